"""What a serving loop needs around the 8-bit cache: attention behind a shared prefix,
the weights that cached tokens receive, eviction by them, and rotary positions of
several axes, on the GPU, against their definitions in 64 bits (tests/_kv8.py,
tests/_kv8_serve.py, which have the bounds). What is moved, and the slots kept, is compared exactly."""
import math

import pytest

import aether_amd as A
from tests import _kv8 as R
from tests import _kv8_serve as S
from tests.test_gpu_kv8 import append, attend, rand, some_layer, stream, within

pytestmark = pytest.mark.gpu


def workspace(torch, need):
    assert need >= 0
    return torch.full((max(need, 16),), 0xFF, dtype=torch.uint8, device="cuda")  # NaN where it is read unwritten


def some_layers(torch, seed, seqs, nkv, hd, max_seq):
    return torch.stack([some_layer(torch, seed + 10 * b, nkv, hd, max_seq) for b in range(seqs)])


def ints(torch, x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ── a shared prefix ───────────────────────────────────────────────────────


def shared(torch, q, prefix, prefix_len, prefix_seq, layers, lens, nkv, hd, max_seq, max_len, window=0, out=None, ws=None):
    L, b, heads = A.lib(), q.shape[0], q.shape[1] // hd
    if ws is None:
        ws = workspace(torch, L.aeth_attn_kv8_shared_ws_bytes(b, heads, nkv, hd, prefix_len, max_len))
    if out is None:
        out = torch.full((b, heads * hd), math.nan, device="cuda")
    A.check(L.aeth_attn_kv8_shared(q.data_ptr(), q.stride(0), prefix.data_ptr() if prefix is not None else None, prefix_seq, prefix_len, layers.data_ptr(),
                                   layers[0].numel(), lens.data_ptr(), b, heads, nkv, hd, max_seq, max_len, window, out.data_ptr(), ws.data_ptr(),
                                   ws.numel(), stream(torch)), "shared")
    return out


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("seqs,prefix_len,lens,nkv,g,window", [
    (1, 1, [1], 1, 1, 0), (1, 64, [0], 2, 4, 0), (2, 65, [0, 1], 2, 3, 0), (3, 0, [5, 0, 70], 2, 4, 0), (2, 1000, [60, 3], 2, 4, 0),
    (17, 300, None, 2, 4, 0), (70, 200, None, 1, 4, 0), (40, 129, None, 2, 7, 0), (5, 640, [1, 64, 65, 130, 40], 1, 17, 0),
    (3, 500, [10, 200, 0], 2, 4, 150), (40, 700, None, 1, 4, 333), (2, 40, [50, 7], 1, 2, 1), (2, 40, [50, 0], 1, 2, 45)])
def test_shared_prefix(gpu, hd, seqs, prefix_len, lens, nkv, g, window):
    torch = gpu
    lens = lens or [(37 * b) % 150 for b in range(seqs)]
    max_len, prefix_seq = max(max(lens), 1), prefix_len + 3
    max_seq = max_len + 5
    prefix = some_layer(torch, 1, nkv, hd, prefix_seq) if prefix_len else None
    layers = some_layers(torch, 50, seqs, nkv, hd, max_seq)
    q = rand(torch, seqs, seqs, nkv * g * hd)
    got = shared(torch, q, prefix, prefix_len, prefix_seq, layers, ints(torch, lens), nkv, hd, max_seq, max_len, window)
    within(torch, got, *S.shared(q, prefix, prefix_len, prefix_seq, layers, lens, nkv, hd, max_seq, window))


@pytest.mark.parametrize("hd,seqs,nkv,g,prefix_len", [(128, 100, 2, 4, 5000), (128, 3, 1, 4, 20000), (64, 64, 1, 8, 6001), (128, 70, 8, 1, 2500), (128, 16, 8, 4, 3000),
                                                           (64, 15, 4, 8, 3000), (256, 16, 4, 4, 2500), (128, 160, 8, 1, 4100)])
def test_shared_prefix_long(gpu, hd, seqs, nkv, g, prefix_len):
    """Many chunks of the prefix, up to 16 parts to join and more, blocks of 16 and 128 columns; the slots behind the prefix and the lengths hold NaN scales."""
    torch = gpu
    lens = [1 + (53 * b) % 300 for b in range(seqs)]
    prefix = some_layer(torch, 1, nkv, hd, prefix_len)
    layers = some_layers(torch, 9, seqs, nkv, hd, 320)
    poison(torch, prefix, nkv, hd, prefix_len, range(prefix_len, -(-prefix_len // 64) * 64))
    for b in range(seqs):
        poison(torch, layers[b], nkv, hd, 320, range(lens[b], 320))
    q = rand(torch, 2, seqs, nkv * g * hd)
    got = shared(torch, q, prefix, prefix_len, prefix_len, layers, ints(torch, lens), nkv, hd, 320, 300)
    within(torch, got, *S.shared(q, prefix, prefix_len, prefix_len, layers, lens, nkv, hd, 320, 0))


@pytest.mark.parametrize("hd,seqs,nkv,g,prefix_len,window", [
    (128, 100, 2, 4, 5000, 3001), (128, 100, 2, 4, 5000, 150), (64, 90, 4, 4, 4001, 2000), (128, 40, 8, 8, 3500, 3333), (256, 40, 1, 4, 1500, 700)])
def test_shared_prefix_long_with_a_window(gpu, hd, seqs, nkv, g, prefix_len, window):
    """Sequences of one block whose windows begin in different tiles of the prefix, and those whose window leaves it; what no window reaches holds NaN scales."""
    torch = gpu
    lens = [(53 * b) % 301 for b in range(seqs)]
    prefix = some_layer(torch, 1, nkv, hd, prefix_len)
    layers = some_layers(torch, 9, seqs, nkv, hd, 320)
    poison(torch, prefix, nkv, hd, prefix_len, range(0, prefix_len - window))
    for b in range(seqs):
        poison(torch, layers[b], nkv, hd, 320, range(lens[b], 320))
    q = rand(torch, 2, seqs, nkv * g * hd)
    got = shared(torch, q, prefix, prefix_len, prefix_len, layers, ints(torch, lens), nkv, hd, 320, 300, window)
    within(torch, got, *S.shared(q, prefix, prefix_len, prefix_len, layers, lens, nkv, hd, 320, window))


def poison(torch, layer, nkv, hd, max_seq, slots, part=2):
    """NaN as the scales of slots: part 0 of K, 1 of V, 2 of both."""
    view = layer.reshape(nkv, -1, 128 * hd + 512)
    for t in slots:
        for p in (0, 1):
            if part in (p, 2):
                at = 128 * hd + 4 * (64 * p + t % 64)
                view[:, t // 64, at:at + 4] = torch.tensor([0, 0, 0xC0, 0x7F], dtype=torch.uint8, device="cuda")


def test_shared_prefix_nan_reaches_those_that_see_it(gpu):
    torch = gpu
    nkv, hd, g, prefix_len, lens = 2, 128, 4, 300, [100, 30, 0, 60]
    layers = some_layers(torch, 3, 4, nkv, hd, 128)
    q = rand(torch, 4, 4, nkv * g * hd)
    for part in (0, 1):
        prefix = some_layer(torch, 1, nkv, hd, 300)
        clean = prefix.clone()
        poison(torch, prefix, nkv, hd, 300, [250], part)
        # window 120: sequence 0 sees the prefix from 280 on, 1 from 210, 2 from 180, 3 from 240
        got = shared(torch, q, prefix, prefix_len, 300, layers, ints(torch, lens), nkv, hd, 128, 100, 120)
        want, bound = S.shared(q, clean, prefix_len, 300, layers, lens, nkv, hd, 128, 120)
        within(torch, got[:1], want[:1], bound[:1])
        assert got[1:].isnan().all()


def test_shared_prefix_takes_strides_and_clamps_lengths(gpu):
    torch = gpu
    nkv, hd, g, seqs = 2, 64, 3, 5
    prefix, layers = some_layer(torch, 1, nkv, hd, 100), some_layers(torch, 2, seqs, nkv, hd, 70)
    q = rand(torch, 3, seqs, nkv * g * hd)
    lens = [70, 1, 20, 33, 64]
    want = shared(torch, q, prefix, 90, 100, layers, ints(torch, lens), nkv, hd, 70, 70)
    for shift, stride in ((0, q.shape[1] + 4), (1, q.shape[1] + 4), (0, q.shape[1] + 1)):
        buf = torch.zeros(seqs * stride + 8, device="cuda")
        rows = torch.as_strided(buf, q.shape, (stride, 1), shift)
        rows.copy_(q)
        out = torch.full((q.numel() + 1,), math.nan, device="cuda")[1:].reshape(q.shape)
        assert torch.equal(shared(torch, rows, prefix, 90, 100, layers, ints(torch, lens), nkv, hd, 70, 70, out=out), want)
    # past max_len, below zero
    wild = shared(torch, q, prefix, 90, 100, layers, ints(torch, [2 ** 31 - 1, 1, -5, 33, 71]), nkv, hd, 70, 70)
    want[2] = shared(torch, q, prefix, 90, 100, layers, ints(torch, [70, 1, 0, 33, 70]), nkv, hd, 70, 70)[2]
    want[4] = shared(torch, q, prefix, 90, 100, layers, ints(torch, [70, 1, 0, 33, 70]), nkv, hd, 70, 70)[4]
    assert torch.equal(wild, want)


def capture(torch, call):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        call()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            call()
    torch.cuda.current_stream().wait_stream(side)
    return graph


def test_shared_prefix_captured(gpu):
    """Two graphs with a workspace each follow the lengths; replays between eager calls, each against the eager result."""
    torch = gpu
    nkv, hd, g, seqs, prefix_len = 2, 128, 4, 20, 700
    prefix, layers = some_layer(torch, 1, nkv, hd, prefix_len), some_layers(torch, 2, seqs, nkv, hd, 200)
    sets = []
    for k in range(2):
        q, lens, out = rand(torch, 7 + k, seqs, nkv * g * hd), ints(torch, [1] * seqs), torch.zeros((seqs, nkv * g * hd), device="cuda")
        ws = workspace(torch, A.lib().aeth_attn_kv8_shared_ws_bytes(seqs, nkv * g, nkv, hd, prefix_len, 200))
        graph = capture(torch, lambda: shared(torch, q, prefix, prefix_len, prefix_len, layers, lens, nkv, hd, 200, 200, out=out, ws=ws))
        sets.append((graph, q, lens, out, ws))
    for step in range(3):
        for k, (graph, q, lens, out, _) in enumerate(sets):
            lens.copy_(ints(torch, [(31 * b + 50 * step + k) % 201 for b in range(seqs)]))
            out.zero_()
        for graph, *_ in sets:
            graph.replay()
        for graph, q, lens, out, _ in sets:
            assert torch.equal(out, shared(torch, q, prefix, prefix_len, prefix_len, layers, lens, nkv, hd, 200, 200))
        torch.cuda.synchronize()


# ── the weights that tokens receive ───────────────────────────────────────


def weigh(torch, q, layer, nkv, hd, max_seq, seq, window=0, prior=None, into=None, ws=None, out=None):
    L, n, heads = A.lib(), q.shape[0], q.shape[1] // hd
    if ws is None:
        ws = workspace(torch, L.aeth_attn_kv8_weights_ws_bytes(1, n, heads, nkv, hd, seq))
    if out is None:
        out = torch.full((n, heads * hd), math.nan, device="cuda")
    if into is None:
        into = torch.full((nkv, max_seq), 7.0, device="cuda")
    A.check(L.aeth_attn_kv8_weights(q.data_ptr(), q.stride(0), layer.data_ptr(), n, heads, nkv, hd, max_seq, seq, window, out.data_ptr(),
                                    prior.data_ptr() if prior is not None else None, into.data_ptr(), ws.data_ptr(), ws.numel(), stream(torch)), "weights")
    return out, into


def weigh_batch(torch, q, layers, lens, nkv, hd, max_seq, max_len, window=0, prior=None, into=None, ws=None, out=None):
    L, b, heads = A.lib(), q.shape[0], q.shape[1] // hd
    if ws is None:
        ws = workspace(torch, L.aeth_attn_kv8_weights_ws_bytes(b, 1, heads, nkv, hd, max_len))
    if out is None:
        out = torch.full((b, heads * hd), math.nan, device="cuda")
    if into is None:
        into = torch.full((b, nkv, max_seq), 7.0, device="cuda")
    A.check(L.aeth_attn_kv8_weights_batch(q.data_ptr(), q.stride(0), layers.data_ptr(), layers[0].numel(), lens.data_ptr(), b, heads, nkv, hd, max_seq,
                                          max_len, window, out.data_ptr(), prior.data_ptr() if prior is not None else None, into.data_ptr(),
                                          ws.data_ptr(), ws.numel(), stream(torch)), "weights batch")
    return out, into


def check_weights(torch, got, want, nkv, seq):
    (out, w), (o, ot, ww, wt) = got, want
    within(torch, out, o, ot)
    within(torch, w[:, :seq], ww, wt)
    assert (w[:, seq:] == 7.0).all()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n,seq,nkv,g,window", [
    (1, 1, 1, 1, 0), (1, 64, 2, 4, 0), (1, 65, 2, 3, 0), (1, 1500, 2, 4, 0), (1, 700, 1, 17, 0), (1, 900, 2, 4, 100), (4, 300, 2, 4, 0), (7, 333, 2, 7, 50),
    (16, 16, 2, 4, 0), (17, 17, 1, 4, 0), (64, 1000, 1, 1, 0), (65, 800, 2, 1, 0), (33, 257, 2, 4, 0), (200, 200, 2, 4, 0), (130, 1025, 1, 8, 0),
    (150, 400, 2, 3, 1), (300, 300, 1, 4, 70), (40, 2000, 2, 4, 700), (256, 513, 1, 2, 0)])
def test_weights(gpu, hd, n, seq, nkv, g, window):
    torch = gpu
    max_seq = seq + 9
    layer = some_layer(torch, n, nkv, hd, max_seq)
    poison(torch, layer, nkv, hd, max_seq, range(seq, max_seq))
    q = rand(torch, seq, n, nkv * g * hd)
    check_weights(torch, weigh(torch, q, layer, nkv, hd, max_seq, seq, window), S.weights(q, layer, nkv, hd, max_seq, seq, window, None), nkv, seq)
    prior = rand(torch, 5, nkv, max_seq).abs()
    want = S.weights(q, layer, nkv, hd, max_seq, seq, window, prior)
    check_weights(torch, weigh(torch, q, layer, nkv, hd, max_seq, seq, window, prior), want, nkv, seq)
    # in place
    kept = prior.clone()
    prior[:, seq:] = 7.0
    check_weights(torch, weigh(torch, q, layer, nkv, hd, max_seq, seq, window, prior, into=prior), S.weights(q, layer, nkv, hd, max_seq, seq, window, kept), nkv,
                  seq)


@pytest.mark.parametrize("hd,n,seq,nkv,g", [(128, 1, 30000, 2, 4), (64, 500, 3000, 2, 4), (128, 1000, 1000, 2, 4)])
def test_weights_long(gpu, hd, n, seq, nkv, g):
    torch = gpu
    layer = some_layer(torch, n, nkv, hd, seq)
    q = rand(torch, seq, n, nkv * g * hd)
    out, w = weigh(torch, q, layer, nkv, hd, seq, seq)
    o, ot, ww, wt = S.weights(q, layer, nkv, hd, seq, seq, 0, None)
    within(torch, out, o, ot)
    within(torch, w, ww, wt)
    again = weigh(torch, q, layer, nkv, hd, seq, seq)
    assert torch.equal(again[0], out) and torch.equal(again[1], w)


@pytest.mark.parametrize("hd,n,seq,nkv,g,window", [
    (128, 60, 9000, 2, 4, 900), (64, 60, 9000, 2, 1, 5), (256, 40, 6000, 1, 4, 1000), (128, 900, 5000, 2, 4, 1500), (64, 300, 7000, 1, 8, 6950),
    (128, 700, 4200, 8, 4, 1)])
def test_weights_of_a_long_cache_with_a_window(gpu, hd, n, seq, nkv, g, window):
    """The columns of a group of keys in one chunk and in several; keys before every window, with NaN scales, keep their prior."""
    torch = gpu
    layer = some_layer(torch, n, nkv, hd, seq)
    poison(torch, layer, nkv, hd, seq, range(0, max(0, seq - n + 1 - window)))
    q = rand(torch, seq, n, nkv * g * hd)
    prior = rand(torch, 5, nkv, seq).abs()
    out, w = weigh(torch, q, layer, nkv, hd, seq, seq, window, prior)
    o, ot, ww, wt = S.weights(q, layer, nkv, hd, seq, seq, window, prior)
    within(torch, out, o, ot)
    within(torch, w, ww, wt)
    dark = max(0, seq - n + 1 - window)
    assert torch.equal(w[:, :dark], prior[:, :dark])


@pytest.mark.parametrize("hd,nkv,g,lens,max_seq,max_len,window", [
    (128, 2, 4, [1, 0, 64, 65, 300], 310, 300, 0), (64, 1, 8, [5, 700, 1, 699], 700, 700, 0), (128, 2, 3, [50, 400, 129], 410, 400, 60),
    (256, 1, 20, [70, 3], 80, 70, 0), (128, 8, 4, [100 + 61 * i for i in range(24)], 1600, 1503, 0), (64, 1, 70, [90, 200], 200, 200, 0),
    (64, 16, 2, [(37 * i) % 301 for i in range(65)], 310, 300, 0), (128, 16, 3, [5000, 1, 700, 4999, 0, 2048, 3333], 5001, 5000, 700)])
def test_weights_batch(gpu, hd, nkv, g, lens, max_seq, max_len, window):
    torch = gpu
    b = len(lens)
    layers = some_layers(torch, 3, b, nkv, hd, max_seq)
    q = rand(torch, 4, b, nkv * g * hd)
    prior = rand(torch, 5, b, nkv, max_seq).abs()
    for before in (None, prior):
        out, w = weigh_batch(torch, q, layers, ints(torch, lens), nkv, hd, max_seq, max_len, window, before)
        for i, seq in enumerate(lens):
            want = S.weights(q[i:i + 1] if seq else q[:0], layers[i], nkv, hd, max_seq, seq, window, None if before is None else before[i])
            if seq == 0:
                assert (out[i] == 0).all() and (w[i] == 7.0).all()
            else:
                check_weights(torch, (out[i:i + 1], w[i]), want, nkv, seq)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n,seq,window", [(1, 700, 0), (3, 700, 100), (90, 700, 0), (90, 700, 33)])
def test_weights_take_strides_and_any_alignment(gpu, hd, n, seq, window):
    torch = gpu
    nkv, g, max_seq = 2, 4, 701
    layer = some_layer(torch, n, nkv, hd, max_seq)
    wide = rand(torch, seq, n, nkv * g * hd + 7)
    q = wide[:, 3:3 + nkv * g * hd]
    out = torch.full((n * nkv * g * hd + 1,), math.nan, device="cuda")[1:].view(n, -1)
    prior = rand(torch, 5, nkv * max_seq + 1).abs()[1:].view(nkv, max_seq)
    into = torch.full((nkv * max_seq + 3,), 7.0, device="cuda")[3:].view(nkv, max_seq)
    got = weigh(torch, q, layer, nkv, hd, max_seq, seq, window, prior, into, out=out)
    check_weights(torch, got, S.weights(q.contiguous(), layer, nkv, hd, max_seq, seq, window, prior), nkv, seq)


def test_weights_without_queries_are_the_prior(gpu):
    torch = gpu
    layer, prior = some_layer(torch, 1, 2, 128, 100), rand(torch, 2, 2, 100)
    q = torch.empty((0, 8 * 128), device="cuda")
    _, w = weigh(torch, q, layer, 2, 128, 100, 70, prior=prior, out=torch.zeros(16, device="cuda"))
    assert torch.equal(w[:, :70], prior[:, :70]) and (w[:, 70:] == 7.0).all()
    _, w = weigh(torch, q, layer, 2, 128, 100, 70, out=torch.zeros(16, device="cuda"))
    assert (w[:, :70] == 0).all() and (w[:, 70:] == 7.0).all()


@pytest.mark.parametrize("n", [1, 40, 100])
def test_weights_of_a_nan_row(gpu, n):
    """A NaN in one query: its row and the weights of what it sees; the other KV head's are numbers."""
    torch = gpu
    nkv, hd, g, seq = 2, 128, 4, 500
    layer = some_layer(torch, 1, nkv, hd, seq)
    q = rand(torch, 2, n, nkv * g * hd)
    q[0, 5] = math.nan
    window = 200
    out, w = weigh(torch, q, layer, nkv, hd, seq, seq, window)
    first, end = max(0, seq - n + 1 - window), seq - n + 1
    assert out[0, :hd].isnan().all() and not out[:, g * hd:].isnan().any() and not out[1:].isnan().any()
    assert w[0, first:end].isnan().all() and not w[0, :first].isnan().any() and not w[0, end:].isnan().any() and not w[1].isnan().any()


def test_weights_captured(gpu):
    """A decode step's and a chunk's graph, replayed over other inputs between eager calls."""
    torch = gpu
    nkv, hd, g, max_seq = 2, 128, 4, 1500
    layers = some_layers(torch, 3, 3, nkv, hd, max_seq)
    q, lens = rand(torch, 4, 3, nkv * g * hd), ints(torch, [3, 2, 1])
    out, w = torch.zeros_like(q), torch.zeros((3, nkv, max_seq), device="cuda")
    ws = workspace(torch, A.lib().aeth_attn_kv8_weights_ws_bytes(3, 1, nkv * g, nkv, hd, max_seq))
    step = capture(torch, lambda: weigh_batch(torch, q, layers, lens, nkv, hd, max_seq, max_seq, into=w, out=out, ws=ws))
    q2 = rand(torch, 6, 100, nkv * g * hd)
    out2, w2 = torch.zeros_like(q2), torch.zeros((nkv, max_seq), device="cuda")
    ws2 = workspace(torch, A.lib().aeth_attn_kv8_weights_ws_bytes(1, 100, nkv * g, nkv, hd, 900))
    chunk = capture(torch, lambda: weigh(torch, q2, layers[1], nkv, hd, max_seq, 900, into=w2, out=out2, ws=ws2))
    for k in range(3):
        lens.copy_(ints(torch, [1 + 700 * k, 1500 - k, 64 * k]))
        q2.copy_(rand(torch, 60 + k, 100, nkv * g * hd))
        for x in (w, w2):
            x.fill_(7.0)
        step.replay()
        chunk.replay()
        for got, want in zip((out, w, out2, w2), weigh_batch(torch, q, layers, lens, nkv, hd, max_seq, max_seq) + weigh(torch, q2, layers[1], nkv, hd, max_seq, 900)):
            assert torch.equal(got, want)
        torch.cuda.synchronize()


# ── eviction ──────────────────────────────────────────────────────────────


def evict(torch, layer, weights, nkv, hd, max_seq, seq, keep, first, recent, dst=None, dst_seq=None, dst_weights=None, kept=True):
    L, in_place = A.lib(), dst is None
    dst, dst_seq = (layer, max_seq) if in_place else (dst, dst_seq)
    listed = torch.full((nkv, keep), -7, dtype=torch.int32, device="cuda") if kept else None
    ws = workspace(torch, L.aeth_kv8_evict_ws_bytes(1, nkv, hd, seq, keep, int(in_place)))
    A.check(L.aeth_kv8_evict(layer.data_ptr(), weights.data_ptr(), nkv, hd, max_seq, seq, keep, first, recent, dst.data_ptr(),
                             dst_weights.data_ptr() if dst_weights is not None else None, dst_seq, listed.data_ptr() if kept else None, ws.data_ptr(),
                             ws.numel(), stream(torch)), "evict")
    return listed


def evict_batch(torch, layers, weights, lens, nkv, hd, max_seq, max_len, keep, first, recent, dst, dst_seq, dst_weights, dst_lens, kept, ws=None):
    L, b = A.lib(), layers.shape[0]
    if ws is None:
        ws = workspace(torch, L.aeth_kv8_evict_ws_bytes(b, nkv, hd, max_len, keep, int(dst is layers)))
    A.check(L.aeth_kv8_evict_batch(layers.data_ptr(), layers[0].numel(), weights.data_ptr(), lens.data_ptr(), b, nkv, hd, max_seq, max_len, keep, first,
                                   recent, dst.data_ptr(), dst[0].numel(), dst_weights.data_ptr() if dst_weights is not None else None, dst_seq,
                                   dst_lens.data_ptr() if dst_lens is not None else None, kept.data_ptr() if kept is not None else None, ws.data_ptr(),
                                   ws.numel(), stream(torch)), "evict batch")


def check_evicted(torch, src, weights, before, after, after_weights, kept, nkv, hd, max_seq, seq, keep, first, recent, dst_seq):
    """src, weights: as they were; before, after: the destination's bytes."""
    s, b, a = R.unpack(src, nkv, hd, max_seq), R.unpack(before, nkv, hd, dst_seq), R.unpack(after, nkv, hd, dst_seq)
    want = [x.clone() for x in b]
    rows = min(seq, keep)
    for h in range(nkv):
        slots = S.evicted(weights[h].tolist(), seq, keep, first, recent)
        at = torch.tensor(slots, dtype=torch.long, device="cuda")
        for x, y in zip(want, s):
            x[h, :rows] = y[h, at]
        if kept is not None:
            assert kept[h, :rows].tolist() == slots
            assert (kept[h, rows:] == -7).all()
        if after_weights is not None:
            assert torch.equal(after_weights[h, :rows].view(torch.int32), weights[h, at].view(torch.int32))
            assert (after_weights[h, rows:] == 0).all()
    for x, y in zip(a, want):
        assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))


def uneven(torch, seed, *shape):
    """Weights with many equal ones, zeros of both signs, infinities and NaN."""
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(2 * torch.randn(shape, generator=g))
    pick = torch.randint(0, 12, shape, generator=g)
    for i, v in enumerate((0.0, -0.0, 1.0, 1.0, math.inf, math.nan, -1.0, -math.inf)):
        w = torch.where(pick == i, torch.tensor(v), w)
    return w.cuda()


EVICTIONS = [(1, 1, 0, 0), (1, 0, 0, 0), (2, 1, 1, 0), (2, 1, 0, 1), (2, 1, 0, 0), (64, 63, 4, 10), (65, 64, 0, 0), (200, 64, 64, 0), (200, 64, 0, 64), (200, 65, 4, 61),
             (200, 130, 3, 20), (333, 300, 4, 100), (333, 333, 4, 100), (333, 400, 4, 100), (1000, 17, 0, 1), (5000, 2500, 4, 64), (4097, 4096, 0, 0),
             (0, 5, 1, 1)]


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("seq,keep,first,recent", EVICTIONS)
def test_evict(gpu, hd, seq, keep, first, recent):
    torch = gpu
    nkv, max_seq, dst_seq = 3, seq + 11, keep + 70
    layer, weights = some_layer(torch, seq, nkv, hd, max_seq), uneven(torch, keep, nkv, max_seq)
    src = layer.clone()
    dst = torch.full(R.layer_shape(nkv, hd, dst_seq), 0xA5, dtype=torch.uint8, device="cuda")
    dst_weights = torch.full((nkv, dst_seq), math.nan, device="cuda")
    before = dst.clone()
    kept = evict(torch, layer, weights, nkv, hd, max_seq, seq, keep, first, recent, dst, dst_seq, dst_weights)
    assert torch.equal(layer, src)
    check_evicted(torch, src, weights, before, dst, dst_weights, kept, nkv, hd, max_seq, seq, keep, first, recent, dst_seq)
    # in place, the weights too; and with neither weights nor slots wanted
    was = weights.clone()
    kept = evict(torch, layer, weights, nkv, hd, max_seq, seq, keep, first, recent, dst_weights=weights)
    check_evicted(torch, src, was, src, layer, weights, kept, nkv, hd, max_seq, seq, keep, first, recent, max_seq)
    layer = src.clone()
    evict(torch, layer, was, nkv, hd, max_seq, seq, keep, first, recent, kept=False)
    check_evicted(torch, src, was, src, layer, None, None, nkv, hd, max_seq, seq, keep, first, recent, max_seq)


@pytest.mark.parametrize("seq,keep", [(131000, 3000), (70000, 60001), (9000, 8191)])
def test_evict_long(gpu, seq, keep):
    torch = gpu
    nkv, hd = 2, 64
    layer = some_layer(torch, seq, nkv, hd, seq)
    src = layer.clone()
    for weights in (torch.rand((nkv, seq), generator=torch.Generator().manual_seed(1)).cuda(), torch.zeros((nkv, seq), device="cuda"), uneven(torch, 3, nkv, seq)):
        layer.copy_(src)
        was = weights.clone()
        kept = evict(torch, layer, weights, nkv, hd, seq, seq, keep, 4, 100, dst_weights=weights)
        check_evicted(torch, src, was, src, layer, weights, kept, nkv, hd, seq, seq, keep, 4, 100, seq)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_batch(gpu, hd, in_place):
    torch = gpu
    nkv, max_seq, keep, first, recent = 2, 700, 200, 4, 30
    lens = [700, 0, 200, 201, 1, 650, 333, 199]
    b = len(lens)
    layers, weights = some_layers(torch, 1, b, nkv, hd, max_seq), uneven(torch, 2, b, nkv, max_seq)
    src, was = layers.clone(), weights.clone()
    kept = torch.full((b, nkv, keep), -7, dtype=torch.int32, device="cuda")
    d_lens = ints(torch, lens)
    if in_place:
        dst, dst_seq, dst_weights, dst_lens = layers, max_seq, weights, d_lens
    else:
        dst_seq = 256
        dst = torch.full((b,) + R.layer_shape(nkv, hd, dst_seq), 0xA5, dtype=torch.uint8, device="cuda")
        dst_weights, dst_lens = torch.full((b, nkv, dst_seq), math.nan, device="cuda"), ints(torch, [-1] * b)
    before = dst.clone()
    evict_batch(torch, layers, weights, d_lens, nkv, hd, max_seq, max_seq, keep, first, recent, dst, dst_seq, dst_weights, dst_lens, kept)
    assert dst_lens.tolist() == [min(l, keep) for l in lens]
    for i, seq in enumerate(lens):
        check_evicted(torch, src[i], was[i], before[i], dst[i], dst_weights[i], kept[i], nkv, hd, max_seq, seq, keep, first, recent, dst_seq)
    if not in_place:
        assert torch.equal(layers, src) and d_lens.tolist() == lens
        # past max_len, below zero
        wild = ints(torch, [2 ** 31 - 1, -3] + lens[2:])
        evict_batch(torch, layers, weights, wild, nkv, hd, max_seq, 700, keep, first, recent, dst, dst_seq, dst_weights, dst_lens, kept)
        assert dst_lens.tolist() == [min(l, keep) for l in lens]
        check_evicted(torch, src[0], was[0], before[0], dst[0], dst_weights[0], kept[0], nkv, hd, max_seq, 700, keep, first, recent, dst_seq)


@pytest.mark.parametrize("keep,first,recent", [(3000, 4, 100), (0, 0, 0), (500, 200, 300), (40000, 0, 0), (1, 0, 0)])
def test_evict_batch_of_many_tokens(gpu, keep, first, recent):
    """Lengths at the borders of what one workgroup holds and of the chunks of many, next to short ones; new lengths in the old ones' place."""
    torch = gpu
    nkv, hd, max_seq = 1, 64, 70000
    lens = [70000, 0, 32768, 32769, 100, 40960, 40961, keep, keep + 1]
    b = len(lens)
    layers = some_layer(torch, 1, b * nkv, hd, max_seq).reshape((b,) + R.layer_shape(nkv, hd, max_seq))
    weights = uneven(torch, keep, b, nkv, max_seq)
    weights[5] = 0.25  # all equal
    weights[0, 0, 5000:] = 1.0 + 2.0 ** -20 * torch.rand(65000, generator=torch.Generator().manual_seed(2)).cuda()  # alike in their first bits
    src, was, d_lens = layers.clone(), weights.clone(), ints(torch, lens)
    kept = torch.full((b, nkv, max(keep, 1)), -7, dtype=torch.int32, device="cuda")
    evict_batch(torch, layers, weights, d_lens, nkv, hd, max_seq, max_seq, keep, first, recent, layers, max_seq, weights, d_lens, kept)
    assert d_lens.tolist() == [min(l, keep) for l in lens]
    for i, seq in enumerate(lens):
        check_evicted(torch, src[i], was[i], src[i], layers[i], weights[i], kept[i] if keep else None, nkv, hd, max_seq, seq, keep, first, recent, max_seq)


def test_evict_captured(gpu):
    torch = gpu
    nkv, hd, max_seq, keep, b = 2, 128, 500, 100, 4
    layers = some_layers(torch, 1, b, nkv, hd, max_seq)
    weights, lens = uneven(torch, 2, b, nkv, max_seq), ints(torch, [500, 400, 300, 50])
    dst = torch.zeros((b,) + R.layer_shape(nkv, hd, 128), dtype=torch.uint8, device="cuda")
    dw, dl, kept = torch.zeros((b, nkv, 128), device="cuda"), ints(torch, [0] * b), torch.full((b, nkv, keep), -7, dtype=torch.int32, device="cuda")
    ws = workspace(torch, A.lib().aeth_kv8_evict_ws_bytes(b, nkv, hd, max_seq, keep, 0))
    graph = capture(torch, lambda: evict_batch(torch, layers, weights, lens, nkv, hd, max_seq, max_seq, keep, 2, 10, dst, 128, dw, dl, kept, ws))
    for k in range(3):
        weights.copy_(uneven(torch, 20 + k, b, nkv, max_seq))
        now = [500 - 99 * k, 100 + k, 7 * k, 450]
        lens.copy_(ints(torch, now))
        kept.fill_(-7)
        before = dst.clone()
        graph.replay()
        for i, seq in enumerate(now):
            check_evicted(torch, layers[i], weights[i], before[i], dst[i], dw[i], kept[i], nkv, hd, max_seq, seq, keep, 2, 10, 128)
        torch.cuda.synchronize()


# ── positions of several axes ─────────────────────────────────────────────


def axes_rope(torch, x, nq, nk, hd, qw, kw, pos, pair_axes, sin, cos, out=None, eps=1e-5):
    axes = torch.tensor(pair_axes, dtype=torch.int32)
    n = x.shape[0]
    if out is None:
        out = torch.full((n, (nq + nk) * hd), math.nan, device="cuda")
    A.check(A.lib().aeth_qk_norm_rope_axes(x.data_ptr(), x.stride(0), n, nq, nk, hd, qw.data_ptr() if qw is not None else None,
                                           kw.data_ptr() if kw is not None else None, eps, pos.data_ptr(), pos.stride(0), pos.shape[0], axes.data_ptr(),
                                           sin.data_ptr(), cos.data_ptr(), sin.shape[0], out.data_ptr(), out.stride(0), stream(torch)), "axes")
    axes.fill_(-1)  # read before the call returned
    return out


def axes_exact(x, nq, nk, hd, qw, kw, pos, pair_axes, sin, cos, eps=1e-5):
    """R.qk_norm_rope with a table row for each token and pair, as tables of one row a token."""
    import torch

    at = pos[torch.tensor(pair_axes, device="cuda")].clamp(0, sin.shape[0] - 1).long().t()  # [n][pairs]
    s, c = torch.gather(sin, 0, at), torch.gather(cos, 0, at)
    return R.qk_norm_rope(x, nq, nk, hd, qw, kw, eps, torch.arange(x.shape[0], device="cuda"), s, c)


def table(torch, rows, hd):
    a = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64) / hd)
    return a.sin().float().cuda(), a.cos().float().cuda()


@pytest.mark.parametrize("hd", [2, 64, 80, 128, 256, 512])
@pytest.mark.parametrize("n,nq,nk,axes,norm", [(1, 4, 2, 3, "qk"), (5, 3, 1, 1, ""), (67, 8, 8, 3, "q"), (9, 1, 0, 16, "k"), (33, 2, 2, 4, "qk")])
def test_axes(gpu, hd, n, nq, nk, axes, norm):
    torch = gpu
    g = torch.Generator().manual_seed(hd + n)
    x = rand(torch, n, n, (nq + nk + 1) * hd)
    qw, kw = (rand(torch, 7, hd) if c in norm else None for c in "qk")
    pos = torch.randint(-3, 130, (axes, n), generator=g, dtype=torch.int32).cuda()  # the table has 100 rows
    pairs = torch.randint(0, axes, (hd // 2,), generator=g).tolist()
    sin, cos = table(torch, 100, hd)
    want, bound = axes_exact(x, nq, nk, hd, qw, kw, pos, pairs, sin, cos)
    within(torch, axes_rope(torch, x, nq, nk, hd, qw, kw, pos, pairs, sin, cos), want, bound)
    # positions further apart than n, rows out of line, in place
    wide = torch.full((axes, n + 3), 99, dtype=torch.int32, device="cuda")
    wide[:, :n] = pos
    buf = torch.zeros(n * (x.shape[1] + 1) + 1, device="cuda")
    rows = torch.as_strided(buf, x.shape, (x.shape[1] + 1, 1), 1)
    rows.copy_(x)
    axes_rope(torch, rows, nq, nk, hd, qw, kw, wide, pairs, sin, cos, out=rows)
    within(torch, rows[:, :(nq + nk) * hd], want, bound)
    assert torch.equal(rows[:, (nq + nk) * hd:], x[:, (nq + nk) * hd:])


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
def test_axes_that_agree_are_one(gpu, hd):
    torch = gpu
    n, nq, nk = 50, 4, 2
    x, qw, kw = rand(torch, 1, n, (nq + nk) * hd), rand(torch, 2, hd), rand(torch, 3, hd)
    sin, cos = table(torch, 200, hd)
    pos = ints(torch, [(7 * i) % 211 for i in range(n)])
    want = torch.empty_like(x)
    A.check(A.lib().aeth_qk_norm_rope(x.data_ptr(), x.shape[1], n, nq, nk, hd, qw.data_ptr(), kw.data_ptr(), 1e-5, 0, pos.data_ptr(), sin.data_ptr(),
                                      cos.data_ptr(), 200, want.data_ptr(), x.shape[1], stream(torch)), "rope")
    got = axes_rope(torch, x, nq, nk, hd, qw, kw, pos.expand(3, n).contiguous(), [j % 3 for j in range(hd // 2)], sin, cos)
    assert torch.equal(got, want)


# ── together ──────────────────────────────────────────────────────────────


def test_a_prompt_weighed_evicted_and_served_behind_a_prefix(gpu):
    """A prompt with an image's positions is appended and attended in two calls, the second of which weighs its tokens; each of three
    sequences' caches is cut to a short one; a decode step appends a token there, weighs again, evicts in place, and attends behind
    a shared prefix. Every step against 64 bits on what the step before left."""
    torch = gpu
    nkv, g, hd, n, tail, keep = 2, 4, 128, 300, 32, 120
    heads, b = nkv * g, 3
    sin, cos = table(torch, 512, hd)
    pairs = [0] * 16 + [1] * 24 + [2] * 24
    i = torch.arange(n, device="cuda")
    pos = torch.stack([torch.where(i < 100, i, 100 + a) for a in (0 * i, i // 20 % 10, i % 20)]).to(torch.int32).contiguous()
    short, short_w = torch.zeros((b,) + R.layer_shape(nkv, hd, 128), dtype=torch.uint8, device="cuda"), torch.zeros((b, nkv, 128), device="cuda")
    for s in range(b):
        x = rand(torch, s, n, (heads + 2 * nkv) * hd)
        qk = axes_rope(torch, x, heads, nkv, hd, None, None, pos, pairs, sin, cos)
        within(torch, qk, *axes_exact(x, heads, nkv, hd, None, None, pos, pairs, sin, cos))
        layer = torch.full(R.layer_shape(nkv, hd, n), 0xA5, dtype=torch.uint8, device="cuda")
        k, v = qk[:, heads * hd:].contiguous(), x[:, (heads + nkv) * hd:].contiguous()
        append(torch, layer, k, v, nkv, hd, n, 0)
        q = qk[:, :heads * hd].contiguous()
        within(torch, attend(torch, q[:n - tail], layer, nkv, hd, n, n - tail), *R.attention(q[:n - tail], layer, nkv, hd, n, n - tail, 0))
        out, w = weigh(torch, q[n - tail:], layer, nkv, hd, n, n)
        check_weights(torch, (out, w), S.weights(q[n - tail:], layer, nkv, hd, n, n, 0, None), nkv, n)
        before = short[s].clone()
        kept = evict(torch, layer, w, nkv, hd, n, n, keep, 4, 32, short[s], 128, short_w[s])
        check_evicted(torch, layer, w, before, short[s], short_w[s], kept, nkv, hd, n, n, keep, 4, 32, 128)
    x = rand(torch, 77, b, (heads + 2 * nkv) * hd)
    where = torch.full((3, b), 130, dtype=torch.int32, device="cuda")
    qk = axes_rope(torch, x, heads, nkv, hd, None, None, where, pairs, sin, cos)
    k, v, q = qk[:, heads * hd:].contiguous(), x[:, (heads + nkv) * hd:].contiguous(), qk[:, :heads * hd].contiguous()
    A.check(A.lib().aeth_kv8_append_batch(short.data_ptr(), short[0].numel(), ints(torch, [keep] * b).data_ptr(), k.data_ptr(), v.data_ptr(), nkv * hd, hd, b, nkv,
                                          hd, 128, stream(torch)), "append batch")
    lens, prior = ints(torch, [keep + 1] * b), short_w.clone()
    out, _ = weigh_batch(torch, q, short, lens, nkv, hd, 128, keep + 1, prior=short_w, into=short_w)
    for s in range(b):
        o, ot, ww, wt = S.weights(q[s:s + 1], short[s], nkv, hd, 128, keep + 1, 0, prior[s])
        within(torch, out[s:s + 1], o, ot)
        within(torch, short_w[s, :, :keep + 1], ww, wt)
    was, weighed = short.clone(), short_w.clone()
    kept = torch.full((b, nkv, 90), -7, dtype=torch.int32, device="cuda")
    evict_batch(torch, short, short_w, lens, nkv, hd, 128, keep + 1, 90, 4, 16, short, 128, short_w, lens, kept)
    for s in range(b):
        check_evicted(torch, was[s], weighed[s], was[s], short[s], short_w[s], kept[s], nkv, hd, 128, keep + 1, 90, 4, 16, 128)
    prefix = some_layer(torch, 5, nkv, hd, 400)
    got = shared(torch, q, prefix, 400, 400, short, lens, nkv, hd, 128, 128)
    within(torch, got, *S.shared(q, prefix, 400, 400, short, [90] * b, nkv, hd, 128, 0))
