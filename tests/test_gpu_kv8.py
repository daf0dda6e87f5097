"""The 8-bit key/value cache, the attention over it and the head norms with the
rotation, on the GPU, against their definitions in 64 bits (tests/_kv8.py, which
also has the bounds). Codes, scales and untouched bytes are compared exactly."""
import math

import pytest

import aether_amd as A
from tests import _kv8 as R

pytestmark = pytest.mark.gpu


def stream(torch):
    return torch.cuda.current_stream().cuda_stream


def new_layer(torch, nkv, hd, max_seq, seqs=None):
    shape = R.layer_shape(nkv, hd, max_seq)
    shape = shape if seqs is None else (seqs,) + shape
    return torch.full(shape, 0xA5, dtype=torch.uint8, device="cuda")


def append(torch, layer, k, v, nkv, hd, max_seq, slot, ts=None, hs=None, n=None):
    A.check(A.lib().aeth_kv8_append(layer.data_ptr(), k.data_ptr(), v.data_ptr(), nkv * hd if ts is None else ts, hd if hs is None else hs,
                                    k.shape[0] if n is None else n, nkv, hd, max_seq, slot, stream(torch)), "append")


def attend(torch, q, layer, nkv, hd, max_seq, seq, window=0, ws=None):
    L, n, heads = A.lib(), q.shape[0], q.shape[1] // hd
    need = L.aeth_attn_kv8_ws_bytes(1, n, heads, nkv, hd, seq)
    if ws is None:
        ws = torch.full((max(need, 16),), 0xFF, dtype=torch.uint8, device="cuda")  # NaN where it is read unwritten
    out = torch.full((n, heads * hd), math.nan, device="cuda")
    A.check(L.aeth_attn_kv8(q.data_ptr(), q.stride(0), layer.data_ptr(), n, heads, nkv, hd, max_seq, seq, window, out.data_ptr(),
                            ws.data_ptr(), ws.numel(), stream(torch)), "attn")
    return out


def attend_batch(torch, q, layers, lens, nkv, hd, max_seq, max_len, window=0, out=None, ws=None):
    L, b, heads = A.lib(), q.shape[0], q.shape[1] // hd
    if ws is None:
        ws = torch.full((max(L.aeth_attn_kv8_ws_bytes(b, 1, heads, nkv, hd, max_len), 16),), 0xFF, dtype=torch.uint8, device="cuda")
    if out is None:
        out = torch.full((b, heads * hd), math.nan, device="cuda")
    A.check(L.aeth_attn_kv8_batch(q.data_ptr(), q.stride(0), layers.data_ptr(), layers[0].numel(), lens.data_ptr(), b, heads, nkv, hd, max_seq,
                                  max_len, window, out.data_ptr(), ws.data_ptr(), ws.numel(), stream(torch)), "attn batch")
    return out


def rand(torch, seed, *shape):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    x[..., ::13] *= 3.0
    return x.cuda()


def within(torch, got, want, bound):
    far = (got.double() - want).abs()
    bad = ~(far <= bound)
    assert not bad.any(), "%d of %d off, the worst %.3g times its bound" % (int(bad.sum()), bad.numel(), float((far / bound).nan_to_num(1e30).max()))


def some_layer(torch, seed, nkv, hd, max_seq):
    slots = -(-max_seq // 64) * 64
    kc, ks = R.codes(rand(torch, seed, nkv, slots, hd))
    vc, vs = R.codes(rand(torch, seed + 1, nkv, slots, hd))
    return R.pack(kc, ks, vc, vs)


# ── writing and reading back ──────────────────────────────────────────────


def check_stored(torch, layer, k, v, nkv, hd, max_seq, slot):
    """Slots slot .. + n hold the codes and scales of k, v; all else is as it was (0xA5)."""
    want = R.unpack(new_layer(torch, nkv, hd, max_seq), nkv, hd, max_seq)
    n = k.shape[0]
    for x, c, s in ((k, want[0], want[2]), (v, want[1], want[3])):
        xc, xs = R.codes(x.reshape(n, nkv, hd).transpose(0, 1))
        c[:, slot:slot + n], s[:, slot:slot + n] = xc, xs
    for g, w in zip(R.unpack(layer, nkv, hd, max_seq), want):
        assert torch.equal(g.contiguous().view(torch.uint8), w.contiguous().view(torch.uint8))


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n,slot,max_seq,nkv", [(1, 0, 1, 1), (1, 63, 64, 3), (1, 64, 65, 8), (7, 61, 100, 2), (64, 64, 192, 2), (65, 63, 128, 1),
                                                (200, 37, 256, 5)])
def test_append_writes_codes_and_nothing_else(gpu, hd, n, slot, max_seq, nkv):
    torch = gpu
    k, v = rand(torch, n + hd, n, nkv * hd), rand(torch, n + hd + 1, n, nkv * hd)
    layer = new_layer(torch, nkv, hd, max_seq)
    append(torch, layer, k, v, nkv, hd, max_seq, slot)
    check_stored(torch, layer, k, v, nkv, hd, max_seq, slot)
    # and back, into rows with a gap between tokens, unaligned
    back = torch.full((2, n * (nkv * hd + 5) + 1), 7.0, device="cuda")
    A.check(A.lib().aeth_kv8_read(layer.data_ptr(), back[0, 1:].data_ptr(), back[1, 1:].data_ptr(), nkv * hd + 5, hd, n, nkv, hd, max_seq, slot,
                                  stream(torch)), "read")
    for x, b in zip((k, v), back):
        c, s = R.codes(x.reshape(n, nkv, hd))
        rows = b[1:].reshape(n, nkv * hd + 5)
        assert torch.equal(rows[:, :nkv * hd].reshape(n, nkv, hd), c.float() * s[..., None])
        assert (rows[:, nkv * hd:] == 7.0).all() and b[0] == 7.0


def test_append_takes_any_strides(gpu):
    """Rows as a fused projection leaves them, and as the f32 cache holds them ([heads][slots][hd]); an odd start."""
    torch = gpu
    nkv, hd, n, max_seq = 4, 128, 70, 128
    x = rand(torch, 3, 2, n, nkv, hd)
    for ts, hs, shift in ((12 * hd, hd, 0), (hd, 90 * hd, 0), (12 * hd + 1, hd, 0), (12 * hd, hd + 3, 1)):
        buf = torch.zeros((2, (n - 1) * ts + (nkv - 1) * hs + hd + shift), device="cuda")
        for b, y in zip(buf, x):
            torch.as_strided(b, (n, nkv, hd), (ts, hs, 1), b.storage_offset() + shift).copy_(y)
        layer = new_layer(torch, nkv, hd, max_seq)
        append(torch, layer, buf[0, shift:], buf[1, shift:], nkv, hd, max_seq, 5, ts, hs, n)
        check_stored(torch, layer, x[0].reshape(n, -1), x[1].reshape(n, -1), nkv, hd, max_seq, 5)


def test_append_of_values_at_a_border(gpu):
    """Ties of 127·x/amax (to even), of amax that divide 127 and that do not, f32 neighbours of ties, the smallest
    and largest numbers."""
    torch = gpu
    hd, rows = 128, []
    for amax in (127.0, 254.0, 381.0, 1.0, 3.0, 2.0 ** -140, 2.0 ** 127, 1e-45, 1.1754944e-38, 0.7, 3.3e38):
        i = torch.arange(hd, dtype=torch.float64)
        near = ((2 * (i % 127) + 1) * amax / 254.0).float()
        bits = near.view(torch.int32) + (torch.arange(hd) // 43 - 1).int()  # one below, at, one above
        for x in (near, bits.view(torch.float32).clamp(-3.4e38, 3.4e38)):
            x = torch.where(torch.arange(hd) % 2 == 0, x, -x)
            x = x.clamp(-float(torch.tensor(amax).float()), float(torch.tensor(amax).float())).clone()
            x[5] = amax
            rows.append(x)
    k = torch.stack(rows).float().cuda()
    layer = new_layer(torch, 1, hd, 64)
    append(torch, layer, k, -k.flip(1), 1, hd, 64, 2)
    check_stored(torch, layer, k, -k.flip(1), 1, hd, 64, 2)


def test_append_of_zeros_infinities_and_nan(gpu):
    torch = gpu
    nkv, hd = 2, 64
    k, v = rand(torch, 1, 8, nkv * hd), rand(torch, 2, 8, nkv * hd)
    k[0] = 0.0
    k[1, 3], k[2, hd + 1], v[3, 7], v[4, 64] = math.inf, -math.inf, math.nan, math.inf
    v[5, :hd] = -0.0
    layer = new_layer(torch, nkv, hd, 64)
    append(torch, layer, k, v, nkv, hd, 64, 0)
    got, want = R.unpack(layer, nkv, hd, 64), [R.codes(x.reshape(8, nkv, hd).transpose(0, 1)) for x in (k, v)]
    for c, s, (wc, ws) in ((got[0], got[2], want[0]), (got[1], got[3], want[1])):
        assert torch.equal(c[:, :8], wc)
        assert torch.equal(torch.isnan(s[:, :8]), torch.isnan(ws)) and torch.equal(s[:, :8].nan_to_num(), ws.nan_to_num())
    back = torch.empty((2, 8, nkv * hd), device="cuda")
    A.check(A.lib().aeth_kv8_read(layer.data_ptr(), back[0].data_ptr(), back[1].data_ptr(), nkv * hd, hd, 8, nkv, hd, 64, 0, stream(torch)), "read")
    assert torch.isnan(back[0, 1, :hd]).all() and torch.isfinite(back[0, 1, hd:]).all() and (back[0, 0] == 0).all()
    assert torch.isnan(back[1, 3, :hd]).all() and torch.isnan(back[1, 4, hd:]).all()


def test_append_in_pieces_leaves_the_same_bytes(gpu):
    torch = gpu
    nkv, hd, n, max_seq = 3, 128, 333, 400
    k, v = rand(torch, 5, n, nkv * hd), rand(torch, 6, n, nkv * hd)
    whole, parts = new_layer(torch, nkv, hd, max_seq), new_layer(torch, nkv, hd, max_seq)
    append(torch, whole, k, v, nkv, hd, max_seq, 20)
    at = 0
    for size in (1, 1, 42, 64, 3, 128, 94):
        append(torch, parts, k[at:at + size], v[at:at + size], nkv, hd, max_seq, 20 + at)
        at += size
    assert at == n and torch.equal(whole, parts)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_batch_append(gpu, hd):
    """One token a sequence at its own slot; slots out of range take nothing; a gap between slices is not touched."""
    torch = gpu
    nkv, max_seq = 2, 130
    slots = [0, 129, 64, -1, 130, 63, 2 ** 31 - 1, -2 ** 31, 100]
    k, v = rand(torch, 7, len(slots), nkv * hd), rand(torch, 8, len(slots), nkv * hd)
    size = A.lib().aeth_kv8_layer_bytes(nkv, hd, max_seq)
    all_ = torch.full((len(slots), size + 48), 0xA5, dtype=torch.uint8, device="cuda")
    d = torch.tensor(slots, dtype=torch.int64).to(torch.int32).cuda()
    A.check(A.lib().aeth_kv8_append_batch(all_.data_ptr(), size + 48, d.data_ptr(), k.data_ptr(), v.data_ptr(), nkv * hd, hd, len(slots), nkv, hd,
                                          max_seq, stream(torch)), "append batch")
    assert (all_[:, size:] == 0xA5).all()
    for i, slot in enumerate(slots):
        layer = all_[i, :size].reshape(R.layer_shape(nkv, hd, max_seq))
        if 0 <= slot < max_seq:
            check_stored(torch, layer, k[i:i + 1], v[i:i + 1], nkv, hd, max_seq, slot)
        else:
            assert (layer == 0xA5).all()


def test_a_cache_past_32_bit_offsets(gpu):
    """Slots whose bytes lie past 4 GiB: 8 heads of 256 over 2^20 positions."""
    torch = gpu
    nkv, hd, max_seq = 8, 256, 1 << 20
    size = A.lib().aeth_kv8_layer_bytes(nkv, hd, max_seq)
    assert size > 1 << 32
    layer = torch.zeros(R.layer_shape(nkv, hd, max_seq), dtype=torch.uint8, device="cuda")
    n, slot = 130, max_seq - 131
    k, v = rand(torch, 9, n, nkv * hd), rand(torch, 10, n, nkv * hd)
    append(torch, layer, k, v, nkv, hd, max_seq, slot)
    back = torch.empty((2, n, nkv * hd), device="cuda")
    A.check(A.lib().aeth_kv8_read(layer.data_ptr(), back[0].data_ptr(), back[1].data_ptr(), nkv * hd, hd, n, nkv, hd, max_seq, slot, stream(torch)), "read")
    for x, b in zip((k, v), back):
        c, s = R.codes(x.reshape(n, nkv, hd))
        assert torch.equal(b.reshape(n, nkv, hd), c.float() * s[..., None])
    # attention at the far end, through a window that keeps to what was appended
    q = rand(torch, 11, 3, 8 * hd)
    got = attend(torch, q, layer, nkv, hd, max_seq, slot + n, 100)
    tail = layer[:, -3:].contiguous()  # the last 192 slots
    want, bound = R.attention(q, tail, nkv, hd, 192, slot + n - (max_seq - 192), 100)
    within(torch, got, want, bound)


# ── attention ─────────────────────────────────────────────────────────────

ATTN = [
    # n, seq, heads, kv_heads, hd, window
    (1, 1, 1, 1, 64, 0), (1, 1, 32, 8, 128, 0), (1, 63, 8, 8, 128, 0), (1, 64, 4, 1, 128, 0), (1, 65, 16, 1, 64, 0), (1, 257, 32, 8, 128, 0),
    (1, 2049, 32, 8, 128, 0), (1, 5000, 6, 2, 256, 0), (1, 3000, 20, 1, 128, 0), (1, 4097, 33, 1, 64, 0), (1, 9000, 8, 8, 64, 0),
    (1, 1000, 32, 8, 128, 100), (1, 129, 8, 2, 128, 1), (1, 128, 8, 2, 128, 64), (1, 128, 8, 2, 128, 127), (1, 128, 8, 2, 128, 128), (1, 6000, 7, 1, 128, 5000),
    (2, 2, 4, 2, 128, 0), (5, 300, 12, 4, 128, 0), (7, 5003, 16, 2, 64, 1024), (8, 64, 8, 1, 256, 0), (3, 1500, 21, 3, 256, 700),
    (64, 64, 4, 4, 64, 0), (65, 65, 32, 8, 128, 0), (100, 163, 10, 2, 128, 0), (250, 1250, 8, 2, 128, 0), (129, 129, 3, 1, 256, 0), (200, 333, 7, 1, 64, 90),
    (512, 512, 32, 8, 128, 0), (700, 700, 16, 2, 128, 1), (1000, 1000, 8, 8, 128, 333), (333, 2000, 14, 2, 128, 0), (1999, 1999, 4, 1, 128, 0),
    (150, 900, 6, 1, 128, 65), (257, 700, 9, 3, 64, 0),
    # every form and its splits: prompts past the small workgroups (hd 64 and 128), a few queries and a chunk over a long past,
    # a window, a prompt for the largest
    (1700, 1700, 32, 8, 128, 0), (3100, 3100, 24, 8, 64, 0), (70, 30000, 16, 8, 128, 0), (250, 20001, 32, 8, 128, 0), (330, 12000, 7, 1, 64, 0),
    (4000, 6000, 32, 8, 128, 555), (3500, 3500, 32, 8, 128, 0), (2000, 2100, 3, 3, 256, 0),
    # 128 columns whole, in a few chunks, in many; with a window
    (600, 600, 64, 8, 64, 0), (600, 1600, 64, 8, 64, 700), (333, 3333, 64, 8, 64, 3000), (600, 7600, 7, 1, 64, 0), (200, 20200, 6, 2, 64, 0),
    (600, 600, 64, 8, 128, 0), (333, 1333, 64, 8, 128, 700), (2000, 3000, 16, 8, 128, 0), (100, 7100, 64, 8, 128, 0), (333, 20333, 8, 8, 128, 0),
    # 256 columns
    (333, 1333, 64, 8, 128, 0), (600, 1600, 64, 8, 128, 700), (600, 3600, 16, 8, 128, 0), (600, 3600, 16, 8, 128, 3000 - 7), (100, 7100, 32, 8, 128, 0),
]


@pytest.mark.parametrize("n,seq,heads,nkv,hd,window", ATTN)
def test_attention(gpu, n, seq, heads, nkv, hd, window):
    torch = gpu
    max_seq = seq + (17 if seq % 2 else 0)
    layer = some_layer(torch, seq + n, nkv, hd, max_seq)
    q = 2.0 * rand(torch, seq, n, heads * hd)
    got = attend(torch, q, layer, nkv, hd, max_seq, seq, window)
    want, bound = R.attention(q, layer, nkv, hd, max_seq, seq, window)
    within(torch, got, want, bound)
    assert torch.equal(attend(torch, q, layer, nkv, hd, max_seq, seq, window), got)  # the same bits again


@pytest.mark.parametrize("n,seq", [(1, 700), (90, 700)])
def test_attention_of_rows_of_any_stride(gpu, n, seq):
    torch = gpu
    nkv, hd, heads = 2, 128, 8
    layer = some_layer(torch, 4, nkv, hd, seq)
    for stride, shift in ((12 * hd, 0), (heads * hd + 3, 1), (heads * hd, 1)):
        buf = torch.zeros((n - 1) * stride + heads * hd + shift, device="cuda")
        rows = torch.as_strided(buf, (n, heads * hd), (stride, 1), shift)
        rows.copy_(rand(torch, 12, n, heads * hd))
        out = torch.full((n * heads * hd + 2,), 7.0, device="cuda")  # from an odd address too
        L = A.lib()
        ws = torch.empty(L.aeth_attn_kv8_ws_bytes(1, n, heads, nkv, hd, seq), dtype=torch.uint8, device="cuda")
        A.check(L.aeth_attn_kv8(rows.data_ptr(), stride, layer.data_ptr(), n, heads, nkv, hd, seq, seq, 0, out[shift:].data_ptr(), ws.data_ptr(), ws.numel(),
                                stream(torch)), "attn")
        want, bound = R.attention(rows.contiguous(), layer, nkv, hd, seq, seq, 0)
        within(torch, out[shift:shift + n * heads * hd].reshape(n, -1), want, bound)
        assert (out[:shift] == 7.0).all() and (out[shift + n * heads * hd:] == 7.0).all()


@pytest.mark.parametrize("n,seq,window", [(1, 200, 50), (1, 1300, 0), (70, 200, 0), (70, 200, 20), (300, 300, 0)])
def test_masked_infinities_and_nan_have_no_effect(gpu, n, seq, window):
    """Slots past the end that were never written, or hold infinities and NaN for scales; masked tokens of a NaN scale;
    a visible one makes its rows NaN and no others."""
    torch = gpu
    nkv, hd, heads, max_seq = 2, 128, 8, 400
    layer = some_layer(torch, 21, nkv, hd, max_seq)
    q = rand(torch, 22, n, heads * hd)
    want, bound = R.attention(q, layer, nkv, hd, max_seq, min(seq, max_seq), window) if seq <= max_seq else (None, None)
    if seq > max_seq:
        max_seq = seq + 60
        layer = some_layer(torch, 21, nkv, hd, max_seq)
        want, bound = R.attention(q, layer, nkv, hd, max_seq, seq, window)
    kc, vc, ks, vs = R.unpack(layer, nkv, hd, max_seq)
    for bad in (math.nan, math.inf, -math.inf):
        ks[:, seq:], vs[:, seq:] = bad, bad
        if window:
            ks[:, :seq - n - window + 1], vs[:, :seq - n - window + 1] = bad, bad  # before every query's window
        got = attend(torch, q, R.pack(kc, ks, vc, vs), nkv, hd, max_seq, seq, window)
        within(torch, got, want, bound)
    # a token that some queries see and some do not
    for which in (ks, vs):
        old = which[1, seq - 1 - n // 2].clone()
        which[1, seq - 1 - n // 2] = math.nan
        got = attend(torch, q, R.pack(kc, ks, vc, vs), nkv, hd, max_seq, seq, window)
        which[1, seq - 1 - n // 2] = old
        pos = torch.arange(seq - n, seq, device="cuda")
        sees = (pos >= seq - 1 - n // 2) & ((pos - window < seq - 1 - n // 2) if window else True)
        nan = torch.isnan(got).reshape(n, nkv, -1)
        assert nan[sees][:, 1].all() and not nan[~sees].any() and not nan[:, 0].any()
        within(torch, got.reshape(n, nkv, -1)[:, 0], want.reshape(n, nkv, -1)[:, 0], bound.reshape(n, nkv, -1)[:, 0])


def test_queries_that_are_no_numbers(gpu):
    torch = gpu
    nkv, hd, heads, seq = 1, 64, 4, 150
    layer = some_layer(torch, 30, nkv, hd, seq)
    q = rand(torch, 31, 6, heads * hd)
    q[0] = 0.0
    q[1, 3], q[2, hd + 3], q[3, 5] = math.nan, math.inf, -math.inf
    q[4] *= 1e-30
    q[5] *= 40.0
    got = attend(torch, q, layer, nkv, hd, seq, seq)
    nan = torch.isnan(got).reshape(6, heads, hd)
    for i in range(6):
        for h in range(heads):
            assert nan[i, h].all() == ((i, h) in ((1, 0), (2, 1), (3, 0))) and (nan[i, h].all() or not nan[i, h].any())
    want, bound = R.attention(q, layer, nkv, hd, seq, seq, 0)
    for i in (0, 4, 5):
        within(torch, got[i], want[i], bound[i])


@pytest.mark.parametrize("n,seq", [(1, 1000), (120, 1000), (1000, 3000)])
def test_attention_over_uneven_rows(gpu, n, seq):
    """What the maximum, the digits and the tiles' exponents have to stand: one key far above the rest, with a value
    of no size; scores that rise from tile to tile by hundreds; a flat row; V scales from 1e-20 to 1e20."""
    torch = gpu
    nkv, hd, heads = 1, 128, 16 if n == 1000 else 2
    slots = -(-seq // 64) * 64
    base = rand(torch, 40, nkv, slots, hd)
    val = rand(torch, 41, nkv, slots, hd)
    q = rand(torch, 42, n, heads * hd)
    t = torch.arange(slots, device="cuda").float()[None, :, None]
    cases = []
    k, v = base.clone(), val.clone()
    k[:, 3] = 12.0 * q[0, :hd] / q[0, :hd].norm()
    v[:, 3] = 1e-7
    cases.append((k, v))
    cases.append((base * (1.0 + t / 20.0), val))
    cases.append((base * (1.0 + (seq - t).clamp_min(0) / 20.0), val))
    cases.append((base * 0.0, val))
    cases.append((base * 1e-3, val * torch.pow(10.0, (t % 41) - 20.0)))
    cases.append((base, val * torch.pow(10.0, -t / 50.0)))
    cases.append((base, val * 1e-24))
    cases.append((base, val * 1e33))
    for k, v in cases:
        kc, ks = R.codes(k)
        vc, vs = R.codes(v)
        layer = R.pack(kc, ks, vc, vs)
        got = attend(torch, q, layer, nkv, hd, slots, seq)
        want, bound = R.attention(q, layer, nkv, hd, slots, seq, 0)
        within(torch, got, want, bound)


WIDE = [  # calls of many columns: 128 whole, with a window, split; 256 split, whole
    (800, 800, 48, 2, 128, 0), (600, 600, 64, 8, 64, 0), (1000, 4000, 32, 2, 128, 600), (600, 7600, 7, 1, 64, 0), (500, 4000, 32, 2, 128, 0),
    (700, 3000, 32, 1, 128, 0), (1500, 1500, 64, 8, 128, 0),
]


@pytest.mark.parametrize("n,seq,heads,nkv,hd,window", WIDE)
def test_many_columns_with_no_numbers_and_any_stride(gpu, n, seq, heads, nkv, hd, window):
    """What the tests above ask of a few columns: slots that no query sees hold infinities and NaN, a token that some
    see is a NaN, a query is one; rows from an odd address with a gap, the result to one."""
    torch = gpu
    max_seq = seq + 70
    layer = some_layer(torch, 24, nkv, hd, max_seq)
    kc, vc, ks, vs = R.unpack(layer, nkv, hd, max_seq)
    ks[:, seq:], vs[:, seq:] = math.nan, math.inf
    if window:
        ks[:, :seq - n - window + 1], vs[:, :seq - n - window + 1] = math.inf, math.nan
    layer = R.pack(kc, ks, vc, vs)
    q = rand(torch, 25, n, heads * hd)
    want, bound = R.attention(q, layer, nkv, hd, max_seq, seq, window)
    within(torch, attend(torch, q, layer, nkv, hd, max_seq, seq, window), want, bound)
    stride = heads * hd + 3
    rows = torch.as_strided(torch.zeros((n - 1) * stride + heads * hd + 1, device="cuda"), (n, heads * hd), (stride, 1), 1)
    rows.copy_(q)
    out = torch.full((n * heads * hd + 2,), 7.0, device="cuda")
    L = A.lib()
    ws = torch.full((max(L.aeth_attn_kv8_ws_bytes(1, n, heads, nkv, hd, seq), 16),), 0xFF, dtype=torch.uint8, device="cuda")
    A.check(L.aeth_attn_kv8(rows.data_ptr(), stride, layer.data_ptr(), n, heads, nkv, hd, max_seq, seq, window, out[1:].data_ptr(), ws.data_ptr(), ws.numel(),
                            stream(torch)), "attn")
    within(torch, out[1:-1].reshape(n, -1), want, bound)
    assert out[0] == 7.0 and out[-1] == 7.0
    # a token of a NaN scale in the last KV head, and a query with one
    at, bad_q = seq - 1 - n // 2, n // 3
    pos = torch.arange(seq - n, seq, device="cuda")
    sees = (pos >= at) & ((pos - window < at) if window else True)
    sees[bad_q] = False
    q[bad_q, 5] = math.inf
    for which in (ks, vs):
        old = which[-1, at].clone()
        which[-1, at] = math.nan
        got = attend(torch, q, R.pack(kc, ks, vc, vs), nkv, hd, max_seq, seq, window)
        which[-1, at] = old
        nan = torch.isnan(got).reshape(n, nkv, -1)
        assert torch.isnan(got[bad_q, :hd]).all()
        rest = torch.arange(n, device="cuda") != bad_q
        assert nan[sees][:, -1].all() and not nan[rest & ~sees].any() and not nan[rest][:, :-1].any()
        fine = ~nan & rest[:, None, None]
        within(torch, got.reshape(n, nkv, -1)[fine], want.reshape(n, nkv, -1)[fine], bound.reshape(n, nkv, -1)[fine])


@pytest.mark.parametrize("n,seq,heads,nkv,hd,window", [w for w in WIDE if w[0] < 1000])
def test_many_columns_over_uneven_rows(gpu, n, seq, heads, nkv, hd, window):
    torch = gpu
    slots = -(-seq // 64) * 64
    base, val = rand(torch, 43, nkv, slots, hd), rand(torch, 44, nkv, slots, hd)
    q = rand(torch, 48, n, heads * hd)
    t = torch.arange(slots, device="cuda").float()[None, :, None]
    for k, v in ((base * (1.0 + t / 20.0), val), (base * (1.0 + (seq - t).clamp_min(0) / 20.0), val), (base * 0.0, val),
                 (base * 1e-3, val * torch.pow(10.0, (t % 41) - 20.0)), (base, val * torch.pow(10.0, -t / 50.0).clamp_min(1e-30)), (base, val * 1e33)):
        layer = R.pack(*R.codes(k), *R.codes(v))
        want, bound = R.attention(q, layer, nkv, hd, slots, seq, window)
        within(torch, attend(torch, q, layer, nkv, hd, slots, seq, window), want, bound)


def test_the_ends_of_the_ranges(gpu):
    """4096 query heads of one KV head, 300 KV heads, a sequence of 2.5 million tokens, 3000 sequences."""
    torch = gpu
    for n, seq, heads, nkv, hd, window in ((1, 70, 4096, 1, 64, 0), (3, 200, 300, 300, 64, 0), (2, 2500000, 4, 1, 64, 0), (1, 2500000, 4, 1, 64, 2 ** 40)):
        layer = some_layer(torch, 27, nkv, hd, seq)
        q = rand(torch, 28, n, heads * hd)
        want, bound = R.attention(q, layer, nkv, hd, seq, seq, 0)
        within(torch, attend(torch, q, layer, nkv, hd, seq, seq, window), want, bound)
    nkv, hd, seqs, max_seq = 1, 64, 3000, 300
    layer = some_layer(torch, 29, nkv, hd, max_seq)
    lens = torch.arange(seqs, dtype=torch.int32, device="cuda") % 301
    q = rand(torch, 30, 1, 2 * hd)
    got = attend_batch(torch, q.expand(seqs, -1).contiguous(), layer[None].expand(seqs, -1, -1, -1).contiguous(), lens, nkv, hd, max_seq, max_seq)
    for n in (0, 1, 64, 65, 129, 300):
        want, bound = R.attention(q, layer, nkv, hd, max_seq, n, 0)
        within(torch, got[n::301], want.expand(len(got[n::301]), -1), bound.expand(len(got[n::301]), -1))


@pytest.mark.parametrize("n,seq,heads,nkv,hd", [(250, 8448, 32, 8, 128), (70, 9000, 16, 8, 128), (90, 9000, 16, 8, 64), (1, 9000, 32, 8, 128),
                                                (100, 7100, 64, 8, 128), (600, 7600, 7, 1, 64), (100, 7100, 32, 8, 128)])
def test_split_rows_of_tiles_that_differ(gpu, n, seq, heads, nkv, hd):
    """Every other tile holds keys a hundred times as long that no query points at: codes of one tile beside the
    scales of another would give scores far above any there is, at the end of a chunk as within it."""
    torch = gpu
    slots = -(-seq // 64) * 64
    k, v = rand(torch, 45, nkv, slots, hd), rand(torch, 46, nkv, slots, hd)
    q = 2.0 * rand(torch, 47, n, heads * hd)
    q.view(n, heads, hd)[..., hd // 2:] = 0.0
    odd = (torch.arange(slots, device="cuda") // 64) % 2 == 1
    for which in (odd, ~odd):
        long = k.clone()
        long[:, which, :hd // 2] = 0.0
        long[:, which, hd // 2:] *= 100.0
        layer = R.pack(*R.codes(long), *R.codes(v))
        got = attend(torch, q, layer, nkv, hd, slots, seq)
        want, bound = R.attention(q, layer, nkv, hd, slots, seq, 0)
        within(torch, got, want, bound)


@pytest.mark.parametrize("heads,nkv,hd,window", [(32, 8, 128, 0), (5, 1, 64, 0), (16, 4, 256, 0), (8, 2, 128, 300), (34, 2, 128, 0)])
def test_batch_attention(gpu, heads, nkv, hd, window):
    """Sequences of no, one and many tokens in one call; rows behind the last one as they were."""
    torch = gpu
    max_seq = 2200
    lens = [0, 1, 64, 65, 2200, 700, 0, 2049, 63, 1999, 2, 1025]
    layers = torch.stack([some_layer(torch, 50 + 2 * i, nkv, hd, max_seq) for i in range(len(lens))])
    q = rand(torch, 49, len(lens), heads * hd)
    d = torch.tensor(lens + [-1], dtype=torch.int32, device="cuda")
    out = torch.full((len(lens) + 1, heads * hd), 7.0, device="cuda")
    attend_batch(torch, q, layers, d, nkv, hd, max_seq, max_seq, window, out)
    assert (out[-1] == 7.0).all()
    for i, n in enumerate(lens):
        want, bound = R.attention(q[i:i + 1], layers[i], nkv, hd, max_seq, n, window)
        within(torch, out[i:i + 1], want, bound)
        if n:
            # the same as the sequence alone, to the order of the sums
            alone = attend(torch, q[i:i + 1], layers[i], nkv, hd, max_seq, n, window)
            within(torch, alone, want, bound)
    # a bound below some lengths: those are taken as the bound; lengths below 0 as 0
    d = torch.tensor([n if n else -5 for n in lens], dtype=torch.int32, device="cuda")
    short = attend_batch(torch, q, layers, d, nkv, hd, max_seq, 700, window)
    for i, n in enumerate(lens):
        want, bound = R.attention(q[i:i + 1], layers[i], nkv, hd, max_seq, min(n, 700), window)
        within(torch, short[i:i + 1], want, bound)


def test_two_streams_with_a_workspace_each(gpu):
    torch = gpu
    nkv, hd, heads, max_seq = 4, 128, 16, 6000
    layer = some_layer(torch, 60, nkv, hd, max_seq)
    need = A.lib().aeth_attn_kv8_ws_bytes(1, 4, heads, nkv, hd, max_seq)
    ws = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in range(2)]
    qs = [rand(torch, 61 + i, 1 + 3 * i, heads * hd) for i in range(2)]
    alone = [attend(torch, q, layer, nkv, hd, max_seq, 6000 - 500 * i) for i, q in enumerate(qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(attend(torch, qs[i], layer, nkv, hd, max_seq, 6000 - 500 * i, ws=ws[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o, alone[i])


# ── head norms and rotation ───────────────────────────────────────────────


def tables(torch, hd, max_seq):
    angle = torch.arange(max_seq, dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64) / hd)
    return angle.sin().float().cuda(), angle.cos().float().cuda()


def qk(torch, x, nq, nk, hd, qw, kw, eps, pos, dpos, sin, cos, out=None, n=None):
    n = x.shape[0] if n is None else n
    if out is None:
        out = torch.full((n, (nq + nk) * hd), math.nan, device="cuda")
    A.check(A.lib().aeth_qk_norm_rope(x.data_ptr(), x.stride(0), n, nq, nk, hd, qw.data_ptr() if qw is not None else None,
                                      kw.data_ptr() if kw is not None else None, eps, pos, dpos.data_ptr() if dpos is not None else None, sin.data_ptr(),
                                      cos.data_ptr(), sin.shape[0], out.data_ptr(), out.stride(0), stream(torch)), "qk")
    return out


@pytest.mark.parametrize("n,nq,nk,hd", [(1, 1, 1, 64), (1, 32, 8, 128), (3, 4, 4, 256), (37, 12, 2, 128), (5, 3, 1, 80), (2, 2, 2, 2), (9, 5, 0, 64),
                                        (9, 0, 5, 128), (4, 2, 1, 514), (513, 8, 1, 64)])
@pytest.mark.parametrize("norm", ["both", "none", "q", "k"])
def test_head_norms_and_rotation(gpu, n, nq, nk, hd, norm):
    torch = gpu
    sin, cos = tables(torch, hd, 300)
    x = rand(torch, n + hd, n, (nq + 2 * nk + 1) * hd)
    qw = rand(torch, 70, hd) if norm in ("both", "q") else None
    kw = rand(torch, 71, hd) if norm in ("both", "k") else None
    positions = torch.arange(n, device="cuda") + 7
    got = qk(torch, x, nq, nk, hd, qw, kw, 1e-5, 7, None, sin, cos)
    want, bound = R.qk_norm_rope(x, nq, nk, hd, qw, kw, 1e-5, positions, sin, cos)
    within(torch, got, want, bound)
    # positions by row, some outside the table; rows that are not 16-byte aligned
    d = torch.randint(-3, 310, (n,), dtype=torch.int32, generator=torch.Generator().manual_seed(n)).cuda()
    wide = torch.zeros((n, x.shape[1] + 1), device="cuda")
    wide[:, 1:] = x
    got = qk(torch, wide[:, 1:], nq, nk, hd, qw, kw, 1e-5, 0, d, sin, cos)
    want, bound = R.qk_norm_rope(x, nq, nk, hd, qw, kw, 1e-5, d, sin, cos)
    within(torch, got, want, bound)
    # in place; what follows the heads in a row stays
    y = x.clone()
    again = qk(torch, x, nq, nk, hd, qw, kw, 1e-5, 0, d, sin, cos)
    qk(torch, y, nq, nk, hd, qw, kw, 1e-5, 0, d, sin, cos, out=y)
    assert torch.equal(y[:, :(nq + nk) * hd], again) and torch.equal(y[:, (nq + nk) * hd:], x[:, (nq + nk) * hd:])


def test_rotation_alone_is_aeth_rope(gpu):
    torch = gpu
    nq, nk, hd, n = 8, 2, 128, 5
    sin, cos = tables(torch, hd, 100)
    x = rand(torch, 80, n, (nq + nk) * hd)
    got = qk(torch, x, nq, nk, hd, None, None, 0.0, 40, None, sin, cos)
    for i in range(n):
        row = x[i].clone()
        A.check(A.lib().aeth_rope(row.data_ptr(), nq + nk, hd, 40 + i, sin.data_ptr(), cos.data_ptr(), 100, stream(torch)), "rope")
        assert torch.equal(got[i], row)


# ── together, as a program uses them ──────────────────────────────────────


def test_a_batch_decodes_under_a_captured_graph(gpu):
    """Prompts of three lengths appended whole, then decode steps of the batch captured once: norm and rotation at each
    sequence's position, append, attention, all following device lengths; replayed with eager work between, each replay
    against the eager calls on another copy."""
    torch = gpu
    nq, nk, hd, max_seq, b = 8, 2, 128, 400, 3
    sin, cos = tables(torch, hd, max_seq)
    qw, kw = rand(torch, 90, hd), rand(torch, 91, hd)
    start = [5, 130, 63]
    L = A.lib()
    width = (nq + 2 * nk) * hd

    def fresh():
        layers = new_layer(torch, nk, hd, max_seq, b)
        for i, n in enumerate(start):
            x = rand(torch, 92 + i, n, width)
            y = qk(torch, x, nq, nk, hd, qw, kw, 1e-5, 0, None, sin, cos)
            A.check(L.aeth_kv8_append(layers[i].data_ptr(), y[:, nq * hd:].data_ptr(), x[:, (nq + nk) * hd:].data_ptr(), width, hd, 0, nk, hd, max_seq, 0,
                                      stream(torch)), "append of nothing")
            k = y[:, nq * hd:].contiguous()
            v = x[:, (nq + nk) * hd:].contiguous()
            append(torch, layers[i], k, v, nk, hd, max_seq, 0)
        return layers, torch.tensor(start, dtype=torch.int32, device="cuda")

    x = torch.empty((b, width), device="cuda")
    ws = torch.empty(L.aeth_attn_kv8_ws_bytes(b, 1, nq, nk, hd, max_seq), dtype=torch.uint8, device="cuda")
    y, out = torch.empty((b, width), device="cuda"), torch.empty((b, nq * hd), device="cuda")

    def step(layers, at, y, out, ws):
        """at: the tokens each sequence has; afterwards one more"""
        y.copy_(x)
        qk(torch, y, nq, nk, hd, qw, kw, 1e-5, 0, at, sin, cos, out=y)
        A.check(L.aeth_kv8_append_batch(layers.data_ptr(), layers[0].numel(), at.data_ptr(), y[:, nq * hd:].data_ptr(), y[:, (nq + nk) * hd:].data_ptr(), width,
                                        hd, b, nk, hd, max_seq, stream(torch)), "append")
        at.add_(1)
        A.check(L.aeth_attn_kv8_batch(y.data_ptr(), width, layers.data_ptr(), layers[0].numel(), at.data_ptr(), b, nq, nk, hd, max_seq, max_seq, 0,
                                      out.data_ptr(), ws.data_ptr(), ws.numel(), stream(torch)), "attn")

    layers, at = fresh()
    twin, at2 = fresh()
    y2, out2, ws2 = torch.empty_like(y), torch.empty_like(out), torch.empty_like(ws)
    x.copy_(rand(torch, 100, b, width))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(layers, at, y, out, ws)
    for i in range(70):
        x.copy_(rand(torch, 101 + i, b, width))
        graph.replay()
        torch.cuda.synchronize()
        step(twin, at2, y2, out2, ws2)
        torch.cuda.synchronize()
        assert torch.equal(out, out2), i
    assert torch.equal(layers, twin) and at.tolist() == [n + 70 for n in start]
    for i in range(b):
        n = start[i] + 70
        want, bound = R.attention(y[i:i + 1, :nq * hd].contiguous(), layers[i], nk, hd, max_seq, n, 0)
        within(torch, out[i:i + 1], want, bound)
