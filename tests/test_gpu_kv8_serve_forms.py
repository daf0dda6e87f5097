"""The forms of the serving calls over the 8-bit cache that take many columns, at shapes that are reckoned to take them on
256 CUs: a prefix in blocks of 128 columns, the weights of tokens behind the attention in blocks of 128 and 256,
four keys a thread of a batch's weights, and four heads a thread of the rotation by several axes; against 64 bits (tests/_kv8.py, tests/_kv8_serve.py).
The attentions of tests/test_gpu_kv8_serve.py take blocks of 16 columns throughout."""
import math

import pytest

import aether_amd as A
from tests import _kv8_serve as S
from tests.test_gpu_kv8 import rand, some_layer, stream, within
from tests.test_gpu_kv8_serve import axes_exact, axes_rope, ints, shared, some_layers, table, weigh, weigh_batch

pytestmark = pytest.mark.gpu


def no_numbers(torch, layer, hd, slots):
    """NaN as the scales of a range of slots, in every head of a layer slice."""
    for at in (128 * hd, 128 * hd + 256):
        scales = layer[..., at:at + 256].contiguous().view(torch.float32)  # [heads][tiles][64]
        scales.reshape(len(layer), -1)[:, slots.start:slots.stop] = math.nan
        layer[..., at:at + 256] = scales.view(torch.uint8)


def apart(torch, x):
    """The same rows at an odd address and stride."""
    buf = torch.zeros(x.shape[0] * (x.shape[1] + 3) + 1, device="cuda")
    rows = torch.as_strided(buf, x.shape, (x.shape[1] + 3, 1), 1)
    rows.copy_(x)
    return rows


# ── a shared prefix in blocks of 128 columns ──────────────────────────────

# (head_dim, sequences, KV heads, query heads of each, prefix, window), with what is joined: parts of the prefix. Columns fill no whole number of
# blocks but in the last two.
BLOCKS = [(128, 17, 64, 32, 64, 0),      # 1
          (128, 17, 8, 32, 6001, 0),     # 6
          (64, 33, 4, 32, 12001, 0),     # 7
          (128, 33, 2, 32, 12001, 0),    # 12
          (64, 65, 2, 32, 20001, 0),     # 14
          (128, 33, 4, 3, 80001, 0),     # 63, less than one block
          (64, 100, 1, 8, 80001, 0),     # 35
          (128, 17, 64, 32, 500, 250),   # 1, and windows that leave the prefix
          (128, 17, 8, 32, 12001, 9001),  # 6
          (64, 33, 4, 32, 20001, 12001),  # 7
          (128, 17, 4, 32, 30001, 20001),  # 12
          (64, 65, 2, 32, 30001, 20001),  # 14
          (128, 160, 8, 4, 6000, 0),     # 6
          (128, 160, 8, 4, 10000, 8000)]


@pytest.mark.parametrize("hd,seqs,nkv,g,prefix_len,window", BLOCKS)
def test_shared_prefix_in_blocks_of_128_columns(gpu, hd, seqs, nkv, g, prefix_len, window):
    """Windows begin in different tiles of the prefix; what no window reaches and the slots behind the prefix and the lengths hold NaN scales."""
    torch = gpu
    own = 300
    lens = [(53 * b) % (own + 1) for b in range(seqs)]
    prefix, layers = some_layer(torch, 1, nkv, hd, prefix_len), some_layers(torch, 9, seqs, nkv, hd, own)
    no_numbers(torch, prefix, hd, range(prefix_len, -(-prefix_len // 64) * 64))
    if window:
        no_numbers(torch, prefix, hd, range(0, prefix_len - window))
    for b in range(seqs):
        no_numbers(torch, layers[b], hd, range(lens[b], 320))
    q = rand(torch, 2, seqs, nkv * g * hd)
    got = shared(torch, q, prefix, prefix_len, prefix_len, layers, ints(torch, lens), nkv, hd, own, own, window)
    assert not got.isnan().any()
    pick = sorted({b * (seqs - 1) // 7 for b in range(8)})
    want, bound = S.shared(q[pick].contiguous(), prefix, prefix_len, prefix_len, layers[pick], [lens[b] for b in pick], nkv, hd, own, window)
    within(torch, got[pick], want, bound)
    out = torch.full((q.numel() + 1,), math.nan, device="cuda")[1:].reshape(q.shape)
    again = shared(torch, apart(torch, q), prefix, prefix_len, prefix_len, layers, ints(torch, lens), nkv, hd, own, own, window, out=out)
    assert torch.equal(again, got)


# ── token weights behind the attention in blocks of many columns ──────────

# (head_dim, queries, tokens, KV heads, query heads of each, window), with the attention's columns of a block and chunks
COLUMNS = [(128, 701, 701, 8, 8, 0),       # 128, 1
           (128, 2000, 2000, 8, 4, 0),     # 128, 1
           (128, 1000, 1000, 4, 8, 500),   # 128, 1
           (128, 150, 8001, 16, 4, 0),     # 128, 4
           (128, 70, 20001, 8, 8, 10000),  # 128, 7
           (128, 300, 20001, 4, 1, 0),     # 128, 20
           (128, 150, 150, 8, 32, 0),      # 256, 1
           (128, 1000, 1500, 4, 16, 700),  # 256, 1
           (128, 150, 2001, 4, 32, 0),     # 256, 4
           (128, 70, 8001, 8, 8, 4000),    # 256, 8
           (128, 40, 20001, 1, 64, 0),     # 256, 20
           (128, 300, 8001, 4, 4, 4000),   # 256, 9
           (64, 301, 301, 8, 32, 0),       # 128, 1
           (64, 1000, 1500, 4, 16, 700),   # 128, 1
           (64, 33, 4001, 8, 32, 0),       # 128, 4
           (64, 70, 20001, 8, 8, 10000),   # 128, 7
           (64, 700, 8001, 1, 4, 0),       # 128, 11
           (64, 150, 40001, 2, 4, 20000)]  # 128, 20


@pytest.mark.parametrize("hd,n,seq,nkv,g,window", COLUMNS)
def test_weights_behind_blocks_of_many_columns(gpu, hd, n, seq, nkv, g, window):
    """What no query sees holds NaN scales; then with a query that is NaN, at an odd address."""
    torch = gpu
    dark = max(0, seq - n + 1 - window) if window else 0
    layer = some_layer(torch, n, nkv, hd, seq)
    no_numbers(torch, layer, hd, range(seq, -(-seq // 64) * 64))
    no_numbers(torch, layer, hd, range(0, dark))
    q, prior = rand(torch, seq, n, nkv * g * hd), rand(torch, 5, nkv, seq).abs()
    out, w = weigh(torch, q, layer, nkv, hd, seq, seq, window, prior)
    o, ot, ww, wt = S.weights(q, layer, nkv, hd, seq, seq, window, prior)
    within(torch, out, o, ot)
    within(torch, w, ww, wt)
    assert torch.equal(w[:, :dark], prior[:, :dark])
    # a query head of the second KV head, or of the only one
    i, head = n // 2, (g if nkv > 1 else 0) + g // 2
    q[i, head * hd + 5] = math.nan
    out, w = weigh(torch, apart(torch, q), layer, nkv, hd, seq, seq, window, prior)
    fine = torch.ones((n, nkv * g), dtype=torch.bool, device="cuda")
    fine[i, head] = False
    at = fine.repeat_interleave(hd, 1)
    assert out[~at].isnan().all()
    within(torch, out[at], o[at], ot[at])
    end = seq - n + i + 1
    lit = torch.ones((nkv, seq), dtype=torch.bool, device="cuda")
    lit[head // g, max(0, end - window) if window else 0:end] = False
    assert w[~lit].isnan().all()
    within(torch, w[lit], ww[lit], wt[lit])


# ── a batch's token weights, four keys a thread ───────────────────────────

# (head_dim, sequences, KV heads, query heads of each, longest, window), with the attention's chunks: more than 2048 pieces of 256 keys
PIECES = [(128, 33, 8, 4, 2100, 0),     # 3, joined with all in flight
          (256, 33, 8, 4, 2100, 0),     # 3
          (64, 20, 8, 10, 4096, 0),     # 4
          (128, 5, 8, 4, 14000, 0),     # 19, a workgroup a column
          (256, 5, 8, 4, 14000, 0),     # 19
          (64, 5, 8, 4, 14000, 0),      # 19
          (64, 12, 8, 4, 6000, 0),      # 8
          (256, 70, 8, 1, 1000, 0),     # 1
          (128, 5, 8, 4, 14000, 9000),  # 18
          (128, 40, 8, 4, 2100, 2000)]  # 1


@pytest.mark.parametrize("hd,seqs,nkv,g,longest,window", PIECES)
def test_batch_weights_of_four_keys_a_thread(gpu, hd, seqs, nkv, g, longest, window):
    """Lengths at the borders of pieces and chunks, some of whose newest tokens are NaN, weights added in place."""
    torch = gpu
    lens = ([longest, 0, 769, 1] + [l for l in (769, 1024, 1025, 1537, 256, 255) if l <= longest] + [(613 * b) % (longest + 1) for b in range(seqs)])[:seqs]
    bad = [b for b in (2, 3, seqs - 1) if lens[b]]
    layers, q, prior = some_layers(torch, 3, seqs, nkv, hd, longest + 3), rand(torch, 4, seqs, nkv * g * hd), rand(torch, 5, seqs, nkv, longest + 3).abs()
    for b in range(seqs):
        no_numbers(torch, layers[b], hd, range(lens[b] - (b in bad), -(-(longest + 3) // 64) * 64))
    w = prior.clone()
    out, _ = weigh_batch(torch, q, layers, ints(torch, lens), nkv, hd, longest + 3, longest, window, w, into=w)
    for b, seq in enumerate(lens):
        first = max(0, seq - window) if window else 0
        assert torch.equal(w[b, :, seq:], prior[b, :, seq:]) and torch.equal(w[b, :, :first], prior[b, :, :first])
        if b in bad:
            assert out[b].isnan().all() and w[b, :, first:seq].isnan().all()
        elif seq:
            o, ot, ww, wt = S.weights(q[b:b + 1], layers[b], nkv, hd, longest + 3, seq, window, prior[b])
            within(torch, out[b:b + 1], o, ot)
            within(torch, w[b, :, :seq], ww, wt)
        else:
            assert (out[b] == 0).all()


# ── four heads a thread by several axes ───────────────────────────────────


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("nq,nk,norm", [(7, 3, "qk"), (7, 3, "q"), (7, 3, "k"), (7, 3, ""), (8, 4, "qk"), (1, 0, "q"), (0, 5, "k"), (2, 1, "qk")])
def test_axes_of_many_rows(gpu, hd, nq, nk, norm, in_place):
    """1024 workgroups and some more, the last one part-filled: heads in groups of four that hold both q's and k's, or end early."""
    torch = gpu
    n = 1024 * 256 // (-(-(nq + nk) // 4) * hd // 8) + 13
    x = rand(torch, n, n, (nq + nk + 1) * hd)
    qw, kw = (rand(torch, 7 + i, hd) if c in norm else None for i, c in enumerate("qk"))
    g = torch.Generator().manual_seed(hd + nq)
    pos = torch.randint(-3, 130, (3, n), generator=g, dtype=torch.int32).cuda()  # the table has 100 rows
    pairs = torch.randint(0, 3, (hd // 2,), generator=g).tolist()
    sin, cos = table(torch, 100, hd)
    want, bound = axes_exact(x, nq, nk, hd, qw, kw, pos, pairs, sin, cos)
    was = x.clone()
    got = axes_rope(torch, x, nq, nk, hd, qw, kw, pos, pairs, sin, cos, out=x if in_place else None)
    within(torch, got[:, :(nq + nk) * hd], want, bound)
    assert torch.equal(x[:, (nq + nk) * hd:] if in_place else x, was[:, (nq + nk) * hd:] if in_place else was)
    # axes that agree give the bits of one
    same = pos[:1].expand(3, n).contiguous()
    one = torch.empty((n, (nq + nk) * hd), device="cuda")
    A.check(A.lib().aeth_qk_norm_rope(was.data_ptr(), was.shape[1], n, nq, nk, hd, qw.data_ptr() if qw is not None else None,
                                      kw.data_ptr() if kw is not None else None, 1e-5, 0, same.data_ptr(), sin.data_ptr(), cos.data_ptr(), 100,
                                      one.data_ptr(), one.shape[1], stream(torch)), "rope")
    assert torch.equal(axes_rope(torch, was, nq, nk, hd, qw, kw, same, pairs, sin, cos), one)
