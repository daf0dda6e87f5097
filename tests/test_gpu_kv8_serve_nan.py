"""What is no number in the serving calls over the 8-bit cache: a query with a NaN or an
infinity, and a cached token with one, where a part of a split row sees nothing else. Rows and
weights that the definition makes NaN are NaN whatever the parts; the others are held to
64 bits (tests/_kv8_serve.py)."""
import math

import pytest

from tests import _kv8_serve as S
from tests.test_gpu_kv8 import rand, some_layer, within
from tests.test_gpu_kv8_serve import ints, poison, shared, some_layers

pytestmark = pytest.mark.gpu

# (head_dim, sequences, KV heads, query heads of each, prefix, own tokens at most): the prefix in blocks of 16 columns and of
# 128, of each with one part of the prefix to join, a few, up to 16, and more; own tokens in several parts too
JOINS = [(128, 3, 2, 4, 200, 12), (64, 3, 2, 4, 1000, 12), (256, 17, 2, 4, 1000, 12), (128, 3, 2, 4, 1000, 2100), (128, 16, 8, 4, 3000, 12),
         (128, 5, 1, 4, 20000, 12), (256, 3, 1, 4, 9000, 12),
         (128, 17, 64, 32, 64, 12), (128, 17, 8, 32, 6001, 12), (64, 33, 4, 32, 12001, 12), (128, 33, 2, 32, 12001, 12), (64, 65, 2, 32, 20001, 12),
         (128, 33, 4, 3, 80001, 12), (64, 100, 1, 8, 80001, 12)]


def some_shared(torch, hd, seqs, nkv, g, prefix_len, own):
    """Queries, a prefix, slices of `own` slots; the first sequences' lengths 1, 1, own."""
    lens = [1, 1, own] + [(5 * b) % (own + 1) for b in range(3, seqs)]
    return rand(torch, 2, seqs, nkv * g * hd), some_layer(torch, 1, nkv, hd, prefix_len), some_layers(torch, 9, seqs, nkv, hd, own), lens


def fine_rows(torch, got, q, prefix, prefix_len, layers, lens, nkv, hd, max_seq, pick, heads=None, window=0):
    """The rows of the sequences `pick` (of every 64-bit row one in a few) are within their bounds, at the heads that `heads` says."""
    pick = sorted(set(pick))
    want, bound = S.shared(q[pick].contiguous(), prefix, prefix_len, prefix_len, layers[pick], [lens[b] for b in pick], nkv, hd, max_seq, window)
    if heads is None:
        within(torch, got[pick], want, bound)
    else:
        at = heads[pick].repeat_interleave(hd, 1)
        within(torch, got[pick][at], want[at], bound[at])


@pytest.mark.parametrize("hd,seqs,nkv,g,prefix_len,own", JOINS)
def test_shared_prefix_queries_that_are_no_numbers(gpu, hd, seqs, nkv, g, prefix_len, own):
    torch = gpu
    q, prefix, layers, lens = some_shared(torch, hd, seqs, nkv, g, prefix_len, own)
    bad, fine = q.clone(), torch.ones((seqs, nkv * g), dtype=torch.bool, device="cuda")
    for b, head, value in ((0, 0, math.nan), (1, nkv * g - 1, math.inf), (2, g // 2, -math.inf), (seqs - 1, 1, math.nan)):
        bad[b, head * hd + 7] = value
        fine[b, head] = False
    got = shared(torch, bad, prefix, prefix_len, prefix_len, layers, ints(torch, lens), nkv, hd, own, own)
    rows = got.reshape(seqs, nkv * g, hd)
    assert rows[~fine].isnan().all() and not rows[fine].isnan().any()
    fine_rows(torch, got, q, prefix, prefix_len, layers, lens, nkv, hd, own, [0, 1, 2, seqs - 1], fine)


@pytest.mark.parametrize("part", [0, 1])
@pytest.mark.parametrize("hd,seqs,nkv,g,prefix_len,own", JOINS)
def test_shared_prefix_own_tokens_that_are_no_numbers(gpu, hd, seqs, nkv, g, prefix_len, own, part):
    """One sequence's only own token, another's newest one; a third's stands behind its length."""
    torch = gpu
    q, prefix, layers, lens = some_shared(torch, hd, seqs, nkv, g, prefix_len, own)
    clean = layers.clone()
    last = seqs - 1 if seqs > 3 else 1
    lens[last] = min(lens[last], own - 1)
    for b, slot in ((0, 0), (2, own - 1), (last, lens[last])):
        poison(torch, layers[b], nkv, hd, own, [slot], part)
    got = shared(torch, q, prefix, prefix_len, prefix_len, layers, ints(torch, lens), nkv, hd, own, own)
    bad = torch.zeros(seqs, dtype=torch.bool, device="cuda")
    bad[[0, 2]] = True
    assert got[bad].isnan().all() and not got[~bad].isnan().any()
    fine_rows(torch, got, q, prefix, prefix_len, clean, lens, nkv, hd, own, [1, last])


@pytest.mark.parametrize("part", [0, 1])
@pytest.mark.parametrize("hd,seqs,nkv,g,prefix_len,own", JOINS)
def test_shared_prefix_a_run_of_tokens_that_are_no_numbers(gpu, hd, seqs, nkv, g, prefix_len, own, part):
    """The prefix's last half in its last KV head: of a long one whole parts. The other heads' rows stay numbers."""
    torch = gpu
    q, prefix, layers, lens = some_shared(torch, hd, seqs, nkv, g, prefix_len, own)
    clean = prefix.clone()
    slots = range(prefix_len // 2, prefix_len)
    at = 128 * hd + 256 * part
    scales = prefix[-1, :, at:at + 256].contiguous().view(torch.float32)  # [tiles][64]
    scales.reshape(-1)[slots.start:slots.stop] = math.nan
    prefix[-1, :, at:at + 256] = scales.view(torch.uint8)
    got = shared(torch, q, prefix, prefix_len, prefix_len, layers, ints(torch, lens), nkv, hd, own, own)
    fine = torch.ones((seqs, nkv * g), dtype=torch.bool, device="cuda")
    fine[:, -g:] = False
    rows = got.reshape(seqs, nkv * g, hd)
    assert rows[~fine].isnan().all() and not rows[fine].isnan().any()
    if nkv > 1:
        fine_rows(torch, got, q, clean, prefix_len, layers, lens, nkv, hd, own, [0, 2, seqs - 1], fine)


@pytest.mark.parametrize("part", [0, 1])
@pytest.mark.parametrize("hd,g,prefix_len", [(128, 4, 300), (64, 4, 321), (256, 2, 64), (128, 17, 65), (128, 4, 5000)])
def test_shared_prefix_a_window_that_leaves_a_token_that_is_no_number(gpu, hd, g, prefix_len, part):
    """The prefix's last token is NaN: alone in some windows, beside own tokens or the one before it in others, and behind others."""
    torch = gpu
    nkv, lens, own = 2, [1, 0, 2, 3, 70], 70
    prefix, layers = some_layer(torch, 1, nkv, hd, prefix_len), some_layers(torch, 9, len(lens), nkv, hd, own)
    q, clean = rand(torch, 2, len(lens), nkv * g * hd), prefix.clone()
    poison(torch, prefix, nkv, hd, prefix_len, [prefix_len - 1], part)
    for window in (1, 2, 3):
        got = shared(torch, q, prefix, prefix_len, prefix_len, layers, ints(torch, lens), nkv, hd, own, own, window)
        sees = [b for b, l in enumerate(lens) if l < window]
        assert got[sees].isnan().all()
        fine_rows(torch, got, q, clean, prefix_len, layers, lens, nkv, hd, own, [b for b in range(len(lens)) if b not in sees], window=window)
