"""Appends of many tokens to the 8-bit cache, which go by whole tiles through LDS (k_kv8_append), against the
definition byte for byte and against the same tokens a few at a time, which do not (k_kv8_append_few)."""
import pytest

import aether_amd as A
from tests import _kv8 as R
from tests.test_gpu_kv8 import append, check_stored, new_layer, rand, some_layer, stream

pytestmark = pytest.mark.gpu


def many(torch, nkv):
    """More tokens than any launch leaves to the kernel for a few: 14 rows and heads a CU, and a tile."""
    return 14 * torch.cuda.get_device_properties(0).multi_processor_count // nkv + 64


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("nkv,extra,slot,behind", [(8, 0, 0, 0), (8, 1, 37, 5), (3, 22, 62, 200), (1, 63, 129, 1), (30, 3, 3, 64), (8, 2, 64, 63)])
def test_many_tokens_from_any_slot(gpu, hd, nkv, extra, slot, behind):
    """Starts and ends anywhere in a tile and in a group of four tokens; slots before, behind, and in the tiles in between."""
    torch = gpu
    n = many(torch, nkv) + extra
    max_seq = slot + n + behind
    k, v = rand(torch, 130 + slot, n, nkv * hd), rand(torch, 131 + slot, n, nkv * hd)
    k[n // 2], v[n // 3] = 0.0, 0.0
    layer = new_layer(torch, nkv, hd, max_seq)
    append(torch, layer, k, v, nkv, hd, max_seq, slot)
    check_stored(torch, layer, k, v, nkv, hd, max_seq, slot)
    back = torch.full((2, n, nkv * hd), 7.0, device="cuda")
    A.check(A.lib().aeth_kv8_read(layer.data_ptr(), back[0].data_ptr(), back[1].data_ptr(), nkv * hd, hd, n, nkv, hd, max_seq, slot, stream(torch)), "read")
    for x, b in zip((k, v), back):
        c, s = R.codes(x.reshape(n, nkv, hd))
        assert torch.equal(b.reshape(n, nkv, hd), c.float() * s[..., None])


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_tokens_of_any_strides(gpu, hd):
    """Rows as a fused projection leaves them, [heads][slots][hd], and ones that are not 16-byte aligned, over a cache that is
    in use: nothing but the new slots changes."""
    torch = gpu
    nkv, slot = 4, 30
    n = many(torch, nkv) + 9
    max_seq = slot + n + 70
    x = rand(torch, 140, 2, n, nkv, hd)
    old = some_layer(torch, 141, nkv, hd, max_seq)
    for ts, hs, shift in ((12 * hd, hd, 0), (hd, (n + 20) * hd, 0), (12 * hd + 1, hd, 0), (12 * hd, hd + 3, 1), (nkv * hd, hd, 3)):
        buf = torch.zeros((2, (n - 1) * ts + (nkv - 1) * hs + hd + shift), device="cuda")
        for b, y in zip(buf, x):
            torch.as_strided(b, (n, nkv, hd), (ts, hs, 1), b.storage_offset() + shift).copy_(y)
        layer = old.clone()
        append(torch, layer, buf[0, shift:], buf[1, shift:], nkv, hd, max_seq, slot, ts, hs, n)
        want = [t.clone() for t in R.unpack(old, nkv, hd, max_seq)]
        for y, c, s in ((x[0], want[0], want[2]), (x[1], want[1], want[3])):
            c[:, slot:slot + n], s[:, slot:slot + n] = R.codes(y.transpose(0, 1))
        assert torch.equal(layer, R.pack(want[0], want[2], want[1], want[3])), (ts, hs, shift)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_tokens_at_once_and_in_pieces(gpu, hd):
    """Infinities, NaN and rows of zeros among them: the bytes of one append are those of many small ones."""
    torch = gpu
    nkv, slot = 8, 21
    n = many(torch, nkv) + 77
    max_seq = slot + n + 3
    k, v = rand(torch, 150, n, nkv * hd), rand(torch, 151, n, nkv * hd)
    k[5, 3], k[n - 2, hd + 1], v[64, 7], v[n // 2, 2 * hd] = float("inf"), float("nan"), float("-inf"), float("nan")
    k[9], v[10, :hd] = 0.0, -0.0
    whole, parts = new_layer(torch, nkv, hd, max_seq), new_layer(torch, nkv, hd, max_seq)
    append(torch, whole, k, v, nkv, hd, max_seq, slot)
    at = 0
    while at < n:
        size = min((1, 7, 64, 100)[at % 4], n - at)
        append(torch, parts, k[at:at + size], v[at:at + size], nkv, hd, max_seq, slot + at)
        at += size
    assert torch.equal(whole, parts)


@pytest.mark.parametrize("n", [4, 4000])
def test_quotients_next_to_a_tie(gpu, n):
    """127·x / amax nearest to a half that two f32 come with x eight binades below amax: 2^-32 from it."""
    torch = gpu
    nkv, hd = 1, 128
    k = torch.zeros((n, hd), device="cuda")
    for i, (amax, x) in enumerate(((16643351.0, 16774401.0 * 2.0 ** -8), (16639922.0, 16770945.0 * 2.0 ** -8), (16643351.0, 16774402.0 * 2.0 ** -8),
                                   (16639922.0, 16770946.0 * 2.0 ** -8))):
        k[i::4] = x
        k[i::4, 1::2] = -x
        k[i::4, 7] = amax
    off = (k[:2, 0].double() * 127.0 / k[:2, 7].double() - 0.5).abs().tolist()
    assert 0.0 < min(off) and max(off) < 2.0 ** -31
    layer = new_layer(torch, nkv, hd, n + 5)
    append(torch, layer, k, -k, nkv, hd, n + 5, 2)
    check_stored(torch, layer, k, -k, nkv, hd, n + 5, 2)
