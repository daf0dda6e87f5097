"""The attention over the 8-bit cache where values grow by many powers of ten from
one run of tokens to the next, in every form: the running power of two that the
many-column form keeps its products at has to follow them both ways."""
import pytest

from tests import _kv8 as R
from tests.test_gpu_kv8 import attend, rand, within

pytestmark = pytest.mark.gpu

# n, seq, heads, kv_heads, hd, window: 16 columns whole and split, 128 whole, with a window, split, 256 whole, split
SHAPES = [(1, 1000, 8, 2, 128, 0), (70, 700, 4, 1, 128, 0), (5, 700, 4, 1, 64, 0), (9, 700, 4, 2, 256, 0), (800, 800, 48, 2, 128, 0),
          (600, 600, 64, 8, 64, 0), (1000, 4000, 32, 2, 128, 600), (600, 7600, 7, 1, 64, 0), (700, 3000, 32, 1, 128, 0), (1500, 1500, 64, 8, 128, 0)]


@pytest.mark.parametrize("run,low,high", [(32, 1e-26, 1e11), (64, 1e-25, 1e25), (100, 1e-24, 1e33), (33, 1e-26, 1e20)])
@pytest.mark.parametrize("n,seq,heads,nkv,hd,window", SHAPES)
def test_values_that_rise(gpu, n, seq, heads, nkv, hd, window, run, low, high):
    """Flat scores and random ones; V of the size `low`, and every second run of tokens, or the last one alone, `high`."""
    torch = gpu
    slots = -(-seq // 64) * 64
    base, val = rand(torch, 120, nkv, slots, hd), rand(torch, 121, nkv, slots, hd)
    q = rand(torch, 122, n, heads * hd)
    t = torch.arange(slots, device="cuda")
    for k, up in ((base * 0.0, t // run % 2 == 1), (base * 0.0, t >= seq - n // 2 - 1), (base, t // run % 2 == 1)):
        v = val * torch.where(up, high, low).float()[None, :, None]
        layer = R.pack(*R.codes(k), *R.codes(v))
        got = attend(torch, q, layer, nkv, hd, slots, seq, window)
        want, bound = R.attention(q, layer, nkv, hd, slots, seq, window)
        within(torch, got, want, bound)


@pytest.mark.parametrize("n,seq,heads,nkv,hd", [(1, 131000, 4, 1, 128), (1, 9000, 32, 8, 128), (5, 9000, 4, 2, 256), (70, 9001, 16, 8, 128), (250, 8448, 32, 8, 128),
                                                (100, 7100, 64, 8, 128), (100, 7100, 32, 8, 128), (600, 7600, 7, 1, 64), (333, 20333, 8, 8, 128), (2500, 2500, 64, 8, 128)])
def test_low_bits_of_the_products_over_long_rows(gpu, n, seq, heads, nkv, hd):
    """Flat scores; the tokens' values are c and -c in turn, of scales 1 + 2^-13 and 1, so that the result, c·2^-14, is what is left of
    bits that half a product's number of bits does not hold. Each product may be rounded to 2^-23 of itself (include/aether_hip.h),
    c·2^-23 a token of the mean; what the 16 products of a matrix instruction and the running sum, never above 16·c and 2·c,
    lose over it is (2·16·U/16 + 2·2·U/4)·c = 3·U·c a token, three roundings of the result 3·U of it: 2^-21·c covers them and the
    last token of an odd row."""
    torch = gpu
    slots = -(-seq // 64) * 64
    t = torch.arange(slots, device="cuda")
    c = 1 + torch.arange(hd, device="cuda") % 31
    vc = (torch.where(t % 2 == 0, 1, -1)[:, None] * c).to(torch.int8).expand(nkv, slots, hd).contiguous()
    vs = torch.where(t % 2 == 0, 1.0 + 2.0 ** -13, 1.0).float().expand(nkv, slots).contiguous()
    layer = R.pack(torch.zeros_like(vc), torch.zeros_like(vs), vc, vs)
    q = rand(torch, 123, n, heads * hd)
    got = attend(torch, q, layer, nkv, hd, slots, seq)
    want, _ = R.attention(q, layer, nkv, hd, slots, seq, 0)
    within(torch, got, want, (2.0 ** -21 * c.double()).repeat(heads).expand(n, -1))


@pytest.mark.parametrize("n,seq,heads,nkv,hd,window", SHAPES)
def test_the_ends_of_the_numbers(gpu, n, seq, heads, nkv, hd, window):
    """Keys up to 2^95 and down to 2^-100 with queries that leave scores of ordinary size, scores up to about 2^20, and values whose sum
    of e^(score - maximum)·|value| stays below 2^119 (tokens times 2^5, what `rand` stays below)."""
    torch = gpu
    slots = -(-seq // 64) * 64
    base, val = rand(torch, 124, nkv, slots, hd), rand(torch, 125, nkv, slots, hd)
    q = rand(torch, 126, n, heads * hd)
    assert base.abs().max() < 16 and val.abs().max() < 32  # keys below 16·2^91 = 2^95, sums below 32·2^(118 - 4) = 2^119
    most = 2.0 ** (118 - 4 - (seq - 1).bit_length())
    for kf, qf, vf in ((2.0 ** 91, 2.0 ** -91, 1.0), (2.0 ** -100, 2.0 ** 100, 1.0), (2.0 ** 8, 2.0 ** 8, 1.0), (1.0, 1.0, most), (0.0, 1.0, most),
                       (1.0, 1.0, 2.0 ** -60)):
        layer = R.pack(*R.codes(base * kf), *R.codes(val * vf))
        qs = q * qf
        got = attend(torch, qs, layer, nkv, hd, slots, seq, window)
        want, bound = R.attention(qs, layer, nkv, hd, slots, seq, window)
        within(torch, got, want, bound)


@pytest.mark.parametrize("n,seq,heads,nkv,hd,window", [(1000, 4000, 32, 2, 128, 600), (600, 1600, 64, 8, 64, 700), (600, 1600, 64, 8, 128, 700), (800, 3000, 48, 2, 128, 65)])
def test_uneven_rows_under_a_window(gpu, n, seq, heads, nkv, hd, window):
    """Many columns over scores that rise and fall by hundreds from tile to tile, flat ones, and V scales that mix, fall or are
    large, where every tile has keys that some column does not see. Values of 1e-30 have scales of 2^-104, and products below
    2^-90 keep fewer bits (include/aether_hip.h): times 2^100, the most that a probability below 2^9 bears beside any V scale up to
    2^18, they stand in two parts whose last place is fp16's 2^-24, so that each is off by up to 2^-125 and a row by
    127 · window · 2^-125, its sum of probabilities being 1 or more."""
    torch = gpu
    slots = -(-seq // 64) * 64
    base, val = rand(torch, 127, nkv, slots, hd), rand(torch, 128, nkv, slots, hd)
    q = rand(torch, 129, n, heads * hd)
    t = torch.arange(slots, device="cuda").float()[None, :, None]
    for k, v in ((base * (1.0 + t / 20.0), val), (base * (1.0 + (seq - t).clamp_min(0) / 20.0), val), (base * 0.0, val),
                 (base * 1e-3, val * torch.pow(10.0, (t % 41) - 20.0)), (base, val * torch.pow(10.0, -t / 50.0).clamp_min(1e-30)), (base, val * 1e30)):
        layer = R.pack(*R.codes(k), *R.codes(v))
        want, bound = R.attention(q, layer, nkv, hd, slots, seq, window)
        within(torch, attend(torch, q, layer, nkv, hd, slots, seq, window), want, bound + 127 * window * 2.0 ** -125)
