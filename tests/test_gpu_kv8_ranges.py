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
