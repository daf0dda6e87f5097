"""Shared-prefix attention, attention weights, eviction and positions of several axes
without a GPU: workspace sizes, and the calls that are refused before any device work (an
accepted one would end in a HIP error here, not in the status asserted)."""
import ctypes

import pytest

import aether_amd as A
from tests.test_kv8 import COMMON, P, call

BYTES = 8 * 64 * 264  # a slice of 64 positions, 8 heads of 128

SHARED = dict(q=P, qs=4096, prefix=P, ps=1000, pl=900, layers=P, stride=64 * BYTES, lens=P, seqs=3, nq=32, nkv=8, hd=128, ms=4096, ml=4096, window=0, out=P, ws=P,
              wsb=1 << 40, stream=None)
SLICES = [(dict(layers=None), -1), (dict(layers=P + 8), -1), (dict(lens=None), -1), (dict(lens=P + 2), -1), (dict(seqs=-1), -1), (dict(seqs=70000), -4),
          (dict(ml=0), -1), (dict(ml=4097), -1), (dict(stride=64 * BYTES - 16), -1), (dict(stride=64 * BYTES + 4), -1), (dict(stride=2 ** 62), -1)]


@pytest.mark.parametrize("change,rc", COMMON + SLICES + [
    (dict(prefix=None), -1), (dict(prefix=P + 4), -1), (dict(pl=-1), -1), (dict(pl=1001), -1), (dict(ps=2 ** 31, pl=2 ** 30 + 1), -1),
    (dict(ps=2 ** 30, pl=2 ** 30), -1), (dict(pl=2 ** 62, ps=2 ** 62), -1)])
def test_shared_refuses(change, rc):
    assert call("aeth_attn_kv8_shared", SHARED, change) == rc
    assert "aeth_attn_kv8_shared" in A.last_error()


def test_shared_refuses_more_than_a_grid():
    change = dict(seqs=60000, nq=128, nkv=128, qs=2 ** 14, hd=64, ms=64, ml=64, stride=128 * 64 * 136)
    assert call("aeth_attn_kv8_shared", SHARED, change) == -4


def test_shared_nothing_to_do():
    assert call("aeth_attn_kv8_shared", SHARED, dict(seqs=0)) == 0
    assert call("aeth_attn_kv8_shared", SHARED, dict(seqs=0, prefix=None, pl=0, ps=0)) == 0


WEIGHTS = dict(q=P, qs=4096, layer=P, n=2, nq=32, nkv=8, hd=128, ms=4096, seq=4096, window=0, out=P, prior=None, weights=P, ws=P, wsb=1 << 40, stream=None)
WEIGHTS_BATCH = dict(q=P, qs=4096, layers=P, stride=64 * BYTES, lens=P, seqs=3, nq=32, nkv=8, hd=128, ms=4096, ml=4096, window=0, out=P, prior=None, weights=P,
                     ws=P, wsb=1 << 40, stream=None)


@pytest.mark.parametrize("change,rc", COMMON + [
    (dict(layer=None), -1), (dict(layer=P + 4), -1), (dict(n=-1), -1), (dict(n=5000), -1), (dict(seq=1), -1), (dict(seq=4097), -1), (dict(seq=-1), -1),
    (dict(weights=None), -1), (dict(weights=P + 2), -1), (dict(prior=P + 1), -1), (dict(prior=P + 4), -1), (dict(prior=P - 8 * 4096 * 4 + 4), -1)])
def test_weights_refuse(change, rc):
    assert call("aeth_attn_kv8_weights", WEIGHTS, change) == rc
    assert "aeth_attn_kv8_weights" in A.last_error()


@pytest.mark.parametrize("change,rc", COMMON + SLICES + [
    (dict(weights=None), -1), (dict(weights=P + 1), -1), (dict(prior=P + 2), -1), (dict(prior=P + 3 * 8 * 4096 * 4 - 4), -1)])
def test_batch_weights_refuse(change, rc):
    assert call("aeth_attn_kv8_weights_batch", WEIGHTS_BATCH, change) == rc
    assert "aeth_attn_kv8_weights_batch" in A.last_error()


def test_weights_refuse_more_than_a_grid():
    change = dict(nq=64, nkv=64, qs=2 ** 14, hd=64, n=1, seq=2 ** 26, ms=2 ** 26, wsb=2 ** 62)
    assert call("aeth_attn_kv8_weights", WEIGHTS, change) == -4


def test_weights_nothing_to_do():
    assert call("aeth_attn_kv8_weights", WEIGHTS, dict(n=0, seq=0)) == 0
    assert call("aeth_attn_kv8_weights", WEIGHTS, dict(n=0, seq=0, q=None, out=None)) == 0
    assert call("aeth_attn_kv8_weights_batch", WEIGHTS_BATCH, dict(seqs=0)) == 0


def test_workspaces():
    L = A.lib()
    for ws, args, sizes in ((L.aeth_attn_kv8_shared_ws_bytes, (3, 32, 8, 128, 1000, 500), (0, 4, 5)),
                            (L.aeth_attn_kv8_weights_ws_bytes, (1, 100, 32, 8, 128, 5000), (0, 1, 5)),
                            (L.aeth_attn_kv8_weights_ws_bytes, (3, 1, 32, 8, 128, 5000), (0, 1, 5)),
                            (L.aeth_kv8_evict_ws_bytes, (3, 8, 128, 5000, 1000, 1), (0, 3, 4, 5))):
        most = ws(*args)
        assert most > 0
        for i in sizes:
            for less in (args[i] - 1, args[i] // 2, 0):
                smaller = list(args)
                smaller[i] = less
                assert 0 <= ws(*smaller) <= most, smaller
    # scores of few columns cost more than the sums of many
    for length in (100, 5000, 100000):
        for n in (1, 11, 12, 13, 15, 16, 17, 64, 500):
            assert L.aeth_attn_kv8_weights_ws_bytes(1, n, 32, 8, 128, length) <= L.aeth_attn_kv8_weights_ws_bytes(1, n + 1, 32, 8, 128, length)
    for bad in ((-1, 32, 8, 128, 10, 10), (3, 30, 8, 128, 10, 10), (3, 32, 8, 96, 10, 10), (3, 32, 8, 128, -1, 10), (3, 32, 8, 128, 10, -1),
                (3, 32, 8, 128, 2 ** 31, 10)):
        assert L.aeth_attn_kv8_shared_ws_bytes(*bad) == -1, bad
    for bad in ((-1, 1, 32, 8, 128, 64), (1, -1, 32, 8, 128, 64), (1, 1, 30, 8, 128, 64), (1, 1, 32, 8, 96, 64), (1, 1, 32, 8, 128, -1)):
        assert L.aeth_attn_kv8_weights_ws_bytes(*bad) == -1, bad
    assert L.aeth_attn_kv8_weights_ws_bytes(65535, 2 ** 24, 4096, 4096, 64, 2 ** 30) == -1  # past 64 bits
    for bad in ((-1, 8, 128, 10, 5, 0), (70000, 8, 128, 10, 5, 0), (1, 0, 128, 10, 5, 0), (1, 8, 100, 10, 5, 0), (1, 8, 128, -1, 5, 0), (1, 8, 128, 10, -1, 0),
                (1, 8, 128, 2 ** 31, 5, 0)):
        assert L.aeth_kv8_evict_ws_bytes(*bad) == -1, bad
        assert "aeth_kv8_evict_ws_bytes" in A.last_error()


FAR = 1 << 40
EVICT = dict(layer=P, weights=FAR, nkv=8, hd=128, ms=4096, seq=3000, keep=1000, first=4, recent=64, dst=2 * FAR, dw=3 * FAR, ds=1024, kept=P, ws=P, wsb=1 << 50,
             stream=None)
EVICT_BATCH = dict(layers=P, stride=64 * BYTES, weights=FAR, lens=P, seqs=3, nkv=8, hd=128, ms=4096, ml=3000, keep=1000, first=4, recent=64, dst=2 * FAR,
                   dstride=16 * BYTES, dw=3 * FAR, ds=1024, dl=P, kept=P, ws=P, wsb=1 << 50, stream=None)
CUTS = [(dict(weights=None), -1), (dict(weights=FAR + 1), -1), (dict(dst=None), -1), (dict(dst=2 * FAR + 8), -1), (dict(dw=3 * FAR + 2), -1),
        (dict(kept=P + 1), -1), (dict(ws=P + 4), -1), (dict(ws=None), -1), (dict(wsb=100), -1), (dict(nkv=0), -1), (dict(nkv=70000), -1), (dict(hd=96), -4),
        (dict(ms=0), -1), (dict(ms=2 ** 31), -1), (dict(ds=0), -1), (dict(ds=999), -1), (dict(ds=2 ** 31), -1), (dict(keep=-1), -1), (dict(first=-1), -1),
        (dict(recent=-1), -1), (dict(first=1001), -1), (dict(recent=997), -1), (dict(first=2 ** 62, recent=2 ** 62), -1),
        (dict(dst=P), -1), (dict(dst=P + 16), -1), (dict(dw=FAR), -1), (dict(dw=FAR + 4), -1), (dict(dw=FAR - 4), -1)]


@pytest.mark.parametrize("change,rc", CUTS + [(dict(layer=None), -1), (dict(layer=P + 8), -1), (dict(seq=-1), -1), (dict(seq=4097), -1),
                                              (dict(dst=P + 64 * BYTES - 16), -1), (dict(dst=P, ds=4032), -1)])
def test_evict_refuses(change, rc):
    assert call("aeth_kv8_evict", EVICT, change) == rc
    assert "aeth_kv8_evict" in A.last_error()


@pytest.mark.parametrize("change,rc", CUTS + [
    (dict(keep=2 ** 62), -1), (dict(layers=None), -1), (dict(lens=None), -1), (dict(lens=P + 1), -1), (dict(dl=P + 2), -1), (dict(seqs=-1), -1), (dict(seqs=70000), -1), (dict(ml=-1), -1),
    (dict(ml=4097), -1), (dict(stride=64 * BYTES - 16), -1), (dict(stride=64 * BYTES + 8), -1), (dict(stride=2 ** 62), -1), (dict(dstride=16 * BYTES - 16), -1),
    (dict(dstride=-16), -1), (dict(dst=P + 64 * BYTES), -1), (dict(dst=P, ds=4096, dstride=65 * BYTES), -1),
    (dict(seqs=60000, nkv=60000, stride=60000 * 64 * 64 * 264, dstride=60000 * 16 * 64 * 264, dst=1 << 62), -1)])
def test_batch_evict_refuses(change, rc):
    assert call("aeth_kv8_evict_batch", EVICT_BATCH, change) == rc
    assert "aeth_kv8_evict_batch" in A.last_error()


def test_evict_nothing_to_do():
    assert call("aeth_kv8_evict_batch", EVICT_BATCH, dict(seqs=0)) == 0


QK = dict(x=P, xs=6144, n=3, nq=32, nk=8, hd=128, qw=P, kw=P, eps=1e-5, pos=P, ps=3, axes=3, pairs=None, sin=P, cos=P, ms=64, out=2 * P, os=5120, stream=None)


def pairs(n, value=0, at=0):
    a = (ctypes.c_int32 * max(n, 1))()
    if n:
        a[at] = value
    return a


@pytest.mark.parametrize("change,rc", [
    (dict(x=None), -1), (dict(out=None), -1), (dict(sin=None), -1), (dict(cos=None), -1), (dict(n=-1), -1), (dict(nq=-1), -1),
    (dict(nk=-1), -1), (dict(hd=127), -1), (dict(hd=0), -1), (dict(ms=0), -1), (dict(pos=None), -1), (dict(pos=P + 2), -1), (dict(pairs=0), -1),
    (dict(xs=5119), -1), (dict(os=5119), -1), (dict(xs=2 ** 62), -1), (dict(out=P), -1), (dict(axes=0), -1), (dict(axes=-1), -1), (dict(axes=17, ps=3), -4),
    (dict(ps=2), -1), (dict(ps=-3), -1), (dict(ps=2 ** 62), -1), (dict(hd=514, xs=2 ** 15, os=2 ** 15), -4), (dict(nq=70000, xs=2 ** 40, os=2 ** 40), -4),
    (dict(n=2 ** 25, xs=2 ** 14, os=2 ** 14, ps=2 ** 25), -4)])
def test_axes_refuse(change, rc):
    table = pairs(257)
    args = dict(change)
    args["pairs"] = None if "pairs" in change else ctypes.addressof(table)
    assert call("aeth_qk_norm_rope_axes", QK, args) == rc
    assert "aeth_qk_norm_rope_axes" in A.last_error()


@pytest.mark.parametrize("value,at", [(3, 0), (-1, 63), (2 ** 31 - 1, 17)])
def test_axes_refuse_a_pair_of_no_axis(value, at):
    table = pairs(64, value, at)
    assert call("aeth_qk_norm_rope_axes", QK, dict(pairs=ctypes.addressof(table))) == -1
    assert "pair %d" % at in A.last_error()


def test_axes_nothing_to_do():
    table = pairs(64)
    assert call("aeth_qk_norm_rope_axes", QK, dict(n=0, pairs=ctypes.addressof(table))) == 0
    assert call("aeth_qk_norm_rope_axes", QK, dict(nq=0, nk=0, pairs=ctypes.addressof(table))) == 0
