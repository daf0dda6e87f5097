"""The 8-bit cache, its attention and the head norms without a GPU: the layout's
size, and the calls that are refused before any device work (an accepted one
would end in a HIP error here, not in the status asserted)."""
import pytest

import aether_amd as A

P = 1 << 20  # an address that is never dereferenced


def test_layer_bytes():
    L = A.lib()
    for nkv, hd, ms in ((8, 128, 4096), (1, 64, 1), (2, 256, 65), (8, 128, 1 << 30)):
        assert L.aeth_kv8_layer_bytes(nkv, hd, ms) == nkv * -(-ms // 64) * 64 * (2 * hd + 8)
    for nkv, hd, ms, rc in ((0, 128, 64, -1), (8, 128, 0, -1), (8, 128, (1 << 30) + 1, -1), (8, 96, 64, -1), (70000, 128, 64, -1)):
        assert L.aeth_kv8_layer_bytes(nkv, hd, ms) == rc, (nkv, hd, ms)
    assert "head_dim" in A.last_error() or "shape" in A.last_error()


def call(name, base, change):
    args = dict(base)
    args.update(change)
    return getattr(A.lib(), name)(*args.values())


APPEND = dict(layer=P, k=P, v=P, ts=1024, hs=128, n=4, nkv=8, hd=128, ms=64, slot=0, stream=None)


@pytest.mark.parametrize("name", ["aeth_kv8_append", "aeth_kv8_read"])
@pytest.mark.parametrize("change,rc", [
    (dict(layer=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(layer=P + 8), -1), (dict(k=P + 2), -1),
    (dict(nkv=0), -1), (dict(nkv=-1), -1), (dict(hd=80), -4), (dict(hd=0), -4), (dict(ms=0), -1), (dict(ms=2 ** 31), -1),
    (dict(n=-1), -1), (dict(n=65), -1), (dict(slot=-1), -1), (dict(slot=61), -1), (dict(slot=65, n=0), -1),
    (dict(slot=2 ** 63 - 1, n=2), -1), (dict(n=2 ** 63 - 1, slot=1), -1),
    (dict(ts=-1), -1), (dict(ts=127), -1), (dict(hs=127), -1), (dict(hs=-128), -1), (dict(ts=2 ** 62), -1), (dict(hs=2 ** 61), -1),
    (dict(n=2 ** 28, ms=2 ** 30, nkv=64), -4)])
def test_append_and_read_refuse(name, change, rc):
    assert call(name, APPEND, change) == rc
    assert name in A.last_error()


def test_nothing_to_do_is_no_error():
    assert call("aeth_kv8_append", APPEND, dict(n=0)) == 0
    assert call("aeth_kv8_read", APPEND, dict(n=0, slot=64)) == 0
    assert call("aeth_kv8_append_batch", BATCH_APPEND, dict(seqs=0)) == 0
    assert call("aeth_attn_kv8", ATTN, dict(n=0)) == 0
    assert call("aeth_attn_kv8_batch", BATCH, dict(seqs=0)) == 0
    assert call("aeth_qk_norm_rope", QK, dict(n=0)) == 0
    assert call("aeth_qk_norm_rope", QK, dict(nq=0, nk=0)) == 0


BYTES = 8 * 64 * 264
BATCH_APPEND = dict(layers=P, stride=BYTES, slots=P, k=P, v=P, ts=1024, hs=128, seqs=3, nkv=8, hd=128, ms=64, stream=None)


@pytest.mark.parametrize("change,rc", [
    (dict(layers=None), -1), (dict(slots=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(slots=P + 1), -1),
    (dict(stride=BYTES - 16), -1), (dict(stride=BYTES + 8), -1), (dict(stride=-BYTES), -1), (dict(stride=2 ** 62), -1),
    (dict(seqs=-1), -1), (dict(seqs=70000), -1), (dict(hd=100), -4), (dict(ts=100), -1), (dict(ms=0), -1)])
def test_batch_append_refuses(change, rc):
    assert call("aeth_kv8_append_batch", BATCH_APPEND, change) == rc
    assert "aeth_kv8_append_batch" in A.last_error()


def test_batch_append_refuses_more_than_a_grid():
    heads = 60000
    change = dict(seqs=60000, nkv=heads, stride=heads * 64 * 264, ts=heads * 128)
    assert call("aeth_kv8_append_batch", BATCH_APPEND, change) == -4


ATTN = dict(q=P, qs=4096, layer=P, n=2, nq=32, nkv=8, hd=128, ms=4096, seq=4096, window=0, out=P, ws=P, wsb=1 << 40, stream=None)
BATCH = dict(q=P, qs=4096, layers=P, stride=64 * BYTES, lens=P, seqs=3, nq=32, nkv=8, hd=128, ms=4096, ml=4096, window=0, out=P, ws=P,
             wsb=1 << 40, stream=None)
COMMON = [
    (dict(q=None), -1), (dict(out=None), -1), (dict(q=P + 1), -1), (dict(out=P + 2), -1), (dict(ws=P + 8), -1),
    (dict(nq=0), -1), (dict(nq=30), -1), (dict(nkv=0), -1), (dict(nkv=-8), -1), (dict(hd=96), -4), (dict(hd=512), -4), (dict(ms=0), -1),
    (dict(ms=2 ** 31), -1), (dict(window=-1), -1), (dict(qs=4095), -1), (dict(qs=-4096), -1), (dict(qs=2 ** 62), -1),
    (dict(ws=None), -1), (dict(wsb=0), -1), (dict(wsb=-1), -1), (dict(nq=8192, qs=2 ** 20), -4)]


@pytest.mark.parametrize("change,rc", COMMON + [
    (dict(layer=None), -1), (dict(layer=P + 4), -1), (dict(n=-1), -1), (dict(n=5000), -1), (dict(seq=1), -1), (dict(seq=4097), -1),
    (dict(seq=-1), -1), (dict(n=2 ** 23, seq=2 ** 24, ms=2 ** 24, nq=4096, nkv=4096, qs=2 ** 20), -4)])
def test_attention_refuses(change, rc):
    assert call("aeth_attn_kv8", ATTN, change) == rc
    assert "aeth_attn_kv8" in A.last_error()


@pytest.mark.parametrize("change,rc", COMMON + [
    (dict(layers=None), -1), (dict(lens=None), -1), (dict(lens=P + 2), -1), (dict(seqs=-1), -1), (dict(seqs=70000), -4),
    (dict(ml=0), -1), (dict(ml=4097), -1), (dict(stride=64 * BYTES - 16), -1), (dict(stride=64 * BYTES + 4), -1), (dict(stride=2 ** 62), -1)])
def test_batch_attention_refuses(change, rc):
    assert call("aeth_attn_kv8_batch", BATCH, change) == rc
    assert "aeth_attn_kv8_batch" in A.last_error()


def test_workspace_covers_smaller_calls():
    ws = A.lib().aeth_attn_kv8_ws_bytes
    assert ws(1, 1, 32, 8, 128, 256) == 0
    for n in (1, 7, 100):
        for length in (257, 4096, 131072):
            w = ws(3, n, 32, 8, 128, length)
            assert w > 0 and w % 4 == 0
            assert ws(2, n, 32, 8, 128, length) <= w and ws(3, max(1, n - 3), 32, 8, 128, length - 1) <= w
    for bad in ((-1, 1, 32, 8, 128, 64), (1, -1, 32, 8, 128, 64), (1, 1, 30, 8, 128, 64), (1, 1, 32, 8, 96, 64), (1, 1, 32, 8, 128, -1),
                (1, 1, 32, 0, 128, 64), (1, 2 ** 40, 32, 8, 128, 64)):
        assert ws(*bad) == -1, bad


QK = dict(x=P, xs=6144, n=3, nq=32, nk=8, hd=128, qw=P, kw=P, eps=1e-5, pos=0, dpos=None, sin=P, cos=P, ms=64, out=2 * P, os=5120, stream=None)


@pytest.mark.parametrize("change,rc", [
    (dict(x=None), -1), (dict(out=None), -1), (dict(sin=None), -1), (dict(cos=None), -1), (dict(n=-1), -1), (dict(nq=-1), -1),
    (dict(nk=-1), -1), (dict(hd=127), -1), (dict(hd=0), -1), (dict(hd=-2), -1), (dict(ms=0), -1), (dict(pos=-1), -1),
    (dict(xs=5119), -1), (dict(os=5119), -1), (dict(xs=2 ** 62), -1), (dict(out=P), -1), (dict(pos=2 ** 63 - 2, n=5), -1),
    (dict(nq=70000, xs=2 ** 40, os=2 ** 40), -4), (dict(n=2 ** 25, xs=2 ** 14, os=2 ** 14), -4)])
def test_head_norms_refuse(change, rc):
    assert call("aeth_qk_norm_rope", QK, change) == rc
    assert "aeth_qk_norm_rope" in A.last_error()
