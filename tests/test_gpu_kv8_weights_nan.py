"""The weights that cached tokens receive beside a token that is no number, where a part of a
split row sees nothing else: a query that sees it has a NaN row and makes the weights of all that
it sees NaN, the others are held to 64 bits (tests/_kv8_serve.py)."""
import pytest

from tests import _kv8_serve as S
from tests.test_gpu_kv8 import rand, some_layer, within
from tests.test_gpu_kv8_serve import ints, poison, some_layers, weigh, weigh_batch

pytestmark = pytest.mark.gpu

# lengths one above what whole parts hold, so that the newest token is a part by itself; few columns, whose scores are kept, in one part, in
# a few and in many, and more, whose scores are formed again
SINGLE = [(128, 1, 2049, 8, 4, 0), (64, 1, 2049, 2, 4, 0), (256, 1, 1025, 2, 4, 0), (128, 1, 257, 1, 1, 0), (128, 1, 769, 2, 17, 0), (128, 1, 20225, 1, 4, 0),
          (128, 1, 2049, 2, 4, 1100), (128, 6, 2049, 8, 4, 0), (64, 12, 1281, 2, 4, 700), (256, 3, 1025, 1, 8, 0), (128, 20, 600, 2, 1, 3),
          (128, 100, 2049, 2, 4, 0), (64, 70, 1281, 2, 4, 1000)]


@pytest.mark.parametrize("part", [0, 1])
@pytest.mark.parametrize("hd,n,seq,nkv,g,window", SINGLE)
def test_weights_of_a_newest_token_that_is_no_number(gpu, hd, n, seq, nkv, g, window, part):
    """Only the last query sees it."""
    torch = gpu
    layer, q, prior = some_layer(torch, n, nkv, hd, seq), rand(torch, 3, n, nkv * g * hd), rand(torch, 5, nkv, seq).abs()
    poison(torch, layer, nkv, hd, seq, [seq - 1], part)
    out, w = weigh(torch, q, layer, nkv, hd, seq, seq, window, prior)
    first = max(0, seq - window) if window else 0
    assert out[n - 1].isnan().all() and w[:, first:].isnan().all()
    o, ot, ww, wt = S.weights(q[:n - 1], layer, nkv, hd, seq, seq - 1, window, prior)
    within(torch, out[:n - 1], o, ot)
    within(torch, w[:, :first], ww[:, :first], wt[:, :first])


@pytest.mark.parametrize("part", [0, 1])
@pytest.mark.parametrize("hd,n,nkv,g", [(128, 1, 2, 4), (64, 6, 2, 4), (256, 2, 3, 4), (128, 60, 2, 4)])
def test_weights_of_a_run_of_tokens_that_are_no_numbers(gpu, hd, n, nkv, g, part):
    """Whole parts of the first KV head; the other heads' rows and weights stay numbers."""
    torch = gpu
    seq = 1700
    layer, q = some_layer(torch, n, nkv, hd, seq), rand(torch, 3, n, nkv * g * hd)
    poison(torch, layer[:1], 1, hd, seq, range(500, 1100), part)
    clean = some_layer(torch, n, nkv, hd, seq)
    out, w = weigh(torch, q, layer, nkv, hd, seq, seq)
    assert out[:, :g * hd].isnan().all() and w[0].isnan()[:seq - n + 1].all()
    o, ot, ww, wt = S.weights(q, clean, nkv, hd, seq, seq, 0, None)
    within(torch, out[:, g * hd:], o[:, g * hd:], ot[:, g * hd:])
    within(torch, w[1:], ww[1:], wt[1:])


@pytest.mark.parametrize("part", [0, 1])
@pytest.mark.parametrize("hd,nkv,g,window", [(128, 8, 4, 0), (64, 2, 8, 0), (256, 2, 2, 0), (128, 2, 70, 0), (128, 2, 4, 600)])
def test_batch_weights_of_newest_tokens_that_are_no_numbers(gpu, hd, nkv, g, window, part):
    torch = gpu
    lens, most, bad = [2049, 1, 257, 2048, 0, 1500, 513], 2100, [0, 1, 2, 6]
    layers, q, prior = some_layers(torch, 3, len(lens), nkv, hd, most), rand(torch, 4, len(lens), nkv * g * hd), rand(torch, 5, len(lens), nkv, most).abs()
    for b in bad:
        poison(torch, layers[b], nkv, hd, most, [lens[b] - 1], part)
    out, w = weigh_batch(torch, q, layers, ints(torch, lens), nkv, hd, most, 2049, window, prior)
    for b, seq in enumerate(lens):
        first = max(0, seq - window) if window else 0
        assert (w[b, :, seq:] == 7.0).all()
        if b in bad:
            assert out[b].isnan().all() and w[b, :, first:seq].isnan().all() and torch.equal(w[b, :, :first], prior[b, :, :first])
        elif seq:
            o, ot, ww, wt = S.weights(q[b:b + 1], layers[b], nkv, hd, most, seq, window, prior[b])
            within(torch, out[b:b + 1], o, ot)
            within(torch, w[b, :, :seq], ww, wt)
        else:
            assert (out[b] == 0).all()
