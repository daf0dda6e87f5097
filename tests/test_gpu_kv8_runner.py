"""The device runner with its cache in 8 bits (AETH_CFG_KV_INT8): the cache's
bytes through the host copies, decode, prefill, generate, windows and long
contexts. References: the CPU oracle's decode step over the values that the
codes stand for, and the model in float64 with an 8-bit cache (tests/_kv8.py)."""
import ctypes

import numpy as np
import pytest

import aether_amd as A
from oracle import oracle as O
from tests import _kv8 as R
from tests._models import TINY, build_tiny, oracle_cfg
from tests._util import Q2_K, Q4_K, Q8_0, assert_close_logits
from tests.test_gpu_context import _random_cache
from tests.test_gpu_decode import make_runner

pytestmark = pytest.mark.gpu

INT8 = dict(TINY, max_seq_len=256, flags=A.CFG_KV_INT8)
# A K or V entry differs between f32 sums and the exact model by up to about 4e-6 of its row's largest, so
# 127 · 8e-6 · 128 = 0.13 of a row's codes fall the other way of a border, a step of 1/127 of the largest each: 2e-3 of the
# row's length where one row decides, in each of the two layers.
FLOOR = 5e-3


def cache_of(r, c):
    kv = np.empty((c["num_layers"], 2, c["num_kv_heads"], c["max_seq_len"], c["head_dim"]), np.float32)
    fill = ctypes.c_int32()
    A.check(A.lib().aeth_runner_kv_to_host(r, kv.ctypes.data, ctypes.byref(fill)))
    return kv, fill.value


def decode(r, c, token, pos):
    logits, nxt = np.empty(c["vocab_size"], np.float32), ctypes.c_int32()
    A.check(A.lib().aeth_runner_decode(r, token, pos, logits.ctypes.data, ctypes.byref(nxt)), "decode")
    assert nxt.value == O.argmax(logits)
    return logits


def prefill(r, c, tokens):
    t, logits = np.asarray(tokens, np.int32), np.empty(c["vocab_size"], np.float32)
    A.check(A.lib().aeth_runner_prefill(r, t.ctypes.data, len(t), logits.ctypes.data, None), "prefill")
    return logits


def test_cache_copies_hold_the_quantised_values(gpu):
    L, c = A.lib(), INT8
    r = make_runner(build_tiny(seed=20, c=c), c)
    try:
        kv, fill = cache_of(r, c)
        assert fill == 0 and not kv.any()
        x = _random_cache(c, 200, 1)
        x[0, 1, 0, 7] = 0.0
        x[1, 0, 1, 8, 5] = np.inf
        A.check(L.aeth_runner_kv_from_host(r, x.ctypes.data, 200))
        kv, fill = cache_of(r, c)
        assert fill == 200 and np.array_equal(kv, R.quantised(x), equal_nan=True) and np.isnan(kv[1, 0, 1, 8]).all()
        # the benchmark's fill: the f32 runner's numbers, quantised, and nothing behind them
        A.check(L.aeth_runner_fill_kv(r, 77, 100))
        kv, fill = cache_of(r, c)
        f = dict(c, flags=0)
        r32 = make_runner(build_tiny(seed=20, c=f), f)
        try:
            A.check(L.aeth_runner_fill_kv(r32, 77, 100))
            kv32, _ = cache_of(r32, f)
        finally:
            L.aeth_runner_free(r32)
        assert fill == 100 and np.array_equal(kv, R.quantised(kv32)) and not kv[:, :, :, 100:].any()
    finally:
        L.aeth_runner_free(r)


@pytest.mark.parametrize("heads,kv_heads,window", [(4, 2, 0), (8, 1, 0), (6, 6, 0), (4, 2, 300), (6, 2, 0)])
def test_decode_over_a_filled_cache_matches_the_oracle(gpu, heads, kv_heads, window):
    """Steps behind 1000 cached tokens, whose values the oracle takes as they stand; the steps' own tokens are
    f32 there (8 bits of one token in a thousand)."""
    L = A.lib()
    c = dict(TINY, max_seq_len=1200, num_heads=heads, num_kv_heads=kv_heads, flags=A.CFG_KV_INT8, sliding_window=window)
    m = build_tiny(seed=21, c=c)
    r = make_runner(m, c)
    try:
        kv = _random_cache(c, 1000, 2)
        A.check(L.aeth_runner_kv_from_host(r, kv.ctypes.data, 1000))
        kv, fill = cache_of(r, c)
        s, co = O.precompute_rope(c["max_seq_len"], c["head_dim"], c["rope_base"])
        for i in range(3):
            logits = decode(r, c, 9 + i, fill)
            ref, fill = O.decode_step(oracle_cfg(c), m["emb"][9 + i], fill, m["layers"], m["layer_dtype"], m["norms"], m["final"], m["lm"], m["lm_dtype"],
                                      s, co, kv, fill)
            assert_close_logits(logits, ref, floor=FLOOR, what="step %d" % i)
        assert L.aeth_runner_seq_len(r) == 1003
    finally:
        L.aeth_runner_free(r)


@pytest.mark.parametrize("layer_dtype", [Q4_K, Q8_0, Q2_K])
@pytest.mark.parametrize("n,window", [(1, 0), (17, 0), (64, 0), (150, 0), (150, 40)])
def test_prefill_and_steps_match_the_exact_model(gpu, layer_dtype, n, window):
    L = A.lib()
    c = dict(INT8, sliding_window=window)
    m = build_tiny(seed=22, layer_dtype=layer_dtype, c=c)
    r = make_runner(m, c)
    tokens = list(np.random.default_rng(n).integers(0, c["vocab_size"], n))
    try:
        got = prefill(r, c, tokens)
        assert_close_logits(got, R.model_logits(c, m, tokens), floor=FLOOR, what="prefill")
        kv, fill = cache_of(r, c)
        assert fill == n and np.array_equal(kv, R.quantised(kv)) and not kv[:, :, :, n:].any()
        for i in range(3):
            tokens.append((31 * i + 5) % c["vocab_size"])
            got = decode(r, c, int(tokens[-1]), n + i)
            assert_close_logits(got, R.model_logits(c, m, tokens), floor=FLOOR, what="step %d" % i)
        kv, fill = cache_of(r, c)
        assert fill == n + 3 and np.array_equal(kv, R.quantised(kv)) and not kv[:, :, :, n + 3:].any()
    finally:
        L.aeth_runner_free(r)


@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (8, 1), (6, 6)])
def test_steps_fill_the_cache_as_a_prompt_does(gpu, heads, kv_heads):
    """Token by token through every place of two tiles, against the same tokens as a prompt. Layer 0 has the same
    inputs: its sums differ in their order, so an entry by at most one code, a step of 1/127 of its row's largest;
    layer 1's inputs then differ by about 2e-3 of their size, and its rows by twice that at most."""
    L = A.lib()
    c = dict(INT8, num_heads=heads, num_kv_heads=kv_heads)
    m = build_tiny(seed=26, c=c)
    tokens = list(np.random.default_rng(8).integers(0, c["vocab_size"], 130))
    r, p = make_runner(m, c), make_runner(m, c)
    try:
        for i, t in enumerate(tokens):
            logits = decode(r, c, int(t), i)
        want = prefill(p, c, tokens)
        (a, fa), (b, fb) = cache_of(r, c), cache_of(p, c)
        assert fa == fb == 130 and not a[:, :, :, 130:].any()
        for layer, slack in ((0, 1.01 / 127), (1, 1.01 / 127 + 8e-3)):
            big = np.abs(b[layer, :, :, :130]).max(-1, keepdims=True)
            assert (np.abs(a[layer, :, :, :130] - b[layer, :, :, :130]) <= slack * big).all(), layer
        exact = R.model_logits(c, m, tokens)
        for got in (logits, want):
            assert np.abs(got - exact).max() <= FLOOR * np.abs(exact).max()
    finally:
        L.aeth_runner_free(r)
        L.aeth_runner_free(p)


def test_long_prompt(gpu):
    """Past the smallest workgroups of the prompt's attention, its split and its join."""
    L = A.lib()
    c = dict(TINY, max_seq_len=1100, flags=A.CFG_KV_INT8)
    m = build_tiny(seed=23, c=c)
    r = make_runner(m, c)
    tokens = list(np.random.default_rng(5).integers(0, c["vocab_size"], 1027))
    try:
        for n in (1027, 300):  # the second in the first's workspace
            assert_close_logits(prefill(r, c, tokens[:n]), R.model_logits(c, m, tokens[:n]), floor=FLOOR, what="%d tokens" % n)
    finally:
        L.aeth_runner_free(r)


def test_generate_graph_matches_eager(gpu):
    L, outs = A.lib(), []
    m = build_tiny(seed=24, c=INT8)
    for graph in (0, 1, 1):
        r = make_runner(m, INT8)
        first, more = (ctypes.c_int32 * 100)(), (ctypes.c_int32 * 100)()
        A.check(L.aeth_runner_generate(r, 1, 0, 100, first, graph), "generate")
        A.check(L.aeth_runner_generate(r, first[99], 100, 100, more, graph), "generate on")
        kv, fill = cache_of(r, INT8)
        assert fill == 200
        outs.append((list(first) + list(more), kv))
        L.aeth_runner_free(r)
    assert outs[0][0] == outs[1][0] == outs[2][0]
    assert np.array_equal(outs[0][1], outs[1][1]) and np.array_equal(outs[0][1], outs[2][1])


def test_contexts_past_the_f32_limit(gpu):
    """20000 positions with AETH_CFG_FULL_CONTEXT; a full cache is refused."""
    L = A.lib()
    c = dict(TINY, max_seq_len=20000, flags=A.CFG_KV_INT8 | A.CFG_FULL_CONTEXT, num_layers=1)
    m = build_tiny(seed=25, c=c)
    r = make_runner(m, c)
    try:
        kv = _random_cache(c, 19999, 3)
        A.check(L.aeth_runner_kv_from_host(r, kv.ctypes.data, 19999))
        kv, fill = cache_of(r, c)
        s, co = O.precompute_rope(c["max_seq_len"], c["head_dim"], c["rope_base"])
        logits = decode(r, c, 3, 19999)
        ref, fill = O.decode_step(oracle_cfg(c), m["emb"][3], 19999, m["layers"], m["layer_dtype"], m["norms"], m["final"], m["lm"], m["lm_dtype"], s, co, kv, fill)
        assert_close_logits(logits, ref, floor=FLOOR, what="the last position")
        assert L.aeth_runner_decode(r, 3, 20000, None, None) == A.AETH_ESTATE
    finally:
        L.aeth_runner_free(r)


def test_refused_configurations(gpu):
    L, r = A.lib(), ctypes.c_void_p()
    for change, rc in ((dict(flags=4), A.AETH_EINVAL), (dict(flags=A.CFG_KV_INT8 | 8), A.AETH_EINVAL),
                       (dict(flags=A.CFG_KV_INT8 | A.CFG_FULL_CONTEXT, max_seq_len=(1 << 20) + 1), A.AETH_EUNSUPPORTED),
                       (dict(flags=A.CFG_KV_INT8, head_dim=64), A.AETH_EUNSUPPORTED)):
        cfg = A.LlamaConfig(**dict(TINY, **change))
        assert L.aeth_runner_create(ctypes.byref(cfg), None, (ctypes.c_int32 * 14)(*([Q4_K] * 14)), None, None, None, 14, None, 1, ctypes.byref(r)) == rc, change
