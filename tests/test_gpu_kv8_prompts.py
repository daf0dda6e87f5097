"""Prompts of the device runner that go over its 8-bit cache in several passes
(AETH_CFG_KV_INT8), against the model in float64 on the device."""
import ctypes
import math

import numpy as np
import pytest

import aether_amd as A
from oracle import oracle as O
from tests import _kv8 as R
from tests._model64 import _deq
from tests._models import TINY, build_tiny
from tests._util import Q2_K, Q4_K, Q8_0, assert_close_logits
from tests.test_gpu_decode import make_runner
from tests.test_gpu_kv8_runner import FLOOR, cache_of, prefill

pytestmark = pytest.mark.gpu

LONG = A.CFG_KV_INT8 | A.CFG_FULL_CONTEXT


def exact_run(torch, c, m, tokens):
    """The model in float64 on the device, K and V in 8 bits: each layer's quantised K and V, and the last position's logits
    (causal over `tokens`, R.model_logits for more tokens than the host has patience for; the last layer's rows but the last one
    are left out where nothing depends on them)."""
    d, nh, nkv, hd, dff, ms = (c[k] for k in ("d_model", "num_heads", "num_kv_heads", "head_dim", "d_ff", "max_seq_len"))
    shapes = [(nh * hd, d), (nkv * hd, d), (nkv * hd, d), (d, nh * hd), (dff, d), (dff, d), (d, dff)]
    n = len(tokens)
    sin, cos = (torch.from_numpy(t.reshape(ms, hd // 2)[:n].astype(np.float64)).cuda()[:, None]
                for t in O.precompute_rope(ms, hd, c["rope_base"]))

    def dev(a):
        return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float64)).cuda()

    def norm(v, w):
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + c["rms_norm_eps"]) * dev(w)

    def rotated(v, at):
        a, b = v[..., :hd // 2], v[..., hd // 2:]
        return torch.cat([a * cos[at] - b * sin[at], a * sin[at] + b * cos[at]], -1)

    def held(v):
        k, s = R.codes(v.float())
        return k.double() * s.double()[..., None]

    x, caches = dev(m["emb"])[torch.tensor(tokens, device="cuda")], []
    for layer, (weights, (w_attn, w_ffn)) in enumerate(zip(m["layers"], m["norms"])):
        wq, wk, wv, wo, wg, wu, wd = (dev(_deq(t, w, *s)).t().contiguous() for t, w, s in zip(m["layer_dtype"], weights, shapes))
        at = slice(n - 1, n) if layer == c["num_layers"] - 1 else slice(0, n)
        h = norm(x, w_attn)
        k, v = held(rotated((h @ wk).reshape(n, nkv, hd), slice(0, n))), held((h @ wv).reshape(n, nkv, hd))
        caches.append((k, v))
        q = rotated((h[at] @ wq).reshape(-1, nh, hd), at)
        rows, heads = torch.arange(n, device="cuda")[at, None], []
        for j in range(nh):
            s = q[:, j] @ k[:, j * nkv // nh].t().contiguous() / math.sqrt(hd)
            p = torch.softmax(torch.where(torch.arange(n, device="cuda") <= rows, s, -math.inf), -1)
            heads.append(p @ v[:, j * nkv // nh])
        x = x[at] + torch.cat(heads, 1) @ wo
        h = norm(x, w_ffn)
        x = x + (torch.nn.functional.silu(h @ wg) * (h @ wu)) @ wd
    return caches, _deq(m["lm_dtype"], m["lm"], c["vocab_size"], d) @ norm(x[-1], m["final"]).cpu().numpy()


def check_cache(r, c, caches, n):
    """An entry differs from the exact model's by at most one code in layer 0, a step of 1/127 of its row's largest; layer 1's
    inputs then differ by about 2e-3 of their size, and its rows by twice that at most."""
    kv, fill = cache_of(r, c)
    assert fill == n and not kv[:, :, :, n:].any()
    for layer, (kc, slack) in enumerate(zip(caches, (1.01 / 127, 1.01 / 127 + 8e-3))):
        for part, want in enumerate(kc):
            want = want.transpose(0, 1).cpu().numpy()
            big = np.abs(want).max(-1, keepdims=True)
            assert (np.abs(kv[layer, part, :, :n] - want) <= slack * big).all(), (layer, part)


@pytest.mark.parametrize("n,dff,layers,dtype", [(8252, 66048, 2, Q4_K), (8192, 66048, 1, Q4_K), (8252, 66048, 1, Q8_0), (70000, 512, 1, Q4_K)])
def test_prompts_of_two_passes(gpu, n, dff, layers, dtype):
    """More rows than a Q4_K GEMM takes of a down projection of k = 66048 (rows times k of 2^29), or than 65535; then a
    shorter prompt in the same buffers, and a refusal of a step, since the cache is full."""
    c = dict(TINY, max_seq_len=n, num_heads=2, num_kv_heads=1, num_layers=layers, d_ff=dff, flags=LONG)
    m = build_tiny(seed=32, layer_dtype=dtype, c=c)
    r = make_runner(m, c)
    tokens = np.random.default_rng(10).integers(0, c["vocab_size"], n).tolist()
    try:
        got = prefill(r, c, tokens)
        caches, want = exact_run(gpu, c, m, tokens)
        assert_close_logits(got, want, floor=FLOOR, what="%d tokens" % n)
        check_cache(r, c, caches, n)
        assert A.lib().aeth_runner_decode(r, 3, n, None, None) == A.AETH_ESTATE
        assert_close_logits(prefill(r, c, tokens[:100]), exact_run(gpu, c, m, tokens[:100])[1], floor=FLOOR, what="100 tokens")
    finally:
        A.lib().aeth_runner_free(r)


def test_a_prompt_refused_midway_leaves_no_sequence(gpu):
    """Over the f32 cache, whose attention takes a prompt whole, the products of the first test still refuse it, in layer 0 and behind
    that layer's writes: no slot counts then, and the next sequence is as on a new runner."""
    L = A.lib()
    c = dict(TINY, max_seq_len=8192, num_heads=2, num_kv_heads=1, num_layers=1, d_ff=66048, flags=A.CFG_FULL_CONTEXT)
    r = make_runner(build_tiny(seed=32, c=c), c)
    tokens = np.random.default_rng(10).integers(0, c["vocab_size"], 8192).astype(np.int32)
    try:
        first = prefill(r, c, tokens[:100])
        assert L.aeth_runner_seq_len(r) == 100
        assert L.aeth_runner_prefill(r, tokens.ctypes.data, 8192, None, None) == A.AETH_EINVAL
        assert L.aeth_runner_seq_len(r) == 0 and cache_of(r, c)[1] == 0
        # arguments refused before anything is written leave the sequence as it is
        assert np.array_equal(prefill(r, c, tokens[:100]), first)
        assert L.aeth_runner_prefill(r, tokens.ctypes.data, 8193, None, None) == A.AETH_EINVAL
        tokens[50] = c["vocab_size"]
        assert L.aeth_runner_prefill(r, tokens.ctypes.data, 60, None, None) == A.AETH_EINVAL
        assert L.aeth_runner_seq_len(r) == 100
    finally:
        L.aeth_runner_free(r)


def test_a_fill_without_memory_leaves_the_cache(gpu):
    """aeth_runner_fill_kv quantises a layer at a time out of an f32 copy; one of 2400 heads over 131072 positions is 322 GB, more than the
    GPU has. The sequence in the cache goes on as if the call had not been."""
    L = A.lib()
    cfg = A.LlamaConfig(vocab_size=512, d_model=256, num_layers=1, num_heads=2400, num_kv_heads=2400, head_dim=128, d_ff=512, max_seq_len=1 << 17,
                        rope_base=10000.0, rms_norm_eps=1e-5, sliding_window=0, flags=LONG)
    got = []
    for fill in (False, True):
        r = ctypes.c_void_p()
        A.check(L.aeth_runner_create(ctypes.byref(cfg), None, (ctypes.c_int32 * 7)(*([Q4_K] * 3 + [Q2_K] + [Q4_K] * 3)), None, None, None, Q4_K, None, 5, ctypes.byref(r)), "create")
        try:
            logits = np.empty(512, np.float32)
            A.check(L.aeth_runner_decode(r, 3, 0, None, None), "decode")
            if fill:
                assert L.aeth_runner_fill_kv(r, 5, 1000) == A.AETH_ENOMEM
            assert L.aeth_runner_seq_len(r) == 1
            A.check(L.aeth_runner_decode(r, 4, 1, logits.ctypes.data, None), "decode")
            got.append(logits)
        finally:
            L.aeth_runner_free(r)
    assert np.array_equal(got[0], got[1])
