"""The attention side of a decode or prefill step over a key/value cache held in 8
bits, as timed cases: the norm and rotation of queries and keys, the cache's
writing and reading back, and the attention over it, through the C ABI of
include/aether_hip.h.

The cache of one layer and sequence is [kv_heads][tiles] tiles of 64 tokens, a
tile being int8 codes of K [64][head_dim], int8 codes of V [head_dim][64] with
token t at byte 16·((t/4)%4) + 4·(t/16) + t%4 of a row, then 64 float scales of K
and 64 of V: a value is code · scale, one scale for each token and head.

Head counts, widths and lengths are those of the repository's benchmark and tests
(32 query / 8 KV heads of 128, caches of 4096 positions, prompts of 512, 2000 and
4000 tokens) and generic ones around them; queries, keys and values are N(0,1),
keys with a few dimensions some times larger, as rotated keys have.
"""
import math

import torch

own = False  # True: the framework's calls; False: their plain form in torch

TILE = 64


def listed():
    return [
        # the q and k heads of one decode step: the smallest call, launch-bound
        dict(name="qk_token", kind="qk", n=1, heads=32, kv_heads=8, head_dim=128, norm=True),
        # the same of a long prompt: a pass over memory
        dict(name="qk_prompt_4000", kind="qk", n=4000, heads=32, kv_heads=8, head_dim=128, norm=True),
        # a decode step's token into its cache, read back
        dict(name="store_token", kind="store", n=1, slot=2048, max_seq=4096, kv_heads=8, head_dim=128),
        # a prompt of odd length behind an odd number of tokens, narrow heads
        dict(name="store_1999_h64", kind="store", n=1999, slot=37, max_seq=4096, kv_heads=8, head_dim=64),
        # a long document's cache
        dict(name="store_30000", kind="store", n=30000, slot=0, max_seq=32768, kv_heads=8, head_dim=128),
        # one decode step of an 8B-shape layer, half way into its 4096-position cache: latency counts
        dict(name="token_2049", kind="attn", n=1, seq=2049, max_seq=4096, heads=32, kv_heads=8, head_dim=128, window=0),
        # one decode step deep into a long context: the cache is read at the memory's rate
        dict(name="token_131000", kind="attn", n=1, seq=131000, max_seq=131072, heads=32, kv_heads=8, head_dim=128, window=0),
        # one decode step of many sequences of different lengths
        dict(name="batch48_4096", kind="batch", seqs=48, longest=4096, max_seq=4096, heads=32, kv_heads=8, head_dim=128, window=0),
        # a drafted continuation checked in one call, sliding window, narrow heads, few KV heads
        dict(name="draft7_w1024_h64", kind="attn", n=7, seq=5003, max_seq=8192, heads=16, kv_heads=2, head_dim=64, window=1024),
        # the benchmark's 512-token prompt
        dict(name="prompt_512", kind="attn", n=512, seq=512, max_seq=4096, heads=32, kv_heads=8, head_dim=128, window=0),
        # a chunk of a long prompt behind what is already cached
        dict(name="chunk_250_of_20000", kind="attn", n=250, seq=20000, max_seq=32768, heads=32, kv_heads=8, head_dim=128, window=0),
        # a whole 4000-token prompt: the largest
        dict(name="prompt_4000", kind="attn", n=4000, seq=4000, max_seq=4096, heads=32, kv_heads=8, head_dim=128, window=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["qk", "store", "attn", "attn", "batch", "prompt"])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 7, 8])
    head_dim = rng.choice([64, 128, 128, 128])
    if kind == "qk":
        return dict(kind="qk", n=_log(rng, 1, 4000), heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim, norm=rng.random() < 0.7)
    if kind == "store":
        n, slot = _log(rng, 1, 30000), _log(rng, 1, 2000) - 1
        return dict(kind="store", n=n, slot=slot, max_seq=n + slot + rng.randrange(0, 500), kv_heads=kv_heads, head_dim=head_dim)
    window = _log(rng, 100, 4000) if rng.random() < 0.25 else 0
    if kind == "batch":
        longest = _log(rng, 50, 4096)
        return dict(kind="batch", seqs=_log(rng, 2, 64), longest=longest, max_seq=longest + rng.randrange(0, 300), heads=kv_heads * group, kv_heads=kv_heads,
                    head_dim=head_dim, window=window)
    if kind == "attn":  # a token, or a few
        n = 1 if rng.random() < 0.6 else rng.randrange(2, 9)
        seq = _log(rng, n, 131000)
    else:
        n = _log(rng, 17, 2500)
        seq = n + (_log(rng, 1, 9000) if rng.random() < 0.5 else 0)
    return dict(kind="attn", n=n, seq=seq, max_seq=seq + rng.randrange(0, 500), heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim, window=window)


def _lengths(c):
    """The lengths of a batch's sequences: spread over 1 .. longest, one of them the longest."""
    return [c["longest"] if i == 0 else 1 + int((c["longest"] - 1) * ((0.6180339887 * i) % 1.0)) for i in range(c["seqs"])]


def _tiles(max_seq):
    return -(-max_seq // TILE)


def _spread(shape, g):
    """N(0,1), every 29th dimension 4 times as large."""
    x = torch.randn(shape, generator=g, device="cuda")
    x[..., ::29] *= 4.0
    return x


def _order():
    """The token at each byte of a row of V codes."""
    t = torch.arange(TILE, device="cuda")
    at = 16 * ((t // 4) % 4) + 4 * (t // 16) + t % 4
    order = torch.empty_like(t)
    order[at] = t
    return order


def _some_cache(c, seqs, g):
    """The cache of `seqs` sequences as it stands before the call: codes that N(0,1) tokens give, laid out in tiles."""
    h, hd, tiles = c["kv_heads"], c["head_dim"], _tiles(c["max_seq"])
    cache = torch.empty((seqs, h, tiles, 2 * TILE * hd + 8 * TILE), dtype=torch.uint8, device="cuda")
    for part in (0, 1):
        x = _spread((seqs, h, tiles, TILE, hd), g) if part == 0 else torch.randn((seqs, h, tiles, TILE, hd), generator=g, device="cuda")
        amax = x.abs().amax(-1, keepdim=True)
        codes = torch.round(x * (127.0 / amax)).to(torch.int8)
        if part:
            codes = codes[..., _order(), :].transpose(-1, -2).contiguous()
        at = part * TILE * hd
        cache[..., at:at + TILE * hd] = codes.reshape(seqs, h, tiles, -1).view(torch.uint8)
        at = 2 * TILE * hd + 4 * TILE * part
        cache[..., at:at + 4 * TILE] = (amax / 127.0).reshape(seqs, h, tiles, TILE).view(torch.uint8)
    return cache


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(1000 + seed)
    hd = c["head_dim"]
    if c["kind"] == "qk":
        rows = c["heads"] + c["kv_heads"]
        c["x"] = _spread((c["n"], (rows + c["kv_heads"]) * hd), g)  # q | k | v, as the projections leave them
        c["qw"], c["kw"] = (1.0 + 0.2 * torch.randn(hd, generator=g, device="cuda") for _ in range(2))
        c["pos"] = int(torch.randint(0, 4000, (1,), generator=g, device="cuda"))
        c["max_seq"] = c["pos"] + c["n"]
        angle = torch.arange(c["max_seq"], dtype=torch.float64)[:, None] * 500000.0 ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64) / hd)
        c["sin"], c["cos"] = angle.sin().float().cuda(), angle.cos().float().cuda()
    elif c["kind"] == "store":
        c["k"] = _spread((c["n"], c["kv_heads"] * hd), g)
        c["v"] = torch.randn((c["n"], c["kv_heads"] * hd), generator=g, device="cuda")
        c["cache"] = torch.zeros((c["kv_heads"], _tiles(c["max_seq"]), 2 * TILE * hd + 8 * TILE), dtype=torch.uint8, device="cuda")
    else:
        seqs = c["seqs"] if c["kind"] == "batch" else 1
        c["cache"] = _some_cache(c, seqs, g)
        c["q"] = _spread((seqs if c["kind"] == "batch" else c["n"], c["heads"] * hd), g)
        if c["kind"] == "batch":
            c["lengths"] = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda")
    return c


# ── the framework's calls ─────────────────────────────────────────────────


def _own(s):
    import aether_amd as A

    L, stream = A.lib(), torch.cuda.current_stream().cuda_stream
    hd, kvh = s["head_dim"], s["kv_heads"]
    if s["kind"] == "qk":
        x = s["x"]
        out = torch.empty((s["n"], (s["heads"] + kvh) * hd), device="cuda")
        qw, kw = (s["qw"].data_ptr(), s["kw"].data_ptr()) if s["norm"] else (None, None)
        A.check(L.aeth_qk_norm_rope(x.data_ptr(), x.shape[1], s["n"], s["heads"], kvh, hd, qw, kw, 1e-5, s["pos"], None, s["sin"].data_ptr(),
                                    s["cos"].data_ptr(), s["max_seq"], out.data_ptr(), out.shape[1], stream), "aeth_qk_norm_rope")
        return out
    if s["kind"] == "store":
        k, v = torch.empty_like(s["k"]), torch.empty_like(s["v"])
        A.check(L.aeth_kv8_append(s["cache"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), kvh * hd, hd, s["n"], kvh, hd, s["max_seq"], s["slot"], stream),
                "aeth_kv8_append")
        A.check(L.aeth_kv8_read(s["cache"].data_ptr(), k.data_ptr(), v.data_ptr(), kvh * hd, hd, s["n"], kvh, hd, s["max_seq"], s["slot"], stream), "aeth_kv8_read")
        return k, v
    q, batch = s["q"], s["kind"] == "batch"
    if "ws" not in s:  # a program keeps its workspace
        need = L.aeth_attn_kv8_ws_bytes(s["seqs"] if batch else 1, 1 if batch else s["n"], s["heads"], kvh, hd, s["longest"] if batch else s["seq"])
        s["ws"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    out, ws = torch.empty_like(q), s["ws"]
    if batch:
        A.check(L.aeth_attn_kv8_batch(q.data_ptr(), q.shape[1], s["cache"].data_ptr(), s["cache"][0].numel(), s["lengths"].data_ptr(), s["seqs"], s["heads"], kvh,
                                      hd, s["max_seq"], s["longest"], s["window"], out.data_ptr(), ws.data_ptr(), ws.numel(), stream), "aeth_attn_kv8_batch")
    else:
        A.check(L.aeth_attn_kv8(q.data_ptr(), q.shape[1], s["cache"].data_ptr(), s["n"], s["heads"], kvh, hd, s["max_seq"], s["seq"], s["window"], out.data_ptr(),
                                ws.data_ptr(), ws.numel(), stream), "aeth_attn_kv8")
    return out


# ── the plain forms ───────────────────────────────────────────────────────


def _plain_qk(s):
    n, h, hd = s["n"], s["heads"] + s["kv_heads"], s["head_dim"]
    y = s["x"][:, :h * hd].reshape(n, h, hd)
    if s["norm"]:
        w = torch.cat([s["qw"].expand(s["heads"], hd), s["kw"].expand(s["kv_heads"], hd)])
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-5) * w
    sin, cos = (t[s["pos"]:s["pos"] + n, None] for t in (s["sin"], s["cos"]))
    a, b = y[..., :hd // 2], y[..., hd // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).reshape(n, h * hd)


def _plain_store(x, heads, hd):
    """x in 8 bits: the codes are the nearest to 127·x/amax, found in 64 bits (a code next to a border), the scale amax/127."""
    x = x.reshape(-1, heads, hd)
    amax = x.abs().amax(-1, keepdim=True).double()
    codes = torch.round(x.double() * 127.0 / amax.clamp_min(1e-300)).to(torch.int8)
    scales = (amax / 127.0).float()
    return (codes.float() * scales).reshape(-1, heads * hd)


def _plain_read(cache, hd):
    """Every token of a cache [...][tiles][bytes] in float: K and V, [...][tokens][hd]."""
    lead = cache.shape[:-2]
    k = cache[..., :TILE * hd].view(torch.int8).unflatten(-1, (TILE, hd)).float()
    v = cache[..., TILE * hd:2 * TILE * hd].view(torch.int8).unflatten(-1, (hd, TILE))
    t = torch.arange(TILE, device=cache.device)
    v = v[..., 16 * ((t // 4) % 4) + 4 * (t // 16) + t % 4].transpose(-1, -2).float()
    scales = cache[..., 2 * TILE * hd:].contiguous().view(torch.float32)
    k, v = k * scales[..., :TILE, None], v * scales[..., TILE:, None]
    return k.reshape(*lead, -1, hd), v.reshape(*lead, -1, hd)


def _plain_attention(q, k, v, first, end, scale):
    """q [heads][rows][hd] over k, v [heads][tokens][hd]: row r of head h sees the tokens first[r] <= t < end[r]."""
    t = torch.arange(k.shape[-2], device=q.device)
    seen = (t >= first[..., None]) & (t < end[..., None])
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    s = torch.where(seen, s, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return torch.matmul(p, v) / p.sum(-1, keepdim=True)


def run(state):
    if own:
        return _own(state)
    s = state
    if s["kind"] == "qk":
        return _plain_qk(s)
    hd, kvh = s["head_dim"], s["kv_heads"]
    if s["kind"] == "store":
        return _plain_store(s["k"], kvh, hd), _plain_store(s["v"], kvh, hd)
    group, scale = s["heads"] // kvh, 1.0 / math.sqrt(hd)
    if s["kind"] == "batch":
        k, v = _plain_read(s["cache"][:, :, :_tiles(s["longest"])], hd)
        q = s["q"].reshape(s["seqs"], kvh, group, hd)
        end = s["lengths"][:, None, None].expand(-1, kvh, group)
        first = end - s["window"] if s["window"] else torch.zeros_like(end)
        return _plain_attention(q, k, v, first, end, scale).reshape(s["seqs"], -1)
    n = s["n"]
    lo = max(0, s["seq"] - n + 1 - s["window"]) // TILE if s["window"] else 0  # the tiles that some query sees
    k, v = _plain_read(s["cache"][0, :, lo:_tiles(s["seq"])], hd)
    q = s["q"].reshape(n, kvh, group, hd).permute(1, 0, 2, 3).reshape(kvh, n * group, hd)
    end = torch.arange(s["seq"] - n + 1, s["seq"] + 1, device="cuda").repeat_interleave(group) - lo * TILE
    first = end - s["window"] if s["window"] else torch.zeros_like(end)
    out = _plain_attention(q, k, v, first, end, scale)
    return out.reshape(kvh, n, group, hd).permute(1, 0, 2, 3).reshape(n, -1)


# ── what a pass cannot do without ─────────────────────────────────────────


def _seen(n, seq, window):
    """(query, key) pairs of n queries at the end of seq, and the keys that some query sees."""
    ends = range(seq - n + 1, seq + 1)
    return sum(min(e, window) if window else e for e in ends), seq - max(0, seq - n + 1 - window) if window else seq


def work(case):
    c, hd = case, case["head_dim"]
    if c["kind"] == "qk":
        el = c["n"] * (c["heads"] + c["kv_heads"]) * hd
        table = c["n"] * hd * 4
        return {"bytes": 8 * el + table + (8 * hd if c["norm"] else 0), "flops": (8 if c["norm"] else 3) * el}
    if c["kind"] == "store":
        el = 2 * c["n"] * c["kv_heads"] * hd
        return {"bytes": (4 + 1 + 1 + 4) * el + 8 * (el // hd), "flops": 6 * el}
    if c["kind"] == "batch":
        pairs = keys = sum(min(l, c["window"]) if c["window"] else l for l in _lengths(c))
        rows = c["seqs"]
    else:
        pairs, keys = _seen(c["n"], c["seq"], c["window"])
        rows = c["n"]
    return {"bytes": keys * c["kv_heads"] * (2 * hd + 8) + 8 * rows * c["heads"] * hd, "flops": 4 * pairs * c["heads"] * hd}


# ── the definition in 64 bits ─────────────────────────────────────────────


def _exact_cache(cache, hd, tokens):
    """K and V of one head's first `tokens` tokens in 64 bits; cache [tiles][bytes]."""
    ks, vs = [], []
    raw = cache[:_tiles(tokens)]
    tiles = raw.shape[0]
    kc = raw[:, :64 * hd].reshape(tiles, 64, hd).view(torch.int8).double()
    vc = raw[:, 64 * hd:128 * hd].reshape(tiles, hd, 64).view(torch.int8).double()
    sc = raw[:, 128 * hd:].contiguous().view(torch.float32).double()
    for t in range(64):
        byte = t % 4 + 4 * (t // 16) + 16 * (t % 16 // 4)
        ks.append(kc[:, t] * sc[:, t, None])
        vs.append(vc[:, :, byte] * sc[:, 64 + t, None])
    return (torch.stack(x, 1).reshape(tiles * 64, hd)[:tokens] for x in (ks, vs))


def exact(case, seed):
    s = prepare(case, seed)
    hd = s["head_dim"]
    if s["kind"] == "qk":
        heads = []
        for h in range(s["heads"] + s["kv_heads"]):
            x = s["x"][:, h * hd:(h + 1) * hd].double()
            if s["norm"]:
                x = x * (x.square().sum(1, keepdim=True) / hd + 1e-5).rsqrt() * (s["qw"] if h < s["heads"] else s["kw"]).double()
            z = torch.complex(x[:, :hd // 2], x[:, hd // 2:])
            at = slice(s["pos"], s["pos"] + s["n"])
            z = z * torch.complex(s["cos"][at].double(), s["sin"][at].double())
            heads += [z.real, z.imag]
        return torch.cat(heads, 1)
    if s["kind"] == "store":
        out = []
        for x in (s["k"], s["v"]):
            rows = x.double().reshape(-1, hd)
            step = rows.abs().max(1, keepdim=True).values / 127
            out.append((torch.round(rows / step) * step).reshape(x.shape))
        return tuple(out)
    group = s["heads"] // s["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    batch = s["kind"] == "batch"
    for b, tokens in enumerate(_lengths(s) if batch else [s["seq"]]):
        for h in range(s["kv_heads"]):
            k, v = _exact_cache(s["cache"][b, h], hd, tokens)
            for g in range(h * group, (h + 1) * group):
                at = (slice(b, b + 1) if batch else slice(None), slice(g * hd, (g + 1) * hd))
                q = s["q"][at].double()
                z = q @ k.T / hd ** 0.5
                ago = torch.arange(tokens - len(q), tokens, device="cuda")[:, None] - torch.arange(tokens, device="cuda")
                z[(ago < 0) | (ago >= (s["window"] or tokens))] = -math.inf
                out[at] = torch.softmax(z, 1) @ v
    return out
