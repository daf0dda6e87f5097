"""What a serving loop needs around the 8-bit key/value cache beyond the calls for single
sequences and batches, as timed cases, through the C ABI of include/aether_hip.h: the
attention of a batch whose sequences share a long prefix, attention that also adds up what
weight each cached token received, the eviction of the tokens that received least, and the
norm and rotation of heads whose positions have several axes.

The cache of one layer and sequence is [kv_heads][tiles] tiles of 64 tokens, a
tile being int8 codes of K [64][head_dim], int8 codes of V [head_dim][64] with
token t at byte 16·((t/4)%4) + 4·(t/16) + t%4 of a row, then 64 float scales of K
and 64 of V: a value is code · scale, one scale for each token and head.

Head counts, widths and lengths are those of the repository's benchmark and tests
(32 query / 8 KV heads of 128, caches of 4096 positions, prompts of 2000 and 4000 tokens)
and generic ones around them; queries, keys and values are N(0,1), keys with a few
dimensions some times larger, as rotated keys have.
"""
import math

import torch

own = False  # True: the framework's calls; False: their plain form in torch

TILE = 64


def listed():
    return [
        # two users behind one system prompt, at the start of their answers: latency counts
        dict(name="shared2_1000", kind="shared", seqs=2, prefix=1000, longest=60, max_seq=4096, heads=32, kv_heads=8, head_dim=128, window=0),
        # a serving batch behind a long system prompt, each with a conversation of its own; odd sizes, narrow heads
        dict(name="shared48_4001_h64", kind="shared", seqs=48, prefix=4001, longest=999, max_seq=1024, heads=32, kv_heads=4, head_dim=64, window=0),
        # many questions about one long document
        dict(name="shared160_20000", kind="shared", seqs=160, prefix=20000, longest=500, max_seq=512, heads=32, kv_heads=8, head_dim=128, window=0),
        # a decode step that keeps count of what its tokens attend to, half way into a 4096-position cache
        dict(name="weights_token_2049", kind="weights", n=1, seq=2049, max_seq=4096, heads=32, kv_heads=8, head_dim=128, window=0),
        # the same of many sequences of different lengths
        dict(name="weights_batch32_4096", kind="weights_batch", seqs=32, longest=4096, max_seq=4096, heads=32, kv_heads=8, head_dim=128, window=0),
        # the last rows of a long prompt, whose weights say which of its tokens to keep; narrow heads
        dict(name="weights_last64_of_20000_h64", kind="weights", n=64, seq=20000, max_seq=20480, heads=16, kv_heads=2, head_dim=64, window=0),
        # the weights of a whole prompt of 2000 tokens: the most arithmetic of this kind
        dict(name="weights_prompt_2000", kind="weights", n=2000, seq=2000, max_seq=4096, heads=32, kv_heads=8, head_dim=128, window=0),
        # a conversation past its budget, cut back to it
        dict(name="evict_2500_to_2048", kind="evict", seq=2500, keep=2048, first=4, recent=256, max_seq=4096, dst_seq=4096, kv_heads=8, head_dim=128),
        # a long document's cache cut down to a short cache of its own
        dict(name="evict_30000_to_4000", kind="evict", seq=30000, keep=4000, first=4, recent=64, max_seq=32768, dst_seq=4096, kv_heads=8, head_dim=128),
        # a batch's caches, of odd and uneven lengths, some within their budget; narrow heads
        dict(name="evict_batch24_4001_to_1501_h64", kind="evict_batch", seqs=24, longest=4001, keep=1501, first=1, recent=33, max_seq=4096, dst_seq=2048,
             kv_heads=4, head_dim=64),
        # the q and k heads of one decode step behind an image: the smallest call, launch-bound
        dict(name="axes_token", kind="axes", n=1, heads=32, kv_heads=8, head_dim=128, axes=3, woven=False, norm=True),
        # a prompt of text and an image's patches: a pass over memory
        dict(name="axes_prompt_4000", kind="axes", n=4000, heads=32, kv_heads=8, head_dim=128, axes=3, woven=True, norm=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["shared", "shared", "weights", "weights", "weights_batch", "evict", "evict_batch", "axes"])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 7, 8])
    head_dim = rng.choice([64, 128, 128, 128, 256])
    shape = dict(heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim)
    window = _log(rng, 100, 4000) if rng.random() < 0.25 else 0
    most = 4 * 160 * 20000 * 32 * 128  # operations of the largest listed case
    if kind == "axes":
        return dict(kind=kind, n=_log(rng, 1, 4000), axes=rng.choice([1, 2, 3, 3, 4]), woven=rng.random() < 0.5, norm=rng.random() < 0.7, **shape)
    if kind == "shared":
        seqs, prefix, longest = _log(rng, 1, 160), _log(rng, 1, 20000), _log(rng, 1, 500)
        while 4 * seqs * (prefix + longest) * shape["heads"] * head_dim > most:
            prefix = prefix // 2 + 1
            longest = longest // 2 + 1
        return dict(kind=kind, seqs=seqs, prefix=prefix, longest=longest, max_seq=longest + rng.randrange(0, 300), window=window, **shape)
    if kind == "weights_batch":
        longest = _log(rng, 20, 4096)
        return dict(kind=kind, seqs=_log(rng, 2, 32), longest=longest, max_seq=longest + rng.randrange(0, 300), window=window, **shape)
    if kind == "weights":
        n = 1 if rng.random() < 0.4 else rng.randrange(2, 100) if rng.random() < 0.6 else _log(rng, 100, 2000)
        seq = n if rng.random() < 0.3 else n + _log(rng, 1, 20000)
        while 4 * n * seq * shape["heads"] * head_dim > most // 2:
            seq = seq // 2 + 1
            n = min(n, seq)
        return dict(kind=kind, n=n, seq=seq, max_seq=seq + rng.randrange(0, 500), window=window, **shape)
    shape.pop("heads")
    longest = _log(rng, 2, 30000 if kind == "evict" else 4096)
    keep = max(1, int(longest * rng.uniform(0.05, 1.1)))
    if kind == "evict":
        keep = min(keep, 8000)
    first = min(rng.randrange(0, 8), keep)
    recent = min(_log(rng, 1, 256), keep - first)
    room = dict(max_seq=longest + rng.randrange(0, 500), dst_seq=keep + rng.randrange(0, 300))
    if kind == "evict":
        return dict(kind=kind, seq=longest, keep=keep, first=first, recent=recent, **room, **shape)
    return dict(kind=kind, seqs=_log(rng, 2, 24), longest=longest, keep=keep, first=first, recent=recent, **room, **shape)


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


def _some_cache(seqs, heads, max_seq, hd, g):
    """The caches of `seqs` sequences as they stand before the call: codes that N(0,1) tokens give, laid out in tiles."""
    tiles = _tiles(max_seq)
    cache = torch.empty((seqs, heads, tiles, 2 * TILE * hd + 8 * TILE), dtype=torch.uint8, device="cuda")
    for part in (0, 1):
        x = _spread((seqs, heads, tiles, TILE, hd), g) if part == 0 else torch.randn((seqs, heads, tiles, TILE, hd), generator=g, device="cuda")
        amax = x.abs().amax(-1, keepdim=True)
        codes = torch.round(x * (127.0 / amax)).to(torch.int8)
        if part:
            codes = codes[..., _order(), :].transpose(-1, -2).contiguous()
        at = part * TILE * hd
        cache[..., at:at + TILE * hd] = codes.reshape(seqs, heads, tiles, -1).view(torch.uint8)
        at = 2 * TILE * hd + 4 * TILE * part
        cache[..., at:at + 4 * TILE] = (amax / 127.0).reshape(seqs, heads, tiles, TILE).view(torch.uint8)
    return cache


def _some_weights(shape, g):
    """Attention weight received so far: a few tokens have most of it, a tenth has none at all (equal to one another)."""
    w = torch.exp(2.0 * torch.randn(shape, generator=g, device="cuda") - 3.0)
    return torch.where(torch.rand(shape, generator=g, device="cuda") < 0.1, 0.0, w)


def _axis_of_pair(c):
    """The axis that turns each pair of a head: woven axis by axis, or in sections, the first the shortest."""
    half, axes = c["head_dim"] // 2, c["axes"]
    if c["woven"]:
        return [j % axes for j in range(half)]
    first = half // (axes + 1) if axes > 1 else half
    return [0 if j < first else 1 + (j - first) * (axes - 1) // (half - first) for j in range(half)]


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(2000 + seed)
    hd, kind = c["head_dim"], c["kind"]
    if kind == "axes":
        c["x"] = _spread((c["n"], (c["heads"] + 2 * c["kv_heads"]) * hd), g)  # q | k | v, as the projections leave them
        c["qw"], c["kw"] = (1.0 + 0.2 * torch.randn(hd, generator=g, device="cuda") for _ in range(2))
        # text, where the axes agree, then an image's patches by frame, row and column
        c["max_seq"], text = 4096, c["n"] // 3
        start = int(torch.randint(0, 2000, (1,), generator=g, device="cuda"))
        i = torch.arange(c["n"], device="cuda")
        patch = i - text
        along = [patch // 1024, patch // 32 % 32, patch % 32, patch % 7]
        pos = [start + torch.where(i < text, i, text + a) for a in along[:c["axes"]]]
        c["pos"] = torch.stack(pos).to(torch.int32).contiguous()
        c["pair_axes"] = torch.tensor(_axis_of_pair(c), dtype=torch.int32)  # on the host, as a model's configuration is
        angle = torch.arange(c["max_seq"], dtype=torch.float64)[:, None] * 500000.0 ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64) / hd)
        c["sin"], c["cos"] = angle.sin().float().cuda(), angle.cos().float().cuda()
        return c
    kvh, seqs = c["kv_heads"], c.get("seqs", 1)
    c["cache"] = _some_cache(seqs, kvh, c["max_seq"], hd, g)
    if "seqs" in c:
        c["lens"] = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda")
    if kind == "shared":
        c["shared"] = _some_cache(1, kvh, c["prefix"], hd, g)
    if kind in ("evict", "evict_batch"):
        c["weights"] = _some_weights((seqs, kvh, c["max_seq"]), g)
        c["dst"] = torch.zeros((seqs, kvh, _tiles(c["dst_seq"]), 2 * TILE * hd + 8 * TILE), dtype=torch.uint8, device="cuda")
        c["dst_weights"] = torch.zeros((seqs, kvh, c["dst_seq"]), device="cuda")
        c["dst_lens"] = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        c["kept"] = torch.zeros((seqs, kvh, c["keep"]), dtype=torch.int32, device="cuda")
        return c
    c["q"] = _spread((c.get("seqs") or c["n"], c["heads"] * hd), g)
    if kind != "shared":
        c["before"] = _some_weights((seqs, kvh, c["max_seq"]), g)
        c["weights"] = torch.zeros_like(c["before"])
    return c


# ── the framework's calls ─────────────────────────────────────────────────


def _workspace(s, need):
    if "ws" not in s:  # a program keeps its workspace
        s["ws"] = torch.empty(max(need(), 16), dtype=torch.uint8, device="cuda")
    return s["ws"]


def _own(s):
    import aether_amd as A

    L, stream = A.lib(), torch.cuda.current_stream().cuda_stream
    hd, kvh, kind = s["head_dim"], s["kv_heads"], s["kind"]
    if kind == "axes":
        x = s["x"]
        out = torch.empty((s["n"], (s["heads"] + kvh) * hd), device="cuda")
        qw, kw = (s["qw"].data_ptr(), s["kw"].data_ptr()) if s["norm"] else (None, None)
        A.check(L.aeth_qk_norm_rope_axes(x.data_ptr(), x.shape[1], s["n"], s["heads"], kvh, hd, qw, kw, 1e-5, s["pos"].data_ptr(), s["n"], s["axes"],
                                         s["pair_axes"].data_ptr(), s["sin"].data_ptr(), s["cos"].data_ptr(), s["max_seq"], out.data_ptr(), out.shape[1],
                                         stream), "aeth_qk_norm_rope_axes")
        return out
    cache, stride = s["cache"], s["cache"][0].numel()
    if kind in ("evict", "evict_batch"):
        seqs, keep, batch = cache.shape[0], s["keep"], kind == "evict_batch"
        ws = _workspace(s, lambda: L.aeth_kv8_evict_ws_bytes(seqs, kvh, hd, s["longest"] if batch else s["seq"], keep, 0))
        dst, kept = s["dst"], s["kept"]
        if batch:
            A.check(L.aeth_kv8_evict_batch(cache.data_ptr(), stride, s["weights"].data_ptr(), s["lens"].data_ptr(), seqs, kvh, hd, s["max_seq"], s["longest"],
                                           keep, s["first"], s["recent"], dst.data_ptr(), dst[0].numel(), s["dst_weights"].data_ptr(), s["dst_seq"],
                                           s["dst_lens"].data_ptr(), kept.data_ptr(), ws.data_ptr(), ws.numel(), stream), "aeth_kv8_evict_batch")
            rows = min(keep, s["longest"])
        else:
            A.check(L.aeth_kv8_evict(cache.data_ptr(), s["weights"].data_ptr(), kvh, hd, s["max_seq"], s["seq"], keep, s["first"], s["recent"],
                                     dst.data_ptr(), s["dst_weights"].data_ptr(), s["dst_seq"], kept.data_ptr(), ws.data_ptr(), ws.numel(), stream),
                    "aeth_kv8_evict")
            rows = min(keep, s["seq"])
        # every sequence's heads lie one behind another: one call reads them all
        k, v = (torch.empty((seqs, kvh, rows, hd), device="cuda") for _ in range(2))
        A.check(L.aeth_kv8_read(dst.data_ptr(), k.data_ptr(), v.data_ptr(), hd, rows * hd, rows, seqs * kvh, hd, s["dst_seq"], 0, stream), "aeth_kv8_read")
        return (kept, s["dst_weights"], k, v) + ((s["dst_lens"],) if batch else ())
    q = s["q"]
    out = torch.empty_like(q)
    if kind == "shared":
        ws = _workspace(s, lambda: L.aeth_attn_kv8_shared_ws_bytes(s["seqs"], s["heads"], kvh, hd, s["prefix"], s["longest"]))
        A.check(L.aeth_attn_kv8_shared(q.data_ptr(), q.shape[1], s["shared"].data_ptr(), s["prefix"], s["prefix"], cache.data_ptr(), stride,
                                       s["lens"].data_ptr(), s["seqs"], s["heads"], kvh, hd, s["max_seq"], s["longest"], s["window"], out.data_ptr(),
                                       ws.data_ptr(), ws.numel(), stream), "aeth_attn_kv8_shared")
        return out
    weights, batch = s["weights"], kind == "weights_batch"
    ws = _workspace(s, lambda: L.aeth_attn_kv8_weights_ws_bytes(s["seqs"] if batch else 1, 1 if batch else s["n"], s["heads"], kvh, hd,
                                                                s["longest"] if batch else s["seq"]))
    if batch:
        A.check(L.aeth_attn_kv8_weights_batch(q.data_ptr(), q.shape[1], cache.data_ptr(), stride, s["lens"].data_ptr(), s["seqs"], s["heads"], kvh, hd,
                                              s["max_seq"], s["longest"], s["window"], out.data_ptr(), s["before"].data_ptr(), weights.data_ptr(),
                                              ws.data_ptr(), ws.numel(), stream), "aeth_attn_kv8_weights_batch")
    else:
        A.check(L.aeth_attn_kv8_weights(q.data_ptr(), q.shape[1], cache.data_ptr(), s["n"], s["heads"], kvh, hd, s["max_seq"], s["seq"], s["window"],
                                        out.data_ptr(), s["before"].data_ptr(), weights.data_ptr(), ws.data_ptr(), ws.numel(), stream),
                "aeth_attn_kv8_weights")
    return out, weights


# ── the plain forms ───────────────────────────────────────────────────────


def _plain_axes(s):
    n, h, hd = s["n"], s["heads"] + s["kv_heads"], s["head_dim"]
    y = s["x"][:, :h * hd].reshape(n, h, hd)
    if s["norm"]:
        w = torch.cat([s["qw"].expand(s["heads"], hd), s["kw"].expand(s["kv_heads"], hd)])
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-5) * w
    row = s["pos"][s["pair_axes"].cuda().long()].long().t()  # [n][pairs]
    sin, cos = (torch.gather(t, 0, row)[:, None] for t in (s["sin"], s["cos"]))
    a, b = y[..., :hd // 2], y[..., hd // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).reshape(n, h * hd)


def _plain_read(cache, hd):
    """Every token of caches [...][tiles][bytes] in float: K and V, [...][tokens][hd]."""
    lead = cache.shape[:-2]
    k = cache[..., :TILE * hd].view(torch.int8).unflatten(-1, (TILE, hd)).float()
    v = cache[..., TILE * hd:2 * TILE * hd].view(torch.int8).unflatten(-1, (hd, TILE))
    t = torch.arange(TILE, device=cache.device)
    v = v[..., 16 * ((t // 4) % 4) + 4 * (t // 16) + t % 4].transpose(-1, -2).float()
    scales = cache[..., 2 * TILE * hd:].contiguous().view(torch.float32)
    k, v = k * scales[..., :TILE, None], v * scales[..., TILE:, None]
    return k.reshape(*lead, -1, hd), v.reshape(*lead, -1, hd)


def _plain_evict(s):
    hd, kvh, keep = s["head_dim"], s["kv_heads"], s["keep"]
    longest = s["longest"] if "lens" in s else s["seq"]
    lens = s["lens"].long() if "lens" in s else torch.tensor([s["seq"]], device="cuda")
    rows = min(keep, longest)
    t = torch.arange(longest, device="cuda")
    w = s["weights"][..., :longest]
    end = lens[:, None, None]
    rank = torch.where((t < s["first"]) | (t >= end - s["recent"]), math.inf, w)  # kept whatever their weight
    rank = torch.where(t < end, rank, -math.inf)
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :rows]
    best = torch.where(best < end, best, longest)  # a sequence shorter than that: none
    best = torch.sort(best, dim=-1).values
    there = best < end
    at = torch.where(there, best, 0)
    kept = torch.zeros(w.shape[0], kvh, keep, dtype=torch.int32, device="cuda")
    kept[..., :rows] = at.to(torch.int32)
    weights = torch.zeros(w.shape[0], kvh, s["dst_seq"], device="cuda")
    weights[..., :rows] = torch.where(there, torch.gather(w, -1, at), 0.0)
    k, v = (torch.where(there[..., None], torch.gather(x, -2, at[..., None].expand(-1, -1, -1, hd)), 0.0) for x in _plain_read(s["cache"], hd))
    return (kept, weights, k, v) + ((torch.clamp(s["lens"], max=keep),) if "lens" in s else ())


def _plain_scores(q, k, first, end, scale):
    """q [heads][rows][hd] over k [heads][tokens][hd]: row r of head h sees the tokens first[r] <= t < end[r], the others get -inf."""
    t = torch.arange(k.shape[-2], device=q.device)
    seen = (t >= first[..., None]) & (t < end[..., None])
    return torch.where(seen, torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale, -math.inf)


def _plain_shared(s):
    hd, kvh, seqs, prefix, window = s["head_dim"], s["kv_heads"], s["seqs"], s["prefix"], s["window"]
    group, scale = s["heads"] // kvh, 1.0 / math.sqrt(hd)
    lens = s["lens"].long()
    total = prefix + lens
    lo = torch.clamp(total - window, min=0) if window else torch.zeros_like(lens)
    q = s["q"].reshape(seqs, kvh, group, hd)
    # the prefix: one product for all, the rows of a head being every sequence's
    pk, pv = _plain_read(s["shared"][0], hd)
    together = q.permute(1, 0, 2, 3).reshape(kvh, seqs * group, hd)
    sp = _plain_scores(together, pk, lo.repeat_interleave(group), torch.full_like(lo, prefix).repeat_interleave(group), scale)
    # each sequence's own tokens
    ok, ov = _plain_read(s["cache"][:, :, :_tiles(s["longest"])], hd)
    each = [x[:, None, None].expand(-1, kvh, group) for x in (torch.clamp(lo - prefix, min=0), lens)]
    so = _plain_scores(q, ok, *each, scale)
    m = torch.maximum(sp.amax(-1).reshape(kvh, seqs, group).permute(1, 0, 2), so.amax(-1))
    mp = m.permute(1, 0, 2).reshape(kvh, seqs * group)
    sp, so = torch.exp(sp - mp[..., None]), torch.exp(so - m[..., None])
    out = torch.matmul(sp, pv).reshape(kvh, seqs, group, hd).permute(1, 0, 2, 3) + torch.matmul(so, ov)
    total = sp.sum(-1).reshape(kvh, seqs, group).permute(1, 0, 2) + so.sum(-1)
    return (out / total[..., None]).reshape(seqs, -1)


def _plain_weights(s):
    hd, kvh, batch = s["head_dim"], s["kv_heads"], s["kind"] == "weights_batch"
    group, scale = s["heads"] // kvh, 1.0 / math.sqrt(hd)
    after = torch.zeros_like(s["before"])
    if batch:
        tokens, n = s["longest"], 1
        end = s["lens"].long()[:, None, None].expand(-1, kvh, group)
        q = s["q"].reshape(s["seqs"], kvh, group, hd)
    else:
        tokens, n = s["seq"], s["n"]
        end = torch.arange(tokens - n + 1, tokens + 1, device="cuda").repeat_interleave(group)
        q = s["q"].reshape(n, kvh, group, hd).permute(1, 0, 2, 3).reshape(1, kvh, n * group, hd)
    k, v = (x[:, :, :tokens] for x in _plain_read(s["cache"][:, :, :_tiles(tokens)], hd))
    first = end - s["window"] if s["window"] else torch.zeros_like(end)
    p = _plain_scores(q, k, first, end, scale)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    # more columns than a few: their sum in 64 bits
    mass = p.sum(-2) if n * group < 64 else torch.stack([h.sum(-2, dtype=torch.float64) for h in p.reshape(kvh, n * group, tokens)])[None]
    out = torch.matmul(p, v)
    out = out.reshape(s["seqs"], -1) if batch else out.reshape(kvh, n, group, hd).permute(1, 0, 2, 3).reshape(n, -1)
    after[..., :tokens] = (s["before"][..., :tokens] + mass).float()
    if batch:
        after[..., :tokens] = torch.where(torch.arange(tokens, device="cuda") < end[..., :1], after[..., :tokens], 0.0)
    return out, after


def run(state):
    if own:
        return _own(state)
    kind = state["kind"]
    if kind == "axes":
        return _plain_axes(state)
    if kind == "shared":
        return _plain_shared(state)
    if kind in ("evict", "evict_batch"):
        return _plain_evict(state)
    return _plain_weights(state)


# ── what a pass cannot do without ─────────────────────────────────────────


def work(case):
    c, hd, kvh, kind = case, case["head_dim"], case["kv_heads"], case["kind"]
    token = 2 * hd + 8  # bytes of a cached token and head
    if kind == "axes":
        el = c["n"] * (c["heads"] + kvh) * hd
        return {"bytes": 8 * el + c["n"] * (4 * hd + 4 * c["axes"]) + (8 * hd if c["norm"] else 0), "flops": (8 if c["norm"] else 3) * el}
    if kind in ("evict", "evict_batch"):
        lens = _lengths(c) if kind == "evict_batch" else [c["seq"]]
        kept = sum(min(l, c["keep"]) for l in lens)
        # the weights of all, the kept tokens from one cache to the other with their weights and numbers, and their values
        return {"bytes": kvh * (4 * sum(lens) + kept * (2 * token + 8 + 8 * hd)), "flops": kvh * (sum(lens) + 2 * kept * hd)}
    window = c["window"] or 1 << 40
    if kind == "shared":
        totals = [c["prefix"] + l for l in _lengths(c)]
        pairs = sum(min(t, window) for t in totals)
        longest_view = max(min(c["prefix"], max(0, window - l)) for l in _lengths(c))  # of the prefix
        keys = longest_view + sum(min(l, window) for l in _lengths(c))
        return {"bytes": keys * kvh * token + 8 * c["seqs"] * c["heads"] * hd, "flops": 4 * pairs * c["heads"] * hd}
    if kind == "weights_batch":
        rows, lens = c["seqs"], _lengths(c)
        pairs = keys = sum(min(l, window) for l in lens)
    else:
        rows, lens = c["n"], [c["seq"]]
        pairs = sum(min(e, window) for e in range(c["seq"] - rows + 1, c["seq"] + 1))
        keys = min(c["seq"], window + rows - 1)
    return {"bytes": keys * kvh * token + 8 * rows * c["heads"] * hd + 8 * kvh * sum(lens), "flops": 4 * pairs * c["heads"] * hd + pairs * c["heads"]}


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


def _exact_axes(s):
    hd, heads = s["head_dim"], []
    pos, axis = s["pos"].long(), s["pair_axes"].tolist()
    turn = torch.stack([torch.complex(s["cos"][pos[a], j].double(), s["sin"][pos[a], j].double()) for j, a in enumerate(axis)], 1)
    for h in range(s["heads"] + s["kv_heads"]):
        x = s["x"][:, h * hd:(h + 1) * hd].double()
        if s["norm"]:
            x = x * (x.square().sum(1, keepdim=True) / hd + 1e-5).rsqrt() * (s["qw"] if h < s["heads"] else s["kw"]).double()
        z = torch.complex(x[:, :hd // 2], x[:, hd // 2:]) * turn
        heads += [z.real, z.imag]
    return torch.cat(heads, 1)


def _exact_evict(s):
    hd, kvh, keep, seqs = s["head_dim"], s["kv_heads"], s["keep"], s["cache"].shape[0]
    lens = _lengths(s) if "lens" in s else [s["seq"]]
    rows = min(keep, max(lens))
    kept = torch.zeros(seqs, kvh, keep, dtype=torch.int32, device="cuda")
    weights = torch.zeros(seqs, kvh, s["dst_seq"], dtype=torch.float64, device="cuda")
    k, v = (torch.zeros(seqs, kvh, rows, hd, dtype=torch.float64, device="cuda") for _ in range(2))
    host = s["weights"].cpu().numpy()
    for b, length in enumerate(lens):
        for h in range(kvh):
            w = host[b, h].tolist()
            must = set(range(min(s["first"], length))) | set(range(max(0, length - s["recent"]), length))
            rest = sorted((t for t in range(length) if t not in must), key=lambda t: (-w[t], t))
            at = sorted(list(must) + rest[:max(0, keep - len(must))]) if length > keep else list(range(length))
            i = torch.tensor(at, device="cuda")
            kept[b, h, :len(at)] = i.to(torch.int32)
            weights[b, h, :len(at)] = s["weights"][b, h].double()[i]
            for x, y in zip((k, v), _exact_cache(s["cache"][b, h], hd, length)):
                x[b, h, :len(at)] = y[i]
    out = (kept, weights, k, v)
    return out + (torch.tensor([min(l, keep) for l in lens], dtype=torch.int32, device="cuda"),) if "lens" in s else out


def exact(case, seed):
    s = prepare(case, seed)
    hd, kind = s["head_dim"], s["kind"]
    if kind == "axes":
        return _exact_axes(s)
    if kind in ("evict", "evict_batch"):
        return _exact_evict(s)
    group = s["heads"] // s["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    after = None if kind == "shared" else torch.zeros_like(s["before"], dtype=torch.float64)
    batch = "seqs" in s
    shared = [tuple(_exact_cache(s["shared"][0, h], hd, s["prefix"])) for h in range(s["kv_heads"])] if kind == "shared" else None
    for b, tokens in enumerate(_lengths(s) if batch else [s["seq"]]):
        for h in range(s["kv_heads"]):
            k, v = _exact_cache(s["cache"][b, h], hd, tokens)
            if shared:
                k, v = (torch.cat(x) for x in zip(shared[h], (k, v)))
            keys = len(k)
            if after is not None:
                after[b, h, :tokens] = s["before"][b, h, :tokens].double()
            for g in range(h * group, (h + 1) * group):
                at = (slice(b, b + 1) if batch else slice(None), slice(g * hd, (g + 1) * hd))
                q = s["q"][at].double()
                z = q @ k.T / hd ** 0.5
                ago = torch.arange(keys - len(q), keys, device="cuda")[:, None] - torch.arange(keys, device="cuda")
                z[(ago < 0) | (ago >= (s["window"] or keys))] = -math.inf
                p = torch.softmax(z, 1)
                out[at] = p @ v
                if after is not None:
                    after[b, h, :tokens] += p.sum(0)
    return out if kind == "shared" else (out, after)
