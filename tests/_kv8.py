"""The 8-bit key/value cache and its attention from their definitions, in 64 bits
(torch on whatever device the tensors are), and the error bounds that the
kernels' roundings allow."""
import math

import torch

TILE = 64
# an f32 value rounded to an integer of 24 bits in balanced digits: the largest component is over 0x7F7F00 / 2
# units, so half a unit is at most this share of it
STEP = 0.5 / 4177792
U = 2.0 ** -24  # half a step of f32, relative


def layer_shape(nkv, hd, max_seq):
    return nkv, -(-max_seq // TILE), 2 * TILE * hd + 8 * TILE


def vbyte(t):
    return 16 * ((t // 4) % 4) + 4 * (t // 16) + t % 4


def codes(x):
    """[..., hd] f32 → int codes (64 bits: exact quotients, ties to even) and f32 scales."""
    amax = x.abs().amax(-1)
    fine = torch.isfinite(amax)
    a = torch.where(fine & (amax > 0), amax, torch.ones_like(amax)).double()
    c = torch.round(x.double() * 127.0 / a[..., None])
    c = torch.where((fine & (amax > 0))[..., None], c, torch.zeros_like(c)).to(torch.int8)
    s = torch.where(fine, (amax.double() / 127.0).float(), torch.full_like(amax, math.nan))
    return c, s


def unpack(layer, nkv, hd, max_seq):
    """The bytes of a layer slice → codes [nkv][slots][hd] of K and V (int8), scales [nkv][slots]."""
    h, tiles, _ = layer_shape(nkv, hd, max_seq)
    b = layer.reshape(h, tiles, -1)
    k = b[..., :TILE * hd].reshape(h, tiles * TILE, hd).view(torch.int8)
    v = b[..., TILE * hd:2 * TILE * hd].reshape(h, tiles, hd, TILE).view(torch.int8)
    at = torch.tensor([vbyte(t) for t in range(TILE)], device=layer.device)
    v = v[..., at].transpose(-1, -2).reshape(h, tiles * TILE, hd)
    s = b[..., 2 * TILE * hd:].contiguous().view(torch.float32)
    return k, v, s[..., :TILE].reshape(h, -1), s[..., TILE:].reshape(h, -1)


def pack(kc, ks, vc, vs):
    """Codes [nkv][slots][hd] (slots a multiple of 64) and scales → the bytes of a layer slice."""
    h, slots, hd = kc.shape
    tiles = slots // TILE
    out = torch.empty((h, tiles, 2 * TILE * hd + 8 * TILE), dtype=torch.uint8, device=kc.device)
    out[..., :TILE * hd] = kc.reshape(h, tiles, -1).contiguous().view(torch.uint8)
    inv = torch.empty(TILE, dtype=torch.long, device=kc.device)
    for t in range(TILE):
        inv[vbyte(t)] = t
    v = vc.reshape(h, tiles, TILE, hd)[:, :, inv].transpose(-1, -2).contiguous()
    out[..., TILE * hd:2 * TILE * hd] = v.reshape(h, tiles, -1).view(torch.uint8)
    s = torch.cat([ks.reshape(h, tiles, TILE), vs.reshape(h, tiles, TILE)], -1).contiguous()
    out[..., 2 * TILE * hd:] = s.view(torch.uint8)
    return out


def attention(q, layer, nkv, hd, max_seq, length, window):
    """q [n][heads·hd] f32 of the last n of `length` tokens → (result, bound), both [n][heads·hd] f64. The
    bound is what the roundings of include/aether_hip.h allow, element by element:
      q:  half a unit of 24 bits of the row's largest component, times Σ|k| of the key;
      score: 8 f32 roundings of it, and as the sum of 16 products at a time in two parts (two roundings a
        step: the products' sum, the running one) hd/4 of Σ|q·k|;
      exponential: 4, and that of its argument, 2·|s - max|·U;
      p·sv: half a unit of 24 bits of the tile's largest, times Σ|code| over the tile, or of itself and
        2^-34 of the row's largest, times the code;
      sums: as the scores', tokens/4 roundings, 16 for what joins waves and chunks, for sum and output each."""
    n, heads = q.shape[0], q.shape[1] // hd
    g = heads // nkv
    kc, vc, ks, vs = unpack(layer, nkv, hd, max_seq)
    out = torch.zeros((n, heads * hd), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    if length == 0:
        return out, tol
    pos = torch.arange(length - n, length, device=q.device)[:, None]
    t = torch.arange(length, device=q.device)[None, :]
    seen = (t <= pos) & ((t > pos - window) if window else (t >= 0))
    tiles = -(-length // TILE)
    pad = tiles * TILE - length
    for h in range(nkv):
        kd = kc[h, :length].double() * ks[h, :length, None].double()
        vd = vc[h, :length].double() * vs[h, :length, None].double()
        some = seen.any(0)
        kd, vd = torch.where(some[:, None], kd, 0.0), torch.where(some[:, None], vd, 0.0)
        for j in range(h * g, (h + 1) * g):
            qd = q[:, j * hd:(j + 1) * hd].double()
            s = (qd @ kd.t().contiguous()) / math.sqrt(hd)
            s = torch.where(seen, s, -math.inf)
            m = s.amax(1, keepdim=True)
            p = torch.exp(s - m)
            l = p.sum(1, keepdim=True)
            cols = slice(j * hd, (j + 1) * hd)
            pv = torch.where(p == 0, 0.0, p)
            out[:, cols] = (pv @ vd) / l
            mass = (pv @ vd.abs()) / l
            es = (qd.abs().amax(1, keepdim=True) * STEP * kd.abs().sum(1)[None] + hd / 4 * U * (qd.abs() @ kd.abs().t().contiguous())) / math.sqrt(hd)
            es = es + 8 * U * s.abs() + 4 * U + 2 * U * (s - m).abs()
            es = torch.where(seen, es, 0.0).amax(1, keepdim=True)
            w = torch.nn.functional.pad(p * torch.where(some, vs[h, :length].double(), 0.0)[None], (0, pad)).reshape(n, tiles, TILE).amax(2)
            far = w.amax(1, keepdim=True) * 2.0 ** -34 * torch.where(some[:, None], vc[h, :length].double().abs(), 0.0).sum(0)
            c = torch.nn.functional.pad(torch.where(some[:, None], vc[h, :length].double().abs(), 0.0), (0, 0, 0, pad)).reshape(tiles, TILE, hd).sum(1)
            tol[:, cols] = 2 * es * mass + (STEP * (w @ c) + far) / l + U * mass + 2 * (length / 4 + 16) * U * mass
    return out, tol + 1e-37


def qk_norm_rope(x, nq, nk, hd, qw, kw, eps, positions, sin, cos):
    """[n][>= (nq + nk)·hd] f32 → (result, bound) [n][(nq + nk)·hd] f64: eight f32 roundings of each factor
    (the sum of squares: hd / 8 in a lane and six joins, halved by the root), three of the rotation."""
    n = x.shape[0]
    y = x[:, :(nq + nk) * hd].double().reshape(n, nq + nk, hd)
    for part, w in ((slice(0, nq), qw), (slice(nq, nq + nk), kw)):
        if w is not None:
            z = y[:, part]
            y[:, part] = z / torch.sqrt((z * z).mean(-1, keepdim=True) + eps) * w.double()
    p = positions.clamp(0, sin.shape[0] - 1).long()
    s, c = sin[p].double()[:, None], cos[p].double()[:, None]
    a, b = y[..., :hd // 2], y[..., hd // 2:]
    out = torch.cat([a * c - b * s, a * s + b * c], -1)
    mag = torch.cat([(a * c).abs() + (b * s).abs()] * 2, -1).maximum(torch.cat([(a * s).abs() + (b * c).abs()] * 2, -1))
    return out.reshape(n, -1), ((hd / 16 + 14) * U * mag).reshape(n, -1) + 1e-37


def quantised(x):
    """numpy [..., hd] f32 → the values its codes stand for (f32)."""
    import numpy as np

    c, s = codes(torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)))
    return (c.float() * s[..., None]).numpy()


def model_logits(c, m, tokens):
    """The last position's logits of a small test model (tests/_models.py) in float64, with every token's K and V
    held in 8 bits: causal over `tokens` at positions 0 .. len-1, c["sliding_window"] as the runner's."""
    import numpy as np

    from oracle import oracle as O
    from tests._model64 import _deq

    d, nh, nkv, hd, dff, ms = (c[k] for k in ("d_model", "num_heads", "num_kv_heads", "head_dim", "d_ff", "max_seq_len"))
    shapes = [(nh * hd, d), (nkv * hd, d), (nkv * hd, d), (d, nh * hd), (dff, d), (dff, d), (d, dff)]
    sin, cos = (t.reshape(ms, hd // 2).astype(np.float64) for t in O.precompute_rope(ms, hd, c["rope_base"]))
    n = len(tokens)
    at = np.minimum(np.arange(n), ms - 1)
    ago = np.arange(n)[:, None] - np.arange(n)
    seen = (ago >= 0) & (ago < (c.get("sliding_window") or n))

    def norm(v, w):
        return v / np.sqrt((v * v).mean(-1, keepdims=True) + c["rms_norm_eps"]) * w.astype(np.float64)

    def rotated(v):
        a, b, s, k = v[..., :hd // 2], v[..., hd // 2:], sin[at][:, None], cos[at][:, None]
        return np.concatenate([a * k - b * s, a * s + b * k], -1)

    x = m["emb"].astype(np.float64)[np.asarray(tokens)]
    for weights, (w_attn, w_ffn) in zip(m["layers"], m["norms"]):
        wq, wk, wv, wo, wg, wu, wd = (_deq(t, w, *s) for t, w, s in zip(m["layer_dtype"], weights, shapes))
        h = norm(x, w_attn)
        q = rotated((h @ wq.T).reshape(n, nh, hd))
        k = quantised(rotated((h @ wk.T).reshape(n, nkv, hd))).astype(np.float64)
        v = quantised((h @ wv.T).reshape(n, nkv, hd)).astype(np.float64)
        heads = []
        for j in range(nh):
            s = np.where(seen, q[:, j] @ k[:, j * nkv // nh].T / math.sqrt(hd), -np.inf)
            p = np.exp(s - s.max(1, keepdims=True))
            heads.append(p @ v[:, j * nkv // nh] / p.sum(1, keepdims=True))
        x = x + np.concatenate(heads, 1) @ wo.T
        h = norm(x, w_ffn)
        g, u = h @ wg.T, h @ wu.T
        with np.errstate(over="ignore"):
            x = x + (g / (1 + np.exp(-g)) * u) @ wd.T
    return _deq(m["lm_dtype"], m["lm"], c["vocab_size"], d) @ norm(x[-1], m["final"])
