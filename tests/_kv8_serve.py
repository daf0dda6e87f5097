"""Attention behind a shared prefix, the weights that cached tokens receive and the
eviction by them, from their definitions in 64 bits over unpacked caches
(tests/_kv8.py), with the bounds that the kernels' roundings allow."""
import math

import torch

from tests import _kv8 as R

TILE, STEP, U = R.TILE, R.STEP, R.U


def padded(parts):
    """Parts [(kc, ks, vc, vs, slots)] of unpacked heads [slots][hd] one behind the other, each from a tile of its own on:
    the joined arrays and the places of the parts' slots in them."""
    out, at, places = [[], [], [], []], 0, []
    for *arrays, slots in parts:
        pad = -slots % TILE
        for o, x in zip(out, arrays):
            o.append(torch.nn.functional.pad(x[:slots], (0, 0, 0, pad) if x.dim() == 2 else (0, pad)))
        places.append(torch.arange(at, at + slots, device=arrays[0].device))
        at += slots + pad
    return [torch.cat(o) for o in out], torch.cat(places)


def rows(q, kc, ks, vc, vs, seen):
    """q [rows][hd] over the tokens of one KV head (a multiple of 64 of them), seen [rows][tokens]: the result, its
    bound, the probabilities and the bounds of those, all f64. The bounds are those that R.attention derives; a probability
    2^(s - m)/l adds its own score's and the sum's: 2·es (score and sum) + (tokens/4 + 16)·U (the sum) + 8·U (difference, exponential, quotient, product)."""
    hd, tokens = kc.shape[1], kc.shape[0]
    some = seen.any(0)
    kd = torch.where(some[:, None], kc.double() * ks[:, None].double(), 0.0)
    vd = torch.where(some[:, None], vc.double() * vs[:, None].double(), 0.0)
    qd = q.double()
    s = torch.where(seen, (qd @ kd.t().contiguous()) / math.sqrt(hd), -math.inf)
    m = s.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(s - m)
    l = p.sum(1, keepdim=True)
    l = torch.where(l == 0, 1.0, l)
    out, mass = (p @ vd) / l, (p @ vd.abs()) / l
    es = (qd.abs().amax(1, keepdim=True) * STEP * kd.abs().sum(1)[None] + hd / 4 * U * (qd.abs() @ kd.abs().t().contiguous())) / math.sqrt(hd)
    es = torch.where(seen, es + 8 * U * s.abs() + 4 * U + 2 * U * (s - m).abs(), 0.0).amax(1, keepdim=True)
    sv = torch.where(some, vs.double(), 0.0)
    w = (p * sv[None]).reshape(len(q), -1, TILE).amax(2)
    vabs = torch.where(some[:, None], vc.double().abs(), 0.0)
    far = w.amax(1, keepdim=True) * 2.0 ** -34 * vabs.sum(0)
    tol = 2 * es * mass + (STEP * (w @ vabs.reshape(-1, TILE, hd).sum(1)) + far) / l + U * mass + 2 * (tokens / 4 + 16) * U * mass
    return out, tol + 1e-37, p / l, p / l * (2 * es + (tokens / 4 + 24) * U)


def shared(q, prefix, prefix_len, prefix_seq, layers, lens, nkv, hd, max_seq, window):
    """q [seqs][heads·hd] → (result, bound)."""
    g = q.shape[1] // hd // nkv
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    pre = R.unpack(prefix, nkv, hd, prefix_seq) if prefix_len else None
    for b, length in enumerate(lens):
        total = prefix_len + length
        if total == 0:
            continue
        own = R.unpack(layers[b], nkv, hd, max_seq)
        for h in range(nkv):
            parts = [(x[0][h], x[2][h], x[1][h], x[3][h], n) for x, n in ((pre, prefix_len), (own, length)) if n]
            arrays, places = padded(parts)
            seen = torch.zeros(1, len(arrays[0]), dtype=torch.bool, device=q.device)
            seen[0, places[max(0, total - window) if window else 0:]] = True
            at = slice(h * g * hd, (h + 1) * g * hd)
            o, t, _, _ = rows(q[b, at].reshape(g, hd), *arrays, seen.expand(g, -1))
            out[b, at], tol[b, at] = o.reshape(-1), t.reshape(-1)
    return out, tol


def weights(q, layer, nkv, hd, max_seq, seq, window, prior):
    """q [n][heads·hd] of the last n of seq tokens, prior [nkv][max_seq] or None → result, bound, weights [nkv][seq], bound. A sum
    of w over r rows: each addition rounds at most by U of what has been added up, r of them, and the prior's."""
    n, g = q.shape[0], q.shape[1] // hd // nkv
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    w, wt = (torch.zeros(nkv, seq, dtype=torch.float64, device=q.device) for _ in range(2))
    if seq and n:
        kc, vc, ks, vs = R.unpack(layer, nkv, hd, max_seq)
        pos = torch.arange(seq - n, seq, device=q.device)[:, None]
        t = torch.arange(-(-seq // TILE) * TILE, device=q.device)[None]
        seen = (t <= pos) & ((t > pos - window) if window else (t >= 0))
        slots = t.shape[1]
        for h in range(nkv):
            for j in range(h * g, (h + 1) * g):
                at = slice(j * hd, (j + 1) * hd)
                out[:, at], tol[:, at], p, pt = rows(q[:, at], kc[h, :slots], ks[h, :slots], vc[h, :slots], vs[h, :slots], seen)
                w[h] += p[:, :seq].sum(0)
                wt[h] += pt[:, :seq].sum(0)
    wt = wt + n * g * U * w + 1e-37 * n * g
    if prior is not None:
        w = w + prior[:, :seq].double()
        wt = wt + U * w.abs()
    return out, tol, w, wt


def evicted(weights, seq, keep, first, recent):
    """The slots of one head that stay, ascending. weights: a list of floats."""
    if seq <= keep:
        return list(range(seq))
    ends = [t for t in range(seq) if t < first or t >= seq - recent]
    rest = [t for t in range(seq) if first <= t < seq - recent]
    rest.sort(key=lambda t: (weights[t] != weights[t], -weights[t] if weights[t] == weights[t] else 0.0, t))
    return sorted(ends + rest[:keep - first - recent])
