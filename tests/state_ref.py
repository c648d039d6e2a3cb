"""Plain 64-bit forms of the state cache's operators (tests): one row, head and slot at a time
where that is clearer than fast."""
import math

import numpy as np
import torch


def quantise(x, group):
    """x [..., D] -> codes [..., D] (uint8) and scales [..., D / group, 2] (bfloat16)."""
    g = x.float().unflatten(-1, (-1, group)).cpu()
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) * torch.tensor(1 / 15, dtype=torch.float32)).to(torch.bfloat16)
    b = lo.to(torch.bfloat16)
    bad = ~(torch.isfinite(g).all(-1) & torch.isfinite(s) & torch.isfinite(b))
    s = torch.where(bad, torch.full_like(s, math.nan), s)
    b = torch.where(bad, torch.full_like(b, math.nan), b)
    quot = (g.double() - b.double()[..., None]) / s.double()[..., None]
    c = torch.nan_to_num(quot, nan=0.0).round().clamp(0, 15)
    c = torch.where((s == 0)[..., None] | bad[..., None], torch.zeros_like(c), c)
    return c.to(torch.uint8).flatten(-2), torch.stack([s, b], -1)


def pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def values(codes, scales):
    """Packed codes and scales -> values, 64 bits."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    s = scales.double()
    return (c.unflatten(-1, (s.shape[-2], -1)) * s[..., :1] + s[..., 1:]).flatten(-2)


def attend(q, cache, table, lens, scale):
    """-> out [rows, q_heads, D], probabilities per head [rows, heads, cap], and per row and query
    head the largest |scale| * sum |q k|, the largest |scale| * sum |q| s (s the scale of the
    channel's group) and the largest |v|; all 64 bits, on the CPU."""
    kc, ks, vc, vs = [t.cpu() for t in (cache.k_codes, cache.k_scales, cache.v_codes,
                                        cache.v_scales)]
    q, table, lens = q.cpu().double(), table.cpu().long(), lens.cpu().long()
    rows, nq, dim = q.shape
    heads, page, group = kc.shape[1], kc.shape[2], dim // ks.shape[3]
    g = nq // heads
    out = torch.zeros(rows, nq, dim, dtype=torch.float64)
    prob = torch.zeros(rows, heads, table.shape[1] * page, dtype=torch.float64)
    size, steps, vmax = (torch.zeros(rows, nq, dtype=torch.float64) for _ in range(3))
    for i in range(rows):
        n = int(lens[i])
        if n == 0:
            continue
        j = torch.arange(n)
        p, o = table[i, j // page], j % page
        for h in range(heads):
            k, v = values(kc[p, h, o], ks[p, h, o]), values(vc[p, h, o], vs[p, h, o])
            mine = slice(h * g, (h + 1) * g)
            qs = q[i, mine]
            e = torch.softmax(qs @ k.T * scale, 1)
            out[i, mine] = e @ v
            prob[i, h, :n] = e.sum(0)
            s = ks[p, h, o, :, 0].double().repeat_interleave(group, 1)
            size[i, mine] = (qs.abs() @ k.abs().T).amax(1) * abs(scale)
            steps[i, mine] = (qs.abs() @ s.T).amax(1) * abs(scale)
            vmax[i, mine] = v.abs().max()
    return out, prob, size, steps, vmax


def evict(weights, positions, lens, budget, sinks, recent):
    """-> new weights, positions, lens (numpy) and the moves [(row, head, source, target)]."""
    rows, heads, cols = weights.shape
    new_w = np.zeros((rows, heads, cols), np.float32)
    new_p = np.full((rows, heads, cols), -1, np.int32)
    moves = []
    for i in range(rows):
        n = int(lens[i])
        for h in range(heads):
            w = weights[i, h, :n].copy()
            p = np.arange(n) if positions is None else positions[i, h, :n]
            keep = list(range(n))
            if n > budget:
                top = int(p.max())
                fixed = (p < sinks) | (p >= top + 1 - recent)
                w2 = np.where(np.isnan(w), -np.inf, w)
                order = sorted(range(n), key=lambda j: (not fixed[j], -w2[j], j))
                keep = sorted(order[:budget])
            kept = set(keep)
            holes = [j for j in range(min(n, budget)) if j not in kept]
            movers = [j for j in keep if j >= budget]
            assert len(holes) == len(movers)
            for j in keep:
                if j < budget:
                    new_w[i, h, j], new_p[i, h, j] = w[j], p[j]
            for d, s in zip(holes, movers):
                new_w[i, h, d], new_p[i, h, d] = w[s], p[s]
                moves.append((i, h, s, d))
    return new_w, new_p, np.minimum(lens, budget), moves
