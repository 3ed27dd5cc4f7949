"""The operators of an fp16 cache in 64 bits, sequence by sequence and head by head, as their definitions read, with the bounds that a computation in 32 bits with outputs
of 16 keeps.  Tensors on the CPU.

HALF: a value rounded to fp16 is off by at most 2^-11 of itself, or half of its smallest step, 2^-25."""
import math

import torch

HALF, TINY, EPS32 = 2.0 ** -11, 2.0 ** -25, 2.0 ** -24


def sizes(lengths, counts, cap, m):
    for b, (n, c) in enumerate(zip(lengths, counts)):
        yield b, min(max(n, 0), cap), min(max(c, 0), m)


def rope(q, k, v, q_out, k_cache, v_cache, inv_freq, lengths, counts, positions=None, gamma_q=None, gamma_k=None, norm=False, eps=1e-6, interleaved=False, sections=None):
    """(q_out, k_cache, v_cache) in 64 bits, and how far each may be off.

    A turn's fraction is rounded to 32 bits, 2^-25 of a turn: 2 pi 2^-25 < 2^-22; sine and cosine within 2^-22, the two products and their sum within 2^-22: each element of the
    pair counts with 2^-20.  A norm's sum of D squares is off by D 2^-24 of itself at most, of which the root has half; root, division and products 2^-21."""
    outs = [x.double().clone() for x in (q_out, k_cache, v_cache)]
    tols = [torch.zeros_like(x) for x in outs]
    pairs = 0 if inv_freq is None else len(inv_freq)
    sections = [pairs] if sections is None else sections
    axis = torch.tensor([a for a, many in enumerate(sections) for _ in range(many)], dtype=torch.long)
    D = q.shape[-1]
    for b, n, c in sizes(lengths, counts, k_cache.shape[2], q.shape[2]):
        for i in range(c):
            at = n - c + i
            where = torch.full((pairs,), float(at), dtype=torch.float64) if positions is None else positions[axis, b, i].double()
            angle = where * inv_freq if pairs else where
            cos, sin = torch.cos(angle), torch.sin(angle)
            for which, (x, gamma) in enumerate(((q, gamma_q), (k, gamma_k), (v, None))):
                if which and at < 0:
                    continue
                y = x[b, :, i].double()
                if which < 2:
                    if norm:
                        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
                        if gamma is not None:
                            y = y * gamma.double()
                    rel = (D * EPS32 / 2 + 2.0 ** -21) if norm else 0.0
                    tol = y.abs() * rel
                    first = torch.arange(pairs) * 2 if interleaved else torch.arange(pairs)
                    second = first + (1 if interleaved else pairs)
                    z, t = y.clone(), tol.clone()
                    z[:, first] = y[:, first] * cos - y[:, second] * sin
                    z[:, second] = y[:, second] * cos + y[:, first] * sin
                    t[:, first] = t[:, second] = (y[:, first].abs() + y[:, second].abs()) * (rel + 2.0 ** -20)
                    y, tol = z, t + z.abs() * HALF * 1.001 + TINY
                    if not norm:
                        still = torch.ones(D, dtype=torch.bool)
                        still[first] = still[second] = False
                        tol[:, still] = 0.0
                else:
                    tol = torch.zeros_like(y)
                if which == 0:
                    outs[0][b, :, i], tols[0][b, :, i] = y, tol
                else:
                    outs[which][b, :, at], tols[which][b, :, at] = y, tol
    return outs, tols


def _attend(q, k, v, scale, sees):
    """One head's queries over keys of which each sees some: outputs and how far they may be off.

    A score is off by (D + 4) 2^-24 of the sum of its products' magnitudes, times the scale s; a weight by as much again and 2^-21; weights enter the product with V as
    fp16 (off by 2^-11, or by half of the smallest step next to a largest weight of 2^7); numerator and sum: twice.  What does not matter (a key that no query
    sees) may be anything."""
    D = q.shape[1]
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for i in range(len(q)):
        mine = sees[i].nonzero()[:, 0]
        if not len(mine):
            continue
        kk, vv, x = k[mine].double(), v[mine].double(), q[i].double()
        t = kk @ x * scale
        size = (kk.abs() @ x.abs() * scale)
        p = torch.softmax(t, 0)
        if not torch.isfinite(vv).all():
            out[i] = (p[:, None] * vv).sum(0)
        else:
            out[i] = p @ vv
        mag = p @ vv.abs()
        tol[i] = mag * (HALF + 2 * (float(size.max()) * (D + 8) * EPS32 + 2.0 ** -21)) + out[i].abs() * HALF + TINY + vv.abs().sum(0) * float(p.max()) * 2.0 ** -32
    return out, tol


def prefix_attention(q, k, v, kp, vp, o, scale, causal, lengths, counts):
    out, tol = o.double().clone(), torch.zeros(o.shape, dtype=torch.float64)
    G, P = q.shape[1] // k.shape[1], kp.shape[1]
    for b, n, c in sizes(lengths, counts, k.shape[2], q.shape[2]):
        own = torch.arange(n)[None] <= (n - c + torch.arange(c))[:, None] if causal else torch.ones(c, n, dtype=torch.bool)
        sees = torch.cat([torch.ones(c, P, dtype=torch.bool), own], 1)
        for h in range(q.shape[1]):
            j = h // G
            out[b, h, :c], tol[b, h, :c] = _attend(q[b, h, :c], torch.cat([kp[j], k[b, j, :n]]), torch.cat([vp[j], v[b, j, :n]]), scale, sees)
    return out, tol


def bounds(k, old, block, lengths, counts):
    """bounds [B,H,blocks,2,D] with the new tokens' blocks brought up to date."""
    out = old.clone()
    for b, n, c in sizes(lengths, counts, k.shape[2], k.shape[2]):
        c = min(c, n)
        for blk in range((n - c) // block, -(-n // block) if c else 0):
            rows = k[b, :, blk * block:min(n, (blk + 1) * block)].double()
            out[b, :, blk, 0] = torch.where(rows.isnan(), math.inf, rows).amin(1).half()
            out[b, :, blk, 1] = torch.where(rows.isnan(), -math.inf, rows).amax(1).half()
    return out


def select(q, bnd, selected, block, top, sink, recent, group, lengths, counts, cap):
    out = selected.clone()
    for b, n, c in sizes(lengths, counts, cap, q.shape[2]):
        for j in range(bnd.shape[1]):
            for i in range(c):
                ends = (n - c + i) // block if n - c + i >= 0 else -1
                score = torch.full((ends + 1,), -math.inf, dtype=torch.float64)
                for g in range(group):
                    x = q[b, j * group + g, i].double()
                    lo, hi = bnd[b, j, :ends + 1, 0].double(), bnd[b, j, :ends + 1, 1].double()
                    score = torch.maximum(score, torch.maximum(x * lo, x * hi).sum(-1))
                score = [float(s) for s in score.float()]
                forced = [s for s in range(ends + 1) if s < sink or s > ends - recent][:top]
                rest = sorted((s for s in range(ends + 1) if s not in forced), key=lambda s: (-score[s], s))
                take = sorted(forced + rest[:top - len(forced)])
                out[b, j, i] = torch.tensor(take + [-1] * (top - len(take)), dtype=torch.int32)
    return out


def sparse_attention(q, k, v, o, selected, block, scale, lengths, counts):
    out, tol = o.double().clone(), torch.zeros(o.shape, dtype=torch.float64)
    G = q.shape[1] // k.shape[1]
    for b, n, c in sizes(lengths, counts, k.shape[2], q.shape[2]):
        for h in range(q.shape[1]):
            sees = torch.zeros(c, n, dtype=torch.bool)
            for i in range(c):
                for s in selected[b, h // G, i].tolist():
                    if s >= 0:
                        sees[i, s * block:min((s + 1) * block, n - c + i + 1)] = True
            out[b, h, :c], tol[b, h, :c] = _attend(q[b, h, :c], k[b, h // G, :n], v[b, h // G, :n], scale, sees)
    return out, tol
