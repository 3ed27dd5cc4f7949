"""8-bit caches and eviction in 64 bits, sequence by sequence and head by head, as their definitions read.  Tensors on the CPU."""
import math

import torch

FLOOR = 2.0 ** -32


def e4m3_values():
    """The 256 codes' values, from their bits: sign, 4 bits of exponent (bias 7), 3 of mantissa; 0x7f and 0xff are NaN."""
    out = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = math.nan if (c & 127) == 127 else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out.append(-v if c & 128 else v)
    return torch.tensor(out, dtype=torch.float64)


VALUES = e4m3_values()


def decode(codes):
    return VALUES[codes.view(torch.uint8).long()]


def encode(x):
    """Codes of the nearest values, the even code of two; not finite, or past 464: NaN."""
    x = x.double()
    grid = VALUES[:127]
    a = x.abs()
    hi = torch.searchsorted(grid, a.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    down, up = a - grid[lo], grid[hi] - a
    code = torch.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    code = torch.where(~torch.isfinite(x) | (a > 464), torch.full_like(code, 127), code)
    return (code + 128 * torch.signbit(x)).to(torch.uint8)


def scale_for(x):
    """The least power of two, from the floor on, by which the finite ones of x come to at most 448."""
    x = x[torch.isfinite(x)].double().abs()
    top, s = (float(x.max()) if x.numel() else 0.0), FLOOR
    while top > 448 * s:
        s *= 2
    return s


def append(x, codes, scale, lengths, counts, block):
    """codes (uint8) and scale with the new rows of x [B,H,M,D], as new tensors."""
    codes, scale = codes.clone(), scale.clone()
    B, H, M, D = x.shape
    for b in range(B):
        n, c = min(max(int(lengths[b]), 0), codes.shape[2]), min(max(int(counts[b]), 0), M)
        first, rows = max(n - c, 0), x[b, :, c - min(c, n):c]
        for blk in range(first // block, -(-n // block) if c else 0):
            lo, hi = max(blk * block, first), min((blk + 1) * block, n)
            if hi <= lo:
                continue
            for h in range(H):
                was = float(scale[b, h, blk]) if lo > blk * block else FLOOR
                now = max(was, scale_for(rows[h, lo - first:hi - first]))
                if lo > blk * block and now != was:
                    codes[b, h, blk * block:lo] = encode(decode(codes[b, h, blk * block:lo]) * (was / now))
                codes[b, h, lo:hi] = encode(rows[h, lo - first:hi - first].double() / now)
                scale[b, h, blk] = now
    return codes, scale


def attention(q, k8, v8, ks, vs, scale, causal, lengths, counts, block):
    """o, lse, key weights [B,Hkv,S] (sums over rows), and how far o, the weights and lse may be off, derived below; rows that are not there are NaN.

    Errors of a kernel that multiplies exact products of fp16 numbers in fp32 and keeps the softmax in fp32.  A score's is at most (D + 8) 2^-24 sum |q k|
    scale, which is the relative error of its exponential; exp2, log2 and a reciprocal add some 2^-21, the sums of n terms in lanes (n / 32 + 64) 2^-24: e.
    The weight is rounded to fp16 before the product with v: 2^-11 of it, or 2^-25 of the largest weight times scale where that is more (subnormal
    numbers).  The output is rounded to fp16 once."""
    B, Hq, M, D = q.shape
    Hkv, S = k8.shape[1:3]
    G = Hq // Hkv
    o = torch.full(q.shape, math.nan, dtype=torch.float64)
    tol = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full((B, Hq, M), math.nan, dtype=torch.float64)
    ltol = torch.zeros((B, Hq, M), dtype=torch.float64)
    w = torch.zeros((B, Hkv, S), dtype=torch.float64)
    wtol = torch.zeros((B, Hkv, S), dtype=torch.float64)
    for b in range(B):
        n, c = min(max(int(lengths[b]), 0), S), min(max(int(counts[b]), 0), M)
        blk = torch.arange(n) // block
        for h in range(Hkv):
            k = decode(k8[b, h, :n]) * ks[b, h].double()[blk][:, None]
            vc = decode(v8[b, h, :n])
            v = vc * vs[b, h].double()[blk][:, None]
            for g in range(G):
                for i in range(c):
                    head, sees = h * G + g, min(n, max(0, n - c + i + 1)) if causal else n
                    if sees == 0:
                        o[b, head, i], lse[b, head, i], tol[b, head, i] = 0.0, -math.inf, 0.0
                        continue
                    x = q[b, head, i].double()
                    s = (k[:sees] * x).sum(1) * scale
                    p = torch.softmax(s, 0)
                    lse[b, head, i] = torch.logsumexp(s, 0)
                    o[b, head, i] = (p[:, None] * v[:sees]).sum(0)
                    size = float(torch.nan_to_num((k[:sees].abs() * x.abs()).sum(1)).max()) * abs(scale)
                    e = (D + 8) * 2.0 ** -24 * size + 2.0 ** -20 + (sees / 32 + 64) * 2.0 ** -24
                    ltol[b, head, i] = 2 * e + 2.0 ** -22 * lse[b, head, i].abs()
                    mass = (p[:, None] * v[:sees].abs()).sum(0)
                    small = 2.0 ** -25 * vc[:sees].abs().sum(0) * (p * vs[b, h].double()[blk[:sees]]).max()
                    tol[b, head, i] = 2.0 ** -11 * o[b, head, i].abs() + 2.0 ** -25 + (2.0 ** -11 + 2 * e) * mass + 2 * e * o[b, head, i].abs() + small
                    w[b, h, :sees] += p
                    wtol[b, h, :sees] += (2 * e + 2.0 ** -23 + (G * M + 8) * 2.0 ** -24) * p
    return o, lse, w, tol, wtol, ltol


def evict(k, v, weights, keep, recent, lengths, ks=None, vs=None, block=64):
    """Per sequence and head: kept positions, and rows of K, V (as codes, or fp16), scales and weights; a dict of nested lists of tensors."""
    B, Hkv, S = k.shape[:3]
    per = weights.shape[1] // Hkv
    out = {n: [[None] * Hkv for _ in range(B)] for n in ("kept", "k", "v", "ks", "vs", "w")}
    for b in range(B):
        n = min(max(int(lengths[b]), 0), S)
        stay = min(n, keep)
        late = min(recent, stay)
        for h in range(Hkv):
            total = weights[b, h * per:(h + 1) * per, :n].double().sum(0).float()
            rank = [(0 if t != t else 1, 0.0 if t != t else t) for t in total.tolist()]
            early = sorted(range(n - late), key=lambda i: (-rank[i][0], -rank[i][1], i))[:stay - late]
            index = torch.tensor(sorted(early) + list(range(n - late, n)), dtype=torch.long)
            out["kept"][b][h] = index
            out["w"][b][h] = weights[b, h * per:(h + 1) * per][:, index]
            for name, x, scale in (("k", k, ks), ("v", v, vs)):
                rows = x[b, h][index]
                if scale is not None:
                    was = scale[b, h].double()[index // block]
                    now = torch.stack([was[i:i + block].max() for i in range(0, stay, block)]) if stay else was
                    ratio = (was.float() / now.repeat_interleave(block)[:stay].float()).double()
                    same = (ratio == 1.0)[:, None]
                    rows = torch.where(same, rows, encode(decode(rows) * ratio[:, None]))
                    out[name + "s"][b][h] = now.float()
                out[name][b][h] = rows
    return out
