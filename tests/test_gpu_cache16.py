"""fp16 caches on the GPU: the rotated append, attention behind a shared prefix, bounds of blocks, selection and attention over what is selected, against the definitions in
64 bits.  Bounds and selections are held to equality, outputs to what oracle/cache16.py derives."""
import math

import pytest
import torch

from oracle import cache16 as ref
from triton_amd import modules, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _laid(x, layout):
    """A GPU copy of [B,H,S,D] in memory of its own order; what lies between the rows is NaN."""
    B, H, S, D = x.shape
    if layout == "token":
        dev = torch.empty(B, S, H, D, dtype=x.dtype, device=DEV).permute(0, 2, 1, 3)
    elif layout == "padded":
        dev = torch.full((B, H, S, D + 16), math.nan, dtype=x.dtype, device=DEV)[..., 8:8 + D]
    else:
        dev = torch.empty(B, H, S, D, dtype=x.dtype, device=DEV)
    return dev.copy_(x)


def _within(got, want, tol, what=""):
    got = got.detach().cpu().double()
    same = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~same & ~torch.isnan(want)], want[~same & ~torch.isnan(want)]), what
    off = ((got - want).abs() - tol)[same]
    assert not off.numel() or float(off.max()) <= 0, f"{what}: {float(off.max())} past the bound"


# ------------------------------------------------------------------------------------------------ rotated append
ROPES = [
    # B, Hq, Hkv, D, new, capacity, lengths, counts, pairs, axes
    (1, 32, 8, 128, 1, 40, [33], [1], 64, 1),
    (2, 4, 2, 64, 3, 50, [3, 50], [3, 2], 32, 1),                       # the first tokens; a padded row; the capacity's end
    (3, 71, 1, 64, 2, 9, [0, 1, 9], [2, 2, 0], 16, 1),                  # no key, more new tokens than keys, nothing new
    (2, 3, 3, 128, 37, 300, [300, 41], [37, 30], 20, 1),
    (1, 8, 2, 128, 70, 80, [75], [70], 64, 3),
    (2, 16, 16, 64, 5, 12, [12, 7], [5, 4], 12, 2),
    (1, 2, 1, 64, 4, 6, [6], [4], 0, 1),                                # nothing is rotated
]


@pytest.mark.parametrize("case", ROPES, ids=lambda c: f"B{c[0]}H{c[1]}_{c[2]}D{c[3]}M{c[4]}p{c[8]}a{c[9]}")
@pytest.mark.parametrize("norm", [None, "plain", "weighted"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ["head", "token", "padded"])
def test_rope(case, norm, interleaved, layout):
    B, Hq, Hkv, D, M, S, lengths, counts, pairs, axes = case
    g = _gen(1)
    q, k, v = (torch.randn(B, h, M, D, generator=g).half() for h in (Hq, Hkv, Hkv))
    for b, c in enumerate(counts):
        for x in (q, k, v):
            x[b, :, c:] = math.nan                                      # padding is not read
    kc, vc, qo = (torch.randn(B, h, s, D, generator=g).half() for h, s in ((Hkv, S), (Hkv, S), (Hq, M)))
    inv = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1)) if pairs else None
    sections = positions = None
    if axes > 1:
        sections = [pairs - (axes - 1) * (pairs // 4)] + [pairs // 4] * (axes - 1)
        positions = torch.randint(0, 200000, (axes, B, M), generator=g).int()
    gq, gk = ((1 + 0.2 * torch.randn(D, generator=g)).half() if norm == "weighted" else None for _ in range(2))
    outs, tols = ref.rope(q, k, v, qo, kc, vc, inv, lengths, counts, positions, gq, gk, norm is not None, 1e-6, interleaved, sections)
    dev = {n: _laid(x, layout) for n, x in dict(q=q, k=k, v=v, q_out=qo, k_cache=kc, v_cache=vc).items()}
    up = lambda t: None if t is None else t.to(DEV)
    ops.cache_rope_append(dev["q"], dev["k"], dev["v"], dev["q_out"], dev["k_cache"], dev["v_cache"], up(inv), _ints(lengths), _ints(counts), up(positions), up(gq), up(gk),
                          norm is not None, 1e-6, interleaved, sections)
    for n, want, tol in zip(("q_out", "k_cache", "v_cache"), outs, tols):
        _within(dev[n], want, tol, n)


def test_rope_far_positions_in_place_and_packed():
    """Positions near the ends of what a long cache has, queries in place, q, k and v beside each other as a projection leaves them, caches in one tensor."""
    B, Hq, Hkv, D, M, S = 2, 4, 2, 64, 3, 5
    g = _gen(2)
    qkv = torch.randn(B, M, Hq + 2 * Hkv, D, generator=g).half()
    inv = 500000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    positions = torch.tensor([[[0, 1, 2 ** 26], [999999, -7, 131072]]], dtype=torch.int32)
    both = torch.zeros(B, 2, Hkv, S, D).half()
    part = lambda t: (t.permute(0, 2, 1, 3)[:, :Hq], t.permute(0, 2, 1, 3)[:, Hq:Hq + Hkv], t.permute(0, 2, 1, 3)[:, Hq + Hkv:])
    q, k, v = part(qkv)
    outs, tols = ref.rope(q, k, v, q, both[:, 0], both[:, 1], inv, [S, 4], [M, M], positions)
    d, db = qkv.to(DEV), both.to(DEV)
    dq, dk, dv = part(d)
    ops.cache_rope_append(dq, dk, dv, dq, db[:, 0], db[:, 1], inv.to(DEV), _ints([S, 4]), None, positions.to(DEV))
    for got, want, tol in zip((dq, db[:, 0], db[:, 1]), outs, tols):
        _within(got, want, tol)
    assert torch.equal(d.cpu()[:, :, Hq:], qkv[:, :, Hq:])


# ------------------------------------------------------------------------------------------------ shared prefix
PREFIXES = [
    # B, Hq, Hkv, D, new, capacity, lengths, counts, prefix, causal
    (1, 32, 8, 128, 1, 40, [33], [1], 100, True),
    (4, 32, 8, 128, 1, 300, [1, 64, 65, 300], [1, 1, 1, 1], 1000, True),       # 16 rows a head
    (9, 32, 8, 128, 1, 70, list(range(1, 70, 8)), [1] * 9, 700, True),         # 36 rows: wide tiles
    (3, 71, 1, 64, 1, 33, [33, 0, 5], [1, 0, 1], 130, True),                   # a sequence without a query; one of no keys
    (3, 4, 2, 64, 3, 10, [10, 2, 0], [3, 3, 2], 5, True),                      # fewer keys than queries
    (3, 4, 2, 64, 3, 10, [10, 2, 0], [3, 3, 2], 0, True),                      # no prefix: rows that see nothing
    (2, 2, 2, 128, 17, 90, [90, 17], [17, 9], 65, True),
    (2, 8, 1, 64, 40, 200, [200, 77], [40, 40], 63, True),                     # tiles of one sequence's rows
    (2, 8, 2, 128, 150, 260, [260, 150], [150, 97], 190, True),
    (2, 8, 2, 128, 150, 260, [260, 150], [150, 97], 0, True),
    (2, 8, 2, 128, 20, 260, [260, 150], [20, 11], 64, False),
    (1, 4, 1, 128, 2, 1, [1], [2], 1, False),
]


@pytest.mark.parametrize("case", PREFIXES, ids=lambda c: f"B{c[0]}H{c[1]}_{c[2]}D{c[3]}M{c[4]}S{c[5]}P{c[8]}{'c' if c[9] else ''}")
@pytest.mark.parametrize("layout", ["head", "token", "padded"])
def test_prefix_attention(case, layout):
    B, Hq, Hkv, D, M, S, lengths, counts, P, causal = case
    g = _gen(3)
    q, k, v = (torch.randn(B, h, s, D, generator=g).half() for h, s in ((Hq, M), (Hkv, S), (Hkv, S)))
    kp, vp = (torch.randn(1, Hkv, P, D, generator=g).half() for _ in range(2))
    o = torch.randn(B, Hq, M, D, generator=g).half()
    for b, (n, c) in enumerate(zip(lengths, counts)):
        k[b, :, n:] = math.nan
        v[b, :, n:] = math.nan
        q[b, :, c:] = math.nan
    want, tol = ref.prefix_attention(q, k, v, kp[0], vp[0], o, D ** -0.5, causal, lengths, counts)
    dq, dk, dv, dkp, dvp, do = (_laid(x, layout) for x in (q, k, v, kp, vp, o))
    modules.get("prefix", "cache", causal=causal).forward(dk, dkp[0], do, dq, dv, dvp[0], _ints(counts), _ints(lengths))
    _within(do, want, tol)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M", [6, 40])
def test_prefix_attention_of_what_is_not_finite(D, M):
    """Infinities and NaN in values and keys of tokens that a query does not see stay out of its output; those that it sees come through."""
    B, Hq, Hkv, S, P = 2, 8, 2, 50, 70
    g = _gen(4)
    q, k, v = (torch.randn(B, h, s, D, generator=g).half() for h, s in ((Hq, M), (Hkv, S), (Hkv, S)))
    kp, vp = (torch.randn(1, Hkv, P, D, generator=g).half() for _ in range(2))
    v[0, 0, S - 1, 3], v[0, 0, S - 2, 4], v[0, 1, S - 3, 5] = math.inf, -math.inf, math.nan
    k[1, 0, S - 1] = math.nan
    k[1, 1, S - 2] = math.inf
    v[1, 1, S - 2] = math.inf
    o = torch.zeros(B, Hq, M, D).half()
    lengths, counts = [S, S], [M, M]
    want, tol = ref.prefix_attention(q, k, v, kp[0], vp[0], o, D ** -0.5, True, lengths, counts)
    args = [x.to(DEV) for x in (k, kp[0], o, q, v, vp[0])]
    modules.get("prefix", "cache").forward(*args, None, None)
    got = args[2].cpu().double()
    # (a key that is not finite makes its queries' rows NaN, whatever else is there)
    for b, h, first in ((1, 0, M - 1), (1, 1, M - 2)):
        rows = slice(h * 4, h * 4 + 4)
        assert torch.isnan(got[b, rows, first:]).any(-1).all()
        got[b, rows, first:] = want[b, rows, first:] = 0.0
        tol[b, rows, first:] = 0.0
    assert torch.equal(torch.isfinite(got), torch.isfinite(want))
    _within(got, want, torch.nan_to_num(tol, nan=0.0, posinf=0.0))


# ------------------------------------------------------------------------------------------------ bounds, selection
SPARSES = [
    # B, Hq, Hkv, D, new, capacity, lengths, counts, block, top, sink, recent
    (1, 32, 8, 128, 1, 1000, [999], [1], 32, 8, 1, 2),
    (3, 8, 2, 64, 1, 700, [700, 1, 333], [1, 1, 1], 64, 4, 0, 1),
    (2, 4, 4, 128, 5, 600, [600, 321], [5, 3], 32, 6, 2, 3),
    (1, 71, 1, 64, 2, 900, [897], [2], 64, 5, 1, 1),
    (2, 4, 1, 128, 40, 300, [300, 20], [40, 33], 128, 2, 0, 1),              # fewer keys than queries
    (1, 2, 1, 64, 70, 2500, [2500], [70], 32, 70, 2, 8),
    (2, 2, 1, 64, 1, 64, [0, 64], [1, 0], 32, 1, 0, 1),                       # no key; no query
    (1, 4, 2, 64, 3, 200, [150], [3], 32, 40, 2, 4),                          # more places than blocks
    (1, 4, 1, 128, 1, 40000, [39999], [1], 32, 128, 1, 4),
]


def _sparse_inputs(case, seed=5):
    B, Hq, Hkv, D, M, S, lengths, counts, block, top, sink, recent = case
    g = _gen(seed)
    q, k, v = (torch.randn(B, h, s, D, generator=g).half() for h, s in ((Hq, M), (Hkv, S), (Hkv, S)))
    o = torch.randn(B, Hq, M, D, generator=g).half()
    for b, (n, c) in enumerate(zip(lengths, counts)):
        k[b, :, n:] = math.nan
        v[b, :, n:] = math.nan
        q[b, :, c:] = math.nan
    blocks = -(-S // block)
    bnd = ref.bounds(k, torch.zeros(B, Hkv, blocks, 2, D).half(), block, lengths, [S] * B)
    return q, k, v, o, bnd, torch.full((B, Hkv, M, top), 77, dtype=torch.int32)


@pytest.mark.parametrize("case", SPARSES, ids=lambda c: f"B{c[0]}H{c[1]}_{c[2]}D{c[3]}M{c[4]}S{c[5]}b{c[8]}t{c[9]}")
@pytest.mark.parametrize("layout", ["head", "token", "padded"])
def test_bounds(case, layout):
    B, Hq, Hkv, D, M, S, lengths, counts, block, *_ = case
    q, k, v, o, bnd, sel = _sparse_inputs(case)
    k[0, :, 0, 1] = math.nan                                                  # does not count
    k[0, :, :, 2] = math.nan                                                  # nothing else is there
    old = torch.randn(bnd.shape, generator=_gen(6)).half()
    want = ref.bounds(k, old, block, lengths, counts)
    got = old.to(DEV)
    modules.get("bounds", "cache", block=block).forward(_laid(k, layout), got, _ints(counts), _ints(lengths))
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("case", SPARSES, ids=lambda c: f"B{c[0]}H{c[1]}_{c[2]}D{c[3]}M{c[4]}S{c[5]}b{c[8]}t{c[9]}")
@pytest.mark.parametrize("layout", ["head", "token", "padded"])
def test_sparse_attention(case, layout):
    B, Hq, Hkv, D, M, S, lengths, counts, block, top, sink, recent = case
    q, k, v, o, bnd, sel = _sparse_inputs(case)
    want_sel = ref.select(q, bnd, sel, block, top, sink, recent, Hq // Hkv, lengths, counts, S)
    want, tol = ref.sparse_attention(q, k, v, o, want_sel, block, D ** -0.5, lengths, counts)
    dq, dk, dv, do = (_laid(x, layout) for x in (q, k, v, o))
    dsel = sel.to(DEV)
    modules.get("sparse", "cache", block=block, top=top, sink=sink, recent=recent).forward(dk, do, dq, dv, bnd.to(DEV), _ints(counts), _ints(lengths), dsel)
    assert torch.equal(dsel.cpu(), want_sel)
    _within(do, want, tol)


def test_selection_of_equals_and_of_what_is_no_number():
    """Equal scores go to the earlier block; NaN is the least, -inf next to it, +inf the largest; zeros of both signs are one."""
    B, Hq, Hkv, D, M, block, top, sink, recent = 1, 2, 1, 64, 1, 32, 9, 1, 2
    S = 32 * 600
    q = torch.zeros(B, Hq, M, D).half()
    q[0, 0, 0, 0], q[0, 1, 0, 1] = 1.0, -1.0
    bnd = torch.zeros(B, Hkv, 600, 2, D).half()
    bnd[0, 0, :, :, 0] = (torch.arange(600) % 7)[:, None].half()
    cases = []
    for fill in (0.0, 3.0, -0.0):
        x = bnd.clone()
        if fill == 3.0:
            x[0, 0, 100:110, :, 0] = math.inf
            x[0, 0, 200:300, :, 0] = math.nan
            x[0, 0, 200:300, :, 1] = math.nan
        if fill == 0.0:
            x[:] = 0.0
            x[0, 0, ::2, 0, 0] = -0.0
        cases.append(x)
    k, v = torch.randn(B, Hkv, S, D, generator=_gen(7)).half(), torch.randn(B, Hkv, S, D, generator=_gen(8)).half()
    for x in cases:
        sel = torch.zeros(B, Hkv, M, top, dtype=torch.int32, device=DEV)
        ws = torch.empty(ops.cache_sparse_attention_workspace_bytes(q, k, top, block), dtype=torch.uint8, device=DEV)
        ops.cache_sparse_attention(q.to(DEV), k.to(DEV), v.to(DEV), x.to(DEV), torch.empty_like(q, device=DEV), sel, top, sink, recent, block, workspace=ws)
        got = sel.cpu()[0, 0, 0].tolist()
        score = torch.maximum(*(torch.nan_to_num((s * x[0, 0, :, :, c].double()).amax(-1), nan=-math.inf, posinf=math.inf) for c, s in ((0, 1.0), (1, -1.0)))).tolist()
        rest = sorted(range(1, 598), key=lambda b: (-score[b], b))[:6]
        assert got == sorted([0, 598, 599] + rest)


MANY = [
    # as SPARSES: blocks of more than 2048, and of more than a workgroup holds
    (1, 4, 1, 64, 2, 32 * 3001, [32 * 3000 + 5], [2], 32, 33, 1, 2),
    (2, 8, 1, 128, 1, 32 * 2100, [32 * 2100, 32 * 1500 + 7], [1, 1], 32, 20, 0, 1),
    (1, 2, 2, 64, 1, 32 * 8300, [32 * 8300 - 1], [1], 32, 40, 2, 3),
    (1, 2, 1, 128, 300, 1500, [1500], [300], 32, 6, 1, 1),
    (5, 8, 8, 64, 30, 900, [900, 30, 500, 31, 0], [30, 30, 17, 1, 30], 64, 4, 1, 1),      # a wave a query
]


@pytest.mark.parametrize("case", MANY, ids=lambda c: f"B{c[0]}H{c[1]}_{c[2]}D{c[3]}M{c[4]}S{c[5]}b{c[8]}t{c[9]}")
@pytest.mark.parametrize("size", [1.0, 2e-4, 300.0])
def test_selection_of_many_blocks(case, size):
    """Scores of ordinary size, of numbers near fp16's least (which a matrix pipe may take for zero), and of large ones; keys alike in all blocks but the last bits."""
    B, Hq, Hkv, D, M, S, lengths, counts, block, top, sink, recent = case
    g = _gen(9)
    q = (torch.randn(B, Hq, M, D, generator=g) * size).half()
    base = torch.randn(B, Hkv, 1, 2, D, generator=g)
    blocks = -(-S // block)
    bnd = ((base + torch.randn(B, Hkv, blocks, 2, D, generator=g) * 0.002).sort(3).values * min(size, 100.0)).half()
    sel = torch.full((B, Hkv, M, top), 5, dtype=torch.int32)
    want = ref.select(q, bnd, sel, block, top, sink, recent, Hq // Hkv, lengths, counts, S)
    k, v = (torch.randn(B, Hkv, S, D, generator=g).half() for _ in range(2))
    dsel, do = sel.to(DEV), torch.zeros_like(q, device=DEV)
    modules.get("sparse", "cache", block=block, top=top, sink=sink, recent=recent).forward(k.to(DEV), do, q.to(DEV), v.to(DEV), bnd.to(DEV), _ints(counts), _ints(lengths), dsel)
    assert torch.equal(dsel.cpu(), want)
    if size == 1.0:
        out, tol = ref.sparse_attention(q, k, v, torch.zeros_like(q), want, block, D ** -0.5, lengths, counts)
        _within(do, out, tol)
