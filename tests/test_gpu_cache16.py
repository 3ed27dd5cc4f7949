"""fp16 caches on the GPU: the rotated append, attention behind a shared prefix, bounds of blocks, selection and attention over what is selected, against the definitions in
64 bits.  Bounds and selections are held to equality, outputs to what oracle/cache16.py derives."""
import math

import pytest
import torch

from oracle import cache16 as ref
from triton_amd import _lib, modules, ops

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


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,M,P,S", [(2, 2, 170, 300), (2, 40, 170, 300), (1, 6, 1300, 700), (12, 1, 2000, 1100), (4, 70, 200, 500)])
def test_infinite_values_that_a_query_sees(B, M, P, S, D):
    """Infinities and NaN in values of the prefix and of the cache, wherever they lie: a channel that has one is no number, as in the formula, and the others keep their numbers."""
    Hq, Hkv = 8, 2
    g = _gen(14)
    q, k, v = (torch.randn(B, h, s, D, generator=g).half() for h, s in ((Hq, M), (Hkv, S), (Hkv, S)))
    kp, vp = (torch.randn(Hkv, P, D, generator=g).half() for _ in range(2))
    vp[0, 40, 3], vp[0, P - 1, 4], vp[1, 70, 5] = math.inf, -math.inf, math.nan
    for b in range(B):
        v[b, 0, 45 + b, 9], v[b, 0, 130, 10], v[b, 1, 64, 11], v[b, 1, 140, 9] = -math.inf, math.nan, math.inf, math.inf
        v[b, 1, 70, 9] = -math.inf if b % 2 else math.inf
    lengths, counts = [S - 9 * b for b in range(B)], [M] * B
    want, tol = ref.prefix_attention(q, k, v, kp, vp, torch.zeros_like(q), D ** -0.5, True, lengths, counts)
    o = torch.zeros(B, Hq, M, D, dtype=torch.float16, device=DEV)
    modules.get("prefix", "cache").forward(*(x.to(DEV) for x in (k, kp)), o, *(x.to(DEV) for x in (q, v, vp)), _ints(counts), _ints(lengths))
    assert torch.equal(o.cpu().isfinite(), want.isfinite())
    _within(o.cpu()[want.isfinite()], want[want.isfinite()], tol[want.isfinite()])
    bnd, sel = torch.zeros(B, Hkv, (S + 63) // 64, 2, D, dtype=torch.float16, device=DEV), torch.zeros(B, Hkv, M, 4, dtype=torch.int32, device=DEV)
    modules.get("bounds", "cache").forward(k.to(DEV), bnd, None, _ints(lengths))
    modules.get("sparse", "cache", top=4).forward(k.to(DEV), o, q.to(DEV), v.to(DEV), bnd, _ints(counts), _ints(lengths), sel)
    want, tol = ref.sparse_attention(q, k, v, torch.zeros_like(q), sel.cpu(), 64, D ** -0.5, lengths, counts)
    assert torch.equal(o.cpu().isfinite(), want.isfinite())
    _within(o.cpu()[want.isfinite()], want[want.isfinite()], tol[want.isfinite()])


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


def test_all_blocks_of_a_long_chunk():
    """No more blocks than places: the attention over the whole cache, and the selection says so."""
    for case in ((2, 8, 2, 128, 150, 260, [260, 150], [150, 97], 64, 5, 1, 1), (1, 71, 1, 64, 2, 3000, [2999], [2], 128, 24, 0, 1)):
        test_sparse_attention(case, "token")


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


# ------------------------------------------------------------------------------------------------ every path of the attention behind a prefix
PATHS = [
    # as PREFIXES: narrow shares of prefix and own keys; two row tiles; wide tiles of 36 and of 300 rows; wide prefix, two narrow blocks of rows; wide rows in shares; no own keys; nothing
    (2, 8, 2, 128, 1, 3000, [3000, 1500], [1, 1], 2500, True),
    (1, 8, 1, 64, 5, 2500, [2500], [5], 1700, True),
    (9, 8, 2, 64, 1, 2700, [2700, 1, 0, 5, 64, 700, 33, 2699, 31], [1, 1, 1, 1, 1, 1, 1, 0, 1], 4001, True),
    (25, 6, 2, 128, 4, 900, [900 - 30 * i for i in range(25)], [1 + i % 4 for i in range(25)], 1500, True),
    (3, 10, 2, 128, 9, 1100, [1100, 9, 300], [9, 9, 4], 1300, True),
    (1, 4, 1, 128, 40, 2600, [2570], [40], 3011, True),
    (1, 5, 1, 64, 33, 3000, [3000], [33], 0, False),
    (2, 4, 2, 64, 2, 0, [0, 0], [2, 1], 70, True),
    (2, 4, 2, 128, 40, 0, [0, 0], [40, 3], 70, True),
    (2, 4, 2, 64, 2, 0, [0, 0], [2, 1], 0, True),
    (1, 8, 8, 128, 1, 700, [1], [1], 0, True),
    (3, 71, 1, 64, 1, 20, [20, 1, 7], [1, 1, 1], 5000, True),
    (2, 71, 1, 64, 3, 100, [100, 50], [3, 2], 300, True),
]


@pytest.mark.parametrize("case", PATHS, ids=lambda c: f"B{c[0]}H{c[1]}_{c[2]}D{c[3]}M{c[4]}S{c[5]}P{c[8]}{'c' if c[9] else ''}")
def test_prefix_attention_paths(case):
    test_prefix_attention(case, "head")


def test_prefix_of_another_layout_than_the_cache():
    """Few keys whose pitches differ between prefix and cache; keys and values likewise."""
    B, Hq, Hkv, D, M, S, P = 2, 4, 2, 64, 2, 60, 45
    g = _gen(11)
    q, k, v = (torch.randn(B, h, s, D, generator=g).half() for h, s in ((Hq, M), (Hkv, S), (Hkv, S)))
    kp, vp = (torch.randn(1, Hkv, P, D, generator=g).half() for _ in range(2))
    want, tol = ref.prefix_attention(q, k, v, kp[0], vp[0], torch.zeros_like(q), D ** -0.5, True, [60, 31], [2, 2])
    for lk, lv, lkp, lvp in (("token", "head", "head", "padded"), ("head", "padded", "token", "head")):
        o = torch.zeros_like(q, device=DEV)
        args = (_laid(k, lk), _laid(kp, lkp)[0], o, q.to(DEV), _laid(v, lv), _laid(vp, lvp)[0], None, _ints([60, 31]))
        modules.get("prefix", "cache").forward(*args)
        _within(o, want, tol)


def test_caches_past_32_bits():
    """Sequences that lie more than 2^32 bytes apart."""
    B, Hq, Hkv, D, M, S, far = 2, 4, 1, 64, 1, 200, (1 << 31) + 4096
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    g = _gen(12)
    q, k, v = (torch.randn(B, h, s, D, generator=g).half() for h, s in ((Hq, M), (Hkv, S), (Hkv, S)))
    new = [torch.randn(B, h, M, D, generator=g).half() for h in (Hq, Hkv, Hkv)]
    room = [torch.empty(far + S * D, dtype=torch.float16, device=DEV) for _ in range(2)]
    dk, dv = (r.as_strided((B, Hkv, S, D), (far, S * D, D, 1)) for r in room)
    dk.copy_(k); dv.copy_(v)
    inv = 100.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    lengths, counts = [200, 150], [1, 1]
    qo = torch.zeros_like(q, device=DEV)
    modules.get("rope", "cache").forward(new[1].to(DEV), dk, new[0].to(DEV), qo, new[2].to(DEV), dv, _ints(counts), None, None, inv.to(DEV), _ints(lengths), None)
    outs, tols = ref.rope(*new, torch.zeros_like(q), k, v, inv, lengths, counts)
    for got, want, tol in zip((qo, dk, dv), outs, tols):
        _within(got, want, tol)
    k, v, q = dk.cpu(), dv.cpu(), qo.cpu()
    o = torch.zeros_like(qo)
    modules.get("prefix", "cache").forward(dk, dk[0, :, :10], o, qo, dv, dv[0, :, :10], _ints(counts), _ints(lengths))
    _within(o, *ref.prefix_attention(q, k, v, k[0, :, :10], v[0, :, :10], torch.zeros_like(q), D ** -0.5, True, lengths, counts))
    bnd, sel = torch.zeros(B, Hkv, 7, 2, D, dtype=torch.float16, device=DEV), torch.zeros(B, Hkv, M, 3, dtype=torch.int32, device=DEV)
    modules.get("bounds", "cache", block=32).forward(dk, bnd, None, _ints(lengths))
    assert torch.equal(bnd.cpu(), ref.bounds(k, torch.zeros(bnd.shape).half(), 32, lengths, [S] * B))
    modules.get("sparse", "cache", block=32, top=3).forward(dk, o, qo, dv, bnd, _ints(counts), _ints(lengths), sel)
    want = ref.select(q, bnd.cpu(), torch.zeros(sel.shape, dtype=torch.int32), 32, 3, 0, 1, 4, lengths, counts, S)
    assert torch.equal(sel.cpu(), want)
    _within(o, *ref.sparse_attention(q, k, v, torch.zeros_like(q), want, 32, D ** -0.5, lengths, counts))


@pytest.mark.parametrize("case", [(2, 64, 4, 300, 280), (1, 128, 4, 300, 280), (2, 64, 1, 1500, 280), (1, 128, 40, 290, 300), (2, 64, 40, 0, 290)], ids=lambda c: "B%dD%dM%dP%dS%d" % c)
def test_rows_far_apart(case):
    """The largest pitch of a token: the keys of one sequence, and those of a prefix, reach past 2^32 bytes."""
    B, D, M, P, S = case
    Hq, Hkv, far = 4, 1, 1 << 23
    rows = P + B * S
    if torch.cuda.mem_get_info()[0] < 2 * rows * far + (4 << 30):
        pytest.skip("needs %d GB" % (2 * rows * far + (4 << 30) >> 30))
    g = _gen(13)
    q = torch.randn(B, Hq, M, D, generator=g).half()
    kv = torch.randn(rows, 2 * D, generator=g).half()
    room = torch.empty(rows * far, dtype=torch.float16, device=DEV).view(rows, far)
    room[:, :2 * D] = kv.to(DEV)
    lengths, counts = [S - 7 * b for b in range(B)], [M] * B

    def parts(x):
        own = x[P:, :].view(B, S, 1, x.shape[1]).permute(0, 2, 1, 3)
        return own[..., :D], own[..., D:2 * D], x[None, :P, :D], x[None, :P, D:2 * D]
    k, v, kp, vp = parts(kv)
    dk, dv, dkp, dvp = parts(room)
    o = torch.zeros(B, Hq, M, D, dtype=torch.float16, device=DEV)
    modules.get("prefix", "cache").forward(dk, dkp, o, q.to(DEV), dv, dvp, _ints(counts), _ints(lengths))
    _within(o, *ref.prefix_attention(q, k, v, kp, vp, torch.zeros_like(q), D ** -0.5, True, lengths, counts))
    nb = (S + 31) // 32
    bnd, sel = torch.zeros(B, Hkv, nb, 2, D, dtype=torch.float16, device=DEV), torch.zeros(B, Hkv, M, 3, dtype=torch.int32, device=DEV)
    modules.get("bounds", "cache", block=32).forward(dk, bnd, None, _ints(lengths))
    assert torch.equal(bnd.cpu(), ref.bounds(k, torch.zeros(bnd.shape).half(), 32, lengths, [S] * B))
    modules.get("sparse", "cache", block=32, top=3).forward(dk, o, q.to(DEV), dv, bnd, _ints(counts), _ints(lengths), sel)
    want = ref.select(q, bnd.cpu(), torch.zeros(sel.shape, dtype=torch.int32), 32, 3, 0, 1, 4, lengths, counts, S)
    assert torch.equal(sel.cpu(), want)
    _within(o, *ref.sparse_attention(q, k, v, torch.zeros_like(q), want, 32, D ** -0.5, lengths, counts))


# ------------------------------------------------------------------------------------------------ together
def _loop(kind, prenorm=False):
    B, Hq, Hkv, D, N, S, P = 3, 8, 2, 64, 192, 500, 90 if kind == "prefix" else 0
    g = _gen(13)
    w = lambda *s: (torch.randn(*s, generator=g) * N ** -0.5).half().to(DEV)
    t = dict(WK=w(N, Hkv * D), WQ=w(N, Hq * D), WV=w(N, Hkv * D), gamma_q=(1 + 0.1 * torch.randn(D, generator=g)).half().to(DEV),
             gamma_k=(1 + 0.1 * torch.randn(D, generator=g)).half().to(DEV), inv_freq=(100.0 ** (-torch.arange(16, dtype=torch.float64) / 16)).to(DEV), positions=None,
             K_cache=torch.zeros(B, Hkv, S, D, dtype=torch.float16, device=DEV), V_cache=torch.zeros(B, Hkv, S, D, dtype=torch.float16, device=DEV))
    if kind == "prefix":
        t.update(K_prefix=torch.randn(Hkv, P, D, generator=g).half().to(DEV), V_prefix=torch.randn(Hkv, P, D, generator=g).half().to(DEV))
        step = modules.get("prenorm" if prenorm else "prefix", "cache16", head_dim=D, qk_norm=True)
    else:
        t.update(bounds=torch.zeros(B, Hkv, -(-S // 32), 2, D, dtype=torch.float16, device=DEV))
        step = modules.get("sparse", "cache16", head_dim=D, qk_norm=True, block=32, top=5, sink=1, recent=2, norm=prenorm)
    return step, t, g, (B, Hq, Hkv, D, N, S)


def _feed(t, g, dims, lengths, counts, M, top=5):
    B, Hq, Hkv, D, N, S = dims
    t.update(X=torch.randn(B, M, N, generator=g).half().to(DEV), O2=torch.zeros(B, M, Hq * D, dtype=torch.float16, device=DEV), lengths=_ints(lengths), counts=_ints(counts),
             selected=torch.full((B, Hkv, M, top), -7, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("kind", ["prefix", "sparse"])
@pytest.mark.parametrize("prenorm", [False, True])
def test_a_serving_loop(kind, prenorm):
    """Prompts, a chunk, single tokens: each step's caches are the last one's with its own tokens behind them, and its outputs are the definition's on them."""
    step, t, g, dims = _loop(kind, prenorm)
    B, Hq, Hkv, D, N, S = dims
    lengths = [0] * B
    for M, counts in ((140, [140, 33, 1]), (17, [17, 0, 17]), (1, [1, 1, 1]), (1, [1, 0, 1]), (4, [2, 4, 3])):
        lengths = [n + c for n, c in zip(lengths, counts)]
        _feed(t, g, dims, lengths, counts, M)
        before = [t[n].cpu() for n in ("K_cache", "V_cache")] + [t["bounds"].cpu() if kind == "sparse" else None]
        step.forward(*[t[n] for n in step.TENSOR_PARAMS])
        # the projection, as the library makes it by itself
        x, qkv = t["X"].view(B * M, N), [torch.zeros(B, M, h, D, dtype=torch.float16, device=DEV) for h in (Hq, Hkv, Hkv)]
        ops.prenorm_qkv(x, None, t["WQ"], t["WK"], t["WV"], *(y.view(B * M, -1, D).permute(1, 0, 2) for y in qkv), 0.0, prenorm)
        q, k, v = (y.permute(0, 2, 1, 3).cpu() for y in qkv)
        outs, tols = ref.rope(q, k, v, q, before[0], before[1], t["inv_freq"].cpu(), lengths, counts, None, t["gamma_q"].cpu(), t["gamma_k"].cpu(), True)
        for n, want, tol in zip(("K_cache", "V_cache"), outs[1:], tols[1:]):
            _within(t[n], want, tol, n)
        # (the queries that the step had: the operator's own)
        qr = torch.zeros_like(qkv[0]).permute(0, 2, 1, 3)
        scratch = [y.clone() for y in (t["K_cache"], t["V_cache"])]
        ops.cache_rope_append(*(y.permute(0, 2, 1, 3) for y in qkv), qr, *scratch, t["inv_freq"], t["lengths"], t["counts"], None, t["gamma_q"], t["gamma_k"], True)
        qr, kc, vc = qr.cpu(), t["K_cache"].cpu(), t["V_cache"].cpu()
        o = t["O2"].view(B, M, Hq, D).permute(0, 2, 1, 3)
        if kind == "prefix":
            _within(o, *ref.prefix_attention(qr, kc, vc, t["K_prefix"].cpu(), t["V_prefix"].cpu(), torch.zeros_like(qr), D ** -0.5, True, lengths, counts))
        else:
            bnd = ref.bounds(kc, before[2], 32, lengths, counts)
            assert torch.equal(t["bounds"].cpu(), bnd)
            sel = ref.select(qr, bnd, torch.full((B, Hkv, M, 5), -7, dtype=torch.int32), 32, 5, 1, 2, Hq // Hkv, lengths, counts, S)
            assert torch.equal(t["selected"].cpu(), sel)
            _within(o, *ref.sparse_attention(qr, kc, vc, torch.zeros_like(qr), sel, 32, D ** -0.5, lengths, counts))


@pytest.mark.parametrize("kind", ["prefix", "sparse"])
def test_a_captured_step_on_caches_that_grow(kind):
    """One token a sequence, captured once and replayed on longer and longer caches, with eager work in between: bit for bit what the eager step leaves."""
    runs = []
    for captured in (False, True):
        step, t, g, dims = _loop(kind)
        _feed(t, g, dims, [150, 40, 7], [150, 40, 7], 150)
        step.forward(*[t[n] for n in step.TENSOR_PARAMS])
        _feed(t, g, dims, [151, 41, 8], [1, 1, 1], 1)
        side, got = torch.cuda.Stream(), []
        step.forward(*[t[n] for n in step.TENSOR_PARAMS])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        if captured:
            with torch.cuda.graph(graph, stream=side):
                step.forward(*[t[n] for n in step.TENSOR_PARAMS])
        for i in range(5):
            t["lengths"] += torch.tensor([1, 1, i % 2], dtype=torch.int32, device=DEV)
            t["counts"].copy_(torch.tensor([1, 1, i % 2]))
            t["X"].copy_(torch.randn(t["X"].shape, generator=g))
            t["O2"].zero_()
            graph.replay() if captured else step.forward(*[t[n] for n in step.TENSOR_PARAMS])
            torch.cuda.synchronize()
            got += [t[n].clone() for n in ("O2", "K_cache", "V_cache") + (("bounds", "selected") if kind == "sparse" else ())]
        runs.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_on_a_stream_of_its_own():
    case = PATHS[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        test_prefix_attention(case, "head")
        test_sparse_attention(SPARSES[1], "token")
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_on_another_device_than_the_current_one():
    B, Hq, Hkv, D, M, S, P = 2, 4, 2, 64, 1, 60, 45
    g = _gen(14)
    q, k, v = (torch.randn(B, h, s, D, generator=g).half() for h, s in ((Hq, M), (Hkv, S), (Hkv, S)))
    with torch.cuda.device(0):
        args = [x.to("cuda:1") for x in (k, k[0], torch.zeros_like(q), q, v, v[0])]
        modules.get("prefix", "cache").forward(*args, None, None)
        torch.cuda.synchronize("cuda:1")
    _within(args[2], *ref.prefix_attention(q, k, v, k[0], v[0], torch.zeros_like(q), D ** -0.5, True, [S] * B, [M] * B))


def test_steps_and_calls_of_nothing():
    for kind in ("prefix", "sparse"):
        step, t, g, dims = _loop(kind)
        B, Hq, Hkv, D, N, S = dims
        _feed(t, g, dims, [5, 0, 1], [0, 0, 0], 0)
        step.forward(*[t[n] for n in step.TENSOR_PARAMS])
        _feed(t, g, dims, [5, 0, 1], [0, 0, 0], 2)
        t["O2"].fill_(3.0)
        step.forward(*[t[n] for n in step.TENSOR_PARAMS])
        assert (t["O2"] == 3.0).all() and (t["selected"] == -7).all() and not t["K_cache"].any()


def test_first_call_inside_a_capture_is_refused():
    q = torch.zeros(1, 4, 1, 64, dtype=torch.float16, device=DEV)
    k = torch.zeros(1, 2, 4000, 64, dtype=torch.float16, device=DEV)
    att = modules.get("prefix", "cache")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side), pytest.raises(RuntimeError, match="eagerly"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            att.forward(k, k[0], q, q.clone(), k, k[0], None, None)


def test_refusals():
    half = lambda *s: torch.zeros(*s, dtype=torch.float16, device=DEV)
    q, o, k, v = half(1, 4, 2, 64), half(1, 4, 2, 64), half(1, 2, 64, 64), half(1, 2, 64, 64)
    n1 = torch.zeros(2, dtype=torch.int32, device=DEV)

    def tried(fn, good):
        fn(**good)

        def bad(error=ValueError, **kw):
            with pytest.raises(error):
                fn(**{**good, **kw})
        return bad
    inv = torch.zeros(32, dtype=torch.float64, device=DEV)
    new = half(1, 2, 2, 64)
    bad = tried(ops.cache_rope_append, dict(q=q, k=new, v=new.clone(), q_out=o, k_cache=k, v_cache=v, inv_freq=inv))
    bad(q=q.float()); bad(q_out=o[:, :2]); bad(k=new[:, :1]); bad(v=new[:, :, :1]); bad(k_cache=k[..., :32]); bad(inv_freq=inv.float()); bad(inv_freq=inv[:30]); bad(inv_freq=inv.cpu())
    bad(lengths=n1); bad(counts=n1[:1].long()); bad(sections=[16, 15]); bad(sections=[]); bad(sections=[8] * 5); bad(sections=[16, 16]); bad(gamma_q=half(64)); bad(q=q.cpu())
    bad(positions=torch.zeros(1, 1, 3, dtype=torch.int32, device=DEV)); bad(norm=True, gamma_k=half(32)); bad(TypeError, sections=3); bad(_lib.TrnError, norm=True, eps=-1.0)
    bad(_lib.TrnError, v_cache=k); bad(_lib.TrnError, q=half(1, 4, 2, 72)[..., 4:68])
    bad = tried(ops.cache_prefix_attention, dict(q=q, k=k, v=v, k_prefix=k[0], v_prefix=v[0], o=o))
    bad(q=q.float()); bad(o=o[:, :2]); bad(q=q[:, :3], o=o[:, :3]); bad(k_prefix=k); bad(v_prefix=v[0, :, :3]); bad(k_prefix=k[0, :1]); bad(v=v[:, :, :3]); bad(lengths=n1); bad(q=q.cpu())
    bad(_lib.TrnError, scale=0.0); bad(_lib.TrnError, o=q); bad(workspace=torch.zeros(4, device=DEV))
    big = half(1, 2, 8000, 64)
    bad(_lib.TrnError, k=big, v=big)                                           # shares without a workspace
    bnd, sel = half(1, 2, 1, 2, 64), torch.zeros(1, 2, 2, 3, dtype=torch.int32, device=DEV)
    bad = tried(ops.cache_bounds, dict(k=k, bounds=bnd))
    bad(block=48); bad(block=32); bad(bounds=bnd.float()); bad(bounds=bnd[0]); bad(k=k[0]); bad(tokens=-1); bad(counts=n1)
    ws = torch.zeros(1 << 20, dtype=torch.uint8, device=DEV)
    bad = tried(ops.cache_sparse_attention, dict(q=q, k=k, v=v, bounds=bnd, o=o, selected=sel, top=3, workspace=ws))
    bad(top=2); bad(top=3, recent=0); bad(sink=3); bad(selected=sel.long()); bad(selected=sel[..., :2]); bad(bounds=half(1, 2, 2, 2, 64)); bad(block=96)
    bad(_lib.TrnError, block=32, bounds=half(1, 2, 2, 2, 64), selected=sel[..., :1].contiguous(), top=1, workspace=None)
    bad(_lib.TrnError, scale=-1.0); bad(v=v.float()); bad(_lib.TrnError, q=half(1, 4, 2, 72)[..., 4:68])
    step = modules.get("prefix", "cache16", head_dim=64)
    with pytest.raises(ValueError):
        step.forward(k, k[0], half(1, 2, 128), v, v[0], half(96, 128), half(96, 256), half(96, 128), half(1, 2, 96), None, None, None, None, None, None)
