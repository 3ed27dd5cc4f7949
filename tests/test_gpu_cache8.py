"""8-bit caches on the GPU: the quantising append, attention over them and the key weights, against the definitions in 64 bits.  Codes and scales are
held to equality; outputs to the bounds that oracle/cache8.py derives."""
import math

import pytest
import torch

from oracle import cache8 as ref
from triton_amd import _lib, modules, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
SPOIL = 0x7f          # a NaN code: what lies behind a sequence's end must not matter


def _cpu(t):
    return t.detach().cpu()


def _cache(B, H, S, D, block, seed, lengths, layout="head", spread=1.0, spoil=True):
    """Codes, scales and their CPU copies; everything behind a sequence's keys is NaN."""
    g = torch.Generator().manual_seed(seed)
    blocks = -(-S // block)
    out = []
    for _ in range(2):
        codes = ref.encode((torch.randn(B, H, S, D, generator=g) * 100.0).clamp(-448, 448))
        scale = torch.exp2(torch.randint(-3, 4, (B, H, blocks), generator=g).float() * spread - 6.0)
        if spoil:
            for b, n in enumerate(lengths):
                codes[b, :, n:] = SPOIL
                scale[b, :, -(-n // block):] = math.nan
        if layout == "token":          # [B, S, H, D] memory
            dev = torch.empty(B, S, H, D, dtype=torch.uint8, device=DEV).permute(0, 2, 1, 3)
        elif layout == "padded":       # rows further apart than they are long
            dev = torch.full((B, H, S, D + 32), SPOIL, dtype=torch.uint8, device=DEV)[..., 16:16 + D]
        else:
            dev = torch.empty(B, H, S, D, dtype=torch.uint8, device=DEV)
        dev.copy_(codes)
        sdev = scale.to(DEV) if layout == "head" else torch.zeros(B, H, blocks + 3, device=DEV)[..., :blocks].copy_(scale)
        out += [codes, scale, dev, sdev]
    return out


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


APPENDS = [
    # B, H, D, new, capacity, block, keys of each sequence with the new ones, new tokens of each
    (1, 8, 128, 1, 64, 64, [1], [1]),                            # the first token
    (2, 2, 64, 1, 100, 32, [33, 64], [1, 1]),                    # one that opens a block, one that fills it
    (3, 3, 128, 5, 300, 64, [62, 66, 300], [5, 3, 5]),           # inside a block, across a border, up to the capacity's end
    (2, 1, 64, 40, 129, 128, [40, 129], [40, 40]),
    (2, 2, 128, 300, 512, 32, [300, 411], [300, 217]),
    (4, 2, 64, 7, 65, 64, [0, 3, 65, 7], [0, 7, 0, 2]),          # no token; more new tokens than keys; nothing new
    (1, 71, 64, 16, 80, 64, [79], [16]),
]


@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"B{c[0]}H{c[1]}D{c[2]}M{c[3]}S{c[4]}b{c[5]}")
@pytest.mark.parametrize("layout", ["head", "token", "padded"])
@pytest.mark.parametrize("size", [1.0, 3e-5, 4000.0])
def test_append(case, layout, size):
    B, H, D, M, S, block, lengths, counts = case
    k8, ks, dk8, dks, v8, vs, dv8, dvs = _cache(B, H, S, D, block, 1, [max(0, n - c) for n, c in zip(lengths, counts)], layout)
    g = torch.Generator().manual_seed(7)
    rows = [(torch.randn(B, H, M, D, generator=g) * size * torch.exp(torch.randn(B, H, M, 1, generator=g))).half() for _ in range(2)]
    dev = [torch.empty(B, M, H, D, dtype=torch.float16, device=DEV).permute(0, 2, 1, 3).copy_(r) if layout == "token" else r.to(DEV) for r in rows]
    ops.cache8_append(*dev, dk8, dv8, dks, dvs, lengths=_ints(lengths), counts=_ints(counts), block=block)
    for x, codes, scale, dc, ds in ((rows[0], k8, ks, dk8, dks), (rows[1], v8, vs, dv8, dvs)):
        want, ws = ref.append(x, codes, scale, lengths, counts, block)
        assert torch.equal(torch.nan_to_num(_cpu(ds), nan=-1.0), torch.nan_to_num(ws, nan=-1.0))
        assert torch.equal(_cpu(dc), want)


def test_append_without_lengths_takes_the_last_rows_and_float8_tensors():
    B, H, D, M, S, block = 2, 2, 128, 9, 70, 32
    k8, ks, dk8, dks, v8, vs, dv8, dvs = _cache(B, H, S, D, block, 3, [S, S])
    g = torch.Generator().manual_seed(8)
    rows = [torch.randn(B, H, M, D, generator=g).half() for _ in range(2)]
    ops.cache8_append(rows[0].to(DEV), rows[1].to(DEV), dk8.view(torch.float8_e4m3fn), dv8.view(torch.float8_e4m3fn), dks, dvs, block=block)
    for x, codes, scale, dc, ds in ((rows[0], k8, ks, dk8, dks), (rows[1], v8, vs, dv8, dvs)):
        want, ws = ref.append(x, codes, scale, [S] * B, [M] * B, block)
        assert torch.equal(_cpu(ds), ws) and torch.equal(_cpu(dc), want)


def test_append_of_what_is_not_finite_and_of_the_type_s_ends():
    B, H, D, M, S, block = 1, 1, 64, 6, 64, 64
    x = torch.zeros(B, H, M, D, dtype=torch.float16)
    x[0, 0, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 1.0]).half()
    x[0, 0, 1, :4] = torch.tensor([65504.0, -65504.0, 2.0 ** -24, -(2.0 ** -24)]).half()
    x[0, 0, 2, :4] = torch.tensor([448.0, 464.0, 480.0, -0.0]).half()
    for rows in ([0], [1], [2], [3], [0, 1], [2, 3], list(range(6))):
        part = x[:, :, rows]
        k8, ks, dk8, dks, v8, vs, dv8, dvs = _cache(B, H, S, D, block, 4, [0])
        ops.cache8_append(part.to(DEV), part.to(DEV), dk8, dv8, dks, dvs, lengths=_ints([len(rows)]))
        want, ws = ref.append(part, k8, ks, [len(rows)], [len(rows)], block)
        assert torch.equal(_cpu(dks), ws)
        got = _cpu(dk8)
        nan = torch.isnan(ref.decode(want))
        assert torch.equal(torch.isnan(ref.decode(got)), nan) and torch.equal(got[~nan], want[~nan])


def test_appends_one_by_one_grow_the_scale():
    """A block filled token by token, each larger than all before: codes are what repeated rescaling of the definition gives."""
    B, H, D, S, block = 1, 2, 128, 64, 64
    k8, ks, dk8, dks, v8, vs, dv8, dvs = _cache(B, H, S, D, block, 5, [0])
    g = torch.Generator().manual_seed(9)
    for n in range(1, 65):
        x = (torch.randn(B, H, 1, D, generator=g) * 1.2 ** n * 1e-3).half()
        ops.cache8_append(x.to(DEV), x.to(DEV), dk8, dv8, dks, dvs, lengths=_ints([n]))
        k8, ks = ref.append(x, k8, ks, [n], [1], block)
    assert torch.equal(_cpu(dk8), k8) and torch.equal(_cpu(dks), ks)


ATTNS = [
    # B, Hq, Hkv, D, queries, capacity, block, lengths, counts, causal
    (1, 32, 8, 128, 1, 70, 64, [70], [1], True),
    (2, 4, 1, 64, 1, 40, 32, [1, 33], [1, 1], True),             # one key; a tile and one more
    (3, 2, 2, 128, 3, 100, 32, [0, 2, 100], [3, 3, 2], True),    # no key at all; fewer keys than queries; a padded query
    (2, 8, 2, 128, 9, 300, 64, [300, 129], [9, 1], True),        # 36 rows: two tiles
    (1, 71, 1, 64, 5, 500, 128, [437], [5], True),
    (2, 6, 2, 64, 4, 160, 64, [160, 31], [4, 0], False),         # all keys for all; no query
    (1, 2, 1, 128, 70, 130, 64, [130], [70], True),              # a prompt's diagonal
    (1, 1, 1, 64, 33, 33, 32, [33], [33], True),
    (1, 8, 8, 128, 1, 2500, 64, [2431], [1], True),              # split over workgroups
    (2, 16, 4, 64, 2, 3000, 128, [3000, 1777], [2, 2], False),
    (1, 4, 2, 128, 1, 1100, 32, [1100], [1], True),
    (2, 8, 2, 128, 150, 400, 64, [400, 260], [150, 101], True),  # many rows: the weights in chunks of row tiles
    (1, 71, 1, 64, 9, 700, 32, [611], [9], False),
    (1, 32, 2, 64, 3, 2600, 64, [2555], [3], True),              # shares, and the weights of many rows behind them
    (2, 12, 2, 128, 4, 1500, 32, [1500, 901], [4, 2], True),
]


def _check(got, want, tol, name):
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - want).abs() / tol.clamp(min=1e-30)).max()):.3g} of the bound"


def _attend(case, layout="head", spread=1.0, seed=11, size=1.0, spoil=True, edit=None):
    B, Hq, Hkv, D, M, S, block, lengths, counts, causal = case
    k8, ks, dk8, dks, v8, vs, dv8, dvs = _cache(B, Hkv, S, D, block, seed, lengths, layout, spread, spoil)
    if edit:
        edit(k8, ks, v8, vs)
        dk8.copy_(k8), dks.copy_(ks), dv8.copy_(v8), dvs.copy_(vs)
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn(B, Hq, M, D, generator=g) * size).half()
    if layout == "token":
        dq = torch.empty(B, M, Hq, D, dtype=torch.float16, device=DEV).permute(0, 2, 1, 3).copy_(q)
        o = torch.full((B, M, Hq, D), 7.0, dtype=torch.float16, device=DEV).permute(0, 2, 1, 3)
    else:
        dq, o = q.to(DEV), torch.full((B, Hq, M, D), 7.0, dtype=torch.float16, device=DEV)
    lse = torch.full((B, Hq, M), 7.0, device=DEV)
    w_in = torch.rand(B, Hkv, S, generator=g)
    w_out = torch.full((B, Hkv, S), 7.0, device=DEV)
    ws = torch.full((ops.cache8_attention_workspace_bytes(dq, dk8, True),), 0xff, dtype=torch.uint8, device=DEV)
    ops.cache8_attention(dq, dk8, dv8, dks, dvs, o, None, causal, _ints(lengths), _ints(counts), lse, w_in.to(DEV), w_out, block, ws)
    want, wlse, w, tol, wtol, ltol = ref.attention(q, k8, v8, ks, vs, D ** -0.5, causal, lengths, counts, block)
    there = torch.arange(M)[None, None, :] < torch.tensor([min(c, M) for c in counts])[:, None, None]
    there = there.expand(B, Hq, M)
    return dict(o=_cpu(o), lse=_cpu(lse), w=_cpu(w_out), w_in=w_in, want=want, wlse=wlse, ww=w, tol=tol, wtol=wtol, ltol=ltol, there=there, q=dq, k8=dk8, v8=dv8, ks=dks, vs=dvs, ws=ws)


def _hold(r, lengths):
    there = r["there"]
    assert torch.equal(r["o"][~there], torch.full_like(r["o"][~there], 7.0)), "outputs of queries that are not there"
    assert (r["lse"][~there] == 7.0).all()
    nan = torch.isnan(r["want"]) & there[..., None]
    assert torch.equal(torch.isnan(r["o"]) & there[..., None], nan)
    fine = there[..., None].expand_as(nan) & ~nan
    _check(r["o"][fine], r["want"][fine], r["tol"][fine], "o")
    empty = there & torch.isinf(r["wlse"])
    assert (r["lse"][empty] == -math.inf).all() and (r["o"][empty] == 0).all()
    some = there & torch.isfinite(r["wlse"])
    _check(r["lse"][some], r["wlse"][some], r["ltol"][some], "lse")
    for b, n in enumerate(lengths):
        assert (r["w"][b, :, n:] == 7.0).all(), "weights behind the last key"
        total = r["w_in"][b, :, :n].double() + r["ww"][b, :, :n]
        ok = torch.isfinite(total)
        _check(r["w"][b, :, :n][ok], total[ok], (r["wtol"][b, :, :n] + 2.0 ** -23 * total.abs())[ok], "weights")


@pytest.mark.parametrize("case", ATTNS, ids=lambda c: f"B{c[0]}q{c[1]}kv{c[2]}D{c[3]}M{c[4]}S{c[5]}b{c[6]}c{int(c[9])}")
@pytest.mark.parametrize("layout", ["head", "token", "padded"])
def test_attention_and_weights(case, layout):
    _hold(_attend(case, layout), case[7])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads, causal", [((8, 8, 40), True), ((20, 16, 16), True), ((33, 16, 16), True), ((33, 16, 16), False)], ids=["two waves", "two, fewer rows", "one wave", "one wave, all keys"])
def test_row_tiles_of_fewer_waves(heads, causal, D):
    """So many rows that two waves share a row tile's keys, or that one has them: most of the batch is padding, for the oracle's sake."""
    B, Hkv, Hq = heads
    M, S, block = (73, 90, 64) if Hq > Hkv else (150, 170, 32)
    lengths = [S, 33, 0, 1, 64, 65, 32] + [40 + b for b in range(B - 7)]
    counts = [M, 33, 2, 1, 5, 0, 70] + [1 + b % 3 for b in range(B - 7)]
    case = (B, Hq, Hkv, D, M, S, block, lengths, counts, causal)
    _hold(_attend(case, "token"), lengths)

    def edit(k8, ks, v8, vs):
        v8[:, :, 20] = 0x7f
    _hold(_attend(case, edit=edit, spoil=False), lengths)


@pytest.mark.parametrize("B, Hq, Hkv, D, M", [(96, 32, 8, 128, 8), (320, 32, 8, 128, 8), (48, 16, 16, 64, 20)], ids=["768 heads", "2560", "768 of 64"])
def test_one_row_tile_of_very_many_heads(B, Hq, Hkv, D, M):
    """Heads enough for row tiles of fewer waves, each of which has a single tile of 17 to 32 rows: its four waves have its keys, and none behind them."""
    S, block = 75, 32
    lengths = [1 + 37 * b % S for b in range(B)]
    lengths[1], lengths[-1] = 0, S
    counts = [M if b in (0, 5, B - 1) else int(b % 4 < 2) for b in range(B)]
    _hold(_attend((B, Hq, Hkv, D, M, S, block, lengths, counts, True), "padded"), lengths)


@pytest.mark.parametrize("spread", [0.0, 4.0])
@pytest.mark.parametrize("case", [ATTNS[3], ATTNS[8], ATTNS[6]], ids=["tiles", "split", "prompt"])
def test_scales_that_differ_by_powers_and_by_nothing(case, spread):
    _hold(_attend(case, spread=spread, size=0.3), case[7])


def test_any_scale_and_none():
    """Scales that are no powers of two, and blocks of zeros whose scale is zero (their keys count in the sum)."""
    def edit(k8, ks, v8, vs):
        ks *= 1.37; vs *= 0.77
        ks[:, :, 0] = 0.0
        vs[:, 0, 1] = 0.0
    case = ATTNS[3]
    _hold(_attend(case, edit=edit), case[7])


def test_large_scores_and_a_single_key_that_takes_all():
    case = ATTNS[8]
    r = _attend(case, size=40.0)
    _hold(r, case[7])


FEW = [ATTNS[0], ATTNS[1], ATTNS[4], ATTNS[8], ATTNS[9], ATTNS[10], ATTNS[14], (1, 8, 2, 128, 1, 900, 64, [900], [1], True), (96, 8, 2, 128, 8, 75, 32, [1 + b % 75 for b in range(96)], [int(b % 8 == 0) * 8 for b in range(96)], True)]


@pytest.mark.parametrize("size", [0.05, 1.0, 8.0, 40.0])
@pytest.mark.parametrize("case", FEW, ids=lambda c: f"B{c[0]}q{c[1]}kv{c[2]}D{c[3]}M{c[4]}S{c[5]}")
def test_weights_of_few_rows_are_not_rounded(case, size):
    """Where all heads have up to 512 rows, or each one row tile, the weight of a key is two numbers of fp16: what the first leaves over, at most 2^-11 of it, is rounded to 2^-11 of
    that, or to 2^-25 of the largest weight.  So of the oracle's bound 2^-22 is left of the term for a weight's rounding, where it has 2^-11; of the output's own
    rounding half a step, 2^-11 of it, or 2^-25."""
    r = _attend(case, size=size)
    there = r["there"][..., None].expand_as(r["want"])
    B, Hq, Hkv, D, M, S, block, lengths, counts, causal = case
    q, k8, v8, ks, vs = (_cpu(r[n]) for n in ("q", "k8", "v8", "ks", "vs"))
    _, _, _, tol, _, _ = ref.attention(q, k8, v8, ks, vs, D ** -0.5, causal, lengths, counts, block)
    mass = ref.attention(q, k8, v8 & 0x7f, ks, vs, D ** -0.5, causal, lengths, counts, block)[0]       # sum of p |v|
    fine = tol - (2.0 ** -11 - 2.0 ** -22) * mass
    assert (fine[there] >= 0).all()       # (zero for a query that sees no key: exactly zeros)
    _check(r["o"][there], r["want"][there], fine[there], "o")


@pytest.mark.parametrize("case", [ATTNS[6], ATTNS[7], ATTNS[3]], ids=["prompt", "tile", "chunk"])
def test_nan_of_a_key_reaches_only_the_queries_that_see_it(case):
    def edit(k8, ks, v8, vs):
        n = case[7][0]
        v8[0, 0, n - 2, 5] = 0x7f
        v8[0, 0, n - 20, 40] = 0xff
    r = _attend(case, edit=edit)
    assert torch.isnan(r["want"]).any() and torch.isfinite(r["want"][r["there"]]).any()
    _hold(r, case[7])


def test_nan_in_a_key_code():
    case = ATTNS[6]
    def edit(k8, ks, v8, vs):
        k8[0, 0, case[7][0] - 30, 3] = 0x7f
    r = _attend(case, edit=edit)
    nan = torch.isnan(r["want"])
    assert nan.any() and not nan.all()
    there = r["there"][..., None].expand_as(nan)
    assert torch.equal(torch.isnan(r["o"])[there], nan[there])
    _check(r["o"][there & ~nan], r["want"][there & ~nan], r["tol"][there & ~nan], "o")


def test_without_a_workspace_lse_or_weights():
    case = ATTNS[8]
    r = _attend(case)
    B, Hq, Hkv, D, M, S, block, lengths, counts, causal = case
    o = torch.zeros(B, Hq, M, D, dtype=torch.float16, device=DEV)
    ops.cache8_attention(r["q"], r["k8"], r["v8"], r["ks"], r["vs"], o, None, causal, _ints(lengths), _ints(counts), block=block)
    _check(_cpu(o), r["want"], r["tol"], "o")


def test_weights_add_up_in_place():
    case = ATTNS[3]
    B, Hq, Hkv, D, M, S, block, lengths, counts, causal = case
    r = _attend(case)
    w = r["w_in"].to(DEV)
    for _ in range(2):
        ops.cache8_attention(r["q"], r["k8"], r["v8"], r["ks"], r["vs"], torch.empty_like(r["q"]), None, causal, _ints(lengths), _ints(counts), None, w, w, block, r["ws"])
    for b, n in enumerate(lengths):
        total = r["w_in"][b, :, :n].double() + 2 * r["ww"][b, :, :n]
        _check(_cpu(w)[b, :, :n], total, 2 * r["wtol"][b, :, :n] + 2.0 ** -22 * total.abs(), "weights")
        assert torch.equal(_cpu(w)[b, :, n:], r["w_in"][b, :, n:])


def test_a_long_cache_past_two_gigabytes_of_offsets():
    """Rows 64 KB apart: the last of 40000 keys lies 2.6 GB behind the first."""
    B, Hq, Hkv, D, M, S, block, pitch = 1, 2, 1, 64, 1, 40000, 128, 1 << 16
    g = torch.Generator().manual_seed(5)
    store = torch.empty(2, S, pitch, dtype=torch.uint8, device=DEV)
    codes = [ref.encode((torch.randn(1, 1, S, D, generator=g) * 30.0).clamp(-448, 448)) for _ in range(2)]
    dev = []
    for i in range(2):
        t = store[i, :, 32:32 + D][None, None]
        t.copy_(codes[i])
        dev.append(t)
    scale = [torch.full((1, 1, -(-S // block)), 2.0 ** -5) for _ in range(2)]
    q = torch.randn(B, Hq, M, D, generator=g).half()
    o = torch.zeros(B, Hq, M, D, dtype=torch.float16, device=DEV)
    ws = torch.empty(ops.cache8_attention_workspace_bytes(q, dev[0]), dtype=torch.uint8, device=DEV)
    ops.cache8_attention(q.to(DEV), dev[0], dev[1], scale[0].to(DEV), scale[1].to(DEV), o, block=block, workspace=ws)
    want, _, _, tol, _, _ = ref.attention(q, codes[0], codes[1], scale[0], scale[1], D ** -0.5, True, [S], [1], block)
    _check(_cpu(o), want, tol, "o")


def test_the_same_bits_again():
    case = ATTNS[8]
    a, b = _attend(case), _attend(case)
    assert torch.equal(a["o"], b["o"]) and torch.equal(a["w"], b["w"]) and torch.equal(a["lse"], b["lse"])


def test_captured_and_replayed_on_a_cache_that_grows():
    """A step of append and attention with weights, captured once and replayed while `lengths` grow on the device."""
    B, Hq, Hkv, D, S, block = 2, 8, 2, 128, 700, 64
    lengths = [600, 65]
    k8, ks, dk8, dks, v8, vs, dv8, dvs = _cache(B, Hkv, S, D, block, 21, lengths)
    g = torch.Generator().manual_seed(22)
    app, att = modules.get("append8", "cache", block=block), modules.get("weights8", "cache", block=block)
    k, v = (torch.zeros(B, Hkv, 1, D, dtype=torch.float16, device=DEV) for _ in range(2))
    q, o = (torch.zeros(B, Hq, 1, D, dtype=torch.float16, device=DEV) for _ in range(2))
    w = torch.zeros(B, Hkv, S, device=DEV)
    n = _ints(lengths)

    def step():
        n.add_(1)
        app.forward(k, dk8, dks, v, dv8, dvs, None, n)
        att.forward(dk8, dks, o, q, dv8, dvs, None, n, w, w)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        att.forward(dk8, dks, o, q, dv8, dvs, None, n, None, torch.zeros_like(w))      # (its workspace)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        step()
    side.synchronize()
    ww = torch.zeros(B, Hkv, S, dtype=torch.float64)
    slack = torch.zeros(B, Hkv, S, dtype=torch.float64)
    for t in range(6):
        rows = [torch.randn(B, h, 1, D, generator=g).half() for h in (Hkv, Hkv, Hq)]
        for dst, src in zip((k, v, q), rows):
            dst.copy_(src)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        lengths = [x + 1 for x in lengths]
        k8, ks = ref.append(rows[0], k8, ks, lengths, [1, 1], block)
        v8, vs = ref.append(rows[1], v8, vs, lengths, [1, 1], block)
        want, _, got_w, tol, wtol, _ = ref.attention(rows[2], k8, v8, ks, vs, D ** -0.5, True, lengths, [1, 1], block)
        _check(_cpu(o), want, tol, f"o of step {t}")
        ww += got_w
        slack += wtol + 2.0 ** -23 * ww
        _check(_cpu(w), ww, slack, f"weights of step {t}")
        assert torch.equal(_cpu(dk8)[0, :, :lengths[0]], k8[0, :, :lengths[0]])


def test_two_instances_on_two_streams():
    case = ATTNS[8]
    B, Hq, Hkv, D, M, S, block, lengths, counts, causal = case
    rs = [_attend(case, seed=s) for s in (41, 51)]
    outs = [torch.zeros_like(r["q"]) for r in rs]
    ws = [torch.zeros(B, Hkv, S, device=DEV) for _ in rs]
    n = _ints(lengths)
    torch.cuda.synchronize()
    mods, streams = [modules.get("weights8", "cache", block=block) for _ in rs], [torch.cuda.Stream() for _ in rs]
    for _ in range(20):
        for r, o, w, mod, st in zip(rs, outs, ws, mods, streams):
            with torch.cuda.stream(st):
                mod.forward(r["k8"], r["ks"], o, r["q"], r["v8"], r["vs"], None, n, None, w)
    torch.cuda.synchronize()
    for r, o, w in zip(rs, outs, ws):
        _check(_cpu(o), r["want"], r["tol"], "o")
        _check(_cpu(w)[0, :, :lengths[0]], r["ww"][0, :, :lengths[0]], r["wtol"][0, :, :lengths[0]], "weights")


def test_caches_and_batches_of_nothing():
    z = lambda *s, dt=torch.uint8: torch.zeros(*s, dtype=dt, device=DEV)
    q, o, lse = z(1, 4, 2, 64, dt=torch.float16), torch.full((1, 4, 2, 64), 7.0, dtype=torch.float16, device=DEV), z(1, 4, 2, dt=torch.float32)
    k8, s = z(1, 2, 0, 64), z(1, 2, 0, dt=torch.float32)
    ops.cache8_append(q[:, :2], q[:, :2], k8, k8, s, s)
    ops.cache8_attention(q, k8, k8, s, s, o, lse=lse)
    assert (o == 0).all() and (lse == -math.inf).all()
    k8, s = z(0, 2, 64, 64), z(0, 2, 1, dt=torch.float32)
    ops.cache8_append(q[:0, :2], q[:0, :2], k8, k8, s, s)
    ops.cache8_attention(q[:0], k8, k8, s, s, o[:0])


@pytest.mark.parametrize("D", [64, 128])
def test_weights_of_no_queries(D):
    """weights_out is weights, or zeros, up to each sequence's length; a cache without keys has none and takes no workspace."""
    B, Hq, Hkv, S, block, lengths = 3, 4, 2, 700, 64, [700, 0, 301]
    k8, ks, dk8, dks, v8, vs, dv8, dvs = _cache(B, Hkv, S, D, block, 71, lengths)
    q = torch.zeros(B, Hq, 0, D, dtype=torch.float16, device=DEV)
    w = torch.rand(B, Hkv, S, generator=torch.Generator().manual_seed(72))
    mod = modules.get("weights8", "cache", block=block)
    for w_in in (None, w):
        for via in ("ops", "module", "counts"):
            out = torch.full((B, Hkv, S), 7.0, device=DEV)
            given = None if w_in is None else w_in.to(DEV)
            if via == "ops":
                ops.cache8_attention(q, dk8, dv8, dks, dvs, q.clone(), lengths=_ints(lengths), lse=torch.zeros(B, Hq, 0, device=DEV), weights=given, weights_out=out, block=block)
            elif via == "module":
                mod.forward(dk8, dks, q.clone(), q, dv8, dvs, None, _ints(lengths), given, out)
            else:
                some = torch.zeros(B, Hq, 3, D, dtype=torch.float16, device=DEV)
                mod.forward(dk8, dks, some.clone(), some, dv8, dvs, _ints([0] * B), _ints(lengths), given, out)
            for b, n in enumerate(lengths):
                assert torch.equal(_cpu(out)[b, :, :n], torch.zeros(Hkv, n) if w_in is None else w[b, :, :n]) and (out[b, :, n:] == 7.0).all()
    same = w.to(DEV)
    mod.forward(dk8, dks, q.clone(), q, dv8, dvs, None, _ints(lengths), same, same)
    assert torch.equal(_cpu(same), w)
    none = lambda *s, dt=torch.uint8: torch.zeros(*s, dtype=dt, device=DEV)
    some, o = torch.ones(B, Hq, 2, D, dtype=torch.float16, device=DEV), torch.full((B, Hq, 2, D), 7.0, dtype=torch.float16, device=DEV)
    k8, s, w0 = none(B, Hkv, 0, D), none(B, Hkv, 0, dt=torch.float32), none(B, Hkv, 0, dt=torch.float32)
    mod.forward(k8, s, o, some, k8, s, None, None, w0, w0)
    assert (o == 0).all()
    # (the C ABI may be given an address for weights of nothing)
    c = _lib.Cache8()
    c.batch, c.n_kv_heads, c.capacity, c.head_dim, c.block = B, Hkv, 0, D, block
    o.fill_(7.0)
    strides = (Hq * 2 * D, 2 * D, D)
    st = _lib.load().trn_cache8_attn_f16(_lib.C.byref(c), some.data_ptr(), o.data_ptr(), Hq, 2, *strides, *strides, 0.125, 1, None, None, same.data_ptr(), None, 0,
                                         torch.cuda.current_stream().cuda_stream)
    assert st == 0 and (o == 0).all() and torch.equal(_cpu(same), w)


@pytest.mark.parametrize("axis", [1, 2, 3], ids=["by sequence", "by head", "by token"])
def test_keys_and_values_of_one_tensor(axis):
    """Append and attention on caches packed into one tensor, scales too: the bits that tensors of their own give.  One tensor for both is refused."""
    B, Hq, Hkv, D, S, block, lengths, counts = 2, 4, 2, 64, 200, 32, [200, 131], [3, 2]
    g = torch.Generator().manual_seed(81)
    k, v = (torch.randn(B, Hkv, 3, D, generator=g).half().to(DEV) for _ in range(2))
    q = torch.randn(B, Hq, 3, D, generator=g).half().to(DEV)
    codes = [ref.encode((torch.randn(B, Hkv, S, D, generator=g) * 100).clamp(-448, 448)).to(DEV) for _ in range(2)]
    scale = [torch.exp2(torch.randint(-3, 4, (B, Hkv, -(-S // block)), generator=g).float()).to(DEV) for _ in range(2)]
    pack = lambda x, a: torch.stack(x, a).unbind(a)
    packed = [t.transpose(1, 2) for t in pack([c.transpose(1, 2) for c in codes], 2)] if axis == 3 else pack(codes, axis)
    packed_scale = pack(scale, min(axis, 2))
    outs = []
    for (k8, v8), (ks, vs) in ((codes, scale), (packed, packed_scale)):
        ops.cache8_append(k, v, k8, v8, ks, vs, _ints(lengths), _ints(counts), block)
        o = torch.zeros_like(q)
        ops.cache8_attention(q, k8, v8, ks, vs, o, lengths=_ints(lengths), counts=_ints(counts), block=block)
        outs.append(o)
    assert torch.equal(outs[0], outs[1])
    for a, b in zip((*codes, *scale), (*packed, *packed_scale)):
        assert torch.equal(a, b)
    for kw in (dict(v8=codes[0]), dict(v_scale=scale[0])):
        with pytest.raises(_lib.TrnError):
            ops.cache8_append(**{**dict(k=k, v=v, k8=codes[0], v8=codes[1], k_scale=scale[0], v_scale=scale[1], block=block), **kw})


@pytest.mark.parametrize("variant", ["vanilla", "prenorm", "weights"])
def test_the_step_of_projection_append_and_attention(variant):
    """modules.get(.., "cache8"): three steps of a ragged, padded batch, with what its projections leave held to the definitions."""
    B, Hq, Hkv, D, N, S, block, M = 2, 4, 2, 64, 256, 120, 32, 5
    g = torch.Generator().manual_seed(61)
    wq, wk, wv = ((torch.randn(N, h * D, generator=g) * N ** -0.5).half().to(DEV) for h in (Hq, Hkv, Hkv))
    mod = modules.get(variant, "cache8", head_dim=D, block=block)
    k8, v8 = (torch.zeros(B, Hkv, S, D, dtype=torch.uint8) for _ in range(2))
    ks, vs = (torch.zeros(B, Hkv, -(-S // block)) for _ in range(2))
    dk8, dv8, dks, dvs = (t.to(DEV) for t in (k8, v8, ks, vs))
    w, ww, slack = torch.zeros(B, Hkv, S, device=DEV), torch.zeros(B, Hkv, S, dtype=torch.float64), torch.zeros(B, Hkv, S, dtype=torch.float64)
    lengths = [0, 0]
    for counts in ([5, 3], [1, 5], [5, 5]):
        x = torch.randn(B, M, N, generator=g).half().to(DEV)
        o = torch.full((B, M, Hq * D), 7.0, dtype=torch.float16, device=DEV)
        lengths = [n + c for n, c in zip(lengths, counts)]
        extra = (w,) if variant == "weights" else ()
        mod.forward(dk8, dks, o, dv8, dvs, wk, wq, wv, x, _ints(counts), _ints(lengths), *extra)
        q, k, v = (torch.empty(B * M, h * D, dtype=torch.float16, device=DEV) for h in (Hq, Hkv, Hkv))
        ops.prenorm_qkv(x.view(B * M, N), None, wq, wk, wv, *(t.view(B * M, -1, D).permute(1, 0, 2) for t in (q, k, v)), 0.0, variant == "prenorm")
        q, k, v = (_cpu(t).view(B, M, -1, D).permute(0, 2, 1, 3) for t in (q, k, v))
        k8, ks = ref.append(k, k8, ks, lengths, counts, block)
        v8, vs = ref.append(v, v8, vs, lengths, counts, block)
        assert torch.equal(_cpu(dk8), k8) and torch.equal(_cpu(dvs), vs)
        want, _, got, tol, wtol, _ = ref.attention(q, k8, v8, ks, vs, D ** -0.5, True, lengths, counts, block)
        for b, c in enumerate(counts):
            _check(_cpu(o)[b, :c].view(c, Hq, D).permute(1, 0, 2), want[b, :, :c], tol[b, :, :c], "O2")
            assert (_cpu(o)[b, c:] == 7.0).all()
        ww += got
        slack += wtol + 2.0 ** -23 * ww
    if variant == "weights":
        _check(_cpu(w), ww, slack + 1e-30, "weights")


@pytest.mark.parametrize("variant", ["vanilla", "prenorm", "weights"])
@pytest.mark.parametrize("B, M", [(2, 0), (0, 3), (0, 0)])
def test_a_step_of_nothing(B, M, variant):
    """No token, or no sequence: cache, scales and weights stay as they are."""
    Hq, Hkv, D, N, S = 4, 2, 64, 256, 120
    mod = modules.get(variant, "cache8", head_dim=D)
    half = lambda *s: torch.ones(*s, dtype=torch.float16, device=DEV)
    codes = [torch.full((B, Hkv, S, D), 5, dtype=torch.uint8, device=DEV) for _ in range(2)]
    scale = [torch.full((B, Hkv, 2), 0.5, device=DEV) for _ in range(2)]
    w = torch.full((B, Hkv, S), 3.0, device=DEV)
    n = _ints([S] * B)
    for lengths, counts in ((None, None), (n, _ints([0] * B))):
        mod.forward(codes[0], scale[0], half(B, M, Hq * D), codes[1], scale[1], half(N, Hkv * D), half(N, Hq * D), half(N, Hkv * D), half(B, M, N), counts, lengths,
                    *((w,) if variant == "weights" else ()))
    assert all((t == 5).all() for t in codes) and all((t == 0.5).all() for t in scale) and (w == 3.0).all()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_a_step_on_another_device_than_the_current_one():
    B, Hq, Hkv, D, N, S, M = 2, 4, 2, 64, 256, 120, 3
    g = torch.Generator().manual_seed(91)
    half = lambda *s: torch.randn(*s, generator=g).half().to("cuda:1")
    wk, wq, wv, x = half(N, Hkv * D), half(N, Hq * D), half(N, Hkv * D), half(B, M, N)
    outs = []
    for current in (0, 1):
        with torch.cuda.device(current):
            codes = [torch.zeros(B, Hkv, S, D, dtype=torch.uint8, device="cuda:1") for _ in range(2)]
            scale = [torch.zeros(B, Hkv, 2, device="cuda:1") for _ in range(2)]
            o, n = torch.zeros(B, M, Hq * D, dtype=torch.float16, device="cuda:1"), torch.full((B,), M, dtype=torch.int32, device="cuda:1")
            modules.get("vanilla", "cache8", head_dim=D).forward(codes[0], scale[0], o, codes[1], scale[1], wk, wq, wv, x, None, n)
            torch.cuda.synchronize("cuda:1")
            assert torch.cuda.current_device() == current
            outs.append((o, *codes, *scale))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    with pytest.raises(ValueError, match="device of x"):
        modules.get("vanilla", "cache8", head_dim=D).forward(codes[0], scale[0], o, codes[1], scale[1], wk.to("cuda:0"), wq, wv, x, None, n)


def test_first_call_inside_a_capture_is_refused():
    k8, ks, dk8, dks, v8, vs, dv8, dvs = _cache(1, 2, 64, 64, 64, 31, [64])
    q = torch.zeros(1, 2, 1, 64, dtype=torch.float16, device=DEV)
    att = modules.get("weights8", "cache")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side), pytest.raises(RuntimeError, match="eagerly"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            att.forward(dk8, dks, q, q.clone(), dv8, dvs, None, None, None, torch.zeros(1, 2, 64, device=DEV))


def test_refusals():
    k8, ks, dk8, dks, v8, vs, dv8, dvs = _cache(1, 2, 64, 64, 64, 31, [64])
    q = torch.zeros(1, 4, 1, 64, dtype=torch.float16, device=DEV)
    o = torch.zeros_like(q)
    good = dict(q=q, k8=dk8, v8=dv8, k_scale=dks, v_scale=dvs, o=o)
    ops.cache8_attention(**good)

    def bad(error=ValueError, **kw):
        with pytest.raises(error):
            ops.cache8_attention(**{**good, **kw})
    bad(q=q.float()); bad(o=o[:, :2]); bad(q=q[:, :3], o=o[:, :3]); bad(k8=dk8.float()); bad(v8=dv8[:, :, :32]); bad(block=48); bad(block=32)
    bad(k_scale=dks.half()); bad(k_scale=dks[..., :0]); bad(lengths=torch.zeros(1, dtype=torch.int64, device=DEV)); bad(lengths=torch.zeros(2, dtype=torch.int32, device=DEV))
    bad(counts=torch.zeros(1, dtype=torch.int32)); bad(weights=torch.zeros(1, 2, 64, device=DEV)); bad(weights_out=torch.zeros(1, 4, 64, device=DEV))
    bad(lse=torch.zeros(1, 4, 2, device=DEV)); bad(workspace=torch.zeros(4, device=DEV)); bad(q=q.cpu())
    bad(_lib.TrnError, scale=0.0); bad(_lib.TrnError, scale=math.nan); bad(_lib.TrnError, weights_out=torch.zeros(1, 2, 64, device=DEV))
    wide = torch.zeros(1, 4, 1, 72, dtype=torch.float16, device=DEV)[..., 4:68]
    bad(_lib.TrnError, q=wide)
    k = torch.zeros(1, 2, 1, 64, dtype=torch.float16, device=DEV)
    ops.cache8_append(k, k, dk8, dv8, dks, dvs)
    for kw in (dict(k=k.float()), dict(k=k[:, :1]), dict(v=torch.zeros(1, 2, 2, 64, dtype=torch.float16, device=DEV)), dict(block=16)):
        with pytest.raises(ValueError):
            ops.cache8_append(**{**dict(k=k, v=k, k8=dk8, v8=dv8, k_scale=dks, v_scale=dvs), **kw})
    with pytest.raises(_lib.TrnError):      # rows that share memory
        ops.cache8_append(torch.zeros(1, 2, 1, 64, dtype=torch.float16, device=DEV), k, dk8[:, :1].expand(1, 2, 64, 64), dv8, dks, dvs)
    ops.cache8_append(k[:, :, :0], k[:, :, :0], dk8, dv8, dks, dvs)
    ops.cache8_attention(**{**good, "q": q[:, :, :0], "o": o[:, :, :0]})
