"""Steps on an fp16 cache: positions behind a shared prefix, positions that are given, heads of 128."""
import math

import pytest
import torch

from oracle import cache16 as ref
from triton_amd import modules, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _half(g, *s, size=1.0):
    return (torch.randn(*s, generator=g) * size).half().to(DEV)


def _within(got, want, tol, what=""):
    off = (got.detach().cpu().double() - want).abs() - tol
    assert not off.numel() or float(off.max()) <= 0, f"{what}: {float(off.max())} past the bound"


@pytest.mark.parametrize("offset", [1000, -7, 2 ** 27, 2 ** 31 - 1])
@pytest.mark.parametrize("D, interleaved", [(64, False), (128, True)])
def test_rope_offset(D, interleaved, offset):
    """A token at place p is rotated by p + offset: as with positions that say so, bit for bit, and within the definition's bound.  More new tokens than keys: places below zero too."""
    B, Hq, Hkv, M, S = 2, 4, 2, 5, 30
    g = torch.Generator().manual_seed(51)
    q, k, v = (_half(g, B, h, M, D) for h in (Hq, Hkv, Hkv))
    inv = (500000.0 ** (-torch.arange(D // 4, dtype=torch.float64) / (D // 4))).to(DEV)
    lengths, counts = [30, 3], [4, 5]
    places = (_ints(lengths) - _ints(counts)).cpu().long()[:, None] + torch.arange(M)
    runs = []
    for how in (dict(offset=offset), dict(positions=(places + offset).clamp(max=2 ** 31 - 1).int()[None].to(DEV))):
        out = [torch.zeros(B, h, s, D, dtype=torch.float16, device=DEV) for h, s in ((Hq, M), (Hkv, S), (Hkv, S))]
        ops.cache_rope_append(q, k, v, *out, inv, _ints(lengths), _ints(counts), interleaved=interleaved, **how)
        runs.append([x.cpu() for x in out])
    if offset < 2 ** 30:
        assert all(torch.equal(a, b) for a, b in zip(*runs))
    # (int64 positions: those past 31 bits too)
    outs, tols = ref.rope(q.cpu(), k.cpu(), v.cpu(), *(torch.zeros_like(x) for x in runs[0]), inv.cpu(), lengths, counts, (places + offset)[None], interleaved=interleaved)
    for got, want, tol in zip(runs[0], outs, tols):
        _within(got, want, tol)


def _weights(g, N, Hq, Hkv, D):
    return dict(WK=_half(g, N, Hkv * D, size=N ** -0.5), WQ=_half(g, N, Hq * D, size=N ** -0.5), WV=_half(g, N, Hkv * D, size=N ** -0.5),
                gamma_q=(1 + 0.1 * torch.randn(D, generator=g)).half().to(DEV), gamma_k=(1 + 0.1 * torch.randn(D, generator=g)).half().to(DEV),
                inv_freq=(10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).to(DEV))


def _call(step, t, **kw):
    t = {**t, **kw}
    step.forward(*(t.get(n) for n in step.TENSOR_PARAMS))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("variant", ["prefix", "prenorm"])
@pytest.mark.parametrize("given", [False, True])
def test_behind_a_prefix_as_in_one_sequence(variant, given, D):
    """Sequences behind a shared prefix, prompts and tokens, against the same tokens in caches that begin with the prefix's own: keys and values bit for bit, and
    outputs within what the definition on the whole sequence allows.  The prefix is made by a step too."""
    B, Hq, Hkv, N, P, S = 3, 8, 2, 192, 70, 60
    g = torch.Generator().manual_seed(52)
    w = _weights(g, N, Hq, Hkv, D)
    nothing = torch.zeros(Hkv, 0, D, dtype=torch.float16, device=DEV)
    whole = modules.get(variant, "cache16", head_dim=D, qk_norm=True)
    step = modules.get(variant, "cache16", head_dim=D, qk_norm=True, after_prefix=None if given else True)
    caches = [torch.zeros(B, Hkv, P + S, D, dtype=torch.float16, device=DEV) for _ in range(2)]
    own = [torch.zeros(B, Hkv, S, D, dtype=torch.float16, device=DEV) for _ in range(2)]
    x = _half(g, 1, P, N).expand(B, P, N).contiguous()
    _call(whole, w, X=x, O2=torch.zeros(B, P, Hq * D, dtype=torch.float16, device=DEV), K_cache=caches[0], V_cache=caches[1], K_prefix=nothing, V_prefix=nothing, lengths=_ints([P] * B))
    kp, vp = (c[0, :, :P].clone() for c in caches)
    lengths = [0] * B
    for M, counts in ((20, [20, 7, 13]), (1, [1, 1, 1]), (1, [1, 0, 1]), (3, [2, 3, 1])):
        lengths = [n + c for n, c in zip(lengths, counts)]
        x = _half(g, B, M, N)
        o1, o2 = (torch.zeros(B, M, Hq * D, dtype=torch.float16, device=DEV) for _ in range(2))
        places = (torch.tensor(lengths) - torch.tensor(counts))[:, None] + torch.arange(M) + P
        _call(whole, w, X=x, O2=o1, K_cache=caches[0], V_cache=caches[1], K_prefix=nothing, V_prefix=nothing, lengths=_ints([P + n for n in lengths]), counts=_ints(counts))
        _call(step, w, X=x, O2=o2, K_cache=own[0], V_cache=own[1], K_prefix=kp, V_prefix=vp, lengths=_ints(lengths), counts=_ints(counts),
              positions=places.int()[None].to(DEV) if given else None)
        for a, b in zip(own, caches):
            assert torch.equal(a, b[:, :, P:])
        qkv = [torch.zeros(B, M, h, D, dtype=torch.float16, device=DEV) for h in (Hq, Hkv, Hkv)]
        ops.prenorm_qkv(x.view(B * M, N), None, w["WQ"], w["WK"], w["WV"], *(y.view(B * M, -1, D).permute(1, 0, 2) for y in qkv), 0.0, variant == "prenorm")
        qr = torch.zeros_like(qkv[0]).permute(0, 2, 1, 3)
        ops.cache_rope_append(*(y.permute(0, 2, 1, 3) for y in qkv), qr, *(c.clone() for c in own), w["inv_freq"], _ints(lengths), _ints(counts), None, w["gamma_q"], w["gamma_k"], True, offset=P)
        kc, vc = (c.cpu() for c in caches)
        want, tol = ref.prefix_attention(qr.cpu(), kc, vc, kc[0, :, :0], vc[0, :, :0], torch.zeros(qr.shape).half(), D ** -0.5, True, [P + n for n in lengths], counts)
        for o in (o1, o2):
            _within(o.view(B, M, Hq, D).permute(0, 2, 1, 3), want, tol)


def test_a_captured_step_behind_a_prefix():
    """One token a sequence, captured once: positions grow with the lengths, which alone are raised between replays."""
    B, Hq, Hkv, N, P, S, D = 2, 4, 2, 192, 33, 40, 128
    runs = []
    for captured in (False, True):
        g = torch.Generator().manual_seed(53)
        w = _weights(g, N, Hq, Hkv, D)
        step = modules.get("prefix", "cache16", head_dim=D, after_prefix=True)
        t = dict(w, gamma_q=None, gamma_k=None, X=_half(g, B, 1, N), O2=torch.zeros(B, 1, Hq * D, dtype=torch.float16, device=DEV), K_prefix=_half(g, Hkv, P, D), V_prefix=_half(g, Hkv, P, D),
                 lengths=_ints([5, 1]), counts=_ints([1, 1]))
        t.update(K_cache=torch.zeros(B, Hkv, S, D, dtype=torch.float16, device=DEV), V_cache=torch.zeros(B, Hkv, S, D, dtype=torch.float16, device=DEV))
        _call(step, t)
        torch.cuda.synchronize()
        graph, got = torch.cuda.CUDAGraph(), []
        if captured:
            with torch.cuda.graph(graph):
                _call(step, t)
        for i in range(4):
            t["lengths"] += 1
            t["X"].copy_(torch.randn(t["X"].shape, generator=g))
            graph.replay() if captured else _call(step, t)
            torch.cuda.synchronize()
            got += [t[n].clone() for n in ("O2", "K_cache", "V_cache")]
        runs.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("variant", ["prefix", "sparse"])
def test_positions_of_several_axes_in_a_step(variant, D):
    B, M, Hq, Hkv, N, S, P = 2, 9, 8, 2, 192, 200, 12
    g = torch.Generator().manual_seed(54)
    w = _weights(g, N, Hq, Hkv, D)
    sections = [D // 2 - 2 * (D // 8), D // 8, D // 8]
    kw = dict(head_dim=D, qk_norm=True, sections=sections)
    step = modules.get("prefix", "cache16", **kw) if variant == "prefix" else modules.get("sparse", "cache16", top=3, sink=1, recent=1, block=32, **kw)
    positions = torch.randint(0, 5000, (3, B, M), generator=g).int()
    lengths, counts = [200, 9], [9, 6]
    before = [_half(g, B, Hkv, S, D) for _ in range(2)]
    kc, vc = (b.clone() for b in before)
    x, o = _half(g, B, M, N), torch.zeros(B, M, Hq * D, dtype=torch.float16, device=DEV)
    bnd, sel = torch.zeros(B, Hkv, 7, 2, D, dtype=torch.float16, device=DEV), torch.zeros(B, Hkv, M, 3, dtype=torch.int32, device=DEV)
    ops.cache_bounds(before[0], bnd, 32, _ints([n - c for n, c in zip(lengths, counts)]))
    old = bnd.cpu()
    kp, vp = _half(g, Hkv, P, D), _half(g, Hkv, P, D)
    _call(step, w, X=x, O2=o, K_cache=kc, V_cache=vc, K_prefix=kp, V_prefix=vp, positions=positions.to(DEV), lengths=_ints(lengths), counts=_ints(counts), bounds=bnd, selected=sel)
    qkv = [torch.zeros(B, M, h, D, dtype=torch.float16, device=DEV) for h in (Hq, Hkv, Hkv)]
    ops.prenorm_qkv(x.view(B * M, N), None, w["WQ"], w["WK"], w["WV"], *(y.view(B * M, -1, D).permute(1, 0, 2) for y in qkv), 0.0, False)
    q, k, v = (y.permute(0, 2, 1, 3).cpu() for y in qkv)
    outs, tols = ref.rope(q, k, v, q, before[0].cpu(), before[1].cpu(), w["inv_freq"].cpu(), lengths, counts, positions, w["gamma_q"].cpu(), w["gamma_k"].cpu(), True, sections=sections)
    for got, want, tol in zip((kc, vc), outs[1:], tols[1:]):
        _within(got, want, tol)
    qr = torch.zeros_like(qkv[0]).permute(0, 2, 1, 3)
    ops.cache_rope_append(*(y.permute(0, 2, 1, 3) for y in qkv), qr, kc.clone(), vc.clone(), w["inv_freq"], _ints(lengths), _ints(counts), positions.to(DEV), w["gamma_q"], w["gamma_k"], True,
                          sections=sections)
    args = (qr.cpu(), kc.cpu(), vc.cpu())
    if variant == "prefix":
        want, tol = ref.prefix_attention(*args, kp.cpu(), vp.cpu(), torch.zeros_like(args[0]), D ** -0.5, True, lengths, counts)
    else:
        assert torch.equal(bnd.cpu(), ref.bounds(args[1], old, 32, lengths, counts))
        want_sel = ref.select(args[0], bnd.cpu(), torch.zeros(sel.shape, dtype=torch.int32), 32, 3, 1, 1, Hq // Hkv, lengths, counts, S)
        assert torch.equal(sel.cpu(), want_sel)
        want, tol = ref.sparse_attention(*args, torch.zeros_like(args[0]), want_sel, 32, D ** -0.5, lengths, counts)
    _within(o.view(B, M, Hq, D).permute(0, 2, 1, 3), want, tol)


@pytest.mark.parametrize("form", ["cache8", "cache16"])
def test_prompts_of_any_length_share_workspaces(form):
    """Numbers of tokens that differ from call to call do not each leave a workspace behind, and a captured step of one keeps its results while others run."""
    B, Hq, Hkv, N, S, D = 1, 8, 2, 192, 1500, 64
    g = torch.Generator().manual_seed(55)
    w = _weights(g, N, Hq, Hkv, D)
    step = modules.get("vanilla" if form == "cache8" else "prefix", form, head_dim=D)
    nothing = torch.zeros(Hkv, 0, D, dtype=torch.float16, device=DEV)
    t = dict(w, gamma_q=None, gamma_k=None, K_cache=torch.zeros(B, Hkv, S, D, dtype=torch.float16, device=DEV), V_cache=torch.zeros(B, Hkv, S, D, dtype=torch.float16, device=DEV), K_prefix=nothing,
             V_prefix=nothing, K8=torch.zeros(B, Hkv, S, D, dtype=torch.float8_e4m3fn, device=DEV), V8=torch.zeros(B, Hkv, S, D, dtype=torch.float8_e4m3fn, device=DEV),
             K_scale=torch.ones(B, Hkv, -(-S // 64), device=DEV), V_scale=torch.ones(B, Hkv, -(-S // 64), device=DEV))
    call = lambda m: dict(X=torch.randn(B, m, N, generator=torch.Generator().manual_seed(m)).half().to(DEV), O2=torch.zeros(B, m, Hq * D, dtype=torch.float16, device=DEV), lengths=_ints([m]))
    seven = call(7)
    _call(step, t, **seven)
    want = seven["O2"].clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        _call(step, t, **seven)
    for m in (1, 6, 30, 200, 333, 700, 701, 1400, 1499, 8):
        _call(step, t, **call(m))
        seven["O2"].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(seven["O2"], want)
    held = [x.numel() * x.element_size() for k, x in step._ws.items() if k[0] == "qkv"]
    # (powers of two from 1 MiB on: the largest, 1499 x 12 x 64 x 2 bytes, takes 4 MiB, and all below it less than as much again)
    assert len(held) <= 3 and sum(held) < 8 << 20
