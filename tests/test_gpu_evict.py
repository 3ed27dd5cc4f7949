"""Eviction from caches by accumulated weight, against the definition: what is kept, where it goes and what is left alone are held to equality."""
import math

import pytest
import torch

from oracle import cache8 as ref
from triton_amd import _lib, modules, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"

CASES = [
    # B, Hkv, rows of weights a head, D, capacity, keep, recent, lengths
    (1, 1, 1, 64, 8, 4, 1, [8]),
    (2, 2, 4, 128, 100, 40, 10, [100, 77]),
    (3, 2, 1, 64, 300, 128, 0, [300, 128, 5]),           # one that is just full, one with room left
    (2, 1, 71, 64, 130, 1, 1, [130, 0]),                 # the last key alone; no key at all
    (2, 3, 2, 128, 1100, 1030, 1030, [1100, 1031]),      # the last ones alone
    (1, 2, 1, 128, 2500, 1300, 64, [2500]),
    (2, 8, 4, 128, 5000, 300, 32, [4999, 2111]),
    (1, 1, 1, 64, 70, 90, 7, [64]),                      # a budget that is larger than the cache
]
KINDS = ["spread", "ties", "ends"]


def _weights(kind, B, rows, S, g):
    w = torch.exp(2 * torch.randn(B, rows, S, generator=g))
    if kind == "ties":
        w = (w * 2).round() / 2
        w[:, :, S // 3:S // 2] = 1.0
    if kind == "ends":
        pick = torch.rand(B, rows, S, generator=g)
        w = torch.where(pick < 0.1, torch.full_like(w, math.nan), torch.where(pick < 0.2, torch.full_like(w, -math.inf), torch.where(
            pick < 0.3, torch.full_like(w, math.inf), torch.where(pick < 0.5, -w, torch.where(pick < 0.6, torch.zeros_like(w), w)))))
        if rows > 1:
            w = torch.nan_to_num(w, nan=math.nan, posinf=1e30, neginf=-1e30)
    return w


def _run(case, kind, half, bits, place, block=64, seed=3, layout="head"):
    B, H, per, D, S, keep, recent, lengths = case
    g = torch.Generator().manual_seed(seed)
    w = _weights(kind, B, H * per, S, g)
    if half:
        w = w.clamp(-60000, 60000).half()
    if bits == 8:
        k, v = (ref.encode((torch.randn(B, H, S, D, generator=g) * 100).clamp(-448, 448)) for _ in range(2))
        ks, vs = (torch.exp2(torch.randint(-4, 5, (B, H, -(-S // block)), generator=g).float()) for _ in range(2))
    else:
        k, v = (torch.randn(B, H, S, D, generator=g).half() for _ in range(2))
        ks = vs = None

    def dev(x):
        if layout == "token":
            return torch.empty(B, x.shape[2], H, D, dtype=x.dtype, device=DEV).permute(0, 2, 1, 3).copy_(x)
        return x.to(DEV)
    dk, dv, dw = dev(k), dev(v), w.to(DEV)
    dks, dvs = (None, None) if bits == 16 else (ks.to(DEV), vs.to(DEV))
    rows = min(keep, S)
    if place == "within":
        ko, vo, wo = dk, dv, dw
        kso, vso = dks, dvs
    else:
        ko, vo = (dev(torch.full((B, H, rows, D), 9, dtype=k.dtype)) for _ in range(2))
        wo = torch.full((B, H * per, keep), 9, dtype=w.dtype, device=DEV)
        kso, vso = (None, None) if bits == 16 else (torch.full((B, H, -(-rows // block)), 9.0, device=DEV) for _ in range(2))
    kept = torch.full((B, H, keep), 77, dtype=torch.int32, device=DEV)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    new = n if place == "within" else torch.full_like(n, 77)
    ws = torch.full((ops.cache_evict_workspace_bytes(dk, dw, keep),), 0xff, dtype=torch.uint8, device=DEV)
    ops.cache_evict(dk, dv, dw, ko, vo, kept, keep, recent, ws, n, new, wo, dks, dvs, kso, vso, block)
    want = ref.evict(k, v, w, keep, recent, lengths, ks, vs, block)
    assert new.tolist() == [min(x, keep) for x in lengths]
    for b, x in enumerate(lengths):
        m = min(x, keep)
        for h in range(H):
            got = kept[b, h].cpu()
            assert torch.equal(got[:m], want["kept"][b][h].int()) and (got[m:] == -1).all()
            for name, out, src in (("k", ko, k), ("v", vo, v)):
                o = out[b, h].cpu()
                assert torch.equal(o[:m].view(torch.uint8), want[name][b][h].view(torch.uint8)), name
                behind = src[b, h, m:] if place == "within" else torch.full_like(o[m:], 9)
                assert torch.equal(o[m:].view(torch.uint8), behind.contiguous().view(torch.uint8)), "rows behind the new length"
            if bits == 8:
                for name, out, src in (("ks", kso, ks), ("vs", vso, vs)):
                    blocks = -(-m // block)
                    o = out[b, h].cpu()
                    assert torch.equal(o[:blocks], want[name][b][h])
                    assert torch.equal(o[blocks:], src[b, h, blocks:] if place == "within" else torch.full_like(o[blocks:], 9))
            ow = wo[b, h * per:(h + 1) * per].cpu().float()
            ww = want["w"][b][h].float()
            assert torch.equal(torch.nan_to_num(ow[:, :m], nan=-5e20), torch.nan_to_num(ww, nan=-5e20))
            if place == "within":
                assert (ow[:, m:x] == 0).all()
                assert torch.equal(torch.nan_to_num(ow[:, x:], nan=-5e20), torch.nan_to_num(w[b, h * per:(h + 1) * per, x:].float(), nan=-5e20))
            else:
                assert (ow[:, m:] == 9).all()


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"B{c[0]}H{c[1]}x{c[2]}D{c[3]}S{c[4]}k{c[5]}r{c[6]}")
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("place", ["apart", "within"])
def test_evict(case, bits, place):
    for kind in KINDS:
        for half in (False, True):
            _run(case, kind, half, bits, place)


@pytest.mark.parametrize("block", [32, 128])
@pytest.mark.parametrize("place", ["apart", "within"])
def test_other_blocks_and_token_major_caches(block, place):
    _run(CASES[6], "spread", False, 8, place, block, layout="token")
    _run(CASES[1], "spread", True, 16, place, layout="token")


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("B, D", [(20, 128), (20, 64), (10, 128)])
def test_many_heads_in_place(B, D, bits):
    """Heads enough for columns of 128 bytes and of whole rows; several steps of each."""
    _run((B, 7, 1, D, 1300, 1100, 9, [1300 - 137 * (b % 10) for b in range(B)]), "spread", False, bits, "within")


@pytest.mark.parametrize("kind", ["spread", "ties"])
@pytest.mark.parametrize("S", [4096, 4097, 8193, 16385, 32768, 32769, 40000])
def test_long_rows(S, kind):
    _run((1, 1, 2, 64, S, S // 2 + 1, 100, [S - 1]), kind, False, 16, "within")
    _run((1, 2, 1, 64, S, S // 3, 0, [S]), kind, True, 8, "apart")
    _run((1, 1, 9, 64, S, S // 2, 3, [S - 5]), kind, True, 16, "apart")


def _sides(place, bits, make):
    """An eviction whose caches, and results, `make` lays out on the device as (k, v, k_out, v_out), held to the definition; rows that are not written stay."""
    B, H, D, S, keep, recent, block, lengths = 2, 3, 64, 300, 130, 20, 32, [300, 207]
    g = torch.Generator().manual_seed(14)
    w = torch.exp(2 * torch.randn(B, H, S, generator=g))
    if bits == 8:
        k, v = (ref.encode((torch.randn(B, H, S, D, generator=g) * 100).clamp(-448, 448)) for _ in range(2))
        ks, vs = (torch.exp2(torch.randint(-4, 5, (B, H, -(-S // block)), generator=g).float()) for _ in range(2))
    else:
        k, v = (torch.randn(B, H, S, D, generator=g).half() for _ in range(2))
        ks = vs = None
    dk, dv, ko, vo = make(k.to(DEV), v.to(DEV))
    scales = [None] * 4 if bits == 16 else [t.to(DEV) for t in (ks, vs, ks, vs)]
    before = [t.cpu() for t in (ko, vo)]
    kept, n = torch.zeros(B, H, keep, dtype=torch.int32, device=DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)
    dw = w.to(DEV)
    ws = torch.full((ops.cache_evict_workspace_bytes(dk, dw, keep),), 0xff, dtype=torch.uint8, device=DEV)
    ops.cache_evict(dk, dv, dw, ko, vo, kept, keep, recent, ws, n, n, None, *scales, block)
    want = ref.evict(k, v, w, keep, recent, lengths, ks, vs, block)
    for b in range(B):
        for h in range(H):
            assert torch.equal(kept[b, h].cpu(), want["kept"][b][h].int())
            for name, out, old in (("k", ko, before[0]), ("v", vo, before[1])):
                o = out[b, h].cpu().contiguous()
                assert torch.equal(o[:keep].view(torch.uint8), want[name][b][h].view(torch.uint8)), (name, b, h)
                assert torch.equal(o[keep:].view(torch.uint8), old[b, h, keep:].contiguous().view(torch.uint8))
            if bits == 8:
                for name, out in (("ks", scales[2]), ("vs", scales[3])):
                    assert torch.equal(out[b, h, :len(want[name][b][h])].cpu(), want[name][b][h])


@pytest.mark.parametrize("axis", [1, 2, 3], ids=["by sequence", "by head", "by token"])
@pytest.mark.parametrize("place", ["apart", "within"])
@pytest.mark.parametrize("bits", [16, 8])
def test_keys_and_values_of_one_tensor(bits, place, axis):
    def make(k, v):
        def pack(a, b):
            a, b = (a.transpose(1, 2), b.transpose(1, 2)) if axis == 3 else (a, b)
            both = torch.stack((a, b), 2 if axis == 3 else axis)
            return [t.transpose(1, 2) if axis == 3 else t for t in both.unbind(2 if axis == 3 else axis)]
        k, v = pack(k, v)
        if place == "within":
            return k, v, k, v
        return k, v, *pack(torch.full((2, 3, 140, 64), 9, dtype=k.dtype, device=DEV), torch.full((2, 3, 140, 64), 8, dtype=k.dtype, device=DEV))
    _sides(place, bits, make)


@pytest.mark.parametrize("stays", ["k", "v"])
@pytest.mark.parametrize("bits", [16, 8])
def test_one_of_keys_and_values_in_place(bits, stays):
    """The other goes into a cache of its own."""
    def make(k, v):
        out = torch.full((2, 3, 140, 64), 9, dtype=k.dtype, device=DEV)
        return (k, v, k, out) if stays == "k" else (k, v, out, v)
    _sides("mixed", bits, make)


def test_keyformer_scores_cut_a_prompt():
    """KeyFormer's prompt module and eviction by its scores, one after the other, as a user has them."""
    B, Hq, Hkv, S, D, keep, recent = 2, 8, 2, 300, 128, 100, 20
    g = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(B, h, S, D, generator=g).half().to(DEV) for h in (Hq, Hkv, Hkv))
    noise = torch.randn(B, Hq, S, S, generator=g).to(DEV)
    score, o = torch.zeros(B, Hq, S, device=DEV), torch.zeros_like(q)
    modules.get("keyformer").forward(score, k, o, q, v, noise)
    ko, vo = (torch.zeros(B, Hkv, keep, D, dtype=torch.float16, device=DEV) for _ in range(2))
    kept = torch.zeros(B, Hkv, keep, dtype=torch.int32, device=DEV)
    modules.get("evict", "cache", keep=keep, recent=recent).forward(k, ko, v, vo, kept, None, None, score, None)
    want = ref.evict(k.cpu(), v.cpu(), score.cpu(), keep, recent, [S] * B)
    for b in range(B):
        for h in range(Hkv):
            assert torch.equal(kept[b, h].cpu(), want["kept"][b][h].int()) and torch.equal(ko[b, h].cpu(), want["k"][b][h])


def test_captured_and_replayed():
    """The same graph on weights that change: each replay against a call of its own."""
    B, H, D, S, keep, recent = 2, 2, 64, 500, 200, 16
    g = torch.Generator().manual_seed(9)
    k, v = (torch.randn(B, H, S, D, generator=g).half().to(DEV) for _ in range(2))
    w = torch.zeros(B, H, S, device=DEV)
    outs = [torch.zeros(B, H, keep, D, dtype=torch.float16, device=DEV) for _ in range(4)]
    kept = [torch.zeros(B, H, keep, dtype=torch.int32, device=DEV) for _ in range(2)]
    mod, other = (modules.get("evict", "cache", keep=keep, recent=recent) for _ in range(2))
    n = torch.tensor([500, 333], dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        mod.forward(k, outs[0], v, outs[1], kept[0], n, None, w, None)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            mod.forward(k, outs[0], v, outs[1], kept[0], n, None, w, None)
    for i in range(5):
        w.copy_(torch.rand(B, H, S, generator=g))
        n.copy_(torch.tensor([500 - 13 * i, 333 - 50 * i], dtype=torch.int32))
        other.forward(k, outs[2], v, outs[3], kept[1], n, None, w, None)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept[0], kept[1])
        m = min(keep, 333 - 50 * i)
        assert torch.equal(outs[0][1, :, :m], outs[2][1, :, :m]) and torch.equal(outs[1][0], outs[3][0])


def test_a_serving_loop():
    """Prompt and tokens appended to an 8-bit cache, attention with weights, eviction when it is full, and on: all together against the definitions."""
    B, Hq, Hkv, D, S, block, keep, recent = 2, 4, 2, 64, 96, 32, 50, 8
    g = torch.Generator().manual_seed(12)
    k8, v8 = (torch.zeros(B, Hkv, S, D, dtype=torch.uint8) for _ in range(2))
    ks, vs = (torch.zeros(B, Hkv, S // block) for _ in range(2))
    dk8, dv8, dks, dvs = (t.to(DEV) for t in (k8, v8, ks, vs))
    w = torch.zeros(B, Hkv, S, device=DEV)
    lengths, n = [0, 0], torch.zeros(B, dtype=torch.int32, device=DEV)
    app, att = modules.get("append8", "cache", block=block), modules.get("weights8", "cache", block=block)
    ev = modules.get("evict8", "cache", keep=keep, recent=recent, block=block)
    kept = torch.zeros(B, Hkv, keep, dtype=torch.int32, device=DEV)
    evicted = 0
    for step in range(40):
        M, counts = (40, [40, 31]) if step == 0 else (3, [3, 1 + step % 3])
        if max(lengths) + M > S:
            wcpu = w.cpu()
            want = ref.evict(k8, v8, wcpu, keep, recent, lengths, ks, vs, block)
            ev.forward(dk8, dk8, dks, dks, dv8, dv8, dvs, dvs, kept, n, n, w, w)
            lengths = [min(x, keep) for x in lengths]
            for b, m in enumerate(lengths):
                for h in range(Hkv):
                    assert torch.equal(kept[b, h, :m].cpu(), want["kept"][b][h].int())
                    k8[b, h, :m], v8[b, h, :m] = want["k"][b][h], want["v"][b][h]
                    ks[b, h, :-(-m // block)], vs[b, h, :-(-m // block)] = want["ks"][b][h], want["vs"][b][h]
            evicted += 1
        q, k, v = (torch.randn(B, h, M, D, generator=g).half() for h in (Hq, Hkv, Hkv))
        o = torch.zeros(B, Hq, M, D, dtype=torch.float16, device=DEV)
        c = torch.tensor(counts, dtype=torch.int32, device=DEV)
        n.add_(c)
        lengths = [x + y for x, y in zip(lengths, counts)]
        app.forward(k.to(DEV), dk8, dks, v.to(DEV), dv8, dvs, c, n)
        before = w.cpu()
        att.forward(dk8, dks, o, q.to(DEV), dv8, dvs, c, n, w, w)
        k8, ks = ref.append(k, k8, ks, lengths, counts, block)
        v8, vs = ref.append(v, v8, vs, lengths, counts, block)
        want, _, ww, tol, wtol, _ = ref.attention(q, k8, v8, ks, vs, D ** -0.5, True, lengths, counts, block)
        for b in range(B):
            y, t = want[b, :, :counts[b]], tol[b, :, :counts[b]]
            assert ((o[b, :, :counts[b]].cpu().double() - y).abs() <= t).all()
            total = before[b, :, :lengths[b]].double() + ww[b, :, :lengths[b]]
            assert ((w[b, :, :lengths[b]].cpu().double() - total).abs() <= wtol[b, :, :lengths[b]] + 2.0 ** -23 * total).all()
        assert torch.equal(dk8[0, :, :lengths[0]].cpu(), k8[0, :, :lengths[0]]) and torch.equal(dvs[1, :, :-(-lengths[1] // block)].cpu(), vs[1, :, :-(-lengths[1] // block)])
    assert n.tolist() == lengths and evicted >= 2


def test_refusals():
    k = torch.zeros(1, 2, 64, 64, dtype=torch.float16, device=DEV)
    v, out, vout = k.clone(), torch.zeros(1, 2, 16, 64, dtype=torch.float16, device=DEV), torch.zeros(1, 2, 16, 64, dtype=torch.float16, device=DEV)
    w, kept = torch.zeros(1, 4, 64, device=DEV), torch.zeros(1, 2, 16, dtype=torch.int32, device=DEV)
    ws = torch.zeros(ops.cache_evict_workspace_bytes(k, w, 16), dtype=torch.uint8, device=DEV)
    good = dict(k=k, v=v, weights=w, k_out=out, v_out=vout, kept=kept, keep=16, recent=4, workspace=ws)
    ops.cache_evict(**good)

    def bad(error=ValueError, **kw):
        with pytest.raises(error):
            ops.cache_evict(**{**good, **kw})
    bad(keep=0); bad(recent=17); bad(recent=-1); bad(kept=kept[:, :1]); bad(kept=kept.long()); bad(weights=w[:, :3].contiguous()); bad(weights=w.double())
    bad(weights=w[:, :, ::2]); bad(v=v[:, :, :32]); bad(k_out=out[:, :, :8]); bad(k_out=out.float()); bad(weights_out=torch.zeros(1, 4, 64, device=DEV))
    bad(k=k.float()); bad(lengths=torch.zeros(1, device=DEV)); bad(workspace=ws.float()); bad(k=k.cpu())
    bad(_lib.TrnError, workspace=ws[:128]); bad(_lib.TrnError, k_out=k[:, :, 8:24]); bad(_lib.TrnError, k_out=v[:, :, :16]); bad(_lib.TrnError, v_out=out)
    bad(_lib.TrnError, k_out=out[:, :1].expand(1, 2, 16, 64))
    codes = torch.zeros(1, 2, 64, 64, dtype=torch.uint8, device=DEV)
    bad(k=codes, v=codes, k_out=codes, v_out=codes)
