"""Layouts of an fp16 cache: strides of axes that have one entry, and caches that have room for more than they hold."""
import pytest
import torch

from oracle import cache16 as ref
from triton_amd import modules

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _one(x, pitch):
    """[.., 1, D] on the GPU whose stride between tokens is 1, or `pitch`."""
    x = x.to(DEV)
    return x[..., 0, :].unsqueeze(-1).transpose(-1, -2) if pitch == 1 else x.as_strided(x.shape, x.stride()[:-2] + (pitch, 1))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("pitch", [1, 3, 1 << 30])
@pytest.mark.parametrize("B, M, P, S", [(1, 1, 1, 1), (2, 1, 1, 90), (2, 3, 90, 1), (1, 1, 1, 5000), (30, 3, 1, 700), (1, 40, 1, 300), (1, 40, 300, 1), (2, 2, 5000, 1)])
def test_one_key_of_any_stride(B, M, P, S, pitch, D):
    """A cache or a prefix of one key, as unsqueeze and transpose leave it: what lies behind that key in memory is not a key."""
    Hq, Hkv = 8, 2
    g = torch.Generator().manual_seed(41)
    q, k, v = (torch.randn(B, h, s, D, generator=g).half() for h, s in ((Hq, M), (Hkv, S), (Hkv, S)))
    kp, vp = (torch.randn(Hkv, P, D, generator=g).half() for _ in range(2))
    want, tol = ref.prefix_attention(q, k, v, kp, vp, torch.zeros_like(q), D ** -0.5, True, [S] * B, [M] * B)
    dk, dv = (_one(x, pitch) if S == 1 else x.to(DEV) for x in (k, v))
    dkp, dvp = (_one(x, pitch) if P == 1 else x.to(DEV) for x in (kp, vp))
    assert (S > 1 or dk.stride(2) == pitch) and (P > 1 or dvp.stride(1) == pitch)
    o = torch.zeros(B, Hq, M, D, dtype=torch.float16, device=DEV)
    modules.get("prefix", "cache").forward(dk, dkp, o, q.to(DEV), dv, dvp, None, None)
    assert ((o.cpu().double() - want).abs() <= tol).all()
    if S == 1:
        bnd, sel = torch.zeros(B, Hkv, 1, 2, D, dtype=torch.float16, device=DEV), torch.zeros(B, Hkv, M, 2, dtype=torch.int32, device=DEV)
        modules.get("bounds", "cache").forward(dk, bnd, None, None)
        assert torch.equal(bnd.cpu(), ref.bounds(k, torch.zeros(bnd.shape).half(), 64, [1] * B, [1] * B))
        modules.get("sparse", "cache", top=2).forward(dk, o, q.to(DEV), dv, bnd, None, None, sel)
        want, tol = ref.prefix_attention(q, k, v, kp[:, :0], vp[:, :0], torch.zeros_like(q), D ** -0.5, True, [1] * B, [M] * B)
        assert ((o.cpu().double() - want).abs() <= tol).all()


ROOMY = [
    # B, Hq, Hkv, D, new, lengths, counts, prefix: in a cache of 9000 places.  Narrow shares; wide tiles on the prefix; two narrow row tiles; tiles of one sequence's rows, one number and two; no prefix;
    # nothing there
    (2, 8, 2, 128, 1, [5, 300], [1, 1], 700),
    (12, 8, 2, 64, 1, list(range(1, 13)), [1] * 12, 900),
    (25, 6, 2, 128, 4, [40 - i for i in range(25)], [1 + i % 4 for i in range(25)], 1500),
    (1, 8, 1, 64, 4, [9], [4], 300),
    (2, 8, 2, 128, 40, [200, 47], [40, 9], 333),
    (2, 8, 2, 64, 150, [260, 150], [150, 97], 190),
    (3, 8, 2, 128, 1, [33, 0, 70], [1, 0, 1], 0),
    (2, 8, 2, 64, 80, [90, 80], [80, 3], 0),
    (2, 4, 2, 64, 2, [0, 0], [2, 1], 100),
]


@pytest.mark.parametrize("case", ROOMY, ids=lambda c: f"B{c[0]}H{c[1]}_{c[2]}D{c[3]}M{c[4]}P{c[7]}")
def test_caches_with_room(case):
    """A cache much larger than what it holds, as a serving loop allocates it: what lies behind the sequences is NaN.  Selected blocks likewise, from few to all of what is there."""
    B, Hq, Hkv, D, M, lengths, counts, P = case
    S, far = max(max(lengths), 1), 9000
    g = torch.Generator().manual_seed(42)
    q, k, v = (torch.randn(B, h, s, D, generator=g).half() for h, s in ((Hq, M), (Hkv, S), (Hkv, S)))
    kp, vp = (torch.randn(Hkv, P, D, generator=g).half() for _ in range(2))
    for b, (n, c) in enumerate(zip(lengths, counts)):
        k[b, :, n:], v[b, :, n:], q[b, :, c:] = float("nan"), float("nan"), float("nan")
    dk, dv = (torch.full((B, Hkv, far, D), float("nan"), dtype=torch.float16, device=DEV) for _ in range(2))
    dk[:, :, :S], dv[:, :, :S] = k.to(DEV), v.to(DEV)
    ln, ct = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (lengths, counts))
    was = torch.randn(q.shape, generator=g).half()
    o = was.to(DEV)
    want, tol = ref.prefix_attention(q, k, v, kp, vp, was, D ** -0.5, True, lengths, counts)
    modules.get("prefix", "cache").forward(dk, kp.to(DEV), o, q.to(DEV), dv, vp.to(DEV), ct, ln)
    assert ((o.cpu().double() - want).abs() <= tol).all()
    for top in (1, 3, 300):
        bnd, sel = torch.zeros(B, Hkv, -(-far // 32), 2, D, dtype=torch.float16, device=DEV), torch.full((B, Hkv, M, top), 7, dtype=torch.int32, device=DEV)
        modules.get("bounds", "cache", block=32).forward(dk, bnd, None, ln)
        o = was.to(DEV)
        modules.get("sparse", "cache", top=top, block=32).forward(dk, o, q.to(DEV), dv, bnd, ct, ln, sel)
        want_sel = ref.select(q, bnd.cpu(), torch.full(sel.shape, 7, dtype=torch.int32), 32, top, 0, 1, Hq // Hkv, lengths, counts, far)
        assert torch.equal(sel.cpu(), want_sel)
        want, tol = ref.sparse_attention(q, k, v, was, want_sel, 32, D ** -0.5, lengths, counts)
        assert ((o.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("B, Hq, Hkv, D, M, S, counts", [(1, 71, 1, 64, 40, 900, [40]), (2, 16, 2, 128, 100, 700, [100, 37]), (1, 8, 1, 64, 128, 500, [128]), (1, 8, 1, 128, 129, 500, [120])])
def test_selection_of_many_heads_and_queries(B, Hq, Hkv, D, M, S, counts):
    """Eight heads and more on a KV head, 12 queries and more: scores by heads up to 128 queries, by queries above."""
    g = torch.Generator().manual_seed(43)
    q, k, v = (torch.randn(B, h, s, D, generator=g).half() for h, s in ((Hq, M), (Hkv, S), (Hkv, S)))
    for b, c in enumerate(counts):
        q[b, :, c:] = float("nan")
    bnd = torch.zeros(B, Hkv, -(-S // 32), 2, D, dtype=torch.float16, device=DEV)
    sel = torch.full((B, Hkv, M, 4), 7, dtype=torch.int32, device=DEV)
    o = torch.zeros(q.shape, dtype=torch.float16, device=DEV)
    modules.get("bounds", "cache", block=32).forward(k.to(DEV), bnd, None, None)
    modules.get("sparse", "cache", top=4, block=32).forward(k.to(DEV), o, q.to(DEV), v.to(DEV), bnd, torch.tensor(counts, dtype=torch.int32, device=DEV), None, sel)
    want_sel = ref.select(q, bnd.cpu(), torch.full(sel.shape, 7, dtype=torch.int32), 32, 4, 0, 1, Hq // Hkv, [S] * B, counts, S)
    assert torch.equal(sel.cpu(), want_sel)
    want, tol = ref.sparse_attention(q, k, v, torch.zeros_like(q), want_sel, 32, D ** -0.5, [S] * B, counts)
    assert ((o.cpu().double() - want).abs() <= tol).all()
