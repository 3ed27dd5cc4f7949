"""Attention over an fp16 cache where one key has nearly all of the weight and a value of zero, as the first token of a long text often has: what the others add up to is the output."""
import math

import pytest
import torch

from triton_amd import modules, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(B, Hkv, M, P, S, D, G, spread=5.0):
    """Queries that look at one channel; there the first key is 16 and the others are 12 to 12 + spread less; values about one, the first key's zero."""
    g = torch.Generator().manual_seed(31)
    q = torch.zeros(B, Hkv * G, M, D)
    q[..., 0] = 1.0 + torch.arange(Hkv * G)[:, None] / 128
    k, v = torch.randn(B, Hkv, P + S, D, generator=g), 1 + 0.5 * torch.randn(B, Hkv, P + S, D, generator=g)
    k[..., 0] = 4.0 - spread * torch.rand(B, Hkv, P + S, generator=g)
    if P:
        k[:, :, :P], v[:, :, :P] = k[:1, :, :P].clone(), v[:1, :, :P].clone()
    k[:, :, 0, 0], v[:, :, 0] = 16.0, 0.0
    return q.half(), k.half(), v.half()


def _check(o, q, k, v, sees, fine):
    """How far a row may be off.  A weight: 2^-32 of the largest, or 2^-22 of itself, as two fp16 numbers; 2^-32 or 2^-11 as one.  Its exponent is below 2^5 and has three roundings of 2^-24
    (the scale, the product, the difference: 2^-18 times ln 2 in all, with those of the largest), the exponential 2^-22: 2^-17 for numerator and sum.  Additions one behind the other: a wave's tiles,
    and 64 for those of a tile, waves and shares, 2^-24 each, in both.  The output's rounding: 2^-11, or 2^-25."""
    G, N = q.shape[1] // k.shape[1], k.shape[2]
    kk, vv = k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    t = (q.double()[..., 0, None] * kk[:, :, None, :, 0]).masked_fill(~sees, -math.inf)
    w = torch.exp(t - t.amax(-1, keepdim=True))
    total = w.sum(-1, keepdim=True)
    want = w @ vv / total
    size = w @ vv.abs() / total
    least, part = 2.0 ** -32, 2.0 ** -22 if fine else 2.0 ** -11
    tol = (sees.double() @ vv.abs()) / total * least + size * (part + 2.0 ** -17 + 2 * (N / 32 + 64) * 2.0 ** -24) + want.abs() * 2.0 ** -11 + 2.0 ** -25
    off = (o.double().cpu() - want).abs() - tol
    assert float(off.max()) <= 0, f"{float(off.max())} past the bound, {float((o.double().cpu() - want).norm() / want.norm()):.2g} of the outputs' size"


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B, M, P, S, fine", [
    (1, 1, 200, 300, True),          # eight waves a row tile
    (1, 2, 3000, 900, True),         # shares of prefix and own keys
    (12, 1, 4000, 500, True),        # wide tiles on the prefix
    (1, 30, 0, 4000, True),          # one sequence's rows, few heads
    (1, 150, 2000, 600, False),      # many
    (4, 90, 0, 1500, False),
])
def test_a_key_that_has_nearly_all_weight(B, M, P, S, fine, D):
    Hkv, G = 2, 4
    q, k, v = _inputs(B, Hkv, M, P, S, D, G)
    o = torch.empty(B, Hkv * G, M, D, dtype=torch.float16, device=DEV)
    kd, vd = k.to(DEV), v.to(DEV)
    modules.get("prefix", "cache", scale=1.0).forward(kd[:, :, P:], kd[0, :, :P], o, q.to(DEV), vd[:, :, P:], vd[0, :, :P], None, None)
    sees = torch.arange(P + S) <= (P + S - M + torch.arange(M))[:, None]
    _check(o, q, k, v, sees.expand(B, Hkv * G, M, P + S), fine)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B, M, P, S, Hkv", [(1, 40, 0, 700, 2), (24, 40, 0, 700, 2), (24, 20, 900, 300, 2), (3, 64, 600, 200, 2), (5, 1, 600, 200, 2), (60, 5, 600, 200, 2), (1, 32, 100, 700, 8), (6, 32, 100, 700, 8)])
def test_a_step_is_as_exact_in_any_batch(B, M, P, S, Hkv, D):
    """Up to 512 rows of a sequence, or 128 of a KV head, alone or beside many: weights are two numbers.  They are equal, so that what one number would lose does not average out."""
    G = 4
    q, k, v = _inputs(B, Hkv, M, P, S, D, G, 0.0)
    o = torch.empty(B, Hkv * G, M, D, dtype=torch.float16, device=DEV)
    kd, vd = k.to(DEV), v.to(DEV)
    modules.get("prefix", "cache", scale=1.0).forward(kd[:, :, P:], kd[0, :, :P], o, q.to(DEV), vd[:, :, P:], vd[0, :, :P], None, None)
    sees = torch.arange(P + S) <= (P + S - M + torch.arange(M))[:, None]
    _check(o, q, k, v, sees.expand(B, Hkv * G, M, P + S), True)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M, S, top", [(1, 9000, 128), (5, 3000, 60), (600, 1500, 40)])
def test_selected_blocks_of_which_the_first_has_nearly_all_weight(M, S, top, D):
    Hkv, G, block = 2, 4, 32
    q, k, v = _inputs(1, Hkv, M, 0, S, D, G)
    o = torch.empty(1, Hkv * G, M, D, dtype=torch.float16, device=DEV)
    bnd = torch.zeros(1, Hkv, -(-S // block), 2, D, dtype=torch.float16, device=DEV)
    sel = torch.zeros(1, Hkv, M, top, dtype=torch.int32, device=DEV)
    ops.cache_bounds(k.to(DEV), bnd, block)
    modules.get("sparse", "cache", top=top, sink=1, recent=2, block=block, scale=1.0).forward(k.to(DEV), o, q.to(DEV), v.to(DEV), bnd, None, None, sel)
    taken = torch.zeros(1, Hkv, M, -(-S // block) + 1, dtype=torch.bool).scatter_(3, sel.cpu().long().where(sel.cpu() >= 0, torch.tensor(-(-S // block))), True)[..., :-1]
    sees = taken.repeat_interleave(block, 3)[..., :S] & (torch.arange(S) <= (S - M + torch.arange(M))[:, None])
    assert sees[..., 0].all()
    _check(o, q, k, v, sees.repeat_interleave(G, 1), True)
