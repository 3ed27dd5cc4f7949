"""Layouts of an fp16 cache that a view may give: strides of axes that have one entry."""
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
