"""Positions behind a shared prefix, what needs no GPU: the append's offset and the step that adds a prefix's keys by itself."""
import pytest
import torch

from test_cache16_host import M, P, _rope, lib, no_gpu  # noqa: F401
from triton_amd import modules


@no_gpu
def test_offset_statuses(lib):  # noqa: F811
    for offset in (1, -7, 2 ** 31 - 1, -2 ** 31):
        assert _rope(lib, offset=offset) == "TRN_E_LAUNCH", offset                # all is well, but for the GPU
    assert _rope(lib, offset=1, positions=P + 7 * M) == "TRN_E_UNSUPPORTED" and _rope(lib, positions=P + 7 * M) == "TRN_E_LAUNCH"


def _step(prefix, **kw):
    """A step's call, which is refused for its X before anything is launched."""
    h = lambda *s: torch.zeros(*s, dtype=torch.float16)
    step = modules.get("prefix", "cache16", head_dim=64, **kw)
    t = dict(K_cache=h(1, 2, 8, 64), K_prefix=h(2, prefix, 64), O2=h(1, 2, 256), V_cache=h(1, 2, 8, 64), V_prefix=h(2, prefix, 64), WK=h(96, 128), WQ=h(96, 256), WV=h(96, 128), X=h(2, 96),
             inv_freq=torch.zeros(32, dtype=torch.float64))
    for _ in range(2):
        with pytest.raises(ValueError):
            step.forward(*(t.get(n) for n in step.TENSOR_PARAMS))


@pytest.mark.filterwarnings("error")
def test_positions_behind_a_prefix_are_asked_for():
    for said in (True, False):
        _step(5, after_prefix=said)
    _step(0)
    with pytest.warns(UserWarning, match="after_prefix=True") as seen:
        _step(5)
    assert len(seen) == 1
    assert modules.get("prenorm", "cache16", head_dim=64, after_prefix=True).after_prefix and modules.get("prefix", "cache16", head_dim=64).after_prefix is None
