"""What a step keeps between calls where a serving loop gives it any number of tokens; needs no GPU."""
import pytest
import torch

from triton_amd import modules


@pytest.mark.parametrize("variant, form, kw", [("vanilla", "cache8", {}), ("weights", "cache8", {}), ("prefix", "cache16", {}), ("sparse", "cache16", dict(top=4))])
def test_projections_of_any_length_share_workspaces(monkeypatch, variant, form, kw):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    step = modules.get(variant, form, head_dim=64, **kw)
    cols, most = 6144, 4000
    for rows in [0, 1, *range(5, most + 1, 37), most]:
        t = step._rows("qkv", rows, cols, torch.float16, torch.device("cpu"))
        assert t.shape == (rows, cols) and t.is_contiguous()
    held = [x.numel() * x.element_size() for x in step._ws.values()]
    assert len(held) <= 8 and sum(held) <= 4 * most * cols * 2
    # the next call of a size finds what the last one had
    assert step._rows("qkv", most, cols, torch.float16, torch.device("cpu")).data_ptr() == t.data_ptr()
