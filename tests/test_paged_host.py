"""Host side of the paged cache's and rotary calls, without a GPU."""

import pytest
import torch

import foveated_kv_b200 as fkv


def _step():
    """A small append on host tensors (its gradients are looked at first)."""
    rows = lambda h: torch.zeros(2, h, 64, dtype=torch.float16)
    pages = torch.zeros(3, 2, 16, 64, dtype=torch.float16)
    return dict(k=rows(2), v=rows(2), k_pages=pages, v_pages=pages.clone(), table=torch.zeros(2, 2, dtype=torch.int32),
                lens=torch.ones(2, dtype=torch.int32), q=rows(4), inv_freq=torch.zeros(32, dtype=torch.float64))


@pytest.mark.parametrize("name", ["k", "v", "q", "inv_freq"])
def test_gradients_are_refused(name):
    kw = _step()
    kw[name].requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        fkv.paged_append(**kw)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        fkv.paged_append(**kw)
    kw, ad = _step(), torch.autograd.forward_ad
    with ad.dual_level():
        kw[name] = ad.make_dual(kw[name], torch.ones_like(kw[name]))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(ValueError, match="forward gradient"):
                fkv.paged_append(**kw)
    with pytest.raises(ValueError, match="CUDA"):                # the tangent is gone with its level
        fkv.paged_append(**kw)
