"""Calls of the group norm operator (nnuzoo_amd/group_norm.py) beside the plain ones: derivatives that it does not have or need not make."""
import pytest
import torch

from test_group_norm_gpu import _data

gpu = pytest.mark.gpu


@gpu
def test_second_derivatives_of_copied_layouts_are_refused(hip_lib):
    """an input whose rows have to be gathered first: a second derivative in x is an error there, too, never a missing term"""
    from nnuzoo_amd.group_norm import group_norm_act
    x = torch.randn(2, 8, 6, device="cuda").requires_grad_(True)
    dx, = torch.autograd.grad(group_norm_act(x.transpose(1, 2), 2), x, torch.ones(2, 6, 8, device="cuda"), create_graph=True)
    assert dx.requires_grad
    with pytest.raises(RuntimeError, match="no second derivative"):
        (dx.square().sum() + x.sum()).backward()
