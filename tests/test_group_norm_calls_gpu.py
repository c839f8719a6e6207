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


@gpu
@pytest.mark.parametrize("S", [300, 40000])
def test_parameter_gradients_alone_make_no_input_gradient(hip_lib, S):
    """behind a frozen part of a network: neither memory nor a pass for the gradient of x, and the same parameter gradients"""
    from nnuzoo_amd.group_norm import group_norm_act
    x, w, b, dy = (t.cuda() for t in _data(2, S, 32, torch.float32, seed=30))
    grads = []
    for frozen in (False, True):
        xr, wr, br = x.clone().requires_grad_(not frozen), w.clone().requires_grad_(True), b.clone().requires_grad_(True)
        y = group_norm_act(xr, 8, wr, br, 1e-5, "silu")
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        grads.append(torch.autograd.grad(y, (wr, br), dy))
        peak = torch.cuda.max_memory_allocated() - before
    assert peak < x.numel() * 4
    for a, c in zip(*grads):
        assert torch.equal(a, c)
