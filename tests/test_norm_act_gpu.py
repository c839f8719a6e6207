"""norm_act (nnuzoo_amd/group_norm.py) takes the place of two module calls: what a caller could do with those - hooks registered for all
modules, forward-mode derivatives, vmap, second derivatives - gives the modules' results on token-major inputs, too."""
import pytest
import torch
from torch import nn

gpu = pytest.mark.gpu
ACTS = [nn.ReLU(inplace=True), nn.SiLU(), nn.LeakyReLU(0.2), nn.Identity()]


def _case(dtype=torch.float32):
    torch.manual_seed(0)
    norm = nn.GroupNorm(4, 16).cuda()
    nn.init.normal_(norm.weight)
    nn.init.normal_(norm.bias)
    return norm, torch.randn(2, 6, 5, 16, device="cuda", dtype=dtype).permute(0, 3, 1, 2)


@gpu
@pytest.mark.parametrize("register", ["register_module_forward_hook", "register_module_forward_pre_hook",
                                      "register_module_full_backward_hook", "register_module_full_backward_pre_hook"])
def test_hooks_of_all_modules(hip_lib, register):
    from nnuzoo_amd.group_norm import norm_act
    norm, x = _case()
    seen = []
    handle = getattr(nn.modules.module, register)(lambda mod, *a: seen.append(type(mod).__name__))
    try:
        norm_act(norm, nn.SiLU(), x.clone().requires_grad_(True)).sum().backward()
    finally:
        handle.remove()
    assert sorted(seen) == ["GroupNorm", "SiLU"]
