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


@gpu
@pytest.mark.parametrize("act", ACTS, ids=lambda a: type(a).__name__)
def test_forward_mode_and_vmap(hip_lib, act):
    from nnuzoo_amd.group_norm import norm_act
    norm, x = _case()
    v, w = torch.randn_like(x), norm.weight.detach()

    def with_weight(f):
        class Both(nn.Module):
            def __init__(self):
                super().__init__()
                self.norm = norm

            def forward(self, t):
                return f(t)
        return lambda u: torch.func.functional_call(Both(), {"norm.weight": u}, (x,))
    ours, mods = (lambda t: norm_act(norm, act, t)), (lambda t: act(norm(t)))
    for f, g, at, d in ((ours, mods, x, v), (with_weight(ours), with_weight(mods), w, torch.ones_like(w))):
        for a, b in zip(torch.func.jvp(f, (at,), (d,)), torch.func.jvp(g, (at,), (d,))):
            assert torch.equal(a, b)
        many = torch.stack((at, d))
        assert torch.equal(torch.func.vmap(f)(many), torch.func.vmap(g)(many))
    with torch.autograd.forward_ad.dual_level():
        a, b = (torch.autograd.forward_ad.unpack_dual(f(torch.autograd.forward_ad.make_dual(x, v))) for f in (ours, mods))
        assert torch.equal(a.primal, b.primal) and torch.equal(a.tangent, b.tangent)
