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


@gpu
@pytest.mark.parametrize("act", ACTS, ids=lambda a: type(a).__name__)
def test_second_derivatives(hip_lib, act):
    """a gradient penalty through token-major activations: the modules' second derivatives, in x, dy and both parameters.  Both sides are
    fp32 computations of sums over 120 terms in different orders: 1e-4 of the largest value is 2^10 roundings"""
    from nnuzoo_amd import backends
    from nnuzoo_amd.group_norm import norm_act
    norm, x = _case()
    dy = torch.randn_like(x).requires_grad_(True)
    out = []
    for f in (lambda t: norm_act(norm, act, t), lambda t: act(norm(t))):
        backends.reset()
        xr = x.clone().requires_grad_(True)
        ins = (xr, norm.weight, norm.bias)
        first = torch.autograd.grad(f(xr), ins, dy, create_graph=True)
        out.append((first, torch.autograd.grad(sum(g.square().sum() for g in first), (*ins, dy), allow_unused=True),
                    any(k[2] == "hip" for k in backends.COUNTS)))
    assert out[0][2] and not out[1][2]          # the operator ran on the one side, the modules on the other
    for got, want in zip(out[0][:2], out[1][:2]):
        for a, b in zip(got, want):
            assert (a is None) == (b is None)
            if a is not None:
                assert float((a - b).abs().max()) <= 1e-4 * float(b.abs().max())
