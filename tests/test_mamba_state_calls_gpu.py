"""Calls of the state-carrying scan and convolution (nnuzoo_amd/mamba_state.py) that a user may make beside the plain ones: derivatives that
the operators do not have, decays at the ends of their range, more sequences than a launch has rows."""
import pytest
import torch

from test_mamba_state_gpu import _conv_data, _scan_data

gpu = pytest.mark.gpu


def _four(v):
    from nnuzoo_amd import mamba_state as ms
    return {
        "causal_conv1d_prompt": lambda: ms.causal_conv1d_prompt(v["x"], v["w"], v["b"], conv_state=v["cs"]),
        "causal_conv1d_token": lambda: ms.causal_conv1d_token(v["x"][:, 0], v["cs"], v["w"], v["b"]),
        "selective_scan_prompt": lambda: ms.selective_scan_prompt(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], z=v["z"],
                                                                  dt_bias=v["dt_bias"], state=v["state"]),
        "selective_scan_token": lambda: ms.selective_scan_token(v["x"][:, 0], v["dt"][:, 0], v["A"], v["B"][:, 0], v["C"][:, 0], v["D"],
                                                                z=v["z"][:, 0], dt_bias=v["dt_bias"], state=v["state"])}


@gpu
@pytest.mark.parametrize("name", ["causal_conv1d_prompt", "causal_conv1d_token", "selective_scan_prompt", "selective_scan_token"])
def test_forward_mode_derivatives_are_refused(hip_lib, name):
    """an input with a tangent - of any argument, also without gradient recording - is an error, not an output without a tangent"""
    from torch.autograd import forward_ad as fw
    v = {k: t.cuda() for k, t in _scan_data(2, 5, 8, 8, 1, 16, "f32", seed=1).items()}
    x, w, b, cs = _conv_data(2, 5, 8, 4, "f32", seed=2)
    v.update(w=w.cuda(), b=b.cuda(), cs=cs.cuda())
    _four(v)[name]()
    args = ("x", "w", "b", "cs") if "conv" in name else ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "state")
    for arg in args:
        with fw.dual_level():
            dual = dict(v, **{arg: fw.make_dual(v[arg], torch.ones_like(v[arg]))})
            for mode in (torch.enable_grad(), torch.no_grad()):
                with mode, pytest.raises(RuntimeError, match="forward-mode"):
                    _four(dual)[name]()
    for transform in (lambda f: torch.func.jvp(f, (v["x"],), (v["x"],)), lambda f: torch.func.vmap(f)(torch.stack((v["x"], v["x"])))):
        with pytest.raises(RuntimeError):
            transform(lambda t: _four(dict(v, x=t))[name]())


@gpu
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("L", [1, 40, 300, 2500])
def test_log_decays_of_minus_infinity_are_decays_of_zero(hip_lib, per_head, L):
    """A_is_log with log(-A) = -inf: the state is never damped, as with A = 0; NaN stays NaN"""
    from nnuzoo_amd.mamba_state import selective_scan_prompt, selective_scan_token
    v = {k: t.cuda() for k, t in _scan_data(2, L, 8, 8, 1, 16, "f32", seed=L, per_head=per_head).items()}
    v["A"][::2] = 0.0
    out = []
    for log in (False, True):
        st = v["state"].clone()
        a = torch.log(-v["A"]) if log else -torch.exp(torch.log(-v["A"]))
        kw = dict(z=v["z"], dt_bias=v["dt_bias"], dt_softplus=True, state=st, A_is_log=log)
        y = selective_scan_prompt(v["x"], v["dt"], a, v["B"], v["C"], v["D"], **kw)
        kw["z"] = v["z"][:, 0]
        t = selective_scan_token(v["x"][:, 0], v["dt"][:, 0], a, v["B"][:, 0], v["C"][:, 0], v["D"], **kw)
        out.append((y[:, :, ::2], t[:, ::2], st[:, ::2]))
    for a, b in zip(*out):
        assert torch.equal(a, b)
    a = torch.log(-v["A"])
    a[1] = float("nan")
    st = v["state"].clone()
    y = selective_scan_prompt(v["x"], v["dt"], a, v["B"], v["C"], v["D"], dt_bias=v["dt_bias"], dt_softplus=True, state=st, A_is_log=True)
    assert bool(torch.isnan(y[:, :, 1]).all()) and bool(torch.isfinite(y[:, :, ::2]).all())


@gpu
def test_sequences_past_a_grid_are_refused_by_name(hip_lib):
    from nnuzoo_amd.mamba_state import selective_scan_prompt, selective_scan_token
    z = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    B = 65536
    with pytest.raises(NotImplementedError, match="65535 sequences"):
        selective_scan_prompt(z(B, 2, 4), z(B, 2, 4), z(4, 4), z(B, 2, 4), z(B, 2, 4))
    assert selective_scan_prompt(z(B - 1, 2, 4), z(B - 1, 2, 4), z(4, 4), z(B - 1, 2, 4), z(B - 1, 2, 4)).shape == (B - 1, 2, 4)
    assert selective_scan_token(z(B, 4), z(B, 4), z(4, 4), z(B, 4), z(B, 4), state=z(B, 4, 4)).shape == (B, 4)
