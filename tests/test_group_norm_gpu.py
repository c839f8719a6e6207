"""Group norm + activation on channels-last tensors (csrc/group_norm.hip) against the 64-bit restatement of
oracle/state_space_block.py, whose bounds follow the roundings of an fp32 computation term by term; gradients also against central
differences.  Shapes: one position, one channel a group, odd channel counts, more channels than a workgroup has threads, rows and
samples that are views of wider tensors."""
import pytest
import torch
from torch import nn

from oracle.state_space_block import close, group_norm_act as oracle

SLOPE = 0.2
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
gpu = pytest.mark.gpu


def _data(N, S, C, dt, seed=0, mean=0.3, std=1.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(N, S, C, generator=g) * std + mean).to(dt)
    w, b = torch.randn(C, generator=g) * 0.4 + 1, torch.randn(C, generator=g) * 0.3
    return x, w, b, torch.randn(N, S, C, generator=g).to(dt)


def _check(x, groups, w, b, dy, act, eps=1e-5, autocast=False):
    from nnuzoo_amd.group_norm import group_norm_act
    xc, wc, bc = (None if t is None else t.cuda().requires_grad_(True) for t in (x, w, b))
    with torch.autocast("cuda", dtype=torch.float16, enabled=autocast):
        y = group_norm_act(xc, groups, wc, bc, eps, act, SLOPE)
    assert y.dtype == (torch.float32 if autocast else x.dtype)
    dy = dy.to(y.dtype)
    y.backward(dy.cuda())
    N, C = x.shape[0], x.shape[-1]
    want = oracle(x.reshape(N, -1, C), groups, w, b, eps, act, SLOPE, dy.reshape(N, -1, C))
    assert xc.grad.dtype == x.dtype
    close(y.reshape(want["y"][0].shape), *want["y"], "y")
    close(xc.grad.reshape(want["dx"][0].shape), *want["dx"], "dx")
    if w is not None:
        assert wc.grad.dtype == w.dtype
        close(wc.grad, *want["dw"], "dw")
    if b is not None:
        close(bc.grad, *want["db"], "db")


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("act", ["none", "relu", "leaky_relu", "silu"])
@pytest.mark.parametrize("N,S,C,groups", [(2, 64, 32, 8), (3, 63, 60, 6), (1, 1, 8, 2), (2, 1, 7, 7), (1, 5, 1, 1), (2, 300, 24, 3),
                                          (1, 1000, 9, 3), (2, 17, 2050, 2)])
def test_against_64_bits(hip_lib, dt, act, N, S, C, groups):
    x, w, b, dy = _data(N, S, C, DT[dt], seed=S + C)
    _check(x, groups, w, b, dy, act)


@gpu
@pytest.mark.parametrize("N,S,C,groups", [(1, 20000, 16, 4), (5, 4099, 64, 1), (2, 130, 4096, 32), (70, 3, 12, 4), (1, 9000, 3, 1)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_many_workgroups(hip_lib, dt, N, S, C, groups):
    x, w, b, dy = _data(N, S, C, DT[dt], seed=C)
    _check(x, groups, w, b, dy, "silu")


@gpu
@pytest.mark.parametrize("N,S,C,groups", [(9, 16, 64, 8), (300, 4, 24, 3), (40, 30, 66, 1), (33, 64, 512, 2), (20, 400, 40, 1),
                                          (1000, 1, 8, 8), (9000, 2, 16, 2), (3000, 5, 60, 6), (12, 100, 600, 1)])
@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_many_small_samples(hip_lib, dt, N, S, C, groups):
    """waves and workgroups that walk several samples of a group, partial weight gradients added up after them"""
    x, w, b, dy = _data(N, S, C, DT[dt], seed=N)
    _check(x, groups, w, b, dy, "silu", eps=1e-2)


@gpu
def test_more_groups_than_a_grid_has_workgroups(hip_lib):
    """600 000 samples x 8 groups: past 2^22 workgroups each takes several groups"""
    x, w, b, dy = _data(600000, 2, 8, torch.float16, seed=14)
    _check(x, 8, w, b, dy, "silu", eps=1e-2)


@gpu
@pytest.mark.parametrize("affine", [(False, False), (True, False), (False, True)])
def test_without_affine_parameters(hip_lib, affine):
    x, w, b, dy = _data(2, 50, 16, torch.float32, seed=3)
    _check(x, 4, w if affine[0] else None, b if affine[1] else None, dy, "relu")


@gpu
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_autocast_gives_fp32(hip_lib, dt):
    x, w, b, dy = _data(2, 77, 32, DT[dt], seed=4)
    _check(x, 8, w, b, dy.float(), "relu", autocast=True)


@gpu
@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_large_mean_keeps_the_variance(hip_lib, dt):
    """mu / sigma = 1000 (fp32) and 60 (fp16): E[x^2] - mu^2 in fp32 would have nothing left of the variance"""
    x, w, b, dy = _data(2, 500, 16, DT[dt], seed=5, mean=1000.0 if dt == "f32" else 60.0, std=1.0)
    _check(x, 4, w, b, dy, "none")


@gpu
def test_half_precision_parameters_and_their_gradients(hip_lib):
    x, w, b, dy = _data(2, 40, 16, torch.float16, seed=6)
    _check(x, 4, w.half(), b.half(), dy, "silu")


@gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_views_of_wider_tensors(hip_lib, dt):
    g = torch.Generator().manual_seed(7)
    wide = torch.randn(3, 5, 7, 40, generator=g).to(DT[dt])
    w, b = torch.randn(16, generator=g), torch.randn(16, generator=g)
    for view in (wide[..., 8:24], wide[..., 3:19], wide[::2, :, :, 8:24], wide[:, :, ::2, 8:24], wide.transpose(1, 2)[..., :16],
                 wide[:, :1].expand(3, 5, 7, 40)[..., :16]):
        dy = torch.randn(view.shape, generator=g).to(DT[dt])
        from nnuzoo_amd.group_norm import group_norm_act
        base = wide.cuda().requires_grad_(True)
        idx = view
        # the same view of the device tensor
        dev = torch.as_strided(base, idx.shape, idx.stride(), idx.storage_offset())
        y = group_norm_act(dev, 4, w.cuda(), b.cuda(), 1e-5, "relu")
        dx, = torch.autograd.grad(y, dev, dy.cuda())
        want = oracle(view.reshape(view.shape[0], -1, 16), 4, w, b, 1e-5, "relu", SLOPE, dy.reshape(view.shape[0], -1, 16))
        close(y.reshape(want["y"][0].shape), *want["y"], "y")
        close(dx.reshape(want["dx"][0].shape), *want["dx"], "dx")


@gpu
def test_gradient_against_differences(hip_lib):
    """central differences of the operator itself: error h^2 |f'''| / 6 + 2^-24 |f| / h each, f = sum(y * dy)"""
    from nnuzoo_amd.group_norm import group_norm_act
    x, w, b, dy = (t.cuda() for t in _data(1, 6, 8, torch.float32, seed=8))
    f = lambda x_, w_, b_: (group_norm_act(x_, 2, w_, b_, 1e-5, "silu").double() * dy.double()).sum()  # noqa: E731
    ins = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(f(*ins), ins)
    h = 2.0 ** -7
    size = float((group_norm_act(x, 2, w, b, 1e-5, "silu").double() * dy.double()).abs().sum())
    for k, t in enumerate((x, w, b)):
        for i in range(0, t.numel(), 5):
            up, dn = [u.clone() for u in (x, w, b)], [u.clone() for u in (x, w, b)]
            up[k].view(-1)[i] += h
            dn[k].view(-1)[i] -= h
            step = float(up[k].view(-1)[i].double() - dn[k].view(-1)[i].double())
            num = float(f(*up) - f(*dn)) / step
            # third derivatives of these normalised sums stay below 8 in units of the sum's size
            assert abs(num - float(grads[k].view(-1)[i])) <= 8 * size * h * h / 6 + 16 * 2.0 ** -24 * size / h


@gpu
def test_nan_and_inf_stay_in_their_group(hip_lib):
    from nnuzoo_amd.group_norm import group_norm_act
    x, w, b, _ = _data(2, 30, 16, torch.float32, seed=9)
    x[0, 3, 5] = float("nan")
    x[1, 7, 0] = float("inf")
    for act in ("none", "relu", "leaky_relu", "silu"):
        y = group_norm_act(x.cuda(), 4, w.cuda(), b.cuda(), 1e-5, act).cpu()
        ref = torch.nn.functional.group_norm(x.transpose(1, 2), 4, w, b).transpose(1, 2)
        assert torch.isnan(y[0, :, 4:8]).all() and torch.isnan(y[1, :, :4]).all()
        assert torch.equal(torch.isnan(y), torch.isnan(ref))


@gpu
def test_constant_rows_and_empty_tensors(hip_lib):
    from nnuzoo_amd.group_norm import group_norm_act
    w, b = torch.full((8,), 2.0).cuda(), torch.arange(8.0).cuda()
    y = group_norm_act(torch.full((2, 9, 8), 3.25).cuda(), 2, w, b)
    assert torch.equal(y, b.expand(2, 9, 8))
    for shape in ((0, 9, 8), (2, 0, 8)):
        x = torch.zeros(shape).cuda().requires_grad_(True)
        wg = w.clone().requires_grad_(True)
        y = group_norm_act(x, 2, wg, b)
        y.sum().backward()
        assert y.shape == shape and x.grad.shape == shape and torch.equal(wg.grad, torch.zeros_like(w))


@gpu
def test_rows_without_spatial_axes_and_single_gradients(hip_lib):
    """x (N, C); gradients of x alone, of the parameters alone, of an expanded dy"""
    from nnuzoo_amd.group_norm import group_norm_act
    x, w, b, _ = _data(37, 1, 24, torch.float32, seed=13)
    dy = torch.full_like(x, 0.5)
    want = oracle(x, 3, w, b, 1e-5, "silu", SLOPE, dy)
    ins = [t.cuda() for t in (x[:, 0], w, b)]
    for need in ((0,), (1,), (2,), (1, 2), (0, 1, 2)):
        args = [t.clone().requires_grad_(i in need) for i, t in enumerate(ins)]
        y = group_norm_act(args[0], 3, args[1], args[2], 1e-5, "silu")
        close(y[:, None], *want["y"], "y")
        (y * 0.5).sum().backward()
        for i, name in enumerate(("dx", "dw", "db")):
            if i in need:
                close(args[i].grad.reshape(want[name][0].shape), *want[name], name)
            else:
                assert args[i].grad is None


@gpu
def test_bit_identical_runs_and_side_stream(hip_lib):
    from nnuzoo_amd.group_norm import group_norm_act
    x, w, b, dy = (t.cuda() for t in _data(2, 5000, 32, torch.float16, seed=10))

    def run():
        xs = [t.clone().requires_grad_(True) for t in (x, w, b)]
        y = group_norm_act(xs[0], 8, xs[1], xs[2], 1e-5, "silu")
        return [y.detach(), *torch.autograd.grad(y, xs, dy)]
    first = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = run()
    s.synchronize()
    for a, c, d in zip(first, second, run()):
        assert torch.equal(a, c) and torch.equal(a, d)


@gpu
def test_captured_and_replayed(hip_lib):
    from nnuzoo_amd.group_norm import group_norm_act
    x, w, b, dy = (t.cuda() for t in _data(2, 300, 32, torch.float32, seed=11))

    def step(x_):
        xr = x_.detach().requires_grad_(True)
        y = group_norm_act(xr, 8, w, b, 1e-5, "relu")
        return y.detach(), torch.autograd.grad(y, xr, dy)[0]
    static = x.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(static)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for k in range(3):
        fresh = torch.randn(x.shape, generator=torch.Generator().manual_seed(k)).cuda()
        static.copy_(fresh)
        graph.replay()
        want = step(fresh)
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want))


@gpu
def test_more_than_2_to_31_elements_apart(hip_lib):
    """two samples whose first elements lie 2^31 + 64 elements apart"""
    from nnuzoo_amd.group_norm import group_norm_act
    gap = 2 ** 31 + 64
    buf = torch.empty(gap + 64 * 16, dtype=torch.float16, device="cuda")
    view = buf.as_strided((2, 64, 16), (gap, 16, 1))
    x, w, b, dy = _data(2, 64, 16, torch.float16, seed=12)
    view.copy_(x.cuda())
    y = group_norm_act(view, 4, w.cuda(), b.cuda(), 1e-5, "relu")
    want = oracle(x, 4, w, b, 1e-5, "relu", SLOPE, dy)
    close(y, *want["y"], "y")


@gpu
def test_module_and_norm_act(hip_lib):
    """GroupNormAct has nn.GroupNorm's state_dict; norm_act takes the operator where the channels lie innermost, in whatever order the
    spatial axes do, keeps the layout, and leaves other layouts to the modules"""
    from nnuzoo_amd import backends
    from nnuzoo_amd.group_norm import GroupNormAct, norm_act
    torch.manual_seed(0)
    ref = nn.GroupNorm(4, 16).cuda()
    nn.init.normal_(ref.weight)
    nn.init.normal_(ref.bias)
    mod = GroupNormAct(4, 16, activation="relu").cuda()
    mod.load_state_dict(ref.state_dict())
    tokens = torch.randn(2, 6, 5, 7, 16, device="cuda")
    for x in (tokens.permute(0, 4, 1, 2, 3), tokens.permute(0, 4, 3, 1, 2), tokens.permute(0, 4, 1, 2, 3).contiguous()):
        want = torch.relu(ref.double()(x.double())).float()
        ref.float()
        backends.reset()
        got = norm_act(ref, nn.ReLU(inplace=True), x)
        hip = any(k[0] == "GroupNorm" and k[2] == "hip" for k in backends.COUNTS)
        assert hip == (not x.is_contiguous())
        assert got.stride() == x.stride() and got.shape == x.shape
        assert torch.allclose(got, want, rtol=1e-5, atol=1e-5)
        assert torch.allclose(mod(x), want, rtol=1e-5, atol=1e-5)
    hooked = nn.GroupNorm(4, 16).cuda()
    seen = []
    hooked.register_forward_hook(lambda *a: seen.append(1))
    norm_act(hooked, nn.SiLU(), tokens.permute(0, 4, 1, 2, 3))
    assert seen


@gpu
def test_refusals(hip_lib):
    from nnuzoo_amd._lib import HipCallError
    from nnuzoo_amd.group_norm import GroupNormAct, group_norm_act
    x, w, b = torch.zeros(2, 4, 8).cuda(), torch.zeros(8).cuda(), torch.zeros(8).cuda()
    with pytest.raises(ValueError, match="groups"):
        group_norm_act(x, 3, w, b)
    with pytest.raises(ValueError, match="groups"):
        group_norm_act(x, 0, w, b)
    with pytest.raises(ValueError, match="weight"):
        group_norm_act(x, 2, w[:4], b)
    with pytest.raises(ValueError, match="spatial"):
        group_norm_act(w, 2, w, b)
    with pytest.raises(NotImplementedError, match="activation"):
        group_norm_act(x, 2, w, b, activation="tanh")
    with pytest.raises(NotImplementedError, match="float32, float16 or bfloat16"):
        group_norm_act(x.double(), 2, w, b)
    with pytest.raises(NotImplementedError, match="4096"):
        group_norm_act(torch.zeros(1, 2, 8192).cuda(), 2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        group_norm_act(x, 2, w.cpu(), b)
    with pytest.raises(NotImplementedError, match="activation"):
        GroupNormAct(2, 8, activation="mish")
    # a gradient of the gradient: the first one is a value, the second an error, whichever of its sources asks for it
    xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, = torch.autograd.grad(group_norm_act(xr, 2, w, b), xr, torch.ones_like(x), create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        (dx.square().sum() + xr.sum()).backward()
    dx, = torch.autograd.grad(group_norm_act(xr, 2, wr, b), xr, torch.ones_like(x), create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(dx.sum(), wr)
    assert issubclass(HipCallError, RuntimeError)


def test_refuses_cpu_tensors_and_bad_calls_without_a_gpu():
    from nnuzoo_amd import _lib
    from nnuzoo_amd.group_norm import GroupNormAct, group_norm_act
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        group_norm_act(torch.zeros(2, 4, 8), 2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        GroupNormAct(2, 8)(torch.zeros(2, 8, 3, 3))
    lib = _lib.load()
    assert lib.nnz_group_norm_act_workspace_bytes(0, 4, 8, 2, 0) == -22
    assert lib.nnz_group_norm_act_workspace_bytes(2, 4, 8, 3, 0) == -22
    assert lib.nnz_group_norm_act_workspace_bytes(2, 4, 8192, 2, 1) == -22
    assert lib.nnz_group_norm_act_workspace_bytes(2, 100000, 8, 2, 1) > 0
    assert lib.nnz_group_norm_act_forward(None, 0, 0, 0, None, None, None, 0, None, None, 0, 2, 4, 8, 2, 1e-5, 0, 0.0, None) == -22


def test_norm_act_leaves_cpu_modules_alone():
    from nnuzoo_amd.group_norm import norm_act
    norm, act, x = nn.GroupNorm(2, 8), nn.ReLU(), torch.randn(2, 8, 3, 3).to(memory_format=torch.channels_last)
    assert torch.equal(norm_act(norm, act, x), act(norm(x)))
