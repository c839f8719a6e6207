"""Dropout from a counter-based generator (csrc/dropout.hip): masks equal, element by element, to an independent numpy restatement of
the generator (itself pinned by published known answers), values equal to fp32 arithmetic with one rounding."""
import numpy as np
import pytest
import torch

from oracle.state_space_block import close, dropout_draws, dropout_kept, philox4x32

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
gpu = pytest.mark.gpu
U = 2.0 ** -24


def test_generator_gives_its_published_known_answers():
    kat = [([0] * 4, [0] * 2, [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]),
           ([0xffffffff] * 4, [0xffffffff] * 2, [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]),
           ([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0], [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1])]
    for ctr, key, want in kat:
        got = philox4x32(np.array([ctr], dtype=np.uint64), np.array([key], dtype=np.uint64))[0]
        assert [int(v) for v in got] == want


def _check(n_shape, dt, p, seed, step, site, residual=None, offset=0):
    from nnuzoo_amd.dropout import dropout, dropout_add, dropout_state
    g = torch.Generator().manual_seed(1)
    numel = int(np.prod(n_shape))
    x = torch.randn(numel + offset, generator=g).to(DT[dt])[offset:].reshape(n_shape)
    state = dropout_state(seed, "cuda", step)
    buf = torch.empty(numel + offset, dtype=x.dtype, device="cuda")
    xc = buf[offset:].view(n_shape).copy_(x).detach().requires_grad_(True)
    kept = dropout_kept(seed & (2 ** 64 - 1), step, site, numel, p).view(n_shape)
    scale = torch.tensor(1.0 / (1.0 - p) if p < 1 else 1.0, dtype=torch.float32)
    drop = lambda t: torch.where(kept, t.float() * scale, torch.zeros((), dtype=torch.float32))  # noqa: E731
    if residual is None:
        y = dropout(xc, p, state, site)
        assert torch.equal(y.cpu(), drop(x).to(x.dtype))
    else:
        r = torch.randn(n_shape, generator=g).to(DT[residual])
        rc = r.cuda().requires_grad_(True)
        y = dropout_add(xc, rc, p, state, site)
        assert y.dtype == torch.promote_types(x.dtype, r.dtype)
        v = torch.where(kept, x.double() / (1 - p) if p < 1 else 0.0, 0.0)
        close(y, v + r.double(), 3 * U * (v.abs() + r.double().abs()), "y")
    dy = torch.randn(n_shape, generator=g).to(y.dtype)
    grads = torch.autograd.grad(y, [xc] if residual is None else [xc, rc], dy.cuda())
    assert torch.equal(grads[0].cpu(), drop(dy).to(x.dtype))
    if residual is not None:
        assert torch.equal(grads[1].cpu(), dy.to(r.dtype))


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 5, 67), (64, 513), (70001,)])
@pytest.mark.parametrize("p", [0.1, 0.5, 0.999])
def test_mask_and_values(hip_lib, dt, shape, p):
    _check(shape, dt, p, 12345, 6, 3)


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("residual", list(DT))
def test_residual(hip_lib, dt, residual):
    _check((33, 65), dt, 0.3, -7, 2 ** 32 - 1, 2 ** 31 - 1, residual)


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("offset", [1, 2, 4])
def test_unaligned(hip_lib, dt, offset):
    _check((1234,), dt, 0.25, 2 ** 63 + 11, 0, 0, offset=offset)


@gpu
@pytest.mark.parametrize("residual", [None, "f32"])
def test_p_of_0_and_1(hip_lib, residual):
    _check((1000,), "f32", 1.0, 3, 3, 3, residual)
    if residual:
        _check((1000,), "f16", 0.0, 3, 3, 3, residual)


@gpu
def test_ties_of_the_upper_halves_use_the_lower_ones(hip_lib):
    """thresholds on both sides of an element's own 32-bit draw: its upper half equals the threshold's, the lower half decides"""
    from nnuzoo_amd.dropout import dropout, dropout_state
    draws = dropout_draws(99, 1, 4, 0, 4096)
    state = dropout_state(99, "cuda", 1)
    x = torch.ones(4096, device="cuda")
    for e in (0, 5, 17, 2047, 4095):
        for d in (0, 1):
            p = (int(draws[e]) + d) / 2 ** 32
            got = dropout(x, p, state, 4).cpu() != 0
            assert torch.equal(got, draws >= int(draws[e]) + d)
            assert bool(got[e]) == (d == 0)


@gpu
def test_share_and_independence(hip_lib):
    """2^24 draws: the share of dropped elements within 5 standard deviations; other steps, sites and seeds give other masks that
    agree with the first as independent ones do"""
    from nnuzoo_amd.dropout import advance, dropout, dropout_state
    n, p = 1 << 24, 0.1
    x = torch.ones(n, device="cuda")
    state = dropout_state(5, "cuda")
    base = dropout(x, p, state, 0) == 0
    sd = (p * (1 - p) / n) ** 0.5
    assert abs(float(base.double().mean()) - p) < 5 * sd
    masks = [dropout(x, p, state, 1) == 0, dropout(x, p, dropout_state(6, "cuda"), 0) == 0]
    advance(state)
    masks.append(dropout(x, p, state, 0) == 0)
    both = (p * p * (1 - p * p) / n) ** 0.5
    for m in masks:
        assert abs(float((m & base).double().mean()) - p * p) < 5 * both
    assert abs(float((base[1:] & base[:-1]).double().mean()) - p * p) < 5 * both


@gpu
def test_mask_is_the_same_for_every_type_and_layout(hip_lib):
    from nnuzoo_amd.dropout import dropout, dropout_state
    state = dropout_state(8, "cuda")
    want = dropout(torch.ones(12, 10, device="cuda"), 0.4, state) != 0
    for dt in DT.values():
        assert torch.equal(dropout(torch.ones(12, 10, device="cuda", dtype=dt), 0.4, state) != 0, want)
    assert torch.equal(dropout(torch.ones(10, 12, device="cuda").t(), 0.4, state) != 0, want)


@gpu
def test_dropped_infinities_are_zero(hip_lib):
    from nnuzoo_amd.dropout import dropout, dropout_state
    x = torch.full((1000,), float("inf"), device="cuda")
    x[::2] = float("nan")
    y = dropout(x, 0.5, dropout_state(1, "cuda"))
    kept = dropout_kept(1, 0, 0, 1000, 0.5).cuda()
    assert torch.equal(torch.isfinite(y), ~kept) and torch.equal(y == 0, ~kept)


@gpu
def test_backward_uses_the_pair_of_its_forward(hip_lib):
    from nnuzoo_amd.dropout import advance, dropout, dropout_state
    state = dropout_state(4, "cuda")
    x = torch.ones(500, device="cuda", requires_grad=True)
    y = dropout(x, 0.5, state)
    advance(state)
    state[0] = 77
    dx, = torch.autograd.grad(y.sum(), x)
    assert torch.equal(dx, y.detach())


@gpu
def test_gradient_against_differences(hip_lib):
    """the operator is linear in x: differences are exact up to roundings"""
    from nnuzoo_amd.dropout import dropout_add, dropout_state
    state = dropout_state(21, "cuda")
    g = torch.Generator().manual_seed(2)
    x, r, dy, v = (torch.randn(300, generator=g).cuda() for _ in range(4))
    x.requires_grad_(True)
    dx, = torch.autograd.grad(dropout_add(x, r, 0.3, state), x, dy)
    with torch.no_grad():
        num = ((dropout_add(x + v, r, 0.3, state).double() - dropout_add(x, r, 0.3, state).double()) * dy.double()).sum()
        size = ((x.abs() + v.abs() + r.abs()) / 0.7 * dy.abs()).double().sum()
    assert abs(float(num) - float((dx.double() * v.double()).sum())) <= 8 * U * float(size)


@gpu
def test_captured_graph_draws_anew(hip_lib):
    from nnuzoo_amd.dropout import advance, dropout, dropout_state
    state = dropout_state(31, "cuda")
    x = torch.ones(5000, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        dropout(x, 0.5, state)
        advance(state)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dropout(x, 0.5, state)
        advance(state)
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal((y != 0).cpu(), dropout_kept(31, 1 + k, 0, 5000, 0.5))
        dropout(x, 0.5, state)      # eager work in between
    assert int(state[1]) == 4


@gpu
def test_elements_past_2_to_32(hip_lib):
    """blocks whose number passes 2^29, elements past 2^32: the last ones of a 4.3 GB call"""
    from nnuzoo_amd.dropout import dropout, dropout_state
    n = 2 ** 32 + 1000
    x = torch.ones(n, dtype=torch.float16, device="cuda")
    y = dropout(x, 0.5, dropout_state(13, "cuda"))
    assert torch.equal((y[-1000:] != 0).cpu(), dropout_kept(13, 0, 0, 1000, 0.5, first=2 ** 32))
    assert torch.equal((y[:1000] != 0).cpu(), dropout_kept(13, 0, 0, 1000, 0.5))


@gpu
def test_module_and_evaluation(hip_lib):
    from nnuzoo_amd.dropout import Dropout, dropout, dropout_add, dropout_state
    state = dropout_state(2, "cuda")
    m = Dropout(0.3, state, site=5)
    x, r = torch.randn(4, 9, device="cuda"), torch.randn(4, 9, device="cuda")
    assert torch.equal(m(x), dropout(x, 0.3, state, 5)) and torch.equal(m(x, r), dropout_add(x, r, 0.3, state, 5))
    m.eval()
    assert m(x) is x and torch.equal(m(x, r), x + r)
    assert dropout(x, 0.0, state) is x


@gpu
def test_gradient_of_the_residual_alone_and_of_one_tensor_twice(hip_lib):
    from nnuzoo_amd.dropout import dropout_add, dropout_state
    state = dropout_state(2, "cuda")
    x, r = torch.randn(70, device="cuda"), torch.randn(70, device="cuda", requires_grad=True)
    dr, = torch.autograd.grad(dropout_add(x, r, 0.5, state).sum(), r)
    assert torch.equal(dr, torch.ones_like(r))
    both, = torch.autograd.grad(dropout_add(r, r, 0.5, state).sum(), r)
    kept = dropout_kept(2, 0, 0, 70, 0.5).cuda()
    assert torch.equal(both, torch.where(kept, 3.0, 1.0))
    view = torch.randn(4, 6, device="cuda").t()                       # gradients of strided inputs and outputs
    v = view.clone().requires_grad_(True)
    y = dropout_add(v.t(), v.t(), 0.5, state)
    y.t().backward(torch.ones(6, 4, device="cuda"))
    assert torch.equal(v.grad, torch.where(dropout_kept(2, 0, 0, 24, 0.5).view(4, 6).cuda(), 3.0, 1.0).t())


@gpu
def test_empty(hip_lib):
    from nnuzoo_amd.dropout import dropout, dropout_add, dropout_state
    x = torch.zeros(0, 4, device="cuda", requires_grad=True)
    state = dropout_state(2, "cuda")
    dropout(x, 0.5, state).sum().backward()
    assert x.grad.shape == (0, 4)
    assert dropout_add(x, x, 0.5, state).shape == (0, 4)


@gpu
def test_refusals(hip_lib):
    from nnuzoo_amd._lib import HipCallError
    from nnuzoo_amd.dropout import Dropout, dropout, dropout_add, dropout_state
    x, state = torch.zeros(4, 4).cuda(), dropout_state(0, "cuda")
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="p must"):
            dropout(x, p, state)
        with pytest.raises(ValueError, match="p must"):
            Dropout(p, state, 0)
    with pytest.raises(ValueError, match="site"):
        dropout(x, 0.5, state, -1)
    with pytest.raises(ValueError, match="differ in shape"):
        dropout_add(x, x[:1], 0.5, state)
    with pytest.raises(HipCallError, match="state"):
        dropout(x, 0.5, state.int())
    with pytest.raises(HipCallError, match="state"):
        dropout(x, 0.5, torch.zeros(3, dtype=torch.int64).cuda())
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        dropout(x, 0.5, state.cpu())
    with pytest.raises(NotImplementedError, match="float32"):
        dropout(x.double(), 0.5, state)
    xr, dy = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(dropout(xr, 0.5, state), xr, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        dx.sum().backward()


def test_refuses_cpu_tensors_and_bad_calls_without_a_gpu():
    from nnuzoo_amd import _lib
    from nnuzoo_amd.dropout import dropout, dropout_add, dropout_state
    x = torch.zeros(4)
    for f in (lambda: dropout(x, 0.5, dropout_state(0, "cpu")), lambda: dropout(x, 0.0, dropout_state(0, "cpu")),
              lambda: dropout_add(x, x, 0.5, dropout_state(0, "cpu"))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f()
    with pytest.raises(ValueError, match="p must"):
        dropout(x, 2.0, dropout_state(0, "cpu"))
    assert dropout_state(2 ** 64 - 1, "cpu", 5).tolist() == [-1, 5]
    lib = _lib.load()
    assert lib.nnz_dropout_forward(None, 0, None, 0, None, 8, 1, 1.0, 0, None, None, None) == -22
    assert lib.nnz_dropout_forward(16, 0, None, 0, 16, 8, 2 ** 32 + 1, 1.0, 0, 16, None, None) == -22
    assert lib.nnz_dropout_forward(16, 3, None, 0, 16, 8, 1, 1.0, 0, 16, None, None) == -22
    assert lib.nnz_dropout_backward(16, 0, 16, 7, 8, 1, 1.0, 0, 16, None) == -22
