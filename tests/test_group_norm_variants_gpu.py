"""The variants of the group norm operator (csrc/group_norm.hip) that large groups take: vectors that span two groups or several, in every
pair of types; more (sample, group) pairs than a launch has teams."""
import pytest
import torch

from oracle.state_space_block import close, group_norm_act as oracle
from test_group_norm_gpu import DT, SLOPE, _check, _data

gpu = pytest.mark.gpu

# (N, S, C, groups): S C / groups is above 16 384, where the workgroups walk whole rows
LARGE = [(2, 9000, 32, 8),       # 4 channels a group: half a vector of 8, a whole one of 4
         (2, 8000, 24, 8),       # 3: vectors over several groups, borders inside
         (2, 4000, 48, 8),       # 6
         (2, 6000, 12, 4),       # 3, and 12 channels are no multiple of 8
         (2, 9000, 16, 8),       # 2
         (2, 3000, 64, 8),       # 8: vectors within a group
         (1, 17000, 8, 8),       # one channel a group
         (2, 3400, 25, 5)]        # odd channels: one at a time


@gpu
@pytest.mark.parametrize("act", ["relu", "silu"])
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("N,S,C,groups", LARGE)
def test_large_groups(hip_lib, dt, act, N, S, C, groups):
    x, w, b, dy = _data(N, S, C, DT[dt], seed=C + S)
    _check(x, groups, w, b, dy, act)


@gpu
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("N,S,C,groups", LARGE)
def test_large_groups_under_autocast(hip_lib, dt, N, S, C, groups):
    x, w, b, dy = _data(N, S, C, DT[dt], seed=C)
    _check(x, groups, w, b, dy.float(), "relu", autocast=True)


@gpu
def test_more_pairs_than_a_launch_has_teams(hip_lib):
    """33.6 million (sample, group) pairs on 2^22 workgroups of 8 waves: the last samples are their waves' second ones"""
    from nnuzoo_amd.group_norm import group_norm_act
    N, S, C = 4200000, 2, 8
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(N, S, C, generator=gen, device="cuda").half().requires_grad_(True)
    w, b = (torch.randn(C, generator=gen, device="cuda") for _ in range(2))
    dy = torch.randn(N, S, C, generator=gen, device="cuda").half()
    y = group_norm_act(x, 8, w, b, 1e-2, "silu")
    dx, = torch.autograd.grad(y, x, dy)
    for part in (slice(0, 1000), slice(N - 7000, N)):
        want = oracle(x[part].detach(), 8, w, b, 1e-2, "silu", SLOPE, dy[part])
        close(y[part], *want["y"], "y")
        close(dx[part], *want["dx"], "dx")


@gpu
def test_many_channels_after_a_call_with_few(hip_lib):
    """4 096 channels take more than 64 KB of LDS; calls of other element types with few channels in between change nothing"""
    wide = _data(1, 200, 4096, torch.bfloat16, seed=20)
    few = _data(2, 9000, 32, torch.bfloat16, seed=21)
    for groups, autocast in ((32, False), (32, True)):
        _check(*wide[:1], groups, *wide[1:3], wide[3].float() if autocast else wide[3], "none", autocast=autocast)
        for g in (8, 4):
            _check(*few[:1], g, *few[1:3], few[3].float(), "none", autocast=True)
            _check(*few[:1], g, *few[1:3], few[3], "none")
        _check(*wide[:1], groups, *wide[1:3], wide[3].float() if autocast else wide[3], "none", autocast=autocast)


@gpu
@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("N,S,C,groups", [(2, 1024, 32, 8), (2, 1025, 32, 8), (2, 4096, 32, 8),        # rows of a group
                                          (32, 512, 32, 8), (33, 512, 32, 8), (600, 300, 32, 8),       # row segments altogether
                                          (3, 129, 32, 8), (8, 128, 32, 8), (9, 128, 32, 8), (33, 256, 32, 8), (12, 102, 60, 6),  # waves
                                          (1, 7, 16, 2), (4, 7, 16, 2), (5, 7, 16, 2)])                # teams of a group
def test_on_both_sides_of_the_borders(hip_lib, dt, N, S, C, groups):
    x, w, b, dy = _data(N, S, C, DT[dt], seed=N + S)
    _check(x, groups, w, b, dy, "leaky_relu")
