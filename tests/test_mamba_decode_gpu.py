"""Decoding with the Mamba and Mamba2 blocks (nnuzoo_amd/nets/mamba_simple.py, mamba2.py) on the state-carrying operators: prompts and
single tokens against the outputs that the reference's own module gave for the whole sequence (tests/golden/mamba_block.npz) and
those of an independent Mamba2 (tests/golden/mamba2_mixer.npz), at the tolerances of the whole-sequence tests; ragged prompts against
each sequence on its own; the group norm of a residual Mamba block in its place."""
import os
from types import SimpleNamespace

import numpy as np
import pytest
import torch
from torch import nn

GOLDEN = os.path.join(os.path.dirname(__file__), "golden")
gpu = pytest.mark.gpu


def _close(got, want, tol, what):
    want = torch.as_tensor(want)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if want.numel():
        err = (got.detach().cpu().float() - want).abs().max().item()
        assert err <= tol * (want.abs().max().item() + 1e-12), f"{what}: {err:.3e}"


def _mamba():
    from nnuzoo_amd.nets.mamba_simple import Mamba
    z = np.load(os.path.join(GOLDEN, "mamba_block.npz"))
    d_model, L, ns = (int(v) for v in z["none_cfg"])
    m = Mamba(d_model, bimamba_type="none", nslices=ns, layer_idx=3)
    with torch.no_grad():
        for n, p in m.named_parameters():
            p.copy_(torch.from_numpy(z[f"none_p_{n}"]))
    return m.cuda(), torch.from_numpy(z["none_x"]).cuda(), z["none_y"]


def _mamba2(tag):
    from nnuzoo_amd.nets.mamba2 import Mamba2
    z = np.load(os.path.join(GOLDEN, "mamba2_mixer.npz"))
    d_model = z[f"{tag}.p.out_proj.weight"].shape[0]
    m = Mamba2(d_model, d_state=16, d_conv=4, expand=2, headdim=int(z[f"{tag}.headdim"]), layer_idx=0)
    with torch.no_grad():
        for n, p in m.named_parameters():
            p.copy_(torch.from_numpy(z[f"{tag}.p.{n}"]))
    return m.cuda(), torch.from_numpy(z[f"{tag}.u"]).cuda(), z[f"{tag}.out"]


BLOCKS = [("mamba", lambda: _mamba()), ("mamba2 a", lambda: _mamba2("a")), ("mamba2 b", lambda: _mamba2("b"))]


@gpu
@pytest.mark.parametrize("name,make", BLOCKS, ids=[b[0] for b in BLOCKS])
@pytest.mark.parametrize("tokens", [0, 1, 5])
def test_prompt_and_steps_give_the_reference_outputs(hip_lib, name, make, tokens):
    m, x, want = make()
    B, L = x.shape[:2]
    conv, ssm = m.allocate_inference_cache(B)
    out = [m.prompt(x[:, :L - tokens], conv, ssm)]
    for t in range(L - tokens, L):
        y, c, s = m.step(x[:, t:t + 1], conv, ssm)
        assert c is conv and s is ssm and y.shape == (B, 1, x.shape[2])
        out.append(y)
    _close(torch.cat(out, 1), want, 3e-4, name)
    assert not out[0].requires_grad


@gpu
@pytest.mark.parametrize("name,make", BLOCKS, ids=[b[0] for b in BLOCKS])
def test_inference_params_and_ragged_prompts(hip_lib, name, make):
    m, x, _ = make()
    B, L = x.shape[:2]
    x = x[:1].expand(3, -1, -1) * torch.tensor([1.0, -0.5, 2.0], device="cuda")[:, None, None]
    lengths = [L - 2, 3, 0]
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    params = SimpleNamespace(key_value_memory_dict={}, seqlen_offset=0, max_seqlen=L, lengths_per_sample=lens)
    first = m(x, inference_params=params)
    assert list(params.key_value_memory_dict) == [m.layer_idx]
    params.seqlen_offset = L
    tok = m(x[:, L - 1:], inference_params=params)
    for i, n in enumerate(lengths):
        own = SimpleNamespace(key_value_memory_dict={}, seqlen_offset=0, max_seqlen=L, lengths_per_sample=None)
        # alone: its tokens and then the last one, as one prompt
        alone = m(torch.cat((x[i:i + 1, :n], x[i:i + 1, L - 1:]), 1), inference_params=own)
        _close(first[i:i + 1, :n], alone[:, :n].cpu(), 3e-4, f"{name} prompt {i}")
        _close(tok[i:i + 1], alone[:, n:].cpu(), 3e-4, f"{name} token {i}")
    # a new prompt on the same params starts from zero states
    params.seqlen_offset = 0
    again = m(x, inference_params=params)
    assert torch.equal(again, first)


@gpu
def test_step_leaves_inactive_sequences_alone(hip_lib):
    m, x, _ = _mamba()
    B = x.shape[0]
    conv, ssm = m.allocate_inference_cache(B, dtype=torch.float32)
    m.prompt(x, conv, ssm)
    c0, s0 = conv.clone(), ssm.clone()
    m.step(x[:, :1], conv, ssm, active=torch.zeros(B, dtype=torch.bool, device="cuda"))
    assert torch.equal(conv, c0) and torch.equal(ssm, s0)


@gpu
@pytest.mark.parametrize("name,make", BLOCKS, ids=[b[0] for b in BLOCKS])
def test_captured_steps(hip_lib, name, make):
    """a decoder's step as one graph: every replay moves the states on and gives what the eager step gives"""
    m, x, _ = make()
    B, L = x.shape[:2]
    token = x[:, :1].clone()
    caches = [m.allocate_inference_cache(B) for _ in range(2)]
    for conv, ssm in caches:
        m.prompt(x, conv, ssm)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            m.step(token, *m.allocate_inference_cache(B))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.step(token, *caches[0])[0]
    for t in range(4):
        token.copy_(x[:, t % L:t % L + 1])
        graph.replay()
        want = m.step(token, *caches[1])[0]
        torch.cuda.synchronize()
        _close(out, want.cpu(), 1e-5, f"{name} replay {t}")
        for a, b in zip(*caches):
            _close(a, b.cpu(), 1e-5, f"{name} state {t}")


@gpu
def test_decoding_under_autocast(hip_lib):
    """fp16 projections around the operators; the scan state stays fp32.  Against fp32: every activation is rounded to 11 bits a few
    times over, and a rounding of the input of the gate or the decays is at most doubled on its way"""
    m, x, want = _mamba()
    conv, ssm = m.allocate_inference_cache(x.shape[0])
    with torch.autocast("cuda", dtype=torch.float16):
        y = m.prompt(x[:, :-1], conv, ssm)
        t, _, _ = m.step(x[:, -1:], conv, ssm)
    assert y.dtype == torch.float16 and ssm.dtype == torch.float32
    _close(torch.cat((y, t), 1), want, 16 * 2.0 ** -11, "autocast")


@gpu
def test_decoding_refusals(hip_lib):
    from nnuzoo_amd.nets.mamba_simple import Mamba
    m, x, _ = _mamba()
    conv, ssm = m.allocate_inference_cache(x.shape[0])
    with pytest.raises(ValueError, match="one token"):
        m.step(x, conv, ssm)
    v2 = Mamba(16, bimamba_type="v2", layer_idx=0).cuda()
    with pytest.raises(NotImplementedError, match="causal"):
        v2.step(torch.zeros(1, 1, 16, device="cuda"), *v2.allocate_inference_cache(1))
    m.layer_idx = None
    with pytest.raises(ValueError, match="layer_idx"):
        m(x, inference_params=SimpleNamespace(key_value_memory_dict={}, seqlen_offset=0))
    with pytest.raises(ValueError, match="conv_state"):
        m.prompt(x, conv[:, :, :3].contiguous(), ssm)


def test_decoding_refuses_cpu_tensors():
    from nnuzoo_amd.nets.mamba2 import Mamba2
    from nnuzoo_amd.nets.mamba_simple import MambaSSM
    for m in (MambaSSM(16, layer_idx=0), Mamba2(16, d_state=16, headdim=2, layer_idx=0)):
        conv, ssm = m.allocate_inference_cache(2)
        assert conv.shape[0] == ssm.shape[0] == 2 and ssm.dtype == torch.float32
        for f in (lambda: m.step(torch.zeros(2, 1, 16), conv, ssm), lambda: m.prompt(torch.zeros(2, 5, 16), conv, ssm)):
            with pytest.raises(RuntimeError, match="no CPU fallback"):
                f()


@gpu
@pytest.mark.parametrize("order", ["h w", "w h"])
def test_residual_mamba_block_takes_the_group_norm_operator(hip_lib, order):
    """the second norm of a ResMambaBlock reads the first mixer's token-major output: the operator runs there, and the block's output and
    gradients stay what the two modules give"""
    from nnuzoo_amd import backends
    from nnuzoo_amd.nets.lm2net import ResMambaBlock
    torch.manual_seed(0)
    blk = ResMambaBlock(2, 16, norm=("GROUP", {"num_groups": 8}), order=order).cuda()
    x = torch.randn(2, 16, 12, 10, device="cuda", requires_grad=True)
    backends.reset()
    y = blk(x)
    assert backends.COUNTS[("GroupNorm", "group norm + activation", "hip")] == 1
    g = torch.randn_like(y)
    ps = [x, blk.norm2.weight, blk.norm2.bias, blk.gsc.proj2.conv.weight]
    got = [y.detach(), *torch.autograd.grad(y, ps, g)]
    hook = blk.norm2.register_forward_hook(lambda *a: None)      # a hooked module runs as a module
    y2 = blk(x)
    assert backends.COUNTS[("GroupNorm", "group norm + activation", "hip")] == 1
    want = [y2.detach(), *torch.autograd.grad(y2, ps, g)]
    hook.remove()
    for a, b, what in zip(got, want, ("y", "dx", "dw", "db", "dproj")):
        _close(a, b.cpu(), 1e-4, what)
    assert isinstance(blk.norm2, nn.GroupNorm)
