"""Calls of the decoding blocks beside the plain ones of test_mamba_decode_gpu.py: what other users of inference_params put there, values
past the half-precision range between the scan and the norm, empty batches."""
from types import SimpleNamespace

import pytest
import torch

from test_mamba_decode_gpu import BLOCKS, _close, _mamba2

gpu = pytest.mark.gpu


def _params(**kw):
    return SimpleNamespace(key_value_memory_dict={}, seqlen_offset=0, max_seqlen=64, **kw)


@gpu
@pytest.mark.parametrize("name,make", BLOCKS, ids=[b[0] for b in BLOCKS])
@pytest.mark.parametrize("cached", [0, 2])
def test_lengths_per_sample_is_the_callers_own_count(hip_lib, name, make, cached):
    """lengths_per_sample counts what each sequence has cached (0 before its prompt, or left over from the last one): the blocks do not
    take it for the prompt's lengths"""
    m, x, want = make()
    B, L = x.shape[:2]
    params = _params(lengths_per_sample=torch.full((B,), cached, dtype=torch.int32, device="cuda"))
    first = m(x[:, :L - 1], inference_params=params)
    params.seqlen_offset = L - 1
    tok = m(x[:, L - 1:], inference_params=params)
    _close(torch.cat((first, tok), 1), want, 3e-4, name)


@gpu
@pytest.mark.parametrize("name,make", BLOCKS, ids=[b[0] for b in BLOCKS])
def test_ragged_prompts_by_prompt_lengths(hip_lib, name, make):
    m, x, _ = make()
    B, L = x.shape[:2]
    x = x[:1].expand(3, -1, -1) * torch.tensor([1.0, -0.5, 2.0], device="cuda")[:, None, None]
    lengths = [L - 2, 3, 0]
    params = _params(prompt_lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    first = m(x, inference_params=params)
    params.seqlen_offset = L
    tok = m(x[:, L - 1:], inference_params=params)
    for i, n in enumerate(lengths):
        alone = m(torch.cat((x[i:i + 1, :n], x[i:i + 1, L - 1:]), 1), inference_params=_params(prompt_lengths=None))
        _close(first[i:i + 1, :n], alone[:, :n].cpu(), 3e-4, f"{name} prompt {i}")
        _close(tok[i:i + 1], alone[:, n:].cpu(), 3e-4, f"{name} token {i}")
    params.seqlen_offset = 0                    # a new prompt starts from zero states
    assert torch.equal(m(x, inference_params=params), first)


@gpu
@pytest.mark.parametrize("half_weights", [False, True])
def test_gated_values_past_the_half_precision_range(hip_lib, half_weights):
    """x silu(z) may pass 65 504 before the RMS norm brings it back: prompt and step keep it in fp32, as forward does.  Against fp32 the
    roundings to 11 bits are those of the input, of in_proj's weight and output (once each in x, z, and the product of both), of the
    convolution's output, of the norm's output, of out_proj's weight and output: 10 relative to their own value, carried on by linear steps
    and by a norm that halves or keeps them; the allowance is the one of the other autocast test, 16"""
    m, x, _ = _mamba2("a")
    with torch.no_grad():
        m.in_proj.weight.mul_(400.0 / (x @ m.in_proj.weight.t()).abs().max())
        n, ds = m.d_state, m.d_ssm
        m.in_proj.weight[2 * ds:2 * ds + 2 * n] *= 0.01        # B, C and dt stay ordinary
        m.in_proj.weight[2 * ds + 2 * n:] *= 0.01
        m.D.fill_(20.0)
    want = m(x)
    if half_weights:
        m, x = m.half(), x.half()
    conv, ssm = m.allocate_inference_cache(x.shape[0])
    with torch.autocast("cuda", dtype=torch.float16, enabled=not half_weights):
        y = m.prompt(x[:, :-1], conv, ssm)
        t = m.step(x[:, -1:], conv, ssm)[0]
    got = torch.cat((y, t), 1)
    assert bool(torch.isfinite(got).all())
    _close(got, want.detach().cpu(), 16 * 2.0 ** -11, "gated")
