"""The variants of the state-carrying scan and convolution (csrc/mamba_state.hip) that only large calls take, against the 64-bit
restatement: two channels a quad (from 4 096 waves on) for whole sequences, for chunks that each workgroup joins by itself and for
chunks with a joining kernel; chunks with several channels a head, several groups and one decay a head; 16 tokens a thread in the
convolution."""
import pytest
import torch

from oracle.state_space_block import causal_conv, causal_conv_rows, close, selective_scan, selective_scan_rows
from test_mamba_state_gpu import DT, _conv_data, _scan_data

gpu = pytest.mark.gpu


def _lengths(B, L, seed):
    """whole, empty, one token, one short, and the rest at random"""
    n = torch.randint(0, L + 1, (B,), generator=torch.Generator().manual_seed(seed))
    for i, v in enumerate((L, 0, 1, L - 1)):
        n[i * (B - 1) // 3 if B > 4 else i % B] = v
    n[-1] = L
    return n


def _oracle(v, lengths, join=0):
    return selective_scan_rows(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], v["dt_bias"], True, v["state"], lengths, join)


def _chunks(B, L, d, H, G, N):
    """(chunks, tokens of a chunk) by the workspace: a state and a sum for each chunk, sequence and channel"""
    from nnuzoo_amd._lib import load
    bytes_ = load().nnz_selective_scan_prompt_workspace_bytes(B, L, d, H, G, N)
    chunks = bytes_ // (B * d * (N + 1) * 4)
    for cl in range(16, L + 16, 16):
        if -(-L // cl) == chunks:
            return chunks, cl
    return 1, L


def _check(B, L, d, H, G, N, dt, per_head=False, chunks=1, slow=0.0):
    from nnuzoo_amd.mamba_state import selective_scan_prompt
    v = _scan_data(B, L, d, H, G, N, dt, seed=B + L, per_head=per_head)
    v["dt_bias"] -= slow
    n = _lengths(B, L, d)
    got, cl = _chunks(B, L, d, H, G, N)
    assert got == chunks
    behind = torch.arange(L) >= n[:, None]
    for k in ("x", "dt", "B", "C", "z"):
        v[k][behind] = float("nan")
    want, new = _oracle(v, n, join=cl if chunks > 1 else 0)
    c = {k: t.cuda() for k, t in v.items()}
    y = selective_scan_prompt(c["x"], c["dt"], c["A"], c["B"], c["C"], c["D"], z=c["z"], dt_bias=c["dt_bias"], dt_softplus=True,
                              state=c["state"], lengths=n.to(torch.int32).cuda())
    close(y, *want, "y")
    close(c["state"], *new, "state")


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("B,L,d,H,G,N", [(4096, 3, 33, 33, 1, 16), (2048, 18, 48, 8, 1, 8), (2048, 35, 66, 66, 2, 4), (4096, 2, 6, 1, 1, 32)])
def test_two_channels_a_quad_whole_sequences(hip_lib, dt, B, L, d, H, G, N):
    _check(B, L, d, H, G, N, dt)


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("d,H,G,N", [(7, 7, 1, 4), (12, 6, 1, 16), (16, 16, 1, 8)])
def test_two_channels_a_quad_in_chunks(hip_lib, dt, d, H, G, N):
    _check(1024, 513, d, H, G, N, dt, chunks=7, slow=2.0)


@gpu
@pytest.mark.parametrize("dt", list(DT))
def test_two_channels_a_quad_in_chunks_with_a_joining_kernel(hip_lib, dt):
    _check(8, 4100, 257, 257, 1, 4, dt, chunks=65, slow=3.0)


@gpu
@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("L,chunks", [(600, 10), (2500, 40)])
@pytest.mark.parametrize("d,H,G,N", [(40, 8, 2, 8), (24, 6, 1, 16), (66, 6, 3, 4)])
def test_chunks_with_heads_and_groups(hip_lib, dt, per_head, L, chunks, d, H, G, N):
    _check(2, L, d, H, G, N, dt, per_head=per_head, chunks=chunks, slow=2.0)


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("B,L,D,W", [(8, 4100, 257, 4), (8, 2053, 512, 8), (6, 2051, 1028, 2)])
def test_convolution_with_16_tokens_a_thread(hip_lib, dt, B, L, D, W):
    """from 131 072 threads of 16 tokens on (V channels each: 4 where D is a multiple of 4)"""
    from nnuzoo_amd.mamba_state import causal_conv1d_prompt
    assert B * (D // 4 if D % 4 == 0 else D) * -(-L // 16) >= 131072
    x, w, b, st = _conv_data(B, L, D, W, dt, seed=L)
    n = _lengths(B, L, W)
    x[torch.arange(L) >= n[:, None]] = float("nan")
    s = st.cuda()
    y = causal_conv1d_prompt(x.cuda(), w.cuda(), b.cuda(), "silu", s, n.cuda())
    want, new = causal_conv_rows(x, w, b, True, st, n)
    close(y, *want, "y")
    assert torch.equal(s.double().cpu(), new)


def test_the_restatements_agree():
    """all sequences at once = sequence by sequence"""
    for per_head in (False, True):
        v = _scan_data(3, 9, 12, 6, 2, 8, "f32", 1, per_head)
        args = [v[k] for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")]
        for a, b in zip(selective_scan(*args, True, v["state"], [9, 0, 4]), selective_scan_rows(*args, True, v["state"], [9, 0, 4])):
            for p, q in zip(a, b):
                assert torch.allclose(p, q, rtol=1e-12, atol=1e-14)
    x, w, b, st = _conv_data(3, 9, 12, 4, "f32", 1)
    (y, e), new = causal_conv(x, w, b, True, st, [9, 0, 3])
    (y2, e2), new2 = causal_conv_rows(x, w, b, True, st, [9, 0, 3])
    assert torch.allclose(y, y2, rtol=1e-12, atol=1e-14) and torch.allclose(e, e2, rtol=1e-12) and torch.equal(new, new2)
