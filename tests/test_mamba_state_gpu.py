"""The state-carrying causal convolution and selective scan (csrc/mamba_state.hip), for prompts and single tokens, against the 64-bit
restatement of oracle/state_space_block.py, whose bounds follow the roundings of an fp32 recurrence step by step.  Lengths from one
token to several chunks, ragged batches with empty sequences, rows that are views of wider tensors, heads and groups, and the
operators together as a decoder uses them."""
import pytest
import torch

from oracle.state_space_block import causal_conv as conv_oracle, close, selective_scan as scan_oracle

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
gpu = pytest.mark.gpu


def _exact(got, want, what):
    assert torch.equal(got.double().cpu(), want), what


# ---- causal convolution ----------------------------------------------------------------------------------------------------------
def _conv_data(B, L, D, W, dt, seed, wide=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, L, D + wide, generator=g).to(DT[dt])
    return x, torch.randn(D, W, generator=g) * 0.5, torch.randn(D, generator=g) * 0.2, torch.randn(B, D, W, generator=g).to(DT[dt])


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("B,L,D,W", [(1, 1, 8, 4), (2, 2, 16, 4), (1, 3, 7, 4), (3, 37, 24, 3), (2, 100, 8, 8), (1, 9, 5, 1), (2, 33, 40, 2),
                                     (1, 64, 3, 5), (2, 20, 16, 6), (1, 31, 8, 7)])
def test_conv_prompt(hip_lib, dt, B, L, D, W):
    from nnuzoo_amd.mamba_state import causal_conv1d_prompt
    x, w, b, st = _conv_data(B, L, D, W, dt, seed=L + W)
    for act, bias, state in (("silu", b, st), (None, None, st), ("silu", b, None)):
        s = None if state is None else state.cuda()
        y = causal_conv1d_prompt(x.cuda(), w.cuda(), None if bias is None else bias.cuda(), act, s)
        want, new = conv_oracle(x, w, bias, act is not None, state, [L] * B)
        assert y.dtype == x.dtype
        close(y, *want, "y")
        if s is not None:
            _exact(s, new, "conv_state")


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("len_type", [torch.int32, torch.int64])
def test_conv_ragged_prompts(hip_lib, dt, len_type):
    """empty, one token, less than the window, whole; NaN behind every sequence is never read"""
    from nnuzoo_amd.mamba_state import causal_conv1d_prompt
    B, L, D, W = 6, 45, 16, 4
    lengths = [0, 1, 2, 3, 29, 45]
    x, w, b, st = _conv_data(B, L, D, W, dt, seed=5)
    for i, n in enumerate(lengths):
        x[i, n:] = float("nan")
    s = st.cuda()
    y = causal_conv1d_prompt(x.cuda(), w.cuda()[:, None], b.cuda(), "swish", s, torch.tensor(lengths, dtype=len_type).cuda())
    want, new = conv_oracle(x, w, b, True, st, lengths)
    close(y, *want, "y")
    _exact(s, new, "conv_state")
    # lengths outside 0 .. L are clamped
    s2, s3 = st.cuda(), st.cuda()
    x = torch.nan_to_num(x)
    y2 = causal_conv1d_prompt(x.cuda(), w.cuda(), b.cuda(), "silu", s2, torch.tensor([-3, -1, 0, 46, 1 << 30, 45], dtype=len_type).cuda())
    y3 = causal_conv1d_prompt(x.cuda(), w.cuda(), b.cuda(), "silu", s3, torch.tensor([0, 0, 0, 45, 45, 45], dtype=len_type).cuda())
    assert torch.equal(y2, y3) and torch.equal(s2, s3)


@gpu
@pytest.mark.parametrize("dt", list(DT))
def test_conv_strides_and_states_of_other_layouts(hip_lib, dt):
    from nnuzoo_amd.mamba_state import causal_conv1d_prompt, causal_conv1d_token
    B, L, D, W = 2, 30, 16, 4
    x, w, b, st = _conv_data(B, L, D, W, dt, seed=6, wide=24)
    big = x.cuda()
    pool = torch.zeros(5, W, D, dtype=st.dtype, device="cuda")
    for lo in (0, 8, 3):
        for state in (st.cuda(), pool[1:3].transpose(1, 2).copy_(st.cuda()), st.cuda().float(), torch.zeros(4, D, W, device="cuda")[::2].copy_(st)):
            xv = x[..., lo:lo + D]
            y = causal_conv1d_prompt(big[..., lo:lo + D], w.cuda(), b.cuda(), "silu", state)
            want, new = conv_oracle(xv, w, b, True, st, [L] * B)
            close(y, *want, "y")
            _exact(state, new, "conv_state")
            tok = big[:, 0, lo:lo + D]
            y = causal_conv1d_token(tok, state, w.cuda(), b.cuda())
            want, new = conv_oracle(tok.cpu()[:, None], w, b, True, new, [1] * B)
            close(y[:, None], *want, "token")
            _exact(state, new, "conv_state")
    # token-major memory the other way round: (L, B, D) and channels-first rows (copied)
    for xv in (x[..., :D].transpose(0, 1).contiguous().transpose(0, 1), x[..., :D].transpose(1, 2).contiguous().transpose(1, 2)):
        y = causal_conv1d_prompt(xv.cuda(), w.cuda(), b.cuda())
        close(y, *conv_oracle(xv, w, b, True, None, [L] * B)[0], "y")


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("B,D,W", [(1, 1, 4), (3, 70, 4), (5, 33, 2), (2, 8, 8), (1, 16, 1)])
def test_conv_token_and_active_rows(hip_lib, dt, B, D, W):
    from nnuzoo_amd.mamba_state import causal_conv1d_token
    x, w, b, st = _conv_data(B, 1, D, W, dt, seed=W)
    s = st.cuda()
    y = causal_conv1d_token(x[:, 0].cuda(), s, w.cuda(), b.cuda())
    want, new = conv_oracle(x, w, b, True, st, [1] * B)
    close(y[:, None], *want, "y")
    _exact(s, new, "conv_state")
    on = torch.arange(B) % 2 == 1
    s = st.cuda()
    y = causal_conv1d_token(x[:, 0].cuda(), s, w.cuda(), b.cuda(), active=on.cuda())
    want, new = conv_oracle(x, w, b, True, st, [int(v) for v in on])
    close(y[:, None], *want, "y")
    _exact(s, new, "conv_state")


@gpu
def test_conv_in_pieces_equals_conv_at_once(hip_lib):
    from nnuzoo_amd.mamba_state import causal_conv1d_prompt, causal_conv1d_token
    x, w, b, st = _conv_data(2, 50, 24, 4, "f16", seed=8)
    x, w, b = x.cuda(), w.cuda(), b.cuda()
    whole, s1, s2 = None, st.cuda(), st.cuda()
    whole = causal_conv1d_prompt(x, w, b, "silu", s1)
    parts = [causal_conv1d_prompt(x[:, :17], w, b, "silu", s2)]
    parts += [causal_conv1d_token(x[:, t], s2, w, b)[:, None] for t in range(17, 21)]
    parts.append(causal_conv1d_prompt(x[:, 21:], w, b, "silu", s2))
    assert torch.equal(torch.cat(parts, 1), whole) and torch.equal(s1, s2)


# ---- selective scan --------------------------------------------------------------------------------------------------------------
def _scan_data(B, L, d, H, G, N, dt, seed, per_head=False):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    dt0 = torch.exp(torch.rand(H, generator=g) * 4.6 - 6.9)
    A = -torch.exp(rn(H)) if per_head else -torch.arange(1.0, N + 1) * (1 + 0.1 * torch.rand(H, N, generator=g))
    cast = lambda t: t.to(DT[dt])  # noqa: E731
    return dict(x=cast(rn(B, L, d)), dt=cast(rn(B, L, H) * 0.5), A=A, B=cast(rn(B, L, G, N)), C=cast(rn(B, L, G, N)), D=rn(H) * 0.2 + 1,
                z=cast(rn(B, L, d)), dt_bias=dt0 + torch.log(-torch.expm1(-dt0)), state=rn(B, d, N))


def _scan_want(v, lengths, softplus=True, join=1 << 30):
    return scan_oracle(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], v["dt_bias"], softplus, v["state"], lengths, join)


def _scan_got(v, softplus=True, lengths=None):
    from nnuzoo_amd.mamba_state import selective_scan_prompt
    c = {k: None if t is None else t.cuda() for k, t in v.items()}
    y = selective_scan_prompt(c["x"], c["dt"], c["A"], c["B"], c["C"], c["D"], z=c["z"], dt_bias=c["dt_bias"], dt_softplus=softplus,
                              state=c["state"], lengths=lengths)
    return y, c["state"]


SHAPES = [(1, 1, 16, 16, 1, 16), (2, 5, 24, 24, 1, 16), (1, 49, 64, 64, 1, 16), (2, 33, 40, 8, 2, 8), (1, 70, 96, 6, 1, 16), (3, 31, 7, 7, 1, 4),
          (1, 130, 20, 4, 2, 32), (2, 64, 130, 130, 1, 16), (1, 300, 33, 33, 1, 16), (1, 32, 1, 1, 1, 4)]


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("B,L,d,H,G,N", SHAPES)
def test_scan_prompt(hip_lib, dt, B, L, d, H, G, N):
    v = _scan_data(B, L, d, H, G, N, dt, seed=L + d)
    y, st = _scan_got(v)
    want, new = _scan_want(v, [L] * B, join=32)
    assert y.dtype == v["x"].dtype and st.dtype == torch.float32
    close(y, *want, "y")
    close(st, *new, "state")


@gpu
@pytest.mark.parametrize("drop", [("z",), ("D",), ("dt_bias",), ("state",), ("z", "D", "dt_bias", "state")])
@pytest.mark.parametrize("softplus", [True, False])
def test_scan_without_optional_inputs(hip_lib, drop, softplus):
    v = _scan_data(2, 40, 24, 24, 1, 16, "f32", seed=3)
    if not softplus:
        v["dt"], v["dt_bias"] = v["dt"].abs() * 0.1, v["dt_bias"].abs() * 0.01
    v.update({k: None for k in drop})
    y, st = _scan_got(v, softplus)
    want, new = _scan_want(v, [40] * 2, softplus, join=32)
    close(y, *want, "y")
    if st is not None:
        close(st, *new, "state")


@gpu
def test_scan_one_decay_a_head(hip_lib):
    """Mamba2's form: A (H,), dt per head, B and C without a group axis"""
    v = _scan_data(2, 37, 48, 6, 1, 16, "f16", seed=4, per_head=True)
    want, new = _scan_want(v, [37] * 2, join=32)
    v["B"], v["C"] = v["B"][:, :, 0], v["C"][:, :, 0]
    y, st = _scan_got(v)
    close(y, *want, "y")
    close(st, *new, "state")


@gpu
@pytest.mark.parametrize("per_head", [False, True])
def test_decays_by_their_logarithm(hip_lib, per_head):
    """A_is_log: the decays are -exp of what is passed, formed in fp32 (|A_log| + 4 roundings more, relative)"""
    from nnuzoo_amd.mamba_state import selective_scan_prompt, selective_scan_token
    v = _scan_data(2, 37, 24, 6, 1, 16, "f32", seed=5, per_head=per_head)
    v["A"] = torch.log(-v["A"])
    c = {k: t.cuda() for k, t in v.items()}
    y = selective_scan_prompt(c["x"], c["dt"], c["A"], c["B"], c["C"], c["D"], z=c["z"], dt_bias=c["dt_bias"], dt_softplus=True,
                              state=c["state"], A_is_log=True)
    t = selective_scan_token(c["x"][:, 0], c["dt"][:, 0], c["A"], c["B"][:, 0], c["C"][:, 0], c["D"], z=c["z"][:, 0], dt_bias=c["dt_bias"],
                             dt_softplus=True, state=c["state"], A_is_log=True)
    slack = 1 + 8 * 2.0 ** -24
    lo, hi = dict(v, A=-torch.exp(v["A"].double()) * slack), dict(v, A=-torch.exp(v["A"].double()))
    cat = lambda d: {k: (torch.cat((u, u[:, :1]), 1) if k in ("x", "dt", "B", "C", "z") else u) for k, u in d.items()}  # noqa: E731
    (ya, ea), (sa, es) = _scan_want(cat(hi), [38] * 2, join=32)
    (yb, _), (sb, _) = _scan_want(cat(lo), [38] * 2, join=32)
    # a relative change of the decays by 8 roundings moves the results by their difference, to first order, in either direction
    close(torch.cat((y, t[:, None]), 1), ya, ea + 2 * (ya - yb).abs() + 2.0 ** -22 * ya.abs().amax(), "y")
    close(c["state"], sa, es + 2 * (sa - sb).abs() + 2.0 ** -22 * sa.abs().amax(), "state")


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("d,L,join", [(16, 1000, 128), (40, 517, 128), (7, 300, 128)])
def test_scan_of_several_chunks_ragged(hip_lib, dt, d, L, join):
    """few channels, long sequences: chunks; lengths that end at, before and after the borders of tiles and chunks, NaN behind them"""
    lengths = [L, 0, 1, 127, 128, 129, L - 1, 256]
    v = _scan_data(len(lengths), L, d, d, 1, 16, dt, seed=L)
    for k in ("x", "dt", "B", "C", "z"):
        for i, n in enumerate(lengths):
            v[k][i, n:] = float("nan")
    for kind in (torch.int32, torch.int64):
        y, st = _scan_got(v, lengths=torch.tensor(lengths, dtype=kind).cuda())
        want, new = _scan_want(v, lengths, join=join)
        close(y, *want, "y")
        close(st, *new, "state")


@gpu
def test_scan_of_many_chunks(hip_lib):
    """more than 64 chunks: runs of them are joined side by side"""
    v = _scan_data(2, 5000, 8, 8, 1, 4, "f32", seed=11)
    v["dt_bias"] -= 3      # slow decays, so that far chunks still matter
    lengths = [5000, 4163]
    y, st = _scan_got(v, lengths=torch.tensor(lengths, dtype=torch.int32).cuda())
    want, new = _scan_want(v, lengths, join=64)
    close(y, *want, "y")
    close(st, *new, "state")


@gpu
def test_scan_repeats_bit_for_bit(hip_lib):
    v = _scan_data(2, 3000, 24, 24, 1, 16, "f16", seed=9)
    first = _scan_got(v)
    for _ in range(2):
        again = _scan_got(v)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@gpu
@pytest.mark.parametrize("dt", list(DT))
def test_scan_views_of_the_projections(hip_lib, dt):
    """x | z halves of one tensor, dt | B | C slices of another, a state that is every other row of a pool"""
    from nnuzoo_amd.mamba_state import selective_scan_prompt, selective_scan_token
    B, L, d, N = 2, 50, 24, 16
    v = _scan_data(B, L, d, d, 1, N, dt, seed=10)
    xz = torch.cat((v["x"], v["z"]), -1).cuda()
    dbc = torch.cat((v["dt"], v["B"][:, :, 0], v["C"][:, :, 0]), -1).cuda()
    pool = torch.zeros(2 * B, d, N, device="cuda")
    st = pool[::2].copy_(v["state"])
    par = {k: v[k].cuda() for k in ("A", "D", "dt_bias")}
    pick = lambda sl: (xz[sl][..., :d], dbc[sl][..., :d], par["A"], dbc[sl][..., d:d + N], dbc[sl][..., d + N:], par["D"])  # noqa: E731
    y = selective_scan_prompt(*pick(slice(None)), z=xz[..., d:], dt_bias=par["dt_bias"], dt_softplus=True, state=st)
    want, new = _scan_want(v, [L] * B, join=32)
    close(y, *want, "y")
    close(st, *new, "state")
    assert not pool[1::2].any()
    sl = (slice(None), 3)
    before = st.cpu()
    y = selective_scan_token(*pick(sl), z=xz[sl][..., d:], dt_bias=par["dt_bias"], dt_softplus=True, state=st)
    one = {k: (t[:, 3:4] if k in ("x", "dt", "B", "C", "z") else t) for k, t in v.items()}
    one["state"] = before
    want, new = _scan_want(one, [1] * B)
    close(y[:, None], *want, "token")
    close(st, *new, "state")


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("B,d,H,G,N", [(1, 16, 16, 1, 16), (3, 40, 8, 2, 8), (2, 7, 7, 1, 4), (5, 64, 4, 4, 32), (1, 1, 1, 1, 16), (4, 130, 130, 1, 16)])
def test_scan_token_and_active_rows(hip_lib, dt, B, d, H, G, N):
    from nnuzoo_amd.mamba_state import selective_scan_token
    v = _scan_data(B, 1, d, H, G, N, dt, seed=d)
    c = {k: t.cuda() for k, t in v.items()}
    on = torch.arange(B) % 2 == 0
    for active in (None, on):
        st = v["state"].cuda()
        y = selective_scan_token(c["x"][:, 0], c["dt"][:, 0], c["A"], c["B"][:, 0], c["C"][:, 0], c["D"], z=c["z"][:, 0],
                                 dt_bias=c["dt_bias"], dt_softplus=True, state=st, active=None if active is None else active.cuda())
        want, new = _scan_want(v, [1] * B if active is None else [int(a) for a in on])
        close(y[:, None], *want, "y")
        close(st, *new, "state")


@gpu
def test_decays_of_zero_and_time_steps_that_vanish(hip_lib):
    """dt = -100: softplus 0, the state stays; dt = 100: softplus 100, the state is replaced; A = 0: the state only grows"""
    v = _scan_data(1, 6, 16, 16, 1, 16, "f32", seed=12)
    v["dt"][:, 0:2], v["dt"][:, 2:4] = -100.0, 100.0
    v["A"][::2] = 0.0
    y, st = _scan_got(v)
    want, new = _scan_want(v, [6], join=32)
    close(y, *want, "y")
    close(st, *new, "state")


# ---- together --------------------------------------------------------------------------------------------------------------------
@gpu
def test_prompt_then_tokens_as_a_decoder_runs_them(hip_lib):
    """two ragged prompts, then tokens of which one sequence sits out a step, captured into a graph after the first: convolution and
    scan in turn on the same states, against the whole sequences at once in 64 bits"""
    from nnuzoo_amd.mamba_state import causal_conv1d_prompt, causal_conv1d_token, selective_scan_prompt, selective_scan_token
    B, L, d, N, W, steps = 3, 40, 32, 16, 4, 5
    v = _scan_data(B, L + steps, d, d, 1, N, "f32", seed=20)
    _, w, b, _ = _conv_data(B, 1, d, W, "f32", seed=21)
    lengths = [40, 13, 0]
    takes = torch.tensor([[1, 1, 1], [1, 0, 1], [1, 1, 1], [0, 1, 1], [1, 1, 0]], dtype=torch.bool)
    c = {k: t.cuda() for k, t in v.items()}
    wc, bc = w.cuda(), b.cuda()
    cs, st = torch.zeros(B, d, W, device="cuda"), torch.zeros(B, d, N, device="cuda")
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    cut = lambda k, t: c[k][:, :L] if t is None else c[k][:, L + t]  # noqa: E731
    u = causal_conv1d_prompt(cut("x", None), wc, bc, "silu", cs, lens)
    y0 = selective_scan_prompt(u, cut("dt", None), c["A"], cut("B", None), cut("C", None), c["D"], z=cut("z", None), dt_bias=c["dt_bias"],
                               dt_softplus=True, state=st, lengths=lens)
    ins = {k: torch.empty_like(c[k][:, 0]) for k in ("x", "dt", "B", "C", "z")}
    act = torch.empty(B, dtype=torch.bool, device="cuda")

    def step():
        u_ = causal_conv1d_token(ins["x"], cs, wc, bc, "silu", act)
        return selective_scan_token(u_, ins["dt"], c["A"], ins["B"], ins["C"], c["D"], z=ins["z"], dt_bias=c["dt_bias"], dt_softplus=True,
                                    state=st, active=act)

    def load(t):
        for k in ins:
            ins[k].copy_(c[k][:, L + t])
        act.copy_(takes[t])
    load(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [step().clone()]
    torch.cuda.current_stream().wait_stream(side)
    keep = (cs.clone(), st.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    assert torch.equal(cs, keep[0]) and torch.equal(st, keep[1])      # capturing runs nothing
    for t in range(1, steps):
        load(t)
        graph.replay()
        torch.cuda.synchronize()
        outs.append(out.clone())
    # every sequence on its own: its prompt and the tokens it took part in
    for i in range(B):
        at = list(range(lengths[i])) + [L + t for t in range(steps) if takes[t, i]]
        one = {k: (t[i:i + 1, at] if k in ins else t) for k, t in v.items()}
        (u64, eu), new_cs = conv_oracle(one["x"], w, b, True, None, [len(at)])
        one.update(x=u64, state=None)
        (y64, ey), (st64, es) = _scan_want(one, [len(at)], join=32)
        # the convolution's own error, through the scan (which is linear in x) with every term taken as positive
        err = dict(one, x=eu, B=one["B"].abs(), C=one["C"].abs(), D=one["D"].abs(), z=None)
        (yu, _), (su, _) = _scan_want(err, [len(at)])
        zz = one["z"].double()
        got = torch.cat([y0[i, :lengths[i]]] + [outs[t][i:i + 1] for t in range(steps) if takes[t, i]])
        close(got, y64[0], ey[0] + 1.01 * (yu * (zz * zz.sigmoid()).abs())[0], "y")
        close(st[i], st64[0], es[0] + 1.01 * su[0], "state")
        assert torch.equal(cs[i].double().cpu(), new_cs[0])
        assert not y0[i, lengths[i]:].any()
        assert all(not outs[t][i].any() for t in range(steps) if not takes[t, i])


@gpu
def test_more_than_2_to_31_elements_apart(hip_lib):
    """rows of one sequence 2^25 elements apart, so that late tokens lie past 2^31 elements"""
    from nnuzoo_amd.mamba_state import causal_conv1d_prompt, selective_scan_prompt
    L, d, N, gap = 70, 16, 16, 1 << 25
    v = _scan_data(1, L, d, d, 1, N, "f16", seed=30)
    buf = torch.empty((L - 1) * gap + 64, dtype=torch.float16, device="cuda")
    xv = buf.as_strided((1, L, d), (gap, gap, 1))
    xv.copy_(v["x"].cuda())
    _, w, b, _ = _conv_data(1, 1, d, 4, "f32", seed=31)
    close(causal_conv1d_prompt(xv, w.cuda(), b.cuda()), *conv_oracle(v["x"], w, b, True, None, [L])[0], "conv")
    c = {k: t.cuda() for k, t in v.items()}
    y = selective_scan_prompt(xv, c["dt"], c["A"], c["B"], c["C"], c["D"], z=c["z"], dt_bias=c["dt_bias"], dt_softplus=True, state=c["state"])
    close(y, *_scan_want(v, [L], join=32)[0], "scan")


@gpu
def test_empty_batches_and_prompts(hip_lib):
    from nnuzoo_amd.mamba_state import causal_conv1d_prompt, causal_conv1d_token, selective_scan_prompt, selective_scan_token
    w = torch.ones(8, 4).cuda()
    A = -torch.ones(8, 16).cuda()
    z = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    for B, L in ((0, 5), (2, 0)):
        st, cs = torch.ones(B, 8, 16, device="cuda"), torch.ones(B, 8, 4, device="cuda")
        assert causal_conv1d_prompt(z(B, L, 8), w, conv_state=cs).shape == (B, L, 8)
        assert selective_scan_prompt(z(B, L, 8), z(B, L, 8), A, z(B, L, 16), z(B, L, 16), state=st).shape == (B, L, 8)
        assert bool((st == 1).all()) and bool((cs == 1).all())
    assert causal_conv1d_token(z(0, 8), z(0, 8, 4), w).shape == (0, 8)
    assert selective_scan_token(z(0, 8), z(0, 8), A, z(0, 16), z(0, 16), state=z(0, 8, 16)).shape == (0, 8)


@gpu
def test_refusals(hip_lib):
    from nnuzoo_amd.mamba_state import causal_conv1d_prompt, causal_conv1d_token, selective_scan_prompt, selective_scan_token
    z = lambda *s, dtype=torch.float32: torch.zeros(s, device="cuda", dtype=dtype)  # noqa: E731
    x, w, cs = z(2, 5, 8), z(8, 4), z(2, 8, 4)

    def conv(err, match, *a, **k):
        with pytest.raises(err, match=match):
            causal_conv1d_prompt(*a, **k)
    conv(NotImplementedError, "activation", x, w, activation="relu")
    conv(NotImplementedError, "widths", x, z(8, 9))
    conv(ValueError, "weight", x, z(7, 4))
    conv(ValueError, "bias", x, w, z(7))
    conv(ValueError, r"\(B, L, D\)", x[0], w)
    conv(ValueError, "conv_state", x, w, conv_state=z(2, 8, 3))
    conv(ValueError, "share memory", x, w, conv_state=z(1, 8, 4).expand(2, 8, 4))
    conv(TypeError, "conv_state", x, w, conv_state=z(2, 8, 4, dtype=torch.float16))
    conv(TypeError, "lengths", x, w, lengths=z(2))
    conv(ValueError, "lengths", x, w, lengths=z(3, dtype=torch.int32))
    conv(NotImplementedError, "float32", x.double(), w)
    conv(RuntimeError, "no backward", x, w.clone().requires_grad_(True))
    conv(RuntimeError, "no CPU fallback", x, w.cpu())
    with pytest.raises(TypeError, match="active"):
        causal_conv1d_token(x[:, 0], cs, w, active=z(2, dtype=torch.int32))
    with torch.no_grad():
        causal_conv1d_prompt(x, w.clone().requires_grad_(True))
    A, B, st = z(8, 16), z(2, 5, 16), z(2, 8, 16)

    def scan(err, match, x_=x, dt=x, A_=A, B_=B, C_=B, **k):
        with pytest.raises(err, match=match):
            selective_scan_prompt(x_, dt, A_, B_, C_, **k)
    scan(ValueError, "heads", dt=z(2, 5, 3), A_=z(3, 16))
    scan(ValueError, "groups", B_=z(2, 5, 3, 16), C_=z(2, 5, 3, 16))
    scan(ValueError, "`A`", A_=z(8, 8))
    scan(ValueError, "`C`", C_=z(2, 5, 8))
    scan(NotImplementedError, "state widths", A_=z(8, 12), B_=z(2, 5, 12), C_=z(2, 5, 12))
    scan(ValueError, "`dt`", dt=z(2, 4, 8))
    scan(TypeError, "one type", dt=x.half())
    scan(ValueError, "`z`", z=z(2, 5, 7))
    scan(TypeError, "float32", state=st.half())
    scan(ValueError, "in place", state=z(2, 16, 8).transpose(1, 2))
    scan(ValueError, "share memory", state=z(1, 8, 16).expand(2, 8, 16))
    scan(ValueError, "`state`", state=z(3, 8, 16))
    scan(RuntimeError, "no backward", A_=A.clone().requires_grad_(True))
    scan(RuntimeError, "no CPU fallback", A_=A.cpu())
    scan(ValueError, "`D`", D=z(7))
    with pytest.raises(ValueError, match=r"\(B, D\)"):
        selective_scan_token(x, x, A, B, B, state=st)


def test_refuses_cpu_tensors_and_bad_calls_without_a_gpu():
    from nnuzoo_amd import _lib
    from nnuzoo_amd.mamba_state import causal_conv1d_prompt, causal_conv1d_token, selective_scan_prompt, selective_scan_token
    x, w, A, B = torch.zeros(2, 5, 8), torch.zeros(8, 4), torch.zeros(8, 16), torch.zeros(2, 5, 16)
    for f in (lambda: causal_conv1d_prompt(x, w), lambda: causal_conv1d_token(x[:, 0], torch.zeros(2, 8, 4), w),
              lambda: selective_scan_prompt(x, x, A, B, B),
              lambda: selective_scan_token(x[:, 0], x[:, 0], A, B[:, 0], B[:, 0], state=torch.zeros(2, 8, 16))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f()
    lib = _lib.load()
    assert lib.nnz_causal_conv1d_prompt(None, 0, 0, 0, None, None, None, None, 0, 0, 0, 0, None, 0, 1, 1, 8, 4, 1, None) == -22
    assert lib.nnz_causal_conv1d_prompt(16, 0, 0, 0, 16, None, 16, None, 0, 0, 0, 0, None, 0, 1, 1, 8, 9, 1, None) == -22
    assert lib.nnz_causal_conv1d_token(16, 0, 0, 16, None, 16, None, 0, 0, 0, 0, None, 1, 8, 4, 1, None) == -22
    for bad in ((0, 5, 8, 8, 1, 16), (1, 0, 8, 8, 1, 16), (1, 5, 8, 3, 1, 16), (1, 5, 8, 8, 3, 16), (1, 5, 8, 8, 1, 12)):
        assert lib.nnz_selective_scan_prompt_workspace_bytes(*bad) == -22
    assert lib.nnz_selective_scan_prompt_workspace_bytes(1, 5, 8, 8, 1, 16) == 0
    assert lib.nnz_selective_scan_prompt_workspace_bytes(1, 4096, 8, 8, 1, 16) > 0
    strides = (_lib.C.c_long * 12)()
    # a call that needs a workspace and gets none
    assert lib.nnz_selective_scan_prompt(16, 16, 16, 16, None, 0, strides, 16, 1, None, None, 0, None, 0, 16, None, 0, None, 0, 1, 4096, 8, 8,
                                         1, 16, None) == -22
    # more sequences than a launch has grid rows for
    assert lib.nnz_selective_scan_prompt(16, 16, 16, 16, None, 0, strides, 16, 1, None, None, 0, None, 0, 16, None, 0, None, 0, 65536, 4, 8,
                                         8, 1, 16, None) == -22
