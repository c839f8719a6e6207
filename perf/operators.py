"""Cases of the operators of a residual state-space block: group norm + activation (channels last), dropout from a counter-based
generator, and the short causal convolution and selective scan with carried states, for prompts and for single tokens.

`run` computes each operator in its plain form (elementary torch operations, 32 bits, one rounding at the end), or, where `own` is
true, through the calls that a user makes of nnuzoo_amd.  `exact` says what `run` returns, in 64 bits."""
import math
from types import SimpleNamespace as State

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS, SLOPE = 1e-5, 0.01
LARGEST = 2 * 2097152 * 32          # elements of the largest case's tensors


def listed():
    return [
        # the deep end of a small residual block with odd sizes: a training step's call is all latency
        dict(name="gn small odd", op="gn", n=3, s=63, c=60, groups=6, act="leaky_relu", dtype="f32"),
        # LightMUNet's first level at 512 x 512, batch 2, 32 filters
        dict(name="gn 512x512 bf16", op="gn", n=2, s=262144, c=32, groups=8, act="relu", dtype="bf16"),
        # the same network's first level at 128^3, batch 2
        dict(name="gn 128^3 f16", op="gn", n=2, s=2097152, c=32, groups=8, act="silu", dtype="f16"),
        # 14 x 14 tokens of two images beside their fp32 residual stream
        dict(name="dropout tokens", op="dropout", n=392, c=384, p=0.1, dtype="bf16", residual="f32"),
        # a full-resolution activation
        dict(name="dropout 512x512", op="dropout", n=524288, c=128, p=0.25, dtype="f16", residual=""),
        # one step of a small batch
        dict(name="conv token", op="conv", b=4, l=0, d=768, w=4, dtype="f32", ragged=False),
        # SegMamba's first stage: 64^3 voxels of two volumes as one sequence each
        dict(name="conv 64^3 tokens", op="conv", b=2, l=262144, d=96, w=4, dtype="f16", ragged=False),
        # one 7 x 7 image through a narrow block
        dict(name="scan 49 tokens", op="scan", b=1, l=49, d=192, h=192, g=1, n=16, dtype="f32", ragged=False),
        # five prompts of different lengths in one padded batch
        dict(name="scan ragged prompts", op="scan", b=5, l=1000, d=768, h=768, g=1, n=16, dtype="bf16", ragged=True),
        # SegMamba's first stage
        dict(name="scan 64^3 tokens", op="scan", b=2, l=262144, d=96, h=96, g=1, n=16, dtype="f16", ragged=False),
        # one token of one sequence: latency
        dict(name="scan token b1", op="scan", b=1, l=0, d=192, h=192, g=1, n=16, dtype="f32", ragged=False),
        # one token of many sequences, heads as Mamba2 has them
        dict(name="scan token b128 heads", op="scan", b=128, l=0, d=1536, h=48, g=1, n=16, dtype="bf16", ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["f32", "f16", "bf16"])
    op = rng.choice(["gn", "gn", "dropout", "conv", "scan", "scan"])
    if op == "gn":
        groups = rng.choice([1, 2, 4, 6, 8, 16, 32])
        c = groups * _log(rng, 1, 512 // groups)
        n = rng.randint(1, 8)
        s = _log(rng, 1, max(1, LARGEST // 4 // (n * c)))
        return dict(op=op, n=n, s=s, c=c, groups=groups, act=rng.choice(["none", "relu", "leaky_relu", "silu"]), dtype=dtype)
    if op == "dropout":
        c = _log(rng, 1, 1024)
        return dict(op=op, n=_log(rng, 1, LARGEST // 4 // c), c=c, p=round(rng.uniform(0.01, 0.9), 4), dtype=dtype,
                    residual=rng.choice(["", "f32", dtype]))
    token = rng.random() < 0.4
    w = rng.randint(2, 8)
    if token:
        b, d = _log(rng, 1, 256), _log(rng, 8, 2048)
    else:
        b, d = rng.randint(1, 8), _log(rng, 8, 1024)
    l = 0 if token else _log(rng, 1, max(1, (LARGEST // 4 if op == "conv" else LARGEST // 16) // (b * d)))
    ragged = not token and rng.random() < 0.5
    if op == "conv":
        return dict(op=op, b=b, l=l, d=d, w=w, dtype=dtype, ragged=ragged)
    h, g = d, 1
    if rng.random() < 0.5:          # heads and groups
        g = rng.choice([1, 2])
        h = g * rng.randint(1, 8)
        d = h * max(1, d // h)
    return dict(op=op, b=b, l=l, d=d, h=h, g=g, n=rng.choice([4, 8, 16, 16, 32]), dtype=dtype, ragged=ragged)


# ---- inputs ----------------------------------------------------------------------------------------------------------------------
def _rand(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def rn(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(shape, generator=gen, device="cuda") * scale + shift).to(dtype)
    return gen, rn


def _lengths(case, seed):
    if not case["ragged"]:
        return None
    r = np.random.RandomState(int(seed) % (1 << 31))
    v = r.randint(0, case["l"] + 1, case["b"])
    v[r.randint(case["b"])] = case["l"]
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen, rn = _rand(case, seed)
    f32 = torch.float32
    if case["op"] == "gn":
        n, s, c = case["n"], case["s"], case["c"]
        x = rn(n, s, c, scale=1.5, shift=0.3).requires_grad_(True)
        w = rn(c, scale=0.3, shift=1.0, dtype=f32).requires_grad_(True)
        b = rn(c, scale=0.2, dtype=f32).requires_grad_(True)
        return State(case=case, x=x, w=w, b=b, dy=rn(n, s, c))
    if case["op"] == "dropout":
        n, c = case["n"], case["c"]
        key = torch.tensor([int(seed) * 0x9E3779B97F4A7C15 % (1 << 63), int(seed) % 1000], dtype=torch.int64, device="cuda")
        x = rn(n, c).requires_grad_(True)
        res = rn(n, c, dtype=DTYPES[case["residual"]]).requires_grad_(True) if case["residual"] else None
        out = torch.promote_types(x.dtype, res.dtype) if res is not None else x.dtype
        return State(case=case, x=x, res=res, key=key, site=int(seed) % 7, dy=rn(n, c, dtype=out))
    b, l, d = case["b"], case["l"], case["d"]
    lengths = _lengths(case, seed)
    rows = (b, l) if l else (b,)
    xz = rn(*rows, 2 * d)           # what in_proj gives: x and z beside each other
    x, z = xz[..., :d], xz[..., d:]
    if case["op"] == "conv":
        w = case["w"]
        return State(case=case, x=x, lengths=lengths, weight=rn(d, w, scale=0.4, dtype=f32), bias=rn(d, scale=0.1, dtype=f32),
                     conv_state=rn(b, d, w))
    h, g, n = case["h"], case["g"], case["n"]
    bc = rn(*rows, 2 * g * n)       # what x_proj gives: B and C beside each other
    B, C = bc[..., :g * n].unflatten(-1, (g, n)), bc[..., g * n:].unflatten(-1, (g, n))
    dt0 = torch.exp(torch.rand(h, generator=gen, device="cuda") * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
    return State(case=case, x=x, z=z, dt=rn(*rows, h, scale=0.5), B=B, C=C, lengths=lengths,
                 A=-torch.arange(1, n + 1, device="cuda", dtype=f32) * (1 + 0.1 * torch.rand(h, n, generator=gen, device="cuda")),
                 D=rn(h, scale=0.1, shift=1.0, dtype=f32), dt_bias=dt0 + torch.log(-torch.expm1(-dt0)),
                 state=rn(b, d, n, scale=0.5, dtype=f32))


# ---- the plain forms -------------------------------------------------------------------------------------------------------------
def _gn(x, w, b, dy, groups, act):
    dt = x.dtype
    n, s, c = x.shape
    xg = x.float().view(n, s, groups, c // groups)
    xc = xg - xg.mean((1, 3), keepdim=True)
    rstd = torch.rsqrt(xc.square().mean((1, 3), keepdim=True) + EPS)
    xh = (xc * rstd).view(n, s, c)
    z = xh * w + b
    g = dy.float()
    if act == "relu":
        y, dz = z.clamp(min=0), g * (z > 0)
    elif act == "leaky_relu":
        y, dz = torch.where(z > 0, z, z * SLOPE), torch.where(z > 0, g, g * SLOPE)
    elif act == "silu":
        sg = 1 / (1 + torch.exp(-z))
        y, dz = z * sg, g * sg * (1 + z * (1 - sg))
    else:
        y, dz = z, g
    db, dw = dz.sum((0, 1)), (dz * xh).sum((0, 1))
    t, xh = (dz * w).view(n, s, groups, -1), xh.view(n, s, groups, -1)
    dx = rstd * (t - t.mean((1, 3), keepdim=True) - xh * (t * xh).mean((1, 3), keepdim=True))
    return [y.to(dt), dx.view(n, s, c).to(dt), dw, db]


M32 = 0xFFFFFFFF


def _philox(c0, c1, c2, c3, k0, k1):
    """Philox-4x32-10 (Salmon, Moraes, Dror, Shaw 2011) on int64 tensors that hold 32-bit words"""
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (p1 >> 32 & M32) ^ c1 ^ k0, p1 & M32, (p0 >> 32 & M32) ^ c3 ^ k1, p0 & M32
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    return torch.stack((c0, c1, c2, c3), -1)


def _halves(words):
    return torch.stack((words & 0xFFFF, words >> 16), -1).flatten(-3)


def _kept(key, site, count, p):
    """whether element e is kept: 16 bits of the call for block e // 8 above 16 bits of the block's second call, against p"""
    blk = torch.arange((count + 7) // 8, device=key.device)
    lo, hi = blk & M32, blk >> 32
    k0, k1, step = key[0] & M32, key[0] >> 32 & M32, (key[1] & M32).expand_as(lo)
    where = torch.full_like(lo, site)
    u = _halves(_philox(lo, hi, where, step, k0, k1)) << 16 | _halves(_philox(lo, hi | 0x80000000, where, step, k0, k1))
    return u[:count] >= round(p * 2 ** 32)


def _dropout(s):
    x, p = s.x.detach(), s.case["p"]
    kept = _kept(s.key, s.site, x.numel(), p).view(x.shape)
    y = torch.where(kept, x.float() * (1 / (1 - p)), 0.0)
    dx = torch.where(kept, s.dy.float() * (1 / (1 - p)), 0.0).to(x.dtype)
    if s.res is None:
        return [y.to(x.dtype), dx]
    return [(y + s.res.detach().float()).to(s.dy.dtype), dx, s.dy.to(s.res.dtype)]


def _valid(lengths, l):
    return (torch.arange(l, device=lengths.device) < lengths[:, None])[..., None]


def _conv(s):
    x = s.x if s.case["l"] else s.x[:, None]
    w, l = s.case["w"], x.shape[1]
    hist = torch.cat((s.conv_state.transpose(1, 2), x), 1)          # (B, W + L, D)
    acc = s.bias + (torch.stack([hist[:, 1 + j:1 + j + l].float() * s.weight[:, j] for j in range(w)])).sum(0)
    y = acc / (1 + torch.exp(-acc))
    end = torch.full((x.shape[0],), l, device=x.device) if s.lengths is None else s.lengths.long()
    if s.lengths is not None:
        y = torch.where(_valid(s.lengths, l), y, 0.0)
    at = (end[:, None] + torch.arange(w, device=x.device))[..., None].expand(-1, -1, x.shape[2])
    s.conv_state.copy_(torch.gather(hist, 1, at).transpose(1, 2))
    y = y.to(x.dtype)
    return [y if s.case["l"] else y[:, 0], s.conv_state]


def _scan(s):
    x, z, dt, B, C = (t if s.case["l"] else t[:, None] for t in (s.x, s.z, s.dt, s.B, s.C))
    b, l, d = x.shape
    rep, grp = d // s.case["h"], d // s.case["g"]
    dl = dt.float() + s.dt_bias
    dl = (dl.clamp(min=0) + torch.log1p(torch.exp(-dl.abs()))).repeat_interleave(rep, -1)
    xf = x.float()
    if s.lengths is not None:       # a token behind its sequence changes nothing
        ok = _valid(s.lengths, l)
        dl, xf = torch.where(ok, dl, 0.0), torch.where(ok, xf, 0.0)
    Bf, Cf = (t.float().repeat_interleave(grp, 2) for t in (B, C))  # (B, L, D, N)
    if s.lengths is not None:
        Bf = torch.where(ok[..., None], Bf, 0.0)
    a = torch.exp(dl[..., None] * s.A.repeat_interleave(rep, 0))
    h = (dl * xf)[..., None] * Bf
    del Bf
    h[:, 0] += a[:, 0] * s.state
    step = 1
    while step < l:                 # h_t <- h_t + a_t h_{t - step}, a_t <- a_t a_{t - step}: all prefixes in log2(L) rounds
        h = torch.cat((h[:, :step], h[:, step:] + a[:, step:] * h[:, :-step]), 1)
        a = torch.cat((a[:, :step], a[:, step:] * a[:, :-step]), 1)
        step *= 2
    del a
    zf = z.float()
    y = ((h * Cf).sum(-1) + s.D.repeat_interleave(rep) * x.float()) * (zf / (1 + torch.exp(-zf)))
    if s.lengths is not None:
        y = torch.where(ok, y, 0.0)
    s.state.copy_(h[:, -1])
    y = y.to(x.dtype)
    return [y if s.case["l"] else y[:, 0], s.state]


# ---- one pass --------------------------------------------------------------------------------------------------------------------
def run(state):
    s, case = state, state.case
    op = case["op"]
    if not own:
        if op == "gn":
            return _gn(s.x.detach(), s.w.detach(), s.b.detach(), s.dy, case["groups"], case["act"])
        return {"dropout": _dropout, "conv": _conv, "scan": _scan}[op](s)
    if op == "gn":
        from nnuzoo_amd.group_norm import group_norm_act
        y = group_norm_act(s.x, case["groups"], s.w, s.b, EPS, activation=case["act"], negative_slope=SLOPE)
        return [y.detach(), *torch.autograd.grad(y, (s.x, s.w, s.b), s.dy)]
    if op == "dropout":
        from nnuzoo_amd.dropout import dropout, dropout_add
        if s.res is None:
            y = dropout(s.x, case["p"], s.key, site=s.site)
            return [y.detach(), *torch.autograd.grad(y, (s.x,), s.dy)]
        y = dropout_add(s.x, s.res, case["p"], s.key, site=s.site)
        return [y.detach(), *torch.autograd.grad(y, (s.x, s.res), s.dy)]
    from nnuzoo_amd import mamba_state as ms
    if op == "conv":
        if case["l"]:
            return [ms.causal_conv1d_prompt(s.x, s.weight, s.bias, "silu", conv_state=s.conv_state, lengths=s.lengths),
                    s.conv_state]
        return [ms.causal_conv1d_token(s.x, s.conv_state, s.weight, s.bias, "silu"), s.conv_state]
    if case["l"]:
        return [ms.selective_scan_prompt(s.x, s.dt, s.A, s.B, s.C, s.D, z=s.z, dt_bias=s.dt_bias, dt_softplus=True,
                                         state=s.state, lengths=s.lengths), s.state]
    return [ms.selective_scan_token(s.x, s.dt, s.A, s.B, s.C, s.D, z=s.z, dt_bias=s.dt_bias, dt_softplus=True, state=s.state),
            s.state]


def work(case):
    e, op = BYTES[case["dtype"]], case["op"]
    if op == "gn":                  # x, dy in; y, dx out
        m = case["n"] * case["s"] * case["c"]
        return {"bytes": 4 * m * e + 4 * case["c"] * 4, "flops": m * (20 if case["act"] == "silu" else 14)}
    if op == "dropout":             # x, dy (and the residual) in; y, dx out
        m = case["n"] * case["c"]
        r = BYTES[case["residual"]] if case["residual"] else 0
        return {"bytes": m * (2 * e + 2 * max(e, r) + r + (r if r and r != max(e, r) else 0)), "flops": 3 * m}
    rows = case["b"] * max(1, case["l"]) * (0.6 if case["ragged"] else 1)
    if op == "conv":
        m = rows * case["d"]
        return {"bytes": 2 * m * e + 2 * case["b"] * case["d"] * case["w"] * e + case["d"] * (case["w"] + 1) * 4,
                "flops": m * (2 * case["w"] + 4)}
    m, n = rows * case["d"], case["n"]
    return {"bytes": 3 * m * e + rows * (case["h"] + 2 * case["g"] * n) * e + 2 * case["b"] * case["d"] * n * 4
            + case["h"] * (n + 2) * 4, "flops": m * (7 * n + 10)}


# ---- in 64 bits ------------------------------------------------------------------------------------------------------------------
def _exact_gn(s):
    case = s.case
    n, m, c = s.x.shape
    q = c // case["groups"]
    x, w, b, g = (t.detach().double() for t in (s.x, s.w, s.b, s.dy))
    ys, dxs, dw, db = [], [], 0, 0
    for i in range(n):              # one sample at a time
        xi, gi = x[i], g[i]
        var, mean = torch.var_mean(xi.reshape(m, -1, q), (0, 2), correction=0)
        mean, sd = mean.repeat_interleave(q), (var + EPS).sqrt().repeat_interleave(q)
        xh = (xi - mean) / sd
        z = w * xh + b
        if case["act"] == "silu":
            y, slope = z * z.sigmoid(), z.sigmoid() + z * z.sigmoid() * z.neg().sigmoid()
        else:
            low = {"none": 1.0, "relu": 0.0, "leaky_relu": SLOPE}[case["act"]]
            slope = torch.where(z > 0, 1.0, low).double()
            y = z * slope
        dz = gi * slope
        db, dw = db + dz.sum(0), dw + (xh * dz).sum(0)
        u = w * dz
        m1 = u.mean(0).view(-1, q).mean(1).repeat_interleave(q)
        m2 = (u * xh).mean(0).view(-1, q).mean(1).repeat_interleave(q)
        ys.append(y)
        dxs.append((u - m1 - xh * m2) / sd)
    return [torch.stack(ys), torch.stack(dxs), dw, db]


def _mul32(a, k):
    """high and low words of a 32 x 32 bit product from 16-bit limbs"""
    k0, k1 = k & 0xFFFF, k >> 16
    a0, a1 = torch.bitwise_and(a, 0xFFFF), torch.bitwise_right_shift(a, 16)
    mid = a1 * k0 + torch.bitwise_right_shift(a0 * k0, 16)
    mid2 = a0 * k1 + torch.bitwise_and(mid, 0xFFFF)
    high = a1 * k1 + torch.bitwise_right_shift(mid, 16) + torch.bitwise_right_shift(mid2, 16)
    low = torch.bitwise_and(mid2, 0xFFFF) * 65536 + torch.bitwise_and(a0 * k0, 0xFFFF)
    return high, low


def _draws(seed, step, site, first, count, second):
    """16-bit draws of elements first .. first + count - 1 (first % 8 == 0)"""
    blk = torch.arange(first // 8, first // 8 + (count + 7) // 8, device="cuda")
    v = [blk % 2 ** 32, blk // 2 ** 32 + (2 ** 31 if second else 0), torch.full_like(blk, site), torch.full_like(blk, step % 2 ** 32)]
    keys = [seed % 2 ** 32, seed // 2 ** 32 % 2 ** 32]
    for r in range(10):
        h0, l0 = _mul32(v[0], 0xD2511F53)
        h1, l1 = _mul32(v[2], 0xCD9E8D57)
        v = [h1 ^ v[1] ^ ((keys[0] + r * 0x9E3779B9) % 2 ** 32), l1, h0 ^ v[3] ^ ((keys[1] + r * 0xBB67AE85) % 2 ** 32), l0]
    out = torch.empty((blk.numel(), 8), dtype=torch.int64, device="cuda")
    for j in range(8):
        out[:, j] = v[j // 2] // 65536 if j % 2 else v[j // 2] % 65536
    return out.flatten()[:count]


def _exact_dropout(s):
    x, dy, p = s.x.detach().double().flatten(), s.dy.double().flatten(), s.case["p"]
    seed, step = (int(v) for v in s.key.tolist())
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    part = 1 << 25
    for i in range(0, x.numel(), part):
        k = min(part, x.numel() - i)
        drop = _draws(seed, step, s.site, i, k, False) * 65536 + _draws(seed, step, s.site, i, k, True) < round(p * 4294967296)
        y[i:i + k] = (x[i:i + k] / (1 - p)).masked_fill(drop, 0)
        dx[i:i + k] = (dy[i:i + k] / (1 - p)).masked_fill(drop, 0)
    y, dx = y.view(s.x.shape), dx.view(s.x.shape)
    return [y, dx] if s.res is None else [y + s.res.detach().double(), dx, s.dy.double()]


def _exact_conv(s):
    x = s.x.double() if s.case["l"] else s.x.double()[:, None]
    w, l = s.case["w"], x.shape[1]
    y, end = torch.zeros_like(x), []
    for i in range(x.shape[0]):
        m = l if s.lengths is None else int(s.lengths[i])
        seen = torch.cat((s.conv_state[i].double(), x[i, :m].t()), 1)       # (D, W + m)
        acc = s.bias.double()[:, None].repeat(1, m)
        for j in range(w):
            acc += s.weight.double()[:, j:j + 1] * seen[:, j + 1:j + 1 + m]
        y[i, :m] = (acc * acc.sigmoid()).t()
        end.append(seen[:, m:])
    return [y if s.case["l"] else y[:, 0], torch.stack(end)]


def _exact_scan(s):
    x, z, dt, B, C = (t.double() if s.case["l"] else t.double()[:, None] for t in (s.x, s.z, s.dt, s.B, s.C))
    b, l, d = x.shape
    rep, grp = d // s.case["h"], d // s.case["g"]
    A, Dv = s.A.double().repeat_interleave(rep, 0), s.D.double().repeat_interleave(rep)
    dl = torch.nn.functional.softplus(dt + s.dt_bias.double()).repeat_interleave(rep, 2)
    if s.lengths is not None:
        dl = dl * (torch.arange(l, device=x.device) < s.lengths[:, None])[..., None]
    m = max(1, math.isqrt(l))       # pieces of m tokens: all pieces at once from zero, then their entry states, then again
    pieces = -(-l // m)

    def cut(t):
        t = torch.cat((t, t.new_zeros((b, pieces * m - l) + t.shape[2:])), 1)
        return t.view((b, pieces, m) + t.shape[2:])
    xs, ds, Bs, Cs = cut(x), cut(dl), cut(B), cut(C)

    def step(h, t):
        u = ds[:, :, t]
        return torch.exp(u[..., None] * A) * h + (u * xs[:, :, t])[..., None] * Bs[:, :, t].repeat_interleave(grp, 2)
    h = x.new_zeros((b, pieces) + A.shape)
    for t in range(m):
        h = step(h, t)
    decay = torch.exp(ds.sum(2)[..., None] * A)
    entry, at = torch.empty_like(h), s.state.double()
    for i in range(pieces):
        entry[:, i] = at
        at = decay[:, i] * at + h[:, i]
    y, h = torch.empty_like(xs), entry
    for t in range(m):
        h = step(h, t)
        y[:, :, t] = (h * Cs[:, :, t].repeat_interleave(grp, 2)).sum(-1)
    y = (y.reshape(b, pieces * m, d)[:, :l] + Dv * x) * z * z.sigmoid()
    if s.lengths is not None:
        y = y * (torch.arange(l, device=x.device) < s.lengths[:, None])[..., None]
    return [y if s.case["l"] else y[:, 0], at]


def exact(case, seed):
    s = prepare(case, seed)
    return {"gn": _exact_gn, "dropout": _exact_dropout, "conv": _exact_conv, "scan": _exact_scan}[case["op"]](s)
