"""Plain 64-bit restatements (CPU, test-only) of the operators of a residual state-space block: group norm + activation with its
gradient, the draws of the counter-based dropout, the causal convolution and the selective scan with carried states.  Each returns
its values together with a bound on what a computation in fp32 may be off by (the output's own rounding not included)."""
from __future__ import annotations

import numpy as np
import torch

U = 2.0 ** -24      # half a unit in the last place of fp32


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def close(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    """|got - want| <= bound + half a step of got's type at want (and the type's smallest steps near zero); NaN where NaN"""
    g, w = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    tiny = 0.0 if got.dtype == torch.float64 else torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    tol = bound + (w.abs() + bound) * half_step(got.dtype) + tiny
    nan = torch.isnan(w)
    assert torch.equal(nan, torch.isnan(g)), f"{what}: NaN in different places"
    bad = ((g - w).abs() > tol) & ~nan & (g != w)
    if bad.any():
        i = int(((g - w).abs() - tol).masked_fill(~bad, -1).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off; worst {g.flatten()[i]} for {w.flatten()[i]}, "
                             f"allowed {tol.flatten()[i]:.3g}")


# ---- group norm + activation -----------------------------------------------------------------------------------------------------
def _act(z, act, slope):
    """value, derivative, bound on |act'| around z"""
    if act == "relu":
        return z.clamp(min=0), (z > 0).double(), torch.ones_like(z)
    if act == "leaky_relu":
        d = torch.where(z > 0, 1.0, slope).double()
        return z * d, d, torch.ones_like(z)
    if act == "silu":
        s = z.sigmoid()
        return z * s, s * (1 + z * (1 - s)), torch.full_like(z, 1.1)
    return z, torch.ones_like(z), torch.ones_like(z)


def group_norm_act(x, groups, w, b, eps, act, slope, dy, additions=512):
    """x, dy (N, S, C), w, b (C,) or None.  -> {name: (value, bound)} for y, dx, dw, db.
    `additions`: the longest chain of fp32 additions in a sum of the backward (rows of a thread + threads of a workgroup)."""
    x, dy = x.double().cpu(), dy.double().cpu()
    N, S, C = x.shape
    q = C // groups
    w = torch.ones(C, dtype=torch.float64) if w is None else w.double().cpu()
    b = torch.zeros(C, dtype=torch.float64) if b is None else b.double().cpu()
    xg = x.view(N, S, groups, q)
    mean = xg.mean((1, 3), keepdim=True)
    var = (xg - mean).square().mean((1, 3), keepdim=True)
    r = (var + eps).rsqrt()
    full = lambda t: t.expand(N, S, groups, q).reshape(N, S, C)  # noqa: E731
    mean_f, r_f = full(mean), full(r)
    xh = (x - mean_f) * r_f
    z = xh * w + b
    # mean and r are rounded once each, then a subtraction, two products and a sum; E[x^2] - mean^2 in fp64 leaves 2^-50 of E[x^2]
    e_var = 2.0 ** -50 * (mean_f.square() + full(var)) * r_f.square()
    e_xh = U * mean_f.abs() * r_f + xh.abs() * (4 * U + e_var)
    e_z = e_xh * w.abs() + 3 * U * ((xh * w).abs() + b.abs())
    y, d, dmax = _act(z, act, slope)
    e_sig = (z.abs() + 6) * 2 * U          # exp of a rounded product, a sum and a reciprocal
    e_y = e_z * dmax + (y.abs() * (e_sig + 2 * U) if act == "silu" else 2 * U * y.abs())
    dz = dy * d
    near = (z.abs() <= 4 * e_z) if act in ("relu", "leaky_relu") else torch.zeros_like(z, dtype=torch.bool)
    e_dz = dy.abs() * (e_z + (e_sig * (1 + z.abs()) * 2 if act == "silu" else 0)) * (0.5 if act == "silu" else 0) \
        + 2 * U * dz.abs() + near * dy.abs()
    t = w * dz
    tg, txg = t.view(N, S, groups, q), (t * xh).view(N, S, groups, q)
    m1, m2 = full(tg.mean((1, 3), keepdim=True)), full(txg.mean((1, 3), keepdim=True))
    e_t = w.abs() * e_dz
    gm = lambda v: full(v.view(N, S, groups, q).mean((1, 3), keepdim=True))  # noqa: E731
    e_m1 = gm(e_t) + additions * U * gm(t.abs())
    e_m2 = gm(e_t * xh.abs() + t.abs() * e_xh) + additions * U * gm((t * xh).abs())
    dx = r_f * (t - m1 - xh * m2)
    size = t.abs() + m1.abs() + (xh * m2).abs()
    e_dx = r_f * (e_t + e_m1 + xh.abs() * e_m2 + m2.abs() * e_xh + 6 * U * size) + 2 * U * dx.abs()
    s = lambda v: v.sum((0, 1))  # noqa: E731
    return {"y": (y, e_y), "dx": (dx, e_dx),
            "dw": (s(dz * xh), s(e_dz * xh.abs() + dz.abs() * e_xh) + additions * U * s((dz * xh).abs())),
            "db": (s(dz), s(e_dz) + additions * U * s(dz.abs()))}


# ---- dropout ---------------------------------------------------------------------------------------------------------------------
def philox4x32(counter, key, rounds=10):
    """Philox-4x32 (Salmon et al. 2011): counter (..., 4) and key (..., 2) of uint32 words -> (..., 4)"""
    c = [np.asarray(counter)[..., i].astype(np.uint64) for i in range(4)]
    k = [np.asarray(key)[..., i].astype(np.uint64) for i in range(2)]
    m = np.uint64(0xFFFFFFFF)
    for _ in range(rounds):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ k[0], p1 & m, (p0 >> np.uint64(32)) ^ c[3] ^ k[1], p0 & m]
        k = [(k[0] + np.uint64(0x9E3779B9)) & m, (k[1] + np.uint64(0xBB67AE85)) & m]
    return np.stack(c, -1)


def dropout_draws(seed, step, site, first, count):
    """32-bit draws of elements first .. first + count - 1 (first a multiple of 8)"""
    blk = np.arange(first // 8, first // 8 + (count + 7) // 8, dtype=np.uint64)
    ctr = np.zeros(blk.shape + (4,), dtype=np.uint64)
    ctr[:, 0], ctr[:, 1] = blk & np.uint64(0xFFFFFFFF), blk >> np.uint64(32)
    ctr[:, 2], ctr[:, 3] = site, step & 0xFFFFFFFF
    key = np.array([seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF], dtype=np.uint64)
    out = []
    for flag in (0, 0x80000000):
        c = ctr.copy()
        c[:, 1] |= np.uint64(flag)
        w = philox4x32(c, np.broadcast_to(key, c.shape[:1] + (2,)))
        out.append(np.stack((w & np.uint64(0xFFFF), w >> np.uint64(16)), -1).reshape(-1))
    return torch.from_numpy(((out[0] << np.uint64(16)) | out[1]).astype(np.int64))[:count]


def dropout_kept(seed, step, site, count, p, first=0):
    return dropout_draws(seed, step, site, first, count) >= round(p * 2 ** 32)


# ---- causal convolution and selective scan with states ---------------------------------------------------------------------------
def _silu(v, e):
    s = v.sigmoid()
    return v * s, 1.1 * e + (v * s).abs() * ((v.abs() + 6) * 2 * U + 2 * U)


def causal_conv(x, w, b, silu, state, lengths):
    """x (B, L, D), w (D, W), state (B, D, W) or None, lengths list -> (y, bound), new state"""
    x, w = x.double().cpu(), w.double().cpu()
    B, L, D = x.shape
    W = w.shape[1]
    b = torch.zeros(D, dtype=torch.float64) if b is None else b.double().cpu()
    hist = torch.zeros(B, D, W, dtype=torch.float64) if state is None else state.double().cpu().clone()
    y, e = torch.zeros(B, L, D, dtype=torch.float64), torch.zeros(B, L, D, dtype=torch.float64)
    for i in range(B):
        for t in range(lengths[i]):
            hist[i] = torch.cat((hist[i][:, 1:], x[i, t][:, None]), 1)
            s = b + (w * hist[i]).sum(1)
            es = (W + 1) * U * (b.abs() + (w * hist[i]).abs().sum(1))
            y[i, t], e[i, t] = _silu(s, es) if silu else (s, es)
    return (y, e), hist


def selective_scan(x, dt, A, Bm, C, D, z, dt_bias, softplus, state, lengths, join=0):
    """x (B, L, D), dt (B, L, H), A (H, N) or (H,), Bm / C (B, L, G, N) -> (y, bound), (state, bound).
    `join`: tokens of the chunks that a fast implementation cuts the sequence into (their decays multiply, their time steps add up)"""
    x, dt, Bm, C = (t.double().cpu() for t in (x, dt, Bm, C))
    B, L, d = x.shape
    H, (G, N) = dt.shape[-1], Bm.shape[-2:]
    A = A.double().cpu()
    A = (A[:, None].expand(H, N) if A.dim() == 1 else A).repeat_interleave(d // H, 0)
    per = lambda t: torch.zeros(d, dtype=torch.float64) if t is None else t.double().cpu().repeat_interleave(d // H)  # noqa: E731
    Dv, bias = per(D), per(dt_bias)
    h = torch.zeros(B, d, N, dtype=torch.float64) if state is None else state.double().cpu().clone()
    eh = torch.zeros_like(h)
    y, e = torch.zeros_like(x), torch.zeros_like(x)
    for i in range(B):
        for t in range(lengths[i]):
            raw = dt[i, t].repeat_interleave(d // H) + bias
            dl = torch.nn.functional.softplus(raw, threshold=1e9) if softplus else raw
            # rounding of dt + bias, then (softplus) exp, reciprocal, series: relative to the result
            e_raw = U * raw.abs()
            e_dl = (e_raw * raw.sigmoid() + 8 * U * dl.abs()) if softplus else e_raw
            a = torch.exp(dl[:, None] * A)
            e_a = a * ((dl[:, None] * A).abs() * 4 * U + A.abs() * e_dl[:, None] + 2 * U)
            bb, cc = Bm[i, t].repeat_interleave(d // G, 0), C[i, t].repeat_interleave(d // G, 0)
            u = dl * x[i, t]
            e_u = e_dl * x[i, t].abs() + U * u.abs()
            new = a * h[i] + u[:, None] * bb
            eh[i] = a * eh[i] + e_a * h[i].abs() + e_a * eh[i] + e_u[:, None] * bb.abs() + 3 * U * ((a * h[i]).abs() + (u[:, None] * bb).abs())
            if join and (t + 1) % join == 0:
                eh[i] = eh[i] + new.abs() * join * U
            h[i] = new
            s = (new * cc).sum(1) + Dv * x[i, t]
            es = (eh[i] * cc.abs()).sum(1) + (N + 3) * U * ((new * cc).abs().sum(1) + (Dv * x[i, t]).abs())
            if z is not None:
                zz = z[i, t].double().cpu()
                g, eg = _silu(zz, torch.zeros_like(zz))
                y[i, t], e[i, t] = s * g, es * g.abs() + s.abs() * eg + 2 * U * (s * g).abs()
            else:
                y[i, t], e[i, t] = s, es
    return (y, e), (h, eh)


def causal_conv_rows(x, w, b, silu, state, lengths):
    """causal_conv for all sequences and tokens at once; the same values and bounds"""
    x, w = x.double().cpu(), w.double().cpu()
    B, L, D = x.shape
    W = w.shape[1]
    b = torch.zeros(D, dtype=torch.float64) if b is None else b.double().cpu()
    state = torch.zeros(B, D, W, dtype=torch.float64) if state is None else state.double().cpu()
    seen = torch.cat((state.transpose(1, 2), x), 1)                     # token t lies at W + t
    s, size = b.expand(B, L, D).clone(), b.abs().expand(B, L, D).clone()
    for j in range(W):
        term = w[:, j] * seen[:, 1 + j:1 + j + L]
        s += term
        size += term.abs()
    es = (W + 1) * U * size
    y, e = _silu(s, es) if silu else (s, es)
    n = torch.as_tensor(lengths)
    there = (torch.arange(L) < n[:, None])[..., None]
    at = (n[:, None] + torch.arange(W))[..., None].expand(B, W, D)
    zero = torch.zeros((), dtype=torch.float64)
    return (torch.where(there, y, zero), torch.where(there, e, zero)), seen.gather(1, at).transpose(1, 2)


def selective_scan_rows(x, dt, A, Bm, C, D, z, dt_bias, softplus, state, lengths, join=0):
    """selective_scan for all sequences at once.  `join`: tokens of the chunks that a fast implementation cuts the sequences into: the
    state behind a chunk is exp(A sum of D_t) entry + the chunk's own, so that beside the recurrence's roundings the sum of `join` time
    steps counts, (join - 1) U of itself, through the exponential (A sum D exp(A sum D) entry), and the roundings of the joining
    itself: |A sum D| 4 U + 2 U of the exponential, one of the FMA"""
    x, dt, Bm, C = (t.double().cpu() for t in (x, dt, Bm, C))
    B, L, d = x.shape
    H, (G, N) = dt.shape[-1], Bm.shape[-2:]
    A = A.double().cpu()
    A = (A[:, None].expand(H, N) if A.dim() == 1 else A).repeat_interleave(d // H, 0)
    per = lambda t: torch.zeros(d, dtype=torch.float64) if t is None else t.double().cpu().repeat_interleave(d // H)  # noqa: E731
    Dv, bias = per(D), per(dt_bias)
    h = torch.zeros(B, d, N, dtype=torch.float64) if state is None else state.double().cpu().clone()
    z = None if z is None else z.double().cpu()
    eh = torch.zeros_like(h)
    y, e = torch.zeros_like(x), torch.zeros_like(x)
    n = torch.as_tensor(lengths)
    entry, steps = h, torch.zeros(B, d, dtype=torch.float64)            # at the chunk's first token; sum of its time steps
    for t in range(int(n.max())):
        on = n > t
        o2, o3 = on[:, None], on[:, None, None]
        raw = dt[:, t].repeat_interleave(d // H, -1) + bias
        dl = torch.nn.functional.softplus(raw, threshold=1e9) if softplus else raw
        e_raw = U * raw.abs()
        e_dl = (e_raw * raw.sigmoid() + 8 * U * dl.abs()) if softplus else e_raw
        dA = dl[..., None] * A
        a = torch.exp(dA)
        e_a = a * (dA.abs() * 4 * U + A.abs() * e_dl[..., None] + 2 * U)
        bb, cc = Bm[:, t].repeat_interleave(d // G, 1), C[:, t].repeat_interleave(d // G, 1)
        u = dl * x[:, t]
        e_u = e_dl * x[:, t].abs() + U * u.abs()
        term = u[..., None] * bb
        new = a * h + term
        e_new = a * eh + e_a * (h.abs() + eh) + e_u[..., None] * bb.abs() + 3 * U * ((a * h).abs() + term.abs())
        steps = steps + dl
        if join and (t + 1) % join == 0:
            sA = (steps[..., None] * A).abs()
            kept = torch.exp(steps[..., None] * A) * entry.abs()
            e_new = e_new + kept * (sA * (join + 3) * U + 2 * U) + U * new.abs()
            entry, steps = new, torch.zeros_like(steps)
        h, eh = torch.where(o3, new, h), torch.where(o3, e_new, eh)
        s = (new * cc).sum(-1) + Dv * x[:, t]
        es = (e_new * cc.abs()).sum(-1) + (N + 3) * U * ((new * cc).abs().sum(-1) + (Dv * x[:, t]).abs())
        if z is not None:
            g, eg = _silu(z[:, t], torch.zeros_like(z[:, t]))
            s, es = s * g, es * g.abs() + s.abs() * eg + 2 * U * (s * g).abs()
        y[:, t], e[:, t] = torch.where(o2, s, torch.zeros_like(s)), torch.where(o2, es, torch.zeros_like(es))
    return (y, e), (h, eh)
