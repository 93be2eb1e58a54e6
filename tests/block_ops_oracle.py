"""Values and error bounds of the block operators in 64 bits, for the tests of both devices.

A rounding to type T errs by at most u(T) = finfo(T).eps / 2 of the value; every bound below is a sum
of such roundings.
"""
import math

import torch

F64 = torch.float64
E4M3 = torch.float8_e4m3fn


def u(dtype):
    return torch.finfo(dtype).eps / 2


def norm_quant(x, w, r, eps):
    """(q unrounded, scale, h as stored) in 64 bits."""
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    f = h.to(F64)
    y = f / torch.sqrt((f * f).mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * w.to(F64)
    scale = (y.abs().amax(-1) / 448.0).clamp_min(1e-30)
    return y / scale[..., None], scale, h


# fp32 sums of squares over a row: a thread adds at most 64 terms in turn and a tree of 10 levels
# joins them (a longer row's threads add dim / 1024 <= 64 here), which rsqrt halves; the scale and the
# reciprocal add a few roundings more: 64 * 2^-24 covers them.
NORM_REL = 64 * 2.0 ** -24


def check_norm_quant(got, x, w, r, eps):
    q, s, h = got
    tq, ts, th = norm_quant(x, w, r, eps)
    assert q.dtype == E4M3 and s.dtype == torch.float32 and q.shape == x.shape and s.shape == x.shape[:-1]
    if r is None:
        assert h is None
    else:
        assert h.dtype == x.dtype and torch.equal(h, th)
    assert ((s.to(F64) - ts).abs() <= NORM_REL * ts).all()
    # e4m3: half a step is 2^-4 of a normal value and 2^-10 below 2^-6
    err = (q.float().to(F64) - tq).abs()
    assert (err <= tq.abs() * (u(E4M3) + 2 * NORM_REL) + 2.0 ** -10).all(), err.max()


def linear(xq, xs, wq, ws, b=None, act=None, residual=None, gate_rows=None):
    """(y, bound on the fp32 part of the error) in 64 bits; gate_rows [M, N]."""
    K = xq.shape[-1]
    x, w = xq.float().to(F64), wq.float().to(F64)
    s = xs.to(F64)[:, None] * ws.to(F64)
    y = (x @ w.T) * s
    # products of e4m3 are exact in fp32; each of the K / 32 steps of the sum may lose 2 units in the last
    # place of the sum so far (<= sum |x w|), joining the parts a few more; scales and bias: 4 roundings
    err = (x.abs() @ w.abs().T) * s * (K / 32 + 16) * 2.0 ** -22
    if b is not None:
        y = y + b.to(F64)
        err = err + y.abs() * 2.0 ** -22
    if act == "gelu":
        t = torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
        # slope below 1.13; the 16-bit forms take tanh within 2^-10.9, the fp32 form errs by a few ulp
        y, err = 0.5 * y * (1 + t), 1.13 * err + y.abs() * (2.0 ** -11.9)
    if gate_rows is not None:
        y, err = y * gate_rows.to(F64), err * gate_rows.to(F64).abs()
    if residual is not None:
        y = y + residual.to(F64)
        err = err + y.abs() * 2.0 ** -22
    return y, err


def check_linear(got, want, err):
    bound = err * (1 + u(got.dtype)) + want.abs() * u(got.dtype) + torch.finfo(got.dtype).tiny
    d = (got.to(F64) - want).abs()
    assert (d <= bound).all(), (d / bound).max()


def rope(x, pos, dims, head_dim, theta, layout, inverse):
    """(y, |x0| + |x1| of every rotated element) in 64 bits, pair by pair."""
    f = x.to(F64).reshape(x.shape[0], -1, head_dim)
    y, size = f.clone(), torch.zeros_like(f)
    p = pos.to(F64).repeat(x.shape[0] // pos.shape[0], 1)
    i, n = 0, sum(dims) // 2
    for a, d in enumerate(dims):
        for j in range(d // 2):
            angle = p[:, a] * theta[a] ** (-2.0 * j / d) * (-1 if inverse else 1)
            c, s = angle.cos()[:, None], angle.sin()[:, None]
            e0, e1 = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
            y[..., e0] = f[..., e0] * c - f[..., e1] * s
            y[..., e1] = f[..., e0] * s + f[..., e1] * c
            size[..., e0] = size[..., e1] = f[..., e0].abs() + f[..., e1].abs()
            i += 1
    return y.reshape(x.shape), size.reshape(x.shape)


def check_rope(got, x, pos, dims, head_dim, theta, layout="interleaved", inverse=False):
    y, size = rope(x, pos, dims, head_dim, theta, layout, inverse)
    # cos and sin in fp32: the reduced angle 2^-23 of up to pi, the functions 2 ulp, two products and a sum;
    # the phase in 64 bits: 2^-51 of the angle on either side
    far = float(pos.to(F64).abs().max()) * 2.0 ** -50 if pos.numel() else 0.0
    bound = size * (12 * 2.0 ** -24 + far) + y.abs() * u(got.dtype) * 1.001 + torch.finfo(got.dtype).tiny
    d = (got.to(F64) - y).abs()
    assert got.dtype == x.dtype and (d <= bound).all(), (d / bound).max()


def cross(q, k, v, heads, heads_kv, allowed, scale):
    """(o, lse, bound on o, bound on lse) in 64 bits; allowed bool [B, Sk]."""
    B, Sq, width = q.shape
    d, T = width // heads, q.dtype
    o = torch.zeros(B, Sq, width, dtype=F64, device=q.device)
    ob = torch.zeros_like(o)
    lse = torch.full((B, heads, Sq), -math.inf, dtype=F64, device=q.device)
    lb = torch.zeros_like(lse)
    for b in range(B):
        keep = allowed[b].nonzero()[:, 0]
        if not keep.numel():
            continue
        for h in range(heads):
            at = slice(h * d, (h + 1) * d)
            g = h // (heads // heads_kv)
            kv = slice(g * d, (g + 1) * d)
            qq, kk, vv = q[b, :, at].to(F64), k[b, keep][:, kv].to(F64), v[b, keep][:, kv].to(F64)
            s = qq @ kk.T * scale
            # scores: products exact in fp32, d / 16 steps of the sum, scaling and base change 4 roundings
            es = (qq.abs() @ kk.abs().T).amax(-1) * scale * (d / 16 + 8) * 2.0 ** -22
            p = torch.softmax(s, -1)
            o[b, :, at] = p @ vv
            size = p @ vv.abs()
            # p rounded to T (u each, below T's smallest normal an absolute tiny * 2u), exponentials 2^-22,
            # the sums over the keys; the weights' errors count against sum p |v|, the total's against |o|
            n = keep.numel()
            rel = u(T) + 4 * es[:, None] + (n / 16 + 32) * 2.0 ** -22
            small = n * torch.finfo(T).tiny * 2 * u(T) * vv.abs().amax(0)
            ob[b, :, at] = size * rel + small + o[b, :, at].abs() * (rel - u(T) + u(T) * 1.01) + torch.finfo(T).tiny
            lse[b, h] = torch.logsumexp(s, -1)
            lb[b, h] = 2 * es + (n / 16 + 32) * 2.0 ** -22 + lse[b, h].abs() * 2.0 ** -22
    return o, lse, ob, lb


def check_cross(got, got_lse, q, k, v, heads, heads_kv=None, allowed=None, scale=None):
    heads_kv = heads_kv or heads
    if allowed is None:
        allowed = torch.ones(k.shape[:2], dtype=torch.bool, device=k.device)
    scale = scale or 1 / math.sqrt(q.shape[-1] // heads)
    o, lse, ob, lb = cross(q, k, v, heads, heads_kv, allowed, scale)
    assert got.dtype == q.dtype and got.shape == q.shape
    d = (got.to(F64) - o).abs()
    assert (d <= ob).all(), (d / ob.clamp_min(1e-30)).max()
    if got_lse is not None:
        assert got_lse.dtype == torch.float32 and got_lse.shape == lse.shape
        none = lse == -math.inf
        assert torch.equal(got_lse == -math.inf, none)
        e = (got_lse.to(F64) - lse).abs()[~none]
        assert (e <= lb[~none]).all(), (e / lb[~none]).max()
    empty = ~allowed.any(1)
    assert not got[empty].any()
