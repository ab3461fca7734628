"""The operators on 8-bit floating point in 64 bits, and how far from that a result may be.

A rounding to e4m3 is off by at most half a step, 2^-4 of the largest power of two below the number, or 2^-10 where it is below 2^-6; a
rounding to fp32 by 2^-24, to bfloat16 by 2^-8 and to fp16 by 2^-11 of the number.
"""
import math

import torch

F64 = torch.float64
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def blocks(n):
    return -(-n // 128)


def make_rows(g, M, K, device, hot=True):
    """Rows in 8 bits as a quantisation leaves them: blocks whose largest is 448, scales over some powers of two."""
    from zse_b200.ops.fp8 import Fp8Rows
    x = torch.randn(M, blocks(K) * 128, generator=g).view(M, -1, 128)
    x = (x / x.abs().amax(-1, keepdim=True) * 448).view(M, -1)[:, :K].to(torch.float8_e4m3fn)
    scale = torch.exp2(torch.randn(blocks(K), M, generator=g) * (2 if hot else 0)) * 0.01
    return Fp8Rows(x.contiguous().to(device), scale.to(device))


def make_weight(g, N, K, device, bias=None, glu=False):
    from zse_b200.ops.fp8 import Fp8Weight
    w = torch.randn((2 if glu else 1) * N, K, generator=g) * (2 / math.sqrt(K))
    b = None if bias is None else torch.randn(N, generator=g).to(bias).to(device)
    q = Fp8Weight.from_dense(w, glu=glu)
    return Fp8Weight(q.data.to(device), q.scale.to(device), b, glu)


def values(rows, M):
    return rows.data[:M].to(F64) * rows.scale[:, :M].to(F64).t().repeat_interleave(128, 1)[:, : rows.data.shape[1]]


def weight(w):
    """[parts of one N each] of the weight in 64 bits."""
    parts = 2 if w.glu else 1
    n = w.data.shape[0] // parts
    out = []
    for p in range(parts):
        s = w.scale[p * blocks(n): (p + 1) * blocks(n)].to(F64)
        out.append(w.data[p * n: (p + 1) * n].to(F64) * s.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, : w.data.shape[1]])
    return out


def product(x, w, on_cpu=False):
    """(x w^T, how far a sum in fp32 may be off) in 64 bits.  A block's 128 products, exact each, are added by four instructions of 32
    whose adder may cut instead of round: 33 numbers a time, 2^-23 of what is added.  Then every block costs a product of the scales, a
    product with it and a sum, 2^-24 each.  (On the CPU: the two values rounded, K products and sums.)"""
    K = x.shape[1]
    off = (K + 6) * 2.0 ** -24 if on_cpu else 4 * 33 * 2.0 ** -23 + (blocks(K) + 3) * 2.0 ** -24
    return x @ w.t(), off * (x.abs() @ w.abs().t())


def gated(g, u, g_off, u_off, gelu):
    """act(g) u, and its bound.  Neither activation is steeper than 1.2; in fp32 it is off by the exponential's few units (the argument of
    gelu's by some more), a sum, a quotient and the product: 2^-20 of the result and, where z is large, 2^-22 |z| of it."""
    z = 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3) if gelu else g
    a = g * torch.sigmoid(z)
    y = a * u
    return y, 1.2 * g_off * u.abs() + a.abs() * u_off + 1.2 * g_off * u_off + y.abs() * (2.0 ** -20 + 2.0 ** -22 * z.abs().clamp_max(110))


def norm(residual, weight_, eps):
    r = residual.to(F64)
    return r / (r.square().mean(-1, keepdim=True) + eps).sqrt() * weight_.to(F64)


def check_rows(y, off, rows, M):
    """Rows in 8 bits that are y up to ``off`` (a number per element, or a share of it): each scale is the block's largest over 448 up to
    what the largest may be off and two roundings to fp32; each element is the nearest to y / scale up to off / scale and three such
    roundings (448 / largest, the product, the scale itself)."""
    C = y.shape[1]
    data, scale = rows.data[:M].to(F64), rows.scale[:, :M].to(F64).t()
    off = off * y.abs() if isinstance(off, float) else off
    fill = lambda t: torch.nn.functional.pad(t, (0, blocks(C) * 128 - C)).view(M, -1, 128)     # noqa: E731
    top, top_off = fill(y).abs().amax(-1), fill(off).amax(-1)
    assert ((scale - top / 448).abs() <= (top_off / 448 + 2 * 2.0 ** -24 * top)).all()
    none = (scale == 0).repeat_interleave(128, 1)[:, :C]
    assert (data[none] == 0).all() and (top[scale == 0] <= 1e-30 + top_off[scale == 0]).all()
    s = scale.clamp_min(1e-300).repeat_interleave(128, 1)[:, :C]
    v = torch.where(none, torch.zeros_like(y), y / s)
    half = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 4)
    slack = torch.where(none, torch.zeros_like(y), off / s) + 4 * 2.0 ** -24 * v.abs()
    # (where the number lies just below a power of two, slack can take it into the next, wider steps)
    over = torch.exp2(torch.floor(torch.log2((v.abs() + slack).clamp_min(2.0 ** -6))) - 4)
    bad = (data - v).abs() > torch.maximum(half, over) + slack
    assert not bad.any(), (int(bad.sum()), torch.nonzero(bad)[:4].tolist(), data[bad][:4].tolist(), v[bad][:4].tolist())


def check_out(y, off, out):
    """A result in ``out``'s type that is y up to ``off``: one more rounding, and fp16's numbers below 2^-14 have steps of 2^-24."""
    t = out.dtype
    if t is torch.float16:
        y = y.clamp(-65504, 65504)
    tol = off + HALF[t] * (y.abs() + off) + (2.0 ** -25 if t is torch.float16 else 1e-37)
    bad = ~((out.to(F64) - y).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), torch.nonzero(bad)[:4].tolist(), out[bad][:4].tolist(), y[bad][:4].tolist())
