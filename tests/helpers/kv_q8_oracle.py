"""The 8-bit KV cache in 64 bits, written from its definition: what the operators' results are compared with."""
import math

import torch

F64 = torch.float64


def make_cache(gen, blocks, nkv, bs, hd, device):
    """A cache that earlier passes have filled: quantised normal rows, key channels and value heads of different size."""
    size = torch.stack([torch.exp(0.6 * torch.randn(nkv, 1, hd, generator=gen)),
                        torch.exp(0.5 * torch.randn(nkv, 1, 1, generator=gen)).expand(nkv, 1, hd) * 0.4])
    x = torch.randn(blocks, 2, nkv, bs, hd, generator=gen) * size
    top = x.abs().amax(-1)
    u = torch.round(x * (127 / top)[..., None]) + 128
    return u.to(torch.uint8).to(device), (top / 127).to(device)


def make_tables(gen, lens, bs, blocks, device, width=None, holes=()):
    """Tables of sequences over shuffled blocks; ``holes``: (sequence, block) pairs that are dropped."""
    need = [-(-n // bs) for n in lens]
    perm = torch.randperm(blocks, generator=gen, dtype=torch.int32)
    assert sum(need) <= blocks
    t = torch.full((max(1, len(lens)), width or max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        t[s, :n] = perm[at: at + n]
        at += n
    for s, b in holes:
        t[s, b] = -1
    return t.to(device)


def rotated(x, positions, freqs, nh, nkv, hd):
    """Rows x [M, (nh + 2 nkv) * hd] -> heads [M, nh + 2 nkv, hd] with q and k rotated, and |a| + |b| of every element's pair."""
    h = x.to(F64).view(x.shape[0], nh + 2 * nkv, hd).clone()
    half = freqs.numel()
    ang = positions.to(F64)[:, None, None] * freqs.to(F64)
    pair = h.abs()
    a, b = h[:, : nh + nkv, :half].clone(), h[:, : nh + nkv, half: 2 * half].clone()
    h[:, : nh + nkv, :half] = a * torch.cos(ang) - b * torch.sin(ang)
    h[:, : nh + nkv, half: 2 * half] = b * torch.cos(ang) + a * torch.sin(ang)
    both = a.abs() + b.abs()
    pair[:, : nh + nkv, :half] = both
    pair[:, : nh + nkv, half: 2 * half] = both
    return h, pair


def check_write(x, positions, freqs, nh, nkv, hd, q, u, scale):
    """``q`` [M, nh * hd], ``u`` [M, 2, nkv, hd] and ``scale`` [M, 2, nkv] as stored, against 64 bits.

    q: half a step of fp16 (2^-11 of the value, 2^-25 below its normal range), and what fp32 adds: the angle rounded to 24 bits
    within one turn (at most 2^-23), sine and cosine (2^-23), two products and a sum (3 * 2^-24 of |a| + |b|): 2^-21 of |a| + |b|.
    u: |x| / scale <= 127, so those 2^-21 of |a| + |b| <= 2 max|x| are 127 * 2^-20 steps in x and in max|x|, and three roundings
    to 24 bits 127 * 2^-22: below 1e-3 beside the half step.  scale: 2^-20 of it from max|x|, 2^-24 from the division."""
    h, pair = rotated(x, positions, freqs, nh, nkv, hd)
    M = x.shape[0]
    h = h.clamp(-65504, 65504)
    want, off = h[:, :nh].reshape(M, -1), pair[:, :nh].reshape(M, -1)
    assert ((q.to(F64) - want).abs() <= want.abs() * 2.0 ** -11 + off * 2.0 ** -21 + 2.0 ** -25).all()
    y = h[:, nh:].view(M, 2, nkv, hd)
    top = y.abs().amax(-1)
    assert ((scale.to(F64) * 127 - top).abs() <= top * 2.0 ** -19).all()
    unit = torch.where(top > 0, 127 / top, torch.zeros_like(top))[..., None]
    assert ((u.to(F64) - 128 - y * unit).abs() <= 0.5 + 1e-3).all()
    assert u.min() >= 1


def attention(q, data, scale, tables, rows, nh, softmax_scale, window=0):
    """``rows``: (sequence, tokens seen) of every row of q.  Returns the result in 64 bits and how far it may be off: half a step of
    the result (2^-11); of every weight the 2^-22 that two fp16 numbers leave, the products' error in its exponent (the bytes'
    products are summed in fp32 with an offset of 128, 24 rounded sums of at most sum|q| * 255 * scale), and 2^-18 for the
    exponential, the running sums and scales in fp32; T * 2^-26 for T / 16 truncated sums of a row; and what lies below the range of
    fp16 (2^-25 each, where the largest weight times value scale is counted as 32 or more): T * 2^-30 of the largest weight times value."""
    nkv, bs, hd = data.shape[2], data.shape[3], data.shape[4]
    out = torch.zeros(len(rows), nh * hd, dtype=F64, device=q.device)
    tol = torch.zeros_like(out)
    for i, (s, n) in enumerate(rows):
        at = torch.arange(n, device=q.device)
        ids = tables[s][at // bs].long()
        at, ids = at[ids >= 0], ids[ids >= 0]
        if window:
            keep = at >= n - window
            at, ids = at[keep], ids[keep]
        if not len(at):
            continue
        k, v = ((data[ids, j, :, at % bs].to(F64) - 128) * scale[ids, j, :, at % bs].to(F64)[..., None] for j in (0, 1))
        qi = q[i, : nh * hd].to(F64).view(nkv, nh // nkv, hd)
        p = torch.softmax(torch.einsum("hgd,thd->hgt", qi, k) * softmax_scale, -1)
        o = torch.einsum("hgt,thd->hgd", p, v)
        size = torch.einsum("hgt,thd->hgd", p, v.abs())
        spread = qi.abs().sum(-1) * 255 * scale[ids, 0, :, at % bs].to(F64).amax(0)[:, None] * softmax_scale * 24 * 2.0 ** -24
        T = len(at)
        out[i] = o.reshape(-1)
        tol[i] = (o.abs() * 2.0 ** -11 + size * (2.0 ** -22 + 2 * spread[..., None] + 2.0 ** -18 + T * 2.0 ** -26)
                  + T * 2.0 ** -30 * torch.einsum("hgt,th->hgt", p, v.abs().amax(2)).amax(2)[..., None] + 2.0 ** -25).reshape(-1)
    return out, tol


def scale_of(hd):
    return 1.0 / math.sqrt(hd)
