"""8-bit floating point calls whose tensors lie beside each other in one buffer give the bytes that tensors of their own give; shared bytes
are refused and nothing is written."""
import pytest
import torch

from tests.helpers.fp8_oracle import blocks, make_rows, make_weight
from zse_b200.ops.fp8 import Fp8Rows, Fp8Weight

pytestmark = pytest.mark.gpu
DEV, F8, U8 = "cuda", torch.float8_e4m3fn, torch.uint8


@pytest.fixture(scope="module")
def ops():
    from zse_b200.ops.backend import make_ops
    return make_ops(DEV)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def same(a, b):
    return torch.equal(a.data.view(U8), b.data.view(U8)) and torch.equal(a.scale, b.scale)


def side_by_side(x, M, columns):
    """x as the left columns of a buffer, and rows to be written as the right ones; their scales as well."""
    K = x.data.shape[1]
    data = torch.zeros(M, K + columns, dtype=U8, device=DEV)
    n = max(blocks(K), blocks(columns))
    scale = torch.zeros(n, 2 * M, device=DEV)
    data[:, :K] = x.data[:M].view(U8)
    scale[: blocks(K), :M] = x.scale[:, :M]
    return (Fp8Rows(data[:, :K].view(F8), scale[: blocks(K), :M]), Fp8Rows(data[:, K:].view(F8), scale[: blocks(columns), M:]))


@pytest.mark.parametrize("M", [1, 40, 600])
def test_side_by_side(ops, M):
    K, ff = 512, 144
    g = gen(M)
    x, up = make_rows(g, M, K, DEV, hot=False), make_weight(g, ff, K, DEV, glu=True)
    want = Fp8Rows.empty(M, ff, DEV)
    ops.linear_swiglu_fp8(up, x, M, want)
    xs, out = side_by_side(x, M, ff)
    ops.linear_swiglu_fp8(up, xs, M, out)
    assert same(out, want) and same(xs, x)
    h = torch.randn(M, K, generator=g).to(DEV)
    ops.quant_fp8(h, M, x)
    whole = torch.zeros(M, 4 * K + K + 4 * blocks(K), dtype=U8, device=DEV)          # a row: fp32 numbers, its bytes, and no scales
    hs = whole[:, : 4 * K].view(torch.float32)
    hs.copy_(h)
    rows = Fp8Rows(whole[:, 4 * K: 5 * K].view(F8), torch.empty(blocks(K), M, device=DEV))
    ops.quant_fp8(hs, M, rows)
    assert same(rows, x) and torch.equal(hs, h)


def test_one_after_the_other(ops):
    """A workspace that holds everything of a run, each piece where the one before ends."""
    M, H, ff = 24, 256, 384
    g = gen(2)
    room, at = torch.zeros(1 << 22, dtype=U8, device=DEV), 0

    def put(t):
        nonlocal at
        t = t.contiguous()
        n = t.numel() * t.element_size()
        place = room[at: at + n].view(t.dtype).view(t.shape)
        place.view(U8).copy_(t.to(DEV).view(U8))
        at += n
        return place

    def rows(columns):
        return Fp8Rows(put(torch.zeros(M, columns, dtype=U8)).view(F8), put(torch.zeros(blocks(columns), M)))
    up, down = make_weight(g, ff, H, "cpu", glu=True), make_weight(g, H, ff, "cpu", torch.float32)
    start, w16 = torch.randn(M, H, generator=g), torch.ones(H).half()
    runs = []
    for place in (lambda t: t.to(DEV), put):
        r, w, x, h, plane = place(start), place(w16), None, None, place(torch.zeros(1, M, H))
        x, h = (rows(H), rows(ff)) if place is put else (Fp8Rows.empty(M, H, DEV), Fp8Rows.empty(M, ff, DEV))
        normed = place(torch.zeros(M, H).half())
        u = Fp8Weight(place(up.data.view(U8)).view(F8), place(up.scale), None, True)
        d = Fp8Weight(place(down.data.view(U8)).view(F8), place(down.scale), place(down.bias))
        ops.add_rmsnorm_fp8(r, None, 0, normed, w, x, M, 1e-6, normed=normed)
        ops.linear_swiglu_fp8(u, x, M, h)
        ops.linear_fp8(d, h, M, plane[0])
        ops.add_rmsnorm_fp8(r, plane, 1, None, w, x, M, 1e-6)
        runs.append((r, x, h, plane, normed))
    (r, x, h, plane, normed), (r2, x2, h2, plane2, normed2) = runs
    assert torch.equal(r, r2) and same(x, x2) and same(h, h2) and torch.equal(plane, plane2) and torch.equal(normed, normed2)


@pytest.mark.parametrize("M", [5, 600])
def test_shared_bytes_are_refused(ops, M):
    from zse_b200.ops.native import NativeError
    K = 256
    g = gen(3)
    x, up, w = make_rows(g, M, K, DEV, hot=False), make_weight(g, K, K, DEV, glu=True), make_weight(g, K, K, DEV)
    out, h, a = Fp8Rows.empty(M, K, DEV), torch.randn(M, K, generator=g).to(DEV), torch.zeros(M, K, device=DEV).half()
    ones, narrow = torch.ones(K, device=DEV).half(), make_weight(g, 2, K, DEV)
    as_f8 = lambda t: t.view(U8)[:, :K].view(F8)                                     # noqa: E731
    calls = [
        lambda: ops.linear_swiglu_fp8(up, x, M, Fp8Rows(out.data, x.scale)),
        lambda: ops.linear_swiglu_fp8(up, Fp8Rows(x.data, out.scale), M, out),
        lambda: ops.linear_fp8(narrow, x, M, x.scale.view(M, 2)),
        lambda: ops.linear_fp8(w, x, 5, w.data.view(torch.bfloat16).view(-1, K)),
        lambda: ops.quant_fp8(h, M, Fp8Rows(out.data, h.view(-1)[: 2 * M].view(2, M))),
        lambda: ops.add_rmsnorm_fp8(h, None, 0, a, ones, Fp8Rows(as_f8(a), out.scale), M, 1e-6),
        lambda: ops.add_rmsnorm_fp8(h, None, 0, a, ones, Fp8Rows(as_f8(h), out.scale), M, 1e-6),
        lambda: ops.add_rmsnorm_fp8(h, h.view(1, M, K), 1, None, ones, out, M, 1e-6),
        lambda: ops.add_rmsnorm_fp8(h, None, 0, None, ones, Fp8Rows(out.data, h.view(-1)[: 2 * M].view(2, M)), M, 1e-6),
        lambda: ops.add_rmsnorm_fp8(h[:-1], None, 0, a[:-1], ones, out, M - 1, 1e-6, normed=a[1:]),
    ]
    kept = [t.clone() for t in (x.data.view(U8), x.scale, w.data.view(U8), h, a)]
    for call in calls:
        with pytest.raises(NativeError):
            call()
    torch.cuda.synchronize()
    assert all(torch.equal(t, k) for t, k in zip((x.data.view(U8), x.scale, w.data.view(U8), h, a), kept))
