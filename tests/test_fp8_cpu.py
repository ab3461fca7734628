"""The operators on 8-bit floating point without a GPU: their torch forms against 64 bits, what they refuse, rows and weights."""
import pytest
import torch

from tests.helpers.fp8_oracle import (check_out, check_rows, gated, make_rows, make_weight, norm, product, values, weight)
from zse_b200.ops.backend import TorchOps
from zse_b200.ops.fp8 import Fp8Rows, Fp8Weight

F8 = torch.float8_e4m3fn


@pytest.fixture()
def ops():
    return TorchOps("cpu")


def gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("H", [16, 144, 384])
@pytest.mark.parametrize("planes,add", [(0, False), (1, False), (3, True)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_norm(ops, H, planes, add, dtype):
    g, M = gen(H + planes), 5
    r, w = torch.randn(M + 1, H, generator=g) * 3, (1 + torch.randn(H, generator=g) * 0.2).to(dtype)
    r[2] = 0
    p = torch.randn(planes, M, H, generator=g) if planes else None
    a = torch.randn(M, H, generator=g).to(dtype) if add else None
    if p is not None:
        p[:, 2] = 0
    if add:
        a[2] = 0
    total = r[:M].double() + (p.double().sum(0) if planes else 0) + (a.double() if add else 0)
    out, normed, last = Fp8Rows.empty(M, H), torch.empty(M, H, dtype=dtype), r[M].clone()
    ops.add_rmsnorm_fp8(r, p, planes, a, w, out, M, 1e-6, normed=normed)
    assert torch.equal(r[:M], total.float()) and torch.equal(r[M], last)
    y = norm(r[:M], w, 1e-6)
    check_rows(y, 5 * 2.0 ** -24, out, M)
    check_out(y, 5 * 2.0 ** -24 * y.abs(), normed)
    assert (out.scale[:, 2] == 0).all() and (out.data[2].float() == 0).all()


@pytest.mark.parametrize("C", [16, 128, 272])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_quant_and_gated(ops, C, dtype):
    g, M = gen(C), 6
    x = (torch.randn(M + 2, 2 * C, generator=g) * 3).to(dtype)
    out = Fp8Rows(torch.full((M + 2, C), 3.0).to(F8), torch.full((-(-C // 128), M + 2), 7.0))
    ops.quant_fp8(x[:, :C], M, out)
    check_rows(x[:M, :C].double(), 0.0, out, M)
    assert (out.data[M:].float() == 3).all() and (out.scale[:, M:] == 7).all()
    for gelu in (False, True):
        ops.swiglu_fp8(x, M, out, gelu=gelu)
        y, off = gated(x[:M, :C].double(), x[:M, C:].double(), 0.0, 0.0, gelu)
        check_rows(y, off, out, M)


@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (3, 130, 144), (5, 48, 384)])
@pytest.mark.parametrize("dtype,bias", [(torch.float16, torch.float16), (torch.bfloat16, None), (torch.float32, torch.float32)])
def test_linear(ops, M, N, K, dtype, bias):
    g = gen(M + N + K)
    x, w = make_rows(g, M + 1, K, "cpu"), make_weight(g, N, K, "cpu", bias)
    x.scale[:, M] = float("nan")
    out = torch.full((M + 1, N + 3), 5.0, dtype=dtype)
    ops.linear_fp8(w, x, M, out)
    y, off = product(values(x, M), weight(w)[0], on_cpu=True)
    if bias is not None:
        y = y + w.bias.double()
        off = off + 2.0 ** -24 * y.abs()
    check_out(y, off, out[:M, :N])
    assert (out[M:] == 5).all() and (out[:, N:] == 5).all()


@pytest.mark.parametrize("M,ff,K,gelu", [(1, 16, 16, False), (4, 144, 272, True), (3, 128, 128, False)])
def test_linear_swiglu(ops, M, ff, K, gelu):
    g = gen(M + ff)
    x, w = make_rows(g, M, K, "cpu", hot=False), make_weight(g, ff, K, "cpu", glu=True)
    out = Fp8Rows.empty(M, ff)
    ops.linear_swiglu_fp8(w, x, M, out, gelu=gelu)
    (gate, g_off), (up, u_off) = (product(values(x, M), p, on_cpu=True) for p in weight(w))
    y, off = gated(gate, up, g_off, u_off, gelu)
    check_rows(y, off, out, M)


def test_weight_from_dense():
    g = gen(1)
    for n, k, glu in ((130, 200, False), (288, 144, True)):
        d = torch.randn(n, k, generator=g)
        d[:128, :128] = 0
        w = Fp8Weight.from_dense(d, glu=glu)
        parts = torch.cat(weight(w))
        half = torch.maximum(2.0 ** -4 * d.abs(), 2.0 ** -10 * d.abs().max() / 448).double()
        assert ((parts - d.double()).abs() <= half * (1 + 2.0 ** -20)).all()
        assert torch.equal(w.dequant().double().float(), parts.float())
        assert w.scale[0, 0] == 0 and (w.N, w.K) == (n, k)


def test_rows_of_infinities_and_nans(ops):
    x = torch.randn(3, 256, generator=gen(2))
    x[0, 5], x[1, 200] = float("inf"), float("nan")
    out = Fp8Rows.empty(3, 256)
    ops.quant_fp8(x, 3, out)
    y = out.dequant()
    assert y[0, :128].isnan().all() and y[1, 128:].isnan().all()
    assert y[0, 128:].isfinite().all() and y[1, :128].isfinite().all() and y[2].isfinite().all()


def test_nothing_to_do(ops):
    out, before = Fp8Rows(torch.ones(2, 32).to(F8), torch.ones(1, 2)), torch.ones(2, 32)
    ops.quant_fp8(torch.zeros(2, 32), 0, out)
    ops.add_rmsnorm_fp8(torch.zeros(2, 32), None, 0, None, torch.ones(32).half(), out, 0, 1e-6)
    w = Fp8Weight.from_dense(torch.ones(64, 32), glu=True)
    ops.linear_swiglu_fp8(w, out, 0, out)
    assert torch.equal(out.data.float(), before)


def test_refusals(ops):
    rows, wide = Fp8Rows.empty(4, 128), Fp8Rows.empty(4, 256)
    r, w16 = torch.zeros(4, 128), torch.ones(128).half()
    w, glu = Fp8Weight.from_dense(torch.ones(32, 128)), Fp8Weight.from_dense(torch.ones(64, 128), glu=True)
    for make in (lambda: Fp8Rows(torch.zeros(4, 128), torch.zeros(1, 4)), lambda: Fp8Weight(torch.zeros(4, 128), torch.zeros(1, 1))):
        with pytest.raises(TypeError):
            make()
    bad = [
        lambda: Fp8Rows(rows.data, torch.zeros(4, 1)),
        lambda: Fp8Weight(w.data, torch.zeros(2, 1)),
        lambda: Fp8Weight(w.data, w.scale, torch.zeros(31)),
        lambda: Fp8Weight(w.data, w.scale, torch.zeros(32, dtype=torch.float64)),
        lambda: Fp8Weight(glu.data, glu.scale, torch.zeros(64), glu=True),
        lambda: Fp8Weight.from_dense(torch.ones(33, 128), glu=True),
        lambda: ops.add_rmsnorm_fp8(r, None, 0, None, w16, rows, 5, 1e-6),                     # more rows than there are
        lambda: ops.add_rmsnorm_fp8(r, None, 0, None, w16, rows, -1, 1e-6),
        lambda: ops.add_rmsnorm_fp8(r, None, 0, None, w16, wide, 4, 1e-6),                     # out of another width
        lambda: ops.add_rmsnorm_fp8(r.half(), None, 0, None, w16, rows, 4, 1e-6),
        lambda: ops.add_rmsnorm_fp8(r, None, 1, None, w16, rows, 4, 1e-6),                     # planes that are not there
        lambda: ops.add_rmsnorm_fp8(r, torch.zeros(3, 128), 1, None, w16, rows, 4, 1e-6),
        lambda: ops.add_rmsnorm_fp8(r, None, 0, torch.zeros(4, 128).bfloat16(), w16, rows, 4, 1e-6),   # two 16-bit types
        lambda: ops.add_rmsnorm_fp8(r, None, 0, None, w16.float(), rows, 4, 1e-6),
        lambda: ops.add_rmsnorm_fp8(r, None, 0, None, w16[:64], rows, 4, 1e-6),
        lambda: ops.add_rmsnorm_fp8(torch.zeros(4, 256)[:, :128], None, 0, None, w16, rows, 4, 1e-6),
        lambda: ops.add_rmsnorm_fp8(r, None, 0, None, w16, rows, 4, 1e-6, normed=torch.zeros(4, 128)),
        lambda: ops.quant_fp8(torch.zeros(4, 120), 4, Fp8Rows.empty(4, 120)),                  # no multiple of 16
        lambda: ops.quant_fp8(torch.zeros(4, 256), 4, rows),
        lambda: ops.quant_fp8(torch.zeros(4, 128, dtype=torch.float64), 4, rows),
        lambda: ops.quant_fp8(torch.zeros(128, 4).t(), 4, rows),
        lambda: ops.swiglu_fp8(torch.zeros(4, 128), 4, rows),
        lambda: ops.linear_fp8(w, wide, 4, torch.zeros(4, 32)),                                # another K
        lambda: ops.linear_fp8(w, rows, 4, torch.zeros(4, 31)),
        lambda: ops.linear_fp8(w, rows, 4, torch.zeros(3, 32)),
        lambda: ops.linear_fp8(w, rows, 5, torch.zeros(5, 32)),
        lambda: ops.linear_fp8(w, rows, 4, torch.zeros(4, 32, dtype=torch.float64)),
        lambda: ops.linear_fp8(w, rows, 4, torch.zeros(32, 4).t()),
        lambda: ops.linear_fp8(glu, rows, 4, torch.zeros(4, 64)),
        lambda: ops.linear_swiglu_fp8(w, rows, 4, Fp8Rows.empty(4, 16)),
        lambda: ops.linear_swiglu_fp8(glu, rows, 4, Fp8Rows.empty(4, 64)),
        lambda: ops.linear_swiglu_fp8(glu, rows, 4, Fp8Rows.empty(3, 32)),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()


def test_layer(ops):
    """Norm, gate and up, down, norm: the run of them as a feed-forward uses them, each step on what the one before left."""
    g, M, H, ff = gen(3), 7, 144, 272
    r, w16 = torch.randn(M, H, generator=g), (1 + torch.randn(H, generator=g) * 0.1).half()
    up, down = make_weight(g, ff, H, "cpu", glu=True), make_weight(g, H, ff, "cpu")
    x, h, plane = Fp8Rows.empty(M, H), Fp8Rows.empty(M, ff), torch.empty(1, M, H)
    ops.add_rmsnorm_fp8(r, None, 0, None, w16, x, M, 1e-6)
    ops.linear_swiglu_fp8(up, x, M, h)
    ops.linear_fp8(down, h, M, plane[0])
    before = r.clone()
    ops.add_rmsnorm_fp8(r, plane, 1, None, w16, x, M, 1e-6)
    y, off = product(values(h, M), weight(down)[0], on_cpu=True)
    check_out(y, off, plane[0])
    assert torch.equal(r, before + plane[0])
    check_rows(norm(r, w16, 1e-6), 5 * 2.0 ** -24, x, M)


def test_refusals_of_the_entries():
    """What the C entries refuse before they touch a GPU (the addresses are not read)."""
    from zse_b200.ops import native as n
    lib = n.load()
    at = [(i + 1) << 30 for i in range(9)]
    SHAPE, ALIGN, LIMIT = -1, -2, -5

    def quant(x=at[0], data=at[1], ldx=64, ld=64, M=4, C=64, act=0, kind=2):
        return lib.zse_quant_fp8(n.QUANT_FP8.pack(x, data, at[2], 0, ldx, ld, M, M, C, act, kind))

    def gemm(x=at[0], w=at[2], bias=0, out=at[5], ldx=64, ldw=64, ldo=64, M=4, N=64, K=64, kind=2, act=0):
        return lib.zse_gemm_fp8(n.GEMM_FP8.pack(x, at[1], w, at[3], bias, out, at[6], at[7], 0, ldx, ldw, ldo, M, M, M, N, K, kind, 2, act))

    def rms(M=4, H=64, data=at[2], ld=64, weight=at[1]):
        return lib.zse_add_rmsnorm_fp8(n.NORM_FP8.pack(at[0], 0, 0, weight, 0, data, at[3], 0, ld, M, 1e-6, 0, M, H, 0))
    assert quant(C=60) == quant(act=3) == quant(kind=3) == SHAPE
    assert quant(x=at[0] + 8) == quant(ldx=66) == quant(data=at[1] + 8) == quant(ld=72) == ALIGN
    assert quant(M=(1 << 30) + 1) == quant(C=(1 << 30) + 16) == LIMIT
    assert quant(data=at[0]) == quant(data=at[0] + 3 * 256 + 240) == quant(x=at[1] + 3 * 64 + 48) == SHAPE       # bytes of both
    assert gemm(N=0) == gemm(K=72) == gemm(act=3) == gemm(act=1, N=72) == gemm(act=1, bias=at[4]) == SHAPE
    assert gemm(x=at[0] + 8) == gemm(w=at[2] + 4) == gemm(ldx=72) == gemm(ldw=72) == gemm(out=at[5] + 2) == gemm(bias=at[4] + 2) == ALIGN
    assert gemm(act=1, out=at[5] + 8) == gemm(act=1, ldo=72) == ALIGN
    assert gemm(M=(1 << 30) + 1) == gemm(N=(1 << 30) + 1) == gemm(act=1, N=(1 << 29) + 16) == gemm(K=(1 << 30) + 16) == LIMIT
    assert gemm(out=at[0], ldx=0, ldo=0) == gemm(out=at[0]) == gemm(out=at[0] + 48) == gemm(act=1, out=at[0] + 32, ldx=128, ldo=128) == SHAPE
    assert rms(H=60) == rms(weight=0) == SHAPE
    assert rms(data=at[2] + 8) == rms(ld=72) == rms(weight=at[1] + 2) == ALIGN
    assert rms(H=32784) == rms(M=(1 << 30) + 1) == LIMIT
