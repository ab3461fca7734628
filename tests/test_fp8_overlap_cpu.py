"""The operators on 8-bit floating point refuse, before anything is launched, what they write sharing bytes with anything else of the
call: rows, scales, planes, weights, a bias.  (The addresses are made up and are not read.)"""
import pytest

from zse_b200.ops import native as n

SHAPE = -1
AT = [(i + 1) << 30 for i in range(9)]
M, H = 6, 256                                                               # two blocks of columns


def norm(residual=AT[0], planes=AT[1], add=AT[2], weight=AT[3], normed=AT[4], data=AT[5], scale=AT[6], ld=H, ld_scale=M, n_planes=2, M=M):
    return n.load().zse_add_rmsnorm_fp8(n.NORM_FP8.pack(residual, planes, add, weight, normed, data, scale, 0, ld, ld_scale, 1e-6, n_planes, M, H, 0))


def quant(x=AT[0], data=AT[1], scale=AT[2], ldx=H, ld=H, ld_scale=M, C=H, act=0, kind=2, M=M):
    return n.load().zse_quant_fp8(n.QUANT_FP8.pack(x, data, scale, 0, ldx, ld, ld_scale, M, C, act, kind))


def gemm(x=AT[0], sx=AT[1], w=AT[2], sw=AT[3], bias=AT[4], out=AT[5], out_scale=0, ldx=H, ldw=H, ldo=H, ld_sx=M, ld_os=M, M=M, N=H, K=H, act=0):
    return n.load().zse_gemm_fp8(n.GEMM_FP8.pack(x, sx, w, sw, bias, out, out_scale, AT[7], 0, ldx, ldw, ldo, ld_sx, ld_os, M, N, K, 2, 2, act))


def gated(out_scale=AT[6], **c):
    return gemm(bias=0, out_scale=out_scale, act=1, **c)


LAST = (M - 1) * H                                                          # bytes before the last of M rows of H bytes


@pytest.mark.parametrize("call", [
    dict(data=AT[0]), dict(data=AT[0] + 4 * LAST + 3 * H), dict(data=AT[1] + 4 * (2 * M * H - 4)), dict(data=AT[2]), dict(data=AT[2] + 2 * LAST),
    dict(data=AT[3] + H), dict(data=AT[4]), dict(data=AT[6]), dict(add=AT[5] + LAST),
    dict(scale=AT[0] + 4), dict(scale=AT[1] + 4 * M * H), dict(scale=AT[2] + 2 * M * H - 4), dict(scale=AT[3] + 2 * H - 4),
    dict(scale=AT[0] - 40, ld_scale=10), dict(scale=AT[4]),
    dict(normed=AT[2] + 2 * H), dict(normed=AT[2] - 16), dict(normed=AT[0]), dict(normed=AT[1] + 4 * M * H), dict(normed=AT[3]),
    dict(residual=AT[1]), dict(residual=AT[1] + 4 * M * H), dict(residual=AT[2]), dict(residual=AT[3]),
    dict(add=AT[1] + 64, normed=AT[1] + 64), dict(add=AT[3], normed=AT[3]), dict(add=AT[0], normed=AT[0]), dict(add=AT[6], normed=AT[6]),
    dict(normed=AT[2], data=AT[2] + 16), dict(M=1, data=AT[2]), dict(M=1, normed=AT[2] + 16),
])
def test_norm(call):
    assert norm(**call) == SHAPE


@pytest.mark.parametrize("call", [
    dict(data=AT[0]), dict(scale=AT[0]), dict(scale=AT[0] + 4 * M * H - 4), dict(scale=AT[0] - 4 * M), dict(scale=AT[1]), dict(scale=AT[1] + LAST + H - 4),
    dict(scale=AT[0] + 4 * H - 4, ldx=H + 16, ld_scale=4 * (H + 16)),
    dict(act=1, ldx=2 * H, scale=AT[0] + 8 * M * H - 4), dict(M=1, scale=AT[0]), dict(M=1, data=AT[0] + 3 * H),
    dict(x=AT[1] + 16, M=1),
])
def test_quant(call):
    assert quant(**call) == SHAPE


@pytest.mark.parametrize("call", [
    dict(out=AT[0]), dict(out=AT[1]), dict(out=AT[1] + 4 * (2 * M - 1)), dict(out=AT[1] - 4 * M * H + 4), dict(out=AT[2]), dict(out=AT[2] + H * H - 16),
    dict(out=AT[3]), dict(out=AT[3] + 12), dict(out=AT[4]), dict(out=AT[4] + 4 * H - 4), dict(out=AT[2], M=1), dict(out=AT[1] + 4, M=1),
    dict(sx=AT[5] + 4 * LAST), dict(sw=AT[5] + 4 * H), dict(w=AT[5] + 64), dict(bias=AT[5] + 4 * H),
    dict(N=1, ldw=0, out=AT[2]),
])
def test_product(call):
    assert gemm(**call) == SHAPE


@pytest.mark.parametrize("call", [
    dict(out_scale=AT[1]), dict(out_scale=AT[1] + 4 * (2 * M - 1)), dict(out_scale=AT[0] + LAST), dict(out_scale=AT[5]), dict(out_scale=AT[5] + LAST + H - 4),
    dict(out_scale=AT[2] + 2 * H * H - 4), dict(out_scale=AT[3] + 28), dict(out=AT[1]), dict(out=AT[2] + 2 * H * H - 16), dict(out=AT[3] + 16), dict(out=AT[0]),
    dict(out_scale=AT[1], M=1), dict(out_scale=AT[1] + 4 * M - 4, ld_sx=2 * M, ld_os=2 * M),
])
def test_gated_product(call):
    assert gated(**call) == SHAPE
