"""Gated 8-bit rows over the whole range of the activation's argument: a block's scale, which is kept in fp32, shows how exact act(g) * u is.

The sigmoid is 1 / (1 + 2^(-z / ln 2)) with 2^x within 2^-22, the reciprocal within 2^-23, the sum within 2^-24; its argument is rounded once and
its constant once, 1.25 |z| 2^-24 of the result where z is negative.  Two products, the scale's division and its product here: 2^-24 each.  So
(11 + 1.25 |z|) 2^-24 in all, and for gelu, whose z comes out of five roundings, (11 + 6.25 |z|) 2^-24.  Where z is positive the exponential's share
of the sum is small and the bound holds by far."""
import pytest
import torch

from zse_b200.ops.fp8 import Fp8Rows

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from zse_b200.ops.backend import make_ops
    return make_ops(DEV)


@pytest.mark.parametrize("gelu", [False, True])
def test_scales_of_gated_rows(ops, gelu):
    g = torch.Generator().manual_seed(5)
    n = 4096
    most = 9.5 if gelu else 85.0                                            # (z of gelu: 76 there)
    gate = (torch.rand(16, n, generator=g) * 2 - 1) * most
    up = torch.exp2(torch.rand(16, n, generator=g) * 20 - 10)
    # one number other than zero in each block, and so large that it is above the least that is kept
    x = torch.zeros(16, 2 * n * 128)
    lift = 2.0 ** 60 if not gelu else 2.0 ** 50
    x[:, : n * 128: 128], x[:, n * 128:: 128] = gate, up * lift
    x = x.to(DEV)
    out = Fp8Rows.empty(16, n * 128, DEV)
    ops.swiglu_fp8(x, 16, out, gelu=gelu)
    v, u = x[:, : n * 128: 128].double(), x[:, n * 128:: 128].double()
    z = 2 * (2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3) if gelu else v
    y = (v * torch.sigmoid(z) * u).abs()
    got = out.scale.t().double() * 448
    off = (got - y).abs() / y
    bound = (11 + (6.25 if gelu else 1.25) * z.abs()) * 2.0 ** -24
    assert (y > 1e-28).all()                                                # (the least: gelu, 9.5 e^-76.3 2^40 = 7e-21; kept from 1e-30 on)
    assert (off <= bound).all(), float((off / bound).max())
    assert (out.data[:, ::128].float().abs() == 448).all()
