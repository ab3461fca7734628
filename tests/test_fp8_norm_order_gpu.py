"""The norm that leaves 8 bits: a row's bytes do not depend on how many rows a call has, not by one rounding either.

The squares are summed in 64 bits and 1 / root is rounded once, to fp32.  Sums taken in two orders differ by a few units of 64 bits, which
changes that rounding only where the root lies next to the middle of two fp32 numbers.  eps is chosen to put it there: of 64 neighbouring
values of mean + eps across such a middle one lies between the two sums wherever they differ."""
import math

import pytest
import torch

from zse_b200.ops.fp8 import Fp8Rows

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from zse_b200.ops.backend import make_ops
    return make_ops(DEV)


def middles(mean):
    """64 values of eps so that mean + eps walks in steps of one unit across a number whose 1 / root is the middle of two in fp32."""
    inv = torch.tensor(1 / math.sqrt(mean * (1 + 1e-6)), dtype=torch.float32)
    below = torch.nextafter(inv, torch.tensor(0.0))
    at = 1 / (((inv.double() + below.double()) / 2).item()) ** 2
    step = math.ulp(mean)
    return [at - mean + k * step for k in range(-32, 32)]


@pytest.mark.parametrize("H", [144, 400, 1040, 2576, 5120, 8192, 20000, 32768])
@pytest.mark.parametrize("planes", [0, 2])
def test_bytes_alone_and_among_others(ops, H, planes):
    g, many = torch.Generator().manual_seed(H), 700
    w = (1 + torch.randn(H, generator=g) * 0.2).half().to(DEV)
    parts = torch.zeros(planes, many, H, device=DEV) if planes else None
    one, all_rows = Fp8Rows.empty(1, H, DEV), Fp8Rows.empty(many, H, DEV)
    for _ in range(4):
        row = (torch.randn(1, H, generator=g) * 3).to(DEV)
        rows = row.expand(many, H).contiguous()
        for eps in middles(row.double().square().mean().item()):
            assert eps > 0
            ops.add_rmsnorm_fp8(row, parts[:, :1].contiguous() if planes else None, planes, None, w, one, 1, eps)
            ops.add_rmsnorm_fp8(rows, parts, planes, None, w, all_rows, many, eps)
            assert torch.equal(one.scale.expand(-1, many), all_rows.scale)
            assert torch.equal(one.data.view(torch.uint8).expand(many, H), all_rows.data.view(torch.uint8))
