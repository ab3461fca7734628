"""A dimension of one says nothing by its stride: layers of a single output take a column and a bias of any stride."""
import pytest
import torch

from tests.helpers.fp8_oracle import check_out, make_rows, make_weight, product, values, weight
from zse_b200.ops.backend import TorchOps
from zse_b200.ops.fp8 import Fp8Weight


def single_output(ops, device, M, on_cpu):
    g = torch.Generator().manual_seed(M)
    x, w = make_rows(g, M, 272, device), make_weight(g, 1, 272, device)
    bias = torch.randn(6, generator=g).to(device)[1::4][:1]
    out = torch.empty(3, M, device=device)[1:2].t()                          # strides (1, M)
    assert bias.stride() == (4,) and out.stride(1) == M
    w = Fp8Weight(w.data, w.scale, bias)
    ops.linear_fp8(w, x, M, out)
    y, off = product(values(x, M), weight(w)[0], on_cpu=on_cpu)
    y = y + bias.double()
    check_out(y, off + 2.0 ** -24 * y.abs(), out)


@pytest.mark.parametrize("M", [2, 5])
def test_single_output(M):
    single_output(TorchOps("cpu"), "cpu", M, True)


def test_a_bias_without_dimensions_is_refused():
    w = make_weight(torch.Generator().manual_seed(1), 1, 16, "cpu")
    for bias in (torch.tensor(1.0), torch.ones(1, 1), torch.ones(2)):
        with pytest.raises(ValueError):
            Fp8Weight(w.data, w.scale, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [2, 5, 130, 700])
def test_single_output_on_the_gpu(M):
    from zse_b200.ops.backend import make_ops
    ops = make_ops("cuda")
    single_output(ops, "cuda", M, False)
    ops.check()
