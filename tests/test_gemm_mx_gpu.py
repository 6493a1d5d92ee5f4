"""The block-scaled tensor-core products (``csrc/gemm_mx_sm100.cu``, ``csrc/gemm_mxf4_sm100.cu``) against the product of the numbers that codes and scales stand for."""
import pytest
import torch

from neuronx_distributed_b200.ops import _ext, gemm_mx
from neuronx_distributed_b200.quantization.microscaling.mx_torch import quantize_mxfp8

pytestmark = pytest.mark.gpu


def close(got, want):
    """A half step of bf16, and sums of products in 32 bits: off by 2^-13 of the largest number of a row at most, hundreds of roundings of 2^-24."""
    want = want.double()
    assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -13 * want.abs().amax(1, keepdim=True)).all())


def eights(M, N, K):
    g = torch.Generator(device="cuda").manual_seed(M + K)
    a, b = (torch.randn(r, K, generator=g, device="cuda") for r in (M, N))
    return (*quantize_mxfp8(a), *quantize_mxfp8(b))


def fours(M, N, K):
    g = torch.Generator(device="cuda").manual_seed(M + K)
    a, b = (torch.randn(r, K, generator=g, device="cuda") for r in (M, N))
    return (*gemm_mx.quantize_mxfp4(a), *gemm_mx.quantize_mxfp4(b))


@pytest.mark.parametrize("M, N, K", [(128, 128, 256), (300, 520, 1024), (4000, 2000, 256)])
def test_waits_that_run_out(M, N, K):
    """Nothing is loaded: the waits give up after a fiftieth of a second, numbers are NaN, and the next call is as ever."""
    a, sa, b, sb = eights(M, N, K)
    call = [t.view(torch.uint8) for t in (a, b)] + [gemm_mx.tile_scales(t) for t in (sa, sb)] + [0, 0]
    assert bool(_ext.ext().gemm_mxfp8(*call, wait_ns=-20000000).isnan().all())
    close(_ext.ext().gemm_mxfp8(*call), gemm_mx.matmul_mxfp8_reference(a, sa, b, sb))
    a, sa, b, sb = fours(M, N, K)
    call = [a, b] + [gemm_mx.tile_scales(t) for t in (sa, sb)] + [32, 1.0]
    assert bool(_ext.ext().gemm_f4(*call, wait_ns=-20000000).isnan().all())
    close(_ext.ext().gemm_f4(*call), gemm_mx.matmul_f4_reference(a, sa, b, sb))


@pytest.mark.parametrize("a_kind, b_kind", [("mxfp8", "mxfp4"), ("mxfp4", "mxfp8"), ("mxfp4", "mxfp4")])
@pytest.mark.parametrize("M, N, K", [(1, 8, 128), (128, 128, 128), (300, 520, 1024), (1000, 2000, 2048)])
def test_operands_of_four_bits(a_kind, b_kind, M, N, K):
    """Numbers of 4 bits, which copies spread over containers of 8: beside 8-bit ones, on either side, and on both."""
    a, b = (f(M, N, K)[i:i + 2] for f, i in ((eights if a_kind == "mxfp8" else fours, 0), (eights if b_kind == "mxfp8" else fours, 2)))
    close(gemm_mx.matmul_mxfp8(*a, *b, a_kind, b_kind), gemm_mx.matmul_mxfp8_reference(*a, *b, a_kind, b_kind))
