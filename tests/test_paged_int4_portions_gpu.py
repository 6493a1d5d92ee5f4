"""Attention over 4-bit pages by the kernels of many rows: pages unpacked to halves for the tensor memory, and row tiles beside them."""
import pytest
import torch

from paged_cases import make as make16
from paged_int4_cases import attention, bound, make
from paged_oracle import attention as oracle16

from neuronx_distributed_b200 import ops
from neuronx_distributed_b200.ops import _ext

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def wide(d, tokens):
    """A table of so many tokens, behind the last page of which there is none: from some width on portions of prompts are unpacked."""
    B, n = d["table"].shape
    cols = -(-tokens // d["k_pages"].codes.shape[1])
    return {**d, "table": torch.cat([d["table"], torch.full((B, max(0, cols - n)), -1, dtype=torch.int32, device="cuda")], 1)}


def attend(d, unpacked=None, **kw):
    """``unpacked``: whether the pages are, by the launches: queries, pages, attention, and often the joining of its parts, for one or two."""
    n = _ext.launches()
    out = ops.paged_int4.attention(d["q"], d["k_pages"], d["v_pages"], d["table"], d["positions"], lens=d["lens"], shared_pages=d["shared_pages"], **kw)
    assert unpacked is None or unpacked == (_ext.launches() - n > 2)
    return out


def check(d, got, scale=None, more=0.0):
    want, size = attention(d, scale)
    off = (got.double() - want).abs() - bound(d["q"].dtype, want, size) - more * size
    assert bool((off <= 0).all()), (float(off.max()), (~(off <= 0)).nonzero()[:4].tolist())


@pytest.mark.parametrize("scale", [None, 1 / 128, 1e-8, 1e-25, 1e-39])
@pytest.mark.parametrize("B, W, H, Hkv, tokens, unpacked", [(2, 80, 8, 2, 8192, True), (2, 6, 8, 2, 0, False), (2, 1, 8, 2, 0, False)])
def test_rows_of_zeros(scale, B, W, H, Hkv, tokens, unpacked):
    """Rows of zeros, as append leaves them for tokens without a slot, and rows of the smallest numbers see the average of the values; so does everybody where the scale is next to
    nothing."""
    d = wide(make(21, "cuda", BF16, B, W, H, Hkv, 128, 16, [100, 37]), tokens)
    d["q"] = d["q"].clone()
    d["q"][0, 0, 1:3] = 0.0
    d["q"][1] = 0.0
    d["q"][0, -1, :2] *= 1e-37
    check(d, attend(d, unpacked, scale=scale), scale)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("W", [1, 60])
def test_scales_below_the_normal_numbers_over_16_bit_pages(dtype, W):
    d = make16(22, "cuda", dtype, 2, W, 8, 2, 128, 16, [100, 37])
    got = ops.paged.attention(d["q"], d["k_cache"], d["v_cache"], d["table"], d["positions"], scale=1e-39)
    want, size = oracle16(d["q"], d["k_cache"], d["v_cache"], d["table"], d["positions"], 1e-39)
    assert bool(((got.double() - want).abs() <= torch.finfo(dtype).eps / 2 * (want.abs() + size) + 2.0 ** -13 * size + 1e-7).all())
