"""8-bit serving operators at the edges of their ranges: calls without a sum's buffer, rows whose
squares leave fp32, the widest product, queries that are huge, tiny or infinite, strides of every
order, and a cache whose offsets pass 32 bits."""

from __future__ import annotations

import math

import pytest
import torch

from kinomlx_b200 import _lib, ops, ops_q8
from oracle import serving_q8 as ref

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
INT8, E4M3 = torch.int8, torch.float8_e4m3fn
DTYPES = [INT8, E4M3]


def _normal(shape, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(BF16)


def _same(a, b):
    a, b = a.cpu().float(), b.cpu().float()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


# ---------------------------------------------------------------- rows
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 16384, 16392, 40000])
@pytest.mark.parametrize("norm", [0, 1])
def test_residual_without_a_buffer_for_the_sum(cuda_device, dtype, dim, norm):
    """The C entry point's `hidden` may be NULL: codes and scales are those of the sum all the same."""
    x, r = _normal((3, dim), dim), _normal((3, dim), dim + 1, 5.0)
    xd, rd = x.to(cuda_device), r.to(cuda_device)
    codes = torch.empty((3, dim), dtype=dtype, device=cuda_device)
    scales = torch.empty(3, device=cuda_device)
    status = _lib.load().kino_q8_rows(
        xd.data_ptr(), dim, rd.data_ptr(), dim, None, 0.0, 1e-6, norm, None, 0, codes.data_ptr(),
        scales.data_ptr(), ops_q8.FORMATS[dtype], 3, dim, torch.cuda.current_stream().cuda_stream)
    assert status == 0, _lib.last_error()
    if norm:
        want = ops_q8.rms_norm_quantize(xd, residual=rd, dtype=dtype)
    else:
        want = ref.quantize_rows((x.float() + r.float()).to(BF16), dtype)
    assert torch.equal(scales.cpu(), want[1].cpu()) and _same(codes, want[0])
    assert torch.equal(xd.cpu(), x) and torch.equal(rd.cpu(), r)


def test_rows_without_values_are_refused(cuda_device):
    for shape in ((4, 0), (2, 3, 0)):
        x = torch.empty(shape, dtype=BF16, device=cuda_device)
        codes = torch.empty(shape, dtype=INT8, device=cuda_device)
        weight = torch.empty((8, 0), dtype=INT8, device=cuda_device)
        with pytest.raises(ValueError, match="width"):
            ops_q8.quantize_tokens(x)
        with pytest.raises(ValueError, match="width"):
            ops_q8.rms_norm_quantize(x, residual=x)
        with pytest.raises(ValueError, match="width"):
            ops_q8.linear_int8(codes, torch.ones(shape[:-1], device=cuda_device), weight,
                               torch.ones(8, device=cuda_device))
    # no rows are nothing to do
    codes, scales = ops_q8.quantize_tokens(torch.empty((2, 0, 64), dtype=BF16, device=cuda_device))
    assert codes.shape == (2, 0, 64) and scales.shape == (2, 0)
    y = ops_q8.linear_int8(codes, scales, *ops_q8.quantize_tokens(
        torch.ones((8, 64), dtype=BF16, device=cuda_device)))
    assert y.shape == (2, 0, 8)


# ---------------------------------------------------------------- product
@pytest.mark.parametrize(("m", "n"), [(3, 16), (300, 6400)])  # both forms
def test_the_widest_product_of_the_lowest_codes(cuda_device, m, n):
    k = 131056  # the widest that the int32 sum holds: 131056 * 2^14 = 2^31 - 2^18
    x = torch.full((m, k), -128, dtype=INT8, device=cuda_device)
    w = torch.full((n, k), -128, dtype=INT8, device=cuda_device)
    w[1] = 127
    ones = torch.ones(max(m, n), device=cuda_device)
    out = ops_q8.linear_int8(x, ones[:m], w, ones[:n])
    ops.device_status()
    want = torch.full((n,), float(128 * 128 * k)).to(BF16)
    want[1] = torch.tensor(-128.0 * 127 * k).to(BF16)
    assert torch.equal(out.cpu(), want.expand(m, n))
