"""Refusals of the 8-bit serving operators at the edges of their shapes, without a GPU."""

from __future__ import annotations

import pytest
import torch

from kinomlx_b200 import _lib, ops_q8
from oracle import serving_q8 as ref

BF16 = torch.bfloat16


@pytest.mark.parametrize("shape", [(4, 0), (2, 3, 0), (0,)])
def test_rows_without_values_are_refused(monkeypatch, shape):
    """Outputs would be left unwritten: rows there are, but no value that the kernels could read."""
    monkeypatch.setattr(ops_q8, "_need", lambda *_: None)  # these tensors are on the CPU
    x, codes = torch.empty(shape, dtype=BF16), torch.empty(shape, dtype=torch.int8)
    for call in (lambda: ops_q8.quantize_tokens(x),
                 lambda: ops_q8.rms_norm_quantize(x, residual=x),
                 lambda: ops_q8.linear_int8(codes, torch.ones(shape[:-1]),
                                            torch.empty((8, 0), dtype=torch.int8), torch.ones(8))):
        with pytest.raises(ValueError, match="width 0"):
            call()


def test_no_rows_are_nothing_to_do(monkeypatch):
    monkeypatch.setattr(ops_q8, "_need", lambda *_: None)
    monkeypatch.setattr(ops_q8, "_launch", None)  # not called
    for shape in ((0, 64), (2, 0, 64), (0, 0)):
        codes, scales = ops_q8.quantize_tokens(torch.empty(shape, dtype=BF16))
        assert codes.shape == shape and scales.shape == shape[:-1]
        y = ops_q8.linear_int8(codes, scales, torch.empty((8, shape[-1]), dtype=torch.int8), torch.ones(8))
        assert y.shape == (*shape[:-1], 8)


@pytest.mark.parametrize("k", [131072, 262144])
def test_products_that_int32_cannot_hold_are_refused(k):
    """131072 products of the code -128 with itself are 2^31."""
    at = 1 << 20  # never read
    lib = _lib.load()
    assert lib.kino_q8_linear(at, k, at, at, k, at, None, at, 64, 4, 64, k, None) == 2
    assert "k <" in _lib.last_error()


@pytest.mark.parametrize("causal", [True, False])
def test_oracle_attention_by_products(causal):
    g = torch.Generator().manual_seed(3)
    codes = [torch.randint(-127, 128, (12, 2, 16, 64), generator=g, dtype=torch.int8) for _ in range(2)]
    scales = [torch.rand((12, 2), generator=g) * 0.02 for _ in range(2)]
    table = torch.randperm(12, generator=g).view(2, 6).to(torch.int32)
    q = torch.randn((150, 6, 64), generator=g).to(BF16)
    lengths, starts = torch.tensor([90, 20]), torch.tensor([0, 120, 148])  # queries in front of the keys
    args = (q, *codes, *scales, table, lengths, starts)
    for a, b in zip(ref.attention(*args, causal=causal), ref.attention_by_products(*args, causal=causal)):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)
