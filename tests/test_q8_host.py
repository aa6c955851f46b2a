"""8-bit serving operators without a GPU: the library exports what include/kino_q8.h declares, the
front end refuses what the kernels cannot take, and the oracle's codes stay within half a code
step of the 64-bit definition."""

from __future__ import annotations

import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

from kinomlx_b200 import _lib, ops_q8
from oracle import serving_q8 as ref

ROOT = Path(__file__).resolve().parents[1]
BF16 = torch.bfloat16


def test_library_exports_the_8bit_entry_points():
    text = (ROOT / "include" / "kino_q8.h").read_text()
    names = sorted(set(re.findall(r"^\s*(?:kino_status|int|int64_t)\s+(kino_q8\w+)\(", text, re.M)))
    assert sorted(_lib.SIGNATURES_Q8) == names
    lib = _lib.load()
    for name in names:
        assert hasattr(lib, name), name
    assert lib.kino_q8_abi_version() == 1


def test_refuses_cpu_tensors_and_types():
    x = torch.zeros((4, 64), dtype=BF16)
    codes, scales = torch.zeros((4, 64), dtype=torch.int8), torch.zeros(4)
    with pytest.raises(ValueError, match="CUDA"):
        ops_q8.quantize_tokens(x)
    with pytest.raises(ValueError, match="CUDA"):
        ops_q8.rms_norm_quantize(x)
    with pytest.raises(ValueError, match="CUDA"):
        ops_q8.linear_int8(codes, scales, codes, scales)
    with pytest.raises(ValueError, match="codes are"):
        ops_q8.quantize_tokens(x, torch.uint8)
    with pytest.raises(ValueError, match="blocks of"):
        ops_q8.new_kv_cache(4, 2, 128, block_tokens=48, device="cpu")
    with pytest.raises(ValueError, match="heads of"):
        ops_q8.new_kv_cache(4, 2, 96, device="cpu")
    cache = ops_q8.new_kv_cache(4, 2, 128, device="cpu")
    table, lengths = torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="contiguous CUDA"):
        ops_q8.kv_cache_read(cache, table, lengths, 4)
    with pytest.raises(ValueError, match="scales"):
        ops_q8.kv_cache_read(cache._replace(k_scales=torch.zeros((4, 3))), table, lengths, 4)
    with pytest.raises(ValueError, match="type and shape"):
        ops_q8.kv_cache_read(cache._replace(v_codes=cache.v_codes[:2]), table, lengths, 4)


# ---- the C entry points refuse before they launch: pointers below are never read
ADDRESS = 1 << 20
OK, EINVAL, UNSUPPORTED = 0, 1, 2


def _rows_status(**over):
    a = dict(x=ADDRESS, ldx=64, residual=None, ld_r=0, weight=None, offset=0.0, eps=1e-6, norm=1,
             hidden=None, ld_h=0, codes=ADDRESS, scales=ADDRESS, fmt=0, rows=4, dim=64) | over
    return _lib.load().kino_q8_rows(*a.values(), None)


@pytest.mark.parametrize(("over", "status"), [
    (dict(x=None), EINVAL), (dict(codes=None), EINVAL), (dict(scales=None), EINVAL),
    (dict(fmt=2), EINVAL), (dict(rows=0), EINVAL), (dict(dim=60), UNSUPPORTED),
    (dict(dim=131080, ldx=131080), UNSUPPORTED), (dict(dim=0), UNSUPPORTED),
    (dict(x=ADDRESS + 8), EINVAL), (dict(codes=ADDRESS + 4), EINVAL), (dict(ldx=68), UNSUPPORTED),
    (dict(ldx=56), EINVAL), (dict(residual=ADDRESS, ld_r=56), EINVAL),
    (dict(residual=ADDRESS + 2, ld_r=64), EINVAL), (dict(hidden=ADDRESS, ld_h=8), EINVAL),
    (dict(norm=0, weight=ADDRESS), EINVAL), (dict(weight=ADDRESS + 8), EINVAL),
])
def test_rows_refusals(over, status):
    assert _rows_status(**over) == status
    assert "kino_q8_rows" in _lib.last_error()


def _linear_status(**over):
    a = dict(x=ADDRESS, ldx=64, sx=ADDRESS, w=ADDRESS, ldw=64, sw=ADDRESS, bias=None, out=ADDRESS,
             ldo=64, m=4, n=64, k=64) | over
    return _lib.load().kino_q8_linear(*a.values(), None)


@pytest.mark.parametrize(("over", "status"), [
    (dict(x=None), EINVAL), (dict(sx=None), EINVAL), (dict(out=None), EINVAL), (dict(m=0), EINVAL),
    (dict(k=72, ldx=80, ldw=80), UNSUPPORTED), (dict(n=60), UNSUPPORTED), (dict(ldx=72), UNSUPPORTED),
    (dict(ldw=68), UNSUPPORTED), (dict(ldo=68), UNSUPPORTED), (dict(ldx=48), EINVAL),
    (dict(ldw=48), EINVAL), (dict(ldo=56), EINVAL), (dict(x=ADDRESS + 8), EINVAL),
    (dict(bias=ADDRESS + 8), EINVAL), (dict(sw=ADDRESS + 4), EINVAL),
    (dict(k=131088, ldx=131088, ldw=131088), UNSUPPORTED), (dict(m=1 << 29), UNSUPPORTED),
])
def test_linear_refusals(over, status):
    assert _linear_status(**over) == status
    assert "kino_q8_linear" in _lib.last_error()


def _cache(**over):
    a = dict(k_codes=ADDRESS, v_codes=ADDRESS, k_scales=ADDRESS, v_scales=ADDRESS, num_blocks=8,
             heads=2, dim=128, block=64, format=0, table=ADDRESS, ld_table=4, table_blocks=4,
             lengths=ADDRESS, batch=2) | over
    return _lib.Q8Cache(**a)


CACHE_REFUSALS = [
    (dict(k_codes=None), EINVAL), (dict(v_scales=None), EINVAL), (dict(table=None), EINVAL),
    (dict(lengths=None), EINVAL), (dict(format=7), EINVAL), (dict(dim=96), UNSUPPORTED),
    (dict(block=48), UNSUPPORTED), (dict(block=256), UNSUPPORTED), (dict(num_blocks=0), EINVAL),
    (dict(batch=0), EINVAL), (dict(table_blocks=0), EINVAL), (dict(ld_table=3), EINVAL),
    (dict(num_blocks=1 << 26), UNSUPPORTED), (dict(heads=70000), UNSUPPORTED),
    (dict(table_blocks=1 << 26, ld_table=1 << 26), UNSUPPORTED), (dict(k_codes=ADDRESS + 8), EINVAL),
]


@pytest.mark.parametrize(("over", "status"), CACHE_REFUSALS)
def test_cache_refusals(over, status):
    lib, c = _lib.load(), _cache(**over)
    assert lib.kino_q8_cache_write(c, ADDRESS, 256, 128, ADDRESS, 256, 128, None, 4, None) == status
    assert lib.kino_q8_cache_read(c, ADDRESS, ADDRESS, 4, None) == status
    args = _attention()
    assert lib.kino_q8_attention(c, args, None) == status
    assert lib.kino_q8_attention_workspace_size(c, args) == -1


@pytest.mark.parametrize(("over", "status"), [
    (dict(k=None), EINVAL), (dict(rows=0), EINVAL), (dict(rows=3), EINVAL),
    (dict(ld_k=252), UNSUPPORTED), (dict(hs_v=100), UNSUPPORTED), (dict(v=ADDRESS + 2), UNSUPPORTED),
])
def test_cache_write_refusals(over, status):
    a = dict(k=ADDRESS, ld_k=256, hs_k=128, v=ADDRESS, ld_v=256, hs_v=128, starts=None, rows=4) | over
    assert _lib.load().kino_q8_cache_write(_cache(), *a.values(), None) == status
    assert "kino_q8_cache_write" in _lib.last_error()


def test_cache_read_refusals():
    lib = _lib.load()
    assert lib.kino_q8_cache_read(_cache(), None, ADDRESS, 4, None) == EINVAL
    assert lib.kino_q8_cache_read(_cache(), ADDRESS + 8, ADDRESS, 4, None) == EINVAL
    assert lib.kino_q8_cache_read(_cache(), ADDRESS, ADDRESS, 0, None) == EINVAL


def _attention(**over):
    a = dict(q=ADDRESS, ld_q=1024, hs_q=128, out=ADDRESS, ld_out=1024, hs_out=128, rows=4,
             q_heads=8, scale=0.1, causal=1, workspace=ADDRESS, workspace_bytes=1 << 40) | over
    return _lib.Q8AttentionArgs(**a)


@pytest.mark.parametrize(("over", "status"), [
    (dict(q=None), EINVAL), (dict(out=None), EINVAL), (dict(rows=0), EINVAL), (dict(rows=3), EINVAL),
    (dict(q_heads=7), EINVAL), (dict(q_heads=0), EINVAL), (dict(q_heads=2 * 129), UNSUPPORTED),
    (dict(ld_q=1020), UNSUPPORTED), (dict(hs_out=4), UNSUPPORTED), (dict(q=ADDRESS + 8), UNSUPPORTED),
    (dict(scale=-1.0), EINVAL), (dict(scale=math.nan), EINVAL), (dict(scale=math.inf), EINVAL),
    (dict(workspace=None), EINVAL), (dict(workspace=ADDRESS + 8), EINVAL),
    (dict(workspace_bytes=1000), EINVAL),
])
def test_attention_refusals(over, status):
    assert _lib.load().kino_q8_attention(_cache(), _attention(**over), None) == status
    assert "kino_q8_attention" in _lib.last_error()
    assert ctypes.sizeof(_lib.Q8AttentionArgs) == 96 and ctypes.sizeof(_lib.Q8Cache) == 112


# ---- the oracle
@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_oracle_codes_are_nearest(dtype):
    g = torch.Generator().manual_seed(1)
    x = (torch.randn((50, 96), generator=g) * torch.logspace(-5, 5, 50)[:, None]).to(BF16)
    codes, scale = ref.quantize_rows(x, dtype)
    want = x.double() / (x.double().abs().amax(-1, keepdim=True) / ref.TOP[dtype])
    off = (codes.double() - want).abs()
    # one fp32 rounding in front of the code's own
    half = 0.5 if dtype == torch.int8 else torch.clamp(want.abs() * 2.0**-4, min=2.0**-10)
    assert bool((off <= half + 2 * 2.0**-24 * want.abs()).all())
    assert bool((codes.double().abs().amax(-1) == ref.TOP[dtype]).all())


def test_oracle_write_follows_its_parts():
    g = torch.Generator().manual_seed(2)
    x = torch.randn((40, 2, 64), generator=g).to(BF16)
    codes, scales = torch.zeros((3, 2, 32, 64), dtype=torch.int8), torch.zeros((3, 2))
    table, zero = torch.tensor([[2, 0]], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    once = ref.cache_write(codes, scales, x, table, zero)
    got = ref.cached(*once, table[0], 40).transpose(0, 1)
    step = x.double().abs().amax() / 127
    assert float((got - x.double()).abs().max()) <= float(step) * 0.51
    # token by token: each growth of the scale rounds again, at most half a step each time
    c, s = codes, scales
    for t in range(40):
        c, s = ref.cache_write(c, s, x[t : t + 1], table, torch.tensor([t], dtype=torch.int32))
    assert torch.equal(s, once[1])
    got = ref.cached(c, s, table[0], 40).transpose(0, 1)
    assert float((got - x.double()).abs().max()) <= float(step) * 4
