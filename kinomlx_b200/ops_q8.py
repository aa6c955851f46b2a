"""8-bit serving operators: torch front end of include/kino_q8.h.

Values are held as 8-bit codes (int8 or float8_e4m3fn) times an fp32 scale for each group: a
token's row, a weight's output channel, or the tokens of one cache block and head. A group's scale
is its largest magnitude over 127 (int8) or 448 (e4m3); a group of zeros (or of magnitudes below
about 1e-36) has scale 0; one that holds an infinity or a NaN has the scale NaN and reads back as
NaN.

    codes, scales, hidden = rms_norm_quantize(x, weight, residual=hidden)
    y = linear_int8(codes, scales, w_codes, w_scales)      # w from quantize_tokens(weight)
    kv_cache_write(cache, k, v, table, lengths)
    out = kv_cache_attention(q, cache, table, lengths + 1)

Like `ops`, these have no CPU path: a tensor of the wrong device, type or shape is a ValueError, a
refusal by the library a RuntimeError. Lengths, token starts and block tables are read on the
device; entries that do not fit are skipped there and `ops.device_status` raises.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _lib, ops

BF16 = torch.bfloat16
I32 = torch.int32
F32 = torch.float32
FORMATS = {torch.int8: _lib.Q8_INT8, torch.float8_e4m3fn: _lib.Q8_E4M3}

__all__ = [
    "KVCache",
    "kv_cache_attention",
    "kv_cache_read",
    "kv_cache_write",
    "linear_int8",
    "new_kv_cache",
    "quantize_tokens",
    "rms_norm_quantize",
]


# Decoded tokens take a few microseconds on the GPU, so the host side of a call counts: one look at
# each tensor, entry points bound once, no wrapper objects.
_entries: dict[str, object] = {}


def _launch(label: str, flops: float, nbytes: float, device: torch.device, name: str, *args) -> None:
    """One kino_q8_* call on the device's current stream."""
    entry = _entries.get(name)
    if entry is None:
        entry = _entries[name] = getattr(_lib.load(), name)
    index = device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return _launch(label, flops, nbytes, device, name, *args)
    stream = torch._C._cuda_getCurrentRawStream(index)
    if ops._log is None:
        ops.launches += 1
        status = entry(*args, stream)
    else:
        with ops._timed(label, flops, nbytes):
            status = entry(*args, stream)
    if status:
        label = _lib.STATUS_NAMES.get(status, str(status))
        raise RuntimeError(f"{name} failed with {label}: {_lib.last_error()}")


def _format(dtype: torch.dtype) -> int:
    try:
        return FORMATS[dtype]
    except KeyError:
        raise ValueError(f"codes are int8 or float8_e4m3fn, not {dtype}") from None


def _need(t: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device | None = None) -> None:
    """A CUDA tensor of this type (on this device) with a unit stride in its last dimension."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (the kinomlx_b200 kernels have no CPU path)")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if not t.is_contiguous() and t.stride(-1) != 1 and t.shape[-1] != 1:
        raise ValueError(f"{name} needs a unit stride in its last dimension")


def _empty_as(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Contiguous, of t's shape (empty_like is the quickest of torch's ways to one)."""
    if t.is_contiguous():
        return torch.empty_like(t, dtype=dtype)
    return torch.empty(t.shape, dtype=dtype, device=t.device)


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    """(..., dim) as (rows, dim) without a copy."""
    if t.dim() == 2:
        return t
    if t.dim() == 0:
        raise ValueError(f"{name} needs rows")
    try:
        return (t.view(-1, t.shape[-1]) if t.numel()
                else t.reshape(math.prod(t.shape[:-1]), t.shape[-1]))
    except RuntimeError:
        raise ValueError(f"{name}: rows of {tuple(t.shape)} are not at one stride") from None


def _quantize_rows(x, weight, eps, residual, dtype, weight_offset, norm, hidden, label):
    fmt = _format(dtype)
    _need(x, "x", BF16)
    x2 = _rows(x, "x")
    rows, dim = x2.shape
    if rows and not dim:
        raise ValueError(f"x {tuple(x.shape)} has rows of width 0")
    device = x.device
    r_ptr = h_ptr = w_ptr = None
    ld_r = ld_h = 0
    if residual is not None:
        _need(residual, "residual", BF16, device)
        if residual.shape != x.shape:
            raise ValueError(f"residual {tuple(residual.shape)} does not match {tuple(x.shape)}")
        if hidden is None:
            hidden = _empty_as(x, BF16)
        else:
            _need(hidden, "hidden", BF16, device)
            if hidden.shape != x.shape:
                raise ValueError(f"hidden {tuple(hidden.shape)} does not match {tuple(x.shape)}")
        r2, h2 = _rows(residual, "residual"), _rows(hidden, "hidden")
        r_ptr, h_ptr = r2.data_ptr(), h2.data_ptr()
        ld_r, ld_h = (r2.stride(0), h2.stride(0)) if rows > 1 else (dim, dim)
    elif hidden is not None:
        raise ValueError("hidden is the sum with a residual: give one")
    if weight is not None:
        _need(weight, "weight", BF16, device)
        if weight.shape != (dim,):
            raise ValueError(f"weight {tuple(weight.shape)} does not match width {dim}")
        w_ptr = weight.data_ptr()
    codes = _empty_as(x, dtype)
    scales = torch.empty(rows if x.dim() == 2 else x.shape[:-1], dtype=F32, device=device)
    if rows:
        _launch(label, 0.0, (3.0 if residual is None else 7.0) * rows * dim, device,
                "kino_q8_rows", x2.data_ptr(), x2.stride(0) if rows > 1 else dim, r_ptr, ld_r, w_ptr, weight_offset, eps,
                norm, h_ptr, ld_h, codes.data_ptr(), scales.data_ptr(), fmt, rows, dim)
    return codes, scales, x if hidden is None else hidden


def quantize_tokens(x: torch.Tensor, dtype: torch.dtype = torch.int8):
    """Codes like x and a scale for each row of x (..., dim) bf16: activations by token, or a
    weight (out, in) by output channel. dim a multiple of 8, at most 131072."""
    codes, scales, _ = _quantize_rows(x, None, 0.0, None, dtype, 0.0, 0, None, "quantize_tokens")
    return codes, scales


def rms_norm_quantize(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    *,
    residual: torch.Tensor | None = None,
    dtype: torch.dtype = torch.int8,
    weight_offset: float = 0.0,
    hidden: torch.Tensor | None = None,
):
    """(codes, scales, hidden): hidden = bf16(x + residual) (x itself without a residual), and the
    codes and row scales of its RMS norm times (weight + weight_offset), which stays in fp32 until
    it is rounded to a code. `hidden` may be given, also as x or residual (in place)."""
    return _quantize_rows(x, weight, eps, residual, dtype, weight_offset, 1, hidden,
                          "rms_norm_quantize")


def linear_int8(
    codes: torch.Tensor,
    scales: torch.Tensor,
    w_codes: torch.Tensor,
    w_scales: torch.Tensor,
    bias: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """bf16(codes @ w_codes.T * scales[:, None] * w_scales + bias) for int8 codes (..., k) with a
    scale for each row and an int8 weight (n, k) with one for each channel; the sum over k is
    exact. k a multiple of 16 below 131072, n of 8."""
    _need(codes, "codes", torch.int8)
    device = codes.device
    _need(w_codes, "w_codes", torch.int8, device)
    _need(scales, "scales", F32, device)
    _need(w_scales, "w_scales", F32, device)
    x2 = _rows(codes, "codes")
    m, k = x2.shape
    if m and not k:
        raise ValueError(f"codes {tuple(codes.shape)} have rows of width 0")
    if w_codes.dim() != 2 or w_codes.shape[1] != k:
        raise ValueError(f"weight {tuple(w_codes.shape)} does not match input width {k}")
    n = w_codes.shape[0]
    if scales.shape != codes.shape[:-1] or not scales.is_contiguous():
        raise ValueError(f"scales {tuple(scales.shape)} are not one for each row, contiguous")
    if w_scales.shape != (n,):
        raise ValueError(f"w_scales {tuple(w_scales.shape)} are not one for each of {n} channels")
    b_ptr = None
    if bias is not None:
        _need(bias, "bias", BF16, device)
        if bias.shape != (n,):
            raise ValueError(f"bias {tuple(bias.shape)} is not one for each of {n} channels")
        b_ptr = bias.data_ptr()
    shape = (*codes.shape[:-1], n)
    if out is None:
        out = torch.empty(shape, dtype=BF16, device=device)
    else:
        _need(out, "out", BF16, device)
        if out.shape != shape:
            raise ValueError(f"out {tuple(out.shape)} does not match {shape}")
    o2 = _rows(out, "out")
    if m and n:
        _launch("linear_int8", 2.0 * m * n * k, 1.0 * m * k + n * k + 2 * m * n, device,
                "kino_q8_linear", x2.data_ptr(), x2.stride(0) if m > 1 else k, scales.data_ptr(),
                w_codes.data_ptr(), w_codes.stride(0) if n > 1 else k, w_scales.data_ptr(), b_ptr,
                out.data_ptr(), o2.stride(0) if m > 1 else n, m, n, k)
    return out


class KVCache(NamedTuple):
    """Keys and values in 8 bits: codes (blocks, heads, block tokens, dim), int8 or float8_e4m3fn,
    with a scale for each block and head, (blocks, heads) fp32. All contiguous; dim 64 or 128,
    block tokens 16, 32, 64 or 128. Token t of sequence b is slot t % block of the block
    table[b, t // block]."""

    k_codes: torch.Tensor
    v_codes: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor


def new_kv_cache(blocks: int, heads: int, dim: int, *, block_tokens: int = 64,
                 dtype: torch.dtype = torch.int8, device: torch.device | str = "cuda") -> KVCache:
    """An empty cache (zeros)."""
    _format(dtype)
    if dim not in (64, 128) or block_tokens not in (16, 32, 64, 128):
        raise ValueError(f"heads of 64 or 128 and blocks of 16, 32, 64 or 128 tokens, not {dim} "
                         f"and {block_tokens}")
    if blocks < 1 or heads < 1:
        raise ValueError(f"a cache of {blocks} blocks and {heads} heads")
    codes = [torch.zeros((blocks, heads, block_tokens, dim), device=device, dtype=torch.int8)
             .view(dtype) for _ in range(2)]
    scales = [torch.zeros((blocks, heads), device=device, dtype=F32) for _ in range(2)]
    return KVCache(*codes, *scales)


def _cache_args(cache: KVCache, table: torch.Tensor, lengths: torch.Tensor) -> _lib.Q8Cache:
    k, v, ks, vs = cache
    fmt = _format(k.dtype)
    if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"codes of keys {tuple(k.shape)} and values {tuple(v.shape)} are not one "
                         "(blocks, heads, tokens, dim) type and shape")
    blocks, heads, block, dim = k.shape
    if ks.shape != (blocks, heads) or vs.shape != (blocks, heads):
        raise ValueError(f"scales {tuple(ks.shape)}, {tuple(vs.shape)} are not (blocks, heads)")
    if not (k.is_cuda and k.is_contiguous() and v.is_contiguous() and ks.is_contiguous()
            and vs.is_contiguous() and ks.dtype == F32 and vs.dtype == F32):
        raise ValueError("a cache is contiguous CUDA tensors with fp32 scales")
    if table.dtype != I32 or lengths.dtype != I32:
        raise ValueError("block table and lengths are int32")
    if table.dim() != 2 or lengths.shape != table.shape[:1]:
        raise ValueError(f"table {tuple(table.shape)} and lengths {tuple(lengths.shape)} are not "
                         "(batch, blocks) and (batch,)")
    batch, wide = table.shape
    if (wide > 1 and table.stride(1) != 1) or not lengths.is_contiguous():
        raise ValueError("block table rows and lengths need unit strides")
    device = k.device
    if not (v.device == ks.device == vs.device == table.device == lengths.device == device):
        raise ValueError(f"cache, table and lengths are not all on {device}")
    return _lib.Q8Cache(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), blocks, heads,
                        dim, block, fmt, table.data_ptr(),
                        table.stride(0) if batch > 1 else max(wide, 1), wide, lengths.data_ptr(),
                        batch)


def _starts(token_starts: torch.Tensor | None, batch: int, rows: int,
            device: torch.device) -> int | None:
    if token_starts is None:
        if rows % batch:
            raise ValueError(f"{rows} rows do not divide over {batch} sequences")
        return None
    if token_starts.dtype != I32 or token_starts.shape != (batch + 1,) \
            or not token_starts.is_contiguous():
        raise ValueError(f"token_starts are batch + 1 = {batch + 1} int32, contiguous")
    if token_starts.device != device:
        raise ValueError(f"token_starts is on {token_starts.device}, not on {device}")
    return token_starts.data_ptr()


def _heads(t: torch.Tensor, name: str, dim: int, device: torch.device) -> None:
    _need(t, name, BF16, device)
    if t.dim() != 3 or t.shape[2] != dim:
        raise ValueError(f"{name} {tuple(t.shape)} is not (rows, heads, {dim})")


def _strides(t: torch.Tensor) -> tuple[int, int]:
    """Row and head strides of (rows, heads, dim); a dimension of one has any, so 0."""
    rows, heads, _ = t.shape
    return t.stride(0) if rows > 1 else 0, t.stride(1) if heads > 1 else 0


def kv_cache_write(
    cache: KVCache,
    k: torch.Tensor,
    v: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    token_starts: torch.Tensor | None = None,
) -> None:
    """Quantise new tokens into the cache, in place. k, v (rows, heads, dim) bf16 (any row and
    head strides that are multiples of 8); block_table (batch, blocks) int32; lengths (batch,)
    int32, the tokens each sequence holds before. Sequence b's rows are token_starts[b] to
    token_starts[b + 1], or rows / batch each; they take positions lengths[b] on. Where a block
    already holds tokens, its scale only grows, and its codes are rounded again when it does.

    A cache block may belong to one sequence of a call only (sequences that share blocks write
    behind them)."""
    args = _cache_args(cache, block_table, lengths)
    device = cache[0].device
    _heads(k, "k", args.dim, device)
    _heads(v, "v", args.dim, device)
    rows = k.shape[0]
    if k.shape != v.shape or k.shape[1] != args.heads:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} are not (rows, {args.heads}, "
                         f"{args.dim})")
    if not rows or not args.batch:
        return
    starts = _starts(token_starts, args.batch, rows, device)
    _launch("kv_cache_write", 0.0, 6.0 * k.numel(), device, "kino_q8_cache_write", args,
            k.data_ptr(), *_strides(k), v.data_ptr(), *_strides(v), starts, rows)


def kv_cache_read(
    cache: KVCache,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    tokens: int,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of tokens [0, tokens) of every sequence as (batch, tokens, heads, dim)
    bf16, zeros from a sequence's length on."""
    args = _cache_args(cache, block_table, lengths)
    device = cache[0].device
    if tokens < 0:
        raise ValueError(f"{tokens} tokens")
    shape = (args.batch, tokens, args.heads, args.dim)
    k, v = (torch.empty(shape, device=device, dtype=BF16) for _ in range(2))
    if k.numel():
        _launch("kv_cache_read", 0.0, 6.0 * k.numel(), device, "kino_q8_cache_read", args,
                k.data_ptr(), v.data_ptr(), tokens)
    return k, v


def kv_cache_attention(
    q: torch.Tensor,
    cache: KVCache,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    token_starts: torch.Tensor | None = None,
    *,
    causal: bool = True,
    scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """softmax(q k^T * scale) v over the cached tokens of each sequence. q (rows, query heads,
    dim) bf16, query heads a multiple of the cache's heads (head h reads cache head h // group);
    lengths (batch,) int32, the tokens in the cache, among them the sequence's queries, which are
    its last tokens: with `causal` query i of n sees keys up to position lengths - n + i. Rows go
    to sequences as in `kv_cache_write`. A query that sees no key gives zeros, an infinite one that
    sees some NaN. Decoded tokens and prompts are faster as calls of their own. Rows of `out`
    outside every sequence are left as they were (uninitialised where `out` is not given)."""
    args = _cache_args(cache, block_table, lengths)
    device = cache[0].device
    _heads(q, "q", args.dim, device)
    rows, heads = q.shape[:2]
    if heads % args.heads:
        raise ValueError(f"{heads} query heads on {args.heads} cache heads")
    if out is None:
        out = _empty_as(q, BF16)
    else:
        _heads(out, "out", args.dim, device)
        if out.shape != q.shape:
            raise ValueError(f"out {tuple(out.shape)} does not match q {tuple(q.shape)}")
    if not rows or not heads or not args.batch:
        return out
    call = _lib.Q8AttentionArgs(
        q.data_ptr(), *_strides(q), out.data_ptr(), *_strides(out),
        _starts(token_starts, args.batch, rows, device), rows, heads,
        args.dim**-0.5 if scale is None else scale, causal)
    size = _entries.get("size") or _entries.setdefault(
        "size", _lib.load().kino_q8_attention_workspace_size)
    if device.index == torch.cuda.current_device():
        nbytes = size(args, call)
    else:  # it goes by the device's SMs
        with torch.cuda.device(device):
            nbytes = size(args, call)
    if nbytes < 0:
        raise RuntimeError(f"kino_q8_attention: {_lib.last_error()}")
    space = torch.empty(nbytes, device=device, dtype=torch.uint8)
    call.workspace, call.workspace_bytes = space.data_ptr(), nbytes
    # (its work goes by lengths that only the device knows: none is logged)
    _launch("kv_cache_attention", 0.0, 0.0, device, "kino_q8_attention", args, call)
    return out
