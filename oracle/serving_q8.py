"""The 8-bit serving operators from their definitions in 64 bits, on the CPU.

Codes are whole numbers (int8) or the values of e4m3 codes, as float64. Quantisation of bf16 values
is given with the roundings of an implementation in fp32 (`scale_f32`, `codes`): the scale is one
correctly rounded quotient, a code the exact quotient x * top / amax rounded to fp32 and then to the
code grid, so that another implementation of the same steps has to give the same codes bit for bit.
"""

from __future__ import annotations

import math

import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
F64 = torch.float64


def scale_f32(amax: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """fp32 scale of groups with these largest magnitudes (NaN where not finite)."""
    s = amax.float() / torch.tensor(TOP[dtype], dtype=torch.float32)
    s = torch.where(s < 2.0**-126, torch.zeros_like(s), s)
    return torch.where(torch.isfinite(amax), s, torch.full_like(s, math.nan))


def codes(quotient: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Codes of float64 quotients; what is not finite gives 0."""
    x = torch.where(torch.isfinite(quotient), quotient, torch.zeros_like(quotient)).float()
    if dtype == torch.int8:
        return x.round().clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def amax(x: torch.Tensor, dims) -> torch.Tensor:
    """Largest magnitudes over dims as float64, NaN where something is not finite."""
    top = torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0).to(F64).abs().amax(dims)
    bad = ~torch.isfinite(x)
    for d in sorted(dims, reverse=True):
        bad = bad.any(d)
    return torch.where(bad, torch.full_like(top, math.nan), top)


def quotients(x: torch.Tensor, top: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype):
    """x * (127 or 448) / top where the scale counts, 0 where it is 0 or NaN."""
    y = x.to(F64) * TOP[dtype] / top
    return torch.where(scale > 0, y, torch.zeros_like(y))


def quantize_rows(x: torch.Tensor, dtype: torch.dtype):
    """(codes, scales) of the last dimension."""
    top = amax(x, (x.dim() - 1,))
    scale = scale_f32(top, dtype)
    return codes(quotients(x, top[..., None], scale[..., None], dtype), dtype), scale


def rms_norm(x, weight=None, eps=1e-6, residual=None, offset=0.0):
    """(hidden bf16, normed float64)."""
    h = x if residual is None else (x.float() + residual.float()).to(torch.bfloat16)
    y = h.to(F64)
    y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)
    return h, y if weight is None else y * (weight.to(F64) + offset)


def linear(codes, scales, w_codes, w_scales, bias=None):
    y = (codes.to(F64) @ w_codes.to(F64).T) * scales.to(F64)[..., None] * w_scales.to(F64)
    return y if bias is None else y + bias.to(F64)


def rows_of(starts, batch: int, rows: int) -> list[tuple[int, int]]:
    if starts is None:
        n = rows // batch
        return [(b * n, n) for b in range(batch)]
    s = starts.tolist()
    return [(s[b], s[b + 1] - s[b]) for b in range(batch)]


def cache_write(held_codes, held_scales, x, table, lengths, starts=None):
    """New (codes, scales) of one of keys or values; x (rows, heads, dim)."""
    dtype, block = held_codes.dtype, held_codes.shape[2]
    out, scales = held_codes.float().clone(), held_scales.clone()
    for b, (first, n) in enumerate(rows_of(starts, len(lengths), x.shape[0])):
        held = int(lengths[b])
        for j in range(held // block, (held + n - 1) // block + 1 if n else 0):
            page = int(table[b, j])
            t0, t1 = max(held, j * block), min(held + n, (j + 1) * block)
            new = x[first + t0 - held : first + t1 - held].float().transpose(0, 1)
            earlier = max(0, held - j * block)
            top = amax(new, (1, 2))[:, None, None]
            own = scale_f32(top, dtype)
            before = scales[page][:, None, None] if earlier else torch.zeros_like(own)
            scale = torch.maximum(own, before)  # NaN wins
            if earlier:
                old = out[page, :, :earlier]
                again = codes(quotients(old.to(F64) * before.to(F64), top, scale, dtype), dtype).float()
                out[page, :, :earlier] = torch.where(scale > before, again, old)
            value = torch.where(scale > before, quotients(new, top, scale, dtype),
                                torch.where(scale > 0, new.to(F64) / before.to(F64), 0.0))
            out[page, :, t0 - j * block : t1 - j * block] = codes(value, dtype).float()
            scales[page] = scale[:, 0, 0]
    return out.to(dtype), scales


def cached(codes, scales, table_row, length: int) -> torch.Tensor:
    """(heads, length, dim) float64 values of one sequence."""
    block = codes.shape[2]
    pages = [codes[int(p)].to(F64) * scales[int(p)].to(F64)[:, None, None]
             for p in table_row[: -(-length // block)]]
    if not pages:
        return torch.zeros((codes.shape[1], 0, codes.shape[3]), dtype=F64)
    return torch.cat(pages, 1)[:, :length]


def attention(q, k_codes, v_codes, k_scales, v_scales, table, lengths, starts=None, *, causal=True,
              scale=None):
    """(out, weight, reach, crowd) float64 like q: softmax attention, zeros for rows without keys.
    What the rounding errors of an implementation in shorter types scale with: weight = softmax @
    |v|, reach = the largest sum of |q k| * scale a row meets, crowd = the keys it sees times the
    largest value that any of their V blocks can hold."""
    rows, heads, dim = q.shape
    group = heads // k_codes.shape[1]
    scale = dim**-0.5 if scale is None else scale
    out, weight = (torch.zeros(q.shape, dtype=F64) for _ in range(2))
    reach, crowd = (torch.zeros((rows, heads, 1), dtype=F64) for _ in range(2))
    for b, (first, n) in enumerate(rows_of(starts, len(lengths), rows)):
        length = int(lengths[b])
        k = cached(k_codes, k_scales, table[b], length)
        v = cached(v_codes, v_scales, table[b], length)
        for i in range(n):
            seen = min(length, max(0, length - n + i + 1)) if causal else length
            if seen == 0:
                continue
            for h in range(heads):
                x, kk, vv = q[first + i, h].to(F64), k[h // group, :seen], v[h // group, :seen]
                p = torch.softmax(kk @ x * scale, 0)
                out[first + i, h] = p @ vv
                weight[first + i, h] = p @ vv.abs()
                reach[first + i, h] = (kk.abs() @ x.abs()).max() * scale
                blocks = [int(p) for p in table[b][: -(-seen // k_codes.shape[2])]]
                crowd[first + i, h] = (seen * TOP[v_codes.dtype]
                                       * v_scales[blocks, h // group].to(F64).max())
    return out, weight, reach, crowd


def attention_by_products(q, k_codes, v_codes, k_scales, v_scales, table, lengths, starts=None, *,
                          causal=True, scale=None):
    """What `attention` gives, for long sequences: matrix products on the tensors' device."""
    rows, heads, dim = q.shape
    cache_heads, block = k_codes.shape[1:3]
    group = heads // cache_heads
    scale = dim**-0.5 if scale is None else scale
    like = dict(dtype=F64, device=q.device)
    out, weight = (torch.zeros(q.shape, **like) for _ in range(2))
    reach, crowd = (torch.zeros((rows, heads, 1), **like) for _ in range(2))
    for b, (first, n) in enumerate(rows_of(starts, len(lengths), rows)):
        length = int(lengths[b])
        if not length or not n:
            continue
        k = cached(k_codes, k_scales, table[b], length)
        v = cached(v_codes, v_scales, table[b], length)
        pages = table[b, : -(-length // block)].long().to(q.device)
        tops = v_scales[pages].to(F64).cummax(0).values  # (pages, heads): the largest so far
        for i0 in range(0, n, 128):
            i = torch.arange(i0, min(n, i0 + 128), device=q.device)
            seen = (length - n + i + 1).clamp(0, length) if causal else torch.full_like(i, length)
            hidden = (torch.arange(length, device=q.device)[None] >= seen[:, None])[:, None]
            last = ((seen - 1).clamp(min=0) // block)
            for h in range(cache_heads):
                at = (slice(first + i0, first + i0 + len(i)), slice(h * group, (h + 1) * group))
                x = q[at].to(F64)
                s = (x @ k[h].T * scale).masked_fill(hidden, -math.inf)
                p = torch.softmax(s, -1).masked_fill((seen == 0)[:, None, None], 0.0)
                out[at], weight[at] = p @ v[h], p @ v[h].abs()
                reach[at] = ((x.abs() @ k[h].abs().T).masked_fill(hidden, 0.0)
                             .amax(-1, keepdim=True) * scale)
                crowd[at] = (seen * TOP[v_codes.dtype] * tops[last, h])[:, None, None]
    return out, weight, reach, crowd
