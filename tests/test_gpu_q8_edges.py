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


def _far_rows(dim):
    """(x, eps) whose squares, products or their sum leave fp32, each beside an ordinary row."""
    base = _normal((6, dim), dim, 1.0).float()
    base[:, 0] = 3.0
    out = []
    for factor, eps in ((1e20, 1e-6), (2.0**126, 1e-6), (1e-30, 0.0), (1e-39, 0.0), (1e-37, 1e-6),
                        (1e-37, 1e-12), (1e-25, 1e-35), (1e19, 0.0)):
        x = base.clone()
        x[1:4] *= factor
        x[2, 1:] *= 1e-3 if factor > 1 else 1.0  # one large value
        x[4] = 0
        out.append((x.clamp(-3.3e38, 3.3e38).to(BF16), eps))
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [8, 128, 5000, 20008])
@pytest.mark.parametrize("form", ["plain", "residual", "weight"])
def test_norm_of_rows_whose_squares_leave_fp32(cuda_device, dtype, dim, form):
    for i, (x, eps) in enumerate(_far_rows(dim)):
        r = (x.float() * -0.5).to(BF16) if form == "residual" else None
        w = None
        if form == "weight":  # products that overflow or vanish before the root is taken
            w = (_normal((dim,), i, 0.5).float() * (1e25 if i % 2 else 1e-10)).to(BF16)
        args = [t if t is None else t.to(cuda_device) for t in (x, w)]
        rd = None if r is None else r.to(cuda_device)
        codes, scales, hidden = ops_q8.rms_norm_quantize(
            *args, eps, residual=rd, dtype=dtype, hidden=rd)  # the sum over the residual
        h, y = ref.rms_norm(x, w, eps, r)
        y = torch.where(h == 0, torch.zeros_like(y), y)  # a row of zeros without eps is 0 / 0
        assert torch.equal(hidden.cpu(), h)
        want = y.abs().amax(-1) / ref.TOP[dtype]
        none = want < 2.0**-126
        assert bool(((want < 0.99 * 2.0**-126) | (want > 1.01 * 2.0**-126)).all())  # no border case
        got = scales.cpu().double()
        # as for ordinary rows: a sum of squares and its root in fp32 below 3e-6, codes below
        # 4 * 2^-24 in front of their own rounding; longer sums only where fp64 is used
        assert not got[none].any() and not codes.cpu().double()[none].any()
        assert bool(((got - want).abs() <= 3e-6 * want)[~none].all()), (i, got, want)
        c = codes.cpu().double()[~none]
        q = y[~none] / want[~none, None]
        half = 0.5 if dtype == INT8 else torch.clamp(q.abs() * 2.0**-4, min=2.0**-10)
        assert bool(((c - q).abs() <= half + 4 * 2.0**-24 * (c.abs() + 1)).all()), i


@pytest.mark.parametrize("dim", [128, 20008])
def test_norm_of_rows_that_are_not_finite(cuda_device, dim):
    x = _normal((5, dim), 3)
    x[0, 5], x[1, 6], x[2, 7], x[3] = math.inf, -math.inf, math.nan, 1e25
    x[3, 9] = math.nan
    w = torch.ones(dim, dtype=BF16)
    w[5] = 0  # infinity times 0
    for weight in (None, w):
        codes, scales, _ = ops_q8.rms_norm_quantize(
            x.to(cuda_device), None if weight is None else weight.to(cuda_device))
        assert scales[:4].isnan().all() and not codes[:4].any()
        alone = ops_q8.rms_norm_quantize(x[4:].to(cuda_device),
                                         None if weight is None else weight.to(cuda_device))
        assert torch.equal(codes[4:], alone[0]) and torch.equal(scales[4:], alone[1])


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


# ---------------------------------------------------------------- attention
def _cache(batch, most, heads, dim, block, dtype, seed, device, codes=127):
    g = torch.Generator().manual_seed(seed)
    per = max(1, -(-most // block))
    table = torch.randperm(batch * per, generator=g).view(batch, per).to(torch.int32)
    cc = [torch.randint(-codes, codes + 1, (batch * per, heads, block, dim), generator=g)
          for _ in range(2)]
    scales = [(torch.rand((batch * per, heads), generator=g) + 0.5) * 0.02 for _ in range(2)]
    cpu = ops_q8.KVCache(*((c if dtype == INT8 else c.float()).to(dtype) for c in cc), *scales)
    return cpu, ops_q8.KVCache(*(t.to(device) for t in cpu)), table


def _check(got, want, weight, reach, crowd, keys):
    # f16 weights 2^-11 (2^-25 below 2^-14, against a largest of at least 1: `crowd`), scores by
    # at most (dim + 4) * 2^-24 of their sum of magnitudes and exponentials 2^-20 (numerator and
    # denominator), sums over the keys 2^-24 an addition (the tensor cores 2^-23), bf16 2^-8
    dim = want.shape[-1]
    inner = ((2.0**-11 + 2 * ((dim + 4) * 2.0**-24 * reach + 2.0**-20) + 3 * keys * 2.0**-24)
             * weight + 2.0**-25 * crowd)
    limit = inner + 2.0**-8 * (want.abs() + inner) + 1e-30
    assert got.isfinite().all()
    assert bool(((got.double() - want).abs() <= limit).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("rows", "group"), [(1, 2), (6, 2), (70, 2)])
@pytest.mark.parametrize("held", [100, 300])
def test_attention_of_the_largest_queries(cuda_device, dtype, rows, group, held):
    """Finite queries up to the largest bf16 values, with keys whose products stay in fp32."""
    dim, heads = 128, 2
    cpu, cache, table = _cache(1, held, heads, dim, 32, dtype, 3, cuda_device, codes=1)
    for t in (cpu, cache):
        t.k_scales.fill_(2.0**-120)
    q = torch.zeros((rows, heads * group, dim))
    g = torch.Generator().manual_seed(4)
    at = torch.randint(0, dim, (rows, heads * group, 1), generator=g)
    q.scatter_(2, at, 2.0**127 * (1 + torch.rand(at.shape, generator=g) * 0.98))
    q = q.to(BF16)
    assert q.isfinite().all()
    lengths = torch.tensor([held], dtype=torch.int32)
    got = ops_q8.kv_cache_attention(q.to(cuda_device), cache, table.to(cuda_device),
                                    lengths.to(cuda_device), scale=0.02)
    _check(got.cpu(), *ref.attention(q, *cpu, table, lengths, scale=0.02), held)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("rows", "group"), [(1, 2), (6, 2)])
def test_attention_of_subnormal_queries(cuda_device, dtype, rows, group):
    dim, heads, held = 128, 2, 150
    cpu, cache, table = _cache(1, held, heads, dim, 32, dtype, 5, cuda_device)
    for t in (cpu, cache):
        t.k_scales.fill_(2.0**112)
    q = (_normal((rows, heads * group, dim), 6).float() * 2.0**-128).to(BF16)
    q[q.abs() >= 2.0**-126] = 2.0**-127
    assert q.any() and bool((q.abs() < 2.0**-126).all())
    lengths = torch.tensor([held], dtype=torch.int32)
    got = ops_q8.kv_cache_attention(q.to(cuda_device), cache, table.to(cuda_device),
                                    lengths.to(cuda_device), scale=32.0)
    _check(got.cpu(), *ref.attention(q, *cpu, table, lengths, scale=32.0), held)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("rows", "group"), [(2, 2), (7, 2), (140, 1)])
@pytest.mark.parametrize("held", [60, 300])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_attention_of_infinite_queries(cuda_device, dtype, rows, group, held, value):
    """Every score of such a row is infinite or NaN, so its softmax is NaN, also where all of them
    are minus infinity; no other row changes, and a row that sees no key stays 0."""
    dim, heads = 64, 2
    cpu, cache, table = _cache(1, held, heads, dim, 16, dtype, 7, cuda_device)
    for t in (cpu, cache):  # all keys on one side: the code of 5
        t.k_codes.view(torch.uint8)[..., 7] = 5 if dtype == INT8 else 0x4A
    q = _normal((rows, heads * group, dim), 8)
    lengths = torch.tensor([held], dtype=torch.int32)
    want = ref.attention(q, *cpu, table, lengths)
    bad = torch.zeros((rows, heads * group), dtype=torch.bool)
    bad[0, 0] = bad[rows - 1, heads * group - 1] = True
    qb = q.clone()
    qb[..., 7][bad] = value
    got = ops_q8.kv_cache_attention(qb.to(cuda_device), cache, table.to(cuda_device),
                                    lengths.to(cuda_device)).cpu()
    ops.device_status()
    if held < rows:
        assert not got[0].any()
        bad[0, 0] = False
    assert got[bad].isnan().all()
    _check(got[~bad], *(t[~bad] for t in want), held)


@pytest.mark.parametrize("rows", [4, 90])
def test_attention_takes_rows_and_heads_in_any_order(cuda_device, rows):
    dim, heads, group = 64, 2, 3
    _, cache, table = _cache(2, 200, heads, dim, 32, INT8, 9, cuda_device)
    lengths = torch.tensor([200, 130], dtype=torch.int32, device=cuda_device)
    args = (cache, table.to(cuda_device), lengths)
    q = _normal((2 * rows, heads * group, dim), 10).to(cuda_device)
    want = ops_q8.kv_cache_attention(q, *args)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)  # heads outside
    assert torch.equal(ops_q8.kv_cache_attention(turned, *args), want)
    out = torch.empty((heads * group, 2 * rows, dim), dtype=BF16, device=cuda_device).transpose(0, 1)
    ops_q8.kv_cache_attention(turned, *args, out=out)
    assert torch.equal(out, want)
    # one head, and one row, for all of them
    for same in (q[:, :1].expand(-1, heads * group, -1), q[:1].expand(2 * rows, -1, -1)):
        assert torch.equal(ops_q8.kv_cache_attention(same, *args),
                           ops_q8.kv_cache_attention(same.contiguous(), *args))


def test_a_cache_whose_offsets_pass_32_bits(cuda_device):
    heads, block, dim, blocks = 8, 128, 128, 32776  # 2^32 + 2^20 bytes of codes, K and V each
    big = ops_q8.new_kv_cache(blocks, heads, dim, block_tokens=block, device=cuda_device)
    small = ops_q8.new_kv_cache(8, heads, dim, block_tokens=block, device=cuda_device)
    pages = torch.tensor([[32775, 3, 16390], [8200, 32769, 32770]], dtype=torch.int32, device=cuda_device)
    near = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device=cuda_device)
    k, v = _normal((2 * 330, heads, dim), 1).to(cuda_device), _normal((2 * 330, heads, dim), 2).to(cuda_device)
    zero = torch.zeros(2, dtype=torch.int32, device=cuda_device)
    after = zero + 330
    for cache, table in ((big, pages), (small, near)):
        ops_q8.kv_cache_write(cache, k, v, table, zero)
    for a, b in zip(ops_q8.kv_cache_read(big, pages, after, 333),
                    ops_q8.kv_cache_read(small, near, after, 333)):
        assert torch.equal(a, b) and a[:, :330].any()
    for rows in (1, 9, 120):
        q = _normal((2 * rows, heads, dim), rows).to(cuda_device)
        assert torch.equal(ops_q8.kv_cache_attention(q, big, pages, after),
                           ops_q8.kv_cache_attention(q, small, near, after))
    ops.device_status()


# ---------------------------------------------------------------- as a program uses them
@pytest.mark.parametrize(("batch", "rows"), [(3, 3), (3, 12), (2, 200)])
def test_graphs_replayed_with_other_lengths_starts_and_tables(cuda_device, batch, rows):
    """Write, read and attention captured once; every replay finds other sizes on the device."""
    dim, heads, group, block, most = 64, 2, 2, 16, 320
    cpu, cache, table = _cache(batch, most, heads, dim, block, E4M3, 21, cuda_device)
    first = [t.clone() for t in cache]
    dev_table = table.to(cuda_device)
    lengths, after, starts = (torch.zeros(n, dtype=torch.int32, device=cuda_device)
                              for n in (batch, batch, batch + 1))
    q = _normal((rows, heads * group, dim), 22).to(cuda_device)
    k, v = (_normal((rows, heads, dim), s).to(cuda_device) for s in (23, 24))
    out = torch.empty_like(q)

    def run():
        ops_q8.kv_cache_write(cache, k, v, dev_table, lengths, starts)
        read = ops_q8.kv_cache_read(cache, dev_table, after, most)
        ops_q8.kv_cache_attention(q, cache, dev_table, after, starts, out=out)
        return read

    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        run()
    stream.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        read = run()
    g = torch.Generator().manual_seed(25)
    for step in range(6):
        cut = torch.sort(torch.randint(0, rows + 1, (batch - 1,), generator=g)).values
        s = torch.cat([torch.zeros(1, dtype=torch.long), cut, torch.tensor([rows if step % 2 else max(cut)])])
        held = torch.randint(0, 100 if step < 5 else 1, (batch,), generator=g).to(torch.int32)
        n = (s[1:] - s[:-1]).to(torch.int32)
        page = table[torch.randperm(batch, generator=g)]
        for t, value in ((starts, s), (lengths, held), (after, held + n), (dev_table, page)):
            t.copy_(value)
        for t, b in zip(cache, first):
            t.copy_(b)
        out.fill_(7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ops.device_status()
        want = [ref.cache_write(cpu[i], cpu[2 + i], x.cpu()[: int(s[-1])], page, held, s)
                for i, x in enumerate((k, v))]
        for i in range(2):
            assert torch.equal(cache[2 + i].cpu(), want[i][1]) and _same(cache[i], want[i][0])
            for b in range(batch):
                length = int(held[b] + n[b])
                y = ref.cached(*want[i], page[b], length).transpose(0, 1)
                assert torch.equal(read[i][b, :length].cpu(), y.float().to(BF16))
                assert not read[i][b, length:].any()
        parts = ref.attention(q.cpu()[: int(s[-1])], want[0][0], want[1][0], want[0][1], want[1][1],
                              page, held + n, s)
        _check(out[: int(s[-1])].cpu(), *parts, most)
        assert bool((out[int(s[-1]):] == 7).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_decoding_token_by_token_behind_a_shared_prefix(cuda_device, dtype):
    """Sequences that share the blocks of a prefix and write behind it, a token at a time: the cache
    holds the oracle's codes after every step, and each step's attention reads it all."""
    dim, heads, group, block, batch, prefix, steps = 128, 2, 4, 32, 3, 64, 40
    cpu = ops_q8.new_kv_cache(2 + 2 * batch, heads, dim, block_tokens=block, dtype=dtype, device="cpu")
    cache = ops_q8.KVCache(*(t.to(cuda_device) for t in cpu))
    table = torch.tensor([[0, 1, 2 + 2 * b, 3 + 2 * b] for b in range(batch)], dtype=torch.int32)
    dev = table.to(cuda_device)
    x = [_normal((prefix, heads, dim), s) for s in (31, 32)]
    zero = torch.zeros(1, dtype=torch.int32)
    ops_q8.kv_cache_write(cache, *(t.to(cuda_device) for t in x), dev[:1], zero.to(cuda_device))
    state = [ref.cache_write(cpu[i], cpu[2 + i], x[i], table[:1], zero) for i in range(2)]
    for step in range(steps):
        held = torch.full((batch,), prefix + step, dtype=torch.int32)
        size = 4.0 if step % 7 == 3 else 1.0  # now and then the blocks' scales grow
        new = [_normal((batch, 1, dim), 100 + step, size), _normal((batch, heads, dim), 200 + step, size)]
        new[0] = new[0].expand(batch, heads, dim)  # one key for all heads, a stride of 0
        ops_q8.kv_cache_write(cache, new[0].to(cuda_device)[:, :1].expand(batch, heads, dim),
                              new[1].to(cuda_device), dev, held.to(cuda_device))
        state = [ref.cache_write(*state[i], new[i], table, held) for i in range(2)]
        for i in range(2):
            assert torch.equal(cache[2 + i].cpu(), state[i][1]), step
            assert _same(cache[i], state[i][0]), step
        if step % 13 == 0:
            q = _normal((batch, heads * group, dim), 300 + step)
            got = ops_q8.kv_cache_attention(q.to(cuda_device), cache, dev, (held + 1).to(cuda_device))
            _check(got.cpu(), *ref.attention(q, state[0][0], state[1][0], state[0][1], state[1][1],
                                             table, held + 1), prefix + step + 1)
    ops.device_status()
