"""8-bit serving operators on the GPU against their definitions in 64 bits.

Where a kernel rounds at the same places as the oracle (quantising bf16 values, the cache) codes and
scales are equal bit for bit. Elsewhere a bound counts the roundings: fp32 2^-24, bf16 2^-8 of the
value each, half a code step for a code.
"""

from __future__ import annotations

import math

import pytest
import torch

from kinomlx_b200 import ops, ops_q8
from oracle import serving_q8 as ref

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
INT8, E4M3 = torch.int8, torch.float8_e4m3fn
DTYPES = [INT8, E4M3]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _normal(shape, seed, std=1.0):
    return (torch.randn(shape, generator=_gen(seed)) * std).to(BF16)


def _same(a, b):
    a, b = a.cpu().float(), b.cpu().float()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


# ---------------------------------------------------------------- rows
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("rows", "dim"), [(1, 8), (3, 64), (5, 504), (17, 1032), (2, 4096),
                                           (3, 8200), (2, 16384), (3, 20008),
                                           (1300, 96), (1, 131072)])
def test_quantize_tokens_is_exact(cuda_device, dtype, rows, dim):
    x = _normal((rows, dim), rows + dim)
    x[0] *= 1e-3
    codes, scales = ops_q8.quantize_tokens(x.to(cuda_device), dtype)
    want, want_scales = ref.quantize_rows(x, dtype)
    assert codes.dtype == dtype and torch.equal(scales.cpu(), want_scales)
    assert _same(codes, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_tokens_special_rows(cuda_device, dtype):
    x = _normal((7, 128), 3)
    x[0] = 0
    x[1] = 1e-37  # scale below 2^-126
    x[2, 5] = math.inf
    x[3, 77] = math.nan
    x[4] = 3.3e38
    x[5] = 1e-34
    codes, scales = ops_q8.quantize_tokens(x.to(cuda_device), dtype)
    want, want_scales = ref.quantize_rows(x, dtype)
    assert _same(scales, want_scales) and _same(codes, want)
    assert scales[:2].tolist() == [0.0, 0.0] and scales[2:4].isnan().all()
    assert not codes[:4].float().any() and scales[4:].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("rows", "dim"), [(1, 8), (3, 264), (9, 2048), (2, 5000), (2, 16384),
                                           (2, 28672), (1250, 80)])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("weight", [False, True])
def test_rms_norm_quantize(cuda_device, dtype, rows, dim, residual, weight):
    x = _normal((rows, dim), dim, 2.0)
    r = _normal((rows, dim), dim + 1, 3.0) if residual else None
    w = _normal((dim,), dim + 2, 0.3) if weight else None
    codes, scales, hidden = ops_q8.rms_norm_quantize(
        x.to(cuda_device), None if w is None else w.to(cuda_device), 1e-5,
        residual=None if r is None else r.to(cuda_device), dtype=dtype,
        weight_offset=1.0 if weight else 0.0)
    h, y = ref.rms_norm(x, w, 1e-5, r, 1.0)
    assert torch.equal(hidden.cpu(), h)
    # scale: a sum of squares of up to 66 fp32 additions in a row, halved by the root; rsqrtf 2 ulp;
    # four products and quotients and the weight's sum: below 3e-6 of the value. Codes do not depend
    # on the root: the weight's sum and two products, below 4 * 2^-24
    want = y.abs().amax(-1) / ref.TOP[dtype]
    assert bool(((scales.cpu().double() - want).abs() <= 3e-6 * want).all())
    c = codes.cpu().double()
    off = (c - y / want[:, None]).abs()
    half = 0.5 if dtype == INT8 else torch.clamp((y / want[:, None]).abs() * 2.0**-4, min=2.0**-10)
    assert bool((off <= half + 4 * 2.0**-24 * (c.abs() + 1)).all())


def test_rms_norm_quantize_in_place_and_strided(cuda_device):
    wide = _normal((6, 3 * 256), 5).to(cuda_device)
    x, r = wide[:, 256:512], _normal((6, 256), 6).to(cuda_device)
    expect = ops_q8.rms_norm_quantize(x.contiguous(), residual=r.clone())
    before = wide.clone()
    codes, scales, hidden = ops_q8.rms_norm_quantize(x, residual=r, hidden=r)
    assert hidden is r
    for got, want in zip((codes, scales, hidden), expect):
        assert torch.equal(got, want)
    assert torch.equal(wide, before)
    one = ops_q8.quantize_tokens(wide[:1, 256:500].as_strided((1, 240), (13, 1)))  # any stride of one row
    assert torch.equal(one[0], ops_q8.quantize_tokens(wide[:1, 256:496].contiguous())[0])
    three = ops_q8.quantize_tokens(r.view(2, 3, 256))
    two = ops_q8.quantize_tokens(r)
    assert three[0].shape == (2, 3, 256) and three[1].shape == (2, 3)
    assert torch.equal(three[0].view(6, 256), two[0]) and torch.equal(three[1].view(6), two[1])


# ---------------------------------------------------------------- product
def _product(m, n, k, seed, bias, device):
    g = _gen(seed)
    x = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8)
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    sx = torch.rand(m, generator=g) * 0.1
    sw = torch.rand(n, generator=g) * 0.01
    b = _normal((n,), seed, 3.0) if bias else None
    return [t if t is None else t.to(device) for t in (x, sx, w, sw, b)], ref.linear(x, sx, w, sw, b)


def _check_product(out, exact, bias):
    # three fp32 roundings of the scaled sum, one of the sum with the bias, one to bf16
    top = exact.abs() + (0 if bias is None else 2 * bias.cpu().double().abs())
    off = (out.cpu().double() - exact).abs()
    assert bool((off <= 2.0**-8 * exact.abs() + 4 * 2.0**-24 * top * (1 + 2.0**-8)).all()), float(off.max())


@pytest.mark.parametrize(("m", "n", "k"), [
    (1, 8, 16), (1, 4096, 4096), (2, 136, 128), (7, 1000, 272), (16, 640, 2064), (17, 384, 1040),
    (33, 256, 512), (64, 128, 144), (65, 264, 384), (126, 520, 1024), (129, 128, 256),
    (256, 512, 768), (257, 256, 128), (300, 1000, 400), (513, 264, 2048), (1025, 768, 640),
    (100, 33800, 64), (300, 6400, 144), (1025, 2600, 640),
])
@pytest.mark.parametrize("bias", [False, True])
def test_linear_int8(cuda_device, m, n, k, bias):
    args, exact = _product(m, n, k, m + n + k, bias, cuda_device)
    _check_product(ops_q8.linear_int8(*args), exact, args[4])
    ops.device_status()


def test_linear_int8_extremes_and_strides(cuda_device):
    # the largest sums that 16384 codes give, beyond fp32's whole numbers
    k = 16384
    x = torch.full((3, k), 127, dtype=torch.int8, device=cuda_device)
    w = torch.full((8, k), -127, dtype=torch.int8, device=cuda_device)
    one = torch.ones(8, device=cuda_device)
    out = ops_q8.linear_int8(x, one[:3].contiguous(), w, one)
    assert bool((out.float() == torch.tensor(-127.0 * 127 * k).to(BF16).float()).all())
    # a slice of wider codes, weights and outputs
    for m in (5, 300):
        args, exact = _product(m, 264, 512, m, True, cuda_device)
        xw = torch.zeros((m, 1024), dtype=torch.int8, device=cuda_device)
        ww = torch.zeros((264, 528), dtype=torch.int8, device=cuda_device)
        xw[:, 512:] = args[0]
        ww[:, 16:] = args[2]
        wide = torch.full((m, 800), 7.0, dtype=BF16, device=cuda_device)
        ops_q8.linear_int8(xw[:, 512:], args[1], ww[:, 16:], args[3], args[4], wide[:, 8:272])
        _check_product(wide[:, 8:272], exact, args[4])
        assert bool((wide[:, :8] == 7).all()) and bool((wide[:, 272:] == 7).all())
    # scales of NaN and 0 stay in their rows and columns
    args, _ = _product(20, 128, 128, 1, False, cuda_device)
    args[1][3], args[1][4], args[3][7] = math.nan, 0.0, math.nan
    out = ops_q8.linear_int8(*args)
    assert out[3].isnan().all() and out[:, 7].isnan().all()
    rest = torch.ones(out.shape, dtype=torch.bool, device=cuda_device)
    rest[3] = False
    rest[:, 7] = False
    assert out[rest].isfinite().all() and not out[4, :7].any()


# ---------------------------------------------------------------- cache
def _cache(batch, most, heads, dim, block, dtype, seed, device, pool=0):
    """A cache with random codes and scales everywhere, and a table of distinct blocks."""
    g = _gen(seed)
    per = max(1, -(-most // block))
    blocks = batch * per + 1 + pool
    table = torch.randperm(blocks, generator=g)[: batch * per].view(batch, per).to(torch.int32)
    codes = [torch.randint(-127, 128, (blocks, heads, block, dim), generator=g) for _ in range(2)]
    if dtype == INT8:
        codes = [c.to(INT8) for c in codes]
    else:
        codes = [(c * 3.5).clamp(-448, 448).to(E4M3) for c in codes]
    scales = [(torch.rand((blocks, heads), generator=g) + 0.5) * 0.02 for _ in range(2)]
    cpu = ops_q8.KVCache(*codes, *scales)
    return cpu, ops_q8.KVCache(*(t.to(device) for t in cpu)), table


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize(("held", "new"), [
    ([0], [1]), ([5, 64, 127], [1, 1, 1]), ([0, 63, 130, 17], [200, 1, 0, 47]),
    ([128, 1], [128, 129]),
])
def test_cache_write_and_read(cuda_device, dtype, block, dim, held, new):
    heads, batch = 3, len(held)
    most = max(h + n for h, n in zip(held, new))
    cpu, cache, table = _cache(batch, most, heads, dim, block, dtype, block + dim, cuda_device)
    rows = sum(new)
    k, v = _normal((rows + 2, heads, dim), 1, 0.5), _normal((rows + 2, heads, dim), 2, 3.0)
    k[0] *= 20  # a token that makes the scales of its block grow
    starts = torch.tensor([0] + [sum(new[: i + 1]) for i in range(batch)], dtype=torch.int32)
    lengths = torch.tensor(held, dtype=torch.int32)
    uniform = len(set(new)) == 1
    if uniform:
        k, v, dev_starts = k[:rows], v[:rows], None
    else:
        dev_starts = starts.to(cuda_device)  # two rows behind the last sequence
    ops_q8.kv_cache_write(cache, k.to(cuda_device), v.to(cuda_device), table.to(cuda_device),
                          lengths.to(cuda_device), dev_starts)
    ops.device_status()
    want = []
    for c, s, x in ((cpu.k_codes, cpu.k_scales, k), (cpu.v_codes, cpu.v_scales, v)):
        want.append(ref.cache_write(c, s, x[:rows], table, lengths, starts))
    for i in range(2):
        assert torch.equal(cache[2 + i].cpu(), want[i][1])
        assert _same(cache[i], want[i][0])  # every block, the untouched ones too
    after = lengths + torch.tensor(new, dtype=torch.int32)
    tokens = most + 3
    got = ops_q8.kv_cache_read(cache, table.to(cuda_device), after.to(cuda_device), tokens)
    ops.device_status()
    for i in range(2):
        for b in range(batch):
            n = int(after[b])
            y = ref.cached(want[i][0], want[i][1], table[b], n).transpose(0, 1)
            assert torch.equal(got[i][b, :n].cpu(), y.float().to(BF16))
            assert not got[i][b, n:].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_cache_write_not_finite_and_zero(cuda_device, dtype):
    cpu, cache, table = _cache(2, 64, 2, 64, 32, dtype, 9, cuda_device)
    k, v = _normal((2, 2, 64), 1), torch.zeros((2, 2, 64), dtype=BF16)
    k[0, 1, 3] = math.nan
    k[1, 0, 9] = -math.inf
    lengths = torch.tensor([0, 40], dtype=torch.int32)
    args = (table.to(cuda_device), lengths.to(cuda_device))
    ops_q8.kv_cache_write(cache, k.to(cuda_device), v.to(cuda_device), *args)
    for i, x in enumerate((k, v)):
        codes, scales = ref.cache_write(cpu[i], cpu[2 + i], x, table, lengths)
        assert _same(cache[2 + i], scales) and _same(cache[i], codes)
    assert cache.k_scales[table[0, 0].long(), 1].isnan() and cache.k_scales[table[1, 1].long(), 0].isnan()
    assert float(cache.v_scales[table[0, 0].long(), 0]) == 0.0
    # a block that held a NaN stays one
    ops_q8.kv_cache_write(cache, _normal((2, 2, 64), 5).to(cuda_device), v.to(cuda_device),
                          args[0], args[1] + 1)
    assert cache.k_scales[table[0, 0].long(), 1].isnan()


def test_cache_write_strides(cuda_device):
    cpu, cache, table = _cache(2, 100, 4, 128, 64, INT8, 4, cuda_device)
    qkv = _normal((20, 3, 4, 128), 8)
    lengths = torch.tensor([60, 3], dtype=torch.int32)
    dev = qkv.to(cuda_device)
    ops_q8.kv_cache_write(cache, dev[:, 1], dev[:, 2], table.to(cuda_device), lengths.to(cuda_device))
    for i in range(2):
        codes, scales = ref.cache_write(cpu[i], cpu[2 + i], qkv[:, 1 + i], table, lengths)
        assert torch.equal(cache[2 + i].cpu(), scales) and _same(cache[i], codes)


# ---------------------------------------------------------------- attention
def _attend(cuda_device, held, new, heads, group, dim, block, dtype, *, causal=True, seed=0,
            scale=None, spread=1.0, packed=None):
    batch = len(held)
    cpu, cache, table = _cache(batch, max(max(held), 1), heads, dim, block, dtype, seed, cuda_device)
    if spread != 1.0:  # scales that differ between blocks by powers of `spread`
        power = torch.randint(-2, 3, cpu.v_scales.shape, generator=_gen(seed + 7)).float()
        cpu.v_scales.mul_(spread**power)
        cache.v_scales.copy_(cpu.v_scales)
    packed = len(set(new)) > 1 if packed is None else packed
    extra = 3 if packed else 0
    rows = sum(new)
    q = _normal((rows + extra, heads * group, dim), seed + 1, 2.0)
    starts = torch.tensor([0] + [sum(new[: i + 1]) for i in range(batch)], dtype=torch.int32)
    lengths = torch.tensor(held, dtype=torch.int32)
    out = torch.full(q.shape, 5.0, dtype=BF16, device=cuda_device)
    got = ops_q8.kv_cache_attention(
        q.to(cuda_device), cache, table.to(cuda_device), lengths.to(cuda_device),
        starts.to(cuda_device) if packed else None, causal=causal, scale=scale, out=out)
    ops.device_status()
    assert got is out and bool((out[rows:] == 5).all())
    want = ref.attention(q[:rows], cpu.k_codes, cpu.v_codes, cpu.k_scales, cpu.v_scales, table,
                         lengths, starts, causal=causal, scale=scale)
    return out[:rows].cpu(), *want


def _check_attention(got, want, weight, reach, crowd):
    # A score's fp32 sum of up to 128 products and its scaling move it by at most 132 * 2^-24 of the
    # sum of magnitudes, numerator and denominator alike; exponentials 2^-20. The weights
    # P = vs exp(s - m) are rounded to f16: 2^-11 of each, and 2^-25 where they are below 2^-14. The
    # largest P of a row is at least 1, so the row sum of P / vs is at least 1 / (largest vs), and
    # the latter is at most 2^-25 * sum |code| * (largest vs) <= 2^-25 * crowd. The result is
    # rounded to bf16, 2^-8 of it.
    dim = want.shape[-1]
    inner = (2.0**-11 + 2 * ((dim + 4) * 2.0**-24 * reach + 2.0**-20)) * weight + 2.0**-25 * crowd
    off = (got.double() - want).abs()
    limit = inner + 2.0**-8 * (want.abs() + inner) + 1e-30
    assert got.isfinite().all()
    assert bool((off <= limit).all()), float((off / limit).max())


SMALL = [  # held (with the new tokens), new, cache heads, group
    ([1], [1], 1, 1),
    ([1, 64, 65, 300], [1, 1, 1, 1], 2, 4),
    ([37, 129], [1, 1], 3, 5),
    ([500], [1], 1, 8),
    ([0, 70], [1, 1], 2, 2),
    ([260, 33], [2, 2], 2, 8),
    ([90, 200, 1], [3, 5, 1], 2, 3),
    ([40, 0, 513], [1, 0, 2], 2, 7),
    ([700], [1], 1, 16),
    ([2, 90], [4, 4], 2, 2),
    ([130, 61], [9, 20], 2, 3),
    ([200], [4], 1, 16),
]


@pytest.mark.parametrize("case", SMALL, ids=range(len(SMALL)))
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("dim", "block"), [(128, 64), (128, 16), (64, 128), (64, 16), (128, 128),
                                            (64, 32)])
def test_attention_few_rows(cuda_device, case, dtype, dim, block):
    held, new, heads, group = case
    _check_attention(*_attend(cuda_device, held, new, heads, group, dim, block, dtype,
                              causal=block != 32, seed=dim + block))


MANY = [  # held (with the new tokens), new, cache heads, group
    ([17], [17], 1, 1),
    ([130], [130], 2, 1),
    ([400], [129], 1, 1),
    ([300, 70], [40, 40], 2, 3),
    ([600, 40, 0, 129], [33, 40, 0, 65], 2, 4),
    ([257], [257], 1, 8),
    ([1000, 5], [9, 1], 1, 7),
    ([64, 200], [70, 20], 1, 5),  # more queries than keys: the first see none
    ([350], [3], 1, 100),
    ([300], [270], 3, 1),
    ([333], [12], 2, 12),
    ([70], [1], 1, 33),
    ([900, 20], [30, 12], 1, 16),
]


@pytest.mark.parametrize("case", MANY, ids=range(len(MANY)))
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("dim", "block", "causal"), [(128, 64, True), (128, 16, True),
                                                      (64, 128, True), (64, 16, False),
                                                      (128, 128, False), (64, 32, True)])
def test_attention_many_rows(cuda_device, case, dtype, dim, block, causal):
    held, new, heads, group = case
    _check_attention(*_attend(cuda_device, held, new, heads, group, dim, block, dtype,
                              causal=causal, seed=dim + block))


# ---------------------------------------------------------------- edges of attention
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("held", "new", "group"), [([90, 200, 33], [1, 1, 1], 4), ([300, 140], [40, 90], 4)])
def test_attention_scales_of_any_size(cuda_device, dtype, held, new, group):
    # V scales that differ by factors of 1000 between blocks, either way
    got = _attend(cuda_device, held, new, 2, group, 128, 16, dtype, spread=1000.0, seed=3)
    _check_attention(*got)
    # scale and no mask
    _check_attention(*_attend(cuda_device, held, new, 2, group, 64, 32, dtype, causal=False, scale=0.3))
    # a scale of 0 averages the keys
    _check_attention(*_attend(cuda_device, held, new, 2, group, 128, 64, dtype, scale=0.0))


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_not_finite_in_masked_places(cuda_device, dtype, rows):
    """Blocks that no query sees, the rest of the last block and keys behind a causal mask hold NaN
    scales and every code pattern; rows that do not see them are as without them."""
    heads, group, dim, block, held = 2, 2, 128, 16, 16 * 7 + 5
    cpu, cache, table = _cache(1, 16 * 9, heads, dim, block, dtype, 5, cuda_device)
    q = _normal((rows, heads * group, dim), 6)
    lengths = torch.tensor([held], dtype=torch.int32)
    for t in (cpu, cache):
        unseen = table[0, 8:].long().to(t.k_codes.device)
        for x in t[2:]:
            x[unseen] = math.nan
        last = int(table[0, 7])
        for x in t[:2]:
            x.view(torch.uint8)[last, :, 5:] = 0x7F  # past the length: NaN patterns in e4m3
    args = (table.to(cuda_device), lengths.to(cuda_device))
    got = ops_q8.kv_cache_attention(q.to(cuda_device), cache, *args)
    _check_attention(got.cpu(), *ref.attention(q, *cpu, table, lengths))
    # a NaN block in sight spoils the rows that see it and no other
    bad = int(table[0, 6])  # keys 96 .. 111
    cache.v_scales[bad, 1] = math.nan
    spoiled = ops_q8.kv_cache_attention(q.to(cuda_device), cache, *args).cpu()
    for i in range(rows):
        sees = held - rows + i >= 96
        assert torch.equal(spoiled[i, :group], got[i, :group].cpu())
        assert bool(spoiled[i, group:].isnan().all()) == sees
        if not sees:
            assert torch.equal(spoiled[i, group:], got[i, group:].cpu())


@pytest.mark.parametrize("rows", [1, 50])
def test_attention_zero_values_and_empty(cuda_device, rows):
    cpu, cache, table = _cache(3, 200, 2, 128, 64, INT8, 8, cuda_device)
    for t in (cpu, cache):
        first = table[0].long().to(t.k_codes.device)
        t.v_codes[first] = 0
        t.v_scales[first] = 0.0
    lengths = torch.tensor([200, 0, 130], dtype=torch.int32)
    q = _normal((3 * rows, 2, 128), 9)
    got = ops_q8.kv_cache_attention(q.to(cuda_device), cache, table.to(cuda_device),
                                    lengths.to(cuda_device))
    assert not got[: 2 * rows].any()
    _check_attention(got.cpu(), *ref.attention(q, *cpu, table, lengths))
    ops.device_status()


@pytest.mark.parametrize("rows", [1, 30])
def test_attention_strides_and_in_place(cuda_device, rows):
    cpu, cache, table = _cache(2, 150, 2, 64, 32, E4M3, 12, cuda_device)
    lengths = torch.tensor([150, 77], dtype=torch.int32)
    qkv = _normal((2 * rows, 3, 6, 64), 10).to(cuda_device)
    args = (table.to(cuda_device), lengths.to(cuda_device))
    want = ops_q8.kv_cache_attention(qkv[:, 1].contiguous(), cache, *args)
    before = qkv.clone()
    out = torch.zeros((2 * rows, 6, 3, 64), dtype=BF16, device=cuda_device)
    got = ops_q8.kv_cache_attention(qkv[:, 1], cache, *args, out=out[:, :, 2])
    assert torch.equal(got, want) and not out[:, :, :2].any()
    ops_q8.kv_cache_attention(qkv[:, 1], cache, *args, out=qkv[:, 1])
    assert torch.equal(qkv[:, 1], want)
    assert torch.equal(qkv[:, 0], before[:, 0]) and torch.equal(qkv[:, 2], before[:, 2])
    _check_attention(want.cpu(), *ref.attention(before[:, 1].cpu(), *cpu, table, lengths))


@pytest.mark.parametrize(("held", "new"), [([5000], [1]), ([3000, 40], [33, 20])])
def test_attention_long_and_repeatable(cuda_device, held, new):
    got = _attend(cuda_device, held, new, 1, 2, 128, 128, INT8, seed=2)
    _check_attention(*got)
    again = _attend(cuda_device, held, new, 1, 2, 128, 128, INT8, seed=2)
    assert torch.equal(got[0], again[0])


def test_many_sequences(cuda_device):
    """More sequences than a warp scans at once, most of them short or empty."""
    held = [(7 * b) % 90 for b in range(75)]
    new = [min(h, b % 3) for b, h in enumerate(held)]
    _check_attention(*_attend(cuda_device, held, new, 1, 2, 64, 16, INT8, packed=True))
    new = [min(h, (11 * b) % 40) for b, h in enumerate(held)]
    _check_attention(*_attend(cuda_device, held, new, 1, 4, 64, 16, E4M3, packed=True))
    cpu, cache, table = _cache(75, 130, 1, 64, 16, INT8, 1, cuda_device)
    x = _normal((sum(new), 1, 64), 4)
    starts = torch.tensor([0] + [sum(new[: i + 1]) for i in range(75)], dtype=torch.int32)
    lengths = torch.tensor(held, dtype=torch.int32)
    dev = x.to(cuda_device)
    ops_q8.kv_cache_write(cache, dev, dev, table.to(cuda_device), lengths.to(cuda_device),
                          starts.to(cuda_device))
    codes, scales = ref.cache_write(cpu.k_codes, cpu.k_scales, x, table, lengths, starts)
    assert torch.equal(cache.k_scales.cpu(), scales) and _same(cache.k_codes, codes)


# ---------------------------------------------------------------- device-side sizes that do not fit
@pytest.mark.parametrize("rows", [1, 40])
def test_sizes_that_do_not_fit_are_skipped_and_reported(cuda_device, rows):
    cpu, cache, table = _cache(2, 100, 2, 64, 16, INT8, 3, cuda_device)
    lengths = torch.tensor([100, 60], dtype=torch.int32)
    q = _normal((2 * rows, 2, 64), 1).to(cuda_device)
    good = ops_q8.kv_cache_attention(q, cache, table.to(cuda_device), lengths.to(cuda_device))
    ops.device_status()
    before = [t.clone() for t in cache]

    def reported():
        with pytest.raises(RuntimeError, match="EINVAL"):
            ops.device_status()
        ops.device_status()  # and forgotten

    for page in (-1, 1 << 20, cache.k_codes.shape[0]):  # a block that the cache does not have
        bad = table.clone()
        bad[0, 2] = page
        got = ops_q8.kv_cache_attention(q, cache, bad.to(cuda_device), lengths.to(cuda_device))
        assert torch.equal(got[rows:], good[rows:]) and got.isfinite().all()
        reported()
        ops_q8.kv_cache_read(cache, bad.to(cuda_device), lengths.to(cuda_device), 100)
        reported()
        x = _normal((2 * rows, 2, 64), 2).to(cuda_device)
        at = torch.tensor([32, 60], dtype=torch.int32, device=cuda_device)
        ops_q8.kv_cache_write(cache, x, x, bad.to(cuda_device), at)
        reported()
        for t, b in zip(cache, before):
            t.copy_(b)
    # a skipped block's keys do not count: as if the sequence had a table without it
    bad = table.clone()
    bad[0, 6] = -1  # keys 96 .. 99, the last block
    got = ops_q8.kv_cache_attention(q[:rows], cache, bad[:1].to(cuda_device),
                                    lengths[:1].to(cuda_device), causal=False)
    reported()
    want = ref.attention(q[:rows].cpu(), *cpu, table[:1], torch.tensor([96]), causal=False)
    _check_attention(got.cpu(), *want)
    # lengths and starts outside the table and the rows
    for wrong in ([-1, 60], [100, 2000]):
        got = ops_q8.kv_cache_attention(q, cache, table.to(cuda_device),
                                        torch.tensor(wrong, dtype=torch.int32, device=cuda_device))
        keep = slice(rows, None) if wrong[0] < 0 else slice(0, rows)
        assert torch.equal(got[keep], good[keep])
        reported()
    full = torch.tensor([111, 60], dtype=torch.int32, device=cuda_device)  # 112 slots
    x = _normal((2 * rows, 2, 64), 2).to(cuda_device)
    ops_q8.kv_cache_write(cache, x, x, table.to(cuda_device), full)
    if rows > 1:
        reported()
    starts = torch.tensor([0, 2 * rows + 1, 2 * rows], dtype=torch.int32, device=cuda_device)
    out = torch.full_like(q, 3.0)
    ops_q8.kv_cache_attention(q, cache, table.to(cuda_device), lengths.to(cuda_device), starts, out=out)
    assert bool((out == 3).all())
    reported()


# ---------------------------------------------------------------- streams, graphs, the whole run
def _layer(dtype, seed, device, batch, tokens, held, width=256, heads=2, group=2, dim=64):
    g = _gen(seed)
    qkv_width = (heads * group + 2 * heads) * dim
    w1 = (torch.randn((qkv_width, width), generator=g) / width**0.5).to(BF16)
    w2 = (torch.randn((width, heads * group * dim), generator=g) / width**0.5).to(BF16)
    s = dict(x=_normal((batch * tokens, width), seed), residual=_normal((batch * tokens, width), seed + 1),
             norm=(1 + _normal((width,), seed + 2, 0.1).float()).to(BF16), w1=w1, w2=w2)
    s = {k: v.to(device) for k, v in s.items()}
    s["q1"], s["q2"] = ops_q8.quantize_tokens(s["w1"]), ops_q8.quantize_tokens(s["w2"])
    _, cache, table = _cache(batch, held + tokens, heads, dim, 32, dtype, seed, device)
    s |= dict(cache=cache, table=table.to(device), heads=heads, group=group, dim=dim,
              lengths=torch.full((batch,), held, dtype=torch.int32, device=device),
              after=torch.full((batch,), held + tokens, dtype=torch.int32, device=device))
    return s


def _run_layer(s):
    """One attention layer in 8 bits: norm, product, cache, attention, quantising, product."""
    codes, scales, hidden = ops_q8.rms_norm_quantize(s["x"], s["norm"], residual=s["residual"])
    qkv = ops_q8.linear_int8(codes, scales, *s["q1"])
    heads, group, dim = s["heads"], s["group"], s["dim"]
    qkv = qkv.view(qkv.shape[0], -1, dim)
    q, k, v = qkv.split([heads * group, heads, heads], 1)
    ops_q8.kv_cache_write(s["cache"], k, v, s["table"], s["lengths"])
    y = ops_q8.kv_cache_attention(q, s["cache"], s["table"], s["after"])
    return hidden, ops_q8.linear_int8(*ops_q8.quantize_tokens(y.flatten(1)), *s["q2"])


@pytest.mark.parametrize(("tokens", "held"), [(1, 70), (1, 0), (45, 20)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_layer_follows_its_64_bit_form(cuda_device, dtype, tokens, held):
    batch = 3
    s = _layer(dtype, 11, cuda_device, batch, tokens, held)
    cache0 = [t.cpu().clone() for t in s["cache"]]
    hidden, out = _run_layer(s)
    ops.device_status()
    c = {k: v.cpu() for k, v in s.items() if isinstance(v, torch.Tensor)}
    h, y = ref.rms_norm(c["x"], c["norm"], 1e-6, c["residual"])
    assert torch.equal(hidden.cpu(), h)
    # the same run without any rounding to 8 bits but the cache's earlier tokens
    heads, group, dim = s["heads"], s["group"], s["dim"]
    qkv = (y @ c["w1"].double().T).view(batch, tokens, -1, dim)
    q, k, v = qkv.split([heads * group, heads, heads], 2)
    att = torch.zeros((batch, tokens, heads * group, dim), dtype=torch.float64)
    for b in range(batch):
        old = [ref.cached(cache0[i], cache0[2 + i], c["table"][b], held) for i in range(2)]
        kk = torch.cat([old[0], k[b].transpose(0, 1)], 1)
        vv = torch.cat([old[1], v[b].transpose(0, 1)], 1)
        for i in range(tokens):
            for hd in range(heads * group):
                p = torch.softmax(kk[hd // group, : held + i + 1] @ q[b, i, hd] * dim**-0.5, 0)
                att[b, i, hd] = p @ vv[hd // group, : held + i + 1]
    want = att.flatten(2).flatten(0, 1) @ c["w2"].double().T
    # Three roundings to codes on the way (activations twice, the new keys and values) and two of
    # weights; a normal row's code error is about 0.29 steps of amax / 127, amax 3 to 4 rms: 1% of
    # the rms each in int8, 3% in e4m3 (2^-4 / sqrt 12 of each value); the sum of five, doubled.
    limit = 0.08 if dtype == INT8 else 0.12
    rel = float((out.cpu().double() - want).norm() / want.norm())
    assert rel < limit, rel


def test_streams_and_graphs(cuda_device):
    s = _layer(INT8, 21, cuda_device, 4, 1, 90)
    start = [t.clone() for t in s["cache"]]
    want = [t.clone() for t in _run_layer(s)]
    kept = [t.clone() for t in s["cache"]]
    for t, b in zip(s["cache"], start):
        t.copy_(b)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):  # another stream than the default
        got = _run_layer(s)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):  # two graphs of the same run, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            res = _run_layer(s)
        graphs.append((g, res))
    for _ in range(3):
        for g, res in graphs:
            for t, b in zip(s["cache"], start):
                t.copy_(b)
            for r in res:
                r.fill_(-1)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(res, want))
            assert all(torch.equal(a, b) for a, b in zip(s["cache"], kept))
    # two at once on two streams
    other = torch.cuda.Stream()
    t = _layer(INT8, 22, cuda_device, 4, 30, 10)
    base = [x.clone() for x in t["cache"]]
    alone = [x.clone() for x in _run_layer(t)]
    torch.cuda.synchronize()
    for _ in range(5):
        for x, b in zip((*s["cache"], *t["cache"]), (*start, *base)):
            x.copy_(b)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            one = _run_layer(s)
        with torch.cuda.stream(other):
            two = _run_layer(t)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(one, want))
        assert all(torch.equal(a, b) for a, b in zip(two, alone))
    ops.device_status()


def test_front_end_refusals(cuda_device):
    x = torch.zeros((4, 64), dtype=BF16, device=cuda_device)
    codes, scales = ops_q8.quantize_tokens(x)
    with pytest.raises(ValueError, match="bfloat16"):
        ops_q8.quantize_tokens(x.float())
    with pytest.raises(ValueError, match="unit stride"):
        ops_q8.quantize_tokens(x.t())
    with pytest.raises(ValueError, match="residual"):
        ops_q8.rms_norm_quantize(x, residual=x[:2])
    with pytest.raises(ValueError, match="give one"):
        ops_q8.rms_norm_quantize(x, hidden=x)
    with pytest.raises(ValueError, match="weight"):
        ops_q8.rms_norm_quantize(x, x[0, :32])
    with pytest.raises(RuntimeError, match="dim"):
        ops_q8.quantize_tokens(x[:, :60].contiguous())
    with pytest.raises(ValueError, match="int8"):
        ops_q8.linear_int8(codes.view(torch.float8_e4m3fn), scales, codes, scales)
    with pytest.raises(ValueError, match="input width"):
        ops_q8.linear_int8(codes, scales, codes[:, :32], scales)
    with pytest.raises(ValueError, match="scales"):
        ops_q8.linear_int8(codes, scales[:3].contiguous(), codes, scales)
    with pytest.raises(ValueError, match="out"):
        ops_q8.linear_int8(codes, scales, codes[:, :], scales, out=x)
    cache = ops_q8.new_kv_cache(4, 2, 64, block_tokens=16)
    table = torch.zeros((2, 2), dtype=torch.int32, device=cuda_device)
    lengths = torch.zeros(2, dtype=torch.int32, device=cuda_device)
    k = torch.zeros((4, 2, 64), dtype=BF16, device=cuda_device)
    with pytest.raises(ValueError, match="divide"):
        ops_q8.kv_cache_write(cache, k[:3], k[:3], table, lengths)
    with pytest.raises(ValueError, match="int32"):
        ops_q8.kv_cache_write(cache, k, k, table.long(), lengths)
    with pytest.raises(ValueError, match="heads"):
        ops_q8.kv_cache_write(cache, k[:, :, :32], k[:, :, :32], table, lengths)
    with pytest.raises(ValueError, match="rows"):
        ops_q8.kv_cache_write(cache, k[:, :1], k[:, :1], table, lengths)
    with pytest.raises(ValueError, match="token_starts"):
        ops_q8.kv_cache_attention(k, cache, table, lengths, lengths)
    with pytest.raises(ValueError, match="query heads"):
        ops_q8.kv_cache_attention(k[:, :1].repeat(1, 3, 1), cache, table, lengths)
    with pytest.raises(RuntimeError, match="scale"):
        ops_q8.kv_cache_attention(k, cache, table, lengths, scale=-1.0)
    # nothing to do is done
    assert ops_q8.quantize_tokens(x[:0])[0].shape == (0, 64)
    assert ops_q8.linear_int8(codes[:0], scales[:0], codes, scales).shape == (0, 4)
    assert ops_q8.kv_cache_attention(k[:0], cache, table, lengths).shape == (0, 2, 64)
    ops_q8.kv_cache_write(cache, k[:0], k[:0], table, lengths)
    assert ops_q8.kv_cache_read(cache, table, lengths, 0)[0].shape == (2, 0, 2, 64)
    assert not ops_q8.kv_cache_attention(k, cache, table, lengths).any()
    ops.device_status()


@pytest.mark.parametrize("new", [[1, 1], [40, 25]])
def test_rows_in_front_and_a_table_of_a_wider_one(cuda_device, new):
    held, heads, group = [120, 70], 2, 3
    cpu, cache, table = _cache(2, 130, heads, 128, 32, E4M3, 31, cuda_device)
    wide = torch.full((2, table.shape[1] + 5), -7, dtype=torch.int32, device=cuda_device)
    wide[:, 2 : 2 + table.shape[1]] = table.to(cuda_device)
    view = wide[:, 2 : 2 + table.shape[1]]
    rows, front = sum(new), 4
    q = _normal((front + rows + 2, heads * group, 128), 32)
    starts = torch.tensor([front, front + new[0], front + rows], dtype=torch.int32, device=cuda_device)
    lengths = torch.tensor(held, dtype=torch.int32, device=cuda_device)
    out = torch.full(q.shape, 9.0, dtype=BF16, device=cuda_device)
    ops_q8.kv_cache_attention(q.to(cuda_device), cache, view, lengths, starts, out=out)
    ops.device_status()
    assert bool((out[:front] == 9).all()) and bool((out[front + rows:] == 9).all())
    _check_attention(out[front : front + rows].cpu(), *ref.attention(
        q[front : front + rows], *cpu, table, lengths.cpu(), (starts - front).cpu()))
    k = _normal((front + rows, heads, 128), 33)
    at = torch.tensor([10, 3], dtype=torch.int32, device=cuda_device)
    ops_q8.kv_cache_write(cache, k.to(cuda_device), k.to(cuda_device), view, at, starts)
    codes, scales = ref.cache_write(cpu.k_codes, cpu.k_scales, k, table, at.cpu(), starts.cpu())
    assert torch.equal(cache.k_scales.cpu(), scales) and _same(cache.k_codes, codes)
    ops.device_status()


def test_leading_dimensions_and_launch_log(cuda_device):
    x = _normal((2, 5, 128), 41).to(cuda_device)
    w = _normal((64, 128), 42).to(cuda_device)
    wq = ops_q8.quantize_tokens(w)
    log = ops.LaunchLog()
    ops.set_launch_log(log)
    try:
        codes, scales, hidden = ops_q8.rms_norm_quantize(x)
        y = ops_q8.linear_int8(codes, scales, *wq)
    finally:
        ops.set_launch_log(None)
    torch.cuda.synchronize()
    assert hidden is x and y.shape == (2, 5, 64)
    assert [r[0] for r in log.records] == ["rms_norm_quantize", "linear_int8"]
    flat = ops_q8.rms_norm_quantize(x.view(10, 128))
    assert torch.equal(y.view(10, 64), ops_q8.linear_int8(*flat[:2], *wq))
