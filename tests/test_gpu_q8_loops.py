"""The 8-bit serving kernels where a CTA takes many units of work: rings that wrap several times,
items that end inside a run and runs that end inside items, whole items of several blocks, output
tiles behind one another. (Small cases give every CTA a single step, so that a fault in what is
carried from one step to the next would pass them.)"""

from __future__ import annotations

import pytest
import torch

import test_gpu_q8 as small
from kinomlx_b200 import ops, ops_q8
from oracle import serving_q8 as ref

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
INT8, E4M3 = torch.int8, torch.float8_e4m3fn


def _sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def _cache(held, heads, dim, block, dtype, seed, device):
    """Random codes and scales; K scales grow threefold along every sequence, so that maxima move
    in late blocks too."""
    g = torch.Generator(device).manual_seed(seed)
    per = [-(-h // block) for h in held]
    order = torch.randperm(sum(per) + 1, generator=g, device=device).to(torch.int32)
    table = torch.full((len(held), max(per)), -1, dtype=torch.int32, device=device)
    codes = [torch.randint(-127, 128, (len(order), heads, block, dim), generator=g, device=device,
                           dtype=INT8) for _ in range(2)]
    if dtype == E4M3:
        codes = [(c.to(BF16) * 3.5).to(E4M3) for c in codes]
    scales = [(torch.rand((len(order), heads), generator=g, device=device) + 0.5) * 0.02
              for _ in range(2)]
    if dtype == E4M3:
        scales = [s / 3.5 for s in scales]
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at : at + n]
        at += n
        scales[0][table[b, :n].long()] *= torch.linspace(1, 3, n, device=device)[:, None] if n else 1
    return ops_q8.KVCache(*codes, *scales), table


def _units(held, new, heads, tokens, width, causal):
    """Units of `width` keys that the items of `tokens` query tokens come to."""
    total = 0
    for length, n in zip(held, new):
        for t in range(-(-n // tokens)):
            keys = max(0, length - n + min(n, (t + 1) * tokens)) if causal else length
            total += max(1, -(-keys // width)) * heads
    return total


def _limit(want, weight, reach, crowd):
    """Weights in f16 2^-11 (2^-25 below 2^-14, against a largest of at least 1: `crowd`); scores by
    at most (dim + 4) * 2^-24 of their sum of magnitudes and exponentials 2^-20, numerator and
    denominator; sums 2^-24 an addition, 2^-23 in the tensor cores, where at most 320 additions
    follow one another here: eight for each of an item's up to 32 blocks of 128 keys, or one for
    each of a run's up to 63 units of 64, twelve warps, and the pieces of an item; the result's
    bf16 2^-8."""
    dim = want.shape[-1]
    inner = ((2.0**-11 + 2 * ((dim + 4) * 2.0**-24 * reach + 2.0**-20) + 3 * 320 * 2.0**-24)
             * weight + 2.0**-25 * crowd)
    return inner + 2.0**-8 * (want.abs() + inner) + 1e-30


def _attend(held, new, heads, group, dim, block, dtype, causal, device):
    cache, table = _cache(held, heads, dim, block, dtype, dim + block, device)
    g = torch.Generator(device).manual_seed(group)
    q = (torch.randn((sum(new), heads * group, dim), generator=g, device=device) * 2).to(BF16)
    starts = torch.tensor([0] + [sum(new[: i + 1]) for i in range(len(new))], dtype=torch.int32,
                          device=device)
    lengths = torch.tensor(held, dtype=torch.int32, device=device)
    args = (q, cache, table, lengths, starts)
    # peaked, so that maxima move, and nearly flat, so that every unit counts
    for scale in (None, 0.01):
        got = ops_q8.kv_cache_attention(*args, causal=causal, scale=scale)
        ops.device_status()
        want, *parts = ref.attention_by_products(q, *cache, table, lengths, starts, causal=causal,
                                                 scale=scale)
        off, limit = (got.double() - want).abs(), _limit(want, *parts)
        assert got.isfinite().all()
        assert bool((off <= limit).all()), float((off / limit).max())
        for _ in range(3):  # the same bits each time
            assert torch.equal(ops_q8.kv_cache_attention(*args, causal=causal, scale=scale), got)
        ops.device_status()


FORMS = [(128, 64, INT8), (128, 16, E4M3), (64, 128, INT8), (64, 32, E4M3), (128, 128, INT8)]


@pytest.mark.parametrize(("dim", "block", "dtype"), FORMS)
@pytest.mark.parametrize(("group", "new", "tiles"), [
    (4, [1] * 8, 1), (8, [1] * 8, 1), (8, [2] * 8, 2), (3, [7, 1, 3, 2, 4, 1, 6, 2], 2),
])
def test_attention_few_rows_many_units(cuda_device, dim, block, dtype, group, new, tiles):
    held, heads = [20000, 900, 15000, 130, 0, 9000, 4000, 700], 8
    units = _units(held, new, heads, 8 * tiles // group, 64, True)
    stages = (9 if tiles == 1 else 8) * (1 if dim == 128 else 2)
    assert 2 * stages < -(-units // _sms()) <= 63  # the ring of loads wraps twice
    _attend(held, new, heads, group, dim, block, dtype, True, cuda_device)


@pytest.mark.parametrize(("dim", "block", "dtype", "causal", "group"), [
    (128, 64, INT8, True, 4), (128, 16, E4M3, True, 1), (64, 128, INT8, True, 7),
    (64, 32, E4M3, False, 4), (128, 128, E4M3, False, 1), (64, 16, INT8, True, 1),
    (128, 32, INT8, True, 48),
])
def test_attention_many_rows_many_units(cuda_device, dim, block, dtype, causal, group):
    held, new, heads = [4000, 700, 0, 2500, 300, 1500], [600, 300, 20, 130, 290, 40], 8
    units = _units(held, new, heads, 4 * (128 // group), 128, causal)
    assert max(held) <= 32 * 128
    assert -(-units // (_sms() // 2)) > 8  # four stages, wrapped twice, over many items
    _attend(held, new, heads, group, dim, block, dtype, causal, cuda_device)


@pytest.mark.parametrize(("m", "n", "k"), [
    (2100, 6408, 272),   # CTA pairs, three or four tiles each, ragged both ways
    (2100, 6408, 912),   # eight blocks of K on six stages, carried over tiles
    (4361, 2056, 144),
    (512, 4104, 1040),   # 64 tokens a tile, four stages
    (384, 5632, 1040),   # 128 tokens a tile, three stages
    (100, 33800, 656),   # the same, the weight's tiles more than fit at once
    (48, 8200, 2064),    # 16 tokens a tile
    (40, 19000, 784),    # 32 or more
])
@pytest.mark.parametrize("bias", [False, True])
def test_linear_int8_many_steps(cuda_device, m, n, k, bias):
    args, exact = small._product(m, n, k, m + n + k, bias, cuda_device)
    out = ops_q8.linear_int8(*args)
    small._check_product(out, exact, args[4])
    assert torch.equal(ops_q8.linear_int8(*args), out)
    ops.device_status()


# ---------------------------------------------------------------- the tcgen05 attention at its edges
# (the same checks with 70 rows a cache head, which that kernel takes)
def test_many_rows_zero_values_and_empty(cuda_device):
    small.test_attention_zero_values_and_empty(cuda_device, 70)


@pytest.mark.parametrize("dtype", [INT8, E4M3])
def test_many_rows_not_finite_in_masked_places(cuda_device, dtype):
    small.test_attention_not_finite_in_masked_places(cuda_device, dtype, 70)


def test_many_rows_sizes_that_do_not_fit(cuda_device):
    small.test_sizes_that_do_not_fit_are_skipped_and_reported(cuda_device, 70)


def test_many_rows_strides_and_in_place(cuda_device):
    small.test_attention_strides_and_in_place(cuda_device, 70)


def test_many_rows_streams_and_graphs(cuda_device):
    """Two layers whose attention has 90 and 100 rows a cache head: by themselves, in two graphs
    replayed in turn, and at once on two streams."""
    layers = [small._layer(INT8, 51, cuda_device, 4, 45, 300), small._layer(E4M3, 52, cuda_device, 3, 50, 150)]
    start = [[t.clone() for t in s["cache"]] for s in layers]

    def restore():
        for s, b in zip(layers, start):
            for x, y in zip(s["cache"], b):
                x.copy_(y)
        torch.cuda.synchronize()

    want = [[t.clone() for t in small._run_layer(s)] for s in layers]
    restore()
    streams, graphs = [torch.cuda.Stream() for _ in layers], []
    for s, stream in zip(layers, streams):
        with torch.cuda.stream(stream):
            small._run_layer(s)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            result = small._run_layer(s)
        graphs.append((graph, result))
    for _ in range(3):
        restore()
        for (graph, result), expect in zip(graphs, want):
            for r in result:
                r.fill_(-1)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(result, expect))
    for _ in range(5):
        restore()
        results = []
        for s, stream in zip(layers, streams):
            with torch.cuda.stream(stream):
                results.append(small._run_layer(s))
        torch.cuda.synchronize()
        for got, expect in zip(results, want):
            assert all(torch.equal(a, b) for a, b in zip(got, expect))
    ops.device_status()
