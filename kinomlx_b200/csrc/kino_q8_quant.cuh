// Quantising kernels of the 8-bit serving path: token rows (with the residual's addition and the
// RMS norm in front), the K/V cache as it is written, and the cache back to bf16.
#pragma once
#include "kino_q8_common.cuh"

namespace kino {

__device__ __forceinline__ void q8_unpack8(const uint4& raw, float (&f)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = unpack_bf16x2(w[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}

// ---------------------------------------------------------------- token rows
// One CTA a row: h = bf16(x + residual), y = h * rsqrt(mean h^2 + eps) * (weight + offset), then
// codes and a scale for the row. The row's common factor r = rsqrt(..) cancels in the codes,
// y top / amax(y) = p top / amax(p) with p = h * (weight + offset), so the sum of squares and the
// largest |p| come from one reduction and r only enters the scale. The row is read once and stays
// in registers: 2 bytes of x, 2 of the residual in, 2 of the sum out and 1 of code per element;
// bound by HBM. The statistics are taken from the rounded sum, which is what the next layer reads,
// so that the fused form equals an addition followed by the norm. (p is exact for bf16 weights
// without an offset.)
constexpr int Q8_ROW_MAX_THREADS = 512;

struct Q8RowArgs {
  const __nv_bfloat16* x;
  int64_t ldx;
  const __nv_bfloat16* residual;  // or null
  int64_t ld_residual;
  const __nv_bfloat16* weight;  // or null
  float weight_offset;
  float eps;
  int norm;
  __nv_bfloat16* hidden;  // or null
  int64_t ld_hidden;
  uint8_t* codes;  // contiguous rows
  float* scales;
  int dim;
};

// Values c of a row in a second pass: the sum that the first one stored (each thread reads back what
// it wrote; x or the residual may be gone under it), or x, and the residual to it, once more.
__device__ __forceinline__ void q8_row_again(const Q8RowArgs& a, int64_t row, int c, float (&v)[8]) {
  if (a.hidden != nullptr) {
    q8_unpack8(reinterpret_cast<const uint4*>(a.hidden + row * a.ld_hidden)[c], v);
    return;
  }
  q8_unpack8(reinterpret_cast<const uint4*>(a.x + row * a.ldx)[c], v);
  if (a.residual != nullptr) {
    float r[8];
    q8_unpack8(reinterpret_cast<const uint4*>(a.residual + row * a.ld_residual)[c], r);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = bf16_round(v[j] + r[j]);
  }
}

// The scale of a normed row, and the factor of its codes, from the sum of squares and the largest
// |p|; false where fp32 cannot give them (the same in all threads): squares or products that left
// its range, or so small that they lost bits. (A term's error is at most 2^-126, so the mean is
// right to 2^-26 from 2^-100 on. Products below 2^-126 have lost bits too, which counts only if the
// root brings the scale back to 2^-126.)
template <int FMT>
__device__ __forceinline__ bool q8_norm_scale(const Q8RowArgs& a, float sum, uint32_t top,
                                              float& scale, Q8Factor& f) {
  const float mean = sum / static_cast<float>(a.dim) + a.eps;
  if (!(mean >= 7.888609e-31f && mean < INFINITY) || top >= 0x7F800000u) return false;
  const float root = rsqrtf(mean);
  if (scale > 0.0f) {
    f = q8_quotient(q8_top<FMT>(), __uint_as_float(top));
    scale *= root;
    if (scale < Q8_LEAST_SCALE) scale = 0.0f;
    return true;
  }
  return (__uint_as_float(top) + 1.401298e-45f) * root < Q8_LEAST_SCALE;
}

// Such a row once more in 64 bits, by the whole CTA. Values of 1e20 and more (their squares pass
// fp32's range), weights that carry h * w out of it, or values below 1e-15 with a smaller eps: no
// path of a model in working order, so nothing here is tuned.
template <int FMT>
__device__ __noinline__ void q8_norm_row_far(const Q8RowArgs& a, int64_t row) {
  __shared__ double s_sum[16], s_max[16];
  __shared__ int s_bad;
  const int nvec = a.dim >> 3;
  auto both = [&](const __nv_bfloat16* at, int i) {
    return unpack_bf16x2(*reinterpret_cast<const uint32_t*>(at + i));
  };
  // values i, i + 1 of the row (as in q8_row_again), and times their weights
  auto values = [&](int i) {
    if (a.hidden != nullptr) return both(a.hidden + row * a.ld_hidden, i);
    float2 h = both(a.x + row * a.ldx, i);
    if (a.residual != nullptr) {
      const float2 r = both(a.residual + row * a.ld_residual, i);
      h = make_float2(bf16_round(h.x + r.x), bf16_round(h.y + r.y));
    }
    return h;
  };
  auto product = [&](float h, float w) {
    return a.weight == nullptr ? static_cast<double>(h) : static_cast<double>(h) * (w + a.weight_offset);
  };
  auto weights = [&](int i) { return a.weight == nullptr ? make_float2(0.0f, 0.0f) : both(a.weight, i); };
  double sum = 0.0, top = 0.0;
  bool bad = false;
#pragma unroll 1
  for (int c = threadIdx.x; c < nvec; c += blockDim.x)
#pragma unroll 1
    for (int i = 8 * c; i < 8 * c + 8; i += 2) {
      const float2 h = values(i), w = weights(i);
      const double p = product(h.x, w.x), q = product(h.y, w.y);
      sum += static_cast<double>(h.x) * h.x + static_cast<double>(h.y) * h.y;
      bad = bad || !isfinite(p) || !isfinite(q);
      top = fmax(top, fmax(fabs(p), fabs(q)));
    }
#pragma unroll 1
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if (threadIdx.x == 0) s_bad = 0;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
    s_sum[threadIdx.x >> 5] = sum;
    s_max[threadIdx.x >> 5] = top;
  }
  if (bad) s_bad = 1;
  __syncthreads();
  sum = top = 0.0;
#pragma unroll 1
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) {
    sum += s_sum[i];
    top = fmax(top, s_max[i]);
  }
  float scale = 0.0f;
  if (s_bad) {
    scale = __uint_as_float(0x7FC00000u);
  } else if (top > 0.0) {
    scale = static_cast<float>(top / (q8_top<FMT>() * sqrt(sum / a.dim + a.eps)));
    if (scale < Q8_LEAST_SCALE) scale = 0.0f;
    if (isinf(scale)) scale = __uint_as_float(0x7FC00000u);  // so is the row's largest value
  }
  if (threadIdx.x == 0) a.scales[row] = scale;
  const double factor = scale > 0.0f ? q8_top<FMT>() / top : 0.0;
#pragma unroll 1
  for (int c = threadIdx.x; c < nvec; c += blockDim.x)
#pragma unroll 1
    for (int i = 8 * c; i < 8 * c + 8; i += 2) {
      uint32_t codes = 0;
      if (scale > 0.0f) {
        const float2 h = values(i), w = weights(i);
        codes = q8_encode4<FMT>(static_cast<float>(product(h.x, w.x) * factor),
                                static_cast<float>(product(h.y, w.y) * factor), 0.0f, 0.0f);
      }
      *reinterpret_cast<uint16_t*>(a.codes + row * a.dim + i) = static_cast<uint16_t>(codes);
    }
}

template <int FMT, int NV>
__global__ void __launch_bounds__(Q8_ROW_MAX_THREADS) q8_rows_kernel(const __grid_constant__ Q8RowArgs a) {
  griddep_wait();
  griddep_launch();
  __shared__ float s_sum[16];
  __shared__ uint32_t s_max[16];
  const int64_t row = blockIdx.x;
  const int warps = blockDim.x >> 5;
  const int nvec = a.dim >> 3;
  const uint4* xr = reinterpret_cast<const uint4*>(a.x + row * a.ldx);
  uint4 raw[NV], rres[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    raw[i] = c < nvec ? __ldcs(xr + c) : make_uint4(0, 0, 0, 0);
  }
  if (a.residual != nullptr) {
    const uint4* rr = reinterpret_cast<const uint4*>(a.residual + row * a.ld_residual);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      rres[i] = c < nvec ? __ldcs(rr + c) : make_uint4(0, 0, 0, 0);
    }
  }
  float v[NV][8];
  float sum = 0.0f;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    q8_unpack8(raw[i], v[i]);
    if (a.residual != nullptr) {
      float r[8];
      q8_unpack8(rres[i], r);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = bf16_round(v[i][j] + r[j]);
    }
    if (a.hidden != nullptr && c < nvec)
      reinterpret_cast<uint4*>(a.hidden + row * a.ld_hidden)[c] =
          make_uint4(pack_bf16x2(v[i][0], v[i][1]), pack_bf16x2(v[i][2], v[i][3]),
                     pack_bf16x2(v[i][4], v[i][5]), pack_bf16x2(v[i][6], v[i][7]));
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(v[i][j], v[i][j], sum);
    if (a.weight != nullptr && c < nvec) {
      float w[8];
      q8_unpack8(__ldg(reinterpret_cast<const uint4*>(a.weight) + c), w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] *= w[j] + a.weight_offset;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, abs_bits(v[i][j]));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (a.norm) sum = warp_sum_f(sum);
  if (warps > 1) {
    if ((threadIdx.x & 31) == 0) {
      s_sum[threadIdx.x >> 5] = sum;
      s_max[threadIdx.x >> 5] = top;
    }
    __syncthreads();
    const int w = threadIdx.x & 31;
    top = __reduce_max_sync(0xffffffffu, w < warps ? s_max[w] : 0u);
    if (a.norm) sum = warp_sum_f(w < warps ? s_sum[w] : 0.0f);
  }
  float scale = q8_scale<FMT>(top);
  Q8Factor f = {0.0f, 0.0f};
  if (a.norm) {
    if (__builtin_expect(!q8_norm_scale<FMT>(a, sum, top, scale, f), 0)) {
      q8_norm_row_far<FMT>(a, row);
      return;
    }
  } else if (scale > 0.0f) {
    f = q8_quotient(q8_top<FMT>(), __uint_as_float(top));
  }
  if (threadIdx.x == 0) a.scales[row] = scale;
  uint2* cr = reinterpret_cast<uint2*>(a.codes + row * a.dim);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (c < nvec)
      cr[c] = !(scale > 0.0f)
                  ? make_uint2(0u, 0u)
                  : make_uint2(q8_encode4<FMT>(f.times(v[i][0]), f.times(v[i][1]),
                                               f.times(v[i][2]), f.times(v[i][3])),
                               q8_encode4<FMT>(f.times(v[i][4]), f.times(v[i][5]),
                                               f.times(v[i][6]), f.times(v[i][7])));
  }
}

// The same for rows that do not fit the registers of a CTA: two passes over the row. (Four CTAs on
// an SM: 2048 x 28672 with a residual 82 us, with three, as the registers of the rare 64-bit rows
// would have it, 88.)
template <int FMT>
__global__ void __launch_bounds__(Q8_ROW_MAX_THREADS, 4) q8_wide_rows_kernel(const __grid_constant__ Q8RowArgs a) {
  griddep_wait();
  griddep_launch();
  __shared__ float s_sum[16];
  __shared__ uint32_t s_max[16];
  const int64_t row = blockIdx.x;
  const int nvec = a.dim >> 3;
  const uint4* xr = reinterpret_cast<const uint4*>(a.x + row * a.ldx);
  uint4* hr = reinterpret_cast<uint4*>(a.hidden + row * a.ld_hidden);
  auto weighted = [&](float (&v)[8], int c) {
    if (a.weight == nullptr) return;
    float w[8];
    q8_unpack8(__ldg(reinterpret_cast<const uint4*>(a.weight) + c), w);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= w[j] + a.weight_offset;
  };
  float sum = 0.0f;
  uint32_t top = 0;
  for (int c = threadIdx.x; c < nvec; c += Q8_ROW_MAX_THREADS) {
    float v[8];
    q8_unpack8(xr[c], v);
    if (a.residual != nullptr) {
      float r[8];
      q8_unpack8(reinterpret_cast<const uint4*>(a.residual + row * a.ld_residual)[c], r);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = bf16_round(v[j] + r[j]);
    }
    if (a.hidden != nullptr)
      hr[c] = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                         pack_bf16x2(v[6], v[7]));
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(v[j], v[j], sum);
    weighted(v, c);
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, abs_bits(v[j]));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  sum = warp_sum_f(sum);
  if ((threadIdx.x & 31) == 0) {
    s_sum[threadIdx.x >> 5] = sum;
    s_max[threadIdx.x >> 5] = top;
  }
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, s_max[threadIdx.x & 15]);
  sum = warp_sum_f((threadIdx.x & 31) < 16 ? s_sum[threadIdx.x & 15] : 0.0f);
  float scale = q8_scale<FMT>(top);
  Q8Factor f = {0.0f, 0.0f};
  if (a.norm) {
    if (__builtin_expect(!q8_norm_scale<FMT>(a, sum, top, scale, f), 0)) {
      q8_norm_row_far<FMT>(a, row);
      return;
    }
  } else if (scale > 0.0f) {
    f = q8_quotient(q8_top<FMT>(), __uint_as_float(top));
  }
  if (threadIdx.x == 0) a.scales[row] = scale;
  uint2* cr = reinterpret_cast<uint2*>(a.codes + row * a.dim);
  for (int c = threadIdx.x; c < nvec; c += Q8_ROW_MAX_THREADS) {
    float v[8];
    q8_row_again(a, row, c, v);
    weighted(v, c);
    cr[c] = !(scale > 0.0f) ? make_uint2(0u, 0u)
                            : make_uint2(q8_encode4<FMT>(f.times(v[0]), f.times(v[1]),
                                                         f.times(v[2]), f.times(v[3])),
                                         q8_encode4<FMT>(f.times(v[4]), f.times(v[5]),
                                                         f.times(v[6]), f.times(v[7])));
  }
}

// ---------------------------------------------------------------- cache write
// Codes live as (block, head, slot, dim): the tokens of one block and head are contiguous, which
// is the unit every kernel here reads. Sequence b's new tokens take positions lengths[b] on.
//
// One CTA per (cache block that gets new tokens, head), K and V together (blocks of 128 tokens of
// 128-wide heads: one of them). The new tokens' values stay in registers between the maximum and
// the rounding. The values are asked for once the block is known, after two dependent reads (lengths
// and starts, then the table) that K and V share; several heads in turn in a CTA were slower (fewer
// loads in flight). A block that holds earlier tokens keeps the larger of its scale and the new
// tokens': where it grows, the earlier codes are rounded again to the new scale (at most a half
// step of the new scale each time).
constexpr int Q8_WRITE_THREADS = 128;

struct Q8WriteArgs {
  const __nv_bfloat16* x[2];  // k, v
  int64_t ld[2], head_stride[2];
  uint8_t* codes[2];
  float* scales[2];
  const int32_t* table;
  int64_t ld_table;
  int table_blocks;
  const int32_t* lengths;  // tokens held before this call
  Q8Rows rows;
  int batch, heads, dim, block, num_blocks;
  int block_shift;  // log2(block)
};

// The item-th cache block that gets new tokens, in order of sequences; false past the last one.
// The same scan in every thread of a warp: each lane counts one sequence's blocks.
__device__ __forceinline__ bool q8_write_item(const Q8WriteArgs& a, int item, int& b, int& index,
                                              int& held, int64_t& first, int& count) {
  int before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    const int mine = b0 + static_cast<int>(lane_id());
    int n = 0;
    if (mine < a.batch) {
      int64_t f;
      int c;
      a.rows.of(mine, f, c);
      const int len = a.lengths[mine];
      if (len < 0) q8_flag(1);
      if (c > 0 && len >= 0) {
        const int last = static_cast<int>((static_cast<int64_t>(len) + c - 1) >> a.block_shift);
        n = last - (len >> a.block_shift) + 1;
      }
    }
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, upto, o);
      if (static_cast<int>(lane_id()) >= o) upto += up;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + upto > item);
    if (hit != 0) {
      const int l = __ffs(hit) - 1;
      b = b0 + l;
      const int skipped = before + __shfl_sync(0xffffffffu, upto - n, l);
      held = a.lengths[b];
      a.rows.of(b, first, count);
      index = (held >> a.block_shift) + (item - skipped);
      return true;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}

template <int FMT, int NV, int KV>
__global__ void __launch_bounds__(Q8_WRITE_THREADS) q8_cache_write_kernel(const Q8WriteArgs a) {
  griddep_wait();
  griddep_launch();
  __shared__ uint32_t s_max[KV][Q8_WRITE_THREADS / 32];
  int b, index, held, count;
  int64_t first;
  // (heads are neighbours in the grid as they are in a token's row)
  const int head = blockIdx.x % a.heads, kv0 = KV == 2 ? 0 : blockIdx.y;
  if (!q8_write_item(a, blockIdx.x / a.heads, b, index, held, first, count)) return;
  const int page = index < a.table_blocks ? a.table[b * a.ld_table + index] : -1;
  if (page < 0 || page >= a.num_blocks) {  // past the table, or no block of this cache
    if (threadIdx.x == 0) q8_flag(1);
    return;
  }
  const int64_t unit = static_cast<int64_t>(page) * a.heads + head;
  const int chunk_bits = a.dim == 128 ? 4 : 3;  // 8-value chunks of a token: 8 or 16
  const int64_t at0 = static_cast<int64_t>(index) << a.block_shift;  // position of slot 0
  const bool earlier = held > at0;
  // slots [fresh0, fresh1) get new tokens, those before fresh0 hold earlier ones
  const int fresh0 = earlier ? static_cast<int>(held - at0) : 0;
  const int fresh1 = static_cast<int>(min(static_cast<int64_t>(a.block), held + static_cast<int64_t>(count) - at0));
  const int64_t row0 = first + at0 - held;  // of slot 0
  uint4 raw[KV][NV];
#pragma unroll
  for (int kv = 0; kv < KV; ++kv) {
    const __nv_bfloat16* src = a.x[kv0 + kv] + head * a.head_stride[kv0 + kv];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = threadIdx.x + i * Q8_WRITE_THREADS;
      const int slot = e >> chunk_bits, c = e & ((1 << chunk_bits) - 1);
      raw[kv][i] = make_uint4(0, 0, 0, 0);
      if (slot >= fresh0 && slot < fresh1)
        raw[kv][i] = __ldcs(reinterpret_cast<const uint4*>(src + (row0 + slot) * a.ld[kv0 + kv]) + c);
    }
  }
  float before[KV];
#pragma unroll
  for (int kv = 0; kv < KV; ++kv) {
    before[kv] = earlier ? a.scales[kv0 + kv][unit] : 0.0f;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t w[4] = {raw[kv][i].x, raw[kv][i].y, raw[kv][i].z, raw[kv][i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        top = max(top, max((w[j] & 0x7FFFu) << 16, w[j] & 0x7FFF0000u));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) s_max[kv][threadIdx.x >> 5] = top;
  }
  __syncthreads();  // (every thread has read the old scales too)
#pragma unroll
  for (int kv = 0; kv < KV; ++kv) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < Q8_WRITE_THREADS / 32; ++i) top = max(top, s_max[kv][i]);
    const float own = q8_scale<FMT>(top), old_scale = before[kv];
    // the larger of the two; NaN wins
    const float scale = old_scale > own ? old_scale : old_scale == old_scale ? own : old_scale;
    Q8Factor f = {0.0f, 0.0f}, again = {0.0f, 0.0f};
    if (scale > 0.0f) {
      if (scale > old_scale) {  // the new tokens' own
        f = q8_quotient(q8_top<FMT>(), __uint_as_float(top));
        again.hi = old_scale * f.hi;  // what the earlier codes are multiplied by
        again.lo = fmaf(old_scale, f.hi, -again.hi) + old_scale * f.lo;
      } else {
        f = q8_quotient(1.0f, old_scale);
      }
    }
    if (threadIdx.x == 0) a.scales[kv0 + kv][unit] = scale;
    const bool grown = scale > old_scale;
    uint2* codes = reinterpret_cast<uint2*>(a.codes[kv0 + kv] + unit * a.block * a.dim);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = threadIdx.x + i * Q8_WRITE_THREADS;
      const int slot = e >> chunk_bits;
      float v[8];
      if (slot >= fresh0 && slot < fresh1) {
        q8_unpack8(raw[kv][i], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = f.times(v[j]);
      } else if (grown && slot < fresh0) {
        const uint2 old = codes[e];
        float lo[4], hi[4];
        q8_decode4<FMT>(old.x, lo);
        q8_decode4<FMT>(old.y, hi);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = again.times(lo[j]);
          v[4 + j] = again.times(hi[j]);
        }
      } else {
        continue;
      }
      codes[e] = !(scale > 0.0f) ? make_uint2(0u, 0u)
                                 : make_uint2(q8_encode4<FMT>(v[0], v[1], v[2], v[3]),
                                              q8_encode4<FMT>(v[4], v[5], v[6], v[7]));
    }
  }
}

// ---------------------------------------------------------------- cache read
// The tokens [0, tokens) of every sequence as (batch, tokens, heads, dim) bf16, zeros past a
// sequence's length: one thread takes 16 codes of K and of V (one scale each) and writes two
// 32-byte runs; threads follow the output, so stores are contiguous and a head's 64 or 128 codes
// are read as whole lines. 1 byte in, 2 out per value, bound by HBM.
struct Q8ReadArgs {
  const uint8_t* codes[2];
  const float* scales[2];
  __nv_bfloat16* out[2];  // contiguous
  const int32_t* table;
  int64_t ld_table;
  int table_blocks;
  const int32_t* lengths;
  int64_t tokens;
  int heads, dim, block, num_blocks;
  int block_shift;  // log2(block)
};

template <int FMT>
__global__ void __launch_bounds__(256) q8_cache_read_kernel(const Q8ReadArgs a) {
  griddep_wait();
  griddep_launch();
  const int b = blockIdx.y;
  // (tokens * heads * dim / 16 fits 31 bits: 64-bit divisions would cost more than the copy)
  const int chunk_bits = a.dim == 128 ? 3 : 2;
  const uint32_t e = blockIdx.x * 256u + threadIdx.x;
  const uint32_t per_token = static_cast<uint32_t>(a.heads) << chunk_bits;
  const uint32_t token = e / per_token;
  if (token >= a.tokens) return;
  const int64_t t = token;
  const int rest = static_cast<int>(e - token * per_token);
  const int head = rest >> chunk_bits, c = rest & ((1 << chunk_bits) - 1);
  const int64_t capacity = static_cast<int64_t>(a.table_blocks) * a.block;
  const int64_t length = a.lengths[b];
  if (length < 0 || length > capacity) q8_flag(1);
  int page = -1;
  if (t < length && t < capacity) {
    page = a.table[b * a.ld_table + (t >> a.block_shift)];
    if (page < 0 || page >= a.num_blocks) {
      q8_flag(1);
      page = -1;
    }
  }
  const int64_t dst = ((b * a.tokens + t) * a.heads + head) * a.dim + c * 16;
  uint4 raw[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  float scale[2] = {0.0f, 0.0f};
  if (page >= 0) {
    const int64_t unit = static_cast<int64_t>(page) * a.heads + head;
    const int64_t src = (unit * a.block + (t & (a.block - 1))) * a.dim + c * 16;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      raw[kv] = __ldcs(reinterpret_cast<const uint4*>(a.codes[kv] + src));
      scale[kv] = a.scales[kv][unit];
    }
  }
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const uint32_t w[4] = {raw[kv].x, raw[kv].y, raw[kv].z, raw[kv].w};
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f[4];
      q8_decode4<FMT>(w[i], f);
      o[2 * i] = pack_bf16x2(f[0] * scale[kv], f[1] * scale[kv]);
      o[2 * i + 1] = pack_bf16x2(f[2] * scale[kv], f[3] * scale[kv]);
    }
    store_16(a.out[kv] + dst, o);
  }
}

}  // namespace kino
