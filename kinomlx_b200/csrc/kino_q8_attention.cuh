// Attention over the 8-bit K/V cache: softmax(q k^T * scale) v with k and v as codes times a scale
// for each cache block and head, fp32 scores, statistics and accumulation, G query heads on each
// K/V head.
//
// Codes are exact as bf16, so the products run on bf16 operands that are converted from the codes
// in registers; a block's K scale multiplies its columns of the scores, its V scale its columns of
// the probabilities (in fp32, before they are rounded to bf16 for the second product).
//
// Work is cut by units of BN keys of one (sequence, query tile, K/V head), the items in that
// order; every CTA of one resident wave takes an equal run of units, whatever the lengths are
// (they are only known on the device). A run that starts or ends inside an item leaves an
// unnormalised partial result with its row maxima and sums; attention_q8_combine adds the pieces
// of each cut item in a fixed order.
#pragma once
#include "kino_attention.cuh"
#include "kino_q8_common.cuh"

namespace kino {

struct Q8Attn {
  const __nv_bfloat16* q;
  int64_t ld_q, hs_q;
  __nv_bfloat16* out;
  int64_t ld_out, hs_out;
  const uint8_t* codes[2];
  const float* scales[2];
  const int32_t* table;
  int64_t ld_table;
  int table_blocks;
  const int32_t* lengths;
  Q8Rows rows;
  int batch, heads, group, block, num_blocks;
  float scale_log2;
  int causal;
  int tile_tokens;  // query tokens of an item
  int tile_rows;    // rows of its partial results (tile_tokens * group, padded)
  int least_units;  // units of a run, at least
  int runs;         // CTAs
  float* part_o;    // [2 * runs][tile_rows][D]
  float* part_ml;   // [2 * runs][tile_rows][2]: row maximum (log2 units), row sum
};

// The items and their units, as every CTA sees them.
template <int BN>
struct Q8Work {
  const Q8Attn& a;
  int b, tile, head;       // the item
  int64_t first;           // its sequence's first query row
  int count, len, tiles;   // the sequence's query tokens, keys, query tiles
  int units;               // the item's
  __device__ __forceinline__ explicit Q8Work(const Q8Attn& args) : a(args) {}

  __device__ __forceinline__ void load(int seq, int64_t& f, int& n, int& l) const {
    a.rows.of(seq, f, n);
    const int64_t capacity = static_cast<int64_t>(a.table_blocks) * a.block;
    l = a.lengths[seq];
    if (l < 0 || l > capacity) {
      q8_flag(1);
      l = l < 0 ? 0 : static_cast<int>(capacity);
    }
  }
  // Keys that the last token of a tile sees.
  __device__ __forceinline__ static int keys(const Q8Attn& a, int n, int l, int t) {
    if (!a.causal) return l;
    const int last = min(n, (t + 1) * a.tile_tokens);
    return max(0, l - n + last);
  }
  __device__ __forceinline__ static int units_of(const Q8Attn& a, int n, int l, int t) {
    return max(1, (keys(a, n, l, t) + BN - 1) / BN);  // an item without keys still writes zeros
  }
  __device__ __forceinline__ int64_t sequence_units(int seq) const {
    int64_t f;
    int n, l;
    load(seq, f, n, l);
    const int nt = (n + a.tile_tokens - 1) / a.tile_tokens;
    int64_t sum = 0;
    if (!a.causal)
      sum = static_cast<int64_t>(nt) * units_of(a, n, l, 0);
    else
      for (int t = 0; t < nt; ++t) sum += units_of(a, n, l, t);
    return sum * a.heads;
  }
  __device__ __forceinline__ void enter(int seq) {
    b = seq;
    load(seq, first, count, len);
    tiles = (count + a.tile_tokens - 1) / a.tile_tokens;
  }
  // By a whole warp: all units of the call.
  __device__ __forceinline__ int64_t total() const {
    int64_t sum = 0;
    for (int s = static_cast<int>(lane_id()); s < a.batch; s += 32) sum += sequence_units(s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
  }
  // By a whole warp: the item that holds unit u (u < total()); returns u's place inside it.
  __device__ __forceinline__ int64_t seek(int64_t u) {
    int64_t before = 0;
    int seq = 0;
    for (int s0 = 0; s0 < a.batch; s0 += 32) {
      const int mine = s0 + static_cast<int>(lane_id());
      const int64_t n = mine < a.batch ? sequence_units(mine) : 0;
      int64_t upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, upto, o);
        if (static_cast<int>(lane_id()) >= o) upto += up;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + upto > u);
      if (hit != 0) {
        const int l = __ffs(hit) - 1;
        seq = s0 + l;
        before += __shfl_sync(0xffffffffu, upto - n, l);
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    enter(seq);
    int64_t at = u - before;
    tile = 0;
    units = units_of(a, count, len, 0);
    while (at >= static_cast<int64_t>(units) * a.heads && tile + 1 < tiles) {
      at -= static_cast<int64_t>(units) * a.heads;
      ++tile;
      units = units_of(a, count, len, tile);
    }
    head = static_cast<int>(at / units);
    return at - static_cast<int64_t>(head) * units;
  }
  __device__ __forceinline__ void next() {
    if (++head < a.heads) return;
    head = 0;
    if (++tile >= tiles) {
      tile = 0;
      do {
        if (b + 1 >= a.batch) {  // past the last item: never asked for by a run inside total()
          units = 1;
          return;
        }
        enter(b + 1);
      } while (tiles == 0);
    }
    units = units_of(a, count, len, tile);
  }
};

// Units of a run.
__device__ __forceinline__ int64_t q8_run_units(const Q8Attn& a, int64_t total) {
  const int64_t even = (total + a.runs - 1) / a.runs;
  return even > a.least_units ? even : a.least_units;
}

// ---------------------------------------------------------------- few query rows
// Up to 8 NT query rows (tokens x group) an item, keys in units of 64. Bound by reading the cache:
// warp 8 brings each unit (K and V of 64 tokens, 128 D bytes) to shared memory by TMA, up to
// Q8D_STAGES units ahead; warps 0..3 and 4..7 take turns on the units, 16 keys a warp.
//
// The products use mma.sync with the keys (then the dims of V) as the 16 rows and the query rows
// as the 8 columns, so that a single decoded token with a group of up to 8 heads fills a tile;
// the tensor pipe is far from its limit here. Each lane reads 16-byte runs of codes and pairs
// them as the fragments want by choosing which dims (of K: 32 t + 4 s ..) or keys and dims (of V)
// a fragment's rows and columns stand for, so nothing is transposed but the 16 x 8
// probabilities (movmatrix).
constexpr int Q8D_BN = 64;
constexpr int Q8D_WARPS = 8;
constexpr int Q8D_THREADS = 32 * (Q8D_WARPS + 1);

template <int D, int NT>
struct Q8DecodeSmem {
  static constexpr int HALF = Q8D_BN * D;  // K or V of a unit
  static constexpr int STAGE = 2 * HALF;
  static constexpr int STAGES = D == 128 ? 8 : 16;
  static constexpr int LDO = D + 4;        // padded row of the merge buffer, in floats
  static constexpr int MERGE_OFF = STAGES * STAGE;
  static constexpr int MERGE = Q8D_WARPS * 8 * NT * LDO * 4;
  static constexpr int ML_OFF = MERGE_OFF + MERGE;      // [warp][8 NT][2]
  static constexpr int SC_OFF = ML_OFF + Q8D_WARPS * 8 * NT * 8;
  // per stage: scales of the four 16-key groups, K then V, and a word of which groups are there
  static constexpr int SC = 48;
  static constexpr int BAR_OFF = SC_OFF + STAGES * SC;
  static constexpr int TOTAL = BAR_OFF + 2 * STAGES * 8 + 64 + 1024;
};

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Byte offset of 16-byte chunk c of row r in a swizzled tile of D-byte rows.
template <int D>
__device__ __forceinline__ uint32_t q8_chunk(int r, int c) {
  return D == 128 ? static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4))
                  : static_cast<uint32_t>(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

template <int D, int NT, int FMT>
__global__ void __launch_bounds__(Q8D_THREADS, 1)
    attention_q8_decode_kernel(const __grid_constant__ CUtensorMap map_k,
                               const __grid_constant__ CUtensorMap map_v, const Q8Attn a) {
  using L = Q8DecodeSmem<D, NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t* empty = full + L::STAGES;
  int64_t* s_run = reinterpret_cast<int64_t*>(empty + L::STAGES);  // u0, u1, at
  int* s_item = reinterpret_cast<int*>(s_run + 3);                 // b, tile, head
  volatile int* abort_flag = s_item + 3;
  const int warp = warp_id();
  const int lane = static_cast<int>(lane_id());
  griddep_wait();
  griddep_launch();
  Q8Work<Q8D_BN> w(a);
  if (warp == 0) {
    const int64_t total = w.total();
    const int64_t run = q8_run_units(a, total);
    const int64_t u0 = blockIdx.x * run;
    int64_t at = 0;
    if (u0 < total) at = w.seek(u0);
    if (lane == 0) {
      s_run[0] = u0;
      s_run[1] = u0 + run < total ? u0 + run : total;
      s_run[2] = at;
      s_item[0] = w.b;
      s_item[1] = w.tile;
      s_item[2] = w.head;
      *abort_flag = 0;
    }
  } else if (warp == 1 && lane == 0) {
    for (int i = 0; i < L::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    fence_barrier_init();
  }
  __syncthreads();
  int64_t left = s_run[1] - s_run[0];
  if (left <= 0) return;
  int at = static_cast<int>(s_run[2]);
  w.enter(s_item[0]);
  w.tile = s_item[1];
  w.head = s_item[2];
  w.units = Q8Work<Q8D_BN>::units_of(a, w.count, w.len, w.tile);

  if (warp == Q8D_WARPS) {
    // ---- loads
    constexpr int PAGES = Q8D_BN / 16;  // cache blocks of a unit, at most
    const int per = a.block >= Q8D_BN ? 1 : Q8D_BN / a.block;
    const int box = a.block >= Q8D_BN ? Q8D_BN : a.block;
    int issued = 0;
    bool ok = true;
    while (left > 0 && ok) {
      const int n = static_cast<int>(left < w.units - at ? left : w.units - at);
      const int keys = Q8Work<Q8D_BN>::keys(a, w.count, w.len, w.tile);
      const int32_t* table = a.table + static_cast<int64_t>(w.b) * a.ld_table;
      // 32 / per units at a time: each lane looks up the place and scales of one load
      const int lot = 32 / per;
      for (int u = 0; u < n && ok; u += lot) {
        const int key = (at + u) * Q8D_BN + lane * box;  // this lane's first key
        int row = -1;
        float ks = 0.0f, vs = 0.0f;
        if (u + lane / per < n && key < keys) {
          const int page = table[key / a.block];
          if (page >= 0 && page < a.num_blocks) {
            const int unit = page * a.heads + w.head;
            row = unit * a.block + key % a.block;
            ks = a.scales[0][unit] * a.scale_log2;
            vs = a.scales[1][unit];
          } else {
            q8_flag(1);
          }
        }
        const int some = min(lot, n - u);
        for (int i = 0; i < some; ++i) {
          const int stage = issued % L::STAGES;
          // (the whole warp goes on or gives up together)
          if (!__all_sync(0xffffffffu, mbar_wait(&empty[stage], ((issued / L::STAGES) & 1) ^ 1u,
                                                 abort_flag))) {
            ok = false;
            break;
          }
          const int l0 = i * per;  // the unit's first lane
          const unsigned there = (__ballot_sync(0xffffffffu, row >= 0) >> l0) & ((1u << per) - 1);
          float* sc = reinterpret_cast<float*>(smem + L::SC_OFF + stage * L::SC);
          // group g of 16 keys belongs to load g * per / 4
          const int src = l0 + (lane & 3) * per / PAGES;
          const float gk = __shfl_sync(0xffffffffu, ks, src);
          const float gv = __shfl_sync(0xffffffffu, vs, src);
          const unsigned groups =
              __ballot_sync(0xffffffffu, lane < PAGES && ((there >> ((lane & 3) * per / PAGES)) & 1));
          if (lane < PAGES) {
            sc[lane] = gk;
            sc[PAGES + lane] = gv;
          }
          if (lane == 0) reinterpret_cast<unsigned*>(sc)[2 * PAGES] = groups;
          __syncwarp();
          if (lane == 0)
            mbar_expect_tx(&full[stage], static_cast<uint32_t>(__popc(there) * box * D * 2));
          __syncwarp();
          if (lane >= l0 && lane < l0 + per && row >= 0) {
            uint8_t* dst = smem + stage * L::STAGE + (lane - l0) * box * D;
            tma_load_2d(dst, &map_k, &full[stage], 0, row);
            tma_load_2d(dst + L::HALF, &map_v, &full[stage], 0, row);
          }
          ++issued;
        }
      }
      left -= n;
      at = 0;
      if (left > 0) w.next();
    }
    if (*abort_flag && lane == 0) {  // copies in flight land before the CTA retires (bounded)
      for (int j = issued - 1; j >= 0 && j >= issued - L::STAGES; --j) {
        const uint64_t t0 = global_ns();
        while (!mbar_try_wait(&full[j % L::STAGES], (j / L::STAGES) & 1) &&
               global_ns() - t0 < 200000000ull) {
        }
      }
    }
    __syncwarp();
  } else {
    // ---- products and softmax
    const int g = lane >> 2, t = lane & 3;
    const int part = warp & 3;   // 16 keys of the unit
    const int turn = warp >> 2;  // which of two units
    constexpr int KS = D / 16;   // steps of the first product, row tiles of the second
    float* merge = reinterpret_cast<float*>(smem + L::MERGE_OFF);
    float* ml = reinterpret_cast<float*>(smem + L::ML_OFF);
    int used = 0;
    int piece = 0;
    bool ok = true;
    while (left > 0) {
      const int n = static_cast<int>(left < w.units - at ? left : w.units - at);
      const bool whole = n == w.units;
      const int keys = Q8Work<Q8D_BN>::keys(a, w.count, w.len, w.tile);
      const int tok0 = w.tile * a.tile_tokens;
      // query row r of the item: token tok0 + r / group, head r % group
      uint32_t qf[NT][2 * KS];
      int limit[NT][2];  // keys that queries 2t and 2t + 1 see
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int r = j * 8 + g, tok = tok0 + r / a.group;
        const bool live = r < a.tile_tokens * a.group && tok < w.count;
        const uint4* src = reinterpret_cast<const uint4*>(
            a.q + (w.first + (live ? tok : 0)) * a.ld_q +
            static_cast<int64_t>(w.head * a.group + (live ? r % a.group : 0)) * a.hs_q + t * (D / 4));
#pragma unroll
        for (int c = 0; c < KS / 2; ++c) {
          const uint4 raw = live ? src[c] : make_uint4(0, 0, 0, 0);
          qf[j][4 * c] = raw.x;
          qf[j][4 * c + 1] = raw.y;
          qf[j][4 * c + 2] = raw.z;
          qf[j][4 * c + 3] = raw.w;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r2 = j * 8 + 2 * t + e, tok2 = tok0 + r2 / a.group;
          const bool in = r2 < a.tile_tokens * a.group && tok2 < w.count;
          limit[j][e] = !in ? 0 : a.causal ? min(keys, w.len - w.count + tok2 + 1) : keys;
        }
      }
      float o[NT][KS][4];
      float m[NT][2], l[NT][2];  // running maximum (0 while there is none), this lane's sums
      bool none[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[j][i][e] = 0.0f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          m[j][e] = 0.0f;
          l[j][e] = 0.0f;
          none[j][e] = true;
        }
      }
      for (int u = 0; u < n; ++u, ++used) {
        if ((used & 1) != turn) continue;
        const int stage = used % L::STAGES;
        ok = ok && __all_sync(0xffffffffu,
                              mbar_wait(&full[stage], (used / L::STAGES) & 1, abort_flag));
        if (!ok) continue;
        const float* sc = reinterpret_cast<const float*>(smem + L::SC_OFF + stage * L::SC);
        const unsigned groups = reinterpret_cast<const unsigned*>(sc)[8];
        const int key0 = (at + u) * Q8D_BN + part * 16;
        if ((groups >> part) & 1) {
          const float ks = sc[part], vs = sc[4 + part];
          const uint8_t* sk = smem + stage * L::STAGE + part * 16 * D;
          const uint8_t* sv = sk + L::HALF;
          // scores of keys g and g + 8 for queries 2t, 2t + 1
          float s[NT][4];
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][e] = 0.0f;
#pragma unroll
          for (int c = 0; c < KS / 4; ++c) {
            const int chunk = t * (KS / 4) + c;
            const uint4 lo = *reinterpret_cast<const uint4*>(sk + q8_chunk<D>(g, chunk));
            const uint4 hi = *reinterpret_cast<const uint4*>(sk + q8_chunk<D>(g + 8, chunk));
            const uint32_t l4[4] = {lo.x, lo.y, lo.z, lo.w}, h4[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t a0 = q8_pair<FMT>(l4[i], 0u, 0, 1), a2 = q8_pair<FMT>(l4[i], 0u, 2, 3);
              const uint32_t a1 = q8_pair<FMT>(h4[i], 0u, 0, 1), a3 = q8_pair<FMT>(h4[i], 0u, 2, 3);
#pragma unroll
              for (int j = 0; j < NT; ++j)
                mma_16816(s[j], a0, a1, a2, a3, qf[j][8 * c + 2 * i], qf[j][8 * c + 2 * i + 1]);
            }
          }
          uint32_t pf[NT][2];
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            bool in[4];
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              in[e] = key0 + g + (e >> 1) * 8 < limit[j][e & 1];
              x[e] = in[e] ? s[j][e] * ks : -INFINITY;
            }
            // The maximum only moves when a score exceeds it by 2^8 (or there was none): the
            // stale one cancels in the division. Decided for the warp, so that every lane of a
            // query keeps the same maximum.
            float top[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
            const bool need = (top[0] > m[j][0] + 8.0f) || (top[1] > m[j][1] + 8.0f) ||
                              (none[j][0] && top[0] > -INFINITY) || (none[j][1] && top[1] > -INFINITY);
            if (__any_sync(0xffffffffu, need)) {
#pragma unroll
              for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int sh = 4; sh < 32; sh <<= 1)
                  top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], sh));
                const float now = none[j][e] ? top[e] : fmaxf(m[j][e], top[e]);
                const bool some = now > -INFINITY;
                const float alpha = none[j][e] || !some ? 0.0f : ex2_approx(m[j][e] - now);
                if (some) {
                  m[j][e] = now;
                  none[j][e] = false;
                  l[j][e] *= alpha;
#pragma unroll
                  for (int i = 0; i < KS; ++i) {
                    o[j][i][e] *= alpha;
                    o[j][i][2 + e] *= alpha;
                  }
                }
              }
            }
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float ex = ex2_approx(x[e] - m[j][e & 1]);
              l[j][e & 1] += ex;
              p[e] = in[e] ? ex * vs : 0.0f;  // a masked key's scale may be NaN
            }
            pf[j][0] = movmatrix(pack_bf16x2(p[0], p[1]));
            pf[j][1] = movmatrix(pack_bf16x2(p[2], p[3]));
          }
          // o[dim, query] += v^T p: keys 2t, 2t + 1, 2t + 8, 2t + 9; dims (D / 8) g + 2i, + 1
          uint32_t vv[4][KS / 2];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row = 2 * t + (r & 1) + (r >> 1) * 8;
            if constexpr (D == 128) {
              const uint4 raw = *reinterpret_cast<const uint4*>(sv + q8_chunk<D>(row, g));
              vv[r][0] = raw.x;
              vv[r][1] = raw.y;
              vv[r][2] = raw.z;
              vv[r][3] = raw.w;
            } else {
              const uint2 raw = *reinterpret_cast<const uint2*>(sv + q8_chunk<D>(row, g >> 1) + (g & 1) * 8);
              vv[r][0] = raw.x;
              vv[r][1] = raw.y;
            }
          }
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            const int by = (i & 1) * 2;
            const uint32_t a0 = q8_pair<FMT>(vv[0][i >> 1], vv[1][i >> 1], by, 4 + by);
            const uint32_t a1 = q8_pair<FMT>(vv[0][i >> 1], vv[1][i >> 1], by + 1, 5 + by);
            const uint32_t a2 = q8_pair<FMT>(vv[2][i >> 1], vv[3][i >> 1], by, 4 + by);
            const uint32_t a3 = q8_pair<FMT>(vv[2][i >> 1], vv[3][i >> 1], by + 1, 5 + by);
#pragma unroll
            for (int j = 0; j < NT; ++j) mma_16816(o[j][i], a0, a1, a2, a3, pf[j][0], pf[j][1]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
      }
      // ---- the eight warps' results of this item
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = j * 8 + 2 * t + e;
#pragma unroll
          for (int sh = 4; sh < 32; sh <<= 1) l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], sh);
          if (g == 0) {
            ml[(warp * 8 * NT + r) * 2] = none[j][e] ? -INFINITY : m[j][e];
            ml[(warp * 8 * NT + r) * 2 + 1] = l[j][e];
          }
          float* dst = merge + (warp * 8 * NT + r) * L::LDO + g * (D / 8);
#pragma unroll
          for (int i = 0; i < KS; ++i)
            *reinterpret_cast<float2*>(dst + 2 * i) = make_float2(o[j][i][e], o[j][i][2 + e]);
        }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const int slot = 2 * static_cast<int>(blockIdx.x) + (piece > 0 ? 1 : 0);
      for (int e = threadIdx.x; e < 8 * NT * (D / 4); e += 32 * Q8D_WARPS) {
        const int r = e / (D / 4), c = (e % (D / 4)) * 4;
        const int tok = tok0 + r / a.group;
        if (r >= a.tile_tokens * a.group || tok >= w.count) continue;
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < Q8D_WARPS; ++k) top = fmaxf(top, ml[(k * 8 * NT + r) * 2]);
        const float ref = top > -INFINITY ? top : 0.0f;
        float sum = 0.0f;
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < Q8D_WARPS; ++k) {
          const float wt = ex2_approx(ml[(k * 8 * NT + r) * 2] - ref);
          sum += wt * ml[(k * 8 * NT + r) * 2 + 1];
          const float4 x = *reinterpret_cast<const float4*>(merge + (k * 8 * NT + r) * L::LDO + c);
          y.x += wt * x.x;
          y.y += wt * x.y;
          y.z += wt * x.z;
          y.w += wt * x.w;
        }
        if (whole) {
          const float inv = top > -INFINITY ? 1.0f / sum : 1.0f;
          *reinterpret_cast<uint2*>(a.out + (w.first + tok) * a.ld_out +
                                    static_cast<int64_t>(w.head * a.group + r % a.group) * a.hs_out + c) =
              make_uint2(pack_bf16x2(y.x * inv, y.y * inv), pack_bf16x2(y.z * inv, y.w * inv));
        } else {
          const int64_t at_row = static_cast<int64_t>(slot) * a.tile_rows + r;
          *reinterpret_cast<float4*>(a.part_o + at_row * D + c) = y;
          if (c == 0) {
            a.part_ml[at_row * 2] = top;
            a.part_ml[at_row * 2 + 1] = sum;
          }
        }
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      left -= n;
      at = 0;
      ++piece;
      if (left > 0) w.next();
    }
  }
}

// ---------------------------------------------------------------- cut items
// CTA c looks at the border between the runs c and c + 1. Where it is the first border inside an
// item, it adds that item's pieces: the last piece of run c, then the first piece of each run up
// to the item's end. (A run's pieces but its first and last are whole items; a piece that is both
// first and last is in slot 0.) gridDim.y CTAs share the rows.
template <int D, int BN>
__global__ void __launch_bounds__(256) attention_q8_combine_kernel(const Q8Attn a) {
  griddep_wait();
  griddep_launch();
  __shared__ int s_item[4];      // b, tile, head, pieces (0: nothing to do)
  __shared__ int s_slot0;
  Q8Work<BN> w(a);
  if (threadIdx.x < 32) {
    const int64_t total = w.total();
    const int64_t run = q8_run_units(a, total);
    const int64_t border = (blockIdx.x + 1) * run;
    int pieces = 0, slot0 = 0;
    if (border < total) {
      const int64_t in = w.seek(border);
      const int64_t start = border - in, end = start + w.units;
      if (in > 0 && start >= border - run) {
        pieces = static_cast<int>((end - 1) / run - blockIdx.x) + 1;
        slot0 = 2 * static_cast<int>(blockIdx.x) + (start > border - run ? 1 : 0);
      }
    }
    if (threadIdx.x == 0) {
      s_item[0] = w.b;
      s_item[1] = w.tile;
      s_item[2] = w.head;
      s_item[3] = pieces;
      s_slot0 = slot0;
    }
  }
  __syncthreads();
  const int pieces = s_item[3];
  if (pieces == 0) return;
  w.enter(s_item[0]);
  const int tok0 = s_item[1] * a.tile_tokens, head = s_item[2];
  const int live = min(a.tile_tokens, w.count - tok0) * a.group;
  for (int e = blockIdx.y * 256 + threadIdx.x; e < live * (D / 4); e += gridDim.y * 256) {
    const int r = e / (D / 4), c = (e % (D / 4)) * 4;
    float top = -INFINITY, sum = 0.0f;
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k = 0; k < pieces; ++k) {
      const int slot = k == 0 ? s_slot0 : 2 * (static_cast<int>(blockIdx.x) + k);
      const int64_t at = static_cast<int64_t>(slot) * a.tile_rows + r;
      const float pm = a.part_ml[at * 2], pl = a.part_ml[at * 2 + 1];
      const float4 x = *reinterpret_cast<const float4*>(a.part_o + at * D + c);
      const float now = fmaxf(top, pm);
      const float ref = now > -INFINITY ? now : 0.0f;
      const float wo = ex2_approx(top - ref), wn = ex2_approx(pm - ref);
      sum = sum * wo + pl * wn;
      y.x = y.x * wo + x.x * wn;
      y.y = y.y * wo + x.y * wn;
      y.z = y.z * wo + x.z * wn;
      y.w = y.w * wo + x.w * wn;
      top = now;
    }
    // rows that see no key: zeros
    const float inv = top > -INFINITY ? 1.0f / sum : 1.0f;
    const int tok = tok0 + r / a.group;
    *reinterpret_cast<uint2*>(a.out + (w.first + tok) * a.ld_out +
                              static_cast<int64_t>(head * a.group + r % a.group) * a.hs_out + c) =
        make_uint2(pack_bf16x2(y.x * inv, y.y * inv), pack_bf16x2(y.z * inv, y.w * inv));
  }
}

}  // namespace kino
