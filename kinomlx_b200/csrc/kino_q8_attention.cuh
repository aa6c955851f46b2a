// Attention over the 8-bit K/V cache: softmax(q k^T * scale) v with k and v as codes times a scale
// for each cache block and head, fp32 scores, statistics and accumulation, G query heads on each
// K/V head.
//
// Codes are exact as bf16 and as f16, so the products run on 16-bit operands converted from the
// codes in registers. A block's K scale multiplies its columns of the scores. Its V scale vs goes
// into the exponent: with one reference m for a query row that follows the largest
// s + log2(vs), the second product's operand is P = exp2(s + log2(vs) - m) = vs exp2(s - m), at
// most 2^8 whatever the scales are, so it is rounded to f16 (2^-11 of its value; bf16 would give
// 2^-8), and the row sum takes each group's sum of P over vs. V scales up to
// 2^-90 count as 0.
//
// Work is cut by units of BN keys of one (sequence, query tile, K/V head), the items in that
// order; every CTA of one resident wave takes an equal run of units, whatever the lengths are
// (they are only known on the device). A run that starts or ends inside an item leaves an
// unnormalised partial result with its row maxima and sums; attention_q8_combine adds the pieces
// of each cut item in a fixed order.
#pragma once
#include <cfloat>
#include <type_traits>

#include "kino_attention.cuh"
#include "kino_q8_common.cuh"
#include "kino_sol.cuh"

namespace kino {

// Where a run starts, for the kernel that adds the pieces.
struct Q8RunStart {
  int64_t run;    // units of a run
  int64_t first;  // the item's first query row of its sequence
  int tile, head, count;
  int at, units;  // the run's first unit of the item's units (units 0: an empty run)
};

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
  int block_shift;  // log2(block)
  float scale_log2;
  int causal;
  int tile_tokens;  // query tokens of an item
  int tile_rows;    // rows of its partial results (tile_tokens * group, padded)
  int runs;         // CTAs (or CTA pairs)
  float* part_o;    // [2 * runs][tile_rows][D]
  float* part_ml;   // [2 * runs][tile_rows][2]: row maximum (log2 units), row sum
  Q8RunStart* starts;  // [runs]
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

constexpr float Q8_LEAST_V = 8.0779356694631609e-28f;  // 2^-90

// Units of a run. (Runs of at least two to eight units for short caches were no faster.)
__device__ __forceinline__ int64_t q8_run_units(const Q8Attn& a, int64_t total) {
  return (total + a.runs - 1) / a.runs;
}

// ---------------------------------------------------------------- few query rows
// Up to 8 NT query rows (tokens x group) an item, keys in units of 64. Bound by reading the cache:
// the last warp brings each unit (K and V of 64 tokens, 128 D bytes) to shared memory by TMA, up to
// STAGES units ahead; the others take turns on the units in groups of four, 16 keys a warp.
//
// The products use mma.sync with the keys (then the dims of V) as the 16 rows and the query rows
// as the 8 columns, so that a single decoded token with a group of up to 8 heads fills a tile;
// the tensor pipe is far from its limit here. Each lane reads 16-byte runs of codes and pairs
// them as the fragments want by choosing which dims (of K: 32 t + 4 s ..) or keys and dims (of V)
// a fragment's rows and columns stand for, so nothing is transposed but the 16 x 8
// probabilities (movmatrix).
constexpr int Q8D_BN = 64;
// Warps that compute (one more loads): three groups of four where the registers allow it (16 x 32768
// tokens, one tile of rows, in a graph: 180 us, 188 with two groups).
constexpr int q8d_warps(int nt) { return nt == 1 ? 12 : 8; }

template <int D, int NT>
struct Q8DecodeSmem {
  static constexpr int HALF = Q8D_BN * D;  // K or V of a unit
  static constexpr int STAGE = 2 * HALF;
  // A multiple of the groups that take turns: a stage then always belongs to the same group, which
  // has seen each earlier phase of its barrier. (Another group could come to a stage whose last
  // load is still on its way, since loads need not arrive in order, and take the phase before that
  // for its own.)
  static constexpr int WARPS = q8d_warps(NT), TURNS = WARPS / 4;
  static constexpr int STAGES = (NT == 1 ? 9 : 8) * (D == 128 ? 1 : 2);
  static_assert(STAGES % TURNS == 0, "a stage belongs to one group of warps");
  static constexpr int LDO = D + 4;        // padded row of the merge buffer, in floats
  static constexpr int MERGE_OFF = STAGES * STAGE;
  static constexpr int MERGE = WARPS * 8 * NT * LDO * 4;
  static constexpr int ML_OFF = MERGE_OFF + MERGE;      // [warp][8 NT][2]
  static constexpr int SC_OFF = ML_OFF + WARPS * 8 * NT * 8;
  // per stage, of the four 16-key groups: K scales (with the softmax scale), 1 / vs, log2(vs), and
  // a word of which groups are there
  static constexpr int SC = 64;
  static constexpr int BAR_OFF = SC_OFF + STAGES * SC;
  static constexpr int TOTAL = BAR_OFF + 2 * STAGES * 8 + 64 + 1024;
};

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
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
__global__ void __launch_bounds__(32 * (q8d_warps(NT) + 1), 1)
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
      a.starts[blockIdx.x] = u0 < total ? Q8RunStart{run, w.first, w.tile, w.head, w.count,
                                                     static_cast<int>(at), w.units}
                                        : Q8RunStart{run, 0, 0, 0, 0, 0, 0};
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
      mbar_init(&full[i], 2);  // the copies, the scales
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

  constexpr int WARPS = L::WARPS;
  if (warp == WARPS) {
    // ---- loads: the places and scales of up to eight units are looked up at once, a lane for each
    // group of 16 keys, while the eight before them are issued (a look-up is two dependent reads,
    // about a microsecond, in which two or three units arrive)
    constexpr int GROUPS = Q8D_BN / 16, LOT = 32 / GROUPS, STEP = 4;
    const int box = a.block >= Q8D_BN ? Q8D_BN : a.block;
    const bool leads = (lane & 3) * 16 % box == 0;  // the copy of its group's box
    const unsigned lead_groups = box == 64 ? 1u : box == 32 ? 5u : 15u;
    int row = -1, count = 0;  // of the next units
    float ks = 0.0f, rv = 0.0f, lv = 0.0f;
    auto look = [&]() {
      count = 0;
      row = -1;
      if (left <= 0) return;
      const int n = static_cast<int>(left < w.units - at ? left : w.units - at);
      count = n < LOT ? n : LOT;
      const int key = (at + lane / GROUPS) * Q8D_BN + (lane & 3) * 16;
      if (lane / GROUPS < count && key < Q8Work<Q8D_BN>::keys(a, w.count, w.len, w.tile)) {
        const int page = a.table[static_cast<int64_t>(w.b) * a.ld_table + (key >> a.block_shift)];
        if (page >= 0 && page < a.num_blocks) {
          const int unit = page * a.heads + w.head;
          row = unit * a.block + (key & (a.block - 1));
          // the codes stand in f16 as their value over q8_f16_unit, those of K and of V
          ks = a.scales[0][unit] * a.scale_log2 * q8_f16_unit<FMT>();
          const float vs = a.scales[1][unit];
          const float v = vs <= Q8_LEAST_V ? Q8_LEAST_V : vs;
          rv = 1.0f / (v * q8_f16_unit<FMT>());
          lv = log2f(v);
        } else {
          q8_flag(1);
        }
      }
      left -= count;
      at += count;
      if (at == w.units) {
        at = 0;
        if (left > 0) w.next();
      }
    };
    int issued = 0;
    bool ok = true;
    look();
    while (count > 0) {
      const int row_now = row, units = count;
      const float ks_now = ks, rv_now = rv, lv_now = lv;
      look();
      const int mine = lane / GROUPS;
      const int unit = issued + mine, stage = unit % L::STAGES;
      for (int u = 0; u < units && ok; u += STEP) {
        const bool active = mine >= u && mine < u + STEP && mine < units;
        // (the whole warp goes on or gives up together)
        ok = __all_sync(0xffffffffu,
                        !active || mbar_wait(&empty[stage], ((unit / L::STAGES) & 1) ^ 1u, abort_flag));
        if (!ok) break;
        const unsigned groups =
            (__ballot_sync(0xffffffffu, active && row_now >= 0) >> (lane & ~3)) & 15u;
        // the copies first: the scales may still be on their way
        if (active && (lane & 3) == 0)
          mbar_expect_tx(&full[stage],
                         static_cast<uint32_t>(__popc(groups & lead_groups) * box * D * 2));
        __syncwarp();
        if (active && row_now >= 0 && leads) {
          uint8_t* dst = smem + stage * L::STAGE + (lane & 3) * 16 * D;
          tma_load_2d(dst, &map_k, &full[stage], 0, row_now);
          tma_load_2d(dst + L::HALF, &map_v, &full[stage], 0, row_now);
        }
        if (active) {
          float* sc = reinterpret_cast<float*>(smem + L::SC_OFF + stage * L::SC);
          sc[lane & 3] = ks_now;
          sc[GROUPS + (lane & 3)] = rv_now;
          sc[2 * GROUPS + (lane & 3)] = lv_now;
          if ((lane & 3) == 0) reinterpret_cast<unsigned*>(sc)[3 * GROUPS] = groups;
        }
        __syncwarp();
        if (active && (lane & 3) == 0) mbar_arrive(&full[stage]);
      }
      if (!ok) break;
      issued += units;
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
    const int turn = warp >> 2;  // which of TURNS units
    constexpr int KS = D / 16;   // steps of the first product, row tiles of the second
    float* merge = reinterpret_cast<float*>(smem + L::MERGE_OFF);
    float* ml = reinterpret_cast<float*>(smem + L::ML_OFF);
    int used = 0, next = 0;  // units so far, and the turn of the one that is next
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
      float qm[NT][2];   // what their rows were divided by
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
        // f16 queries: a power of two brings the row's largest value to [1, 2), and is taken back
        // with the K scale (values below 2^-14 of the largest lose low bits, 2^-25 of it at most)
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i)
          top = max(top, max((qf[j][i] & 0x7FFFu) << 16, qf[j][i] & 0x7FFF0000u));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // (the factors of zeros, subnormals and the largest values are the nearest normal ones)
        const uint32_t ex = min(max(top >> 23, 1u), 253u);
        const float down = __uint_as_float((254u - ex) << 23);
        // (a row that is not finite has only infinite and NaN scores, whose softmax is NaN also
        // where all of them are -infinity: its factor makes them NaN)
        const float up = __uint_as_float(top < 0x7F800000u ? ex << 23 : 0x7FC00000u);
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i) {
          const float2 f = unpack_bf16x2(qf[j][i]);
          qf[j][i] = pack_f16x2(f.x * down, f.y * down);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) qm[j][e] = __shfl_sync(0xffffffffu, up, (2 * t + e) * 4);
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
        const bool take = next == turn;
        next = next + 1 == L::TURNS ? 0 : next + 1;
        if (!take) continue;
        const int stage = used % L::STAGES;
        ok = ok && __all_sync(0xffffffffu,
                              mbar_wait(&full[stage], (used / L::STAGES) & 1, abort_flag));
        if (!ok) continue;
        const float* sc = reinterpret_cast<const float*>(smem + L::SC_OFF + stage * L::SC);
        const unsigned groups = reinterpret_cast<const unsigned*>(sc)[12];
        const int key0 = (at + u) * Q8D_BN + part * 16;
        if ((groups >> part) & 1) {
          const float ks = sc[part], rv = sc[4 + part], lv = sc[8 + part];
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
              const uint32_t wl = q8_f16_bias<FMT>(l4[i]), wh = q8_f16_bias<FMT>(h4[i]);
              const uint32_t a0 = q8_f16_pair<FMT>(wl, 0), a2 = q8_f16_pair<FMT>(wl, 1);
              const uint32_t a1 = q8_f16_pair<FMT>(wh, 0), a3 = q8_f16_pair<FMT>(wh, 1);
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
              x[e] = in[e] ? fmaf(s[j][e], ks * qm[j][e & 1], lv) : -INFINITY;
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
              p[e] = ex2_approx(x[e] - m[j][e & 1]);
              if (in[e]) l[j][e & 1] = fmaf(p[e], rv, l[j][e & 1]);  // a masked key's rv may be NaN
            }
            if (lv == -90.0f) p[0] = p[1] = p[2] = p[3] = 0.0f;  // a V scale of 0
            pf[j][0] = movmatrix(pack_f16x2(p[0], p[1]));
            pf[j][1] = movmatrix(pack_f16x2(p[2], p[3]));
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
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < KS / 2; ++i) vv[r][i] = q8_f16_bias<FMT>(vv[r][i]);
#pragma unroll
          for (int i = 0; i < KS / 2; ++i) {
            // bytes of the two keys side by side: dims 4i, 4i + 1 and 4i + 2, 4i + 3 of the run
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t lo = __byte_perm(vv[0][i], vv[1][i], h ? 0x7362 : 0x5140);
              const uint32_t hi = __byte_perm(vv[2][i], vv[3][i], h ? 0x7362 : 0x5140);
              const uint32_t a0 = q8_f16_pair<FMT>(lo, 0), a1 = q8_f16_pair<FMT>(lo, 1);
              const uint32_t a2 = q8_f16_pair<FMT>(hi, 0), a3 = q8_f16_pair<FMT>(hi, 1);
#pragma unroll
              for (int j = 0; j < NT; ++j)
                mma_16816(o[j][2 * i + h], a0, a1, a2, a3, pf[j][0], pf[j][1]);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
      }
      // ---- the warps' results of this item
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
      asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory");
      const int slot = 2 * static_cast<int>(blockIdx.x) + (piece > 0 ? 1 : 0);
      for (int e = threadIdx.x; e < 8 * NT * (D / 4); e += 32 * WARPS) {
        const int r = e / (D / 4), c = (e % (D / 4)) * 4;
        const int tok = tok0 + r / a.group;
        if (r >= a.tile_tokens * a.group || tok >= w.count) continue;
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < WARPS; ++k) top = fmaxf(top, ml[(k * 8 * NT + r) * 2]);
        const float ref = top > -INFINITY ? top : 0.0f;
        float sum = 0.0f;
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < WARPS; ++k) {
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
      asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory");
      left -= n;
      at = 0;
      ++piece;
      if (left > 0) w.next();
    }
  }
}

// ---------------------------------------------------------------- many query rows
// tcgen05 on CTA pairs (cta_group::2): an item is up to two tiles of 256 query rows, 128 of each
// in either CTA (chunks of 128 / group tokens x group heads, so that grouped heads share the keys'
// tile), over blocks of 128 keys. A pair shares a block's operands: each CTA converts 64 of its
// keys for the first product and half of the dims of its V for the second, which halves the
// conversion and the shared-memory traffic.
//   warp 0        Q chunks by TMA, when the last item's first products are done
//   warp 1        tensor memory; in the even CTA the products, issued from code that the compiler
//                 knows to be uniform (from one divergent thread they took twice as long); in the
//                 odd CTA the word to the even one that a block's operands are there (by a thread
//                 without loads in flight, which a release at cluster scope would wait for)
//   warps 2..9    softmax of the CTA's rows, four warps a tile and a thread a row, 64 keys at a time
//   warps 10..13  codes -> bf16 (K), f16 (V) in the layout TMA would write (128-byte swizzle);
//                 each thread keeps the next block's codes in registers
// Tensor memory: S_A in columns [0, 128), S_B [128, 256), O_A [256, 256 + D), O_B [384, 384 + D).
// Each S is two buffers of 64 keys, so that a tile's next scores are there while its warps work on
// these (keys 32 h .. and 64 + 32 h .. of the block for buffer h: 32 of each CTA's 64). P of a buffer
// overlies its scores. All roles of both CTAs walk the same run of items; the pipelines' phases go
// on over items. Tile A sees a prefix of the item's keys under a causal mask and leaves the blocks
// behind it out.
//
// 4608 queries x 9216 keys, 24 heads of 128: 600 us in a graph, 870 TFLOP/s, 620 in calls one after
// another (the cache read to bf16 and the dense bf16 kernel, two calls: 455);
// on single CTAs with two warps a row 1400, in pairs 1100, a row a thread 810, with the issue and
// the words between CTAs as above 655, in half blocks 608, with maxima that select nothing in
// unmasked blocks 600. Neither pipe is full: the tensor pipe
// is busy for about 2400 of 5000 cycles a block, exponentials for 2048; the chain score ->
// maximum -> P -> product of either tile is what remains, and the conversion (100 us of the 600).
constexpr int Q8P_BN = 128;
constexpr int Q8P_THREADS = 448;

template <int D>
struct Q8PrefillSmem {
  static constexpr int HALF = 128 * 64 * 2;  // Q: 128 rows x 64 dims
  static constexpr int KHALF = 64 * 64 * 2;  // K: this CTA's 64 keys x 64 dims
  static constexpr int K_BYTES = D / 64 * KHALF;
  static constexpr int V_BYTES = 128 * D;    // V: 128 keys x D / 2 dims
  static constexpr int Q_OFF = 0;            // tile t at t * 2 * HALF
  static constexpr int KV_OFF = 4 * HALF;
  static constexpr int STAGE = K_BYTES + V_BYTES;
  static constexpr int STAGES = 4;
  static constexpr int SC_OFF = KV_OFF + STAGES * STAGE;
  // a stage's 8 groups of 16 keys: (K scale times the softmax scale, log2(vs)) each, and a mask of
  // the groups that are there
  static constexpr int SC = 80;
  static constexpr int BAR_OFF = SC_OFF + STAGES * SC;
  // q_full, q_empty, kv_full[S], kv_empty[S], kv_peer[S], s_full[4], p_full[4], pv_done[2], o_full,
  // o_empty, drain
  static constexpr int NBAR = 2 + 3 * STAGES + 4 + 4 + 2 + 3;
  static constexpr int USED = BAR_OFF + NBAR * 8 + 64 + 1024;
  // No CTA of another kernel that holds tensor memory while it waits for its cluster may share an SM
  // (each could wait for columns that the other holds on the cluster's other SM): heads of 64 ask
  // for more than they use.
  static constexpr int TOTAL = USED > 140 * 1024 ? USED : 140 * 1024;
};

// sdesc_mn128 for 32 elements a row: 64-byte rows along K with the 64-byte swizzle, 8-row groups
// 512 bytes apart.
__device__ __forceinline__ uint64_t sdesc_mn64(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(1u) << 16;
  d |= static_cast<uint64_t>(512u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(4u) << 61;
  return d;
}

// D += A (each CTA's tensor memory) * B (halves of N in both CTAs' shared memory).
__device__ __forceinline__ void umma_f16_ts_pair(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                                 uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, "
      "p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}

// One lane of the warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}
// The same value in every lane (which the compiler then knows).
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
// mbar_wait by a whole warp, which goes on or gives up together.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort));
}

template <int D, int FMT>
__global__ void __launch_bounds__(Q8P_THREADS, 1)
    attention_q8_prefill_kernel(const __grid_constant__ CUtensorMap map_q, const Q8Attn a) {
  using L = Q8PrefillSmem<D>;
  using Work = Q8Work<Q8P_BN>;
  constexpr int NH = D / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t* q_full = bars;                      // even CTA's
  uint64_t* q_empty = bars + 1;
  uint64_t* kv_full = bars + 2;                 // this CTA's converted operands and scales
  uint64_t* kv_empty = kv_full + L::STAGES;
  uint64_t* kv_peer = kv_empty + L::STAGES;     // even CTA's: the odd one's operands
  uint64_t* s_full = kv_peer + L::STAGES;
  uint64_t* p_full = s_full + 4;                // even CTA's; both [half][tile]
  uint64_t* pv_done = p_full + 4;               // [tile]
  uint64_t* o_full = pv_done + 2;
  uint64_t* o_empty = o_full + 1;               // even CTA's
  uint64_t* drain = o_empty + 1;
  int64_t* s_run = reinterpret_cast<int64_t*>(bars + L::NBAR);  // u0, u1, at
  int* s_item = reinterpret_cast<int*>(s_run + 3);              // b, tile, head
  volatile int* abort_flag = s_item + 3;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_item + 4);

  const int warp = uniform(warp_id());
  const int lane = static_cast<int>(lane_id());
  const int rank = static_cast<int>(cluster_rank());
  const int pair = static_cast<int>(blockIdx.x >> 1);
  griddep_wait();
  Work w(a);
  if (warp == 0) {
    const int64_t total = w.total();
    const int64_t run = q8_run_units(a, total);
    const int64_t u0 = pair * run;
    int64_t in = 0;
    if (u0 < total) in = w.seek(u0);
    if (lane == 0) {
      if (rank == 0)
        a.starts[pair] = u0 < total ? Q8RunStart{run, w.first, w.tile, w.head, w.count,
                                                 static_cast<int>(in), w.units}
                                    : Q8RunStart{run, 0, 0, 0, 0, 0, 0};
      s_run[0] = u0;
      s_run[1] = u0 + run < total ? u0 + run : total;
      s_run[2] = in;
      s_item[0] = w.b;
      s_item[1] = w.tile;
      s_item[2] = w.head;
      *abort_flag = 0;
    }
  } else if (warp == 1) {
    if (lane == 0) {
      mbar_init(q_full, 1);
      mbar_init(q_empty, 1);
      for (int i = 0; i < L::STAGES; ++i) {
        mbar_init(&kv_full[i], 4);  // the converting warps
        mbar_init(&kv_empty[i], 1);
        mbar_init(&kv_peer[i], 1);
      }
      for (int t = 0; t < 2; ++t) {
        for (int h = 0; h < 2; ++h) {
          mbar_init(&s_full[h * 2 + t], 1);
          mbar_init(&p_full[h * 2 + t], 8);  // the tile's softmax warps of both CTAs
        }
        mbar_init(&pv_done[t], 1);
      }
      mbar_init(o_full, 1);
      mbar_init(o_empty, 16);
      mbar_init(drain, 1);
      fence_barrier_init();
    }
    __syncwarp();
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist before any remote arrive
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  griddep_launch();
  int64_t left = s_run[1] - s_run[0];
  int at = static_cast<int>(s_run[2]);
  if (left > 0) {
    w.enter(s_item[0]);
    w.tile = s_item[1];
    w.head = s_item[2];
    w.units = Work::units_of(a, w.count, w.len, w.tile);
  }
  const int chunk = a.tile_tokens >> 2;  // tokens of 128 rows
  // Blocks that tile A takes part in: those its last token sees, all if there is no tile B.
  auto blocks_a = [&](int ntile) {
    if (ntile == 1 || !a.causal) return w.units;
    const int last = min(w.count, w.tile * a.tile_tokens + 2 * chunk);
    return (max(0, w.len - w.count + last) + Q8P_BN - 1) / Q8P_BN;
  };

  if (warp < 2) {
    if (warp == 0 && lane == 0) {
      // ---- queries
      int items = 0;
      while (left > 0) {
        const int n = static_cast<int>(left < w.units - at ? left : w.units - at);
        if (Work::keys(a, w.count, w.len, w.tile) > 0) {
          const int tok0 = w.tile * a.tile_tokens;
          const int ntile = w.count - tok0 > 2 * chunk ? 2 : 1;
          if (!mbar_wait(q_empty, (items & 1) ^ 1u, abort_flag)) break;
          if (rank == 0)
            mbar_expect_tx(q_full, static_cast<uint32_t>(ntile * 2 * D * 2 * a.group * chunk));
          for (int t = 0; t < ntile; ++t)
            for (int h = 0; h < NH; ++h)
              tma_load_3d_pair(smem + L::Q_OFF + (t * 2 + h) * L::HALF, &map_q,
                               smem_u32(q_full) & kPairLeaderMask, h * 64, w.head * a.group,
                               static_cast<int>(w.first) + tok0 + (2 * t + rank) * chunk);
          ++items;
        }
        left -= n;
        at = 0;
        if (left > 0) w.next();
      }
      if (*abort_flag && items > 0) {  // a bounded moment for copies in flight
        const uint64_t t0 = global_ns();
        while (global_ns() - t0 < 100000000ull) {
        }
      }
    } else if (warp == 1 && rank == 0) {
      // ---- products: the whole warp walks the run, with values that the compiler knows to be the
      // same in all lanes, and one lane issues
      const bool issue = elect_one();
      constexpr uint32_t idesc_s = idesc_bf16(256, 64);
      constexpr uint32_t idesc_o = idesc_f16(256, D) | (1u << 16);  // V: MN-major
      // (descriptors hold addresses in units of 16 bytes: steps are plain additions)
      auto s_mma = [&](int t, int jb, int half) {
        const uint64_t sq = sdesc_k128(smem_u32(smem + L::Q_OFF + t * 2 * L::HALF));
        const uint64_t sk =
            sdesc_k128(smem_u32(smem + L::KV_OFF + (jb % L::STAGES) * L::STAGE + half * 32 * 128));
        if (issue) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_bf16_pair(tmem + t * 128 + half * 64,
                           sq + ((kk >> 2) * L::HALF + (kk & 3) * 32) / 16,
                           sk + ((kk >> 2) * L::KHALF + (kk & 3) * 32) / 16, idesc_s,
                           kk > 0 ? 1u : 0u);
          umma_commit_pair(&s_full[half * 2 + t], 0x3);
        }
      };
      auto pv_mma = [&](int t, int jb, int half, bool first, bool free_stage) {
        const uint32_t at_v =
            smem_u32(smem + L::KV_OFF + (jb % L::STAGES) * L::STAGE + L::K_BYTES);
        const uint64_t sv = (D == 128 ? sdesc_mn128(at_v, L::V_BYTES) : sdesc_mn64(at_v)) +
                            half * 32 * D / 16;
        if (issue) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)  // keys 32 half + 16 kk, then 64 + 32 half + 16 (kk - 2)
            umma_f16_ts_pair(tmem + 256 + t * 128, tmem + t * 128 + half * 64 + kk * 8,
                             sv + (kk * 16 + (kk >= 2 ? 32 : 0)) * D / 16, idesc_o,
                             (!first || kk > 0) ? 1u : 0u);
          umma_commit_pair(&pv_done[t], 0x3);
          if (free_stage) umma_commit_pair(&kv_empty[jb % L::STAGES], 0x3);
        }
      };
      auto block_there = [&](int jb) {
        const uint32_t parity = (jb / L::STAGES) & 1;
        return warp_wait(&kv_full[jb % L::STAGES], parity, abort_flag) &&
               warp_wait(&kv_peer[jb % L::STAGES], parity, abort_flag);
      };
      int items = 0, jb = 0;
      uint32_t parity = 0;  // bit t: of the blocks that tile t has been given
      bool ok = true;
      while (__any_sync(0xffffffffu, left > 0) && ok) {
        const int n = uniform(static_cast<int>(left < w.units - at ? left : w.units - at));
        if (__any_sync(0xffffffffu, Work::keys(a, w.count, w.len, w.tile) > 0)) {
          const int ntile = uniform(w.count - w.tile * a.tile_tokens > 2 * chunk ? 2 : 1);
          const int na = uniform(blocks_a(ntile) - at);  // of this piece's blocks
          ok = warp_wait(q_full, items & 1, abort_flag) && block_there(jb);
          if (!ok) break;
          tc_fence_after();
          for (int half = 0; half < 2; ++half)
            for (int t = na > 0 ? 0 : 1; t < ntile; ++t) s_mma(t, jb, half);
          ok = warp_wait(o_empty, (items & 1) ^ 1u, abort_flag);  // the last output was read
          for (int j = 0; j < n && ok; ++j, ++jb) {
            // (before the wait for P, which takes longer)
            if (j + 1 < n) {
              ok = block_there(jb + 1);
              if (!ok) break;
            }
#pragma unroll 1
            for (int half = 0; half < 2 && ok; ++half)
#pragma unroll 1
              for (int t = j < na ? 0 : 1; t < ntile; ++t) {
                ok = warp_wait(&p_full[half * 2 + t], (parity >> t) & 1, abort_flag);
                if (!ok) break;
                parity ^= static_cast<uint32_t>(half) << t;
                tc_fence_after();
                pv_mma(t, jb, half, j == 0 && half == 0, half == 1 && t == ntile - 1);
                if (j + 1 < n && (t == 1 || j + 1 < na)) s_mma(t, jb + 1, half);
              }
          }
          if (!ok) break;
          if (issue) umma_commit_pair(q_empty, 0x3);
          if (issue) umma_commit_pair(o_full, 0x3);
          ++items;
        }
        left -= n;
        at = 0;
        if (left > 0) w.next();
      }
      // all issued products end before tensor memory is released (bounded)
      if (issue) umma_commit_pair(drain, 0x1);
      const uint64_t t0 = global_ns();
      while (!mbar_try_wait(drain, 0) && global_ns() - t0 < 200000000ull) {
      }
    }
    if (warp == 1 && lane == 0 && rank == 1) {
      // ---- word to the even CTA
      const uint32_t there = cluster_addr(smem_u32(kv_peer), 0);
      int jb = 0;
      bool ok = true;
      while (left > 0 && ok) {
        const int n = static_cast<int>(left < w.units - at ? left : w.units - at);
        if (Work::keys(a, w.count, w.len, w.tile) > 0)
          for (int j = 0; j < n && ok; ++j, ++jb) {
            ok = mbar_wait(&kv_full[jb % L::STAGES], (jb / L::STAGES) & 1, abort_flag);
            if (ok) mbar_arrive_cluster(there + (jb % L::STAGES) * 8);
          }
        left -= n;
        at = 0;
        if (left > 0) w.next();
      }
    }
    __syncwarp();
  } else if (warp >= 10) {
    // ---- codes to 16 bits
    const int cw = warp - 10;
    // K: runs of 16 codes of this CTA's 64 keys; V: of D / 2 dims of 128 keys. The lanes of a
    // quarter warp are laid so that its 16-byte stores fall on different banks.
    constexpr int KPR = D / 16, VPR = D / 32;            // runs a row
    constexpr int KROWS = 128 / KPR, VROWS = 128 / VPR;  // rows that the four warps read at once
    constexpr int NK = 64 / KROWS, NVV = 128 / VROWS;    // reads a thread
    const int k_run = D == 128 ? (lane & 3) + ((lane >> 3) & 1) * 4 : lane & 3;
    const int k_row = cw * (32 / KPR) + (D == 128 ? ((lane >> 2) & 1) + (lane >> 4) * 2 : lane >> 2);
    const int v_run = D == 128 ? lane & 3 : lane & 1;
    const int v_row = cw * (32 / VPR) + (D == 128 ? lane >> 2 : lane >> 1);
    const uint32_t k_dst = smem_u32(smem + L::KV_OFF) + (k_run >> 2) * L::KHALF + k_row * 128;
    const uint32_t k0 = k_dst + ((((k_run & 3) * 2) ^ (k_row & 7)) << 4);
    const uint32_t k1 = k_dst + ((((k_run & 3) * 2 + 1) ^ (k_row & 7)) << 4);
    const uint32_t v_dst = smem_u32(smem + L::KV_OFF) + L::K_BYTES + v_row * D;
    const int v_swz = D == 128 ? v_row & 7 : (v_row >> 1) & 3;
    const uint32_t v0 = v_dst + (((v_run * 2) ^ v_swz) << 4);
    const uint32_t v1 = v_dst + (((v_run * 2 + 1) ^ v_swz) << 4);
    int n = 0;  // units of the item that are left to look up
    auto settle = [&]() {  // on to a unit with keys (an item without any has one unit), or the end
      while (left > 0) {
        n = static_cast<int>(left < w.units - at ? left : w.units - at);
        if (Work::keys(a, w.count, w.len, w.tile) > 0) return;
        left -= n;
        at = 0;
        if (left > 0) w.next();
      }
    };
    auto step = [&]() {
      ++at;
      --left;
      if (--n == 0) {
        at = 0;
        if (left > 0) {
          w.next();
          settle();
        }
      }
    };
    // lanes 0..7: where the cursor's 16-key groups are (K and V), and their scales
    int k_there = -1, v_there = -1;
    float ks = 0.0f, vs = 0.0f;
    auto look = [&]() {
      k_there = v_there = -1;
      ks = vs = 0.0f;
      if (left > 0 && lane < 8) {
        const int key = at * Q8P_BN + lane * 16;
        if (key < Work::keys(a, w.count, w.len, w.tile)) {
          const int page = a.table[static_cast<int64_t>(w.b) * a.ld_table + (key >> a.block_shift)];
          if (page >= 0 && page < a.num_blocks) {
            const int unit = page * a.heads + w.head;
            k_there = unit * a.block + (key & (a.block - 1));
            ks = a.scales[0][unit] * a.scale_log2;
            vs = a.scales[1][unit];
            v_there = vs <= Q8_LEAST_V ? -1 : k_there;  // taken as zero codes
          } else {
            q8_flag(1);
          }
        }
      }
    };
    uint4 kraw[NK], vraw[NVV];
    auto fetch_k = [&](int i) {
      const int r = rank * 64 + i * KROWS + k_row;
      const int base = __shfl_sync(0xffffffffu, k_there, r >> 4);
      kraw[i] = make_uint4(0, 0, 0, 0);
      if (base >= 0)
        kraw[i] = __ldg(reinterpret_cast<const uint4*>(
            a.codes[0] + static_cast<int64_t>(base + (r & 15)) * D + k_run * 16));
    };
    auto fetch_v = [&](int i) {
      const int r = i * VROWS + v_row;
      const int base = __shfl_sync(0xffffffffu, v_there, r >> 4);
      vraw[i] = make_uint4(0, 0, 0, 0);
      if (base >= 0)
        vraw[i] = __ldg(reinterpret_cast<const uint4*>(
            a.codes[1] + static_cast<int64_t>(base + (r & 15)) * D + rank * (D / 2) + v_run * 16));
    };
    auto store = [&](uint32_t dst, uint32_t x, uint32_t y, uint32_t z, uint32_t t) {
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(x), "r"(y), "r"(z),
                   "r"(t)
                   : "memory");
    };
    settle();
    look();
    bool todo = left > 0;
    if (todo) {
#pragma unroll
      for (int i = 0; i < NK; ++i) fetch_k(i);
#pragma unroll
      for (int i = 0; i < NVV; ++i) fetch_v(i);
    }
    int jb = 0;
    while (todo) {
      const float ks_now = ks, vs_now = vs;
      const unsigned groups = __ballot_sync(0xffffffffu, k_there >= 0) & 0xFFu;
      step();
      look();
      todo = left > 0;
      const int stage = jb % L::STAGES;
      if (!__all_sync(0xffffffffu, mbar_wait(&kv_empty[stage], ((jb / L::STAGES) & 1) ^ 1u,
                                             abort_flag)))
        break;
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        const uint32_t off = stage * L::STAGE + i * KROWS * 128;
        const uint4 v = kraw[i];
        store(k0 + off, q8_pair<FMT>(v.x, 0u, 0, 1), q8_pair<FMT>(v.x, 0u, 2, 3),
              q8_pair<FMT>(v.y, 0u, 0, 1), q8_pair<FMT>(v.y, 0u, 2, 3));
        store(k1 + off, q8_pair<FMT>(v.z, 0u, 0, 1), q8_pair<FMT>(v.z, 0u, 2, 3),
              q8_pair<FMT>(v.w, 0u, 0, 1), q8_pair<FMT>(v.w, 0u, 2, 3));
      }
      if (todo) {
#pragma unroll
        for (int i = 0; i < NK; ++i) fetch_k(i);
      }
#pragma unroll
      for (int i = 0; i < NVV; ++i) {
        const uint32_t off = stage * L::STAGE + i * VROWS * D;
        const uint32_t x = q8_f16_bias<FMT>(vraw[i].x), y = q8_f16_bias<FMT>(vraw[i].y);
        const uint32_t z = q8_f16_bias<FMT>(vraw[i].z), t = q8_f16_bias<FMT>(vraw[i].w);
        store(v0 + off, q8_f16_pair<FMT>(x, 0), q8_f16_pair<FMT>(x, 1), q8_f16_pair<FMT>(y, 0),
              q8_f16_pair<FMT>(y, 1));
        store(v1 + off, q8_f16_pair<FMT>(z, 0), q8_f16_pair<FMT>(z, 1), q8_f16_pair<FMT>(t, 0),
              q8_f16_pair<FMT>(t, 1));
      }
      if (todo) {
#pragma unroll
        for (int i = 0; i < NVV; ++i) fetch_v(i);
      }
      if (cw == 0) {
        float* sc = reinterpret_cast<float*>(smem + L::SC_OFF + stage * L::SC);
        if (lane < 8) {
          sc[2 * lane] = ks_now;
          sc[2 * lane + 1] = log2f(vs_now <= Q8_LEAST_V ? Q8_LEAST_V : vs_now);
        }
        if (lane == 0) reinterpret_cast<unsigned*>(sc)[16] = groups;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&kv_full[stage]);
      ++jb;
    }
  } else {
    // ---- softmax: one row a thread, 64 of the block's keys at a time
    const int t = (warp - 2) >> 2;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t o_col = tmem + lane_base + 256 + t * 128;
    const int row_tok = row / a.group, row_head = row % a.group;
    const bool in_row = row < chunk * a.group;
    const uint32_t p_full0 = cluster_addr(smem_u32(&p_full[t]), 0);
    const uint32_t o_empty0 = cluster_addr(smem_u32(o_empty), 0);
    int items = 0, jb = 0, piece = 0;
    int cnt = 0;  // half blocks of this tile
    bool ok = true;
    while (left > 0) {
      const int n = static_cast<int>(left < w.units - at ? left : w.units - at);
      const bool whole = n == w.units;
      const int keys = Work::keys(a, w.count, w.len, w.tile);
      const int ntile = w.count - w.tile * a.tile_tokens > 2 * chunk ? 2 : 1;
      const int tok = w.tile * a.tile_tokens + (2 * t + rank) * chunk + row_tok;
      const bool live = in_row && tok < w.count;
      // keys that this row sees (rows of no query are computed with whatever is there and not
      // stored), and the least of the warp's rows
      const int limit = !live ? 0x7fffffff
                              : a.causal ? max(0, min(keys, w.len - w.count + tok + 1)) : keys;
      const int least = __reduce_min_sync(0xffffffffu, limit);
      int blocks = 0;  // that the tile takes part in
      if (keys > 0 && t < ntile) blocks = t == 1 ? n : min(n, blocks_a(ntile) - at);
      float m_run = -INFINITY, l_run = 0.0f;
#pragma unroll 1
      for (int hj = 0; hj < 2 * blocks; ++hj, ++cnt) {
        const int half = hj & 1, j = hj >> 1;
        const int stage = (jb + j) % L::STAGES;
        ok = __all_sync(0xffffffffu,
                        mbar_wait(&kv_full[stage], ((jb + j) / L::STAGES) & 1, abort_flag) &&
                            mbar_wait(&s_full[half * 2 + t], (cnt >> 1) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        // Row i of the tile keeps one reference m, and the second product's operand is
        //   P = vs exp2(s ks - m) = exp2(s ks + log2(vs) - m),
        // so the reference follows the largest s ks + log2(vs) and P stays within f16's range
        // whatever the blocks' V scales are; the row sum takes a group's sum of P over vs.
        const uint32_t s_col = tmem + lane_base + t * 128 + half * 64;
        uint32_t sr[2][32];
        tmem_ld32(s_col, sr[0]);
        tmem_ld32(s_col + 32, sr[1]);
        // columns 0..31 are keys key0 .., columns 32..63 keys key0 + 64 ..
        const int key0 = (at + j) * Q8P_BN + half * 32;
        const float4* sc = reinterpret_cast<const float4*>(smem + L::SC_OFF + stage * L::SC) + half;
        const float4 sc2[2] = {sc[0], sc[2]};
        const unsigned word =
            reinterpret_cast<const unsigned*>(smem + L::SC_OFF + stage * L::SC)[16] >> (2 * half);
        const unsigned groups = (word & 3u) | ((word >> 2) & 12u);
        const bool masked = key0 + 96 > least || groups != 15u;  // warp-uniform
        const int valid[2] = {masked ? limit - key0 : 32, masked ? limit - key0 - 64 : 32};
        tmem_wait_ld();
        // (scales are not negative: a group's largest score gives its largest scaled one)
        float best[4];
        if (masked) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const uint32_t* v = sr[g >> 1] + (g & 1) * 16;
            const int of = (g & 1) * 16;
            float x = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i)
              x = fmaxf(x, of + i < valid[g >> 1] ? __uint_as_float(v[i]) : -INFINITY);
            best[g] = x;
          }
        } else {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const uint32_t* v = sr[g >> 1] + (g & 1) * 16;
            auto f = [&](int i) { return __uint_as_float(v[i]); };
            const float x = max3f(f(0), f(1), f(2)), y = max3f(f(3), f(4), f(5));
            const float z = max3f(f(6), f(7), f(8)), u = max3f(f(9), f(10), f(11));
            best[g] = max3f(max3f(x, y, z), max3f(u, f(12), f(13)), fmaxf(f(14), f(15)));
          }
        }
        float y[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 s4 = sc2[g >> 1];
          y[g] = fmaf(best[g], g & 1 ? s4.z : s4.x, g & 1 ? s4.w : s4.y);
        }
        // A masked group stays at -inf whatever its scales are. One in sight counts as the lowest
        // finite value at least: a row whose scores are all -inf then ends as 0 / 0, and not as
        // one that sees no key.
        float mine = -INFINITY;
        if (masked) {
#pragma unroll
          for (int g = 0; g < 4; ++g)
            if ((g & 1) * 16 < valid[g >> 1] && ((groups >> g) & 1))
              mine = max3f(mine, y[g], -FLT_MAX);
        } else {
          mine = max3f(max3f(y[0], y[1], y[2]), y[3], -FLT_MAX);
        }
        // The reference moves only when it is exceeded by 2^8 (the stale one cancels in the
        // division).
        float alpha = 1.0f;
        bool rescale = false;
        if (hj > 0) {
          const bool need = mine > m_run + 8.0f;
          rescale = __any_sync(0xffffffffu, need);
          if (need) {
            alpha = ex2_approx(m_run - mine);
            m_run = mine;
            l_run *= alpha;
          }
        } else {
          m_run = mine;
        }
        const float ref = m_run == -INFINITY ? 0.0f : m_run;
        auto exps = [&](auto tag) {
          constexpr bool MASKED = decltype(tag)::value;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const uint32_t* v = sr[g >> 1] + (g & 1) * 16;
            const float4 s4 = sc2[g >> 1];
            const float kg = g & 1 ? s4.z : s4.x, lg = g & 1 ? s4.w : s4.y, cg = lg - ref;
            const uint64_t k2 = f2_pack(kg, kg), c2 = f2_pack(cg, cg);
            uint64_t sum2[2] = {f2_pack(0.0f, 0.0f), f2_pack(0.0f, 0.0f)};
            uint32_t packed[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const int e = 2 * u;
              const uint64_t xs =
                  f2_fma(f2_pack(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), k2, c2);
              const float2 xv = f2_unpack(xs);
              float2 p2 = make_float2(ex2_approx(xv.x), ex2_approx(xv.y));
              if constexpr (MASKED) {  // a masked key counts for nothing, its scales may be NaN
                const bool in = (groups >> g) & 1;
                p2.x = in && (g & 1) * 16 + e < valid[g >> 1] ? p2.x : 0.0f;
                p2.y = in && (g & 1) * 16 + e + 1 < valid[g >> 1] ? p2.y : 0.0f;
              }
              sum2[u & 1] = f2_add(sum2[u & 1], f2_pack(p2.x, p2.y));
              packed[u] = pack_f16x2(p2.x, p2.y);
            }
            const float2 s2 = f2_unpack(f2_add(sum2[0], sum2[1]));
            if (!MASKED || (((groups >> g) & 1) && (g & 1) * 16 < valid[g >> 1]))
              l_run = fmaf(s2.x + s2.y, ex2_approx(-lg), l_run);
            tmem_st8(s_col + g * 8, packed);  // over the scores, which are in registers
          }
        };
        if (masked)
          exps(std::true_type{});
        else
          exps(std::false_type{});
        if (rescale) {
          // the product of the half block before this one has to be in the output
          ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[t], (cnt - 1) & 1, abort_flag));
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(o_col + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(o_col + c * 32, o);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        // (tensor memory only, written above: no memory to release)
        if (lane == 0) mbar_arrive_cluster_relaxed(p_full0 + half * 16);
      }
      if (keys > 0) {
        ok = ok && __all_sync(0xffffffffu, mbar_wait(o_full, items & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        jb += n;
      }
      l_run *= 1.0f / q8_f16_unit<FMT>();  // the V codes stand as their value over it
      if (t < ntile) {
        const float inv = m_run == -INFINITY ? 1.0f : 1.0f / l_run;
        const int64_t part = static_cast<int64_t>(2 * pair + (piece > 0 ? 1 : 0)) * a.tile_rows +
                             (2 * t + rank) * chunk * a.group + row;
        if (!whole && live) {
          a.part_ml[part * 2] = m_run;
          a.part_ml[part * 2 + 1] = l_run;
        }
        __nv_bfloat16* out = a.out + (w.first + tok) * a.ld_out +
                             static_cast<int64_t>(w.head * a.group + row_head) * a.hs_out;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          if (blocks > 0) {
            tmem_ld32(o_col + c * 32, o);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0;
          }
          if (live && whole) {
            uint32_t w16[16];
#pragma unroll
            for (int i = 0; i < 16; ++i)
              w16[i] = pack_bf16x2(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
            store_row32(out + c * 32, w16, 32);
          } else if (live) {
            uint4* dst = reinterpret_cast<uint4*>(a.part_o + part * D + c * 32);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              dst[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
        }
      }
      if (keys > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(o_empty0);
        ++items;
      }
      left -= n;
      at = 0;
      ++piece;
      if (left > 0) w.next();
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the products have drained; neither CTA's memory is in use any more
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ---------------------------------------------------------------- cut items
// CTA c looks at the border between the runs c and c + 1. Where it is the first border inside an
// item, it adds that item's pieces: the last piece of run c, then the first piece of each run up
// to the item's end. (A run's pieces but its first and last are whole items; a piece that is both
// first and last is in slot 0.) gridDim.y CTAs share the rows, D / 4 threads a row. One sequence on
// one head may be in as many pieces as there are CTAs: then all groups of D / 4 threads of a CTA
// share a row's pieces (32000 keys on one head: 14 us, 46 with one group a row).
template <int D>
__global__ void __launch_bounds__(256) attention_q8_combine_kernel(const Q8Attn a) {
  griddep_wait();
  griddep_launch();
  constexpr int LANES = D / 4, GROUPS = 256 / LANES;
  __shared__ float4 s_y[GROUPS][LANES];
  __shared__ float2 s_ml[GROUPS];
  const Q8RunStart s = a.starts[blockIdx.x + 1];
  const int64_t border = (blockIdx.x + 1) * s.run, start = border - s.at;
  if (s.units == 0 || s.at == 0 || start < border - s.run) return;
  const int pieces = static_cast<int>((start + s.units - 1) / s.run - blockIdx.x) + 1;
  const int slot0 = 2 * static_cast<int>(blockIdx.x) + (start > border - s.run ? 1 : 0);
  const int tok0 = s.tile * a.tile_tokens;
  const int live = min(a.tile_tokens, s.count - tok0) * a.group;
  const int group = threadIdx.x / LANES, c = threadIdx.x % LANES * 4;
  const bool share = pieces >= 2 * GROUPS;
  const int first = share ? group : 0, stride = share ? GROUPS : 1;
  for (int r = share ? blockIdx.y : blockIdx.y * GROUPS + group; r < live;
       r += gridDim.y * (share ? 1 : GROUPS)) {
    auto place = [&](int k) {
      const int slot = k == 0 ? slot0 : 2 * (static_cast<int>(blockIdx.x) + k);
      return static_cast<int64_t>(slot) * a.tile_rows + r;
    };
    float top = -INFINITY, sum = 0.0f;
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](float wt, float l, const float4 x) {
      sum = fmaf(l, wt, sum);
      y.x = fmaf(x.x, wt, y.x);
      y.y = fmaf(x.y, wt, y.y);
      y.z = fmaf(x.z, wt, y.z);
      y.w = fmaf(x.w, wt, y.w);
    };
    constexpr int LOT = 8;  // pieces whose reads are in flight together
    for (int k0 = first; k0 < pieces; k0 += LOT * stride) {
      float2 ml[LOT];
      float4 x[LOT];
#pragma unroll
      for (int i = 0; i < LOT; ++i) {
        const int k = k0 + i * stride;
        ml[i] = make_float2(-INFINITY, 0.0f);
        x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (k < pieces) {
          const int64_t at = place(k);
          ml[i] = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
          x[i] = *reinterpret_cast<const float4*>(a.part_o + at * D + c);
        }
      }
      float now = top;
#pragma unroll
      for (int i = 0; i < LOT; ++i) now = fmaxf(now, ml[i].x);
      const float ref = now > -INFINITY ? now : 0.0f;
      const float keep = ex2_approx(top - ref);
      sum *= keep;
      y.x *= keep;
      y.y *= keep;
      y.z *= keep;
      y.w *= keep;
      top = now;
#pragma unroll
      for (int i = 0; i < LOT; ++i) add(ex2_approx(ml[i].x - ref), ml[i].y, x[i]);
    }
    if (share) {
      s_y[group][c / 4] = y;
      if (c == 0) s_ml[group] = make_float2(top, sum);
      __syncthreads();
      if (group == 0) {
#pragma unroll
        for (int g = 1; g < GROUPS; ++g) top = fmaxf(top, s_ml[g].x);
        const float ref = top > -INFINITY ? top : 0.0f;
        sum = 0.0f;
        y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) add(ex2_approx(s_ml[g].x - ref), s_ml[g].y, s_y[g][c / 4]);
      }
      __syncthreads();
      if (group != 0) continue;
    }
    // rows that see no key: zeros
    const float inv = top > -INFINITY ? 1.0f / sum : 1.0f;
    const int tok = tok0 + r / a.group;
    *reinterpret_cast<uint2*>(a.out + (s.first + tok) * a.ld_out +
                              static_cast<int64_t>(s.head * a.group + r % a.group) * a.hs_out + c) =
        make_uint2(pack_bf16x2(y.x * inv, y.y * inv), pack_bf16x2(y.z * inv, y.w * inv));
  }
}

}  // namespace kino
