// 8-bit integer product on tcgen05 (kind::i8, exact int32 sums in tensor memory):
//
//   out[m, n] = bf16( float(sum_k x[m, k] * w[n, k]) * sx[m] * sw[n] + bias[n] )
//
// x holds int8 codes of tokens, w of output channels, both K-contiguous; sx and sw are the fp32
// scales of each token and channel. A K-step of one instruction is 32 bytes in both this and the
// bf16 kernel, so the tiles have the same bytes (128-byte swizzled rows = 128 codes) and half as
// many K steps.
//
// Two forms:
//   q8_gemm_pair_kernel   CTA pairs, 256 x 256 output tiles, persistent (the layout of the bf16
//                         pair kernel): large token counts, bound by the tensor cores.
//   q8_gemm_wide_kernel   128 channels x NT tokens, channels on the accumulator's lanes, so that
//                         few tokens waste no rows of the tensor tile and the weight is read
//                         once; the K range is cut over a cluster of up to 8 CTAs whose int32
//                         partial tiles are added through distributed shared memory. Integer sums
//                         do not depend on the cut. Few tokens: bound by reading the weight.
#pragma once
#include "kino_q8_common.cuh"
#include "kino_gemm.cuh"

namespace kino {

constexpr int Q8G_BK = 128;  // codes per shared-memory row

struct Q8GemmArgs {
  const float* sx;
  const float* sw;
  const __nv_bfloat16* bias;  // or null
  __nv_bfloat16* out;
  int64_t ldo;
  int m, n;
  int tiles_m, tiles_n, num_tiles, kblocks;
};

// Instruction descriptor for kind::i8: signed A and B, int32 accumulator, both K-major.
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) {
  return (2u << 4)                                  // D format: s32
         | (1u << 7)                                // A format: signed 8 bit
         | (1u << 10)                               // B format: signed 8 bit
         | (static_cast<uint32_t>(n >> 3) << 17)    // N / 8
         | (static_cast<uint32_t>(m >> 4) << 24);   // M / 16
}

__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                             uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// ---------------------------------------------------------------- CTA pairs
constexpr int Q8G_STAGES = 6;

__global__ void __launch_bounds__(GEMM_THREADS, 1)
    q8_gemm_pair_kernel(const __grid_constant__ CUtensorMap map_x,
                        const __grid_constant__ CUtensorMap map_w, const Q8GemmArgs a) {
  using L = Gemm2SmSmem<Q8G_STAGES>;  // 128 rows x 128 bytes of each operand a stage and CTA
  constexpr int BN = 256;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::TILE_BYTES);
  uint64_t* empty = full + Q8G_STAGES;
  uint64_t* tfull = empty + Q8G_STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);

  const int warp = warp_id();
  const uint32_t lane = lane_id();
  const uint32_t rank = cluster_rank();  // 0: leader (issues the MMAs), 1: peer
  const int pair = blockIdx.x >> 1;
  const int pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < Q8G_STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 2 * GEMM_EPI_WARPS);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch(&map_x);
    tma_prefetch(&map_w);
  }
  griddep_wait();
  if (warp == 1) {
    tmem_alloc_pair(tmem_base_slot, 2 * BN);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist before any remote arrive
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_slot;
  griddep_launch();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      for (int t = pair; t < a.num_tiles; t += pairs) {
        const int nt = t / a.tiles_m, mt = t % a.tiles_m;
        for (int kb = 0; kb < a.kblocks; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag)) goto producer_done;
          uint8_t* sa = smem + stage * L::STAGE_BYTES;
          uint8_t* sb = sa + L::A_BYTES;
          const uint32_t leader_full = smem_u32(&full[stage]) & kPairLeaderMask;
          if (rank == 0) mbar_expect_tx(&full[stage], 2 * L::STAGE_BYTES);
          tma_load_2d_pair(sa, &map_x, leader_full, kb * Q8G_BK, mt * 256 + rank * 128);
          tma_load_2d_pair(sb, &map_w, leader_full, kb * Q8G_BK, nt * BN + rank * 128);
          ++issued;
          if (++stage == Q8G_STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    producer_done:
      if (*abort_flag && issued > 0) {  // after a timeout: a bounded moment for loads in flight
        const uint64_t t0 = global_ns();
        while (global_ns() - t0 < 100000000ull) {
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = idesc_i8(256, BN);
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      for (int t = pair; t < a.num_tiles; t += pairs, ++local) {
        const int acc = local & 1;
        const uint32_t acc_phase = (local >> 1) & 1;
        if (!mbar_wait(&tempty[acc], acc_phase ^ 1u, abort_flag)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        bool ok = true;
        for (int kb = 0; kb < a.kblocks; ++kb) {
          if (!mbar_wait(&full[stage], phase, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * L::STAGE_BYTES);
          const uint32_t sb = sa + L::A_BYTES;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_i8_pair(d_tmem, sdesc_k128(sa + kk * 32), sdesc_k128(sb + kk * 32), idesc,
                         (kb > 0 || kk > 0) ? 1u : 0u);
          umma_commit_pair(&empty[stage], 0x3);
          if (++stage == Q8G_STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit_pair(&tfull[acc], 0x3);
      }
      umma_commit_pair(drain, 0x1);
      const uint64_t t0 = global_ns();
      while (!mbar_try_wait(drain, 0) && global_ns() - t0 < 200000000ull) {
      }
    }
  } else {
    const int quarter = warp & 3;
    const int half = (warp - 2) >> 2;  // column half of the tile
    const int row_in_tile = static_cast<int>(rank) * 128 + quarter * 32 + static_cast<int>(lane);
    const uint32_t leader_tempty0 = cluster_addr(smem_u32(&tempty[0]), 0);
    int local = 0;
    for (int t = pair; t < a.num_tiles; t += pairs, ++local) {
      const int nt = t / a.tiles_m, mt = t % a.tiles_m;
      const int acc = local & 1;
      const uint32_t acc_phase = (local >> 1) & 1;
      const int row = mt * 256 + row_in_tile;
      const bool live = row < a.m;
      const float sx = live ? a.sx[row] : 0.0f;
      if (!mbar_wait(&tfull[acc], acc_phase, abort_flag)) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((quarter * 32) << 16) + acc * BN + half * 128;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t r[32];
        tmem_ld32(taddr + c * 32, r);
        tmem_wait_ld();
        const int col = nt * BN + half * 128 + c * 32;
        if (live && col < a.n) {
          uint32_t packed[16];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            if (col + g * 8 < a.n) {
              const float4 s0 = __ldg(reinterpret_cast<const float4*>(a.sw + col + g * 8));
              const float4 s1 = __ldg(reinterpret_cast<const float4*>(a.sw + col + g * 8) + 1);
              float v[8];
              const float sw[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
              for (int j = 0; j < 8; ++j)
                v[j] = __fmul_rn(__fmul_rn(static_cast<float>(static_cast<int>(r[g * 8 + j])), sx), sw[j]);
              if (a.bias != nullptr) {
                const uint4 raw = __ldg(reinterpret_cast<const uint4*>(a.bias + col + g * 8));
                const uint32_t w4[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  const float2 f = unpack_bf16x2(w4[q]);
                  v[2 * q] = __fadd_rn(v[2 * q], f.x);
                  v[2 * q + 1] = __fadd_rn(v[2 * q + 1], f.y);
                }
              }
#pragma unroll
              for (int q = 0; q < 4; ++q) packed[g * 4 + q] = pack_bf16x2(v[2 * q], v[2 * q + 1]);
            } else {
#pragma unroll
              for (int q = 0; q < 4; ++q) packed[g * 4 + q] = 0;
            }
          }
          store_row32(a.out + static_cast<int64_t>(row) * a.ldo + col, packed, a.n - col);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster_relaxed(leader_tempty0 + acc * 8);
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * BN);
  }
}

// ---------------------------------------------------------------- few tokens
// One tile per CTA (and cluster along K): warp 0 loads, warp 1 issues, then all six warps add and
// store. After the products the pipeline's shared memory holds this CTA's int32 partial tile,
// [token][128 channels]; CTA r of the cluster finishes tokens r, r + splits, ...
constexpr int Q8W_THREADS = 192;

template <int NT>
struct Q8WideSmem {
  static constexpr int A_BYTES = 128 * Q8G_BK;  // weight rows
  static constexpr int B_BYTES = NT * Q8G_BK;   // token rows
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  // about 100 KB of loads in flight, and room for two CTAs on an SM
  static constexpr int STAGES = NT <= 32 ? 5 : NT <= 64 ? 4 : 3;
  static constexpr int PARTIAL_BYTES = NT * 128 * 4;
  static constexpr int TILE_BYTES =
      STAGES * STAGE_BYTES > PARTIAL_BYTES ? STAGES * STAGE_BYTES : PARTIAL_BYTES;
  static constexpr int BAR_BYTES = (2 * STAGES + 1) * 8 + 16;
  static constexpr int TOTAL = TILE_BYTES + BAR_BYTES + 1024;
  static constexpr int COLS = NT < 32 ? 32 : NT;
};

template <int NT>
__global__ void __launch_bounds__(Q8W_THREADS)
    q8_gemm_wide_kernel(const __grid_constant__ CUtensorMap map_x,
                        const __grid_constant__ CUtensorMap map_w, const Q8GemmArgs a,
                        const int splits) {
  using L = Q8WideSmem<NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::TILE_BYTES);
  uint64_t* empty = full + L::STAGES;
  uint64_t* done = empty + L::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id();
  const uint32_t lane = lane_id();
  const int split = blockIdx.x % splits;  // == rank in the cluster
  const int tile = blockIdx.x / splits;
  const int nt = tile / a.tiles_m, mt = tile % a.tiles_m;
  const int kb0 = static_cast<int>(static_cast<int64_t>(split) * a.kblocks / splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(split + 1) * a.kblocks / splits);
  const int nkb = kb1 - kb0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch(&map_x);
    tma_prefetch(&map_w);
  }
  griddep_wait();
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_launch();

  if (warp == 0) {
    if (lane == 0) {
      int issued = 0;
      for (int i = 0; i < nkb; ++i) {
        const int stage = i % L::STAGES;
        if (!mbar_wait(&empty[stage], ((i / L::STAGES) & 1) ^ 1u, abort_flag)) break;
        uint8_t* sa = smem + stage * L::STAGE_BYTES;
        mbar_expect_tx(&full[stage], L::STAGE_BYTES);
        tma_load_2d(sa, &map_w, &full[stage], (kb0 + i) * Q8G_BK, nt * 128);
        tma_load_2d(sa + L::A_BYTES, &map_x, &full[stage], (kb0 + i) * Q8G_BK, mt * NT);
        ++issued;
      }
      if (*abort_flag) {  // copies in flight land before the CTA goes on (bounded)
        for (int j = issued - 1; j >= 0 && j >= issued - L::STAGES; --j) {
          const uint64_t t0 = global_ns();
          while (!mbar_try_wait(&full[j % L::STAGES], (j / L::STAGES) & 1) &&
                 global_ns() - t0 < 200000000ull) {
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_i8(128, NT);
      for (int i = 0; i < nkb; ++i) {
        const int stage = i % L::STAGES;
        if (!mbar_wait(&full[stage], (i / L::STAGES) & 1, abort_flag)) break;
        tc_fence_after();
        const uint32_t sa = smem_u32(smem + stage * L::STAGE_BYTES);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          umma_i8(tmem, sdesc_k128(sa + kk * 32), sdesc_k128(sa + L::A_BYTES + kk * 32), idesc,
                  (i > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&empty[stage]);
      }
      umma_commit(done);
      // after a timeout elsewhere: issued products still end before tensor memory is released
      const uint64_t t0 = global_ns();
      while (!mbar_try_wait(done, 0) && global_ns() - t0 < 200000000ull) {
      }
    }
    __syncwarp();
  }
  // the products are complete: the stages' memory is free for the partial tile
  const bool ok = mbar_wait(done, 0, abort_flag);
  tc_fence_after();
  __syncthreads();
  int* part = reinterpret_cast<int*>(smem);
  if (ok && warp >= 2) {
    const int quarter = warp & 3;
#pragma unroll 1
    for (int c = 0; c < NT; c += 32) {
      uint32_t r[32];
      tmem_ld32(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + c, r);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (c + j < NT) part[(c + j) * 128 + quarter * 32 + lane] = static_cast<int>(r[j]);
    }
  }
  tc_fence_before();
  if (splits > 1)
    cluster_sync();
  else
    __syncthreads();
  if (ok) {
    // 16 threads a token, 8 channels each
    const int ch = nt * 128 + static_cast<int>(threadIdx.x & 15) * 8;
    float sw[8], bias[8];
    if (ch < a.n) {
      const float4 s0 = __ldg(reinterpret_cast<const float4*>(a.sw + ch));
      const float4 s1 = __ldg(reinterpret_cast<const float4*>(a.sw + ch) + 1);
      sw[0] = s0.x, sw[1] = s0.y, sw[2] = s0.z, sw[3] = s0.w;
      sw[4] = s1.x, sw[5] = s1.y, sw[6] = s1.z, sw[7] = s1.w;
      uint4 raw = make_uint4(0, 0, 0, 0);
      if (a.bias != nullptr) raw = __ldg(reinterpret_cast<const uint4*>(a.bias + ch));
      const uint32_t w4[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 f = unpack_bf16x2(w4[q]);
        bias[2 * q] = f.x;
        bias[2 * q + 1] = f.y;
      }
      const int most = min(NT, a.m - mt * NT);
      for (int t = split + static_cast<int>(threadIdx.x >> 4) * splits; t < most;
           t += (Q8W_THREADS / 16) * splits) {
        int acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        const uint32_t local = smem_u32(part + t * 128 + (threadIdx.x & 15) * 8);
        for (int r = 0; r < splits; ++r) {
          const uint32_t addr = splits > 1 ? cluster_addr(local, r) : local;
          int p[8];
          if (splits > 1) {
            asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(p[0]), "=r"(p[1]), "=r"(p[2]), "=r"(p[3])
                         : "r"(addr));
            asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(p[4]), "=r"(p[5]), "=r"(p[6]), "=r"(p[7])
                         : "r"(addr + 16));
          } else {
            asm volatile("ld.shared.v4.s32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(p[0]), "=r"(p[1]), "=r"(p[2]), "=r"(p[3])
                         : "r"(addr));
            asm volatile("ld.shared.v4.s32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(p[4]), "=r"(p[5]), "=r"(p[6]), "=r"(p[7])
                         : "r"(addr + 16));
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[j] += p[j];
        }
        const int row = mt * NT + t;
        const float sx = a.sx[row];
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[j] = __fmul_rn(__fmul_rn(static_cast<float>(acc[j]), sx), sw[j]);
          if (a.bias != nullptr) v[j] = __fadd_rn(v[j], bias[j]);
        }
        *reinterpret_cast<uint4*>(a.out + static_cast<int64_t>(row) * a.ldo + ch) =
            make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                       pack_bf16x2(v[6], v[7]));
      }
    }
  }
  if (splits > 1)
    cluster_sync();  // no CTA leaves while another reads its partial tile
  else
    __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, L::COLS);
  }
}

}  // namespace kino
