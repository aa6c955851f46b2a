// Host side of the 8-bit serving entry points (include/kino_q8.h): argument checks and launches.
// Part of the library's translation unit; uses kino_capi.cu's launch and error helpers.
#pragma once

namespace {

bool q8_format(int format) { return format == KINO_Q8_INT8 || format == KINO_Q8_E4M3; }

// 8-bit tensor map of `rows` rows of `width` bytes at `stride` bytes; boxes of 128 x box_rows (or
// the whole width where it is less than 128) bytes with the swizzle of that width.
kino_status make_map8(CUtensorMap* map, const void* base, uint64_t width, uint64_t rows,
                      uint64_t stride, uint32_t box_width, uint32_t box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return fail(KINO_ECUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t d[2] = {width, rows};
  const cuuint64_t s[1] = {stride};
  const cuuint32_t b[2] = {box_width, box_rows};
  const cuuint32_t e[2] = {1, 1};
  const CUresult r =
      fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), d, s, b, e,
         CU_TENSOR_MAP_INTERLEAVE_NONE,
         box_width == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(KINO_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return KINO_OK;
}

// Raises a kernel's dynamic shared memory limit, once per kernel and device.
template <auto Kernel>
kino_status q8_smem(int bytes) {
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && done[dev]) return KINO_OK;
  const cudaError_t e =
      cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(KINO_ECUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  if (dev >= 0 && dev < 64) done[dev] = true;
  return KINO_OK;
}

template <int FMT>
void launch_q8_rows(const kino::Q8RowArgs& a, int64_t rows, cudaStream_t stream) {
  // Four 16-byte vectors a thread where there are rows enough for many CTAs on an SM (9216 x 4096:
  // 48.0 us, 52.8 with two, 80.5 with one), two for few rows, whose latency counts.
  const int nvec = a.dim / 8, each = rows >= 8 * device_sms() ? 4 : 2;
  int threads = ((nvec + each - 1) / each + 31) / 32 * 32;
  if (threads > kino::Q8_ROW_MAX_THREADS) threads = kino::Q8_ROW_MAX_THREADS;
  const int nv = (nvec + threads - 1) / threads;
  auto run = [&](auto kernel) {
    launch_pdl(kernel, dim3(static_cast<unsigned>(rows)), dim3(threads), 0, stream, a);
  };
  if (nv <= 2)
    run(kino::q8_rows_kernel<FMT, 2>);
  else if (nv <= 4)
    run(kino::q8_rows_kernel<FMT, 4>);
  else
    run(kino::q8_wide_rows_kernel<FMT>);
}

int log2_block(int64_t block) { return block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7; }

template <int FMT>
void launch_q8_write(const kino::Q8WriteArgs& a, int64_t items, cudaStream_t stream) {
  auto run = [&](auto kernel, unsigned parts) {
    launch_pdl(kernel, dim3(static_cast<unsigned>(items * a.heads), parts),
               dim3(kino::Q8_WRITE_THREADS), 0, stream, a);
  };
  switch (a.block * a.dim / 1024) {
    case 1:
      return run(kino::q8_cache_write_kernel<FMT, 1, 2>, 1);
    case 2:
      return run(kino::q8_cache_write_kernel<FMT, 2, 2>, 1);
    case 4:
      return run(kino::q8_cache_write_kernel<FMT, 4, 2>, 1);
    case 8:
      return run(kino::q8_cache_write_kernel<FMT, 8, 2>, 1);
    default:
      return run(kino::q8_cache_write_kernel<FMT, 16, 1>, 2);
  }
}

kino_status check_q8_cache(const kino_q8_cache* c, const char* what) {
  if (c == nullptr || c->k_codes == nullptr || c->v_codes == nullptr || c->k_scales == nullptr ||
      c->v_scales == nullptr || c->table == nullptr || c->lengths == nullptr)
    return fail(KINO_EINVAL, "%s: null", what);
  if (!q8_format(c->format)) return fail(KINO_EINVAL, "%s: format %d", what, c->format);
  if (c->dim != 64 && c->dim != 128)
    return fail(KINO_ENOTSUPPORTED, "%s: heads are 64 or 128 wide, not %lld", what,
                (long long)c->dim);
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128)
    return fail(KINO_ENOTSUPPORTED, "%s: blocks hold 16, 32, 64 or 128 tokens, not %lld", what,
                (long long)c->block);
  if (c->num_blocks < 1 || c->heads < 1 || c->batch < 1 || c->table_blocks < 1 ||
      c->ld_table < c->table_blocks)
    return fail(KINO_EINVAL, "%s: empty cache, batch or table", what);
  if (c->heads > 65535 || c->batch > 65535 ||
      c->num_blocks > 0x7fffffffLL / (c->heads * c->block) ||
      c->table_blocks > 0x3fffffffLL / c->block)
    return fail(KINO_ENOTSUPPORTED, "%s: cache too large", what);
  if (!aligned16(c->k_codes) || !aligned16(c->v_codes))
    return fail(KINO_EINVAL, "%s: codes not 16-byte aligned", what);
  return KINO_OK;
}

template <int NT>
kino_status launch_q8_wide(const CUtensorMap& mw, const void* x, int64_t ldx, int64_t k,
                           kino::Q8GemmArgs a, int splits, cudaStream_t stream) {
  using L = kino::Q8WideSmem<NT>;
  CUtensorMap mx;
  kino_status st = make_map8(&mx, x, static_cast<uint64_t>(k), static_cast<uint64_t>(a.m),
                             static_cast<uint64_t>(ldx), 128, NT);
  if (st != KINO_OK) return st;
  constexpr auto kernel = kino::q8_gemm_wide_kernel<NT>;
  st = q8_smem<kernel>(L::TOTAL);
  if (st != KINO_OK) return st;
  a.tiles_m = (a.m + NT - 1) / NT;
  a.tiles_n = (a.n + 127) / 128;
  a.num_tiles = a.tiles_m * a.tiles_n;
  launch_ex(kernel, dim3(static_cast<unsigned>(a.num_tiles * splits)), dim3(kino::Q8W_THREADS),
            L::TOTAL, stream, splits, mx, mw, a, splits);
  return check_launch("kino_q8_linear");
}

// ---- attention: which kernel, and how its work is cut
struct Q8AttnPlan {
  int decode_tiles;  // 8-row tiles of the few-rows kernel (1 or 2), 0: the tcgen05 kernel
  int tile_tokens, tile_rows, runs;
  int64_t bytes;
};

kino_status plan_q8_attention(const kino_q8_cache* c, const kino_q8_attention_args* g,
                              Q8AttnPlan* p) {
  const char* what = "kino_q8_attention";
  kino_status st = check_q8_cache(c, what);
  if (st != KINO_OK) return st;
  if (g == nullptr) return fail(KINO_EINVAL, "%s: null", what);
  if (g->rows < 1 || g->rows > 0x3fffffffLL) return fail(KINO_EINVAL, "%s: rows", what);
  if (g->token_starts == nullptr && g->rows % c->batch)
    return fail(KINO_EINVAL, "%s: %lld rows do not divide over %lld sequences", what,
                (long long)g->rows, (long long)c->batch);
  if (g->q_heads < 1 || g->q_heads % c->heads)
    return fail(KINO_EINVAL, "%s: %lld query heads on %lld cache heads", what,
                (long long)g->q_heads, (long long)c->heads);
  const int64_t group = g->q_heads / c->heads;
  if (group > 128)
    return fail(KINO_ENOTSUPPORTED, "%s: at most 128 query heads on a cache head", what);
  // Query rows of a sequence on one cache head, on average (the lengths are on the device; both
  // kernels take any). Up to 64 rows the kernel for few rows is the faster one although it reads
  // the cache again for each 16 of them (16 sequences of 8192 tokens, 8 heads of 128: 32 rows
  // 131 us, with tcgen05 287; 64 rows 247 and 287; 8 sequences of 2000 with 128 rows 84 and 48).
  // One kernel for the call: a prompt's chunk beside decoded tokens is better a call of its own.
  const int64_t rows = (g->rows + c->batch - 1) / c->batch * group;
  p->decode_tiles = rows <= 8 ? 1 : rows <= 64 && group <= 16 ? 2 : 0;
  const int64_t tile = p->decode_tiles ? 8 * p->decode_tiles : 512;
  p->tile_tokens = static_cast<int>(p->decode_tiles ? tile / group : 4 * (128 / group));
  p->tile_rows = static_cast<int>(tile);
  p->runs = p->decode_tiles ? device_sms() : device_sms() / 2;  // CTAs, or pairs of them
  p->bytes = 2LL * p->runs * tile * (c->dim + 2) * 4 +
             p->runs * static_cast<int64_t>(sizeof(kino::Q8RunStart));
  return KINO_OK;
}

template <int D, int NT, int FMT>
kino_status launch_q8_decode(const kino_q8_cache* c, const kino::Q8Attn& a, cudaStream_t stream) {
  using L = kino::Q8DecodeSmem<D, NT>;
  CUtensorMap mk, mv;
  const uint64_t rows = static_cast<uint64_t>(c->num_blocks * c->heads * c->block);
  const uint32_t box = static_cast<uint32_t>(std::min<int64_t>(c->block, kino::Q8D_BN));
  kino_status st = make_map8(&mk, c->k_codes, D, rows, D, D, box);
  if (st != KINO_OK) return st;
  st = make_map8(&mv, c->v_codes, D, rows, D, D, box);
  if (st != KINO_OK) return st;
  constexpr auto kernel = kino::attention_q8_decode_kernel<D, NT, FMT>;
  st = q8_smem<kernel>(L::TOTAL);
  if (st != KINO_OK) return st;
  launch_pdl(kernel, dim3(a.runs), dim3(32 * (L::WARPS + 1)), L::TOTAL, stream, mk, mv, a);
  if (a.runs > 1)
    launch_pdl(kino::attention_q8_combine_kernel<D>, dim3(a.runs - 1, 2),
               dim3(256), 0, stream, a);
  return check_launch("kino_q8_attention");
}

// (see Q8PrefillSmem; 228 KB an SM, 1 KB of them for each CTA)
static_assert(kino::Q8PrefillSmem<64>::TOTAL + kino::Q8WideSmem<16>::TOTAL + 2048 > 228 * 1024,
              "the product's cluster form does not fit beside the attention");

template <int D, int FMT>
kino_status launch_q8_attention(const kino_q8_cache* c, kino::Q8Attn& a, int decode_tiles,
                                cudaStream_t stream) {
  if (decode_tiles == 1) return launch_q8_decode<D, 1, FMT>(c, a, stream);
  if (decode_tiles == 2) return launch_q8_decode<D, 2, FMT>(c, a, stream);
  // queries as (rows, heads, dim): a box is 64 dims of the group's heads of 128 / group tokens
  CUtensorMap mq;
  const uint64_t dims[3] = {D, static_cast<uint64_t>(a.heads) * a.group,
                            static_cast<uint64_t>(a.rows.rows)};
  // (the stride of a dimension of one counts for nothing but the map's own checks)
  const uint64_t strides[2] = {dims[1] > 1 ? static_cast<uint64_t>(a.hs_q) : D,
                               dims[2] > 1 ? static_cast<uint64_t>(a.ld_q) : D * dims[1]};
  const uint32_t box[3] = {64, static_cast<uint32_t>(a.group),
                           static_cast<uint32_t>(a.tile_tokens / 4)};
  kino_status st = make_map(&mq, a.q, 3, dims, strides, box);
  if (st != KINO_OK) return st;
  using L = kino::Q8PrefillSmem<D>;
  constexpr auto kernel = kino::attention_q8_prefill_kernel<D, FMT>;
  st = q8_smem<kernel>(L::TOTAL);
  if (st != KINO_OK) return st;
  launch_ex(kernel, dim3(2 * a.runs), dim3(kino::Q8P_THREADS), L::TOTAL, stream, 2, mq, a);
  if (a.runs > 1)
    launch_pdl(kino::attention_q8_combine_kernel<D>, dim3(a.runs - 1, 32), dim3(256),
               0, stream, a);
  return check_launch("kino_q8_attention");
}

}  // namespace

extern "C" {

int kino_q8_abi_version(void) { return 1; }

kino_status kino_q8_rows(const void* x, int64_t ldx, const void* residual, int64_t ld_residual,
                         const void* weight, float weight_offset, float eps, int norm,
                         void* hidden, int64_t ld_hidden, void* codes, float* scales, int format,
                         int64_t rows, int64_t dim, void* stream) {
  if (x == nullptr || codes == nullptr || scales == nullptr)
    return fail(KINO_EINVAL, "kino_q8_rows: null");
  if (!q8_format(format)) return fail(KINO_EINVAL, "kino_q8_rows: format %d", format);
  if (rows < 1 || rows > 0x7fffffffLL) return fail(KINO_EINVAL, "kino_q8_rows: rows");
  if (dim < 8 || dim % 8 || dim > 131072)
    return fail(KINO_ENOTSUPPORTED, "kino_q8_rows: dim %% 8 == 0 and dim <= 131072, not %lld",
                (long long)dim);
  if (!aligned16(x) || !aligned16(residual) || !aligned16(weight) || !aligned16(hidden) ||
      (reinterpret_cast<uintptr_t>(codes) & 7u))
    return fail(KINO_EINVAL, "kino_q8_rows: operands not aligned");
  if (ldx % 8 || ld_residual % 8 || ld_hidden % 8)
    return fail(KINO_ENOTSUPPORTED, "kino_q8_rows: row strides must be multiples of 8");
  if (rows > 1 && (ldx < dim || (residual != nullptr && ld_residual < dim) ||
                   (hidden != nullptr && ld_hidden < dim)))
    return fail(KINO_EINVAL, "kino_q8_rows: stride below width");
  if (!norm && weight != nullptr) return fail(KINO_EINVAL, "kino_q8_rows: a weight without a norm");
  kino::Q8RowArgs a;
  a.x = static_cast<const __nv_bfloat16*>(x);
  a.ldx = ldx;
  a.residual = static_cast<const __nv_bfloat16*>(residual);
  a.ld_residual = ld_residual;
  a.weight = static_cast<const __nv_bfloat16*>(weight);
  a.weight_offset = weight_offset;
  a.eps = eps;
  a.norm = norm;
  a.hidden = static_cast<__nv_bfloat16*>(hidden);
  a.ld_hidden = ld_hidden;
  a.codes = static_cast<uint8_t*>(codes);
  a.scales = scales;
  a.dim = static_cast<int>(dim);
  if (format == KINO_Q8_INT8)
    launch_q8_rows<kino::Q8_INT8>(a, rows, static_cast<cudaStream_t>(stream));
  else
    launch_q8_rows<kino::Q8_E4M3>(a, rows, static_cast<cudaStream_t>(stream));
  return check_launch("kino_q8_rows");
}

kino_status kino_q8_linear(const void* x, int64_t ldx, const float* x_scales, const void* w,
                           int64_t ldw, const float* w_scales, const void* bias, void* out,
                           int64_t ldo, int64_t m, int64_t n, int64_t k, void* stream) {
  if (x == nullptr || x_scales == nullptr || w == nullptr || w_scales == nullptr || out == nullptr)
    return fail(KINO_EINVAL, "kino_q8_linear: null");
  if (m < 1 || n < 1 || k < 1) return fail(KINO_EINVAL, "kino_q8_linear: empty shape");
  if (k % 16 || n % 8 || ldx % 16 || ldw % 16 || ldo % 8)
    return fail(KINO_ENOTSUPPORTED, "kino_q8_linear: k and the code strides must be multiples of "
                "16, n and the output stride of 8 (k=%lld n=%lld)", (long long)k, (long long)n);
  if (k >= 131072)  // 131072 products of -128 with itself are 2^31, one more than int32 holds
    return fail(KINO_ENOTSUPPORTED, "kino_q8_linear: k < 131072, not %lld", (long long)k);
  if (m > (1 << 28) || n > (1 << 28))
    return fail(KINO_ENOTSUPPORTED, "kino_q8_linear: shape too large");
  if (ldx < k || ldw < k || ldo < n) return fail(KINO_EINVAL, "kino_q8_linear: stride below width");
  if (!aligned16(x) || !aligned16(w) || !aligned16(w_scales) || !aligned16(bias) || !aligned16(out))
    return fail(KINO_EINVAL, "kino_q8_linear: operands not 16-byte aligned");
  kino::Q8GemmArgs a;
  a.sx = x_scales;
  a.sw = w_scales;
  a.bias = static_cast<const __nv_bfloat16*>(bias);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.ldo = ldo;
  a.m = static_cast<int>(m);
  a.n = static_cast<int>(n);
  a.kblocks = static_cast<int>((k + kino::Q8G_BK - 1) / kino::Q8G_BK);
  CUtensorMap mw;
  kino_status st = make_map8(&mw, w, static_cast<uint64_t>(k), static_cast<uint64_t>(n),
                             static_cast<uint64_t>(ldw), 128, 128);
  if (st != KINO_OK) return st;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Which form (device times at k = 4096 unless said, one SM count of 148):
  //  - the wide form with the least token tile that needs no more CTAs than fit at once (two on an
  //    SM, not quite filled): many small tiles read the weight from L2 again but finish sooner
  //    than few large ones (126 x 8192, k 2048: 8.6 us with 32 tokens a tile, 14.0 with 128;
  //    512 x 4096: 14.9 with 64, 17.6 in pairs); K cut only up to one CTA an SM (1 x 4096: 9.9
  //    whole, 7.0 cut by four; 64 x 4096 with 32 tokens: 9.0 cut by two, 9.2 by four);
  //  - CTA pairs once 256 x 256 tiles occupy two thirds of them (1024 x 4096: 18.3 us, wide 20.1;
  //    256 x 16384: 21.1, wide 21.9; 512 x 4096, 32 tiles on 74 pairs: 17.6, wide 14.9);
  //  - neither (few tokens, a very wide weight): one token tile, the weight read once.
  const int64_t sms = device_sms();
  const int64_t tiles_n = (n + 127) / 128;
  const int64_t pair_tiles = ((m + 255) / 256) * ((n + 255) / 256);
  int nt = 0;
  if (m <= 128 || 3 * pair_tiles < sms)
    for (nt = 16; nt <= 128; nt *= 2)
      if (4 * tiles_n * ((m + nt - 1) / nt) <= 7 * sms) break;
  if (nt > 128 && m <= 128)
    for (nt = 16; nt < m; nt *= 2) {
    }
  if (nt == 0 || nt > 128) {
    CUtensorMap mx;
    st = make_map8(&mx, x, static_cast<uint64_t>(k), static_cast<uint64_t>(m),
                   static_cast<uint64_t>(ldx), 128, 128);
    if (st != KINO_OK) return st;
    a.tiles_m = static_cast<int>((m + 255) / 256);
    a.tiles_n = static_cast<int>((n + 255) / 256);
    if (pair_tiles > 0x3fffffffLL) return fail(KINO_ENOTSUPPORTED, "kino_q8_linear: shape too large");
    a.num_tiles = static_cast<int>(pair_tiles);
    using L = kino::Gemm2SmSmem<kino::Q8G_STAGES>;
    constexpr auto kernel = kino::q8_gemm_pair_kernel;
    st = q8_smem<kernel>(L::TOTAL);
    if (st != KINO_OK) return st;
    const int pairs = static_cast<int>(std::min<int64_t>(a.num_tiles, sms / 2));
    launch_ex(kernel, dim3(2 * pairs), dim3(kino::GEMM_THREADS), L::TOTAL, s, 2, mx, mw, a);
    return check_launch("kino_q8_linear");
  }
  const int64_t tiles = tiles_n * ((m + nt - 1) / nt);
  int splits = 1;
  while (splits < 8 && tiles * splits * 2 <= sms && a.kblocks >= 8 * splits) splits *= 2;
  switch (nt) {
    case 16:
      return launch_q8_wide<16>(mw, x, ldx, k, a, splits, s);
    case 32:
      return launch_q8_wide<32>(mw, x, ldx, k, a, splits, s);
    case 64:
      return launch_q8_wide<64>(mw, x, ldx, k, a, splits, s);
    default:
      return launch_q8_wide<128>(mw, x, ldx, k, a, splits, s);
  }
}

kino_status kino_q8_cache_write(const kino_q8_cache* cache, const void* k, int64_t ld_k,
                                int64_t hs_k, const void* v, int64_t ld_v, int64_t hs_v,
                                const int32_t* token_starts, int64_t rows, void* stream) {
  kino_status st = check_q8_cache(cache, "kino_q8_cache_write");
  if (st != KINO_OK) return st;
  if (k == nullptr || v == nullptr) return fail(KINO_EINVAL, "kino_q8_cache_write: null");
  if (rows < 1 || rows > 0x3fffffffLL) return fail(KINO_EINVAL, "kino_q8_cache_write: rows");
  if (token_starts == nullptr && rows % cache->batch)
    return fail(KINO_EINVAL, "kino_q8_cache_write: %lld rows do not divide over %lld sequences",
                (long long)rows, (long long)cache->batch);
  if (ld_k % 8 || ld_v % 8 || hs_k % 8 || hs_v % 8 || !aligned16(k) || !aligned16(v))
    return fail(KINO_ENOTSUPPORTED, "kino_q8_cache_write: strides must be multiples of 8 with "
                "16-byte aligned operands");
  kino::Q8WriteArgs a;
  a.x[0] = static_cast<const __nv_bfloat16*>(k);
  a.x[1] = static_cast<const __nv_bfloat16*>(v);
  a.ld[0] = ld_k;
  a.ld[1] = ld_v;
  a.head_stride[0] = hs_k;
  a.head_stride[1] = hs_v;
  a.codes[0] = static_cast<uint8_t*>(cache->k_codes);
  a.codes[1] = static_cast<uint8_t*>(cache->v_codes);
  a.scales[0] = cache->k_scales;
  a.scales[1] = cache->v_scales;
  a.table = cache->table;
  a.ld_table = cache->ld_table;
  a.table_blocks = static_cast<int>(cache->table_blocks);
  a.lengths = cache->lengths;
  a.rows.starts = token_starts;
  a.rows.each = static_cast<int>(rows / cache->batch);
  a.rows.rows = rows;
  a.batch = static_cast<int>(cache->batch);
  a.heads = static_cast<int>(cache->heads);
  a.dim = static_cast<int>(cache->dim);
  a.block = static_cast<int>(cache->block);
  a.num_blocks = static_cast<int>(cache->num_blocks);
  a.block_shift = log2_block(cache->block);
  // n tokens fall into at most (n - 1) / block + 2 blocks (n >= 1)
  const int64_t block = cache->block, batch = cache->batch;
  const int64_t items = token_starts == nullptr
                            ? batch * ((rows / batch + block - 2) / block + 1)
                            : rows / block + 2 * std::min(batch, rows);
  if (items * cache->heads > 0x7fffffffLL)
    return fail(KINO_ENOTSUPPORTED, "kino_q8_cache_write: too many blocks");
  if (cache->format == KINO_Q8_INT8)
    launch_q8_write<kino::Q8_INT8>(a, items, static_cast<cudaStream_t>(stream));
  else
    launch_q8_write<kino::Q8_E4M3>(a, items, static_cast<cudaStream_t>(stream));
  return check_launch("kino_q8_cache_write");
}

kino_status kino_q8_cache_read(const kino_q8_cache* cache, void* k_out, void* v_out,
                               int64_t tokens, void* stream) {
  kino_status st = check_q8_cache(cache, "kino_q8_cache_read");
  if (st != KINO_OK) return st;
  if (k_out == nullptr || v_out == nullptr) return fail(KINO_EINVAL, "kino_q8_cache_read: null");
  if (!aligned16(k_out) || !aligned16(v_out))
    return fail(KINO_EINVAL, "kino_q8_cache_read: outputs not 16-byte aligned");
  if (tokens < 1) return fail(KINO_EINVAL, "kino_q8_cache_read: tokens");
  kino::Q8ReadArgs a;
  a.codes[0] = static_cast<const uint8_t*>(cache->k_codes);
  a.codes[1] = static_cast<const uint8_t*>(cache->v_codes);
  a.scales[0] = cache->k_scales;
  a.scales[1] = cache->v_scales;
  a.out[0] = static_cast<__nv_bfloat16*>(k_out);
  a.out[1] = static_cast<__nv_bfloat16*>(v_out);
  a.table = cache->table;
  a.ld_table = cache->ld_table;
  a.table_blocks = static_cast<int>(cache->table_blocks);
  a.lengths = cache->lengths;
  a.tokens = tokens;
  a.heads = static_cast<int>(cache->heads);
  a.dim = static_cast<int>(cache->dim);
  a.block = static_cast<int>(cache->block);
  a.num_blocks = static_cast<int>(cache->num_blocks);
  a.block_shift = log2_block(cache->block);
  const int64_t per_token = cache->heads * (cache->dim / 16);
  if (tokens > (0x7fffffffLL - 256) / per_token)
    return fail(KINO_ENOTSUPPORTED, "kino_q8_cache_read: shape too large");
  const dim3 grid(static_cast<unsigned>((tokens * per_token + 255) / 256),
                  static_cast<unsigned>(cache->batch));
  if (cache->format == KINO_Q8_INT8)
    launch_pdl(kino::q8_cache_read_kernel<kino::Q8_INT8>, grid, dim3(256), 0,
               static_cast<cudaStream_t>(stream), a);
  else
    launch_pdl(kino::q8_cache_read_kernel<kino::Q8_E4M3>, grid, dim3(256), 0,
               static_cast<cudaStream_t>(stream), a);
  return check_launch("kino_q8_cache_read");
}

int64_t kino_q8_attention_workspace_size(const kino_q8_cache* cache,
                                         const kino_q8_attention_args* args) {
  Q8AttnPlan p;
  return plan_q8_attention(cache, args, &p) == KINO_OK ? p.bytes : -1;
}

kino_status kino_q8_attention(const kino_q8_cache* cache, const kino_q8_attention_args* args,
                              void* stream) {
  Q8AttnPlan p;
  kino_status st = plan_q8_attention(cache, args, &p);
  if (st != KINO_OK) return st;
  if (args->q == nullptr || args->out == nullptr)
    return fail(KINO_EINVAL, "kino_q8_attention: null");
  if (args->ld_q % 8 || args->hs_q % 8 || args->ld_out % 8 || args->hs_out % 8 ||
      !aligned16(args->q) || !aligned16(args->out))
    return fail(KINO_ENOTSUPPORTED, "kino_q8_attention: strides must be multiples of 8 with "
                "16-byte aligned operands");
  if (!(args->scale >= 0.0f) || args->scale > 1e30f)
    return fail(KINO_EINVAL, "kino_q8_attention: scale %g", static_cast<double>(args->scale));
  if (args->workspace == nullptr || !aligned16(args->workspace) || args->workspace_bytes < p.bytes)
    return fail(KINO_EINVAL, "kino_q8_attention: %lld bytes of aligned workspace",
                (long long)p.bytes);
  kino::Q8Attn a;
  a.q = static_cast<const __nv_bfloat16*>(args->q);
  a.ld_q = args->ld_q;
  a.hs_q = args->hs_q;
  a.out = static_cast<__nv_bfloat16*>(args->out);
  a.ld_out = args->ld_out;
  a.hs_out = args->hs_out;
  a.codes[0] = static_cast<const uint8_t*>(cache->k_codes);
  a.codes[1] = static_cast<const uint8_t*>(cache->v_codes);
  a.scales[0] = cache->k_scales;
  a.scales[1] = cache->v_scales;
  a.table = cache->table;
  a.ld_table = cache->ld_table;
  a.table_blocks = static_cast<int>(cache->table_blocks);
  a.lengths = cache->lengths;
  a.rows.starts = args->token_starts;
  a.rows.each = static_cast<int>(args->rows / cache->batch);
  a.rows.rows = args->rows;
  a.batch = static_cast<int>(cache->batch);
  a.heads = static_cast<int>(cache->heads);
  a.group = static_cast<int>(args->q_heads / cache->heads);
  a.block = static_cast<int>(cache->block);
  a.num_blocks = static_cast<int>(cache->num_blocks);
  a.block_shift = log2_block(cache->block);
  a.scale_log2 = args->scale * 1.4426950408889634f;
  a.causal = args->causal != 0;
  a.tile_tokens = p.tile_tokens;
  a.tile_rows = p.tile_rows;
  a.runs = p.runs;
  a.part_o = static_cast<float*>(args->workspace);
  a.part_ml = a.part_o + 2LL * p.runs * p.tile_rows * cache->dim;
  a.starts = reinterpret_cast<kino::Q8RunStart*>(a.part_ml + 2LL * p.runs * p.tile_rows * 2);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool i8 = cache->format == KINO_Q8_INT8;
  if (cache->dim == 128)
    return i8 ? launch_q8_attention<128, kino::Q8_INT8>(cache, a, p.decode_tiles, s)
              : launch_q8_attention<128, kino::Q8_E4M3>(cache, a, p.decode_tiles, s);
  return i8 ? launch_q8_attention<64, kino::Q8_INT8>(cache, a, p.decode_tiles, s)
            : launch_q8_attention<64, kino::Q8_E4M3>(cache, a, p.decode_tiles, s);
}

}  // extern "C"
