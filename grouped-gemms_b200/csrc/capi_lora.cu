// C ABI of the low-rank adapters (see include/mxgg.h): argument checks and
// launches only; nothing synchronises or allocates.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/mxgg.h"
#include "host.cuh"
#include "lora.cuh"
#include "lora_rows.cuh"
#include "lora_tc.cuh"

namespace mxgg {
namespace {

constexpr int64_t kExtent = (int64_t)1 << 30;

int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }
int64_t v_bytes(int64_t M, int64_t R) { return M * 2 * lora_rp((int)R) * 2; }

bool out_type_ok(int t) { return t == MXGG_DTYPE_BF16 || t == MXGG_DTYPE_F16 || t == MXGG_DTYPE_F32; }

int lora_check(const char* what, const int32_t* offs, int64_t S, const int32_t* adapter, int64_t M, int64_t K,
               int64_t N, int64_t R, int64_t L) {
  if (M < 0 || K < 1 || N < 1 || R < 1 || L < 1 || S < 0)
    return fail(MXGG_ERR_INVALID, "%s: bad sizes (rows %lld, d_in %lld, d_out %lld, rank %lld, adapters %lld, "
                "segments %lld)", what, (long long)M, (long long)K, (long long)N, (long long)R, (long long)L,
                (long long)S);
  if (M >= kExtent || K >= kExtent || N >= kExtent || L >= kExtent || L * std::max(K, N) >= kExtent * 2)
    return fail(MXGG_ERR_UNSUPPORTED, "%s: extents beyond 2^30", what);
  if (L > 65535) return fail(MXGG_ERR_UNSUPPORTED, "%s: %lld adapters, at most 65535", what, (long long)L);
  if (R > kMaxLoraRank || R % 8 != 0)
    return fail(MXGG_ERR_UNSUPPORTED, "%s: rank %lld: multiples of 8 up to %d", what, (long long)R, kMaxLoraRank);
  if (K % 8 != 0 || N % 8 != 0)
    return fail(MXGG_ERR_UNSUPPORTED, "%s: d_in %lld and d_out %lld must be multiples of 8", what, (long long)K,
                (long long)N);
  if (offs) {
    if (S > kMaxLoraSegments)
      return fail(MXGG_ERR_UNSUPPORTED, "%s: %lld segments, at most %d", what, (long long)S, kMaxLoraSegments);
    if (!adapter && S > L)
      return fail(MXGG_ERR_INVALID, "%s: %lld segments need an adapter map for %lld adapters", what, (long long)S,
                  (long long)L);
  } else {
    if (S != M) return fail(MXGG_ERR_INVALID, "%s: without offsets every row is a segment", what);
    if (!adapter && S > 0) return fail(MXGG_ERR_INVALID, "%s: rows without offsets need their adapters", what);
  }
  return MXGG_OK;
}

int rows_check(const char* what, const char* name, const void* p, int64_t ld, int64_t cols, int64_t M, int es) {
  if (M == 0) return MXGG_OK;
  if (!p) return fail(MXGG_ERR_INVALID, "%s: null %s", what, name);
  if (ld < cols || (ld * es) % 16 != 0 || !aligned(p, 16))
    return fail(MXGG_ERR_INVALID, "%s: %s rows must be 16-byte aligned and not overlap (row stride %lld of %lld "
                "elements)", what, name, (long long)ld, (long long)cols);
  return MXGG_OK;
}

int out_es(int t) { return t == MXGG_DTYPE_F32 ? 4 : 2; }

constexpr CUtensorMapDataType kBf16Map = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
constexpr CUtensorMapSwizzle kSwz = CU_TENSOR_MAP_SWIZZLE_128B;

// Shared memory of a CTA's ring and tables, at most: two CTAs to an SM, and one.
// A stage of the shrink is 32 KB at most, so it has three; the expand's tiles of
// v count too.
constexpr int kShrinkSmem = 96 * 1024;
static_assert(kShrinkSmem / (kShrinkXBytes + kMaxLoraRank * 128) >= 3, "stages of the shrink");
constexpr int kExpandPairSmem = 98 * 1024, kExpandSmem = 212 * 1024;
constexpr int kWgradSmem = 108 * 1024;

int run_shrink(DeviceState* st, const LoraSegs& g, const void* x, int64_t ld, const void* w, int r_contig,
               const float* scaling, int64_t C, int64_t R, void* v, cudaStream_t stream) {
  ShrinkParams p{};
  p.g = g;
  p.scaling = scaling;
  p.C = (int)C;
  p.R = (int)R;
  p.Rp = lora_rp((int)R);
  p.r_contig = r_contig;
  p.w_bytes = r_contig ? ((int)R + 63) / 64 * kLoraBK * 128 : p.Rp * 128;
  p.v = static_cast<__nv_bfloat16*>(v);
  p.status = st->status;
  p.wait_ns = wait_limit_ns();
  const long long tiles = ((long long)g.M + kLoraBM - 1) / kLoraBM + std::min(g.S, g.M) - 1;
  const int kiters = (int)((C + kLoraBK - 1) / kLoraBK);
  // Split the contraction until the CTAs cover the SMs, each keeping 4 stages of work.
  p.ksplit = 1;
  while (p.ksplit < 8 && tiles * p.ksplit < st->num_sms && kiters / (2 * p.ksplit) >= 4) p.ksplit *= 2;
  // two CTAs share an SM
  const int stage = kShrinkXBytes + p.w_bytes;
  p.stages = std::min(kShrinkMaxStages, kShrinkSmem / stage);
  const size_t smem = (size_t)p.stages * stage + 1024;
  CUtensorMap mx, mx32, mw;
  if (int rc = make_tmap_2d(&mx, x, kBf16Map, 2, (uint64_t)g.M, (uint64_t)C, (uint64_t)ld, kLoraBK, kLoraBM, kSwz))
    return rc;
  if (int rc = make_tmap_2d(&mx32, x, kBf16Map, 2, (uint64_t)g.M, (uint64_t)C, (uint64_t)ld, kLoraBK, 32, kSwz))
    return rc;
  if (int rc = r_contig ? make_tmap_3d(&mw, w, kBf16Map, 2, (uint64_t)g.L, (uint64_t)C, (uint64_t)R, (uint64_t)R,
                                       (uint64_t)(C * R), 64, kLoraBK, 1, kSwz)
                        : make_tmap_3d(&mw, w, kBf16Map, 2, (uint64_t)g.L, (uint64_t)R, (uint64_t)C, (uint64_t)C,
                                       (uint64_t)(C * R), kLoraBK, (uint32_t)p.Rp, 1, kSwz))
    return rc;
  if (int rc = allow_smem<lora_shrink_kernel>(*st, kShrinkSmem + 1024)) return rc;
  MXGG_CUDA_TRY(launch(lora_shrink_kernel, dim3((unsigned)(tiles * p.ksplit)), dim3(128), smem, p.ksplit, false, stream,
                       mx, mx32, mw, p));
  return MXGG_OK;
}

CUtensorMapDataType map_type(int dtype) {
  return dtype == MXGG_DTYPE_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
         : dtype == MXGG_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                   : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

// v (M, 2, Rp): `rows` rows of both halves side by side when they fit 64
// columns (lora_v_pieces), else of 64 columns of one half (zeros past Rp)
int make_v_map(CUtensorMap* m, const void* v, int M, int Rp, int rows) {
  if (lora_v_pieces(Rp) == 1)
    return make_tmap_3d(m, v, kBf16Map, 2, (uint64_t)M, 1, (uint64_t)(2 * Rp), (uint64_t)(2 * Rp), (uint64_t)(2 * Rp),
                        64, 1, (uint32_t)rows, kSwz);
  return make_tmap_3d(m, v, kBf16Map, 2, (uint64_t)M, 2, (uint64_t)Rp, (uint64_t)Rp, (uint64_t)(2 * Rp), 64, 1,
                      (uint32_t)rows, kSwz);
}

template <typename O>
int expand_as(DeviceState* st, const LoraSegs& g, const void* v, const void* w, int r_contig, const void* base,
              int64_t base_ld, void* out, int64_t out_ld, int out_dtype, int64_t C, int64_t R, bool more,
              cudaStream_t stream) {
  ExpandParams p{};
  p.more = more;
  p.g = g;
  p.C = (int)C;
  p.Rp = lora_rp((int)R);
  p.r_contig = r_contig;
  const int rc = (p.Rp + 63) / 64, es = out_es(out_dtype);
  p.base_bytes = kLoraBM * kExpandBN * es;
  p.w_row = p.Rp <= 16 ? 32 : p.Rp <= 32 ? 64 : 128;
  p.w_bytes = r_contig ? rc * kExpandBN * p.w_row : p.Rp * 128;
  p.v_pieces = lora_v_pieces(p.Rp);
  p.base = base;
  p.base_ld = base_ld;
  p.out = out;
  p.out_ld = out_ld;
  p.status = st->status;
  p.wait_ns = wait_limit_ns();
  const long long tiles = ((long long)g.M + kLoraBM - 1) / kLoraBM + std::min(g.S, g.M) - 1;
  const int nt = (int)((C + kExpandBN - 1) / kExpandBN);
  // Cut the columns until two CTAs to an SM fill the GPU once, each keeping two tiles (v is loaded once per CTA).  Where
  // one fits (fp32 results; 16-bit ones above rank 32, grad_x above 48) they come in two rounds.
  p.nsplit = (int)std::max<long long>(1, std::min<long long>((nt + 1) / 2, 2LL * st->num_sms / tiles));
  const int vb = p.v_pieces * kLoraBM * 128, stage = p.base_bytes + p.w_bytes;
  // two CTAs share an SM where that leaves each three stages
  const int pair = (kExpandPairSmem - vb) / stage;
  p.stages = std::min(kExpandMaxStages, pair >= 3 ? pair : (kExpandSmem - vb) / stage);
  const size_t smem = (size_t)vb + (size_t)p.stages * stage + 1024;
  CUtensorMap mv, mw, mb, mb32, mo;
  if (int rc2 = make_v_map(&mv, v, g.M, p.Rp, kLoraBM)) return rc2;
  if (int rc2 = r_contig ? make_tmap_3d(&mw, w, kBf16Map, 2, (uint64_t)g.L, (uint64_t)C, (uint64_t)R, (uint64_t)R,
                                        (uint64_t)(C * R), (uint32_t)p.w_row / 2, kExpandBN, 1,
                                        p.w_row == 32   ? CU_TENSOR_MAP_SWIZZLE_32B
                                        : p.w_row == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                        : kSwz)
                         : make_tmap_3d(&mw, w, kBf16Map, 2, (uint64_t)g.L, (uint64_t)R, (uint64_t)C, (uint64_t)C,
                                        (uint64_t)(C * R), kExpandBN, (uint32_t)p.Rp, 1, kSwz))
    return rc2;
  if (int rc2 = make_tmap_2d(&mo, out, map_type(out_dtype), es, (uint64_t)g.M, (uint64_t)C, (uint64_t)out_ld,
                             (uint32_t)(128 / es), 32, kSwz))
    return rc2;
  mb = mb32 = mo;
  if (base) {
    if (int rc2 = make_tmap_2d(&mb, base, map_type(out_dtype), es, (uint64_t)g.M, (uint64_t)C, (uint64_t)base_ld,
                               (uint32_t)(128 / es), kLoraBM, kSwz))
      return rc2;
    if (base != out)
      if (int rc2 = make_tmap_2d(&mb32, base, map_type(out_dtype), es, (uint64_t)g.M, (uint64_t)C, (uint64_t)base_ld,
                                 (uint32_t)(128 / es), 32, kSwz))
        return rc2;
  }
  if (int rc2 = allow_smem<lora_expand_kernel<O>>(*st, kExpandSmem + 1024)) return rc2;
  MXGG_CUDA_TRY(launch(lora_expand_kernel<O>, dim3((unsigned)(tiles * p.nsplit)), dim3(kExpandThreads), smem, 1, true,
                       stream, mv, mw, mb, mb32, mo, p));
  return MXGG_OK;
}

int run_expand(DeviceState* st, const LoraSegs& g, const void* v, const void* w, int r_contig, const void* base,
               int64_t base_ld, void* out, int64_t out_ld, int out_dtype, int64_t C, int64_t R, bool more,
               cudaStream_t stream) {
  auto f = out_dtype == MXGG_DTYPE_BF16  ? expand_as<__nv_bfloat16>
           : out_dtype == MXGG_DTYPE_F16 ? expand_as<__half>
                                         : expand_as<float>;
  return f(st, g, v, w, r_contig, base, base_ld, out, out_ld, out_dtype, C, R, more, stream);
}

// Launch shape of the weight gradients: no more CTAs than there are stages.
// kWgradMaxCtas, not the device's SMs: the workspace query has no device.
struct WgradPlan {
  int64_t ctas, bytes;   // CTAs; the partials' size
};
int64_t wgrad_tiles(int64_t C) { return (C + kWgradBC - 1) / kWgradBC; }
WgradPlan wgrad_plan(int64_t M, int64_t C, int64_t R, int64_t L, int64_t S) {
  WgradPlan w;
  const int64_t tiles = wgrad_tiles(C);
  const int64_t stages = M > 0 && S > 0 ? ((M + kWgradBT - 1) / kWgradBT + std::min(S, M) - 1) * tiles : 0;
  w.ctas = std::min<int64_t>(stages, kWgradMaxCtas);
  w.bytes = align256(stages > 0 ? (tiles * wgrad_slots((int)L, (int)S) + w.ctas) * kWgradBC * lora_rp((int)R) * 4 : 0);
  return w;
}

struct WgradArgs {
  const void *v, *z;
  int64_t ld, C;
  int transposed;
  void* out;
};

// One or two weight gradients: the partials, then their sums.
int run_wgrad(DeviceState* st, const LoraSegs& g, const WgradArgs* jobs, int n, int64_t R, int out_dtype, uint8_t* part,
              bool pdl, cudaStream_t stream) {
  WgradParams p{};
  p.g = g;
  p.R = (int)R;
  p.Rp = lora_rp((int)R);
  p.status = st->status;
  p.wait_ns = wait_limit_ns();
  const int stage = kWgradZBytes + lora_v_pieces(p.Rp) * kWgradBT * 128;
  const int tables = wgrad_table_bytes(g.S);
  p.stages = std::min(kWgradMaxStages, (kWgradSmem - tables) / stage);   // two CTAs to an SM
  const size_t smem = (size_t)p.stages * stage + tables + 1024;
  CUtensorMap mv[2], mz[2];
  long long sum_blocks = 0;
  int ctas = 0;
  for (int i = 0; i < n; ++i) {
    p.job[i].C = (int)jobs[i].C;
    p.job[i].ctiles = (int)wgrad_tiles(jobs[i].C);
    p.job[i].transposed = jobs[i].transposed;
    p.job[i].out = jobs[i].out;
    const WgradPlan w = wgrad_plan(g.M, jobs[i].C, R, g.L, g.S);
    p.job[i].ctas = (int)w.ctas;
    p.job[i].part = reinterpret_cast<float*>(part);
    part += w.bytes;
    ctas = std::max(ctas, p.job[i].ctas);
    sum_blocks += (jobs[i].C + wgrad_sum_cols(p.Rp) - 1) / wgrad_sum_cols(p.Rp);
    if (int rc = make_v_map(&mv[i], jobs[i].v, g.M, p.Rp, kWgradBT)) return rc;
    if (int rc = make_tmap_2d(&mz[i], jobs[i].z, kBf16Map, 2, (uint64_t)g.M, (uint64_t)jobs[i].C,
                              (uint64_t)jobs[i].ld, 64, kWgradBT, kSwz))
      return rc;
  }
  if (n == 1) {
    mv[1] = mv[0];
    mz[1] = mz[0];
  }
  if (int rc = allow_smem<lora_wgrad_kernel>(*st, kWgradSmem + 1024)) return rc;
  MXGG_CUDA_TRY(launch(lora_wgrad_kernel, dim3((unsigned)ctas), dim3(kWgradThreads), smem, 1, pdl, stream, mv[0],
                       mz[0], mv[1], mz[1], p));
  auto k = out_dtype == MXGG_DTYPE_BF16  ? lora_wgrad_sum_kernel<__nv_bfloat16>
           : out_dtype == MXGG_DTYPE_F16 ? lora_wgrad_sum_kernel<__half>
                                         : lora_wgrad_sum_kernel<float>;
  const size_t sum_smem = (size_t)wgrad_sum_cols(p.Rp) * (p.Rp + 1) * 4 + (size_t)(2 * g.S + 2) * 4;   // below 48 KB
  MXGG_CUDA_TRY(launch(k, dim3((unsigned)sum_blocks, (unsigned)g.L), dim3(256), sum_smem, 1, true, stream, p));
  return MXGG_OK;
}

constexpr int64_t kRowsFew = 4;

// Single rows always take the 16-row clusters.  Of segments, measured against
// 128-row tiles (5120 -> 8192, 8192 -> 5120 and 2048 -> 2048, ranks 16 to 128):
// a cluster's weights come once per 16 rows, a tile's once per 128, but tiles
// are two launches of few CTAs.  Up to 64 rows the clusters win always (11 us
// against 15 for rank 16), beyond 256 never (23 against 16 us at 512 rows);
// between, when segments are short (256 rows in 8: 25 against 31 us for rank 64)
// or the rank is small (256 rows in one: 15.1 against 15.4 us for rank 16, but
// 26 against 19 us for rank 64).
bool rows_form(const int32_t* offs, int64_t S, int64_t M, int64_t R) {
  if (!offs || M <= 64) return true;
  return M <= 256 && (M <= 32 * S || M * lora_rp((int)R) <= 8192);
}

constexpr int rows_threads(int KC, int wanted) { return KC <= 4 ? wanted : 256; }
constexpr int rows_smem(int threads, int Rp) { return threads / 32 * kRowsGroup * rows_red_ld(Rp) * 4; }

template <typename O, int KC>
int rows_launch(const DeviceState& st, RowsParams p, cudaStream_t stream) {
  auto k = lora_rows_kernel<O, KC>;
  const int threads = rows_threads(KC, p.threads);
  const size_t smem = rows_smem(threads, p.Rp);
  if (int rc = allow_smem<lora_rows_kernel<O, KC>>(st, rows_smem(rows_threads(KC, kRowsMaxThreads), 16 * KC), true))
    return rc;
  if (p.cluster > 8) {
    // a device (or a slice of one) without 16 free SMs in a GPC takes clusters of 8
    const cudaError_t e = launch(k, dim3((unsigned)p.g.M * (unsigned)p.cluster), dim3(threads), smem, p.cluster, false,
                                 stream, p);
    if (e == cudaSuccess) return MXGG_OK;
    if (e != cudaErrorInvalidClusterSize) return fail(MXGG_ERR_CUDA, "mxgg_lora_mm: %s", cudaGetErrorString(e));
    cudaGetLastError();
    p.cluster = 8;
  }
  MXGG_CUDA_TRY(launch(k, dim3((unsigned)p.g.M * (unsigned)p.cluster), dim3(threads), smem, p.cluster, false, stream, p));
  return MXGG_OK;
}

template <typename O>
int rows_as(const DeviceState& st, const RowsParams& p, cudaStream_t stream) {
  return p.Rp <= 16   ? rows_launch<O, 1>(st, p, stream)
         : p.Rp <= 32 ? rows_launch<O, 2>(st, p, stream)
         : p.Rp <= 64 ? rows_launch<O, 4>(st, p, stream)
                      : rows_launch<O, 8>(st, p, stream);
}

}  // namespace
}  // namespace mxgg

using namespace mxgg;

extern "C" {

int64_t mxgg_lora_v_bytes(int64_t M, int64_t R) {
  if (M < 0 || M >= kExtent || R < 1 || R > kMaxLoraRank || R % 8 != 0) return -1;
  return v_bytes(M, R);
}

int mxgg_lora_mm(const void* x, int64_t x_ld, const void* a, const void* b, const int32_t* segment_end_offsets,
                 int64_t n_segments, const int32_t* segment_adapter, const float* scaling, const void* base,
                 int64_t base_ld, void* out, int64_t out_ld, int out_dtype, int64_t M, int64_t K, int64_t N, int64_t R,
                 int64_t L, void* v, void* stream_v) {
  const char* what = "mxgg_lora_mm";
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (int rc = lora_check(what, segment_end_offsets, n_segments, segment_adapter, M, K, N, R, L)) return rc;
  if (!out_type_ok(out_dtype)) return fail(MXGG_ERR_INVALID, "%s: unknown out_dtype %d", what, out_dtype);
  if (M == 0 || n_segments == 0) return MXGG_OK;
  if (int rc = rows_check(what, "x", x, x_ld, K, M, 2)) return rc;
  if (int rc = rows_check(what, "out", out, out_ld, N, M, out_es(out_dtype))) return rc;
  if (base) {
    if (int rc = rows_check(what, "base", base, base_ld, N, M, out_es(out_dtype))) return rc;
    if (base == out && base_ld != out_ld)
      return fail(MXGG_ERR_INVALID, "%s: base is out, with another row stride", what);
  }
  if (!segment_end_offsets && M > ((int64_t)1 << 27))
    return fail(MXGG_ERR_UNSUPPORTED, "%s: more than 2^27 single rows", what);
  if (!a || !b || (!v && segment_end_offsets) || !aligned(a, 16) || !aligned(b, 16) || !aligned(v, 16))
    return fail(MXGG_ERR_INVALID, "%s: a, b and v must be 16-byte aligned", what);
  DeviceState* st = nullptr;
  if (int rc = get_device_state(&st)) return rc;
  const LoraSegs g{segment_end_offsets, segment_adapter, (int)n_segments, (int)L, (int)M};
  if (rows_form(segment_end_offsets, n_segments, M, R)) {
    RowsParams p{};
    p.g = g;
    p.x = static_cast<const __nv_bfloat16*>(x);
    p.x_ld = x_ld;
    p.a = static_cast<const __nv_bfloat16*>(a);
    p.b = static_cast<const __nv_bfloat16*>(b);
    p.scaling = scaling;
    p.base = base;
    p.base_ld = base_ld;
    p.out = out;
    p.out_ld = out_ld;
    p.v = static_cast<__nv_bfloat16*>(v);
    p.K = (int)K;
    p.N = (int)N;
    p.R = (int)R;
    p.Rp = lora_rp((int)R);
    // a few rows: more CTAs and warps for each, as there is nothing else to fill the GPU with
    p.cluster = M <= kRowsFew ? 16 : 8;
    p.threads = M <= kRowsFew ? 512 : 256;
    switch (out_dtype) {
      case MXGG_DTYPE_BF16: return rows_as<__nv_bfloat16>(*st, p, stream);
      case MXGG_DTYPE_F16: return rows_as<__half>(*st, p, stream);
      default: return rows_as<float>(*st, p, stream);
    }
  }
  if (int rc = run_shrink(st, g, x, x_ld, a, 0, scaling, K, R, v, stream)) return rc;
  return run_expand(st, g, v, b, 1, base, base_ld, out, out_ld, out_dtype, N, R, false, stream);
}

int64_t mxgg_lora_mm_backward_workspace_size(int64_t M, int64_t K, int64_t N, int64_t R, int64_t L,
                                             int64_t n_segments) {
  if (M < 0 || M >= kExtent || K < 1 || N < 1 || R < 1 || R > kMaxLoraRank || R % 8 != 0 || L < 1 || n_segments < 0 ||
      K >= kExtent || N >= kExtent || L >= kExtent || n_segments > kMaxLoraSegments)
    return -1;
  return align256(v_bytes(M, R)) + wgrad_plan(M, K, R, L, n_segments).bytes +
         wgrad_plan(M, N, R, L, n_segments).bytes;
}

int mxgg_lora_mm_backward(const void* grad_out, int64_t grad_out_ld, const void* x, int64_t x_ld, const void* a,
                          const void* b, const void* v, const int32_t* segment_end_offsets, int64_t n_segments,
                          const int32_t* segment_adapter, const float* scaling, const void* grad_base,
                          int64_t grad_base_ld, void* grad_x, int64_t grad_x_ld, int grad_x_dtype, void* grad_a,
                          void* grad_b, int grad_w_dtype, int64_t M, int64_t K, int64_t N, int64_t R, int64_t L,
                          void* workspace, int64_t workspace_bytes, void* stream_v) {
  const char* what = "mxgg_lora_mm_backward";
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (int rc = lora_check(what, segment_end_offsets, n_segments, segment_adapter, M, K, N, R, L)) return rc;
  if (!segment_end_offsets) return fail(MXGG_ERR_UNSUPPORTED, "%s: the gradients take segments, not rows", what);
  if (!out_type_ok(grad_x_dtype) || !out_type_ok(grad_w_dtype))
    return fail(MXGG_ERR_INVALID, "%s: unknown dtype (%d, %d)", what, grad_x_dtype, grad_w_dtype);
  if (!grad_x && !grad_a && !grad_b) return fail(MXGG_ERR_INVALID, "%s: no gradient asked for", what);
  if (int rc = rows_check(what, "grad_out", grad_out, grad_out_ld, N, M, 2)) return rc;
  if (grad_a)
    if (int rc = rows_check(what, "x", x, x_ld, K, M, 2)) return rc;
  if (grad_x) {
    if (int rc = rows_check(what, "grad_x", grad_x, grad_x_ld, K, M, out_es(grad_x_dtype))) return rc;
    if (grad_base) {
      if (int rc = rows_check(what, "grad_base", grad_base, grad_base_ld, K, M, out_es(grad_x_dtype))) return rc;
      if (grad_base == grad_x && grad_base_ld != grad_x_ld)
        return fail(MXGG_ERR_INVALID, "%s: grad_base is grad_x, with another row stride", what);
    }
  }
  if (!a || !b || !aligned(a, 16) || !aligned(b, 16) || !aligned(v, 16) || (M > 0 && grad_b && !v) ||
      !aligned(grad_a, 16) || !aligned(grad_b, 16))
    return fail(MXGG_ERR_INVALID, "%s: a, b, v, grad_a and grad_b must be 16-byte aligned", what);
  const int64_t need = mxgg_lora_mm_backward_workspace_size(M, K, N, R, L, n_segments);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 256)))
    return fail(MXGG_ERR_INVALID, "%s: workspace of %lld bytes (256-byte aligned) required", what, (long long)need);
  DeviceState* st = nullptr;
  if (int rc = get_device_state(&st)) return rc;
  const int64_t wb = out_es(grad_w_dtype) * L * R;
  if (M == 0 || n_segments == 0) {
    if (grad_a) MXGG_CUDA_TRY(cudaMemsetAsync(grad_a, 0, (size_t)(wb * K), stream));
    if (grad_b) MXGG_CUDA_TRY(cudaMemsetAsync(grad_b, 0, (size_t)(wb * N), stream));
    return MXGG_OK;
  }
  const LoraSegs g{segment_end_offsets, segment_adapter, (int)n_segments, (int)L, (int)M};
  uint8_t* dv = static_cast<uint8_t*>(workspace);
  // Each launch but the first is programmatic: what it reads before its wait
  // (offsets, adapters, weights, bases) was complete when the first started.
  bool pdl = false;
  if (grad_x || grad_a) {
    if (int rc = run_shrink(st, g, grad_out, grad_out_ld, b, 1, scaling, N, R, dv, stream)) return rc;
    pdl = true;
  }
  if (grad_x)
    if (int rc = run_expand(st, g, dv, a, 0, grad_base, grad_base_ld, grad_x, grad_x_ld, grad_x_dtype, K, R,
                            grad_a || grad_b, stream))
      return rc;
  WgradArgs jobs[2];
  int n = 0;
  if (grad_a) jobs[n++] = WgradArgs{dv, x, x_ld, K, 0, grad_a};
  if (grad_b) jobs[n++] = WgradArgs{v, grad_out, grad_out_ld, N, 1, grad_b};
  if (n) return run_wgrad(st, g, jobs, n, R, grad_w_dtype, dv + align256(v_bytes(M, R)), pdl, stream);
  return MXGG_OK;
}

}  // extern "C"
