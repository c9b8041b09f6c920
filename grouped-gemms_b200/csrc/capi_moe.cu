// C ABI of the routed layer's operators (see include/mxgg.h): router, dispatch
// plan, gradients of the combine and the dispatch.  Argument checks and
// launches only; nothing synchronises or allocates.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/mxgg.h"
#include "host.cuh"
#include "moe_grad.cuh"
#include "router.cuh"

namespace mxgg {
namespace {

constexpr int64_t kExtent = (int64_t)1 << 30;

// Launch shape of route_topk: blocks of 4 warps until every SM has one, of 16
// (fewer partials to add) beyond that.  kRouteSms, not the device's count: the
// workspace query has no device.
constexpr int kRouteSms = 148;
int route_lanes(int64_t E) {   // lanes per token
  int g = 1;
  while (g < 32 && g * 8 < E) g *= 2;
  return g;
}
struct RouteShape {
  int warps, blocks;
};
RouteShape route_shape(int64_t T, int64_t E) {
  const int64_t groups = 32 / route_lanes(E), warps = (T + groups - 1) / groups;
  RouteShape s;
  s.warps = warps > 4 * kRouteSms ? 16 : 4;
  s.blocks = (int)std::max<int64_t>(1, std::min<int64_t>((warps + s.warps - 1) / s.warps, 2 * kRouteSms));
  return s;
}

struct RouteWs {
  int64_t p, c, z, n, total;   // byte offsets, size
};
RouteWs route_ws(int64_t T, int64_t E) {
  const int64_t blocks = route_shape(T, E).blocks;
  RouteWs w;
  w.p = 0;
  w.c = w.p + blocks * E * 4;
  w.z = w.c + blocks * E * 4;
  w.n = w.z + blocks * 4;
  w.total = w.n + blocks * 4;
  return w;
}

int route_check(const char* what, int dtype, int64_t ld, int64_t T, int64_t E, int64_t k) {
  if (dtype != MXGG_DTYPE_BF16 && dtype != MXGG_DTYPE_F16 && dtype != MXGG_DTYPE_F32)
    return fail(MXGG_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
  if (T < 0 || E < 1 || k < 1 || k > E || ld < E)
    return fail(MXGG_ERR_INVALID, "%s: bad sizes (tokens %lld, experts %lld, k %lld, row stride %lld)", what,
                (long long)T, (long long)E, (long long)k, (long long)ld);
  if (E > kMaxRouteExperts || k > kMaxRouteK)
    return fail(MXGG_ERR_UNSUPPORTED, "%s: at most %d experts and k %d", what, kMaxRouteExperts, kMaxRouteK);
  if (T >= kExtent) return fail(MXGG_ERR_UNSUPPORTED, "%s: extents beyond 2^30", what);
  return MXGG_OK;
}

// 16-byte rows: base, row stride and length all multiples of 16 bytes
bool route_vec(const void* p, int64_t ld, int64_t E, int es) {
  return aligned(p, 16) && (ld * es) % 16 == 0 && (E * es) % 16 == 0;
}

template <typename T, int G, int V>
int launch_route(const RouteParams& p, int, cudaStream_t stream) {
  const RouteShape s = route_shape(p.T, p.E);
  route_topk_kernel<T, G, V><<<s.blocks, s.warps * 32, 0, stream>>>(p);
  MXGG_CUDA_TRY(cudaGetLastError());
  if (s.blocks > 1) {
    const int ctas = p.E > 32 ? kRouteFinishCtas : 1;
    MXGG_CUDA_TRY(launch(route_finish_kernel, dim3(ctas), dim3(1024), 0, ctas, true, stream, p, s.blocks));
  }
  return MXGG_OK;
}

template <typename T, int G, int V>
int launch_route_grad(const RouteGradParams& p, int num_sms, cudaStream_t stream) {
  constexpr int kGroups = 32 / G;
  const long long warps = (p.T + kGroups - 1) / kGroups;
  const int nw = warps > 4LL * num_sms ? 8 : 4;
  const int blocks = (int)std::max(1LL, std::min<long long>((warps + nw - 1) / nw, (long long)num_sms * 8));
  route_grad_kernel<T, G, V><<<blocks, nw * 32, 0, stream>>>(p);
  MXGG_CUDA_TRY(cudaGetLastError());
  return MXGG_OK;
}

// Lanes per token (G) and elements per lane (V): V stays at 8 while 32 lanes
// hold the row, so a row of 16-bit logits is one 16-byte load per lane.
#define MXGG_ROUTE_PICK(FN, TYPE)                              \
  (E <= 8     ? FN<TYPE, 1, 8>(p, sms, stream)                 \
   : E <= 16  ? FN<TYPE, 2, 8>(p, sms, stream)                 \
   : E <= 32  ? FN<TYPE, 4, 8>(p, sms, stream)                 \
   : E <= 64  ? FN<TYPE, 8, 8>(p, sms, stream)                 \
   : E <= 128 ? FN<TYPE, 16, 8>(p, sms, stream)                \
   : E <= 256 ? FN<TYPE, 32, 8>(p, sms, stream)                \
   : E <= 512 ? FN<TYPE, 32, 16>(p, sms, stream)               \
              : FN<TYPE, 32, 32>(p, sms, stream))

template <typename T>
int route_for(int64_t E, const RouteParams& p, int sms, cudaStream_t stream) {
  return MXGG_ROUTE_PICK(launch_route, T);
}
template <typename T>
int route_grad_for(int64_t E, const RouteGradParams& p, int sms, cudaStream_t stream) {
  return MXGG_ROUTE_PICK(launch_route_grad, T);
}
#undef MXGG_ROUTE_PICK

// Threads for a row of N bf16 elements, 8 to a thread and round: whole warps, rounds of even length.
unsigned row_threads(int64_t N) {
  const int64_t pieces = std::max<int64_t>(1, N / 8), rounds = (pieces + 255) / 256;
  return (unsigned)(((pieces + rounds - 1) / rounds + 31) / 32 * 32);
}

// Pairs per block of a dispatch plan: enough blocks to fill the GPU, chunks of at least 2048 pairs.
constexpr int kPlanMaxBlocks = 148;
int plan_per(int64_t pairs) {
  const int64_t per = std::max<int64_t>(2048, (pairs + kPlanMaxBlocks - 1) / kPlanMaxBlocks);
  return (int)((per + kPlanThreads - 1) / kPlanThreads * kPlanThreads);
}

}  // namespace
}  // namespace mxgg

using namespace mxgg;

extern "C" {

int64_t mxgg_route_workspace_size(int64_t tokens, int64_t experts) {
  if (tokens < 0 || tokens >= kExtent || experts < 1 || experts > kMaxRouteExperts) return -1;
  return route_ws(tokens, experts).total;
}

int mxgg_route_topk(const void* logits, int dtype, int64_t ld, const uint8_t* mask, int64_t tokens, int64_t experts,
                    int32_t k, int32_t renormalise, int32_t* chosen, float* weights, float* stats, int32_t* counts,
                    float* losses, int32_t* n_counted, void* workspace, int64_t workspace_bytes, void* stream_v) {
  const char* what = "mxgg_route_topk";
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (int rc = route_check(what, dtype, ld, tokens, experts, k)) return rc;
  if (!counts || !losses || !n_counted || (tokens > 0 && (!logits || !chosen || !weights || !stats)))
    return fail(MXGG_ERR_INVALID, "%s: null pointer", what);
  const RouteWs ws = route_ws(tokens, experts);
  if (!workspace || workspace_bytes < ws.total || !aligned(workspace, 16))
    return fail(MXGG_ERR_INVALID, "%s: workspace of %lld bytes (16-byte aligned) required", what, (long long)ws.total);
  if (!aligned(stats, 8)) return fail(MXGG_ERR_INVALID, "%s: stats must be 8-byte aligned", what);
  DeviceState* st = nullptr;
  if (int rc = get_device_state(&st)) return rc;
  RouteParams p{};
  p.logits = logits;
  p.ld = ld;
  p.mask = mask;
  p.T = (int)tokens;
  p.E = (int)experts;
  p.k = k;
  p.renormalise = renormalise ? 1 : 0;
  p.experts = chosen;
  p.weights = weights;
  p.stats = reinterpret_cast<float2*>(stats);
  p.counts = counts;
  p.losses = losses;
  p.tokens = n_counted;
  uint8_t* w = static_cast<uint8_t*>(workspace);
  p.part_p = reinterpret_cast<float*>(w + ws.p);
  p.part_c = reinterpret_cast<int32_t*>(w + ws.c);
  p.part_z = reinterpret_cast<float*>(w + ws.z);
  p.part_n = reinterpret_cast<int32_t*>(w + ws.n);
  p.vec = route_vec(logits, ld, experts, dtype == MXGG_DTYPE_F32 ? 4 : 2);
  switch (dtype) {
    case MXGG_DTYPE_BF16: return route_for<__nv_bfloat16>(experts, p, st->num_sms, stream);
    case MXGG_DTYPE_F16: return route_for<__half>(experts, p, st->num_sms, stream);
    default: return route_for<float>(experts, p, st->num_sms, stream);
  }
}

int mxgg_route_topk_backward(const void* logits, int dtype, int64_t ld, int64_t tokens, int64_t experts, int32_t k,
                             int32_t renormalise, const int32_t* chosen, const float* weights, const float* stats,
                             const int32_t* counts, const int32_t* n_counted, const float* grad_weights,
                             const float* grad_balance, float balance_coef, const float* grad_z, float z_coef,
                             void* grad_logits, void* stream_v) {
  const char* what = "mxgg_route_topk_backward";
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (int rc = route_check(what, dtype, ld, tokens, experts, k)) return rc;
  if (tokens == 0) return MXGG_OK;
  if (!logits || !chosen || !weights || !stats || !counts || !n_counted || !grad_logits)
    return fail(MXGG_ERR_INVALID, "%s: null pointer", what);
  if (!aligned(stats, 8)) return fail(MXGG_ERR_INVALID, "%s: stats must be 8-byte aligned", what);
  DeviceState* st = nullptr;
  if (int rc = get_device_state(&st)) return rc;
  RouteGradParams p{};
  p.logits = logits;
  p.ld = ld;
  p.T = (int)tokens;
  p.E = (int)experts;
  p.k = k;
  p.renormalise = renormalise ? 1 : 0;
  p.experts = chosen;
  p.weights = weights;
  p.stats = reinterpret_cast<const float2*>(stats);
  p.counts = counts;
  p.tokens = n_counted;
  p.grad_w = grad_weights;
  p.grad_bal = grad_balance;
  p.grad_z = grad_z;
  p.bal_coef = balance_coef;
  p.z_coef = z_coef;
  p.grad = grad_logits;
  const int es = dtype == MXGG_DTYPE_F32 ? 4 : 2;
  p.vec = route_vec(logits, ld, experts, es) && route_vec(grad_logits, experts, experts, es);
  switch (dtype) {
    case MXGG_DTYPE_BF16: return route_grad_for<__nv_bfloat16>(experts, p, st->num_sms, stream);
    case MXGG_DTYPE_F16: return route_grad_for<__half>(experts, p, st->num_sms, stream);
    default: return route_grad_for<float>(experts, p, st->num_sms, stream);
  }
}

int64_t mxgg_dispatch_plan_rows(int64_t tokens, int64_t k, int64_t experts, int64_t pad) {
  if (tokens < 0 || k < 1 || experts < 1 || pad < 1) return -1;
  if (tokens >= kExtent || k >= kExtent || pad >= kExtent) return -1;
  const int64_t pairs = tokens * k;
  const int64_t used = std::min(experts, pairs);
  if (pairs >= kExtent || used * (pad - 1) >= kExtent) return -1;
  return (pairs + used * (pad - 1)) / pad * pad;
}

int64_t mxgg_dispatch_plan_workspace_size(int64_t tokens, int64_t k, int64_t experts) {
  if (tokens < 0 || k < 1 || experts < 1 || experts > kMaxRouteExperts || tokens >= kExtent || k >= kExtent ||
      tokens * k >= kExtent)
    return -1;
  const int64_t pairs = tokens * k;
  const int64_t per = plan_per(pairs);
  const int64_t blocks = std::max<int64_t>(1, (pairs + per - 1) / per);
  return blocks > 1 ? blocks * experts * 4 : 0;   // one block counts for itself
}

int mxgg_dispatch_plan(const int32_t* chosen, int64_t tokens, int32_t k, int64_t experts, int32_t pad,
                       int32_t* group_end_offsets, int32_t* counts, int32_t* row_index, int64_t rows,
                       int64_t* pair_pos, void* workspace, int64_t workspace_bytes, void* stream_v) {
  const char* what = "mxgg_dispatch_plan";
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (tokens < 0 || k < 1 || experts < 1 || pad < 1)
    return fail(MXGG_ERR_INVALID, "%s: bad sizes (tokens %lld, k %d, experts %lld, pad %d)", what, (long long)tokens, k,
                (long long)experts, pad);
  if (experts > kMaxRouteExperts)
    return fail(MXGG_ERR_UNSUPPORTED, "%s: at most %d experts", what, kMaxRouteExperts);
  const int64_t need_rows = mxgg_dispatch_plan_rows(tokens, k, experts, pad);
  if (need_rows < 0 || need_rows >= kExtent) return fail(MXGG_ERR_UNSUPPORTED, "%s: extents beyond 2^30", what);
  if (rows != need_rows)
    return fail(MXGG_ERR_INVALID, "%s: row_index must hold mxgg_dispatch_plan_rows = %lld entries, got %lld", what,
                (long long)need_rows, (long long)rows);
  const int64_t need = mxgg_dispatch_plan_workspace_size(tokens, k, experts);
  if (!group_end_offsets || !counts || (tokens > 0 && (!chosen || !row_index || !pair_pos)))
    return fail(MXGG_ERR_INVALID, "%s: null pointer", what);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(MXGG_ERR_INVALID, "%s: workspace of %lld bytes (16-byte aligned) required", what, (long long)need);
  DeviceState* st = nullptr;
  if (int rc = get_device_state(&st)) return rc;
  PlanParams p{};
  p.experts = chosen;
  p.pairs = (int)(tokens * k);
  p.k = k;
  p.E = (int)experts;
  p.pad = pad;
  p.rows = (int)rows;
  p.per = plan_per(p.pairs);
  p.hist = static_cast<int32_t*>(workspace);
  p.offs = group_end_offsets;
  p.counts = counts;
  p.row_index = row_index;
  p.pair_pos = pair_pos;
  const int blocks = std::max(1, (p.pairs + p.per - 1) / p.per);
  const int smem = (kPlanWarps + 3) * p.E * 4;
  if (int rc = allow_smem<plan_place_kernel>(*st, (kPlanWarps + 3) * kMaxRouteExperts * 4)) return rc;
  if (blocks == 1) {
    plan_place_kernel<<<1, kPlanThreads, smem, stream>>>(p);
    MXGG_CUDA_TRY(cudaGetLastError());
    return MXGG_OK;
  }
  plan_count_kernel<<<blocks, kPlanThreads, p.E * 4, stream>>>(p);
  MXGG_CUDA_TRY(cudaGetLastError());
  MXGG_CUDA_TRY(launch(plan_place_kernel, dim3(blocks), dim3(kPlanThreads), (size_t)smem, 1, true, stream, p));
  return MXGG_OK;
}

int mxgg_combine_topk_backward(const void* grad_out, const void* y, int64_t y_rows, const int64_t* pos,
                               const float* weights, const int32_t* row_index, int64_t tokens, int64_t N, int32_t k,
                               void* grad_y, float* grad_weights, void* stream_v) {
  const char* what = "mxgg_combine_topk_backward";
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (tokens < 0 || N < 0 || k < 1 || y_rows < 0) return fail(MXGG_ERR_INVALID, "%s: bad sizes", what);
  if (tokens >= kExtent || y_rows >= kExtent || N >= kExtent)
    return fail(MXGG_ERR_UNSUPPORTED, "%s: extents beyond 2^30", what);
  if (N % 8 != 0) return fail(MXGG_ERR_UNSUPPORTED, "%s: N %% 8 != 0", what);
  if ((tokens > 0 && (!pos || !weights || !grad_weights)) || (y_rows > 0 && !row_index))
    return fail(MXGG_ERR_INVALID, "%s: null pointer", what);
  if (N > 0 && ((tokens > 0 && (!grad_out || !aligned(grad_out, 16))) ||
                (y_rows > 0 && (!y || !grad_y || !aligned(y, 16) || !aligned(grad_y, 16)))))
    return fail(MXGG_ERR_INVALID, "%s: null or unaligned pointer", what);
  DeviceState* st = nullptr;
  if (int rc = get_device_state(&st)) return rc;
  CombineGradParams p{};
  p.grad_out = static_cast<const __nv_bfloat16*>(grad_out);
  p.y = static_cast<const __nv_bfloat16*>(y);
  p.pos = pos;
  p.weights = weights;
  p.row_index = row_index;
  p.rows = y_rows;
  p.T = (int)tokens;
  p.N = (int)N;
  p.k = k;
  p.grad_y = static_cast<__nv_bfloat16*>(grad_y);
  p.grad_w = grad_weights;
  const unsigned zero = (unsigned)((y_rows + kCombineZeroRows - 1) / kCombineZeroRows);
  const unsigned threads = row_threads(N);
  for (int j = 0; j < k; j += 8) {
    const unsigned blocks = (unsigned)tokens + (j == 0 ? zero : 0u);
    if (blocks == 0) continue;
    switch (std::min(8, k - j)) {
      case 1: combine_grad_kernel<1><<<blocks, threads, 0, stream>>>(p, j); break;
      case 2: combine_grad_kernel<2><<<blocks, threads, 0, stream>>>(p, j); break;
      case 3: combine_grad_kernel<3><<<blocks, threads, 0, stream>>>(p, j); break;
      case 4: combine_grad_kernel<4><<<blocks, threads, 0, stream>>>(p, j); break;
      case 5: combine_grad_kernel<5><<<blocks, threads, 0, stream>>>(p, j); break;
      case 6: combine_grad_kernel<6><<<blocks, threads, 0, stream>>>(p, j); break;
      case 7: combine_grad_kernel<7><<<blocks, threads, 0, stream>>>(p, j); break;
      default: combine_grad_kernel<8><<<blocks, threads, 0, stream>>>(p, j); break;
    }
    MXGG_CUDA_TRY(cudaGetLastError());
  }
  return MXGG_OK;
}

int mxgg_dispatch_backward(const void* grad_rows, int64_t rows, const int64_t* pos, int64_t tokens, int64_t N,
                           int32_t k, void* grad_x, void* stream_v) {
  const char* what = "mxgg_dispatch_backward";
  if (tokens < 0 || N < 0 || k < 1 || rows < 0) return fail(MXGG_ERR_INVALID, "%s: bad sizes", what);
  if (tokens >= kExtent || rows >= kExtent || N >= kExtent)
    return fail(MXGG_ERR_UNSUPPORTED, "%s: extents beyond 2^30", what);
  if (N % 8 != 0) return fail(MXGG_ERR_UNSUPPORTED, "%s: N %% 8 != 0", what);
  if (tokens == 0 || N == 0) return MXGG_OK;
  if (!pos || !grad_x || !aligned(grad_x, 16) || (rows > 0 && (!grad_rows || !aligned(grad_rows, 16))))
    return fail(MXGG_ERR_INVALID, "%s: null or unaligned pointer", what);
  DeviceState* st = nullptr;
  if (int rc = get_device_state(&st)) return rc;
  dispatch_grad_kernel<<<(unsigned)tokens, row_threads(N), 0, static_cast<cudaStream_t>(stream_v)>>>(
      static_cast<const __nv_bfloat16*>(grad_rows), pos, rows, (int)N, (int)k, static_cast<__nv_bfloat16*>(grad_x));
  MXGG_CUDA_TRY(cudaGetLastError());
  return MXGG_OK;
}

}  // extern "C"
