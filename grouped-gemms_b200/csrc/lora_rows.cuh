// Low-rank adapters for few rows each (a decode step): both products in one
// launch (formulas in lora.cuh).
//
// A cluster of CTAs takes up to 16 rows that carry one adapter: its CTAs split
// the first product's contraction, add their partial v through distributed
// shared memory, and split the second product's columns.  Cluster m looks at
// row m: it works when row m is the first, 17th, 33rd ... row of its adapter
// within a window of 1024 rows and takes the next 16 of them, so rows need no
// sorting, weights are read once per 16 rows, and nothing depends on timing.
//
// Bound: the adapters' bytes (HBM, or latency for a few rows).  16-row
// mma.sync products take the weights straight from global memory into
// registers; tcgen05 would need 128-row tiles, 1 to 16 rows of them real.
// From a cold L2: 64 rows with adapters of their own, 5120 -> 8192, rank 16: 16 us
// (30 MB); rank 64: 44 us (112 MB); one row, 8192 -> 5120, rank 64: 9.4 us.
#pragma once

#include "lora_tc.cuh"

namespace mxgg {

constexpr int kRowsMaxThreads = 512;
constexpr int kRowsWindow = 1024;
constexpr int kRowsGroup = 16;

struct RowsParams {
  LoraSegs g;                 // offs null: adapter per row
  const __nv_bfloat16* x;
  long long x_ld;
  const __nv_bfloat16* a;     // (L, R, K)
  const __nv_bfloat16* b;     // (L, N, R)
  const float* scaling;
  const void* base;
  long long base_ld;
  void* out;
  long long out_ld;
  __nv_bfloat16* v;           // or null
  int K, N, R, Rp, cluster;
  int threads;                // wanted (ranks above 64 take 256)
};

// Floats between the rows of a warp's partial v in shared memory: 8 more than a
// multiple of 32, so that the 8 rows a store touches lie on different banks.
__host__ __device__ constexpr int rows_red_ld(int Rp) { return (Rp + 31) / 32 * 32 + 8; }

// KC: 16-wide pieces of the rank (Rp <= 16 KC).
template <typename O, int KC>
__global__ void __launch_bounds__(KC <= 4 ? kRowsMaxThreads : 256) lora_rows_kernel(const RowsParams p) {
  const int nth = blockDim.x, nw = nth >> 5;
  extern __shared__ float sh_red[];                       // [warps][16][rows_red_ld(Rp)]
  __shared__ int sh_ad[kRowsWindow];
  __shared__ int sh_start[kMaxLoraSegments + 1], sh_tiles[kMaxLoraSegments + 1];
  __shared__ __align__(16) float sh_part[kRowsGroup * 16 * KC];
  __shared__ __align__(16) float sh_v[kRowsGroup][16 * KC + 4];
  __shared__ int sh_rows[kRowsGroup];
  __shared__ int sh_n;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int q = blockIdx.x % p.cluster, m = blockIdx.x / p.cluster;
  const int w0 = m / kRowsWindow * kRowsWindow, w1 = min(w0 + kRowsWindow, p.g.M);
  if (p.g.offs) {
    if (warp == 0) lora_build_table(p.g, 1, sh_start, sh_tiles);
    __syncthreads();
  }
  for (int j = w0 + tid; j < w1; j += nth) {
    int l;
    if (p.g.offs) l = j < sh_start[p.g.S] ? lora_adapter(p.g, lora_find(sh_tiles, p.g.S, j)) : -2;
    else l = lora_adapter(p.g, j);
    sh_ad[j - w0] = l;
  }
  __syncthreads();
  const int l = sh_ad[m - w0];
  if (l == -2) return;                                    // past the last segment (the whole cluster leaves)
  constexpr int kPer16 = 16 / (int)sizeof(O);
  if (l < 0) {
    // no adapter: the base's row (nothing to do in place), or zeros; v is zero
    const int n16 = p.N / kPer16, per = (n16 + p.cluster - 1) / p.cluster;
    const int i1 = min(n16, (q + 1) * per);
    if (p.base != p.out)
      for (int i = q * per + tid; i < i1; i += nth) {
        uint4 z = make_uint4(0, 0, 0, 0);
        if (p.base) z = *(reinterpret_cast<const uint4*>(static_cast<const O*>(p.base) + m * p.base_ld) + i);
        *(reinterpret_cast<uint4*>(static_cast<O*>(p.out) + m * p.out_ld) + i) = z;
      }
    if (p.v && q == 0)
      for (int i = tid; i < p.Rp / 4; i += nth)
        *(reinterpret_cast<uint4*>(p.v + (long long)m * 2 * p.Rp) + i) = make_uint4(0, 0, 0, 0);
    return;
  }
  if (warp == 0) {
    int before = 0;
    for (int j0 = w0; j0 < m; j0 += 32) {
      const int j = j0 + lane;
      before += __popc(__ballot_sync(0xFFFFFFFFu, j < m && sh_ad[j - w0] == l));
    }
    int n = 0;
    if (before % kRowsGroup == 0) {
      for (int j0 = m; j0 < w1 && n < kRowsGroup; j0 += 32) {
        const int j = j0 + lane;
        const bool hit = j < w1 && sh_ad[j - w0] == l;
        const unsigned b = __ballot_sync(0xFFFFFFFFu, hit);
        const int at = n + __popc(b & ((1u << lane) - 1u));
        if (hit && at < kRowsGroup) sh_rows[at] = j;
        n += __popc(b);
      }
    }
    if (lane == 0) sh_n = min(n, kRowsGroup);
  }
  __syncthreads();
  const int nrows = sh_n;
  if (nrows == 0) return;                                 // another cluster takes this row

  const int g = lane >> 2, t = lane & 3;
  const int step = p.cluster * nw, first = q * nw + warp;
  const __nv_bfloat16* wa = p.a + (long long)l * p.R * p.K;
  const __nv_bfloat16* wb = p.b + (long long)l * p.N * p.R;
  // the second product's weights start on their way while the first runs
  for (int gi = first; gi * 32 < p.N; gi += step) {
    const char* src = reinterpret_cast<const char*>(wb + (long long)gi * 32 * p.R);
    const int bytes = min(32, p.N - gi * 32) * p.R * 2;
    for (int o = lane * 128; o < bytes; o += 32 * 128) ptx::prefetch_l2(src + o);
    if (p.base && lane < nrows)
      ptx::prefetch_l2(static_cast<const O*>(p.base) + sh_rows[lane] * p.base_ld + gi * 32);
  }
  const int row_lo = g < nrows ? sh_rows[g] : -1, row_hi = g + 8 < nrows ? sh_rows[g + 8] : -1;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  {
    float acc[2 * KC][4];
#pragma unroll
    for (int j = 0; j < 2 * KC; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
    // 32 contraction elements a round: lane t of a quad holds 8 contiguous ones of its row (both operands in
    // the same order, so the products need no shuffle)
    // Loads are unconditional (addresses clamped, what lies outside replaced by 0 afterwards) and come before the
    // products, so that a round's loads are all in flight at once; a branch around each kept them one by one
    // (1.7 TB/s for 64 adapters of rank 64).
    const __nv_bfloat16* xl = p.x + (row_lo >= 0 ? row_lo : sh_rows[0]) * p.x_ld;
    const __nv_bfloat16* xh = p.x + (row_hi >= 0 ? row_hi : sh_rows[0]) * p.x_ld;
#pragma unroll(KC == 1 ? 4 : KC <= 4 ? 2 : 1)
    for (int c = first; c * 32 < p.K; c += step) {
      const int k0 = c * 32 + t * 8;
      const bool in = k0 < p.K;
      const int k = in ? k0 : p.K - 8;
      uint4 xa = __ldg(reinterpret_cast<const uint4*>(xl + k));
      uint4 xb = __ldg(reinterpret_cast<const uint4*>(xh + k));
      uint4 w[2 * KC];
#pragma unroll
      for (int j = 0; j < 2 * KC; ++j)
        w[j] = __ldg(reinterpret_cast<const uint4*>(wa + (long long)min(j * 8 + g, p.R - 1) * p.K + k));
      xa = in && row_lo >= 0 ? xa : zero;
      xb = in && row_hi >= 0 ? xb : zero;
#pragma unroll
      for (int j = 0; j < 2 * KC; ++j) {
        const uint4 u = in && j * 8 + g < p.R ? w[j] : zero;
        ptx::mma_m16n8k16_bf16(acc[j], xa.x, xb.x, xa.y, xb.y, u.x, u.y);
        ptx::mma_m16n8k16_bf16(acc[j], xa.z, xb.z, xa.w, xb.w, u.z, u.w);
      }
    }
    float* red = sh_red + warp * kRowsGroup * rows_red_ld(p.Rp);
#pragma unroll
    for (int j = 0; j < 2 * KC; ++j) {
      const int r = j * 8 + 2 * t;
      if (r < p.Rp) {
        if (row_lo >= 0)
          *reinterpret_cast<float2*>(red + g * rows_red_ld(p.Rp) + r) = make_float2(acc[j][0], acc[j][1]);
        if (row_hi >= 0)
          *reinterpret_cast<float2*>(red + (g + 8) * rows_red_ld(p.Rp) + r) = make_float2(acc[j][2], acc[j][3]);
      }
    }
  }
  for (int i = tid; i < kRowsGroup * (16 * KC + 4) / 4; i += nth)
    *(reinterpret_cast<float4*>(&sh_v[0][0]) + i) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  __syncthreads();
  const int quads = nrows * p.Rp / 4;                     // only the rows there are
  for (int i = tid; i < quads; i += nth) {
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int w = 0; w < nw; ++w) {
      const float4 u = *reinterpret_cast<const float4*>(sh_red + (w * kRowsGroup + i * 4 / p.Rp) * rows_red_ld(p.Rp) +
                                                        i * 4 % p.Rp);
      s.x += u.x; s.y += u.y; s.z += u.z; s.w += u.w;
    }
    *reinterpret_cast<float4*>(sh_part + i * 4) = s;
  }
  ptx::cluster_sync();
  const float scale = p.scaling ? p.scaling[l] : 1.0f;
  for (int i = tid; i < quads; i += nth) {
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const uint32_t src = ptx::smem_u32(sh_part + i * 4);
    // a remote load takes hundreds of cycles: eight at a time (the cluster has 8 or 16 CTAs), added in rank order
    for (int c0 = 0; c0 < p.cluster; c0 += 8) {
      float4 u[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) u[c] = ptx::ld_cluster_f32x4(ptx::mapa(src, c0 + c));
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        s.x += u[c].x; s.y += u[c].y; s.z += u[c].z; s.w += u[c].w;
      }
    }
    const int r = i * 4 / p.Rp, c = i * 4 % p.Rp;
    // ranks past R stay 0: their sums of x times 0 are NaN beside an infinite x
    if (c < p.R)
      *reinterpret_cast<float4*>(&sh_v[r][c]) = make_float4(scale * s.x, scale * s.y, scale * s.z, scale * s.w);
  }
  ptx::cluster_arrive();                                  // waited for at the end: no CTA leaves while it is read
  __syncthreads();
  if (p.v && q == 0)
    for (int i = tid; i < nrows * (p.Rp / 8); i += nth) {
      const int r = i / (p.Rp / 8), c = i % (p.Rp / 8) * 8;
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = sh_v[r][c + j];
      uint4 hi, lo;
      split_halves(f, hi, lo);
      __nv_bfloat16* row = p.v + (long long)sh_rows[r] * 2 * p.Rp;
      *reinterpret_cast<uint4*>(row + c) = hi;
      *reinterpret_cast<uint4*>(row + p.Rp + c) = lo;
    }
  // v's halves as the first operand, rank pieces of 16 (lane t: ranks 4 t .. 4 t + 3 of its rows)
  uint32_t hi[KC][4], lo[KC][4];
#pragma unroll
  for (int kc = 0; kc < KC; ++kc) {
    const int c = kc * 16 + 4 * t;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (c < p.Rp) f = *reinterpret_cast<const float4*>(&sh_v[g + 8 * h][c]);
      split2(f.x, f.y, hi[kc][h], lo[kc][h]);
      split2(f.z, f.w, hi[kc][2 + h], lo[kc][2 + h]);
    }
  }
#pragma unroll(KC == 1 ? 2 : 1)
  for (int gi = first; gi * 32 < p.N; gi += step) {
    // four 8-column products whose columns interleave so that a lane ends with 8 neighbours of each row
    uint2 w[4][KC];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = min(gi * 32 + (g >> 1) * 8 + 2 * j + (g & 1), p.N - 1);   // columns past N are not stored
#pragma unroll
      for (int kc = 0; kc < KC; ++kc)
        w[j][kc] = __ldg(reinterpret_cast<const uint2*>(wb + (long long)n * p.R + min(kc * 16 + 4 * t, p.R - 4)));
    }
    float d[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) d[j][i] = 0.0f;
#pragma unroll
      for (int kc = 0; kc < KC; ++kc) {
        const uint2 u = kc * 16 + 4 * t < p.R ? w[j][kc] : make_uint2(0, 0);
        ptx::mma_m16n8k16_bf16(d[j], hi[kc][0], hi[kc][1], hi[kc][2], hi[kc][3], u.x, u.y);
        ptx::mma_m16n8k16_bf16(d[j], lo[kc][0], lo[kc][1], lo[kc][2], lo[kc][3], finite_pair(u.x), finite_pair(u.y));
      }
    }
    const int c = gi * 32 + t * 8;
    if (c >= p.N) continue;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = h ? row_hi : row_lo;
      if (row < 0) continue;
      float f[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[2 * j] = d[j][2 * h];
        f[2 * j + 1] = d[j][2 * h + 1];
      }
      O* dst = static_cast<O*>(p.out) + row * p.out_ld + c;
      __align__(16) O o[8];
      if (p.base) {
        __align__(16) O bs[8];
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const O*>(p.base) + row * p.base_ld + c);
#pragma unroll
        for (int i = 0; i < 8 / kPer16; ++i) reinterpret_cast<uint4*>(bs)[i] = src[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] += lora_to_f32<O>(bs[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = lora_from_f32<O>(f[i]);
#pragma unroll
      for (int i = 0; i < 8 / kPer16; ++i) reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(o)[i];
    }
  }
  ptx::cluster_wait();
}

}  // namespace mxgg
