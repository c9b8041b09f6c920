// Top-k router and dispatch plan of a routed layer.
//
// Router, for a token t with logits l (E of them): p = softmax(l); the k
// largest logits are chosen (lowest index first among equals); their weights
// are p (or p over their sum).  A token counts when its mask is on and some
// logit is above -inf; n tokens count.  With counts_e the choices of expert e,
// f_e = counts_e / (k n) and P_e = mean p_e over the counted tokens:
//   balance loss = E sum_e f_e P_e       z loss = mean (log sum exp l)^2
// Derivative to l_e (f_e held, as counts are not differentiable):
//   p_e (c_e - sum p c) + g_z (2 / n) lse p_e + [e chosen: its weight's share]
//   with c_e = g_balance E f_e / n.
//
// Bound: latency for a decode step; the logits' bytes once per pass for few
// experts; for many the selection's integer instructions.  65521 tokens, 256
// experts, top-8, bf16: forward 35 us (34 MB; the integer pipe is the busiest,
// issue slots 64 %), the losses' sums 7 us, backward 22 us (67 MB, 3.1 TB/s).
// 16384 tokens, 8 experts, top-2, fp32: 4.3, 4.9 (its start overlapped) and 3.5 us.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "ptx.cuh"

namespace mxgg {

constexpr int kMaxRouteExperts = 1024;
constexpr int kMaxRouteK = 16;
constexpr int kRouteMaxThreads = 512;

// logits element e of a row as fp32 (exact for every type)
__device__ __forceinline__ float route_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float route_load(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float route_load(const float* p) { return *p; }
__device__ __forceinline__ void route_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void route_store(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void route_store(float* p, float v) { *p = v; }

// Keys order logits as unsigned integers with the element's index below, the
// lower index winning among equals.  A negative has all bits flipped, a positive
// its sign; adding 0 first makes -0 equal to +0 and turns every NaN into the
// canonical one (all ones below the sign), which ranks above +inf.  What lies
// below `kNone` -- -inf (an expert switched off), a key given out (0) -- is never
// chosen.  16-bit logits fit 32-bit keys and are made two at a time.
template <typename T>
struct RouteKey;
template <>
struct RouteKey<float> {
  using K = unsigned long long;
  static constexpr K kNone = (K)0x00800000u << 32;
  template <int V, typename E>
  static __device__ __forceinline__ void make(const float* t, E elem, K (&k)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t b = __float_as_uint(t[i] + 0.0f);
      k[i] = ((K)(b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u)) << 32) | (uint32_t)~elem(i);
    }
  }
  static __device__ __forceinline__ int index(K k) { return (int)~(uint32_t)k; }
  static __device__ __forceinline__ float value(K k) {
    const uint32_t h = (uint32_t)(k >> 32);
    return __uint_as_float((h & 0x80000000u) ? (h & 0x7FFFFFFFu) : ~h);
  }
  static __device__ __forceinline__ K warp_max(K k) {
    const uint32_t hi = __reduce_max_sync(0xFFFFFFFFu, (uint32_t)(k >> 32));
    const uint32_t lo = __reduce_max_sync(0xFFFFFFFFu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return ((K)hi << 32) | lo;
  }
};
__device__ __forceinline__ uint32_t route_add0(const __nv_bfloat16* t) {
  const __nv_bfloat162 v = __hadd2_rn(*reinterpret_cast<const __nv_bfloat162*>(t), __float2bfloat162_rn(0.0f));
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t route_add0(const __half* t) {
  const __half2 v = __hadd2_rn(*reinterpret_cast<const __half2*>(t), __float2half2_rn(0.0f));
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
struct RouteKey16 {
  using K = uint32_t;
  // the key of the lowest finite value
  static constexpr K kNone = std::is_same<T, __half>::value ? 0x04000000u : 0x00800000u;
  template <int V, typename E>
  static __device__ __forceinline__ void make(const T* t, E elem, K (&k)[V]) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const uint32_t w = route_add0(t + i);
      const uint32_t f = w ^ ((((w >> 15) & 0x00010001u) * 0x7FFFu) | 0x80008000u);
      k[i] = (f << 16) + (uint32_t)(0xFFFF - elem(i));
      k[i + 1] = (f & 0xFFFF0000u) | (uint32_t)(0xFFFF - elem(i + 1));
    }
  }
  static __device__ __forceinline__ int index(K k) { return 0xFFFF - (int)(k & 0xFFFFu); }
  static __device__ __forceinline__ float value(K k) {
    const uint32_t h = k >> 16, r = (h & 0x8000u) ? (h & 0x7FFFu) : (~h & 0xFFFFu);
    if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)r));
    else return __uint_as_float(r << 16);
  }
  static __device__ __forceinline__ K warp_max(K k) { return __reduce_max_sync(0xFFFFFFFFu, k); }
};
template <>
struct RouteKey<__nv_bfloat16> : RouteKey16<__nv_bfloat16> {};
template <>
struct RouteKey<__half> : RouteKey16<__half> {};

// 2^x, off by 2 ulp at most, tiny results flushed to 0.
__device__ __forceinline__ float route_ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// exp(d), d <= 0, for the weights, as 2^t with t = d log2(e): log2(e) is taken
// as the sum of two floats and the product's error e found with fmas (Dekker
// 1971), since t's own rounding, 2^-24 of an exponent that may be large, would
// show; 2^(t + e) = 2^t (1 + e ln 2) to first order.  The sums
// take it up to 128 experts; beyond, their terms are many and it would cost 3 us
// of 35 (256 experts).
__device__ __forceinline__ float route_exp(float d) {
  constexpr float kLog2e = 1.44269502f, kLog2eLow = 1.92596303e-8f, kLn2 = 0.693147181f;
  const float t = d * kLog2e;
  const float e = fmaf(d, kLog2eLow, fmaf(d, kLog2e, -t));
  const float r = route_ex2(t);
  // beside an infinite d, 0 as it is; a NaN stays one through r
  return d > -126.0f ? fmaf(r, e * kLn2, r) : r;
}
// exp(d - s), s_log2e = s log2(e), for the gradient and, beyond 128 experts, the sums: off by (|d| + |s|) 2^-24 and
// the 2 ulp of 2^x, tiny results flushed to 0.  The rounding of d = x - max alone is |d| 2^-24 of the result, in
// whatever exponential: the gradient of 16384 x 8 is 9.9e-8 of its norm off float64, 9.5e-8 in plain fp32 operations.
__device__ __forceinline__ float route_exp(float d, float s_log2e) {
  return route_ex2(fmaf(d, 1.44269504089f, -s_log2e));
}

template <typename K>
__device__ __forceinline__ void sort_desc(K& a, K& b) {
  const K hi = a > b ? a : b, lo = a > b ? b : a;
  a = hi;
  b = lo;
}

// Sorts 8 keys, largest first: an optimal 19-comparator network (Knuth, TAOCP 3, 5.3.4).
template <typename K>
__device__ __forceinline__ void sort8_desc(K (&k)[8]) {
  sort_desc(k[0], k[2]); sort_desc(k[1], k[3]); sort_desc(k[4], k[6]); sort_desc(k[5], k[7]);
  sort_desc(k[0], k[4]); sort_desc(k[1], k[5]); sort_desc(k[2], k[6]); sort_desc(k[3], k[7]);
  sort_desc(k[0], k[1]); sort_desc(k[2], k[3]); sort_desc(k[4], k[5]); sort_desc(k[6], k[7]);
  sort_desc(k[2], k[4]); sort_desc(k[3], k[5]);
  sort_desc(k[1], k[4]); sort_desc(k[3], k[6]);
  sort_desc(k[1], k[2]); sort_desc(k[3], k[4]); sort_desc(k[5], k[6]);
}

// A token's E logits lie with G neighbouring lanes, V in each; lane g's i-th
// is element (i / W) * G * W + g * W + i % W: runs of W elements (16 bytes)
// interleaved across the lanes, so a 16-byte load per run coalesces, and i
// grows with the element index within a lane.
template <typename T, int G, int V>
struct RouteRow {
  static constexpr int kVec = 16 / (int)sizeof(T);
  static constexpr int W = V < kVec ? V : kVec;
  static __device__ __forceinline__ int elem(int g, int i) { return (i / W) * (G * W) + g * W + i % W; }
  // A lane's elements as they lie in memory; -inf past E and (all of them) without a row.
  struct alignas(16) Raw {
    T t[V < kVec ? kVec : V];
  };
  static __device__ __forceinline__ T off() {
    T t;
    route_store(&t, __uint_as_float(0xFF800000u));
    return t;
  }
  static __device__ __forceinline__ void fetch(const T* row, bool has, int E, int g, bool vec, Raw& raw) {
    if (vec && W == kVec) {                // E is a multiple of kVec here
#pragma unroll
      for (int i = 0; i < V; i += W) {
        const int e = elem(g, i);
        if (has && e < E) {
          *reinterpret_cast<uint4*>(raw.t + i) = __ldg(reinterpret_cast<const uint4*>(row + e));
        } else {
#pragma unroll
          for (int j = 0; j < W; ++j) raw.t[i + j] = off();
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = elem(g, i);
        raw.t[i] = has && e < E ? row[e] : off();
      }
    }
  }
  static __device__ __forceinline__ void unpack(const Raw& raw, float (&x)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = route_load(raw.t + i);
  }
  static __device__ __forceinline__ void store(T* row, int E, int g, bool vec, const float (&x)[V]) {
    if (vec && W == kVec) {
#pragma unroll
      for (int i = 0; i < V; i += W) {
        const int e = elem(g, i);
        if (e < E) {
          uint4 q;
          T* t = reinterpret_cast<T*>(&q);
#pragma unroll
          for (int j = 0; j < W; ++j) route_store(t + j, x[i + j]);
          *reinterpret_cast<uint4*>(row + e) = q;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = elem(g, i);
        if (e < E) route_store(row + e, x[i]);
      }
    }
  }
};

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

struct RouteParams {
  const void* logits;
  long long ld;            // elements between rows
  const uint8_t* mask;     // (T,) or null
  int T, E, k;
  int renormalise;
  int vec;                 // 16-byte row loads allowed
  int32_t* experts;        // (T, k)
  float* weights;          // (T, k)
  float2* stats;           // (T,): the largest logit and log sum exp(l - it); (-inf, 0) for a token that does not count
  int32_t* counts;         // (E,)
  float* losses;           // balance, z
  int32_t* tokens;         // counted tokens
  // per-block partials: [blocks][E] sums of p, [blocks][E] choices, [blocks] z sums, [blocks] tokens
  float* part_p;
  int32_t* part_c;
  float* part_z;
  int32_t* part_n;
};

// Losses from the per-block partials, summed in a fixed order (the result does
// not depend on timing).  CTA q of `ctas` (a cluster, or one) takes a run of
// the experts; lanes run along experts, warps along blocks.
__device__ __forceinline__ void route_finish(const RouteParams& p, int blocks, int q, int ctas) {
  __shared__ float sh_p[32][33];
  __shared__ int sh_c[32][33];
  __shared__ float sh_f[32];
  __shared__ int sh_i[32];
  __shared__ float sh_bal;
  const int tid = threadIdx.x, nth = blockDim.x, warp = tid >> 5, lane = tid & 31, nw = nth >> 5;
  const int chunks = (p.E + 31) / 32, c0 = chunks * q / ctas, c1 = chunks * (q + 1) / ctas;
  float bal = 0.0f;
  for (int ch = c0; ch < c1; ++ch) {
    const int e = ch * 32 + lane;
    float s = 0.0f;
    int c = 0;
    if (e < p.E)
#pragma unroll 8
      for (int b = warp; b < blocks; b += nw) {
        s += p.part_p[(long long)b * p.E + e];
        c += p.part_c[(long long)b * p.E + e];
      }
    sh_p[warp][lane] = s;
    sh_c[warp][lane] = c;
    __syncthreads();
    // warp w adds up expert w, w + nw, ... of the chunk
    for (int i = warp; i < 32; i += nw) {
      s = lane < nw ? sh_p[lane][i] : 0.0f;
      c = lane < nw ? sh_c[lane][i] : 0;
      s = group_sum<32>(s);
      c = __reduce_add_sync(0xFFFFFFFFu, c);
      if (ch * 32 + i < p.E) {
        if (lane == 0) p.counts[ch * 32 + i] = c;
        bal += (float)c * s;
      }
    }
    __syncthreads();
  }
  float z = 0.0f;
  int n = 0;
  if (q == 0)
    for (int b = tid; b < blocks; b += nth) {
      z += p.part_z[b];
      n += p.part_n[b];
    }
  z = group_sum<32>(z);
  n = __reduce_add_sync(0xFFFFFFFFu, n);
  if (lane == 0) {
    sh_p[0][warp] = bal;
    sh_f[warp] = z;
    sh_i[warp] = n;
  }
  __syncthreads();
  if (tid == 0) {
    bal = 0.0f;
    for (int w = 0; w < nw; ++w) bal += sh_p[0][w];
    sh_bal = bal;
  }
  if (ctas > 1) ptx::cluster_sync();
  if (q == 0 && tid == 0) {
    for (int r = 1; r < ctas; ++r) bal += ptx::ld_cluster_f32(ptx::mapa(ptx::smem_u32(&sh_bal), r));
    z = 0.0f;
    n = 0;
    for (int w = 0; w < nw; ++w) { z += sh_f[w]; n += sh_i[w]; }
    const float fn = (float)(n > 0 ? n : 1);
    p.losses[0] = bal * ((float)p.E / ((float)p.k * fn)) / fn;
    p.losses[1] = z / fn;
    *p.tokens = n;
  }
  if (ctas > 1) ptx::cluster_sync();                      // no CTA leaves while its sum is being read
}

// The k largest of a group's keys, largest first: lane j % G keeps choice j in
// slot j / G.  kMost bounds k.  Eight keys a lane come sorted and are given out
// from the top; after round j only the next kMost - 1 - j of a lane can still be
// asked for, so no more are moved up.  More keys are searched anew each round.
template <typename Key, int G, int V, int kMost, int kSlots>
__device__ __forceinline__ void route_choose(typename Key::K (&key)[V], int g, int k, typename Key::K (&mine)[kSlots]) {
  using K = typename Key::K;
#pragma unroll
  for (int j = 0; j < kMost; ++j) {
    if (j >= k) break;
    K best = key[0];
    if constexpr (V != 8) {
#pragma unroll
      for (int i = 1; i < V; ++i) best = key[i] > best ? key[i] : best;
    }
    const K own = best;
    if constexpr (G == 32) {
      best = Key::warp_max(best);
    } else {
#pragma unroll
      for (int o = G / 2; o; o >>= 1) {
        const K other = __shfl_xor_sync(0xFFFFFFFFu, best, o);
        best = other > best ? other : best;
      }
    }
    if (g == j % G) mine[j / G] = best;
    // keys that can be chosen are distinct: the lane that held it moves on
    if constexpr (V == 8) {
      const bool won = own == best;
      constexpr int kKeep = kMost < V ? kMost : V;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (kMost > V || i < kKeep - 1 - j) key[i] = won ? (i + 1 < V ? key[i + 1 < V ? i + 1 : i] : (K)0) : key[i];
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) key[i] = key[i] == best ? (K)0 : key[i];
    }
  }
}

template <typename T, int G, int V>
__global__ void __launch_bounds__(kRouteMaxThreads) route_topk_kernel(const RouteParams p) {
  using Row = RouteRow<T, G, V>;
  using Key = RouteKey<T>;
  using K = typename Key::K;
  constexpr int kGroups = 32 / G;
  // choices a lane keeps: lane j % G holds choice j
  constexpr int kMostK = G * V < kMaxRouteK ? G * V : kMaxRouteK;
  constexpr int kSlots = (kMostK + G - 1) / G;
  const float ninf = __uint_as_float(0xFF800000u);
  __shared__ float sh_p[kMaxRouteExperts];
  __shared__ int sh_c[kMaxRouteExperts];
  __shared__ float sh_f[32];
  __shared__ int sh_i[32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nw = blockDim.x >> 5;
  const int g = lane % G, grp = lane / G;
  for (int e = tid; e < p.E; e += blockDim.x) {
    sh_p[e] = 0.0f;
    sh_c[e] = 0;
  }
  __syncthreads();
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.0f;
  float zsum = 0.0f;
  int ntok = 0;
  const int step = gridDim.x * nw * kGroups;
  const long long row_step = (long long)step * p.ld;
  // The next token's row is on its way while this one is worked on: a token is
  // a chain of dependent steps, and one load's latency would be half of it.
  int t0 = (blockIdx.x * nw + warp) * kGroups;
  const T* row = static_cast<const T*>(p.logits) + (long long)(t0 + grp) * p.ld;
  typename Row::Raw raw;
  Row::fetch(row, t0 + grp < p.T && (!p.mask || p.mask[t0 + grp]), p.E, g, p.vec, raw);
  // every lane of a warp runs the same number of rounds: the shuffles need all of them
  for (; t0 < p.T; t0 += step) {
    const long long t = t0 + grp;
    float x[V];
    Row::unpack(raw, x);
    K key[V];
    Key::template make<V>(raw.t, [g](int i) { return Row::elem(g, i); }, key);
    row += row_step;
    const int tn = t0 + step + grp;
    Row::fetch(row, tn < p.T && (!p.mask || p.mask[tn]), p.E, g, p.vec, raw);
    if constexpr (V == 8) sort8_desc(key);
    K mine[kSlots];
#pragma unroll
    for (int s = 0; s < kSlots; ++s) mine[s] = 0;
    if constexpr (kMostK > 8) {
      if (p.k > 8) route_choose<Key, G, V, kMostK>(key, g, p.k, mine);
      else route_choose<Key, G, V, 8>(key, g, p.k, mine);
    } else {
      route_choose<Key, G, V, kMostK>(key, g, p.k, mine);
    }
    const K first = G == 1 ? mine[0] : __shfl_sync(0xFFFFFFFFu, mine[0], lane - g);
    const bool counted = first >= Key::kNone;
    const float top = counted ? Key::value(first) : 0.0f;
    float total = 0.0f;
    // softmax terms against the row's maximum: x - top is <= 0 or -inf (elements past E, masked rows), or
    // NaN beside a NaN or +inf
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[i] = G < 32 ? route_exp(x[i] - top) : route_exp(x[i] - top, 0.0f);
      total += x[i];
    }
    total = group_sum<G>(total);
    float ex[kSlots], csum = 0.0f;
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      ex[s] = mine[s] >= Key::kNone ? route_exp(Key::value(mine[s]) - top) : 0.0f;
      csum += ex[s];
    }
    csum = group_sum<G>(csum);
    const float d = __frcp_rn(p.renormalise ? csum : total);
    if (t < p.T) {
#pragma unroll
      for (int s = 0; s < kSlots; ++s) {
        const int j = s * G + g;
        if (j < p.k) {
          const bool has = mine[s] >= Key::kNone;
          const int e = has ? Key::index(mine[s]) : -1;
          p.experts[t * p.k + j] = e;
          p.weights[t * p.k + j] = has ? ex[s] * d : 0.0f;
          if (has) atomicAdd(&sh_c[e], 1);
        }
      }
      if (g == 0) {
        const float lt = counted ? logf(total) : 0.0f, lse = top + lt;
        p.stats[t] = make_float2(counted ? top : ninf, lt);
        if (counted) {
          zsum += lse * lse;
          ++ntok;
        }
      }
    }
    const float inv = counted ? __frcp_rn(total) : 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] += x[i] * inv;
  }
  // block sums in a fixed order: lanes of a warp by shuffles, warps one after another
#pragma unroll
  for (int o = G; o < 32; o <<= 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] += __shfl_xor_sync(0xFFFFFFFFu, acc[i], o);
  }
  zsum = group_sum<32>(zsum);
  ntok = __reduce_add_sync(0xFFFFFFFFu, ntok);
  if (lane == 0) { sh_f[warp] = zsum; sh_i[warp] = ntok; }
  for (int w = 0; w < nw; ++w) {
    if (warp == w && grp == 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = Row::elem(g, i);
        if (e < p.E) sh_p[e] += acc[i];
      }
    }
    __syncthreads();
  }
  for (int e = tid; e < p.E; e += blockDim.x) {
    p.part_p[(long long)blockIdx.x * p.E + e] = sh_p[e];
    p.part_c[(long long)blockIdx.x * p.E + e] = sh_c[e];
  }
  if (tid == 0) {
    float z = 0.0f;
    int n = 0;
    for (int w = 0; w < nw; ++w) { z += sh_f[w]; n += sh_i[w]; }
    p.part_z[blockIdx.x] = z;
    p.part_n[blockIdx.x] = n;
  }
  if (gridDim.x == 1) {
    __syncthreads();
    route_finish(p, 1, 0, 1);
  } else {
    ptx::griddep_launch_dependents();
  }
}

constexpr int kRouteFinishCtas = 8;
__global__ void __launch_bounds__(1024) route_finish_kernel(const RouteParams p, int blocks) {
  ptx::griddep_wait();
  route_finish(p, blocks, (int)blockIdx.x, (int)gridDim.x);
}

struct RouteGradParams {
  const void* logits;
  long long ld;
  int T, E, k;
  int renormalise;
  int vec;                  // 16-byte loads of logits rows and stores of grad rows allowed
  const int32_t* experts;   // (T, k)
  const float* weights;     // (T, k)
  const float2* stats;      // (T,)
  const int32_t* counts;    // (E,)
  const int32_t* tokens;
  const float* grad_w;      // (T, k) or null
  const float* grad_bal;    // scalar on the device, or null
  const float* grad_z;
  float bal_coef, z_coef;   // factors of the scalars (the gradients themselves when those are null)
  void* grad;               // (T, E)
};

template <typename T, int G, int V>
__global__ void __launch_bounds__(256) route_grad_kernel(const RouteGradParams p) {
  using Row = RouteRow<T, G, V>;
  constexpr int kGroups = 32 / G;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nw = blockDim.x >> 5;
  const int g = lane % G, grp = lane / G;
  const int n_i = *p.tokens;
  const float n = (float)(n_i > 0 ? n_i : 1);
  const float gb = p.bal_coef * (p.grad_bal ? *p.grad_bal : 1.0f);
  const float gz = p.z_coef * (p.grad_z ? *p.grad_z : 1.0f) * 2.0f / n;
  const float cf = (gb * (float)p.E / n) / (n * (float)p.k);
  float c[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = Row::elem(g, i);
    c[i] = e < p.E ? cf * (float)p.counts[e] : 0.0f;
  }
  const int step = gridDim.x * nw * kGroups;
  const long long row_step = (long long)step * p.ld;
  const float ninf = __uint_as_float(0xFF800000u);
  // one token ahead, as in the forward
  int t0 = (blockIdx.x * nw + warp) * kGroups;
  const T* row = static_cast<const T*>(p.logits) + (long long)(t0 + grp) * p.ld;
  typename Row::Raw raw;
  float2 next = t0 + grp < p.T ? p.stats[t0 + grp] : make_float2(ninf, 0.0f);
  Row::fetch(row, t0 + grp < p.T, p.E, g, p.vec, raw);
  for (; t0 < p.T; t0 += step) {
    const long long t = t0 + grp;
    const float2 st = next;
    // p = exp((l - largest) - log sum): one rounded log-sum-exp would lose the
    // sum beside a large |l| (a row of the type's lowest value)
    const bool counted = st.x != ninf;
    const float lse = st.x + st.y;
    const float top = counted ? st.x : 0.0f, lt = st.y * 1.44269504089f;
    const T* cur = row;
    float x[V];
    float s = 0.0f;
    Row::unpack(raw, x);
    row += row_step;
    const int tn = t0 + step + grp;
    next = tn < p.T ? p.stats[tn] : make_float2(ninf, 0.0f);
    Row::fetch(row, tn < p.T, p.E, g, p.vec, raw);
    // this token's choices: the first of a lane's by registers, further ones (k > G) from memory
    int e0 = -1;
    float w0 = 0.0f, g0 = 0.0f;
    if (p.grad_w && counted && g < p.k) {
      e0 = p.experts[t * p.k + g];
      w0 = p.weights[t * p.k + g];
      g0 = p.grad_w[t * p.k + g];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[i] = counted ? route_exp(x[i] - top, lt) : 0.0f;
      s += x[i] * c[i];
    }
    s = group_sum<G>(s);
    float inner = 0.0f;
    if (p.grad_w) {
      if (e0 >= 0) inner = w0 * g0;
      if constexpr (G < kMaxRouteK) {
        if (counted)
          for (int j = g + G; j < p.k; j += G)
            if (p.experts[t * p.k + j] >= 0) inner += p.weights[t * p.k + j] * p.grad_w[t * p.k + j];
      }
      inner = group_sum<G>(inner);
    }
    const float all = counted ? gz * lse - s - (p.renormalise ? 0.0f : inner) : 0.0f;
    float d[V];
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = x[i] * (c[i] + all);
    T* out = static_cast<T*>(p.grad) + t * p.E;
    if (t < p.T) Row::store(out, p.E, g, p.vec, d);
    if (!p.grad_w) continue;
    // the chosen experts' elements again, whole, by the lane that holds the choice
    __syncwarp();
    const float cut = p.renormalise ? inner : 0.0f;
    if (e0 >= 0) {
      const float pe = route_exp(route_load(cur + e0) - top, lt);
      route_store(out + e0, pe * (cf * (float)p.counts[e0] + all) + w0 * (g0 - cut));
    }
    if constexpr (G < kMaxRouteK) {
      if (counted)
        for (int j = g + G; j < p.k; j += G) {
          const int e = p.experts[t * p.k + j];
          if (e < 0) continue;
          const float pe = route_exp(route_load(cur + e) - top, lt);
          route_store(out + e, pe * (cf * (float)p.counts[e] + all) +
                                   p.weights[t * p.k + j] * (p.grad_w[t * p.k + j] - cut));
        }
    }
  }
}

// ------------------------------------------------------------ dispatch plan
// A stable counting sort of the T * k choices by expert into groups padded to
// `pad` rows: pair_pos[pair] = start_pad[e] + rank of the pair among e's
// choices in (token, choice) order, row_index its inverse, -1 in padding.
// Blocks take contiguous chunks; a chunk's first rank of e is the sum of the
// earlier chunks' choices of e (a first launch counts them; one chunk needs
// no such launch).  Bound: latency; 131072 x 2 choices of 64 experts take 2.2 us
// to count and 8.6 us to place (4.2 MB in all), a decode step's 122 choices 4.7 us.
constexpr int kPlanThreads = 512;
constexpr int kPlanWarps = kPlanThreads / 32;

struct PlanParams {
  const int32_t* experts;    // (pairs,)
  int pairs, k, E, pad;
  int rows;                  // length of row_index
  int per;                   // pairs per block
  int32_t* hist;             // [blocks][E]
  int32_t* offs;             // (E,) cumulative padded ends
  int32_t* counts;           // (E,)
  int32_t* row_index;        // (rows,)
  int64_t* pair_pos;         // (pairs,)
};

__global__ void __launch_bounds__(kPlanThreads) plan_count_kernel(const PlanParams p) {
  extern __shared__ int sh[];
  for (int e = threadIdx.x; e < p.E; e += kPlanThreads) sh[e] = 0;
  __syncthreads();
  const int b0 = blockIdx.x * p.per, b1 = min(b0 + p.per, p.pairs);
  for (int i = b0 + threadIdx.x; i < b1; i += kPlanThreads) {
    const int e = p.experts[i];
    if (e >= 0 && e < p.E) atomicAdd(&sh[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += kPlanThreads) p.hist[(long long)blockIdx.x * p.E + e] = sh[e];
  ptx::griddep_launch_dependents();
}

// dynamic shared memory: warp counters [kPlanWarps][E], base [E], start [E], total [E]
__global__ void __launch_bounds__(kPlanThreads) plan_place_kernel(const PlanParams p) {
  extern __shared__ int sh[];
  int* wc = sh;
  int* base = wc + kPlanWarps * p.E;
  int* start = base + p.E;
  int* total = start + p.E;
  __shared__ int sh_end;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int blocks = gridDim.x;
  for (int i = tid; i < kPlanWarps * p.E; i += kPlanThreads) wc[i] = 0;
  for (int i = tid; i < p.E; i += kPlanThreads) { base[i] = 0; total[i] = 0; }
  __syncthreads();
  ptx::griddep_wait();
  // warp w's run of the block's chunk, in order
  const int b0 = blockIdx.x * p.per, b1 = min(b0 + p.per, p.pairs);
  const int wper = ((p.per + kPlanWarps - 1) / kPlanWarps + 31) / 32 * 32;
  const int w0 = min(b0 + warp * wper, b1), w1 = min(w0 + wper, b1);
  for (int i = w0 + lane; i < w1; i += 32) {
    const int e = p.experts[i];
    if (e >= 0 && e < p.E) atomicAdd(&wc[warp * p.E + e], 1);
  }
  if (blocks > 1) {
    for (int i = tid; i < blocks * p.E; i += kPlanThreads) {
      const int h = p.hist[i];
      const int b = i / p.E, e = i - b * p.E;
      if (h) {
        atomicAdd(&total[e], h);
        if (b < (int)blockIdx.x) atomicAdd(&base[e], h);
      }
    }
  }
  __syncthreads();
  for (int e = tid; e < p.E; e += kPlanThreads) {
    int s = base[e];
    for (int w = 0; w < kPlanWarps; ++w) {
      const int c = wc[w * p.E + e];
      wc[w * p.E + e] = s;
      s += c;
    }
    if (blocks == 1) total[e] = s;
  }
  __syncthreads();
  // padded starts: an exclusive scan over the experts by one warp
  if (warp == 0) {
    int carry = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane;
      const int v = e < p.E ? (total[e] + p.pad - 1) / p.pad * p.pad : 0;
      int s = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, s, o);
        if (lane >= o) s += u;
      }
      if (e < p.E) start[e] = carry + s - v;
      if (blockIdx.x == 0 && e < p.E) {
        p.offs[e] = carry + s;
        p.counts[e] = total[e];
      }
      carry += __shfl_sync(0xFFFFFFFFu, s, 31);
    }
    if (lane == 0) sh_end = carry;
  }
  __syncthreads();
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const int i = i0 + lane;
    const int e = i < w1 ? p.experts[i] : -1;
    const bool ok = e >= 0 && e < p.E;
    const unsigned same = __match_any_sync(0xFFFFFFFFu, ok ? e : -1);
    const int before = __popc(same & ((1u << lane) - 1u));
    int pos = -1;
    if (ok) pos = start[e] + wc[warp * p.E + e] + before;
    __syncwarp();
    if (ok && before == 0) wc[warp * p.E + e] += __popc(same);
    __syncwarp();
    if (i < w1) {
      p.pair_pos[i] = pos;
      if (ok) p.row_index[pos] = i / p.k;
    }
  }
  // padding rows: the groups' tails, then everything past the last group
  for (int e = blockIdx.x * kPlanWarps + warp; e < p.E; e += blocks * kPlanWarps) {
    const int r1 = start[e] + (total[e] + p.pad - 1) / p.pad * p.pad;
    for (int r = start[e] + total[e] + lane; r < r1; r += 32) p.row_index[r] = -1;
  }
  for (int r = sh_end + blockIdx.x * kPlanThreads + tid; r < p.rows; r += blocks * kPlanThreads) p.row_index[r] = -1;
}

}  // namespace mxgg
