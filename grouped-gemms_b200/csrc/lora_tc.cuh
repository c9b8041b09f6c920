// Tensor-core kernels of the low-rank adapters (formulas in lora.cuh): TMA
// tiles in a shared-memory ring, tcgen05.mma with the accumulator in TMEM, one
// thread issuing the loads and one the products.
//
// Every wait is bounded: one that runs out sets kErrLoraWait in the device
// status word and ends the roles' loops.  Behind the barrier that all of them
// reach, the copies still in flight are waited for (whichever role's wait ran
// out, also after the last load was issued), then the kernel frees its TMEM and
// returns: shared memory that a copy may still write never goes to another CTA.
#pragma once

#include "lora.cuh"

namespace mxgg {

constexpr uint32_t kErrLoraWait = 512u;
// A wait for a whole loop's end, in units of the limit of one stage's wait (whose own failure ends it early).
constexpr unsigned long long kLoraWaitSpan = 64;
constexpr int kLoraBM = 128;    // rows of a tile
constexpr int kLoraBK = 64;     // contraction elements of a stage: a 128-byte swizzled row

__device__ __forceinline__ int lora_adapter(const LoraSegs& g, int s) {
  const int l = g.adapter ? g.adapter[s] : s;
  return l >= 0 && l < g.L ? l : -1;
}

// Segment starts and the prefix sum of their tiles of `tile` rows, by one warp.
// start[S] is the last end, tiles[S] the number of tiles.  adapters (or null):
// the segments' adapters, loaded along with the ends (one latency, not two).
__device__ __forceinline__ void lora_build_table(const LoraSegs& g, int tile, int* start, int* tiles,
                                                 int* adapters = nullptr) {
  const int lane = threadIdx.x & 31;
  int carry_end = 0, carry_tiles = 0;
  for (int s0 = 0; s0 < g.S; s0 += 32) {
    const int s = s0 + lane;
    int end = s < g.S ? min(g.offs[s], g.M) : 0;
    if (adapters && s < g.S) adapters[s] = lora_adapter(g, s);
    end = max(end, carry_end);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xFFFFFFFFu, end, o);
      if (lane >= o) end = max(end, u);
    }
    int begin = __shfl_up_sync(0xFFFFFFFFu, end, 1);
    if (lane == 0) begin = carry_end;
    const int mine = s < g.S ? (end - begin + tile - 1) / tile : 0;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xFFFFFFFFu, sum, o);
      if (lane >= o) sum += u;
    }
    if (s < g.S) {
      start[s] = begin;
      tiles[s] = carry_tiles + sum - mine;
    }
    carry_end = __shfl_sync(0xFFFFFFFFu, end, 31);
    carry_tiles += __shfl_sync(0xFFFFFFFFu, sum, 31);
  }
  if (lane == 0) {
    start[g.S] = carry_end;
    tiles[g.S] = carry_tiles;
  }
}

// Segment of tile t (t < tiles[S]): the last s with tiles[s] <= t.
__device__ __forceinline__ int lora_find(const int* tiles, int S, int t) {
  int lo = 0, hi = S - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tiles[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// v - hi, and 0 beside an infinite hi (inf - inf would make a NaN of an infinite v).
__device__ __forceinline__ float low_half(float v, float hi) {
  return (__float_as_uint(hi) & 0x7FFFFFFFu) == 0x7F800000u ? 0.0f : v - hi;
}
// Two values as their packed high and low halves.
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16(a, b);
  lo = pack_bf16(low_half(a, __uint_as_float(hi << 16)), low_half(b, __uint_as_float(hi & 0xFFFF0000u)));
}
// Beside an infinite weight the high half alone gives the product (it has v's sign, and is 0 where v is); the low
// half's own sign, or its 0, would make a NaN of it.  So the low half is multiplied by a packed pair of weights with 0
// for infinities and NaNs.
__device__ __forceinline__ uint32_t finite_pair(uint32_t w) {
  return w & ~(((((w & 0x7F807F80u) + 0x00800080u) >> 15) & 0x00010001u) * 0xFFFFu);
}
// Eight values as v's two halves, 16 bytes each.
__device__ __forceinline__ void split_halves(const float (&f)[8], uint4& hi, uint4& lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) split2(f[2 * i], f[2 * i + 1], h[i], l[i]);
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
}

__device__ __forceinline__ uint32_t smem_align1024(const void* p) { return (ptx::smem_u32(p) + 1023u) & ~1023u; }

// Waits (bounded) for a ring's loads that may be in flight, the last ones issued:
// load j went to stage j % stages in that stage's round j / stages.
__device__ __forceinline__ void lora_drain(uint64_t* full, int issued, int stages, unsigned long long wait_ns) {
  volatile int never = 0;
  for (int j = max(0, issued - stages); j < issued; ++j)
    ptx::mbar_wait(ptx::smem_u32(full + j % stages), (j / stages) & 1, &never, wait_ns);
}

// ------------------------------------------------------------------ shrink
// A cluster of `ksplit` CTAs owns 128 rows; each CTA multiplies its share of
// the contraction and the cluster adds the partial tiles through distributed
// shared memory, in rank order, before one rounding to v's halves.  The ranks
// past R are set to 0 there: their sums of x times 0 are NaN beside an infinite x,
// and would make a NaN of the whole row in the second product.
// Bound: HBM, x once.  16384 x 5120, rank 16: 36 us, 4.7 TB/s (a plain read of
// as much, 28 us; about 8 us are the launch's start and the join); 16384 x 8192:
// 57 us.  Three to five stages, one or two CTAs to an SM measured the same.
struct ShrinkParams {
  LoraSegs g;
  const float* scaling;
  int C, R, Rp;
  int r_contig;            // weights (L, C, R) instead of (L, R, C)
  int ksplit, stages;
  int w_bytes;             // weight bytes of a stage
  __nv_bfloat16* v;
  uint32_t* status;
  unsigned long long wait_ns;
};
constexpr int kShrinkMaxStages = 8;
constexpr int kShrinkXBytes = kLoraBM * kLoraBK * 2;

__global__ void __launch_bounds__(128) lora_shrink_kernel(const __grid_constant__ CUtensorMap map_x,
                                                          const __grid_constant__ CUtensorMap map_x32,
                                                          const __grid_constant__ CUtensorMap map_w,
                                                          const ShrinkParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ int sh_start[kMaxLoraSegments + 1], sh_tiles[kMaxLoraSegments + 1], sh_ad[kMaxLoraSegments];
  __shared__ alignas(8) uint64_t sh_full[kShrinkMaxStages], sh_empty[kShrinkMaxStages], sh_done;
  __shared__ uint32_t sh_tmem;
  __shared__ int sh_abort, sh_issued;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kq = blockIdx.x % p.ksplit, tile = blockIdx.x / p.ksplit;
  const uint32_t ring = smem_align1024(smem_raw);
  const uint32_t stage_bytes = kShrinkXBytes + p.w_bytes;
  uint32_t ncols = 32;
  while ((int)ncols < p.Rp) ncols <<= 1;
  if (tid == 32) {
    ptx::prefetch_tmap(&map_x);
    ptx::prefetch_tmap(&map_w);
    for (int i = 0; i < p.stages; ++i) {
      ptx::mbar_init(ptx::smem_u32(&sh_full[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&sh_empty[i]), 1);
    }
    ptx::mbar_init(ptx::smem_u32(&sh_done), 1);
    ptx::fence_mbar_init();
    sh_abort = 0;
  }
  if (warp == 2) {
    ptx::tmem_alloc(ptx::smem_u32(&sh_tmem), ncols);
    ptx::tmem_relinquish();
  }
  if (warp == 0) lora_build_table(p.g, kLoraBM, sh_start, sh_tiles, sh_ad);
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = sh_tmem;
  const bool past = tile >= sh_tiles[p.g.S];
  const int s = past ? 0 : lora_find(sh_tiles, p.g.S, tile);
  const int row0 = sh_start[s] + (tile - sh_tiles[s]) * kLoraBM;
  const int end = min(sh_start[s + 1], row0 + kLoraBM);
  const int l = past ? -1 : sh_ad[s];
  const int vld = 2 * p.Rp;
  if (l < 0) {                                         // the whole cluster leaves
    if (!past && kq == 0) {
      const int n = (end - row0) * (vld / 8);
      uint4* dst = reinterpret_cast<uint4*>(p.v + (long long)row0 * vld);
      for (int i = tid; i < n; i += 128) dst[i] = make_uint4(0, 0, 0, 0);
    }
    if (warp == 2) ptx::tmem_dealloc(tmem, ncols);
    return;
  }
  ptx::griddep_launch_dependents();      // only now: a dependent CTA must not take this one's TMEM
  volatile int* abort = &sh_abort;
  const float scale = p.scaling ? p.scaling[l] : 1.0f;
  const int live = (end - row0 + 31) / 32;   // 32-row runs with rows in them; the products' other rows are not stored
  const int kiters = (p.C + kLoraBK - 1) / kLoraBK;
  const int i0 = (int)((long long)kiters * kq / p.ksplit), i1 = (int)((long long)kiters * (kq + 1) / p.ksplit);

  if (warp == 0) {
    if (lane == 0) {
      int issued = 0;
      for (int i = i0; i < i1; ++i, ++issued) {
        const int st = issued % p.stages, round = issued / p.stages;
        if (round > 0 && !ptx::mbar_wait(ptx::smem_u32(&sh_empty[st]), (round - 1) & 1, abort, p.wait_ns)) {
          atomicOr(p.status, kErrLoraWait);
          sh_abort = 1;
          break;
        }
        const uint32_t full = ptx::smem_u32(&sh_full[st]);
        const uint32_t dst = ring + st * stage_bytes;
        ptx::mbar_arrive_expect_tx(full, p.w_bytes + live * (kShrinkXBytes / 4));
        if (live == 4) {
          ptx::tma_load_2d(dst, &map_x, full, i * kLoraBK, row0);
        } else {
          for (int q = 0; q < live; ++q)
            ptx::tma_load_2d(dst + q * (kShrinkXBytes / 4), &map_x32, full, i * kLoraBK, row0 + q * 32);
        }
        if (p.r_contig) {
          for (int c = 0; c * 64 < p.R; ++c)
            ptx::tma_load_3d(dst + kShrinkXBytes + c * (kLoraBK * 128), &map_w, full, c * 64, i * kLoraBK, l);
        } else {
          ptx::tma_load_3d(dst + kShrinkXBytes, &map_w, full, i * kLoraBK, 0, l);
        }
      }
      sh_issued = issued;
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = ptx::idesc_bf16(128, p.Rp, 0, p.r_contig);
      for (int n = 0; n < i1 - i0; ++n) {
        const int st = n % p.stages;
        if (!ptx::mbar_wait(ptx::smem_u32(&sh_full[st]), (n / p.stages) & 1, abort, p.wait_ns)) {
          atomicOr(p.status, kErrLoraWait);
          sh_abort = 1;
          break;
        }
        ptx::tc_fence_after();
        const uint32_t xs = ring + st * stage_bytes, ws = xs + kShrinkXBytes;
#pragma unroll
        for (int j = 0; j < kLoraBK / 16; ++j) {
          const uint64_t ad = ptx::kmajor_sw128_desc(xs + j * 32);
          const uint64_t bd = p.r_contig ? ptx::mnmajor_sw128_desc(ws + j * 2048, kLoraBK * 128)
                                         : ptx::kmajor_sw128_desc(ws + j * 32);
          ptx::tc_mma_bf16(tmem, ad, bd, idesc, (n | j) != 0);
        }
        ptx::tc_commit(ptx::smem_u32(&sh_empty[st]));
      }
      ptx::tc_commit(ptx::smem_u32(&sh_done));
    }
    __syncwarp();
  }
  {
    volatile int never = 0;
    if (!ptx::mbar_wait(ptx::smem_u32(&sh_done), 0, &never, kLoraWaitSpan * p.wait_ns)) {
      atomicOr(p.status, kErrLoraWait);
      sh_abort = 1;
    }
  }
  ptx::tc_fence_after();
  const uint32_t lane_addr = tmem + ((uint32_t)(warp * 32) << 16);
  if (p.ksplit == 1) {
    const int m = row0 + tid;
    __nv_bfloat16* row = p.v + (long long)m * vld;
    for (int c = 0; c < p.Rp; c += 16) {
      uint32_t r[16];
      ptx::tmem_ld_32x32b_x16(lane_addr + c, r);
      ptx::tmem_wait_ld();
      if (m < end) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float f[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = c + h * 8 < p.R ? scale * __uint_as_float(r[h * 8 + i]) : 0.0f;
          uint4 hi, lo;
          split_halves(f, hi, lo);
          *reinterpret_cast<uint4*>(row + c + h * 8) = hi;
          *reinterpret_cast<uint4*>(row + p.Rp + c + h * 8) = lo;
        }
      }
    }
  } else {
    // the ring is free: every load was consumed and every product is done
    const int ld = p.Rp + 4;                           // floats between rows: 16-byte aligned, off the banks
    const uint32_t buf = ring;
    for (int c = 0; c < p.Rp; c += 16) {
      uint32_t r[16];
      ptx::tmem_ld_32x32b_x16(lane_addr + c, r);
      ptx::tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(buf + (tid * ld + c + i) * 4), "r"(r[i]),
                     "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3])
                     : "memory");
    }
    ptx::cluster_sync();
    const int rows = kLoraBM / p.ksplit, per_row = p.Rp / 8;
    for (int i = tid; i < rows * per_row; i += 128) {
      const int rr = kq * rows + i / per_row, c = (i % per_row) * 8;
      float f[8] = {};
      // remote loads take hundreds of cycles: two CTAs' at a time (ksplit is a power of two), added in rank order
      for (int q = 0; q < p.ksplit; q += 2) {
        float4 u[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t src = ptx::mapa(buf + (rr * ld + c) * 4, q + h);
          u[2 * h] = ptx::ld_cluster_f32x4(src);
          u[2 * h + 1] = ptx::ld_cluster_f32x4(src + 16);
        }
#pragma unroll
        for (int h = 0; h < 4; h += 2) {
          f[0] += u[h].x; f[1] += u[h].y; f[2] += u[h].z; f[3] += u[h].w;
          f[4] += u[h + 1].x; f[5] += u[h + 1].y; f[6] += u[h + 1].z; f[7] += u[h + 1].w;
        }
      }
      const int m = row0 + rr;
      if (m < end) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = c < p.R ? f[j] * scale : 0.0f;
        uint4 hi, lo;
        split_halves(f, hi, lo);
        __nv_bfloat16* row = p.v + (long long)m * vld;
        *reinterpret_cast<uint4*>(row + c) = hi;
        *reinterpret_cast<uint4*>(row + p.Rp + c) = lo;
      }
    }
    ptx::cluster_sync();                               // no CTA leaves while its tile is being read
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (sh_abort) {
    if (tid == 0) lora_drain(sh_full, sh_issued, p.stages, p.wait_ns);
    __syncthreads();
  }
  if (warp == 2) ptx::tmem_dealloc(tmem, ncols);
}

// ------------------------------------------------------------------ expand
// out = base + v W^T for 128 rows, 64 columns at a time: the base tile and the
// weight tile come by TMA into a ring, the two halves of v (loaded once) go
// through the same products into one of two TMEM accumulators, and two groups
// of four epilogue warps take tiles in turn: they add the base in place in
// shared memory and store the tile by TMA (32 full rows of a warp) or row by
// row (rows that end inside).  Two groups, as one spends most of a tile waiting
// (accumulator, shared memory, its store's read of the stage).  A product that
// comes out NaN is taken again from shared memory, infinite weights times v's high
// half alone (finite_pair): looking through the weights before the products took 1
// to 30 % of the kernel (ranks 16 to 128), looking for NaNs afterwards none.
// Bound: HBM, the base's read and the output's write.  16384 x 8192, rank 16:
// 90 us, 6.0 TB/s.  One epilogue group with CTAs for 2.3 rounds took 185 us.
struct ExpandParams {
  LoraSegs g;
  int C, Rp;
  int r_contig;            // weights (L, C, R) instead of (L, R, C)
  int nsplit, stages;
  int base_bytes, w_bytes; // of a stage: its output tile (the base is loaded there), its weights
  int w_row;               // bytes of a weight row in shared memory (r_contig): its swizzle, 32, 64 or 128
  int v_pieces;            // 128-byte wide tiles of v
  int more;                // a launch of the same call follows (no other may start before this one's output stands)
  const void* base;        // null: zeros
  long long base_ld;
  void* out;
  long long out_ld;
  uint32_t* status;
  unsigned long long wait_ns;
};
constexpr int kExpandBN = 64;
constexpr int kExpandMaxStages = 6;
constexpr int kExpandThreads = 320;     // TMA, MMA, eight epilogue warps

// v's tiles in shared memory: both halves side by side in one 128-byte row when
// they fit (Rp <= 32), else ceil(Rp / 64) tiles for each half.
__host__ __device__ constexpr int lora_v_pieces(int Rp) { return Rp <= 32 ? 1 : 2 * ((Rp + 63) / 64); }
// Byte offset of half h, 16 ranks j, in tiles of `tile` bytes.
__device__ __forceinline__ uint32_t lora_v_off(int Rp, int h, int j, uint32_t tile) {
  if (Rp <= 32) return (uint32_t)(h * Rp + j * 16) * 2;
  return (uint32_t)(h * ((Rp + 63) / 64) + j / 4) * tile + (uint32_t)(j % 4) * 32;
}

__device__ __forceinline__ float lds_bf16(uint32_t a) {
  unsigned short u;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(a));
  return __uint_as_float((uint32_t)u << 16);
}
// Byte `at` of a tile in the swizzle pattern of `row` (32, 64 or 128) bytes.
__device__ __forceinline__ uint32_t swizzled(uint32_t at, uint32_t row) {
  return at ^ (((at >> 7) & (row / 16 - 1)) << 4);
}
// v W^T of row r and column c of a tile, infinite weights times v's high half alone.  It ends at the first NaN:
// whole adapters of them would take milliseconds.
__device__ __noinline__ float lora_product(uint32_t vbuf, uint32_t ws, int Rp, int r_contig, int w_row, int r, int c) {
  float sum = 0.0f;
  for (int k = 0; k < Rp && !isnan(sum); ++k) {
    const uint32_t at = lora_v_off(Rp, 0, k / 16, kLoraBM * 128) + k % 16 * 2, high = swizzled(at + r * 128, 128);
    const uint32_t al = lora_v_off(Rp, 1, k / 16, kLoraBM * 128) + k % 16 * 2, low = swizzled(al + r * 128, 128);
    const float w = lds_bf16(ws + (r_contig ? (k / 64) * (kExpandBN * 128) + swizzled(c * w_row + k % 64 * 2, w_row)
                                            : swizzled(k * 128 + c * 2, 128)));
    sum = fmaf(lds_bf16(vbuf + high), w, sum);
    if (isfinite(w)) sum = fmaf(lds_bf16(vbuf + low), w, sum);
  }
  return sum;
}

// NaN if one of the values is.
__device__ __forceinline__ float any_nan(const uint32_t (&a)[32]) {
  float m = __uint_as_float(a[0]);
#pragma unroll
  for (int i = 1; i < 32; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(__uint_as_float(a[i])));
  return m;
}

template <typename O>
__device__ __forceinline__ void lora_add8(float (&f)[8], const uint4& q) {
  if constexpr (sizeof(O) == 2) {
    const O* t = reinterpret_cast<const O*>(&q);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] += lora_to_f32<O>(t[i]);
  }
}

// Two to an SM: left alone the compiler takes 64 registers and spills in the loop (117 us instead of 101, rank 32).
template <typename O>
__global__ void __launch_bounds__(kExpandThreads, 2)
lora_expand_kernel(const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_w,
                   const __grid_constant__ CUtensorMap map_base, const __grid_constant__ CUtensorMap map_base32,
                   const __grid_constant__ CUtensorMap map_out, const ExpandParams p) {
  constexpr int kPer16 = 16 / (int)sizeof(O);            // elements in 16 bytes
  constexpr int kBoxCols = 128 / (int)sizeof(O);         // columns of a 128-byte box row
  constexpr int kBoxes = kExpandBN / kBoxCols;           // boxes side by side in an output tile
  extern __shared__ uint8_t smem_raw[];
  __shared__ int sh_start[kMaxLoraSegments + 1], sh_tiles[kMaxLoraSegments + 1], sh_ad[kMaxLoraSegments];
  __shared__ alignas(8) uint64_t sh_full[kExpandMaxStages], sh_empty[kExpandMaxStages];
  __shared__ alignas(8) uint64_t sh_acc_full[2], sh_acc_empty[2], sh_v;
  __shared__ uint32_t sh_tmem;
  __shared__ int sh_abort, sh_issued;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int part = blockIdx.x % p.nsplit, tile = blockIdx.x / p.nsplit;
  if (warp == 0) lora_build_table(p.g, kLoraBM, sh_start, sh_tiles, sh_ad);
  __syncthreads();
  if (tile >= sh_tiles[p.g.S]) {
    ptx::griddep_wait();
    return;
  }
  const int s = lora_find(sh_tiles, p.g.S, tile);
  const int row0 = sh_start[s] + (tile - sh_tiles[s]) * kLoraBM;
  const int end = min(sh_start[s + 1], row0 + kLoraBM);
  const int l = sh_ad[s];
  const int nt = (p.C + kExpandBN - 1) / kExpandBN;
  const int t0 = (int)((long long)nt * part / p.nsplit), t1 = (int)((long long)nt * (part + 1) / p.nsplit);
  if (l < 0) {
    // no adapter: the base's rows (nothing to do in place), or zeros
    ptx::griddep_wait();
    if (p.base == p.out) return;
    const int c0 = t0 * kExpandBN, c1 = min(t1 * kExpandBN, p.C), per = (c1 - c0) / kPer16;
    for (int i = tid; i < (end - row0) * per; i += kExpandThreads) {
      const long long m = row0 + i / per;
      const int c = c0 + (i % per) * kPer16;
      uint4 q = make_uint4(0, 0, 0, 0);
      if (p.base) q = *reinterpret_cast<const uint4*>(static_cast<const O*>(p.base) + m * p.base_ld + c);
      *reinterpret_cast<uint4*>(static_cast<O*>(p.out) + m * p.out_ld + c) = q;
    }
    return;
  }
  const int rc = (p.Rp + 63) / 64;                       // 64-wide pieces of the rank
  const uint32_t vbuf = smem_align1024(smem_raw);        // v's tiles of 128 rows x 128 bytes
  const uint32_t ring = vbuf + p.v_pieces * (kLoraBM * 128);
  const int live = (end - row0 + 31) / 32;               // 32-row runs with rows in them
  const uint32_t stage_bytes = p.base_bytes + p.w_bytes;
  if (tid == 32) {
    for (int i = 0; i < p.stages; ++i) {
      ptx::mbar_init(ptx::smem_u32(&sh_full[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&sh_empty[i]), 4);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(ptx::smem_u32(&sh_acc_full[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&sh_acc_empty[i]), 4);
    }
    ptx::mbar_init(ptx::smem_u32(&sh_v), 1);
    ptx::fence_mbar_init();
    sh_abort = 0;
  }
  if (warp == 2) {
    ptx::tmem_alloc(ptx::smem_u32(&sh_tmem), 2 * kExpandBN);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (p.more) ptx::griddep_launch_dependents();
  const uint32_t tmem = sh_tmem;
  volatile int* abort = &sh_abort;
  const int n = t1 - t0;

  if (warp == 0) {
    if (lane == 0) {
      int issued = 0;
      for (int i = 0; i < n; ++i, ++issued) {
        const int st = i % p.stages, round = i / p.stages;
        if (round > 0 && !ptx::mbar_wait(ptx::smem_u32(&sh_empty[st]), (round - 1) & 1, abort, p.wait_ns)) {
          atomicOr(p.status, kErrLoraWait);
          sh_abort = 1;
          break;
        }
        const uint32_t full = ptx::smem_u32(&sh_full[st]);
        const uint32_t dst = ring + st * stage_bytes;
        const int c = (t0 + i) * kExpandBN;
        ptx::mbar_arrive_expect_tx(full, p.w_bytes + (p.base ? live * (p.base_bytes / 4) : 0));
        if (p.r_contig) {
          for (int j = 0; j < rc; ++j)
            ptx::tma_load_3d(dst + p.base_bytes + j * (kExpandBN * 128), &map_w, full, j * 64, c, l);
        } else {
          ptx::tma_load_3d(dst + p.base_bytes, &map_w, full, c, 0, l);
        }
        if (p.base)
          for (int j = 0; j < kBoxes; ++j) {
            const uint32_t d = dst + j * (kLoraBM * 128);
            if (live == 4) {
              ptx::tma_load_2d(d, &map_base, full, c + j * kBoxCols, row0);
            } else {
              for (int q = 0; q < live; ++q)
                ptx::tma_load_2d(d + q * (32 * 128), &map_base32, full, c + j * kBoxCols, row0 + q * 32);
            }
          }
        if (i == 0) {
          // v comes from the launch before this one; weights and base do not
          ptx::griddep_wait();
          const uint32_t vb = ptx::smem_u32(&sh_v);
          ptx::mbar_arrive_expect_tx(vb, p.v_pieces * (kLoraBM * 128));
          for (int j = 0; j < p.v_pieces; ++j)
            ptx::tma_load_3d(vbuf + j * (kLoraBM * 128), &map_v, vb, p.v_pieces == 1 ? 0 : (j % rc) * 64,
                             p.v_pieces == 1 ? 0 : j / rc, row0);
        }
      }
      sh_issued = issued;
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = ptx::idesc_bf16(128, kExpandBN, 0, !p.r_contig);
      ptx::griddep_wait();       // a wait's limit must not count the launch before
      bool ok = ptx::mbar_wait(ptx::smem_u32(&sh_v), 0, abort, p.wait_ns);
      for (int i = 0; ok && i < n; ++i) {
        const int st = i % p.stages, buf = i & 1;
        if (i >= 2) ok = ptx::mbar_wait(ptx::smem_u32(&sh_acc_empty[buf]), ((i >> 1) - 1) & 1, abort, p.wait_ns);
        ok = ok && ptx::mbar_wait(ptx::smem_u32(&sh_full[st]), (i / p.stages) & 1, abort, p.wait_ns);
        if (!ok) break;
        ptx::tc_fence_after();
        const uint32_t ws = ring + st * stage_bytes + p.base_bytes;
        for (int h = 0; h < 2; ++h)
          for (int j = 0; j < p.Rp / 16; ++j) {
            const uint64_t ad = ptx::kmajor_sw128_desc(vbuf + lora_v_off(p.Rp, h, j, kLoraBM * 128));
            const uint64_t bd = p.r_contig ? ptx::kmajor_desc(ws + (j / 4) * (kExpandBN * 128) + (j % 4) * 32, p.w_row)
                                           : ptx::mnmajor_sw128_desc(ws + j * 2048, 8192);
            ptx::tc_mma_bf16(tmem + buf * kExpandBN, ad, bd, idesc, (h | j) != 0);
          }
        ptx::tc_commit(ptx::smem_u32(&sh_acc_full[buf]));
      }
      if (!ok) {
        atomicOr(p.status, kErrLoraWait);
        sh_abort = 1;
      }
    }
    __syncwarp();
  } else {
    // epilogue: warp w may read TMEM lanes 32 (w % 4) .. + 31; tile i goes to group i % 2, accumulator i % 2
    const int q = warp & 3, group = (warp - 2) >> 2;
    const int r = q * 32 + lane;                          // row of the tile
    const bool full_rows = row0 + q * 32 + 32 <= end;
    const uint32_t lane_addr = tmem + ((uint32_t)(q * 32) << 16);
    const uint32_t sw = (uint32_t)(r & 7);
    bool ok = true;
    ptx::griddep_wait();
    for (int i = group; i < n; i += 2) {
      const int st = i % p.stages, buf = group;
      if (i >= 2 && lane == 0) {
        // the last tile's stage may be loaded again once its store has been read
        ptx::bulk_wait_read<0>();
        ptx::mbar_arrive(ptx::smem_u32(&sh_empty[(i - 2) % p.stages]));
      }
      __syncwarp();
      const uint32_t tile_s = ring + st * stage_bytes + r * 128;
      // the loads' own barrier makes the base tile visible to these threads
      ok = ptx::mbar_wait(ptx::smem_u32(&sh_full[st]), (i / p.stages) & 1, abort, p.wait_ns) &&
           ptx::mbar_wait(ptx::smem_u32(&sh_acc_full[buf]), (i >> 1) & 1, abort, p.wait_ns);
      if (!__all_sync(0xFFFFFFFFu, ok)) {
        if (lane == 0) {
          atomicOr(p.status, kErrLoraWait);
          sh_abort = 1;
        }
        break;
      }
      ptx::tc_fence_after();
      const int c = (t0 + i) * kExpandBN;
      const bool mine = row0 + r < end;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t a[32];
        ptx::tmem_ld_32x32b_x32(lane_addr + buf * kExpandBN + half * 32, a);
        ptx::tmem_wait_ld();
        if (__any_sync(0xFFFFFFFFu, isnan(any_nan(a)) && mine)) {
          ptx::mbar_wait(ptx::smem_u32(&sh_v), 0, abort, p.wait_ns);   // long done: these threads see v by it
          const uint32_t ws = ring + st * stage_bytes + p.base_bytes;
#pragma unroll
          for (int u = 0; u < 32; ++u)
            if (isnan(__uint_as_float(a[u])) && mine)
              a[u] = __float_as_uint(lora_product(vbuf, ws, p.Rp, p.r_contig, p.w_row, r, half * 32 + u));
          __syncwarp();
        }
#pragma unroll
        for (int u = 0; u < 32; u += kPer16) {
          const int col = half * 32 + u;
          const uint32_t addr = tile_s + (col / kBoxCols) * (kLoraBM * 128) + ((((col % kBoxCols) / kPer16) ^ sw) << 4);
          uint4 o;
          if constexpr (sizeof(O) == 2) {
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(a[u + j]);
            if (p.base) {
              uint4 b;
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w) : "r"(addr));
              lora_add8<O>(f, b);
            }
            O t[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = lora_from_f32<O>(f[j]);
            o = *reinterpret_cast<const uint4*>(t);
          } else {
            o = make_uint4(a[u], a[u + 1], a[u + 2], a[u + 3]);
            if (p.base) {
              uint4 b;
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w) : "r"(addr));
              o.x = __float_as_uint(__uint_as_float(o.x) + __uint_as_float(b.x));
              o.y = __float_as_uint(__uint_as_float(o.y) + __uint_as_float(b.y));
              o.z = __float_as_uint(__uint_as_float(o.z) + __uint_as_float(b.z));
              o.w = __float_as_uint(__uint_as_float(o.w) + __uint_as_float(b.w));
            }
          }
          if (full_rows) {
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(o.x), "r"(o.y), "r"(o.z), "r"(o.w)
                         : "memory");
          } else if (mine && c + col < p.C) {
            *reinterpret_cast<uint4*>(static_cast<O*>(p.out) + (long long)(row0 + r) * p.out_ld + c + col) = o;
          }
        }
      }
      ptx::tc_fence_before();
      if (full_rows) {
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive(ptx::smem_u32(&sh_acc_empty[buf]));
          for (int j = 0; j < kBoxes; ++j)
            if (c + j * kBoxCols < p.C)
              ptx::tma_store_2d(&map_out, ring + st * stage_bytes + j * (kLoraBM * 128) + q * (32 * 128),
                                c + j * kBoxCols, row0 + q * 32);
          ptx::bulk_commit();
        }
      } else {
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sh_acc_empty[buf]));
      }
    }
    if (lane == 0) ptx::bulk_wait<0>();
    __syncwarp();
  }
  ptx::griddep_wait();
  ptx::tc_fence_before();
  __syncthreads();
  if (sh_abort) {
    if (tid == 32) {
      // v's load, the ring's, and (before their accumulators go) the products in flight
      volatile int never = 0;
      ptx::mbar_wait(ptx::smem_u32(&sh_v), 0, &never, p.wait_ns);
      lora_drain(sh_full, sh_issued, p.stages, p.wait_ns);
      ptx::tc_commit(ptx::smem_u32(&sh_v));
      ptx::mbar_wait(ptx::smem_u32(&sh_v), 1, &never, p.wait_ns);
    }
    __syncthreads();
  }
  if (warp == 2) ptx::tmem_dealloc(tmem, 2 * kExpandBN);
}

// --------------------------------------------------------- weight gradients
// G_l[c, r] = sum over adapter l's rows m of z[m, c] v[m, r], both operands with
// the contraction along their rows, 128 columns c at a time.
//
// The work of a (v, z) pair is one axis of 64-row stages: column tiles, within a
// tile the segments by adapter, then in order.  CTA b of G takes the b-th G-th of
// the first pair's axis and then of the second's, so that all end together
// whatever the segments' lengths (whole pieces dealt out left the last CTAs with
// 15 % more), and a pair's sums do not depend on the other's presence.
// A CTA keeps one of two accumulators until the adapter or the tile changes and
// then writes an fp32 partial; a second launch adds a block's partials in CTA
// order.  Loads run ahead across those ends.  Rows of a stage past its segment's
// end belong to others: they are zeroed in shared memory, as 0 * NaN would not
// be 0.  Where v's halves have accumulators of their own (Rp <= 32) the low one's
// sum counts only where it is finite: beside an infinite z the high one's is the
// result (finite_pair).  Above, an infinite z gives NaN for an infinity; sums of
// their own took 6 to 14 % of the kernel there (ranks 64 and 128).
// Bound: HBM, z once (two CTAs to an SM keep 128 KB of it on the way).  16384
// rows, 5120 + 8192 columns, rank 16 (436 MB): 87 us, 5.0 TB/s, and 6 us for the
// sums; one CTA to an SM took half as long again, its products' issue and waits
// (1100 cycles a stage) lying bare.
struct WgradJob {
  int C;                     // columns
  int ctiles;                // 128-column tiles
  int ctas;                  // CTAs that share the axis (the first ones of the grid)
  int transposed;            // output (L, C, R) instead of (L, R, C)
  void* out;
  // partial of (tile i, adapter l, CTA b): slot i * slots + wgrad_slot(l) + b, [128][Rp] floats; the slots of what
  // occurs are distinct, as a step along the axis raises i * slots + wgrad_slot(l) or b
  float* part;
};
// Slots of a tile: an adapter's own number, or, when there are more adapters than segments, the number of segments
// with rows of lower ones.  A table of many adapters, of which a batch carries a few, takes no more than the few.
__host__ __device__ constexpr int wgrad_slots(int L, int S) { return L < S ? L : S; }

struct WgradParams {
  LoraSegs g;
  int R, Rp, stages;
  WgradJob job[2];           // the second without columns when there is one pair
  uint32_t* status;
  unsigned long long wait_ns;
};
constexpr int kWgradBC = 128;
constexpr int kWgradBT = 64;        // rows of a stage
constexpr int kWgradMaxStages = 6;
constexpr int kWgradZBytes = kWgradBC * kWgradBT * 2;
constexpr int kWgradMaxCtas = 2 * 148;   // two to an SM
constexpr int kWgradThreads = 192;   // TMA, MMA, four epilogue warps

__host__ __device__ constexpr int wgrad_table_bytes(int S) { return (6 * S + 2) * 4; }
__device__ __forceinline__ long long wgrad_cut(long long total, int b, int ctas) { return total * b / ctas; }

__global__ void __launch_bounds__(kWgradThreads)
lora_wgrad_kernel(const __grid_constant__ CUtensorMap map_v0, const __grid_constant__ CUtensorMap map_z0,
                  const __grid_constant__ CUtensorMap map_v1, const __grid_constant__ CUtensorMap map_z1,
                  const __grid_constant__ WgradParams p) {
  extern __shared__ uint8_t smem_raw[];
  // tables of the segments: start and stages before (in order), adapter; by adapter: segment, stages before, slot
  int* sh_start = reinterpret_cast<int*>(smem_raw);
  int* sh_tiles = sh_start + p.g.S + 1;
  int* sh_ad = sh_tiles + p.g.S + 1;
  int* sh_seg = sh_ad + p.g.S;
  int* sh_pre = sh_seg + p.g.S;
  int* sh_slot = sh_pre + p.g.S;
  const int slots = wgrad_slots(p.g.L, p.g.S);
  __shared__ int sh_n;
  __shared__ alignas(8) uint64_t sh_full[kWgradMaxStages], sh_empty[kWgradMaxStages];
  __shared__ alignas(8) uint64_t sh_acc_full[2], sh_acc_empty[2], sh_done;
  __shared__ uint32_t sh_tmem;
  __shared__ int sh_abort, sh_issued;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rc = (p.Rp + 63) / 64;
  const uint32_t ring = smem_align1024(smem_raw + wgrad_table_bytes(p.g.S));
  const int v_pieces = lora_v_pieces(p.Rp);
  const uint32_t stage_bytes = kWgradZBytes + v_pieces * (kWgradBT * 128);
  // Rp <= 32: both halves lie side by side, one product of 2 Rp columns; their accumulators are added at the end
  const bool joined = p.Rp <= 32;
  const int acc_cols = joined ? 2 * p.Rp : p.Rp;
  uint32_t ncols = 32;
  while ((int)ncols < 2 * acc_cols) ncols <<= 1;
  if (warp == 0) lora_build_table(p.g, kWgradBT, sh_start, sh_tiles, sh_ad);
  if (tid == 32) {
    for (int i = 0; i < p.stages; ++i) {
      ptx::mbar_init(ptx::smem_u32(&sh_full[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&sh_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(ptx::smem_u32(&sh_acc_full[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&sh_acc_empty[i]), 4);
    }
    ptx::mbar_init(ptx::smem_u32(&sh_done), 1);
    ptx::fence_mbar_init();
    sh_abort = 0;
    sh_n = 0;
  }
  if (warp == 2) {
    ptx::tmem_alloc(ptx::smem_u32(&sh_tmem), ncols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  ptx::griddep_launch_dependents();
  // place of every segment with rows and an adapter among them, by adapter and then in order
  for (int s = tid; s < p.g.S; s += kWgradThreads) {
    const int l = sh_ad[s], n = sh_tiles[s + 1] - sh_tiles[s];
    if (l < 0 || n == 0) continue;
    int rank = 0, pre = 0, lower = 0;
    for (int o = 0; o < p.g.S; ++o) {
      const int lo = sh_ad[o], no = sh_tiles[o + 1] - sh_tiles[o];
      if (lo >= 0 && no > 0 && (lo < l || (lo == l && o < s))) {
        ++rank;
        pre += no;
        lower += lo < l;
      }
    }
    sh_seg[rank] = s;
    sh_pre[rank] = pre;
    sh_slot[rank] = slots == p.g.L ? l : lower;
    atomicAdd(&sh_n, 1);
  }
  __syncthreads();
  const int nseg = sh_n;
  const uint32_t tmem = sh_tmem;
  volatile int* abort = &sh_abort;
  const int last = nseg > 0 ? sh_seg[nseg - 1] : 0;
  const int W = nseg > 0 ? sh_pre[nseg - 1] + sh_tiles[last + 1] - sh_tiles[last] : 0;   // stages of a column tile
  // this CTA's range of a job's axis
  auto range = [&](int j, long long& t0, long long& t1) {
    const long long total = (long long)W * p.job[j].ctiles;
    const bool has = (int)blockIdx.x < p.job[j].ctas;
    t0 = has ? wgrad_cut(total, blockIdx.x, p.job[j].ctas) : 0;
    t1 = has ? wgrad_cut(total, blockIdx.x + 1, p.job[j].ctas) : 0;
  };

  // A run of stages in one segment and tile; every role walks the same runs.
  struct Run {
    int tile, adapter, slot, row, end, n;
    bool flush;                    // the accumulator ends with it
  };
  auto run = [&](long long t, long long t1) {
    Run w;
    w.tile = (int)(t / W);
    const int q = (int)(t - (long long)w.tile * W);
    int lo = 0, hi = nseg - 1;     // the last place whose stages start at or before q
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (sh_pre[mid] <= q) lo = mid;
      else hi = mid - 1;
    }
    const int s = sh_seg[lo], after = lo + 1 < nseg ? sh_pre[lo + 1] : W;
    w.adapter = sh_ad[s];
    w.slot = sh_slot[lo];
    w.row = sh_start[s] + (q - sh_pre[lo]) * kWgradBT;
    w.end = sh_start[s + 1];
    const long long left = t1 - t;
    w.n = left < after - q ? (int)left : after - q;
    w.flush = t + w.n == t1 || q + w.n == W || (q + w.n == after && sh_ad[sh_seg[lo + 1]] != w.adapter);
    return w;
  };

  if (warp == 0) {
    if (lane == 0) {
      ptx::griddep_wait();
      int issued = 0, st = 0, phase = 1;          // a fresh ring is empty: its (phase 1) wait passes at once
      bool ok = true;
      for (int jb = 0; jb < 2; ++jb) {
        long long t, t1;
        range(jb, t, t1);
        const CUtensorMap* map_v = jb ? &map_v1 : &map_v0;
        const CUtensorMap* map_z = jb ? &map_z1 : &map_z0;
        while (ok && t < t1) {
          const Run w = run(t, t1);
          const int c = w.tile * kWgradBC;
          for (int i = 0; i < w.n; ++i) {
            if (!ptx::mbar_wait(ptx::smem_u32(&sh_empty[st]), phase, abort, p.wait_ns)) {
              atomicOr(p.status, kErrLoraWait);
              sh_abort = 1;
              ok = false;
              break;
            }
            const uint32_t full = ptx::smem_u32(&sh_full[st]);
            const uint32_t dst = ring + st * stage_bytes;
            const int m = w.row + i * kWgradBT;
            ptx::mbar_arrive_expect_tx(full, stage_bytes);
            for (int j = 0; j < kWgradBC / 64; ++j)
              ptx::tma_load_2d(dst + j * (kWgradBT * 128), map_z, full, c + j * 64, m);
            for (int j = 0; j < v_pieces; ++j)
              ptx::tma_load_3d(dst + kWgradZBytes + j * (kWgradBT * 128), map_v, full, joined ? 0 : (j % rc) * 64,
                               joined ? 0 : j / rc, m);
            ++issued;
            if (++st == p.stages) {
              st = 0;
              phase ^= 1;
            }
          }
          t += w.n;
        }
      }
      sh_issued = issued;
    }
    __syncwarp();
  } else if (warp == 1) {
    const uint32_t idesc = ptx::idesc_bf16(128, acc_cols, 1, 1);
    ptx::griddep_wait();         // a wait's limit must not count the launch before
    int n = 0, st = 0, phase = 0;
    bool ok = true, fresh = true;
    for (int jb = 0; jb < 2; ++jb) {
      long long t, t1;
      range(jb, t, t1);
      while (ok && t < t1) {
        const Run w = run(t, t1);
        const int buf = n & 1;
        const uint32_t acc = tmem + buf * acc_cols;
        if (fresh && n >= 2) ok = ptx::mbar_wait(ptx::smem_u32(&sh_acc_empty[buf]), ((n >> 1) - 1) & 1, abort, p.wait_ns);
        for (int i = 0; i < w.n; ++i) {
          ok = ok && ptx::mbar_wait(ptx::smem_u32(&sh_full[st]), phase, abort, p.wait_ns);
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (!ok) {
            if (lane == 0) {
              atomicOr(p.status, kErrLoraWait);
              sh_abort = 1;
            }
            break;
          }
          const int rows = min(kWgradBT, w.end - w.row - i * kWgradBT);
          const int ksteps = (rows + 15) / 16;
          const uint32_t zs = ring + st * stage_bytes, vs = zs + kWgradZBytes;
          if (rows % 16 != 0) {
            // rows past the end, up to the last product's 16: 128 bytes in every tile, whatever the swizzle
            const int tiles = kWgradBC / 64 + v_pieces, per = (ksteps * 16 - rows) * 8;
            for (int e = lane; e < tiles * per; e += 32) {
              const uint32_t a = zs + (e / per) * (kWgradBT * 128) + rows * 128 + (e % per) * 16;
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(a), "r"(0) : "memory");
            }
            ptx::fence_proxy_async_smem();
            __syncwarp();
          }
          if (lane == 0) {
            ptx::tc_fence_after();
            // 16 rows further: 2048 bytes, 128 in a descriptor's address field
            const uint64_t ad = ptx::mnmajor_sw128_desc(zs, kWgradBT * 128);
            for (int h = 0; h < (joined ? 1 : 2); ++h) {
              const uint64_t bd = ptx::mnmajor_sw128_desc(vs + h * rc * (kWgradBT * 128), kWgradBT * 128);
#pragma unroll
              for (int j = 0; j < kWgradBT / 16; ++j)
                if (j < ksteps) ptx::tc_mma_bf16(acc, ad + j * 128, bd + j * 128, idesc, !fresh || (i | j | h) != 0);
            }
            ptx::tc_commit(ptx::smem_u32(&sh_empty[st]));
          }
          __syncwarp();
          if (++st == p.stages) {
            st = 0;
            phase ^= 1;
          }
        }
        fresh = w.flush;
        if (w.flush) {
          if (ok && lane == 0) ptx::tc_commit(ptx::smem_u32(&sh_acc_full[buf]));
          __syncwarp();
          ++n;
        }
        t += w.n;
      }
    }
    if (lane == 0) ptx::tc_commit(ptx::smem_u32(&sh_done));
    __syncwarp();
  } else {
    ptx::griddep_wait();
    const int q = warp & 3;                      // TMEM lanes this warp may read: 32 q ..
    int n = 0;
    bool ok = true;
    for (int jb = 0; jb < 2; ++jb) {
      long long t, t1;
      range(jb, t, t1);
      while (ok && t < t1) {
        const Run w = run(t, t1);
        t += w.n;
        if (!w.flush) continue;
        const int buf = n & 1;
        // an accumulator takes as many stages as there are rows: this wait spans many of theirs
        ok = ptx::mbar_wait(ptx::smem_u32(&sh_acc_full[buf]), (n >> 1) & 1, abort, kLoraWaitSpan * p.wait_ns);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) {
          if (lane == 0) {
            atomicOr(p.status, kErrLoraWait);
            sh_abort = 1;
          }
          break;
        }
        ptx::tc_fence_after();
        const int c = q * 32 + lane;
        const bool in = w.tile * kWgradBC + c < p.job[jb].C;
        float* dst = p.job[jb].part +
                     ((long long)w.tile * slots + w.slot + blockIdx.x) * (kWgradBC * p.Rp) + c * p.Rp;
        const uint32_t lane_addr = tmem + ((uint32_t)(q * 32) << 16) + buf * acc_cols;
        for (int r = 0; r < p.Rp; r += 16) {
          uint32_t a[16], b[16];
          ptx::tmem_ld_32x32b_x16(lane_addr + r, a);
          if (joined) ptx::tmem_ld_32x32b_x16(lane_addr + p.Rp + r, b);
          ptx::tmem_wait_ld();
          if (in) {
            if (joined)
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float l = __uint_as_float(b[i]);
                a[i] = __float_as_uint(__uint_as_float(a[i]) + (isfinite(l) ? l : 0.0f));
              }
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              *reinterpret_cast<uint4*>(dst + r + i) = make_uint4(a[i], a[i + 1], a[i + 2], a[i + 3]);
          }
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sh_acc_empty[buf]));
        ++n;
      }
    }
  }
  ptx::griddep_wait();
  {
    volatile int never = 0;
    if (!ptx::mbar_wait(ptx::smem_u32(&sh_done), 0, &never, kLoraWaitSpan * p.wait_ns)) {
      atomicOr(p.status, kErrLoraWait);
      sh_abort = 1;
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (sh_abort) {
    if (tid == 0) lora_drain(sh_full, sh_issued, p.stages, p.wait_ns);
    __syncthreads();
  }
  if (warp == 2) ptx::tmem_dealloc(tmem, ncols);
}

// Columns of a block of the sums: a whole tile while its shared memory stays small (fewer, longer blocks: one
// round of them for 8 adapters of rank 16).
__host__ __device__ constexpr int wgrad_sum_cols(int Rp) { return Rp <= 64 ? 128 : 64; }
// Adds an adapter's partials in CTA order: a block takes columns c of one
// adapter and writes its (c, r) tile through shared memory, so both output
// orders store runs.
template <typename O>
__global__ void __launch_bounds__(256) lora_wgrad_sum_kernel(const __grid_constant__ WgradParams p) {
  const int ncols = wgrad_sum_cols(p.Rp);
  extern __shared__ float sh[];                            // [columns][ld], then the segments' tables
  const int ld = p.Rp + 1;
  int* sh_start = reinterpret_cast<int*>(sh + ncols * ld);
  int* sh_tiles = sh_start + p.g.S + 1;
  __shared__ int sh_before, sh_mine, sh_all, sh_lower;
  __shared__ bool sh_has[kWgradMaxCtas];
  const int tid = threadIdx.x, lane = tid & 31;
  const int blocks0 = (p.job[0].C + ncols - 1) / ncols;
  const int which = (int)blockIdx.x >= blocks0;
  const WgradJob& job = p.job[which];
  const int c0 = ((int)blockIdx.x - (which ? blocks0 : 0)) * ncols, l = blockIdx.y;
  if (tid == 0) sh_before = sh_mine = sh_all = sh_lower = 0;
  if (tid < 32) lora_build_table(p.g, kWgradBT, sh_start, sh_tiles);
  __syncthreads();
  // stages of a column tile: of lower adapters, of this one, of all; segments with rows of lower adapters
  int before = 0, mine = 0, all = 0, lower = 0;
  for (int s = tid; s < p.g.S; s += 256) {
    const int a = lora_adapter(p.g, s), n = a < 0 ? 0 : sh_tiles[s + 1] - sh_tiles[s];
    all += n;
    before += a < l ? n : 0;
    mine += a == l ? n : 0;
    lower += a < l && n > 0;
  }
  before = __reduce_add_sync(0xFFFFFFFFu, before);
  mine = __reduce_add_sync(0xFFFFFFFFu, mine);
  all = __reduce_add_sync(0xFFFFFFFFu, all);
  lower = __reduce_add_sync(0xFFFFFFFFu, lower);
  if (lane == 0) {
    atomicAdd(&sh_lower, lower);
    atomicAdd(&sh_before, before);
    atomicAdd(&sh_mine, mine);
    atomicAdd(&sh_all, all);
  }
  __syncthreads();
  const int tile = c0 / kWgradBC;
  const long long total = (long long)sh_all * job.ctiles;
  const long long lo = (long long)tile * sh_all + sh_before, hi = lo + sh_mine;
  // CTA of a position t: the last b with total * b / ctas <= t
  int b0 = 0, b1 = -1;
  if (sh_mine > 0) {
    b0 = (int)(((lo + 1) * job.ctas + total - 1) / total) - 1;
    b1 = (int)((hi * job.ctas + total - 1) / total) - 1;
  }
  // with fewer stages than CTAs some have none, and wrote no partial
  for (int b = b0 + tid; b <= b1; b += 256)
    sh_has[b - b0] = wgrad_cut(total, b, job.ctas) != wgrad_cut(total, b + 1, job.ctas);
  __syncthreads();
  ptx::griddep_wait();
  const int cols = min(ncols, job.C - c0), quads = p.Rp / 4;
  const int slots = wgrad_slots(p.g.L, p.g.S);
  const float* part = job.part + ((long long)tile * slots + (slots == p.g.L ? l : sh_lower)) * (kWgradBC * p.Rp) +
                      (long long)(c0 % kWgradBC) * p.Rp;
  for (int e = tid; e < cols * quads; e += 256) {
    const int c = e / quads, r = (e % quads) * 4;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int b = b0; b <= b1; ++b) {
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (sh_has[b - b0]) v = *reinterpret_cast<const float4*>(part + (long long)b * (kWgradBC * p.Rp) + c * p.Rp + r);
      sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
    }
    float* d = sh + c * ld + r;
    d[0] = sum.x; d[1] = sum.y; d[2] = sum.z; d[3] = sum.w;
  }
  __syncthreads();
  O* out = static_cast<O*>(job.out);
  if (job.transposed) {
    O* dst = out + ((long long)l * job.C + c0) * p.R;
    for (int e = tid; e < cols * p.R; e += 256) dst[e] = lora_from_f32<O>(sh[e / p.R * ld + e % p.R]);
  } else {
    for (int e = tid; e < p.R * ncols; e += 256) {
      const int r = e / ncols, c = e % ncols;
      if (c < cols) out[((long long)l * p.R + r) * job.C + c0 + c] = lora_from_f32<O>(sh[c * ld + r]);
    }
  }
}

}  // namespace mxgg
