// qz_kv4.cuh -- the paged 4-bit KV cache: block tables and slot maps built from
// request lengths, 4-bit append and read back, and decode attention over the
// packed pages.
//
// Pool layout (one layer): uint8 [pages, n_kv, ps * (hd + 8)]. One block is a
// page (ps positions) of one kv head:
//   K codes [ps, hd / 2] | V codes [ps, hd / 2] | K (s, z) [ps, 2] | V (s, z) [ps, 2]
// Codes are unsigned 4-bit, two per byte, element 2j in the low half of byte
// j; s (step) and z (zero) are bf16. A row stands for z + c * s.
//
// z and s are bf16 because they are read with every row: 4 bytes beside hd/2
// of codes instead of 8 (11 % of the traffic at hd = 64). Rounding them costs
// nothing in the codes, which are chosen against the rounded z and s; only the
// smallest values of a row can fall below z, by at most |z| * 2^-9.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "qz_device.cuh"

namespace qz {
namespace kv4 {

enum : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ f2_t f2_mul(f2_t a, f2_t b) {
  f2_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f2_t f2_add(f2_t a, f2_t b) {
  f2_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f2_t f2_set(float a, float b) {
  return f2_pack(__float_as_uint(a), __float_as_uint(b));
}

// n consecutive elements as fp32; `vec`: p is 16-byte aligned and n * sizeof(T)
// a multiple of 16.
template <int n, class T>
__device__ __forceinline__ void load_row(const T* p, bool vec, float (&x)[n]) {
  if (vec) {
    constexpr int per = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < n / per; ++j) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + j);
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int k = 0; k < per; ++k) x[j * per + k] = to_f(e[k]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < n; ++j) x[j] = to_f(p[j]);
  }
}

// (s, z) of a packed parameter word: s in the low half, z in the high half.
__device__ __forceinline__ float par_s(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float par_z(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// ---------------------------------------------------------------------------
// block tables and slot maps
// ---------------------------------------------------------------------------
// Requests in order: request b holds lens[b] positions and new_rows[b] rows
// join. It is granted when its rows fit the row capacity, its pages the
// table's width, and the free pages left by the requests before it suffice;
// a refused request keeps its length and its rows get slot -1. Page j of a
// request's new ones is free[used + (pages of the requests before it) + j].
//
// Latency-bound (a few hundred bytes to about a megabyte): one launch, no
// atomics. Every CTA scans all requests in shared memory, then CTAs share out
// the rows (binary search of the row's request). Where lens or used are updated
// in place, kPlanCluster CTAs form one cluster whose barrier separates the
// reading from the writing; else a CTA for every 1024 rows needs no barrier
// (1024 requests, 49000 rows: 7.0 us, in a cluster of 8 13.6 us).
constexpr int kPlanThreads = 1024;
constexpr int kPlanPer = 4;
constexpr int kPlanMaxB = kPlanThreads * kPlanPer;
constexpr int kPlanCluster = 8;

struct PlanArgs {
  const int64_t* lens;
  const int64_t* joins;
  int32_t* table;
  const int32_t* free_pages;
  const int64_t* used;
  int64_t* cu_rows;
  int64_t* lens_out;
  int64_t* used_out;
  int64_t* slots;
  int64_t* positions;
  int64_t width, n_free, rows;
  int B, shift;   // page size = 1 << shift
};

__host__ __device__ constexpr int plan_smem(int B) { return 512 + B * 16 + 16; }

__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

// Exclusive prefix of v over the block; total: the sum.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* warp_sums, int64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int64_t w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  *total = warp_sums[31];
  return x - v + (warp ? warp_sums[warp - 1] : 0);
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanArgs a) {
  extern __shared__ __align__(16) uint8_t plan_sh[];
  int64_t* warp_sums = reinterpret_cast<int64_t*>(plan_sh);             // [32] (+ 32 spare)
  int64_t* s_len = reinterpret_cast<int64_t*>(plan_sh + 512);           // [B]
  int32_t* s_page = reinterpret_cast<int32_t*>(s_len + a.B);            // [B] free index, -1: refused
  int32_t* s_cu = s_page + a.B;                                         // [B + 1]
  const int tid = threadIdx.x, B = a.B, shift = a.shift;
  const int64_t ps = int64_t(1) << shift, cap = a.width << shift;

  pdl_wait();
  int64_t len[kPlanPer], n[kPlanPer], need[kPlanPer];
  bool ok[kPlanPer];
  int64_t mine = 0;
#pragma unroll
  for (int k = 0; k < kPlanPer; ++k) {
    const int b = tid * kPlanPer + k;
    len[k] = b < B ? a.lens[b] : 0;
    n[k] = b < B ? a.joins[b] : 0;
    ok[k] = len[k] >= 0 && n[k] >= 0 && len[k] <= cap;
    n[k] = n[k] < 0 ? 0 : (n[k] > a.rows ? a.rows + 1 : n[k]);
    mine += n[k];
  }
  const int64_t used = *a.used;
  const int64_t left = used < 0 || used > a.n_free ? 0 : a.n_free - used;
  int64_t total;
  int64_t row = block_scan(mine, warp_sums, &total);
  if (tid == 0) s_cu[0] = 0;
  mine = 0;
#pragma unroll
  for (int k = 0; k < kPlanPer; ++k) {
    const int b = tid * kPlanPer + k;
    row += n[k];
    if (b < B) {
      s_len[b] = len[k];
      s_cu[b + 1] = static_cast<int32_t>(row < a.rows ? row : a.rows);
    }
    need[k] = 0;
    if (ok[k]) {
      const int64_t want = (len[k] + n[k] + ps - 1) >> shift;
      ok[k] = row <= a.rows && want <= a.width;
      if (ok[k]) need[k] = want - ((len[k] + ps - 1) >> shift);
    }
    mine += need[k];
  }
  int64_t at = block_scan(mine, warp_sums, &total);
  int64_t granted = 0;   // pages handed out to this thread's requests
#pragma unroll
  for (int k = 0; k < kPlanPer; ++k) {
    const int b = tid * kPlanPer + k;
    const bool g = ok[k] && (need[k] == 0 || at + need[k] <= left);
    if (b < B) s_page[b] = g ? static_cast<int32_t>(need[k] ? used + at : 0) : -1;
    granted += g ? need[k] : 0;
    at += need[k];
  }
  block_scan(granted, warp_sums, &total);   // also orders the shared arrays before their use
  cluster_sync_all();

  const int nthreads = gridDim.x * kPlanThreads, gt = blockIdx.x * kPlanThreads + tid;
  for (int b = gt; b < B; b += nthreads) {
    a.cu_rows[b + 1] = s_cu[b + 1];
    const int64_t l = s_len[b];
    const int64_t j = a.joins[b];
    a.lens_out[b] = s_page[b] >= 0 ? l + j : l;
  }
  if (gt == 0) {
    a.cu_rows[0] = 0;
    *a.used_out = used + total;
  }
  const int live = s_cu[B];
  // A new page's first position is always one of the request's new rows: that row
  // writes the table entry (and none of those that are read here).
  const int top = 1 << (31 - __clz(B));
  for (int64_t r = gt; r < a.rows; r += nthreads) {
    int64_t slot = -1, pos = -1;
    if (r < live) {
      int b = 0;   // the last request whose rows begin at r or before
      for (int s = top; s > 0; s >>= 1)
        if (b + s < B && s_cu[b + s] <= r) b += s;
      const int64_t l = s_len[b];
      const int32_t first = s_page[b];
      pos = l + r - s_cu[b];
      if (first >= 0) {
        const int64_t have = (l + ps - 1) >> shift, p = pos >> shift, in_page = pos & (ps - 1);
        int32_t* entry = a.table + static_cast<int64_t>(b) * a.width + p;
        const int32_t page = p < have ? *entry : a.free_pages[first + (p - have)];
        if (p >= have && in_page == 0) *entry = page;
        if (page >= 0) slot = (static_cast<int64_t>(page) << shift) + in_page;
      }
    }
    a.slots[r] = slot;
    a.positions[r] = pos;
  }
}

// ---------------------------------------------------------------------------
// append: rows of K and V -> 4-bit codes at their slots
// ---------------------------------------------------------------------------
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Extremes of n values, NaN if one is (three-input min and max: half the instructions).
template <int n>
__device__ __forceinline__ void extremes(const float (&x)[n], float& mn, float& mx) {
  mn = mx = x[0];
#pragma unroll
  for (int j = 1; j + 1 < n; j += 2) {
    asm("min.NaN.f32 %0, %0, %1, %2;" : "+f"(mn) : "f"(x[j]), "f"(x[j + 1]));
    asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(mx) : "f"(x[j]), "f"(x[j + 1]));
  }
  if constexpr (n % 2 == 0) {
    mn = min_nan(mn, x[n - 1]);
    mx = max_nan(mx, x[n - 1]);
  }
}

// The parameter word and the fp32 values of s and z for a row's extremes. A row
// with a non-finite value, or whose z or s leaves bf16's range, gets NaN for
// both (it reads back as NaN); a row whose maximum does not exceed z gets s = 0.
__device__ __forceinline__ uint32_t row_params(float mn, float mx, float& s, float& z) {
  const uint32_t zb = __bfloat16_as_ushort(__float2bfloat16_rn(mn));
  z = __uint_as_float(zb << 16);
  const float span = __fsub_rn(mx, z);
  const float st = span > 0.f ? __fdiv_rn(span, 15.0f) : 0.0f;
  const uint32_t sb = __bfloat16_as_ushort(__float2bfloat16_rn(st));
  s = __uint_as_float(sb << 16);
  if (!(isfinite(mn) && isfinite(mx) && isfinite(s) && isfinite(z))) {
    s = 0.f;
    return 0x7FC07FC0u;
  }
  return sb | (zb << 16);
}

// Codes of n <= 16 values, value j in bits 4 j ...: clamp(round((x - z) / s), 0, 15)
// of the real quotient, ties to even; zero when s is. t = (x - z) * (1 / s) in fp32
// (an approximate reciprocal) is within 4 * 2^-24 * 15.1 < 4e-6 of it, so only a t
// within 1e-5 of the middle of two codes is decided again, by comparing x - z with
// (m + 1/2) s in fp64, where nothing that matters is lost. s is the row's
// (max - z) / 15 within 2^-9, so no t reaches 15.5. Adding 1.5 * 2^23 rounds t to
// an integer in the low mantissa bits; the words are summed with their constant
// exponent bits, which one subtraction takes out. Pairs go through the packed
// fp32 operations: the rounds of 32 values, not HBM, bound a simpler form.
template <int n>
__device__ __forceinline__ uint2 codes_of(const float (&x)[n], float s, float z) {
  uint32_t w[2] = {0u, 0u};
  if (!(s > 0.f)) return make_uint2(0u, 0u);
  if (s < 1e-30f) {               // 1 / s could overflow
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      float xj = x[0];
#pragma unroll
      for (int k = 1; k < n; ++k) xj = j == k ? x[k] : xj;
      const double d = rint((static_cast<double>(xj) - static_cast<double>(z)) / static_cast<double>(s));
      const uint32_t c = d >= 15.0 ? 15u : (d > 0.0 ? static_cast<uint32_t>(d) : 0u);
      if (j < 8) w[0] |= c << (4 * j); else w[1] |= c << (4 * (j - 8));
    }
    return make_uint2(w[0], w[1]);
  }
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  constexpr float kMagic = 12582912.0f;   // 0x4B400000
  const f2_t z2 = f2_set(z, z), inv2 = f2_set(inv, inv), magic2 = f2_set(kMagic, kMagic);
  uint32_t bias[2] = {0u, 0u};
  float border = 0.f;                     // largest distance from an integer
#pragma unroll
  for (int j = 0; j < n; j += 2) {
    const float2 q = f2_unpack(f2_mul(f2_sub(f2_set(x[j], x[j + 1]), z2), inv2));
    const f2_t t2 = f2_set(fmaxf(q.x, 0.f), fmaxf(q.y, 0.f));
    const f2_t r2 = f2_add(t2, magic2);
    const float2 r = f2_unpack(r2), d = f2_unpack(f2_sub(t2, f2_sub(r2, magic2)));
    border = fmaxf(border, fmaxf(fabsf(d.x), fabsf(d.y)));
    w[j >> 3] += __float_as_uint(r.x) << (4 * (j & 7));
    w[j >> 3] += __float_as_uint(r.y) << (4 * ((j & 7) + 1));
    bias[j >> 3] += (0x4B400000u << (4 * (j & 7))) + (0x4B400000u << (4 * ((j & 7) + 1)));
  }
  w[0] -= bias[0];
  w[1] -= bias[1];
  if (border > 0.49999f) {
#pragma unroll
    for (int j = 0; j < n; ++j) {
      const float t = fmaxf(__fsub_rn(x[j], z) * inv, 0.f), m = floorf(t);
      if (fabsf(t - m - 0.5f) < 2e-5f) {
        const double d = static_cast<double>(x[j]) - static_cast<double>(z);
        const double half = (static_cast<double>(m) + 0.5) * static_cast<double>(s);
        const uint32_t lo = static_cast<uint32_t>(m);
        const uint32_t c = lo + (d > half || (d == half && (lo & 1u)) ? 1u : 0u);
        w[j >> 3] = (w[j >> 3] & ~(15u << (4 * (j & 7)))) | (c << (4 * (j & 7)));
      }
    }
  }
  return make_uint2(w[0], w[1]);
}

struct AppendArgs {
  const void* k;
  const void* v;
  int64_t k_rs, k_hs, v_rs, v_hs;   // element strides of rows and heads
  uint8_t* pool;
  const int64_t* slots;
  int64_t n, slots_max;             // slots_max = pages * page size
  int nkv, shift;
  int vec;                          // 16-byte loads are aligned
};

constexpr int kAppendThreads = 256;
constexpr int kAppendPerSm = 3;   // CTAs; 80 registers a thread

// Bound by HBM (the rows are read once, hd/2 + 4 bytes written). HD / 16 lanes
// take the K and the V row of one head, 16 values each, as 16-byte chunks dealt
// out in turn, so that each load instruction reads whole lines; three (two)
// shuffle rounds find a row's extremes. K and V together, and rows read before
// the slot is known to be valid, keep twice the loads in flight: 16391 rows of
// 8 x 128 fp32 take 31 us (4.6 TB/s), one row at a time 51.
template <class T, int HD>
__global__ void __launch_bounds__(kAppendThreads, kAppendPerSm) append_kernel(const AppendArgs a) {
  constexpr int LPR = HD / 16;
  constexpr int E = 16 / sizeof(T), C = 16 / E;   // elements of a chunk, chunks of a lane
  const int lane = threadIdx.x & (LPR - 1);
  const int64_t total = a.n * a.nkv;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kAppendThreads / LPR);
  const int64_t ps = int64_t(1) << a.shift;
  pdl_wait();
  // warp-uniform loop: all lanes run the same number of rounds for the shuffles
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kAppendThreads / LPR);
  for (int64_t base = first; base < total; base += step) {
    const int64_t id = base + threadIdx.x / LPR;
    const int64_t row = id >> 31 ? id / a.nkv
                                 : static_cast<int64_t>(static_cast<unsigned>(id) / static_cast<unsigned>(a.nkv));
    const int h = static_cast<int>(id - row * a.nkv);
    const bool in = id < total;
    const int64_t slot = in ? __ldg(a.slots + row) : -1;
    float x[2][16];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const T* p = static_cast<const T*>(kv ? a.v : a.k) + row * (kv ? a.v_rs : a.k_rs) +
                   h * (kv ? a.v_hs : a.k_hs) + lane * E;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float e[E];
#pragma unroll
        for (int j = 0; j < E; ++j) e[j] = 0.f;
        if (in) load_row(p + c * (LPR * E), a.vec, e);
#pragma unroll
        for (int j = 0; j < E; ++j) x[kv][c * E + j] = e[j];
      }
    }
    float mn[2], mx[2];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      extremes(x[kv], mn[kv], mx[kv]);
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) {
        mn[kv] = min_nan(mn[kv], __shfl_xor_sync(0xffffffffu, mn[kv], o));
        mx[kv] = max_nan(mx[kv], __shfl_xor_sync(0xffffffffu, mx[kv], o));
      }
    }
    if (slot < 0 || slot >= a.slots_max) continue;
    const int64_t off = slot & (ps - 1);
    uint8_t* blk = a.pool + ((slot >> a.shift) * a.nkv + h) * (ps * (HD + 8));
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      float s, z;
      const uint32_t par = row_params(mn[kv], mx[kv], s, z);
      const uint2 w = codes_of(x[kv], s, z);
      uint8_t* at = blk + (kv ? ps * (HD / 2) : 0) + off * (HD / 2) + lane * (E / 2);
      if constexpr (E == 4) {
        *reinterpret_cast<uint16_t*>(at) = static_cast<uint16_t>(w.x);
        *reinterpret_cast<uint16_t*>(at + 2 * LPR) = static_cast<uint16_t>(w.x >> 16);
        *reinterpret_cast<uint16_t*>(at + 4 * LPR) = static_cast<uint16_t>(w.y);
        *reinterpret_cast<uint16_t*>(at + 6 * LPR) = static_cast<uint16_t>(w.y >> 16);
      } else {
        *reinterpret_cast<uint32_t*>(at) = w.x;
        *reinterpret_cast<uint32_t*>(at + 4 * LPR) = w.y;
      }
      if (lane == 0) *reinterpret_cast<uint32_t*>(blk + ps * HD + (kv ? ps * 4 : 0) + off * 4) = par;
    }
  }
}

struct GatherArgs {
  const uint8_t* pool;
  const int64_t* slots;
  float* k;
  float* v;
  int64_t n, slots_max;
  int nkv, shift;
};

constexpr int kGatherThreads = 256;

// The values of rows: z + c * s (one rounding), fp32 [n, nkv, hd]; zeros for a
// slot outside the pool. Bound by the fp32 stores: HD / 4 lanes take the K and the
// V row of one head, read 2 bytes of codes each and store float4s; kGatherFly
// rows are in flight per lane, for the load of a slot and the loads behind it.
constexpr int kGatherFly = 2;
template <int HD>
__global__ void __launch_bounds__(kGatherThreads) gather_kernel(const GatherArgs a) {
  constexpr int LPR = HD / 4;
  const int lane = threadIdx.x & (LPR - 1);
  const int64_t total = a.n * a.nkv;
  const int64_t rows_per_block = kGatherThreads / LPR;
  const int64_t ps = int64_t(1) << a.shift;
  pdl_wait();
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * (rows_per_block * kGatherFly) + threadIdx.x / LPR;
       base < total; base += static_cast<int64_t>(gridDim.x) * (rows_per_block * kGatherFly)) {
    uint32_t c[kGatherFly][2], par[kGatherFly][2];
    int64_t id[kGatherFly];
#pragma unroll
    for (int f = 0; f < kGatherFly; ++f) {
      id[f] = base + f * rows_per_block;
      c[f][0] = c[f][1] = par[f][0] = par[f][1] = 0u;        // s = z = 0: zeros
      if (id[f] >= total) continue;
      const int64_t row = id[f] >> 31
          ? id[f] / a.nkv : static_cast<int64_t>(static_cast<unsigned>(id[f]) / static_cast<unsigned>(a.nkv));
      const int h = static_cast<int>(id[f] - row * a.nkv);
      const int64_t slot = __ldg(a.slots + row);
      if (slot < 0 || slot >= a.slots_max) continue;
      const int64_t off = slot & (ps - 1);
      const uint8_t* blk = a.pool + ((slot >> a.shift) * a.nkv + h) * (ps * (HD + 8));
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        c[f][kv] = *reinterpret_cast<const uint16_t*>(blk + kv * (ps * (HD / 2)) + off * (HD / 2) + lane * 2);
        par[f][kv] = *reinterpret_cast<const uint32_t*>(blk + ps * HD + kv * (ps * 4) + off * 4);
      }
    }
#pragma unroll
    for (int f = 0; f < kGatherFly; ++f) {
      if (id[f] >= total) continue;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const float s = par_s(par[f][kv]), z = par_z(par[f][kv]);
        const uint32_t w = c[f][kv];
        const float4 o = make_float4(fmaf(static_cast<float>(w & 15u), s, z),
                                     fmaf(static_cast<float>((w >> 4) & 15u), s, z),
                                     fmaf(static_cast<float>((w >> 8) & 15u), s, z),
                                     fmaf(static_cast<float>(w >> 12), s, z));
        __stcs(reinterpret_cast<float4*>((kv ? a.v : a.k) + id[f] * HD) + lane, o);
      }
    }
  }
}

// q/k norm, RoPE and append of projection rows in one pass
struct RopeArgs {
  const float* qkv;        // [M, (nq + 2 nkv) hd]
  const float* qn_w;       // [hd] or null
  const float* kn_w;
  const float* inv_freq;   // [hd / 2]
  float* q_out;            // [M, nq hd]
  uint8_t* pool;
  const int64_t* positions;
  const int64_t* slots;
  int64_t m, slots_max;
  int nq, nkv, shift;
  float eps;
};

constexpr int kRopeThreads = 128;

// A warp per (row, head), HD / 32 dimensions a lane: q heads are normed, rotated
// and written, k heads normed, rotated and quantised, v heads quantised, each
// straight from the projection (the roped k never goes to memory). The pair of
// dimension j under the half-split rotation, j +- HD / 2, lies 16 lanes away.
// Latency-bound at decode sizes (16 rows of 48 heads: 0.4 MB).
template <int HD>
__global__ void __launch_bounds__(kRopeThreads) qk_rope_kv4_kernel(const RopeArgs a) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  const int heads = a.nq + 2 * a.nkv;
  pdl_wait();
  const int64_t id = static_cast<int64_t>(blockIdx.x) * (kRopeThreads / 32) + (threadIdx.x >> 5);
  if (id >= a.m * heads) return;
  const int64_t row = id / heads;
  const int head = static_cast<int>(id - row * heads);
  const bool is_q = head < a.nq, is_v = head >= a.nq + a.nkv;
  const float* src = a.qkv + (row * heads + head) * HD + lane * E;
  float x[E];
#pragma unroll
  for (int j = 0; j < E; ++j) x[j] = src[j];
  if (!is_v) {
    const float* w = is_q ? a.qn_w : a.kn_w;
    if (w) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < E; ++j) ss = fmaf(x[j], x[j], ss);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = 1.0f / sqrtf(ss / static_cast<float>(HD) + a.eps);
#pragma unroll
      for (int j = 0; j < E; ++j) x[j] = x[j] * r * w[lane * E + j];
    }
    const int64_t pos = a.positions[row];
    const float fpos = static_cast<float>(pos < 0 ? 0 : pos);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const float ang = fpos * a.inv_freq[(lane * E + j) & (HD / 2 - 1)];
      const float c = cosf(ang), s = sinf(ang);
      const float y = __shfl_xor_sync(0xffffffffu, x[j], 16);
      x[j] = lane < 16 ? x[j] * c - y * s : x[j] * c + y * s;
    }
  }
  if (is_q) {
    float* dst = a.q_out + (row * a.nq + head) * HD + lane * E;
#pragma unroll
    for (int j = 0; j < E; ++j) dst[j] = x[j];
    return;
  }
  const int64_t slot = a.slots[row];
  if (slot < 0 || slot >= a.slots_max) return;
  float mn, mx;
  extremes(x, mn, mx);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mn = min_nan(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  float s, z;
  const uint32_t par = row_params(mn, mx, s, z);
  const uint32_t c = codes_of(x, s, z).x;
  const int h = head - a.nq - (is_v ? a.nkv : 0);
  const int64_t ps = int64_t(1) << a.shift, off = slot & (ps - 1);
  uint8_t* blk = a.pool + ((slot >> a.shift) * a.nkv + h) * (ps * (HD + 8));
  uint8_t* at = blk + (is_v ? ps * (HD / 2) : 0) + off * (HD / 2) + lane * (E / 2);
  if constexpr (E == 4)
    *reinterpret_cast<uint16_t*>(at) = static_cast<uint16_t>(c);
  else
    *at = static_cast<uint8_t>(c);
  if (lane == 0) *reinterpret_cast<uint32_t*>(blk + ps * HD + (is_v ? ps * 4 : 0) + off * 4) = par;
}

// ---------------------------------------------------------------------------
// attention, rows against a long context
// ---------------------------------------------------------------------------
// o = sum_t softmax(scale * q . k_t) v_t with k_t = zk_t + sk_t c_t and
// v_t = zv_t + sv_t d_t, so with the integer codes as one MMA operand
//   q . k_t = sk_t (q . c_t) + zk_t sum(q)
//   o       = sum_t (p_t sv_t) (d_t - 8) + sum_t p_t (zv_t + 8 sv_t)
// The codes are exact in fp16, so only q and the weights p sv are rounded:
// each is split into two fp16 values (22 bits), which stand as two columns of
// the other operand. A warp handles 16 positions at a time with m16n8k16 MMAs:
//   S [16 positions x 8 columns]  = K codes x q    (4 queries x {hi, lo})
//   O [hd x 8 columns]           += (V codes - 8)^T x w
// These MMAs see 8 columns per kv head and position block; the pages stream at
// HBM speed and the tensor pipe is not the bound, so mma.sync serves here (a
// tcgen05 tile of 128 rows would be 94 % padding).
//
// Each warp streams its own 32 positions at a time: bulk copies bring the packed
// blocks of one stage into shared memory, kAttnDepth - 1 stages ahead of the
// math, so no registers hold data in flight. (cp.async by all lanes: 4 to 6 %
// slower for pages of 16 and 32, for its instructions; 5 % faster for larger
// pages, which take four copies a stage here.) A lane's share of a K row is 16
// (hd 64: 8) consecutive bytes. The order of dimensions inside an MMA's K
// axis is free as long as q has the same one, so nibbles 0 and 4 of a word
// (w & 0x000F000F) form one fp16 pair: the bits c are the subnormal c * 2^-24,
// exact. Nibbles 1 and 5 lie four bits higher, as 16 c * 2^-24; q's values for
// them are divided by 16. For V, pairs run along positions: one PRMT joins the
// halves of two positions' words; 0x6400 | d is 1024 + d, and one HADD2 (HFMA2
// for the nibbles four bits higher) leaves d - 8. Centring V keeps the sums as
// small as their result. An MMA's accumulation truncates (about 3e-8 of the
// accumulator each time), so for fp32 rows one or two MMAs start from zero, the sums
// are added up in fp32, and K is centred like V: with subnormal K codes and
// accumulation in place, results were 1.3e-6 to 2.4e-6 off 64 bits. 16-bit rows take
// both cheaper forms for up to kAttnFlush stages, 128 MMAs that leave 2e-6; then a
// warp's sums go to fp32 sums of its own in the workspace (fp32 sums in registers
// spill at four CTAs per SM). Row r of the
// eight positions an MMA fragment pairs up is position r / 2 + 4 (r & 1), so
// that the V rows a quarter-warp reads are neighbours (fewer bank conflicts).
//
// Work is cut into steps of 128 positions over all (request, kv head, block of
// queries), shared out evenly over a fixed grid whatever the lengths, which
// only the device knows (graph replay). A CTA's share may begin or end within an item; those partials
// (max, sum, accumulator) go to the workspace and the last of an item's CTAs
// to arrive merges them in CTA order, so results do not depend on timing.
//
// The running maximum is only renewed when a score passes it by 2^3 (weights
// stay below 2^3 relative to it): one vote per stage instead of a reduction. The
// same vote sees to the power of two that brings a query's weights p sv into fp16's
// range (see kAttnSpare).
//
// Measured: 64 x 16384 positions, 8 kv heads of 128, bf16 139 us (56 % of the copy
// rate; 730 instructions per 32 positions and head, issue slots 57 %, no pipe full);
// 16 x 2048 fp32 17.4 us; one request of 131071 positions, 8 kv heads of 64, fp32 45 us
// (635 instructions, issue 65 %). Graphs of 10 calls.

constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = kAttnWarps * 32;
constexpr int kAttnStage = 32;    // positions per warp and stage
constexpr int kAttnDepth = 3;     // stages of a warp
constexpr int kAttnStep = kAttnWarps * kAttnStage;
constexpr int kAttnMaxB = 4096;
// Steps of positions (so stages of a warp) between the places where a warp's sums of
// 16-bit rows leave the MMA's accumulator: after steps 63, 127, ... of an item (a power
// of two).
constexpr int kAttnFlush = 64;
// Weights p sv enter the MMAs as fp16 pairs times up = 2^(11 - ev), so whatever lies
// below 2^-25 of that scale is lost. ev is the exponent of the largest step sv seen, but
// at most kAttnSpare above that of the largest p sv: a row of V with a large step and a
// vanishing weight costs the others nothing (they keep 2^-26 of the largest weight), and
// steps that differ by less than 2^10 need no attention from stage to stage.
constexpr int kAttnSpare = 10;
// What an item costs beside its positions (its query fragments, the merge), in
// steps: the shares of short and long contexts take about as long.
constexpr int kAttnItemUnits = 1;

struct AttnArgs {
  const void* q;
  void* out;
  int64_t q_rs, q_hs, o_rs, o_hs;   // element strides of rows and heads
  const uint8_t* pool;
  const int32_t* table;
  const int64_t* lens;
  const int64_t* cu;                // [B + 1] or null: request b has row b
  float* part;
  float* sums;                      // [CTAs][warps][attn_sum_floats][32]; not used for fp32 rows
  unsigned int* tickets;
  int64_t pages, width, n;
  int B, nkv, group, shift;
  float scale;                      // softmax scale * log2(e)
  int vec;                          // q rows are 16-byte aligned
  int rows_lo, rows_hi;             // requests with rows_lo < rows <= rows_hi are handled
};

// CTAs per SM that the register file and shared memory hold (fp32 rows at hd 128: the
// fp32 sums want more than the 128 registers of four).
constexpr int kAttnMaxPerSm = 5;
__host__ __device__ constexpr int attn_per_sm(int hd, int nb, bool wide) {
  return nb == 1 ? (hd == 64 ? 5 : (wide ? 3 : 4)) : (hd == 64 ? 4 : 2);
}
template <int HD, int NB>
__host__ __device__ constexpr int attn_queries() { return 4 * NB; }
template <int HD, int NB>
__host__ __device__ constexpr int attn_part_floats() { return 4 * NB * (HD + 2); }
// A lane's share of a warp's sums, and the maximum of each query that they stand relative to.
__host__ __device__ constexpr int attn_sum_floats(int hd, int nb) { return nb * (hd / 8 + 1); }
template <int HD>
__host__ __device__ constexpr int attn_stage_bytes() { return kAttnStage * (HD + 8); }
constexpr int kAttnHead = kAttnThreads * 8 + 64 + kAttnWarps * kAttnDepth * 8;
// The warps' rings; their results take the same place afterwards.
template <int HD, int NB>
__host__ __device__ constexpr int attn_smem() {
  constexpr int ring = kAttnWarps * kAttnDepth * attn_stage_bytes<HD>();
  constexpr int merge = kAttnWarps * attn_part_floats<HD, NB>() * 4;
  return 2048 + (ring > merge ? ring : merge);
}
static_assert(kAttnHead <= 2048, "the rings start 2 KB in");

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same from a zero accumulator.
__device__ __forceinline__ void mma_f16_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                            uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ uint32_t trans8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^e for e in [-126, 127], floor(log2 x) for a normal x >= 0 (-127 for what is smaller).
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }
__device__ __forceinline__ int exponent(float x) { return static_cast<int>((__float_as_uint(x) >> 23) & 255u) - 127; }

// The four position pairs of one 16-bit half of two rows' words, less 8:
// h[n] = (d(row a, nibble n) - 8, d(row b, nibble n) - 8) as fp16.
__device__ __forceinline__ void centred4(uint32_t x, uint32_t (&h)[4]) {
  const uint32_t y = x >> 8;
  const __half2 m8 = __half2half2(__ushort_as_half(0xE408));    // -1032
  const __half2 m72 = __half2half2(__ushort_as_half(0xD480));   // -72
  const __half2 r16 = __half2half2(__ushort_as_half(0x2C00));   // 1 / 16
  auto put = [](uint32_t w) { return *reinterpret_cast<const __half2*>(&w); };
  auto get = [](__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); };
  h[0] = get(__hadd2(put((x & 0x000F000Fu) | 0x64006400u), m8));
  h[1] = get(__hfma2(put((x & 0x00F000F0u) | 0x64006400u), r16, m72));
  h[2] = get(__hadd2(put((y & 0x000F000Fu) | 0x64006400u), m8));
  h[3] = get(__hfma2(put((y & 0x00F000F0u) | 0x64006400u), r16, m72));
}

template <int W>
__device__ __forceinline__ void lds(uint32_t addr, uint32_t (&v)[W]) {
  if constexpr (W == 4)
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr));
  else if constexpr (W == 2)
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(addr));
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(addr));
}

// 1-D bulk copy global -> this CTA's shared memory (no cluster multicast).
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void fence_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ int64_t rows_of(const AttnArgs& a, int64_t b, int64_t* first) {
  int64_t r0 = b, r1 = b + 1;
  if (a.cu) {
    r0 = a.cu[b];
    r1 = a.cu[b + 1];
  }
  r0 = r0 < 0 ? 0 : r0;
  r1 = r1 > a.n ? a.n : r1;
  *first = r0;
  const int64_t n = r1 > r0 ? r1 - r0 : 0;
  return n > a.rows_lo && n <= a.rows_hi ? n : 0;
}

template <int NB>
__device__ __forceinline__ int64_t steps_of(const AttnArgs& a, int64_t len) {
  const int64_t cap = a.width << a.shift;
  const int64_t t = len < 0 ? 0 : (len > cap ? cap : len);
  const int64_t s = (t + kAttnStep - 1) / kAttnStep;
  return s > 0 ? s : 1;   // an empty context still has its (zero) rows to write
}

// floor(x / y) for 0 <= x < 2^52 with inv = 1 / y: the product is off by less
// than one, which the remainder shows.
__device__ __forceinline__ int64_t div_floor(int64_t x, int64_t y, double inv) {
  int64_t q = static_cast<int64_t>(static_cast<double>(x) * inv);
  const int64_t r = x - q * y;
  q += r >= y ? 1 : (r < 0 ? -1 : 0);
  return q;
}

template <class T, int HD, int NB>
__global__ void __launch_bounds__(kAttnThreads, attn_per_sm(HD, NB, sizeof(T) == 4)) attn_kernel(const AttnArgs a) {
  constexpr int Q = attn_queries<HD, NB>();   // queries (row, head) of an item
  constexpr int KS = HD / 16;                 // MMAs along the head dimension, and O tiles
  constexpr int KW = HD / 32;                 // K words of a lane and row
  constexpr int VW = HD / 64;                 // V words of a lane and position
  constexpr bool kWide = sizeof(T) == 4;      // the more exact forms
  constexpr bool kPairs = kWide && !(HD == 128 && NB == 2);   // (there pairs of MMAs would spill)
  constexpr float kNegInf = -INFINITY;
  constexpr int SB = attn_stage_bytes<HD>();
  extern __shared__ __align__(128) uint8_t attn_sh[];
  int64_t* s_scan = reinterpret_cast<int64_t*>(attn_sh);                        // [threads]
  int64_t* s_at = reinterpret_cast<int64_t*>(attn_sh + kAttnThreads * 8);       // {b, its first unit}
  int* s_last = reinterpret_cast<int*>(s_at + 2);
  float* s_wm = reinterpret_cast<float*>(attn_sh);                              // [threads][2], after s_scan
  float* s_o = reinterpret_cast<float*>(attn_sh + 2048);                        // [warps][Q][HD]
  float* s_ml = s_o + kAttnWarps * Q * HD;                                      // [warps][Q][2]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, i = lane & 3;
  const uint32_t bars = smem_u32(attn_sh + kAttnThreads * 8 + 64) + warp * (kAttnDepth * 8);
  const uint32_t ring = smem_u32(attn_sh + 2048) + warp * (kAttnDepth * SB);
  if (lane == 0) {
    for (int k = 0; k < kAttnDepth; ++k) mbar_init(bars + 8 * k, 1);
    fence_mbar_init();
  }
  // A stage is one block of 32 positions, or (pages of 16) two of 16. Copies: a
  // whole block each, or the four parts of 32 positions of a larger page.
  const bool small = a.shift == 4, parts = a.shift > 5;
  const int copies = parts ? 4 : (small ? 2 : 1);
  const uint32_t bytes = parts ? (lane < 2 ? kAttnStage * (HD / 2) : kAttnStage * 4)
                               : (small ? SB / 2 : SB);
  const uint32_t to = parts ? (lane < 2 ? lane * (kAttnStage * (HD / 2))
                                        : kAttnStage * HD + (lane - 2) * (kAttnStage * 4))
                            : lane * (SB / 2);
  const int64_t ps = int64_t(1) << a.shift, page_bytes = a.nkv * (ps * (HD + 8));
  // this lane's offsets within a stage: K row and parameters of its first score
  // row, V row of its first position; from 16 positions to the next
  const int blk = small ? 16 : 32, tau = (g >> 1) + 4 * (g & 1);
  const uint32_t k_at = tau * (HD / 2) + i * (HD / 8);
  const uint32_t v_at = blk * (HD / 2) + i * (HD / 2) + g * (HD / 16);
  const uint32_t p_at = blk * HD + tau * 4;
  const uint32_t k_next = small ? SB / 2 : 16 * (HD / 2), p_next = small ? SB / 2 : 64;
  int st = 0;            // the ring position of the next stage to be used
  uint32_t phase = 0;    // its parity

  pdl_wait();
  // ---- this CTA's share [u0, u1) of all units --------------------------------
  // An item (request, kv head, block of queries) is kAttnItemUnits units for its
  // fixed costs and one for each step of its positions.
  const int per_thread = (a.B + kAttnThreads - 1) / kAttnThreads;
  auto units = [&](int64_t b) -> int64_t {
    int64_t r0;
    const int64_t n = rows_of(a, b, &r0);
    if (n == 0) return 0;
    return a.nkv * static_cast<int64_t>((static_cast<unsigned>(n * a.group) + Q - 1) / Q) *
           (steps_of<NB>(a, a.lens[b]) + kAttnItemUnits);
  };
  int64_t mine = 0;
  for (int k = 0; k < per_thread; ++k) {
    const int64_t b = static_cast<int64_t>(tid) * per_thread + k;
    if (b < a.B) mine += units(b);
  }
  s_scan[tid] = mine;
  __syncthreads();
  int64_t before = 0, U = 0;
  for (int k = 0; k * per_thread < a.B; ++k) {
    const int64_t v = s_scan[k];
    before += k < tid ? v : 0;
    U += v;
  }
  if (U == 0) return;
  const int64_t C = U < gridDim.x ? U : gridDim.x;
  const int64_t c = blockIdx.x;
  if (c >= C) return;
  const double inv_c = 1.0 / static_cast<double>(C), inv_u = 1.0 / static_cast<double>(U);
  // CTA k's share begins at k U / C; unit x belongs to CTA ((x + 1) C - 1) / U
  auto begin_of = [&](int64_t k) -> int64_t { return div_floor(k * U, C, inv_c); };
  auto cta_of = [&](int64_t x) -> int64_t { return div_floor((x + 1) * C - 1, U, inv_u); };
  const int64_t u0 = begin_of(c), u1 = begin_of(c + 1);
  if (u0 >= before && u0 < before + mine) {
    int64_t b = static_cast<int64_t>(tid) * per_thread, at = before;
    for (int64_t n = units(b); u0 >= at + n; n = units(b)) {
      at += n;
      ++b;
    }
    s_at[0] = b;
    s_at[1] = at;
  }
  __syncthreads();
  int64_t b = s_at[0], ub = s_at[1];
  const int cap = static_cast<int>(a.width << a.shift);

  for (int64_t u = u0; u < u1;) {
    int64_t r0;
    const int n = static_cast<int>(rows_of(a, b, &r0));
    const int64_t len = n ? a.lens[b] : 0;
    const int64_t size = steps_of<NB>(a, len) + kAttnItemUnits;   // units of an item
    const int nqueries = n * a.group;
    const int nqb = (nqueries + Q - 1) / Q;
    const int64_t all = a.nkv * nqb * size;
    if (u >= ub + all) {
      ub += all;
      ++b;
      continue;
    }
    const int64_t in_b = u - ub;
    const int64_t item = in_b >> 31 ? in_b / size
                                    : static_cast<int64_t>(static_cast<unsigned>(in_b) / static_cast<unsigned>(size));
    const int64_t i0 = ub + item * size, i1 = i0 + size < u1 ? i0 + size : u1;
    // steps [s0, s1) of the item
    const int s0 = u - i0 < kAttnItemUnits ? 0 : static_cast<int>(u - i0) - kAttnItemUnits;
    const int s1 = static_cast<int>(i1 - i0) - kAttnItemUnits;
    u = i1;
    if (s1 <= s0) continue;                  // (the item's steps are the next CTA's)
    const int h = static_cast<int>(static_cast<unsigned>(item) / static_cast<unsigned>(nqb));
    const int q0 = (static_cast<int>(item) - h * nqb) * Q;   // first query of the item

    // positions [0, lim) that a query sees; rows and positions are at most 2^30
    const int64_t far = int64_t(1) << 30, off64 = len - n;
    const int off = static_cast<int>(off64 > far ? far : (off64 < -far ? -far : off64));
    auto limit = [&](int qi) -> int {
      const int l = off + static_cast<int>(static_cast<unsigned>(qi) / static_cast<unsigned>(a.group)) + 1;
      return l < 0 ? 0 : (l > cap ? cap : l);
    };
    int lim[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int qi = q0 + nb * 4 + i;
      lim[nb] = limit(qi < nqueries ? qi : nqueries - 1);   // (more queries than there are: q = 0)
    }
    const int all_see = limit(q0);                 // the first query sees least ...
    const int seen = limit(q0 + Q < nqueries ? q0 + Q - 1 : nqueries - 1);   // ... and the last most

    // ---- q: two fp16 columns per query, scaled by a power of two --------------
    uint32_t qf[NB][KS][2];
    float F[NB], Qs[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int qi = q0 + nb * 4 + (g >> 1);
      float x[HD / 4];
      if (qi < nqueries) {
        const int r = static_cast<int>(static_cast<unsigned>(qi) / static_cast<unsigned>(a.group));
        const T* p = static_cast<const T*>(a.q) + (r0 + r) * a.q_rs +
                     (h * a.group + (qi - r * a.group)) * a.q_hs + i * (HD / 4);
        load_row(p, a.vec, x);
      } else {
#pragma unroll
        for (int j = 0; j < HD / 4; ++j) x[j] = 0.f;
      }
      float mx = 0.f, sum = 0.f;
#pragma unroll
      for (int j = 0; j < HD / 4; ++j) {
        mx = fmaxf(mx, fabsf(x[j]));
        sum += x[j];
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
      }
      // |x| * 2^(14 - e) < 2^15 for the row's largest; e bounded so that both
      // powers of two are normal
      int e = static_cast<int>((__float_as_uint(mx) >> 23) & 255u) - 127;
      e = e < -112 ? -112 : (e > 117 ? 117 : e);
      const float up = pow2i(14 - e);
      const float f = pow2i(e + (kWide ? -14 : 10)) * a.scale, qs = sum * a.scale;
      F[nb] = __shfl_sync(0xffffffffu, f, 8 * i);
      Qs[nb] = __shfl_sync(0xffffffffu, qs, 8 * i);
      // pairs (0 4) (1 5) (2 6) (3 7) of each eight; subnormal odd nibbles are 16 c
#pragma unroll
      for (int m = 0; m < KW; ++m)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float s = !kWide && (k & 1) ? up * 0.0625f : up;
          const float y0 = x[8 * m + k] * s, y1 = x[8 * m + k + 4] * s;
          const __half2 hi = __floats2half2_rn(y0, y1);
          const float2 back = __half22float2(hi);
          const __half2 lo = __floats2half2_rn(y0 - back.x, y1 - back.y);
          const __half2 v = g & 1 ? lo : hi;
          qf[nb][2 * m + (k >> 1)][k & 1] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }

    // m: maximum; rel: what scores are taken relative to (0 until there is a maximum)
    float acc[NB][KS][4], m[NB], rel[NB], l[NB], zs[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      m[nb] = kNegInf;
      rel[nb] = l[nb] = zs[nb] = 0.f;
#pragma unroll
      for (int t = 0; t < KS; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[nb][t][j] = 0.f;
    }
    // a query's weights are p sv up; wm: their largest when up was last settled, without up
    float up[NB];
    volatile float* wm = s_wm + tid * 2;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      up[nb] = pow2i(111);               // ev = -100
      wm[nb] = 0.f;
    }

    // ---- stages of this warp ---------------------------------------------------
    auto own_sums = [&](int k) -> float* {   // (formed where it is used: registers)
      return a.sums + static_cast<size_t>(blockIdx.x * kAttnWarps + warp) * (attn_sum_floats(HD, NB) * 32) +
             k * 32 + lane;
    };
    const int32_t* tab = a.table + b * a.width;
    const int t_end = s1 * kAttnStep < seen ? s1 * kAttnStep : seen;
    int pos = s0 * kAttnStep + warp * kAttnStage;
    int ahead = pos;                       // first position of the next stage to be copied
    auto page_at = [&](int p) -> int {
      p += small ? lane * 16 : 0;
      return lane < copies && p < t_end ? __ldg(tab + (p >> a.shift)) : -1;
    };
    int page = page_at(ahead);
    const uint8_t* head = a.pool + static_cast<int64_t>(h) * (ps * (HD + 8));
    if (parts) head += lane < 2 ? lane * (ps * (HD / 2)) : ps * HD + (lane - 2) * (ps * 4);
    const uint32_t per_pos = parts ? (lane < 2 ? HD / 2 : 4) : 0;
    // bit (stage's 16-position half) of ring position k: that half was copied
    uint32_t there = 0;
    auto issue = [&](int k) {
      const bool have = page >= 0 && page < a.pages;
      const uint32_t vote = __ballot_sync(0xffffffffu, have);
      const uint32_t halves = small ? vote & 3u : (vote & 1u) * 3u;
      there = (there & ~(3u << (2 * k))) | (halves << (2 * k));
      const uint32_t bar = bars + 8 * k;
      if (lane == 0) mbar_arrive_expect_tx(bar, small ? __popc(vote) * (SB / 2) : (vote ? SB : 0));
      __syncwarp();
      if (have) {
        const uint8_t* from = head + page * page_bytes + (ahead & (static_cast<int>(ps) - 1)) * per_pos;
        bulk_copy(ring + k * SB + to, from, bytes, bar);
      }
      ahead += kAttnStep;
      page = page_at(ahead);
    };
    {
      int k = st;
      for (int j = 0; j < kAttnDepth - 1 && ahead < t_end; ++j) {
        issue(k);
        k = k + 1 == kAttnDepth ? 0 : k + 1;
      }
    }
    // 16-bit rows: where the chain of MMAs ends; whether one did
    int stop = kWide ? t_end : min(t_end, (s0 / kAttnFlush + 1) * (kAttnFlush * kAttnStep));
    bool flushed = false;
#pragma unroll 1
    while (true) {
#pragma unroll 1
      for (; pos < stop; pos += kAttnStep) {
        if (ahead < t_end) issue(st == 0 ? kAttnDepth - 1 : st - 1);   // the stage used last
        const bool landed = __all_sync(0xffffffffu, mbar_wait(bars + 8 * st, phase));
        if (!landed) {   // reported; the copy gets as long again before its place is used
          if (lane == 0) report_error(ERR_WAIT_FULL, 0x430u);
          mbar_wait(bars + 8 * st, phase);
        }
        const uint32_t base = ring + st * SB, half_ok = landed ? (there >> (2 * st)) & 3u : 0u;
        const bool whole = half_ok == 3u && pos + kAttnStage <= all_see;
        // scores of rows g, g + 8 of both halves, and their V parameters
        float x[2][2][NB];
        uint32_t vp[2][2][NB];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          uint32_t k0[KW], k1[KW], kp[2], one[1];
          lds(base + k_at + t * k_next, k0);
          lds(base + k_at + t * k_next + 8 * (HD / 2), k1);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            lds(base + p_at + t * p_next + 32 * r, one);
            kp[r] = one[0];
            lds(base + p_at + t * p_next + 32 * r + blk * 4, one);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) vp[t][r][nb] = one[0];
          }
          float sc[NB][4];
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[nb][j] = 0.f;
#pragma unroll
          for (int w = 0; w < KW; ++w) {
            if constexpr (kWide) {
              // two MMAs from zero for each word, summed in fp32
              uint32_t c0[4], c1[4];
              centred4(k0[w], c0);
              centred4(k1[w], c1);
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) {
                float d[4];
                mma_f16_new(d, c0[0], c1[0], c0[1], c1[1], qf[nb][2 * w][0], qf[nb][2 * w][1]);
                mma_f16(d, c0[2], c1[2], c0[3], c1[3], qf[nb][2 * w + 1][0], qf[nb][2 * w + 1][1]);
#pragma unroll
                for (int j = 0; j < 4; ++j) sc[nb][j] += d[j];
              }
            } else {
              const uint32_t c0 = k0[w], c1 = k1[w], d0 = c0 >> 8, d1 = c1 >> 8;
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) {
                mma_f16(sc[nb], c0 & 0x000F000Fu, c1 & 0x000F000Fu, c0 & 0x00F000F0u, c1 & 0x00F000F0u,
                        qf[nb][2 * w][0], qf[nb][2 * w][1]);
                mma_f16(sc[nb], d0 & 0x000F000Fu, d1 & 0x000F000Fu, d0 & 0x00F000F0u, d1 & 0x00F000F0u,
                        qf[nb][2 * w + 1][0], qf[nb][2 * w + 1][1]);
              }
            }
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float sk = par_s(kp[r]), zk = kWide ? fmaf(8.f, sk, par_z(kp[r])) : par_z(kp[r]);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
              x[t][r][nb] = fmaf((sc[nb][2 * r] + sc[nb][2 * r + 1]) * F[nb], sk, zk * Qs[nb]);
          }
        }
        if (!whole) {
          // hidden positions, which may hold anything: no score, no V
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int p = (half_ok >> t) & 1u ? pos + 16 * t + 8 * r + tau : 0x7FFFFFFF;
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
                if (p >= lim[nb]) {
                  x[t][r][nb] = kNegInf;
                  vp[t][r][nb] = 0u;
                }
            }
        }
        float top[NB], sm[NB];
        bool renew = false;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          top[nb] = fmaxf(fmaxf(x[0][0][nb], x[0][1][nb]), fmaxf(x[1][0][nb], x[1][1][nb]));
          sm[nb] = fmaxf(fmaxf(fmaxf(0.f, par_s(vp[0][0][nb])), par_s(vp[0][1][nb])),
                         fmaxf(par_s(vp[1][0][nb]), par_s(vp[1][1][nb])));
          // p < 2^3 and sv up < 2^12
          renew = renew || top[nb] > m[nb] + 3.f || sm[nb] * up[nb] >= 4096.f;
        }
        if (__any_sync(0xffffffffu, renew)) {
          // new maximum and new scale of every query
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            float t = top[nb];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
            const float mn = fmaxf(m[nb], t);
            const float al = m[nb] == kNegInf ? 1.f : ex2(m[nb] - mn);
            m[nb] = mn;
            rel[nb] = mn == kNegInf ? 0.f : mn;
            float w = wm[nb] * al, sv = sm[nb];
#pragma unroll
            for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
              for (int r = 0; r < 2; ++r) w = fmaxf(w, ex2(x[h2][r][nb] - rel[nb]) * par_s(vp[h2][r][nb]));
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
              w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, o));
              sv = fmaxf(sv, __shfl_xor_sync(0xffffffffu, sv, o));
            }
            wm[nb] = w;
            const int ew = exponent(w), ev_old = 11 - exponent(up[nb]);
            int ev = max(ev_old, exponent(sv));
            ev = max(ew, min(ev, ew + kAttnSpare));
            ev = min(max(ev, -100), 127);
            up[nb] = pow2i(11 - ev);
            const float down = al * pow2i(min(max(ev_old - ev, -126), 127));
            l[nb] *= al;
            zs[nb] *= al;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[nb][k][j] *= down;
          }
        }
        // weights of 16 positions: (hi, lo) of each row's side by side, transposed
        auto weights = [&](int t, uint32_t (&wb)[NB][2]) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            float w[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float p = ex2(x[t][r][nb] - rel[nb]), sv = par_s(vp[t][r][nb]);
              l[nb] += p;
              zs[nb] = fmaf(p, fmaf(8.f, sv, par_z(vp[t][r][nb])), zs[nb]);
              w[r] = (p * sv) * up[nb];
            }
            const __half2 hi = __floats2half2_rn(w[0], w[1]);
            const float2 back = __half22float2(hi);
            const __half2 lo = __floats2half2_rn(w[0] - back.x, w[1] - back.y);
            const uint32_t h2 = *reinterpret_cast<const uint32_t*>(&hi), l2 = *reinterpret_cast<const uint32_t*>(&lo);
            wb[nb][0] = trans8x8(prmt(h2, l2, 0x5410u));
            wb[nb][1] = trans8x8(prmt(h2, l2, 0x7632u));
          }
        };
        if constexpr (kPairs) {
          // two MMAs from zero for each output tile, added in fp32
          uint32_t wb[2][NB][2];
          weights(0, wb[0]);
          weights(1, wb[1]);
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            uint32_t v[2][4];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                uint32_t one[1];
                lds(base + v_at + t * k_next + r * 4 * (HD / 2) + 4 * w, one);
                v[t][r] = one[0];
              }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t sel = half ? 0x7632u : 0x5410u;
              float d[NB][2][4];
#pragma unroll
              for (int t = 0; t < 2; ++t) {
                uint32_t ha[4], hb[4];
                centred4(prmt(v[t][0], v[t][1], sel), ha);
                centred4(prmt(v[t][2], v[t][3], sel), hb);
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                  for (int nb = 0; nb < NB; ++nb) {
                    if (t == 0)
                      mma_f16_new(d[nb][p], ha[2 * p], ha[2 * p + 1], hb[2 * p], hb[2 * p + 1],
                                  wb[t][nb][0], wb[t][nb][1]);
                    else
                      mma_f16(d[nb][p], ha[2 * p], ha[2 * p + 1], hb[2 * p], hb[2 * p + 1], wb[t][nb][0],
                              wb[t][nb][1]);
                  }
              }
#pragma unroll
              for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                  for (int j = 0; j < 4; ++j) acc[nb][w * 4 + half * 2 + p][j] += d[nb][p][j];
            }
          }
        } else {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            uint32_t v[4][VW];
#pragma unroll
            for (int r = 0; r < 4; ++r) lds(base + v_at + t * k_next + r * 4 * (HD / 2), v[r]);
            uint32_t wb[NB][2];
            weights(t, wb);
#pragma unroll
            for (int w = 0; w < VW; ++w) {
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const uint32_t sel = half ? 0x7632u : 0x5410u;
                uint32_t ha[4], hb[4];
                centred4(prmt(v[0][w], v[1][w], sel), ha);
                centred4(prmt(v[2][w], v[3][w], sel), hb);
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                  for (int nb = 0; nb < NB; ++nb) {
                    float(&o)[4] = acc[nb][w * 4 + half * 2 + p];
                    if constexpr (kWide) {
                      float d[4];
                      mma_f16_new(d, ha[2 * p], ha[2 * p + 1], hb[2 * p], hb[2 * p + 1], wb[nb][0], wb[nb][1]);
#pragma unroll
                      for (int j = 0; j < 4; ++j) o[j] += d[j];
                    } else {
                      mma_f16(o, ha[2 * p], ha[2 * p + 1], hb[2 * p], hb[2 * p + 1], wb[nb][0], wb[nb][1]);
                    }
                  }
              }
            }
          }
        }
        __syncwarp();                        // the stage may be copied over
        st = st + 1 == kAttnDepth ? 0 : st + 1;
        phase ^= st == 0 ? 1u : 0u;
      }
      if (kWide || pos >= t_end) break;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const float w_down = __uint_as_float(0x7F000000u - __float_as_uint(up[nb]));   // 1 / up
        float* const own_m = own_sums(NB * KS * 2 + nb);
        const float mf = flushed ? __ldcg(own_m) : kNegInf, f = mf == kNegInf ? 1.f : ex2(mf - m[nb]);
        __stcg(own_m, m[nb]);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float* const at = own_sums((nb * KS + k) * 2 + j);
            const float v = (acc[nb][k][2 * j] + acc[nb][k][2 * j + 1]) * w_down;
            __stcg(at, flushed ? fmaf(__ldcg(at), f, v) : v);
            acc[nb][k][2 * j] = acc[nb][k][2 * j + 1] = 0.f;
          }
      }
      flushed = true;
      stop = min(t_end, stop + kAttnFlush * kAttnStep);
    }
    __syncthreads();   // the rings are done with: the results take their place

    // ---- the warps' partials, relative to each warp's maximum -----------------
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float w_down = __uint_as_float(0x7F000000u - __float_as_uint(up[nb]));   // 1 / up
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l[nb] += __shfl_xor_sync(0xffffffffu, l[nb], o);
        zs[nb] += __shfl_xor_sync(0xffffffffu, zs[nb], o);
      }
      float* o = s_o + (warp * Q + nb * 4 + i) * HD + g * (HD / 8);
#pragma unroll
      for (int t = 0; t < KS; ++t) {
        o[2 * t] = fmaf(acc[nb][t][0] + acc[nb][t][1], w_down, zs[nb]);
        o[2 * t + 1] = fmaf(acc[nb][t][2] + acc[nb][t][3], w_down, zs[nb]);
      }
      if (flushed) {
        const float mf = __ldcg(own_sums(NB * KS * 2 + nb)), f = mf == kNegInf ? 1.f : ex2(mf - m[nb]);
#pragma unroll
        for (int t = 0; t < 2 * KS; ++t) o[t] = fmaf(__ldcg(own_sums(nb * KS * 2 + t)), f, o[t]);
      }
      if (g == 0) {
        s_ml[(warp * Q + nb * 4 + i) * 2] = m[nb];
        s_ml[(warp * Q + nb * 4 + i) * 2 + 1] = l[nb];
      }
    }
    __syncthreads();

    // ---- merge: the warps, then (for a shared item) the CTAs -------------------
    const int64_t c_first = cta_of(i0 + kAttnItemUnits), c_last = cta_of(i0 + size - 1);
    const int parts = static_cast<int>(c_last - c_first) + 1;
    auto store = [&](int qq, int d, const float4& o, float lsum) {
      const int qi = q0 + qq;
      if (qi >= nqueries) return;
      const int r = static_cast<int>(static_cast<unsigned>(qi) / static_cast<unsigned>(a.group));
      T* p = static_cast<T*>(a.out) + (r0 + r) * a.o_rs + (h * a.group + (qi - r * a.group)) * a.o_hs + d;
      const float inv = lsum == 0.f ? 0.f : 1.0f / lsum;
      p[0] = from_f<T>(o.x * inv);
      p[1] = from_f<T>(o.y * inv);
      p[2] = from_f<T>(o.z * inv);
      p[3] = from_f<T>(o.w * inv);
    };
    auto add = [](float4& o, float f, const float4& v) {
      o.x = fmaf(f, v.x, o.x);
      o.y = fmaf(f, v.y, o.y);
      o.z = fmaf(f, v.z, o.z);
      o.w = fmaf(f, v.w, o.w);
    };
    float* mypart = a.part + (c * 2 + (c == c_first && u0 < i0 ? 1 : 0)) * (Q * (HD + 2));
    for (int e = tid; e < Q * HD / 4; e += kAttnThreads) {
      const int qq = e / (HD / 4), d = (e - qq * (HD / 4)) * 4;
      float M = kNegInf;
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) M = fmaxf(M, s_ml[(w * Q + qq) * 2]);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float ls = 0.f;
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) {
        const float mw = s_ml[(w * Q + qq) * 2];
        const float f = mw == kNegInf ? 0.f : ex2(mw - M);
        add(o, f, *reinterpret_cast<const float4*>(s_o + (w * Q + qq) * HD + d));
        ls = fmaf(f, s_ml[(w * Q + qq) * 2 + 1], ls);
      }
      if (parts == 1) {
        store(qq, d, o, ls);
      } else {
        __stcg(reinterpret_cast<float4*>(mypart + qq * HD + d), o);
        if (d == 0) __stcg(reinterpret_cast<float2*>(mypart + Q * HD + qq * 2), make_float2(M, ls));
      }
    }
    if (parts > 1) {
      __syncthreads();
      if (tid == 0) {
        __threadfence();                     // the CTA's partial before its ticket
        const unsigned old = atomicAdd(a.tickets + c_first, 1u);
        *s_last = old == static_cast<unsigned>(parts - 1);
        __threadfence();
      }
      __syncthreads();
      if (*s_last) {
        // an item begins in its first CTA's last segment (slot 1 unless that CTA begins with
        // it) and is the first segment (slot 0) of the others
        const float* base = a.part + c_first * 2 * (Q * (HD + 2));
        const int skip = begin_of(c_first) < i0 ? Q * (HD + 2) : 0;
        // Threads take four dimensions; where that leaves threads over, groups of
        // them take every G-th part and meet in shared memory. The running maximum
        // is renewed every kFly parts, which are in flight together: one CTA reads
        // all of a long context's parts, so it is latency that counts here.
        constexpr int E = Q * HD / 4, G = E < kAttnThreads ? kAttnThreads / E : 1, kFly = 8;
        for (int e0 = 0; e0 < E; e0 += kAttnThreads) {
          const int e = e0 + tid % (E < kAttnThreads ? E : kAttnThreads), grp = tid / E % G;
          const int qq = e / (HD / 4), d = (e - qq * (HD / 4)) * 4;
          float M = kNegInf, ls = 0.f;
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int k0 = grp; k0 < parts; k0 += kFly * G) {
            float2 ml[kFly];
            float4 v[kFly];
            float mn = M;
#pragma unroll
            for (int k = 0; k < kFly; ++k) {
              const int part = k0 + k * G;
              const float* p = base + static_cast<int64_t>(part) * 2 * (Q * (HD + 2)) + (part == 0 ? skip : 0);
              const bool have = part < parts;
              ml[k] = have ? __ldcg(reinterpret_cast<const float2*>(p + Q * HD + qq * 2))
                           : make_float2(kNegInf, 0.f);
              v[k] = have ? __ldcg(reinterpret_cast<const float4*>(p + qq * HD + d))
                          : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int k = 0; k < kFly; ++k) mn = fmaxf(mn, ml[k].x);
            const float al = M == kNegInf ? 1.f : ex2(M - mn);   // (sums of 0, or NaN, without a maximum)
            M = mn;
            ls *= al;
            o = make_float4(o.x * al, o.y * al, o.z * al, o.w * al);
#pragma unroll
            for (int k = 0; k < kFly; ++k) {
              const float f = ml[k].x == kNegInf ? 0.f : ex2(ml[k].x - M);
              add(o, f, v[k]);
              ls = fmaf(f, ml[k].y, ls);
            }
          }
          if constexpr (G == 1) {
            store(qq, d, o, ls);
          } else {
            float4* g_o = reinterpret_cast<float4*>(s_o);             // [G][E]
            float2* g_ml = reinterpret_cast<float2*>(g_o + G * E);    // [G][E]
            __syncthreads();
            g_o[grp * E + e] = o;
            g_ml[grp * E + e] = make_float2(M, ls);
            __syncthreads();
            if (grp == 0) {
              float mn = M;
#pragma unroll
              for (int k = 1; k < G; ++k) mn = fmaxf(mn, g_ml[k * E + e].x);
              const float al = M == kNegInf ? 1.f : ex2(M - mn);
              ls *= al;
              o = make_float4(o.x * al, o.y * al, o.z * al, o.w * al);
#pragma unroll
              for (int k = 1; k < G; ++k) {
                const float2 t = g_ml[k * E + e];
                const float f = t.x == kNegInf ? 0.f : ex2(t.x - mn);
                add(o, f, g_o[k * E + e]);
                ls = fmaf(f, t.y, ls);
              }
              store(qq, d, o, ls);
            }
          }
        }
        if (tid == 0) a.tickets[c_first] = 0u;   // ready for the next call
      }
    }
    fence_async_smem();   // these reads and writes come before the next segment's copies
    __syncthreads();
  }
}

}  // namespace kv4
}  // namespace qz
