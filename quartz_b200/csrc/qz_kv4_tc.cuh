// qz_kv4_tc.cuh -- attention of many query rows (prompts and prompt chunks) over
// the paged 4-bit cache on the 5th-generation tensor cores (tcgen05 / TMEM).
//
// The same mathematics as attn_kernel (qz_kv4.cuh): the 4-bit codes are one
// operand, exact in fp16; q and the weights p * s_v are the other. fp32 rows are
// split into two fp16 limbs (22 bits); 16-bit rows take one: q then is exact
// (bf16 and fp16 fit fp16 after the row's power of two) and the weights' 2^-11
// is no more than the output's own rounding.
//
// An item is 128 (row, head) pairs of one kv head; heads of a group share the
// keys, so a tile is 128 / group query rows. Per tile of 128 positions
//   S [128 x 128] = Q codes(K)^T        A = Q from TMEM, B = K codes, K-major
//   O [128 x hd] += W (codes(V) - 8)    A = W from TMEM, B = V codes, MN-major
// Both A operands live in TMEM: with Q in shared memory an MMA would read 8 KB
// for 64 cycles of work, the whole bandwidth of shared memory, before the
// producers store anything. W overwrites S in place (a thread's own columns).
// TMEM columns: Q limbs 0..127, O 128..255, S/W double-buffered 256..511.
//
// 16 warps, one CTA per SM:
//   0-7   softmax; thread = (row, half of the tile's columns), warps w and w + 4
//         share rows and agree on a new maximum through one barrier reduction
//   8-14  producers: bulk copies bring the packed pages of a tile to shared
//         memory kTcRaw tiles ahead (issued by warp 8, one lane per page and
//         part); all seven turn them into fp16 tiles in the swizzled layout the
//         MMA reads, and (s, z) of each position into fp32
//   15    one thread issues the MMAs: S(t + 1) before O(t), so that the next
//         scores are ready when the softmax of this tile ends
// K and V tiles of a position row hold their dimensions in nibble order
// (0 4 1 5 2 6 3 7 of each word); Q is stored in the same order, and the
// epilogue puts O's columns back.
#pragma once

#include "qz_kv4.cuh"
#include "qz_tc_gemm.cuh"

namespace qz {
namespace kv4 {

constexpr int kTcThreads = 16 * 32;
constexpr int kTcProducers = 7 * 32;
constexpr int kTcRows = 128;    // (row, head) pairs per item
constexpr int kTcKeys = 128;    // positions per tile
constexpr int kTcRing = 4;      // parameter stages
constexpr int kTcRaw = 3;       // stages of packed tiles
constexpr uint32_t kColQ = 0, kColO = 128, kColS = 256;

struct TcArgs {
  AttnArgs a;
  int out_vec;   // out rows are 16-byte aligned
};

template <int HD>
__host__ __device__ constexpr int tc_tile_bytes() { return kTcKeys * HD * 2; }
// A packed tile: K codes, V codes, K's and V's (s, z) words.
template <int HD>
__host__ __device__ constexpr int tc_raw_bytes() { return kTcKeys * (HD + 8); }

// Shared memory: K and V tiles (two stages each), parameters, exchange words,
// barriers. At least 116 KB is asked for, so that one CTA (and its 512 TMEM
// columns) occupies an SM.
struct TcShared {
  float sk[kTcRing][kTcKeys], zk[kTcRing][kTcKeys];   // K's step and zero
  float sv[kTcRing][kTcKeys], zc[kTcRing][kTcKeys];   // V's step * 2^(9 - ev), zero + 8 step
  uint32_t valid[kTcRing][4];   // positions that exist, one bit each
  float down[kTcRing];          // 2^(ev before - ev): O's factor when V's exponent grows
  float w_down[kTcRing];        // 2^(ev - 9)
  float xa[2][kTcRows], xb[2][kTcRows];   // exchange between the two halves of a row
  float dmax[2][4];
  int64_t scan[128];
  int64_t item[2];              // request, tile within it
  uint64_t k_full[2], v_full[2], s_full[2], p_full[2], v_empty[2], par_full[kTcRing], q_ready, drain;
  uint64_t raw_full[kTcRaw], raw_empty[kTcRaw];
  uint32_t raw_groups[kTcRaw];  // which 16-position groups of a packed tile exist
  uint32_t tmem;
};

template <int HD>
__host__ __device__ constexpr int tc_smem() {
  constexpr int n = 4 * tc_tile_bytes<HD>() + kTcRaw * tc_raw_bytes<HD>() +
                    static_cast<int>(sizeof(TcShared)) + 1024;
  return n > 116 * 1024 ? n : 116 * 1024;
}

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

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
        "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
        "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// D[tmem] (+)= A[tmem] * B[smem], fp16 operands, fp32 accumulation.
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// D fp32, A / B fp16, M = 128; b_mn: B's memory is contiguous along N.
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(128 >> 4) << 24);
}

// MN-major operand, 128-byte swizzle: 64 elements of N per 128-byte row, eight
// rows (along K) per 1024-byte group, the next 64 elements of N `lead` bytes on.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t addr, uint32_t lead) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>((lead >> 4) & 0x3FFFu) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
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

// Whether `q` holds for any of the `n` threads at named barrier `id`.
__device__ __forceinline__ bool bar_any(int id, int n, bool q) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, o;\n\t"
      "setp.ne.b32 p, %3, 0;\n\t"
      "barrier.cta.red.or.pred o, %1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, o;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(n), "r"(q ? 1u : 0u)
      : "memory");
  return r != 0u;
}

// One word of eight codes as fp16 pairs, in nibble order 0 4 1 5 2 6 3 7: the
// subnormals c * 2^-24 (16 c * 2^-24 for nibbles 1, 5, 3, 7) for K ...
__device__ __forceinline__ uint4 k_pairs(uint32_t w) {
  const uint32_t y = w >> 8;
  return make_uint4(w & 0x000F000Fu, w & 0x00F000F0u, y & 0x000F000Fu, y & 0x00F000F0u);
}
// ... and c - 8 for V.
__device__ __forceinline__ uint4 v_pairs(uint32_t w) {
  uint32_t h[4];
  centred4(w, h);
  return make_uint4(h[0], h[1], h[2], h[3]);
}

template <class T, int HD>
__global__ void __launch_bounds__(kTcThreads, 1) attn_tc_kernel(const TcArgs args) {
  constexpr int L = sizeof(T) == 4 ? 2 : 1;      // fp16 limbs of q and of the weights
  constexpr int TB = tc_tile_bytes<HD>();
  constexpr int BLK = kTcKeys * 128;             // bytes of 64 dimensions of a tile
  constexpr float kNegInf = -INFINITY;
  const AttnArgs& a = args.a;
  extern __shared__ __align__(128) uint8_t tc_raw[];
  uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tc_raw) + 1023) &
                                              ~static_cast<uintptr_t>(1023));
  uint8_t* raws = tiles + 4 * TB;
  TcShared& sh = *reinterpret_cast<TcShared*>(raws + kTcRaw * tc_raw_bytes<HD>());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  pdl_wait();
  // ---- which item: tiles of `per` query rows of every handled request ---------
  const int per = kTcRows / a.group;
  if (tid < 128) {
    const int chunk = (a.B + 127) / 128;
    int64_t mine = 0;
    for (int k = 0; k < chunk; ++k) {
      const int64_t b = static_cast<int64_t>(tid) * chunk + k;
      int64_t r0;
      if (b < a.B) mine += (rows_of(a, b, &r0) + per - 1) / per;
    }
    sh.scan[tid] = mine;
  }
  if (tid == 0) {
    sh.item[0] = -1;
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&sh.k_full[s]), kTcProducers);
      mbar_init(smem_u32(&sh.v_full[s]), kTcProducers);
      mbar_init(smem_u32(&sh.s_full[s]), 1);
      mbar_init(smem_u32(&sh.p_full[s]), 256);
      mbar_init(smem_u32(&sh.v_empty[s]), 1);
    }
    for (int s = 0; s < kTcRing; ++s) mbar_init(smem_u32(&sh.par_full[s]), kTcProducers);
    for (int s = 0; s < kTcRaw; ++s) {
      mbar_init(smem_u32(&sh.raw_full[s]), 1);
      mbar_init(smem_u32(&sh.raw_empty[s]), kTcProducers);
    }
    mbar_init(smem_u32(&sh.q_ready), 256);
    mbar_init(smem_u32(&sh.drain), 1);
    fence_mbar_init();
  }
  __syncthreads();
  if (tid < 128) {
    const int chunk = (a.B + 127) / 128;
    int64_t before = 0, total = 0;
    for (int k = 0; k * chunk < a.B; ++k) {
      const int64_t v = sh.scan[k];
      before += k < tid ? v : 0;
      total += v;
    }
    // a request's later tiles see more: they start first
    const int64_t t = total - 1 - blockIdx.x / a.nkv;
    if (t >= 0 && t >= before && t < before + sh.scan[tid]) {
      int64_t b = static_cast<int64_t>(tid) * chunk, at = before, r0;
      for (int64_t n = (rows_of(a, b, &r0) + per - 1) / per; t >= at + n;
           n = (rows_of(a, b, &r0) + per - 1) / per) {
        at += n;
        ++b;
      }
      sh.item[0] = b;
      sh.item[1] = t - at;
    }
  }
  __syncthreads();
  const int64_t b = sh.item[0];
  if (b < 0) return;                       // the grid is an upper bound
  if (warp == 15) {
    tc::tmem_alloc(smem_u32(&sh.tmem), 512);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = sh.tmem;

  const int h = blockIdx.x % a.nkv;
  int64_t r0;
  const int64_t n = rows_of(a, b, &r0);
  const int64_t row0 = sh.item[1] * per;                       // first row of the item
  const int64_t len = a.lens[b], cap = a.width << a.shift;
  auto limit = [&](int64_t row) -> int {                       // positions [0, limit) are seen
    const int64_t l = len - n + row + 1;
    return static_cast<int>(l < 0 ? 0 : (l > cap ? cap : l));
  };
  const int seen = limit(row0 + per < n ? row0 + per - 1 : n - 1);
  const int nt = (seen + kTcKeys - 1) / kTcKeys;

  if (warp < 8) {
    // ======================= softmax =======================================
    const int r = tid & 127, half = tid >> 7, pair = 1 + (warp & 3);
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
    const int64_t row = row0 + r / a.group;
    const int head = h * a.group + r % a.group;
    const bool real = r < per * a.group && row < n;
    const int lim = real ? limit(row) : 0;

    // ---- q: this thread's half of the row, as fp16 limbs in TMEM --------------
    float F, Qs;
    {
      float x[HD / 2];
      if (real) {
        const T* p = static_cast<const T*>(a.q) + (r0 + row) * a.q_rs + head * a.q_hs + half * (HD / 2);
        load_row(p, a.vec, x);
      } else {
#pragma unroll
        for (int j = 0; j < HD / 2; ++j) x[j] = 0.f;
      }
      float mx = 0.f, sum = 0.f;
#pragma unroll
      for (int j = 0; j < HD / 2; ++j) {
        mx = fmaxf(mx, fabsf(x[j]));
        sum += x[j];
      }
      sh.xa[half][r] = mx;
      sh.xb[half][r] = sum;
      named_bar_sync(pair, 64);
      mx = fmaxf(mx, sh.xa[half ^ 1][r]);
      sum = sh.xb[0][r] + sh.xb[1][r];
      int e = static_cast<int>((__float_as_uint(mx) >> 23) & 255u) - 127;
      e = e < -113 ? -113 : (e > 117 ? 117 : e);
      const float up = pow2i(14 - e);
      F = pow2i(10 + e) * a.scale;
      Qs = sum * a.scale;
      const __half r16 = __ushort_as_half(0x2C00);   // 1 / 16
#pragma unroll
      for (int m = 0; m < HD / 16; m += 2) {
        uint32_t w[L][8];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t s[8];                             // (hi, lo) of eight dimensions
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            s[j] = split_h2(x[8 * (m + k) + j] * up);
            if (j & 1) {                             // odd nibbles stand as 16 c
              const __half2 t = __hmul2(*reinterpret_cast<const __half2*>(&s[j]), __half2half2(r16));
              s[j] = *reinterpret_cast<const uint32_t*>(&t);
            }
          }
#pragma unroll
          for (int l = 0; l < L; ++l) {
            const uint32_t sel = l ? 0x7632u : 0x5410u;
            w[l][4 * k] = prmt(s[0], s[4], sel);
            w[l][4 * k + 1] = prmt(s[1], s[5], sel);
            w[l][4 * k + 2] = prmt(s[2], s[6], sel);
            w[l][4 * k + 3] = prmt(s[3], s[7], sel);
          }
        }
#pragma unroll
        for (int l = 0; l < L; ++l)
          tmem_st8(lane_addr + kColQ + l * (HD / 2) + half * (HD / 4) + 4 * m, w[l]);
      }
      tmem_wait_st();
      tc::tc_fence_before();
      mbar_arrive(smem_u32(&sh.q_ready));
      named_bar_sync(pair, 64);   // xa is used again below
    }

    const f2_t F2 = f2_set(F, F), Q2 = f2_set(Qs, Qs);
    float m = kNegInf;
    f2_t l2 = f2_set(0.f, 0.f), zs2 = f2_set(0.f, 0.f);
    bool failed = false;
    for (int j = 0; j < nt; ++j) {
      const int ring = j & (kTcRing - 1), buf = j & 1;
      const int p0 = j * kTcKeys + half * 64;           // this thread's first position
      bool ok = mbar_wait(smem_u32(&sh.par_full[ring]), (j / kTcRing) & 1) &&
                mbar_wait(smem_u32(&sh.s_full[buf]), (j >> 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      tc::tc_fence_after();
      float top = kNegInf;
      const uint32_t va = sh.valid[ring][half * 2], vb = sh.valid[ring][half * 2 + 1];
      const bool whole = (va & vb) == 0xFFFFFFFFu && __all_sync(0xffffffffu, lim >= p0 + 64);
      // scores (base 2) of 16 positions; they are formed twice, for the maximum
      // and for the weights, which costs three instructions per two positions
      // and saves holding 64 of them
      const float4* sk4 = reinterpret_cast<const float4*>(&sh.sk[ring][half * 64]);
      const float4* zk4 = reinterpret_cast<const float4*>(&sh.zk[ring][half * 64]);
      auto scores = [&](int c, f2_t (&x)[8]) {
        uint32_t v[16];
        tc::tmem_ld16(lane_addr + kColS + buf * 128 + half * 64 + 16 * c, v);
        tc::tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float4 s = sk4[4 * c + k], z = zk4[4 * c + k];
          x[2 * k] = f2_fma(f2_mul(f2_pack(v[4 * k], v[4 * k + 1]), F2), f2_set(s.x, s.y),
                            f2_mul(f2_set(z.x, z.y), Q2));
          x[2 * k + 1] = f2_fma(f2_mul(f2_pack(v[4 * k + 2], v[4 * k + 3]), F2),
                                f2_set(s.z, s.w), f2_mul(f2_set(z.z, z.w), Q2));
        }
        if (!whole) {
          const uint32_t bits = (c < 2 ? va : vb) >> (16 * (c & 1));
          const int left = lim - p0 - 16 * c;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float2 t = f2_unpack(x[k]);
            x[k] = f2_set((bits >> (2 * k)) & 1u && 2 * k < left ? t.x : kNegInf,
                          (bits >> (2 * k)) & 2u && 2 * k + 1 < left ? t.y : kNegInf);
          }
        }
      };
      if (ok) {
#pragma unroll 2
        for (int c = 0; c < 4; ++c) {
          f2_t x[8];
          scores(c, x);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float2 t = f2_unpack(x[k]);
            top = fmaxf(top, fmaxf(t.x, t.y));
          }
        }
      }
      const float down = sh.down[ring];
      if (bar_any(pair, 64, !ok || top > m + 4.f || down != 1.f)) {
        // a new maximum for the pair's rows (or a new exponent of V's steps)
        sh.xa[half][r] = top;
        if (bar_any(pair, 64, !ok)) {
          failed = true;
          break;
        }
        const float mn = fmaxf(m, fmaxf(top, sh.xa[half ^ 1][r]));
        const float al = m == kNegInf ? 1.f : ex2(m - mn);
        m = mn;
        l2 = f2_mul(l2, f2_set(al, al));
        zs2 = f2_mul(zs2, f2_set(al, al));
        if (j > 0) {
          bool done = mbar_wait(smem_u32(&sh.v_empty[(j - 1) & 1]), ((j - 1) >> 1) & 1);
          done = __all_sync(0xffffffffu, done);
          if (!done && lane == 0) report_error(ERR_WAIT_FULL, 0x401u);
          tc::tc_fence_after();
          const float f = al * down;
#pragma unroll
          for (int c = 0; c < HD / 2; c += 16) {
            uint32_t o[16];
            const uint32_t at = lane_addr + kColO + half * (HD / 2) + c;
            tc::tmem_ld16(at, o);
            tc::tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
            tmem_st8(at, o);
            tmem_st8(at + 8, o + 8);
          }
          tmem_wait_st();
        }
        named_bar_sync(pair, 64);   // xa is free again
      }
      // weights, over this thread's own columns of S
      const float mu = m == kNegInf ? 0.f : -m;
      const f2_t mu2 = f2_set(mu, mu);
      const float4* sv4 = reinterpret_cast<const float4*>(&sh.sv[ring][half * 64]);
      const float4* zc4 = reinterpret_cast<const float4*>(&sh.zc[ring][half * 64]);
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {       // 16 positions: one K step of the MMA
        f2_t x[8];
        scores(c, x);
        uint32_t w[8 * L];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float4 s = sv4[4 * c + q], z = zc4[4 * c + q];
          if (!whole) {
            // selected, not multiplied, away: a hidden position may hold anything
            const float2 a0 = f2_unpack(x[2 * q]), a1 = f2_unpack(x[2 * q + 1]);
            if (a0.x == kNegInf) s.x = z.x = 0.f;
            if (a0.y == kNegInf) s.y = z.y = 0.f;
            if (a1.x == kNegInf) s.z = z.z = 0.f;
            if (a1.y == kNegInf) s.w = z.w = 0.f;
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 t = f2_unpack(f2_add(x[2 * q + e], mu2));
            const f2_t p = f2_set(ex2(t.x), ex2(t.y));
            l2 = f2_add(l2, p);
            zs2 = f2_fma(p, e ? f2_set(z.z, z.w) : f2_set(z.x, z.y), zs2);
            const float2 y = f2_unpack(f2_mul(p, e ? f2_set(s.z, s.w) : f2_set(s.x, s.y)));
            const __half2 hi = __floats2half2_rn(y.x, y.y);
            w[2 * q + e] = *reinterpret_cast<const uint32_t*>(&hi);
            if constexpr (L == 2) {
              const float2 back = __half22float2(hi);
              const __half2 lo = __floats2half2_rn(y.x - back.x, y.y - back.y);
              w[8 + 2 * q + e] = *reinterpret_cast<const uint32_t*>(&lo);
            }
          }
        }
        const uint32_t at = lane_addr + kColS + buf * 128 + half * 64 + c * (8 * L);
#pragma unroll
        for (int l = 0; l < L; ++l) tmem_st8(at + 8 * l, w + 8 * l);
      }
      tmem_wait_st();
      tc::tc_fence_before();
      mbar_arrive(smem_u32(&sh.p_full[buf]));
    }
    if (failed && lane == 0) report_error(ERR_WAIT_FULL, 0x400u);
    // ---- epilogue ---------------------------------------------------------------
    const float2 lt = f2_unpack(l2), zt = f2_unpack(zs2);
    sh.xa[half][r] = lt.x + lt.y;
    sh.xb[half][r] = zt.x + zt.y;
    named_bar_sync(pair, 64);
    const float l = sh.xa[0][r] + sh.xa[1][r], zs = sh.xb[0][r] + sh.xb[1][r];
    bool ok = !failed;
    if (nt > 0 && ok) ok = mbar_wait(smem_u32(&sh.v_empty[(nt - 1) & 1]), ((nt - 1) >> 1) & 1);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok && lane == 0) report_error(ERR_WAIT_FULL, 0x402u);
    tc::tc_fence_after();
    const float wd = nt > 0 ? sh.w_down[(nt - 1) & (kTcRing - 1)] : 0.f;
    T* o = static_cast<T*>(a.out) + (r0 + row) * a.o_rs + head * a.o_hs + half * (HD / 2);
    if (ok) {
#pragma unroll
      for (int c = 0; c < HD / 2; c += 32) {
        uint32_t u[32];
        if (nt > 0) {
          tmem_ld32(lane_addr + kColO + half * (HD / 2) + c, u);
          tc::tmem_wait_ld();
        }
        T y[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          // column 8 w + k holds dimension 8 w + (k / 2) + (k odd ? 4 : 0)
          const int d = (k & ~7) + ((k & 7) >> 1) + ((k & 1) << 2);
          const float t = nt > 0 ? fmaf(__uint_as_float(u[k]), wd, zs) : 0.f;
          y[d] = from_f<T>(l == 0.f ? 0.f : t / l);
        }
        if (real) {
          if (args.out_vec) {
            constexpr int pv = 16 / sizeof(T);
#pragma unroll
            for (int k = 0; k < 32 / pv; ++k)
              reinterpret_cast<uint4*>(o + c)[k] = *reinterpret_cast<const uint4*>(y + k * pv);
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) o[c + k] = y[k];
          }
        }
      }
    }
  } else if (warp < 15) {
    // ======================= producers =====================================
    const int dt = tid - 256;
    constexpr int LPR = HD / 32;                 // 16-byte chunks per code row
    constexpr int NC = 128 * LPR;                // ... per tile
    constexpr int RB = tc_raw_bytes<HD>();
    const int64_t ps = int64_t(1) << a.shift;
    const int32_t* tab = a.table + b * a.width;
    // ---- the copies of one tile: lane = (page of the tile, part of its block) --
    const int cnt = a.shift < 7 ? 1 << a.shift : kTcKeys;        // positions per copy
    const int pg = lane >> 2, part = lane & 3;
    auto page_of = [&](int j) -> int {
      const int p = j * kTcKeys + pg * cnt;
      return pg * cnt < kTcKeys && p < seen ? __ldg(tab + (p >> a.shift)) : -1;
    };
    int page = -1;
    auto issue = [&](int j) {      // warp 8; `page` is page_of(j)
      const int st = j % kTcRaw;
      const bool have = page >= 0 && page < a.pages;
      const uint32_t bytes = cnt * (part < 2 ? HD / 2 : 4);
      const uint32_t total = __reduce_add_sync(0xffffffffu, have ? bytes : 0u);
      const uint32_t groups = __reduce_or_sync(
          0xffffffffu, have ? ((1u << (cnt >> 4)) - 1u) << (pg * (cnt >> 4)) : 0u);
      const uint32_t bar = smem_u32(&sh.raw_full[st]);
      if (lane == 0) {
        sh.raw_groups[st] = groups;
        mbar_arrive_expect_tx(bar, total);
      }
      __syncwarp();
      if (have) {
        const int64_t off = (j * kTcKeys + pg * cnt) & (ps - 1);
        const uint8_t* src = a.pool + (static_cast<int64_t>(page) * a.nkv + h) * (ps * (HD + 8));
        src += part < 2 ? part * (ps * (HD / 2)) + off * (HD / 2) : ps * HD + (part - 2) * (ps * 4) + off * 4;
        const uint32_t dst = smem_u32(raws + st * RB) +
                             (part < 2 ? part * (kTcKeys * (HD / 2)) + pg * cnt * (HD / 2)
                                       : kTcKeys * HD + (part - 2) * (kTcKeys * 4) + pg * cnt * 4);
        bulk_copy(dst, src, bytes, bar);
      }
      page = page_of(j + 1);
    };
    // Codes of the tile -> fp16. The eight threads of one store phase hold two
    // rows (hd 128) and four chunks of each; taking the last two chunks' words
    // in the order 2 3 0 1 keeps their sixteen-byte columns apart.
    auto put = [&](uint8_t* tile, const uint8_t* codes, uint32_t groups, bool is_v) {
#pragma unroll 2
      for (int t = dt; t < NC; t += kTcProducers) {
        const int row = t / LPR, ci = t % LPR;
        uint4 c4 = *reinterpret_cast<const uint4*>(codes + t * 16);
        if (!((groups >> (row >> 4)) & 1u)) c4 = make_uint4(0u, 0u, 0u, 0u);   // never copied
        const bool swap = LPR == 4 && (ci & 2);
        const uint32_t w[4] = {swap ? c4.z : c4.x, swap ? c4.w : c4.y, swap ? c4.x : c4.z,
                               swap ? c4.y : c4.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int c = ci * 4 + (swap ? k ^ 2 : k);       // word of the row
          const uint4 u = is_v ? v_pairs(w[k]) : k_pairs(w[k]);
          *reinterpret_cast<uint4*>(tile + (c >> 3) * BLK + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = u;
        }
      }
    };
    bool fail = false;
    int ev = -100, issued = 0, landed = 0;
    if (warp == 8) {
      page = page_of(0);
      for (; issued < kTcRaw - 1 && issued < nt; ++issued) issue(issued);
    }
    for (int j = 0; j < nt; ++j) {
      const int ring = j & (kTcRing - 1), buf = j & 1, st = j % kTcRaw;
      if (warp == 8 && issued < nt && !fail) {
        // the stage of tile j - 1, read by every producer before it arrived there
        if (j > 0 && !mbar_wait(smem_u32(&sh.raw_empty[(j - 1) % kTcRaw]), ((j - 1) / kTcRaw) & 1)) {
          report_error(ERR_WAIT_EMPTY, 0x412u);
          fail = true;
        }
        fail = __any_sync(0xffffffffu, fail);
        if (!fail) issue(issued++);
      }
      if (!fail && !mbar_wait(smem_u32(&sh.raw_full[st]), (j / kTcRaw) & 1)) {
        report_error(ERR_WAIT_FULL, 0x413u);
        fail = true;
      }
      if (!fail) landed = j + 1;
      const uint8_t* raw = raws + st * RB;
      const uint32_t groups = sh.raw_groups[st];
      // parameters, one position a thread; weights are p * s_v * 2^(9 - ev), ev
      // the largest exponent so far
      const bool mine = dt < kTcKeys;            // whole warps
      const bool here = mine && j * kTcKeys + dt < seen && ((groups >> (dt >> 4)) & 1u);
      uint32_t kpar = 0u, vpar = 0u;             // positions that do not exist: s = z = 0
      if (here) {
        kpar = *reinterpret_cast<const uint32_t*>(raw + kTcKeys * HD + dt * 4);
        vpar = *reinterpret_cast<const uint32_t*>(raw + kTcKeys * (HD + 4) + dt * 4);
      }
      const float sv = par_s(vpar);
      if (mine) {
        float t = fmaxf(sv, 0.f);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
        const uint32_t bits = __ballot_sync(0xffffffffu, here);
        if (lane == 0) {
          sh.dmax[j & 1][warp - 8] = t;
          sh.valid[ring][warp - 8] = bits;
        }
      }
      if (bar_any(5, kTcProducers, fail)) {
        fail = true;
        break;
      }
      const float mx = fmaxf(fmaxf(sh.dmax[j & 1][0], sh.dmax[j & 1][1]),
                             fmaxf(sh.dmax[j & 1][2], sh.dmax[j & 1][3]));
      int e = static_cast<int>((__float_as_uint(mx) >> 23) & 255u) - 127;
      e = e > 127 ? 127 : e;
      const int ev_old = ev;
      ev = e > ev ? e : ev;
      if (mine) {
        sh.sk[ring][dt] = par_s(kpar);
        sh.zk[ring][dt] = par_z(kpar);
        sh.sv[ring][dt] = sv * pow2i(9 - ev);
        sh.zc[ring][dt] = fmaf(8.f, sv, par_z(vpar));
      }
      if (dt == 0) {
        sh.down[ring] = j == 0 || ev_old - ev < -126 ? (j == 0 ? 1.f : 0.f) : pow2i(ev_old - ev);
        sh.w_down[ring] = pow2i(ev - 9);
      }
      mbar_arrive(smem_u32(&sh.par_full[ring]));
      // K (its stage is free once S(j - 2) is done), then V (once O(j - 2) is)
      if (j >= 2 && !mbar_wait(smem_u32(&sh.s_full[buf]), ((j >> 1) - 1) & 1)) {
        report_error(ERR_WAIT_EMPTY, 0x410u);
        fail = true;
      }
      if (!fail) {
        put(tiles + buf * TB, raw, groups, false);
        fence_async_smem();
        mbar_arrive(smem_u32(&sh.k_full[buf]));
      }
      if (!fail && j >= 2 && !mbar_wait(smem_u32(&sh.v_empty[buf]), ((j >> 1) - 1) & 1)) {
        report_error(ERR_WAIT_EMPTY, 0x411u);
        fail = true;
      }
      if (!fail) {
        put(tiles + (2 + buf) * TB, raw + kTcKeys * (HD / 2), groups, true);
        fence_async_smem();
        mbar_arrive(smem_u32(&sh.v_full[buf]));
        mbar_arrive(smem_u32(&sh.raw_empty[st]));
      }
    }
    // after a failed wait: no copy stays in flight into memory that is given up
    for (int t = landed; t < issued; ++t)
      if (!mbar_wait(smem_u32(&sh.raw_full[t % kTcRaw]), (t / kTcRaw) & 1)) {
        report_error(ERR_DRAIN, 0x414u);
        break;
      }
  } else if (lane == 0 && nt > 0) {
    // ======================= MMA issuer ====================================
    constexpr uint32_t id_s = idesc_f16(kTcKeys, false), id_o = idesc_f16(HD, true);
    auto scores = [&](int j) {
      const uint32_t kt = smem_u32(tiles + (j & 1) * TB), d = tmem + kColS + (j & 1) * 128;
#pragma unroll
      for (int s = 0; s < HD / 16; ++s)
#pragma unroll
        for (int l = 0; l < L; ++l)
          mma_f16_ts(d, tmem + kColQ + l * (HD / 2) + s * 8,
                     tc::smem_desc_sw128(kt + (s >> 2) * BLK + (s & 3) * 32), id_s, (s | l) != 0);
      tc::tc_commit(smem_u32(&sh.s_full[j & 1]));
    };
    bool ok = mbar_wait(smem_u32(&sh.q_ready), 0) && mbar_wait(smem_u32(&sh.k_full[0]), 0);
    tc::tc_fence_after();
    if (ok) scores(0);
    for (int j = 0; ok && j < nt; ++j) {
      if (j + 1 < nt) {
        // S(j + 1) goes where W(j - 1) was; the MMAs run in the order of issue
        ok = mbar_wait(smem_u32(&sh.k_full[(j + 1) & 1]), ((j + 1) >> 1) & 1);
        if (!ok) break;
        tc::tc_fence_after();
        scores(j + 1);
      }
      ok = mbar_wait(smem_u32(&sh.v_full[j & 1]), (j >> 1) & 1) &&
           mbar_wait(smem_u32(&sh.p_full[j & 1]), (j >> 1) & 1);
      if (!ok) break;
      tc::tc_fence_after();
      const uint32_t vt = smem_u32(tiles + (2 + (j & 1)) * TB), w = tmem + kColS + (j & 1) * 128;
#pragma unroll
      for (int s = 0; s < kTcKeys / 16; ++s)
#pragma unroll
        for (int l = 0; l < L; ++l)
          mma_f16_ts(tmem + kColO, w + (s >> 2) * 64 + (s & 3) * (8 * L) + 8 * l,
                     smem_desc_mn(vt + s * 2048, BLK), id_o, (j | s | l) != 0);
      tc::tc_commit(smem_u32(&sh.v_empty[j & 1]));
    }
    if (!ok) report_error(ERR_WAIT_FULL, 0x420u);
    // TMEM and shared memory are given up only after every issued MMA has finished
    tc::tc_commit(smem_u32(&sh.drain));
    if (!mbar_wait(smem_u32(&sh.drain), 0)) report_error(ERR_DRAIN, 0x421u);
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 15) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

}  // namespace kv4
}  // namespace qz
