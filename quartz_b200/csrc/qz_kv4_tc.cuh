// qz_kv4_tc.cuh -- attention of many query rows (prompts and prompt chunks) over
// the paged 4-bit cache on the 5th-generation tensor cores (tcgen05 / TMEM).
//
// The same mathematics as attn_kernel (qz_kv4.cuh): the 4-bit codes are one
// operand, exact in fp16; q and the weights p * s_v are the other. The weights are
// split into two fp16 limbs (22 bits), and so is q of fp32 rows; q of 16-bit rows
// takes one, which is exact (bf16 and fp16 fit fp16 after the row's power of two).
// One limb for the weights of 16-bit rows would add an error of the size of fp16's
// rounding (2^-12 each: results 2.6e-4 off 64 bits where the rounding is 2.1e-4).
//
// An item is 128 (row, head) pairs of one kv head; heads of a group share the
// keys, so a tile is 128 / group query rows. Per tile of 128 positions
//   S [128 x 128] = Q codes(K)^T        A = Q from TMEM, B = K codes (fp32 rows:
//                                       less 8), K-major
//   O [128 x hd] += W (codes(V) - 8)    A = W from TMEM, B = V codes, MN-major
// Both A operands live in TMEM: with Q in shared memory an MMA would read 8 KB
// for 64 cycles of work, the whole bandwidth of shared memory, before the
// producers store anything. W overwrites S in place (a thread's own columns).
// TMEM columns: Q limbs 0..127, O 128..255, S/W double-buffered 256..511.
//
// 24 warps, one CTA per SM:
//   0-15  softmax. A row of a tile has two threads, one for each 64 positions;
//         groups of four warps take (even tiles, first half), (odd, first),
//         (even, second), (odd, second), so each scheduler has four warps in
//         different phases to hide latency behind. A row's maximum is agreed
//         between its two threads and passed on from tile to tile through
//         shared memory, before the weights are formed.
//   16-19 converters: packed codes -> fp16 tiles in the swizzled layout the MMA
//         reads
//   20    parameters: (s, z) of each position -> fp32 arrays
//   21    loader: one bulk copy per page brings a tile's packed blocks to shared
//         memory, kTcRaw tiles ahead
//   22    issues the MMAs: S(t + 1) before O(t), so that the next scores are
//         ready when the softmax of this tile ends
//   23    takes a place of the workspace for the item's fp32 sums
// A row's weights p s_v go into fp16 as p s_v 2^(10 - ev), p relative to the row's
// running maximum (below 2^4) and ev the largest exponent so far of a position's
// u = max(s_v, |z_v + 8 s_v| / 8), a bound of what a code can add; what lies below
// 2^-25 of that is lost. While all u seen lie within 2^8 of each other a row's largest
// weight keeps 2^-26 of itself, whatever its scores. Where they do not (`wide`, from
// that tile of an item on), a row with no weight near the largest u is taken relative
// to less than its maximum, as far as its largest p u asks for: tiles then take the
// largest of score + log2 u of each row too.
//
// K and V tiles of a position row hold their dimensions in nibble order
// (0 4 1 5 2 6 3 7 of each word); Q is stored in the same order, and the
// epilogue puts O's columns back.
//
// Measured: a prompt of 4096, 32 heads, 8 kv heads of 128: 392 us (fp32), tensor pipe
// 28 %; a tile takes 2.6 us (fp32) or 2.2 us (16 bits), of which the MMAs are 1.0 or 0.8:
// two tiles are in flight and each is a chain of scores, maximum, weights and sums. A
// prompt with `wide` tiles takes 424 us.
#pragma once

#include "qz_kv4.cuh"
#include "qz_tc_gemm.cuh"

namespace qz {
namespace kv4 {

constexpr int kTcThreads = 24 * 32;
constexpr int kTcSoftmax = 16 * 32;
constexpr int kTcConverters = 4 * 32;
constexpr int kTcRows = 128;    // (row, head) pairs per item
constexpr int kTcKeys = 128;    // positions per tile
// Parameter stages. Tile j's are written once its packed tile has landed, so
// after tile j - kTcRaw was converted, so after O(j - kTcRaw - 2) was issued:
// the softmax is at most kTcRaw + 1 tiles behind.
constexpr int kTcRing = 8;
constexpr int kTcRaw = 3;       // stages of packed tiles
constexpr int kTcSpare = 8;     // how far u's exponents may spread before `wide`
constexpr uint32_t kColQ = 0, kColO = 128, kColS = 256;

struct TcArgs {
  AttnArgs a;
  int out_vec;      // out rows are 16-byte aligned
  int slots;        // places of `sums`, one for each SM
  float4* sums;     // [slots][HD / 4][kTcRows]
  unsigned* taken;  // [slots]: 1 while a CTA owns the place, 0 between calls
};

// Tiles that O accumulates in TMEM before it is added to fp32 sums in the
// workspace (L2). The MMA truncates its accumulator, 16 times a tile and by about
// 3e-8 of it each time, so a chain of n tiles that grows evenly ends 16 n 3e-8 / 2
// low: 1e-5 of itself after 40 tiles, 2e-4 after 100000 positions. Even: the odd
// tiles' threads do it, while the even ones work on the next tile. fp32 rows, every
// two tiles: 5e-7 off 64 bits at 4096 positions; every four 1.1e-6 and 4 % faster.
// 16-bit rows round by 2^-12 at least, 16 tiles drift by 4e-6 (fp16 over 40000
// positions 2.08e-4 off 64 bits, the rounding 2.07e-4; every 8 tiles 2.5 % slower).
template <int L>
__host__ __device__ constexpr int tc_flush() { return L == 2 ? 2 : 16; }

__device__ __forceinline__ uint32_t sm_id() {
  uint32_t id;
  asm volatile("mov.u32 %0, %%smid;" : "=r"(id));
  return id;
}
// A place of `sums` for this CTA alone. At most one CTA per SM runs, so there is one that
// is free; the SM's number only says where to look first (a CTA may be moved while it
// runs, so the number owns nothing). -1, and an error, where a workspace is shared with a
// call that runs at the same time.
__device__ __forceinline__ int take_place(unsigned* taken, int slots) {
  const unsigned first = sm_id();
  for (unsigned k = 0; k < 64u * slots; ++k) {
    const int p = static_cast<int>((first + k) % static_cast<unsigned>(slots));
    if (atomicCAS(taken + p, 0u, 1u) == 0u) {
      __threadfence();                   // what its last owner wrote comes first
      return p;
    }
  }
  report_error(ERR_WAIT_EMPTY, 0x404u);
  return -1;
}
__device__ __forceinline__ void leave_place(unsigned* taken, int p) {
  if (p < 0) return;
  __threadfence();
  atomicExch(taken + p, 0u);
}
template <int HD>
__device__ __forceinline__ float4* sums_of(const TcArgs& args, int place) {
  return args.sums + static_cast<size_t>(place) * (HD / 4 * kTcRows);
}

template <int HD>
__host__ __device__ constexpr int tc_tile_bytes() { return kTcKeys * HD * 2; }
// A packed tile: K codes, V codes, K's and V's (s, z) words.
template <int HD>
__host__ __device__ constexpr int tc_raw_bytes() { return kTcKeys * (HD + 8); }

// Shared memory: K and V tiles (two stages each), parameters, exchange words,
// barriers. At least 116 KB is asked for, so that one CTA (and its 512 TMEM
// columns) occupies an SM.
struct TcShared {
  float sk[kTcRing][kTcKeys], zk[kTcRing][kTcKeys];   // K's step, zero (+ 8 step if centred)
  float sv[kTcRing][kTcKeys], zc[kTcRing][kTcKeys];   // V's step * 2^(10 - ev), zero + 8 step
  float lu[kTcRing][kTcKeys];   // log2(u) + 10 - ev
  alignas(16) uint32_t valid[kTcRing][4];   // positions that exist, one bit each
  float down[kTcRing];          // 2^(ev before - ev): O's factor when V's exponent grows
  float w_down[kTcRing];        // 2^(ev - 10)
  uint32_t wide[kTcRing];       // the u so far differ by more than 2^kTcSpare
  float top[2][2][kTcRows];     // [tile & 1][half]: maximum of a row's half tile
  float topu[2][2][kTcRows];    // and of score + lu, of all tiles so far (wide tiles only)
  float max[2][kTcRows];        // [tile & 1]: what a row's scores are taken relative to
  // [tile & 1]: the largest score and score + lu so far, relative to `max` (wide tiles only)
  float peak[2][kTcRows], peaku[2][kTcRows];
  // exchange between a row's four threads, when q is read and at the end (a group
  // without a tile reaches the end while others still read q)
  float ex_q[2][4][kTcRows], ex[3][4][kTcRows];
  // [half]: what a row's sums in the workspace stand relative to, and their w_down
  float flushed[2][kTcRows], flushed_w[2][kTcRows];
  int place;                    // in the workspace (or -1: none was free)
  uint32_t odd[kTcRing];        // a V parameter of the tile is not finite
  int64_t scan[128];
  int item[6];                  // request, first row, rows, first row of q, len - rows, positions seen
  uint64_t k_full[2], v_full[2], s_full[2], p_full[2], v_empty[2], par_full[kTcRing], q_ready, drain;
  uint64_t raw_full[kTcRaw], raw_empty[kTcRaw], t_full[2][4], m_full[2][4], o_free;
  uint32_t raw_groups[kTcRaw];  // which 16-position groups of a packed tile exist
  uint32_t tmem;
};

template <int HD>
__host__ __device__ constexpr int tc_smem() {
  constexpr int n = 4 * tc_tile_bytes<HD>() + kTcRaw * tc_raw_bytes<HD>() +
                    static_cast<int>(sizeof(TcShared)) + 1024;
  return n > 116 * 1024 ? n : 116 * 1024;
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

// The four pairs of a word's codes, in nibble order 0 4 1 5 2 6 3 7, as they lie:
// c * 2^-24, and 16 c * 2^-24 for nibbles 1, 5, 3, 7.
__device__ __forceinline__ void subnormal4(uint32_t x, uint32_t (&h)[4]) {
  const uint32_t y = x >> 8;
  h[0] = x & 0x000F000Fu;
  h[1] = x & 0x00F000F0u;
  h[2] = y & 0x000F000Fu;
  h[3] = y & 0x00F000F0u;
}

// One word of eight codes as fp16 pairs in nibble order 0 4 1 5 2 6 3 7: less 8, or
// (SUB) as the subnormals that they are, for K of 16-bit rows (see attn_kernel).
template <bool SUB>
__device__ __forceinline__ uint4 pairs_of(uint32_t w) {
  uint32_t h[4];
  if constexpr (SUB) subnormal4(w, h); else centred4(w, h);
  return make_uint4(h[0], h[1], h[2], h[3]);
}

// Registers per thread of a warpgroup (all four warps call it). The shares of
// the six warpgroups, 4 * 88 + 72 + 56, are the launch's 6 * 80.
template <int N>
__device__ __forceinline__ void regs_more() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_less() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xFFFFFFFF;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0u;
}

// mbar_wait by a whole warp: true if every lane saw the phase complete.
__device__ __forceinline__ bool warp_wait(const uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity));
}

// What a thread has summed of its row, relative to 2^m.
struct RowState {
  float m;         // what the sums stand relative to
  f2_t l, zs;      // sum of p, sum of p (z_v + 8 s_v)
};

// x = score + mu of 64 positions, in TMEM in place of S; returns their maximum. MASK: positions
// that do not exist (bits of `valid`) or lie at `lim` or behind it, counted from the first, become
// -inf.
template <bool MASK>
__device__ __forceinline__ float tc_scores(uint32_t taddr, const float* sk, const float* zk, f2_t F2,
                                           f2_t Q2, f2_t mu2, const uint32_t* valid, int lim) {
  float t0 = -INFINITY, t1 = -INFINITY;
  uint32_t v[2][16];
  tc::tmem_ld16(taddr, v[0]);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    tc::tmem_wait_ld();
    if (c < 3) tc::tmem_ld16(taddr + 16 * (c + 1), v[(c + 1) & 1]);
    uint32_t(&u)[16] = v[c & 1];
    const uint32_t bits = MASK ? valid[c >> 1] >> (16 * (c & 1)) : 0u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 s = reinterpret_cast<const float4*>(sk)[4 * c + k];
      const float4 z = reinterpret_cast<const float4*>(zk)[4 * c + k];
      float2 a = f2_unpack(f2_fma(f2_mul(f2_pack(u[4 * k], u[4 * k + 1]), F2), f2_set(s.x, s.y),
                                  f2_fma(f2_set(z.x, z.y), Q2, mu2)));
      float2 b = f2_unpack(f2_fma(f2_mul(f2_pack(u[4 * k + 2], u[4 * k + 3]), F2), f2_set(s.z, s.w),
                                  f2_fma(f2_set(z.z, z.w), Q2, mu2)));
      if constexpr (MASK) {
        const int left = lim - 16 * c - 4 * k;
        const uint32_t four = bits >> (4 * k);
        a.x = (four & 1u) && left > 0 ? a.x : -INFINITY;
        a.y = (four & 2u) && left > 1 ? a.y : -INFINITY;
        b.x = (four & 4u) && left > 2 ? b.x : -INFINITY;
        b.y = (four & 8u) && left > 3 ? b.y : -INFINITY;
      }
      t0 = fmaxf(t0, fmaxf(a.x, a.y));
      t1 = fmaxf(t1, fmaxf(b.x, b.y));
      u[4 * k] = __float_as_uint(a.x);
      u[4 * k + 1] = __float_as_uint(a.y);
      u[4 * k + 2] = __float_as_uint(b.x);
      u[4 * k + 3] = __float_as_uint(b.y);
    }
    tmem_st8(taddr + 16 * c, u);
    tmem_st8(taddr + 16 * c + 8, u + 8);
  }
  tmem_wait_st();
  return fmaxf(t0, t1);
}

// The maximum of x + lu over 64 positions.
__device__ __forceinline__ float tc_top_u(uint32_t taddr, const float* lu) {
  float t = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < 64; c += 16) {
    uint32_t x[16];
    tc::tmem_ld16(taddr + c, x);
    tc::tmem_wait_ld();
#pragma unroll
    for (int k = 0; k < 16; ++k) t = fmaxf(t, __uint_as_float(x[k]) + lu[c + k]);
  }
  return t;
}

// n columns of this row times f plus d.
template <int n>
__device__ __forceinline__ void tc_rescale(uint32_t taddr, float f, float d) {
#pragma unroll 1
  for (int c = 0; c < n; c += 16) {
    uint32_t o[16];
    tc::tmem_ld16(taddr + c, o);
    tc::tmem_wait_ld();
#pragma unroll
    for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(fmaf(__uint_as_float(o[k]), f, d));
    tmem_st8(taddr + c, o);
    tmem_st8(taddr + c + 8, o + 8);
  }
  tmem_wait_st();
}

// Weights of 64 positions into TMEM, in place of x (the two limbs of 16 positions side
// by side, as many columns as x). SELECT: parameters of hidden positions may be NaN, so they are selected
// away; otherwise p = 0 makes their products vanish.
template <bool SELECT>
__device__ __forceinline__ void tc_weights(uint32_t taddr, const float* sv, const float* zc,
                                           RowState& st) {
  uint32_t v[2][16];
  tc::tmem_ld16(taddr, v[0]);
  f2_t l = f2_set(0.f, 0.f), zs = f2_set(0.f, 0.f);   // this tile's, then added: long sums stay exact
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    tc::tmem_wait_ld();
    if (c < 3) tc::tmem_ld16(taddr + 16 * (c + 1), v[(c + 1) & 1]);
    const uint32_t(&x)[16] = v[c & 1];
    uint32_t w[16];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float4 s = reinterpret_cast<const float4*>(sv)[4 * c + q];
      float4 z = reinterpret_cast<const float4*>(zc)[4 * c + q];
      if constexpr (SELECT) {
        constexpr uint32_t kHidden = 0xFF800000u;   // -inf
        if (x[4 * q] == kHidden) s.x = z.x = 0.f;
        if (x[4 * q + 1] == kHidden) s.y = z.y = 0.f;
        if (x[4 * q + 2] == kHidden) s.z = z.z = 0.f;
        if (x[4 * q + 3] == kHidden) s.w = z.w = 0.f;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const f2_t p = f2_set(ex2(__uint_as_float(x[4 * q + 2 * e])),
                              ex2(__uint_as_float(x[4 * q + 2 * e + 1])));
        l = f2_add(l, p);
        zs = f2_fma(p, e ? f2_set(z.z, z.w) : f2_set(z.x, z.y), zs);
        const f2_t y2 = f2_mul(p, e ? f2_set(s.z, s.w) : f2_set(s.x, s.y));
        const float2 y = f2_unpack(y2);
        const __half2 hi = __floats2half2_rn(y.x, y.y);
        w[2 * q + e] = *reinterpret_cast<const uint32_t*>(&hi);
        const float2 back = __half22float2(hi);
        const float2 d = f2_unpack(f2_sub(y2, f2_set(back.x, back.y)));
        const __half2 lo = __floats2half2_rn(d.x, d.y);
        w[8 + 2 * q + e] = *reinterpret_cast<const uint32_t*>(&lo);
      }
    }
    tmem_st8(taddr + 16 * c, w);
    tmem_st8(taddr + 16 * c + 8, w + 8);
  }
  st.l = f2_add(st.l, l);
  st.zs = f2_add(st.zs, zs);
}

template <class T, int HD>
__global__ void __launch_bounds__(kTcThreads, 1) attn_tc_kernel(const TcArgs args) {
  constexpr int L = sizeof(T) == 4 ? 2 : 1;      // fp16 limbs of q (the weights have two)
  constexpr int TB = tc_tile_bytes<HD>();
  constexpr int RB = tc_raw_bytes<HD>();
  constexpr int BLK = kTcKeys * 128;             // bytes of 64 dimensions of a tile
  constexpr int kFlush = tc_flush<L>();
  constexpr float kNegInf = -INFINITY;
  const AttnArgs& a = args.a;
  extern __shared__ __align__(128) uint8_t tc_raw[];
  // pointer arithmetic, not integer rounding, keeps these shared-memory accesses
  uint8_t* tiles = tc_raw + ((1024u - (smem_u32(tc_raw) & 1023u)) & 1023u);
  uint8_t* raws = tiles + 4 * TB;                // K stages, V stages, packed stages
  TcShared& sh = *reinterpret_cast<TcShared*>(raws + kTcRaw * RB);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  pdl_wait();
  // ---- which item: tiles of `per` query rows of every handled request ---------
  const int per = kTcRows / a.group;
  const int cap = static_cast<int>(a.width << a.shift);
  const int chunk = (a.B + 127) / 128;
  auto tiles_of = [&](int64_t b) -> int {        // n <= 2^30 rows
    int64_t r0;
    return (static_cast<int>(rows_of(a, b, &r0)) + per - 1) / per;
  };
  int64_t len0 = 0;                              // of the thread's first request
  if (tid < 128) {
    int64_t mine = 0;
    if (static_cast<int64_t>(tid) * chunk < a.B) len0 = a.lens[static_cast<int64_t>(tid) * chunk];
    for (int k = 0; k < chunk; ++k) {
      const int64_t b = static_cast<int64_t>(tid) * chunk + k;
      if (b < a.B) mine += tiles_of(b);
    }
    sh.scan[tid] = mine;
  }
  if (tid == 0) {
    sh.item[0] = sh.place = -1;
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&sh.k_full[s]), kTcConverters);
      mbar_init(smem_u32(&sh.v_full[s]), kTcConverters);
      mbar_init(smem_u32(&sh.s_full[s]), 1);
      mbar_init(smem_u32(&sh.p_full[s]), 256);
      for (int w = 0; w < 4; ++w) {
        mbar_init(smem_u32(&sh.t_full[s][w]), 2);
        mbar_init(smem_u32(&sh.m_full[s][w]), 1);
      }
      mbar_init(smem_u32(&sh.v_empty[s]), 1);
    }
    for (int s = 0; s < kTcRing; ++s) mbar_init(smem_u32(&sh.par_full[s]), 32);
    for (int s = 0; s < kTcRaw; ++s) {
      mbar_init(smem_u32(&sh.raw_full[s]), 1);
      mbar_init(smem_u32(&sh.raw_empty[s]), kTcConverters + 32);
    }
    mbar_init(smem_u32(&sh.q_ready), kTcSoftmax);
    mbar_init(smem_u32(&sh.drain), 1);
    mbar_init(smem_u32(&sh.o_free), 256);
    fence_mbar_init();
  }
  __syncthreads();
  if (tid == kTcThreads - 32) sh.place = take_place(args.taken, args.slots);
  if (warp == 22) {
    tc::tmem_alloc(smem_u32(&sh.tmem), 512);
    tc::tmem_relinquish();
    tc::tc_fence_before();
  }
  if (tid < 128) {
    int64_t before = 0, total = 0;
    for (int k = 0; k * chunk < a.B; ++k) {
      const int64_t v = sh.scan[k];
      before += k < tid ? v : 0;
      total += v;
    }
    // a request's later tiles see more: they start first
    const int64_t t = total - 1 - blockIdx.x / a.nkv;
    if (t >= 0 && t >= before && t < before + sh.scan[tid]) {
      int64_t b = static_cast<int64_t>(tid) * chunk, at = before;
      for (int n = tiles_of(b); t >= at + n; n = tiles_of(b)) {
        at += n;
        ++b;
      }
      int64_t r0;
      const int64_t n = rows_of(a, b, &r0), row0 = (t - at) * per, lim = int64_t(1) << 30;
      const int64_t len = b == static_cast<int64_t>(tid) * chunk ? len0 : a.lens[b];
      const int64_t off = len - n, last = (row0 + per < n ? row0 + per : n) + off;
      sh.item[0] = static_cast<int>(b);
      sh.item[1] = static_cast<int>(row0);
      sh.item[2] = static_cast<int>(n);
      sh.item[3] = static_cast<int>(r0);
      // rows and positions are at most 2^30, so more than that changes no limit
      sh.item[4] = static_cast<int>(off > lim ? lim : (off < -lim ? -lim : off));
      sh.item[5] = static_cast<int>(last < 0 ? 0 : (last > cap ? cap : last));
    }
  }
  __syncthreads();
  tc::tc_fence_after();
  if (sh.item[0] < 0) {                    // the grid is an upper bound
    if (warp == 22) tc::tmem_dealloc(*const_cast<volatile uint32_t*>(&sh.tmem), 512);
    if (tid == kTcThreads - 32) leave_place(args.taken, sh.place);
    return;
  }
  // (each role reads these for itself: kept from here on, they would spill)
  auto tmem_base = [&]() -> uint32_t { return *const_cast<volatile uint32_t*>(&sh.tmem); };
  auto item = [&](int k) -> int { return *const_cast<volatile int*>(&sh.item[k]); };
  auto seen_by = [&]() -> int { return item(5); };
  auto nt_of = [&]() -> int { return (seen_by() + kTcKeys - 1) / kTcKeys; };   // tiles of the item
  if (warp < 16) {
    // ======================= softmax =======================================
    regs_more<88>();
    // row r of the item; quarter: which TMEM lanes; odd / half: which tiles and positions
    const int r = tid & 127, quarter = warp & 3, odd = (warp >> 2) & 1, half = warp >> 3;
    const int part = warp >> 2;               // this thread's share of the row's dimensions
    const uint32_t lane_addr = tmem_base() + (static_cast<uint32_t>(32 * quarter) << 16);
    const int nt = nt_of(), h = blockIdx.x % a.nkv;
    // r / group for r < 128: the error of the rounded-up reciprocal, 128 / 65536,
    // is below 1 / group
    const uint32_t inv_group = (65535u + a.group) / a.group;
    const int rg = static_cast<int>((r * inv_group) >> 16);
    const int row0 = item(1), n = item(2);
    const int64_t r0 = item(3);
    const int row = row0 + rg, head = h * a.group + (r - rg * a.group);
    const bool real = r < per * a.group && row < n;
    const int sees = sh.item[4] + row + 1;          // positions [0, lim) are seen
    const int lim = !real || sees < 0 ? 0 : (sees > cap ? cap : sees);
    constexpr int DP = HD / 4;                      // dimensions per thread

    // ---- q: this thread's share of the row, as fp16 limbs in TMEM --------------
    float F, Qs;
    {
      float x[DP];
      if (a.vec) {
        // through the second K and V stages (the converters leave them alone
        // until q_ready): whole rows per warp, 16-byte chunk c of row r at c ^ (r & 7)
        constexpr int CH = HD * static_cast<int>(sizeof(T)) / 16;
        auto at = [&](int rr, int c) -> uint4* {
          return reinterpret_cast<uint4*>(tiles + (rr < 64 ? TB : 3 * TB) + (rr & 63) * (CH * 16) +
                                          ((c ^ (rr & 7)) << 4));
        };
        // all loads before the first store; rows that are not real read the item's last
        // (a load under a condition would wait for the one before it)
        uint4 u[CH / 4];
#pragma unroll
        for (int i = 0; i < CH / 4; ++i) {
          const int idx = i * kTcSoftmax + tid, rr = idx / CH, c = idx % CH;
          const int g = static_cast<int>((rr * inv_group) >> 16), gr = row0 + g < n ? g : n - 1 - row0;
          u[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (r0 + row0 + gr) * a.q_rs +
                                                      (h * a.group + (rr - g * a.group)) * a.q_hs) + c);
        }
#pragma unroll
        for (int i = 0; i < CH / 4; ++i) {
          const int idx = i * kTcSoftmax + tid, rr = idx / CH, c = idx % CH;
          const int g = static_cast<int>((rr * inv_group) >> 16);
          *at(rr, c) = rr < per * a.group && row0 + g < n ? u[i] : make_uint4(0u, 0u, 0u, 0u);
        }
        named_bar_sync(6, kTcSoftmax);
        constexpr int pv = 16 / sizeof(T);
#pragma unroll
        for (int j = 0; j < CH / 4; ++j) {
          const uint4 u = *at(r, part * (CH / 4) + j);
          const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
          for (int k = 0; k < pv; ++k) x[j * pv + k] = to_f(e[k]);
        }
      } else if (real) {
        load_row(static_cast<const T*>(a.q) + (r0 + row) * a.q_rs + head * a.q_hs + part * DP, false,
                 x);
      } else {
#pragma unroll
        for (int j = 0; j < DP; ++j) x[j] = 0.f;
      }
      float m4[4] = {0.f, 0.f, 0.f, 0.f}, s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < DP; ++j) {
        m4[j & 3] = fmaxf(m4[j & 3], fabsf(x[j]));
        s4[j & 3] += x[j];
      }
      float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
      float sum = (s4[0] + s4[1]) + (s4[2] + s4[3]);
      sh.ex_q[0][part][r] = mx;
      sh.ex_q[1][part][r] = sum;
      named_bar_sync(1 + quarter, 128);
      mx = fmaxf(fmaxf(sh.ex_q[0][0][r], sh.ex_q[0][1][r]), fmaxf(sh.ex_q[0][2][r], sh.ex_q[0][3][r]));
      sum = (sh.ex_q[1][0][r] + sh.ex_q[1][1][r]) + (sh.ex_q[1][2][r] + sh.ex_q[1][3][r]);
      int e = static_cast<int>((__float_as_uint(mx) >> 23) & 255u) - 127;
      e = e < -112 ? -112 : (e > 117 ? 117 : e);
      const float up = pow2i(14 - e);
      F = pow2i(e + (L == 2 ? -14 : 10)) * a.scale;
      Qs = sum * a.scale;
      // pairs (0 4) (1 5) (2 6) (3 7) of each eight, as K's codes lie (subnormal odd
      // nibbles are 16 c)
      const float up_odd = L == 2 ? up : up * 0.0625f;
#pragma unroll
      for (int m = 0; m < DP / 8; m += 2) {
        uint32_t w[L][8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int at = 8 * (m + (k >> 2)) + (k & 3);
          const f2_t y2 = f2_mul(f2_set(x[at], x[at + 4]), k & 1 ? f2_set(up_odd, up_odd) : f2_set(up, up));
          const float2 y = f2_unpack(y2);
          const __half2 hi = __floats2half2_rn(y.x, y.y);
          w[0][k] = *reinterpret_cast<const uint32_t*>(&hi);
          if constexpr (L == 2) {
            const float2 back = __half22float2(hi);
            const float2 d = f2_unpack(f2_sub(y2, f2_set(back.x, back.y)));
            const __half2 lo = __floats2half2_rn(d.x, d.y);
            w[L - 1][k] = *reinterpret_cast<const uint32_t*>(&lo);
          }
        }
#pragma unroll
        for (int l = 0; l < L; ++l)
          tmem_st8(lane_addr + kColQ + l * (HD / 2) + part * (DP / 2) + 4 * m, w[l]);
      }
      tmem_wait_st();
      tc::tc_fence_before();
      mbar_arrive(smem_u32(&sh.q_ready));
    }

    const f2_t F2 = f2_set(F, F), Q2 = f2_set(Qs, Qs);
    RowState st{kNegInf, f2_set(0.f, 0.f), f2_set(0.f, 0.f)};
    bool failed = false;
#pragma unroll 1
    for (int j = odd; j < nt; j += 2) {
      const int ring = j & (kTcRing - 1), p0 = j * kTcKeys + half * 64;
      bool ok = mbar_wait(smem_u32(&sh.par_full[ring]), (j / kTcRing) & 1) &&
                mbar_wait(smem_u32(&sh.s_full[odd]), (j >> 1) & 1);
      // the row's maximum up to tile j - 1
      if (j > 0) ok = ok && mbar_wait(smem_u32(&sh.m_full[odd ^ 1][quarter]), ((j - 1) >> 1) & 1);
      failed = !__all_sync(0xffffffffu, ok);
      if (failed) break;
      tc::tc_fence_after();
      const float before = j > 0 ? sh.max[odd ^ 1][r] : kNegInf;
      const uint32_t cols = lane_addr + kColS + odd * 128 + half * 64;
      const float mu = before == kNegInf ? 0.f : -before;
      const uint2 vb = *reinterpret_cast<const uint2*>(&sh.valid[ring][2 * half]);
      const bool whole = (vb.x & vb.y) == 0xFFFFFFFFu && __all_sync(0xffffffffu, lim >= p0 + 64);
      const f2_t mu2 = f2_set(mu, mu);
      const float* sk = sh.sk[ring] + half * 64;
      const float* zk = sh.zk[ring] + half * 64;
      float top = whole ? tc_scores<false>(cols, sk, zk, F2, Q2, mu2, nullptr, 0)
                        : tc_scores<true>(cols, sk, zk, F2, Q2, mu2, &sh.valid[ring][2 * half], lim - p0);
      const bool wide = sh.wide[ring] != 0u;
      float topu = kNegInf, peak = kNegInf;
      if (wide) {
        topu = tc_top_u(cols, sh.lu[ring] + half * 64);
        if (before != kNegInf) {
          // Of the tiles before: what was agreed on, or, when those were not wide, p in
          // [1, 2^4] and u of 2^-kTcSpare of the largest at least.
          const bool was = j > 0 && sh.wide[(j - 1) & (kTcRing - 1)] != 0u;
          peak = was ? sh.peak[odd ^ 1][r] : 4.f;
          topu = fmaxf(topu, (was ? sh.peaku[odd ^ 1][r] : 10.f - kTcSpare) + __log2f(sh.down[ring]));
        }
        sh.topu[odd][half][r] = topu;
      }
      // both halves' maximum; the arrays it takes are free again once O(j) is issued
      sh.top[odd][half][r] = top;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.t_full[odd][quarter]));
      failed = !warp_wait(&sh.t_full[odd][quarter], (j >> 1) & 1);
      if (failed) break;
      top = fmaxf(top, sh.top[odd][half ^ 1][r]);
      // a maximum that rose by more than 2^4 is renewed (x stands relative to -mu)
      float now = before;
      if (wide) {
        topu = fmaxf(topu, sh.topu[odd][half ^ 1][r]);
        peak = fmaxf(peak, top);
        // by how much the reference moves: p u 2^(10 - ev) of 2^10 to 2^11 where it has left
        // [2^2, 2^14], and no p above 2^90
        float d = 0.f;
        if (topu == kNegInf)
          d = before == kNegInf || top > 4.f ? top : 0.f;
        else if (before == kNegInf || topu > 14.f || topu < 2.f)
          d = floorf(topu) - 10.f;
        d = fmaxf(d, peak - 90.f);
        now = (before == kNegInf ? 0.f : before) + d;
        if (half == 0) {
          sh.peak[odd][r] = peak - d;
          sh.peaku[odd][r] = topu - d;
        }
      } else if (top > (before == kNegInf ? kNegInf : 4.f)) {
        now = fmaxf(before, top - mu);
      }
      if (half == 0) {
        sh.max[odd][r] = now;
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.m_full[odd][quarter]));
      }
      const float down = sh.down[ring];
      if (__any_sync(0xffffffffu, now != before || down != 1.f)) {
        tc_rescale<64>(cols, 1.f, now == kNegInf ? 0.f : -mu - now);
        if (j % kFlush) {
          // O holds tiles up to j - 1 relative to `before`, V's steps to the old exponent
          const bool done = warp_wait(&sh.v_empty[odd ^ 1], ((j - 1) >> 1) & 1);
          if (!done && lane == 0) report_error(ERR_WAIT_FULL, 0x401u);
          tc::tc_fence_after();
          tc_rescale<HD / 2>(lane_addr + kColO + half * (HD / 2),
                             (before == kNegInf ? 1.f : ex2(before - now)) * down, 0.f);
        }
      }
      if (__any_sync(0xffffffffu, now != st.m)) {        // this thread's own sums
        const float al = st.m == kNegInf ? 1.f : ex2(st.m - now);
        st.m = now;
        st.l = f2_mul(st.l, f2_set(al, al));
        st.zs = f2_mul(st.zs, f2_set(al, al));
      }
      // weights, over this thread's columns of S
      const float* sv = sh.sv[ring] + half * 64;
      const float* zc = sh.zc[ring] + half * 64;
      if (sh.odd[ring])
        tc_weights<true>(cols, sv, zc, st);
      else
        tc_weights<false>(cols, sv, zc, st);
      tmem_wait_st();
      tc::tc_fence_before();
      mbar_arrive(smem_u32(&sh.p_full[odd]));
      if (j % kFlush == kFlush - 1 && j + 1 < nt) {
        // O to the sums, this thread's half of the row; the next tile starts it anew
        const bool first = j < kFlush;
        const float wd = sh.w_down[ring];
        failed = sh.place < 0;
        if (failed) break;
        float4* const mine = sums_of<HD>(args, sh.place) + half * (HD / 8) * kTcRows + r;
        float4 t[4];
        auto fetch = [&](int c) {                 // sums of 16 columns, ahead of their use
#pragma unroll
          for (int k = 0; k < 4; ++k)
            t[k] = first ? make_float4(0.f, 0.f, 0.f, 0.f) : __ldcg(mine + (4 * c + k) * kTcRows);
        };
        fetch(0);
        float al = 1.f;                           // from the sums' terms to O's
        if (!first) {
          const float fl = sh.flushed[half][r], fw = sh.flushed_w[half][r];
          if (fl != now && fl != kNegInf) al = ex2(fl - now);
          if (fw != wd) al *= fw / wd;
        }
        sh.flushed[half][r] = now;
        sh.flushed_w[half][r] = wd;
        failed = !warp_wait(&sh.v_empty[odd], (j >> 1) & 1);
        if (failed) break;
        tc::tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[16];
          tc::tmem_ld16(lane_addr + kColO + half * (HD / 2) + 16 * c, o);
          tc::tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float4 s = t[k];
            __stcg(mine + (4 * c + k) * kTcRows,
                   make_float4(fmaf(s.x, al, __uint_as_float(o[4 * k])),
                               fmaf(s.y, al, __uint_as_float(o[4 * k + 1])),
                               fmaf(s.z, al, __uint_as_float(o[4 * k + 2])),
                               fmaf(s.w, al, __uint_as_float(o[4 * k + 3]))));
          }
          if (c + 1 < HD / 32) fetch(c + 1);
        }
        tc::tc_fence_before();
        mbar_arrive(smem_u32(&sh.o_free));
      }
    }
    if (failed && lane == 0) report_error(ERR_WAIT_FULL, 0x400u);
    // ---- epilogue: the four threads' sums, relative to what the last tile's are -----
    const float2 lt = f2_unpack(st.l), zt = f2_unpack(st.zs);
    sh.ex[0][part][r] = st.m;
    sh.ex[1][part][r] = lt.x + lt.y;
    sh.ex[2][part][r] = zt.x + zt.y;
    named_bar_sync(1 + quarter, 128);
    // (parts 0 and 2 had the even tiles, 1 and 3 the odd ones)
    const float mf = sh.ex[0][(nt - 1) & 1][r];
    float l = 0.f, zs = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float m = sh.ex[0][k][r], al = m == kNegInf ? 1.f : ex2(m - mf);
      l = fmaf(sh.ex[1][k][r], al, l);
      zs = fmaf(sh.ex[2][k][r], al, zs);
    }
    // the sums of this thread's columns, ahead of the last tile's MMAs
    const bool summed = nt > kFlush && !failed && sh.place >= 0;
    float4 t[DP / 4];
#pragma unroll
    for (int k = 0; k < DP / 4; ++k)
      t[k] = summed ? __ldcg(sums_of<HD>(args, sh.place) + (part * DP / 4 + k) * kTcRows + r)
                    : make_float4(0.f, 0.f, 0.f, 0.f);
    bool ok = !failed;
    if (nt > 0 && ok) ok = mbar_wait(smem_u32(&sh.v_empty[(nt - 1) & 1]), ((nt - 1) >> 1) & 1);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok && lane == 0) report_error(ERR_WAIT_FULL, 0x402u);
    tc::tc_fence_after();
    const float wd = nt > 0 ? sh.w_down[(nt - 1) & (kTcRing - 1)] : 0.f;
    constexpr int CH = HD * static_cast<int>(sizeof(T)) / 16, pv = 16 / sizeof(T);
    if (ok) {
      // The tiles are free now: rows of 16-byte chunks (chunk c of row r at
      // c ^ (r & 7)) go through them, so that a warp stores whole rows.
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      const float fl = summed ? sh.flushed[0][r] : kNegInf, as = fl == kNegInf ? 1.f : ex2(fl - mf);
      const float asw = summed ? as * sh.flushed_w[0][r] : 0.f;
#pragma unroll
      for (int c = 0; c < DP; c += 16) {
        uint32_t u[16];
        if (nt > 0) {
          tc::tmem_ld16(lane_addr + kColO + part * DP + c, u);
          tc::tmem_wait_ld();
        }
#pragma unroll
        for (int k8 = 0; k8 < 16; k8 += 8) {
          T y[8];
#pragma unroll
          for (int k4 = 0; k4 < 8; k4 += 4) {
            const float4 t4 = t[(c + k8 + k4) / 4];
            const float e[4] = {t4.x, t4.y, t4.z, t4.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              // column 8 w + k holds dimension 8 w + (k / 2) + (k odd ? 4 : 0)
              const int col = k4 + k, d = (col >> 1) + ((col & 1) << 2);
              y[d] = from_f<T>(nt > 0 ? fmaf(__uint_as_float(u[k8 + col]), wd, fmaf(e[k], asw, zs)) * inv : 0.f);
            }
          }
          if (args.out_vec) {
#pragma unroll
            for (int k = 0; k < 8 / pv; ++k) {
              const int ch = (part * DP + c + k8) / pv + k;
              *reinterpret_cast<uint4*>(tiles + r * (CH * 16) + ((ch ^ (r & 7)) << 4)) =
                  *reinterpret_cast<const uint4*>(y + k * pv);
            }
          } else if (r < per * a.group && item(1) + rg < item(2)) {
            T* o = static_cast<T*>(a.out) + (static_cast<int64_t>(item(3)) + item(1) + rg) * a.o_rs +
                   (h * a.group + (r - rg * a.group)) * a.o_hs + part * DP + c + k8;
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] = y[k];
          }
        }
      }
    }
    // every softmax warp comes here, whatever happened
    if (!bar_any(6, kTcSoftmax, !ok) && args.out_vec) {
      const int first = item(1), rows = item(2);
      const int64_t base = item(3);
#pragma unroll 4
      for (int i = 0; i < CH / 4; ++i) {
        const int idx = i * kTcSoftmax + tid, rr = idx / CH, c = idx % CH;
        const int g = static_cast<int>((rr * inv_group) >> 16);
        if (rr < per * a.group && first + g < rows)
          *(reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (base + first + g) * a.o_rs +
                                     (h * a.group + (rr - g * a.group)) * a.o_hs) + c) =
              *reinterpret_cast<const uint4*>(tiles + rr * (CH * 16) + ((c ^ (rr & 7)) << 4));
      }
    }
  } else if (warp < 20) {
    // ======================= converters ====================================
    regs_less<72>();
    const int nt = nt_of();
    // 16-byte chunks of code rows, LPR per row; a thread has the same chunk of
    // every RPI-th row, so its addresses are fixed. The eight threads of one
    // store phase hold two rows (hd 128) and four chunks of each; taking the
    // last two chunks' words in the order 2 3 0 1 keeps their sixteen-byte
    // columns apart.
    const int dt = tid - kTcSoftmax;
    constexpr int LPR = HD / 32, RPI = kTcConverters / LPR, NI = kTcKeys / RPI;
    const int s7 = a.shift < 7 ? a.shift : 7, cnt = 1 << s7;   // positions per packed block
    const int rr = dt / LPR, ci = dt % LPR;
    const bool swap = LPR == 4 && (ci & 2);
    uint32_t src[NI], dst[4];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int p = rr + i * RPI;
      src[i] = (p >> s7) * (cnt * (HD + 8)) + (p & (cnt - 1)) * (HD / 2) + ci * 16;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = ci * 4 + (swap ? k ^ 2 : k);       // word of the row
      dst[k] = (c >> 3) * BLK + rr * 128 + (((c & 7) ^ (rr & 7)) << 4);
    }
    auto put = [&](uint8_t* tile, const uint8_t* codes, uint32_t groups, auto pairs) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        uint4 c4 = *reinterpret_cast<const uint4*>(codes + src[i]);
        if (!((groups >> ((rr + i * RPI) >> 4)) & 1u)) c4 = make_uint4(0u, 0u, 0u, 0u);   // never copied
        const uint32_t w[4] = {swap ? c4.z : c4.x, swap ? c4.w : c4.y, swap ? c4.x : c4.z,
                               swap ? c4.y : c4.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<uint4*>(tile + dst[k] + i * (RPI * 128)) = pairs(w[k]);
      }
      fence_async_smem();
    };
#pragma unroll 1
    for (int j = 0; j < nt; ++j) {
      const int buf = j & 1, st = j % kTcRaw;
      if (!mbar_wait(smem_u32(&sh.raw_full[st]), (j / kTcRaw) & 1)) {
        report_error(ERR_WAIT_FULL, 0x413u);
        break;
      }
      const uint8_t* raw = raws + st * RB;
      const uint32_t groups = sh.raw_groups[st];
      // q goes through the second stages
      if (j == 1 && !mbar_wait(smem_u32(&sh.q_ready), 0)) {
        report_error(ERR_WAIT_FULL, 0x415u);
        break;
      }
      // K's stage is free once S(j - 2) is done, V's once O(j - 2) is
      if (j >= 2 && !mbar_wait(smem_u32(&sh.s_full[buf]), ((j >> 1) - 1) & 1)) {
        report_error(ERR_WAIT_EMPTY, 0x410u);
        break;
      }
      put(tiles + buf * TB, raw, groups, [](uint32_t w) { return pairs_of<L == 1>(w); });
      mbar_arrive(smem_u32(&sh.k_full[buf]));
      if (j >= 2 && !mbar_wait(smem_u32(&sh.v_empty[buf]), ((j >> 1) - 1) & 1)) {
        report_error(ERR_WAIT_EMPTY, 0x411u);
        break;
      }
      put(tiles + (2 + buf) * TB, raw + cnt * (HD / 2), groups, [](uint32_t w) { return pairs_of<false>(w); });
      mbar_arrive(smem_u32(&sh.v_full[buf]));
      mbar_arrive(smem_u32(&sh.raw_empty[st]));
    }
  } else {
  regs_less<56>();
  if (warp == 20) {
    // ======================= parameters ====================================
    // weights are p * s_v * 2^(10 - ev), ev the largest exponent of u so far
    const int s7 = a.shift < 7 ? a.shift : 7, cnt = 1 << s7;
    const int seen = seen_by(), nt = (seen + kTcKeys - 1) / kTcKeys;
    int ev = -100, least = 127;              // the largest and the smallest exponent of u
#pragma unroll 1
    for (int j = 0; j < nt; ++j) {
      const int ring = j & (kTcRing - 1), st = j % kTcRaw;
      if (!warp_wait(&sh.raw_full[st], (j / kTcRaw) & 1)) {
        if (lane == 0) report_error(ERR_WAIT_FULL, 0x416u);
        break;
      }
      const uint32_t groups = sh.raw_groups[st];
      uint32_t kp[4], vp[4];
      float mx = 0.f, mn = INFINITY, u[4];
      bool odd = false;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int p = lane + 32 * k;
        const bool here = j * kTcKeys + p < seen && ((groups >> (p >> 4)) & 1u);
        kp[k] = vp[k] = 0u;                    // positions that do not exist: s = z = 0
        if (here) {
          const uint8_t* q = raws + st * RB + (p >> s7) * (cnt * (HD + 8)) + cnt * HD + (p & (cnt - 1)) * 4;
          kp[k] = *reinterpret_cast<const uint32_t*>(q);
          vp[k] = *reinterpret_cast<const uint32_t*>(q + cnt * 4);
        }
        const uint32_t bits = __ballot_sync(0xffffffffu, here);
        if (lane == 0) sh.valid[ring][k] = bits;
        u[k] = fmaxf(par_s(vp[k]), 0.125f * fabsf(fmaf(8.f, par_s(vp[k]), par_z(vp[k]))));
        mx = fmaxf(mx, u[k]);
        mn = here ? fminf(mn, u[k]) : mn;
        odd = odd || !isfinite(par_s(vp[k])) || !isfinite(par_z(vp[k]));
      }
      mbar_arrive(smem_u32(&sh.raw_empty[st]));
      const int e = exponent(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mx))));
      const int f = exponent(__uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(mn))));
      const int ev_old = ev;
      ev = min(max(e, ev), 127);
      least = min(least, max(f, -100));
      const float up = pow2i(10 - ev);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int p = lane + 32 * k;
        const float sv = par_s(vp[k]);
        sh.sk[ring][p] = par_s(kp[k]);
        sh.zk[ring][p] = L == 2 ? fmaf(8.f, par_s(kp[k]), par_z(kp[k])) : par_z(kp[k]);
        sh.sv[ring][p] = sv * up;
        sh.zc[ring][p] = fmaf(8.f, sv, par_z(vp[k]));
        sh.lu[ring][p] = __log2f(u[k]) + (10.f - ev);
      }
      odd = __any_sync(0xffffffffu, odd);
      if (lane == 0) {
        sh.odd[ring] = odd ? 1u : 0u;
        sh.down[ring] = j == 0 ? 1.f : (ev_old - ev < -126 ? 0.f : pow2i(ev_old - ev));
        sh.w_down[ring] = pow2i(ev - 10);
        sh.wide[ring] = ev - least > kTcSpare ? 1u : 0u;
      }
      mbar_arrive(smem_u32(&sh.par_full[ring]));
    }
  } else if (warp == 21) {
    // ======================= loader ========================================
    // lane = page of the tile (its whole block), or, for pages of more than a
    // tile, one of the four parts of 128 of its positions
    const int64_t ps = int64_t(1) << a.shift;
    const int32_t* tab = a.table + static_cast<int64_t>(sh.item[0]) * a.width;
    const bool parts = a.shift > 7;
    const int seen = seen_by(), nt = (seen + kTcKeys - 1) / kTcKeys, h = blockIdx.x % a.nkv;
    const int cnt = parts ? kTcKeys : 1 << a.shift, copies = parts ? 4 : kTcKeys >> a.shift;
    const int pg = parts ? 0 : lane;
    const uint32_t bytes = parts ? (lane < 2 ? kTcKeys * (HD / 2) : kTcKeys * 4) : cnt * (HD + 8);
    auto page_of = [&](int j) -> int {
      const int p = j * kTcKeys + pg * cnt;
      return lane < copies && p < seen ? __ldg(tab + (p >> a.shift)) : -1;
    };
    int page = page_of(0), j = 0;
#pragma unroll 1
    for (; j < nt; ++j) {
      const int st = j % kTcRaw;
      if (j >= kTcRaw && !warp_wait(&sh.raw_empty[st], ((j / kTcRaw) - 1) & 1)) {
        if (lane == 0) report_error(ERR_WAIT_EMPTY, 0x412u);
        break;
      }
      const bool have = page >= 0 && page < a.pages;
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
        const uint8_t* from = a.pool + (static_cast<int64_t>(page) * a.nkv + h) * (ps * (HD + 8));
        uint32_t to = smem_u32(raws + st * RB);
        if (parts) {
          const int64_t off = (j * kTcKeys) & (ps - 1);
          from += lane < 2 ? lane * (ps * (HD / 2)) + off * (HD / 2)
                           : ps * HD + (lane - 2) * (ps * 4) + off * 4;
          to += lane < 2 ? lane * (kTcKeys * (HD / 2)) : kTcKeys * HD + (lane - 2) * (kTcKeys * 4);
        } else {
          to += pg * bytes;
        }
        bulk_copy(to, from, bytes, bar);
      }
      page = page_of(j + 1);
    }
    // no copy stays in flight into memory that is given up
    for (int t = j > kTcRaw ? j - kTcRaw : 0; t < j; ++t)
      if (!warp_wait(&sh.raw_full[t % kTcRaw], (t / kTcRaw) & 1)) {
        if (lane == 0) report_error(ERR_DRAIN, 0x414u);
        break;
      }
  } else if (warp == 22 && seen_by() > 0) {
    // ======================= MMA issuer ====================================
    const int nt = nt_of();
    const uint32_t tmem = tmem_base();
    constexpr uint32_t id_s = idesc_f16(kTcKeys, false), id_o = idesc_f16(HD, true);
    const bool leader = elect_one();
    const uint64_t kdesc = tc::smem_desc_sw128(smem_u32(tiles));
    const uint64_t vdesc = smem_desc_mn(smem_u32(tiles + 2 * TB), BLK);
    auto scores = [&](int j) {
      const uint64_t kd = kdesc + (j & 1) * (TB >> 4);
      const uint32_t d = tmem + kColS + (j & 1) * 128;
      if (leader) {
#pragma unroll
        for (int l = L - 1; l >= 0; --l)       // low limbs first: what they truncate is small
#pragma unroll
          for (int s = 0; s < HD / 16; ++s)
            mma_f16_ts(d, tmem + kColQ + l * (HD / 2) + s * 8,
                       kd + (((s >> 2) * BLK + (s & 3) * 32) >> 4), id_s, s != 0 || l != L - 1);
        tc::tc_commit(smem_u32(&sh.s_full[j & 1]));
      }
      __syncwarp();
    };
    bool ok = warp_wait(&sh.q_ready, 0) && warp_wait(&sh.k_full[0], 0);
    tc::tc_fence_after();
    if (ok) scores(0);
#pragma unroll 1
    for (int j = 0; ok && j < nt; ++j) {
      if (j + 1 < nt) {
        // S(j + 1) goes where W(j - 1) was; the MMAs run in the order of issue
        ok = warp_wait(&sh.k_full[(j + 1) & 1], ((j + 1) >> 1) & 1);
        if (!ok) break;
        tc::tc_fence_after();
        scores(j + 1);
      }
      ok = warp_wait(&sh.v_full[j & 1], (j >> 1) & 1) && warp_wait(&sh.p_full[j & 1], (j >> 1) & 1);
      const bool anew = j % kFlush == 0;
      if (anew && j > 0) ok = ok && warp_wait(&sh.o_free, (j / kFlush - 1) & 1);
      if (!ok) break;
      tc::tc_fence_after();
      const uint64_t vd = vdesc + (j & 1) * (TB >> 4);
      const uint32_t w = tmem + kColS + (j & 1) * 128;
      if (leader) {
#pragma unroll
        for (int l = 1; l >= 0; --l)
#pragma unroll
          for (int s = 0; s < kTcKeys / 16; ++s)
            mma_f16_ts(tmem + kColO, w + (s >> 2) * 64 + (s & 3) * 16 + 8 * l,
                       vd + ((s * 2048) >> 4), id_o, !anew || s != 0 || l != 1);
        tc::tc_commit(smem_u32(&sh.v_empty[j & 1]));
      }
      __syncwarp();
    }
    if (!ok && lane == 0) report_error(ERR_WAIT_FULL, 0x420u);
    // TMEM and shared memory are given up only after every issued MMA has finished
    if (leader) tc::tc_commit(smem_u32(&sh.drain));
    __syncwarp();
    if (!warp_wait(&sh.drain, 0) && lane == 0) report_error(ERR_DRAIN, 0x421u);
  }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (tid == kTcThreads - 32) leave_place(args.taken, sh.place);
  if (warp == 22) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem_base(), 512);
  }
}

}  // namespace kv4
}  // namespace qz
