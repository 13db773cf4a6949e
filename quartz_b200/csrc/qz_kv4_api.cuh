// qz_kv4_api.cuh -- C entry points of the paged 4-bit KV cache (the last part of
// qz_api.cu's translation unit): argument checks, variant choice, launches.
#pragma once

#include "qz_kv4.cuh"
#include "qz_kv4_tc.cuh"

namespace {

// Programmatic dependent launch of a kernel that waits for its predecessors
// itself (pdl_wait), optionally as clusters of `cluster` CTAs.
template <class A>
int launch_kv4(void (*fn)(A), int grid, int threads, int smem, cudaStream_t st, const A& args,
               int cluster = 1) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[n].val.programmaticStreamSerializationAllowed = 1;
  ++n;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = static_cast<unsigned>(n);
  QZ_CUDA(cudaLaunchKernelEx(&cfg, fn, args));
  return QZ_OK;
}

// The dynamic shared memory of `fn`, allowed once per device.
template <class F>
int allow_smem_once(F* fn, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  QZ_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = uint64_t(1) << (dev & 63);      // device_info() refuses devices beyond 64
  if (!(done.load(std::memory_order_acquire) & bit)) {
    QZ_CUDA(allow_smem(fn, bytes));
    done.fetch_or(bit, std::memory_order_release);
  }
  return QZ_OK;
}

// log2 of a page size the kernels take (16 .. 256, a power of two), else -1.
int page_shift(int64_t page_size) {
  for (int s = 4; s <= 8; ++s)
    if (page_size == (int64_t(1) << s)) return s;
  return -1;
}

int check_kv4_pool(const void* pool, int64_t pages, int64_t page_size, int nkv, int hd,
                   const std::string& who) {
  if (nkv < 1) return fail(QZ_ERR_INVALID, who + ": n_kv must be >= 1");
  if (hd != 64 && hd != 128) return fail(QZ_ERR_INVALID, who + ": head_dim must be 64 or 128");
  if (page_shift(page_size) < 0)
    return fail(QZ_ERR_INVALID, who + ": page size must be 16, 32, 64, 128 or 256");
  if (pages < 1 || pages > 0x7FFFFFFFll) return fail(QZ_ERR_INVALID, who + ": bad page count");
  if (!pool || !aligned16(pool))
    return fail(QZ_ERR_INVALID, who + ": null or unaligned pool (16 bytes)");
  return QZ_OK;
}

int check_kv4_heads(int nq, int nkv, const std::string& who) {
  if (nq < 1 || nkv < 1 || nq % nkv)
    return fail(QZ_ERR_INVALID, who + ": query heads must be a multiple of kv heads");
  return QZ_OK;
}

int dtype_bytes(int dtype) { return dtype == qz::kv4::kF32 ? 4 : 2; }

// Whether rows of `hd` elements at p + i * rs + j * hs all start on 16 bytes.
bool rows_aligned(const void* p, int64_t rs, int64_t hs, int dtype) {
  const int64_t b = dtype_bytes(dtype);
  return aligned16(p) && (rs * b) % 16 == 0 && (hs * b) % 16 == 0;
}

template <class T>
int launch_append(const DeviceInfo& d, int hd, const qz::kv4::AppendArgs& a, cudaStream_t st) {
  const int per_block = qz::kv4::kAppendThreads / (hd / 16);
  const int64_t want = qz::cdiv(a.n * a.nkv, per_block);
  const int grid = static_cast<int>(std::min<int64_t>(want, int64_t(d.sms) * qz::kv4::kAppendPerSm));
  return hd == 64 ? launch_kv4(qz::kv4::append_kernel<T, 64>, grid, qz::kv4::kAppendThreads, 0, st, a)
                  : launch_kv4(qz::kv4::append_kernel<T, 128>, grid, qz::kv4::kAppendThreads, 0, st, a);
}

// Blocks of 4 queries (row, head) of a kv head per item of the split kernel: one where
// no request has more than 8, else two. 8 kv heads of 128, bf16, one and two blocks:
// 64 x 2048 positions, 8 queries 40.3 and 45.1 us, 16 59.0 and 60.9; 1 x 16384
// positions, 8 queries 21.7 and 21.2, 16 28.5 and 26.7, 32 45.1 and 36.1.
int attn_blocks(int64_t max_rows, int group) { return max_rows * group > 8 ? 2 : 1; }

struct Kv4AttnLayout {
  int grid;
  int64_t part_off, own_off, sums_off, total;
};

// Requests with more rows than this may take the tensor-core kernel, whose items are
// 128 queries of a kv head over the whole context: with 64 of them real the split kernel
// is as fast (64 requests x 2048 positions, fp32: 138 and 140 us; 128 queries: 250 and
// 140). Groups that fit no tile take the split kernel.
constexpr int kTcMinQueries = 64;
int64_t tc_rows(int group) {
  return group > qz::kv4::kTcRows ? 0x7FFFFFFF : std::max(1, kTcMinQueries / group);
}

// ... and do where its items fill half of the GPU at least, as far as the host can tell
// (all rows but one per request, or the most of one request). The split kernel shares out
// positions too: 8 items over 16384 positions take it 112 us, the other 344; 64 items
// over 2048 positions 51 and 72; a tile of the one is 2.3 us an SM, its work in the other
// 30 ns of the whole GPU, so that they meet at 78 items.
int64_t split_rows(const DeviceInfo& d, int64_t B, int64_t n, int64_t max_rows, int group, int nkv) {
  const int64_t rows = std::max(n - B + 1, std::min(n, max_rows));
  return nkv * qz::cdiv(rows * group, qz::kv4::kTcRows) < d.sms / 2 ? 0x7FFFFFFF : tc_rows(group);
}

Kv4AttnLayout kv4_attn_layout(const DeviceInfo& d, int64_t max_rows, int group, int hd, bool wide) {
  const int nb = attn_blocks(max_rows, group);
  Kv4AttnLayout l;
  l.grid = d.sms * qz::kv4::attn_per_sm(hd, nb, wide);
  // the tickets' place is the same for every variant, so that one workspace
  // serves calls of different shapes in turn; what lies behind it keeps nothing
  // (five tickets and one place of `sums` an SM: 148 SMs take 3.5 KB of the head)
  l.part_off = QZ_KV4_WORKSPACE_HEAD;
  l.own_off = l.part_off + qz::cdiv(int64_t(l.grid) * 2 * 4 * nb * (hd + 2) * 4, 256) * 256;
  l.sums_off = l.own_off + (wide ? 0 : int64_t(l.grid) * qz::kv4::kAttnWarps *
                                           qz::kv4::attn_sum_floats(hd, nb) * 32 * 4);
  l.total = l.sums_off + (max_rows > tc_rows(group) ? int64_t(d.sms) * qz::kv4::kTcRows * hd * 4 : 0);
  return l;
}

template <class T, int HD, int NB>
int launch_kv4_attn(const qz::kv4::AttnArgs& a, int grid, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  if (int rc = allow_smem_once(qz::kv4::attn_kernel<T, HD, NB>, qz::kv4::attn_smem<HD, NB>(), done))
    return rc;
  return launch_kv4(qz::kv4::attn_kernel<T, HD, NB>, grid, qz::kv4::kAttnThreads,
                    qz::kv4::attn_smem<HD, NB>(), st, a);
}

template <class T>
int launch_kv4_attn_t(int hd, int nb, const qz::kv4::AttnArgs& a, int grid, cudaStream_t st) {
  if (hd == 64)
    return nb == 1 ? launch_kv4_attn<T, 64, 1>(a, grid, st) : launch_kv4_attn<T, 64, 2>(a, grid, st);
  return nb == 1 ? launch_kv4_attn<T, 128, 1>(a, grid, st) : launch_kv4_attn<T, 128, 2>(a, grid, st);
}

template <class T, int HD>
int launch_kv4_tc(const qz::kv4::TcArgs& a, int64_t grid, cudaStream_t st) {
  constexpr int smem = qz::kv4::tc_smem<HD>();
  static std::atomic<uint64_t> done{0};
  if (int rc = allow_smem_once(qz::kv4::attn_tc_kernel<T, HD>, smem, done)) return rc;
  return launch_kv4(qz::kv4::attn_tc_kernel<T, HD>, static_cast<int>(grid), qz::kv4::kTcThreads,
                    smem, st, a);
}

}  // namespace

extern "C" {

int qz_kv4_plan(const int64_t* lens, const int64_t* new_rows, int64_t B, int32_t* block_table,
                int64_t width, const int32_t* free_pages, int64_t n_free, const int64_t* used,
                int64_t page_size, int64_t rows, int64_t* cu_rows, int64_t* lens_out,
                int64_t* used_out, int64_t* slots, int64_t* positions, void* stream) {
  if (B < 1 || B > qz::kv4::kPlanMaxB)
    return fail(QZ_ERR_INVALID, "qz_kv4_plan: requests must be 1 .. 4096");
  const int shift = page_shift(page_size);
  if (shift < 0)
    return fail(QZ_ERR_INVALID, "qz_kv4_plan: page size must be 16, 32, 64, 128 or 256");
  if (width < 1 || width > (int64_t(1) << 30) / page_size)
    return fail(QZ_ERR_INVALID, "qz_kv4_plan: table width must be 1 .. 2^30 / page size");
  if (n_free < 0 || n_free > 0x7FFFFFFFll || rows < 0 || rows > (int64_t(1) << 30))
    return fail(QZ_ERR_INVALID, "qz_kv4_plan: bad free-page or row count");
  if (!lens || !new_rows || !block_table || (n_free && !free_pages) || !used || !cu_rows ||
      !lens_out || !used_out || (rows && (!slots || !positions)))
    return fail(QZ_ERR_INVALID, "qz_kv4_plan: null pointer");
  DeviceInfo* d = nullptr;
  if (int rc = device_info(&d)) return rc;
  qz::kv4::PlanArgs a{lens, new_rows, block_table, free_pages, used, cu_rows, lens_out, used_out,
                      slots, positions, width, n_free, rows, static_cast<int>(B), shift};
  const int smem = qz::kv4::plan_smem(static_cast<int>(B));
  if (smem > 48 * 1024)
    QZ_CUDA(allow_smem(qz::kv4::plan_kernel, qz::kv4::plan_smem(qz::kv4::kPlanMaxB)));
  // One CTA writes a small plan. A large one is shared out: over a cluster where lengths
  // or the cursor are updated in place, else over as many CTAs as give each thread a row.
  // In place, us for one CTA / a cluster (B x rows each): 64 x 1 6.1 / 6.6, 768 x 1 6.8 / 7.3,
  // 1 x 3048 7.1 / 6.5, 1024 x 1 7.2 / 7.8, 8 x 512 8.8 / 6.8, 4096 x 1 13.4 / 8.7,
  // 1024 x 48 66 / 14.
  const bool large = rows + 4 * B > 4096;
  auto meets = [](const int64_t* p, int64_t n, const int64_t* q, int64_t m) { return p < q + m && q < p + n; };
  const bool in_place = meets(lens_out, B, lens, B) || meets(lens_out, B, new_rows, B) ||
                        meets(lens_out, B, used, 1) || meets(used_out, 1, lens, B) ||
                        meets(used_out, 1, new_rows, B) || meets(used_out, 1, used, 1);
  const int64_t ctas = (rows + qz::kv4::kPlanThreads - 1) / qz::kv4::kPlanThreads;
  const int cluster = large && in_place ? qz::kv4::kPlanCluster : 1;
  const int grid = in_place ? cluster : static_cast<int>(ctas < 1 ? 1 : (ctas > d->sms ? d->sms : ctas));
  return launch_kv4(qz::kv4::plan_kernel, grid, qz::kv4::kPlanThreads, smem,
                    static_cast<cudaStream_t>(stream), a, cluster);
}

int qz_kv4_append(const void* k, const void* v, int dtype, int64_t k_row_stride,
                  int64_t k_head_stride, int64_t v_row_stride, int64_t v_head_stride, int64_t n,
                  int nkv, int hd, uint8_t* pool, int64_t pages, int64_t page_size,
                  const int64_t* slots, void* stream) {
  if (int rc = check_kv4_pool(pool, pages, page_size, nkv, hd, "qz_kv4_append")) return rc;
  if (dtype < 0 || dtype > 2) return fail(QZ_ERR_INVALID, "qz_kv4_append: unknown dtype");
  if (n < 0 || n > (int64_t(1) << 40) / nkv) return fail(QZ_ERR_INVALID, "qz_kv4_append: bad row count");
  if (n == 0) return QZ_OK;
  if (!k || !v || !slots) return fail(QZ_ERR_INVALID, "qz_kv4_append: null pointer");
  DeviceInfo* d = nullptr;
  if (int rc = device_info(&d)) return rc;
  qz::kv4::AppendArgs a{k, v, k_row_stride, k_head_stride, v_row_stride, v_head_stride, pool,
                        slots, n, pages * page_size, nkv, page_shift(page_size), 0};
  a.vec = rows_aligned(k, k_row_stride, k_head_stride, dtype) &&
          rows_aligned(v, v_row_stride, v_head_stride, dtype);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case qz::kv4::kF32: return launch_append<float>(*d, hd, a, st);
    case qz::kv4::kBF16: return launch_append<__nv_bfloat16>(*d, hd, a, st);
    default: return launch_append<__half>(*d, hd, a, st);
  }
}

int qz_kv4_gather(const uint8_t* pool, int64_t pages, int64_t page_size, int nkv, int hd,
                  const int64_t* slots, int64_t n, float* k, float* v, void* stream) {
  if (int rc = check_kv4_pool(pool, pages, page_size, nkv, hd, "qz_kv4_gather")) return rc;
  if (n < 0 || n > (int64_t(1) << 40) / nkv) return fail(QZ_ERR_INVALID, "qz_kv4_gather: bad row count");
  if (n == 0) return QZ_OK;
  if (!k || !v || !slots) return fail(QZ_ERR_INVALID, "qz_kv4_gather: null pointer");
  if (!aligned16(k) || !aligned16(v))
    return fail(QZ_ERR_INVALID, "qz_kv4_gather: k and v must be 16-byte aligned");
  DeviceInfo* d = nullptr;
  if (int rc = device_info(&d)) return rc;
  const qz::kv4::GatherArgs a{pool, slots, k, v, n, pages * page_size, nkv, page_shift(page_size)};
  const int per_block = qz::kv4::kGatherThreads / (hd / 4) * qz::kv4::kGatherFly;
  const int grid = static_cast<int>(
      std::min<int64_t>(qz::cdiv(n * nkv, per_block), int64_t(d->sms) * 8));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return hd == 64 ? launch_kv4(qz::kv4::gather_kernel<64>, grid, qz::kv4::kGatherThreads, 0, st, a)
                  : launch_kv4(qz::kv4::gather_kernel<128>, grid, qz::kv4::kGatherThreads, 0, st, a);
}

int qz_qk_rope_kv4(const float* qkv, const float* q_norm_w, const float* k_norm_w,
                   const float* inv_freq, float* q_out, int64_t M, int nq, int nkv, int hd,
                   const int64_t* positions, uint8_t* pool, int64_t pages, int64_t page_size,
                   const int64_t* slots, float eps, void* stream) {
  if (int rc = check_kv4_heads(nq, nkv, "qz_qk_rope_kv4")) return rc;
  if (int rc = check_kv4_pool(pool, pages, page_size, nkv, hd, "qz_qk_rope_kv4")) return rc;
  if (M < 0 || M > (int64_t(1) << 32) / (nq + 2 * nkv))
    return fail(QZ_ERR_INVALID, "qz_qk_rope_kv4: bad row count");
  if ((q_norm_w == nullptr) != (k_norm_w == nullptr))
    return fail(QZ_ERR_INVALID, "qz_qk_rope_kv4: pass both norm weights or neither");
  if (M == 0) return QZ_OK;
  if (!qkv || !inv_freq || !q_out || !positions || !slots)
    return fail(QZ_ERR_INVALID, "qz_qk_rope_kv4: null pointer");
  DeviceInfo* d = nullptr;
  if (int rc = device_info(&d)) return rc;
  const qz::kv4::RopeArgs a{qkv, q_norm_w, k_norm_w, inv_freq, q_out, pool, positions, slots, M,
                            pages * page_size, nq, nkv, page_shift(page_size), eps};
  const int64_t warps = M * (nq + 2 * nkv);
  const int grid = static_cast<int>(qz::cdiv(warps, qz::kv4::kRopeThreads / 32));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return hd == 64 ? launch_kv4(qz::kv4::qk_rope_kv4_kernel<64>, grid, qz::kv4::kRopeThreads, 0, st, a)
                  : launch_kv4(qz::kv4::qk_rope_kv4_kernel<128>, grid, qz::kv4::kRopeThreads, 0, st, a);
}

int qz_kv4_attention_workspace_bytes(int nq, int nkv, int hd, int64_t max_rows, int64_t* bytes) {
  if (!bytes) return fail(QZ_ERR_INVALID, "qz_kv4_attention_workspace_bytes: null pointer");
  if (int rc = check_kv4_heads(nq, nkv, "qz_kv4_attention_workspace_bytes")) return rc;
  if (hd != 64 && hd != 128)
    return fail(QZ_ERR_INVALID, "qz_kv4_attention_workspace_bytes: head_dim must be 64 or 128");
  if (max_rows < 1)
    return fail(QZ_ERR_INVALID, "qz_kv4_attention_workspace_bytes: max_rows must be >= 1");
  DeviceInfo* d = nullptr;
  if (int rc = device_info(&d)) return rc;
  // (16-bit rows take the larger grid)
  *bytes = kv4_attn_layout(*d, max_rows, nq / nkv, hd, false).total;
  return QZ_OK;
}

int qz_kv4_attention(const void* q, int dtype, int64_t q_row_stride, int64_t q_head_stride,
                     void* out, int64_t out_row_stride, int64_t out_head_stride,
                     const uint8_t* pool, int64_t pages, int64_t page_size,
                     const int32_t* block_table, int64_t width, const int64_t* lens,
                     const int64_t* cu_rows, int64_t B, int64_t n, int64_t max_rows, int nq,
                     int nkv, int hd, float scale, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = check_kv4_heads(nq, nkv, "qz_kv4_attention")) return rc;
  if (int rc = check_kv4_pool(pool, pages, page_size, nkv, hd, "qz_kv4_attention")) return rc;
  if (dtype < 0 || dtype > 2) return fail(QZ_ERR_INVALID, "qz_kv4_attention: unknown dtype");
  if (B < 0 || B > qz::kv4::kAttnMaxB)
    return fail(QZ_ERR_INVALID, "qz_kv4_attention: requests must be 0 .. 4096");
  if (n < 0 || n > (int64_t(1) << 30) / (nq / nkv))
    return fail(QZ_ERR_INVALID, "qz_kv4_attention: bad row count");
  if (width < 1 || width > (int64_t(1) << 30) / page_size)
    return fail(QZ_ERR_INVALID, "qz_kv4_attention: table width must be 1 .. 2^30 / page size");
  if (max_rows < 1 || (!cu_rows && max_rows != 1))
    return fail(QZ_ERR_INVALID, "qz_kv4_attention: max_rows must be >= 1, and 1 without cu_rows");
  if (B == 0 || n == 0) return QZ_OK;
  if (!q || !out || !block_table || !lens || !ws)
    return fail(QZ_ERR_INVALID, "qz_kv4_attention: null pointer");
  DeviceInfo* d = nullptr;
  if (int rc = device_info(&d)) return rc;
  const int group = nq / nkv, nb = attn_blocks(max_rows, group);
  const Kv4AttnLayout L = kv4_attn_layout(*d, max_rows, group, hd, dtype == qz::kv4::kF32);
  if (static_cast<int64_t>(ws_bytes) < L.total || !aligned_to(ws, 256))
    return fail(QZ_ERR_INVALID, "qz_kv4_attention: workspace too small or not 256-byte aligned");
  qz::kv4::AttnArgs a{};
  a.q = q;
  a.out = out;
  a.q_rs = q_row_stride;
  a.q_hs = q_head_stride;
  a.o_rs = out_row_stride;
  a.o_hs = out_head_stride;
  a.pool = pool;
  a.table = block_table;
  a.lens = lens;
  a.cu = cu_rows;
  a.tickets = static_cast<unsigned*>(ws);
  a.part = reinterpret_cast<float*>(static_cast<char*>(ws) + L.part_off);
  a.sums = reinterpret_cast<float*>(static_cast<char*>(ws) + L.own_off);
  a.pages = pages;
  a.width = width;
  a.n = n;
  a.B = static_cast<int>(B);
  a.nkv = nkv;
  a.group = group;
  a.shift = page_shift(page_size);
  a.scale = scale * 1.44269504088896341f;
  a.vec = rows_aligned(q, q_row_stride, q_head_stride, dtype);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t few = split_rows(*d, B, n, max_rows, group, nkv);
  if (few < 0x7FFFFFFF && max_rows > few) {
    qz::kv4::TcArgs t{a, 0, d->sms, reinterpret_cast<float4*>(static_cast<char*>(ws) + L.sums_off),
                        a.tickets + int64_t(d->sms) * qz::kv4::kAttnMaxPerSm};
    t.out_vec = rows_aligned(out, out_row_stride, out_head_stride, dtype);
    t.a.rows_lo = static_cast<int>(few);
    t.a.rows_hi = static_cast<int>(std::min<int64_t>(max_rows, 0x7FFFFFFF));
    const int64_t per = qz::kv4::kTcRows / group;
    const int64_t grid = (n / per + std::min<int64_t>(B, n / (few + 1))) * nkv;
    if (grid > 0x7FFFFFFFll) return fail(QZ_ERR_INVALID, "qz_kv4_attention: too many rows");
    if (grid > 0) {
      int rc;
      if (dtype == qz::kv4::kF32)
        rc = hd == 64 ? launch_kv4_tc<float, 64>(t, grid, st) : launch_kv4_tc<float, 128>(t, grid, st);
      else if (dtype == qz::kv4::kBF16)
        rc = hd == 64 ? launch_kv4_tc<__nv_bfloat16, 64>(t, grid, st)
                      : launch_kv4_tc<__nv_bfloat16, 128>(t, grid, st);
      else
        rc = hd == 64 ? launch_kv4_tc<__half, 64>(t, grid, st) : launch_kv4_tc<__half, 128>(t, grid, st);
      if (rc) return rc;
    }
  }
  a.rows_lo = 0;
  a.rows_hi = static_cast<int>(std::min<int64_t>(max_rows, few));
  switch (dtype) {
    case qz::kv4::kF32: return launch_kv4_attn_t<float>(hd, nb, a, L.grid, st);
    case qz::kv4::kBF16: return launch_kv4_attn_t<__nv_bfloat16>(hd, nb, a, L.grid, st);
    default: return launch_kv4_attn_t<__half>(hd, nb, a, L.grid, st);
  }
}

}  // extern "C"
