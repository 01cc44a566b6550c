// Host entries of the paged key-value cache operators (kernels: paged.cuh).
#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/qdecode.h"
#include "internal.cuh"
#include "overlap.hpp"
#include "paged.cuh"
#include "paged_decode.cuh"
#include "paged_prompt.cuh"

namespace qd {

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static bool known_dtype(int d) { return d == QD_KV_F16 || d == QD_KV_F32 || d == QD_KV_BF16; }

static void need(bool ok, const char* msg) {
  if (!ok) throw QdError{QD_E_INVALID, msg};
}

// (Rows of a ragged batch may be padding that no memory stands behind: the host is sure of the first alone.)
static Rows rows_of(const void* p, int dtype, int64_t rows, int64_t elements, int64_t stride) {
  const int64_t size = dtype == QD_KV_F32 ? 4 : 2;
  return {p, rows, elements * size, stride * size};
}
static void need_apart_from_pools(const qd_paged_kv* kv, const Rows& x, const char* msg) {
  const int64_t bytes = (int64_t)kv->num_pages * kv->kv_heads * kv->page_size * kHeadDim * 2;
  need(apart(x, Rows{kv->k, 1, bytes, bytes}) && apart(x, Rows{kv->v, 1, bytes, bytes}), msg);
}

static PagedArgs check_paged(const qd_paged_kv* kv) {
  need(kv != nullptr, "paged cache: NULL pointer");
  need(kv->dtype == QD_KV_F16 || kv->dtype == QD_KV_BF16, "paged cache: dtype must be QD_KV_F16 or QD_KV_BF16");
  need(kv->head_dim == kHeadDim, "paged cache: head_dim must be 128");
  need(kv->page_size >= 16 && kv->page_size <= 256 && (kv->page_size & (kv->page_size - 1)) == 0,
       "paged cache: page_size must be a power of two from 16 to 256");
  need(kv->kv_heads >= 1 && kv->kv_heads <= 1024, "paged cache: bad kv_heads");
  need(kv->batch >= 0 && kv->batch <= 4096, "paged cache: batch must be 0..4096");
  need(kv->num_pages >= 0 && kv->table_width >= 0 && kv->table_stride >= kv->table_width,
       "paged cache: bad num_pages, table_width or table_stride");
  need((long long)kv->table_width * kv->page_size <= 0x40000000LL, "paged cache: table_width * page_size beyond 2^30");
  need(kv->batch == 0 || (kv->block_table && kv->seq_lens) , "paged cache: NULL block_table or seq_lens");
  need(kv->num_pages == 0 || (kv->k && kv->v), "paged cache: NULL pool");
  need(aligned16(kv->k) && aligned16(kv->v), "paged cache: pools must be 16-byte aligned");
  PagedArgs a{};
  a.k = kv->k;
  a.v = kv->v;
  a.num_pages = kv->num_pages;
  while ((1 << a.page_shift) < kv->page_size) ++a.page_shift;
  a.kv_heads = kv->kv_heads;
  a.batch = kv->batch;
  a.table = kv->block_table;
  a.table_width = kv->table_width;
  a.table_stride = kv->table_stride;
  a.seq_lens = kv->seq_lens;
  a.status = kv->status;
  return a;
}

static PAttnArgs check_attn(const qd_paged_kv* kv, const void* q, int dtype, int64_t q_stride, int rows, int q_heads,
                            int window, int sinks, float scale, void* y, int64_t y_stride, int sure) {
  PAttnArgs a{};
  a.kv = check_paged(kv);
  need(rows >= 0, "paged attention: negative rows");
  need(dtype == QD_KV_F32 || dtype == kv->dtype, "paged attention: q and y are QD_KV_F32 or of the cache's dtype");
  need(q_heads >= 1 && q_heads % kv->kv_heads == 0 && q_heads / kv->kv_heads <= 64,
       "paged attention: q_heads must be a multiple of kv_heads, at most 64 times it");
  need(window >= 0 && sinks >= 0, "paged attention: window and sinks must not be negative");
  need(std::isfinite(scale), "paged attention: scale must be finite");
  need(rows == 0 || (q && y), "paged attention: NULL pointer");
  need(aligned16(q) && aligned16(y), "paged attention: q and y must be 16-byte aligned");
  need(q_stride >= (int64_t)q_heads * kHeadDim && y_stride >= (int64_t)q_heads * kHeadDim && q_stride % 8 == 0 &&
           y_stride % 8 == 0,
       "paged attention: row strides must be multiples of 8, at least q_heads * 128");
  // (several CTAs read a row of q, and one of them may be done first)
  const Rows out = rows_of(y, dtype, sure, (int64_t)q_heads * kHeadDim, y_stride);
  need(apart(out, rows_of(q, dtype, sure, (int64_t)q_heads * kHeadDim, q_stride)), "paged attention: y overlaps q");
  need_apart_from_pools(kv, out, "paged attention: y overlaps the pools");
  a.q = q;
  a.q_stride = q_stride;
  a.rows = rows;
  a.q_heads = q_heads;
  a.window = std::min(window, 1 << 30);  // positions end at 2^30: the same keys, and no overflow
  a.sinks = std::min(sinks, 1 << 30);
  a.scale = scale == 0.0f ? 1.0f / std::sqrt((float)kHeadDim) : scale;
  a.y = y;
  a.dtype = dtype;
  a.y_stride = y_stride;
  return a;
}

template <int HEADS>
static void launch_append(const AppendArgs& a, int qkv_dtype, long long heads, cudaStream_t s) {
  const long long warps = a.rows * ((heads + HEADS - 1) / HEADS);
  need(warps <= 0x7fffffffLL, "qd_paged_append: too many rows");
  const dim3 grid((unsigned)((warps + 7) / 8)), block(256);
  if (qkv_dtype == QD_KV_F32) launch_ex(k_paged_append<float, HEADS>, grid, block, 0, s, a);
  else if (qkv_dtype == QD_KV_F16) launch_ex(k_paged_append<__half, HEADS>, grid, block, 0, s, a);
  else launch_ex(k_paged_append<__nv_bfloat16, HEADS>, grid, block, 0, s, a);
}

template <typename T, bool THREE>
static void launch_decode(const PAttnArgs& a, void* workspace, cudaStream_t s) {
  static unsigned long long smem_set = 0;
  allow_smem(k_paged_decode<T, THREE>, pd_smem(4096), smem_set);
  const int nh = a.kv.kv_heads * ((a.q_heads / a.kv.kv_heads + 7) / 8);
  // two CTAs an SM hold all of them at once; no more than there can be units
  const long long most = (long long)a.kv.batch * nh * (((long long)a.kv.table_width << a.kv.page_shift) / kPdTile + 1);
  if (most > 0x7fffffffLL) throw QdError{QD_E_RANGE, "qd_paged_attn_decode: batch * heads * table beyond 2^31 units"};
  const int ctas = (int)std::max(1LL, std::min<long long>(most, std::min(2 * current_sms(), kPdMaxCtas)));
  launch_ex(k_paged_decode<T, THREE>, dim3(ctas), dim3(kPdThreads), (size_t)pd_smem(a.kv.batch), s, a, workspace);
  // (a table of one unit leaves nothing to join)
  if ((a.kv.table_width << a.kv.page_shift) > kPdTile)
    launch_ex(k_paged_decode_join, dim3(a.kv.batch * nh), dim3(256), 0, s, a, workspace, ctas);
}

// Row tiles of a call (at most), and the parts that their keys are split into: enough to give
// every SM a CTA, none where the row tiles alone do.
static int prompt_items(int batch, int rows, int group, int cta_rows) {
  return (int)((long long)rows * group / cta_rows) + std::min(batch, rows);
}
static int prompt_splits(int items, int kv_heads) {
  const long long n = (long long)items * kv_heads;
  return n == 0 ? 1 : (int)std::max(1LL, std::min<long long>(kPpMaxSplits, current_sms() / n));
}

static thread_local bool stall_next = false;  // qd_paged_inject_stall

template <typename T, int PARTS>
static void launch_prompt(const PAttnArgs& a, const void* q_any, void* workspace, cudaStream_t s) {
  constexpr int kRows = 128 * pp_tiles<PARTS>();
  const int G = a.q_heads / a.kv.kv_heads, items = prompt_items(a.kv.batch, a.rows, G, kRows);
  PPromptArgs p{};
  p.a = a;
  p.cta_rows = kRows;
  p.stall = stall_next;
  stall_next = false;
  p.splits = prompt_splits(items, a.kv.kv_heads);
  p.po = static_cast<float4*>(workspace);
  p.pml = reinterpret_cast<float2*>(p.po + (size_t)items * a.kv.kv_heads * p.splits * kRows * (kHeadDim / 4));
  // a table that holds few tiles never splits them into more parts than this
  const long long tiles = (((long long)a.kv.table_width << a.kv.page_shift) + kPpKeys - 1) / kPpKeys;
  p.splits = (int)std::max(1LL, std::min<long long>(p.splits, tiles / 2));
  const long long grid = (long long)items * a.kv.kv_heads * p.splits;
  if (grid * 32 > 0x7fffffffLL) throw QdError{QD_E_RANGE, "qd_paged_attn_prompt: too many rows"};
  const CUtensorMapDataType type =
      std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const unsigned box = std::min(1 << a.kv.page_shift, kPpKeys);
  // (an empty pool has no page that could be copied: any address will do)
  const uint64_t pool = std::max<uint64_t>((uint64_t)a.kv.num_pages * a.kv.kv_heads << a.kv.page_shift, box);
  if (pool > 0x7fffffffULL) throw QdError{QD_E_RANGE, "qd_paged_attn_prompt: a pool beyond 2^31 rows"};
  std::string err;
  if (!make_tmap_2d(&p.tk, a.kv.num_pages ? a.kv.k : q_any, type, kHeadDim, pool, kHeadDim * 2, 64, box,
                    CU_TENSOR_MAP_SWIZZLE_128B, &err) ||
      !make_tmap_2d(&p.tv, a.kv.num_pages ? a.kv.v : q_any, type, kHeadDim, pool, kHeadDim * 2, 64, box,
                    CU_TENSOR_MAP_SWIZZLE_128B, &err) ||
      !make_tmap_2d(&p.tv16, a.kv.num_pages ? a.kv.v : q_any, type, kHeadDim, pool, kHeadDim * 2, 64, 16,
                    CU_TENSOR_MAP_SWIZZLE_128B, &err))
    throw QdError{QD_E_CUDA, err};
  // More blocks than SMs: they take each other's work (5 ragged chunks in 480 blocks 109 -> 98 us; a prompt of
  // 8 rows, whose blocks have nothing to take, 9.6 us without that and 10.8 with it).
  static unsigned long long smem_set[2] = {};
  const bool claim = grid > current_sms();
  auto kernel = claim ? k_paged_prompt<T, PARTS, true> : k_paged_prompt<T, PARTS, false>;
  allow_smem(kernel, pp_smem<PARTS>(), smem_set[claim]);
  launch_ex(kernel, dim3((unsigned)grid), dim3(kPpThreads), (size_t)pp_smem<PARTS>(), s, p);
  if (p.splits > 1) launch_ex(k_paged_prompt_join, dim3(items * a.kv.kv_heads * (kRows / 8)), dim3(256), 0, s, p);
}

}  // namespace qd

using namespace qd;

// Runs a checked body, turning every exception into the C status and message.
template <typename F>
static int guarded(F&& body) {
  try {
    body();
  } catch (const QdError& err) {
    set_thread_error(err.msg);
    return err.code;
  } catch (const std::exception& err) {
    set_thread_error(err.what());
    return QD_E_NOMEM;
  }
  return QD_OK;
}

extern "C" {

int qd_paged_append(const qd_paged_kv* kv, const void* qkv, int qkv_dtype, int64_t qkv_stride, int rows,
                    const int32_t* q_starts, int q_heads, const float* q_norm, const float* k_norm, float eps,
                    const float* cos, const float* sin, int64_t rope_len, int64_t rope_stride, void* q_out,
                    int q_out_dtype, int64_t q_out_stride, void* stream) {
  return guarded([&] {
    AppendArgs a{};
    a.kv = check_paged(kv);
    need(rows >= 0, "qd_paged_append: negative rows");
    need(q_starts || rows == kv->batch, "qd_paged_append: without q_starts rows must equal the batch");
    need(known_dtype(qkv_dtype) && known_dtype(q_out_dtype), "qd_paged_append: unknown dtype");
    need(q_heads >= 0 && q_heads <= 65536, "qd_paged_append: bad q_heads");
    const int64_t heads = (int64_t)q_heads + 2 * kv->kv_heads;
    need(qkv_stride >= heads * kHeadDim && qkv_stride % 8 == 0,
         "qd_paged_append: qkv_stride must be a multiple of 8, at least (q_heads + 2 kv_heads) * 128");
    need(q_heads == 0 || (q_out_stride >= (int64_t)q_heads * kHeadDim && q_out_stride % 8 == 0),
         "qd_paged_append: q_out_stride must be a multiple of 8, at least q_heads * 128");
    need(std::isfinite(eps) && eps >= 0.0f, "qd_paged_append: eps must be finite and not negative");
    need((cos == nullptr) == (sin == nullptr), "qd_paged_append: cos and sin go together");
    need(!cos || (rope_len >= 0 && rope_stride >= 0 && rope_stride % 4 == 0),
         "qd_paged_append: rope_stride must be a multiple of 4, not negative");
    need(rows == 0 || (qkv && (q_out || q_heads == 0)), "qd_paged_append: NULL pointer");
    need(aligned16(qkv) && aligned16(q_out) && aligned16(cos) && aligned16(sin) && aligned16(q_norm) &&
             aligned16(k_norm),
         "qd_paged_append: pointers must be 16-byte aligned");
    const int sure = q_starts ? std::min(rows, 1) : rows;
    const Rows in = rows_of(qkv, qkv_dtype, sure, heads * kHeadDim, qkv_stride);
    const Rows out = rows_of(q_out, q_out_dtype, sure, (int64_t)q_heads * kHeadDim, q_out_stride);
    const bool in_place = q_out == qkv && q_out_dtype == qkv_dtype && (q_out_stride == qkv_stride || rows == 1);
    need(in_place || apart(out, in),
         "qd_paged_append: q_out overlaps qkv (it may be qkv itself, with its type and stride)");
    need_apart_from_pools(kv, out, "qd_paged_append: q_out overlaps the pools");
    need_apart_from_pools(kv, in, "qd_paged_append: qkv overlaps the pools");
    if (rows == 0 || kv->batch == 0) return;
    a.kv_dtype = kv->dtype;
    a.qkv = qkv;
    a.qkv_stride = qkv_stride;
    a.rows = rows;
    a.q_starts = q_starts;
    a.q_heads = q_heads;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.eps = eps;
    a.cos_t = cos;
    a.sin_t = sin;
    a.rope_len = rope_len;
    a.rope_stride = rope_stride;
    a.q_out = q_out;
    a.q_out_dtype = q_out_dtype;
    a.q_out_stride = q_out_stride;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // four heads a warp once that gives every SM four CTAs, else two
    if (rows * ((heads + 3) / 4) >= 32LL * current_sms()) launch_append<4>(a, qkv_dtype, heads, s);
    else launch_append<2>(a, qkv_dtype, heads, s);
  });
}

size_t qd_paged_attn_decode_workspace_bytes(int batch, int q_heads) {
  return batch < 0 || q_heads < 0 ? 0 : pd_ws_bytes(batch);
}

int qd_paged_attn_decode(const qd_paged_kv* kv, const void* q, int dtype, int64_t q_stride, int q_heads, int window,
                         int sinks, float scale, void* y, int64_t y_stride, void* workspace, void* stream) {
  return guarded([&] {
    need(kv != nullptr, "paged cache: NULL pointer");
    PAttnArgs a = check_attn(kv, q, dtype, q_stride, kv->batch, q_heads, window, sinks, scale, y, y_stride, kv->batch);
    if (a.rows == 0) return;
    need(workspace != nullptr, "qd_paged_attn_decode: NULL workspace");
    need(aligned16(workspace), "qd_paged_attn_decode: the workspace must be 16-byte aligned");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (kv->dtype == QD_KV_F16) launch_decode<__half, false>(a, workspace, s);
    else if (dtype == QD_KV_F32) launch_decode<__nv_bfloat16, true>(a, workspace, s);
    else launch_decode<__nv_bfloat16, false>(a, workspace, s);
  });
}

size_t qd_paged_attn_prompt_workspace_bytes(int batch, int rows, int q_heads, int kv_heads, int dtype) {
  if (batch < 0 || rows < 0 || q_heads < 1 || kv_heads < 1 || q_heads % kv_heads) return 0;
  size_t most = 256;
  for (const int cta_rows : {128, 256}) {  // (a CTA's rows depend on the types)
    const int items = prompt_items(batch, rows, q_heads / kv_heads, cta_rows), splits = prompt_splits(items, kv_heads);
    if (splits > 1 || dtype == QD_KV_F32)
      most = std::max(most, (size_t)items * kv_heads * splits * cta_rows * (kHeadDim * 4 + 8));
  }
  return most;
}

int qd_paged_attn_prompt(const qd_paged_kv* kv, const void* q, int dtype, int64_t q_stride, int rows,
                         const int32_t* q_starts, int q_heads, int window, int sinks, float scale, void* y,
                         int64_t y_stride, void* workspace, void* stream) {
  return guarded([&] {
    PAttnArgs a =
        check_attn(kv, q, dtype, q_stride, rows, q_heads, window, sinks, scale, y, y_stride, std::min(rows, 1));
    if (rows == 0 || kv->batch == 0) return;
    need(q_starts != nullptr, "qd_paged_attn_prompt: NULL q_starts");
    need(workspace != nullptr, "qd_paged_attn_prompt: NULL workspace");
    a.q_starts = q_starts;
    need(aligned16(workspace), "qd_paged_attn_prompt: the workspace must be 16-byte aligned");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (kv->dtype == QD_KV_F16) {
      if (dtype == QD_KV_F32) launch_prompt<__half, 2>(a, q, workspace, s);
      else launch_prompt<__half, 1>(a, q, workspace, s);
    } else {
      if (dtype == QD_KV_F32) launch_prompt<__nv_bfloat16, 3>(a, q, workspace, s);
      else launch_prompt<__nv_bfloat16, 1>(a, q, workspace, s);
    }
  });
}

void qd_paged_inject_stall(void) { stall_next = true; }

}  // extern "C"
