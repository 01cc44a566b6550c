// Host entries of the paged key-value cache operators (kernels: paged.cuh).
#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "../../include/qdecode.h"
#include "internal.cuh"
#include "overlap.hpp"
#include "paged.cuh"
#include "paged_decode.cuh"
#include "paged_prompt.cuh"
#include "paged_q8.cuh"
#include "paged_shared.cuh"

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

static PagedArgs check_q8(const qd_paged_q8* kv) {
  need(kv != nullptr, "paged cache: NULL pointer");
  const qd_paged_kv same{kv->k, kv->v, QD_KV_F16, kv->num_pages, kv->page_size, kv->kv_heads, kv->head_dim, kv->batch,
                         kv->block_table, kv->table_width, kv->table_stride, kv->seq_lens, kv->status};
  const PagedArgs a = check_paged(&same);
  need(kv->num_pages == 0 || (kv->k_scale && kv->v_scale), "paged cache: NULL scales");
  need(aligned16(kv->k_scale) && aligned16(kv->v_scale), "paged cache: scales must be 16-byte aligned");
  return a;
}
static void need_apart_from_q8(const qd_paged_q8* kv, const Rows& x, const char* msg) {
  const int64_t rows = (int64_t)kv->num_pages * kv->kv_heads * kv->page_size;
  for (const void* pool : {kv->k, kv->v}) need(apart(x, Rows{pool, 1, rows * kHeadDim, rows * kHeadDim}), msg);
  for (const void* scales : {kv->k_scale, kv->v_scale}) need(apart(x, Rows{scales, 1, rows * 4, rows * 4}), msg);
}

static PAttnArgs check_attn(const qd_paged_kv* kv, const void* q, int dtype, int64_t q_stride, int rows, int q_heads,
                            int window, int sinks, float scale, void* y, int64_t y_stride, int sure,
                            const qd_paged_q8* q8 = nullptr) {
  PAttnArgs a{};
  a.kv = q8 ? check_q8(q8) : check_paged(kv);
  need(rows >= 0, "paged attention: negative rows");
  need(q8 ? known_dtype(dtype) : dtype == QD_KV_F32 || dtype == kv->dtype,
       q8 ? "paged attention: unknown dtype" : "paged attention: q and y are QD_KV_F32 or of the cache's dtype");
  need(q_heads >= 1 && q_heads % a.kv.kv_heads == 0 && q_heads / a.kv.kv_heads <= 64,
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
  if (q8) need_apart_from_q8(q8, out, "paged attention: y overlaps the pools");
  else need_apart_from_pools(kv, out, "paged attention: y overlaps the pools");
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

template <int HEADS, bool Q8>
static void launch_append(const AppendArgs& a, int qkv_dtype, long long heads, cudaStream_t s) {
  const long long warps = a.rows * ((heads + HEADS - 1) / HEADS);
  need(warps <= 0x7fffffffLL, "qd_paged_append: too many rows");
  const dim3 grid((unsigned)((warps + 7) / 8)), block(256);
  if constexpr (Q8) {
    if (qkv_dtype == QD_KV_F32) launch_ex(k_paged_append_q8<float, HEADS / 2>, grid, block, 0, s, a);
    else if (qkv_dtype == QD_KV_F16) launch_ex(k_paged_append_q8<__half, HEADS / 2>, grid, block, 0, s, a);
    else launch_ex(k_paged_append_q8<__nv_bfloat16, HEADS / 2>, grid, block, 0, s, a);
  } else {
    if (qkv_dtype == QD_KV_F32) launch_ex(k_paged_append<float, HEADS>, grid, block, 0, s, a);
    else if (qkv_dtype == QD_KV_F16) launch_ex(k_paged_append<__half, HEADS>, grid, block, 0, s, a);
    else launch_ex(k_paged_append<__nv_bfloat16, HEADS>, grid, block, 0, s, a);
  }
}

// The append calls, over a checked cache; need_apart refuses rows that lie over it.
struct Scales {
  float *k, *v;
};
template <bool Q8, typename F>
static void append(const PagedArgs& kv, int kv_dtype, Scales scales, F&& need_apart, const void* qkv, int qkv_dtype,
                   int64_t qkv_stride, int rows, const int32_t* q_starts, int q_heads, const float* q_norm,
                   const float* k_norm, float eps, const float* cos, const float* sin, int64_t rope_len,
                   int64_t rope_stride, void* q_out, int q_out_dtype, int64_t q_out_stride, void* stream) {
  need(rows >= 0, "qd_paged_append: negative rows");
  need(q_starts || rows == kv.batch, "qd_paged_append: without q_starts rows must equal the batch");
  need(known_dtype(qkv_dtype) && known_dtype(q_out_dtype), "qd_paged_append: unknown dtype");
  need(q_heads >= 0 && q_heads <= 65536, "qd_paged_append: bad q_heads");
  const int64_t heads = (int64_t)q_heads + 2 * kv.kv_heads;
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
  need_apart(out, "qd_paged_append: q_out overlaps the pools");
  need_apart(in, "qd_paged_append: qkv overlaps the pools");
  if (rows == 0 || kv.batch == 0) return;
  AppendArgs a{};
  a.kv = kv;
  a.kv_dtype = kv_dtype;
  a.k_scale = scales.k;
  a.v_scale = scales.v;
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
  if (rows * ((heads + 3) / 4) >= 32LL * current_sms()) launch_append<4, Q8>(a, qkv_dtype, heads, s);
  else launch_append<2, Q8>(a, qkv_dtype, heads, s);
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
    launch_ex(k_paged_decode_join<8, true>, dim3(a.kv.batch * nh), dim3(256), 0, s, a, workspace, ctas);
}

// qd_paged_inject_stall and qd_paged_inject_stall_at, taken by the thread's next call.
static thread_local int stall_next = kPpStallNone;
static int take_stall() {
  const int stall = stall_next;
  stall_next = kPpStallNone;
  return stall;
}

template <typename Heads>
static void launch_decode_q8(Q8Args q, void* workspace, cudaStream_t s) {
  const PAttnArgs& a = q.a;
  const int nh = a.kv.kv_heads * ((a.q_heads / a.kv.kv_heads + Heads::kHeads - 1) / Heads::kHeads);
  const long long most = (long long)a.kv.batch * nh * (((long long)a.kv.table_width << a.kv.page_shift) / kQ8Tile + 1);
  if (most > 0x7fffffffLL)
    throw QdError{QD_E_RANGE, "qd_paged_attn_decode_q8: batch * heads * table beyond 2^31 units"};
  // (an empty pool has no page that could be copied: any address will do)
  const uint64_t pool = std::max<uint64_t>((uint64_t)a.kv.num_pages * a.kv.kv_heads << a.kv.page_shift, 16);
  if (pool > 0x7fffffffULL) throw QdError{QD_E_RANGE, "qd_paged_attn_decode_q8: a pool beyond 2^31 rows"};
  std::string err;
  for (const bool v : {false, true})
    if (!make_tmap_2d(v ? &q.tv : &q.tk, a.kv.num_pages == 0 ? a.q : v ? a.kv.v : a.kv.k, CU_TENSOR_MAP_DATA_TYPE_UINT8,
                      kHeadDim, pool, kHeadDim, kHeadDim, 16, CU_TENSOR_MAP_SWIZZLE_128B, &err))
      throw QdError{QD_E_CUDA, err};
  static unsigned long long smem_set = 0;
  allow_smem(k_paged_decode_q8<Heads>, pq8_smem(4096), smem_set);
  const int ctas = (int)std::max(1LL, std::min<long long>(most, std::min(Heads::kCtas * current_sms(), kPdMaxCtas)));
  launch_ex(k_paged_decode_q8<Heads>, dim3(ctas), dim3(kPdThreads), (size_t)pq8_smem(a.kv.batch), s, q, workspace);
  // (a table of one unit leaves nothing to join)
  // What follows starts when the join's CTAs have left: three CTAs of the next call fill an SM, and among the join's some
  // did not find their place in one piece until others had ended (64 sequences of 2048 positions, call after call: 70 us
  // instead of 56).
  if ((a.kv.table_width << a.kv.page_shift) > kQ8Tile)
    launch_ex(k_paged_decode_join<Heads::kHeads, false>, dim3(a.kv.batch * nh), dim3(256), 0, s, a, workspace, ctas);
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

template <typename T>
static void pool_maps(PPromptArgs& p, const void* any, const char* too_large) {
  const PagedArgs& kv = p.a.kv;
  const CUtensorMapDataType type =
      std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const unsigned box = std::min(1 << kv.page_shift, kPpKeys);
  // (an empty pool has no page that could be copied: any address will do)
  const uint64_t pool = std::max<uint64_t>((uint64_t)kv.num_pages * kv.kv_heads << kv.page_shift, box);
  if (pool > 0x7fffffffULL) throw QdError{QD_E_RANGE, too_large};
  std::string err;
  if (!make_tmap_2d(&p.tk, kv.num_pages ? kv.k : any, type, kHeadDim, pool, kHeadDim * 2, 64, box,
                    CU_TENSOR_MAP_SWIZZLE_128B, &err) ||
      !make_tmap_2d(&p.tv, kv.num_pages ? kv.v : any, type, kHeadDim, pool, kHeadDim * 2, 64, box,
                    CU_TENSOR_MAP_SWIZZLE_128B, &err) ||
      !make_tmap_2d(&p.tv16, kv.num_pages ? kv.v : any, type, kHeadDim, pool, kHeadDim * 2, 64, 16,
                    CU_TENSOR_MAP_SWIZZLE_128B, &err))
    throw QdError{QD_E_CUDA, err};
}

template <typename T, int PARTS>
static void launch_prompt(const PAttnArgs& a, const void* q_any, void* workspace, cudaStream_t s) {
  constexpr int kRows = 128 * pp_tiles<PARTS>();
  const int G = a.q_heads / a.kv.kv_heads, items = prompt_items(a.kv.batch, a.rows, G, kRows);
  PPromptArgs p{};
  p.a = a;
  p.cta_rows = kRows;
  p.stall = take_stall();
  p.splits = prompt_splits(items, a.kv.kv_heads);
  p.po = static_cast<float4*>(workspace);
  p.pml = reinterpret_cast<float2*>(p.po + (size_t)items * a.kv.kv_heads * p.splits * kRows * (kHeadDim / 4));
  // a table that holds few tiles never splits them into more parts than this
  const long long tiles = (((long long)a.kv.table_width << a.kv.page_shift) + kPpKeys - 1) / kPpKeys;
  p.splits = (int)std::max(1LL, std::min<long long>(p.splits, tiles / 2));
  const long long grid = (long long)items * a.kv.kv_heads * p.splits;
  if (grid * 32 > 0x7fffffffLL) throw QdError{QD_E_RANGE, "qd_paged_attn_prompt: too many rows"};
  pool_maps<T>(p, q_any, "qd_paged_attn_prompt: a pool beyond 2^31 rows");
  // More blocks than SMs: they take each other's work (5 ragged chunks in 480 blocks 109 -> 98 us; a prompt of
  // 8 rows, whose blocks have nothing to take, 9.6 us without that and 10.8 with it).
  static unsigned long long smem_set[2] = {};
  const bool claim = grid > current_sms();
  auto kernel = claim ? k_paged_prompt<T, PARTS, true> : k_paged_prompt<T, PARTS, false>;
  allow_smem(kernel, pp_smem<PARTS>(), smem_set[claim]);
  launch_ex(kernel, dim3((unsigned)grid), dim3(kPpThreads), (size_t)pp_smem<PARTS>(), s, p);
  if (p.splits > 1) launch_ex(k_paged_prompt_join, dim3(items * a.kv.kv_heads * (kRows / 8)), dim3(256), 0, s, p);
}

// Attention over shared prefixes: its workspace is the sums of both kinds of positions.
struct SharedWs {
  size_t po, pml, rows, tail_o, tail_ml, mark, decode, bytes;
};
constexpr int kSharedRows = 128;  // rows of a CTA (sequences times query heads of a KV head)
// Row tiles of the groups, at most.
static int shared_items(int batch, int groups, int group) {
  return (int)(((long long)batch * group + (long long)groups * (kSharedRows - 1)) / kSharedRows);
}
static SharedWs shared_ws(int batch, int groups, int q_heads, int kv_heads) {
  const int G = q_heads / kv_heads, items = shared_items(batch, groups, G);
  const size_t rows = (size_t)items * kv_heads * prompt_splits(items, kv_heads) * 2 * kSharedRows;  // (two sets)
  SharedWs w{};
  const auto take = [&](size_t n) {
    const size_t at = w.bytes;
    w.bytes += (n + 255) / 256 * 256;
    return at;
  };
  w.po = take(rows * kHeadDim * 4);
  w.pml = take(rows * 8);
  w.rows = take((size_t)batch * G * 8);
  w.tail_o = take((size_t)batch * q_heads * kHeadDim * 4);
  w.tail_ml = take((size_t)batch * q_heads * 8);
  w.mark = take(8);
  w.decode = take(pd_ws_bytes(batch));
  return w;
}

// A number that no call had before and that a workspace's old contents will hardly be.
static uint64_t next_ticket() {
  static std::atomic<uint64_t> calls{0};
  return (calls.fetch_add(1, std::memory_order_relaxed) + 1) * 0x9e3779b97f4a7c15ull;
}

template <typename T, int PARTS>
static void launch_shared(PAttnArgs a, void* workspace, cudaStream_t s) {
  constexpr int kSets = pp_tiles<PARTS>();
  const int B = a.kv.batch, kvh = a.kv.kv_heads, G = a.q_heads / kvh, subs = (G + 7) / 8;
  const long long most = (long long)B * kvh * subs * (((long long)a.kv.table_width << a.kv.page_shift) / kPdTile + 1);
  if (most > 0x7fffffffLL)
    throw QdError{QD_E_RANGE, "qd_paged_attn_decode_shared: batch * heads * table beyond 2^31 units"};
  const SharedWs w = shared_ws(B, a.groups, a.q_heads, kvh);
  char* base = static_cast<char*>(workspace);
  a.mark = reinterpret_cast<unsigned long long*>(base + w.mark);
  a.ticket = next_ticket();
  PPromptArgs p{};
  p.a = a;
  p.a.kv.batch = a.groups;
  p.stall = take_stall();
  p.cta_rows = kSharedRows;
  const int items = shared_items(B, a.groups, G);
  p.splits = prompt_splits(items, kvh);
  p.po = reinterpret_cast<float4*>(base + w.po);
  p.pml = reinterpret_cast<float2*>(base + w.pml);
  p.rows = reinterpret_cast<int2*>(base + w.rows);
  const long long grid = (long long)items * kvh * p.splits;  // (at least one)
  if (grid * 32 > 0x7fffffffLL) throw QdError{QD_E_RANGE, "qd_paged_attn_decode_shared: too many rows"};
  pool_maps<T>(p, a.q, "qd_paged_attn_decode_shared: a pool beyond 2^31 rows");
  static unsigned long long prefix_set[2] = {}, tail_set = 0;
  const bool claim = grid > current_sms();
  auto prefix = claim ? k_paged_prompt<T, PARTS, true, true> : k_paged_prompt<T, PARTS, false, true>;
  allow_smem(prefix, pp_smem<PARTS>(), prefix_set[claim]);
  launch_ex(prefix, dim3((unsigned)grid), dim3(kPpThreads), (size_t)pp_smem<PARTS>(), s, p);
  PSharedArgs j{};
  j.a = a;
  j.a.tail_o = reinterpret_cast<float*>(base + w.tail_o);
  j.a.tail_ml = reinterpret_cast<float2*>(base + w.tail_ml);
  j.po = p.po;
  j.pml = p.pml;
  j.rows = p.rows;
  j.splits = p.splits * kSets;
  j.cta_rows = kSharedRows;
  j.all_rows = items * kSharedRows;
  j.decode_ws = base + w.decode;
  j.ctas = (int)std::max(1LL, std::min<long long>(most, std::min(2 * current_sms(), kPdMaxCtas)));
  allow_smem(k_paged_decode<T, PARTS == 3, true>, pd_smem(4096), tail_set);
  launch_ex(k_paged_decode<T, PARTS == 3, true>, dim3(j.ctas), dim3(kPdThreads), (size_t)pd_smem(B), s, j.a,
            (void*)j.decode_ws);
  launch_ex(k_paged_shared_join, dim3((B * G + 7) / 8, kvh), dim3(kPsThreads), 0, s, j);
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
    const PagedArgs cache = check_paged(kv);
    append<false>(cache, kv->dtype, {}, [&](const Rows& x, const char* msg) { need_apart_from_pools(kv, x, msg); }, qkv, qkv_dtype,
                  qkv_stride, rows, q_starts, q_heads, q_norm, k_norm, eps, cos, sin, rope_len, rope_stride, q_out,
                  q_out_dtype, q_out_stride, stream);
  });
}

int qd_paged_append_q8(const qd_paged_q8* kv, const void* qkv, int qkv_dtype, int64_t qkv_stride, int rows,
                       const int32_t* q_starts, int q_heads, const float* q_norm, const float* k_norm, float eps,
                       const float* cos, const float* sin, int64_t rope_len, int64_t rope_stride, void* q_out,
                       int q_out_dtype, int64_t q_out_stride, void* stream) {
  return guarded([&] {
    const PagedArgs cache = check_q8(kv);
    append<true>(cache, QD_KV_F16, {kv->k_scale, kv->v_scale},
                 [&](const Rows& x, const char* msg) { need_apart_from_q8(kv, x, msg); }, qkv, qkv_dtype, qkv_stride, rows,
                 q_starts, q_heads, q_norm, k_norm, eps, cos, sin, rope_len, rope_stride, q_out, q_out_dtype,
                 q_out_stride, stream);
  });
}

int qd_paged_read_q8(const qd_paged_q8* kv, const int32_t* first, const qd_paged_kv* to, void* stream) {
  return guarded([&] {
    ReadArgs a{};
    a.src = check_q8(kv);
    need(to != nullptr, "paged cache: NULL pointer");
    qd_paged_kv out = *to;
    out.seq_lens = kv->seq_lens;  // (those of `to` are not looked at)
    a.dst = check_paged(&out);
    need(to->batch == kv->batch && to->kv_heads == kv->kv_heads,
         "qd_paged_read_q8: both caches must have the same batch and kv_heads");
    for (const void* pool : {to->k, to->v}) {
      const int64_t bytes = (int64_t)to->num_pages * to->kv_heads * to->page_size * kHeadDim * 2;
      need_apart_from_q8(kv, Rows{pool, 1, bytes, bytes}, "qd_paged_read_q8: the 16-bit pools overlap the 8-bit ones");
    }
    a.scale = {kv->k_scale, kv->v_scale};
    a.first = first;
    a.dtype = to->dtype;
    if (kv->batch == 0) return;
    const long long most = (long long)kv->batch * kv->kv_heads * (((long long)kv->table_width << a.src.page_shift) / 16 + 1);
    if (most > 0x7fffffffLL) throw QdError{QD_E_RANGE, "qd_paged_read_q8: batch * heads * table beyond 2^31 units"};
    const int ctas = (int)std::max(1LL, std::min<long long>((most + 3) / 4, 32 * current_sms()));
    const size_t smem = (size_t)(kv->batch + 1) * 4;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (to->dtype == QD_KV_F16) launch_ex(k_paged_read_q8<__half>, dim3(ctas), dim3(kPdThreads), smem, s, a);
    else launch_ex(k_paged_read_q8<__nv_bfloat16>, dim3(ctas), dim3(kPdThreads), smem, s, a);
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

int qd_paged_attn_decode_q8(const qd_paged_q8* kv, const void* q, int dtype, int64_t q_stride, int q_heads, int window,
                            int sinks, float scale, void* y, int64_t y_stride, void* workspace, void* stream) {
  return guarded([&] {
    need(kv != nullptr, "paged cache: NULL pointer");
    PAttnArgs a =
        check_attn(nullptr, q, dtype, q_stride, kv->batch, q_heads, window, sinks, scale, y, y_stride, kv->batch, kv);
    if (a.rows == 0) return;
    need(workspace != nullptr, "qd_paged_attn_decode_q8: NULL workspace");
    need(aligned16(workspace), "qd_paged_attn_decode_q8: the workspace must be 16-byte aligned");
    Q8Args args{};
    args.a = a;
    args.scale = {kv->k_scale, kv->v_scale};
    args.stall = take_stall() == kPpStallFirst;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int group = q_heads / kv->kv_heads;
    if (group <= 2) launch_decode_q8<Q8Whole>(args, workspace, s);
    else if (group <= 4) launch_decode_q8<Q8Half<1>>(args, workspace, s);
    else launch_decode_q8<Q8Half<2>>(args, workspace, s);
  });
}

size_t qd_paged_attn_decode_shared_workspace_bytes(int batch, int groups, int q_heads, int kv_heads) {
  if (batch < 0 || groups < 0 || groups > batch || q_heads < 1 || kv_heads < 1 || q_heads % kv_heads) return 0;
  return shared_ws(batch, groups, q_heads, kv_heads).bytes;
}

int qd_paged_attn_decode_shared(const qd_paged_kv* kv, const void* q, int dtype, int64_t q_stride, int q_heads,
                                int groups, const int32_t* group_starts, const int32_t* shared_lens, float scale,
                                void* y, int64_t y_stride, void* workspace, void* stream) {
  return guarded([&] {
    need(kv != nullptr, "paged cache: NULL pointer");
    PAttnArgs a = check_attn(kv, q, dtype, q_stride, kv->batch, q_heads, 0, 0, scale, y, y_stride, kv->batch);
    need(groups >= 0 && groups <= kv->batch, "qd_paged_attn_decode_shared: groups must be 0..batch");
    if (a.rows == 0 || groups == 0) return;
    need(group_starts && shared_lens, "qd_paged_attn_decode_shared: NULL group_starts or shared_lens");
    need(workspace != nullptr, "qd_paged_attn_decode_shared: NULL workspace");
    need(aligned16(workspace), "qd_paged_attn_decode_shared: the workspace must be 16-byte aligned");
    a.q_starts = group_starts;
    a.groups = groups;
    a.shared_lens = shared_lens;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (kv->dtype == QD_KV_F16) {
      if (dtype == QD_KV_F32) launch_shared<__half, 2>(a, workspace, s);
      else launch_shared<__half, 1>(a, workspace, s);
    } else {
      if (dtype == QD_KV_F32) launch_shared<__nv_bfloat16, 3>(a, workspace, s);
      else launch_shared<__nv_bfloat16, 1>(a, workspace, s);
    }
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

void qd_paged_inject_stall(void) { stall_next = kPpStallFirst; }
int qd_paged_inject_stall_at(int where) {
  return guarded([&] {
    need(where == kPpStallFirst || where == kPpStallLate || where == kPpStallLast, "qd_paged_inject_stall_at: no such place");
    stall_next = where;
  });
}

}  // extern "C"
