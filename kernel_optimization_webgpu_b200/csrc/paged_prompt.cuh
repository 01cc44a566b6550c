// Attention of a ragged batch of prompt chunks over a paged cache, on the tcgen05 tensor cores.
//
// Rows: the (token, query head) pairs of one sequence and KV head, token-major, so that all the
// query heads that share a KV head share its tiles whatever their number. A CTA takes 256
// consecutive rows as two M = 128 tiles and walks the 128-key tiles that any of its rows sees:
//   S = Q K^T      -> TMEM (f32)                     M 128, N 128 keys, K 128 dims
//   P = exp2(S c - m)   two threads per row: maximum, weights, their sum, all in f32
//   O += P V       -> TMEM (f32), P read from TMEM   M 128, N 128 dims, K 128 keys
// The two tiles alternate: while one's softmax runs, the tensor cores work for the other. P
// replaces its S in TMEM (S0 S1 O0 O1 = 512 columns); the MMAs of one issuer run in order, so
// S of the next key tile may be issued right behind the product that reads P. What bounds it:
// 2048 cycles of products and as many of exponentials per 256 rows and 128 keys, in a loop of
// 3460 (scores ready -> weights ready 1900, products -> next scores ready 1460, for each tile in
// turn): 8192 causal rows of 16 heads take 250 us = 1100 TFLOP/s in a burst at 1965 MHz, and 292 us one
// after the other for a second, at 1620 to 1680 MHz under the power cap (3 us more before the products of the
// first half of P's keys started ahead of the second). Beside it at 266 us: one thread per row
// instead of two 301 us, an exp2 by polynomial for 3 to 8 of 16 weights 269 to 287 us
// (the softmax warps wait on each other's instructions, not on the special-function unit).
//
// O is rescaled only when a row's maximum has grown by more than 2^kPpLag since the last time
// (weights then stay below 2^(kPpLag + kPpShift), inside f16); the final division makes up for
// it, so the result is exact to rounding. P is rounded to the cache's 16-bit type (half a step
// relative, as the tensor cores take 16-bit operands); its sum is taken in f32 before that.
// With f32 queries q and P are each a sum of PARTS 16-bit operands, and every product is issued that
// many times: two f16 keep 22 bits (of a row of q that a power of two has brought to the upper end of f16's
// range; the factor of the row's scores takes it back), two bf16 only 16 (the results were 5e-6 off),
// so a bf16 cache takes three. Three parts of P do not fit over S in TMEM, so such a CTA has one row tile. The
// tensor cores drop the bits below an accumulator's last place, towards zero, at every step, which
// over a long row shows in f32: every kPpFlush tiles O moves from TMEM to sums in the workspace that
// are added with rounding (rows over 4000 keys with values of one sign: 4e-6 off, 3e-5 without; it costs a
// causal prompt of 4096 rows 154 us against 122, with three parts 257 against 218).
//
// Where the grid does not fit the GPU at once, a CTA goes on with the work of blocks that have not started
// (cluster launch control), looked up by a warp of its own while the last key tiles are still on
// their way: K and V of the next rows flow through the ring without a pause, their Q is on its
// way into L2, and one row tile ends while the other still has products. 5 ragged chunks (480
// blocks of 30 us, 8 of them start and end): 109 -> 98 us, 1.5 of them by Q's prefetch.
//
// K and V come page by page by TMA (128-byte swizzle; rows of a page and head are contiguous)
// into a ring of 32 KB tiles. V rows that no query of the CTA sees are zeros in shared memory: their
// weight is 0, but 0 times what a recycled page holds could be NaN.
//
// Few rows over a long cache (a chunk behind a long context): the key tiles of a CTA's rows are
// split over gridDim parts whose sums k_paged_prompt_join adds in order.
#pragma once

#include <climits>
#include <type_traits>

#include "gemm_tc.cuh"
#include "paged_decode.cuh"

namespace qd {

constexpr int kPpSoftmax = 512;    // softmax threads: two a row, 64 keys of a tile each
constexpr int kPpThreads = 640;    // and the MMA warp, the copy warp, the scheduling warp and an idle one
// Registers: 96 a thread at launch (61440 in all); a softmax thread holds 64 scores, so the last
// warpgroup gives some of its share up: 512 * 104 + 128 * 64 = 61440.
constexpr int kPpRegsMany = 104, kPpRegsFew = 64;
constexpr int kPpKeys = 128;
constexpr int kPpTileBytes = 128 * 256;  // a 128 x 128 tile of 16-bit elements
constexpr int kPpMaxSplits = 32;
constexpr int kPpFlush = 4;        // tiles between two moves of O to the workspace (f32 results)
constexpr float kPpLag = 8.0f, kPpShift = 7.0f;

// First: block 0 withholds its first key tile. Late (SHARED): the second softmax set begins each work 40 us late. Last:
// block 0 withholds the last key tile of its first work, whose successor it has then taken.
enum PpStall : int { kPpStallNone = 0, kPpStallFirst = 1, kPpStallLate = 2, kPpStallLast = 3 };
struct PPromptArgs {
  CUtensorMap tk, tv, tv16;  // boxes of a page (at most 128 rows), and of 16 rows
  PAttnArgs a;
  int splits;
  int cta_rows;  // 128 times the row tiles of a CTA
  int stall;     // test hook (qd_paged_inject_stall, qd_paged_inject_stall_at), one of PpStall
  // Unnormalised sums (f32 results, or parts > 1): [item][KV head][split][32 groups of 4 dims][cta_rows], so
  // that a warp's rows lie side by side; and their maxima and weights: [item][KV head][split][cta_rows].
  float4* po;
  float2* pml;
  int2* rows;    // SHARED: [batch][query heads of a KV head]: where a row's sums are (item * cta_rows + row), its parts
};

template <int PARTS>
__host__ __device__ constexpr int pp_tiles() { return PARTS == 3 ? 1 : 2; }  // row tiles of a CTA
template <int PARTS>
__host__ __device__ constexpr int pp_slots() { return PARTS == 1 ? 5 : PARTS == 2 ? 3 : 4; }
template <int PARTS>
__host__ __device__ constexpr int pp_smem() {
  return (pp_tiles<PARTS>() * PARTS + pp_slots<PARTS>()) * kPpTileBytes + 1024;
}
// With SHARED: one tile of queries, the rest of that memory goes to the ring.
template <int PARTS>
__host__ __device__ constexpr int pp_shared_slots() { return pp_slots<PARTS>() + (pp_tiles<PARTS>() - 1) * PARTS; }

// The item-th tile of rows, counted from the last (the latest rows of a prompt see the most keys
// and start first): its sequence, tile, first row, new tokens and length, or false. Called by
// whole warps; up to 32 sequences take one round trip to memory.
__device__ __forceinline__ bool pp_item(const PAttnArgs& a, int G, int cta_rows, int item, int& seq, int& tile, int& start,
                                        int& fresh, int& asked) {
  const int lane = threadIdx.x & 31, B = a.kv.batch;
  int n0 = 0, s0 = 0, len0 = 0;  // of the first 32 sequences
  int total = 0;
  for (int b0 = 0; b0 < B; b0 += 32) {
    const int b = b0 + lane;
    int n = 0, s = 0;
    if (b < B) {
      s = a.q_starts[b];
      n = max(a.q_starts[b + 1] - s, 0);
      if (b0 == 0) len0 = a.kv.seq_lens[b];
    }
    if (b0 == 0) {
      n0 = n;
      s0 = s;
    }
    int t = (n * G + cta_rows - 1) / cta_rows;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    total += t;
  }
  int want = total - 1 - item;
  if (want < 0) return false;
  for (int b0 = 0; b0 < B; b0 += 32) {
    const int b = b0 + lane;
    const int n = b0 == 0 ? n0 : b < B ? max(a.q_starts[b + 1] - a.q_starts[b], 0) : 0;
    const int t = (n * G + cta_rows - 1) / cta_rows;
    int incl = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    const unsigned past = __ballot_sync(0xffffffffu, incl > want);
    if (past) {
      const int src = __ffs(past) - 1;
      seq = b0 + src;
      tile = want - __shfl_sync(0xffffffffu, incl - t, src);
      fresh = __shfl_sync(0xffffffffu, n, src);
      start = b0 == 0 ? __shfl_sync(0xffffffffu, s0, src) : a.q_starts[seq];
      asked = b0 == 0 ? __shfl_sync(0xffffffffu, len0, src) : a.kv.seq_lens[seq];
      return true;
    }
    want -= __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
}

// What the rows of an item are: first token, positions, and the keys that any of them sees.
struct PpItem {
  int seq, tok0, n_rows, pos0, len;  // row r: token tok0 + r / G at position pos0 + r / G
  Visible v;
};
__device__ __forceinline__ PpItem pp_rows(const PAttnArgs& a, int G, int cta_rows, int tile, int start, int fresh,
                                          int asked) {
  PpItem it;
  it.len = min(max(asked, 0), a.kv.table_width << a.kv.page_shift);
  it.tok0 = start;
  it.pos0 = asked - fresh;
  it.n_rows = fresh * G;
  const int r0 = tile * cta_rows, r1 = min(r0 + cta_rows, it.n_rows);
  const int plo = it.pos0 + r0 / G, phi = it.pos0 + (r1 - 1) / G;
  Visible& v = it.v;
  v.end = max(0, min(phi + 1, it.len));
  v.lo = a.window > 0 ? max(0, plo + 1 - a.window) : 0;
  v.ns = min(min(a.sinks, v.lo), v.end);
  v.st = (v.ns + kPpKeys - 1) / kPpKeys;
  v.w0 = max(v.lo / kPpKeys, v.st);
  v.tiles = v.st + max(0, (v.end + kPpKeys - 1) / kPpKeys - v.w0);
  return it;
}
// The same for queries of a group of sequences over the positions that they share with its first: row r belongs to
// sequence tok0 + r / G and sees what of them its own length leaves (pp_shares). Whole warps.
__device__ __forceinline__ int pp_shares(const PAttnArgs& a, int seq) {
  return max(0, min(paged_len(a.kv, seq), a.shared_lens[seq]));
}
__device__ __forceinline__ PpItem pp_shared_rows(const PAttnArgs& a, int G, int cta_rows, int tile, int start, int n) {
  PpItem it;
  it.tok0 = start;
  it.pos0 = 0;
  it.n_rows = n * G;
  const int r0 = tile * cta_rows, r1 = min(r0 + cta_rows, it.n_rows);
  int most = 0;
  for (int s = start + r0 / G + (threadIdx.x & 31); s <= start + (r1 - 1) / G; s += 32)
    if ((unsigned)s < (unsigned)a.rows) most = max(most, pp_shares(a, s));
  it.len = __reduce_max_sync(0xffffffffu, most);
  it.v = Visible{it.len, 0, 0, 0, 0, (it.len + kPpKeys - 1) / kPpKeys};
  return it;
}
// Largest of three, NaN if one of them is.
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
// Whether any of a pair of warps says so, and their plain meeting.
__device__ __forceinline__ bool pp_any(int barrier, bool mine) {
  unsigned r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbarrier.cta.red.or.pred p, %2, 64, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"((unsigned)mine), "r"(barrier)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void pp_meet(int barrier) { asm volatile("barrier.cta.sync %0, 64;" ::"r"(barrier) : "memory"); }
// Bits 0 .. n - 1.
__device__ __forceinline__ unsigned pp_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
// Parts that an item's key tiles are really split into: at least two tiles each.
__device__ __forceinline__ int pp_parts(int tiles, int splits) { return min(splits, max(1, tiles >> 1)); }

// Bounded wait that gives up at once where another role already has.
__device__ __forceinline__ bool pp_wait(unsigned long long* bar, unsigned parity, volatile int* failed,
                                        unsigned long long limit = kTcWaitNs) {
  if (tc_mbar_test(bar, parity)) return true;
  const unsigned long long t0 = tc_now();
  while (!tc_mbar_test(bar, parity)) {
    if (*failed) return false;
    if (tc_now() - t0 > limit) {
      *failed = 1;
      return false;
    }
  }
  return true;
}
// The limit of a wait for work of so many key tiles to come to its end (a tile takes 2 to 4 us).
__device__ __forceinline__ unsigned long long pp_patience(int tiles) { return kTcWaitNs + 16384ull * (unsigned)tiles; }
__device__ __forceinline__ void pp_arrive(unsigned long long* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc_smem(bar)) : "memory");
}

// What a CTA does next, as its scheduling warp writes it for the others. halves: row tiles, 0 at the end.
struct PpWork {
  PpItem it;
  int item, row0, g, z, parts, t0, nk, halves;
};
// Takes a block of the grid that has not started yet; its index and true, or false when all have.
__device__ __forceinline__ void pp_claim(void* answer, unsigned long long* bar) {
  asm volatile(
      "mbarrier.arrive.expect_tx.shared::cta.b64 _, [%1], 16;\n\t"
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
          tc_smem(answer)),
      "r"(tc_smem(bar))
      : "memory");
}
__device__ __forceinline__ bool pp_claimed(const void* answer, int& block) {
  unsigned got, x;
  asm volatile(
      "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\tld.shared.b128 h, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
      : "=r"(got), "=r"(x)
      : "r"(tc_smem(answer))
      : "memory");
  block = (int)x;
  return got != 0;
}

// B operand with its N index (dims) contiguous: 64-dim rows of 128 bytes, 128-byte swizzle; the
// next 64 dims kPpTileBytes / 2 on, the next 8 keys 1024 bytes on.
__device__ __forceinline__ unsigned long long umma_desc_mn_sw128(unsigned smem_addr) {
  return (unsigned long long)((smem_addr >> 4) & 0x3FFFu) | ((unsigned long long)(kPpTileBytes / 2 >> 4) << 16) |
         ((unsigned long long)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// f32 accumulator, 16-bit operands (f16 or bf16), B with N contiguous where mn.
template <typename T>
__device__ __forceinline__ unsigned pp_idesc(bool mn) {
  const unsigned fmt = sizeof(T) == 2 && !std::is_same<T, __half>::value ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (mn ? 1u << 16 : 0u) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
}
// D (+)= A B, issued by the lane whose `leader` is set: A from shared memory, or from TMEM.
template <bool kAccumulate>
__device__ __forceinline__ void pp_mma_ss(unsigned d_tmem, unsigned long long a, unsigned long long b, unsigned idesc,
                                          unsigned leader) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 e, %4, 0;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(leader), "n"(kAccumulate ? 1 : 0)
      : "memory");
}
__device__ __forceinline__ void pp_mma_ts(unsigned d_tmem, unsigned a_tmem, unsigned long long b, unsigned idesc,
                                          bool accumulate, unsigned leader) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 e, %4, 0;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b), "r"(idesc), "r"(leader), "r"((unsigned)accumulate)
      : "memory");
}
// All products issued so far by that lane arrive on the barrier when they are done.
__device__ __forceinline__ void pp_commit(unsigned long long* bar, unsigned leader) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(tc_smem(bar)),
      "r"(leader)
      : "memory");
}
#define PP_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
// 64 consecutive TMEM columns of this warp's lanes.
__device__ __forceinline__ void tmem_ld64(unsigned taddr, unsigned* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : PP_R8(r, 0), PP_R8(r, 8), PP_R8(r, 16), PP_R8(r, 24), PP_R8(r, 32), PP_R8(r, 40), PP_R8(r, 48), PP_R8(r, 56)
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(unsigned taddr, unsigned* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : PP_R8(r, 0), PP_R8(r, 8)
      : "r"(taddr)
      : "memory");
}
#undef PP_R8
#define PP_W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
__device__ __forceinline__ void tmem_st16(unsigned taddr, const unsigned* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::PP_W8(r, 0),
      PP_W8(r, 8), "r"(taddr)
      : "memory");
}
#undef PP_W8
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <typename T>
__device__ __forceinline__ unsigned pack2(float x, float y);
template <>
__device__ __forceinline__ unsigned pack2<__half>(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const unsigned*>(&h);
}
template <>
__device__ __forceinline__ unsigned pack2<__nv_bfloat16>(float x, float y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const unsigned*>(&h);
}

// x, y as the sum of PARTS packed pairs, each the rounded rest of those before.
template <typename T, int PARTS>
__device__ __forceinline__ void split_parts(float x, float y, unsigned (&u)[PARTS]) {
  if constexpr (PARTS == 1) {
    u[0] = pack2<T>(x, y);
  } else if constexpr (PARTS == 2) {
    split2<T>(x, y, u[0], u[1]);
  } else {
    const float2 rest = split2_rest<T>(x, y, u[0]);
    split2<T>(rest.x, rest.y, u[1], u[2]);
  }
}

// CLAIM: blocks take the work of others that have not started (a grid that does not fit the GPU at once).
// SHARED: the rows of a "sequence" are the queries of a group, all of which see the positions that the group shares
// (a.q_starts: the groups' first sequences, a.kv.batch of them); every row's sums go to the workspace. A CTA has one
// tile of 128 rows, as few queries share a prefix, and its two sets of softmax threads take every other key
// tile of it: S_t = Q K_j^T for t = j % 2, with a maximum, sums and an O of their own, joined like the parts of
// several CTAs: 64 f32 queries behind 16384 shared keys, 16 query and 8 KV heads, 62 -> 56 us for the whole call
// (16-bit queries gained nothing: the loop over key tiles already took them at 5.4 TB/s).
template <typename T, int PARTS, bool CLAIM, bool SHARED = false>
__global__ void __launch_bounds__(kPpThreads, 1) k_paged_prompt(const __grid_constant__ PPromptArgs pa) {
  const PAttnArgs& a = pa.a;
  constexpr int kTiles = pp_tiles<PARTS>(), kQTiles = SHARED ? 1 : kTiles, kRows = 128 * kQTiles;
  constexpr int S = SHARED ? pp_shared_slots<PARTS>() : pp_slots<PARTS>();
  constexpr int kAlt = SHARED ? kTiles : 1;  // sets that share the key tiles of a row
  // (with three parts and one set, a tile's 24 products into O cost 1.7e-6 of the result with moves every four tiles, 1.0e-6 so)
  constexpr int kFlush = SHARED && PARTS == 3 ? 2 : kPpFlush;
  constexpr int kQTile = PARTS * kPpTileBytes;  // the parts of 128 rows
  // Parts of a weight: those of q, but two for 16-bit queries over shared positions, as k_paged_decode takes them for
  // the positions behind and for all of a sequence alone. With one, f16 results were 2.8e-4 off and bf16 results
  // 2.0e-3, where their own rounding is 2.1e-4 and 1.7e-3; 64 of 16384 took 49 us, 7 groups of bf16 56 (51 and 59 with two).
  constexpr int kParts = SHARED && PARTS == 1 ? 2 : PARTS;
  // O moves to the workspace every kFlush tiles. Not for 16-bit results: what the products drop on the way, 3e-5 of
  // a sum of 8192 values of one sign that one CTA takes, is a sixth of their rounding (moves every 4 tiles: 3e-6, 65
  // us for the 7 groups; every 16: 1.4e-5, 60 us).
  constexpr bool kMoves = PARTS > 1;
  // TMEM columns: S_t | O_t with P over S, or S | P (three parts) | O
  constexpr unsigned kColP = kTiles == 2 ? 0 : 128, kColO = kTiles == 2 ? 256 : 384;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* qs =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* ring = qs + kQTiles * kQTile;
  __shared__ unsigned long long full[S], empty[S], s_full[2], p_half[2], p_full[2], o_done[2], q_full[2], drain;
  __shared__ unsigned long long work_full[2], work_empty[2], ask, answered;
  __shared__ __align__(16) uint4 answer;
  __shared__ PpWork work[3];  // two in turn; one that was taken and could not be handed on
  __shared__ unsigned bad_rows[8];  // of key tile j: bit i set where 16-key chunk i has no usable page
  __shared__ unsigned tmem_base;
  __shared__ float shared_row[256];  // between a row's two threads: a maximum (NaN: given up), then a sum
  __shared__ unsigned char q_exp[2][SHARED ? 128 : 1];  // largest exponents of the queries, for the other set
  __shared__ int failed;
  // (values read back from lane 0 are warp-uniform to the compiler: the MMA warp's operands then live
  // in uniform registers)
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int kvh = a.kv.kv_heads, G = a.q_heads / kvh;
  if (tid == 0) {
    tma_prefetch_map(&pa.tk);
    tma_prefetch_map(&pa.tv);
    tma_prefetch_map(&pa.tv16);
  }
  pdl_wait();
  if (SHARED && blockIdx.x == 0 && tid == 0)
    asm volatile("st.release.gpu.global.u64 [%0], %1;" ::"l"(a.mark), "l"(a.ticket) : "memory");
  pdl_trigger();
  // What block `b` of the grid is to do, if anything (whole warps).
  auto find_work = [&](int b, PpWork& w) {
    w.g = b % kvh;
    w.z = (b / kvh) % pa.splits;
    w.item = b / (kvh * pa.splits);
    int seq = 0, tile = 0, start = 0, fresh = 0, asked = 0;
    if (!pp_item(a, G, kRows, w.item, seq, tile, start, fresh, asked)) return false;
    if constexpr (SHARED) {
      if ((unsigned)start >= (unsigned)a.rows) return false;  // (no such sequence)
      w.it = pp_shared_rows(a, G, kRows, tile, start, fresh);
      seq = start;  // (whose pages are the group's)
    } else {
      w.it = pp_rows(a, G, kRows, tile, start, fresh, asked);
    }
    w.it.seq = seq;
    // beyond the table, or new tokens before position 0 (a length of 0 is a padded sequence)
    if (!SHARED && (asked > w.it.len || (asked != 0 && asked < fresh)) && lane == 0) paged_flag(a.kv, QD_PAGED_BAD_LENGTH);
    w.parts = pp_parts(w.it.v.tiles, pa.splits);
    if (w.z >= w.parts) return false;
    w.t0 = w.it.v.tiles * w.z / w.parts;  // (at most 2^23 tiles, 32 parts)
    w.nk = w.it.v.tiles * (w.z + 1) / w.parts - w.t0;
    w.row0 = tile * kRows;
    w.halves = kTiles == 2 && (SHARED ? w.nk > 1 : w.it.n_rows - w.row0 > 128) ? 2 : 1;
    return true;
  };
  PpWork first;
  if (!find_work(blockIdx.x, first)) return;
  // The n-th work of the block, when it is there (the one before has `tiles`); false: given up.
  auto wait_work = [&](int n, int tiles) {
    return !CLAIM ||
           __all_sync(0xffffffffu, pp_wait(&work_full[n & 1], (unsigned)(n >> 1) & 1u, &failed, pp_patience(tiles)));
  };
  // SHARED: where a work's row has its sums, and how many of them.
  auto place = [&](const PpWork& w, int lr) {
    return make_int2(w.item * kRows + lr, w.it.v.tiles < 2 ? w.it.v.tiles : w.parts * kAlt);
  };
  auto work_of = [&](int n) -> const PpWork& { return CLAIM ? work[n & 1] : first; };
  auto work_done = [&](int n) {
    __syncwarp();
    if (CLAIM && lane == 0) pp_arrive(&work_empty[n & 1]);
  };

  if (warp == kPpSoftmax / 32) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem(&tmem_base)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    for (int i = 0; i < S; ++i) {
      tc_mbar_init(&full[i]);
      tc_mbar_init(&empty[i]);
    }
    tc_mbar_init(&drain);
    for (int i = 0; i < 2; ++i) {
      tc_mbar_init(&s_full[i]);
      tc_mbar_init(&o_done[i]);
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 256;" ::"r"(tc_smem(&p_full[i])) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 256;" ::"r"(tc_smem(&p_half[i])) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 256;" ::"r"(tc_smem(&q_full[i])) : "memory");
      tc_mbar_init(&work_full[i]);
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(tc_smem(&work_empty[i])), "n"(kPpSoftmax / 32 + 2)
                   : "memory");
    }
    tc_mbar_init(&ask);
    tc_mbar_init(&answered);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    failed = 0;
    work[0] = first;
    work[1].halves = work[2].halves = 0;
    if (CLAIM) pp_arrive(&work_full[0]);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = __shfl_sync(0xffffffffu, tmem_base, 0);

  if (warp >= kPpSoftmax / 32) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPpRegsFew));
    if (CLAIM && warp == kPpSoftmax / 32 + 2) {
      // ---- schedule: this block's work, then that of blocks that have not started ----
      // (asked for by the copy warp when it comes to the last tile)
      int next = 1, claims = 0, block = 0, tiles = work[0].nk;
      bool ok = true, more = true;
      auto free_slot = [&] {
        return next < 2 ||
               __all_sync(0xffffffffu, pp_wait(&work_empty[next & 1], (unsigned)(next / 2 - 1) & 1u, &failed));
      };
      while (ok && more) {
        ok = __all_sync(0xffffffffu, pp_wait(&ask, (unsigned)(next - 1) & 1u, &failed, pp_patience(tiles)));
        if (!ok) break;
        PpWork w;
        do {
          if (lane == 0) pp_claim(&answer, &answered);
          ok = __all_sync(0xffffffffu, tc_mbar_wait(&answered, (unsigned)claims++ & 1u));
          if (!ok) failed = 1;
          more = ok && pp_claimed(&answer, block);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (read before the next answer lands)
          __syncwarp();
        } while (more && !find_work(__shfl_sync(0xffffffffu, block, 0), w));
        if (!more) break;
        for (int r = w.row0 + lane; r < min(w.row0 + kRows, w.it.n_rows); r += 32) {  // Q, to L2
          const int tok = w.it.tok0 + r / G;
          if ((unsigned)tok < (unsigned)a.rows) {
            constexpr int kSize = PARTS > 1 ? 4 : 2;
            const char* q = static_cast<const char*>(a.q) +
                            ((long long)tok * a.q_stride + ((long long)w.g * G + r % G) * kHeadDim) * kSize;
#pragma unroll
            for (int i = 0; i < kHeadDim * kSize; i += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + i));
          }
        }
        tiles = w.nk;
        ok = free_slot();
        if (lane == 0) {
          work[ok ? next & 1 : 2] = w;
          if (ok) pp_arrive(&work_full[next & 1]);
        }
        ++next;
      }
      if (ok && free_slot() && lane == 0) {
        work[next & 1].halves = 0;
        pp_arrive(&work_full[next & 1]);
      }
    } else if (warp == kPpSoftmax / 32 + 1) {
      // ---- copies: K and V tiles alternate through the ring ----
      const int ps = 1 << a.kv.page_shift, box = min(ps, kPpKeys), boxes = kPpKeys / box;
      int issued_to = -1, done = 0;  // ring slots of the works before
      bool ok = !(pa.stall == kPpStallFirst && blockIdx.x == 0);
      for (int n = 0, nk = 0; ok && (CLAIM || n == 0); ++n) {
        ok = wait_work(n, nk);
        if (!ok || work_of(n).halves == 0) break;
        const PpItem it = work_of(n).it;
        const int seq = it.seq, g = work_of(n).g, t0 = work_of(n).t0;
        nk = __shfl_sync(0xffffffffu, work_of(n).nk, 0);
        if (CLAIM && nk == 0 && lane == 0) pp_arrive(&ask);
        for (int i = 0; i < 2 * nk && ok; ++i) {
          // the scheduling warp has the time of the ring's tiles to find the next work; earlier, a CTA would hold
          // work that another one could begin
          if (CLAIM && i == max(0, 2 * nk - 3) && lane == 0) pp_arrive(&ask);
          if (pa.stall == kPpStallLast && blockIdx.x == 0 && n == 0 && i == 2 * nk - 2) {
            ok = false;
            break;
          }
          const int j = i >> 1, at = done + i, slot = at % S;
          const bool is_v = i & 1;
          const int k0 = it.v.tile(t0 + j) * kPpKeys;
          // lane n: the page of the n-th box, if any row of the CTA sees it
          int page = -1;
          const int p0 = k0 + lane * box;
          const bool any = lane < boxes && p0 < it.v.end && (p0 + box > it.v.lo || p0 < it.v.ns);
          if (any) page = paged_page(a.kv, seq, p0);
          const unsigned seen = __ballot_sync(0xffffffffu, any), good = __ballot_sync(0xffffffffu, page >= 0);
          if (at >= S) ok = pp_wait(&empty[slot], (unsigned)(at / S - 1) & 1u, &failed);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const bool partial =
              !(k0 + kPpKeys <= it.v.end && (k0 >= it.v.lo || k0 + kPpKeys <= it.v.ns)) || good != seen;
          unsigned char* dst = ring + slot * kPpTileBytes;
          if (lane == 0 && !is_v) {
            unsigned bad = 0;
            for (int n = 0; n < boxes; ++n)
              if (((seen & ~good) >> n) & 1u) bad |= ((1u << (box / 16)) - 1u) << (n * (box / 16));
            bad_rows[(at >> 1) & 7] = bad;
            if (bad) paged_flag(a.kv, QD_PAGED_BAD_PAGE);
          }
          if (!(is_v && partial)) {  // whole boxes (what they hold of hidden keys gives scores that are masked)
            if (lane == 0)
              asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc_smem(&full[slot])),
                           "r"(__popc(good) * box * 256)
                           : "memory");
            __syncwarp();
            if (page >= 0) {
              const int y = (page * kvh + g) * ps + (p0 & (ps - 1));
              unsigned char* d = dst + lane * box * 128;
              tma_load_2d(d, is_v ? &pa.tv : &pa.tk, 0, y, &full[slot]);
              tma_load_2d(d + kPpTileBytes / 2, is_v ? &pa.tv : &pa.tk, 64, y, &full[slot]);
            }
          } else {
            // V of a tile with hidden rows, by groups of 16: TMA copies a group that is wholly visible and, from
            // outside the tensor, the zeros of one that is wholly hidden; the rows of a group with both
            // are copied or cleared one by one. (Clearing after the copy, row by row, cost 33 of 158 us
            // where every row has a window: 5 ragged chunks of up to 1500 tokens.)
            const int g0 = k0 + 16 * lane, gpage = __shfl_sync(0xffffffffu, page, (16 * (lane & 7)) / box);
            bool all = lane < 8 && gpage >= 0, some = false;
            if (all) {
              some = g0 < it.v.end && (g0 + 16 > it.v.lo || g0 < it.v.ns);
              all = g0 + 16 <= it.v.end && (g0 >= it.v.lo || g0 + 16 <= it.v.ns);
            }
            const unsigned edge = __ballot_sync(0xffffffffu, some && !all);
            if (lane == 0)
              asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(tc_smem(&full[slot])),
                           "r"((8 - __popc(edge)) * 4096)
                           : "memory");
            __syncwarp();
            if (lane < 8 && !((edge >> lane) & 1u)) {
              const int y = all ? (gpage * kvh + g) * ps + (g0 & (ps - 1)) : -16;
              unsigned char* d = dst + lane * 16 * 128;
              tma_load_2d(d, &pa.tv16, 0, y, &full[slot]);
              tma_load_2d(d + kPpTileBytes / 2, &pa.tv16, 64, y, &full[slot]);
            }
            for (unsigned left = edge; left; left &= left - 1) {
              const int n = __ffs(left) - 1, q0 = k0 + 16 * n;
              const long long row = ((long long)__shfl_sync(0xffffffffu, gpage, n) * kvh + g) * ps + (q0 & (ps - 1));
              const char* src = static_cast<const char*>(a.kv.v) + row * 256 + (lane & 15) * 16;
              const unsigned d = tc_smem(dst) + ((lane & 15) >> 3) * (kPpTileBytes / 2) + n * 16 * 128;
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const int r = 2 * e + (lane >> 4);
                cp_async16(d + r * 128 + (((lane ^ r) & 7) << 4), src + r * 256, it.v.at(q0 + r));
              }
            }
            if (edge) {
              asm volatile("cp.async.wait_all;" ::: "memory");
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              __syncwarp();
            }
            if (lane == 0) pp_arrive(&full[slot]);
          }
          issued_to = at;
        }
        done += 2 * nk;
        work_done(n);
      }
      // nothing may still be landing when the CTA ends
      for (int i = max(0, issued_to - S + 1); i <= issued_to; ++i)
        (void)tc_mbar_wait(&full[i % S], (unsigned)(i / S) & 1u);
    } else if (warp == kPpSoftmax / 32) {
      // ---- MMA issue ----
      // The whole warp runs the loop, so that the descriptors are warp-uniform values, and one lane issues.
      // (Under `if (lane == 0)` each of the 16 products of a tile and its operands took 90 cycles to issue,
      // more than the 64 that it runs.)
      const unsigned id_s = pp_idesc<T>(false), id_o = pp_idesc<T>(true), leader = lane == 0;
      const unsigned long long dq = umma_desc_k_sw128(tc_smem(qs)), dk = umma_desc_k_sw128(tc_smem(ring));
      const unsigned long long dv = umma_desc_mn_sw128(tc_smem(ring));
      // S_t = Q_t K^T. The smallest part goes first: the accumulator drops bits towards zero at every step,
      // and that costs the less the smaller the sum still is (f32 results at 64 + 3500 keys: 2.0e-6 off
      // with the largest part first, 0.9e-6 so).
      auto scores = [&](int t, int slot) {
        const unsigned long long q0 = dq + (SHARED ? 0u : (unsigned)(t * (kQTile >> 4)));
        const unsigned long long k0 = dk + (unsigned)(slot * (kPpTileBytes >> 4));
#pragma unroll
        for (int part = 0; part < PARTS; ++part)
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const unsigned off = ((ks >> 2) * (kPpTileBytes / 2) + (ks & 3) * 32) >> 4;
            const unsigned qo = (PARTS - 1 - part) * (kPpTileBytes >> 4) + off;
            if (part == 0 && ks == 0) pp_mma_ss<false>(tmem + t * 128, q0 + qo, k0, id_s, leader);
            else pp_mma_ss<true>(tmem + t * 128, q0 + qo, k0 + off, id_s, leader);
          }
        pp_commit(&s_full[t], leader);
      };
      bool ok = true;
      unsigned turn = 0, q_turn = 0;  // bit t: parity of row tile t's barriers before this work (SHARED: works in q_turn)
      int done = 0;                   // ring slots of the works before
      for (int n = 0, nk = 0; ok && (CLAIM || n == 0); ++n) {
        ok = wait_work(n, nk);
        if (!ok) break;
        nk = __shfl_sync(0xffffffffu, work_of(n).nk, 0);
        const int halves = __shfl_sync(0xffffffffu, work_of(n).halves, 0);
        work_done(n);
        if (halves == 0) break;
        if (nk == 0) continue;
        auto ring_slot = [&](int i) { return (done + i) % S; };
        auto ring_phase = [&](int i) { return (unsigned)((done + i) / S) & 1u; };
        // O_t += P_t V for the n-th tile of row tile t
        auto product = [&](int t, int n, int slot) {
          const unsigned long long v0 = dv + (unsigned)(slot * (kPpTileBytes >> 4));
          const unsigned od = tmem + kColO + t * 128, pd = tmem + kColP + t * 128;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            ok = __all_sync(0xffffffffu,
                            pp_wait(half ? &p_full[t] : &p_half[t], (unsigned)(n ^ (turn >> t)) & 1u, &failed));
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int part = 0; part < kParts; ++part)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int ks = 2 * half + (i & 1) + 4 * (i >> 1);  // keys 0-31 and 64-95, then the others
                const unsigned po = (kParts - 1 - part) * 64 + ks * 8;
                if (half == 0 && part == 0 && i == 0)
                  pp_mma_ts(od, pd + po, v0, id_o, kMoves ? n % kFlush != 0 : n > 0, leader);
                else
                  pp_mma_ts(od, pd + po, v0 + ks * (2048 >> 4), id_o, true, leader);
              }
          }
        };
        if constexpr (SHARED) {
          auto landed = [&](int i) { return __all_sync(0xffffffffu, pp_wait(&full[ring_slot(i)], ring_phase(i), &failed)); };
          auto scores_of = [&](int j) {
            ok = ok && landed(2 * j);
            tc_fence_after();
            if (!ok) return;
            scores(j % kAlt, ring_slot(2 * j));
            pp_commit(&empty[ring_slot(2 * j)], leader);
          };
          ok = __all_sync(0xffffffffu, pp_wait(&q_full[q_turn & 1u], q_turn >> 1 & 1u, &failed));
          ++q_turn;
          for (int j = 0; j < halves; ++j) scores_of(j);
          for (int j = 0; j < nk && ok; ++j) {
            const int t = j % kAlt;
            ok = landed(2 * j + 1);
            if (ok) product(t, j / kAlt, ring_slot(2 * j + 1));
            if (!ok) break;
            pp_commit(&o_done[t], leader);
            pp_commit(&empty[ring_slot(2 * j + 1)], leader);
            if (j + kAlt < nk) scores_of(j + kAlt);
          }
          done += 2 * nk;
          for (int t = 0; t < kAlt; ++t)
            if ((nk + kAlt - 1 - t) / kAlt & 1) turn ^= 1u << t;
          continue;
        }
        ok = __all_sync(0xffffffffu, pp_wait(&full[ring_slot(0)], ring_phase(0), &failed));
        for (int t = 0; t < halves && ok; ++t) {
          ok = __all_sync(0xffffffffu, pp_wait(&q_full[t], (q_turn >> t) & 1u, &failed));
          tc_fence_after();
          if (ok) scores(t, ring_slot(0));
        }
        q_turn ^= halves == 2 ? 3u : 1u;
        if (ok) pp_commit(&empty[ring_slot(0)], leader);
        int vs = ring_slot(1), ks_slot = ring_slot(2);           // ring slots of V of tile j and K of tile j + 1,
        unsigned vph = ring_phase(1), kph = ring_phase(2);       // and their phases
        for (int j = 0; j < nk && ok; ++j) {
          ok = pp_wait(&full[vs], vph, &failed);
          if (j + 1 < nk) ok = pp_wait(&full[ks_slot], kph, &failed) && ok;
          ok = __all_sync(0xffffffffu, ok);
          for (int t = 0; t < halves && ok; ++t) {
            product(t, j, vs);
            if (!ok) break;
            pp_commit(&o_done[t], leader);
            if (t == halves - 1) pp_commit(&empty[vs], leader);
            if (j + 1 < nk) {
              scores(t, ks_slot);
              if (t == halves - 1) pp_commit(&empty[ks_slot], leader);
            }
          }
          vs += 2;
          if (vs >= S) vs -= S, vph ^= 1u;
          ks_slot += 2;
          if (ks_slot >= S) ks_slot -= S, kph ^= 1u;
        }
        done += 2 * nk;
        if (nk & 1) turn ^= halves == 2 ? 3u : 1u;
      }
      if (!ok) {  // given up: let what was issued finish before the CTA ends
        pp_commit(&drain, leader);
        (void)tc_mbar_wait(&drain, 0);
      }
    }
    tc_fence_before();
    __syncthreads();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPpRegsMany));
    // ---- softmax: half a row per thread ----
    const int t = (tid >> 8) & 1, hf = (tid >> 7) & 1, own = t * 128 + (tid & 127), lr = SHARED ? tid & 127 : own;
    const int pair = 1 + t * 4 + (warp & 3);  // named barrier of the two warps that share 32 rows
    int done = 0;       // key tiles of the works before
    int works = 0;      // those with any
    unsigned turn = 0;  // parity of this row tile's among them
    bool ok = true;  // (a warp that has given up still meets its partner at their barriers, where both end)
    for (int n = 0, nk = 0; CLAIM || n == 0; ++n) {
      if (CLAIM) {
        ok = ok && wait_work(n, nk);
        if (pp_any(pair, !ok)) break;
      }
      const PpItem it = work_of(n).it;
      const int item = work_of(n).item, g = work_of(n).g, z = work_of(n).z, parts = work_of(n).parts,
                t0 = work_of(n).t0, halves = __shfl_sync(0xffffffffu, work_of(n).halves, 0);
      nk = __shfl_sync(0xffffffffu, work_of(n).nk, 0);
      if (halves == 0) break;
      const int row = work_of(n).row0 + lr, tok = row / G, hs = row - tok * G;
      const bool live = lr < kRows && row < it.n_rows && (unsigned)(it.tok0 + tok) < (unsigned)a.rows;
      // key tiles of this set: all, or every other one
      const int mine_nk = kAlt == 2 ? (nk + 1 - t) >> 1 : nk;
      if (t < halves && nk > 0) {
        // Q: K-major with the 128-byte swizzle; dead rows are zero. A warp copies its 32 rows' 64 dims row by
        // row, neighbouring lanes on neighbouring chunks (a row per lane took 4.5 us of a busy GPU's
        // time). A negative scale changes the sign of q, so that the softmax always has a positive one.
        const int wr = (warp & 3) * 32;  // first of the warp's rows in its tile
        unsigned char* wq = qs + (SHARED ? 0 : t * kQTile) + hf * (kPpTileBytes / 2);
        const long long q_at =
            live ? (long long)(it.tok0 + tok) * a.q_stride + ((long long)g * G + hs) * kHeadDim + 64 * hf : -1;
        float c = fabsf(a.scale) * kLog2e;  // of the row's scores
        if (SHARED && t == 1) {
          // The other set brings the queries. It may end this work and bring the next one's before this set has looked
          // (of two key tiles it waits for its own only), so works have two barriers in turn; the work behind the
          // next is handed out when this one has been left.
          if (pa.stall == kPpStallLate) __nanosleep(40000);
          ok = ok && __all_sync(0xffffffffu, pp_wait(&q_full[works & 1], (unsigned)works >> 1 & 1u, &failed));
          if constexpr (PARTS == 2) c = fmaxf(c * f16_fit(q_exp[works & 1][wr + lane]).y, 1.0e-37f);
        } else {
        if constexpr (PARTS > 1) {
          const int c4 = lane & 15;
          constexpr int N = PARTS == 2 ? 16 : 8;
#pragma unroll
          for (int i0 = 0; i0 < 16; i0 += N) {
            float4 x[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const long long at = __shfl_sync(0xffffffffu, q_at, 2 * (i0 + i) + (lane >> 4));
              x[i] = at >= 0 ? load4<float>(a.q, at + 4 * c4) : make_float4(0.f, 0.f, 0.f, 0.f);
              if (a.scale < 0.0f) x[i] = make_float4(-x[i].x, -x[i].y, -x[i].z, -x[i].w);
            }
            if constexpr (PARTS == 2) {
              // Each row by its own power of two to where two f16 hold 22 bits of it (f16_fit). The largest of
              // a row's 64 dims, for the i-th pair of rows in lane i of each half; the partner warp has the others:
              // the two exponents go to the halves of the row's word.
              float top[16];
#pragma unroll
              for (int i = 0; i < 16; ++i)
                top[i] = fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w)));
#pragma unroll
              for (int o = 8; o > 0; o >>= 1)
#pragma unroll
                for (int i = 0; i < o; ++i) {
                  const float theirs = lane & o ? top[i] : top[i + o], ours = lane & o ? top[i + o] : top[i];
                  top[i] = fmaxf(ours, __shfl_xor_sync(0xffffffffu, theirs, o));
                }
              const unsigned* tops = reinterpret_cast<const unsigned*>(shared_row) + t * 128;
              reinterpret_cast<unsigned short*>(shared_row)[2 * (t * 128 + wr + 2 * c4 + (lane >> 4)) + hf] =
                  (unsigned short)(__float_as_int(top[0]) >> 23);
              pp_meet(pair);
              auto fit = [&](int r) { return f16_fit((int)max(tops[r] & 0xffffu, tops[r] >> 16)); };
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float up = fit(wr + 2 * i + (lane >> 4)).x;
                x[i] = make_float4(x[i].x * up, x[i].y * up, x[i].z * up, x[i].w * up);
              }
              c = fmaxf(c * fit(wr + lane).y, 1.0e-37f);  // (never 0: a hidden key's score is -inf)
              if (SHARED && hf == 0) {
                const unsigned both = tops[wr + lane];
                q_exp[works & 1][wr + lane] = (unsigned char)max(both & 0xffffu, both >> 16);
              }
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const int r = wr + 2 * (i0 + i) + (lane >> 4);
              unsigned u[2][PARTS];
              split_parts<T, PARTS>(x[i].x, x[i].y, u[0]);
              split_parts<T, PARTS>(x[i].z, x[i].w, u[1]);
              const unsigned off = r * 128 + ((((c4 >> 1) ^ r) & 7) << 4) + (c4 & 1) * 8;
#pragma unroll
              for (int part = 0; part < PARTS; ++part)
                *reinterpret_cast<uint2*>(wq + part * kPpTileBytes + off) = make_uint2(u[0][part], u[1][part]);
            }
          }
        } else {
          uint4 x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const long long at = __shfl_sync(0xffffffffu, q_at, 4 * i + (lane >> 3));
            x[i] = at >= 0 ? *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + at + 8 * (lane & 7))
                           : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (a.scale < 0.0f)
              x[i] = make_uint4(x[i].x ^ 0x80008000u, x[i].y ^ 0x80008000u, x[i].z ^ 0x80008000u, x[i].w ^ 0x80008000u);
            const int r = wr + 4 * i + (lane >> 3);
            *reinterpret_cast<uint4*>(wq + r * 128 + (((lane ^ r) & 7) << 4)) = x[i];
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        pp_arrive(&q_full[SHARED ? works & 1 : t]);
        }
        float m = -INFINITY, l = 0.0f;
        const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
        const unsigned ts = tmem + t * 128 + lanes, tp = tmem + kColP + t * 128 + 32 * hf + lanes;
        const unsigned to = tmem + kColO + t * 128 + 64 * hf + lanes;
        const int p = !live ? -1 : SHARED ? pp_shares(a, it.tok0 + tok) - 1 : it.pos0 + tok;
        const int pmax = min(p, it.len - 1);
        const int phi = a.window > 0 ? p - a.window : -2;  // keys up to here are hidden, unless sinks
        // positions of the warp's first and last live rows
        const unsigned lv = __ballot_sync(0xffffffffu, live);
        const int pw0 = SHARED ? __reduce_min_sync(0xffffffffu, p) : __shfl_sync(0xffffffffu, p, 0), pw1 = __shfl_sync(0xffffffffu, p, lv ? 31 - __clz(lv) : 0);
        const long long part0 = ((((long long)item * kvh + g) * pa.splits + z) * kAlt + (kAlt == 2 ? t : 0)) * kRows;
        float4* mine = pa.po + part0 * (kHeadDim / 4) + lr;
        float moved = -INFINITY;  // the maximum that the sums in the workspace go by
        for (int j = 0; j < mine_nk; ++j) {
          const int jt = kAlt == 2 ? 2 * j + t : j;  // of the work's tiles
          ok = ok && __all_sync(0xffffffffu, pp_wait(&s_full[t], (unsigned)(j ^ turn) & 1u, &failed));
          tc_fence_after();
          unsigned sr[64];
          tmem_ld64(ts + 64 * hf, sr);
          const int k0 = it.v.tile(t0 + jt) * kPpKeys;
          const unsigned bad = bad_rows[(done + jt) & 7];
          const bool inside = lv == 0xffffffffu && bad == 0 && k0 + kPpKeys - 1 <= min(pw0, it.len - 1) &&
                              (a.window == 0 || k0 > pw1 - a.window || k0 + kPpKeys <= a.sinks);
          if (!inside) {
            // bit i of a word: key at + i is visible to this row
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const int at = k0 + 64 * hf + 32 * w, b = bad >> (4 * hf + 2 * w);
              unsigned see = pp_below(pmax + 1 - at) & (~pp_below(phi + 1 - at) | pp_below(a.sinks - at));
              if (b & 1) see &= 0xffff0000u;
              if (b & 2) see &= 0x0000ffffu;
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!((see >> i) & 1u)) sr[32 * w + i] = 0xff800000u;
            }
          }
          float mx[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e] = __uint_as_float(sr[e]);
#pragma unroll
          for (int i = 4; i < 60; i += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(sr[i + e]), __uint_as_float(sr[i + 4 + e]));
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(sr[60 + e]), -INFINITY);
          float mt = max3(max3(mx[0], mx[1], mx[2]), mx[3], -INFINITY) * c;  // NaN where a score is
          // This barrier also stands between every read of S and the writes of P over it.
          if (pp_any(pair, !ok || mt > m + kPpLag)) {
            // The first thread's maximum to the second, the larger one back. (A NaN maximum moves nothing: its
            // row becomes NaN by its weights.)
            const float gone = __int_as_float(0x7fffffff);
            if (!(mt == mt)) mt = -INFINITY;
            if (hf == 0) shared_row[own] = ok ? mt : gone;
            pp_meet(pair);
            if (hf == 1) {
              const float other = shared_row[own];
              shared_row[own] = ok && other == other ? fmaxf(mt, other) : gone;
            }
            pp_meet(pair);
            mt = shared_row[own];
            ok = __all_sync(0xffffffffu, mt == mt);
            if (!ok) break;
            // each row by its own maximum (a factor of 1 where it has not moved), so that a row's result
            // does not depend on the rows beside it
            const float mn = mt > m + kPpLag ? mt : m;
            const float f = m == -INFINITY ? 0.0f : exp2_fast(m - mn);
            m = mn;
            l *= f;
            if (j > 0) {  // the product of the tile before must have reached O
              ok = __all_sync(0xffffffffu, pp_wait(&o_done[t], (unsigned)((j - 1) ^ turn) & 1u, &failed));
              tc_fence_after();
#pragma unroll 1
              for (int h = 0; h < 4; ++h) {
                unsigned o[16];
                tmem_ld16(to + 16 * h, o);
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                tmem_st16(to + 16 * h, o);
              }
            }
          }
          if (kMoves && j > 0 && j % kFlush == 0) {
            ok = ok && __all_sync(0xffffffffu, pp_wait(&o_done[t], (unsigned)((j - 1) ^ turn) & 1u, &failed));
            tc_fence_after();
            const float f = moved == -INFINITY ? 0.0f : exp2_fast(moved - m);
#pragma unroll 1
            for (int h = 0; h < 4; ++h) {
              unsigned o[16];
              tmem_ld16(to + 16 * h, o);
              float4* dst = mine + (16 * hf + 4 * h) * kRows;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float4 x = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                       __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
                if (j > kFlush) {
                  const float4 y = dst[i * kRows];
                  x = make_float4(fmaf(y.x, f, x.x), fmaf(y.y, f, x.y), fmaf(y.z, f, x.z), fmaf(y.w, f, x.w));
                }
                dst[i * kRows] = x;
              }
            }
            moved = m;
            tc_fence_before();
          }
          const float ref = m == -INFINITY ? 0.0f : kPpShift - m;
          float2 sum = make_float2(0.f, 0.f);
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // 32 keys: 16 packed columns
            unsigned w[kParts][16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float s0 = __uint_as_float(sr[32 * h + 2 * i]), s1 = __uint_as_float(sr[32 * h + 2 * i + 1]);
              float2 e = __ffma2_rn(make_float2(s0, s1), make_float2(c, c), make_float2(ref, ref));
              e = make_float2(exp2_fast(e.x), exp2_fast(e.y));
              sum = __fadd2_rn(sum, e);
              unsigned u[kParts];
              split_parts<T, kParts>(e.x, e.y, u);
#pragma unroll
              for (int part = 0; part < kParts; ++part) w[part][i] = u[part];
            }
#pragma unroll
            for (int part = 0; part < kParts; ++part) tmem_st16(tp + 64 * part + 16 * h, w[part]);
            if (h == 0) {  // the products of the first half of both threads' keys may start
              tmem_wait_st();
              tc_fence_before();
              if (ok) pp_arrive(&p_half[t]);
            }
          }
          l += sum.x + sum.y;
          tmem_wait_st();
          tc_fence_before();
          if (ok) pp_arrive(&p_full[t]);
        }
        pp_meet(pair);  // (the last maximum has been read)
        if (hf == 0) shared_row[own] = l;
        pp_meet(pair);
        if (hf == 1) shared_row[own] += l;
        pp_meet(pair);
        l = shared_row[own];
        if (ok) ok = __all_sync(0xffffffffu, pp_wait(&o_done[t], (unsigned)((mine_nk - 1) ^ turn) & 1u, &failed));
        if (ok) {
          tc_fence_after();
          const bool whole = !SHARED && parts == 1;
          const float f = whole ? inv_sum(l) : 1.0f;
          const long long y_at =
              live ? (long long)(it.tok0 + tok) * a.y_stride + ((long long)g * G + hs) * kHeadDim + 64 * hf : -1;
          if (!whole && hf == 0) pa.pml[part0 + lr] = make_float2(m, l);
          // Whole rows leave through the warp's part of Q's shared memory (every product that read it is done),
          // 32 dims at a time, so that neighbouring lanes write neighbouring chunks.
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            float o[32];
            tmem_ld32(to + 32 * h, o);
            if (kMoves && mine_nk > kFlush) {
              const float fm = moved == -INFINITY ? 0.0f : exp2_fast(moved - m);
              const float4* src = mine + (16 * hf + 8 * h) * kRows;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float4 y = src[i * kRows];
                o[4 * i] = fmaf(y.x, fm, o[4 * i]);
                o[4 * i + 1] = fmaf(y.y, fm, o[4 * i + 1]);
                o[4 * i + 2] = fmaf(y.z, fm, o[4 * i + 2]);
                o[4 * i + 3] = fmaf(y.w, fm, o[4 * i + 3]);
              }
            }
            if (!whole) {
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                mine[(16 * hf + 8 * h + i / 4) * kRows] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
              continue;
            }
            constexpr int kChunks = PARTS > 1 ? 8 : 4;  // 16-byte chunks of 32 dims
            unsigned char* my_row = wq + (wr + lane) * 128;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
              uint4 x;
              if constexpr (PARTS > 1)
                x = make_uint4(__float_as_uint(o[4 * c] * f), __float_as_uint(o[4 * c + 1] * f),
                               __float_as_uint(o[4 * c + 2] * f), __float_as_uint(o[4 * c + 3] * f));
              else
                x = make_uint4(pack2<T>(o[8 * c] * f, o[8 * c + 1] * f),
                               pack2<T>(o[8 * c + 2] * f, o[8 * c + 3] * f),
                               pack2<T>(o[8 * c + 4] * f, o[8 * c + 5] * f),
                               pack2<T>(o[8 * c + 6] * f, o[8 * c + 7] * f));
              *reinterpret_cast<uint4*>(my_row + (((c ^ lane) & 7) << 4)) = x;
            }
            __syncwarp();
            constexpr int kAtOnce = 32 / kChunks;  // rows a step of the warp writes
#pragma unroll
            for (int i = 0; i < 32 / kAtOnce; ++i) {
              const int r = i * kAtOnce + lane / kChunks, c = lane % kChunks;
              const long long at = __shfl_sync(0xffffffffu, y_at, r);
              const uint4 x = *reinterpret_cast<const uint4*>(wq + (wr + r) * 128 + (((c ^ r) & 7) << 4));
              if (at >= 0)
                *reinterpret_cast<uint4*>(static_cast<unsigned char*>(a.y) +
                                          (at + 32 * h) * (PARTS > 1 ? 4 : (int)sizeof(T)) + 16 * c) = x;
            }
            __syncwarp();
          }
        }
        tc_fence_before();
        turn ^= (unsigned)mine_nk;
      }
      done += nk;
      if (nk > 0) ++works;
      if (SHARED && live && t == 0 && hf == 0 && g == 0 && z == 0)
        pa.rows[(long long)(it.tok0 + tok) * G + hs] = place(work_of(n), lr);
      if (!SHARED && nk == 0 && live) {  // no key is visible to any row
        const long long base = (long long)(it.tok0 + tok) * a.y_stride + ((long long)g * G + hs) * kHeadDim + 64 * hf;
        for (int i = 0; i < kHeadDim / 2; i += 4) store4(a.y, base + i, a.dtype, make_float4(0.f, 0.f, 0.f, 0.f));
      }
      work_done(n);
    }
    tc_fence_before();
    __syncthreads();  // (the other roles' is at their end)
    if (failed) {
      // What this block held becomes NaN, so that nobody takes it for an answer. (Here, where the softmax threads'
      // registers are, and after the barrier, behind which no work is handed on any more.)
      if (tid == 0) paged_flag(a.kv, QD_PAGED_TIMEOUT);
      const float gone = __int_as_float(0x7fffffff);
#pragma unroll 1
      for (int i = 0; i < 3; ++i) {
        const PpWork& w = work[i];
        if (w.halves == 0) continue;
        const int n_rows = min(kRows, w.it.n_rows - w.row0);
#pragma unroll 1
        for (int e = tid; e < 32 * n_rows; e += kPpSoftmax) {
          const int lr = e >> 5, row = w.row0 + lr, tok = w.it.tok0 + row / G;
          if ((unsigned)tok >= (unsigned)a.rows) continue;
          // (and where the rows of a work are that was taken and not begun)
          if (SHARED && w.g == 0 && w.z == 0 && lane == 0) pa.rows[(long long)tok * G + row % G] = place(w, lr);
          if (SHARED || w.parts > 1)
            for (int x = 0; x < kAlt; ++x)
              pa.pml[((((long long)w.item * kvh + w.g) * pa.splits + w.z) * kAlt + x) * kRows + lr] = make_float2(gone, gone);
          else
            store4(a.y, (long long)tok * a.y_stride + ((long long)w.g * G + row % G) * kHeadDim + 4 * lane, a.dtype,
                   make_float4(gone, gone, gone, gone));
        }
      }
    }
  }
  if (warp == kPpSoftmax / 32) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// Adds the parts of rows whose key tiles were split. A CTA takes eight rows, a thread four dims of
// one; grid: items * kv_heads * cta_rows / 8.
__global__ void __launch_bounds__(256) k_paged_prompt_join(const __grid_constant__ PPromptArgs pa) {
  const PAttnArgs& a = pa.a;
  const int kvh = a.kv.kv_heads, G = a.q_heads / kvh, R = pa.cta_rows, per = R >> 3;
  const int r = (blockIdx.x % per) * 8 + (threadIdx.x & 7), d4 = threadIdx.x >> 3;
  const int ig = blockIdx.x / per, g = ig % kvh, item = ig / kvh;
  pdl_wait();
  pdl_trigger();
  int seq = 0, tile = 0, start = 0, fresh = 0, asked = 0;
  if (!pp_item(a, G, R, item, seq, tile, start, fresh, asked)) return;
  const PpItem it = pp_rows(a, G, R, tile, start, fresh, asked);
  const int parts = pp_parts(it.v.tiles, pa.splits), row = tile * R + r, tok = row / G;
  if (parts == 1 || row >= it.n_rows || (unsigned)(it.tok0 + tok) >= (unsigned)a.rows) return;
  const long long p0 = ((long long)item * kvh + g) * pa.splits * R;
  float M = -INFINITY;
  for (int k = 0; k < parts; ++k) M = fmaxf(M, pa.pml[p0 + k * R + r].x);
  float L = 0.0f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = 0; k < parts; ++k) {
    const float2 ml = pa.pml[p0 + k * R + r];
    const float4 x = pa.po[(p0 + (long long)k * R) * (kHeadDim / 4) + (long long)d4 * R + r];
    const float f = ml.x == -INFINITY ? 0.0f : exp2_fast(ml.x - M);
    L = fmaf(ml.y, f, L);
    y = make_float4(fmaf(x.x, f, y.x), fmaf(x.y, f, y.y), fmaf(x.z, f, y.z), fmaf(x.w, f, y.w));
  }
  const float zf = inv_sum(L);
  store4(a.y, (long long)(it.tok0 + tok) * a.y_stride + ((long long)g * G + row % G) * kHeadDim + 4 * d4, a.dtype,
         make_float4(y.x * zf, y.y * zf, y.z * zf, y.w * zf));
}

}  // namespace qd
