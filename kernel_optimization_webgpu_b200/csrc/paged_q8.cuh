// Operators over a paged cache of 8-bit integers: reading it back into 16-bit pages, and attention of one new
// token per sequence over it. (Writing it: k_paged_append with Q8.)
//
// Pools K, V: int8 [page][kv_head][page_size][128], scales f32 [page][kv_head][page_size]; an element stands for
// its integer times its row's scale.
#pragma once

#include "paged_prompt.cuh"

namespace qd {

struct PagedScales {
  const float* k;
  const float* v;
};

// Four 8-bit integers as f16, exactly: byte n + 128 under the exponent of 1024 is the f16 1152 + n. Pairs
// (0, 1) and (2, 3); the bytes come with their upper bit flipped.
__device__ __forceinline__ unsigned q8_half2(unsigned w, unsigned sel) {
  const unsigned u = __byte_perm(w, 0x64646464u, sel), bias = 0x64806480u;
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), *reinterpret_cast<const __half2*>(&bias));
  return *reinterpret_cast<const unsigned*>(&h);
}
constexpr unsigned kQ8Lo = 0x4140, kQ8Hi = 0x4342;

// ---- reading back ------------------------------------------------------------------------
struct ReadArgs {
  PagedArgs src, dst;  // dst: pools, pages and table
  PagedScales scale;
  const int* first;    // positions from first[b] on; NULL: all
  int dtype;           // of dst
};

__device__ __forceinline__ float4 q8_float4(unsigned w, float s) {
  const unsigned lo = q8_half2(w, kQ8Lo), hi = q8_half2(w, kQ8Hi);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return make_float4(a.x * s, a.y * s, b.x * s, b.y * s);
}
// A warp takes 16 positions (which one page holds) of one sequence and KV head, K and V: lane l the eight elements
// 8 (l % 16) of every other row, all sixteen loads before the first store. What it has to move bounds it (132 bytes
// of a row in, 256 out). Units are counted through a scan of the lengths, so that a table wider than they are costs
// nothing.
template <typename T>
__global__ void __launch_bounds__(kPdThreads) k_paged_read_q8(const __grid_constant__ ReadArgs a) {
  extern __shared__ int first[];
  const int tid = threadIdx.x, lane = tid & 31, B = a.src.batch, kvh = a.src.kv_heads;
  pdl_wait();
  pdl_trigger();
  auto end_of = [&](int b) { return min(paged_len(a.src, b), a.dst.table_width << a.dst.page_shift); };
  auto from = [&](int b) { return a.first ? max(a.first[b], 0) : 0; };
  struct Tiles { int tiles; };
  pd_units(B, first, [&](int b) {
    const int n = end_of(b), f = min(from(b), n);
    return Tiles{f < n ? (n + 15) / 16 - f / 16 : 0};
  });
  if (blockIdx.x == 0)
    for (int b = tid; b < B; b += kPdThreads)
      if (a.src.seq_lens[b] != end_of(b)) paged_flag(a.src, QD_PAGED_BAD_LENGTH);
  const long long units = (long long)first[B] * kvh;
  const int warps = gridDim.x * (kPdThreads / 32);
  for (long long u = blockIdx.x * (kPdThreads / 32) + (tid >> 5); u < units; u += warps) {
    int lo = 0, hi = B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((long long)first[mid] * kvh <= u) lo = mid;
      else hi = mid;
    }
    const int rest = (int)(u - (long long)first[lo] * kvh), tiles = first[lo + 1] - first[lo];
    const int g = rest / tiles, f = from(lo), end = end_of(lo), p0 = (f / 16 + rest % tiles) * 16;
    const int ps = paged_page(a.src, lo, p0), pd = paged_page(a.dst, lo, p0);
    if (ps < 0 || pd < 0) {
      if (lane == 0) paged_flag(a.src, QD_PAGED_BAD_PAGE);
      continue;
    }
    const long long rs = (((long long)ps * kvh + g) << a.src.page_shift) + (p0 & ((1 << a.src.page_shift) - 1));
    const long long rd = (((long long)pd * kvh + g) << a.dst.page_shift) + (p0 & ((1 << a.dst.page_shift) - 1));
    const int r0 = lane >> 4, c = lane & 15;
    // lane l: the scale of row l % 16, of K in the first half, of V in the second (rows of the page that no
    // sequence holds are memory too, and their values are not used)
    const float mine = (lane < 16 ? a.scale.k : a.scale.v)[rs + c];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const uint2* src = reinterpret_cast<const uint2*>(static_cast<const int8_t*>(x ? a.src.v : a.src.k) + rs * kHeadDim) + lane;
      uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(x ? a.dst.v : a.dst.k) + rd * kHeadDim) + lane;
      uint2 w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = src[i * 32];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int p = p0 + 2 * i + r0;
        const float s = __shfl_sync(0xffffffffu, mine, 16 * x + 2 * i + r0);
        const float4 y = q8_float4(w[i].x ^ 0x80808080u, s), z = q8_float4(w[i].y ^ 0x80808080u, s);
        if (p >= f && p < end)
          dst[i * 32] = make_uint4(pack2<T>(y.x, y.y), pack2<T>(y.z, y.w), pack2<T>(z.x, z.y), pack2<T>(z.z, z.w));
      }
    }
  }
}

// ---- attention of one new token per sequence ---------------------------------------------------
// As k_paged_decode (units in equal runs per CTA, a ring of copies per warp, parts joined by
// k_paged_decode_join), over half the bytes, which leaves instructions as the next bound, so:
//  - A warp takes 32 positions of a unit of 128. TMA copies them, 16 rows of one page at a time, with the swizzle
//    that the loads from shared memory want; one lane per 16 rows asks for them.
//  - The integers are exact in f16 and feed the products as they are (byte permutes and one subtraction per pair, in
//    registers). A K row's scale multiplies its scores, a V row's its weight: y = sum_j (p_j vs_j) n_j.
//  - mma.sync m16n8k16 with keys (dims of V) as the 16 rows and query heads as the 8 columns: four heads, each as a
//    column of its 16-bit part and one of the rest, which meet in one thread, so that nothing is
//    spent on the eight rows that two heads would leave empty the other way round (82 us for the 64 sequences below).
//    The contraction's index may have any order that both operands share: thread t of a quad takes dims 32 t .. + 31
//    of a K row (two 16-byte loads) and 16 consecutive dims of four positions of V. The weights'
//    fragments are those of the scores transposed (movmatrix).
//  - The weights p_j vs_j go into f16 parts, and a V row's scale may have any size beside its weight (the first
//    token's V is small in many models, and its weight large), so they have a running maximum of their own, of
//    s_j + log2 vs_j, next to that of s_j, by which the weights' sum goes.
// SETS: column sets of four heads; one for up to four query heads to a KV head, else two.
constexpr int kQ8Tile = 128, kQ8Stages = 2;
constexpr int kQ8Rows = 32;                 // positions of a warp
constexpr int kQ8Slot = 2 * kQ8Rows * 128;  // K and V
constexpr int kQ8Scales = 2 * kQ8Rows * 4;  // their scales
constexpr int kQ8PerSm = 3;                 // CTAs
static_assert(8 * kPdSumRow * 4 <= kQ8Slot, "a slot holds eight heads' sums");
__host__ __device__ constexpr int pq8_smem(int batch) {
  return 1024 + 4 * kQ8Stages * (kQ8Slot + kQ8Scales) + (batch + 1) * 4;
}

struct Q8Args {
  CUtensorMap tk, tv;  // boxes of 16 rows
  PAttnArgs a;
  PagedScales scale;
};

__device__ __forceinline__ float log2_fast(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint4 lds128(unsigned addr) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr));
  return r;
}
__device__ __forceinline__ float lds32f(unsigned addr) {
  float r;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ unsigned transpose_b16(unsigned x) {  // an 8 x 8 matrix over the warp
  unsigned y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int SETS>
__global__ void __launch_bounds__(kPdThreads, SETS == 1 ? kQ8PerSm : 2) k_paged_decode_q8(const __grid_constant__ Q8Args qa,
                                                                                       void* workspace) {
  const PAttnArgs& a = qa.a;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  unsigned char* ring = smem + warp * kQ8Stages * kQ8Slot;
  unsigned char* scales = smem + 4 * kQ8Stages * kQ8Slot + warp * kQ8Stages * kQ8Scales;
  int* first = reinterpret_cast<int*>(smem + 4 * kQ8Stages * (kQ8Slot + kQ8Scales));
  __shared__ unsigned long long full[4][kQ8Stages];
  __shared__ float2 sml[4][8];  // maximum and sum of weights of each warp and head,
  __shared__ float smo[4][8];   // the maximum that its sums go by
  const int G = a.q_heads / a.kv.kv_heads, subs = (G + 7) >> 3, nh = a.kv.kv_heads * subs, B = a.kv.batch;
  const PDecodeWs ws = pd_ws(workspace);
  if (tid == 0) {
    tma_prefetch_map(&qa.tk);
    tma_prefetch_map(&qa.tv);
    for (int i = 0; i < 4 * kQ8Stages; ++i) tc_mbar_init(&full[0][0] + i);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  pdl_trigger();
  auto see = [&](int b) { return visible<kQ8Tile>(a.kv.seq_lens[b], paged_len(a.kv, b), a.window, a.sinks); };
  pd_units(B, first, see);  // (its barriers are the mbarriers' too)
  if (blockIdx.x == 0) {
    for (int b = tid; b <= B; b += kPdThreads) ws.first[b] = first[b];
    for (int b = tid; b < B; b += kPdThreads)  // (paged_len cuts both)
      if (a.kv.seq_lens[b] != paged_len(a.kv, b)) paged_flag(a.kv, QD_PAGED_BAD_LENGTH);
  }
  for (int b = blockIdx.x; b < B; b += gridDim.x)  // nothing visible: zeros
    if (first[b + 1] == first[b])
      for (int i = tid; i < a.q_heads * kHeadDim; i += kPdThreads) store1(a.y, b * a.y_stride + i, a.dtype, 0.0f);
  const long long U = (long long)first[B] * nh;
  const int ctas = (int)min((long long)gridDim.x, U);  // none of them empty
  if ((int)blockIdx.x >= ctas) return;
  const int u0 = (int)(U * blockIdx.x / ctas), u1 = (int)(U * (blockIdx.x + 1) / ctas);
  auto step = [&](PdCursor& c) { pd_step(c, first, a.kv.kv_heads, subs, see); };
  PdCursor cur = pd_place(B, first, nh, subs, u0, see);
  PdCursor pre = cur;  // the copies run ahead of the sums
  const int n_units = u1 - u0;

  // page of the 16 positions that this half of the warp asks for of the unit at `pre`; -1: nothing visible there, -2: bad
  auto page_of = [&](const PdCursor& c) {
    const int p0 = c.v.tile(c.t) * kQ8Tile + kQ8Rows * warp + (lane & 16);
    const bool any = p0 < c.v.end && (p0 + 16 > c.v.lo || p0 < c.v.ns);
    if (!any) return -1;
    const int page = paged_page(a.kv, c.b, p0);
    return page < 0 ? -2 : page;
  };
  int next_page = page_of(pre);
  unsigned live_ring = 0;  // bits 2 i, 2 i + 1: the halves of slot i hold rows
  unsigned phases = 0;     // bit i: parity of slot i's barrier
  int issued = 0, in_slot = 0;
  bool gone = false;  // a copy has not come in time
  auto issue = [&]() {
    if (issued >= n_units || gone) return;
    const int page = next_page;
    const unsigned good = __ballot_sync(0xffffffffu, page >= 0);
    const unsigned halves = (good & 1u) | (good >> 16 & 1u) << 1;
    live_ring = (live_ring & ~(3u << (2 * in_slot))) | halves << (2 * in_slot);
    if (page == -2 && (lane & 15) == 0) paged_flag(a.kv, QD_PAGED_BAD_PAGE);
    unsigned long long* bar = &full[warp][in_slot];
    if (lane == 0 && halves)
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc_smem(bar)),
                   "r"((halves == 3u ? 2 : 1) * (2 * 16 * 128 + 2 * 16 * 4))
                   : "memory");
    __syncwarp();
    if ((lane & 15) == 0 && page >= 0) {
      const int p0 = pre.v.tile(pre.t) * kQ8Tile + kQ8Rows * warp + lane;
      const int row = ((page * a.kv.kv_heads + pre.g) << a.kv.page_shift) + (p0 & ((1 << a.kv.page_shift) - 1));
      unsigned char* d = ring + in_slot * kQ8Slot + lane * 128;
      unsigned char* s = scales + in_slot * kQ8Scales + lane * 4;
      tma_load_2d(d, &qa.tk, 0, row, bar);
      tma_load_2d(d + kQ8Rows * 128, &qa.tv, 0, row, bar);
      bulk_load(s, qa.scale.k + row, 64, bar);
      bulk_load(s + kQ8Rows * 4, qa.scale.v + row, 64, bar);
    }
    ++issued;
    in_slot = in_slot + 1 == kQ8Stages ? 0 : in_slot + 1;
    if (issued < n_units) {
      step(pre);
      next_page = page_of(pre);
    }
  };
#pragma unroll
  for (int i = 0; i < kQ8Stages - 1; ++i) issue();

  // The queries of a (sequence, head): lane l has column l / 4 of the products (of set s head 4 s + l / 8, its 16-bit part
  // or the rest), dims 32 (l % 4) .. + 31; the scores and sums of head 4 s + l % 4.
  const float qs = a.scale * kLog2e;
  const int t4 = lane & 3, g8 = lane >> 2;
  unsigned q[SETS][8][2];
  float o[SETS][8][4], m[SETS], mo[SETS], l[SETS], factor[SETS];
  bool fresh = true;  // a new (sequence, head): take its q, clear the sums
  int seg = 0;        // segments finished by this CTA
  bool from_start = cur.t == 0;
  int slot = 0;
  for (int i = 0; i < n_units; ++i) {
    issue();
    if (fresh) {
      fresh = false;
#pragma unroll
      for (int n = 0; n < SETS; ++n) {
        const int hs = cur.sub * 8 + 4 * n + (g8 >> 1);
        const bool live = hs < G;
        const long long base = cur.b * a.q_stride + ((long long)cur.g * G + (live ? hs : 0)) * kHeadDim + 32 * t4;
        float2 x[16];
        float top = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; ++k) x[k] = load2(a.q, base + 2 * k, a.dtype);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          if (!live) x[k] = make_float2(0.f, 0.f);
          top = fmaxf(top, fmaxf(fabsf(x[k].x), fabsf(x[k].y)));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float2 fit = f16_fit(__float_as_int(top) >> 23);
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            unsigned hi, lo;
            split2<__half>(x[2 * k + e].x * fit.x, x[2 * k + e].y * fit.x, hi, lo);
            q[n][k][e] = g8 & 1 ? lo : hi;
          }
        factor[n] = qs * __shfl_sync(0xffffffffu, fit.y, 8 * t4);  // of head t4: columns 2 t4, 2 t4 + 1
#pragma unroll
        for (int j = 0; j < 8; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.0f;
        m[n] = mo[n] = -INFINITY;
        l[n] = 0.0f;
      }
    }
    const bool last_t = cur.t + 1 == cur.v.tiles, more = i + 1 < n_units;
    unsigned halves = live_ring >> (2 * slot) & 3u;
    if (halves && !gone) {
      gone = !__all_sync(0xffffffffu, tc_mbar_wait(&full[warp][slot], phases >> slot & 1u));
      if (gone) {
        if (lane == 0) paged_flag(a.kv, QD_PAGED_TIMEOUT);
      } else {
        phases ^= 1u << slot;
        live_ring &= ~(3u << (2 * slot));
      }
    }
    if (gone) {  // what this warp held becomes NaN
      halves = 0;
#pragma unroll
      for (int n = 0; n < SETS; ++n) l[n] = __int_as_float(0x7fffffff);
    }
    if (halves) {
      const unsigned kb = tc_smem(ring) + slot * kQ8Slot, vb = kb + kQ8Rows * 128;
      const unsigned sb = tc_smem(scales) + slot * kQ8Scales + g8 * 4;
      const int p0 = cur.v.tile(cur.t) * kQ8Tile + kQ8Rows * warp;
      const bool inside = halves == 3u && p0 + 32 <= cur.v.end && (p0 >= cur.v.lo || p0 + 32 <= cur.v.ns);
      float p[SETS][4], u[SETS][4];  // of positions 8 j + g8: scores, and with V's scale
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float s[SETS][2][4];
#pragma unroll
        for (int n = 0; n < SETS; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) s[n][e][0] = s[n][e][1] = s[n][e][2] = s[n][e][3] = 0.0f;
        const unsigned row = kb + (16 * h + g8) * 128;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const unsigned at = row + (((2 * t4 + c) ^ g8) << 4);
          const uint4 x = lds128(at), y = lds128(at + 1024);
          const unsigned xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const unsigned v = xw[k] ^ 0x80808080u, w = yw[k] ^ 0x80808080u;
            const unsigned f[4] = {q8_half2(v, kQ8Lo), q8_half2(w, kQ8Lo), q8_half2(v, kQ8Hi), q8_half2(w, kQ8Hi)};
#pragma unroll
            for (int n = 0; n < SETS; ++n) mma_16816<__half>(s[n][k & 1], f, q[n][4 * c + k][0], q[n][4 * c + k][1]);
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = 2 * h + e;
          const float ks = lds32f(sb + 32 * j), lv = log2_fast(lds32f(sb + 32 * j + kQ8Rows * 4));
#pragma unroll
          for (int n = 0; n < SETS; ++n) {
            p[n][j] = ((s[n][0][2 * e] + s[n][1][2 * e]) + (s[n][0][2 * e + 1] + s[n][1][2 * e + 1])) * (factor[n] * ks);
            u[n][j] = p[n][j] + lv;
          }
        }
      }
      if (!inside) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (!(halves >> (j >> 1) & 1u) || !cur.v.at(p0 + 8 * j + g8))
#pragma unroll
            for (int n = 0; n < SETS; ++n) p[n][j] = u[n][j] = -INFINITY;
      }
#pragma unroll
      for (int n = 0; n < SETS; ++n) {
        float mt = fmaxf(fmaxf(p[n][0], p[n][1]), fmaxf(p[n][2], p[n][3]));
        float ut = fmaxf(fmaxf(u[n][0], u[n][1]), fmaxf(u[n][2], u[n][3]));
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, x));
          ut = fmaxf(ut, __shfl_xor_sync(0xffffffffu, ut, x));
        }
        if (__any_sync(0xffffffffu, mt > m[n] + kPdLag || ut > mo[n] + kPdLag)) {  // some head's maximum moved: rescale
          const float mn = mt > m[n] + kPdLag ? mt : m[n], un = ut > mo[n] + kPdLag ? ut : mo[n];
          l[n] *= m[n] == -INFINITY ? 0.0f : exp2_fast(m[n] - mn);
          const float f = mo[n] == -INFINITY ? 0.0f : exp2_fast(mo[n] - un);
          m[n] = mn;
          mo[n] = un;
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][j][e] *= f;
        }
        const float ref = m[n] == -INFINITY ? 0.0f : m[n], uref = mo[n] == -INFINITY ? 0.0f : mo[n] - kPdShift;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          l[n] += exp2_fast(p[n][j] - ref);
          u[n][j] = exp2_fast(u[n][j] - uref);
        }
      }
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        unsigned w[SETS][2];
#pragma unroll
        for (int n = 0; n < SETS; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {  // a weight as its 16-bit part and the rest, for the columns of its head
            const float x = u[n][2 * st + e];
            const float hi = __half2float(__float2half_rn(x));
            w[n][e] = transpose_b16(pack2<__half>(hi, x - hi));
          }
        // rows 16 st + 2 t + {0, 1, 8, 9}, chunk g8
        const unsigned row = vb + (16 * st + 2 * t4) * 128, c0 = (g8 ^ (2 * t4)) << 4, c1 = (g8 ^ (2 * t4 + 1)) << 4;
        const uint4 x0 = lds128(row + c0), x1 = lds128(row + 128 + c1);
        const uint4 x2 = lds128(row + 1024 + c0), x3 = lds128(row + 1152 + c1);
        const unsigned va[4] = {x0.x, x0.y, x0.z, x0.w}, vc[4] = {x1.x, x1.y, x1.z, x1.w};
        const unsigned vd[4] = {x2.x, x2.y, x2.z, x2.w}, ve[4] = {x3.x, x3.y, x3.z, x3.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const unsigned a0 = __byte_perm(va[k], vc[k], 0x5140) ^ 0x80808080u, a1 = __byte_perm(va[k], vc[k], 0x7362) ^ 0x80808080u;
          const unsigned b0 = __byte_perm(vd[k], ve[k], 0x5140) ^ 0x80808080u, b1 = __byte_perm(vd[k], ve[k], 0x7362) ^ 0x80808080u;
          const unsigned f[4] = {q8_half2(a0, kQ8Lo), q8_half2(a0, kQ8Hi), q8_half2(b0, kQ8Lo), q8_half2(b0, kQ8Hi)};
          const unsigned f2[4] = {q8_half2(a1, kQ8Lo), q8_half2(a1, kQ8Hi), q8_half2(b1, kQ8Lo), q8_half2(b1, kQ8Hi)};
#pragma unroll
          for (int n = 0; n < SETS; ++n) {
            mma_16816<__half>(o[n][2 * k], f, w[n][0], w[n][1]);
            mma_16816<__half>(o[n][2 * k + 1], f2, w[n][0], w[n][1]);
          }
        }
      }
    }
    __syncwarp();  // the slot may be refilled
    if (last_t || !more) {
      // The (sequence, head), or this CTA's part of it, ends: join the four warps. The sums go to the slot that has
      // just been read: dims 16 g8 .. + 15 of head t4 of each set.
#pragma unroll
      for (int n = 0; n < SETS; ++n) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[n] += __shfl_xor_sync(0xffffffffu, l[n], x);
        float* mine = reinterpret_cast<float*>(ring + slot * kQ8Slot) + (4 * n + t4) * kPdSumRow + 16 * g8;
#pragma unroll
        for (int j = 0; j < 8; j += 2)
          *reinterpret_cast<float4*>(mine + 2 * j) = make_float4(o[n][j][0] + o[n][j][1], o[n][j][2] + o[n][j][3],
                                                                 o[n][j + 1][0] + o[n][j + 1][1], o[n][j + 1][2] + o[n][j + 1][3]);
        if (g8 == 0) {
          sml[warp][4 * n + t4] = make_float2(m[n], l[n]);
          smo[warp][4 * n + t4] = mo[n];
        }
      }
      __syncthreads();
      const int live = min(8, G - cur.sub * 8);
      const bool whole = from_start && last_t;
      const long long out = cur.b * a.y_stride + ((long long)cur.g * G + cur.sub * 8) * kHeadDim + tid;
      const long long part = (2ll * blockIdx.x + (seg ? 1 : 0)) * 8;
      for (int h = 0; h < live; ++h) {  // thread tid: dim tid
        const float M = fmaxf(fmaxf(sml[0][h].x, sml[1][h].x), fmaxf(sml[2][h].x, sml[3][h].x));
        float L = 0.0f, x = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          L += sml[w][h].y * (sml[w][h].x == -INFINITY ? 0.0f : exp2_fast(sml[w][h].x - M));  // (NaN stays)
          const float f = smo[w][h] == -INFINITY ? 0.0f : exp2_fast(smo[w][h] - kPdShift - M);
          x += reinterpret_cast<const float*>(smem + (w * kQ8Stages + slot) * kQ8Slot)[h * kPdSumRow + tid] * f;
        }
        if (whole) {
          store1(a.y, out + h * kHeadDim, a.dtype, x * inv_sum(L));
        } else {
          ws.o[(part + h) * kHeadDim + tid] = x;
          if (tid == 0) ws.ml[part + h] = make_float2(M, L);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncthreads();  // before the slots are refilled
      ++seg;
      fresh = true;
      from_start = true;
    }
    if (more) step(cur);
    slot = slot + 1 == kQ8Stages ? 0 : slot + 1;
  }
  if (gone)  // nothing may still be landing when the CTA ends
    for (int i = 0; i < kQ8Stages; ++i)
      if (live_ring >> (2 * i) & 3u) (void)tc_mbar_wait(&full[warp][i], phases >> i & 1u);
}

}  // namespace qd
