// Attention of one new token per sequence over a paged cache, split over the cache's length.
//
// y = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = scale q.k_j, over the visible keys. Each
// key is read once and takes part in 4 * 128 flops per query head that shares it, far below
// what the tensor cores do per byte: the kernel is bound by the bytes of K and V, so the
// design is about keeping copies in flight on every SM from the first cycle to the last.
//
//  - Work is cut into units of 64 positions of one (sequence, KV head), and the flat list of all
//    units into one run of equal length per CTA, whatever the lengths of the sequences. A run
//    crosses from one sequence to the next without draining its copies. A (sequence, head) that
//    one CTA holds whole is written by it; the others leave partial sums (at most two per CTA),
//    which k_paged_decode_join adds in the order of the CTAs: no atomics, the same bits each time.
//  - Warp w of a CTA owns positions 16w .. 16w+15 of every unit: its own ring of kPdStages slots
//    filled by cp.async, its own running maximum and sum. No CTA barrier until a (sequence, head)
//    ends. 16 positions lie in one page, so a slot needs one table entry, loaded a unit ahead.
//    Rows that are not visible are filled with zeros instead of being read.
//  - Products on mma.sync m16n8k16, 16 rows = up to 8 query heads twice: rows 0-7 hold the
//    operand rounded to 16 bits, rows 8-15 what that rounding left. The two sums of a head meet
//    in one thread (accumulator rows r and r + 8), so q and the weights keep twice 16 bits'
//    precision at no extra instruction. (tcgen05 wants 64 rows or more; 56 of them would idle.)
//    Two bf16 hold only 16 of f32's 24 bits (results were 5e-6 off): with f32 queries on a bf16
//    cache a second set of products takes the rest of both operands (THREE).
//    Two f16 hold 22 bits of what lies well inside f16's range: each head's q is brought there by a
//    power of two, which its scores' factor takes back (f16_fit).
//
// 64 sequences of 2048 positions, 8 KV heads: 93 us for 537 MB = 5.8 TB/s; of 8192: 338 us = 6.35 TB/s.
// About 10 us of either are the two launches and the chain of lookups before the first row (lengths,
// table, row), which is why 1 x 32768 (134 MB) takes 32 us. Three slots and two CTAs an SM; two
// slots and three CTAs: 112 us.
#pragma once

#include <type_traits>

#include "paged.cuh"

namespace qd {

constexpr int kPdThreads = 128;
constexpr int kPdTile = 64;          // positions per unit
constexpr int kPdStages = 3;
constexpr int kPdSlot = 2 * 16 * 256;  // K and V rows of 16 positions
constexpr int kPdMaxCtas = 320;
constexpr float kPdLag = 8.0f;       // log2 a running maximum may fall behind before the sums are rescaled
constexpr float kPdShift = 7.0f;     // weights are kept times 2^7: with the lag below 2^15 < 65504, and small
                                     // weights stay in f16's normal range down to 2^-21 of the largest
constexpr float kLog2e = 1.4426950408889634f;

struct PDecodeWs {
  float* o;      // [2 * ctas][8][128]
  float2* ml;    // [2 * ctas][8]
  int* first;    // [batch + 1]: units of the sequences before b, one KV head's
};
__host__ __device__ inline size_t pd_ws_bytes(int batch) {
  return (size_t)2 * kPdMaxCtas * 8 * (kHeadDim * 4 + 8) + (size_t)(batch + 1) * 4 + 256;
}
__host__ __device__ inline PDecodeWs pd_ws(void* p) {
  PDecodeWs w;
  w.o = static_cast<float*>(p);
  w.ml = reinterpret_cast<float2*>(w.o + (size_t)2 * kPdMaxCtas * 8 * kHeadDim);
  w.first = reinterpret_cast<int*>(w.ml + (size_t)2 * kPdMaxCtas * 8);
  return w;
}

// The visible positions of a query at position asked - 1: [0, ns) and [lo, end), in tiles of
// TILE positions: st of the sinks, then from w0 on.
struct Visible {
  int end, lo, ns, st, w0, tiles;
  __device__ __forceinline__ bool at(int pos) const { return pos < end && (pos >= lo || pos < ns); }
  __device__ __forceinline__ int tile(int i) const { return i < st ? i : w0 + (i - st); }
};
template <int TILE>
__device__ __forceinline__ Visible visible(int asked, int len, int window, int sinks) {
  Visible v;
  v.end = len;
  v.lo = window > 0 ? max(0, asked - window) : 0;
  v.ns = min(min(sinks, v.lo), v.end);
  v.st = (v.ns + TILE - 1) / TILE;
  v.w0 = max(v.lo / TILE, v.st);
  v.tiles = v.st + max(0, (v.end + TILE - 1) / TILE - v.w0);
  return v;
}

__device__ __forceinline__ void cp_async16(unsigned dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1);
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&d)[4], const unsigned (&a)[4], unsigned b0,
                                                         unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(unsigned addr, unsigned (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(unsigned addr, unsigned (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// hi = the pair rounded to 16 bits, lo = the rest, rounded again.
template <typename T>
__device__ __forceinline__ void split2(float x, float y, unsigned& hi, unsigned& lo);
template <>
__device__ __forceinline__ void split2<__half>(float x, float y, unsigned& hi, unsigned& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const unsigned*>(&h);
  lo = *reinterpret_cast<const unsigned*>(&l);
}
template <>
__device__ __forceinline__ void split2<__nv_bfloat16>(float x, float y, unsigned& hi, unsigned& lo) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  const float2 f = __bfloat1622float2(h);
  const __nv_bfloat162 l = __floats2bfloat162_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const unsigned*>(&h);
  lo = *reinterpret_cast<const unsigned*>(&l);
}
// The pair rounded to 16 bits, and the rest.
template <typename T>
__device__ __forceinline__ float2 split2_rest(float x, float y, unsigned& hi) {
  unsigned lo;
  split2<T>(x, y, hi, lo);
  const float2 f = std::is_same<T, __half>::value
                       ? __half22float2(*reinterpret_cast<const __half2*>(&hi))
                       : make_float2(__uint_as_float(hi << 16), __uint_as_float(hi & 0xffff0000u));
  return make_float2(x - f.x, y - f.y);
}
// The power of two that brings values whose largest has the (biased) exponent e into f16's upper range (the
// largest to 2^13 .. 2^14), so that the second of two f16 parts keeps its bits, and its inverse.
__device__ __forceinline__ float2 f16_fit(int e) {
  e = min(max(e, 14), 254);  // (an infinity stays one, zeros stay zeros)
  return make_float2(__int_as_float((267 - e) << 23), __int_as_float((e - 13) << 23));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float2 load2(const void* p, long long e, int dtype) {
  if (dtype == QD_KV_F32) return *reinterpret_cast<const float2*>(static_cast<const float*>(p) + e);
  const unsigned u = *reinterpret_cast<const unsigned*>(static_cast<const __half*>(p) + e);
  if (dtype == QD_KV_F16) return __half22float2(*reinterpret_cast<const __half2*>(&u));
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ void store1(void* p, long long e, int dtype, float x) {
  if (dtype == QD_KV_F32) static_cast<float*>(p)[e] = x;
  else if (dtype == QD_KV_F16) static_cast<__half*>(p)[e] = __float2half_rn(x);
  else static_cast<__nv_bfloat16*>(p)[e] = __float2bfloat16_rn(x);
}

// Sum times the reciprocal of its weights; nothing seen gives zero.
__device__ __forceinline__ float inv_sum(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

// A place in the flat list of units: unit t of sequence b, KV head g, and the sub-th eight of its
// query heads.
struct PdCursor {
  int b, g, sub, t;
  Visible v;
};

// Dynamic shared memory: 4 rings | units before each sequence. Where a (sequence, head) ends, each
// warp's sums go to the ring slot it has just read, rows kPdSumRow floats apart (8 heads on
// distinct banks).
constexpr int kPdSumRow = 136;
static_assert(8 * kPdSumRow * 4 <= kPdSlot, "a slot holds eight heads' sums");
__host__ __device__ constexpr int pd_smem(int batch) { return 4 * kPdStages * kPdSlot + (batch + 1) * 4; }

template <typename T, bool THREE>
__global__ void __launch_bounds__(kPdThreads) k_paged_decode(const __grid_constant__ PAttnArgs a, void* workspace) {
  extern __shared__ __align__(128) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned char* ring = smem + warp * kPdStages * kPdSlot;
  int* first = reinterpret_cast<int*>(smem + 4 * kPdStages * kPdSlot);
  __shared__ float2 sml[4][8];  // maximum and sum of each warp and head
  const int G = a.q_heads / a.kv.kv_heads, subs = (G + 7) >> 3, nh = a.kv.kv_heads * subs, B = a.kv.batch;
  const PDecodeWs ws = pd_ws(workspace);
  pdl_wait();
  pdl_trigger();

  // units before each sequence (an exclusive scan of the tile counts)
  {
    __shared__ int wsum[4];
    const int per = (B + kPdThreads - 1) / kPdThreads;
    const int b0 = min(tid * per, B), b1 = min(b0 + per, B);
    int n = 0;
    for (int b = b0; b < b1; ++b) {
      const int t = visible<kPdTile>(a.kv.seq_lens[b], paged_len(a.kv, b), a.window, a.sinks).tiles;
      first[b] = t;
      n += t;
    }
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    int at = incl - n;
    for (int w = 0; w < warp; ++w) at += wsum[w];
    for (int b = b0; b < b1; ++b) {
      const int t = first[b];
      first[b] = at;
      at += t;
    }
    if (tid == kPdThreads - 1) first[B] = wsum[0] + wsum[1] + wsum[2] + wsum[3];
    __syncthreads();
  }
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

  auto see = [&](PdCursor& c) {
    c.v = visible<kPdTile>(a.kv.seq_lens[c.b], paged_len(a.kv, c.b), a.window, a.sinks);
  };
  auto step = [&](PdCursor& c) {  // to the next unit (there is one)
    if (++c.t < c.v.tiles) return;
    c.t = 0;
    if (++c.sub < subs) return;
    c.sub = 0;
    if (++c.g < a.kv.kv_heads) return;
    c.g = 0;
    do ++c.b;
    while (first[c.b + 1] == first[c.b]);
    see(c);
  };
  PdCursor cur;
  {
    int lo = 0, hi = B;  // the last sequence whose units start at or before u0
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((long long)first[mid] * nh <= u0) lo = mid;
      else hi = mid;
    }
    cur.b = lo;
    see(cur);
    const int rest = u0 - first[lo] * nh;
    const int h = rest / cur.v.tiles;
    cur.t = rest - h * cur.v.tiles;
    cur.g = h / subs;
    cur.sub = h - cur.g * subs;
  }
  PdCursor pre = cur;  // the copies run ahead of the sums
  const int n_units = u1 - u0;

  // page of this warp's 16 positions of the unit at `pre`; -1: nothing visible there, -2: bad
  auto page_of = [&](const PdCursor& c) {
    const int p0 = c.v.tile(c.t) * kPdTile + 16 * warp;
    const bool any = p0 < c.v.end && (p0 + 16 > c.v.lo || p0 < c.v.ns);
    if (!any) return -1;
    const int page = paged_page(a.kv, c.b, p0);
    return page < 0 ? -2 : page;
  };
  int next_page = page_of(pre);
  unsigned live_ring = 0;  // bit i: slot i holds rows
  int issued = 0, in_slot = 0;
  const int pmask = (1 << a.kv.page_shift) - 1;
  const unsigned ring_s = (unsigned)__cvta_generic_to_shared(ring);
  // lane -> 16-byte chunk lane % 16 of rows 2i + lane / 16; chunk c of row r sits at c ^ (r % 8)
  unsigned to[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 2 * i + (lane >> 4);
    to[i] = ring_s + r * 256 + (((lane & 15) ^ r) << 4);
  }
  auto issue = [&]() {
    if (issued < n_units) {
      const int page = next_page;
      live_ring &= ~(1u << in_slot);
      if (page >= 0) {
        const int p0 = pre.v.tile(pre.t) * kPdTile + 16 * warp;
        const long long row0 = (((long long)page * a.kv.kv_heads + pre.g) << a.kv.page_shift) + (p0 & pmask);
        const char* ks = static_cast<const char*>(a.kv.k) + row0 * 256 + lane * 16;
        const char* vs = static_cast<const char*>(a.kv.v) + row0 * 256 + lane * 16;
        const unsigned dst = in_slot * kPdSlot;
        const bool all = p0 + 16 <= pre.v.end && (p0 >= pre.v.lo || p0 + 16 <= pre.v.ns);
        if (all) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            cp_async16(to[i & 3] + dst + (i >> 2) * 2048, ks + i * 512, true);
            cp_async16(to[i & 3] + dst + (i >> 2) * 2048 + 4096, vs + i * 512, true);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const bool ok = pre.v.at(p0 + 2 * i + (lane >> 4));
            cp_async16(to[i & 3] + dst + (i >> 2) * 2048, ks + i * 512, ok);
            cp_async16(to[i & 3] + dst + (i >> 2) * 2048 + 4096, vs + i * 512, ok);
          }
        }
        live_ring |= 1u << in_slot;
      } else if (page == -2 && lane == 0) {
        paged_flag(a.kv, QD_PAGED_BAD_PAGE);
      }
      ++issued;
      in_slot = in_slot + 1 == kPdStages ? 0 : in_slot + 1;
      if (issued < n_units) {
        step(pre);
        next_page = page_of(pre);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kPdStages - 1; ++i) issue();

  // The queries of a (sequence, head): lane -> head lane / 4, dims 16 kk + 2 (lane % 4) + {0, 1, 8, 9}.
  // They are fetched a unit before they are needed.
  const float qs = a.scale * kLog2e;
  float2 qn[16];
  auto fetch_q = [&](const PdCursor& c) {
    const int hs = c.sub * 8 + (lane >> 2);
    const bool live = hs < G;
    const long long base = c.b * a.q_stride + ((long long)c.g * G + (live ? hs : 0)) * kHeadDim + 2 * (lane & 3);
#pragma unroll
    for (int kk = 0; kk < 16; ++kk) qn[kk] = load2(a.q, base + 8 * kk, a.dtype);
    if (!live) {
#pragma unroll
      for (int kk = 0; kk < 16; ++kk) qn[kk] = make_float2(0.f, 0.f);
    }
  };
  fetch_q(cur);
  unsigned q[8][4], q3[THREE ? 8 : 1][2];
  float o[16][4], m = -INFINITY, l = 0.0f;
  float factor = qs;   // of q's products
  bool fresh = true;   // a new (sequence, head): take its q, clear the sums
  int seg = 0;         // segments finished by this CTA
  bool from_start = cur.t == 0;
  int slot = 0;
  for (int i = 0; i < n_units; ++i) {
    issue();
    if (fresh) {
      fresh = false;
      if constexpr (std::is_same<T, __half>::value) {
        float top = 0.0f;
#pragma unroll
        for (int kk = 0; kk < 16; ++kk) top = fmaxf(top, fmaxf(fabsf(qn[kk].x), fabsf(qn[kk].y)));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float2 fit = f16_fit(__float_as_int(top) >> 23);
#pragma unroll
        for (int kk = 0; kk < 16; ++kk) qn[kk] = make_float2(qn[kk].x * fit.x, qn[kk].y * fit.x);
        factor = qs * fit.y;
      }
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        if constexpr (THREE) {
          const float2 x = split2_rest<T>(qn[2 * kk].x, qn[2 * kk].y, q[kk][0]);
          const float2 y = split2_rest<T>(qn[2 * kk + 1].x, qn[2 * kk + 1].y, q[kk][2]);
          split2<T>(x.x, x.y, q[kk][1], q3[kk][0]);
          split2<T>(y.x, y.y, q[kk][3], q3[kk][1]);
        } else {
          split2<T>(qn[2 * kk].x, qn[2 * kk].y, q[kk][0], q[kk][1]);
          split2<T>(qn[2 * kk + 1].x, qn[2 * kk + 1].y, q[kk][2], q[kk][3]);
        }
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
      m = -INFINITY;
      l = 0.0f;
    }
    const bool last_t = cur.t + 1 == cur.v.tiles, more = i + 1 < n_units;
    PdCursor nxt = cur;
    if (more) {
      step(nxt);
      if (last_t) fetch_q(nxt);
    }
    const bool rows = (live_ring >> slot) & 1u;
    asm volatile("cp.async.wait_group %0;" ::"n"(kPdStages - 1) : "memory");
    __syncwarp();
    if (rows) {
      const unsigned kb = ring_s + slot * kPdSlot, vb = kb + 4096;
      float s[4][4];  // two key halves, each in two chains of products (even and odd steps)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
      const int mi = lane >> 3, r8 = lane & 7;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        unsigned b[4];
        ldsm4(kb + (8 * (mi >> 1) + r8) * 256 + (((2 * kk + (mi & 1)) ^ r8) << 4), b);
        mma_16816<T>(s[2 * (kk & 1)], q[kk], b[0], b[1]);
        mma_16816<T>(s[2 * (kk & 1) + 1], q[kk], b[2], b[3]);
        if constexpr (THREE) {
          const unsigned q2[4] = {q3[kk][0], 0u, q3[kk][1], 0u};
          mma_16816<T>(s[2 * (kk & 1)], q2, b[0], b[1]);
          mma_16816<T>(s[2 * (kk & 1) + 1], q2, b[2], b[3]);
        }
      }
      const int p0 = cur.v.tile(cur.t) * kPdTile + 16 * warp;
      float p[2][2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) p[j][e] = ((s[j][e] + s[2 + j][e]) + (s[j][2 + e] + s[2 + j][2 + e])) * factor;
      if (!(p0 + 16 <= cur.v.end && (p0 >= cur.v.lo || p0 + 16 <= cur.v.ns))) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (!cur.v.at(p0 + 8 * j + 2 * (lane & 3) + e)) p[j][e] = -INFINITY;
      }
      float mt = fmaxf(fmaxf(p[0][0], p[0][1]), fmaxf(p[1][0], p[1][1]));
      mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
      mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
      if (__any_sync(0xffffffffu, mt > m + kPdLag)) {  // some head's maximum moved: rescale
        const float mn = mt > m + kPdLag ? mt : m;
        const float f = m == -INFINITY ? 0.0f : exp2_fast(m - mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          o[j][0] *= f;
          o[j][1] *= f;
          o[j][2] *= f;
          o[j][3] *= f;
        }
      }
      const float ref = m == -INFINITY ? 0.0f : m - kPdShift;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          p[j][e] = exp2_fast(p[j][e] - ref);
          l += p[j][e];
        }
      unsigned w[4], w3[4] = {0u, 0u, 0u, 0u};
      if constexpr (THREE) {
        const float2 x = split2_rest<T>(p[0][0], p[0][1], w[0]), y = split2_rest<T>(p[1][0], p[1][1], w[2]);
        split2<T>(x.x, x.y, w[1], w3[0]);
        split2<T>(y.x, y.y, w[3], w3[2]);
      } else {
        split2<T>(p[0][0], p[0][1], w[0], w[1]);
        split2<T>(p[1][0], p[1][1], w[2], w[3]);
      }
#pragma unroll
      for (int dn = 0; dn < 16; dn += 2) {
        unsigned b[4];
        ldsm4_t(vb + (r8 + 8 * (mi & 1)) * 256 + (((dn + (mi >> 1)) ^ r8) << 4), b);
        mma_16816<T>(o[dn], w, b[0], b[1]);
        mma_16816<T>(o[dn + 1], w, b[2], b[3]);
        if constexpr (THREE) {
          mma_16816<T>(o[dn], w3, b[0], b[1]);
          mma_16816<T>(o[dn + 1], w3, b[2], b[3]);
        }
      }
    }
    __syncwarp();  // the slot may be refilled
    if (last_t || !more) {
      // The (sequence, head), or this CTA's part of it, ends: join the four warps.
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      float* mine = reinterpret_cast<float*>(ring + slot * kPdSlot) + (lane >> 2) * kPdSumRow + 2 * (lane & 3);
#pragma unroll
      for (int j = 0; j < 16; ++j)
        *reinterpret_cast<float2*>(mine + 8 * j) = make_float2(o[j][0] + o[j][2], o[j][1] + o[j][3]);
      if ((lane & 3) == 0) sml[warp][lane >> 2] = make_float2(m, l);
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
          const float f = sml[w][h].x == -INFINITY ? 0.0f : exp2_fast(sml[w][h].x - M);
          L += sml[w][h].y * f;
          x += reinterpret_cast<const float*>(smem + (w * kPdStages + slot) * kPdSlot)[h * kPdSumRow + tid] * f;
        }
        if (whole) {
          store1(a.y, out + h * kHeadDim, a.dtype, x * inv_sum(L));
        } else {
          ws.o[(part + h) * kHeadDim + tid] = x;
          if (tid == 0) ws.ml[part + h] = make_float2(M, L);
        }
      }
      __syncthreads();  // before the slots are refilled
      ++seg;
      fresh = true;
      from_start = true;
    }
    cur = nxt;
    slot = slot + 1 == kPdStages ? 0 : slot + 1;
  }
}

// Joins the parts of each (sequence, query group) that several CTAs hold. Grid: batch * nh. Warp w takes head w / per of the group
// and every per-th part (per = 8 / heads, a power of two): each lane's loads of up to eight
// parts are in flight together (with one warp per head, 37 parts took 6 us).
__global__ void __launch_bounds__(256) k_paged_decode_join(const __grid_constant__ PAttnArgs a, void* workspace,
                                                           int grid) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = a.q_heads / a.kv.kv_heads, subs = (G + 7) >> 3, nh = a.kv.kv_heads * subs;
  const int b = blockIdx.x / nh, h = blockIdx.x % nh, heads = min(8, G - (h % subs) * 8);
  const PDecodeWs ws = pd_ws(workspace);
  pdl_wait();
  pdl_trigger();
  const int f0 = ws.first[b], tiles = ws.first[b + 1] - f0;
  const long long U = (long long)ws.first[a.kv.batch] * nh;
  const int ctas = (int)min((long long)grid, U);
  const long long v0 = (long long)f0 * nh + (long long)h * tiles, v1 = v0 + tiles;
  if (tiles == 0) return;
  const int c0 = (int)(((v0 + 1) * ctas - 1) / U), c1 = (int)((v1 * ctas - 1) / U);
  if (c0 == c1) return;  // written whole
  const int lg = heads > 4 ? 0 : heads > 2 ? 1 : heads > 1 ? 2 : 3, per = 1 << lg;
  const int hw = warp >> lg, k0 = warp & (per - 1);
  float M = -INFINITY, L = 0.0f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  if (hw < heads) {
    for (int c = c0 + k0; c <= c1; c += 8 * per) {
      float2 ml[8];
      float4 x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int cc = c + k * per;
        ml[k] = make_float2(-INFINITY, 0.0f);
        x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (cc <= c1) {
          const long long slot = (2ll * cc + (U * cc / ctas >= v0 ? 0 : 1)) * 8 + hw;
          ml[k] = ws.ml[slot];
          x[k] = *reinterpret_cast<const float4*>(ws.o + slot * kHeadDim + 4 * lane);
        }
      }
      float mn = M;
#pragma unroll
      for (int k = 0; k < 8; ++k) mn = fmaxf(mn, ml[k].x);
      const float fo = M == -INFINITY ? 0.0f : exp2_fast(M - mn);
      L *= fo;
      y = make_float4(y.x * fo, y.y * fo, y.z * fo, y.w * fo);
      M = mn;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float f = ml[k].x == -INFINITY ? 0.0f : exp2_fast(ml[k].x - M);
        L += ml[k].y * f;
        y = make_float4(y.x + x[k].x * f, y.y + x[k].y * f, y.z + x[k].z * f, y.w + x[k].w * f);
      }
    }
  }
  __shared__ float2 sml[8];
  __shared__ float4 so[8][32];
  if (lane == 0) sml[warp] = make_float2(M, L);
  so[warp][lane] = y;
  __syncthreads();
  if (hw >= heads || k0) return;
  for (int w = 1; w < per; ++w) {
    const float2 ml = sml[warp + w];
    const float4 x = so[warp + w][lane];
    const float mn = fmaxf(M, ml.x);
    const float fa = M == -INFINITY ? 0.0f : exp2_fast(M - mn), fb = ml.x == -INFINITY ? 0.0f : exp2_fast(ml.x - mn);
    L = L * fa + ml.y * fb;
    y = make_float4(y.x * fa + x.x * fb, y.y * fa + x.y * fb, y.z * fa + x.z * fb, y.w * fa + x.w * fb);
    M = mn;
  }
  const float z = inv_sum(L);
  store4(a.y, b * a.y_stride + ((long long)(h / subs) * G + (h % subs) * 8 + hw) * kHeadDim + 4 * lane, a.dtype,
         make_float4(y.x * z, y.y * z, y.z * z, y.w * z));
}

}  // namespace qd
