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
// As k_paged_decode (units in equal runs per CTA, a ring of copies per warp, hi / lo operand rows on mma.sync,
// parts joined by k_paged_decode_join), over half the bytes, so a warp takes 32 positions of a unit of 128:
//  - The integers are exact in f16 and feed the products as they are (byte permutes and one subtraction per pair, in
//    registers). A K row's scale multiplies its scores, a V row's its weight: y = sum_j (p_j vs_j) n_j.
//  - Products may take the contraction's index in any order that both operands share. Thread t of a quad takes dims
//    32 t .. 32 t + 31 of a K row (two 16-byte loads, no transposition) and of V, for the quad's
//    8 dim groups, 16 consecutive dims of its own four positions of 16.
//  - The weights p_j vs_j go into f16 parts, and a V row's scale may have any size beside its weight (the first
//    token's V is small in many models, and its weight large), so they have a running maximum of their own, of
//    s_j + log2 vs_j, next to that of s_j, by which the weights' sum goes.
constexpr int kQ8Tile = 128, kQ8Stages = 3;
constexpr int kQ8Rows = 32;                                  // positions of a warp
constexpr int kQ8Slot = 2 * kQ8Rows * 128 + 2 * kQ8Rows * 4;  // K, V, their scales
static_assert(8 * kPdSumRow * 4 <= kQ8Slot, "a slot holds eight heads' sums");
__host__ __device__ constexpr int pq8_smem(int batch) { return 4 * kQ8Stages * kQ8Slot + (batch + 1) * 4; }

__device__ __forceinline__ void cp_async4(unsigned dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
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
__device__ __forceinline__ float2 lds64f(unsigned addr) {
  float2 r;
  asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(r.x), "=f"(r.y) : "r"(addr));
  return r;
}

__global__ void __launch_bounds__(kPdThreads) k_paged_decode_q8(const __grid_constant__ PAttnArgs a,
                                                                const __grid_constant__ PagedScales scale,
                                                                void* workspace) {
  extern __shared__ __align__(128) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned char* ring = smem + warp * kQ8Stages * kQ8Slot;
  int* first = reinterpret_cast<int*>(smem + 4 * kQ8Stages * kQ8Slot);
  __shared__ float2 sml[4][8];  // maximum and sum of weights of each warp and head,
  __shared__ float smo[4][8];   // the maximum that its sums go by
  const int G = a.q_heads / a.kv.kv_heads, subs = (G + 7) >> 3, nh = a.kv.kv_heads * subs, B = a.kv.batch;
  const PDecodeWs ws = pd_ws(workspace);
  pdl_wait();
  pdl_trigger();
  auto see = [&](int b) { return visible<kQ8Tile>(a.kv.seq_lens[b], paged_len(a.kv, b), a.window, a.sinks); };
  pd_units(B, first, see);
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

  // page of the 16 positions that this half of the warp copies of the unit at `pre`; -1: nothing visible there, -2: bad
  auto page_of = [&](const PdCursor& c) {
    const int p0 = c.v.tile(c.t) * kQ8Tile + kQ8Rows * warp + (lane & 16);
    const bool any = p0 < c.v.end && (p0 + 16 > c.v.lo || p0 < c.v.ns);
    if (!any) return -1;
    const int page = paged_page(a.kv, c.b, p0);
    return page < 0 ? -2 : page;
  };
  int next_page = page_of(pre);
  unsigned live_ring = 0;  // bits 2 i, 2 i + 1: the halves of slot i hold rows
  int issued = 0, in_slot = 0;
  const int pmask = (1 << a.kv.page_shift) - 1;
  const unsigned ring_s = (unsigned)__cvta_generic_to_shared(ring);
  // lane l copies chunk l % 8 of rows 4 i + l / 8; chunk c of row r sits at c ^ (r % 8). Scales: lane l row l.
  unsigned to[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 4 * i + (lane >> 3);
    to[i] = ring_s + r * 128 + (((lane & 7) ^ (r & 7)) << 4);
  }
  auto issue = [&]() {
    if (issued < n_units) {
      const int page = next_page;
      const unsigned good = __ballot_sync(0xffffffffu, page >= 0);
      const unsigned halves = (good & 1u) | ((good >> 16 & 1u) << 1);
      live_ring = (live_ring & ~(3u << (2 * in_slot))) | halves << (2 * in_slot);
      if (page == -2 && (lane & 15) == 0) paged_flag(a.kv, QD_PAGED_BAD_PAGE);
      const int p0 = pre.v.tile(pre.t) * kQ8Tile + kQ8Rows * warp;
      const unsigned dst = in_slot * kQ8Slot;
      // first row of this lane's half (of its scale), and of both halves
      const long long mine = (((long long)max(page, 0) * a.kv.kv_heads + pre.g) << a.kv.page_shift) + ((p0 + (lane & 16)) & pmask);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long long row0 = __shfl_sync(0xffffffffu, mine, 16 * h);
        if (!(halves >> h & 1u)) continue;
        const char* ks = static_cast<const char*>(a.kv.k) + row0 * 128 + lane * 16;
        const char* vs = static_cast<const char*>(a.kv.v) + row0 * 128 + lane * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool ok = pre.v.at(p0 + 16 * h + 4 * i + (lane >> 3));
          cp_async16(to[i & 1] + dst + 2048 * h + (i >> 1) * 1024, ks + i * 512, ok);
          cp_async16(to[i & 1] + dst + 2048 * h + (i >> 1) * 1024 + 4096, vs + i * 512, ok);
        }
      }
      if (page >= 0) {
        const bool ok = pre.v.at(p0 + lane);
        cp_async4(ring_s + dst + 8192 + lane * 4, scale.k + mine + (lane & 15), ok);
        cp_async4(ring_s + dst + 8320 + lane * 4, scale.v + mine + (lane & 15), ok);
      }
      ++issued;
      in_slot = in_slot + 1 == kQ8Stages ? 0 : in_slot + 1;
      if (issued < n_units) {
        step(pre);
        next_page = page_of(pre);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kQ8Stages - 1; ++i) issue();

  // The queries of a (sequence, head), fetched a unit before they are needed: lane l has head l / 4, dims
  // 32 (l % 4) .. + 31, pairs qn[i] of them.
  const float qs = a.scale * kLog2e;
  const int t4 = lane & 3, g8 = lane >> 2;
  float2 qn[16];
  auto fetch_q = [&](const PdCursor& c) {
    const int hs = c.sub * 8 + g8;
    const bool live = hs < G;
    const long long base = c.b * a.q_stride + ((long long)c.g * G + (live ? hs : 0)) * kHeadDim + 32 * t4;
#pragma unroll
    for (int i = 0; i < 16; ++i) qn[i] = load2(a.q, base + 2 * i, a.dtype);
    if (!live) {
#pragma unroll
      for (int i = 0; i < 16; ++i) qn[i] = make_float2(0.f, 0.f);
    }
  };
  fetch_q(cur);
  unsigned q[8][4];
  float o[16][4], m = -INFINITY, mo = -INFINITY, l = 0.0f;
  float factor = qs;   // of q's products
  bool fresh = true;   // a new (sequence, head): take its q, clear the sums
  int seg = 0;         // segments finished by this CTA
  bool from_start = cur.t == 0;
  int slot = 0;
  for (int i = 0; i < n_units; ++i) {
    issue();
    if (fresh) {
      fresh = false;
      float top = 0.0f;
#pragma unroll
      for (int k = 0; k < 16; ++k) top = fmaxf(top, fmaxf(fabsf(qn[k].x), fabsf(qn[k].y)));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float2 fit = f16_fit(__float_as_int(top) >> 23);
      factor = qs * fit.y;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        split2<__half>(qn[2 * k].x * fit.x, qn[2 * k].y * fit.x, q[k][0], q[k][1]);
        split2<__half>(qn[2 * k + 1].x * fit.x, qn[2 * k + 1].y * fit.x, q[k][2], q[k][3]);
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
      m = mo = -INFINITY;
      l = 0.0f;
    }
    const bool last_t = cur.t + 1 == cur.v.tiles, more = i + 1 < n_units;
    PdCursor nxt = cur;
    if (more) {
      step(nxt);
      if (last_t) fetch_q(nxt);
    }
    const unsigned halves = live_ring >> (2 * slot) & 3u;
    asm volatile("cp.async.wait_group %0;" ::"n"(kQ8Stages - 1) : "memory");
    __syncwarp();
    if (halves) {
      const unsigned kb = ring_s + slot * kQ8Slot, vb = kb + 4096;
      const int p0 = cur.v.tile(cur.t) * kQ8Tile + kQ8Rows * warp;
      const bool inside = halves == 3u && p0 + 32 <= cur.v.end && (p0 >= cur.v.lo || p0 + 32 <= cur.v.ns);
      float p[4][2], u[4][2];  // of positions 8 j + 2 t + {0, 1}: scores, and with V's scale
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float s[2][4];
#pragma unroll
        for (int e = 0; e < 2; ++e) s[e][0] = s[e][1] = s[e][2] = s[e][3] = 0.0f;
        const unsigned row = kb + (8 * j + g8) * 128;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint4 x = lds128(row + (((2 * t4 + c) ^ g8) << 4));
          const unsigned w[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, x.z ^ 0x80808080u, x.w ^ 0x80808080u};
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_16816<__half>(s[c], q[4 * c + k], q8_half2(w[k], kQ8Lo), q8_half2(w[k], kQ8Hi));
        }
        const float2 ks = lds64f(kb + 8192 + (8 * j + 2 * t4) * 4), vs = lds64f(kb + 8320 + (8 * j + 2 * t4) * 4);
        p[j][0] = ((s[0][0] + s[1][0]) + (s[0][2] + s[1][2])) * (factor * ks.x);
        p[j][1] = ((s[0][1] + s[1][1]) + (s[0][3] + s[1][3])) * (factor * ks.y);
        u[j][0] = p[j][0] + log2_fast(vs.x);
        u[j][1] = p[j][1] + log2_fast(vs.y);
      }
      if (!inside) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (!(halves >> (j >> 1) & 1u) || !cur.v.at(p0 + 8 * j + 2 * t4 + e)) p[j][e] = u[j][e] = -INFINITY;
      }
      float mt = -INFINITY, ut = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mt = fmaxf(mt, fmaxf(p[j][0], p[j][1]));
        ut = fmaxf(ut, fmaxf(u[j][0], u[j][1]));
      }
      mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
      ut = fmaxf(ut, __shfl_xor_sync(0xffffffffu, ut, 1));
      mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
      ut = fmaxf(ut, __shfl_xor_sync(0xffffffffu, ut, 2));
      if (__any_sync(0xffffffffu, mt > m + kPdLag || ut > mo + kPdLag)) {  // some head's maximum moved: rescale
        const float mn = mt > m + kPdLag ? mt : m, un = ut > mo + kPdLag ? ut : mo;
        l *= m == -INFINITY ? 0.0f : exp2_fast(m - mn);
        const float f = mo == -INFINITY ? 0.0f : exp2_fast(mo - un);
        m = mn;
        mo = un;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          o[j][0] *= f;
          o[j][1] *= f;
          o[j][2] *= f;
          o[j][3] *= f;
        }
      }
      const float ref = m == -INFINITY ? 0.0f : m, uref = mo == -INFINITY ? 0.0f : mo - kPdShift;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l += exp2_fast(p[j][e] - ref);
          u[j][e] = exp2_fast(u[j][e] - uref);
        }
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        unsigned w[4];
        split2<__half>(u[2 * st][0], u[2 * st][1], w[0], w[1]);
        split2<__half>(u[2 * st + 1][0], u[2 * st + 1][1], w[2], w[3]);
        // rows 16 st + 2 t + {0, 1, 8, 9}, chunk g8
        const int r = 2 * t4;
        const unsigned row = vb + (16 * st + r) * 128;
        const uint4 x0 = lds128(row + ((g8 ^ r) << 4)), x1 = lds128(row + 128 + ((g8 ^ (r + 1)) << 4));
        const uint4 x2 = lds128(row + 1024 + ((g8 ^ r) << 4)), x3 = lds128(row + 1152 + ((g8 ^ (r + 1)) << 4));
        const unsigned va[4] = {x0.x, x0.y, x0.z, x0.w}, vbb[4] = {x1.x, x1.y, x1.z, x1.w};
        const unsigned vc[4] = {x2.x, x2.y, x2.z, x2.w}, vd[4] = {x3.x, x3.y, x3.z, x3.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const unsigned a0 = __byte_perm(va[k], vbb[k], 0x5140) ^ 0x80808080u, a1 = __byte_perm(va[k], vbb[k], 0x7362) ^ 0x80808080u;
          const unsigned b0 = __byte_perm(vc[k], vd[k], 0x5140) ^ 0x80808080u, b1 = __byte_perm(vc[k], vd[k], 0x7362) ^ 0x80808080u;
          mma_16816<__half>(o[4 * k], w, q8_half2(a0, kQ8Lo), q8_half2(b0, kQ8Lo));
          mma_16816<__half>(o[4 * k + 1], w, q8_half2(a0, kQ8Hi), q8_half2(b0, kQ8Hi));
          mma_16816<__half>(o[4 * k + 2], w, q8_half2(a1, kQ8Lo), q8_half2(b1, kQ8Lo));
          mma_16816<__half>(o[4 * k + 3], w, q8_half2(a1, kQ8Hi), q8_half2(b1, kQ8Hi));
        }
      }
    }
    __syncwarp();  // the slot may be refilled
    if (last_t || !more) {
      // The (sequence, head), or this CTA's part of it, ends: join the four warps.
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      float* mine = reinterpret_cast<float*>(ring + slot * kQ8Slot) + g8 * kPdSumRow + 32 * t4;
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        *reinterpret_cast<float4*>(mine + j) = make_float4(o[j][0] + o[j][2], o[j + 1][0] + o[j + 1][2],
                                                           o[j + 2][0] + o[j + 2][2], o[j + 3][0] + o[j + 3][2]);
        *reinterpret_cast<float4*>(mine + 16 + j) = make_float4(o[j][1] + o[j][3], o[j + 1][1] + o[j + 1][3],
                                                                o[j + 2][1] + o[j + 2][3], o[j + 3][1] + o[j + 3][3]);
      }
      if (t4 == 0) {
        sml[warp][g8] = make_float2(m, l);
        smo[warp][g8] = mo;
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
          L += sml[w][h].x == -INFINITY ? sml[w][h].y * 0.0f : sml[w][h].y * exp2_fast(sml[w][h].x - M);
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
      __syncthreads();  // before the slots are refilled
      ++seg;
      fresh = true;
      from_start = true;
    }
    cur = nxt;
    slot = slot + 1 == kQ8Stages ? 0 : slot + 1;
  }
}

}  // namespace qd
