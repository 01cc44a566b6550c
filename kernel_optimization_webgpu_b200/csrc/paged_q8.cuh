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
// 8 (l % 16) of every other row, all sixteen loads together, and while they are on their way it finds the next 16 and looks
// up their pages. What it has to move bounds it (132 bytes of a row in, 256 out): 24 sequences of up to 9001 positions, 527 MB,
// 86 us = 6.1 TB/s. Units are counted through a scan of the lengths, so that a table wider than they are costs nothing, and
// shared out over more CTAs than run at once (32 per SM; 93 us with 8), as the SMs' share of the memory's rate is not even.
template <typename T>
__global__ void __launch_bounds__(kPdThreads) k_paged_read_q8(const __grid_constant__ ReadArgs a) {
  extern __shared__ int first[];
  const int tid = threadIdx.x, lane = tid & 31, B = a.src.batch, kvh = a.src.kv_heads;
  pdl_wait();
  pdl_trigger();
  auto end_of = [&](int b) { return min(paged_len(a.src, b), a.dst.table_width << a.dst.page_shift); };
  auto from = [&](int b) { return a.first ? max(a.first[b], 0) : 0; };
  struct Tiles { int tiles; };
  __shared__ int wsum[4];
  pd_units(B, first, tid, lane, tid >> 5, wsum, [&](int b) {
    const int n = end_of(b), f = min(from(b), n);
    return Tiles{f < n ? (n + 15) / 16 - f / 16 : 0};
  });
  if (blockIdx.x == 0)
    for (int b = tid; b < B; b += kPdThreads)
      if (a.src.seq_lens[b] != end_of(b)) paged_flag(a.src, QD_PAGED_BAD_LENGTH);
  const long long units = (long long)first[B] * kvh;
  const int warps = gridDim.x * (kPdThreads / 32);
  struct Unit {
    int g, f, end, p0, ps, pd;  // its positions are those of p0 .. p0 + 15 in [f, end); entries of both tables
  };
  auto find = [&](long long u) {
    int lo = 0, hi = B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((long long)first[mid] * kvh <= u) lo = mid;
      else hi = mid;
    }
    const int rest = (int)(u - (long long)first[lo] * kvh), tiles = first[lo + 1] - first[lo];
    Unit x;
    x.g = rest / tiles;
    x.f = from(lo);
    x.end = end_of(lo);
    x.p0 = (x.f / 16 + rest - x.g * tiles) * 16;
    x.ps = a.src.table[(long long)lo * a.src.table_stride + (x.p0 >> a.src.page_shift)];
    x.pd = a.dst.table[(long long)lo * a.dst.table_stride + (x.p0 >> a.dst.page_shift)];
    return x;
  };
  long long u = blockIdx.x * (kPdThreads / 32) + (tid >> 5);
  if (u >= units) return;
  const int r0 = lane >> 4, c = lane & 15;
  for (Unit x = find(u);;) {
    const bool ok = (unsigned)x.ps < (unsigned)a.src.num_pages && (unsigned)x.pd < (unsigned)a.dst.num_pages;
    uint2 w[2][8];
    float mine = 0.0f;
    if (ok) {
      const long long rs = (((long long)x.ps * kvh + x.g) << a.src.page_shift) + (x.p0 & ((1 << a.src.page_shift) - 1));
      // lane l: the scale of row l % 16, of K in the first half, of V in the second (rows of the page that no
      // sequence holds are memory too, and their values are not used)
      mine = (lane < 16 ? a.scale.k : a.scale.v)[rs + c];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[0][i] = reinterpret_cast<const uint2*>(static_cast<const int8_t*>(a.src.k) + rs * kHeadDim)[i * 32 + lane];
        w[1][i] = reinterpret_cast<const uint2*>(static_cast<const int8_t*>(a.src.v) + rs * kHeadDim)[i * 32 + lane];
      }
    } else if (lane == 0) {
      paged_flag(a.src, QD_PAGED_BAD_PAGE);
    }
    u += warps;
    const bool more = u < units;
    Unit next = x;
    if (more) next = find(u);
    if (ok) {
      const long long rd = (((long long)x.pd * kvh + x.g) << a.dst.page_shift) + (x.p0 & ((1 << a.dst.page_shift) - 1));
      const bool all = x.p0 >= x.f && x.p0 + 16 <= x.end;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(n ? a.dst.v : a.dst.k) + rd * kHeadDim) + lane;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int p = x.p0 + 2 * i + r0;
          const float s = __shfl_sync(0xffffffffu, mine, 16 * n + 2 * i + r0);
          const float4 y = q8_float4(w[n][i].x ^ 0x80808080u, s), z = q8_float4(w[n][i].y ^ 0x80808080u, s);
          if (all || (p >= x.f && p < x.end))
            dst[i * 32] = make_uint4(pack2<T>(y.x, y.y), pack2<T>(y.z, y.w), pack2<T>(z.x, z.y), pack2<T>(z.z, z.w));
        }
      }
    }
    if (!more) break;
    x = next;
  }
}

// ---- attention of one new token per sequence ---------------------------------------------------
// As k_paged_decode (units in equal runs per CTA, a ring of copies per warp, parts joined by
// k_paged_decode_join), over half the bytes, which leaves instructions as the next bound, so:
//  - A warp takes 32 positions of a unit of 128. TMA copies them, 16 rows of one page at a time, with the swizzle
//    that the loads from shared memory want; one lane per 16 rows asks for them.
//  - mma.sync with keys (dims of V) as the 16 rows and query heads as the 8 columns, so that nothing is spent on
//    the eight rows that two heads would leave empty the other way round.
//  - A K row's scale multiplies its scores, a V row's its weight: y = sum_j (p_j vs_j) n_j. The products take the
//    cache's integers, and the other operand as a sum of parts that are columns side by side:
//      one or two heads to a KV head (Q8Whole): m16n8k32 of 8-bit integers, q and the weights as 31-bit fixed-point
//      numbers in four signed bytes, exact sums in 32 bits. K goes into it as it lies in memory, V transposed by bytes
//      in registers;
//      more heads (Q8Half): m16n8k16 of f16, the integers made f16 (byte permutes and a subtraction per pair), q and the
//      weights as two f16. Its columns hold twice the heads, and its sums take a third of the registers.
//    64 sequences of 2048 positions, 8 KV heads: 16 query heads 55 us with Q8Whole and 58 with Q8Half; 32 query heads 71 and
//    66 (with four heads in Q8Whole); 4 KV heads and 32 query heads 52 with Q8Half, 75 with Q8Whole twice.
//  - The contraction's index may have any order that both operands share: thread t of a quad takes dims
//    32 t .. + 31 of a K row (two 16-byte loads) and 16 consecutive dims of some positions of V.
//  - A V row's scale may have any size beside its weight (the first token's V is small in many models, and its weight
//    large), so the weights p_j vs_j have a running maximum of their own, of s_j and the scale's exponent, next to that
//    of s_j, by which the weights' sum goes.
constexpr int kQ8Tile = 128, kQ8Stages = 2;
constexpr int kQ8Rows = 32;                 // positions of a warp
constexpr int kQ8Slot = 2 * kQ8Rows * 128;  // K and V
constexpr int kQ8Scales = 2 * kQ8Rows * 4;  // their scales
static_assert(8 * kPdSumRow * 4 <= kQ8Slot, "a slot holds eight heads' sums");
__host__ __device__ constexpr int pq8_smem(int batch) {
  return 1024 + 4 * kQ8Stages * (kQ8Slot + kQ8Scales) + (batch + 1) * 4;
}

struct Q8Args {
  CUtensorMap tk, tv;  // boxes of 16 rows
  PAttnArgs a;
  PagedScales scale;
  int stall;  // test hook (qd_paged_inject_stall): block 0's first warp withholds its first copies
};

// A scale as f * 2^k, 1 <= |f| < 2 (0 and below 2^-126: k is -inf; not finite: f is the scale itself). A weight times it is
// exp2(s + k - reference) f: the sum with k loses less than one with a logarithm does (f32 queries on 1 x 31
// positions: 9e-7 off with a logarithm, 2 - 4e-7 so; 64 x 2048: 54.2 -> 55.3 us, 64 x 8192: 182 -> 177).
__device__ __forceinline__ void q8_scale(float s, float& k, float& f) {
  const unsigned u = __float_as_uint(s), e = (u >> 23) & 255u;
  k = e == 0u ? -INFINITY : __uint_as_float(0x4b000000u | e) - 8388735.0f;  // (2^23 + e less 2^23 + 127)
  f = e == 255u ? s : __uint_as_float((u & 0x807fffffu) | 0x3f800000u);
}
// (not volatile: the loads and products of a unit may be interleaved as their latencies ask)
__device__ __forceinline__ void q8_mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned transpose_b16(unsigned x) {  // an 8 x 8 matrix over the warp
  unsigned y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// What both kinds share of a unit: the visible positions of the warp's 32.
struct Q8Seen {
  bool inside;      // all of them
  unsigned halves;  // bit i: rows 16 i .. + 15 are there
  int p0;
  Visible v;
  __device__ __forceinline__ bool at(int i) const { return (halves >> (i >> 4) & 1u) && v.at(p0 + i); }
};
__device__ __forceinline__ uint4 q8_lds(const unsigned char* at) { return *reinterpret_cast<const uint4*>(at); }

// One or two heads: columns 4 h + part, part 3 the most significant byte. Thread (g8, t4) has the scores of head t4 / 2 at
// positions order(g8) + 8 j, j < 4 (as its neighbour t4 ^ 1 has), and dims 16 g8 .. + 15 of two of the head's parts.
// Positions are taken in an order for which the rows that a quarter warp reads from shared memory lie on distinct banks.
struct Q8Whole {
  static constexpr int kHeads = 2, kCtas = 3;  // heads, CTAs per SM
  static constexpr float kShift = 29.0f;       // weights are kept times 2^29 (below 2^30), off by 2^-30 of the largest
  static constexpr int kFlush = 2048;          // units after which the 32-bit sums are moved (each adds below 2^19)
  unsigned q[4][2];
  int acc[8][4];
  float o[16], m, mo, l, factor;
  int since;

  static __device__ __forceinline__ int order(int c) { return 2 * (c & 3) + ((c ^ (c >> 2)) & 1); }
  // A number of at most 2^30 in size as four signed bytes.
  static __device__ __forceinline__ unsigned digits(int x) { return (unsigned)(x + 0x00808080) ^ 0x00808080u; }
  // Four words as the columns of their bytes.
  static __device__ __forceinline__ void turn(unsigned a, unsigned b, unsigned c, unsigned d, unsigned (&r)[4]) {
    const unsigned ab0 = __byte_perm(a, b, 0x5140), ab1 = __byte_perm(a, b, 0x7362);
    const unsigned cd0 = __byte_perm(c, d, 0x5140), cd1 = __byte_perm(c, d, 0x7362);
    r[0] = __byte_perm(ab0, cd0, 0x5410);
    r[1] = __byte_perm(ab0, cd0, 0x7632);
    r[2] = __byte_perm(ab1, cd1, 0x5410);
    r[3] = __byte_perm(ab1, cd1, 0x7632);
  }
  static __device__ __forceinline__ void mma(int (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                             unsigned b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }

  __device__ __forceinline__ void start(const PAttnArgs& a, const PdCursor& c, int G, int g8, int t4) {
    since = 0;
    const int hs = c.sub * kHeads + (g8 >> 2);
    const bool live = hs < G;
    const long long base = c.b * a.q_stride + ((long long)c.g * G + (live ? hs : 0)) * kHeadDim + 32 * t4;
    float2 x[16];
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) x[k] = load2(a.q, base + 2 * k, a.dtype);
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      if (!live) x[k] = make_float2(0.f, 0.f);
      top = max(top, max(__float_as_uint(x[k].x) & 0x7fffffffu, __float_as_uint(x[k].y) & 0x7fffffffu));
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // by a power of two (in two steps from very small ones) to below 2^30
    const int e = (int)(top >> 23), small = e < 60;
    const float up0 = small ? 18446744073709551616.0f : 1.0f, down0 = small ? 5.421010862427522e-20f : 1.0f;
    const int f = min(small ? e + 64 : e, 254);
    const float up = __int_as_float((283 - f) << 23), down = __int_as_float((f - 29) << 23);
    const unsigned sel = 0x0040u + 0x11u * (g8 & 3);  // byte g8 % 4 of two words
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      unsigned d[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float y = i & 1 ? x[2 * k + (i >> 1)].y : x[2 * k + (i >> 1)].x;
        d[i] = digits(__float2int_rn(y * up0 * up));
      }
      q[k >> 1][k & 1] = __byte_perm(__byte_perm(d[0], d[1], sel), __byte_perm(d[2], d[3], sel), 0x5410);
    }
    // of the head whose scores this thread has; not finite: its scores are NaN
    const float mine = e == 255 ? __int_as_float(0x7fffffff) : a.scale * kLog2e * down0 * down;
    factor = __shfl_sync(0xffffffffu, mine, 16 * (t4 >> 1));
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j] = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0;
    m = mo = -INFINITY;
    l = 0.0f;
  }
  // Moves the 32-bit sums to the f32 ones, times f.
  __device__ __forceinline__ void flush(float f) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        o[2 * j + e] = (o[2 * j + e] + fmaf((float)acc[j][2 * e + 1], 256.0f, (float)acc[j][2 * e])) * f;
        acc[j][2 * e] = acc[j][2 * e + 1] = 0;
      }
  }
  __device__ __forceinline__ void unit(const unsigned char* kb, const unsigned char* vb, const float* ks, const float* vs,
                                       const Q8Seen& seen, int g8, int t4) {
    const int r0 = order(g8);
    float p[4], u[4], vf[4];  // of positions r0 + 8 j: scores, and with V's scale but for its factor vf
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      int s[4] = {0, 0, 0, 0};
      const unsigned char* row = kb + (16 * h + r0) * 128;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const unsigned char* at = row + (((2 * t4 + c) ^ r0) << 4);
        const uint4 x = q8_lds(at), y = q8_lds(at + 1024);
        mma(s, x.x, y.x, x.y, y.y, q[2 * c][0], q[2 * c][1]);
        mma(s, x.z, y.z, x.w, y.w, q[2 * c + 1][0], q[2 * c + 1][1]);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = 2 * h + e;
        const float sc = ks[r0 + 8 * j];
        float k;
        q8_scale(vs[r0 + 8 * j], k, vf[j]);
        // two bytes of q here (below 2^30 together), two in the neighbour
        const float x = (float)(s[2 * e] + 256 * s[2 * e + 1]) * (t4 & 1 ? 65536.0f : 1.0f);
        p[j] = (x + __shfl_xor_sync(0xffffffffu, x, 1)) * (factor * sc);
        u[j] = p[j] + k;
      }
    }
    if (!seen.inside) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (!seen.at(r0 + 8 * j)) p[j] = u[j] = -INFINITY, vf[j] = 0.0f;  // (what lies there may be no scale)
    }
    const bool full = ++since == kFlush;
    if (full) since = 0;
    unsigned w[2];
    float mt = fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3]));
    float ut = fmaxf(fmaxf(u[0], u[1]), fmaxf(u[2], u[3]));
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, x));
      ut = fmaxf(ut, __shfl_xor_sync(0xffffffffu, ut, x));
    }
    if (__any_sync(0xffffffffu, full || mt > m + kPdLag || ut > mo)) {  // some head's maximum moved
      const float mn = mt > m + kPdLag ? mt : m, un = ut > mo ? ut : mo;
      l *= m == -INFINITY ? 0.0f : exp2_fast(m - mn);
      flush(mo == -INFINITY ? 0.0f : exp2_fast(mo - un));
      m = mn;
      mo = un;
    }
    const float ref = m == -INFINITY ? 0.0f : m, uref = mo == -INFINITY ? 0.0f : mo - kShift;
    unsigned d[4], r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = exp2_fast(u[j] - uref) * vf[j];
      l = fmaf(x, 0.0f, l) + exp2_fast(p[j] - ref);  // (a NaN weight is no integer)
      d[j] = digits(__float2int_rn(x));
    }
    // the parts of four positions each; thread (g8, t4) wants part g8 % 4 of head g8 / 4 of those that rows t4 and t4 + 4 have
    turn(d[0], d[1], d[2], d[3], r);
    const unsigned even = t4 & 1 ? r[2] : r[0], odd = t4 & 1 ? r[3] : r[1];
    const int from = 4 * t4 + 2 * (g8 >> 2) + ((g8 >> 1) & 1);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const unsigned x = __shfl_sync(0xffffffffu, even, from + 16 * e), y = __shfl_sync(0xffffffffu, odd, from + 16 * e);
      w[e] = g8 & 1 ? y : x;
    }
    // V: positions order(t4) + 8 j and order(t4 + 4) + 8 j, dims 16 g8 .. + 15
    const int ra = order(t4), rb = order(t4 + 4);
    const unsigned char *va = vb + ra * 128 + ((g8 ^ ra) << 4), *vc = vb + rb * 128 + ((g8 ^ rb) << 4);
    uint4 x[4], y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = q8_lds(va + 1024 * j);
      y[j] = q8_lds(vc + 1024 * j);
    }
    auto dims = [&](int k, unsigned xa, unsigned xb, unsigned xc, unsigned xd, unsigned ya, unsigned yb, unsigned yc,
                    unsigned yd) {  // 4 k .. + 3 of both
      unsigned e[4], f[4];
      turn(xa, xb, xc, xd, e);
      turn(ya, yb, yc, yd, f);
      mma(acc[2 * k], e[0], e[1], f[0], f[1], w[0], w[1]);
      mma(acc[2 * k + 1], e[2], e[3], f[2], f[3], w[0], w[1]);
    };
    dims(0, x[0].x, x[1].x, x[2].x, x[3].x, y[0].x, y[1].x, y[2].x, y[3].x);
    dims(1, x[0].y, x[1].y, x[2].y, x[3].y, y[0].y, y[1].y, y[2].y, y[3].y);
    dims(2, x[0].z, x[1].z, x[2].z, x[3].z, y[0].z, y[1].z, y[2].z, y[3].z);
    dims(3, x[0].w, x[1].w, x[2].w, x[3].w, y[0].w, y[1].w, y[2].w, y[3].w);
  }
  __device__ __forceinline__ void give_up() { l = __int_as_float(0x7fffffff); }
  // The warp's sums of head h to sums[h * kPdSumRow + dim], maximum and weights to ml[h], the maximum of the sums to mos[h].
  __device__ __forceinline__ void finish(float* sums, float2* ml, float* mos, int g8, int t4) {
    flush(1.0f);
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
    float y[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float x = o[j] * (t4 & 1 ? 65536.0f : 1.0f);
      y[j] = x + __shfl_xor_sync(0xffffffffu, x, 1);
    }
    const int h = t4 >> 1;
    float* mine = sums + h * kPdSumRow + 16 * g8 + 8 * (t4 & 1);
#pragma unroll
    for (int j = 0; j < 8; j += 4)
      *reinterpret_cast<float4*>(mine + j) = t4 & 1 ? make_float4(y[8 + j], y[9 + j], y[10 + j], y[11 + j])
                                                   : make_float4(y[j], y[j + 1], y[j + 2], y[j + 3]);
    if (g8 == 0 && !(t4 & 1)) {
      ml[h] = make_float2(m, l);
      mos[h] = mo;
    }
  }
};

// Up to 4 * SETS heads. Set n has heads 4 n .. + 3: columns 2 (h % 4) (the 16-bit part) and + 1 (the rest). Thread (g8, t4) has
// the scores of head 4 n + t4 at positions g8 + 8 j, and its dims 16 g8 .. + 15.
template <int SETS>
struct Q8Half {
  static constexpr int kHeads = 4 * SETS, kCtas = SETS == 1 ? 3 : 2;
  // a maximum may fall behind by 2^7: weights, and their scales' factors below 2, then stay below 2^15
  static constexpr float kLag = 7.0f, kShift = kPdShift;
  unsigned q[SETS][8][2];
  float o[SETS][8][4], m[SETS], mo[SETS], l[SETS], factor[SETS];

  __device__ __forceinline__ void start(const PAttnArgs& a, const PdCursor& c, int G, int g8, int t4) {
#pragma unroll
    for (int n = 0; n < SETS; ++n) {
      const int hs = c.sub * kHeads + 4 * n + (g8 >> 1);
      const bool live = hs < G;
      const long long base = c.b * a.q_stride + ((long long)c.g * G + (live ? hs : 0)) * kHeadDim + 32 * t4;
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
      factor[n] = a.scale * kLog2e * __shfl_sync(0xffffffffu, fit.y, 8 * t4);  // of head t4: columns 2 t4, 2 t4 + 1
#pragma unroll
      for (int j = 0; j < 8; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.0f;
      m[n] = mo[n] = -INFINITY;
      l[n] = 0.0f;
    }
  }
  __device__ __forceinline__ void unit(const unsigned char* kb, const unsigned char* vb, const float* ks, const float* vs,
                                       const Q8Seen& seen, int g8, int t4) {
    float p[SETS][4], u[SETS][4], vf[4];  // of positions 8 j + g8: scores, and with V's scale
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float s[SETS][2][4];
#pragma unroll
      for (int n = 0; n < SETS; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) s[n][e][0] = s[n][e][1] = s[n][e][2] = s[n][e][3] = 0.0f;
      const unsigned char* row = kb + (16 * h + g8) * 128;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const unsigned char* at = row + (((2 * t4 + c) ^ g8) << 4);
        const uint4 x = q8_lds(at), y = q8_lds(at + 1024);
        const unsigned xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const unsigned v = xw[k] ^ 0x80808080u, w = yw[k] ^ 0x80808080u;
          const unsigned f[4] = {q8_half2(v, kQ8Lo), q8_half2(w, kQ8Lo), q8_half2(v, kQ8Hi), q8_half2(w, kQ8Hi)};
#pragma unroll
          for (int n = 0; n < SETS; ++n) q8_mma(s[n][k & 1], f, q[n][4 * c + k][0], q[n][4 * c + k][1]);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = 2 * h + e;
        const float sc = ks[8 * j + g8];
        float kv;
        q8_scale(vs[8 * j + g8], kv, vf[j]);
#pragma unroll
        for (int n = 0; n < SETS; ++n) {
          p[n][j] = ((s[n][0][2 * e] + s[n][1][2 * e]) + (s[n][0][2 * e + 1] + s[n][1][2 * e + 1])) * (factor[n] * sc);
          u[n][j] = p[n][j] + kv;
        }
      }
    }
    if (!seen.inside) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (!seen.at(8 * j + g8)) {
          vf[j] = 0.0f;  // (what lies there may be no scale)
#pragma unroll
          for (int n = 0; n < SETS; ++n) p[n][j] = u[n][j] = -INFINITY;
        }
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
      if (__any_sync(0xffffffffu, mt > m[n] + kPdLag || ut > mo[n] + kLag)) {  // some head's maximum moved: rescale
        const float mn = mt > m[n] + kPdLag ? mt : m[n], un = ut > mo[n] + kLag ? ut : mo[n];
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
        u[n][j] = exp2_fast(u[n][j] - uref) * vf[j];
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
      const unsigned char* row = vb + (16 * st + 2 * t4) * 128;
      const unsigned c0 = (g8 ^ (2 * t4)) << 4, c1 = (g8 ^ (2 * t4 + 1)) << 4;
      const uint4 x0 = q8_lds(row + c0), x1 = q8_lds(row + 128 + c1);
      const uint4 x2 = q8_lds(row + 1024 + c0), x3 = q8_lds(row + 1152 + c1);
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
          q8_mma(o[n][2 * k], f, w[n][0], w[n][1]);
          q8_mma(o[n][2 * k + 1], f2, w[n][0], w[n][1]);
        }
      }
    }
  }
  __device__ __forceinline__ void give_up() {
#pragma unroll
    for (int n = 0; n < SETS; ++n) l[n] = __int_as_float(0x7fffffff);
  }
  __device__ __forceinline__ void finish(float* sums, float2* ml, float* mos, int g8, int t4) {
#pragma unroll
    for (int n = 0; n < SETS; ++n) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[n] += __shfl_xor_sync(0xffffffffu, l[n], x);
      float* mine = sums + (4 * n + t4) * kPdSumRow + 16 * g8;
#pragma unroll
      for (int j = 0; j < 8; j += 2)
        *reinterpret_cast<float4*>(mine + 2 * j) = make_float4(o[n][j][0] + o[n][j][1], o[n][j][2] + o[n][j][3],
                                                               o[n][j + 1][0] + o[n][j + 1][1], o[n][j + 1][2] + o[n][j + 1][3]);
      if (g8 == 0) {
        ml[4 * n + t4] = make_float2(m[n], l[n]);
        mos[4 * n + t4] = mo[n];
      }
    }
  }
};

template <typename Heads>
__global__ void __launch_bounds__(kPdThreads, Heads::kCtas) k_paged_decode_q8(const __grid_constant__ Q8Args qa, void* workspace) {
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
  const int G = a.q_heads / a.kv.kv_heads, subs = (G + Heads::kHeads - 1) / Heads::kHeads, nh = a.kv.kv_heads * subs, B = a.kv.batch;
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
  __shared__ int wsum[4];
  pd_units(B, first, tid, lane, warp, wsum, see);  // (its barriers are the mbarriers' too)
  const long long U = (long long)first[B] * nh;
  const int ctas = (int)min((long long)gridDim.x, U);  // none of them empty
  auto aside = [&] {  // what is not on the way to the first copies
    if (blockIdx.x == 0) {
      for (int b = tid; b <= B; b += kPdThreads) ws.first[b] = first[b];
      for (int b = tid; b < B; b += kPdThreads)  // (paged_len cuts both)
        if (a.kv.seq_lens[b] != paged_len(a.kv, b)) paged_flag(a.kv, QD_PAGED_BAD_LENGTH);
    }
    for (int b = blockIdx.x; b < B; b += gridDim.x)  // nothing visible: zeros
      if (first[b + 1] == first[b])
        for (int i = tid; i < a.q_heads * kHeadDim; i += kPdThreads) store1(a.y, b * a.y_stride + i, a.dtype, 0.0f);
  };
  if ((int)blockIdx.x >= ctas) {
    aside();
    return;
  }
  const int u0 = pd_div(U * blockIdx.x, ctas), u1 = pd_div(U * (blockIdx.x + 1), ctas);
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
  // the queries of a (sequence, head) brought near before they are needed
  const int q_bytes = a.dtype == QD_KV_F32 ? 4 : 2;
  auto near_q = [&](const PdCursor& c) {
    const char* at = static_cast<const char*>(a.q) + (c.b * a.q_stride + ((long long)c.g * G + c.sub * Heads::kHeads) * kHeadDim) * q_bytes;
    if (lane * 128 < min(Heads::kHeads, G - c.sub * Heads::kHeads) * kHeadDim * q_bytes) asm volatile("prefetch.global.L1 [%0];" ::"l"(at + lane * 128));
  };
  int next_page = page_of(pre);
  near_q(pre);
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
    if ((lane & 15) == 0 && page >= 0 && !(qa.stall && issued == 0 && warp == 0 && blockIdx.x == 0)) {
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
      if (pre.t == 0) near_q(pre);
    }
  };
#pragma unroll
  for (int i = 0; i < kQ8Stages - 1; ++i) issue();
  aside();

  const int t4 = lane & 3, g8 = lane >> 2;
  Heads heads;
  bool fresh = true;  // a new (sequence, head): take its q, clear the sums
  int seg = 0;        // segments finished by this CTA
  bool from_start = cur.t == 0;
  int slot = 0;
  for (int i = 0; i < n_units; ++i) {
    issue();
    if (fresh) heads.start(a, cur, G, g8, t4);
    fresh = false;
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
      heads.give_up();
    }
    if (halves) {
      const unsigned char* kb = ring + slot * kQ8Slot;
      const float* ks = reinterpret_cast<const float*>(scales + slot * kQ8Scales);
      Q8Seen seen{false, halves, cur.v.tile(cur.t) * kQ8Tile + kQ8Rows * warp, cur.v};
      seen.inside = halves == 3u && seen.p0 + 32 <= cur.v.end && (seen.p0 >= cur.v.lo || seen.p0 + 32 <= cur.v.ns);
      heads.unit(kb, kb + kQ8Rows * 128, ks, ks + kQ8Rows, seen, g8, t4);
    }
    __syncwarp();  // the slot may be refilled
    if (last_t || !more) {
      // The (sequence, head), or this CTA's part of it, ends: join the four warps. The sums go to the slot that has
      // just been read.
      heads.finish(reinterpret_cast<float*>(ring + slot * kQ8Slot), sml[warp], smo[warp], g8, t4);
      __syncthreads();
      const int live = min(Heads::kHeads, G - cur.sub * Heads::kHeads);
      const bool whole = from_start && last_t;
      const long long out = cur.b * a.y_stride + ((long long)cur.g * G + cur.sub * Heads::kHeads) * kHeadDim + tid;
      const long long part = (2ll * blockIdx.x + (seg ? 1 : 0)) * 8;
      for (int h = 0; h < live; ++h) {  // thread tid: dim tid
        const float M = fmaxf(fmaxf(sml[0][h].x, sml[1][h].x), fmaxf(sml[2][h].x, sml[3][h].x));
        float L = 0.0f, x = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          L += sml[w][h].y * (sml[w][h].x == -INFINITY ? 0.0f : exp2_fast(sml[w][h].x - M));  // (NaN stays)
          // (the exponential has no results below 2^-126, the sums may: V scales go down to there)
          const float e = smo[w][h] - M, lift = e < -64.0f ? 64.0f : 0.0f;
          const float f = smo[w][h] == -INFINITY ? 0.0f : exp2_fast(e + lift);
          const float sum = reinterpret_cast<const float*>(smem + (w * kQ8Stages + slot) * kQ8Slot)[h * kPdSumRow + tid];
          x += sum * (1.0f / (1 << (int)Heads::kShift)) * f * (lift == 0.0f ? 1.0f : 0x1p-64f);
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
