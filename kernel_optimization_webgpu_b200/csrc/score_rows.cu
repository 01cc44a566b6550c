// Per row of logits: the log probability of a given token, the entropy of the softmax, and the largest tokens.
//
//   log p_t = x_t - m - log S,  H = log S - sum (x - m) e^(x - m) / S,  S = sum e^(x - m),  m = max x
//
// One thread-block cluster per row, a contiguous share per CTA, read once from memory: each thread keeps a running
// maximum and both sums by it, joined over warps and the cluster at the end. The largest tokens need a border first,
// below which nothing has to be looked at: the row's threads form 128 groups, and the top-th largest of the groups'
// maxima is a value that at least `top` tokens reach and that hardly more than those do. Of the batches of loads whose
// maximum (kept in shared memory) reaches it, a few dozen, the tokens are listed, and the list is put in order by
// counting.
//
// Many rows: bound by the latency of the loads and, with 16-bit logits, by the exponentials (one per token: 17 of
// 39 us of the special-function unit), so the next batch is on its way while one is worked on. 512 x 151936 bf16 with 20
// alternatives: 39 us (156 MB, 4.0 TB/s; 35 without alternatives), 256 x 151936 f32: 27 us (5.75 TB/s). One row of f32:
// 7.9 us, of which a chain of loads, barriers of the cluster and the border's search, not bytes.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/qdecode.h"
#include "internal.cuh"
#include "overlap.hpp"
#include "rows.cuh"

namespace qd {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int kScoreThreads = 256;
constexpr int kScoreCluster = 8;
constexpr int kScoreTop = 64;      // largest `top`
constexpr int kScoreGroups = 128;  // of a row's threads: at least kScoreTop
constexpr int kScoreList = 1024;   // tokens at or above the border that a CTA lists
constexpr int kScoreUnroll = 4;    // 16-byte loads of a thread's batch
constexpr int kScoreSlots = 12;    // batches whose maxima are kept apart

struct ScoreArgs {
  const void* logits;
  int vocab, per;  // per: 16-byte vectors a CTA takes
  long long row_stride;
  const int* tokens;
  int top;
  float* logprobs;
  float* entropy;
  int* top_ids;
  float* top_logprobs;
};

constexpr float kLog2E = 1.4426950408889634f;

// Sums by a maximum: s0 = sum e^d, s1 = sum d e^d, d = x - m.
struct ScoreSums {
  float m, s0, s1;
};
__device__ __forceinline__ float score_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The factor of sums by the maximum m, for sums by mn >= m: e^d.
__device__ __forceinline__ float score_shift(float m, float mn, float& d) {
  d = m == mn || m == -INFINITY ? 0.0f : fmaxf(m - mn, -150.0f);
  return m == -INFINITY ? 0.0f : score_exp2(d * kLog2E);
}
// The sums of a warp's lanes, in all of them.
__device__ __forceinline__ ScoreSums score_join(ScoreSums s) {
  float mn = s.m, d;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
  const float f = score_shift(s.m, mn, d);
  s = ScoreSums{mn, s.s0 * f, fmaf(d, s.s0, s.s1) * f};
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s.s0 += __shfl_xor_sync(0xffffffffu, s.s0, o);
    s.s1 += __shfl_xor_sync(0xffffffffu, s.s1, o);
  }
  return s;
}
// A row as 16-byte vectors of VE tokens; what of its first and last one lies outside is -inf.
template <typename T>
struct ScoreRow {
  static constexpr int VE = 16 / sizeof(T);
  const char* base;  // 16-byte boundary at or below the row's first token
  int head, vocab;   // tokens between them
  __device__ __forceinline__ bool whole(int v) const { return v * VE >= head && v * VE - head + VE <= vocab; }
  __device__ __forceinline__ uint4 load(int v) const {
    if (whole(v)) return *reinterpret_cast<const uint4*>(base + (long long)v * 16);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        const int e = v * VE - head + i;
        w[i] = e >= 0 && e < vocab ? reinterpret_cast<const uint32_t*>(base)[(long long)v * VE + i] : kNone;
      } else {
        w[i] = kNone;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int e = v * VE - head + 2 * i + h;
          if (e >= 0 && e < vocab)
            w[i] = __byte_perm(w[i], reinterpret_cast<const uint16_t*>(base)[(long long)v * VE + 2 * i + h],
                               h ? 0x5410 : 0x3254);
        }
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // -inf, or a pair of them
  static constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  static __device__ __forceinline__ uint4 none() { return make_uint4(kNone, kNone, kNone, kNone); }
  // Pair i of a vector.
  static __device__ __forceinline__ float2 pair(const uint4& u, int i) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    else return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  static __device__ __forceinline__ float2 pair_at(const uint4& u, int i) {  // (an index of run time)
    const uint32_t w = i & 2 ? (i & 1 ? u.w : u.z) : (i & 1 ? u.y : u.x);
    if constexpr (sizeof(T) == 4) return i ? make_float2(__uint_as_float(u.z), __uint_as_float(u.w)) : pair(u, 0);
    else return pair(make_uint4(w, 0, 0, 0), 0);
  }
  // A bound below which a weight by the maximum m is 0, as a pair of T: a finite one, so that d e^d is 0 there too.
  // (There is none for a maximum next to the type's lowest value.)
  static constexpr float kLow = sizeof(T) == 4 ? -3.402823466e38f : std::is_same<T, __half>::value ? -65504.0f : -3.389531389e38f;
  static __device__ __forceinline__ bool has_floor(float m) { return m - kLow > 150.0f; }
  static __device__ __forceinline__ uint32_t floor_of(float m) {
    const float f = fmaxf(m - fmaf(fabsf(m), 0.125f, 1.0e4f), kLow);
    if constexpr (sizeof(T) == 4) {
      return __float_as_uint(f);
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __float2half2_rn(f);
      return *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __float2bfloat162_rn(f);
      return *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  // Word i of a vector, its numbers at least `floor` (NaN stays).
  static __device__ __forceinline__ uint32_t lifted(uint32_t w, uint32_t floor) {
    if constexpr (sizeof(T) == 4) {
      float r;
      asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(w)), "f"(__uint_as_float(floor)));
      return __float_as_uint(r);
    } else {
      using V = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      const V h = __hmax2_nan(*reinterpret_cast<const V*>(&w), *reinterpret_cast<const V*>(&floor));
      return *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  // The largest of a vector that is a number (-inf where none is).
  static __device__ __forceinline__ float most(const uint4& u) {
    if constexpr (sizeof(T) == 4) {
      return fmaxf(fmaxf(fmaxf(__uint_as_float(u.x), -INFINITY), __uint_as_float(u.y)),
                   fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
    } else {
      using V = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      const V a = __hmax2(*reinterpret_cast<const V*>(&u.x), *reinterpret_cast<const V*>(&u.y));
      const V b = __hmax2(*reinterpret_cast<const V*>(&u.z), *reinterpret_cast<const V*>(&u.w));
      const V c = __hmax2(a, b);
      const float2 f = pair(make_uint4(*reinterpret_cast<const uint32_t*>(&c), 0, 0, 0), 0);
      return fmaxf(fmaxf(f.x, -INFINITY), f.y);
    }
  }
};

struct ScoreShared {
  ScoreSums warp[kScoreThreads / 32];
  float groups[kScoreGroups];  // this CTA's maxima
  u64 best[kScoreTop];         // this CTA's largest tokens in order, 0 behind the last
  float border, M, log_s;
  int listed, batches;
  u64 red[kScoreThreads / 32];
  u64 list[kScoreList];
  float most[kScoreSlots][kScoreThreads];              // of each thread's batches
  unsigned short again[kScoreSlots * kScoreThreads];   // batches that hold what reaches the border
};

// Position in the order of sample_rows: larger first.
__device__ __forceinline__ u64 score_key(float x, int i) { return (u64)row_key(x) << 32 | (uint32_t)~i; }

template <typename T>
__global__ void __launch_bounds__(kScoreThreads, 4) k_score_rows(const __grid_constant__ ScoreArgs a) {
  using Row = ScoreRow<T>;
  constexpr int VE = Row::VE, U = kScoreUnroll, kSlots = kScoreSlots, N = kScoreThreads;
  __shared__ ScoreShared sh;
  cg::cluster_group cl = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank(), r = blockIdx.x / C, K = a.top;
  auto meet = [&] {  // of the row's CTAs
    if (C > 1) cl.sync();
    else __syncthreads();
  };
  pdl_wait();
  pdl_trigger();
  Row row;
  {
    const char* at = static_cast<const char*>(a.logits) + r * a.row_stride * (long long)sizeof(T);
    const int off = (int)(reinterpret_cast<uintptr_t>(at) & 15);
    row.base = at - off;
    row.head = off / (int)sizeof(T);
    row.vocab = a.vocab;
  }
  const int nv = (row.head + a.vocab + VE - 1) / VE;
  const int v0 = min(rank * a.per, nv), v1 = min(v0 + a.per, nv);
  float given = 0.0f;
  int token = 0;
  if (rank == 0 && tid == 32) {
    token = a.tokens[r];
    if ((unsigned)token < (unsigned)a.vocab) given = rows_value<T>(row.base, (long long)row.head + token);
  }

  ScoreSums s{-INFINITY, 0.0f, 0.0f};
  {
    float2 s0 = make_float2(0.f, 0.f), s1 = s0;
    int slot = 0;
    // vectors [vb, ve) lie wholly inside the row and this share
    const int vb = max(v0, row.head > 0), ve = row.whole(nv - 1) ? v1 : min(v1, nv - 1);
    uint4 next[U];
    auto fetch = [&](int v) {
      if (v >= vb && v + (U - 1) * N < ve) {
#pragma unroll
        for (int k = 0; k < U; ++k) next[k] = *reinterpret_cast<const uint4*>(row.base + (long long)(v + k * N) * 16);
      } else {
#pragma unroll
        for (int k = 0; k < U; ++k) next[k] = v + k * N < v1 ? row.load(v + k * N) : Row::none();
      }
    };
    fetch(v0 + tid);
    for (int v = v0 + tid; v < v1; v += U * N) {
      uint4 x[U];
#pragma unroll
      for (int k = 0; k < U; ++k) x[k] = next[k];
      if (v + U * N < v1) fetch(v + U * N);
      float mx = Row::most(x[0]);
#pragma unroll
      for (int k = 1; k < U; ++k) mx = fmaxf(mx, Row::most(x[k]));
      // (more batches than slots: a slot stands for several)
      sh.most[slot][tid] = v - (v0 + tid) < kSlots * U * N ? mx : fmaxf(mx, sh.most[slot][tid]);
      slot = slot + 1 == kSlots ? 0 : slot + 1;
      if (mx > s.m) {
        float d;
        const float f = score_shift(s.m, mx, d);
        s1 = make_float2(fmaf(d, s0.x, s1.x) * f, fmaf(d, s0.y, s1.y) * f);
        s0 = make_float2(s0.x * f, s0.y * f);
        s.m = mx;
      }
      // (before the first finite value: everything -inf, or NaN, which stays NaN)
      const float m = s.m == -INFINITY ? 0.0f : s.m;
      if (!Row::has_floor(m)) {  // (a mask of the lowest value that covers the whole batch)
        for (int k = 0; k < U * VE / 2; ++k) {
          const int w = v + k / (VE / 2) * N;
          const float2 f = w < v1 ? Row::pair_at(row.load(w), k % (VE / 2)) : make_float2(-INFINITY, -INFINITY);
          const float dx = f.x - m, dy = f.y - m, ex = score_exp2(dx * kLog2E), ey = score_exp2(dy * kLog2E);
          s0 = __fadd2_rn(s0, make_float2(ex, ey));
          s1 = __fadd2_rn(s1, make_float2(ex > 0.0f ? dx * ex : 0.0f, ey > 0.0f ? dy * ey : 0.0f));
        }
        continue;
      }
      const uint32_t floor = Row::floor_of(m);
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const uint4 u = make_uint4(Row::lifted(x[k].x, floor), Row::lifted(x[k].y, floor), Row::lifted(x[k].z, floor),
                                   Row::lifted(x[k].w, floor));
#pragma unroll
        for (int i = 0; i < VE / 2; ++i) {
          const float2 d = __fadd2_rn(Row::pair(u, i), make_float2(-m, -m));
          const float2 y = __fmul2_rn(d, make_float2(kLog2E, kLog2E));
          const float2 e = make_float2(score_exp2(y.x), score_exp2(y.y));
          s0 = __fadd2_rn(s0, e);
          s1 = __ffma2_rn(d, e, s1);
        }
      }
    }
    s.s0 = s0.x + s0.y;
    s.s1 = s1.x + s1.y;
  }
  // maxima of the row's groups of `per` neighbouring threads
  const int per = N * C / kScoreGroups, mine = N / per;  // (groups of this CTA)
  float top = s.m;
  for (int o = 1; o < per; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane % per == 0) sh.groups[tid / per] = top;
  s = score_join(s);
  if (lane == 0) sh.warp[warp] = s;
  if (tid == 0) sh.listed = sh.batches = 0;
  if (tid < kScoreTop) sh.best[tid] = 0;
  meet();

  if (warp == 1 && rank == 0) {  // the whole row's sums
    s = ScoreSums{-INFINITY, 0.0f, 0.0f};
    for (int i = lane; i < C * (N / 32); i += 32) {
      const ScoreSums o = cl.map_shared_rank(&sh, i / (N / 32))->warp[i % (N / 32)];
      const float mn = fmaxf(s.m, o.m);
      float ds, d;
      const float fs = score_shift(s.m, mn, ds), f = score_shift(o.m, mn, d);
      s = ScoreSums{mn, s.s0 * fs + o.s0 * f, fmaf(ds, s.s0, s.s1) * fs + fmaf(d, o.s0, o.s1) * f};
    }
    s = score_join(s);
    const float log_s = logf(s.s0);
    if (lane == 0) {
      const float none = __int_as_float(0x7fffffff), h = log_s - s.s1 / s.s0;
      a.logprobs[r] = (unsigned)token < (unsigned)a.vocab ? (given - s.m) - log_s : none;
      if (a.entropy) a.entropy[r] = s.m == -INFINITY ? none : h < 0.0f ? 0.0f : h;  // (NaN stays)
      sh.M = s.m;
      sh.log_s = log_s;
    }
  }
  if (K > 0) {
    if (warp == 0) {
      // The border, from the top bit down: the largest key that K groups reach, or of 12 bits or more one that no other
      // group reaches. (To the type's last bit: with f32 keys of 16 bits a row whose values lie close together beside
      // their size, as under a common offset, had tens of thousands of tokens at the border, and each of the largest
      // took a pass.)
      constexpr int kLast = sizeof(T) == 4 ? 0 : std::is_same<T, __half>::value ? 13 : 16;
      uint32_t key[kScoreGroups / 32];
#pragma unroll
      for (int i = 0; i < kScoreGroups / 32; ++i) {
        const int at = i * 32 + lane;
        key[i] = row_key(cl.map_shared_rank(&sh, at / mine)->groups[at % mine]);
      }
      uint32_t low = 0;
#pragma unroll
      for (int bit = 31; bit >= kLast; --bit) {
        const uint32_t want = low | 1u << bit;
        int reach = 0;
#pragma unroll
        for (int i = 0; i < kScoreGroups / 32; ++i) reach += key[i] >= want;
        reach = __reduce_add_sync(0xffffffffu, reach);
        if (reach >= K) low = want;
        if (bit <= 20 && reach == K) break;
      }
      if (lane == 0) sh.border = low > 0x007fffffu ? row_key_value(low) : -INFINITY;  // (the key of -inf)
    }
    __syncthreads();
    const float border = sh.border;
    // A border of -inf: fewer than `top` groups hold anything above it. Then all that is above it is listed, and of
    // what is not, the first few by index, which is their order.
    const bool few = border == -INFINITY;
    const int first = v0 * VE - row.head, last = min(v1 * VE - row.head, a.vocab);  // this CTA's tokens (first may be < 0)
    auto put = [&](int at, u64 key) {
      a.top_ids[(long long)r * K + at] = (int)~(uint32_t)key;
      a.top_logprobs[(long long)r * K + at] = (row_key_value((uint32_t)(key >> 32)) - sh.M) - sh.log_s;
    };
    auto list = [&](float x, int i) {
      const int at = atomicAdd(&sh.listed, 1);
      if (at < kScoreList) sh.list[at] = score_key(x, i);
    };
    // The batches that reach it, and then their vectors side by side (one trip to memory, where a thread's own
    // batches in turn took a trip per vector: 512 rows of bf16 60 us).
    for (int i = 0; i < kSlots && v0 + tid + i * U * N < v1; ++i)
      if (sh.most[i][tid] >= border) sh.again[atomicAdd(&sh.batches, 1)] = (unsigned short)(i * N + tid);
    __syncthreads();
    for (int j = tid; j < sh.batches * U; j += N) {
      const int at = sh.again[j / U];
      for (int w = v0 + at % N + (at / N * U + j % U) * N; w < v1; w += kSlots * U * N) {
        const uint4 x = row.load(w);
        if (!(Row::most(x) >= border)) continue;
#pragma unroll
        for (int c = 0; c < VE / 2; ++c) {
          const float2 f = Row::pair(x, c);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float y = h ? f.y : f.x;
            const int e = w * VE - row.head + 2 * c + h;
            if (few ? y > -INFINITY || (y == -INFINITY && e >= 0 && e < last && e < first + kScoreList / 2) : y >= border)
              list(y, e);
          }
        }
      }
    }
    __syncthreads();
    int n = sh.listed;
    bool whole = n <= kScoreList && (!few || n >= K || n == last - max(first, 0));
    if (!whole) {
      // Too many (a mask that leaves much of this CTA's share and little else, say): all of the share once more, with a
      // border of its own, the top-th largest of its threads' maxima. (6 rows of 151936 tokens of which a mask leaves 5000
      // neighbours: one after the other, as below, the largest 20 took 105 us, so 30. 600 rows of 32000 whose positive
      // tokens 40 threads hold, the largest 21: 657 and 51 us.)
      __syncthreads();
      if (warp == 0) {
        uint32_t key[N / 32], low = 0;
        for (int k = 0; k < N / 32; ++k) {
          const int t = 32 * k + lane;
          float most = -INFINITY;
          for (int i = 0; i < kSlots && v0 + t + i * U * N < v1; ++i) most = fmaxf(most, sh.most[i][t]);
          key[k] = row_key(most);
        }
#pragma unroll 1
        for (int bit = 31; bit >= 0; --bit) {
          const uint32_t want = low | 1u << bit;
          int reach = 0;
          for (int k = 0; k < N / 32; ++k) reach += key[k] >= want;
          if (__reduce_add_sync(0xffffffffu, reach) >= K) low = want;
        }
        if (lane == 0) {
          sh.border = low > 0x007fffffu ? row_key_value(low) : -INFINITY;
          sh.listed = 0;
        }
      }
      __syncthreads();
      const float own = sh.border;
      if (own > -INFINITY) {
        for (int v = v0 + tid; v < v1; v += N) {
          const uint4 x = row.load(v);
          if (!(Row::most(x) >= own)) continue;
          for (int i = 0; i < VE; ++i) {
            const float2 f = Row::pair_at(x, i / 2);
            const float y = i & 1 ? f.y : f.x;
            if (y >= own) list(y, v * VE - row.head + i);
          }
        }
      }
      __syncthreads();
      n = sh.listed;
      whole = own > -INFINITY && n <= kScoreList;
    }
    if (whole) {
      for (int i = tid; i < n; i += N) {
        const u64 mine = sh.list[i];
        int before = 0;
        for (int j = 0; j < n; ++j) before += sh.list[j] > mine;
        if (before < K) {
          if (C == 1) put(before, mine);
          else sh.best[before] = mine;
        }
      }
    } else {  // values that occur a thousand times: one after the other
      u64 below = ~0ull;
      for (int k = 0; k < K; ++k) {
        u64 best = 0;
        for (int v = v0 + tid; v < v1; v += N) {
          const uint4 x = row.load(v);
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            const int e = v * VE - row.head + i;
            const float2 f = Row::pair(x, i / 2);
            const u64 key = score_key(i & 1 ? f.y : f.x, e);
            if (e >= 0 && e < last && key < below && key > best) best = key;
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (lane == 0) sh.red[warp] = best;
        __syncthreads();
        best = sh.red[lane % (N / 32)];
#pragma unroll
        for (int o = (N / 32) / 2; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (best == 0) break;  // (the same in every thread)
        if (tid == 0) {
          if (C == 1) put(k, best);
          else sh.best[k] = best;
        }
        below = best;
        __syncthreads();
      }
    }
    if (C > 1) cl.sync();
    if (C > 1 && rank == 0) {  // the CTAs' largest in order
      const int m = C * K;
      for (int i = tid; i < m; i += N) sh.list[i] = cl.map_shared_rank(&sh, i / K)->best[i % K];
      __syncthreads();
      for (int i = tid; i < m; i += N) {
        const u64 mine = sh.list[i];
        int before = 0;
        for (int j = 0; j < m; ++j) before += sh.list[j] > mine;
        if (mine != 0 && before < K) put(before, mine);
      }
    }
  }
  if (C > 1) cl.sync();  // shared memory is read by others until here
}

template <typename T>
static void launch_score_rows(ScoreArgs a, int rows, cudaStream_t s) {
  constexpr int VE = 16 / sizeof(T);
  // CTAs per row: as many as fill the GPU twice (a CTA pays 4 us beside its loads: 512 rows of bf16 40 us with one,
  // 44 with two, 94 with eight; 64 rows of f32 37, 23 and 15.5), but 2048 tokens are not split.
  int C = 1;
  while (C < kScoreCluster && (long long)rows * C < 2 * current_sms() && (a.vocab + C - 1) / C > 2048) C *= 2;
  a.per = ((a.vocab + VE - 1) / VE + 1 + C - 1) / C;  // (a row that starts inside a vector has one more)
  if ((long long)rows * C > 0x7fffffffLL) throw QdError{QD_E_RANGE, "qd_score_rows: too many rows"};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * C));
  cfg.blockDim = dim3(kScoreThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  QD_CK(cudaLaunchKernelEx(&cfg, k_score_rows<T>, a));
}
}  // namespace qd

extern "C" int qd_score_rows(const void* logits, int dtype, int rows, uint32_t vocab, int64_t row_stride,
                             const int32_t* tokens, int top, float* logprobs, float* entropy, int32_t* top_ids,
                             float* top_logprobs, void* stream) {
  try {
    using namespace qd;
    if (rows < 0 || vocab == 0) throw QdError{QD_E_INVALID, "qd_score_rows: bad rows or vocab"};
    if (vocab > 0x40000000u) throw QdError{QD_E_RANGE, "qd_score_rows: vocab beyond 2^30"};
    if (dtype != QD_KV_F32 && dtype != QD_KV_F16 && dtype != QD_KV_BF16)
      throw QdError{QD_E_INVALID, "qd_score_rows: unknown dtype"};
    if (row_stride < (int64_t)vocab) throw QdError{QD_E_INVALID, "qd_score_rows: row_stride below vocab"};
    if (top < 0 || top > kScoreTop || (uint32_t)top > vocab)
      throw QdError{QD_E_INVALID, "qd_score_rows: top must be 0..64, at most vocab"};
    if (rows == 0) return QD_OK;
    if (!logits || !tokens || !logprobs || (top && (!top_ids || !top_logprobs)))
      throw QdError{QD_E_INVALID, "qd_score_rows: NULL argument"};
    const int64_t size = dtype == QD_KV_F32 ? 4 : 2, n = rows;
    const Rows in{logits, n, (int64_t)vocab * size, row_stride * size}, given{tokens, 1, n * 4, n * 4};
    for (const Rows& out : {Rows{logprobs, 1, n * 4, n * 4}, Rows{entropy, entropy ? 1 : 0, n * 4, n * 4},
                            Rows{top_ids, top ? 1 : 0, n * top * 4, n * top * 4},
                            Rows{top_logprobs, top ? 1 : 0, n * top * 4, n * top * 4}})
      if (!apart(out, in) || !apart(out, given))
        throw QdError{QD_E_INVALID, "qd_score_rows: an output overlaps logits or tokens"};
    ScoreArgs a{logits, (int)vocab, 0, row_stride, tokens, top, logprobs, entropy, top_ids, top_logprobs};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == QD_KV_F32) launch_score_rows<float>(a, rows, s);
    else if (dtype == QD_KV_F16) launch_score_rows<__half>(a, rows, s);
    else launch_score_rows<__nv_bfloat16>(a, rows, s);
  } catch (const qd::QdError& err) {
    qd::set_thread_error(err.msg);
    return err.code;
  } catch (const std::exception& err) {
    qd::set_thread_error(err.what());
    return QD_E_NOMEM;
  }
  return QD_OK;
}
