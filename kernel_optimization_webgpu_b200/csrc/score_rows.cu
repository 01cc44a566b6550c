// Per row of logits: the log probability of a given token, the entropy of the softmax, and the largest tokens.
//
//   log p_t = x_t - m - log S,  H = log S - sum (x - m) e^(x - m) / S,  S = sum e^(x - m),  m = max x
//
// One thread-block cluster per row, a contiguous share per CTA, read once from memory: each thread keeps a running
// maximum, S and the entropy's sum by it (in base 2), joined over warps, CTAs and the cluster at the end. The
// largest tokens need a border first, below which nothing has to be looked at: the row's threads form 128 groups,
// and the top-th largest of the groups' maxima is a value that at least `top` tokens reach and that
// hardly more than those do. A second look at the CTA's share (in L1 by now) lists what reaches it; the lists, a few
// tokens each, are put in order by counting.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/qdecode.h"
#include "internal.cuh"
#include "rows.cuh"

namespace qd {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int kScoreThreads = 512;
constexpr int kScoreWarps = kScoreThreads / 32;
constexpr int kScoreCluster = 8;
constexpr int kScoreTop = 64;     // largest `top`
constexpr int kScoreGroups = 128;  // of a row's threads: at least kScoreTop
constexpr int kScoreList = 1024;  // tokens at or above the border that a CTA lists
constexpr int kScoreUnroll = 4;   // 16-byte loads in flight per thread

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

// Sums by a maximum: s0 = sum 2^y, s1 = sum y 2^y, y = (x - m) log2 e.
struct ScoreSums {
  float m, s0, s1;
};
__device__ __forceinline__ float score_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The same sums by the maximum mn >= s.m.
__device__ __forceinline__ ScoreSums score_by(ScoreSums s, float mn) {
  const float d = s.m == mn || s.m == -INFINITY ? 0.0f : fmaxf((s.m - mn) * 1.4426950408889634f, -200.0f);
  const float f = s.m == -INFINITY ? 0.0f : score_exp2(d);
  return ScoreSums{mn, s.s0 * f, fmaf(d, s.s0, s.s1) * f};
}
__device__ __forceinline__ ScoreSums score_join(ScoreSums a, ScoreSums b) {
  const float mn = fmaxf(a.m, b.m);
  a = score_by(a, mn);
  b = score_by(b, mn);
  return ScoreSums{mn, a.s0 + b.s0, a.s1 + b.s1};
}
__device__ __forceinline__ float score_max_nan(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}

template <typename T>
struct ScoreRow {
  static constexpr int VE = 16 / sizeof(T);
  const char* base;  // 16-byte boundary at or below the row's first element
  int head, vocab;   // elements between them
  // Vector v: elements v * VE - head ..; what lies outside the row is -inf.
  __device__ __forceinline__ bool whole(int v) const { return v * VE >= head && v * VE - head + VE <= vocab; }
  __device__ __forceinline__ void load(int v, float (&x)[VE]) const {
    if (whole(v)) {
      const uint4 u = *reinterpret_cast<const uint4*>(base + (long long)v * 16);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
          x[i] = __uint_as_float(w[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          x[2 * i] = f.x;
          x[2 * i + 1] = f.y;
        } else {
          x[2 * i] = __uint_as_float(w[i] << 16);
          x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const int e = v * VE - head + i;
        x[i] = e >= 0 && e < vocab ? rows_value<T>(base, (long long)v * VE + i) : -INFINITY;
      }
    }
  }
};

struct ScoreShared {
  ScoreSums sums;               // this CTA's
  ScoreSums warp[kScoreWarps];
  float groups[kScoreGroups];   // this CTA's maxima (kScoreGroups / C of them)
  u64 best[kScoreTop];          // this CTA's largest tokens in order, 0 behind the last
  float all[kScoreGroups];      // the row's
  float border;
  int listed;
  u64 red[kScoreWarps];
  u64 list[kScoreList];
};

// Position in the order of sample_rows: larger first.
__device__ __forceinline__ u64 score_key(float x, int i) { return (u64)row_key(x) << 32 | (uint32_t)~i; }

template <typename T>
__global__ void __launch_bounds__(kScoreThreads, 2) k_score_rows(const __grid_constant__ ScoreArgs a) {
  constexpr int VE = 16 / sizeof(T), U = kScoreUnroll;
  __shared__ ScoreShared sh;
  cg::cluster_group cl = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank(), r = blockIdx.x / C, K = a.top;
  pdl_wait();
  pdl_trigger();
  ScoreRow<T> row;
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
  if (rank == 0 && tid == 0) {
    token = a.tokens[r];
    if ((unsigned)token < (unsigned)a.vocab) given = rows_value<T>(row.base, (long long)row.head + token);
  }

  ScoreSums s{-INFINITY, 0.0f, 0.0f};
  for (int v = v0 + tid; v < v1; v += U * kScoreThreads) {
    float x[U][VE];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (v + k * kScoreThreads < v1) {
        row.load(v + k * kScoreThreads, x[k]);
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) x[k][i] = -INFINITY;
      }
    }
    float mx = x[0][0];
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int i = 0; i < VE; ++i) mx = fmaxf(mx, x[k][i]);
    if (mx > s.m) s = score_by(s, mx);
    // (before the first finite value: everything -inf, or NaN, which stays NaN)
    const float m = s.m == -INFINITY ? 0.0f : s.m;
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        // below 2^-126 a weight is as good as none, and its place in the entropy's sum stays finite
        const float y = score_max_nan((x[k][i] - m) * 1.4426950408889634f, -126.0f);
        const float e = score_exp2(y);
        s.s0 += e;
        s.s1 = fmaf(y, e, s.s1);
      }
  }
  // maxima of the row's 128 groups of 4 C neighbouring threads
  float top = s.m;
  for (int o = 1; o < 4 * C; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane % (4 * C) == 0) sh.groups[tid / (4 * C)] = top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    s = score_join(s, ScoreSums{__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.s0, o),
                                __shfl_xor_sync(0xffffffffu, s.s1, o)});
  if (lane == 0) sh.warp[warp] = s;
  __syncthreads();
  if (warp == 0) {
    s = sh.warp[lane % kScoreWarps];
#pragma unroll
    for (int o = kScoreWarps / 2; o > 0; o >>= 1)
      s = score_join(s, ScoreSums{__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.s0, o),
                                  __shfl_xor_sync(0xffffffffu, s.s1, o)});
    if (lane == 0) sh.sums = s;
  }
  cl.sync();

  float M = 0.0f, log_s = 0.0f;
  if (rank == 0) {  // the whole row's sums, in the order of the CTAs
    s = cl.map_shared_rank(&sh, 0)->sums;
    for (int c = 1; c < C; ++c) s = score_join(s, cl.map_shared_rank(&sh, c)->sums);
    M = s.m;
    log_s = logf(s.s0);
    if (tid == 0) {
      const float none = __int_as_float(0x7fffffff);
      a.logprobs[r] = (unsigned)token < (unsigned)a.vocab ? (given - M) - log_s : none;
      const float h = fmaf(-0.6931471805599453f, s.s1 / s.s0, log_s);
      if (a.entropy) a.entropy[r] = M == -INFINITY ? none : h < 0.0f ? 0.0f : h;  // (NaN stays)
    }
  }
  if (K > 0) {
    if (tid < kScoreGroups) sh.all[tid] = cl.map_shared_rank(&sh, tid / (kScoreGroups / C))->groups[tid % (kScoreGroups / C)];
    if (tid < kScoreTop) sh.best[tid] = 0;
    if (tid == 0) sh.listed = 0;
    __syncthreads();
    if (tid < kScoreGroups) {
      const float mine = sh.all[tid];
      int before = 0;
      for (int j = 0; j < kScoreGroups; ++j) before += sh.all[j] > mine || (sh.all[j] == mine && j < tid);
      if (before == K - 1) sh.border = mine;
    }
    __syncthreads();
    const float border = sh.border;
    // A border of -inf: fewer than `top` groups hold anything above it. Then all that is above it is listed, and of
    // what is not, the first few by index, which is their order.
    const bool few = border == -INFINITY;
    const int first = v0 * VE - row.head, last = min(v1 * VE - row.head, a.vocab);  // this CTA's tokens (first may be < 0)
    auto list = [&](float x, int i) {
      const int at = atomicAdd(&sh.listed, 1);
      if (at < kScoreList) sh.list[at] = score_key(x, i);
    };
    for (int v = v0 + tid; v < v1; v += kScoreThreads) {
      float x[VE];
      row.load(v, x);
      float mx = x[0];
#pragma unroll
      for (int i = 1; i < VE; ++i) mx = fmaxf(mx, x[i]);
      if (mx >= border) {
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const int e = v * VE - row.head + i;
          if (few ? x[i] > -INFINITY || (x[i] == -INFINITY && e >= 0 && e < last && e < first + kScoreList / 2) : x[i] >= border)
            list(x[i], e);
        }
      }
    }
    __syncthreads();
    const int n = sh.listed;
    if (n <= kScoreList && (!few || n >= K || n == last - max(first, 0))) {
      for (int i = tid; i < n; i += kScoreThreads) {
        const u64 mine = sh.list[i];
        int before = 0;
        for (int j = 0; j < n; ++j) before += sh.list[j] > mine;
        if (before < K) sh.best[before] = mine;
      }
    } else {  // too many tokens reach the border (long classes of equal values): one after the other
      u64 below = ~0ull;
      for (int k = 0; k < K; ++k) {
        u64 best = 0;
        for (int v = v0 + tid; v < v1; v += kScoreThreads) {
          float x[VE];
          row.load(v, x);
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            const int e = v * VE - row.head + i;
            const u64 key = score_key(x[i], e);
            if (e >= 0 && e < last && key < below && key > best) best = key;
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (lane == 0) sh.red[warp] = best;
        __syncthreads();
        best = sh.red[lane % kScoreWarps];
#pragma unroll
        for (int o = kScoreWarps / 2; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (best == 0) break;  // (the same in every thread)
        if (tid == 0) sh.best[k] = best;
        below = best;
        __syncthreads();
      }
    }
    cl.sync();
    if (rank == 0) {  // the CTAs' largest in order
      const int m = C * K;
      if (tid < m) sh.list[tid] = cl.map_shared_rank(&sh, tid / K)->best[tid % K];
      __syncthreads();
      if (tid < m) {
        const u64 mine = sh.list[tid];
        int before = 0;
        for (int j = 0; j < m; ++j) before += sh.list[j] > mine;
        if (mine != 0 && before < K) {
          a.top_ids[(long long)r * K + before] = (int)~(uint32_t)mine;
          a.top_logprobs[(long long)r * K + before] = (row_key_value((uint32_t)(mine >> 32)) - M) - log_s;
        }
      }
    }
  }
  cl.sync();  // shared memory is read by others until here
}

template <typename T>
static void launch_score_rows(ScoreArgs a, int rows, cudaStream_t s) {
  constexpr int VE = 16 / sizeof(T);
  int C = 1;
  while (C < kScoreCluster && ((a.vocab + C - 1) / C > 20480 ||
                               ((long long)rows * C < 2 * current_sms() && (a.vocab + C - 1) / C > 2048)))
    C *= 2;
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
