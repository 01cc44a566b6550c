// One token per row of logits, every row with its own temperature, top-k, top-p, min-p and
// given random number, over the whole vocabulary.
//
// The tokens that survive the cuts are always a prefix of the row's order (value, then lower
// index), and the drawn token ends a prefix too, so each step is the same question: where
// does a running count, or a running sum of weights, first pass a target? It is answered on
// order-preserving integer keys. The weights w = exp((v - v_max) / T) are 44-bit fixed-point
// numbers from a double-precision exponential and are summed as 64-bit integers: exact, so
// the answer does not depend on the order of summation, and a border is misplaced only where
// the random number falls within about 2^-40 of it.
#include <cmath>
#include <string>

#include "../../include/qdecode.h"
#include "internal.cuh"
#include "paged.cuh"

namespace qd {

typedef unsigned long long u64;

constexpr int kRowsThreads = 1024;
constexpr int kRowsMaxVocab = 393216;
constexpr double kRowsOne = 17592186044416.0;  // weight 1 = 2^44

struct SampleRowsArgs {
  const void* logits;
  int vocab;
  long long row_stride;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  int* ids;
  float* logprobs;
};

template <typename T>
__device__ __forceinline__ float row_value(const void* p, long long i);
template <>
__device__ __forceinline__ float row_value<float>(const void* p, long long i) {
  return static_cast<const float*>(p)[i];
}
template <>
__device__ __forceinline__ float row_value<__half>(const void* p, long long i) {
  return __half2float(static_cast<const __half*>(p)[i]);
}
template <>
__device__ __forceinline__ float row_value<__nv_bfloat16>(const void* p, long long i) {
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// Larger value, larger key; -0 as +0; NaN 0, below every number.
__device__ __forceinline__ uint32_t row_key(float v) {
  if (v != v) return 0u;
  const uint32_t u = __float_as_uint(v + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float row_key_value(uint32_t k) {
  if (k == 0u) return __int_as_float(0x7fc00000);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

__device__ __forceinline__ u64 row_weight(uint32_t key, double vmax, double inv_t) {
  if (key == 0u) return 0ull;
  return (u64)__double2ll_rn(exp(((double)row_key_value(key) - vmax) * inv_t) * kRowsOne);
}

__device__ u64 rows_sum(u64 v, u64* sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 t = 0;
  for (int w = 0; w < kRowsThreads / 32; ++w) t += sm[w];
  return t;
}

// A prefix of the row's order: every key above `key`, and the first `ties` of those equal to it.
struct RowPrefix {
  uint32_t key;
  u64 ties;
};

// One CTA per row; every question is answered by bisecting the 32-bit key.
template <typename T>
__global__ void __launch_bounds__(kRowsThreads) k_sample_rows(const __grid_constant__ SampleRowsArgs a) {
  __shared__ u64 sm[kRowsThreads / 32];
  const int r = blockIdx.x, tid = threadIdx.x;
  pdl_wait();
  const long long base = r * a.row_stride;
  const float temperature = a.temperature ? a.temperature[r] : 1.0f;
  const int top_k = a.top_k ? a.top_k[r] : 0;
  const float top_p = a.top_p ? a.top_p[r] : 1.0f, min_p = a.min_p ? a.min_p[r] : 0.0f;
  const float u = a.u[r];
  const double inv_t = 1.0 / (double)temperature;
  double vmax = 0.0;
  // sum over keys in [lo, hi] of weights (by = 0) or of ones (by = 1)
  auto over = [&](uint32_t lo, uint32_t hi, bool count) {
    u64 s = 0;
    for (int i = tid; i < a.vocab; i += kRowsThreads) {
      const uint32_t k = row_key(row_value<T>(a.logits, base + i));
      if (k >= lo && k <= hi) s += count ? 1ull : row_weight(k, vmax, inv_t);
    }
    return rows_sum(s, sm);
  };
  // the key at which the sum over keys >= key first reaches `goal` (goal <= the whole sum, > 0)
  auto find = [&](u64 goal, bool count) {
    uint32_t lo = 0u, hi = 0xffffffffu;
    while (lo < hi) {
      const uint32_t mid = lo + ((hi - lo) >> 1) + 1u;
      if (over(mid, 0xffffffffu, count) >= goal) lo = mid;
      else hi = mid - 1u;
    }
    return lo;
  };
  // index of the n-th (from 0) token whose key is `key`
  auto nth = [&](uint32_t key, u64 n) {
    int lo = 0, hi = a.vocab - 1;
    while (lo < hi) {
      const int mid = lo + (hi - lo) / 2;
      u64 s = 0;
      for (int i = tid; i <= mid; i += kRowsThreads) s += row_key(row_value<T>(a.logits, base + i)) == key;
      if (rows_sum(s, sm) > n) hi = mid;
      else lo = mid + 1;
    }
    return lo;
  };
  const uint32_t kmax = find(1, true);
  const float vm = row_key_value(kmax);
  if (!(temperature > 0.0f) || top_k == 1 || !(fabsf(vm) < INFINITY)) {
    const int id = nth(kmax, 0);
    if (tid == 0) {
      a.ids[r] = id;
      if (a.logprobs) a.logprobs[r] = 0.0f;
    }
    return;
  }
  vmax = (double)vm;
  auto mass = [&](RowPrefix p) {
    return (p.key == 0xffffffffu ? 0ull : over(p.key + 1u, 0xffffffffu, false)) +
           p.ties * row_weight(p.key, vmax, inv_t);
  };
  RowPrefix keep{0u, (u64)a.vocab};
  keep.ties = over(0u, 0u, true);
  if (top_k > 0 && top_k < a.vocab) {
    keep.key = find(top_k, true);
    keep.ties = top_k - (keep.key == 0xffffffffu ? 0ull : over(keep.key + 1u, 0xffffffffu, true));
  }
  auto shorter = [](RowPrefix x, RowPrefix y) {
    return x.key > y.key || (x.key == y.key && x.ties < y.ties) ? x : y;
  };
  u64 total = mass(keep);
  if (top_p < 1.0f) {
    const double goal = fmax((double)top_p, 0.0) * (double)total;
    const u64 g = max((u64)ceil(goal), 1ull);
    const uint32_t k = find(g, false);
    const u64 above = k == 0xffffffffu ? 0ull : over(k + 1u, 0xffffffffu, false), w = row_weight(k, vmax, inv_t);
    keep = shorter(RowPrefix{k, (g - above + w - 1) / w}, keep);
  }
  if (min_p > 0.0f) {
    // the smallest key whose value reaches v_max + T ln(min_p), never above the largest
    uint32_t lo = 1u, hi = kmax;
    while (lo < hi) {
      const uint32_t mid = lo + ((hi - lo) >> 1);
      if (exp(((double)row_key_value(mid) - vmax) * inv_t) >= (double)min_p) hi = mid;
      else lo = mid + 1u;
    }
    if (min_p > 1.0f) keep = RowPrefix{kmax, 1};
    else keep = shorter(keep, RowPrefix{lo, over(lo, lo, true)});
  }
  total = mass(keep);
  const u64 goal = min((u64)floor((double)u * (double)total), total - 1) + 1;  // running sum > u * total
  const uint32_t k = find(goal, false);
  const u64 above = k == 0xffffffffu ? 0ull : over(k + 1u, 0xffffffffu, false), w = row_weight(k, vmax, inv_t);
  const int id = nth(k, (goal - above + w - 1) / w - 1);
  if (tid == 0) {
    a.ids[r] = id;
    if (a.logprobs)
      a.logprobs[r] = (float)(((double)row_key_value(k) - vmax) * inv_t - log((double)total / kRowsOne));
  }
}

}  // namespace qd

extern "C" int qd_sample_rows(const void* logits, int dtype, int rows, uint32_t vocab, int64_t row_stride,
                              const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                              const float* u, int32_t* ids, float* logprobs, void* stream) {
  try {
    using namespace qd;
    if (rows < 0 || vocab == 0) throw QdError{QD_E_INVALID, "qd_sample_rows: bad rows or vocab"};
    if (vocab > (uint32_t)kRowsMaxVocab)
      throw QdError{QD_E_RANGE, "qd_sample_rows: vocab beyond " + std::to_string(kRowsMaxVocab)};
    if (dtype != QD_KV_F32 && dtype != QD_KV_F16 && dtype != QD_KV_BF16)
      throw QdError{QD_E_INVALID, "qd_sample_rows: unknown dtype"};
    if (row_stride < (int64_t)vocab) throw QdError{QD_E_INVALID, "qd_sample_rows: row_stride below vocab"};
    if (rows == 0) return QD_OK;
    if (!logits || !u || !ids) throw QdError{QD_E_INVALID, "qd_sample_rows: NULL argument"};
    SampleRowsArgs a{logits, (int)vocab, row_stride, temperature, top_k, top_p, min_p, u, ids, logprobs};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const dim3 grid(rows), block(kRowsThreads);
    if (dtype == QD_KV_F32) launch_ex(k_sample_rows<float>, grid, block, 0, s, a);
    else if (dtype == QD_KV_F16) launch_ex(k_sample_rows<__half>, grid, block, 0, s, a);
    else launch_ex(k_sample_rows<__nv_bfloat16>, grid, block, 0, s, a);
  } catch (const qd::QdError& err) {
    qd::set_thread_error(err.msg);
    return err.code;
  } catch (const std::exception& err) {
    qd::set_thread_error(err.what());
    return QD_E_NOMEM;
  }
  return QD_OK;
}
