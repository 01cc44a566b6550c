// One token per row of logits, every row with its own temperature, top-k, top-p, min-p and
// given random number, over the whole vocabulary.
//
// The tokens that survive the cuts are always a prefix of the row's order (value, then lower
// index), and the drawn token ends a prefix too, so each step is the same question: where
// does a running count, or a running sum of weights, first pass a target? The weights
// w = exp((v - v_max) / T) are 44-bit fixed-point numbers from a double-precision exponential,
// summed as 64-bit integers: exact, so the answer does not depend on the order of summation, and
// a border is misplaced only where the random number falls within about 2^-40 of it.
//
// One thread-block cluster per row. The row is read once, into the CTAs' shared memory; what is
// bound is then the latency of a few passes over it, so the work of a pass is spread over the
// cluster and the passes are few:
//  1. maximum and minimum;
//  2. histogram over kRowsBins equal steps of value between them (or 31 T nats, beyond which a
//     weight is zero): counts, and sums of weights where a cut needs them, by integer atomics in
//     shared memory. Steps are monotone in the value, so every border lies in a known step;
//  3. the steps that hold all tokens that can be kept, when these are at most kRowsList, are
//     gathered into the first CTA, sorted, and all cuts and the draw are done there.
// Otherwise (a large nucleus, the whole vocabulary) each border is resolved alone: the tokens of
// its step are gathered and sorted, a step with too many is cut into finer ones by key, and where
// all of them are equal their order is their index. The first CTA of the cluster leads: it
// tells the others what to do next and ends them.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <utility>

#include "../../include/qdecode.h"
#include "internal.cuh"
#include "paged.cuh"

namespace qd {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int kRowsThreads = 512;
constexpr int kRowsWarps = kRowsThreads / 32;
constexpr int kRowsMaxVocab = 393216;
constexpr int kRowsMaxCluster = 8;
constexpr int kRowsBins = 1024;   // two a thread of the leader
constexpr int kRowsList = 1024;
constexpr double kRowsOne = 17592186044416.0;  // weight 1 = 2^44

struct SampleRowsArgs {
  const void* logits;
  int vocab, per;  // per: tokens a CTA holds
  long long row_stride;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  int* ids;
  float* logprobs;
};

// Larger value, larger key.
__device__ __forceinline__ uint32_t row_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);  // -0 as +0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float row_key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// What the leader asks of every CTA.
enum RowsOp : int { kOpEnd = 0, kOpHist, kOpGather, kOpRange, kOpMass, kOpCount, kOpPick };
struct RowsCmd {
  int op;
  int by_bin;         // members: bins [lo, hi] of the first histogram; else keys [lo, hi]
  uint32_t lo, hi;
  int shift;          // kOpHist by key: bin = (hi - key) >> shift
  int rank, n;        // kOpPick: CTA `rank` finds its n-th member by index
};
// A prefix of the row's order: every key above `key` and the first `ties` of those equal to it.
struct RowsPrefix {
  uint32_t key;
  int ties;
  u64 mass;
};

struct RowsShared {
  RowsCmd cmd;
  float mx[kRowsMaxCluster], mn[kRowsMaxCluster];
  u64 part[kRowsMaxCluster];      // per-CTA sums for the leader
  uint32_t key_min, key_max;      // leader
  int found;                      // leader: an index
  int listed;                     // leader: entries of the list
  u64 red[kRowsWarps];
  u64 pick_mass;                  // results of searches over the leader's threads
  int pick_bin, pick_at;
  u64 pick_base;
  int pick_count;
};

template <typename T>
__device__ __forceinline__ float rows_value(const void* p, long long i) {
  if constexpr (sizeof(T) == 4) return static_cast<const float*>(p)[i];
  else if constexpr (std::is_same<T, __half>::value) return __half2float(static_cast<const __half*>(p)[i]);
  else return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// One CTA's view of its row.
struct RowsCta {
  cg::cluster_group cl;
  RowsShared* sh;
  float* val;      // [per], NaN as -inf
  uint4* hist;     // [kRowsBins] {count, weights in three 32-bit sums of 16 + 14 + 14 bits}
  u64* list;       // leader: {~key, index}
  int n, base, C, rank;
  float vmax, scale;
  double inv_t;

  __device__ __forceinline__ int bin(float v) const {  // ascending as v descends
    return v == -INFINITY ? kRowsBins - 1 : (int)fminf((vmax - v) * scale, (float)(kRowsBins - 1));
  }
  __device__ __forceinline__ u64 weight(float v) const {
    return v == -INFINITY ? 0ull : (u64)__double2ll_rn(exp(((double)v - (double)vmax) * inv_t) * kRowsOne);
  }
  __device__ __forceinline__ bool member(const RowsCmd& c, float v) const {
    if (c.by_bin) {
      const uint32_t b = (uint32_t)bin(v);
      return b >= c.lo && b <= c.hi;
    }
    const uint32_t k = row_key(v);
    return k >= c.lo && k <= c.hi;
  }
  __device__ u64 block_sum64(u64 v) {  // in every thread
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh->red[threadIdx.x >> 5] = v;
    __syncthreads();
    u64 t = 0;
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) t += sh->red[w];
    return t;
  }

  // Histogram of the members; afterwards this CTA's share of the bins holds the whole row's sums
  // as {count, weight low, weight high, -}.
  __device__ void histogram(const RowsCmd& c, bool mass) {
    for (int i = threadIdx.x; i < kRowsBins; i += kRowsThreads) hist[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kRowsThreads) {
      const float v = val[i];
      int b;
      if (c.by_bin) {
        b = bin(v);
      } else {
        const uint32_t k = row_key(v);
        if (k < c.lo || k > c.hi) continue;
        b = (int)((c.hi - k) >> c.shift);
      }
      atomicAdd(&hist[b].x, 1u);
      if (mass) {
        const u64 w = weight(v);
        atomicAdd(&hist[b].y, (uint32_t)w & 0xffffu);
        atomicAdd(&hist[b].z, (uint32_t)(w >> 16) & 0x3fffu);
        atomicAdd(&hist[b].w, (uint32_t)(w >> 30));
      }
    }
    cl.sync();
    const int share = kRowsBins / C;
    for (int i = threadIdx.x; i < share; i += kRowsThreads) {
      const int b = rank * share + i;
      uint32_t count = 0;
      u64 w = 0;
      for (int r = 0; r < C; ++r) {
        const uint4 h = *cl.map_shared_rank(&hist[b], r);
        count += h.x;
        w += (u64)h.y + ((u64)h.z << 16) + ((u64)h.w << 30);
      }
      hist[b] = make_uint4(count, (uint32_t)w, (uint32_t)(w >> 32), 0);
    }
  }

  // What a command makes every CTA do (the caller synchronises the cluster around it).
  __device__ void perform(const RowsCmd& c) {
    RowsShared* lead = cl.map_shared_rank(sh, 0);
    const int lane = threadIdx.x & 31;
    if (c.op == kOpHist) {
      histogram(c, true);
    } else if (c.op == kOpGather) {
      u64* out = cl.map_shared_rank(list, 0);
      for (int i0 = 0; i0 < n; i0 += kRowsThreads) {
        const int i = i0 + threadIdx.x;
        const float v = i < n ? val[i] : 0.0f;
        const bool in = i < n && member(c, v);
        const unsigned who = __ballot_sync(0xffffffffu, in);
        if (who) {
          int at = 0;
          if (lane == 0) at = atomicAdd(&lead->listed, __popc(who));
          at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1u));
          if (in && at < kRowsList) out[at] = ((u64)~row_key(v) << 32) | (unsigned)(base + i);
        }
      }
    } else if (c.op == kOpRange) {
      uint32_t lo = 0xffffffffu, hi = 0u;
      for (int i = threadIdx.x; i < n; i += kRowsThreads)
        if (member(c, val[i])) {
          const uint32_t k = row_key(val[i]);
          lo = min(lo, k);
          hi = max(hi, k);
        }
      lo = __reduce_min_sync(0xffffffffu, lo);
      hi = __reduce_max_sync(0xffffffffu, hi);
      if (lane == 0 && lo <= hi) {
        atomicMin(&lead->key_min, lo);
        atomicMax(&lead->key_max, hi);
      }
    } else if (c.op == kOpMass || c.op == kOpCount) {
      u64 s = 0;
      for (int i = threadIdx.x; i < n; i += kRowsThreads)
        if (member(c, val[i])) s += c.op == kOpMass ? weight(val[i]) : 1ull;
      s = block_sum64(s);
      if (threadIdx.x == 0) lead->part[rank] = s;
    } else if (c.op == kOpPick && c.rank == rank) {
      // warps hold consecutive runs of the slice: count by warp, then walk the run that holds it
      const int warp = threadIdx.x >> 5, run = ((n + kRowsWarps - 1) / kRowsWarps + 31) / 32 * 32;
      const int i0 = min(warp * run, n), i1 = min(i0 + run, n);
      int count = 0;
      for (int i = i0; i < i1; i += 32) count += __popc(__ballot_sync(0xffffffffu, i + lane < i1 && member(c, val[i + lane])));
      __syncthreads();
      if (lane == 0) sh->red[warp] = (u64)count;
      __syncthreads();
      int want = c.n;
      for (int w = 0; w < warp; ++w) want -= (int)sh->red[w];
      if (want >= 0 && want < count) {
        for (int i = i0; i < i1; i += 32) {
          const bool in = i + lane < i1 && member(c, val[i + lane]);
          const unsigned who = __ballot_sync(0xffffffffu, in);
          if (in && __popc(who & ((1u << lane) - 1u)) == want) lead->found = base + i + lane;
          want -= __popc(who);
        }
      }
    }
  }

  // ---- the leader's side (every thread of its CTA calls these together) ----
  __device__ void command(const RowsCmd& c) {
    __syncthreads();
    if ((int)threadIdx.x < C) *cl.map_shared_rank(&sh->cmd, threadIdx.x) = c;
    if (threadIdx.x == 0 && c.op == kOpGather) sh->listed = 0;
    if (threadIdx.x == 0 && c.op == kOpRange) {
      sh->key_min = 0xffffffffu;
      sh->key_max = 0u;
    }
    cl.sync();
    if (c.op == kOpEnd) return;
    perform(c);
    cl.sync();
  }
  __device__ u64 total_of(const RowsCmd& c) {
    command(c);
    u64 s = 0;
    for (int r = 0; r < C; ++r) s += sh->part[r];
    return s;
  }
  __device__ int index_of(uint32_t key, int nth) {  // the nth token (from 0) of that key
    RowsCmd c{kOpCount, 0, key, key, 0, 0, 0};
    command(c);
    c.op = kOpPick;
    c.n = nth;
    for (c.rank = 0; c.rank < C - 1 && c.n >= (int)sh->part[c.rank]; ++c.rank) c.n -= (int)sh->part[c.rank];
    command(c);
    return sh->found;
  }

  // This thread's two bins of the reduced histogram, and inclusive running sums at their ends.
  struct Bins {
    uint32_t count[2], run[2];
    u64 mass[2], mrun[2];
  };
  __device__ Bins read_bins() {
    Bins b;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = 2 * threadIdx.x + e;
      const uint4 h = *cl.map_shared_rank(&hist[i], i / (kRowsBins / C));
      b.count[e] = h.x;
      b.mass[e] = (u64)h.y | ((u64)h.z << 32);
    }
    uint32_t c = b.count[0] + b.count[1];
    u64 m = b.mass[0] + b.mass[1];
    const uint32_t c0 = c;
    const u64 m0 = m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, c, o);
      const u64 y = __shfl_up_sync(0xffffffffu, m, o);
      if (lane >= o) {
        c += x;
        m += y;
      }
    }
    __shared__ uint32_t wc[kRowsWarps];
    __shared__ u64 wm[kRowsWarps];
    __syncthreads();
    if (lane == 31) {
      wc[warp] = c;
      wm[warp] = m;
    }
    __syncthreads();
    for (int w = 0; w < warp; ++w) {
      c += wc[w];
      m += wm[w];
    }
    b.run[0] = c - c0 + b.count[0];
    b.run[1] = c;
    b.mrun[0] = m - m0 + b.mass[0];
    b.mrun[1] = m;
    return b;
  }
  // The bin at which the running count (by_count) or weight first reaches goal: its number, size
  // and what comes before it, in sh->pick_*. (goal lies within the whole sum.)
  __device__ void find_bin(const Bins& b, u64 goal, bool by_count) {
    __syncthreads();
    if (threadIdx.x == 0) sh->pick_bin = -1;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const u64 hi = by_count ? b.run[e] : b.mrun[e], own = by_count ? b.count[e] : b.mass[e];
      if (hi >= goal && hi - own < goal) {
        sh->pick_bin = 2 * threadIdx.x + e;
        sh->pick_count = (int)b.count[e];
        sh->pick_base = b.run[e] - b.count[e];
        sh->pick_mass = b.mrun[e] - b.mass[e];
      }
    }
    __syncthreads();
  }

  // Sorts the gathered list (value descending, then index) and leaves its running weights in
  // cum (over the leader's histogram, whose bins were read before).
  __device__ int sort_list(u64* cum) {
    const int m = min(sh->listed, kRowsList);
    int p2 = 64;
    while (p2 < m) p2 <<= 1;
    for (int i = m + threadIdx.x; i < p2; i += kRowsThreads) list[i] = ~0ull;
    __syncthreads();
    if (m <= 256) {  // rank by counting
      u64 x = 0;
      int r = 0;
      if ((int)threadIdx.x < m) {
        x = list[threadIdx.x];
        for (int i = 0; i < m; ++i) r += list[i] < x;
      }
      __syncthreads();
      if ((int)threadIdx.x < m) list[r] = x;
      __syncthreads();
    } else {
      for (int k = 2; k <= p2; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
          for (int i = threadIdx.x; i < p2 / 2; i += kRowsThreads) {
            const int a = ((i & ~(j - 1)) << 1) | (i & (j - 1)), b = a | j;
            const u64 x = list[a], y = list[b];
            if ((x > y) == ((a & k) == 0)) {
              list[a] = y;
              list[b] = x;
            }
          }
          __syncthreads();
        }
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i0 = 2 * threadIdx.x;
    const u64 w0 = i0 < m ? weight(entry_value(list[i0])) : 0ull, w1 = i0 + 1 < m ? weight(entry_value(list[i0 + 1])) : 0ull;
    u64 s = w0 + w1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    __syncthreads();
    if (lane == 31) sh->red[warp] = s;
    __syncthreads();
    for (int w = 0; w < warp; ++w) s += sh->red[w];
    if (i0 < m) cum[i0] = s - w1;
    if (i0 + 1 < m) cum[i0 + 1] = s;
    __syncthreads();
    return m;
  }
  __device__ __forceinline__ static float entry_value(u64 e) { return row_key_value(~(uint32_t)(e >> 32)); }
  // First entry whose running weight reaches goal (goal <= cum[m - 1]), in every thread.
  __device__ int find_entry(const u64* cum, int m, u64 goal) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = 2 * threadIdx.x + e;
      if (i < m && cum[i] >= goal && (i == 0 || cum[i - 1] < goal)) sh->pick_at = i;
    }
    __syncthreads();
    return sh->pick_at;
  }

  // The prefix at whose end the running count or weight first reaches goal, and (want_index) the
  // token that ends it. b: the row's first histogram.
  __device__ RowsPrefix resolve(const Bins& first, u64 goal, bool by_count, bool want_index, int* index) {
    find_bin(first, goal, by_count);
    u64 before = sh->pick_base, mass = sh->pick_mass;
    int count = sh->pick_count;
    RowsCmd c{kOpGather, 1, (uint32_t)sh->pick_bin, (uint32_t)sh->pick_bin, 0, 0, 0};
    // (32 bits of key, ten a round: five rounds always reach a single key)
    for (int round = 0; round < 6 && count > kRowsList; ++round) {
      if (c.by_bin) {
        c.op = kOpRange;
        command(c);
        c.lo = sh->key_min;
        c.hi = sh->key_max;
        c.by_bin = 0;
      }
      if (c.lo == c.hi) break;
      c.op = kOpHist;
      c.shift = 0;
      while (((c.hi - c.lo) >> c.shift) >= (uint32_t)kRowsBins) ++c.shift;
      command(c);
      const Bins b = read_bins();
      find_bin(b, goal - (by_count ? before : mass), by_count);
      before += sh->pick_base;
      mass += sh->pick_mass;
      count = sh->pick_count;
      const uint32_t top = c.hi - ((uint32_t)sh->pick_bin << c.shift), span = (1u << c.shift) - 1u;
      c.lo = max(c.lo, top - min(top, span));
      c.hi = top;
    }
    RowsPrefix p;
    if (count > kRowsList) {  // equal values: the order is the index
      const u64 w = weight(row_key_value(c.lo));
      p.key = c.lo;
      p.ties = (int)(by_count ? goal - before : (goal - mass + w - 1) / w);
      p.mass = mass + p.ties * w;
      if (want_index) *index = index_of(p.key, p.ties - 1);
      return p;
    }
    c.op = kOpGather;
    command(c);
    u64* cum = reinterpret_cast<u64*>(hist);
    const int m = sort_list(cum);
    const int at = by_count ? (int)(goal - before) - 1 : find_entry(cum, m, goal - mass);
    p.key = ~(uint32_t)(list[at] >> 32);
    p.mass = mass + cum[at];
    int lo = at;
    while (lo > 0 && ~(uint32_t)(list[lo - 1] >> 32) == p.key) --lo;
    p.ties = at - lo + 1;
    *index = (int)(uint32_t)list[at];
    return p;
  }
};

// The key of the smallest float v with (v - v_max) / T >= ln(min_p), which is w >= min_p.
__device__ __forceinline__ uint32_t rows_min_key(float min_p, float vmax, double temperature) {
  if (min_p >= 1.0f) return row_key(vmax);
  return row_key(__double2float_ru(fma(log((double)min_p), temperature, (double)vmax)));
}

template <typename T>
__global__ void __launch_bounds__(kRowsThreads, 2) k_sample_rows(const __grid_constant__ SampleRowsArgs a) {
  extern __shared__ __align__(16) unsigned char rows_smem[];
  __shared__ RowsShared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  RowsCta x{cg::this_cluster()};
  x.sh = &sh;
  x.C = (int)x.cl.num_blocks();
  x.rank = (int)x.cl.block_rank();
  x.hist = reinterpret_cast<uint4*>(rows_smem);
  x.list = reinterpret_cast<u64*>(rows_smem + kRowsBins * 16);
  x.val = reinterpret_cast<float*>(rows_smem + kRowsBins * 16 + kRowsList * 8);
  const int r = blockIdx.x / x.C;
  x.base = x.rank * a.per;
  x.n = max(0, min(a.per, a.vocab - x.base));
  auto started = x.cl.barrier_arrive();  // waited for before the first access to another CTA's memory
  pdl_wait();
  pdl_trigger();
  // (beyond 1e30 every weight of a finite row is 1 as it is)
  float temperature = a.temperature ? a.temperature[r] : 1.0f;
  if (temperature > 1.0e30f) temperature = 1.0e30f;
  const int top_k = a.top_k ? a.top_k[r] : 0;
  const float top_p = a.top_p ? a.top_p[r] : 1.0f, min_p = a.min_p ? a.min_p[r] : 0.0f;
  const float u = a.u[r];

  // ---- the row into shared memory, its maximum and its smallest finite value ----
  const char* row = static_cast<const char*>(a.logits) + (r * a.row_stride + x.base) * (long long)sizeof(T);
  float mx = -INFINITY, mn = INFINITY;
  auto take = [&](float v) {
    if (!(v == v)) v = -INFINITY;
    mx = fmaxf(mx, v);
    if (v > -INFINITY) mn = fminf(mn, v);
    return v;
  };
  constexpr int V16 = 16 / sizeof(T);
  int done = 0;
  if ((reinterpret_cast<uintptr_t>(row) & 15) == 0) {
    const int chunks = x.n / V16;
#pragma unroll 4
    for (int i = tid; i < chunks; i += kRowsThreads) {
      const uint4 q = ld_stream(reinterpret_cast<const uint4*>(row) + i);
      T t[V16];
      memcpy(t, &q, 16);
      float f[V16];
#pragma unroll
      for (int e = 0; e < V16; ++e) f[e] = take(rows_value<T>(t, e));
#pragma unroll
      for (int e = 0; e < V16; e += 4)
        *reinterpret_cast<float4*>(x.val + i * V16 + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
    }
    done = chunks * V16;
  }
  for (int i = done + tid; i < x.n; i += kRowsThreads) x.val[i] = take(rows_value<T>(row, i));
  mx = warp_max(mx);
  mn = -warp_max(-mn);
  if (lane == 0) {
    sh.red[warp] = ((u64)__float_as_uint(mx) << 32) | __float_as_uint(mn);
  }
  if (tid == 0) sh.found = 0x7fffffff;
  __syncthreads();
  for (int w = 0; w < kRowsWarps; ++w) {
    mx = fmaxf(mx, __uint_as_float((uint32_t)(sh.red[w] >> 32)));
    mn = fminf(mn, __uint_as_float((uint32_t)sh.red[w]));
  }
  x.cl.barrier_wait(std::move(started));
  if (tid < x.C) {
    *x.cl.map_shared_rank(&sh.mx[x.rank], tid) = mx;
    *x.cl.map_shared_rank(&sh.mn[x.rank], tid) = mn;
  }
  x.cl.sync();
  for (int c = 0; c < x.C; ++c) {
    mx = fmaxf(mx, sh.mx[c]);
    mn = fminf(mn, sh.mn[c]);
  }
  x.vmax = mx;

  const bool few = top_k > 0 && top_k < a.vocab;
  if (!(temperature > 0.0f) || top_k == 1 || !(fabsf(mx) < INFINITY)) {
    // greedy: the first token of the largest value; where all are -inf or NaN the first that is not NaN
    int at = 0x7fffffff;
    for (int i = tid; i < x.n; i += kRowsThreads) {
      const bool is = mx > -INFINITY ? x.val[i] == mx : !isnan(rows_value<T>(row, i));
      if (is) at = min(at, x.base + i);
    }
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) atomicMin(&x.cl.map_shared_rank(&sh, 0)->found, at);
    x.cl.sync();
    if (x.rank == 0 && tid == 0) {
      a.ids[r] = sh.found == 0x7fffffff ? 0 : sh.found;
      if (a.logprobs) a.logprobs[r] = 0.0f;
    }
    return;
  }
  x.inv_t = 1.0 / (double)temperature;
  const float range = fminf(31.0f * temperature, mx - mn);
  x.scale = range > 0.0f ? fminf((float)(kRowsBins - 1) / range, 3.0e38f) : 0.0f;

  // weights are summed at once where a cut or the draw will need them; a top-k cut, or a min-p cut
  // without a top-p one, usually leaves a short list that does not
  const bool cut_p = top_p < 1.0f, cut_m = min_p > 0.0f;
  bool mass = !few && (cut_p || !cut_m);
  x.histogram(RowsCmd{kOpHist, 1, 0, kRowsBins - 1, 0, 0, 0}, mass);
  x.cl.sync();
  if (x.rank != 0) {
    for (;;) {
      x.cl.sync();
      const RowsCmd c = sh.cmd;
      if (c.op == kOpEnd) return;
      x.perform(c);
      x.cl.sync();
    }
  }

  // ---- the leader ----
  const RowsCmd end{kOpEnd, 0, 0, 0, 0, 0, 0};
  RowsCta::Bins bins = x.read_bins();
  const uint32_t kmin = cut_m ? rows_min_key(min_p, mx, (double)temperature) : 0u;
  // the last step that can hold a kept token, and how many tokens there are up to it
  int last = kRowsBins - 1, upto = a.vocab;
  if (few) {
    x.find_bin(bins, (u64)top_k, true);
    last = sh.pick_bin;
    upto = (int)sh.pick_base + sh.pick_count;
  } else if (cut_p) {
    if (tid == kRowsThreads - 1) sh.part[0] = bins.mrun[1];
    __syncthreads();
    x.find_bin(bins, max((u64)ceil(fmax((double)top_p, 0.0) * (double)sh.part[0]), 1ull), false);
    last = sh.pick_bin;
    upto = (int)sh.pick_base + sh.pick_count;
  }
  if (cut_m && !(few && cut_p)) {  // (top-p after top-k needs the whole top-k's sum)
    const int mb = x.bin(row_key_value(kmin));
    if (mb < last) {
      last = mb;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (2 * tid + e == mb) sh.pick_count = (int)bins.run[e];
      __syncthreads();
      upto = sh.pick_count;
    }
  }
  u64 total = 0;
  int id = 0;
  float logp = 0.0f;
  auto share = [&](uint32_t key) {
    return (float)(((double)row_key_value(key) - (double)mx) * x.inv_t - log((double)total / kRowsOne));
  };
  if (upto <= kRowsList) {
    u64 all = 0;
    if (!few && cut_p) all = sh.part[0];
    __syncthreads();
    x.command(RowsCmd{kOpGather, 1, 0, (uint32_t)last, 0, 0, 0});
    x.command(end);
    u64* cum = reinterpret_cast<u64*>(x.hist);
    int m = x.sort_list(cum);
    if (few) m = min(m, top_k);
    if (cut_p) {
      const u64 sum = few ? cum[m - 1] : all;
      m = min(m, x.find_entry(cum, m, min(max((u64)ceil(fmax((double)top_p, 0.0) * (double)sum), 1ull), cum[m - 1])) + 1);
    }
    if (cut_m) {
      __syncthreads();
      if (tid == 0) sh.pick_at = 1;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * tid + e;
        if (i < m && ~(uint32_t)(x.list[i] >> 32) >= kmin && (i + 1 == m || ~(uint32_t)(x.list[i + 1] >> 32) < kmin))
          sh.pick_at = i + 1;
      }
      __syncthreads();
      m = sh.pick_at;
      if (min_p > 1.0f) m = 1;
    }
    total = cum[m - 1];
    const int at = x.find_entry(cum, m, min((u64)floor((double)u * (double)total), total - 1) + 1);
    id = (int)(uint32_t)x.list[at];
    logp = share(~(uint32_t)(x.list[at] >> 32));
  } else {
    if (!mass) {
      x.command(RowsCmd{kOpHist, 1, 0, kRowsBins - 1, 0, 0, 0});
      bins = x.read_bins();
    }
    if (tid == kRowsThreads - 1) sh.pick_mass = bins.mrun[1];
    __syncthreads();
    RowsPrefix keep{0u, a.vocab, sh.pick_mass};
    int unused;
    if (few) keep = x.resolve(bins, (u64)top_k, true, false, &unused);
    if (cut_p) {
      const RowsPrefix p =
          x.resolve(bins, max((u64)ceil(fmax((double)top_p, 0.0) * (double)keep.mass), 1ull), false, false, &unused);
      if (p.key > keep.key || (p.key == keep.key && p.ties < keep.ties)) keep = p;
    }
    if (min_p > 1.0f) {
      keep.mass = x.weight(mx);
    } else if (cut_m && kmin > keep.key) {
      keep.mass = x.total_of(RowsCmd{kOpMass, 0, kmin, 0xffffffffu, 0, 0, 0});
    }
    total = keep.mass;
    const RowsPrefix p = x.resolve(bins, min((u64)floor((double)u * (double)total), total - 1) + 1, false, true, &id);
    logp = share(p.key);
    x.command(end);
  }
  if (tid == 0) {
    a.ids[r] = id;
    if (a.logprobs) a.logprobs[r] = logp;
  }
}

template <typename T>
static void launch_sample_rows(SampleRowsArgs a, int rows, cudaStream_t s) {
  // CTAs per row: enough that a CTA holds at most 20480 tokens (two CTAs an SM) and, with few rows,
  // that the SMs are used; a CTA below 2048 tokens gains nothing any more.
  int C = 1;
  while (C < kRowsMaxCluster && ((a.vocab + C - 1) / C > 20480 ||
                                 ((long long)rows * C < 2 * current_sms() && (a.vocab + C - 1) / C > 2048)))
    C *= 2;
  a.per = ((a.vocab + C - 1) / C + 7) / 8 * 8;
  const size_t smem = kRowsBins * 16 + kRowsList * 8 + (size_t)a.per * 4;
  static unsigned long long smem_set = 0;
  allow_smem(k_sample_rows<T>, kRowsBins * 16 + kRowsList * 8 + (size_t)(kRowsMaxVocab / kRowsMaxCluster + 8) * 4, smem_set);
  if ((long long)rows * C > 0x7fffffffLL) throw QdError{QD_E_RANGE, "qd_sample_rows: too many rows"};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * C));
  cfg.blockDim = dim3(kRowsThreads);
  cfg.dynamicSmemBytes = smem;
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
  QD_CK(cudaLaunchKernelEx(&cfg, k_sample_rows<T>, a));
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
    SampleRowsArgs a{logits, (int)vocab, 0, row_stride, temperature, top_k, top_p, min_p, u, ids, logprobs};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == QD_KV_F32) launch_sample_rows<float>(a, rows, s);
    else if (dtype == QD_KV_F16) launch_sample_rows<__half>(a, rows, s);
    else launch_sample_rows<__nv_bfloat16>(a, rows, s);
  } catch (const qd::QdError& err) {
    qd::set_thread_error(err.msg);
    return err.code;
  } catch (const std::exception& err) {
    qd::set_thread_error(err.what());
    return QD_E_NOMEM;
  }
  return QD_OK;
}
