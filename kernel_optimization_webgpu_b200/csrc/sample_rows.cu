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
// One thread-block cluster per row. The row is read once, into the CTAs' shared memory; what bounds
// it is then the latency of a few passes and cluster barriers and, with many rows, the
// instructions per token, so the passes are few and the work of each is spread over the cluster:
//  1. maximum and minimum;
//  2. histogram over kRowsBins equal steps of value between them (or 32 T nats, beyond which a
//     weight is zero): counts, and the sums of the places within a step, by 32-bit atomics in
//     shared memory. Steps are monotone in the value. Count times the weight at the mean place
//     is a step's sum of weights to within s^2 / 8 + 1e-5 of itself, s the step in nats (the
//     exponential's curvature over one step, and f32 roundings), which tells for every border
//     in which few steps it must lie;
//  3. the tokens of those steps are gathered into the first CTA; in the same pass the exact
//     weights of all tokens, and of those above each such range, are summed in registers. The
//     leader sorts the gathered ones and finds the borders exactly.
//     The border's range and the draw's share one such pass, or take one each where only both
//     together are too long for the list (64 rows as below: 66 -> 65 us; a row that then needed the
//     resolution below took 43 us, and takes 25 to 28).
// Where a range holds more than kRowsList tokens (long classes of equal values, a large top-k), each border
// is resolved alone: exact sums by step, the tokens of one step gathered and sorted, a step with
// too many cut into finer ones by key, and where all of them are equal their order is their
// index. The first CTA of the cluster leads: it tells the others what to do next and ends them.
//
// One row of 151936 f32 logits, top-k 40 and top-p 0.9: 14.5 us. 64 rows with settings of their own,
// most of them over the whole vocabulary: 65 us (38.9 MB), two CTAs an SM in two waves; of a
// cluster's 28 us there, 11 are the exact sums of all weights, 5 the histogram, 8 the leader's steps.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <utility>

#include "../../include/qdecode.h"
#include "internal.cuh"
#include "paged.cuh"
#include "rows.cuh"

namespace qd {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int kRowsThreads = 512;
constexpr int kRowsWarps = kRowsThreads / 32;
constexpr int kRowsMaxVocab = 393216;
constexpr int kRowsMaxCluster = 8;
constexpr int kRowsMaxPer = kRowsMaxVocab / kRowsMaxCluster;  // tokens a CTA takes: its 32-bit sums of 16 bits fit
constexpr int kRowsBins = 2048;       // four a thread of the leader
constexpr int kRowsExact = kRowsBins / 2;  // bins of an exact histogram (twice the words a bin)
constexpr int kRowsList = 1024;
constexpr double kRowsOne = 17592186044416.0;  // weight 1 = 2^44

struct SampleRowsArgs {
  const void* logits;
  int vocab, per;  // per: tokens a CTA takes, a multiple of 8
  long long row_stride;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  int* ids;
  float* logprobs;
};

// What the leader asks of every CTA.
enum RowsOp : int { kOpEnd = 0, kOpHist, kOpGather, kOpRange, kOpMass, kOpCount, kOpPick };
struct RowsCmd {
  int op;
  int by_bin;         // members: bins [lo, hi] (2: of the exact histogram), else keys [lo, hi]
  uint32_t lo, hi;
  int shift;          // kOpHist by key: bin = (hi - key) >> shift
  int rank, n;        // kOpPick: CTA `rank` finds its n-th member by index
  int sums;           // kOpGather: also the weights of all tokens, and of those in bins below lo and lo2;
                      // 2: [lo2, hi2] are no members
  uint32_t lo2, hi2;  // kOpGather by bin: a second range of members (lo2 > hi2: none)
};
// A prefix of the row's order: every key above `key` and the first `ties` of those equal to it.
struct RowsPrefix {
  uint32_t key;
  int ties;
  u64 mass;
};

// A bin, its tokens, and the tokens and weight before it.
struct RowsAt {
  int bin, count, before;
  u64 mass;
};

struct RowsShared {
  RowsCmd cmd;
  float mx[kRowsMaxCluster], mn[kRowsMaxCluster];
  u64 part[kRowsMaxCluster];      // per-CTA sums for the leader
  u64 above[3][kRowsMaxCluster];  // kOpGather with sums: all, below lo, below lo2
  u64 sums[3][kRowsWarps];        // of this CTA's warps
  int taken;                      // entries of this CTA's own list
  uint32_t key_min, key_max;      // leader
  int found;                      // leader: an index
  u64 red[kRowsWarps];
  RowsAt at[4];                   // results of searches over the leader's threads
  int pick_at, upto;
  u64 whole;
};

// One CTA's view of its row.
struct RowsCta {
  cg::cluster_group cl;
  RowsShared* sh;
  float* val;       // this CTA's tokens, filled up to a multiple of 4 with NaN
  uint32_t* hist;   // [2][kRowsBins]: counts, places; or [4][kRowsExact]: counts, and weights in three sums
  const double* pow2;  // 2^(44 + i / 128)
  u64* list;       // leader: {~key, index}
  int n, base, C, lg, rank;  // C = 1 << lg CTAs
  float vmax, scale, range;  // scale: places per unit of value
  double inv_t, z_scale;  // 1 / T and 128 log2(e) / T
  float step;             // width of a bin in the weight's logarithm to base 2

  // A value's place: 4096ths of a bin below the maximum, rounded by an addition of 2^23 (conversions
  // run at an eighth of its rate). Ascending as v descends. kNoPlace for what has no weight (NaN,
  // -inf, beyond the range; the scale keeps the range's end below it): those are the last bin.
  static constexpr uint32_t kNoPlace = (kRowsBins - 1) << 12;
  __device__ __forceinline__ uint32_t place(float v) const {
    return __float_as_uint(fminf(fmaf(vmax - v, scale, 8388608.0f), 8388608.0f + (float)kNoPlace)) & 0x7fffffu;
  }
  __device__ __forceinline__ int bin(float v) const { return (int)(place(v) >> 12); }
  __device__ __forceinline__ int exact_bin(float v) const { return (int)(place(v) >> 13); }
  // exp((v - v_max) / T) * 2^44, rounded: with z = 128 log2(e) (v - v_max) / T = 128 e + i + r, it is
  // 2^(44 + e) 2^(i / 128) 2^(r / 128), |r| <= 1 / 2, the last factor by its Taylor sum to the fourth
  // power (the rest is below 2^-49): table-driven, after Tang, ACM TOMS 15 (1989). Roundings to
  // an integer are additions of 1.5 * 2^52 and 2^52.
  // (before the last rounding; of a value beyond the range it is meaningless)
  __device__ __forceinline__ double raw_weight(float v) const {
    const double d = (double)v - (double)vmax;
    const double near = fma(d, z_scale, 6755399441055744.0);
    const int k = __double2loint(near);
    const double r = fma(d, z_scale, 6755399441055744.0 - near);
    constexpr double c = 0.6931471805599453 / 128.0;
    const double p = fma(fma(fma(fma(c * c * c * c / 24.0, r, c * c * c / 6.0), r, c * c / 2.0), r, c), r, 1.0);
    const double w = p * pow2[k & 127];
    return __hiloint2double(__double2hiint(w) + ((k << 13) & 0xfff00000), __double2loint(w));
  }
  __device__ __forceinline__ u64 weight(float v) const {
    if (!(vmax - v <= range)) return 0ull;
    return (u64)__double_as_longlong(raw_weight(v) + 4503599627370496.0) & 0xfffffffffffffull;
  }
  // f(values, index of the first) for every four tokens of this CTA, the last ones filled up with NaN
  // (which has no weight and sorts last), two loads before their work.
  template <typename F>
  __device__ __forceinline__ void each4(F&& f) const {
    int i = 4 * threadIdx.x;
    for (; i + 4 * kRowsThreads < n; i += 8 * kRowsThreads) {
      const float4 x = *reinterpret_cast<const float4*>(val + i);
      const float4 y = *reinterpret_cast<const float4*>(val + i + 4 * kRowsThreads);
      const float v[4] = {x.x, x.y, x.z, x.w}, w[4] = {y.x, y.y, y.z, y.w};
      f(v, i);
      f(w, i + 4 * kRowsThreads);
    }
    if (i < n) {
      const float4 x = *reinterpret_cast<const float4*>(val + i);
      const float v[4] = {x.x, x.y, x.z, x.w};
      f(v, i);
    }
  }
  // f(value, index) for every token.
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    each4([&](const float (&v)[4], int i) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < n) f(v[k], i + k);
    });
  }
  __device__ __forceinline__ bool member(const RowsCmd& c, float v) const {
    if (c.by_bin) {
      const uint32_t b = (uint32_t)(c.by_bin == 2 ? exact_bin(v) : bin(v));
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

  // Histogram of the members; afterwards this CTA's share of the bins holds the whole row's sums:
  // the count, and the sum of weights (kExact) or of places (kPlaces) as two words.
  enum HistKind : int { kCounts, kPlaces, kExact };
  __device__ void histogram(const RowsCmd& c, HistKind kind) {
    const int nb = kind == kExact ? kRowsExact : kRowsBins;
    for (int i = threadIdx.x; i < kRowsBins / 2; i += kRowsThreads)
      reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (kind == kCounts) {
      each4([&](const float (&v)[4], int) {
        int b[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) b[k] = bin(v[k]);
#pragma unroll
        for (int k = 0; k < 4; ++k) atomicAdd(&hist[b[k]], 1u);
      });
    } else if (kind == kPlaces) {
      each4([&](const float (&v)[4], int) {
        uint32_t u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = place(v[k]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          atomicAdd(&hist[u[k] >> 12], 1u);
          atomicAdd(&hist[kRowsBins + (u[k] >> 12)], u[k] & 4095u);
        }
      });
    } else {
      each([&](float v, int) {
        int b;
        if (c.by_bin) {
          b = exact_bin(v);
        } else {
          const uint32_t k = row_key(v);
          if (k < c.lo || k > c.hi) return;
          b = (int)((c.hi - k) >> c.shift);
        }
        atomicAdd(&hist[b], 1u);
        const u64 w = weight(v);
        const uint32_t low = (uint32_t)w & 0x3fffu, mid = (uint32_t)(w >> 14) & 0x3fffu, high = (uint32_t)(w >> 28);
        if (low) atomicAdd(&hist[nb + b], low);
        if (mid) atomicAdd(&hist[2 * nb + b], mid);
        if (high) atomicAdd(&hist[3 * nb + b], high);
      });
    }
    cl.sync();
    const int share = nb >> lg;
    for (int i = threadIdx.x; i < share; i += kRowsThreads) {
      const int b = rank * share + i;
      uint32_t h[4][kRowsMaxCluster];
      const int fields = kind == kCounts ? 1 : kind == kPlaces ? 2 : 4;
#pragma unroll
      for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int r = 0; r < kRowsMaxCluster; ++r)  // all loads in flight together
          h[f][r] = f < fields && r < C ? cl.map_shared_rank(hist, r)[f * nb + b] : 0u;
      uint32_t count = 0;
      u64 w = 0;
#pragma unroll
      for (int r = 0; r < kRowsMaxCluster; ++r) {
        count += h[0][r];
        w += (u64)h[1][r] + ((u64)h[2][r] << 14) + ((u64)h[3][r] << 28);
      }
      hist[b] = count;
      if (kind == kPlaces) {  // (a row's sum of places fits: at most 393216 times 4095)
        hist[kRowsBins + b] = (uint32_t)w;
      } else if (kind == kExact) {
        hist[nb + b] = (uint32_t)w;
        hist[2 * nb + b] = (uint32_t)(w >> 32);
      }
    }
  }

  // What a command makes every CTA do (the caller synchronises the cluster around it).
  __device__ void perform(const RowsCmd& c) {
    RowsShared* lead = cl.map_shared_rank(sh, 0);
    const int lane = threadIdx.x & 31;
    if (c.op == kOpHist) {
      histogram(c, kExact);
    } else if (c.op == kOpGather) {  // into this CTA's own list; the leader collects them
      if (threadIdx.x == 0) sh->taken = 0;
      __syncthreads();
      auto keep = [&](float v, int i) {
        const int at = atomicAdd(&sh->taken, 1);
        if (at < kRowsList) list[at] = ((u64)~row_key(v) << 32) | (unsigned)(base + i);
      };
      if (c.sums) {  // by bin
        // Each thread adds at most 96 weights below 2^45 to 2^52: additions there round every weight to an
        // integer and are exact otherwise.
        double sum[3] = {4503599627370496.0, 4503599627370496.0, 4503599627370496.0};
        const bool two = c.sums == 2 || c.lo2 <= c.hi2;
        const uint32_t lo = c.lo << 12, span = ((c.hi + 1) << 12) - lo, lo2 = c.lo2 << 12;
        const uint32_t span2 = c.sums == 1 && two ? ((c.hi2 + 1) << 12) - lo2 : 0u;
        each4([&](const float (&v)[4], int i) {
          double w[4];
          uint32_t u[4];
          bool any = false;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            u[k] = place(v[k]);
            w[k] = raw_weight(v[k]);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (u[k] < kNoPlace) sum[0] += w[k];
            if (u[k] < lo) sum[1] += w[k];
            any = any || u[k] - lo < span;
          }
          if (two) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (u[k] < lo2) sum[2] += w[k];
              any = any || u[k] - lo2 < span2;
            }
          }
          if (any) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if ((u[k] - lo < span || u[k] - lo2 < span2) && i + k < n) keep(v[k], i + k);
          }
        });
        u64 all[3];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          all[k] = (u64)__double_as_longlong(sum[k]) & 0xfffffffffffffull;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) all[k] += __shfl_xor_sync(0xffffffffu, all[k], o);
          if (lane == 0) sh->sums[k][threadIdx.x >> 5] = all[k];
        }
        __syncthreads();
        if (threadIdx.x < 3) {
          u64 total = 0;
          for (int w = 0; w < kRowsWarps; ++w) total += sh->sums[threadIdx.x][w];
          lead->above[threadIdx.x][rank] = total;
        }
      } else if (c.by_bin == 1) {
        const uint32_t lo = c.lo << 12, span = ((c.hi + 1) << 12) - lo;
        each4([&](const float (&v)[4], int i) {
          bool in[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) in[k] = place(v[k]) - lo < span;
          if (in[0] || in[1] || in[2] || in[3]) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (in[k] && i + k < n) keep(v[k], i + k);
          }
        });
      } else {
        each([&](float v, int i) {
          if (member(c, v)) keep(v, i);
        });
      }
      __syncthreads();
      if (threadIdx.x == 0) lead->part[rank] = (u64)min(sh->taken, kRowsList);
    } else if (c.op == kOpRange) {
      uint32_t lo = 0xffffffffu, hi = 0u;
      each([&](float v, int) {
        if (member(c, v)) {
          lo = min(lo, row_key(v));
          hi = max(hi, row_key(v));
        }
      });
      lo = __reduce_min_sync(0xffffffffu, lo);
      hi = __reduce_max_sync(0xffffffffu, hi);
      if (lane == 0 && lo <= hi) {
        atomicMin(&lead->key_min, lo);
        atomicMax(&lead->key_max, hi);
      }
    } else if (c.op == kOpMass || c.op == kOpCount) {
      u64 s = 0;
      each([&](float v, int) {
        if (member(c, v)) s += c.op == kOpMass ? weight(v) : 1ull;
      });
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
    if (threadIdx.x == 0 && c.op == kOpRange) {
      sh->key_min = 0xffffffffu;
      sh->key_max = 0u;
    }
    if (c.op == kOpEnd) {  // nothing more passes between the CTAs: the leader need not wait
      (void)cl.barrier_arrive();
      return;
    }
    cl.sync();
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
    RowsCmd c{kOpCount, 0, key, key, 0, 0, 0, 0, 1, 0};
    command(c);
    c.op = kOpPick;
    c.n = nth;
    for (c.rank = 0; c.rank < C - 1 && c.n >= (int)sh->part[c.rank]; ++c.rank) c.n -= (int)sh->part[c.rank];
    command(c);
    return sh->found;
  }

  // This thread's bins of the reduced histogram (four neighbours; two of an exact one), and running
  // sums up to and with each. Weights are exact after kExact, estimates after kPlaces.
  struct Bins {
    int per;
    uint32_t count[4], run[4];
    u64 mass[4], mrun[4];
  };
  __device__ Bins read_bins(HistKind kind) {
    Bins b;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nb = kind == kExact ? kRowsExact : kRowsBins;
    b.per = kind == kExact ? 2 : 4;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      b.count[e] = 0;
      b.mass[e] = 0;
      if (e >= b.per) continue;
      const int i = b.per * threadIdx.x + e;
      const uint32_t* h = cl.map_shared_rank(hist, i / (nb >> lg)) + i;
      b.count[e] = h[0];
      if (kind == kExact) {
        b.mass[e] = (u64)h[nb] | ((u64)h[2 * nb] << 32);
      } else if (kind == kPlaces && b.count[e] && i < kRowsBins - 1) {
        const float at = (float)i + (float)h[nb] / (4096.0f * (float)b.count[e]);
        b.mass[e] = (u64)((float)b.count[e] * exp2f(44.0f - at * step));
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      b.run[e] = (e ? b.run[e - 1] : 0u) + b.count[e];
      b.mrun[e] = (e ? b.mrun[e - 1] : 0ull) + b.mass[e];
    }
    uint32_t c = b.run[3];
    u64 m = b.mrun[3];
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
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      b.run[e] += c - c0;
      b.mrun[e] += m - m0;
    }
    return b;
  }
  // For each goal: the bin at which the running count (by_count) or weight first reaches it, and the
  // tokens and weight before it, in sh->at. (A goal lies between 1 and the whole sum, as an integer:
  // a sum beyond 2^53 that became a double may have grown.)
  __device__ void find_bins(const Bins& b, const u64* goal, int n_goals, bool by_count) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const u64 hi = by_count ? b.run[e] : b.mrun[e], own = by_count ? b.count[e] : b.mass[e];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < n_goals && hi >= goal[k] && hi - own < goal[k])
          sh->at[k] = RowsAt{b.per * (int)threadIdx.x + e, (int)b.count[e], (int)(b.run[e] - b.count[e]), b.mrun[e] - b.mass[e]};
    }
    __syncthreads();
  }

  // Collects the CTAs' lists behind the leader's own.
  __device__ int collect() {
    int off[kRowsMaxCluster + 1];
    off[0] = 0;
#pragma unroll
    for (int r = 0; r < kRowsMaxCluster; ++r) off[r + 1] = off[r] + (r < C ? (int)sh->part[r] : 0);
    const int m = min(off[kRowsMaxCluster], kRowsList);
    for (int i = off[1] + threadIdx.x; i < m; i += kRowsThreads) {
      int r = 1;
#pragma unroll
      for (int k = 2; k < kRowsMaxCluster; ++k) r += i >= off[k];
      int at = 0;
#pragma unroll
      for (int k = 1; k < kRowsMaxCluster; ++k)
        if (r == k) at = i - off[k];
      list[i] = cl.map_shared_rank(list, r)[at];
    }
    __syncthreads();
    return m;
  }
  // Bitonic sort of the list padded to kRowsList: each warp keeps 64 neighbours in registers (two a
  // lane, 32 apart) and exchanges by shuffles; only distances of 64 and more go through shared memory
  // (10 steps with a barrier instead of 55).
  __device__ void sort_all(int m) {
    const int lane = threadIdx.x & 31, i0 = (threadIdx.x >> 5) * 64 + lane;
    u64 x = i0 < m ? list[i0] : ~0ull, y = i0 + 32 < m ? list[i0 + 32] : ~0ull;
    auto order = [](u64& a, u64& b, bool up) {
      if ((a > b) == up) {
        const u64 t = a;
        a = b;
        b = t;
      }
    };
    auto swap = [&](u64& a, int j, bool up) {  // against the lane j away; `up`: the lower index keeps the smaller
      const u64 o = __shfl_xor_sync(0xffffffffu, a, j);
      if ((a > o) == (((lane & j) == 0) == up)) a = o;
    };
    for (int k = 2; k <= kRowsList; k <<= 1) {
      for (int j = k >> 1; j >= 64; j >>= 1) {
        __syncthreads();
        list[i0] = x;
        list[i0 + 32] = y;
        __syncthreads();
        const bool up = ((i0 & k) == 0) == ((i0 & j) == 0);
        const u64 ox = list[i0 ^ j], oy = list[(i0 + 32) ^ j];
        if ((x > ox) == up) x = ox;
        if ((y > oy) == up) y = oy;
      }
      if (k >= 64) order(x, y, (i0 & k) == 0);
      for (int j = min(k >> 1, 16); j > 0; j >>= 1) {
        swap(x, j, (i0 & k) == 0);
        swap(y, j, ((i0 + 32) & k) == 0);
      }
    }
    __syncthreads();
    list[i0] = x;
    list[i0 + 32] = y;
    __syncthreads();
  }
  // Sorts the collected list (value descending, then index) and leaves its running weights in
  // cum (over the leader's histogram, whose bins were read before).
  __device__ void sort_list(u64* cum, int m) {
    if (m <= 256) {  // rank by counting
      u64 x = 0;
      int r = 0;
      if ((int)threadIdx.x < m) {
        x = list[threadIdx.x];
#pragma unroll 8
        for (int i = 0; i < m; ++i) r += list[i] < x;
      }
      __syncthreads();
      if ((int)threadIdx.x < m) list[r] = x;
      __syncthreads();
    } else {
      sort_all(m);
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
    u64 goals[4] = {goal, 0, 0, 0};
    find_bins(first, goals, 1, by_count);
    u64 before = sh->at[0].before, mass = sh->at[0].mass;
    int count = sh->at[0].count;
    RowsCmd c{kOpGather, 2, (uint32_t)sh->at[0].bin, (uint32_t)sh->at[0].bin, 0, 0, 0, 0, 1, 0};
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
      while (((c.hi - c.lo) >> c.shift) >= (uint32_t)kRowsExact) ++c.shift;
      command(c);
      const Bins b = read_bins(kExact);
      goals[0] = goal - (by_count ? before : mass);
      find_bins(b, goals, 1, by_count);
      before += sh->at[0].before;
      mass += sh->at[0].mass;
      count = sh->at[0].count;
      const uint32_t top = c.hi - ((uint32_t)sh->at[0].bin << c.shift), span = (1u << c.shift) - 1u;
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
    const int m = collect();
    sort_list(cum, m);
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
  __shared__ double pow2[128];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  RowsCta x{cg::this_cluster()};
  x.sh = &sh;
  x.C = (int)x.cl.num_blocks();
  x.rank = (int)x.cl.block_rank();
  x.lg = 31 - __clz(x.C);
  x.hist = reinterpret_cast<uint32_t*>(rows_smem);
  x.list = reinterpret_cast<u64*>(rows_smem + kRowsBins * 8);
  x.val = reinterpret_cast<float*>(rows_smem + kRowsBins * 8 + kRowsList * 8);
  const int r = blockIdx.x / x.C;
  x.base = x.rank * a.per;
  x.n = max(0, min(a.per, a.vocab - x.base));
  x.pow2 = pow2;
  if (tid < 128) pow2[tid] = exp2(tid / 128.0) * kRowsOne;
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
    mx = fmaxf(mx, v);
    mn = fminf(mn, v > -INFINITY ? v : INFINITY);
  };
  constexpr int V = 16 / sizeof(T);
  int done = 0;
  if ((reinterpret_cast<uintptr_t>(row) & 15) == 0) {
    const uint4* src = reinterpret_cast<const uint4*>(row);
    const int chunks = x.n / V;
#pragma unroll 5
    for (int i = tid; i < chunks; i += kRowsThreads) {
      const uint4 q = ld_stream(src + i);
      T t[V];
      memcpy(t, &q, 16);
#pragma unroll
      for (int k = 0; k < V; k += 4) {
        const float4 f = make_float4(rows_value<T>(t, k), rows_value<T>(t, k + 1), rows_value<T>(t, k + 2), rows_value<T>(t, k + 3));
        take(f.x);
        take(f.y);
        take(f.z);
        take(f.w);
        *reinterpret_cast<float4*>(x.val + i * V + k) = f;
      }
    }
    done = chunks * V;
  }
  for (int i = done + tid; i < x.n; i += kRowsThreads) {
    const float v = rows_value<T>(row, i);
    take(v);
    x.val[i] = v;
  }
  if (tid < ((4 - x.n % 4) & 3)) x.val[x.n + tid] = __int_as_float(0x7fc00000);
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
    x.each([&](float v, int i) {
      if (mx > -INFINITY ? v == mx : !isnan(v)) at = min(at, x.base + i);
    });
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
  x.z_scale = x.inv_t * (128.0 * 1.4426950408889634);
  // 32 T: 2^44 exp(-32) < 1/2, so that what lies beyond weighs nothing
  x.range = fminf(32.0f * temperature, mx - mn);
  x.scale = x.range > 0.0f ? (float)(RowsCta::kNoPlace - 8) / x.range : 0.0f;
  // A temperature (or a row) below 1e-33 wants more places per unit than f32 has: places then still ascend,
  // but lie close together and reach beyond the range, and tell nothing about weights. Such a row takes the
  // exact passes.
  const bool coarse = x.scale > 3.0e38f;
  if (coarse) x.scale = 3.0e38f;
  x.step = x.scale > 0.0f ? (float)(x.z_scale * (4096.0 / 128.0) / (double)x.scale) : 0.0f;

  // weights matter unless a top-k cut (or a min-p cut without a top-p one) leaves a short list
  const bool cut_p = top_p < 1.0f, cut_m = min_p > 0.0f;
  const RowsCta::HistKind kind = few || coarse || (cut_m && !cut_p) ? RowsCta::kCounts : RowsCta::kPlaces;
  x.histogram(RowsCmd{}, kind);
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
  const RowsCmd all_bins{kOpHist, 2, 0, kRowsExact - 1, 0, 0, 0, 0, 1, 0}, end{};
  RowsCta::Bins bins = x.read_bins(kind);
  const uint32_t kmin = cut_m ? rows_min_key(min_p, mx, (double)temperature) : 0u;
  const double p_share = fmax((double)top_p, 0.0);
  const int mbin = cut_m ? x.bin(row_key_value(kmin)) : kRowsBins - 1;
  if (tid == kRowsThreads - 1) sh.whole = bins.mrun[3];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (4 * tid + e == mbin) sh.upto = (int)bins.run[e];
  __syncthreads();
  // Where the top-p border and the draw must lie, by the estimated running weights (kPlaces).
  const double about = (double)sh.whole, nats = (double)x.step * 0.6931471805599453;
  const double slack = 3.0 * (nats * nats / 8.0 + 1.0e-5);
  const double p_goal = cut_p ? p_share * about : about, uu = fmin(fmax((double)u, 0.0), 1.0);
  // (the token that reaches the top-p border is kept whole: at most one weight more)
  const double d_lo_goal = uu * (cut_p ? p_goal * (1.0 - slack) : about),
               d_hi_goal = uu * (cut_p ? p_goal * (1.0 + slack) + kRowsOne : about);
  u64 goals[4];
  auto within = [&](double goal) { return min((u64)fmax(goal, 1.0), sh.whole); };
  goals[0] = few ? (u64)top_k : within(p_goal * (1.0 + slack));
  goals[1] = within(p_goal * (1.0 - slack));
  goals[2] = within(d_hi_goal * (1.0 + slack) + 1.0);
  goals[3] = within(d_lo_goal * (1.0 - slack));
  if (kind == RowsCta::kPlaces || few) x.find_bins(bins, goals, few ? 1 : 4, few);
  // the last bin that can hold a kept token, and the tokens up to it
  int last = kRowsBins - 1, upto = a.vocab;
  if (few || (cut_p && !coarse)) {
    last = sh.at[0].bin;
    upto = sh.at[0].before + sh.at[0].count;
  }
  if (cut_m && !(few && cut_p) && mbin < last) {  // (top-p after top-k needs the whole top-k's sum)
    last = mbin;
    upto = sh.upto;
  }
  // without a top-k or min-p cut: the ranges of bins of the border and of the draw, if short enough
  const int p_lo = sh.at[1].bin, p_hi = last, d_lo = min(sh.at[3].bin, last), d_hi = min(sh.at[2].bin, last);
  bool ranges = upto > kRowsList && kind == RowsCta::kPlaces && !cut_m, apart = false;
  if (ranges) {
    const int n_draw = sh.at[2].before + sh.at[2].count - sh.at[3].before;
    const int n_border = cut_p ? upto - sh.at[1].before : 0;
    apart = n_draw + n_border > kRowsList;  // one after the other, if each fits alone
    ranges = n_draw <= kRowsList && n_border <= kRowsList;
  }
  u64 total = 0;
  int id = 0;
  float logp = 0.0f;
  auto share = [&](uint32_t key) {
    return (float)(((double)row_key_value(key) - (double)mx) * x.inv_t - log((double)total / kRowsOne));
  };
  u64* cum = reinterpret_cast<u64*>(x.hist);
  bool settled = false;
  if (upto <= kRowsList && (few || !cut_p || !coarse)) {
    x.command(RowsCmd{kOpGather, 1, 0, (uint32_t)last, 0, 0, 0, cut_p && !few, 1, 0});
    int m = x.collect();
    const bool known = few || !cut_p;  // `last` is certain, not estimated: the other CTAs are done
    if (known) x.command(end);
    x.sort_list(cum, m);
    settled = true;
    if (few) m = min(m, top_k);
    if (cut_p) {
      u64 sum = 0;
      if (few) sum = cum[m - 1];
      else
        for (int c = 0; c < x.C; ++c) sum += sh.above[0][c];
      const u64 goal = max((u64)ceil(p_share * (double)sum), 1ull);
      settled = known || goal <= cum[m - 1] || (cut_m && last == mbin);
      m = min(m, x.find_entry(cum, m, min(goal, cum[m - 1])) + 1);
    }
    if (!known && settled) x.command(end);
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
  } else if (ranges) {
    // Both ranges in one list, in order: the draw's tokens lie at or before the border's. Where the
    // ranges overlap they are one. Running weights: exact, from those above each range. (Apart: the
    // border's list first, then the draw's.)
    RowsCmd c{kOpGather, 1, (uint32_t)d_lo, (uint32_t)d_hi, 0, 0, 0, 1, 1, 0};
    if (apart) {
      c = RowsCmd{kOpGather, 1, (uint32_t)p_lo, (uint32_t)p_hi, 0, 0, 0, 2, (uint32_t)d_lo, (uint32_t)d_lo};
    } else if (cut_p) {
      if (p_lo <= d_hi + 1) {
        c.hi = (uint32_t)p_hi;
      } else {
        c.lo2 = (uint32_t)p_lo;
        c.hi2 = (uint32_t)p_hi;
      }
    }
    x.command(c);
    int m = x.collect();
    u64 all = 0, above = 0, above2 = 0;
    for (int k = 0; k < x.C; ++k) {
      all += sh.above[0][k];
      above += sh.above[1][k];
      above2 += sh.above[2][k];
    }
    const bool split = !apart && c.lo2 <= c.hi2;
    x.sort_list(cum, m);
    // entries of the first range, then what the second one's running weights lack
    int m1 = m;
    if (split) {
      __syncthreads();
      if (tid == 0) sh.pick_at = 0;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * tid + e;
        if (i < m && x.bin(x.entry_value(x.list[i])) <= d_hi && (i + 1 == m || x.bin(x.entry_value(x.list[i + 1])) > d_hi))
          sh.pick_at = i + 1;
      }
      __syncthreads();
      m1 = sh.pick_at;
    }
    u64 first = m1 > 0 ? cum[m1 - 1] : 0ull;
    const u64 lift = split ? above2 - above - first : 0ull;  // weights between the ranges
    const u64 span = m > 0 ? above + cum[m - 1] + lift : 0ull;
    total = all;
    bool ok = m > 0;
    if (cut_p && ok) {
      const u64 goal = max((u64)ceil(p_share * (double)all), 1ull);
      const u64 from = split ? above + first + lift : above;  // before the border's range
      ok = goal > from && goal <= span;
      if (ok) total = above + lift + cum[x.find_entry(cum, m, goal - above - lift)];
    }
    if (ok && apart) {
      x.command(RowsCmd{kOpGather, 1, (uint32_t)d_lo, (uint32_t)d_hi, 0, 0, 0, 0, 1, 0});
      m = m1 = x.collect();
      x.sort_list(cum, m);
      above = above2;
      first = m > 0 ? cum[m - 1] : 0ull;
    }
    if (ok) {
      const u64 goal = min((u64)floor((double)u * (double)total), total - 1) + 1;
      ok = m1 > 0 && goal > above && goal <= above + first;
      if (ok) {
        const int at = x.find_entry(cum, m1, goal - above);
        id = (int)(uint32_t)x.list[at];
        logp = share(~(uint32_t)(x.list[at] >> 32));
        settled = true;
        x.command(end);
      }
    }
  }
  if (!settled) {
    x.command(all_bins);
    bins = x.read_bins(RowsCta::kExact);
    if (tid == kRowsThreads - 1) sh.whole = bins.mrun[3];
    __syncthreads();
    RowsPrefix keep{0u, a.vocab, sh.whole};
    int unused;
    if (few) keep = x.resolve(bins, (u64)top_k, true, false, &unused);
    if (cut_p) {
      const RowsPrefix p = x.resolve(bins, max((u64)ceil(p_share * (double)keep.mass), 1ull), false, false, &unused);
      if (p.key > keep.key || (p.key == keep.key && p.ties < keep.ties)) keep = p;
    }
    if (min_p > 1.0f) {
      keep.mass = x.weight(mx);
    } else if (cut_m && kmin > keep.key) {
      keep.mass = x.total_of(RowsCmd{kOpMass, 0, kmin, 0xffffffffu, 0, 0, 0, 0, 1, 0});
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
  // CTAs per row: enough that a CTA holds at most 20480 tokens (two CTAs an SM; without a copy in shared
  // memory, passes over L1 and L2 took 1.2 to 1.5 times as long) and, with few rows, that the SMs are
  // used; a CTA below 2048 tokens gains nothing any more.
  int C = 1;
  while (C < kRowsMaxCluster && ((a.vocab + C - 1) / C > 20480 ||
                                 ((long long)rows * C < 2 * current_sms() && (a.vocab + C - 1) / C > 2048)))
    C *= 2;
  a.per = ((a.vocab + C - 1) / C + 7) / 8 * 8;
  const size_t smem = kRowsBins * 8 + kRowsList * 8 + (size_t)a.per * 4;
  static unsigned long long smem_set = 0;
  allow_smem(k_sample_rows<T>, kRowsBins * 8 + kRowsList * 8 + (size_t)kRowsMaxPer * 4, smem_set);
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
