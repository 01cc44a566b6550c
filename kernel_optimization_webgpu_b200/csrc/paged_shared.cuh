// Decode attention of groups of sequences that share their first positions.
//
// Sequence b of a group sees its first shared_lens[b] positions through the group's first sequence's row of the
// block table and the others through its own:
//   y = (sum over both of exp(s_j - m) v_j) / (sum over both of exp(s_j - m)),
// and each sum is taken where its keys are cheapest:
//  - the shared ones once for all the group's queries (k_paged_prompt with SHARED: the queries of a KV head of all
//    the group's sequences are the rows of its 128-row tiles, so the prefix is read once a group, and what was
//    4 * 128 operations per byte of K and V becomes as many for each of the group's queries, on tcgen05);
//  - each sequence's own by k_paged_decode with TAIL, in equal runs of units per CTA;
//  - k_paged_shared_join adds the parts of a row in order: those of the shared positions, then its own.
#pragma once

#include "paged_decode.cuh"
#include "paged_prompt.cuh"

namespace qd {

struct PSharedArgs {
  PAttnArgs a;  // kv.batch: sequences
  const float4* po;
  const float2* pml;
  const int2* rows;
  int splits, cta_rows, all_rows;  // all_rows: places in `rows`' numbering
  void* decode_ws;
  int ctas;  // grid of the TAIL launch
};

// A sum and where its maximum and weight are.
struct PsSum {
  float m, l;
  float4 o;
};
__device__ __forceinline__ void ps_add(PsSum& s, float2 ml, float4 x) {
  const float mn = fmaxf(s.m, ml.x);
  const float f = s.m == -INFINITY ? 0.0f : exp2_fast(s.m - mn), e = ml.x == -INFINITY ? 0.0f : exp2_fast(ml.x - mn);
  s.m = mn;
  s.l = fmaf(s.l, f, ml.y * e);
  s.o = make_float4(fmaf(s.o.x, f, x.x * e), fmaf(s.o.y, f, x.y * e), fmaf(s.o.z, f, x.z * e), fmaf(s.o.w, f, x.w * e));
}

// A CTA takes eight rows (sequence, query head of KV head g), a thread four dims of one; grid: (rows / 8, kv_heads).
__global__ void __launch_bounds__(256) k_paged_shared_join(const __grid_constant__ PSharedArgs pa) {
  const PAttnArgs& a = pa.a;
  const int kvh = a.kv.kv_heads, G = a.q_heads / kvh, subs = (G + 7) >> 3, nh = kvh * subs;
  const int row = blockIdx.x * 8 + (threadIdx.x & 7), d4 = threadIdx.x >> 3, g = blockIdx.y;
  const int b = row / G, hs = row - b * G;
  pdl_wait();
  pdl_trigger();
  if (b >= a.kv.batch || b < a.q_starts[0] || b >= a.q_starts[a.groups]) return;  // padding
  PsSum s{-INFINITY, 0.0f, make_float4(0.f, 0.f, 0.f, 0.f)};
  int2 at = pa.rows[row];
  if ((unsigned)at.x >= (unsigned)pa.all_rows || at.y > pa.splits) at = make_int2(0, 0);  // (starts that do not ascend)
  const long long p0 = ((long long)(at.x / pa.cta_rows) * kvh + g) * pa.splits * pa.cta_rows + at.x % pa.cta_rows;
#pragma unroll 4
  for (int z = 0; z < at.y; ++z) {
    const long long p = p0 + (long long)z * pa.cta_rows;
    ps_add(s, pa.pml[p], pa.po[(p - at.x % pa.cta_rows) * (kHeadDim / 4) + (long long)d4 * pa.cta_rows + at.x % pa.cta_rows]);
  }
  const PDecodeWs ws = pd_ws(pa.decode_ws);
  const int f0 = ws.first[b], tiles = ws.first[b + 1] - f0;
  if (tiles > 0) {
    const long long U = (long long)ws.first[a.kv.batch] * nh;
    const int ctas = (int)min((long long)pa.ctas, U);
    const long long v0 = (long long)f0 * nh + (long long)(g * subs + (hs >> 3)) * tiles, v1 = v0 + tiles;
    const int c0 = pd_div((v0 + 1) * ctas - 1, U), c1 = pd_div(v1 * ctas - 1, U);
    if (c0 == c1) {
      const long long i = (long long)b * a.q_heads + g * G + hs;
      ps_add(s, a.tail_ml[i], *reinterpret_cast<const float4*>(a.tail_o + i * kHeadDim + 4 * d4));
    } else {
      for (int c = c0; c <= c1; ++c) {
        const long long i = (2ll * c + (pd_div(U * c, ctas) >= v0 ? 0 : 1)) * 8 + (hs & 7);
        ps_add(s, ws.ml[i], *reinterpret_cast<const float4*>(ws.o + i * kHeadDim + 4 * d4));
      }
    }
  }
  const float z = inv_sum(s.l);
  store4(a.y, b * a.y_stride + ((long long)g * G + hs) * kHeadDim + 4 * d4, a.dtype,
         make_float4(s.o.x * z, s.o.y * z, s.o.z * z, s.o.w * z));
}

}  // namespace qd
