// Decode attention of groups of sequences that share their first positions.
//
// Sequence b of a group sees its first shared_lens[b] positions through the group's first sequence's row of the
// block table and the others through its own:
//   y = (sum over both of exp(s_j - m) v_j) / (sum over both of exp(s_j - m)),
// and each sum is taken where its keys are cheapest:
//  - the shared ones once for all the group's queries (k_paged_prompt with SHARED: the queries of a KV head of all
//    the group's sequences are the rows of its 128-row tiles, so the prefix is read once a tile, and what was
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

// A CTA takes eight rows (sequence, query head of KV head g), a thread four dims of one and every fourth part; grid:
// (rows / 8, kv_heads). What bounds it is the chain of lookups, each a trip to L2, so there are two: the
// row's places, all its parts (one thread for all of a row's parts took 9 us for 64 sequences and 18 parts).
constexpr int kPsThreads = 1024;
__global__ void __launch_bounds__(kPsThreads) k_paged_shared_join(const __grid_constant__ PSharedArgs pa) {
  const PAttnArgs& a = pa.a;
  __shared__ float2 sml[3][8];
  __shared__ float4 so[3][256];
  const int kvh = a.kv.kv_heads, G = a.q_heads / kvh, subs = (G + 7) >> 3, nh = kvh * subs;
  const int tid = threadIdx.x & 255, zl = threadIdx.x >> 8;
  const int row = blockIdx.x * 8 + (tid & 7), d4 = tid >> 3, g = blockIdx.y;
  const int b = min(row / G, a.kv.batch - 1), hs = row % G;
  pdl_wait();
  pdl_trigger();
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.mark = 0;  // (a captured call has one ticket for all replays)
  const PDecodeWs ws = pd_ws(pa.decode_ws);
  int2 at = pa.rows[min(row, a.kv.batch * G - 1)];
  const int f0 = ws.first[b], f1 = ws.first[b + 1], all = ws.first[a.kv.batch];
  const bool live = row < a.kv.batch * G && b >= a.q_starts[0] && b < a.q_starts[a.groups];  // (others are padding)
  if (!live || (unsigned)at.x >= (unsigned)pa.all_rows || at.y > pa.splits) at = make_int2(0, 0);  // (or starts do not ascend)
  const int item = at.x / pa.cta_rows, lr = at.x - item * pa.cta_rows;
  const long long p0 = ((long long)item * kvh + g) * pa.splits * pa.cta_rows;
  const float2* ml = pa.pml + p0 + lr;
  const float4* po = pa.po + p0 * (kHeadDim / 4) + (long long)d4 * pa.cta_rows + lr;
  // its own positions: the CTAs c0 .. c0 + own - 1 of the TAIL launch, or one that held them whole
  const int tiles = live ? f1 - f0 : 0;
  const long long U = (long long)all * nh;
  const int ctas = (int)min((long long)pa.ctas, U);
  const long long v0 = (long long)f0 * nh + (long long)(g * subs + (hs >> 3)) * tiles;
  int c0 = 0, own = 0;
  if (tiles > 0) {
    c0 = pd_div((v0 + 1) * ctas - 1, U);
    own = pd_div((v0 + tiles) * ctas - 1, U) - c0 + 1;
  }
  const long long mine = (long long)b * a.q_heads + g * G + hs;
  float M = -INFINITY, L = 0.0f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  const int n = at.y + own;
  constexpr int N = 4;  // parts in flight
  for (int z0 = zl; z0 < n; z0 += 4 * N) {
    float2 s[N];
    float4 x[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int z = z0 + 4 * k;
      s[k] = make_float2(-INFINITY, 0.0f);
      x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (z < at.y) {
        s[k] = ml[z * pa.cta_rows];
        x[k] = po[(long long)z * pa.cta_rows * (kHeadDim / 4)];
      } else if (z < n) {
        const int c = c0 + z - at.y;
        const long long i = own == 1 ? mine : (2ll * c + (pd_div(U * c, ctas) >= v0 ? 0 : 1)) * 8 + (hs & 7);
        s[k] = (own == 1 ? a.tail_ml : ws.ml)[i];
        x[k] = *reinterpret_cast<const float4*>((own == 1 ? a.tail_o : ws.o) + i * kHeadDim + 4 * d4);
      }
    }
    float mn = M;
#pragma unroll
    for (int k = 0; k < N; ++k) mn = fmaxf(mn, s[k].x);
    const float fo = M == -INFINITY ? 0.0f : exp2_fast(M - mn);
    M = mn;
    L *= fo;
    y = make_float4(y.x * fo, y.y * fo, y.z * fo, y.w * fo);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float f = s[k].x == -INFINITY ? 0.0f : exp2_fast(s[k].x - M);
      L = fmaf(s[k].y, f, L);
      y = make_float4(fmaf(x[k].x, f, y.x), fmaf(x[k].y, f, y.y), fmaf(x[k].z, f, y.z), fmaf(x[k].w, f, y.w));
    }
  }
  if (zl) {
    so[zl - 1][tid] = y;
    if (d4 == 0) sml[zl - 1][tid & 7] = make_float2(M, L);
  }
  __syncthreads();
  if (zl || !live) return;
  float top = M;
#pragma unroll
  for (int k = 0; k < 3; ++k) top = fmaxf(top, sml[k][tid & 7].x);
  const float fo = M == -INFINITY ? 0.0f : exp2_fast(M - top);
  L *= fo;
  y = make_float4(y.x * fo, y.y * fo, y.z * fo, y.w * fo);
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const float2 s = sml[k][tid & 7];
    const float4 x = so[k][tid];
    const float f = s.x == -INFINITY ? 0.0f : exp2_fast(s.x - top);
    L = fmaf(s.y, f, L);
    y = make_float4(fmaf(x.x, f, y.x), fmaf(x.y, f, y.y), fmaf(x.z, f, y.z), fmaf(x.w, f, y.w));
  }
  const float z = inv_sum(L);
  store4(a.y, b * a.y_stride + ((long long)g * G + hs) * kHeadDim + 4 * d4, a.dtype,
         make_float4(y.x * z, y.y * z, y.z * z, y.w * z));
}

}  // namespace qd
