// Operators over a paged key-value cache: the fused head norm + rotation + append, and
// attention of new tokens over the pages.
//
// Pools K, V: [page][kv_head][page_size][128]; the page_size rows of one (page, KV head) are
// one contiguous range, which is what the attention kernels copy. Position p of sequence b
// lives in page table[b][p / page_size], row p % page_size.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace qd {

struct PagedArgs {
  void* k;
  void* v;
  int num_pages, page_shift;  // page_size = 1 << page_shift
  int kv_heads, batch;
  const int* table;
  int table_width, table_stride;
  const int* seq_lens;
  int* status;
};

__device__ __forceinline__ void paged_flag(const PagedArgs& a, int bits) {
  if (a.status) atomicOr(a.status, bits);
}

// Length of sequence b, cut to what its table row can name.
__device__ __forceinline__ int paged_len(const PagedArgs& a, int b) {
  return min(max(a.seq_lens[b], 0), a.table_width << a.page_shift);
}

// Page of position p (inside the table), or -1.
__device__ __forceinline__ int paged_page(const PagedArgs& a, int b, int p) {
  const int page = a.table[(long long)b * a.table_stride + (p >> a.page_shift)];
  return (unsigned)page < (unsigned)a.num_pages ? page : -1;
}

// Sequence of row r: the b with q_starts[b] <= r < q_starts[b + 1], or -1 (padding rows).
// Every lane of a warp calls it with the same r; 32 entries are compared per round trip. The first
// trip tells whether the row is padding; if it is not, load() is called then, and what it
// reads comes under the rest of the search (up to 32 sequences have none).
template <typename F>
__device__ __forceinline__ int paged_find_seq(const int* q_starts, int batch, int r, F&& load) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = batch;  // entries [lo, hi] bracket the answer: q_starts[lo] <= r
  bool first = true;
  do {
    const int step = (hi - lo + 31) >> 5;
    const int e = q_starts[min(lo + (lane + 1) * step, hi)];
    const unsigned le = __ballot_sync(0xffffffffu, e <= r);
    if (first) {
      if (r < q_starts[0] || le >> 31) return -1;  // (the last lane holds entry hi)
      load();
      first = false;
    }
    const int n = __popc(le);  // ascending entries: the lanes at or below r are a prefix
    const int nlo = lo + n * step;
    hi = min(nlo + step, hi);
    lo = min(nlo, hi - 1);
  } while (hi - lo > 1);
  return lo;
}

// Four consecutive elements as f32, and back with one rounding.
template <typename T>
__device__ __forceinline__ float4 load4(const void* base, long long e);
template <>
__device__ __forceinline__ float4 load4<float>(const void* base, long long e) {
  return *reinterpret_cast<const float4*>(static_cast<const float*>(base) + e);
}
template <>
__device__ __forceinline__ float4 load4<__half>(const void* base, long long e) {
  const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __half*>(base) + e);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
template <>
__device__ __forceinline__ float4 load4<__nv_bfloat16>(const void* base, long long e) {
  const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(base) + e);
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xffff0000u));
}

__device__ __forceinline__ void store4(void* base, long long e, int dtype, float4 x) {
  if (dtype == QD_KV_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(base) + e) = x;
  } else if (dtype == QD_KV_F16) {
    const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
    *reinterpret_cast<uint2*>(static_cast<__half*>(base) + e) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  } else {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(base) + e) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
}

// ---- head RMSNorm + rotation + append ------------------------------------------------
struct AppendArgs {
  PagedArgs kv;
  int kv_dtype;
  const void* qkv;
  long long qkv_stride;
  int rows;
  const int* q_starts;
  int q_heads;
  const float* q_norm;
  const float* k_norm;
  float eps;
  const float* cos_t;
  const float* sin_t;
  long long rope_len, rope_stride;
  void* q_out;
  int q_out_dtype;
  long long q_out_stride;
  float *k_scale, *v_scale;  // of an 8-bit cache
};

// One warp per row and HEADS consecutive heads of its [q | k | v]; lane l holds dims 4l .. 4l+3, so
// the rotation's partner dims are 16 lanes away. What it has to move bounds it (per row and head 512
// bytes of f32 in, 512 or 256 out), so the heads' loads go out as soon as the row is known not to be
// padding, and its sequence, position and page are looked up under them; the heads' sums of squares
// then run side by side.
// HEADS: 4 keep 2 KB in flight per warp at 40 warps an SM (16384 rows of 16 + 8 + 8 heads, f32, 470 MB:
// 82 us = 5.7 TB/s, 88 with 8); with few rows 2 spread the work over more warps (1 row: 2.5 us, 3.2
// with 4).
template <typename T, int HEADS>
__global__ void __launch_bounds__(256, HEADS == 4 ? 5 : 6) k_paged_append(const __grid_constant__ AppendArgs a) {
  const int lane = threadIdx.x & 31;
  const int heads = a.q_heads + 2 * a.kv.kv_heads;
  const unsigned per_row = (unsigned)(heads + HEADS - 1) / HEADS;
  const unsigned w = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int r = (int)(w / per_row), h0 = (int)(w % per_row) * HEADS;
  if (r >= a.rows) return;
  pdl_wait();
  float4 x[HEADS];
  auto load = [&] {
#pragma unroll
    for (int i = 0; i < HEADS; ++i)
      x[i] = load4<T>(a.qkv, r * a.qkv_stride + (long long)min(h0 + i, heads - 1) * kHeadDim + 4 * lane);
  };
  int b = r, back = 1;
  if (a.q_starts) {
    b = paged_find_seq(a.q_starts, a.kv.batch, r, load);
    if (b < 0) return;
    back = a.q_starts[b + 1] - r;
  } else {
    load();
  }
  const int p = a.kv.seq_lens[b] - back;
  const long long t = (long long)p * a.rope_stride + 4 * (lane & 15);
  const bool turned = a.cos_t != nullptr;
  const bool live = p >= 0 && p < (a.kv.table_width << a.kv.page_shift) &&
                    (!turned || (long long)p * a.rope_stride + kHeadDim / 2 <= a.rope_len);
  if (!live) {
    if (lane == 0) paged_flag(a.kv, QD_PAGED_BAD_LENGTH);
    return;
  }
  float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (turned) {
    c = *reinterpret_cast<const float4*>(a.cos_t + t);
    s = *reinterpret_cast<const float4*>(a.sin_t + t);
    if (lane < 16) s = make_float4(-s.x, -s.y, -s.z, -s.w);
  }
  int page = -1;
  if (h0 + HEADS > a.q_heads) {
    page = paged_page(a.kv, b, p);
    if (page < 0 && lane == 0) paged_flag(a.kv, QD_PAGED_BAD_PAGE);
  }
  const int k0 = a.q_heads, v0 = a.q_heads + a.kv.kv_heads;
  float ss[HEADS];
#pragma unroll
  for (int i = 0; i < HEADS; ++i) ss[i] = x[i].x * x[i].x + x[i].y * x[i].y + x[i].z * x[i].z + x[i].w * x[i].w;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < HEADS; ++i) ss[i] += __shfl_xor_sync(0xffffffffu, ss[i], o);
  const int in_page = p & ((1 << a.kv.page_shift) - 1);
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const int h = h0 + i;
    if (h >= heads) break;
    float4 y = x[i];
    if (h < v0) {
      const float* wn = h < k0 ? a.q_norm : a.k_norm;
      if (wn) {
        const float f = rsqrtf(ss[i] * (1.0f / kHeadDim) + a.eps);
        const float4 n = *reinterpret_cast<const float4*>(wn + 4 * lane);
        y = make_float4(y.x * f * n.x, y.y * f * n.y, y.z * f * n.z, y.w * f * n.w);
      }
      if (turned) {
        const float4 o = make_float4(__shfl_xor_sync(0xffffffffu, y.x, 16), __shfl_xor_sync(0xffffffffu, y.y, 16),
                                     __shfl_xor_sync(0xffffffffu, y.z, 16), __shfl_xor_sync(0xffffffffu, y.w, 16));
        y = make_float4(y.x * c.x + o.x * s.x, y.y * c.y + o.y * s.y, y.z * c.z + o.z * s.z, y.w * c.w + o.w * s.w);
      }
    }
    if (h < k0) {
      store4(a.q_out, r * a.q_out_stride + (long long)h * kHeadDim + 4 * lane, a.q_out_dtype, y);
    } else if (page >= 0) {
      const int g = h < v0 ? h - k0 : h - v0;
      const long long row = (((long long)page * a.kv.kv_heads + g) << a.kv.page_shift) + in_page;
      store4(h < v0 ? a.kv.k : a.kv.v, row * kHeadDim + 4 * lane, a.kv_dtype, y);
    }
  }
}

// The same into a cache of 8-bit integers n with a scale per row: scale = the largest magnitude / 127, n = 127 x / the largest
// rounded, halves to even, by an addition of 1.5 * 2^23 whose sum's low byte is n. Halves are common (any element that
// is half the largest), so the quotient q = x / scale gets one residual: q + (127 x - q max) / max is off by no more than its
// own rounding, 2^-17 of a step, and a half comes out as one. (Without it about half of the halves of 16-bit rows went to
// the other integer: read back in f16, V was 6.5e-4 off from bf16 rows and 3.7e-4 from f16 rows, both 2.0e-4 so; it takes 2.3
// us of 16384 rows.) With f32 rows 127 x is the product and what it rounds off. All of it over 128, so that no product
// leaves f32. A row with an element that is not
// finite gets a NaN scale (all of it reads as NaN), one whose largest is below 2^-100 a scale of 0.
//
// Half a warp per head: lane h of it holds dims 4 h .. + 3 and 64 + 4 h .. + 3, which the rotation turns into
// each other, and a sum or maximum takes four steps for two heads at once. (The other kernel's lanes, with the rows'
// maxima and divisions added, were bound by instructions: 16384 rows of 16 + 8 + 8 heads, f32, 437 MB, 98 us; so 73 us = 6.0 TB/s.
// Rows of f16 or bf16, 236 MB, take 73 us too: 75 % of the issue slots are taken with either.)
// Sums run in that kernel's order: q comes out the same to the bit.
template <typename T, int PAIRS>
__global__ void __launch_bounds__(256, PAIRS == 2 ? 5 : 6) k_paged_append_q8(const __grid_constant__ AppendArgs a) {
  const int lane = threadIdx.x & 31, hl = lane & 15, half = lane >> 4;
  const int heads = a.q_heads + 2 * a.kv.kv_heads, k0 = a.q_heads, v0 = a.q_heads + a.kv.kv_heads;
  const unsigned per_row = (unsigned)(heads + 2 * PAIRS - 1) / (2 * PAIRS);
  const unsigned w = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int r = (int)(w / per_row), h0 = (int)(w % per_row) * (2 * PAIRS);
  if (r >= a.rows) return;
  pdl_wait();
  float4 x[PAIRS][2];
  auto load = [&] {
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      const long long at = r * a.qkv_stride + (long long)min(h0 + 2 * i + half, heads - 1) * kHeadDim + 4 * hl;
      x[i][0] = load4<T>(a.qkv, at);
      x[i][1] = load4<T>(a.qkv, at + kHeadDim / 2);
    }
  };
  int b = r, back = 1;
  if (a.q_starts) {
    b = paged_find_seq(a.q_starts, a.kv.batch, r, load);
    if (b < 0) return;
    back = a.q_starts[b + 1] - r;
  } else {
    load();
  }
  const int p = a.kv.seq_lens[b] - back;
  const long long t = (long long)p * a.rope_stride + 4 * hl;
  const bool turned = a.cos_t != nullptr;
  const bool live = p >= 0 && p < (a.kv.table_width << a.kv.page_shift) &&
                    (!turned || (long long)p * a.rope_stride + kHeadDim / 2 <= a.rope_len);
  if (!live) {
    if (lane == 0) paged_flag(a.kv, QD_PAGED_BAD_LENGTH);
    return;
  }
  float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (turned && h0 < v0) {
    c = *reinterpret_cast<const float4*>(a.cos_t + t);
    s = *reinterpret_cast<const float4*>(a.sin_t + t);
  }
  int page = -1;
  if (h0 + 2 * PAIRS > k0) {
    page = paged_page(a.kv, b, p);
    if (page < 0 && lane == 0) paged_flag(a.kv, QD_PAGED_BAD_PAGE);
  }
  if (h0 < v0) {  // (warp-uniform: V rows are written as they are)
    float ss[PAIRS];
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      const float4 u = x[i][0], v = x[i][1];
      const float su = fmaf(u.w, u.w, fmaf(u.z, u.z, fmaf(u.x, u.x, u.y * u.y)));
      const float sv = fmaf(v.w, v.w, fmaf(v.z, v.z, fmaf(v.x, v.x, v.y * v.y)));
      ss[i] = su + sv;
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) ss[i] += __shfl_xor_sync(0xffffffffu, ss[i], o);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      const int h = h0 + 2 * i + half;
      if (h >= v0) continue;
      float4 u = x[i][0], v = x[i][1];
      const float* wn = h < k0 ? a.q_norm : a.k_norm;
      if (wn) {
        const float f = rsqrtf(ss[i] * (1.0f / kHeadDim) + a.eps);
        const float4 n = *reinterpret_cast<const float4*>(wn + 4 * hl);
        const float4 m = *reinterpret_cast<const float4*>(wn + kHeadDim / 2 + 4 * hl);
        u = make_float4(u.x * f * n.x, u.y * f * n.y, u.z * f * n.z, u.w * f * n.w);
        v = make_float4(v.x * f * m.x, v.y * f * m.y, v.z * f * m.z, v.w * f * m.w);
      }
      if (turned) {
        // (which product is rounded, as in the other kernel)
        x[i][0] = make_float4(fmaf(u.x, c.x, v.x * -s.x), fmaf(u.y, c.y, v.y * -s.y), fmaf(u.z, c.z, v.z * -s.z),
                              fmaf(u.w, c.w, v.w * -s.w));
        x[i][1] = make_float4(fmaf(v.x, c.x, u.x * s.x), fmaf(v.y, c.y, u.y * s.y), fmaf(v.z, c.z, u.z * s.z),
                              fmaf(v.w, c.w, u.w * s.w));
      } else {
        x[i][0] = u;
        x[i][1] = v;
      }
      if (h < k0) {
        const long long at = r * a.q_out_stride + (long long)h * kHeadDim + 4 * hl;
        store4(a.q_out, at, a.q_out_dtype, x[i][0]);
        store4(a.q_out, at + kHeadDim / 2, a.q_out_dtype, x[i][1]);
      }
    }
  }
  if (page < 0) return;
  const int in_page = p & ((1 << a.kv.page_shift) - 1);
  const unsigned none = 0x7fffffffu;
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    if (h0 + 2 * i + 1 < k0) continue;  // (both heads are q's)
    const float4 u = x[i][0], v = x[i][1];
    // the largest magnitude (NaN above infinity above every number)
    unsigned top = max(max(max(__float_as_uint(u.x) & none, __float_as_uint(u.y) & none),
                           max(__float_as_uint(u.z) & none, __float_as_uint(u.w) & none)),
                       max(max(__float_as_uint(v.x) & none, __float_as_uint(v.y) & none),
                           max(__float_as_uint(v.z) & none, __float_as_uint(v.w) & none)));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float most = __uint_as_float(top), near = most * (1.0f / 127.0f);
    const float scale = fmaf(fmaf(-near, 127.0f, most), 1.0f / 127.0f, near);
    const float up = __fdividef(1.0f, scale), most7 = most * 0.0078125f, up7 = up * (128.0f / 127.0f);
    auto both = [](float y) { return make_float2(y, y); };
    auto whole = [&](float2 y) {
      const float2 q = __fmul2_rn(y, both(up)), z = __fmul2_rn(y, both(0.9921875f));  // 127 / 128
      float2 rest = __ffma2_rn(make_float2(-q.x, -q.y), both(most7), z);
      if constexpr (sizeof(T) == 4) rest = __fadd2_rn(rest, __ffma2_rn(y, both(0.9921875f), make_float2(-z.x, -z.y)));
      return __fadd2_rn(__ffma2_rn(rest, both(up7), q), both(12582912.0f));
    };
    auto bytes = [&](float4 y) {
      const float2 d = whole(make_float2(y.x, y.y)), e = whole(make_float2(y.z, y.w));
      return __byte_perm(__byte_perm(__float_as_uint(d.x), __float_as_uint(d.y), 0x0040),
                         __byte_perm(__float_as_uint(e.x), __float_as_uint(e.y), 0x0040), 0x5410);
    };
    const int h = h0 + 2 * i + half;
    if (h < k0 || h >= heads) continue;
    const bool fits = top < 0x7f800000u && top >= 27u << 23;
    const int g = h < v0 ? h - k0 : h - v0;
    const long long row = (((long long)page * a.kv.kv_heads + g) << a.kv.page_shift) + in_page;
    unsigned* n = reinterpret_cast<unsigned*>(static_cast<int8_t*>(h < v0 ? a.kv.k : a.kv.v) + row * kHeadDim) + hl;
    n[0] = fits ? bytes(u) : 0u;
    n[16] = fits ? bytes(v) : 0u;
    if (hl == 0) (h < v0 ? a.k_scale : a.v_scale)[row] = fits ? scale : top >= 0x7f800000u ? __uint_as_float(none) : 0.0f;
  }
}

// ---- attention of new tokens -----------------------------------------------------------
struct PAttnArgs {
  PagedArgs kv;
  const void* q;
  long long q_stride;
  int rows;
  const int* q_starts;
  int q_heads;
  int window, sinks;
  float scale;
  void* y;
  int dtype;  // of q and y
  long long y_stride;
  // Shared prefixes: q_starts holds the groups' first sequences (groups + 1 entries).
  int groups;
  const int* shared_lens;  // [batch]
  float* tail_o;           // [batch][q_heads][128]: unnormalised sums of the positions behind them,
  float2* tail_ml;         // [batch][q_heads]: with their maxima and weights
  // The launch over the shared positions writes the call's ticket here when all before it is done, the join clears it.
  unsigned long long *mark, ticket;
};

}  // namespace qd
