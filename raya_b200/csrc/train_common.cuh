// train_common.cuh — what the kernels of the training operators share: their
// launch arguments, the table of the relative position bias by distance, and
// the sum of the bias gradient's partials.
//
// The operators (include/raya_attn.h, raya_attn_forward_bias and
// raya_attn_backward).  For query i and key j = i + rel that the mask allows,
//   x_ij  = scale * q_i . k_j + table[head][bucket(rel)],
//   m_i   = max_j x_ij,   l_i = sum_j exp(x_ij - m_i),   p_ij = exp(x_ij - m_i) / l_i,
//   out_i = sum_j p_ij v_j,
// and backward, with delta_i = dout_i . out_i and ds_ij = p_ij (dout_i . v_j - delta_i),
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij dout_i,
//   dtable[head][b] = sum of ds_ij over bucket(j - i) = b.
// The exponentials are taken as powers of two: scores enter as x * log2(e),
// so qscale and the bias carry that factor.
//
// Every mask of this library is symmetric in i and j, so the queries that
// see key j are key_range(j).
#pragma once

#include "common.cuh"

namespace raya {
namespace train {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// A bias at or below this masks its bucket, as -inf does: the type's lowest
// value times log2(e) is no float, and no real score comes near it.
constexpr float kMaskedBias = -1.2676506e30f;  // -2^100

constexpr int kMaxBuckets = 64;

struct TrainArgs {
  AttnArgs a;              // q, k, v, out, valid_len, the mask, qscale = scale * log2(e)
  const float* dout;       // [rows][head_dim]
  const float2* stats;     // [rows] (m, l): read by the backward kernels
  float2* stats_out;       // [rows] or nullptr: written by the forward kernels
  float* dq;
  float* dk;
  float* dv;
  const float* rel_bias;   // [heads][2 * rel_half]: bias * log2(e) of rel = index - rel_half, or nullptr
  const uint8_t* rel_id;   // [2 * rel_half]: its bucket (the row-wise kernels)
  int rel_half;
  int buckets;
  float scale;
  float* delta;            // [rows]: dout . out (the row-wise kernels)
  float* part;             // [slices][parts][buckets]: partials of the table's gradient, or nullptr
  int parts;               // partials per slice
};

// Statistics as the kernels use them: the base-2 exponent of the row's
// maximum and 1 / l, both 0 for a row without keys (a NaN sum stays NaN).
__device__ __forceinline__ void row_stats(float2 st, float& m2, float& linv) {
  const bool some = st.y != 0.f;
  m2 = some ? st.x * kLog2e : 0.f;
  linv = some ? 1.0f / st.y : 0.f;
}

// The statistics of a row whose scores, in powers of two, have the maximum
// m2 and the sum l2 of 2^(x - base).  m is rounded to fp32, and l is taken
// against the exponent that row_stats gives back for the rounded m, so that
// forward and backward use the same p to the last rounding of l.
__device__ __forceinline__ float2 make_stats(float m2, float base, float l2) {
  if (!(l2 > 0.f)) return make_float2(l2 != l2 ? l2 : -INFINITY, l2 != l2 ? l2 : 0.f);
  const float m = m2 * kLn2;
  return make_float2(m, l2 * ex2(base - m * kLog2e));
}

// Bounds of the distance buckets of one half: bucket k holds the distances
// from at[k] up to at[k + 1].
struct BucketBounds {
  int at[kMaxBuckets / 2];
};

// The bias by distance: vec[head][rel + half] = table[head][bucket(rel)] *
// log2(e), and where ids is given ids[rel + half] = bucket(rel).  Thread
// `first` of `step` takes every step-th distance; once per call, so that the
// attention kernels copy the slice that a tile needs instead of searching
// buckets.
__device__ __forceinline__ void rel_table(const float* __restrict__ table, int heads, int buckets, int half,
                                          const BucketBounds& b, float* __restrict__ vec, uint8_t* __restrict__ ids,
                                          long long first, long long step) {
  const long long n = 2ll * half;
  for (long long t = first; t < n; t += step) {
    const int rel = static_cast<int>(t - half), dist = rel < 0 ? -rel : rel;
    int lo = 0, hi = buckets / 2 - 1;  // the last bound at or below dist
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (b.at[mid] <= dist)
        lo = mid;
      else
        hi = mid - 1;
    }
    const int id = lo + (rel > 0 ? buckets / 2 : 0);
    for (int h = 0; h < heads; ++h) {
      const float x = table[static_cast<size_t>(h) * buckets + id];
      vec[static_cast<size_t>(h) * n + t] = x <= kMaskedBias ? -INFINITY : x * kLog2e;
    }
    if (ids) ids[t] = static_cast<uint8_t>(id);
  }
}
__global__ void __launch_bounds__(256) rel_table_kernel(const float* table, int heads, int buckets, int half,
                                                        const __grid_constant__ BucketBounds b, float* vec, uint8_t* ids) {
  rel_table(table, heads, buckets, half, b, vec, ids, blockIdx.x * 256ll + threadIdx.x, gridDim.x * 256ll);
}

// Programmatic dependent launch.  A kernel that says launch_dependents lets the
// next one's CTAs start where it leaves room; wait_for_primary returns when
// the kernel before is complete and its writes are visible.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_primary() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// What a kernel learned by that wait, passed on to the kernels behind it that
// do not wait themselves: one lane of a warp that has waited says so, a whole
// warp of the later kernel asks.  Where the word is not (yet) to be seen, that
// warp waits for the launch before it to be complete, which is always enough.
__device__ __forceinline__ void publish_primary(unsigned* word) {
  asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(word), "r"(1u) : "memory");
}
__device__ __forceinline__ void see_primary(const unsigned* word) {
  unsigned seen;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(word) : "memory");
  if (!__all_sync(0xffffffffu, seen == 1u)) wait_for_primary();
  fence_proxy_async_global();
}

// dtable[head][b] = the sum of its partials over the batch and the parts of
// each slice, always in the same order (one block per head and bucket; 256
// strided sums, then a tree), in 64 bits: thousands of partials of either
// sign meet here.  Its blocks wait beside the end of the launch before, while
// the partials are still being written: they are no read-only data, and are
// read from L2.
__global__ void __launch_bounds__(256) bias_grad_kernel(const float* part, int batch, int heads, int parts, int buckets,
                                                        float* dtable) {
  __shared__ double sum[256];
  const int h = blockIdx.x, b = blockIdx.y;
  double s = 0.0;
  wait_for_primary();
  const long long n = static_cast<long long>(batch) * parts;
  for (long long t = threadIdx.x; t < n; t += 256) {
    const long long seq = t / parts, at = (seq * heads + h) * parts + t % parts;
    s += static_cast<double>(__ldcg(part + at * buckets + b));
  }
  sum[threadIdx.x] = s;
  __syncthreads();
  for (int w = 128; w > 0; w >>= 1) {
    if (threadIdx.x < static_cast<unsigned>(w)) sum[threadIdx.x] += sum[threadIdx.x + w];
    __syncthreads();
  }
  if (threadIdx.x == 0) dtable[static_cast<size_t>(h) * buckets + b] = static_cast<float>(sum[0]);
}

}  // namespace train
}  // namespace raya
