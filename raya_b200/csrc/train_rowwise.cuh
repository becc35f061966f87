// train_rowwise.cuh — the training operators for any head_dim (a multiple of
// 8, at most 256): one warp per row, partners in chunks of 32, one lane per
// partner for the dot products and one lane per column for the sums.  Every
// sum is held in 32 bits and taken in a fixed order.
#pragma once

#include "train_common.cuh"

namespace raya {
namespace train {

constexpr int kRowWarps = 4;
constexpr int kRowThreads = kRowWarps * 32;
constexpr int kRowMaxD = 256;
constexpr int kRowCols = kRowMaxD / 32;

// x . y over d floats, x in shared memory, y in global memory (both 16-byte aligned).
__device__ __forceinline__ float dot_row(const float* xs, const float* __restrict__ y, int d) {
  float acc = 0.f;
  for (int c = 0; c < d; c += 4) {
    const float4 a = *reinterpret_cast<const float4*>(xs + c);
    const float4 b = __ldg(reinterpret_cast<const float4*>(y + c));
    acc = fmaf(a.x, b.x, acc);
    acc = fmaf(a.y, b.y, acc);
    acc = fmaf(a.z, b.z, acc);
    acc = fmaf(a.w, b.w, acc);
  }
  return acc;
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
  return x;
}

// Block b of the grid runs rows w, w + step, ... of slice b / parts, where w
// counts its warps among the slice's.
struct RowJob {
  long long bh;
  int head, valid, first, step;
};
__device__ __forceinline__ RowJob row_job(const TrainArgs& t, int warp) {
  RowJob j;
  j.bh = blockIdx.x / t.parts;
  const int part = static_cast<int>(blockIdx.x - j.bh * t.parts);
  j.head = static_cast<int>(j.bh % t.a.heads);
  const int v = t.a.valid_len ? t.a.valid_len[j.bh / t.a.heads] : t.a.seq;
  j.valid = v < 0 ? 0 : (v > t.a.seq ? t.a.seq : v);
  j.first = part * kRowWarps + warp;
  j.step = t.parts * kRowWarps;
  return j;
}

__global__ void __launch_bounds__(kRowThreads) rowwise_train_fwd(const __grid_constant__ TrainArgs t) {
  __shared__ __align__(16) float qs[kRowWarps][kRowMaxD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = t.a.head_dim;
  const RowJob job = row_job(t, warp);
  const float* bias = t.rel_bias ? t.rel_bias + (2ll * job.head + 1) * t.rel_half : nullptr;
  const size_t base = static_cast<size_t>(job.bh) * t.a.seq;
  for (int i = job.first; i < t.a.seq; i += job.step) {
    float* orow = t.a.out + (base + i) * d;
    int lo = 0, hi = 0;
    if (i < job.valid) {
      key_range(t.a, i, job.valid, lo, hi);
      for (int c = lane; c < d; c += 32) qs[warp][c] = t.a.q[(base + i) * d + c];
    }
    __syncwarp();
    float o[kRowCols];
#pragma unroll
    for (int u = 0; u < kRowCols; ++u) o[u] = 0.f;
    float m = -INFINITY, l = 0.f;  // l: this lane's share
    for (int j0 = lo; j0 < hi; j0 += 32) {
      const int j = j0 + lane;
      float x = -INFINITY;
      if (j < hi) x = fmaf(dot_row(qs[warp], t.a.k + (base + j) * d, d), t.a.qscale, bias ? bias[j - i] : 0.f);
      const float mnew = fmaxf(m, warp_max(x));
      const float mbase = mnew == -INFINITY ? 0.f : mnew;
      const float alpha = ex2(m - mbase), p = ex2(x - mbase);
      m = mnew;
      l = fmaf(l, alpha, p);
#pragma unroll
      for (int u = 0; u < kRowCols; ++u) o[u] *= alpha;
      const int nk = min(32, hi - j0);
      for (int jj = 0; jj < nk; ++jj) {
        const float pj = __shfl_sync(0xffffffffu, p, jj);
        const float* vrow = t.a.v + (base + j0 + jj) * d;
        if (pj != 0.f) {  // also false for none: a NaN weight counts
#pragma unroll
          for (int u = 0; u < kRowCols; ++u)
            if (lane + 32 * u < d) o[u] = fmaf(pj, vrow[lane + 32 * u], o[u]);
        }
      }
    }
    l = warp_sum(l);
    const float inv = l > 0.f ? 1.0f / l : l != l ? l : 0.f;
#pragma unroll
    for (int u = 0; u < kRowCols; ++u)
      if (lane + 32 * u < d) orow[lane + 32 * u] = o[u] * inv;
    if (t.stats_out && lane == 0) t.stats_out[base + i] = make_stats(m, m == -INFINITY ? 0.f : m, l);
    __syncwarp();
  }
}

// dq and delta, and the partials of the table's gradient: each thread adds
// its ds into a column of its own of acc[bucket][thread], which the block
// sums in a fixed order at its end.
__global__ void __launch_bounds__(kRowThreads) rowwise_train_dq(const __grid_constant__ TrainArgs t) {
  __shared__ __align__(16) float qs[kRowWarps][kRowMaxD], gs[kRowWarps][kRowMaxD];
  extern __shared__ float acc[];  // [buckets][kRowThreads] with t.part
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = t.a.head_dim;
  const RowJob job = row_job(t, warp);
  const float* bias = t.rel_bias ? t.rel_bias + (2ll * job.head + 1) * t.rel_half : nullptr;
  const uint8_t* ids = t.rel_id + t.rel_half;
  const size_t base = static_cast<size_t>(job.bh) * t.a.seq;
  if (t.part)
    for (int b = 0; b < t.buckets; ++b) acc[b * kRowThreads + threadIdx.x] = 0.f;
  for (int i = job.first; i < t.a.seq; i += job.step) {
    float* dqrow = t.dq + (base + i) * d;
    int lo = 0, hi = 0;
    float delta = 0.f, m2 = 0.f, linv = 0.f;
    if (i < job.valid) {
      key_range(t.a, i, job.valid, lo, hi);
      for (int c = lane; c < d; c += 32) {
        qs[warp][c] = t.a.q[(base + i) * d + c];
        const float g = t.dout[(base + i) * d + c];
        gs[warp][c] = g;
        delta = fmaf(g, t.a.out[(base + i) * d + c], delta);
      }
      delta = warp_sum(delta);
      row_stats(t.stats[base + i], m2, linv);
    }
    if (lane == 0) t.delta[base + i] = delta;
    __syncwarp();
    float o[kRowCols];
#pragma unroll
    for (int u = 0; u < kRowCols; ++u) o[u] = 0.f;
    for (int j0 = lo; j0 < hi; j0 += 32) {
      const int j = j0 + lane;
      float ds = 0.f;
      if (j < hi) {
        const float x = fmaf(dot_row(qs[warp], t.a.k + (base + j) * d, d), t.a.qscale, bias ? bias[j - i] : 0.f);
        const float p = ex2(x - m2) * linv;
        if (p != 0.f) ds = p * (dot_row(gs[warp], t.a.v + (base + j) * d, d) - delta);
        if (t.part) acc[ids[j - i] * kRowThreads + threadIdx.x] += ds;
      }
      const int nk = min(32, hi - j0);
      for (int jj = 0; jj < nk; ++jj) {
        const float w = __shfl_sync(0xffffffffu, ds, jj);
        const float* krow = t.a.k + (base + j0 + jj) * d;
#pragma unroll
        for (int u = 0; u < kRowCols; ++u)
          if (lane + 32 * u < d) o[u] = fmaf(w, krow[lane + 32 * u], o[u]);
      }
    }
    const float f = i < job.valid ? t.scale : 1.f;  // padded rows stay +0 under a negative scale
#pragma unroll
    for (int u = 0; u < kRowCols; ++u)
      if (lane + 32 * u < d) dqrow[lane + 32 * u] = o[u] * f;
    __syncwarp();
  }
  if (t.part) {
    __syncthreads();
    for (int b = warp; b < t.buckets; b += kRowWarps) {
      float s = 0.f;
      for (int u = lane; u < kRowThreads; u += 32) s += acc[b * kRowThreads + u];
      s = warp_sum(s);
      if (lane == 0) t.part[static_cast<size_t>(blockIdx.x) * t.buckets + b] = s;
    }
  }
}

// dk and dv: one warp per key row, its queries in chunks of 32.
__global__ void __launch_bounds__(kRowThreads) rowwise_train_dkv(const __grid_constant__ TrainArgs t) {
  __shared__ __align__(16) float ks[kRowWarps][kRowMaxD], vs[kRowWarps][kRowMaxD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = t.a.head_dim;
  const RowJob job = row_job(t, warp);
  const float* bias = t.rel_bias ? t.rel_bias + (2ll * job.head + 1) * t.rel_half : nullptr;
  const size_t base = static_cast<size_t>(job.bh) * t.a.seq;
  for (int j = job.first; j < t.a.seq; j += job.step) {
    int lo = 0, hi = 0;
    if (j < job.valid) {
      key_range(t.a, j, job.valid, lo, hi);
      for (int c = lane; c < d; c += 32) {
        ks[warp][c] = t.a.k[(base + j) * d + c];
        vs[warp][c] = t.a.v[(base + j) * d + c];
      }
    }
    __syncwarp();
    float ok[kRowCols], ov[kRowCols];
#pragma unroll
    for (int u = 0; u < kRowCols; ++u) ok[u] = ov[u] = 0.f;
    for (int i0 = lo; i0 < hi; i0 += 32) {
      const int i = i0 + lane;
      float p = 0.f, ds = 0.f;
      if (i < hi) {
        float m2, linv;
        row_stats(t.stats[base + i], m2, linv);
        const float x = fmaf(dot_row(ks[warp], t.a.q + (base + i) * d, d), t.a.qscale, bias ? bias[j - i] : 0.f);
        p = ex2(x - m2) * linv;
        if (p != 0.f) ds = p * (dot_row(vs[warp], t.dout + (base + i) * d, d) - t.delta[base + i]);
      }
      const int nq = min(32, hi - i0);
      for (int ii = 0; ii < nq; ++ii) {
        const float w = __shfl_sync(0xffffffffu, ds, ii), pw = __shfl_sync(0xffffffffu, p, ii);
        const float* qrow = t.a.q + (base + i0 + ii) * d;
        const float* grow = t.dout + (base + i0 + ii) * d;
#pragma unroll
        for (int u = 0; u < kRowCols; ++u)
          if (lane + 32 * u < d) {
            ok[u] = fmaf(w, qrow[lane + 32 * u], ok[u]);
            ov[u] = fmaf(pw, grow[lane + 32 * u], ov[u]);
          }
      }
    }
    const float f = j < job.valid ? t.scale : 1.f;  // as in rowwise_train_dq
#pragma unroll
    for (int u = 0; u < kRowCols; ++u)
      if (lane + 32 * u < d) {
        t.dk[(base + j) * d + lane + 32 * u] = ok[u] * f;
        t.dv[(base + j) * d + lane + 32 * u] = ov[u];
      }
    __syncwarp();
  }
}

}  // namespace train
}  // namespace raya
