// train_tc.cuh — the training operators on the tensor cores (sm_100a,
// tcgen05.mma kind::f16 in 3xFP16), head_dim <= 128.
//
// Numbers.  An fp32 operand x enters as x * 2^e = hi + lo, two fp16 numbers
// (hi rounded to nearest, lo the rest), with one exponent e per 64 rows that
// brings their largest magnitude into [2^14, 2^15); a product is hi*lo +
// lo*hi + hi*hi into fp32, and the softmax threads take the exponents off
// with the factor that they multiply by anyway.  An operand is good to 2^-22
// of its value, and absolutely to 2^-40 of its tile's largest.  The weights
// that meet the second operand (w, ds) are scaled per row: w by a constant,
// ds by an exponent of its own for each row and tile.  Every tile's product
// is added into fp32 registers with rounding to nearest, since the tensor
// core's accumulation truncates.
//
// split_kernel writes the operands once into the workspace, as the shared
// memory images that the products read: per tensor, slice and 64 rows, hi
// and lo as [64 rows][128 bytes] under the 128-byte swizzle (one such panel
// per 64 columns of head_dim, zeros behind it).  One image serves as K-major
// operand (scores) and as MN-major operand (sums over rows), so a tile needs
// one plain bulk copy per operand and no warp of the product kernels splits
// anything.  Rows at or past valid_len are zeros, so nothing there is ever
// multiplied.  1 / l goes into the rows of dout and into delta = dout . out:
// with g_i = dout_i / l_i and w_ij = 2^(x_ij - m_i) <= 1,
//   dv_j = sum_i w_ij g_i,   ds_ij = w_ij (g_i . v_j - g_i . out_i),
// so no product multiplies by it, and the exponent's argument stays a small
// difference (m and log2(l) in one fp32 offset cost 6e-7 of every p).
//
// A CTA computes one 128-row tile of one output; with the rows R, the
// columns C (64 per step) and the second operand X of its kind:
//   kForward: R = q,      C = k,  out  = softmax(R C^T) v
//   kDv:      R = k,      C = q,  dv   = W^T g
//   kDq:      R = q, g    C = k, v  dq = dS k,   dS = W * (g v^T - delta)
//   kDk:      R = k, v    C = q, g  dk = dS^T q
// 7 products where a single pass over the pairs would take 5, but every sum
// stays in its own CTA: no atomics, the same bits on every run.  Per 128x64
// tile and kind: 12 MMAs (M 128, N 64, K 16) per product, ~32 cycles each.
//
// Two CTAs share an SM (head_dim <= 64: 256 tensor-memory columns each; one
// CTA of 512 columns above), so one's softmax runs beside the other's
// products and its start and end beside the other's middle.  Within a CTA
// the steps are serial, except that kForward and kDv compute the next scores
// during the softmax (two score buffers).
//
// Roles (320 threads): warps 0-7 the rows (TMEM lane = row), warps 0-3 the
// first and 4-7 the second half of the columns of the scores and of the
// output; what a row's two threads share (its maximum) passes through shared
// memory at a barrier of their two warps.  Warp 8 issues the MMAs, warp 9 the
// bulk copies; both run their loops on the whole warp and issue from one
// lane.  With one thread per row (192 threads) the softmax's own latencies
// set the pace: 3.4k cycles per tile and 31% of the issue slots used.
//
// Tensor memory, columns (P = panels): rows' operands (hi 32 P, lo 32 P,
// twice for kDq and kDk), then scores: kForward and kDv two buffers of 64 and
// the partial of 64 P; kDq and kDk S (64), dP (64) and the partial, which for
// P = 1 takes dP's place once that has been read.  The weights overwrite
// their scores: k-step s (16 columns) has its hi part in columns 32 (s / 2) +
// 8 (s % 2) and lo 16 further.
//
// Every wait is bounded, as in the forward kernels.
#pragma once

#include <cuda_fp16.h>

#include "tc16_ws.cuh"
#include "train_common.cuh"

namespace raya {
namespace train {

constexpr int kTileRows = 128, kTileCols = 64;
constexpr int kTcThreads = 320;
constexpr int kRowThreadsTc = 256;
constexpr int kIssueWarp = 8, kCopyWarp = 9;
constexpr int kPairBarrier = 1, kRowBarrier = 5;  // named barriers: 1-4 the warps of the same rows, 5 all row warps
constexpr int kMaxStages = 3;
constexpr int kPanelBytes = 64 * 128;              // 64 rows of 64 fp16
constexpr int kVec = 192;                          // distances that a 128x64 tile covers (191, and one for alignment)
constexpr float kWeightLog2 = 14.f;                // kDv: w enters as w * 2^14, so that small ones keep their bits
constexpr float kRescale = 8.f, kForwardLog2 = 7.f;  // kForward: p <= 2^8 of the kept maximum, times 2^7

enum TcKind { kForward = 0, kDq = 1, kDk = 2, kDv = 3 };
enum { kImgQ = 0, kImgK = 1, kImgV = 2, kImgG = 3 };

// What the tensor-core kernels read besides TrainArgs.  The workspace holds
// one chunk of slices at a time: images, exponents and row values are
// indexed from slice0.
struct TcArgs {
  TrainArgs t;
  uint8_t* img[4];     // [chunk slices][tiles][2 P panels]: q, k, v, dout
  int4* exps;          // [chunk slices][tiles]: their exponents
  float* rows;         // [chunk slices][tiles][2][64]: m * log2(e) (inf: no key), and delta / l
  int tiles;           // 64-row tiles per slice (even)
  long long slice0;
  int stages;
};

__device__ __forceinline__ int valid_of(const AttnArgs& a, long long bh) {
  const int v = a.valid_len ? a.valid_len[bh / a.heads] : a.seq;
  return v < 0 ? 0 : (v > a.seq ? a.seq : v);
}

// 64 rows of one tensor into their image.  256 threads: 16 lanes take a row's
// 64 columns of a panel (16-byte loads, 8-byte stores), 16 rows at a time.
// blockIdx.y: the tensor.  Bound by HBM: 4 bytes read and 4 written per
// element (dout: 8 read).
template <int P>
__global__ void __launch_bounds__(256) split_kernel(const __grid_constant__ TcArgs c) {
  __shared__ uint32_t red[8];
  const AttnArgs& a = c.t.a;
  const int tid = threadIdx.x, which = blockIdx.y, d = a.head_dim;
  const long long local = blockIdx.x / static_cast<unsigned>(c.tiles), bh = c.slice0 + local;
  const int tile = static_cast<int>(blockIdx.x - local * c.tiles);
  const int valid = valid_of(a, bh);
  const int r0 = tile * 64;
  if (r0 >= (valid + 127) / 128 * 128) return;  // no 128-row tile reads it
  const float* src = which == kImgQ ? a.q : which == kImgK ? a.k : which == kImgV ? a.v : c.t.dout;
  src += static_cast<size_t>(bh) * a.seq * d;
  const float* out = a.out + static_cast<size_t>(bh) * a.seq * d;
  const int c4 = (tid & 15) * 4, r = tid >> 4;
  float4 x[4][P];
  float big = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = r0 + r + 16 * i;
    float m2 = 0.f, linv = 0.f, dot = 0.f;
    if (which == kImgG && row < valid) row_stats(c.t.stats[static_cast<size_t>(bh) * a.seq + row], m2, linv);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int col = 64 * p + c4;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < valid && col < d) {
        y = *reinterpret_cast<const float4*>(src + static_cast<size_t>(row) * d + col);
        if (which == kImgG) {
          y = make_float4(y.x * linv, y.y * linv, y.z * linv, y.w * linv);
          const float4 o = *reinterpret_cast<const float4*>(out + static_cast<size_t>(row) * d + col);
          dot = fmaf(y.x, o.x, fmaf(y.y, o.y, fmaf(y.z, o.z, fmaf(y.w, o.w, dot))));
        }
      }
      x[i][p] = y;
      // Infinities and NaN stay out of the exponent: they spoil their own products only.
      const float m = fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w)));
      if (m < INFINITY) big = fmaxf(big, m);
    }
    if (which == kImgG) {
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
      if ((tid & 15) == 0) {
        float* rows = c.rows + (local * c.tiles + tile) * 128;
        rows[r + 16 * i] = linv != 0.f ? m2 : INFINITY;  // 2^(x - inf) = 0: no key, or past valid_len
        rows[64 + r + 16 * i] = dot;
      }
    }
  }
  const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(big));
  if ((tid & 31) == 0) red[tid >> 5] = bits;
  __syncthreads();
  uint32_t most = red[0];
#pragma unroll
  for (int w = 1; w < 8; ++w) most = max(most, red[w]);
  const int e = tc16::scale_exp(most);
  const float sc = tc16::pow2(e);
  if (tid == 0) reinterpret_cast<int*>(c.exps + local * c.tiles + tile)[which] = e;
  uint8_t* img = c.img[which] + (local * c.tiles + tile) * (2ll * P * kPanelBytes);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rr = r + 16 * i;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const float v[4] = {x[i][p].x * sc, x[i][p].y * sc, x[i][p].z * sc, x[i][p].w * sc};
      uint32_t h[2], l[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const __half2 hh = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
        const float2 back = __half22float2(hh);
        h[k] = *reinterpret_cast<const uint32_t*>(&hh);
        l[k] = tc16::pack_f16x2(v[2 * k] - back.x, v[2 * k + 1] - back.y);
      }
      const uint32_t at = p * kPanelBytes + tc16::op_off(rr, c4 >> 3) + (c4 & 4) * 2;
      *reinterpret_cast<uint2*>(img + at) = make_uint2(h[0], h[1]);
      *reinterpret_cast<uint2*>(img + P * kPanelBytes + at) = make_uint2(l[0], l[1]);
    }
  }
}

// Shared memory behind the operand stages.
struct TcTail {
  float vec[kMaxStages][kVec];       // bias * log2(e) by distance
  float rows[kMaxStages][2 * 64];    // kDk, kDv: the columns' exponent and delta
  uint8_t ids[kMaxStages][kVec];     // kDq: buckets by distance
  int exps[kMaxStages][4];           // exponents of the columns' 64 rows, by tensor
  float red[2][2][kTileRows];        // [tile parity][half]: what a row's threads exchange
  uint64_t full[kMaxStages], freed[kMaxStages];
  uint64_t s_full[2], w_ready[2], part_full, part_free, a_ready;
  uint32_t tmem_base;
  int abort_flag;
};

template <int P>
constexpr size_t stage_bytes() { return 2ull * 2 * P * kPanelBytes; }
template <int P>
constexpr size_t tc_smem(int stages, int buckets) {
  return 1024 + stages * stage_bytes<P>() + sizeof(TcTail) + static_cast<size_t>(buckets) * kRowThreadsTc * sizeof(float);
}
// head_dim <= 64: at most half of an SM's shared memory, and more than a
// third, so that exactly two CTAs (2 x 256 tensor-memory columns) share it.
constexpr size_t kHalfSm = (233472 - 2 * 1024) / 2, kWholeCta = 232448;
constexpr size_t kThirdSm = 233472 / 3;
static_assert(tc_smem<1>(3, 0) <= kHalfSm, "two CTAs per SM");
static_assert(tc_smem<1>(2, kMaxBuckets) <= kWholeCta && tc_smem<2>(2, kMaxBuckets) <= kWholeCta, "shared memory of a block");

// A product of scales that would be infinite, as the largest float: 0 times it is 0.
__device__ __forceinline__ float finite(float x) { return fmaxf(fminf(x, 3.4028235e38f), -3.4028235e38f); }

// 128 bytes of an operand's row r (64 fp16 of one panel) as 32 words, from
// its image.  Straight from global memory: each row is read once, a whole
// line per panel and half.
__device__ __forceinline__ void load_row(const uint8_t* panel, int r, uint32_t* w) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint4 x = *reinterpret_cast<const uint4*>(panel + tc16::op_off(r, k));
    w[4 * k] = x.x;
    w[4 * k + 1] = x.y;
    w[4 * k + 2] = x.z;
    w[4 * k + 3] = x.w;
  }
}

// Weights w[32] (fp32, already scaled) as fp16 hi and lo over their scores.
__device__ __forceinline__ void store_weights(uint32_t taddr, const float* w) {
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    uint32_t h[8], l[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) tc16::split2(w[16 * s + 2 * k], w[16 * s + 2 * k + 1], h[k], l[k]);
    tc16::tmem_st8u(taddr + 8 * s, h);
    tc16::tmem_st8u(taddr + 8 * s + 16, l);
  }
}

// 32 scores in place: s * mult (+ bias), -inf outside [lo, hi).
template <bool BIAS, int STEP>
__device__ __forceinline__ void mask_scores(float* s, float mult, const float* vec, int lo, int hi, bool inside) {
#pragma unroll
  for (int i = 0; i < 32; ++i) s[i] = BIAS ? fmaf(s[i], mult, vec[STEP * i]) : s[i] * mult;
  if (!inside) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < lo || i >= hi) s[i] = -INFINITY;
  }
}

template <int KIND, int P, bool BIAS>
__device__ void run_tile(const TcArgs& c, long long local, int tile128, unsigned char* smem, int part_index) {
  using namespace tc32;
  constexpr bool kScores2 = KIND == kDq || KIND == kDk;      // S and dP, serial
  constexpr bool kByKey = KIND == kDk || KIND == kDv;        // rows are keys, columns queries
  constexpr bool kShared = KIND != kDv;                      // a row's threads share a maximum
  constexpr uint32_t kCols = 256 * P;
  constexpr uint32_t kColA2 = 64 * P;
  constexpr uint32_t kColS = kScores2 ? 128 * P : 64 * P;
  constexpr uint32_t kColS2 = kColS + 64;                    // dP, or the second score buffer
  constexpr uint32_t kColPart = kScores2 ? (P == 1 ? kColS2 : kColS2 + 64) : kColS2 + 64;
  static_assert(kColPart + 64 * P <= kCols, "tensor memory");
  constexpr int kB1 = kByKey ? kImgQ : kImgK, kB2 = kByKey ? kImgG : kImgV;  // the columns' operands
  constexpr int kA1 = kByKey ? kImgK : kImgQ, kA2 = kByKey ? kImgV : kImgG;  // the rows'
  constexpr uint32_t kOp = 2 * P * kPanelBytes;
  constexpr int kOutCols = 32 * P;                           // output columns of a thread

  const AttnArgs& a = c.t.a;
  const int tid = threadIdx.x, warp = tid >> 5;
  const long long bh = c.slice0 + local;
  const int valid = valid_of(a, bh);
  const int r0 = tile128 * kTileRows, d = a.head_dim;
  float* outp = KIND == kForward ? a.out : KIND == kDq ? c.t.dq : KIND == kDk ? c.t.dk : c.t.dv;
  const bool with_grad = KIND == kDq && c.t.part != nullptr;
  float* partial = with_grad ? c.t.part + (static_cast<size_t>(bh) * c.t.parts + part_index) * c.t.buckets : nullptr;

  int lo = 0, hi = 0, unused;
  if (r0 < valid) {
    key_range(a, r0, valid, lo, unused);
    key_range(a, min(r0 + kTileRows, valid) - 1, valid, unused, hi);
  }
  const int t0 = lo / kTileCols, n = hi > lo ? (hi + kTileCols - 1) / kTileCols - t0 : 0;
  if (n == 0) {  // padding only
    const int rows = min(kTileRows, a.seq - r0);
    float* o = outp + (static_cast<size_t>(bh) * a.seq + r0) * d;
    for (int i = tid; i < rows * d / 4; i += kTcThreads) st_stream(o + 4 * i, make_float4(0.f, 0.f, 0.f, 0.f));
    if (KIND == kForward && c.t.stats_out && tid < rows)
      c.t.stats_out[static_cast<size_t>(bh) * a.seq + r0 + tid] = make_float2(-INFINITY, 0.f);
    if (with_grad && tid < c.t.buckets) partial[tid] = 0.f;
    return;
  }

  TcTail& sm = *reinterpret_cast<TcTail*>(smem + c.stages * stage_bytes<P>());
  float* acc = reinterpret_cast<float*>(&sm + 1);  // with_grad: [buckets][kRowThreadsTc]
  const int stages = c.stages;
  const long long tile_base = local * c.tiles;

  // Copies the operands and values of step g into its stage (one lane).
  auto copy_stage = [&](int g) {
    const int st = g % stages, c0 = (t0 + g) * kTileCols;
    const long long tile = tile_base + t0 + g;
    const int head = static_cast<int>(bh % a.heads);
    // The tile's first distance j - i: rows' i from r0, or columns' i from c0.
    const int rel = kByKey ? r0 - c0 - 64 : c0 - r0 - 128;
    unsigned char* op = smem + st * stage_bytes<P>();
    mbar_arrive_expect_tx(&sm.full[st], 2 * kOp + 16u + (BIAS ? kVec * 4u : 0u) + (kByKey ? 512u : 0u) +
                                            (with_grad ? kVec : 0u));
    tma_load_1d(op, c.img[kB1] + tile * static_cast<long long>(kOp), kOp, &sm.full[st]);
    tma_load_1d(op + kOp, c.img[kB2] + tile * static_cast<long long>(kOp), kOp, &sm.full[st]);
    tma_load_1d(sm.exps[st], c.exps + tile, 16u, &sm.full[st]);
    if constexpr (BIAS)
      tma_load_1d(sm.vec[st], c.t.rel_bias + (2ll * head + 1) * c.t.rel_half + rel, kVec * 4u, &sm.full[st]);
    if (with_grad) tma_load_1d(sm.ids[st], c.t.rel_id + c.t.rel_half + rel, kVec, &sm.full[st]);
    if constexpr (kByKey) tma_load_1d(sm.rows[st], c.rows + tile * 128, 512u, &sm.full[st]);
  };

  // Before the CTA's first barrier: the copy warp fills the stages, the
  // issuing warp takes tensor memory, and the row threads load their rows
  // (first halves of the row threads: the first operand, or its hi parts).
  constexpr int kParts = kScores2 ? 2 * P : P;  // 32-word pieces of this thread
  uint32_t arow[kParts][32];
  const int half = warp >> 2, rt = tid & 127;
  int4 ae = make_int4(0, 0, 0, 0);
  if (warp < 8) {
    const int which = kScores2 && half ? kA2 : kA1;
    const uint8_t* img = c.img[which] + (tile_base + 2 * tile128 + (rt >> 6)) * static_cast<long long>(kOp) +
                         (kScores2 ? 0 : half * P * kPanelBytes);
#pragma unroll
    for (int p = 0; p < kParts; ++p) load_row(img + p * kPanelBytes, rt & 63, arow[p]);
    ae = c.exps[tile_base + 2 * tile128 + (rt >> 6)];
  } else if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sm.tmem_base)),
                 "r"(kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (tc16::lane_is_first(tid)) {
    for (int s = 0; s < kMaxStages; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.freed[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&sm.s_full[s], 1);
      mbar_init(&sm.w_ready[s], kRowThreadsTc);
    }
    mbar_init(&sm.part_full, 1);
    mbar_init(&sm.part_free, kRowThreadsTc);
    mbar_init(&sm.a_ready, kRowThreadsTc);
    sm.abort_flag = 0;
    fence_mbar_init();
    for (int g = 0; g < min(n, stages); ++g) copy_stage(g);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  volatile int* abort_flag = &sm.abort_flag;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return mbar_wait_bounded(bar, parity & 1u, abort_flag, a.status, a.timeout_cycles);
  };
  // A bounded wait whose outcome is the same on every lane of the warp.
  auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)); };
  // Read after the roles, by the warps that set them: the last copies and the last commit in flight.
  int last_g = min(n, stages) - 1;
  uint64_t* last_commit = nullptr;
  uint32_t last_parity = 0;

  if (warp < 8) {
    // ---------------- half a row per thread ----------------
    const uint32_t lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
#pragma unroll
    for (int p = 0; p < kParts; ++p)
      tmem_st32(lane + (kScores2 ? half * kColA2 : half * 32 * P) + 32 * p, reinterpret_cast<const float*>(arow[p]));
    tmem_wait_st();
    tc_fence_before();
    mbar_arrive(&sm.a_ready);

    const int row = r0 + rt;
    const int ea1 = kByKey ? ae.y : ae.x, ea2 = kByKey ? ae.z : ae.w;
    const float qmul = a.qscale * tc16::pow2(-ea1), unit1 = tc16::pow2(-ea2);
    float my_off = 0.f, my_delta = 0.f;
    if constexpr (KIND == kDq) {
      const float* mine = c.rows + (tile_base + 2 * tile128 + (rt >> 6)) * 128 + (rt & 63);
      my_off = mine[0];
      my_delta = mine[64];
    }
    if (with_grad)
      for (int b = 0; b < c.t.buckets; ++b) acc[b * kRowThreadsTc + tid] = 0.f;
    int rlo = 0, rhi = 0;
    key_range(a, min(row, valid - 1), valid, rlo, rhi);

    // Where the thread's first column finds its distance: j - i relative to
    // the tile's first one (kByKey: i runs with the column, so backwards).
    constexpr int kStep = kByKey ? -1 : 1;
    const int vec_at = (kByKey ? rt + 64 : 128 - rt) + kStep * 32 * half;
    float o[kOutCols];
#pragma unroll
    for (int i = 0; i < kOutCols; ++i) o[i] = 0.f;
    float m_used = -INFINITY, m_true = -INFINITY, lsum = 0.f;
    bool ok = true;      // the same on every lane of the warp
    float factor = 0.f;  // of the partial that is in flight

    // o += partial of tile g * factor, and the partial's columns are free.
    auto add_partial = [&](int g) {
      if (!warp_wait(&sm.part_full, g)) return false;
      tc_fence_after();
      const float2 f2 = make_float2(factor, factor);
#pragma unroll
      for (int q = 0; q < 2 * P; ++q) {
        float x[16];
        tc16::tmem_ld16(lane + kColPart + kOutCols * half + 16 * q, x);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float2 r = __ffma2_rn(make_float2(x[i], x[i + 1]), f2, make_float2(o[16 * q + i], o[16 * q + i + 1]));
          o[16 * q + i] = r.x;
          o[16 * q + i + 1] = r.y;
        }
      }
      tc_fence_before();
      mbar_arrive(&sm.part_free);
      return true;
    };
    // The larger of the row's two values x; false if either thread's warp gave up.
    auto share_max = [&](int g, float& x) {
      sm.red[g & 1][half][rt] = x;
      if (bar_any(kPairBarrier + (warp & 3), 64, !ok)) return false;
      x = fmaxf(x, sm.red[g & 1][half ^ 1][rt]);
      return true;
    };

    for (int g = 0; g < n; ++g) {
      const int st = g % stages, c0 = (t0 + g) * kTileCols + 32 * half;
      const int sb = kScores2 ? 0 : g & 1;
      if (ok) ok = warp_wait(&sm.full[st], g / stages) && warp_wait(&sm.s_full[sb], kScores2 ? g : g >> 1);
      if (!kShared && !ok) break;
      tc_fence_after();
      const uint32_t scol = lane + kColS + 64 * sb + 32 * half;
      const int e1 = sm.exps[st][kB1], e2 = sm.exps[st][kB2];
      const int mlo = rlo - c0, mhi = rhi - c0;
      float s[32];
      if (ok) {
        const bool inside = __all_sync(0xffffffffu, mlo <= 0 && mhi >= 32);
        tmem_ld32(scol, s);
        mask_scores<BIAS, kStep>(s, finite(qmul * tc16::pow2(-e1)), &sm.vec[st][vec_at], mlo, mhi, inside);
      }

      if constexpr (KIND == kForward) {
        float mx = -INFINITY;
        if (ok) {
#pragma unroll
          for (int i = 0; i < 32; i += 2) mx = fmax3(mx, s[i], s[i + 1]);
        }
        if (!share_max(g, mx)) { ok = false; break; }
        float alpha = 1.f;
        m_true = fmaxf(m_true, mx);
        if (mx > m_used + kRescale) {
          alpha = ex2(m_used - mx);
          m_used = mx;
        }
        const float base = (m_used == -INFINITY ? 0.f : m_used) - kForwardLog2;
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          s[i] = ex2(s[i] - base);
          s[i + 1] = ex2(s[i + 1] - base);
          sum = __fadd2_rn(sum, make_float2(s[i], s[i + 1]));
        }
        lsum = fmaf(lsum, alpha, sum.x + sum.y);
        store_weights(scol, s);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&sm.w_ready[sb]);
        if (g > 0) {
          ok = add_partial(g - 1);
          if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
            for (int i = 0; i < kOutCols; ++i) o[i] *= alpha;
          }
        }
        factor = tc16::pow2(-e2);
      } else if constexpr (KIND == kDv) {
        const float* off = sm.rows[st] + 32 * half;
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 f = *reinterpret_cast<const float4*>(off + i);
          s[i] = ex2(s[i] - f.x + kWeightLog2);
          s[i + 1] = ex2(s[i + 1] - f.y + kWeightLog2);
          s[i + 2] = ex2(s[i + 2] - f.z + kWeightLog2);
          s[i + 3] = ex2(s[i + 3] - f.w + kWeightLog2);
        }
        store_weights(scol, s);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&sm.w_ready[sb]);
        if (g > 0) ok = add_partial(g - 1);
        factor = tc16::pow2(-e2) * 6.103515625e-05f;  // 2^-14
      } else {
        // ds = w (dP - delta), then an exponent for the row: its largest |ds| to [2^14, 2^15)
        float big = 0.f;
        if (ok) {
          const float unit = finite(unit1 * tc16::pow2(-e2));
          const float* off = sm.rows[st] + 32 * half;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float dp[16];
            tc16::tmem_ld16(lane + kColS2 + 32 * half + 16 * q, dp);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int k = 16 * q + i;
              const float w = ex2(s[k] - (KIND == kDk ? off[k] : my_off));
              s[k] = w * fmaf(dp[i], unit, -(KIND == kDk ? off[64 + k] : my_delta));
            }
#pragma unroll
            for (int i = 0; i < 16; i += 2) big = fmax3(big, fabsf(s[16 * q + i]), fabsf(s[16 * q + i + 1]));
          }
        }
        if (!share_max(g, big)) { ok = false; break; }
        const int e = tc16::scale_exp(__float_as_uint(big));
        if (with_grad) {
          // This thread's column of acc: runs of equal buckets along the row.
          const uint8_t* ids = &sm.ids[st][vec_at];
          const int first = ids[0], last = ids[31];
          if (__all_sync(0xffffffffu, first == last)) {  // ends equal: one bucket
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) sum += s[i];
            acc[first * kRowThreadsTc + tid] += sum;
          } else {
            int cur = first;
            float run = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const int id = ids[i];
              if (id != cur) {
                acc[cur * kRowThreadsTc + tid] += run;
                run = 0.f;
                cur = id;
              }
              run += s[i];
            }
            acc[cur * kRowThreadsTc + tid] += run;
          }
          __syncwarp();  // the lanes' runs end at different columns
        }
        const float up = tc16::pow2(e);
#pragma unroll
        for (int i = 0; i < 32; ++i) s[i] *= up;
        store_weights(scol, s);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&sm.w_ready[sb]);
        factor = finite(tc16::pow2(-e) * tc16::pow2(-e1));
        ok = add_partial(g);
      }
    }
    if constexpr (!kScores2)
      if (ok) ok = add_partial(n - 1);
    float f = KIND == kDv ? 1.f : c.t.scale;
    if constexpr (KIND == kForward) {  // the row's sum: first half + second half
      sm.red[0][half][rt] = lsum;  // the last exchange is read: part_full follows both threads' w_ready
      bar_named(kRowBarrier, kRowThreadsTc);
      lsum = sm.red[0][0][rt] + sm.red[0][1][rt];
      f = lsum > 0.f ? 1.0f / lsum : lsum != lsum ? lsum : 0.f;
      if (ok && c.t.stats_out && half == 0 && row < a.seq)
        c.t.stats_out[static_cast<size_t>(bh) * a.seq + row] =
            row < valid ? make_stats(m_true, (m_used == -INFINITY ? 0.f : m_used) - kForwardLog2, lsum)
                        : make_float2(-INFINITY, 0.f);
      __syncwarp();
    }
    // The warp's rows through shared memory (the stages are idle: every copy
    // and product is complete), so that eight lanes store 128 bytes of a row.
    if (ok) {
      constexpr int kPitch = 64 * P + 4;  // 16-byte accesses of 8 rows or of one row meet no bank twice
      static_assert(kTileRows * kPitch * 4 <= 2 * stage_bytes<P>(), "row staging");
      float* stage = reinterpret_cast<float*>(smem) + (warp & 3) * 32 * kPitch + kOutCols * half;
      const bool live = row < valid;
#pragma unroll
      for (int i = 0; i < kOutCols; i += 4)
        *reinterpret_cast<float4*>(stage + (tid & 31) * kPitch + i) =
            live ? make_float4(o[i] * f, o[i + 1] * f, o[i + 2] * f, o[i + 3] * f) : make_float4(0.f, 0.f, 0.f, 0.f);
      __syncwarp();
      const int wr0 = r0 + (warp & 3) * 32, wrows = min(32, a.seq - wr0);
      float* dst = outp + (static_cast<size_t>(bh) * a.seq + wr0) * d + kOutCols * half;
      constexpr int kLanes = kOutCols / 4;  // lanes of a row
      const int col = (tid % kLanes) * 4;
#pragma unroll
      for (int i = 0; i < kLanes; ++i) {
        const int r = i * (32 / kLanes) + (tid & 31) / kLanes;
        if (r < wrows && kOutCols * half + col < d)
          st_stream(dst + static_cast<size_t>(r) * d + col, *reinterpret_cast<const float4*>(stage + r * kPitch + col));
      }
    }
    __syncwarp();
    if (with_grad) {
      // The threads' columns, bucket by bucket, in a fixed order.
      bar_named(kRowBarrier, kRowThreadsTc);
      for (int b = warp; b < c.t.buckets; b += 8) {
        float x = 0.f;
        for (int u = tid & 31; u < kRowThreadsTc; u += 32) x += acc[b * kRowThreadsTc + u];
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
        if ((tid & 31) == 0) partial[b] = x;
      }
    }
  } else if (warp == kIssueWarp) {
    // ---------------- MMA issue ----------------
    bool ok = warp_wait(&sm.a_ready, 0);
    if (ok) tc_fence_after();
    auto commit = [&](uint64_t* bar, uint32_t parity) {
      mma_commit_e(bar);
      last_commit = bar;
      last_parity = parity & 1u;
    };
    const uint32_t ops = smem_addr(smem);
    auto operand = [&](int g, int which) {
      return ops + static_cast<uint32_t>((g % stages) * stage_bytes<P>() + which * (2 * P * kPanelBytes));
    };
    // rows x columns^T into dcol: the small products first
    auto scores = [&](uint32_t dcol, uint32_t acol, uint32_t b) {
      const uint32_t ah = tmem + acol, al = ah + 32 * P, bl = b + P * kPanelBytes;
      uint32_t add = 0;
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          tc16::mma_f16_ts_e<tc16::kIdescQK>(tmem + dcol, ah + 32 * p + 8 * k, tc16::b_desc(bl + p * kPanelBytes, k), add);
          add = 1;
        }
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          tc16::mma_f16_ts_e<tc16::kIdescQK>(tmem + dcol, al + 32 * p + 8 * k, tc16::b_desc(b + p * kPanelBytes, k), 1u);
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          tc16::mma_f16_ts_e<tc16::kIdescQK>(tmem + dcol, ah + 32 * p + 8 * k, tc16::b_desc(b + p * kPanelBytes, k), 1u);
    };
    // weights x operand (its 64 rows are the inner dimension) into the partial
    auto sums = [&](uint32_t wcol, uint32_t b) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const uint32_t dcol = tmem + kColPart + 64 * p, bhi = b + p * kPanelBytes, blo = bhi + P * kPanelBytes;
        auto hi_at = [&](int k) { return tmem + wcol + 32 * (k >> 1) + 8 * (k & 1); };
#pragma unroll
        for (int k = 0; k < 4; ++k)
          tc16::mma_f16_ts_e<tc16::kIdescPV>(dcol, hi_at(k), tc16::v_desc(blo, k), k > 0 ? 1u : 0u);
#pragma unroll
        for (int k = 0; k < 4; ++k) tc16::mma_f16_ts_e<tc16::kIdescPV>(dcol, hi_at(k) + 16, tc16::v_desc(bhi, k), 1u);
#pragma unroll
        for (int k = 0; k < 4; ++k) tc16::mma_f16_ts_e<tc16::kIdescPV>(dcol, hi_at(k), tc16::v_desc(bhi, k), 1u);
      }
    };
    if constexpr (kScores2) {
      for (int g = 0; ok && g < n; ++g) {
        ok = warp_wait(&sm.full[g % stages], g / stages);
        // The row threads have added the last partial, so its columns (dP's, for P = 1) and the weights' are free.
        if (ok && g > 0) ok = warp_wait(&sm.part_free, g - 1);
        if (!ok) break;
        tc_fence_after();
        scores(kColS, 0, operand(g, 0));
        scores(kColS2, kColA2, operand(g, 1));
        commit(&sm.s_full[0], g);
        ok = warp_wait(&sm.w_ready[0], g);
        if (!ok) break;
        tc_fence_after();
        sums(kColS, operand(g, 0));
        commit(&sm.part_full, g);
        if (g + stages < n) commit(&sm.freed[g % stages], g / stages);
      }
    } else {
      if (ok) ok = warp_wait(&sm.full[0], 0);
      if (ok) {
        tc_fence_after();
        scores(kColS, 0, operand(0, 0));
        commit(&sm.s_full[0], 0);
      }
      for (int g = 0; ok && g < n; ++g) {
        if (g + 1 < n) {
          // The other score buffer held the weights of tile g - 1: its product is complete.
          if (g > 0) ok = warp_wait(&sm.part_full, g - 1);
          if (ok) ok = warp_wait(&sm.full[(g + 1) % stages], (g + 1) / stages);
          if (!ok) break;
          tc_fence_after();
          scores(kColS + 64 * ((g + 1) & 1), 0, operand(g + 1, 0));
          commit(&sm.s_full[(g + 1) & 1], (g + 1) >> 1);
        }
        ok = warp_wait(&sm.w_ready[g & 1], g >> 1);
        if (ok && g > 0) ok = warp_wait(&sm.part_free, g - 1);
        if (!ok) break;
        tc_fence_after();
        sums(kColS + 64 * (g & 1), operand(g, 1));
        commit(&sm.part_full, g);
        if (g + stages < n) commit(&sm.freed[g % stages], g / stages);
      }
    }
  } else {
    // ---------------- bulk copies (the first `stages` are on their way) ----------------
    for (int g = stages; g < n; ++g) {
      if (!warp_wait(&sm.freed[g % stages], g / stages - 1)) break;
      if (tc16::lane_is_first(tid)) {
        fence_proxy_async_smem();  // the row threads' reads of this stage, before the copies
        copy_stage(g);
      }
      last_g = g;
      __syncwarp();
    }
  }
  __syncwarp();

  // After a timeout, drain what is in flight (bounded) before tensor memory is freed and the CTA ends.
  tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0) {
    const long long t_end = clock64() + a.timeout_cycles;
    auto drain = [&](uint64_t* bar, uint32_t parity) {
      while (!mbar_try_wait(bar, parity & 1u) && clock64() < t_end) {
      }
    };
    if (tid == kCopyWarp * 32)
      for (int g = max(0, last_g - stages + 1); g <= last_g; ++g) drain(&sm.full[g % stages], g / stages);
    if (tid == kIssueWarp * 32 && last_commit) drain(last_commit, last_parity);
  }
  __syncthreads();
  if (warp == kIssueWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
  }
}

__device__ __forceinline__ unsigned char* aligned_smem(unsigned char* raw) {
  const uint32_t at = smem_addr(raw);
  return raw + (((at + 1023u) & ~1023u) - at);
}

// One CTA per 128-row tile of the chunk's slices.  A launch per kind: with
// the three gradients in one grid, CTAs of different kinds on an SM evicted
// one another's code from the instruction cache (4.0 of 17 stall cycles per
// instruction were instruction fetch).
template <int KIND, int P, bool BIAS>
__global__ void __launch_bounds__(kTcThreads, P == 1 ? 2 : 1) tc_train(const __grid_constant__ TcArgs c) {
  extern __shared__ unsigned char raw[];
  const unsigned tiles = static_cast<unsigned>(c.tiles) / 2, local = blockIdx.x / tiles;
  const int tile = static_cast<int>(blockIdx.x - local * tiles);
  run_tile<KIND, P, BIAS>(c, local, tile, aligned_smem(raw), tile);
}

}  // namespace train
}  // namespace raya
