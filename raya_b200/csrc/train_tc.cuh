// train_tc.cuh — the training operators on the tensor cores (sm_100a,
// tcgen05.mma kind::f16 in 3xFP16), head_dim <= 128.
//
// Numbers.  An fp32 operand x enters as x * 2^e = hi + lo, two fp16 numbers
// (hi rounded to nearest, lo the rest), with one exponent e per 64 rows that
// brings their largest magnitude into [2^14, 2^15); a product is hi*lo +
// lo*hi + hi*hi into fp32, and the softmax threads take the exponents off
// with the factor that they multiply by anyway.  An operand is good to 2^-22
// of its value, and absolutely to 2^-40 of its tile's largest.  The weights
// that meet the second operand (w, ds) are scaled too: w by a constant, ds by
// an exponent from a bound for each row and tile, and for dv and dk, where a
// key may have nothing but small ones, by a second exponent where the first
// would leave them to fp16's smallest steps.  Every tile's product
// is added into fp32 registers with rounding to nearest, since the tensor
// core's accumulation truncates.
//
// split_kernel writes the operands once into the workspace, as the shared
// memory images that the products read: per tensor, slice and 64 rows, hi
// and lo as [64 rows][128 bytes] under the 128-byte swizzle (one such panel
// per 64 columns of head_dim, zeros behind it).  One image serves as K-major
// operand (scores) and as MN-major operand (sums over rows), so a tile needs
// one plain bulk copy per operand and no warp of the product kernels splits
// anything but its weights (and, in the forward pass with head_dim <= 64, q,
// which only its own rows meet: a tensor less to write and read back, 10%).
// Rows at or past valid_len are zeros, so nothing there is ever multiplied.
// What is not finite stays in the products of its own row with every row of
// the tiles that see it.  1 / l goes into the rows of dout and into delta = dout . out:
// with g_i = dout_i / l_i and w_ij = 2^(x_ij - m_i) <= 1,
//   dv_j = sum_i w_ij g_i,   ds_ij = w_ij (g_i . v_j - g_i . out_i),
// so no product multiplies by it, and the exponent's argument stays a small
// difference (m and log2(l) in one fp32 offset cost 6e-7 of every p).
//
// A unit of work is one 128-row tile of one output; with the rows R, the
// columns C (64 per step) and the second operand of its kind:
//   kForward: R = q,      C = k,  out  = softmax(R C^T) v
//   kDv:      R = k,      C = q,  dv   = W^T g
//   kDq:      R = q, g    C = k, v  dq = dS k,   dS = W * (g v^T - delta)
//   kDk:      R = k, v    C = q, g  dk = dS^T q
// 7 products where a single pass over the pairs would take 5 (dk and dv in
// one CTA would need 384 columns of tensor memory and could not share an SM),
// but every sum stays in its own CTA: no atomics, the same bits on every run.
// Per 128x64 tile and kind: 12 MMAs (M 128, N 64, K 16) per product and
// panel, ~32 cycles each.
//
// Two CTAs share an SM (head_dim <= 64: 256 tensor-memory columns each; one
// CTA of 512 columns above), so one's softmax runs beside the other's
// products: 1.6 times one CTA's rate.  Within a CTA the steps follow one
// another, except that kForward and kDv compute the next scores during the
// softmax (two score buffers).  The CTAs are persistent and take units from a
// queue; the next unit's rows are on their way before the last tile of this.
//
// Roles (256 threads; 384 for two panels): warps 0-3 one row per thread (TMEM
// lane = row), for two panels warps 4-7 the second half of the columns of
// the scores and of the output (what a row's two threads share, its maximum,
// passes through shared memory).  Then one warp that issues the MMAs, one
// that takes the units and issues the bulk copies, and two that sum the
// table's gradient; the first two run their loops on the whole warp and issue
// from one lane.
//
// Tensor memory, columns (P = panels): rows' operands (hi 32 P, lo 32 P,
// twice for kDq and kDk), then scores: kForward and kDv two buffers of 64 and
// the partial of 64 P; kDq and kDk S (64), dP (64) and the partial, which for
// P = 1 takes dP's place once that has been read.  The weights overwrite
// their scores: k-step s (16 columns) has its hi part in columns 32 (s / 2) +
// 8 (s % 2) and lo 16 further.
//
// What bounds it.  The chain of a tile: scores, a round trip through the row
// threads (tensor memory to registers and back), the second product, its
// sum.  One CTA alone takes 3.5k cycles a tile (kForward), two on an SM 2.1k
// each tile of either, of which the tensor core works 37%, the issue slots
// 44%.  Taking two thirds of the MMAs out changed 8 to 17%, all exponentials 5%, the
// split of the weights 4%, the bulk copies nothing.  Measured and left: two
// threads per row (the same time with 30% more instructions), unrolled 64-column
// code (instruction fetch: 419 against 314 us), a grid of all three gradients
// (likewise), a workspace that stays in L2 (each chunk's tail costs more).
//
// Every wait is bounded, as in the forward kernels.
#pragma once

#include <cuda_fp16.h>

#include "tc16_ws.cuh"
#include "train_common.cuh"

namespace raya {
namespace train {

constexpr int kTileRows = 128, kTileCols = 64;
// Threads per row: one where two CTAs share an SM, two where one has it alone.
constexpr int kRowWarpsOf(int panels) { return 4 * panels; }
constexpr int tc_threads(int panels) { return 128 * panels + 128; }
// Registers (setmaxnreg): a row thread holds a row of scores next to a row of
// the output.  The shares add up to what the launch gives its threads: 256
// threads of 128 registers (two CTAs per SM), 384 of 168.
constexpr int row_regs(int panels) { return panels == 1 ? 192 : 208; }
constexpr int other_regs(int panels) { return panels == 1 ? 64 : 88; }
static_assert(row_regs(1) + other_regs(1) <= 2 * 128 && 2 * row_regs(2) + other_regs(2) <= 3 * 168, "register shares");
// Named barriers, which have no bound: between warps that leave together only.
// 1-4 the two warps of the same rows, 5 the table's.
constexpr int kPairBarrier = 1, kTableBarrier = 5;
constexpr int kStages = 2;
constexpr int kPanelBytes = 64 * 128;              // 64 rows of 64 fp16
constexpr int kVec = 192;                          // distances that a 128x64 tile covers (191, and one for alignment)
constexpr float kWeightScale = 16384.f;            // kDv: w <= 1 enters as w * 2^14, fp16's last power of two with room above it
constexpr float kSmallWeight = 0.25f;              // kDk, kDv: what is scaled once more where a row has nothing larger
constexpr int kRowValues = 3 * 64;                 // values per 64 rows of dout; kDk and kDv read the first two of each
constexpr float kRescale = 8.f, kForwardLog2 = 7.f;  // kForward: p <= 2^8 of the kept maximum, times 2^7

enum TcKind { kForward = 0, kDq = 1, kDk = 2, kDv = 3 };
enum { kImgQ = 0, kImgK = 1, kImgV = 2, kImgG = 3 };

// What goes with 64 rows of a slice's images: their exponents by tensor, and
// in units of these (2^e times the value) the longest row of v and of g; the
// largest |delta|.  Rows that are not finite do not count.
struct alignas(16) TileScale {
  int e[4];
  float v_norm, g_norm, delta, unused;
};

// What the tensor-core kernels read besides TrainArgs.  The workspace holds
// one chunk of slices at a time: images, exponents and row values are
// indexed from slice0.
struct TcArgs {
  TrainArgs t;
  uint8_t* img[4];     // [chunk slices][tiles][2 P panels]: q, k, v, dout
  TileScale* scales;   // [chunk slices][tiles]
  float* rows;         // [chunk slices][tiles][3][64]: m * log2(e) (inf: no key, no dout), delta = g . out, |g| 2^e
  const float* table;  // the bias, or nullptr
  float* vec;          // where it goes by distance (t.rel_bias)
  int tiles;           // 64-row tiles per slice (even)
  int first_image;     // kImgK where the forward kernel splits q itself, else kImgQ
  long long slice0;
  unsigned units;      // 128-row tiles of the chunk
  unsigned* next;      // [4] by kind: units handed out beyond the first one of each CTA; split_kernel clears them.
                       // Backward, [kForward]: 1 once kDq has seen split_kernel complete
  BucketBounds bounds;
  int far;             // the last bucket's first distance
  // With t.part, the table's gradient by distance:
  int slots;           // dist_slots(far)
  float* dist;         // [CTAs][8][slots] where shared memory does not hold them, or nullptr
};

__device__ __forceinline__ int valid_of(const AttnArgs& a, long long bh) {
  const int v = a.valid_len ? a.valid_len[static_cast<unsigned>(bh) / static_cast<unsigned>(a.heads)] : a.seq;  // bh < 2^31
  return v < 0 ? 0 : (v > a.seq ? a.seq : v);
}

// Two scaled values as fp16 hi (rounded to nearest) and lo (the rest).
__device__ __forceinline__ void split_near(float x, float y, uint32_t& h, uint32_t& l) {
  const __half2 hh = __floats2half2_rn(x, y);
  const float2 back = __half22float2(hh);
  h = *reinterpret_cast<const uint32_t*>(&hh);
  l = tc16::pack_f16x2(x - back.x, y - back.y);
}

// 64 rows of one tensor into their image.  256 threads: 16 lanes take a row's
// 64 columns of a panel (16-byte loads, 8-byte stores), 16 rows at a time.
// blockIdx.y: the tensor, and behind them the bias by distance.  Tiles of
// padding write the zeros of the results there instead.  Bound by HBM: 4 bytes
// read and 4 written per element (dout: 8 read), 96% of the copy rate forward
// (8 x 16 x 8192: 0.88 GB in 140 us), 88% backward (64 x 12 x 512, half of it
// valid: 0.67 GB in 116 us).  With four blocks on an SM, which the registers
// of all of dout's and out's loads at once allow, it was 176 and 131.
template <int P, bool BACK>
__global__ void __launch_bounds__(256, P == 1 ? (BACK ? 5 : 6) : 3) split_kernel(const __grid_constant__ TcArgs c) {
  __shared__ uint32_t red[8];
  __shared__ float norms[8], deltas[8];
  const AttnArgs& a = c.t.a;
  const int tid = threadIdx.x, which = c.first_image + blockIdx.y, d = a.head_dim;
  launch_dependents();
  if (which == 4 || (which == 3 && !BACK)) {
    rel_table(c.table, a.heads, c.t.buckets, c.t.rel_half, c.bounds, c.vec, nullptr, blockIdx.x * 256ll + tid,
              gridDim.x * 256ll);
    return;
  }
  const unsigned local = blockIdx.x / static_cast<unsigned>(c.tiles);
  const long long bh = c.slice0 + local;
  const int tile = static_cast<int>(blockIdx.x - local * static_cast<unsigned>(c.tiles));
  if (blockIdx.x == 0 && blockIdx.y == 0 && tid < 4) c.next[tid] = 0;
  const int valid = valid_of(a, bh);
  const int r0 = tile * 64;
  const size_t first = static_cast<size_t>(bh) * a.seq + r0;
  if (r0 >= (valid + 127) / 128 * 128) {  // no 128-row tile reads it: padding, whose results are zero
    float* o = nullptr;
    if (BACK)
      o = which == kImgQ ? c.t.dq : which == kImgK ? c.t.dk : which == kImgV ? c.t.dv : nullptr;
    else if (which == kImgV)
      o = a.out;
    const int rows = min(64, a.seq - r0);
    if (o)
      for (int i = tid; i < rows * d / 4; i += 256) st_stream(o + first * d + 4 * i, make_float4(0.f, 0.f, 0.f, 0.f));
    if (!BACK && which == kImgV && c.t.stats_out && tid < rows) c.t.stats_out[first + tid] = make_float2(-INFINITY, 0.f);
    if (c.t.part && which == kImgQ && tile % 2 == 0 && tid < c.t.buckets)
      c.t.part[(static_cast<size_t>(bh) * c.t.parts + tile / 2) * c.t.buckets + tid] = 0.f;
    return;
  }
  const float* __restrict__ src = (which == kImgQ ? a.q : which == kImgK ? a.k : which == kImgV ? a.v : c.t.dout) + first * d;
  const float* __restrict__ out = a.out + first * d;
  const bool grad = BACK && which == kImgG;
  const int c4 = (tid & 15) * 4, r = tid >> 4, live = valid - r0;  // rows below `live` are read
  float4 x[4][P];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int row = r + 16 * i, col = 64 * p + c4;
      x[i][p] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < live && col < d) x[i][p] = __ldcs(reinterpret_cast<const float4*>(src + static_cast<size_t>(row) * d + col));
    }
  float delta = 0.f;
  if (grad) {
#pragma unroll
    for (int half = 0; half < 4; half += 2) {  // two rows of out at a time, for a fifth block on the SM
      float4 y[2][P];
      float2 st[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = r + 16 * (half + i);
        st[i] = make_float2(0.f, 0.f);
        if (row < live) st[i] = __ldg(c.t.stats + first + row);
#pragma unroll
        for (int p = 0; p < P; ++p) {
          const int col = 64 * p + c4;
          y[i][p] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (row < live && col < d) y[i][p] = __ldcs(reinterpret_cast<const float4*>(out + static_cast<size_t>(row) * d + col));
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float m2, linv, dot = 0.f;
        row_stats(st[i], m2, linv);
#pragma unroll
        for (int p = 0; p < P; ++p) {
          float4& g = x[half + i][p];
          const float4 o = y[i][p];
          g = make_float4(g.x * linv, g.y * linv, g.z * linv, g.w * linv);
          dot = fmaf(g.x, o.x, fmaf(g.y, o.y, fmaf(g.z, o.z, fmaf(g.w, o.w, dot))));
        }
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
        if ((tid & 15) == 0) {
          float* rows = c.rows + (static_cast<size_t>(local) * c.tiles + tile) * kRowValues + r + 16 * (half + i);
          const float off = linv != 0.f ? m2 : INFINITY;  // 2^(x - inf) = 0: no key, or past valid_len
          rows[0] = off;
          rows[64] = dot;
        }
        if (fabsf(dot) < INFINITY) delta = fmaxf(delta, fabsf(dot));
      }
    }
  }
  float big = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int p = 0; p < P; ++p) {
      // Infinities and NaN stay out of the exponent: they spoil their own products only.
      const float4 g = x[i][p];
      const float m = fmaxf(fmaxf(fabsf(g.x), fabsf(g.y)), fmaxf(fabsf(g.z), fabsf(g.w)));
      if (m < INFINITY) big = fmaxf(big, m);
    }
  const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(big));
  if ((tid & 31) == 0) red[tid >> 5] = bits;
  __syncthreads();
  uint32_t most = red[0];
#pragma unroll
  for (int w = 1; w < 8; ++w) most = max(most, red[w]);
  const int e = tc16::scale_exp(most);
  const float sc = tc16::pow2(e);
  const size_t at_tile = static_cast<size_t>(local) * c.tiles + tile;
  if (tid == 0) c.scales[at_tile].e[which] = e;
  uint8_t* img = c.img[which] + at_tile * (2 * P * kPanelBytes);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const float4 g = x[i][p];
      uint32_t h[2], l[2];
      split_near(g.x * sc, g.y * sc, h[0], l[0]);
      split_near(g.z * sc, g.w * sc, h[1], l[1]);
      const uint32_t at = p * kPanelBytes + tc16::op_off(r + 16 * i, c4 >> 3) + (c4 & 4) * 2;
      *reinterpret_cast<uint2*>(img + at) = make_uint2(h[0], h[1]);
      *reinterpret_cast<uint2*>(img + P * kPanelBytes + at) = make_uint2(l[0], l[1]);
    }
  if (!BACK || which < kImgV) return;
  // The rows' lengths, for the bound on ds (kDq, kDk).
  float longest = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float square = 0.f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const float4 g = make_float4(x[i][p].x * sc, x[i][p].y * sc, x[i][p].z * sc, x[i][p].w * sc);
      square = fmaf(g.x, g.x, fmaf(g.y, g.y, fmaf(g.z, g.z, fmaf(g.w, g.w, square))));
    }
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) square += __shfl_xor_sync(0xffffffffu, square, off);
    const float norm = square < INFINITY ? sqrtf(square) : 0.f;
    longest = fmaxf(longest, norm);
    if (grad && (tid & 15) == 0) {
      float* rows = c.rows + at_tile * kRowValues + r + 16 * i;
      rows[128] = norm;
      // A row without a dout adds nothing to any gradient.  Its weights become 0
      // too, so that they do not hide how small those of the other rows are.
      if (square == 0.f) rows[0] = INFINITY;
    }
  }
  longest = fmaxf(longest, __shfl_xor_sync(0xffffffffu, longest, 16));
  delta = fmaxf(delta, __shfl_xor_sync(0xffffffffu, delta, 16));
  if ((tid & 31) == 0) {
    norms[tid >> 5] = longest;
    deltas[tid >> 5] = delta;
  }
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < 8; ++w) {
      longest = fmaxf(longest, norms[w]);
      delta = fmaxf(delta, deltas[w]);
    }
    TileScale& t = c.scales[at_tile];
    if (grad) {
      t.g_norm = longest;
      t.delta = delta;
    } else {
      t.v_norm = longest;
    }
  }
}

// One unit of work: a 128-row tile of one slice.
struct TcUnit {
  int local;   // slice within the chunk
  int valid, r0;
  int t0, n;   // 64-column tiles [t0, t0 + n) that its rows see; n = 0: padding only (not queued), -1: no more units
};

// Shared memory behind the operand stages.
constexpr int kQueue = 2;
template <int P>
struct alignas(16) TcTail {
  float vec[kStages][kVec];       // bias * log2(e) by distance
  float rows[kStages][128];       // kDk, kDv: the columns' exponents and delta
  TileScale scales[kStages];      // of the columns' 64 rows
  int flat[kStages];              // the tile's pairs all lie in one distance bucket
  float red[2][2][P == 2 ? kTileRows : 1];  // [tile parity][half]: what a row's threads exchange
  TcUnit unit[kQueue];            // the units that the copy warp has begun
  uint64_t u_full[kQueue], u_free[kQueue];
  uint64_t full[kStages], freed[kStages];
  uint64_t s_full[2], w_ready[2], part_full, part_free, a_ready;
  uint64_t rows_full[8];          // by row warp
  // The table's gradient: each row warp's blocks of ds in its buffer, and at a
  // unit's end each row's sums beyond the last bound on either side.
  uint64_t ds_ready[8], ds_free[8], far_ready, far_free;
  float2 far[4 * P][32];
  uint32_t tmem_base;
  int abort_flag;
};

template <int P>
constexpr size_t stage_bytes() { return 2ull * 2 * P * kPanelBytes; }
// Each row warp's buffer: two blocks of 32 rows x 128 bytes under the 128-byte
// swizzle.  The next unit's rows come in through it by bulk copies, the
// output leaves through it by tensor stores (which clip rows past seq and
// columns past head_dim), and neither holds the row threads up: with loads
// and stores of their own these took 5 to 7k of a unit's 30k cycles.  Whatever
// writes into the buffer (rows coming in, ds for the table's gradient, the
// output) first waits for the store that reads it.
constexpr int kBlockBytes = 32 * 128, kRowBuf = 2 * kBlockBytes;
template <int P>
constexpr size_t tc_smem() {
  return 1024 + kStages * stage_bytes<P>() + kRowWarpsOf(P) * kRowBuf + sizeof(TcTail<P>);
}
// head_dim <= 64: two CTAs (2 x 256 tensor-memory columns) share an SM and a
// third does not fit beside them.
constexpr size_t kHalfSm = (233472 - 2 * 1024) / 2, kWholeSm = 232448;
static_assert(tc_smem<1>() <= kHalfSm && tc_smem<1>() > 233472 / 3 && tc_smem<2>() <= kWholeSm, "CTAs per SM");

// A product of scales that would be infinite, as the largest float: 0 times it is 0.
__device__ __forceinline__ float finite(float x) { return fmaxf(fminf(x, 3.4028235e38f), -3.4028235e38f); }

// 2^e, of two factors: the sum of some exponents may be beyond one float's.
__device__ __forceinline__ float two_to(int e) {
  const int a = e >> 1, b = e - a;
  return tc16::pow2(max(-126, min(127, a))) * tc16::pow2(max(-126, min(127, b)));
}

// One tensor-map tile into shared memory, completing on `bar`; zeros outside the tensor.
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void prefetch_l2(const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
}

// 32 columns from each of two places of this thread's TMEM lane, both on the
// way at once (a round trip takes the row threads 200 cycles).  Loads and wait
// in one statement, so that no use can be scheduled between them.
__device__ __forceinline__ void tmem_ld32x2(uint32_t at0, float* v0, uint32_t at1, float* v1) {
  uint32_t a[32], b[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%65];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]), "=r"(a[8]), "=r"(a[9]), "=r"(a[10]), "=r"(a[11]), "=r"(a[12]), "=r"(a[13]), "=r"(a[14]), "=r"(a[15]), "=r"(a[16]), "=r"(a[17]), "=r"(a[18]), "=r"(a[19]), "=r"(a[20]), "=r"(a[21]), "=r"(a[22]), "=r"(a[23]), "=r"(a[24]), "=r"(a[25]), "=r"(a[26]), "=r"(a[27]), "=r"(a[28]), "=r"(a[29]), "=r"(a[30]), "=r"(a[31]),
        "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3]), "=r"(b[4]), "=r"(b[5]), "=r"(b[6]), "=r"(b[7]), "=r"(b[8]), "=r"(b[9]), "=r"(b[10]), "=r"(b[11]), "=r"(b[12]), "=r"(b[13]), "=r"(b[14]), "=r"(b[15]), "=r"(b[16]), "=r"(b[17]), "=r"(b[18]), "=r"(b[19]), "=r"(b[20]), "=r"(b[21]), "=r"(b[22]), "=r"(b[23]), "=r"(b[24]), "=r"(b[25]), "=r"(b[26]), "=r"(b[27]), "=r"(b[28]), "=r"(b[29]), "=r"(b[30]), "=r"(b[31])
      : "r"(at0), "r"(at1)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    v0[i] = __uint_as_float(a[i]);
    v1[i] = __uint_as_float(b[i]);
  }
}

// D (+)= A B over 64 of the inner dimension in split fp16, A from tensor memory:
// hi lo + lo hi + hi hi, the small products first, each in four k-steps of 16:
// A's steps A1, A2 and A3 columns behind the first, B's descriptors STEP
// apart.  As tc16::mma_f16_ts_e, but one statement: with a statement for each
// of the twelve, 47 cycles apart where the tensor core takes 32, the kernels
// took 2 to 4% longer.
template <uint32_t IDESC, int STEP, int A1, int A2, int A3>
__device__ __forceinline__ void mma12_ts_e(uint32_t d, uint32_t a_hi, uint32_t a_lo, uint64_t b_hi, uint64_t b_lo, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, t, e;\n\t.reg .b32 r;\n\t.reg .b32 h0, h1, h2, h3, l0, l1, l2, l3;\n\t"
      ".reg .b64 x0, x1, x2, x3, y0, y1, y2, y3;\n\t"
      "mov.b32 h0, %1;\n\t"
      "add.u32 h1, %1, %8;\n\t"
      "add.u32 h2, %1, %9;\n\t"
      "add.u32 h3, %1, %10;\n\t"
      "mov.b32 l0, %2;\n\t"
      "add.u32 l1, %2, %8;\n\t"
      "add.u32 l2, %2, %9;\n\t"
      "add.u32 l3, %2, %10;\n\t"
      "mov.b64 x0, %3;\n\t"
      "add.u64 x1, %3, 1 * %11;\n\t"
      "add.u64 x2, %3, 2 * %11;\n\t"
      "add.u64 x3, %3, 3 * %11;\n\t"
      "mov.b64 y0, %4;\n\t"
      "add.u64 y1, %4, 1 * %11;\n\t"
      "add.u64 y2, %4, 2 * %11;\n\t"
      "add.u64 y3, %4, 3 * %11;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "setp.eq.b32 t, %7, 0;\n\t"
      "elect.sync r|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [h0], y0, %5, {%7, %7, %7, %7}, p;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [h1], y1, %5, {%7, %7, %7, %7}, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [h2], y2, %5, {%7, %7, %7, %7}, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [h3], y3, %5, {%7, %7, %7, %7}, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [l0], x0, %5, {%7, %7, %7, %7}, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [l1], x1, %5, {%7, %7, %7, %7}, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [l2], x2, %5, {%7, %7, %7, %7}, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [l3], x3, %5, {%7, %7, %7, %7}, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [h0], x0, %5, {%7, %7, %7, %7}, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [h1], x1, %5, {%7, %7, %7, %7}, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [h2], x2, %5, {%7, %7, %7, %7}, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [h3], x3, %5, {%7, %7, %7, %7}, t;\n\t"
      "}" ::"r"(d),
      "r"(a_hi), "r"(a_lo), "l"(b_hi), "l"(b_lo), "n"(IDESC), "r"(accumulate), "r"(0u), "n"(A1), "n"(A2), "n"(A3), "n"(STEP)
      : "memory");
}

// One of the three products: four k-steps.
template <uint32_t IDESC, int STEP, int A1, int A2, int A3>
__device__ __forceinline__ void mma4_ts_e(uint32_t d, uint32_t a, uint64_t b, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, t, e;\n\t.reg .b32 r;\n\t.reg .b32 a1, a2, a3;\n\t.reg .b64 b1, b2, b3;\n\t"
      "add.u32 a1, %1, %6;\n\t"
      "add.u32 a2, %1, %7;\n\t"
      "add.u32 a3, %1, %8;\n\t"
      "add.u64 b1, %2, %9;\n\t"
      "add.u64 b2, %2, 2 * %9;\n\t"
      "add.u64 b3, %2, 3 * %9;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.eq.b32 t, %5, 0;\n\t"
      "elect.sync r|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, {%5, %5, %5, %5}, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, {%5, %5, %5, %5}, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, {%5, %5, %5, %5}, t;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "n"(IDESC), "r"(accumulate), "r"(0u), "n"(A1), "n"(A2), "n"(A3), "n"(STEP)
      : "memory");
}

// Weights w[32] (fp32, already scaled) as fp16 hi and lo over their scores.
// Returns the OR of the hi halves.
__device__ __forceinline__ uint32_t store_weights(uint32_t taddr, const float* w) {
  uint32_t all = 0;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    uint32_t h[8], l[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      tc16::split2(w[16 * s + 2 * k], w[16 * s + 2 * k + 1], h[k], l[k]);
      all |= h[k];
    }
    tc16::tmem_st8u(taddr + 8 * s, h);
    tc16::tmem_st8u(taddr + 8 * s + 16, l);
  }
  return all;
}

// What is left to do for a tile with small weights (see SmallWeights): no part of
// the loops that call it.  A row's blocks of 32 columns that the bits of `blocks`
// name are in their places as they are, in fp32.  settle_rows scales and splits
// them and returns their largest magnitude, or `big`; the two threads of a row
// do it in two steps, with an exchange between.
__device__ __forceinline__ float largest(float big, const float* w) {
#pragma unroll
  for (int i = 0; i < 32; i += 2) big = tc32::fmax3(big, fabsf(w[i]), fabsf(w[i + 1]));
  return big;
}
__device__ __forceinline__ void scale_and_store(uint32_t taddr, float* w, float f) {
#pragma unroll
  for (int i = 0; i < 32; ++i) w[i] *= f;
  store_weights(taddr, w);
}
__device__ __forceinline__ int small_exp(float big) { return big < kSmallWeight ? tc16::scale_exp(__float_as_uint(big)) : 0; }
__device__ __noinline__ float settle_rows(uint32_t taddr, uint32_t blocks, float big) {
  float w[32], x[32];
  tc32::tmem_wait_st();
  tmem_ld32x2(taddr, w, taddr + 32, x);
  if (blocks & 1u) big = largest(big, w);
  if (blocks & 2u) big = largest(big, x);
  const float f = tc16::pow2(small_exp(big));
  if (blocks & 1u) scale_and_store(taddr, w, f);
  if (blocks & 2u) scale_and_store(taddr + 32, x, f);
  return big;
}
__device__ __noinline__ float largest_weight(uint32_t taddr, float big) {
  float w[32];
  tc32::tmem_wait_st();
  tc32::tmem_ld32(taddr, w);
  return largest(big, w);
}
__device__ __noinline__ void split_again(uint32_t taddr, float big) {
  float w[32];
  tc32::tmem_ld32(taddr, w);
  scale_and_store(taddr, w, tc16::pow2(small_exp(big)));
}

// Two neighbouring values for the packed operations.
__device__ __forceinline__ float2 get2(const float* x) { return make_float2(x[0], x[1]); }
__device__ __forceinline__ void put2(float* x, float2 y) {
  x[0] = y.x;
  x[1] = y.y;
}

__device__ __forceinline__ float2 sub2(float2 x, float2 y) { return __ffma2_rn(y, make_float2(-1.f, -1.f), x); }

// N scores in place: s * mult (+ bias), -inf outside [lo, hi).
// flat: one bias for all of them.
template <int N, bool BIAS, int STEP>
__device__ __forceinline__ void mask_scores(float* s, float mult, const float* vec, bool flat, int lo, int hi, bool inside) {
  const float2 m2 = make_float2(mult, mult);
  if (!BIAS || flat) {
    const float2 b = BIAS ? make_float2(vec[0], vec[0]) : make_float2(-0.f, -0.f);
#pragma unroll
    for (int i = 0; i < N; i += 2) put2(s + i, BIAS ? __ffma2_rn(get2(s + i), m2, b) : __fmul2_rn(get2(s + i), m2));
  } else {
#pragma unroll
    for (int q = 0; q < N; q += 16) {  // 16 loads in flight
      float2 b[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) b[i] = make_float2(vec[STEP * (q + 2 * i)], vec[STEP * (q + 2 * i + 1)]);
#pragma unroll
      for (int i = 0; i < 8; ++i) put2(s + q + 2 * i, __ffma2_rn(get2(s + q + 2 * i), m2, b[i]));
    }
  }
  if (!inside) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < lo || i >= hi) s[i] = -INFINITY;
  }
}

// The sums along the diagonals of a 32 x 32 block (32 rows of 128 bytes under
// the 128-byte swizzle).  Lane (a, b) = (lane / 8, lane % 8) takes row 4 m + a,
// columns 4 ((m + b) mod 8) ... + 3 for m = 0 ... 7: column - row + a is 4 b ...
// + 3 while m + b < 8 (in `upper`), 32 less behind that (in `lower`).
// 16-byte loads without a bank conflict, and half the instructions of one
// column per lane and row.
__device__ __forceinline__ void diagonal_sums(const float* block, int lane, float2* upper, float2* lower) {
  const int a = lane >> 3, b = lane & 7;
  float4 x[8];
#pragma unroll
  for (int m = 0; m < 8; ++m)
    x[m] = *reinterpret_cast<const float4*>(block + (4 * m + a) * 32 + ((((m + b) & 7) ^ ((4 * m + a) & 7)) << 2));
  upper[0] = upper[1] = lower[0] = lower[1] = make_float2(0.f, 0.f);
#pragma unroll
  for (int m = 0; m < 8; ++m) {
    if (m + b < 8) {
      upper[0] = __fadd2_rn(upper[0], make_float2(x[m].x, x[m].y));
      upper[1] = __fadd2_rn(upper[1], make_float2(x[m].z, x[m].w));
    } else {
      lower[0] = __fadd2_rn(lower[0], make_float2(x[m].x, x[m].y));
      lower[1] = __fadd2_rn(lower[1], make_float2(x[m].z, x[m].w));
    }
  }
}

// Whether some pair of a block of 32 x 32 lies below the last bucket's bound;
// base: column - row of its first pair.
__device__ __forceinline__ bool near_block(int base, int far) { return base - 31 < far && base + 31 > -far; }
// Distances are kept in four copies by a, that of D at slot mid + D + a.  Near
// blocks have -far - 61 ... far + 61 and touch 64 slots from mid + base - 32.
constexpr int dist_mid(int far) { return (far + 67) / 4 * 4; }
constexpr int dist_slots(int far) { return (dist_mid(far) + far + 68) / 4 * 4; }

// The launches of a call overlap.  kForward and kDq start while split_kernel
// ends and wait for it before they read what it wrote; kDk and kDv start
// where the gradient before leaves room, which is after every CTA of kDq has
// waited for split_kernel, published that and said launch_dependents.  They
// acquire the published word before they read an image, so that its writes are
// ordered before their loads and bulk copies, and wait for the launch before
// them only at their end (whatever is behind them, the sum of the partials
// first, is to find all three complete).  The word alone cannot tell this
// call's 1 from one that was in the workspace before: split_kernel has cleared
// it long before a kDk can exist, and atomics and acquiring loads read L2,
// where that is the only copy.
//
// Persistent: the copy warp takes one unit after the other (the first by
// blockIdx, the others from a counter, since padding makes them uneven) and
// hands them to the other warps.  Every barrier and ring runs on across them:
// G counts the CTA's 64-column tiles, U its units with any.  GRAD (kDq): the
// table's gradient as well.
template <int KIND, int P, bool BIAS, bool GRAD = false>
__global__ void __launch_bounds__(tc_threads(P), P == 1 ? 2 : 1) tc_train(
    const __grid_constant__ TcArgs c, const __grid_constant__ CUtensorMap out_map,
    const __grid_constant__ CUtensorMap q_map) {
  using namespace tc32;
  constexpr bool kScores2 = KIND == kDq || KIND == kDk;      // S and dP, serial
  constexpr bool kByKey = KIND == kDk || KIND == kDv;        // rows are keys, columns queries
  constexpr bool kOwnRows = KIND == kForward && P == 1;      // q straight from its tensor, split by its row threads
  constexpr bool kBehindSplit = !kByKey;                     // the launch before is split_kernel
  constexpr int kHalves = P;                                 // threads per row
  constexpr int kW = 64 / kHalves;                           // score columns of a thread
  constexpr int kBlocks = kW / 32;
  constexpr bool kShared = KIND != kDq && kHalves == 2;      // a row's threads share a maximum
  constexpr int kRowThreadsTc = 128 * kHalves;
  constexpr int kIssueWarp = kRowWarpsOf(P);                 // then the copy warp and two for the table's gradient
  constexpr uint32_t kCols = 256 * P;
  constexpr uint32_t kColA2 = 64 * P;
  constexpr uint32_t kColS = kScores2 ? 128 * P : 64 * P;
  constexpr uint32_t kColS2 = kColS + 64;                    // dP, or the second score buffer
  constexpr uint32_t kColPart = kScores2 ? (P == 1 ? kColS2 : kColS2 + 64) : kColS2 + 64;
  static_assert(kColPart + 64 * P <= kCols, "tensor memory");
  constexpr int kB1 = kByKey ? kImgQ : kImgK, kB2 = kByKey ? kImgG : kImgV;  // the columns' operands
  constexpr int kA1 = kByKey ? kImgK : kImgQ, kA2 = kByKey ? kImgV : kImgG;  // the rows'
  constexpr uint32_t kOp = 2 * P * kPanelBytes;
  constexpr int kOutCols = kW * P;                           // output columns of a thread

  extern __shared__ unsigned char raw[];
  unsigned char* const smem = raw + (((smem_addr(raw) + 1023u) & ~1023u) - smem_addr(raw));
  unsigned char* const row_bufs = smem + kStages * stage_bytes<P>();
  TcTail<P>& sm = *reinterpret_cast<TcTail<P>*>(row_bufs + kRowWarpsOf(P) * kRowBuf);

  const AttnArgs& a = c.t.a;
  const int tid = threadIdx.x, warp = tid >> 5, d = a.head_dim;
  static_assert(!GRAD || (KIND == kDq && BIAS), "the table's gradient goes with dq");

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
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
    for (int s = 0; s < kIssueWarp; ++s) mbar_init(&sm.rows_full[s], 1);
    for (int s = 0; s < 8; ++s) {
      mbar_init(&sm.ds_ready[s], 1);
      mbar_init(&sm.ds_free[s], 1);
    }
    mbar_init(&sm.far_ready, kIssueWarp);
    mbar_init(&sm.far_free, 1);
    for (int s = 0; s < kQueue; ++s) {
      mbar_init(&sm.u_full[s], 1);
      mbar_init(&sm.u_free[s], kIssueWarp + (GRAD ? 3 : 1));
    }
    sm.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sm.tmem_base)),
                 "r"(kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
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
  // Read after the roles, by the warps that set them: the tiles copied and the products committed.
  int copied = 0, committed = 0;
  uint64_t* last_commit = nullptr;
  uint32_t last_parity = 0;

  // The consumers' next unit (n = -1 after the last one, or a timeout).
  int queued = 0;
  auto take_unit = [&](TcUnit& u) {
    const int s = queued % kQueue;
    const bool got = warp_wait(&sm.u_full[s], queued / kQueue);
    u = sm.unit[s];
    if (!got) u.n = -1;
    __syncwarp();
    if ((tid & 31) == 0) mbar_arrive(&sm.u_free[s]);
    ++queued;
    return got;
  };

  if (warp < kIssueWarp)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(row_regs(P)));
  else
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(other_regs(P)));
  if (warp < kIssueWarp) {
    // ---------------- rows ----------------
    if constexpr (kBehindSplit) wait_for_primary();
    const int half = warp >> 2, rt = tid & 127, ln = tid & 31;
    unsigned char* const buf = row_bufs + warp * kRowBuf;
    const uint32_t lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    constexpr int kStep = kByKey ? -1 : 1;
    // Where the thread's first column finds its distance: j - i relative to
    // the tile's first one (kByKey: i runs with the column, so backwards).
    const int vec_at = (kByKey ? rt + 64 : 128 - rt) + kStep * kW * half;

    // What a row needs besides its operands: 2^-e of these, the columns that
    // it sees, for kDq and kDk the (longest) length of the second, and for
    // kDq its exponent and delta.
    struct Row {
      float qmul, unit, off, delta, norm;
      int lo, hi;
    };
    // Unit u's rows, in rounds of two 32-word pieces of a thread (hi and lo
    // panels of the first operand, then of the second): from the images into
    // the warp's buffer, and on into tensor memory.
    constexpr int kRounds = (kScores2 ? 2 : 1) * P / kHalves;
    int fetched = 0;
    bool in_flight = false;
    auto fetch_rows = [&](const TcUnit& u, int round) {
      fence_proxy_async_smem();  // the warp's own accesses of the buffer, before the copies
      __syncwarp();
      if (ln == 0) {
        tma_store_wait_read();  // and the last unit's way out
        const long long tile = static_cast<long long>(u.local) * c.tiles + u.r0 / 64 + ((warp & 3) >> 1);
        mbar_arrive_expect_tx(&sm.rows_full[warp], kRowBuf);
        if constexpr (kOwnRows) {
#pragma unroll
          for (int p = 0; p < 2; ++p)
            tma_load_3d(buf + p * kBlockBytes, &q_map, 32 * p, u.r0 + warp * 32, static_cast<int>(c.slice0 + u.local),
                        &sm.rows_full[warp]);
        }
#pragma unroll
        for (int p = 0; p < 2 && !kOwnRows; ++p) {
          const int piece = (half * kRounds + round) * 2 + p;
          tma_load_1d(buf + p * kBlockBytes,
                      c.img[piece < 2 * P ? kA1 : kA2] + tile * static_cast<long long>(kOp) +
                          piece % (2 * P) * kPanelBytes + (warp & 1) * kBlockBytes,
                      kBlockBytes, &sm.rows_full[warp]);
        }
      }
      __syncwarp();
      in_flight = true;
    };
    // Piece p of the buffer: this lane's row of block p.
    auto buffered = [&](int p, float* w) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float4 x = *reinterpret_cast<const float4*>(buf + p * kBlockBytes + ln * 128 + ((k ^ (ln & 7)) << 4));
        w[4 * k] = x.x;
        w[4 * k + 1] = x.y;
        w[4 * k + 2] = x.z;
        w[4 * k + 3] = x.w;
      }
    };
    auto place_rows = [&](int round) {
      if (!warp_wait(&sm.rows_full[warp], fetched)) return false;
      in_flight = false;
      ++fetched;
      if constexpr (!kOwnRows) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          float w[32];
          buffered(p, w);
          tmem_st32(lane + 32 * ((half * kRounds + round) * 2 + p), w);
        }
      }
      return true;
    };
    // kOwnRows: the row of q in the buffer, scaled by an exponent of its own,
    // hi and lo into tensor memory (columns k / 2 and 32 + k / 2).  Returns 2^-e.
    auto split_row = [&](bool live) {
      float w[64];
      buffered(0, w);
      buffered(1, w + 32);
      float big = 0.f;
#pragma unroll
      for (int i = 0; i < 64; ++i) {
        if (!live) w[i] = 0.f;  // padding may hold anything
        if (fabsf(w[i]) < INFINITY) big = fmaxf(big, fabsf(w[i]));
      }
      const int e = tc16::scale_exp(__float_as_uint(big));
      const float2 up = make_float2(tc16::pow2(e), tc16::pow2(e));
#pragma unroll
      for (int q = 0; q < 64; q += 16) {
        uint32_t h[8], l[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float2 x = __fmul2_rn(get2(w + q + 2 * k), up);
          split_near(x.x, x.y, h[k], l[k]);
        }
        tc16::tmem_st8u(lane + q / 2, h);
        tc16::tmem_st8u(lane + 32 + q / 2, l);
      }
      return tc16::pow2(-e);
    };
    // A unit's rows (their first round is on the way) and what goes with them,
    // in two steps so that something can be done while the second round comes.
    // Called when the scores of the unit before are complete.
    static_assert(kRounds <= 2, "rounds of a unit's rows");
    auto load_first = [&](const TcUnit& u, Row& r) -> bool {
      const long long tile = static_cast<long long>(u.local) * c.tiles + u.r0 / 64 + ((warp & 3) >> 1);
      if constexpr (!kOwnRows) {
        const TileScale& s = c.scales[tile];
        r.qmul = a.qscale * tc16::pow2(-s.e[kA1]);
        r.unit = kScores2 ? tc16::pow2(-s.e[kA2]) : 0.f;
        r.norm = KIND == kDk ? s.v_norm : 0.f;
      }
      r.off = r.delta = 0.f;
      if constexpr (KIND == kDq) {
        r.off = c.rows[tile * kRowValues + (rt & 63)];
        r.delta = c.rows[tile * kRowValues + 64 + (rt & 63)];
        r.norm = c.rows[tile * kRowValues + 128 + (rt & 63)];
      }
      key_range(a, min(u.r0 + rt, u.valid - 1), u.valid, r.lo, r.hi);
      if (!place_rows(0)) return false;
      if constexpr (kRounds == 2) fetch_rows(u, 1);
      if constexpr (kOwnRows) r.qmul = a.qscale * split_row(u.r0 + rt < u.valid);
      return true;
    };
    auto load_rest = [&]() -> bool {
      if constexpr (kRounds == 2)
        if (!place_rows(1)) return false;
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&sm.a_ready);
      return true;
    };

    TcUnit u, nu;
    Row r, nr;
    int G = 0;
    bool ok = true;  // the same on every lane of the warp
    int units = 0;
    uint32_t ds_used = 0, ds_phase = 0;  // GRAD, by block: whether it is with the table's warps, the parity of its next return
    ok = take_unit(u);
    if constexpr (kByKey) fence_proxy_async_global();  // behind the copy warp's see_primary: the images, before the copies
    if (u.n > 0) {
      fetch_rows(u, 0);
      ok = load_first(u, r) && load_rest();
    }
    for (;;) {
      // Warps that meet at barriers of their own leave together.
      const bool leave = !ok || u.n <= 0;
      if (kShared ? bar_any(kPairBarrier + (warp & 3), 64, leave) : leave) break;
      const int row = u.r0 + rt;
      const size_t first_row = static_cast<size_t>(c.slice0 + u.local) * a.seq + u.r0;
      float far_before = 0.f, far_after = 0.f;
      if constexpr (GRAD) {
        if (ln == 0) tma_store_wait_read();  // the last unit's way out, before the columns of ds
        __syncwarp();
      }
      float o[kOutCols];
#pragma unroll
      for (int i = 0; i < kOutCols; ++i) o[i] = 0.f;
      float m_used = -INFINITY, m_true = -INFINITY, lsum = 0.f;
      float factor = 0.f;  // of the partial that is in flight
      // o += partial of tile g * factor, and the partial's columns are free.
      auto add_partial = [&](int g) {
        if (!warp_wait(&sm.part_full, g)) return false;
        tc_fence_after();
        static_assert(kOutCols == 64, "two loads of a thread's output columns");
        const uint32_t at = lane + kColPart + kOutCols * half;
        float x[64];
        tmem_ld32x2(at, x, at + 32, x + 32);
        tc_fence_before();
        mbar_arrive(&sm.part_free);
        const float2 f2 = make_float2(factor, factor);
#pragma unroll
        for (int i = 0; i < 64; i += 2) put2(o + i, __ffma2_rn(get2(x + i), f2, get2(o + i)));
        return true;
      };
      // Block q of the buffer is back from the table's warps.
      auto ds_return = [&](int q) -> bool {
        if (!(ds_used >> q & 1u)) return true;
        if (!warp_wait(&sm.ds_free[warp * kBlocks + q], ds_phase >> q)) return false;
        ds_phase ^= 1u << q;
        ds_used &= ~(1u << q);
        return true;
      };
      // The larger of the row's two values x; false if either thread's warp gave up.
      auto share_max = [&](int g, float& x) {
        if constexpr (kHalves == 1) return ok;
        sm.red[g & 1][half][rt] = x;
        if (bar_any(kPairBarrier + (warp & 3), 64, !ok)) return false;
        x = fmaxf(x, sm.red[g & 1][half ^ 1][rt]);
        return true;
      };
      // kDk and kDv: a key may have nothing but small weights.  Where its largest
      // so far, in this tile's scale, is kSmallWeight or more, fp16 holds the
      // tile's to 2^-24 (half a step of hi and of lo), 2^-22 of that one.  The
      // weights of a row that has had none are scaled by 2^e more, which brings
      // the largest to 2^14.  A block with such rows is put over its scores once
      // more as it is (`raw`), and split when the row is known.  The loops pay an
      // OR of the hi parts, whose exponents have their top bit from 2 on, and a
      // vote, both behind the stores: a branch before them, or the rest in line,
      // cost every tile 4%.  With it: every key 478 to 502 us, window 233 to 242.
      float top = 0.f;  // the row's largest in the unit, unscaled, or less where it is large enough
      struct SmallWeights {
        float big;        // that in the tile's scale, with the tile's own
        int e = 0;
        bool seen = false;
        uint32_t raw = 0;  // the same on every lane of the warp
      };
      // Behind the store of block q, which gave `bits`; seen: some of the row's
      // weights in it may not be zero.
      auto weigh = [&](SmallWeights& sw, int q, uint32_t scol, const float* w, uint32_t bits, bool seen) {
        if (bits & 0x40004000u) sw.big = fmaxf(sw.big, 2.f);
        sw.seen |= seen;
        if (__any_sync(0xffffffffu, sw.seen && !(sw.big >= kSmallWeight))) {
          tmem_wait_st();
          tmem_st32(scol + 32 * q, w);
          sw.raw |= 1u << q;
        }
      };
      // Behind the last block; down: one over the tile's scale.  False if a
      // pair's other warp gave up.
      auto settle = [&](SmallWeights& sw, uint32_t scol, float down, int g) -> bool {
        if constexpr (kHalves == 1) {
          if (sw.raw) sw.big = settle_rows(scol, sw.raw, sw.big);
        } else {
          if (sw.raw) sw.big = largest_weight(scol, sw.big);
          if (!share_max(g, sw.big)) return ok = false;
          if (sw.raw) split_again(scol, sw.big);
        }
        sw.e = small_exp(sw.big);
        top = fmaxf(top, fminf(sw.big, 32768.f) * down);
        return true;
      };
      nu.n = -1;
      // The next unit's rows: begun before the last tile (with the table's
      // gradient behind it, when the buffer is back), placed behind it.
      auto begin_next = [&] {
        if (ok && take_unit(nu) && nu.n > 0) fetch_rows(nu, 0);
      };
      auto prepare_next = [&](int t) {
        if (t + 1 < u.n) return;
        if constexpr (GRAD) {
#pragma unroll
          for (int q = 0; q < kBlocks; ++q) ok = ok && ds_return(q);
          begin_next();
        }
        if (ok && nu.n > 0) ok = load_first(nu, nr) && (kScores2 || load_rest());
      };

      for (int t = 0; t < u.n; ++t, ++G) {
        const int st = G % kStages, c0 = (u.t0 + t) * kTileCols + kW * half;
        const int sb = kScores2 ? 0 : G & 1;
        if (!GRAD && t + 1 == u.n) begin_next();
        if (ok) ok = warp_wait(&sm.full[st], G / kStages) && warp_wait(&sm.s_full[sb], kScores2 ? G : G >> 1);
        if (!kShared && !ok) break;
        tc_fence_after();
        const uint32_t scol = lane + kColS + 64 * sb + kW * half;
        const int e1 = sm.scales[st].e[kB1], e2 = sm.scales[st].e[kB2];
        const int mlo = r.lo - c0, mhi = r.hi - c0;
        const bool inside = __all_sync(0xffffffffu, mlo <= 0 && mhi >= kW);
        const float mult = finite(r.qmul * tc16::pow2(-e1));
        const bool flat = BIAS && sm.flat[st] != 0;
        const float* const vec = &sm.vec[st][vec_at];
        const bool some = !flat || vec[0] != -INFINITY;  // the bias leaves the tile
        // 32 columns at a time, in rolled loops (the loop over the tiles is to
        // fit the instruction cache nearest to the scheduler): block q's masked
        // scores, and back into tensor memory until the row's maximum is known.
        auto block_scores = [&](int q, float* s, float* dp) {
          if constexpr (kScores2)
            tmem_ld32x2(scol + 32 * q, s, lane + kColS2 + kW * half + 32 * q, dp);
          else
            tmem_ld32(scol + 32 * q, s);
          mask_scores<32, BIAS, kStep>(s, mult, vec + kStep * 32 * q, flat, mlo - 32 * q, mhi - 32 * q, inside);
        };

        if constexpr (KIND == kForward) {
          float mx = -INFINITY;
          if (ok) {
#pragma unroll 1
            for (int q = 0; q < kBlocks; ++q) {
              float s[32];
              block_scores(q, s, nullptr);
#pragma unroll
              for (int i = 0; i < 32; i += 2) mx = fmax3(mx, s[i], s[i + 1]);
              tmem_st32(scol + 32 * q, s);
            }
            tmem_wait_st();
          }
          if (!share_max(G, mx)) { ok = false; break; }
          float alpha = 1.f;
          m_true = fmaxf(m_true, mx);
          if (mx > m_used + kRescale) {
            alpha = ex2(m_used - mx);
            m_used = mx;
          }
          const float base = (m_used == -INFINITY ? 0.f : m_used) - kForwardLog2;
          const float2 nb = make_float2(-base, -base);
          float2 sum = make_float2(0.f, 0.f), sum1 = sum;
#pragma unroll 1
          for (int q = 0; q < kBlocks; ++q) {
            float s[32];
            tmem_ld32(scol + 32 * q, s);
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float2 x = __fadd2_rn(get2(s + i), nb), y = __fadd2_rn(get2(s + i + 2), nb);
              put2(s + i, make_float2(ex2(x.x), ex2(x.y)));
              put2(s + i + 2, make_float2(ex2(y.x), ex2(y.y)));
              sum = __fadd2_rn(sum, get2(s + i));
              sum1 = __fadd2_rn(sum1, get2(s + i + 2));
            }
            store_weights(scol + 32 * q, s);
          }
          sum = __fadd2_rn(sum, sum1);
          lsum = fmaf(lsum, alpha, sum.x + sum.y);
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&sm.w_ready[sb]);
          if (t > 0) {
            ok = add_partial(G - 1);
            if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
              for (int i = 0; i < kOutCols; i += 2) put2(o + i, __fmul2_rn(get2(o + i), make_float2(alpha, alpha)));
            }
          }
          factor = tc16::pow2(-e2);
          prepare_next(t);
        } else if constexpr (KIND == kDv) {
          SmallWeights sw;
          sw.big = top * tc16::pow2(e2) * kWeightScale;
#pragma unroll 1
          for (int q = 0; q < kBlocks; ++q) {
            const float* off = sm.rows[st] + kW * half + 32 * q;
            float s[32];
            block_scores(q, s, nullptr);
            const float2 up = make_float2(kWeightScale, kWeightScale);
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 f = *reinterpret_cast<const float4*>(off + i);
              const float2 x = sub2(get2(s + i), make_float2(f.x, f.y)), y = sub2(get2(s + i + 2), make_float2(f.z, f.w));
              put2(s + i, __fmul2_rn(make_float2(ex2(x.x), ex2(x.y)), up));
              put2(s + i + 2, __fmul2_rn(make_float2(ex2(y.x), ex2(y.y)), up));
            }
            const uint32_t bits = store_weights(scol + 32 * q, s);
            weigh(sw, q, scol, s, bits, some && sm.scales[st].g_norm > 0.f && mlo < 32 * q + 32 && mhi > 32 * q);
          }
          if (!settle(sw, scol, tc16::pow2(-e2) * (1.f / kWeightScale), G)) break;
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&sm.w_ready[sb]);
          if (t > 0) ok = add_partial(G - 1);
          factor = tc16::pow2(-e2) * (1.f / kWeightScale) * tc16::pow2(-sw.e);
          prepare_next(t);
        } else {
          // ds = w (g . v - delta) times 2^e, which brings the bound |g| |v| +
          // |delta| (w <= 1, the column's or the row's longest vector) to
          // [2^13, 2^14): four times that still fit, should rounding bring a
          // weight above 1.  fp16 holds what is 2^-37 of the bound.  That will
          // do for dq, where some weight of the row is of the size of 1.
          const float unit = finite(r.unit * tc16::pow2(-e2));
          const float bound = KIND == kDq ? fmaf(r.norm * sm.scales[st].v_norm, unit, fabsf(r.delta))
                                          : fmaf(r.norm * sm.scales[st].g_norm, unit, sm.scales[st].delta);
          const int e = tc16::scale_exp(__float_as_uint(finite(bound))) - 1;
          const float up = tc16::pow2(e), down = tc16::pow2(-e);
          const float unit_up = finite(unit * up), minus_up = KIND == kDq ? -r.delta * up : -up;
          const float2 unit2 = make_float2(unit_up, unit_up), minus2 = make_float2(minus_up, minus_up);
          SmallWeights sw;
          sw.big = top * up;
#pragma unroll 1
          for (int q = 0; q < kBlocks; ++q) {
            const float* off = sm.rows[st] + kW * half + 32 * q;
            float s[32], dp[32];
            block_scores(q, s, dp);
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              float4 f;
              float2 g0 = minus2, g1 = minus2;
              if constexpr (KIND == kDk) {
                f = *reinterpret_cast<const float4*>(off + i);
                const float4 g = *reinterpret_cast<const float4*>(off + 64 + i);
                g0 = __fmul2_rn(make_float2(g.x, g.y), minus2);
                g1 = __fmul2_rn(make_float2(g.z, g.w), minus2);
              } else {
                f = make_float4(r.off, r.off, r.off, r.off);
              }
              const float2 x = sub2(get2(s + i), make_float2(f.x, f.y));
              const float2 y = sub2(get2(s + i + 2), make_float2(f.z, f.w));
              put2(s + i, __fmul2_rn(make_float2(ex2(x.x), ex2(x.y)), __ffma2_rn(get2(dp + i), unit2, g0)));
              put2(s + i + 2, __fmul2_rn(make_float2(ex2(y.x), ex2(y.y)), __ffma2_rn(get2(dp + i + 2), unit2, g1)));
            }
            const uint32_t bits = store_weights(scol + 32 * q, s);
            if constexpr (KIND == kDk)
              weigh(sw, q, scol, s, bits, some && bound > 0.f && mlo < 32 * q + 32 && mhi > 32 * q);
            if constexpr (GRAD) {
              const int base = c0 + 32 * q - (u.r0 + (warp & 3) * 32);  // column - row of the block's first pair
              if (!near_block(base, c.far)) {
                float2 x = get2(s), y = get2(s + 2);
#pragma unroll
                for (int i = 4; i < 32; i += 4) {
                  x = __fadd2_rn(x, get2(s + i));
                  y = __fadd2_rn(y, get2(s + i + 2));
                }
                const float sum = ((x.x + x.y) + (y.x + y.y)) * down;
                if (base > 0)
                  far_after += sum;
                else
                  far_before += sum;
              } else {
                ok = ok && ds_return(q);
                if (ok) {
                  const float2 down2 = make_float2(down, down);
#pragma unroll
                  for (int i = 0; i < 32; i += 4) {
                    const float2 x = __fmul2_rn(get2(s + i), down2), y = __fmul2_rn(get2(s + i + 2), down2);
                    *reinterpret_cast<float4*>(buf + q * kBlockBytes + ln * 128 + (((i >> 2) ^ (ln & 7)) << 4)) =
                        make_float4(x.x, x.y, y.x, y.y);
                  }
                  __syncwarp();
                  if (ln == 0) mbar_arrive(&sm.ds_ready[warp * kBlocks + q]);
                  ds_used |= 1u << q;
                }
              }
            }
          }
          if constexpr (KIND == kDk) {
            if (!settle(sw, scol, down, G)) break;
          }
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&sm.w_ready[sb]);
          factor = finite(KIND == kDk ? two_to(-(e + e1 + sw.e)) : tc16::pow2(-e) * tc16::pow2(-e1));
          prepare_next(t);
          if (ok) ok = add_partial(G);
          if (ok && t + 1 == u.n && nu.n > 0) ok = load_rest();
        }
      }
      if constexpr (!kScores2)
        if (ok) ok = add_partial(G - 1);

      float f = KIND == kDv ? 1.f : c.t.scale;
      if constexpr (KIND == kForward) {
        if constexpr (kHalves == 2) {  // the row's sum: first half + second half
          sm.red[0][half][rt] = lsum;  // the last exchange is read: part_full follows both threads' w_ready
          if (bar_any(kPairBarrier + (warp & 3), 64, !ok)) { ok = false; break; }
          lsum = sm.red[0][0][rt] + sm.red[0][1][rt];  // and read before the pair meets at the loop's top
        }
        f = lsum > 0.f ? 1.0f / lsum : lsum != lsum ? lsum : 0.f;
        if (ok && c.t.stats_out && half == 0 && row < a.seq)
          c.t.stats_out[first_row + rt] =
              row < u.valid ? make_stats(m_true, (m_used == -INFINITY ? 0.f : m_used) - kForwardLog2, lsum)
                            : make_float2(-INFINITY, 0.f);
        __syncwarp();
      }
      if constexpr (GRAD) {
        // The rows' sums beyond the last bound, to the table's warps.
        if (ok && units > 0) ok = warp_wait(&sm.far_free, units - 1);
        if (ok) {
          sm.far[warp][ln] = make_float2(far_before, far_after);
          __syncwarp();
          if (ln == 0) mbar_arrive(&sm.far_ready);
          ++units;
        }
      }
      if (ok) {
        const bool live = row < u.valid;
        const int wr0 = u.r0 + (warp & 3) * 32;
        if (ln == 0) tma_store_wait_read();  // a last unit fetches no rows: the one before may still be on its way out
        __syncwarp();
#pragma unroll
        for (int q = 0; q < kOutCols; q += 32) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(buf + q * 128 + ln * 128 + (((i >> 2) ^ (ln & 7)) << 4)) =
                live ? make_float4(o[q + i] * f, o[q + i + 1] * f, o[q + i + 2] * f, o[q + i + 3] * f)
                     : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (ln == 0 && wr0 < a.seq) {
#pragma unroll
          for (int q = 0; q < kOutCols; q += 32)
            if (kOutCols * half + q < d)
              tma_store_3d(&out_map, buf + q * 128, kOutCols * half + q, wr0, static_cast<int>(c.slice0 + u.local));
          tma_store_commit();
        }
        __syncwarp();
      }
      u = nu;
      r = nr;
    }
    if (ln == 0) tma_store_wait_read();
    if (in_flight) {  // only after a timeout: bounded, as the drains below
      const long long t_end = clock64() + a.timeout_cycles;
      while (!mbar_try_wait(&sm.rows_full[warp], fetched & 1u) && clock64() < t_end) {
      }
    }
    __syncwarp();
  } else if (warp == kIssueWarp) {
    // ---------------- MMA issue ----------------
    auto commit = [&](uint64_t* bar, uint32_t parity) {
      mma_commit_e(bar);
      last_commit = bar;
      last_parity = parity & 1u;
    };
    const uint32_t ops = smem_addr(smem);
    auto operand = [&](int g, int which) {
      return ops + static_cast<uint32_t>((g % kStages) * stage_bytes<P>() + which * kOp);
    };
    // rows x columns^T into dcol.  Both panels' small products come before the
    // large ones: panel by panel, what the accumulation truncates put the
    // table's gradient at head size 96 1.1e-6 off its largest value, not 7.6e-7.
    auto scores = [&](uint32_t dcol, uint32_t acol, uint32_t b) {
      const uint32_t hi = tmem + acol, lo = hi + 32 * P, blo = b + P * kPanelBytes;
      if constexpr (P == 1) {
        mma12_ts_e<tc16::kIdescQK, 2, 8, 16, 24>(tmem + dcol, hi, lo, tc16::b_desc(b, 0), tc16::b_desc(blo, 0), 0u);
      } else {
        auto four = [&](uint32_t at, uint32_t op, uint32_t add) {
          mma4_ts_e<tc16::kIdescQK, 2, 8, 16, 24>(tmem + dcol, at, tc16::b_desc(op, 0), add);
        };
#pragma unroll
        for (int p = 0; p < P; ++p) four(hi + 32 * p, blo + p * kPanelBytes, p > 0 ? 1u : 0u);
#pragma unroll
        for (int p = 0; p < P; ++p) four(lo + 32 * p, b + p * kPanelBytes, 1u);
#pragma unroll
        for (int p = 0; p < P; ++p) four(hi + 32 * p, b + p * kPanelBytes, 1u);
      }
    };
    // weights x operand (its 64 rows are the inner dimension) into the partial
    auto sums = [&](uint32_t wcol, uint32_t b) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const uint32_t hi = tmem + wcol, bhi = b + p * kPanelBytes;
        mma12_ts_e<tc16::kIdescPV, 128, 8, 32, 40>(tmem + kColPart + 64 * p, hi, hi + 16, tc16::v_desc(bhi, 0),
                                                   tc16::v_desc(bhi + P * kPanelBytes, 0), 0u);
      }
    };
    int G = 0, U = 0;
    bool ok = true;
    TcUnit u;
    while (ok && take_unit(u) && u.n > 0) {
      const int n = u.n;
      ok = warp_wait(&sm.a_ready, U++);
      for (int t = 0; ok && t < n; ++t, ++G) {
        if constexpr (kScores2) {
          ok = warp_wait(&sm.full[G % kStages], G / kStages);
          // S takes the place of the last weights, whose product is complete,
          // dP (for P = 1) that of its sum, which the row threads have added.
          if (ok && G > 0) ok = warp_wait(&sm.part_full, G - 1);
          if (!ok) break;
          tc_fence_after();
          scores(kColS, 0, operand(G, 0));
          if (G > 0) ok = warp_wait(&sm.part_free, G - 1);
          if (!ok) break;
          tc_fence_after();
          scores(kColS2, kColA2, operand(G, 1));
          commit(&sm.s_full[0], G);
        } else {
          // The scores of tile g go to the buffer that held the weights of tile g - 2, whose product is complete.
          auto scores_of = [&](int g) {
            ok = warp_wait(&sm.full[g % kStages], g / kStages);
            if (!ok) return;
            tc_fence_after();
            scores(kColS + 64 * (g & 1), 0, operand(g, 0));
            commit(&sm.s_full[g & 1], g >> 1);
          };
          if (t == 0) scores_of(G);
          if (ok && t + 1 < n) {
            if (G > 0) ok = warp_wait(&sm.part_full, G - 1);
            if (ok) scores_of(G + 1);
          }
        }
        if (ok) ok = warp_wait(&sm.w_ready[kScores2 ? 0 : G & 1], kScores2 ? G : G >> 1);
        if (!kScores2 && ok && G > 0) ok = warp_wait(&sm.part_free, G - 1);
        if (!ok) break;
        tc_fence_after();
        sums(kScores2 ? kColS : kColS + 64 * (G & 1), operand(G, kScores2 ? 0 : 1));
        commit(&sm.freed[G % kStages], G / kStages);
        commit(&sm.part_full, G);
        committed = G + 1;
      }
    }
    // Nothing arrives on a barrier after the CTA has ended.
    for (int g = max(0, committed - kStages); ok && g < committed; ++g) ok = warp_wait(&sm.freed[g % kStages], g / kStages);
  } else if (GRAD && warp > kIssueWarp + 1) {
    // ---------------- the table's gradient ----------------
    // Two warps, each with the row warps of its parity: their near blocks of
    // ds (some pair below the last bound) by distance, and at the unit's end
    // the distances by bucket, everything in a fixed order.  Beside the row
    // threads, whose own diagonal sums took 1.6k cycles a block and 7k a unit.
    const int me = warp - (kIssueWarp + 2), ln = tid & 31;
    float* const all = c.dist ? c.dist + static_cast<size_t>(blockIdx.x) * 8 * c.slots : reinterpret_cast<float*>(&sm + 1);
    float* const dist = all + 4 * me * c.slots;
    const int mid = dist_mid(c.far);
    uint32_t phase = 0;
    bool ok = true;
    TcUnit u;
    for (int units = 0;; ++units) {
      const bool got = take_unit(u);
      if (bar_any(kTableBarrier, 64, !got) || u.n <= 0) break;  // both leave together
      for (int i = ln; i < c.slots; i += 32) reinterpret_cast<float4*>(dist)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      __syncwarp();
      for (int t = 0; ok && t < u.n; ++t)
        for (int w = me; ok && w < kIssueWarp; w += 2)
          for (int q = 0; ok && q < kBlocks; ++q) {
            const int base = (u.t0 + t) * kTileCols + kW * (w >> 2) + 32 * q - (u.r0 + (w & 3) * 32);
            if (!near_block(base, c.far)) continue;
            const int i = w * kBlocks + q;
            ok = warp_wait(&sm.ds_ready[i], phase >> i);
            if (!ok) break;
            phase ^= 1u << i;
            float2 upper[2], lower[2];
            diagonal_sums(reinterpret_cast<const float*>(row_bufs + w * kRowBuf + q * kBlockBytes), ln, upper, lower);
            __syncwarp();
            if (ln == 0) mbar_arrive(&sm.ds_free[i]);
            float4* const at = reinterpret_cast<float4*>(dist + (ln >> 3) * c.slots + mid + base) + (ln & 7);
            const float4 x = at[0], y = at[-8];
            at[0] = make_float4(x.x + upper[0].x, x.y + upper[0].y, x.z + upper[1].x, x.w + upper[1].y);
            at[-8] = make_float4(y.x + lower[0].x, y.y + lower[0].y, y.z + lower[1].x, y.w + lower[1].y);
            __syncwarp();
          }
      if (ok) ok = warp_wait(&sm.far_ready, units);
      if (bar_any(kTableBarrier, 64, !ok)) break;
      // Warp 0 has the keys up to the query, warp 1 those behind it.  First
      // each distance's eight copies into one (in its own slot of the first
      // copy), those from the last bound on into `beyond`.
      const bool behind = me == 1;
      float beyond = 0.f;
      for (int w = 0; w < kIssueWarp; ++w) beyond += behind ? sm.far[w][ln].y : sm.far[w][ln].x;
      for (int i = me + ln; i < c.far + 62; i += 32) {
        float* const at = all + mid + (behind ? i : -i);
        float y[8];
#pragma unroll
        for (int p = 0; p < 8; ++p) y[p] = at[p * c.slots + (p & 3)];
        const float x = ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
        if (i >= c.far)
          beyond += x;
        else
          at[0] = x;
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) beyond += __shfl_xor_sync(0xffffffffu, beyond, off);
      __syncwarp();
      const int sides = c.t.buckets / 2;
      float* const partial = c.t.part + (static_cast<size_t>(c.slice0 + u.local) * c.t.parts + u.r0 / kTileRows) * c.t.buckets + me * sides;
      for (int k0 = 0; k0 < sides; k0 += 8) {  // four lanes to a bucket
        const int k = k0 + (ln >> 2);
        float x = 0.f;
        if (k + 1 < sides) {
          const int to = min(c.bounds.at[k + 1], c.far);
          for (int i = max(c.bounds.at[k], me) + (ln & 3); i < to; i += 4) x += all[mid + (behind ? i : -i)];
        }
        x += __shfl_xor_sync(0xffffffffu, x, 1);
        x += __shfl_xor_sync(0xffffffffu, x, 2);
        if (k < sides && (ln & 3) == 0) partial[k] = k + 1 == sides ? beyond : x;
      }
      if (bar_any(kTableBarrier, 64, false)) break;  // both are done with the distances and the far sums
      if (me == 0 && ln == 0) mbar_arrive(&sm.far_free);
      __syncwarp();
    }
  } else if (warp == kIssueWarp + 1) {
    // ---------------- units and bulk copies ----------------
    bool ok = true, first = true;
    unsigned unit = blockIdx.x;
    for (int k = 0; ok;) {
      TcUnit u{0, 0, 0, 0, -1};
      if (unit < c.units) {
        const unsigned tiles = static_cast<unsigned>(c.tiles) / 2;
        u.local = static_cast<int>(unit / tiles);
        u.valid = valid_of(a, c.slice0 + u.local);
        u.r0 = static_cast<int>(unit - u.local * tiles) * kTileRows;
        int lo = 0, hi = 0, unused;
        if (u.r0 < u.valid) {
          key_range(a, u.r0, u.valid, lo, unused);
          key_range(a, min(u.r0 + kTileRows, u.valid) - 1, u.valid, unused, hi);
        }
        u.t0 = lo / kTileCols;
        u.n = hi > lo ? (hi + kTileCols - 1) / kTileCols - u.t0 : 0;
      }
      if (first) {
        if constexpr (kBehindSplit)
          wait_for_primary();
        else
          see_primary(c.next + kForward);
        if constexpr (KIND == kDq) {
          if ((tid & 31) == 0) publish_primary(c.next + kForward);
          __syncwarp();
        }
        if constexpr (KIND != kForward) launch_dependents();
        first = false;
      }
      if ((tid & 31) == 0) unit = gridDim.x + atomicAdd(c.next + KIND, 1u);  // the next one, used a unit later
      if (u.n == 0) {  // padding only: split_kernel has written its zeros
        unit = __shfl_sync(0xffffffffu, unit, 0);
        continue;
      }
      if (k >= kQueue) ok = warp_wait(&sm.u_free[k % kQueue], k / kQueue - 1);
      if (!ok) break;
      if ((tid & 31) == 0) {
        sm.unit[k % kQueue] = u;
        mbar_arrive(&sm.u_full[k % kQueue]);
        if (!kOwnRows && u.n > 0) {  // its rows, a unit ahead of their use
          const long long tile = static_cast<long long>(u.local) * c.tiles + u.r0 / 64;
          prefetch_l2(c.img[kA1] + tile * static_cast<long long>(kOp), 2 * kOp);
          if constexpr (kScores2) prefetch_l2(c.img[kA2] + tile * static_cast<long long>(kOp), 2 * kOp);
        }
      }
      __syncwarp();
      ++k;
      if (u.n < 0) break;
      const int head = static_cast<int>((c.slice0 + u.local) % a.heads);
      for (int t = 0; t < u.n; ++t) {
        const int st = copied % kStages, c0 = (u.t0 + t) * kTileCols;
        if (copied >= kStages) ok = warp_wait(&sm.freed[st], copied / kStages - 1);
        if (!ok) break;
        if (tc16::lane_is_first(tid)) {
          fence_proxy_async_smem();  // the row threads' reads of this stage, before the copies
          const long long tile = static_cast<long long>(u.local) * c.tiles + u.t0 + t;
          // The tile's first distance j - i: rows' i from r0, or columns' i from c0.
          const int rel = kByKey ? u.r0 - c0 - 64 : c0 - u.r0 - 128;
          unsigned char* op = smem + st * stage_bytes<P>();
          uint64_t* bar = &sm.full[st];
          if constexpr (BIAS) sm.flat[st] = rel + 1 >= c.far || rel + kVec - 1 <= -c.far;
          constexpr uint32_t kScaleBytes = sizeof(TileScale), kRowBytes = 128 * 4;
          mbar_arrive_expect_tx(bar, 2 * kOp + kScaleBytes + (BIAS ? kVec * 4u : 0u) + (kByKey ? kRowBytes : 0u));
          tma_load_1d(op, c.img[kB1] + tile * static_cast<long long>(kOp), kOp, bar);
          tma_load_1d(op + kOp, c.img[kB2] + tile * static_cast<long long>(kOp), kOp, bar);
          tma_load_1d(&sm.scales[st], c.scales + tile, kScaleBytes, bar);
          if constexpr (BIAS)
            tma_load_1d(sm.vec[st], c.t.rel_bias + (2ll * head + 1) * c.t.rel_half + rel, kVec * 4u, bar);
          if constexpr (kByKey) tma_load_1d(sm.rows[st], c.rows + tile * kRowValues, kRowBytes, bar);
        }
        __syncwarp();
        ++copied;
      }
      unit = __shfl_sync(0xffffffffu, unit, 0);
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
    if (tid == (kIssueWarp + 1) * 32)
      for (int g = max(0, copied - kStages); g < copied; ++g) drain(&sm.full[g % kStages], g / kStages);
    if (tid == kIssueWarp * 32 && last_commit) drain(last_commit, last_parity);
  }
  __syncthreads();
  if (warp == kIssueWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
  }
  if constexpr (!kBehindSplit) {
    if (tid == 0) wait_for_primary();
  }
}

}  // namespace train
}  // namespace raya
