// train_host.cuh — the host side of the training operators: argument checks,
// the bias's bucket bounds, the workspace's layout and the launches.
// Included by raya_attn.cu inside its anonymous namespace.

constexpr int kMinBuckets = 4;
constexpr int kMaxBucketPowers = train::kMaxBuckets / 4;
constexpr long long kMaxDistance = 1ll << 29;

raya_attn_status check_buckets(int32_t buckets, int32_t max_distance) {
  if (buckets < kMinBuckets || buckets > train::kMaxBuckets || buckets % 2 != 0)
    return fail(RAYA_ATTN_ERR_UNSUPPORTED, "unsupported: %d bias buckets (an even number, %d to %d)", buckets,
                kMinBuckets, train::kMaxBuckets);
  if (max_distance <= buckets / 4 || max_distance >= kMaxDistance)
    return fail(RAYA_ATTN_ERR_SHAPE, "invalid shape: max_distance %d (above %d, below %lld for %d buckets)",
                max_distance, buckets / 4, kMaxDistance, buckets);
  return RAYA_ATTN_OK;
}

// a^p * b^q as base-2^32 digits, least significant first (p + q <= 32
// factors below 2^32, so 33 digits hold it).
struct Digits {
  uint32_t at[kMaxBucketPowers + 1];
  int n;
};
Digits power_product(uint32_t a, int p, uint32_t b, int q) {
  Digits x{{1}, 1};
  for (int i = 0; i < p + q; ++i) {
    const uint32_t factor = i < p ? a : b;
    uint64_t carry = 0;
    for (int k = 0; k < x.n; ++k) {
      carry += static_cast<uint64_t>(x.at[k]) * factor;
      x.at[k] = static_cast<uint32_t>(carry);
      carry >>= 32;
    }
    if (carry) x.at[x.n++] = static_cast<uint32_t>(carry);
  }
  return x;
}

bool at_least(const Digits& x, const Digits& y) {  // x >= y
  if (x.n != y.n) return x.n > y.n;
  for (int k = x.n - 1; k >= 0; --k)
    if (x.at[k] != y.at[k]) return x.at[k] > y.at[k];
  return true;
}

// Bucket first + k begins at the least whole n >= first * (max / first)^(k /
// rest).  Where that number is no whole one within double's error, rounding
// up is safe; next to a whole number r the powers r^rest and first^(rest - k)
// * max^k are compared exactly.
train::BucketBounds bucket_bounds(int buckets, int max_distance) {
  train::BucketBounds b{};
  const int half = buckets / 2, first = half / 2, rest = half - first;
  for (int k = 0; k < first; ++k) b.at[k] = k;
  for (int k = 0; k < rest; ++k) {
    const double x = first * std::pow(static_cast<double>(max_distance) / first, static_cast<double>(k) / rest);
    const double r = std::round(x);
    if (std::fabs(x - r) > 1e-9 * r)
      b.at[first + k] = static_cast<int>(std::ceil(x));
    else
      b.at[first + k] = static_cast<int>(r) + (at_least(power_product(static_cast<uint32_t>(r), rest, 1, 0),
                                                        power_product(static_cast<uint32_t>(first), rest - k,
                                                                      static_cast<uint32_t>(max_distance), k))
                                                   ? 0
                                                   : 1);
  }
  return b;
}

// Where the workspace keeps what; offsets in bytes, each 16-byte aligned.
struct TrainPlan {
  int rel_half = 0;  // the bias table by distance covers rel in [-rel_half, rel_half)
  int parts = 1;     // partials of the table's gradient per slice
  int panels = 0;    // 64-column panels of head_dim on the tensor cores; 0: the row-wise kernels
  int tiles = 0;     // 64-row tiles per slice, an even number
  long long chunk = 0;  // slices whose images the workspace holds at a time
  size_t rel_bias = 0, rel_id = 0, delta = 0, part = 0;
  size_t img[4] = {}, scales = 0, rows = 0, next = 0;
  int far = 0, slots = 0;           // the table's gradient by distance (train_tc.cuh)
  size_t dist = 0;                  // where it does not fit into shared memory,
  long long dist_ctas = 0;          // for that many CTAs (0: it fits)
  size_t bytes = 0;
};

// The images of one chunk of slices.  A chunk ends with a tail of units, so
// smaller ones are slower even where they stay in L2: 8 x 16 x 8192 backward
// took 1.73 ms within this bound, 2.03, 2.33 and 2.91 with 192, 96 and 48 MB.
constexpr size_t kMaxImageBytes = size_t{2} << 30;
constexpr long long kMaxResident = 2 * 148;  // persistent CTAs: two on each SM

raya_attn_status train_plan(const raya_attn_desc* d, const raya_attn_bias* bias, bool backward, TrainPlan* plan) {
  raya_attn_status st = check_shape(d);
  if (st != RAYA_ATTN_OK) return st;
  if (bias && (st = check_buckets(bias->buckets, bias->max_distance)) != RAYA_ATTN_OK) return st;
  // Below these every index of the kernels fits its type.
  const long long kMaxRows = 1ll << 40, kMaxSlices = 0x7fffffffll;
  if (d->batch > kMaxSlices / d->heads || d->batch * d->heads > kMaxRows / std::max<int64_t>(d->seq, 1))
    return fail(RAYA_ATTN_ERR_UNSUPPORTED, "unsupported: %lld sequences of %lld heads and %lld rows",
                static_cast<long long>(d->batch), static_cast<long long>(d->heads), static_cast<long long>(d->seq));
  *plan = TrainPlan{};
  if (d->seq == 0) return RAYA_ATTN_OK;
  const long long slices = d->batch * d->heads;
  auto take = [plan](size_t bytes) {
    const size_t at = plan->bytes;
    plan->bytes += (bytes + 15) & ~static_cast<size_t>(15);
    return at;
  };
  if (bias) {
    plan->rel_half = static_cast<int>((d->seq + 127) / 128 * 128 + 128);
    plan->rel_bias = take(static_cast<size_t>(d->heads) * 2 * plan->rel_half * sizeof(float));
    if (d->head_dim > 128) plan->rel_id = take(2 * static_cast<size_t>(plan->rel_half));
  }
  if (d->head_dim <= 128) {
    plan->panels = d->head_dim <= 64 ? 1 : 2;
    const int first = !backward && plan->panels == 1 ? train::kImgK : train::kImgQ, last = backward ? 4 : 3;
    plan->tiles = static_cast<int>((d->seq + 127) / 128 * 2);
    plan->parts = plan->tiles / 2;
    const size_t image = static_cast<size_t>(plan->tiles) * 2 * plan->panels * train::kPanelBytes;
    // The split's grid: one block per 64-row tile (and tensor), below 2^31; the kernels behind it have a CTA per resident one.
    plan->chunk = std::max<long long>(1, std::min<long long>({slices, static_cast<long long>(kMaxImageBytes / ((last - first) * image)),
                                                              0x7fffffffll / (2ll * plan->tiles)}));
    for (int i = first; i < last; ++i) plan->img[i] = take(plan->chunk * image);
    plan->scales = take(plan->chunk * plan->tiles * sizeof(train::TileScale));
    if (backward) plan->rows = take(static_cast<size_t>(plan->chunk) * plan->tiles * train::kRowValues * sizeof(float));
    plan->next = take(4 * sizeof(unsigned));
    if (bias)  // distances beyond seq do not occur
      plan->far = static_cast<int>(std::min<int64_t>(bucket_bounds(bias->buckets, bias->max_distance).at[bias->buckets / 2 - 1], d->seq));
    if (backward && bias) {
      plan->slots = train::dist_slots(plan->far);
      const size_t bytes = size_t{8} * plan->slots * sizeof(float);
      const size_t spare = plan->panels == 1 ? train::kHalfSm - train::tc_smem<1>() : train::kWholeSm - train::tc_smem<2>();
      if (bytes > spare) {
        // Tables of very many distances: fewer CTAs rather than more than 1 GiB.
        plan->dist_ctas = std::max<long long>(1, std::min<long long>(kMaxResident, (1ll << 30) / static_cast<long long>(bytes)));
        plan->dist = take(plan->dist_ctas * bytes);
      }
    }
  } else {
    // Blocks per slice for about eight blocks on each of the 148 SMs (more
    // leaves warps with a row or two, and more partials).
    const long long want = (d->seq + train::kRowWarps - 1) / train::kRowWarps;
    plan->parts = static_cast<int>(std::min(want, std::max<long long>(1, 8 * 148 / slices)));
    if (slices * plan->parts > 0x7fffffffll)
      return fail(RAYA_ATTN_ERR_UNSUPPORTED, "unsupported: %lld CTAs exceed the grid limit", slices * plan->parts);
    if (backward) plan->delta = take(static_cast<size_t>(slices) * d->seq * sizeof(float));
  }
  if (backward && bias) plan->part = take(static_cast<size_t>(slices) * plan->parts * bias->buckets * sizeof(float));
  return RAYA_ATTN_OK;
}

template <typename T>
T* at(void* workspace, size_t offset) {
  return reinterpret_cast<T*>(static_cast<char*>(workspace) + offset);
}

raya_attn_status check_launch(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? RAYA_ATTN_OK : cuda_fail(e, what);
}

// The tensors of a training call, in the order of the entry points.
struct TrainIo {
  const float *q, *k, *v, *out;
  float* out_w;          // forward
  const float* stats;    // backward
  float* stats_w;        // forward, or nullptr
  const float* dout;
  float *dq, *dk, *dv, *dtable;
  const int32_t* valid_len;
};

raya_attn_status launch_rowwise(const TrainPlan& plan, train::TrainArgs t, const float* table,
                                const train::BucketBounds& bounds, void* workspace, cudaStream_t stream, bool backward) {
  const unsigned grid = static_cast<unsigned>(static_cast<long long>(t.a.batch) * t.a.heads * plan.parts);
  if (table) {
    const unsigned blocks = static_cast<unsigned>(std::min<long long>((2ll * plan.rel_half + 255) / 256, 1024));
    train::rel_table_kernel<<<blocks, 256, 0, stream>>>(table, t.a.heads, t.buckets, plan.rel_half, bounds,
                                                        at<float>(workspace, plan.rel_bias), at<uint8_t>(workspace, plan.rel_id));
    const raya_attn_status st = check_launch("bias table launch");
    if (st != RAYA_ATTN_OK) return st;
  }
  if (!backward) {
    train::rowwise_train_fwd<<<grid, train::kRowThreads, 0, stream>>>(t);
    return check_launch("forward launch");
  }
  t.delta = at<float>(workspace, plan.delta);
  const size_t smem = t.part ? static_cast<size_t>(t.buckets) * train::kRowThreads * sizeof(float) : 0;
  train::rowwise_train_dq<<<grid, train::kRowThreads, smem, stream>>>(t);
  const raya_attn_status st = check_launch("query gradient launch");
  if (st != RAYA_ATTN_OK) return st;
  train::rowwise_train_dkv<<<grid, train::kRowThreads, 0, stream>>>(t);
  return check_launch("key gradient launch");
}

// A 3-D tensor map over a [slices][seq][head_dim] fp32 tensor with boxes of
// [1][32 rows][32 floats], 128-byte swizzle: a store clips rows past seq and
// columns past head_dim, a load gives zeros there.
raya_attn_status encode_rows3d(CUtensorMap* map, const float* base, uint64_t head_dim, uint64_t seq, uint64_t slices) {
  raya_attn_status st = load_encoder();
  if (st != RAYA_ATTN_OK) return st;
  const cuuint64_t gdim[3] = {head_dim, seq, slices};
  const cuuint64_t gstride[2] = {head_dim * sizeof(float), seq * head_dim * sizeof(float)};
  const cuuint32_t box[3] = {32, 32, 1};
  const cuuint32_t estride[3] = {1, 1, 1};
  const CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<float*>(base), gdim, gstride, box, estride,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(RAYA_ATTN_ERR_CUDA, "cuda: cuTensorMapEncodeTiled (rows) failed (%d)", static_cast<int>(r));
  return RAYA_ATTN_OK;
}

// A launch that may begin where the one before leaves room (train_common.cuh).
cudaLaunchAttribute early_launch() {
  cudaLaunchAttribute overlap{};
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  return overlap;
}

// Chunk by chunk: the images of its slices, then every 128-row tile of them.
template <int P>
raya_attn_status launch_tc(const TrainPlan& plan, const train::TrainArgs& t, const float* table, const train::BucketBounds& bounds,
                           void* workspace, int sms, cudaStream_t stream, bool backward) {
  train::TcArgs c{};
  c.t = t;
  c.tiles = plan.tiles;
  c.first_image = !backward && P == 1 ? train::kImgK : train::kImgQ;
  for (int i = c.first_image; i < (backward ? 4 : 3); ++i) c.img[i] = at<uint8_t>(workspace, plan.img[i]);
  c.scales = at<train::TileScale>(workspace, plan.scales);
  if (backward) c.rows = at<float>(workspace, plan.rows);
  c.next = at<unsigned>(workspace, plan.next);
  c.table = table;
  c.vec = at<float>(workspace, plan.rel_bias);
  c.bounds = bounds;
  c.far = plan.far;
  const size_t smem = train::tc_smem<P>();
  size_t dist = 0;
  if (t.part) {
    c.slots = plan.slots;
    if (plan.dist_ctas > 0)
      c.dist = at<float>(workspace, plan.dist);
    else
      dist = size_t{8} * plan.slots * sizeof(float);
  }
  const long long resident = std::min(kMaxResident, static_cast<long long>(sms) * (P == 1 ? 2 : 1));
  const bool bias = t.rel_bias != nullptr;
  const long long slices = static_cast<long long>(t.a.batch) * t.a.heads;
  for (c.slice0 = 0; c.slice0 < slices; c.slice0 += plan.chunk) {
    const long long n = std::min(plan.chunk, slices - c.slice0) * plan.tiles;
    c.units = static_cast<unsigned>(n / 2);
    const dim3 split_grid(static_cast<unsigned>(n), (backward ? 4 : 3) - c.first_image + (bias ? 1 : 0));
    if (backward)
      train::split_kernel<P, true><<<split_grid, 256, 0, stream>>>(c);
    else
      train::split_kernel<P, false><<<split_grid, 256, 0, stream>>>(c);
    raya_attn_status st = check_launch("operand split launch");
    if (st != RAYA_ATTN_OK) return st;
    auto launch_kind = [&](void (*fn)(train::TcArgs, CUtensorMap, CUtensorMap), size_t shared, long long ctas, float* out, const char* what) {
      CUtensorMap map, q_map{};
      raya_attn_status encoded = encode_rows3d(&map, out, t.a.head_dim, t.a.seq, slices);
      if (encoded == RAYA_ATTN_OK && c.first_image == train::kImgK)
        encoded = encode_rows3d(&q_map, t.a.q, t.a.head_dim, t.a.seq, slices);
      if (encoded != RAYA_ATTN_OK) return encoded;
      cudaLaunchAttribute overlap = early_launch();
      cudaLaunchConfig_t config{};
      config.gridDim = dim3(static_cast<unsigned>(std::min(n / 2, ctas)));
      config.blockDim = dim3(train::tc_threads(P));
      config.dynamicSmemBytes = shared;
      config.stream = stream;
      config.attrs = &overlap;
      config.numAttrs = 1;
      const cudaError_t e = cudaLaunchKernelEx(&config, fn, c, map, q_map);
      return e == cudaSuccess ? check_launch(what) : cuda_fail(e, what);
    };
    using train::tc_train;
    if (!backward) {
      st = launch_kind(bias ? tc_train<train::kForward, P, true> : tc_train<train::kForward, P, false>, smem, resident, t.a.out, "forward launch");
      if (st != RAYA_ATTN_OK) return st;
      continue;
    }
    st = launch_kind(t.part  ? tc_train<train::kDq, P, true, true>
                     : bias ? tc_train<train::kDq, P, true>
                            : tc_train<train::kDq, P, false>,
                     smem + dist, c.dist ? std::min(resident, plan.dist_ctas) : resident, t.dq, "query gradient launch");
    if (st == RAYA_ATTN_OK)
      st = launch_kind(bias ? tc_train<train::kDk, P, true> : tc_train<train::kDk, P, false>, smem, resident, t.dk, "key gradient launch");
    if (st == RAYA_ATTN_OK)
      st = launch_kind(bias ? tc_train<train::kDv, P, true> : tc_train<train::kDv, P, false>, smem, resident, t.dv, "value gradient launch");
    if (st != RAYA_ATTN_OK) return st;
  }
  return RAYA_ATTN_OK;
}

raya_attn_status train_call(const raya_attn_desc* d, const TrainIo& io, const raya_attn_bias* bias, void* workspace,
                            size_t workspace_bytes, cudaStream_t stream, bool backward) {
  TrainPlan plan;
  raya_attn_status st = train_plan(d, bias, backward, &plan);
  if (st != RAYA_ATTN_OK) return st;
  if (!bias && io.dtable) return fail(RAYA_ATTN_ERR_SHAPE, "invalid shape: dtable without a bias");
  if (bias && !bias->table) return fail(RAYA_ATTN_ERR_SHAPE, "invalid shape: null bias table");
  if (d->seq == 0) {  // no rows; a gradient over none is zero
    if (!io.dtable) return RAYA_ATTN_OK;
    const cudaError_t e = cudaMemsetAsync(io.dtable, 0, static_cast<size_t>(d->heads) * bias->buckets * sizeof(float), stream);
    return e == cudaSuccess ? RAYA_ATTN_OK : cuda_fail(e, "cudaMemsetAsync(dtable)");
  }
  const void* used[] = {io.q, io.k, io.v, backward ? io.out : io.out_w, backward ? io.stats : io.q,
                        backward ? io.dout : io.q, backward ? io.dq : io.q, backward ? io.dk : io.q,
                        backward ? io.dv : io.q};
  for (const void* p : used)
    if (!p) return fail(RAYA_ATTN_ERR_SHAPE, "invalid shape: null tensor pointer");
  for (const void* p : used)
    if (p != io.stats && !aligned16(p))
      return fail(RAYA_ATTN_ERR_UNSUPPORTED, "unsupported: tensors must be 16-byte aligned");
  const float* stats = backward ? io.stats : io.stats_w;
  if ((reinterpret_cast<uintptr_t>(stats) & 7u) != 0)
    return fail(RAYA_ATTN_ERR_UNSUPPORTED, "unsupported: stats must be 8-byte aligned");
  if (plan.bytes > 0 && (!workspace || workspace_bytes < plan.bytes))
    return fail_length("workspace", workspace ? workspace_bytes : 0, plan.bytes);
  if (workspace && !aligned16(workspace))
    return fail(RAYA_ATTN_ERR_UNSUPPORTED, "unsupported: the workspace must be 16-byte aligned");
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  DeviceCtx* ctx = nullptr;
  st = ensure_ready(dev, &ctx);
  if (st != RAYA_ATTN_OK) return st;

  train::TrainArgs t{};
  t.a = make_args(d, io.q, io.k, io.v, backward ? const_cast<float*>(io.out) : io.out_w, io.valid_len, ctx->status);
  t.scale = d->scale;
  t.stats = reinterpret_cast<const float2*>(io.stats);
  t.stats_out = reinterpret_cast<float2*>(io.stats_w);
  t.dout = io.dout;
  t.dq = io.dq;
  t.dk = io.dk;
  t.dv = io.dv;
  t.parts = plan.parts;
  train::BucketBounds bounds{};
  if (bias) {
    bounds = bucket_bounds(bias->buckets, bias->max_distance);
    t.rel_half = plan.rel_half;
    t.buckets = bias->buckets;
    t.rel_bias = at<float>(workspace, plan.rel_bias);
    if (plan.panels == 0) t.rel_id = at<uint8_t>(workspace, plan.rel_id);
  }
  if (io.dtable) t.part = at<float>(workspace, plan.part);
  if (plan.panels > 0)
    st = plan.panels == 1 ? launch_tc<1>(plan, t, bias ? bias->table : nullptr, bounds, workspace, ctx->sms, stream, backward)
                          : launch_tc<2>(plan, t, bias ? bias->table : nullptr, bounds, workspace, ctx->sms, stream, backward);
  else
    st = launch_rowwise(plan, t, bias ? bias->table : nullptr, bounds, workspace, stream, backward);
  if (st != RAYA_ATTN_OK) return st;
  if (io.dtable) {
    cudaLaunchAttribute overlap = early_launch();
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(d->heads), static_cast<unsigned>(bias->buckets));
    config.blockDim = dim3(256);
    config.stream = stream;
    config.attrs = &overlap;
    config.numAttrs = 1;
    const cudaError_t launched = cudaLaunchKernelEx(&config, train::bias_grad_kernel, static_cast<const float*>(t.part), static_cast<int>(d->batch),
                                                    static_cast<int>(d->heads), plan.parts, static_cast<int>(bias->buckets), io.dtable);
    st = launched == cudaSuccess ? check_launch("bias gradient launch") : cuda_fail(launched, "bias gradient launch");
  }
  return st;
}
