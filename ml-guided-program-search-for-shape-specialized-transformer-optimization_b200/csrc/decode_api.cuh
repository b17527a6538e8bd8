// decode_api.cuh -- argument checks and launches of the decoding operators:
// norm and rotation of queries and keys, the 8-bit key/value cache, and 4-bit
// linear layers.  Part of b200tx.cu's translation unit.
#pragma once

namespace {

constexpr int64_t kRopeManyTokens = 4096;
constexpr int kRopeChunks = 4;
constexpr int64_t kKv8ShortSteps = 24;

// Values a lane: eight of bf16, four of fp32 (16 bytes; 25 x 420 tokens of 6 heads of 64
// in fp32: four 8.0 us, eight 13.7), four of bf16 where the pairs' halves do not lie
// eight apart, eight of fp32 for head_dim 256 (a head is at most one warp).
bool eight_values(const b200tx::RopeTable& rope, int dtype, int64_t head_dim) {
  if (head_dim == 256) return true;
  return dtype == B200TX_BF16 && (rope.cos == nullptr || rope.interleaved || rope.rotary % 16 == 0);
}

int rope_table(const char* what, const b200tx_rope* rope, int64_t head_dim, b200tx::RopeTable* out) {
  *out = b200tx::RopeTable{};
  if (rope == nullptr) return B200TX_OK;
  if (rope->cos == nullptr || rope->sin == nullptr || rope->positions <= 0 || rope->positions > 0x7fffffffLL)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "%s: bad rotation table", what);
  if (!aligned16(rope->cos) || !aligned16(rope->sin))
    return fail(B200TX_ERR_INVALID_ARGUMENT, "%s: the rotation tables must be 16-byte aligned", what);
  const int64_t step = head_dim == 256 ? 16 : 8;
  if (rope->rotary <= 0 || rope->rotary > head_dim || rope->rotary % step != 0)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "%s: rotary %lld is not a multiple of %lld up to head_dim %lld", what,
                (long long)rope->rotary, (long long)step, (long long)head_dim);
  out->cos = rope->cos;
  out->sin = rope->sin;
  out->positions = static_cast<int>(rope->positions);
  out->rotary = static_cast<int>(rope->rotary);
  out->interleaved = rope->interleaved != 0;
  return B200TX_OK;
}

int heads_shape(const char* what, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads) {
  if (batch <= 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || batch > (1 << 20) || tokens > (1 << 26) ||
      heads > (1 << 14) || kv_heads > heads)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "%s: bad shape batch %lld tokens %lld heads %lld kv_heads %lld", what,
                (long long)batch, (long long)tokens, (long long)heads, (long long)kv_heads);
  return B200TX_OK;
}

int kv8_view(const char* what, const b200tx_kv8_cache* c, b200tx::Kv8Cache* out) {
  if (c == nullptr || c->codes == nullptr || c->scales == nullptr || c->tail == nullptr || c->page_table == nullptr ||
      c->lengths == nullptr)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "%s: null cache pointer", what);
  if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail(B200TX_ERR_UNSUPPORTED, "%s: head_dim %lld (32, 64, 128 and 256 are built)", what,
                (long long)c->head_dim);
  if (c->pages <= 0 || c->pages > 0x7fffffffLL || c->slots <= 0 || c->slots > (1 << 20) || c->max_blocks <= 0 ||
      c->max_blocks > 0x7fffffffLL / b200tx::kKv8Block || c->kv_heads <= 0 || c->kv_heads > (1 << 14))
    return fail(B200TX_ERR_INVALID_ARGUMENT, "%s: bad cache shape", what);
  if (!aligned16(c->codes) || !aligned16(c->tail))
    return fail(B200TX_ERR_INVALID_ARGUMENT, "%s: the cache's codes and tail must be 16-byte aligned", what);
  out->codes = static_cast<uint8_t*>(c->codes);
  out->scales = c->scales;
  out->tail = static_cast<__nv_bfloat16*>(c->tail);
  out->page_table = c->page_table;
  out->lengths = c->lengths;
  out->pages = c->pages;
  out->slots = static_cast<int>(c->slots);
  out->max_blocks = static_cast<int>(c->max_blocks);
  out->kv_heads = static_cast<int>(c->kv_heads);
  return B200TX_OK;
}

// Chunks of heads for a warp: one, for the shortest step, or where there are
// tokens enough to fill the SMs several, so that angles and factors are made
// fewer times (append of 4 x 4000 tokens: one 114 us, four 103; 2 x 5776 tokens of
// 48 heads of 64: one 35.8 us, four 31.9).
int rope_chunks(int64_t tokens) { return tokens >= kRopeManyTokens ? kRopeChunks : 1; }

template <int D, int E, typename T>
cudaError_t launch_rope(b200tx::RopeArgs& a, cudaStream_t stream) {
  a.chunks = rope_chunks(a.total_tokens);
  const int64_t rounds = b200tx::rope_rounds<D, E>(a.heads, a.chunks) +
                         (a.copy_values ? 2 : 1) * b200tx::rope_rounds<D, E>(a.kv_heads, a.chunks);
  const int64_t ctas = (a.total_tokens + b200tx::kRopeWarps - 1) / b200tx::kRopeWarps * rounds;
  return launch(b200tx::qk_norm_rope_kernel<D, E, T>, dim3(static_cast<unsigned>(ctas)), dim3(b200tx::kRopeWarps * 32), 0,
                stream, a);
}

cudaError_t launch_rope_dim(int64_t head_dim, int dtype, b200tx::RopeArgs& a, cudaStream_t stream) {
  using bf16 = __nv_bfloat16;
  if (eight_values(a.norm.rope, dtype, head_dim)) {
    switch (head_dim) {
      case 8: return launch_rope<8, 8, bf16>(a, stream);
      case 16: return launch_rope<16, 8, bf16>(a, stream);
      case 32: return launch_rope<32, 8, bf16>(a, stream);
      case 64: return launch_rope<64, 8, bf16>(a, stream);
      case 128: return launch_rope<128, 8, bf16>(a, stream);
      default: return dtype == B200TX_F32 ? launch_rope<256, 8, float>(a, stream) : launch_rope<256, 8, bf16>(a, stream);
    }
  }
  const bool f32 = dtype == B200TX_F32;
  switch (head_dim) {
    case 8: return f32 ? launch_rope<8, 4, float>(a, stream) : launch_rope<8, 4, bf16>(a, stream);
    case 16: return f32 ? launch_rope<16, 4, float>(a, stream) : launch_rope<16, 4, bf16>(a, stream);
    case 32: return f32 ? launch_rope<32, 4, float>(a, stream) : launch_rope<32, 4, bf16>(a, stream);
    case 64: return f32 ? launch_rope<64, 4, float>(a, stream) : launch_rope<64, 4, bf16>(a, stream);
    default: return f32 ? launch_rope<128, 4, float>(a, stream) : launch_rope<128, 4, bf16>(a, stream);
  }
}

template <int D, int E, typename T>
cudaError_t launch_kv8_append(b200tx::Kv8AppendArgs& a, cudaStream_t stream) {
  a.chunks = rope_chunks(static_cast<int64_t>(a.batch) * a.tokens);
  const int64_t units = static_cast<int64_t>(a.batch) * a.tokens * b200tx::rope_rounds<D, E>(a.heads, a.chunks);
  const int64_t q_ctas = (units + b200tx::kKv8AppendWarps - 1) / b200tx::kKv8AppendWarps;
  return launch(b200tx::kv8_append_kernel<D, E, T>, dim3(static_cast<unsigned>(a.kv_ctas + q_ctas)),
                dim3(b200tx::kKv8AppendWarps * 32), 0, stream, a);
}

cudaError_t launch_kv8_append_dim(int64_t head_dim, int dtype, b200tx::Kv8AppendArgs& a, cudaStream_t stream) {
  using bf16 = __nv_bfloat16;
  if (eight_values(a.norm.rope, dtype, head_dim)) {
    switch (head_dim) {
      case 32: return launch_kv8_append<32, 8, bf16>(a, stream);
      case 64: return launch_kv8_append<64, 8, bf16>(a, stream);
      case 128: return launch_kv8_append<128, 8, bf16>(a, stream);
      default: return dtype == B200TX_F32 ? launch_kv8_append<256, 8, float>(a, stream) : launch_kv8_append<256, 8, bf16>(a, stream);
    }
  }
  const bool f32 = dtype == B200TX_F32;
  switch (head_dim) {
    case 32: return f32 ? launch_kv8_append<32, 4, float>(a, stream) : launch_kv8_append<32, 4, bf16>(a, stream);
    case 64: return f32 ? launch_kv8_append<64, 4, float>(a, stream) : launch_kv8_append<64, 4, bf16>(a, stream);
    default: return f32 ? launch_kv8_append<128, 4, float>(a, stream) : launch_kv8_append<128, 4, bf16>(a, stream);
  }
}

template <int D>
cudaError_t launch_kv8_gather(b200tx::Kv8GatherArgs& a, cudaStream_t stream) {
  const int64_t threads = static_cast<int64_t>(a.most) * a.cache.kv_heads * (D / 8);
  a.ctas = static_cast<int>((threads + 255) / 256);
  return launch(b200tx::kv8_gather_kernel<D>, dim3(static_cast<unsigned>(a.ctas) * static_cast<unsigned>(a.batch)),
                dim3(256), 0, stream, a);
}

// The workspace of the attention: arrival counters, then the parts of tiles
// that lie in two or more CTAs.
constexpr int64_t kKv8ArrivalBytes = B200TX_KV8_COUNTER_BYTES;

template <int D, int NR>
int kv8_attention_grid(int sm_count) {
  return sm_count * b200tx::Kv8Shape<D, NR>::CTAS;
}

template <int D, int NR>
int64_t kv8_part_bytes(int sm_count) {
  return static_cast<int64_t>(kv8_attention_grid<D, NR>(sm_count)) * 2 * b200tx::Kv8Shape<D, NR>::PART_FLOATS * 4;
}

// Row groups of 8 in a tile, for which a code is expanded once: up to 4 where the
// outputs of 32 rows fit in the registers (head_dim 32 and 64), 2 for 128, 1 for 256.
// Where tiles of 8 rows are short work even for a full cache, 24 steps a CTA, one:
// their beginning and join take less (64 rows: 4 x 2 heads of 128 over 3001 tokens, 20
// steps, one 12.3 us, two 15.3; over 12000, 81 steps, 34.9 and 30.8; 4 x 2 heads of 64 over
// 3001, 7 steps, one 12.2 us, four 14.7; 8 x 4 of 64 over 3000, 27 steps, 22.8 and 20.7).
int kv8_row_groups(int64_t head_dim, int64_t rows, int64_t sequence_heads, int64_t max_blocks, int sm_count) {
  if (rows <= 8 || head_dim == 256) return 1;
  const int64_t steps = sequence_heads * ((rows + 7) / 8) * max_blocks * (head_dim == 128 ? 2 : 1);
  const int ctas = head_dim == 128   ? kv8_attention_grid<128, 1>(sm_count)
                   : head_dim == 64 ? kv8_attention_grid<64, 1>(sm_count)
                                    : kv8_attention_grid<32, 1>(sm_count);
  if (steps <= kKv8ShortSteps * ctas) return 1;
  if (rows <= 16 || head_dim == 128) return 2;
  return 4;
}

template <int D>
int64_t kv8_workspace(int sm_count) {
  int64_t most = kv8_part_bytes<D, 1>(sm_count);
  if constexpr (D <= 128) most = std::max(most, kv8_part_bytes<D, 2>(sm_count));
  if constexpr (D <= 64) most = std::max(most, kv8_part_bytes<D, 4>(sm_count));
  return kKv8ArrivalBytes + most;
}

template <int D, int NR>
cudaError_t launch_kv8_attention(b200tx::Kv8AttnArgs& a, DeviceState* dev, int index, cudaStream_t stream) {
  using S = b200tx::Kv8Shape<D, NR>;
  if (!dev->kv8_attr[index]) {
    cudaError_t err =
        cudaFuncSetAttribute(b200tx::kv8_attention_kernel<D, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::MAIN);
    if (err != cudaSuccess) return err;
    dev->kv8_attr[index] = true;
  }
  return launch(b200tx::kv8_attention_kernel<D, NR>, dim3(static_cast<unsigned>(kv8_attention_grid<D, NR>(dev->sm_count))),
                dim3(b200tx::kKv8Warps * 32), S::MAIN, stream, a);
}

template <int TN, int RT, int GROUP>
cudaError_t launch_w4(b200tx::W4Args& a, DeviceState* dev, int index, cudaStream_t stream) {
  constexpr int kMost = 112 * 1024;  // two CTAs for each SM
  if (!dev->w4_attr[index]) {
    cudaError_t err = cudaFuncSetAttribute(b200tx::linear_w4_kernel<TN, RT, GROUP>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (err != cudaSuccess) return err;
    dev->w4_attr[index] = true;
  }
  // Slices of K: the fewest (they are joined at the end) that give most SMs a second
  // CTA (1 x 8192 -> 8192: 128 CTAs 20.3 us, 256 CTAs 15.9; 8 x 8192 -> 28672:
  // 224 CTAs 38.6 us, 448 CTAs 41.9).
  const int tiles = (a.outer + 16 * RT - 1) / (16 * RT), all_stages = (a.runs + b200tx::kW4Runs - 1) / b200tx::kW4Runs;
  a.slices = 1;
  while (a.slices < b200tx::kW4Warps && a.slices < all_stages &&
         (tiles * a.slices + b200tx::kW4Warps - 1) / b200tx::kW4Warps < dev->sm_count * 5 / 4 &&
         2 * b200tx::w4_stage_bytes<TN, RT>(2 * a.slices) <= kMost)
    a.slices *= 2;
  const int stage = b200tx::w4_stage_bytes<TN, RT>(a.slices);
  a.stages = 4 * stage <= kMost ? 4 : 3 * stage <= kMost ? 3 : 2;
  const int join = b200tx::kW4Warps * RT * TN * 512;
  const int per = b200tx::kW4Warps / a.slices;
  const dim3 grid(static_cast<unsigned>((tiles + per - 1) / per), static_cast<unsigned>((a.rows + TN * 8 - 1) / (TN * 8)));
  return launch(b200tx::linear_w4_kernel<TN, RT, GROUP>, grid, dim3(b200tx::kW4Warps * 32),
                static_cast<size_t>(std::max(a.stages * stage, join)), stream, a);
}

constexpr int64_t kW4GridRows = 65535;     // of x tiles: the grid's second dimension
constexpr int kW4LineShared = 227 * 1024;  // of a CTA that has an SM to itself
constexpr int64_t kW4LineUnits = 48;       // (16 columns, stage) units for each SM

template <int TN, int GROUP>
cudaError_t launch_w4_line(b200tx::W4Args& a, DeviceState* dev, int index, cudaStream_t stream) {
  if (!dev->w4_line_attr[index]) {
    cudaError_t err = cudaFuncSetAttribute(b200tx::linear_w4_line_kernel<TN, GROUP>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize, kW4LineShared);
    if (err != cudaSuccess) return err;
    dev->w4_line_attr[index] = true;
  }
  const int all_stages = (a.runs + b200tx::kW4Runs - 1) / b200tx::kW4Runs;
  const int x_bytes = a.rows * all_stages * b200tx::kW4Runs * b200tx::kW4Run * 2;
  const int stage = b200tx::kW4LineWarps * b200tx::kW4LineStage;
  a.stages = x_bytes + 4 * stage <= kW4LineShared ? 4 : 3;
  return launch(b200tx::linear_w4_line_kernel<TN, GROUP>, dim3(static_cast<unsigned>(std::min(dev->sm_count, (a.outer + 15) / 16))),
                dim3(b200tx::kW4LineWarps * 32), static_cast<size_t>(x_bytes + a.stages * stage), stream, a);
}

template <int TN>
cudaError_t launch_w4_line_group(int64_t group, b200tx::W4Args& a, DeviceState* dev, int index, cudaStream_t stream) {
  switch (group) {
    case 32: return launch_w4_line<TN, 32>(a, dev, index, stream);
    case 64: return launch_w4_line<TN, 64>(a, dev, index + 1, stream);
    default: return launch_w4_line<TN, 128>(a, dev, index + 2, stream);
  }
}

// The kernel with x in shared memory, where x and three stages for each warp fit and
// there are units enough for its warps (8 x 8192 -> 28672, 387 units an SM: 31.2 us
// against 38.2; 16 x 4096 -> 14336, 97: 15.4 against 16.2; 1 x 4096 -> 4096, 28: 5.74 against
// 5.64; 1 x 1024 -> 4096, 7: 4.8 against 3.3).
bool w4_in_line(const b200tx::W4Args& a, const DeviceState* dev) {
  const int64_t all_stages = (a.runs + b200tx::kW4Runs - 1) / b200tx::kW4Runs;
  return a.rows <= 16 && a.rows * all_stages * b200tx::kW4Runs * b200tx::kW4Run * 2 +
                                 3 * b200tx::kW4LineWarps * b200tx::kW4LineStage <= kW4LineShared &&
         (a.outer + 15) / 16 * all_stages >= kW4LineUnits * dev->sm_count;
}

template <int TN, int RT>
cudaError_t launch_w4_group(int64_t group, b200tx::W4Args& a, DeviceState* dev, int index, cudaStream_t stream) {
  switch (group) {
    case 32: return launch_w4<TN, RT, 32>(a, dev, index, stream);
    case 64: return launch_w4<TN, RT, 64>(a, dev, index + 1, stream);
    default: return launch_w4<TN, RT, 128>(a, dev, index + 2, stream);
  }
}

// Column tiles of a warp: two, sharing the x fragments, where the columns are many
// (8 x 4096 -> 14336: one 13.8 us, two 12.9; 1 x 8192 -> 8192: one 15.9, two 18.9) and the
// accumulators fit (32 x 4096 -> 14336: one 24.9 us, two 43.1).
template <int TN>
cudaError_t launch_w4_tiles(int64_t group, b200tx::W4Args& a, DeviceState* dev, int index, cudaStream_t stream) {
  if constexpr (TN <= 2) {
    if (a.outer >= 80 * dev->sm_count) return launch_w4_group<TN, 2>(group, a, dev, index, stream);
  }
  return launch_w4_group<TN, 1>(group, a, dev, index + 3, stream);
}

}  // namespace

extern "C" {

int b200tx_qk_norm_rope(const void* qkv, void* out, int dtype, int64_t batch, int64_t tokens, int64_t heads,
                        int64_t kv_heads, int64_t head_dim, int64_t in_batch_stride, int64_t in_token_stride,
                        int64_t out_batch_stride, int64_t out_token_stride, const float* q_weight,
                        const float* k_weight, float eps, const b200tx_rope* rope, const void* positions,
                        int positions_64, int64_t position_batch_stride, cudaStream_t stream) {
  if (qkv == nullptr || out == nullptr)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "qk_norm_rope: null tensor pointer");
  int rc = heads_shape("qk_norm_rope", batch, tokens, heads, kv_heads);
  if (rc != B200TX_OK) return rc;
  if (head_dim < 8 || head_dim > 256 || (head_dim & (head_dim - 1)) != 0)
    return fail(B200TX_ERR_UNSUPPORTED, "qk_norm_rope: head_dim %lld (8, 16, 32, 64, 128 and 256 are built)",
                (long long)head_dim);
  if (dtype != B200TX_F32 && dtype != B200TX_BF16)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "qk_norm_rope: dtype %d", dtype);
  if (!aligned16(qkv) || !aligned16(out) || (in_batch_stride | in_token_stride | out_batch_stride | out_token_stride) % 8 != 0)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "qk_norm_rope: pointers must be 16-byte aligned, strides multiples of 8");
  if ((q_weight != nullptr && !aligned16(q_weight)) || (k_weight != nullptr && !aligned16(k_weight)))
    return fail(B200TX_ERR_INVALID_ARGUMENT, "qk_norm_rope: the norm weights must be 16-byte aligned");
  b200tx::RopeArgs a{};
  rc = rope_table("qk_norm_rope", rope, head_dim, &a.norm.rope);
  if (rc != B200TX_OK) return rc;
  DeviceState* dev = nullptr;
  rc = current_device(&dev);
  if (rc != B200TX_OK) return rc;
  a.in = qkv;
  a.out = out;
  a.in_batch_stride = in_batch_stride;
  a.in_token_stride = in_token_stride;
  a.out_batch_stride = out_batch_stride;
  a.out_token_stride = out_token_stride;
  a.positions = positions;
  a.positions_64 = positions_64;
  a.position_batch_stride = position_batch_stride;
  a.tokens = static_cast<int>(tokens);
  a.heads = static_cast<int>(heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.copy_values = out != qkv;
  a.total_tokens = batch * tokens;
  a.norm.q_weight = q_weight;
  a.norm.k_weight = k_weight;
  a.norm.eps = eps;
  if (static_cast<double>(a.total_tokens) * (heads + 2 * kv_heads) > 2147483647.0)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "qk_norm_rope: too many tokens");
  cudaError_t err = launch_rope_dim(head_dim, dtype, a, stream);
  return err == cudaSuccess ? B200TX_OK : cuda_fail(err, "qk_norm_rope");
}

int b200tx_kv8_append(const b200tx_kv8_cache* cache, const void* qkv, int dtype, void* q_out, int64_t batch,
                      int64_t tokens, int64_t heads, int64_t batch_stride, int64_t token_stride,
                      const int32_t* slot_ids, const int32_t* counts, const float* q_weight, const float* k_weight,
                      float eps, const b200tx_rope* rope, cudaStream_t stream) {
  b200tx::Kv8AppendArgs a{};
  int rc = kv8_view("kv8_append", cache, &a.cache);
  if (rc != B200TX_OK) return rc;
  if (qkv == nullptr || q_out == nullptr) return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_append: null tensor pointer");
  rc = heads_shape("kv8_append", batch, tokens, heads, cache->kv_heads);
  if (rc != B200TX_OK) return rc;
  if (dtype != B200TX_F32 && dtype != B200TX_BF16)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_append: dtype %d", dtype);
  if (!aligned16(qkv) || !aligned16(q_out) || (batch_stride | token_stride) % 8 != 0)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_append: pointers must be 16-byte aligned, strides multiples of 8");
  if ((q_weight != nullptr && !aligned16(q_weight)) || (k_weight != nullptr && !aligned16(k_weight)))
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_append: the norm weights must be 16-byte aligned");
  if (slot_ids == nullptr && batch > cache->slots)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_append: batch %lld in a cache of %lld slots", (long long)batch,
                (long long)cache->slots);
  rc = rope_table("kv8_append", rope, cache->head_dim, &a.norm.rope);
  if (rc != B200TX_OK) return rc;
  DeviceState* dev = nullptr;
  rc = current_device(&dev);
  if (rc != B200TX_OK) return rc;
  a.qkv = qkv;
  a.q_out = static_cast<__nv_bfloat16*>(q_out);
  a.batch_stride = batch_stride;
  a.token_stride = token_stride;
  a.slot_ids = slot_ids;
  a.counts = counts;
  a.batch = static_cast<int>(batch);
  a.tokens = static_cast<int>(tokens);
  a.heads = static_cast<int>(heads);
  a.block_span = static_cast<int>((tokens + b200tx::kKv8Block - 2) / b200tx::kKv8Block + 1);
  a.kv_ctas = batch * cache->kv_heads * a.block_span;
  a.norm.q_weight = q_weight;
  a.norm.k_weight = k_weight;
  a.norm.eps = eps;
  if (static_cast<double>(batch) * tokens * heads > 1073741823.0 || a.kv_ctas > 0x3fffffffLL)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_append: too many tokens");
  cudaError_t err = launch_kv8_append_dim(cache->head_dim, dtype, a, stream);
  return err == cudaSuccess ? B200TX_OK : cuda_fail(err, "kv8_append");
}

int b200tx_kv8_gather(const b200tx_kv8_cache* cache, void* k_out, void* v_out, int64_t batch, int64_t most,
                      int64_t tokens, const int32_t* slot_ids, const int32_t* counts, cudaStream_t stream) {
  b200tx::Kv8GatherArgs a{};
  int rc = kv8_view("kv8_gather", cache, &a.cache);
  if (rc != B200TX_OK) return rc;
  if (k_out == nullptr || v_out == nullptr || !aligned16(k_out) || !aligned16(v_out))
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_gather: outputs must be 16-byte aligned");
  if (batch <= 0 || batch > (1 << 20) || most <= 0 || most > 0x7fffffffLL || tokens < 0 || tokens > (1 << 26))
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_gather: bad shape batch %lld tokens %lld", (long long)batch,
                (long long)most);
  if (slot_ids == nullptr && batch > cache->slots)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_gather: batch %lld in a cache of %lld slots", (long long)batch,
                (long long)cache->slots);
  if (static_cast<double>(batch) * most * cache->kv_heads * (cache->head_dim / 8) > 2147483647.0)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_gather: too many values");
  DeviceState* dev = nullptr;
  rc = current_device(&dev);
  if (rc != B200TX_OK) return rc;
  a.slot_ids = slot_ids;
  a.counts = counts;
  a.tokens = static_cast<int>(tokens);
  a.batch = static_cast<int>(batch);
  a.most = static_cast<int>(most);
  a.k = static_cast<__nv_bfloat16*>(k_out);
  a.v = static_cast<__nv_bfloat16*>(v_out);
  cudaError_t err;
  switch (cache->head_dim) {
    case 32: err = launch_kv8_gather<32>(a, stream); break;
    case 64: err = launch_kv8_gather<64>(a, stream); break;
    case 128: err = launch_kv8_gather<128>(a, stream); break;
    default: err = launch_kv8_gather<256>(a, stream); break;
  }
  return err == cudaSuccess ? B200TX_OK : cuda_fail(err, "kv8_gather");
}

int b200tx_kv8_workspace_bytes(int64_t head_dim, int64_t* bytes_out) {
  if (bytes_out == nullptr) return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_workspace_bytes: null result");
  DeviceState* dev = nullptr;
  int rc = current_device(&dev);
  if (rc != B200TX_OK) return rc;
  switch (head_dim) {
    case 32: *bytes_out = kv8_workspace<32>(dev->sm_count); return B200TX_OK;
    case 64: *bytes_out = kv8_workspace<64>(dev->sm_count); return B200TX_OK;
    case 128: *bytes_out = kv8_workspace<128>(dev->sm_count); return B200TX_OK;
    case 256: *bytes_out = kv8_workspace<256>(dev->sm_count); return B200TX_OK;
    default: return fail(B200TX_ERR_UNSUPPORTED, "kv8_workspace_bytes: head_dim %lld", (long long)head_dim);
  }
}

int b200tx_kv8_attention(const b200tx_kv8_cache* cache, const void* q, void* out, int64_t batch, int64_t tokens,
                         int64_t heads, int64_t q_batch_stride, int64_t q_token_stride, const int32_t* slot_ids,
                         const int32_t* counts, float scale, void* workspace, int64_t workspace_bytes,
                         cudaStream_t stream) {
  b200tx::Kv8AttnArgs a{};
  int rc = kv8_view("kv8_attention", cache, &a.cache);
  if (rc != B200TX_OK) return rc;
  if (q == nullptr || out == nullptr || workspace == nullptr)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_attention: null tensor pointer");
  rc = heads_shape("kv8_attention", batch, tokens, heads, cache->kv_heads);
  if (rc != B200TX_OK) return rc;
  if (heads % cache->kv_heads != 0)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_attention: %lld heads do not share %lld kv heads evenly",
                (long long)heads, (long long)cache->kv_heads);
  if (tokens * heads > (1 << 26)) return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_attention: too many query rows");
  if (!aligned16(q) || !aligned16(out) || !aligned16(workspace) || (q_batch_stride | q_token_stride) % 8 != 0)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_attention: pointers must be 16-byte aligned, strides multiples of 8");
  if (!(scale > 0.f) || scale > 1e30f) return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_attention: scale must be positive");
  if (slot_ids == nullptr && batch > cache->slots)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_attention: batch %lld in a cache of %lld slots", (long long)batch,
                (long long)cache->slots);
  DeviceState* dev = nullptr;
  rc = current_device(&dev);
  if (rc != B200TX_OK) return rc;
  int64_t need = 0;
  rc = b200tx_kv8_workspace_bytes(cache->head_dim, &need);
  if (rc != B200TX_OK) return rc;
  if (workspace_bytes < need)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_attention: workspace of %lld bytes, %lld needed",
                (long long)workspace_bytes, (long long)need);
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.q_batch_stride = q_batch_stride;
  a.q_token_stride = q_token_stride;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.slot_ids = slot_ids;
  a.counts = counts;
  a.batch = static_cast<int>(batch);
  a.tokens = static_cast<int>(tokens);
  a.heads = static_cast<int>(heads);
  a.group = static_cast<int>(heads / cache->kv_heads);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.arrivals = static_cast<unsigned int*>(workspace);
  a.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kKv8ArrivalBytes);
  cudaError_t err;
  const int groups =
      kv8_row_groups(cache->head_dim, tokens * a.group, batch * cache->kv_heads, cache->max_blocks, dev->sm_count);
  // all steps of the longest sequences that the page table can hold, and the tiles' own cost
  const double units = static_cast<double>(batch) * cache->kv_heads * ((tokens * a.group + 8 * groups - 1) / (8 * groups)) *
                       (4.0 * cache->max_blocks + 8 + b200tx::kKv8TileCost);
  if (units >= 4294967296.0)
    return fail(B200TX_ERR_UNSUPPORTED, "kv8_attention: batch x heads x rows x blocks of this call pass 2^32 steps");
  switch (cache->head_dim + groups) {
    case 33: err = launch_kv8_attention<32, 1>(a, dev, 0, stream); break;
    case 34: err = launch_kv8_attention<32, 2>(a, dev, 1, stream); break;
    case 36: err = launch_kv8_attention<32, 4>(a, dev, 2, stream); break;
    case 65: err = launch_kv8_attention<64, 1>(a, dev, 3, stream); break;
    case 66: err = launch_kv8_attention<64, 2>(a, dev, 4, stream); break;
    case 68: err = launch_kv8_attention<64, 4>(a, dev, 5, stream); break;
    case 129: err = launch_kv8_attention<128, 1>(a, dev, 6, stream); break;
    case 130: err = launch_kv8_attention<128, 2>(a, dev, 7, stream); break;
    default: err = launch_kv8_attention<256, 1>(a, dev, 8, stream); break;
  }
  return err == cudaSuccess ? B200TX_OK : cuda_fail(err, "kv8_attention");
}

int b200tx_linear_w4(const void* x, int64_t x_stride, const void* packed, const void* scales, const float* bias,
                     void* out, int out_dtype, int64_t M, int64_t N, int64_t K, int64_t group, int epilogue,
                     cudaStream_t stream) {
  if (x == nullptr || packed == nullptr || scales == nullptr || out == nullptr)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "linear_w4: null tensor pointer");
  if (M <= 0 || N <= 0 || K <= 0 || M > (1 << 20) || N > (1 << 24) || K > (1 << 24) || K % 8 != 0)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "linear_w4: bad shape M %lld N %lld K %lld (K a multiple of 8)",
                (long long)M, (long long)N, (long long)K);
  if (group != 32 && group != 64 && group != 128)
    return fail(B200TX_ERR_UNSUPPORTED, "linear_w4: group %lld (32, 64 and 128 are built)", (long long)group);
  if (out_dtype != B200TX_F32 && out_dtype != B200TX_BF16)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "linear_w4: out_dtype %d", out_dtype);
  if (epilogue != B200TX_EPI_BIAS && epilogue != B200TX_EPI_BIAS_GELU)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "linear_w4: epilogue %d", epilogue);
  if (!aligned16(x) || !aligned16(packed) || x_stride % 8 != 0)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "linear_w4: x and packed must be 16-byte aligned, x_stride a multiple of 8");
  DeviceState* dev = nullptr;
  int rc = current_device(&dev);
  if (rc != B200TX_OK) return rc;
  b200tx::W4Args a{};
  a.x = static_cast<const __nv_bfloat16*>(x);
  a.packed = static_cast<const uint8_t*>(packed);
  a.scales = static_cast<const __nv_bfloat16*>(scales);
  a.bias = bias;
  a.out = out;
  a.x_stride = x_stride;
  a.rows = static_cast<int>(M);
  a.outer = static_cast<int>(N);
  a.inner = static_cast<int>(K);
  a.runs = static_cast<int>((K + b200tx::kW4Run - 1) / b200tx::kW4Run);
  a.gelu = epilogue == B200TX_EPI_BIAS_GELU;
  a.out_f32 = out_dtype == B200TX_F32;
  if (w4_in_line(a, dev)) {
    cudaError_t err = M <= 8 ? launch_w4_line_group<1>(group, a, dev, 0, stream) : launch_w4_line_group<2>(group, a, dev, 3, stream);
    return err == cudaSuccess ? B200TX_OK : cuda_fail(err, "linear_w4");
  }
  // Rows of x by eights: 1, 2 or 4 MMA columns.  Four only where the columns of W
  // fill the SMs; with fewer the rows go 16 at a time, which makes twice the CTAs
  // and reads the weights again from L2 (29 x 4744 -> 5003: four 23.9 us, twice two 22.4).
  const bool by_16 = M <= 16 || (a.outer < 80 * dev->sm_count && M <= 16 * kW4GridRows);
  cudaError_t err = M <= 8   ? launch_w4_tiles<1>(group, a, dev, 0, stream)
                    : by_16 ? launch_w4_tiles<2>(group, a, dev, 6, stream)
                             : launch_w4_tiles<4>(group, a, dev, 12, stream);
  return err == cudaSuccess ? B200TX_OK : cuda_fail(err, "linear_w4");
}

}  // extern "C"
