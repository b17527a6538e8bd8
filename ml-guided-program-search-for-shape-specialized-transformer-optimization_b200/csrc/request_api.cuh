// request_api.cuh -- argument checks and launches of the operators for batches of
// many requests: low-rank adapters beside a shared projection, pages of the 8-bit cache,
// verification of drafted tokens.  Part of b200tx.cu's translation unit.
#pragma once

namespace {

constexpr int kLrShared = 220 * 1024;  // most that a build asks for

// Clusters of 1 << shift CTAs that run at once: those of 4 and 8 do not fill each part of the GPU (33 of eight CTAs with two on an
// SM, 15 with one, where 148 SMs would have room for 37 and 18).
template <typename Kernel>
cudaError_t low_rank_resident(Kernel kernel, int bytes, int shift, int* clusters) {
  if (*clusters > 0) return cudaSuccess;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(1u << shift);
  config.blockDim = dim3(b200tx::kLrThreads);
  config.dynamicSmemBytes = bytes;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = 1u << shift;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  int found = 0;
  cudaError_t err = cudaOccupancyMaxActiveClusters(&found, kernel, &config);
  if (err == cudaSuccess) *clusters = std::max(1, found);
  return err;
}

template <int RT, bool F32, bool WHOLE>
cudaError_t launch_low_rank(b200tx::LowRankArgs& a, DeviceState* dev, int index, cudaStream_t stream) {
  using S = b200tx::LrShape<RT>;
  static_assert(S::bytes(8, 3) <= kLrShared, "the sums of eight CTAs do not fit");
  if (!dev->low_rank_attr[index]) {
    cudaError_t err = cudaFuncSetAttribute(b200tx::low_rank_kernel<RT, F32, WHOLE>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize, kLrShared);
    if (err != cudaSuccess) return err;
    dev->low_rank_attr[index] = true;
  }
  const int64_t windows = (a.rows + b200tx::kLrWindow - 1) / b200tx::kLrWindow;
  const int64_t rows = std::min<int64_t>(a.rows, b200tx::kLrWindow);
  const int terms = a.out_f32 ? 3 : 2;
  // Groups of a window as far as can be told here: where its rows share an adapter, and half a group more for each
  // adapter that they may differ in.
  const int64_t differ = std::min<int64_t>(a.count, (rows + a.per_index - 1) / a.per_index);
  auto groups_of = [&](int64_t size) { return windows * std::min(rows, (rows + size - 1) / size + differ / 2); };
  const int64_t tiles = (a.outer + b200tx::kLrTile - 1) / b200tx::kLrTile, steps = (a.inner + 31) / 32;
  int64_t resident[4];  // clusters of 1, 2, 4 and 8 CTAs that run at once
  for (int i = 0; i < 4; ++i) {
    cudaError_t err = low_rank_resident(b200tx::low_rank_kernel<RT, F32, WHOLE>, S::bytes(1 << i, terms), i,
                                        &dev->low_rank_resident[index][terms - 2][i]);
    if (err != cudaSuccess) return err;
    resident[i] = dev->low_rank_resident[index][terms - 2][i];
  }
  // Groups of as few rows as let all run at once, in clusters of the size for which a warp has least to do: steps of K, and
  // rounds of columns, which take eight times as long.  A second wave costs more than all else (256 rows of 8 adapters,
  // 4096 -> 4096, rank 32: 8 rows by four CTAs 11.6 us, by eight 16.5; rank 128 by two 20.3, by eight 37.0; 203 rows of
  // 4744 -> 5003: by two CTAs, with one round, 15.1, by eight, with two, 17.5, and 32 rows by eight 27).
  int shift = -1;
  int64_t least = 0;
  for (a.group = 8;; a.group *= 2) {
    const int64_t groups = groups_of(a.group);
    for (int i = 0; i < 4; ++i) {
      if (groups > resident[i] || (i == 0 && steps > 8 * b200tx::kLrWarps)) continue;  // one CTA only where K is short
      const int64_t units = b200tx::kLrWarps << i;
      const int64_t split = std::min(resident[i] / groups, (tiles + units - 1) / units);
      const int64_t cost = 2 * ((steps + units - 1) / units) + 16 * ((tiles + units * split - 1) / (units * split)) +
                           (i > 0) * 2 + (i == 3);
      if (shift >= 0 && cost >= least) continue;
      least = cost;
      shift = i;
    }
    if (shift >= 0 || a.group == S::G) break;
  }
  // Too many for that: several waves of small clusters (1024 rows of 32 adapters, 4096 -> 4096: rank 32 by one CTA 34.4 us, two
  // 27.1, four 39; rank 64 37.7, 46.5 and 58).
  if (shift < 0) shift = S::TWO ? 1 : 0;
  const int ctas = 1 << shift, bytes = S::bytes(ctas, terms);
  // Groups that can be: one more for each further index that occurs.
  const int64_t most = std::min<int64_t>(rows, (rows + a.group - 1) / a.group + a.count + 1);
  a.parts = static_cast<int>((tiles + ctas * b200tx::kLrWarps - 1) / (ctas * b200tx::kLrWarps));
  a.clusters = static_cast<int>(std::min(std::max(groups_of(a.group), resident[shift]) / windows, most * a.parts));
  return launch_clustered(b200tx::low_rank_kernel<RT, F32, WHOLE>, dim3(static_cast<unsigned>(windows * a.clusters * ctas)),
                          dim3(b200tx::kLrThreads), static_cast<size_t>(bytes), static_cast<unsigned>(ctas), stream, a);
}

template <int RT>
cudaError_t launch_low_rank_io(b200tx::LowRankArgs& a, bool f32, DeviceState* dev, int index, cudaStream_t stream) {
  if (a.outer % 8 == 0)
    return f32 ? launch_low_rank<RT, true, true>(a, dev, index, stream) : launch_low_rank<RT, false, true>(a, dev, index + 1, stream);
  return f32 ? launch_low_rank<RT, true, false>(a, dev, index + 2, stream) : launch_low_rank<RT, false, false>(a, dev, index + 3, stream);
}

template <int RA, bool F32>
int launch_low_rank_tile(b200tx::LowRankArgs& a, DeviceState* dev, int index, cudaStream_t stream) {
  using S = b200tx::LtShape<RA>;
  constexpr int kMost = 215 * 1024;
  static_assert(S::bytes(RA * 64, 3) <= kMost, "the terms do not fit");
  if (!dev->low_rank_tile_attr[index]) {
    cudaError_t err = cudaFuncSetAttribute(b200tx::low_rank_tile_kernel<RA, F32>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (err != cudaSuccess) return cuda_fail(err, "low_rank_add");
    dev->low_rank_tile_attr[index] = true;
  }
  const int rank16 = (a.rank + 15) / 16 * 16;
  const int bytes = static_cast<int>(S::bytes(rank16, a.out_f32 ? 3 : 2));
  const int64_t windows = (a.rows + b200tx::kLrWindow - 1) / b200tx::kLrWindow;
  const int64_t rows = std::min<int64_t>(a.rows, b200tx::kLrWindow);
  a.group = b200tx::kLtRows;
  const int64_t least = (rows + a.group - 1) / a.group;
  // The columns are cut into parts, for each of which the sums are taken anew, while all CTAs then run at once.
  const int64_t resident = dev->sm_count;
  const int64_t rounds = (a.outer + b200tx::kLtColumns - 1) / b200tx::kLtColumns;
  a.parts = static_cast<int>(std::min(rounds, std::max<int64_t>(1, resident / (windows * least))));
  a.clusters = static_cast<int>(least * a.parts);
  using u64 = uint64_t;
  CUtensorMap x_map, down_map, up_map;
  const u64 inner = a.inner, rank = a.rank, count = a.count;
  const u64 x_dims[2] = {inner, static_cast<u64>(a.rows)}, down_dims[2] = {inner, count * rank}, k_stride[1] = {inner * 2};
  const uint32_t x_box[2] = {64, b200tx::kLtRows}, down_box[2] = {64, static_cast<uint32_t>(rank16)};
  const u64 up_dims[3] = {rank, 8, count * a.outer / 8}, up_strides[2] = {rank * 2, rank * 16};
  const uint32_t up_box[3] = {64, 2, b200tx::kLtColumns / 8};
  int rc = encode_bf16_map(&x_map, a.x, 2, x_dims, k_stride, x_box);
  if (rc == B200TX_OK) rc = encode_bf16_map(&down_map, a.down, 2, down_dims, k_stride, down_box);
  if (rc == B200TX_OK) rc = encode_bf16_map(&up_map, a.up, 3, up_dims, up_strides, up_box);
  if (rc != B200TX_OK) return rc;
  cudaError_t err = launch(b200tx::low_rank_tile_kernel<RA, F32>, dim3(static_cast<unsigned>(windows * a.clusters)),
                           dim3(b200tx::kLtThreads), static_cast<size_t>(bytes), stream, a, x_map, down_map, up_map);
  return err == cudaSuccess ? B200TX_OK : cuda_fail(err, "low_rank_add");
}

// Rows go by 128 on tcgen05 where there are many, in runs of one adapter, and rows of base and the result are multiples of 16
// bytes.  The warp MMAs' time grows with rows x ranks, the UMMAs' with K: a group's sums are one CTA's (1024 -> 4096: 1024 rows of rank
// 16 13.1 us by warps, 14.2 so; rank 32 16.1 and 14.7, rank 64 20.3 and 15.0; 4096 rows of rank 64 57 and 27.  4096 -> 4096:
// 1024 rows of rank 64 23.6 and 31.0, 2048 38.5 and 34.1, 4096 76 and 41.5; 4096 rows of rank 16 33.9 and 41, 8192 66.6 and 52.8).
// Runs are told by how many rows an index stands for, which is known here; with an index for each row the warp MMAs take
// all (8 x 2048 rows of rank 64, 1024 -> 4096, GELU: 238 us in runs and 275 in no order, where 8 indices take 79.8).
constexpr int64_t kLtLeastRows = 1024, kLtLeastRun = 64, kLtLeastRanks = 32, kLtLeastInner = 1024;

int kv8_pool(const char* what, const b200tx_kv8_pool* c, b200tx::Kv8Pool* out) {
  if (c == nullptr) return fail(B200TX_ERR_INVALID_ARGUMENT, "%s: null pool", what);
  b200tx::Kv8Cache view;
  int rc = kv8_view(what, &c->cache, &view);
  if (rc != B200TX_OK) return rc;
  if (c->refs == nullptr || c->scratch == nullptr)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "%s: null pool pointer", what);
  if (!aligned16(c->refs) || !aligned16(c->scratch))
    return fail(B200TX_ERR_INVALID_ARGUMENT, "%s: refs and scratch must be 16-byte aligned", what);
  if (c->layers <= 0 || c->layers > (1 << 16)) return fail(B200TX_ERR_INVALID_ARGUMENT, "%s: %lld layers", what, (long long)c->layers);
  if (c->cache.pages > (1 << 30)) return fail(B200TX_ERR_INVALID_ARGUMENT, "%s: %lld pages", what, (long long)c->cache.pages);
  out->codes = view.codes;
  out->scales = view.scales;
  out->tail = reinterpret_cast<uint4*>(view.tail);
  out->page_table = const_cast<int32_t*>(view.page_table);
  out->lengths = const_cast<int32_t*>(view.lengths);
  out->refs = c->refs;
  out->scratch = c->scratch;
  out->pages = view.pages;
  out->slots = view.slots;
  out->max_blocks = view.max_blocks;
  out->kv_heads = view.kv_heads;
  out->dim = static_cast<int>(c->cache.head_dim);
  out->layers = static_cast<int>(c->layers);
  return B200TX_OK;
}

// Places of the table of slots: a power of two, at least twice the rows.
int slot_places(int64_t rows) {
  int places = 2;
  while (places < 2 * rows) places *= 2;
  return places;
}

int low_log2(int64_t v) {
  int shift = 0;
  while ((int64_t{2} << shift) <= v) ++shift;
  return shift;
}

constexpr int kPoolShared = 96 * 1024;  // of 2048 rows' records and places

// CTAs for an order over so many pages and entries: one, without exchanges, while its threads take few of them
// each (free and reserve with 1320 pages: one 10.3 us, a cluster 12.4; 10320: 14.9 and 16.4; 20640: 19.3 and 17.9; 82080: 51
// and 21; compaction of 3572 pages 11.6 and 14.7, of 14286 23.5 and 19.8).
constexpr int64_t kPoolFew = 12288;
unsigned pool_cluster(int64_t pages, int64_t entries) { return std::max(pages, entries) <= kPoolFew ? 1 : b200tx::kPoolCtas; }

template <typename Kernel>
cudaError_t pool_attribute(Kernel kernel, bool* done) {
  if (*done) return cudaSuccess;
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPoolShared);
  if (err == cudaSuccess) err = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (err == cudaSuccess) *done = true;
  return err;
}

template <typename T, bool VEC>
cudaError_t launch_verify(b200tx::VerifyArgs& a, int64_t batch, cudaStream_t stream) {
  return launch_clustered(b200tx::verify_draft_kernel<T, VEC>, dim3(static_cast<unsigned>(batch) * b200tx::kVerifyMostCtas),
                          dim3(b200tx::kVerifyThreads), 0, b200tx::kVerifyMostCtas, stream, a);
}

}  // namespace

extern "C" {

int b200tx_low_rank_add(const void* x, const void* base, int base_dtype, void* out, int out_dtype, const void* down,
                        const void* up, const float* scales, const int32_t* indices, int64_t index_count, int64_t M,
                        int64_t N, int64_t K, int64_t rank, int64_t adapters, int epilogue, cudaStream_t stream) {
  if (x == nullptr || base == nullptr || out == nullptr || down == nullptr || up == nullptr || scales == nullptr ||
      indices == nullptr)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "low_rank_add: null tensor pointer");
  if (M <= 0 || N <= 0 || K <= 0 || M > (1 << 26) || N > (1 << 24) || K > (1 << 24) || K % 8 != 0)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "low_rank_add: bad shape M %lld N %lld K %lld (K a multiple of 8)",
                (long long)M, (long long)N, (long long)K);
  if (rank <= 0 || rank > 128 || rank % 8 != 0)
    return fail(B200TX_ERR_UNSUPPORTED, "low_rank_add: rank %lld (multiples of 8 up to 128 are built)", (long long)rank);
  if (adapters <= 0 || adapters > (1 << 20))
    return fail(B200TX_ERR_INVALID_ARGUMENT, "low_rank_add: %lld adapters", (long long)adapters);
  if (index_count <= 0 || M % index_count != 0)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "low_rank_add: %lld indices for %lld rows", (long long)index_count, (long long)M);
  if ((base_dtype != B200TX_F32 && base_dtype != B200TX_BF16) || (out_dtype != B200TX_F32 && out_dtype != B200TX_BF16))
    return fail(B200TX_ERR_INVALID_ARGUMENT, "low_rank_add: dtypes %d and %d", base_dtype, out_dtype);
  if (epilogue != B200TX_EPI_BIAS && epilogue != B200TX_EPI_BIAS_GELU)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "low_rank_add: epilogue %d", epilogue);
  if (!aligned16(x) || !aligned16(base) || !aligned16(out) || !aligned16(down) || !aligned16(up))
    return fail(B200TX_ERR_INVALID_ARGUMENT, "low_rank_add: x, base, out, down and up must be 16-byte aligned");
  if (base == out && base_dtype != out_dtype)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "low_rank_add: out is base in another type");
  DeviceState* dev = nullptr;
  int rc = current_device(&dev);
  if (rc != B200TX_OK) return rc;
  b200tx::LowRankArgs a{};
  a.x = static_cast<const __nv_bfloat16*>(x);
  a.base = base;
  a.out = out;
  a.down = static_cast<const __nv_bfloat16*>(down);
  a.up = static_cast<const __nv_bfloat16*>(up);
  a.scales = scales;
  a.indices = indices;
  a.rows = M;
  a.per_index = static_cast<int>(M / index_count);
  a.inner = static_cast<int>(K);
  a.outer = static_cast<int>(N);
  a.rank = static_cast<int>(rank);
  a.count = static_cast<int>(adapters);
  a.out_f32 = out_dtype == B200TX_F32;
  a.gelu = epilogue == B200TX_EPI_BIAS_GELU;
  a.skip_bare = base == out && !a.gelu;
  const bool f32 = base_dtype == B200TX_F32;
  if (M >= kLtLeastRows && M * rank >= kLtLeastRanks * std::max(K, kLtLeastInner) && a.per_index >= kLtLeastRun &&
      N % 8 == 0 && adapters * N < (int64_t{1} << 34)) {
    return rank <= 64 ? f32 ? launch_low_rank_tile<1, true>(a, dev, 0, stream) : launch_low_rank_tile<1, false>(a, dev, 1, stream)
           : f32      ? launch_low_rank_tile<2, true>(a, dev, 2, stream)
                      : launch_low_rank_tile<2, false>(a, dev, 3, stream);
  }
  cudaError_t err = rank <= 16   ? launch_low_rank_io<1>(a, f32, dev, 0, stream)
                    : rank <= 32 ? launch_low_rank_io<2>(a, f32, dev, 4, stream)
                    : rank <= 64 ? launch_low_rank_io<4>(a, f32, dev, 8, stream)
                                 : launch_low_rank_io<8>(a, f32, dev, 12, stream);
  return err == cudaSuccess ? B200TX_OK : cuda_fail(err, "low_rank_add");
}

int b200tx_kv8_pool_scratch(int64_t pages, int64_t* ints_out) {
  if (ints_out == nullptr || pages <= 0 || pages > (1 << 30))
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_pool_scratch: %lld pages", (long long)pages);
  *ints_out = b200tx::kPoolCounters + 2 * pages;
  return B200TX_OK;
}

int b200tx_kv8_fork(const b200tx_kv8_pool* pool, const int32_t* source, const int32_t* target, int64_t pairs,
                    cudaStream_t stream) {
  b200tx::Kv8ForkArgs a{};
  int rc = kv8_pool("kv8_fork", pool, &a.pool);
  if (rc != B200TX_OK) return rc;
  if (pairs < 0 || pairs > b200tx::kPoolRows)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_fork: %lld sequences (%d at most)", (long long)pairs, b200tx::kPoolRows);
  if (pairs == 0) return B200TX_OK;
  if (target == nullptr) return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_fork: null target");
  DeviceState* dev = nullptr;
  rc = current_device(&dev);
  if (rc != B200TX_OK) return rc;
  a.source = source;
  a.target = target;
  a.pairs = static_cast<int>(pairs);
  a.owners = slot_places(pairs);
  const int region = b200tx::kKv8Block * a.pool.dim / 8;
  a.region_log2 = low_log2(region);
  a.piece_shift = std::min(low_log2(b200tx::kForkPieces / pairs), a.region_log2);
  if (source != nullptr && static_cast<double>(a.pool.slots) * 4 * a.pool.kv_heads * region >= 4294967295.0)
    return fail(B200TX_ERR_UNSUPPORTED, "kv8_fork: a layer's tails pass 64 GB");
  a.column_shift = low_log2(b200tx::kForkPieces / pairs);
  const int64_t tail_items =
      source == nullptr ? 0 : static_cast<int64_t>(a.pool.layers) * 2 * a.pool.kv_heads * (region >> a.piece_shift);
  const int64_t table_items = ((a.pool.max_blocks - 1) >> a.column_shift) + 1;
  if (tail_items + table_items > (1 << 30))
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_fork: too many layers and heads");
  a.tail_items = static_cast<int>(tail_items);
  a.table_items = static_cast<int>(table_items);
  cudaError_t err = pool_attribute(b200tx::kv8_fork_kernel, &dev->fork_attr);
  const int64_t grid = std::min<int64_t>(tail_items + table_items, b200tx::kForkCtas * dev->sm_count);
  if (err == cudaSuccess)
    err = launch(b200tx::kv8_fork_kernel, dim3(static_cast<unsigned>(grid)), dim3(b200tx::kForkThreads),
                 pairs * sizeof(b200tx::ForkPair) + 8 * a.owners, stream, a);
  return err == cudaSuccess ? B200TX_OK : cuda_fail(err, "kv8_fork");
}

int b200tx_kv8_reserve(const b200tx_kv8_pool* pool, const int32_t* slot_ids, const int32_t* counts, int64_t tokens,
                       int64_t rows, int32_t* missing, cudaStream_t stream) {
  b200tx::Kv8ReserveArgs a{};
  int rc = kv8_pool("kv8_reserve", pool, &a.pool);
  if (rc != B200TX_OK) return rc;
  if (rows <= 0 || rows > b200tx::kPoolRows || tokens < 0 || tokens > (1 << 26))
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_reserve: %lld tokens of %lld sequences (%d at most)", (long long)tokens,
                (long long)rows, b200tx::kPoolRows);
  if (missing == nullptr) return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_reserve: null result");
  if (slot_ids == nullptr && rows > a.pool.slots)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_reserve: %lld sequences in a cache of %d slots", (long long)rows, a.pool.slots);
  const int64_t entries = rows * std::min<int64_t>(a.pool.max_blocks, tokens / b200tx::kKv8Block + 1);
  if (entries > (1 << 30))
    return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_reserve: too many blocks");
  DeviceState* dev = nullptr;
  rc = current_device(&dev);
  if (rc != B200TX_OK) return rc;
  a.slot_ids = slot_ids;
  a.counts = counts;
  a.missing = missing;
  a.tokens = static_cast<int>(tokens);
  a.rows = static_cast<int>(rows);
  a.owners = slot_places(rows);
  cudaError_t err = pool_attribute(b200tx::kv8_reserve_kernel, &dev->reserve_attr);
  const unsigned ctas = pool_cluster(a.pool.pages, entries);
  if (err == cudaSuccess)
    err = launch_clustered(b200tx::kv8_reserve_kernel, dim3(ctas), dim3(b200tx::kPoolThreads),
                           static_cast<size_t>(12 * rows + 8 * a.owners), ctas, stream, a);
  return err == cudaSuccess ? B200TX_OK : cuda_fail(err, "kv8_reserve");
}

int b200tx_kv8_compact(const b200tx_kv8_pool* pool, int32_t* used, cudaStream_t stream) {
  b200tx::Kv8CompactArgs a{};
  int rc = kv8_pool("kv8_compact", pool, &a.pool);
  if (rc != B200TX_OK) return rc;
  if (used == nullptr) return fail(B200TX_ERR_INVALID_ARGUMENT, "kv8_compact: null result");
  DeviceState* dev = nullptr;
  rc = current_device(&dev);
  if (rc != B200TX_OK) return rc;
  a.used = used;
  a.page_bytes = static_cast<int64_t>(2) * a.pool.kv_heads * b200tx::kKv8Block * a.pool.dim;
  constexpr int64_t kPiece = b200tx::kCompactThreads * b200tx::kCompactHeld * 16;
  a.piece = static_cast<int>(std::min(a.page_bytes, kPiece));
  a.pieces = static_cast<int>((a.page_bytes + a.piece - 1) / a.piece);
  const unsigned ctas = pool_cluster(a.pool.pages, 0);
  cudaError_t err = pool_attribute(b200tx::kv8_compact_plan_kernel, &dev->compact_attr);
  if (err == cudaSuccess)
    err = launch_clustered(b200tx::kv8_compact_plan_kernel, dim3(ctas), dim3(b200tx::kPoolThreads), 0, ctas, stream, a);
  if (err == cudaSuccess)
    err = launch(b200tx::kv8_compact_move_kernel,
                 dim3(static_cast<unsigned>(std::min<int64_t>(4 * dev->sm_count, (a.pool.pages + 1) / 2 * a.pool.layers * a.pieces))),
                 dim3(b200tx::kCompactThreads), 0, stream, a);
  return err == cudaSuccess ? B200TX_OK : cuda_fail(err, "kv8_compact");
}

int b200tx_verify_draft(const void* target, int64_t target_batch_stride, int64_t target_token_stride, const void* draft,
                        int64_t draft_batch_stride, int64_t draft_token_stride, int dtype, const void* drafted,
                        int drafted_64, const float* uniform, const int32_t* counts, int64_t batch, int64_t tokens,
                        int64_t vocab, void* out, int32_t* accepted, cudaStream_t stream) {
  if (target == nullptr || (drafted == nullptr && tokens > 0) || uniform == nullptr || out == nullptr || accepted == nullptr)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "verify_draft: null tensor pointer");
  if (batch <= 0 || batch > (1 << 20) || tokens < 0 || tokens > b200tx::kVerifyTokens || vocab <= 0 || vocab > (1 << 28))
    return fail(B200TX_ERR_INVALID_ARGUMENT, "verify_draft: bad shape batch %lld tokens %lld (%d at most) vocab %lld",
                (long long)batch, (long long)tokens, b200tx::kVerifyTokens, (long long)vocab);
  if (dtype != B200TX_F32 && dtype != B200TX_BF16)
    return fail(B200TX_ERR_INVALID_ARGUMENT, "verify_draft: dtype %d", dtype);
  DeviceState* dev = nullptr;
  int rc = current_device(&dev);
  if (rc != B200TX_OK) return rc;
  b200tx::VerifyArgs a{};
  a.target = target;
  a.draft = draft;
  a.drafted = drafted;
  a.uniform = uniform;
  a.counts = counts;
  a.out = out;
  a.accepted = accepted;
  a.target_batch_stride = target_batch_stride;
  a.target_token_stride = target_token_stride;
  a.draft_batch_stride = draft_batch_stride;
  a.draft_token_stride = draft_token_stride;
  a.tokens = static_cast<int>(tokens);
  a.vocab = static_cast<int>(vocab);
  a.wide = drafted_64 != 0;
  const int per = dtype == B200TX_F32 ? 4 : 8;  // values in 16 bytes
  const int64_t strides = target_batch_stride | target_token_stride | (draft == nullptr ? 0 : draft_batch_stride | draft_token_stride);
  const bool vec = aligned16(target) && (draft == nullptr || aligned16(draft)) && strides % per == 0;
  cudaError_t err;
  if (dtype == B200TX_F32)
    err = vec ? launch_verify<float, true>(a, batch, stream) : launch_verify<float, false>(a, batch, stream);
  else
    err = vec ? launch_verify<__nv_bfloat16, true>(a, batch, stream) : launch_verify<__nv_bfloat16, false>(a, batch, stream);
  return err == cudaSuccess ? B200TX_OK : cuda_fail(err, "verify_draft");
}

}  // extern "C"
