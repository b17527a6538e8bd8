// low_rank_kernels.cuh -- low-rank adapters of many requests beside a shared
// projection:
//     out[r] = act(base[r] + scale_a * (x[r] . down_a^T) . up_a^T)
// with the adapter a of each row (a request's), down_a [R, K], up_a [N, R], R
// up to 128.  Rows with a negative index have none, rows with an index past the
// set are NaN.
//
// Two thin products with R between them: the work is the bytes of x, base and out, and
// of the adapters in use.  One launch does both.  Rows that share an adapter are
// found on the way: within a window of 256 rows each thread ranks its row
// among those with the same index, and every G-th rank leads a group of up to
// G rows (in any places of the window), so an adapter is read once for G rows
// whatever order the rows come in, and nothing is sorted or laid out before.
//
// A cluster takes a group.  Its warps split K: a warp's sums of down . x^T are
// joined in shared memory, the CTAs' in each other's (distributed shared memory),
// in a fixed order.  Then the warps split N.
//
// Both products are warp MMAs (m16n8k16) with the weights as the A operand and
// the rows as its 8 columns: 8 rows are a full tile, and weights and x go from global memory
// to registers as they lie, 16 bytes a lane.  That works because the
// order of a contraction's terms is free: a lane's 8 neighbouring values of k
// stand where the fragment wants (2t, 2t + 1, 2t + 8, 2t + 9) twice.  In the second product
// the rows of up are dealt out so that a lane holds 8 neighbouring columns of
// the result.  tcgen05 would want x and the weights in shared memory first, for
// tiles of 128 rows that share an adapter; the tensor pipe is not what bounds this.
//
// The R sums of a row are fp32.  The second product takes them as bf16 terms, each the rounded rest of the
// ones before: two (2^-17 of the sum is left) where the result has 16 bits, three (2^-25) where it has 32.
#pragma once

#include "attention_mma_kernels.cuh"
#include "gemm_kernels.cuh"

namespace b200tx {

constexpr int kLrWarps = 8;
constexpr int kLrThreads = kLrWarps * 32;
constexpr int kLrWindow = kLrThreads;  // rows among which groups are formed
constexpr int kLrTile = 64;            // columns of the result that a warp takes at a time
constexpr int kLrStageRow = kLrTile + 4;

struct LowRankArgs {
  const __nv_bfloat16* x;     // [rows, inner]
  const void* base;           // [rows, outer]
  void* out;                  // [rows, outer], base's memory or other
  const __nv_bfloat16* down;  // [count, rank, inner]
  const __nv_bfloat16* up;    // [count, outer, rank]
  const float* scales;        // [count]
  const int32_t* indices;     // [rows / per_index]
  int64_t rows;
  int per_index, inner, outer, rank, count;
  int out_f32, gelu;
  int clusters;     // for each window
  int parts;        // most that the columns are cut into between clusters
  int skip_bare;    // out is base and has nothing done to it where there is no adapter
};

// The groups of a window's rows.
template <int G>
struct LrGroups {
  __align__(16) int key[kLrWindow];  // the row's adapter, -1: none, count: past the set
  int rank[kLrWindow];               // its place among the rows of that key
  int lead[kLrWindow];               // the first row of each group
  int warp_leads[kLrWarps];
  int rows[G];                       // of the group at hand, -1 past its end

  // Ranks the window's n rows; returns the number of groups.
  __device__ __forceinline__ int form(const LowRankArgs& a, int64_t first, int n) {
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    int mine = -2;
    if (tid < n) {
      const int index = a.indices[static_cast<unsigned>(first + tid) / static_cast<unsigned>(a.per_index)];
      key[tid] = mine = index < 0 ? -1 : min(index, a.count);
    }
    __syncthreads();
    int before = 0;
    if (tid < n) {
      for (int j = 0; j < (tid & ~31); j += 4) {
        const int4 k = *reinterpret_cast<const int4*>(key + j);
        before += (k.x == mine) + (k.y == mine) + (k.z == mine) + (k.w == mine);
      }
    }
    const uint32_t same = __match_any_sync(0xffffffffu, mine);
    before += __popc(same & ((1u << lane) - 1));
    const bool leads = tid < n && before % G == 0;
    const uint32_t leaders = __ballot_sync(0xffffffffu, leads);
    rank[tid] = before;
    if (lane == 0) warp_leads[warp] = __popc(leaders);
    __syncthreads();
    int groups = 0, at = 0;
#pragma unroll
    for (int w = 0; w < kLrWarps; ++w) {
      if (w == warp) at = groups;
      groups += warp_leads[w];
    }
    if (leads) lead[at + __popc(leaders & ((1u << lane) - 1))] = tid;
    __syncthreads();
    return groups;
  }

  // Fills `rows` with the group's; all threads, which are done with the one before.  Returns how many.
  __device__ __forceinline__ int take(int group, int n) {
    const int tid = threadIdx.x, leader = lead[group], adapter = key[leader], from = rank[leader];
    const bool in = tid < n && key[tid] == adapter && rank[tid] >= from && rank[tid] < from + G;
    if (tid < G) rows[tid] = -1;
    const int many = __syncthreads_count(in);
    if (in) rows[rank[tid] - from] = tid;
    __syncthreads();
    return many;
  }
};

// Floats of a group's sums, as the MMA leaves them: RT tiles of 16 ranks, NT of 8 rows.
template <int RT, int NT>
struct LrShape {
  static constexpr int G = NT * 8;
  static constexpr int SUMS = RT * NT * 128;
  static constexpr int H_ROW = RT * 16 + 8;  // padded: a lane's 16 bytes of 8 rows fall into different banks
  static constexpr int TERM = G * H_ROW;             // of one of the terms
  static constexpr int STAGE = 8 * kLrStageRow;      // floats in which a warp turns its results
  static constexpr int JOIN = kLrWarps * (SUMS > STAGE ? SUMS : STAGE) * 4;
  // shared memory with `ctas` in a cluster: warps' sums, two rounds of the CTAs' sums, the terms
  static constexpr int bytes(int ctas, int terms) { return JOIN + (ctas > 1 ? 2 * ctas * SUMS * 4 : 0) + terms * TERM * 2; }
};

__device__ __forceinline__ void st_cluster_v4(uint32_t addr, const float4& v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}

// GELU of two values: with the library's erf where the result has 32 bits, by the approximation of the
// projections' epilogue (1.5e-7 of the value) where it has 16.  There infinity is no number in the product of its factors.
__device__ __forceinline__ void lr_gelu(float& x, float& y, bool f32) {
  if (f32) {
    x = 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
    y = 0.5f * y * (1.f + erff(y * 0.70710678118654752f));
    return;
  }
  const float inf = __int_as_float(0x7f800000), x0 = x, y0 = y;
  gelu_erf_x2(x, y);
  x = x0 == inf ? inf : x;
  y = y0 == inf ? inf : y;
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// Eight neighbouring values of a row of base, as they lie.
template <bool F32>
struct LrEight {
  uint4 w[F32 ? 2 : 1];

  __device__ __forceinline__ void load(const LowRankArgs& a, int64_t at) {
    const uint4* const p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.base) + at * (F32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < (F32 ? 2 : 1); ++i) w[i] = p[i];
  }

  __device__ __forceinline__ void values(float (&y)[8]) const {
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        y[4 * i] = __uint_as_float(w[i].x), y[4 * i + 1] = __uint_as_float(w[i].y);
        y[4 * i + 2] = __uint_as_float(w[i].z), y[4 * i + 3] = __uint_as_float(w[i].w);
      }
    } else {
      const uint32_t v[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[2 * i] = __uint_as_float(v[i] << 16);
        y[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
      }
    }
  }
};

__device__ __forceinline__ void lr_store_eight(const LowRankArgs& a, int64_t at, float (&y)[8]) {
  if (a.gelu) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) lr_gelu(y[i], y[i + 1], a.out_f32);
  }
  if (a.out_f32) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.out) + at);
    p[0] = make_float4(y[0], y[1], y[2], y[3]);
    p[1] = make_float4(y[4], y[5], y[6], y[7]);
  } else {
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + at) =
        make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]));
  }
}

template <bool F32>
__device__ __forceinline__ float lr_load_one(const LowRankArgs& a, int64_t at) {
  if constexpr (F32)
    return static_cast<const float*>(a.base)[at];
  else
    return __bfloat162float(static_cast<const __nv_bfloat16*>(a.base)[at]);
}

__device__ __forceinline__ void lr_store_one(const LowRankArgs& a, int64_t at, float y) {
  if (a.out_f32)
    static_cast<float*>(a.out)[at] = y;
  else
    static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16(y);
}

// A value as two or three bf16 terms, `apart` from one another: each the rounded rest.
__device__ __forceinline__ void lr_terms(float h, int parts, __nv_bfloat16* to, int apart) {
  const bool finite = fabsf(h) <= 3.38e38f;  // else the first term is all
  for (int i = 0; i < parts; ++i) {
    const __nv_bfloat16 near = __float2bfloat16(h);
    to[i * apart] = near;
    h = finite ? h - __bfloat162float(near) : 0.f;
  }
}

// What the column part of a group works on.
struct LrColumns {
  int64_t first;                // the window's first row
  const int* rows;              // of the group, in the window
  const __nv_bfloat16* up;      // the adapter's, or null: nothing is added
  const __nv_bfloat16* terms;   // [parts][G][H_ROW]
  float* stage;                 // the warp's
  int parts;                    // terms that the sums are split into
  bool bad;                     // an index past the set: NaN
};

// TILES tiles of 64 columns, `stride` apart, for the first NTU * 8 rows of the group.
template <int RT, int NT, int NTU, int TILES, bool F32>
__device__ __forceinline__ void lr_columns(const LowRankArgs& a, const LrColumns& o, int tile0, int stride, int tiles) {
  using S = LrShape<RT, NT>;
  const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const bool whole = a.outer % 8 == 0;
  // base goes out first: no load of it waits behind a store that might be to the same place
  LrEight<F32> base[TILES][NTU][2];
  if (whole) {
#pragma unroll
    for (int q = 0; q < TILES; ++q) {
      const int col = (tile0 + q * stride) * kLrTile + 8 * g;
#pragma unroll
      for (int i = 0; i < NTU; ++i) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = o.rows[i * 8 + 2 * t + e];
          if (row >= 0 && tile0 + q * stride < tiles && col < a.outer) base[q][i][e].load(a, (o.first + row) * a.outer + col);
        }
      }
    }
  }
  float acc[TILES][4][NTU][4] = {};
  if (o.up != nullptr) {
    constexpr int CHUNKS = RT == 1 ? 1 : RT / 2;  // of 16 or 32 ranks
#pragma unroll(TILES * CHUNKS <= 2 ? CHUNKS : 1)
    for (int r = 0; r < CHUNKS; ++r) {
      // 4 ranks a lane, or 8
      uint4 w[TILES][4][2];
#pragma unroll
      for (int q = 0; q < TILES; ++q) {
        const int col = (tile0 + q * stride) * kLrTile + 8 * g;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int at = col + 2 * m + h, rank = RT == 1 ? 4 * t : r * 32 + 8 * t;
            const __nv_bfloat16* const p = o.up + static_cast<int64_t>(at) * a.rank + rank;
            const bool in = tile0 + q * stride < tiles && at < a.outer && rank < a.rank;
            w[q][m][h] = make_uint4(0, 0, 0, 0);
            if constexpr (RT == 1) {
              if (in) {
                const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
                w[q][m][h].x = v.x, w[q][m][h].y = v.y;
              }
            } else {
              if (in) w[q][m][h] = __ldg(reinterpret_cast<const uint4*>(p));
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NTU; ++i) {
        for (int part = 0; part < o.parts; ++part) {
          const __nv_bfloat16* const p = o.terms + part * S::TERM + (i * 8 + g) * S::H_ROW + (RT == 1 ? 4 * t : r * 32 + 8 * t);
          uint4 b = make_uint4(0, 0, 0, 0);
          if constexpr (RT == 1) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            b.x = v.x, b.y = v.y;
          } else {
            b = *reinterpret_cast<const uint4*>(p);
          }
#pragma unroll
          for (int q = 0; q < TILES; ++q) {
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              const uint32_t one[4] = {w[q][m][0].x, w[q][m][1].x, w[q][m][0].y, w[q][m][1].y};
              mma_m16n8k16_bf16(acc[q][m][i], one, b.x, b.y);
              if constexpr (RT > 1) {
                const uint32_t two[4] = {w[q][m][0].z, w[q][m][1].z, w[q][m][0].w, w[q][m][1].w};
                mma_m16n8k16_bf16(acc[q][m][i], two, b.z, b.w);
              }
            }
          }
        }
      }
    }
  }
  const float nan = __int_as_float(0x7fffffff);
#pragma unroll
  for (int q = 0; q < TILES; ++q) {
    const int tile = tile0 + q * stride, col = tile * kLrTile + 8 * g;
    if (tile >= tiles) break;
#pragma unroll
    for (int i = 0; i < NTU; ++i) {
      if (whole) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = o.rows[i * 8 + 2 * t + e];
          if (row < 0 || col >= a.outer) continue;
          float y[8];
          base[q][i][e].values(y);
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            y[2 * m] = o.bad ? nan : y[2 * m] + acc[q][m][i][e];
            y[2 * m + 1] = o.bad ? nan : y[2 * m + 1] + acc[q][m][i][2 + e];
          }
          lr_store_eight(a, (o.first + row) * a.outer + col, y);
        }
        continue;
      }
      // Rows that start anywhere: turned in shared memory, so that a warp reads and writes 32 neighbouring values.
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float4* const to = reinterpret_cast<float4*>(o.stage + (2 * t + e) * kLrStageRow + 8 * g);
        to[0] = make_float4(acc[q][0][i][e], acc[q][0][i][2 + e], acc[q][1][i][e], acc[q][1][i][2 + e]);
        to[1] = make_float4(acc[q][2][i][e], acc[q][2][i][2 + e], acc[q][3][i][e], acc[q][3][i][2 + e]);
      }
      __syncwarp();
      float y[8][2];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int row = o.rows[i * 8 + r];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = tile * kLrTile + h * 32 + lane;
          y[r][h] = row >= 0 && at < a.outer ? lr_load_one<F32>(a, (o.first + row) * a.outer + at) : 0.f;
        }
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int row = o.rows[i * 8 + r];
        if (row < 0) break;
        float lo = y[r][0] + o.stage[r * kLrStageRow + lane], hi = y[r][1] + o.stage[r * kLrStageRow + 32 + lane];
        if (a.gelu) lr_gelu(lo, hi, a.out_f32);
        const int at = tile * kLrTile + lane;
        const int64_t where = (o.first + row) * a.outer + at;
        if (at < a.outer) lr_store_one(a, where, o.bad ? nan : lo);
        if (at + 32 < a.outer) lr_store_one(a, where + 32, o.bad ? nan : hi);
      }
      __syncwarp();
    }
  }
}

template <int RT, int NT, bool F32>
__global__ void __launch_bounds__(kLrThreads, RT * NT <= (F32 ? 4 : 8) ? 2 : 1) low_rank_kernel(const __grid_constant__ LowRankArgs a) {
  using S = LrShape<RT, NT>;
  extern __shared__ __align__(16) uint8_t lr_smem[];
  __shared__ LrGroups<S::G> s;

  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  uint32_t ctas;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  const int C = static_cast<int>(ctas), c = C > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  float* const join = reinterpret_cast<float*>(lr_smem);
  float* const sums = join + S::JOIN / 4;  // [2][C][SUMS], where C > 1
  __nv_bfloat16* const terms = reinterpret_cast<__nv_bfloat16*>(sums + (C > 1 ? 2 * C * S::SUMS : 0));

  // the CTAs of the cluster all run before any writes into another's shared memory
  if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  griddep_wait();
  griddep_launch_dependents();

  const int cluster = static_cast<int>(blockIdx.x) / C;
  const int mine = cluster % a.clusters;
  LrColumns o;
  o.first = static_cast<int64_t>(cluster / a.clusters) * kLrWindow;
  o.rows = s.rows;
  o.terms = terms;
  o.stage = join + warp * S::STAGE;
  o.parts = a.out_f32 ? 3 : 2;
  const int n = static_cast<int>(min(static_cast<int64_t>(kLrWindow), a.rows - o.first));
  const int groups = s.form(a, o.first, n);
  if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

  // fewer groups than clusters: several share a group and split its columns
  const int split = max(1, min(a.clusters / groups, a.parts));
  const int part = split == 1 ? 0 : mine / groups;
  const int tiles = (a.outer + kLrTile - 1) / kLrTile;
  const int tile0 = (part * C + c) * kLrWarps + warp, stride = split * C * kLrWarps;
  int round = 0;  // of sums exchanged: two buffers, so that one barrier a round is enough
  for (int group = split == 1 ? mine : part < split ? mine % groups : groups; group < groups;
       group += split == 1 ? a.clusters : groups) {
    const int adapter = s.key[s.lead[group]];
    if (adapter < 0 && a.skip_bare) continue;
    __syncthreads();  // the rows, terms and stages of the group before are read
    const int many = s.take(group, n);
    o.bad = adapter >= a.count;
    o.up = adapter < 0 || o.bad ? nullptr : a.up + static_cast<int64_t>(adapter) * a.outer * a.rank;

    if (o.up != nullptr) {
      // the warp's first columns of up are on their way while the sums are taken
      for (int tile = tile0, k = 0; tile < tiles && k < 4; tile += stride, ++k) {
        const char* const p = reinterpret_cast<const char*>(o.up + static_cast<int64_t>(tile) * kLrTile * a.rank);
        const int bytes = min(kLrTile, a.outer - tile * kLrTile) * a.rank * 2;
        for (int at = lane * 128; at < bytes; at += 32 * 128) prefetch_l2(p + at);
      }
      // ---- sums over K: [ranks] x [rows of the group]
      float acc[RT][NT][4] = {};
      const __nv_bfloat16* xp[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int row = s.rows[i * 8 + g];
        xp[i] = row < 0 ? nullptr : a.x + (o.first + row) * a.inner + 8 * t;
      }
      const __nv_bfloat16* const dp = a.down + (static_cast<int64_t>(adapter) * a.rank + g) * a.inner + 8 * t;
      const int steps = (a.inner + 31) / 32, units = C * kLrWarps, unit = c * kLrWarps + warp;
      const int from = static_cast<int>(static_cast<int64_t>(steps) * unit / units);
      const int to = static_cast<int>(static_cast<int64_t>(steps) * (unit + 1) / units);
      const uint4 zero = make_uint4(0, 0, 0, 0);
      constexpr int U = RT * 2 + NT <= 6 ? 4 : RT * 2 + NT <= 12 ? 2 : 1;  // steps whose loads go out together
      for (int at = from; at < to; at += U) {
        uint4 w[U][RT][2], v[U][NT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int k = (at + u) * 32;
          const bool in = at + u < to && k + 8 * t < a.inner;
#pragma unroll
          for (int r = 0; r < RT; ++r) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int row = r * 16 + h * 8;
              w[u][r][h] = in && row + g < a.rank
                               ? __ldg(reinterpret_cast<const uint4*>(dp + static_cast<int64_t>(row) * a.inner + k))
                               : zero;
            }
          }
#pragma unroll
          for (int i = 0; i < NT; ++i)
            v[u][i] = in && xp[i] != nullptr ? __ldg(reinterpret_cast<const uint4*>(xp[i] + k)) : zero;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const uint4 lo = w[u][r][0], hi = w[u][r][1];
            const uint32_t one[4] = {lo.x, hi.x, lo.y, hi.y}, two[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
            for (int i = 0; i < NT; ++i) {
              if (i * 8 >= many) break;
              mma_m16n8k16_bf16(acc[r][i], one, v[u][i].x, v[u][i].y);
              mma_m16n8k16_bf16(acc[r][i], two, v[u][i].z, v[u][i].w);
            }
          }
        }
      }
      // ---- joined: warps, then CTAs, each in order
#pragma unroll
      for (int r = 0; r < RT; ++r) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
          *reinterpret_cast<float4*>(join + warp * S::SUMS + ((r * NT + i) * 32 + lane) * 4) =
              make_float4(acc[r][i][0], acc[r][i][1], acc[r][i][2], acc[r][i][3]);
      }
      __syncthreads();
      float* const shared_sums = sums + (round++ & 1) * C * S::SUMS;
      if (C > 1) {
        for (int i = tid; i < S::SUMS / 4; i += kLrThreads) {
          float4 v = *reinterpret_cast<const float4*>(join + i * 4);
#pragma unroll
          for (int w = 1; w < kLrWarps; ++w) {
            const float4 u = *reinterpret_cast<const float4*>(join + w * S::SUMS + i * 4);
            v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
          }
          for (int peer = 0; peer < C; ++peer) st_cluster_v4(peer_smem_addr(shared_sums + c * S::SUMS + i * 4, peer), v);
        }
        cluster_sync();
      }
      const float scale = __ldg(a.scales + adapter);
      const float* const from_all = C > 1 ? shared_sums : join;
      const int pieces = C > 1 ? C : kLrWarps;
      for (int i = tid; i < S::SUMS / 4; i += kLrThreads) {
        float4 v = *reinterpret_cast<const float4*>(from_all + i * 4);
        for (int w = 1; w < pieces; ++w) {
          const float4 u = *reinterpret_cast<const float4*>(from_all + w * S::SUMS + i * 4);
          v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
        }
        const int l = i % 32, tile = i / 32, r = tile / NT, q = tile % NT;
        const float y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at_rank = r * 16 + l / 4 + (e / 2) * 8, at_row = q * 8 + 2 * (l % 4) + e % 2;
          // no rank there: 0, also where x is infinite
          lr_terms(at_rank < a.rank ? y[e] * scale : 0.f, o.parts, terms + at_row * S::H_ROW + at_rank, S::TERM);
        }
      }
      __syncthreads();
    }

    // ---- columns
    if (many <= 8) {
      constexpr int TILES = RT * (F32 ? 2 : 1) <= 4 ? 2 : 1;
      for (int tile = tile0; tile < tiles; tile += TILES * stride) lr_columns<RT, NT, 1, TILES, F32>(a, o, tile, stride, tiles);
    } else if constexpr (NT > 1) {
      for (int tile = tile0; tile < tiles; tile += stride) lr_columns<RT, NT, NT, 1, F32>(a, o, tile, stride, tiles);
    }
  }
}

}  // namespace b200tx
