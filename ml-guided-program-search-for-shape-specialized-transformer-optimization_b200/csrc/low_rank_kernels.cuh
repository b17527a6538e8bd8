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
// tiles of 128 rows that share an adapter (low_rank_tile_kernels.cuh, for prompts); the tensor pipe is not what bounds this.
//
// What bounds it: the chain launch -> indices -> ranks -> sums over K -> exchange in the cluster -> columns, each about
// a microsecond, most of it trips to memory and barriers; and beyond a few groups the instructions of a tile (issue
// 32 % with two CTAs on an SM).  One row of 1024 -> 4096, rank 16: 5.0 us in a graph (0.6 indices, 0.5 ranks, 1.2 sums, 0.7 exchange,
// 0.35 terms, 0.8 columns).  64 rows of 32 adapters, 4096 -> 14336: 12 us for 19.9 MB (3.0 us at the copy rate; cold 16).  203 rows
// in no order, 4744 -> 5003, rank 24, 32 bits: 15 us for 12.4 MB.
//
// The R sums of a row are fp32.  The second product takes them as bf16 terms, each the rounded rest of the
// ones before: two (2^-17 of the sum is left) where the result has 16 bits, three (2^-25) where it has 32.  An infinity
// among up's values meets terms of either sign and zeros, so that NaN may stand where the formula has an infinity.
#pragma once

#include "attention_mma_kernels.cuh"

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
  int group;        // most rows of a group
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

  // Ranks the window's n rows; returns the number of groups.  All threads of the CTA, kLrThreads or more.
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
    const bool leads = tid < n && before % a.group == 0;
    const uint32_t leaders = __ballot_sync(0xffffffffu, leads);
    if (tid < kLrWindow) rank[tid] = before;
    if (lane == 0 && warp < kLrWarps) warp_leads[warp] = __popc(leaders);
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
  __device__ __forceinline__ int take(int group, int n, int most) {
    const int tid = threadIdx.x, leader = lead[group], adapter = key[leader], from = rank[leader];
    const bool in = tid < n && key[tid] == adapter && rank[tid] >= from && rank[tid] < from + most;
    if (tid < G) rows[tid] = -1;
    const int many = __syncthreads_count(in);
    if (in) rows[rank[tid] - from] = tid;
    __syncthreads();
    return many;
  }
};

// A build for RT tiles of 16 ranks: groups of up to NT eights of rows.  With more ranks two eights are enough for the
// registers (rank 64, 4096 -> 1024: 16 rows 7.9 us, with four 8.1; 256 rows 17.2 and 17.9).
template <int RT>
struct LrShape {
  static constexpr int NT = RT <= 2 ? 4 : 2;
  static constexpr int G = NT * 8;
  static constexpr bool TWO = RT <= 2;               // the registers leave room for two CTAs on an SM
  static constexpr int SUMS = RT * NT * 128;         // floats of a group's sums, as the MMA leaves them
  static constexpr int H_ROW = RT * 16 + 8;          // padded: a lane's 16 bytes of 8 rows fall into different banks
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

__device__ __noinline__ float lr_gelu_32(float x) { return 0.5f * x * (1.f + erff(x * 0.70710678118654752f)); }

// GELU for a result of 16 bits.  With a = |x|, GELU(x) = max(x, 0) - a Q(a), Q the normal distribution's tail,
// and -log2 Q is smooth: a polynomial of degree 7, fitted on [0, 6] for the least error of a Q(a).  The bound is an absolute
// one: with the polynomial in fp32 (1.05e-7) and the exponential (4.1e-8) a value is off by less than 1.5e-7.  That is 4e-4
// of the value itself down to x = -6, at most a fifth of the rounding of the result; below, where a value is smaller than
// 6e-9, 1.3 % at -7, and past -10 the size is wrong.  13 instructions; one value at a time, as pairs of values in one
// instruction want their constants in registers, and moves for them.
__device__ __forceinline__ float lr_gelu_16(float x) {
  float positive;  // with NaN kept
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(positive) : "f"(x));
  const float a = fminf(fabsf(x), 16.f);  // where the exponential is 0 by now, and the polynomial does not go down for ever
  float p = fmaf(-7.928164222903433e-07f, a, 4.487410114961676e-05f);
  p = fmaf(p, a, -0.0008306637755595148f);
  p = fmaf(p, a, 0.008231189101934433f);
  p = fmaf(p, a, -0.05359907075762749f);
  p = fmaf(p, a, -0.45865529775619507f);
  p = fmaf(p, a, -1.151233434677124f);
  p = fmaf(p, a, -0.9999903440475464f);
  // -a, without the clamp where x is negative: -infinity times 0 is NaN, as in x Phi(x)
  return fmaf(fminf(x, -a), fast_exp2(p), positive);
}

// GELU of two values, by the library's erf where the result has 32 bits.
__device__ __forceinline__ void lr_gelu(float& x, float& y, bool f32) {
  if (f32) {
    x = lr_gelu_32(x);
    y = lr_gelu_32(y);
  } else {
    x = lr_gelu_16(x);
    y = lr_gelu_16(y);
  }
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// Eight neighbouring values of a row of base, as they lie.
template <bool F32>
struct LrEight {
  uint4 w[F32 ? 2 : 1];

  __device__ __forceinline__ void load(const uint8_t* p) {
#pragma unroll
    for (int i = 0; i < (F32 ? 2 : 1); ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
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

// A warp's 64 columns of up, as the MMA takes them: 4 ranks a lane of its 8 columns, or 8 of each 32.
template <int RT>
struct LrUp {
  static constexpr int CHUNKS = RT == 1 ? 1 : RT / 2;
  static constexpr int KEPT = CHUNKS <= 2 ? CHUNKS : 1;  // more than the registers hold are read for each eight of rows
  uint32_t w[KEPT][8][RT == 1 ? 2 : 4];

  // p: the adapter's up at the lane's first column and rank
  __device__ __forceinline__ void load(const LowRankArgs& a, const __nv_bfloat16* p, int to, int chunk, int columns) {
    const int rank = (RT == 1 ? 4 : 8) * (threadIdx.x % 4) + chunk * 32;
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const __nv_bfloat16* const at = p + m * a.rank + chunk * 32;
      const bool in = m < columns && rank < a.rank;
      if constexpr (RT == 1) {
        const uint2 v = in ? __ldg(reinterpret_cast<const uint2*>(at)) : make_uint2(0, 0);
        w[to][m][0] = v.x, w[to][m][1] = v.y;
      } else {
        const uint4 v = in ? __ldg(reinterpret_cast<const uint4*>(at)) : make_uint4(0, 0, 0, 0);
        w[to][m][0] = v.x, w[to][m][1] = v.y, w[to][m][2] = v.z, w[to][m][3] = v.w;
      }
    }
  }

  // Adds the product with the rows' terms at p (16 or 32 ranks).
  __device__ __forceinline__ void add(int from, const __nv_bfloat16* p, float (&acc)[4][4]) const {
    if constexpr (RT == 1) {
      const uint2 b = *reinterpret_cast<const uint2*>(p);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const uint32_t f[4] = {w[from][2 * m][0], w[from][2 * m + 1][0], w[from][2 * m][1], w[from][2 * m + 1][1]};
        mma_m16n8k16_bf16(acc[m], f, b.x, b.y);
      }
    } else {
      const uint4 b = *reinterpret_cast<const uint4*>(p);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const uint32_t f[4] = {w[from][2 * m][0], w[from][2 * m + 1][0], w[from][2 * m][1], w[from][2 * m + 1][1]};
        const uint32_t h[4] = {w[from][2 * m][2], w[from][2 * m + 1][2], w[from][2 * m][3], w[from][2 * m + 1][3]};
        mma_m16n8k16_bf16(acc[m], f, b.x, b.y);
        mma_m16n8k16_bf16(acc[m], h, b.z, b.w);
      }
    }
  }
};

// F32: base has 32 bits.  WHOLE: the rows of base and out are multiples of 16 bytes.
// The code is kept short (few copies of the inner parts): a call lasts so few microseconds
// that instructions which are run once cost what fetching them takes.
template <int RT, bool F32, bool WHOLE>
__global__ void __launch_bounds__(kLrThreads, LrShape<RT>::TWO ? 2 : 1) low_rank_kernel(const __grid_constant__ LowRankArgs a) {
  using S = LrShape<RT>;
  constexpr int NT = S::NT;
  constexpr bool EARLY = RT <= 2;  // up's first columns are loaded before the sums are taken
  extern __shared__ __align__(16) uint8_t lr_smem[];
  __shared__ LrGroups<S::G> s;

  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  uint32_t ctas;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  const int C = static_cast<int>(ctas), c = C > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  float* const join = reinterpret_cast<float*>(lr_smem);
  float* const sums = join + S::JOIN / 4;  // [2][C][SUMS], where C > 1
  __nv_bfloat16* const terms = reinterpret_cast<__nv_bfloat16*>(sums + (C > 1 ? 2 * C * S::SUMS : 0));
  float* const stage = join + warp * S::STAGE;

  // the CTAs of the cluster all run before any writes into another's shared memory
  if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  griddep_wait();
  griddep_launch_dependents();

  const int cluster = static_cast<int>(blockIdx.x) / C;
  const int mine = cluster % a.clusters;
  const int64_t first = static_cast<int64_t>(cluster / a.clusters) * kLrWindow;
  const int n = static_cast<int>(min(static_cast<int64_t>(kLrWindow), a.rows - first));
  const int groups = s.form(a, first, n);
  if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

  const int parts = a.out_f32 ? 3 : 2;  // terms that the sums are split into
  const float nan = __int_as_float(0x7fffffff);
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
    const int many = s.take(group, n, a.group);
    const bool bad = adapter >= a.count, bare = adapter < 0 || bad;

    // the warp's columns, from its first tile on
    LrUp<RT> next;
    LrEight<F32> next_base[2];
    const __nv_bfloat16* const up = a.up + (static_cast<int64_t>(bare ? 0 : adapter) * a.outer + 8 * g) * a.rank + (RT == 1 ? 4 : 8) * t;
    auto load_up = [&](int tile, int to, int chunk) {
      const int col = tile * kLrTile;
      next.load(a, up + static_cast<int64_t>(col) * a.rank, to, chunk, a.outer - col - 8 * g);
    };
    auto load_base = [&](int tile, int i) {
      const int col = tile * kLrTile + 8 * g;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = s.rows[i * 8 + 2 * t + e];
        if (row >= 0 && col < a.outer)
          next_base[e].load(static_cast<const uint8_t*>(a.base) + ((first + row) * a.outer + col) * (F32 ? 4 : 2));
      }
    };
    // where rows start anywhere: 64 neighbouring values of each of 8 rows by a warp
    float next_y[8][2] = {};
    auto load_ragged = [&](int tile, int i) {
      const int at = tile * kLrTile + lane, here = many - i * 8;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        if (r >= here) break;
        const int64_t where = (first + s.rows[i * 8 + r]) * a.outer + at;
        if (at < a.outer) next_y[r][0] = lr_load_one<F32>(a, where);
        if (at + 32 < a.outer) next_y[r][1] = lr_load_one<F32>(a, where + 32);
      }
    };
    auto load_rows = [&](int tile, int i) {
      if constexpr (WHOLE)
        load_base(tile, i);
      else
        load_ragged(tile, i);
    };
    if (tile0 < tiles) load_rows(tile0, 0);

    if (!bare) {
      if (EARLY && tile0 < tiles) {
#pragma unroll
        for (int r = 0; r < LrUp<RT>::KEPT; ++r) load_up(tile0, r, r);
      }
      // the columns after these come nearer while the sums are taken
      for (int tile = EARLY ? tile0 + stride : tile0, k = 0; tile < tiles && k < 4; tile += stride, ++k) {
        const char* const p = reinterpret_cast<const char*>(a.up + (static_cast<int64_t>(adapter) * a.outer + tile * kLrTile) * a.rank);
        const int bytes = min(kLrTile, a.outer - tile * kLrTile) * a.rank * 2;
        for (int at = lane * 128; at < bytes; at += 32 * 128) prefetch_l2(p + at);
      }
      // ---- sums over K: [ranks] x [rows of the group]
      float acc[RT][NT][4] = {};
      const int steps = (a.inner + 31) / 32, units = C * kLrWarps, unit = c * kLrWarps + warp;
      const int from = static_cast<int>(static_cast<int64_t>(steps) * unit / units);
      const int to = static_cast<int>(static_cast<int64_t>(steps) * (unit + 1) / units);
      const __nv_bfloat16* xp[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) xp[i] = a.x + (first + max(s.rows[i * 8 + g], 0)) * a.inner + from * 32 + 8 * t;
      const __nv_bfloat16* dp = a.down + (static_cast<int64_t>(adapter) * a.rank + g) * a.inner + from * 32 + 8 * t;
      const uint4 zero = make_uint4(0, 0, 0, 0);
      constexpr int U = RT == 1 ? 2 : 1;  // steps whose loads go out together
#pragma unroll 1
      for (int at = from; at < to; at += U) {
        uint4 w[U][RT][2], v[U][NT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const bool in = at + u < to && (at + u) * 32 + 8 * t < a.inner;
#pragma unroll
          for (int r = 0; r < RT; ++r) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int row = r * 16 + h * 8;
              w[u][r][h] = in && row + g < a.rank
                               ? __ldg(reinterpret_cast<const uint4*>(dp + static_cast<int64_t>(row) * a.inner + u * 32))
                               : zero;
            }
          }
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            if (i * 8 >= many) break;
            v[u][i] = in && i * 8 + g < many ? __ldg(reinterpret_cast<const uint4*>(xp[i] + u * 32)) : zero;
          }
        }
        dp += U * 32;
#pragma unroll
        for (int i = 0; i < NT; ++i) xp[i] += U * 32;
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            if (i * 8 >= many) break;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              const uint4 lo = w[u][r][0], hi = w[u][r][1];
              const uint32_t one[4] = {lo.x, hi.x, lo.y, hi.y}, two[4] = {lo.z, hi.z, lo.w, hi.w};
              mma_m16n8k16_bf16(acc[r][i], one, v[u][i].x, v[u][i].y);
              mma_m16n8k16_bf16(acc[r][i], two, v[u][i].z, v[u][i].w);
            }
          }
        }
      }
      // ---- joined: warps, then CTAs, each in order
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        if (i * 8 >= many) break;
#pragma unroll
        for (int r = 0; r < RT; ++r)
          *reinterpret_cast<float4*>(join + warp * S::SUMS + ((i * RT + r) * 32 + lane) * 4) =
              make_float4(acc[r][i][0], acc[r][i][1], acc[r][i][2], acc[r][i][3]);
      }
      __syncthreads();
      const int held = (many + 7) / 8 * RT * 32;  // float4s of the rows that there are
      float* const shared_sums = sums + (round++ & 1) * C * S::SUMS;
      if (C > 1) {
        // a warp for each CTA that the sums go to, in turn
        for (int i = lane; i < held; i += 32) {
          float4 v = *reinterpret_cast<const float4*>(join + i * 4);
#pragma unroll
          for (int w = 1; w < kLrWarps; ++w) {
            const float4 u = *reinterpret_cast<const float4*>(join + w * S::SUMS + i * 4);
            v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
          }
          for (int peer = warp; peer < C; peer += kLrWarps) st_cluster_v4(peer_smem_addr(shared_sums + c * S::SUMS + i * 4, peer), v);
        }
        cluster_sync();
      }
      const float scale = __ldg(a.scales + adapter);
      const float* const from_all = C > 1 ? shared_sums : join;
      const int pieces = C > 1 ? C : kLrWarps;
      for (int i = tid; i < held * 4; i += kLrThreads) {
        float v = from_all[i];
        for (int w = 1; w < pieces; ++w) v += from_all[w * S::SUMS + i];
        const int e = i % 4, l = i / 4 % 32, tile = i / 128, q = tile / RT, r = tile % RT;
        const int at_rank = r * 16 + l / 4 + (e / 2) * 8, at_row = q * 8 + 2 * (l % 4) + e % 2;
        // no rank there: 0, also where x is infinite
        lr_terms(at_rank < a.rank ? v * scale : 0.f, parts, terms + at_row * S::H_ROW + at_rank, S::TERM);
      }
      __syncthreads();
    }

    // ---- columns
#pragma unroll 1
    for (int tile = tile0; tile < tiles; tile += stride) {
      if (!EARLY && !bare) {
#pragma unroll
        for (int r = 0; r < LrUp<RT>::KEPT; ++r)
          if (LrUp<RT>::CHUNKS == LrUp<RT>::KEPT) load_up(tile, r, r);
      }
      const LrUp<RT> now = next;
      if (EARLY && !bare && tile + stride < tiles) {
#pragma unroll
        for (int r = 0; r < LrUp<RT>::KEPT; ++r) load_up(tile + stride, r, r);
      }
      const int col = tile * kLrTile + 8 * g;
#pragma unroll 1
      for (int i = 0; i * 8 < many; ++i) {
        const LrEight<F32> base[2] = {next_base[0], next_base[1]};
        float y8[8][2];
#pragma unroll
        for (int r = 0; r < 8; ++r) y8[r][0] = next_y[r][0], y8[r][1] = next_y[r][1];
        // the next eight rows' values, or the next columns', before a store that might be to the same place
        if ((i + 1) * 8 < many)
          load_rows(tile, i + 1);
        else if (tile + stride < tiles)
          load_rows(tile + stride, 0);
        float acc[4][4] = {};
        if (!bare) {
          const __nv_bfloat16* const p = terms + (i * 8 + g) * S::H_ROW + (RT == 1 ? 4 : 8) * t;
          if constexpr (LrUp<RT>::CHUNKS == LrUp<RT>::KEPT) {
#pragma unroll
            for (int r = 0; r < LrUp<RT>::KEPT; ++r) {
#pragma unroll 1
              for (int k = 0; k < parts; ++k) now.add(r, p + k * S::TERM + r * 32, acc);
            }
          } else {
#pragma unroll 1
            for (int r = 0; r < LrUp<RT>::CHUNKS; ++r) {
              load_up(tile, 0, r);
#pragma unroll 1
              for (int k = 0; k < parts; ++k) next.add(0, p + k * S::TERM + r * 32, acc);
            }
          }
        }
        if constexpr (WHOLE) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = s.rows[i * 8 + 2 * t + e];
            if (row < 0 || col >= a.outer) continue;
            float y[8];
            base[e].values(y);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              y[2 * m] += acc[m][e];
              y[2 * m + 1] += acc[m][2 + e];
            }
            if (bad) {
#pragma unroll
              for (int m = 0; m < 8; ++m) y[m] = nan;
            }
            lr_store_eight(a, (first + row) * a.outer + col, y);
          }
        } else {
          // Rows that start anywhere: turned in shared memory, so that a warp reads and writes 32 neighbouring values.
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float4* const to = reinterpret_cast<float4*>(stage + (2 * t + e) * kLrStageRow + 8 * g);
            to[0] = make_float4(acc[0][e], acc[0][2 + e], acc[1][e], acc[1][2 + e]);
            to[1] = make_float4(acc[2][e], acc[2][2 + e], acc[3][e], acc[3][2 + e]);
          }
          __syncwarp();
          const int at = tile * kLrTile + lane, here = min(many - i * 8, 8);
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            if (r >= here) break;
            float lo = y8[r][0] + stage[r * kLrStageRow + lane], hi = y8[r][1] + stage[r * kLrStageRow + 32 + lane];
            if (a.gelu) lr_gelu(lo, hi, a.out_f32);
            const int64_t where = (first + s.rows[i * 8 + r]) * a.outer + at;
            if (at < a.outer) lr_store_one(a, where, bad ? nan : lo);
            if (at + 32 < a.outer) lr_store_one(a, where + 32, bad ? nan : hi);
          }
          __syncwarp();
        }
      }
    }
  }
}

}  // namespace b200tx
