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
// The R sums of a row are fp32.  The second product takes them as two bf16 terms, the rounded value and
// the rounded rest (2^-17 relative), so that they cost no accuracy beside fp32.
#pragma once

#include "attention_mma_kernels.cuh"
#include "gemm_kernels.cuh"

namespace b200tx {

constexpr int kLrWarps = 8;
constexpr int kLrThreads = kLrWarps * 32;
constexpr int kLrWindow = kLrThreads;  // rows among which groups are formed
constexpr int kLrTile = 64;            // columns of the result that a warp takes at a time

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

// Floats of a group's sums, as the MMA leaves them: RT tiles of 16 ranks, NT of 8 rows.
template <int RT, int NT>
struct LrShape {
  static constexpr int G = NT * 8;
  static constexpr int SUMS = RT * NT * 128;
  static constexpr int H_ROW = RT * 16 + 8;  // padded: a lane's 16 bytes of 8 rows fall into different banks
  static constexpr int H_BYTES = 2 * G * H_ROW * 2;
  static constexpr int JOIN = kLrWarps * SUMS * 4;
  // shared memory with `ctas` in a cluster: warps' sums, two rounds of the CTAs' sums, the terms
  static constexpr int bytes(int ctas) { return JOIN + (ctas > 1 ? 2 * ctas * SUMS * 4 : 0) + H_BYTES; }
};

__device__ __forceinline__ void st_cluster_v4(uint32_t addr, const float4& v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}

__device__ __forceinline__ float lr_activate(float y, bool gelu) {
  return gelu ? 0.5f * y * (1.f + erff(y * 0.70710678118654752f)) : y;
}

// Eight neighbouring values of a row of base, as they lie.
template <bool F32>
struct LrEight {
  uint4 w[F32 ? 2 : 1];

  __device__ __forceinline__ void load(const LowRankArgs& a, int64_t at, int valid) {
    const uint8_t* const p = static_cast<const uint8_t*>(a.base) + at * (F32 ? 4 : 2);
    if (valid == 8 && a.outer % 8 == 0) {
#pragma unroll
      for (int i = 0; i < (F32 ? 2 : 1); ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
      return;
    }
    uint32_t v[F32 ? 8 : 4] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i >= valid) break;
      if (F32)
        v[i] = reinterpret_cast<const uint32_t*>(p)[i];
      else
        v[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[i]) << (i % 2 * 16);
    }
#pragma unroll
    for (int i = 0; i < (F32 ? 2 : 1); ++i) w[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
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

__device__ __forceinline__ void lr_store(const LowRankArgs& a, int64_t at, int valid, float (&y)[8]) {
  if (a.gelu) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = lr_activate(y[i], true);
  }
  if (valid == 8 && a.outer % 8 == 0) {
    if (a.out_f32) {
      float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.out) + at);
      p[0] = make_float4(y[0], y[1], y[2], y[3]);
      p[1] = make_float4(y[4], y[5], y[6], y[7]);
    } else {
      *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + at) =
          make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i >= valid) break;
    if (a.out_f32)
      static_cast<float*>(a.out)[at + i] = y[i];
    else
      static_cast<__nv_bfloat16*>(a.out)[at + i] = __float2bfloat16(y[i]);
  }
}

template <int RT, int NT, bool F32>
__global__ void __launch_bounds__(kLrThreads, RT * NT <= (F32 ? 4 : 8) ? 2 : 1) low_rank_kernel(const __grid_constant__ LowRankArgs a) {
  using S = LrShape<RT, NT>;
  extern __shared__ __align__(16) uint8_t lr_smem[];
  __shared__ __align__(16) int s_key[kLrWindow];
  __shared__ __align__(16) int s_rank[kLrWindow];
  __shared__ __align__(16) int s_lead[kLrWindow];
  __shared__ int s_warp_leads[kLrWarps];
  __shared__ int s_rows[S::G];

  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  uint32_t ctas;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  const int C = static_cast<int>(ctas), c = C > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  float* const join = reinterpret_cast<float*>(lr_smem);
  float* const sums = join + kLrWarps * S::SUMS;  // [2][C][SUMS], where C > 1
  __nv_bfloat16* const terms = reinterpret_cast<__nv_bfloat16*>(sums + (C > 1 ? 2 * C * S::SUMS : 0));  // [2][G][H_ROW]

  // the CTAs of the cluster all run before any writes into another's shared memory
  if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  griddep_wait();
  griddep_launch_dependents();

  const int cluster = static_cast<int>(blockIdx.x) / C;
  const int64_t first = static_cast<int64_t>(cluster / a.clusters) * kLrWindow;
  const int mine = cluster % a.clusters;
  const int n = static_cast<int>(min(static_cast<int64_t>(kLrWindow), a.rows - first));

  // groups: equal indices by their order
  if (tid < n) {
    const int index = a.indices[static_cast<unsigned>(first + tid) / static_cast<unsigned>(a.per_index)];
    s_key[tid] = index < 0 ? -1 : min(index, a.count);
  }
  __syncthreads();
  int rank = 0;
  const int key = tid < n ? s_key[tid] : 0;
  if (tid < n) {
    for (int j = 0; j < (tid & ~31); j += 4) {
      const int4 k = *reinterpret_cast<const int4*>(s_key + j);
      rank += (k.x == key) + (k.y == key) + (k.z == key) + (k.w == key);
    }
  }
  const uint32_t same = __match_any_sync(0xffffffffu, tid < n ? key : -2);
  rank += __popc(same & ((1u << lane) - 1));
  const bool leads = tid < n && rank % S::G == 0;
  const uint32_t leaders = __ballot_sync(0xffffffffu, leads);
  s_rank[tid] = rank;
  if (lane == 0) s_warp_leads[warp] = __popc(leaders);
  __syncthreads();
  int groups = 0, before = 0;
#pragma unroll
  for (int w = 0; w < kLrWarps; ++w) {
    if (w == warp) before = groups;
    groups += s_warp_leads[w];
  }
  if (leads) s_lead[before + __popc(leaders & ((1u << lane) - 1))] = tid;
  __syncthreads();
  if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

  // fewer groups than clusters: several share a group and split its columns
  const int split = max(1, min(a.clusters / groups, a.parts));
  const int part = split == 1 ? 0 : mine / groups;
  int round = 0;  // of sums exchanged: two buffers, so that one barrier a round is enough
  for (int group = split == 1 ? mine : part < split ? mine % groups : groups; group < groups;
       group += split == 1 ? a.clusters : groups) {
    const int leader = s_lead[group];
    const int adapter = s_key[leader], rank0 = s_rank[leader];
    if (adapter < 0 && a.skip_bare) continue;
    __syncthreads();  // s_rows and terms of the group before are read
    if (tid < S::G) s_rows[tid] = -1;
    __syncthreads();
    if (tid < n && s_key[tid] == adapter && s_rank[tid] >= rank0 && s_rank[tid] < rank0 + S::G) s_rows[s_rank[tid] - rank0] = tid;
    __syncthreads();
    const bool bare = adapter < 0 || adapter >= a.count;

    if (!bare) {
      // ---- sums over K: [ranks] x [rows of the group]
      float acc[RT][NT][4] = {};
      const __nv_bfloat16* xp[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int row = s_rows[i * 8 + g];
        xp[i] = row < 0 ? nullptr : a.x + (first + row) * a.inner + 8 * t;
      }
      const __nv_bfloat16* const dp = a.down + (static_cast<int64_t>(adapter) * a.rank + g) * a.inner + 8 * t;
      const int steps = (a.inner + 31) / 32, units = C * kLrWarps, unit = c * kLrWarps + warp;
      const int from = static_cast<int>(static_cast<int64_t>(steps) * unit / units);
      const int to = static_cast<int>(static_cast<int64_t>(steps) * (unit + 1) / units);
      const uint4 zero = make_uint4(0, 0, 0, 0);
      constexpr int U = RT * 2 + NT <= 6 ? 4 : RT * 2 + NT <= 12 ? 2 : 1;  // steps whose loads go out together
      for (int s = from; s < to; s += U) {
        uint4 w[U][RT][2], v[U][NT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int k = (s + u) * 32;
          const bool in = s + u < to && k + 8 * t < a.inner;
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
          float4 s = *reinterpret_cast<const float4*>(join + i * 4);
#pragma unroll
          for (int w = 1; w < kLrWarps; ++w) {
            const float4 o = *reinterpret_cast<const float4*>(join + w * S::SUMS + i * 4);
            s.x += o.x, s.y += o.y, s.z += o.z, s.w += o.w;
          }
          for (int peer = 0; peer < C; ++peer) st_cluster_v4(peer_smem_addr(shared_sums + c * S::SUMS + i * 4, peer), s);
        }
        cluster_sync();
      }
      const float scale = __ldg(a.scales + adapter);
      const float* const from_all = C > 1 ? shared_sums : join;
      const int many = C > 1 ? C : kLrWarps;
      for (int i = tid; i < S::SUMS / 4; i += kLrThreads) {
        float4 s = *reinterpret_cast<const float4*>(from_all + i * 4);
        for (int w = 1; w < many; ++w) {
          const float4 o = *reinterpret_cast<const float4*>(from_all + w * S::SUMS + i * 4);
          s.x += o.x, s.y += o.y, s.z += o.z, s.w += o.w;
        }
        const int l = i % 32, tile = i / 32, r = tile / NT, q = tile % NT;
        const float y[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at_rank = r * 16 + l / 4 + (e / 2) * 8, at_row = q * 8 + 2 * (l % 4) + e % 2;
          // no rank there: 0, also where x is infinite
          const float h = at_rank < a.rank ? y[e] * scale : 0.f;
          const __nv_bfloat16 near = __float2bfloat16(h);
          const float rest = h - __bfloat162float(near);
          terms[at_row * S::H_ROW + at_rank] = near;
          terms[(S::G + at_row) * S::H_ROW + at_rank] = __float2bfloat16(fabsf(h) <= 3.38e38f ? rest : 0.f);
        }
      }
      __syncthreads();
    }

    // ---- columns
    const int tiles = (a.outer + kLrTile - 1) / kLrTile;
    const __nv_bfloat16* const up = a.up + static_cast<int64_t>(bare ? 0 : adapter) * a.outer * a.rank;
    for (int tile = (part * C + c) * kLrWarps + warp; tile < tiles; tile += split * C * kLrWarps) {
      const int col = tile * kLrTile + 8 * g;
      const int valid = min(max(a.outer - col, 0), 8);
      // base goes out first: no load of it waits behind a store that might be to the same place
      LrEight<F32> base[NT][2];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = s_rows[i * 8 + 2 * t + e];
          if (row >= 0 && valid > 0) base[i][e].load(a, (first + row) * a.outer + col, valid);
        }
      }
      float acc[4][NT][4] = {};
      if (!bare) {
        if constexpr (RT == 1) {
          // 4 ranks a lane
          uint2 w[4][2];
#pragma unroll
          for (int m = 0; m < 4; ++m) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              w[m][h] = 2 * m + h < valid && 4 * t < a.rank
                            ? __ldg(reinterpret_cast<const uint2*>(up + static_cast<int64_t>(col + 2 * m + h) * a.rank + 4 * t))
                            : make_uint2(0, 0);
            }
          }
#pragma unroll
          for (int i = 0; i < NT; ++i) {
#pragma unroll
            for (int part2 = 0; part2 < 2; ++part2) {
              const uint2 b = *reinterpret_cast<const uint2*>(terms + (part2 * S::G + i * 8 + g) * S::H_ROW + 4 * t);
#pragma unroll
              for (int m = 0; m < 4; ++m) {
                const uint32_t f[4] = {w[m][0].x, w[m][1].x, w[m][0].y, w[m][1].y};
                mma_m16n8k16_bf16(acc[m][i], f, b.x, b.y);
              }
            }
          }
        } else {
#pragma unroll(RT <= 4 ? RT / 2 : 2)
          for (int r = 0; r < RT / 2; ++r) {
            uint4 w[4][2];
#pragma unroll
            for (int m = 0; m < 4; ++m) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                w[m][h] = 2 * m + h < valid && r * 32 + 8 * t < a.rank
                              ? __ldg(reinterpret_cast<const uint4*>(up + static_cast<int64_t>(col + 2 * m + h) * a.rank + r * 32 + 8 * t))
                              : make_uint4(0, 0, 0, 0);
              }
            }
#pragma unroll
            for (int i = 0; i < NT; ++i) {
#pragma unroll
              for (int part2 = 0; part2 < 2; ++part2) {
                const uint4 b = *reinterpret_cast<const uint4*>(terms + (part2 * S::G + i * 8 + g) * S::H_ROW + r * 32 + 8 * t);
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                  const uint32_t one[4] = {w[m][0].x, w[m][1].x, w[m][0].y, w[m][1].y};
                  const uint32_t two[4] = {w[m][0].z, w[m][1].z, w[m][0].w, w[m][1].w};
                  mma_m16n8k16_bf16(acc[m][i], one, b.x, b.y);
                  mma_m16n8k16_bf16(acc[m][i], two, b.z, b.w);
                }
              }
            }
          }
        }
      }
      if (valid == 0) continue;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = s_rows[i * 8 + 2 * t + e];
          if (row < 0) continue;
          const int64_t at = (first + row) * a.outer + col;
          float y[8];
          if (adapter >= a.count) {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = __int_as_float(0x7fffffff);
          } else {
            base[i][e].values(y);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              y[2 * m] += acc[m][i][e];
              y[2 * m + 1] += acc[m][i][2 + e];
            }
          }
          lr_store(a, at, valid, y);
        }
      }
    }
  }
}

}  // namespace b200tx
