// low_rank_tile_kernels.cuh -- low-rank adapters beside a shared projection, for
// many rows with few adapters (prompts): what low_rank_kernels.cuh computes,
// 128 rows of an adapter at a time on tcgen05.
//
// A CTA takes a group of up to 128 rows (found as there) and a part of the columns:
//   1. sums = x . down^T over K, 128 x R, accumulated in TMEM; x (rows gathered from
//      anywhere) and down come in 64-column stages by cp.async into the 128-byte swizzled
//      layout that the UMMA reads, which leaves the rows free and any multiple of 8 for K;
//   2. the sums, scaled, become bf16 terms in shared memory (each the rounded rest of the ones before);
//   3. for each 128 columns: terms . up^T into one of two TMEM buffers, while the warps bring
//      the buffer before to the result: a warp turns 32 rows x 32 columns in shared memory, so
//      that base is read and the result written in whole 64-byte pieces of rows.
//
// Bound by the bytes of base and the result, which are 9 of 10 of a feed-forward layer's: the weights of
// an adapter are read (from L2) once for 128 rows, and two CTAs on an SM cover each other's waits.
// The warp MMA form of this reads them for every 32 rows and keeps the tensor pipe busy for as long as the bytes take.
//
// All threads do all of it in step; one of them issues the UMMAs.  Waits are bounded as everywhere.
#pragma once

#include "kv8_attention_kernels.cuh"
#include "low_rank_kernels.cuh"

namespace b200tx {

constexpr int kLtRows = 128;
constexpr int kLtColumns = 128;          // of the result, for one round
constexpr int kLtStages = 4;             // of 64 values of K
constexpr int kLtTurnRow = 36;           // floats: 32, padded so that 8 rows fall into different banks
constexpr uint32_t kLtXBytes = kLtRows * 128;
constexpr uint32_t kLtTurnBytes = kLrWarps * 32 * kLtTurnRow * 4;
constexpr int kErrLowRankWait = 0x501;

// RA atoms of 64 ranks.
template <int RA>
struct LtShape {
  static constexpr uint32_t UP = RA * kLtColumns * 128;  // a round's columns of up
  static constexpr uint32_t TERM = RA * kLtRows * 128;
  __host__ __device__ static constexpr uint32_t stage(int rank16) { return kLtXBytes + rank16 * 128; }
  // the stages of the sums, and later the terms, two rounds' columns and the turned results, in the same place
  __host__ __device__ static constexpr uint32_t bytes(int rank16, int terms) {
    return (kLtStages * stage(rank16) > terms * TERM + 2 * UP + kLtTurnBytes ? kLtStages * stage(rank16)
                                                                            : terms * TERM + 2 * UP + kLtTurnBytes) + 1024;
  }
};

// Where 16 bytes of a 128-byte row stand under the 128-byte swizzle.
__device__ __forceinline__ uint32_t lt_place(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

template <int RA, bool F32, bool WHOLE>
__global__ void __launch_bounds__(kLrThreads, RA == 1 ? 2 : 1) low_rank_tile_kernel(const __grid_constant__ LowRankArgs a) {
  using S = LtShape<RA>;
  extern __shared__ uint8_t lt_smem[];
  __shared__ LrGroups<kLtRows> s;
  __shared__ uint64_t stage_bar[kLtStages], round_bar[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;

  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  uint8_t* const smem = align_1024(lt_smem);
  const uint32_t smem0 = smem_u32(smem);
  const int rank16 = (a.rank + 15) / 16 * 16, parts = a.out_f32 ? 3 : 2;
  const uint32_t up0 = smem0 + parts * S::TERM;
  float* const turn = reinterpret_cast<float*>(smem + parts * S::TERM + 2 * S::UP) + warp * 32 * kLtTurnRow;

  if (tid == 0) {
    for (int i = 0; i < kLtStages; ++i) mbar_init(&stage_bar[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&round_bar[i], 1);
    fence_barrier_init();
    abort_flag = 0;
  }
  if (warp == 0) {
    tmem_alloc(&tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  const int mine = blockIdx.x % a.clusters;
  const int64_t first = static_cast<int64_t>(blockIdx.x / a.clusters) * kLrWindow;
  const int n = static_cast<int>(min(static_cast<int64_t>(kLrWindow), a.rows - first));
  const int groups = s.form(a, first, n);
  const int split = max(1, min(a.clusters / groups, a.parts));
  const int part = split == 1 ? 0 : mine / groups;
  const int all_rounds = (a.outer + kLtColumns - 1) / kLtColumns;
  const int round0 = all_rounds * part / split, rounds = all_rounds * (part + 1) / split - round0;
  const float nan = __int_as_float(0x7fffffff);
  const uint32_t sums_tmem = tmem + 128;  // the second round's columns: free until then
  uint32_t steps_done = 0, rounds_done = 0;
  bool ok = true;

  for (int group = split == 1 ? mine : part < split ? mine % groups : groups; group < groups && ok;
       group += split == 1 ? a.clusters : groups) {
    const int adapter = s.key[s.lead[group]];
    if (adapter < 0 && a.skip_bare) continue;
    tc_fence_before();
    __syncthreads();
    const int many = s.take(group, n, a.group);
    const bool bad = adapter >= a.count, bare = adapter < 0 || bad;
    const __nv_bfloat16* const up = a.up + static_cast<int64_t>(bare ? 0 : adapter) * a.outer * a.rank;

    // 128 columns of up, K-major; ranks past the adapter's up to a multiple of 16, and columns past the last, are zero
    auto load_up = [&](int round) {
      const int chunks = rank16 / 8;
      const uint32_t to = up0 + (round & 1) * S::UP;
      for (int i = tid; i < kLtColumns * chunks; i += kLrThreads) {
        const int col = i / chunks, chunk = i - col * chunks, at = (round0 + round) * kLtColumns + col;
        const bool in = at < a.outer && chunk * 8 < a.rank;
        cp_async_or_zero(to + chunk / 8 * (kLtColumns * 128) + lt_place(col, chunk % 8),
                         up + (in ? static_cast<int64_t>(at) * a.rank + chunk * 8 : 0), in);
      }
      cp_async_commit();
    };

    if (!bare) {
      // ---- sums over K
      const int steps = (a.inner + 63) / 64;
      const uint32_t stage_bytes = S::stage(rank16);
      const __nv_bfloat16* const down = a.down + static_cast<int64_t>(adapter) * a.rank * a.inner;
      // a thread's pieces: 16 bytes at the same place of every 32nd row
      const int chunk = tid % 8, row0 = tid / 8;
      const __nv_bfloat16* xp[kLtRows / 32];
#pragma unroll
      for (int i = 0; i < kLtRows / 32; ++i) xp[i] = a.x + (first + max(s.rows[row0 + 32 * i], 0)) * a.inner + chunk * 8;
      auto load_stage = [&](int step) {
        const uint32_t to = smem0 + (steps_done + step) % kLtStages * stage_bytes;
        const bool in = step * 64 + chunk * 8 < a.inner;
#pragma unroll
        for (int i = 0; i < kLtRows / 32; ++i) {
          const bool take = in && row0 + 32 * i < many;
          cp_async_or_zero(to + lt_place(row0 + 32 * i, chunk), take ? xp[i] + step * 64 : a.x, take);
        }
        for (int row = row0; row < rank16; row += 32) {
          const bool take = in && row < a.rank;
          cp_async_or_zero(to + kLtXBytes + lt_place(row, chunk),
                           down + (take ? static_cast<int64_t>(row) * a.inner + step * 64 + chunk * 8 : 0), take);
        }
      };
      for (int i = 0; i < kLtStages - 1; ++i) {
        if (i < steps) load_stage(i);
        cp_async_commit();
      }
      const uint32_t idesc = umma_idesc_bf16(kLtRows, rank16, false, false);
      for (int step = 0; step < steps; ++step) {
        cp_async_wait<kLtStages - 2>();
        fence_proxy_async_smem();
        if (__syncthreads_or(abort_flag)) break;
        const uint32_t slot = (steps_done + step) % kLtStages;
        if (tid == 0) {
          tc_fence_after();
          const uint32_t x = smem0 + slot * stage_bytes, w = x + kLtXBytes;
          for (int k = 0; k < 4; ++k)
            umma_bf16_ss(sums_tmem, sw128_desc(x + k * 32, 16, 1024), sw128_desc(w + k * 32, 16, 1024), idesc, step + k > 0);
          umma_commit(&stage_bar[slot]);
        }
        // the stage before is free when its UMMAs are done
        if (step > 0) {
          const uint32_t at = steps_done + step - 1;
          mbar_wait(&stage_bar[at % kLtStages], at / kLtStages & 1, kErrLowRankWait, &abort_flag);
        }
        if (step + kLtStages - 1 < steps) load_stage(step + kLtStages - 1);
        cp_async_commit();
      }
      if (abort_flag == 0) {
        const uint32_t at = steps_done + steps - 1;
        mbar_wait(&stage_bar[at % kLtStages], at / kLtStages & 1, kErrLowRankWait, &abort_flag);
      }
      cp_async_wait<0>();
      if (__syncthreads_or(abort_flag)) {  // else every stage is read: its place is free
        ok = false;
        break;
      }
      steps_done += steps;
      tc_fence_after();
      load_up(0);
      // ---- terms
      const float scale = __ldg(a.scales + adapter);
      const int row = warp % 4 * 32 + lane;
      for (int col = warp / 4 * 32; col < rank16; col += 64) {
        uint32_t r[32];
        tmem_ld_32cols(sums_tmem + (static_cast<uint32_t>(warp % 4 * 32) << 16) + col, r);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (col + c * 8 >= rank16) break;
          float h[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) h[i] = col + c * 8 + i < a.rank ? __uint_as_float(r[c * 8 + i]) * scale : 0.f;
          const int chunk8 = (col + c * 8) / 8;
          uint8_t* const to = smem + chunk8 / 8 * (kLtRows * 128) + lt_place(row, chunk8 % 8);
          for (int k = 0; k < parts; ++k) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              w[i] = pack_bf16x2(h[2 * i], h[2 * i + 1]);
              // infinities and NaN are whole in the first term
              h[2 * i] = fabsf(h[2 * i]) <= 3.38e38f ? h[2 * i] - __uint_as_float(w[i] << 16) : 0.f;
              h[2 * i + 1] = fabsf(h[2 * i + 1]) <= 3.38e38f ? h[2 * i + 1] - __uint_as_float(w[i] & 0xffff0000u) : 0.f;
            }
            *reinterpret_cast<uint4*>(to + k * S::TERM) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      tc_fence_before();
    }

    // ---- columns: round j's UMMAs run while round j - 1 is brought to the result
    const uint32_t idesc = umma_idesc_bf16(kLtRows, kLtColumns, false, false);
    const int quarter = warp % 4 * 32, half = warp / 4 * 64;
    // base's values of this lane, 4 neighbouring columns of every 4th row, on their way before they are wanted
    float4 next[8];
    auto load_base = [&](int round, int sub) {
      const int column = (round0 + round) * kLtColumns + half + sub + lane % 8 * 4;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = s.rows[quarter + i * 4 + lane / 8];
        if (row < 0 || column >= a.outer) continue;
        const int64_t at = (first + row) * a.outer + column;
        if constexpr (WHOLE && F32) {
          next[i] = *reinterpret_cast<const float4*>(static_cast<const float*>(a.base) + at);
        } else if constexpr (WHOLE) {
          const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(a.base) + at);
          next[i].x = __uint_as_float(v.x), next[i].y = __uint_as_float(v.y);  // taken apart where it is used
        } else {
          next[i].x = lr_load_one<F32>(a, at);
          if (column + 1 < a.outer) next[i].y = lr_load_one<F32>(a, at + 1);
          if (column + 2 < a.outer) next[i].z = lr_load_one<F32>(a, at + 2);
          if (column + 3 < a.outer) next[i].w = lr_load_one<F32>(a, at + 3);
        }
      }
    };
    load_base(0, 0);
    for (int j = 0; j <= rounds; ++j) {
      if (!bare) {
        cp_async_wait<0>();
        fence_proxy_async_smem();
        tc_fence_before();
        if (__syncthreads_or(abort_flag)) {  // else the round's columns (and the terms) are there, and its TMEM buffer is read
          ok = false;
          break;
        }
        if (j < rounds && tid == 0) {
          tc_fence_after();
          const uint32_t d = tmem + (j & 1) * 128, w = up0 + (j & 1) * S::UP;
          uint32_t more = 0;
          for (int k = 0; k < parts; ++k) {
            for (int r = 0; r < rank16 / 16; ++r) {
              const uint32_t at = r / 4 * (kLtRows * 128) + r % 4 * 32;
              umma_bf16_ss(d, sw128_desc(smem0 + k * S::TERM + at, 16, 1024), sw128_desc(w + at, 16, 1024), idesc, more);
              more = 1;
            }
          }
          umma_commit(&round_bar[(rounds_done + j) & 1]);
        }
        if (j > 0) {
          const uint32_t at = rounds_done + j - 1;
          mbar_wait(&round_bar[at & 1], at >> 1 & 1, kErrLowRankWait, &abort_flag);  // if it runs out, all see it at the next barrier
          tc_fence_after();
        }
        if (j + 1 < rounds) load_up(j + 1);
      }
      if (j == 0) continue;
      const int column0 = (round0 + j - 1) * kLtColumns + half;
#pragma unroll 1
      for (int sub = 0; sub < 64; sub += 32) {
        const int column = column0 + sub + lane % 8 * 4;
        float4 base[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) base[i] = next[i];
        if (sub == 0)
          load_base(j - 1, 32);
        else if (j < rounds)
          load_base(j, 0);
        if (!bare) {
          uint32_t r[32];
          tmem_ld_32cols(tmem + ((j - 1) & 1) * 128 + (static_cast<uint32_t>(quarter) << 16) + half + sub, r);
          tmem_wait_ld();
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<uint4*>(turn + lane * kLtTurnRow + i * 4) = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
          __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = s.rows[quarter + i * 4 + lane / 8];
          if (row < 0 || column >= a.outer) continue;
          float4 y = base[i];
          if constexpr (WHOLE && !F32) {
            const uint32_t lo = __float_as_uint(y.x), hi = __float_as_uint(y.y);
            y = make_float4(__uint_as_float(lo << 16), __uint_as_float(lo & 0xffff0000u), __uint_as_float(hi << 16),
                            __uint_as_float(hi & 0xffff0000u));
          }
          if (!bare) {
            const float4 v = *reinterpret_cast<const float4*>(turn + (i * 4 + lane / 8) * kLtTurnRow + lane % 8 * 4);
            y.x += v.x, y.y += v.y, y.z += v.z, y.w += v.w;
          }
          if (bad) y = make_float4(nan, nan, nan, nan);
          if (a.gelu) {
            lr_gelu(y.x, y.y, a.out_f32);
            lr_gelu(y.z, y.w, a.out_f32);
          }
          const int64_t at = (first + row) * a.outer + column;
          if constexpr (WHOLE) {
            if (a.out_f32)
              *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = y;
            else
              *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) = make_uint2(pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
          } else {
            lr_store_one(a, at, y.x);
            if (column + 1 < a.outer) lr_store_one(a, at + 1, y.y);
            if (column + 2 < a.outer) lr_store_one(a, at + 2, y.z);
            if (column + 3 < a.outer) lr_store_one(a, at + 3, y.w);
          }
        }
      }
    }
    if (!bare) rounds_done += rounds;
  }

  cp_async_wait<0>();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 256);
}

}  // namespace b200tx
