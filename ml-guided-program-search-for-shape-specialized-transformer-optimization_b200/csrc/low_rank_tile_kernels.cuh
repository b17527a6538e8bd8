// low_rank_tile_kernels.cuh -- low-rank adapters beside a shared projection, for
// many rows with few adapters (prompts): what low_rank_kernels.cuh computes,
// 128 rows of an adapter at a time on tcgen05.
//
// A CTA takes a group of up to 128 rows (found as there) and a part of the columns:
//   1. sums = x . down^T over K, 128 x R, accumulated in TMEM from stages of 64 values of K.  Rows that
//      follow one another (a prompt's) come by TMA, others by cp.async from where they are,
//      into the same 128-byte swizzled layout;
//   2. the sums, scaled, become bf16 terms in shared memory (each the rounded rest of the ones before);
//   3. for each 128 columns: terms . up^T into one of two TMEM buffers, while the warps bring
//      the buffer before to the result.  up comes by TMA, two neighbouring columns of
//      each eight at a time, so that a lane that reads two neighbouring ones of each eight of the buffer (tcgen05.ld of
//      16 lanes x 256 bits) has 8 neighbouring columns of the result, of two rows: it reads base and writes the
//      result 16 bytes at a time, four lanes 64 that lie together, and nothing is turned in shared memory.
//
// The bytes are base's and the result's, 9 of 10 of a feed-forward layer's: the weights of
// an adapter are read (from L2) once for 128 rows.  The warp MMA form of this reads them for every 32 rows
// and keeps the tensor pipe busy for as long as the bytes take.
//
// What bounds it: 8 x 2048 rows of 1024 -> 4096, rank 64, GELU: 79.8 us, 3.85 TB/s of the measured 6.55 (46.7 us; the warp MMAs
// take 238).  Of these 3 are launch and ranks, 8.7 the sums (0.33 us a stage: the issuing thread), 1 the terms, and 32 rounds
// of 2.0 us: 22 instructions a value, 13 of them GELU, issued in 65 % of cycles on 128 of 148 SMs (a group to an SM; cutting a
// group's columns would take its sums twice).  With base in 32 bits, 436 MB: 124 us, 3.5 TB/s.
//
// One thread brings the stages and up's columns, one of another warp issues the UMMAs (in one thread the two take 0.57 us
// for a stage); 16 warps make the terms and bring the results out, each for itself: they all meet at the
// buffers' barriers only.  Waits are bounded as everywhere.
#pragma once

#include "kv8_attention_kernels.cuh"
#include "low_rank_kernels.cuh"

namespace b200tx {

constexpr int kLtRows = 128;
constexpr int kLtColumns = 128;          // of the result, for one round
constexpr int kLtStages = 6;             // of 64 values of K
constexpr uint32_t kLtXBytes = kLtRows * 128;
constexpr int kLtWorkers = 512;          // threads that make the terms and bring the results out
constexpr int kLtThreads = kLtWorkers + 64;

// RA atoms of 64 ranks.
template <int RA>
struct LtShape {
  static constexpr uint32_t UP = RA * kLtColumns * 128;  // a round's columns of up
  static constexpr int UPS = RA == 1 ? 4 : 3;            // rounds whose columns are there or on their way
  static constexpr uint32_t TERM = RA * kLtRows * 128;
  __host__ __device__ static constexpr uint32_t stage(int rank16) { return kLtXBytes + rank16 * 128; }
  // the stages of the sums, and later the terms and the rounds' columns, in the same place
  __host__ __device__ static constexpr uint32_t bytes(int rank16, int terms) {
    return (kLtStages * stage(rank16) > terms * TERM + UPS * UP ? kLtStages * stage(rank16) : terms * TERM + UPS * UP) + 1024;
  }
};

// Column 32 g + 8 t + 2 i + b of a round stands in its buffer at 32 i + 8 g + 2 t + b.  Of 16 rows, a lane reads columns
// 2 t and 2 t + 1 (t = lane % 4) of the eight at 32 i + 8 g for each i: r[4 i + b] of row lane / 4, r[4 i + 2 + b] of row lane / 4 + 8.
__device__ __forceinline__ void tmem_ld_16x32(uint32_t taddr, uint32_t (&r)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[4 * i]), "=r"(r[4 * i + 1]), "=r"(r[4 * i + 2]), "=r"(r[4 * i + 3])
                 : "r"(taddr + 32 * i));
}

// Where 16 bytes of a 128-byte row stand under the 128-byte swizzle.
__device__ __forceinline__ uint32_t lt_place(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

template <int RA, bool F32>
__global__ void __launch_bounds__(kLtThreads, 1)
    low_rank_tile_kernel(const __grid_constant__ LowRankArgs a, const __grid_constant__ CUtensorMap x_map,
                         const __grid_constant__ CUtensorMap down_map, const __grid_constant__ CUtensorMap up_map) {
  using S = LtShape<RA>;
  extern __shared__ uint8_t lt_smem[];
  __shared__ LrGroups<kLtRows> s;
  __shared__ uint64_t copied_bar[kLtStages], free_bar[kLtStages], stage_bar[kLtStages];
  __shared__ uint64_t up_bar[S::UPS], up_free_bar[S::UPS], full_bar[2], empty_bar[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;

  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  uint8_t* const smem = align_1024(lt_smem);
  const uint32_t smem0 = smem_u32(smem);
  const int rank16 = (a.rank + 15) / 16 * 16, parts = a.out_f32 ? 3 : 2;
  if (tid == 0) {
    for (int i = 0; i < kLtStages; ++i) {
      mbar_init(&copied_bar[i], 1);
      mbar_init(&free_bar[i], 1);
      mbar_init(&stage_bar[i], 1);
    }
    for (int i = 0; i < S::UPS; ++i) {
      mbar_init(&up_bar[i], 1);
      mbar_init(&up_free_bar[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&full_bar[i], 1);
      mbar_init(&empty_bar[i], kLtWorkers / 32);
    }
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
  auto column_of = [&](int j) { return static_cast<uint32_t>(round0 + j) * kLtColumns; };
  const float nan = __int_as_float(0x7fffffff);
  const uint32_t sums_tmem = tmem + 128;  // the second round's columns: free until then
  const uint64_t smem_desc = sw128_desc(smem0, 16, 1024);  // an operand's place is its 16-byte units more
  const bool copies = tid == kLtWorkers, issues = tid == kLtWorkers + 32;
  uint32_t steps_done = 0, copied_done = 0, rounds_done = 0;
  uint32_t asked = 0, asked_up = 0;  // copies that the copying thread has asked for, of stages and of up's columns

  for (int group = split == 1 ? mine : part < split ? mine % groups : groups; group < groups;
       group += split == 1 ? a.clusters : groups) {
    const int adapter = s.key[s.lead[group]];
    if (adapter < 0 && a.skip_bare) continue;
    tc_fence_before();
    fence_proxy_async_smem();
    if (__syncthreads_or(abort_flag)) break;
    const int many = s.take(group, n, a.group);
    const bool bad = adapter >= a.count, bare = adapter < 0 || bad;
    const __nv_bfloat16* const up = a.up + static_cast<int64_t>(bare ? 0 : adapter) * a.outer * a.rank;

    if (!bare) {
      // ---- sums over K
      const int steps = (a.inner + 63) / 64;
      const uint32_t stage_bytes = S::stage(rank16);
      const uint32_t idesc = umma_idesc_bf16(kLtRows, rank16, false, false);
      auto add_step = [&](uint32_t slot, bool more, uint64_t* bar) {
        tc_fence_after();
        const uint64_t x = smem_desc + (slot * stage_bytes >> 4), w = x + (kLtXBytes >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_bf16_ss(sums_tmem, x + 2 * k, w + 2 * k, idesc, more || k > 0);
        umma_commit(bar);
      };
      if (s.rows[many - 1] - s.rows[0] == many - 1) {
        // rows in a row; those behind the group's come along, and what becomes of them is not written
        if (copies) {
          const int row = static_cast<int>(first) + s.rows[0];
          uint32_t slot = copied_done % kLtStages, phase = copied_done / kLtStages & 1;
          for (int step = 0; step < steps; ++step) {
            if (!mbar_wait(&free_bar[slot], phase ^ 1, kErrLowRankWait, &abort_flag)) break;
            mbar_arrive_expect_tx(&copied_bar[slot], stage_bytes);
            tma_load_2d(smem + slot * stage_bytes, &x_map, &copied_bar[slot], step * 64, row);
            tma_load_2d(smem + slot * stage_bytes + kLtXBytes, &down_map, &copied_bar[slot], step * 64, adapter * a.rank);
            if (++slot == kLtStages) slot = 0, phase ^= 1;
            ++asked;
          }
        } else if (issues) {
          uint32_t slot = copied_done % kLtStages, phase = copied_done / kLtStages & 1;
          for (int step = 0; step < steps; ++step) {
            if (!mbar_wait(&copied_bar[slot], phase, kErrLowRankWait, &abort_flag)) break;
            add_step(slot, step > 0, &free_bar[slot]);
            if (++slot == kLtStages) slot = 0, phase ^= 1;
          }
          // the others wait at the barrier below, which costs no instructions that this thread would wait behind
          const uint32_t at = copied_done + steps - 1;
          mbar_wait(&free_bar[at % kLtStages], at / kLtStages & 1, kErrLowRankWait, &abort_flag);
        }
        copied_done += steps;
      } else {
        const __nv_bfloat16* const down = a.down + static_cast<int64_t>(adapter) * a.rank * a.inner;
        // a thread's pieces: 16 bytes at the same place of every 64th row
        constexpr int APART = kLtWorkers / 8;
        const int chunk = tid % 8, row0 = tid / 8;
        const bool loads = tid < kLtWorkers;
        const __nv_bfloat16* xp[kLtRows / APART];
#pragma unroll
        for (int i = 0; i < kLtRows / APART; ++i)
          xp[i] = a.x + (first + (loads ? max(s.rows[row0 + APART * i], 0) : 0)) * a.inner + chunk * 8;
        auto load_stage = [&](int step) {
          const uint32_t to = smem0 + (steps_done + step) % kLtStages * stage_bytes;
          const bool in = step * 64 + chunk * 8 < a.inner;
#pragma unroll
          for (int i = 0; i < kLtRows / APART; ++i) {
            const bool take = in && row0 + APART * i < many;
            cp_async_or_zero(to + lt_place(row0 + APART * i, chunk), take ? xp[i] + step * 64 : a.x, take);
          }
          for (int row = row0; row < rank16; row += APART) {
            const bool take = in && row < a.rank;
            cp_async_or_zero(to + kLtXBytes + lt_place(row, chunk),
                             down + (take ? static_cast<int64_t>(row) * a.inner + step * 64 + chunk * 8 : 0), take);
          }
        };
        for (int i = 0; i < kLtStages - 1; ++i) {
          if (i < steps && loads) load_stage(i);
          cp_async_commit();
        }
        for (int step = 0; step < steps; ++step) {
          cp_async_wait<kLtStages - 2>();
          fence_proxy_async_smem();
          if (__syncthreads_or(abort_flag)) break;
          const uint32_t at = steps_done + step;
          if (issues) add_step(at % kLtStages, step > 0, &stage_bar[at % kLtStages]);
          // the stage before is free when its UMMAs are done
          if (step > 0) mbar_wait(&stage_bar[(at - 1) % kLtStages], (at - 1) / kLtStages & 1, kErrLowRankWait, &abort_flag);
          if (step + kLtStages - 1 < steps && loads) load_stage(step + kLtStages - 1);
          cp_async_commit();
        }
        const uint32_t at = steps_done + steps - 1;
        if (abort_flag == 0) mbar_wait(&stage_bar[at % kLtStages], at / kLtStages & 1, kErrLowRankWait, &abort_flag);
        cp_async_wait<0>();
        steps_done += steps;
      }
      if (__syncthreads_or(abort_flag)) break;  // else every stage is read: its place is free
      tc_fence_after();
      // ---- terms
      const float scale = __ldg(a.scales + adapter);
      const int row = warp % 4 * 32 + lane;
      if (const int col = warp / 4 * 32; warp < kLtWorkers / 32 && col < rank16) {
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
      fence_proxy_async_smem();
      __syncthreads();  // the terms are there, and the sums' place is free
    }

    // ---- columns
    if (tid >= kLtWorkers) {
      if (copies && !bare) {
        // 8 columns of up are one of the map's outermost dimension; those past the adapter's last come along
        const int eight0 = static_cast<int>(static_cast<int64_t>(adapter) * a.outer / 8);
        uint32_t slot = rounds_done % S::UPS, phase = rounds_done / S::UPS & 1;
        for (int j = 0; j < rounds; ++j) {
          if (!mbar_wait(&up_free_bar[slot], phase ^ 1, kErrLowRankWait, &abort_flag)) break;
          uint8_t* const to = smem + parts * S::TERM + slot * S::UP;
          mbar_arrive_expect_tx(&up_bar[slot], S::UP);
#pragma unroll
          for (int r = 0; r < 4 * RA; ++r)
            tma_load_3d(to + r * 32 * 128, &up_map, &up_bar[slot], r / 4 * 64, r % 4 * 2, eight0 + static_cast<int>(column_of(j) / 8));
          if (++slot == S::UPS) slot = 0, phase ^= 1;
          ++asked_up;
        }
      } else if (issues && !bare) {
        const uint32_t idesc = umma_idesc_bf16(kLtRows, kLtColumns, false, false);
        uint32_t slot = rounds_done % S::UPS, phase = rounds_done / S::UPS & 1;
        for (int j = 0; j < rounds; ++j) {
          const uint32_t at = rounds_done + j, buffer = at & 1;
          if (!mbar_wait(&up_bar[slot], phase, kErrLowRankWait, &abort_flag)) break;
          if (!mbar_wait(&empty_bar[buffer], (at >> 1 & 1) ^ 1, kErrLowRankWait, &abort_flag)) break;
          tc_fence_after();
          const uint64_t w = smem_desc + (parts * S::TERM + slot * S::UP >> 4);
          for (int k = 0; k < parts; ++k) {
#pragma unroll
            for (int r = 0; r < 4 * RA; ++r) {
              const uint32_t in = (r / 4 * (kLtRows * 128) + r % 4 * 32) >> 4;
              if (r * 16 < rank16)
                umma_bf16_ss(tmem + buffer * 128, smem_desc + (k * S::TERM >> 4) + in, w + in, idesc, k + r > 0);
            }
          }
          umma_commit(&up_free_bar[slot]);
          umma_commit(&full_bar[buffer]);
          if (++slot == S::UPS) slot = 0, phase ^= 1;
        }
      }
      if (!bare) rounds_done += rounds;
      continue;
    }
    const int quarter = warp % 4 * 32, columns = warp / 4 * 32;  // this warp's rows and columns of a round
    // This lane's values: 8 neighbouring columns of four rows.  Places in the window have 32 bits (256 rows of 2^24 columns).
    uint32_t place[4];
    uint32_t live = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = s.rows[quarter + i * 8 + lane / 4];
      live |= static_cast<uint32_t>(row >= 0) << i;
      place[i] = static_cast<uint32_t>(max(row, 0)) * a.outer + columns + lane % 4 * 8;
    }
    const uint8_t* const base0 = static_cast<const uint8_t*>(a.base) + first * a.outer * (F32 ? 4 : 2);
    uint8_t* const out0 = static_cast<uint8_t*>(a.out) + first * a.outer * (a.out_f32 ? 4 : 2);
    // A warp with all its rows takes whole rounds without a check between the values; base's are on their way then a
    // round before they are wanted: rows 2 i and 2 i + 1 of the four.
    const bool plain = __all_sync(0xffffffffu, live == 0xf) && !bad;
    auto whole = [&](int j) { return plain && column_of(j) + kLtColumns <= static_cast<uint32_t>(a.outer); };
    LrEight<F32> ahead[2][2];
    auto load_base = [&](int j, int i) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        ahead[i][e].load(base0 + static_cast<uint64_t>(place[2 * i + e] + column_of(j)) * (F32 ? 4 : 2));
    };
    auto store = [&](uint8_t* to, float (&y)[8]) {
      if (a.out_f32) {
        if (a.gelu) {
#pragma unroll
          for (int k = 0; k < 8; ++k) y[k] = lr_gelu_32(y[k]);
        }
        reinterpret_cast<float4*>(to)[0] = make_float4(y[0], y[1], y[2], y[3]);
        reinterpret_cast<float4*>(to)[1] = make_float4(y[4], y[5], y[6], y[7]);
      } else {
        if (a.gelu) {
#pragma unroll
          for (int k = 0; k < 8; ++k) y[k] = lr_gelu_16(y[k]);
        }
        *reinterpret_cast<uint4*>(to) =
            make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]));
      }
    };
    if (whole(0)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) load_base(0, i);
    }
    for (int j = 0; j < rounds; ++j) {
      const uint32_t at = rounds_done + j;
      // the warp goes on, or stops, together
      if (!__all_sync(0xffffffffu, bare || mbar_wait(&full_bar[at & 1], at >> 1 & 1, kErrLowRankWait, &abort_flag))) break;
      tc_fence_after();
      const uint32_t column = column_of(j);
      const int size = a.out_f32 ? 4 : 2;
      const uint32_t d = tmem + (at & 1) * 128 + (static_cast<uint32_t>(quarter) << 16) + columns / 4;
      auto done = [&]() {  // the buffer is read
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty_bar[at & 1]);
      };
      if (whole(j)) {
        const bool more = j + 1 < rounds && whole(j + 1);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t r[16] = {};
          if (!bare) tmem_ld_16x32(d + (static_cast<uint32_t>(i * 16) << 16), r);
          float y[2][8];
#pragma unroll
          for (int e = 0; e < 2; ++e) ahead[i][e].values(y[e]);
          if (more) load_base(j + 1, i);
          if (!bare) {
            tmem_wait_ld();
            if (i == 1) done();
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int m = 0; m < 8; ++m) y[e][m] += __uint_as_float(r[m / 2 * 4 + 2 * e + m % 2]);
            store(out0 + static_cast<uint64_t>(place[2 * i + e] + column) * size, y[e]);
          }
        }
        continue;
      }
      // rows or columns are missing, or all is NaN
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        uint32_t r[16] = {};
        if (!bare) {
          tmem_ld_16x32(d + (static_cast<uint32_t>(i * 16) << 16), r);
          tmem_wait_ld();
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t here = column + columns + lane % 4 * 8;
          const int row = s.rows[quarter + i * 16 + e * 8 + lane / 4];
          if (row < 0 || here >= static_cast<uint32_t>(a.outer)) continue;
          const uint64_t from = static_cast<uint64_t>(static_cast<uint32_t>(row) * a.outer + here);
          LrEight<F32> base;
          base.load(base0 + from * (F32 ? 4 : 2));
          float y[8];
          base.values(y);
#pragma unroll
          for (int m = 0; m < 8; ++m) y[m] = bad ? nan : y[m] + __uint_as_float(r[m / 2 * 4 + 2 * e + m % 2]);
          store(out0 + from * size, y);
        }
      }
      if (!bare) done();
    }
    if (!bare) rounds_done += rounds;
  }

  cp_async_wait<0>();
  if (copies) {  // no copy is left on its way, also where a wait has run out
    for (uint32_t i = asked > kLtStages ? asked - kLtStages : 0; i < asked; ++i)
      mbar_drain_wait(&copied_bar[i % kLtStages], i / kLtStages & 1);
    for (uint32_t i = asked_up > S::UPS ? asked_up - S::UPS : 0; i < asked_up; ++i)
      mbar_drain_wait(&up_bar[i % S::UPS], i / S::UPS & 1);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 256);
}

}  // namespace b200tx
