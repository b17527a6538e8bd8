// linear_w4_kernels.cuh -- y = epilogue(x . W^T + b) for a few rows of x, with W
// held in 4 bits and a bf16 scale for each group of weights along K:
//   W[n, k] = scale[k / group, n] * (code[n, k] - 8),   code in 0..15
//
// What bounds it: with few rows the weights' bytes over HBM, N K / 2 (and 2 N K / group
// of scales); next to it the instructions, of which turning codes into numbers is 11
// for a word of 8; with 17 rows and more x, which every CTA copies for its own columns.
//
// Layout.  A word is 8 consecutive weights of a row, ordered so that one mask
// takes two neighbours (nibble i holds weight {0,2,4,6,1,3,5,7}[i]): the
// nibbles under bf16's 128.0 are 128 + code, and subtracting 136 is exact.  A run of
// 128 weights is 16 words, word (a, b) of the 4 x 4 stored at (b, a): lane t of
// a quad reads 16 bytes and has words of four consecutive 32-weight pieces,
// so that whatever the group is, a product of the tensor core stays within one.
//
// The weights are the A operand (m16: output columns), x the B operand (n8: rows
// of x), so 8 rows of x cost one MMA.  A CTA is 8 warps: 8 / KS tiles of 16 RT
// columns x KS slices of K.  A slice goes through K two runs at a time, weights
// and x by cp.async into a ring (8 lanes copy one 128-byte line of two runs, chunks
// permuted by the row so that the fragments are read without bank conflicts); its
// warps share x.  The sum of a group is multiplied by its scale and added in fp32; the
// slices are joined in shared memory in a fixed order.
//
// Measured: 1 x 1024 -> 4096 in 3.0 us, 32 x 4096 -> 14336 in 25 us, 8 x 8192 -> 28672 (122
// MB) in 38 us.  Masks and shifts run at half rate, and 224 CTAs on 148 SMs leave
// half of the SMs less to do; for up to 16 rows and many units the kernel at the end
// of this file keeps x in shared memory and shares evenly: 31 us, 3.9 TB/s.
#pragma once

#include "attention_mma_kernels.cuh"
#include "kv8_attention_kernels.cuh"

namespace b200tx {

constexpr int kW4Warps = 8;
constexpr int kW4Run = 128;   // weights of a row that lie together
constexpr int kW4Runs = 2;    // runs of a stage: a whole line

struct W4Args {
  const __nv_bfloat16* x;        // [M, K]
  const uint8_t* packed;         // [N, runs * 64]
  const __nv_bfloat16* scales;   // [runs * 128 / group, N]
  const float* bias;             // [N] or null
  void* out;                     // [M, N]
  int64_t x_stride;
  int rows, outer, inner, runs;
  int gelu, out_f32;
  int slices;                    // warps along K, a power of two up to 8
  int stages;                    // of the ring
};

// The lowest nibbles of both halves as bf16 numbers code - 8, the usual way to expand
// 4-bit codes.  The mask and the
// exponent are one three-input operation: these and the shifts run at half
// rate and are what the kernel issues most.
__device__ __forceinline__ uint32_t nibbles_bf16x2(uint32_t w) {
  uint32_t biased;
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xEA;" : "=r"(biased) : "r"(w), "r"(0x43004300u));  // (w & mask) | 128.0
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&biased),
                                   __bfloat162bfloat162(__ushort_as_bfloat16(0x4308)));  // 136
  return *reinterpret_cast<const uint32_t*>(&v);
}

// d = a b
__device__ __forceinline__ void mma_m16n8k16_bf16_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ void w4_write(const W4Args& a, int m, int n, float y) {
  if (a.gelu) y = 0.5f * y * (1.f + erff(y * 0.70710678118654752f));
  const int64_t at = static_cast<int64_t>(m) * a.outer + n;
  if (a.out_f32) {
    static_cast<float*>(a.out)[at] = y;
  } else {
    static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
  }
}

// Bytes of a ring stage: 8 warps' weights, then the slices' x.
template <int TN, int RT>
constexpr int w4_stage_bytes(int slices) {
  return kW4Warps * RT * 16 * (kW4Runs * kW4Run / 2) + slices * TN * 8 * kW4Runs * kW4Run * 2;
}

// TN: n8 tiles of x rows; RT: m16 tiles of columns of a warp.
template <int TN, int RT, int GROUP>
__global__ void __launch_bounds__(kW4Warps * 32, 2) linear_w4_kernel(W4Args a) {
  constexpr int GROUPS = kW4Run / GROUP;  // groups per run
  constexpr int WORDS = 4 / GROUPS;       // words per group and lane
  constexpr int STAGE = kW4Runs * kW4Run;               // weights of a row in a stage
  constexpr int ROW = STAGE / 2;                     // their bytes
  constexpr int W_BYTES = RT * 16 * ROW;             // of a warp's stage
  constexpr int X_ROW = STAGE * 2;                   // bytes of a row of x
  constexpr int X_BYTES = TN * 8 * X_ROW;            // of a slice's stage
  constexpr int CHUNKS = ROW / 16, ROWS_A_COPY = 32 / CHUNKS;
  constexpr int COPIES = RT * 16 / ROWS_A_COPY;
  extern __shared__ __align__(128) uint8_t w4_smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t4 = lane % 4;
  const int per = kW4Warps / a.slices;  // warps of a slice
  const int slice = warp / per, tile = warp % per;
  const int n0 = (blockIdx.x * per + tile) * (16 * RT);
  const int m0 = blockIdx.y * (TN * 8);
  const int stage_bytes = kW4Warps * W_BYTES + a.slices * X_BYTES;
  const int all_stages = (a.runs + kW4Runs - 1) / kW4Runs, each = (all_stages + a.slices - 1) / a.slices;
  const int begin = min(all_stages, slice * each), count = min(all_stages, begin + each) - begin;
  griddep_wait();
  griddep_launch_dependents();

  // ---- copies: 512 bytes of weights (4 or 8 rows) at a time, and this warp's rows of the slice's x
  const int64_t pitch = static_cast<int64_t>(a.runs) * (kW4Run / 2);
  const int first_row = min(n0, a.outer - 1);  // columns past the end read the last one and are not written
  const uint8_t* const w_src = a.packed + first_row * pitch + lane % CHUNKS * 16;
  unsigned w_off[COPIES];
#pragma unroll
  for (int i = 0; i < COPIES; ++i)
    w_off[i] = static_cast<unsigned>(min(n0 + i * ROWS_A_COPY + lane / CHUNKS, a.outer - 1) - first_row) * static_cast<unsigned>(pitch);
  const uint32_t ring = smem_u32(w4_smem);
  const uint32_t w_put = ring + warp * W_BYTES + kv8_k_place<128>(lane * 16);
  static_assert(X_ROW == 512, "a copy of 32 lanes is a row of x");
  const __nv_bfloat16* const x_src = a.x + (m0 + tile) * a.x_stride + lane * 8;
  const int64_t x_step = per * a.x_stride;
  const uint32_t x_put = ring + kW4Warps * W_BYTES + slice * X_BYTES + tile * X_ROW;
  auto issue = [&](int s) {
    if (s < count) {
      const int at = begin + s;
      const uint32_t stage = (s % a.stages) * stage_bytes;
      const bool take = at * kW4Runs + (lane % CHUNKS) / 4 < a.runs;
#pragma unroll
      for (int i = 0; i < COPIES; ++i)
        cp_async_or_zero(w_put + stage + i * 512, w_src + w_off[i] + static_cast<int64_t>(at) * ROW, take);
      // x rows tile, tile + per, ... of the CTA's; a row is a copy
      const __nv_bfloat16* from = x_src + at * STAGE;
      uint32_t to = x_put + stage;
      const int left = at * STAGE + lane * 8 < a.inner ? a.rows - m0 : 0;
      for (int row = tile; row < TN * 8; row += per, from += x_step, to += per * X_ROW)
        cp_async_or_zero(to + ((row & 1) << 6 ^ lane * 16), row < left ? from : a.x, row < left);
    }
    cp_async_commit();
  };
  for (int s = 0; s < a.stages - 1; ++s) issue(s);

  // ---- scales: lane = a column of the tile (RT 2), or of one of two groups (RT 1)
  constexpr int STAGE_GROUPS = kW4Runs * GROUPS;
  constexpr int SCALES = (STAGE_GROUPS * RT + 1) / 2;
  const int s_col = min(n0 + lane % (16 * RT), a.outer - 1);
  const int all_groups = a.runs * GROUPS;
  auto load_scales = [&](int s, uint16_t (&to)[SCALES]) {
#pragma unroll
    for (int i = 0; i < SCALES; ++i) {
      const int q = (begin + s) * STAGE_GROUPS + (RT == 2 ? i : 2 * i + lane / 16);
      to[i] = 0;
      if (s < count && q < all_groups)
        to[i] = __ldg(reinterpret_cast<const uint16_t*>(a.scales) + static_cast<int64_t>(q) * a.outer + s_col);
    }
  };
  uint16_t scales[SCALES], next_scales[SCALES];
  load_scales(0, scales);

  float sum[RT][TN][4] = {};
  const uint32_t w_get = warp * W_BYTES + kv8_k_place<128>(g * 128 + t4 * 16);
  const uint32_t x_get = kW4Warps * W_BYTES + slice * X_BYTES + g * X_ROW;
  const uint32_t x_low = (t4 * 16) ^ ((g & 1) << 6);
#pragma unroll 1
  for (int s = 0; s < count; ++s) {
    if (a.stages == 2) cp_async_wait<0>();
    else if (a.stages == 3) cp_async_wait<1>();
    else cp_async_wait<2>();
    asm volatile("bar.sync %0, %1;" ::"r"(1 + slice), "r"(per * 32) : "memory");
    issue(s + a.stages - 1);
    load_scales(s + 1, next_scales);
    const uint8_t* const stage = w4_smem + (s % a.stages) * stage_bytes;
#pragma unroll
    for (int r = 0; r < kW4Runs; ++r) {
      uint32_t w[RT][2][4];
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        lds_words<16>(stage + (w_get ^ (r * 64)) + i * 16 * ROW, w[i][0]);
        lds_words<16>(stage + (w_get ^ (r * 64)) + i * 16 * ROW + 8 * ROW, w[i][1]);
      }
#pragma unroll
      for (int q = 0; q < GROUPS; ++q) {
        float acc[RT][TN][4];
#pragma unroll
        for (int c = q * WORDS; c < (q + 1) * WORDS; ++c) {
          uint32_t xf[TN][4];
#pragma unroll
          for (int j = 0; j < TN; ++j)
            lds_words<16>(stage + x_get + (x_low ^ ((c & 1) << 6)) + (c >> 1) * 128 + r * 256 + j * 8 * X_ROW, xf[j]);
#pragma unroll
          for (int i = 0; i < RT; ++i) {
            const uint32_t wa = w[i][0][c], wb = w[i][1][c];
            const uint32_t a0[4] = {nibbles_bf16x2(wa), nibbles_bf16x2(wb), nibbles_bf16x2(wa >> 4), nibbles_bf16x2(wb >> 4)};
            const uint32_t a1[4] = {nibbles_bf16x2(wa >> 8), nibbles_bf16x2(wb >> 8), nibbles_bf16x2(wa >> 12),
                                    nibbles_bf16x2(wb >> 12)};
#pragma unroll
            for (int j = 0; j < TN; ++j) {
              if (c == q * WORDS) {
                mma_m16n8k16_bf16_first(acc[i][j], a0, xf[j][0], xf[j][1]);
              } else {
                mma_m16n8k16_bf16(acc[i][j], a0, xf[j][0], xf[j][1]);
              }
              mma_m16n8k16_bf16(acc[i][j], a1, xf[j][2], xf[j][3]);
            }
          }
        }
        const int group = r * GROUPS + q;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          const uint32_t held = scales[RT == 2 ? group : group / 2];
          const int from = RT == 2 ? i * 16 : group % 2 * 16;
          const float s0 = __uint_as_float(__shfl_sync(0xffffffffu, held, from + g) << 16);
          const float s1 = __uint_as_float(__shfl_sync(0xffffffffu, held, from + g + 8) << 16);
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            sum[i][j][0] = fmaf(s0, acc[i][j][0], sum[i][j][0]);
            sum[i][j][1] = fmaf(s0, acc[i][j][1], sum[i][j][1]);
            sum[i][j][2] = fmaf(s1, acc[i][j][2], sum[i][j][2]);
            sum[i][j][3] = fmaf(s1, acc[i][j][3], sum[i][j][3]);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < SCALES; ++i) scales[i] = next_scales[i];
  }

  if (a.slices > 1) {
    cp_async_wait<0>();
    __syncthreads();
    float4* const join = reinterpret_cast<float4*>(w4_smem);  // [warp][RT * TN][32]
#pragma unroll
    for (int i = 0; i < RT; ++i) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
        join[(warp * RT * TN + i * TN + j) * 32 + lane] = make_float4(sum[i][j][0], sum[i][j][1], sum[i][j][2], sum[i][j][3]);
    }
    __syncthreads();
    if (slice != 0) return;
    for (int w = 1; w < a.slices; ++w) {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const float4 v = join[((w * per + tile) * RT * TN + i * TN + j) * 32 + lane];
          sum[i][j][0] += v.x; sum[i][j][1] += v.y; sum[i][j][2] += v.z; sum[i][j][3] += v.w;
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < RT; ++i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = n0 + i * 16 + g + 8 * h;
      if (n >= a.outer) continue;
      const float bias = a.bias == nullptr ? 0.f : a.bias[n];
#pragma unroll
      for (int j = 0; j < TN; ++j) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int m = m0 + j * 8 + 2 * t4 + e;
          if (m < a.rows) w4_write(a, m, n, sum[i][j][2 * h + e] + bias);
        }
      }
    }
  }
}

// ---- the same product with all of x in shared memory ------------------------
// One CTA of 16 warps for each SM.  It holds x, so that the main loop copies
// weights only and needs no barrier: each warp has a ring of its own.  A CTA has an
// equal share of the 16-column tiles; its (tile, stage) units form one line that the
// warps cut into equal ranges.  Tiles that lie in several ranges are joined in shared
// memory, in the order of the ranges.  8 x 8192 -> 28672 takes 30.9 us (3.9 TB/s; 38.2
// above), bound by its instructions, 363 for 16 columns x 256 weights: schedulers issue in
// two of three cycles.

constexpr int kW4LineWarps = 16;
constexpr int kW4LineStage = 16 * (kW4Runs * kW4Run / 2);  // bytes of a warp's stage

template <int TN, int GROUP>
__global__ void __launch_bounds__(kW4LineWarps * 32, 1) linear_w4_line_kernel(W4Args a) {
  constexpr int GROUPS = kW4Run / GROUP, WORDS = 4 / GROUPS;
  constexpr int STAGE = kW4Runs * kW4Run, ROW = STAGE / 2;
  constexpr int COPIES = 4;  // of 4 rows' lines
  constexpr int STAGE_GROUPS = kW4Runs * GROUPS, SCALES = STAGE_GROUPS / 2;
  extern __shared__ __align__(128) uint8_t w4_smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t4 = lane % 4;
  const int all_stages = (a.runs + kW4Runs - 1) / kW4Runs;
  const int tiles = (a.outer + 15) / 16;
  auto cut = [](int64_t of, int i, int parts) { return static_cast<int>(of * i / parts); };
  const int first_tile = cut(tiles, blockIdx.x, gridDim.x);
  const int units = (cut(tiles, blockIdx.x + 1, gridDim.x) - first_tile) * all_stages;
  const int begin = cut(units, warp, kW4LineWarps), end = cut(units, warp + 1, kW4LineWarps);
  griddep_wait();
  griddep_launch_dependents();

  // ---- x: rows of whole stages, odd rows' halves of a line exchanged
  const int x_pitch = all_stages * STAGE * 2;
  const uint32_t x_at = smem_u32(w4_smem);
  for (int row = 0; row < a.rows; ++row) {
    const __nv_bfloat16* const from = a.x + row * a.x_stride;
    for (int chunk = threadIdx.x; chunk < all_stages * (STAGE / 8); chunk += kW4LineWarps * 32) {
      const bool take = chunk * 8 < a.inner;
      cp_async_or_zero(x_at + row * x_pitch + (chunk * 16 ^ (row & 1) << 6), take ? from + chunk * 8 : a.x, take);
    }
  }
  cp_async_commit();

  // ---- a warp's copies: 4 rows' lines at a time
  const int64_t pitch = static_cast<int64_t>(a.runs) * (kW4Run / 2);
  const int ring_at = a.rows * x_pitch + warp * a.stages * kW4LineStage;
  const uint32_t w_put = x_at + ring_at + kv8_k_place<128>(lane * 16);
  struct Cursor { int unit, tile, at; };
  auto advance = [&](Cursor& c) {
    ++c.unit;
    if (++c.at == all_stages) { c.at = 0; ++c.tile; }
  };
  Cursor copy{begin, first_tile + begin / all_stages, begin % all_stages};
  uint32_t put = w_put;
  const uint32_t put_end = w_put + a.stages * kW4LineStage;
  const uint8_t* from = nullptr;
  unsigned row_off[COPIES];
  auto enter_tile = [&]() {  // columns past the end read the last one and are not written
    const int row = min(copy.tile * 16 + lane / 8, a.outer - 1);
    from = a.packed + row * pitch + copy.at * ROW + lane % 8 * 16;
#pragma unroll
    for (int i = 0; i < COPIES; ++i)
      row_off[i] = static_cast<unsigned>(min(row + i * 4, a.outer - 1) - row) * static_cast<unsigned>(pitch);
  };
  enter_tile();
  auto issue = [&]() {
    if (copy.unit < end) {
      const bool take = copy.at * kW4Runs + lane % 8 / 4 < a.runs;
#pragma unroll
      for (int i = 0; i < COPIES; ++i) cp_async_or_zero(put + i * 512, from + row_off[i], take);
      advance(copy);
      from += ROW;
      if (copy.at == 0) enter_tile();
      put += kW4LineStage;
      if (put == put_end) put = w_put;
    }
    cp_async_commit();
  };
  for (int s = 0; s < a.stages - 1; ++s) issue();

  // ---- scales, two units ahead: lane = a column of one of two groups
  const int all_groups = a.runs * GROUPS;
  Cursor now{begin, first_tile + begin / all_stages, begin % all_stages}, ahead = now;
  auto load_scales = [&](uint16_t (&to)[SCALES]) {
    const int col = min(ahead.tile * 16 + lane % 16, a.outer - 1);
#pragma unroll
    for (int i = 0; i < SCALES; ++i) {
      const int q = ahead.at * STAGE_GROUPS + 2 * i + lane / 16;
      to[i] = 0;
      if (ahead.unit < end && q < all_groups)
        to[i] = __ldg(reinterpret_cast<const uint16_t*>(a.scales) + static_cast<int64_t>(q) * a.outer + col);
    }
    advance(ahead);
  };
  uint16_t scales[3][SCALES];
  load_scales(scales[0]);
  load_scales(scales[1]);

  if (a.stages == 3) cp_async_wait<2>();
  else cp_async_wait<3>();
  __syncthreads();  // x is there

  auto write = [&](int tile, const float (&sum)[TN][4]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = tile * 16 + g + 8 * h;
      if (n >= a.outer) continue;
      const float bias = a.bias == nullptr ? 0.f : a.bias[n];
#pragma unroll
      for (int j = 0; j < TN; ++j) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int m = j * 8 + 2 * t4 + e;
          if (m < a.rows) w4_write(a, m, n, sum[j][2 * h + e] + bias);
        }
      }
    }
  };

  float sum[TN][4] = {}, head[TN][4] = {};  // head: the range's first piece, if another range has part of its tile
  int piece = begin;                        // first unit of the piece
  const int w_get = ring_at + kv8_k_place<128>(g * 128 + t4 * 16);
  int x_get[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int row = min(j * 8 + g, a.rows - 1);  // rows past the end are not written
    x_get[j] = row * x_pitch + (t4 * 16 ^ (row & 1) << 6);
  }
  int get = 0;
#pragma unroll 1
  while (now.unit < end) {
    if (a.stages == 3) cp_async_wait<1>();
    else cp_async_wait<2>();
    __syncwarp();
    issue();
    load_scales(scales[2]);
    const uint8_t* const stage = w4_smem + get * kW4LineStage;
    const uint8_t* const x_stage = w4_smem + now.at * (STAGE * 2);
#pragma unroll
    for (int r = 0; r < kW4Runs; ++r) {
      uint32_t w[2][4];
      lds_words<16>(stage + (w_get ^ (r * 64)), w[0]);
      lds_words<16>(stage + (w_get ^ (r * 64)) + 8 * ROW, w[1]);
#pragma unroll
      for (int q = 0; q < GROUPS; ++q) {
        float acc[TN][4];
#pragma unroll
        for (int c = q * WORDS; c < (q + 1) * WORDS; ++c) {
          const uint32_t wa = w[0][c], wb = w[1][c];
          const uint32_t a0[4] = {nibbles_bf16x2(wa), nibbles_bf16x2(wb), nibbles_bf16x2(wa >> 4), nibbles_bf16x2(wb >> 4)};
          const uint32_t a1[4] = {nibbles_bf16x2(wa >> 8), nibbles_bf16x2(wb >> 8), nibbles_bf16x2(wa >> 12),
                                  nibbles_bf16x2(wb >> 12)};
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            uint32_t xf[4];
            lds_words<16>(x_stage + (x_get[j] ^ ((c & 1) << 6)) + (c >> 1) * 128 + r * 256, xf);
            if (c == q * WORDS) {
              mma_m16n8k16_bf16_first(acc[j], a0, xf[0], xf[1]);
            } else {
              mma_m16n8k16_bf16(acc[j], a0, xf[0], xf[1]);
            }
            mma_m16n8k16_bf16(acc[j], a1, xf[2], xf[3]);
          }
        }
        const int group = r * GROUPS + q;
        const uint32_t held = scales[0][group / 2];
        const float s0 = __uint_as_float(__shfl_sync(0xffffffffu, held, group % 2 * 16 + g) << 16);
        const float s1 = __uint_as_float(__shfl_sync(0xffffffffu, held, group % 2 * 16 + g + 8) << 16);
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          sum[j][0] = fmaf(s0, acc[j][0], sum[j][0]);
          sum[j][1] = fmaf(s0, acc[j][1], sum[j][1]);
          sum[j][2] = fmaf(s1, acc[j][2], sum[j][2]);
          sum[j][3] = fmaf(s1, acc[j][3], sum[j][3]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < SCALES; ++i) {
      scales[0][i] = scales[1][i];
      scales[1][i] = scales[2][i];
    }
    get = get + 1 == a.stages ? 0 : get + 1;
    if (now.at == all_stages - 1) {  // the tile ends here
      const bool whole = now.unit - piece == all_stages - 1;
      if (whole) write(now.tile, sum);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!whole) head[j][e] = sum[j][e];
          sum[j][e] = 0.f;
        }
      }
      piece = now.unit + 1;
    }
    advance(now);
  }

  // ---- join: a range's first piece if it begins in a tile, and its last if it ends in one
  cp_async_wait<0>();
  __syncwarp();
  const bool ends_inside = piece < end;  // the last piece's tile goes on in the next range
  const bool only = piece == begin;      // and it is the first piece, too
  float4* const mine = reinterpret_cast<float4*>(w4_smem + ring_at);
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const float(&h)[4] = ends_inside && only ? sum[j] : head[j];
    mine[j * 32 + lane] = make_float4(h[0], h[1], h[2], h[3]);
  }
  __syncthreads();
  // the range that has a tile's first unit, but not its last, joins it
  if (!ends_inside || piece % all_stages != 0) return;
  const int tile_end = piece + all_stages;
  for (int w = warp + 1; w < kW4LineWarps; ++w) {
    const int from = cut(units, w, kW4LineWarps);
    if (from >= tile_end) break;
    if (from == cut(units, w + 1, kW4LineWarps)) continue;
    const float4* const other = reinterpret_cast<const float4*>(w4_smem + a.rows * x_pitch + w * a.stages * kW4LineStage);
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const float4 v = other[j * 32 + lane];
      sum[j][0] += v.x; sum[j][1] += v.y; sum[j][2] += v.z; sum[j][3] += v.w;
    }
  }
  write(first_tile + piece / all_stages, sum);
}

}  // namespace b200tx
