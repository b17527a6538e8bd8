// linear_w4_kernels.cuh -- y = epilogue(x . W^T + b) for a few rows of x, with W
// held in 4 bits and a bf16 scale for each group of weights along K:
//   W[n, k] = scale[k / group, n] * (code[n, k] - 8),   code in 0..15
//
// What bounds it: with up to 32 rows the weights' bytes over HBM, N K / 2 (and
// 2 N K / group of scales).
//
// Layout.  A word is 8 consecutive weights of a row, ordered so that one mask
// takes two neighbours (nibble i holds weight {0,2,4,6,1,3,5,7}[i]): the
// nibbles under bf16's 128.0 are 128 + code, and subtracting 136 is exact.  A run of
// 128 weights is 16 words, word (a, b) of the 4 x 4 stored at (b, a): lane t of
// a quad loads 16 bytes and has words of four consecutive 32-weight pieces,
// so that whatever the group is, a product of the tensor core stays within one.
//
// The weights are the A operand (m16: output columns), x the B operand (n8: rows
// of x), so 8 rows of x cost one MMA.  Weights go from HBM to registers to the
// tensor core without shared memory; x comes from L1.  The sum of a group is
// multiplied by its scale and added in fp32.  A CTA is 8 warps: column tiles x
// splits of K (runs dealt in turn), joined in shared memory in a fixed order.
#pragma once

#include "attention_mma_kernels.cuh"

namespace b200tx {

constexpr int kW4Warps = 8;
constexpr int kW4Run = 128;  // weights of a row that lie together

struct W4Args {
  const __nv_bfloat16* x;        // [M, K]
  const uint8_t* packed;         // [N, runs * 64]
  const __nv_bfloat16* scales;   // [runs * 128 / group, N]
  const float* bias;             // [N] or null
  void* out;                     // [M, N]
  int64_t x_stride;
  int rows, outer, inner, runs;
  int gelu;
  int split;                     // warps along K, a power of two up to 8
};

__device__ __forceinline__ uint32_t nibbles_bf16x2(uint32_t w) {
  const uint32_t biased = (w & 0x000f000fu) | 0x43004300u;
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&biased),
                                   __bfloat162bfloat162(__ushort_as_bfloat16(0x4308)));  // 136
  return *reinterpret_cast<const uint32_t*>(&v);
}

// TN: n8 tiles of x rows; AHEAD: runs whose loads are in flight together.
template <int TN, int GROUP, typename OutT>
__global__ void __launch_bounds__(kW4Warps * 32) linear_w4_kernel(W4Args a) {
  constexpr int AHEAD = TN == 4 ? 2 : 4;
  constexpr int GROUPS = kW4Run / GROUP;  // groups per run
  constexpr int WORDS = 4 / GROUPS;       // words per group and lane
  __shared__ float4 join[kW4Warps][TN][32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t4 = lane % 4;
  const int part = warp % a.split, tile = warp / a.split;
  const int n0 = (blockIdx.x * (kW4Warps / a.split) + tile) * 16;
  const int m0 = blockIdx.y * (TN * 8);
  // columns past the end read the last one and are not written
  const int col[2] = {min(n0 + g, a.outer - 1), min(n0 + g + 8, a.outer - 1)};
  const int64_t pitch = static_cast<int64_t>(a.runs) * (kW4Run / 2);
  const uint8_t* w_row[2] = {a.packed + col[0] * pitch + t4 * 16, a.packed + col[1] * pitch + t4 * 16};
  griddep_wait();
  griddep_launch_dependents();

  const __nv_bfloat16* x_row[TN];
  bool x_in[TN];
#pragma unroll
  for (int i = 0; i < TN; ++i) {
    const int m = m0 + i * 8 + g;
    x_in[i] = m < a.rows;
    x_row[i] = a.x + (x_in[i] ? m : 0) * a.x_stride + t4 * 8;
  }

  float sum[TN][4];
#pragma unroll
  for (int i = 0; i < TN; ++i) sum[i][0] = sum[i][1] = sum[i][2] = sum[i][3] = 0.f;

  for (int r0 = part; r0 < a.runs; r0 += a.split * AHEAD) {
    uint4 w[AHEAD][2];
    __nv_bfloat16 s[AHEAD][GROUPS][2];
#pragma unroll
    for (int p = 0; p < AHEAD; ++p) {
      const int r = r0 + p * a.split;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        w[p][h] = make_uint4(0u, 0u, 0u, 0u);
        if (r < a.runs) w[p][h] = __ldg(reinterpret_cast<const uint4*>(w_row[h] + static_cast<int64_t>(r) * (kW4Run / 2)));
#pragma unroll
        for (int q = 0; q < GROUPS; ++q) {
          s[p][q][h] = __ushort_as_bfloat16(0);
          if (r < a.runs) s[p][q][h] = a.scales[static_cast<int64_t>(r * GROUPS + q) * a.outer + col[h]];
        }
      }
    }
#pragma unroll
    for (int p = 0; p < AHEAD; ++p) {
      const int r = r0 + p * a.split;
      if (r >= a.runs) break;
      const uint32_t wa[4] = {w[p][0].x, w[p][0].y, w[p][0].z, w[p][0].w};
      const uint32_t wb[4] = {w[p][1].x, w[p][1].y, w[p][1].z, w[p][1].w};
#pragma unroll
      for (int q = 0; q < GROUPS; ++q) {
        float acc[TN][4] = {};
#pragma unroll
        for (int c = q * WORDS; c < (q + 1) * WORDS; ++c) {
          const uint32_t a0[4] = {nibbles_bf16x2(wa[c]), nibbles_bf16x2(wb[c]), nibbles_bf16x2(wa[c] >> 4),
                                  nibbles_bf16x2(wb[c] >> 4)};
          const uint32_t a1[4] = {nibbles_bf16x2(wa[c] >> 8), nibbles_bf16x2(wb[c] >> 8), nibbles_bf16x2(wa[c] >> 12),
                                  nibbles_bf16x2(wb[c] >> 12)};
          const int k = r * kW4Run + c * 32;
#pragma unroll
          for (int i = 0; i < TN; ++i) {
            uint4 x = make_uint4(0u, 0u, 0u, 0u);
            if (x_in[i] && k + t4 * 8 < a.inner) x = *reinterpret_cast<const uint4*>(x_row[i] + k);
            mma_m16n8k16_bf16(acc[i], a0, x.x, x.y);
            mma_m16n8k16_bf16(acc[i], a1, x.z, x.w);
          }
        }
        const float s0 = __bfloat162float(s[p][q][0]), s1 = __bfloat162float(s[p][q][1]);
#pragma unroll
        for (int i = 0; i < TN; ++i) {
          sum[i][0] = fmaf(s0, acc[i][0], sum[i][0]);
          sum[i][1] = fmaf(s0, acc[i][1], sum[i][1]);
          sum[i][2] = fmaf(s1, acc[i][2], sum[i][2]);
          sum[i][3] = fmaf(s1, acc[i][3], sum[i][3]);
        }
      }
    }
  }

  if (a.split > 1) {
#pragma unroll
    for (int i = 0; i < TN; ++i) join[warp][i][lane] = make_float4(sum[i][0], sum[i][1], sum[i][2], sum[i][3]);
    __syncthreads();
    if (part != 0) return;
    for (int w = 1; w < a.split; ++w) {
#pragma unroll
      for (int i = 0; i < TN; ++i) {
        const float4 v = join[warp + w][i][lane];
        sum[i][0] += v.x; sum[i][1] += v.y; sum[i][2] += v.z; sum[i][3] += v.w;
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int n = n0 + g + 8 * h;
    if (n >= a.outer) continue;
    const float bias = a.bias == nullptr ? 0.f : a.bias[n];
#pragma unroll
    for (int i = 0; i < TN; ++i) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int m = m0 + i * 8 + 2 * t4 + e;
        if (m >= a.rows) continue;
        float y = sum[i][2 * h + e] + bias;
        if (a.gelu) y = 0.5f * y * (1.f + erff(y * 0.70710678118654752f));
        OutT* dst = static_cast<OutT*>(a.out) + static_cast<int64_t>(m) * a.outer + n;
        if constexpr (sizeof(OutT) == 4) {
          *dst = y;
        } else {
          *dst = __float2bfloat16_rn(y);
        }
      }
    }
  }
}

}  // namespace b200tx
