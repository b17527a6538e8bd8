// kv8_attention_kernels.cuh -- attention of a few new tokens over the 8-bit
// cache of kv8_cache_kernels.cuh.
//
//   out_i = sum_j p_ij v_j,   p_i = softmax over j <= position(i) of scale q_i . k_j
//   k_j = ks (code_j - 128),  v_j likewise; the open block's tokens are bf16
//
// What bounds it: a cached token is 2 Hkv D bytes read once, and 4 Hq D
// operations; with a few queries that is far below the tensor cores' rate, so
// the cache's bytes over HBM bound it, and the split has to give every SM an
// equal share of them whatever the lengths are.
//
// Split.  The rows of a (sequence, kv head) are its tokens x the query heads of
// the group, in tiles of 16, one m16 MMA tile.  A tile's keys are cut into
// steps of 32 codes (16 tokens in the open block: as many bytes).  All steps
// of all tiles form one line, cut into equal ranges, one per CTA: a CTA ends
// within a tile's keys, or does several tiles, and no length of any sequence
// leaves SMs idle.  A tile that lies in several CTAs is joined by the one
// that finishes last, in the order of the ranges, so results do not depend on
// the order of arrival.
//
// Within a CTA the steps of a tile go round the four warps.  Each lane copies
// exactly the bytes that it will use itself (cp.async into its own place of a
// ring in shared memory): a queue with neither barriers nor bank conflicts,
// deep enough to cover the HBM latency.
//
// Numbers.  Codes become fp16 by one permute and one subtraction (exact), the
// queries are scaled by a power of two per row into fp16 (exact but for what
// is 2^-24 of the row's largest value), products accumulate in fp32, the
// block scale multiplies the sum.  Probabilities are rounded to fp16 (2^-11,
// finer than the bf16 output's 2^-8).  In the open block keys and
// queries are bf16 and each probability is the sum of two bf16 numbers.  The
// running maximum moves only when a score exceeds it by more than 2^8, which
// leaves room in fp16 and saves most rescalings.
#pragma once

#include "attention_mma_kernels.cuh"
#include "kv8_cache_kernels.cuh"

namespace b200tx {

constexpr int kKv8Warps = 4;
constexpr int kKv8Step = 32;      // tokens per step in full blocks
constexpr int kKv8TailStep = 16;  // tokens per step in the open block
constexpr int kKv8Rows = 16;      // rows per tile
constexpr float kKv8Headroom = 8.f;  // log2 of how far a score may pass the running maximum

template <int D>
struct Kv8Shape {
  static constexpr int STAGES = D >= 128 ? 3 : D == 64 ? 4 : 6;
  static constexpr int CTAS = D == 256 ? 1 : D == 128 ? 2 : D == 64 ? 3 : 4;  // per SM
  static constexpr int KB = D / 4 < 16 ? D / 4 : 16;  // bytes per key copy
  static constexpr int KC = D / 4 / KB;               // key copies per row and lane
  static constexpr int VB = D / 8 < 16 ? D / 8 : 16;  // bytes per value copy
  static constexpr int VC = D / 8 / VB;
  static constexpr int HALF = kKv8Step * D;           // bytes of a step's keys (or values)
  static constexpr int STAGE = 2 * HALF + 16;         // and the two scales
  static constexpr int KSTEPS = D / 16;               // k16 steps of q . k
  static constexpr int NT = D / 8;                    // n8 tiles of the output
  static constexpr int RING = kKv8Warps * STAGES * STAGE;
  static constexpr int JOIN = kKv8Warps * kKv8Rows * D * 4;  // the warps' outputs, over the ring
  static constexpr int MAIN = RING > JOIN ? RING : JOIN;
  // a CTA's part of a tile: outputs as fragments, then (max, sum) of 16 rows
  static constexpr int PART_FLOATS = kKv8Rows * D + 2 * kKv8Rows;
};

struct Kv8AttnArgs {
  Kv8Cache cache;
  const __nv_bfloat16* q;               // [batch, tokens, heads, D], heads dense
  int64_t q_batch_stride, q_token_stride;
  __nv_bfloat16* out;                   // [batch, tokens, heads, D]
  const int32_t* slot_ids;
  const int32_t* counts;
  int batch, tokens, heads, group, row_tiles;
  float scale_log2;                     // scale * log2(e)
  float* parts;                         // [grid, 2, PART_FLOATS]
  unsigned int* arrivals;               // [grid], zero between launches
};

template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool take) {
  const int n = take ? BYTES : 0;  // what is not taken reads as zero
  if constexpr (BYTES == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  } else {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
  }
}

__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma_m16n8k16_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Two codes (bytes SEL of the words) as fp16 numbers code - 128: the byte under
// 0x64 is 1024 + code.
template <int SEL>
__device__ __forceinline__ uint32_t codes_f16x2(uint32_t w) {
  const uint32_t biased = __byte_perm(w, 0x64646464u, SEL);
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&biased), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <int BYTES>
__device__ __forceinline__ void lds_words(const uint8_t* p, uint32_t (&w)[BYTES / 4]) {
  if constexpr (BYTES == 16) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (BYTES == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// What one sequence asks for: its tokens in all, and the steps over them.
struct Kv8Sequence {
  int slot, total, count, steps;
  bool bad;  // no such slot, or longer than its page table: outputs are NaN
};

__device__ __forceinline__ Kv8Sequence kv8_sequence(const Kv8AttnArgs& a, int b) {
  Kv8Sequence s;
  s.slot = a.slot_ids == nullptr ? b : a.slot_ids[b];
  s.count = a.counts == nullptr ? a.tokens : min(max(a.counts[b], 0), a.tokens);
  s.bad = s.slot < 0 || s.slot >= a.cache.slots;
  const int64_t total = s.bad ? 0 : static_cast<int64_t>(max(0, a.cache.lengths[s.slot])) + s.count;
  s.bad = s.bad || total > static_cast<int64_t>(a.cache.max_blocks) * kKv8Block;
  s.total = s.bad ? 0 : static_cast<int>(total);
  const int open = s.total % kKv8Block;
  s.steps = s.bad || s.count == 0
                ? 0
                : s.total / kKv8Block * (kKv8Block / kKv8Step) + (open + kKv8TailStep - 1) / kKv8TailStep;
  return s;
}

template <int D>
__global__ void __launch_bounds__(kKv8Warps * 32, Kv8Shape<D>::CTAS) kv8_attention_kernel(Kv8AttnArgs a) {
  using S = Kv8Shape<D>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t scan[kKv8Warps];
  __shared__ int64_t found_offset;
  __shared__ int found_b;
  __shared__ float2 warp_ml[kKv8Warps][kKv8Rows];
  __shared__ float row_sum[kKv8Rows];
  __shared__ float row_part[8][kKv8Rows];
  __shared__ int is_last;

  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t4 = lane % 4;
  const int tiles = a.cache.kv_heads * a.row_tiles;  // of a sequence
  griddep_wait();
  griddep_launch_dependents();

  // ---- where this CTA's range begins
  const int chunk = (a.batch + kKv8Warps * 32 - 1) / (kKv8Warps * 32);
  int64_t mine = 0;
  for (int b = tid * chunk; b < min(a.batch, (tid + 1) * chunk); ++b) {
    const Kv8Sequence s = kv8_sequence(a, b);
    mine += s.steps;
    if (s.steps == 0 && b % gridDim.x == blockIdx.x) {
      // nothing to attend to: zeros (NaN if the sequence is not one)
      const uint32_t fill = s.bad ? 0x7fff7fffu : 0u;
      uint4* o = reinterpret_cast<uint4*>(a.out + static_cast<int64_t>(b) * a.tokens * a.heads * D);
      for (int64_t i = 0; i < static_cast<int64_t>(a.tokens) * a.heads * D / 8; ++i) o[i] = make_uint4(fill, fill, fill, fill);
    }
  }
  int64_t before = mine;  // inclusive sum over the warp, then exclusive over the CTA
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int64_t n = __shfl_up_sync(0xffffffffu, before, d);
    if (lane >= d) before += n;
  }
  if (lane == 31) scan[warp] = before;
  __syncthreads();
  before -= mine;
  int64_t all = 0;
#pragma unroll
  for (int w = 0; w < kKv8Warps; ++w) {
    if (w < warp) before += scan[w];
    all += scan[w];
  }
  const int64_t total = all * tiles;
  // at least one step a warp, so that short contexts are not cut into crumbs
  const int64_t ctas = min(static_cast<int64_t>(gridDim.x), (total + kKv8Warps - 1) / kKv8Warps);
  if (blockIdx.x >= ctas) return;
  const int64_t lo = total * blockIdx.x / ctas, hi = total * (blockIdx.x + 1) / ctas;
  if (lo >= before * tiles && lo < (before + mine) * tiles) {
    int64_t offset = before * tiles;
    int b = tid * chunk;
    for (;; ++b) {
      const int64_t n = static_cast<int64_t>(kv8_sequence(a, b).steps) * tiles;
      if (lo < offset + n) break;
      offset += n;
    }
    found_b = b;
    found_offset = offset;
  }
  __syncthreads();

  int b = found_b;
  int64_t offset = found_offset;  // of sequence b in the line
  Kv8Sequence seq = kv8_sequence(a, b);
  uint8_t* const ring = smem + warp * S::STAGES * S::STAGE;
  int64_t cur = lo;
  while (cur < hi) {
    while (cur >= offset + static_cast<int64_t>(seq.steps) * tiles) {
      offset += static_cast<int64_t>(seq.steps) * tiles;
      seq = kv8_sequence(a, ++b);
    }
    const int tile = static_cast<int>((cur - offset) / seq.steps);
    const int64_t tile_begin = offset + static_cast<int64_t>(tile) * seq.steps;
    const int step0 = static_cast<int>(cur - tile_begin);
    const int step1 = static_cast<int>(min(static_cast<int64_t>(seq.steps), hi - tile_begin));
    const int head = tile % a.cache.kv_heads;
    const int row0 = tile / a.cache.kv_heads * kKv8Rows;
    const int rows = min(kKv8Rows, a.tokens * a.group - row0);
    const int full = seq.total / kKv8Block;
    const int open = seq.total - full * kKv8Block;
    const int start = seq.total - seq.count;
    const int mine_steps = max(0, (step1 - step0 - warp + kKv8Warps - 1) / kKv8Warps);
    bool poisoned = false;

    // ---- this warp's copies.  Step k of the warp is step step0 + warp + 4 k.
    int pages = 0;  // lane i: the page of step (k & ~31) + i of the warp
    auto issue = [&](int k) {
      if (k < mine_steps) {
        if ((k & 31) == 0) {
          const int step = step0 + warp + kKv8Warps * (k + lane);
          pages = step < 2 * full && k + lane < mine_steps ? kv8_page(a.cache, seq.slot, step / 2) : 0;
        }
        const int step = step0 + warp + kKv8Warps * k;
        const int page = __shfl_sync(0xffffffffu, pages, k & 31);
        const uint32_t stage = smem_u32(ring + (k % S::STAGES) * S::STAGE);
        if (step < 2 * full) {
          const bool good = page >= 0;
          poisoned = poisoned || !good;
          const int64_t at = static_cast<int64_t>(good ? page : 0) * 2 * a.cache.kv_heads + head;
          const uint8_t* kp = a.cache.codes + at * kKv8Block * D + (step & 1) * S::HALF;
          const uint8_t* vp = kp + static_cast<int64_t>(a.cache.kv_heads) * kKv8Block * D;
#pragma unroll
          for (int n = 0; n < 4; ++n) {
#pragma unroll
            for (int c = 0; c < S::KC; ++c)
              cp_async<S::KB>(stage + ((n * S::KC + c) * 32 + lane) * S::KB, kp + (n * 8 + g) * D + c * 64 + t4 * S::KB, good);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {  // tokens (i / 4) * 16 + {2t, 2t+1, 2t+8, 2t+9}
            const int token = (i / 4) * 16 + 2 * t4 + (i & 1) + ((i >> 1) & 1) * 8;
#pragma unroll
            for (int c = 0; c < S::VC; ++c)
              cp_async<S::VB>(stage + S::HALF + ((i * S::VC + c) * 32 + lane) * S::VB, vp + token * D + c * 128 + g * S::VB, good);
          }
          if (lane < 2) cp_async<4>(stage + 2 * S::HALF + 4 * lane, a.cache.scales + at + lane * a.cache.kv_heads, good);
        } else {
          const int first = (step - 2 * full) * kKv8TailStep;
          const __nv_bfloat16* kp = kv8_tail(a.cache, seq.slot, full & 1, 0, head, D);
          const __nv_bfloat16* vp = kv8_tail(a.cache, seq.slot, full & 1, 1, head, D);
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int token = first + n * 8 + g;
#pragma unroll
            for (int c = 0; c < S::KC; ++c) {
#pragma unroll
              for (int h = 0; h < 2; ++h)
                cp_async<S::KB>(stage + (((n * S::KC + c) * 2 + h) * 32 + lane) * S::KB,
                                kp + token * D + c * 64 + t4 * S::KB + h * (S::KB / 2), token < open);
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int token = first + 2 * t4 + (i & 1) + (i >> 1) * 8;
#pragma unroll
            for (int c = 0; c < S::VC; ++c) {
#pragma unroll
              for (int h = 0; h < 2; ++h)
                cp_async<S::VB>(stage + S::HALF + (((i * S::VC + c) * 2 + h) * 32 + lane) * S::VB,
                                vp + token * D + c * 128 + g * S::VB + h * (S::VB / 2), token < open);
            }
          }
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int k = 0; k < S::STAGES - 1; ++k) issue(k);

    // ---- queries: rows g and g + 8 of the tile, scaled by a power of two into fp16
    uint32_t qf[S::KSTEPS][4];
    float row_scale[2];  // turns a sum of products into a log2 score
    int limit[2];        // the row's own position: the last key that it sees
    int least = 0x7fffffff;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = row0 + g + 8 * r;
      const int token = row / a.group;
      const bool real = row < a.tokens * a.group && token < seq.count;
      limit[r] = real ? start + token : -1;
      if (real) least = min(least, limit[r]);
      const __nv_bfloat16* src = a.q + static_cast<int64_t>(b) * a.q_batch_stride + token * a.q_token_stride +
                                 (head * a.group + row % a.group) * D;
      float x[S::KSTEPS][4];
      float peak = 0.f;
      bool finite = true;
#pragma unroll
      for (int c = 0; c < S::KC; ++c) {
#pragma unroll
        for (int i = 0; i < S::KB / 4; ++i) {
          uint2 w = make_uint2(0u, 0u);
          if (real) w = *reinterpret_cast<const uint2*>(src + c * 64 + t4 * S::KB + 4 * i);
          float* y = x[c * (S::KB / 4) + i];
          y[0] = __uint_as_float(w.x << 16); y[1] = __uint_as_float(w.x & 0xffff0000u);
          y[2] = __uint_as_float(w.y << 16); y[3] = __uint_as_float(w.y & 0xffff0000u);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            peak = fmaxf(peak, fabsf(y[e]));
            finite = finite && fabsf(y[e]) < __int_as_float(0x7f800000);
          }
        }
      }
      peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
      peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
      const unsigned ok = __ballot_sync(0xffffffffu, finite);
      finite = ((ok >> (lane & ~3)) & 15u) == 15u;
      // 2^e <= peak < 2^(e+1), clamped so that 2^e and 2^-e are normal numbers
      const int e = min(126, max(-100, static_cast<int>(__float_as_uint(peak) >> 23) - 127));
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      row_scale[r] = finite ? up * a.scale_log2 : __int_as_float(0x7fffffff);
#pragma unroll
      for (int k = 0; k < S::KSTEPS; ++k) {
        qf[k][r] = finite ? pack_f16x2(x[k][0] * down, x[k][1] * down) : 0u;
        qf[k][2 + r] = finite ? pack_f16x2(x[k][2] * down, x[k][3] * down) : 0u;
      }
    }
    least = __reduce_min_sync(0xffffffffu, least);

    float o[S::NT][4];
#pragma unroll
    for (int j = 0; j < S::NT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    const float minus_inf = __int_as_float(0xff800000);
    float m[2] = {minus_inf, minus_inf}, l[2] = {0.f, 0.f};

    // Scores (log2) in place to probabilities; `factor` turns sums into scores.
    auto softmax = [&](auto& s, const float (&factor)[2], int first_token, bool masked) {
      constexpr int N = sizeof(s) / sizeof(s[0]);
      float top[2] = {minus_inf, minus_inf};
#pragma unroll
      for (int n = 0; n < N; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] *= factor[e >> 1];
          if (masked && first_token + n * 8 + 2 * t4 + (e & 1) > limit[e >> 1]) s[n][e] = minus_inf;
          top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      }
      if (__any_sync(0xffffffffu, top[0] > m[0] + kKv8Headroom || top[1] > m[1] + kKv8Headroom)) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float next = fmaxf(m[r], top[r]);
          const float by = m[r] == minus_inf ? 0.f : fast_exp2(m[r] - next);
          m[r] = next;
          l[r] *= by;
#pragma unroll
          for (int j = 0; j < S::NT; ++j) {
            o[j][2 * r] *= by;
            o[j][2 * r + 1] *= by;
          }
        }
      }
      const float from[2] = {m[0] == minus_inf ? 0.f : m[0], m[1] == minus_inf ? 0.f : m[1]};
#pragma unroll
      for (int n = 0; n < N; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] = fast_exp2(s[n][e] - from[e >> 1]);
          l[e >> 1] += s[n][e];
        }
      }
    };

    for (int k = 0; k < mine_steps; ++k) {
      cp_async_wait<S::STAGES - 2>();
      __syncwarp();
      issue(k + S::STAGES - 1);
      const int step = step0 + warp + kKv8Warps * k;
      uint8_t* stage = ring + (k % S::STAGES) * S::STAGE;
      if (step < 2 * full) {
        const int first_token = step * kKv8Step;
        const float2 scales = *reinterpret_cast<const float2*>(stage + 2 * S::HALF);
        float s[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
          for (int c = 0; c < S::KC; ++c) {
            uint32_t w[S::KB / 4];
            lds_words<S::KB>(stage + ((n * S::KC + c) * 32 + lane) * S::KB, w);
#pragma unroll
            for (int i = 0; i < S::KB / 4; ++i)
              mma_m16n8k16_f16(s[n], qf[c * (S::KB / 4) + i], codes_f16x2<0x4140>(w[i]), codes_f16x2<0x4342>(w[i]));
          }
        }
        const bool masked = first_token + kKv8Step - 1 > least;
        const float factor[2] = {row_scale[0] * scales.x, row_scale[1] * scales.x};
        softmax(s, factor, first_token, masked);
        // a row that sees none of these keys takes nothing of them, whatever the scale
        const float vs[2] = {masked && first_token > limit[0] ? 0.f : scales.y, masked && first_token > limit[1] ? 0.f : scales.y};
        uint32_t p[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          p[h][0] = pack_f16x2(s[2 * h][0], s[2 * h][1]);
          p[h][1] = pack_f16x2(s[2 * h][2], s[2 * h][3]);
          p[h][2] = pack_f16x2(s[2 * h + 1][0], s[2 * h + 1][1]);
          p[h][3] = pack_f16x2(s[2 * h + 1][2], s[2 * h + 1][3]);
        }
#pragma unroll
        for (int c = 0; c < S::VC; ++c) {
          uint32_t w[8][S::VB / 4];
#pragma unroll
          for (int i = 0; i < 8; ++i) lds_words<S::VB>(stage + S::HALF + ((i * S::VC + c) * 32 + lane) * S::VB, w[i]);
#pragma unroll
          for (int i = 0; i < S::VB / 4; ++i) {
            float acc[4][4] = {};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              // bytes of two tokens side by side: the b fragments' pairs along k
              const uint32_t ab0 = __byte_perm(w[4 * h][i], w[4 * h + 1][i], 0x5140);
              const uint32_t ab1 = __byte_perm(w[4 * h][i], w[4 * h + 1][i], 0x7362);
              const uint32_t cd0 = __byte_perm(w[4 * h + 2][i], w[4 * h + 3][i], 0x5140);
              const uint32_t cd1 = __byte_perm(w[4 * h + 2][i], w[4 * h + 3][i], 0x7362);
              mma_m16n8k16_f16(acc[0], p[h], codes_f16x2<0x4140>(ab0), codes_f16x2<0x4140>(cd0));
              mma_m16n8k16_f16(acc[1], p[h], codes_f16x2<0x4342>(ab0), codes_f16x2<0x4342>(cd0));
              mma_m16n8k16_f16(acc[2], p[h], codes_f16x2<0x4140>(ab1), codes_f16x2<0x4140>(cd1));
              mma_m16n8k16_f16(acc[3], p[h], codes_f16x2<0x4342>(ab1), codes_f16x2<0x4342>(cd1));
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float(&dst)[4] = o[c * S::VB + 4 * i + e];
              dst[0] = fmaf(vs[0], acc[e][0], dst[0]);
              dst[1] = fmaf(vs[0], acc[e][1], dst[1]);
              dst[2] = fmaf(vs[1], acc[e][2], dst[2]);
              dst[3] = fmaf(vs[1], acc[e][3], dst[3]);
            }
          }
        }
      } else {
        const int in_tail = (step - 2 * full) * kKv8TailStep;
        const int first_token = full * kKv8Block + in_tail;
        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
          for (int c = 0; c < 2 * S::KC; ++c) {
            uint32_t w[S::KB / 4];
            lds_words<S::KB>(stage + ((n * 2 * S::KC + c) * 32 + lane) * S::KB, w);
#pragma unroll
            for (int i = 0; i < S::KB / 8; ++i) {
              const int ks = c * (S::KB / 8) + i;
              uint32_t qb[4];  // fp16 -> bf16, exact: they came from bf16
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&qf[ks][e]));
                qb[e] = pack_bf16x2(v.x, v.y);
              }
              mma_m16n8k16_bf16(s[n], qb, w[2 * i], w[2 * i + 1]);
            }
          }
        }
        softmax(s, row_scale, first_token, true);
        uint32_t hi[4], low[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = s[e >> 1][2 * (e & 1)], y = s[e >> 1][2 * (e & 1) + 1];
          hi[e] = pack_bf16x2(x, y);
          low[e] = pack_bf16x2(x - __uint_as_float(hi[e] << 16), y - __uint_as_float(hi[e] & 0xffff0000u));
        }
        // Values that are not finite, and rows that must not see them: 0 x inf
        // would be NaN, so such a step goes value by value.
        bool odd = false;
        if (seq.count > 1) {
#pragma unroll
          for (int i = 0; i < 8 * S::VC; ++i) {
            uint32_t w[S::VB / 4];
            lds_words<S::VB>(stage + S::HALF + (i * 32 + lane) * S::VB, w);
#pragma unroll
            for (int e = 0; e < S::VB / 4; ++e)
              odd = odd || (w[e] & 0x7f80u) == 0x7f80u || (w[e] & 0x7f800000u) == 0x7f800000u;
          }
          odd = __any_sync(0xffffffffu, odd);
        }
        if (!odd) {
#pragma unroll
          for (int c = 0; c < S::VC; ++c) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t w[4][S::VB / 4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                lds_words<S::VB>(stage + S::HALF + (((i * S::VC + c) * 2 + h) * 32 + lane) * S::VB, w[i]);
#pragma unroll
              for (int i = 0; i < S::VB / 4; ++i) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  float(&dst)[4] = o[c * S::VB + h * (S::VB / 2) + 2 * i + e];
                  const uint32_t b0 = __byte_perm(w[0][i], w[1][i], e ? 0x7632 : 0x5410);
                  const uint32_t b1 = __byte_perm(w[2][i], w[3][i], e ? 0x7632 : 0x5410);
                  mma_m16n8k16_bf16(dst, hi, b0, b1);
                  mma_m16n8k16_bf16(dst, low, b0, b1);
                }
              }
            }
          }
        } else {
          // probabilities over the step's keys, which are used up: [16 rows][16 tokens]
          __syncwarp();
          float* pr = reinterpret_cast<float*>(stage);
#pragma unroll
          for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) pr[(g + 8 * (e >> 1)) * 16 + n * 8 + 2 * t4 + (e & 1)] = s[n][e];
          }
          __syncwarp();
          for (int token = 0; token < kKv8TailStep; ++token) {
            // token = 2t' + (i & 1) + (i >> 1) * 8 lies with lanes t' in copy i
            const int from_t = (token % 8) / 2, i = (token & 1) + (token / 8) * 2;
            const int where = first_token + token;
#pragma unroll
            for (int j = 0; j < S::NT; ++j) {
              const int c = j / S::VB, h = (j % S::VB) / (S::VB / 2), at = j % (S::VB / 2);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int from = (2 * t4 + (e & 1)) * 4 + from_t;
                const uint8_t* p = stage + S::HALF + (((i * S::VC + c) * 2 + h) * 32 + from) * S::VB + 2 * at;
                const float v = __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p)) << 16);
                if (where <= limit[e >> 1]) o[j][e] = fmaf(pr[(g + 8 * (e >> 1)) * 16 + token], v, o[j][e]);
              }
            }
          }
          __syncwarp();
        }
      }
    }
    cp_async_wait<0>();

    // ---- join the warps: fragments [warp][n tile][lane], a quarter of the n tiles each
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (poisoned) l[r] = __int_as_float(0x7fffffff);
      if (t4 == 0) warp_ml[warp][g + 8 * r] = make_float2(m[r], l[r]);
    }
    __syncthreads();  // everyone is done with the ring
    float4* const join = reinterpret_cast<float4*>(smem);
#pragma unroll
    for (int j = 0; j < S::NT; ++j) join[(warp * S::NT + j) * 32 + lane] = make_float4(o[j][0], o[j][1], o[j][2], o[j][3]);
    __syncthreads();
    float weight[kKv8Warps][2], top[2], sum[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float2 ml[kKv8Warps];
      top[r] = minus_inf;
      sum[r] = 0.f;
#pragma unroll
      for (int w = 0; w < kKv8Warps; ++w) {
        ml[w] = warp_ml[w][g + 8 * r];
        top[r] = fmaxf(top[r], ml[w].x);
      }
#pragma unroll
      for (int w = 0; w < kKv8Warps; ++w) {
        weight[w][r] = ml[w].x == minus_inf ? 0.f : fast_exp2(ml[w].x - top[r]);
        sum[r] += ml[w].x == minus_inf && ml[w].y == 0.f ? 0.f : weight[w][r] * ml[w].y;
      }
    }
    constexpr int QUARTER = S::NT / kKv8Warps;
    float4 acc[QUARTER];
#pragma unroll
    for (int i = 0; i < QUARTER; ++i) {
      const int j = warp * QUARTER + i;
      acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kKv8Warps; ++w) {
        const float4 v = join[(w * S::NT + j) * 32 + lane];
        acc[i].x = fmaf(weight[w][0], v.x, acc[i].x);
        acc[i].y = fmaf(weight[w][0], v.y, acc[i].y);
        acc[i].z = fmaf(weight[w][1], v.z, acc[i].z);
        acc[i].w = fmaf(weight[w][1], v.w, acc[i].w);
      }
    }

    // ---- a tile in several CTAs: leave the part, the last to arrive joins them
    bool write = step0 == 0 && step1 == seq.steps;
    if (!write) {
      const int64_t c0 = ((tile_begin + 1) * ctas - 1) / total;
      const int64_t c1 = ((tile_begin + seq.steps) * ctas - 1) / total;
      const int n_parts = static_cast<int>(c1 - c0) + 1;
      float* part = a.parts + (static_cast<int64_t>(blockIdx.x) * 2 + (cur == lo ? 0 : 1)) * S::PART_FLOATS;
#pragma unroll
      for (int i = 0; i < QUARTER; ++i)
        __stcg(reinterpret_cast<float4*>(part) + (warp * QUARTER + i) * 32 + lane, acc[i]);
      if (warp == 0 && t4 == 0) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
          __stcg(reinterpret_cast<float2*>(part + kKv8Rows * D) + g + 8 * r, make_float2(top[r], sum[r]));
      }
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const unsigned int had = atomicAdd(a.arrivals + c0, 1u);
        is_last = had + 1 == static_cast<unsigned int>(n_parts);
        if (is_last) a.arrivals[c0] = 0;  // ready for the next launch
      }
      __syncthreads();
      write = is_last;
      if (write) {
        __threadfence();
        const int64_t first_lo = total * c0 / ctas;
        auto part_of = [&](int i) {
          const int which = i == 0 && first_lo != tile_begin ? 1 : 0;
          return a.parts + ((c0 + i) * 2 + which) * S::PART_FLOATS;
        };
        // every row's maximum and sum over the parts; the parts' weights go to shared memory
        float2* const ml = reinterpret_cast<float2*>(smem);
        const int row = tid % kKv8Rows, lane8 = tid / kKv8Rows;
        float best = minus_inf;
        for (int i = lane8; i < n_parts; i += 8) {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(part_of(i) + kKv8Rows * D) + row);
          ml[i * kKv8Rows + row] = v;
          best = fmaxf(best, v.x);
        }
        row_part[lane8][row] = best;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) best = fmaxf(best, row_part[i][row]);
        __syncthreads();
        float part_sum = 0.f;
        for (int i = lane8; i < n_parts; i += 8) {
          const float2 v = ml[i * kKv8Rows + row];
          const float w = v.x == minus_inf ? 0.f : fast_exp2(v.x - best);
          part_sum += v.x == minus_inf && v.y == 0.f ? 0.f : w * v.y;
          ml[i * kKv8Rows + row].x = w;
        }
        row_part[lane8][row] = part_sum;
        __syncthreads();
        if (tid < kKv8Rows) {
          float s = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) s += row_part[i][tid];
          row_sum[tid] = s;
        }
        __syncthreads();
        sum[0] = row_sum[g];
        sum[1] = row_sum[g + 8];
#pragma unroll
        for (int i = 0; i < QUARTER; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int i = 0; i < n_parts; ++i) {
          const float w0 = ml[i * kKv8Rows + g].x, w1 = ml[i * kKv8Rows + g + 8].x;
          const float4* src = reinterpret_cast<const float4*>(part_of(i)) + warp * QUARTER * 32 + lane;
#pragma unroll
          for (int j = 0; j < QUARTER; ++j) {
            const float4 v = __ldcg(src + j * 32);
            acc[j].x = fmaf(w0, v.x, acc[j].x);
            acc[j].y = fmaf(w0, v.y, acc[j].y);
            acc[j].z = fmaf(w1, v.z, acc[j].z);
            acc[j].w = fmaf(w1, v.w, acc[j].w);
          }
        }
      }
    }
    if (write) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = g + 8 * r;
        if (row >= rows) continue;
        const int token = (row0 + row) / a.group;
        const bool real = token < seq.count && sum[r] != 0.f;  // padding rows are zero
        const float by = real ? 1.f / sum[r] : 0.f;
        __nv_bfloat16* dst = a.out + ((static_cast<int64_t>(b) * a.tokens + token) * a.heads + head * a.group +
                                      (row0 + row) % a.group) * D;
#pragma unroll
        for (int i = 0; i < QUARTER; ++i) {
          const int j = warp * QUARTER + i;  // dims c * 128 + n * VB + j % VB of columns n = 2t, 2t + 1
          const int d = j / S::VB * 128 + j % S::VB;
          dst[d + (2 * t4) * S::VB] = __float2bfloat16_rn(real ? (r ? acc[i].z : acc[i].x) * by : 0.f);
          dst[d + (2 * t4 + 1) * S::VB] = __float2bfloat16_rn(real ? (r ? acc[i].w : acc[i].y) * by : 0.f);
        }
      }
    }
    __syncthreads();  // the ring and the shared rows are free again
    cur = tile_begin + step1;
  }
}

}  // namespace b200tx
