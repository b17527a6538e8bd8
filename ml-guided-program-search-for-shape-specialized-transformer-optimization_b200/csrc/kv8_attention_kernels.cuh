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
// the group, in tiles of 8 NR.  A tile's keys are cut into steps of 16 to 64
// codes, 8 KB of keys and values (4 KB for head_dim 32), and half as many tokens in
// the open block.  All steps of all tiles, and a fixed cost for each tile, form
// one line, cut into equal ranges, one per CTA: a CTA ends within a tile's keys,
// or does several tiles, and no length of any sequence leaves SMs idle.  A tile
// that lies in several CTAs is joined by the one that finishes last, in the order
// of the ranges, so results do not depend on the order of arrival.
//
// Within a CTA the steps of a tile go round the four warps.  Each warp has a ring
// of steps in shared memory of its own, filled by cp.async: no barrier between
// warps, deep enough to cover the HBM latency.  A copy of 8 lanes is one
// 128-byte line; with the lanes in the fragments' order instead (rows 2 t for
// values) the call took 1.29 times as long (16 sequences x 8192 tokens, 8 heads of
// 128).  Within a line the 16-byte chunks are permuted by
// the row, so that the fragments are read without bank conflicts.
//
// Products.  Keys and values are the A operand (16 tokens, or 16 dims), queries
// and probabilities the B operand (8 rows), so that 8 rows cost one MMA and a
// code is expanded once for all rows of a tile.  The dims' order within a product
// is free: a lane's bytes are consecutive in memory, and the queries are laid out to match.
//
// Numbers.  A code byte under a zero byte is the fp16 number code 2^-24, a
// subnormal, which the tensor cores take as exactly as any other: expanding two
// codes is one instruction.  The offset of 128 comes out of the sums, as the
// accumulators start at -128 2^-24 times the row's sum of queries (or
// probabilities; both are MMAs with a constant, and the latter also gives the softmax's
// denominator).  The queries are scaled by a power of two per row into fp16
// (exact but for what is 2^-24 of the row's largest value), products accumulate
// in fp32, the block's scale multiplies the sum.  Probabilities are rounded to
// fp16: to 2^-11 of themselves (finer than the bf16 output's 2^-8) down to 2^-21 of
// the row's largest so far, below that to 2^-32 of it, which takes a million tokens a
// warp to reach 2^-12.  For that a row's exponents are taken from a base 2^7 under its
// running maximum; the base moves only when a score exceeds it by more than 2^15,
// fp16's room, which saves most rescalings and most reductions.  In the open block keys
// and queries are bf16 and each probability is the sum of two bf16 numbers.
//
// Measured: 100000 tokens of 16 heads of 64 in 43 us (4.8 TB/s), 16 x 8192 of 8 heads of
// 128 in 55 us (4.9 TB/s), 64 ragged sequences up to 8192 in 33 us, 1000 tokens of 16
// heads of 64 in 7.9 us.  Of a long call some 8 us are launch, ramp and the last join;
// the rest runs at 6 TB/s.  With 8 to 12 warps an SM the instructions of a step are
// the next bound.
#pragma once

#include "attention_mma_kernels.cuh"
#include "kv8_cache_kernels.cuh"

namespace b200tx {

constexpr int kKv8Warps = 4;
// What beginning and joining a tile costs, in steps, one number for all head_dims.  64 ragged sequences up
// to 8192, with 6 / 12 / 24 steps: head_dim 128 40.5 / 33.9 / 38.5 us, 256 50.1 / 37.6 / 36.0, 32 28.1 / 26.3 /
// 30.4, 64 22.3 / 22.9 / 27.2; 16 x 8 tokens over up to 4000: 128 35.7 / 28.8 / 32.0, 256 27.2 / 22.9 / 23.7,
// 64 21.1 / 21.4 / 24.5; 128 sequences up to 500: 128 20.4 / 21.7 / 23.5, 64 15.0 / 15.8 / 16.3.
constexpr int kKv8TileCost = 12;
constexpr float kKv8JoinShare = 0.5f;  // what a part costs to join, against a step: its root
constexpr float kKv8Under = 7.f;      // log2 of how far a row's base lies under its maximum when it moves
constexpr float kKv8Headroom = 15.f;  // and of how far a score may pass the base: fp16 ends at 2^16
constexpr float kKv8Unit = 16777216.f;  // 2^24: a code's fp16 number is code / 2^24
constexpr uint32_t kKv8OffsetF16 = 0x80808080u;   // two fp16 -2^-17 = -128 / 2^24
constexpr uint32_t kKv8OffsetBf16 = 0xb700b700u;  // two bf16 -2^-17
constexpr float kKv8SumUnit = -131072.f;          // -2^17

template <int D, int NR>
struct Kv8Shape {
  static constexpr int TOK = D <= 64 ? 64 : D == 128 ? 32 : 16;  // tokens per step in full blocks
  static constexpr int TAIL = TOK / 2;                // and in the open block
  static constexpr int T16 = TOK / 16;
  static constexpr int TAIL16 = TAIL < 16 ? 1 : TAIL / 16;  // tiles of a step in the open block,
  static constexpr bool TAIL_HALF = TAIL < 16;              // the only one half empty
  static constexpr int STAGES = D == 32 ? 4 : D == 64 ? 2 : 3;
  static constexpr int CTAS = D >= 128 || NR == 4 ? 2 : 3;  // per SM
  static constexpr int ROWS = 8 * NR;                 // rows per tile
  static constexpr int KB = D / 4 < 16 ? D / 4 : 16;  // bytes per key copy
  static constexpr int KC = D / 4 / KB;               // key copies per row and lane
  static constexpr int VB = D / 8 < 16 ? D / 8 : 16;  // bytes per value copy
  static constexpr int VC = D / 8 / VB;
  static constexpr int HALF = TOK * D;                // bytes of a step's keys (or values)
  static constexpr int STAGE = 2 * HALF + 16;         // and the two scales
  static constexpr int KSTEPS = D / 16;               // k16 steps of q . k
  static constexpr int MT = D / 16;                   // m16 tiles of the output
  static constexpr int FRAGS = MT * NR;               // fragments (4 floats a lane) of the output
  static constexpr int SHARE = FRAGS >= kKv8Warps ? FRAGS / kKv8Warps : 1;  // of one warp, when joining
  static_assert(SHARE <= MT && MT % SHARE == 0, "a warp's share lies in one row group");
  static constexpr int RING = kKv8Warps * STAGES * STAGE;
  static constexpr int JOIN = kKv8Warps * ROWS * D * 4;  // the warps' outputs, over the ring
  static constexpr int MAIN = RING > JOIN ? RING : JOIN;
  // a CTA's part of a tile: outputs as fragments, then (max, sum) of the rows
  static constexpr int PART_FLOATS = ROWS * D + 2 * ROWS;
};

struct Kv8AttnArgs {
  Kv8Cache cache;
  const __nv_bfloat16* q;               // [batch, tokens, heads, D], heads dense
  int64_t q_batch_stride, q_token_stride;
  __nv_bfloat16* out;                   // [batch, tokens, heads, D]
  const int32_t* slot_ids;
  const int32_t* counts;
  int batch, tokens, heads, group;
  float scale_log2;                     // scale * log2(e)
  float* parts;                         // [grid, 2, PART_FLOATS]
  unsigned int* arrivals;               // [grid], zero between launches
};

template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  } else {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
  }
}

// 16 bytes; what is not taken is written as zero, and not read.
__device__ __forceinline__ void cp_async_or_zero(uint32_t dst, const void* src, bool take) {
  const int n = take ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
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

// The same with the accumulator read from elsewhere: d = a b + (c0, c1, c0, c1).
__device__ __forceinline__ void mma_m16n8k16_f16_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                                      float c0, float c1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %10, %11};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}

// An 8 x 8 matrix of 16-bit values, row lane / 4 and columns 2 (lane % 4) + {0, 1}
// in each lane, transposed.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Codes 0 and 2 (1 and 3) of a word as fp16 numbers code 2^-24.
__device__ __forceinline__ uint32_t codes_even(uint32_t w) { return w & 0x00ff00ffu; }
__device__ __forceinline__ uint32_t codes_odd(uint32_t w) { return __byte_perm(w, 0u, 0x4341); }

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

// Where byte `at` of a step's keys or values lies in its half of a stage: chunk
// bits (4..6) exchanged by row bits.  All are linear over exclusive or, so a
// lane's part and a constant part are permuted apart.
template <int D>
__host__ __device__ constexpr uint32_t kv8_k_place(uint32_t at) {  // rows of D codes, read 8 rows x 4 chunks
  return D >= 128 ? at ^ (((at / D) & 1u) << 6) : at;
}
template <int D>
__host__ __device__ constexpr uint32_t kv8_v_place(uint32_t at) {  // read rows {0, 2, 4, 6} x 2 chunks
  return D >= 128 ? at ^ (((at / (2 * D)) & 3u) << 5) : D == 64 ? at ^ (((at >> 7) & 3u) << 5) : at ^ (((at >> 7) & 1u) << 5);
}
template <int D>
__host__ __device__ constexpr uint32_t kv8_tail_k_place(uint32_t at) {  // rows of D bf16, read every other chunk
  return D >= 64 ? at ^ (((at / (2 * D)) & 1u) << 4) : at;
}
template <int D>
__host__ __device__ constexpr uint32_t kv8_tail_v_place(uint32_t at) {
  const uint32_t pair = at / (4 * D);
  return D >= 64 ? at ^ (((pair & 1u) << 4) | ((pair & 2u) << 5)) : at;
}

// What one sequence asks for: its tokens in all, the steps over them, and the units of the
// line: a tile's steps and its fixed cost, for the tiles that its own new tokens fill.
struct Kv8Sequence {
  int slot, total, count, steps;
  unsigned tiles, cost, units;  // cost: of one tile; units: of all
  bool bad;                     // no such slot, or longer than its page table: outputs are NaN
};

template <int TOK, int ROWS>
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
                : s.total / kKv8Block * (kKv8Block / TOK) + (open + TOK / 2 - 1) / (TOK / 2);
  s.cost = s.steps == 0 ? 0u : static_cast<unsigned>(s.steps + kKv8TileCost);
  s.tiles = s.steps == 0 ? 0u : a.cache.kv_heads * ((static_cast<unsigned>(s.count) * a.group + ROWS - 1) / ROWS);
  s.units = s.cost * s.tiles;
  return s;
}

// The line of all units cut into ranges: the first `more` have each + 1.
struct Kv8Ranges {
  unsigned each, more;
  __device__ __forceinline__ unsigned begin(unsigned cta) const { return cta * each + min(cta, more); }
  __device__ __forceinline__ unsigned of(unsigned unit) const {
    const unsigned big = more * (each + 1);
    return unit < big ? unit / (each + 1) : more + (unit - big) / each;
  }
};

template <int D, int NR>
__global__ void __launch_bounds__(kKv8Warps * 32, Kv8Shape<D, NR>::CTAS) kv8_attention_kernel(Kv8AttnArgs a) {
  using S = Kv8Shape<D, NR>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ unsigned scan[kKv8Warps], scan_tiles[kKv8Warps], scan_gaps[kKv8Warps];
  __shared__ unsigned found_offset;
  __shared__ int found_b;
  __shared__ float2 warp_ml[kKv8Warps][S::ROWS];
  __shared__ int is_last;

  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t4 = lane % 4;
  auto sequence = [&](int b) { return kv8_sequence<S::TOK, S::ROWS>(a, b); };
  const float minus_inf = __int_as_float(0xff800000), nan = __int_as_float(0x7fffffff);
  griddep_wait();
  griddep_launch_dependents();

  // ---- where this CTA's range begins
  const int chunk = (a.batch + kKv8Warps * 32 - 1) / (kKv8Warps * 32);
  unsigned mine = 0, mine_tiles = 0;
  bool gaps = false;
  for (int b = tid * chunk; b < min(a.batch, (tid + 1) * chunk); ++b) {
    const Kv8Sequence s = sequence(b);
    mine += s.units;
    mine_tiles += s.tiles;
    gaps = gaps || s.bad || s.count < a.tokens;
  }
  // inclusive sums over the warp, then exclusive over the CTA
  unsigned before = mine;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const unsigned n = __shfl_up_sync(0xffffffffu, before, d);
    if (lane >= d) before += n;
  }
  mine_tiles = __reduce_add_sync(0xffffffffu, mine_tiles);
  const unsigned warp_gaps = __any_sync(0xffffffffu, gaps);
  if (lane == 31) {
    scan[warp] = before;
    scan_tiles[warp] = mine_tiles;
    scan_gaps[warp] = warp_gaps;
  }
  __syncthreads();  // a barrier that joins the flags costs 0.6 us of 1000 tokens of 16 heads of 64
  before -= mine;
  unsigned total = 0, tiles = 0, all_gaps = 0;  // the host has checked that they fit
#pragma unroll
  for (int w = 0; w < kKv8Warps; ++w) {
    if (w < warp) before += scan[w];
    total += scan[w];
    tiles += scan_tiles[w];
    all_gaps |= scan_gaps[w];
  }
  if (all_gaps != 0) {
    // Rows past the counts are zero, all rows of what is no sequence NaN: no tile has them.  A
    // sequence's rows for each CTA, or a part of them where the sequences are fewer.
    const unsigned parts = max(1u, gridDim.x / a.batch);
    for (unsigned item = blockIdx.x; item < parts * a.batch; item += gridDim.x) {
      const unsigned b = item % a.batch, part = item / a.batch;
      const Kv8Sequence s = sequence(b);
      const int first = s.bad ? 0 : s.count;
      const uint32_t fill = s.bad ? 0x7fff7fffu : 0u;
      const int64_t values = static_cast<int64_t>(a.heads) * D / 8, n = (a.tokens - first) * values;
      uint4* const o = reinterpret_cast<uint4*>(a.out) + (static_cast<int64_t>(b) * a.tokens + first) * values;
      for (int64_t i = part * (kKv8Warps * 32) + tid; i < n; i += parts * (kKv8Warps * 32)) o[i] = make_uint4(fill, fill, fill, fill);
    }
  }
  // Units of a CTA: at least a step for each warp, so that short contexts are not cut
  // into crumbs; and where few long tiles are left to all CTAs, not so few that joining
  // a tile's n parts takes longer than reading its units / n (their sum is least at
  // n ~ sqrt(units); by the mean tile: 32768 tokens of one kv head 31.6 -> 16.4 us).
  const float mean_units = __fdividef(static_cast<float>(total), fmaxf(1.f, static_cast<float>(tiles)));
  const float least_units = fmaxf(kKv8Warps, kKv8JoinShare * __fsqrt_rn(mean_units));
  const unsigned ctas = min(static_cast<unsigned>(__fdividef(static_cast<float>(total), least_units)) + (total != 0), gridDim.x);
  if (blockIdx.x >= ctas) return;
  Kv8Ranges ranges;
  ranges.each = total / ctas;
  ranges.more = total - ranges.each * ctas;
  const unsigned lo = ranges.begin(blockIdx.x), hi = ranges.begin(blockIdx.x + 1);
  if (lo >= before && lo < before + mine) {
    unsigned offset = before;
    int b = tid * chunk;
    for (;; ++b) {
      const unsigned n = sequence(b).units;
      if (lo < offset + n) break;
      offset += n;
    }
    found_b = b;
    found_offset = offset;
  }
  __syncthreads();

  int b = found_b;
  unsigned offset = found_offset;  // of sequence b in the line
  Kv8Sequence seq = sequence(b);
  uint8_t* const ring = smem + warp * S::STAGES * S::STAGE;
  unsigned cur = lo;
  bool first_piece = true;
  while (cur < hi) {
    while (cur >= offset + seq.units) {
      offset += seq.units;
      seq = sequence(++b);
    }
    const unsigned cost = seq.cost;
    const int tile = static_cast<int>((cur - offset) / cost);
    const unsigned tile_begin = offset + tile * cost;
    // a tile's units are its fixed cost, then its steps
    const int from_unit = static_cast<int>(cur - tile_begin);
    const int to_unit = static_cast<int>(min(cost, hi - tile_begin));
    const int step0 = max(0, from_unit - kKv8TileCost);
    const int step1 = max(0, to_unit - kKv8TileCost);
    cur = tile_begin + to_unit;
    const int which = first_piece ? 0 : 1;
    if (step1 <= step0) continue;  // the range ends within the fixed cost: nothing to do here
    first_piece = false;

    const int head = tile % a.cache.kv_heads;
    const int row0 = tile / a.cache.kv_heads * S::ROWS;
    const int full = seq.total / kKv8Block;
    const int open = seq.total - full * kKv8Block;
    const int start = seq.total - seq.count;
    const int mine_steps = max(0, (step1 - step0 - warp + kKv8Warps - 1) / kKv8Warps);

    // ---- queries: lane (g, t) has dims of row g of each row group, as B fragments.
    // Their loads go out first, to wait together with the page numbers'.
    uint2 q_bits[NR][S::KSTEPS];
    int my_limit[NR];
    int least = 0x7fffffff;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int row = row0 + r * 8 + g;
      const int token = a.tokens == 1 ? row >= a.group : row / a.group;
      const bool real = token < seq.count;
      my_limit[r] = real ? start + token : -1;
      if (real) least = min(least, my_limit[r]);
      const __nv_bfloat16* src = a.q + static_cast<int64_t>(b) * a.q_batch_stride + token * a.q_token_stride +
                                 (head * a.group + row - token * a.group) * D + t4 * S::KB;
#pragma unroll
      for (int k = 0; k < S::KSTEPS; ++k) {
        q_bits[r][k] = make_uint2(0u, 0u);
        if (real) q_bits[r][k] = *reinterpret_cast<const uint2*>(src + k / (S::KB / 4) * 64 + 4 * (k % (S::KB / 4)));
      }
    }

    // ---- this warp's copies.  Step k of the warp is step step0 + warp + 4 k.
    const int coded_steps = full * (kKv8Block / S::TOK);
    int pages = 0;  // lane i: the page of step (k & ~31) + i of the warp
    auto issue = [&](int k) {
      if (k < mine_steps) {
        if ((k & 31) == 0) {
          const int step = step0 + warp + kKv8Warps * (k + lane);
          pages = step < coded_steps && k + lane < mine_steps ? kv8_page(a.cache, seq.slot, step / (kKv8Block / S::TOK)) : 0;
        }
        const int step = step0 + warp + kKv8Warps * k;
        int page = __shfl_sync(0xffffffffu, pages, k & 31);
        const uint32_t stage = smem_u32(ring + (k % S::STAGES) * S::STAGE);
        constexpr int COPIES = S::HALF / 512;  // of 16 bytes a lane
        if (step < coded_steps) {
          const bool known = page >= 0;
          page = max(page, 0);  // page 0 is always there
          const int64_t at = static_cast<int64_t>(page) * 2 * a.cache.kv_heads + head;
          const uint8_t* kp = a.cache.codes + at * kKv8Block * D + step % (kKv8Block / S::TOK) * S::HALF + lane * 16;
          const uint8_t* vp = kp + static_cast<int64_t>(a.cache.kv_heads) * kKv8Block * D;
#pragma unroll
          for (int x = 0; x < COPIES; ++x) cp_async<16>(stage + kv8_k_place<D>(lane * 16) + x * 512, kp + x * 512);
#pragma unroll
          for (int x = 0; x < COPIES; ++x)
            cp_async<16>(stage + S::HALF + (kv8_v_place<D>(lane * 16) ^ (kv8_v_place<D>(x * 512) & 511u)) + x * 512, vp + x * 512);
          if (lane < 2) {
            // a block whose page is not in the table counts as one whose scales are NaN
            if (known) {
              cp_async<4>(stage + 2 * S::HALF + 4 * lane, a.cache.scales + at + lane * a.cache.kv_heads);
            } else {
              *reinterpret_cast<float*>(ring + (k % S::STAGES) * S::STAGE + 2 * S::HALF + 4 * lane) = nan;
            }
          }
        } else {
          const int first = (step - coded_steps) * S::TAIL;
          const __nv_bfloat16* kp = kv8_tail(a.cache, seq.slot, full & 1, 0, head, D) + first * D + lane * 8;
          const __nv_bfloat16* vp = kv8_tail(a.cache, seq.slot, full & 1, 1, head, D) + first * D + lane * 8;
#pragma unroll
          for (int x = 0; x < COPIES; ++x) {
            const bool take = first + (x * 256 + lane * 8) / D < open;
            cp_async_or_zero(stage + (kv8_tail_k_place<D>(lane * 16) ^ (kv8_tail_k_place<D>(x * 512) & 511u)) + x * 512,
                             kp + x * 256, take);
            cp_async_or_zero(stage + S::HALF + (kv8_tail_v_place<D>(lane * 16) ^ (kv8_tail_v_place<D>(x * 512) & 511u)) + x * 512,
                             vp + x * 256, take);
          }
        }
      }
      cp_async_commit();
    };
#pragma unroll 1  // straight-line code that runs once costs its fetch
    for (int k = 0; k < S::STAGES - 1; ++k) issue(k);

    uint32_t qf[NR][S::KSTEPS][2];
    // of rows 2 t and 2 t + 1 of each group, the columns of the accumulators:
    float row_scale[NR][2];  // turns a sum of products into a log2 score
    float q_start[NR][2];    // where the sum starts, -128 2^-24 times the sum of the queries
    int limit[NR][2];        // the row's own position: the last key that it sees
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const uint2(&x)[S::KSTEPS] = q_bits[r];
      uint32_t peak_bits = 0;
#pragma unroll
      for (int k = 0; k < S::KSTEPS; ++k)
        peak_bits = max(peak_bits, max(max((x[k].x << 16) & 0x7fff0000u, x[k].x & 0x7fff0000u),
                                       max((x[k].y << 16) & 0x7fff0000u, x[k].y & 0x7fff0000u)));
      peak_bits = max(peak_bits, __shfl_xor_sync(0xffffffffu, peak_bits, 1));
      peak_bits = max(peak_bits, __shfl_xor_sync(0xffffffffu, peak_bits, 2));
      const bool finite = peak_bits < 0x7f800000u;
      // 2^e <= peak < 2^(e+1), clamped so that 2^e and 2^-e are normal numbers
      const int e = min(126, max(-100, static_cast<int>(peak_bits >> 23) - 127));
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      float start_sum[4];
#pragma unroll
      for (int k = 0; k < S::KSTEPS; ++k) {
        const float y0 = __uint_as_float(x[k].x << 16), y1 = __uint_as_float(x[k].x & 0xffff0000u);
        const float y2 = __uint_as_float(x[k].y << 16), y3 = __uint_as_float(x[k].y & 0xffff0000u);
        qf[r][k][0] = finite ? pack_f16x2(y0 * down, y2 * down) : 0u;
        qf[r][k][1] = finite ? pack_f16x2(y1 * down, y3 * down) : 0u;
        const uint32_t offset[4] = {kKv8OffsetF16, kKv8OffsetF16, kKv8OffsetF16, kKv8OffsetF16};
        if (k == 0) {
          mma_m16n8k16_f16_from(start_sum, offset, qf[r][k][0], qf[r][k][1], 0.f, 0.f);
        } else {
          mma_m16n8k16_f16(start_sum, offset, qf[r][k][0], qf[r][k][1]);
        }
      }
      const float my_scale = finite ? up * a.scale_log2 : nan;
#pragma unroll
      for (int e2 = 0; e2 < 2; ++e2) {
        const int from = (2 * t4 + e2) * 4;
        row_scale[r][e2] = __shfl_sync(0xffffffffu, my_scale, from);
        limit[r][e2] = __shfl_sync(0xffffffffu, my_limit[r], from);
        q_start[r][e2] = start_sum[e2];
      }
    }
    least = __reduce_min_sync(0xffffffffu, least);

    float o[NR][S::MT][4];
    float m[NR][2], l[NR][2];  // the rows' bases and sums
#pragma unroll
    for (int r = 0; r < NR; ++r) {
#pragma unroll
      for (int j = 0; j < S::MT; ++j) o[r][j][0] = o[r][j][1] = o[r][j][2] = o[r][j][3] = 0.f;
      m[r][0] = m[r][1] = minus_inf;
      l[r][0] = l[r][1] = 0.f;
    }

    // Sums s (tokens 16 i + g and + 8, rows 2 t and 2 t + 1) to probabilities 2^(s factor - m).
    auto softmax = [&](auto& s, float (&factor)[NR][2], int first_token, bool masked, bool half) {
      constexpr int TILES = sizeof(s) / sizeof(s[0]);
      float top[NR][2];
      bool above = false;
#pragma unroll
      for (int r = 0; r < NR; ++r) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float t = minus_inf;
          // never 0, so that a masked -inf stays -inf (a block of zeros has scale 0)
          factor[r][e] = factor[r][e] == 0.f ? 1e-30f : factor[r][e];
          if (masked) {
            if (first_token > limit[r][e]) factor[r][e] = 1e-30f;  // sees none: a NaN scale is not its own
#pragma unroll
            for (int i = 0; i < TILES; ++i) {
#pragma unroll
              for (int h = 0; h < 2; ++h)
                if (first_token + i * 16 + h * 8 + g > limit[r][e] || (half && h == 1)) s[i][r][2 * h + e] = minus_inf;
            }
          }
#pragma unroll
          for (int i = 0; i < TILES; ++i) t = max3(t, s[i][r][e], s[i][r][2 + e]);
          top[r][e] = t * factor[r][e];
          above = above || top[r][e] > m[r][e] + kKv8Headroom;
        }
      }
      if (__any_sync(0xffffffffu, above)) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float next = fmaxf(top[r][e], __shfl_xor_sync(0xffffffffu, top[r][e], 4));
            next = fmaxf(next, __shfl_xor_sync(0xffffffffu, next, 8));
            next = fmaxf(fmaxf(next, __shfl_xor_sync(0xffffffffu, next, 16)) - kKv8Under, m[r][e]);
            const float by = m[r][e] == minus_inf ? 0.f : fast_exp2(m[r][e] - next);
            m[r][e] = next;
            l[r][e] *= by;
#pragma unroll
            for (int j = 0; j < S::MT; ++j) {
              o[r][j][e] *= by;
              o[r][j][2 + e] *= by;
            }
          }
        }
      }
#pragma unroll
      for (int r = 0; r < NR; ++r) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float from = m[r][e] == minus_inf ? 0.f : m[r][e];
#pragma unroll
          for (int i = 0; i < TILES; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              s[i][r][2 * h + e] = fast_exp2(fmaf(s[i][r][2 * h + e], factor[r][e], -from));
          }
        }
      }
    };

    // a lane's place in a step: the parts of its fragments that do not depend on the step
    const uint32_t k_at = kv8_k_place<D>(g * D + t4 * S::KB), v_at = kv8_v_place<D>(2 * t4 * D + g * S::VB);
    const uint32_t tail_k_at = kv8_tail_k_place<D>(g * 2 * D + t4 * 2 * S::KB);
    const uint32_t tail_v_at = kv8_tail_v_place<D>(2 * t4 * 2 * D + g * 2 * S::VB);
#pragma unroll 1
    for (int k = 0; k < mine_steps; ++k) {
      cp_async_wait<S::STAGES - 2>();
      __syncwarp();
      issue(k + S::STAGES - 1);
      const int step = step0 + warp + kKv8Warps * k;
      uint8_t* stage = ring + (k % S::STAGES) * S::STAGE;
      if (step < coded_steps) {
        const int first_token = step * S::TOK;
        const float2 scales = *reinterpret_cast<const float2*>(stage + 2 * S::HALF);
        float s[S::T16][NR][4];
#pragma unroll
        for (int c = 0; c < S::KC; ++c) {
          uint32_t w[2 * S::T16][S::KB / 4];
#pragma unroll
          for (int n = 0; n < 2 * S::T16; ++n) lds_words<S::KB>(stage + (k_at ^ (c * 64)) + n * 8 * D, w[n]);
#pragma unroll
          for (int i = 0; i < S::KB / 4; ++i) {
            const int ks = c * (S::KB / 4) + i;
#pragma unroll
            for (int t = 0; t < S::T16; ++t) {
              const uint32_t kf[4] = {codes_even(w[2 * t][i]), codes_even(w[2 * t + 1][i]), codes_odd(w[2 * t][i]),
                                      codes_odd(w[2 * t + 1][i])};
#pragma unroll
              for (int r = 0; r < NR; ++r) {
                if (ks == 0) {
                  mma_m16n8k16_f16_from(s[t][r], kf, qf[r][0][0], qf[r][0][1], q_start[r][0], q_start[r][1]);
                } else {
                  mma_m16n8k16_f16(s[t][r], kf, qf[r][ks][0], qf[r][ks][1]);
                }
              }
            }
          }
        }
        const bool masked = first_token + S::TOK - 1 > least;
        float factor[NR][2];
        const float k_unit = scales.x * kKv8Unit, v_unit = scales.y * kKv8Unit;
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          factor[r][0] = row_scale[r][0] * k_unit;
          factor[r][1] = row_scale[r][1] * k_unit;
        }
        softmax(s, factor, first_token, masked, false);
        uint32_t p[S::T16][NR][2];
        float v_start[NR][2], v_scale[NR][2];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          float sum[4];
          const uint32_t offset[4] = {kKv8OffsetF16, kKv8OffsetF16, kKv8OffsetF16, kKv8OffsetF16};
#pragma unroll
          for (int t = 0; t < S::T16; ++t) {
            p[t][r][0] = transpose_8x8(pack_f16x2(s[t][r][0], s[t][r][1]));
            p[t][r][1] = transpose_8x8(pack_f16x2(s[t][r][2], s[t][r][3]));
            if (t == 0) {
              mma_m16n8k16_f16_from(sum, offset, p[0][r][0], p[0][r][1], 0.f, 0.f);
            } else {
              mma_m16n8k16_f16(sum, offset, p[t][r][0], p[t][r][1]);
            }
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            l[r][e] += sum[e];
            v_start[r][e] = sum[e];
            // a row that sees none of these keys takes nothing of them, whatever the scale
            v_scale[r][e] = masked && first_token > limit[r][e] ? 0.f : v_unit;
          }
        }
#pragma unroll
        for (int c = 0; c < S::VC; ++c) {
          uint32_t w[4 * S::T16][S::VB / 4];
#pragma unroll
          for (int i = 0; i < 4 * S::T16; ++i) {  // tokens 16 (i / 4) + {2t, 2t + 1, 2t + 8, 2t + 9}
            const uint32_t at = D <= 64 ? v_at ^ ((i & 1) * D) : v_at + (i & 1) * D;
            lds_words<S::VB>(stage + S::HALF + at + ((i / 4) * 16 + (i >> 1 & 1) * 8) * D + c * 128, w[i]);
          }
#pragma unroll
          for (int i = 0; i < S::VB / 4; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // dims 4 i + 2 h and + 1 of the lane's bytes
              float acc[NR][4];
#pragma unroll
              for (int t = 0; t < S::T16; ++t) {
                // two tokens' bytes of two dims each, then the tokens' pairs per dim
                const uint32_t ab = __byte_perm(w[4 * t][i], w[4 * t + 1][i], h ? 0x7632 : 0x5410);
                const uint32_t cd = __byte_perm(w[4 * t + 2][i], w[4 * t + 3][i], h ? 0x7632 : 0x5410);
                const uint32_t vf[4] = {codes_even(ab), codes_odd(ab), codes_even(cd), codes_odd(cd)};
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                  if (t == 0) {
                    mma_m16n8k16_f16_from(acc[r], vf, p[0][r][0], p[0][r][1], v_start[r][0], v_start[r][1]);
                  } else {
                    mma_m16n8k16_f16(acc[r], vf, p[t][r][0], p[t][r][1]);
                  }
                }
              }
#pragma unroll
              for (int r = 0; r < NR; ++r) {
                float(&dst)[4] = o[r][c * (S::VB / 2) + 2 * i + h];
#pragma unroll
                for (int e = 0; e < 4; ++e) dst[e] = fmaf(v_scale[r][e & 1], acc[r][e], dst[e]);
              }
            }
          }
        }
      } else {
        constexpr int TT = S::TAIL16;  // 16-token groups
        const int first_token = full * kKv8Block + (step - coded_steps) * S::TAIL;
        float s[TT][NR][4];
#pragma unroll
        for (int c = 0; c < 2 * S::KC; ++c) {
          uint32_t w[2 * TT][S::KB / 4];
#pragma unroll
          for (int n = 0; n < S::TAIL / 8; ++n)
            lds_words<S::KB>(stage + (tail_k_at ^ (c % 2 * S::KB)) + c / 2 * 128 + n * 16 * D, w[n]);
#pragma unroll
          for (int i = 0; i < S::KB / 8; ++i) {
            const int ks = c * (S::KB / 8) + i;
            uint32_t qb[NR][2];  // fp16 -> bf16, exact: they came from bf16
#pragma unroll
            for (int r = 0; r < NR; ++r) {
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&qf[r][ks][e]));
                qb[r][e] = pack_bf16x2(v.x, v.y);
              }
            }
#pragma unroll
            for (int t = 0; t < TT; ++t) {
              const uint32_t(&wa)[S::KB / 4] = w[2 * t];
              const uint32_t(&wb)[S::KB / 4] = w[S::TAIL_HALF ? 0 : 2 * t + 1];
              const uint32_t kf[4] = {__byte_perm(wa[2 * i], wa[2 * i + 1], 0x5410),
                                      S::TAIL_HALF ? 0u : __byte_perm(wb[2 * i], wb[2 * i + 1], 0x5410),
                                      __byte_perm(wa[2 * i], wa[2 * i + 1], 0x7632),
                                      S::TAIL_HALF ? 0u : __byte_perm(wb[2 * i], wb[2 * i + 1], 0x7632)};
#pragma unroll
              for (int r = 0; r < NR; ++r) {
                if (ks == 0) s[t][r][0] = s[t][r][1] = s[t][r][2] = s[t][r][3] = 0.f;
                mma_m16n8k16_bf16(s[t][r], kf, qb[r][0], qb[r][1]);
              }
            }
          }
        }
        float factor[NR][2];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          factor[r][0] = row_scale[r][0];
          factor[r][1] = row_scale[r][1];
        }
        softmax(s, factor, first_token, true, S::TAIL_HALF);
        uint32_t high[TT][NR][2], low[TT][NR][2];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const uint32_t offset[4] = {kKv8OffsetBf16, kKv8OffsetBf16, kKv8OffsetBf16, kKv8OffsetBf16};
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int t = 0; t < TT; ++t) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float x = s[t][r][2 * h], y = s[t][r][2 * h + 1];
              const uint32_t hi2 = pack_bf16x2(x, y);
              const uint32_t lo2 = pack_bf16x2(x - __uint_as_float(hi2 << 16), y - __uint_as_float(hi2 & 0xffff0000u));
              high[t][r][h] = transpose_8x8(hi2);
              low[t][r][h] = transpose_8x8(lo2);
            }
            mma_m16n8k16_bf16(sum, offset, high[t][r][0], high[t][r][1]);
            mma_m16n8k16_bf16(sum, offset, low[t][r][0], low[t][r][1]);
          }
          l[r][0] += sum[0];
          l[r][1] += sum[1];
        }
        // Values that are not finite, and rows that must not see them: 0 x inf
        // would be NaN, so such a step goes value by value.
        bool odd = false;
        if (seq.count > 1 && first_token + S::TAIL - 1 > least) {
#pragma unroll
          for (int i = 0; i < S::HALF / 512; ++i) {
            uint32_t w[4];
            lds_words<16>(stage + S::HALF + i * 512 + lane * 16, w);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              odd = odd || (w[e] & 0x7f80u) == 0x7f80u || (w[e] & 0x7f800000u) == 0x7f800000u;
          }
          odd = __any_sync(0xffffffffu, odd);
        }
        if (!odd) {
#pragma unroll
          for (int c = 0; c < S::VC; ++c) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t w[4 * TT][S::VB / 4];
#pragma unroll
              for (int i = 0; i < S::TAIL / 4; ++i)
                lds_words<S::VB>(stage + S::HALF + (tail_v_at ^ (h * S::VB)) + c * 256 +
                                     ((i / 4) * 16 + (i & 1) + (i >> 1 & 1) * 8) * 2 * D, w[i]);
#pragma unroll
              for (int i = 0; i < S::VB / 4; ++i) {
#pragma unroll
                for (int t = 0; t < TT; ++t) {
                  constexpr int C = S::TAIL_HALF ? 0 : 2;
                  const uint32_t vf[4] = {
                      __byte_perm(w[4 * t][i], w[4 * t + 1][i], 0x5410), __byte_perm(w[4 * t][i], w[4 * t + 1][i], 0x7632),
                      S::TAIL_HALF ? 0u : __byte_perm(w[4 * t + C][i], w[4 * t + C + 1][i], 0x5410),
                      S::TAIL_HALF ? 0u : __byte_perm(w[4 * t + C][i], w[4 * t + C + 1][i], 0x7632)};
#pragma unroll
                  for (int r = 0; r < NR; ++r) {
                    float(&dst)[4] = o[r][c * (S::VB / 2) + h * (S::VB / 4) + i];
                    mma_m16n8k16_bf16(dst, vf, high[t][r][0], high[t][r][1]);
                    mma_m16n8k16_bf16(dst, vf, low[t][r][0], low[t][r][1]);
                  }
                }
              }
            }
          }
        } else {
          // 16 tokens of a row group's probabilities at a time, over the step's keys, which are used up
          float* pr = reinterpret_cast<float*>(stage);
#pragma unroll
          for (int rt = 0; rt < NR * TT; ++rt) {
            const int r = rt / TT, t = rt % TT;
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 4; ++e) pr[(2 * t4 + (e & 1)) * 16 + g + 8 * (e >> 1)] = s[t][r][e];
            __syncwarp();
#pragma unroll 1
            for (int token = 0; token < (S::TAIL_HALF ? 8 : 16); ++token) {
              const int where = first_token + 16 * t + token;
#pragma unroll
              for (int j = 0; j < S::MT; ++j) {
                const int c = j / (S::VB / 2), h = j % (S::VB / 2) / (S::VB / 4), at = j % (S::VB / 4);
                const uint32_t two = *reinterpret_cast<const uint32_t*>(
                    stage + S::HALF + kv8_tail_v_place<D>((16 * t + token) * 2 * D + (c * 128 + g * S::VB) * 2 + h * S::VB + 4 * at));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float v = __uint_as_float(e < 2 ? two << 16 : two & 0xffff0000u);
                  if (where <= limit[r][e & 1]) o[r][j][e] = fmaf(pr[(2 * t4 + (e & 1)) * 16 + token], v, o[r][j][e]);
                }
              }
            }
          }
          __syncwarp();
        }
      }
    }
    cp_async_wait<0>();

    // ---- join the warps: fragments [warp][r, j][lane], a share of them for each warp
    if (g == 0) {
#pragma unroll
      for (int r = 0; r < NR; ++r) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          warp_ml[warp][r * 8 + 2 * t4 + e] = make_float2(m[r][e], l[r][e] * kKv8SumUnit);
      }
    }
    __syncthreads();  // everyone is done with the ring
    float4* const join = reinterpret_cast<float4*>(smem);
#pragma unroll
    for (int r = 0; r < NR; ++r) {
#pragma unroll
      for (int j = 0; j < S::MT; ++j)
        join[(warp * S::FRAGS + r * S::MT + j) * 32 + lane] = make_float4(o[r][j][0], o[r][j][1], o[r][j][2], o[r][j][3]);
    }
    __syncthreads();
    const int frag0 = warp * S::SHARE;
    const bool has_share = frag0 < S::FRAGS;
    // the maximum and the sum of one row over n (max, sum) pairs, the pairs' weights
    auto weigh = [&](const float2 (&ml)[kKv8Warps], float (&weight)[kKv8Warps]) {
      float top = minus_inf, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kKv8Warps; ++w) top = fmaxf(top, ml[w].x);
      const float from = top == minus_inf ? 0.f : top;
#pragma unroll
      for (int w = 0; w < kKv8Warps; ++w) {
        weight[w] = fast_exp2(ml[w].x - from);
        sum = fmaf(weight[w], ml[w].y, sum);
      }
      return make_float2(top, sum);
    };
    // a warp's share lies in one row group
    const int share_rows = frag0 / S::MT;
    float4 acc[S::SHARE];
    float2 ml_out[2] = {};
    if (has_share) {
      float weight[2][kKv8Warps];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float2 ml[kKv8Warps];
#pragma unroll
        for (int w = 0; w < kKv8Warps; ++w) ml[w] = warp_ml[w][share_rows * 8 + 2 * t4 + e];
        ml_out[e] = weigh(ml, weight[e]);
      }
#pragma unroll
      for (int i = 0; i < S::SHARE; ++i) {
        acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kKv8Warps; ++w) {
          const float4 v = join[(w * S::FRAGS + frag0 + i) * 32 + lane];
          acc[i].x = fmaf(weight[0][w], v.x, acc[i].x);
          acc[i].y = fmaf(weight[1][w], v.y, acc[i].y);
          acc[i].z = fmaf(weight[0][w], v.z, acc[i].z);
          acc[i].w = fmaf(weight[1][w], v.w, acc[i].w);
        }
      }
    }

    // ---- a tile in several CTAs: leave the part, the last to arrive joins them
    bool write = step0 == 0 && step1 == seq.steps;
    if (!write) {
      const unsigned c0 = ranges.of(tile_begin + kKv8TileCost);
      const unsigned c1 = ranges.of(tile_begin + cost - 1);
      const int n_parts = static_cast<int>(c1 - c0) + 1;
      float* part = a.parts + (static_cast<int64_t>(blockIdx.x) * 2 + which) * S::PART_FLOATS;
      if (has_share) {
#pragma unroll
        for (int i = 0; i < S::SHARE; ++i) __stcg(reinterpret_cast<float4*>(part) + (frag0 + i) * 32 + lane, acc[i]);
        if (frag0 % S::MT == 0 && g == 0)
          __stcg(reinterpret_cast<float4*>(part + S::ROWS * D) + share_rows * 4 + t4,
                 make_float4(ml_out[0].x, ml_out[0].y, ml_out[1].x, ml_out[1].y));
      }
      __syncthreads();
      if (tid == 0) {
        // releases the CTA's part (ordered before by the barrier), acquires the others'
        unsigned int had;
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(had) : "l"(a.arrivals + c0) : "memory");
        is_last = had + 1 == static_cast<unsigned int>(n_parts);
        if (is_last) a.arrivals[c0] = 0;  // ready for the next launch
      }
      __syncthreads();
      write = is_last;
      if (write && has_share) {
        // The parts in the order of the ranges, kAhead at a time with all loads
        // in flight: the latency of L2 is what this costs.
        constexpr int kAhead = S::SHARE == 1 ? 16 : S::SHARE == 2 ? 12 : 8;
        // in the tile's first CTA it is the second part if the range begins before the tile
        const float* first_part = a.parts + (static_cast<int64_t>(c0) * 2 + (ranges.begin(c0) < tile_begin ? 1 : 0)) * S::PART_FLOATS;
        const float* next_part = a.parts + static_cast<int64_t>(c0) * 2 * S::PART_FLOATS;
        float top[2] = {minus_inf, minus_inf}, sum[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < S::SHARE; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int n0 = 0; n0 < n_parts; n0 += kAhead) {
          float4 v[kAhead][S::SHARE], ml[kAhead];  // ml: (max, sum) of rows 2 t and 2 t + 1
#pragma unroll
          for (int n = 0; n < kAhead; ++n) {
            const float* part_n = n0 + n == 0 ? first_part : next_part + static_cast<int64_t>(n0 + n) * 2 * S::PART_FLOATS;
            ml[n] = make_float4(minus_inf, 0.f, minus_inf, 0.f);
            if (n0 + n < n_parts) ml[n] = __ldcg(reinterpret_cast<const float4*>(part_n + S::ROWS * D) + share_rows * 4 + t4);
#pragma unroll
            for (int i = 0; i < S::SHARE; ++i) {
              v[n][i] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (n0 + n < n_parts) v[n][i] = __ldcg(reinterpret_cast<const float4*>(part_n) + (frag0 + i) * 32 + lane);
            }
          }
          float next[2] = {top[0], top[1]}, from[2], by[2];
#pragma unroll
          for (int n = 0; n < kAhead; ++n) {
            next[0] = fmaxf(next[0], ml[n].x);
            next[1] = fmaxf(next[1], ml[n].z);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            from[e] = next[e] == minus_inf ? 0.f : next[e];
            by[e] = fast_exp2(top[e] - from[e]);
            top[e] = next[e];
            sum[e] *= by[e];
          }
#pragma unroll
          for (int i = 0; i < S::SHARE; ++i) acc[i] = make_float4(acc[i].x * by[0], acc[i].y * by[1], acc[i].z * by[0], acc[i].w * by[1]);
#pragma unroll
          for (int n = 0; n < kAhead; ++n) {
            const float w0 = fast_exp2(ml[n].x - from[0]), w1 = fast_exp2(ml[n].z - from[1]);
            sum[0] = fmaf(w0, ml[n].y, sum[0]);
            sum[1] = fmaf(w1, ml[n].w, sum[1]);
#pragma unroll
            for (int i = 0; i < S::SHARE; ++i) {
              acc[i].x = fmaf(w0, v[n][i].x, acc[i].x);
              acc[i].y = fmaf(w1, v[n][i].y, acc[i].y);
              acc[i].z = fmaf(w0, v[n][i].z, acc[i].z);
              acc[i].w = fmaf(w1, v[n][i].w, acc[i].w);
            }
          }
        }
        ml_out[0].y = sum[0];
        ml_out[1].y = sum[1];
      }
    }
    if (write && has_share) {
#pragma unroll
      for (int i = 0; i < S::SHARE; ++i) {
        const int j = (frag0 + i) % S::MT;
        // fragment j has bytes 2 j' and 2 j' + 1 of copy c of lane g
        const int d = j / (S::VB / 2) * 128 + g * S::VB + j % (S::VB / 2) * 2;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = row0 + share_rows * 8 + 2 * t4 + e;
          const int token = row / a.group;
          if (token >= seq.count) continue;
          // A row sees its own key at least, so that its sum is zero only where all its scores
          // are -infinity: 0 / 0, as softmax has it.
          const float by = 1.f / ml_out[e].y;
          const uint32_t two = pack_bf16x2((e ? acc[i].y : acc[i].x) * by, (e ? acc[i].w : acc[i].z) * by);
          *reinterpret_cast<uint32_t*>(a.out + ((static_cast<int64_t>(b) * a.tokens + token) * a.heads + head * a.group +
                                                row % a.group) * D + d) = two;
        }
      }
    }
    __syncthreads();  // the ring and the shared rows are free again
  }
}

}  // namespace b200tx
