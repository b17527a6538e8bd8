// kv8_cache_kernels.cuh -- the paged key/value cache held in 8 bits: appending
// tokens and reading values back.
//
// A sequence's tokens lie in blocks of 64.  A block that is full is held as
// 8-bit codes with one fp32 scale per kv head, for keys and for values:
//     scale = max |x| / 127 over the block's 64 x D values of the head
//     code  = rint(x / scale) + 128,           x ~ (code - 128) * scale
// The block that is still open is held in bf16 in the sequence's tail.  Its
// scale is only known when its last token arrives; with the open block in 16
// bits nothing is ever quantised twice, and a prompt appended at once gives
// the same bits as the same tokens one at a time.  Keys and values are
// rounded to bf16 when they enter, whichever way they take.
//
// The offset of 128 keeps a code positive: under a zero byte it is an fp16
// number as it stands, two to an instruction, and the attention takes the
// offset out of its sums.
//
// What bounds them: HBM, each value read and written once, and beside it the latency of the
// loads.  An append of 4 x 4000 tokens (32 + 2 x 8 heads of 128) moves 360 MB in 85 us, 4.3
// TB/s, with 22 of 64 warps on an SM (80 registers a thread); schedulers issue in 61 % of
// cycles, and a warp waits three cycles for loads to one in which it issues.  The read-back
// of its values moves 98 MB in 20 us, 4.9 TB/s.
//
// The tail has two slots, taken by the parity of the block index.  A call of
// up to 64 tokens touches two blocks at most, and leaves both in their slots;
// a caller may therefore keep any number of the tokens that it appended last
// (drafted tokens, say) by the length that it sets afterwards.
//
// A block with a value that is not finite gets the scale NaN: whoever attends
// to it sees NaN rather than a plausible number.
#pragma once

#include "rope_kernels.cuh"

namespace b200tx {

constexpr int kKv8Block = 64;

// A slot is that of one sequence of a call at most.
struct Kv8Cache {
  uint8_t* codes;           // [pages, 2, kv_heads, 64, D]
  float* scales;            // [pages, 2, kv_heads]
  __nv_bfloat16* tail;      // [slots, 2 (block parity), 2, kv_heads, 64, D]
  const int32_t* page_table;  // [slots, max_blocks]
  const int32_t* lengths;     // [slots]
  int64_t pages;
  int slots, max_blocks, kv_heads;
};

__device__ __forceinline__ __nv_bfloat16* kv8_tail(const Kv8Cache& c, int slot, int parity, int kv, int head, int dim) {
  const int64_t at = ((static_cast<int64_t>(slot) * 2 + parity) * 2 + kv) * c.kv_heads + head;
  return c.tail + at * kKv8Block * dim;
}

// The page of a block, or -1 where the table does not hold it.
__device__ __forceinline__ int kv8_page(const Kv8Cache& c, int slot, int block) {
  if (block < 0 || block >= c.max_blocks) return -1;
  const int page = __ldg(c.page_table + static_cast<int64_t>(slot) * c.max_blocks + block);
  return page >= 0 && page < c.pages ? page : -1;
}

struct Kv8AppendArgs {
  Kv8Cache cache;
  const void* qkv;
  __nv_bfloat16* q_out;  // [batch, tokens, heads, D]
  int64_t batch_stride, token_stride;  // elements of qkv
  const int32_t* slot_ids;             // [batch] or null = identity
  const int32_t* counts;               // [batch] new tokens, or null = tokens
  int batch, tokens, heads;
  int block_span;                      // blocks a sequence's new tokens can touch
  int64_t kv_ctas;                     // batch * kv_heads * block_span
  int chunks;                          // query part: as in RopeArgs
  QkNormArgs norm;
};

constexpr int kKv8AppendWarps = 8;
constexpr float kKv8Tiny = 5.421010862427522e-20f;    // 2^-64
constexpr float kKv8Raise = 7.922816251426434e+28f;  // 2^96

// One block of one kv head: its new tokens normed, rotated and stored, and the
// block quantised if it is full now.
template <int D, int E, typename T>
__device__ __forceinline__ void kv8_append_block(const Kv8AppendArgs& a, int b, int slot, int head, int block, int start,
                                                 int count, uint32_t (*peak)[kKv8AppendWarps]) {
  using Lanes = HeadLanes<D, E>;
  constexpr int L = Lanes::L;
  constexpr int TOKENS = Lanes::HEADS;                      // per warp and pass
  constexpr int PASS = kKv8AppendWarps * TOKENS;            // tokens per pass
  constexpr int PASSES = (kKv8Block + PASS - 1) / PASS;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, in_head = lane % L;
  const int first = block * kKv8Block;
  const int end = start + count;
  const bool full = first + kKv8Block <= end;
  const bool keep = !full || a.tokens <= kKv8Block;
  const T* src = static_cast<const T*>(a.qkv) + b * a.batch_stride + (a.heads + head) * D + in_head * E;
  __nv_bfloat16* const tail_k = kv8_tail(a.cache, slot, block & 1, 0, head, D) + in_head * E;
  __nv_bfloat16* const tail_v = kv8_tail(a.cache, slot, block & 1, 1, head, D) + in_head * E;
  const int partner = partner_lane<D, E>(a.norm.rope, lane);

  uint32_t k_bits[PASSES][E / 2], v_bits[PASSES][E / 2];  // bf16 pairs
  // every pass's loads go out before the first is used
  Raw<T, E> k_raw[PASSES], v_raw[PASSES];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int in_block = p * PASS + warp * TOKENS + lane / L;
    const int token = first + in_block;
    k_raw[p].zero();
    v_raw[p].zero();
    if (in_block < kKv8Block && token >= start && token < end) {
      k_raw[p].load(src + (token - start) * a.token_stride);
      v_raw[p].load(src + (token - start) * a.token_stride + a.cache.kv_heads * D);
    }
  }
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int in_block = p * PASS + warp * TOKENS + lane / L;
    const int token = first + in_block;
    const bool fresh = in_block < kKv8Block && token >= start && token < end;
    Raw<__nv_bfloat16, E> k, v;
    k.zero();
    v.zero();
    if (__any_sync(0xffffffffu, fresh)) {
      LaneAngles<D, E> angles;
      angles.load(a.norm.rope, fresh ? token : 0, in_head);
      LaneFactors<D, E> f;
      f.set(a.norm.k_weight, angles, a.norm.rope, lane);
      float y[E];
      norm_rotate<D, E, T>(k_raw[p], y, f, a.norm.k_weight != nullptr, a.norm.eps, angles.turned, a.norm.rope, partner);
      k.set(y);
      if constexpr (sizeof(T) == 2) {
        v = v_raw[p];
      } else {
        float x[E];
        v_raw[p].values(x);
        v.set(x);
      }
    }
    if (fresh && keep) {
      k.store(tail_k + in_block * D);
      v.store(tail_v + in_block * D);
    } else if (!fresh && full && in_block < kKv8Block && token < start) {
      k.load(tail_k + in_block * D);
      v.load(tail_v + in_block * D);
    }
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      k_bits[p][i] = k.w[i];
      v_bits[p][i] = v.w[i];
    }
  }
  if (!full) return;

  // The largest magnitude as a bit pattern, two bf16 at a time: the order of
  // non-negative floats, with infinity and then NaN above every finite value.
  uint32_t k_two = 0, v_two = 0;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      k_two = __vmaxu2(k_two, k_bits[p][i] & 0x7fff7fffu);
      v_two = __vmaxu2(v_two, v_bits[p][i] & 0x7fff7fffu);
    }
  }
  uint32_t k_max = __reduce_max_sync(0xffffffffu, max(k_two << 16, k_two & 0xffff0000u));
  uint32_t v_max = __reduce_max_sync(0xffffffffu, max(v_two << 16, v_two & 0xffff0000u));
  __syncthreads();  // a block before this one may still read peak
  if (lane == 0) {
    peak[0][warp] = k_max;
    peak[1][warp] = v_max;
  }
  __syncthreads();
  const int page = kv8_page(a.cache, slot, block);
  if (page < 0) return;
#pragma unroll
  for (int i = 0; i < kKv8AppendWarps; ++i) {
    k_max = max(k_max, peak[0][i]);
    v_max = max(v_max, peak[1][i]);
  }
  const float nan = __int_as_float(0x7fffffff);
  const float k_scale = k_max >= 0x7f800000u ? nan : __uint_as_float(k_max) / 127.f;
  const float v_scale = v_max >= 0x7f800000u ? nan : __uint_as_float(v_max) / 127.f;
  const int64_t at = (static_cast<int64_t>(page) * 2) * a.cache.kv_heads + head;
  if (threadIdx.x == 0) {
    a.cache.scales[at] = k_scale;
    a.cache.scales[at + a.cache.kv_heads] = v_scale;
  }
  uint8_t* const k_codes = a.cache.codes + at * kKv8Block * D;
  uint8_t* const v_codes = k_codes + static_cast<int64_t>(a.cache.kv_heads) * kKv8Block * D;
  // Below 2^-64 a block is taken up by 2^96, values and scale alike and exactly, so that the
  // scale is a normal number and its reciprocal a finite one whatever the block's peak is.
  auto raise = [](uint32_t (&bits)[PASSES][E / 2], float scale) {
    if (scale >= kKv8Tiny) return scale;  // NaN is no matter, as below
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
#pragma unroll
      for (int i = 0; i < E / 2; ++i)
        bits[p][i] = pack_bf16x2(__uint_as_float(bits[p][i] << 16) * kKv8Raise,
                                 __uint_as_float(bits[p][i] & 0xffff0000u) * kKv8Raise);
    }
    return scale * kKv8Raise;
  };
  const float k_unit = raise(k_bits, k_scale), v_unit = raise(v_bits, v_scale);
  // scale 0: a block of zeros, codes 128; scale NaN: any code, the scale says it all
  const float k_inv = k_unit > 0.f ? 1.f / k_unit : 0.f, v_inv = v_unit > 0.f ? 1.f / v_unit : 0.f;
  // The quotient x / scale in 32 bits, correctly rounded, by Markstein's method ("Computation
  // of elementary functions on the IBM RISC System/6000 processor", 1990): a first
  // quotient by the rounded reciprocal, and its exact remainder times the reciprocal.
  // A product with the reciprocal alone takes values halfway between two codes, such as
  // half the block's peak, to either side.  Then 1.5 2^23 + 128 + quotient, rounded to an
  // integer by the addition: the low byte is the code.  Two values at a time.
  auto codes = [](uint32_t lo, uint32_t hi, float unit, float inv) -> uint32_t {
    const uint64_t by = f32x2(inv, inv), unit2 = f32x2(-unit, -unit), shift = f32x2(12583040.f, 12583040.f);
    auto two = [&](uint32_t w) {
      const uint64_t x = f32x2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
      const uint64_t near = mul_f32x2(x, by);
      return unpack_f32x2(add_f32x2(fma_f32x2(fma_f32x2(near, unit2, x), by, near), shift));
    };
    const float2 c01 = two(lo), c23 = two(hi);
    return __byte_perm(__byte_perm(__float_as_uint(c01.x), __float_as_uint(c01.y), 0x0040),
                       __byte_perm(__float_as_uint(c23.x), __float_as_uint(c23.y), 0x0040), 0x5410);
  };
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int in_block = p * PASS + warp * TOKENS + lane / L;
    if (in_block >= kKv8Block) continue;
    uint32_t kc[E / 4], vc[E / 4];
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
      kc[i] = codes(k_bits[p][2 * i], k_bits[p][2 * i + 1], k_unit, k_inv);
      vc[i] = codes(v_bits[p][2 * i], v_bits[p][2 * i + 1], v_unit, v_inv);
    }
    uint8_t* const k_to = k_codes + in_block * D + in_head * E;
    uint8_t* const v_to = v_codes + in_block * D + in_head * E;
    if constexpr (E == 8) {
      *reinterpret_cast<uint2*>(k_to) = make_uint2(kc[0], kc[1]);
      *reinterpret_cast<uint2*>(v_to) = make_uint2(vc[0], vc[1]);
    } else {
      *reinterpret_cast<uint32_t*>(k_to) = kc[0];
      *reinterpret_cast<uint32_t*>(v_to) = vc[0];
    }
  }
}

// CTAs below kv_ctas each take one block of one kv head; the rest norm and
// rotate the queries, a warp for a round of a token's heads as in qk_norm_rope_kernel.
template <int D, int E, typename T>
__global__ void __launch_bounds__(kKv8AppendWarps * 32, D == 256 ? 1 : 3) kv8_append_kernel(Kv8AppendArgs a) {
  __shared__ uint32_t peak[2][kKv8AppendWarps];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x % 32;

  if (blockIdx.x < a.kv_ctas) {
    const int64_t item = blockIdx.x / a.cache.kv_heads;
    const int head = static_cast<int>(blockIdx.x - item * a.cache.kv_heads);
    const int b = static_cast<int>(item / a.block_span);
    const int at = static_cast<int>(item - static_cast<int64_t>(b) * a.block_span);
    const int slot = a.slot_ids == nullptr ? b : a.slot_ids[b];
    if (slot < 0 || slot >= a.cache.slots) return;
    const int start = max(0, a.cache.lengths[slot]);
    const int count = a.counts == nullptr ? a.tokens : min(max(a.counts[b], 0), a.tokens);
    if (count == 0) return;
    const int first = start / kKv8Block, last = (start + count - 1) / kKv8Block;
    const int block = first + at;
    if (block > last) return;
    // A call of more than 64 tokens can end in an open block that has the tail
    // slot of its first one.  The first block's CTA then takes both, the
    // last after it has read the old tokens.
    const bool shared_slot = at == 0 ? last > first && ((last - first) & 1) == 0
                                     : block == last && (at & 1) == 0;
    if (at != 0 && shared_slot) return;
    for (int now = block;; now = last) {
      kv8_append_block<D, E, T>(a, b, slot, head, now, start, count, peak);
      if (!shared_slot || now == last) return;
      __syncthreads();
    }
  }

  const int PER = a.chunks * kRopeUnroll * HeadLanes<D, E>::HEADS;
  const unsigned rounds = rope_rounds<D, E>(a.heads, a.chunks);
  const unsigned unit = (blockIdx.x - static_cast<unsigned>(a.kv_ctas)) * kKv8AppendWarps + threadIdx.x / 32;
  const unsigned token = unit / rounds;
  if (token >= static_cast<unsigned>(a.batch) * a.tokens) return;
  const int first = static_cast<int>(unit - token * rounds) * PER;
  const unsigned b = token / a.tokens, t = token - b * a.tokens;
  const int slot = a.slot_ids == nullptr ? b : a.slot_ids[b];
  // a slot that is none has no position: its queries become NaN where there is a rotation
  const int64_t position = slot < 0 || slot >= a.cache.slots ? -1 : static_cast<int64_t>(max(0, a.cache.lengths[slot])) + t;
  norm_rotate_round<D, E, T, __nv_bfloat16>(static_cast<const T*>(a.qkv) + b * a.batch_stride + t * a.token_stride,
                                            a.q_out + static_cast<int64_t>(token) * a.heads * D, first,
                                            min(first + PER, a.heads), a.norm.q_weight, position, a.norm, lane);
}

struct Kv8GatherArgs {
  Kv8Cache cache;
  const int32_t* slot_ids;
  const int32_t* counts;
  int tokens;        // tokens appended since the lengths were set, where counts is null
  int batch, most;   // tokens given out per sequence
  int ctas;          // per sequence
  __nv_bfloat16* k;  // [batch, most, kv_heads, D]
  __nv_bfloat16* v;
};

// Eight codes as bf16 values.
__device__ __forceinline__ uint4 kv8_values(const uint2& c, float scale) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // a byte under 2^23 is 2^23 + code
    const uint32_t two = i < 2 ? c.x : c.y;
    const float lo = __uint_as_float(__byte_perm(two, 0x4b000000u, i % 2 ? 0x7542 : 0x7540)) - 8388736.f;
    const float hi = __uint_as_float(__byte_perm(two, 0x4b000000u, i % 2 ? 0x7543 : 0x7541)) - 8388736.f;
    w[i] = pack_bf16x2(lo * scale, hi * scale);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Eight values a thread, keys and values: codes in, bf16 out (16 bytes, so that a warp's
// store is whole lines).  Tokens past a sequence's end are zero; a block whose
// page is not in the table is NaN.
template <int D>
__global__ void __launch_bounds__(256) kv8_gather_kernel(Kv8GatherArgs a) {
  constexpr unsigned PER = D / 8;
  griddep_wait();
  griddep_launch_dependents();
  const unsigned b = blockIdx.x / a.ctas;
  const unsigned at = (blockIdx.x - b * a.ctas) * 256 + threadIdx.x;  // (token, head, part)
  const unsigned row = at / PER, part = at % PER * 8;
  const unsigned t = row / a.cache.kv_heads, head = row - t * a.cache.kv_heads;
  if (t >= static_cast<unsigned>(a.most)) return;
  const int slot = a.slot_ids == nullptr ? static_cast<int>(b) : a.slot_ids[b];
  const bool known = slot >= 0 && slot < a.cache.slots;
  const int64_t total =
      known ? static_cast<int64_t>(max(0, a.cache.lengths[slot])) + (a.counts == nullptr ? a.tokens : max(0, a.counts[b])) : 0;
  const uint32_t fill = known ? 0u : 0x7fff7fffu;
  uint4 out[2] = {make_uint4(fill, fill, fill, fill), make_uint4(fill, fill, fill, fill)};
  if (known && t < total) {
    const int block = t / kKv8Block, in_block = t % kKv8Block;
    if (block == total / kKv8Block) {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
        out[kv] = *reinterpret_cast<const uint4*>(kv8_tail(a.cache, slot, block & 1, kv, head, D) + in_block * D + part);
    } else {
      const int page = kv8_page(a.cache, slot, block);
      const int64_t where = static_cast<int64_t>(max(page, 0)) * 2 * a.cache.kv_heads + head;  // page 0 is always there
      uint2 c[2];
      float scale[2];
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int64_t w = where + kv * a.cache.kv_heads;
        scale[kv] = a.cache.scales[w];
        c[kv] = *reinterpret_cast<const uint2*>(a.cache.codes + (w * kKv8Block + in_block) * D + part);
      }
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) out[kv] = kv8_values(c[kv], page < 0 ? __int_as_float(0x7fffffff) : scale[kv]);
    }
  }
  const int64_t to = ((static_cast<int64_t>(b) * a.most + t) * a.cache.kv_heads + head) * D + part;
  *reinterpret_cast<uint4*>(a.k + to) = out[0];
  *reinterpret_cast<uint4*>(a.v + to) = out[1];
}

}  // namespace b200tx
