// kv8_cache_kernels.cuh -- the paged key/value cache held in 8 bits: appending
// tokens and reading values back.
//
// A sequence's tokens lie in blocks of 64.  A block that is full is held as
// 8-bit codes with one fp32 scale per kv head, for keys and for values:
//     scale = max |x| / 127 over the block's 64 x D values of the head
//     code  = rint(x / scale) + 128,       x ~ (code - 128) * scale
// The block that is still open is held in bf16 in the sequence's tail.  Its
// scale is only known when its last token arrives; with the open block in 16
// bits nothing is ever quantised twice, and a prompt appended at once gives
// the same bits as the same tokens one at a time.  Keys and values are
// rounded to bf16 when they enter, whichever way they take.
//
// The offset of 128 makes a code the low byte of an fp16 number 1024 + code:
// the attention turns bytes into numbers with one byte permute and one
// subtraction for two of them.
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
  QkNormArgs norm;
};

constexpr int kKv8AppendWarps = 8;

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
      float y[E], x[E];
      norm_rotate<D, E, T>(k_raw[p], y, f, a.norm.k_weight != nullptr, a.norm.eps, angles.turned, a.norm.rope, partner);
      v_raw[p].values(x);
      k.set(y);
      v.set(x);
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

  // The largest magnitude as a bit pattern: the order of non-negative floats,
  // with infinity and then NaN above every finite value.
  uint32_t k_max = 0, v_max = 0;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      k_max = max(k_max, max((k_bits[p][i] << 16) & 0x7fff0000u, k_bits[p][i] & 0x7fff0000u));
      v_max = max(v_max, max((v_bits[p][i] << 16) & 0x7fff0000u, v_bits[p][i] & 0x7fff0000u));
    }
  }
  k_max = __reduce_max_sync(0xffffffffu, k_max);
  v_max = __reduce_max_sync(0xffffffffu, v_max);
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
  auto code = [](uint32_t bits, float scale) -> uint32_t {
    // scale 0: a block of zeros; scale NaN: any code, the scale says it all
    return scale > 0.f ? static_cast<uint32_t>(__float2int_rn(__uint_as_float(bits) / scale) + 128) : 128u;
  };
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int in_block = p * PASS + warp * TOKENS + lane / L;
    if (in_block >= kKv8Block) continue;
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
      uint32_t kc = 0, vc = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t kb = k_bits[p][2 * i + j], vb = v_bits[p][2 * i + j];
        kc |= (code(kb << 16, k_scale) | code(kb & 0xffff0000u, k_scale) << 8) << (16 * j);
        vc |= (code(vb << 16, v_scale) | code(vb & 0xffff0000u, v_scale) << 8) << (16 * j);
      }
      reinterpret_cast<uint32_t*>(k_codes + in_block * D + in_head * E)[i] = kc;
      reinterpret_cast<uint32_t*>(v_codes + in_block * D + in_head * E)[i] = vc;
    }
  }
}

// CTAs below kv_ctas each take one block of one kv head; the rest norm and
// rotate the queries, a warp for a round of a token's heads as in qk_norm_rope_kernel.
template <int D, int E, typename T>
__global__ void __launch_bounds__(kKv8AppendWarps * 32) kv8_append_kernel(Kv8AppendArgs a) {
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

  constexpr int PER = kRopeUnroll * HeadLanes<D, E>::HEADS;
  const unsigned rounds = rope_rounds<D, E>(a.heads);
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
  __nv_bfloat16* k;  // [batch, most, kv_heads, D]
  __nv_bfloat16* v;
};

// Eight values a thread, keys and values: codes in, bf16 out.  Tokens past a
// sequence's end are zero; a block whose page is not in the table is NaN.
template <int D>
__global__ void __launch_bounds__(256) kv8_gather_kernel(Kv8GatherArgs a) {
  constexpr int PER = D / 8;
  griddep_wait();
  griddep_launch_dependents();
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = at / PER;  // (b, token, head)
  const int part = static_cast<int>(at % PER) * 8;
  const int64_t bt = row / a.cache.kv_heads;
  const int head = static_cast<int>(row % a.cache.kv_heads);
  const int64_t b = bt / a.most;
  const int t = static_cast<int>(bt % a.most);
  if (b >= a.batch) return;
  const int slot = a.slot_ids == nullptr ? static_cast<int>(b) : a.slot_ids[b];
  const bool known = slot >= 0 && slot < a.cache.slots;
  const int total = known ? max(0, a.cache.lengths[slot]) + (a.counts == nullptr ? a.tokens : max(0, a.counts[b])) : 0;
  uint4 out[2] = {};
  if (!known) {
    out[0] = out[1] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
  } else if (t < total) {
    const int block = t / kKv8Block, in_block = t % kKv8Block;
    if (block == total / kKv8Block) {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
        out[kv] = *reinterpret_cast<const uint4*>(kv8_tail(a.cache, slot, block & 1, kv, head, D) + in_block * D + part);
    } else {
      const int page = kv8_page(a.cache, slot, block);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        float scale = __int_as_float(0x7fffffff);
        uint2 c = make_uint2(0u, 0u);
        if (page >= 0) {
          const int64_t where = (static_cast<int64_t>(page) * 2 + kv) * a.cache.kv_heads + head;
          scale = a.cache.scales[where];
          c = *reinterpret_cast<const uint2*>(a.cache.codes + (where * kKv8Block + in_block) * D + part);
        }
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t two = (i < 2 ? c.x : c.y) >> (16 * (i & 1));
          w[i] = pack_bf16x2((static_cast<int>(two & 255u) - 128) * scale, (static_cast<int>((two >> 8) & 255u) - 128) * scale);
        }
        out[kv] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  const int64_t to = row * D + part;
  *reinterpret_cast<uint4*>(a.k + to) = out[0];
  *reinterpret_cast<uint4*>(a.v + to) = out[1];
}

}  // namespace b200tx
