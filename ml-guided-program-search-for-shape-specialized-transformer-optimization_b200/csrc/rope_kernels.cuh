// rope_kernels.cuh -- RMS norm of each query and key head and the rotation by
// position, in one pass over the packed projection [B, T, (Hq + 2 Hkv) * D].
//
// A head x in R^D becomes  y = x / sqrt(mean(x^2) + eps) * w  (no weight: y = x),
// and its first R dims are turned by the position p: a pair (a, b) becomes
// (a cos - b sin, b cos + a sin), with the angles of row p of the tables.
// Pairs are (i, i + R/2), or (2i, 2i + 1) when interleaved.  Value heads are
// copied.  Everything is computed in fp32 and rounded once.
//
// The work is elementwise, so HBM bounds it: each value is read and written
// once.  A head lies across L = D / E lanes with E = 8 (or 4) consecutive values
// each, one 16-byte access of bf16, so that the sum of squares and the pair's
// other half are shuffles and never leave the registers.  The factor of the norm
// is common to a head, so the pair's other half is exchanged as it was read (two
// bf16 a shuffle) and
//   y = r (x (w c) + x' (w' s))
// with w c and w' s computed once for the four groups of heads that a warp takes
// of a token (a lane holds the same dims of every head); their loads go out
// together.  8 x 2048 tokens of 48 heads of 64 (201 MB) take 38 us, 5.3 TB/s.
#pragma once

#include "sm100_common.cuh"

namespace b200tx {

constexpr int kRopeWarps = 4;   // warps per CTA (8: 42 us for 8 x 2048 tokens of 48 heads of 64, 4: 38 us)
constexpr int kRopeUnroll = 4;  // head groups of a warp

struct RopeTable {
  const float* cos;  // [positions, rotary/2]; null = no rotation
  const float* sin;
  int positions, rotary, interleaved;
};

struct QkNormArgs {
  const float* q_weight;  // [D] or null
  const float* k_weight;
  float eps;
  RopeTable rope;
};

template <int D, int E>
struct HeadLanes {
  static constexpr int L = D / E;      // lanes per head
  static constexpr int HEADS = 32 / L;  // heads per warp
};

// 1 / sqrt(x) to 2^-22; x is a mean of squares plus eps.
__device__ __forceinline__ float fast_rsqrt(float x) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// E consecutive values as they lie in memory: one access of up to 16 bytes, two of fp32.
template <typename T, int E>
struct Raw {
  static constexpr int WORDS = E * static_cast<int>(sizeof(T)) / 4;
  uint32_t w[WORDS];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (WORDS == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; i += 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + i);
        w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
      }
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (WORDS == 2) {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; i += 4)
        *reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(p) + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    }
  }
  __device__ __forceinline__ void values(float (&x)[E]) const {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = __uint_as_float(w[i]);
    }
  }
  __device__ __forceinline__ void set(const float (&x)[E]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) w[i] = __float_as_uint(x[i]);
    }
  }
};

// The angles of a lane's dims at one position: c multiplies the value, s the
// pair's other half (-sin for the first of a pair).  A position outside the table
// gives NaN, which marks the head.
template <int D, int E>
struct LaneAngles {
  float c[E], s[E];
  bool turned;  // the lane's dims are among the first `rotary`

  __device__ __forceinline__ void load(const RopeTable& r, int64_t position, int lane_in_head) {
    const int d0 = lane_in_head * E;
    turned = r.cos != nullptr && d0 < r.rotary;
    if (!turned) {
#pragma unroll
      for (int i = 0; i < E; ++i) { c[i] = 1.f; s[i] = 0.f; }
      return;
    }
    if (position < 0 || position >= r.positions) {
#pragma unroll
      for (int i = 0; i < E; ++i) c[i] = s[i] = __int_as_float(0x7fffffff);
      return;
    }
    const int half = r.rotary / 2;
    const float* cr = r.cos + position * half;
    const float* sr = r.sin + position * half;
    if (r.interleaved) {
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        const float cv = __ldg(cr + d0 / 2 + i / 2), sv = __ldg(sr + d0 / 2 + i / 2);
        c[i] = c[i + 1] = cv;
        s[i] = -sv;
        s[i + 1] = sv;
      }
    } else {
      const bool first = d0 < half;
      const int at = first ? d0 : d0 - half;
#pragma unroll
      for (int i = 0; i < E; i += 4) {
        const float4 cv = *reinterpret_cast<const float4*>(cr + at + i);
        const float4 sv = *reinterpret_cast<const float4*>(sr + at + i);
        c[i] = cv.x; c[i + 1] = cv.y; c[i + 2] = cv.z; c[i + 3] = cv.w;
        s[i] = sv.x; s[i + 1] = sv.y; s[i + 2] = sv.z; s[i + 3] = sv.w;
      }
#pragma unroll
      for (int i = 0; i < E; ++i) s[i] = first ? -s[i] : s[i];
    }
  }
};

// The lane that has the pair's other half (itself where there is none).
template <int D, int E>
__device__ __forceinline__ int partner_lane(const RopeTable& r, int lane) {
  const int apart = r.rotary / (2 * E);
  const int l = lane % HeadLanes<D, E>::L;
  return l < apart ? lane + apart : l < 2 * apart ? lane - apart : lane;
}

// w c and w' s of a lane's dims, for one kind of head at one position.
template <int D, int E>
struct LaneFactors {
  float own[E], other[E];

  __device__ __forceinline__ void set(const float* weight, const LaneAngles<D, E>& a, const RopeTable& r, int lane) {
    const int d0 = lane % HeadLanes<D, E>::L * E;
    const int p0 = r.interleaved ? d0 : partner_lane<D, E>(r, lane) % HeadLanes<D, E>::L * E;
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      float4 w = make_float4(1.f, 1.f, 1.f, 1.f), p = w;
      if (weight != nullptr) {
        w = __ldg(reinterpret_cast<const float4*>(weight + d0 + i));
        p = __ldg(reinterpret_cast<const float4*>(weight + p0 + i));
        if (r.interleaved) p = make_float4(p.y, p.x, p.w, p.z);
      }
      own[i] = a.c[i] * w.x; own[i + 1] = a.c[i + 1] * w.y; own[i + 2] = a.c[i + 2] * w.z; own[i + 3] = a.c[i + 3] * w.w;
      other[i] = a.s[i] * p.x; other[i + 1] = a.s[i + 1] * p.y; other[i + 2] = a.s[i + 2] * p.z; other[i + 3] = a.s[i + 3] * p.w;
    }
  }
};

// One head's values in a lane, normed and turned.  All lanes of the warp take part.
template <int D, int E, typename T>
__device__ __forceinline__ void norm_rotate(const Raw<T, E>& raw, float (&y)[E], const LaneFactors<D, E>& f, bool normed,
                                            float eps, bool turned, const RopeTable& rope, int partner) {
  float x[E];
  raw.values(x);
  float r = 1.f;
  if (normed) {
    uint64_t two = f32x2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const uint64_t v = f32x2(x[i], x[i + 1]);
      two = fma_f32x2(v, v, two);
    }
    float sum = unpack_f32x2(two).x + unpack_f32x2(two).y;
#pragma unroll
    for (int o = HeadLanes<D, E>::L / 2; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    r = fast_rsqrt(fmaf(sum, 1.f / D, eps));
  }
  float z[E];
  if (rope.cos != nullptr && !rope.interleaved) {
    Raw<T, E> other;
#pragma unroll
    for (int i = 0; i < Raw<T, E>::WORDS; ++i) other.w[i] = __shfl_sync(0xffffffffu, raw.w[i], partner);
    other.values(z);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) z[i] = x[i ^ 1];
  }
  const uint64_t rr = f32x2(r, r);
#pragma unroll
  for (int i = 0; i < E; i += 2) {
    uint64_t v = mul_f32x2(f32x2(x[i], x[i + 1]), f32x2(f.own[i], f.own[i + 1]));
    if (turned) v = fma_f32x2(f32x2(z[i], z[i + 1]), f32x2(f.other[i], f.other[i + 1]), v);
    const float2 out = unpack_f32x2(mul_f32x2(v, rr));
    y[i] = out.x;
    y[i + 1] = out.y;
  }
}

// Heads [first, last) of one kind at one token, kRopeUnroll x HEADS of them at a time.
template <int D, int E, typename T, typename OutT>
__device__ __forceinline__ void norm_rotate_round(const T* src, OutT* dst, int first, int last, const float* weight,
                                                  int64_t position, const QkNormArgs& norm, int lane) {
  constexpr int HEADS = HeadLanes<D, E>::HEADS;
  constexpr int L = HeadLanes<D, E>::L;
  constexpr int PER = kRopeUnroll * HEADS;
  const int mine = first + lane / L;
  src += mine * D + lane % L * E;
  dst += mine * D + lane % L * E;
  int left = last - mine;  // this lane's heads come every HEADS
  Raw<T, E> x[kRopeUnroll];
#pragma unroll
  for (int u = 0; u < kRopeUnroll; ++u) {
    x[u].zero();
    if (u * HEADS < left) x[u].load(src + u * HEADS * D);
  }
  LaneAngles<D, E> angles;
  angles.load(norm.rope, position, lane % L);
  LaneFactors<D, E> f;
  f.set(weight, angles, norm.rope, lane);
  const int partner = partner_lane<D, E>(norm.rope, lane);
  for (;;) {
#pragma unroll
    for (int u = 0; u < kRopeUnroll; ++u) {
      if (first + u * HEADS >= last) break;
      float y[E];
      norm_rotate<D, E, T>(x[u], y, f, weight != nullptr, norm.eps, angles.turned, norm.rope, partner);
      Raw<OutT, E> out;
      out.set(y);
      if (u * HEADS < left) out.store(dst + u * HEADS * D);
    }
    first += PER;
    if (first >= last) return;
    left -= PER;
    src += PER * D;
    dst += PER * D;
#pragma unroll
    for (int u = 0; u < kRopeUnroll; ++u)
      if (u * HEADS < left) x[u].load(src + u * HEADS * D);
  }
}

// Warps for a kind of head of one token, each taking `chunks` times PER heads.
template <int D, int E>
__host__ __device__ constexpr int rope_rounds(int heads, int chunks) {
  const int per = chunks * kRopeUnroll * HeadLanes<D, E>::HEADS;
  return (heads + per - 1) / per;
}

struct RopeArgs {
  const void* in;
  void* out;
  int64_t in_batch_stride, in_token_stride;    // elements
  int64_t out_batch_stride, out_token_stride;
  const void* positions;  // int32 or int64, null = the token's index
  int64_t position_batch_stride;
  int positions_64;
  int tokens, heads, kv_heads;
  int copy_values;        // 0: the values are left as they are (in place)
  int64_t total_tokens;   // batch * tokens
  int chunks;             // of kRopeUnroll head groups that a warp takes
  QkNormArgs norm;
};

// A CTA takes a round (of the queries, keys or values) of 4 tokens, a warp each;
// the rounds of the same tokens are neighbours, as they are in memory.
template <int D, int E, typename T>
__global__ void __launch_bounds__(kRopeWarps * 32) qk_norm_rope_kernel(RopeArgs a) {
  constexpr int HEADS = HeadLanes<D, E>::HEADS;
  const int PER = a.chunks * kRopeUnroll * HEADS;
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x % 32;
  const int q_rounds = rope_rounds<D, E>(a.heads, a.chunks), k_rounds = rope_rounds<D, E>(a.kv_heads, a.chunks);
  const unsigned rounds = q_rounds + k_rounds + (a.copy_values ? k_rounds : 0);
  const unsigned first_token = blockIdx.x / rounds * kRopeWarps;
  const int round = static_cast<int>(blockIdx.x % rounds);
  const unsigned token = first_token + threadIdx.x / 32;
  if (token >= a.total_tokens) return;
  const unsigned b = token / a.tokens, t = token - b * a.tokens;
  const T* src = static_cast<const T*>(a.in) + b * a.in_batch_stride + t * a.in_token_stride;
  T* dst = static_cast<T*>(a.out) + b * a.out_batch_stride + t * a.out_token_stride;

  if (round < q_rounds + k_rounds) {
    int64_t position = t;
    if (a.positions != nullptr) {
      const int64_t at = b * a.position_batch_stride + t;
      position = a.positions_64 ? static_cast<const int64_t*>(a.positions)[at] : static_cast<const int32_t*>(a.positions)[at];
    }
    const bool is_q = round < q_rounds;
    const int first = is_q ? round * PER : a.heads + (round - q_rounds) * PER;
    const int last = min(first + PER, is_q ? a.heads : a.heads + a.kv_heads);
    norm_rotate_round<D, E, T, T>(src, dst, first, last, is_q ? a.norm.q_weight : a.norm.k_weight, position, a.norm, lane);
    return;
  }
  constexpr int L = HeadLanes<D, E>::L;
  int first = a.heads + a.kv_heads + (round - q_rounds - k_rounds) * PER + lane / L;
  const int last = min(first + PER, a.heads + 2 * a.kv_heads);
  for (; first < last; first += kRopeUnroll * HEADS) {
    Raw<T, E> x[kRopeUnroll];
#pragma unroll
    for (int u = 0; u < kRopeUnroll; ++u)
      if (first + u * HEADS < last) x[u].load(src + (first + u * HEADS) * D + lane % L * E);
#pragma unroll
    for (int u = 0; u < kRopeUnroll; ++u)
      if (first + u * HEADS < last) x[u].store(dst + (first + u * HEADS) * D + lane % L * E);
  }
}

}  // namespace b200tx
