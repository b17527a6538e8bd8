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
// once.  A head lies across L = D / E lanes with E = max(4, D/32) consecutive
// values each (one 8- or 16-byte access), so that the sum of squares and the
// pair's other half are shuffles and never leave the registers.  A lane holds
// the same dims of every head, so a warp loads its token's angles once and
// walks over the token's heads, four at a time to keep loads in flight.
#pragma once

#include "sm100_common.cuh"

namespace b200tx {

constexpr int kRopeWarps = 8;   // warps per CTA
constexpr int kRopeUnroll = 4;  // head groups in flight per warp

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

template <int D>
struct HeadLanes {
  static constexpr int E = D / 32 > 4 ? D / 32 : 4;  // values per lane
  static constexpr int L = D / E;                    // lanes per head
  static constexpr int HEADS = 32 / L;               // heads per warp
};

// E consecutive values as fp32.
template <int E>
__device__ __forceinline__ void load_values(const float* p, float (&x)[E]) {
#pragma unroll
  for (int i = 0; i < E; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(p + i);
    x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
  }
}

template <int E>
__device__ __forceinline__ void load_values(const __nv_bfloat16* p, float (&x)[E]) {
  uint32_t w[E / 2];
  if constexpr (E == 4) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

template <int E>
__device__ __forceinline__ void store_values(float* p, const float (&x)[E]) {
#pragma unroll
  for (int i = 0; i < E; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
}

template <int E>
__device__ __forceinline__ void store_values(__nv_bfloat16* p, const float (&x)[E]) {
  if constexpr (E == 4) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                                              pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
  }
}

// The angles of a lane's dims at one position.  c multiplies the value, s its
// partner: dims past `rotary` get (1, 0); the first of a pair carries -sin.
// A position outside the table gives NaN, which marks the head.
template <int D>
struct LaneAngles {
  static constexpr int E = HeadLanes<D>::E;
  float c[E], s[E];

  __device__ __forceinline__ void load(const RopeTable& r, int64_t position, int lane_in_head) {
    const int d0 = lane_in_head * E;
    if (r.cos == nullptr || d0 >= r.rotary) {
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
      for (int i = 0; i < E; ++i) {
        c[i] = __ldg(cr + at + i);
        const float sv = __ldg(sr + at + i);
        s[i] = first ? -sv : sv;
      }
    }
  }
};

// One head's values in a lane: the norm if this lane's head has one, then the
// rotation.  All lanes of the warp take part in the shuffles.
template <int D>
__device__ __forceinline__ void norm_rotate(float (&x)[HeadLanes<D>::E], const float (&w)[HeadLanes<D>::E], bool normed,
                                            float eps, const LaneAngles<D>& angles, const RopeTable& rope, int lane) {
  constexpr int E = HeadLanes<D>::E;
  constexpr int L = HeadLanes<D>::L;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
  for (int o = L / 2; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (normed) {
    const float r = rsqrtf(sum * (1.f / D) + eps);
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = x[i] * r * w[i];
  }
  if (rope.cos == nullptr) return;
  if (rope.interleaved) {
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float a = x[i], b = x[i + 1];
      x[i] = fmaf(a, angles.c[i], b * angles.s[i]);
      x[i + 1] = fmaf(b, angles.c[i + 1], a * angles.s[i + 1]);
    }
  } else {
    const int apart = rope.rotary / (2 * E);  // lanes between the halves of a pair
    const int l = lane % L;
    const int from = l < apart ? lane + apart : l < 2 * apart ? lane - apart : lane;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float other = __shfl_sync(0xffffffffu, x[i], from);
      x[i] = fmaf(x[i], angles.c[i], other * angles.s[i]);
    }
  }
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
  int splits, span;       // warps per token, head groups per warp
  QkNormArgs norm;
};

template <int D, typename T>
__global__ void __launch_bounds__(kRopeWarps * 32) qk_norm_rope_kernel(RopeArgs a) {
  constexpr int E = HeadLanes<D>::E;
  constexpr int L = HeadLanes<D>::L;
  constexpr int HEADS = HeadLanes<D>::HEADS;
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x % 32;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kRopeWarps + threadIdx.x / 32;
  const int64_t token = unit / a.splits;
  if (token >= a.total_tokens) return;
  const int split = static_cast<int>(unit - token * a.splits);
  const int64_t b = token / a.tokens;
  const int64_t t = token - b * a.tokens;
  const int in_head = lane % L;

  int64_t position = t;
  if (a.positions != nullptr) {
    const int64_t at = b * a.position_batch_stride + t;
    position = a.positions_64 ? static_cast<const int64_t*>(a.positions)[at] : static_cast<const int32_t*>(a.positions)[at];
  }
  LaneAngles<D> angles;
  angles.load(a.norm.rope, position, in_head);
  float qw[E] = {}, kw[E] = {};
  if (a.norm.q_weight != nullptr) load_values<E>(a.norm.q_weight + in_head * E, qw);
  if (a.norm.k_weight != nullptr) load_values<E>(a.norm.k_weight + in_head * E, kw);

  const T* src = static_cast<const T*>(a.in) + b * a.in_batch_stride + t * a.in_token_stride;
  T* dst = static_cast<T*>(a.out) + b * a.out_batch_stride + t * a.out_token_stride;
  const int turned = a.heads + a.kv_heads;
  const int all = a.copy_values ? turned + a.kv_heads : turned;
  const int first = split * a.span * HEADS;
  const int last = min(all, first + a.span * HEADS);
  for (int h0 = first; h0 < last; h0 += kRopeUnroll * HEADS) {
    float x[kRopeUnroll][E];
#pragma unroll
    for (int u = 0; u < kRopeUnroll; ++u) {
      const int h = h0 + u * HEADS + lane / L;
      if (h < last) {
        load_values<E>(src + h * D + in_head * E, x[u]);
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) x[u][i] = 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < kRopeUnroll; ++u) {
      const int h = h0 + u * HEADS + lane / L;
      const bool is_q = h < a.heads;
      float y[E], w[E];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        y[i] = x[u][i];
        w[i] = is_q ? qw[i] : kw[i];
      }
      const bool normed = is_q ? a.norm.q_weight != nullptr : a.norm.k_weight != nullptr;
      norm_rotate<D>(y, w, normed, a.norm.eps, angles, a.norm.rope, lane);
      if (h < turned) {
#pragma unroll
        for (int i = 0; i < E; ++i) x[u][i] = y[i];
      }
      if (h < last) store_values<E>(dst + h * D + in_head * E, x[u]);
    }
  }
}

}  // namespace b200tx
