// verify_kernels.cuh -- how many drafted tokens count, and the token after them.
//
// Token d_t, drafted with probability q_t(d_t), counts while u_t q_t(d_t) < p_t(d_t), p the
// target's probabilities and u given random numbers; the tokens counted this way, with the one that
// follows, are distributed as the target's own.  The one that follows is drawn from max(p_t - q_t, 0) at
// the first refusal, from p where every draft counts: the first index whose running sum
// passes u_T times the whole.  A draft without probabilities has q = 1 at its token.
//
// All sums are in 64 bits, products and differences of 32-bit numbers exact or nearly so,
// which decides borders as the definition does.  The work is one row of p and of q a
// sequence (not T + 1 of them): the row is known after one trip to memory for the drafts' tokens and one for
// their probabilities.  A cluster takes a sequence: its CTAs sum stretches of the row,
// exchange the sums, and the one CTA where the sum is passed looks through one stretch again.
#pragma once

#include "sm100_common.cuh"

namespace b200tx {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyParts = 64;     // stretches of a CTA's part of the row
constexpr int kVerifyTokens = 1024;  // drafted tokens of a sequence

struct VerifyArgs {
  const void* target;  // [batch, tokens + 1, vocab]
  const void* draft;   // [batch, tokens, vocab] or null
  const void* drafted; // [batch, tokens] int32 or int64
  const float* uniform;   // [batch, tokens + 1]
  const int32_t* counts;  // [batch] or null = tokens
  void* out;              // [batch, tokens + 1], drafted's type
  int32_t* accepted;      // [batch]
  int64_t target_batch_stride, target_token_stride, draft_batch_stride, draft_token_stride;
  int tokens, vocab, bf16, wide, vec;
};

template <typename T>
__device__ __forceinline__ double verify_value(const T* p) {
  if constexpr (sizeof(T) == 2)
    return __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p)) << 16);
  else
    return *p;
}

// Four neighbouring values.
template <typename T>
__device__ __forceinline__ void verify_four(const T* p, bool vec, int valid, float (&v)[4]) {
  if (vec && valid == 4) {
    if constexpr (sizeof(T) == 2) {
      const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
      v[0] = __uint_as_float(w.x << 16), v[1] = __uint_as_float(w.x & 0xffff0000u);
      v[2] = __uint_as_float(w.y << 16), v[3] = __uint_as_float(w.y & 0xffff0000u);
    } else {
      const float4 w = __ldg(reinterpret_cast<const float4*>(p));
      v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = i < valid ? static_cast<float>(verify_value<T>(p + i)) : 0.f;
}

// The mass of token i of four: what is left of p where the draft is refused.  NaN counts as nothing.
__device__ __forceinline__ double verify_mass(float p, float q) {
  const double d = static_cast<double>(p) - static_cast<double>(q);
  return d > 0.0 ? d : 0.0;
}

template <typename T>
__global__ void __launch_bounds__(kVerifyThreads) verify_draft_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ int s_first, s_token;
  __shared__ double s_part[kVerifyParts];
  __shared__ double s_cta[2][8];
  __shared__ int s_last[2][8];  // the last index of a CTA's part with mass, -1: none
  __shared__ int s_warp_last[kVerifyWarps];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  uint32_t ctas;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  const int C = static_cast<int>(ctas), c = static_cast<int>(cluster_ctarank());
  const int64_t b = blockIdx.x / ctas;
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  griddep_wait();
  griddep_launch_dependents();

  const T* const target = static_cast<const T*>(a.target) + b * a.target_batch_stride;
  const T* const draft = a.draft == nullptr ? nullptr : static_cast<const T*>(a.draft) + b * a.draft_batch_stride;
  const float* const uniform = a.uniform + b * (a.tokens + 1);
  const int n = a.counts == nullptr ? a.tokens : min(max(a.counts[b], 0), a.tokens);
  auto drafted = [&](int t) -> int64_t {
    const int64_t at = b * a.tokens + t;
    return a.wide ? static_cast<const int64_t*>(a.drafted)[at] : static_cast<const int32_t*>(a.drafted)[at];
  };
  if (tid == 0) s_first = n;
  __syncthreads();
  for (int t = tid; t < n; t += kVerifyThreads) {
    const int64_t token = drafted(t);
    bool good = false;  // a token outside of the vocabulary is refused
    if (token >= 0 && token < a.vocab) {
      const double p = verify_value<T>(target + t * a.target_token_stride + token);
      const double q = draft == nullptr ? 1.0 : verify_value<T>(draft + t * a.draft_token_stride + token);
      good = static_cast<double>(uniform[t]) * q < p;
    }
    if (!good) atomicMin(&s_first, t);
  }
  __syncthreads();
  const int first = s_first;
  const bool refused = first < n;
  const int64_t token = refused ? drafted(first) : -1;
  const T* const p_row = target + first * a.target_token_stride;
  const T* const q_row = refused && draft != nullptr ? draft + first * a.draft_token_stride : nullptr;
  const double u = fmax(static_cast<double>(uniform[a.tokens]), 0.0);
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

  // stretches: parts of the row for CTAs, of these for warps, whole fours for 32 lanes
  const int stretch = static_cast<int>((static_cast<int64_t>(a.vocab) + C * kVerifyParts * 128 - 1) / (C * kVerifyParts * 128)) * 128;
  const int begin = min(static_cast<int64_t>(a.vocab), static_cast<int64_t>(c) * kVerifyParts * stretch);
  // what is left of p; where nothing is, p itself
  for (int whole = refused ? 0 : 1; whole < 2; ++whole) {
    auto mass_of = [&](int at, float (&v)[4], double (&mass)[4]) {
      const int valid = min(max(a.vocab - at, 0), 4);
      float q[4] = {};
      verify_four<T>(p_row + at, a.vec, valid, v);
      if (whole == 0 && q_row != nullptr) verify_four<T>(q_row + at, a.vec, valid, q);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        mass[i] = whole == 0 && q_row == nullptr && at + i == token ? 0.0 : verify_mass(v[i], q[i]);
    };
    int last = -1;
    for (int part = warp; part < kVerifyParts; part += kVerifyWarps) {
      double sum = 0.0;
      const int64_t from = begin + static_cast<int64_t>(part) * stretch, to = min(static_cast<int64_t>(a.vocab), from + stretch);
#pragma unroll 4
      for (int64_t at = from + lane * 4; at < to; at += 128) {
        float v[4];
        double mass[4];
        mass_of(static_cast<int>(at), v, mass);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sum += mass[i];
          if (mass[i] > 0.0) last = static_cast<int>(at) + i;
        }
      }
#pragma unroll
      for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (lane == 0) s_part[part] = sum;
    }
    last = __reduce_max_sync(0xffffffffu, last);
    if (lane == 0) s_warp_last[warp] = last;
    __syncthreads();
    if (warp == 0) {
      double sum = 0.0;
      for (int i = 0; i < kVerifyParts; ++i) sum += s_part[i];
      int most = -1;
      for (int i = 0; i < kVerifyWarps; ++i) most = max(most, s_warp_last[i]);
      if (lane < C) {
        asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(peer_smem_addr(&s_cta[whole][c], lane)), "d"(sum) : "memory");
        asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(peer_smem_addr(&s_last[whole][c], lane)), "r"(most) : "memory");
      }
    }
    cluster_sync();
    double all = 0.0;
    int end = -1;
    for (int i = 0; i < C; ++i) {
      all += s_cta[whole][i];
      end = max(end, s_last[whole][i]);
    }
    if (end < 0 && whole == 0) continue;  // the same in every CTA
    const double wanted = u * all;
    // the first CTA in which the running sum passes what is wanted; if none, the last index with mass
    double running = 0.0;
    int owner = -1;
    for (int i = 0; i < C; ++i) {
      if (running + s_cta[whole][i] > wanted) {
        owner = i;
        break;
      }
      running += s_cta[whole][i];
    }
    if (owner < 0) {
      if (c == 0 && tid == 0) s_token = end;
      owner = 0;
    } else if (owner == c && warp == 0) {
      int part = 0;
      for (; part < kVerifyParts - 1; ++part) {
        if (running + s_part[part] > wanted) break;
        running += s_part[part];
      }
      // 128 values at a time, in order
      int found = -1, latest = -1;
      const int64_t from = begin + static_cast<int64_t>(part) * stretch, to = min(static_cast<int64_t>(a.vocab), from + stretch);
      for (int64_t base = from; base < to && found < 0; base += 128) {
        float v[4];
        double mass[4];
        const int at = static_cast<int>(base) + lane * 4;
        mass_of(at, v, mass);
        const double mine = mass[0] + mass[1] + mass[2] + mass[3];
        double sum = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
          const double o = __shfl_up_sync(0xffffffffu, sum, d);
          if (lane >= d) sum += o;
        }
        double at_sum = running + (sum - mine);
        int here = -1, held = -1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          at_sum += mass[i];
          if (mass[i] > 0.0) held = at + i;
          if (here < 0 && mass[i] > 0.0 && at_sum > wanted) here = at + i;
        }
        const uint32_t bits = __ballot_sync(0xffffffffu, here >= 0);
        if (bits != 0) found = __shfl_sync(0xffffffffu, here, __ffs(bits) - 1);
        latest = max(latest, __reduce_max_sync(0xffffffffu, held));
        running += __shfl_sync(0xffffffffu, sum, 31);
      }
      // rounding may leave the sum of one's parts short of their total: then the last with mass is it
      if (lane == 0) s_token = found >= 0 ? found : latest >= 0 ? latest : s_last[whole][c];
    }
    __syncthreads();
    if (owner == c) {
      for (int t = tid; t <= a.tokens; t += kVerifyThreads) {
        const int64_t value = t < first ? drafted(t) : t == first ? s_token : -1;
        const int64_t at = b * (a.tokens + 1) + t;
        if (a.wide)
          static_cast<int64_t*>(a.out)[at] = value;
        else
          static_cast<int32_t*>(a.out)[at] = static_cast<int32_t>(value);
      }
      if (tid == 0) a.accepted[b] = first;
    }
    return;
  }
}

}  // namespace b200tx
