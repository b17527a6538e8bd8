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
// exchange the sums, and the one CTA where the sum is passed looks through one warp's stretch again.
//
// What bounds it: 64 sequences x 128000, both rows fp32: 15.5 us for 52 MB (8.0 at the copy rate): 1.2 to 2.5 until the row is known, the
// rows at the copy rate, then exchange, choice and the second look 2 to 4 more.  One sequence x 32000: 5.1 us, five trips to memory.
#pragma once

#include "sm100_common.cuh"

namespace b200tx {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyMostCtas = 8;
constexpr int kVerifyTokens = 1024;  // drafted tokens of a sequence
constexpr int kVerifyLook = 256;     // values that a warp looks through one by one, the CTA's warps at the same time

struct VerifyArgs {
  const void* target;  // [batch, tokens + 1, vocab]
  const void* draft;   // [batch, tokens, vocab] or null
  const void* drafted; // [batch, tokens] int32 or int64
  const float* uniform;   // [batch, tokens + 1]
  const int32_t* counts;  // [batch] or null = tokens
  void* out;              // [batch, tokens + 1], drafted's type
  int32_t* accepted;      // [batch]
  int64_t target_batch_stride, target_token_stride, draft_batch_stride, draft_token_stride;
  int tokens, vocab, wide;
};

template <typename T>
__device__ __forceinline__ float verify_value(const T* p) {
  if constexpr (sizeof(T) == 2)
    return __uint_as_float(static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(p))) << 16);
  else
    return __ldg(p);
}

// A row's masses: what is left of p where the draft is refused.  A mass that is NaN counts as nothing.
template <typename T, bool VEC>
struct VerifyRow {
  const T* p;
  const T* q;    // or null
  int excluded;  // a token whose mass is taken away whole, or -1

  __device__ __forceinline__ double mass(float a, float b, int at) const {
    const double d = static_cast<double>(a) - static_cast<double>(b);
    return d > 0.0 && at != excluded ? d : 0.0;
  }

  __device__ __forceinline__ double one(int at) const { return mass(verify_value(p + at), q == nullptr ? 0.f : verify_value(q + at), at); }

  // Values that a lane reads at once, 16 bytes, or one where rows start anywhere.
  static constexpr int PER = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;

  template <bool TWO>
  __device__ __forceinline__ double sum_of(int from, int to) const {
    constexpr int U = VEC ? 4 : 16, STEP = 32 * PER;
    const int lane = threadIdx.x % 32;
    double sum = 0.0, other = 0.0;  // two sums, for the latency of an addition
    int at = from + lane * PER;
    if constexpr (VEC) {
      // whole steps, their loads together
      for (; at + (U - 1) * STEP + PER <= to; at += U * STEP) {
        uint4 v[U], w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          v[u] = __ldg(reinterpret_cast<const uint4*>(p + at + u * STEP));
          if (TWO) w[u] = __ldg(reinterpret_cast<const uint4*>(q + at + u * STEP));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t x[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
          const uint32_t y[4] = {TWO ? w[u].x : 0u, TWO ? w[u].y : 0u, TWO ? w[u].z : 0u, TWO ? w[u].w : 0u};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int where = at + u * STEP;
            if constexpr (sizeof(T) == 2) {
              sum += mass(__uint_as_float(x[i] << 16), __uint_as_float(y[i] << 16), where + 2 * i);
              other += mass(__uint_as_float(x[i] & 0xffff0000u), __uint_as_float(y[i] & 0xffff0000u), where + 2 * i + 1);
            } else if (i % 2) {
              other += mass(__uint_as_float(x[i]), __uint_as_float(y[i]), where + i);
            } else {
              sum += mass(__uint_as_float(x[i]), __uint_as_float(y[i]), where + i);
            }
          }
        }
      }
    } else {
      for (; at + (U - 1) * STEP < to; at += U * STEP) {
        float v[U], w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          v[u] = verify_value(p + at + u * STEP);
          w[u] = TWO ? verify_value(q + at + u * STEP) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) (u % 2 ? other : sum) += mass(v[u], w[u], at + u * STEP);
      }
    }
    for (; at < to; at += STEP) {
      for (int i = 0; i < PER && at + i < to; ++i) sum += one(at + i);
    }
    sum += other;
#pragma unroll
    for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    return sum;
  }

  // The masses from..to - 1 summed by a warp; the same in all lanes.
  __device__ __forceinline__ double sum(int from, int to) const {
    return q != nullptr ? sum_of<true>(from, to) : sum_of<false>(from, to);
  }
};

// Of n sums in order the one in which the running sum passes `wanted`; where rounding, or a wish past the whole, leaves
// none, the last with mass, and from then on.
__device__ __forceinline__ int verify_pick(const double* sums, int n, double& running, double& wanted) {
  int last = 0;
  double before = running;
  for (int i = 0; i < n; ++i) {
    if (running + sums[i] > wanted) return i;
    if (sums[i] > 0.0) {
      last = i;
      before = running;
    }
    running += sums[i];
  }
  running = before;
  wanted = __longlong_as_double(0x7ff0000000000000ll);
  return last;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kVerifyThreads) verify_draft_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ int s_first;
  __shared__ double s_part[2][kVerifyWarps];
  __shared__ double s_cta[2][kVerifyMostCtas];
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
  const double u = fmax(static_cast<double>(uniform[a.tokens]), 0.0);
  const int n = a.counts == nullptr ? a.tokens : min(max(a.counts[b], 0), a.tokens);
  auto drafted = [&](int t) -> int64_t {
    const int64_t at = b * a.tokens + t;
    return a.wide ? static_cast<const int64_t*>(a.drafted)[at] : static_cast<const int32_t*>(a.drafted)[at];
  };
  if (tid == 0) s_first = n;
  __syncthreads();
  for (int t = tid; t < n; t += kVerifyThreads) {
    const float mine = uniform[t];
    const int64_t token = drafted(t);
    bool good = false;  // a token outside of the vocabulary is refused
    if (token >= 0 && token < a.vocab) {
      const double p = verify_value<T>(target + t * a.target_token_stride + token);
      const double q = draft == nullptr ? 1.0 : static_cast<double>(verify_value<T>(draft + t * a.draft_token_stride + token));
      good = static_cast<double>(mine) * q < p;
    }
    if (!good) atomicMin(&s_first, t);
  }
  __syncthreads();
  const int first = s_first;
  const bool refused = first < n;
  VerifyRow<T, VEC> row;
  row.p = target + first * a.target_token_stride;
  row.q = nullptr;
  row.excluded = -1;
  if (refused && draft != nullptr) row.q = draft + first * a.draft_token_stride;
  if (refused && draft == nullptr) {
    const int64_t token = drafted(first);
    row.excluded = token >= 0 && token < a.vocab ? static_cast<int>(token) : -1;
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

  // a part of the row for each warp of the cluster, in order
  const int64_t parts = C * kVerifyWarps;
  int length = static_cast<int>((a.vocab + parts * 256 - 1) / (parts * 256) * 256);
  auto end = [&](int64_t from, int64_t many) { return static_cast<int>(min(static_cast<int64_t>(a.vocab), from + many)); };
  double all = 0.0;
  int turn = 0;
  // what is left of p; where nothing is, p itself
  for (;; ++turn) {
    const int64_t from = static_cast<int64_t>(c * kVerifyWarps + warp) * length;
    const double sum = from < a.vocab ? row.sum(static_cast<int>(from), end(from, length)) : 0.0;
    if (lane == 0) s_part[0][warp] = sum;
    __syncthreads();
    if (warp == 0 && lane < C) {
      double mine = 0.0;
      for (int i = 0; i < kVerifyWarps; ++i) mine += s_part[0][i];
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(peer_smem_addr(&s_cta[turn][c], lane)), "d"(mine) : "memory");
    }
    cluster_sync();
    all = 0.0;
    for (int i = 0; i < C; ++i) all += s_cta[turn][i];
    if (turn == 1 || (row.q == nullptr && row.excluded < 0) || all > 0.0) break;  // the same in every CTA
    row.q = nullptr;
    row.excluded = -1;
  }
  double wanted = u * all, running = 0.0;
  if (verify_pick(s_cta[turn], C, running, wanted) != c) return;

  int64_t token = -1;
  if (all > 0.0) {
    // a part, the eighth of it, and so on, until the warps look through what is left
    int pick = verify_pick(s_part[0], kVerifyWarps, running, wanted);
    int64_t from = static_cast<int64_t>(c * kVerifyWarps + pick) * length;
    int limit = end(from, length), level = 1;
    for (; length > kVerifyWarps * kVerifyLook; ++level) {
      length = (length + kVerifyWarps * 256 - 1) / (kVerifyWarps * 256) * 256;
      const int64_t mine = from + static_cast<int64_t>(warp) * length;
      const double sum = mine < limit ? row.sum(static_cast<int>(mine), min(limit, end(mine, length))) : 0.0;
      if (lane == 0) s_part[level & 1][warp] = sum;
      __syncthreads();
      pick = verify_pick(s_part[level & 1], kVerifyWarps, running, wanted);
      from += static_cast<int64_t>(pick) * length;
      limit = min(limit, end(from, length));
    }
    // eight neighbouring values a lane
    from += warp * kVerifyLook + lane * kVerifyLook / 32;
    double mass[kVerifyLook / 32], mine = 0.0;
#pragma unroll
    for (int i = 0; i < kVerifyLook / 32; ++i) mass[i] = from + i < limit ? row.one(static_cast<int>(from + i)) : 0.0;
#pragma unroll
    for (int i = 0; i < kVerifyLook / 32; ++i) mine += mass[i];
    double upto = mine;  // with the lanes before
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const double o = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += o;
    }
    if (lane == 31) s_part[level & 1][warp] = upto;
    __syncthreads();
    if (verify_pick(s_part[level & 1], kVerifyWarps, running, wanted) != warp) return;
    running += upto - mine;
    int latest = -1, found = -1;
#pragma unroll
    for (int i = 0; i < kVerifyLook / 32; ++i) {
      running += mass[i];
      if (mass[i] > 0.0) {
        latest = i;
        if (found < 0 && running > wanted) found = i;
      }
    }
    const uint32_t passed = __ballot_sync(0xffffffffu, found >= 0), held = __ballot_sync(0xffffffffu, latest >= 0);
    const int64_t at = from + (passed != 0 ? found : latest);
    token = __shfl_sync(0xffffffffu, at, passed != 0 ? __ffs(passed) - 1 : 31 - __clz(held));
  } else if (warp != 0) {
    return;
  }
  // one warp of one CTA is left
  for (int t = lane; t <= a.tokens; t += 32) {
    const int64_t value = t < first ? drafted(t) : t == first ? token : -1;
    const int64_t at = b * (a.tokens + 1) + t;
    if (a.wide)
      static_cast<int64_t*>(a.out)[at] = value;
    else
      static_cast<int32_t*>(a.out)[at] = static_cast<int32_t>(value);
  }
  if (lane == 0) a.accepted[b] = first;
}

}  // namespace b200tx
