// A router's scores to experts and weights, and the balance loss, with gradients.
//
// logits[t, e] are T rows of E scores (E <= 1024).  With p = softmax of a row:
//
//   route      the k largest scores of a row, descending, ties to the lower
//              expert: experts[t, j], weights[t, j] = p at them, divided by
//              their sum with `normalize`.
//   its        normalize:  dl[id_j] = w_j (g_j - sum_i w_i g_i), 0 elsewhere
//   gradient   otherwise:  dl[e] = [e = id_j] p_e g_j - p_e sum_i p_i g_i
//   balance    c[e] = entries with experts[t, j] = e of the tokens counted,
//              S = sum c, n = tokens counted,
//              loss = E sum_e (c[e] / S) (sum_t p[t, e] / n),  0 when S or n is 0
//   its        a[e] = g E c[e] / (S n),  dl[t, e] = p_e (a[e] - sum_i a_i p_i),
//   gradient   0 for tokens not counted
//
// A score of -inf has p = 0 and is never chosen: a row with fewer than k others
// ends with entries -1 of weight 0 (which expert_sort drops), a row of them alone
// has p = 0 throughout.  A NaN counts as the largest score, and NaN or +inf make
// the row's p NaN, as the formula does.  Scores as low as the type goes are
// ordinary numbers.  Numbers outside 0..E-1 in `experts` mark dropped entries.
//
// One warp takes a row, NV scores a lane, in registers; exponentials, sums and
// gradients are fp32.  Sums over tokens have a fixed order: a warp's rows, the
// warps of a block, the blocks; the counts are integers.  Results repeat bit for
// bit.
#pragma once
#include "mb_common.cuh"
#include "quantize.cuh"

namespace mb {
namespace router {

constexpr int MAX_EXPERTS = 1024;
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_PARTS = 256;      // blocks that sum up the balance, at most
constexpr int MAX_K = 64;

struct RouteArgs {
  const void *logits;
  int64_t ld;          // between rows of logits
  int T, E, k, normalize;
  float *weights;      // [T, k]
  int *experts;        // [T, k]
  const float *grad;   // [T, k]
  void *dlogits;       // [T, E]
};

struct BalanceArgs {
  const void *logits;
  int64_t ld;
  int T, E, k;
  const int *experts;      // [T, k]
  const uint8_t *mask;     // [T] or null: 0 leaves a token out
  float *part_p;           // [parts, E]
  int *part_c;             // [parts, E + 1]: counts, tokens
  int parts;
  float *loss;
  int *counts, *tokens;    // [E], one
  const float *grad;       // one
  void *dlogits;           // [T, E]
};

// Lane's score i of a row is expert slot(i): V neighbours at a time, so that a lane
// loads whole words.  V goes by E alone, and rows off such words (AL false) are loaded
// score by score into the same places: sums have one order whatever the layout.
template <int V> __device__ __forceinline__ int slot(int i, int lane) { return (i / V) * 32 * V + lane * V + i % V; }

// A row's scores, -inf past E.
template <class T, int NV, int V, bool AL>
__device__ __forceinline__ void load_scores(const T *row, int E, int lane, float (&x)[NV]) {
#pragma unroll
  for (int i = 0; i < NV; i += V) {
    const int e = slot<V>(i, lane);
    if constexpr (V == 1 || !AL) {
#pragma unroll
      for (int v = 0; v < V; ++v) x[i + v] = e + v < E ? to_f32(row[e + v]) : -INFINITY;
    } else {
      T t[V];
      constexpr int B = V * (int)sizeof(T);
      if (e < E) {   // E is a multiple of V
        if constexpr (B == 16) *reinterpret_cast<uint4 *>(t) = *reinterpret_cast<const uint4 *>(row + e);
        else if constexpr (B == 8) *reinterpret_cast<uint2 *>(t) = *reinterpret_cast<const uint2 *>(row + e);
        else *reinterpret_cast<uint32_t *>(t) = *reinterpret_cast<const uint32_t *>(row + e);
      }
#pragma unroll
      for (int v = 0; v < V; ++v) x[i + v] = e < E ? to_f32(t[v]) : -INFINITY;
    }
  }
}
template <class T, int NV, int V, bool AL>
__device__ __forceinline__ void store_scores(T *row, int E, int lane, const float (&x)[NV]) {
#pragma unroll
  for (int i = 0; i < NV; i += V) {
    const int e = slot<V>(i, lane);
    if (e >= E) continue;
    T t[V];
#pragma unroll
    for (int v = 0; v < V; ++v) t[v] = Elem<T>::store(x[i + v]);
    constexpr int B = V * (int)sizeof(T);
    if constexpr (V == 1 || !AL) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (e + v < E) row[e + v] = t[v];
    } else if constexpr (B == 16) *reinterpret_cast<uint4 *>(row + e) = *reinterpret_cast<uint4 *>(t);
    else if constexpr (B == 8) *reinterpret_cast<uint2 *>(row + e) = *reinterpret_cast<uint2 *>(t);
    else *reinterpret_cast<uint32_t *>(row + e) = *reinterpret_cast<uint32_t *>(t);
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// Order-preserving bits of a score: equal zeros, NaN above everything, 0 below everything.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);   // -0 becomes 0
  return x != x ? 0xffffffffu : (b & 0x80000000u ? ~b : b | 0x80000000u);
}
constexpr uint32_t kNever = 0x007fffffu;         // order_bits(-inf)
__device__ __forceinline__ float from_order_bits(uint32_t o) {
  return __uint_as_float(o == 0xffffffffu ? 0x7fc00000u : (o & 0x80000000u ? o ^ 0x80000000u : ~o));
}

// The row's largest score, or 0 when there is no number above -inf (a base of exponentials).
template <int NV> __device__ __forceinline__ float base_of(const float (&x)[NV]) {
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) m = fmaxf(m, x[i]);
  m = from_order_bits(__reduce_max_sync(0xffffffffu, order_bits(m)));
  return m == -INFINITY ? 0.f : m;
}
// exp(x - base) in place, and 1 / their sum over the row (0 for a sum of 0).
template <int NV> __device__ __forceinline__ float exponentials(float (&x)[NV]) {
  const float base = base_of(x);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    x[i] = expf(x[i] - base);
    s += x[i];
  }
  s = warp_sum(s);
  return s == 0.f ? 0.f : __fdividef(1.f, s);
}

template <class T, int NV, int V, bool AL>
__global__ void __launch_bounds__(THREADS) route_kernel(const RouteArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_trigger();
  pdl_wait();
  for (int64_t t = (int64_t)blockIdx.x * WARPS + warp; t < a.T; t += (int64_t)gridDim.x * WARPS) {
    float x[NV];
    load_scores<T, NV, V, AL>(static_cast<const T *>(a.logits) + t * a.ld, a.E, lane, x);
    uint32_t key[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) key[i] = order_bits(x[i]);
    const float base = base_of(x);
    float total = 0.f;
    if (!a.normalize) {
#pragma unroll
      for (int i = 0; i < NV; ++i) total += expf(x[i] - base);
      total = warp_sum(total);
    }
    // k rounds: the largest key, the lowest expert that has it
    float chosen = 0.f;      // of round `lane` (and 32 + lane): exp(score - base)
    float chosen2 = 0.f, sum = 0.f;
    int id = -1, id2 = -1;
    uint32_t best = 0;
    int at = 0;
    auto scan = [&]() {
      best = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (key[i] > best) { best = key[i]; at = i; }
    };
    scan();
    for (int j = 0; j < a.k; ++j) {
      const uint32_t top = __reduce_max_sync(0xffffffffu, best);
      if (top <= kNever) break;
      const uint32_t e = __reduce_min_sync(0xffffffffu, best == top ? (uint32_t)slot<V>(at, lane) : 0xffffffffu);
      const float w = expf(from_order_bits(top) - base);
      sum += w;
      if (lane == (j & 31)) {
        if (j < 32) { chosen = w; id = (int)e; }
        else { chosen2 = w; id2 = (int)e; }
      }
      if (best == top && (uint32_t)slot<V>(at, lane) == e) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (i == at) key[i] = 0;
        scan();
      }
    }
    const float all = a.normalize ? sum : total;
    const float inv = all == 0.f ? 0.f : __fdividef(1.f, all);
    if (lane < a.k) {
      a.weights[t * a.k + lane] = chosen * inv;
      a.experts[t * a.k + lane] = id;
    }
    if (lane + 32 < a.k) {
      a.weights[t * a.k + 32 + lane] = chosen2 * inv;
      a.experts[t * a.k + 32 + lane] = id2;
    }
  }
}

template <class T, int NV, int V, bool AL>
__global__ void __launch_bounds__(THREADS) route_backward_kernel(const RouteArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_trigger();
  pdl_wait();
  for (int64_t t = (int64_t)blockIdx.x * WARPS + warp; t < a.T; t += (int64_t)gridDim.x * WARPS) {
    float x[NV], d[NV];
    load_scores<T, NV, V, AL>(static_cast<const T *>(a.logits) + t * a.ld, a.E, lane, x);
    const float inv = exponentials(x);
#pragma unroll
    for (int i = 0; i < NV; ++i) d[i] = 0.f;
    // each entry's exponential and gradient go to the lane that holds its expert
    float total = 0.f, dot = 0.f;   // of this lane's entries
    for (int j0 = 0; j0 < a.k; j0 += 32) {
      const bool on = j0 + lane < a.k;
      const int mine = on ? a.experts[t * a.k + j0 + lane] : -1;
      const float g = on ? a.grad[t * a.k + j0 + lane] : 0.f;
      const int n = min(32, a.k - j0);
      for (int j = 0; j < n; ++j) {
        const int e = __shfl_sync(0xffffffffu, mine, j);
        const float gj = __shfl_sync(0xffffffffu, g, j);
        if ((unsigned)e >= (unsigned)a.E) continue;
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (slot<V>(i, lane) == e) {
            d[i] += x[i] * gj;
            dot += x[i] * gj;
            total += x[i];
          }
      }
    }
    dot = warp_sum(dot);
    if (a.normalize) {
      // w_j = x_j / total over the entries; an expert named twice counts twice
      total = warp_sum(total);
      const float r = total == 0.f ? 0.f : __fdividef(1.f, total);
      const float mean = dot * r;
      float c[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) c[i] = 0.f;
      for (int j0 = 0; j0 < a.k; j0 += 32) {
        const int mine = j0 + lane < a.k ? a.experts[t * a.k + j0 + lane] : -1;
        const int n = min(32, a.k - j0);
        for (int j = 0; j < n; ++j) {
          const int e = __shfl_sync(0xffffffffu, mine, j);
#pragma unroll
          for (int i = 0; i < NV; ++i) c[i] += slot<V>(i, lane) == e ? 1.f : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) d[i] = c[i] == 0.f ? 0.f : (d[i] - c[i] * x[i] * mean) * r;
    } else {
      const float mean = dot * inv;
#pragma unroll
      for (int i = 0; i < NV; ++i) d[i] = (d[i] - x[i] * mean) * inv;
    }
    store_scores<T, NV, V, AL>(static_cast<T *>(a.dlogits) + t * a.E, a.E, lane, d);
  }
}

// Sums of probabilities and counts of a block's tokens.
template <class T, int NV, int V, bool AL>
__global__ void __launch_bounds__(THREADS) balance_kernel(const BalanceArgs a) {
  extern __shared__ float sums[];                            // [WARPS][E]
  int *hist = reinterpret_cast<int *>(sums + WARPS * a.E);   // [E + 1], the last one the tokens
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e <= a.E; e += THREADS) hist[e] = 0;
  __syncthreads();
  pdl_trigger();
  pdl_wait();
  float p[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) p[i] = 0.f;
  int tokens = 0;
  for (int64_t t = (int64_t)blockIdx.x * WARPS + warp; t < a.T; t += (int64_t)gridDim.x * WARPS) {
    if (a.mask && !a.mask[t]) continue;
    float x[NV];
    load_scores<T, NV, V, AL>(static_cast<const T *>(a.logits) + t * a.ld, a.E, lane, x);
    for (int j = lane; j < a.k; j += 32) {
      const int e = a.experts[t * a.k + j];
      if ((unsigned)e < (unsigned)a.E) atomicAdd(hist + e, 1);
    }
    const float inv = exponentials(x);
#pragma unroll
    for (int i = 0; i < NV; ++i) p[i] = fmaf(x[i], inv, p[i]);
    ++tokens;
  }
  if (lane == 0 && tokens) atomicAdd(hist + a.E, tokens);
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (slot<V>(i, lane) < a.E) sums[warp * a.E + slot<V>(i, lane)] = p[i];
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += THREADS) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) s += sums[w * a.E + e];
    a.part_p[(int64_t)blockIdx.x * a.E + e] = s;
  }
  for (int e = threadIdx.x; e <= a.E; e += THREADS) a.part_c[(int64_t)blockIdx.x * (a.E + 1) + e] = hist[e];
}

// The blocks' sums to counts, tokens and loss: one block, in the order of the blocks.
__global__ static void __launch_bounds__(1024) balance_finish_kernel(const BalanceArgs a) {
  __shared__ float red[32];
  __shared__ int redi[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_trigger();
  pdl_wait();
  float dot = 0.f;
  int total = 0, n = 0;
  for (int i = threadIdx.x; i < a.parts; i += 1024) n += a.part_c[(int64_t)i * (a.E + 1) + a.E];
  for (int e = threadIdx.x; e < a.E; e += 1024) {
    float s = 0.f;
    int c = 0;
    for (int i = 0; i < a.parts; ++i) {
      s += a.part_p[(int64_t)i * a.E + e];
      c += a.part_c[(int64_t)i * (a.E + 1) + e];
    }
    a.counts[e] = c;
    total += c;
    dot = fmaf((float)c, s, dot);
  }
  auto block_int = [&](int v) {
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if (lane == 0) redi[warp] = v;
    __syncthreads();
    return __reduce_add_sync(0xffffffffu, redi[lane]);
  };
  n = block_int(n);
  total = block_int(total);
  dot = warp_sum(dot);
  if (lane == 0) red[warp] = dot;
  __syncthreads();
  if (warp == 0) {
    dot = warp_sum(red[lane]);
    if (lane == 0) {
      *a.tokens = n;
      *a.loss = n == 0 || total == 0 ? 0.f : (float)((double)a.E * dot / ((double)total * n));
    }
  }
}

template <class T, int NV, int V, bool AL>
__global__ void __launch_bounds__(THREADS) balance_backward_kernel(const BalanceArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_trigger();
  pdl_wait();
  float s[NV];
  int total = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = slot<V>(i, lane);
    const int c = e < a.E ? a.counts[e] : 0;
    total += c;
    s[i] = (float)c;
  }
  total = __reduce_add_sync(0xffffffffu, total);
  const int n = *a.tokens;
  const float f = n == 0 || total == 0 ? 0.f : (float)((double)*a.grad * a.E / ((double)total * n));
#pragma unroll
  for (int i = 0; i < NV; ++i) s[i] *= f;
  for (int64_t t = (int64_t)blockIdx.x * WARPS + warp; t < a.T; t += (int64_t)gridDim.x * WARPS) {
    float x[NV];
    if (a.mask && !a.mask[t]) {
#pragma unroll
      for (int i = 0; i < NV; ++i) x[i] = 0.f;
    } else {
      load_scores<T, NV, V, AL>(static_cast<const T *>(a.logits) + t * a.ld, a.E, lane, x);
      const float inv = exponentials(x);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        x[i] *= inv;
        dot = fmaf(x[i], s[i], dot);
      }
      dot = warp_sum(dot);
#pragma unroll
      for (int i = 0; i < NV; ++i) x[i] *= s[i] - dot;
    }
    store_scores<T, NV, V, AL>(static_cast<T *>(a.dlogits) + t * a.E, a.E, lane, x);
  }
}

}  // namespace router
}  // namespace mb
