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
// A warp takes a row, NV scores a lane, in registers, and several rows at once where
// registers allow: a row is a chain of shuffles and reductions, and what it waits for
// is latency.  Exponentials, sums and gradients are fp32.  Sums over tokens have a
// fixed order (a warp's rows, the warps of a block, the blocks of a cluster, the
// clusters); the counts are integers.  Results repeat bit for bit.
//
// 65536 x 128 fp32 scores, 8 experts each: route 32.2 us and its gradient 21.6, balance
// 20.1 and 15.0 (33.5 MB of scores are 5.1 us).  The logic pipe, at half rate, binds the choice
// (83 % in use: k rounds of reductions over a warp) and is the busiest of the others (40 to
// 44 %, issue slots 60 to 62 %).
#pragma once
#include "mb_common.cuh"
#include "quantize.cuh"

namespace mb {
namespace router {

constexpr int MAX_EXPERTS = 1024;
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int CLUSTER = 8;          // blocks that sum up the balance together
constexpr int FINISH_THREADS = 512;
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
  float *part_p;           // [parts, E], a part a cluster
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

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A word of shared memory of the cluster's block `rank`.
__device__ __forceinline__ int ld_cluster_s32(const int *p, uint32_t rank) {
  uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(p)), r;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(r) : "memory");
  return v;
}
__device__ __forceinline__ float ld_cluster_f32(const float *p, uint32_t rank) {
  return __int_as_float(ld_cluster_s32(reinterpret_cast<const int *>(p), rank));
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

// exp(y) for y <= 0: CUDA states 2 + floor(1.173 |y|) units in the last place.  What rounds is the exponent
// y / ln 2, and where that is large the result is small against the row's sum; below 2^-126 it is 0.
// (expf takes three times as many instructions, a fifth of all in the kernels without a choice of experts.)
__device__ __forceinline__ float exponential(float y) { return __expf(y); }

// The row's largest score, or 0 when there is no number above -inf (a base of exponentials).
template <int NV> __device__ __forceinline__ float base_of(const float (&x)[NV]) {
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) m = fmaxf(m, x[i]);
  // signed integers in the order of the floats (fmaxf leaves NaN out: the exponential of one is NaN whatever
  // the base)
  auto flip = [](int b) { return b ^ ((b >> 31) & 0x7fffffff); };
  m = __int_as_float(flip(__reduce_max_sync(0xffffffffu, flip(__float_as_int(m)))));
  return m == -INFINITY ? 0.f : m;
}
// exp(x - base) in place, and 1 / their sum over the row (0 for a sum of 0).
template <int NV> __device__ __forceinline__ float exponentials(float (&x)[NV]) {
  const float base = base_of(x);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    x[i] = exponential(x[i] - base);
    s += x[i];
  }
  s = warp_sum(s);
  return s == 0.f ? 0.f : __fdividef(1.f, s);
}

// Rows that a warp takes at once.
template <int NV> struct Rows { static constexpr int R = NV <= 4 ? 4 : NV <= 8 ? 2 : 1; };

// A lane's keys as a queue: the largest in front, equal ones in their order.  Short
// lists are sorted once (neighbours exchanged, so equal keys keep their order), long
// ones searched again when their front has gone.
template <int NV> struct Queue {
  static constexpr bool SORTED = NV <= 4;
  uint32_t key[NV], best;
  int at, place[SORTED ? NV : 1];
  __device__ __forceinline__ void search() {
    best = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (key[i] > best) { best = key[i]; at = i; }
  }
  __device__ __forceinline__ void init(const float (&x)[NV]) {
    at = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) key[i] = order_bits(x[i]);
    if constexpr (SORTED) {
#pragma unroll
      for (int i = 0; i < NV; ++i) place[i] = i;
#pragma unroll
      for (int r = 0; r < NV; ++r)
#pragma unroll
        for (int i = r & 1; i + 1 < NV; i += 2) {
          const bool swap = key[i + 1] > key[i];
          const uint32_t a = key[i], b = key[i + 1];
          const int p = place[i], q = place[i + 1];
          key[i] = swap ? b : a;
          key[i + 1] = swap ? a : b;
          place[i] = swap ? q : p;
          place[i + 1] = swap ? p : q;
        }
      best = key[0];
      at = place[0];
    } else {
      search();
    }
  }
  __device__ __forceinline__ void pop(bool mine) {
    if constexpr (SORTED) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        key[i] = mine ? (i + 1 < NV ? key[i + 1 < NV ? i + 1 : i] : 0u) : key[i];
        place[i] = mine && i + 1 < NV ? place[i + 1 < NV ? i + 1 : i] : place[i];
      }
      best = key[0];
      at = place[0];
    } else if (mine) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (i == at) key[i] = 0;
      search();
    }
  }
};

// MANY: k above 32, a second result a lane.
template <class T, int NV, int V, bool AL, bool MANY>
__global__ void __launch_bounds__(THREADS) route_kernel(const RouteArgs a) {
  constexpr int R = MANY ? 1 : Rows<NV>::R;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_trigger();
  pdl_wait();
  for (int64_t t0 = ((int64_t)blockIdx.x * WARPS + warp) * R; t0 < a.T; t0 += (int64_t)gridDim.x * WARPS * R) {
    float x[R][NV];
#pragma unroll
    for (int r = 0; r < R; ++r)   // (rows past the last are the last again)
      load_scores<T, NV, V, AL>(static_cast<const T *>(a.logits) + min(t0 + r, (int64_t)a.T - 1) * a.ld, a.E, lane, x[r]);
    float base[R], total[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      base[r] = base_of(x[r]);
      total[r] = 0.f;
    }
    if (!a.normalize) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int i = 0; i < NV; ++i) total[r] += exponential(x[r][i] - base[r]);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) total[r] = warp_sum(total[r]);
    }
    // k rounds: the largest key, the lowest expert that has it; lane j keeps round j's
    // (its exponential is taken once at the end, not by every lane in every round).
    Queue<NV> q[R];
    uint32_t top[R], top2 = 0;
    int id[R], id2 = -1;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      q[r].init(x[r]);
      top[r] = kNever;
      id[r] = -1;
    }
    for (int j = 0; j < a.k; ++j) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, q[r].best);
        const uint32_t own = (uint32_t)slot<V>(q[r].at, lane);
        const uint32_t e = __reduce_min_sync(0xffffffffu, q[r].best == m ? own : 0xffffffffu);
        if (m > kNever) {
          if constexpr (MANY) {
            if (lane == j) { top[r] = m; id[r] = (int)e; }
            if (lane + 32 == j) { top2 = m; id2 = (int)e; }
          } else {
            top[r] = lane == j ? m : top[r];
            id[r] = lane == j ? (int)e : id[r];
          }
        }
        q[r].pop(q[r].best == m && own == e);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      // exp(-inf) for entries that name no expert
      float w = id[r] < 0 ? 0.f : exponential(from_order_bits(top[r]) - base[r]), w2 = 0.f;
      if constexpr (MANY) w2 = id2 < 0 ? 0.f : exponential(from_order_bits(top2) - base[r]);
      const float all = a.normalize ? warp_sum(w + w2) : total[r];
      const float inv = all == 0.f ? 0.f : __fdividef(1.f, all);
      const int64_t at = (t0 + r) * a.k + lane;
      if (t0 + r < a.T) {
        if (lane < a.k) {
          a.weights[at] = w * inv;
          a.experts[at] = id[r];
        }
        if (MANY && lane + 32 < a.k) {
          a.weights[at + 32] = w2 * inv;
          a.experts[at + 32] = id2;
        }
      }
    }
  }
}

// An expert's entries' gradients and their number go through shared memory, {G, n} a
// place, E places a row: lanes write their entries and read their experts.  Two
// entries with one number (each writes its lane and reads it back) are added one
// after another instead.
template <class T, int NV, int V, bool AL>
__global__ void __launch_bounds__(THREADS) route_backward_kernel(const RouteArgs a) {
  constexpr int R = Rows<NV>::R;
  extern __shared__ float2 places[];   // [WARPS][R][32 NV]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float2 *own = places + warp * (R * 32 * NV);
  pdl_trigger();
  pdl_wait();
  for (int64_t t0 = ((int64_t)blockIdx.x * WARPS + warp) * R; t0 < a.T; t0 += (int64_t)gridDim.x * WARPS * R) {
    float x[R][NV];
#pragma unroll
    for (int r = 0; r < R; ++r)   // (rows past the last are the last again)
      load_scores<T, NV, V, AL>(static_cast<const T *>(a.logits) + min(t0 + r, (int64_t)a.T - 1) * a.ld, a.E, lane, x[r]);
    int e[R], e2[R];
    float g[R], g2[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t at = min(t0 + r, (int64_t)a.T - 1) * a.k + lane;
      e[r] = lane < a.k ? a.experts[at] : -1;
      g[r] = lane < a.k ? a.grad[at] : 0.f;
      e2[r] = lane + 32 < a.k ? a.experts[at + 32] : -1;
      g2[r] = lane + 32 < a.k ? a.grad[at + 32] : 0.f;
    }
    __syncwarp();   // the last rows' places have been read
#pragma unroll
    for (int i = 0; i < R * NV; ++i) own[i * 32 + lane] = make_float2(0.f, 0.f);
    __syncwarp();
    auto put = [&](int r, int e, float g) {   // by the whole warp
      float2 *p = own + r * 32 * NV;
      const bool on = (unsigned)e < (unsigned)a.E;
      const float before = on ? p[e].y : 0.f;
      __syncwarp();
      if (on) p[e].y = (float)(lane + 1);
      __syncwarp();
      const bool alone = !on || (before == 0.f && p[e].y == (float)(lane + 1));
      if (__all_sync(0xffffffffu, alone)) {
        if (on) p[e] = make_float2(g, 1.f);
        __syncwarp();
        return;
      }
      if (on) p[e].y = before;
      __syncwarp();
      for (int l = 0; l < 32; ++l) {
        if (lane == l && on) p[e] = make_float2(p[e].x + g, p[e].y + 1.f);
        __syncwarp();
      }
    };
#pragma unroll
    for (int r = 0; r < R; ++r) put(r, e[r], g[r]);
    if (a.k > 32) {
#pragma unroll
      for (int r = 0; r < R; ++r) put(r, e2[r], g2[r]);
    }
    float inv[R], total[R], dot[R];
#pragma unroll
    for (int r = 0; r < R; ++r) inv[r] = exponentials(x[r]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      total[r] = dot[r] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const float2 p = own[r * 32 * NV + slot<V>(i, lane)];
        dot[r] = fmaf(x[r][i], p.x, dot[r]);
        total[r] = fmaf(x[r][i], p.y, total[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      dot[r] = warp_sum(dot[r]);
      if (a.normalize) {
        total[r] = warp_sum(total[r]);
        inv[r] = total[r] == 0.f ? 0.f : __fdividef(1.f, total[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float mean = dot[r] * inv[r];
      float d[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const float2 p = own[r * 32 * NV + slot<V>(i, lane)];
        // normalize: the sum goes over the entries, an expert named twice counts twice
        if (a.normalize) d[i] = p.y == 0.f ? 0.f : x[r][i] * (p.x - p.y * mean) * inv[r];
        else d[i] = x[r][i] * (p.x - mean) * inv[r];
      }
      if (t0 + r < a.T) store_scores<T, NV, V, AL>(static_cast<T *>(a.dlogits) + (t0 + r) * a.E, a.E, lane, d);
    }
  }
}

// A block's sum of integers, the same in every thread.
__device__ __forceinline__ int block_sum(int v, int *red) {
  v = __reduce_add_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = blockDim.x / 32, lane = threadIdx.x & 31;
  return __reduce_add_sync(0xffffffffu, lane < warps ? red[lane] : 0);
}
__device__ __forceinline__ float balance_loss(int E, float dot, int total, int n) {
  return n == 0 || total == 0 ? 0.f : (float)((double)E * dot / ((double)total * n));
}

// Sums of probabilities and counts of a cluster's tokens; with one cluster the loss too.
template <class T, int NV, int V, bool AL>
__global__ void __launch_bounds__(THREADS) balance_kernel(const BalanceArgs a) {
  constexpr int R = Rows<NV>::R;
  extern __shared__ float sums[];                            // [WARPS][E], then the block's in the first E
  int *hist = reinterpret_cast<int *>(sums + WARPS * a.E);   // [E + 1], the last one the tokens
  __shared__ int red[WARPS];
  __shared__ float dots[CLUSTER];
  __shared__ int totals[CLUSTER];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  for (int e = threadIdx.x; e <= a.E; e += THREADS) hist[e] = 0;
  __syncthreads();
  pdl_trigger();
  pdl_wait();
  float p[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) p[i] = 0.f;
  int tokens = 0;
  for (int64_t t0 = ((int64_t)blockIdx.x * WARPS + warp) * R; t0 < a.T; t0 += (int64_t)gridDim.x * WARPS * R) {
    float x[R][NV], inv[R];
    bool on[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      on[r] = t0 + r < a.T && (!a.mask || a.mask[t0 + r]);
#pragma unroll
      for (int i = 0; i < NV; ++i) x[r][i] = -INFINITY;
      if (on[r]) {
        load_scores<T, NV, V, AL>(static_cast<const T *>(a.logits) + (t0 + r) * a.ld, a.E, lane, x[r]);
        ++tokens;
      }
    }
    const int *ids = a.experts + t0 * a.k;
    const int entries = (int)min((int64_t)R, a.T - t0) * a.k;   // of the rows, next to one another
    for (int j = lane; j < entries; j += 32) {
      const int e = ids[j];
      bool count = (unsigned)e < (unsigned)a.E;
      if (a.mask) count = count && a.mask[t0 + j / a.k];
      if (count) atomicAdd(hist + e, 1);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) inv[r] = exponentials(x[r]);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < NV; ++i) p[i] = fmaf(x[r][i], inv[r], p[i]);   // (of a token left out all are 0)
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
    sums[e] = s;   // (this thread alone reads column e)
  }
  cluster_barrier();
  // each rank adds up its share of the experts, in the order of the ranks
  const int part = blockIdx.x / CLUSTER;
  int total = 0, n = 0;
  float dot = 0.f;
  for (int e = threadIdx.x * CLUSTER + rank; e <= a.E; e += THREADS * CLUSTER) {
    float s = 0.f;
    int c = 0;
#pragma unroll
    for (int w = 0; w < CLUSTER; ++w) {
      if (e < a.E) s += ld_cluster_f32(sums + e, w);
      c += ld_cluster_s32(hist + e, w);
    }
    if (a.parts > 1) {
      if (e < a.E) a.part_p[(int64_t)part * a.E + e] = s;
      a.part_c[(int64_t)part * (a.E + 1) + e] = c;
    } else if (e < a.E) {
      a.counts[e] = c;
      total += c;
      dot = fmaf((float)c, s, dot);
    }
  }
  if (a.parts > 1) {
    cluster_barrier();   // no block leaves while others still read its sums
    return;
  }
  if (threadIdx.x < CLUSTER) n = ld_cluster_s32(hist + a.E, threadIdx.x);
  n = block_sum(n, red);
  total = block_sum(total, red);
  // the dot products of a block's warps and of the blocks, in order
  dot = warp_sum(dot);
  __shared__ float warp_dot[WARPS];
  if (lane == 0) warp_dot[warp] = dot;
  __syncthreads();
  if (threadIdx.x == 0) {
    dot = 0.f;
    for (int w = 0; w < WARPS; ++w) dot += warp_dot[w];
    dots[0] = dot;
    totals[0] = total;
  }
  cluster_barrier();
  if (rank == 0 && threadIdx.x == 0) {
    dot = 0.f;
    total = 0;
    for (int w = 0; w < CLUSTER; ++w) {
      dot += ld_cluster_f32(dots, w);
      total += ld_cluster_s32(totals, w);
    }
    *a.tokens = n;
    *a.loss = balance_loss(a.E, dot, total, n);
  }
  cluster_barrier();
}

// The clusters' sums to counts, tokens and loss, in the order of the clusters: one block (E < FINISH_THREADS)
// or one cluster, each of its blocks a share of the experts.
__global__ static void __launch_bounds__(FINISH_THREADS) balance_finish_kernel(const BalanceArgs a) {
  __shared__ float ps[FINISH_THREADS], dots[1];
  __shared__ int cs[FINISH_THREADS], red[32], totals[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  pdl_trigger();
  pdl_wait();
  // this block's experts (the last is the tokens' count), and threads that share each one's parts
  const int E1 = a.E + 1, ranks = gridDim.x, per = (E1 + ranks - 1) / ranks, share = FINISH_THREADS / per;
  const int mine = threadIdx.x / per, e = rank * per + (threadIdx.x - mine * per);
  float s = 0.f;
  int c = 0;
  if (mine < share && e < E1) {
    const int i0 = a.parts * mine / share, i1 = a.parts * (mine + 1) / share;
#pragma unroll 4
    for (int i = i0; i < i1; ++i) {
      s += e < a.E ? a.part_p[(int64_t)i * a.E + e] : 0.f;
      c += a.part_c[(int64_t)i * E1 + e];
    }
  }
  ps[threadIdx.x] = s;
  cs[threadIdx.x] = c;
  __syncthreads();
  float dot = 0.f;
  int total = 0, n = 0;
  if (threadIdx.x < per && e < E1) {
    for (int w = 1; w < share; ++w) {
      s += ps[w * per + threadIdx.x];
      c += cs[w * per + threadIdx.x];
    }
    if (e < a.E) {
      a.counts[e] = c;
      total = c;
      dot = (float)c * s;
    } else {
      n = c;
    }
  }
  n = block_sum(n, red);
  total = block_sum(total, red);
  dot = warp_sum(dot);
  __syncthreads();
  if (lane == 0) ps[warp] = dot;
  __syncthreads();
  if (warp == 0) {
    dot = warp_sum(lane < FINISH_THREADS / 32 ? ps[lane] : 0.f);
    if (lane == 0) {
      dots[0] = dot;
      totals[0] = total;
      totals[1] = n;
    }
  }
  cluster_barrier();
  if (rank == 0 && threadIdx.x == 0) {
    dot = 0.f;
    total = n = 0;
    for (int w = 0; w < ranks; ++w) {
      dot += ld_cluster_f32(dots, w);
      total += ld_cluster_s32(totals, w);
      n += ld_cluster_s32(totals + 1, w);
    }
    *a.tokens = n;
    *a.loss = balance_loss(a.E, dot, total, n);
  }
  cluster_barrier();   // no block leaves while its sums are read
}

template <class T, int NV, int V, bool AL>
__global__ void __launch_bounds__(THREADS) balance_backward_kernel(const BalanceArgs a) {
  constexpr int R = Rows<NV>::R;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_trigger();
  pdl_wait();
  // a[e] less their mean over the experts, which cancels (the p of a row sum to 1): what is left of an
  // even load is 0, not what rounding makes of equal numbers
  float s[NV];
  int c[NV], total = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = slot<V>(i, lane);
    c[i] = e < a.E ? a.counts[e] : 0;
    total += c[i];
  }
  total = __reduce_add_sync(0xffffffffu, total);
  const int n = *a.tokens;
  const float f = n == 0 || total == 0 ? 0.f : (float)((double)*a.grad / ((double)total * n));
#pragma unroll
  for (int i = 0; i < NV; ++i) s[i] = (float)((long long)c[i] * a.E - total) * f;
  for (int64_t t0 = ((int64_t)blockIdx.x * WARPS + warp) * R; t0 < a.T; t0 += (int64_t)gridDim.x * WARPS * R) {
    float x[R][NV], inv[R], dot[R];
    bool on[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      on[r] = t0 + r < a.T && (!a.mask || a.mask[t0 + r]);
#pragma unroll
      for (int i = 0; i < NV; ++i) x[r][i] = -INFINITY;   // of a token left out: no probabilities, no gradient
      if (on[r]) load_scores<T, NV, V, AL>(static_cast<const T *>(a.logits) + (t0 + r) * a.ld, a.E, lane, x[r]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) inv[r] = exponentials(x[r]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      dot[r] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        x[r][i] *= inv[r];
        dot[r] = fmaf(x[r][i], s[i], dot[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) dot[r] = warp_sum(dot[r]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int i = 0; i < NV; ++i) x[r][i] *= s[i] - dot[r];
      if (t0 + r < a.T) store_scores<T, NV, V, AL>(static_cast<T *>(a.dlogits) + (t0 + r) * a.E, a.E, lane, x[r]);
    }
  }
}

}  // namespace router
}  // namespace mb
