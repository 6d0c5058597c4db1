// Tokens sorted by expert and back.
//
// A router gives each of T tokens k expert numbers ids[t, j] (entry i = t k + j).
// expert_sort orders the n = T k entries by expert, entries of one expert in
// their own order (stable), numbers outside [0, E) ("dropped") last:
//
//   order[slot] = i,  position[i] = slot,  offsets[e] = first slot of expert e,
//   offsets[E] = number of entries kept.
//
// `order` is a whole permutation, so every row of the sorted buffers has one
// owner: the kernels below run over tokens, read a token's row once and touch
// its k slots, and slots at or past offsets[E] hold zeros.
//
//   gather    xs[position[t, j]] = x[t]
//   combine   out[t] = sum_j w[t, j] y[position[t, j]]       (j ascending, fp32)
//   backward  dy[position[t, j]] = w[t, j] dout[t],  dw[t, j] = <dout[t], y[position[t, j]]>
//             dx[t] = sum_j dxs[position[t, j]]               (combine with w = 1)
//
// Sums have a fixed order and nothing is accumulated with atomics, so results
// repeat bit for bit.
#pragma once
#include "mb_common.cuh"
#include "quantize.cuh"

namespace mb {

constexpr int kMaxExperts = 1024;

struct SortParams {
  const void *ids;
  int n, E;
  int *order, *position, *offsets;
};

// One block, one pass per phase.
template <class I>
__global__ void __launch_bounds__(1024) expert_sort_kernel(const SortParams p) {
  extern __shared__ int sm[];  // hist[32][E + 1]
  const int W = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int B = p.E + 1;
  const I *ids = static_cast<const I *>(p.ids);
  pdl_trigger();
  pdl_wait();
  for (int i = threadIdx.x; i < W * B; i += blockDim.x) sm[i] = 0;
  __syncthreads();
  const int per = ((p.n + W - 1) / W + 31) / 32 * 32;
  const int lo = min(p.n, warp * per), hi = min(p.n, lo + per);
  int *h = sm + warp * B;
  auto bin = [&](int i) -> int {
    if (i >= hi) return -1;
    const I e = ids[i];
    return (e < 0 || e >= (I)p.E) ? p.E : (int)e;
  };
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int e = bin(i0 + lane);
    const unsigned same = __match_any_sync(0xffffffffu, e);
    if (e >= 0 && lane == __ffs(same) - 1) h[e] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int at = 0;
    for (int e = 0; e < B; ++e) {
      p.offsets[e] = at;
      for (int w = 0; w < W; ++w) {
        const int c = sm[w * B + e];
        sm[w * B + e] = at;
        at += c;
      }
    }
  }
  __syncthreads();
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int i = i0 + lane, e = bin(i);
    const unsigned same = __match_any_sync(0xffffffffu, e);
    int slot = 0;
    if (e >= 0) slot = h[e] + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (e >= 0 && lane == __ffs(same) - 1) h[e] += __popc(same);
    __syncwarp();
    if (e >= 0) {
      p.order[slot] = i;
      p.position[i] = slot;
    }
  }
}

struct RouteParams {
  int64_t T, H;
  int k;
  const int *position;  // [T, k]
  const int *kept;      // offsets + E: slots at or past *kept are dropped
  const void *src, *src2;
  int64_t ld_src, ld_src2;
  const void *w;        // [T, k] weights, or null for ones
  void *dst, *dst2;
  int64_t ld_dst;
  float *scale;
};

// Slot of entry (t, j): negative when dropped (or not a slot of the buffer).
__device__ __forceinline__ int64_t slot_of_entry(const RouteParams &p, int64_t t, int j, int kept) {
  return p.position[t * p.k + j];
}
__device__ __forceinline__ bool slot_in(const RouteParams &p, int64_t s) { return s >= 0 && s < p.T * p.k; }

template <class T, int V>
__global__ void __launch_bounds__(256) expert_gather_kernel(const RouteParams p) {
  pdl_trigger();
  pdl_wait();
  const int64_t t = blockIdx.x;
  const int kept = *p.kept;
  const T *x = static_cast<const T *>(p.src) + t * p.ld_src;
  for (int64_t c = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * V; c < p.H;
       c += (int64_t)gridDim.y * blockDim.x * V) {
    Vec<T, V> v, z;
    v.load(x + c);
    z.zero();
    for (int j = 0; j < p.k; ++j) {
      const int64_t s = slot_of_entry(p, t, j, kept);
      if (!slot_in(p, s)) continue;
      T *d = static_cast<T *>(p.dst) + s * p.ld_dst + c;
      if (s < kept) v.store(d);
      else z.store(d);
    }
  }
}

template <class T, class TW, int V>
__global__ void __launch_bounds__(256) expert_combine_kernel(const RouteParams p) {
  pdl_trigger();
  pdl_wait();
  const int64_t t = blockIdx.x;
  const int kept = min(*p.kept, (int)min(p.T * p.k, (int64_t)0x7fffffff));
  const TW *w = static_cast<const TW *>(p.w);
  for (int64_t c = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * V; c < p.H;
       c += (int64_t)gridDim.y * blockDim.x * V) {
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    for (int j = 0; j < p.k; ++j) {
      const int64_t s = slot_of_entry(p, t, j, kept);
      if (s < 0 || s >= kept) continue;
      const float wj = w ? to_f32(w[t * p.k + j]) : 1.f;
      Vec<T, V> v;
      v.load(static_cast<const T *>(p.src) + s * p.ld_src + c);
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = fmaf(wj, v.f(i), acc[i]);
    }
    Vec<T, V> o;
#pragma unroll
    for (int i = 0; i < V; ++i) o.set(i, acc[i]);
    o.store(static_cast<T *>(p.dst) + t * p.ld_dst + c);
  }
}

// src = dout, src2 = y, dst = dy, dst2 = dw.  One block per token.
template <class T, class TW, int V>
__global__ void __launch_bounds__(256) expert_combine_backward_kernel(const RouteParams p) {
  __shared__ float part[8];
  pdl_trigger();
  pdl_wait();
  const int64_t t = blockIdx.x;
  const int kept = min(*p.kept, (int)min(p.T * p.k, (int64_t)0x7fffffff));
  const TW *w = static_cast<const TW *>(p.w);
  const T *dout = static_cast<const T *>(p.src) + t * p.ld_src;
  for (int j = 0; j < p.k; ++j) {
    const int64_t s = slot_of_entry(p, t, j, kept);
    const bool in = slot_in(p, s), live = in && s < kept;
    const float wj = live ? to_f32(w[t * p.k + j]) : 0.f;
    float dot = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * V; c < p.H; c += (int64_t)blockDim.x * V) {
      Vec<T, V> d, y, o;
      o.zero();
      if (live) {
        d.load(dout + c);
        y.load(static_cast<const T *>(p.src2) + s * p.ld_src2 + c);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          dot = fmaf(d.f(i), y.f(i), dot);
          o.set(i, wj * d.f(i));
        }
      }
      if (in) o.store(static_cast<T *>(p.dst) + s * p.ld_dst + c);
    }
    for (int m = 16; m; m >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, m);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = dot;
    __syncthreads();
    if (threadIdx.x == 0) {
      float sum = 0.f;
      for (int i = 0; i < (int)(blockDim.x >> 5); ++i) sum += part[i];
      static_cast<TW *>(p.dst2)[t * p.k + j] = Elem<TW>::store(sum);
    }
    __syncthreads();
  }
}

// Rows to int8 (see quantize.cuh): row t of src goes to the k slots of token t,
// or, with position == null, to row t.
template <class T, int V>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const RouteParams p) {
  __shared__ uint32_t part[8];
  pdl_trigger();
  pdl_wait();
  const int64_t t = blockIdx.x;
  const T *x = static_cast<const T *>(p.src) + t * p.ld_src;
  uint32_t m = 0;
  for (int64_t c = (int64_t)threadIdx.x * V; c < p.H; c += (int64_t)blockDim.x * V) {
    Vec<T, V> v;
    v.load(x + c);
#pragma unroll
    for (int i = 0; i < V; ++i) m = max(m, abs_bits(v.f(i)));
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  __syncthreads();
  for (int i = 0; i < 8; ++i) m = max(m, part[i]);
  const RowQuant rq(m);
  const int kept = p.kept ? *p.kept : 0;
  const int k = p.position ? p.k : 1;
  for (int64_t c = (int64_t)threadIdx.x * V; c < p.H; c += (int64_t)blockDim.x * V) {
    Vec<T, V> v;
    v.load(x + c);
    int8_t q[V];
#pragma unroll
    for (int i = 0; i < V; ++i) q[i] = rq.dead ? 0 : (int8_t)rq.q(v.f(i));
    for (int j = 0; j < k; ++j) {
      const int64_t s = p.position ? slot_of_entry(p, t, j, kept) : t;
      if (p.position && !slot_in(p, s)) continue;
      int8_t *d = static_cast<int8_t *>(p.dst) + s * p.ld_dst + c;
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] = (p.position && s >= kept) ? 0 : q[i];
    }
  }
  if (threadIdx.x < k) {
    for (int j = threadIdx.x; j < k; j += blockDim.x) {
      const int64_t s = p.position ? slot_of_entry(p, t, j, kept) : t;
      if (!p.position || slot_in(p, s)) p.scale[s] = (p.position && s >= kept) ? 0.f : rq.scale;
    }
  }
}

}  // namespace mb
