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
// Sums have a fixed order and nothing is accumulated with floating-point
// atomics, so results repeat bit for bit.
#pragma once
#include "mb_common.cuh"
#include "quantize.cuh"

namespace mb {

constexpr int kMaxExperts = 1024;
constexpr int kSortBatch = 8;  // entries a lane holds at a time

struct SortParams {
  const void *ids;
  int n, E;
  int *order, *position, *offsets;
};

__device__ __forceinline__ int ld_cluster_s32(const int *p, uint32_t rank) {
  uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(p)), r;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(r) : "memory");
  return v;
}

// A counting sort in one launch of one cluster.  Each warp owns a run of
// entries and a histogram of its own in shared memory; the warps' counts are
// summed down the block, the blocks' totals across the cluster through
// distributed shared memory, and the experts' starts by a scan, which turns
// every histogram cell into the slot of that warp's next entry of that expert.
// Within a warp entries of equal experts are ranked by lane, so the order is
// stable.
template <class I>
__global__ void __launch_bounds__(1024) expert_sort_kernel(const SortParams p) {
  extern __shared__ int sm[];  // next[W][E + 1], total[E + 1], warp sums[32]
  const int W = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int B = p.E + 1;
  const int rank = blockIdx.x, ranks = gridDim.x;
  int *total = sm + W * B, *sums = total + B;
  int *h = sm + warp * B;
  const I *ids = static_cast<const I *>(p.ids);
  for (int i = threadIdx.x; i < W * B; i += blockDim.x) sm[i] = 0;
  pdl_trigger();
  pdl_wait();
  const int step = 32 * kSortBatch;
  const int per = ((p.n + ranks * W - 1) / (ranks * W) + 31) / 32 * 32;
  const int lo = (int)min((int64_t)p.n, (int64_t)(rank * W + warp) * per), hi = min(p.n, lo + per);
  int e[kSortBatch];
  auto load = [&](int i0) {
    I v[kSortBatch];
#pragma unroll
    for (int b = 0; b < kSortBatch; ++b) {
      const int i = i0 + b * 32 + lane;
      v[b] = i < hi ? ids[i] : 0;
    }
#pragma unroll
    for (int b = 0; b < kSortBatch; ++b) {
      const int i = i0 + b * 32 + lane;
      e[b] = i >= hi ? -1 : ((v[b] < 0 || v[b] >= (I)p.E) ? p.E : (int)v[b]);
    }
  };
  __syncthreads();
  for (int i0 = lo; i0 < hi; i0 += step) {
    load(i0);
#pragma unroll
    for (int b = 0; b < kSortBatch; ++b)
      if (e[b] >= 0) atomicAdd(h + e[b], 1);
  }
  __syncthreads();
  // down the block: each cell becomes the number of that expert's entries in the warps before
  for (int x = threadIdx.x; x < B; x += blockDim.x) {
    int at = 0;
    for (int w = 0; w < W; ++w) {
      const int c = sm[w * B + x];
      sm[w * B + x] = at;
      at += c;
    }
    total[x] = at;
  }
  __syncthreads();
  if (ranks > 1)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  // thread x < E (E <= blockDim.x): entries of expert x in the ranks before this
  // one, and in all; thread 0 also the dropped ones before
  const int x = threadIdx.x;
  auto total_of = [&](int bin, int r) { return ranks > 1 ? ld_cluster_s32(total + bin, r) : total[bin]; };
  int before = 0, count = 0, dropped = 0;
  if (x < p.E) {
    for (int r = 0; r < ranks; ++r) {
      const int c = total_of(x, r);
      if (r < rank) before += c;
      count += c;
    }
  }
  if (x == 0)
    for (int r = 0; r < rank; ++r) dropped += total_of(p.E, r);
  int upto = count;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  for (int w = 0; w < warp; ++w) upto += sums[w];
  if (ranks > 1)  // the others have read this block's totals
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  // total[] becomes the slot of this block's first entry of each expert
  if (x < p.E) {
    const int start = upto - count;
    total[x] = start + before;
    if (rank == 0) p.offsets[x] = start;
    if (x == p.E - 1) {
      total[p.E] = upto;  // dropped entries follow the last expert's
      if (rank == 0) p.offsets[p.E] = upto;
    }
  }
  __syncthreads();
  if (x == 0) total[p.E] += dropped;
  __syncthreads();
  const bool held = hi - lo <= step;  // e[] still holds this warp's entries
  for (int i0 = lo; i0 < hi; i0 += step) {
    if (!held) load(i0);
#pragma unroll
    for (int b = 0; b < kSortBatch; ++b) {
      const unsigned same = __match_any_sync(0xffffffffu, e[b]);
      int slot = 0;
      if (e[b] >= 0) slot = h[e[b]];
      __syncwarp();
      if (e[b] >= 0) {
        const int i = i0 + b * 32 + lane;
        if (lane == __ffs(same) - 1) h[e[b]] = slot + __popc(same);
        slot += total[e[b]] + __popc(same & ((1u << lane) - 1u));
        p.order[slot] = i;
        p.position[i] = slot;
      }
      __syncwarp();
    }
  }
}

struct RouteParams {
  int T, H, k;
  const int *position;  // [T, k]
  const int *kept;      // offsets + E: slots at or past *kept are dropped
  const void *src, *src2;
  int64_t ld_src, ld_src2;
  const void *w;        // [T, k] weights, or null for ones
  void *dst, *dst2;
  int64_t ld_dst;
  float *scale;
};

// The kernels run blocks of 256 threads, `lanes` (32, 128 or 256) of them to a
// token, so that short rows still fill warps and long ones have a block; a
// token's columns are shared out over blockIdx.y as well.
constexpr int kRouteThreads = 256;
constexpr int kEntries = 8;  // entries of a token worked on at a time

// Slots of entries j0 .. j0+7 of token t: -1 for none (past k, or a number that
// is no row of the buffer).
__device__ __forceinline__ void load_slots(const RouteParams &p, int t, int j0, int (&slot)[kEntries]) {
  const int n = p.T * p.k;
#pragma unroll
  for (int j = 0; j < kEntries; ++j) {
    const int s = j0 + j < p.k ? p.position[(int64_t)t * p.k + j0 + j] : -1;
    slot[j] = s < n ? s : -1;
  }
}

template <class T, bool AL>
__global__ void __launch_bounds__(kRouteThreads) expert_gather_kernel(const RouteParams p, int lanes) {
  constexpr int V = Vec<T>::V;
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x * (kRouteThreads / lanes) + threadIdx.x / lanes;
  if (t >= p.T) return;
  const int kept = p.kept ? *p.kept : 0;
  const T *x = static_cast<const T *>(p.src) + t * p.ld_src;
  const int v0 = blockIdx.y * lanes + threadIdx.x % lanes, dv = gridDim.y * lanes;
  for (int j0 = 0; j0 < p.k; j0 += kEntries) {
    int slot[kEntries];
    load_slots(p, t, j0, slot);
    for (int c = v0 * V; c < p.H + (AL ? 0 : V); c += dv * V) {
      Vec<T> v;
      if constexpr (AL) v = load_vec<T, AL>(x, c, p.H);
#pragma unroll
      for (int j = 0; j < kEntries; ++j) {
        if (slot[j] < 0) continue;
        T *d = static_cast<T *>(p.dst) + slot[j] * p.ld_dst;
        const int cc = c + frame<T, AL>(d);
        if constexpr (!AL) v = load_vec<T, AL>(x, cc, p.H);
        Vec<T> o = v;
        if (slot[j] >= kept) o.zero();
        store_vec(d, cc, p.H, o);
      }
    }
  }
}

// The k rows of a token are fetched together (eight 16-byte loads in flight per
// thread) and summed in order.
template <class T, class TW, bool AL>
__global__ void __launch_bounds__(kRouteThreads) expert_combine_kernel(const RouteParams p, int lanes) {
  constexpr int V = Vec<T>::V;
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x * (kRouteThreads / lanes) + threadIdx.x / lanes;
  if (t >= p.T) return;
  const int kept = p.kept ? *p.kept : 0;
  const TW *w = static_cast<const TW *>(p.w);
  T *out = static_cast<T *>(p.dst) + t * p.ld_dst;
  const int c0 = frame<T, AL>(out);
  const int v0 = blockIdx.y * lanes + threadIdx.x % lanes, dv = gridDim.y * lanes;
  for (int c = c0 + v0 * V; c < p.H; c += dv * V) {
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    for (int j0 = 0; j0 < p.k; j0 += kEntries) {
      int slot[kEntries];
      float wj[kEntries];
      load_slots(p, t, j0, slot);
      Vec<T> v[kEntries];
#pragma unroll
      for (int j = 0; j < kEntries; ++j) {
        const bool live = slot[j] >= 0 && slot[j] < kept;
        wj[j] = live ? (w ? to_f32(w[(int64_t)t * p.k + j0 + j]) : 1.f) : 0.f;
        if (live) v[j] = load_vec<T, AL>(static_cast<const T *>(p.src) + slot[j] * p.ld_src, c, p.H);
        else v[j].zero();
      }
#pragma unroll
      for (int j = 0; j < kEntries; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = fmaf(wj[j], v[j].f(i), acc[i]);
    }
    Vec<T> o;
#pragma unroll
    for (int i = 0; i < V; ++i) o.set(i, acc[i]);
    store_vec(out, c, p.H, o);
  }
}

// src = dout, src2 = y, dst = dy, dst2 = dw.  A token's lanes see its whole rows
// (blockIdx.y unused), so that the dot products are summed here.
template <class T, class TW, bool AL>
__global__ void __launch_bounds__(kRouteThreads) expert_combine_backward_kernel(const RouteParams p, int lanes) {
  constexpr int V = Vec<T>::V;
  __shared__ float part[kRouteThreads / 32][kEntries];
  pdl_trigger();
  pdl_wait();
  const int per = kRouteThreads / lanes, tb = threadIdx.x / lanes, tl = threadIdx.x % lanes;
  const int t = blockIdx.x * per + tb;
  const int kept = p.kept ? *p.kept : 0;
  const TW *w = static_cast<const TW *>(p.w);
  const T *dout = static_cast<const T *>(p.src) + t * p.ld_src;
  for (int j0 = 0; j0 < p.k; j0 += kEntries) {
    int slot[kEntries];
    float wj[kEntries], dot[kEntries];
#pragma unroll
    for (int j = 0; j < kEntries; ++j) {
      slot[j] = -1;
      dot[j] = 0.f;
    }
    if (t < p.T) {
      load_slots(p, t, j0, slot);
#pragma unroll
      for (int j = 0; j < kEntries; ++j)
        wj[j] = slot[j] >= 0 && slot[j] < kept ? to_f32(w[(int64_t)t * p.k + j0 + j]) : 0.f;
      for (int c = tl * V; c < p.H + (AL ? 0 : V); c += lanes * V) {
        Vec<T> d, y[kEntries];
        if constexpr (AL) d = load_vec<T, AL>(dout, c, p.H);
#pragma unroll
        for (int j = 0; j < kEntries; ++j) {
          if (slot[j] >= 0 && slot[j] < kept) {
            const int cc = c + frame<T, AL>(static_cast<T *>(p.dst) + slot[j] * p.ld_dst);
            y[j] = load_vec<T, AL>(static_cast<const T *>(p.src2) + slot[j] * p.ld_src2, cc, p.H);
          } else {
            y[j].zero();
          }
        }
#pragma unroll
        for (int j = 0; j < kEntries; ++j) {
          if (slot[j] < 0) continue;
          T *dy = static_cast<T *>(p.dst) + slot[j] * p.ld_dst;
          const int cc = c + frame<T, AL>(dy);
          Vec<T> o;
          o.zero();
          if (slot[j] < kept) {
            if constexpr (!AL) d = load_vec<T, AL>(dout, cc, p.H);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              dot[j] = fmaf(d.f(i), y[j].f(i), dot[j]);
              o.set(i, wj[j] * d.f(i));
            }
          }
          store_vec(dy, cc, p.H, o);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kEntries; ++j) {
#pragma unroll
      for (int m = 16; m; m >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], m);
      if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5][j] = dot[j];
    }
    __syncthreads();
    if (t < p.T && tl < kEntries && j0 + tl < p.k) {
      float sum = 0.f;
      for (int i = 0; i < lanes / 32; ++i) sum += part[tb * (lanes / 32) + i][tl];
      static_cast<TW *>(p.dst2)[(int64_t)t * p.k + j0 + tl] = Elem<TW>::store(sum);
    }
    __syncthreads();
  }
}

// Rows to int8 (see quantize.cuh): row t of src goes to the k slots of token t,
// or, with position == null, to row t.  TPR threads hold a row's vectors, up to
// HELD each, in registers between the maximum and the rounding; longer rows are
// read again (from L2).
template <class T, bool AL, int TPR>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) quantize_rows_kernel(const RouteParams p, int q_vec) {
  constexpr int V = Vec<T>::V, HELD = 4, THREADS = TPR < 256 ? 256 : TPR;
  __shared__ uint32_t part[THREADS / 32];
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x * (THREADS / TPR) + threadIdx.x / TPR, tl = threadIdx.x % TPR;
  const bool row = t < p.T;
  const T *x = static_cast<const T *>(p.src) + t * p.ld_src;
  Vec<T> v[HELD];
  uint32_t m = 0;
  auto largest = [&](const Vec<T> &a) {
#pragma unroll
    for (int i = 0; i < V; ++i) m = max(m, abs_bits(a.f(i)));
  };
  if (row) {
#pragma unroll
    for (int g = 0; g < HELD; ++g) {
      const int c = (g * TPR + tl) * V;
      if (c < p.H) v[g] = load_vec<T, AL>(x, c, p.H);
      else v[g].zero();
    }
#pragma unroll
    for (int g = 0; g < HELD; ++g) largest(v[g]);
    for (int c = (HELD * TPR + tl) * V; c < p.H; c += TPR * V) largest(load_vec<T, AL>(x, c, p.H));
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    const int w0 = threadIdx.x / TPR * (TPR / 32);
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) m = max(m, part[w0 + i]);
  }
  if (!row) return;
  const RowQuant rq(m);
  const int kept = p.kept ? *p.kept : 0, k = p.position ? p.k : 1;
  auto put = [&](int c, const Vec<T> &a) {
    union { int8_t b[V]; uint32_t w[V / 4]; } q;
#pragma unroll
    for (int i = 0; i < V; ++i) q.b[i] = rq.dead ? 0 : (int8_t)rq.q(a.f(i));
    for (int j = 0; j < k; ++j) {
      int64_t s = t;
      bool zero = false;
      if (p.position) {
        s = p.position[(int64_t)t * p.k + j];
        if (s < 0 || s >= (int64_t)p.T * p.k) continue;
        zero = s >= kept;
      }
      int8_t *d = static_cast<int8_t *>(p.dst) + s * p.ld_dst + c;
      if (q_vec && c + V <= p.H) {
        if constexpr (V == 8) *reinterpret_cast<uint2 *>(d) = zero ? make_uint2(0, 0) : make_uint2(q.w[0], q.w[1]);
        else *reinterpret_cast<uint32_t *>(d) = zero ? 0u : q.w[0];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (c + i < p.H) d[i] = zero ? 0 : q.b[i];
      }
    }
  };
#pragma unroll
  for (int g = 0; g < HELD; ++g) {
    const int c = (g * TPR + tl) * V;
    if (c < p.H) put(c, v[g]);
  }
  for (int c = (HELD * TPR + tl) * V; c < p.H; c += TPR * V) put(c, load_vec<T, AL>(x, c, p.H));
  for (int j = tl; j < k; j += TPR) {
    int64_t s = t;
    bool zero = false;
    if (p.position) {
      s = p.position[(int64_t)t * p.k + j];
      if (s < 0 || s >= (int64_t)p.T * p.k) continue;
      zero = s >= kept;
    }
    p.scale[s] = zero ? 0.f : rq.scale;
  }
}

}  // namespace mb
