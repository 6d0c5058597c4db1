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
//
// All but the sort are bound by HBM: they move each row once, 16 bytes a thread,
// with as many rows in flight as registers allow.  Measured on B200 at 8192
// tokens x 8 experts each, 4096 bf16 columns (a copy moves 6.54 TB/s): gather
// 104.5 us (5.8 TB/s), gather to int8 57.7 us (5.8), combine 95.5 us (6.3), its
// gradient 184 us (6.2); the sort of those 65536 entries 11 us, of 32 entries
// 2.2 us, where launch and latency are all there is.
#pragma once
#include "mb_common.cuh"
#include "quantize.cuh"

namespace mb {

constexpr int kMaxExperts = 1024;
constexpr int kSortBatch = 8;   // entries a lane holds at a time
constexpr int kSortRanks = 16;  // blocks of a cluster, at most

struct SortParams {
  const void *ids;
  int n, E;
  int *order, *position, *offsets;
};

__device__ __forceinline__ int ld_cluster_s32(const int *p, uint32_t rank) {
  uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(p)), r;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(r));  // ordered by the barriers' assembly
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
  const int B = p.E + 1, S = B | 1;  // an odd pitch spreads a column over the banks
  const int rank = blockIdx.x, ranks = gridDim.x;
  int *total = sm + W * S, *sums = total + B;
  int *h = sm + warp * S;
  const I *ids = static_cast<const I *>(p.ids);
  for (int i = threadIdx.x; i < W * S; i += blockDim.x) sm[i] = 0;
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
  // Counts the batch into h and leaves each entry's place among the warp's
  // entries of its expert counted so far (plus what h held) in at[].
  // The lanes of equal experts are found by a vote per bit of the number, several
  // times faster than the match instruction (65536 entries: 18.8 us with it).
  int at[kSortBatch];
  const int bits = 32 - __clz(p.E);
  auto count_batch = [&](int i0) {
#pragma unroll
    for (int b = 0; b < kSortBatch; ++b) {
      if (i0 + b * 32 >= hi) break;  // e[] holds no entry from here on
      unsigned same = __ballot_sync(0xffffffffu, e[b] >= 0);
      for (int i = 0; i < bits; ++i) {
        const bool one = (e[b] >> i) & 1;
        const unsigned m = __ballot_sync(0xffffffffu, one);
        same &= one ? m : ~m;
      }
      const int base = e[b] >= 0 ? h[e[b]] : 0;
      __syncwarp();
      if (e[b] >= 0 && lane == __ffs(same) - 1) h[e[b]] = base + __popc(same);
      __syncwarp();
      at[b] = base + __popc(same & ((1u << lane) - 1u));
    }
  };
  __syncthreads();
  for (int i0 = lo; i0 < hi; i0 += step) {
    load(i0);
    count_batch(i0);
  }
  __syncthreads();
  // down the block: each cell becomes the number of that expert's entries in the
  // warps before (a thread scans a column, eight cells in flight)
  for (int x = threadIdx.x; x < B; x += blockDim.x) {
    int upto = 0;
    for (int w0 = 0; w0 < W; w0 += 8) {
      int c[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = w0 + i < W ? sm[(w0 + i) * S + x] : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (w0 + i < W) sm[(w0 + i) * S + x] = upto;
        upto += c[i];
      }
    }
    total[x] = upto;
  }
  __syncthreads();
  if (ranks > 1)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  // thread x < E (E <= blockDim.x): entries of expert x in the ranks before this
  // one, and in all; thread 0 also the dropped ones before
  const int x = threadIdx.x;
  int before = 0, count = 0, dropped = 0;
  if (ranks == 1) {
    if (x < p.E) count = total[x];
  } else {
    // the ranks' totals are fetched together: one round trip, not `ranks` of them
    auto add = [&](int bin, int &pre, int &all) {
      int c[kSortRanks];
#pragma unroll
      for (int r = 0; r < kSortRanks; ++r) c[r] = ld_cluster_s32(total + bin, r < ranks ? r : 0);
#pragma unroll
      for (int r = 0; r < kSortRanks; ++r) {
        if (r < rank) pre += c[r];
        if (r < ranks) all += c[r];
      }
    };
    int unused = 0;
    if (x < p.E) add(x, before, count);
    if (x == 0) add(p.E, dropped, unused);
  }
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
  auto place = [&](int i0) {
#pragma unroll
    for (int b = 0; b < kSortBatch; ++b) {
      if (e[b] < 0) continue;
      const int i = i0 + b * 32 + lane;
      p.order[at[b]] = i;
      p.position[i] = at[b];
    }
  };
  if (lo >= hi) return;  // a warp without entries has loaded none
  if (hi - lo <= step) {  // e[] and at[] still hold the warp's entries
#pragma unroll
    for (int b = 0; b < kSortBatch; ++b)
      if (e[b] >= 0) at[b] += total[e[b]] + h[e[b]];
    place(lo);
  } else {
    for (int i0 = lo; i0 < hi; i0 += step) {
      load(i0);
      count_batch(i0);
#pragma unroll
      for (int b = 0; b < kSortBatch; ++b)
        if (e[b] >= 0) at[b] += total[e[b]];
      place(i0);
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

// The kernels run blocks of 256 threads, `lanes` (16, 32, 128 or 256; whole warps
// in combine's gradient) of them to a token, so that short rows still fill warps
// and long ones have a block; a token's columns are shared out over blockIdx.y
// as well.
constexpr int kRouteThreads = 256;
// A token's entries are worked on NE (2, 4 or 8) at a time: the rows of a batch
// are in flight together, a batch wider than k is spent on nothing (k = 2 in
// batches of 8: combine of 8192 tokens of 4096 bf16 84 us against 36), and a
// batch's registers cost threads.  Measured at k = 8: combine of aligned bf16 rows
// 95.7 us in eights and 102 in fours, of fp32 rows 219 and 190, of unaligned bf16
// rows 170 and 159; its gradient 191 and 183.

// Slots of entries j0 .. j0+NE-1 of token t: -1 for none (past k, or a number that
// is no row of the buffer).
template <int NE>
__device__ __forceinline__ void load_slots(const RouteParams &p, int t, int j0, int (&slot)[NE]) {
  const int n = p.T * p.k;
#pragma unroll
  for (int j = 0; j < NE; ++j) {
    const int s = j0 + j < p.k ? p.position[(int64_t)t * p.k + j0 + j] : -1;
    slot[j] = s < n ? s : -1;
  }
}

template <class T> __device__ __forceinline__ T *row_of(void *base, int64_t r, int64_t ld) {
  return static_cast<T *>(base) + r * ld;
}
template <class T> __device__ __forceinline__ const T *row_of(const void *base, int64_t r, int64_t ld) {
  return static_cast<const T *>(base) + r * ld;
}

// AL below: every row starts on 16 bytes and holds whole vectors.
//
// The elements of a row that no whole vector of its frame holds: the first `head`
// ones and those from `tail` on, fewer than two vectors of them.  The kernels
// below give them a lane each after the vectors; taken by the vectors' own
// threads, one by one, they cost more than the row (combine of 8192 x 8 x 4099
// bf16: 243 us).
struct Edges {
  int head, tail, H;
  __device__ __forceinline__ Edges(int frame, int H_, int V) : H(H_) {
    head = frame < 0 ? min(V + frame, H) : 0;
    tail = max(head, frame + (H - frame) / V * V);
  }
  __device__ __forceinline__ int count() const { return head + H - tail; }
  __device__ __forceinline__ int column(int e) const { return e < head ? e : tail + e - head; }
};

template <class T, int NE, bool AL>
__global__ void __launch_bounds__(kRouteThreads) expert_gather_kernel(const RouteParams p, int lanes) {
  constexpr int V = Vec<T>::V;
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x * (kRouteThreads / lanes) + threadIdx.x / lanes, tl = threadIdx.x % lanes;
  if (t >= p.T) return;
  const int kept = p.kept ? *p.kept : 0;
  const T *x = row_of<T>(p.src, t, p.ld_src);
  const int v0 = blockIdx.y * lanes + tl, dv = gridDim.y * lanes;
  for (int j0 = 0; j0 < p.k; j0 += NE) {
    int slot[NE];
    load_slots(p, t, j0, slot);
    for (int c = v0 * V; c < p.H + (AL ? 0 : V); c += dv * V) {
      Vec<T> v;
      if constexpr (AL) v = load16<T, AL>(x + c);
#pragma unroll
      for (int j = 0; j < NE; ++j) {
        if (slot[j] < 0) continue;
        T *d = row_of<T>(p.dst, slot[j], p.ld_dst);
        const int cc = c + frame<T, AL>(d);
        if (!AL && (cc < 0 || cc + V > p.H)) continue;
        if constexpr (!AL) v = load16<T, AL>(x + cc);
        Vec<T> o = v;
        if (slot[j] >= kept) o.zero();
        *reinterpret_cast<uint4 *>(d + cc) = o.u.q;
      }
    }
    if constexpr (!AL) {
      if (blockIdx.y) continue;
#pragma unroll
      for (int j = 0; j < NE; ++j) {
        if (slot[j] < 0) continue;
        T *d = row_of<T>(p.dst, slot[j], p.ld_dst);
        const Edges g(frame<T, AL>(d), p.H, V);
        for (int e = tl; e < g.count(); e += lanes) {
          const int c = g.column(e);
          d[c] = slot[j] < kept ? x[c] : Elem<T>::store(0.f);
        }
      }
    }
  }
}

// The rows of a token are fetched together (NE 16-byte loads in flight per
// thread) and summed in order.
template <class T, class TW, int NE, bool AL>
__global__ void __launch_bounds__(kRouteThreads) expert_combine_kernel(const RouteParams p, int lanes) {
  constexpr int V = Vec<T>::V;
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x * (kRouteThreads / lanes) + threadIdx.x / lanes, tl = threadIdx.x % lanes;
  if (t >= p.T) return;
  const int kept = p.kept ? *p.kept : 0;
  const TW *w = static_cast<const TW *>(p.w);
  T *out = row_of<T>(p.dst, t, p.ld_dst);
  const int c0 = frame<T, AL>(out);
  const int v0 = blockIdx.y * lanes + tl, dv = gridDim.y * lanes;
  int slot[NE];
  float wj[NE];
  auto entries = [&](int j0) {
    load_slots(p, t, j0, slot);
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      if (slot[j] >= kept) slot[j] = -1;
      wj[j] = slot[j] < 0 ? 0.f : w ? to_f32(w[(int64_t)t * p.k + j0 + j]) : 1.f;
    }
  };
  if (p.k <= NE) entries(0);
  for (int c = c0 + v0 * V; AL ? c < p.H : c + V <= p.H; c += dv * V) {
    if (!AL && c < 0) continue;
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    for (int j0 = 0; j0 < p.k; j0 += NE) {
      if (p.k > NE) entries(j0);
      Vec<T> v[NE];
      uint4 next[AL ? 1 : NE];
#pragma unroll
      for (int j = 0; j < NE; ++j) {
        const T *y = row_of<T>(p.src, max(slot[j], 0), p.ld_src) + c;
        const uint32_t off = AL ? 0u : (uint32_t)(reinterpret_cast<uintptr_t>(y) & 15);
        const char *word = reinterpret_cast<const char *>(y) - off;
        v[j].u.q = load_once<!AL>(word, slot[j] >= 0);
        if constexpr (!AL) next[j] = load_once<true>(word + 16, slot[j] >= 0 && off);
      }
      if constexpr (!AL) {
#pragma unroll
        for (int j = 0; j < NE; ++j)
          v[j].u.q = cut16(v[j].u.q, next[j],
                           (uint32_t)reinterpret_cast<uintptr_t>(row_of<T>(p.src, max(slot[j], 0), p.ld_src) + c) & 15);
      }
#pragma unroll
      for (int j = 0; j < NE; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = fmaf(wj[j], v[j].f(i), acc[i]);
    }
    Vec<T> o;
#pragma unroll
    for (int i = 0; i < V; ++i) o.set(i, acc[i]);
    *reinterpret_cast<uint4 *>(out + c) = o.u.q;
  }
  if constexpr (!AL) {
    if (blockIdx.y) return;
    const Edges g(c0, p.H, V);
    for (int e = tl; e < g.count(); e += lanes) {
      const int c = g.column(e);
      float acc = 0.f;
      for (int j0 = 0; j0 < p.k; j0 += NE) {
        if (p.k > NE) entries(j0);
        float y[NE];
#pragma unroll
        for (int j = 0; j < NE; ++j) y[j] = slot[j] >= 0 ? to_f32(row_of<T>(p.src, slot[j], p.ld_src)[c]) : 0.f;
#pragma unroll
        for (int j = 0; j < NE; ++j) acc = fmaf(wj[j], y[j], acc);
      }
      out[c] = Elem<T>::store(acc);
    }
  }
}

// src = dout, src2 = y, dst = dy, dst2 = dw.  A token's lanes see its whole rows
// (blockIdx.y unused), so that the dot products are summed here: by thread along
// the row, then over lanes and warps in a fixed order.  With aligned rows dout is
// read once for the NE entries of a batch; otherwise every entry has a vector
// frame of its own (its row of dy's) and is worked on alone.
template <class T, class TW, int NE, bool AL>
__global__ void __launch_bounds__(kRouteThreads) expert_combine_backward_kernel(const RouteParams p, int lanes) {
  constexpr int V = Vec<T>::V;
  __shared__ float part[kRouteThreads / 32][NE];
  pdl_trigger();
  pdl_wait();
  const int per = kRouteThreads / lanes, tb = threadIdx.x / lanes, tl = threadIdx.x % lanes;
  const int t = blockIdx.x * per + tb;
  const int kept = p.kept ? *p.kept : 0;
  const TW *w = static_cast<const TW *>(p.w);
  const T *dout = row_of<T>(p.src, t, p.ld_src);
  // The edge elements of entry slot s with weight ws; returns their share of its dot product.
  auto edges = [&](int s, float ws, int frame_) {
    T *dy = row_of<T>(p.dst, s, p.ld_dst);
    const T *y = row_of<T>(p.src2, s, p.ld_src2);
    const Edges g(frame_, p.H, V);
    float sum = 0.f;
    for (int e = tl; e < g.count(); e += lanes) {
      const int c = g.column(e);
      const float d = to_f32(dout[c]);
      dy[c] = Elem<T>::store(s < kept ? ws * d : 0.f);
      if (s < kept) sum = fmaf(d, to_f32(y[c]), sum);
    }
    return sum;
  };
  auto warp_sum = [](float v) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
  };
  for (int j0 = 0; j0 < p.k; j0 += NE) {
    int slot[NE];
    float wj[NE];
#pragma unroll
    for (int j = 0; j < NE; ++j) slot[j] = -1;
    if (t < p.T) load_slots(p, t, j0, slot);
#pragma unroll
    for (int j = 0; j < NE; ++j)
      wj[j] = slot[j] >= 0 && slot[j] < kept ? to_f32(w[(int64_t)t * p.k + j0 + j]) : 0.f;
    if constexpr (AL) {
      float dot[NE];
#pragma unroll
      for (int j = 0; j < NE; ++j) dot[j] = 0.f;
      if (t < p.T) {
        for (int c = tl * V; c < p.H; c += lanes * V) {
          const Vec<T> d = load16<T, AL>(dout + c);
          Vec<T> y[NE];
#pragma unroll
          for (int j = 0; j < NE; ++j) {
            y[j].u.q = load_once(row_of<T>(p.src2, max(slot[j], 0), p.ld_src2) + c, slot[j] >= 0 && slot[j] < kept);
          }
#pragma unroll
          for (int j = 0; j < NE; ++j) {
            if (slot[j] < 0) continue;
            Vec<T> o;
            o.zero();
            if (slot[j] < kept) {
#pragma unroll
              for (int i = 0; i < V; ++i) {
                dot[j] = fmaf(d.f(i), y[j].f(i), dot[j]);
                o.set(i, wj[j] * d.f(i));
              }
            }
            *reinterpret_cast<uint4 *>(row_of<T>(p.dst, slot[j], p.ld_dst) + c) = o.u.q;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NE; ++j) {
        dot[j] = warp_sum(dot[j]);
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5][j] = dot[j];
      }
    } else {
#pragma unroll 1
      for (int j = 0; j < NE; ++j) {
        const int s = t < p.T && j0 + j < p.k ? p.position[(int64_t)t * p.k + j0 + j] : -1;
        float dot = 0.f;
        if (s >= 0 && s < p.T * p.k) {
          T *dy = row_of<T>(p.dst, s, p.ld_dst);
          const T *y = row_of<T>(p.src2, s, p.ld_src2);
          const float ws = s < kept ? to_f32(w[(int64_t)t * p.k + j0 + j]) : 0.f;
          const int c0 = frame<T, AL>(dy);
#pragma unroll 4
          for (int c = c0 + tl * V; c + V <= p.H; c += lanes * V) {
            if (c < 0) continue;
            Vec<T> o;
            o.zero();
            if (s < kept) {
              const Vec<T> d = load16<T, AL>(dout + c), yv = load16<T, AL>(y + c);
#pragma unroll
              for (int i = 0; i < V; ++i) {
                dot = fmaf(d.f(i), yv.f(i), dot);
                o.set(i, ws * d.f(i));
              }
            }
            *reinterpret_cast<uint4 *>(dy + c) = o.u.q;
          }
          dot += edges(s, ws, c0);
        }
        dot = warp_sum(dot);
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5][j] = dot;
      }
    }
    __syncthreads();
    if (t < p.T && tl < NE && j0 + tl < p.k) {
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
// read again (from L2).  It is bound by how much of its loads an SM can keep in
// flight between the barriers and roundings (issue slots 77 % in use), and by HBM
// behind that: 16384 x 8192 bf16 72.8 us (5.5 TB/s) with four vectors a thread,
// 87 with two and twice the threads, 79 with eight and half of them; copies into
// shared memory ahead of a persistent block gave 79.
template <class T, bool AL, int TPR, int HELD>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR, (HELD > 4 ? 768 : HELD > 2 || !AL ? 1280 : 2048) / (TPR < 256 ? 256 : TPR)) quantize_rows_kernel(const RouteParams p, int q_vec) {
  constexpr int V = Vec<T>::V, THREADS = TPR < 256 ? 256 : TPR;
  __shared__ uint32_t part[THREADS / 32];
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x * (THREADS / TPR) + threadIdx.x / TPR, tl = threadIdx.x % TPR;
  const bool row = t < p.T;
  const T *x = static_cast<const T *>(p.src) + t * p.ld_src;
  Vec<T> v[HELD];
  MaxAbs<T> largest;
  if (row) {
    if constexpr (AL) {
#pragma unroll
      for (int g = 0; g < HELD; ++g) {
        const int c = (g * TPR + tl) * V;
        if (c < p.H) v[g] = load_vec<T, AL>(x, c, p.H);
        else v[g].zero();
      }
    } else {
      // the aligned words that hold elements of the row, all on their way before
      // the first is cut (397 x 10609 fp32 17.6 to 12.7 us; 7601 x 5403 bf16 42.8 to
      // 38.8, aligned 30.8); elements past the row's end count as zeros
      const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(x) & 15);
      const char *word = reinterpret_cast<const char *>(x) - off;
      const int past = (int)((16 - off) / sizeof(T));  // elements of a vector in its first word
      uint4 next[HELD];
#pragma unroll
      for (int g = 0; g < HELD; ++g) {
        const int i = g * TPR + tl;
        v[g].u.q = load_once<true>(word + (int64_t)i * 16, i * V < p.H);
        next[g] = load_once<true>(word + (int64_t)i * 16 + 16, off && i * V + past < p.H);
      }
#pragma unroll
      for (int g = 0; g < HELD; ++g) {
        v[g].u.q = cut16(v[g].u.q, next[g], off);
        keep_first(v[g], p.H - (g * TPR + tl) * V);
      }
    }
#pragma unroll
    for (int g = 0; g < HELD; ++g) largest.add(v[g]);
    for (int c = (HELD * TPR + tl) * V; c < p.H; c += TPR * V) largest.add(load_vec<T, AL>(x, c, p.H));
  }
  uint32_t m = largest.bits();
  if constexpr (TPR < 32) {
#pragma unroll
    for (int d = TPR / 2; d; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
  } else {
    m = __reduce_max_sync(0xffffffffu, m);
  }
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    const int w0 = threadIdx.x / TPR * (TPR / 32);
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) m = max(m, part[w0 + i]);
  }
  if (!row) return;
  const RowQuant<T> rq(m);
  const int kept = p.kept ? *p.kept : 0, k = p.position ? p.k : 1;
  auto put = [&](int c, const Vec<T> &a) {
    union { int8_t b[V]; uint32_t w[V / 4]; } q;
    float f[V];
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = a.f(i);
    rq.q(f, q.w);
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
    p.scale[s] = zero ? 0.f : RowQuant<T>::scale(m);
  }
}

}  // namespace mb
