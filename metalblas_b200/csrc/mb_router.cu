// C ABI of the router and its balance loss (router.cuh).
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "mb_host.cuh"
#include "mb_common.cuh"
#include "router.cuh"

using namespace mb;
using namespace mb::host;

namespace {

using namespace mb::router;

int check(const char *what, int dtype, int64_t T, int64_t E, int64_t k, int64_t ld, const void *logits) {
  if (dtype != MB_F32 && dtype != MB_F16 && dtype != MB_BF16)
    return fail(MB_ERR_UNSUPPORTED, "%s: scores must be fp32, fp16 or bf16, got %d", what, dtype);
  if (T < 0 || k < 0) return fail(MB_ERR_INVALID, "%s: negative extent", what);
  if (E < 1 || E > MAX_EXPERTS) return fail(MB_ERR_INVALID, "%s: %lld experts (1 to %d)", what, (long long)E, MAX_EXPERTS);
  if (T > 0x7fff0000ll || (k && T > 0x7fff0000ll / k)) return fail(MB_ERR_INVALID, "%s: tokens * k must stay below 2^31 - 2^16", what);
  if (T > 1 && ld < E) return fail(MB_ERR_INVALID, "%s: rows of logits overlap", what);
  if (T > 0 && !logits) return fail(MB_ERR_INVALID, "%s: null logits", what);
  return MB_OK;
}

// f(element tag, scores a lane, neighbours among them, whether they are one word in memory).
template <class F>
int by_shape(int dtype, int64_t E, const void *p, int64_t ld, const void *p2, F &&f) {
  using std::integral_constant;
  auto of = [&](auto *tag) {
    auto go = [&](auto nv, auto v) {
      constexpr int V = decltype(v)::value;
      const uintptr_t at = reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(p2);
      const bool al = E % V == 0 && ld % V == 0 && at % (V * sizeof(*tag)) == 0;
      return al ? f(tag, nv, v, std::true_type()) : f(tag, nv, v, std::false_type());
    };
    if (E <= 32) return go(integral_constant<int, 1>(), integral_constant<int, 1>());
    if (E <= 64) return go(integral_constant<int, 2>(), integral_constant<int, 2>());
    if (E <= 128) return go(integral_constant<int, 4>(), integral_constant<int, 4>());
    if (E <= 256) return go(integral_constant<int, 8>(), integral_constant<int, 4>());
    if (E <= 512) return go(integral_constant<int, 16>(), integral_constant<int, 4>());
    return go(integral_constant<int, 32>(), integral_constant<int, 4>());
  };
  switch (dtype) {
    case MB_F32: return of((float *)nullptr);
    case MB_F16: return of((__half *)nullptr);
    default: return of((__nv_bfloat16 *)nullptr);
  }
}

// Rows that a warp takes at once (Rows in router.cuh), by the experts.
int rows_at_once(int64_t E) { return E <= 128 ? 4 : E <= 256 ? 2 : 1; }
// Blocks of T rows: resident ones, each through its share.
unsigned row_grid(int64_t T, int rows) {
  return (unsigned)std::min<int64_t>(ceil_div(T, WARPS * rows), (int64_t)device_sms() * 6);
}
// Clusters that sum up the balance of T tokens.  One makes the loss in the same launch: up to two
// rounds of its rows it is as fast as several and a second launch (64 experts, 512 tokens 6.2 and 6.0 us,
// 1000 tokens 9.5 and 5.8, 4096 tokens 28.7 and 7.1; 256 experts, 256 tokens 6.0 and 6.3).
int64_t parts_of(int64_t T, int64_t E) {
  const int64_t rows = (int64_t)CLUSTER * WARPS * rows_at_once(E);
  if (T <= 2 * rows) return 1;
  return std::min<int64_t>(ceil_div(T, rows), device_sms() * 4 / CLUSTER);
}

}  // namespace

extern "C" {

int mb_expert_route(int32_t dtype, int64_t tokens, int64_t experts, int64_t k, int32_t normalize, const void *logits,
                    int64_t ldl, float *weights, int32_t *ids, void *stream) {
  const int rc = check("expert_route", dtype, tokens, experts, k, ldl, logits);
  if (rc) return rc;
  if (k > experts || k > MAX_K) return fail(MB_ERR_INVALID, "expert_route: k = %lld of %lld experts (at most %d)", (long long)k, (long long)experts, MAX_K);
  if (tokens * k == 0) return MB_OK;
  if (!weights || !ids) return fail(MB_ERR_INVALID, "expert_route: null pointer");
  RouteArgs a{logits, ldl, (int)tokens, (int)experts, (int)k, normalize, weights, ids, nullptr, nullptr};
  return by_shape(dtype, experts, logits, ldl, nullptr, [&](auto *t, auto nv, auto v, auto al) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int NV = decltype(nv)::value, V = decltype(v)::value;
    constexpr bool AL = decltype(al)::value;
    if constexpr (NV > 1)
      if (k > 32)
        return launch_pdl(route_kernel<T, NV, V, AL, true>, dim3(row_grid(tokens, 1)), dim3(THREADS), 0, (cudaStream_t)stream, 1,
                          "expert_route", a);
    return launch_pdl(route_kernel<T, NV, V, AL, false>, dim3(row_grid(tokens, rows_at_once(experts))), dim3(THREADS), 0,
                      (cudaStream_t)stream, 1, "expert_route", a);
  });
}

int mb_expert_route_backward(int32_t dtype, int64_t tokens, int64_t experts, int64_t k, int32_t normalize,
                             const float *grad, const void *logits, int64_t ldl, const int32_t *ids, void *dlogits,
                             void *stream) {
  const int rc = check("expert_route_backward", dtype, tokens, experts, k, ldl, logits);
  if (rc) return rc;
  if (k > MAX_K) return fail(MB_ERR_INVALID, "expert_route_backward: k = %lld (at most %d)", (long long)k, MAX_K);
  if (tokens == 0) return MB_OK;
  if (!dlogits || (k && (!grad || !ids))) return fail(MB_ERR_INVALID, "expert_route_backward: null pointer");
  RouteArgs a{logits, ldl, (int)tokens, (int)experts, (int)k, normalize, nullptr, const_cast<int32_t *>(ids), grad, dlogits};
  return by_shape(dtype, experts, logits, ldl, dlogits, [&](auto *t, auto nv, auto v, auto al) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int NV = decltype(nv)::value;
    constexpr auto kern = route_backward_kernel<T, NV, decltype(v)::value, decltype(al)::value>;
    constexpr int smem = WARPS * Rows<NV>::R * 32 * NV * 8;   // 64 KB at most
    const int rc = allow_smem<kern>(smem);
    if (rc) return rc;
    return launch_pdl(kern, dim3(row_grid(tokens, Rows<NV>::R)), dim3(THREADS), smem, (cudaStream_t)stream, 1,
                      "expert_route_backward", a);
  });
}

int64_t mb_expert_balance_workspace_size(int64_t tokens, int64_t experts) {
  if (tokens < 0 || experts < 1 || experts > MAX_EXPERTS) return 0;
  return parts_of(tokens, experts) * (2 * experts + 1) * 4;
}

int mb_expert_balance(int32_t dtype, int64_t tokens, int64_t experts, int64_t k, const void *logits, int64_t ldl,
                      const int32_t *ids, const uint8_t *mask, float *loss, int32_t *counts, int32_t *counted,
                      void *workspace, int64_t workspace_bytes, void *stream) {
  const int rc = check("expert_balance", dtype, tokens, experts, k, ldl, logits);
  if (rc) return rc;
  if (!loss || !counts || !counted || (tokens * k && !ids)) return fail(MB_ERR_INVALID, "expert_balance: null pointer");
  const int64_t need = mb_expert_balance_workspace_size(tokens, experts);
  if (!workspace || workspace_bytes < need) return fail(MB_ERR_WORKSPACE, "expert_balance: workspace of %lld bytes required", (long long)need);
  if (reinterpret_cast<uintptr_t>(workspace) & 3) return fail(MB_ERR_WORKSPACE, "expert_balance: the workspace must start on a 4-byte boundary");
  const int64_t parts = parts_of(tokens, experts);
  BalanceArgs a{};
  a.logits = logits; a.ld = ldl; a.T = (int)tokens; a.E = (int)experts; a.k = (int)k;
  a.experts = ids; a.mask = mask;
  a.part_p = static_cast<float *>(workspace);
  a.part_c = static_cast<int *>(workspace) + parts * experts;
  a.parts = (int)parts;
  a.loss = loss; a.counts = counts; a.tokens = counted;
  const int r = by_shape(dtype, experts, logits, ldl, nullptr, [&](auto *t, auto nv, auto v, auto al) {
    using T = std::remove_pointer_t<decltype(t)>;
    const size_t smem = (size_t)(WARPS * experts + experts + 1) * 4;   // 36 KB at 1024 experts
    return launch_pdl(balance_kernel<T, decltype(nv)::value, decltype(v)::value, decltype(al)::value>, dim3((unsigned)parts * CLUSTER), dim3(THREADS),
                      smem, (cudaStream_t)stream, CLUSTER, "expert_balance", a);
  });
  if (r || parts == 1) return r;
  // one block adds up a few sums, a cluster many (64 experts, 1000 tokens 5.8 and 6.8 us; 256 experts, 2048
  // tokens 9.5 and 8.3; 128 experts, 65536 tokens 20.9 and 19.9)
  const int blocks = parts * (experts + 1) <= 3 * FINISH_THREADS && experts < FINISH_THREADS ? 1 : CLUSTER;
  return launch_pdl(balance_finish_kernel, dim3(blocks), dim3(FINISH_THREADS), 0, (cudaStream_t)stream, blocks, "expert_balance", a);
}

int mb_expert_balance_backward(int32_t dtype, int64_t tokens, int64_t experts, const float *grad, const void *logits,
                               int64_t ldl, const int32_t *counts, const int32_t *counted, const uint8_t *mask,
                               void *dlogits, void *stream) {
  const int rc = check("expert_balance_backward", dtype, tokens, experts, 1, ldl, logits);
  if (rc || tokens == 0) return rc;
  if (!grad || !counts || !counted || !dlogits) return fail(MB_ERR_INVALID, "expert_balance_backward: null pointer");
  BalanceArgs a{};
  a.logits = logits; a.ld = ldl; a.T = (int)tokens; a.E = (int)experts; a.mask = mask;
  a.counts = const_cast<int32_t *>(counts); a.tokens = const_cast<int32_t *>(counted);
  a.grad = grad; a.dlogits = dlogits;
  return by_shape(dtype, experts, logits, ldl, dlogits, [&](auto *t, auto nv, auto v, auto al) {
    using T = std::remove_pointer_t<decltype(t)>;
    return launch_pdl(balance_backward_kernel<T, decltype(nv)::value, decltype(v)::value, decltype(al)::value>,
                      dim3(row_grid(tokens, rows_at_once(experts))),
                      dim3(THREADS), 0, (cudaStream_t)stream, 1, "expert_balance_backward", a);
  });
}

}  // extern "C"
