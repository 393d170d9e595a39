// Stateless router on given logits: the experts of every token and their weights (route_select.cuh has the rule).
// One warp per token, the row in registers: lane i holds npl = ceil(E / 32) neighbouring experts.
//
// Bound by instructions, not by bytes: 16384 rows of 256 float32 logits are 16.8 MB, 2.6 us at the measured copy rate, and take
// 10.5 us for 8 of softmax scores, 11.8 us with sigmoid scores and a bias, 18.8 us with the best 4 of 8 groups as well (some 750
// instructions a row, 2.7 a cycle and SM). One token to 64 take 2.1 to 3.3 us, launch included. What it took to get there (the
// last case): integer divisions and group geometry out of the loop over rows, numbers ranked as numbers (redux.sync of floats)
// instead of as ordered integers: 28 -> 20 us; the exact ranking of a row with close neighbours by its candidates alone, one
// lane each, instead of all its experts: 64 tokens, one of them such a row, 9.7 -> 3.9 us.
#include <algorithm>

#include "route_select.cuh"

namespace pm {
namespace {

constexpr int kRouteWarps = 4;
constexpr int kRouteMaxExperts = 1024;

// Plain loads: the 16-bit forms of __ldg are pure inline assembly, which the compiler may move in front of a bounds test.
__device__ __forceinline__ float load_logit(const float* p) { return *p; }
__device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_logit(const __half* p) { return __half2float(*p); }

// Resident blocks, each row of warps taking one token after the other. More of them with fewer registers: 256 experts in groups
// 20.3 -> 22 us (8 blocks), 512 experts 10.9 -> 12.0 us (5); one block per four tokens instead, launched one after another:
// 25 us.
constexpr int blocks_per_sm(int npl) { return npl <= 8 ? 6 : npl <= 16 ? 4 : 3; }

template <class T, int NPL, int KIND>
__global__ void __launch_bounds__(kRouteWarps * 32, blocks_per_sm(NPL))
route_kernel(const T* __restrict__ logits, int64_t ld, int n_tok, const __grid_constant__ RouteRule rule, int vector_loads,
             int32_t* __restrict__ topk_ids, float* __restrict__ topk_w) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int E = rule.E, npl = (E + 31) / 32, e0 = lane * npl;
  RouteScratch* scratch = reinterpret_cast<RouteScratch*>(smem_raw + warp * route_scratch_bytes(E));
  wait_for_predecessor();

  float b[NPL];
  const float bias_max = load_choice_bias<NPL>(rule, npl, lane, b);
  const RouteGroups groups(rule, npl, lane);
  constexpr int kVec = 16 / sizeof(T);
  float l[NPL];
  auto load = [&](int64_t t) {
    const T* row = logits + t * ld;
    if (vector_loads) {  // E = 32 npl, npl a multiple of kVec, rows on 16-byte boundaries
      if constexpr (NPL % kVec == 0) {
#pragma unroll
        for (int j = 0; j < NPL; j += kVec)
          if (j < npl) {
            const uint4 v = *reinterpret_cast<const uint4*>(row + e0 + j);
            const T* p = reinterpret_cast<const T*>(&v);
#pragma unroll
            for (int i = 0; i < kVec; ++i) l[j + i] = (float)p[i];
          }
      }
    } else {
#pragma unroll
      for (int j = 0; j < NPL; ++j)
        if (j < npl && e0 + j < E) l[j] = load_logit(row + e0 + j);
    }
  };
#pragma unroll
  for (int j = 0; j < NPL; ++j) l[j] = -CUDART_INF_F;
  const int64_t step = (int64_t)gridDim.x * kRouteWarps;
  for (int64_t t = (int64_t)blockIdx.x * kRouteWarps + warp; t < n_tok; t += step) {
    load(t);
    const T* row = logits + t * ld;
    route_token<NPL, KIND>(l, npl, rule, b, bias_max, groups, scratch, lane, [&](int e) { return load_logit(row + e); },
                     [&](int j, int id, float w) {
                       topk_ids[t * rule.k + j] = id;
                       topk_w[t * rule.k + j] = w;
                     });
  }
}

template <class T, int NPL>
cudaError_t launch(const T* logits, int64_t ld, int n_tok, const RouteRule& rule, int32_t* ids, float* w, cudaStream_t s) {
  const int npl = (rule.E + 31) / 32, vec = 16 / (int)sizeof(T);
  const int vector_loads = NPL % vec == 0 && npl % vec == 0 && rule.E == 32 * npl && ((uintptr_t)logits & 15) == 0 &&
                           (ld * (int64_t)sizeof(T)) % 16 == 0;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
  // One row after the other per warp once every SM has its blocks; at most 35 KB of shared memory per block.
  const int blocks = std::min((n_tok + kRouteWarps - 1) / kRouteWarps, sms * blocks_per_sm(NPL));
  // Kernels of their own for the usual kinds of rules: 16384 tokens of 256 experts, softmax 11.8 -> 10.5 us, sigmoid and bias 13.5 ->
  // 11.8, with groups 20.3 -> 18.8. Wider rows are too rare for that. Dropped choices of 0 take the general kernel: 17.5-18.7 us become
  // 19.1-20.4 there, of 64 tokens 3.0 become 3.2 (a test in the fixed kinds would cost those that drop by -inf).
  auto kern = route_kernel<T, NPL, kAnyRule>;
  if constexpr (NPL <= 16) {
    switch (rule.drop_zero ? (int)kAnyRule : route_kind(rule)) {
      case 0: kern = route_kernel<T, NPL, 0>; break;
      case kGrouped: kern = route_kernel<T, NPL, kGrouped>; break;
      case kSigmoid | kHasBias: kern = route_kernel<T, NPL, kSigmoid | kHasBias>; break;
      case kSigmoid | kHasBias | kGrouped: kern = route_kernel<T, NPL, kSigmoid | kHasBias | kGrouped>; break;
    }
  }
  return launch_behind(kern, blocks, kRouteWarps * 32, kRouteWarps * route_scratch_bytes(rule.E), s, logits, ld,
                       n_tok, rule, vector_loads, ids, w);
}

template <class T>
cudaError_t pick(const T* logits, int64_t ld, int n_tok, const RouteRule& rule, int32_t* ids, float* w, cudaStream_t s) {
  const int npl = (rule.E + 31) / 32;
  // Registers of a lane: the next size up. 4096 rows of 512 experts in 16 registers 10.9 us, in 32 of them 18.8 us.
  if (npl <= 2) return launch<T, 2>(logits, ld, n_tok, rule, ids, w, s);
  if (npl <= 8) return launch<T, 8>(logits, ld, n_tok, rule, ids, w, s);
  if (npl <= 16) return launch<T, 16>(logits, ld, n_tok, rule, ids, w, s);
  return launch<T, 32>(logits, ld, n_tok, rule, ids, w, s);
}

}  // namespace

int check_route_rule(const RouteRule& r, const char* who) {
  const std::string name(who);
  if (r.E <= 0 || r.E > kRouteMaxExperts) return fail(PM_ERR_INVALID, name + ": num_expert must be in [1, 1024]");
  if (r.k <= 0 || r.k > 32 || r.k > r.E) return fail(PM_ERR_INVALID, name + ": top_k must be in [1, min(32, num_expert)]");
  if (r.n_group < 1 || r.n_group > 32 || r.E % r.n_group != 0)
    return fail(PM_ERR_INVALID, name + ": n_group must be in [1, 32] and divide num_expert");
  if (r.topk_group < 1 || r.topk_group > r.n_group) return fail(PM_ERR_INVALID, name + ": topk_group must be in [1, n_group]");
  if (r.k > r.topk_group * (r.E / r.n_group))
    return fail(PM_ERR_INVALID, name + ": topk_group groups hold fewer than top_k experts");
  if (r.drop_zero && r.bias == nullptr) return fail(PM_ERR_INVALID, name + ": PM_GROUP_DROPPED_ZERO is for routers with a choice_bias");
  return PM_OK;
}

cudaError_t launch_route(const void* logits, int dtype, int64_t ld, int n_tok, const RouteRule& rule, int32_t* ids, float* w,
                         cudaStream_t s) {
  if (n_tok <= 0) return cudaSuccess;
  if (dtype == PM_F32) return pick((const float*)logits, ld, n_tok, rule, ids, w, s);
  if (dtype == PM_BF16) return pick((const __nv_bfloat16*)logits, ld, n_tok, rule, ids, w, s);
  return pick((const __half*)logits, ld, n_tok, rule, ids, w, s);
}

}  // namespace pm
