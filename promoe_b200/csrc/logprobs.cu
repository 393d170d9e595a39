// Log probability of a given token, entropy and the best alternatives of every row of vocabulary logits, in one pass:
//   M = max l, S = sum 2^(l log2e - c), U = sum 2^(l log2e - c) (l log2e - c), c = M log2e rounded
//   lse = c ln2 + ln S,  logp = l_target - lse,  H = ln S - ln2 U / S,  top: l - lse of the n largest
// c is rounded once and used everywhere, so its rounding cancels; a logit costs one multiply-add, one exponential, one
// addition, one multiply-add and the maximum.
//
// A row is read by a cluster of CTAs (one where there are many rows); every thread keeps its own running maximum and
// sums and rescales them when a batch of its values raises the maximum.
//
// The n best come out of the same pass. The first batch gives a threshold (of 32 groups of threads the n-th best
// maximum: n values reach it); every value that reaches it goes to a list in shared memory, about 1.5 n per batch, and at the
// end a value's place is the number of list entries before it. Entries are (ordered value, reversed index), so ties go to
// the lower index and the result does not depend on the order in which the list was filled. A row whose list
// overflows (many equal values, ascending rows) finds its n-th best entry by radix selection over the row instead.
//
// Masked logits: -inf has probability 0 and is never an alternative (id -1, log probability -inf where fewer than n are
// left). A row that holds NaN or +inf, or whose logits are all -inf, is no distribution: NaN and id -1. A negative target names
// no token (log probability 0), one beyond the row is NaN.
#include <math_constants.h>

#include "pm_common.cuh"
#include "sm100_ptx.cuh"

namespace pm {
namespace {

using sm100::cluster_rank;
using sm100::cluster_sync;
using sm100::map_to_rank;
using sm100::smem_u32;

constexpr int kListCap = 1024;
constexpr int kMaxTop = 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.69314718055994531;
constexpr int kUnroll = 4;  // 16-byte vectors per thread and batch

using Entry = unsigned long long;  // ordered value above the reversed index

__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ Entry entry_of(float v, uint32_t index) { return ((Entry)order_of(v) << 32) | (0xffffffffu - index); }
constexpr uint32_t kOrderNegInf = 0x007fffffu;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// volatile: a load that the compiler could move would pass the test for the row's end
__device__ __forceinline__ uint4 load_stream(const uint4* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}

template <class T> struct Vec;
template <> struct Vec<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ void widen(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ void widen(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <> struct Vec<__half> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ void widen(const uint4& v, float (&f)[8]) {
    const __half2* p = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __half22float2(p[i]);
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
};
template <class T> __device__ __forceinline__ float widen_one(T v);
template <> __device__ __forceinline__ float widen_one(float v) { return v; }
template <> __device__ __forceinline__ float widen_one(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float widen_one(__half v) { return __half2float(v); }

// Running sums of one thread, or of a part of the row. m: largest value so far, c: m log2e (0 while m is -inf). For values
// near the type's limits c stops at a number that float32 holds: below, the sum is then 0, as it should be beside any ordinary
// value; rows whose maximum lies out there are summed again at the end.
struct Sums {
  float m, c, s, u;
};
__device__ __forceinline__ Sums no_sums() { return Sums{-CUDART_INF_F, 0.f, 0.f, 0.f}; }

__device__ __forceinline__ void raise(Sums& a, float m) {  // m > a.m
  const float c = fminf(fmaxf(m, -2e38f), 2e38f) * kLog2e, d = a.c - c;
  const float f = a.s > 0.f ? exp2_fast(d) : 0.f;
  a.u = a.s > 0.f ? f * (a.u + d * a.s) : (a.s != a.s ? a.s : 0.f);
  a.s = a.s != a.s ? a.s : a.s * f;
  a.m = m;
  a.c = c;
}
__device__ __forceinline__ void add_value(Sums& a, float l) {
  const float t = fmaf(l, kLog2e, -a.c), e = exp2_fast(t);
  a.s += e;
  a.u = fmaf(e, fmaxf(t, -1e4f), a.u);  // masked values: 0 times a finite number
}
__device__ __forceinline__ void join(Sums& a, const Sums& b) {
  if (b.m > a.m) raise(a, b.m);
  const float d = b.m == -CUDART_INF_F ? 0.f : b.c - a.c;  // sums of a part without a finite value are 0 or NaN
  const float f = exp2_fast(d);
  a.u += b.s == 0.f ? 0.f : f * (b.u + fmaxf(d, -1e4f) * b.s);
  a.s += f * b.s;
}

struct LogprobArgs {
  const void* logits;
  int64_t ld;
  const int64_t* targets;
  int32_t T, V, n;
  float *logp, *entropy;
  int32_t* top_ids;
  float* top_logp;
};

template <int THREADS>
struct LogprobShared {
  Sums warp_sums[THREADS / 32];
  Sums part;              // this CTA's sums, read by rank 0
  Entry best[kMaxTop];    // this CTA's n best in order, read by rank 0
  float seg[32];
  Entry list[kListCap];
  int count;
  uint32_t hist[256];
  Entry prefix;
  int need;
  double lse;
  int dead;
};

// Entries of `list` in order: out[r] = the r-th largest, r < n; 0 where there are fewer.
template <int THREADS>
__device__ __forceinline__ void rank_list(const Entry* list, int count, Entry* out, int n) {
  const int tid = threadIdx.x;
  for (int r = tid; r < n; r += THREADS)
    if (r >= count) out[r] = 0;
  for (int i = tid; i < count; i += THREADS) {
    const Entry mine = list[i];
    int before = 0;
    for (int j = 0; j < count; ++j) before += list[j] > mine;
    if (before < n) out[before] = mine;
  }
}

template <class T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
logprobs_kernel(const __grid_constant__ LogprobArgs a, int parts) {
  __shared__ LogprobShared<THREADS> sh;
  constexpr int N = Vec<T>::kN;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank();
  const int row = blockIdx.x / parts, n = a.n;
  wait_for_predecessor();

  const T* l = static_cast<const T*>(a.logits) + (int64_t)row * a.ld;
  const int head = min(a.V, (int)(((16 - ((uintptr_t)l & 15)) & 15) / sizeof(T)));
  const int n_vec = (a.V - head) / N, tail0 = head + n_vec * N;
  const int v0 = (int)((long long)n_vec * rank / parts), v1 = (int)((long long)n_vec * (rank + 1) / parts);
  const uint4* body = reinterpret_cast<const uint4*>(l + head);

  Sums a0 = no_sums();
  if (tid == 0) sh.count = 0;
  __syncthreads();
  auto push = [&](Entry e) {
    const int at = atomicAdd(&sh.count, 1);
    if (at < kListCap) sh.list[at] = e;
  };
  // values before the first and behind the last 16-byte boundary
  if (rank == 0) {
    const int loose = head + (a.V - tail0);
    if (tid < loose) {
      const int i = tid < head ? tid : tail0 + tid - head;
      const float v = widen_one(l[i]);
      if (v > a0.m) raise(a0, v);
      add_value(a0, v);
      if (n > 0 && order_of(v) > kOrderNegInf && v == v) push(entry_of(v, (uint32_t)i));
    }
  }
  Entry threshold = ((Entry)kOrderNegInf << 32) | 0xffffffffu;
  float floor_v = -CUDART_INF_F;
  uint4 next[kUnroll];
  auto fetch = [&](int base) {
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int v = base + k * THREADS + tid;
      if (v < v1) next[k] = load_stream(body + v);
    }
  };
  fetch(v0);
  for (int base = v0; base < v1; base += kUnroll * THREADS) {
    uint4 cur[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) cur[k] = next[k];
    if (base + kUnroll * THREADS < v1) fetch(base + kUnroll * THREADS);
    float top[kUnroll], all = -CUDART_INF_F;
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      top[k] = -CUDART_INF_F;
      if (base + k * THREADS + tid < v1) {
        float f[N];
        Vec<T>::widen(cur[k], f);
#pragma unroll
        for (int i = 0; i < N; ++i) top[k] = fmaxf(top[k], f[i]);
      }
      all = fmaxf(all, top[k]);
    }
    if (all > a0.m) raise(a0, all);
#pragma unroll
    for (int k = 0; k < kUnroll; ++k)
      if (base + k * THREADS + tid < v1) {
        float f[N];
        Vec<T>::widen(cur[k], f);
#pragma unroll
        for (int i = 0; i < N; ++i) add_value(a0, f[i]);
      }
    if (n == 0) continue;
    if (base == v0) {
      // threshold: the n-th best of 32 groups' maxima
      constexpr int kGroup = THREADS / 32;
      float g = all;
#pragma unroll
      for (int m = kGroup / 2; m >= 1; m >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, m));
      if (tid % kGroup == 0) sh.seg[tid / kGroup] = g;
      __syncthreads();
      const float mine = sh.seg[lane];
      int before = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float o = __shfl_sync(0xffffffffu, mine, i);
        before += o > mine || (o == mine && i < lane);
      }
      floor_v = __shfl_sync(0xffffffffu, mine, __ffs(__ballot_sync(0xffffffffu, before == n - 1)) - 1);
      if (floor_v > -CUDART_INF_F) threshold = (Entry)order_of(floor_v) << 32;
    }
    if (all >= floor_v && all > -CUDART_INF_F) {
#pragma unroll
      for (int k = 0; k < kUnroll; ++k)
        if (top[k] >= floor_v && top[k] > -CUDART_INF_F) {
          float f[N];
          Vec<T>::widen(cur[k], f);
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (f[i] >= floor_v) {
              const Entry e = entry_of(f[i], (uint32_t)(head + (base + k * THREADS + tid) * N + i));
              if (e > threshold) push(e);
            }
        }
    }
  }

  // sums of the warp, the CTA, the row
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) {
    Sums o;
    o.m = __shfl_xor_sync(0xffffffffu, a0.m, m);
    o.c = __shfl_xor_sync(0xffffffffu, a0.c, m);
    o.s = __shfl_xor_sync(0xffffffffu, a0.s, m);
    o.u = __shfl_xor_sync(0xffffffffu, a0.u, m);
    join(a0, o);
  }
  if (lane == 0) sh.warp_sums[warp] = a0;
  __syncthreads();
  if (tid == 0) {
    Sums t = sh.warp_sums[0];
    for (int w = 1; w < THREADS / 32; ++w) join(t, sh.warp_sums[w]);
    sh.part = t;
  }
  if (n > 0) {
    int count = sh.count;
    if (count > kListCap) {
      // radix selection of the n-th largest entry of this part, eight bits at a time from the top
      if (tid == 0) {
        sh.prefix = 0;
        sh.need = n;
      }
      const int lo = rank == 0 ? 0 : head + v0 * N, hi = rank == (uint32_t)parts - 1 ? a.V : head + v1 * N;
      auto of = [&](int i, bool& in) {
        const float v = widen_one(l[i]);
        in = v == v && v > -CUDART_INF_F;
        // loose values at the end of the row belong to rank 0
        if (i >= tail0 && rank != 0) in = false;
        return entry_of(v, (uint32_t)i);
      };
      for (int shift = 56; shift >= 0; shift -= 8) {
        for (int b = tid; b < 256; b += THREADS) sh.hist[b] = 0;
        __syncthreads();
        const Entry prefix = sh.prefix;
        for (int pass = 0; pass < 2; ++pass) {
          const int from = pass ? max(hi, tail0) : lo, to = pass ? (rank == 0 ? a.V : 0) : hi;
          for (int i0 = from; i0 < to; i0 += THREADS) {
            bool in = i0 + tid < to;
            Entry e = 0;
            if (in) e = of(i0 + tid, in);
            in = in && (shift == 56 || (e >> (shift + 8)) == (prefix >> (shift + 8)));
            const uint32_t digit = in ? (uint32_t)(e >> shift) & 255u : 256u;
            const unsigned same = __match_any_sync(0xffffffffu, digit);  // equal values are what brings rows here
            if (in && lane == __ffs(same) - 1) atomicAdd(&sh.hist[digit], (uint32_t)__popc(same));
          }
        }
        __syncthreads();
        if (tid == 0) {
          int need = sh.need, b = 255;
          for (; b > 0 && (int)sh.hist[b] < need; --b) need -= (int)sh.hist[b];
          sh.need = need;
          sh.prefix = prefix | ((Entry)b << shift);
        }
        __syncthreads();
      }
      const Entry least = sh.prefix;  // the n-th largest (there are more than kListCap)
      if (tid == 0) sh.count = 0;
      __syncthreads();
      for (int pass = 0; pass < 2; ++pass) {
        const int from = pass ? max(hi, tail0) : lo, to = pass ? (rank == 0 ? a.V : 0) : hi;
        for (int i = from + tid; i < to; i += THREADS) {
          bool in;
          const Entry e = of(i, in);
          if (in && e >= least) push(e);
        }
      }
      __syncthreads();
      count = sh.count;
    }
    rank_list<THREADS>(sh.list, count, sh.best, n);
  }
  if (parts > 1) {
    cluster_sync();
    if (rank == 0) {
      if (tid == 0) {
        Sums t = sh.part;
        for (int p = 1; p < parts; ++p) {
          const uint32_t at = map_to_rank(smem_u32(&sh.part), p);
          Sums o;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.m) : "r"(at));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.c) : "r"(at + 4));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.s) : "r"(at + 8));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.u) : "r"(at + 12));
          join(t, o);
        }
        sh.part = t;
        sh.count = 0;
      }
      __syncthreads();
      if (n > 0) {
        for (int i = tid; i < parts * n; i += THREADS) {
          Entry e;
          asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(e) : "r"(map_to_rank(smem_u32(&sh.best[i % n]), i / n)));
          if (e != 0) push(e);
        }
      }
    }
    cluster_sync();  // nobody leaves before its part was read
    if (rank != 0) return;
    if (n > 0) rank_list<THREADS>(sh.list, sh.count, sh.best, n);
  }
  __syncthreads();

  Sums t = sh.part;
  if (fabsf(t.m) > 1e37f && fabsf(t.m) < CUDART_INF_F) {
    // m log2e may have overflowed (a row of the type's lowest value): once more, relative to the maximum
    Sums b = no_sums();
    bool bad = false;
    for (int i = tid; i < a.V; i += THREADS) {
      const float v = widen_one(l[i]), d = (v - t.m) * kLog2e, e = exp2_fast(d);
      bad |= v != v;
      b.s += e;
      b.u = fmaf(e, fmaxf(d, -1e4f), b.u);
    }
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) {
      b.s += __shfl_xor_sync(0xffffffffu, b.s, m);
      b.u += __shfl_xor_sync(0xffffffffu, b.u, m);
    }
    if (lane == 0) sh.warp_sums[warp] = b;
    __syncthreads();
    t.s = t.u = 0.f;
    for (int w = 0; w < THREADS / 32; ++w) {
      t.s += sh.warp_sums[w].s;
      t.u += sh.warp_sums[w].u;
    }
    if (__syncthreads_or(bad)) t.s = CUDART_NAN_F;
  }
  const bool dead = !(t.s > 0.f) || !(fabsf(t.m) < CUDART_INF_F);
  const double log_s = log((double)t.s);
  const double lse = dead ? CUDART_NAN : (fabsf(t.m) > 1e37f ? (double)t.m : (double)t.c * kLn2) + log_s;
  if (tid == 0) {
    if (a.logp != nullptr) {
      const int64_t target = a.targets[row];
      a.logp[row] = target < 0 ? 0.f : (dead || target >= a.V) ? CUDART_NAN_F : (float)((double)widen_one(l[target]) - lse);
    }
    if (a.entropy != nullptr)
      a.entropy[row] = dead ? CUDART_NAN_F : (float)(log_s - kLn2 * (double)t.u / (double)t.s);
  }
  for (int r = tid; r < n; r += THREADS) {
    const Entry e = dead ? 0 : sh.best[r];
    a.top_ids[(int64_t)row * n + r] = e == 0 ? -1 : (int32_t)(0xffffffffu - (uint32_t)e);
    a.top_logp[(int64_t)row * n + r] =
        dead ? CUDART_NAN_F : e == 0 ? -CUDART_INF_F : (float)((double)value_of((uint32_t)(e >> 32)) - lse);
  }
}

template <class T, int THREADS>
cudaError_t launch(const LogprobArgs& a, int parts, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = (unsigned)a.T * (unsigned)parts;
  cfg.blockDim = THREADS;
  cfg.stream = s;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)parts, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, logprobs_kernel<T, THREADS>, a, parts);
}

template <class T>
cudaError_t pick(const LogprobArgs& a, int sms, cudaStream_t s) {
  // a cluster per row while that fills the GPU no more than about twice and a part stays longer than a batch of 128 threads
  int parts = 1;
  while (parts < 8 && (int64_t)a.T * parts * 2 <= 2 * sms && a.V / (2 * parts) >= 4096) parts *= 2;
  // a thread should have a whole batch, and each of the 32 groups of threads values for the threshold
  if (a.V / parts >= 512 * kUnroll * Vec<T>::kN / 2) return launch<T, 512>(a, parts, s);
  return launch<T, 128>(a, parts, s);
}

}  // namespace

cudaError_t launch_token_logprobs(const void* logits, int dtype, int64_t ld, int T, int V, const int64_t* targets, int n,
                                  float* logp, float* entropy, int32_t* top_ids, float* top_logp, cudaStream_t s) {
  if (T <= 0) return cudaSuccess;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
  const LogprobArgs a{logits, ld, targets, T, V, n, logp, entropy, top_ids, top_logp};
  if (dtype == PM_F32) return pick<float>(a, sms, s);
  if (dtype == PM_BF16) return pick<__nv_bfloat16>(a, sms, s);
  return pick<__half>(a, sms, s);
}

}  // namespace pm
