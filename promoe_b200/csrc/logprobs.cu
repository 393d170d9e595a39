// Log probability of a given token, entropy and the best alternatives of every row of vocabulary logits, in one pass:
//   M = max l, S = sum 2^(l k - c), U = sum 2^(l k - c) (l k - c), k = log2 e and c = M k, both rounded
//   lse = c / k + ln S,  logp = l_target - lse,  H = ln S - ln2 U / S,  top: l - lse of the n largest
// c is rounded once and used everywhere, so its rounding cancels. k's does where c is divided by the same k (times ln 2 it was
// off by 1.3e-8 M); in the terms it leaves 1.3e-8 of (l - M). Two logits cost two exponentials and three packed
// float32 instructions besides the widening and the maximum. Logits are raised to a value that has no probability beside any
// other (kLow), which keeps 0 times infinity out of U; rows whose maximum is down there are summed again. (Raising only
// once a thread has met a masked logit changed nothing.)
//
// A row is read by a cluster of CTAs (one where there are many rows); every thread keeps its own running maximum and
// sums and rescales them when a batch of its values raises the maximum.
//
// The n best come out of the same pass. The first batch gives a floor (of 32 or 64 groups of threads the n-th best
// maximum: n values reach it), later ones raise it; every 16-byte vector with a value that reaches the floor is noted, about
// 1.5 n of them each time the part read doubles. At the end their values that reach the last floor go to a list, where a
// value's place is the number of entries before it. Entries are (ordered value, reversed index), so ties go to the lower index and
// the result does not depend on the order in which the list was filled, nor on the floors. A row whose lists overflow (many
// equal values, ascending rows) finds its n-th best entry by radix selection over the row instead. (Sorting out the values of
// a vector inside the loop costs registers and code there: 53 and, for n = 20, 90 us instead of 55 and 58 for 1024 rows of 131072.)
//
// What bounds it: long rows HBM. 4096 rows of 131072 bf16 take 166 us = 6.49 TB/s without alternatives, 190 us = 5.65 TB/s with
// five and 211 us with twenty: the end of a row (two rankings, the noted vectors' way from L2) is latency that four CTAs per SM
// cover in part. That is at 1965 MHz; after some hundred passes the 1000 W limit takes the clock to 1680 MHz, and the same
// passes take 197, 223 and about 250 us. Short rows that end too (4096 of 2048: 12 us without alternatives, 21 with five; one warp per row
// instead of four changed that by less than a fifth). One row of 131072 takes 3.7 us without alternatives, 6 to 6.5 with five, 8
// with twenty: a chain of load, floor, sums, cluster barrier and ranking, each of them 500 to 1500 cycles, most of which go into the
// first fetch of its instructions. Hence few unrolled loops and one copy of the ranking. The parts of a row write their
// sums and best into rank 0's shared memory before the only barrier that anyone waits for (reading them from there
// behind it: 0.5 us more). First form, with scalar arithmetic and the lists sorted out in the loop: 281 us for 4096 rows, 11.5 for one.
//
// Masked logits: -inf has probability 0 and is never an alternative (id -1, log probability -inf where fewer than n are
// left). A row that holds NaN or +inf, or whose logits are all -inf, is no distribution: NaN and id -1. A negative target names
// no token (log probability 0), one beyond the row is NaN.
#include <math_constants.h>

#include "pm_common.cuh"
#include "sm100_ptx.cuh"

namespace pm {
namespace {

using sm100::cluster_arrive_diverged;
using sm100::cluster_rank;
using sm100::cluster_wait_diverged;
using sm100::map_to_rank;
using sm100::smem_u32;

constexpr int kCap = 1024;  // room in the lists
constexpr int kMaxTop = 32;
constexpr int kMaxParts = 8;  // CTAs of a row
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kPerC = 1.0 / (double)kLog2e;
constexpr float kLn2 = 0.69314718f;
constexpr int kUnroll = 4;  // 16-byte vectors per thread and batch

using Entry = unsigned long long;  // ordered value above the reversed index

__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ Entry entry_of(float v, uint32_t index) { return ((Entry)order_of(v) << 32) | (0xffffffffu - index); }

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

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 16 bytes of logits. kLow: no logit counts beside one that is more than kFar above it, and -inf is raised to it. kLowBits: a
// register of it. raise(): all values at least kLow, NaN kept. top(): the larger (NaN ignored). pair(i): values 2i, 2i + 1. first(): the
// lowest value of a 64-bit word.
constexpr float kFar = 300.f;
// Rows with a larger maximum are summed again. c is off by half a step, at most 4 between kLow and here, which the exponents of the sums
// can hold; a maximum of 1e10 would be off by 512, one of 1e33 would take the sums' rescaling to infinity, and a thread that meets
// values of -1e9 first (masks) before any ordinary one would make them infinite too, hence kLow.
constexpr float kPlain = 1e8f;
template <class T> struct Vec;
template <> struct Vec<float> {
  static constexpr int kN = 4;
  static constexpr float kLow = -0x1p26f;
  static constexpr uint32_t kLowBits = 0xCC800000u;
  static __device__ __forceinline__ uint32_t raise(uint32_t w) { return __float_as_uint(max_nan(__uint_as_float(w), kLow)); }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ float top(uint32_t w) { return __uint_as_float(w); }
  static __device__ __forceinline__ float first(uint64_t v) { return __uint_as_float((uint32_t)v); }
  static __device__ __forceinline__ uint64_t pair(const uint4& v, int i) {
    return i == 0 ? pack2(__uint_as_float(v.x), __uint_as_float(v.y)) : pack2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int kN = 8;
  static constexpr float kLow = -0x1p26f;
  static constexpr uint32_t kLowBits = 0xCC80CC80u;
  static __device__ __forceinline__ uint32_t raise(uint32_t w) {
    const uint32_t low = kLowBits;
    const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&w), *reinterpret_cast<const __nv_bfloat162*>(&low));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ float top(uint32_t w) {
    return fmaxf(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ float first(uint64_t v) { return __uint_as_float((uint32_t)v << 16); }
  static __device__ __forceinline__ uint64_t pair(const uint4& v, int i) {
    const uint32_t w = (&v.x)[i];
    return pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
};
template <> struct Vec<__half> {
  static constexpr int kN = 8;
  static constexpr float kLow = -65504.f;
  static constexpr uint32_t kLowBits = 0xFBFFFBFFu;
  static __device__ __forceinline__ uint32_t raise(uint32_t w) {
    const uint32_t low = kLowBits;
    const __half2 r = __hmax2_nan(*reinterpret_cast<const __half2*>(&w), *reinterpret_cast<const __half2*>(&low));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    const __half2 r = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ float top(uint32_t w) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return fmaxf(f.x, f.y);
  }
  static __device__ __forceinline__ float first(uint64_t v) { return __half2float(__ushort_as_half((unsigned short)v)); }
  static __device__ __forceinline__ uint64_t pair(const uint4& v, int i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&(&v.x)[i]));
    return pack2(f.x, f.y);
  }
};
template <class T> __device__ __forceinline__ float widen_one(T v);
template <> __device__ __forceinline__ float widen_one(float v) { return v; }
template <> __device__ __forceinline__ float widen_one(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float widen_one(__half v) { return __half2float(v); }

// Running sums of one thread, or of a part of the row. m: largest value so far (at least kLow), c: m log2e.
struct Sums {
  float m, c, s, u;
};
template <class T>
__device__ __forceinline__ Sums no_sums() { return Sums{Vec<T>::kLow, Vec<T>::kLow * kLog2e, 0.f, 0.f}; }
__device__ __forceinline__ void join(Sums& a, const Sums& b) {
  const float m = fmaxf(a.m, b.m), c = m * kLog2e;
  const float da = a.c - c, db = b.c - c, fa = exp2_fast(da), fb = exp2_fast(db);
  a.u = fa * (a.u + da * a.s) + fb * (b.u + db * b.s);
  a.s = fa * a.s + fb * b.s;
  a.m = m;
  a.c = c;
}
// Over the first `width` lanes of every group of `width`; the group's first lane has the result.
__device__ __forceinline__ void join_lanes(Sums& a, int width) {
  for (int d = width >> 1; d >= 1; d >>= 1) {
    Sums o;
    o.m = __shfl_down_sync(0xffffffffu, a.m, d, width);
    o.c = __shfl_down_sync(0xffffffffu, a.c, d, width);
    o.s = __shfl_down_sync(0xffffffffu, a.s, d, width);
    o.u = __shfl_down_sync(0xffffffffu, a.u, d, width);
    join(a, o);
  }
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
  alignas(16) Entry list[kCap];
  Sums warp_sums[32];
  alignas(16) Sums part;  // the row's sums
  Entry best[kMaxTop];    // the row's n best in order; 0 to begin with
  // in rank 0, which the others write to: sums and n best of each part
  alignas(16) Sums part_sums[kMaxParts];
  alignas(16) Entry part_best[kMaxParts * kMaxTop];
  float seg[64];          // largest value of each group of threads so far
  int count, n_hot;
  int32_t hot[kCap];   // 16-byte vectors that held a value that reached the floor
  uint32_t hist[256];
  Entry prefix;
  int need;
};

// Entries of `list` in order: the r-th largest to shared memory (of any CTA of the cluster) at out + 8 r, r < n; 0 where there
// are fewer. Four neighbouring threads compare for one entry. All threads call it; `list` is aligned to 16 bytes. One
// copy of the code for both rankings of a row: fetching it costs more than running it.
template <int THREADS>
__device__ __noinline__ void rank_list(const Entry* list, int count, int n, uint32_t out) {
  const int tid = threadIdx.x, quarter = tid & 3;
  auto put = [&](int r, Entry e) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(out + 8u * (uint32_t)r), "l"(e) : "memory"); };
  for (int r = count + tid; r < n; r += THREADS) put(r, 0);
  const uint32_t pairs = smem_u32(list);
#pragma unroll 1
  for (int i0 = 0; i0 < count; i0 += THREADS / 4) {
    const int i = i0 + (tid >> 2);
    const Entry mine = i < count ? list[i] : ~(Entry)0;
    int before = 0;
#pragma unroll 2
    for (int j = quarter; 2 * j < count; j += 4) {
      const uint4 o = sm100::lds128(pairs + 16u * (uint32_t)j);
      before += (((Entry)o.y << 32 | o.x) > mine) + (2 * j + 1 < count && ((Entry)o.w << 32 | o.z) > mine);
    }
    before += __shfl_xor_sync(0xffffffffu, before, 1);
    before += __shfl_xor_sync(0xffffffffu, before, 2);
    if (i < count && before < n && quarter == 0) put(before, mine);
  }
}

// The n-th largest of seg[0 .. 32 or 64): the least of those that fewer than n exceed. Read once: they may rise meanwhile.
__device__ __forceinline__ float nth_best(const volatile float* seg, bool wide, int n) {
  const int lane = threadIdx.x & 31;
  const float a = seg[lane];
  int above = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) above += __shfl_sync(0xffffffffu, a, i) > a;
  uint32_t least = 0xffffffffu;
  if (wide) {
    const float b = seg[lane + 32];
    int above_b = 0;
#pragma unroll 4
    for (int i = 0; i < 32; ++i) {
      const float oa = __shfl_sync(0xffffffffu, a, i), ob = __shfl_sync(0xffffffffu, b, i);
      above += ob > a;
      above_b += (oa > b) + (ob > b);
    }
    if (above_b < n) least = order_of(b);
  }
  if (above < n) least = min(least, order_of(a));
  return value_of(__reduce_min_sync(0xffffffffu, least));
}

template <class T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
logprobs_kernel(const __grid_constant__ LogprobArgs a, int parts) {
  __shared__ LogprobShared<THREADS> sh;
  using V = Vec<T>;
  constexpr int N = V::kN, kBatch = kUnroll * THREADS;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank();
  const int row = blockIdx.x / parts, n = a.n;
  if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");  // waited for before rank 0's shared memory is written
  wait_for_predecessor();

  const T* l = static_cast<const T*>(a.logits) + (int64_t)row * a.ld;
  const int head = min(a.V, (int)(((16 - ((uintptr_t)l & 15)) & 15) / sizeof(T)));
  const int n_vec = (a.V - head) / N, tail0 = head + n_vec * N;
  const int v0 = (int)((unsigned)n_vec * rank / (unsigned)parts), v1 = (int)((unsigned)n_vec * (rank + 1) / (unsigned)parts);  // n_vec < 2^29
  const uint4* body = reinterpret_cast<const uint4*>(l + head);

  uint4 cur[kUnroll], next[kUnroll];
  auto fetch = [&](int base) {
    if (base + kBatch <= v1) {
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) next[k] = load_stream(body + base + k * THREADS + tid);
    } else {
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        next[k] = make_uint4(V::kLowBits, V::kLowBits, V::kLowBits, V::kLowBits);  // adds nothing
        if (base + k * THREADS + tid < v1) next[k] = load_stream(body + base + k * THREADS + tid);
      }
    }
  };
  if (v0 < v1) fetch(v0);
  // The target's logit is asked for in two steps, each well before its result is needed.
  int64_t target = -1;
  T at_target{};
  if (tid == 0 && rank == 0 && a.logp != nullptr) target = a.targets[row];
  if (tid == 0) sh.count = sh.n_hot = 0;
  if (tid < kMaxTop) sh.best[tid] = 0;
  __syncthreads();
  auto push = [&](Entry e) {
    const int at = atomicAdd(&sh.count, 1);
    if (at < kCap) sh.list[at] = e;
  };
  float m = V::kLow, c = V::kLow * kLog2e;
  uint64_t s2 = 0, u2 = 0, s3 = 0, u3 = 0;  // two pairs of running sums
  auto raise_to = [&](float top) {
    const float nc = top * kLog2e, d = c - nc, f = exp2_fast(d);
    const uint64_t ff = pack2(f, f), dd = pack2(d, d);
    u2 = fma2(ff, fma2(dd, s2, u2), 0);
    u3 = fma2(ff, fma2(dd, s3, u3), 0);
    s2 = fma2(ff, s2, 0);
    s3 = fma2(ff, s3, 0);
    m = top;
    c = nc;
  };
  auto add_pair = [&](uint64_t v, uint64_t minus_c, uint64_t& s, uint64_t& u) {
    const uint64_t t = fma2(v, pack2(kLog2e, kLog2e), minus_c);
    float lo, hi;
    unpack2(t, lo, hi);
    const uint64_t e = pack2(exp2_fast(lo), exp2_fast(hi));
    s = add2(s, e);
    u = fma2(e, t, u);
  };
  // values before the first and behind the last 16-byte boundary
  if (rank == 0 && tid < head + a.V - tail0) {
    const int i = tid < head ? tid : tail0 + tid - head;
    const float v = widen_one(l[i]), raised = max_nan(v, V::kLow);
    if (raised > m) raise_to(raised);
    add_pair(pack2(raised, V::kLow), pack2(-c, -c), s2, u2);
    if (raised == V::kLow) s2 = u2 = 0;  // what a masked value and the filler would count for beside nothing else
    if (n > 0 && v > V::kLow) push(entry_of(v, (uint32_t)i));  // lower ones below, with those of the body
  }
  const float above_low = __int_as_float(__float_as_int(V::kLow) - 1);  // the next number; raised values are not noted
  float floor_v = above_low;
  // Many alternatives want more groups: the 32nd best of 32 maxima is their least, which some 130 values reach, and the lists of
  // rows of 50000 overflowed (300 of them, n = 32: 220 to 490 us; of 64 groups 27 us). Ranking 64 values takes every warp
  // three times as many shuffles (one row of 131072, n = 20, where 31 values reach the floor of 32 groups: 8.3 -> 9.6 us).
  const bool wide = n > 24;
  auto group_best = [&]() {
    float g = m;
#pragma unroll
    for (int d = 1; d < THREADS / 64; d <<= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, d));
    if (!wide) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, THREADS / 64));
    if (tid % (wide ? THREADS / 64 : THREADS / 32) == 0) sh.seg[tid / (wide ? THREADS / 64 : THREADS / 32)] = g;
  };
  int batch = 0;
  for (int base = v0; base < v1; base += kBatch, ++batch) {
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) cur[k] = next[k];
    if (base + kBatch < v1) fetch(base + kBatch);
    uint32_t top_w = V::kLowBits;
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      cur[k].x = V::raise(cur[k].x);
      cur[k].y = V::raise(cur[k].y);
      cur[k].z = V::raise(cur[k].z);
      cur[k].w = V::raise(cur[k].w);
      top_w = V::larger(top_w, V::larger(V::larger(cur[k].x, cur[k].y), V::larger(cur[k].z, cur[k].w)));
    }
    const float all = V::top(top_w);
    if (all > m) raise_to(all);
    const uint64_t minus_c = pack2(-c, -c);
#pragma unroll
    for (int k = 0; k < kUnroll; ++k)
#pragma unroll
      for (int i = 0; i < N / 2; i += 2) {
        add_pair(V::pair(cur[k], i), minus_c, s2, u2);
        add_pair(V::pair(cur[k], i + 1), minus_c, s3, u3);
      }
    if (n == 0) continue;
    if ((batch & (batch + 1)) == 0 && (batch == 0 || base + kBatch < v1)) {  // batches 0, 1, 3, 7, ...
      group_best();
      // At first every group has to have its value there. Later a warp may see other groups' older, lower ones: they are
      // maxima of those groups all the same. (It takes them once: they may rise while it compares them.)
      if (batch == 0) __syncthreads();
      else __syncwarp();
      floor_v = fmaxf(nth_best(sh.seg, wide, n), above_low);
    }
    if (all >= floor_v) {
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int v = base + k * THREADS + tid;
        if (V::top(V::larger(V::larger(cur[k].x, cur[k].y), V::larger(cur[k].z, cur[k].w))) >= floor_v && v < v1) {
          const int at = atomicAdd(&sh.n_hot, 1);
          if (at < kCap) sh.hot[at] = v;
        }
      }
    }
  }

  if (target >= 0 && target < a.V) at_target = l[target];

  // sums of the thread, the warp, the CTA
  Sums a0;
  {
    float s_lo, s_hi, u_lo, u_hi;
    unpack2(add2(s2, s3), s_lo, s_hi);
    unpack2(add2(u2, u3), u_lo, u_hi);
    a0 = Sums{m, c, s_lo + s_hi, u_lo + u_hi};
  }
  join_lanes(a0, 32);
  if (lane == 0) sh.warp_sums[warp] = a0;
  if (n > 0 && batch > 1) group_best();
  __syncthreads();
  if (parts > 1) cluster_wait_diverged();
  if (warp == 0) {
    Sums t = lane < THREADS / 32 ? sh.warp_sums[lane] : no_sums<T>();
    join_lanes(t, THREADS / 32);
    if (lane == 0) {
      if (parts == 1) sh.part = t;
      else
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(map_to_rank(smem_u32(&sh.part_sums[rank]), 0)),
                     "f"(t.m), "f"(t.c), "f"(t.s), "f"(t.u) : "memory");
    }
  }
  if (n > 0) {
    const bool all_hot = sh.n_hot <= kCap;
    int count = 0;
    if (all_hot) {
      // the noted vectors once more, against the last floor
      // (after a single batch the loop's is the last)
      if (batch > 1) floor_v = fmaxf(nth_best(sh.seg, wide, n), above_low);
      const bool low = floor_v == above_low;
      for (int i = tid; i < sh.n_hot; i += THREADS) {
        const int at = head + sh.hot[i] * N;
        const uint4 w = body[sh.hot[i]];
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float x = widen_one(reinterpret_cast<const T*>(&w)[j]);
          if (x >= floor_v) push(entry_of(x, (uint32_t)(at + j)));
        }
      }
      __syncthreads();
      count = sh.count;
      if (low) __syncthreads();
      if (low && count < n) {  // finite values from kLow down, if there are any
        for (int v = v0 + tid; v < v1; v += 4 * THREADS) {
          uint4 w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (v + k * THREADS < v1) w[k] = body[v + k * THREADS];
#pragma unroll 1
          for (int k = 0; k < 4; ++k) {
            if (v + k * THREADS >= v1) break;
            const uint4 x4 = k == 0 ? w[0] : k == 1 ? w[1] : k == 2 ? w[2] : w[3];
#pragma unroll
            for (int j = 0; j < N; ++j) {
              const float x = widen_one(reinterpret_cast<const T*>(&x4)[j]);
              if (x > -CUDART_INF_F && x <= V::kLow) push(entry_of(x, (uint32_t)(head + (v + k * THREADS) * N + j)));
            }
          }
        }
        if (rank == 0 && tid < head + a.V - tail0) {
          const int i = tid < head ? tid : tail0 + tid - head;
          const float x = widen_one(l[i]);
          if (x > -CUDART_INF_F && x <= V::kLow) push(entry_of(x, (uint32_t)i));
        }
        __syncthreads();
        count = sh.count;
      }
    }
    if (!all_hot || count > kCap) {
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
      const Entry least = sh.prefix;  // the n-th largest, or the lowest if there are fewer
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
    rank_list<THREADS>(sh.list, count, n, parts == 1 ? smem_u32(sh.best) : map_to_rank(smem_u32(&sh.part_best[rank * n]), 0));
  }
  if (parts > 1) {
    cluster_arrive_diverged();
    if (rank != 0) return;
    cluster_wait_diverged();  // the parts' sums and best are there
    if (warp == 0) {
      Sums t = lane < parts ? sh.part_sums[lane] : no_sums<T>();
      join_lanes(t, kMaxParts);
      if (lane == 0) sh.part = t;
    }
    // Entries of 0 rank behind every other. Of many, only those that reach the least of the parts' ceil(n / parts)-th best, at least
    // n of them, are ranked (160 of 8 parts: 1.8 us all of them).
    if (n > 0 && parts * n <= THREADS / 4) {
      rank_list<THREADS>(sh.part_best, parts * n, n, smem_u32(sh.best));
    } else if (n > 0) {
      Entry least = ~(Entry)0;
      for (int p = 0; p < parts; ++p) least = min(least, sh.part_best[p * n + (n - 1) / parts]);
      if (tid == 0) sh.count = 0;
      __syncthreads();
      for (int i = tid; i < parts * n; i += THREADS)
        if (sh.part_best[i] >= least && sh.part_best[i] != 0) push(sh.part_best[i]);
      __syncthreads();
      rank_list<THREADS>(sh.list, sh.count, n, smem_u32(sh.best));
    }
  }
  __syncthreads();

  Sums t = sh.part;
  bool again = !(t.m > V::kLow + kFar) || t.m > kPlain;
  // Neither NaN nor anything above -inf: no distribution, without a second look (33 x 50001 with one such row: 9.5 -> 6.0 us).
  if (again && n > 0 && sh.best[0] == 0 && t.m == V::kLow && t.s == t.s) {
    again = false;
    t.s = 0.f;
  }
  if (again) {
    // A row of the type's lowest values, or of a size at which c is too coarse: its true maximum, and everything relative to it
    auto whole_row = [&](auto f) {
      if (tid < head + a.V - tail0) f(widen_one(l[tid < head ? tid : tail0 + tid - head]));
      for (int v = tid; v < n_vec; v += 4 * THREADS) {
        uint4 w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (v + k * THREADS < n_vec) w[k] = body[v + k * THREADS];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (v + k * THREADS < n_vec) {
#pragma unroll
            for (int j = 0; j < N; ++j) f(widen_one(reinterpret_cast<const T*>(&w[k])[j]));
          }
      }
    };
    float top = -CUDART_INF_F;
    bool bad = false;
    whole_row([&](float v) {
      bad |= v != v;
      top = fmaxf(top, v);
    });
    top = value_of(__reduce_max_sync(0xffffffffu, order_of(top)));
    if (lane == 0) sh.warp_sums[warp].m = top;
    bad = __syncthreads_or(bad);
    for (int w = 0; w < THREADS / 32; ++w) top = fmaxf(top, sh.warp_sums[w].m);
    float s = 0.f, u = 0.f;
    if (fabsf(top) < CUDART_INF_F)
      whole_row([&](float v) {
        const float d = (v - top) * kLog2e, e = exp2_fast(d);
        s += e;
        u = fmaf(e, fmaxf(d, -1e4f), u);
      });
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, d);
      u += __shfl_xor_sync(0xffffffffu, u, d);
    }
    __syncthreads();
    if (lane == 0) {
      sh.warp_sums[warp].s = s;
      sh.warp_sums[warp].u = u;
    }
    __syncthreads();
    t = Sums{top, 0.f, 0.f, 0.f};
    for (int w = 0; w < THREADS / 32; ++w) {
      t.s += sh.warp_sums[w].s;
      t.u += sh.warp_sums[w].u;
    }
    if (bad) t.s = CUDART_NAN_F;
  }
  if (warp != 0) return;
  const bool dead = !(t.s > 0.f) || !(fabsf(t.m) < CUDART_INF_F);
  const float log_s = logf(t.s);
  const double lse = dead ? CUDART_NAN : (again ? (double)t.m : (double)t.c * kPerC) + (double)log_s;
  if (lane == 0) {
    if (a.logp != nullptr) {
      a.logp[row] = target < 0 ? 0.f : dead || target >= a.V ? CUDART_NAN_F : (float)((double)widen_one(at_target) - lse);
    }
    if (a.entropy != nullptr) a.entropy[row] = dead ? CUDART_NAN_F : fmaf(-kLn2, t.u / t.s, log_s);
  }
  if (lane < n) {
    const Entry e = dead ? 0 : sh.best[lane];
    a.top_ids[(int64_t)row * n + lane] = e == 0 ? -1 : (int32_t)(0xffffffffu - (uint32_t)e);
    a.top_logp[(int64_t)row * n + lane] =
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
  while (parts < kMaxParts && (int64_t)a.T * parts * 2 <= 2 * sms && a.V / (2 * parts) >= 4096) parts *= 2;
  // Every thread should have half a batch, and each of the 32 groups of threads values for the floor. Parts of a row are
  // short: more threads finish sooner. Whole rows leave room for other rows' CTAs, which work while one row is finished.
  const int vectors = a.V / parts / Vec<T>::kN;
  if (parts > 1 && vectors >= 512 * kUnroll / 2) return launch<T, 512>(a, parts, s);
  if (vectors >= 256 * kUnroll / 2) return launch<T, 256>(a, parts, s);
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
