// y = act(x w^T + bias) + residual: x [M, K] tokens, w [N, K] weights, bf16 or fp16, float32 sums, one rounding at the end.
//
// Tensor-core kernel (linear_tc_kernel): weight rows are the M operand of tcgen05.mma, token rows the N operand, because N
// can be any multiple of 16: one token costs a 16-column tile, a prompt of 777 four tiles of 208. TMA brings both in steps
// of 64 k into a ring, one thread issues the MMAs, eight warps drain the accumulators (double-buffered in
// tensor memory) through bias, activation and residual. A lane holds one weight row, so the bias is one load per tile and
// the lanes of a warp store 32 neighbouring outputs of a token, whatever the alignment of y.
// Three shapes of it, chosen by launch_linear:
//   pairs   CTA pairs (cta_group::2) on 256 weight rows x up to 256 tokens, persistent: many tokens
//   single  one CTA on 128 weight rows, persistent: few tokens against many weight rows
//   split   a cluster of up to 8 CTAs shares the k steps of one tile and adds its partial sums through distributed shared
//           memory, in the order of the ranks: too few tiles for the GPU
//
// Rows that do not start on 16-byte boundaries cannot be fetched by TMA: linear_plain_kernel (mma.sync, plain loads).
//
// Every mbarrier wait is bounded. On a give-up the outputs of the tile become NaN and *err (optional) a code.
#include <algorithm>

#include "pm_common.cuh"
#include "sm100_ptx.cuh"

namespace pm {
namespace {

using namespace sm100;

constexpr int kEpiWarps = 8;
constexpr int kTcThreads = (4 + kEpiWarps) * 32;
constexpr int kWBytes = 128 * 128;  // a CTA's 128 weight rows of a k step
constexpr int kMaxStages = 12;
constexpr int kSmemMost = 232448;

struct LinearTc {
  void* y;
  const void *res, *bias;
  int64_t ldy, ldr;
  int32_t M, N, k_tiles, act, bias_type, f16;
  int32_t width, tok_tiles, w_tiles;  // token columns of a tile; tiles
  int32_t stage_bytes, n_stages, ring_bytes;
  int32_t split, tmem_cols;
  int32_t* err;
};

struct LinShared {
  uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  volatile int abort;
};

template <class T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float(float v) { return v; }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }

// Plain loads: the 16-bit forms of __ldg are pure inline assembly, which the compiler may move in front of the test for a
// null pointer or an end.
__device__ __forceinline__ float load_bias(const void* bias, int type, int n) {
  if (bias == nullptr) return 0.f;
  if (type == PM_F32) return static_cast<const float*>(bias)[n];
  if (type == PM_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[n]);
  return __half2float(static_cast<const __half*>(bias)[n]);
}

template <int ACT>
__device__ __forceinline__ float activate(float v) {
  if (ACT == PM_ACT_RELU) return v < 0.f ? 0.f : v;  // NaN stays
  if (ACT == PM_ACT_SILU) return v / (1.f + __expf(-v));
  if (ACT == PM_ACT_GELU) return 0.5f * v * erfcf(v * -0.70710678118654752f);
  if (ACT == PM_ACT_GELU_TANH)  // 0.5 v (1 + tanh u) = v / (1 + exp(-2u))
    return v / (1.f + __expf(-1.5957691216057308f * (v + 0.044715f * v * v * v)));
  return v;
}
template <int N>
__device__ __forceinline__ void activate_all(float (&v)[N], int act) {
  auto all = [&](auto f) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = f(v[i]);
  };
  switch (act) {
    case PM_ACT_RELU: return all(activate<PM_ACT_RELU>);
    case PM_ACT_SILU: return all(activate<PM_ACT_SILU>);
    case PM_ACT_GELU: return all(activate<PM_ACT_GELU>);
    case PM_ACT_GELU_TANH: return all(activate<PM_ACT_GELU_TANH>);
  }
}
__device__ __forceinline__ float activate_one(float v, int act) {
  float a[1] = {v};
  activate_all(a, act);
  return a[0];
}

// Weight tile and token tile of a position: eight weight tiles at a time against all token tiles, so that what the GPU
// works on at once is a nearly square part of y.
__device__ __forceinline__ void tile_at(const LinearTc& a, int tile, int& wt, int& tt) {
  constexpr int kBand = 8;
  const int band = tile / (kBand * a.tok_tiles), in = tile - band * kBand * a.tok_tiles;
  const int high = min(kBand, a.w_tiles - band * kBand);
  tt = in / high;
  wt = band * kBand + in - tt * high;
}

template <int CG, class OT>
__global__ void __launch_bounds__(kTcThreads, 1)
linear_tc_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                 const __grid_constant__ LinearTc a) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* stages = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  LinShared& sh = *reinterpret_cast<LinShared*>(stages + a.ring_bytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int per_tile = CG == 2 ? 2 : a.split;  // CTAs on one tile
  const int first = blockIdx.x / per_tile, step = gridDim.x / per_tile;
  const int n_tiles = a.w_tiles * a.tok_tiles, n_stages = a.n_stages;
  const bool split = CG == 1 && a.split > 1;
  const int k0 = split ? (int)((long long)a.k_tiles * rank / a.split) : 0;
  const int k1 = split ? (int)((long long)a.k_tiles * (rank + 1) / a.split) : a.k_tiles;

  if (threadIdx.x == 0) {
    for (int s = 0; s < n_stages; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.acc_full[i], 1);
      mbar_init(&sh.acc_empty[i], CG * kEpiWarps);
    }
    sh.abort = 0;
    fence_barrier_init();
  }
  if (warp == 2) {
    if (CG == 2) tmem_alloc(&sh.tmem_base, a.tmem_cols);
    else tmem_alloc_single(&sh.tmem_base, a.tmem_cols);
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync_diverged();
  tc_fence_after();
  const uint32_t tmem_base = sh.tmem_base;
  const uint32_t acc_cols = a.tmem_cols / 2;  // distance of the two accumulators
  let_successor_start();
  wait_for_predecessor();

  if (warp == 0 && lane == 0) {
    // ---- producer: 128 weight rows and this CTA's share of the token rows ----------------------------
    const int rows = a.width / CG;
    int at = 0, steps = 0;
    uint32_t turn = 0;
    bool ok = true;
    for (int tile = first; tile < n_tiles && ok; tile += step) {
      int wt, tt;
      tile_at(a, tile, wt, tt);
      const int w_row = wt * 128 * CG + (CG == 2 ? (int)rank * 128 : 0);
      const int x_row = tt * a.width + (CG == 2 ? (int)rank * rows : 0);
      for (int kt = k0; kt < k1; ++kt, ++steps) {
        if (turn > 0 && !mbar_wait(&sh.empty[at], (turn - 1) & 1, &sh.abort)) {
          ok = false;
          break;
        }
        unsigned char* dst = stages + (size_t)at * a.stage_bytes;
        if (CG == 2) {
          if (rank == 0) mbar_arrive_expect_tx(&sh.full[at], 2 * a.stage_bytes);
          const uint32_t bar = map_to_rank(smem_u32(&sh.full[at]), 0);
          tma_load_2d(dst, &map_w, bar, kt * 64, w_row);
          tma_load_2d(dst + kWBytes, &map_x, bar, kt * 64, x_row);
        } else {
          mbar_arrive_expect_tx(&sh.full[at], a.stage_bytes);
          tma_load_2d_single(dst, &map_w, &sh.full[at], kt * 64, w_row);
          tma_load_2d_single(dst + kWBytes, &map_x, &sh.full[at], kt * 64, x_row);
        }
        if (++at == n_stages) {
          at = 0;
          ++turn;
        }
      }
    }
    // the last arrivals on this CTA's barriers must have landed before its shared memory goes away
    for (int k = max(0, steps - n_stages); k < steps && ok; ++k)
      ok = mbar_wait(&sh.empty[k % n_stages], (k / n_stages) & 1, &sh.abort);
    if (!ok) sh.abort = 1;
  } else if (warp == 1 && lane == 0 && (CG == 1 || rank == 0)) {
    // ---- MMA issuer ----------------------------------------------------------------------------------
    const uint32_t idesc = a.f16 ? umma_idesc_f16(128 * CG, a.width) : umma_idesc_bf16(128 * CG, a.width);
    int at = 0, it = 0;
    uint32_t turn = 0;
    bool ok = true;
    for (int tile = first; tile < n_tiles && ok; tile += step, ++it) {
      const int acc = it & 1;
      if (it >= 2 && !mbar_wait(&sh.acc_empty[acc], ((it >> 1) - 1) & 1, &sh.abort)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t d = tmem_base + (uint32_t)acc * acc_cols;
      for (int kt = k0; kt < k1; ++kt) {
        if (!mbar_wait(&sh.full[at], turn & 1, &sh.abort)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t addr = smem_u32(stages + (size_t)at * a.stage_bytes);
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // 16 k = 32 bytes inside the swizzled row
          const uint64_t da = umma_desc_k_sw128(addr + k * 32), db = umma_desc_k_sw128(addr + kWBytes + k * 32);
          const uint32_t more = (kt > k0 || k > 0) ? 1u : 0u;
          if (CG == 2) umma_bf16(d, da, db, idesc, more);
          else umma_single(d, da, db, idesc, more);
        }
        if (CG == 2) umma_commit_pair(&sh.empty[at]);
        else umma_commit_single(&sh.empty[at]);
        if (++at == n_stages) {
          at = 0;
          ++turn;
        }
      }
      if (ok) {
        if (CG == 2) umma_commit_pair(&sh.acc_full[acc]);
        else umma_commit_single(&sh.acc_full[acc]);
      }
    }
    if (!ok) sh.abort = 1;
  } else if (warp >= 4) {
    // ---- epilogue: warp w drains accumulator rows 32w .. 32w+31, two warps of a quadrant share the columns ------
    const int w = warp & 3, half = (warp - 4) >> 2;
    const float nan = __int_as_float(0x7fffffff);
    int it = 0;
    bool ok = true;
    for (int tile = first; tile < n_tiles; tile += step, ++it) {
      int wt, tt;
      tile_at(a, tile, wt, tt);
      const int acc = it & 1;
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&sh.acc_full[acc], (it >> 1) & 1, &sh.abort));
      tc_fence_after();
      const uint32_t taddr = tmem_base + (uint32_t)acc * acc_cols + ((uint32_t)(32 * w) << 16);
      const int n = wt * 128 * CG + (CG == 2 ? (int)rank * 128 : 0) + 32 * w + lane;
      const int m0 = tt * a.width, cols = min(a.width, a.M - m0);
      if (split) {
        // partial sums to shared memory (the ring is empty now), column by column
        float* part = reinterpret_cast<float*>(stages);
        for (int c0 = half * 32; c0 < cols; c0 += 64) {
          uint32_t v[32];
          tmem_ld32(taddr + c0, v);
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (c0 + c < cols) part[(c0 + c) * 128 + 32 * w + lane] = ok ? __uint_as_float(v[c]) : nan;
        }
        continue;
      }
      const float b = n < a.N ? load_bias(a.bias, a.bias_type, n) : 0.f;
      for (int c0 = half * 32; c0 < cols; c0 += 64) {
        uint32_t v[32];
        tmem_ld32(taddr + c0, v);
        const int left = n < a.N ? cols - c0 : 0;
        OT r[32];
        if (a.res != nullptr) {
          const OT* src = static_cast<const OT*>(a.res) + (int64_t)(m0 + c0) * a.ldr + n;
#pragma unroll
          for (int c = 0; c < 32; ++c) r[c] = c < left ? src[c * a.ldr] : from_float<OT>(0.f);
        }
        tmem_ld_wait();
        float o[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) o[c] = ok ? __uint_as_float(v[c]) + b : nan;
        activate_all(o, a.act);
        if (a.res != nullptr) {
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] += to_float<OT>(r[c]);
        }
        OT* dst = static_cast<OT*>(a.y) + (int64_t)(m0 + c0) * a.ldy + n;
#pragma unroll
        for (int c = 0; c < 32; ++c)
          if (c < left) dst[c * a.ldy] = from_float<OT>(o[c]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CG == 2) mbar_arrive_cluster(map_to_rank(smem_u32(&sh.acc_empty[acc]), 0));
        else mbar_arrive(smem_u32(&sh.acc_empty[acc]));
      }
    }
    if (!ok && lane == 0) sh.abort = 1;
  }
  __syncwarp();
  if (split) {
    __syncthreads();
    cluster_sync_diverged();  // every rank's partial sums are in place
    if (warp >= 4) {
      int wt, tt;
      tile_at(a, first, wt, tt);
      const int m0 = tt * a.width, cols = min(a.width, a.M - m0);
      const uint32_t part = smem_u32(stages);
      for (int task = (warp - 4) + kEpiWarps * (int)rank; task < cols * 4; task += kEpiWarps * a.split) {
        const int c = task >> 2, row = (task & 3) * 32 + lane, n = wt * 128 + row;
        float v = 0.f;
        for (int r = 0; r < a.split; ++r) {
          float p;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(p) : "r"(map_to_rank(part, r) + 4u * (uint32_t)(c * 128 + row)));
          v += p;
        }
        if (n < a.N) {
          v = activate_one(v + load_bias(a.bias, a.bias_type, n), a.act);
          if (a.res != nullptr) v += to_float<OT>(static_cast<const OT*>(a.res)[(int64_t)(m0 + c) * a.ldr + n]);
          static_cast<OT*>(a.y)[(int64_t)(m0 + c) * a.ldy + n] = from_float<OT>(v);
        }
      }
    }
  }
  __syncthreads();
  if (sh.abort) {
    if (threadIdx.x == 0 && a.err != nullptr) atomicExch(a.err, 1);
    // give loads that are still in flight time to land before the shared memory is released
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2 || split) cluster_sync_diverged();
  tc_fence_after();
  if (warp == 2) {
    if (CG == 2) tmem_dealloc(tmem_base, a.tmem_cols);
    else tmem_dealloc_single(tmem_base, a.tmem_cols);
  }
}

// ---- rows that TMA cannot fetch -------------------------------------------------------------------------
// Tiles of 64 tokens x 64 weight rows, steps of 32 k through shared memory, eight warps of 32 x 16 outputs, the next step's
// values fetched into registers while the present one is multiplied. Loads are 2 bytes per lane, a warp reads one row's 64 bytes.
constexpr int kPlainTok = 64, kPlainW = 64, kPlainK = 32, kPlainPitch = kPlainK + 8;

template <class T>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&x)[4], const uint32_t (&w)[2]);
template <>
__device__ __forceinline__ void mma_16x8x16<__nv_bfloat16>(float (&d)[4], const uint32_t (&x)[4], const uint32_t (&w)[2]) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(w[0]), "r"(w[1]));
}
template <>
__device__ __forceinline__ void mma_16x8x16<__half>(float (&d)[4], const uint32_t (&x)[4], const uint32_t (&w)[2]) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(w[0]), "r"(w[1]));
}

template <class T, class OT>
__global__ void __launch_bounds__(256)
linear_plain_kernel(const __grid_constant__ LinearCall a) {
  __shared__ __align__(16) uint16_t xs[kPlainTok * kPlainPitch], ws[kPlainW * kPlainPitch];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int w_tiles = (a.N + kPlainW - 1) / kPlainW;
  const int m0 = blockIdx.x / w_tiles * kPlainTok, n0 = blockIdx.x % w_tiles * kPlainW;
  const int wm = (warp & 1) * 32, wn = (warp >> 1) * 16;
  wait_for_predecessor();
  const uint16_t* __restrict__ x = static_cast<const uint16_t*>(a.x);
  const uint16_t* __restrict__ w = static_cast<const uint16_t*>(a.w);
  float acc[2][2][4] = {};
  uint16_t xr[8], wr[8];
  auto fetch = [&](int k0) {
    const int k = k0 + lane;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int m = m0 + warp + 8 * i, n = n0 + warp + 8 * i;
      xr[i] = m < a.M && k < a.K ? x[(int64_t)m * a.ldx + k] : (uint16_t)0;
      wr[i] = n < a.N && k < a.K ? w[(int64_t)n * a.ldw + k] : (uint16_t)0;
    }
  };
  fetch(0);
  for (int k0 = 0; k0 < a.K; k0 += kPlainK) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      xs[(warp + 8 * i) * kPlainPitch + lane] = xr[i];
      ws[(warp + 8 * i) * kPlainPitch + lane] = wr[i];
    }
    __syncthreads();
    if (k0 + kPlainK < a.K) fetch(k0 + kPlainK);
    const int g = lane >> 2, q = (lane & 3) * 2;
#pragma unroll
    for (int kk = 0; kk < kPlainK; kk += 16) {
      uint32_t xf[2][4], wf[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint16_t* p = xs + (wm + 16 * i + g) * kPlainPitch + kk + q;
        xf[i][0] = *reinterpret_cast<const uint32_t*>(p);
        xf[i][1] = *reinterpret_cast<const uint32_t*>(p + 8 * kPlainPitch);
        xf[i][2] = *reinterpret_cast<const uint32_t*>(p + 8);
        xf[i][3] = *reinterpret_cast<const uint32_t*>(p + 8 * kPlainPitch + 8);
        const uint16_t* v = ws + (wn + 8 * i + g) * kPlainPitch + kk + q;
        wf[i][0] = *reinterpret_cast<const uint32_t*>(v);
        wf[i][1] = *reinterpret_cast<const uint32_t*>(v + 8);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) mma_16x8x16<T>(acc[i][j], xf[i], wf[j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int m = m0 + wm + 16 * i + (lane >> 2) + (e >> 1) * 8, n = n0 + wn + 8 * j + (lane & 3) * 2 + (e & 1);
        if (m < a.M && n < a.N) {
          float v = activate_one(acc[i][j][e] + load_bias(a.bias, a.bias_type, n), a.act);
          if (a.res != nullptr) v += to_float<OT>(static_cast<const OT*>(a.res)[(int64_t)m * a.ldr + n]);
          static_cast<OT*>(a.y)[(int64_t)m * a.ldy + n] = from_float<OT>(v);
        }
      }
}

template <class T>
cudaError_t launch_plain(const LinearCall& a, cudaStream_t s) {
  const long long tiles = (long long)((a.N + kPlainW - 1) / kPlainW) * ((a.M + kPlainTok - 1) / kPlainTok);
  if (tiles > 0x7fffffffll) return cudaErrorInvalidValue;
  const unsigned grid = (unsigned)tiles;
  if (a.out_type == PM_F32) return launch_behind(linear_plain_kernel<T, float>, grid, 256, 0, s, a);
  return launch_behind(linear_plain_kernel<T, T>, grid, 256, 0, s, a);
}

// ---- launch plan ------------------------------------------------------------------------------------------
struct LinearShape {
  int cg = 1, split = 1, tok_tiles = 1, width = 16;
};

// Estimated cycles of a shape. A k step of 64 takes 2 cycles per token column on the tensor cores, and its operands
// come from L2 at about 48 bytes per cycle and SM; the rest is what a tile and a launch cost besides.
double shape_cost(const LinearShape& c, int N, int k_tiles, int sms) {
  const int w_tiles = (N + 128 * c.cg - 1) / (128 * c.cg), units = sms / c.cg;
  const long long ctas = (long long)w_tiles * c.tok_tiles * c.split;
  const long long waves = (ctas + units - 1) / units;
  const double step = std::max(2.0 * c.width, (kWBytes + c.width / c.cg * 128) / 48.0);
  const int steps = (k_tiles + c.split - 1) / c.split;
  return waves * (steps * step + 600.0 + (c.split > 1 ? 1200.0 + 8.0 * c.width : 0.0)) + 2.0 * c.width;
}

LinearShape choose_shape(int M, int N, int k_tiles, int sms) {
  LinearShape best;
  double cost = 0;
  for (int cg = 1; cg <= 2; ++cg) {
    const int grain = 16 * cg, least = (M + 255) / 256;
    for (int t = least; t <= least + 3; ++t)
      for (int split = 1; split <= (cg == 1 ? 8 : 1); ++split) {
        if (split > k_tiles) break;
        LinearShape c;
        c.cg = cg;
        c.split = split;
        c.width = ((M + t - 1) / t + grain - 1) / grain * grain;
        c.tok_tiles = (M + c.width - 1) / c.width;
        const double x = shape_cost(c, N, k_tiles, sms);
        if (cost == 0 || x < cost) {
          cost = x;
          best = c;
        }
      }
  }
  return best;
}

template <int CG, class OT>
cudaError_t launch_tc(const CUtensorMap& map_w, const CUtensorMap& map_x, const LinearTc& t, int grid, int cluster, size_t smem,
                      cudaStream_t s) {
  static SmemOptIn once;
  auto kern = linear_tc_kernel<CG, OT>;
  cudaError_t e = opt_in_smem(once, kern);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = kTcThreads;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)cluster, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, map_w, map_x, t);
}

template <int CG>
cudaError_t launch_tc_for(int out_type, const CUtensorMap& map_w, const CUtensorMap& map_x, const LinearTc& t, int grid,
                          int cluster, size_t smem, cudaStream_t s) {
  if (out_type == PM_F32) return launch_tc<CG, float>(map_w, map_x, t, grid, cluster, smem, s);
  if (out_type == PM_BF16) return launch_tc<CG, __nv_bfloat16>(map_w, map_x, t, grid, cluster, smem, s);
  return launch_tc<CG, __half>(map_w, map_x, t, grid, cluster, smem, s);
}

bool tma_rows(const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && ld < ((int64_t)1 << 38); }

}  // namespace

int launch_linear(const LinearCall& a, cudaStream_t s) {
  if (!tma_rows(a.x, a.ldx) || !tma_rows(a.w, a.ldw)) {
    PM_CUDA(a.type == PM_BF16 ? launch_plain<__nv_bfloat16>(a, s) : launch_plain<__half>(a, s));
    return PM_OK;
  }
  int dev = 0, sms = 0;
  PM_CUDA(cudaGetDevice(&dev));
  PM_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  const int k_tiles = (a.K + 63) / 64;
  const LinearShape c = choose_shape(a.M, a.N, k_tiles, sms);
  LinearTc t{};
  t.y = a.y; t.res = a.res; t.bias = a.bias;
  t.ldy = a.ldy; t.ldr = a.ldr;
  t.M = a.M; t.N = a.N; t.k_tiles = k_tiles; t.act = a.act; t.bias_type = a.bias_type; t.f16 = a.type == PM_F16;
  t.width = c.width; t.tok_tiles = c.tok_tiles; t.w_tiles = (a.N + 128 * c.cg - 1) / (128 * c.cg);
  t.split = c.split; t.err = a.err;
  t.stage_bytes = kWBytes + c.width / c.cg * 128;
  const int room = kSmemMost - 1024 - (int)sizeof(LinShared), steps = (k_tiles + c.split - 1) / c.split;
  const long long n_tiles = (long long)t.w_tiles * t.tok_tiles, units = sms / c.cg;
  const long long tiles_each = c.split > 1 ? 1 : (n_tiles + units - 1) / units;
  t.n_stages = (int)std::min<long long>(std::min(kMaxStages, room / t.stage_bytes), steps * tiles_each);
  t.ring_bytes = t.stage_bytes * t.n_stages;
  if (c.split > 1) t.ring_bytes = std::max(t.ring_bytes, c.width * 512);
  t.tmem_cols = 64;  // two accumulators, each at a multiple of 32 columns; the allocation is a power of two
  while (t.tmem_cols < 2 * c.width) t.tmem_cols *= 2;
  CUtensorMap map_w, map_x;
  int rc = tc_encode_matrix(&map_w, a.w, a.K, a.N, a.ldw, 128);
  if (rc != PM_OK) return rc;
  rc = tc_encode_matrix(&map_x, a.x, a.K, a.M, a.ldx, c.width / c.cg);
  if (rc != PM_OK) return rc;
  // Beside the grouped FFN's kernel, which takes all tensor memory after it has let its successor in, no block of this one
  // may start (each would wait for the other): 64 KB do not fit there. Pairs allocate together, so only one per SM.
  const size_t smem = std::max<size_t>(1024 + t.ring_bytes + sizeof(LinShared), (c.cg == 2 ? 120 : 64) * 1024);
  const int cluster = c.cg == 2 ? 2 : c.split;
  if (n_tiles * c.split > 0x7fffffffll) return fail(PM_ERR_INVALID, "linear: too many tiles");
  const long long grid = c.split > 1 ? n_tiles * c.split : std::min(n_tiles, units) * c.cg;
  PM_CUDA(c.cg == 2 ? launch_tc_for<2>(a.out_type, map_w, map_x, t, (int)grid, cluster, smem, s)
                    : launch_tc_for<1>(a.out_type, map_w, map_x, t, (int)grid, cluster, smem, s));
  return PM_OK;
}

}  // namespace pm
