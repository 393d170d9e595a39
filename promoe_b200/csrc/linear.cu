// y = act(x w^T + bias) + residual: x [M, K] tokens, w [N, K] weights, bf16 or fp16, float32 sums, one rounding at the end.
//
// More than 16 tokens: linear_tc_kernel. Weight rows are the M operand of tcgen05.mma, token rows the N operand, because N can
// be any multiple of 16: 33 tokens cost 48 columns, a prompt of 777 nine tiles of 96. TMA brings both in steps of 64 or 128 k
// into a ring, one thread issues the MMAs, eight warps drain the accumulators (double-buffered in tensor memory)
// through bias, activation and residual. A lane holds one weight row, so the bias is one load per tile and the lanes of a
// warp store 32 neighbouring outputs of a token, whatever the alignment of y. Three shapes of it, chosen by an estimate of
// their time (shape_cost):
//   pairs   CTA pairs (cta_group::2) on 256 weight rows x up to 256 tokens, persistent
//   single  one CTA on 128 weight rows, persistent
//   split   a cluster of up to 8 CTAs shares the k steps of one tile and adds its partial sums through distributed shared
//           memory, in the order of the ranks: too few tiles for the GPU
// What bounds it. Large products the tensor cores under the power limit: 8192 x 4096 -> 14336 takes 645 us in a burst = 1.49 PFLOP/s,
// 0.92 of measured, and 742 us sustained. Few tokens against many weights HBM: 33 x 2048 -> 100003 68 us = 6.0 TB/s, 0.92 of measured. Between them an
// SM's intake, 124 bytes per ns at most: 777 x 5632 -> 2048 (tiles of 256 x 96, 22 KB for 64 k and SM) 25 us where the
// MMAs alone would take 9. And what comes before and after the k steps: setup and first load 1.5 us, a tile's epilogue
// 0.3 us for each 16 columns and half (a warp's store or remote store of 16 columns takes 600 cycles), joining partial sums 0.7 us for the
// cluster barrier and as much for the sums. 64 x 4096 -> 4096 11 us, 512 x 3584 -> 4608 18 us.
//
// At most 16 tokens: linear_few_kernel (mma.sync), which streams the weights straight into registers. Rows that do not start on
// 16-byte boundaries cannot be fetched by TMA: linear_plain_kernel (mma.sync, plain loads) for more tokens than that.
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
// k of one accumulator of float32 outputs. The tensor cores cut their running sums off where float32 ends, which shrinks a sum by
// about 2^-24 of itself per addition of 16 k: 2.1e-6 for K = 2048 in one accumulator, 4.7e-7 in four. (16-bit results take one: their own
// rounding is 2^-9 or 2^-12, which that reaches where K is half a million or 65536; the sums of 256 columns would not fit the
// epilogue's registers.)
constexpr int kPromoteK = 512;

struct LinearTc {
  void* y;
  const void *res, *bias;
  int64_t ldy, ldr;
  int32_t M, N, k_tiles, act, bias_type, f16;
  int32_t width, tok_tiles, w_tiles;  // token columns of a tile; tiles
  int32_t atoms, stage_bytes, n_stages;  // 64-k atoms of a step; k_tiles counts steps
  int32_t chunk;                         // steps that one accumulator takes
  int32_t split, part_offset, shared_bytes;  // CTAs (pairs) on a tile; their partial sums behind the ring; all of these bytes
  int32_t part_cols;                         // columns that each of them finishes, a multiple of 4
  int32_t tmem_cols;
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

// sigma(z) = (z > 0 ? 1 : e) / (1 + e), e = exp(-|z|): nothing overflows, and small values keep their digits. Results of 16 bits take the
// quick exponential, off by 2 + 1.2 |z| steps of float32 (their own rounding is 2^-9 or 2^-12), float32 results the one that is
// good to a step (512 x 3584 -> 4608 22.6 -> 23.7 us with SiLU, 8192 x 64 -> 8192 105 -> 134). The quick division is good to two steps
// for such denominators (1 to 7). The code is short on purpose: the epilogue is unrolled over columns, and a launch of few tiles pays
// for every instruction it fetches.
template <bool QUICK> __device__ __forceinline__ float exponential(float v) { return QUICK ? __expf(v) : expf(v); }
template <bool QUICK>
__device__ __forceinline__ float times_sigmoid(float v, float z) {
  const float e = exponential<QUICK>(-fabsf(z));
  return v * __fdividef(z > 0.f ? 1.f : e, 1.f + e);
}
// The complement of the error function for x = |v| / sqrt 2, as exp(-v^2 / 2) t P(t), t = 1 / (1 + 0.375 x). P was fitted to
// exp(x^2) erfc(x) / t over 0 <= x <= 9.4 (least largest relative error, 1.1e-8); in float32 the whole is off by 2^-21 of itself at most,
// in the tail too, where 1 - erf has lost every digit. exp(-v^2 / 2) takes the rounding of v^2 along.
template <bool QUICK>
__device__ __forceinline__ float erfc_of(float v) {
  const float t = __fdividef(1.f, fmaf(0.375f * 0.70710678f, fabsf(v), 1.f)), sq = v * v;
  float p = 0.0616966151f;
  p = fmaf(p, t, -0.288075387f);
  p = fmaf(p, t, 0.433893770f);
  p = fmaf(p, t, -0.231076419f);
  p = fmaf(p, t, 0.274844110f);
  p = fmaf(p, t, 0.121038958f);
  p = fmaf(p, t, 0.205430418f);
  p = fmaf(p, t, 0.210633501f);
  p = fmaf(p, t, 0.211614415f);
  float e = exponential<QUICK>(-0.5f * sq);
  if (!QUICK) e = fmaf(e, -0.5f * fmaf(v, v, -sq), e);
  return sq < 400.f ? p * t * e : 0.f;
}
template <int ACT, bool QUICK>
__device__ __forceinline__ float activate(float v) {
  if (ACT == PM_ACT_RELU) return v < 0.f ? 0.f : v;  // NaN stays
  if (ACT == PM_ACT_SILU) return times_sigmoid<QUICK>(v, v);
  if (ACT == PM_ACT_GELU) {  // v/2 erfc(-v / sqrt 2)
    const float tail = erfc_of<QUICK>(v);
    return 0.5f * v * (v > 0.f ? 2.f - tail : tail);
  }
  if (ACT == PM_ACT_GELU_TANH)  // v/2 (1 + tanh u) = v sigma(2 u)
    return times_sigmoid<QUICK>(v, 1.5957691216057308f * (v + 0.044715f * v * v * v));
  return v;
}
template <bool QUICK, int N>
__device__ __forceinline__ void activate_all(float (&v)[N], int act) {
  auto all = [&](auto f) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = f(v[i]);
  };
  switch (act) {
    case PM_ACT_RELU: return all(activate<PM_ACT_RELU, QUICK>);
    case PM_ACT_SILU: return all(activate<PM_ACT_SILU, QUICK>);
    case PM_ACT_GELU: return all(activate<PM_ACT_GELU, QUICK>);
    case PM_ACT_GELU_TANH: return all(activate<PM_ACT_GELU_TANH, QUICK>);
  }
}
template <class OT>
__device__ __forceinline__ float activate_one(float v, int act) {
  float a[1] = {v};
  activate_all<sizeof(OT) == 2>(a, act);
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

// C neighbouring tokens from token m on of weight row n (one row per lane), `left` of them inside y: their residual; and bias,
// activation, residual, rounding, store. A chunk that lies inside y as a whole takes forms without tests: those made 17
// instructions of the 6 per output, which bounds products with a short K.
template <class OT, int C>
__device__ __forceinline__ void load_residual(const LinearTc& a, OT (&r)[C], int64_t m, int n, int left) {
  const OT* src = static_cast<const OT*>(a.res) + m * a.ldr + n;
  if (__all_sync(0xffffffffu, left >= C)) {
#pragma unroll
    for (int c = 0; c < C; ++c, src += a.ldr) r[c] = *src;
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c, src += a.ldr) r[c] = c < left ? *src : from_float<OT>(0.f);
  }
}
template <class OT, int C, bool ADD>
__device__ __forceinline__ void finish(const LinearTc& a, float (&o)[C], const OT (&r)[C], float bias, int64_t m, int n, int left) {
  const bool whole = __all_sync(0xffffffffu, left >= C);
#pragma unroll
  for (int c = 0; c < C; ++c) o[c] += bias;
  activate_all<sizeof(OT) == 2>(o, a.act);
  if (ADD) {
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] += to_float<OT>(r[c]);
  }
  OT* dst = static_cast<OT*>(a.y) + m * a.ldy + n;
  if (whole) {
#pragma unroll
    for (int c = 0; c < C; ++c, dst += a.ldy) *dst = from_float<OT>(o[c]);
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c, dst += a.ldy)
      if (c < left) *dst = from_float<OT>(o[c]);
  }
}

template <int CG, class OT>
__global__ void __launch_bounds__(kTcThreads, 1)
linear_tc_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                 const __grid_constant__ LinearTc a) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* stages = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  LinShared& sh = *reinterpret_cast<LinShared*>(stages + a.shared_bytes);
  constexpr bool kPromote = sizeof(OT) == 4;  // float32 outputs: accumulators of a.chunk steps, added up in registers
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = cluster_rank(), rank = CG == 2 ? cta & 1 : 0, part_rank = CG == 2 ? cta >> 1 : cta;
  const int per_tile = CG * a.split;
  const int first = blockIdx.x / per_tile, step = gridDim.x / per_tile;
  const int n_tiles = a.w_tiles * a.tok_tiles, n_stages = a.n_stages;
  const bool split = a.split > 1;
  const int k0 = split ? a.k_tiles * (int)part_rank / a.split : 0;  // k_tiles <= 2^25, split <= 8
  const int k1 = split ? a.k_tiles * ((int)part_rank + 1) / a.split : a.k_tiles;

  if (warp == 0) {
    if (lane == 0) prefetch_tensor_map(&map_w);
    if (lane < n_stages) {
      mbar_init(&sh.full[lane], 2);  // the two producers
      mbar_init(&sh.empty[lane], 1);
    }
    if (lane < 2) {
      mbar_init(&sh.acc_full[lane], 1);
      mbar_init(&sh.acc_empty[lane], CG * kEpiWarps);
    }
    if (lane == 0) sh.abort = 0;
    fence_barrier_init();
    __syncwarp();
  }
  if (warp == 3 && lane == 0) prefetch_tensor_map(&map_x);
  if (warp == 2) {
    if (CG == 2) tmem_alloc(&sh.tmem_base, a.tmem_cols);
    else tmem_alloc_single(&sh.tmem_base, a.tmem_cols);
  }
  tc_fence_before();
  if (CG == 2) {
    __syncthreads();
    cluster_sync_diverged();
  } else {
    // The weights' producer needs nothing but its own barriers: it goes ahead, by some 500 ns.
    if (warp == 0) asm volatile("barrier.cta.arrive 1, %0;" ::"n"(kTcThreads) : "memory");
    else asm volatile("barrier.cta.sync 1, %0;" ::"n"(kTcThreads) : "memory");
    if (split) cluster_arrive_diverged();  // waited for before the partial sums are sent
  }
  tc_fence_after();
  const uint32_t tmem_base = sh.tmem_base;    // not yet there for warp 0, which does not use it
  const uint32_t acc_cols = a.tmem_cols / 2;  // distance of the two accumulators
  if (CG == 2 || warp != 0) let_successor_start();  // not before the tensor memory is allocated
  wait_for_predecessor();

  const uint32_t full0 = smem_u32(&sh.full[0]), empty0 = smem_u32(&sh.empty[0]), stage0 = smem_u32(stages);
  const int lead = CG == 2 ? (int)(cta & ~1u) : 0;  // the pair's first CTA
  float bias = 0.f;
  if ((warp == 0 || warp == 3) && lane == 0) {
    // ---- producers: one thread for this CTA's 128 weight rows, one for its share of the token rows ------------------
    const bool tokens = warp == 3;
    const int rows = a.width / CG;
    const uint32_t bytes = CG * a.atoms * (tokens ? (uint32_t)rows * 128 : (uint32_t)kWBytes), atom_bytes = kWBytes + rows * 128;
    const CUtensorMap* map = tokens ? &map_x : &map_w;
    const uint32_t dst0 = stage0 + (tokens ? kWBytes : 0), full_of_pair = CG == 2 ? map_to_rank(full0, lead) : full0;
    int at = 0, steps = 0;
    uint32_t turn = 0;
    bool ok = true;
    for (int tile = first; tile < n_tiles && ok; tile += step) {
      int wt, tt;
      tile_at(a, tile, wt, tt);
      const int row = tokens ? tt * a.width + (int)rank * rows : wt * 128 * CG + (int)rank * 128;
      for (int kt = k0; kt < k1; ++kt, ++steps) {
        if (turn > 0 && !mbar_wait(empty0 + at * 8, (turn - 1) & 1, &sh.abort)) {
          ok = false;
          break;
        }
        if (rank == 0) mbar_arrive_expect_tx(full0 + at * 8, bytes);
        for (int i = 0; i < a.atoms; ++i)
          tma_load_2d_at<CG>(dst0 + at * a.stage_bytes + i * atom_bytes, map, full_of_pair + at * 8, (kt * a.atoms + i) * 64, row);
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
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // ---- MMA issuer ----------------------------------------------------------------------------------
    const uint32_t idesc = a.f16 ? umma_idesc_f16(128 * CG, a.width) : umma_idesc_bf16(128 * CG, a.width);
    const uint64_t desc0 = umma_desc_k_sw128(stage0);
    const uint32_t atom16 = (uint32_t)(kWBytes + a.width / CG * 128) >> 4;
    const uint16_t both = (uint16_t)(3u << lead);
    int at = 0, it = 0;
    uint32_t turn = 0;
    bool ok = true;
    for (int tile = first; tile < n_tiles && ok; tile += step)
      for (int kc = k0; kc < k1 && ok; kc += a.chunk, ++it) {
        const int acc = it & 1, end = min(k1, kc + a.chunk);
        if (it >= 2 && !mbar_wait(&sh.acc_empty[acc], ((it >> 1) - 1) & 1, &sh.abort)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + (uint32_t)acc * acc_cols;
        uint32_t more = 0;
        for (int kt = kc; kt < end; ++kt) {
          if (!mbar_wait(full0 + at * 8, turn & 1, &sh.abort)) {
            ok = false;
            break;
          }
          tc_fence_after();
          uint64_t da = desc0 + (uint32_t)(at * (a.stage_bytes >> 4));
          for (int i = 0; i < a.atoms; ++i, da += atom16) {
            const uint64_t db = da + (kWBytes >> 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // 16 k = 32 bytes inside the swizzled row
              umma_at<CG>(d, da + 2 * k, db + 2 * k, idesc, more);
              more = 1;
            }
          }
          umma_commit_at<CG>(empty0 + at * 8, both);
          if (++at == n_stages) {
            at = 0;
            ++turn;
          }
        }
        if (ok) umma_commit_at<CG>(smem_u32(&sh.acc_full[acc]), both);
      }
    if (!ok) sh.abort = 1;
  } else if (warp >= 4) {  // `bias` of this lane's row stays for the joining of partial sums
    // ---- epilogue: warp w drains accumulator rows 32w .. 32w+31, two warps of a quadrant share the columns ------
    const int w = warp & 3, half = (warp - 4) >> 2;
    const float nan = __int_as_float(0x7fffffff);
    const uint32_t acc_free = CG == 2 ? map_to_rank(smem_u32(&sh.acc_empty[0]), lead) : smem_u32(&sh.acc_empty[0]);
    int it = 0;
    bool ok = true;
    for (int tile = first; tile < n_tiles; tile += step) {
      int wt, tt;
      tile_at(a, tile, wt, tt);
      const int n = (wt * CG + (int)rank) * 128 + 32 * w + lane;
      const int m0 = tt * a.width, cols = min(a.width, a.M - m0);
      bias = n < a.N ? load_bias(a.bias, a.bias_type, n) : 0.f;
      // The residual of a chunk is asked for one chunk ahead, the first one's while the tile is still being multiplied (777 x
      // 5632 -> 2048 27.6 -> 26.9 us, 8192 x 64 -> 8192 137 -> 128 us).
      const bool add = a.res != nullptr && !split;
      OT ahead[16] = {};
      auto ask = [&](int c0) {
        if (add && c0 < cols) load_residual<OT, 16>(a, ahead, m0 + c0, n, n < a.N ? cols - c0 : 0);
      };
      ask(half * 16);
      auto give = [&](float (&o)[16], int c0) {
        if (!ok) {
#pragma unroll
          for (int c = 0; c < 16; ++c) o[c] = nan;
        }
        if (!split) {
          const int left = n < a.N ? cols - c0 : 0;
          if (!add) {
            finish<OT, 16, false>(a, o, ahead, bias, m0 + c0, n, left);
          } else {
            OT r[16];
#pragma unroll
            for (int c = 0; c < 16; ++c) r[c] = ahead[c];
            ask(c0 + 32);
            finish<OT, 16, true>(a, o, r, bias, m0 + c0, n, left);
          }
        } else {
          // four columns at a time to the CTA that finishes them, which keeps [source][its fours of columns][128 rows][4]
          const int per = a.part_cols;
          const uint32_t mine = stage0 + a.part_offset + 16u * (uint32_t)((int)part_rank * (per >> 2) * 128 + 32 * w + lane);
          int owner = c0 / per, at = c0 - owner * per;
          uint32_t dst = map_to_rank(mine, CG * owner + rank) + 512u * (uint32_t)at;
#pragma unroll
          for (int c = 0; c < 16; c += 4)
            if (c0 + c < cols) {
              asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "f"(o[c]), "f"(o[c + 1]), "f"(o[c + 2]),
                           "f"(o[c + 3]) : "memory");
              dst += 2048;
              at += 4;
              if (at == per) {
                at = 0;
                ++owner;
                if (owner < a.split) dst = map_to_rank(mine, CG * owner + rank);
              }
            }
        }
      };
      if (CG == 1 && split) cluster_wait_diverged();
      float sums[kPromote ? 4 : 1][16];
      for (int kc = k0; kc < k1; kc += a.chunk, ++it) {
        const int acc = it & 1;
        ok = ok && __all_sync(0xffffffffu, mbar_wait(&sh.acc_full[acc], (it >> 1) & 1, &sh.abort));
        tc_fence_after();
        const uint32_t taddr = tmem_base + (uint32_t)acc * acc_cols + ((uint32_t)(32 * w) << 16);
        if (kPromote) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // at most 128 columns
            const int c0 = half * 16 + 32 * i;
            if (c0 < cols) {
              uint32_t v[16];
              tmem_ld16(taddr + c0, v);
              tmem_ld_wait();
              float(&to)[16] = sums[kPromote ? i : 0];
#pragma unroll
              for (int c = 0; c < 16; ++c) to[c] = kc == k0 ? __uint_as_float(v[c]) : to[c] + __uint_as_float(v[c]);
            }
          }
        } else {
#pragma unroll 1
          for (int c0 = half * 16; c0 < cols; c0 += 32) {
            uint32_t v[16];
            tmem_ld16(taddr + c0, v);
            tmem_ld_wait();
            float o[16];
#pragma unroll
            for (int c = 0; c < 16; ++c) o[c] = __uint_as_float(v[c]);
            give(o, c0);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (CG == 2) mbar_arrive_cluster(acc_free + acc * 8);
          else mbar_arrive(acc_free + acc * 8);
        }
      }
      if (kPromote) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (half * 16 + 32 * i < cols) give(sums[kPromote ? i : 0], half * 16 + 32 * i);
      }
    }
    if (!ok && lane == 0) sh.abort = 1;
  }
  __syncwarp();
  if (split) {
    if (CG == 1 && warp < 4) cluster_wait_diverged();
    __syncthreads();
    cluster_sync_diverged();  // every CTA's partial sums have arrived where they are finished
    if (warp >= 4) {
      int wt, tt;
      tile_at(a, first, wt, tt);
      const int per = a.part_cols, c_first = (int)part_rank * per;
      const int m0 = tt * a.width, mine = min(per, min(a.width, a.M - m0) - c_first);
      const int row = (warp & 3) * 32 + lane, n = (wt * CG + (int)rank) * 128 + row;
      for (int c0 = ((warp - 4) >> 2) * 8; c0 < mine; c0 += 16) {
        float o[8] = {};
        const float4* part = reinterpret_cast<const float4*>(stages + a.part_offset) + (c0 >> 2) * 128 + row;
        for (int r = 0; r < a.split; ++r, part += (per >> 2) * 128) {
          const float4 u = part[0], v = c0 + 4 < per ? part[128] : make_float4(0.f, 0.f, 0.f, 0.f);
          o[0] += u.x, o[1] += u.y, o[2] += u.z, o[3] += u.w;
          o[4] += v.x, o[5] += v.y, o[6] += v.z, o[7] += v.w;
        }
        const int left = n < a.N ? mine - c0 : 0;
        OT r[8] = {};
        if (a.res != nullptr) load_residual<OT, 8>(a, r, m0 + c_first + c0, n, left);
        finish<OT, 8, true>(a, o, r, bias, m0 + c_first + c0, n, left);
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
  if (CG == 2) cluster_sync_diverged();
  tc_fence_after();
  if (warp == 2) {
    if (CG == 2) tmem_dealloc(tmem_base, a.tmem_cols);
    else tmem_dealloc_single(tmem_base, a.tmem_cols);
  }
}

// ---- rows that TMA cannot fetch -------------------------------------------------------------------------
// Tiles of BM tokens x BN weight rows in steps of 64 k, eight warps (mma.sync). Rows may start at any multiple of two bytes:
// the aligned 16-byte words that hold a step's values come into a ring of kRing steps (cp.async; each word holds at least one
// of the row's bytes, so it is mapped memory), and a thread shifts its eight values out of two of them into the tile: 15
// instructions instead of eight loads. What bounds it: the steps' two barriers and, with few tiles, the SMs that have none.
// 86 rows of 2611 -> 15580 take 90 us (180 with two-byte loads straight into the tile), 4000 of 2001 -> 2001 295 us = 109
// TFLOP/s, 125 of 1506 -> 111 20 us (36). Rows on 16-byte boundaries are three to eight times faster. Up to 16 tokens take
// linear_few_kernel instead.
constexpr int kPlainThreads = 256;

template <class T>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&x)[4], uint32_t w0, uint32_t w1);
template <>
__device__ __forceinline__ void mma_16x8x16<__nv_bfloat16>(float (&d)[4], const uint32_t (&x)[4], uint32_t w0, uint32_t w1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(w0), "r"(w1));
}
template <>
__device__ __forceinline__ void mma_16x8x16<__half>(float (&d)[4], const uint32_t (&x)[4], uint32_t w0, uint32_t w1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(w0), "r"(w1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix2(uint32_t& r0, uint32_t& r1, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];" : "=r"(r0), "=r"(r1) : "r"(addr));
}

// The eight values that start `shift` bytes into lo, of which `valid` are the row's, the others zero.
__device__ __forceinline__ uint4 eight_from(const uint4& lo, const uint4& hi, int shift, int valid) {
  uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  if (shift & 8) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (shift & 4) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  const int bits = (shift & 2) * 8;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], bits);
  if (valid < 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = 2 * i + 1 < valid ? w[i] : 2 * i < valid ? w[i] & 0xffffu : 0u;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void cp_async_16(uint32_t dst, uintptr_t src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

template <int BM, int BN>
struct PlainTile {
  static constexpr int kK = 64, kPitch = kK + 8, kVec = kK / 8;  // 16 bytes of padding: ldmatrix meets every bank once
  static constexpr int kRows = BM + BN, kWords = kVec + 1, kRing = BM >= 64 ? 3 : 4;
  static constexpr int kPer = (kRows + 31) / 32;  // rows per thread: eight threads take a row's eights
  static constexpr size_t bytes() { return (size_t)kRows * kPitch * 2 + (size_t)kRing * kRows * kWords * 16; }
};

template <class T, class OT, int BM, int BN>
__global__ void __launch_bounds__(kPlainThreads)
linear_plain_kernel(const __grid_constant__ LinearCall a) {
  using P = PlainTile<BM, BN>;
  constexpr int kWarpsM = BM >= 32 ? BM / 32 : 1, kWarpsN = 8 / kWarpsM;
  constexpr int kM = BM >= 32 ? 2 : 1, kN = BN / kWarpsN / 8;  // 16 x 8 pieces of a warp
  static_assert(BN % (kWarpsN * 8) == 0, "whole pieces");
  extern __shared__ __align__(16) unsigned char smem_raw[];
  uint16_t* tile = reinterpret_cast<uint16_t*>(smem_raw);  // token rows, then weight rows
  unsigned char* ring = smem_raw + (size_t)P::kRows * P::kPitch * 2;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int w_tiles = (a.N + BN - 1) / BN;
  const int m0 = blockIdx.x / w_tiles * BM, n0 = blockIdx.x % w_tiles * BN;
  const int wm = warp % kWarpsM * 16 * kM, wn = warp / kWarpsM * 8 * kN;
  const int steps = (a.K + P::kK - 1) / P::kK;
  wait_for_predecessor();
  // Eight neighbouring threads take the first eight words of a row, rows tid / 8, + 32, ...; the ninth word of row r is thread r's.
  const int v = tid & 7, r0 = tid >> 3;
  auto row_at = [&](int r) -> uintptr_t {  // 0 outside the matrices
    const bool tok = r < BM;
    const int row = tok ? m0 + r : n0 + r - BM;
    if (r >= P::kRows || row >= (tok ? a.M : a.N)) return 0;
    return (uintptr_t)(tok ? a.x : a.w) + (uintptr_t)((int64_t)row * (tok ? a.ldx : a.ldw) * 2);
  };
  uintptr_t word[P::kPer];
  uint32_t shifts = 0, rows_in = 0;  // of each row: half the byte offset in its first word; whether it exists
#pragma unroll
  for (int i = 0; i < P::kPer; ++i) {
    const uintptr_t row = row_at(r0 + 32 * i);
    word[i] = (row & ~(uintptr_t)15) + 16u * v;
    shifts |= (uint32_t)(row & 14) >> 1 << (4 * i);
    rows_in |= (uint32_t)(row != 0) << i;
  }
  const uintptr_t ninth_row = row_at(tid), ninth = (ninth_row & ~(uintptr_t)15) + 128u;
  const uint32_t ninth_end = ninth_row != 0 ? 2u * (uint32_t)a.K + (uint32_t)(ninth_row & 15) : 0u;  // words start before it
  const uint32_t ring0 = smem_u32(ring);
  auto fetch = [&](int step) {
    if (step < steps) {
      const uint32_t dst = ring0 + (uint32_t)(step % P::kRing) * (P::kRows * P::kWords * 16), off = (uint32_t)step * (P::kK * 2);
#pragma unroll
      for (int i = 0; i < P::kPer; ++i)
        if ((rows_in >> i & 1) && off + 16u * v < 2u * (uint32_t)a.K + (shifts >> (4 * i) & 7) * 2u)
          cp_async_16(dst + 16u * (uint32_t)((r0 + 32 * i) * P::kWords + v), word[i] + off);
      if (off + 128u < ninth_end) cp_async_16(dst + 16u * (uint32_t)(tid * P::kWords + P::kVec), ninth + off);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  constexpr bool kPromote = sizeof(OT) == 4;  // as in the tensor-memory kernel
  float acc[kM][kN][4] = {}, sum[kPromote ? kM : 1][kPromote ? kN : 1][4] = {};
  const uint32_t base = smem_u32(tile);
  // ldmatrix: lanes 0-15 give the rows of the first 8 k, lanes 16-31 of the next
  const uint32_t x_at = base + 2u * (uint32_t)((wm + (lane & 15)) * P::kPitch + (lane >> 4) * 8);
  const uint32_t w_at = base + 2u * (uint32_t)((BM + wn + (lane & 7)) * P::kPitch + (lane >> 3 & 1) * 8);
#pragma unroll
  for (int i = 0; i < P::kRing - 1; ++i) fetch(i);
  for (int step = 0; step < steps; ++step) {
    asm volatile("cp.async.wait_group %0;" ::"n"(P::kRing - 2) : "memory");
    __syncthreads();  // the step's words are there, and the tile has been read
    const uint4* words = reinterpret_cast<const uint4*>(ring + (size_t)(step % P::kRing) * (P::kRows * P::kWords * 16));
    const int valid = min(8, a.K - step * P::kK - v * 8);
#pragma unroll
    for (int i = 0; i < P::kPer; ++i) {
      const int r = r0 + 32 * i;
      if (P::kRows % 32 == 0 || r < P::kRows) {
        uint4 e = make_uint4(0, 0, 0, 0);
        if ((rows_in >> i & 1) && valid > 0)
          e = eight_from(words[r * P::kWords + v], words[r * P::kWords + v + 1], (int)(shifts >> (4 * i) & 7) * 2, valid);
        *reinterpret_cast<uint4*>(tile + r * P::kPitch + v * 8) = e;
      }
    }
    __syncthreads();
    fetch(step + P::kRing - 1);  // over the words of the step before this one
#pragma unroll
    for (int kk = 0; kk < P::kK; kk += 16) {
      uint32_t xf[kM][4];
#pragma unroll
      for (int i = 0; i < kM; ++i) ldmatrix4(xf[i], x_at + 2u * (uint32_t)(16 * i * P::kPitch + kk));
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        uint32_t w0, w1;
        ldmatrix2(w0, w1, w_at + 2u * (uint32_t)(8 * j * P::kPitch + kk));
#pragma unroll
        for (int i = 0; i < kM; ++i) mma_16x8x16<T>(acc[i][j], xf[i], w0, w1);
      }
    }
    if constexpr (kPromote) {
      if ((step + 1) % (kPromoteK / P::kK) == 0 || step + 1 == steps) {
#pragma unroll
        for (int i = 0; i < kM; ++i)
#pragma unroll
          for (int j = 0; j < kN; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              sum[i][j][c] += acc[i][j][c];
              acc[i][j][c] = 0.f;
            }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kN; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int n = n0 + wn + 8 * j + (lane & 3) * 2 + e;
      if (n >= a.N) continue;
      const float b = load_bias(a.bias, a.bias_type, n);
#pragma unroll
      for (int i = 0; i < kM; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int m = m0 + wm + 16 * i + (lane >> 2) + 8 * h;
          if (m >= a.M) continue;
          float v = activate_one<OT>((kPromote ? sum[kPromote ? i : 0][kPromote ? j : 0] : acc[i][j])[2 * h + e] + b, a.act);
          if (a.res != nullptr) v += to_float<OT>(static_cast<const OT*>(a.res)[(int64_t)m * a.ldr + n]);
          static_cast<OT*>(a.y)[(int64_t)m * a.ldy + n] = from_float<OT>(v);
        }
    }
}

template <class T, class OT, int BM, int BN>
cudaError_t launch_plain_tiles(const LinearCall& a, cudaStream_t s) {
  const long long tiles = (long long)((a.N + BN - 1) / BN) * ((a.M + BM - 1) / BM);
  if (tiles > 0x7fffffffll) return cudaErrorInvalidValue;
  auto kern = linear_plain_kernel<T, OT, BM, BN>;
  static SmemOptIn once;
  cudaError_t e = opt_in_smem(once, kern);
  if (e != cudaSuccess) return e;
  return launch_behind(kern, (unsigned)tiles, kPlainThreads, PlainTile<BM, BN>::bytes(), s, a);
}

// ---- few tokens -----------------------------------------------------------------------------------------
// 16 RT weight rows per CTA, its warps on one step of 64 k after the other in turn (mma.sync; weight rows are its M operand, MT
// tiles of eight tokens its N operand). A lane loads 16 bytes of a row, eight neighbouring k, and gives them to two MMAs as
// the k it has there: both operands come in the same order, so that neither goes through shared memory. Weights pass the L1
// by, two steps of a warp are under way at a time. The warps' sums are added in order through shared memory.
// Rows off 16-byte boundaries (ALIGNED = false): a lane's eight values are shifted out of two aligned words; their registers leave
// room for one step per warp, more warps make up for it. 1 x 3001 -> 4001 8.6 us, 7 x 1628 -> 80637 60 us = 4.4 TB/s, where
// tiles through shared memory took 28 and 90.
// Bound by the weights' way from HBM, once a launch has started: 8 x 3584 -> 4608 (33 MB) takes 6.2 us in a chain of products, of
// which 5.0 are the bytes at the measured copy rate. The tensor-core kernel needs 3 us more for its setup, the joining of partial sums and the
// longer way of the operands.

__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// Eight values from `at` on of which `left` lie inside the row; the others are zero.
template <class T>
__device__ __forceinline__ uint4 load_end(const T* row, int left) {
  if (left >= 8) return *reinterpret_cast<const uint4*>(row);
  uint4 v = make_uint4(0, 0, 0, 0);
  const unsigned short* src = reinterpret_cast<const unsigned short*>(row);
  if (left > 0) v.x = src[0];
  if (left > 1) v.x |= (uint32_t)src[1] << 16;
  if (left > 2) v.y = src[2];
  if (left > 3) v.y |= (uint32_t)src[3] << 16;
  if (left > 4) v.z = src[4];
  if (left > 5) v.z |= (uint32_t)src[5] << 16;
  if (left > 6) v.w = src[6];
  return v;
}

template <class T, class OT, int RT, int MT, int WARPS, bool ALIGNED = true>
__global__ void __launch_bounds__(WARPS * 32, (ALIGNED ? 16 : 24) / WARPS) linear_few_kernel(const __grid_constant__ LinearCall a) {
  __shared__ float part[WARPS][MT * 8][16 * RT + 4];  // the lanes of a store meet different banks
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16 * RT, steps = a.K / 64;
  if (ALIGNED && threadIdx.x < 16 * RT && n0 + (int)threadIdx.x < a.N && a.ahead > 0)
    prefetch_to_l2(static_cast<const T*>(a.w) + (int64_t)(n0 + (int)threadIdx.x) * a.ldw, (uint32_t)a.ahead);
  let_successor_start();
  wait_for_predecessor();
  const T *w[2 * RT], *x[MT];  // rows beyond the last are the last again, their sums are not used
#pragma unroll
  for (int i = 0; i < 2 * RT; ++i) w[i] = static_cast<const T*>(a.w) + (int64_t)min(n0 + g + 8 * i, a.N - 1) * a.ldw + 8 * t;
#pragma unroll
  for (int i = 0; i < MT; ++i) x[i] = static_cast<const T*>(a.x) + (int64_t)min(g + 8 * i, a.M - 1) * a.ldx + 8 * t;

  struct Step {
    uint4 w[2 * RT][2], x[MT][2];
  };
  // Rows that start anywhere: the two 16-byte words that hold a lane's eight values, if they hold any of the row's `left` values
  // from the step's start on (else they may lie in memory that is not there), and the values shifted out of them.
  auto load_shifted = [&](Step& s, int step, int left) {
    auto two = [&](const T* row, uint4& v) {
      const uintptr_t at = (uintptr_t)(row + step * 64), word = at & ~(uintptr_t)15;
      const int shift = (int)(at & 15), valid = left - 8 * t;
      const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int in = valid - 32 * h;
        const uint4* p = reinterpret_cast<const uint4*>(word + 64 * h);
        const uint4 lo = in > 0 ? p[0] : none, hi = 2 * in + shift > 16 && shift > 0 ? p[1] : none;
        (&v)[h] = eight_from(lo, hi, shift, in < 8 ? in : 8);
      }
    };
#pragma unroll
    for (int i = 0; i < 2 * RT; ++i) two(w[i], s.w[i][0]);
#pragma unroll
    for (int i = 0; i < MT; ++i) two(x[i], s.x[i][0]);
  };
  auto load = [&](Step& s, int step) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 2 * RT; ++i) s.w[i][h] = load_once(w[i] + step * 64 + 32 * h);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < MT; ++i) s.x[i][h] = *reinterpret_cast<const uint4*>(x[i] + step * 64 + 32 * h);
    }
  };
  float acc[RT][MT][4] = {}, sum[RT][MT][4] = {};
  auto multiply = [&](const Step& s) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const uint4 lo = s.w[2 * r][h], hi = s.w[2 * r + 1][h];
        const uint32_t first[4] = {lo.x, hi.x, lo.y, hi.y}, second[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          mma_16x8x16<T>(acc[r][i], first, s.x[i][h].x, s.x[i][h].y);
          mma_16x8x16<T>(acc[r][i], second, s.x[i][h].z, s.x[i][h].w);
        }
      }
  };
  auto promote = [&]() {  // the tensor cores cut their running sums off
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          sum[r][i][c] += acc[r][i][c];
          acc[r][i][c] = 0.f;
        }
  };
  if constexpr (!ALIGNED) {
    Step one;  // the other blocks' warps have theirs under way meanwhile
    for (int s = warp, n = 1; s < steps; s += WARPS, ++n) {
      load_shifted(one, s, 64);
      multiply(one);
      if (n % (kPromoteK / 64) == 0) promote();
    }
    if (steps * 64 < a.K && warp == steps % WARPS) {
      load_shifted(one, steps, a.K - steps * 64);
      multiply(one);
    }
  } else {
    Step even, odd;
    int s = warp;
    if (s < steps) load(even, s);
    for (int n = 1; s < steps; s += 2 * WARPS, ++n) {
      if (s + WARPS < steps) load(odd, s + WARPS);
      multiply(even);
      if (s + 2 * WARPS < steps) load(even, s + 2 * WARPS);
      if (s + WARPS < steps) multiply(odd);
      if (n % (kPromoteK / 128) == 0) promote();
    }
    if (steps * 64 < a.K && warp == steps % WARPS) {  // the rest of the rows, less than a step
      Step end;
      const int left = a.K - steps * 64 - 8 * t;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < 2 * RT; ++i) end.w[i][h] = load_end(w[i] + steps * 64 + 32 * h, left - 32 * h);
#pragma unroll
        for (int i = 0; i < MT; ++i) end.x[i][h] = load_end(x[i] + steps * 64 + 32 * h, left - 32 * h);
      }
      multiply(end);
    }
  }
  promote();
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) part[warp][8 * i + 2 * t + (c & 1)][16 * r + g + 8 * (c >> 1)] = sum[r][i][c];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * RT * 8 * MT; i += WARPS * 32) {
    const int row = i % (16 * RT), m = i / (16 * RT), n = n0 + row;
    if (m >= a.M || n >= a.N) continue;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) v += part[k][m][row];
    v = activate_one<OT>(v + load_bias(a.bias, a.bias_type, n), a.act);
    if (a.res != nullptr) v += to_float<OT>(static_cast<const OT*>(a.res)[(int64_t)m * a.ldr + n]);
    static_cast<OT*>(a.y)[(int64_t)m * a.ldy + n] = from_float<OT>(v);
  }
}

// What an SM's blocks ask L2 for before they wait for the kernel in front of them, where all blocks are resident at once: the fetch
// overlaps that kernel's end. Cold weights in a chain of products, 0 / 64 / 128 / 192 KB: 8 x 3584 -> 4608 7.39 / 6.56 / 6.22 / 6.56 us, 1 x
// 4096 -> 4096 7.6 / 6.7 / 6.3 / 6.2, 1 x 2048 -> 512 3.1 / 2.5 / 2.5 / 2.5, 1 x 14336 -> 4096 20.4 / 19.2 / 18.4 / 17.4. With more blocks than fit
// it takes bandwidth from the rows that are being read (8 x 7168 -> 18432 42.0 -> 44.2). (The tensor-core kernel gained nothing.)
constexpr int kAheadBytes = 131072;

// Which of them a product of M tokens takes, none (false) for the tensor-core kernel. All blocks should be resident at once, 16
// warps per SM; 32 weight rows a block halve the fetches of x, but only for one tile of tokens have they the registers.
// Cold weights, the others of {16, 32 rows} x {4, 8, 16 warps} and the tensor-core kernel in turn: 8 x 2048 -> 2048 16x16 3.7 us, 16x8
// 4.7, tensor cores 6.5; 8 x 3584 -> 4608 32x16 7.4, 16x8 7.6, 10.3; 8 x 2048 -> 8192 32x8 7.4, 16x4 7.5, 10.2; 8 x 1024 -> 30000 32x8
// 12.3, 16x4 12.8, 14.0; 8 x 4096 -> 128000 32x8 170, tensor cores 166. 16 x 3584 -> 4608 16x8 8.1, 32x16 9.7, 10.4; 16 x 2048 -> 6000
// 16x4 7.3, 16x8 8.7, 9.5; 16 x 7168 -> 18432 16x4 44.6, tensor cores 43.3. 32 tokens (four tiles): 2048 -> 512 6.0 against 5.3.
struct FewShape {
  int rows, warps;
};
bool few_shape(int M, int N, int sms, FewShape& f) {
  const int narrow = (N + 15) / 16, wide = (N + 31) / 32;
  if (M > 16) return false;
  f = {16, 16};
  if (narrow <= sms) return true;
  if (M <= 8) {
    f = {32, wide <= sms ? 16 : 8};
    return wide <= 8 * sms;
  }
  f = {16, narrow <= 2 * sms ? 8 : 4};
  return narrow <= 4 * sms;
}

template <class T, class OT>
cudaError_t launch_few_for(const LinearCall& a, FewShape f, cudaStream_t s) {
  const unsigned blocks = (unsigned)((a.N + f.rows - 1) / f.rows), threads = (unsigned)f.warps * 32;
  if (a.M <= 8) {
    if (f.rows == 16) return launch_behind(linear_few_kernel<T, OT, 1, 1, 16>, blocks, threads, 0, s, a);
    if (f.warps == 16) return launch_behind(linear_few_kernel<T, OT, 2, 1, 16>, blocks, threads, 0, s, a);
    return launch_behind(linear_few_kernel<T, OT, 2, 1, 8>, blocks, threads, 0, s, a);
  }
  if (f.warps == 16) return launch_behind(linear_few_kernel<T, OT, 1, 2, 16>, blocks, threads, 0, s, a);
  if (f.warps == 8) return launch_behind(linear_few_kernel<T, OT, 1, 2, 8>, blocks, threads, 0, s, a);
  return launch_behind(linear_few_kernel<T, OT, 1, 2, 4>, blocks, threads, 0, s, a);
}
template <class T, class OT, int MT>
cudaError_t launch_few_shifted_for(const LinearCall& a, int sms, cudaStream_t s) {
  const int blocks = (a.N + 15) / 16;
  if (blocks <= sms) return launch_behind(linear_few_kernel<T, OT, 1, MT, 16, false>, blocks, 512, 0, s, a);
  if (blocks <= 3 * sms) return launch_behind(linear_few_kernel<T, OT, 1, MT, 8, false>, blocks, 256, 0, s, a);
  return launch_behind(linear_few_kernel<T, OT, 1, MT, 4, false>, blocks, 128, 0, s, a);
}
template <class T, class OT>
cudaError_t launch_few_shifted(const LinearCall& a, int sms, cudaStream_t s) {
  return a.M <= 8 ? launch_few_shifted_for<T, OT, 1>(a, sms, s) : launch_few_shifted_for<T, OT, 2>(a, sms, s);
}
template <class T>
cudaError_t launch_few(const LinearCall& a, FewShape f, cudaStream_t s) {
  return a.out_type == PM_F32 ? launch_few_for<T, float>(a, f, s) : launch_few_for<T, T>(a, f, s);
}

template <class T, class OT>
cudaError_t launch_plain_for(const LinearCall& a, int sms, cudaStream_t s) {
  // narrow weight tiles where wide ones would leave SMs without any
  if ((long long)((a.N + 127) / 128) * ((a.M + 63) / 64) < sms) return launch_plain_tiles<T, OT, 32, 64>(a, s);
  return launch_plain_tiles<T, OT, 64, 128>(a, s);
}

template <class T>
cudaError_t launch_plain(const LinearCall& a, int sms, cudaStream_t s) {
  if (a.M <= 16) return a.out_type == PM_F32 ? launch_few_shifted<T, float>(a, sms, s) : launch_few_shifted<T, T>(a, sms, s);
  return a.out_type == PM_F32 ? launch_plain_for<T, float>(a, sms, s) : launch_plain_for<T, T>(a, sms, s);
}

// ---- launch plan ------------------------------------------------------------------------------------------
struct LinearShape {
  int cg = 1, split = 1, tok_tiles = 1, width = 16, atoms = 1;
};

// Narrow steps take two atoms of 64 k: waits and commits cost 75 ns per step.
int atoms_for(int cg, int width) { return kWBytes + width / cg * 128 <= 24 * 1024 ? 2 : 1; }

// Estimated ns of a shape. The constants were fitted to 2966 measured times (176 sizes of 24 to 2048 tokens, K from 64 to 8192, N
// from 256 to 100003, cold weights; 8 % off in the middle): the shape with the least estimate is 0.9 % slower than the best of a
// size on average, 11 % at worst. An atom's MMAs take 0.74 ns per token column, 170 at least (the weight rows' way from
// shared memory), a step's waits and commits 173 more; an SM takes in 124 bytes per ns; a tile's epilogue 8.7 ns per column, which
// counts where it is longer than the next tile's k steps and after the last one. Joining partial sums costs 1.1 us and 10 ns per
// column. cap: clusters of cg * split CTAs that the GPU holds at once.
double shape_cost(const LinearShape& c, int M, int N, int K, int cap) {
  const long long tiles = (long long)((N + 128 * c.cg - 1) / (128 * c.cg)) * c.tok_tiles;
  const double rounds = (double)((tiles + cap - 1) / cap), bytes = kWBytes + c.width / c.cg * 128;
  const double atom = std::max(std::max(170.0, 0.74 * c.width) + 173.0 / c.atoms, bytes / 124.0);
  const int steps = (K + 64 * c.atoms - 1) / (64 * c.atoms);
  const double tile = std::max((steps + c.split - 1) / c.split * c.atoms * atom, rounds > 1 ? 8.7 * c.width : 0.0);
  const double fixed = 2175.0 + 10.85 * c.width + 525.0 * rounds + (c.cg == 2 ? 225.0 : 0.0) +
                       (c.split > 1 ? 1120.0 + 10.1 * c.width : 0.0);
  return std::max(rounds * tile, ((double)N * K + (double)M * K) * 2 / 6500.0) + fixed;
}

constexpr int kMaxCluster = 8;

// Clusters of each size that the current device holds, one CTA per SM.
cudaError_t cluster_capacity(int dev, int (&cap)[kMaxCluster + 1]);

struct PlanKey {
  int M, N, K, promote, dev;
  bool operator==(const PlanKey& o) const { return M == o.M && N == o.N && K == o.K && promote == o.promote && dev == o.dev; }
};

LinearShape choose_shape(int M, int N, int K, bool promote, const int (&cap)[kMaxCluster + 1]) {
  LinearShape best;
  double cost = 0;
  const int most = promote ? 128 : 256;  // float32 outputs keep their sums in registers
  for (int cg = 1; cg <= 2; ++cg) {
    const int grain = 16 * cg;
    for (int w = grain; w <= most; w += grain) {
      LinearShape c;
      c.cg = cg;
      c.tok_tiles = (M + w - 1) / w;
      c.width = ((M + c.tok_tiles - 1) / c.tok_tiles + grain - 1) / grain * grain;  // tiles of equal width
      c.atoms = atoms_for(cg, c.width);
      const int steps = (K + 64 * c.atoms - 1) / (64 * c.atoms);
      for (c.split = 1; c.split * cg <= kMaxCluster && c.split <= steps; ++c.split) {
        // shared tiles: one round of clusters, and partial sums that leave the ring enough room
        if (c.split > 1 && (c.width > 128 || (long long)((N + 128 * cg - 1) / (128 * cg)) * c.tok_tiles > cap[cg * c.split])) break;
        const double x = shape_cost(c, M, N, K, cap[cg * c.split]);
        if (cost == 0 || x < cost) {
          cost = x;
          best = c;
        }
      }
      if (c.tok_tiles == 1) break;
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

cudaError_t cluster_capacity(int dev, int (&cap)[kMaxCluster + 1]) {
  static std::atomic<int> known[64][kMaxCluster + 1];
  auto kern = linear_tc_kernel<1, __nv_bfloat16>;
  for (int c = 1; c <= kMaxCluster; ++c) {
    const bool keep = dev >= 0 && dev < 64;
    int n = keep ? known[dev][c].load(std::memory_order_relaxed) : 0;
    if (n == 0) {
      cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
      if (e != cudaSuccess) return e;
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = 1024 * c;
      cfg.blockDim = kTcThreads;
      cfg.dynamicSmemBytes = kSmemMost;
      cudaLaunchAttribute attr{};
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim = {(unsigned)c, 1, 1};
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      if ((e = cudaOccupancyMaxActiveClusters(&n, kern, &cfg)) != cudaSuccess) return e;
      if (n <= 0) return cudaErrorNotSupported;
      if (keep) known[dev][c].store(n, std::memory_order_relaxed);
    }
    cap[c] = n;
  }
  return cudaSuccess;
}

bool tma_rows(const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && ld < ((int64_t)1 << 38); }

}  // namespace

int launch_linear(const LinearCall& a, cudaStream_t s) {
  int dev = 0, cap[kMaxCluster + 1];
  PM_CUDA(cudaGetDevice(&dev));
  PM_CUDA(cluster_capacity(dev, cap));
  if (!tma_rows(a.x, a.ldx) || !tma_rows(a.w, a.ldw)) {
    PM_CUDA(a.type == PM_BF16 ? launch_plain<__nv_bfloat16>(a, cap[1], s) : launch_plain<__half>(a, cap[1], s));
    return PM_OK;
  }
  FewShape few;
  if (few_shape(a.M, a.N, cap[1], few)) {
    LinearCall c = a;
    const int blocks = (a.N + few.rows - 1) / few.rows, per_sm = 16 / few.warps;
    if (blocks <= per_sm * cap[1]) c.ahead = std::min(std::min(a.K, kAheadBytes) / 8 * 16, kAheadBytes / (per_sm * few.rows) & ~15);
    PM_CUDA(a.type == PM_BF16 ? launch_few<__nv_bfloat16>(c, few, s) : launch_few<__half>(c, few, s));
    return PM_OK;
  }
  // The shape follows from the sizes alone; a thread remembers the last few.
  const bool promote = a.out_type == PM_F32;
  const PlanKey key{a.M, a.N, a.K, promote, dev};
  struct Plan {
    PlanKey key;
    LinearShape shape;
  };
  static thread_local Plan plans[16] = {};
  Plan& plan = plans[((unsigned)a.M * 31u + (unsigned)a.N * 7u + (unsigned)a.K) % 16u];
  if (!(plan.key == key)) plan = Plan{key, choose_shape(a.M, a.N, a.K, promote, cap)};
  const LinearShape& c = plan.shape;
  LinearTc t{};
  t.y = a.y; t.res = a.res; t.bias = a.bias;
  t.ldy = a.ldy; t.ldr = a.ldr;
  t.M = a.M; t.N = a.N; t.act = a.act; t.bias_type = a.bias_type; t.f16 = a.type == PM_F16;
  t.width = c.width; t.tok_tiles = c.tok_tiles; t.w_tiles = (a.N + 128 * c.cg - 1) / (128 * c.cg);
  t.atoms = c.atoms; t.k_tiles = (a.K + 64 * c.atoms - 1) / (64 * c.atoms);
  t.chunk = promote ? kPromoteK / 64 / c.atoms : t.k_tiles;
  t.split = c.split; t.err = a.err;
  t.stage_bytes = c.atoms * (kWBytes + c.width / c.cg * 128);
  t.part_cols = ((c.width + c.split - 1) / c.split + 3) & ~3;
  const int part_bytes = c.split > 1 ? t.part_cols * c.split * 512 : 0;
  const int room = kSmemMost - 1024 - (int)sizeof(LinShared) - part_bytes, steps = (t.k_tiles + c.split - 1) / c.split;
  const long long n_tiles = (long long)t.w_tiles * t.tok_tiles, units = cap[c.cg * c.split];
  const long long tiles_each = c.split > 1 ? 1 : (n_tiles + units - 1) / units;
  t.n_stages = (int)std::min<long long>(std::min(kMaxStages, room / t.stage_bytes), steps * tiles_each);
  t.part_offset = t.stage_bytes * t.n_stages;
  t.shared_bytes = t.part_offset + part_bytes;
  t.tmem_cols = 64;  // two accumulators, each at a multiple of 32 columns; the allocation is a power of two
  while (t.tmem_cols < 2 * c.width) t.tmem_cols *= 2;
  CUtensorMap map_w, map_x;
  int rc = tc_encode_matrix(&map_w, a.w, a.K, a.N, a.ldw, 128);
  if (rc != PM_OK) return rc;
  rc = tc_encode_matrix(&map_x, a.x, a.K, a.M, a.ldx, c.width / c.cg);
  if (rc != PM_OK) return rc;
  // Beside the grouped FFN's kernel, which takes all tensor memory after it has let its successor in, no block of this one
  // may start (each would wait for the other): 64 KB do not fit there. Pairs allocate together, so only one per SM.
  const size_t smem = std::max<size_t>(1024 + t.shared_bytes + sizeof(LinShared), (c.cg == 2 ? 120 : 64) * 1024);
  const int cluster = c.cg * c.split;
  if (n_tiles * cluster > 0x7fffffffll) return fail(PM_ERR_INVALID, "linear: too many tiles");
  const long long grid = (c.split > 1 ? n_tiles : std::min(n_tiles, units)) * cluster;
  PM_CUDA(c.cg == 2 ? launch_tc_for<2>(a.out_type, map_w, map_x, t, (int)grid, cluster, smem, s)
                    : launch_tc_for<1>(a.out_type, map_w, map_x, t, (int)grid, cluster, smem, s));
  return PM_OK;
}

}  // namespace pm
