// One warp chooses the experts of one token from its router logits: softmax or sigmoid scores, a correction bias that
// takes part in the choice only, groups of neighbouring experts of which the best few stay, the k best of what is left,
// their scores as weights, renormalised and scaled. Used by the stateless router (route.cu) and by the
// layer call's router (gate_topk.cu) for layers with a router rule.
//
//   score   s_e = softmax(l)_e  or  1 / (1 + exp(-l_e))
//   choice  c_e = s_e + b_e; an expert whose logit or choice is -inf cannot be chosen
//   group   max of its choices, or the sum of its two largest (a missing second counts as nothing);
//           the topk_group best groups stay, ties to the lower group
//   ids     the k largest choices among them, descending, ties to the lower id; -1 where there are fewer
//   weight  s_id, divided by (sum of the k + 1e-20) if asked for, times the scale; 0 for id -1
// A row that holds a NaN (softmax: or +inf) has no scores: its ids are -1 and its weights NaN.
//
// Which expert is chosen must not depend on float32 rounding. Without a bias experts are ranked by their logits (scores are
// monotonic in them). Choices with a bias and sums of two are ranked in float32, and a row in which two neighbours of a
// ranking lie closer than the error bound of those numbers is ranked again in 64 bits (a few rows in a thousand).
#pragma once
#include <math_constants.h>

#include "pm_common.cuh"

namespace pm {

// Numbers as integers in the same order; the key of -inf, kNone, stands for what cannot be chosen.
constexpr uint32_t kNone = 0x007fffffu;
__device__ __forceinline__ uint32_t order_key(float v) {  // not for -0
  const uint32_t b = __float_as_uint(v);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// Lanes that share a group: the same power of two for each of G <= 32 groups.
__device__ __forceinline__ int lanes_per_group(int G) { return 1 << (31 - __clz(32 / G)); }

// ---- the same ranking in 64 bits; c[E] is shared memory of the warp ------------------------------------------
// Logits in c become choices.
static __device__ __noinline__ void exact_choices(double* c, const RouteRule* rule, int lane) {
  const int E = rule->E;
  double mx = -CUDART_INF, sum = 0.0;
  __syncwarp();
  if (!rule->sigmoid) {
    for (int e = lane; e < E; e += 32) mx = fmax(mx, c[e]);
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) mx = fmax(mx, __shfl_xor_sync(0xffffffffu, mx, m));
    for (int e = lane; e < E; e += 32) sum += exp(c[e] - mx);
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  }
  for (int e = lane; e < E; e += 32) {
    const double l = c[e];
    const double s = rule->sigmoid ? 1.0 / (1.0 + exp(-l)) : exp(l - mx) / sum;
    const double v = s + (rule->bias != nullptr ? (double)rule->bias[e] : 0.0);
    c[e] = l == -CUDART_INF || v != v ? -CUDART_INF : v;
  }
  __syncwarp();
}

// The groups that stay, as bits.
static __device__ __noinline__ uint32_t exact_groups(const double* c, const RouteRule* rule, int lane) {
  const int per = rule->E / rule->n_group;
  double value = -CUDART_INF;  // lane g: group g
  if (lane < rule->n_group) {
    double a = -CUDART_INF, b = -CUDART_INF;
    for (int i = 0; i < per; ++i) {
      const double v = c[lane * per + i];
      if (v > a) {
        b = a;
        a = v;
      } else if (v > b) {
        b = v;
      }
    }
    value = rule->group_top2 && b > -CUDART_INF ? a + b : a;
  }
  int before = 0;  // groups that rank before this one
  for (int g = 0; g < rule->n_group; ++g) {
    const double o = __shfl_sync(0xffffffffu, value, g);
    before += o > value || (o == value && g < lane);
  }
  return __ballot_sync(0xffffffffu, lane < rule->n_group && before < rule->topk_group && value > -CUDART_INF);
}

// Lane j < k returns the j-th of the experts in the groups `kept`, -1 if there are fewer. Uses c up.
static __device__ __noinline__ int exact_rank(double* c, const RouteRule* rule, uint32_t kept, int lane) {
  const int E = rule->E, per = E / rule->n_group;
  for (int e = lane; e < E; e += 32)
    if (!((kept >> (e / per)) & 1u)) c[e] = -CUDART_INF;
  int mine = -1;
  for (int j = 0; j < rule->k; ++j) {
    double best = -CUDART_INF;
    int at = E;
    for (int e = lane; e < E; e += 32)
      if (c[e] > best) {
        best = c[e];
        at = e;
      }
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) {
      const double ob = __shfl_xor_sync(0xffffffffu, best, m);
      const int oa = __shfl_xor_sync(0xffffffffu, at, m);
      if (ob > best || (ob == best && oa < at)) {
        best = ob;
        at = oa;
      }
    }
    if (at >= E) break;  // the same in every lane: nothing is left
    if (lane == j) mine = at;
    if ((at & 31) == lane) c[at] = -CUDART_INF;
  }
  return mine;
}

// How the warp chooses. Lane i holds npl neighbouring experts, so lower lanes hold lower ids. The k-th largest of the lanes'
// maxima is a floor that k experts reach, and usually few more do: those are laid out one per lane, in the order of
// their ids, and each counts how many rank before it. Where more than 32 experts reach the floor (many equal logits,
// large k) there are k rounds of arg-max over all experts instead.
struct alignas(16) RouteScratch {  // shared memory of one warp, followed by E doubles
  uint32_t key[36];                // candidates; then their values in rank order
  uint32_t id[36];
};
__host__ __device__ __forceinline__ size_t route_scratch_bytes(int E) { return sizeof(RouteScratch) + 8 * (size_t)((E + 1) / 2 * 2); }

__device__ __forceinline__ float fast_sigmoid(float l) {  // off by 2e-7; 0 for -inf, 1 for +inf
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.f + exp2f(l * -1.4426950408889634f)));
  return y;
}

// A router's correction bias in the registers of a warp: what route_token's b holds. Returns the largest finite magnitude.
template <int NPL>
__device__ __forceinline__ float load_choice_bias(const RouteRule& r, int npl, int lane, float (&b)[NPL]) {
  float most = 0.f;
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    const int e = lane * npl + j;
    float v = 0.f;
    if (r.bias != nullptr && j < npl && e < r.E) v = r.bias[e];
    if (fabsf(v) <= 3.402823466e38f) most = fmaxf(most, fabsf(v));
    b[j] = v == v ? v : -CUDART_INF_F;  // no choice can be made with a NaN
  }
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
}

// Row of a token: experts lane * npl .. lane * npl + npl - 1 are l[0 .. npl) of this lane (-inf beyond E; npl <= NPL), b and
// bias_max from load_choice_bias. logit(e) reads the row again. write(j, id, weight) is called once for each j < k, by any lane.
template <int NPL, class Logit, class Write>
__device__ __forceinline__ void route_token(const float (&l)[NPL], int npl, const RouteRule& r, const float (&b)[NPL], float bias_max,
                                            RouteScratch* scratch, int lane, const Logit& logit, const Write& write) {
  const int E = r.E, e0 = lane * npl;
  double* work = reinterpret_cast<double*>(scratch + 1);
  const bool by_logit = r.bias == nullptr, grouped = r.n_group > 1 && r.topk_group < r.n_group, sums = grouped && r.group_top2 != 0;
  bool odd = false;
#pragma unroll
  for (int j = 0; j < NPL; ++j) odd |= !(l[j] < CUDART_INF_F);
  if (__any_sync(0xffffffffu, odd)) {
    bool dead = false;
#pragma unroll
    for (int j = 0; j < NPL; ++j) dead |= l[j] != l[j] || (!r.sigmoid && l[j] == CUDART_INF_F);
    if (__any_sync(0xffffffffu, dead)) {
      if (lane < r.k) write(lane, -1, CUDART_NAN_F);
      return;
    }
  }
  // A float32 score is off by at most 1e-6 of the largest (the exponential's argument is off by half a step, the
  // exponential and the division by about two), a choice by that and half a step of its own.
  float sum = 0.f, top = 0.f, margin = 0.f;
  uint32_t key[NPL];  // ordered choices
  if (!r.sigmoid) {
    top = -CUDART_INF_F;
#pragma unroll
    for (int j = 0; j < NPL; ++j) top = fmaxf(top, l[j]);
    top = key_value(__reduce_max_sync(0xffffffffu, order_key(top)));
    if (top == -CUDART_INF_F) top = 0.f;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      const float e = __expf(l[j] - top);
      key[j] = __float_as_uint(e);
      sum += e;
    }
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  }
  if (!by_logit || sums) {
    const float inv = r.sigmoid ? 1.f : 1.f / sum;
    margin = 4e-6f * (inv + bias_max);
    if (r.sigmoid) {
#pragma unroll
      for (int j = 0; j < NPL; ++j) key[j] = __float_as_uint(fast_sigmoid(l[j]) + b[j]);
    } else {
#pragma unroll
      for (int j = 0; j < NPL; ++j) key[j] = __float_as_uint(fmaf(__uint_as_float(key[j]), inv, b[j]));
    }
#pragma unroll
    for (int j = 0; j < NPL; ++j) key[j] = l[j] > -CUDART_INF_F ? order_key(__uint_as_float(key[j])) : kNone;
  } else {
#pragma unroll
    for (int j = 0; j < NPL; ++j) key[j] = order_key(l[j] + 0.f);
  }
  auto stage_exact = [&]() {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (j < npl && e0 + j < E) work[e0 + j] = (double)l[j];
    exact_choices(work, &r, lane);
  };
  bool staged = false;
  uint32_t kept = 0xffffffffu;
  if (grouped) {
    const int G = r.n_group, per = E / G, L = lanes_per_group(G);
    const bool aligned = npl * 32 == E && 32 % G == 0;  // lane i's experts all belong to group i / L
    const int group = lane / L;                         // this lane's share of the valuation, and with `aligned` its experts'
    uint32_t a = kNone, a2 = kNone;                     // the two best of it
    auto take = [&](uint32_t v) {
      a2 = max(a2, min(a, v));
      a = max(a, v);
    };
    if (aligned) {
#pragma unroll
      for (int j = 0; j < NPL; ++j) take(key[j]);
    } else {
      uint32_t* all = reinterpret_cast<uint32_t*>(work);
      __syncwarp();
#pragma unroll
      for (int j = 0; j < NPL; ++j)
        if (j < npl && e0 + j < E) all[e0 + j] = key[j];
      __syncwarp();
      const int q = lane % L, steps = (per + L - 1) / L;
      if (group < G) {
        int x = group % steps;  // groups start at different steps, so that they meet different banks
        for (int i = 0; i < steps; ++i) {
          const int at = q + L * x;
          take(at < per ? all[group * per + at] : kNone);
          if (++x == steps) x = 0;
        }
      }
    }
    for (int m = L >> 1; m >= 1; m >>= 1) {
      const uint32_t oa = __shfl_xor_sync(0xffffffffu, a, m), ob = __shfl_xor_sync(0xffffffffu, a2, m);
      a2 = max(max(a2, ob), min(a, oa));
      a = max(a, oa);
    }
    uint32_t value = a;  // the same in every lane of a group; kNone in lanes without one
    if (sums && a2 != kNone) value = order_key(key_value(a) + key_value(a2) + 0.f);
    bool in = false;
    float last = 0.f;
    for (int i = 0; i < r.topk_group; ++i) {
      const uint32_t m = __reduce_max_sync(0xffffffffu, value);
      if (m == kNone) break;
      bool mine = value == m;
      const unsigned who = __ballot_sync(0xffffffffu, mine);
      if (__popc(who) != L) mine = group == (__ffs(who) - 1) / L;  // equal groups: the lowest
      in |= mine;
      if (mine) value = kNone;
      last = key_value(m);
    }
    kept = __ballot_sync(0xffffffffu, in);
    const uint32_t next = __reduce_max_sync(0xffffffffu, value);
    const bool close = (!by_logit || sums) && next != kNone && last - key_value(next) < 2.f * margin;  // sums of two choices
    if (L > 1) {  // from bits of lanes to bits of groups
      uint32_t of_groups = 0u;
      for (int g = 0; g < G; ++g) of_groups |= ((kept >> (g * L)) & 1u) << g;
      kept = of_groups;
    }
    if (close) {
      stage_exact();
      staged = true;
      kept = exact_groups(work, &r, lane);
      in = (kept >> group) & 1u;
    }
    if (by_logit && sums) {  // from here on by the logits
#pragma unroll
      for (int j = 0; j < NPL; ++j) key[j] = order_key(l[j] + 0.f);
    }
    if (aligned) {
#pragma unroll
      for (int j = 0; j < NPL; ++j) key[j] = in ? key[j] : kNone;
    } else {
      int g = e0 / per, rem = e0 - g * per;
#pragma unroll
      for (int j = 0; j < NPL; ++j) {
        if (!((kept >> (g & 31)) & 1u)) key[j] = kNone;
        if (++rem == per) {
          rem = 0;
          ++g;
        }
      }
    }
  }
  const int want = by_logit ? r.k : r.k + 1;  // one more to compare the last with
  uint32_t floor_key = kNone;
  {
    uint32_t best = kNone;
#pragma unroll
    for (int j = 0; j < NPL; ++j) best = max(best, key[j]);
    for (int i = 0; i < want; ++i) {  // equal maxima leave together, which only lowers the floor
      floor_key = __reduce_max_sync(0xffffffffu, best);
      if (floor_key == kNone) break;
      if (best == floor_key) best = kNone;
    }
  }
  floor_key = max(floor_key, kNone + 1u);  // fewer lanes than that: everything that can be chosen
  int mine = 0;
#pragma unroll
  for (int j = 0; j < NPL; ++j) mine += key[j] >= floor_key;
  int before = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, before, d);
    if (lane >= d) before += v;
  }
  const int n = __shfl_sync(0xffffffffu, before, 31);
  before -= mine;
  bool close = false;
  int rank = 32, id = -1;
  __syncwarp();
  if (n <= 32) {
    scratch->key[lane] = 0u;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (key[j] >= floor_key) {
        scratch->key[before] = key[j];
        scratch->id[before] = (uint32_t)(e0 + j);
        ++before;
      }
    __syncwarp();
    const uint32_t v = scratch->key[lane];
    const uint4* four = reinterpret_cast<const uint4*>(scratch->key);
    rank = 0;
    for (int i = 0; i < n; i += 4) {  // of equals the one in the lower lane, with the lower id, ranks first
      const uint4 o = four[i / 4];
      rank += (o.x + (i < lane ? 1u : 0u) > v) + (o.y + (i + 1 < lane ? 1u : 0u) > v) + (o.z + (i + 2 < lane ? 1u : 0u) > v) +
              (o.w + (i + 3 < lane ? 1u : 0u) > v);
    }
    if (lane < n) id = (int)scratch->id[lane];
    else rank = 32;
    if (!by_logit) {
      __syncwarp();
      if (lane < n) scratch->key[rank] = v;
      __syncwarp();
      const uint32_t next = lane < n && rank + 1 < n ? scratch->key[rank + 1] : 0u;
      close = __any_sync(0xffffffffu, rank < r.k && next != 0u && key_value(v) - key_value(next) < margin);
    }
  } else {
    // k rounds: the best of every lane, the warp's best of those; a lane keeps the first of equals
    uint32_t best = kNone;
    int at = 0;
    auto scan = [&]() {
      best = kNone;
#pragma unroll
      for (int j = 0; j < NPL; ++j)
        if (key[j] > best) {
          best = key[j];
          at = j;
        }
    };
    scan();
    float last = 0.f;
    for (int i = 0; i < want && !close; ++i) {
      const uint32_t m = __reduce_max_sync(0xffffffffu, best);
      if (m == kNone) break;
      const int win = __ffs(__ballot_sync(0xffffffffu, best == m)) - 1;
      const int e = __shfl_sync(0xffffffffu, e0 + at, win);
      if (!by_logit) {
        const float v = key_value(m);
        if (i > 0) close = last - v < margin;
        last = v;
      }
      if (i < r.k && lane == i) id = e;
      if (lane == win) {
#pragma unroll
        for (int j = 0; j < NPL; ++j)
          if (j == at) key[j] = kNone;
        scan();
      }
    }
    rank = lane;
  }
  if (close) {
    if (!staged) stage_exact();
    id = exact_rank(work, &r, kept, lane);
    rank = lane;
  }
  const bool chosen = id >= 0 && rank < r.k;
  float w = 0.f;
  if (chosen) {
    const float v = logit(id);
    w = r.sigmoid ? __fdividef(1.f, 1.f + expf(-v)) : __fdividef(expf(v - top), sum);
  }
  if (r.norm) {
    float all = w;
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) all += __shfl_xor_sync(0xffffffffu, all, m);
    w = __fdividef(w, all + 1e-20f);
  }
  if (chosen) write(rank, id, w * r.scale);
  const int found = __popc(__ballot_sync(0xffffffffu, chosen));
  if (lane >= found && lane < r.k) write(lane, -1, 0.f);
}

}  // namespace pm
