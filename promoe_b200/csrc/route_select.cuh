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

__device__ __forceinline__ uint32_t order_key(float v) {  // ascending with v; 0 is below every number
  const uint32_t b = __float_as_uint(v + 0.f);            // -0 and 0 are the same
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// Lanes that share a group: the same power of two for each of G <= 32 groups.
__device__ __forceinline__ int lanes_per_group(int G) { return 1 << (31 - __clz(32 / G)); }

// ---- the same ranking in 64 bits; c[E] is shared memory of the warp ------------------------------------------
// Logits in c become choices.
__device__ __noinline__ void exact_choices(double* c, const RouteRule* rule, int lane) {
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
__device__ __noinline__ uint32_t exact_groups(const double* c, const RouteRule* rule, int lane) {
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
__device__ __noinline__ int exact_rank(double* c, const RouteRule* rule, uint32_t kept, int lane) {
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

// Experts lane * npl .. lane * npl + npl - 1 of the row are l[0 .. npl) of this lane (-inf beyond E; npl <= NPL).
// work: E doubles of shared memory of this warp. bias_max: largest |finite bias|, 0 without one. logit(e) reads the row again.
// Lane j < k gets the j-th id and its weight.
template <int NPL, class Logit>
__device__ __forceinline__ void route_token(const float (&l)[NPL], int npl, const RouteRule& r, float bias_max, double* work,
                                            int lane, const Logit& logit, int& id, float& weight) {
  const int E = r.E, e0 = lane * npl;
  const bool by_logit = r.bias == nullptr, grouped = r.n_group > 1 && r.topk_group < r.n_group, sums = grouped && r.group_top2 != 0;
  float top = -CUDART_INF_F;
  bool odd = false;
#pragma unroll
  for (int j = 0; j < NPL; ++j)
    if (j < npl) {
      odd |= !(l[j] <= 3.402823466e38f) && (l[j] != l[j] || !r.sigmoid);
      top = fmaxf(top, l[j]);
    }
  id = -1;
  if (__any_sync(0xffffffffu, odd)) {
    weight = CUDART_NAN_F;
    return;
  }
  weight = 0.f;
  top = key_value(__reduce_max_sync(0xffffffffu, order_key(top)));
  if (top == -CUDART_INF_F) return;  // nothing to choose from
  float sum = 0.f;
  float s[NPL];
  if (!r.sigmoid) {
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      s[j] = j < npl ? __expf(l[j] - top) : 0.f;
      sum += s[j];
    }
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  }
  uint32_t key[NPL];  // 0: cannot be chosen
#pragma unroll
  for (int j = 0; j < NPL; ++j) key[j] = j < npl && l[j] > -CUDART_INF_F ? order_key(l[j]) : 0u;
  // A float32 score is off by at most 1e-6 of the largest (the exponential's argument is off by half a step, the
  // exponential and the division by about two), a choice by that and half a step of its own.
  float margin = 0.f;
  uint32_t* ck = reinterpret_cast<uint32_t*>(work);  // what the groups are valued by
  if (grouped) __syncwarp();
  if (!by_logit || sums) {
    const float inv = r.sigmoid ? 1.f : 1.f / sum;
    margin = 4e-6f * (inv + bias_max);
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (j < npl && e0 + j < E) {
        uint32_t ckey = 0u;
        if (key[j] != 0u) {
          float c = r.sigmoid ? __fdividef(1.f, 1.f + __expf(-fmaxf(l[j], -80.f))) : s[j] * inv;
          if (!by_logit) c += r.bias[e0 + j];
          if (c > -CUDART_INF_F) ckey = order_key(c);  // not NaN either
        }
        if (grouped) ck[e0 + j] = ckey;
        if (!by_logit) key[j] = ckey;
      }
  } else if (grouped) {
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (j < npl && e0 + j < E) ck[e0 + j] = key[j];
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
    __syncwarp();
    const int per = E / r.n_group, L = lanes_per_group(r.n_group);
    const int g = lane / L, q = lane % L, steps = (per + L - 1) / L;
    uint32_t a = 0u, b = 0u;  // the group's two best
    if (g < r.n_group) {
      int x = g % steps;  // groups start at different steps, so that they meet different banks
      for (int i = 0; i < steps; ++i) {
        const int at = q + L * x;
        const uint32_t v = at < per ? ck[g * per + at] : 0u;
        b = max(b, min(a, v));
        a = max(a, v);
        if (++x == steps) x = 0;
      }
    }
    for (int m = L >> 1; m >= 1; m >>= 1) {
      const uint32_t oa = __shfl_xor_sync(0xffffffffu, a, m), ob = __shfl_xor_sync(0xffffffffu, b, m);
      b = max(max(b, ob), min(a, oa));
      a = max(a, oa);
    }
    uint32_t value = q == 0 ? a : 0u;
    if (sums && value != 0u && b != 0u) value = order_key(key_value(a) + key_value(b));
    kept = 0u;
    float last = 0.f;
    bool close = false;
    for (int i = 0; i <= r.topk_group; ++i) {
      const uint32_t m = __reduce_max_sync(0xffffffffu, value);
      if (m == 0u) break;
      const int win = __ffs(__ballot_sync(0xffffffffu, value == m)) - 1;
      if (i < r.topk_group) {
        kept |= 1u << (win / L);
        last = key_value(m);
        if (lane == win) value = 0u;
      } else {
        close = (!by_logit || sums) && last - key_value(m) < 2.f * margin;  // sums of two choices
      }
    }
    if (close) {
      stage_exact();
      staged = true;
      kept = exact_groups(work, &r, lane);
    }
    int gj = e0 / per, rem = e0 - gj * per;
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (j < npl) {
        if (!((kept >> (gj & 31)) & 1u)) key[j] = 0u;
        if (++rem == per) {
          rem = 0;
          ++gj;
        }
      }
  }
  // k rounds: the best of every lane, the warp's best of those. Lower lanes hold lower ids, a lane keeps the first of equals.
  uint32_t best = 0u;
  int at = 0;
  auto scan = [&]() {
    best = 0u;
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (j < npl && key[j] > best) {
        best = key[j];
        at = j;
      }
  };
  scan();
  float last = 0.f;
  bool close = false;
  const int rounds = by_logit ? r.k : r.k + 1;
  for (int i = 0; i < rounds && !close; ++i) {
    const uint32_t m = __reduce_max_sync(0xffffffffu, best);
    if (m == 0u) break;
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
        if (j == at) key[j] = 0u;
      scan();
    }
  }
  if (close) {
    if (!staged) stage_exact();
    id = exact_rank(work, &r, kept, lane);
  }
  if (lane >= r.k) id = -1;
  float w = 0.f;
  if (id >= 0) {
    const float v = logit(id);
    w = r.sigmoid ? 1.f / (1.f + expf(-v)) : expf(v - top) / sum;
  }
  if (r.norm) {
    float all = w;
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) all += __shfl_xor_sync(0xffffffffu, all, m);
    w = w / (all + 1e-20f);
  }
  weight = w * r.scale;
}

}  // namespace pm
