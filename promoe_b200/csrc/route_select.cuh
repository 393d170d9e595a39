// One warp chooses the experts of one token from its router logits: softmax or sigmoid scores, a correction bias that
// takes part in the choice only, groups of neighbouring experts of which the best few stay, the k best of what is left,
// their scores as weights, renormalised and scaled. Used by the stateless router (route.cu) and by the
// layer call's router (gate_topk.cu) for layers with a router rule.
//
//   score   s_e = softmax(l)_e  or  1 / (1 + exp(-l_e))
//   choice  c_e = s_e + b_e; an expert whose logit or choice is -inf cannot be chosen
//   group   max of its choices, or the sum of its two largest (a missing second counts as nothing);
//           the topk_group best groups stay, ties to the lower group; the others' experts leave, or (drop_zero) their
//           choices become 0
//   ids     the k largest choices among them, descending, ties to the lower id; -1 where there are fewer
//   weight  s_id, divided by (sum of the k + 1e-20) if asked for, times the scale; 0 for id -1
// A row that holds a NaN (softmax: or +inf) has no scores: its ids are -1 and its weights NaN.
//
// Which expert is chosen must not depend on float32 rounding. Without a bias experts are ranked by their logits (scores are
// monotonic in them). Choices with a bias and sums of two are ranked in float32, and a row in which two neighbours of a
// ranking lie closer than the error bound of those numbers is ranked again in 64 bits (about one row in a thousand).
#pragma once
#include <math_constants.h>

#include "pm_common.cuh"

namespace pm {

// The choice of what cannot be chosen is -inf.

// The largest of a warp's numbers, in one instruction; no NaN among them.
__device__ __forceinline__ float warp_top(float v) {
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
__device__ __forceinline__ uint32_t order_key(float v) {  // integers in the order of the numbers; not for -0
  const uint32_t b = __float_as_uint(v);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

// A lane's place in the rule's groups.
struct RouteGroups {
  int lanes;     // that share the valuation of a group: the same power of two for each of at most 32 groups
  int per;       // experts of a group
  int group;     // this lane's, n_group and more without one
  bool aligned;  // lane i's own experts all belong to its group
  __device__ __forceinline__ RouteGroups(const RouteRule& r, int npl, int lane) {
    const int shift = 31 - __clz(32 / r.n_group);
    lanes = 1 << shift;
    per = r.E / r.n_group;
    group = lane >> shift;
    aligned = npl * 32 == r.E && 32 % r.n_group == 0;
  }
};

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

// The sum behind the softmax scores; c holds the logits.
static __device__ __noinline__ double exact_sum(const double* c, int E, double top, int lane) {
  double sum = 0.0;
  __syncwarp();
  for (int e = lane; e < E; e += 32) sum += exp(c[e] - top);
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  return sum;
}

// Rank of each of the n <= 32 candidates, one per lane in the order of their ids, by a choice that `sum` (softmax) makes exact; 0
// for one of a dropped group.
static __device__ __noinline__ int exact_candidates(double logit, float bias, double top, double sum, int sigmoid, bool dropped, int n,
                                                    int lane) {
  const double v = dropped ? 0.0 : (sigmoid ? 1.0 / (1.0 + exp(-logit)) : exp(logit - top) / sum) + (double)bias;
  int rank = 0;
  for (int i = 0; i < n; ++i) {
    const double o = __shfl_sync(0xffffffffu, v, i);
    rank += o > v || (o == v && i < lane);
  }
  return lane < n ? rank : 32;
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

// Lane j < k returns the j-th of the experts in the groups `kept` (drop_zero: of all), -1 if there are fewer. Uses c up.
static __device__ __noinline__ int exact_rank(double* c, const RouteRule* rule, uint32_t kept, int lane) {
  const int E = rule->E, per = E / rule->n_group;
  for (int e = lane; e < E; e += 32)
    if (!((kept >> (e / per)) & 1u)) c[e] = rule->drop_zero && c[e] > -CUDART_INF ? 0.0 : -CUDART_INF;
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
  uint32_t key[36];                // candidates as ordered integers; then their choices in rank order
  float2 candidate[32];            // choice and id
};
__host__ __device__ __forceinline__ size_t route_scratch_bytes(int E) { return sizeof(RouteScratch) + 8 * (size_t)((E + 1) / 2 * 2); }

// Off by less than 3e-7: the exponential by 2^-22 of itself and by what half a step of its argument makes of it, which moves
// the quotient by a quarter of that at most; the sum by half a step, the reciprocal by one. 0 for -inf, 1 for +inf.
__device__ __forceinline__ float fast_sigmoid(float l) {
  float t, y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(l * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.f + t));
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
// bias_max from load_choice_bias, groups of this lane. logit(e) reads the row again. write(j, id, weight) is called once for each j < k, by any lane.
// KIND: what of the rule is fixed when the code is compiled (route_kind), or kAnyRule.
constexpr int kAnyRule = -1, kHasBias = 1, kGrouped = 2, kSigmoid = 4;
__host__ __device__ __forceinline__ int route_kind(const RouteRule& r) {
  return (r.bias != nullptr ? kHasBias : 0) | (r.n_group > 1 && r.topk_group < r.n_group ? kGrouped : 0) | (r.sigmoid ? kSigmoid : 0);
}
template <int NPL, int KIND, class Logit, class Write>
__device__ __forceinline__ void route_token(const float (&l)[NPL], int npl, const RouteRule& r, const float (&b)[NPL], float bias_max,
                                            const RouteGroups& groups, RouteScratch* scratch, int lane, const Logit& logit, const Write& write) {
  const int E = r.E, e0 = lane * npl;
  double* work = reinterpret_cast<double*>(scratch + 1);
  const int kind = KIND == kAnyRule ? route_kind(r) : KIND;
  const bool by_logit = !(kind & kHasBias), grouped = (kind & kGrouped) != 0, sigmoid = (kind & kSigmoid) != 0;
  const bool sums = grouped && r.group_top2 != 0;
  const bool zero = KIND == kAnyRule && grouped && r.drop_zero != 0;  // the fixed kinds let the experts of dropped groups leave
  bool odd = false;
#pragma unroll
  for (int j = 0; j < NPL; ++j) odd |= !(fabsf(l[j]) < CUDART_INF_F);
  odd = __any_sync(0xffffffffu, odd);
  if (odd) {
    bool dead = false;
#pragma unroll
    for (int j = 0; j < NPL; ++j) dead |= l[j] != l[j] || (!sigmoid && l[j] == CUDART_INF_F);
    if (__any_sync(0xffffffffu, dead)) {
      if (lane < r.k) write(lane, -1, CUDART_NAN_F);
      return;
    }
  }
  // How far apart two float32 choices have to be for their order to be certain: twice the error of one. A sigmoid score is
  // off by 3e-7, a softmax score by 1.5e-6 of the largest (the sum of up to 37 roundings, the exponential and the division by
  // two or three), a choice by that and half a step of its own.
  float sum = 0.f, top = 0.f, margin = 0.f;
  float c[NPL];  // choices
  if (!sigmoid) {
    top = -CUDART_INF_F;
#pragma unroll
    for (int j = 0; j < NPL; ++j) top = fmaxf(top, l[j]);
    top = warp_top(top);
    if (top == -CUDART_INF_F) top = 0.f;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      c[j] = __expf(l[j] - top);
      sum += c[j];
    }
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  }
  if (!by_logit || sums) {
    const float inv = sigmoid ? 1.f : 1.f / sum;
    margin = (sigmoid ? 1e-6f : 4e-6f * inv) + 1e-6f * bias_max;
    if (sigmoid) {
#pragma unroll
      for (int j = 0; j < NPL; ++j) c[j] = fast_sigmoid(l[j]) + b[j];
    } else {
#pragma unroll
      for (int j = 0; j < NPL; ++j) c[j] = fmaf(c[j], inv, b[j]);
    }
    if (odd) {
#pragma unroll
      for (int j = 0; j < NPL; ++j) c[j] = l[j] > -CUDART_INF_F ? c[j] : -CUDART_INF_F;
    }
  } else {
#pragma unroll
    for (int j = 0; j < NPL; ++j) c[j] = l[j] + 0.f;  // no -0
  }
  auto stage_logits = [&]() {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (j < npl && e0 + j < E) work[e0 + j] = (double)l[j];
  };
  uint32_t lanes_in = 0xffffffffu;  // lanes whose group stays
  auto kept_groups = [&]() {        // the same as bits of groups
    uint32_t kept = 0u;
    for (int g = 0; g < r.n_group; ++g) kept |= ((lanes_in >> (g * groups.lanes)) & 1u) << g;
    return kept;
  };
  if (grouped) {
    const int G = r.n_group, per = groups.per, L = groups.lanes, group = groups.group;
    const bool aligned = groups.aligned;
    float a = -CUDART_INF_F, a2 = -CUDART_INF_F;  // the two best of this lane's share of its group
    auto take = [&](float v) {
      a2 = fmaxf(a2, fminf(a, v));
      a = fmaxf(a, v);
    };
    if (aligned) {
#pragma unroll
      for (int j = 0; j < NPL; ++j) take(c[j]);
    } else {
      float* all = reinterpret_cast<float*>(work);
      __syncwarp();
#pragma unroll
      for (int j = 0; j < NPL; ++j)
        if (j < npl && e0 + j < E) all[e0 + j] = c[j];
      __syncwarp();
      const int q = lane & (L - 1), steps = (per + L - 1) / L;
      if (group < G) {
        int x = group % steps;  // groups start at different steps, so that they meet different banks
        for (int i = 0; i < steps; ++i) {
          const int at = q + L * x;
          take(at < per ? all[group * per + at] : -CUDART_INF_F);
          if (++x == steps) x = 0;
        }
      }
    }
    for (int m = L >> 1; m >= 1; m >>= 1) {
      const float oa = __shfl_xor_sync(0xffffffffu, a, m), ob = __shfl_xor_sync(0xffffffffu, a2, m);
      a2 = fmaxf(fmaxf(a2, ob), fminf(a, oa));
      a = fmaxf(a, oa);
    }
    float value = a;  // the same in every lane of a group; -CUDART_INF_F in lanes without one
    if (sums && a2 > -CUDART_INF_F) value = a + a2;
    int before = 0;  // groups that rank before this one
    for (int g = 0; g < G; ++g) {
      const float o = __shfl_sync(0xffffffffu, value, g * L);
      before += g < group ? o >= value : o > value;
    }
    bool in = before < r.topk_group && value > -CUDART_INF_F;
    bool close = false;
    if (!by_logit || sums) {  // sums of two choices
      const float next = warp_top(in ? -CUDART_INF_F : value), last = -warp_top(in ? -value : -CUDART_INF_F);
      close = next > -CUDART_INF_F && last - next < 2.f * margin;
    }
    if (close) {
      stage_logits();
      exact_choices(work, &r, lane);
      const uint32_t kept = exact_groups(work, &r, lane);
      in = (kept >> group) & 1u;
    }
    lanes_in = __ballot_sync(0xffffffffu, in);
    if (by_logit && sums) {  // from here on by the logits
#pragma unroll
      for (int j = 0; j < NPL; ++j) c[j] = l[j] + 0.f;
    }
    if (aligned) {
#pragma unroll
      for (int j = 0; j < NPL; ++j) c[j] = in ? c[j] : zero && c[j] > -CUDART_INF_F ? 0.f : -CUDART_INF_F;
    } else {
      const uint32_t kept = kept_groups();
      int g = e0 / per, rem = e0 - g * per;
#pragma unroll
      for (int j = 0; j < NPL; ++j) {
        if (!((kept >> (g & 31)) & 1u)) c[j] = zero && c[j] > -CUDART_INF_F ? 0.f : -CUDART_INF_F;
        if (++rem == per) {
          rem = 0;
          ++g;
        }
      }
    }
  }
  const int want = by_logit ? r.k : r.k + 1;  // one more to compare the last with
  float floor = -CUDART_INF_F;
  {
    float best = -CUDART_INF_F;
#pragma unroll
    for (int j = 0; j < NPL; ++j) best = fmaxf(best, c[j]);
    for (int i = 0; i < want; ++i) {  // equal maxima leave together, which only lowers the floor
      floor = warp_top(best);
      if (best == floor) best = -CUDART_INF_F;
    }
  }
  // Fewer lanes than that: everything that can be chosen. Else also what float32 may have put below the floor.
  if (!by_logit) floor -= margin;
  floor = fmaxf(floor, -3.402823466e38f);
  int mine = 0;
#pragma unroll
  for (int j = 0; j < NPL; ++j) mine += c[j] >= floor;
  int before = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, before, d);
    if (lane >= d) before += v;
  }
  const int n = __shfl_sync(0xffffffffu, before, 31);
  before -= mine;
  int rank = 32, id = -1;
  float v_id = 0.f;  // the logit of id
  __syncwarp();
  if (n <= 32) {
    scratch->candidate[lane].x = -CUDART_INF_F;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (c[j] >= floor) {
        scratch->candidate[before] = make_float2(c[j], __int_as_float(e0 + j));
        ++before;
      }
    __syncwarp();
    const float choice = scratch->candidate[lane].x;
    const uint32_t v = order_key(choice);
    scratch->key[lane] = v;
    __syncwarp();
    const uint4* four = reinterpret_cast<const uint4*>(scratch->key);
    rank = 0;
    for (int i = 0; i < n; i += 4) {  // of equals the one in the lower lane, with the lower id, ranks first
      const uint4 o = four[i / 4];
      rank += (o.x + (i < lane ? 1u : 0u) > v) + (o.y + (i + 1 < lane ? 1u : 0u) > v) + (o.z + (i + 2 < lane ? 1u : 0u) > v) +
              (o.w + (i + 3 < lane ? 1u : 0u) > v);
    }
    if (lane < n) {
      id = __float_as_int(scratch->candidate[lane].y);
      v_id = logit(id);
    } else {
      rank = 32;
    }
    if (!by_logit) {
      __syncwarp();
      if (lane < n) scratch->key[rank] = __float_as_uint(choice);
      __syncwarp();
      const bool close = rank < r.k && rank + 1 < n && choice - __uint_as_float(scratch->key[rank + 1]) < margin;
      if (__any_sync(0xffffffffu, close)) {
        double sum64 = 1.0;
        if (!sigmoid) {
          stage_logits();
          sum64 = exact_sum(work, E, (double)top, lane);
        }
        const bool dropped = zero && lane < n && !((kept_groups() >> (id / groups.per)) & 1u);
        rank = exact_candidates((double)v_id, lane < n ? r.bias[id] : 0.f, (double)top, sum64, sigmoid, dropped, n, lane);
      }
    }
  } else {
    // k rounds: the best of every lane, the warp's best of those; a lane keeps the first of equals
    float best = -CUDART_INF_F;
    int at = 0;
    auto scan = [&]() {
      best = -CUDART_INF_F;
#pragma unroll
      for (int j = 0; j < NPL; ++j)
        if (c[j] > best) {
          best = c[j];
          at = j;
        }
    };
    scan();
    float last = 0.f;
    bool close = false;
    for (int i = 0; i < want && !close; ++i) {
      const float m = warp_top(best);
      if (m == -CUDART_INF_F) break;
      const int win = __ffs(__ballot_sync(0xffffffffu, best == m)) - 1;
      const int e = __shfl_sync(0xffffffffu, e0 + at, win);
      if (!by_logit) {
        if (i > 0) close = last - m < margin;
        last = m;
      }
      if (i < r.k && lane == i) id = e;
      if (lane == win) {
#pragma unroll
        for (int j = 0; j < NPL; ++j)
          if (j == at) c[j] = -CUDART_INF_F;
        scan();
      }
    }
    if (close) {
      stage_logits();
      exact_choices(work, &r, lane);
      id = exact_rank(work, &r, kept_groups(), lane);
    }
    rank = lane;
    if (id >= 0) v_id = logit(id);
  }
  const bool chosen = id >= 0 && rank < r.k;
  float w = 0.f;
  if (chosen) {
    const float e = expf(sigmoid ? -fabsf(v_id) : v_id - top);  // at most 1: the quick division gives 0 for quotients by more than 2^126
    w = __fdividef(sigmoid && v_id >= 0.f ? 1.f : e, sigmoid ? 1.f + e : sum);
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
