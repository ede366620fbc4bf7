// Routing of tokens to experts from the router's logits l (rows, E):
//   s_e = sigmoid(l_e) or softmax(l)_e
//   ranked by s_e + bias_e, or without a bias by l_e (the order of the scores,
//   without the ties that rounding a score makes)
//   with groups of E / G experts: the best `top_groups` groups, a group
//   counting as its best expert or as the sum of its two best, and then the
//   best k experts of those; ties go to the lower index
//   gates_i = scale · s_i / Σ_selected s, or scale · s_i
// Scores that are compared are held in 64 bits: two experts whose scores
// differ by less than fp32 resolves still have one order.  An expert whose
// logit is -inf or NaN, or whose bias is, takes no part: it comes after every
// other expert of the chosen groups and its gate is 0, so that a row with
// nothing left has valid, distinct experts and gates of 0.
#include "common.h"
#include "route.h"

#include <math.h>

namespace rwkvmoe {
namespace {

constexpr float kInf = __builtin_inff();

template <typename T> RWKV_DEV float load_logit(const T* p) {
  const float l = to_f(*p);
  return l == l ? l : -kInf;  // a NaN takes no part
}

// The group's score from its best two keys (-inf: none left).
RWKV_DEV double group_score(double a, double b, bool top2) {
  return top2 && b > -(double)kInf ? a + b : a;
}

// L lanes a row, V keys a lane: lane i holds experts [i·per, (i + 1)·per).
//   KT     double, or float where the logits themselves are compared
//   LDSG   groups that do not lie on whole lanes: their scores go through LDS
template <typename T, typename KT, int L, int V, bool LDSG>
__global__ __launch_bounds__(256) void route_kernel(Route p, int per) {
  constexpr int RW = 64 / L, RPB = 256 / L;
  static_assert(!LDSG || L == 64, "one row a wave");
  __shared__ double sk[LDSG ? RPB : 1][LDSG ? kRouteMaxE : 1];
  __shared__ double sg[LDSG ? RPB : 1][LDSG ? kRouteMaxGroups : 1];
  __shared__ unsigned char sok[LDSG ? RPB : 1][LDSG ? kRouteMaxGroups : 1];
  const int lane = threadIdx.x & 63, sub = lane % L;
  const int row_raw = (blockIdx.x * 4 + (threadIdx.x >> 6)) * RW + lane / L;
  const int row = min(row_raw, p.rows - 1);  // (rows past the end repeat the last one and are not written)
  const T* lg = (const T*)p.logits + (size_t)row * p.stride;
  const int e0 = sub * per;
  const KT ninf = -(KT)kInf;

  KT key[V];
  unsigned alive = 0;
  float lmax = -kInf;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const bool in = i < per && e0 + i < p.E;
    const float l = in ? load_logit(lg + e0 + i) : -kInf;
    key[i] = (KT)l;
    lmax = fmaxf(lmax, l);
    if (in) alive |= 1u << i;
  }
  const bool need_max = !p.sigmoid && (!p.renorm || sizeof(KT) == 8);
  double total = 1.0;
  if (need_max) {
#pragma unroll
    for (int d = 1; d < L; d <<= 1) lmax = fmaxf(lmax, __shfl_xor(lmax, d));
  }
  // (l - max as 0 where both are the same infinity)
  auto ex = [&](float l, float m) { return l == m && l > -kInf ? 1.0 : exp((double)l - (double)m); };
  if constexpr (sizeof(KT) == 8) {
    if (p.sigmoid) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < per && key[i] > ninf) key[i] = 1.0 / (1.0 + exp(-key[i]));
    } else if (lmax > -kInf) {
      total = 0.0;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < per && key[i] > ninf) {
          key[i] = ex((float)key[i], lmax);
          total += key[i];
        }
#pragma unroll
      for (int d = 1; d < L; d <<= 1) total += __shfl_xor(total, d);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < per && key[i] > ninf) key[i] /= total;
    }
    if (p.bias) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (alive >> i & 1) {
          const float b = p.bias[e0 + i];
          key[i] = b > -kInf && key[i] > ninf ? key[i] + (double)b : ninf;  // (a NaN bias is no bias > -inf)
        }
    }
  } else {
    if (!p.sigmoid && !p.renorm && lmax > -kInf) {  // the softmax's sum over all experts
      total = 0.0;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < per && key[i] > ninf) total += ex((float)key[i], lmax);
#pragma unroll
      for (int d = 1; d < L; d <<= 1) total += __shfl_xor(total, d);
    }
  }

  if (p.groups > 1) {
    const int S = p.E / p.groups;
    if constexpr (LDSG) {
      const int wr = threadIdx.x >> 6;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (alive >> i & 1) sk[wr][e0 + i] = (double)key[i];
      __syncthreads();
      if (sub < p.groups) {
        double a = ninf, b = ninf;
        for (int i = 0; i < S; ++i) {
          const double v = sk[wr][sub * S + i];
          b = v > a ? a : (v > b ? v : b);
          a = v > a ? v : a;
        }
        sg[wr][sub] = group_score(a, b, p.top2);
      }
      __syncthreads();
      if (sub < p.groups) {
        const double mine = sg[wr][sub];
        int above = 0;
        for (int g = 0; g < p.groups; ++g) above += sg[wr][g] > mine || (sg[wr][g] == mine && g < sub);
        sok[wr][sub] = above < p.top_groups;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < V; ++i)
        if ((alive >> i & 1) && !sok[wr][(e0 + i) / S]) alive &= ~(1u << i);
    } else {
      // a group is 2^j whole lanes
      const int lpg = S / per, g = sub / lpg;
      KT a = ninf, b = ninf;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < per) {
          b = key[i] > a ? a : (key[i] > b ? key[i] : b);
          a = key[i] > a ? key[i] : a;
        }
      for (int d = 1; d < lpg; d <<= 1) {
        const KT oa = __shfl_xor(a, d), ob = __shfl_xor(b, d);
        const KT lo = oa > a ? a : oa, hb = ob > b ? ob : b;
        a = oa > a ? oa : a;
        b = lo > hb ? lo : hb;
      }
      const double mine = group_score((double)a, (double)b, p.top2);
      int above = 0;
      for (int q = 0; q < p.groups; ++q) {
        const double v = __shfl(mine, (lane - sub) + q * lpg);
        above += v > mine || (v == mine && q < g);
      }
      if (above >= p.top_groups) alive = 0;
    }
  }

  // k times the best of what is left
  int mine = 0;  // slot `sub` (and sub + L) of the row
  int mine2 = 0;
  bool live = false, live2 = false;
  for (int j = 0; j < p.k; ++j) {
    KT best = ninf;
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const bool take = (alive >> i & 1) && (key[i] > best || at == 0x7fffffff);
      best = take ? key[i] : best;
      at = take ? e0 + i : at;
    }
#pragma unroll
    for (int d = 1; d < L; d <<= 1) {
      const KT ob = __shfl_xor(best, d);
      const int oa = __shfl_xor(at, d);
      const bool take = ob > best || (ob == best && oa < at);
      best = take ? ob : best;
      at = take ? oa : at;
    }
    const int i = at - e0;
    if (i >= 0 && i < per) alive &= ~(1u << i);
    if (j % L == sub) {
      if (j < L) {
        mine = at;
        live = best > ninf;
      } else {
        mine2 = at;
        live2 = best > ninf;
      }
    }
  }

  // the gates: one slot a lane (two where k is more than L)
  auto score = [&](int e, bool on, float m) {
    if (!on) return 0.0;
    const float l = load_logit(lg + e);
    return p.sigmoid ? 1.0 / (1.0 + exp(-(double)l)) : ex(l, m);
  };
  float m = lmax;
  if (!p.sigmoid && p.renorm) {  // relative to the largest that is selected
    m = live ? load_logit(lg + mine) : -kInf;
    if (live2) m = fmaxf(m, load_logit(lg + mine2));
#pragma unroll
    for (int d = 1; d < L; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  }
  const double s1 = sub < p.k ? score(mine, live, m) : 0.0;
  const double s2 = sub + L < p.k ? score(mine2, live2, m) : 0.0;
  double div = p.sigmoid ? 1.0 : total;
  if (p.renorm) {
    div = s1 + s2;
#pragma unroll
    for (int d = 1; d < L; d <<= 1) div += __shfl_xor(div, d);
  }
  const double c = div > 0.0 ? (double)p.scale / div : 0.0;
  if (row_raw < p.rows) {
    if (sub < p.k) {
      p.inds[(size_t)row * p.k + sub] = mine;
      p.gates[(size_t)row * p.k + sub] = (float)(s1 * c);
    }
    if (sub + L < p.k) {
      p.inds[(size_t)row * p.k + sub + L] = mine2;
      p.gates[(size_t)row * p.k + sub + L] = (float)(s2 * c);
    }
  }
}

// d_logits from the gates' cotangents.  With u_i = s_i over the selected and
// U = Σ u:  renormalised d s_i = (scale / U)(d_i - Σ_j d_j u_j / U), else
// scale · d_i;  sigmoid d l_i = d s_i · s_i (1 - s_i);  softmax
// d l_e = s_e ([e selected] d s_e - Σ_i d s_i s_i), which is 0 off the selected
// experts where the gates are renormalised.  Half a wave a row, a lane a slot;
// every expert of the row is written.  A slot whose gate is 0 took no part.
template <typename T>
__global__ __launch_bounds__(256) void route_bwd_kernel(Route p) {
  const int lane = threadIdx.x & 31;
  const int row_raw = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int row = min(row_raw, p.rows - 1);
  const T* lg = (const T*)p.logits + (size_t)row * p.stride;
  auto sum = [&](double v) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) v += __shfl_xor(v, d);
    return v;
  };
  int e = -1;
  float l = -kInf;
  double dg = 0.0;
  if (lane < p.k) {
    e = p.inds_in[(size_t)row * p.k + lane];
    if (e >= 0 && e < p.E && p.gates_in[(size_t)row * p.k + lane] != 0.f) {
      l = load_logit(lg + e);
      dg = (double)p.d_gates[(size_t)row * p.k + lane];
    } else {
      e = -1;  // (an id that no expert has is dropped)
    }
  }
  const bool on = e >= 0 && l > -kInf;
  const bool dense = !p.sigmoid && !p.renorm;
  float m = l;
  if (dense)
    for (int i = lane; i < p.E; i += 32) m = fmaxf(m, load_logit(lg + i));
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  auto ex = [&](float v) { return v == m && v > -kInf ? 1.0 : exp((double)v - (double)m); };
  double total = 1.0, s = 0.0, rest = 0.0;
  if (p.sigmoid) {
    if (on) {
      s = 1.0 / (1.0 + exp(-(double)l));
      rest = 1.0 / (1.0 + exp((double)l));  // 1 - s
    }
  } else {
    if (dense) {
      total = 0.0;
      for (int i = lane; i < p.E; i += 32) {
        const float v = load_logit(lg + i);
        if (v > -kInf) total += ex(v);
      }
      total = sum(total);
    }
    if (on) s = ex(l) / total;
  }
  double ds = dg * (double)p.scale;
  if (p.renorm) {
    const double U = sum(s);
    const double mean = sum(ds * s);
    ds = U > 0.0 ? (ds - mean / U) / U : 0.0;
  }
  double dl = on ? ds * s : 0.0;
  double back = 0.0;
  if (p.sigmoid) dl *= rest;
  else if (dense) back = sum(dl);

  T* out = (T*)p.d_logits + (size_t)row * p.E;
  const bool vec = p.E % 4 == 0;
  for (int c = 0; c < p.E; c += 128) {
    const int i0 = c + lane * 4;
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    if (dense) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (i0 + q < p.E) {
          const float x = load_logit(lg + i0 + q);
          if (x > -kInf) v[q] = -back * (ex(x) / total);
        }
    }
    for (int j = 0; j < p.k; ++j) {
      const int d = __shfl(e, (threadIdx.x & 32) + j) - i0;
      const double add = __shfl(dl, (threadIdx.x & 32) + j);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] += d == q ? add : 0.0;
    }
    if (row_raw >= p.rows) continue;
    if (vec) {
      if (i0 < p.E) {
        union { T e[4]; unsigned u[sizeof(T)]; } w;
#pragma unroll
        for (int q = 0; q < 4; ++q) w.e[q] = from_f<T>((float)v[q]);
        typedef unsigned uvec __attribute__((ext_vector_type(sizeof(T))));
        *(uvec*)(out + i0) = *(const uvec*)w.u;
      }
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (i0 + q < p.E) out[i0 + q] = from_f<T>((float)v[q]);
    }
  }
}

template <typename T, typename KT, int L, int V, bool LDSG>
hipError_t run(const Route& p, int per, hipStream_t s) {
  constexpr int RPB = 256 / L;
  launch_kernel(route_kernel<T, KT, L, V, LDSG>, dim3((p.rows + RPB - 1) / RPB), dim3(256), 0, s, p, per);
  return hipGetLastError();
}

inline bool on_lanes(const Route& p, int L, int per) {
  if (p.groups == 1) return true;
  const int S = p.E / p.groups;
  if (S % per) return false;
  const int lpg = S / per;
  return (lpg & (lpg - 1)) == 0 && lpg * p.groups <= L;
}

template <typename T, typename KT>
hipError_t run_key(const Route& p, hipStream_t s) {
  const int per64 = (p.E + 63) / 64, per16 = (p.E + 15) / 16;
  // 16 lanes a row take four rows a wave through the reductions at once; with
  // too few rows to fill the card 64 lanes have less to do each
  const bool many = p.rows >= 4096;
  if (many && on_lanes(p, 16, per16)) {
    if (per16 <= 4) return run<T, KT, 16, 4, false>(p, per16, s);
    if (per16 <= 8) return run<T, KT, 16, 8, false>(p, per16, s);
    if (per16 <= 16) return run<T, KT, 16, 16, false>(p, per16, s);
    return run<T, KT, 16, 32, false>(p, per16, s);
  }
  if (on_lanes(p, 64, per64))
    return per64 <= 4 ? run<T, KT, 64, 4, false>(p, per64, s) : run<T, KT, 64, 8, false>(p, per64, s);
  return per64 <= 4 ? run<T, KT, 64, 4, true>(p, per64, s) : run<T, KT, 64, 8, true>(p, per64, s);
}

}  // namespace

hipError_t launch_route(const Route& p, hipStream_t s) {
  // without a bias, and without sums of scores, the logits are compared
  const bool scores = p.bias || (p.groups > 1 && p.top2);
  hipError_t e = hipErrorInvalidValue;
  RWKV_DISPATCH_DTYPE(p.dtype, T, { e = scores ? run_key<T, double>(p, s) : run_key<T, float>(p, s); });
  return mark(e, "route", s);
}

hipError_t launch_route_backward(const Route& p, hipStream_t s) {
  RWKV_DISPATCH_DTYPE(p.dtype, T, {
    launch_kernel(route_bwd_kernel<T>, dim3((p.rows + 7) / 8), dim3(256), 0, s, p);
  });
  return mark(hipGetLastError(), "route_bwd", s);
}

}  // namespace rwkvmoe
