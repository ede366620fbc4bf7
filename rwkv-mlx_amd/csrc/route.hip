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

#include <type_traits>

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

// exp(l - m), with 1 where both are the same infinity.
RWKV_DEV double ex(float l, float m) { return l == m && l > -kInf ? 1.0 : exp((double)l - (double)m); }

// The gates of a row from its selected experts: slot `sub` of the row in
// `mine` (slot sub + L in mine2), live where the expert takes part.  lmax and
// total: the row's largest logit and Σ exp(l - lmax), for a softmax that is
// not renormalised.
template <typename T, int L>
RWKV_DEV void write_gates(const Route& p, const T* lg, int row, int mine, int mine2, bool live, bool live2, float lmax,
                          double total) {
  const int sub = (threadIdx.x & 63) % L;
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
  if (row < p.rows) {
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

// The selection of a row with keys in 64 bits: L lanes a row, V keys a lane,
// lane i with experts [i·per, (i + 1)·per).
//   KT     double, or float where the logits themselves are compared
//   LDSG   groups that do not lie on whole lanes: their scores go through LDS
template <typename T, typename KT, int L, int V, bool LDSG>
RWKV_DEV void route_rows(const Route& p, int per) {
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

  if constexpr (sizeof(KT) == 8) {
    if (!p.bias) {  // (the scores were for the groups)
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (alive >> i & 1) key[i] = (double)load_logit(lg + e0 + i);
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

  write_gates<T, L>(p, lg, row_raw, mine, mine2, live, live2, lmax, total);
}

template <typename T, typename KT, int V, bool LDSG>
__global__ __launch_bounds__(256) void route_wide_kernel(Route p, int per) {
  route_rows<T, KT, 64, V, LDSG>(p, per);
}

// Largest of the 16 lanes of a DPP row, in every one of them.
RWKV_DEV unsigned row_max(unsigned v) {
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));  // row_ror:8
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
  return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
}
template <int L> RWKV_DEV unsigned lanes_max(unsigned v) {
  v = row_max(v);
  if constexpr (L == 64) {
    const unsigned a = max((unsigned)__builtin_amdgcn_readlane((int)v, 0), (unsigned)__builtin_amdgcn_readlane((int)v, 16));
    const unsigned b = max((unsigned)__builtin_amdgcn_readlane((int)v, 32), (unsigned)__builtin_amdgcn_readlane((int)v, 48));
    v = max(a, b);
  }
  return v;
}

// Floats as integers of the same order.  The least finite one is 0x00800000:
// below it, 0 is a key that is gone and 1 an expert that takes no part.
constexpr unsigned kGone = 0, kMasked = 1;
RWKV_DEV unsigned order_of(float v) {
  const unsigned b = __builtin_bit_cast(unsigned, v + 0.f);  // (-0 as 0)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
RWKV_DEV float value_of(unsigned o) {
  return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// A lane's V values at byte `at` of r; what lies past their row's end is any
// number.  All loads are under way before the first value is used.
template <typename T, int V, bool VEC>
RWKV_DEV void load_row(__amdgpu_buffer_rsrc_t r, unsigned at, float (&l)[V]) {
  if constexpr (sizeof(T) == 4) {
    static_assert(V % 4 == 0, "chunks");
    u32x4 c[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i) c[i] = buf_load16(r, at + i * 16);
#pragma unroll
    for (int i = 0; i < V; ++i) l[i] = __builtin_bit_cast(float, (unsigned)c[i / 4][i % 4]);
  } else if constexpr (VEC) {  // pairs
    unsigned c[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) c[i] = buf_load4(r, at + i * 4);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      union { unsigned u; T e[2]; } w;
      w.u = c[i / 2];
      l[i] = to_f(w.e[i % 2]);
    }
  } else {
    unsigned short c[V];
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = buf_load2(r, at + i * 2);
#pragma unroll
    for (int i = 0; i < V; ++i) l[i] = to_f(__builtin_bit_cast(T, c[i]));
  }
}

// The same selection with 32-bit keys.
//   RANK_LOGITS  logits are compared as they are
//   RANK_SUMS    and groups by the sums of two scores
//   RANK_SCORES  scores with a bias
// Scores come from the fp32 exponential, each within kRouteTol · (1 + |bias|)
// of its value.  Where two groups at the border lie closer than both errors
// together, the groups are compared again in 64 bits; where two neighbours of
// the order do, up to 8 more experts are picked and the picked ones ranked in
// 64 bits (about one row in 500 of N(0, 1.5) logits over 256 experts, so that
// every large launch has some: they may not take many times as long).  Only a
// row with more near ties than that is done again whole.
// 16384 fp32 rows of 256, biased, 4 of 8 groups, top 8: 23.7 us (34 with 64-bit
// keys alone); the logits' 16.8 MB would take 3.4, the picks' chains of
// exchanges between lanes are what bounds it.  16 such rows: 6.6 us, latency.
// 8191 rows of 64, top 4 of the logits: 4.8 us.
constexpr float kRouteTol = 0x1p-20f;
enum { RANK_LOGITS = 0, RANK_SUMS = 1, RANK_SCORES = 2 };

// exp(v) to about 2^-23 |v|.
RWKV_DEV float exp_near(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504088896340736f); }
RWKV_DEV float score_near(bool sigmoid, float l, float lmax) {
  if (sigmoid) return __builtin_amdgcn_rcpf(1.f + exp_near(-l));
  const float e = exp_near(l - lmax);
  return l == lmax ? 1.f : e;
}

// A score in 64 bits; total: the softmax's Σ exp(l - lmax).
RWKV_DEV double score_of(bool sigmoid, float l, float lmax, double total) {
  return sigmoid ? 1.0 / (1.0 + exp(-(double)l)) : ex(l, lmax) / total;
}
template <int L, int V>
RWKV_DEV double softmax_total(const float (&l)[V], float lmax) {
  double t = 0.0;
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (l[i] > -kInf) t += ex(l[i], lmax);
#pragma unroll
  for (int d = 1; d < L; d <<= 1) t += __shfl_xor(t, d);
  return t;
}

// How many groups are above this lane's (2^j whole lanes a group), in 64 bits.
template <int L, int V, bool BIAS>
RWKV_DEV int exact_above(const Route& p, const float (&l)[V], const float* bias, const unsigned (&key)[V], float lmax,
                         int sub, int lpg) {
  const int lane = threadIdx.x & 63;
  const double ninf = -(double)kInf, total = p.sigmoid ? 1.0 : softmax_total<L>(l, lmax);
  double a = ninf, b = ninf;
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (key[i] > kMasked) {
      double v = score_of(p.sigmoid, l[i], lmax, total);
      if constexpr (BIAS) v += (double)bias[i];
      b = v > a ? a : (v > b ? v : b);
      a = v > a ? v : a;
    }
  for (int d = 1; d < lpg; d <<= 1) {
    const double oa = __shfl_xor(a, d), ob = __shfl_xor(b, d);
    const double lo = oa > a ? a : oa, hb = ob > b ? ob : b;
    a = oa > a ? oa : a;
    b = lo > hb ? lo : hb;
  }
  const double mine = group_score(a, b, p.top2);
  int above = 0;
  for (int q = 0; q < p.groups; ++q) {
    const double v = __shfl(mine, (lane - sub) + q * lpg);
    above += v > mine || (v == mine && q < sub / lpg);
  }
  return above;
}

template <typename T, int L, int V, bool VEC, int RANK>
__global__ __launch_bounds__(256) void route_kernel(Route p, int per) {
  constexpr bool SCORES = RANK == RANK_SCORES;
  constexpr int RW = 64 / L;
  const int lane = threadIdx.x & 63, sub = lane % L;
  const int row_raw = (blockIdx.x * 4 + (threadIdx.x >> 6)) * RW + lane / L;
  const int row = min(row_raw, p.rows - 1);
  const T* lg = (const T*)p.logits + (size_t)row * p.stride;
  const int e0 = sub * per;
  float l[V];
  // one descriptor for the rows of the wave (run() keeps their span below 2 GB)
  const int row0 = __builtin_amdgcn_readfirstlane(row), rowl = __builtin_amdgcn_readlane(row, 63);
  const __amdgpu_buffer_rsrc_t rl =
      buf_rsrc((const T*)p.logits + (size_t)row0 * p.stride, ((unsigned)(rowl - row0) * (unsigned)p.stride + p.E) * (unsigned)sizeof(T));
  load_row<T, V, VEC>(rl, ((unsigned)(row - row0) * (unsigned)p.stride + e0) * (unsigned)sizeof(T), l);
  float bias[SCORES ? V : 1];
  if constexpr (SCORES) {
    load_row<float, V, true>(buf_rsrc(p.bias, (unsigned)p.E * 4u), (unsigned)e0 * 4u, bias);
  }
  bool in[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    in[i] = (int)(i < per) & (int)(e0 + i < p.E);
    l[i] = (int)in[i] & (int)(l[i] > -kInf) ? l[i] : -kInf;  // (a NaN takes no part)
  }
  float lmax = -kInf;
  double total = 1.0;
  if (!p.sigmoid && (RANK != RANK_LOGITS || !p.renorm)) {
#pragma unroll
    for (int i = 0; i < V; ++i) lmax = fmaxf(lmax, l[i]);
#pragma unroll
    for (int d = 1; d < L; d <<= 1) lmax = fmaxf(lmax, __shfl_xor(lmax, d));
    if (!p.renorm && lmax > -kInf) total = softmax_total<L>(l, lmax);  // the gates' divisor
  }

  unsigned key[V];
  float tol = 2.f * kRouteTol;  // of two scores
  if constexpr (SCORES) {
    float sc[V], inv = 1.f;
    if (p.sigmoid) {
#pragma unroll
      for (int i = 0; i < V; ++i) sc[i] = score_near(true, l[i], lmax);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) sc[i] = score_near(false, l[i], lmax);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) sum += l[i] > -kInf ? sc[i] : 0.f;
#pragma unroll
      for (int d = 1; d < L; d <<= 1) sum += __shfl_xor(sum, d);
      inv = __builtin_amdgcn_rcpf(sum);
    }
    float bm = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      // (bitwise: a branch would wait for every load on its own)
      const bool on = (int)in[i] & (int)(l[i] > -kInf) & (int)(bias[i] > -kInf);
      const unsigned o = order_of(sc[i] * inv + bias[i]);
      key[i] = on ? o : in[i] ? kMasked : kGone;
      bm = fmaxf(bm, on ? fabsf(bias[i]) : 0.f);
    }
#pragma unroll
    for (int d = 1; d < L; d <<= 1) bm = fmaxf(bm, __shfl_xor(bm, d));
    tol = 2.f * kRouteTol * (1.f + bm);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = l[i] > -kInf ? order_of(l[i]) : in[i] ? kMasked : kGone;
  }

  if (p.groups > 1) {  // a group is 2^j whole lanes
    const int S = p.E / p.groups, lpg = S / per, g = sub / lpg;
    unsigned a = kGone, b = kGone;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      b = max(b, min(a, key[i]));
      a = max(a, key[i]);
    }
    for (int d = 1; d < lpg; d <<= 1) {
      const unsigned oa = (unsigned)__shfl_xor((int)a, d), ob = (unsigned)__shfl_xor((int)b, d);
      b = max(max(b, ob), min(a, oa));
      a = max(a, oa);
    }
    int above = 0;
    if constexpr (RANK == RANK_LOGITS) {
      for (int q = 0; q < p.groups; ++q) {
        const unsigned v = (unsigned)__shfl((int)a, (lane - sub) + q * lpg);
        above += v > a || (v == a && q < g);
      }
    } else {
      auto worth = [&](unsigned o) { return SCORES ? value_of(o) : score_near(p.sigmoid, value_of(o), lmax); };
      const float mine = a <= kMasked ? -kInf : p.top2 && b > kMasked ? worth(a) + worth(b) : worth(a);
      int sure = 0, near = 0;  // groups that are above for certain; that may stand either way round
      for (int q = 0; q < p.groups; ++q) {
        const float v = __shfl(mine, (lane - sub) + q * lpg);
        above += v > mine || (v == mine && q < g);
        const bool n = q != g && v > -kInf && fabsf(v - mine) <= 2.f * tol;
        near += n;
        sure += v > mine && !n;
      }
      if (__ballot(near > 0 && sure < p.top_groups && sure + near >= p.top_groups))
        above = exact_above<L, V, SCORES>(p, l, bias, key, lmax, sub, lpg);
    }
    if (above >= p.top_groups) {
#pragma unroll
      for (int i = 0; i < V; ++i) key[i] = kGone;
    }
  }

  // the best of what is left, n of them from slot j0 on
  int mine = 0, mine2 = 0;
  bool live = false, live2 = false, close = false;
  unsigned last = 0xffffffffu;
  auto best_left = [&]() {
    unsigned best = kGone;
#pragma unroll
    for (int i = 0; i < V; ++i) best = max(best, key[i]);
    return best;
  };
  auto pick = [&](int j0, int n) {
    for (int j = j0; j < j0 + n; ++j) {
      const unsigned best = best_left(), m = lanes_max<L>(best);
      if constexpr (SCORES) close |= j > 0 && m > kMasked && value_of(last) - value_of(m) <= tol;
      last = m;
      // the lowest lane of the row that has it, and its lowest expert
      const unsigned long long eq = __ballot(best == m) >> (lane - sub);
      const int win = __builtin_ctzll(L == 64 ? eq : eq & ((1ull << L) - 1));
      int at = 0;
      bool found = sub != win;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const bool hit = (int)!found & (int)(key[i] == m);
        at = hit ? i : at;
        key[i] = hit ? kGone : key[i];
        found |= hit;
      }
      at = __shfl(e0 + at, (lane - sub) + win);
      if (j % L == sub) {
        if (j < L) {
          mine = at;
          live = m > kMasked;
        } else {
          mine2 = at;
          live2 = m > kMasked;
        }
      }
    }
  };
  pick(0, p.k);
  if constexpr (SCORES) {
    const unsigned kth = last, next = lanes_max<L>(best_left());
    close |= next > kMasked && value_of(kth) - value_of(next) <= tol;
    if (__ballot(close)) {
      const int more = min(8, L - p.k);
      if (more < 4) {
        route_rows<T, double, L, V, false>(p, per);
        return;
      }
      pick(p.k, more);  // (where fewer are left, lanes repeat experts that are gone: not live)
      if (__ballot(last > kMasked && value_of(kth) - value_of(last) <= tol)) {
        route_rows<T, double, L, V, false>(p, per);
        return;
      }
      const int n = p.k + more;
      const double sum = p.sigmoid ? 1.0 : softmax_total<L>(l, lmax);
      double v = -(double)kInf;
      if (sub < n && live) v = score_of(p.sigmoid, load_logit(lg + mine), lmax, sum) + (double)p.bias[mine];
      // not live: in the order they were picked, after all others
      int rank = live ? 0 : sub;
      for (int q = 0; q < n; ++q) {
        const double o = __shfl(v, (lane - sub) + q);
        const int oi = __shfl(mine, (lane - sub) + q);
        if (live) rank += o > v || (o == v && oi < mine);
      }
      const int to = (lane - sub + (sub < n ? rank : sub)) * 4;
      mine = __builtin_amdgcn_ds_permute(to, mine);
      live = __builtin_amdgcn_ds_permute(to, (int)live) != 0;
    }
  }
  write_gates<T, L>(p, lg, row_raw, mine, mine2, live, live2, lmax, total);
}

// d_logits from the gates' cotangents.  With u_i = s_i over the selected and
// U = Σ u:  renormalised d s_i = (scale / U)(d_i - Σ_j d_j u_j / U), else
// scale · d_i;  sigmoid d l_i = d s_i · s_i (1 - s_i);  softmax
// d l_e = s_e ([e selected] d s_e - Σ_i d s_i s_i), which is 0 off the selected
// experts where the gates are renormalised.  Half a wave a row, a lane a slot;
// every expert of the row is written.  A slot whose gate is 0 took no part.
// The row is put together in LDS: cleared, the k values added, and stored with
// 4 values a lane.  65536 fp32 rows of 160, 6 selected: 18.6 us, 42 MB of
// gradients at 2.3 TB/s and a cache line for every selected logit.
template <typename T, bool DENSE>
__global__ __launch_bounds__(256) void route_bwd_kernel(Route p, int kpow) {
  // (a softmax's dense gradient is a difference: it stays in 64 bits)
  typedef typename std::conditional<DENSE, double, float>::type A;
  typedef A avec __attribute__((ext_vector_type(4)));
  extern __shared__ __attribute__((aligned(32))) unsigned char rows_lds[];
  const int lane = threadIdx.x & 31;
  const int row_raw = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int row = min(row_raw, p.rows - 1);
  const T* lg = (const T*)p.logits + (size_t)row * p.stride;
  const int E4 = (p.E + 3) / 4 * 4;
  A* acc = (A*)rows_lds + (threadIdx.x >> 5) * E4;
  // over the lanes that hold slots
  auto sum = [&](double v) {
    for (int d = 1; d < kpow; d <<= 1) v += __shfl_xor(v, d);
    return v;
  };
  auto sum_all = [&](double v) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) v += __shfl_xor(v, d);
    return v;
  };
  int e = -1;
  float l = -kInf;
  double dg = 0.0;
  if (lane < p.k) {
    e = p.inds_in[(size_t)row * p.k + lane];
    const float g = p.gates_in[(size_t)row * p.k + lane], d = p.d_gates[(size_t)row * p.k + lane];
    if (e >= 0 && e < p.E && g != 0.f) {
      l = load_logit(lg + e);
      dg = (double)d;
    } else {
      e = -1;  // (an id that no expert has is dropped)
    }
  }
  for (int i = lane * 4; i < E4; i += 128) *(avec*)(acc + i) = avec{0, 0, 0, 0};
  const bool on = e >= 0 && l > -kInf;
  float m = l;
  if constexpr (DENSE)
    for (int i = lane; i < p.E; i += 32) m = fmaxf(m, load_logit(lg + i));
  if (!p.sigmoid)
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  double total = 1.0, s = 0.0, rest = 0.0;
  if (p.sigmoid) {
    if (on) {  // s and 1 - s
      const double t = exp(-fabs((double)l)), q = 1.0 / (1.0 + t);
      s = l >= 0.f ? q : t * q;
      rest = l >= 0.f ? t * q : q;
    }
  } else {
    if constexpr (DENSE) {
      total = 0.0;
      for (int i = lane; i < p.E; i += 32) {
        const float v = load_logit(lg + i);
        if (v > -kInf) total += ex(v, m);
      }
      total = sum_all(total);
    }
    if (on) s = ex(l, m) / total;
  }
  double ds = dg * (double)p.scale;
  if (p.renorm) {
    const double U = sum(s);
    const double mean = sum(ds * s);
    ds = U > 0.0 ? (ds - mean / U) / U : 0.0;
  }
  double dl = on ? ds * s : 0.0, back = 0.0;
  if (p.sigmoid) dl *= rest;
  if constexpr (DENSE) back = sum_all(dl);
  __syncthreads();
  if (on) atomicAdd(acc + e, (A)dl);  // (the forward's experts are distinct)
  __syncthreads();
  if (row_raw >= p.rows) return;
  T* out = (T*)p.d_logits + (size_t)row * p.E;
  for (int i0 = lane * 4; i0 < p.E; i0 += 128) {
    avec v = *(const avec*)(acc + i0);
    if constexpr (DENSE) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (i0 + q < p.E) {
          const float x = load_logit(lg + i0 + q);
          if (x > -kInf) v[q] -= back * (ex(x, m) / total);
        }
    }
    if (p.E % 4 == 0) {
      union { T e[4]; unsigned u[sizeof(T)]; } w;
#pragma unroll
      for (int q = 0; q < 4; ++q) w.e[q] = from_f<T>((float)v[q]);
      typedef unsigned uvec __attribute__((ext_vector_type(sizeof(T))));
      uvec o;
#pragma unroll
      for (int q = 0; q < (int)sizeof(T); ++q) o[q] = w.u[q];
      *(uvec*)(out + i0) = o;
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (i0 + q < p.E) out[i0 + q] = from_f<T>((float)v[q]);
    }
  }
}

template <typename T, int L, int V, int RANK>
hipError_t run(const Route& p, int per, hipStream_t s) {
  constexpr int RPB = 256 / L;
  const dim3 grid((p.rows + RPB - 1) / RPB), block(256);
  // 16-bit logits are read in pairs where every lane's first is on 4 bytes
  const bool vec = sizeof(T) == 4 || (per % 2 == 0 && p.stride % 2 == 0 && (uintptr_t)p.logits % 4 == 0);
  if (vec) launch_kernel(route_kernel<T, L, V, true, RANK>, grid, block, 0, s, p, per);
  else if constexpr (sizeof(T) == 2) launch_kernel(route_kernel<T, L, V, false, RANK>, grid, block, 0, s, p, per);
  return hipGetLastError();
}

inline bool on_lanes(const Route& p, int L, int per) {
  if (p.groups == 1) return true;
  const int S = p.E / p.groups;
  if (S % per) return false;
  const int lpg = S / per;
  return (lpg & (lpg - 1)) == 0 && lpg * p.groups <= L;
}

template <typename T, int RANK>
hipError_t run_key(const Route& p, hipStream_t s) {
  typedef typename std::conditional<RANK != RANK_LOGITS, double, float>::type KT;
  const int per64 = (p.E + 63) / 64, per16 = (p.E + 15) / 16;
  // 16 lanes a row take four rows a wave through the reductions at once; with
  // too few rows to fill the card 64 lanes have less to do each
  const bool many = p.rows >= 4096 && per16 <= 16 && p.stride < (1 << 27);
  if (many && on_lanes(p, 16, per16)) {
    if (per16 <= 4) return run<T, 16, 4, RANK>(p, per16, s);
    if (per16 <= 8) return run<T, 16, 8, RANK>(p, per16, s);
    if (per16 <= 12) return run<T, 16, 12, RANK>(p, per16, s);
    return run<T, 16, 16, RANK>(p, per16, s);
  }
  if (on_lanes(p, 64, per64))
    return per64 <= 4 ? run<T, 64, 4, RANK>(p, per64, s) : run<T, 64, 8, RANK>(p, per64, s);
  const dim3 grid((p.rows + 3) / 4), block(256);
  if (per64 <= 4) launch_kernel(route_wide_kernel<T, KT, 4, true>, grid, block, 0, s, p, per64);
  else launch_kernel(route_wide_kernel<T, KT, 8, true>, grid, block, 0, s, p, per64);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_route(const Route& p, hipStream_t s) {
  hipError_t e = hipErrorInvalidValue;
  RWKV_DISPATCH_DTYPE(p.dtype, T, {
    e = p.bias ? run_key<T, RANK_SCORES>(p, s)
               : p.groups > 1 && p.top2 ? run_key<T, RANK_SUMS>(p, s) : run_key<T, RANK_LOGITS>(p, s);
  });
  return mark(e, "route", s);
}

hipError_t launch_route_backward(const Route& p, hipStream_t s) {
  int kpow = 1;
  while (kpow < p.k) kpow *= 2;
  RWKV_DISPATCH_DTYPE(p.dtype, T, {
    const bool dense = !p.sigmoid && !p.renorm;
    const unsigned lds = 8u * ((p.E + 3) / 4 * 4) * (dense ? sizeof(double) : sizeof(float));
    launch_kernel(dense ? route_bwd_kernel<T, true> : route_bwd_kernel<T, false>,
                  dim3((p.rows + 7) / 8), dim3(256), lds, s, p, kpow);
  });
  return mark(hipGetLastError(), "route_bwd", s);
}

}  // namespace rwkvmoe
