// Routing of tokens to experts with a balance bias and groups, from given logits [T, E], and its
// gradient.  For a token with logits l:
//   s = sigmoid(l) or softmax(l);  c = s + b   (b: the experts' balance bias, may be null)
//   experts lie in G groups of E / G side by side; a group's score is the sum of its two largest
//   c, without a bias too (routing that ranks groups by their best expert alone is another rule);
//   only experts of the best `keep` groups are eligible
//   ids = the k eligible experts with the largest c, in that order; ties to the lower index
//   w = scale * s[ids] (/ (sum of s[ids] + 1e-20))
// A NaN c ranks below every other value; a row of softmax without a value above -inf has s = 0.
//
// Which of two experts is ahead is decided in 64 bits: the differences between neighbouring
// scores of a few hundred experts are small enough for the order to depend on fp32 rounding in
// about one token of a thousand.  fp64 arithmetic runs at fp32's rate here (not counting packed
// forms), and the bytes, 2 to 4 per logit, are what the kernels wait for.
//
// L lanes share a token (16 where the token fits and there are many tokens, else 64), expert
// l + L * slot to lane l.  Bound by latency: 32 tokens of 256 experts, 8 of them, 9-10 us, 4096
// of 128 10-11 and the gradient 5.6.
#include <type_traits>

#include "mm_common.h"
#include "mm_mx.h"
#include "mmfp4.h"

namespace {

constexpr int NT = 256;
constexpr int MAX_E = 1024, MAX_K = 64, MAX_G = 64;
constexpr double EPS = 1e-20;

// Joins over groups of lanes, step D: a value of the other half of the lane's 2 D, for operands that
// all D lanes of a half hold alike, as they do where a join goes D = 1, 2, 4, ..  Moves between
// registers, mirrored where that is what there is: a selection of 8 among 256 waits for 48 such
// steps (the call of 32 tokens 10.3 us, through LDS 10.8).
template <int D>
MM_DEV uint32_t other(uint32_t v) {
  static_assert(D == 1 || D == 2 || D == 4 || D == 8 || D == 16 || D == 32, "steps of a wave");
  if constexpr (D == 1) return __builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 15, 15, true);
  else if constexpr (D == 2) return __builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 15, 15, true);
  else if constexpr (D == 4) return __builtin_amdgcn_update_dpp(0, (int)v, 0x141, 15, 15, true);
  else if constexpr (D == 8) return __builtin_amdgcn_update_dpp(0, (int)v, 0x140, 15, 15, true);
  else if constexpr (D == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return threadIdx.x & 16 ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & 32 ? r[0] : r[1];
  }
}
template <int D>
MM_DEV float other(float v) {
  return __builtin_bit_cast(float, other<D>(__builtin_bit_cast(uint32_t, v)));
}
template <int D>
MM_DEV double other(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)other<D>((uint32_t)(u >> 32)) << 32 |
                                        other<D>((uint32_t)u));
}
// f(D) for D = 1, 2, 4, .. below L.
template <int L, int D = 1, class F>
MM_DEV void steps(F&& f) {
  if constexpr (D < L) {
    f(std::integral_constant<int, D>{});
    steps<L, 2 * D>(f);
  }
}

template <int L>
MM_DEV double all_sum(double v) {
  steps<L>([&](auto d) { v += other<decltype(d)::value>(v); });
  return v;
}
template <int L>
MM_DEV float all_max(float v) {   // the largest, a NaN if there is one
  steps<L>([&](auto d) {
    const float o = other<decltype(d)::value>(v);
    v = (o > v || o != o) ? o : v;
  });
  return v;
}

// The lane's logits, -inf past E.  All loads leave before one is waited for: one type for all, and
// the last expert's again past E.
template <int L, int SL>
MM_DEV void load_logits(const void* p, int type, size_t base, int E, float (&x)[SL]) {
  const int l = threadIdx.x % L;
  if (type == mmmx::F32) {
#pragma unroll
    for (int i = 0; i < SL; ++i) x[i] = ((const float*)p)[base + min(l + L * i, E - 1)];
  } else {
    uint16_t v[SL];
#pragma unroll
    for (int i = 0; i < SL; ++i) v[i] = ((const uint16_t*)p)[base + min(l + L * i, E - 1)];
#pragma unroll
    for (int i = 0; i < SL; ++i)
      x[i] = type == mmmx::F16 ? (float)__builtin_bit_cast(f16, v[i])
                               : __builtin_bit_cast(float, (uint32_t)v[i] << 16);
  }
#pragma unroll
  for (int i = 0; i < SL; ++i)
    if (l + L * i >= E) x[i] = -__builtin_inff();
}

// s of the lane's experts; lanes past E get 0.
template <int L, int SL>
MM_DEV void scores(const void* logits, int type, size_t base, int E, bool softmax, double (&s)[SL]) {
  const int l = threadIdx.x % L;
  float x[SL];
  load_logits<L, SL>(logits, type, base, E, x);
  if (!softmax) {
#pragma unroll
    for (int i = 0; i < SL; ++i) s[i] = 1.0 / (1.0 + exp(-(double)x[i]));
    return;
  }
  float m = x[0];
#pragma unroll
  for (int i = 1; i < SL; ++i) m = (x[i] > m || x[i] != x[i]) ? x[i] : m;
  m = all_max<L>(m);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < SL; ++i) {
    s[i] = l + L * i < E ? exp((double)x[i] - (double)m) : 0.0;
    sum += s[i];
  }
  sum = all_sum<L>(sum);
  const double r = m == -__builtin_inff() ? 0.0 : 1.0 / sum;
#pragma unroll
  for (int i = 0; i < SL; ++i) s[i] = r == 0.0 ? 0.0 : s[i] * r;
}

MM_DEV double not_nan(double v) { return v == v ? v : -__builtin_inf(); }

struct Route {
  const void* logits;
  const float* bias;
  int64_t* ids;
  float* w;
  float scale;
  int type, T, E, k, softmax, groups, keep, renorm;
};

template <int L, int SL>
__global__ void __launch_bounds__(NT) k_moe_route(Route a) {
  extern __shared__ double lds[];                    // [tokens of the block][2][E]: s and c
  constexpr int TOK = NT / L;
  const int l = threadIdx.x % L, mine = threadIdx.x / L;
  const int E = a.E, k = a.k;
  const int t = min((int)blockIdx.x * TOK + mine, a.T - 1);   // surplus lanes repeat the last
  double* const ls = lds + (size_t)mine * 2 * E;
  double* const lc = ls + E;
  double s[SL], c[SL];
  float b[SL];
#pragma unroll
  for (int i = 0; i < SL; ++i) b[i] = 0.0f;
  if (a.bias)
#pragma unroll
    for (int i = 0; i < SL; ++i) b[i] = a.bias[min(l + L * i, E - 1)];
  scores<L, SL>(a.logits, a.type, (size_t)t * E, E, a.softmax, s);
  uint32_t out = 0;                                  // slots that cannot be taken (any more)
#pragma unroll
  for (int i = 0; i < SL; ++i) {
    const int e = l + L * i;
    if (e < E) {
      c[i] = not_nan(s[i] + (double)b[i]);
      ls[e] = s[i];
      lc[e] = c[i];
    } else {
      c[i] = -__builtin_inf();
      out |= 1u << i;
    }
  }
  __syncthreads();
  if (a.groups > 1) {
    // P lanes per group, G * P <= L; each looks at every P-th of the group's experts
    const int G = a.groups, n = E / G;
    int gp = 1;
    while (gp < G) gp <<= 1;
    const int P = L / gp, g = l / P;
    double b1 = -__builtin_inf(), b2 = b1;
    for (int j = l % P; g < G && j < n; j += P) {
      const double v = lc[g * n + j];
      b2 = v > b1 ? b1 : (v > b2 ? v : b2);
      b1 = v > b1 ? v : b1;
    }
    steps<L>([&](auto d) {
      constexpr int D = decltype(d)::value;
      if (D >= P) return;
      const double o1 = other<D>(b1), o2 = other<D>(b2);
      b2 = o1 > b1 ? (b1 > o2 ? b1 : o2) : (o1 > b2 ? o1 : b2);
      b1 = o1 > b1 ? o1 : b1;
    });
    const double best = not_nan(n == 1 ? b1 : b1 + b2);
    int ahead = 0;
    for (int j = 0; j < G; ++j) {
      const double o = __shfl(best, j * P, L);
      ahead += o > best || (o == best && j < g);
    }
    const uint64_t kept = __ballot(g < G && ahead < a.keep) >> (threadIdx.x % 64 / L * L);
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const int e = l + L * i;
      if (e < E && !((kept >> (e / n * P)) & 1)) out |= 1u << i;
    }
  }
  double total = 0.0;
  double my_s = 0.0;                                 // round r is kept by lane r % L
  int my_id = 0;
  const bool write = blockIdx.x * TOK + mine < a.T;
  for (int r = 0; r < k; ++r) {
    double bv = -__builtin_inf();
    int bi = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < SL; ++i)                     // slots ascend in e: ties keep the lower
      if (!((out >> i) & 1) && (c[i] > bv || bi == 0x7fffffff)) {
        bv = c[i];
        bi = l + L * i;
      }
    steps<L>([&](auto d) {
      constexpr int D = decltype(d)::value;
      const double ov = other<D>(bv);
      const int oi = (int)other<D>((uint32_t)bi);
      const bool take = oi != 0x7fffffff && (bi == 0x7fffffff || ov > bv || (ov == bv && oi < bi));
      bv = take ? ov : bv;
      bi = take ? oi : bi;
    });
    if (bi % L == l) out |= 1u << (bi / L);
    const double v = ls[bi];
    total += v;
    if (r % L == l) {
      my_s = v;
      my_id = bi;
    }
    // a full round of lanes, or the end: ids out; weights wait for the sum unless there is none
    if ((r % L == L - 1 || r == k - 1) && write) {
      const int at = r / L * L + l;
      if (at <= r) {
        a.ids[(size_t)t * k + at] = my_id;
        if (!a.renorm) a.w[(size_t)t * k + at] = (float)((double)a.scale * my_s);
      }
    }
  }
  if (a.renorm && write)
    for (int j = l; j < k; j += L) {
      // one round of lanes: still held; more: read back what this lane wrote
      const double v = k <= L ? my_s : ls[a.ids[(size_t)t * k + j]];
      a.w[(size_t)t * k + j] = (float)((double)a.scale * (v / (total + EPS)));
    }
}

struct RouteGrad {
  const float* dw;
  const void* logits;
  const int64_t* ids;
  void* dl;
  float scale;
  int type, T, E, k, softmax, renorm;
};

// dl = J^T dw.  With u = dw * scale, and under renormalisation S = sum of s[ids] + 1e-20 and
// u <- (u - (u . s[ids]) / S) / S; v = u scattered to the experts (an index that comes twice
// gets both):
//   sigmoid  dl = v s (1 - s);   softmax  dl = s (v - (v . s))
// Ids outside [0, E) have s = 0 and get nothing.
template <int L, int SL>
__global__ void __launch_bounds__(NT) k_moe_route_grad(RouteGrad a) {
  extern __shared__ double lds[];                    // [tokens of the block][2][E]: s and v
  constexpr int TOK = NT / L;
  const int l = threadIdx.x % L, mine = threadIdx.x / L;
  const int E = a.E, k = a.k;
  const int t = min((int)blockIdx.x * TOK + mine, a.T - 1);
  double* const ls = lds + (size_t)mine * 2 * E;
  double* const lv = ls + E;
  double s[SL];
  scores<L, SL>(a.logits, a.type, (size_t)t * E, E, a.softmax, s);
#pragma unroll
  for (int i = 0; i < SL; ++i) {
    const int e = l + L * i;
    if (e < E) {
      ls[e] = s[i];
      lv[e] = 0.0;
    }
  }
  __syncthreads();
  double sum = EPS, us = 0.0;                        // S and u . s[ids]
  if (a.renorm) {
    double p = 0.0, q = 0.0;
    for (int j = l; j < k; j += L) {
      const int64_t id = a.ids[(size_t)t * k + j];
      const double sj = id >= 0 && id < E ? ls[id] : 0.0;
      p += sj;
      q += sj * ((double)a.dw[(size_t)t * k + j] * (double)a.scale);
    }
    sum += all_sum<L>(p);
    us = all_sum<L>(q);
  }
  double vs = 0.0;                                   // v . s
  for (int j0 = 0; j0 < k; j0 += L) {
    const int j = j0 + l;
    const int64_t id = j < k ? a.ids[(size_t)t * k + j] : -1;
    const bool live = id >= 0 && id < E;
    const int which = live ? (int)id : -1;
    double u = j < k ? (double)a.dw[(size_t)t * k + j] * (double)a.scale : 0.0;
    if (a.renorm) u = (u - us / sum) / sum;
    // the first lane of those with one index adds them up, in order
    double mine_all = 0.0;
    bool first = live;
    for (int o = 0; o < min(L, k - j0); ++o) {
      const double ou = __shfl(u, o, L);
      if (__shfl(which, o, L) == which) {
        mine_all += ou;
        first = first && o >= l;
      }
    }
    if (first) {
      lv[id] += mine_all;
      vs += mine_all * ls[id];
    }
  }
  __syncthreads();
  vs = all_sum<L>(vs);
  if (blockIdx.x * TOK + mine >= a.T) return;
#pragma unroll
  for (int i = 0; i < SL; ++i) {
    const int e = l + L * i;
    if (e < E) {
      const double d = a.softmax ? s[i] * (lv[e] - vs) : lv[e] * (s[i] * (1.0 - s[i]));
      mmmx::store1(a.dl, a.type, (size_t)t * E + e, (float)d);
    }
  }
}

// Lanes per token and slots per lane.
struct Shape {
  int L, SL;
};
Shape shape_of(int T, int E, int groups) {
  if (E <= 256 && groups <= 16 && T >= 2048)
    return {16, E <= 64 ? 4 : (E <= 128 ? 8 : 16)};
  return {64, E <= 64 ? 1 : (E <= 128 ? 2 : (E <= 256 ? 4 : (E <= 512 ? 8 : 16)))};
}

#define MM_ROUTE(KERNEL, ARGS)                                                                  \
  do {                                                                                          \
    const Shape sh = shape_of(T, E, groups);                                                    \
    const int tok = NT / sh.L;                                                                  \
    const size_t blocks = ((size_t)T + tok - 1) / tok;                                          \
    MM_CHECK_ARG(mmmx::launch_holds(blocks, NT), "routing: %d tokens are too many", T);         \
    const dim3 grid((unsigned)blocks);                                                          \
    const size_t bytes = (size_t)tok * 2 * E * sizeof(double);                                  \
    const hipStream_t st = (hipStream_t)stream;                                                 \
    if (sh.L == 16) {                                                                           \
      if (sh.SL == 4) hipLaunchKernelGGL((KERNEL<16, 4>), grid, dim3(NT), bytes, st, ARGS);       \
      else if (sh.SL == 8) hipLaunchKernelGGL((KERNEL<16, 8>), grid, dim3(NT), bytes, st, ARGS);  \
      else hipLaunchKernelGGL((KERNEL<16, 16>), grid, dim3(NT), bytes, st, ARGS);                 \
    } else {                                                                                    \
      if (sh.SL == 1) hipLaunchKernelGGL((KERNEL<64, 1>), grid, dim3(NT), bytes, st, ARGS);       \
      else if (sh.SL == 2) hipLaunchKernelGGL((KERNEL<64, 2>), grid, dim3(NT), bytes, st, ARGS);  \
      else if (sh.SL == 4) hipLaunchKernelGGL((KERNEL<64, 4>), grid, dim3(NT), bytes, st, ARGS);  \
      else if (sh.SL == 8) hipLaunchKernelGGL((KERNEL<64, 8>), grid, dim3(NT), bytes, st, ARGS);  \
      else hipLaunchKernelGGL((KERNEL<64, 16>), grid, dim3(NT), bytes, st, ARGS);                 \
    }                                                                                           \
  } while (0)

}  // namespace

extern "C" int mm_moe_route(const void* logits, int type, const float* bias, int T, int E, int k,
                            int softmax, int groups, int keep, int renorm, float scale,
                            int64_t* ids, float* weights, void* stream) {
  MM_CHECK_ARG(T >= 0 && E > 0 && E <= MAX_E, "mm_moe_route: T=%d, E=%d: at most %d experts", T, E,
               MAX_E);
  MM_CHECK_ARG(groups > 0 && groups <= MAX_G && E % groups == 0,
               "mm_moe_route: groups=%d must divide E=%d and be at most %d", groups, E, MAX_G);
  MM_CHECK_ARG(keep > 0 && keep <= groups, "mm_moe_route: topk_groups=%d of %d groups", keep,
               groups);
  MM_CHECK_ARG(k > 0 && k <= MAX_K && k <= E / groups * keep,
               "mm_moe_route: k=%d must be at most %d and the %d experts of the groups kept", k,
               MAX_K, E / groups * keep);
  MM_CHECK_ARG(type >= 0 && type <= 2, "mm_moe_route: unknown type %d", type);
  if (T == 0) return 0;
  MM_CHECK_ARG(logits && ids && weights, "mm_moe_route: null argument");
  const Route a{logits, bias, ids, weights, scale, type, T, E, k, softmax, groups, keep, renorm};
  MM_ROUTE(k_moe_route, a);
  MM_CHECK_LAUNCH("mm_moe_route");
  return 0;
}

extern "C" int mm_moe_route_backward(const float* dw, const void* logits, int type,
                                     const int64_t* ids, int T, int E, int k, int softmax,
                                     int renorm, float scale, void* dlogits, void* stream) {
  MM_CHECK_ARG(T >= 0 && E > 0 && E <= MAX_E,
               "mm_moe_route_backward: T=%d, E=%d: at most %d experts", T, E, MAX_E);
  MM_CHECK_ARG(k > 0 && k <= MAX_K, "mm_moe_route_backward: k=%d must be 1..%d", k, MAX_K);
  MM_CHECK_ARG(type >= 0 && type <= 2, "mm_moe_route_backward: unknown type %d", type);
  if (T == 0) return 0;
  MM_CHECK_ARG(dw && logits && ids && dlogits, "mm_moe_route_backward: null argument");
  const int groups = 1;
  const RouteGrad a{dw, logits, ids, dlogits, scale, type, T, E, k, softmax, renorm};
  MM_ROUTE(k_moe_route_grad, a);
  MM_CHECK_LAUNCH("mm_moe_route_backward");
  return 0;
}
