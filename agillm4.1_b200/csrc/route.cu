// General expert routing: softmax or sigmoid scores of router logits, a
// selection bias, groups of experts, top-k, renormalised and scaled weights,
// and the gradient of the weights with respect to the logits.
//
//   s = softmax(l) or sigmoid(l);   key c = l without a bias, s + b with one
//   group score = sum of the group's two largest s (c with a bias)
//   idx = the k largest c within the top groups, ties to the lowest index
//   w_r = scale * s[idx_r]  (/ sum_j s[idx_j] when renormalised)
//
// An expert whose key is -inf or NaN is never chosen: its slot gets index -1
// and weight 0. A NaN logit (or +inf under softmax) makes the row's weights
// NaN.
//
// The order of the keys is decided in real arithmetic: without a bias a key is
// the logit itself, exact. Otherwise the keys are computed in fp32 (error
// below 2^-20 (1 + |c|)); where two neighbours of the sorted top k + 1, or
// the last kept and first dropped group, are closer than that allows, the
// token is selected again with fp64 scores. So the indices do not depend on
// how an exponential is rounded. Equal logits with equal biases are equal
// keys and need no second look.
//
// Mapping: L lanes hold a token's E logits in registers, V each (lane i holds
// experts i, i + L, ...). Few experts take few lanes, so a warp routes 8
// tokens of a 16-expert block; grouped routing takes the whole warp.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace agm {

namespace {

constexpr int kRouteThreads = 256;
constexpr float kNegInf = -INFINITY;

template <typename F>
__device__ __forceinline__ F exp_of(F v) {
  if constexpr (std::is_same<F, double>::value)
    return exp(v);
  else
    return expf(v);
}

template <typename F, int L>
__device__ __forceinline__ F lanes_max(F v) {
#pragma unroll
  for (int o = L / 2; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <typename F, int L>
__device__ __forceinline__ F lanes_sum(F v) {
#pragma unroll
  for (int o = L / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Largest (v, then lowest id) over the L lanes; every lane gets the winner.
template <typename F, int L>
__device__ __forceinline__ void lanes_best(F& v, int& id) {
  if constexpr (L == 32 && std::is_same<F, float>::value) {
    const uint32_t b = __float_as_uint(v);
    const uint32_t u = (b & 0x80000000u) ? ~b : (b | 0x80000000u);  // order of the floats
    const uint32_t m = __reduce_max_sync(0xffffffffu, u);
    id = __reduce_min_sync(0xffffffffu, u == m ? id : INT32_MAX);
    v = __uint_as_float((m & 0x80000000u) ? (m ^ 0x80000000u) : ~m);
  } else {
#pragma unroll
    for (int o = L / 2; o; o >>= 1) {
      const F ov = __shfl_xor_sync(0xffffffffu, v, o);
      const int oi = __shfl_xor_sync(0xffffffffu, id, o);
      if (ov > v || (ov == v && oi < id)) {
        v = ov;
        id = oi;
      }
    }
  }
}

// Selects one token's experts; slot r = sub + L * i of lane `sub` gets sel[i].
// Returns whether the fp32 keys leave the choice open.
template <typename F, int L, int V, int KS>
__device__ __forceinline__ bool select_experts(const float (&l)[V], const RouteArgs& a, int sub, int (&sel)[KS]) {
  constexpr bool kFast = std::is_same<F, float>::value;
  const bool grouped = a.top_groups < a.n_groups;
  F key[V];
  bool near = false;
  if (!a.bias && !grouped) {
#pragma unroll
    for (int j = 0; j < V; ++j) key[j] = static_cast<F>(l[j]);
  } else {
    F s[V];
    if (a.score == AGM_ROUTE_SIGMOID) {
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] = F(1) / (F(1) + exp_of(-static_cast<F>(l[j])));
    } else {
      float m = kNegInf;
#pragma unroll
      for (int j = 0; j < V; ++j) m = fmaxf(m, l[j]);
      m = lanes_max<float, L>(m);
      F t = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s[j] = l[j] > kNegInf ? exp_of(static_cast<F>(l[j]) - static_cast<F>(m)) : F(0);
        t += s[j];
      }
      t = lanes_sum<F, L>(t);
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] = s[j] / t;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = sub + L * j;
      key[j] = a.bias ? (e < a.n_experts ? s[j] + static_cast<F>(a.bias[e]) : F(kNegInf)) : static_cast<F>(l[j]);
      if (!(l[j] > kNegInf)) key[j] = F(kNegInf);
    }
    if (grouped) {
      if constexpr (L == 32) {
        const int size = a.n_experts / a.n_groups;
        int grp[V];
#pragma unroll
        for (int j = 0; j < V; ++j) grp[j] = (sub + L * j) / size;
        F mine = F(kNegInf);  // lane g: score of group g
        for (int g = 0; g < a.n_groups; ++g) {
          F t1 = F(kNegInf), t2 = F(kNegInf);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            F v = a.bias ? key[j] : s[j];
            if (grp[j] != g || !(key[j] > F(kNegInf))) v = F(kNegInf);
            t2 = max(t2, min(t1, v));
            t1 = max(t1, v);
          }
#pragma unroll
          for (int o = 16; o; o >>= 1) {
            const F o1 = __shfl_xor_sync(0xffffffffu, t1, o), o2 = __shfl_xor_sync(0xffffffffu, t2, o);
            t2 = max(min(t1, o1), max(t2, o2));
            t1 = max(t1, o1);
          }
          if (sub == g) mine = t2 > F(kNegInf) ? t1 + t2 : t1;
        }
        uint32_t kept = 0;
        F last = 0;
        for (int i = 0; i <= a.top_groups; ++i) {
          F v = ((kept >> sub) & 1u) ? F(kNegInf) : mine + F(0);
          int id = sub;
          lanes_best<F, 32>(v, id);
          if (!(v > F(kNegInf))) break;
          if (i == a.top_groups) {
            near = kFast && last - v <= F(3.8e-6f) * (F(1) + fabs(v));  // 2^-18
            break;
          }
          kept |= 1u << id;
          last = v;
        }
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (!((kept >> (grp[j] & 31)) & 1u)) key[j] = F(kNegInf);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) key[j] = key[j] > F(kNegInf) ? key[j] + F(0) : F(kNegInf);  // NaN: never chosen; -0 = 0
#pragma unroll
  for (int i = 0; i < KS; ++i) sel[i] = -1;
  const bool inexact = kFast && a.bias != nullptr;
  uint32_t used = 0;
  F prev = F(INFINITY);
  float prev_l = 0.f, prev_b = 0.f;
  const int picks = a.k + (inexact ? 1 : 0);
  for (int r = 0; r < picks; ++r) {
    F v = F(kNegInf);
    int id = INT32_MAX;
    float vl = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (!((used >> j) & 1u) && key[j] > v) {
        v = key[j];
        id = sub + L * j;
        if (inexact) vl = l[j];
      }
    const int own = id;
    lanes_best<F, L>(v, id);
    const bool any = v > F(kNegInf);
    if (inexact) {
      const int src = (threadIdx.x & 31 & ~(L - 1)) | (id & (L - 1));
      vl = __shfl_sync(0xffffffffu, vl, any ? src : 0);
      const float vb = any ? a.bias[id] : 0.f;
      if (any && r > 0 && prev - v <= F(1.9e-6f) * (F(1) + fabs(v)) && !(vl == prev_l && vb == prev_b)) near = true;
      prev = v;
      prev_l = vl;
      prev_b = vb;
    }
    if (any && own == id) used |= 1u << (id / L);
    if (r < a.k && any) {
#pragma unroll
      for (int i = 0; i < KS; ++i)
        if (r == sub + L * i) sel[i] = id;
    }
  }
  return near;
}

template <typename T, int L, int V>
__global__ void __launch_bounds__(kRouteThreads)
    route_kernel(const T* __restrict__ logits, RouteArgs a, int32_t* __restrict__ idx, float* __restrict__ weights) {
  constexpr int KS = L == 32 ? 1 : AGM_ROUTE_MAX_TOPK / 8;  // L = 4 serves at most 16 experts
  constexpr int TOK = 32 / L;
  pdl_wait();
  pdl_trigger();
  const int lane = lane_id(), sub = lane & (L - 1);
  const int64_t step = static_cast<int64_t>(gridDim.x) * (blockDim.x / 32) * TOK;
  for (int64_t t0 = (static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + warp_id()) * TOK; t0 < a.n; t0 += step) {
    const int64_t t = t0 + lane / L;
    const bool live = t < a.n;
    const T* row = logits + (live ? t : t0) * a.n_experts;
    float l[V];
    bool bad = false;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = sub + L * j;
      l[j] = e < a.n_experts ? Traits<T>::to_f(row[e]) : kNegInf;
      bad |= l[j] != l[j] || (a.score == AGM_ROUTE_SOFTMAX && l[j] == INFINITY);
    }
#pragma unroll
    for (int o = L / 2; o; o >>= 1) bad |= __shfl_xor_sync(0xffffffffu, static_cast<int>(bad), o) != 0;
    int sel[KS];
    const bool near = select_experts<float, L, V, KS>(l, a, sub, sel);
    if (__any_sync(0xffffffffu, near)) {
      int again[KS];
      select_experts<double, L, V, KS>(l, a, sub, again);
#pragma unroll
      for (int i = 0; i < KS; ++i) sel[i] = near ? again[i] : sel[i];
    }
    // Weights of the chosen experts, from their logits. Renormalised weights
    // are ratios: the factor exp(m) common to all scores is left out, so that
    // they do not underflow where every chosen score does.
    float p[KS], total = 0.f;
    if (!a.renormalize && a.score == AGM_ROUTE_SOFTMAX) {
      float m = kNegInf;
#pragma unroll
      for (int j = 0; j < V; ++j) m = fmaxf(m, l[j]);
      m = lanes_max<float, L>(m);
#pragma unroll
      for (int j = 0; j < V; ++j) total += l[j] > kNegInf ? expf(l[j] - m) : 0.f;
      total = lanes_sum<float, L>(total);
#pragma unroll
      for (int i = 0; i < KS; ++i) p[i] = sel[i] >= 0 ? expf(Traits<T>::to_f(row[sel[i]]) - m) : 0.f;
    } else {
      float c[KS], m = kNegInf;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        c[i] = sel[i] >= 0 ? Traits<T>::to_f(row[sel[i]]) : kNegInf;
        m = fmaxf(m, a.score == AGM_ROUTE_SIGMOID ? fminf(c[i], 0.f) : c[i]);
      }
      m = lanes_max<float, L>(m);
      if (!a.renormalize) m = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        if (a.score == AGM_ROUTE_SIGMOID)
          p[i] = c[i] > kNegInf ? expf(fminf(c[i], 0.f) - m) / (1.f + expf(-fabsf(c[i]))) : 0.f;
        else
          p[i] = c[i] > kNegInf ? expf(c[i] - m) : 0.f;
        total += p[i];
      }
      total = a.renormalize ? lanes_sum<float, L>(total) : 1.f;
    }
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const int r = sub + L * i;
      if (live && r < a.k) {
        idx[t * a.k + r] = sel[i];
        weights[t * a.k + r] = bad ? NAN : (sel[i] >= 0 ? a.scale * (p[i] / total) : 0.f);
      }
    }
  }
}

// d l from d w. With s the scores and w' the renormalised weights:
//   softmax, renormalised   dl_r = scale w'_r (dw_r - sum_j dw_j w'_j)
//   sigmoid, renormalised   dl_r = scale w'_r (1 - s_r) (dw_r - sum_j dw_j w'_j)
//   sigmoid                 dl_r = scale dw_r s_r (1 - s_r)
//   softmax                 dl_e = s_e (scale dw_e - scale sum_j dw_j s_j), every e
// All but the last are zero outside the chosen experts. An index outside
// [0, E) is an empty slot; a repeated one adds up.
template <typename T, int L, int V>
__global__ void __launch_bounds__(kRouteThreads)
    route_backward_kernel(const float* __restrict__ dw, const T* __restrict__ logits, const int32_t* __restrict__ idx,
                          RouteArgs a, T* __restrict__ dl) {
  constexpr int KS = L == 32 ? 1 : AGM_ROUTE_MAX_TOPK / 8;
  constexpr int TOK = 32 / L;
  pdl_wait();
  pdl_trigger();
  const int lane = lane_id(), sub = lane & (L - 1);
  const bool sigmoid = a.score == AGM_ROUTE_SIGMOID;
  const bool dense = !sigmoid && !a.renormalize;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (blockDim.x / 32) * TOK;
  for (int64_t t0 = (static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + warp_id()) * TOK; t0 < a.n; t0 += step) {
    const int64_t t = t0 + lane / L;
    const bool live = t < a.n;
    const int64_t tt = live ? t : t0;
    const T* row = logits + tt * a.n_experts;
    float l[V], m = kNegInf, total = 0.f;
    if (dense) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int e = sub + L * j;
        l[j] = e < a.n_experts ? Traits<T>::to_f(row[e]) : kNegInf;
        m = fmaxf(m, l[j]);
      }
      m = lanes_max<float, L>(m);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        l[j] = l[j] != kNegInf ? expf(l[j] - m) : 0.f;  // NaN stays
        total += l[j];
      }
      total = lanes_sum<float, L>(total);
    }
    int id[KS];
    float c[KS], g[KS], p[KS], mc = kNegInf;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const int r = sub + L * i;
      id[i] = r < a.k ? idx[tt * a.k + r] : -1;
      if (id[i] >= a.n_experts) id[i] = -1;
      c[i] = id[i] >= 0 ? Traits<T>::to_f(row[id[i]]) : kNegInf;
      g[i] = id[i] >= 0 ? a.scale * dw[tt * a.k + r] : 0.f;
      mc = fmaxf(mc, sigmoid ? fminf(c[i], 0.f) : c[i]);
    }
    mc = lanes_max<float, L>(mc);
    float sum = 0.f, inner = 0.f;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      if (dense)
        p[i] = c[i] != kNegInf ? expf(c[i] - m) / total : 0.f;
      else if (sigmoid)
        p[i] = c[i] != kNegInf ? expf(fminf(c[i], 0.f) - (a.renormalize ? mc : 0.f)) / (1.f + expf(-fabsf(c[i]))) : 0.f;
      else
        p[i] = c[i] != kNegInf ? expf(c[i] - mc) : 0.f;
      sum += p[i];
    }
    if (a.renormalize) {
      sum = lanes_sum<float, L>(sum);
#pragma unroll
      for (int i = 0; i < KS; ++i) p[i] = id[i] >= 0 && sum != 0.f ? p[i] / sum : 0.f;
    }
    if (a.renormalize || dense) {
#pragma unroll
      for (int i = 0; i < KS; ++i) inner += g[i] * p[i];
      inner = lanes_sum<float, L>(inner);
    }
    float out[V];
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = dense && total != 0.f ? -inner * (l[j] / total) : 0.f;
    // Slot values: what slot r adds to its expert.
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      if (dense)
        g[i] = p[i] * g[i];
      else if (sigmoid) {
        const float z = expf(-fabsf(c[i]));
        g[i] = p[i] * ((c[i] > 0.f ? z : 1.f) / (1.f + z)) * (g[i] - (a.renormalize ? inner : 0.f));
      } else {
        g[i] = p[i] * (g[i] - inner);
      }
      if (id[i] < 0) g[i] = 0.f;
    }
    for (int r = 0; r < a.k; ++r) {
      int e = -1;
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i)
        if (r / L == i) {
          e = id[i];
          v = g[i];
        }
      const int src = (lane & ~(L - 1)) | (r & (L - 1));
      e = __shfl_sync(0xffffffffu, e, src);
      v = __shfl_sync(0xffffffffu, v, src);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (e == sub + L * j) out[j] += v;
    }
    if (live) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int e = sub + L * j;
        if (e < a.n_experts) dl[t * a.n_experts + e] = Traits<T>::from_f(out[j]);
      }
    }
  }
}

// Lanes per token: enough registers' worth of experts on the fewest lanes.
template <typename Call>
cudaError_t by_width(int n_experts, bool grouped, Call&& call) {
  using std::integral_constant;
  if (!grouped && n_experts <= 16) return call(integral_constant<int, 4>{}, integral_constant<int, 4>{});
  if (!grouped && n_experts <= 64) return call(integral_constant<int, 8>{}, integral_constant<int, 8>{});
  if (n_experts <= 128) return call(integral_constant<int, 32>{}, integral_constant<int, 4>{});
  if (n_experts <= 256) return call(integral_constant<int, 32>{}, integral_constant<int, 8>{});
  return call(integral_constant<int, 32>{}, integral_constant<int, 16>{});
}

unsigned route_grid(int64_t n, int lanes, int num_sms) {
  const int64_t per_cta = kRouteThreads / lanes;
  return static_cast<unsigned>(std::min<int64_t>((n + per_cta - 1) / per_cta, static_cast<int64_t>(num_sms) * 8));
}

template <typename T>
cudaError_t route_t(const void* logits, const RouteArgs& a, int32_t* idx, float* weights, int num_sms,
                    cudaStream_t stream) {
  return by_width(a.n_experts, a.top_groups < a.n_groups, [&](auto l, auto v) {
    return launch_kernel(route_kernel<T, l.value, v.value>, dim3(route_grid(a.n, l.value, num_sms)),
                         dim3(kRouteThreads), 0, stream, static_cast<const T*>(logits), a, idx, weights);
  });
}

template <typename T>
cudaError_t route_backward_t(const float* dw, const void* logits, const int32_t* idx, const RouteArgs& a, void* dl,
                             int num_sms, cudaStream_t stream) {
  return by_width(a.n_experts, false, [&](auto l, auto v) {
    return launch_kernel(route_backward_kernel<T, l.value, v.value>, dim3(route_grid(a.n, l.value, num_sms)),
                         dim3(kRouteThreads), 0, stream, dw, static_cast<const T*>(logits), idx, a,
                         static_cast<T*>(dl));
  });
}

}  // namespace

cudaError_t route_experts(int dtype, const void* logits, const RouteArgs& a, int32_t* idx, float* weights, int num_sms,
                          cudaStream_t stream) {
  switch (dtype) {
    case AGM_F32: return route_t<float>(logits, a, idx, weights, num_sms, stream);
    case AGM_BF16: return route_t<__nv_bfloat16>(logits, a, idx, weights, num_sms, stream);
    case AGM_F16: return route_t<__half>(logits, a, idx, weights, num_sms, stream);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t route_experts_backward(int dtype, const float* dw, const void* logits, const int32_t* idx,
                                   const RouteArgs& a, void* dl, int num_sms, cudaStream_t stream) {
  switch (dtype) {
    case AGM_F32: return route_backward_t<float>(dw, logits, idx, a, dl, num_sms, stream);
    case AGM_BF16: return route_backward_t<__nv_bfloat16>(dw, logits, idx, a, dl, num_sms, stream);
    case AGM_F16: return route_backward_t<__half>(dw, logits, idx, a, dl, num_sms, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace agm
