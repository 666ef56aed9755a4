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
// and weight 0. A NaN logit takes its own expert out of the scores, and +inf
// under softmax is the limit of a large logit (the experts that have it share
// a score of 1), so such a row still chooses; its weights are NaN.
//
// The order of the keys is decided in real arithmetic: without a bias a key is
// the logit itself, exact. Otherwise the keys are computed in fp32 (error
// below 2^-20 (1 + |c|)); where two neighbours of the sorted top k + 1, or
// the last kept and first dropped group, are closer than that allows, the
// token is selected again with fp64 scores. So the indices do not depend on
// how an exponential is rounded. Equal logits with equal biases are equal
// keys and need no second look.
//
// Two forward kernels:
//
// * route_kernel, any E <= 512, k <= 32 and grouping: L lanes hold a token's
//   logits, V each (lane i holds experts i, i + L, ...) and pick k times the
//   largest key. Few experts take few lanes, so a warp routes 8 tokens of a
//   16-expert block; grouped routing takes the whole warp. Its picks make large
//   k slow where tokens are many: 65,536 x 256 without bias or groups take 94 us
//   at k = 10, 134 at 16, 239 at 32 (25 at 8, on the kernel below).
//
// * route_wide_kernel, E >= 32 and k <= 8, bound by its instructions rather
//   than by memory if it picked that way (65,536 x 256 grouped top-8 took 232
//   us). Lane c of L holds the experts [c * per, (c + 1) * per), a whole group
//   or a whole part of one, so a group's two largest keys are found without
//   talking to other lanes. The k-th largest of the maxima of 4 L sub-blocks
//   bounds the k-th largest key from below; the few keys that reach it (9 to
//   12 for k = 8) go to a list in index order, where each finds its rank by
//   counting. Where keys are too close to be told apart, those of the list,
//   or the two that make a group's score, are formed again in fp64. Only rows
//   with more than 32 keys at the border, or a NaN or infinite softmax, go
//   through the other kernel's code, one by one. That case now takes 37 us:
//   71 MB at 1.9 TB/s. Neither memory nor the issue slots (60% taken) are full:
//   the chain of a token's dependent steps bounds it, at the 24 warps per SM
//   that fit. Two CTAs per SM with 128 registers took 45 us, 16 lanes a token
//   48, 64 registers with the keys written over the logits 47. 262,144 x 64
//   bf16, top-6: 45 us.
//
// Few tokens (64 x 14: 2.3 us on the device) cost a launch and one pass's
// latency.
#include <algorithm>
#include <cfloat>
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

// Whether the order of real numbers may keep other groups than the fp32 scores
// (one a lane) do. They are half scores, h1 + h2 of the halved keys, since the
// sum of two keys near 3.4e38 is no fp32 number; `size_of` is |h1| + |h2|. A
// half key is off by its expert's score, `error` / 2 * 2^-24 at most, and by the
// rounding of the bias' add, and their sum and the ends here by a rounding
// each, which is 3 size_of 2^-24 in all (keys of opposite signs cancel in the
// score, not in its error). Infinite scores are exact.
template <int L>
__device__ __forceinline__ bool groups_near(float score, float size_of, float error, bool kept) {
  const float e = fabsf(score) < INFINITY ? (error + 4.f * size_of) * 0x1p-24f : 0.f;
  const float hi = lanes_max<float, L>(kept ? kNegInf : score + e);
  const float lo = -lanes_max<float, L>(kept && score > kNegInf ? e - score : kNegInf);
  return !(lo > hi) && hi > kNegInf;
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
        // min: +inf - +inf is NaN, for which it gives 0
        s[j] = l[j] > kNegInf ? exp_of(min(static_cast<F>(l[j]) - static_cast<F>(m), F(0))) : F(0);
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
        F mine = F(kNegInf), size_of = F(0);  // lane g: half the score of group g, and the magnitudes that went into it
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
          if (sub == g) {
            const F h1 = F(0.5) * t1, h2 = F(0.5) * t2;
            mine = t2 > F(kNegInf) ? h1 + h2 : h1;
            size_of = fabs(h1) + (t2 > F(kNegInf) ? fabs(h2) : F(0));
          }
        }
        uint32_t kept = 0;
        for (int i = 0; i < a.top_groups; ++i) {
          F v = ((kept >> sub) & 1u) ? F(kNegInf) : mine + F(0);
          int id = sub;
          lanes_best<F, 32>(v, id);
          if (!(v > F(kNegInf))) break;
          kept |= 1u << id;
        }
        if constexpr (kFast) near = groups_near<32>(mine, size_of, 16.f, (kept >> sub) & 1u);
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
  bool same = false;  // the last two picks are equal in logit and bias
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
      same = any && r > 0 && vl == prev_l && vb == prev_b;
      if (any && r > 0 && prev - v <= F(1.9e-6f) * (F(1) + fabs(v)) && !same) near = true;
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
  if constexpr (kFast) {
    // Equal experts on both sides of the border need no second look at one
    // another, but hide a later one that fp32 takes for equal.
    bool hidden = false;
    if (same)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (!((used >> j) & 1u) && prev - key[j] <= F(1.9e-6f) * (F(1) + fabs(prev)) &&
            !(l[j] == prev_l && a.bias[sub + L * j] == prev_b))
          hidden = true;
    const uint32_t token = L == 32 ? 0xffffffffu : ((1u << (L & 31)) - 1u) << (threadIdx.x & 31 & ~(L - 1));
    near |= (__ballot_sync(0xffffffffu, hidden) & token) != 0;
  }
  return near;
}

// Routes the warp's 32 / L tokens t0, t0 + 1, ...; a lane holds KS of its token's slots.
template <typename T, int L, int V, int KS>
__device__ __forceinline__ void route_tokens(const T* __restrict__ logits, const RouteArgs& a, int64_t t0,
                                             int32_t* __restrict__ idx, float* __restrict__ weights) {
  const int lane = lane_id(), sub = lane & (L - 1);
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

template <typename T, int L, int V, int KS>
__global__ void __launch_bounds__(kRouteThreads)
    route_kernel(const T* __restrict__ logits, RouteArgs a, int32_t* __restrict__ idx, float* __restrict__ weights) {
  constexpr int TOK = 32 / L;
  pdl_wait();
  pdl_trigger();
  const int64_t step = static_cast<int64_t>(gridDim.x) * (blockDim.x / 32) * TOK;
  for (int64_t t0 = (static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + warp_id()) * TOK; t0 < a.n; t0 += step)
    route_tokens<T, L, V, KS>(logits, a, t0, idx, weights);
}

// One token by a whole warp, out of line.
template <typename T>
__device__ __noinline__ void route_one(const T* __restrict__ logits, const RouteArgs& a, int64_t t,
                                       int32_t* __restrict__ idx, float* __restrict__ weights) {
  route_tokens<T, 32, AGM_ROUTE_MAX_EXPERTS / 32, 1>(logits, a, t, idx, weights);
}

// Approximate exponential (within 2^-22, relative, and 1.5 |v| 2^-24 for its
// rounded argument) and reciprocal (2^-23). A sigmoid 1 / (1 + e^-l) formed
// from them is off by at most s (1 - s) times the exponential's error, which
// is below 1.4 * 2^-24, plus s * 3 * 2^-24: two keys by 10 * 2^-24 (1 + |c|)
// together with the bias' add. A softmax score s is off by at most 30 s 2^-24
// (the sum's terms and tree for E <= 512), and all scores sum to 1, so two
// keys by 32 * 2^-24 (1 + |c|). For sums of two see groups_near.
__device__ __forceinline__ float fast_exp(float v) {
  float o;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(o) : "f"(v * 1.4426950408889634f));
  return o;
}
__device__ __forceinline__ float fast_rcp(float v) {
  float o;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(o) : "f"(v));
  return o;
}

__device__ __forceinline__ void order2(float& a, float& b) {  // a >= b
  const float t = fminf(a, b);
  a = fmaxf(a, b);
  b = t;
}
__device__ __forceinline__ void bitonic8(float (&v)[8]) {  // a bitonic sequence, to descending order
#pragma unroll
  for (int d = 4; d; d >>= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (!(i & d)) order2(v[i], v[i + d]);
}

// e / per for e < 512 (the quotient is at least 1 / 64 away from the next integer).
__device__ __forceinline__ int owner(int e, float inv_per) { return static_cast<int>((e + 0.5f) * inv_per); }

// Score in fp64; m and t: the softmax's maximum and sum.
__device__ __forceinline__ double exact_score(float l, bool sigmoid, float m, double t) {
  const double z = exp(sigmoid ? -static_cast<double>(l) : static_cast<double>(l) - m);
  return sigmoid ? 1.0 / (1.0 + z) : z / t;
}

constexpr int kWideTopK = 8;
constexpr int kWideList = 32;
constexpr int kWideOdd = kWideTopK + 1;

template <int L, int V>
struct WideSmem {
  static constexpr int kTok = 32 / L;
  static constexpr int kSlots = L < kWideTopK ? kWideTopK / L : 1;  // slots of a lane
  static constexpr int kLane = V + 4;  // floats between two lanes' experts: 16-byte rows, no bank conflicts
  float logit[kTok][L * kLane];
  double exact[kTok][kWideList];       // keys formed again
  float key[kTok][kWideList];
  int id[kTok][kWideList];
  float sorted[kTok][kWideTopK + 4];   // keys by rank, the first k + 1
  int sel[kTok][kWideTopK + 4];        // their experts; at kWideOdd: the token has no finite scores
};

template <typename T>
__device__ __forceinline__ float4 load4(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return __ldcs(reinterpret_cast<const float4*>(p));
  } else {
    const uint2 u = __ldcs(reinterpret_cast<const uint2*>(p));
    const T* h = reinterpret_cast<const T*>(&u);
    return make_float4(Traits<T>::to_f(h[0]), Traits<T>::to_f(h[1]), Traits<T>::to_f(h[2]), Traits<T>::to_f(h[3]));
  }
}

// max that keeps NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float o;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(o) : "f"(a), "f"(b));
  return o;
}
// bits |= v >= bound ? bit : 0
__device__ __forceinline__ void mark_if_ge(uint32_t& bits, float v, float bound, uint32_t bit) {
  asm("{\n\t.reg .pred p;\n\tsetp.ge.f32 p, %1, %2;\n\t@p or.b32 %0, %0, %3;\n\t}"
      : "+r"(bits)
      : "f"(v), "f"(bound), "r"(bit));
}

// CTAs per SM: as many as shared memory lets in (4 lanes take 59 KB a CTA, three
// an SM, and gain 1% from the registers: 65,536 x 32 with groups 23.5 us
// against 23.9) or, for 32 experts a lane, as registers do.
//
// KEYS: what orders the experts. kLogits: neither bias nor groups, the logit
// itself. kGroupsThenLogits: groups without a bias; the register key is the
// approximate score until the groups are chosen, then the logit, which orders
// as the scores do, exactly, also where those of a confident row (or sigmoids
// near zero) are below their error: 65,536 x 256 with logits of deviation 10
// take 98 us, mostly for group scores in fp64, where a bound from the scores
// let whole groups into the list and took 942; of deviation 1, 41 and 43.
// kBiased: the register key is the approximate score plus bias.
enum WideKeys { kLogits, kGroupsThenLogits, kBiased };

template <typename T, int L, int V, WideKeys KEYS>
__global__ void __launch_bounds__(kRouteThreads, V <= 16 && L > 4 ? 4 : 3)
    route_wide_kernel(const T* __restrict__ logits, RouteArgs a, int per, int run, int32_t* __restrict__ idx,
                      float* __restrict__ weights) {
  using Smem = WideSmem<L, V>;
  constexpr int TOK = Smem::kTok, LD = Smem::kLane, SB = V / 4;
  constexpr uint32_t kAll = 0xffffffffu;
  static_assert(sizeof(Smem) % 16 == 0, "the warps' parts are read in 16-byte units");
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Smem& sm = reinterpret_cast<Smem*>(smem_raw)[warp_id()];
  float* bias_s = reinterpret_cast<float*>(smem_raw + sizeof(Smem) * (kRouteThreads / 32));  // [L * LD]
  const int lane = lane_id(), sub = lane & (L - 1), tok = lane / L;
  const int E = a.n_experts;
  const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * (kRouteThreads / 32) + warp_id()) * TOK;
  const int toks = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(TOK), a.n - t0)));
  constexpr bool RAW = KEYS == kLogits, BIASED = KEYS == kBiased;
  const bool grouped = KEYS == kGroupsThenLogits || (BIASED && a.top_groups < a.n_groups);
  const bool sigmoid = a.score == AGM_ROUTE_SIGMOID;
  const float inv_per = 1.f / per;
  pdl_wait();
  pdl_trigger();
  // 1. The tokens' logits to shared memory, as fp32 in the lanes' order;
  // places of no expert hold -inf.
  const T* src = logits + t0 * E;
  if (run) {  // E == L * V, aligned rows: the tokens are one run of 16-byte (8-byte) units
    constexpr int N = TOK * L * V / 128;
    float4 f[N];
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const int i = 128 * q + 4 * lane;
      f[q] = i / (L * V) < toks ? load4<T>(src + i) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if constexpr (BIASED)
      for (int e = threadIdx.x; e < E; e += kRouteThreads) bias_s[e / V * LD + e % V] = a.bias[e];
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const int i = 128 * q + 4 * lane, c = i / V;  // c counts lanes over all tokens
      *reinterpret_cast<float4*>(&sm.logit[0][c * LD + (i - c * V)]) = f[q];
    }
  } else {
    for (int i = lane; i < TOK * L * LD; i += 32) sm.logit[0][i] = kNegInf;
    __syncwarp();
    for (int k = 0; k < toks; ++k)
      for (int e = lane; e < E; e += 32) {
        const int c = owner(e, inv_per);
        sm.logit[k][c * LD + (e - c * per)] = Traits<T>::to_f(src[k * E + e]);
      }
    if constexpr (BIASED)
      for (int e = threadIdx.x; e < E; e += kRouteThreads) {
        const int c = owner(e, inv_per);
        bias_s[c * LD + (e - c * per)] = a.bias[e];
      }
  }
  __syncthreads();
  if (toks == 0) return;  // whole warps; no barrier of the CTA follows
  const uint32_t part = L == 32 ? kAll : ((1u << (L & 31)) - 1u) << (tok * L);
  const float* my_logit = &sm.logit[tok][sub * LD];
  auto place = [&](int e) {  // of expert e among the lanes' experts
    const int c = owner(e, inv_per);
    return c * LD + (e - c * per);
  };
  // 2. Keys, and per quarter of the lane's experts the two largest.
  float key[V], m = 0.f, inv_t = 0.f;
#pragma unroll
  for (int q = 0; q < V / 4; ++q) {
    const float4 f = *reinterpret_cast<const float4*>(my_logit + 4 * q);
    key[4 * q] = f.x, key[4 * q + 1] = f.y, key[4 * q + 2] = f.z, key[4 * q + 3] = f.w;
  }
  bool bad = false;
  if (!sigmoid && !(RAW && a.renormalize)) {
    m = kNegInf;
#pragma unroll
    for (int j = 0; j < V; ++j) m = fmaxf(m, key[j]);
    m = lanes_max<float, L>(m);
    bad = m == INFINITY;
    if (m == kNegInf) m = 0.f;  // exp(-inf - 0) = 0
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) t += fast_exp(key[j] - m);
    t = lanes_sum<float, L>(t);
    // t is NaN beside a NaN or +inf logit: the scores below are none then, and the other kernel's code routes the
    // token (a flag kept in a register cost spills).
    if (!RAW) sm.sel[tok][kWideOdd] = t != t;
    inv_t = t > 0.f ? 1.f / t : 0.f;
  }
  float top[8], g1 = kNegInf, g2 = kNegInf;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    float k1 = kNegInf, k2 = kNegInf;
    if constexpr (!RAW) {
      float s[SB];
      if (sigmoid) {
#pragma unroll
        for (int j = 0; j < SB; ++j) s[j] = fast_rcp(1.f + fast_exp(-key[b * SB + j]));
      } else {
#pragma unroll
        for (int j = 0; j < SB; ++j) s[j] = fast_exp(key[b * SB + j] - m) * inv_t;
      }
      if constexpr (BIASED) {
        if constexpr (SB % 4 == 0) {
#pragma unroll
          for (int j = 0; j < SB; j += 4) {
            const float4 f = *reinterpret_cast<const float4*>(bias_s + sub * LD + b * SB + j);
            s[j] += f.x, s[j + 1] += f.y, s[j + 2] += f.z, s[j + 3] += f.w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < SB; ++j) s[j] += bias_s[sub * LD + b * SB + j];
        }
      }
      float h[SB], w[SB];  // the two largest of 2, 4, ... keys
#pragma unroll
      for (int j = 0; j < SB; ++j) {
        const float c = key[b * SB + j] == kNegInf ? kNegInf : s[j];
        key[b * SB + j] = c;
        h[j] = c;
        w[j] = kNegInf;
      }
#pragma unroll
      for (int o = 1; o < SB; o <<= 1)
#pragma unroll
        for (int j = 0; j + o < SB; j += 2 * o) {
          const float mid = fminf(h[j], h[j + o]);
          w[j] = o == 1 ? mid : fmaxf(fmaxf(w[j], w[j + o]), mid);
          h[j] = max_nan(h[j], h[j + o]);
        }
      k1 = h[0];
      k2 = w[0];
    } else {
#pragma unroll
      for (int j = 0; j < SB; ++j) k1 = max_nan(k1, key[b * SB + j]);
    }
    if (k1 != k1) {  // NaN among them: never chosen
      bad = true;
      k1 = k2 = kNegInf;
#pragma unroll
      for (int j = b * SB; j < (b + 1) * SB; ++j) {
        if (!(key[j] > kNegInf)) key[j] = kNegInf;
        k2 = fmaxf(k2, fminf(k1, key[j]));
        k1 = fmaxf(k1, key[j]);
      }
    }
    g2 = fmaxf(fmaxf(g2, k2), fminf(g1, k1));
    g1 = fmaxf(g1, k1);
    top[b] = k1;
  }
  bool near = false, kept = true;
  double exact_t = 1.0;
  bool have_t = sigmoid;
  // The softmax's sum in fp64, formed when first needed (whole warps).
  auto need_sum = [&]() {
    if (have_t) return;
    have_t = true;
    double t = 0.0;
    for (int j = 0; j < V; ++j) t += exact_score(my_logit[j], false, m, 1.0);
    exact_t = lanes_sum<double, L>(t);
  };
  if (grouped) {
    const int span = L / a.n_groups;  // lanes of a group
    const float lane2 = g2;           // the lane's own second key
    for (int o = 1; o < span; o <<= 1) {
      const float o1 = __shfl_xor_sync(kAll, g1, o), o2 = __shfl_xor_sync(kAll, g2, o);
      g2 = fmaxf(fminf(g1, o1), fmaxf(g2, o2));
      g1 = fmaxf(g1, o1);
    }
    const float h1 = 0.5f * g1, h2 = 0.5f * g2;
    const float score = g2 > kNegInf ? h1 + h2 : h1;
    const float size_of = fabsf(h1) + (g2 > kNegInf ? fabsf(h2) : 0.f);
    int rank = 0;
    for (int o = span; o < L; o += span) {
      const int other = (sub + o) & (L - 1);
      const float so = __shfl_sync(kAll, score, (lane & ~(L - 1)) | other);
      rank += so > score || (so == score && other < sub);
    }
    near = groups_near<L>(score, size_of, sigmoid ? 5.f : 8.f, rank < a.top_groups);
    if (__any_sync(kAll, near)) {
      // The group scores again, from the exact keys of the one or two (more
      // only where they are close) largest in every lane.
      need_sum();
      const float cut = lane2 == INFINITY ? lane2 : fmaxf(lane2 - (sigmoid ? 20.f : 64.f) * 0x1p-24f * (1.f + fabsf(lane2)), -FLT_MAX);
      uint32_t pair = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) mark_if_ge(pair, key[j], lane2 > kNegInf ? cut : -FLT_MAX, 1u << j);
      double e1 = -INFINITY, e2 = -INFINITY;
      while (pair) {
        const int j = __ffs(pair) - 1;
        pair &= pair - 1;
        const double d = exact_score(my_logit[j], sigmoid, m, exact_t) + (BIASED ? bias_s[sub * LD + j] : 0.f);
        e2 = fmax(e2, fmin(e1, d));
        e1 = fmax(e1, d);
      }
      for (int o = 1; o < span; o <<= 1) {
        const double o1 = __shfl_xor_sync(kAll, e1, o), o2 = __shfl_xor_sync(kAll, e2, o);
        e2 = fmax(fmin(e1, o1), fmax(e2, o2));
        e1 = fmax(e1, o1);
      }
      const double exact = e2 > -INFINITY ? e1 + e2 : e1;
      rank = 0;
      for (int o = span; o < L; o += span) {
        const int other = (sub + o) & (L - 1);
        const double so = __shfl_sync(kAll, exact, (lane & ~(L - 1)) | other);
        rank += so > exact || (so == exact && other < sub);
      }
      near = false;
    }
    kept = rank < a.top_groups;
    if (!kept)
#pragma unroll
      for (int b = 0; b < 4; ++b) top[b] = kNegInf;
  }
  if constexpr (KEYS == kGroupsThenLogits) {
    // NaN reaches neither a maximum nor a bound, -inf no bound.
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      const float4 f = *reinterpret_cast<const float4*>(my_logit + 4 * q);
      key[4 * q] = f.x, key[4 * q + 1] = f.y, key[4 * q + 2] = f.z, key[4 * q + 3] = f.w;
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      top[b] = kNegInf;
#pragma unroll
      for (int j = b * SB; j < (b + 1) * SB; ++j) top[b] = fmaxf(top[b], key[j]);
      if (!kept) top[b] = kNegInf;
    }
  }
  // 3. A bound that at least k keys reach: the k-th largest quarter maximum.
  order2(top[0], top[1]);
  order2(top[2], top[3]);
  order2(top[0], top[2]);
  order2(top[1], top[3]);
  order2(top[1], top[2]);
#pragma unroll
  for (int i = 0; i < 4; ++i) top[7 - i] = __shfl_xor_sync(kAll, top[i], 1);
  bitonic8(top);
#pragma unroll
  for (int o = 2; o < L; o <<= 1) {
    float other[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) other[i] = __shfl_xor_sync(kAll, top[i], o);
#pragma unroll
    for (int i = 0; i < 8; ++i) top[i] = fmaxf(top[i], other[7 - i]);
    bitonic8(top);
  }
  float bound = top[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) bound = i < a.k ? top[i] : bound;
  const float error = (sigmoid ? 10.f : 32.f) * 0x1p-24f;  // of (1 + |key|)
  if (BIASED) bound -= 2.f * error * (1.f + fabsf(bound));
  if (!(bound > kNegInf)) bound = -FLT_MAX;
  // 4. The keys that reach it, in index order.
  uint32_t hit = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) mark_if_ge(hit, key[j], bound, 1u << j);
  if (!kept) hit = 0;
  const int count = __popc(hit);
  int upto = count;
#pragma unroll
  for (int o = 1; o < L; o <<= 1) {
    const int u = __shfl_up_sync(kAll, upto, o, L);
    if (sub >= o) upto += u;
  }
  const int total = __shfl_sync(kAll, upto, (lane & ~(L - 1)) | (L - 1));
  bad = (__ballot_sync(kAll, bad) & part) != 0;
  const bool crowded = total > kWideList;
  for (int at = upto - count; hit && at < kWideList; ++at) {
    const int j = __ffs(hit) - 1;
    hit &= hit - 1;
    sm.id[tok][at] = sub * per + j;
    sm.key[tok][at] = BIASED ? __int_as_float(sub * LD + j) : my_logit[j] + 0.f;  // its place; or -0 = 0
  }
  const int len = min(total, kWideList);
  const int len4 = (len + 3) & ~3;
  if constexpr (!BIASED) {
    for (int i = len + sub; i < len4; i += L) sm.key[tok][i] = kNegInf;
  } else {
    // The keys again, shared out over the lanes: few hold most of the list.
    __syncwarp();
    for (int i = sub; i < len4; i += L) {
      float v = kNegInf;
      if (i < len) {
        const int at = __float_as_int(sm.key[tok][i]);
        v = sm.logit[tok][at];
        v = sigmoid ? fast_rcp(1.f + fast_exp(-v)) : fast_exp(v - m) * inv_t;  // as in 2
        v += bias_s[at];
      }
      sm.key[tok][i] = v + 0.f;  // -0 = 0
    }
  }
  for (int i = sub; i <= kWideTopK; i += L) sm.sel[tok][i] = -1;
  __syncwarp();
  // 5. Each finds its rank: the number of keys above it.
  const bool live = tok < toks;
  for (int p = sub; p < len; p += L) {
    const float c = sm.key[tok][p];
    int above = 0;
    if constexpr (!BIASED) {
      // Keys are exact: an equal one before p is above it too, o > c being o >= the float after c.
      const float up = __int_as_float(__float_as_int(c) + (c < 0.f ? -1 : 1));
      for (int q = 0; q < len4; q += 4) {
        const float4 o = *reinterpret_cast<const float4*>(&sm.key[tok][q]);
        above += (o.x >= (q < p ? c : up)) + (o.y >= (q + 1 < p ? c : up)) + (o.z >= (q + 2 < p ? c : up)) +
                 (o.w >= (q + 3 < p ? c : up));
      }
    } else {
      for (int q = 0; q < len4; q += 4) {
        const float4 o = *reinterpret_cast<const float4*>(&sm.key[tok][q]);
        above += (o.x > c) + (o.y > c) + (o.z > c) + (o.w > c);
      }
    }
    if (above <= a.k) {
      sm.sel[tok][above] = sm.id[tok][p];
      sm.sorted[tok][above] = c;
    }
  }
  __syncwarp();
  // Neighbours closer than the error of keys leave the order open; equal keys
  // leave a rank empty.
  for (int r = sub; BIASED && r < a.k && r < len; r += L) {
    const float c = sm.sorted[tok][r];
    const bool more = r + 1 < len;
    near |= sm.sel[tok][r] < 0 || (more && sm.sel[tok][r + 1] < 0) ||
            (more && c - sm.sorted[tok][r + 1] <= error * (1.f + fabsf(c)));
  }
  if (BIASED && __any_sync(kAll, near && live)) {
    need_sum();
    near = (__ballot_sync(kAll, near) & part) != 0 && live;
    __syncwarp();
    // Again with exact keys, equal ones by index.
    if (near)
      for (int p = sub; p < len; p += L) {
        const int e = sm.id[tok][p];
        sm.exact[tok][p] = exact_score(sm.logit[tok][place(e)], sigmoid, m, exact_t) + a.bias[e];
      }
    __syncwarp();
    if (near)
      for (int p = sub; p < len; p += L) {
        const double c = sm.exact[tok][p];
        int above = 0;
        for (int q = 0; q < len; ++q) above += sm.exact[tok][q] > c || (sm.exact[tok][q] == c && q < p);
        if (above < a.k) sm.sel[tok][above] = sm.id[tok][p];
      }
  }
  __syncwarp();
  // 6. Weights.
  constexpr int SLOTS = Smem::kSlots;
  int e[SLOTS];
  float l[SLOTS], p[SLOTS], total_p = 1.f;
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const int r = sub + L * i;
    e[i] = live && r < a.k ? sm.sel[tok][r] : -1;
    l[i] = e[i] >= 0 ? sm.logit[tok][place(e[i])] : kNegInf;
    p[i] = 0.f;
  }
  if (a.renormalize) {
    float mx = kNegInf;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) mx = fmaxf(mx, sigmoid ? fminf(l[i], 0.f) : l[i]);
    mx = lanes_max<float, L>(mx);
    total_p = 0.f;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      if (e[i] >= 0) p[i] = expf((sigmoid ? fminf(l[i], 0.f) : l[i]) - mx) / (sigmoid ? 1.f + expf(-fabsf(l[i])) : 1.f);
      total_p += p[i];
    }
    total_p = lanes_sum<float, L>(total_p);
    // A renormalised softmax does not look at the other logits: +inf among them is met here.
    bad |= !sigmoid && mx == INFINITY;
  } else {
#pragma unroll
    for (int i = 0; i < SLOTS; ++i)
      if (e[i] >= 0) p[i] = sigmoid ? expf(fminf(l[i], 0.f)) / (1.f + expf(-fabsf(l[i]))) : expf(l[i] - m) * inv_t;
  }
  bool nan_row = false;
  if (bad && live) {  // a NaN bias is no NaN logit
    for (int i = 0; i < E; ++i) {
      const float v = sm.logit[tok][place(i)];
      nan_row |= v != v || (!sigmoid && v == INFINITY);
    }
  }
  const bool alone = crowded || (!RAW && !sigmoid && sm.sel[tok][kWideOdd] != 0);
  if (live && !alone) {
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      const int r = sub + L * i;
      if (r < a.k) {
        idx[(t0 + tok) * a.k + r] = e[i];
        weights[(t0 + tok) * a.k + r] = nan_row ? NAN : (e[i] >= 0 ? a.scale * (p[i] / total_p) : 0.f);
      }
    }
  }
  // 7. Tokens with more keys at the border than the list holds, or without finite scores, one by one.
  // Last, so that the call keeps nothing of the above alive.
  for (uint32_t open = __ballot_sync(kAll, alone && live && sub == 0); open; open &= open - 1)
    route_one<T>(logits, a, t0 + (__ffs(open) - 1) / L, idx, weights);
}

// Exponential of the gradient for logits of type T.
template <typename T>
__device__ __forceinline__ float grad_exp(float v) {
  if constexpr (std::is_same<T, float>::value)
    return expf(v);
  else
    return fast_exp(v);
}

// d l from d w. With s the scores, w' the renormalised weights, G_e the sum of
// scale dw over the slots that chose e and n_e their number:
//   softmax, renormalised   dl_e = w'_e (G_e - n_e inner),           inner = sum_e w'_e G_e
//   sigmoid, renormalised   dl_e = w'_e (1 - s_e) (G_e - n_e inner)
//   sigmoid                 dl_e = s_e (1 - s_e) G_e
//   softmax                 dl_e = s_e (G_e - sum_j s_j G_j)
// All but the last are zero outside the chosen experts. An index outside
// [0, E) is an empty slot; a repeated one adds up.
// Lane i of L holds the experts [i V, (i + 1) V), so that whole rows move in
// 16-byte (8-byte) units where they are aligned. A span as it is in memory:
template <typename T, int V>
struct RawSpan {
  T v[V];
  __device__ __forceinline__ void load(const T* __restrict__ row, int e0, int E, int vec) {
    if (vec) {
#pragma unroll
      for (int q = 0; q < V; q += 4) {
        if (e0 + q < E) {
          if constexpr (sizeof(T) == 4)
            *reinterpret_cast<float4*>(&v[q]) = *reinterpret_cast<const float4*>(row + e0 + q);
          else
            *reinterpret_cast<uint2*>(&v[q]) = *reinterpret_cast<const uint2*>(row + e0 + q);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (e0 + j < E) v[j] = row[e0 + j];
    }
  }
  __device__ __forceinline__ void get(float (&l)[V], int e0, int E) const {
#pragma unroll
    for (int j = 0; j < V; ++j) l[j] = e0 + j < E ? Traits<T>::to_f(v[j]) : kNegInf;
  }
};
template <typename T, int V>
__device__ __forceinline__ void store_span(T* __restrict__ row, int e0, int E, int vec, const float (&v)[V]) {
  if (vec) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      if (e0 + 4 * q < E) {
        if constexpr (sizeof(T) == 4)
          *reinterpret_cast<float4*>(row + e0 + 4 * q) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        else
          *reinterpret_cast<uint2*>(row + e0 + 4 * q) =
              make_uint2(pack2<T>(v[4 * q], v[4 * q + 1]), pack2<T>(v[4 * q + 2], v[4 * q + 3]));
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (e0 + j < E) row[e0 + j] = Traits<T>::from_f(v[j]);
  }
}

// The slots' values go to their experts' lanes through shared memory: of the
// slots that chose an expert the first adds up all of them, in slot order.
// For 16-bit logits the exponentials are the approximate ones: an expert |v|
// below the row's maximum is off by (4 + 1.5 |v|) 2^-24, which at |v| = 80,
// where e^-v nearly leaves fp32, is 1.5% of fp16's half step and
// 0.2% of bf16's. fp32 logits take expf (262,144 x 64, top-6: 63 us where the
// approximate ones took 56). A lane holds KS of its token's slots: one where
// k <= L, which leaves registers for a fourth CTA per SM and cuts the slots'
// code by KS^2.
//
// Bound by the latency of its steps at 32 warps per SM (60% of the issue slots
// are taken), not by memory: 262,144 x 64 bf16, top-6, takes 42 us, 45
// renormalised (80 MB, 1.9 TB/s; with four slots a lane throughout a quarter
// more), 49,151 x 64 10.5 us.
template <typename T, int L, int V, int KS>
__global__ void __launch_bounds__(kRouteThreads)
    route_backward_kernel(const float* __restrict__ dw, const T* __restrict__ logits, const int32_t* __restrict__ idx,
                          RouteArgs a, int vec, T* __restrict__ dl) {
  constexpr int TOK = 32 / L;
  constexpr uint32_t kAll = 0xffffffffu;
  __shared__ __align__(16) float grad_s[kRouteThreads / 32][TOK][L * V];
  __shared__ __align__(16) float count_s[kRouteThreads / 32][TOK][L * V];
  const int lane = lane_id(), sub = lane & (L - 1), tok = lane / L;
  float* mine_g = &grad_s[warp_id()][tok][sub * V];
  float* mine_n = &count_s[warp_id()][tok][sub * V];
#pragma unroll
  for (int j = 0; j < V; j += 4) {
    *reinterpret_cast<float4*>(mine_g + j) = make_float4(0.f, 0.f, 0.f, 0.f);
    *reinterpret_cast<float4*>(mine_n + j) = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  pdl_wait();
  pdl_trigger();
  const bool sigmoid = a.score == AGM_ROUTE_SIGMOID;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (blockDim.x / 32) * TOK;
  int64_t t0 = (static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + warp_id()) * TOK;
  // The next tokens' values are in flight while these are worked on.
  RawSpan<T, V> raw;
  int next_id[KS];
  float next_g[KS];
  auto fetch = [&](int64_t first) {
    if (first >= a.n) return;
    const int64_t tt = min(first + tok, a.n - 1);
    raw.load(logits + tt * a.n_experts, sub * V, a.n_experts, vec);
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const int r = sub + L * i;
      next_id[i] = r < a.k ? idx[tt * a.k + r] : -1;
      next_g[i] = r < a.k ? dw[tt * a.k + r] : 0.f;
    }
  };
  fetch(t0);
  for (; t0 < a.n; t0 += step) {
    const int64_t t = t0 + tok;
    const bool live = t < a.n;
    float l[V];
    raw.get(l, sub * V, a.n_experts);
    int id[KS];
    float g[KS];
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      id[i] = next_id[i] < a.n_experts ? next_id[i] : -1;
      g[i] = id[i] >= 0 ? a.scale * next_g[i] : 0.f;
    }
    fetch(t0 + step);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      if (L * i >= a.k) break;
      float sum = 0.f, n = 0.f;
      bool first = true;
#pragma unroll
      for (int o = 0; o < KS; ++o) {
        if (L * o >= a.k) break;
        for (int q = 0; q < L && L * o + q < a.k; ++q) {
          const int src = (lane & ~(L - 1)) | q;
          const int oe = __shfl_sync(kAll, id[o], src);
          const float og = __shfl_sync(kAll, g[o], src);
          if (oe == id[i]) {
            sum += og;
            n += 1.f;
            if (L * o + q < sub + L * i) first = false;
          }
        }
      }
      if (first && id[i] >= 0) {
        grad_s[warp_id()][tok][id[i]] = sum;
        count_s[warp_id()][tok][id[i]] = n;
      }
    }
    __syncwarp();
    float G[V], n[V];
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const float4 x = *reinterpret_cast<const float4*>(mine_g + j), y = *reinterpret_cast<const float4*>(mine_n + j);
      G[j] = x.x, G[j + 1] = x.y, G[j + 2] = x.z, G[j + 3] = x.w;
      n[j] = y.x, n[j + 1] = y.y, n[j + 2] = y.z, n[j + 3] = y.w;
      *reinterpret_cast<float4*>(mine_g + j) = make_float4(0.f, 0.f, 0.f, 0.f);
      *reinterpret_cast<float4*>(mine_n + j) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    // Scores, up to a common factor: over all experts, or (renormalised) the chosen ones.
    float m = kNegInf, total = 0.f, inner = 0.f;
    if (!sigmoid || a.renormalize) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (!a.renormalize || n[j] > 0.f) m = fmaxf(m, sigmoid ? fminf(l[j], 0.f) : l[j]);
      m = lanes_max<float, L>(m);
    }
    float p[V], rest[V];  // score; 1 - score (sigmoid)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      rest[j] = 1.f;
      if (sigmoid) {
        const float z = grad_exp<T>(-fabsf(l[j]));
        const float inv = fast_rcp(1.f + z);
        rest[j] = (l[j] > 0.f ? z : 1.f) * inv;
        // s = e^min(l, 0) / (1 + z); renormalised, e^-m times that, which does not underflow with all of them.
        p[j] = a.renormalize ? grad_exp<T>(fminf(l[j], 0.f) - m) * inv : (l[j] > 0.f ? 1.f : z) * inv;
      } else {
        p[j] = l[j] != kNegInf ? grad_exp<T>(l[j] - m) : 0.f;  // NaN stays
      }
      if (l[j] == kNegInf || (a.renormalize && !(n[j] > 0.f))) p[j] = 0.f;
      total += a.renormalize ? n[j] * p[j] : p[j];
      inner += p[j] * G[j];
    }
    if (!sigmoid || a.renormalize) {
      total = lanes_sum<float, L>(total);
      const float inv = total > 0.f ? 1.f / total : total;  // 0 where nothing is left; NaN stays
      inner = lanes_sum<float, L>(inner) * inv;
#pragma unroll
      for (int j = 0; j < V; ++j) p[j] *= inv;
    } else {
      inner = 0.f;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = G[j] - (a.renormalize ? n[j] * inner : inner);
      l[j] = p[j] * rest[j] * d;
    }
    if (live) store_span<T, V>(dl + t * a.n_experts, sub * V, a.n_experts, vec, l);
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

// At most `per_sm` CTAs per SM. The forward takes more than are resident: its
// tokens differ (65,536 x 24, top-4: 18.5 us on 4, 15.8 on 8). The gradient
// takes the resident 4: each CTA prefetches its next tokens (262,144 x 64, top-6:
// 43.5 us on 4, 50.9 on 6, 44.0 on 8).
unsigned route_grid(int64_t n, int lanes, int num_sms, int per_sm) {
  const int64_t per_cta = kRouteThreads / lanes;
  return static_cast<unsigned>(std::min<int64_t>((n + per_cta - 1) / per_cta, static_cast<int64_t>(num_sms) * per_sm));
}

template <typename T, int L, int V>
cudaError_t launch_wide(const T* logits, const RouteArgs& a, int per, int32_t* idx, float* weights,
                        cudaStream_t stream) {
  const int smem = static_cast<int>(sizeof(WideSmem<L, V>)) * (kRouteThreads / 32) + L * WideSmem<L, V>::kLane * 4;
  const int run = a.n_experts == L * V && reinterpret_cast<uintptr_t>(logits) % (4 * sizeof(T)) == 0;
  const auto kernel = a.bias                       ? route_wide_kernel<T, L, V, kBiased>
                      : a.top_groups < a.n_groups ? route_wide_kernel<T, L, V, kGroupsThenLogits>
                                                  : route_wide_kernel<T, L, V, kLogits>;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return e;
  const int64_t per_cta = kRouteThreads / L;
  const int64_t ctas = (a.n + per_cta - 1) / per_cta;
  if (ctas > INT32_MAX) return cudaErrorInvalidValue;
  return launch_kernel(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kRouteThreads), smem, stream, logits, a, per, run,
                       idx, weights);
}

// Lanes per token and experts per lane of the wide kernel, or false where it
// does not apply: with groups, a lane holds a whole group or an equal part.
bool wide_shape(const RouteArgs& a, int& lanes, int& per) {
  if (a.k > kWideTopK || a.n_experts < 32) return false;
  const bool grouped = a.top_groups < a.n_groups;
  if (grouped && (a.n_groups & (a.n_groups - 1))) return false;
  lanes = std::max(a.n_experts <= 64 ? 4 : 8, grouped ? a.n_groups : 1);
  while (a.n_experts > 32 * lanes) lanes *= 2;
  if (grouped && a.n_experts % lanes) return false;
  per = (a.n_experts + lanes - 1) / lanes;
  return per <= 32;
}

template <typename T>
cudaError_t route_t(const void* logits, const RouteArgs& a, int32_t* idx, float* weights, int num_sms,
                    cudaStream_t stream) {
  int lanes, per;
  if (wide_shape(a, lanes, per)) {
    const T* x = static_cast<const T*>(logits);
    if (lanes == 4) return launch_wide<T, 4, 16>(x, a, per, idx, weights, stream);  // at most 64 experts
    if (lanes == 8)
      return per <= 8    ? launch_wide<T, 8, 8>(x, a, per, idx, weights, stream)
             : per <= 16 ? launch_wide<T, 8, 16>(x, a, per, idx, weights, stream)
                         : launch_wide<T, 8, 32>(x, a, per, idx, weights, stream);
    if (lanes == 16)
      return per <= 16 ? launch_wide<T, 16, 16>(x, a, per, idx, weights, stream)
                       : launch_wide<T, 16, 32>(x, a, per, idx, weights, stream);
    return launch_wide<T, 32, 16>(x, a, per, idx, weights, stream);
  }
  return by_width(a.n_experts, a.top_groups < a.n_groups, [&](auto l, auto v) {
    constexpr int L = l.value, V = v.value;
    constexpr int kMost = L == 32 ? 1 : AGM_ROUTE_MAX_TOPK / 8;  // 4 lanes serve at most 16 experts
    const auto kernel = a.k <= L ? route_kernel<T, L, V, 1> : route_kernel<T, L, V, kMost>;
    return launch_kernel(kernel, dim3(route_grid(a.n, L, num_sms, 8)), dim3(kRouteThreads), 0, stream,
                         static_cast<const T*>(logits), a, idx, weights);
  });
}

template <typename T>
cudaError_t route_backward_t(const float* dw, const void* logits, const int32_t* idx, const RouteArgs& a, void* dl,
                             int num_sms, cudaStream_t stream) {
  using std::integral_constant;
  const uintptr_t at = reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(dl);
  const int vec = a.n_experts % 4 == 0 && at % (4 * sizeof(T)) == 0;
  auto launch = [&](auto l, auto v) {
    constexpr int L = l.value, V = v.value;
    const auto kernel = a.k <= L ? route_backward_kernel<T, L, V, 1>
                                 : route_backward_kernel<T, L, V, AGM_ROUTE_MAX_TOPK / L>;
    return launch_kernel(kernel, dim3(route_grid(a.n, L, num_sms, 4)), dim3(kRouteThreads), 0, stream, dw,
                         static_cast<const T*>(logits), idx, a, vec, static_cast<T*>(dl));
  };
  const integral_constant<int, 8> v8;
  if (a.n_experts <= 32) return launch(integral_constant<int, 4>{}, v8);
  if (a.n_experts <= 64) return launch(integral_constant<int, 8>{}, v8);
  if (a.n_experts <= 128) return launch(integral_constant<int, 16>{}, v8);
  if (a.n_experts <= 256) return launch(integral_constant<int, 32>{}, v8);
  return launch(integral_constant<int, 32>{}, integral_constant<int, 16>{});
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
