// Block-scaled e4m3: quantisation of rows and of weights, the inverse, and the
// expert dispatch and weighted sum around the 8-bit grouped products.
//
// All of these move memory and are bound by it. A lane owns 16 consecutive
// elements (one 16-byte store of e4m3), 8 lanes a block of 128, a warp 512
// columns of a row, whose four scales are one 32-bit word of the row's scale
// tile.
#include <algorithm>
#include <type_traits>

#include "fp8.cuh"
#include "kernels.h"

namespace agm {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTokBlk = AGM_DISPATCH_BLOCK;

// The lane's 16 elements as they are in memory, so that several units can be in flight.
template <typename T>
struct Raw16 {
  uint4 u[sizeof(T)];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) u[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) u[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void unpack(float (&v)[16]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[4 * i] = __uint_as_float(u[i].x);
        v[4 * i + 1] = __uint_as_float(u[i].y);
        v[4 * i + 2] = __uint_as_float(u[i].z);
        v[4 * i + 3] = __uint_as_float(u[i].w);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float f[8];
        unpack8<T>(u[i], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[8 * i + j] = f[j];
      }
    }
  }
};

__device__ __forceinline__ float amax16(const float (&v)[16]) {
  float m[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 16; ++i) m[i & 1] = fmaxf(m[i & 1], fabsf(v[i]));  // passes over NaN
  return fmaxf(m[0], m[1]);
}

__device__ __forceinline__ bool is_inf(float v) { return v == __uint_as_float(0x7f800000u); }

// The lane's values without infinities (as NaN), and their largest finite magnitude.
__device__ __forceinline__ float drop_inf(float (&v)[16]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    m = fmaxf(m, finite_abs(v[i]));
    v[i] = inf_to_nan(v[i]);
  }
  return m;
}

__device__ __forceinline__ uint4 encode16(const float (&v)[16], float inv) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = __float_as_uint(v[4 * i + j]);
    scale2(x[0], x[1], inv);
    scale2(x[2], x[3], inv);
    w[i] = pack_e4m3x4(__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]), __uint_as_float(x[3]));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Quantises the lane's 16 elements of 512 columns of a row; word is the row's
// scale word (in every lane).
__device__ __forceinline__ uint4 encode_unit(float (&v)[16], int lane, uint32_t& word) {
  float m = amax16(v);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (__any_sync(0xffffffffu, is_inf(m))) {
    m = drop_inf(v);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  }
  const uint32_t byte = scale_byte(m);
  uint32_t w = byte << (8 * (lane >> 3));
  w |= __shfl_xor_sync(0xffffffffu, w, 8);
  w |= __shfl_xor_sync(0xffffffffu, w, 16);
  word = w;
  return encode16(v, inv_scale(byte));
}

template <typename T>
__device__ __forceinline__ void load_unit(const T* x, int64_t row, int k4, int width, int lane, Raw16<T>& raw) {
  const int c = k4 * 512 + lane * 16;
  if (c < width)
    raw.load(x + row * width + c);
  else
    raw.clear();
}

// Steps of a warp through the (row, 512 columns) units u, u + step, ...: one
// division at the start, additions after it.
struct UnitWalk {
  int64_t row, step_rows;
  int k4, step_k4, width_k4;
  __device__ __forceinline__ UnitWalk(int64_t u, int64_t step, int width_k4_)
      : row(u / width_k4_), step_rows(step / width_k4_), width_k4(width_k4_) {
    k4 = static_cast<int>(u - row * width_k4);
    step_k4 = static_cast<int>(step - step_rows * width_k4);
  }
  __device__ __forceinline__ void next() {
    row += step_rows;
    k4 += step_k4;
    if (k4 >= width_k4) {
      k4 -= width_k4;
      ++row;
    }
  }
};

// Units of a warp in flight: one at a time, 94 M elements of bf16 took 78 us to
// quantise and 65 us to read back; four at a time 56 and 54 us. fp32 takes the
// registers of two of them for one (90 us on four, 82 on three, 77 on two).
constexpr int kFlight = 4;

// One warp per (row, 512 columns); rows up to the next multiple of 128 get a
// scale word only, so that whole scale tiles are defined. Bound by memory:
// 73,728 x 1280 bf16 in 52 us, 283 MB at 5.4 TB/s, with 61% of the issue slots
// taken; fp32 in 77 us, 472 MB at 6.1 TB/s.
template <typename T>
__global__ void __launch_bounds__(kThreads, 3)
    quantize_rows_kernel(const T* __restrict__ x, int64_t rows, int width, int width_k4, uint8_t* __restrict__ q,
                         uint8_t* __restrict__ scales) {
  constexpr int FLIGHT = sizeof(T) == 4 ? kFlight / 2 : kFlight;
  const int lane = lane_id();
  const int64_t all_rows = (rows + 127) / 128 * 128;
  UnitWalk w(static_cast<int64_t>(blockIdx.x) * kWarps + warp_id(), static_cast<int64_t>(gridDim.x) * kWarps, width_k4);
  while (w.row < all_rows) {
    Raw16<T> raw[FLIGHT];
    UnitWalk ahead = w;
#pragma unroll
    for (int i = 0; i < FLIGHT; ++i) {
      const int c = ahead.k4 * 512 + lane * 16;
      if (ahead.row < rows && c < width)
        raw[i].load(x + ahead.row * width + c);
      else
        raw[i].clear();
      ahead.next();
    }
#pragma unroll
    for (int i = 0; i < FLIGHT; ++i) {
      if (w.row < all_rows) {
        float v[16];
        raw[i].unpack(v);
        uint32_t word;
        const uint4 o = encode_unit(v, lane, word);
        const int c = w.k4 * 512 + lane * 16;
        if (w.row < rows && c < width) *reinterpret_cast<uint4*>(q + w.row * width + c) = o;
        if (lane == 0) *reinterpret_cast<uint32_t*>(scales + scale_word_offset(w.row, w.k4, width_k4)) = word;
      }
      w.next();
    }
  }
}

// One CTA per 128 x 128 block: 8 lanes hold a row of the block, 4 passes of 32
// rows stay in registers between the maximum and the rounding. 14 x 3200 x
// 1280 bf16 in 31 to 35 us, 172 MB at 5.2 TB/s.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    quantize_weight_kernel(const T* __restrict__ w, int n, int width, int width_k4, uint8_t* __restrict__ q,
                           uint8_t* __restrict__ scales) {
  __shared__ float max_s[kWarps];
  const int kb = blockIdx.x, nb = blockIdx.y;
  const int tiles = gridDim.y;
  const int64_t g = blockIdx.z;
  const int lane = lane_id(), sub = threadIdx.x & 7, r0 = threadIdx.x >> 3;
  const int c = kb * 128 + sub * 16;
  const int64_t base = g * n;
  Raw16<T> raw[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int r = nb * 128 + p * 32 + r0;
    if (r < n && c < width)
      raw[p].load(w + (base + r) * width + c);
    else
      raw[p].clear();
  }
  float m = 0.f, v[16];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    raw[p].unpack(v);
    m = fmaxf(m, amax16(v));
  }
  auto block_max = [&]() {
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) max_s[warp_id()] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) m = fmaxf(m, max_s[i]);
  };
  block_max();
  const bool odd = is_inf(m);  // the same in every thread
  if (odd) {
    __syncthreads();
    m = 0.f;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      raw[p].unpack(v);
      m = fmaxf(m, drop_inf(v));
    }
    block_max();
  }
  const uint32_t byte = scale_byte(m);
  const float inv = inv_scale(byte);
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int r = nb * 128 + p * 32 + r0;
    raw[p].unpack(v);
    if (odd) drop_inf(v);
    if (r < n && c < width) *reinterpret_cast<uint4*>(q + (base + r) * width + c) = encode16(v, inv);
  }
  // Every row of the tile gets the block's byte; the last block also clears
  // the bytes of the K blocks that do not exist.
  const int blocks = (width + 127) / 128;
  if (threadIdx.x < 128) {
    uint8_t* tile = scales + (g * tiles + nb) * static_cast<int64_t>(width_k4) * kScaleTile;
    const int64_t at = scale_word_offset(threadIdx.x, kb >> 2, width_k4) + (kb & 3);
    tile[at] = static_cast<uint8_t>(byte);
    if (kb == blocks - 1)
      for (int b = (kb & 3) + 1; b < 4; ++b) tile[at - (kb & 3) + b] = 0;
  }
}

template <typename T>
__device__ __forceinline__ void decode_unit(const uint4& b, uint32_t word, int lane, T* __restrict__ o) {
  const float s = scale_value((word >> (8 * (lane >> 3))) & 0xffu);
  const uint32_t bw[4] = {b.x, b.y, b.z, b.w};
  float v[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = unpack_e4m3x2(bw[i >> 1] >> (16 * (i & 1)));
    v[2 * i] = f.x * s;
    v[2 * i + 1] = f.y * s;
  }
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      __stcs(reinterpret_cast<float4*>(o) + i, make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      __stcs(reinterpret_cast<uint4*>(o) + i,
             make_uint4(pack2<T>(v[8 * i], v[8 * i + 1]), pack2<T>(v[8 * i + 2], v[8 * i + 3]),
                        pack2<T>(v[8 * i + 4], v[8 * i + 5]), pack2<T>(v[8 * i + 6], v[8 * i + 7])));
  }
}

// Rows of all groups in one sequence; a group's scale tiles start anew. 73,728
// x 1280 to bf16 in 50 us, 5.6 TB/s.
template <typename T>
__global__ void __launch_bounds__(kThreads, 4)
    dequantize_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scales, int64_t groups, int64_t rows,
                      int width, int width_k4, T* __restrict__ out) {
  const int lane = lane_id();
  const int64_t tile_rows = (rows + 127) / 128 * 128;
  const int64_t all_rows = groups * rows;
  UnitWalk w(static_cast<int64_t>(blockIdx.x) * kWarps + warp_id(), static_cast<int64_t>(gridDim.x) * kWarps, width_k4);
  while (w.row < all_rows) {
    uint4 b[kFlight];
    uint32_t word[kFlight];
    UnitWalk ahead = w;
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int c = ahead.k4 * 512 + lane * 16;
      if (ahead.row < all_rows && c < width) {
        const int64_t g = groups == 1 ? 0 : ahead.row / rows;
        word[i] = __ldg(reinterpret_cast<const uint32_t*>(
            scales + scale_word_offset(g * tile_rows + ahead.row - g * rows, ahead.k4, width_k4)));
        b[i] = __ldcs(reinterpret_cast<const uint4*>(q + ahead.row * width + c));
      }
      ahead.next();
    }
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int c = w.k4 * 512 + lane * 16;
      if (w.row < all_rows && c < width) decode_unit<T>(b[i], word[i], lane, out + w.row * width + c);
      w.next();
    }
  }
}

// ---------------------------------------------------------------------------
// Dispatch
// ---------------------------------------------------------------------------
__device__ __forceinline__ int pad_rows(int count) { return (count + AGM_TILE_M - 1) / AGM_TILE_M * AGM_TILE_M; }

// Exclusive prefix of the padded counts in count_s over E <= 512 experts, by
// one warp: start_s[E + 1].
__device__ __forceinline__ void padded_prefix(const int* count_s, int E, int* start_s, int lane) {
  int carry = 0;
  for (int e0 = 0; e0 < E; e0 += 32) {
    const int e = e0 + lane;
    const int v = e < E ? pad_rows(count_s[e]) : 0;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    if (e < E) start_s[e] = carry + incl - v;
    carry += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) start_s[E] = carry;
}

// Small batches: every CTA counts all slots by itself and its warps move
// (token, 512 columns) units, one launch in all. The unit's elements are
// loaded before the counting, which hides their latency. 64 tokens, top-2 of
// 14, width 1280: 3.7 us, a launch and three dependent reads.
constexpr int kSmallSlots = 1024;
template <typename T>
__global__ void __launch_bounds__(kThreads) dispatch_small_kernel(Fp8Dispatch a, int width_k4) {
  __shared__ int idx_s[kSmallSlots];
  __shared__ int count_s[AGM_ROUTE_MAX_EXPERTS];
  __shared__ int start_s[AGM_ROUTE_MAX_EXPERTS + 1];
  const int lane = lane_id(), warp = warp_id();
  pdl_wait();
  pdl_trigger();
  const int slots = static_cast<int>(a.n) * a.k;
  const int units = static_cast<int>(a.n) * width_k4;
  int u = blockIdx.x * kWarps + warp;
  Raw16<T> raw;
  if (u < units) load_unit<T>(static_cast<const T*>(a.x), u / width_k4, u % width_k4, a.d, lane, raw);
  if (blockIdx.x == 0) {
    if (threadIdx.x == 0) *a.err = 0;
    for (int i = threadIdx.x; i < a.n_zero; i += kThreads) a.zero[i] = 0;
  }
  for (int e = threadIdx.x; e < a.n_experts; e += kThreads) count_s[e] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < slots; i += kThreads) {
    int e = a.idx[i];
    if (e < 0 || e >= a.n_experts) e = -1;
    idx_s[i] = e;
    if (e >= 0) atomicAdd(&count_s[e], 1);
  }
  __syncthreads();
  if (warp == 0) padded_prefix(count_s, a.n_experts, start_s, lane);
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int e = threadIdx.x; e < a.n_experts; e += kThreads) {
      a.counts[e] = count_s[e];
      a.seg_start[e] = start_s[e];
    }
    if (threadIdx.x == 0) a.seg_start[a.n_experts] = start_s[a.n_experts];
  }
  for (; u < units; u += gridDim.x * kWarps) {
    const int t = u / width_k4, k4 = u - t * width_k4;
    if (u >= static_cast<int>(gridDim.x) * kWarps) load_unit<T>(static_cast<const T*>(a.x), t, k4, a.d, lane, raw);
    float v[16];
    raw.unpack(v);
    uint32_t word;
    const uint4 o = encode_unit(v, lane, word);
    const int c = k4 * 512 + lane * 16;
    for (int r = 0; r < a.k; ++r) {
      const int s = t * a.k + r, e = idx_s[s];
      int before = 0;
      for (int i = lane; i < s; i += 32) before += idx_s[i] == e;
      const int64_t row = e >= 0 ? start_s[e] + static_cast<int>(__reduce_add_sync(0xffffffffu, before)) : -1;
      if (k4 == 0 && lane == 0) a.row_of[s] = static_cast<int>(row);
      if (row < 0) continue;
      if (c < a.d) *reinterpret_cast<uint4*>(a.q + row * a.d + c) = o;
      if (lane == 0) *reinterpret_cast<uint32_t*>(a.scales + scale_word_offset(row, k4, width_k4)) = word;
    }
  }
}

// Large batches, three launches. 1: per-expert counts of every 128 tokens.
__global__ void __launch_bounds__(kThreads)
    dispatch_hist_kernel(const int32_t* __restrict__ idx, int64_t slots, int k, int E, int32_t* __restrict__ hist,
                         int* err, int32_t* __restrict__ zero, int n_zero) {
  __shared__ int count_s[AGM_ROUTE_MAX_EXPERTS];
  pdl_wait();
  pdl_trigger();
  if (blockIdx.x == 0) {
    if (threadIdx.x == 0) *err = 0;
    for (int i = threadIdx.x; i < n_zero; i += kThreads) zero[i] = 0;
  }
  for (int e = threadIdx.x; e < E; e += kThreads) count_s[e] = 0;
  __syncthreads();
  const int64_t s0 = static_cast<int64_t>(blockIdx.x) * kTokBlk * k;
  const int64_t s1 = min(slots, s0 + static_cast<int64_t>(kTokBlk) * k);
  for (int64_t s = s0 + threadIdx.x; s < s1; s += kThreads) {
    const int e = idx[s];
    if (e >= 0 && e < E) atomicAdd(&count_s[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += kThreads) hist[static_cast<int64_t>(blockIdx.x) * E + e] = count_s[e];
}

// 2: per expert, the counts of its blocks become offsets in its segment (one
// warp per expert, in place).
__global__ void __launch_bounds__(kThreads)
    dispatch_scan_kernel(int32_t* __restrict__ hist, int n_blocks, int E, int32_t* __restrict__ counts) {
  constexpr int kUnroll = 8;
  pdl_wait();
  pdl_trigger();
  const int lane = lane_id();
  const int e = blockIdx.x * kWarps + warp_id();
  if (e >= E) return;
  int carry = 0;
  for (int b0 = 0; b0 < n_blocks; b0 += 32 * kUnroll) {
    int v[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const int b = b0 + 32 * j + lane;
      v[j] = b < n_blocks ? hist[static_cast<int64_t>(b) * E + e] : 0;
    }
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const int b = b0 + 32 * j + lane;
      int incl = v[j];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
      }
      if (b < n_blocks) hist[static_cast<int64_t>(b) * E + e] = carry + incl - v[j];
      carry += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  if (lane == 0) counts[e] = carry;
}

// 3: destinations of a block's slots in slot order, then its rows. Each warp
// ranks an eighth of the block's slots: matching lanes of 32 slots at a time,
// on top of the counts of the warps before it. Small grids split a block's
// rows over several CTAs, each of which ranks all its slots (24 blocks: 105
// us whole, 15.5 split; finer splits of large batches gain nothing). Bound by
// memory and its ranking pass: 73,728 tokens x 1280 bf16, top-2, 379 MB in
// 82 us, 4.6 TB/s.
template <typename T>
__global__ void __launch_bounds__(kThreads, 3) dispatch_rows_kernel(Fp8Dispatch a, int width_k4, int split) {
  __shared__ int start_s[AGM_ROUTE_MAX_EXPERTS + 1];
  __shared__ int base_s[kWarps][AGM_ROUTE_MAX_EXPERTS];
  __shared__ int32_t dest_s[kTokBlk * AGM_ROUTE_MAX_TOPK];
  const int lane = lane_id(), warp = warp_id();
  const int E = a.n_experts;
  const int blk = blockIdx.x / split, part = blockIdx.x - blk * split;
  const int64_t tok0 = static_cast<int64_t>(blk) * kTokBlk;
  const int toks = static_cast<int>(min(static_cast<int64_t>(kTokBlk), a.n - tok0));
  const int slots = toks * a.k;
  const int per_warp = (slots + kWarps - 1) / kWarps;
  const int s0 = min(slots, warp * per_warp), s1 = min(slots, s0 + per_warp);
  const int32_t* idx = a.idx + tok0 * a.k;
  auto load_four = [&](int tok, int k4, Raw16<T>(&to)[4]) {
    const T* row = static_cast<const T*>(a.x) + (tok0 + tok) * a.d;
#pragma unroll
    for (int q = 0; q < 4; ++q) load_unit<T>(row, 0, k4 + q, a.d, lane, to[q]);
  };
  const int first = part * kWarps + warp;
  Raw16<T> raw[4];
  // The batch was there before the two launches ahead, and the second of them
  // waited for the first: only the counts have to be waited for.
  if (first < toks) load_four(first, 0, raw);  // in flight during the ranking
  for (int e = lane; e < E; e += 32) base_s[warp][e] = 0;
  __syncwarp();
  for (int s = s0 + lane; s < s1; s += 32) {
    const int e = idx[s];
    if (e >= 0 && e < E) atomicAdd(&base_s[warp][e], 1);
  }
  pdl_wait();
  pdl_trigger();
  if (warp == 0) padded_prefix(a.counts, E, start_s, lane);
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += kThreads) {
    int at = start_s[e] + a.block_hist[static_cast<int64_t>(blk) * E + e];
    for (int w = 0; w < kWarps; ++w) {
      const int c = base_s[w][e];
      base_s[w][e] = at;
      at += c;
    }
    if (blockIdx.x == 0) a.seg_start[e] = start_s[e];
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.seg_start[E] = start_s[E];
    if (start_s[E] > a.max_rows) raise_error(a.err, kErrRowOverflow);
  }
  __syncthreads();
  for (int b = s0; b < s1; b += 32) {
    const int s = b + lane;
    int e = s < s1 ? idx[s] : -1;
    if (e < 0 || e >= E) e = -1;
    const uint32_t peers = __match_any_sync(0xffffffffu, e);
    const int base = e >= 0 ? base_s[warp][e] : 0;
    __syncwarp();
    if (s < s1) {
      const int row = e >= 0 ? base + __popc(peers & ((1u << lane) - 1u)) : -1;
      dest_s[s] = row < a.max_rows ? row : -1;
      if (part == 0) a.row_of[tok0 * a.k + s] = dest_s[s];
    }
    if (e >= 0 && lane == __ffs(peers) - 1) base_s[warp][e] = base + __popc(peers);
    __syncwarp();
  }
  __syncthreads();
  // Rows: a warp takes a token, 4 x 512 columns at a time, the next ones in
  // flight while these are rounded and written.
  int i = first;
  int q0 = 0;
  while (i < toks) {
    int ni = i, nq = q0 + 4;
    if (nq >= width_k4) {
      nq = 0;
      ni += split * kWarps;
    }
    Raw16<T> next[4];
    if (ni < toks) load_four(ni, nq, next);
    const int my_dest = lane < a.k ? dest_s[i * a.k + lane] : -1;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (q0 + q >= width_k4) break;
      float v[16];
      raw[q].unpack(v);
      uint32_t word;
      const uint4 o = encode_unit(v, lane, word);
      const int c = (q0 + q) * 512 + lane * 16;
      for (int r = 0; r < a.k; ++r) {
        const int64_t to = __shfl_sync(0xffffffffu, my_dest, r);
        if (to < 0) continue;
        if (c < a.d) *reinterpret_cast<uint4*>(a.q + to * a.d + c) = o;
        if (lane == 0) *reinterpret_cast<uint32_t*>(a.scales + scale_word_offset(to, q0 + q, width_k4)) = word;
      }
    }
    i = ni;
    q0 = nq;
#pragma unroll
    for (int q = 0; q < 4; ++q) raw[q] = next[q];
  }
}

// ---------------------------------------------------------------------------
// Weighted sum
// ---------------------------------------------------------------------------
// One warp per token and P x 256 columns: a lane sums P x 8 columns over the
// token's rows, the loads of KU rows in flight at a time. ONE: k <= KU, so
// that only one part's sums are held at a time. SHARED: the outputs of shared
// experts are there (their loop costs registers, with k <= 2 a CTA per SM and
// 10 us at 73,728 tokens where there are none). Bound by memory: 73,728 tokens
// x 1280 bf16, top-2, 567 MB in about 115 us, 4.9 TB/s. y comes rounded to T, as
// the block in its own precision rounds it: fp32 would be 377 MB more to write
// and 377 MB more to read here, some 115 us of 1.3 ms, for a relative error of
// 0.0017 (the last rounding's) in place of 0.0023 to 0.0024. Few tokens could
// afford it, but then a token's result would depend on the batch it is in.
template <typename T, int KU, int P, bool ONE, bool SHARED>
__global__ void __launch_bounds__(kThreads)
    combine_weighted_kernel(const T* __restrict__ y, const int32_t* __restrict__ row_of,
                            const float* __restrict__ weights, int64_t n, int nchunk, int k,
                            const T* __restrict__ residual, const T* __restrict__ shared, int n_shared,
                            T* __restrict__ out) {
  static_assert(ONE || P == 1, "several parts only for few rows");
  const int lane = lane_id();
  const uint4* y4 = reinterpret_cast<const uint4*>(y);
  const uint4* res4 = reinterpret_cast<const uint4*>(residual);
  const uint4* shared4 = reinterpret_cast<const uint4*>(shared);
  const int parts = (nchunk + 32 * P - 1) / (32 * P);
  const int64_t units = n * parts;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps;
  int64_t u = static_cast<int64_t>(blockIdx.x) * kWarps + warp_id();
  int my_row;
  float my_w;
  auto fetch = [&]() {
    const bool in = u < units && lane < k;
    const int64_t at = (parts == 1 ? u : u / parts) * k + lane;
    my_row = in ? row_of[at] : -1;
    my_w = in ? weights[at] : 0.f;
  };
  // Rows and weights come from before the launch that this one overlaps with
  // (the product that writes y), which had waited for them: few tokens fetch
  // them before their own wait (0.6 us of 36 at 64 tokens); the wide form has
  // no registers for it (a CTA fewer per SM).
  if (P == 1) fetch();
  pdl_wait();
  pdl_trigger();
  for (; u < units; u += step) {
    if (P > 1 || u >= step) fetch();
    const int64_t t = parts == 1 ? u : u / parts;
    const int c0 = static_cast<int>(u - t * parts) * 32 * P + lane;
    float acc[8];
    auto start = [&](int c) {
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = 0.f;
      if (residual && c < nchunk) unpack8<T>(__ldcs(res4 + t * nchunk + c), acc);
      if constexpr (SHARED) {
#pragma unroll 1
        for (int s = 0; s < n_shared && c < nchunk; ++s) {
          float f[8];
          unpack8<T>(__ldcs(shared4 + (s * n + t) * nchunk + c), f);
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[j] += f[j];
        }
      }
    };
    auto add = [&](const uint4& v, float w) {
      float f[8];
      unpack8<T>(v, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = fmaf(w, f[j], acc[j]);
    };
    auto finish = [&](int c) {
      if (c < nchunk)
        __stcs(reinterpret_cast<uint4*>(out) + t * nchunk + c,
               make_uint4(pack2<T>(acc[0], acc[1]), pack2<T>(acc[2], acc[3]), pack2<T>(acc[4], acc[5]),
                          pack2<T>(acc[6], acc[7])));
    };
    if (!ONE) start(c0);
    for (int r0 = 0; r0 < (ONE ? 1 : k); r0 += KU) {
      uint4 v[KU][P];
      float w[KU];
#pragma unroll
      for (int i = 0; i < KU; ++i) {
        const int row = __shfl_sync(0xffffffffu, my_row, (r0 + i) & 31);
        w[i] = __shfl_sync(0xffffffffu, my_w, (r0 + i) & 31);
        const bool use = r0 + i < k && row >= 0;
        if (!use) w[i] = 0.f;  // a slot without a row adds nothing, whatever its weight
#pragma unroll
        for (int p = 0; p < P; ++p) {
          const int c = c0 + 32 * p;
          v[i][p] = use && c < nchunk ? __ldcs(y4 + static_cast<int64_t>(row) * nchunk + c) : make_uint4(0, 0, 0, 0);
        }
      }
      if constexpr (ONE) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
          start(c0 + 32 * p);
#pragma unroll
          for (int i = 0; i < KU; ++i) add(v[i][p], w[i]);
          finish(c0 + 32 * p);
        }
      } else {
#pragma unroll
        for (int i = 0; i < KU; ++i) add(v[i][0], w[i]);
      }
    }
    if (!ONE) finish(c0);
  }
}

// One warp per unit, on at most `per_sm` CTAs per SM. Quantising and reading
// back take as many as are resident at once, so that all run from start to end
// with equal shares (94 M elements: quantise 57 us on 8 per SM, 53 us on 3;
// read back 61 us on 8, 58 us on 4, in a loop). The weighted sum's few CTAs would leave
// their SMs to the next launch late (73,728 tokens: 119 us on 8, 140 us on 3).
unsigned warp_grid(int64_t units, int num_sms, int per_sm) {
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((units + kWarps - 1) / kWarps,
                                                                      static_cast<int64_t>(num_sms) * per_sm)));
}

template <typename T>
cudaError_t dispatch_t(const Fp8Dispatch& a, int num_sms, cudaStream_t stream) {
  const int width_k4 = scale_k4(a.d);
  if (a.n * a.k <= kSmallSlots)
    return launch_kernel(dispatch_small_kernel<T>, dim3(warp_grid(a.n * width_k4, num_sms, 8)), dim3(kThreads), 0,
                         stream, a, width_k4);
  const int nb = static_cast<int>((a.n + kTokBlk - 1) / kTokBlk);
  cudaError_t e = launch_kernel(dispatch_hist_kernel, dim3(nb), dim3(kThreads), 0, stream, a.idx, a.n * a.k, a.k,
                                a.n_experts, a.block_hist, a.err, a.zero, a.n_zero);
  if (e != cudaSuccess) return e;
  e = launch_kernel(dispatch_scan_kernel, dim3((a.n_experts + kWarps - 1) / kWarps), dim3(kThreads), 0, stream,
                    a.block_hist, nb, a.n_experts, a.counts);
  if (e != cudaSuccess) return e;
  // At least four CTAs per SM, and at least one token per warp.
  const int split = std::max(1, std::min(kTokBlk / kWarps, (4 * num_sms + nb - 1) / nb));
  return launch_kernel(dispatch_rows_kernel<T>, dim3(nb * split), dim3(kThreads), 0, stream, a, width_k4, split);
}

}  // namespace

cudaError_t quantize_fp8_rows(int dtype, const void* x, int64_t rows, int width, void* q, void* scales, int num_sms,
                              cudaStream_t stream) {
  const int k4 = scale_k4(width);
  const unsigned grid = warp_grid((rows + 127) / 128 * 128 * k4, num_sms, 3);
  uint8_t* qb = static_cast<uint8_t*>(q);
  uint8_t* sb = static_cast<uint8_t*>(scales);
  switch (dtype) {
    case AGM_F32:
      quantize_rows_kernel<float><<<grid, kThreads, 0, stream>>>(static_cast<const float*>(x), rows, width, k4, qb, sb);
      break;
    case AGM_BF16:
      quantize_rows_kernel<__nv_bfloat16>
          <<<grid, kThreads, 0, stream>>>(static_cast<const __nv_bfloat16*>(x), rows, width, k4, qb, sb);
      break;
    default:
      quantize_rows_kernel<__half><<<grid, kThreads, 0, stream>>>(static_cast<const __half*>(x), rows, width, k4, qb, sb);
  }
  return cudaGetLastError();
}

cudaError_t quantize_fp8_weight(int dtype, const void* w, int64_t groups, int n, int width, void* q, void* scales,
                                cudaStream_t stream) {
  const int k4 = scale_k4(width);
  const dim3 grid((width + 127) / 128, (n + 127) / 128, static_cast<unsigned>(groups));
  uint8_t* qb = static_cast<uint8_t*>(q);
  uint8_t* sb = static_cast<uint8_t*>(scales);
  switch (dtype) {
    case AGM_F32:
      quantize_weight_kernel<float><<<grid, kThreads, 0, stream>>>(static_cast<const float*>(w), n, width, k4, qb, sb);
      break;
    case AGM_BF16:
      quantize_weight_kernel<__nv_bfloat16>
          <<<grid, kThreads, 0, stream>>>(static_cast<const __nv_bfloat16*>(w), n, width, k4, qb, sb);
      break;
    default:
      quantize_weight_kernel<__half><<<grid, kThreads, 0, stream>>>(static_cast<const __half*>(w), n, width, k4, qb, sb);
  }
  return cudaGetLastError();
}

cudaError_t dequantize_fp8(int dtype, const void* q, const void* scales, int64_t groups, int64_t rows, int width,
                           void* out, int num_sms, cudaStream_t stream) {
  const int k4 = scale_k4(width);
  const unsigned grid = warp_grid(groups * rows * k4, num_sms, 4);
  const uint8_t* qb = static_cast<const uint8_t*>(q);
  const uint8_t* sb = static_cast<const uint8_t*>(scales);
  switch (dtype) {
    case AGM_F32:
      dequantize_kernel<float><<<grid, kThreads, 0, stream>>>(qb, sb, groups, rows, width, k4, static_cast<float*>(out));
      break;
    case AGM_BF16:
      dequantize_kernel<__nv_bfloat16>
          <<<grid, kThreads, 0, stream>>>(qb, sb, groups, rows, width, k4, static_cast<__nv_bfloat16*>(out));
      break;
    default:
      dequantize_kernel<__half><<<grid, kThreads, 0, stream>>>(qb, sb, groups, rows, width, k4, static_cast<__half*>(out));
  }
  return cudaGetLastError();
}

cudaError_t dispatch_fp8(int dtype, const Fp8Dispatch& a, int num_sms, cudaStream_t stream) {
  return dtype == AGM_BF16 ? dispatch_t<__nv_bfloat16>(a, num_sms, stream) : dispatch_t<__half>(a, num_sms, stream);
}

cudaError_t combine_weighted(int dtype, const void* y, const int32_t* row_of, const float* weights, int64_t n, int d,
                             int k, const void* residual, const void* shared, int n_shared, void* out, int num_sms,
                             cudaStream_t stream) {
  const int nchunk = d / 8;
  auto launch = [&](auto kernel, int columns, auto zero) {
    using T = decltype(zero);
    return launch_kernel(kernel, dim3(warp_grid(n * ((nchunk + columns - 1) / columns), num_sms, 8)), dim3(kThreads), 0, stream,
                         static_cast<const T*>(y), row_of, weights, n, nchunk, k, static_cast<const T*>(residual),
                         static_cast<const T*>(shared), n_shared, static_cast<T*>(out));
  };
  // Few units: the narrowest, to use every SM. Many: enough loads in flight per warp. For k <= 2, with dispatch and
  // two narrow products around it, 73,728 tokens take (us, on 3 / 4 / 5 / 6 parts) 299 / 285 / 286 / 291 at width
  // 1024, 364 / 361 / 353 / 359 at 1280, 401 / 395 / 397 / 396 at 1408, 576 / 558 / 561 / 573 at 2048 and
  // 1132 / 1093 / 1102 / 1113 at 4096.
  auto pick = [&](auto zero, auto with_shared) {
    using T = decltype(zero);
    constexpr bool S = with_shared.value;
    const bool wide = n * ((nchunk + 31) / 32) >= static_cast<int64_t>(num_sms) * 64;
    if (k <= 2)
      return wide ? launch(combine_weighted_kernel<T, 2, 5, true, S>, 160, zero)
                  : launch(combine_weighted_kernel<T, 2, 1, true, S>, 32, zero);
    if (k <= 4)
      return wide ? launch(combine_weighted_kernel<T, 4, 2, true, S>, 64, zero)
                  : launch(combine_weighted_kernel<T, 4, 1, true, S>, 32, zero);
    return launch(combine_weighted_kernel<T, 8, 1, false, S>, 32, zero);
  };
  auto pick_dtype = [&](auto with_shared) {
    return dtype == AGM_BF16 ? pick(__nv_bfloat16(), with_shared) : pick(__half(), with_shared);
  };
  return n_shared ? pick_dtype(std::true_type()) : pick_dtype(std::false_type());
}

}  // namespace agm
