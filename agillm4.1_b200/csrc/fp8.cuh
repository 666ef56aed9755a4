// Device helpers of the block-scaled 8-bit floating point path: the e4m3 block
// format and the tcgen05 forms that multiply it.
//
// Format. A matrix [rows, width] is stored as e4m3 bytes, row-major, with one
// power-of-two scale per block of 128 consecutive elements of a row (weights:
// per 128 x 128 block, written once for each of its rows). The scale is the
// exponent p biased by 127 in one byte (E8M0); an element stands for q * 2^p.
// p is the least integer with amax <= 448 * 2^p, so a block uses the whole
// e4m3 range and x * 2^-p is exact: the only rounding is e4m3's own.
//
// Scale tiles. The tensor core reads scales from tensor memory as 32 lanes x
// 32-bit words, word = 4 consecutive K blocks of one row, the row's four
// 32-row groups side by side. Memory holds exactly that image: for every 128
// rows and every 4 K blocks one 512-byte tile, row r and block b at byte
// 16 * (r % 32) + 4 * (r % 128 / 32) + b % 4, tiles ordered [row tile][b / 4].
// So a tile goes from global memory to tensor memory without being touched.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace agm {

constexpr int kFp8Block = 128;      // elements per scale
constexpr int kScaleTile = 512;     // bytes of one scale tile

__host__ __device__ __forceinline__ int scale_k4(int width) { return (width + 4 * kFp8Block - 1) / (4 * kFp8Block); }

// Byte offset of row r's scale word (4 K blocks) in the scale tiles of a matrix.
__device__ __forceinline__ int64_t scale_word_offset(int64_t r, int k4, int width_k4) {
  const int rr = static_cast<int>(r & 127);
  return ((r >> 7) * width_k4 + k4) * kScaleTile + (rr & 31) * 16 + (rr >> 5) * 4;
}

// Biased exponent of the least power of two s with amax <= 448 s (448 = 1.75 * 2^8),
// for a finite amax >= 0; never below 2^-127.
__device__ __forceinline__ uint32_t scale_byte(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = static_cast<int>(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return static_cast<uint32_t>(max(e, 0));
}
// 2^-(byte - 127): exact for every byte scale_byte returns (0 .. 247).
__device__ __forceinline__ float inv_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// 2^(byte - 127); byte 0 is the subnormal 2^-127.
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __uint_as_float(byte ? byte << 23 : 0x00400000u);
}

// |v| for the block maximum: what has no e4m3 form (NaN, infinities) does not
// set the scale of its neighbours.
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a < __uint_as_float(0x7f800000u) ? a : 0.f;  // false for NaN
}
// Infinities become NaN (e4m3 has none and would turn them into +-448).
__device__ __forceinline__ float inf_to_nan(float v) {
  return fabsf(v) == __uint_as_float(0x7f800000u) ? __uint_as_float(0x7fc00000u) : v;
}
// 4 scaled values -> 4 e4m3 bytes (round to nearest even), first in the low byte.
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ float2 unpack_e4m3x2(uint32_t v) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v & 0xffffu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));  // every e4m3 value is a half
}

// Packed fp32 pairs (one instruction for two adds or products).
__device__ __forceinline__ void add2(uint32_t& x, uint32_t& y, float a, float b) {
  asm("{\n\t.reg .b64 v, w;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 w, {%2, %3};\n\tadd.rn.f32x2 v, v, w;\n\t"
      "mov.b64 {%0, %1}, v;\n\t}"
      : "+r"(x), "+r"(y)
      : "f"(a), "f"(b));
}
__device__ __forceinline__ void scale2(uint32_t& x, uint32_t& y, float s) {
  asm("{\n\t.reg .b64 v, w;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 w, {%2, %2};\n\tmul.rn.f32x2 v, v, w;\n\t"
      "mov.b64 {%0, %1}, v;\n\t}"
      : "+r"(x), "+r"(y)
      : "f"(s));
}
// max(v, 0) that keeps NaN.
__device__ __forceinline__ float relu_keep_nan(float v) {
  float o;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(o) : "f"(v));
  return o;
}

// One lane of the converged warp. The compiler issues tcgen05 and TMA
// instructions behind it once; behind `lane == 0` it loops over the active
// lanes around every one of them, which held the MMA issue to 2.06 PFLOP/s
// where it now reaches 2.47 (rows kernel, 75,776 x 3200 by 1280 x 3200).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(p)
      :
      : "memory");
  return p != 0;
}

// Arrive on an mbarrier of another CTA of the cluster (cluster address). It
// orders this CTA's work only: a release at cluster scope also waits for the
// thread's outstanding global stores, over a microsecond in an epilogue.
__device__ __forceinline__ void mbar_arrive_peer(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cta.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// ---------------------------------------------------------------------------
// tcgen05 with block scales
// ---------------------------------------------------------------------------
// Instruction descriptor, kind::mxf8f6f4: B scale byte of the word at bits
// 4-5, A and B format e4m3 (bits 7-9, 10-12 = 0), both K-major, N >> 3 at bits
// 17-22, E8M0 scales (bit 23), M >> 4 at bits 24-28, A scale byte at 29-30.
__host__ __device__ constexpr uint32_t idesc_mxf8(int M, int N, int sf) {
  return (static_cast<uint32_t>(sf) << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (1u << 23) |
         (static_cast<uint32_t>(M >> 4) << 24) | (static_cast<uint32_t>(sf) << 29);
}

// Shared-memory descriptor of a scale tile for tcgen05.cp.32x128b: 32 rows of
// 16 bytes, no swizzle, 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_scale(uint32_t smem_addr) {
  return static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(128u >> 4) << 32) |
         (static_cast<uint64_t>(1u) << 46);
}

// Scale tile in shared memory -> 4 columns of tensor memory (in all four
// 32-lane groups), in order with the MMAs the same thread issues after it.
template <int GROUP>
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint64_t desc) {
  if constexpr (GROUP == 2)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// D (+)= (A * 2^pa) (B * 2^pb)^T over K = 32, scales from tensor memory.
template <int GROUP>
__device__ __forceinline__ void umma_mxf8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if constexpr (GROUP == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

}  // namespace agm
