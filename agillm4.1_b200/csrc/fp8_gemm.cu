// Grouped product of block-scaled e4m3 operands on the 5th-generation tensor
// cores:
//
//   c[r, n] = act( sum_k a[r, k] w[g(r), n, k] + bias[g(r), n] )
//
// kind::mxf8f6f4 multiplies e4m3 by e4m3 and applies the blocks' power-of-two
// scales inside the tensor core (one scale per 32 elements of K; a block of
// 128 uses its scale four times), accumulating in fp32. So the scales cost no
// arithmetic outside the MMA: a 512-byte scale tile per 128 rows and 512
// elements of K rides along with the operands (TMA to shared memory,
// tcgen05.cp to tensor memory) and a k-block selects its byte of the word
// through the instruction descriptor.
//
// Two kernels:
//
// * fp8_rows_kernel, many rows per group (bound by the tensor cores): a
//   cluster of two CTAs computes 256 rows x 256 columns with cta_group::2.
//   Each CTA loads its own 128 rows of a and half of the weight tile, 32 KB
//   per 128-deep k-block and CTA. Two 256-column accumulators and the scales
//   do not fit in the 512 columns of tensor memory, so the accumulators
//   overlap in 32 columns (0..255 and 224..479): the epilogue takes a tile's
//   128 columns per warp into registers at once and releases the shared
//   columns first, so the next tile waits for that load and not for the
//   epilogue's arithmetic.
//
// * fp8_weights_kernel, few rows per group (bound by reading the weights): the
//   weight tile is the 128-row operand and the group's rows the N operand (32
//   of them, or up to 128), so no bandwidth goes to padding rows and the ring
//   of stages keeps 144 KB of weights in flight per SM.
//
// Both walk units numbered from the device-side row counts (no host sync;
// empty groups cost nothing), are persistent and warp-specialised (warp 0 TMA,
// warp 1 MMA, warps 2-9 epilogue), bound every wait, and can write their
// result as e4m3 blocks: 128 output columns of a row are one block, which an
// epilogue thread (rows kernel) or warp (weights kernel) has whole, so the
// quantisation of the next product's input costs no pass over memory.
#include <algorithm>

#include "fp8.cuh"
#include "kernels.h"

namespace agm {

namespace {

constexpr int kBK = 128;              // e4m3 elements (and bytes) per k-block: one 128-byte swizzled row
constexpr int kEpi = 8;
constexpr int kThreads = 64 + 32 * kEpi;
constexpr int kMaxGroups = AGM_ROUTE_MAX_EXPERTS;

// ---- rows kernel ----
constexpr int kPN = 256;                      // columns per pair tile
constexpr int kPStages = 5;
constexpr int kPA = 128 * kBK;                // 16 KB
constexpr int kPB = 128 * kBK;                // 16 KB: half of the weight tile
constexpr int kPSf = 3 * kScaleTile;          // scale tiles of a stage: a, and both halves of w
constexpr int kPStg = 32 * 128;               // output chunk of one epilogue warp
constexpr int kPBias = 128 * 4;               // its bias values
constexpr int kAccStep = kPN - 32;            // second accumulator's first column
constexpr int kSfCol = kAccStep + kPN;        // 480: two slots of 16 columns
constexpr int kGroupPairs = 8;                // rasterisation: 8 row blocks per group of column tiles
constexpr int kPSmem = kPStages * (kPA + kPB + kPSf) + kEpi * (kPStg + kPBias) + 256 + 1024;
static_assert(kPSmem + kMaxGroups * 12 + 16 <= 227 * 1024, "rows kernel shared memory");

// ---- weights kernel ----
template <int ROWS>
struct SwapCfg {
  static constexpr int kStages = ROWS == 32 ? 9 : 6;
  static constexpr int kW = 128 * kBK;
  static constexpr int kA = ROWS * kBK;
  static constexpr int kSf = 2 * kScaleTile;
  static constexpr int kStgLd = 132;          // floats per staged row
  static constexpr int kStg = 32 * kStgLd * 4;
  static constexpr int kTmemCols = ROWS == 32 ? 128 : 512;
  static constexpr int kSfCol = 2 * ROWS;
  static constexpr int kSmem = kStages * (kW + kA + kSf) + kStg + 512 + 1024;
};

// Row counts and starts of the groups, checked, and the prefix sum of their
// blocks of `ROWS` rows.
struct Groups {
  int count[kMaxGroups];
  int start[kMaxGroups];
  int first[kMaxGroups + 1];
};

__device__ __forceinline__ void load_groups(const Fp8GemmArgs& args, int block_rows, Groups& s) {
  // All threads; the caller synchronises.
  for (int g = threadIdx.x; g < args.groups; g += blockDim.x) {
    int64_t c = args.counts ? args.counts[g] : args.a_rows;
    int64_t r = args.counts ? args.seg_start[g] : 0;
    if (c < 0 || (c > 0 && (r < 0 || (r & 127) || r + c > args.a_rows))) {
      if (blockIdx.x == 0) raise_error(args.err, kErrRowOverflow);
      c = 0;
    }
    s.count[g] = static_cast<int>(c);
    s.start[g] = static_cast<int>(r);
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int carry = 0;
    for (int g0 = 0; g0 < args.groups; g0 += 32) {
      const int g = g0 + lane;
      const int v = g < args.groups ? (s.count[g] + block_rows - 1) / block_rows : 0;
      int incl = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
      }
      if (g < args.groups) s.first[g] = carry + incl - v;
      carry += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) s.first[args.groups] = carry;
  }
}

// Group of block b (first[g] <= b < first[g + 1]).
__device__ __forceinline__ int find_group(const Groups& s, int groups, int b) {
  int lo = 0, hi = groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s.first[mid] <= b)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

struct Unit {
  int g;      // weight group
  int row0;   // first row
  int valid;  // rows of the group from row0 on
  int nb;     // column tile
};

__device__ __forceinline__ Unit rows_unit(const Groups& s, int groups, int t, int num_p, int num_n) {
  const int span = kGroupPairs * num_n;
  const int grp = t / span;
  const int first = grp * kGroupPairs;
  const int gp = min(num_p - first, kGroupPairs);
  const int r = t - grp * span;
  const int b = first + r % gp;
  Unit u;
  u.nb = r / gp;
  u.g = find_group(s, groups, b);
  const int j = b - s.first[u.g];
  u.row0 = s.start[u.g] + j * 256;
  u.valid = s.count[u.g] - j * 256;
  return u;
}

template <int ROWS>
__device__ __forceinline__ Unit weights_unit(const Groups& s, int groups, int t, int num_n) {
  const int b = t / num_n;
  Unit u;
  u.nb = t - b * num_n;
  u.g = find_group(s, groups, b);
  const int j = b - s.first[u.g];
  u.row0 = s.start[u.g] + j * ROWS;
  u.valid = s.count[u.g] - j * ROWS;
  return u;
}

// OUT: __nv_bfloat16, __half, or __nv_fp8_e4m3 (block-scaled output).
template <typename OUT, bool RELU>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    fp8_rows_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmSA,
                    const __grid_constant__ CUtensorMap tmSB, const __grid_constant__ CUtensorMap tmA32,
                    Fp8GemmArgs args) {
  constexpr bool OUT8 = sizeof(OUT) == 1;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Groups grp;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + kPStages * kPA;
  uint8_t* sStg = sB + kPStages * kPB;
  uint8_t* sSf = sStg + kEpi * kPStg;
  float* sBias = reinterpret_cast<float*>(sSf + kPStages * kPSf);
  uint64_t* full = reinterpret_cast<uint64_t*>(sBias + kEpi * kPBias / 4);  // rank 0's are used
  uint64_t* empty = full + kPStages;                                    // both ranks
  uint64_t* acc_full = empty + kPStages;                                // both ranks
  uint64_t* acc_empty = acc_full + 2;                                   // rank 0's are used, as the rest
  uint64_t* shared_cols = acc_empty + 2;                                // the accumulators' common columns are free
  uint64_t* sf_done = shared_cols + 1;                                  // MMAs of a scale slot have completed
  uint64_t* drain = sf_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id(), lane = lane_id();
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int cluster = static_cast<int>(cluster_id_x());
  const int nclusters = static_cast<int>(cluster_count_x());

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 2 * kEpi);
      mbar_init(&sf_done[i], 1);
    }
    mbar_init(shared_cols, kEpi);
    mbar_init(drain, 1);
    *abort_s = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmC);
    tma_prefetch_desc(&tmSA);
    tma_prefetch_desc(&tmSB);
  }
  pdl_wait();
  pdl_trigger();
  load_groups(args, 256, grp);
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist before any cross-CTA arrive or copy
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int num_p = grp.first[args.groups];
  const int num_n = (args.n + kPN - 1) / kPN;
  const int total = num_p * num_n;
  const int num_kb = (args.k + kBK - 1) / kBK;
  const int w_tiles = (args.n + 127) / 128;

  if (warp == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    const uint32_t full0 = cluster_map(smem_u32(full), 0);
    int stage = 0;
    uint32_t phase = 0, armed = 0, armed_parity = 0;
    bool ok = true;
    for (int t = cluster; t < total && ok; t += nclusters) {
      const Unit u = rows_unit(grp, args.groups, t, num_p, num_n);
      // Rank 1 loads the block's second 128 rows. Of a block that the group
      // does not fill only the 32-row boxes with live rows are loaded: what
      // stays in shared memory for the others reaches their own results only.
      const int a_row = u.row0 + (leader ? 0 : 128);
      const int boxes0 = min(4, (u.valid + 31) / 32), boxes1 = max(0, min(4, (u.valid - 97) / 32));
      const int boxes = leader ? boxes0 : boxes1;
      const uint32_t bytes = 2 * kPB + (boxes0 + boxes1) * 32 * kBK;
      const uint32_t sf_bytes = 4 * kScaleTile + (boxes0 ? kScaleTile : 0) + (boxes1 ? kScaleTile : 0);
      const int n_mma = min(kPN, (args.n - u.nb * kPN + 31) / 32 * 32);
      const int b_row = u.nb * kPN + static_cast<int>(rank) * (n_mma / 2);
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1, args.err, kErrTimeoutEmpty) || *abort_s) {
          *abort_s = 1;
          ok = false;
          break;
        }
        if (elect_one()) {
          const bool sf = (kb & 3) == 0;
          if (leader) mbar_arrive_expect_tx(&full[stage], bytes + (sf ? sf_bytes : 0));
          const uint32_t fb = full0 + stage * 8;
          tma_load_3d_pair(sB + stage * kPB, &tmB, kb * kBK, b_row, u.g, fb);
          if (boxes == 4)
            tma_load_2d_pair(sA + stage * kPA, &tmA, kb * kBK, a_row, fb);
          else
            for (int i = 0; i < boxes; ++i)
              tma_load_2d_pair(sA + stage * kPA + i * 32 * kBK, &tmA32, kb * kBK, a_row + 32 * i, fb);
          if (sf) {
            uint8_t* dst = sSf + stage * kPSf;
            if (boxes) tma_load_3d_pair(dst, &tmSA, 0, kb >> 2, a_row >> 7, fb);
            tma_load_3d_pair(dst + kScaleTile, &tmSB, 0, kb >> 2, u.g * w_tiles + 2 * u.nb, fb);
          }
        }
        armed |= 1u << stage;
        armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
        __syncwarp();
        if (++stage == kPStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    __syncwarp();
    bool drained = true;
    for (int s = 0; s < kPStages && drained; ++s)
      if (armed & (1u << s)) drained = mbar_wait(&empty[s], (armed_parity >> s) & 1, args.err, kErrTimeoutDrain);
  } else if (warp == 1) {
    if (leader) {
      // ---------------- MMA issuer (rank 0) ----------------
      const uint32_t sA_addr = smem_u32(sA), sB_addr = smem_u32(sB), sSf_addr = smem_u32(sSf);
      int stage = 0, it = 0, sf_use = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = cluster; t < total && ok; t += nclusters, ++it) {
        const Unit u = rows_unit(grp, args.groups, t, num_p, num_n);
        const int n_mma = min(kPN, (args.n - u.nb * kPN + 31) / 32 * 32);
        const int acc = it & 1;
        // Two tiles back: the whole accumulator; the tile before: the common columns.
        if (!mbar_wait(&acc_empty[acc], ((it >> 1) & 1) ^ 1, args.err, kErrTimeoutAcc) ||
            (it > 0 && !mbar_wait(shared_cols, (it - 1) & 1, args.err, kErrTimeoutAcc)) || *abort_s) {
          *abort_s = 1;
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * kAccStep;
        uint32_t sfa = 0, sfb = 0;
        int slot = 0;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&full[stage], phase, args.err, kErrTimeoutFull) || *abort_s) {
            *abort_s = 1;
            ok = false;
            break;
          }
          if ((kb & 3) == 0) {
            slot = sf_use & 1;
            if (sf_use >= 2 && !mbar_wait(&sf_done[slot], ((sf_use >> 1) - 1) & 1, args.err, kErrTimeoutAcc)) {
              *abort_s = 1;
              ok = false;
              break;
            }
            ++sf_use;
            sfa = tmem_base + kSfCol + slot * 16;
            sfb = sfa + 4;
          }
          tc_fence_after();
          if (elect_one()) {
            if ((kb & 3) == 0) {
              const uint32_t src = sSf_addr + stage * kPSf;
              tmem_copy_scales<2>(sfa, smem_desc_scale(src));
              tmem_copy_scales<2>(sfb, smem_desc_scale(src + kScaleTile));
              tmem_copy_scales<2>(sfb + 4, smem_desc_scale(src + 2 * kScaleTile));
            }
            const uint64_t a_desc = smem_desc_k_sw128(sA_addr + stage * kPA);
            const uint64_t b_desc = smem_desc_k_sw128(sB_addr + stage * kPB);
            const uint32_t idesc = idesc_mxf8(256, n_mma, kb & 3);
#pragma unroll
            for (int kk = 0; kk < kBK / 32; ++kk)
              umma_mxf8<2>(d_tmem, a_desc + 2 * kk, b_desc + 2 * kk, idesc, sfa, sfb, (kb > 0 || kk > 0) ? 1u : 0u);
            umma_commit_pair(&empty[stage], 0x3);
            if ((kb & 3) == 3 || kb == num_kb - 1) umma_commit_pair(&sf_done[slot], 0x1);
            if (kb == num_kb - 1) umma_commit_pair(&acc_full[acc], 0x3);
          }
          __syncwarp();
          if (++stage == kPStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (elect_one()) umma_commit_pair(drain, 0x1);
      __syncwarp();
      mbar_wait(drain, 0, args.err, kErrTimeoutDrain);
    }
  } else {
    // ---------------- Epilogue (warps 2..9, both CTAs) ----------------
    const int ew = warp - 2;
    const int quarter = warp & 3;
    const int half = ew >> 2;  // columns [128 * half, + 128) of the tile
    uint8_t* stg = sStg + ew * kPStg;
    const uint32_t acc_empty0 = cluster_map(smem_u32(acc_empty), 0);
    const uint32_t shared0 = cluster_map(smem_u32(shared_cols), 0);
    const int out_k4 = scale_k4(args.n);
    int it = 0;
    for (int t = cluster; t < total; t += nclusters, ++it) {
      const Unit u = rows_unit(grp, args.groups, t, num_p, num_n);
      const int acc = it & 1;
      const int n0 = u.nb * kPN + half * 128;
      const int n_valid = args.n - n0;                                       // may be <= 0
      const int r_valid = u.valid - static_cast<int>(rank) * 128 - quarter * 32;  // live rows from the warp's first on
      const int row0 = u.row0 + static_cast<int>(rank) * 128 + quarter * 32;
      // A second 128 rows exist only where the group reaches them; of 128 rows that exist, those behind
      // the count are written (as zeros) when asked.
      const bool exists = leader || u.valid > 128;
      const bool work = exists && n_valid > 0 && (r_valid > 0 || args.zero_pad);
      // The tile's bias values to shared memory while its products run: read
      // from global memory at their use they cost a sixth of a short tile.
      float* bias_s = sBias + ew * (kPBias / 4);
      if (args.bias) {
        const bool in = work && 4 * lane < n_valid;
        const float4 b = in ? __ldg(reinterpret_cast<const float4*>(args.bias + static_cast<int64_t>(u.g) * args.n + n0) + lane)
                            : make_float4(0.f, 0.f, 0.f, 0.f);
        reinterpret_cast<float4*>(bias_s)[lane] = b;
        __syncwarp();
      }
      if (!mbar_wait(&acc_full[acc], (it >> 1) & 1, args.err, kErrTimeoutAcc) || *abort_s) {
        *abort_s = 1;
        break;
      }
      tc_fence_after();
      uint32_t r[128];
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * kAccStep + half * 128;
      // The common columns are the last 32 of accumulator 0 and the first 32
      // of accumulator 1: they are read and released before the others.
      if (half != acc) {
        if (work) {
          if (acc)
            tmem_ld_32x32b_x32(taddr, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
          else
            tmem_ld_32x32b_x32(taddr + 96, *reinterpret_cast<uint32_t(*)[32]>(&r[96]));
          tmem_ld_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (leader)
            mbar_arrive(shared_cols);
          else
            mbar_arrive_peer(shared0);
        }
      }
      if (work) {
        if (half == acc || !acc) tmem_ld_32x32b_x32(taddr, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
        tmem_ld_32x32b_x32(taddr + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
        tmem_ld_32x32b_x32(taddr + 64, *reinterpret_cast<uint32_t(*)[32]>(&r[64]));
        if (half == acc || acc) tmem_ld_32x32b_x32(taddr + 96, *reinterpret_cast<uint32_t(*)[32]>(&r[96]));
        tmem_ld_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (leader)
          mbar_arrive(&acc_empty[acc]);
        else
          mbar_arrive_peer(acc_empty0 + acc * 8);
      }
      if (!work) continue;
      const bool whole = r_valid >= 32 && n_valid >= 128;
      if (args.bias) {
#pragma unroll
        for (int q = 0; q < 32; ++q) {
          const float4 b = reinterpret_cast<const float4*>(bias_s)[q];
          add2(r[4 * q], r[4 * q + 1], b.x, b.y);
          add2(r[4 * q + 2], r[4 * q + 3], b.z, b.w);
        }
        __syncwarp();  // before the next tile's values
      }
      if (RELU) {
#pragma unroll
        for (int j = 0; j < 128; ++j) r[j] = __float_as_uint(relu_keep_nan(__uint_as_float(r[j])));
      }
      if (!whole) {
        const bool live = lane < r_valid;
#pragma unroll
        for (int j = 0; j < 128; ++j) r[j] = live && j < n_valid ? r[j] : 0u;
      }
      if constexpr (OUT8) {
        float mx[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 128; ++j) mx[j & 3] = fmaxf(mx[j & 3], fabsf(__uint_as_float(r[j])));  // passes over NaN
        float m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        if (m == __uint_as_float(0x7f800000u)) {
          m = 0.f;
#pragma unroll
          for (int j = 0; j < 128; ++j) {
            m = fmaxf(m, finite_abs(__uint_as_float(r[j])));
            r[j] = __float_as_uint(inf_to_nan(__uint_as_float(r[j])));
          }
        }
        const uint32_t byte = scale_byte(m);
        const float inv = inv_scale(byte);
        if (lane == 0) bulk_wait_group_read0();
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = 16 * q + 4 * i;
            scale2(r[j], r[j + 1], inv);
            scale2(r[j + 2], r[j + 3], inv);
            w[i] = pack_e4m3x4(__uint_as_float(r[j]), __uint_as_float(r[j + 1]), __uint_as_float(r[j + 2]),
                               __uint_as_float(r[j + 3]));
          }
          *reinterpret_cast<uint4*>(stg + lane * 128 + ((q ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        const int kb = n0 >> 7;
        static_cast<uint8_t*>(args.c_scales)[scale_word_offset(row0 + lane, kb >> 2, out_k4) + (kb & 3)] =
            static_cast<uint8_t>(byte);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&tmC, stg, n0, row0);
          bulk_commit_group();
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (64 * h < n_valid) {
            if (lane == 0) bulk_wait_group_read0();
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int j = 64 * h + 8 * q + 2 * i;
                w[i] = pack2<OUT>(__uint_as_float(r[j]), __uint_as_float(r[j + 1]));
              }
              *reinterpret_cast<uint4*>(stg + lane * 128 + ((q ^ (lane & 7)) << 4)) =
                  make_uint4(w[0], w[1], w[2], w[3]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmC, stg, n0 + 64 * h, row0);
              bulk_commit_group();
            }
          }
        }
      }
    }
    if (lane == 0) {
      bulk_wait_group0();
      asm volatile("fence.proxy.async.global;" ::: "memory");
    }
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs are done with the pair's tensor memory and shared memory
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// Barrier among the epilogue warps that also tells all of them whether any
// passed `stop`.
__device__ __forceinline__ bool epilogue_any(bool stop) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "bar.red.or.pred p, 1, %2, q;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(stop)), "n"(32 * kEpi)
      : "memory");
  return any != 0;
}

template <typename OUT, bool RELU, int ROWS>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_weights_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                       const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSW,
                       Fp8GemmArgs args) {
  using Cfg = SwapCfg<ROWS>;
  constexpr bool OUT8 = sizeof(OUT) == 1;
  constexpr int kStages = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Groups grp;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sW = smem;
  uint8_t* sA = sW + kStages * Cfg::kW;
  uint8_t* sSf = sA + kStages * Cfg::kA;
  float* sStg = reinterpret_cast<float*>(sSf + kStages * Cfg::kSf);
  uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(sStg) + Cfg::kStg);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* sf_done = acc_empty + 2;
  uint64_t* drain = sf_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id(), lane = lane_id();
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kEpi);
      mbar_init(&sf_done[i], 1);
    }
    mbar_init(drain, 1);
    *abort_s = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmSA);
    tma_prefetch_desc(&tmSW);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  if (!args.early) {
    pdl_wait();
    pdl_trigger();
  }
  load_groups(args, ROWS, grp);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int num_n = (args.n + 127) / 128;
  const int total = grp.first[args.groups] * num_n;
  const int num_kb = (args.k + kBK - 1) / kBK;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    int stage = 0;
    uint32_t phase = 0, armed = 0, armed_parity = 0;
    bool ok = true;
    auto load_rows = [&](int st, int kb, const Unit& u, int boxes) {  // the elected lane
      for (int i = 0; i < boxes; ++i)
        tma_load_2d(sA + st * Cfg::kA + i * 32 * kBK, &tmA, kb * kBK, u.row0 + 32 * i, &full[st]);
      if ((kb & 3) == 0) tma_load_3d(sSf + st * Cfg::kSf + kScaleTile, &tmSA, 0, kb >> 2, u.row0 >> 7, &full[st]);
    };
    // With `early`, the first unit's first stages get their weights before
    // the wait for the previous kernel and their rows after it.
    bool waited = !args.early;
    int deferred = 0;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
      const Unit u = weights_unit<ROWS>(grp, args.groups, t, num_n);
      const int boxes = (min(u.valid, ROWS) + 31) / 32;
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1, args.err, kErrTimeoutEmpty) || *abort_s) {
          *abort_s = 1;
          ok = false;
          break;
        }
        if (elect_one()) {
          const bool sf = (kb & 3) == 0;
          mbar_arrive_expect_tx(&full[stage], Cfg::kW + boxes * 32 * kBK + (sf ? Cfg::kSf : 0));
          tma_load_3d(sW + stage * Cfg::kW, &tmW, kb * kBK, u.nb * 128, u.g, &full[stage]);
          if (sf) tma_load_3d(sSf + stage * Cfg::kSf, &tmSW, 0, kb >> 2, u.g * num_n + u.nb, &full[stage]);
          if (waited) load_rows(stage, kb, u, boxes);
        }
        if (!waited && (++deferred == kStages || deferred == num_kb)) {
          pdl_wait();
          pdl_trigger();
          waited = true;
          if (elect_one())
            for (int j = 0; j < deferred; ++j) load_rows(j, j, u, boxes);
        }
        armed |= 1u << stage;
        armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
        __syncwarp();
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (!waited) {
      // No unit (a unit's stages end the wait above): still order after the previous kernel.
      pdl_wait();
      pdl_trigger();
    }
    __syncwarp();
    for (int s = 0; s < kStages; ++s)
      if (armed & (1u << s)) mbar_wait(&full[s], (armed_parity >> s) & 1, args.err, kErrTimeoutDrain);
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    const uint32_t sW_addr = smem_u32(sW), sA_addr = smem_u32(sA), sSf_addr = smem_u32(sSf);
    int stage = 0, it = 0, sf_use = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x, ++it) {
      const Unit u = weights_unit<ROWS>(grp, args.groups, t, num_n);
      const int n_mma = (min(u.valid, ROWS) + 31) / 32 * 32;
      const int acc = it & 1;
      if (!mbar_wait(&acc_empty[acc], ((it >> 1) & 1) ^ 1, args.err, kErrTimeoutAcc) || *abort_s) {
        *abort_s = 1;
        break;
      }
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + acc * ROWS;
      uint32_t sfw = 0, sfa = 0;
      int slot = 0;
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait(&full[stage], phase, args.err, kErrTimeoutFull) || *abort_s) {
          *abort_s = 1;
          ok = false;
          break;
        }
        if ((kb & 3) == 0) {
          slot = sf_use & 1;
          if (sf_use >= 2 && !mbar_wait(&sf_done[slot], ((sf_use >> 1) - 1) & 1, args.err, kErrTimeoutAcc)) {
            *abort_s = 1;
            ok = false;
            break;
          }
          ++sf_use;
          sfw = tmem_base + Cfg::kSfCol + slot * 8;
          sfa = sfw + 4;
          // The MMA takes the scales of its 32 rows from the first of the
          // tile's four columns (it reads scales at multiples of 4 columns
          // only), so the words of a later 32-row group move there.
          const int q = ROWS == 32 ? (u.row0 >> 5) & 3 : 0;
          if (q) {
            uint32_t* tile = reinterpret_cast<uint32_t*>(sSf + stage * Cfg::kSf + kScaleTile);
            tile[4 * lane] = tile[4 * lane + q];
            fence_proxy_async_smem();
            __syncwarp();
          }
        }
        tc_fence_after();
        if (elect_one()) {
          if ((kb & 3) == 0) {
            const uint32_t src = sSf_addr + stage * Cfg::kSf;
            const uint32_t dst = tmem_base + Cfg::kSfCol + slot * 8;
            tmem_copy_scales<1>(dst, smem_desc_scale(src));
            tmem_copy_scales<1>(dst + 4, smem_desc_scale(src + kScaleTile));
          }
          const uint64_t w_desc = smem_desc_k_sw128(sW_addr + stage * Cfg::kW);
          const uint64_t a_desc = smem_desc_k_sw128(sA_addr + stage * Cfg::kA);
          const uint32_t idesc = idesc_mxf8(128, n_mma, kb & 3);
#pragma unroll
          for (int kk = 0; kk < kBK / 32; ++kk)
            umma_mxf8<1>(d_tmem, w_desc + 2 * kk, a_desc + 2 * kk, idesc, sfw, sfa, (kb > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&empty[stage]);
          if ((kb & 3) == 3 || kb == num_kb - 1) umma_commit(&sf_done[slot]);
          if (kb == num_kb - 1) umma_commit(&acc_full[acc]);
        }
        __syncwarp();
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (elect_one()) umma_commit(drain);
    __syncwarp();
    mbar_wait(drain, 0, args.err, kErrTimeoutDrain);
  } else {
    // ---------------- Epilogue (warps 2..9) ----------------
    // The accumulator has an output column n per lane and a row per column:
    // 32 rows at a time go through shared memory, after which a warp holds a
    // row's 128 columns, 4 per lane.
    const int ew = warp - 2;
    const int quarter = warp & 3;
    const int half = ew >> 2;
    const int out_k4 = scale_k4(args.n);
    int it = 0;
    for (int t = blockIdx.x; t < total; t += gridDim.x, ++it) {
      const Unit u = weights_unit<ROWS>(grp, args.groups, t, num_n);
      const int acc = it & 1;
      const int n0 = u.nb * 128;
      const int live = min(u.valid, ROWS);
      // Rows this unit writes: its live rows, and behind a segment's last row zeros up to the next multiple of 128.
      const int rows = (args.zero_pad && u.valid <= ROWS) ? live + ((-(u.row0 + live)) & 127) : live;
      const int chunks = (live + 31) / 32;
      const bool in_n = n0 + quarter * 32 + lane < args.n;
      const float b = args.bias && in_n ? __ldg(args.bias + static_cast<int64_t>(u.g) * args.n + n0 + quarter * 32 + lane)
                                        : 0.f;
      const bool got = mbar_wait(&acc_full[acc], (it >> 1) & 1, args.err, kErrTimeoutAcc);
      if (!got) *abort_s = 1;
      tc_fence_after();
      for (int ch = 0; ch * 32 < rows; ++ch) {
        // Also: the staged rows of the chunk before have been read.
        if (epilogue_any(!got || *abort_s)) {
          if (lane == 0) *abort_s = 1;
          goto done;
        }
        if (ch < chunks) {
          uint32_t r[16];
          tmem_ld_32x32b_x16(
              tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * ROWS + 32 * ch + 16 * half, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float v = __uint_as_float(r[i]) + b;
            if (RELU) v = relu_keep_nan(v);
            const bool ok_row = 32 * ch + 16 * half + i < live;
            sStg[(16 * half + i) * Cfg::kStgLd + quarter * 32 + lane] = ok_row && in_n ? v : 0.f;
          }
          if (ch == chunks - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[acc]);  // the accumulator has been read
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) sStg[(16 * half + i) * Cfg::kStgLd + quarter * 32 + lane] = 0.f;
        }
        named_bar_sync(1, 32 * kEpi);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int rr = ew * 4 + i;
          if (32 * ch + rr >= rows) continue;
          const int64_t row = static_cast<int64_t>(u.row0) + 32 * ch + rr;
          const float4 v = *reinterpret_cast<const float4*>(&sStg[rr * Cfg::kStgLd + 4 * lane]);
          const int n = n0 + 4 * lane;
          if constexpr (OUT8) {
            float m = fmaxf(fmaxf(finite_abs(v.x), finite_abs(v.y)), fmaxf(finite_abs(v.z), finite_abs(v.w)));
            m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));  // non-negative floats order as ints
            const uint32_t byte = scale_byte(m);
            const float inv = inv_scale(byte);
            if (n < args.n)
              *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(args.c) + row * args.n + n) =
                  pack_e4m3x4(inf_to_nan(v.x) * inv, inf_to_nan(v.y) * inv, inf_to_nan(v.z) * inv, inf_to_nan(v.w) * inv);
            if (lane == 0)
              static_cast<uint8_t*>(args.c_scales)[scale_word_offset(row, u.nb >> 2, out_k4) + (u.nb & 3)] =
                  static_cast<uint8_t>(byte);
          } else if (n < args.n) {
            *reinterpret_cast<uint2*>(static_cast<OUT*>(args.c) + row * args.n + n) =
                make_uint2(pack2<OUT>(v.x, v.y), pack2<OUT>(v.z, v.w));
          }
        }
      }
    }
  }
done:
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::kTmemCols);
  }
}

// Scale tiles [tiles][k4][512 bytes] as 32-bit words; a box takes `tiles_box` tiles at one k4.
bool encode_scales(CUtensorMap* m, const void* base, int64_t tiles, int k4, int tiles_box) {
  const uint64_t dims[3] = {128, static_cast<uint64_t>(k4), static_cast<uint64_t>(tiles)};
  const uint64_t str[2] = {kScaleTile, static_cast<uint64_t>(k4) * kScaleTile};
  const uint32_t box[3] = {128, 1, static_cast<uint32_t>(tiles_box)};
  return encode_tmap(m, base, 3, dims, str, box, CU_TENSOR_MAP_DATA_TYPE_UINT32, CU_TENSOR_MAP_SWIZZLE_NONE);
}

bool encode_rows(const Fp8GemmArgs& args, uint32_t box_rows, CUtensorMap* tmA) {
  const uint64_t dims[2] = {static_cast<uint64_t>(args.k), static_cast<uint64_t>(args.a_rows)};
  const uint64_t str[1] = {static_cast<uint64_t>(args.k)};
  const uint32_t box[2] = {kBK, box_rows};
  return encode_tmap(tmA, args.a, 2, dims, str, box, CU_TENSOR_MAP_DATA_TYPE_UINT8);
}

// Both kernels' operands: rows in boxes of 32, weights in boxes of 128, scale tiles.
bool encode_operands(const Fp8GemmArgs& args, int w_tiles_box, CUtensorMap* tmA, CUtensorMap* tmW, CUtensorMap* tmSA,
                     CUtensorMap* tmSW) {
  const uint64_t k = static_cast<uint64_t>(args.k), n = static_cast<uint64_t>(args.n);
  const int k4 = scale_k4(args.k);
  if (!encode_rows(args, 32, tmA)) return false;
  {
    const uint64_t dims[3] = {k, n, static_cast<uint64_t>(args.groups)};
    const uint64_t str[2] = {k, k * n};
    const uint32_t box[3] = {kBK, 128, 1};
    if (!encode_tmap(tmW, args.w, 3, dims, str, box, CU_TENSOR_MAP_DATA_TYPE_UINT8)) return false;
  }
  return encode_scales(tmSA, args.a_scales, (args.a_rows + 127) / 128, k4, 1) &&
         encode_scales(tmSW, args.w_scales, args.groups * static_cast<int64_t>((args.n + 127) / 128), k4, w_tiles_box);
}

template <typename OUT, bool RELU>
cudaError_t launch_rows(const Fp8GemmArgs& args, int num_sms, cudaStream_t stream) {
  CUtensorMap tmA, tmA32, tmB, tmC, tmSA, tmSB;
  if (!encode_operands(args, 2, &tmA32, &tmB, &tmSA, &tmSB) || !encode_rows(args, 128, &tmA)) return cudaErrorInvalidValue;
  {
    const uint64_t dims[2] = {static_cast<uint64_t>(args.n), static_cast<uint64_t>(args.a_rows)};
    const uint64_t str[1] = {static_cast<uint64_t>(args.n) * sizeof(OUT)};
    const uint32_t box[2] = {128 / sizeof(OUT), 32};
    const CUtensorMapDataType dt = sizeof(OUT) == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    if (!encode_tmap(&tmC, args.c, 2, dims, str, box, dt)) return cudaErrorInvalidValue;
  }
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(fp8_rows_kernel<OUT, RELU>), kPSmem);
  if (e != cudaSuccess) return e;
  const int64_t units = (args.live_rows / 256 + args.groups) * static_cast<int64_t>((args.n + kPN - 1) / kPN);
  const int ctas = std::max(2, static_cast<int>(std::min<int64_t>(num_sms, 2 * units)) & ~1);
  return launch_kernel(fp8_rows_kernel<OUT, RELU>, dim3(ctas), dim3(kThreads), kPSmem, stream, tmA, tmB, tmC, tmSA,
                       tmSB, tmA32, args);
}

template <typename OUT, bool RELU, int ROWS>
cudaError_t launch_weights(const Fp8GemmArgs& args, int num_sms, cudaStream_t stream) {
  CUtensorMap tmA, tmW, tmSA, tmSW;
  if (!encode_operands(args, 1, &tmA, &tmW, &tmSA, &tmSW)) return cudaErrorInvalidValue;
  const int smem = SwapCfg<ROWS>::kSmem;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(fp8_weights_kernel<OUT, RELU, ROWS>), smem);
  if (e != cudaSuccess) return e;
  const int64_t units = (args.live_rows / ROWS + args.groups) * static_cast<int64_t>((args.n + 127) / 128);
  const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(num_sms, units)));
  return launch_kernel(fp8_weights_kernel<OUT, RELU, ROWS>, dim3(grid), dim3(kThreads), smem, stream, tmA, tmW, tmSA,
                       tmSW, args);
}

template <typename OUT, bool RELU>
cudaError_t launch_mode(const Fp8GemmArgs& args, int mode, int num_sms, cudaStream_t stream) {
  if (mode == AGM_FP8_ROWS) return launch_rows<OUT, RELU>(args, num_sms, stream);
  // Up to 32 rows per group on average: blocks of 32 rows and a deeper ring.
  if (args.live_rows <= 32 * static_cast<int64_t>(args.groups)) return launch_weights<OUT, RELU, 32>(args, num_sms, stream);
  return launch_weights<OUT, RELU, 128>(args, num_sms, stream);
}

template <typename OUT>
cudaError_t launch_out(const Fp8GemmArgs& args, int mode, int num_sms, cudaStream_t stream) {
  return args.relu ? launch_mode<OUT, true>(args, mode, num_sms, stream)
                   : launch_mode<OUT, false>(args, mode, num_sms, stream);
}

}  // namespace

cudaError_t grouped_gemm_fp8(int c_dtype, const Fp8GemmArgs& args, int mode, int num_sms, cudaStream_t stream) {
  if (mode == AGM_FP8_AUTO)
    mode = args.live_rows >= 128 * static_cast<int64_t>(args.groups) ? AGM_FP8_ROWS : AGM_FP8_WEIGHTS;
  if (args.c_scales) return launch_out<__nv_fp8_e4m3>(args, mode, num_sms, stream);
  return c_dtype == AGM_BF16 ? launch_out<__nv_bfloat16>(args, mode, num_sms, stream)
                             : launch_out<__half>(args, mode, num_sms, stream);
}

}  // namespace agm
