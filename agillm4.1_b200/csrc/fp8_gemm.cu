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
//   epilogue's arithmetic. 147,456 rows over 14 groups: 1280 -> 3200 with
//   e4m3 output 507 us (2.38 PFLOP/s), 3200 -> 1280 with bf16 output 469 us
//   (2.58), in runs of a few launches; back to back for seconds, under the 1 kW
//   cap, 588 us (2.05) and 547 to 584 us (2.07 to 2.21). A k-block of a pair takes 0.43 us, 0.28 when nothing is loaded:
//   what bounds it is the 64 KB that come from L2 meanwhile (11 TB/s over all
//   SMs). A change of tiles adds 0.8 us. Three and four stages instead of five
//   were 17% and 5% slower.
//
// * fp8_weights_kernel, few rows per group (bound by reading the weights): the
//   weight tile is the 128-row operand and up to 128 of the group's rows the N
//   operand, of which only the 32-row boxes with live rows are loaded and
//   multiplied. The ring keeps 96 KB of weights in flight per SM; 144 KB, with
//   room for 32 rows only, was not faster at 8 rows per group (42 against 40
//   us for 61 x 1488 x 2000) and slower from 32 on. A further group of 3200 x
//   1280 takes its weights' time at 5.75 TB/s; 7.3 us are fixed (launch, the
//   first weights' latency, the last tile's epilogue).
//
//   It also runs both products of a block of experts in one launch: units of
//   the first product, then of the second, are drawn from a ticket counter.
//   A unit of the second waits until all columns of its rows have been
//   written (a counter per 128-row block), after its first weights are on
//   their way, so the weights stream through the change from one product to
//   the other. Tickets keep this free of deadlocks whatever part of the grid
//   is running: a unit that is waited for was drawn earlier, by a CTA that
//   runs and waits for nothing but units drawn before. 64 tokens, top-2 of 14,
//   1280 -> 3200 -> 1280, dispatch to weighted sum: 39 us in two launches, 36
//   in one. Prefetching the first weights into L2 during the dispatch gained
//   0.4 us there and cost 4 us at one token, so it is not done.
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
constexpr int kWStages = 6;
constexpr int kWRows = 128;                   // rows of a unit
constexpr int kWW = 128 * kBK;                // 16 KB of weights
constexpr int kWA = kWRows * kBK;
constexpr int kWSf = 2 * kScaleTile;
constexpr int kWStgLd = 132;                  // floats per staged row
constexpr int kWStg = 32 * kWStgLd * 4;
constexpr int kWSfCol = 2 * kWRows;           // behind the two accumulators: two slots of 8 columns
constexpr int kWQueue = 4;                    // units drawn ahead
constexpr int kWSmem = kWStages * (kWW + kWA + kWSf) + kWStg + 512 + 1024;

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

__device__ __forceinline__ Unit weights_unit(const Groups& s, int groups, int b, int nb) {
  Unit u;
  u.nb = nb;
  u.g = find_group(s, groups, b);
  const int j = b - s.first[u.g];
  u.row0 = s.start[u.g] + j * kWRows;
  u.valid = s.count[u.g] - j * kWRows;
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
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist before any cross-CTA arrive or copy
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  pdl_wait();
  pdl_trigger();
  load_groups(args, 256, grp);
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

// One product, or (FUSED) the two of a block of experts.
struct WeightsArgs {
  Fp8GemmArgs p[2];
  int32_t* ticket;  // FUSED: next unit
  int32_t* done;    // FUSED: per 128-row block, finished units of the first product
};
struct WeightsMaps {
  CUtensorMap a[2], w[2], sa[2], sw[2];
};

__device__ __forceinline__ int ld_acquire_gpu(const int32_t* p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// T: the 16-bit output type (of the second product when FUSED, whose first
// writes e4m3).
template <typename T, bool FUSED>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_weights_kernel(const __grid_constant__ WeightsMaps maps, const __grid_constant__ WeightsArgs args) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ Groups grp;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sW = smem;
  uint8_t* sA = sW + kWStages * kWW;
  uint8_t* sSf = sA + kWStages * kWA;
  float* sStg = reinterpret_cast<float*>(sSf + kWStages * kWSf);
  uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(sStg) + kWStg);
  uint64_t* empty = full + kWStages;
  uint64_t* acc_full = empty + kWStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* sf_done = acc_empty + 2;
  uint64_t* q_full = sf_done + 2;
  uint64_t* q_empty = q_full + kWQueue;
  uint64_t* drain = q_empty + kWQueue;
  volatile int* queue = reinterpret_cast<volatile int*>(drain + 1);  // [kWQueue], -1: no more units
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1) + kWQueue;
  volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id(), lane = lane_id();
  int* err = args.p[0].err;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kWStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kEpi);
      mbar_init(&sf_done[i], 1);
    }
    for (int i = 0; i < kWQueue; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1 + kEpi);
    }
    mbar_init(drain, 1);
    *abort_s = 0;
    fence_barrier_init();
    for (int i = 0; i < (FUSED ? 2 : 1); ++i) {
      tma_prefetch_desc(&maps.a[i]);
      tma_prefetch_desc(&maps.w[i]);
      tma_prefetch_desc(&maps.sa[i]);
      tma_prefetch_desc(&maps.sw[i]);
    }
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_trigger();
  int first_ticket = blockIdx.x;
  if (FUSED && threadIdx.x == 0) first_ticket = atomicAdd(args.ticket, 1);  // answered while the groups are read
  load_groups(args.p[0], kWRows, grp);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int groups = args.p[0].groups;
  const int blocks = grp.first[groups];
  const int num_n0 = (args.p[0].n + 127) / 128;
  const int num_n1 = FUSED ? (args.p[1].n + 127) / 128 : 0;
  const int total0 = blocks * num_n0;
  const int total = total0 + blocks * num_n1;
  // Unit t: product, 128-row block, column tile.
  auto decode = [&](int t, int& ph, int& b) {
    ph = FUSED && t >= total0 ? 1 : 0;
    const int r = t - (ph ? total0 : 0), n = ph ? num_n1 : num_n0;
    b = r / n;
    return weights_unit(grp, groups, b, r - b * n);
  };
  // The consumers' next unit (-1: none): drawn by the producer when FUSED.
  int taken = 0;
  auto next_unit = [&](int t) -> int {
    if constexpr (!FUSED) {
      t = taken++ ? t + static_cast<int>(gridDim.x) : static_cast<int>(blockIdx.x);
      return t < total ? t : -1;
    } else {
      const int s = taken % kWQueue;
      if (!mbar_wait(&q_full[s], (taken / kWQueue) & 1, err, kErrTimeoutFull)) {
        *abort_s = 1;
        return -1;
      }
      t = queue[s];
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_empty[s]);
      ++taken;
      return t;
    }
  };

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    int stage = 0;
    uint32_t phase = 0, armed = 0, armed_parity = 0;
    int drawn = 0, ahead = __shfl_sync(0xffffffffu, first_ticket, 0);
    bool ok = true;
    while (ok) {
      const int t = ahead < total ? ahead : -1;
      if (FUSED) {
        const int s = drawn % kWQueue;
        if (!mbar_wait(&q_empty[s], ((drawn / kWQueue) & 1) ^ 1, err, kErrTimeoutEmpty) || *abort_s) {
          *abort_s = 1;
          break;
        }
        if (lane == 0) {
          queue[s] = t;
          mbar_arrive(&q_full[s]);  // releases the store
        }
        __syncwarp();
        ++drawn;
      }
      if (t < 0) break;
      int ticket = 0;
      if (FUSED && lane == 0) ticket = atomicAdd(args.ticket, 1);  // answered while this unit loads
      int ph, b;
      const Unit u = decode(t, ph, b);
      const int num_kb = ((ph ? args.p[1].k : args.p[0].k) + kBK - 1) / kBK;
      const int num_n = ph ? num_n1 : num_n0;
      const int boxes = (min(u.valid, kWRows) + 31) / 32;
      const CUtensorMap *mA = &maps.a[ph], *mW = &maps.w[ph], *mSA = &maps.sa[ph], *mSW = &maps.sw[ph];
      auto load_rows = [&](int st, int kb) {  // the elected lane
        for (int i = 0; i < boxes; ++i)
          tma_load_2d(sA + st * kWA + i * 32 * kBK, mA, kb * kBK, u.row0 + 32 * i, &full[st]);
        if ((kb & 3) == 0) tma_load_3d(sSf + st * kWSf + kScaleTile, mSA, 0, kb >> 2, u.row0 >> 7, &full[st]);
      };
      // Whether the unit's rows have been written; those of the second
      // product come from the first. Its proxy fence orders the TMA loads
      // behind the counter's acquire.
      bool ready = !FUSED || ph == 0;
      auto poll = [&]() {
        int v = lane == 0 ? ld_acquire_gpu(args.done + b) : 0;
        v = __shfl_sync(0xffffffffu, v, 0);
        __syncwarp();  // a shuffle orders no memory, and the elected lane need not be the one that acquired
        if (v >= num_n0) {
          asm volatile("fence.proxy.async.global;" ::: "memory");
          ready = true;
        }
      };
      int waiting = 0, first_stage = stage;  // stages that have their weights only
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1, err, kErrTimeoutEmpty) || *abort_s) {
          *abort_s = 1;
          ok = false;
          break;
        }
        if (elect_one()) {
          const bool sf = (kb & 3) == 0;
          mbar_arrive_expect_tx(&full[stage], kWW + boxes * 32 * kBK + (sf ? kWSf : 0));
          tma_load_3d(sW + stage * kWW, mW, kb * kBK, u.nb * 128, u.g, &full[stage]);
          if (sf) tma_load_3d(sSf + stage * kWSf, mSW, 0, kb >> 2, u.g * num_n + u.nb, &full[stage]);
          if (ready) load_rows(stage, kb);
        }
        __syncwarp();
        if (FUSED && !ready) {
          ++waiting;
          poll();
          if (!ready && (waiting == kWStages || waiting == num_kb)) {
            const uint64_t t0 = globaltimer_ns();
            while (!ready) {
              __nanosleep(64);
              poll();
              if (!ready && (globaltimer_ns() - t0 > AGM_WAIT_LIMIT_NS || *abort_s)) {
                if (lane == 0) raise_error(err, kErrTimeoutFull);
                *abort_s = 1;
                break;
              }
              __syncwarp();
            }
            // On time-out the rows are loaded all the same, so that every armed stage completes.
            ok = ready;
          }
          if (ready || !ok) {
            if (elect_one())
              for (int j = 0; j < waiting; ++j) load_rows((first_stage + j) % kWStages, j);
            __syncwarp();
          }
        }
        armed |= 1u << stage;
        armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
        if (++stage == kWStages) {
          stage = 0;
          phase ^= 1;
        }
        if (!ok) break;
      }
      ahead = FUSED ? __shfl_sync(0xffffffffu, ticket, 0) : t + static_cast<int>(gridDim.x);
    }
    __syncwarp();
    for (int s = 0; s < kWStages; ++s)
      if (armed & (1u << s)) mbar_wait(&full[s], (armed_parity >> s) & 1, err, kErrTimeoutDrain);
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    const uint32_t sW_addr = smem_u32(sW), sA_addr = smem_u32(sA), sSf_addr = smem_u32(sSf);
    int stage = 0, it = 0, sf_use = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = next_unit(0); t >= 0 && ok; t = next_unit(t), ++it) {
      int ph, b;
      const Unit u = decode(t, ph, b);
      const int num_kb = ((ph ? args.p[1].k : args.p[0].k) + kBK - 1) / kBK;
      const int n_mma = (min(u.valid, kWRows) + 31) / 32 * 32;
      const int acc = it & 1;
      if (!mbar_wait(&acc_empty[acc], ((it >> 1) & 1) ^ 1, err, kErrTimeoutAcc) || *abort_s) {
        *abort_s = 1;
        break;
      }
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + acc * kWRows;
      uint32_t sfw = 0;
      int slot = 0;
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait(&full[stage], phase, err, kErrTimeoutFull) || *abort_s) {
          *abort_s = 1;
          ok = false;
          break;
        }
        if ((kb & 3) == 0) {
          slot = sf_use & 1;
          if (sf_use >= 2 && !mbar_wait(&sf_done[slot], ((sf_use >> 1) - 1) & 1, err, kErrTimeoutAcc)) {
            *abort_s = 1;
            ok = false;
            break;
          }
          ++sf_use;
          sfw = tmem_base + kWSfCol + slot * 8;
        }
        tc_fence_after();
        if (elect_one()) {
          if ((kb & 3) == 0) {
            const uint32_t src = sSf_addr + stage * kWSf;
            tmem_copy_scales<1>(sfw, smem_desc_scale(src));
            tmem_copy_scales<1>(sfw + 4, smem_desc_scale(src + kScaleTile));
          }
          const uint64_t w_desc = smem_desc_k_sw128(sW_addr + stage * kWW);
          const uint64_t a_desc = smem_desc_k_sw128(sA_addr + stage * kWA);
          const uint32_t idesc = idesc_mxf8(128, n_mma, kb & 3);
#pragma unroll
          for (int kk = 0; kk < kBK / 32; ++kk)
            umma_mxf8<1>(d_tmem, w_desc + 2 * kk, a_desc + 2 * kk, idesc, sfw, sfw + 4, (kb > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&empty[stage]);
          if ((kb & 3) == 3 || kb == num_kb - 1) umma_commit(&sf_done[slot]);
          if (kb == num_kb - 1) umma_commit(&acc_full[acc]);
        }
        __syncwarp();
        if (++stage == kWStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (elect_one()) umma_commit(drain);
    __syncwarp();
    mbar_wait(drain, 0, err, kErrTimeoutDrain);
  } else {
    // ---------------- Epilogue (warps 2..9) ----------------
    // The accumulator has an output column n per lane and a row per column:
    // 32 rows at a time go through shared memory, after which a warp holds a
    // row's 128 columns, 4 per lane.
    const int ew = warp - 2;
    const int quarter = warp & 3;
    const int half = ew >> 2;
    int it = 0;
    for (int t = next_unit(0);; t = next_unit(t), ++it) {
      // All epilogue warps leave together: one may have met a time-out.
      if (epilogue_any(t < 0 || *abort_s)) break;
      int ph, b;
      const Unit u = decode(t, ph, b);
      const Fp8GemmArgs& g = args.p[ph];
      const bool out8 = g.c_scales != nullptr;
      const int acc = it & 1;
      const int n0 = u.nb * 128;
      const int live = min(u.valid, kWRows);
      // Rows this unit writes: its live rows, and behind a segment's last row zeros up to the next multiple of 128
      // or the last row there is.
      const int rows = (g.zero_pad && u.valid <= kWRows)
                           ? static_cast<int>(min(static_cast<int64_t>(live + ((-(u.row0 + live)) & 127)), g.a_rows - u.row0))
                           : live;
      const int chunks = (live + 31) / 32;
      const int out_k4 = scale_k4(g.n);
      const bool in_n = n0 + quarter * 32 + lane < g.n;
      const float bias = g.bias && in_n ? __ldg(g.bias + static_cast<int64_t>(u.g) * g.n + n0 + quarter * 32 + lane) : 0.f;
      const bool got = mbar_wait(&acc_full[acc], (it >> 1) & 1, err, kErrTimeoutAcc);
      if (!got) *abort_s = 1;
      tc_fence_after();
      bool stop = false;
      for (int ch = 0; ch * 32 < rows && !stop; ++ch) {
        // Also: the staged rows of the chunk before have been read.
        if (epilogue_any(!got || *abort_s)) {
          stop = true;
          break;
        }
        if (ch < chunks) {
          uint32_t r[16];
          tmem_ld_32x32b_x16(
              tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * kWRows + 32 * ch + 16 * half, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float v = __uint_as_float(r[i]) + bias;
            if (g.relu) v = relu_keep_nan(v);
            const bool ok_row = 32 * ch + 16 * half + i < live;
            sStg[(16 * half + i) * kWStgLd + quarter * 32 + lane] = ok_row && in_n ? v : 0.f;
          }
          if (ch == chunks - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[acc]);  // the accumulator has been read
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) sStg[(16 * half + i) * kWStgLd + quarter * 32 + lane] = 0.f;
        }
        named_bar_sync(1, 32 * kEpi);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int rr = ew * 4 + i;
          if (32 * ch + rr >= rows) continue;
          const int64_t row = static_cast<int64_t>(u.row0) + 32 * ch + rr;
          const float4 v = *reinterpret_cast<const float4*>(&sStg[rr * kWStgLd + 4 * lane]);
          const int n = n0 + 4 * lane;
          if (out8) {
            float m = fmaxf(fmaxf(finite_abs(v.x), finite_abs(v.y)), fmaxf(finite_abs(v.z), finite_abs(v.w)));
            m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));  // non-negative floats order as ints
            const uint32_t byte = scale_byte(m);
            const float inv = inv_scale(byte);
            if (n < g.n)
              *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(g.c) + row * g.n + n) =
                  pack_e4m3x4(inf_to_nan(v.x) * inv, inf_to_nan(v.y) * inv, inf_to_nan(v.z) * inv, inf_to_nan(v.w) * inv);
            if (lane == 0)
              static_cast<uint8_t*>(g.c_scales)[scale_word_offset(row, u.nb >> 2, out_k4) + (u.nb & 3)] =
                  static_cast<uint8_t>(byte);
          } else if (n < g.n) {
            *reinterpret_cast<uint2*>(static_cast<T*>(g.c) + row * g.n + n) =
                make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
          }
        }
      }
      if (stop) break;
      if (FUSED && ph == 0) {
        // The block's rows have one more column tile: publish it.
        named_bar_sync(1, 32 * kEpi);
        if (threadIdx.x == 64) {
          __threadfence();
          atomicAdd(args.done + b, 1);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
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

template <typename T>
cudaError_t launch_weights(const Fp8GemmArgs& args, int num_sms, cudaStream_t stream) {
  WeightsMaps maps = {};
  if (!encode_operands(args, 1, &maps.a[0], &maps.w[0], &maps.sa[0], &maps.sw[0])) return cudaErrorInvalidValue;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(fp8_weights_kernel<T, false>), kWSmem);
  if (e != cudaSuccess) return e;
  WeightsArgs wa = {};
  wa.p[0] = args;
  const int64_t units = (args.live_rows / kWRows + args.groups) * static_cast<int64_t>((args.n + 127) / 128);
  const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(num_sms, units)));
  return launch_kernel(fp8_weights_kernel<T, false>, dim3(grid), dim3(kThreads), kWSmem, stream, maps, wa);
}

template <typename T>
cudaError_t launch_both(const Fp8GemmArgs& first, const Fp8GemmArgs& second, int32_t* ticket, int32_t* done, int num_sms,
                        cudaStream_t stream) {
  WeightsMaps maps;
  if (!encode_operands(first, 1, &maps.a[0], &maps.w[0], &maps.sa[0], &maps.sw[0]) ||
      !encode_operands(second, 1, &maps.a[1], &maps.w[1], &maps.sa[1], &maps.sw[1]))
    return cudaErrorInvalidValue;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(fp8_weights_kernel<T, true>), kWSmem);
  if (e != cudaSuccess) return e;
  const WeightsArgs wa{{first, second}, ticket, done};
  return launch_kernel(fp8_weights_kernel<T, true>, dim3(num_sms), dim3(kThreads), kWSmem, stream, maps, wa);
}

template <typename OUT>
cudaError_t launch_rows_relu(const Fp8GemmArgs& args, int num_sms, cudaStream_t stream) {
  return args.relu ? launch_rows<OUT, true>(args, num_sms, stream) : launch_rows<OUT, false>(args, num_sms, stream);
}

}  // namespace

// The rows kernel fills its 256-row tiles from about 96 rows per group on (14
// groups, 3200 -> 1280: 16.6 us against 14.2 at 64 rows, 16.9 against 24.0 at
// 128; 61 groups, 2000 -> 1488: 51 against 44 at 80 rows, 56 against 74 at 160).
bool fp8_rows_pay(int64_t rows, int groups) { return rows >= 96 * static_cast<int64_t>(groups); }

cudaError_t grouped_gemm_fp8(int c_dtype, const Fp8GemmArgs& args, int mode, int num_sms, cudaStream_t stream) {
  const bool rows = mode == AGM_FP8_AUTO ? fp8_rows_pay(args.live_rows, args.groups) : mode == AGM_FP8_ROWS;
  if (!rows)
    return c_dtype == AGM_BF16 || args.c_scales ? launch_weights<__nv_bfloat16>(args, num_sms, stream)
                                                : launch_weights<__half>(args, num_sms, stream);
  if (args.c_scales) return launch_rows_relu<__nv_fp8_e4m3>(args, num_sms, stream);
  return c_dtype == AGM_BF16 ? launch_rows_relu<__nv_bfloat16>(args, num_sms, stream)
                             : launch_rows_relu<__half>(args, num_sms, stream);
}

cudaError_t expert_products_fp8(int dtype, const Fp8GemmArgs& first, const Fp8GemmArgs& second, int32_t* ticket,
                                int32_t* done, int num_sms, cudaStream_t stream) {
  return dtype == AGM_BF16 ? launch_both<__nv_bfloat16>(first, second, ticket, done, num_sms, stream)
                           : launch_both<__half>(first, second, ticket, done, num_sms, stream);
}

}  // namespace agm
