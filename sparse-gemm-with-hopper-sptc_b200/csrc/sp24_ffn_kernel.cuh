// sp24_ffn_kernel.cuh — the gated feed-forward block's products on CTA pairs:
// dense 16-bit operands, tcgen05.mma.cta_group::2 with M = 256, N = 256,
// fp32 accumulators in TMEM.
//
//   kFfnForward  act(x Wg^T) * (x Wu^T): tokens along M, 128 features of Wg and
//                the same 128 of Wu along N.  CTA 0 of the pair stages Wg's
//                rows and CTA 1 Wu's, so one MMA fills columns 0-127 of the
//                accumulator with g and columns 128-255 with u: every epilogue
//                thread holds both sums of its elements, and no second pass
//                over x or over h is needed.
//   kFfnDx       [dg | du] [Wg; Wu]: K runs through f twice, first dg with Wg,
//                then du with Wu, into one accumulator.
//   kFfnDw       dg^T x and du^T x: M runs through f twice (one output each),
//                K through the tokens.
//
// Operands are read where they lie: K-major rows (x and W forward, dg forward
// of Wg) or, where the summed index is the row, MN-major (W in dx, dg and x in
// dw), in SWIZZLE_128B boxes of 64 x 64 elements; no transposed copy is made.
// Rows and columns past the end are zero-filled by TMA and not stored.
//
// Roles per CTA (11 warps), as in the 2:4 pair kernel (sp24_gemm2sm_kernel.cuh):
// warps 0 and 10 load A and B, warp 1 of the leader issues the MMAs, warps 2-9
// drain the accumulator.  It is double-buffered (2 x 256 columns fill TMEM), so
// a tile's epilogue overlaps the next tile's products.
//
// Bound by the tensor pipe: a 256 x 256 tile takes in 32 KB per 512 clocks and SM,
// about what an SM can take (64 bytes a clock), and the pipe is 95-96% active in
// all three products.  B200, 4096 tokens, 4096 -> 14336 bf16, 962 GFLOP each:
// forward 608 us in a burst (1.58 PFLOP/s; cuBLAS's burst rate is 1.67), 690 held
// under the 1000 W cap at 1.25-1.3 GHz, where cuBLAS takes 720 for the product
// alone; dx 640, dw 625 (cuBLAS 713, 728).  Row-tile groups of 16 (all the tokens
// of this size) against 8 forward: 655 against 699 us.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "sp24_gemm2sm_kernel.cuh"
#include "sp24_ptx.cuh"
#include "sp24_rows.cuh"

namespace sp24 {

enum : int { kFfnForward = 0, kFfnDx = 1, kFfnDw = 2 };
constexpr int kFfnMaxSplits = 4;   // pairs per cluster of the K-split forms: 8 CTAs

struct FfnParams {
  int m, n;                // rows of a plane's output, output columns (forward: f)
  int m_tiles, n_tiles;    // of the whole launch (dw: both planes' row tiles)
  int k_stages;            // 64-deep stages of one tile
  int plane;               // dx: stages per plane; dw: row tiles per plane
  int group_m;
  int splits;              // K-split forms: pairs per cluster; dx: else K slices a tile
  float* partial;          // planes of m x ld_partial sums, a slice each, or null
  long long ld_partial;
  void *out0, *out1;       // dw: dw_gate, dw_up; else out0
  long long ld_out0, ld_out1;
  int vec_out;             // 2: rows start on 32 bytes, 1: on 16, 0: neither
  float* saved;            // forward: planes g and u, m x ld_saved each, or null
  long long ld_saved;
  int act;
  int* status;
  unsigned long long timeout_ns;
};

// Dense MMA of a CTA pair, both operands from shared memory.
SP24_DEV void tc_mma_dense_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Instruction descriptor, dense kind::f16 with fp32 accumulation (fields as in
// make_idesc_sparse, plus A's major bit).
__host__ __device__ constexpr uint32_t make_idesc_dense(uint32_t fmt, uint32_t n, uint32_t m,
                                                        bool a_mn_major, bool b_mn_major) {
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((a_mn_major ? 1u : 0u) << 15) |
         ((b_mn_major ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

template <int DT, int MODE>
struct FfnCfg {
  static constexpr bool A_MN = MODE == kFfnDw;
  static constexpr bool B_MN = MODE != kFfnForward;
  static constexpr int BK = 64;                       // elements of K per stage
  static constexpr int OPERAND = 128 * BK * 2;        // 16 KB: this CTA's 128 rows of A or B
  static constexpr int STAGE_BYTES = 2 * OPERAND;
  static constexpr int STAGES = 7;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024;
  // MN-major boxes hold 64 of the 128 rows: two of them, 8 KB apart.
  static constexpr int A_BOXES = A_MN ? 2 : 1;
  static constexpr int B_BOXES = B_MN ? 2 : 1;
  static constexpr uint32_t A_LBO = A_MN ? OPERAND / 2 : 16;
  static constexpr uint32_t B_LBO = B_MN ? OPERAND / 2 : 16;
  // Bytes from one MMA's operand (16 of K) to the next: 16 rows of 128 bytes,
  // or 32 bytes along a row.
  static constexpr uint32_t A_STEP = A_MN ? 16 * 128 : 32;
  static constexpr uint32_t B_STEP = B_MN ? 16 * 128 : 32;
  static constexpr uint32_t IDESC = make_idesc_dense(DT == 1 ? 1 : 0, 256, 256, A_MN, B_MN);
  static constexpr int RS = 256 + 4;                  // parked partial row stride (floats)
  static_assert(128 * RS * 4 <= STAGES * STAGE_BYTES, "a parked partial tile fits the ring");
};

// Warp-collective: 64 consecutive 16-bit columns of the lane's own row, as 32
// words of two; the warp's rows are row0 .. row0 + 31 and rows >= m and columns
// >= n are absent.  After the quad transpose (sp24_gemm2sm_kernel.cuh) four lanes
// hold one row's 128 bytes between them and store them in one piece; a ragged
// end costs the last eight columns' lane single elements.
SP24_DEV void store_run64(void* out, long long ld, int vec, uint32_t (&u)[32], int row0, int m,
                          int col0, int n) {
  if (col0 >= n) return;   // warp-uniform
  const int lane = threadIdx.x & 31;
  quad_transpose_units(u);
  const int c = col0 + 16 * (lane & 3), g = lane >> 2;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int row = row0 + 4 * g + q;
    if (row >= m) continue;
    uint16_t* dst = static_cast<uint16_t*>(out) + row * ld + c;
    if (vec == 2 && c + 16 <= n) {
      st_global_v8_u32(dst, &u[8 * q]);
      continue;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t* w = &u[8 * q + 4 * h];
      if (vec > 0 && c + 8 * h + 8 <= n) {
        *reinterpret_cast<uint4*>(dst + 8 * h) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + 8 * h + j < n) dst[8 * h + j] = static_cast<uint16_t>(w[j / 2] >> (16 * (j & 1)));
      }
    }
  }
}

// The same for 32 fp32 columns on rows that start on 32 bytes and are padded to
// multiples of eight: whole units of eight, the last one over the padding.
SP24_DEV void store_run32_f32(float* out, long long ld, uint32_t (&u)[32], int row0, int m, int col0,
                              int n) {
  if (col0 >= n) return;
  const int lane = threadIdx.x & 31;
  quad_transpose_units(u);
  const int c = col0 + 8 * (lane & 3), g = lane >> 2;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int row = row0 + 4 * g + q;
    if (row < m && c < n) st_global_v8_u32(out + row * ld + c, &u[8 * q]);
  }
}

// Activations of the gate (sp24_activation).  Both are g times a sigmoid: silu of g
// itself, the tanh form of gelu of k(g) = sqrt(8 / pi) (g + 0.044715 g^3), since
// (1 + tanh z) / 2 = sigmoid(2 z).  The quotient is the approximate one: the IEEE
// division takes its slow path for the zeroes of absent rows (255 x 64, f = 128,
// one tile less a row: 16.3 -> 6.1 us).
enum : int { kGateNone = 0, kGateSilu = 1, kGateGelu = 2 };
constexpr float kGeluC = 1.5957691216057308f, kGeluA = 0.044715f;

SP24_DEV float gate_act(float g, int act) {
  if (act == kGateSilu) return silu_of(g);
  if (act == kGateGelu) return g * sigmoid_of(kGeluC * g * fmaf(kGeluA * g, g, 1.0f));
  return g;
}

// The activation and its derivative: with s = sigmoid(k), a = g s and
// a' = s + g s (1 - s) k'.
SP24_DEV void gate_act_grad(float g, int act, float& a, float& da) {
  if (act == kGateNone) {
    a = g;
    da = 1.0f;
    return;
  }
  float k = g, dk = 1.0f, gc = g;
  if (act == kGateGelu) {
    // Beyond +-30 the sigmoid is 0 or 1 and g^2 must not overflow into 0 * inf.
    gc = g > 30.0f ? 30.0f : g < -30.0f ? -30.0f : g;
    const float q = kGeluA * gc * gc;
    k = kGeluC * gc * (1.0f + q);
    dk = kGeluC * fmaf(3.0f, q, 1.0f);
  }
  const float s = sigmoid_of(k);
  a = g * s;
  da = s * fmaf(gc * (1.0f - s), dk, 1.0f);
}

SP24_DEV void ffn_tile(const FfnParams& P, int t, int& mt, int& nt) {
  const int per_group = P.group_m * P.n_tiles;
  const int g = t / per_group;
  const int first = g * P.group_m;
  const int gm = min(P.m_tiles - first, P.group_m);
  const int r = t - g * per_group;
  mt = first + r % gm;
  nt = r / gm;
}

// tmA0 / tmA1, tmB0 / tmB1: the operands' two planes (forward: A is x, B0 and B1
// are Wg and Wu; dx: A planes dg and du, B planes Wg and Wu; dw: A planes dg
// and du, B is x).
// KS = 0: clusters of 2, persistent over the units of work.  These are the tiles,
// or (dx over so few tiles that four pairs each would leave most idle) K slices
// of them, whose fp32 sums go to a plane of the workspace each and are added up
// by ffn_dx_sum_kernel.
// KS = 1 (forward or dx over few tiles): a cluster of 2 S CTAs computes one tile, pair p its
// K slice p; each CTA parks its fp32 partial tile in its idle ring, and the
// pairs' partials are summed in order over distributed shared memory.
template <int DT, int MODE, int KS>
SP24_DEV void ffn_pair_body(const CUtensorMap& tmA0, const CUtensorMap& tmA1, const CUtensorMap& tmB0,
                            const CUtensorMap& tmB1, const FfnParams& P) {
#if defined(__CUDA_ARCH__) && (__CUDA_ARCH__ >= 1000)
  using C = FfnCfg<DT, MODE>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[C::STAGES];
  __shared__ __align__(8) uint64_t empty_bar[C::STAGES];
  __shared__ __align__(8) uint64_t accf_bar[2];
  __shared__ __align__(8) uint64_t acce_bar[2];
  __shared__ __align__(8) uint64_t drain_bar;
  __shared__ uint32_t tmem_base_sh;
  __shared__ volatile int abort_sh;

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const uint32_t lead = KS ? (rank & ~1u) : 0u;   // cluster rank of this pair's leader
  const int prank = static_cast<int>(rank - lead);
  const bool leader = prank == 0;
  const uint16_t pair_mask = static_cast<uint16_t>(3u << lead);
  const int pair = KS ? static_cast<int>(blockIdx.x) / (2 * P.splits) : static_cast<int>(blockIdx.x >> 1);
  const int slices = !KS && MODE == kFfnDx ? P.splits : 1;   // units a tile
  const int num_units = P.m_tiles * P.n_tiles * slices;
  const int npairs = KS ? num_units : static_cast<int>(gridDim.x >> 1);   // KS: one tile
  // K stages [first, last) of unit t.
  auto k_range = [&](int t, int& first, int& last) {
    const int all = KS ? P.splits : slices, one = KS ? static_cast<int>(rank >> 1) : t % slices;
    first = static_cast<int>(static_cast<long long>(P.k_stages) * one / all);
    last = static_cast<int>(static_cast<long long>(P.k_stages) * (one + 1) / all);
  };
  const uint64_t tmo = P.timeout_ns;

  if (threadIdx.x == 0) {
    abort_sh = 0;
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accf_bar[b], 1);
      mbar_init(&acce_bar[b], 2 * kPairEpiWarps);
    }
    mbar_init(&drain_bar, 1);
    fence_barrier_init();
    // Every slot is armed for its first use here and re-armed by the MMA warp
    // as soon as it has seen it full.  Both CTAs' bytes land on the leader's
    // barrier; TMA counts zero-filled elements too, so all stages are alike.
    if (leader)
      for (int s = 0; s < C::STAGES; ++s) mbar_arrive_expect_tx(&full_bar[s], 2 * C::STAGE_BYTES);
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA0);
    tma_prefetch_desc(&tmA1);
    tma_prefetch_desc(&tmB0);
    tma_prefetch_desc(&tmB1);
  }
  if (warp == 1) {
    tmem_alloc_pair(&tmem_base_sh, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_sh;
  griddep_launch_dependents();

  if (warp == 0 || warp == kPairBWarp) {
    // ------------------------------------------------------------ producers
    griddep_wait();
    const bool is_b = warp == kPairBWarp;
    const bool mn = is_b ? C::B_MN : C::A_MN;
    const int boxes = is_b ? C::B_BOXES : C::A_BOXES;
    const uint32_t full0 = mapa_shared(smem_u32(&full_bar[0]), lead);
    const uint32_t off = (is_b ? C::OPERAND : 0) + lane * (C::OPERAND / 2);
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    uint32_t used_mask = 0, used_ph = 0;   // slots of the leader's barrier with copies in flight
    for (int t = pair; t < num_units && ok; t += npairs) {
      int mt, nt, ks0, ks1;
      ffn_tile(P, t / slices, mt, nt);
      k_range(t, ks0, ks1);
      const int mplane = MODE == kFfnDw && mt >= P.plane ? 1 : 0;
      if (MODE == kFfnDw) mt -= mplane * P.plane;
      // First row (or, MN-major, first column) of this CTA's 128.
      const int first = is_b ? (MODE == kFfnForward ? nt * 128 : nt * 256 + prank * 128)
                             : mt * 256 + prank * 128;
      for (int ks = ks0; ks < ks1; ++ks) {
        int good = 1;
        if (lane == 0) good = mbar_wait_fast(&empty_bar[s], ph ^ 1u, &abort_sh, tmo) ? 1 : 0;
        if (__shfl_sync(0xffffffffu, good, 0) == 0) {
          ok = false;
          break;
        }
        if (leader && lane == 0) {
          used_mask |= 1u << s;
          used_ph = (used_ph & ~(1u << s)) | (ph << s);
        }
        if (lane < boxes) {
          const int kplane = MODE == kFfnDx && ks >= P.plane ? 1 : 0;
          const int k0 = (ks - kplane * P.plane) * C::BK;
          const bool second = is_b ? (MODE == kFfnForward ? prank == 1 : kplane == 1)
                                   : (mplane | kplane) == 1;
          const CUtensorMap* map = is_b ? (second ? &tmB1 : &tmB0) : (second ? &tmA1 : &tmA0);
          tma_load_2d_pair(smem + s * C::STAGE_BYTES + off, map, full0 + s * sizeof(uint64_t),
                           mn ? first + lane * 64 : k0, mn ? k0 : first);
        }
        if (++s == C::STAGES) s = 0, ph ^= 1u;
      }
    }
    if (!ok && leader && lane == 0) {
      // Error path: copies in flight land before the CTA leaves.
      volatile int dummy = 0;
      for (int i = 0; i < C::STAGES; ++i)
        if (used_mask & (1u << i)) mbar_wait(&full_bar[i], (used_ph >> i) & 1u, &dummy, tmo);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader)
    if (leader) {
      const uint32_t base = smem_u32(smem);
      const uint64_t adesc0 = make_sdesc(base, C::A_LBO, 1024, kLayoutSW128);
      const uint64_t bdesc0 = make_sdesc(base + C::OPERAND, C::B_LBO, 1024, kLayoutSW128);
      int s = 0, buf = 0;
      uint32_t ph = 0, aph = 0;
      bool ok = true, any = false;
      for (int t = pair; t < num_units && ok; t += npairs) {
        int ks0, ks1;
        k_range(t, ks0, ks1);
        if (!mbar_wait_warp<true>(&acce_bar[buf], aph ^ 1u, &abort_sh, tmo)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + static_cast<uint32_t>(buf * 256);
        for (int ks = ks0; ks < ks1; ++ks) {
          if (!mbar_wait_warp(&full_bar[s], ph, &abort_sh, tmo)) {
            ok = false;
            break;
          }
          if (lane == 0) mbar_arrive_expect_tx(&full_bar[s], 2 * C::STAGE_BYTES);
          tc_fence_after();
          if (elect_one()) {
            const uint64_t so = static_cast<uint64_t>(s * (C::STAGE_BYTES >> 4));
#pragma unroll
            for (int j = 0; j < C::BK / 16; ++j)
              tc_mma_dense_pair(d, adesc0 + so + j * (C::A_STEP >> 4),
                                bdesc0 + so + j * (C::B_STEP >> 4), C::IDESC,
                                (ks > ks0 || j > 0) ? 1u : 0u);
            tc_commit_pair(&empty_bar[s], pair_mask);
          }
          __syncwarp();
          any = true;
          if (++s == C::STAGES) s = 0, ph ^= 1u;
        }
        if (!ok) break;
        if (elect_one()) tc_commit_pair(&accf_bar[buf], pair_mask);
        __syncwarp();
        buf ^= 1;
        if (buf == 0) aph ^= 1u;
      }
      if (!ok && any) {
        volatile int dummy = 0;
        if (elect_one()) tc_commit_pair(&drain_bar, static_cast<uint16_t>(1u << lead));
        __syncwarp();
        if (lane == 0) mbar_wait(&drain_bar, 0, &dummy, tmo);
        __syncwarp();
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3;             // TMEM lane quarter
    const int half = (warp - 2) >> 2;   // which half of the tile's columns
    const uint32_t acce0 = mapa_shared(smem_u32(&acce_bar[0]), lead);
    int buf = 0;
    uint32_t aph = 0;
    for (int t = pair; t < num_units; t += npairs) {
      int mt, nt;
      ffn_tile(P, t / slices, mt, nt);
      const int mplane = MODE == kFfnDw && mt >= P.plane ? 1 : 0;
      if (MODE == kFfnDw) mt -= mplane * P.plane;
      bool ok = true;
      if (lane == 0) ok = mbar_wait_sleepy(&accf_bar[buf], aph, &abort_sh, tmo);
      if (__shfl_sync(0xffffffffu, ok ? 1 : 0, 0) == 0) break;
      tc_fence_after();
      const int row0 = mt * 256 + prank * 128 + q * 32;
      const uint32_t tb = tmem_base + (static_cast<uint32_t>(q * 32) << 16) +
                          static_cast<uint32_t>(buf * 256);
      // Two passes: 32 features' g and u (forward), or 64 output columns.
      uint32_t pk[32];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t r0[32], r1[32];
        const uint32_t c0 = tb + (MODE == kFfnForward ? half * 64 + c * 32 : half * 128 + c * 64);
        tmem_ld_x32(c0, r0);
        tmem_ld_x32(c0 + (MODE == kFfnForward ? 128 : 32), r1);
        tmem_ld_wait(r0);
        tmem_ld_wait(r1);
        if (c == 1) {   // all of this warp's columns read: the accumulator is free
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(acce0 + buf * sizeof(uint64_t));
        }
        if constexpr (KS) {
          // Parked at the accumulator's own columns.
          constexpr int R1 = MODE == kFfnForward ? 128 : 32;
          float* red = reinterpret_cast<float*>(smem) + (q * 32 + lane) * C::RS + (c0 - tb);
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            *reinterpret_cast<uint4*>(red + j) = make_uint4(r0[j], r0[j + 1], r0[j + 2], r0[j + 3]);
            *reinterpret_cast<uint4*>(red + R1 + j) = make_uint4(r1[j], r1[j + 1], r1[j + 2], r1[j + 3]);
          }
        } else if (MODE == kFfnDx && P.partial != nullptr) {
          float* part = P.partial + (t % slices) * (P.m * P.ld_partial);
          const int col0 = nt * 256 + half * 128 + c * 64;
          store_run32_f32(part, P.ld_partial, r0, row0, P.m, col0, P.n);
          store_run32_f32(part, P.ld_partial, r1, row0, P.m, col0 + 32, P.n);
        } else if constexpr (MODE == kFfnForward) {
          const int col0 = nt * 128 + half * 64;
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            float h[2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
              h[e] = gate_act(__uint_as_float(r0[j + e]), P.act) * __uint_as_float(r1[j + e]);
            pk[(c * 32 + j) / 2] = pack16<DT>(h[0], h[1]);
          }
          if (P.saved != nullptr) {
            store_run32_f32(P.saved, P.ld_saved, r0, row0, P.m, col0 + c * 32, P.n);
            store_run32_f32(P.saved + P.m * P.ld_saved, P.ld_saved, r1, row0, P.m, col0 + c * 32, P.n);
          }
          if (c == 1) store_run64(P.out0, P.ld_out0, P.vec_out, pk, row0, P.m, col0, P.n);
        } else {
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            pk[j / 2] = pack16<DT>(__uint_as_float(r0[j]), __uint_as_float(r0[j + 1]));
            pk[16 + j / 2] = pack16<DT>(__uint_as_float(r1[j]), __uint_as_float(r1[j + 1]));
          }
          store_run64(mplane ? P.out1 : P.out0, mplane ? P.ld_out1 : P.ld_out0, P.vec_out, pk, row0,
                      P.m, nt * 256 + half * 128 + c * 64, P.n);
        }
      }
      buf ^= 1;
      if (buf == 0) aph ^= 1u;
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();   // KS: every pair's partial is parked and visible (release / acquire)
  if constexpr (KS) {
    // CTA (slice p, half h) finishes rows [128 p / S, 128 (p + 1) / S) of its half
    // of the tile, four output columns a thread.
    static_assert(MODE != kFfnDw, "the K-split forms");
    const int S = P.splits;
    int mt, nt;
    ffn_tile(P, pair, mt, nt);
    const int split = static_cast<int>(rank >> 1);
    const int r0 = 128 * split / S, rows = 128 * (split + 1) / S - r0;
    const float* red = reinterpret_cast<const float*>(smem);
    // Sum over the slices of four parked columns; all loads on their way first.
    auto total = [&](int rl, int cl) {
      const uint32_t la = smem_u32(red + rl * C::RS + cl);
      float4 v[kFfnMaxSplits];
#pragma unroll
      for (int sp = 0; sp < kFfnMaxSplits; ++sp)
        if (sp < S) v[sp] = ld_dsmem_f4(mapa_shared(la, static_cast<uint32_t>(2 * sp + prank)));
      float4 a = v[0];
#pragma unroll
      for (int sp = 1; sp < kFfnMaxSplits; ++sp)
        if (sp < S) a.x += v[sp].x, a.y += v[sp].y, a.z += v[sp].z, a.w += v[sp].w;
      return a;
    };
    constexpr int COLS = MODE == kFfnForward ? 128 : 256;   // output columns of a tile
    for (int i = threadIdx.x; i < rows * (COLS / 4); i += kPairThreads) {
      const int rl = r0 + i / (COLS / 4), cl = i % (COLS / 4) * 4;
      float4 a = total(rl, cl);
      const int row = mt * 256 + prank * 128 + rl, col = nt * COLS + cl;
      if constexpr (MODE == kFfnForward) {
        const float4 u = total(rl, 128 + cl);
        if (P.saved != nullptr && row < P.m && col < P.n) {   // whole units, the last over the padding
          float* g = P.saved + row * P.ld_saved + col;
          *reinterpret_cast<float4*>(g) = a;
          *reinterpret_cast<float4*>(g + P.m * P.ld_saved) = u;
        }
        a = make_float4(gate_act(a.x, P.act) * u.x, gate_act(a.y, P.act) * u.y, gate_act(a.z, P.act) * u.z,
                        gate_act(a.w, P.act) * u.w);
      }
      if (row >= P.m) continue;
      uint16_t* dst = static_cast<uint16_t*>(P.out0) + row * P.ld_out0 + col;
      const uint32_t w[2] = {pack16<DT>(a.x, a.y), pack16<DT>(a.z, a.w)};
      if (P.vec_out > 0 && col + 4 <= P.n) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (col + j < P.n) dst[j] = static_cast<uint16_t>(w[j / 2] >> (16 * (j & 1)));
      }
    }
    cluster_sync();   // no CTA leaves while others still read its shared memory
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
  if (threadIdx.x == 0 && abort_sh != 0 && P.status != nullptr) atomicExch(P.status, 1);
#endif
}

template <int DT, int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    ffn_pair_kernel(const __grid_constant__ CUtensorMap tmA0, const __grid_constant__ CUtensorMap tmA1,
                    const __grid_constant__ CUtensorMap tmB0, const __grid_constant__ CUtensorMap tmB1,
                    const FfnParams P) {
  ffn_pair_body<DT, MODE, 0>(tmA0, tmA1, tmB0, tmB1, P);
}

// Launched with a run-time cluster of 2 * P.splits CTAs.
template <int DT, int MODE>
__global__ void __launch_bounds__(kPairThreads, 1)
    ffn_split_kernel(const __grid_constant__ CUtensorMap tmA0, const __grid_constant__ CUtensorMap tmA1,
                        const __grid_constant__ CUtensorMap tmB0, const __grid_constant__ CUtensorMap tmB1,
                        const FfnParams P) {
  ffn_pair_body<DT, MODE, 1>(tmA0, tmA1, tmB0, tmB1, P);
}

// dx from the K slices' planes of m x ld fp32 sums: a block finishes 32 runs of
// eight columns, its warp w adding up slices [w S / 8, (w + 1) S / 8) of each (the
// slices are many where the runs are few, and one thread's chain of loads would
// be all latency); the eight sums are then added in order.  VEC: dx's rows start
// on 16 bytes.
template <int DT, int VEC>
__global__ void __launch_bounds__(256)
    ffn_dx_sum_kernel(const float* __restrict__ part, int splits, int m, int n, long long ld, void* __restrict__ out,
                      long long ldo) {
  __shared__ float4 sums[8][2][32];
  griddep_launch_dependents();
  griddep_wait();
  const int per_row = (n + 7) / 8, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const long long unit = blockIdx.x * 32LL + lane, plane = m * ld;
  const long long row = unit / per_row;
  const int col = static_cast<int>(unit - row * per_row) * 8;
  float4 a = make_float4(0, 0, 0, 0), b = a;
  if (row < m) {
    const float* p = part + row * ld + col;
#pragma unroll 4
    for (int s = splits * w / 8; s < splits * (w + 1) / 8; ++s) {
      const float4 x = *reinterpret_cast<const float4*>(p + s * plane);
      const float4 y = *reinterpret_cast<const float4*>(p + s * plane + 4);
      a.x += x.x, a.y += x.y, a.z += x.z, a.w += x.w;
      b.x += y.x, b.y += y.y, b.z += y.z, b.w += y.w;
    }
  }
  sums[w][0][lane] = a;
  sums[w][1][lane] = b;
  __syncthreads();
  if (w != 0 || row >= m) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    const float4 x = sums[i][0][lane], y = sums[i][1][lane];
    a.x += x.x, a.y += x.y, a.z += x.z, a.w += x.w;
    b.x += y.x, b.y += y.y, b.z += y.z, b.w += y.w;
  }
  const uint32_t k[4] = {pack16<DT>(a.x, a.y), pack16<DT>(a.z, a.w), pack16<DT>(b.x, b.y), pack16<DT>(b.z, b.w)};
  uint16_t* o = static_cast<uint16_t*>(out) + row * ldo + col;
  if (VEC && col + 8 <= n) {
    *reinterpret_cast<uint4*>(o) = make_uint4(k[0], k[1], k[2], k[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + j < n) o[j] = static_cast<uint16_t>(k[j / 2] >> (16 * (j & 1)));
  }
}

// dg = d_out u act'(g) and du = d_out act(g) from the saved fp32 sums, rounded
// to 16 bits: eight columns a thread, rows of ld (a multiple of 8) elements.
// Bound by HBM: 14 bytes an element (4096 x 14336: 822 MB in 126 us, 6.5 TB/s).
// Only the units of eight that hold a column below f are walked: d_out has no
// padding to read, and the products' tensor maps end at f.  A last unit past f is
// written whole (the saved sums there are whatever the buffer holds).
// VEC: d_out's rows start on 16 bytes and f is a multiple of 8.
template <int DT, int VEC>
__global__ void __launch_bounds__(256)
    ffn_dgate_kernel(int t, int f, const float* __restrict__ saved, long long ld,
                     const void* __restrict__ d_out, long long ldd, int act,
                     uint16_t* __restrict__ dgu) {
  griddep_launch_dependents();
  griddep_wait();
  const long long per_row = (f + 7) / 8, total = per_row * t, plane = ld * t;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const long long row = i / per_row;
    const int col = static_cast<int>(i - row * per_row) * 8;
    const float* gp = saved + row * ld + col;
    float g[8], u[8], d[8];
    *reinterpret_cast<float4*>(g) = *reinterpret_cast<const float4*>(gp);
    *reinterpret_cast<float4*>(g + 4) = *reinterpret_cast<const float4*>(gp + 4);
    *reinterpret_cast<float4*>(u) = *reinterpret_cast<const float4*>(gp + plane);
    *reinterpret_cast<float4*>(u + 4) = *reinterpret_cast<const float4*>(gp + plane + 4);
    if constexpr (VEC) {
      const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(d_out) + row * ldd + col);
      const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = load16<DT>(&ws[j / 2], j & 1);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = col + j < f ? load16<DT>(d_out, row * ldd + col + j) : 0.0f;
    }
    uint32_t og[4], ou[4];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      float dg[2], du[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float x = g[j + e];
        float a, da;
        gate_act_grad(x, act, a, da);
        du[e] = d[j + e] * a;
        dg[e] = d[j + e] * u[j + e] * da;
      }
      og[j / 2] = pack16<DT>(dg[0], dg[1]);
      ou[j / 2] = pack16<DT>(du[0], du[1]);
    }
    uint16_t* o = dgu + row * ld + col;
    *reinterpret_cast<uint4*>(o) = make_uint4(og[0], og[1], og[2], og[3]);
    *reinterpret_cast<uint4*>(o + plane) = make_uint4(ou[0], ou[1], ou[2], ou[3]);
  }
}

}  // namespace sp24
