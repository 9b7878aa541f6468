// sp24_scaled_pair_kernel.cuh — the 8-bit 2:4 product with channel and token
// scales on CTA pairs, for many tokens.
//
//   acc[r][t] = sum_k W[r][k] x[t][k]        tcgen05.mma.sp.cta_group::2, M = 256,
//   c[t][r]   = acc * scale_m[r] * scale_n[t] + bias[r]    N = BN, K = 64 per MMA
//
// Two tiles.  The tensor pipe takes about 11.6k multiply-adds a clock and SM of
// this kind, an SM takes in about 64 bytes a clock (bin/sp24_feed_probe),
// and compressed weights are the cheaper operand (half the values, plus an eighth
// for the codes).
//   MB = 2, BN = 224  two blocks of 256 weight rows against one staged block of
//                     tokens: 68 KB per 1270 clocks of MMAs and 256 of K.  The
//                     accumulators take 2 x 224 TMEM columns and the metadata
//                     buffers most of the rest, so they are single-buffered;
//                     the epilogue hands each back once its columns are in
//                     registers.  A last wave that would fill at most half the
//                     pairs is dealt block by block.
//   MB = 1, BN = 128  36 KB per 360 clocks: more loading per product, but twice
//                     as many tiles in both directions and two accumulator
//                     buffers, for calls that do not fill the GPU with the other.
// 14336 x 4096 int8, 4096 tokens (481 dense-equivalent GFLOP): 130-134 us in a
// burst, 145-148 held under the 1000 W cap at 1.69 GHz, where the MMAs alone would
// take 86.  Filling the stages and feeding the MMAs slow each other: without its
// stores the kernel takes 115 us, without its MMAs 114, without its loads 117.
// Measured and not kept (times held under the cap): 128-byte store lines (144 against 144), cache policies on weights or
// output (the same), both accumulators packed before the first store (164),
// starting block 0 while block 1 drains (148; with three stages ahead 147), three
// accumulators of 160 columns, so that every epilogue overlaps (155 against 141),
// one block x 224 tokens with two accumulators (146 against 144), 128-deep stages
// in a ring twice as long (188: their 64-byte weight rows load slower).
//
// Accumulator lanes are weight rows, i.e. neighbouring features of a token's
// output row: a warp's store of one token is one contiguous 64-byte run.
//
// Roles per CTA: warps 0-7 drain the accumulators, warp 8 loads weights and
// metadata, warp 10 the tokens, warp 9 of the leader issues the MMAs.
#pragma once

#include "sp24_gemm2sm_kernel.cuh"
#include "sp24_ptx.cuh"
#include "sp24_stream_kernel.cuh"

namespace sp24 {

constexpr int kScaledThreads = 352;   // 11 warps: 0-7 epilogue, then one role each
constexpr int kScaledAWarp = 8, kScaledMmaWarp = 9, kScaledBWarp = 10;

struct ScaledPairParams {
  int m, n, k;
  int m_tiles, n_tiles, k_stages;
  int items;          // units of work: whole tiles, then
  int whole_items;    // single blocks of the tiles from whole_items on (MB = 2)
  int group_m;
  int meta_mblocks;
  const float *scale_m, *scale_n, *bias;
  void* out;
  long long ldo;
  int out_type;
  int words;          // 16-bit output rows start on 4-byte boundaries
  int static_weights;
  int* status;
  unsigned long long timeout_ns;
};

template <int I8, int MB, int BN>
struct ScaledPairCfg {
  static constexpr int BKD = 256;                       // dense K per stage (rows of 128 bytes)
  static constexpr int MMAS = BKD / 64;
  static constexpr int A_BOX = kBlockM * 128;
  static constexpr int A_BYTES = MB * A_BOX;
  static constexpr int HALF = BN / 2;                   // tokens staged per CTA
  static constexpr int B_BOX = HALF * 128;
  static constexpr int B_BOXES = BKD / 128;
  static constexpr int B_BYTES = B_BOXES * B_BOX;
  static constexpr int ATOMS = BKD / 128;               // per block
  static constexpr int E_BYTES = MB * ATOMS * kAtomBytes;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + E_BYTES;
  static constexpr int STAGES_RAW = (kSmemBudget - 5 * 1024) / STAGE_BYTES;
  static constexpr int STAGES = STAGES_RAW > 8 ? 8 : STAGES_RAW;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024;
  // TMEM: accumulator b at column 256 b, two of four metadata buffers after each.
  static constexpr int E_COL = BN;
  static constexpr uint32_t IDESC =
      I8 ? ((1u << 2) | (2u << 4) | (1u << 7) | (1u << 10) | ((BN >> 3) << 17) | ((256u >> 4) << 24))
         : make_idesc_sparse(0, BN, 256, false);
  static constexpr int CW = BN / 2;                     // columns per epilogue warp
  static_assert(BN % 32 == 0 && BN + 2 * MB * ATOMS * 4 <= 256, "tokens per tile");
  static_assert(B_BOX % 1024 == 0 && STAGE_BYTES % 1024 == 0, "boxes stay 1024-aligned");
  static_assert(STAGES >= 3, "ring");
};

SP24_DEV void tc_mma_sp_pair_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t e, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.sp.cta_group::2.kind::i8 [%0], %1, %2, [%3], %4, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(e), "r"(idesc), "r"(acc)
      : "memory");
}

// Unit of work `it`: tile column nt, `blocks` blocks of 256 weight rows from `block`.
template <int MB>
SP24_DEV void scaled_item(const ScaledPairParams& P, int it, int& nt, int& block, int& blocks) {
  const int half = it - P.whole_items;
  const int t = half < 0 ? it : P.whole_items + half / MB;
  const int per_group = P.group_m * P.n_tiles;
  const int g = t / per_group;
  const int first = g * P.group_m;
  const int gm = min(P.m_tiles - first, P.group_m);
  const int r = t - g * per_group;
  nt = r / gm;
  block = (first + r % gm) * MB + (half < 0 ? 0 : half % MB);
  blocks = half < 0 ? MB : 1;
}

template <int I8>
SP24_DEV float sum_value(uint32_t a) {
  return I8 ? static_cast<float>(static_cast<int>(a)) : __uint_as_float(a);
}

// Warp-collective: CW accumulator columns (tokens t0 ..) of 32 weight rows, lane
// l holding row `row` = row0 + l, scaled and stored.  sn: the tokens' scales in
// shared memory.  The epilogue is bound by instruction issue (eight warps, two
// blocks of 112 columns each), hence the paired arithmetic, and 16-bit outputs
// leave as whole words: neighbouring lanes swap halves, so that even lanes store
// two rows of one token and odd lanes of the next (words: rows start on words).
template <int I8, int CW, int OUT>
SP24_DEV void scaled_emit(const ScaledPairParams& P, const uint32_t (&r)[CW], int row, int t0, const float* sn) {
  const int lane = threadIdx.x & 31;
  const bool live = row < P.m;
  const float sm1 = live && P.scale_m != nullptr ? P.scale_m[row] : 1.0f;
  const float b1 = live && P.bias != nullptr ? P.bias[row] : 0.0f;
  const float2 sm = make_float2(sm1, sm1), bias = make_float2(b1, b1);
  auto value2 = [&](int j) {
    const float2 s = *reinterpret_cast<const float2*>(sn + j);
    return fma2(make_float2(sum_value<I8>(r[j]), sum_value<I8>(r[j + 1])), mul2(sm, s), bias);
  };
  const int left = P.n - t0;   // tokens from t0 on
  if constexpr (OUT == 2) {
    if (!live) return;
    float* p = static_cast<float*>(P.out) + t0 * P.ldo + row;
#pragma unroll
    for (int j = 0; j < CW; j += 2) {
      const float2 v = value2(j);
      if (j < left) p[0] = v.x;
      if (j + 1 < left) p[P.ldo] = v.y;
      p += 2 * P.ldo;
    }
  } else if (P.words && left >= CW && row - lane + 32 <= P.m) {
    const int odd = lane & 1;
    const uint32_t sel = odd ? 0x3276u : 0x5410u;
    uint16_t* p = static_cast<uint16_t*>(P.out) + (t0 + odd) * P.ldo + (row - odd);
#pragma unroll
    for (int j = 0; j < CW; j += 2) {
      const float2 v = value2(j);
      const uint32_t mine = pack16<OUT>(v.x, v.y);
      *reinterpret_cast<uint32_t*>(p) = __byte_perm(mine, __shfl_xor_sync(0xffffffffu, mine, 1), sel);
      p += 2 * P.ldo;
    }
  } else if (live) {
    uint16_t* p = static_cast<uint16_t*>(P.out) + t0 * P.ldo + row;
#pragma unroll
    for (int j = 0; j < CW; j += 2) {
      const float2 v = value2(j);
      const uint32_t w = pack16<OUT>(v.x, v.y);
      if (j < left) p[0] = static_cast<uint16_t>(w);
      if (j + 1 < left) p[P.ldo] = static_cast<uint16_t>(w >> 16);
      p += 2 * P.ldo;
    }
  }
}

// tmA: a_c, tmB: tokens, tmE: the metadata image as rows of 256 bytes (8 to an atom).
template <int I8, int MB, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kScaledThreads, 1)
    scaled_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                       const __grid_constant__ CUtensorMap tmE, const ScaledPairParams P) {
#if defined(__CUDA_ARCH__) && (__CUDA_ARCH__ >= 1000)
  using C = ScaledPairCfg<I8, MB, BN>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[C::STAGES];
  __shared__ __align__(8) uint64_t empty_bar[C::STAGES];
  __shared__ __align__(8) uint64_t accf_bar[2 / MB];
  __shared__ __align__(8) uint64_t acce_bar[2];
  __shared__ __align__(8) uint64_t drain_bar;
  __shared__ __align__(16) float sn_sh[kPairEpiWarps][C::CW];   // each epilogue warp's token scales
  __shared__ uint32_t tmem_base_sh;
  __shared__ volatile int abort_sh;

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int prank = static_cast<int>(cluster_ctarank());
  const bool leader = prank == 0;
  const int pair = static_cast<int>(blockIdx.x >> 1);
  const int npairs = static_cast<int>(gridDim.x >> 1);
  const uint64_t tmo = P.timeout_ns;
  // Bytes of both CTAs for the stage `ahead` of the first stage of unit `it`.
  auto stage_tx = [&](int it, int ahead) {
    if (ahead >= P.k_stages) it += ahead / P.k_stages * npairs;
    const int blocks = it < P.whole_items ? MB : 1;
    return static_cast<uint32_t>(2 * (blocks * (C::A_BOX + C::ATOMS * kAtomBytes) + C::B_BYTES));
  };

  if (threadIdx.x == 0) {
    abort_sh = 0;
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2 / MB; ++b) mbar_init(&accf_bar[b], 1);
    for (int b = 0; b < 2; ++b) mbar_init(&acce_bar[b], 2 * kPairEpiWarps);
    mbar_init(&drain_bar, 1);
    fence_barrier_init();
    // Armed here for the first use, by the MMA warp for later ones; both CTAs'
    // bytes land on the leader's barriers (TMA counts zero-filled ones too).
    if (leader)
      for (int s = 0; s < C::STAGES; ++s) mbar_arrive_expect_tx(&full_bar[s], stage_tx(pair, s));
  }
  if (warp == kScaledAWarp && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmE);
  }
  if (warp == kScaledMmaWarp) {
    tmem_alloc_pair(&tmem_base_sh, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_sh;
  griddep_launch_dependents();

  if (warp == kScaledAWarp || warp == kScaledBWarp) {
    // ------------------------------------------------------------ producers
    // A: lanes 0 .. MB-1 a block of 128 a_c rows each, then an atom a lane;
    // B: the stage's tokens in boxes 128 bytes wide.
    const bool is_b = warp == kScaledBWarp;
    if (is_b || !P.static_weights) griddep_wait();
    const bool is_a = !is_b && lane < MB;
    const int el = lane - MB;                           // block el / ATOMS, its atom el % ATOMS
    const CUtensorMap* map = is_b ? &tmB : is_a ? &tmA : &tmE;
    const uint32_t off = is_b   ? C::A_BYTES + lane * C::B_BOX
                         : is_a ? lane * C::A_BOX
                                : C::A_BYTES + C::B_BYTES + el * kAtomBytes;
    const int dx = is_b ? C::BKD : is_a ? C::BKD / 2 : 0;
    const int dy = is_b || is_a ? 0 : C::ATOMS * P.meta_mblocks * 8;
    const uint32_t full0 = mapa_shared(smem_u32(&full_bar[0]), 0);
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    uint32_t used_mask = 0, used_ph = 0;
    for (int it = pair; it < P.items && ok; it += npairs) {
      int nt, block, blocks;
      scaled_item<MB>(P, it, nt, block, blocks);
      int x = is_b ? lane * 128 : 0, y;
      bool loads;
      if (is_b) {
        loads = lane < C::B_BOXES;
        y = nt * BN + prank * C::HALF;
      } else if (is_a) {
        loads = lane < blocks;
        y = (block + lane) * 256 + prank * 128;
      } else {
        loads = el < blocks * C::ATOMS;
        // Blocks past the image belong to rows past m: any valid codes serve.
        const int mb = min((block + el / C::ATOMS) * 2 + prank, P.meta_mblocks - 1);
        y = ((el % C::ATOMS) * P.meta_mblocks + mb) * 8;
      }
      for (int ks = 0; ks < P.k_stages; ++ks) {
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
        if (loads)
          tma_load_2d_pair(smem + s * C::STAGE_BYTES + off, map, full0 + s * sizeof(uint64_t), x, y);
        x += dx;
        y += dy;
        if (++s == C::STAGES) s = 0, ph ^= 1u;
      }
    }
    if (!ok && leader && lane == 0) {
      // Error path: copies in flight land before the CTA leaves.
      volatile int dummy = 0;
      for (int i = 0; i < C::STAGES; ++i)
        if (used_mask & (1u << i)) mbar_wait(&full_bar[i], (used_ph >> i) & 1u, &dummy, tmo);
    }
  } else if (warp == kScaledMmaWarp) {
    // ------------------------------------------------------------ MMA issuer (leader)
    if (leader) {
      const uint32_t base = smem_u32(smem);
      const uint64_t adesc0 = make_sdesc(base, 16, 1024, kLayoutSW128);
      const uint64_t bdesc0 = make_sdesc(base + C::A_BYTES, 16, 1024, kLayoutSW128);
      const uint64_t edesc0 = make_sdesc(base + C::A_BYTES + C::B_BYTES, kAtomBytes, 128, kLayoutNone);
      int s = 0;
      uint32_t ph = 0, aph = 0, eb = 0, acc0 = 0;   // acc0: this unit's first accumulator
      bool ok = true, any = false;
      for (int it = pair; it < P.items && ok; it += npairs) {
        int nt, block, blocks;
        scaled_item<MB>(P, it, nt, block, blocks);
        // Block b of a stage: its products, once the metadata is on its way.
        auto products = [&](int ks, uint32_t e, int b) {
          const int kleft = P.k - ks * C::BKD;
          const uint64_t so = static_cast<uint64_t>(s * (C::STAGE_BYTES >> 4));
          if ((block + b) * 256 < P.m && elect_one()) {
#pragma unroll
            for (int j = 0; j < C::MMAS; ++j)
              if (j * 64 < kleft) {   // past K there is no metadata
                const uint64_t ad = adesc0 + so + b * (C::A_BOX >> 4) + j * 2;
                const uint64_t bd = bdesc0 + so + (j >> 1) * (C::B_BOX >> 4) + (j & 1) * 4;
                const uint32_t d = tmem_base + (acc0 + b) * 256, ec = e + b * C::ATOMS * 4 + j * 2;
                const uint32_t acc = (ks > 0 || j > 0) ? 1u : 0u;
                if constexpr (I8) tc_mma_sp_pair_i8(d, ad, bd, ec, C::IDESC, acc);
                else tc_mma_sp_pair<1>(d, ad, bd, ec, C::IDESC, acc);
              }
          }
          __syncwarp();
        };
        // The last unit's columns of these accumulators are in registers.
        for (int b = 0; b < blocks && ok; ++b) ok = mbar_wait_warp<true>(&acce_bar[acc0 + b], aph ^ 1u, &abort_sh, tmo);
        if (!ok) break;
        tc_fence_after();
        for (int ks = 0; ks < P.k_stages; ++ks) {
          if (!mbar_wait_warp(&full_bar[s], ph, &abort_sh, tmo)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t e = tmem_base + (eb & 1u) * 256 + C::E_COL + (eb >> 1 & 1u) * (MB * C::ATOMS * 4);
          ++eb;
          if (elect_one()) {
            const uint64_t ed = edesc0 + static_cast<uint64_t>(s * (C::STAGE_BYTES >> 4));
#pragma unroll
            for (int a = 0; a < MB * C::ATOMS; ++a)
              if (a < blocks * C::ATOMS) tc_cp<2>(e + 4 * a, ed + a * (kAtomBytes >> 4));
          }
          __syncwarp();
          any = true;
          products(ks, e, 0);
          if (blocks == 2) products(ks, e, 1);
          // Armed for the slot's next use only now, off the products' path; freed
          // once they are done.
          if (lane == 0) mbar_arrive_expect_tx(&full_bar[s], stage_tx(it, ks + C::STAGES));
          __syncwarp();
          if (elect_one()) tc_commit_pair(&empty_bar[s], 3);
          __syncwarp();
          if (++s == C::STAGES) s = 0, ph ^= 1u;
        }
        if (!ok) break;
        if (elect_one()) tc_commit_pair(&accf_bar[MB == 1 ? acc0 : 0], 3);
        __syncwarp();
        if (MB == 1) acc0 ^= 1u;
        if (acc0 == 0) aph ^= 1u;
      }
      if (!ok && any) {
        volatile int dummy = 0;
        if (elect_one()) tc_commit_pair(&drain_bar, 1);
        __syncwarp();
        if (lane == 0) mbar_wait(&drain_bar, 0, &dummy, tmo);
        __syncwarp();
      }
    }
  } else if (warp < kPairEpiWarps) {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3;
    const int half = warp >> 2;
    const uint32_t acce0 = mapa_shared(smem_u32(&acce_bar[0]), 0);
    uint32_t aph = 0, acc0 = 0;
    griddep_wait();   // scales and bias may come from the previous kernel
    for (int it = pair; it < P.items; it += npairs) {
      int nt, block, blocks;
      scaled_item<MB>(P, it, nt, block, blocks);
      float* sn = sn_sh[warp];
      __syncwarp();
      for (int j = lane; j < C::CW; j += 32) {
        const int tok = nt * BN + half * C::CW + j;
        sn[j] = P.scale_n != nullptr && tok < P.n ? P.scale_n[tok] : 1.0f;
      }
      __syncwarp();
      bool ok = true;
      if (lane == 0) ok = mbar_wait_sleepy(&accf_bar[MB == 1 ? acc0 : 0], aph, &abort_sh, tmo);
      if (__shfl_sync(0xffffffffu, ok ? 1 : 0, 0) == 0) break;
      tc_fence_after();
      const int t0 = nt * BN + half * C::CW;
#pragma unroll 1
      for (int b = 0; b < MB; ++b) {
        const int row = (block + b) * 256 + prank * 128 + q * 32 + lane;
        if (b >= blocks) {
          if (lane == 0) mbar_arrive_cluster(acce0 + (acc0 + b) * sizeof(uint64_t));
          continue;
        }
        uint32_t r[C::CW];
        const uint32_t tb = tmem_base + (static_cast<uint32_t>(q * 32) << 16) +
                            (acc0 + b) * 256 + half * C::CW;
#pragma unroll
        for (int c = 0; c < C::CW; c += 16) tmem_ld_x16(tb + c, *reinterpret_cast<uint32_t(*)[16]>(&r[c]));
        tmem_ld_wait(r);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(acce0 + (acc0 + b) * sizeof(uint64_t));
        if (row - lane >= P.m) continue;
        if (P.out_type == 2) scaled_emit<I8, C::CW, 2>(P, r, row, t0, sn);
        else if (P.out_type == 1) scaled_emit<I8, C::CW, 1>(P, r, row, t0, sn);
        else scaled_emit<I8, C::CW, 0>(P, r, row, t0, sn);
      }
      if (MB == 1) acc0 ^= 1u;
      if (acc0 == 0) aph ^= 1u;
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == kScaledMmaWarp) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
  if (threadIdx.x == 0 && abort_sh != 0 && P.status != nullptr) atomicExch(P.status, 1);
#endif
}

}  // namespace sp24
