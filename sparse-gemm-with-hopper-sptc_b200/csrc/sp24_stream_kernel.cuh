// sp24_stream_kernel.cuh — the MLP block's products over few tokens, bound by
// streaming the weights from HBM once:
//   scaled   8-bit 2:4 weights x tokens with channel and token scales
//            (tcgen05.mma.sp, kind::i8 or kind::f8f6f4);
//   ffn      dense 16-bit Wg and Wu x tokens, act(g) * u (tcgen05.mma,
//            kind::f16): both weights stream through one ring against one
//            staged B, into two accumulators.
//
// The weights' rows are the MMA's M (128 a CTA) and the tokens its N (BN), so a
// single token costs a 16-column MMA and not a 128-row one.  Both operands are
// K-major as they lie in memory.  Where the row blocks alone cannot occupy the
// GPU, K is split over the S CTAs of a cluster; their partial tiles are summed
// in rank order over distributed shared memory (int32 for kind::i8), so results
// do not depend on timing.  No workspace, no atomics, one launch.
//
// Accumulator lanes are weight rows, i.e. neighbouring features of a token's
// output row: a warp's stores of one column are one contiguous run.
//
// Measured (device time in a graph, B200, weights from HBM at a copy rate of 6.5
// TB/s): gated block 4096 -> 14336 bf16, one token: 235 MB in 39-41 us, 5.7-6.0 TB/s;
// int8 product 4096 -> 14336, one token: 36.8 MB in 9.5 us, of which about 4 are
// launch, first loads and drain (a 10 MB product takes 5.5); 32 tokens through
// 14336 -> 4096 e4m3, K split in four: 11.5 us.  Bytes in flight decide the rest: a
// ring of 110 KB instead of 190 costs 20%, and two CTAs an SM with half a ring
// each 5-8%.
//
// Roles (6 warps): warp 0 loads (one copy a lane), warp 1 issues the MMAs,
// warps 2-5 drain the accumulator.
#pragma once

#include "sp24_ffn_kernel.cuh"
#include "sp24_gemm_kernel.cuh"
#include "sp24_ptx.cuh"
#include "sp24_rows.cuh"

namespace sp24 {

enum : int { kStreamI8 = 0, kStreamE4M3 = 1, kStreamF16 = 2, kStreamBF16 = 3 };
constexpr int kStreamThreads = 192;
constexpr int kStreamMaxSplits = 8;

struct StreamParams {
  int m, n, k;              // weight rows, tokens, K
  int m_blocks;
  int splits;               // S
  int stages;               // K stages over all splits
  int ring;                 // slots, at most C::STAGES
  const uint8_t* meta;      // scaled: tcgen05 metadata image
  int meta_mblocks, katoms;
  const float *scale_m, *scale_n, *bias;
  void* out;                // n x m
  long long ldo;
  int out_type;             // 0 f16, 1 bf16, 2 f32
  float* saved;             // ffn: planes of n x ld_saved, or null
  long long ld_saved;
  int act;
  int static_weights;       // weights are not written by in-flight work: their first
                            // ring of loads may precede the wait for it
  int* status;
  unsigned long long timeout_ns;
};

template <int OP, int BN>
struct StreamCfg {
  static constexpr bool SPARSE = OP <= kStreamE4M3;
  static constexpr int G = SPARSE ? 1 : 2;               // weights streamed
  static constexpr int BKD = SPARSE ? 256 : 64;          // dense K per stage: 128 bytes of A
  static constexpr int MMA_K = SPARSE ? 64 : 16;
  static constexpr int MMAS = BKD / MMA_K;               // 4
  static constexpr int A_COLS = SPARSE ? 128 : 64;       // elements of an A box row
  static constexpr int A_BOX = kBlockM * 128;
  static constexpr int A_BYTES = G * A_BOX;
  static constexpr int B_BOXES = SPARSE ? 2 : 1;         // 128-byte wide boxes of BN tokens
  static constexpr int B_COLS = SPARSE ? 128 : 64;
  static constexpr int B_BOX = BN * 128;
  static constexpr int B_BYTES = B_BOXES * B_BOX;
  static constexpr int ATOMS = SPARSE ? 2 : 0;           // metadata atoms per stage
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + ATOMS * kAtomBytes;
  static constexpr int STAGES_RAW = (kSmemBudget - 1024) / STAGE_BYTES;
  static constexpr int STAGES = STAGES_RAW > 8 ? 8 : STAGES_RAW;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024;
  static constexpr int PARKED = G * BN * (kBlockM + 4) * 4;   // a partial tile, in the idle ring
  static constexpr int LOADS = G + B_BOXES + ATOMS;
  static constexpr int E_COL = G * BN;
  static constexpr int COLS_NEEDED = E_COL + 2 * ATOMS * 4;
  static constexpr uint32_t TMEM_COLS = COLS_NEEDED <= 32    ? 32
                                        : COLS_NEEDED <= 64  ? 64
                                        : COLS_NEEDED <= 128 ? 128
                                        : COLS_NEEDED <= 256 ? 256
                                                             : 512;
  // The least shared memory a launch asks for.  CTAs that wait on one another
  // (clusters) must never wait for TMEM that another waiting CTA holds, so no mix
  // of this library's CTAs that fits an SM's shared memory may want more than its
  // 512 columns: a CTA asks for at least the share of 228 KB that its columns are
  // of 512, and for more than the pair kernels, which take all columns, leave free
  // (50 KB).
  static constexpr int MIN_SMEM = (TMEM_COLS * 228 / 512 < 56 ? 56 : static_cast<int>(TMEM_COLS * 228 / 512)) * 1024;
  static_assert(MIN_SMEM <= SMEM_BYTES, "room for the least request");
  // Descriptor fields as in make_idesc_sparse; kind::i8 has D = s32 (2) and
  // signed A and B (1).
  static constexpr uint32_t IDESC =
      !SPARSE ? make_idesc_dense(OP == kStreamBF16 ? 1 : 0, BN, kBlockM, false, false)
      : OP == kStreamI8
          ? ((1u << 2) | (2u << 4) | (1u << 7) | (1u << 10) | ((BN >> 3) << 17) | ((kBlockM >> 4) << 24))
          : make_idesc_sparse(0, BN, kBlockM, false);
  static constexpr int RS = kBlockM + 4;                 // parked column stride (words)
  static_assert(BN % 16 == 0 && BN >= 16 && BN <= 128, "token tile");
  static_assert(STAGE_BYTES % 1024 == 0, "stage regions must stay 1024-aligned");
  static_assert(PARKED <= STAGES * STAGE_BYTES, "parked partial tiles must fit the ring");
};

template <int OP>
SP24_DEV void stream_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t e, uint32_t idesc, uint32_t acc) {
  if constexpr (OP == kStreamI8) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.sp.cta_group::1.kind::i8 [%0], %1, %2, [%3], %4, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(e), "r"(idesc), "r"(acc)
        : "memory");
  } else if constexpr (OP == kStreamE4M3) {
    tc_mma_sp<1>(d, a, b, e, idesc, acc);
  } else {
    (void)e;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  }
}

SP24_DEV void store_out(void* out, int type, long long i, float v) {
  if (type == 0) store16<0>(out, i, v);
  else if (type == 1) store16<1>(out, i, v);
  else static_cast<float*>(out)[i] = v;
}

// An output element from its sums.  s0 (and s1 = u in the ffn) are raw 32-bit
// accumulator words.
template <int OP>
SP24_DEV float stream_value(const StreamParams& P, uint32_t s0, uint32_t s1, float scale_m, float bias,
                            float scale_n) {
  if constexpr (OP == kStreamI8) return fmaf(static_cast<float>(static_cast<int>(s0)), scale_m * scale_n, bias);
  else if constexpr (OP == kStreamE4M3) return fmaf(__uint_as_float(s0), scale_m * scale_n, bias);
  else return gate_act(__uint_as_float(s0), P.act) * __uint_as_float(s1);
}

template <int OP>
SP24_DEV uint32_t stream_add(uint32_t a, uint32_t b) {
  if constexpr (OP == kStreamI8) return a + b;
  else return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
}

// Grid: m_blocks * n_tiles * S CTAs in clusters of S; rank r of a cluster sums
// stages [stages r / S, stages (r + 1) / S).
// tmA, tmA2: the weights (tmA2: Wu in the ffn); tmB: the tokens.
template <int OP, int BN>
__global__ void __launch_bounds__(kStreamThreads, 1)
    stream_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmA2,
                  const __grid_constant__ CUtensorMap tmB, const StreamParams P) {
#if defined(__CUDA_ARCH__) && (__CUDA_ARCH__ >= 1000)
  using C = StreamCfg<OP, BN>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[C::STAGES];
  __shared__ __align__(8) uint64_t empty_bar[C::STAGES];
  __shared__ __align__(8) uint64_t accf_bar;
  __shared__ __align__(8) uint64_t drain_bar;
  __shared__ uint32_t tmem_base_sh;
  __shared__ volatile int abort_sh;

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int S = P.splits;
  const int rank = S > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int tile = static_cast<int>(blockIdx.x) / S;
  const int mb = tile % P.m_blocks;
  const int nb = tile / P.m_blocks;
  const int g0 = static_cast<int>(static_cast<long long>(P.stages) * rank / S);
  const int g1 = static_cast<int>(static_cast<long long>(P.stages) * (rank + 1) / S);
  const int nst = g1 - g0;
  const uint64_t tmo = P.timeout_ns;
  // Bytes of global stage g: whole boxes (zero-filled parts count), and the
  // metadata atoms that exist.
  auto stage_tx = [&](int g) {
    int atoms = P.katoms - g * C::ATOMS;
    atoms = atoms < 0 ? 0 : (atoms > C::ATOMS ? C::ATOMS : atoms);
    return static_cast<uint32_t>(C::A_BYTES + C::B_BYTES + atoms * kAtomBytes);
  };

  if (threadIdx.x == 0) {
    abort_sh = 0;
    for (int s = 0; s < P.ring; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(&accf_bar, 1);
    mbar_init(&drain_bar, 1);
    fence_barrier_init();
    // Armed here for the first use, by the MMA warp for later ones.
    for (int s = 0; s < P.ring && s < nst; ++s) mbar_arrive_expect_tx(&full_bar[s], stage_tx(g0 + s));
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    if constexpr (C::G == 2) tma_prefetch_desc(&tmA2);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_base_sh, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_sh;
  griddep_launch_dependents();

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    // Lanes 0 .. G-1 load A boxes, the next B_BOXES the tokens, the rest metadata.
    const bool is_a = lane < C::G;
    const bool is_b = !is_a && lane < C::G + C::B_BOXES;
    const int bl = lane - C::G, el = lane - C::G - C::B_BOXES;
    auto issue = [&](int slot, int g) {
      uint8_t* st = smem + slot * C::STAGE_BYTES;
      if (is_a) {
        tma_load_2d(st + lane * C::A_BOX, lane == 1 ? &tmA2 : &tmA, &full_bar[slot], g * C::A_COLS,
                    mb * kBlockM);
      } else if (is_b) {
        tma_load_2d(st + C::A_BYTES + bl * C::B_BOX, &tmB, &full_bar[slot],
                    (g * C::B_BOXES + bl) * C::B_COLS, nb * BN);
      } else {
        const int atom = g * C::ATOMS + el;
        if (atom < P.katoms)
          bulk_load(st + C::A_BYTES + C::B_BYTES + el * kAtomBytes,
                    P.meta + (static_cast<size_t>(atom) * P.meta_mblocks + mb) * kAtomBytes, kAtomBytes,
                    &full_bar[slot]);
      }
    };
    const int pre = min(P.ring, nst);
    const bool loads = lane < C::LOADS;
    if (P.static_weights && loads && !is_b)
      for (int i = 0; i < pre; ++i) issue(i, g0 + i);
    griddep_wait();
    if (loads && (is_b || !P.static_weights))
      for (int i = 0; i < pre; ++i) issue(i, g0 + i);
    int s = pre == P.ring ? 0 : pre;
    uint32_t ph = pre == P.ring ? 1u : 0u;
    uint32_t used_mask = (1u << pre) - 1u, used_ph = 0;
    bool ok = true;
    for (int i = pre; i < nst; ++i) {
      int good = 1;
      if (lane == 0) good = mbar_wait_fast(&empty_bar[s], ph ^ 1u, &abort_sh, tmo) ? 1 : 0;
      if (__shfl_sync(0xffffffffu, good, 0) == 0) {
        ok = false;
        break;
      }
      if (loads) issue(s, g0 + i);
      used_ph = (used_ph & ~(1u << s)) | (ph << s);
      if (++s == P.ring) s = 0, ph ^= 1u;
    }
    if (!ok && lane == 0) {
      // Error path: copies in flight land before the CTA leaves.
      volatile int dummy = 0;
      for (int j = 0; j < P.ring; ++j)
        if (used_mask & (1u << j)) mbar_wait(&full_bar[j], (used_ph >> j) & 1u, &dummy, tmo);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    const uint32_t base = smem_u32(smem);
    const uint64_t adesc0 = make_sdesc(base, 16, 1024, kLayoutSW128);
    const uint64_t bdesc0 = make_sdesc(base + C::A_BYTES, 16, 1024, kLayoutSW128);
    const uint64_t edesc0 = make_sdesc(base + C::A_BYTES + C::B_BYTES, kAtomBytes, 128, kLayoutNone);
    int s = 0;
    uint32_t ph = 0, ebuf = 0;
    bool ok = true, any = false;
    for (int i = 0; i < nst; ++i) {
      const int g = g0 + i;
      if (!mbar_wait_warp(&full_bar[s], ph, &abort_sh, tmo)) {
        ok = false;
        break;
      }
      if (lane == 0 && i + P.ring < nst) mbar_arrive_expect_tx(&full_bar[s], stage_tx(g + P.ring));
      tc_fence_after();
      ebuf ^= static_cast<uint32_t>(C::ATOMS * 4);
      const uint32_t e = tmem_base + static_cast<uint32_t>(C::E_COL) + ebuf;
      const int kleft = P.k - g * C::BKD;
      if (elect_one()) {
        const uint64_t so = static_cast<uint64_t>(s * (C::STAGE_BYTES >> 4));
#pragma unroll
        for (int a = 0; a < C::ATOMS; ++a)
          if (g * C::ATOMS + a < P.katoms) tc_cp<1>(e + 4 * a, edesc0 + so + a * (kAtomBytes >> 4));
#pragma unroll
        for (int w = 0; w < C::G; ++w)
#pragma unroll
          for (int j = 0; j < C::MMAS; ++j) {
            // Past K a 2:4 MMA has no metadata; a dense one would add zeroes.
            if (j * C::MMA_K < kleft) {
              const uint64_t boff = C::SPARSE ? (j >> 1) * (C::B_BOX >> 4) + (j & 1) * 4 : j * 2;
              stream_mma<OP>(tmem_base + static_cast<uint32_t>(w * BN),
                             adesc0 + so + w * (C::A_BOX >> 4) + j * 2, bdesc0 + so + boff,
                             e + 2 * j, C::IDESC, (i > 0 || j > 0) ? 1u : 0u);
            }
          }
        tc_commit(&empty_bar[s]);
      }
      __syncwarp();
      any = true;
      if (++s == P.ring) s = 0, ph ^= 1u;
    }
    if (ok && elect_one()) tc_commit(&accf_bar);
    __syncwarp();
    if (!ok && any) {
      volatile int dummy = 0;
      if (elect_one()) tc_commit(&drain_bar);
      __syncwarp();
      if (lane == 0) mbar_wait(&drain_bar, 0, &dummy, tmo);
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3;
    const int row_l = q * 32 + lane;
    const int row = mb * kBlockM + row_l;
    const bool live = row < P.m;
    const int cols = min(BN, P.n - nb * BN);
    float sm = 1.0f, bias = 0.0f;
    if (C::SPARSE && live) {
      griddep_wait();   // scales and bias may come from the previous kernel
      if (P.scale_m != nullptr) sm = P.scale_m[row];
      if (P.bias != nullptr) bias = P.bias[row];
    }
    bool ok = true;
    if (lane == 0) ok = mbar_wait(&accf_bar, 0, &abort_sh, tmo);
    if (__shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0) {
      tc_fence_after();
      const uint32_t tb = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
      uint32_t* red = reinterpret_cast<uint32_t*>(smem);   // the ring is idle now
#pragma unroll 1
      for (int c = 0; c < cols; c += 16) {
        uint32_t r[C::G][16];
#pragma unroll
        for (int w = 0; w < C::G; ++w) tmem_ld_x16(tb + static_cast<uint32_t>(w * BN + c), r[w]);
#pragma unroll
        for (int w = 0; w < C::G; ++w) tmem_ld_wait(r[w]);
        if (S > 1) {
#pragma unroll
          for (int w = 0; w < C::G; ++w)
#pragma unroll
            for (int j = 0; j < 16; ++j) red[(w * BN + c + j) * C::RS + row_l] = r[w][j];
        } else if (live) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const long long t = nb * BN + c + j;
            if (c + j < cols) {
              const float sn = C::SPARSE && P.scale_n != nullptr ? P.scale_n[t] : 1.0f;
              if (!C::SPARSE && P.saved != nullptr) {
                P.saved[t * P.ld_saved + row] = __uint_as_float(r[0][j]);
                P.saved[(P.n + t) * P.ld_saved + row] = __uint_as_float(r[C::G - 1][j]);
              }
              store_out(P.out, P.out_type, t * P.ldo + row,
                        stream_value<OP>(P, r[0][j], r[C::G - 1][j], sm, bias, sn));
            }
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (S > 1) {
    // Every rank's partial tile is parked and visible after this barrier.  The
    // live columns' groups of four rows are dealt out to the ranks in turn.
    cluster_sync();
    const uint32_t* red = reinterpret_cast<const uint32_t*>(smem);
    const int cols = min(BN, P.n - nb * BN);
    const int total = cols * (kBlockM / 4);
    for (int idx = threadIdx.x + kStreamThreads * rank; idx < total; idx += kStreamThreads * S) {
      const int c = idx / (kBlockM / 4);
      const int rl = (idx - c * (kBlockM / 4)) * 4;
      const int row = mb * kBlockM + rl;
      uint32_t acc[C::G][4];
#pragma unroll
      for (int w = 0; w < C::G; ++w) {
        const uint32_t la = smem_u32(red + (w * BN + c) * C::RS + rl);
#pragma unroll 1
        for (int s0 = 0; s0 < S; s0 += 4) {   // four loads on their way before the first sum
          float4 v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (s0 + i < S) v[i] = ld_dsmem_f4(mapa_shared(la, static_cast<uint32_t>(s0 + i)));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (s0 + i >= S) break;
            const uint32_t p[4] = {__float_as_uint(v[i].x), __float_as_uint(v[i].y), __float_as_uint(v[i].z),
                                   __float_as_uint(v[i].w)};
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[w][j] = s0 + i == 0 ? p[j] : stream_add<OP>(acc[w][j], p[j]);
          }
        }
      }
      const long long t = nb * BN + c;
      const float sn = C::SPARSE && P.scale_n != nullptr ? P.scale_n[t] : 1.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (row + j < P.m) {
          const float sm = C::SPARSE && P.scale_m != nullptr ? P.scale_m[row + j] : 1.0f;
          const float bias = C::SPARSE && P.bias != nullptr ? P.bias[row + j] : 0.0f;
          if (!C::SPARSE && P.saved != nullptr) {
            P.saved[t * P.ld_saved + row + j] = __uint_as_float(acc[0][j]);
            P.saved[(P.n + t) * P.ld_saved + row + j] = __uint_as_float(acc[C::G - 1][j]);
          }
          store_out(P.out, P.out_type, t * P.ldo + row + j,
                    stream_value<OP>(P, acc[0][j], acc[C::G - 1][j], sm, bias, sn));
        }
      }
    }
    // No CTA leaves (and releases its shared memory) while others still read it.
    cluster_sync();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
  if (threadIdx.x == 0 && abort_sh != 0 && P.status != nullptr) atomicExch(P.status, 1);
#endif
}

// The gated block over 33 to 128 tokens, still bound by the weights' bytes: a CTA
// pair takes 256 rows of Wg and the same 256 of Wu as the M of two MMAs
// (tcgen05.mma.cta_group::2, M = 256, N = BN) against one staged block of tokens,
// of which each CTA loads half.  Staging half the tokens leaves the ring to the
// weights: at 128 tokens 32 of a stage's 40 KB, where a single CTA's stages hold
// 32 of 48 (4096 -> 14336 bf16, 128 tokens: 48.2 us against 57.6).  Both
// accumulators of a feature lie in one lane, at columns 0 and 256.
template <int BN>
struct FewPairCfg {
  static constexpr int BK = 64;
  static constexpr int A_BOX = kBlockM * 128;
  static constexpr int A_BYTES = 2 * A_BOX;             // Wg's rows, then Wu's
  static constexpr int HALF = BN / 2;                   // tokens staged per CTA
  static constexpr int B_BYTES = HALF * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES_RAW = (kSmemBudget - 1024) / STAGE_BYTES;
  static constexpr int STAGES = STAGES_RAW > 8 ? 8 : STAGES_RAW;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024;
  static constexpr int CW = BN / 2;                     // columns per epilogue warp
  static_assert(BN % 64 == 0 && BN <= 128 && STAGE_BYTES % 1024 == 0, "token tile");
};

// tmA, tmA2: Wg and Wu; tmB: the tokens.  One pair per 256 features.
template <int DT, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    few_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmA2,
                    const __grid_constant__ CUtensorMap tmB, const StreamParams P) {
#if defined(__CUDA_ARCH__) && (__CUDA_ARCH__ >= 1000)
  using C = FewPairCfg<BN>;
  constexpr uint32_t IDESC = make_idesc_dense(DT, BN, 256, false, false);
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[C::STAGES];
  __shared__ __align__(8) uint64_t empty_bar[C::STAGES];
  __shared__ __align__(8) uint64_t accf_bar;
  __shared__ __align__(8) uint64_t drain_bar;
  __shared__ uint32_t tmem_base_sh;
  __shared__ volatile int abort_sh;

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int prank = static_cast<int>(cluster_ctarank());
  const bool leader = prank == 0;
  const int row_cta = static_cast<int>(blockIdx.x >> 1) * 256 + prank * 128;   // this CTA's first feature
  const uint64_t tmo = P.timeout_ns;

  if (threadIdx.x == 0) {
    abort_sh = 0;
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(&accf_bar, 1);
    mbar_init(&drain_bar, 1);
    fence_barrier_init();
    // Both CTAs' bytes land on the leader's barriers, armed here for the first
    // use and by the MMA warp for later ones.
    if (leader)
      for (int s = 0; s < C::STAGES; ++s) mbar_arrive_expect_tx(&full_bar[s], 2 * C::STAGE_BYTES);
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmA2);
    tma_prefetch_desc(&tmB);
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
    const bool is_b = warp == kPairBWarp;
    if (is_b || !P.static_weights) griddep_wait();
    const CUtensorMap* map = is_b ? &tmB : lane == 1 ? &tmA2 : &tmA;
    const uint32_t off = is_b ? C::A_BYTES : lane * C::A_BOX;
    const int y = is_b ? prank * C::HALF : row_cta;
    const uint32_t full0 = mapa_shared(smem_u32(&full_bar[0]), 0);
    int s = 0;
    uint32_t ph = 0, used_mask = 0, used_ph = 0;
    bool ok = true;
    for (int ks = 0; ks < P.stages; ++ks) {
      int good = 1;
      if (lane == 0) good = mbar_wait_fast(&empty_bar[s], ph ^ 1u, &abort_sh, tmo) ? 1 : 0;
      if (__shfl_sync(0xffffffffu, good, 0) == 0) {
        ok = false;
        break;
      }
      used_mask |= 1u << s;
      used_ph = (used_ph & ~(1u << s)) | (ph << s);
      if (lane < (is_b ? 1 : 2))
        tma_load_2d_pair(smem + s * C::STAGE_BYTES + off, map, full0 + s * sizeof(uint64_t), ks * C::BK, y);
      if (++s == C::STAGES) s = 0, ph ^= 1u;
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
      const uint64_t adesc0 = make_sdesc(base, 16, 1024, kLayoutSW128);
      const uint64_t bdesc0 = make_sdesc(base + C::A_BYTES, 16, 1024, kLayoutSW128);
      int s = 0;
      uint32_t ph = 0;
      bool ok = true, any = false;
      for (int ks = 0; ks < P.stages; ++ks) {
        if (!mbar_wait_warp(&full_bar[s], ph, &abort_sh, tmo)) {
          ok = false;
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&full_bar[s], 2 * C::STAGE_BYTES);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t so = static_cast<uint64_t>(s * (C::STAGE_BYTES >> 4));
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int j = 0; j < C::BK / 16; ++j)
              tc_mma_dense_pair(tmem_base + w * 256, adesc0 + so + w * (C::A_BOX >> 4) + j * 2,
                                bdesc0 + so + j * 2, IDESC, (ks > 0 || j > 0) ? 1u : 0u);
          tc_commit_pair(&empty_bar[s], 3);
        }
        __syncwarp();
        any = true;
        if (++s == C::STAGES) s = 0, ph ^= 1u;
      }
      if (ok && elect_one()) tc_commit_pair(&accf_bar, 3);
      __syncwarp();
      if (!ok && any) {
        volatile int dummy = 0;
        if (elect_one()) tc_commit_pair(&drain_bar, 1);
        __syncwarp();
        if (lane == 0) mbar_wait(&drain_bar, 0, &dummy, tmo);
        __syncwarp();
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3, half = (warp - 2) >> 2;
    bool ok = true;
    if (lane == 0) ok = mbar_wait_sleepy(&accf_bar, 0, &abort_sh, tmo);
    if (__shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0) {
      tc_fence_after();
      const int row = row_cta + q * 32 + lane;
      const int t0 = half * C::CW, t1 = min(P.n, t0 + C::CW);
      const uint32_t tb = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll 1
      for (int t = t0; t < t1; t += 16) {
        uint32_t g[16], u[16];
        tmem_ld_x16(tb + t, g);
        tmem_ld_x16(tb + 256 + t, u);
        tmem_ld_wait(g);
        tmem_ld_wait(u);
        if (row >= P.m) continue;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const long long tok = t + j;
          if (tok < t1) {
            if (P.saved != nullptr) {
              P.saved[tok * P.ld_saved + row] = __uint_as_float(g[j]);
              P.saved[(P.n + tok) * P.ld_saved + row] = __uint_as_float(u[j]);
            }
            store16<DT>(P.out, tok * P.ldo + row,
                        gate_act(__uint_as_float(g[j]), P.act) * __uint_as_float(u[j]));
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
  if (threadIdx.x == 0 && abort_sh != 0 && P.status != nullptr) atomicExch(P.status, 1);
#endif
}

}  // namespace sp24
