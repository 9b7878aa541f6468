// sp24_mlp.cu — C ABI of the MLP-block operators declared in include/sp24.h:
// argument checks and launches of the row kernels (sp24_rows.cuh), the 8-bit
// scaled product and the gated feed-forward block.
#include <algorithm>

#include "sp24_ffn_kernel.cuh"
#include "sp24_host.cuh"
#include "sp24_rows.cuh"
#include "sp24_scaled_pair_kernel.cuh"
#include "sp24_stream_kernel.cuh"

using namespace sp24host;

namespace {

inline bool is_16bit(int dt) { return dt == SP24_F16 || dt == SP24_BF16; }

// A row stride given as 0 means the row's length.
inline int64_t stride_or(int64_t ld, int64_t len) { return ld ? ld : len; }

// ------------------------------------------------------------------ rows to 8 bits
sp24_status check_rows(const sp24_rowquant_desc* d, int mode, sp24::RowsParams* p) {
  if (d == nullptr) return SP24_ERR_ARG;
  if (!is_16bit(d->dtype) || (d->qdtype != SP24_I8 && d->qdtype != SP24_E4M3))
    return SP24_ERR_ARG;
  if (d->rows < 0 || d->cols <= 0) return SP24_ERR_SHAPE;
  p->rows = d->rows;
  p->cols = d->cols;
  p->ldx = stride_or(d->ldx, d->cols);
  p->ldq = stride_or(d->ldq, d->cols);
  p->ld_up = stride_or(d->ld_up, d->cols);
  p->ld_residual = stride_or(d->ld_residual, d->cols);
  p->ld_residual_out = stride_or(d->ld_residual_out, d->cols);
  if (p->ldx < d->cols || p->ldq < d->cols) return SP24_ERR_SHAPE;
  if (mode == sp24::kRowsNorm) {
    if (d->weight == nullptr || !(d->eps >= 0.0f)) return SP24_ERR_ARG;
    if (d->residual_out != nullptr && d->residual == nullptr) return SP24_ERR_ARG;
    if (p->ld_residual < d->cols || p->ld_residual_out < d->cols) return SP24_ERR_SHAPE;
  } else if (d->residual != nullptr || d->residual_out != nullptr || d->weight != nullptr) {
    return SP24_ERR_ARG;
  }
  if (mode == sp24::kRowsSwiglu) {
    if (p->ld_up < d->cols) return SP24_ERR_SHAPE;
  } else if (d->up != nullptr) {
    return SP24_ERR_ARG;
  }
  if (d->rows > 0 && (d->x == nullptr || d->q == nullptr || d->scale == nullptr ||
                      (mode == sp24::kRowsSwiglu && d->up == nullptr)))
    return SP24_ERR_ARG;
  p->x = d->x;
  p->up = d->up;
  p->residual = d->residual;
  p->residual_out = d->residual_out;
  p->weight = d->weight;
  p->eps = d->eps;
  p->inv_cols = 1.0f / static_cast<float>(d->cols);
  p->q = static_cast<uint8_t*>(d->q);
  p->scale = d->scale;
  return SP24_OK;
}

// A resident grid: as many blocks as fit the registers, threads and shared
// memory of the SMs.
template <int DT, int MODE, int I8, int V, int VPT, bool ONE_WARP>
sp24_status launch_rows_kernel(const sp24::RowsParams& p, const DeviceInfo& di, unsigned threads, cudaStream_t s) {
  constexpr int kSmem = 200 * 1024;   // of an SM, for the slots
  auto kern = sp24::rows_quant_kernel<DT, MODE, I8, V, VPT, ONE_WARP>;
  static std::atomic<bool> attr_set[kMaxDevices];
  static std::atomic<int> regs{0};
  sp24_status st = ensure_kernel_attrs(kern, attr_set, V > 1 ? 2 * VPT * (ONE_WARP ? 256 : 1024) * 2 * V : 0);
  if (st != SP24_OK) return st;
  if (regs.load(std::memory_order_relaxed) == 0) {
    cudaFuncAttributes a{};
    SP24_CUDA_TRY(cudaFuncGetAttributes(&a, kern));
    regs.store((a.numRegs + 7) / 8 * 8, std::memory_order_relaxed);
  }
  const int inputs = p.up != nullptr || p.residual != nullptr ? 2 : 1;
  const int smem = V > 1 ? inputs * VPT * static_cast<int>(threads) * 2 * V : 0;
  const int t = static_cast<int>(threads);
  int blocks = std::min({2048 / t, 65536 / (regs.load(std::memory_order_relaxed) * t), 32});
  if (V > 1) blocks = std::min(blocks, kSmem / std::max(smem, 1));
  blocks = std::max(blocks, 1);
  const long long per_block = ONE_WARP ? t / 32 : 1;
  const long long want = (p.rows + per_block - 1) / per_block;
  const unsigned grid = static_cast<unsigned>(std::min<long long>(want, static_cast<long long>(blocks) * di.sm_count));
  return launch_gemm_kernel(kern, grid, threads, smem, s, 0, true, p);
}

// Rows of more than LO and at most HI vectors, VPT of them a thread; only the
// forms that such rows reach are built.
template <int DT, int MODE, int I8, int V, int VPT, int LO, int HI>
sp24_status launch_rows_vpt(const sp24::RowsParams& p, const DeviceInfo& di, int vecs, cudaStream_t s) {
  constexpr int kWarp = 32 * VPT;   // vectors that one warp holds
  if constexpr (LO < kWarp)
    if (HI <= kWarp || vecs <= kWarp) return launch_rows_kernel<DT, MODE, I8, V, VPT, true>(p, di, 256, s);
  if constexpr (HI > kWarp) {
    const unsigned threads = static_cast<unsigned>(round_up((vecs + VPT - 1) / VPT, 32));
    return launch_rows_kernel<DT, MODE, I8, V, VPT, false>(p, di, threads, s);
  }
  return SP24_ERR_SHAPE;   // not reached
}

// Vectors a thread holds.  The norm waits for a row's two inputs, sum and weight
// at once and wants many threads with little each: one vector up to 4096 columns
// (8192 x 4096: 39.0 us; 40.2 with two, 46.1 with four), two up to 16384 (8192 x
// 8192: 79.9; 85.0 with one, 82.5 with four).  Rows without it have less to keep
// and more to gain from few warps a row: four (8192 x 4096 plain: 18.5 us; 20.6
// with two, 22.7 with one), unless a warp covers the row with one (8192 x 256:
// 4.4 us; 6.0 with four) or there are few rows, whose loads then go out at once.
// Vectors of four and two values: four where they reach (norm 8192 x 4092 / 4094:
// 43.9 / 62.5 us; 64.4 / 80.2 with eight), single elements eight (4096 x 1001
// swiglu: 10.3 us; 12.0 with four, 12.7 with sixteen).
template <int DT, int MODE, int I8, int V>
sp24_status launch_rows_v(const sp24::RowsParams& p, const DeviceInfo& di, cudaStream_t s) {
  const int vecs = (p.cols + V - 1) / V;
  if constexpr (V == 8 && MODE == sp24::kRowsNorm) {
    if (vecs <= 512) return launch_rows_vpt<DT, MODE, I8, V, 1, 0, 512>(p, di, vecs, s);
    if (vecs <= 2048) return launch_rows_vpt<DT, MODE, I8, V, 2, 512, 2048>(p, di, vecs, s);
    if (vecs <= 4096) return launch_rows_vpt<DT, MODE, I8, V, 4, 2048, 4096>(p, di, vecs, s);
  } else if constexpr (V == 8) {
    if (vecs <= 32) return launch_rows_vpt<DT, MODE, I8, V, 1, 0, 32>(p, di, vecs, s);
    const bool few = p.rows <= 2 * di.sm_count;
    if (few && vecs <= 2048) return launch_rows_vpt<DT, MODE, I8, V, 2, 32, 2048>(p, di, vecs, s);
    if (vecs <= 4096) return launch_rows_vpt<DT, MODE, I8, V, 4, 32, 4096>(p, di, vecs, s);
  } else if constexpr (V == 4) {
    if (vecs <= 4096) return launch_rows_vpt<DT, MODE, I8, V, 4, 0, 4096>(p, di, vecs, s);
  } else if constexpr (V == 2) {
    if (vecs <= 4096) return launch_rows_vpt<DT, MODE, I8, V, 4, 0, 4096>(p, di, vecs, s);
    if (vecs <= 8192) return launch_rows_vpt<DT, MODE, I8, V, 8, 4096, 8192>(p, di, vecs, s);
  } else {
    if (vecs <= 8192) return launch_rows_vpt<DT, MODE, I8, V, 8, 0, 8192>(p, di, vecs, s);
  }
  return launch_gemm_kernel(sp24::rows_quant_long_kernel<DT, MODE, I8>,
                            static_cast<unsigned>(p.rows), 1024, 0, s, 0, true, p);
}

template <int DT, int MODE, int I8>
sp24_status launch_rows(const sp24::RowsParams& p, const DeviceInfo& di, cudaStream_t s) {
  // The widest vector that divides the rows and starts all of them aligned.
  auto fits = [&](int v) {
    auto in = [v](const void* q, long long ld) {
      return q == nullptr || (reinterpret_cast<uintptr_t>(q) % (2 * v) == 0 && ld % v == 0);
    };
    return p.cols % v == 0 && in(p.x, p.ldx) && in(p.up, p.ld_up) && in(p.residual, p.ld_residual) &&
           in(p.residual_out, p.ld_residual_out) && in(p.weight, 0) &&
           reinterpret_cast<uintptr_t>(p.q) % v == 0 && p.ldq % v == 0;
  };
  return fits(8)   ? launch_rows_v<DT, MODE, I8, 8>(p, di, s)
         : fits(4) ? launch_rows_v<DT, MODE, I8, 4>(p, di, s)
         : fits(2) ? launch_rows_v<DT, MODE, I8, 2>(p, di, s)
                   : launch_rows_v<DT, MODE, I8, 1>(p, di, s);
}

template <int MODE>
sp24_status rows_quant(const sp24_rowquant_desc* d, sp24_stream_t stream) {
  sp24::RowsParams p{};
  sp24_status st = check_rows(d, MODE, &p);
  if (st != SP24_OK || d->rows == 0) return st;
  DeviceInfo* di = nullptr;
  st = device_info(&di);
  if (st != SP24_OK) return st;
  cudaStream_t s = as_stream(stream);
  const bool i8 = d->qdtype == SP24_I8;
  if (d->dtype == SP24_F16)
    return i8 ? launch_rows<0, MODE, 1>(p, *di, s) : launch_rows<0, MODE, 0>(p, *di, s);
  return i8 ? launch_rows<1, MODE, 1>(p, *di, s) : launch_rows<1, MODE, 0>(p, *di, s);
}

// ------------------------------------------------------------------ scaled product
constexpr int kMaxScaledK = 131072;   // 2:4 int8 sums stay below 2^31 with room to spare

sp24_status check_scaled(const sp24_scaled_desc* d) {
  if (d == nullptr) return SP24_ERR_ARG;
  if (d->dtype != SP24_I8 && d->dtype != SP24_E4M3) return SP24_ERR_ARG;
  if (!is_16bit(d->cdtype) && d->cdtype != SP24_F32) return SP24_ERR_ARG;
  if (d->m <= 0 || d->n < 0 || d->k <= 0 || d->k % 64 != 0) return SP24_ERR_SHAPE;
  if (d->dtype == SP24_I8 && d->k > kMaxScaledK) return SP24_ERR_SHAPE;
  const int64_t lda = stride_or(d->lda_c, d->k / 2), ldx = stride_or(d->ldx, d->k);
  if (lda < d->k / 2 || ldx < d->k || stride_or(d->ldc, d->m) < d->m) return SP24_ERR_SHAPE;
  if (d->a_c == nullptr || d->meta == nullptr) return SP24_ERR_ARG;
  if (d->n > 0 && (d->x == nullptr || d->c == nullptr)) return SP24_ERR_ARG;
  if (!aligned16(d->a_c) || !aligned16(d->meta) || !aligned16(d->x) || lda % 16 || ldx % 16)
    return SP24_ERR_ALIGN;
  return SP24_OK;
}

// ------------------------------------------------------------------ gated feed-forward
// Row stride of the saved fp32 planes and of the 16-bit dg / du planes: whole
// 128-byte lines, so that no row of a TMA box straddles two.
inline int64_t ffn_ld(int f) { return static_cast<int64_t>(round_up(static_cast<size_t>(f), 64)); }

inline size_t dgu_bytes(int t, int f) { return static_cast<size_t>(t) * 2 * ffn_ld(f) * 2; }

// K slices of a dx tile that go through the workspace: where the tiles are so few
// that clusters of four pairs would leave most of the pairs idle, as many slices as
// there are pairs for them, of at least eight stages each; else none.  The
// workspace, whose size is asked for without a device, has room for the slices of a
// whole B200 (74 pairs); a part with fewer SMs takes fewer.
constexpr int kMaxPairs = 74;
int dx_slices(int t, int h, int f, int pairs = kMaxPairs) {
  const long long tiles = ((t + 255LL) / 256) * ((h + 255LL) / 256);
  const long long stages = 2 * ((f + 63LL) / 64);
  const long long slices = std::min(pairs / tiles, stages / 8);
  return slices > sp24::kFfnMaxSplits ? static_cast<int>(slices) : 0;
}

sp24_status check_ffn(const sp24_ffn_desc* d) {
  if (d == nullptr) return SP24_ERR_ARG;
  if (!is_16bit(d->dtype)) return SP24_ERR_ARG;
  if (d->act != SP24_ACT_SILU && d->act != SP24_ACT_GELU_TANH && d->act != SP24_ACT_NONE) return SP24_ERR_ARG;
  if (d->t < 0 || d->h <= 0 || d->f <= 0) return SP24_ERR_SHAPE;
  const int64_t ldx = stride_or(d->ldx, d->h), ldg = stride_or(d->ld_gate, d->h),
                ldu = stride_or(d->ld_up, d->h);
  if (ldx < d->h || ldg < d->h || ldu < d->h) return SP24_ERR_SHAPE;
  if (d->w_gate == nullptr || d->w_up == nullptr || (d->t > 0 && d->x == nullptr))
    return SP24_ERR_ARG;
  if (!aligned16(d->x) || !aligned16(d->w_gate) || !aligned16(d->w_up) || ldx % 8 || ldg % 8 ||
      ldu % 8 || !aligned32(d->saved))
    return SP24_ERR_ALIGN;
  return SP24_OK;
}

// What the three products of a call share.
struct FfnCall {
  int sm_count;
  int* status;
  cudaStream_t stream;
};

int out_vec(const void* p, int64_t ld) {
  return aligned32(p) && ld % 16 == 0 ? 2 : aligned16(p) && ld % 8 == 0 ? 1 : 0;
}

template <int DT, int MODE>
sp24_status launch_ffn_pair(const FfnCall& c, const CUtensorMap (&a)[2], const CUtensorMap (&b)[2],
                            sp24::FfnParams p) {
  using C = sp24::FfnCfg<DT, MODE>;
  auto kern = sp24::ffn_pair_kernel<DT, MODE>;
  static std::atomic<bool> attr_set[kMaxDevices];
  const sp24_status st = ensure_kernel_attrs(kern, attr_set, C::SMEM_BYTES);
  if (st != SP24_OK) return st;
  p.status = c.status;
  p.timeout_ns = kDefaultTimeoutNs;
  const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles * std::max(1, p.splits);
  if (tiles > 0x7fffffff / 2) return SP24_ERR_SHAPE;
  const unsigned pairs = static_cast<unsigned>(std::min<long long>(tiles, c.sm_count / 2));
  return launch_gemm_kernel(kern, 2 * pairs, sp24::kPairThreads, C::SMEM_BYTES, c.stream, 0, true,
                            a[0], a[1], b[0], b[1], p);
}

// The largest number of K splits, at most `want`, whose clusters (`per_split`
// CTAs each) are all resident at once: a second wave of clusters would cost
// more than the split saves.
template <auto Kern>
int resident_splits(int threads, int smem, long long clusters, int per_split, int want) {
  static std::atomic<int> cache[kMaxDevices][9];   // by CTAs per cluster; 0 = not asked yet
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 1;
  for (int s = want; s > 1; --s) {
    std::atomic<int>& slot = cache[dev][s * per_split];
    int n = slot.load(std::memory_order_relaxed);
    if (n == 0) {
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(static_cast<unsigned>(s * per_split));
      cfg.blockDim = dim3(static_cast<unsigned>(threads));
      cfg.dynamicSmemBytes = static_cast<size_t>(smem);
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = static_cast<unsigned>(s * per_split);
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&n, Kern, &cfg) != cudaSuccess) {
        (void)cudaGetLastError();
        n = 0;
      }
      n = n > 0 ? n : -1;
      slot.store(n, std::memory_order_relaxed);
    }
    if (n >= clusters) return s;
  }
  return 1;
}

// Tensor map of a 16-bit matrix in boxes of 64 columns (128 bytes).
sp24_status encode_16(CUtensorMap* map, const void* base, int rows, int cols, int64_t ld, int box_rows) {
  return encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, base, static_cast<uint64_t>(cols),
                   static_cast<uint64_t>(rows), static_cast<uint64_t>(ld) * 2, 64,
                   static_cast<uint32_t>(box_rows), CU_TENSOR_MAP_SWIZZLE_128B);
}

// ------------------------------------------------------------------ few tokens
constexpr int kStreamMaxTokens = 128;

template <int OP, int BN>
sp24_status launch_stream_bn(const FfnCall& c, const CUtensorMap& a, const CUtensorMap& a2,
                             const CUtensorMap& b, sp24::StreamParams p) {
  using C = sp24::StreamCfg<OP, BN>;
  auto kern = sp24::stream_kernel<OP, BN>;
  static std::atomic<bool> attr_set[kMaxDevices];
  const sp24_status st = ensure_kernel_attrs(kern, attr_set, C::SMEM_BYTES);
  if (st != SP24_OK) return st;
  p.stages = (p.k + C::BKD - 1) / C::BKD;
  const int n_tiles = (p.n + BN - 1) / BN;
  const long long tiles = static_cast<long long>(p.m_blocks) * n_tiles;
  if (tiles * sp24::kStreamMaxSplits > 0x7fffffff) return SP24_ERR_SHAPE;
  const int want = static_cast<int>(std::min<long long>({c.sm_count / tiles, sp24::kStreamMaxSplits, p.stages}));
  p.splits = resident_splits<sp24::stream_kernel<OP, BN>>(sp24::kStreamThreads, C::SMEM_BYTES, tiles, 1, want);
  // No more slots than a CTA has stages: what is left of the SM's shared memory
  // lets the next kernel's CTAs start their prologue beside this one's tail
  // (4096 x 4096, 1 token, back to back: 6.1 -> 5.6 us).
  p.ring = std::min(C::STAGES, (p.stages + p.splits - 1) / p.splits);
  const int smem = std::max({p.ring * C::STAGE_BYTES + 1024, p.splits > 1 ? C::PARKED + 1024 : 0, C::MIN_SMEM});
  p.status = c.status;
  p.timeout_ns = kDefaultTimeoutNs;
  return launch_gemm_kernel(kern, static_cast<unsigned>(tiles * p.splits), sp24::kStreamThreads,
                            static_cast<size_t>(smem), c.stream, static_cast<unsigned>(p.splits), true, a, a2, b, p);
}

// rows of a TMA box of B for n tokens
inline int stream_bn(int n) { return n <= 16 ? 16 : n <= 32 ? 32 : n <= 64 ? 64 : 128; }

template <int OP>
sp24_status launch_stream(const FfnCall& c, const CUtensorMap& a, const CUtensorMap& a2,
                          const CUtensorMap& b, const sp24::StreamParams& p) {
  switch (stream_bn(p.n)) {
    case 16: return launch_stream_bn<OP, 16>(c, a, a2, b, p);
    case 32: return launch_stream_bn<OP, 32>(c, a, a2, b, p);
    case 64: return launch_stream_bn<OP, 64>(c, a, a2, b, p);
    default: return launch_stream_bn<OP, 128>(c, a, a2, b, p);
  }
}

// Tensor map of 8-bit rows in boxes of 128 columns.
sp24_status encode_8(CUtensorMap* map, const void* base, int rows, int cols, int64_t ld, int box_rows) {
  return encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, static_cast<uint64_t>(cols),
                   static_cast<uint64_t>(rows), static_cast<uint64_t>(ld), 128,
                   static_cast<uint32_t>(box_rows), CU_TENSOR_MAP_SWIZZLE_128B);
}

inline int out_type(const sp24_scaled_desc* d) { return d->cdtype == SP24_F32 ? 2 : static_cast<int>(d->cdtype); }
inline int static_weights() { return (sp24_get_launch_hints() & SP24_HINT_STATIC_WEIGHTS) != 0; }

template <int I8>
sp24_status scaled_few(const FfnCall& c, const sp24_scaled_desc* d) {
  CUtensorMap a, b;
  sp24_status st = encode_8(&a, d->a_c, d->m, d->k / 2, stride_or(d->lda_c, d->k / 2), 128);
  if (st == SP24_OK) st = encode_8(&b, d->x, d->n, d->k, stride_or(d->ldx, d->k), stream_bn(d->n));
  if (st != SP24_OK) return st;
  sp24::StreamParams p{};
  p.m = d->m, p.n = d->n, p.k = d->k;
  p.m_blocks = (d->m + 127) / 128;
  p.meta = d->meta;
  p.meta_mblocks = meta_mblocks(d->m), p.katoms = meta_katoms(d->k);
  p.scale_m = d->scale_m, p.scale_n = d->scale_n, p.bias = d->bias;
  p.out = d->c, p.ldo = stride_or(d->ldc, d->m), p.out_type = out_type(d);
  p.static_weights = static_weights();
  return launch_stream<I8 ? sp24::kStreamI8 : sp24::kStreamE4M3>(c, a, a, b, p);
}

template <int I8, int MB, int BN>
sp24_status scaled_pair(const FfnCall& c, const sp24_scaled_desc* d) {
  using C = sp24::ScaledPairCfg<I8, MB, BN>;
  auto kern = sp24::scaled_pair_kernel<I8, MB, BN>;
  static std::atomic<bool> attr_set[kMaxDevices];
  sp24_status st = ensure_kernel_attrs(kern, attr_set, C::SMEM_BYTES);
  if (st != SP24_OK) return st;
  CUtensorMap a, b, e;
  const int mblocks = meta_mblocks(d->m), katoms = meta_katoms(d->k);
  st = encode_8(&a, d->a_c, d->m, d->k / 2, stride_or(d->lda_c, d->k / 2), 128);
  if (st == SP24_OK) st = encode_8(&b, d->x, d->n, d->k, stride_or(d->ldx, d->k), C::HALF);
  if (st == SP24_OK)
    st = encode_2d(&e, CU_TENSOR_MAP_DATA_TYPE_UINT8, d->meta, 256,
                   static_cast<uint64_t>(katoms) * mblocks * 8, 256, 256, 8, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (st != SP24_OK) return st;
  sp24::ScaledPairParams p{};
  p.m = d->m, p.n = d->n, p.k = d->k;
  p.m_tiles = (d->m + MB * 256 - 1) / (MB * 256), p.n_tiles = (d->n + BN - 1) / BN;
  p.k_stages = (d->k + C::BKD - 1) / C::BKD;
  p.group_m = 8;
  p.meta_mblocks = mblocks;
  p.scale_m = d->scale_m, p.scale_n = d->scale_n, p.bias = d->bias;
  p.out = d->c, p.ldo = stride_or(d->ldc, d->m), p.out_type = out_type(d);
  p.words = reinterpret_cast<uintptr_t>(d->c) % 4 == 0 && p.ldo % 2 == 0;
  p.static_weights = static_weights();
  p.status = c.status;
  p.timeout_ns = kDefaultTimeoutNs;
  const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles;
  if (tiles > 0x7fffffff / 4) return SP24_ERR_SHAPE;
  // A last wave that half the pairs could cover is dealt block by block.
  const int pairs = c.sm_count / 2;
  const int last = static_cast<int>(tiles % pairs);
  const bool halve = MB == 2 && 2 * last <= pairs;
  p.whole_items = static_cast<int>(halve ? tiles - last : tiles);
  p.items = p.whole_items + (halve ? 2 * last : 0);
  return launch_gemm_kernel(kern, static_cast<unsigned>(2 * std::min(p.items, pairs)), sp24::kScaledThreads,
                            C::SMEM_BYTES, c.stream, 0, true, a, b, e, p);
}

// Which kernel.  Up to 32 tokens the weights' bytes decide, and the streaming
// kernel splits K over as many SMs as there are.  From 33 to 128 tokens a pair
// that stages half the tokens per SM wins where 256-row tiles alone occupy
// three quarters of the pairs (14336 x 4096, 64 / 128 tokens: 13.7 / 13.9 us
// against 15.0 / 21.8; 4096 x 14336 has 16 such tiles: 28 us against 13 / 17).
// Beyond, tiles of one 256-row block x 128 tokens fill few waves, and tiles of
// two blocks x 224 tokens load less per product: a wave of the large tile takes
// twice as long as one of the small (K = 14336: 47 and 25 us; K = 4096: 18 and 8),
// and its last wave may go in halves.  The large tile is taken where it ends
// sooner.  Device times of both in a burst / held under the power cap: 4096 tokens x
// 4096 x 14336, 2.5 large waves or 7 small, 125 / 140 and 160 / 180 us; 1024 tokens x
// 14336 x 4096, 2 or 7, 41 / 45 and 54 / 56 us; 333 x 5003 x 4160, half a wave or
// one, 18.7 / 18.4 and 14.0 / 13.8 us, and a tie goes to the small.
template <int I8>
sp24_status scaled(const FfnCall& c, const sp24_scaled_desc* d) {
  const long long pairs = c.sm_count / 2;
  const long long blocks = (d->m + 255) / 256;
  if (d->n <= 32 || (d->n <= kStreamMaxTokens && 4 * blocks < 3 * pairs)) return scaled_few<I8>(c, d);
  const long long small_tiles = blocks * ((d->n + 127LL) / 128);
  const long long large_tiles = (d->m + 511LL) / 512 * ((d->n + 223LL) / 224);
  const long long small = (small_tiles + pairs - 1) / pairs;
  const long long last = large_tiles % pairs;
  const long long halves = large_tiles / pairs * 2 + (last == 0 ? 0 : 2 * last <= pairs ? 1 : 2);
  return small > halves ? scaled_pair<I8, 2, 224>(c, d) : scaled_pair<I8, 1, 128>(c, d);
}

template <int DT, int BN>
sp24_status launch_few_pair(const FfnCall& c, const CUtensorMap& a, const CUtensorMap& a2,
                            const CUtensorMap& b, sp24::StreamParams p) {
  using C = sp24::FewPairCfg<BN>;
  auto kern = sp24::few_pair_kernel<DT, BN>;
  static std::atomic<bool> attr_set[kMaxDevices];
  const sp24_status st = ensure_kernel_attrs(kern, attr_set, C::SMEM_BYTES);
  if (st != SP24_OK) return st;
  p.stages = (p.k + C::BK - 1) / C::BK;
  p.status = c.status;
  p.timeout_ns = kDefaultTimeoutNs;
  return launch_gemm_kernel(kern, static_cast<unsigned>((p.m + 255) / 256 * 2), sp24::kPairThreads,
                            C::SMEM_BYTES, c.stream, 0, true, a, a2, b, p);
}

// Token tile of the pair form.
inline int few_pair_bn(int n) { return n <= 64 ? 64 : 128; }

// The pair form of the gated block: from 33 tokens on, where its 256-feature
// tiles occupy three quarters of the pairs in one wave (4096 -> 14336: 64 / 128
// tokens 41.8 / 48.2 us against the single CTAs' 46.5 / 57.6; 4096 -> 8192, 32
// tiles: 38.4 against 35.7 at 100 tokens).  Beyond 128 tokens the tiles with tokens
// on M are faster (256 tokens: 62.1 us against 71.2).
bool few_pairs(const FfnCall& c, const sp24_ffn_desc* d) {
  const int tiles = (d->f + 255) / 256, pairs = c.sm_count / 2;
  return d->t > 32 && d->t <= kStreamMaxTokens && tiles <= pairs && 4 * tiles >= 3 * pairs;
}

template <int DT>
sp24_status ffn_forward_few(const FfnCall& c, const sp24_ffn_desc* d, void* out, int64_t ld_out) {
  CUtensorMap a, a2, b;
  const bool pairs = few_pairs(c, d);
  const int box = pairs ? few_pair_bn(d->t) / 2 : stream_bn(d->t);
  sp24_status st = encode_16(&a, d->w_gate, d->f, d->h, stride_or(d->ld_gate, d->h), 128);
  if (st == SP24_OK) st = encode_16(&a2, d->w_up, d->f, d->h, stride_or(d->ld_up, d->h), 128);
  if (st == SP24_OK) st = encode_16(&b, d->x, d->t, d->h, stride_or(d->ldx, d->h), box);
  if (st != SP24_OK) return st;
  sp24::StreamParams p{};
  p.m = d->f, p.n = d->t, p.k = d->h;
  p.m_blocks = (d->f + 127) / 128;
  p.out = out, p.ldo = ld_out, p.out_type = DT;
  p.saved = static_cast<float*>(d->saved), p.ld_saved = ffn_ld(d->f);
  p.act = d->act;
  p.static_weights = static_weights();
  if (pairs) {
    return few_pair_bn(d->t) == 64 ? launch_few_pair<DT, 64>(c, a, a2, b, p)
                                   : launch_few_pair<DT, 128>(c, a, a2, b, p);
  }
  return launch_stream<DT == 0 ? sp24::kStreamF16 : sp24::kStreamBF16>(c, a, a2, b, p);
}

// Few tiles of the forward pass or of dx, K split over the pairs of a cluster;
// p.splits = 1 where that does not apply (no two pairs a tile, no such clusters).
template <int DT, int MODE>
sp24_status launch_ffn_split(const FfnCall& c, const CUtensorMap (&a)[2], const CUtensorMap (&b)[2],
                             sp24::FfnParams p, int want) {
  using C = sp24::FfnCfg<DT, MODE>;
  constexpr auto kern = sp24::ffn_split_kernel<DT, MODE>;
  const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles;
  p.splits = 1;
  if (want > 1) {
    static std::atomic<bool> attr_set[kMaxDevices];
    const sp24_status st = ensure_kernel_attrs(kern, attr_set, C::SMEM_BYTES);
    if (st != SP24_OK) return st;
    p.splits = resident_splits<kern>(sp24::kPairThreads, C::SMEM_BYTES, tiles, 2, want);
  }
  if (p.splits <= 1) return launch_ffn_pair<DT, MODE>(c, a, b, p);
  p.status = c.status;
  p.timeout_ns = kDefaultTimeoutNs;
  return launch_gemm_kernel(kern, static_cast<unsigned>(tiles * 2 * p.splits), sp24::kPairThreads, C::SMEM_BYTES,
                            c.stream, static_cast<unsigned>(2 * p.splits), true, a[0], a[1], b[0], b[1], p);
}

template <int DT>
sp24_status ffn_forward(const FfnCall& c, const sp24_ffn_desc* d, void* out, int64_t ld_out) {
  if (d->t <= kStreamMaxTokens) return ffn_forward_few<DT>(c, d, out, ld_out);
  CUtensorMap a[2], b[2];
  sp24_status st = encode_16(&a[0], d->x, d->t, d->h, stride_or(d->ldx, d->h), 128);
  if (st == SP24_OK) st = encode_16(&b[0], d->w_gate, d->f, d->h, stride_or(d->ld_gate, d->h), 128);
  if (st == SP24_OK) st = encode_16(&b[1], d->w_up, d->f, d->h, stride_or(d->ld_up, d->h), 128);
  if (st != SP24_OK) return st;
  a[1] = a[0];
  sp24::FfnParams p{};
  p.m = d->t, p.n = d->f;
  p.m_tiles = (d->t + 255) / 256, p.n_tiles = (d->f + 127) / 128;
  p.k_stages = (d->h + 63) / 64;
  p.group_m = 16;
  p.out0 = out, p.ld_out0 = ld_out, p.vec_out = out_vec(out, ld_out);
  p.saved = static_cast<float*>(d->saved), p.ld_saved = ffn_ld(d->f);
  p.act = d->act;
  // Few tiles and a long sum: K split over the pairs of a cluster, eight stages a
  // slice at least (1199 x 3704, f = 744, 30 tiles: 29.3 -> 19.7 us; 300 x 1000, f =
  // 776: 13.0 -> 10.8; slices of four stages gain nothing more).
  const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles;
  const int want =
      static_cast<int>(std::min<long long>({c.sm_count / 2 / tiles, sp24::kFfnMaxSplits, p.k_stages / 8}));
  return launch_ffn_split<DT, sp24::kFfnForward>(c, a, b, p, want);
}

template <int DT>
sp24_status ffn_backward(const FfnCall& c, const sp24_ffn_desc* d, const sp24_ffn_grads* g) {
  const int64_t ldw = ffn_ld(d->f), ldd = stride_or(g->ld_d_out, d->f);
  uint16_t* dg = static_cast<uint16_t*>(g->workspace);
  uint16_t* du = dg + static_cast<size_t>(d->t) * ldw;
  const long long chunks = static_cast<long long>(d->t) * ((d->f + 7) / 8);
  const unsigned grid = static_cast<unsigned>(std::min<long long>((chunks + 255) / 256, c.sm_count * 8));
  const bool vec = aligned16(g->d_out) && ldd % 8 == 0 && d->f % 8 == 0;
  auto kern = vec ? sp24::ffn_dgate_kernel<DT, 1> : sp24::ffn_dgate_kernel<DT, 0>;
  sp24_status st = launch_gemm_kernel(kern, grid, 256, 0, c.stream, 0, true, d->t, d->f,
                                      static_cast<const float*>(d->saved), static_cast<long long>(ldw),
                                      static_cast<const void*>(g->d_out), static_cast<long long>(ldd),
                                      static_cast<int>(d->act), dg);
  if (st != SP24_OK) return st;
  CUtensorMap a[2], b[2];
  if (g->dx != nullptr) {
    st = encode_16(&a[0], dg, d->t, d->f, ldw, 128);
    if (st == SP24_OK) st = encode_16(&a[1], du, d->t, d->f, ldw, 128);
    if (st == SP24_OK) st = encode_16(&b[0], d->w_gate, d->f, d->h, stride_or(d->ld_gate, d->h), 64);
    if (st == SP24_OK) st = encode_16(&b[1], d->w_up, d->f, d->h, stride_or(d->ld_up, d->h), 64);
    if (st != SP24_OK) return st;
    sp24::FfnParams p{};
    p.m = d->t, p.n = d->h;
    p.m_tiles = (d->t + 255) / 256, p.n_tiles = (d->h + 255) / 256;
    p.plane = (d->f + 63) / 64, p.k_stages = 2 * p.plane;
    p.group_m = 8;
    p.out0 = g->dx, p.ld_out0 = stride_or(g->ld_dx, d->h), p.vec_out = out_vec(g->dx, p.ld_out0);
    // Few tiles: K split over the pairs of a cluster (777 x 1000, f = 2744, 16
    // tiles of 86 stages: 45.0 -> 19.8 us with four; through the workspace 23.4).
    // Very few: split further, through the workspace (40 x 112, f = 12344, one tile:
    // 35.4 us with four pairs, 11.7 with 48 slices; 64 x 4096, f = 14336 keeps four).
    const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles;
    const int slices = dx_slices(d->t, d->h, d->f, std::min(kMaxPairs, c.sm_count / 2));
    const int want = static_cast<int>(std::min<long long>({c.sm_count / 2 / tiles, sp24::kFfnMaxSplits, p.k_stages}));
    if (slices > 0) {
      p.splits = slices;
      p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(g->workspace) + dgu_bytes(d->t, d->f));
      p.ld_partial = ffn_ld(d->h);
    }
    st = slices > 0 ? launch_ffn_pair<DT, sp24::kFfnDx>(c, a, b, p)
                    : launch_ffn_split<DT, sp24::kFfnDx>(c, a, b, p, want);
    if (st != SP24_OK) return st;
    if (slices > 0) {
      const long long runs = static_cast<long long>(d->t) * ((d->h + 7) / 8);
      auto sum = p.vec_out > 0 ? sp24::ffn_dx_sum_kernel<DT, 1> : sp24::ffn_dx_sum_kernel<DT, 0>;
      st = launch_gemm_kernel(sum, static_cast<unsigned>((runs + 31) / 32), 256, 0, c.stream, 0, true,
                              static_cast<const float*>(p.partial), p.splits, d->t, d->h, p.ld_partial, p.out0,
                              p.ld_out0);
      if (st != SP24_OK) return st;
    }
  }
  if (g->dw_gate != nullptr) {
    st = encode_16(&a[0], dg, d->t, d->f, ldw, 64);
    if (st == SP24_OK) st = encode_16(&a[1], du, d->t, d->f, ldw, 64);
    if (st == SP24_OK) st = encode_16(&b[0], d->x, d->t, d->h, stride_or(d->ldx, d->h), 64);
    if (st != SP24_OK) return st;
    b[1] = b[0];
    sp24::FfnParams p{};
    p.m = d->f, p.n = d->h;
    p.plane = (d->f + 255) / 256, p.m_tiles = 2 * p.plane, p.n_tiles = (d->h + 255) / 256;
    p.k_stages = (d->t + 63) / 64;
    p.group_m = 8;
    p.out0 = g->dw_gate, p.ld_out0 = stride_or(g->ld_dgate, d->h);
    p.out1 = g->dw_up, p.ld_out1 = stride_or(g->ld_dup, d->h);
    p.vec_out = std::min(out_vec(p.out0, p.ld_out0), out_vec(p.out1, p.ld_out1));
    st = launch_ffn_pair<DT, sp24::kFfnDw>(c, a, b, p);
  }
  return st;
}

}  // namespace

extern "C" {

sp24_status sp24_rmsnorm_quant(const sp24_rowquant_desc* d, sp24_stream_t stream) {
  return rows_quant<sp24::kRowsNorm>(d, stream);
}

sp24_status sp24_swiglu_quant(const sp24_rowquant_desc* d, sp24_stream_t stream) {
  return rows_quant<sp24::kRowsSwiglu>(d, stream);
}

sp24_status sp24_quantize_rows(const sp24_rowquant_desc* d, sp24_stream_t stream) {
  return rows_quant<sp24::kRowsPlain>(d, stream);
}

sp24_status sp24_gemm_scaled(const sp24_scaled_desc* d, sp24_stream_t stream) {
  sp24_status st = check_scaled(d);
  if (st != SP24_OK || d->n == 0) return st;
  DeviceInfo* di = nullptr;
  st = device_info(&di);
  if (st != SP24_OK) return st;
  const FfnCall c{di->sm_count, d->status_dev ? d->status_dev : di->status_word, as_stream(stream)};
  return d->dtype == SP24_I8 ? scaled<1>(c, d) : scaled<0>(c, d);
}

size_t sp24_ffn_saved_bytes(int t, int f) {
  return t <= 0 || f <= 0 ? 0 : static_cast<size_t>(t) * 2 * ffn_ld(f) * sizeof(float);
}

size_t sp24_ffn_workspace_bytes(int t, int h, int f) {
  if (t <= 0 || h <= 0 || f <= 0) return 0;
  // planes of dg and du, then the slices' sums
  return dgu_bytes(t, f) + static_cast<size_t>(dx_slices(t, h, f)) * t * ffn_ld(h) * sizeof(float);
}

sp24_status sp24_ffn_forward(const sp24_ffn_desc* d, void* out, int64_t ld_out,
                             sp24_stream_t stream) {
  sp24_status st = check_ffn(d);
  if (st != SP24_OK) return st;
  ld_out = stride_or(ld_out, d->f);
  if (ld_out < d->f) return SP24_ERR_SHAPE;
  if (d->t == 0) return SP24_OK;
  if (out == nullptr) return SP24_ERR_ARG;
  if (d->saved != nullptr && d->saved_bytes < sp24_ffn_saved_bytes(d->t, d->f))
    return SP24_ERR_WORKSPACE;
  DeviceInfo* di = nullptr;
  st = device_info(&di);
  if (st != SP24_OK) return st;
  const FfnCall c{di->sm_count, d->status_dev ? d->status_dev : di->status_word, as_stream(stream)};
  return d->dtype == SP24_F16 ? ffn_forward<0>(c, d, out, ld_out) : ffn_forward<1>(c, d, out, ld_out);
}

sp24_status sp24_ffn_backward(const sp24_ffn_desc* d, const sp24_ffn_grads* g,
                              sp24_stream_t stream) {
  sp24_status st = check_ffn(d);
  if (st != SP24_OK) return st;
  if (g == nullptr) return SP24_ERR_ARG;
  if ((g->dw_gate == nullptr) != (g->dw_up == nullptr)) return SP24_ERR_ARG;
  const int64_t ldd = stride_or(g->ld_d_out, d->f), lddx = stride_or(g->ld_dx, d->h),
                ldg = stride_or(g->ld_dgate, d->h), ldu = stride_or(g->ld_dup, d->h);
  if (ldd < d->f || lddx < d->h || ldg < d->h || ldu < d->h) return SP24_ERR_SHAPE;
  if (d->t > 0) {
    if (g->d_out == nullptr || d->saved == nullptr) return SP24_ERR_ARG;
    if (d->saved_bytes < sp24_ffn_saved_bytes(d->t, d->f) || g->workspace == nullptr ||
        g->workspace_bytes < sp24_ffn_workspace_bytes(d->t, d->h, d->f))
      return SP24_ERR_WORKSPACE;
    if (!aligned32(g->workspace)) return SP24_ERR_ALIGN;
  }
  DeviceInfo* di = nullptr;
  st = device_info(&di);
  if (st != SP24_OK) return st;
  cudaStream_t s = as_stream(stream);
  if (d->t == 0) {   // sums over no token
    if (g->dw_gate != nullptr) {
      SP24_CUDA_TRY(cudaMemset2DAsync(g->dw_gate, ldg * 2, 0, d->h * 2, d->f, s));
      SP24_CUDA_TRY(cudaMemset2DAsync(g->dw_up, ldu * 2, 0, d->h * 2, d->f, s));
    }
    return SP24_OK;
  }
  const FfnCall c{di->sm_count, d->status_dev ? d->status_dev : di->status_word, s};
  return d->dtype == SP24_F16 ? ffn_backward<0>(c, d, g) : ffn_backward<1>(c, d, g);
}

}  // extern "C"
