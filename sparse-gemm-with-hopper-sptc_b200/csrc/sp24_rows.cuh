// sp24_rows.cuh — rows of 16-bit activations to 8-bit codes with one scale per
// row: after a residual addition and a root-mean-square norm, after the SwiGLU
// product, or as they are.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "sp24_ptx.cuh"

namespace sp24 {

enum : int { kRowsPlain = 0, kRowsNorm = 1, kRowsSwiglu = 2 };

struct RowsParams {
  int rows, cols;
  const void *x, *up, *residual, *weight;
  void* residual_out;
  long long ldx, ld_up, ld_residual, ld_residual_out, ldq;
  float eps;
  uint8_t* q;
  float* scale;
};

template <int DT>
SP24_DEV float load16(const void* p, long long i) {
  if constexpr (DT == 0) return __half2float(static_cast<const __half*>(p)[i]);
  else return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
template <int DT>
SP24_DEV void store16(void* p, long long i, float v) {
  if constexpr (DT == 0) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// Two neighbouring 8-bit codes, the first in the low byte.  |v| <= Q up to a
// rounding step, so the integers stay within +-127; e4m3 saturates.
template <int I8>
SP24_DEV uint32_t codes2(float a, float b) {
  if constexpr (I8) {
    return __byte_perm(static_cast<uint32_t>(__float2int_rn(a)),
                       static_cast<uint32_t>(__float2int_rn(b)), 0x0040) & 0xFFFFu;
  } else {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  }
}

// V values of a row, V = 8: one 16-byte load; V = 1: one element.
template <int DT, int V>
SP24_DEV void load_vec(const void* p, long long i, float (&v)[V]) {
  if constexpr (V == 8) {
    const uint4 w = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i));
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == 0) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&ws[j]));
        v[2 * j] = f.x, v[2 * j + 1] = f.y;
      } else {
        v[2 * j] = __uint_as_float(ws[j] << 16);
        v[2 * j + 1] = __uint_as_float(ws[j] & 0xFFFF0000u);
      }
    }
  } else {
    v[0] = load16<DT>(p, i);
  }
}

template <int DT>
SP24_DEV uint32_t pack16(float lo, float hi) {
  if constexpr (DT == 0) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

SP24_DEV float silu_of(float v) { return v / (1.0f + __expf(-v)); }

// Reduction over the threads of one row: a warp (W = 1) or the whole block.
template <bool ONE_WARP, typename F>
SP24_DEV uint32_t row_reduce(uint32_t v, uint32_t* sh, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  if constexpr (!ONE_WARP) {
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    // Every warp folds the warps' values again, in the same order.
    v = sh[(threadIdx.x & 31) % warps];
    uint32_t r = __shfl_sync(0xffffffffu, v, 0);
    for (int w = 1; w < warps; ++w) r = f(r, __shfl_sync(0xffffffffu, v, w));
    v = r;
  }
  return v;
}

// Scale of a row from the bits of its largest |y| (these order as unsigned
// numbers, infinity and NaN on top), and the factor that gives its codes.
struct RowScale {
  float scale, lift, inv;
  bool bad;
};
template <int I8>
SP24_DEV RowScale row_scale(uint32_t mx) {
  constexpr float Q = I8 ? 127.0f : 448.0f;
  RowScale r;
  const float amax = __uint_as_float(mx);
  r.bad = mx >= 0x7F800000u;
  // Q / amax overflows for the smallest rows: those are scaled up first.
  r.lift = amax < 1e-30f ? 0x1p100f : 1.0f;
  r.inv = (r.bad || mx == 0) ? 0.0f : Q / (amax * r.lift);
  r.scale = r.bad ? __uint_as_float(0x7FC00000u) : amax / Q;
  return r;
}

// One pass over memory: a row's values stay in registers as fp32 from the load
// to the codes (VPT vectors of V columns a thread), between the two row-wide
// reductions (the norm's sum of squares, then the largest magnitude).
// ONE_WARP: a warp per row, blockDim.x / 32 rows a block; else a block per row.
template <int DT, int MODE, int I8, int V, int VPT, bool ONE_WARP>
__global__ void __launch_bounds__(1024) rows_quant_kernel(const RowsParams P) {
  __shared__ uint32_t sh[2][32];
  griddep_launch_dependents();
  const int tid = ONE_WARP ? threadIdx.x & 31 : threadIdx.x;
  const int step = ONE_WARP ? 32 : blockDim.x;
  const long long r = ONE_WARP ? blockIdx.x * static_cast<long long>(blockDim.x >> 5) + (threadIdx.x >> 5)
                               : blockIdx.x;
  if (ONE_WARP && r >= P.rows) return;
  griddep_wait();
  float v[VPT][V];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (tid + i * step) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) v[i][j] = 0.0f;
    if (c < P.cols) load_vec<DT, V>(P.x, r * P.ldx + c, v[i]);
  }
  if (MODE == kRowsSwiglu || (MODE == kRowsNorm && P.residual != nullptr)) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * step) * V;
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = 0.0f;
      if (c < P.cols)
        load_vec<DT, V>(MODE == kRowsSwiglu ? P.up : P.residual,
                        r * (MODE == kRowsSwiglu ? P.ld_up : P.ld_residual) + c, o);
#pragma unroll
      for (int j = 0; j < V; ++j)
        v[i][j] = MODE == kRowsSwiglu ? silu_of(v[i][j]) * o[j] : v[i][j] + o[j];
    }
  }
  if constexpr (MODE == kRowsNorm) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * step) * V;
      if (P.residual_out != nullptr && c < P.cols) {
        const long long o = r * P.ld_residual_out + c;
        if constexpr (V == 8) {
          __stcs(reinterpret_cast<uint4*>(static_cast<uint16_t*>(P.residual_out) + o),
                 make_uint4(pack16<DT>(v[i][0], v[i][1]), pack16<DT>(v[i][2], v[i][3]),
                            pack16<DT>(v[i][4], v[i][5]), pack16<DT>(v[i][6], v[i][7])));
        } else {
          store16<DT>(P.residual_out, o, v[i][0]);
        }
      }
#pragma unroll
      for (int j = 0; j < V; ++j) ss += v[i][j] * v[i][j];
    }
    ss = __uint_as_float(row_reduce<ONE_WARP>(__float_as_uint(ss), sh[0], [](uint32_t a, uint32_t b) {
      return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
    const float rstd = rsqrtf(ss / static_cast<float>(P.cols) + P.eps);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * step) * V;
      float w[V];
#pragma unroll
      for (int j = 0; j < V; ++j) w[j] = 0.0f;
      if (c < P.cols) {
        if constexpr (V == 8) {
          const uint4 u = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(P.weight) + c));
          const uint32_t us[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = load16<DT>(&us[j / 2], j & 1);
        } else {
          w[0] = load16<DT>(P.weight, c);
        }
      }
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = c < P.cols ? v[i][j] * rstd * w[j] : 0.0f;
    }
  }
  uint32_t mx = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) mx = max(mx, __float_as_uint(v[i][j]) & 0x7FFFFFFFu);
  mx = row_reduce<ONE_WARP>(mx, sh[1], [](uint32_t a, uint32_t b) { return max(a, b); });
  const RowScale s = row_scale<I8>(mx);
  if (tid == 0) P.scale[r] = s.scale;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (tid + i * step) * V;
    if (c >= P.cols) continue;
#pragma unroll
    for (int j = 0; j < V; ++j) v[i][j] = s.bad ? 0.0f : v[i][j] * s.lift * s.inv;
    uint8_t* q = P.q + r * P.ldq + c;
    if constexpr (V == 8) {
      *reinterpret_cast<uint2*>(q) =
          make_uint2(codes2<I8>(v[i][0], v[i][1]) | codes2<I8>(v[i][2], v[i][3]) << 16,
                     codes2<I8>(v[i][4], v[i][5]) | codes2<I8>(v[i][6], v[i][7]) << 16);
    } else {
      q[0] = static_cast<uint8_t>(codes2<I8>(v[i][0], 0.0f));
    }
  }
}

// Rows too long for the registers of one block: three passes over each, the
// later ones from cache.
template <int DT, int MODE, int I8>
__global__ void __launch_bounds__(1024) rows_quant_long_kernel(const RowsParams P) {
  __shared__ uint32_t sh[2][32];
  griddep_launch_dependents();
  griddep_wait();
  const long long r = blockIdx.x;
  auto base = [&](int c) -> float {
    const float v = load16<DT>(P.x, r * P.ldx + c);
    if constexpr (MODE == kRowsNorm) {
      return P.residual != nullptr ? v + load16<DT>(P.residual, r * P.ld_residual + c) : v;
    } else if constexpr (MODE == kRowsSwiglu) {
      return silu_of(v) * load16<DT>(P.up, r * P.ld_up + c);
    } else {
      return v;
    }
  };
  float rstd = 1.0f;
  if constexpr (MODE == kRowsNorm) {
    float ss = 0.0f;
    for (int c = threadIdx.x; c < P.cols; c += blockDim.x) {
      const float v = base(c);
      ss += v * v;
    }
    ss = __uint_as_float(row_reduce<false>(__float_as_uint(ss), sh[0], [](uint32_t a, uint32_t b) {
      return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
    rstd = rsqrtf(ss / static_cast<float>(P.cols) + P.eps);
  }
  auto value = [&](float b, int c) {
    if constexpr (MODE == kRowsNorm) return b * rstd * load16<DT>(P.weight, c);
    else return b;
  };
  uint32_t mx = 0;
  for (int c = threadIdx.x; c < P.cols; c += blockDim.x)
    mx = max(mx, __float_as_uint(value(base(c), c)) & 0x7FFFFFFFu);
  mx = row_reduce<false>(mx, sh[1], [](uint32_t a, uint32_t b) { return max(a, b); });
  const RowScale s = row_scale<I8>(mx);
  if (threadIdx.x == 0) P.scale[r] = s.scale;
  for (int c = threadIdx.x; c < P.cols; c += blockDim.x) {
    // The sum is written last: residual_out may be the residual itself.
    const float b = base(c);
    const float v = s.bad ? 0.0f : value(b, c) * s.lift * s.inv;
    if (MODE == kRowsNorm && P.residual_out != nullptr)
      store16<DT>(P.residual_out, r * P.ld_residual_out + c, b);
    P.q[r * P.ldq + c] = static_cast<uint8_t>(codes2<I8>(v, 0.0f));
  }
}

}  // namespace sp24
