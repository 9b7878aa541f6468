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

// 8-bit code of v * inv, |v * inv| <= Q up to rounding.
template <int I8>
SP24_DEV uint32_t to_code(float v) {
  if constexpr (I8) {
    return static_cast<uint32_t>(max(-127, min(127, __float2int_rn(v)))) & 0xFFu;
  } else {
    return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
  }
}

template <typename F>
SP24_DEV uint32_t block_reduce(uint32_t v, uint32_t* sh, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  const int warps = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh[0];
  for (int w = 1; w < warps; ++w) v = f(v, sh[w]);
  __syncthreads();
  return v;
}

// One block per row; three passes over it, the later ones from cache.
template <int DT, int MODE, int I8>
__global__ void __launch_bounds__(256) rows_quant_kernel(const RowsParams P) {
  __shared__ uint32_t sh[8];
  constexpr float Q = I8 ? 127.0f : 448.0f;
  const long long r = blockIdx.x;
  auto base = [&](int c) -> float {
    const float v = load16<DT>(P.x, r * P.ldx + c);
    if constexpr (MODE == kRowsNorm) {
      return P.residual != nullptr ? v + load16<DT>(P.residual, r * P.ld_residual + c) : v;
    } else if constexpr (MODE == kRowsSwiglu) {
      return v / (1.0f + __expf(-v)) * load16<DT>(P.up, r * P.ld_up + c);
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
    ss = __uint_as_float(block_reduce(__float_as_uint(ss), sh, [](uint32_t a, uint32_t b) {
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
  mx = block_reduce(mx, sh, [](uint32_t a, uint32_t b) { return max(a, b); });
  // The bits of |y| order as unsigned numbers, infinity and NaN on top.
  const float amax = __uint_as_float(mx);
  const bool bad = mx >= 0x7F800000u;
  // Q / amax overflows for the smallest rows: those are scaled up first.
  const float lift = amax < 1e-30f ? 0x1p100f : 1.0f;
  const float inv = (bad || mx == 0) ? 0.0f : Q / (amax * lift);
  for (int c = threadIdx.x; c < P.cols; c += blockDim.x) {
    const float b = base(c);
    if (MODE == kRowsNorm && P.residual_out != nullptr)
      store16<DT>(P.residual_out, r * P.ld_residual_out + c, b);
    const float v = bad ? 0.0f : value(b, c) * lift * inv;
    P.q[r * P.ldq + c] = static_cast<uint8_t>(to_code<I8>(v));
  }
  if (threadIdx.x == 0) P.scale[r] = bad ? __uint_as_float(0x7FC00000u) : amax / Q;
}

}  // namespace sp24
