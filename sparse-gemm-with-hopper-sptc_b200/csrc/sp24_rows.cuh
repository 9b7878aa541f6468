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
// rounding step, so the integers stay within +-127; e4m3 saturates.  Integers
// are rounded by adding 1.5 * 2^23, which leaves v's nearest integer (halves to
// even) in the low bits of the sum: an addition where a conversion would take
// the slow unit that the exponentials need (4096 x 14336 SwiGLU: 64 us with
// conversions, 54 us in e4m3).
template <int I8>
SP24_DEV uint32_t codes2(float a, float b) {
  if constexpr (I8) {
    return __byte_perm(__float_as_uint(a + 12582912.0f), __float_as_uint(b + 12582912.0f), 0x0040) & 0xFFFFu;
  } else {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  }
}

// V neighbouring values of a row as they lie in memory: 16 bytes (V = 8) or one
// element.
template <int V>
SP24_DEV uint4 load_raw(const void* p, long long i) {
  const uint16_t* q = static_cast<const uint16_t*>(p) + i;
  if constexpr (V == 8) return *reinterpret_cast<const uint4*>(q);
  else return make_uint4(*q, 0, 0, 0);
}
template <int DT, int V>
SP24_DEV void unpack_raw(const uint4& w, float (&v)[V]) {
  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const uint32_t h = ws[j / 2] >> (16 * (j & 1));
    if constexpr (DT == 0) v[j] = __half2float(__ushort_as_half(static_cast<unsigned short>(h)));
    else v[j] = (j & 1) ? __uint_as_float(ws[j / 2] & 0xFFFF0000u) : __uint_as_float(ws[j / 2] << 16);
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

// x sigmoid(x) = x / (1 + 2^(-x log2 e)), the reciprocal and the power each to
// about two ulp: beside the 8-bit step that cannot be seen, and the IEEE
// division made the SwiGLU compute-bound.  Far below zero the power is infinite
// and the result -0 (true size < 1e-36); -infinity gives NaN, as the formula does.
SP24_DEV float silu_of(float v) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return v * r;
}

// Reduction over the threads of one row: a warp, or the whole block (one
// barrier; every warp folds the warps' values itself, in the same order).  0
// is the identity of both uses.  Successive calls alternate between two `sh`.
template <bool ONE_WARP, typename F>
SP24_DEV uint32_t row_reduce(uint32_t v, uint32_t* sh, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  if constexpr (!ONE_WARP) {
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? sh[lane] : 0u;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  }
  return v;
}

// max(a, |b|), NaN if either is: its bits then order above infinity's.
SP24_DEV float max_abs(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}

SP24_DEV void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
SP24_DEV void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

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
//
// The grid is resident and walks the rows.  With V = 8 every thread has a slot
// in shared memory for each of its vectors: it issues the copies of its next
// row (cp.async) as soon as it has unpacked the current one, so loads stay in
// flight through the reductions and stores.  A slot has one owner: no barrier
// guards it, only the owner's own wait.
template <int DT, int MODE, int I8, int V, int VPT, bool ONE_WARP>
__global__ void __launch_bounds__(ONE_WARP ? 256 : 1024) rows_quant_kernel(const RowsParams P) {
  extern __shared__ uint4 slots[];   // V = 8: [input][VPT][blockDim.x]
  __shared__ uint32_t sh[2][32];
  griddep_launch_dependents();
  const int tid = ONE_WARP ? threadIdx.x & 31 : threadIdx.x;
  const int step = ONE_WARP ? 32 : blockDim.x;
  const int per_block = ONE_WARP ? blockDim.x >> 5 : 1;
  const long long stride = static_cast<long long>(gridDim.x) * per_block;
  long long r = blockIdx.x * static_cast<long long>(per_block) + (ONE_WARP ? threadIdx.x >> 5 : 0);
  const void* other = MODE == kRowsSwiglu ? P.up : P.residual;
  const long long ld_other = MODE == kRowsSwiglu ? P.ld_up : P.ld_residual;
  const bool two = MODE == kRowsSwiglu || (MODE == kRowsNorm && other != nullptr);
  uint4* mine = slots + threadIdx.x;
  auto fetch = [&](long long row) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * step) * V;
      if (c < P.cols) {
        cp_async16(mine + i * blockDim.x, static_cast<const uint16_t*>(P.x) + row * P.ldx + c);
        if (two)
          cp_async16(mine + (VPT + i) * blockDim.x, static_cast<const uint16_t*>(other) + row * ld_other + c);
      }
    }
  };
  if (r >= P.rows) return;
  griddep_wait();
  if constexpr (V == 8) fetch(r);
  uint4 rw[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (tid + i * step) * V;
    rw[i] = make_uint4(0, 0, 0, 0);
    if (MODE == kRowsNorm && c < P.cols) rw[i] = load_raw<V>(P.weight, c);
  }
  for (; r < P.rows; r += stride) {
    float v[VPT][V];
    if constexpr (V == 8) cp_async_wait_all();
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * step) * V;
      uint4 rx = make_uint4(0, 0, 0, 0), ro = rx;
      if (c < P.cols) {
        rx = V == 8 ? mine[i * blockDim.x] : load_raw<V>(P.x, r * P.ldx + c);
        if (two) ro = V == 8 ? mine[(VPT + i) * blockDim.x] : load_raw<V>(other, r * ld_other + c);
      }
      float o[V];
      unpack_raw<DT, V>(rx, v[i]);
      unpack_raw<DT, V>(ro, o);   // zeroes where there is no second input
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (MODE == kRowsSwiglu) v[i][j] = silu_of(v[i][j]) * o[j];
        if (MODE == kRowsNorm) v[i][j] += o[j];
      }
    }
    if constexpr (V == 8)
      if (r + stride < P.rows) fetch(r + stride);
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
        float w[V];
        unpack_raw<DT, V>(rw[i], w);
        const bool in = (tid + i * step) * V < P.cols;   // past the end 0, even if rstd is not finite
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = in ? v[i][j] * rstd * w[j] : 0.0f;
      }
    }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) top = max_abs(top, v[i][j]);
    const uint32_t mx = row_reduce<ONE_WARP>(__float_as_uint(top), sh[1],
                                             [](uint32_t a, uint32_t b) { return max(a, b); });
    const RowScale s = row_scale<I8>(mx);
    if (tid == 0) P.scale[r] = s.scale;
    if (s.bad || s.lift != 1.0f) {   // rare, the same for the whole row
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = s.bad ? 0.0f : v[i][j] * s.lift;
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * step) * V;
      if (c >= P.cols) continue;
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] *= s.inv;
      uint8_t* q = P.q + r * P.ldq + c;
      if constexpr (V == 8) {
        __stcs(reinterpret_cast<uint2*>(q),
               make_uint2(codes2<I8>(v[i][0], v[i][1]) | codes2<I8>(v[i][2], v[i][3]) << 16,
                          codes2<I8>(v[i][4], v[i][5]) | codes2<I8>(v[i][6], v[i][7]) << 16));
      } else {
        q[0] = static_cast<uint8_t>(codes2<I8>(v[i][0], 0.0f));
      }
    }
    // The norm's two barriers order the uses of sh between rows; the other
    // modes have one a row and need a second before sh[1] is written again.
    if constexpr (!ONE_WARP && MODE != kRowsNorm) __syncthreads();
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
