// sp24_rows.cuh — rows of 16-bit activations to 8-bit codes with one scale per
// row: after a residual addition and a root-mean-square norm, after the SwiGLU
// product, or as they are.
//
// Bound by HBM: each input is read once and each output written once.  B200,
// measured copy rate 6.5 TB/s, device time over rotating buffers: norm with residual
// 8192 x 4096 bf16 (235 MB) 36.6 us, 6.4 TB/s; SwiGLU 4096 x 14336 (294 MB) 47.9 us,
// 6.1 TB/s; plain 8192 x 14336 (352 MB) 55.7 us, 6.3 TB/s.  The SwiGLU is nearest to
// another limit: its exponential and reciprocal keep their unit busy half of the
// time.
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
  float eps, inv_cols;
  uint8_t* q;
  float* scale;
};

// Two fp32 operations in one instruction.
SP24_DEV uint64_t bits2(float2 a) { return *reinterpret_cast<uint64_t*>(&a); }
SP24_DEV float2 from_bits2(uint64_t r) { return *reinterpret_cast<float2*>(&r); }
SP24_DEV float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return from_bits2(r);
}
SP24_DEV float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return from_bits2(r);
}
SP24_DEV float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return from_bits2(r);
}

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
// the slow unit that the exponentials need (4096 x 14336 SwiGLU, before later
// steps: 63.7 us with conversions, 55.3 with additions).
template <int I8>
SP24_DEV uint32_t codes2(float a, float b) {
  if constexpr (I8) {
    return __byte_perm(__float_as_uint(a + 12582912.0f), __float_as_uint(b + 12582912.0f), 0x0040) & 0xFFFFu;
  } else {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  }
}

// V neighbouring values of a row as they lie in memory: one load of 2 V bytes, in
// the low words of the result.
template <int V>
SP24_DEV uint4 load_raw(const void* p, long long i) {
  const uint16_t* q = static_cast<const uint16_t*>(p) + i;
  if constexpr (V == 8) {
    return *reinterpret_cast<const uint4*>(q);
  } else if constexpr (V == 4) {
    const uint2 w = *reinterpret_cast<const uint2*>(q);
    return make_uint4(w.x, w.y, 0, 0);
  } else if constexpr (V == 2) {
    return make_uint4(*reinterpret_cast<const uint32_t*>(q), 0, 0, 0);
  } else {
    return make_uint4(*q, 0, 0, 0);
  }
}
// ... and V codes, two to a half word, or V 16-bit values, two to a word, back.
template <int V>
SP24_DEV void store_codes(uint8_t* q, const uint32_t (&k)[4]) {
  if constexpr (V == 8) __stcs(reinterpret_cast<uint2*>(q), make_uint2(k[0] | k[1] << 16, k[2] | k[3] << 16));
  else if constexpr (V == 4) __stcs(reinterpret_cast<uint32_t*>(q), k[0] | k[1] << 16);
  else if constexpr (V == 2) *reinterpret_cast<uint16_t*>(q) = static_cast<uint16_t>(k[0]);
  else *q = static_cast<uint8_t>(k[0]);
}
template <int V>
SP24_DEV void store_raw(void* p, long long i, const uint32_t (&w)[4]) {
  uint16_t* q = static_cast<uint16_t*>(p) + i;
  if constexpr (V == 8) __stcs(reinterpret_cast<uint4*>(q), make_uint4(w[0], w[1], w[2], w[3]));
  else if constexpr (V == 4) __stcs(reinterpret_cast<uint2*>(q), make_uint2(w[0], w[1]));
  else if constexpr (V == 2) *reinterpret_cast<uint32_t*>(q) = w[0];
  else *q = static_cast<uint16_t>(w[0]);
}

// The two values of one 32-bit word (V = 1: the one value and a zero).
template <int DT>
SP24_DEV float2 unpack2(uint32_t w) {
  if constexpr (DT == 0) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
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

// sigmoid(x) = 1 / (1 + 2^(-x log2 e)), the reciprocal and the power each to
// about two ulp: beside the 8-bit step that cannot be seen, and the IEEE
// division made the SwiGLU compute-bound.  Far below zero the power is infinite
// and the result 0 (true size < 1e-37).
SP24_DEV float sigmoid_of(float v) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return r;
}
SP24_DEV float silu_of(float v) { return v * sigmoid_of(v); }   // -infinity: NaN, as the formula

// What the threads of a row agree on.
struct RowStats {
  float sum;      // of squares (the norm)
  uint32_t top;   // bits of the largest magnitude
};

// Reduces both over the row's threads: a warp, or the whole block with one
// barrier (every warp folds the warps' values itself, in the same order).
// Successive rows alternate between two `sh`: a warp can be at most one barrier
// ahead of another, so none still reads what the next row overwrites.
template <bool ONE_WARP, bool SUM>
SP24_DEV RowStats row_reduce(float sum, uint32_t top, uint2* sh) {
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (SUM) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  if constexpr (!ONE_WARP) {
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) sh[threadIdx.x >> 5] = make_uint2(__float_as_uint(sum), top);
    __syncthreads();
    const uint2 v = lane < warps ? sh[lane] : make_uint2(0, 0);
    top = __reduce_max_sync(0xffffffffu, v.y);
    if constexpr (SUM) {
      sum = __uint_as_float(v.x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
  }
  return {sum, top};
}

// max(a, |b|), NaN if either is: its bits then order above infinity's.
SP24_DEV float max_abs(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}

// Asynchronous copy of V 16-bit values (V = 8, 4, 2).
template <int V>
SP24_DEV void cp_async(void* dst, const void* src) {
  if constexpr (V == 8)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(2 * V) : "memory");
}
SP24_DEV void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// The factor that turns a row's values into codes, from the bits of the largest
// magnitude (these order as unsigned numbers, infinity and NaN on top), and the
// row's scale for values that are `gain` times those.  Quotients to two ulp.
struct RowScale {
  float scale, lift, inv;
  bool bad;
};
template <int I8>
SP24_DEV RowScale row_scale(uint32_t top, float gain) {
  constexpr float Q = I8 ? 127.0f : 448.0f;
  RowScale r;
  const float amax = __uint_as_float(top);
  // The approximate quotient wants its divisor within 2^+-126: rows outside are
  // brought in first.
  r.lift = amax < 1e-30f ? 0x1p100f : amax > 1e30f ? 0x1p-40f : 1.0f;
  const float bounded = amax * r.lift;
  // A gain of 0: the squares overflowed; NaN: they met one; above 2^63: their mean
  // is below fp32's normal range, and the subnormal sum has lost digits.
  r.bad = !(bounded < 3e38f) || (top != 0 && !(gain > 0.0f && gain <= 0x1p63f));
  r.inv = (r.bad || top == 0) ? 0.0f : __fdividef(Q, bounded);
  r.scale = r.bad ? __uint_as_float(0x7FC00000u) : top == 0 ? 0.0f : amax * gain * (1.0f / Q);
  return r;
}

// One pass over memory: a row's values stay in registers as fp32 from the load
// to the codes (VPT vectors of V columns a thread).  The norm's factor
// r = 1 / sqrt(mean s^2 + eps) is the same for the whole row, so it cancels in
// the codes: with a = max |s w|, q = round(s w Q / a) and scale = r a / Q.  The sum
// of squares and the largest magnitude are therefore reduced together, and a
// row costs one barrier (8192 x 4096: 39.6 us with one after the other).
// ONE_WARP: a warp per row, blockDim.x / 32 rows a block; else a block per row.
//
// The grid is resident and walks the rows.  With V > 1 every thread has a slot
// in shared memory for each of its vectors: it issues the copies of its next
// row (cp.async) as soon as it has unpacked the current one, so loads stay in
// flight through the reductions and stores.  A slot has one owner: no barrier
// guards it, only the owner's own wait.
template <int DT, int MODE, int I8, int V, int VPT, bool ONE_WARP>
__global__ void __launch_bounds__(ONE_WARP ? 256 : 1024) rows_quant_kernel(const RowsParams P) {
  extern __shared__ __align__(16) uint8_t slots[];   // V > 1: [input][VPT][blockDim.x] vectors
  __shared__ uint2 sh[2][32];
  constexpr int H = V > 1 ? V / 2 : 1;   // words of two values a vector
  griddep_launch_dependents();
  const int tid = ONE_WARP ? threadIdx.x & 31 : threadIdx.x;
  const int step = ONE_WARP ? 32 : blockDim.x;
  const int per_block = ONE_WARP ? blockDim.x >> 5 : 1;
  const long long stride = static_cast<long long>(gridDim.x) * per_block;
  long long r = blockIdx.x * static_cast<long long>(per_block) + (ONE_WARP ? threadIdx.x >> 5 : 0);
  const void* other = MODE == kRowsSwiglu ? P.up : P.residual;
  const long long ld_other = MODE == kRowsSwiglu ? P.ld_up : P.ld_residual;
  const bool two = MODE == kRowsSwiglu || (MODE == kRowsNorm && other != nullptr);
  // Slot of vector i of input w.
  auto slot = [&](int w, int i) { return slots + ((w * VPT + i) * blockDim.x + threadIdx.x) * (2 * V); };
  auto fetch = [&](long long row) {
    const uint16_t* px = static_cast<const uint16_t*>(P.x) + row * P.ldx;
    const uint16_t* po = static_cast<const uint16_t*>(other) + row * ld_other;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * step) * V;
      if (c < P.cols) {
        cp_async<V>(slot(0, i), px + c);
        if (two) cp_async<V>(slot(1, i), po + c);
      }
    }
  };
  if (r >= P.rows) return;
  griddep_wait();
  if constexpr (V > 1) fetch(r);
  uint4 rw[VPT];   // past the row's end 0
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (tid + i * step) * V;
    rw[i] = make_uint4(0, 0, 0, 0);
    if (MODE == kRowsNorm && c < P.cols) rw[i] = load_raw<V>(P.weight, c);
  }
  int parity = 0;
  for (; r < P.rows; r += stride) {
    float2 v[VPT][H];
    float2 ss = make_float2(0.0f, 0.0f);
    float top = 0.0f;
    if constexpr (V > 1) cp_async_wait_all();
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * step) * V;
      uint4 rx = make_uint4(0, 0, 0, 0), ro = rx;
      if (c < P.cols) {
        rx = V > 1 ? load_raw<V>(slot(0, i), 0) : load_raw<V>(P.x, r * P.ldx + c);
        if (two) ro = V > 1 ? load_raw<V>(slot(1, i), 0) : load_raw<V>(other, r * ld_other + c);
      }
      const uint32_t wx[4] = {rx.x, rx.y, rx.z, rx.w}, wo[4] = {ro.x, ro.y, ro.z, ro.w};
      const uint32_t ww[4] = {rw[i].x, rw[i].y, rw[i].z, rw[i].w};
#pragma unroll
      for (int j = 0; j < H; ++j) {
        float2 a = unpack2<DT>(wx[j]);
        if constexpr (MODE == kRowsSwiglu) a = mul2(make_float2(silu_of(a.x), silu_of(a.y)), unpack2<DT>(wo[j]));
        if constexpr (MODE == kRowsNorm) {
          if (two) a = add2(a, unpack2<DT>(wo[j]));
          ss = fma2(a, a, ss);
        }
        v[i][j] = a;
      }
      if (MODE == kRowsNorm && P.residual_out != nullptr && c < P.cols) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < H; ++j) w[j] = pack16<DT>(v[i][j].x, v[i][j].y);
        store_raw<V>(P.residual_out, r * P.ld_residual_out + c, w);
      }
#pragma unroll
      for (int j = 0; j < H; ++j) {
        if constexpr (MODE == kRowsNorm) v[i][j] = mul2(v[i][j], unpack2<DT>(ww[j]));
        top = max_abs(max_abs(top, v[i][j].x), v[i][j].y);
      }
    }
    if constexpr (V > 1)
      if (r + stride < P.rows) fetch(r + stride);
    const RowStats st = row_reduce<ONE_WARP, MODE == kRowsNorm>(ss.x + ss.y, __float_as_uint(top), sh[parity]);
    parity ^= 1;
    const float gain = MODE == kRowsNorm ? rsqrtf(st.sum * P.inv_cols + P.eps) : 1.0f;
    const RowScale s = row_scale<I8>(st.top, gain);
    if (tid == 0) P.scale[r] = s.scale;
    if (s.bad || s.lift != 1.0f) {   // rare, the same for the whole row
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < H; ++j)
          v[i][j] = s.bad ? make_float2(0.0f, 0.0f) : make_float2(v[i][j].x * s.lift, v[i][j].y * s.lift);
    }
    const float2 inv = make_float2(s.inv, s.inv);
    uint8_t* q = P.q + r * P.ldq;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * step) * V;
      if (c >= P.cols) continue;
      uint32_t k[4];
#pragma unroll
      for (int j = 0; j < H; ++j) {
        const float2 a = mul2(v[i][j], inv);
        k[j] = codes2<I8>(a.x, a.y);
      }
      store_codes<V>(q + c, k);
    }
  }
}

// Rows too long for the registers of one block: two passes over each, the
// second from cache.
template <int DT, int MODE, int I8>
__global__ void __launch_bounds__(1024) rows_quant_long_kernel(const RowsParams P) {
  __shared__ uint2 sh[32];
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
  auto weight = [&](int c) { return MODE == kRowsNorm ? load16<DT>(P.weight, c) : 1.0f; };
  float ss = 0.0f, top = 0.0f;
  for (int c = threadIdx.x; c < P.cols; c += blockDim.x) {
    const float b = base(c);
    ss += b * b;
    top = max_abs(top, b * weight(c));
  }
  const RowStats st = row_reduce<false, MODE == kRowsNorm>(ss, __float_as_uint(top), sh);
  const RowScale s =
      row_scale<I8>(st.top, MODE == kRowsNorm ? rsqrtf(st.sum * P.inv_cols + P.eps) : 1.0f);
  if (threadIdx.x == 0) P.scale[r] = s.scale;
  for (int c = threadIdx.x; c < P.cols; c += blockDim.x) {
    // The sum is written last: residual_out may be the residual itself.
    const float b = base(c);
    const float v = s.bad ? 0.0f : b * weight(c) * s.lift * s.inv;
    if (MODE == kRowsNorm && P.residual_out != nullptr)
      store16<DT>(P.residual_out, r * P.ld_residual_out + c, b);
    P.q[r * P.ldq + c] = static_cast<uint8_t>(codes2<I8>(v, 0.0f));
  }
}

}  // namespace sp24
