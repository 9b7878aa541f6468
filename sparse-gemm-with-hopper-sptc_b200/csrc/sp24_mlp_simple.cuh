// sp24_mlp_simple.cuh — the plain tiled scaled product on the CUDA cores: one
// thread per output, operands staged in shared memory.
#pragma once

#include "sp24_rows.cuh"

namespace sp24 {

struct ScaledParams {
  int m, n, k;
  const uint8_t* a_c;
  long long lda_c;
  const uint8_t* meta;
  int meta_mblocks;
  const uint8_t* x;
  long long ldx;
  const float *scale_m, *scale_n, *bias;
  void* c;
  long long ldc;
  int cdtype;
};

template <int I8>
__global__ void __launch_bounds__(256) scaled_simple_kernel(const ScaledParams P) {
  __shared__ float ws[16][65];
  __shared__ float xs[16][65];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int row0 = blockIdx.x * 16, tok0 = blockIdx.y * 16;
  auto val = [](uint8_t b) {
    if constexpr (I8) return static_cast<float>(static_cast<int8_t>(b));
    else return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
  };
  float acc = 0.0f;
  int iacc = 0;
  for (int k0 = 0; k0 < P.k; k0 += 64) {
    for (int i = threadIdx.x; i < 16 * 16; i += 256) {   // row i / 16, group i % 16
      const int row = row0 + i / 16, g = k0 / 4 + i % 16;
      float w[4] = {0, 0, 0, 0};
      if (row < P.m) {
        const uint8_t* atom = P.meta + (static_cast<size_t>(g / 32) * P.meta_mblocks + row / 128) * 2048;
        const uint32_t code = (atom[(row % 128) * 16 + (g % 32) / 2] >> (4 * (g & 1))) & 15u;
        w[code & 3] = val(P.a_c[row * P.lda_c + 2 * g]);
        w[code >> 2] = val(P.a_c[row * P.lda_c + 2 * g + 1]);
      }
      for (int j = 0; j < 4; ++j) ws[i / 16][(i % 16) * 4 + j] = w[j];
    }
    for (int i = threadIdx.x; i < 16 * 64; i += 256) {
      const int tok = tok0 + i / 64;
      xs[i / 64][i % 64] = tok < P.n ? val(P.x[tok * P.ldx + k0 + i % 64]) : 0.0f;
    }
    __syncthreads();
    float part = 0.0f;
    for (int j = 0; j < 64; ++j) part += ws[tx][j] * xs[ty][j];
    if constexpr (I8) iacc += static_cast<int>(part);   // exact: below 2^24
    else acc += part;
    __syncthreads();
  }
  const int row = row0 + tx, tok = tok0 + ty;
  if (row >= P.m || tok >= P.n) return;
  float v = I8 ? static_cast<float>(iacc) : acc;
  v *= (P.scale_m ? P.scale_m[row] : 1.0f) * (P.scale_n ? P.scale_n[tok] : 1.0f);
  if (P.bias) v += P.bias[row];
  const long long o = tok * P.ldc + row;
  if (P.cdtype == 0) store16<0>(P.c, o, v);
  else if (P.cdtype == 1) store16<1>(P.c, o, v);
  else static_cast<float*>(P.c)[o] = v;
}

}  // namespace sp24
