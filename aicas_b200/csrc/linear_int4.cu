// Decode-side products with 4-bit weights:
//   y[r, n] = sum_k x'[r, k] * scale[n, k / g] * (q[n, k] - zero[n, k / g])
// with x' = x or its RMSNorm, and a residual or SiLU(gate) * up epilogue.  The
// sum of a group is taken over the whole numbers q - zero in fp32 and scaled
// once a group, the groups are added in fp32, and the result is rounded once.
// A warp computes one output feature for all rows.
#include <cstdio>

#include "common.cuh"
#include "linear_int4.cuh"

namespace aicas {
namespace {

constexpr int kWarps = 8;

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) linear_int4_kernel(const aicas_linear_int4_params p) {
  __shared__ float rstd[AICAS_LINEAR_MAX_ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int K = p.in_features, g = p.group_size;
  const T* nw = static_cast<const T*>(p.norm_weight);
  for (int r = warp; r < p.rows; r += kWarps) {
    const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
    float ss = 0.f;
    if (nw != nullptr)
      for (int k = lane; k < K; k += 32) ss += Elem<T>::to_float(x[k]) * Elem<T>::to_float(x[k]);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    if (lane == 0) rstd[r] = nw != nullptr ? rsqrtf(ss / (float)K + p.eps) : 1.f;
  }
  __syncthreads();
  const int n = blockIdx.x * kWarps + warp;
  if (n >= p.out_features) return;
  const int mats = p.mode == AICAS_LINEAR_SWIGLU ? 2 : 1;
  for (int r0 = 0; r0 < p.rows; r0 += 4) {
    float y[2][4] = {};
    for (int j = 0; j < mats; ++j) {
      const aicas_int4_weight& w = p.w[j];
      const uint8_t* q = static_cast<const uint8_t*>(w.q) + n * w.q_stride;
      for (int i = lane; i < K / 2; i += 32) {
        const int64_t grp = (int64_t)n * (K / g) + 2 * i / g;
        const float z = w.zeros != nullptr ? (float)static_cast<const uint8_t*>(w.zeros)[grp] : 8.f;
        const float sc = Elem<T>::to_float(static_cast<const T*>(w.scales)[grp]);
        const float w0 = (float)(q[i] & 15) - z, w1 = (float)(q[i] >> 4) - z;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (r0 + r >= p.rows) continue;
          const T* x = static_cast<const T*>(p.x) + (r0 + r) * p.x_stride + 2 * i;
          float x0 = Elem<T>::to_float(x[0]), x1 = Elem<T>::to_float(x[1]);
          if (nw != nullptr) {
            x0 = Elem<T>::to_float(Elem<T>::from_float(x0 * rstd[r0 + r] * Elem<T>::to_float(nw[2 * i])));
            x1 = Elem<T>::to_float(Elem<T>::from_float(x1 * rstd[r0 + r] * Elem<T>::to_float(nw[2 * i + 1])));
          }
          y[j][r] += sc * (w0 * x0 + w1 * x1);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) y[j][r] += __shfl_xor_sync(0xffffffffu, y[j][r], off);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (r0 + r >= p.rows || lane != 0) continue;
      float v = y[0][r];
      if (p.mode == AICAS_LINEAR_SWIGLU) v = v / (1.f + __expf(-v)) * y[1][r];
      if (p.mode == AICAS_LINEAR_RESIDUAL)
        v += Elem<T>::to_float(static_cast<const T*>(p.residual)[(r0 + r) * p.residual_stride + n]);
      static_cast<T*>(p.out)[(r0 + r) * p.out_stride + n] = Elem<T>::from_float(v);
    }
  }
}

}  // namespace

int run_linear_int4(const aicas_linear_int4_params* p, int, cudaStream_t stream, unsigned int*, char* err,
                    size_t errlen) {
  const unsigned grid = (unsigned)((p->out_features + kWarps - 1) / kWarps);
  if (p->dtype == AICAS_DTYPE_BF16)
    linear_int4_kernel<__nv_bfloat16><<<grid, kWarps * 32, 0, stream>>>(*p);
  else
    linear_int4_kernel<__half><<<grid, kWarps * 32, 0, stream>>>(*p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    snprintf(err, errlen, "int4 linear launch: %s (%s)", cudaGetErrorString(e), cudaGetErrorName(e));
    return AICAS_ERR_CUDA;
  }
  return AICAS_OK;
}

}  // namespace aicas
