// out = residual + act(a . w^T + bias): tiled on CUDA cores, fp32 sums.
#include "elem.cuh"
#include "kernels.h"

namespace gdc {
namespace {

constexpr int kTile = 64, kStep = 16;

__device__ __forceinline__ float activate(float z, int act) {
  if (act == kActGelu) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  if (act == kActRelu) return z > 0.f ? z : (z != z ? z : 0.f);
  if (act == kActSilu) return z / (1.f + expf(-z));
  return z;
}

template <typename T>
__global__ void __launch_bounds__(256)
    linear_residual_kernel(const T* __restrict__ a, const T* __restrict__ w, const T* __restrict__ bias, const T* residual,
                           T* out, long long lda, long long ldw, long long ldr, long long ldo, long long m_cap,
                           const int32_t* __restrict__ rows_dev, int N, int K, int act) {
  using E = ElemOps<T>;
  __shared__ float sa[kStep][kTile + 1], sw[kStep][kTile + 1];
  const long long M = rows_dev != nullptr ? min(m_cap, (long long)*rows_dev) : m_cap;
  const long long m0 = (long long)blockIdx.x * kTile;
  const int n0 = blockIdx.y * kTile;
  if (m0 >= M) return;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += kStep) {
    for (int i = threadIdx.x; i < kTile * kStep; i += 256) {
      const int r = i / kStep, k = i % kStep;
      sa[k][r] = m0 + r < M && k0 + k < K ? E::to_f32(a[(m0 + r) * lda + k0 + k]) : 0.f;
      sw[k][r] = n0 + r < N && k0 + k < K ? E::to_f32(w[(long long)(n0 + r) * ldw + k0 + k]) : 0.f;
    }
    __syncthreads();
    for (int k = 0; k < kStep; ++k)
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty + 16 * i], sw[k][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const long long m = m0 + ty + 16 * i;
      const int n = n0 + tx + 16 * j;
      if (m >= M || n >= N) continue;
      float z = activate(acc[i][j] + (bias != nullptr ? E::to_f32(bias[n]) : 0.f), act);
      if (residual != nullptr) z += E::to_f32(residual[m * ldr + n]);
      out[m * ldo + n] = E::from_f32(z);
    }
}

template <typename T>
gdc_status launch_typed(const LinearResidualArgs& p, cudaStream_t stream) {
  const dim3 grid(unsigned((p.M + kTile - 1) / kTile), unsigned((p.N + kTile - 1) / kTile));
  if (grid.y > 65535) return set_error(GDC_ERR_UNSUPPORTED, "gdc_linear_residual: N=%d too large", p.N);
  linear_residual_kernel<T><<<grid, 256, 0, stream>>>(
      static_cast<const T*>(p.a), static_cast<const T*>(p.w), static_cast<const T*>(p.bias),
      static_cast<const T*>(p.residual), static_cast<T*>(p.out), p.lda, p.ldw, p.ldr, p.ldo, p.M, p.rows_dev, p.N, p.K,
      p.act);
  return check_launch("linear_residual_kernel");
}

}  // namespace

gdc_status launch_linear_residual(Elem t, const LinearResidualArgs& a, cudaStream_t stream, int*) {
  return t == Elem::kF16 ? launch_typed<__half>(a, stream) : launch_typed<__nv_bfloat16>(a, stream);
}

}  // namespace gdc
