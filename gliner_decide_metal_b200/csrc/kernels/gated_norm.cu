// The norms before and after a transformer block with its gate and residual scale:
//   x' = x + scale * gate * N_post(y),  n = N_pre(x').
//
// One pass over HBM: a row's y and x are read once, held in registers through both norms, and
// x' and n written once (8 bytes a value); n is computed from the unrounded x'. Statistics are
// fp32 and two-pass in registers (the mean first, then the squares of the differences), so a
// row with a large mean loses nothing.
//
// A row belongs to TPR = 32 * 2^w threads of one block, each holding CH chunks of 8 values.
#include "elem.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace gdc {
namespace {

constexpr int kThreads = 256;  // threads of a block when rows take fewer; wide rows take up to 512

// Sum over the TPR threads of a row. red: two halves used in turn, so one barrier a sum is enough.
struct RowSum {
  float* red;
  int tpr, lane, warp_in_row, first_warp;
  int turn = 0;
  __device__ __forceinline__ float operator()(float v) {
    v = ptx::warp_sum(v);
    if (tpr == 32) return v;
    float* r = red + turn * 32;
    turn ^= 1;
    if (lane == 0) r[first_warp + warp_in_row] = v;
    __syncthreads();
    const int n = tpr >> 5;
    float s = 0.f;
    for (int i = 0; i < n; ++i) s += r[first_warp + i];
    return s;
  }
};

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int col, int stride, int cols, float (&v)[8]) {
  using E = ElemOps<T>;
  if (VEC) {
    if (col < cols) {
      const uint4 r = __ldg(reinterpret_cast<const uint4*>(p + col));
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = E::unpack(w[j]);
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = col + j * stride < cols ? E::to_f32(p[col + j * stride]) : 0.f;
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int col, int stride, int cols, const float (&v)[8]) {
  using E = ElemOps<T>;
  if (VEC) {
    if (col < cols)
      *reinterpret_cast<uint4*>(p + col) =
          make_uint4(E::pack(v[0], v[1]), E::pack(v[2], v[3]), E::pack(v[4], v[5]), E::pack(v[6], v[7]));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + j * stride < cols) p[col + j * stride] = E::from_f32(v[j]);
  }
}

// v <- N(v) over the row; columns at or past `cols` are zero and stay out of the sums.
template <typename T, bool VEC, int CH>
__device__ __forceinline__ void normalise(float (&v)[CH][8], int kind, const T* w, const T* b, int col0, int step,
                                          int stride, int cols, float eps, RowSum& sum) {
  float mean = 0.f;
  if (kind == 1) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[c][j];
    mean = sum(s) / float(cols);
  }
  float q = 0.f;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool in = VEC ? col0 + c * step < cols : col0 + c * step + j * stride < cols;
      const float d = v[c][j] - mean;
      q += in ? d * d : 0.f;
    }
  const float inv = rsqrtf(sum(q) / float(cols) + eps);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    float wv[8], bv[8];
    const int col = col0 + c * step;
    if (w != nullptr) load8<T, VEC>(w, col, stride, cols, wv);
    if (b != nullptr) load8<T, VEC>(b, col, stride, cols, bv);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float z = (v[c][j] - mean) * inv;
      if (w != nullptr) z *= wv[j];
      if (b != nullptr) z += bv[j];
      v[c][j] = z;
    }
  }
}

template <typename T, bool VEC, int CH>
__global__ void __launch_bounds__(512)
    gated_norm_kernel(const T* __restrict__ y, const T* x, const T* __restrict__ post_w, const T* __restrict__ post_b,
                      const T* __restrict__ gate, const T* __restrict__ pre_w, const T* __restrict__ pre_b, T* x_out,
                      T* n_out, long long ldy, long long ldx, long long ldxo, long long ldno, long long rows,
                      long long gate_rows, const int32_t* __restrict__ gate_index, const int32_t* __restrict__ rows_dev,
                      int post, int pre, int cols, float scale, float eps, int tpr, int* err) {
  __shared__ float red[64];
  ptx::grid_launch_next();
  ptx::grid_wait();
  const int in_row = threadIdx.x & (tpr - 1);
  const int rows_per_block = blockDim.x / tpr;
  const long long row = (long long)blockIdx.x * rows_per_block + threadIdx.x / tpr;
  const long long n_rows = rows_dev != nullptr ? min(rows, (long long)*rows_dev) : rows;
  bool live = row < n_rows;
  const int col0 = VEC ? in_row * 8 : in_row;
  const int step = tpr * 8, stride = VEC ? 1 : tpr;
  RowSum sum{red, tpr, int(threadIdx.x & 31), in_row >> 5, int(threadIdx.x / tpr) * (tpr >> 5)};

  const T* g = nullptr;
  if (live && gate != nullptr) {
    long long gr = gate_rows == 1 ? 0 : row;
    if (gate_index != nullptr) {
      gr = gate_index[row];
      if (gr < 0 || gr >= gate_rows) {  // uniform over the row's threads
        if (in_row == 0) atomicOr(err, kErrBadGateIndex);
        live = false;
      }
    }
    if (live) g = gate + gr * cols;
  }
  const int my_cols = live ? cols : 0;  // a skipped row takes part in the barriers only
  float xv[CH][8];
#pragma unroll
  for (int c = 0; c < CH; ++c) load8<T, VEC>(x + (live ? row * ldx : 0), col0 + c * step, stride, my_cols, xv[c]);
  if (y != nullptr) {
    float z[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c) load8<T, VEC>(y + (live ? row * ldy : 0), col0 + c * step, stride, my_cols, z[c]);
    if (post != 0) normalise<T, VEC, CH>(z, post, post_w, post_b, col0, step, stride, cols, eps, sum);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (g != nullptr) {
        float gv[8];
        load8<T, VEC>(g, col0 + c * step, stride, my_cols, gv);
#pragma unroll
        for (int j = 0; j < 8; ++j) z[c][j] *= gv[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool in = VEC ? col0 + c * step < my_cols : col0 + c * step + j * stride < my_cols;
        xv[c][j] = in ? fmaf(scale, z[c][j], xv[c][j]) : 0.f;
      }
    }
  }
  if (x_out != nullptr) {
#pragma unroll
    for (int c = 0; c < CH; ++c) store8<T, VEC>(x_out + (live ? row * ldxo : 0), col0 + c * step, stride, my_cols, xv[c]);
  }
  if (pre != 0) {
    normalise<T, VEC, CH>(xv, pre, pre_w, pre_b, col0, step, stride, cols, eps, sum);
#pragma unroll
    for (int c = 0; c < CH; ++c) store8<T, VEC>(n_out + (live ? row * ldno : 0), col0 + c * step, stride, my_cols, xv[c]);
  }
}

bool vec_ok(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, bool VEC, int CH>
gdc_status launch_variant(const GatedNormArgs& a, int tpr, cudaStream_t stream, int* err) {
  const int threads = tpr > kThreads ? tpr : kThreads;
  const int per_block = threads / tpr;
  const long long blocks = (a.rows + per_block - 1) / per_block;
  GDC_CUDA_TRY(launch_overlapped(
      gated_norm_kernel<T, VEC, CH>, unsigned(blocks), unsigned(threads), 0, 1, stream, static_cast<const T*>(a.y),
      static_cast<const T*>(a.x), static_cast<const T*>(a.post_w), static_cast<const T*>(a.post_b), static_cast<const T*>(a.gate),
      static_cast<const T*>(a.pre_w), static_cast<const T*>(a.pre_b), static_cast<T*>(a.x_out), static_cast<T*>(a.n_out), a.ldy, a.ldx,
      a.ldxo, a.ldno, a.rows, a.gate_rows, a.gate_index, a.rows_dev, a.post, a.pre, a.cols, a.scale, a.eps, tpr, err));
  return GDC_OK;
}

template <typename T>
gdc_status launch_typed(const GatedNormArgs& a, cudaStream_t stream, int* err) {
  bool vec = a.cols % 8 == 0 && a.ldy % 8 == 0 && a.ldx % 8 == 0 && a.ldxo % 8 == 0 && a.ldno % 8 == 0;
  const void* all[] = {a.y, a.x, a.post_w, a.post_b, a.gate, a.pre_w, a.pre_b, a.x_out, a.n_out};
  for (const void* p : all) vec = vec && vec_ok(p);
  // 16 values a thread up to 512 threads a row, then 32
  int tpr = 32;
  while (tpr < 512 && tpr * 16 < a.cols) tpr *= 2;
  const int ch = (a.cols + tpr * 8 - 1) / (tpr * 8);
  if (ch <= 1) return vec ? launch_variant<T, true, 1>(a, tpr, stream, err) : launch_variant<T, false, 1>(a, tpr, stream, err);
  if (ch <= 2) return vec ? launch_variant<T, true, 2>(a, tpr, stream, err) : launch_variant<T, false, 2>(a, tpr, stream, err);
  return vec ? launch_variant<T, true, 4>(a, tpr, stream, err) : launch_variant<T, false, 4>(a, tpr, stream, err);
}

}  // namespace

gdc_status launch_gated_residual_norm(Elem t, const GatedNormArgs& a, cudaStream_t stream, int* err) {
  return t == Elem::kF16 ? launch_typed<__half>(a, stream, err) : launch_typed<__nv_bfloat16>(a, stream, err);
}

}  // namespace gdc
