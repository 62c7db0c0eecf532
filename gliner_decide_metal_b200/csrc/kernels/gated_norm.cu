// The norms before and after a transformer block with its gate and residual scale:
//   x' = x + scale * gate * N_post(y),  n = N_pre(x').
//
// One pass over HBM: a row's y and x are read once, held in registers through both norms, and
// x' and n written once (8 bytes a value); n is computed from the unrounded x'. Statistics are
// fp32 and two-pass in registers (the mean first, then the squares of the differences), so a
// row with a large mean loses nothing.
//
// What bounds it is bytes in flight: the sums are a chain of up to four reductions a row. So the
// grid is persistent and every thread has its values of the next row on their way to its own
// slots of shared memory (cp.async; no other thread reads them, so nothing is synchronised) while
// it works on this one, and a row belongs to few threads: one warp up to 512
// columns (reductions without a barrier, four rows a block), one block of 64 to 512 threads above.
// Weights and gate rows are read again for every row, from L1, by plain loads: the kernel may be resident while
// the one before it writes them, so they are not read-only for its lifetime. Rows at odd 2-byte addresses are read
// value by value when their turn comes.
//
// On a B200, two norms and a gate (8 bytes a value), captured back to back: 16384 x 4096 RMSNorm 90 to 94 us, 5.7 to
// 6.0 TB/s (0.87 to 0.91 of a plain copy; its instructions are next, 0.68 issued a cycle; 97 us one C call after another),
// LayerNorm 107 us (one reduction more a norm); 4885 x 1024 LayerNorm 10 to 13 us, 3.2 TB/s at most from HBM (two
// rows a block in all: start and chain of reductions); 16384 x 4095, value by value, 187 us (these variants also spill
// up to 236 bytes a thread at 64 registers).
#include <algorithm>

#include "elem.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace gdc {
namespace {

struct NormParams {
  const void *y, *x, *post_w, *post_b, *gate, *pre_w, *pre_b;
  void *x_out, *n_out;
  long long ldy, ldx, ldxo, ldno, rows, gate_rows;
  const int32_t *gate_index, *rows_dev;
  int post, pre, cols;
  float scale, eps;
  int* err;
};

// Values of one thread: N of them in chunks of V neighbours (8: 16-byte accesses, 2: 4-byte, 1),
// chunk c at columns (c * TPR + thread) * V. Raw 16-bit pairs.
template <typename T, int V, int N>
struct Values {
  static constexpr int kWords = V == 1 ? N : N / 2;
  uint32_t w[kWords];

  template <bool STREAM>
  __device__ __forceinline__ void load(const T* p, int first, int step, int cols) {
#pragma unroll
    for (int c = 0; c < N / V; ++c) {
      const int col = first + c * step;
      if (V == 8) {
        uint4 r = make_uint4(0u, 0u, 0u, 0u);
        if (col < cols) r = STREAM ? __ldcs(reinterpret_cast<const uint4*>(p + col)) : *reinterpret_cast<const uint4*>(p + col);
        w[c * 4 % kWords] = r.x;
        w[(c * 4 + 1) % kWords] = r.y;
        w[(c * 4 + 2) % kWords] = r.z;
        w[(c * 4 + 3) % kWords] = r.w;
      } else if (V == 2) {
        const uint32_t* q = reinterpret_cast<const uint32_t*>(p + col);
        w[c % kWords] = col < cols ? (STREAM ? __ldcs(q) : *q) : 0u;
      } else {
        const uint16_t* q = reinterpret_cast<const uint16_t*>(p + col);
        w[c % kWords] = col < cols ? uint32_t(STREAM ? __ldcs(q) : *q) : 0u;
      }
    }
  }
  // The same through shared memory: chunk c of this thread at slot + c * threads * 2 V bytes.
  static constexpr int kChunkBytes = 2 * V;
  static __device__ __forceinline__ void fetch(uint32_t slot, const T* p, int first, int step, int cols) {
#pragma unroll
    for (int c = 0; c < N / V; ++c) {
      const int col = first + c * step;
      const uint32_t dst = slot + c * blockDim.x * kChunkBytes;
      const int bytes = col < cols ? kChunkBytes : 0;  // nothing read, the slot zeroed, behind the row's end
      const T* src = p + (col < cols ? col : 0);
      if (V == 8)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
      else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    }
  }
  __device__ __forceinline__ void take(uint32_t slot) {
#pragma unroll
    for (int c = 0; c < N / V; ++c) {
      const uint32_t src = slot + c * blockDim.x * kChunkBytes;
      if (V == 8)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[c * 4 % kWords]), "=r"(w[(c * 4 + 1) % kWords]), "=r"(w[(c * 4 + 2) % kWords]), "=r"(w[(c * 4 + 3) % kWords])
                     : "r"(src)
                     : "memory");
      else
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[c % kWords]) : "r"(src) : "memory");
    }
  }
  __device__ __forceinline__ float2 pair(int i) const {  // values 2 i, 2 i + 1
    if (V == 1) return make_float2(one(2 * i), one(2 * i + 1));
    return ElemOps<T>::unpack(w[i % kWords]);
  }
  __device__ __forceinline__ float one(int i) const {
    const uint16_t h = uint16_t(w[i % kWords]);
    return ElemOps<T>::to_f32(*reinterpret_cast<const T*>(&h));
  }
};

template <typename T, int V, int N>
__device__ __forceinline__ void store(T* p, const float (&v)[N], int first, int step, int cols) {
  using E = ElemOps<T>;
#pragma unroll
  for (int c = 0; c < N / V; ++c) {
    const int col = first + c * step;
    if (col >= cols) continue;
    const float* f = v + c * V;
    if (V == 8)
      __stcs(reinterpret_cast<uint4*>(p + col), make_uint4(E::pack(f[0], f[1 % V]), E::pack(f[2 % V], f[3 % V]), E::pack(f[4 % V], f[5 % V]),
                                                           E::pack(f[6 % V], f[7 % V])));
    else if (V == 2)
      __stcs(reinterpret_cast<uint32_t*>(p + col), E::pack(f[0], f[1 % V]));
    else
      p[col] = E::from_f32(f[0]);
  }
}

// Sum over the TPR threads of a row; red has two halves used in turn, so one barrier a sum is enough.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red, int& turn) {
  v = ptx::warp_sum(v);
  if (TPR == 32) return v;
  float* r = red + turn * 16;
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < TPR / 32; ++i) s += r[i];
  return s;
}

// v <- N(v); values at or past `cols` stay out of the sums.
template <typename T, int V, int N, int TPR>
__device__ __forceinline__ void normalise(float (&v)[N], int kind, const T* w, const T* b, int first, int step, int cols, float inv_cols,
                                          float eps, float* red, int& turn) {
  float mean = 0.f;
  if (kind == 1) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < N / V; ++c)
      if (first + c * step < cols) {
#pragma unroll
        for (int j = 0; j < V; ++j) s += v[c * V + j];
      }
    mean = row_sum<TPR>(s, red, turn) * inv_cols;
  }
  float q = 0.f;
#pragma unroll
  for (int c = 0; c < N / V; ++c)
    if (first + c * step < cols) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = v[c * V + j] - mean;
        q = fmaf(d, d, q);
      }
    }
  const float inv = rsqrtf(row_sum<TPR>(q, red, turn) * inv_cols + eps);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = (v[i] - mean) * inv;
  if (w != nullptr) {
    Values<T, V, N> wv;
    wv.template load<false>(w, first, step, cols);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 a = wv.pair(i);
      v[2 * i] *= a.x;
      v[2 * i + 1] *= a.y;
    }
  }
  if (b != nullptr) {
    Values<T, V, N> bv;
    bv.template load<false>(b, first, step, cols);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 a = bv.pair(i);
      v[2 * i] += a.x;
      v[2 * i + 1] += a.y;
    }
  }
}

constexpr int kStages = 2;  // rows of a thread in shared memory: the current one and the next (a third costs the weights their L1)

template <int V, int N, int TPR>
struct NormShape {
  static constexpr int kThreads = TPR == 32 ? 128 : TPR, kRows = TPR == 32 ? 4 : 1;  // rows a block holds at once
  static constexpr bool kAsync = V > 1;
  static constexpr int kRowBytes = kThreads * N * 2;  // one tensor of the block's rows
  static constexpr int kSmemBytes = kAsync ? kStages * 2 * kRowBytes : 0;
  static constexpr int kBlocks = N == 32 ? (TPR <= 128 ? 4 : TPR == 256 ? 2 : 1) : 1024 / kThreads;  // resident on an SM
};

template <typename T, int V, int N, int TPR>
__global__ void __launch_bounds__(NormShape<V, N, TPR>::kThreads, NormShape<V, N, TPR>::kBlocks) gated_norm_kernel(const NormParams p) {
  using S = NormShape<V, N, TPR>;
  __shared__ float red[32];
  extern __shared__ __align__(16) uint8_t slots[];
  ptx::grid_launch_next();
  ptx::grid_wait();
  const int in_row = TPR == 32 ? int(threadIdx.x & 31) : int(threadIdx.x);
  const int first = in_row * V, step = TPR * V, cols = p.cols;
  const float inv_cols = 1.f / float(cols);
  const T *y = static_cast<const T*>(p.y), *x = static_cast<const T*>(p.x);
  const long long n_rows = p.rows_dev != nullptr ? min(p.rows, (long long)*p.rows_dev) : p.rows;
  const long long stride = (long long)gridDim.x * S::kRows;
  long long row = (long long)blockIdx.x * S::kRows + (TPR == 32 ? threadIdx.x >> 5 : 0);
  const uint32_t my_slot = ptx::smem_u32(slots) + threadIdx.x * Values<T, V, N>::kChunkBytes;
  int turn = 0, stage = 0;
  auto fetch = [&](long long r, int s) {
    if (r < n_rows) {
      Values<T, V, N>::fetch(my_slot + (2 * s) * S::kRowBytes, x + r * p.ldx, first, step, cols);
      if (y != nullptr) Values<T, V, N>::fetch(my_slot + (2 * s + 1) * S::kRowBytes, y + r * p.ldy, first, step, cols);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (S::kAsync)
    for (int s = 0; s < kStages - 1; ++s) fetch(row + s * stride, s);
  for (; row < n_rows; row += stride) {  // (uniform over the threads of a row, which share its barriers)
    long long g_row = p.gate_rows == 1 ? 0 : row;
    if (p.gate_index != nullptr) g_row = p.gate_index[row];
    float xv[N], z[N];
    {
      Values<T, V, N> xr, yr;
      if (S::kAsync) {
        int ahead = stage + kStages - 1;
        if (ahead >= kStages) ahead -= kStages;
        fetch(row + (kStages - 1) * stride, ahead);
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        xr.take(my_slot + (2 * stage) * S::kRowBytes);
        if (y != nullptr) yr.take(my_slot + (2 * stage + 1) * S::kRowBytes);
        if (++stage == kStages) stage = 0;
      } else {
        xr.template load<true>(x + row * p.ldx, first, step, cols);
        if (y != nullptr) yr.template load<true>(y + row * p.ldy, first, step, cols);
      }
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float2 a = xr.pair(i);
        xv[2 * i] = a.x;
        xv[2 * i + 1] = a.y;
        if (y != nullptr) {
          const float2 b = yr.pair(i);
          z[2 * i] = b.x;
          z[2 * i + 1] = b.y;
        }
      }
    }
    if (p.gate_index != nullptr && (g_row < 0 || g_row >= p.gate_rows)) {
      if (in_row == 0) atomicOr(p.err, kErrBadGateIndex);
      continue;
    }
    if (y != nullptr) {
      if (p.post != 0)
        normalise<T, V, N, TPR>(z, p.post, static_cast<const T*>(p.post_w), static_cast<const T*>(p.post_b), first, step, cols, inv_cols,
                                p.eps, red, turn);
      if (p.gate != nullptr) {
        Values<T, V, N> gv;
        gv.template load<false>(static_cast<const T*>(p.gate) + g_row * cols, first, step, cols);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          const float2 a = gv.pair(i);
          z[2 * i] *= a.x;
          z[2 * i + 1] *= a.y;
        }
      }
#pragma unroll
      for (int i = 0; i < N; ++i) xv[i] = fmaf(p.scale, z[i], xv[i]);
    }
    if (p.x_out != nullptr) store<T, V, N>(static_cast<T*>(p.x_out) + row * p.ldxo, xv, first, step, cols);
    if (p.pre != 0) {
      normalise<T, V, N, TPR>(xv, p.pre, static_cast<const T*>(p.pre_w), static_cast<const T*>(p.pre_b), first, step, cols, inv_cols, p.eps,
                              red, turn);
      store<T, V, N>(static_cast<T*>(p.n_out) + row * p.ldno, xv, first, step, cols);
    }
  }
  if (S::kAsync) asm volatile("cp.async.wait_group 0;" ::: "memory");  // (empty groups only)
}

template <typename T, int V, int N, int TPR>
gdc_status launch_variant(const NormParams& p, cudaStream_t stream) {
  using S = NormShape<V, N, TPR>;
  auto kern = gated_norm_kernel<T, V, N, TPR>;
  static PerDeviceOnce resident;  // blocks the device holds at once
  int dev = 0;
  GDC_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return set_error(GDC_ERR_CUDA, "device ordinal out of range");
  const int most = per_device_once(resident, dev, [&] {
    int b = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmemBytes) != cudaSuccess) return 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&b, kern, S::kThreads, S::kSmemBytes) != cudaSuccess) return 0;
    return b * device_sm_count(dev);
  });
  if (most < 1) return set_error(GDC_ERR_CUDA, "gated residual norm: no block fits on device %d", dev);
  const long long blocks = std::min<long long>((p.rows + S::kRows - 1) / S::kRows, most);
  GDC_CUDA_TRY(launch_overlapped(kern, unsigned(blocks), unsigned(S::kThreads), S::kSmemBytes, 1, stream, p));
  return GDC_OK;
}

template <typename T, int V>
gdc_status launch_width(const NormParams& p, cudaStream_t stream) {
  // Values a thread and threads a row, measured: 16 x 64 against 32 x 32 at 1024 columns (16384 rows:
  // 25.4 against 26.1 us; one row: 3.2 against 3.7; single values 8 x 128: 42 against 55), 32 x 128
  // against 16 x 256 at 4096 (two LayerNorms over 16384 rows: 108 against 118 us).
  const int c = p.cols;
  if (c <= 256) return launch_variant<T, V, 8, 32>(p, stream);
  if (c <= 512) return launch_variant<T, V, 16, 32>(p, stream);
  if (c <= 1024) return V == 1 ? launch_variant<T, V, 8, 128>(p, stream) : launch_variant<T, V, 16, 64>(p, stream);
  if (c <= 2048) return launch_variant<T, V, 16, 128>(p, stream);
  if (c <= 4096) return launch_variant<T, V, 32, 128>(p, stream);
  if (c <= 8192) return launch_variant<T, V, 16, 512>(p, stream);
  return launch_variant<T, V, 32, 512>(p, stream);
}

template <typename T>
gdc_status launch_typed(const GatedNormArgs& a, cudaStream_t stream, int* err) {
  const NormParams p{a.y, a.x, a.post_w, a.post_b, a.gate, a.pre_w, a.pre_b, a.x_out, a.n_out, a.ldy, a.ldx, a.ldxo, a.ldno, a.rows,
                     a.gate_rows, a.gate_index, a.rows_dev, a.post, a.pre, a.cols, a.scale, a.eps, err};
  // the widest access that every row of every tensor is aligned to
  uintptr_t bits = uintptr_t(a.cols) * 2;
  for (const void* q : {a.y, a.x, a.post_w, a.post_b, a.gate, a.pre_w, a.pre_b, (const void*)a.x_out, (const void*)a.n_out})
    bits |= reinterpret_cast<uintptr_t>(q);
  bits |= uintptr_t(a.ldx) * 2;
  if (a.y != nullptr) bits |= uintptr_t(a.ldy) * 2;
  if (a.x_out != nullptr) bits |= uintptr_t(a.ldxo) * 2;
  if (a.n_out != nullptr) bits |= uintptr_t(a.ldno) * 2;
  if (bits % 16 == 0) return launch_width<T, 8>(p, stream);
  if (bits % 4 == 0) return launch_width<T, 2>(p, stream);
  return launch_width<T, 1>(p, stream);
}

}  // namespace

gdc_status launch_gated_residual_norm(Elem t, const GatedNormArgs& a, cudaStream_t stream, int* err) {
  return t == Elem::kF16 ? launch_typed<__half>(a, stream, err) : launch_typed<__nv_bfloat16>(a, stream, err);
}

}  // namespace gdc
