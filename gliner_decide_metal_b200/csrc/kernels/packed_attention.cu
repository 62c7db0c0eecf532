// Softmax attention with grouped heads over packed sequences: one warp per query row and head,
// online softmax in fp32 on CUDA cores.
#include "elem.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace gdc {
namespace {

// Index of the sequence that holds `row`: the last b with off[b] <= row among those whose rows
// [off[b], off[b+1]) are valid. -1: none.
__device__ __forceinline__ int find_sequence(const int32_t* off, int batch, int row) {
  for (int b = 0; b < batch; ++b)
    if (off[b] <= row && row < off[b + 1]) return b;
  return -1;
}

template <typename T, int D>
__global__ void __launch_bounds__(128)
    packed_attention_rows_kernel(PackedAttentionArgs a, int* err) {
  using E = ElemOps<T>;
  constexpr int PER = D / 32;
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int row = int(item / a.heads), h = int(item % a.heads);
  if (item < a.batch && lane == 0) {  // sequences without a row of their own are checked too
    const int b = int(item);
    if (a.q_off[b] > a.q_off[b + 1] || a.k_off[b] > a.k_off[b + 1]) atomicOr(err, kErrBadOffsets);
  }
  if (row >= a.q_rows) return;
  const int b = find_sequence(a.q_off, a.batch, row);
  if (b < 0) return;
  const int q0 = a.q_off[b], q1 = a.q_off[b + 1], k0 = a.k_off[b], k1 = a.k_off[b + 1];
  if (q0 < 0 || q1 > a.q_rows || k0 < 0 || k1 < k0 || k1 > a.k_rows) {
    if (lane == 0) atomicOr(err, kErrBadOffsets);
    return;
  }
  const int seen = a.causal ? max(0, min(k1 - k0, row - q1 + 1 + (k1 - k0))) : k1 - k0;
  const T* q = static_cast<const T*>(a.q) + (long long)row * a.ldq + h * D + lane * PER;
  const int hk = h / (a.heads / a.kv_heads);
  const T* k = static_cast<const T*>(a.k) + (long long)k0 * a.ldk + hk * D + lane * PER;
  const T* v = static_cast<const T*>(a.v) + (long long)k0 * a.ldv + hk * D + lane * PER;
  float qv[PER], o[PER] = {}, m = -INFINITY, l = 0.f;
  for (int i = 0; i < PER; ++i) qv[i] = E::to_f32(q[i]) * a.scale;
  for (int j = 0; j < seen; ++j) {
    float s = 0.f;
    for (int i = 0; i < PER; ++i) s = fmaf(qv[i], E::to_f32(k[(long long)j * a.ldk + i]), s);
    s = ptx::warp_sum(s);
    const float mn = fmaxf(m, s);
    const float r = m == mn ? 1.f : expf(m - mn), p = expf(s - mn);
    l = l * r + p;
    for (int i = 0; i < PER; ++i) o[i] = o[i] * r + p * E::to_f32(v[(long long)j * a.ldv + i]);
    m = mn;
  }
  T* out = static_cast<T*>(a.out) + (long long)row * a.ldo + h * D + lane * PER;
  for (int i = 0; i < PER; ++i) out[i] = E::from_f32(seen > 0 ? o[i] / l : 0.f);
}

}  // namespace

size_t packed_attention_workspace(int, int64_t, int64_t, int, int, int) { return 256; }

gdc_status launch_packed_attention(Elem t, const PackedAttentionArgs& a, cudaStream_t stream, int* err) {
  const int64_t items = a.q_rows * a.heads > a.batch ? a.q_rows * a.heads : a.batch;
  const unsigned blocks = unsigned((items + 3) / 4);
  if (t == Elem::kF16) {
    if (a.dim == 64) packed_attention_rows_kernel<__half, 64><<<blocks, 128, 0, stream>>>(a, err);
    else packed_attention_rows_kernel<__half, 128><<<blocks, 128, 0, stream>>>(a, err);
  } else {
    if (a.dim == 64) packed_attention_rows_kernel<__nv_bfloat16, 64><<<blocks, 128, 0, stream>>>(a, err);
    else packed_attention_rows_kernel<__nv_bfloat16, 128><<<blocks, 128, 0, stream>>>(a, err);
  }
  return check_launch("packed_attention_rows_kernel");
}

}  // namespace gdc
