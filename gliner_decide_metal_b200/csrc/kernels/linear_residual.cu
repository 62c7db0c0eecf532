// out = residual + act(a . w^T + bias) on tcgen05 tensor cores, any M, N and K.
//
// The product is computed transposed: the MMA's 128 rows are weight rows (output columns n) and
// its N dimension is `bt` rows of a (m), chosen per call: a multiple of 16 up to 256, or one of 32 up
// to 512 as two MMAs side by side. So
//   * few rows of a cost a narrow MMA (bt = 16 for a single token) while the weights, which are
//     then all the traffic, stream through the wide operand;
//   * in the epilogue a thread owns one n (its bias is one register) and walks over m: a warp
//     reads residuals and writes results 32 neighbouring n at a time, 64 bytes a row, at any
//     alignment, pitch and width, and a row count only the device knows limits a loop.
//
// Two forms, one kernel:
//   PAIR    two CTAs (cta_group::2) make a 256 (n) x bt (m) tile: each loads its 128 weight rows
//           and half of the a rows, the leader issues the MMAs for both. Persistent; up to bt = 256
//           two accumulators in TMEM, so a tile's epilogue runs beside the next tile's products.
//   single  a CTA makes a 128 x bt tile; where tiles are fewer than SMs, a cluster of 2, 4 or 8 CTAs
//           splits K, and each sums its share of the columns from all of them, in rank order,
//           through distributed shared memory.
//
// Roles: warp 0 TMA (128-column K blocks of w and a into a ring), warp 1 MMA issue, warps 2-17
// epilogue (TMEM lane quarter warp % 4; the four warps of a quarter take 16-column chunks in turn).
// An epilogue warp has the residuals of its first three 16-column chunks (48 rows, 64 bytes each) on
// their way before it waits for the accumulators, and those of three chunks ahead from then on.
// Sums are fp32 over K in order (K split: in order inside a share, shares in rank order): the
// same call gives the same bits.
//
// What bounds it, and what it reaches on a B200 (bias and residual included, fp16; 20 calls captured in a graph, their
// tensors in turn out of 400 MB; in brackets a library's product alone the same way; "in calls": one
// C call after another, where the clock is the power cap's):
//   8192 x 8192 x 4096 (M, N, K), GELU   the tensor cores: 390 to 405 us, 1360 to 1410 TFLOP/s (393 to 416); in calls
//                      440 to 468, 1170 to 1250 TFLOP/s
//   4885 x 1024 x 4096 136 of 148 SMs in one round of 288-row tiles, its start and its epilogue not
//                      overlapped: 34 us, 1190 TFLOP/s (31); in calls 41
//   4885 x 4096 x 1024, GELU   epilogues, 8 K blocks a tile long: 51 us, 796 TFLOP/s (35); bf16 4% less
//   64 x 4096 x 4096, SiLU     operand tiles arriving: 14 us, 2.5 TB/s (9.7)
//   1 x 4096 x 4096    weights streaming: 10.8 us, 3.1 TB/s (11.8)
// Tried and slower: 64-column K blocks (406 -> 575 us on the first), prefetching weights to L2 (15.4 ->
// 17.5 us for 64 rows); polling waits and one TMA box an operand made no difference.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "elem.cuh"
#include "gelu.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace gdc {

PFN_cuTensorMapEncodeTiled_v12000 get_encode_fn();

namespace {

constexpr int kBK = 128;         // K columns of a stage: two 128-byte swizzle atoms an operand
constexpr int kEpiWarps = 16;    // four a TMEM lane quarter, each every fourth 16-column chunk
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kMaxStages = 6;
constexpr int kWBytes = 128 * kBK * 2;
constexpr int kRingBytes = 225 * 1024, kSplitRing = 192 * 1024;  // (split K keeps partial sums beside the ring)
constexpr int kMaxSplitBt = 64;  // split K: columns x 128 lanes x 4 bytes of partial sums, 32 KB
constexpr int kCtrlBytes = 256;
constexpr int kMaxSmem = kRingBytes + kCtrlBytes + 1024;
static_assert(kSplitRing + kMaxSplitBt * 512 <= kRingBytes && kMaxSmem <= 232448, "shared memory of a CTA");

struct LinearParams {
  const void *bias, *residual;
  void* out;
  long long ldr, ldo, m_cap;
  const int32_t* rows_dev;
  int N, K, bt, subs, split, stages, stage_bytes;  // subs: MMAs side by side in a tile
  int acc_cols, tmem_cols;  // TMEM columns between accumulators, and in all
  int* err;
};

// Tile t of num_n x num_m: groups of 8 n tiles, so that the tiles in flight share both operands.
__device__ __forceinline__ void tile_at(long long t, int num_n, int num_m, int& nb, int& mb) {
  const long long per_group = 8ll * num_m;
  const int g = int(t / per_group);
  const int width = min(8, num_n - g * 8);
  const int u = int(t - g * per_group);
  nb = g * 8 + u % width;
  mb = u / width;
}

// The activation of two values (rows m, m + 1 of one n).
template <typename T, int ACT>
__device__ __forceinline__ float2 activate(float2 z) {
  if (ACT == kActGelu) {
    const float2 g = ElemOps<T>::kMmaFormat == 1 ? gelu_erf2_wide(z) : gelu_erf2(z);
    return make_float2(z.x > 16.f ? z.x : g.x, z.y > 16.f ? z.y : g.y);  // GELU(x) = x there; keeps +inf
  }
  if (ACT == kActRelu) {
    asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(z.x));
    asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(z.y));
  }
  if (ACT == kActSilu)
    return make_float2(__fdividef(z.x, 1.f + ex2_approx_f32(-kGeluLog2e * z.x)),
                       __fdividef(z.y, 1.f + ex2_approx_f32(-kGeluLog2e * z.y)));
  return z;
}

// Column n of the outputs: rows are fetched and stored 16 at a time.
template <typename T, int ACT>
struct Column {
  using E = ElemOps<T>;
  const T* res;
  T* out;
  long long ldr, ldo, M;
  float bias;
  // residuals of rows m0 .. m0 + 15 (those outside the matrix stay unset)
  __device__ __forceinline__ void fetch(long long m0, uint16_t (&r)[16]) const {
    const uint16_t* src = reinterpret_cast<const uint16_t*>(res) + m0 * ldr;
    if (m0 + 16 <= M) {
#pragma unroll
      for (int i = 0; i < 16; ++i, src += ldr) r[i] = *src;
    } else {
      const int rows = int(max(0ll, M - m0));
#pragma unroll
      for (int i = 0; i < 16; ++i, src += ldr)
        if (i < rows) r[i] = *src;
    }
  }
  __device__ __forceinline__ void store(long long m0, const uint32_t (&z)[16], const uint16_t (&r)[16]) const {
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float2 x = activate<T, ACT>(__fadd2_rn(make_float2(__uint_as_float(z[i]), __uint_as_float(z[i + 1])), make_float2(bias, bias)));
      v[i] = x.x;
      v[i + 1] = x.y;
    }
    if (res != nullptr) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] += E::to_f32(*reinterpret_cast<const T*>(&r[i]));
    }
    T* dst = out + m0 * ldo;
    if (m0 + 16 <= M) {
#pragma unroll
      for (int i = 0; i < 16; ++i, dst += ldo) *dst = E::from_f32(v[i]);
    } else {
      const int rows = int(max(0ll, M - m0));
#pragma unroll
      for (int i = 0; i < 16; ++i, dst += ldo)
        if (i < rows) *dst = E::from_f32(v[i]);
    }
  }
};

template <typename T, bool PAIR, int ACT>
__global__ void __launch_bounds__(kThreads, 1)
    linear_residual_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a, const LinearParams p) {
  using E = ElemOps<T>;
  const int warp = ptx::warp_index(), lane = threadIdx.x & 31;
  ptx::grid_launch_next();
  if (threadIdx.x == 0) {
    ptx::prefetch_tensor_map(&tm_w);
    ptx::prefetch_tensor_map(&tm_a);
  }
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + p.stages * p.stage_bytes);
  float* red = reinterpret_cast<float*>(ring + p.stages * p.stage_bytes + kCtrlBytes);
  uint64_t* empty = full + kMaxStages;
  uint64_t* tfull = empty + kMaxStages;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  const bool clustered = PAIR || p.split > 1;
  const uint32_t rank = clustered ? ptx::cluster_ctarank() : 0;
  const bool leader = !PAIR || rank == 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      ptx::mbar_init(&full[s], 1);
      ptx::mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(&tfull[a], 1);
      ptx::mbar_init(&tempty[a], (PAIR ? 2 : 1) * kEpiWarps);
    }
    ptx::mbar_init(drain, 1);
    ptx::fence_barrier_init();
  }
  if (warp == 1) {
    if (PAIR) {
      ptx::tmem_alloc_pair(tmem_slot, p.tmem_cols);
      ptx::tmem_relinquish_pair();
    } else {
      ptx::tmem_alloc(tmem_slot, p.tmem_cols);
      ptx::tmem_relinquish();
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (clustered) ptx::cluster_sync();  // every barrier is initialised before a peer signals or writes
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  ptx::grid_wait();

  const long long M = p.rows_dev != nullptr ? min(p.m_cap, (long long)*p.rows_dev) : p.m_cap;
  const int bt = p.bt;
  const int num_m = M > 0 ? int((M + bt - 1) / bt) : 0;
  constexpr int kTileN = PAIR ? 256 : 128;
  const int num_n = (p.N + kTileN - 1) / kTileN;
  const long long tiles = (long long)num_m * num_n;
  const int share = PAIR ? 2 : p.split;  // CTAs that work on one tile
  const long long first = blockIdx.x / share, stride = gridDim.x / share;
  // this CTA's K blocks
  const int kblocks = (p.K + kBK - 1) / kBK;
  const int kb0 = PAIR ? 0 : int((long long)kblocks * rank / p.split);
  const int kb1 = PAIR ? kblocks : int((long long)kblocks * (rank + 1) / p.split);
  const int a_rows = PAIR ? bt / 2 : bt;  // rows of a this CTA loads
  const int sub_rows = a_rows / p.subs, a_atom = sub_rows * 128, sub_bytes = 2 * a_atom;  // [sub][atom][rows][64]

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      long long issued = 0;
      bool ok = true;
      const uint32_t tx = uint32_t(PAIR ? 2 : 1) * uint32_t(kWBytes + p.subs * sub_bytes);
      for (long long t = first; t < tiles && ok; t += stride) {
        int nb, mb;
        tile_at(t, num_n, num_m, nb, mb);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = ptx::mbar_wait(&empty[stage], phase ^ 1u, p.err))) break;
          uint8_t* s_w = ring + stage * p.stage_bytes;
          uint8_t* s_a = s_w + kWBytes;
          const int n0 = nb * kTileN + int(PAIR ? rank * 128 : 0), m0 = mb * bt + int(PAIR ? rank * sub_rows : 0);
          if (PAIR) {
            const uint32_t bar = ptx::mapa_shared(ptx::smem_u32(&full[stage]), 0);
            if (leader) ptx::mbar_arrive_expect_tx(&full[stage], tx);
            for (int u = 0; u < 2; ++u) {
              ptx::tma_load_2d_pair(s_w + u * 16384, &tm_w, kb * kBK + u * 64, n0, bar);
              for (int h = 0; h < p.subs; ++h)
                ptx::tma_load_2d_pair(s_a + h * sub_bytes + u * a_atom, &tm_a, kb * kBK + u * 64, m0 + h * 2 * sub_rows, bar);
            }
          } else {
            ptx::mbar_arrive_expect_tx(&full[stage], tx);
            for (int u = 0; u < 2; ++u) {
              ptx::tma_load_2d(s_w + u * 16384, &tm_w, kb * kBK + u * 64, n0, &full[stage]);
              for (int h = 0; h < p.subs; ++h)
                ptx::tma_load_2d(s_a + h * sub_bytes + u * a_atom, &tm_a, kb * kBK + u * 64, m0 + h * sub_rows, &full[stage]);
            }
          }
          ++issued;
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // Every slot's last load has landed and been consumed ("empty" again) before the CTA can exit
      // (bounded; in a pair this is also what keeps the leader's reads of this CTA's slots valid).
      for (long long j = std::max(0ll, issued - p.stages); j < issued; ++j) {
        uint64_t* bar = &empty[j % p.stages];
        const uint32_t parity = uint32_t((j / p.stages) & 1);
        const unsigned long long t0 = ptx::globaltimer();
        while (!ptx::mbar_try_wait(bar, parity) && ptx::globaltimer() - t0 < ptx::kTimeoutNs) {
        }
      }
    }
  } else if (warp == 1) {
    if (leader) {
      const uint32_t idesc =
          ptx::idesc_f16_f32(PAIR ? 256 : 128, uint32_t(bt / p.subs)) | (E::kMmaFormat << 7) | (E::kMmaFormat << 10);
      int stage = 0, local = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (long long t = first; t < tiles && ok; t += stride, ++local) {
        const int acc = local & 1;
        if (!(ok = __all_sync(0xffffffffu, ptx::mbar_wait(&tempty[acc], ((local >> 1) & 1) ^ 1, p.err)))) break;
        ptx::tc_fence_after();
        const uint32_t d = tmem + uint32_t(acc * p.acc_cols);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = __all_sync(0xffffffffu, ptx::mbar_wait(&full[stage], phase, p.err)))) break;
          ptx::tc_fence_after();
          const uint32_t w_addr = ptx::smem_u32(ring + stage * p.stage_bytes), a_addr = w_addr + kWBytes;
          for (int h = 0; h < p.subs; ++h) {
            const uint32_t dh = d + uint32_t(h * (bt / 2));
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k) {
              const uint64_t dw = ptx::desc_kmajor_sw128(w_addr + (k >> 2) * 16384 + (k & 3) * 32);
              const uint64_t da = ptx::desc_kmajor_sw128(a_addr + h * sub_bytes + (k >> 2) * a_atom + (k & 3) * 32);
              if (PAIR)
                ptx::umma_f16_ss_pair_warp(dh, dw, da, idesc, (kb != kb0) | (k != 0));
              else
                ptx::umma_f16_ss_warp(dh, dw, da, idesc, (kb != kb0) | (k != 0));
            }
          }
          if (PAIR)
            ptx::umma_commit_pair_mc_warp(&empty[stage], 0x3);
          else
            ptx::umma_commit_warp(&empty[stage]);
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if (PAIR)
          ptx::umma_commit_pair_mc_warp(&tfull[acc], 0x3);
        else
          ptx::umma_commit_warp(&tfull[acc]);
      }
      // every issued MMA is done before TMEM is released
      if (PAIR)
        ptx::umma_commit_pair_mc_warp(drain, 0x1);
      else
        ptx::umma_commit_warp(drain);
      const unsigned long long t0 = ptx::globaltimer();
      while (!ptx::mbar_try_wait(drain, 0) && ptx::globaltimer() - t0 < ptx::kTimeoutNs) {
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, part = (warp - 2) >> 2;
    int local = 0;
    for (long long t = first; t < tiles; t += stride, ++local) {
      const int acc = local & 1;
      int nb, mb;
      tile_at(t, num_n, num_m, nb, mb);
      const int n = nb * kTileN + int(PAIR ? rank * 128 : 0) + quarter * 32 + lane;
      const bool live = n < p.N;
      Column<T, ACT> col{static_cast<const T*>(p.residual), static_cast<T*>(p.out) + n, p.ldr, p.ldo, M, 0.f};
      if (col.res != nullptr) col.res += n;
      if (p.bias != nullptr && live) col.bias = E::to_f32(static_cast<const T*>(p.bias)[n]);
      const long long m_tile = (long long)mb * bt;
      const uint32_t t_row = tmem + (uint32_t(quarter * 32) << 16) + uint32_t(acc * p.acc_cols);
      const int chunks = bt / 16;
      if (!PAIR && p.split > 1) {
        // this share's sums to the CTA that finishes each column: red[source][column of its share][lane]
        if (!__all_sync(0xffffffffu, ptx::mbar_wait(&tfull[acc], 0, p.err))) break;
        ptx::tc_fence_after();
        const int mine = bt / p.split;  // columns each CTA finishes
        for (int c = part; c < chunks; c += 4) {
          uint32_t z[16];
          ptx::tmem_ld_32x32b_x16(t_row + c * 16, z);
          ptx::tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int column = c * 16 + i;
            const uint32_t dst = ptx::mapa_shared(
                ptx::smem_u32(red + (int(rank) * mine + column % mine) * 128 + quarter * 32 + lane), uint32_t(column / mine));
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(__uint_as_float(z[i])) : "memory");
          }
        }
        break;  // one tile a cluster; finished below
      }
      const bool has_res = col.res != nullptr && live;
      const int count = (chunks - part + 3) / 4;  // chunks part, part + 4, ...
      uint16_t r[3][16];
      if (has_res) {
#pragma unroll
        for (int u = 0; u < 3; ++u)
          if (u < count) col.fetch(m_tile + (part + 4 * u) * 16, r[u]);
      }
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(&tfull[acc], (local >> 1) & 1, p.err))) break;
      ptx::tc_fence_after();
      for (int i = 0; i < count; i += 3) {
#pragma unroll
        for (int u = 0; u < 3; ++u) {
          if (i + u < count) {
            const int c = part + 4 * (i + u);
            uint32_t z[16];
            ptx::tmem_ld_32x32b_x16(t_row + c * 16, z);
            ptx::tmem_wait_ld();
            if (live) col.store(m_tile + c * 16, z, r[u]);
            if (has_res && i + u + 3 < count) col.fetch(m_tile + (c + 12) * 16, r[u]);
          }
        }
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR)
          ptx::mbar_arrive_cluster_relaxed(ptx::mapa_shared(ptx::smem_u32(&tempty[acc]), 0));
        else
          ptx::mbar_arrive(&tempty[acc]);
      }
    }
  }
  __syncwarp();
  if (!PAIR && p.split > 1) {
    ptx::cluster_sync();  // all shares' sums have arrived
    if (warp >= 2 && first < tiles) {
      const int quarter = warp & 3, part = (warp - 2) >> 2;
      int nb, mb;
      tile_at(first, num_n, num_m, nb, mb);
      const int n = nb * 128 + quarter * 32 + lane, mine = bt / p.split;
      const bool live = n < p.N;
      const T* res = static_cast<const T*>(p.residual);
      T* out = static_cast<T*>(p.out);
      const float bias = p.bias != nullptr && live ? E::to_f32(static_cast<const T*>(p.bias)[n]) : 0.f;
      for (int j = part; j < mine; j += 4) {
        const long long m = (long long)mb * bt + int(rank) * mine + j;
        if (!live || m >= M) continue;
        float z = 0.f;
        for (int s = 0; s < p.split; ++s) z += red[(s * mine + j) * 128 + quarter * 32 + lane];
        z = activate<T, ACT>(make_float2(z + bias, 0.f)).x;
        if (res != nullptr) z += E::to_f32(res[m * p.ldr + n]);
        out[m * p.ldo + n] = E::from_f32(z);
      }
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (PAIR) ptx::cluster_sync();  // neither CTA leaves while the pair may still touch its memory
  if (warp == 1) {
    ptx::tc_fence_after();
    if (PAIR)
      ptx::tmem_dealloc_pair(tmem, p.tmem_cols);
    else
      ptx::tmem_dealloc(tmem, p.tmem_cols);
  }
}

// ------------------------------------------------------------------------------------- host

gdc_status encode(CUtensorMap* map, bool bf16, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows) {
  auto fn = get_encode_fn();
  if (!fn) return set_error(GDC_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {ld * 2};
  const cuuint32_t box[2] = {64, box_rows}, estr[2] = {1, 1};
  const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base), dims,
                        strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(GDC_ERR_CUDA, "cuTensorMapEncodeTiled (linear residual) failed (%d)", int(r));
  return GDC_OK;
}

struct Config {
  bool pair;
  int bt, split;
};

// What a device can run at once: SMs, and clusters of 2, 4 and 8 CTAs of the single form.
struct DeviceLimits {
  int sms = 148, clusters[4] = {148, 74, 36, 16};
};

// The form of a call: the least of each form's estimate in microseconds wins. The constants order the forms of one
// call as they were measured; they do not predict times. Operand tiles: 95 bytes a nanosecond and SM when all
// SMs load, 130 when half of them do, which is what tiles that other CTAs have brought into L2 come at; weights that
// come from HBM, as with few rows, arrive at half of that or less (all SMs: 44). An epilogue: 11 ns a column,
// 9 more for a residual or a GELU; joining split K 1.2 us; a launch's start is left out. Estimate and time in us:
// 1 x 4096 x 4096 4.4 and 10.8, 64 x 4096 x 4096 5.7 and 14, 4885 x 1024 x 4096 29 and 34, 4885 x 4096 x 1024 GELU 37 and
// 51, 8192 x 8192 x 4096 GELU 317 and 390 to 405.
Config choose(int64_t M, int N, int K, bool residual, int act, const DeviceLimits& dev) {
  Config best{false, 16, 1};
  double best_time = 1e300;
  const int64_t kblocks = (K + kBK - 1) / kBK;
  auto consider = [&](const Config& c) {
    const int64_t tile_n = c.pair ? 256 : 128;
    const int64_t tiles = ((N + tile_n - 1) / tile_n) * ((M + c.bt - 1) / c.bt);
    const int64_t at_once = c.pair ? dev.clusters[1] : (c.split == 1 ? dev.sms : dev.clusters[c.split == 2 ? 1 : c.split == 4 ? 2 : 3]);
    if (c.split > 1 && tiles > at_once) return;
    const int64_t rounds = (tiles + at_once - 1) / at_once;
    if (c.bt > 256 && rounds > 1) return;  // one accumulator only
    const double ctas = double(std::min(tiles, at_once)) * (c.pair ? 2 : c.split);
    const double rate = ctas > dev.sms / 2 ? 95e3 : 130e3;
    const double a_rows = c.pair ? c.bt / 2 : c.bt;
    const double block = std::max((128 + a_rows) * kBK * 2 / rate, 4.0 * c.bt / 1850.0);
    const double main = double((kblocks + c.split - 1) / c.split) * block;
    const double epilogue = c.bt * (0.011 + (residual ? 0.009 : 0) + (act == kActGelu ? 0.009 : 0)) / c.split + (c.split > 1 ? 1.2 : 0);
    const double time = main + double(rounds - 1) * std::max(main, epilogue) + epilogue;
    if (time < best_time * 0.999) {
      best_time = time;
      best = c;
    }
  };
  const int64_t bt_max = std::min<int64_t>(512, (M + 15) / 16 * 16);
  for (int bt = 16; bt <= bt_max || bt == 16; bt += bt < 256 ? 16 : 32) {
    if (M > 64 && bt >= 32) consider({true, bt, 1});
    consider({false, bt, 1});
    if (bt <= kMaxSplitBt)
      for (int s = 2; s <= 8; s *= 2)
        if (s <= kblocks) consider({false, bt, s});
  }
  return best;
}

template <typename T, bool PAIR, int ACT>
gdc_status launch_form(const CUtensorMap& tw, const CUtensorMap& ta, const LinearParams& p, int grid, int cluster, cudaStream_t stream,
                       int dev) {
  auto kern = linear_residual_kernel<T, PAIR, ACT>;
  static PerDeviceOnce configured;
  const cudaError_t ce = cudaError_t(per_device_once(
      configured, dev, [&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem); }));
  if (ce != cudaSuccess) return set_error(GDC_ERR_CUDA, "linear residual smem attribute: %s", cudaGetErrorString(ce));
  const size_t smem = size_t(p.stages) * p.stage_bytes + kCtrlBytes + 1024 + (p.split > 1 ? size_t(p.bt) * 512 : 0);
  GDC_CUDA_TRY(launch_overlapped(kern, unsigned(grid), kThreads, smem, unsigned(cluster), stream, tw, ta, p));
  return GDC_OK;
}

// Limits of a device, asked once: how many clusters fit depends on how its SMs are grouped.
gdc_status device_limits(int dev, DeviceLimits* out) {
  static PerDeviceOnce once;
  static DeviceLimits limits[64];
  auto kern = linear_residual_kernel<__half, false, kActNone>;
  const cudaError_t ce = cudaError_t(per_device_once(once, dev, [&] {
    DeviceLimits& l = limits[dev];
    l.sms = l.clusters[0] = device_sm_count(dev);
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
    for (int i = 1; i < 4 && e == cudaSuccess; ++i) {
      cudaLaunchAttribute attr{};
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = 1u << i;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(unsigned(l.sms) >> i << i);
      cfg.blockDim = dim3(kThreads);
      cfg.dynamicSmemBytes = kMaxSmem;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      e = cudaOccupancyMaxActiveClusters(&l.clusters[i], kern, &cfg);
    }
    return e;
  }));
  if (ce != cudaSuccess) return set_error(GDC_ERR_CUDA, "linear residual cluster limits: %s", cudaGetErrorString(ce));
  *out = limits[dev];
  return GDC_OK;
}

template <typename T>
gdc_status launch_typed(const LinearResidualArgs& a, cudaStream_t stream, int* err) {
  constexpr bool bf16 = ElemOps<T>::kMmaFormat == 1;
  int dev = 0;
  GDC_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return set_error(GDC_ERR_CUDA, "device ordinal out of range");
  DeviceLimits lim;
  GDC_TRY(device_limits(dev, &lim));
  const int sms = lim.sms;
  const Config c = choose(a.M, a.N, a.K, a.residual != nullptr, a.act, lim);
  const int a_rows = c.pair ? c.bt / 2 : c.bt, subs = c.bt > 256 ? 2 : 1;
  CUtensorMap tw, ta;
  GDC_TRY(encode(&tw, bf16, a.w, uint64_t(a.N), uint64_t(a.K), uint64_t(a.ldw), 128));
  GDC_TRY(encode(&ta, bf16, a.a, uint64_t(a.M), uint64_t(a.K), uint64_t(a.lda), uint32_t(a_rows / subs)));
  LinearParams p{};
  p.bias = a.bias;
  p.residual = a.residual;
  p.out = a.out;
  p.ldr = a.ldr;
  p.ldo = a.ldo;
  p.m_cap = a.M;
  p.rows_dev = a.rows_dev;
  p.N = a.N;
  p.K = a.K;
  p.bt = c.bt;
  p.subs = subs;
  p.split = c.split;
  p.stage_bytes = kWBytes + a_rows * kBK * 2;
  const int64_t tile_n = c.pair ? 256 : 128;
  const int64_t tiles = ((a.N + tile_n - 1) / tile_n) * ((a.M + c.bt - 1) / c.bt);
  const int64_t at_once = c.pair ? lim.clusters[1] : (c.split == 1 ? sms : tiles);
  const int64_t blocks = ((a.K + kBK - 1) / kBK + c.split - 1) / c.split;  // K blocks of a CTA's tile
  // As many stages as fit and, where a CTA has one tile, as it has K blocks. (576 threads of 96 registers keep a second
  // CTA of this kernel off the SM whatever the ring's size; only kernels of up to 10,000 registers, such as a small
  // norm, start beside it, and chains of norms and small linears took the same time with rings of any size.)
  const bool one = tiles <= at_once;
  p.stages = std::min(kMaxStages, (c.split > 1 ? kSplitRing : kRingBytes) / p.stage_bytes);
  if (one) p.stages = int(std::min<int64_t>(p.stages, blocks));
  p.acc_cols = (c.bt + 31) / 32 * 32;
  p.tmem_cols = 32;
  while (p.tmem_cols < (one ? 1 : 2) * p.acc_cols) p.tmem_cols *= 2;
  p.err = err;
  const int cluster = c.pair ? 2 : c.split;
  const int grid = c.pair ? 2 * int(std::min<int64_t>(tiles, at_once))
                          : (c.split > 1 ? int(tiles * c.split) : int(std::min<int64_t>(tiles, sms)));
  switch (a.act * 2 + c.pair) {
    case 2 * kActNone: return launch_form<T, false, kActNone>(tw, ta, p, grid, cluster, stream, dev);
    case 2 * kActNone + 1: return launch_form<T, true, kActNone>(tw, ta, p, grid, cluster, stream, dev);
    case 2 * kActGelu: return launch_form<T, false, kActGelu>(tw, ta, p, grid, cluster, stream, dev);
    case 2 * kActGelu + 1: return launch_form<T, true, kActGelu>(tw, ta, p, grid, cluster, stream, dev);
    case 2 * kActRelu: return launch_form<T, false, kActRelu>(tw, ta, p, grid, cluster, stream, dev);
    case 2 * kActRelu + 1: return launch_form<T, true, kActRelu>(tw, ta, p, grid, cluster, stream, dev);
    case 2 * kActSilu: return launch_form<T, false, kActSilu>(tw, ta, p, grid, cluster, stream, dev);
    default: return launch_form<T, true, kActSilu>(tw, ta, p, grid, cluster, stream, dev);
  }
}

}  // namespace

gdc_status launch_linear_residual(Elem t, const LinearResidualArgs& a, cudaStream_t stream, int* err) {
  return t == Elem::kF16 ? launch_typed<__half>(a, stream, err) : launch_typed<__nv_bfloat16>(a, stream, err);
}

}  // namespace gdc
