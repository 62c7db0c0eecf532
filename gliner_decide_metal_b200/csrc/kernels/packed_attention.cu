// Softmax attention with grouped heads over packed sequences on tcgen05 tensor cores.
//
//   s_ij = scale * q_i . k_j over the keys j that query i sees,
//   o_i  = sum_j 2^(c s'_ij - c m_i) v_j / sum_j 2^(c s'_ij - c m_i),   s' = q.k, c = scale log2 e
//
// in one pass over the keys: a running reference m_i of the row's maximum and the running sum
// stay in registers, the unnormalised o_i in TMEM.
//
// Rows. A query tile is 128 MMA rows: row r holds query position pos + r / G and head
// hk * G + r % G of key head hk (G = heads / kv_heads), so a key / value tile is read once for
// all heads of its group and a single token's G heads fill one tile. One work item is two such
// tiles (256 rows) of one sequence and key head against a range of 128-key tiles.
//
// Roles of a CTA (one per SM, persistent over items; each role waits for jobs from warp 9's ring):
//   warps 0-3, 4-7  softmax of tile 0 / tile 1: one thread a row. Reads its 128 scores from TMEM,
//                   writes the weights back over them as 16-bit MMA operands, and at an item's
//                   end divides and stores the row (or stores the split's partial row).
//   warp 8          issues the MMAs: S_t = Q_t K_j^T (both operands in shared memory), then
//                   O_t += P_t V_j (P_t from TMEM); the tensor cores work on one tile while the
//                   softmax warps work on the other.
//   warp 9          the CTA's jobs, and TMA: Q tiles of the item and a ring of K and V tiles, running
//                   ahead into the next item.
// TMEM: S_0 [0, 128), S_1 [128, 256), O_0 [256, 256 + D), O_1 behind it; P_t lies over S_t at D = 128 and
// behind the O's at D = 64, where S_t(j + 1) can then be computed beside the softmax of S_t(j).
// An item of one query tile (tokens taken one at a time) is shared by both row groups, which take
// its key tiles in turn (shared_item).
//
// The reference m_i moves only when a row's maximum has grown by more than 2^8 (then the tile's
// O rows are rescaled in TMEM), so most key tiles need no rescale. S_t(j) complete implies P_t V(j-1) complete
// (one thread issues them in that order) at D = 128, so the rescale needs no wait of its own; at D = 64
// the row warps wait for P_t V(j-1) before they write O_t or P_t.
//
// The weights are rounded to the tensors' type for the second product, the row's sum is of the unrounded
// ones. bf16 has fp32's range; in fp16 the weights are computed 2^7 larger (the factor is in O and in the row's
// sum alike), so they reach up to 2^15, the range's end, and its lower end is that much further away: a
// weight is off by 2^-11 of itself or by 2^-32 of the largest one, whichever is more.
//
// A value that no visible key contributes must not reach a row, but 0 * inf is NaN: a row whose
// result is not finite is computed again from memory by one warp over exactly its visible keys
// (row_by_definition); value rows behind the last key of a sequence are zeroed in shared memory
// first, so ordinary padding never takes that path.
//
// Plan. Lengths are device data. When there are more items than SMs, or few items with many keys,
// plan_kernel lists the items, splits long key ranges into chunks (their partial rows are joined
// by combine_kernel), and orders them by descending cost; otherwise, and for small batches of single
// tokens (plan_layout), a CTA finds its items itself.
//
// What bounds it, and what it reaches on a B200:
//   prompts   256 rows x 128 keys at D = 128 take the tensor cores 2048 cycles and the exponential
//             unit 2048, but a row group's chain (scores 1250 from its weights on, maximum 500,
//             exponentials and rounding 1450, hand-over 300) takes 3550, and two groups fill it to
//             1.7 times the longer of the two. 8192 tokens, 32 / 8 heads of 128, causal: 534 to 541 us, 1030 TFLOP/s,
//             one C call after another (the power cap's clock); 459 to 516 us in short captured bursts. Tried and
//             slower: part of the exponentials as polynomials, two threads a row, weights in halves signalled
//             apart, two issuing warps, 64-key steps with two score buffers.
//   D = 64    S_t is ready when its group is: waits 300, scores 300, maximum 500, exponentials 1600, 3000 in
//             all with both groups on the exponential unit. Four prompts of 4096, 16 / 4 heads: 215 to 225 us,
//             610 to 640 TFLOP/s (242 us with the weights over the scores).
//   tokens    HBM: 48 tokens over 212,000 keys of 8 heads of 128, captured: 154 us, 5.6 TB/s; over 196,000 more uneven
//             ones, one C call after another, 164 to 173 us, 4.6 to 4.9 TB/s. One token over 8000: 18 to 25 us from one GPU
//             to the next, of which 10 its keys and 3 the joining.
//   short     32 sequences of 64 to 256 rows, 16 / 4 heads of 64: 30 us, of which 5 plan, 7 to 12 the
//             first item of each CTA (its instructions are cold), 4 to 5 each further one and up to 4.7 a joining
//             launch that finds nothing.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "elem.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace gdc {

PFN_cuTensorMapEncodeTiled_v12000 get_encode_fn();

namespace {

constexpr int kKeys = 128;       // keys of a tile
constexpr int kThreads = 384;     // three warpgroups; two of the third's warps only take part in barriers
constexpr int kRowRegs = 216, kIssueRegs = 72;  // 256 * 216 + 128 * 72 = 384 * 168, the launch's registers
constexpr int kPlanThreads = 512;
constexpr int kPlanSms = 148;    // the planner's unit of work (the workspace size depends on it)
constexpr float kGrowth = 8.0f;  // log2 growth of a row's maximum that moves its reference
constexpr float kHalfLift = 7.0f;  // log2 of the factor of fp16 weights
// A row's reference in log2 units is rounded to fp32. Beyond this (scores of 2.9 million) the rounding would
// move its weights by more than a quarter of a binade, and further out past what 16 bits hold: such a
// row is computed by its definition (row_by_definition), from differences of scores.
constexpr float kMaxReference = 4194304.f;

// One work item (32 bytes).
struct Item {
  int q_row, lq;   // first query row and number of queries of the sequence
  int k_row, lk;   // first key row and number of keys
  int pos;         // first query position of the item
  int t0, t1;      // key tiles [t0, t1)
  int slot;        // partial rows' slot, -1: the item's only range
};
struct Job {  // an item and the key head to do it for
  Item it;
  int hk, more, pad[2];  // more: 0 ends the CTA's work
};
struct SplitItem {  // an item whose key range was split: slots [slot, slot + n)
  int q_row, lq, k_row, lk, pos, slot, n, pad;
};
struct PlanHeader {
  int n_items, n_splits, split_rows;  // split_rows: rows of the largest split item
};

// Workspace: header, items, split items, partial rows (fp32 O, then reference and sum).
struct PlanLayout {
  int64_t items_ub;    // upper bound of (sequence, item) pairs
  int rows_cap;        // rows of an item that can be used
  int chunks_cap;      // planned items per key head, splits included
  bool planned, split;  // split and not planned: every CTA lists the ranges itself
  size_t items_at, splits_at, part_o_at, part_ml_at, bytes;
};

PlanLayout plan_layout(int batch, int64_t q_rows, int64_t k_rows, int heads, int kv_heads, int dim) {
  PlanLayout l{};
  const int G = heads / kv_heads;
  const int per_item = 2 * (kKeys / G);
  l.items_ub = q_rows / per_item + std::min<int64_t>(batch, q_rows);
  l.rows_cap = int(std::min<int64_t>(int64_t(per_item) * G, q_rows * G));
  const int64_t jobs = l.items_ub * kv_heads;
  // Splitting pays while there are few jobs to an SM (many even out by themselves), the fewer the larger a
  // partial result is (256 rows of 128 columns, written and read again, cost as much as three key tiles):
  // at most eight jobs an SM up to 64 KB, four at 128 KB. Partial rows are bounded to 64 MB.
  const int64_t row_bytes = int64_t(l.rows_cap) * (dim + 2) * 4;
  const int64_t cap = std::min<int64_t>((int64_t(64) << 20) / row_bytes, jobs + 8 * kPlanSms);
  const int64_t most = kPlanSms * std::max<int64_t>(2, std::min<int64_t>(8, 131072 / (int64_t(l.rows_cap) * dim)));
  l.split = k_rows > 2 * kKeys && jobs <= most && cap >= jobs + kPlanSms / 2;
  // Up to 128 sequences of one item each (tokens taken one at a time) and about 48 key tiles an SM: every CTA
  // goes over the offsets itself, which spares a launch (one token over 8000 keys 22.1 -> 18.2 us, 32 over
  // 1000 38.8 -> 35.1, 48 over 95,000 in all 92.7 -> 81.8). With more the planner's order by cost is worth it
  // (48 over 212,000: 154 us planned, 166 so). Measured at head size 128; at 64, whose tiles are half as large, the same
  // limit is used unmeasured.
  const bool direct = q_rows <= per_item && batch <= 128 && (k_rows / kKeys + batch) * kv_heads <= 48 * kPlanSms;
  l.planned = l.split ? !direct : jobs > kPlanSms;
  l.chunks_cap = int(l.split ? cap / kv_heads : std::min<int64_t>(l.items_ub, INT32_MAX));
  auto up = [](size_t v) { return (v + 255) & ~size_t(255); };
  l.items_at = 256;
  l.splits_at = l.items_at + (l.planned ? up(size_t(l.chunks_cap) * sizeof(Item)) : 0);
  l.part_o_at = l.splits_at + (l.split ? up(size_t(l.items_ub) * sizeof(SplitItem)) : 0);
  l.part_ml_at = l.part_o_at + (l.split ? up(size_t(l.chunks_cap) * kv_heads * l.rows_cap * dim * 4) : 0);
  l.bytes = l.part_ml_at + (l.split ? up(size_t(l.chunks_cap) * kv_heads * l.rows_cap * 8) : 0);
  return l;
}

struct Params {
  const void *q, *k, *v;
  void* out;
  long long ldq, ldk, ldv, ldo;
  const int32_t *q_off, *k_off;
  int batch, q_rows, k_rows, heads, kv_heads, dim, group, tile_pos;  // tile_pos: positions of a tile
  int causal;
  float scale, scale_log2;
  // plan
  PlanHeader* header;
  Item* items;
  SplitItem* splits;
  float* part_o;   // [slot * kv_heads + hk][rows_cap][D]
  float2* part_ml; // [slot * kv_heads + hk][rows_cap]
  int rows_cap, chunks_cap;
  long long items_ub;
  int wide_out;  // out's rows are 32-byte aligned
  int can_split;
  unsigned long long wait_ns;  // limit of the waits that rows computed by their definition can hold up (not of those for loads)
  int* err;
};

// Offsets of sequence b; false (and reported by `lane`) where they are not those of the buffers.
__device__ __forceinline__ bool sequence(const Params& p, int b, bool report, int& q0, int& lq, int& k0, int& lk) {
  q0 = p.q_off[b];
  const int q1 = p.q_off[b + 1];
  k0 = p.k_off[b];
  const int k1 = p.k_off[b + 1];
  lq = q1 - q0;
  lk = k1 - k0;
  const bool ok = q0 >= 0 && q1 >= q0 && q1 <= p.q_rows && k0 >= 0 && k1 >= k0 && k1 <= p.k_rows;
  if (!ok && report) atomicOr(p.err, kErrBadOffsets);
  return ok;
}

// Keys that query position `pos` sees (a prefix of the sequence's keys).
__device__ __forceinline__ int seen_keys(int pos, int lq, int lk, int causal) {
  return causal ? max(0, min(lk, pos + 1 + lk - lq)) : lk;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// 64 bytes of one row. A warp's rows lie in different lines, and the store unit takes a line at a time
// whatever its width, so the widest stores cost least.
__device__ __forceinline__ void store64(void* dst, const uint32_t (&w)[16], bool wide) {
  if (wide) {
#pragma unroll
    for (int e = 0; e < 16; e += 8)
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(static_cast<uint32_t*>(dst) + e), "r"(w[e]),
                   "r"(w[e + 1]), "r"(w[e + 2]), "r"(w[e + 3]), "r"(w[e + 4]), "r"(w[e + 5]), "r"(w[e + 6]), "r"(w[e + 7])
                   : "memory");
  } else {
#pragma unroll
    for (int e = 0; e < 16; e += 4)
      *reinterpret_cast<uint4*>(static_cast<uint32_t*>(dst) + e) = make_uint4(w[e], w[e + 1], w[e + 2], w[e + 3]);
  }
}

// One output row from memory over exactly its visible keys: plain softmax in fp32, one warp, 32 keys at
// a time (a lane has one's score, every lane its columns of their values); about 170 ns a key
// (480 key by key).
// The result is left in the lanes' o[D / 32] (columns lane * D / 32 ...).
template <typename T, int D>
__device__ void row_by_definition(const Params& p, int q_row, int lq, int k_row, int lk, int pos, int head, float (&o)[D / 32]) {
  using E = ElemOps<T>;
  constexpr int PER = D / 32;
  const int lane = threadIdx.x & 31;
  const int hk = head / p.group;
  const T* q = static_cast<const T*>(p.q) + (long long)(q_row + pos) * p.ldq + head * D + lane * PER;
  const T* k = static_cast<const T*>(p.k) + (long long)k_row * p.ldk + hk * D;
  const T* v = static_cast<const T*>(p.v) + (long long)k_row * p.ldv + hk * D + lane * PER;
  const int n = seen_keys(pos, lq, lk, p.causal);
  float qv[PER], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    qv[i] = E::to_f32(q[i]);
    o[i] = 0.f;
  }
#pragma unroll 1
  for (int j0 = 0; j0 < n; j0 += 32) {
    const int count = min(32, n - j0);
    const uint4* row = reinterpret_cast<const uint4*>(k + (long long)(j0 + min(lane, count - 1)) * p.ldk);
    float s = 0.f;
#pragma unroll 4
    for (int c = 0; c < D / 8; ++c) {
      const uint4 u = row[c];
      const uint32_t u4[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float2 x = E::unpack(u4[e / 2]);
        s = fmaf(__shfl_sync(0xffffffffu, qv[e % PER], c * (8 / PER) + e / PER), x.x, s);
        s = fmaf(__shfl_sync(0xffffffffu, qv[(e + 1) % PER], c * (8 / PER) + (e + 1) / PER), x.y, s);
      }
    }
    s = lane < count ? s * p.scale : -INFINITY;
    float mn = fmaxf(m, s);  // (passes over NaN, whose weight below is NaN)
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, d));
    const float r = m == mn ? 1.f : expf(m - mn), w = s == -INFINITY ? 0.f : expf(s - mn);
    l = l * r + ptx::warp_sum(w);
    if (l != l) break;  // every column is NaN
    m = mn;
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] *= r;
#pragma unroll 8
    for (int j = 0; j < count; ++j) {
      const float wj = __shfl_sync(0xffffffffu, w, j);
      const uint32_t* src = reinterpret_cast<const uint32_t*>(v + (long long)(j0 + j) * p.ldv);
#pragma unroll
      for (int i = 0; i < PER; i += 2) {
        const float2 x = E::unpack(src[i / 2]);
        o[i] = fmaf(wj, x.x, o[i]);
        o[i + 1] = fmaf(wj, x.y, o[i + 1]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) o[i] = n > 0 ? o[i] / l : 0.f;
}

template <typename T, int D>
__device__ void store_row_by_definition(const Params& p, int q_row, int lq, int k_row, int lk, int pos, int head) {
  using E = ElemOps<T>;
  constexpr int PER = D / 32;
  float o[PER];
  row_by_definition<T, D>(p, q_row, lq, k_row, lk, pos, head, o);
  uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + (long long)(q_row + pos) * p.ldo + head * D +
                                              (threadIdx.x & 31) * PER);
#pragma unroll
  for (int i = 0; i < PER / 2; ++i) dst[i] = E::pack(o[2 * i], o[2 * i + 1]);
}

// ------------------------------------------------------------------------------------- plan

// Length of the chunks that key ranges are split into, in tiles (at most chunks_cap chunks a key head:
// their number is below work / length + items; work, items and the longest item are of one key head).
// One round of chunks where the work allows short ones; otherwise about eight chunks an SM, none so
// short that its partial rows (which cost as much as `over` tiles) weigh much. Two sequences
// of 256 rows after 6000 keys: 103 us in chunks of four tiles, 77 to 86 us so; a prompt of 4096 tokens
// in 16 heads of 128: 99 us split, joining not counted, 74 us whole; prompts of 6000, 700 and 300 in 16
// heads of 64: 157 us split, 123 us whole; 16 tokens over 700 to 2500 keys of 8 heads: 42 us in chunks of
// four tiles, 31 us whole.
template <typename I>
__device__ __forceinline__ int chunk_length(const Params& p, I head_work, int items, int longest) {
  constexpr I kSms = kPlanSms, kWhole = 1 << 30;
  const I work = head_work * p.kv_heads, jobs = I(items) * p.kv_heads;
  auto ceil_div = [](I a, I b) { return (a + b - 1) / b; };
  // rows * dim * 8 bytes at an SM's 44 bytes a nanosecond, over 1.9 us a tile
  const I over = p.rows_cap * p.dim / 10500;
  I c = max(4 + 8 * over, ceil_div(work, 8 * kSms));
  if (jobs <= kSms / 2) {
    const I one = max(2 + 2 * over, ceil_div(work, kSms - jobs));
    if (one <= 8 + 8 * over) c = one;
  } else if ((over > 0 && I(longest) * kSms <= work + work / 4) || (jobs <= kSms && I(longest) * kSms <= 2 * work)) {
    c = kWhole;  // the items even out by themselves, or fill a round whose longest item is near the mean
  }
  const I room = I(p.chunks_cap) * p.kv_heads - jobs;
  return int(min(kWhole, max(c, ceil_div(work, max(I(1), room)))));
}

constexpr int kBuckets = 512;

// Lists the items by descending cost (key tiles of the chunk; a counting sort in shared memory)
// and the split items, in one CTA. Each warp has a run of sequences, a lane one of up to 32 at a time;
// where a sequence has many items the lanes share them out.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(Params p) {
  __shared__ int hist[kBuckets];
  __shared__ unsigned long long s_work, s_items;
  __shared__ int s_max, s_slots, s_splits, s_rows;
  ptx::grid_launch_next();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = kPlanThreads / 32;
  const int per_item = 2 * p.tile_pos;
  if (threadIdx.x == 0) {
    s_work = s_items = 0;
    s_max = s_slots = s_splits = s_rows = 0;
  }
  for (int i = threadIdx.x; i < kBuckets; i += kPlanThreads) hist[i] = 0;
  ptx::grid_wait();
  __syncthreads();
  const int run = (p.batch + warps - 1) / warps;  // sequences of a warp
  // f(q0, lq, k0, lk, position, key tiles) for every item; a sequence of bad offsets has none. The first pass
  // reports those and counts the warp's items, in 64 bits: offsets that decrease can make 2^19 sequences
  // overlap, each of them as long as the query rows. A warp that has counted more than the rows can hold
  // goes over no more items (nothing will be computed), so that the passes end whatever the offsets are.
  auto for_each_item = [&](bool first, auto&& f) {
    const int last = min(p.batch, (warp + 1) * run);
    long long count = 0;
    for (int b0 = warp * run; b0 < last; b0 += 32) {
      int q0 = 0, lq = 0, k0 = 0, lk = 0;
      if (b0 + lane < last && !sequence(p, b0 + lane, first, q0, lq, k0, lk)) lq = 0;
      const int n = (lq + per_item - 1) / per_item;  // (below 2^30)
      if (first) {
        count += __reduce_add_sync(0xffffffffu, n & 0xffff) + ((long long)__reduce_add_sync(0xffffffffu, n >> 16) << 16);
        if (count > p.items_ub) continue;
      }
      auto item = [&](int q, int l, int k, int m, int i) {
        const int pos = i * per_item;
        f(q, l, k, m, pos, (seen_keys(min(pos + per_item, l) - 1, l, m, p.causal) + kKeys - 1) / kKeys);
      };
      if (__reduce_max_sync(0xffffffffu, n) <= 4) {
        for (int i = 0; i < n; ++i) item(q0, lq, k0, lk, i);
      } else {
        for (int s = 0; s < min(32, last - b0); ++s) {
          const int q = __shfl_sync(0xffffffffu, q0, s), l = __shfl_sync(0xffffffffu, lq, s), k = __shfl_sync(0xffffffffu, k0, s),
                    m = __shfl_sync(0xffffffffu, lk, s), ns = __shfl_sync(0xffffffffu, n, s);
          for (int i = lane; i < ns; i += 32) item(q, l, k, m, i);
        }
      }
    }
    __syncwarp();
    return count;
  };
  {
    unsigned long long work = 0;
    int most = 0;
    const long long items = for_each_item(true, [&](int, int, int, int, int, int t) {
      work += t;
      most = max(most, t);
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) work += __shfl_xor_sync(0xffffffffu, work, o);
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) {
      atomicAdd(&s_work, work);
      atomicAdd(&s_items, (unsigned long long)items);
      atomicMax(&s_max, most);
    }
  }
  __syncthreads();
  // More items than the query rows can hold: sequences overlap, so that some offset decreases, which has been
  // reported; nothing is computed. (This is what keeps the lists below inside the workspace.)
  if (s_items > (unsigned long long)p.items_ub) {
    if (threadIdx.x == 0) *p.header = PlanHeader{0, 0, 0};
    return;
  }
  const int chunk = p.can_split ? chunk_length<long long>(p, (long long)s_work, int(s_items), s_max) : 1 << 30;
  int shift = 0;
  while ((min(chunk, s_max) >> shift) >= kBuckets) ++shift;
  auto bucket = [&](int tiles) { return kBuckets - 1 - min(kBuckets - 1, tiles >> shift); };
  for (int pass = 0; pass < 2; ++pass) {
    for_each_item(false, [&](int q0, int lq, int k0, int lk, int pos, int t) {
      const int parts = t > chunk ? (t + chunk - 1) / chunk : 1;
      const int len = (t + parts - 1) / parts;
      int slot = -1;
      if (pass == 1 && parts > 1) {
        slot = atomicAdd(&s_slots, parts);
        atomicMax(&s_rows, min(per_item, lq - pos) * p.group);
        p.splits[atomicAdd(&s_splits, 1)] = SplitItem{q0, lq, k0, lk, pos, slot, parts, 0};
      }
      for (int c = 0; c < parts; ++c) {
        const int t0 = min(t, c * len), t1 = min(t, t0 + len);
        const int at = atomicAdd(&hist[bucket(t1 - t0)], 1);
        if (pass == 1) p.items[at] = Item{q0, lq, k0, lk, pos, t0, t1, parts > 1 ? slot + c : -1};
      }
    });
    __syncthreads();
    if (pass == 0) {
      // exclusive prefix sum of the histogram (descending cost: bucket 0 holds the longest)
      int v = threadIdx.x < kBuckets ? hist[threadIdx.x] : 0;
      int incl = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
      }
      __shared__ int sums[32];
      if (lane == 31) sums[warp] = incl;
      __syncthreads();
      int before = 0;
      for (int w = 0; w < warp; ++w) before += sums[w];
      if (threadIdx.x < kBuckets) hist[threadIdx.x] = before + incl - v;
      __syncthreads();
    }
  }
  if (threadIdx.x == 0) {
    p.header->n_items = hist[kBuckets - 1];
    p.header->n_splits = s_splits;
    p.header->split_rows = s_rows;
  }
}

// ------------------------------------------------------------------------------------- main

template <int D>
struct Shape {
  static constexpr int kAtoms = D / 64;
  static constexpr int kTileBytes = 128 * D * 2;
  static constexpr int kStages = D == 128 ? 5 : 10;
  // D = 64 leaves TMEM columns for the weights beside the scores, so S_t(j + 1) is on its way while the
  // softmax of S_t(j) is; at D = 128 the weights lie over the scores they come from.
  static constexpr bool kOwnP = D == 64;
  static constexpr int kAhead = kOwnP ? 2 : 1;  // key tiles before an item's first value tile
  static constexpr int kOffQ = 0;
  static constexpr int kOffRing = 2 * kTileBytes;
  static constexpr int kOffBar = kOffRing + kStages * kTileBytes;
  static constexpr int kOffMl = kOffBar + 512;  // tile 1's references and sums of a shared item
  static constexpr int kSmemBytes = kOffMl + 128 * 8 + 1024;
  static_assert(kSmemBytes <= 232448, "shared memory of a CTA");
};

struct Bars {
  uint64_t full[10], empty[10];
  uint64_t q_full[2], q_empty[2], s_full[2], p_ready[2], o_full[2], o_free[2], s_free[2], drain;
  uint64_t job_full[2], job_empty[2], ml_ready;
  uint32_t tmem, pad;
  Job job[2];
};
static_assert(sizeof(Bars) <= 512, "barrier block");

__device__ __forceinline__ uint64_t desc_v(uint32_t addr) {
  // MN-major, 128-byte swizzle: 64-column atoms 16 KB apart (leading offset), 8-key groups 1 KB
  // apart (stride offset)
  uint64_t d = uint64_t((addr >> 4) & 0x3FFFu);
  d |= uint64_t(16384u >> 4) << 16;
  d |= uint64_t(1024u >> 4) << 32;
  d |= uint64_t(1u) << 46;
  d |= uint64_t(2u) << 61;
  return d;
}

// Key tiles of query tile `t` inside the item's range: [t0, t0 + n).
__device__ __forceinline__ int tile_count(const Params& p, const Item& it, int t) {
  const int first = it.pos + t * p.tile_pos;
  if (first >= it.lq) return 0;
  const int last = min(first + p.tile_pos, it.lq) - 1;
  const int need = (seen_keys(last, it.lq, it.lk, p.causal) + kKeys - 1) / kKeys;
  return max(0, min(it.t1, need) - it.t0);
}

// An item whose rows fill one query tile at most and that has several key tiles (tokens taken one at a
// time): both row groups work on that tile, group 0 on the even key tiles and group 1 on the odd ones,
// each with its own reference, sum and O; group 0 joins them at the end. One group alone takes
// about 1.9 us a 64 KB key and value tile, twice what memory needs for it.
__device__ __forceinline__ bool shared_item(const Params& p, const Item& it) {
  return it.pos + p.tile_pos >= it.lq && tile_count(p, it, 0) > 1;
}

// The CTA's next job, by its producer (one lane): planned ones from the list, every other round
// backwards (the list is in descending cost, so a CTA's share evens out).
__device__ __forceinline__ bool next_planned(const Params& p, int round, Job& job) {
  const long long g = gridDim.x;
  const long long at = (long long)round * g + ((round & 1) ? g - 1 - blockIdx.x : blockIdx.x);
  if (at >= (long long)p.header->n_items * p.kv_heads) return false;  // only in the last round: earlier ones are full
  const int4* src = reinterpret_cast<const int4*>(p.items + at / p.kv_heads);
  const int4 a = src[0], b = src[1];
  job.it = Item{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  job.hk = int(at % p.kv_heads);
  return true;
}

// Inclusive sum over the warp's lanes up to this one.
__device__ __forceinline__ int warp_prefix(int v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// The unplanned job of this CTA: the (blockIdx.x / kv_heads)-th item in sequence order. One warp;
// the result is the same in every lane.
__device__ __forceinline__ bool find_job(const Params& p, Job& job) {
  const int lane = threadIdx.x & 31, per_item = 2 * p.tile_pos;
  int want = blockIdx.x / p.kv_heads;
  job.hk = blockIdx.x % p.kv_heads;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    int q0 = 0, lq = 0, k0 = 0, lk = 0, n = 0;
    if (b0 + lane < p.batch && sequence(p, b0 + lane, true, q0, lq, k0, lk)) n = (lq + per_item - 1) / per_item;
    const int incl = warp_prefix(n);
    const int i = want - (incl - n);
    const uint32_t hit = __ballot_sync(0xffffffffu, i >= 0 && i < n);
    if (hit != 0) {
      const int src = __ffs(hit) - 1;
      Item& it = job.it;
      it.q_row = __shfl_sync(0xffffffffu, q0, src);
      it.lq = __shfl_sync(0xffffffffu, lq, src);
      it.k_row = __shfl_sync(0xffffffffu, k0, src);
      it.lk = __shfl_sync(0xffffffffu, lk, src);
      it.pos = __shfl_sync(0xffffffffu, i, src) * per_item;
      it.t0 = 0;
      it.t1 = (seen_keys(min(it.pos + per_item, it.lq) - 1, it.lq, it.lk, p.causal) + kKeys - 1) / kKeys;
      it.slot = -1;
      return true;
    }
    want -= __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
}

// Calls whose sequences have an item each at most (split, not planned): sequence b of this lane, its key
// tiles (-1: no item). One warp.
__device__ __forceinline__ int only_item(const Params& p, int b, bool report, int& q0, int& lq, int& k0, int& lk) {
  q0 = lq = k0 = lk = 0;
  if (b >= p.batch || !sequence(p, b, report, q0, lq, k0, lk) || lq == 0) return -1;
  return (seen_keys(lq - 1, lq, lk, p.causal) + kKeys - 1) / kKeys;
}

// The chunk length of up to 32 such sequences whose items fill more than a round or are uneven: each lane
// weighs one length (the last: no splitting) by the rounds that its chunks take: 1.2 us a tile, 5.5 a round, 3
// for joining. Measured against chunk_length: 24 tokens over 500 to 2000 keys of 8 heads of 128: 43 -> 35 us,
// 12 over 300 to 4000: 32 -> 27 us, 32 over 1000: 35.4 both; of 64 short ones
// the weighing costs more than it gives (22.0 -> 23.3). The constants are head size 128's, at 64 as well (there 24 over
// 500 to 2000 take 30 us and 12 over 300 to 4000 26).
__device__ __forceinline__ int weighed_length(const Params& p, int t, int longest) {
  const int lane = threadIdx.x & 31;
  const int whole = max(longest, 1), mine = lane == 31 ? whole : min(whole, (lane + 2) * (1 + longest / 48));
  const float inv = 1.f / float(mine);
  int chunks = 0;
#pragma unroll 8
  for (int i = 0; i < 32; ++i) {
    const int u = __shfl_sync(0xffffffffu, t, i);
    chunks += u < 0 ? 0 : max(1, int((float(u) - 0.5f) * inv) + 1);
  }
  const int rounds = (chunks * p.kv_heads + int(gridDim.x) - 1) / int(gridDim.x);
  const bool fits = chunks <= p.chunks_cap || mine == whole;  // no more chunks than there are slots
  const float us = fits ? float(rounds) * (1.2f * float(mine) + 5.5f) + (mine < whole ? 3.f : 0.f) : INFINITY;
  const float best = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(us)));  // (positive: ordered as integers)
  const int chunk = __shfl_sync(0xffffffffu, mine, __ffs(__ballot_sync(0xffffffffu, us == best)) - 1);
  const int count = t > chunk ? (t + chunk - 1) / chunk : int(t >= 0);  // (the same exactly)
  return __reduce_add_sync(0xffffffffu, count) <= p.chunks_cap ? chunk : whole;
}

// The chunk length of such a call (0: nothing to do); CTA 0 lists the split items for combine_kernel.
__device__ __forceinline__ int plan_in_place(const Params& p) {
  const int lane = threadIdx.x & 31;
  int work = 0, items = 0, longest = 0, t = -1, q0, lq, k0, lk;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    t = only_item(p, b0 + lane, true, q0, lq, k0, lk);
    items += t >= 0;
    work += max(t, 0);
    longest = max(longest, t);
  }
  work = __reduce_add_sync(0xffffffffu, work);
  items = __reduce_add_sync(0xffffffffu, items);
  longest = __reduce_max_sync(0xffffffffu, longest);
  const bool none = items == 0 || items > p.items_ub;  // (overlapping sequences, as in plan_kernel)
  int chunk = none ? 0 : chunk_length<int>(p, work, items, longest);
  const int jobs = items * p.kv_heads;
  if (!none && p.batch <= 32 && jobs > kPlanSms / 2 && (jobs > kPlanSms || longest * kPlanSms > 2 * work * p.kv_heads))
    chunk = weighed_length(p, t, longest);
  if (blockIdx.x == 0) {
    int splits = 0, slots = 0, rows = 0;
    for (int b0 = 0; !none && b0 < p.batch; b0 += 32) {
      const int t = only_item(p, b0 + lane, false, q0, lq, k0, lk);
      const int parts = t > chunk ? (t + chunk - 1) / chunk : 0;
      const uint32_t split = __ballot_sync(0xffffffffu, parts > 0);
      const int incl = warp_prefix(parts);
      if (parts > 0)
        p.splits[splits + __popc(split & ((1u << lane) - 1))] = SplitItem{q0, lq, k0, lk, 0, slots + incl - parts, parts, 0};
      if (parts > 0) rows = max(rows, lq * p.group);
      splits += __popc(split);
      slots += __shfl_sync(0xffffffffu, incl, 31);
    }
    rows = __reduce_max_sync(0xffffffffu, rows);
    if (lane == 0) *p.header = PlanHeader{0, splits, rows};
  }
  return chunk;
}

// The CTA's job of a round: its number counts the chunks of all sequences in order, every other round backwards.
__device__ __forceinline__ bool find_chunk(const Params& p, int chunk, int round, Job& job) {
  if (chunk == 0) return false;
  const int lane = threadIdx.x & 31, g = gridDim.x;
  const int at = round * g + ((round & 1) ? g - 1 - int(blockIdx.x) : int(blockIdx.x));
  int want = at / p.kv_heads, slots = 0;
  job.hk = at % p.kv_heads;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    int q0, lq, k0, lk;
    const int t = only_item(p, b0 + lane, false, q0, lq, k0, lk);
    const int parts = t > chunk ? (t + chunk - 1) / chunk : int(t >= 0), slotted = parts > 1 ? parts : 0;
    const int incl = warp_prefix(parts), slots_incl = warp_prefix(slotted);
    const int i = want - (incl - parts);
    const uint32_t hit = __ballot_sync(0xffffffffu, i >= 0 && i < parts);
    if (hit != 0) {
      const int len = parts > 0 ? (t + parts - 1) / parts : 0;
      const int t0 = min(t, i * len), slot = parts > 1 ? slots + slots_incl - slotted + i : -1;
      const int src = __ffs(hit) - 1;
      auto of = [&](int v) { return __shfl_sync(0xffffffffu, v, src); };
      job.it = Item{of(q0), of(lq), of(k0), of(lk), 0, of(t0), of(min(t, t0 + len)), of(slot)};
      return true;
    }
    want -= __shfl_sync(0xffffffffu, incl, 31);
    slots += __shfl_sync(0xffffffffu, slots_incl, 31);
  }
  return false;
}

// A consumer's view of the job ring.
struct Jobs {
  Bars* bars;
  uint32_t n = 0;
  // Waits for the next job (all lanes of a warp); null: no more, or a wait gave up.
  __device__ __forceinline__ const Job* next(int* err, unsigned long long wait_ns) {
    if (!__all_sync(0xffffffffu, ptx::mbar_wait(&bars->job_full[n & 1], (n >> 1) & 1, err, wait_ns))) return nullptr;
    const Job* job = &bars->job[n & 1];
    return job->more ? job : nullptr;
  }
  __device__ __forceinline__ void done() {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(&bars->job_empty[n & 1]);
    ++n;
  }
};

template <typename T, int D, bool PLANNED>
__global__ void __launch_bounds__(kThreads, 1)
    packed_attention_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                            const __grid_constant__ CUtensorMap tm_v, const Params p) {
  using S = Shape<D>;
  using E = ElemOps<T>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_q = smem + S::kOffQ;
  uint8_t* s_ring = smem + S::kOffRing;
  Bars* bars = reinterpret_cast<Bars*>(smem + S::kOffBar);
  const int warp = ptx::warp_index(), lane = threadIdx.x & 31;
  int* err = p.err;

  ptx::grid_launch_next();
  if (threadIdx.x == 0) {
    ptx::prefetch_tensor_map(&tm_q);
    ptx::prefetch_tensor_map(&tm_k);
    ptx::prefetch_tensor_map(&tm_v);
    for (int i = 0; i < S::kStages; ++i) {
      ptx::mbar_init(&bars->full[i], 1);
      ptx::mbar_init(&bars->empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      ptx::mbar_init(&bars->q_full[t], 1);
      ptx::mbar_init(&bars->q_empty[t], 1);
      ptx::mbar_init(&bars->s_full[t], 1);
      ptx::mbar_init(&bars->p_ready[t], 4);
      ptx::mbar_init(&bars->o_full[t], 1);
      ptx::mbar_init(&bars->o_free[t], 4);
      ptx::mbar_init(&bars->s_free[t], 4);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&bars->job_full[i], 1);
      ptx::mbar_init(&bars->job_empty[i], 9);  // the MMA warp and the eight row warps
    }
    ptx::mbar_init(&bars->ml_ready, 4);
    ptx::mbar_init(&bars->drain, 1);
    ptx::fence_barrier_init();
  }
  if (warp == 8) {
    ptx::tmem_alloc(&bars->tmem, 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  ptx::grid_wait();
  const uint32_t tmem = bars->tmem;
  Jobs jobs{bars};

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    if (warp == 9) {
      Job job;
      int stage = 0;
      uint32_t phase = 0;
      uint32_t q_uses[2] = {0, 0};
      long long issued = 0;
      const int chunk = !PLANNED && p.can_split ? plan_in_place(p) : 0;
      for (int round = 0;; ++round) {  // the warp finds a job, one lane hands it out and loads its tiles
        bool more;
        if (PLANNED)
          more = next_planned(p, round, job);
        else
          more = p.can_split ? find_chunk(p, chunk, round, job) : round == 0 && find_job(p, job);
        bool ok = true;
        if (lane == 0) {
          job.more = more;
          Bars* b = bars;
          if ((ok = ptx::mbar_wait(&b->job_empty[round & 1], ((round >> 1) & 1) ^ 1, err, p.wait_ns))) {
            b->job[round & 1] = job;
            ptx::mbar_arrive(&b->job_full[round & 1]);
          }
        }
        if (lane == 0 && ok && more) {
          const Item& it = job.it;
          const int hk = job.hk;
          const int n0 = tile_count(p, it, 0), n1 = tile_count(p, it, 1), n = max(n0, n1);
          auto load_q = [&](int t) {
            if (!(ok = ok && ptx::mbar_wait(&bars->q_empty[t], (q_uses[t] & 1) ^ 1, err, p.wait_ns))) return;
            ++q_uses[t];
            ptx::mbar_arrive_expect_tx(&bars->q_full[t], uint32_t(S::kAtoms * p.tile_pos * p.group * 128));
            for (int a = 0; a < S::kAtoms; ++a)
              ptx::tma_load_3d(s_q + t * S::kTileBytes + a * 16384, &tm_q, a * 64, hk * p.group,
                               it.q_row + it.pos + t * p.tile_pos, &bars->q_full[t]);
          };
          auto load_kv = [&](const CUtensorMap* map, int j) {
            if (!(ok = ok && ptx::mbar_wait(&bars->empty[stage], phase ^ 1, err, p.wait_ns))) return;
            ptx::mbar_arrive_expect_tx(&bars->full[stage], uint32_t(S::kTileBytes));
            for (int a = 0; a < S::kAtoms; ++a)
              ptx::tma_load_2d(s_ring + stage * S::kTileBytes + a * 16384, map, hk * D + a * 64,
                               it.k_row + (it.t0 + j) * kKeys, &bars->full[stage]);
            ++issued;
            if (++stage == S::kStages) {
              stage = 0;
              phase ^= 1;
            }
          };
          if (n > 0) {
            if (n0 > 0) load_q(0);
            load_kv(&tm_k, 0);
            if (n1 > 0) load_q(1);
            const int ahead = shared_item(p, it) ? 2 : S::kAhead;
            if (ahead == 2 && n > 1) load_kv(&tm_k, 1);
            for (int j = 0; j < n && ok; ++j) {
              load_kv(&tm_v, j);
              if (j + ahead < n) load_kv(&tm_k, j + ahead);
            }
          }
        }
        if (!__shfl_sync(0xffffffffu, int(ok && more), 0)) break;
      }
      if (lane == 0) {
        // the loads in flight land before the CTA can exit (bounded)
        auto landed = [&](uint64_t* bar, uint32_t parity) {
          const unsigned long long t0 = ptx::globaltimer();
          while (!ptx::mbar_try_wait(bar, parity) && ptx::globaltimer() - t0 < ptx::kTimeoutNs) {
          }
        };
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (q_uses[t] > 0) landed(&bars->q_full[t], (q_uses[t] - 1) & 1);
        for (long long j = std::max(0ll, issued - S::kStages); j < issued; ++j)
          landed(&bars->full[j % S::kStages], uint32_t((j / S::kStages) & 1));
      }
    }
    if (warp == 8) {
      constexpr uint32_t fmt = (E::kMmaFormat << 7) | (E::kMmaFormat << 10);
      constexpr uint32_t idesc_s = ptx::idesc_f16_f32(128, kKeys) | fmt;
      constexpr uint32_t idesc_o = ptx::idesc_f16_f32(128, D, 1) | fmt;
      int stage = 0;
      uint32_t phase = 0;
      uint32_t items_of[2] = {0, 0}, p_uses[2] = {0, 0};
      uint32_t q1_skipped = 0;  // shared items: group 1 took part without a query tile of its own
      bool ok = true;
      while (ok) {
        const Job* job = jobs.next(err, p.wait_ns);
        if (job == nullptr) break;
        const int cnt[2] = {tile_count(p, job->it, 0), tile_count(p, job->it, 1)};
        const int n = max(cnt[0], cnt[1]);
        const int keys_left = job->it.lk - job->it.t0 * kKeys;
        const bool shared = shared_item(p, job->it);
        jobs.done();
        if (n == 0) continue;
        auto advance = [&] {
          if (++stage == S::kStages) {
            stage = 0;
            phase ^= 1;
          }
        };
        // S_t = Q_tq K^T
        auto products = [&](int t, int tq, uint32_t k_addr) {
          const uint32_t q_addr = ptx::smem_u32(s_q + tq * S::kTileBytes);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = uint32_t(k >> 2) * 16384 + (k & 3) * 32;
            ptx::umma_f16_ss_warp(tmem + t * 128, ptx::desc_kmajor_sw128(q_addr + off), ptx::desc_kmajor_sw128(k_addr + off), idesc_s,
                                  k != 0);
          }
          ptx::umma_commit_warp(&bars->s_full[t]);
        };
        auto wait_tile = [&] {
          const bool got = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->full[stage], phase, err));
          ptx::tc_fence_after();
          return got;
        };
        // value rows behind the sequence's last key (valid ones before them): zero, whatever the buffer holds there
        auto zero_tail = [&](uint8_t* v_tile, int valid) {
          if (valid >= kKeys) return;
          for (int i = lane; i < (kKeys - valid) * 8; i += 32)
#pragma unroll
            for (int a = 0; a < S::kAtoms; ++a)
              *reinterpret_cast<uint4*>(v_tile + a * 16384 + valid * 128 + i * 16) = make_uint4(0, 0, 0, 0);
          ptx::fence_proxy_async_smem();
          __syncwarp();
        };
        // O_t (+)= P_t V; o_full: of the item's last one, or where the weights have columns of their own of each
        auto values = [&](int t, uint32_t v_addr, bool first, bool last) {
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)
            ptx::umma_f16_ts_warp(tmem + 256 + t * D, tmem + (S::kOwnP ? 384 + t * 64 : t * 128) + k * 8, desc_v(v_addr + k * 2048),
                                  idesc_o, !first | (k != 0));
          if (S::kOwnP || last) ptx::umma_commit_warp(&bars->o_full[t]);
        };
        // the weights of P_t, and before its first product of an item, O_t's columns
        auto weights_ready = [&](int t, bool first) {
          bool got = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->p_ready[t], p_uses[t] & 1, err, p.wait_ns));
          ++p_uses[t];
          if (got && first) got = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->o_free[t], (items_of[t] & 1) ^ 1, err));
          ptx::tc_fence_after();
          return got;
        };
        if (shared) {
          // tiles in the order K0 K1 V0 K2 V1 K3 ..., group j % 2 takes tile j
          ok = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->q_full[0], items_of[0] & 1, err));
          auto next_scores = [&](int t) {
            ok = wait_tile();
            if (!ok) return;
            products(t, 0, ptx::smem_u32(s_ring + stage * S::kTileBytes));
            ptx::umma_commit_warp(&bars->empty[stage]);
            advance();
          };
          if (ok) next_scores(0);
          if (ok) next_scores(1);
          if (ok && n == 2) ptx::umma_commit_warp(&bars->q_empty[0]);
          for (int j = 0; j < n && ok; j += 2) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (!ok || j + t >= n) continue;
              if (!(ok = wait_tile())) continue;
              zero_tail(s_ring + stage * S::kTileBytes, keys_left - (j + t) * kKeys);
              if (!(ok = weights_ready(t, j == 0))) continue;
              values(t, ptx::smem_u32(s_ring + stage * S::kTileBytes), j == 0, j + t + 2 >= n);
              ptx::umma_commit_warp(&bars->empty[stage]);
              advance();
              if (j + t + 2 < n) {
                next_scores(t);
                if (ok && j + t + 3 == n) ptx::umma_commit_warp(&bars->q_empty[0]);
              }
            }
          }
          ++items_of[0];
          ++items_of[1];
          ++q1_skipped;
          continue;
        }
        auto scores = [&](int t, int j, uint32_t k_addr) {
          products(t, t, k_addr);
          if (j + 1 == cnt[t]) ptx::umma_commit_warp(&bars->q_empty[t]);
        };
        // S_t(0)
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->full[stage], phase, err));
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (ok && cnt[t] > 0) {
            ok = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->q_full[t], (items_of[t] - (t == 1 ? q1_skipped : 0u)) & 1, err));
            ptx::tc_fence_after();
            if (ok) scores(t, 0, ptx::smem_u32(s_ring + stage * S::kTileBytes));
          }
        if (!ok) break;
        ptx::umma_commit_warp(&bars->empty[stage]);
        advance();
        // S_t's columns have been read (step p_uses[t] of this tile, counted over the items)
        auto scores_read = [&](int t) {
          const bool got = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->s_free[t], p_uses[t] & 1, err, p.wait_ns));
          ptx::tc_fence_after();
          return got;
        };
        if (S::kOwnP && n > 1) {
          ok = wait_tile();
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (ok && cnt[t] > 1 && (ok = scores_read(t))) scores(t, 1, ptx::smem_u32(s_ring + stage * S::kTileBytes));
          if (!ok) break;
          ptx::umma_commit_warp(&bars->empty[stage]);
          advance();
        }
        for (int j = 0; j < n && ok; ++j) {
          const int v_stage = stage;
          const uint32_t v_phase = phase;
          advance();
          ok = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->full[v_stage], v_phase, err));
          if (!ok) break;
          uint8_t* v_tile = s_ring + v_stage * S::kTileBytes;
          zero_tail(v_tile, keys_left - j * kKeys);
          const bool more = j + S::kAhead < n;
          bool k_ready = false;
          const uint32_t v_addr = ptx::smem_u32(v_tile);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!ok || j >= cnt[t]) continue;
            if (!(ok = weights_ready(t, j == 0))) continue;
            values(t, v_addr, j == 0, j + 1 == cnt[t]);
            if (j + S::kAhead < cnt[t]) {
              if (!k_ready) {
                ok = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->full[stage], phase, err));
                if (!ok) continue;
                ptx::tc_fence_after();
                k_ready = true;
              }
              if (S::kOwnP && !(ok = scores_read(t))) continue;
              scores(t, j + S::kAhead, ptx::smem_u32(s_ring + stage * S::kTileBytes));
            }
          }
          if (!ok) break;
          ptx::umma_commit_warp(&bars->empty[v_stage]);
          if (more) {
            ptx::umma_commit_warp(&bars->empty[stage]);
            advance();
          }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (cnt[t] > 0) ++items_of[t];
      }
      // every issued MMA is done before TMEM is released
      ptx::umma_commit_warp(&bars->drain);
      if (lane == 0) {
        const unsigned long long t0 = ptx::globaltimer();
        while (!ptx::mbar_try_wait(&bars->drain, 0) && ptx::globaltimer() - t0 < ptx::kTimeoutNs) {
        }
      }
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRowRegs));
    const int t = warp >> 2;
    const int r = (warp & 3) * 32 + lane;
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + t * 128 + lanes, t_o = tmem + 256 + t * D + lanes;
    const uint32_t t_p = S::kOwnP ? tmem + 384 + t * 64 + lanes : t_s;
    const int row_pos = r / p.group, row_head = r % p.group;
    const int warp_pos = ((warp & 3) * 32) / p.group;
    const float c = p.scale_log2;
    constexpr float kLift = E::kMmaFormat == 0 ? kHalfLift : 0.f;
    uint32_t s_uses = 0, o_uses = 0, joins = 0;
    float2* ml = reinterpret_cast<float2*>(smem + S::kOffMl) + r;
    bool ok = true;
    while (true) {
      const Job* job = jobs.next(err, p.wait_ns);
      if (job == nullptr) break;
      // key tiles of this group; keys that the row, and the warp's first row, see from the range's first on;
      // keys from one of the group's tiles to the next
      int n, rel, warp_rel, stride = kKeys;
      const bool shared = shared_item(p, job->it);
      const int tq = shared ? 0 : t;  // query tile
      {
        const Item& it = job->it;
        n = tile_count(p, it, tq);
        const int pos = it.pos + tq * p.tile_pos + row_pos;
        rel = (row_pos < p.tile_pos && pos < it.lq ? seen_keys(pos, it.lq, it.lk, p.causal) : 0) - it.t0 * kKeys;
        warp_rel = seen_keys(min(it.pos + tq * p.tile_pos + warp_pos, it.lq - 1), it.lq, it.lk, p.causal) - it.t0 * kKeys;
        if (shared) {
          n = (n + 1 - t) / 2;
          rel -= t * kKeys;
          warp_rel -= t * kKeys;
          stride = 2 * kKeys;
        }
      }
      float m = -INFINITY, mc = 0.f;
      float2 sum0 = make_float2(0.f, 0.f), sum1 = make_float2(0.f, 0.f);
      for (int j = 0; j < n; ++j) {
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->s_full[t], s_uses & 1, err, p.wait_ns));
        ++s_uses;
        if (!ok) break;
        ptx::tc_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int i = 0; i < 4; ++i) ptx::tmem_ld_32x32b_x32(t_s + i * 32, s[i]);
        ptx::tmem_wait_ld();
        if (S::kOwnP) {
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(&bars->s_free[t]);
        }
        if (j * stride + kKeys > warp_rel) {  // some row of the warp does not see the whole tile
          const int vis = rel - j * stride;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (i * 32 + e >= vis) s[i][e] = 0xff800000u;
        }
        float mx[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          mx[i] = __uint_as_float(s[i][0]);
#pragma unroll
          for (int e = 1; e < 31; e += 2) mx[i] = max3_nan(mx[i], __uint_as_float(s[i][e]), __uint_as_float(s[i][e + 1]));
          mx[i] = max3_nan(mx[i], __uint_as_float(s[i][31]), __uint_as_float(s[i][31]));
        }
        const float top = max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], m);
        if (j == 0) {
          m = top;
          mc = m == -INFINITY ? 0.f : fmaf(m, c, -kLift);
        } else {
          if (S::kOwnP) {  // the last product has read the weights and written O
            ok = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->o_full[t], o_uses & 1, err, p.wait_ns));
            ++o_uses;
            if (!ok) break;
            ptx::tc_fence_after();
          }
          const bool grow = !((top - m) * c <= kGrowth) && top != m;
          if (__any_sync(0xffffffffu, grow)) {
            const float f = grow ? ex2(m * c - top * c) : 1.f;
            if (grow) {
              m = top;
              mc = fmaf(m, c, -kLift);
            }
            sum0.x *= f;
            sum0.y *= f;
            sum1.x *= f;
            sum1.y *= f;
#pragma unroll 1
            for (int i = 0; i < D / 16; ++i) {  // rare: few registers beside the scores
              uint32_t o[16];
              ptx::tmem_ld_32x32b_x16(t_o + i * 16, o);
              ptx::tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              ptx::tmem_st_32x32b_x16(t_o + i * 16, o);
            }
          }
        }
        const float2 c2 = make_float2(c, c), mc2 = make_float2(-mc, -mc);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float2 x = __ffma2_rn(make_float2(__uint_as_float(s[i][2 * e]), __uint_as_float(s[i][2 * e + 1])), c2, mc2);
            x.x = ex2(x.x);
            x.y = ex2(x.y);
            if (e & 1)
              sum1 = __fadd2_rn(sum1, x);
            else
              sum0 = __fadd2_rn(sum0, x);
            w[e] = E::pack(x.x, x.y);
          }
          ptx::tmem_st_32x32b_x16(t_p + i * 16, w);
        }
        ptx::tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&bars->p_ready[t]);
      }
      if (!ok) break;
      // ---- the item's rows of this tile
      float l = (sum0.x + sum0.y) + (sum1.x + sum1.y);
      if (fabsf(mc) > kMaxReference) l = NAN;  // (in a split's or group's partial row: of the joined row)
      const Item it = job->it;
      const int hk = job->hk;
      const int head = hk * p.group + row_head, pos = it.pos + t * p.tile_pos + row_pos;
      const bool live = row_pos < p.tile_pos && pos < it.lq;
      const int seen = live ? seen_keys(pos, it.lq, it.lk, p.causal) : 0;
      const long long at = it.slot < 0 ? 0 : ((long long)it.slot * p.kv_heads + hk) * p.rows_cap + t * p.tile_pos * p.group + r;
      T* dst = static_cast<T*>(p.out) + (long long)(it.q_row + pos) * p.ldo + head * D;
      float* part = p.part_o + at * D;
      const bool scaled = it.slot < 0;  // a split's partial row is left unnormalised
      // factors of O_t and, in a shared item, of group 1's O
      float f0 = !scaled ? 1.f : seen > 0 ? 1.f / l : 0.f, f1 = 0.f;
      if (n > 0) {
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->o_full[t], o_uses & 1, err, p.wait_ns));
        ++o_uses;
        if (!ok) break;
        ptx::tc_fence_after();
      }
      if (shared && t == 1) {
        // group 0 joins the two (the wait above also says that it has read the last item's)
        *ml = make_float2(m, l);
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&bars->ml_ready);
        jobs.done();
        continue;
      }
      if (shared) {
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->ml_ready, joins & 1, err, p.wait_ns));  // O_1 is complete too
        if (!ok) break;
        ptx::tc_fence_after();
        ++joins;
        const float2 o = *ml;
        const float top = max3_nan(m, o.x, o.x), tc = top == -INFINITY ? 0.f : top * c;
        f0 = ex2(fmaf(m, c, -tc));
        f1 = ex2(fmaf(o.x, c, -tc));
        l = f0 * l + f1 * o.y;
        m = top;
        const float inv = !scaled ? 1.f : seen > 0 ? 1.f / l : 0.f;
        f0 *= inv;
        f1 *= inv;
      }
      float bad = 0.f;
#pragma unroll 1
      for (int i = 0; i < D; i += 32) {  // (unrolled, its registers would spill into the key loop)
        uint32_t o[32];
        if (n > 0) {
          ptx::tmem_ld_32x32b_x32(t_o + i, o);
          ptx::tmem_wait_ld_of(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f0);
          if (shared) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t u[16];
              ptx::tmem_ld_32x32b_x16(t_o + D + i + h * 16, u);
              ptx::tmem_wait_ld_of(u);
#pragma unroll
              for (int e = 0; e < 16; ++e)
                o[h * 16 + e] = __float_as_uint(fmaf(f1, __uint_as_float(u[e]), __uint_as_float(o[h * 16 + e])));
            }
          }
        }
        if (n == 0 || (it.slot < 0 && seen == 0)) {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        if (live && it.slot < 0) {
          uint32_t w[16];
          float2 not_finite[2] = {};  // NaN as soon as one value is not finite
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 a = make_float2(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
            not_finite[e & 1] = __ffma2_rn(a, make_float2(0.f, 0.f), not_finite[e & 1]);
            w[e] = E::pack(a.x, a.y);
          }
          bad += (not_finite[0].x + not_finite[0].y) + (not_finite[1].x + not_finite[1].y);
          store64(dst + i, w, p.wide_out);
        } else if (live) {
          store64(part + i, reinterpret_cast<const uint32_t(&)[16]>(o[0]), true);
          store64(part + i + 16, reinterpret_cast<const uint32_t(&)[16]>(o[16]), true);
        }
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (n > 0 && lane == 0) {
        ptx::mbar_arrive(&bars->o_free[t]);
        if (shared) ptx::mbar_arrive(&bars->o_free[1]);
      }
      if (it.slot >= 0) {
        if (live) p.part_ml[at] = make_float2(m, l);
      } else {
        uint32_t again = __ballot_sync(0xffffffffu, bad != 0.f);
        while (again != 0) {  // rare: a result that is not finite
          const int src = __ffs(again) - 1;
          again &= again - 1;
          store_row_by_definition<T, D>(p, it.q_row, it.lq, it.k_row, it.lk, __shfl_sync(0xffffffffu, pos, src),
                                        __shfl_sync(0xffffffffu, head, src));
        }
      }
      jobs.done();
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// Joins the partial rows of split items: weights 2^(c m_s - c m) of the splits, one warp a row.
template <typename T, int D>
__global__ void __launch_bounds__(256) combine_kernel(const Params p) {
  using E = ElemOps<T>;
  constexpr int PER = D / 32;
  ptx::grid_wait();
  const int lane = threadIdx.x & 31;
  const int rows = p.header->split_rows;  // (few where single tokens of long sequences are split, whatever rows_cap)
  const long long total = (long long)p.header->n_splits * p.kv_heads * rows;
  for (long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); w < total; w += (long long)gridDim.x * 8) {
    const int row = int(w % rows);
    const int hk = int(w / rows % p.kv_heads);
    const SplitItem it = p.splits[w / rows / p.kv_heads];
    const int pos = it.pos + row / p.group, head = hk * p.group + row % p.group;
    if (pos >= it.lq) continue;
    // 32 splits at a time: a lane has one's reference and sum, every lane its columns of all of them
    float m = -INFINITY, l = 0.f, acc[PER] = {};
    for (int s0 = 0; s0 < it.n; s0 += 32) {
      const int count = min(32, it.n - s0);
      const long long first = ((long long)(it.slot + s0) * p.kv_heads + hk) * p.rows_cap + row;
      const long long step = (long long)p.kv_heads * p.rows_cap;
      const float2 ml = lane < count ? p.part_ml[first + lane * step] : make_float2(-INFINITY, 0.f);
      float top = max3_nan(m, ml.x, ml.x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float u = __shfl_xor_sync(0xffffffffu, top, o);
        top = max3_nan(top, u, u);
      }
      const float tc = top == -INFINITY ? 0.f : top * p.scale_log2;
      const float old = ex2(fmaf(m, p.scale_log2, -tc)), f = ex2(fmaf(ml.x, p.scale_log2, -tc));
      m = top;
      l = fmaf(l, old, ptx::warp_sum(f * ml.y));
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[i] *= old;
#pragma unroll 8
      for (int s = 0; s < count; ++s) {
        const float fs = __shfl_sync(0xffffffffu, f, s);
        const float* src = p.part_o + (first + s * step) * D + lane * PER;
#pragma unroll
        for (int i = 0; i < PER; i += 2) {
          const float2 v = *reinterpret_cast<const float2*>(src + i);
          acc[i] = fmaf(fs, v.x, acc[i]);
          acc[i + 1] = fmaf(fs, v.y, acc[i + 1]);
        }
      }
    }
    const int seen = seen_keys(pos, it.lq, it.lk, p.causal);
    const float inv = seen > 0 ? 1.f / l : 0.f;
    float bad = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      acc[i] = seen > 0 ? acc[i] * inv : 0.f;
      bad = fmaf(acc[i], 0.f, bad);
    }
    if (__any_sync(0xffffffffu, bad != 0.f)) row_by_definition<T, D>(p, it.q_row, it.lq, it.k_row, it.lk, pos, head, acc);
    uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + (long long)(it.q_row + pos) * p.ldo + head * D + lane * PER);
#pragma unroll
    for (int i = 0; i < PER / 2; ++i) dst[i] = E::pack(acc[2 * i], acc[2 * i + 1]);
  }
}

// ------------------------------------------------------------------------------------- host

// 16-bit tensor map with 128-byte swizzled boxes of 64 columns.
gdc_status encode(CUtensorMap* map, bool bf16, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                  const cuuint32_t* box) {
  auto fn = get_encode_fn();
  if (!fn) return set_error(GDC_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r =
      fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, cuuint32_t(rank), const_cast<void*>(base), dims,
         strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(GDC_ERR_CUDA, "cuTensorMapEncodeTiled (packed attention) failed (%d)", int(r));
  return GDC_OK;
}

template <typename T, int D>
gdc_status launch_typed(const PackedAttentionArgs& a, cudaStream_t stream, int* err) {
  using S = Shape<D>;
  constexpr bool bf16 = ElemOps<T>::kMmaFormat == 1;
  int dev = 0;
  GDC_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return set_error(GDC_ERR_CUDA, "device ordinal out of range");
  const PlanLayout l = plan_layout(a.batch, a.q_rows, a.k_rows, a.heads, a.kv_heads, D);
  const int sms = device_sm_count(dev);
  const int group = a.heads / a.kv_heads, tile_pos = kKeys / group;

  CUtensorMap tq, tk, tv;
  {
    const cuuint64_t dims[3] = {D, cuuint64_t(a.heads), cuuint64_t(a.q_rows)};
    const cuuint64_t strides[2] = {D * 2, cuuint64_t(a.ldq) * 2};
    const cuuint32_t box[3] = {64, cuuint32_t(group), cuuint32_t(tile_pos)};
    GDC_TRY(encode(&tq, bf16, a.q, 3, dims, strides, box));
  }
  // without keys nothing is loaded; the maps then describe the queries
  const bool keys = a.k_rows > 0;
  for (int i = 0; i < 2; ++i) {
    const cuuint64_t dims[2] = {cuuint64_t(keys ? a.kv_heads : a.heads) * D, cuuint64_t(keys ? a.k_rows : a.q_rows)};
    const cuuint64_t strides[1] = {cuuint64_t(keys ? (i ? a.ldv : a.ldk) : a.ldq) * 2};
    const cuuint32_t box[2] = {64, kKeys};
    GDC_TRY(encode(i ? &tv : &tk, bf16, keys ? (i ? a.v : a.k) : a.q, 2, dims, strides, box));
  }
  Params p{};
  p.q = a.q;
  p.k = a.k;
  p.v = a.v;
  p.out = a.out;
  p.ldq = a.ldq;
  p.ldk = a.ldk;
  p.ldv = a.ldv;
  p.ldo = a.ldo;
  p.q_off = a.q_off;
  p.k_off = a.k_off;
  p.batch = a.batch;
  p.q_rows = int(a.q_rows);
  p.k_rows = int(a.k_rows);
  p.heads = a.heads;
  p.kv_heads = a.kv_heads;
  p.dim = D;
  p.group = group;
  p.tile_pos = tile_pos;
  p.causal = a.causal;
  p.scale = a.scale;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.header = reinterpret_cast<PlanHeader*>(a.workspace);
  p.items = reinterpret_cast<Item*>(a.workspace + l.items_at);
  p.splits = reinterpret_cast<SplitItem*>(a.workspace + l.splits_at);
  p.part_o = reinterpret_cast<float*>(a.workspace + l.part_o_at);
  p.part_ml = reinterpret_cast<float2*>(a.workspace + l.part_ml_at);
  p.rows_cap = l.rows_cap;
  p.chunks_cap = l.chunks_cap;
  p.items_ub = l.items_ub;
  p.can_split = l.split;
  // A warp may have 32 rows to compute by their definition, 130 to 190 ns a key each, while others wait for it, and a
  // wait may see two such warps one after the other: 2 s would be over with 180,000 keys. A microsecond a key and row.
  p.wait_ns = ptx::kTimeoutNs + 64 * 1000ull * (unsigned long long)a.k_rows;
  p.err = err;
  p.wide_out = reinterpret_cast<uintptr_t>(a.out) % 32 == 0 && a.ldo % 16 == 0;

  static PerDeviceOnce configured;
  const cudaError_t ce = cudaError_t(per_device_once(configured, dev, [&] {
    const cudaError_t e = cudaFuncSetAttribute(packed_attention_kernel<T, D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmemBytes);
    return e != cudaSuccess ? e
                            : cudaFuncSetAttribute(packed_attention_kernel<T, D, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   S::kSmemBytes);
  }));
  if (ce != cudaSuccess) return set_error(GDC_ERR_CUDA, "packed attention smem attribute: %s", cudaGetErrorString(ce));
  const int64_t jobs = (l.planned || l.split ? l.chunks_cap : l.items_ub) * a.kv_heads;
  const unsigned grid = unsigned(l.planned || l.split ? std::min<int64_t>(sms, jobs) : jobs);
  if (l.planned) {
    GDC_CUDA_TRY(launch_overlapped(plan_kernel, 1, kPlanThreads, 0, 1, stream, p));
    GDC_CUDA_TRY(launch_overlapped(packed_attention_kernel<T, D, true>, grid, kThreads, S::kSmemBytes, 1, stream, tq, tk, tv, p));
  } else {
    GDC_CUDA_TRY(launch_overlapped(packed_attention_kernel<T, D, false>, grid, kThreads, S::kSmemBytes, 1, stream, tq, tk, tv, p));
  }
  if (l.split) {
    const int64_t rows = l.items_ub * a.kv_heads * l.rows_cap;
    GDC_CUDA_TRY(launch_overlapped(combine_kernel<T, D>, unsigned(std::min<int64_t>(4 * sms, (rows + 7) / 8)), 256, 0, 1, stream, p));
  }
  return GDC_OK;
}

}  // namespace

size_t packed_attention_workspace(int batch, int64_t q_rows, int64_t k_rows, int heads, int kv_heads, int dim) {
  if (batch <= 0 || q_rows <= 0) return 0;
  return plan_layout(batch, q_rows, k_rows, heads, kv_heads, dim).bytes;
}

gdc_status launch_packed_attention(Elem t, const PackedAttentionArgs& a, cudaStream_t stream, int* err) {
  if (t == Elem::kF16)
    return a.dim == 64 ? launch_typed<__half, 64>(a, stream, err) : launch_typed<__half, 128>(a, stream, err);
  return a.dim == 64 ? launch_typed<__nv_bfloat16, 64>(a, stream, err) : launch_typed<__nv_bfloat16, 128>(a, stream, err);
}

}  // namespace gdc
