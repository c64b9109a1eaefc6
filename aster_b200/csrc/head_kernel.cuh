// The products behind the loss of a language model's head, z = x . w^T with x [tokens, hidden] and
// w [vocab, hidden], as one persistent tcgen05 kernel with three endings:
//
//   kStats    a tile of z becomes, per row, its maximum and its sum of exponentials (one pass, running
//             rescale), the logits at the row's labels, and (label smoothing) its plain sum.  Nothing of
//             size tokens x vocab leaves the SM.
//   kGrad     the same tile of z, computed again, becomes a 16-bit tile of
//             G = dL/dz = c_t (softmax - labels), the only thing of that shape that is ever stored,
//             and only for a range of the vocabulary at a time.
//   kProduct  two products in one launch, dX = G . W and dW = G^T . X (16-bit out, or fp32 partial
//             sums where the long axis is cut).
//
// Roles and pipeline are those of the GEMM kernel (producer warp, one MMA-issuing warp, four epilogue
// warps, a ring of 128-byte-swizzled stages, two accumulators in TMEM); CG = 2 runs CTA pairs on 256-row
// tiles.  What differs: the tile width `bn` is a run-time number (the instruction descriptor carries
// it), so that a narrow problem can give every SM the same share of the vocabulary, and an operand may
// lie with its rows along K ("MN-major"): dX reads W and dW reads G and X as they lie in memory.  A
// stage of such an operand is a row of boxes [64 of K][64 columns], 8 KB each with the same swizzle; its
// descriptor has the 64-column groups 8192 bytes apart (leading offset) and the groups of 8 K rows 1024
// bytes apart (stride offset), and an MMA (16 of K) advances it by 2048 bytes.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "gemm_kernel.cuh"

namespace head {

using gemm::kBM;
using gemm::kRowBytes;

// Epilogue warps: one per quarter of the TMEM lanes; two, each with half of a tile's columns, where a tile has so
// few K blocks that its output decides (a warp's read of 64 columns takes 512 cycles, 16 bytes per cycle and
// quarter, which the other warp's arithmetic then fills).
constexpr int threads(int epilogue_warps) { return 64 + 32 * epilogue_warps; }
constexpr int kStageK = 64;            // elements of K per stage (16-bit operands, 128 bytes)
constexpr int kBoxBytes = 64 * kRowBytes;  // one box of an MN-major operand
constexpr int kMaxStages = 16;
constexpr int kMaxBn = 256;            // accumulator stride in TMEM
constexpr int kNoLabel = 0x7FFFFFFF;

enum Mode : int { kStats = 0, kGrad = 1, kProduct = 2 };
// Codes of the status words, beside those of the GEMM kernel (status[1..2] = block, item).
constexpr int kStatusWords = 16;

// Division by a launch constant: floor(n / d) for 0 <= n, d < 2^31 as the high word of n 2 (floor(2^63 / d) + 1).
// (The excess of the factor over 2^63 / d is at most 1, so the product is off by less than n / 2^63 < 1 / d.)
struct FastDiv {
  uint64_t m;
  int d;
  __host__ __device__ static FastDiv of(int d) { return {(1ull << 63) / static_cast<uint64_t>(d) + 1u, d}; }
  __device__ __forceinline__ int div(int n) const { return static_cast<int>(__umul64hi(static_cast<uint64_t>(n) << 1, m)); }
};

struct Problem {
  int M, N;          // rows of A, rows of B (columns of the tile space)
  int num_kb;        // K blocks over the whole K
  int kb_per_split;  // K blocks of one part
  int splits;
  int m_blocks, n_blocks;
  int raster_group;
  int items;         // m_blocks * n_blocks * splits
  FastDiv tiles;     // m_blocks * n_blocks
  FastDiv span;      // raster_group * n_blocks
  FastDiv group;     // raster_group
  FastDiv last_group;  // m-blocks of the last raster group
  int a_mn, b_mn;    // operand lies with its rows along K
  int b_row0;        // first row of B in its tensor map
  int b_k0;          // first K coordinate of B in its tensor map
  uint32_t idesc;
  // kProduct
  void* out16;       // [M][ld], or null: fp32 partial sums
  int64_t ld;
  float* partial;    // [splits][M][N]
  int accumulate;    // partial sums are added to what an earlier launch left there
};

struct Params {
  Problem prob[2];
  int num_probs;
  int bn;            // tile width
  int am;            // rows of A per stage: 128, or 32 / 64 when M is no larger (one CTA, K-major)
  int stages;
  int extra_rounds;  // see Walk
  uint32_t* status;
  unsigned wait_limit_ms;  // 0 = gemm::kWaitTimeoutNs
  // labels: `top` entries per row in rising order of their ids (top = 1: the target itself)
  int tokens, vocab;
  int col0;          // first column of the vocabulary in this launch (kGrad)
  int top;
  const void* target;      // cross entropy: int64 or int32
  int target64;
  long long ignore_index;
  const int32_t* ids;      // distillation: sorted, kNoLabel at the end
  const float* probs;      // distillation: their probabilities
  float label_prob;        // cross entropy: 1 - smoothing
  float scale2;            // log2(e) / temperature
  // kStats
  float2* part;            // [n_blocks][tokens]: maximum (times scale2) and sum of 2^(z scale2 - maximum)
  float* part_z;           // [n_blocks][tokens] sums of z, or null
  float* label_z;          // [tokens][top]
  uint32_t* ticket;        // cleared for the reduction that follows
  // kGrad
  const float* lse;        // [tokens]
  const float* coef;       // [tokens] row factors; null: `coef_top` for every row that has a loss
  float coef_top;
  const float* weight;     // distillation: [tokens] 1, 0 (no loss) or NaN
  float base;              // smoothing / vocab
  void* g;                 // [tokens][g_ld]
  int64_t g_ld;
  // kProduct
  const float* unscale;    // one factor on everything; null: *share * *grad_loss * unscale_factor
  const float* share;
  const float* grad_loss;
  float unscale_factor;
};

__host__ __device__ constexpr int stage_bytes(int bn, int cg, int am) { return (am + bn / cg) * kRowBytes; }
// Bytes behind the last stage that the MMA's 128-row read of a short A tile still touches.
__host__ __device__ constexpr int overrun_bytes(int bn, int cg, int am) {
  return kBM * kRowBytes > stage_bytes(bn, cg, am) ? kBM * kRowBytes - stage_bytes(bn, cg, am) : 0;
}
constexpr int kBarrierBytes = 384;
// 4 KB per epilogue warp in which 32 rows x 128 bytes of output are turned around (a lane per row writes them,
// eight lanes per row read them), so that they leave as whole lines.
constexpr int kTurnBytes = 32 * 128;
__host__ __device__ constexpr int smem_bytes(int bn, int stages, int cg, int am, int epilogue_warps) {
  return stages * stage_bytes(bn, cg, am) + epilogue_warps * kTurnBytes + overrun_bytes(bn, cg, am) + kBarrierBytes + 1024;
}

// 2^x for the softmax: the hardware's approximation (2 ulp) with results below 2^-126 flushed; the
// largest term of a sum is 2^0.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Has a bounded wait given up since the status words were last read?  What it left out is then missing from the
// sums of the kernels that follow: their results are made NaN.
__device__ __forceinline__ bool wait_lost(const uint32_t* status) { return *reinterpret_cast<const volatile uint32_t*>(status) != gemm::kStatusOk; }

// Four MMAs of one stage; `a_step` / `b_step` advance an operand's descriptor by 16 elements of K.
#define B200_HEAD_STAGE_ASM(GROUP)                                                              \
  asm volatile(                                                                                 \
      "{\n"                                                                                     \
      ".reg .pred p, q;\n"                                                                      \
      ".reg .b64 da, db;\n"                                                                     \
      ".reg .b32 la, lb;\n"                                                                     \
      "setp.ne.b32 p, %5, 0;\n"                                                                 \
      "setp.eq.b32 q, 0, 0;\n"                                                                  \
      "mov.b64 da, {%1, %3};\n"                                                                 \
      "mov.b64 db, {%2, %3};\n"                                                                 \
      "tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], da, db, %4, p;\n"                       \
      "add.u32 la, %1, %6;\n"                                                                   \
      "add.u32 lb, %2, %7;\n"                                                                   \
      "mov.b64 da, {la, %3};\n"                                                                 \
      "mov.b64 db, {lb, %3};\n"                                                                 \
      "tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], da, db, %4, q;\n"                       \
      "add.u32 la, la, %6;\n"                                                                   \
      "add.u32 lb, lb, %7;\n"                                                                   \
      "mov.b64 da, {la, %3};\n"                                                                 \
      "mov.b64 db, {lb, %3};\n"                                                                 \
      "tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], da, db, %4, q;\n"                       \
      "add.u32 la, la, %6;\n"                                                                   \
      "add.u32 lb, lb, %7;\n"                                                                   \
      "mov.b64 da, {la, %3};\n"                                                                 \
      "mov.b64 db, {lb, %3};\n"                                                                 \
      "tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], da, db, %4, q;\n"                       \
      "}\n" ::"r"(tmem_d),                                                                      \
      "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate_first), "r"(a_step), "r"(b_step) \
      : "memory")

template <int CG>
__device__ __forceinline__ void mma_stage(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc,
                                          uint32_t accumulate_first, uint32_t a_step, uint32_t b_step) {
  if constexpr (CG == 1) {
    B200_HEAD_STAGE_ASM("1");
  } else {
    B200_HEAD_STAGE_ASM("2");
  }
}
#undef B200_HEAD_STAGE_ASM

// Low word of a descriptor: start address, leading offset (64-column groups of an MN-major operand).
__device__ __forceinline__ uint32_t desc_lo(uint32_t smem_addr, int mn) {
  return ((smem_addr >> 4) & 0x3FFFu) | ((mn ? static_cast<uint32_t>(kBoxBytes >> 4) : 1u) << 16);
}

// The items of a unit (CTA or pair), one after the other, -1 at the end.  Items of problem 0 (the longer ones)
// are dealt round-robin; the units that got one fewer then take `extra_rounds` items of problem 1 more, which
// is how many of them take as long as one of problem 0, and the rest is dealt round-robin again.
struct Walk {
  int at, step;       // next item of the current phase
  int left;           // items left in it
  int extra_at, extra_step, extra_left;
  int rest_at, units, total;

  __device__ __forceinline__ Walk(const Params& p, int unit, int n_units) {
    const int items0 = p.prob[0].items;
    const int rem = items0 % n_units;
    units = n_units;
    total = items0 + (p.num_probs > 1 ? p.prob[1].items : 0);
    at = unit;
    step = n_units;
    left = items0 / n_units + (unit < rem ? 1 : 0);
    const int extra = rem != 0 ? p.extra_rounds : 0;
    extra_at = items0 + unit - rem;
    extra_step = n_units - rem;
    extra_left = rem != 0 && unit >= rem ? extra : 0;
    rest_at = items0 + extra * (n_units - rem) + unit;
  }
  __device__ __forceinline__ int next() {
    if (left == 0) {
      if (extra_left > 0) {
        at = extra_at;
        step = extra_step;
        left = extra_left;
        extra_left = 0;
      } else {
        at = rest_at;
        step = units;
        left = 0x7FFFFFFF;
      }
    }
    --left;
    const int item = at;
    if (item >= total) {
      left = 1;  // stays behind the end
      return -1;
    }
    at += step;
    return item;
  }
};

struct Item {
  int prob, m_blk, n_blk, split, kb0, nkb;
};

__device__ __forceinline__ Item decode(const Params& p, int item) {
  Item w;
  w.prob = item >= p.prob[0].items ? 1 : 0;
  const Problem& q = p.prob[w.prob];
  int t = w.prob ? item - p.prob[0].items : item;
  w.split = q.splits > 1 ? q.tiles.div(t) : 0;
  t -= w.split * q.tiles.d;
  const int group = q.span.div(t);
  const int first = group * q.raster_group;
  const int in_group = t - group * q.span.d;
  const FastDiv& rows = first + q.raster_group <= q.m_blocks ? q.group : q.last_group;
  w.n_blk = rows.div(in_group);
  w.m_blk = first + in_group - w.n_blk * rows.d;
  w.kb0 = w.split * q.kb_per_split;
  w.nkb = min(q.kb_per_split, q.num_kb - w.kb0);
  return w;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A warp's 32 rows x 128 bytes on their way from a lane per row to whole lines: lane l writes row l (16-byte
// piece j at position j ^ (l % 8)) and reads pieces of rows 4 i + l / 8, piece l % 8, for i = 0..7.
struct TurnAround {
  uint32_t buf;

  __device__ __forceinline__ uint32_t piece(uint32_t row, uint32_t j) const { return buf + row * 128u + ((j ^ (row & 7u)) << 4); }
  // Pieces [first, first + N / 4) of this lane's row.  The first call of a round waits for the previous round's reads.
  template <int N>
  __device__ __forceinline__ void put(int first, const uint32_t (&w)[N]) const {
    const uint32_t lane = threadIdx.x & 31;
    if (first == 0) __syncwarp();
#pragma unroll
    for (int j = 0; j < N / 4; ++j) sm100::st_shared_u4(piece(lane, first + j), w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
  }
  // Element `at` (16 bits) of this lane's row, after its piece has been put.
  __device__ __forceinline__ void patch16(int at, uint32_t bits) const {
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(piece(threadIdx.x & 31, at >> 3) + 2u * (at & 7)), "h"(static_cast<unsigned short>(bits)) : "memory");
  }
  // Element `at` (32 bits) of this lane's row.
  __device__ __forceinline__ float own32(int at) const {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(piece(threadIdx.x & 31, at >> 2) + 4u * (at & 3)) : "memory");
    return v;
  }
  template <typename Use>
  __device__ __forceinline__ void get(Use use) const {
    const uint32_t lane = threadIdx.x & 31;
    __syncwarp();
    uint4 t[8];  // all reads before the first use: their latencies overlap
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = sm100::ld_shared_u4(piece(4u * i + (lane >> 3), lane & 7u));
#pragma unroll
    for (int i = 0; i < 8; ++i) use(i, t[i]);
  }
};

// x[at] by halving: five selects deep.
__device__ __forceinline__ float pick(const float (&x)[32], int at) {
  float a[16], b[8], c[4];
#pragma unroll
  for (int j = 0; j < 16; ++j) a[j] = at & 16 ? x[j + 16] : x[j];
#pragma unroll
  for (int j = 0; j < 8; ++j) b[j] = at & 8 ? a[j + 8] : a[j];
#pragma unroll
  for (int j = 0; j < 4; ++j) c[j] = at & 4 ? b[j + 4] : b[j];
  const float d = at & 2 ? c[2] : c[0], e = at & 2 ? c[3] : c[1];
  return at & 1 ? e : d;
}

// A row's labels during the walk over a tile's columns, in rising order.  The entry behind the next one is
// fetched ahead: the lists of a tile's rows do not fit what the ring leaves of the L1, and a label should not
// wait for the L2.
struct Labels {
  const int32_t* ids;  // null: one label (cross entropy)
  const float* probs;
  int top, at;
  int next, ahead;     // the next label's column and the one behind it, kNoLabel: none left
  float prob, prob_ahead;

  __device__ __forceinline__ void fetch_ahead() {
    const bool more = at + 1 < top;
    ahead = more ? __ldg(ids + at + 1) : kNoLabel;
    prob_ahead = more ? __ldg(probs + at + 1) : 0.0f;
  }
  __device__ __forceinline__ void start() {
    next = at < top ? __ldg(ids + at) : kNoLabel;
    prob = at < top ? __ldg(probs + at) : 0.0f;
    fetch_ahead();
  }
  __device__ __forceinline__ void advance() {
    ++at;
    next = ahead;
    prob = prob_ahead;
    if (ids != nullptr) fetch_ahead();
  }
};

// The class of cross entropy's row, or kNoLabel (ignored, or outside the vocabulary).
__device__ __forceinline__ int target_class(const Params& p, int row) {
  const long long t = p.target64 ? __ldg(static_cast<const long long*>(p.target) + row) : static_cast<long long>(__ldg(static_cast<const int*>(p.target) + row));
  return t != p.ignore_index && t >= 0 && t < p.vocab ? static_cast<int>(t) : kNoLabel;
}

// 1 for a row with a loss, 0 for one without, NaN for one with a bad label.
__device__ __forceinline__ float row_weight(const Params& p, int row) {
  if (p.weight != nullptr) return __ldg(p.weight + row);
  const long long t = p.target64 ? __ldg(static_cast<const long long*>(p.target) + row) : static_cast<long long>(__ldg(static_cast<const int*>(p.target) + row));
  return t == p.ignore_index ? 0.0f : (t >= 0 && t < p.vocab ? 1.0f : NAN);
}

// Labels of `row` from column `col` on.
__device__ __forceinline__ Labels labels_from(const Params& p, int row, bool row_ok, int col) {
  Labels l;
  l.ids = nullptr;
  l.probs = nullptr;
  l.top = p.top;
  l.at = 0;
  l.next = l.ahead = kNoLabel;
  l.prob = p.label_prob;
  l.prob_ahead = 0.0f;
  if (!row_ok) return l;
  if (p.ids == nullptr) {
    const int t = target_class(p, row);
    if (t >= col) l.next = t;
    return l;
  }
  l.ids = p.ids + static_cast<size_t>(row) * p.top;
  l.probs = p.probs + static_cast<size_t>(row) * p.top;
  // First entry at or behind `col`, by eighths: the eight probes of a round are independent loads, so that 64
  // entries take two trips to the L2 instead of six.
  int lo = 0, n = p.top;
  while (n > 0) {
    const int step = (n + 7) >> 3, end = lo + n;
    int below = 0;
#pragma unroll
    for (int i = 1; i <= 8; ++i) {
      const int at = lo + i * step - 1;
      below += at < end && __ldg(l.ids + at) < col ? 1 : 0;
    }
    lo += below * step;  // the last entry of the next eighth is at or behind `col`
    lo = min(lo, end);
    n = min(step - 1, end - lo);
  }
  l.at = lo;
  l.start();
  return l;
}

// T16: the 16-bit type of the operands, of G and of the gradients.  EW: epilogue warps, 4 or (kProduct) 8.
template <int CG, int MODE, typename T16, int EW>
__global__ void __launch_bounds__(threads(EW), 1)
head_kernel(const __grid_constant__ CUtensorMap map_a0, const __grid_constant__ CUtensorMap map_b0, const __grid_constant__ CUtensorMap map_a1,
            const __grid_constant__ CUtensorMap map_b1, const __grid_constant__ Params p) {
#if defined(__CUDA_ARCH_FEAT_SM100_ALL)
  using namespace sm100;
  static_assert(EW == 4 || (EW == 8 && MODE == kProduct), "a second epilogue warp per quarter: products only");
  constexpr int kTileM = kBM * CG;
  constexpr uint32_t kTmemCols = 2 * kMaxBn;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_raw_u32 = smem_u32(smem_raw);
  const uint32_t smem_base = (smem_raw_u32 + 1023u) & ~1023u;
  const uint32_t a_bytes = static_cast<uint32_t>(p.am) * kRowBytes;
  const uint32_t b_rows = static_cast<uint32_t>(p.bn) / CG;
  const uint32_t b_bytes = b_rows * kRowBytes;
  const uint32_t st_bytes = a_bytes + b_bytes;
  // (what a short A stage's 128-row read touches behind the ring is the turn-around buffers, and what follows them)
  [[maybe_unused]] const uint32_t turn_base = smem_base + static_cast<uint32_t>(p.stages) * st_bytes;
  const uint32_t bar_base = turn_base + EW * kTurnBytes + static_cast<uint32_t>(overrun_bytes(p.bn, CG, p.am));
  uint8_t* bar_ptr = smem_raw + (bar_base - smem_raw_u32);
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 128u + 8u * s; };
  auto acc_full_bar = [&](int a) { return bar_base + 256u + 8u * a; };
  auto acc_empty_bar = [&](int a) { return bar_base + 272u + 8u * a; };
  const uint32_t drain_bar = bar_base + 288u;
  const uint32_t tmem_slot = bar_base + 296u;
  volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(bar_ptr + 296);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(bar_ptr + 300);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const gemm::Waiter waiter{abort_flag, p.status, p.wait_limit_ms != 0 ? p.wait_limit_ms * 1000000ull : gemm::kWaitTimeoutNs};
  const uint32_t cta_rank = CG == 2 ? cluster_ctarank() : 0u;
  const bool leader = cta_rank == 0u;
  const int unit = static_cast<int>(blockIdx.x) / CG;
  const int units = static_cast<int>(gridDim.x) / CG;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(acc_full_bar(a), 1);
      mbar_init(acc_empty_bar(a), EW * CG);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0u;
    fence_barrier_init();
    fence_proxy_async_smem();
    prefetch_tensormap(&map_a0);
    prefetch_tensormap(&map_b0);
    if constexpr (MODE == kProduct) {
      prefetch_tensormap(&map_a1);
      prefetch_tensormap(&map_b1);
    }
  }
  if (warp == 1) tmem_alloc<CG>(tmem_slot, kTmemCols);
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot_ptr;
  griddep_launch_dependents();
  griddep_wait();  // global memory from here on
  if constexpr (MODE == kStats) {
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.ticket = 0u;
  }

  if (warp == 0) {
    // ------------------------------- producer -------------------------------
    int stage = 0;
    uint32_t phase = 0;
    long long issued = 0;
    bool ok = true;
    for (Walk walk(p, unit, units); ok;) {
      const int item = walk.next();
      if (item < 0) break;
      const Item w = decode(p, item);
      const Problem& q = p.prob[w.prob];
      const CUtensorMap* ma = MODE == kProduct && w.prob ? &map_a1 : &map_a0;
      const CUtensorMap* mb = MODE == kProduct && w.prob ? &map_b1 : &map_b0;
      const bool a_mn = MODE == kProduct && q.a_mn != 0;
      const bool b_mn = MODE == kProduct && q.b_mn != 0;
      const int a_row = w.m_blk * kTileM + static_cast<int>(cta_rank) * kBM;
      const int b_row = q.b_row0 + w.n_blk * p.bn + static_cast<int>(cta_rank * b_rows);
      for (int kb = 0; kb < w.nkb; ++kb) {
        if (!waiter.wait(empty_bar(stage), phase ^ 1u, gemm::kStatusProducerEmptyWait, item, kb)) {
          ok = false;
          break;
        }
        if (elect_one()) {
          const uint32_t a_dst = smem_base + static_cast<uint32_t>(stage) * st_bytes;
          const uint32_t b_dst = a_dst + a_bytes;
          const int ka = (w.kb0 + kb) * kStageK;
          const int kbq = q.b_k0 + (w.kb0 + kb) * kStageK;
          uint32_t bar = full_bar(stage);
          if constexpr (CG == 1) {
            mbar_arrive_expect_tx(bar, st_bytes);
          } else {
            if (leader) mbar_arrive_expect_tx(bar, 2u * st_bytes);
            bar = map_to_cta(bar, 0u);
          }
          auto load = [&](uint32_t dst, const CUtensorMap* m, int c0, int c1) {
            if constexpr (CG == 1) {
              tma_load_2d(dst, m, bar, c0, c1);
            } else {
              tma_load_2d_pair(dst, m, bar, c0, c1);
            }
          };
          if (a_mn) {
#pragma unroll
            for (int b = 0; b < kBM / 64; ++b) load(a_dst + b * kBoxBytes, ma, a_row + b * 64, ka);
          } else {
            load(a_dst, ma, ka, a_row);
          }
          if (b_mn) {
            for (uint32_t b = 0; b < b_rows / 64u; ++b) load(b_dst + b * kBoxBytes, mb, b_row + static_cast<int>(b) * 64, kbq);
          } else {
            load(b_dst, mb, kbq, b_row);
          }
        }
        __syncwarp();
        ++issued;
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (!ok && leader) {
      // Aborting: let the copies already issued land before the CTA may exit.
      for (int s = 0; s < p.stages; ++s) {
        if (issued > s) {
          const long long last = (issued - 1) - ((issued - 1 - s) % p.stages);
          waiter.wait(full_bar(s), static_cast<uint32_t>((last / p.stages) & 1), 0u, 0, 0, gemm::kDrainTimeoutNs);
        }
      }
    } else if (!ok) {
      waiter.settle();
    }
  } else if (warp == 1) {
    // ------------------------------- MMA issuer (leader CTA only) -------------------------------
    if (leader) {
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      const uint32_t desc_hi = smem_desc_hi_sw128();
      const uint32_t peer_delta = CG == 2 ? map_to_cta(bar_base, 1u) - bar_base : 0u;
      for (Walk walk(p, unit, units); ok;) {
        const int item = walk.next();
        if (item < 0) break;
        const Item w = decode(p, item);
        const Problem& q = p.prob[w.prob];
        const int a_mn = MODE == kProduct ? q.a_mn : 0;
        const int b_mn = MODE == kProduct ? q.b_mn : 0;
        const uint32_t a_step = a_mn ? 128u : 2u;
        const uint32_t b_step = b_mn ? 128u : 2u;
        const uint32_t idesc = q.idesc;
        if (!waiter.wait(acc_empty_bar(acc), acc_phase ^ 1u, gemm::kStatusMmaAccEmptyWait, item, 0)) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(acc * kMaxBn);
        uint32_t a_lo = desc_lo(smem_base + static_cast<uint32_t>(stage) * st_bytes, a_mn);
        uint32_t b_lo = desc_lo(smem_base + static_cast<uint32_t>(stage) * st_bytes + a_bytes, b_mn);
        for (int kb = 0; kb < w.nkb; ++kb) {
          if (!waiter.wait(full_bar(stage), phase, gemm::kStatusMmaFullWait, item, kb)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          if (elect_one()) {
            mma_stage<CG>(tmem_d, a_lo, b_lo, desc_hi, idesc, kb != 0 ? 1u : 0u, a_step, b_step);
            umma_commit<CG>(empty_bar(stage));
            if constexpr (CG == 2) umma_commit<CG>(empty_bar(stage) + peer_delta);
          }
          __syncwarp();
          a_lo += st_bytes >> 4;
          b_lo += st_bytes >> 4;
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
            a_lo = desc_lo(smem_base, a_mn);
            b_lo = desc_lo(smem_base + a_bytes, b_mn);
          }
        }
        if (!ok) break;
        if (elect_one()) {
          umma_commit<CG>(acc_full_bar(acc));
          if constexpr (CG == 2) umma_commit<CG>(acc_full_bar(acc) + peer_delta);
        }
        __syncwarp();
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
      if (!ok) {
        // Aborting: wait for the MMAs already issued before TMEM and shared memory go away.
        if (elect_one()) umma_commit<CG>(drain_bar);
        __syncwarp();
        waiter.wait(drain_bar, 0u, 0u, 0, 0, gemm::kDrainTimeoutNs);
      }
    }
  } else {
    // ------------------------------- epilogue -------------------------------
    const int quarter = warp & 3;
    [[maybe_unused]] const TurnAround turn{turn_base + static_cast<uint32_t>(warp - 2) * kTurnBytes};
    const int row_in_tile = static_cast<int>(cta_rank) * kBM + quarter * 32 + lane;
    float unscale = 1.0f;
    if constexpr (MODE == kProduct) {
      unscale = p.unscale != nullptr ? __ldg(p.unscale) : __ldg(p.share) * __ldg(p.grad_loss) * p.unscale_factor;
      if (wait_lost(p.status)) unscale = NAN;  // z or G are not what they should be
    }
    int acc = 0;
    uint32_t acc_phase = 0;
    for (Walk walk(p, unit, units);;) {
      const int item = walk.next();
      if (item < 0) break;
      const Item w = decode(p, item);
      const Problem& q = p.prob[w.prob];
      const int row = w.m_blk * kTileM + row_in_tile;
      const bool row_ok = row < q.M;
      // What the row needs, and the search for the tile's first label, come while the tile's MMAs run.
      [[maybe_unused]] Labels l;
      if constexpr (MODE != kProduct) l = labels_from(p, row, row_ok, p.col0 + w.n_blk * p.bn);
      [[maybe_unused]] float coef = 0.0f, lse2 = 0.0f;
      if constexpr (MODE == kGrad) {
        if (row_ok) {
          coef = p.coef != nullptr ? __ldg(p.coef + row) : p.coef_top * row_weight(p, row);
          lse2 = __ldg(p.lse + row) * 1.4426950408889634f;
        }
      }
      if (!waiter.wait_relaxed(acc_full_bar(acc), acc_phase, gemm::kStatusEpilogueAccFullWait, item, w.nkb <= 4 ? 20u : 64u)) break;
      tc_fence_after_sync();
      const bool slab_ok = row - lane < q.M;  // does any of the warp's rows exist?
      const int tile_col = w.n_blk * p.bn;    // in the columns of this launch
      const int cols = min(p.bn, q.N - tile_col);
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * kMaxBn);
      if constexpr (MODE == kStats) {
        float m = -INFINITY, s = 0.0f, zsum = 0.0f;
#pragma unroll 1
        for (int c = 0; c < (slab_ok ? cols : 0); c += 32) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(taddr + static_cast<uint32_t>(c), v);
          tmem_ld_wait();
          float x[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] = __uint_as_float(v[j]);
          if (c + 32 > cols) {  // ragged edge: what lies beyond the vocabulary adds nothing
            if (p.part_z != nullptr) {
#pragma unroll
              for (int j = 0; j < 32; ++j) zsum += c + j < cols ? x[j] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] = c + j < cols ? x[j] : -INFINITY;
          } else if (p.part_z != nullptr) {
            float t = 0.0f;
#pragma unroll
            for (int j = 0; j < 32; ++j) t += x[j];
            zsum += t;
          }
          float cm = x[0];
#pragma unroll
          for (int j = 1; j < 32; ++j) cm = fmaxf(cm, x[j]);
          const float nm = fmaxf(m, cm);
          const float m2 = nm == -INFINITY ? 0.0f : nm * p.scale2;  // a row of minus infinities sums to 0
          float t0 = 0.0f, t1 = 0.0f;
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            t0 += ex2(fmaf(x[j], p.scale2, -m2));
            t1 += ex2(fmaf(x[j + 1], p.scale2, -m2));
          }
          s = fmaf(s, ex2(fmaf(m, p.scale2, -m2)), t0 + t1);
          m = nm;
          const int end = tile_col + c + 32;
          if (__any_sync(0xffffffffu, l.next < end)) {
            // Registers cannot be indexed: the lane's 32 logits go through its row of shared memory.
            uint32_t zs[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) zs[j] = __float_as_uint(x[j]);
            turn.put(0, zs);
            while (l.next < end) {
              p.label_z[static_cast<size_t>(row) * p.top + l.at] = turn.own32(l.next - (tile_col + c));
              l.advance();
            }
            __syncwarp();
          }
        }
        if (row_ok) {
          const size_t at = static_cast<size_t>(w.n_blk) * p.tokens + row;
          p.part[at] = make_float2(m * p.scale2, s);
          if (p.part_z != nullptr) p.part_z[at] = zsum;
        }
      } else if constexpr (MODE == kGrad) {
        const int vcol = p.col0 + tile_col;
        const float shift = coef * p.base;
        const int piece_row = row - lane + (lane >> 3), piece_col = (lane & 7) * 8;  // of every 4 rows, of every 64 columns
        T16* const dst = static_cast<T16*>(p.g) + static_cast<size_t>(piece_row) * p.g_ld + tile_col + piece_col;
#pragma unroll 1
        for (int c = 0; c < (slab_ok ? cols : 0); c += 64) {
          uint32_t v[64];
          tmem_ld_32x32b_x64(taddr + static_cast<uint32_t>(c), v);
          tmem_ld_wait();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] = fmaf(coef, ex2(fmaf(__uint_as_float(v[32 * h + j]), p.scale2, -lse2)), -shift);
            if (coef == 0.0f) {  // a row without a loss has no gradient, whatever its logits are
#pragma unroll
              for (int j = 0; j < 32; ++j) x[j] = 0.0f;
            }
            uint32_t out[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) out[j] = pack2<T16>(x[2 * j], x[2 * j + 1]);
            turn.put(4 * h, out);
            // The few entries at labels are taken out of the 32, corrected (an id may be listed more than once)
            // and written over the rounded ones: cheaper than touching all 32 for each of them (4096 x 1024 x 16384
            // with 64 labels per row: 159 -> 137 us; 105 with one label).
            const int col = vcol + c + 32 * h;
            const int end = c + 32 * h < cols ? col + 32 : 0;  // a tile may end after the first half
            while (__any_sync(0xffffffffu, l.next < end)) {
              if (l.next < end) {
                const int id = l.next;
                float g = pick(x, id - col);
                do {
                  g -= coef * l.prob;
                  l.advance();
                } while (l.next == id);
                turn.patch16(32 * h + id - col, pack2<T16>(g, 0.0f));
              }
              __syncwarp();
            }
          }
          // Rows of G are whole 64-column groups: what a piece writes behind the last column is never read.
          const bool col_ok = c + piece_col < cols;
          turn.get([&](int i, const uint4& t) {
            if (col_ok && piece_row + 4 * i < q.M) *reinterpret_cast<uint4*>(dst + static_cast<size_t>(4 * i) * p.g_ld + c) = t;
          });
        }
      } else {
        const int piece_row = row - lane + (lane >> 3);
        const int half = EW == 8 ? (warp - 2) >> 2 : 0;
        const int c_first = half * (kMaxBn / 2), c_end = !slab_ok ? 0 : (EW == 8 && half == 0 ? min(cols, kMaxBn / 2) : cols);
        if (q.out16 != nullptr) {
          const int piece_col = (lane & 7) * 8;
          T16* const dst = static_cast<T16*>(q.out16) + static_cast<size_t>(piece_row) * q.ld + tile_col + piece_col;
#pragma unroll 1
          for (int c = c_first; c < c_end; c += 64) {
            uint32_t v[64];
            tmem_ld_32x32b_x64(taddr + static_cast<uint32_t>(c), v);
            tmem_ld_wait();
            uint32_t out[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) out[j] = pack2<T16>(__uint_as_float(v[2 * j]) * unscale, __uint_as_float(v[2 * j + 1]) * unscale);
            const bool col_ok = c + piece_col < cols;  // the columns are a multiple of 8: a piece exists or does not
            turn.put(0, out);
            turn.get([&](int i, const uint4& t) {
              if (col_ok && piece_row + 4 * i < q.M) *reinterpret_cast<uint4*>(dst + static_cast<size_t>(4 * i) * q.ld + c) = t;
            });
          }
        } else {
          const int piece_col = (lane & 7) * 4;
          float* const dst = q.partial + (static_cast<size_t>(w.split) * q.M + piece_row) * q.N + tile_col + piece_col;
#pragma unroll 1
          for (int c = c_first; c < c_end; c += 32) {
            uint32_t v[32];
            tmem_ld_32x32b_x32(taddr + static_cast<uint32_t>(c), v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * unscale);
            const bool col_ok = c + piece_col < cols;
            turn.put(0, v);
            turn.get([&](int i, const uint4& t) {
              if (col_ok && piece_row + 4 * i < q.M) {
                float4* const d = reinterpret_cast<float4*>(dst + static_cast<size_t>(4 * i) * q.N + c);
                float4 f = make_float4(__uint_as_float(t.x), __uint_as_float(t.y), __uint_as_float(t.z), __uint_as_float(t.w));
                if (q.accumulate) {
                  const float4 o = *d;
                  f = make_float4(f.x + o.x, f.y + o.y, f.z + o.z, f.w + o.w);
                }
                *d = f;
              }
            });
          }
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 1) {
          mbar_arrive(acc_empty_bar(acc));
        } else {
          mbar_arrive_remote(map_to_cta(acc_empty_bar(acc), 0u));
        }
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
  }

  // ------------------------------- teardown -------------------------------
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc<CG>(tmem_base, kTmemCols);
  }
#endif
}

}  // namespace head
