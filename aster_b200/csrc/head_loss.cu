// Cross entropy and distillation of a language model's head (b200_head_loss_*): schedules of the three
// products in head_kernel.cuh and the small kernels between them.
//
// Forward:   [teacher rows: probabilities, sorted ids]  ->  kStats over z  ->  join the tiles' maxima and
//            sums per row, losses, their deterministic sum
// Backward:  row factors  ->  per range of the vocabulary: kGrad (z again, G in 16 bits), then dX += G . W
//            and dW = G^T . X in one launch  ->  [sum of dX's parts]
//
// 8 tokens*vocab*hidden operations instead of the 6 of a program that keeps z: recomputing z costs one
// product, keeping it would cost tokens*vocab*4 bytes for the whole time between the passes.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>

#include "common.h"
#include "head_kernel.cuh"

namespace {

using head::Params;
using head::Problem;

constexpr int kMaxTop = 1024;
constexpr int kSms = 148;
constexpr int kMaxSmem = 232448;
constexpr int64_t kGradBytes = 256ll << 20;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHalfTop = 8192.0f;  // largest row factor of fp16's dL/dz

__device__ uint32_t g_status[head::kStatusWords];

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// ---------------------------------------------------------------------------------------------
// small kernels
// ---------------------------------------------------------------------------------------------
// Sum, maximum over a block of 32-thread warps, the same value in all threads; `buf` holds 32 floats.
__device__ __forceinline__ float block_reduce(float v, bool max_op, float* buf) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (blockDim.x + 31) >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float t = __shfl_xor_sync(0xffffffffu, v, o);
    v = max_op ? fmaxf(v, t) : v + t;
  }
  __syncthreads();  // a previous call's reads of buf
  if (lane == 0) buf[warp] = v;
  __syncthreads();
  v = lane < warps ? buf[lane] : (max_op ? -INFINITY : 0.0f);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float t = __shfl_xor_sync(0xffffffffu, v, o);
    v = max_op ? fmaxf(v, t) : v + t;
  }
  return v;
}

__device__ __forceinline__ float load_float(const void* p, int dtype, size_t i) {
  if (dtype == B200_F32) return __ldg(static_cast<const float*>(p) + i);
  const unsigned short b = __ldg(static_cast<const unsigned short*>(p) + i);
  return dtype == B200_BF16 ? __uint_as_float(static_cast<uint32_t>(b) << 16) : __half2float(__ushort_as_half(b));
}

__device__ __forceinline__ long long load_index(const void* p, int bits, size_t i) {
  return bits == 64 ? __ldg(static_cast<const long long*>(p) + i) : static_cast<long long>(__ldg(static_cast<const int*>(p) + i));
}

// One block per row: the teacher's probabilities over its listed entries, sorted by id (a bitonic network over
// the next power of two `n`; the key's low half is the listing order, so that equal ids stay in it and no two
// keys are equal).  The temperature divides differences to the row's maximum, never the logits themselves: those
// may be as large as fp32 goes (masks of the type's lowest value), and minus infinity alone leaves an entry out.
__global__ void __launch_bounds__(kMaxTop / 2) teacher_kernel(const void* __restrict__ logits, int dtype, const void* __restrict__ ids_in, int bits, int top, int n,
                                                              int vocab, float inv_t, int32_t* __restrict__ ids, float* __restrict__ probs,
                                                              float* __restrict__ weight, float* __restrict__ neg_entropy) {
  extern __shared__ uint64_t key[];  // [n], then [n] floats: as little as the rows need, so that an SM holds 32 of them
  float* const s_t = reinterpret_cast<float*>(key + n);
  __shared__ float buf[32];
  const size_t row = blockIdx.x, base = row * top;
  sm100::griddep_launch_dependents();
  sm100::griddep_wait();
  float mx = -INFINITY;
  int any = 0, bad = 0;
  for (int j = threadIdx.x; j < n; j += blockDim.x) {
    uint32_t id32 = head::kNoLabel;
    if (j < top) {
      const long long id = load_index(ids_in, bits, base + j);
      float t = load_float(logits, dtype, base + j);
      const bool listed = id >= 0 && t != -INFINITY;
      if (listed) {
        any = 1;
        if (id >= vocab || !(t < INFINITY)) bad = 1;
        if (id < vocab) id32 = static_cast<uint32_t>(id);
        mx = fmaxf(mx, t);
      } else {
        t = -INFINITY;
      }
      s_t[j] = t;
    }
    key[j] = (static_cast<uint64_t>(id32) << 32) | static_cast<uint32_t>(j);
  }
  any = __syncthreads_or(any);
  bad = __syncthreads_or(bad);
  mx = block_reduce(mx, true, buf);
  float sum = 0.0f;
  for (int j = threadIdx.x; j < top; j += blockDim.x) sum += any ? expf((s_t[j] - mx) * inv_t) : 0.0f;
  sum = block_reduce(sum, false, buf);
  for (int size = 2; size <= n; size <<= 1) {
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      for (int i = threadIdx.x; i < n / 2; i += blockDim.x) {
        const int lo = ((i & ~(stride - 1)) << 1) | (i & (stride - 1)), hi = lo + stride;
        const uint64_t a = key[lo], b = key[hi];
        if ((a > b) == ((lo & size) == 0)) {
          key[lo] = b;
          key[hi] = a;
        }
      }
      __syncthreads();
    }
  }
  const float log_sum = logf(sum), inv = any ? 1.0f / sum : 0.0f;
  float ent = 0.0f;
  for (int place = threadIdx.x; place < top; place += blockDim.x) {
    const uint64_t k = key[place];
    const int32_t id = static_cast<int32_t>(k >> 32);
    const float d = (s_t[static_cast<uint32_t>(k)] - mx) * inv_t;
    const float p = id != head::kNoLabel ? expf(d) * inv : 0.0f;
    ids[base + place] = id;
    probs[base + place] = p;
    if (p > 0.0f) ent += p * (d - log_sum);
  }
  ent = block_reduce(ent, false, buf);
  if (threadIdx.x == 0) {
    weight[row] = !any ? 0.0f : (bad ? NAN : 1.0f);
    neg_entropy[row] = ent;
  }
}

struct JoinParams {
  const float2* part;
  const float* part_z;
  const float* label_z;
  const float* probs;        // distillation
  const int32_t* ids;
  const float* weight;
  const float* neg_entropy;
  const void* target;        // cross entropy
  int index_bits;
  long long ignore_index;
  int tokens, vocab, n_blocks, top, reduction;
  float smoothing, inv_t, row_scale;
  float* loss;
  float* lse;
  float* share;              // what a row's gradient is divided by, as a factor
  float2* block_sums;
  uint32_t* ticket;
  const uint32_t* status;
  struct {
    uint32_t* at;
    int words;
  } pad[4];                  // what lies between the parts of `saved`: it is an output, all of which is defined
};

// 8 rows per block of 8 warps.  A thread joins every 32nd tile of one row (8 lanes read 8 neighbouring rows
// of a tile, 64 bytes), then warp r finishes row r.  The last block to finish adds the blocks' sums in their
// order, so that a repeated call gives the same bits.
constexpr int kJoinRows = 8;
constexpr int kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const JoinParams p) {
  __shared__ float s_m[32][kJoinRows + 1], s_s[32][kJoinRows + 1], s_z[32][kJoinRows + 1];
  __shared__ float s_loss[kJoinRows], s_kept[kJoinRows];
  __shared__ uint32_t s_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  sm100::griddep_wait();
  const bool lost = head::wait_lost(p.status);
  if (blockIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (static_cast<int>(threadIdx.x) < p.pad[i].words) p.pad[i].at[threadIdx.x] = 0u;  // fewer than 256 bytes
    }
  }
  {
    const int r = threadIdx.x % kJoinRows, group = threadIdx.x / kJoinRows;
    const int row = blockIdx.x * kJoinRows + r;
    float m = -INFINITY, s = 0.0f, z = 0.0f;
    if (row < p.tokens) {
#pragma unroll 4
      for (int n = group; n < p.n_blocks; n += 32) {
        const float2 t = __ldcs(p.part + static_cast<size_t>(n) * p.tokens + row);
        const float nm = fmaxf(m, t.x);
        const float b = nm == -INFINITY ? 0.0f : nm;
        s = s * head::ex2(m - b) + t.y * head::ex2(t.x - b);
        m = nm;
        if (p.part_z != nullptr) z += __ldcs(p.part_z + static_cast<size_t>(n) * p.tokens + row);
      }
    }
    s_m[group][r] = m;
    s_s[group][r] = s;
    s_z[group][r] = z;
  }
  __syncthreads();
  const int row = blockIdx.x * kJoinRows + warp;
  const float my_m = s_m[lane][warp];
  float m = my_m, s = s_s[lane][warp], z = s_z[lane][warp];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  s *= head::ex2(my_m - (m == -INFINITY ? 0.0f : m));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    z += __shfl_xor_sync(0xffffffffu, z, o);
  }
  const float lse = (m + log2f(s)) * 0.6931471805599453f;
  float loss = 0.0f, kept = 0.0f;
  if (row < p.tokens) {
    if (p.probs != nullptr) {
      const float w = p.weight[row];
      if (w != 0.0f) {
        float dot = 0.0f;
        for (int j = lane; j < p.top; j += 32) {
          const size_t at = static_cast<size_t>(row) * p.top + j;
          if (p.ids[at] != head::kNoLabel) dot += p.probs[at] * p.label_z[at];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        loss = w * (p.neg_entropy[row] + lse - dot * p.inv_t) * p.row_scale;
        kept = 1.0f;
      }
    } else {
      const long long t = load_index(p.target, p.index_bits, row);
      if (t != p.ignore_index) {
        loss = t >= 0 && t < p.vocab ? lse - (1.0f - p.smoothing) * p.label_z[row] : NAN;
        if (p.part_z != nullptr) loss -= p.smoothing * (z / static_cast<float>(p.vocab));
        kept = 1.0f;
      }
    }
    if (lost) loss = NAN;
    if (lane == 0) {
      p.lse[row] = lse;
      if (p.reduction == B200_REDUCE_NONE) p.loss[row] = loss;
    }
  }
  if (p.reduction == B200_REDUCE_NONE) {
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.share = 1.0f;
    return;
  }
  if (lane == 0) {
    s_loss[warp] = loss;
    s_kept[warp] = kept;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    float a = 0.0f, k = 0.0f;
#pragma unroll
    for (int r = 0; r < kJoinRows; ++r) {
      a += s_loss[r];
      k += s_kept[r];
    }
    p.block_sums[blockIdx.x] = make_float2(a, k);
    __threadfence();
    s_last = atomicAdd(p.ticket, 1u) == gridDim.x - 1 ? 1u : 0u;
  }
  __syncthreads();
  if (s_last == 0u) return;
  __threadfence();
  double a = 0.0, k = 0.0;  // counts beyond 2^24 stay exact
  for (unsigned i = threadIdx.x; i < gridDim.x; i += blockDim.x) {
    const float2 t = __ldcg(p.block_sums + i);
    a += t.x;
    k += t.y;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    k += __shfl_xor_sync(0xffffffffu, k, o);
  }
  __shared__ double d_a[kJoinThreads / 32], d_k[kJoinThreads / 32];
  if (lane == 0) {
    d_a[warp] = a;
    d_k[warp] = k;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    a = k = 0.0;
    for (int i = 0; i < kJoinThreads / 32; ++i) {
      a += d_a[i];
      k += d_k[i];
    }
    const bool mean = p.reduction == B200_REDUCE_MEAN;
    *p.loss = static_cast<float>(mean ? a / k : a);
    *p.share = lost ? NAN : !mean ? 1.0f : (k > 0.0 ? static_cast<float>(1.0 / k) : 0.0f);  // without any row the gradients are zero
  }
}

// Row factors c_t = dL/dL_t * dL_t/d(softmax - labels), 0 for rows without a loss, divided by the largest
// of them: G = c_t (softmax - labels) is rounded to 16 bits, and with equal factors its entries at the labels
// are then close to 1 and -- nearly -- exact.  (Under the plain factor 1/N all of them carried the one rounding
// error of 1/N: the gradients were off by 0.0035 instead of 0.0017, which is the rounding of the result.)
// fp16: the largest factor is 2^13, so that small probabilities keep their digits, too.  `unscale` takes the
// divisor out of the gradients again, in fp32.  Mean and sum have equal factors and need no launch for this:
// the row's own 1, 0 or NaN is its factor, and everything else is in the divisor.
__global__ void __launch_bounds__(1024) factor_kernel(const float* __restrict__ grad_loss, float row_scale, const void* __restrict__ target, int index_bits,
                                                      long long ignore_index, int vocab, const float* __restrict__ weight, int tokens, float top,
                                                      float* __restrict__ coef, float* __restrict__ unscale) {
  __shared__ float buf[32];
  sm100::griddep_launch_dependents();
  sm100::griddep_wait();
  auto factor = [&](int t) -> float {
    float w;
    if (weight != nullptr) {
      w = weight[t];
    } else {
      const long long y = load_index(target, index_bits, t);
      w = y == ignore_index ? 0.0f : (y >= 0 && y < vocab ? 1.0f : NAN);
    }
    return w == 0.0f ? 0.0f : w * row_scale * grad_loss[t];
  };
  float mx = 0.0f;
  for (int t = threadIdx.x; t < tokens; t += blockDim.x) {
    const float c = fabsf(factor(t));
    if (c < INFINITY) mx = fmaxf(mx, c);
  }
  mx = block_reduce(mx, true, buf);
  if (mx == 0.0f) mx = 1.0f;
  for (int t = threadIdx.x; t < tokens; t += blockDim.x) coef[t] = factor(t) / mx * top;
  if (threadIdx.x == 0) *unscale = mx / top;
}

// A gradient as the sum of its fp32 parts, in their order, rounded once.  n4 = elements / 4.
template <typename T16>
__global__ void __launch_bounds__(256) sum_parts_kernel(const float* __restrict__ parts, int splits, size_t n4, T16* __restrict__ out, const uint32_t* status) {
  sm100::griddep_wait();
  const float lost = head::wait_lost(status) ? NAN : 0.0f;
  for (size_t i = static_cast<size_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n4; i += static_cast<size_t>(gridDim.x) * blockDim.x) {
    float4 a = __ldcs(reinterpret_cast<const float4*>(parts) + i);
    for (int s = 1; s < splits; ++s) {
      const float4 b = __ldcs(reinterpret_cast<const float4*>(parts) + s * n4 + i);
      a = make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
    }
    if (lost != 0.0f) a = make_float4(lost, lost, lost, lost);
    reinterpret_cast<uint2*>(out)[i] = make_uint2(head::pack2<T16>(a.x, a.y), head::pack2<T16>(a.z, a.w));
  }
}

// ---------------------------------------------------------------------------------------------
// schedules
// ---------------------------------------------------------------------------------------------
struct Tiling {
  int cg, bn, am, stages, smem;
  int warps;  // epilogue warps
};

int ring(Tiling* t) {
  const int room = kMaxSmem - head::kBarrierBytes - 1024 - t->warps * head::kTurnBytes - head::overrun_bytes(t->bn, t->cg, t->am);
  // With few rows the product streams w from DRAM, and 140 KB of it on request per SM are enough (8 x 4096 x 32768
  // forward: 61 / 55 / 54 / 53 / 53 us with 2 / 3 / 4 / 5 / 6 stages of 28 KB).
  const int cap = t->am < 128 ? std::min(head::kMaxStages, std::max(4, 140 * 1024 / (t->bn * head::kRowBytes))) : 8;
  t->stages = std::min(cap, room / head::stage_bytes(t->bn, t->cg, t->am));
  t->smem = head::smem_bytes(t->bn, t->stages, t->cg, t->am, t->warps);
  // One CTA per SM: each takes all of TMEM.
  if (t->smem <= kMaxSmem / 2) t->smem = kMaxSmem / 2 + 1024;
  return t->stages;
}

// CTA pairs (256-row tiles) unless single CTAs (128 rows) leave at least a fifth fewer padded rows.
int choose_cg(int64_t tokens) { return div_up(tokens, 128) * 128 * 5 <= div_up(tokens, 256) * 256 * 4 ? 1 : 2; }

// Tile of z: of the widths from 256 down, the one whose rounds of tiles cost least.  A K block of a tile costs
// what the L2 sends its SM, the rows of A and of B that a CTA stages: at 64 bytes a cycle that is 512 cycles
// for a pair's 256 x 256, as long as its MMAs, and longer than them for everything narrower.
Tiling z_tiling(int64_t tokens, int64_t cols) {
  Tiling t = {};
  t.warps = 4;
  t.cg = choose_cg(tokens);
  t.am = t.cg == 1 && tokens <= 64 ? (tokens <= 32 ? 32 : 64) : 128;
  const int64_t units = kSms / t.cg, m_blocks = div_up(tokens, 128 * t.cg);
  int64_t best = 0;
  for (int bn = 256; bn >= 64; bn -= 32) {
    const int64_t cost = div_up(m_blocks * div_up(cols, bn), units) * (t.am + bn / t.cg);
    if (t.bn == 0 || cost < best) {
      t.bn = bn;
      best = cost;
    }
  }
  ring(&t);
  return t;
}

struct Plan {
  Tiling z, grad, prod;
  int64_t n_blocks;       // tiles along the vocabulary, forward
  int64_t range, ranges;  // columns of G at a time
  int64_t g_ld;
  int splits, kb_per_split;      // of dX's K, the range
  int w_splits, w_kb_per_split;  // of dW's K, the tokens
  bool direct;            // dX is written by the product itself
  // byte offsets
  size_t f_part, f_part_z, f_label_z, f_entropy, f_sums, f_ticket, f_bytes;
  size_t s_weight, s_probs, s_ids, s_bytes;
  size_t b_g, b_coef, b_unscale, b_parts, b_w_parts, b_bytes;
};

int make_plan(const b200_head_desc& d, Plan* p) {
  B200_REQUIRE(d.kind == B200_HEAD_CROSS_ENTROPY || d.kind == B200_HEAD_DISTILL, "head_loss: kind=%d", d.kind);
  B200_REQUIRE(d.tokens >= 1 && d.hidden >= 8 && d.vocab >= 1, "head_loss: tokens and vocab must be >= 1 and hidden >= 8 (got %lld, %lld, %lld)",
               (long long)d.tokens, (long long)d.vocab, (long long)d.hidden);
  const int64_t limit = (1ll << 31) - 1024;
  B200_REQUIRE(d.tokens < limit && d.hidden < limit && d.vocab < limit, "head_loss: tokens, hidden and vocab must be below 2^31");
  B200_REQUIRE(d.hidden % 8 == 0, "head_loss: hidden=%lld is not a multiple of 8 (16-byte rows)", (long long)d.hidden);
  B200_REQUIRE(d.x_stride >= d.hidden && d.w_stride >= d.hidden && d.x_stride % 8 == 0 && d.w_stride % 8 == 0,
               "head_loss: x_stride=%lld and w_stride=%lld must be multiples of 8 of at least hidden", (long long)d.x_stride, (long long)d.w_stride);
  B200_REQUIRE(d.dtype == B200_F16 || d.dtype == B200_BF16, "head_loss: dtype=%d is not f16 or bf16", d.dtype);
  B200_REQUIRE(d.reduction >= B200_REDUCE_NONE && d.reduction <= B200_REDUCE_SUM, "head_loss: reduction=%d", d.reduction);
  B200_REQUIRE(d.index_bits == 32 || d.index_bits == 64, "head_loss: index_bits=%d is not 32 or 64", d.index_bits);
  B200_REQUIRE(d.grad_bytes >= 0, "head_loss: grad_bytes must be >= 0");
  B200_REQUIRE(d.wait_limit_ms >= 0, "head_loss: wait_limit_ms must be >= 0");
  if (d.kind == B200_HEAD_DISTILL) {
    B200_REQUIRE(d.top >= 1 && d.top <= kMaxTop, "head_loss: top=%d outside [1, %d]", d.top, kMaxTop);
    B200_REQUIRE(d.dtype_teacher == B200_F32 || d.dtype_teacher == B200_BF16 || d.dtype_teacher == B200_F16, "head_loss: dtype_teacher=%d is not f32, bf16 or f16", d.dtype_teacher);
    // 1 / T and T^2 have to be numbers that fp32 holds in full.
    B200_REQUIRE(d.temperature >= 0x1p-60f && d.temperature <= 0x1p60f, "head_loss: temperature=%g is outside [2^-60, 2^60]", d.temperature);
  } else {
    B200_REQUIRE(d.label_smoothing >= 0.0f && d.label_smoothing < 1.0f, "head_loss: label_smoothing must be in [0, 1)");
  }
  const size_t T = static_cast<size_t>(d.tokens), top = d.kind == B200_HEAD_DISTILL ? static_cast<size_t>(d.top) : 1u;
  p->z = z_tiling(d.tokens, d.vocab);
  p->n_blocks = div_up(d.vocab, p->z.bn);
  size_t at = 0;
  auto take = [&at](size_t bytes) {
    const size_t off = at;
    at = align256(at + bytes);
    return off;
  };
  p->f_part = take(static_cast<size_t>(p->n_blocks) * T * sizeof(float2));
  p->f_part_z = take(d.kind == B200_HEAD_CROSS_ENTROPY && d.label_smoothing > 0.0f ? static_cast<size_t>(p->n_blocks) * T * sizeof(float) : 0);
  p->f_label_z = take(T * top * sizeof(float));
  p->f_entropy = take(d.kind == B200_HEAD_DISTILL ? T * sizeof(float) : 0);
  p->f_sums = take(static_cast<size_t>(div_up(d.tokens, kJoinRows)) * sizeof(float2));
  p->f_ticket = take(sizeof(uint32_t));
  p->f_bytes = at;
  at = 0;
  take(sizeof(float));  // share
  p->s_weight = take(d.kind == B200_HEAD_DISTILL ? T * sizeof(float) : 0);
  p->s_probs = take(d.kind == B200_HEAD_DISTILL ? T * top * sizeof(float) : 0);
  p->s_ids = take(d.kind == B200_HEAD_DISTILL ? T * top * sizeof(int32_t) : 0);
  p->s_bytes = at;

  // Ranges of the vocabulary: as few as the limit allows, of equal width, whole tiles.
  const int64_t most = std::max<int64_t>(256, (d.grad_bytes > 0 ? d.grad_bytes : kGradBytes) / (2 * d.tokens) / 256 * 256);
  p->ranges = div_up(d.vocab, most);
  p->range = std::min<int64_t>(div_up(div_up(d.vocab, p->ranges), 256) * 256, div_up(d.vocab, 64) * 64);
  p->ranges = div_up(d.vocab, p->range);
  p->g_ld = p->range;
  p->grad = z_tiling(d.tokens, p->range);
  p->prod = {};
  p->prod.cg = p->z.cg;
  p->prod.bn = 256;
  p->prod.am = 128;
  // dW's tiles have tokens / 64 K blocks.  With two of them or fewer its output decides, and eight epilogue
  // warps pay (8 x 4096 x 32768: backward 181 -> 168 us); with more they only take power from the MMAs (333 tokens: 50 -> 53 us).
  p->prod.warps = p->prod.cg == 1 && d.tokens <= 128 ? 8 : 4;
  ring(&p->prod);
  // dX has few tiles with a long K (the range), dW many with a short one (the tokens).  dX is cut until a
  // part is at most half of what an SM does in all, which keeps the last round short.
  const int64_t units = kSms / p->prod.cg, tile_m = 128 * p->prod.cg, n_tiles = div_up(d.hidden, p->prod.bn);
  const int64_t x_kb = div_up(p->range, head::kStageK), x_tiles = div_up(d.tokens, tile_m) * n_tiles;
  const int64_t w_kb = div_up(d.tokens, head::kStageK), w_tiles = div_up(p->range, tile_m) * n_tiles;
  const int64_t share = (x_kb * x_tiles + w_kb * w_tiles) / units;
  const int64_t want = std::max<int64_t>(16, share / 2);
  const int64_t parts = std::min<int64_t>(32, div_up(x_kb, want));
  p->kb_per_split = static_cast<int>(div_up(x_kb, parts));
  p->splits = static_cast<int>(div_up(x_kb, p->kb_per_split));
  p->direct = p->splits == 1 && p->ranges == 1;
  // dW likewise where one of its tiles is more than an SM's share of all the work (a small vocabulary or hidden axis
  // and many tokens: 65536 x 256 x 4000 backward 1111 -> 720 us, 8192 x 256 x 4000 98 -> 86) and the fp32 parts stay
  // below 256 MiB; with shorter tiles the parts only cost (8192 x 1024 x 4096: 152 -> 162).
  const int64_t part_bytes = p->range * d.hidden * 4;
  const int64_t w_parts = w_kb > share ? std::min<int64_t>({16, div_up(w_kb, want), std::max<int64_t>(1, kGradBytes / part_bytes)}) : 1;
  p->w_kb_per_split = static_cast<int>(div_up(w_kb, w_parts));
  p->w_splits = static_cast<int>(div_up(w_kb, p->w_kb_per_split));
  at = 0;
  p->b_g = take(T * static_cast<size_t>(p->g_ld) * 2);
  p->b_coef = take(T * sizeof(float));
  p->b_unscale = take(sizeof(float));
  p->b_parts = take(p->direct ? 0 : static_cast<size_t>(p->splits) * T * static_cast<size_t>(d.hidden) * sizeof(float));
  p->b_w_parts = take(p->w_splits > 1 ? static_cast<size_t>(p->w_splits) * static_cast<size_t>(part_bytes) : 0);
  p->b_bytes = at;
  return B200_OK;
}

int raster(int64_t m_blocks, int64_t tile_m, int64_t k) {
  const int64_t g = (32ll << 20) / std::max<int64_t>(1, tile_m * k * 2);
  return static_cast<int>(std::max<int64_t>(1, std::min(g, m_blocks)));
}

using KernelFn = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const CUtensorMap, const Params);

template <int MODE>
KernelFn kernel_for(int cg, int dtype, int warps = 4) {
  if constexpr (MODE == head::kProduct) {
    if (warps == 8) return dtype == B200_F16 ? head::head_kernel<1, MODE, __half, 8> : head::head_kernel<1, MODE, __nv_bfloat16, 8>;
  }
  if (dtype == B200_F16) return cg == 2 ? head::head_kernel<2, MODE, __half, 4> : head::head_kernel<1, MODE, __half, 4>;
  return cg == 2 ? head::head_kernel<2, MODE, __nv_bfloat16, 4> : head::head_kernel<1, MODE, __nv_bfloat16, 4>;
}

uint32_t idesc(int dtype, const Tiling& t, bool a_mn, bool b_mn) {
  const uint32_t f = dtype == B200_BF16 ? 1u : 0u;
  return sm100::make_idesc(1u, f, f, static_cast<uint32_t>(head::kBM * t.cg), static_cast<uint32_t>(t.bn)) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
}

// What a device needs to be asked or told once: that it is an sm_100 part, the address of its status words,
// and the kernels' shared-memory limit there.
constexpr int kMaxDevices = 64;
struct DeviceState {
  std::atomic<bool> ready{false};  // set once everything below is known; a failed attempt is made again by the next call
  uint32_t* status = nullptr;
};
std::mutex g_devices_mu;
DeviceState g_devices[kMaxDevices];

int init_device(int dev, DeviceState* st) {
  int major = 0;
  B200_CUDA_OK(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev));
  if (major != 10) return b200::fail(B200_ERR_NO_DEVICE, "device %d has compute capability %d.x; the kernels need sm_100", dev, major);
  for (int dtype : {B200_F16, B200_BF16}) {
    for (int cg : {1, 2}) {
      for (KernelFn fn : {kernel_for<head::kStats>(cg, dtype), kernel_for<head::kGrad>(cg, dtype), kernel_for<head::kProduct>(cg, dtype), kernel_for<head::kProduct>(1, dtype, 8)}) {
        B200_CUDA_OK(cudaFuncSetAttribute(reinterpret_cast<const void*>(fn), cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
      }
    }
  }
  void* p = nullptr;
  B200_CUDA_OK(cudaGetSymbolAddress(&p, g_status));
  st->status = static_cast<uint32_t*>(p);
  return B200_OK;
}

int current_device(DeviceState** out) {
  int dev = 0;
  B200_CUDA_OK(cudaGetDevice(&dev));
  B200_REQUIRE(dev >= 0 && dev < kMaxDevices, "head_loss: device index %d", dev);
  DeviceState& st = g_devices[dev];
  if (!st.ready.load(std::memory_order_acquire)) {
    std::lock_guard<std::mutex> lock(g_devices_mu);
    if (!st.ready.load(std::memory_order_relaxed)) {
      const int rc = init_device(dev, &st);
      if (rc != B200_OK) return rc;
      st.ready.store(true, std::memory_order_release);
    }
  }
  *out = &st;
  return B200_OK;
}

int launch(KernelFn fn, const Tiling& t, Params* p, const CUtensorMap (&maps)[4], cudaStream_t stream) {
  int64_t items = p->prob[0].items;
  if (p->num_probs > 1) items += p->prob[1].items;
  p->bn = t.bn;
  p->am = t.am;
  p->stages = t.stages;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(items, kSms / t.cg)) * t.cg);
  cfg.blockDim = dim3(static_cast<unsigned>(head::threads(t.warps)));
  cfg.dynamicSmemBytes = static_cast<size_t>(t.smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (t.cg == 2) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = 2;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  // The prologue overlaps the previous kernel's end; the kernel waits for that kernel before it touches global memory.
  attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[n].val.programmaticStreamSerializationAllowed = 1;
  ++n;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  B200_CUDA_OK(cudaLaunchKernelEx(&cfg, fn, maps[0], maps[1], maps[2], maps[3], *p));
  b200::count_launch();
  B200_CUDA_OK(cudaGetLastError());
  return B200_OK;
}

// A small kernel that begins with griddep_wait: its launch overlaps the end of the kernel before it.
template <typename... Args, typename... Actual>
int launch_small(void (*fn)(Args...), unsigned grid, unsigned threads, size_t smem, cudaStream_t stream, Actual... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.dynamicSmemBytes = smem;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  B200_CUDA_OK(cudaLaunchKernelEx(&cfg, fn, static_cast<Args>(args)...));
  b200::count_launch();
  B200_CUDA_OK(cudaGetLastError());
  return B200_OK;
}

int launch_sum_parts(int dtype, const float* parts, int splits, size_t n, void* out, const uint32_t* status, cudaStream_t stream) {
  const size_t n4 = n / 4;
  const unsigned blocks = static_cast<unsigned>(std::min<size_t>((n4 + 255) / 256, kSms * 8));
  if (dtype == B200_F16) return launch_small(sum_parts_kernel<__half>, blocks, 256u, 0u, stream, parts, splits, n4, static_cast<__half*>(out), status);
  return launch_small(sum_parts_kernel<__nv_bfloat16>, blocks, 256u, 0u, stream, parts, splits, n4, static_cast<__nv_bfloat16*>(out), status);
}

// z = x . w^T over the columns [col0, col0 + cols).
Problem z_problem(const b200_head_desc& d, const Tiling& t, int64_t col0, int64_t cols) {
  Problem q = {};
  q.M = static_cast<int>(d.tokens);
  q.N = static_cast<int>(cols);
  q.num_kb = q.kb_per_split = static_cast<int>(div_up(d.hidden, head::kStageK));
  q.splits = 1;
  q.m_blocks = static_cast<int>(div_up(d.tokens, 128 * t.cg));
  q.n_blocks = static_cast<int>(div_up(cols, t.bn));
  q.raster_group = raster(q.m_blocks, 128 * t.cg, d.hidden);
  q.b_row0 = static_cast<int>(col0);
  q.idesc = idesc(d.dtype, t, false, false);
  return q;
}

int set_items(Problem* q) {
  const int64_t items = static_cast<int64_t>(q->m_blocks) * q->n_blocks * q->splits;
  B200_REQUIRE(items < (1ll << 30), "head_loss: %lld tiles are more than one launch covers", (long long)items);
  q->items = static_cast<int>(items);
  q->tiles = head::FastDiv::of(q->m_blocks * q->n_blocks);
  q->span = head::FastDiv::of(q->raster_group * q->n_blocks);
  q->group = head::FastDiv::of(q->raster_group);
  q->last_group = head::FastDiv::of(q->m_blocks % q->raster_group != 0 ? q->m_blocks % q->raster_group : q->raster_group);
  return B200_OK;
}

void set_labels(const b200_head_desc& d, const Plan& pl, const void* labels, const void* saved, uint32_t* status, Params* p) {
  std::memset(p, 0, sizeof(*p));
  p->status = status;
  p->wait_limit_ms = static_cast<unsigned>(d.wait_limit_ms);
  p->num_probs = 1;
  p->tokens = static_cast<int>(d.tokens);
  p->vocab = static_cast<int>(d.vocab);
  p->top = 1;
  p->scale2 = kLog2e;
  if (d.kind == B200_HEAD_DISTILL) {
    const uint8_t* s = static_cast<const uint8_t*>(saved);
    p->top = d.top;
    p->ids = reinterpret_cast<const int32_t*>(s + pl.s_ids);
    p->probs = reinterpret_cast<const float*>(s + pl.s_probs);
    p->scale2 = kLog2e / d.temperature;
  } else {
    p->target = labels;
    p->target64 = d.index_bits == 64;
    p->ignore_index = d.ignore_index;
    p->label_prob = 1.0f - d.label_smoothing;
    p->base = d.label_smoothing / static_cast<float>(d.vocab);
  }
}

int common_checks(const b200_head_desc* desc, const void* x, const void* w, const void* labels, const void* saved, const void* workspace, size_t bytes,
                  size_t need) {
  B200_REQUIRE(x != nullptr && w != nullptr && labels != nullptr && saved != nullptr, "head_loss: NULL argument");
  B200_REQUIRE(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(saved) | reinterpret_cast<uintptr_t>(workspace)) & 15u) == 0,
               "head_loss: x, w, saved and workspace must be 16-byte aligned");
  B200_REQUIRE((reinterpret_cast<uintptr_t>(labels) & static_cast<uintptr_t>(desc->index_bits / 8 - 1)) == 0, "head_loss: labels must be aligned to their elements");
  if (workspace == nullptr || bytes < need) return b200::fail(B200_ERR_WORKSPACE, "head_loss: needs a %zu-byte workspace, got %zu", need, bytes);
  return B200_OK;
}

int status_words(uint32_t** words) {
  DeviceState* st = nullptr;
  const int rc = current_device(&st);
  if (rc == B200_OK) *words = st->status;
  return rc;
}

}  // namespace

extern "C" {

int b200_head_loss_sizes(const b200_head_desc* desc, b200_head_sizes* sizes) {
  B200_REQUIRE(desc != nullptr && sizes != nullptr, "head_loss_sizes: NULL argument");
  std::memset(sizes, 0, sizeof(*sizes));
  Plan pl;
  const int rc = make_plan(*desc, &pl);
  if (rc != B200_OK) return rc;
  sizes->forward_workspace = pl.f_bytes;
  sizes->backward_workspace = pl.b_bytes;
  sizes->saved = pl.s_bytes;
  sizes->grad_columns = pl.range;
  sizes->grad_splits = pl.splits;
  sizes->cta_group = pl.z.cg;
  sizes->tile_n = pl.z.bn;
  return B200_OK;
}

int b200_head_loss_forward(const b200_head_desc* desc, const void* x, const void* w, const void* labels, const void* teacher_logits, float* loss, float* lse,
                           void* saved, void* workspace, size_t workspace_bytes, void* stream) {
  B200_REQUIRE(desc != nullptr && loss != nullptr && lse != nullptr, "head_loss_forward: NULL argument");
  const b200_head_desc& d = *desc;
  Plan pl;
  int rc = make_plan(d, &pl);
  if (rc != B200_OK) return rc;
  B200_REQUIRE((d.kind == B200_HEAD_DISTILL) == (teacher_logits != nullptr), "head_loss_forward: teacher_logits belong to distillation, and only to it");
  rc = common_checks(desc, x, w, labels, saved, workspace, workspace_bytes, pl.f_bytes);
  if (rc != B200_OK) return rc;
  const cudaStream_t s = b200::as_stream(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  uint8_t* sv = static_cast<uint8_t*>(saved);
  uint32_t* status = nullptr;
  rc = status_words(&status);
  if (rc != B200_OK) return rc;
  if (d.kind == B200_HEAD_DISTILL) {
    int n = 2;
    while (n < d.top) n *= 2;
    const unsigned threads = static_cast<unsigned>(std::max(32, n / 2));
    rc = launch_small(teacher_kernel, static_cast<unsigned>(d.tokens), threads, static_cast<size_t>(n) * 12u, s, teacher_logits, d.dtype_teacher, labels, d.index_bits, d.top, n, static_cast<int>(d.vocab),
                      1.0f / d.temperature, reinterpret_cast<int32_t*>(sv + pl.s_ids), reinterpret_cast<float*>(sv + pl.s_probs), reinterpret_cast<float*>(sv + pl.s_weight),
                      reinterpret_cast<float*>(ws + pl.f_entropy));
    if (rc != B200_OK) return rc;
  }
  Params p;
  set_labels(d, pl, labels, saved, status, &p);
  p.prob[0] = z_problem(d, pl.z, 0, d.vocab);
  rc = set_items(&p.prob[0]);
  if (rc != B200_OK) return rc;
  p.part = reinterpret_cast<float2*>(ws + pl.f_part);
  const bool smooth = d.kind == B200_HEAD_CROSS_ENTROPY && d.label_smoothing > 0.0f;
  p.part_z = smooth ? reinterpret_cast<float*>(ws + pl.f_part_z) : nullptr;
  p.label_z = reinterpret_cast<float*>(ws + pl.f_label_z);
  p.ticket = reinterpret_cast<uint32_t*>(ws + pl.f_ticket);
  CUtensorMap maps[4] = {};
  rc = b200::make_strided_operand_map(&maps[0], x, d.dtype, d.tokens, d.hidden, d.x_stride, static_cast<uint32_t>(pl.z.am));
  if (rc != B200_OK) return rc;
  rc = b200::make_strided_operand_map(&maps[1], w, d.dtype, d.vocab, d.hidden, d.w_stride, static_cast<uint32_t>(pl.z.bn / pl.z.cg));
  if (rc != B200_OK) return rc;
  rc = launch(kernel_for<head::kStats>(pl.z.cg, d.dtype), pl.z, &p, maps, s);
  if (rc != B200_OK) return rc;
  JoinParams j = {};
  j.part = p.part;
  j.part_z = p.part_z;
  j.label_z = p.label_z;
  j.target = p.target;
  j.index_bits = d.index_bits;
  j.ignore_index = d.ignore_index;
  j.tokens = p.tokens;
  j.vocab = p.vocab;
  j.n_blocks = static_cast<int>(pl.n_blocks);
  j.top = p.top;
  j.reduction = d.reduction;
  j.smoothing = smooth ? d.label_smoothing : 0.0f;
  j.inv_t = j.row_scale = 1.0f;
  if (d.kind == B200_HEAD_DISTILL) {
    j.probs = p.probs;
    j.ids = p.ids;
    j.weight = reinterpret_cast<const float*>(sv + pl.s_weight);
    j.neg_entropy = reinterpret_cast<const float*>(ws + pl.f_entropy);
    j.inv_t = 1.0f / d.temperature;
    j.row_scale = d.temperature * d.temperature;
  }
  j.loss = loss;
  j.lse = lse;
  j.share = reinterpret_cast<float*>(sv);
  j.block_sums = reinterpret_cast<float2*>(ws + pl.f_sums);
  j.ticket = p.ticket;
  j.status = status;
  auto pad = [&](int i, size_t part, size_t words) {
    const size_t end = part + words * 4;
    j.pad[i] = {reinterpret_cast<uint32_t*>(sv + end), static_cast<int>((align256(end) - end) / 4)};
  };
  pad(0, 0, 1);
  if (d.kind == B200_HEAD_DISTILL) {
    const size_t rows = static_cast<size_t>(d.tokens), entries = rows * static_cast<size_t>(d.top);
    pad(1, pl.s_weight, rows);
    pad(2, pl.s_probs, entries);
    pad(3, pl.s_ids, entries);
  }
  return launch_small(join_kernel, static_cast<unsigned>(div_up(d.tokens, kJoinRows)), kJoinThreads, 0u, s, j);
}

int b200_head_loss_backward(const b200_head_desc* desc, const void* x, const void* w, const void* labels, const float* lse, const void* saved,
                            const float* grad_loss, void* grad_x, void* grad_w, void* workspace, size_t workspace_bytes, void* stream) {
  B200_REQUIRE(desc != nullptr && lse != nullptr && grad_loss != nullptr, "head_loss_backward: NULL argument");
  const b200_head_desc& d = *desc;
  Plan pl;
  int rc = make_plan(d, &pl);
  if (rc != B200_OK) return rc;
  rc = common_checks(desc, x, w, labels, saved, workspace, workspace_bytes, pl.b_bytes);
  if (rc != B200_OK) return rc;
  B200_REQUIRE(((reinterpret_cast<uintptr_t>(grad_x) | reinterpret_cast<uintptr_t>(grad_w)) & 15u) == 0, "head_loss_backward: grad_x and grad_w must be 16-byte aligned");
  if (grad_x == nullptr && grad_w == nullptr) return B200_OK;
  const cudaStream_t s = b200::as_stream(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const uint8_t* sv = static_cast<const uint8_t*>(saved);
  uint32_t* status = nullptr;
  rc = status_words(&status);
  if (rc != B200_OK) return rc;
  const bool distill = d.kind == B200_HEAD_DISTILL;
  float* coef = reinterpret_cast<float*>(ws + pl.b_coef);
  float* unscale = reinterpret_cast<float*>(ws + pl.b_unscale);
  float* parts = reinterpret_cast<float*>(ws + pl.b_parts);
  void* g = ws + pl.b_g;
  const bool per_row = d.reduction == B200_REDUCE_NONE;
  const float row_scale = distill ? d.temperature : 1.0f, coef_top = d.dtype == B200_F16 ? kHalfTop : 1.0f;
  const float* weight = distill ? reinterpret_cast<const float*>(sv + pl.s_weight) : nullptr;
  const float* share = reinterpret_cast<const float*>(sv);
  if (per_row) {
    rc = launch_small(factor_kernel, 1u, 1024u, 0u, s, grad_loss, row_scale, labels, d.index_bits, d.ignore_index, static_cast<int>(d.vocab), weight,
                      static_cast<int>(d.tokens), coef_top, coef, unscale);
    if (rc != B200_OK) return rc;
  }

  CUtensorMap z_maps[4] = {};
  rc = b200::make_strided_operand_map(&z_maps[0], x, d.dtype, d.tokens, d.hidden, d.x_stride, static_cast<uint32_t>(pl.grad.am));
  if (rc != B200_OK) return rc;
  rc = b200::make_strided_operand_map(&z_maps[1], w, d.dtype, d.vocab, d.hidden, d.w_stride, static_cast<uint32_t>(pl.grad.bn / pl.grad.cg));
  if (rc != B200_OK) return rc;
  CUtensorMap w_rows, x_rows;  // boxes of 64 K rows
  rc = b200::make_strided_operand_map(&w_rows, w, d.dtype, d.vocab, d.hidden, d.w_stride, 64);
  if (rc != B200_OK) return rc;
  rc = b200::make_strided_operand_map(&x_rows, x, d.dtype, d.tokens, d.hidden, d.x_stride, 64);
  if (rc != B200_OK) return rc;

  for (int64_t r = 0; r < pl.ranges; ++r) {
    const int64_t col0 = r * pl.range, cols = std::min(pl.range, d.vocab - col0);
    Params p;
    set_labels(d, pl, labels, saved, status, &p);
    p.prob[0] = z_problem(d, pl.grad, col0, cols);
    rc = set_items(&p.prob[0]);
    if (rc != B200_OK) return rc;
    p.col0 = static_cast<int>(col0);
    p.lse = lse;
    p.coef = per_row ? coef : nullptr;
    p.coef_top = coef_top;
    p.weight = weight;
    p.g = g;
    p.g_ld = pl.g_ld;
    rc = launch(kernel_for<head::kGrad>(pl.grad.cg, d.dtype), pl.grad, &p, z_maps, s);
    if (rc != B200_OK) return rc;

    // dX and dW of the range in one launch.  G's maps end at the range's last column: what lies behind
    // it in a row of G is read as zero.
    Params q;
    std::memset(&q, 0, sizeof(q));
    q.status = status;
    q.wait_limit_ms = static_cast<unsigned>(d.wait_limit_ms);
    q.unscale = per_row ? unscale : nullptr;
    q.share = share;
    q.grad_loss = grad_loss;
    q.unscale_factor = row_scale / coef_top;
    CUtensorMap maps[4] = {};
    if (grad_x != nullptr) {
      Problem& dx = q.prob[q.num_probs];
      rc = b200::make_strided_operand_map(&maps[0], g, d.dtype, d.tokens, cols, pl.g_ld, 128);
      if (rc != B200_OK) return rc;
      maps[1] = w_rows;
      dx.M = static_cast<int>(d.tokens);
      dx.N = static_cast<int>(d.hidden);
      dx.num_kb = static_cast<int>(div_up(cols, head::kStageK));
      dx.kb_per_split = pl.kb_per_split;
      dx.splits = static_cast<int>(div_up(dx.num_kb, pl.kb_per_split));
      dx.m_blocks = static_cast<int>(div_up(d.tokens, 128 * pl.prod.cg));
      dx.n_blocks = static_cast<int>(div_up(d.hidden, pl.prod.bn));
      dx.raster_group = raster(dx.m_blocks, 128 * pl.prod.cg, cols);
      dx.b_mn = 1;
      dx.b_k0 = static_cast<int>(col0);
      dx.idesc = idesc(d.dtype, pl.prod, false, true);
      dx.ld = d.hidden;
      dx.out16 = pl.direct ? grad_x : nullptr;
      dx.partial = parts;
      dx.accumulate = r > 0;
      rc = set_items(&dx);
      if (rc != B200_OK) return rc;
      ++q.num_probs;
    }
    if (grad_w != nullptr) {
      Problem& dw = q.prob[q.num_probs];
      rc = b200::make_strided_operand_map(&maps[2 * q.num_probs], g, d.dtype, d.tokens, cols, pl.g_ld, 64);
      if (rc != B200_OK) return rc;
      maps[2 * q.num_probs + 1] = x_rows;
      dw.M = static_cast<int>(cols);
      dw.N = static_cast<int>(d.hidden);
      dw.num_kb = static_cast<int>(div_up(d.tokens, head::kStageK));
      dw.kb_per_split = pl.w_kb_per_split;
      dw.splits = pl.w_splits;
      dw.m_blocks = static_cast<int>(div_up(cols, 128 * pl.prod.cg));
      dw.n_blocks = static_cast<int>(div_up(d.hidden, pl.prod.bn));
      dw.raster_group = raster(dw.m_blocks, 128 * pl.prod.cg, d.tokens);
      dw.a_mn = dw.b_mn = 1;
      dw.idesc = idesc(d.dtype, pl.prod, true, true);
      dw.ld = d.hidden;
      dw.out16 = pl.w_splits > 1 ? nullptr : static_cast<uint8_t*>(grad_w) + static_cast<size_t>(col0) * d.hidden * 2;
      dw.partial = reinterpret_cast<float*>(ws + pl.b_w_parts);
      rc = set_items(&dw);
      if (rc != B200_OK) return rc;
      ++q.num_probs;
    }
    if (q.num_probs == 2) q.extra_rounds = std::max(1, q.prob[0].kb_per_split / q.prob[1].kb_per_split);
    rc = launch(kernel_for<head::kProduct>(pl.prod.cg, d.dtype, pl.prod.warps), pl.prod, &q, maps, s);
    if (rc != B200_OK) return rc;
    if (grad_w != nullptr && pl.w_splits > 1) {
      rc = launch_sum_parts(d.dtype, reinterpret_cast<const float*>(ws + pl.b_w_parts), pl.w_splits, static_cast<size_t>(cols) * static_cast<size_t>(d.hidden),
                            static_cast<uint8_t*>(grad_w) + static_cast<size_t>(col0) * d.hidden * 2, status, s);
      if (rc != B200_OK) return rc;
    }
  }
  if (grad_x != nullptr && !pl.direct) {
    return launch_sum_parts(d.dtype, parts, pl.splits, static_cast<size_t>(d.tokens) * static_cast<size_t>(d.hidden), grad_x, status, s);
  }
  return B200_OK;
}

int b200_head_loss_status(uint32_t words[4]) {
  B200_REQUIRE(words != nullptr, "head_loss_status: NULL argument");
  uint32_t* dev = nullptr;
  const int rc = status_words(&dev);
  if (rc != B200_OK) return rc;
  B200_CUDA_OK(cudaDeviceSynchronize());
  B200_CUDA_OK(cudaMemcpy(words, dev, 4 * sizeof(uint32_t), cudaMemcpyDeviceToHost));
  if (words[0] != 0) {
    B200_CUDA_OK(cudaMemset(dev, 0, 4 * sizeof(uint32_t)));
    return b200::fail(B200_ERR_TIMEOUT, "device wait timed out: code 0x%x cta %u item %u k-block %u", words[0], words[1], words[2], words[3]);
  }
  return B200_OK;
}

}  // extern "C"
