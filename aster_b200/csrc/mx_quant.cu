// Block-scaled 4-bit floats on the device: values -> E2M1 codes and E8M0 scales, and back.
//
// A block is 32 consecutive values of a row.  With a = max |x| over the block, the shared exponent
// is e = floor(log2 a) - 2 (2 is the exponent of E2M1's largest magnitude, 6 = 1.5 * 2^2), clamped
// to [-127, 127]; the scale byte is e + 127 and the codes are x * 2^-e rounded to nearest even with
// magnitudes above 6 saturating.  A block of zeros has scale byte 127.  A block that holds a NaN or
// an infinity has scale byte 255 (E8M0's NaN): all 32 values then read as NaN, here and in the
// tensor core.  All of it is exact in fp32 but for the one rounding to E2M1: a product with a power
// of two only rounds where the result is below 2^-126, and that is code 0 either way.
//
// The scales are written in the order the product streams them (blocks of [128 rows][4 K blocks],
// row r of a block at byte (r % 32) * 16 + (r / 32) * 4; see pack_mx_scales_kernel), so that no
// second pass over them is needed.
//
// Both kernels are bound by DRAM.  A lane moves 8 values (16 or 32 bytes, one vector access) and 4 lanes
// share a block, so a warp's accesses are contiguous and the block maximum is two shuffles.  A warp takes
// 256 of K in the eight rows {r, r + 1} + {0, 32, 64, 96} of 128, whose scales are two whole 32-byte sectors
// of the packed order: it needs no other warp, and has eight vectors per lane on their way at once.  (Tiles
// of 128 rows whose scales meet in shared memory: 36 us instead of 31 for 8192 x 8192 bf16, 5.5 TB/s; back 28 us, 6.0; more threads
// per CTA: 39 to 48.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>

#include "common.h"
#include "ptx_sm100.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kPerLane = 8;               // values per lane and row
constexpr int kTileK = 32 * kPerLane;     // of K per warp: 8 blocks of 32 per row
constexpr int kTileRows = 128;
constexpr int kRows = 8;                  // rows per warp
constexpr int kCtasPerTile = kTileRows / kRows / kWarps;
constexpr int kScaleBlockBytes = 512;

// 8 consecutive values as raw 32-bit words.
template <typename T>
struct Raw {
  uint32_t w[kPerLane * sizeof(T) / 4];
};

// Largest magnitude of the 8 values as fp32 bits (magnitudes compare as integers; infinities and NaN come out
// largest), still within the lane; and the maximum over the 4 lanes of a block.
__device__ __forceinline__ uint32_t block_max(uint32_t m) {
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  return max(m, __shfl_xor_sync(0xffffffffu, m, 2));
}
__device__ __forceinline__ uint32_t amax_bits(const Raw<float>& r) {
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) m = max(m, r.w[i] & 0x7FFFFFFFu);
  return block_max(m);
}
// Two 16-bit magnitudes at a time.
__device__ __forceinline__ uint32_t amax_16(const uint32_t (&w)[kPerLane / 2]) {
  uint32_t m = w[0] & 0x7FFF7FFFu;
#pragma unroll
  for (int i = 1; i < kPerLane / 2; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
  return block_max(max(m & 0xFFFFu, m >> 16));
}
__device__ __forceinline__ uint32_t amax_bits(const Raw<__nv_bfloat16>& r) { return amax_16(r.w) << 16; }
__device__ __forceinline__ uint32_t amax_bits(const Raw<__half>& r) { return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(amax_16(r.w))))); }

template <typename T>
__device__ __forceinline__ float value(const Raw<T>& r, int i);
template <>
__device__ __forceinline__ float value<float>(const Raw<float>& r, int i) { return __uint_as_float(r.w[i]); }
template <>
__device__ __forceinline__ float value<__nv_bfloat16>(const Raw<__nv_bfloat16>& r, int i) {
  return __uint_as_float((i & 1) ? (r.w[i >> 1] & 0xFFFF0000u) : (r.w[i >> 1] << 16));
}
template <>
__device__ __forceinline__ float value<__half>(const Raw<__half>& r, int i) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>((i & 1) ? (r.w[i >> 1] >> 16) : (r.w[i >> 1] & 0xFFFFu))));
}

template <typename T, bool kVec>
__device__ __forceinline__ Raw<T> load8(const T* p) {
  Raw<T> r;
  if constexpr (kVec) {
#pragma unroll
    for (int j = 0; j < static_cast<int>(sizeof(r.w) / 16); ++j) {
      const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p) + j);
      r.w[4 * j] = v.x;
      r.w[4 * j + 1] = v.y;
      r.w[4 * j + 2] = v.z;
      r.w[4 * j + 3] = v.w;
    }
  } else {
    T v[kPerLane];
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) v[i] = p[i];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) r.w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kPerLane / 2; ++i) {
        r.w[i] = static_cast<uint32_t>(*reinterpret_cast<const unsigned short*>(&v[2 * i])) |
                 (static_cast<uint32_t>(*reinterpret_cast<const unsigned short*>(&v[2 * i + 1])) << 16);
      }
    }
  }
  return r;
}

// Two values -> one byte, `lo` in the low nibble (round to nearest even, saturating at 6).
__device__ __forceinline__ uint32_t e2m1_pair(float lo, float hi) {
  return static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(make_float2(lo, hi), __NV_E2M1, cudaRoundNearest));
}

// What a warp covers: rows row0 + r + 32 j and row0 + r + 1 + 32 j, columns from k0 on.
struct Tile {
  int64_t row0, k0;
  int r;          // even, below 32
  int rows;       // rows that exist from row0 on, at most 128
  int groups;     // scale blocks (128 of K) that exist: 1 or 2
  size_t scales;  // first byte of the warp's 32 in the first of them
};
__device__ __forceinline__ Tile tile_of(int64_t rows, int64_t K, unsigned tiles_k) {
  Tile t;
  const unsigned tile = blockIdx.x / kCtasPerTile;
  const unsigned rb = tile / tiles_k;
  const unsigned kt = tile - rb * tiles_k;
  t.r = 2 * static_cast<int>((blockIdx.x % kCtasPerTile) * kWarps + (threadIdx.x >> 5));
  t.row0 = static_cast<int64_t>(rb) * kTileRows;
  t.k0 = static_cast<int64_t>(kt) * kTileK;
  t.rows = static_cast<int>(rows - t.row0 < kTileRows ? rows - t.row0 : kTileRows);
  const int64_t k_groups = (K + 127) / 128;
  t.groups = k_groups - 2 * static_cast<int64_t>(kt) >= 2 ? 2 : 1;
  t.scales = (static_cast<size_t>(rb) * k_groups + 2 * static_cast<size_t>(kt)) * kScaleBlockBytes + static_cast<size_t>(t.r) * 16;
  return t;
}
// Row a (0..7) of the warp, in the order of their scale words.
__device__ __forceinline__ int warp_row(const Tile& t, int a) { return t.r + (a >> 2) + 32 * (a & 3); }

// Rows behind the last and blocks behind K get scale bytes of 127, so that every byte of the packed
// scales is defined.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads) quantize_mx4_kernel(const T* __restrict__ x, uint8_t* __restrict__ q, uint8_t* __restrict__ scales,
                                                                int64_t rows, int64_t K, int64_t row_stride, unsigned tiles_k) {
  const int lane = threadIdx.x & 31;
  const Tile t = tile_of(rows, K, tiles_k);
  const int64_t k = t.k0 + lane * kPerLane;
  const bool k_ok = k < K;
  const T* const src = x + t.row0 * row_stride + k;
  uint8_t* const dst = q + (t.row0 * K + k) / 2;
  Raw<T> raw[kRows];
#pragma unroll
  for (int a = 0; a < kRows; ++a) {
    const int r = warp_row(t, a);
    if (r < t.rows && k_ok) {
      raw[a] = load8<T, kVec>(src + r * row_stride);
    } else {
#pragma unroll
      for (int j = 0; j < static_cast<int>(sizeof(raw[a].w) / 4); ++j) raw[a].w[j] = 0u;
    }
  }
  uint32_t words[kRows];  // of lanes 0 and 16: the scale words of the rows
#pragma unroll
  for (int a = 0; a < kRows; ++a) {
    const int r = warp_row(t, a);
    const uint32_t amax = amax_bits(raw[a]);
    const uint32_t field = amax >> 23;  // biased exponent of the maximum; 0 below 2^-126
    uint32_t byte = field > 2u ? field - 2u : 0u;
    if (amax == 0u) byte = 127u;
    const bool bad = field == 255u;
    if (bad) byte = 255u;
    const float inv = __uint_as_float((254u - (bad ? 127u : byte)) << 23);
    uint32_t codes = 0u;
#pragma unroll
    for (int i = 0; i < kPerLane / 2; ++i) codes |= e2m1_pair(value<T>(raw[a], 2 * i) * inv, value<T>(raw[a], 2 * i + 1) * inv) << (8 * i);
    if (bad) codes = 0u;
    if (r < t.rows && k_ok) *reinterpret_cast<uint32_t*>(dst + r * (K / 2)) = codes;
    uint32_t word = byte << (8 * ((lane >> 2) & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    words[a] = word;
  }
  if ((lane & 15) == 0 && (lane >> 4) < t.groups) {
    uint4* const s = reinterpret_cast<uint4*>(scales + t.scales + (lane >> 4) * kScaleBlockBytes);
    s[0] = make_uint4(words[0], words[1], words[2], words[3]);
    s[1] = make_uint4(words[4], words[5], words[6], words[7]);
  }
}

// Rounding into the output type; for bf16 and fp32 it never rounds (two significant bits, and the
// smallest value, 2^-128, is a bf16 subnormal).
__device__ __forceinline__ void store8(float* p, const float (&v)[kPerLane]) {
  if ((reinterpret_cast<uintptr_t>(p) & 31u) != 0) {  // a caller's buffer may be aligned to 16 bytes only
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    return;
  }
  sm100::st_global_v8(p, __float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]), __float_as_uint(v[4]),
                      __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[kPerLane]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store8(__half* p, const float (&v)[kPerLane]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) dequantize_mx4_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scales, T* __restrict__ out,
                                                                  int64_t rows, int64_t K, unsigned tiles_k) {
  const int lane = threadIdx.x & 31;
  const Tile t = tile_of(rows, K, tiles_k);
  const int64_t k = t.k0 + lane * kPerLane;
  if (k >= K) return;
  const uint8_t* const src = q + (t.row0 * K + k) / 2;
  T* const dst = out + t.row0 * K + k;
  uint32_t codes[kRows];
#pragma unroll
  for (int a = 0; a < kRows; ++a) {
    const int r = warp_row(t, a);
    codes[a] = r < t.rows ? __ldcs(reinterpret_cast<const uint32_t*>(src + r * (K / 2))) : 0u;
  }
  const uint4* const s = reinterpret_cast<const uint4*>(scales + t.scales + (lane >> 4) * kScaleBlockBytes);
  const uint4 s0 = __ldg(s), s1 = __ldg(s + 1);
  const uint32_t words[kRows] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
  for (int a = 0; a < kRows; ++a) {
    const int r = warp_row(t, a);
    if (r >= t.rows) continue;
    const uint32_t byte = (words[a] >> (8 * ((lane >> 2) & 3))) & 255u;
    // 2^(byte - 127): byte 0 is a subnormal, 255 is NaN
    const float scale = byte == 255u ? __uint_as_float(0x7FC00000u) : (byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23));
    float v[kPerLane];
#pragma unroll
    for (int i = 0; i < kPerLane / 2; ++i) {
      const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>((codes[a] >> (8 * i)) & 0xFFu), __NV_E2M1);
      const float2 f = __half22float2(__half2(h));
      v[2 * i] = f.x * scale;
      v[2 * i + 1] = f.y * scale;
    }
    store8(dst + r * K, v);
  }
}

int check_shape(const char* who, int64_t rows, int64_t K, int dtype_q) {
  B200_REQUIRE(dtype_q == B200_MXE2M1, "%s: dtype_q=%d is not the block-scaled fp4 type", who, dtype_q);
  B200_REQUIRE(rows >= 1 && K >= 32 && K % 32 == 0, "%s: rows must be >= 1 and K a positive multiple of 32 (got %lld, %lld)", who, (long long)rows, (long long)K);
  B200_REQUIRE(rows < (1ll << 31) - 256 && K < (1ll << 31) - 256, "%s: rows and K must be below 2^31", who);
  return B200_OK;
}

int grid_for(const char* who, int64_t rows, int64_t K, unsigned* grid, unsigned* tiles_k) {
  const int64_t tk = (K + kTileK - 1) / kTileK, tiles = (rows + kTileRows - 1) / kTileRows * tk * kCtasPerTile;
  B200_REQUIRE(tiles < (1ll << 31), "%s: %lld x %lld values are more than one launch covers", who, (long long)rows, (long long)K);
  *grid = static_cast<unsigned>(tiles);
  *tiles_k = static_cast<unsigned>(tk);
  return B200_OK;
}

template <typename T>
int launch_quantize(const void* x, void* q, void* scales, int64_t rows, int64_t K, int64_t row_stride, cudaStream_t stream) {
  unsigned grid = 0, tiles_k = 0;
  const int rc = grid_for("quantize_mx", rows, K, &grid, &tiles_k);
  if (rc != B200_OK) return rc;
  // Vector loads need every row to start on a 16-byte boundary (a lane's 8 values then do, too).
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && (row_stride * static_cast<int64_t>(sizeof(T))) % 16 == 0;
  const T* xt = static_cast<const T*>(x);
  uint8_t* qb = static_cast<uint8_t*>(q);
  uint8_t* sb = static_cast<uint8_t*>(scales);
  if (vec) {
    quantize_mx4_kernel<T, true><<<grid, kThreads, 0, stream>>>(xt, qb, sb, rows, K, row_stride, tiles_k);
  } else {
    quantize_mx4_kernel<T, false><<<grid, kThreads, 0, stream>>>(xt, qb, sb, rows, K, row_stride, tiles_k);
  }
  b200::count_launch();
  B200_CUDA_OK(cudaGetLastError());
  return B200_OK;
}

template <typename T>
int launch_dequantize(const void* q, const void* scales, void* out, int64_t rows, int64_t K, cudaStream_t stream) {
  unsigned grid = 0, tiles_k = 0;
  const int rc = grid_for("dequantize_mx", rows, K, &grid, &tiles_k);
  if (rc != B200_OK) return rc;
  dequantize_mx4_kernel<T><<<grid, kThreads, 0, stream>>>(static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(scales), static_cast<T*>(out), rows, K, tiles_k);
  b200::count_launch();
  B200_CUDA_OK(cudaGetLastError());
  return B200_OK;
}

}  // namespace

extern "C" {

int b200_quantize_mx(const void* x, int32_t dtype_x, int64_t rows, int64_t K, int64_t row_stride, int32_t dtype_q, void* q, void* scales_packed, void* stream) {
  B200_REQUIRE(x != nullptr && q != nullptr && scales_packed != nullptr, "quantize_mx: NULL argument");
  const int rc = check_shape("quantize_mx", rows, K, dtype_q);
  if (rc != B200_OK) return rc;
  B200_REQUIRE(row_stride >= K || rows == 1, "quantize_mx: row_stride=%lld is below K=%lld", (long long)row_stride, (long long)K);
  B200_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(scales_packed)) & 15u) == 0, "quantize_mx: q and scales must be 16-byte aligned");
  const uintptr_t eb = dtype_x == B200_F32 ? 4u : 2u;
  B200_REQUIRE((reinterpret_cast<uintptr_t>(x) & (eb - 1u)) == 0, "quantize_mx: x must be aligned to its elements");
  const cudaStream_t s = b200::as_stream(stream);
  switch (dtype_x) {
    case B200_F32: return launch_quantize<float>(x, q, scales_packed, rows, K, row_stride, s);
    case B200_BF16: return launch_quantize<__nv_bfloat16>(x, q, scales_packed, rows, K, row_stride, s);
    case B200_F16: return launch_quantize<__half>(x, q, scales_packed, rows, K, row_stride, s);
    default: return b200::fail(B200_ERR_INVALID, "quantize_mx: dtype_x=%d is not f32, bf16 or f16", dtype_x);
  }
}

int b200_dequantize_mx(const void* q, const void* scales_packed, int32_t dtype_q, int64_t rows, int64_t K, int32_t dtype_out, void* out, void* stream) {
  B200_REQUIRE(q != nullptr && scales_packed != nullptr && out != nullptr, "dequantize_mx: NULL argument");
  const int rc = check_shape("dequantize_mx", rows, K, dtype_q);
  if (rc != B200_OK) return rc;
  B200_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(scales_packed) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0,
               "dequantize_mx: q, scales and out must be 16-byte aligned");
  const cudaStream_t s = b200::as_stream(stream);
  switch (dtype_out) {
    case B200_F32: return launch_dequantize<float>(q, scales_packed, out, rows, K, s);
    case B200_BF16: return launch_dequantize<__nv_bfloat16>(q, scales_packed, out, rows, K, s);
    case B200_F16: return launch_dequantize<__half>(q, scales_packed, out, rows, K, s);
    default: return b200::fail(B200_ERR_INVALID, "dequantize_mx: dtype_out=%d is not f32, bf16 or f16", dtype_out);
  }
}

}  // extern "C"
