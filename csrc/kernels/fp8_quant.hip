// Block-scaled 8-bit floating point: quantise, give back, transpose.
//
// A block of 128 values (1 x 128, or 128 x 128 for weights) shares one power of two, 2^e with
//   e = min { e >= -127 : amax <= L 2^e },   amax = the block's largest finite magnitude,
// L = 448 (e4m3) or 57344 (e5m2); a block of zeros has e = 0.  Both L are 1.75 * 2^p (p = 8,
// 15), so for amax = m * 2^E, 1 <= m < 2, e = E - p + (m > 1.75): exact from the float's bits.
// A power of two is what the scaled matrix instruction takes (a byte, e + 127) and what the scaled
// conversions of this chip take (a float with that byte as its exponent; they divide or multiply by it
// exactly, all 256 bytes checked), so a value is rounded ONCE, to nearest even, by the conversion; an
// infinity becomes the type's infinity (e5m2) or NaN (e4m3), a NaN stays NaN.
//
// All kernels here are bound by memory: 3 bytes move for each bfloat16 value that is quantised.
#include <type_traits>

#include "fp8_device.h"

namespace gpuexp {

namespace {

constexpr int kQThreads = 256;

// ---- 8 values next to each other: 4 words of 16-bit values, or 8 of 32 ----
template <int kX>
struct Eight {
  static constexpr int kWords = kX == kF32 ? 8 : 4;
  uint32_t w[kWords];
};

// 16 bytes at any element's address: one instruction (rows of odd length), as the memory unit takes
// unaligned accesses
typedef u32x4 u32x4_any __attribute__((aligned(2)));

// From element i of x; those behind the first n read as 0 and are not touched in memory.
template <int kX>
__device__ __forceinline__ Eight<kX> load8(const void* x, int64_t i, int n) {
  Eight<kX> v;
  if (n >= 8) {
    const u32x4_any* p = reinterpret_cast<const u32x4_any*>(static_cast<const char*>(x) + i * (kX == kF32 ? 4 : 2));
#pragma unroll
    for (int j = 0; j < Eight<kX>::kWords; ++j) v.w[j] = p[j >> 2][j & 3];
    return v;
  }
  // a row's end: the loads go out together (behind the end the first value again)
  uint32_t one[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) one[j] = 0;
  if (n > 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t at = i + (j < n ? j : 0);
      if constexpr (kX == kF32) one[j] = static_cast<const uint32_t*>(x)[at];
      else one[j] = static_cast<const uint16_t*>(x)[at];
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) one[j] = j < n ? one[j] : 0;
#pragma unroll
  for (int j = 0; j < Eight<kX>::kWords; ++j) {
    if constexpr (kX == kF32) v.w[j] = one[j];
    else v.w[j] = one[2 * j] | (one[2 * j + 1] << 16);
  }
  return v;
}

// largest finite magnitude of the eight
template <int kX>
__device__ __forceinline__ uint32_t max8(const Eight<kX>& v) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < Eight<kX>::kWords; ++j) m = max_mag<kX>(m, mag<kX>(v.w[j]));
  m = widest<kX>(m);
  if (m >= kInf<kX>) {  // hardly ever
    m = 0;
#pragma unroll
    for (int j = 0; j < Eight<kX>::kWords; ++j) m = max_mag<kX>(m, finite_mag<kX>(v.w[j]));
    m = widest<kX>(m);
  }
  return m;
}

// the columns' largest finite magnitudes over 8 rows, packed as the values are
template <int kX>
__device__ __forceinline__ void column_maxima(const Eight<kX> (&v)[8], uint32_t (&m)[Eight<kX>::kWords]) {
  constexpr int kWords = Eight<kX>::kWords;
  uint32_t all = 0;
#pragma unroll
  for (int j = 0; j < kWords; ++j) {
    m[j] = mag<kX>(v[0].w[j]);
#pragma unroll
    for (int i = 1; i < 8; ++i) m[j] = max_mag<kX>(m[j], mag<kX>(v[i].w[j]));
    all = max_mag<kX>(all, m[j]);
  }
  if (widest<kX>(all) >= kInf<kX>) {  // hardly ever
#pragma unroll
    for (int j = 0; j < kWords; ++j) {
      m[j] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m[j] = max_mag<kX>(m[j], finite_mag<kX>(v[i].w[j]));
    }
  }
}

// largest of 16 lanes next to each other: three xors and a mirror inside the lanes' data path
__device__ __forceinline__ uint32_t max16(uint32_t m) {
  m = max(m, uint32_t(__builtin_amdgcn_update_dpp(0, int(m), 0xB1, 0xf, 0xf, true)));   // lane ^ 1
  m = max(m, uint32_t(__builtin_amdgcn_update_dpp(0, int(m), 0x4E, 0xf, 0xf, true)));   // lane ^ 2
  m = max(m, uint32_t(__builtin_amdgcn_update_dpp(0, int(m), 0x141, 0xf, 0xf, true)));  // mirrored in 8
  m = max(m, uint32_t(__builtin_amdgcn_update_dpp(0, int(m), 0x140, 0xf, 0xf, true)));  // mirrored in 16
  return m;
}

template <int kX, int kType>
__device__ __forceinline__ u32x2 convert8(const Eight<kX>& v, float scale) {
  if constexpr (kX == kF32)
    return u32x2{convert4<kType>(v.w[0], v.w[1], v.w[2], v.w[3], scale), convert4<kType>(v.w[4], v.w[5], v.w[6], v.w[7], scale)};
  else
    return u32x2{convert4<kX, kType>(v.w[0], v.w[1], scale), convert4<kX, kType>(v.w[2], v.w[3], scale)};
}

// A tensor's rows start at multiples of 16 bytes and are padded to them, so an 8-byte access at a
// multiple of 8 below its columns never leaves the row.
__device__ __forceinline__ void store_q8(uint8_t* q, u32x2 w) { *reinterpret_cast<u32x2*>(q) = w; }

// u / d for u < 2^31: m = ceil(2^(31 + s) / d) with 2^(s-1) < d <= 2^s is at most 2^32 - 1
struct FastDiv {
  uint32_t d, m;
  int s;
};
FastDiv fast_div(uint32_t d) {
  int s = 0;
  while ((uint64_t(1) << s) < d) ++s;
  return {d, uint32_t(((uint64_t(1) << (31 + s)) + d - 1) / d), s};
}
__device__ __forceinline__ uint32_t div(uint32_t u, FastDiv f) {
  return uint32_t((uint64_t(u) * f.m) >> (31 + f.s));
}

// ---- 1 x 128 blocks along the rows: 16 lanes hold a block, 8 values each ----
template <int kX, int kType>
__global__ void __launch_bounds__(kQThreads)
quantize_rows_kernel(const void* __restrict__ x, int64_t ldx, int cols, uint32_t units, FastDiv nb, Fp8Out out) {
  const uint32_t u = blockIdx.x * (kQThreads / 16) + (threadIdx.x >> 4);
  if (u >= units) return;  // whole groups of 16 lanes
  const uint32_t row = div(u, nb), blk = u - row * nb.d;
  const int col = int(blk) * kFp8Block + (threadIdx.x & 15) * 8;
  const Eight<kX> v = load8<kX>(x, int64_t(row) * ldx + col, cols - col);
  const int byte = scale_byte<kType>(mag_bits<kX>(max16(max8<kX>(v))));
  if (col < cols) store_q8(out.q + int64_t(row) * out.ld + col, convert8<kX, kType>(v, scale_of(byte)));
  if ((threadIdx.x & 15) == 0) out.scale[int64_t(row) * out.lds + blk] = uint8_t(byte);
}

// ---- a 128 x 128 tile: 256 threads, each 8 rows x 8 columns ----
// Thread t holds rows (t/16)*8 + i and columns (t%16)*8 + j, so 16 lanes read a row's 128
// values together, a row's largest is 4 exchanges between those lanes, and the 8 bytes of one
// column are one 8-byte write into the transposed tile in LDS.  16-bit values stay as they were read,
// two columns to a word, in maxima and conversions alike: 3 instructions a value, and few registers.
//   square: one scale for the tile.   rows: a scale for each row (out) and each column (outT).
// The LDS image is [column][row] bytes; the 8-byte slot of a column is swizzled by the column's
// group of 8 so that the 16 lanes of a write, 8 columns apart, fall into different banks.
__device__ __forceinline__ int slot(int col, int r8) { return col * 128 + ((r8 ^ ((col >> 3) & 15)) << 3); }

// columns 2 c and 2 c + 1 (16-bit: of word c; 32-bit: columns c) of 8 rows, each 8 bytes to its slot
template <int kX, int kType, int kC>
__device__ __forceinline__ void column_to_tile(const Eight<kX> (&v)[8], uint8_t* tile, int cj, int r8, int lo, int hi) {
  if constexpr (kX == kF32) {
    const float s = scale_of(lo);
    *reinterpret_cast<u32x2*>(tile + slot(cj + kC, r8)) =
        u32x2{convert4<kType>(v[0].w[kC], v[1].w[kC], v[2].w[kC], v[3].w[kC], s),
              convert4<kType>(v[4].w[kC], v[5].w[kC], v[6].w[kC], v[7].w[kC], s)};
  } else {
    uint32_t a[4], b[4];  // the low and the high column, two rows to a word
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = __builtin_amdgcn_perm(v[2 * i + 1].w[kC], v[2 * i].w[kC], 0x05040100u);
      b[i] = __builtin_amdgcn_perm(v[2 * i + 1].w[kC], v[2 * i].w[kC], 0x07060302u);
    }
    const float s = scale_of(lo), t = scale_of(hi);
    *reinterpret_cast<u32x2*>(tile + slot(cj + 2 * kC, r8)) =
        u32x2{convert4<kX, kType>(a[0], a[1], s), convert4<kX, kType>(a[2], a[3], s)};
    *reinterpret_cast<u32x2*>(tile + slot(cj + 2 * kC + 1, r8)) =
        u32x2{convert4<kX, kType>(b[0], b[1], t), convert4<kX, kType>(b[2], b[3], t)};
  }
}

template <int kX, int kType>
__device__ __forceinline__ void columns_to_tile(const Eight<kX> (&v)[8], uint8_t* tile, int cj, int r8,
                                                const int (&bytes)[8]) {
  if constexpr (kX == kF32) {
    column_to_tile<kX, kType, 0>(v, tile, cj, r8, bytes[0], 0);
    column_to_tile<kX, kType, 1>(v, tile, cj, r8, bytes[1], 0);
    column_to_tile<kX, kType, 2>(v, tile, cj, r8, bytes[2], 0);
    column_to_tile<kX, kType, 3>(v, tile, cj, r8, bytes[3], 0);
    column_to_tile<kX, kType, 4>(v, tile, cj, r8, bytes[4], 0);
    column_to_tile<kX, kType, 5>(v, tile, cj, r8, bytes[5], 0);
    column_to_tile<kX, kType, 6>(v, tile, cj, r8, bytes[6], 0);
    column_to_tile<kX, kType, 7>(v, tile, cj, r8, bytes[7], 0);
  } else {
    column_to_tile<kX, kType, 0>(v, tile, cj, r8, bytes[0], bytes[1]);
    column_to_tile<kX, kType, 1>(v, tile, cj, r8, bytes[2], bytes[3]);
    column_to_tile<kX, kType, 2>(v, tile, cj, r8, bytes[4], bytes[5]);
    column_to_tile<kX, kType, 3>(v, tile, cj, r8, bytes[6], bytes[7]);
  }
}

// 16 lanes write 128 bytes of one column of the tile in LDS
__device__ __forceinline__ void tile_to_rows(const uint8_t* tile, Fp8Out outT, int64_t rows, int64_t cols, int64_t r0,
                                             int64_t c0) {
  const int t = threadIdx.x;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = i * 16 + (t >> 4), k8 = t & 15;
    if (c0 + c < cols && r0 + k8 * 8 < rows)
      store_q8(outT.q + (c0 + c) * outT.ld + r0 + k8 * 8, *reinterpret_cast<const u32x2*>(tile + slot(c, k8)));
  }
}

template <int kX, int kType, bool kSquare>
__global__ void __launch_bounds__(kQThreads, kX == kF32 ? 2 : 4)
quantize_tile_kernel(const void* __restrict__ x, int64_t ldx, int64_t rows, int64_t cols, uint32_t tiles_n,
                     Fp8Out out, Fp8Out outT) {
  constexpr int kWords = Eight<kX>::kWords;
  __shared__ __attribute__((aligned(16))) uint8_t tile[128 * 128];
  __shared__ uint32_t colmax[4][16 * kWords];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t r0 = int64_t(blockIdx.x / tiles_n) * 128;
  const int64_t c0 = int64_t(blockIdx.x % tiles_n) * 128;
  const int r8 = t >> 4, cj = (t & 15) * 8;
  const int64_t col = c0 + cj;
  const int ncol = col < cols ? int(cols - col < 8 ? cols - col : 8) : 0;
  const int nrow = int(rows - r0 - r8 * 8 < 8 ? rows - r0 - r8 * 8 : 8);  // may be <= 0
  Eight<kX> v[8];
  const int64_t first = (r0 + r8 * 8) * ldx + col;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = load8<kX>(x, first + i * ldx, i < nrow ? ncol : 0);
  uint32_t m[kWords];
  column_maxima<kX>(v, m);
  uint8_t* const q = out.q + (r0 + r8 * 8) * out.ld + col;
  int bytes[8];  // of the columns
  if constexpr (kSquare) {
    uint32_t all = m[0];
#pragma unroll
    for (int j = 1; j < kWords; ++j) all = max_mag<kX>(all, m[j]);
    all = max16(widest<kX>(all));
    all = max(all, uint32_t(__shfl_xor(int(all), 16)));
    all = max(all, uint32_t(__shfl_xor(int(all), 32)));
    if (lane == 0) colmax[wave][0] = all;
    __syncthreads();
    all = max(max(colmax[0][0], colmax[1][0]), max(colmax[2][0], colmax[3][0]));
    const int byte = scale_byte<kType>(mag_bits<kX>(all));
#pragma unroll
    for (int j = 0; j < 8; ++j) bytes[j] = byte;
    if (out.q && ncol > 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < nrow) store_q8(q + i * out.ld, convert8<kX, kType>(v[i], scale_of(byte)));
    }
    if (t == 0) {
      if (out.q) out.scale[(r0 / 128) * out.lds + c0 / 128] = uint8_t(byte);
      if (outT.q) outT.scale[(c0 / 128) * outT.lds + r0 / 128] = uint8_t(byte);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kWords; ++j) {
      m[j] = max_mag<kX>(m[j], uint32_t(__shfl_xor(int(m[j]), 16)));
      m[j] = max_mag<kX>(m[j], uint32_t(__shfl_xor(int(m[j]), 32)));
    }
    if (lane < 16) {
#pragma unroll
      for (int j = 0; j < kWords; ++j) colmax[wave][lane * kWords + j] = m[j];
    }
    if (out.q) {  // rows, while the columns' maxima travel
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int byte = scale_byte<kType>(mag_bits<kX>(max16(max8<kX>(v[i]))));
        if (i < nrow) {
          if (ncol > 0) store_q8(q + i * out.ld, convert8<kX, kType>(v[i], scale_of(byte)));
          if ((t & 15) == 0) out.scale[(r0 + r8 * 8 + i) * out.lds + c0 / 128] = uint8_t(byte);
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kWords; ++j) {
      const int c = (t & 15) * kWords + j;
      const uint32_t top = max_mag<kX>(max_mag<kX>(colmax[0][c], colmax[1][c]), max_mag<kX>(colmax[2][c], colmax[3][c]));
      if constexpr (kX == kF32) {
        bytes[j] = scale_byte<kType>(top);
      } else {
        bytes[2 * j] = scale_byte<kType>(mag_bits<kX>(top & 0xffffu));
        bytes[2 * j + 1] = scale_byte<kType>(mag_bits<kX>(top >> 16));
      }
    }
    if (r8 == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < ncol) outT.scale[(col + j) * outT.lds + r0 / 128] = uint8_t(bytes[j]);
    }
  }
  if (!outT.q) return;
  columns_to_tile<kX, kType>(v, tile, cj, r8, bytes);
  __syncthreads();
  tile_to_rows(tile, outT, rows, cols, r0, c0);
}

// ---- 8 bits -> 16 or 32 bits: exact but for the one rounding into f16 / bf16 (a value of 8
// bits times a power of two has at most 4 significant bits); a scale of NaN gives NaN ----
template <int kX, int kType, bool kHigh>
__device__ __forceinline__ void widen2(uint32_t w, float scale, uint32_t* out) {
  if constexpr (kX == kF32) {
    f32x2 v;
    if constexpr (kType == kE4M3) v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, kHigh);
    else v = __builtin_amdgcn_cvt_scalef32_pk_f32_bf8(w, scale, kHigh);
    out[0] = __float_as_uint(v[0]);
    out[1] = __float_as_uint(v[1]);
  } else if constexpr (kX == kBF16) {
    if constexpr (kType == kE4M3)
      *out = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, kHigh));
    else
      *out = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, scale, kHigh));
  } else {
    if constexpr (kType == kE4M3)
      *out = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, kHigh));
    else
      *out = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, scale, kHigh));
  }
}

template <int kX, int kType>
__global__ void __launch_bounds__(kQThreads)
dequantize_kernel(Fp8In in, int cols, uint32_t units, FastDiv nb, int row_shift, void* __restrict__ x, int64_t ldx) {
  const uint32_t u = blockIdx.x * (kQThreads / 16) + (threadIdx.x >> 4);
  if (u >= units) return;
  const uint32_t row = div(u, nb), blk = u - row * nb.d;
  const int col = int(blk) * kFp8Block + (threadIdx.x & 15) * 8;
  if (col >= cols) return;
  const u32x2 w = *reinterpret_cast<const u32x2*>(in.q + int64_t(row) * in.ld + col);
  const float s = scale_of(in.scale[int64_t(row >> row_shift) * in.lds + blk]);
  constexpr int kTwo = kX == kF32 ? 2 : 1;  // words of two values
  Eight<kX> v;
  widen2<kX, kType, false>(w[0], s, v.w);
  widen2<kX, kType, true>(w[0], s, v.w + kTwo);
  widen2<kX, kType, false>(w[1], s, v.w + 2 * kTwo);
  widen2<kX, kType, true>(w[1], s, v.w + 3 * kTwo);
  const int64_t i = int64_t(row) * ldx + col;
  const int n = cols - col;
  if (n >= 8) {
    u32x4_any* p = reinterpret_cast<u32x4_any*>(static_cast<char*>(x) + i * (kX == kF32 ? 4 : 2));
#pragma unroll
    for (int j = 0; j < Eight<kX>::kWords / 4; ++j) p[j] = u32x4{v.w[4 * j], v.w[4 * j + 1], v.w[4 * j + 2], v.w[4 * j + 3]};
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < n) {
      if constexpr (kX == kF32) static_cast<uint32_t*>(x)[i + j] = v.w[j];
      else static_cast<uint16_t*>(x)[i + j] = uint16_t(v.w[j >> 1] >> (16 * (j & 1)));
    }
}

// ---- transpose: the layout of a tile is that of quantize_tile_kernel ----
// square: bytes move, scales move.  rows: every column of 128 rows gets its own scale; the new value is
// q 2^(e - e'), rounded once: with powers of two on both sides it changes only where it leaves the type's
// normal range, that is 2^-14 below its block's largest (e4m3).
// While the tile's scales are within 2^64 of each other (always, in practice), its values relative to the
// largest scale are exact in bf16, and the columns go the way of quantize_tile_kernel's.  Otherwise the
// columns' largest are found by the bits of |q| as a 32-bit float plus the row's scale byte in the
// exponent's place, which order the products as unsigned integers (exponents sum to at most 142 + 254 <
// 512), and q is shifted by the difference of the exponents.
template <int kType, bool kHigh>
__device__ __forceinline__ f32x2 values2(uint32_t w) {
  if constexpr (kType == kE4M3) return __builtin_amdgcn_cvt_pk_f32_fp8(int(w), kHigh);
  else return __builtin_amdgcn_cvt_pk_f32_bf8(int(w), kHigh);
}
template <int kType>
__device__ __forceinline__ uint32_t shifted4(const uint32_t (&w)[4], int byte, const int (&shift)[4]) {
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t one = (w[i] >> (8 * byte)) & 255u;
    v[i] = __builtin_ldexpf(values2<kType, false>(one)[0], shift[i]);
  }
  const s16x2 lo = convert2<kType, false>(s16x2{0, 0}, v[0], v[1], 1.f);
  return __builtin_bit_cast(uint32_t, convert2<kType, true>(lo, v[2], v[3], 1.f));
}

template <int kType, bool kSquare>
__global__ void __launch_bounds__(kQThreads, 3)
transpose_kernel(Fp8In in, int64_t rows, int64_t cols, uint32_t tiles_n, Fp8Out outT) {
  __shared__ __attribute__((aligned(16))) uint8_t tile[128 * 128];
  __shared__ uint32_t colmax[4][128];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t r0 = int64_t(blockIdx.x / tiles_n) * 128;
  const int64_t c0 = int64_t(blockIdx.x % tiles_n) * 128;
  const int r8 = t >> 4, cj = (t & 15) * 8;
  const int64_t col = c0 + cj;
  const bool on = col < cols;
  const int nrow = int(rows - r0 - r8 * 8 < 8 ? rows - r0 - r8 * 8 : 8);
  const uint8_t* const q = in.q + (r0 + r8 * 8) * in.ld + col;
  u32x2 w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = on && i < nrow ? *reinterpret_cast<const u32x2*>(q + i * in.ld) : u32x2{0, 0};
  if constexpr (kSquare) {
    if (t == 0) outT.scale[(c0 / 128) * outT.lds + r0 / 128] = in.scale[(r0 / 128) * in.lds + c0 / 128];
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // columns 4 h .. + 4
      uint32_t o[4][2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {  // of rows 4 g .. + 4: 4 x 4 bytes
        const uint32_t a = w[4 * g][h], b = w[4 * g + 1][h], c = w[4 * g + 2][h], d = w[4 * g + 3][h];
        const uint32_t ab = __builtin_amdgcn_perm(b, a, 0x05010400u), ab2 = __builtin_amdgcn_perm(b, a, 0x07030602u);
        const uint32_t cd = __builtin_amdgcn_perm(d, c, 0x05010400u), cd2 = __builtin_amdgcn_perm(d, c, 0x07030602u);
        o[0][g] = __builtin_amdgcn_perm(cd, ab, 0x05040100u);
        o[1][g] = __builtin_amdgcn_perm(cd, ab, 0x07060302u);
        o[2][g] = __builtin_amdgcn_perm(cd2, ab2, 0x05040100u);
        o[3][g] = __builtin_amdgcn_perm(cd2, ab2, 0x07060302u);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) *reinterpret_cast<u32x2*>(tile + slot(cj + 4 * h + k, r8)) = u32x2{o[k][0], o[k][1]};
    }
  } else {
    const uint8_t* const scales = in.scale + r0 * in.lds + c0 / 128;
    // the tile's largest and smallest scale: each wave looks at all 128 rows
    const int last = int(rows - r0 < 128 ? rows - r0 : 128) - 1;
    const int s0 = scales[(lane < last ? lane : last) * in.lds], s1 = scales[(lane + 64 < last ? lane + 64 : last) * in.lds];
    int top = max(s0, s1), low = 255 - min(s0, s1);
    uint32_t both = uint32_t(top) | (uint32_t(low) << 16);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) both = max2x16(both, uint32_t(__shfl_xor(int(both), d)));
    top = int(both & 0xffffu);
    low = 255 - int(both >> 16);
    int e[8];  // the rows' scale bytes
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = scales[(r8 * 8 + i < last ? r8 * 8 + i : last) * in.lds];
    int bytes[8];  // the columns'
    if (top - low <= 64 && top < 255) {
      Eight<kBF16> v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float s = scale_of(e[i] - top + 127);
        widen2<kBF16, kType, false>(w[i][0], s, v[i].w);
        widen2<kBF16, kType, true>(w[i][0], s, v[i].w + 1);
        widen2<kBF16, kType, false>(w[i][1], s, v[i].w + 2);
        widen2<kBF16, kType, true>(w[i][1], s, v[i].w + 3);
      }
      uint32_t m[4];
      column_maxima<kBF16>(v, m);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m[j] = max2x16(m[j], uint32_t(__shfl_xor(int(m[j]), 16)));
        m[j] = max2x16(m[j], uint32_t(__shfl_xor(int(m[j]), 32)));
      }
      if (lane < 16) {
#pragma unroll
        for (int j = 0; j < 4; ++j) colmax[wave][lane * 4 + j] = m[j];
      }
      __syncthreads();
      // a column's byte is at least 0, relative to the largest scale at least 127 - top
      const int least = 127 - top;
      int rel[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = (t & 15) * 4 + j;
        const uint32_t a = max2x16(max2x16(colmax[0][c], colmax[1][c]), max2x16(colmax[2][c], colmax[3][c]));
        const uint32_t lo = a & 0xffffu, hi = a >> 16;
        rel[2 * j] = max(scale_byte<kType>(lo << 16), least);
        rel[2 * j + 1] = max(scale_byte<kType>(hi << 16), least);
        bytes[2 * j] = lo == 0 ? 127 : rel[2 * j] - least;
        bytes[2 * j + 1] = hi == 0 ? 127 : rel[2 * j + 1] - least;
      }
      columns_to_tile<kBF16, kType>(v, tile, cj, r8, rel);
    } else {
      constexpr uint32_t kNan = kType == kE4M3 ? 0x7f7f7f7fu : 0x7e7e7e7eu;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (e[i] == 255) w[i] = u32x2{kNan, kNan};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t one = (w[i][j >> 2] >> (8 * (j & 3))) & 255u;
          const uint32_t b = __float_as_uint(values2<kType, false>(one)[0]) & 0x7fffffffu;
          m = max(m, b - 1 < 0x7f7fffffu ? b + (uint32_t(e[i]) << 23) : 0u);  // finite and not zero
        }
        m = max(m, uint32_t(__shfl_xor(int(m), 16)));
        m = max(m, uint32_t(__shfl_xor(int(m), 32)));
        if (lane < 16) colmax[wave][cj + j] = m;
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = cj + j;
        const uint32_t m = max(max(colmax[0][c], colmax[1][c]), max(colmax[2][c], colmax[3][c]));
        constexpr int p = kType == kE4M3 ? 8 : 15;
        // as scale_byte, the exponent's field being 127 too large
        const int byte = int(m >> 23) - 127 - p + ((m & 0x7fffffu) > 0x600000u ? 1 : 0);
        bytes[j] = m == 0 ? 127 : byte < 0 ? 0 : byte;
        u32x2 o;
#pragma unroll
        for (int g = 0; g < 2; ++g)
          o[g] = shifted4<kType>({w[4 * g][j >> 2], w[4 * g + 1][j >> 2], w[4 * g + 2][j >> 2], w[4 * g + 3][j >> 2]}, j & 3,
                                 {e[4 * g] - bytes[j], e[4 * g + 1] - bytes[j], e[4 * g + 2] - bytes[j], e[4 * g + 3] - bytes[j]});
        *reinterpret_cast<u32x2*>(tile + slot(c, r8)) = o;
      }
    }
    if (r8 == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < cols) outT.scale[(col + j) * outT.lds + r0 / 128] = uint8_t(bytes[j]);
    }
  }
  __syncthreads();
  tile_to_rows(tile, outT, rows, cols, r0, c0);
}

template <typename F>
void by_types(int xtype, int type, F f) {
  auto t = [&](auto x) {
    if (type == kE4M3) f(x, std::integral_constant<int, kE4M3>{});
    else f(x, std::integral_constant<int, kE5M2>{});
  };
  if (xtype == kBF16) t(std::integral_constant<int, kBF16>{});
  else if (xtype == kF16) t(std::integral_constant<int, kF16>{});
  else t(std::integral_constant<int, kF32>{});
}

}  // namespace

hipError_t launch_quantize_fp8(const void* x, int xtype, int64_t ldx, int64_t rows, int64_t cols, int type,
                               int block_rows, Fp8Out out, Fp8Out outT, hipStream_t stream) {
  if (!fp8_blocks_ok(rows, cols)) return hipErrorInvalidValue;
  if (rows == 0 || cols == 0) return hipSuccess;
  const uint32_t nb = uint32_t((cols + 127) / 128);
  by_types(xtype, type, [&](auto kx, auto kt) {
    constexpr int X = decltype(kx)::value, T = decltype(kt)::value;
    if (block_rows == 1 && !outT.q) {
      const uint32_t units = uint32_t(rows) * nb;
      auto k = quantize_rows_kernel<X, T>;
      hipLaunchKernelGGL(k, dim3((units + 15) / 16), dim3(kQThreads), 0, stream, x, ldx, int(cols), units,
                         fast_div(nb), out);
    } else {
      const uint32_t tiles = uint32_t((rows + 127) / 128) * nb;
      auto k = block_rows == 1 ? quantize_tile_kernel<X, T, false> : quantize_tile_kernel<X, T, true>;
      hipLaunchKernelGGL(k, dim3(tiles), dim3(kQThreads), 0, stream, x, ldx, rows, cols, nb, out, outT);
    }
  });
  return hipGetLastError();
}

hipError_t launch_dequantize_fp8(Fp8In in, int64_t rows, int64_t cols, void* x, int xtype, int64_t ldx,
                                 hipStream_t stream) {
  if (!fp8_blocks_ok(rows, cols)) return hipErrorInvalidValue;
  if (rows == 0 || cols == 0) return hipSuccess;
  const uint32_t nb = uint32_t((cols + 127) / 128), units = uint32_t(rows) * nb;
  by_types(xtype, in.type, [&](auto kx, auto kt) {
    constexpr int X = decltype(kx)::value, T = decltype(kt)::value;
    auto k = dequantize_kernel<X, T>;
    hipLaunchKernelGGL(k, dim3((units + 15) / 16), dim3(kQThreads), 0, stream, in, int(cols), units, fast_div(nb),
                       in.block_rows == 1 ? 0 : 7, x, ldx);
  });
  return hipGetLastError();
}

hipError_t launch_transpose_fp8(Fp8In in, int64_t rows, int64_t cols, Fp8Out outT, hipStream_t stream) {
  if (!fp8_blocks_ok(rows, cols)) return hipErrorInvalidValue;
  if (rows == 0 || cols == 0) return hipSuccess;
  const uint32_t nb = uint32_t((cols + 127) / 128), tiles = uint32_t((rows + 127) / 128) * nb;
  auto k = in.type == kE4M3 ? (in.block_rows == 1 ? transpose_kernel<kE4M3, false> : transpose_kernel<kE4M3, true>)
                            : (in.block_rows == 1 ? transpose_kernel<kE5M2, false> : transpose_kernel<kE5M2, true>);
  hipLaunchKernelGGL(k, dim3(tiles), dim3(kQThreads), 0, stream, in, rows, cols, nb, outT);
  return hipGetLastError();
}

}  // namespace gpuexp
