// Block-scaled 8-bit floating point: quantise, give back, transpose.
//
// A block of 128 values (1 x 128, or 128 x 128 for weights) shares one power of two, 2^e with
//   e = min { e >= -127 : amax <= L 2^e },   amax = the block's largest finite magnitude,
// L = 448 (e4m3) or 57344 (e5m2); a block of zeros has e = 0.  Both L are 1.75 * 2^p (p = 8,
// 15), so for amax = m * 2^E, 1 <= m < 2, e = E - p + (m > 1.75): exact from the float's bits.
// A power of two is what the scaled matrix instruction takes (a byte, e + 127), its product
// with the values is exact, so a value is rounded ONCE, to nearest even, by the conversion;
// an infinity becomes the type's infinity (e5m2) or NaN (e4m3), a NaN stays NaN.
// A 16- or 32-bit input is read as it is: nothing is rounded before the conversion.
//
// All kernels here are bound by memory: 3 bytes move for each bfloat16 value that is quantised.
#include "fp8_launch.h"

#include <type_traits>

namespace gpuexp {

namespace {

typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;

constexpr int kQThreads = 256;

__device__ __forceinline__ uint32_t bits(float v) { return __float_as_uint(v); }

// finite magnitudes order as their bits; infinities and NaN count as zero
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = bits(v) & 0x7fffffffu;
  return b >= 0x7f800000u ? 0u : b;
}

template <int kType>
__device__ __forceinline__ int block_exponent(uint32_t amax) {
  constexpr int p = kType == kE4M3 ? 8 : 15;
  if (amax == 0) return 0;
  const int e = int(amax >> 23) - 127 - p + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < -127 ? -127 : e;  // (subnormal amax included: its exponent field is 0)
}

// 2^-e as a float: e in [-127, 120], so always a normal number
__device__ __forceinline__ float inv_scale(int e) { return __uint_as_float(uint32_t(127 - e) << 23); }

template <int kType>
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  int r = 0;
  if constexpr (kType == kE4M3) {
    r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, r, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
  } else {
    r = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, r, false);
    r = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, r, true);
  }
  return uint32_t(r);
}

template <int kType>
__device__ __forceinline__ void unpack4(uint32_t w, float* v) {
  typedef __attribute__((ext_vector_type(2))) float f32x2;
  f32x2 lo, hi;
  if constexpr (kType == kE4M3) {
    lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false);
    hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
  } else {
    lo = __builtin_amdgcn_cvt_pk_f32_bf8(int(w), false);
    hi = __builtin_amdgcn_cvt_pk_f32_bf8(int(w), true);
  }
  v[0] = lo[0];
  v[1] = lo[1];
  v[2] = hi[0];
  v[3] = hi[1];
}

template <int kX>
__device__ __forceinline__ float widen(const void* p, int64_t i) {
  if constexpr (kX == kBF16) return __uint_as_float(uint32_t(static_cast<const uint16_t*>(p)[i]) << 16);
  if constexpr (kX == kF16) return float(static_cast<const _Float16*>(p)[i]);
  if constexpr (kX == kF32) return static_cast<const float*>(p)[i];
}

// 8 consecutive values from element i of x; those behind the first n read as 0 and are not
// touched in memory.  kVec: i is a multiple of 8 elements on a 16-byte boundary.
template <int kX, bool kVec>
__device__ __forceinline__ void load8(const void* x, int64_t i, int n, float* v) {
  if (kVec && n >= 8) {
    if constexpr (kX == kF32) {
      const u32x4* p = reinterpret_cast<const u32x4*>(static_cast<const float*>(x) + i);
      const u32x4 a = p[0], b = p[1];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = __uint_as_float(a[j]);
        v[4 + j] = __uint_as_float(b[j]);
      }
    } else {
      const u32x4 a = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(x) + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (kX == kBF16) {
          v[2 * j] = __uint_as_float(a[j] << 16);
          v[2 * j + 1] = __uint_as_float(a[j] & 0xffff0000u);
        } else {
          typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
          const uint32_t w = a[j];
          const f16x2 h = __builtin_bit_cast(f16x2, w);
          v[2 * j] = float(h[0]);
          v[2 * j + 1] = float(h[1]);
        }
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = j < n ? widen<kX>(x, i + j) : 0.f;
}

template <int kX>
__device__ __forceinline__ uint32_t narrow(float v) {  // one rounding, to nearest even
  if constexpr (kX == kBF16) {
    const __bf16 h = (__bf16)v;
    return __builtin_bit_cast(uint16_t, h);
  } else {
    const _Float16 h = (_Float16)v;
    return __builtin_bit_cast(uint16_t, h);
  }
}

template <int kX, bool kVec>
__device__ __forceinline__ void store8(void* x, int64_t i, int n, const float* v) {
  if (kVec && n >= 8) {
    if constexpr (kX == kF32) {
      u32x4 a, b;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        a[j] = bits(v[j]);
        b[j] = bits(v[4 + j]);
      }
      u32x4* p = reinterpret_cast<u32x4*>(static_cast<float*>(x) + i);
      p[0] = a;
      p[1] = b;
    } else {
      u32x4 a;
#pragma unroll
      for (int j = 0; j < 4; ++j) a[j] = narrow<kX>(v[2 * j]) | (narrow<kX>(v[2 * j + 1]) << 16);
      *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(x) + i) = a;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < n) {
      if constexpr (kX == kF32) static_cast<float*>(x)[i + j] = v[j];
      else static_cast<uint16_t*>(x)[i + j] = uint16_t(narrow<kX>(v[j]));
    }
}

// the first n of 8 bytes; a tensor's rows start at multiples of 16 bytes and are padded to
// them, so a whole 8-byte store never leaves the row (n >= 1)
__device__ __forceinline__ void store_q8(uint8_t* q, u32x2 w) { *reinterpret_cast<u32x2*>(q) = w; }

template <int kType>
__device__ __forceinline__ u32x2 quantize8(const float* v, float inv) {
  return u32x2{pack4<kType>(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
               pack4<kType>(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv)};
}

__device__ __forceinline__ uint32_t max8(const float* v) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, finite_bits(v[j]));
  return m;
}

// largest of the 16 lanes that share a block's row
__device__ __forceinline__ uint32_t max16(uint32_t m) {
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) m = max(m, uint32_t(__shfl_xor(int(m), d)));
  return m;
}

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
template <int kX, int kType, bool kVec>
__global__ void __launch_bounds__(kQThreads)
quantize_rows_kernel(const void* __restrict__ x, int64_t ldx, int cols, uint32_t units, FastDiv nb, Fp8Out out) {
  const uint32_t u = blockIdx.x * (kQThreads / 16) + (threadIdx.x >> 4);
  if (u >= units) return;  // whole groups of 16 lanes
  const uint32_t row = div(u, nb), blk = u - row * nb.d;
  const int col = int(blk) * kFp8Block + (threadIdx.x & 15) * 8;
  float v[8];
  load8<kX, kVec>(x, int64_t(row) * ldx + col, cols - col, v);
  const int e = block_exponent<kType>(max16(max8(v)));
  if (col < cols) store_q8(out.q + int64_t(row) * out.ld + col, quantize8<kType>(v, inv_scale(e)));
  if ((threadIdx.x & 15) == 0) out.scale[int64_t(row) * out.lds + blk] = uint8_t(e + 127);
}

// ---- a 128 x 128 tile: 256 threads, each 8 rows x 8 columns ----
// Thread t holds rows (t/16)*8 + i and columns (t%16)*8 + j, so 16 lanes read a row's 128
// values together, a row's largest is 4 exchanges between those lanes, and the 8 bytes of one
// column are one 8-byte write into the transposed tile in LDS.
//   square: one scale for the tile.   rows: a scale for each row (out) and each column (outT).
// The LDS image is [column][row] bytes; the 8-byte slot of a column is swizzled by the column's
// group of 8 so that the 16 lanes of a write, 8 columns apart, fall into different banks.
__device__ __forceinline__ int slot(int col, int r8) { return col * 128 + ((r8 ^ ((col >> 3) & 15)) << 3); }

template <int kX, int kType, bool kSquare, bool kVec>
__global__ void __launch_bounds__(kQThreads)
quantize_tile_kernel(const void* __restrict__ x, int64_t ldx, int64_t rows, int64_t cols, uint32_t tiles_n,
                     Fp8Out out, Fp8Out outT) {
  __shared__ __attribute__((aligned(16))) uint8_t tile[128 * 128];
  __shared__ uint32_t colmax[4][128];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t r0 = int64_t(blockIdx.x / tiles_n) * 128;
  const int64_t c0 = int64_t(blockIdx.x % tiles_n) * 128;
  const int r8 = t >> 4, cj = (t & 15) * 8;
  const int64_t col = c0 + cj;
  const int ncol = col < cols ? int(cols - col < 8 ? cols - col : 8) : 0;
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = r0 + r8 * 8 + i;
    load8<kX, kVec>(x, row * ldx + col, row < rows ? ncol : 0, v[i]);
  }
  int ecol[8];
  if constexpr (kSquare) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, max8(v[i]));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = max(m, uint32_t(__shfl_xor(int(m), d)));
    if (lane == 0) colmax[wave][0] = m;
    __syncthreads();
    m = max(max(colmax[0][0], colmax[1][0]), max(colmax[2][0], colmax[3][0]));
    const int e = block_exponent<kType>(m);
#pragma unroll
    for (int j = 0; j < 8; ++j) ecol[j] = e;
    const float inv = inv_scale(e);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t row = r0 + r8 * 8 + i;
      if (out.q && row < rows && ncol > 0) store_q8(out.q + row * out.ld + col, quantize8<kType>(v[i], inv));
    }
    if (t == 0) {
      if (out.q) out.scale[(r0 / 128) * out.lds + c0 / 128] = uint8_t(e + 127);
      if (outT.q) outT.scale[(c0 / 128) * outT.lds + r0 / 128] = uint8_t(e + 127);
    }
  } else {
    uint32_t m[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) m[j] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) m[j] = max(m[j], finite_bits(v[i][j]));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = max(m[j], uint32_t(__shfl_xor(int(m[j]), 16)));
      m[j] = max(m[j], uint32_t(__shfl_xor(int(m[j]), 32)));
    }
    if (lane < 16) {
#pragma unroll
      for (int j = 0; j < 8; ++j) colmax[wave][cj + j] = m[j];
    }
    // rows, while the column maxima travel
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t row = r0 + r8 * 8 + i;
      const int e = block_exponent<kType>(max16(max8(v[i])));
      if (out.q && row < rows) {
        if (ncol > 0) store_q8(out.q + row * out.ld + col, quantize8<kType>(v[i], inv_scale(e)));
        if ((t & 15) == 0) out.scale[row * out.lds + c0 / 128] = uint8_t(e + 127);
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = cj + j;
      ecol[j] = block_exponent<kType>(max(max(colmax[0][c], colmax[1][c]), max(colmax[2][c], colmax[3][c])));
    }
    if (r8 == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < ncol) outT.scale[(col + j) * outT.lds + r0 / 128] = uint8_t(ecol[j] + 127);
    }
  }
  if (!outT.q) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float inv = inv_scale(ecol[j]);
    u32x2 w;
    w[0] = pack4<kType>(v[0][j] * inv, v[1][j] * inv, v[2][j] * inv, v[3][j] * inv);
    w[1] = pack4<kType>(v[4][j] * inv, v[5][j] * inv, v[6][j] * inv, v[7][j] * inv);
    *reinterpret_cast<u32x2*>(tile + slot(cj + j, r8)) = w;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) {  // 16 lanes write 128 bytes of one column
    const int c = i * 16 + (t >> 4), k8 = t & 15;
    if (c0 + c < cols && r0 + k8 * 8 < rows)
      store_q8(outT.q + (c0 + c) * outT.ld + r0 + k8 * 8, *reinterpret_cast<const u32x2*>(tile + slot(c, k8)));
  }
}

// ---- 8 bits -> 16 or 32 bits: exact but for the one rounding into f16 / bf16 (a value of 8
// bits times a power of two has at most 4 significant bits) ----
__device__ __forceinline__ float scaled(float v, int byte) {  // byte 255 is NaN
  return byte == 255 ? __uint_as_float(0x7fc00000u) : __builtin_ldexpf(v, byte - 127);
}

template <int kX, int kType, bool kVec>
__global__ void __launch_bounds__(kQThreads)
dequantize_kernel(Fp8In in, int cols, uint32_t units, FastDiv nb, int row_shift, void* __restrict__ x, int64_t ldx) {
  const uint32_t u = blockIdx.x * (kQThreads / 16) + (threadIdx.x >> 4);
  if (u >= units) return;
  const uint32_t row = div(u, nb), blk = u - row * nb.d;
  const int col = int(blk) * kFp8Block + (threadIdx.x & 15) * 8;
  if (col >= cols) return;
  const u32x2 w = *reinterpret_cast<const u32x2*>(in.q + int64_t(row) * in.ld + col);
  const int s = in.scale[int64_t(row >> row_shift) * in.lds + blk];
  float v[8];
  unpack4<kType>(w[0], v);
  unpack4<kType>(w[1], v + 4);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = scaled(v[j], s);
  store8<kX, kVec>(x, int64_t(row) * ldx + col, cols - col, v);
}

// ---- transpose: the layout of a tile is that of quantize_tile_kernel ----
// rows: every column of 128 rows gets its own scale.  Its largest magnitude is found without
// rounding: |q| 2^(e - 16) is a float for every e (the shift keeps the largest below infinity),
// and what falls below the smallest subnormal, which only blocks reach whose exponent is
// clamped anyway, still counts as not zero.  The new value is q 2^(e - e'), rounded once: with
// powers of two on both sides it changes only where it leaves the type's normal range, that is
// 2^-14 below its block's largest (e4m3).
template <int kType, bool kSquare>
__global__ void __launch_bounds__(kQThreads)
transpose_kernel(Fp8In in, int64_t rows, int64_t cols, uint32_t tiles_n, Fp8Out outT) {
  __shared__ __attribute__((aligned(16))) uint8_t tile[128 * 128];
  __shared__ uint32_t colmax[4][128];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t r0 = int64_t(blockIdx.x / tiles_n) * 128;
  const int64_t c0 = int64_t(blockIdx.x % tiles_n) * 128;
  const int r8 = t >> 4, cj = (t & 15) * 8;
  const int64_t col = c0 + cj;
  const bool on = col < cols;
  u32x2 w[8];
  int e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = r0 + r8 * 8 + i;
    const bool here = on && row < rows;
    w[i] = here ? *reinterpret_cast<const u32x2*>(in.q + row * in.ld + col) : u32x2{0, 0};
    e[i] = 127;
    if (!kSquare && here) e[i] = in.scale[row * in.lds + c0 / 128];
  }
  if constexpr (kSquare) {
    if (t == 0) outT.scale[(c0 / 128) * outT.lds + r0 / 128] = in.scale[(r0 / 128) * in.lds + c0 / 128];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      u32x2 o{0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i >> 2] |= ((w[i][j >> 2] >> (8 * (j & 3))) & 255u) << (8 * (i & 3));
      *reinterpret_cast<u32x2*>(tile + slot(cj + j, r8)) = o;
    }
  } else {
    float v[8][8];
    uint32_t m[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) m[j] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      unpack4<kType>(w[i][0], v[i]);
      unpack4<kType>(w[i][1], v[i] + 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (e[i] == 255) v[i][j] = __uint_as_float(0x7fc00000u);
        const uint32_t b = finite_bits(__builtin_ldexpf(v[i][j], e[i] - 127 - 16));
        const bool some = (bits(v[i][j]) & 0x7fffffffu) - 1u < 0x7f7fffffu;  // finite and not zero
        m[j] = max(m[j], some && b == 0 ? 1u : b);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = max(m[j], uint32_t(__shfl_xor(int(m[j]), 16)));
      m[j] = max(m[j], uint32_t(__shfl_xor(int(m[j]), 32)));
    }
    if (lane < 16) {
#pragma unroll
      for (int j = 0; j < 8; ++j) colmax[wave][cj + j] = m[j];
    }
    __syncthreads();
    int en[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = cj + j;
      const uint32_t top = max(max(colmax[0][c], colmax[1][c]), max(colmax[2][c], colmax[3][c]));
      constexpr int p = kType == kE4M3 ? 8 : 15;
      // as block_exponent, of the shifted magnitude
      const int ee = int(top >> 23) - 127 - p + 16 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
      en[j] = top == 0 ? 0 : top < 0x800000u || ee < -127 ? -127 : ee;
    }
    if (r8 == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < cols) outT.scale[(col + j) * outT.lds + r0 / 128] = uint8_t(en[j] + 127);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float q[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = __builtin_ldexpf(v[i][j], e[i] - 127 - en[j]);
      u32x2 o;
      o[0] = pack4<kType>(q[0], q[1], q[2], q[3]);
      o[1] = pack4<kType>(q[4], q[5], q[6], q[7]);
      *reinterpret_cast<u32x2*>(tile + slot(cj + j, r8)) = o;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = i * 16 + (t >> 4), k8 = t & 15;
    if (c0 + c < cols && r0 + k8 * 8 < rows)
      store_q8(outT.q + (c0 + c) * outT.ld + r0 + k8 * 8, *reinterpret_cast<const u32x2*>(tile + slot(c, k8)));
  }
}

bool wide_vec(const void* x, int xtype, int64_t ldx, int64_t rows) {
  const int64_t size = xtype == kF32 ? 4 : 2;
  return reinterpret_cast<uintptr_t>(x) % 16 == 0 && (rows <= 1 || (ldx * size) % 16 == 0);
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

// 16 lanes for each block of 128 values, and a launch has less than 2^32 threads
bool count_ok(int64_t rows, int64_t cols) {
  return rows >= 0 && cols >= 0 && rows < (int64_t(1) << 28) && cols < (int64_t(1) << 31) - 128 &&
         rows * ((cols + 127) / 128) < (int64_t(1) << 28) - 16;
}

}  // namespace

hipError_t launch_quantize_fp8(const void* x, int xtype, int64_t ldx, int64_t rows, int64_t cols, int type,
                               int block_rows, Fp8Out out, Fp8Out outT, hipStream_t stream) {
  if (!count_ok(rows, cols)) return hipErrorInvalidValue;
  if (rows == 0 || cols == 0) return hipSuccess;
  const uint32_t nb = uint32_t((cols + 127) / 128);
  const bool vec = wide_vec(x, xtype, ldx, rows);
  by_types(xtype, type, [&](auto kx, auto kt) {
    constexpr int X = decltype(kx)::value, T = decltype(kt)::value;
    if (block_rows == 1 && !outT.q) {
      const uint32_t units = uint32_t(rows) * nb;
      auto k = vec ? quantize_rows_kernel<X, T, true> : quantize_rows_kernel<X, T, false>;
      hipLaunchKernelGGL(k, dim3((units + 15) / 16), dim3(kQThreads), 0, stream, x, ldx, int(cols), units,
                         fast_div(nb), out);
    } else {
      const uint32_t tiles = uint32_t((rows + 127) / 128) * nb;
      auto k = block_rows == 1 ? (vec ? quantize_tile_kernel<X, T, false, true> : quantize_tile_kernel<X, T, false, false>)
                               : (vec ? quantize_tile_kernel<X, T, true, true> : quantize_tile_kernel<X, T, true, false>);
      hipLaunchKernelGGL(k, dim3(tiles), dim3(kQThreads), 0, stream, x, ldx, rows, cols, nb, out, outT);
    }
  });
  return hipGetLastError();
}

hipError_t launch_dequantize_fp8(Fp8In in, int64_t rows, int64_t cols, void* x, int xtype, int64_t ldx,
                                 hipStream_t stream) {
  if (!count_ok(rows, cols)) return hipErrorInvalidValue;
  if (rows == 0 || cols == 0) return hipSuccess;
  const uint32_t nb = uint32_t((cols + 127) / 128), units = uint32_t(rows) * nb;
  const bool vec = wide_vec(x, xtype, ldx, rows);
  by_types(xtype, in.type, [&](auto kx, auto kt) {
    constexpr int X = decltype(kx)::value, T = decltype(kt)::value;
    auto k = vec ? dequantize_kernel<X, T, true> : dequantize_kernel<X, T, false>;
    hipLaunchKernelGGL(k, dim3((units + 15) / 16), dim3(kQThreads), 0, stream, in, int(cols), units, fast_div(nb),
                       in.block_rows == 1 ? 0 : 7, x, ldx);
  });
  return hipGetLastError();
}

hipError_t launch_transpose_fp8(Fp8In in, int64_t rows, int64_t cols, Fp8Out outT, hipStream_t stream) {
  if (!count_ok(rows, cols)) return hipErrorInvalidValue;
  if (rows == 0 || cols == 0) return hipSuccess;
  const uint32_t nb = uint32_t((cols + 127) / 128), tiles = uint32_t((rows + 127) / 128) * nb;
  auto k = in.type == kE4M3 ? (in.block_rows == 1 ? transpose_kernel<kE4M3, false> : transpose_kernel<kE4M3, true>)
                            : (in.block_rows == 1 ? transpose_kernel<kE5M2, false> : transpose_kernel<kE5M2, true>);
  hipLaunchKernelGGL(k, dim3(tiles), dim3(kQThreads), 0, stream, in, rows, cols, nb, outT);
  return hipGetLastError();
}

}  // namespace gpuexp
