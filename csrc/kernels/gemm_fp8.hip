// C[M,N] = A[M,K] . B[N,K]^T of two operands in 8 bits (e4m3 or e5m2 each) with one power of two
// for each block of 128 along K (and 1 or 128 rows), C in bf16 or f16:
//   C[i][j] = sum over blocks b of 2^(ea[i][b] + eb[j][b]) * sum over k in b of a[i][k] b[j][k]
// v_mfma_scale_f32_16x16x128_f8f6f4 takes one such block of K per instruction with the two
// exponents as bytes (lane l holds row l % 16, k (l / 16) * 32 .. + 32, and that row's scale), so
// the scales cost no arithmetic, and its rate is twice bf16's.  All four k groups of a row share
// the scale, so which 32 of a block's 128 k a lane holds does not matter as long as A and B agree.
//
// Precision: the accumulators are 32-bit floats.  Inside the instruction, products of 8-bit
// values are aligned to the largest of their group and what lies about 2^-14 below it is cut off
// (measured; the older fp8 instructions do the same), which leaves a result 1.5e-5 off in norm on
// random operands -- a hundredth of the rounding to bf16 that follows, and 2^-10 of the 8-bit
// rounding that the largest product itself carries.  C is rounded once.
//
// Operands are read with raw buffer loads straight into LDS: a lane whose row or 16-byte chunk is
// past the end gets an offset past the buffer's end and reads zeros, so ragged sizes need no other
// path; where K ends inside a 16-byte chunk the fragments of the last block are masked, so what
// follows the last value in a row has no effect.
#include "fp8_launch.h"

#include <type_traits>

namespace gpuexp {

namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((address_space(3))) void* lds_ptr_t;

constexpr int kBK = 128;  // bytes of K per tile: one scale block
constexpr uint32_t kOob = 0x80000000u;

struct Operand {
  const uint8_t* q;
  const uint8_t* scale;
  int64_t ld, lds;
  int rows;   // of the operand
  int shift;  // 0 or 7: rows that share a scale, as a shift
};

__device__ __forceinline__ int swz(int row, int chunk) { return chunk ^ ((row >> 1) & 7); }

typedef decltype(__builtin_amdgcn_make_buffer_rsrc(static_cast<void*>(nullptr), 0, 0, 0)) rsrc_t;

// rows [row0, row0 + 128 or 256) of an operand as a raw buffer that ends with the operand's last row
__device__ __forceinline__ rsrc_t tile_rsrc(const Operand& o, int row0, int tile_rows, int K) {
  int left = o.rows - row0;
  left = left < tile_rows ? left : tile_rows;
  const uint32_t bytes = uint32_t(left - 1) * uint32_t(o.ld) + uint32_t((K + 15) & ~15);
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(o.q) + int64_t(row0) * o.ld, 0, int(bytes), 0x00020000);
}

// zeroes the bytes of a fragment whose k (within the block) is at or past `left`; the fragment is
// two 16-byte chunks c0, c1
__device__ __forceinline__ void mask_frag(i32x8& f, int c0, int c1, int left) {
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const int k = (w < 4 ? c0 * 16 : c1 * 16) + (w & 3) * 4;
    const int n = left - k;  // bytes of this word that are in range
    if (n < 4) f[w] = n <= 0 ? 0 : f[w] & int((1u << (8 * n)) - 1u);
  }
}

template <int kA, int kB>
__device__ __forceinline__ f32x4 mfma(const i32x8& a, const i32x8& b, f32x4 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, kA, kB, 0, sa, 0, sb);
}

template <typename T>
__device__ __forceinline__ uint16_t to16(float v) {
  const T h = (T)v;
  return __builtin_bit_cast(uint16_t, h);
}

// ---- 128 x 128 tile, 4 waves of 64 x 64, two tiles of K in LDS ----
template <int kA, int kB, typename TC>
__global__ void __launch_bounds__(256, 2)
gemm_fp8_128_kernel(Operand A, Operand B, uint16_t* __restrict__ C, int64_t ldc, int K) {
  __shared__ __attribute__((aligned(16))) uint8_t smem[2 * 2 * 128 * kBK];  // [buf][A|B][128][128]
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int nbn = (B.rows + 127) / 128;
  const int row_a = int(blockIdx.x / nbn) * 128, row_b = int(blockIdx.x % nbn) * 128;
  const rsrc_t ra = tile_rsrc(A, row_a, 128, K), rb = tile_rsrc(B, row_b, 128, K);
  const int nk = (K + kBK - 1) / kBK;

  auto stage = [&](int t) {
    uint8_t* buf = smem + (t & 1) * 2 * 128 * kBK;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int rblk = (wave * 4 + i) * 8, row = rblk + (lane >> 3);
      const int k = t * kBK + swz(row, lane & 7) * 16;
      const uint32_t oa = k < K ? uint32_t(row) * uint32_t(A.ld) + k : kOob;
      const uint32_t ob = k < K ? uint32_t(row) * uint32_t(B.ld) + k : kOob;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_ptr_t)(buf + rblk * kBK), 16, oa, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_ptr_t)(buf + (128 + rblk) * kBK), 16, ob, 0, 0, 0);
    }
  };

  // scales: one dword holds a row's next four blocks
  const uint32_t *pa[4], *pb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    int r = row_a + wm * 64 + i * 16 + (lane & 15);
    r = (r < A.rows ? r : A.rows - 1) >> A.shift;
    pa[i] = reinterpret_cast<const uint32_t*>(A.scale + int64_t(r) * A.lds);
    r = row_b + wn * 64 + i * 16 + (lane & 15);
    r = (r < B.rows ? r : B.rows - 1) >> B.shift;
    pb[i] = reinterpret_cast<const uint32_t*>(B.scale + int64_t(r) * B.lds);
  }
  uint32_t sa[4], sb[4];
  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (nk > 0) stage(0);
  for (int t = 0; t < nk; ++t) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // tile t landed for every wave; the other buffer is free
    if (t + 1 < nk) stage(t + 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if ((t & 3) == 0) {
        sa[i] = pa[i][t >> 2];
        sb[i] = pb[i][t >> 2];
      } else {
        sa[i] >>= 8;
        sb[i] >>= 8;
      }
    }
    const uint8_t* As = smem + (t & 1) * 2 * 128 * kBK;
    const uint8_t* Bs = As + 128 * kBK;
    const int c0 = lane >> 4, c1 = 4 + (lane >> 4);
    i32x8 af[4], bf[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int x = wm * 64 + i * 16 + (lane & 15), y = wn * 64 + i * 16 + (lane & 15);
      const i32x4 a0 = *reinterpret_cast<const i32x4*>(As + x * kBK + swz(x, c0) * 16);
      const i32x4 a1 = *reinterpret_cast<const i32x4*>(As + x * kBK + swz(x, c1) * 16);
      const i32x4 b0 = *reinterpret_cast<const i32x4*>(Bs + y * kBK + swz(y, c0) * 16);
      const i32x4 b1 = *reinterpret_cast<const i32x4*>(Bs + y * kBK + swz(y, c1) * 16);
      af[i] = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
      bf[i] = __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    const int left = K - t * kBK;
    if (left < kBK && (left & 15)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mask_frag(af[i], c0, c1, left);
        mask_frag(bf[i], c0, c1, left);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = mfma<kA, kB>(af[i], bf[j], acc[i][j], int(sa[i]), int(sb[j]));
  }

  // C/D map of 16x16x128: col = lane % 16, row = (lane / 16) * 4 + r
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = row_a + wm * 64 + i * 16 + (lane >> 4) * 4 + r;
        const int col = row_b + wn * 64 + j * 16 + (lane & 15);
        if (row < A.rows && col < B.rows) C[int64_t(row) * ldc + col] = to16<TC>(acc[i][j][r]);
      }
}

Operand operand(const Fp8In& in, int64_t rows) {
  return {in.q, in.scale, in.ld, in.lds, int(rows), in.block_rows == 1 ? 0 : 7};
}

template <typename F>
void by_types(int a, int b, int c, F f) {
  auto u = [&](auto ta, auto tb) {
    if (c == kBF16) f(ta, tb, __bf16{});
    else f(ta, tb, _Float16{});
  };
  auto t = [&](auto ta) {
    if (b == kE4M3) u(ta, std::integral_constant<int, kE4M3>{});
    else u(ta, std::integral_constant<int, kE5M2>{});
  };
  if (a == kE4M3) t(std::integral_constant<int, kE4M3>{});
  else t(std::integral_constant<int, kE5M2>{});
}

bool side_ok(const Fp8In& in, int64_t rows, int64_t K) {
  // a tile of 256 rows has to fit in a buffer's 31 bits
  return rows < (int64_t(1) << 31) - 256 && in.ld >= K && in.ld % 16 == 0 && in.ld <= (int64_t(1) << 22) &&
         in.lds % 4 == 0 && in.lds * 128 >= K && reinterpret_cast<uintptr_t>(in.q) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(in.scale) % 4 == 0;
}

}  // namespace

hipError_t launch_gemm_fp8(const GemmFp8Args& g, hipStream_t stream) {
  if (g.M < 0 || g.N < 0 || g.K < 0 || !side_ok(g.a, g.M, g.K) || !side_ok(g.b, g.N, g.K)) return hipErrorInvalidValue;
  if (g.M == 0 || g.N == 0) return hipSuccess;
  const int64_t tiles = ((g.M + 127) / 128) * ((g.N + 127) / 128);
  if (tiles >= (int64_t(1) << 24)) return hipErrorInvalidValue;  // 2^32 threads
  by_types(g.a.type, g.b.type, g.ctype, [&](auto ta, auto tb, auto tc) {
    constexpr int a = decltype(ta)::value, b = decltype(tb)::value;
    hipLaunchKernelGGL((gemm_fp8_128_kernel<a, b, decltype(tc)>), dim3(uint32_t(tiles)), dim3(256), 0, stream,
                       operand(g.a, g.M), operand(g.b, g.N), static_cast<uint16_t*>(g.c), g.ldc, int(g.K));
  });
  return hipGetLastError();
}

}  // namespace gpuexp
