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
// path; where K ends inside a 16-byte chunk, that chunk is a step of its own with its rest zeroed, so
// what follows the last value in a row has no effect.
#include <type_traits>

#include "fp8_device.h"

namespace gpuexp {

namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
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

// kByte: the byte of sa and sb that holds the scale
template <int kA, int kB, int kByte = 0>
__device__ __forceinline__ f32x4 mfma(const i32x8& a, const i32x8& b, f32x4 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, kA, kB, kByte, sa, kByte, sb);
}

template <typename T>
__device__ __forceinline__ uint16_t to16(float v) {
  const T h = (T)v;
  return __builtin_bit_cast(uint16_t, h);
}

// Where K ends inside a 16-byte chunk, the tiles stop before that chunk and this fragment makes one
// more step of it: the lanes that hold chunk 0 of `row` (others: on = false) read it with what
// follows K zeroed, the rest is zero.
__device__ __forceinline__ i32x8 tail_frag(rsrc_t rsrc, int64_t ld, int row, bool on, int K) {
  const int k = K & ~15;
  const uint32_t off = on ? uint32_t(row) * uint32_t(ld) + k : kOob;
  i32x4 v = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, 0));
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int n = K - k - 4 * w;  // bytes of this word that count
    if (n < 4) v[w] = n <= 0 ? 0 : v[w] & int((1u << (8 * n)) - 1u);
  }
  const i32x4 zero{0, 0, 0, 0};
  return __builtin_shufflevector(v, zero, 0, 1, 2, 3, 4, 5, 6, 7);
}
// the scale of `row` in K's last block
__device__ __forceinline__ int tail_scale(const Operand& o, int row, int K) {
  row = (row < o.rows ? row : o.rows - 1) >> o.shift;
  return o.scale[int64_t(row) * o.lds + (K - 1) / kBK];
}

// The first rows of this block's tile.  Blocks are dealt to the 8 XCDs in turn: each XCD gets a
// contiguous range of tiles, ordered in groups of kGroupM row panels x all column panels, so the tiles
// that run at once share panels in its L2.
template <int kBM, int kBN, int kGroupM>
__device__ __forceinline__ void tile_of_block(int M, int N, int& row_a, int& row_b) {
  const int nbn = (N + kBN - 1) / kBN, nbm = (M + kBM - 1) / kBM;
  const int nwg = nbm * nbn;
  const int orig = blockIdx.x;
  const int xcd = orig & 7, q = nwg >> 3, r = nwg & 7;
  const int wgid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (orig >> 3);
  const int in_group = kGroupM * nbn;
  const int first_m = (wgid / in_group) * kGroupM;
  const int gsize = nbm - first_m < kGroupM ? nbm - first_m : kGroupM;
  row_a = (first_m + (wgid % in_group) % gsize) * kBM;
  row_b = ((wgid % in_group) / gsize) * kBN;
}

// gfx9 encoding: vmcnt [3:0] and [15:14], expcnt [6:4], lgkmcnt [11:8]
constexpr int waitcnt_vm(int n) { return (n & 0xF) | (0x7 << 4) | (0xF << 8) | (((n >> 4) & 3) << 14); }
constexpr int kWaitLgkm0 = 0xF | (0x7 << 4) | (0x3 << 14);

template <int N>
__device__ __forceinline__ void wait_vm() {
  __builtin_amdgcn_s_waitcnt(waitcnt_vm(N));
}

// A fragment of 32 rows x 64 k: lane l holds row l % 32 and, with g = l / 32, the chunks 2 h + g and
// 2 h + g + 4 of the row's 8, h = 0, 1 for the two halves of a K tile.  Any assignment does that A
// and B share, and in this one the four places are xors of each other, alike for rows 32 apart.
struct FragAt {
  const uint8_t *p0, *p1;  // h = 0: chunks g, g + 4
  const uint8_t *p2, *p3;  // h = 1
};
__device__ __forceinline__ FragAt frag_at(const uint8_t* rows, int lane) {
  const int at = (lane & 31) * kBK, c = swz(lane & 31, lane >> 5) * 16;
  return {rows + at + c, rows + at + (c ^ 64), rows + at + (c ^ 32), rows + at + (c ^ 96)};
}
__device__ __forceinline__ void read_frag(const FragAt& f, int offset, i32x8 (&out)[2]) {
  const i32x4 a = *reinterpret_cast<const i32x4*>(f.p0 + offset);
  const i32x4 b = *reinterpret_cast<const i32x4*>(f.p1 + offset);
  const i32x4 c = *reinterpret_cast<const i32x4*>(f.p2 + offset);
  const i32x4 d = *reinterpret_cast<const i32x4*>(f.p3 + offset);
  out[0] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  out[1] = __builtin_shufflevector(c, d, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <int kA, int kB, int kByte>
__device__ __forceinline__ f32x16 mfma32(const i32x8& a, const i32x8& b, f32x16 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, kA, kB, kByte, sa, kByte, sb);
}

// C leaves through LDS, so that every global store is 16 bytes of a row.  D of 32x32x64: column (here
// a row of C, B being the first operand) = lane % 32, row (a column of C) = (e / 4) * 8 + (lane / 32) * 4
// + e % 4: a lane writes 8 bytes, the two halves of a wave the two halves of 16-byte chunks, which are
// xored with the row so that the 32 rows fall into different banks.
template <int kBN, typename TC>
__device__ __forceinline__ void tile_to_lds(uint8_t* smem, int row0, int col0, int lane, const f32x16& v) {
  const int row = row0 + (lane & 31);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int c = col0 / 8 + e;
    const u32x2 w{uint32_t(to16<TC>(v[4 * e])) | (uint32_t(to16<TC>(v[4 * e + 1])) << 16),
                  uint32_t(to16<TC>(v[4 * e + 2])) | (uint32_t(to16<TC>(v[4 * e + 3])) << 16)};
    *reinterpret_cast<u32x2*>(smem + row * kBN * 2 + ((c ^ (row & (kBN / 8 - 1) & 31)) << 4) + (lane >> 5) * 8) = w;
  }
}
template <int kBM, int kBN, int kThreads>
__device__ __forceinline__ void lds_to_c(const uint8_t* smem, uint16_t* C, int64_t ldc, int M, int N, int row_a,
                                         int row_b) {
  constexpr int kChunks = kBN / 8;
#pragma unroll 4
  for (int p = 0; p < kBM * kChunks / kThreads; ++p) {
    const int idx = p * kThreads + threadIdx.x;
    const int row = idx / kChunks, c = idx % kChunks;
    if (row_a + row >= M) break;
    const i32x4 v = *reinterpret_cast<const i32x4*>(smem + row * kBN * 2 + ((c ^ (row & (kChunks - 1) & 31)) << 4));
    const int col = row_b + c * 8;
    uint16_t* dst = C + int64_t(row_a + row) * ldc + col;
    if (col + 8 <= N) {
      typedef i32x4 wide_t __attribute__((aligned(2)));  // (one store at any address)
      *reinterpret_cast<wide_t*>(dst) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (col + e < N) dst[e] = uint16_t(uint32_t(v[e >> 1]) >> (16 * (e & 1)));
    }
  }
}

// the place, in f32x4, of a tile's sums over part `part` of K: [part][tile][32 x 32 fragment][4][lane]
template <int kBM, int kBN>
__device__ __forceinline__ int64_t part_at(int M, int N, int part, int tile_m, int tile_n) {
  const int64_t nbn = (N + kBN - 1) / kBN, nbm = (M + kBM - 1) / kBM;
  return ((part * nbm + tile_m) * nbn + tile_n) * (kBM * kBN / 4);
}

template <typename TC>
__device__ __forceinline__ void store4(uint16_t* dst, const f32x4& v, int columns) {
  typedef __attribute__((ext_vector_type(4))) uint16_t u16x4;
  const u16x4 h{to16<TC>(v[0]), to16<TC>(v[1]), to16<TC>(v[2]), to16<TC>(v[3])};
  if (columns >= 4) {
    typedef u16x4 wide_t __attribute__((aligned(2)));  // (one store at any address)
    *reinterpret_cast<wide_t*>(dst) = h;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < columns) dst[e] = h[e];
  }
}

// ---- 128 x 128 and 64 x 64 tiles, 4 waves, 2 or 4 tiles of K in LDS ----
// For sizes with too few 256 x 256 tiles to fill the card.  Waves are 2 x 2, each with a quarter of the
// tile.  While K tile t is multiplied from registers, t + 1 is read from LDS and t + kStages is loaded
// into the buffer that t left; one barrier per K tile.  Behind it every wave has its part of tile t + 1
// (a counted wait: loads complete in order) and has tile t in registers.  Past the end of K the loads go
// on out of range, so the count holds.  The K loop is unrolled by 4, so with 2 or 4 stages every LDS
// address is a constant.  The scales come as in the 256 x 256 kernel; a quad's words are read with its
// first K tile, and the next quad's loaded then, which the count covers.
// From memory a CU gets 56 GB/s this way, 0.30 us for a K tile of 64 x 64 (64 blocks; from the caches
// 0.18), and 8 stages get no more.  So where there are fewer tiles than CUs, K is cut into parts at multiples of 512 (a row's four
// scales are one word), blockIdx.y of them: TC = float stores the sums of a part in 32 bits as the lanes
// hold them, and join_parts_kernel adds them.
template <int kA, int kB, typename TC, int kBM, int kBN, int kStages>
__global__ void __launch_bounds__(256, 1)
gemm_fp8_tile_kernel(Operand A, Operand B, uint16_t* __restrict__ C, int64_t ldc, int K, float* __restrict__ sums) {
  constexpr bool kParts = std::is_same_v<TC, float>;
  constexpr int kStage = (kBM + kBN) * kBK, kScales = kStages * kStage, kRows = kBM + kBN;
  constexpr int kMI = kBM / 64, kNI = kBN / 64, kLoads = kRows / 32;  // 32-row fragments and loads per wave
  static_assert((kStages == 2 || kStages == 4) && kBM * kBN * 2 <= kScales, "slots are t % 4's, and C fits");
  __shared__ __attribute__((aligned(16))) uint8_t smem[kScales + 2 * kRows * 4];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  int row_a, row_b;
  tile_of_block<kBM, kBN, 8>(A.rows, B.rows, row_a, row_b);
  const int quads = (K + 4 * kBK - 1) / (4 * kBK);
  // this block's quads of K, and its K tiles and bytes, without a last part of 16 bytes
  const int q0 = kParts ? int(quads * blockIdx.y / gridDim.y) : 0;
  const int q1 = kParts ? int(quads * (blockIdx.y + 1) / gridDim.y) : quads;
  const int end = q1 == quads ? K & ~15 : q1 * 4 * kBK, t0 = q0 * 4, nk = (end + kBK - 1) / kBK;
  const rsrc_t ra = tile_rsrc(A, row_a, kBM, K), rb = tile_rsrc(B, row_b, kBN, K);

  // load i of a wave covers rows (wave + 4 i) * 8 .. + 8 of [A rows, B rows]
  const int lrow = lane >> 3;
  const int chunk = swz((wave & 1) * 8 + lrow, lane & 7) * 16;  // (the swizzle sees the parity of row / 8)
  const uint32_t va = uint32_t(lrow) * uint32_t(A.ld) + chunk, vb = uint32_t(lrow) * uint32_t(B.ld) + chunk;
  auto stage = [&](int t, int slot) {  // slot: t % kStages
    uint8_t* buf = smem + slot * kStage;
    const bool in = chunk < end - t * kBK;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = (wave + 4 * i) * 8;
      if (i < kBM / 32)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_ptr_t)(buf + row * kBK), 16, in ? va : kOob,
                                                 uint32_t(row) * uint32_t(A.ld) + t * kBK, 0, 0);
      else
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_ptr_t)(buf + row * kBK), 16, in ? vb : kOob,
                                                 uint32_t(row - kBM) * uint32_t(B.ld) + t * kBK, 0, 0);
    }
  };
  // scales: wave w loads those of rows w * 64 + lane of [A rows, B rows]
  const bool loads_scales = wave * 64 < kRows;
  const bool of_a = wave * 64 < kBM;
  const Operand& S = of_a ? A : B;
  int srow = (of_a ? row_a + wave * 64 : row_b + wave * 64 - kBM) + lane;
  srow = (srow < S.rows ? srow : S.rows - 1) >> S.shift;
  const uint8_t* sptr = S.scale + int64_t(srow) * S.lds;
  auto stage_scales = [&](int quad) {
    typedef __attribute__((address_space(1))) void* gptr_t;
    if (loads_scales)
      __builtin_amdgcn_global_load_lds((gptr_t)(sptr + (quad < quads ? quad : quads - 1) * 4),
                                       (lds_ptr_t)(smem + kScales + (quad & 1) * kRows * 4 + wave * 256), 4, 0, 0);
  };

  f32x16 acc[kMI][kNI];
#pragma unroll
  for (int i = 0; i < kMI; ++i)
#pragma unroll
    for (int j = 0; j < kNI; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  i32x8 af[2][kMI][2], bf[2][kNI][2];  // K tiles t and t + 1
  uint32_t sa[kMI], sb[kNI], sa_next[kMI], sb_next[kNI];
  const FragAt a_at = frag_at(smem + wm * (kBM / 2) * kBK, lane);
  const FragAt b_at = frag_at(smem + (kBM + wn * (kBN / 2)) * kBK, lane);
  auto read = [&](int slot, i32x8 (&fa)[kMI][2], i32x8 (&fb)[kNI][2]) {
    const int buf = slot * kStage;
#pragma unroll
    for (int i = 0; i < kMI; ++i) read_frag(a_at, buf + i * 32 * kBK, fa[i]);
#pragma unroll
    for (int j = 0; j < kNI; ++j) read_frag(b_at, buf + j * 32 * kBK, fb[j]);
  };
  auto read_scales = [&](int quad, uint32_t (&a)[kMI], uint32_t (&b)[kNI]) {
    const uint8_t* sc = smem + kScales + (quad & 1) * kRows * 4 + (lane & 31) * 4;
#pragma unroll
    for (int i = 0; i < kMI; ++i) a[i] = *reinterpret_cast<const uint32_t*>(sc + (wm * (kBM / 2) + i * 32) * 4);
#pragma unroll
    for (int j = 0; j < kNI; ++j)
      b[j] = *reinterpret_cast<const uint32_t*>(sc + (kBM + wn * (kBN / 2) + j * 32) * 4);
  };

  auto tile = [&](int t, auto byte_tag) {
    constexpr int byte = decltype(byte_tag)::value, cur = byte & 1;
    // tile t + 1 is here, and the reads of tile t have landed
    __builtin_amdgcn_s_waitcnt(waitcnt_vm((kStages - 2) * kLoads) & ~0xF00);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if constexpr (byte == 3) {
      read_scales((t + 1) >> 2, sa_next, sb_next);
      stage_scales(((t + 1) >> 2) + 1);
    }
    stage(t + kStages, byte % kStages);
    read((byte + 1) % kStages, af[1 - cur], bf[1 - cur]);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < kMI; ++i)
#pragma unroll
        for (int j = 0; j < kNI; ++j)
          acc[i][j] = mfma32<kB, kA, byte>(bf[cur][j][h], af[cur][i][h], acc[i][j], int(sb[j]), int(sa[i]));
    // the reads and loads go out between the MFMA: in a burst they would hold up the wave at issue
#pragma unroll
    for (int i = 0; i < 2 * kMI * kNI; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2 * (kMI + kNI) / (kMI * kNI), 0);
      __builtin_amdgcn_sched_group_barrier(0x010, kLoads / (2 * kMI * kNI), 0);
    }
    if constexpr (byte == 3) {
#pragma unroll
      for (int i = 0; i < kMI; ++i) sa[i] = sa_next[i];
#pragma unroll
      for (int j = 0; j < kNI; ++j) sb[j] = sb_next[j];
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  if (nk > t0) {
    stage_scales(q0);
    stage_scales(q0 + 1);
#pragma unroll
    for (int t = 0; t < kStages; ++t) stage(t0 + t, t);
    wait_vm<(kStages - 1) * kLoads>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read_scales(q0, sa, sb);
    read(0, af[0], bf[0]);
    for (int t = t0;; t += 4) {
      tile(t, std::integral_constant<int, 0>{});
      if (t + 1 >= nk) break;
      tile(t + 1, std::integral_constant<int, 1>{});
      if (t + 2 >= nk) break;
      tile(t + 2, std::integral_constant<int, 2>{});
      if (t + 3 >= nk) break;
      tile(t + 3, std::integral_constant<int, 3>{});
      if (t + 4 >= nk) break;
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();  // no load in flight, every wave's reads done: LDS is free
  }
  if (end != K && q1 == quads) {
#pragma unroll
    for (int i = 0; i < kMI; ++i) {
      const int x = wm * (kBM / 2) + i * 32 + (lane & 31);
      const i32x8 a = tail_frag(ra, A.ld, x, lane < 32, K);
      const int s = tail_scale(A, row_a + x, K);
#pragma unroll
      for (int j = 0; j < kNI; ++j) {
        const int y = wn * (kBN / 2) + j * 32 + (lane & 31);
        acc[i][j] = mfma32<kB, kA, 0>(tail_frag(rb, B.ld, y, lane < 32, K), a, acc[i][j], tail_scale(B, row_b + y, K),
                                      s);
      }
    }
  }
  if constexpr (kParts) {
    f32x4* at = reinterpret_cast<f32x4*>(sums) + part_at<kBM, kBN>(A.rows, B.rows, blockIdx.y, row_a / kBM, row_b / kBN);
#pragma unroll
    for (int i = 0; i < kMI; ++i)
#pragma unroll
      for (int j = 0; j < kNI; ++j) {
        const int f = (wm * kMI + i) * (kBN / 32) + wn * kNI + j;
        if (row_a + (wm * kMI + i) * 32 < A.rows && row_b + (wn * kNI + j) * 32 < B.rows)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            at[(f * 4 + g) * 64 + lane] = f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
      }
  } else {
#pragma unroll
    for (int i = 0; i < kMI; ++i)
#pragma unroll
      for (int j = 0; j < kNI; ++j)
        tile_to_lds<kBN, TC>(smem, wm * (kBM / 2) + i * 32, wn * (kBN / 2) + j * 32, lane, acc[i][j]);
    __syncthreads();
    lds_to_c<kBM, kBN, 256>(smem, C, ldc, A.rows, B.rows, row_a, row_b);
  }
}

// C from the parts' sums, added in the parts' order, so results do not depend on timing.  A thread has 4
// columns of a row, as they lie in the matrix instruction's result, and its loads are in flight together.
// Bound by the launch and its bytes: 3.3 to 4.2 us for 4 parts of 64 x 4096.  (Joining in the last block to arrive would want counters that someone has cleared: a launch too.)
template <typename TC, int kBM, int kBN>
__global__ void __launch_bounds__(256)
join_parts_kernel(const f32x4* __restrict__ sums, uint16_t* __restrict__ C, int64_t ldc, int M, int N, int parts) {
  constexpr int kOf = kBM * kBN / 4;  // threads of a tile
  const int64_t nbn = (N + kBN - 1) / kBN;
  const int64_t tile = int64_t(blockIdx.x) / (kOf / 256);
  const int at = int(blockIdx.x % (kOf / 256)) * 256 + threadIdx.x;
  const int lane = at & 63, g = (at >> 6) & 3, f = at >> 8;
  const int row = int(tile / nbn) * kBM + f / (kBN / 32) * 32 + (lane & 31);
  const int col = int(tile % nbn) * kBN + f % (kBN / 32) * 32 + g * 8 + (lane >> 5) * 4;
  if (row >= M || col >= N) return;
  const int64_t step = part_at<kBM, kBN>(M, N, 1, 0, 0);
  const f32x4* from = sums + tile * kOf + at;
  f32x4 v = *from;
#pragma unroll 4
  for (int p = 1; p < parts; ++p) v += from[p * step];
  store4<TC>(C + int64_t(row) * ldc + col, v, N - col);
}

// ---- 256 x 256 tile, 8 waves, two barriers per phase ----
// Waves are 2 along M x 4 along N, each a 128 x 64 block of C as 2 x 2 quadrants of 64 x 32; a
// K tile (128 bytes of K) is four phases, one quadrant of 8 MFMA (256 cycles) each.  A "group" is
// the 128 rows of a tile that one phase reads: A-M0 / A-M1 = the first / second 64 rows of each
// wave row, B-N0 / B-N1 = the first / second 32 rows of each wave column; 16 KiB, two 16-byte loads
// into LDS per thread.  Wave row 1 runs one barrier behind wave row 0, so that on every SIMD one
// wave's MFMA run while the other reads LDS and issues loads.  With Bf / Bs = B-N0 / B-N1 for even
// K tiles and the reverse for odd ones, phase p of K tile t
//   P1  loads A-M1(t+1), reads A-M0(t),   multiplies (M0, Bf)
//   P2  loads Bf(t+2),   reads Bs(t),     multiplies (M0, Bs)
//   P3  loads A-M0(t+2), reads A-M1(t),   multiplies (M1, Bs)
//   P4  loads Bs(t+2),   reads Bf(t+1),   multiplies (M1, Bf)
// so a group's rows are loaded 2 phases after their last read in that buffer and 6 before their
// next, and the wait in each phase (loads complete in order) retires the group issued 5 phases
// earlier, one phase before it is read.  Past the end of K the same loads go on with every lane out
// of range (zeros, no memory traffic), so the counts hold to the last tile.
//
// The rows' scales go the same way: 4 bytes hold a row's next 4 blocks, so each wave loads those of
// 64 rows with one instruction every 4 K tiles, 4 K tiles ahead, into 2 x 2 KiB of LDS; a lane keeps
// its 8 + 4 rows' words, and the instruction picks the byte: the K loop is unrolled by 4.
// LDS is [A|B][buffer][256][128]: every read of an operand is then within an immediate offset (16
// bits) of one address per chunk.
constexpr int kTile256 = 256 * kBK;
constexpr int kScales256 = 4 * kTile256;

// every wave's counted wait is behind this barrier; this wave's LDS reads have landed
__device__ __forceinline__ void barrier_before_mfma() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
  __builtin_amdgcn_sched_barrier(0);
}

__device__ __forceinline__ void barrier_after_mfma() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <int kA, int kB, typename TC>
__global__ void __launch_bounds__(512, 1)
gemm_fp8_256_kernel(Operand A, Operand B, uint16_t* __restrict__ C, int64_t ldc, int K) {
  __shared__ __attribute__((aligned(16))) uint8_t smem[kScales256 + 2 * 2048];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave >> 2, wc = wave & 3;

  int row_a, row_b;
  tile_of_block<256, 256, 4>(A.rows, B.rows, row_a, row_b);

  const int K16 = K & ~15;
  const int nk = (K16 + kBK - 1) / kBK;  // >= 2
  const rsrc_t ra = tile_rsrc(A, row_a, 256, K), rb = tile_rsrc(B, row_b, 256, K);

  // A load instruction covers 8 rows x 128 bytes; its first row is a multiple of 8 whose parity (in
  // eights) is that of `i` below, on which the swizzle depends.  The row and K tile go into the
  // scalar offset, which the range check counts: rows past the end read as zeros.  Chunks past K16
  // are sent past the buffer's end.
  const int lrow = lane >> 3;
  const int chunk[2] = {swz(lrow, lane & 7) * 16, swz(8 + lrow, lane & 7) * 16};
  const uint32_t va[2] = {uint32_t(lrow) * uint32_t(A.ld) + chunk[0], uint32_t(lrow) * uint32_t(A.ld) + chunk[1]};
  const uint32_t vb[2] = {uint32_t(lrow) * uint32_t(B.ld) + chunk[0], uint32_t(lrow) * uint32_t(B.ld) + chunk[1]};
  auto stage_a = [&](int half, int t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int rb8 = wave * 2 + i;
      const int row = (rb8 / 8) * 128 + half * 64 + (rb8 % 8) * 8;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_ptr_t)(smem + (t & 1) * kTile256 + row * kBK), 16,
                                               chunk[i] < K16 - t * kBK ? va[i] : kOob,
                                               uint32_t(row) * uint32_t(A.ld) + t * kBK, 0, 0);
    }
  };
  auto stage_b = [&](int half, int t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int rb8 = wave * 2 + i;
      const int row = (rb8 / 4) * 64 + half * 32 + (rb8 % 4) * 8;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_ptr_t)(smem + (2 + (t & 1)) * kTile256 + row * kBK), 16,
                                               chunk[i] < K16 - t * kBK ? vb[i] : kOob,
                                               uint32_t(row) * uint32_t(B.ld) + t * kBK, 0, 0);
    }
  };
  // scales: wave w < 4 loads A's rows w * 64 + lane, the others B's
  const Operand& S = wave < 4 ? A : B;
  int srow = (wave < 4 ? row_a : row_b) + (wave & 3) * 64 + lane;
  srow = (srow < S.rows ? srow : S.rows - 1) >> S.shift;
  const uint8_t* sptr = S.scale + int64_t(srow) * S.lds;
  const int quads = (nk + 3) / 4;
  auto stage_scales = [&](int quad) {  // the words of K tiles quad * 4 .. + 4; past the end the last again
    typedef __attribute__((address_space(1))) void* gptr_t;
    __builtin_amdgcn_global_load_lds((gptr_t)(sptr + (quad < quads ? quad : quads - 1) * 4),
                                     (lds_ptr_t)(smem + kScales256 + (quad & 1) * 2048 + wave * 256), 4, 0, 0);
  };

  f32x16 acc[2][2][2];  // [m half][n half][32 rows of A], each 32 columns of C x 32 rows
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[a][b][i][e] = 0.f;
  i32x8 af[2][2], b0[2], b1[2];  // [32 rows][k half]
  uint32_t sa[4], sb[2];
  const FragAt a_at = frag_at(smem + wr * 128 * kBK, lane), b_at = frag_at(smem + 2 * kTile256 + wc * 64 * kBK, lane);

  stage_scales(0);
  stage_b(0, 0); stage_a(0, 0); stage_b(1, 0); stage_a(1, 0);
  stage_b(1, 1); stage_a(0, 1); stage_b(0, 1);
  wait_vm<6>();
  __builtin_amdgcn_s_barrier();
  if (wr == 1) __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  read_frag(b_at, 0, b0);

  // B is the first operand, so that a lane's results lie along a row of C: 4 columns next to each
  // other.  (The two halves of K chain through an accumulator, so they are two MFMA apart.)
  auto quadrant = [&](f32x16 (&c)[2], const i32x8 (&bf)[2], int m, int n, auto byte_tag) {
    constexpr int byte = decltype(byte_tag)::value;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        c[i] = mfma32<kB, kA, byte>(bf[h], af[i][h], c[i], int(sb[n]), int(sa[m * 2 + i]));
  };
  auto read_a = [&](int buf, int half) {
#pragma unroll
    for (int i = 0; i < 2; ++i) read_frag(a_at, buf * kTile256 + (half * 64 + i * 32) * kBK, af[i]);
  };
  auto read_b = [&](int buf, int half, i32x8 (&bf)[2]) { read_frag(b_at, buf * kTile256 + half * 32 * kBK, bf); };

  auto tile = [&](int t, auto byte_tag) {  // byte: t % 4
    constexpr int byte = decltype(byte_tag)::value;
    constexpr bool odd = byte & 1;
    constexpr int cur = byte & 1;
    // P1
    if constexpr (byte == 0) {
      const uint8_t* sc = smem + kScales256 + ((t >> 2) & 1) * 2048 + (lane & 31) * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) sa[i] = *reinterpret_cast<const uint32_t*>(sc + (wr * 128 + i * 32) * 4);
#pragma unroll
      for (int i = 0; i < 2; ++i) sb[i] = *reinterpret_cast<const uint32_t*>(sc + 1024 + (wc * 64 + i * 32) * 4);
      stage_scales((t >> 2) + 1);
    }
    stage_a(1, t + 1);
    read_a(cur, 0);
    wait_vm<10>();
    barrier_before_mfma();
    if constexpr (odd) quadrant(acc[0][1], b1, 0, 1, byte_tag); else quadrant(acc[0][0], b0, 0, 0, byte_tag);
    barrier_after_mfma();
    // P2
    stage_b(odd ? 1 : 0, t + 2);
    if constexpr (odd) read_b(cur, 0, b0); else read_b(cur, 1, b1);
    wait_vm<10>();
    barrier_before_mfma();
    if constexpr (odd) quadrant(acc[0][0], b0, 0, 0, byte_tag); else quadrant(acc[0][1], b1, 0, 1, byte_tag);
    barrier_after_mfma();
    // P3
    stage_a(0, t + 2);
    read_a(cur, 1);
    wait_vm<10>();
    barrier_before_mfma();
    if constexpr (odd) quadrant(acc[1][0], b0, 1, 0, byte_tag); else quadrant(acc[1][1], b1, 1, 1, byte_tag);
    barrier_after_mfma();
    // P4 (after the last tile the read finds what an earlier tile left; nothing uses it)
    stage_b(odd ? 0 : 1, t + 2);
    if constexpr (odd) read_b(1 - cur, 0, b0); else read_b(1 - cur, 1, b1);
    wait_vm<10>();
    barrier_before_mfma();
    if constexpr (odd) quadrant(acc[1][1], b1, 1, 1, byte_tag); else quadrant(acc[1][0], b0, 1, 0, byte_tag);
    barrier_after_mfma();
  };
  for (int t = 0;; t += 4) {
    tile(t, std::integral_constant<int, 0>{});
    if (t + 1 >= nk) break;
    tile(t + 1, std::integral_constant<int, 1>{});
    if (t + 2 >= nk) break;
    tile(t + 2, std::integral_constant<int, 2>{});
    if (t + 3 >= nk) break;
    tile(t + 3, std::integral_constant<int, 3>{});
    if (t + 4 >= nk) break;
  }
  if (wr == 0) __builtin_amdgcn_s_barrier();  // wave row 1 is one barrier behind
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();  // no load in flight, every wave's reads done: LDS is free

  if (K != K16) {
    i32x8 at[4], bt[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = wr * 128 + i * 32 + (lane & 31);
      at[i] = tail_frag(ra, A.ld, row, lane < 32, K);
      sa[i] = tail_scale(A, row_a + row, K);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int row = wc * 64 + n * 32 + (lane & 31);
      bt[n] = tail_frag(rb, B.ld, row, lane < 32, K);
      sb[n] = tail_scale(B, row_b + row, K);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc[i >> 1][n][i & 1] = mfma32<kB, kA, 0>(bt[n], at[i], acc[i >> 1][n][i & 1], int(sb[n]), int(sa[i]));
  }

#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        tile_to_lds<256, TC>(smem, wr * 128 + m * 64 + i * 32, wc * 64 + n * 32, lane, acc[m][n][i]);
  __syncthreads();
  lds_to_c<256, 256, 512>(smem, C, ldc, A.rows, B.rows, row_a, row_b);
}

// ---- up to 16 rows of A (tokens of a decoding step): B goes from memory straight to registers ----
// Bound by B's bytes, read once.  A block takes 16 * kR rows of B; its waves divide K in units of 512
// bytes (four scale blocks, so that a row's four scales are one word), whose loads are in flight
// together, and many waves run on a CU.  Nothing is staged, since no two waves read the same of B (a ring
// in LDS for each wave, which reads whole lines, took the same time).  A comes from the caches; 32 rows
// of B per wave halve what is read of it.  The waves' sums are joined in LDS in the waves' order, so
// results do not depend on timing.
// B is the matrix instruction's first operand: a lane then holds 4 columns of C next to each other.
constexpr int kQuad = 4 * kBK;

// 32 values of 16 bits in 8, with the scale byte of the block they share with the lanes 16, 32 and 48 on
template <int kType, int kX>
__device__ __forceinline__ void quantize32(const i32x4 (&w)[4], i32x8& out, int& byte) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max_mag<kX>(m, mag<kX>(uint32_t(w[i >> 2][i & 3])));
  m = widest<kX>(m);
  if (m >= kInf<kX>) {  // hardly ever
    m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max_mag<kX>(m, finite_mag<kX>(uint32_t(w[i >> 2][i & 3])));
    m = widest<kX>(m);
  }
  m = max(m, uint32_t(__shfl_xor(int(m), 16)));
  m = max(m, uint32_t(__shfl_xor(int(m), 32)));
  byte = scale_byte<kType>(mag_bits<kX>(m));
  const float scale = scale_of(byte);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    out[i] = int(convert4<kX, kType>(uint32_t(w[i >> 1][(i & 1) * 2]), uint32_t(w[i >> 1][(i & 1) * 2 + 1]), scale));
}

// kWide >= 0: A is [M][ld] values of 16 bits (WideType kWide, K a multiple of 16), quantised to kA on
// their way as quantize_fp8 does: a lane has 32 values of a row's block, its three neighbours 16 lanes
// apart the others.
template <int kA, int kB, int kR, int kWide>
__global__ void __launch_bounds__(1024)
gemm_fp8_rows_kernel(Operand A, Operand B, uint16_t* __restrict__ C, int64_t ldc, int K, int c_is_f16) {
  __shared__ f32x4 part[16 * kR * 64];  // [wave][kR][lane]
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int row_b = blockIdx.x * (16 * kR);
  const int K16 = K & ~15;
  const int nk = (K16 + kBK - 1) / kBK, quads = (nk + 3) / 4;
  const int q0 = quads * wave / waves, q1 = quads * (wave + 1) / waves;
  const rsrc_t ra = tile_rsrc(A, 0, 16, kWide < 0 ? K : 2 * K), rb = tile_rsrc(B, row_b, 16 * kR, K);
  const int l15 = lane & 15, chunk = (lane >> 4) * 16;  // this lane's chunks of a block: chunk, chunk + 64

  const uint32_t* psb[kR];
#pragma unroll
  for (int r = 0; r < kR; ++r) {
    int n = row_b + r * 16 + l15;
    n = (n < B.rows ? n : B.rows - 1) >> B.shift;
    psb[r] = reinterpret_cast<const uint32_t*>(B.scale + int64_t(n) * B.lds);
  }
  const uint32_t* psa = nullptr;
  if constexpr (kWide < 0)
    psa = reinterpret_cast<const uint32_t*>(A.scale + int64_t((l15 < A.rows ? l15 : A.rows - 1) >> A.shift) * A.lds);
  // One scale block (128 bytes of K) of 16 rows; past K16 zeros.  `first`: which of its two chunks a lane
  // loads first.  Every other row of A the other half of its line: 16 x 64 bytes of equal halves take the
  // first-level cache twice as long (16 x 1024 x 4096 6.3 us, so 4.7).  B's rows so too where the card is
  // not full (16 x 1024 x 16384 18.2 / 15.5); else whole lines in turn come faster from memory.  32 rows of
  // B gain nothing (16 x 8192 x 8192 15.9 / 16.8).
  const int first_a = kR == 1 ? (l15 & 1) * 64 : 0, first_b = gridDim.x < 256 ? first_a : 0;
  auto load = [&](rsrc_t rsrc, uint32_t at, int k, int first) {
    const i32x4 x = __builtin_bit_cast(
        i32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, chunk + first < K16 - k ? at + first : kOob, k, 0));
    const i32x4 y = __builtin_bit_cast(
        i32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, chunk + (first ^ 64) < K16 - k ? at + (first ^ 64) : kOob, k, 0));
    return __builtin_shufflevector(first ? y : x, first ? x : y, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  const uint32_t at_a = uint32_t(l15) * uint32_t(A.ld) + (kWide < 0 ? chunk : 2 * chunk), at_b = uint32_t(l15) * uint32_t(B.ld) + chunk;

  f32x4 acc[kR];
#pragma unroll
  for (int r = 0; r < kR; ++r) acc[r] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int q = q0; q < q1; ++q) {
    i32x8 a[4], b[kR][4];
    i32x4 wide[4][4];  // of a block, the values of chunk and of chunk + 64
    uint32_t sb[kR], sa = 0;
    if constexpr (kWide >= 0) {  // first: loads complete in order, and A is quantised while B comes
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = q * kQuad + i * kBK;
          const bool in = (j < 2 ? chunk : chunk + 64) < K - k;
          wide[i][j] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                     ra, in ? at_a + (j >> 1) * 128 + (j & 1) * 16 : kOob, 2 * k, 0));
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int r = 0; r < kR; ++r) b[r][i] = load(rb, at_b + r * 16 * uint32_t(B.ld), q * kQuad + i * kBK, first_b);
      if constexpr (kWide < 0) a[i] = load(ra, at_a, q * kQuad + i * kBK, first_a);
    }
#pragma unroll
    for (int r = 0; r < kR; ++r) sb[r] = psb[r][q];
    if constexpr (kWide < 0) {
      sa = psa[q];
    } else {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int byte;
        quantize32<kA, kWide>(wide[i], a[i], byte);
        sa |= uint32_t(byte) << (8 * i);
      }
    }
    // behind K the scales are whatever pads their rows, and the values are zeros: 2^0 will do
    const int blocks = nk - q * 4;
    const uint32_t pad = blocks >= 4 ? 0u : 0xffffffffu << (8 * blocks);
    sa = (sa & ~pad) | (0x7f7f7f7fu & pad);
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      sb[r] = (sb[r] & ~pad) | (0x7f7f7f7fu & pad);
      acc[r] = mfma<kB, kA, 0>(b[r][0], a[0], acc[r], int(sb[r]), int(sa));
      acc[r] = mfma<kB, kA, 1>(b[r][1], a[1], acc[r], int(sb[r]), int(sa));
      acc[r] = mfma<kB, kA, 2>(b[r][2], a[2], acc[r], int(sb[r]), int(sa));
      acc[r] = mfma<kB, kA, 3>(b[r][3], a[3], acc[r], int(sb[r]), int(sa));
    }
  }
  if (kWide < 0 && K != K16 && wave == waves - 1) {
    const i32x8 a = tail_frag(ra, A.ld, l15, lane < 16, K);
    const int s = tail_scale(A, l15, K);
#pragma unroll
    for (int r = 0; r < kR; ++r)
      acc[r] = mfma<kB, kA>(tail_frag(rb, B.ld, r * 16 + l15, lane < 16, K), a, acc[r],
                            tail_scale(B, row_b + r * 16 + l15, K), s);
  }
#pragma unroll
  for (int r = 0; r < kR; ++r) part[(wave * kR + r) * 64 + lane] = acc[r];
  __syncthreads();
  for (int i = threadIdx.x; i < kR * 64; i += blockDim.x) {
    f32x4 v = part[i];
    for (int w = 1; w < waves; ++w) v += part[w * kR * 64 + i];
    const int l = i & 63, r = i >> 6;
    const int row = l & 15, col = row_b + r * 16 + (l >> 4) * 4;
    if (row >= A.rows) continue;
    uint16_t h[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = c_is_f16 ? to16<_Float16>(v[e]) : to16<__bf16>(v[e]);
    uint16_t* dst = C + int64_t(row) * ldc + col;
    if (col + 4 <= B.rows) {
      typedef __attribute__((ext_vector_type(4))) uint16_t u16x4;
      typedef u16x4 wide_t __attribute__((aligned(2)));  // (one store at any address)
      *reinterpret_cast<wide_t*>(dst) = u16x4{h[0], h[1], h[2], h[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < B.rows) dst[e] = h[e];
    }
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

// a tile of 256 rows has to fit in a buffer's 31 bits
constexpr int64_t kMaxRows = (int64_t(1) << 31) - 256, kMaxLd = int64_t(1) << 22;

bool side_ok(const Fp8In& in, int64_t rows, int64_t K) {
  return rows < kMaxRows && in.ld >= K && in.ld % 16 == 0 && in.ld <= kMaxLd &&
         in.lds % 4 == 0 && in.lds * 128 >= K && reinterpret_cast<uintptr_t>(in.q) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(in.scale) % 4 == 0;
}

}  // namespace

namespace {

// What a call takes on this card, in microseconds, by the kernel and the parts of K: a line in the tiles
// of K (`nk`) for each round of 256 blocks, whose slope grows with the part of the card that loads at
// once.  In parts there is a second kernel and its bytes, and 1 us for a launch and a workspace more.
// The numbers are those of 600 random sizes (1 to 8192 x 64 to 16384 x 128 to 16384, B in the caches and
// from memory) with which the choice costs least: on 520 others 0.6 % against the fastest kernel in the
// mean, up to 16 rows 1.3 %, on 160 more 0.7 and 0.6 %.  Examples,
// B from memory, us:                          128 x 128   two per CU   256 x 256   64 x 64
//   256 x 4096 x 4096                          21.9        30.3         42.7        12.1
//   1024 x 4096 x 4096                         23.1        31.4         42.4        33.6
//   4096 x 4096 x 4096 (from the caches)       76.4        64.0         55.9        101.3
//                                             few rows   32 of B per wave   64 x 64
//   1 / 16 x 4096 x 8192                       9.4 / 10.9   11.6 / 15.1      18.7 / 19.1
//   1 / 16 x 8192 x 8192                       16.0 / 19.4  14.2 / 16.0      19.5 / 20.0
//   1 / 16 x 16384 x 2048                      8.5 / 9.9    8.8 / 9.6        8.3 / 8.4
//                                             whole   in parts
//   17 x 1024 x 8192                           18.4    8.7 (16 of 64 x 64)
//   64 x 4096 x 14336                          39.1    18.0 (4 of 64 x 64)
//   512 x 4096 x 14336                         64      51 (2 of 128 x 128)
double estimate_us(int variant, int64_t M, int64_t blocks, double nk) {
  const double rounds = blocks <= 256 ? 1 : double((blocks + 255) >> 8);
  const double full = blocks < 256 ? double(blocks) * (1.0 / 256) : 1;
  switch (variant) {
    case 1: return 2.2 + rounds * (3.7 + (0.38 + 0.14 * full) * nk);
    case 2: return 0.3 + rounds * (13 + (1.05 + 0.2 * full) * nk);
    case 3: return 1.1 + rounds * (0.19 + (0.068 + 0.002 * double(M)) * nk);
    case 4: return 2.7 + rounds * (1 + (0.165 + 0.05 * full) * nk);
    case 5: return 3.9 + rounds * (1.9 + (0.4 + 0.125 * full) * nk);
    default: return 2 + rounds * (0.1 + (0.117 + 0.001 * double(M)) * nk);
  }
}

}  // namespace

// waves of a few-rows block: each takes at least a unit of 512 bytes of K
static int rows_waves(int64_t K) {
  const int64_t quads = ((K & ~int64_t(15)) + 4 * kBK - 1) / (4 * kBK);
  int waves = 1;
  while (waves < 16 && waves < quads) waves *= 2;
  return waves;
}

// whether a launch has less than 2^32 threads
static bool grid_ok(int64_t variant, int64_t parts, int64_t M, int64_t N, int64_t K) {
  const auto blocks = [](int64_t n, int64_t edge) { return (n + edge - 1) / edge; };
  constexpr int64_t kThreads = int64_t(1) << 32;
  if (variant == 3 || variant == 6) return blocks(N, variant == 3 ? 16 : 32) * rows_waves(K) * 64 < kThreads;
  if (variant == 2) return blocks(M, 256) * blocks(N, 256) * 512 < kThreads;
  const int64_t edge = variant == 4 ? 64 : 128;
  return blocks(M, edge) * blocks(N, edge) * (parts > 1 ? 16 : 1) * 256 < kThreads;  // (16: join_parts_kernel's)
}

// variant 0 = by the sizes, 1 = 128 x 128 tile, 2 = 256 x 256 tile, 3 = few rows (M <= 16), 4 = 64 x 64
// tile, 5 = 128 x 128 tile with two K tiles in LDS (two blocks per CU), 6 = few rows, 32 of B per wave;
// parts 0 = by the sizes, with a variant 1
GemmFp8Plan plan_gemm_fp8(int64_t M, int64_t N, int64_t K, int64_t variant, int64_t parts) {
  const auto takes = [&](int64_t v, int64_t p) {
    return (v == 2 ? K >= kBK + 16 : v == 3 || v == 6 ? M <= 16 : v >= 1 && v <= 5) && grid_ok(v, p, M, N, K);
  };
  const int64_t quads = (K + 4 * kBK - 1) / (4 * kBK);
  if (variant != 0) {
    const bool ok = takes(variant, parts) && parts >= 0 &&
                    (parts <= 1 || ((variant == 1 || variant == 4) && parts <= 16 && parts <= quads));
    return {ok ? int(variant) : -1, ok && parts > 1 ? int(parts) : 1};
  }
  if (parts < 0 || parts > 1) return {-1, 1};
  const double nk = double(K) * (1.0 / kBK);
  const auto tiles = [&](int edge) { return ((M + edge - 1) / edge) * ((N + edge - 1) / edge); };
  const int64_t of_64 = tiles(64), of_128 = tiles(128);
  GemmFp8Plan plan{-1, 1};
  double best = 0;
  const auto consider = [&](int v, int p, double us) {
    if ((plan.variant < 0 || us < best) && takes(v, p)) best = us, plan = {v, p};
  };
  consider(4, 1, estimate_us(4, M, of_64, nk));
  consider(1, 1, estimate_us(1, M, of_128, nk));
  consider(5, 1, estimate_us(5, M, of_128, nk));
  consider(2, 1, estimate_us(2, M, tiles(256), nk));
  if (M <= 16) {
    consider(3, 1, estimate_us(3, M, (N + 15) / 16, nk));
    consider(6, 1, estimate_us(6, M, (N + 31) / 32, nk));
  }
  if (parts == 0 && of_128 > 0) {
    const double join = double((M + 31) / 32 * 32) * double(N) * (8 / 4.6e6);  // a part's sums, written and read
    for (int p = 2; p <= 16 && p <= quads && of_128 * p <= 512; ++p) {
      const double part = double((int(quads) + p - 1) / p * 4), more = 2 + p * join;
      if (of_64 * p <= 512) consider(4, p, estimate_us(4, M, of_64 * p, part) + more);
      consider(1, p, estimate_us(1, M, of_128 * p, part) + more);
    }
  }
  return plan;
}

bool gemm_fp8_ok(int64_t M, int64_t N, int64_t K) {
  return M < kMaxRows && N < kMaxRows && fp8_row_bytes(K) <= kMaxLd &&
         (grid_ok(4, 1, M, N, K) || grid_ok(1, 1, M, N, K) || (K >= kBK + 16 && grid_ok(2, 1, M, N, K)) ||
          (M <= 16 && grid_ok(6, 1, M, N, K)));
}

int64_t gemm_fp8_temp_bytes(int64_t M, int64_t N, const GemmFp8Plan& plan) {
  const int64_t edge = plan.variant == 4 ? 64 : 128;
  return plan.variant < 0 || plan.parts <= 1 ? 0 : plan.parts * ((M + edge - 1) / edge) * ((N + edge - 1) / edge) * edge * edge * 4;
}

namespace {

template <int a, int b, int kR, int kWide = -1>
void launch_rows(const GemmFp8Args& g, Operand oa, Operand ob, hipStream_t stream) {
  hipLaunchKernelGGL((gemm_fp8_rows_kernel<a, b, kR, kWide>), dim3(uint32_t((g.N + 16 * kR - 1) / (16 * kR))),
                     dim3(rows_waves(g.K) * 64), 0, stream, oa, ob, static_cast<uint16_t*>(g.c), g.ldc, int(g.K),
                     g.ctype == kF16);
}

}  // namespace

hipError_t launch_gemm_fp8(const GemmFp8Args& g, hipStream_t stream) {
  if (g.M < 0 || g.N < 0 || g.K < 0 || !side_ok(g.a, g.M, g.K) || !side_ok(g.b, g.N, g.K)) return hipErrorInvalidValue;
  if (g.M == 0 || g.N == 0) return hipSuccess;
  const GemmFp8Plan plan = plan_gemm_fp8(g.M, g.N, g.K, g.variant, g.parts);
  const int variant = plan.variant, parts = plan.parts;
  if (variant < 0 || (parts > 1 && !g.temp)) return hipErrorInvalidValue;
  const int64_t edge = variant == 2 ? 256 : variant == 4 ? 64 : 128;
  const int64_t tiles = ((g.M + edge - 1) / edge) * ((g.N + edge - 1) / edge);
  by_types(g.a.type, g.b.type, g.ctype, [&](auto ta, auto tb, auto tc) {
    constexpr int a = decltype(ta)::value, b = decltype(tb)::value;
    const Operand oa = operand(g.a, g.M), ob = operand(g.b, g.N);
    uint16_t* c = static_cast<uint16_t*>(g.c);
    if (variant == 3 || variant == 6) {
      if (variant == 3) launch_rows<a, b, 1>(g, oa, ob, stream);
      else launch_rows<a, b, 2>(g, oa, ob, stream);
    } else if (variant == 2) {
      hipLaunchKernelGGL((gemm_fp8_256_kernel<a, b, decltype(tc)>), dim3(uint32_t(tiles)), dim3(512), 0, stream, oa, ob,
                         c, g.ldc, int(g.K));
    } else if (parts > 1) {
      float* sums = static_cast<float*>(g.temp);
      auto run = [&](auto edge_tag) {
        constexpr int e = decltype(edge_tag)::value;
        hipLaunchKernelGGL((gemm_fp8_tile_kernel<a, b, float, e, e, 4>), dim3(uint32_t(tiles), uint32_t(parts)), dim3(256),
                           0, stream, oa, ob, nullptr, 0, int(g.K), sums);
        hipLaunchKernelGGL((join_parts_kernel<decltype(tc), e, e>), dim3(uint32_t(tiles * (e * e / 1024))), dim3(256), 0,
                           stream, reinterpret_cast<const f32x4*>(sums), c, g.ldc, int(g.M), int(g.N), parts);
      };
      if (variant == 1) run(std::integral_constant<int, 128>{});
      else run(std::integral_constant<int, 64>{});
    } else {
      auto k = variant == 1   ? gemm_fp8_tile_kernel<a, b, decltype(tc), 128, 128, 4>
               : variant == 5 ? gemm_fp8_tile_kernel<a, b, decltype(tc), 128, 128, 2>
                              : gemm_fp8_tile_kernel<a, b, decltype(tc), 64, 64, 4>;
      hipLaunchKernelGGL(k, dim3(uint32_t(tiles)), dim3(256), 0, stream, oa, ob, c, g.ldc, int(g.K),
                         static_cast<float*>(nullptr));
    }
  });
  return hipGetLastError();
}

// Every block quantises the rows of x that it needs, which takes the place of a launch (1, 4, 8 and 16 tokens, weights
// from memory, us, this way: 512 x 512 3.0 3.1 3.1 3.1, by two launches 5.1 5.2 5.4 5.5; 4096 x 2048 4.8 5.0 5.1 5.3 and
// 7.1 7.2 7.3 7.4) until every block's repetition costs as much.  That is near 2^24 weights (4096 x 4096 7.7 7.9 8.1 9.2
// and 8.3 8.5 8.6 9.0), up to 8 tokens near 2^25 (16384 x 2048 10.1 10.7 11.4 and 11.1 11.4 11.7; 8192 x 4096 11.5 11.9
// 12.6 and 11.9 12.2 12.4; from the caches 8 tokens 11.2 and 10.3), and beyond it is more (8 x 8192 x 8192 23.2 and 17.3);
// likewise up to 2^16 values of x (16 x 1024 x 8192 13.2 and 11.1).  The limits cost up to 5 % from memory and 10 % from
// the caches where they are reached.  The vector loads of x want its rows at multiples of 16 bytes and no row to end
// inside 16 values.
bool gemm_fp8_takes_wide(const void* x, int64_t ldx, int64_t M, int64_t N, int64_t K) {
  return M >= 1 && M <= 16 && K >= 1 && K % 16 == 0 && K <= 8192 && M * K <= 65536 &&
         N * K <= (int64_t(1) << (M <= 8 ? 25 : 24)) &&
         reinterpret_cast<uintptr_t>(x) % 16 == 0 && (M == 1 || (ldx % 8 == 0 && ldx <= (int64_t(1) << 21)));
}

hipError_t launch_gemm_fp8_wide(const void* x, int type, int64_t ldx, Fp8In w, int64_t M, int64_t N, int64_t K,
                                void* y, hipStream_t stream) {
  if (!gemm_fp8_takes_wide(x, ldx, M, N, K) || !side_ok(w, N, K) || !grid_ok(3, 1, M, N, K))
    return hipErrorInvalidValue;
  if (N == 0) return hipSuccess;
  GemmFp8Args g{};
  g.c = y;
  g.ldc = N;
  g.M = M;
  g.N = N;
  g.K = K;
  g.ctype = type;
  const Operand oa{static_cast<const uint8_t*>(x), nullptr, 2 * (M == 1 ? K : ldx), 0, int(M), 0};
  const Operand ob = operand(w, N);
  auto by_b = [&](auto tb) {
    constexpr int b = decltype(tb)::value;
    if (type == kBF16) launch_rows<kE4M3, b, 1, kBF16>(g, oa, ob, stream);
    else launch_rows<kE4M3, b, 1, kF16>(g, oa, ob, stream);
  };
  if (w.type == kE4M3) by_b(std::integral_constant<int, kE4M3>{});
  else by_b(std::integral_constant<int, kE5M2>{});
  return hipGetLastError();
}

}  // namespace gpuexp
