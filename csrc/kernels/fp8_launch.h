// Launchers of the 8-bit operators (fp8_quant.hip, gemm_fp8.hip) and their host-side rules.
// A tensor in 8 bits is [rows][cols] bytes with a row stride `ld` (bytes); its scales are E8M0
// bytes (2^(byte - 127)) [rows / block_rows][ceil(cols / 128)] with a row stride `lds`.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace gpuexp {

enum Fp8Type { kE4M3 = 0, kE5M2 = 1 };               // also the matrix instruction's type codes
enum WideType { kBF16 = 0, kF16 = 1, kF32 = 2 };     // types of 16 and 32 bits
constexpr int kFp8Block = 128;

// Bytes between the rows of a tensor of 8-bit values that this code lays out.  The kernels want multiples of
// 16; where an eighth more memory is enough, rows start at lines of 128 bytes: a block of 128 values is then
// one line, and no line is written by two blocks that share no cache (4112 x 4112 x 4112 112 -> 93 us,
// 64 x 4000 x 5001 14.0 -> 12.2, the transpose of 4112 x 8208 27 -> 20).
inline int64_t fp8_row_bytes(int64_t cols) {
  const int64_t lines = (cols + 127) / 128 * 128;
  return lines - cols <= cols / 8 ? lines : (cols + 15) / 16 * 16;
}

struct Fp8Out {  // a tensor in 8 bits to write; q == nullptr: not wanted
  uint8_t* q;
  uint8_t* scale;
  int64_t ld;
  int64_t lds;
};

struct Fp8In {
  const uint8_t* q;
  const uint8_t* scale;
  int64_t ld;
  int64_t lds;
  int block_rows;  // 1 or 128 rows share a scale
  int type;        // Fp8Type
};

// what the kernels index: of a tensor to quantise, give back or transpose its blocks of 128 along rows
inline bool fp8_blocks_ok(int64_t rows, int64_t cols) {  // (16 lanes for each, and a launch has less than 2^32 threads)
  return rows >= 0 && cols >= 0 && rows < (int64_t(1) << 28) && cols < (int64_t(1) << 31) - 128 &&
         rows * ((cols + 127) / 128) < (int64_t(1) << 28) - 16;
}

// out = x[rows][cols] in 8 bits; outT = its transpose [cols][rows].  block_rows 1: blocks of
// 1 x 128 along each output's own rows; 128: blocks of 128 x 128, the transpose the same values.
hipError_t launch_quantize_fp8(const void* x, int xtype, int64_t ldx, int64_t rows, int64_t cols, int type,
                               int block_rows, Fp8Out out, Fp8Out outT, hipStream_t stream);
hipError_t launch_dequantize_fp8(Fp8In in, int64_t rows, int64_t cols, void* x, int xtype, int64_t ldx,
                                 hipStream_t stream);
// outT = in's transpose; block_rows 1: requantised in blocks of 1 x 128 along in's rows
hipError_t launch_transpose_fp8(Fp8In in, int64_t rows, int64_t cols, Fp8Out outT, hipStream_t stream);

struct GemmFp8Args {
  Fp8In a, b;  // [M][K], [N][K]
  void* c;     // [M][ldc] of ctype (kBF16 or kF16)
  int64_t ldc;
  int64_t M, N, K;
  int ctype;
  int variant;  // 0: by the sizes; 1: 128 x 128 tile, 2: 256 x 256 (K >= 144), 3: few rows (M <= 16), 4: 64 x 64,
                // 5: 128 x 128 with two K tiles in LDS, so two blocks per CU, 6: few rows, 32 of B per wave
  int parts;    // of K, multiplied by different blocks: 0: by the sizes; more than one: variants 1 and 4, at most 16
  void* temp;   // gemm_fp8_temp_bytes, read and written during the call
};
// what a call runs (0 resolved); variant -1 if the sizes do not fit it
struct GemmFp8Plan {
  int variant, parts;
};
GemmFp8Plan plan_gemm_fp8(int64_t M, int64_t N, int64_t K, int64_t variant, int64_t parts);
bool gemm_fp8_ok(int64_t M, int64_t N, int64_t K);  // whether a product of these sizes has a kernel
int64_t gemm_fp8_temp_bytes(int64_t M, int64_t N, const GemmFp8Plan& plan);
hipError_t launch_gemm_fp8(const GemmFp8Args& g, hipStream_t stream);
// the same for x[M][ldx] in bf16 or f16, quantised on its way (blocks of 1 x 128, e4m3), where it takes x
bool gemm_fp8_takes_wide(const void* x, int64_t ldx, int64_t M, int64_t N, int64_t K);
hipError_t launch_gemm_fp8_wide(const void* x, int type, int64_t ldx, Fp8In w, int64_t M, int64_t N, int64_t K,
                                void* y, hipStream_t stream);

// y[M][N] = x[M][K] . w[N][K]^T in 8 bits and its backward pass, several launches behind one call.
// Two workspaces in device memory: `kept` holds between the passes what the backward pass reads (x in
// 8 bits for dw, the transposed weight in 8 bits for dx), `temp` only during a pass.
struct LinearFp8Args {
  int64_t M, N, K;
  bool keep_dx, keep_dw;  // what `kept` is laid out for
  bool want_dx, want_dw;  // what a backward pass computes, of these
  const void* x;  // [M][ldx], type
  int64_t ldx;
  const void* w;  // [N][ldw], wtype; not read by the backward pass
  int64_t ldw;
  int type, wtype;  // of x, y and their gradients, and of w and dw: kBF16 or kF16
  uint8_t* kept;
  uint8_t* temp;
};
// whether every launch of the passes takes these sizes, so that none is refused behind others
bool linear_fp8_ok(int64_t M, int64_t N, int64_t K, bool keep_dx, bool keep_dw);
int64_t linear_fp8_kept_bytes(int64_t M, int64_t N, int64_t K, bool keep_dx, bool keep_dw);
int64_t linear_fp8_forward_bytes(int64_t M, int64_t N, int64_t K, bool keep_dx, bool keep_dw);   // temp
int64_t linear_fp8_backward_bytes(int64_t M, int64_t N, int64_t K, bool want_dx, bool want_dw);  // temp
hipError_t launch_linear_fp8_forward(const LinearFp8Args& a, void* y, hipStream_t stream);
hipError_t launch_linear_fp8_backward(const LinearFp8Args& a, const void* dy, int64_t lddy, void* dx, void* dw,
                                      hipStream_t stream);
// the same with a weight that is in 8 bits already; temp: x in 8 bits, where the product
// does not make it, and the product's own
bool serve_fp8_ok(int64_t M, int64_t N, int64_t K, bool want_dx);
int64_t serve_fp8_bytes(const void* x, int64_t ldx, int64_t M, int64_t N, int64_t K);
hipError_t launch_serve_fp8(const void* x, int type, int64_t ldx, Fp8In w, int64_t M, int64_t N, int64_t K, void* y,
                            uint8_t* temp, hipStream_t stream);

}  // namespace gpuexp
