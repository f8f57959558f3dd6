// A linear layer in 8 bits: what its passes launch, and where in two workspaces they keep it.
//   forward    x -> Q(x) (kept if the weight takes a gradient), w -> Q(w) and its transpose (kept if x
//              takes one), y = Q(x) Q(w)^T
//   backward   dy -> Q(dy) and Q(dy^T) in one pass over dy, dx = Q(dy) Q(w), dw = Q(dy^T) T(Q(x))^T
//              with T the kept x transposed and requantised along the tokens; of these what is asked for
// Host code only; one call from Python per pass, since a small step is bound by the host.
#include <algorithm>

#include "fp8_launch.h"

namespace gpuexp {

namespace {

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// a tensor in 8 bits inside a workspace: values, then scales
struct Piece {
  int64_t rows, cols, at;
  int block_rows;
  int64_t ld() const { return fp8_row_bytes(cols); }
  int64_t lds() const { return up(up(cols, kFp8Block) / kFp8Block, 4); }
  int64_t scales_at() const { return at + up(rows * ld(), 256); }
  int64_t end() const { return scales_at() + up(up(rows, block_rows) / block_rows * lds(), 256); }
  Fp8Out out(uint8_t* base) const { return {base + at, base + scales_at(), ld(), lds()}; }
  Fp8In in(const uint8_t* base) const { return {base + at, base + scales_at(), ld(), lds(), block_rows, kE4M3}; }
};

// a product, and where in a workspace it keeps the sums of the parts of K
struct Product {
  int64_t M, N, K;
  GemmFp8Plan plan;
  Product(int64_t M, int64_t N, int64_t K) : M(M), N(N), K(K), plan(plan_gemm_fp8(M, N, K, 0, 0)) {}
  int64_t bytes() const { return up(gemm_fp8_temp_bytes(M, N, plan), 256); }
  hipError_t run(Fp8In a, Fp8In b, void* c, int ctype, void* temp, hipStream_t stream) const {
    return launch_gemm_fp8({a, b, c, N, M, N, K, ctype, plan.variant, plan.parts, temp}, stream);
  }
};

void take(Piece& p, int64_t& at, int64_t rows, int64_t cols, int block_rows) {
  p = {rows, cols, at, block_rows};
  at = p.end();
}

// Bytes are without the products' sums, which follow in a pass's workspace.
struct Forward {
  Piece xq, wq, wt;  // x, w; w transposed
  int64_t kept = 0, temp = 0;
  Forward(int64_t M, int64_t N, int64_t K, bool keep_dx, bool keep_dw) {
    take(xq, keep_dw ? kept : temp, M, K, 1);
    take(wq, temp, N, K, kFp8Block);
    if (keep_dx) take(wt, kept, K, N, kFp8Block);
  }
};
struct Backward {
  Piece gq, gt, xt;  // dy, dy transposed, x transposed
  int64_t temp = 0;
  Backward(int64_t M, int64_t N, int64_t K, bool want_dx, bool want_dw) {
    if (want_dx) take(gq, temp, M, N, 1);
    if (want_dw) {
      take(gt, temp, N, M, 1);
      take(xt, temp, K, M, 1);
    }
  }
};

#define GPUEXP_RETURN_IF(call)                   \
  if (hipError_t e_ = (call); e_ != hipSuccess) \
  return e_

}  // namespace

bool linear_fp8_ok(int64_t M, int64_t N, int64_t K, bool keep_dx, bool keep_dw) {
  return fp8_blocks_ok(M, K) && fp8_blocks_ok(N, K) && gemm_fp8_ok(M, N, K) &&
         (!(keep_dx || keep_dw) || fp8_blocks_ok(M, N)) && (!keep_dx || gemm_fp8_ok(M, K, N)) &&
         (!keep_dw || gemm_fp8_ok(N, K, M));
}

int64_t linear_fp8_kept_bytes(int64_t M, int64_t N, int64_t K, bool keep_dx, bool keep_dw) {
  return Forward(M, N, K, keep_dx, keep_dw).kept;
}

int64_t linear_fp8_forward_bytes(int64_t M, int64_t N, int64_t K, bool keep_dx, bool keep_dw) {
  return Forward(M, N, K, keep_dx, keep_dw).temp + Product(M, N, K).bytes();
}

// the two products take turns at the same place
int64_t linear_fp8_backward_bytes(int64_t M, int64_t N, int64_t K, bool want_dx, bool want_dw) {
  return Backward(M, N, K, want_dx, want_dw).temp +
         std::max(want_dx ? Product(M, K, N).bytes() : 0, want_dw ? Product(N, K, M).bytes() : 0);
}

hipError_t launch_linear_fp8_forward(const LinearFp8Args& a, void* y, hipStream_t stream) {
  const Forward p(a.M, a.N, a.K, a.keep_dx, a.keep_dw);
  uint8_t* x_at = a.keep_dw ? a.kept : a.temp;
  GPUEXP_RETURN_IF(launch_quantize_fp8(a.x, a.type, a.ldx, a.M, a.K, kE4M3, 1, p.xq.out(x_at), {}, stream));
  GPUEXP_RETURN_IF(launch_quantize_fp8(a.w, a.wtype, a.ldw, a.N, a.K, kE4M3, kFp8Block, p.wq.out(a.temp),
                                       a.keep_dx ? p.wt.out(a.kept) : Fp8Out{}, stream));
  return Product(a.M, a.N, a.K).run(p.xq.in(x_at), p.wq.in(a.temp), y, a.type, a.temp + p.temp, stream);
}

hipError_t launch_linear_fp8_backward(const LinearFp8Args& a, const void* dy, int64_t lddy, void* dx, void* dw,
                                      hipStream_t stream) {
  if ((a.want_dx && !a.keep_dx) || (a.want_dw && !a.keep_dw)) return hipErrorInvalidValue;
  if (!a.want_dx && !a.want_dw) return hipSuccess;
  const Forward f(a.M, a.N, a.K, a.keep_dx, a.keep_dw);
  const Backward p(a.M, a.N, a.K, a.want_dx, a.want_dw);
  uint8_t* sums = a.temp + p.temp;
  GPUEXP_RETURN_IF(launch_quantize_fp8(dy, a.type, lddy, a.M, a.N, kE4M3, 1,
                                       a.want_dx ? p.gq.out(a.temp) : Fp8Out{},
                                       a.want_dw ? p.gt.out(a.temp) : Fp8Out{}, stream));
  if (a.want_dx)
    GPUEXP_RETURN_IF(Product(a.M, a.K, a.N).run(p.gq.in(a.temp), f.wt.in(a.kept), dx, a.type, sums, stream));
  if (a.want_dw) {
    GPUEXP_RETURN_IF(launch_transpose_fp8(f.xq.in(a.kept), a.M, a.K, p.xt.out(a.temp), stream));
    GPUEXP_RETURN_IF(Product(a.N, a.K, a.M).run(p.gt.in(a.temp), p.xt.in(a.temp), dw, a.wtype, sums, stream));
  }
  return hipSuccess;
}

bool serve_fp8_ok(int64_t M, int64_t N, int64_t K, bool want_dx) {
  return fp8_blocks_ok(M, K) && gemm_fp8_ok(M, N, K) &&
         (!want_dx || (fp8_blocks_ok(M, N) && fp8_blocks_ok(N, K) && gemm_fp8_ok(M, K, N)));
}

int64_t serve_fp8_bytes(const void* x, int64_t ldx, int64_t M, int64_t N, int64_t K) {
  return gemm_fp8_takes_wide(x, ldx, M, N, K) ? 0 : Piece{M, K, 0, 1}.end() + Product(M, N, K).bytes();
}

hipError_t launch_serve_fp8(const void* x, int type, int64_t ldx, Fp8In w, int64_t M, int64_t N, int64_t K, void* y,
                            uint8_t* temp, hipStream_t stream) {
  if (gemm_fp8_takes_wide(x, ldx, M, N, K)) return launch_gemm_fp8_wide(x, type, ldx, w, M, N, K, y, stream);
  const Piece xq{M, K, 0, 1};
  GPUEXP_RETURN_IF(launch_quantize_fp8(x, type, ldx, M, K, kE4M3, 1, xq.out(temp), {}, stream));
  return Product(M, N, K).run(xq.in(temp), w, y, type, temp + xq.end(), stream);
}

}  // namespace gpuexp
