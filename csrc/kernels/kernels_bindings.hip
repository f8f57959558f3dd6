// Python bindings for the HIP workload kernels (raw device pointers + stream handles, so
// they work with torch tensors via .data_ptr() and without torch at all via gemm_burn).
#include <hip/hip_runtime.h>
#include <pybind11/pybind11.h>

#include <chrono>
#include <stdexcept>
#include <string>

#include "fp8_launch.h"

namespace py = pybind11;

namespace gpuexp {
bool gemm_shape_ok(int M, int N, int K);
bool gemm256_shape_ok(int M, int N, int K);
int resolve_gemm_variant(int M, int N, int K, int variant);
hipError_t launch_gemm_bf16_tn(const void* A, const void* B, void* C, int M, int N, int K, hipStream_t stream,
                               int variant);
hipError_t launch_fill_bf16(void* p, size_t n, uint32_t seed, hipStream_t stream);
hipError_t launch_stream_copy(const void* src, void* dst, size_t bytes, int blocks, hipStream_t stream);
hipError_t launch_lds_probe(float* out, int blocks, int iters, int stride, hipStream_t stream);
hipError_t launch_occupancy_hog(int kind, float* out, int blocks, double seconds, hipStream_t stream);
hipError_t launch_mfma_duty(float* out, uint64_t* counts, int blocks, double duty, double period_s, double seconds,
                            uint32_t xcc_mask, hipStream_t stream);
}  // namespace gpuexp

namespace {

void check(hipError_t e, const char* what) {
  if (e != hipSuccess) throw std::runtime_error(std::string(what) + ": " + hipGetErrorString(e));
}

// 8-bit tensors arrive as raw addresses; the Python wrappers (ops/fp8.py) check the tensors, these
// check what the kernels' vector accesses and index arithmetic assume.
gpuexp::Fp8In fp8_in(uintptr_t q, uintptr_t scale, int64_t ld, int64_t lds, int block_rows, int type, int64_t rows,
                     int64_t cols) {
  if (rows < 0 || cols < 0 || (block_rows != 1 && block_rows != 128) || type < 0 || type > 1)
    throw std::invalid_argument("8-bit operand: sizes >= 0, block_rows 1 or 128, type 0 (e4m3) or 1 (e5m2)");
  if (rows && cols && (!q || !scale)) throw std::invalid_argument("8-bit operand: null pointer");
  if (q % 16 || scale % 4 || ld % 16 || lds % 4 || ld < cols || lds < (cols + 127) / 128)
    throw std::invalid_argument("8-bit operand: rows must start at multiples of 16 bytes (scales: 4) and not overlap");
  return {reinterpret_cast<const uint8_t*>(q), reinterpret_cast<const uint8_t*>(scale), ld, lds, block_rows, type};
}

gpuexp::Fp8Out fp8_out(uintptr_t q, uintptr_t scale, int64_t ld, int64_t lds, int64_t cols) {
  if (!q) return {};
  if (!scale || q % 16 || ld % 16 || ld < cols || lds < (cols + 127) / 128)
    throw std::invalid_argument("8-bit result: rows must start at multiples of 16 bytes and not overlap");
  return {reinterpret_cast<uint8_t*>(q), reinterpret_cast<uint8_t*>(scale), ld, lds};
}

gpuexp::LinearFp8Args linear_args(int64_t M, int64_t N, int64_t K, bool want_dx, bool want_dw, int type, int wtype,
                                  uintptr_t kept, uintptr_t temp) {
  if (M < 0 || N < 0 || K < 0 || type < 0 || type > 1 || wtype < 0 || wtype > 1)
    throw std::invalid_argument("linear_fp8: sizes >= 0, types 0 (bf16) or 1 (f16)");
  if (kept % 256 || temp % 256) throw std::invalid_argument("linear_fp8: workspaces start at multiples of 256 bytes");
  gpuexp::LinearFp8Args a{};
  a.M = M;
  a.N = N;
  a.K = K;
  a.want_dx = want_dx;
  a.want_dw = want_dw;
  a.type = type;
  a.wtype = wtype;
  a.kept = reinterpret_cast<uint8_t*>(kept);
  a.temp = reinterpret_cast<uint8_t*>(temp);
  return a;
}

}  // namespace

// Separate module from the telemetry core: it links a HIP runtime, so it is imported
// only AFTER torch (when torch is used) to bind to torch's runtime — see ops/gemm.py.
PYBIND11_MODULE(_gpuexp_kernels, m) {
  m.doc() = "HIP/CDNA4 workload kernels (bf16 MFMA GEMM) for synthetic GPU pods";
  m.def("hip_device_count", []() {
    int n = 0;
    if (hipGetDeviceCount(&n) != hipSuccess) return 0;
    return n;
  });
  m.def("gemm_shape_ok", &gpuexp::gemm_shape_ok);
  m.def("gemm256_shape_ok", &gpuexp::gemm256_shape_ok);
  m.def("gemm_variant", &gpuexp::resolve_gemm_variant, py::arg("M"), py::arg("N"), py::arg("K"),
        py::arg("variant") = 0,
        "The GEMM kernel variant a gemm_bf16 call with these arguments runs (0 = auto resolved), -1 if the shape "
        "does not fit it.  Host-only: no GPU needed.");
  m.def("gemm_bf16", [](uintptr_t a, uintptr_t b, uintptr_t c, int M, int N, int K, uintptr_t stream, int variant) {
    if (!gpuexp::gemm_shape_ok(M, N, K))
      throw std::invalid_argument("gemm_bf16 needs M%128==0, N%128==0, K%64==0");
    if (variant >= 2 && !gpuexp::gemm256_shape_ok(M, N, K))
      throw std::invalid_argument("the 256x256 kernel needs M%256==0, N%256==0, K%64==0, K>=128");
    if (variant < 0 || variant > 9)
      throw std::invalid_argument("variant is 0 (auto), 1 (128x128), 2-9 (256x256 tile orders / priority / read schedules / ping-pong / 4 waves)");
    if (!a || !b || !c) throw std::invalid_argument("null pointer");
    check(gpuexp::launch_gemm_bf16_tn(reinterpret_cast<const void*>(a), reinterpret_cast<const void*>(b),
                                      reinterpret_cast<void*>(c), M, N, K, reinterpret_cast<hipStream_t>(stream),
                                      variant),
          "gemm_bf16 launch");
  }, py::arg("a"), py::arg("b"), py::arg("c"), py::arg("M"), py::arg("N"), py::arg("K"), py::arg("stream") = 0,
     py::arg("variant") = 0,
     "C[M,N] = A[M,K] @ B[N,K]^T; bf16 row-major, fp32 accumulate (MFMA 16x16x32). variant: 0 auto, "
     "1 = 128x128 tile, 2 = 256x256 tile");
  m.def("fill_bf16", [](uintptr_t p, size_t n, uint32_t seed, uintptr_t stream) {
    check(gpuexp::launch_fill_bf16(reinterpret_cast<void*>(p), n, seed, reinterpret_cast<hipStream_t>(stream)),
          "fill_bf16 launch");
  }, py::arg("ptr"), py::arg("n"), py::arg("seed") = 1, py::arg("stream") = 0);
  // PMC calibration workloads (csrc/kernels/probe_kernels.hip)
  m.def("stream_copy", [](uintptr_t src, uintptr_t dst, size_t nbytes, int blocks, uintptr_t stream) {
    if (!src || !dst || nbytes % 16 || blocks < 1 || blocks > (1 << 20))
      throw std::invalid_argument("stream_copy needs non-null pointers, nbytes % 16 == 0, 1 <= blocks <= 2^20");
    check(gpuexp::launch_stream_copy(reinterpret_cast<const void*>(src), reinterpret_cast<void*>(dst), nbytes, blocks,
                                     reinterpret_cast<hipStream_t>(stream)),
          "stream_copy launch");
  }, py::call_guard<py::gil_scoped_release>(), py::arg("src"), py::arg("dst"), py::arg("nbytes"),
     py::arg("blocks") = 4096, py::arg("stream") = 0,
     "dst[:nbytes] = src[:nbytes] (each byte read once from and written once to HBM)");
  m.def("lds_probe", [](uintptr_t out, int blocks, int iters, int stride, uintptr_t stream) {
    // `out` must hold >= blocks floats (checked by the Python wrapper)
    if (!out || blocks < 1 || blocks > (1 << 20) || iters < 1 || (stride != 1 && stride != 32))
      throw std::invalid_argument("lds_probe needs out, 1 <= blocks <= 2^20, iters >= 1, stride 1 or 32");
    check(gpuexp::launch_lds_probe(reinterpret_cast<float*>(out), blocks, iters, stride,
                                   reinterpret_cast<hipStream_t>(stream)),
          "lds_probe launch");
  }, py::call_guard<py::gil_scoped_release>(), py::arg("out"), py::arg("blocks"), py::arg("iters"),
     py::arg("stride"), py::arg("stream") = 0,
     "256-thread blocks (4 waves) of ds_read_b32 from LDS: stride 1 conflict-free, stride 32 32-way conflicts");
  m.def("mfma_duty", [](uintptr_t out, uintptr_t counts, int blocks, double duty, double period_s, double seconds,
                        uintptr_t stream, uint32_t xcc_mask) {
    // `out` >= blocks floats, `counts` >= blocks * 4 uint64 (checked by the Python wrapper)
    check(gpuexp::launch_mfma_duty(reinterpret_cast<float*>(out), reinterpret_cast<uint64_t*>(counts), blocks, duty,
                                   period_s, seconds, xcc_mask, reinterpret_cast<hipStream_t>(stream)),
          "mfma_duty launch");
  }, py::call_guard<py::gil_scoped_release>(), py::arg("out"), py::arg("counts"), py::arg("blocks"), py::arg("duty"),
     py::arg("period_s") = 0.002, py::arg("seconds") = 1.0, py::arg("stream") = 0, py::arg("xcc_mask") = 0,
     "256-thread blocks alternating back-to-back v_mfma_f32_32x32x16_bf16 (duty x period) with s_sleep, for "
     "`seconds` (s_memrealtime-timed); 2 blocks per CU = 2 waves per SIMD keep the matrix cores busy `duty` of "
     "the wall time.  xcc_mask != 0: only blocks on those XCCs (HW_REG_XCC_ID) run, the rest exit at once");
  m.def("occupancy_hog", [](int kind, uintptr_t out, int blocks, double seconds, uintptr_t stream) {
    // `out` >= blocks floats (checked by the Python wrapper)
    check(gpuexp::launch_occupancy_hog(kind, reinterpret_cast<float*>(out), blocks, seconds,
                                       reinterpret_cast<hipStream_t>(stream)),
          "occupancy_hog launch");
  }, py::call_guard<py::gil_scoped_release>(), py::arg("kind"), py::arg("out"), py::arg("blocks"),
     py::arg("seconds"), py::arg("stream") = 0,
     "Blocks that hold a resource for `seconds` each: kind 0 = 1 wave + 64 KiB LDS per block (LDS-limited), "
     "kind 1 = 8 waves per block, no LDS (wave-slot-limited)");
  // 8-bit floating point with block scales (csrc/kernels/fp8_quant.hip, gemm_fp8.hip)
  m.def("quantize_fp8", [](uintptr_t x, int xtype, int64_t ldx, int64_t rows, int64_t cols, int type, int block_rows,
                           uintptr_t q, uintptr_t scale, int64_t ld, int64_t lds, uintptr_t qt, uintptr_t scale_t,
                           int64_t ldt, int64_t ldst, uintptr_t stream) {
    if (!x || rows < 1 || cols < 1 || ldx < cols || xtype < 0 || xtype > 2 || type < 0 || type > 1 ||
        (block_rows != 1 && block_rows != 128) || (!q && !qt))
      throw std::invalid_argument("quantize_fp8: sizes >= 1, ldx >= cols, types 0-2 / 0-1, block_rows 1 or 128, a result");
    check(gpuexp::launch_quantize_fp8(reinterpret_cast<const void*>(x), xtype, ldx, rows, cols, type, block_rows,
                                      fp8_out(q, scale, ld, lds, cols), fp8_out(qt, scale_t, ldt, ldst, rows),
                                      reinterpret_cast<hipStream_t>(stream)),
          "quantize_fp8 launch");
  }, "x[rows][cols] (0 bf16, 1 f16, 2 f32) in 8 bits (0 e4m3, 1 e5m2) with block scales, and / or its transpose");
  m.def("dequantize_fp8", [](uintptr_t q, uintptr_t scale, int64_t ld, int64_t lds, int block_rows, int type,
                             int64_t rows, int64_t cols, uintptr_t x, int xtype, int64_t ldx, uintptr_t stream) {
    const gpuexp::Fp8In in = fp8_in(q, scale, ld, lds, block_rows, type, rows, cols);
    if (!x || xtype < 0 || xtype > 2 || ldx < cols) throw std::invalid_argument("dequantize_fp8: bad result");
    check(gpuexp::launch_dequantize_fp8(in, rows, cols, reinterpret_cast<void*>(x), xtype, ldx,
                                        reinterpret_cast<hipStream_t>(stream)),
          "dequantize_fp8 launch");
  }, "x[rows][cols] = the values that the 8-bit tensor stands for");
  m.def("transpose_fp8", [](uintptr_t q, uintptr_t scale, int64_t ld, int64_t lds, int block_rows, int type,
                            int64_t rows, int64_t cols, uintptr_t qt, uintptr_t scale_t, int64_t ldt, int64_t ldst,
                            uintptr_t stream) {
    const gpuexp::Fp8In in = fp8_in(q, scale, ld, lds, block_rows, type, rows, cols);
    if (!qt) throw std::invalid_argument("transpose_fp8: null pointer");
    check(gpuexp::launch_transpose_fp8(in, rows, cols, fp8_out(qt, scale_t, ldt, ldst, rows),
                                       reinterpret_cast<hipStream_t>(stream)),
          "transpose_fp8 launch");
  }, "The transpose of an 8-bit tensor; blocks of 1 x 128 are quantised anew along its own rows");
  m.def("gemm_fp8", [](uintptr_t a, uintptr_t sa, int64_t lda, int64_t ldsa, int block_a, int type_a, uintptr_t b,
                       uintptr_t sb, int64_t ldb, int64_t ldsb, int block_b, int type_b, uintptr_t c, int64_t ldc,
                       int64_t M, int64_t N, int64_t K, int ctype, int variant, uintptr_t stream) {
    gpuexp::GemmFp8Args g{};
    if (gpuexp::resolve_gemm_fp8_variant(M, N, K, variant) < 0)
      throw std::invalid_argument("gemm_fp8: variant is 0 (auto), 1 (128x128), 2 (256x256, K >= 144), 3 (few rows, M <= 16), 4 (64x64), 5 (128x128, "
                                  "two blocks per CU) or 6 (few rows, 32 of B per wave)");
    g.a = fp8_in(a, sa, lda, ldsa, block_a, type_a, M, K);
    g.b = fp8_in(b, sb, ldb, ldsb, block_b, type_b, N, K);
    if (!c || ldc < N || c % 2 || (ctype != 0 && ctype != 1))
      throw std::invalid_argument("gemm_fp8: a result with ldc >= N of type 0 (bf16) or 1 (f16)");
    g.c = reinterpret_cast<void*>(c);
    g.ldc = ldc;
    g.M = M;
    g.N = N;
    g.K = K;
    g.ctype = ctype;
    g.variant = variant;
    check(gpuexp::launch_gemm_fp8(g, reinterpret_cast<hipStream_t>(stream)), "gemm_fp8 launch");
  }, "C[M,N] = A[M,K] @ B[N,K]^T; 8-bit operands with block scales, fp32 accumulate (scaled MFMA). The last argument but "
     "the stream, variant: 0 auto, 1 = 128x128 tile, 2 = 256x256 tile, 3 = few rows, 4 = 64x64, 5 = 128x128 with two "
     "blocks per CU, 6 = few rows, 32 of B per wave");
  m.def("gemm_fp8_variant", &gpuexp::resolve_gemm_fp8_variant, py::arg("M"), py::arg("N"), py::arg("K"),
        py::arg("variant") = 0,
        "The kernel variant a gemm_fp8 call with these sizes runs (0 = auto resolved), -1 if they do not fit it. "
        "Host-only: no GPU needed.");
  m.def("linear_fp8_bytes", [](int64_t M, int64_t N, int64_t K, bool want_dx, bool want_dw) {
    if (M < 0 || N < 0 || K < 0) throw std::invalid_argument("linear_fp8: sizes >= 0");
    const gpuexp::LinearFp8Bytes b = gpuexp::linear_fp8_bytes(M, N, K, want_dx, want_dw);
    return py::make_tuple(b.kept, b.forward_temp, b.backward_temp);
  }, "Bytes of the workspaces of a linear layer in 8 bits: (kept between the passes, forward, backward)");
  m.def("linear_fp8_forward", [](int64_t M, int64_t N, int64_t K, bool want_dx, bool want_dw, uintptr_t x, int64_t ldx,
                                 int type, uintptr_t w, int64_t ldw, int wtype, uintptr_t kept, uintptr_t temp,
                                 uintptr_t y, uintptr_t stream) {
    gpuexp::LinearFp8Args a = linear_args(M, N, K, want_dx, want_dw, type, wtype, kept, temp);
    if ((M && K && (!x || ldx < K)) || (N && K && (!w || ldw < K)) || (M && N && !y))
      throw std::invalid_argument("linear_fp8_forward: null pointer, or rows that overlap");
    a.x = reinterpret_cast<const void*>(x);
    a.ldx = ldx;
    a.w = reinterpret_cast<const void*>(w);
    a.ldw = ldw;
    check(gpuexp::launch_linear_fp8_forward(a, reinterpret_cast<void*>(y), reinterpret_cast<hipStream_t>(stream)),
          "linear_fp8 forward launch");
  }, "y[M,N] = x[M,K] @ w[N,K]^T in 8 bits (types 0 bf16, 1 f16); `kept` holds what the backward pass needs");
  m.def("linear_fp8_backward", [](int64_t M, int64_t N, int64_t K, bool want_dx, bool want_dw, uintptr_t dy,
                                  int64_t lddy, int type, int wtype, uintptr_t kept, uintptr_t temp, uintptr_t dx,
                                  uintptr_t dw, uintptr_t stream) {
    const gpuexp::LinearFp8Args a = linear_args(M, N, K, want_dx, want_dw, type, wtype, kept, temp);
    if ((M && N && (!dy || lddy < N)) || (want_dx && M && K && !dx) || (want_dw && N && K && !dw))
      throw std::invalid_argument("linear_fp8_backward: null pointer, or rows that overlap");
    check(gpuexp::launch_linear_fp8_backward(a, reinterpret_cast<const void*>(dy), lddy, reinterpret_cast<void*>(dx),
                                             reinterpret_cast<void*>(dw), reinterpret_cast<hipStream_t>(stream)),
          "linear_fp8 backward launch");
  }, "dx[M,K] and / or dw[N,K] of linear_fp8_forward");
  m.def("serve_fp8_bytes", &gpuexp::serve_fp8_bytes, "Bytes of serve_fp8's workspace");
  m.def("serve_fp8", [](uintptr_t x, int type, int64_t ldx, uintptr_t w, uintptr_t scale, int64_t ld, int64_t lds,
                        int block_rows, int wtype, int64_t M, int64_t N, int64_t K, uintptr_t y, uintptr_t temp,
                        uintptr_t stream) {
    const gpuexp::Fp8In in = fp8_in(w, scale, ld, lds, block_rows, wtype, N, K);
    if (M < 0 || type < 0 || type > 1 || (M && K && (!x || ldx < K)) || (M && N && !y) || temp % 256)
      throw std::invalid_argument("serve_fp8: types 0-1, rows that do not overlap, a workspace at a multiple of 256");
    check(gpuexp::launch_serve_fp8(reinterpret_cast<const void*>(x), type, ldx, in, M, N, K, reinterpret_cast<void*>(y),
                                   reinterpret_cast<uint8_t*>(temp), reinterpret_cast<hipStream_t>(stream)),
          "serve_fp8 launch");
  }, "y[M,N] = x[M,K] @ w[N,K]^T; x bf16 / f16 is quantised on the way, w is in 8 bits");
  m.def("gemm_burn", [](int device, int M, int N, int K, double seconds, int iters_per_sync, int variant) {
    // Torch-free synthetic GEMM pod: keeps one GPU busy for `seconds` and reports the
    // achieved bf16 TFLOP/s (random operands).
    if (!gpuexp::gemm_shape_ok(M, N, K) || (variant >= 2 && !gpuexp::gemm256_shape_ok(M, N, K)))
      throw std::invalid_argument("bad GEMM shape");
    if (seconds <= 0 || seconds > 3600) throw std::invalid_argument("seconds out of range");
    double tflops = 0;
    long iters = 0;
    double elapsed = 0;
    {
      py::gil_scoped_release rel;
      check(hipSetDevice(device), "hipSetDevice");
      void *a = nullptr, *b = nullptr, *c = nullptr;
      check(hipMalloc(&a, size_t(M) * K * 2), "hipMalloc A");
      check(hipMalloc(&b, size_t(N) * K * 2), "hipMalloc B");
      check(hipMalloc(&c, size_t(M) * N * 2), "hipMalloc C");
      hipStream_t s;
      check(hipStreamCreate(&s), "hipStreamCreate");
      (void)gpuexp::launch_fill_bf16(a, size_t(M) * K, 1, s);
      (void)gpuexp::launch_fill_bf16(b, size_t(N) * K, 2, s);
      check(hipStreamSynchronize(s), "fill");
      auto t0 = std::chrono::steady_clock::now();
      int per = iters_per_sync > 0 ? iters_per_sync : 8;
      for (;;) {
        for (int i = 0; i < per; ++i) check(gpuexp::launch_gemm_bf16_tn(a, b, c, M, N, K, s, variant), "gemm");
        check(hipStreamSynchronize(s), "gemm");
        iters += per;
        elapsed = std::chrono::duration<double>(std::chrono::steady_clock::now() - t0).count();
        if (elapsed >= seconds) break;
      }
      tflops = 2.0 * M * N * double(K) * double(iters) / elapsed / 1e12;
      (void)hipStreamDestroy(s);
      (void)hipFree(a);
      (void)hipFree(b);
      (void)hipFree(c);
    }
    py::dict d;
    d["tflops"] = tflops;
    d["iters"] = iters;
    d["seconds"] = elapsed;
    return d;
  }, py::arg("device"), py::arg("M") = 4096, py::arg("N") = 4096, py::arg("K") = 4096, py::arg("seconds") = 1.0,
     py::arg("iters_per_sync") = 8, py::arg("variant") = 0);
}
