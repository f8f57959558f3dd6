// torch bindings of the 8-bit operators: checks of arguments, allocation, autograd.  In C++ because a
// small call is bound by the host: the launches of a training step take 20 us, its Python took 100.
// Tensors come in and go out as torch tensors, work goes to torch's current stream of their device.
// The operators are torch.ops.gpuexp's, and Python calls them through torch's dispatcher: what records a
// program (torch.jit.trace, make_fx) then records the operator, not the empty tensors that it fills.
// The documentation is in ops/fp8.py.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

#include "fp8_launch.h"

namespace {

using at::Tensor;
using gpuexp::Fp8In;
using gpuexp::Fp8Out;
using gpuexp::kFp8Block;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Pair = std::tuple<Tensor, Tensor>;
using Four = std::tuple<Tensor, Tensor, Tensor, Tensor>;

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
int64_t blocks(int64_t n) { return (n + kFp8Block - 1) / kFp8Block; }

// the longest row of a product's operand: a tile of 256 of them has to fit in a buffer's 31 bits
constexpr int64_t kLongest = int64_t(1) << 22;

constexpr const char* kLimits =
    "larger than the kernels index: of a tensor to quantise, give back or transpose fewer than 2^28 rows and 2^28 - 16 blocks "
    "of 128 values along them, of a product's operand fewer than 2^31 - 256 rows at most 4 MiB apart, and fewer than 2^32 "
    "threads in a launch";

void check(hipError_t e, const char* what) {
  TORCH_CHECK_VALUE(e != hipErrorInvalidValue, what, ": ", kLimits);
  TORCH_CHECK(e == hipSuccess, what, ": ", hipGetErrorString(e));
}

// the current device and torch's current stream for the launches of a call
struct On {
  explicit On(const Tensor& t)
      : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
  c10::DeviceGuard guard;
  hipStream_t stream;
};

int fp8_type(at::ScalarType t) {
  return t == at::kFloat8_e4m3fn ? gpuexp::kE4M3 : t == at::kFloat8_e5m2 ? gpuexp::kE5M2 : -1;
}
int wide_type(at::ScalarType t) {
  return t == at::kBFloat16 ? gpuexp::kBF16 : t == at::kHalf ? gpuexp::kF16 : t == at::kFloat ? gpuexp::kF32 : -1;
}

template <typename... T>
void check_gpu(const char* name, const Tensor& first, const T&... rest) {
  TORCH_CHECK_VALUE(first.device().is_cuda() && (... && (rest.device() == first.device())), name,
                    ": tensors must be on the same GPU, got ", first.device(), ((" " + rest.device().str()) + ...));
}
void check_gpu(const char* name, const Tensor& t) {
  TORCH_CHECK_VALUE(t.device().is_cuda(), name, ": tensors must be on the same GPU, got ", t.device());
}

// A 1-byte tensor [rows, cols] whose rows start at multiples of `pad`: the bytes between them.
struct Rows {
  bool columns_ok, ok;
  int64_t ld, off;
  Rows(const Tensor& t, int64_t pad) : columns_ok(true), ok(true), ld(up(t.size(1), pad)), off(0) {
    if (!t.numel()) return;  // (an empty view may have any address)
    columns_ok = t.size(1) == 1 || t.stride(1) == 1;
    if (t.size(0) > 1) ld = t.stride(0);
    off = int64_t(reinterpret_cast<uintptr_t>(t.const_data_ptr()) % pad);
    ok = columns_ok && ld % pad == 0 && ld >= t.size(1) && off == 0;
  }
};
int64_t row_stride(const char* name, const char* of, const Tensor& t, int64_t pad) {
  const Rows r(t, pad);
  TORCH_CHECK_VALUE(r.columns_ok, of, name, " must have its columns next to each other, got strides ", t.strides());
  TORCH_CHECK_VALUE(r.ok, of, name, "'s rows must start at multiples of ", pad, " bytes and not overlap (row stride ", r.ld,
                    ", address % ", pad, " = ", r.off, "); quantize_fp8 makes such tensors, align_fp8 lays out copies");
  return r.ld;
}

// the checks of types and sizes: whether (q, scale) has blocks of 1 x 128
bool check_pair(const char* name, const Tensor& q, const Tensor& scale) {
  TORCH_CHECK_TYPE(fp8_type(q.scalar_type()) >= 0, name, " must be float8_e4m3fn or float8_e5m2, got ", q.scalar_type());
  TORCH_CHECK_TYPE(scale.scalar_type() == at::kFloat8_e8m0fnu, "the scales of ", name, " must be float8_e8m0fnu, got ",
                   scale.scalar_type());
  TORCH_CHECK_VALUE(q.dim() == 2 && scale.dim() == 2, name, " and its scales must be 2-dimensional, got ", q.sizes(),
                    " and ", scale.sizes());
  const int64_t rows = q.size(0), cols = q.size(1), nb = blocks(cols);
  const bool per_row = scale.size(0) == rows;
  TORCH_CHECK_VALUE(scale.size(1) == nb && (per_row || scale.size(0) == blocks(rows)), "the scales of ", name, " ",
                    q.sizes(), " must be [", rows, ", ", nb, "] (blocks of 1 x 128) or [", blocks(rows), ", ", nb,
                    "] (128 x 128), got ", scale.sizes());
  return per_row;
}

Fp8In operand(const char* name, const Tensor& q, const Tensor& scale) {
  const bool per_row = check_pair(name, q, scale);
  Fp8In in{nullptr, nullptr, row_stride(name, "", q, 16), row_stride(name, "the scales of ", scale, 4),
           per_row ? 1 : kFp8Block, fp8_type(q.scalar_type())};
  if (q.numel()) {
    in.q = static_cast<const uint8_t*>(q.const_data_ptr());
    in.scale = static_cast<const uint8_t*>(scale.const_data_ptr());
  }
  return in;
}

// columns next to each other, rows that do not overlap
bool row_major(const Tensor& x) {
  const int64_t rows = x.size(0), cols = x.size(1);
  return !x.numel() || ((cols == 1 || x.stride(1) == 1) && (rows == 1 || x.stride(0) >= cols));
}
// whether the memory from the first to the last value of each meets
bool overlap(const Tensor& x, const Tensor& y) {
  if (!x.numel() || !y.numel()) return false;
  const auto begin = [](const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()); };
  const auto end = [&](const Tensor& t) {
    return begin(t) + ((t.size(0) - 1) * t.stride(0) + (t.size(1) - 1) * t.stride(1) + 1) * t.element_size();
  };
  return begin(x) < end(y) && begin(y) < end(x);
}
int64_t wide_stride(const Tensor& x) { return x.size(0) > 1 && x.size(1) ? x.stride(0) : x.size(1); }

Tensor empty(at::IntArrayRef size, const Tensor& like, at::ScalarType type) {
  return at::empty(size, like.options().dtype(type));
}

Tensor bytes(int64_t n, const Tensor& like) { return empty({n}, like, at::kByte); }

// [rows, cols] of 1-byte values whose rows start `ld` bytes apart
Tensor empty_rows(int64_t rows, int64_t cols, const Tensor& like, at::ScalarType type, int64_t ld) {
  const Tensor t = empty({rows, ld}, like, type);
  return ld == cols ? t : t.narrow(1, 0, cols);
}

struct Made {  // a tensor in 8 bits and where a kernel writes it
  Tensor q, scale;
  Fp8Out out{};
  Made() = default;
  Made(int64_t rows, int64_t cols, const Tensor& like, at::ScalarType type, int block_rows)
      : q(empty_rows(rows, cols, like, type, gpuexp::fp8_row_bytes(cols))),
        scale(empty_rows((rows + block_rows - 1) / block_rows, blocks(cols), like, at::kFloat8_e8m0fnu,
                         up(blocks(cols), 4))),
        out{static_cast<uint8_t*>(q.mutable_data_ptr()), static_cast<uint8_t*>(scale.mutable_data_ptr()),
            gpuexp::fp8_row_bytes(cols), up(blocks(cols), 4)} {}
};

// (q, scale) with rows that start where the kernels want them: what does already is given back as it is
Pair align_fp8(const Tensor& q, const Tensor& scale) {
  check_pair("q", q, scale);
  const at::NoGradGuard none;
  const auto aligned = [](const Tensor& t, int64_t pad, int64_t ld) {
    if (Rows(t, pad).ok) return t;
    const Tensor rows = empty_rows(t.size(0), t.size(1), t, t.scalar_type(), ld);
    rows.copy_(t);
    return rows;
  };
  return {aligned(q, 16, gpuexp::fp8_row_bytes(q.size(1))), aligned(scale, 4, up(scale.size(1), 4))};
}

std::pair<Made, Made> quantize(const Tensor& x, at::ScalarType dtype, int64_t block_rows, bool columns) {
  TORCH_CHECK_TYPE(fp8_type(dtype) >= 0, "quantize_fp8 makes float8_e4m3fn or float8_e5m2, not ", dtype);
  TORCH_CHECK_VALUE(block_rows == 1 || block_rows == kFp8Block, "block_rows is 1 or 128, got ", block_rows);
  TORCH_CHECK_TYPE(wide_type(x.scalar_type()) >= 0, "x must be bfloat16, float16 or float32, got ", x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() == 2, "x must be 2-dimensional, got ", x.sizes());
  TORCH_CHECK_VALUE(row_major(x), "x must be row-major with its columns next to each other, got strides ", x.strides());
  check_gpu("quantize_fp8", x);
  const int64_t m = x.size(0), k = x.size(1);
  const On on(x);
  Made out, out_t;
  out = Made(m, k, x, dtype, int(block_rows));
  if (columns) out_t = Made(k, m, x, dtype, int(block_rows));
  if (m && k)
    check(gpuexp::launch_quantize_fp8(x.const_data_ptr(), wide_type(x.scalar_type()), wide_stride(x), m, k,
                                      fp8_type(dtype), int(block_rows), out.out, out_t.out, on.stream),
          "quantize_fp8");
  return {std::move(out), std::move(out_t)};
}

Pair quantize_fp8(const Tensor& x, at::ScalarType dtype, int64_t block_rows) {
  auto [out, none] = quantize(x, dtype, block_rows, false);
  return {std::move(out.q), std::move(out.scale)};
}

Four quantize_fp8_both(const Tensor& x, at::ScalarType dtype, int64_t block_rows) {
  auto [out, out_t] = quantize(x, dtype, block_rows, true);
  return {std::move(out.q), std::move(out.scale), std::move(out_t.q), std::move(out_t.scale)};
}

Tensor dequantize_fp8(const Tensor& q, const Tensor& scale, at::ScalarType dtype) {
  const Fp8In in = operand("q", q, scale);
  TORCH_CHECK_TYPE(wide_type(dtype) >= 0, "dequantize_fp8 gives bfloat16, float16 or float32, not ", dtype);
  check_gpu("dequantize_fp8", q, scale);
  const int64_t rows = q.size(0), cols = q.size(1);
  const On on(q);
  Tensor x = empty({rows, cols}, q, dtype);
  if (rows && cols)
    check(gpuexp::launch_dequantize_fp8(in, rows, cols, x.mutable_data_ptr(), wide_type(dtype), cols, on.stream),
          "dequantize_fp8");
  return x;
}

Pair transpose_fp8(const Tensor& q, const Tensor& scale) {
  const Fp8In in = operand("q", q, scale);
  check_gpu("transpose_fp8", q, scale);
  const int64_t rows = q.size(0), cols = q.size(1);
  const On on(q);
  Made out(cols, rows, q, q.scalar_type(), in.block_rows);
  if (rows && cols) check(gpuexp::launch_transpose_fp8(in, rows, cols, out.out, on.stream), "transpose_fp8");
  return {std::move(out.q), std::move(out.scale)};
}

Tensor product(const Tensor& a, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale, const Tensor* given,
               at::ScalarType out_dtype, int64_t variant, int64_t parts) {
  const Fp8In oa = operand("a", a, a_scale), ob = operand("b", b, b_scale);
  const int64_t M = a.size(0), K = a.size(1), N = b.size(0);
  TORCH_CHECK_VALUE(b.size(1) == K, "shape mismatch ", a.sizes(), " x ", b.sizes(), "^T");
  const at::ScalarType dtype = given ? given->scalar_type() : out_dtype;
  TORCH_CHECK_TYPE(dtype == at::kBFloat16 || dtype == at::kHalf, "gemm_fp8 writes bfloat16 or float16, not ", dtype);
  if (given)
    TORCH_CHECK_VALUE(given->dim() == 2 && given->size(0) == M && given->size(1) == N && row_major(*given),
                      "out must be [", M, ", ", N, "] with its columns next to each other, got ", given->sizes(),
                      ", strides ", given->strides());
  const gpuexp::GemmFp8Plan plan = gpuexp::plan_gemm_fp8(M, N, K, variant, parts);
  TORCH_CHECK_VALUE(plan.variant >= 0, "variant ", variant, " with ", parts, " parts does not take these sizes (", M, ", ",
                    N, ", ", K, ")", variant == 0 && parts == 0 ? ": more blocks than a launch has" : "");
  check_gpu("gemm_fp8", a, a_scale, b, b_scale, given ? *given : a);
  TORCH_CHECK_VALUE(K <= kLongest, "gemm_fp8: rows of at most ", kLongest, " values, got ", K);
  const On on(a);
  Tensor out = given ? *given : empty({M, N}, a, dtype);
  if (given) {
    TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() && given->requires_grad()), "out takes a gradient, which gemm_fp8 "
                      "has none to give");
    for (const Tensor* t : {&a, &a_scale, &b, &b_scale})
      TORCH_CHECK_VALUE(!overlap(*given, *t), "out must not overlap an input");
    out.unsafeGetTensorImpl()->bump_version();  // an in-place change, to whoever saved `out`
  }
  if (M && N) {
    Tensor temp;
    if (const int64_t need = gpuexp::gemm_fp8_temp_bytes(M, N, plan)) temp = bytes(need, a);
    check(gpuexp::launch_gemm_fp8({oa, ob, out.mutable_data_ptr(), wide_stride(out), M, N, K, wide_type(dtype),
                                   plan.variant, plan.parts, temp.defined() ? temp.mutable_data_ptr() : nullptr},
                                  on.stream),
          "gemm_fp8");
  }
  return out;
}

Tensor gemm_fp8(const Tensor& a, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale,
                at::ScalarType out_dtype, int64_t variant, int64_t parts) {
  return product(a, a_scale, b, b_scale, nullptr, out_dtype, variant, parts);
}

void gemm_fp8_out(const Tensor& a, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale, const Tensor& out,
                  int64_t variant, int64_t parts) {
  product(a, a_scale, b, b_scale, &out, out.scalar_type(), variant, parts);
}

Tensor rows_of(const Tensor& x) { return row_major(x) ? x : x.contiguous(); }

// what a layer's passes take: x [M, K] and w [N, K] as checked_linear passes them on
void check_layer(const Tensor& x, at::ScalarType wtype) {
  TORCH_CHECK_TYPE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf,
                   "linear_fp8 takes bfloat16 or float16 activations, got ", x.scalar_type());
  TORCH_CHECK_TYPE(wtype == at::kBFloat16 || wtype == at::kHalf,
                   "linear_fp8 takes bfloat16 or float16 weights, or 8-bit ones with weight_scale, got ", wtype);
}

// y = x w^T of x [M, K], w [N, K] and the workspace that the backward pass needs
Pair linear_fp8_forward(const Tensor& x, const Tensor& w, bool keep_dx, bool keep_dw) {
  check_layer(x, w.scalar_type());
  check_gpu("linear_fp8", x, w);
  TORCH_CHECK_VALUE(x.dim() == 2 && w.dim() == 2 && x.size(1) == w.size(1) && row_major(x) && row_major(w),
                    "linear_fp8_forward takes row-major x [M, K] and w [N, K], got ", x.sizes(), " and ", w.sizes());
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  const On on(x);
  Tensor y = empty({M, N}, x, x.scalar_type()),
         kept = bytes(gpuexp::linear_fp8_kept_bytes(M, N, K, keep_dx, keep_dw), x),
         temp = bytes(gpuexp::linear_fp8_forward_bytes(M, N, K, keep_dx, keep_dw), x);
  gpuexp::LinearFp8Args a{M, N, K, keep_dx, keep_dw, false, false, x.const_data_ptr(), wide_stride(x), w.const_data_ptr(),
                          wide_stride(w), wide_type(x.scalar_type()), wide_type(w.scalar_type()),
                          static_cast<uint8_t*>(kept.mutable_data_ptr()), static_cast<uint8_t*>(temp.mutable_data_ptr())};
  check(gpuexp::launch_linear_fp8_forward(a, y.mutable_data_ptr(), on.stream), "linear_fp8");
  return {std::move(y), std::move(kept)};
}

// (dx, dw) of dy [M, N] and what the forward pass kept for them; one that is not wanted is undefined
Pair linear_fp8_backward(const Tensor& given, const Tensor& kept, int64_t K, at::ScalarType wtype, bool kept_dx,
                         bool kept_dw, bool want_dx, bool want_dw) {
  const Tensor dy = rows_of(given);
  check_layer(dy, wtype);
  check_gpu("linear_fp8", dy, kept);
  const int64_t M = dy.size(0), N = dy.size(1);
  TORCH_CHECK_VALUE(dy.dim() == 2 && kept.scalar_type() == at::kByte && kept.is_contiguous() &&
                        kept.numel() == gpuexp::linear_fp8_kept_bytes(M, N, K, kept_dx, kept_dw) &&
                        (kept_dx || !want_dx) && (kept_dw || !want_dw),
                    "linear_fp8_backward: what was kept is not of these sizes, or not for these gradients");
  const On on(dy);
  Tensor dx, dw;
  if (want_dx) dx = empty({M, K}, dy, dy.scalar_type());
  if (want_dw) dw = empty({N, K}, dy, wtype);
  const Tensor temp = bytes(gpuexp::linear_fp8_backward_bytes(M, N, K, want_dx, want_dw), dy);
  gpuexp::LinearFp8Args a{M, N, K, kept_dx, kept_dw, want_dx, want_dw, nullptr, 0, nullptr, 0,
                          wide_type(dy.scalar_type()), wide_type(wtype),
                          static_cast<uint8_t*>(kept.mutable_data_ptr()), static_cast<uint8_t*>(temp.mutable_data_ptr())};
  check(gpuexp::launch_linear_fp8_backward(a, dy.const_data_ptr(), wide_stride(dy),
                                           want_dx ? dx.mutable_data_ptr() : nullptr,
                                           want_dw ? dw.mutable_data_ptr() : nullptr, on.stream),
        "linear_fp8's backward pass");
  return {std::move(dx), std::move(dw)};
}

Tensor serve(const Tensor& x, const Tensor& w, const Tensor& scale) {
  const Fp8In in = operand("weight", w, scale);
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  const On on(x);
  Tensor y = empty({M, N}, x, x.scalar_type());
  const int64_t need = gpuexp::serve_fp8_bytes(x.const_data_ptr(), wide_stride(x), M, N, K);
  Tensor temp;
  if (need) temp = bytes(need, x);
  check(gpuexp::launch_serve_fp8(x.const_data_ptr(), wide_type(x.scalar_type()), wide_stride(x), in, M, N, K,
                                 y.mutable_data_ptr(), need ? static_cast<uint8_t*>(temp.mutable_data_ptr()) : nullptr,
                                 on.stream),
        "linear_fp8");
  return y;
}

// the checks of a layer's arguments, and x's rows [M, K]
Tensor checked_linear(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& scale, bool want_dx,
                      bool want_dw) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 2 && x.size(-1) == weight.size(1), "shape mismatch ", x.sizes(),
                    " x ", weight.sizes(), "^T");
  check_layer(x, scale ? x.scalar_type() : weight.scalar_type());
  if (scale) {
    TORCH_CHECK_VALUE(!weight.requires_grad(), "weights in 8 bits take no gradient");
    operand("weight", weight, *scale);
  }
  const int64_t N = weight.size(0), K = x.size(-1);
  int64_t M = 1;
  for (int64_t d = 0; d < x.dim() - 1; ++d) M *= x.size(d);
  TORCH_CHECK_VALUE(K <= kLongest && (!want_dx || N <= kLongest) && (!want_dw || M <= kLongest),
                    "linear_fp8: at most ", kLongest, " inputs, for x's gradient as many outputs and for the weight's as "
                    "many rows of x, got ", K, ", ", N, " and ", M);
  // (here, so that no backward pass is refused after its forward pass has run)
  TORCH_CHECK_VALUE(scale ? gpuexp::serve_fp8_ok(M, N, K, want_dx) : gpuexp::linear_fp8_ok(M, N, K, want_dx, want_dw),
                    "linear_fp8: ", M, " rows of ", K, " inputs and ", N, " outputs are ", kLimits);
  if (scale) check_gpu("linear_fp8", x, weight, *scale);
  else check_gpu("linear_fp8", x, weight);
  return rows_of(x.dim() == 2 ? x : x.reshape({M, K}));
}

Tensor as_given(const Tensor& y, const Tensor& x) {
  if (x.dim() == 2) return y;
  std::vector<int64_t> size(x.sizes().begin(), x.sizes().end());
  size.back() = y.size(1);
  return y.reshape(size);
}

// without autograd
Tensor linear_fp8(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& scale) {
  const Tensor x2 = checked_linear(x, weight, scale, false, false);
  return as_given(scale ? serve(x2, weight, *scale) : std::get<0>(linear_fp8_forward(x2, rows_of(weight), false, false)), x);
}

// ---- the operators through torch's dispatcher ----
template <typename F>
c10::TypedOperatorHandle<F> find(const char* name, F*) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
#define GPUEXP_CALL(op, ...)                            \
  ([&] {                                                \
    static const auto handle = find("gpuexp::" #op, op); \
    return handle.call(__VA_ARGS__);                    \
  }())

variable_list once(variable_list results) {
  // Gradients of gradients are refused where they are asked for, not where the first ones are made; also for a
  // constant dy, since dx depends on the weight and dw on x.
  if (!at::GradMode::is_enabled()) return results;
  for (Tensor& t : results) {  // DelayedError hangs its refusal only on tensors that take a gradient
    if (t.defined()) t.set_requires_grad(true);
  }
  auto error = std::make_shared<torch::autograd::DelayedError>("linear_fp8 cannot be differentiated twice",
                                                               int(results.size()));
  return (*error)(std::move(results));
}

struct LinearFp8 : torch::autograd::Function<LinearFp8> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w) {
    const bool keep_dx = x.requires_grad(), keep_dw = w.requires_grad();
    auto [y, kept] = GPUEXP_CALL(linear_fp8_forward, x, w, keep_dx, keep_dw);
    ctx->save_for_backward({kept});
    ctx->saved_data["sizes"] = std::vector<int64_t>{x.size(1), keep_dx, keep_dw, int64_t(w.scalar_type())};
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor kept = ctx->get_saved_variables()[0];
    const std::vector<int64_t> s = ctx->saved_data["sizes"].toIntVector();
    const bool kept_dx = s[1] != 0, kept_dw = s[2] != 0;
    // a call may ask for one gradient alone (torch.autograd.grad(y, x), backward(inputs=[w]))
    const bool want_dx = kept_dx && ctx->needs_input_grad(0), want_dw = kept_dw && ctx->needs_input_grad(1);
    variable_list results(2);
    {
      at::AutoGradMode off(false);
      std::tie(results[0], results[1]) = GPUEXP_CALL(linear_fp8_backward, grads[0], kept, s[0], at::ScalarType(s[3]),
                                                     kept_dx, kept_dw, want_dx, want_dw);
    }
    return once(std::move(results));
  }
};

struct ServeFp8 : torch::autograd::Function<ServeFp8> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& scale) {
    ctx->save_for_backward({w, scale});
    return GPUEXP_CALL(linear_fp8, x, w, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list results(3);
    {
      at::AutoGradMode off(false);
      const Pair g = GPUEXP_CALL(quantize_fp8, rows_of(grads[0]), at::kFloat8_e4m3fn, 1);
      const Pair wt = GPUEXP_CALL(transpose_fp8, saved[0], saved[1]);
      results[0] = GPUEXP_CALL(gemm_fp8, std::get<0>(g), std::get<1>(g), std::get<0>(wt), std::get<1>(wt),
                               grads[0].scalar_type(), 0, 0);
    }
    return once(std::move(results));
  }
};

// (below autograd the tangent would be dropped without a word)
void check_no_tangent(const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(),
                              "linear_fp8 has no forward-mode derivative");
}

Tensor linear_fp8_autograd(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& scale) {
  check_no_tangent(x);
  check_no_tangent(weight);
  const bool grad = at::GradMode::is_enabled(), want_dx = grad && x.requires_grad(),
             want_dw = grad && weight.requires_grad();
  if (!want_dx && !want_dw) {
    at::AutoDispatchBelowADInplaceOrView below;
    return GPUEXP_CALL(linear_fp8, x, weight, scale);
  }
  const Tensor x2 = checked_linear(x, weight, scale, want_dx, want_dw);
  return as_given(scale ? ServeFp8::apply(x2, weight, *scale) : LinearFp8::apply(x2, rows_of(weight)), x);
}

TORCH_LIBRARY(gpuexp, m) {
  m.def("quantize_fp8(Tensor x, ScalarType dtype, int block_rows) -> (Tensor, Tensor)");
  m.def("quantize_fp8_both(Tensor x, ScalarType dtype, int block_rows) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("dequantize_fp8(Tensor q, Tensor scale, ScalarType dtype) -> Tensor");
  m.def("transpose_fp8(Tensor q, Tensor scale) -> (Tensor, Tensor)");
  m.def("gemm_fp8(Tensor a, Tensor a_scale, Tensor b, Tensor b_scale, ScalarType out_dtype, int variant, int parts) "
        "-> Tensor");
  m.def("gemm_fp8_out(Tensor a, Tensor a_scale, Tensor b, Tensor b_scale, Tensor(a!) out, int variant, int parts) -> ()");
  m.def("linear_fp8(Tensor x, Tensor weight, Tensor? weight_scale) -> Tensor");
  m.def("linear_fp8_forward(Tensor x, Tensor weight, bool keep_dx, bool keep_dw) -> (Tensor, Tensor)");
  m.def("linear_fp8_backward(Tensor dy, Tensor kept, int inputs, ScalarType weight_dtype, bool kept_dx, bool kept_dw, "
        "bool want_dx, bool want_dw) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(gpuexp, CompositeExplicitAutograd, m) {
  m.impl("quantize_fp8", quantize_fp8);
  m.impl("quantize_fp8_both", quantize_fp8_both);
  m.impl("dequantize_fp8", dequantize_fp8);
  m.impl("transpose_fp8", transpose_fp8);
  m.impl("gemm_fp8", gemm_fp8);
  m.impl("gemm_fp8_out", gemm_fp8_out);
  m.impl("linear_fp8", linear_fp8);
  m.impl("linear_fp8_forward", linear_fp8_forward);
  m.impl("linear_fp8_backward", linear_fp8_backward);
}

TORCH_LIBRARY_IMPL(gpuexp, Autograd, m) {
  m.impl("linear_fp8", linear_fp8_autograd);
  // the others take no part in autograd
  for (const char* name : {"quantize_fp8", "quantize_fp8_both", "dequantize_fp8", "transpose_fp8", "gemm_fp8",
                           "gemm_fp8_out", "linear_fp8_forward", "linear_fp8_backward"})
    m.impl(name, torch::CppFunction::makeFallthrough());
}

}  // namespace

// Loaded after torch, whose HIP runtime it then shares (see ops/gemm.py).
PYBIND11_MODULE(_gpuexp_fp8, m) {
  m.doc() = "8-bit floating point with block scales on torch tensors (ops/fp8.py)";
  m.def("quantize_fp8", [](const Tensor& x, at::ScalarType dtype, int64_t block_rows) {
    return GPUEXP_CALL(quantize_fp8, x, dtype, block_rows);
  });
  m.def("quantize_fp8_both", [](const Tensor& x, at::ScalarType dtype, int64_t block_rows) {
    auto [q, scale, q_t, scale_t] = GPUEXP_CALL(quantize_fp8_both, x, dtype, block_rows);
    return std::make_tuple(Pair{std::move(q), std::move(scale)}, Pair{std::move(q_t), std::move(scale_t)});
  });
  m.def("dequantize_fp8", [](const Tensor& q, const Tensor& scale, at::ScalarType dtype) {
    return GPUEXP_CALL(dequantize_fp8, q, scale, dtype);
  });
  m.def("align_fp8", align_fp8);
  m.def("transpose_fp8", [](const Tensor& q, const Tensor& scale) { return GPUEXP_CALL(transpose_fp8, q, scale); });
  m.def("gemm_fp8", [](const Tensor& a, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale,
                       const std::optional<Tensor>& out, at::ScalarType out_dtype, int64_t variant, int64_t parts) {
    if (!out) return GPUEXP_CALL(gemm_fp8, a, a_scale, b, b_scale, out_dtype, variant, parts);
    GPUEXP_CALL(gemm_fp8_out, a, a_scale, b, b_scale, *out, variant, parts);
    return *out;
  });
  m.def("linear_fp8", [](const Tensor& x, const Tensor& weight, const std::optional<Tensor>& weight_scale) {
    return GPUEXP_CALL(linear_fp8, x, weight, weight_scale);
  });
  m.def("gemm_fp8_plan", [](int64_t M, int64_t N, int64_t K, int64_t variant, int64_t parts) {
    const gpuexp::GemmFp8Plan plan = gpuexp::plan_gemm_fp8(M, N, K, variant, parts);
    return std::make_pair(plan.variant, plan.parts);
  }, py::arg("M"), py::arg("N"), py::arg("K"), py::arg("variant") = 0, py::arg("parts") = 0,
     "The kernel variant and the parts of K a gemm_fp8 call with these sizes runs (0 resolved); variant -1 if they do "
     "not fit it. Host-only: no GPU needed.");
}
