// Host-side launchers of the per-token kernels as a thin torch extension over
// the C ABI (include/mi355_fused.h): argument checks, the row / stride logic
// and the output allocation of the Python launchers in kernels/*.py, done in
// C++ so an eager call costs one pybind11 dispatch instead of Python
// attribute accesses, a torch.empty from Python and a 12-argument ctypes
// call.  Torch types stop here: every kernel is reached through the
// plain-pointer entry points of libmi355_fused.so, on torch's current HIP
// stream.
//
// The behaviour is the Python launchers', which keep the reference's
// launcher contracts (src/kernels/fused_rmsnorm_triton.py:52-71,
// src/kernels/fused_swiglu_triton.py:39-53, src/kernels/w8a16_matmul_triton.py:
// 102-134): a failed precondition raises AssertionError with the same
// message, a malformed weight shape the ValueError of Python's tuple
// unpacking, and a failing C-ABI call the package's KernelError (registered
// by _lib at import) with the library's message.
#include <torch/extension.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>

#include <sstream>
#include <string>

#include "../../include/mi355_fused.h"

namespace py = pybind11;

namespace {

// The package's KernelError class.  Held through a pointer that is never
// freed: a py::object with static storage would be released after the
// interpreter has finalised, at process exit.
py::object* g_kernel_error = nullptr;

[[noreturn]] void fail_assert(const std::string& msg) {
  PyErr_SetString(PyExc_AssertionError, msg.c_str());
  throw py::error_already_set();
}

void check(const char* fn, int status) {
  if (status == MI355_OK) return;
  const std::string msg = mi355_last_error();
  if (g_kernel_error != nullptr) {
    PyErr_SetObject(g_kernel_error->ptr(), py::make_tuple(fn, status, msg).ptr());
    throw py::error_already_set();
  }
  throw std::runtime_error(std::string(fn) + " failed with status " + std::to_string(status) + ": " + msg);
}

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return MI355_F32;
    case at::kHalf: return MI355_F16;
    case at::kBFloat16: return MI355_BF16;
    default: return -1;
  }
}

// str(torch.dtype) as Python prints it, for the assertion messages.
std::string dtype_str(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kDouble: return "torch.float64";
    case at::kChar: return "torch.int8";
    case at::kByte: return "torch.uint8";
    case at::kShort: return "torch.int16";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    case at::kBool: return "torch.bool";
    default: return std::string("torch.") + c10::toString(t);
  }
}

// tuple(t.shape) as Python prints it.
std::string shape_str(at::IntArrayRef s) {
  std::ostringstream o;
  o << "(";
  for (size_t i = 0; i < s.size(); ++i) o << (i ? ", " : "") << s[i];
  if (s.size() == 1) o << ",";
  o << ")";
  return o.str();
}

// `n, k = w.shape` for a 2-D weight; Python's unpacking error otherwise.
std::pair<int64_t, int64_t> unpack2(const at::Tensor& w) {
  if (w.dim() > 2) throw py::value_error("too many values to unpack (expected 2)");
  if (w.dim() < 2) throw py::value_error("not enough values to unpack (expected 2, got " + std::to_string(w.dim()) + ")");
  return {w.size(0), w.size(1)};
}

// Launch context: `dev` current for the call (switched only when it is not),
// torch's current stream on it.
struct Launch {
  c10::optional<c10::hip::HIPGuard> guard;
  void* stream;
  explicit Launch(int dev) {
    if (c10::hip::current_device() != dev) guard.emplace(static_cast<c10::DeviceIndex>(dev));
    stream = c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(dev)).stream();
  }
};

// Rows view of t over its last dimension n: (view, row count, row stride),
// copying only when the last dimension itself is strided (a row-strided view
// is passed with its stride).
struct Rows {
  at::Tensor t;
  int64_t m, stride;
};
Rows rows_of(const at::Tensor& t, int64_t n) {
  if (t.is_contiguous()) return {t, n ? t.numel() / n : 0, n};
  at::Tensor t2 = t.reshape({-1, n});
  if (t2.stride(-1) != 1 || (t2.size(0) > 1 && t2.stride(0) < n)) t2 = t2.contiguous();
  const int64_t m = t2.size(0);
  return {t2, m, m > 1 ? t2.stride(0) : n};
}

// x as [rows, k] rows a projection kernel can stream: unit element stride
// and, over more than one row, rows that do not overlap (row stride >= k).
// A broadcast or overlapping view -- expand() gives row stride 0 -- is
// copied, as the reference's `x.reshape(-1, K).contiguous()` copies it.
at::Tensor matrix_rows(const at::Tensor& x, int64_t k) {
  at::Tensor x2 = x.reshape({-1, k});
  if (x2.stride(-1) != 1 || (x2.size(0) > 1 && x2.stride(0) < k)) x2 = x2.contiguous();
  return x2;
}

// Weight matrices [n, k] the kernels stream row by row: each with unit
// element stride and non-overlapping rows, and (for a pair read together)
// one shared row stride; copied otherwise.
bool streamable(const at::Tensor& w) {
  return w.stride(-1) == 1 && (w.size(0) <= 1 || w.stride(0) >= w.size(1));
}
std::pair<at::Tensor, at::Tensor> weight_pair(const at::Tensor& a, const at::Tensor& b) {
  if (streamable(a) && streamable(b) && a.stride(0) == b.stride(0)) return {a, b};
  return {a.contiguous(), b.contiguous()};
}

std::vector<int64_t> with_last(at::IntArrayRef s, int64_t last) {
  std::vector<int64_t> v(s.begin(), s.end());
  v.back() = last;
  return v;
}

void* ptr(const at::Tensor& t) { return t.data_ptr(); }

// Whether the split-K kernels take these operands (the alignment that the
// linears' launchers ask of everything but their generic kernels): row starts
// on 16 bytes, whole 16-byte packets per row.
bool packets(const at::Tensor& x, int64_t xs, const at::Tensor& w, int64_t ws, int64_t k) {
  const int64_t xe = x.element_size(), we = w.element_size();
  return xs * xe % 16 == 0 && ws * we % 16 == 0 && k * we % 16 == 0 &&
         (reinterpret_cast<uintptr_t>(ptr(x)) | reinterpret_cast<uintptr_t>(ptr(w))) % 16 == 0;
}

// A call's scratch memory: `bytes` from torch's allocator on the current
// stream (the launch stream, so its reuse is ordered after the call's kernels;
// a captured graph keeps it in its pool).  Undefined for 0 bytes, and where
// the memory is not to be had: the call then runs the unsplit kernels.
at::Tensor workspace(int64_t bytes, const at::Tensor& like) {
  if (bytes <= 0) return {};
  try {
    return at::empty({bytes}, like.options().dtype(at::kByte));
  } catch (const c10::OutOfMemoryError&) {
    return {};
  }
}

// ------------------------------------------------------------------ RMSNorm

at::Tensor rmsnorm(const at::Tensor& x, const at::Tensor& weight, double eps) {
  if (!(x.is_cuda() && weight.is_cuda())) fail_assert("x and weight must be ROCm GPU tensors");
  const int64_t N = x.size(-1);
  if (!(weight.dim() == 1 && weight.size(0) == N))
    fail_assert("weight shape " + shape_str(weight.sizes()) + " != (" + std::to_string(N) + ",)");
  const int code = code_of(x.scalar_type()), wcode = code_of(weight.scalar_type());
  if (code < 0 || wcode < 0)
    fail_assert("unsupported dtypes x=" + dtype_str(x.scalar_type()) + " weight=" + dtype_str(weight.scalar_type()) +
                " (fp16, bf16, fp32)");
  const int dev = x.get_device();
  if (weight.get_device() != dev) fail_assert("x and weight must be on the same device");
  const Rows r = rows_of(x, N);
  const at::Tensor w = weight.stride(0) != 1 ? weight.contiguous() : weight;
  at::Tensor out = x.is_contiguous() ? at::empty_like(x) : at::empty(x.sizes(), x.options());
  if (r.m && N) {
    Launch l(dev);
    check("mi355_rmsnorm_fwd", mi355_rmsnorm_fwd(ptr(r.t), ptr(w), ptr(out), r.m, N, r.stride, N,
                                                 static_cast<float>(eps), code, wcode, code, l.stream));
  }
  return out;
}

std::tuple<at::Tensor, at::Tensor> add_rmsnorm(const at::Tensor& x, const at::Tensor& residual,
                                               const at::Tensor& weight, double eps) {
  if (!(x.is_cuda() && residual.is_cuda() && weight.is_cuda()))
    fail_assert("x, residual and weight must be ROCm GPU tensors");
  if (x.sizes() != residual.sizes())
    fail_assert("shape mismatch " + shape_str(x.sizes()) + " vs " + shape_str(residual.sizes()));
  if (x.scalar_type() != residual.scalar_type())
    fail_assert("dtype mismatch " + dtype_str(x.scalar_type()) + " vs " + dtype_str(residual.scalar_type()));
  const int64_t N = x.size(-1);
  if (!(weight.dim() == 1 && weight.size(0) == N))
    fail_assert("weight shape " + shape_str(weight.sizes()) + " != (" + std::to_string(N) + ",)");
  const int code = code_of(x.scalar_type()), wcode = code_of(weight.scalar_type());
  if (code < 0 || wcode < 0)
    fail_assert("unsupported dtypes x=" + dtype_str(x.scalar_type()) + " weight=" + dtype_str(weight.scalar_type()) +
                " (fp16, bf16, fp32)");
  const int dev = x.get_device();
  if (residual.get_device() != dev || weight.get_device() != dev)
    fail_assert("x, residual and weight must be on the same device");
  const Rows xr = rows_of(x, N), rr = rows_of(residual, N);
  const at::Tensor w = weight.stride(0) != 1 ? weight.contiguous() : weight;
  at::Tensor out = at::empty(x.sizes(), x.options());
  at::Tensor h = at::empty(x.sizes(), x.options());
  if (xr.m && N) {
    Launch l(dev);
    check("mi355_add_rmsnorm_fwd",
          mi355_add_rmsnorm_fwd(ptr(xr.t), ptr(rr.t), ptr(w), ptr(out), ptr(h), xr.m, N, xr.stride, rr.stride, N, N,
                                static_cast<float>(eps), code, wcode, code, l.stream));
  }
  return {out, h};
}

// ------------------------------------------------------------- SiLU-and-mul

at::Tensor silu_mul(const at::Tensor& gate, const at::Tensor& up) {
  if (gate.sizes() != up.sizes())
    fail_assert("shape mismatch " + shape_str(gate.sizes()) + " vs " + shape_str(up.sizes()));
  if (!(gate.is_cuda() && up.is_cuda())) fail_assert("gate and up must be ROCm GPU tensors");
  int code = code_of(gate.scalar_type());
  const int ucode = code_of(up.scalar_type());
  if (code < 0 || ucode < 0)
    fail_assert("unsupported dtypes gate=" + dtype_str(gate.scalar_type()) + " up=" + dtype_str(up.scalar_type()) +
                " (fp16, bf16, fp32)");
  const int dev = gate.get_device();
  if (up.get_device() != dev) fail_assert("gate and up must be on the same device");
  at::Tensor g, u;
  if (code != ucode) {
    // the reference widens each input to fp32 separately; widening both here
    // is exact, and the fp32 result is rounded once below
    g = gate.contiguous().to(at::kFloat);
    u = up.contiguous().to(at::kFloat);
    code = MI355_F32;
  } else {
    g = gate.is_contiguous() ? gate : gate.contiguous();
    u = up.is_contiguous() ? up : up.contiguous();
  }
  at::Tensor out = at::empty_like(g);
  const int64_t n = g.numel();
  if (n) {
    Launch l(dev);
    check("mi355_silu_mul_fwd", mi355_silu_mul_fwd(ptr(g), ptr(u), ptr(out), n, code, code, l.stream));
  }
  if (out.scalar_type() != gate.scalar_type()) out = out.to(gate.scalar_type());
  return out.view(gate.sizes());
}

// ------------------------------------------------- gate/up + SiLU-and-mul

at::Tensor gate_up_silu(const at::Tensor& x, const at::Tensor& w_gate, const at::Tensor& w_up, bool out_f32) {
  if (!(x.is_cuda() && w_gate.is_cuda() && w_up.is_cuda())) fail_assert("x and the weights must be ROCm GPU tensors");
  if (x.scalar_type() != at::kHalf && x.scalar_type() != at::kBFloat16)
    fail_assert("x must be fp16 or bf16, got " + dtype_str(x.scalar_type()));
  if (w_gate.scalar_type() != x.scalar_type() || w_up.scalar_type() != x.scalar_type())
    fail_assert("dtype mismatch x=" + dtype_str(x.scalar_type()) + " w_gate=" + dtype_str(w_gate.scalar_type()) +
                " w_up=" + dtype_str(w_up.scalar_type()));
  const int64_t k = x.size(-1);
  if (!(w_gate.dim() == 2 && w_gate.sizes() == w_up.sizes() && w_gate.size(1) == k))
    fail_assert("weights must be [n_out, " + std::to_string(k) + "], got " + shape_str(w_gate.sizes()) + " and " +
                shape_str(w_up.sizes()));
  const int dev = x.get_device();
  if (w_gate.get_device() != dev || w_up.get_device() != dev) fail_assert("x and the weights must share a device");
  const at::ScalarType odt = out_f32 ? at::kFloat : x.scalar_type();

  const int64_t n_out = w_gate.size(0);
  const at::Tensor x2 = matrix_rows(x, k);
  const auto [wg, wu] = weight_pair(w_gate, w_up);
  const int64_t rows = x2.size(0);
  at::Tensor out = at::empty({rows, n_out}, x.options().dtype(odt));
  if (rows && n_out) {
    // a single row's stride is arbitrary in torch (even 0); the kernel reads one row then
    const int64_t xs = rows > 1 ? x2.stride(0) : k;
    const int64_t ws = n_out > 1 ? wg.stride(0) : k;
    Launch l(dev);
    check("mi355_gate_up_silu_fwd",
          mi355_gate_up_silu_fwd(ptr(x2), ptr(wg), ptr(wu), ptr(out), rows, k, n_out, xs, ws, n_out,
                                 code_of(x.scalar_type()), code_of(odt), l.stream));
  }
  return out.view(with_last(x.sizes(), n_out));
}

// ------------------------------------------------------------ 16-bit linear

at::Tensor linear16(const at::Tensor& x, const at::Tensor& weight, const c10::optional<at::Tensor>& bias,
                    bool out_f32) {
  if (!(x.is_cuda() && weight.is_cuda())) fail_assert("x and weight must be ROCm GPU tensors");
  if (x.scalar_type() != at::kHalf && x.scalar_type() != at::kBFloat16)
    fail_assert("x must be fp16 or bf16, got " + dtype_str(x.scalar_type()));
  if (weight.scalar_type() != x.scalar_type())
    fail_assert("dtype mismatch x=" + dtype_str(x.scalar_type()) + " weight=" + dtype_str(weight.scalar_type()));
  if (weight.dim() != 2) fail_assert("weight must be (N, K), got " + shape_str(weight.sizes()));
  const int64_t N = weight.size(0), K = weight.size(1);
  if (x.size(-1) != K)
    fail_assert("x last dim " + std::to_string(x.size(-1)) + " != weight in_features " + std::to_string(K));
  const bool has_bias = bias.has_value() && bias->defined();
  if (has_bias && !(bias->is_cuda() && bias->dim() == 1 && bias->size(0) == N && code_of(bias->scalar_type()) >= 0))
    fail_assert("bias must be a (" + std::to_string(N) + ",) float GPU tensor, got " + shape_str(bias->sizes()) + " " +
                dtype_str(bias->scalar_type()));
  const int dev = x.get_device();
  if (weight.get_device() != dev || (has_bias && bias->get_device() != dev))
    fail_assert("x, weight and bias must share a device");
  const at::ScalarType odt = out_f32 ? at::kFloat : x.scalar_type();

  const at::Tensor x2 = matrix_rows(x, K);
  const at::Tensor w = streamable(weight) ? weight : weight.contiguous();
  const at::Tensor b = has_bias ? bias->contiguous() : at::Tensor();
  const int64_t M = x2.size(0);
  at::Tensor out = at::empty({M, N}, x.options().dtype(odt));
  if (M && N) {
    const int64_t xs = M > 1 ? x2.stride(0) : K;
    const int64_t ws = N > 1 ? w.stride(0) : K;
    Launch l(dev);
    const at::Tensor work = workspace(packets(x2, xs, w, ws, K) ? mi355_linear16_workspace(M, K, N) : 0, x);
    check("mi355_linear16_fwd",
          mi355_linear16_ws_fwd(ptr(x2), ptr(w), has_bias ? ptr(b) : nullptr, ptr(out), M, K, N, xs, ws, N,
                                code_of(x.scalar_type()), has_bias ? code_of(b.scalar_type()) : 0, code_of(odt),
                                work.defined() ? ptr(work) : nullptr, work.defined() ? work.numel() : 0, l.stream));
  }
  return out.reshape(with_last(x.sizes(), N));
}

// ------------------------------------------------------------------- W8A16

at::Tensor w8a16_linear(const at::Tensor& x, const at::Tensor& w_q, const at::Tensor& scale,
                        const c10::optional<at::Tensor>& bias, bool out_f32) {
  if (!(x.is_cuda() && w_q.is_cuda())) fail_assert("x and w_q must be ROCm GPU tensors");
  if (w_q.scalar_type() != at::kChar) fail_assert("w_q must be int8, got " + dtype_str(w_q.scalar_type()));
  const auto [N, K] = unpack2(w_q);
  if (x.size(-1) != K)
    fail_assert("x last dim " + std::to_string(x.size(-1)) + " != weight in_features " + std::to_string(K));
  if (x.scalar_type() != at::kHalf && x.scalar_type() != at::kBFloat16)
    fail_assert("x must be fp16 or bf16, got " + dtype_str(x.scalar_type()));
  if (!(scale.is_cuda() && scale.dim() == 1 && scale.size(0) == N && code_of(scale.scalar_type()) >= 0))
    fail_assert("scale must be a (" + std::to_string(N) + ",) float GPU tensor, got " + shape_str(scale.sizes()) + " " +
                dtype_str(scale.scalar_type()));
  const bool has_bias = bias.has_value() && bias->defined();
  if (has_bias && !(bias->is_cuda() && bias->dim() == 1 && bias->size(0) == N && code_of(bias->scalar_type()) >= 0))
    fail_assert("bias must be a (" + std::to_string(N) + ",) float GPU tensor, got " + shape_str(bias->sizes()) + " " +
                dtype_str(bias->scalar_type()));
  const int dev = x.get_device();
  if (w_q.get_device() != dev || scale.get_device() != dev || (has_bias && bias->get_device() != dev))
    fail_assert("x, w_q, scale and bias must share a device");
  const at::ScalarType odt = out_f32 ? at::kFloat : x.scalar_type();

  const at::Tensor x2 = matrix_rows(x, K);
  const at::Tensor q = streamable(w_q) ? w_q : w_q.contiguous();
  const at::Tensor s = scale.contiguous();
  const at::Tensor b = has_bias ? bias->contiguous() : at::Tensor();
  const int64_t M = x2.size(0);
  at::Tensor out = at::empty({M, N}, x.options().dtype(odt));
  if (M && N) {
    const int64_t xs = M > 1 ? x2.stride(0) : K;
    const int64_t ws = N > 1 ? q.stride(0) : K;
    Launch l(dev);
    const at::Tensor work = workspace(packets(x2, xs, q, ws, K) ? mi355_w8a16_linear_workspace(M, K, N) : 0, x);
    check("mi355_w8a16_linear_fwd",
          mi355_w8a16_linear_ws_fwd(ptr(x2), ptr(q), ptr(s), has_bias ? ptr(b) : nullptr, ptr(out), M, K, N, xs, ws, N,
                                    code_of(x.scalar_type()), code_of(s.scalar_type()),
                                    has_bias ? code_of(b.scalar_type()) : 0, code_of(odt),
                                    work.defined() ? ptr(work) : nullptr, work.defined() ? work.numel() : 0, l.stream));
  }
  return out.reshape(with_last(x.sizes(), N));
}

at::Tensor gate_up_silu_w8a16(const at::Tensor& x, const at::Tensor& wq_gate, const at::Tensor& scale_gate,
                              const at::Tensor& wq_up, const at::Tensor& scale_up, bool out_f32) {
  if (!(x.is_cuda() && wq_gate.is_cuda() && wq_up.is_cuda())) fail_assert("x and the weights must be ROCm GPU tensors");
  if (!(wq_gate.scalar_type() == at::kChar && wq_up.scalar_type() == at::kChar)) fail_assert("weights must be int8");
  if (wq_gate.sizes() != wq_up.sizes())
    fail_assert("weight shapes differ: " + shape_str(wq_gate.sizes()) + " vs " + shape_str(wq_up.sizes()));
  const auto [N, K] = unpack2(wq_gate);
  if (x.size(-1) != K)
    fail_assert("x last dim " + std::to_string(x.size(-1)) + " != weight in_features " + std::to_string(K));
  if (x.scalar_type() != at::kHalf && x.scalar_type() != at::kBFloat16)
    fail_assert("x must be fp16 or bf16, got " + dtype_str(x.scalar_type()));
  for (const at::Tensor* sc : {&scale_gate, &scale_up}) {
    if (!(sc->is_cuda() && sc->dim() == 1 && sc->size(0) == N && code_of(sc->scalar_type()) >= 0))
      fail_assert("scales must be (" + std::to_string(N) + ",) float GPU tensors, got " + shape_str(sc->sizes()) + " " +
                  dtype_str(sc->scalar_type()));
  }
  if (scale_gate.scalar_type() != scale_up.scalar_type()) fail_assert("the two scales must share a dtype");
  const int dev = x.get_device();
  for (const at::Tensor* t : {&wq_gate, &wq_up, &scale_gate, &scale_up}) {
    if (t->get_device() != dev) fail_assert("all inputs must share a device");
  }
  const at::ScalarType odt = out_f32 ? at::kFloat : x.scalar_type();

  const at::Tensor x2 = matrix_rows(x, K);
  const auto [qg, qu] = weight_pair(wq_gate, wq_up);
  const at::Tensor sg = scale_gate.contiguous(), su = scale_up.contiguous();
  const int64_t M = x2.size(0);
  at::Tensor out = at::empty({M, N}, x.options().dtype(odt));
  if (M && N) {
    const int64_t xs = M > 1 ? x2.stride(0) : K;
    const int64_t ws = N > 1 ? qg.stride(0) : K;
    Launch l(dev);
    check("mi355_gate_up_silu_w8a16_fwd",
          mi355_gate_up_silu_w8a16_fwd(ptr(x2), ptr(qg), ptr(qu), ptr(sg), ptr(su), ptr(out), M, K, N, xs, ws, N,
                                       code_of(x.scalar_type()), code_of(sg.scalar_type()), code_of(odt), l.stream));
  }
  return out.reshape(with_last(x.sizes(), N));
}

// -------------------------------------- rotary positions, key/value cache

typedef c10::optional<at::Tensor> OptTensor;
bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

// x [batch, tokens, heads, d] by its strides; copied where d is strided or
// (packets) a row does not start on 16 bytes.
struct Heads4 {
  at::Tensor t;  // 4-d
  int64_t batch, tokens, heads, d;
  int64_t strides[3];
};
Heads4 heads4(const char* what, const at::Tensor& x, bool packets) {
  if (x.dim() != 4) fail_assert(std::string(what) + " must be [batch, tokens, heads, head_dim], got " + shape_str(x.sizes()));
  Heads4 r{x, x.size(0), x.size(1), x.size(2), x.size(3), {0, 0, 0}};
  bool fits = x.numel() == 0 || x.stride(3) == 1 || r.d == 1;
  if (packets && x.numel() != 0) {
    fits = fits && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; ++i) fits = fits && (x.size(i) == 1 || x.stride(i) % 8 == 0);
  }
  if (!fits) r.t = x.clone(at::MemoryFormat::Contiguous);
  for (int i = 0; i < 3; ++i) r.strides[i] = r.t.size(i) == 1 ? 0 : r.t.stride(i);  // a lone row's stride says nothing
  return r;
}

// The cache's tensors (pools [pages, kv_heads, page_size, head_dim]).
struct Cache {
  at::Tensor table;  // keeps a copy alive
  mi355_kv_cache c;
  at::ScalarType values;  // the dtype of a 16-bit cache
};
Cache cache_of(const at::Tensor& k, const at::Tensor& v, const at::Tensor& table, const OptTensor& k_scale,
               const OptTensor& v_scale) {
  if (!(k.is_cuda() && v.is_cuda() && table.is_cuda())) fail_assert("the cache must be on a ROCm GPU");
  if (k.dim() != 4 || k.sizes() != v.sizes())
    fail_assert("cache.k and cache.v must be [pages, kv_heads, page_size, head_dim], got " + shape_str(k.sizes()) +
                " and " + shape_str(v.sizes()));
  const at::ScalarType t = k.scalar_type();
  if (t != v.scalar_type()) fail_assert("cache dtypes differ: " + dtype_str(t) + " and " + dtype_str(v.scalar_type()));
  int format;
  if (t == at::kHalf || t == at::kBFloat16) format = MI355_KV_16BIT;
  else if (t == at::kChar) format = MI355_KV_INT8;
  else if (t == at::kFloat8_e4m3fn) format = MI355_KV_E4M3;
  else fail_assert("cache dtype must be fp16, bf16, int8 or float8_e4m3fn, got " + dtype_str(t));
  if (!(k.is_contiguous() && v.is_contiguous())) fail_assert("cache.k and cache.v must be contiguous");
  if (!(table.dim() == 2 && table.scalar_type() == at::kInt))
    fail_assert("page_table must be int32 [batch, pages], got " + dtype_str(table.scalar_type()) + " " +
                shape_str(table.sizes()));
  const int dev = k.get_device();
  if (v.get_device() != dev || table.get_device() != dev) fail_assert("the cache's tensors must share a device");
  Cache r{table, {}, t};
  if (table.numel() && (table.stride(1) != 1 || (table.size(0) > 1 && table.stride(0) < table.size(1))))
    r.table = table.contiguous();
  const bool quantised = format != MI355_KV_16BIT;
  if (quantised != has(k_scale) || quantised != has(v_scale))
    fail_assert(quantised ? "a quantised cache needs k_scale and v_scale" : "a 16-bit cache has no scales");
  if (quantised) {
    for (const OptTensor* s : {&k_scale, &v_scale}) {
      const at::Tensor& x = **s;
      if (!(x.is_cuda() && x.get_device() == dev && x.scalar_type() == at::kFloat && x.is_contiguous() &&
            x.sizes() == k.sizes().slice(0, 3)))
        fail_assert("the cache's scales must be contiguous float32 " + shape_str(k.sizes().slice(0, 3)) +
                    " on its device, got " + dtype_str(x.scalar_type()) + " " + shape_str(x.sizes()));
    }
  }
  r.c.k = ptr(k);
  r.c.v = ptr(v);
  r.c.k_scale = quantised ? static_cast<float*>(ptr(*k_scale)) : nullptr;
  r.c.v_scale = quantised ? static_cast<float*>(ptr(*v_scale)) : nullptr;
  r.c.page_table = static_cast<const int32_t*>(ptr(r.table));
  r.c.table_width = r.table.size(1);
  r.c.table_stride = r.table.size(0) > 1 ? r.table.stride(0) : r.table.size(1);
  r.c.pages = k.size(0);
  r.c.kv_heads = k.size(1);
  r.c.page_size = k.size(2);
  r.c.head_dim = k.size(3);
  r.c.format = format;
  return r;
}

// int32 [batch] on the cache's device, contiguous (copied if need be).
at::Tensor lengths(const char* what, const at::Tensor& t, int64_t batch, int dev) {
  if (!(t.is_cuda() && t.get_device() == dev && t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == batch))
    fail_assert(std::string(what) + " must be int32 (" + std::to_string(batch) + ",) on the cache's device, got " +
                dtype_str(t.scalar_type()) + " " + shape_str(t.sizes()));
  return t.contiguous();
}
const int32_t* ints(const at::Tensor& t) { return t.defined() ? static_cast<const int32_t*>(ptr(t)) : nullptr; }

// positions (int64, or int32 widened) broadcast to [batch, tokens].
at::Tensor positions_of(const at::Tensor& p, int64_t batch, int64_t tokens, int dev) {
  if (!(p.is_cuda() && p.get_device() == dev && (p.scalar_type() == at::kLong || p.scalar_type() == at::kInt)))
    fail_assert("positions must be an int64 or int32 tensor on x's device, got " + dtype_str(p.scalar_type()));
  const bool fits = p.dim() <= 2 && (p.dim() < 1 || p.size(-1) == tokens || p.size(-1) == 1) &&
                    (p.dim() < 2 || p.size(0) == batch || p.size(0) == 1);
  if (!fits)
    fail_assert("positions " + shape_str(p.sizes()) + " do not broadcast to (" + std::to_string(batch) + ", " +
                std::to_string(tokens) + ")");
  return (p.scalar_type() == at::kLong ? p : p.to(at::kLong)).expand({batch, tokens});
}
at::Tensor frequencies(const at::Tensor& f, int64_t d, int dev) {
  if (!(f.is_cuda() && f.get_device() == dev && f.scalar_type() == at::kFloat && f.dim() == 1))
    fail_assert("inv_freq must be a 1-d float32 tensor on x's device, got " + dtype_str(f.scalar_type()) + " " +
                shape_str(f.sizes()));
  if (2 * f.size(0) > d)
    fail_assert("inv_freq has " + std::to_string(f.size(0)) + " pairs, more than head_dim " + std::to_string(d) + " holds");
  return f.contiguous();
}

at::Tensor rotary(const at::Tensor& x, const at::Tensor& positions, const at::Tensor& inv_freq, double scale,
                  bool interleaved) {
  if (!x.is_cuda()) fail_assert("x must be a ROCm GPU tensor");
  const int code = code_of(x.scalar_type());
  if (code < 0) fail_assert("unsupported dtype x=" + dtype_str(x.scalar_type()) + " (fp16, bf16, fp32)");
  const Heads4 h = heads4("x", x, false);
  const int dev = x.get_device();
  const at::Tensor p = positions_of(positions, h.batch, h.tokens, dev), f = frequencies(inv_freq, h.d, dev);
  at::Tensor out = at::empty(x.sizes(), x.options());
  if (out.numel()) {
    Launch l(dev);
    check("mi355_rotary_fwd",
          mi355_rotary_fwd(ptr(h.t), ptr(out), static_cast<const int64_t*>(ptr(p)), static_cast<const float*>(ptr(f)),
                           h.batch, h.tokens, h.heads, h.d, 2 * f.size(0), h.strides[0], h.strides[1], h.strides[2],
                           p.stride(0), p.stride(1), static_cast<float>(scale), interleaved, code, l.stream));
  }
  return out;
}

int check_new(const char* what, const at::Tensor& x, const Cache& cache, int dev) {
  if (!(x.is_cuda() && x.get_device() == dev)) fail_assert(std::string(what) + " must be on the cache's GPU");
  if (x.scalar_type() != at::kHalf && x.scalar_type() != at::kBFloat16)
    fail_assert(std::string(what) + " must be fp16 or bf16, got " + dtype_str(x.scalar_type()));
  if (cache.c.format == MI355_KV_16BIT && x.scalar_type() != cache.values)
    fail_assert(std::string(what) + " is " + dtype_str(x.scalar_type()) + ", the cache " + dtype_str(cache.values));
  return code_of(x.scalar_type());
}

OptTensor kv_append(const at::Tensor& ck, const at::Tensor& cv, const at::Tensor& table, const OptTensor& ks,
                    const OptTensor& vs, const at::Tensor& k, const at::Tensor& v, const at::Tensor& seq_lens,
                    const OptTensor& new_lens, const OptTensor& q, const OptTensor& positions,
                    const OptTensor& inv_freq, double scale, bool interleaved) {
  const Cache cache = cache_of(ck, cv, table, ks, vs);
  const int dev = ck.get_device();
  const int code = check_new("k", k, cache, dev);
  if (k.sizes() != v.sizes()) fail_assert("k and v differ: " + shape_str(k.sizes()) + " vs " + shape_str(v.sizes()));
  if (check_new("v", v, cache, dev) != code) fail_assert("k and v must share a dtype");
  const Heads4 kh = heads4("k", k, true), vh = heads4("v", v, true);
  if (kh.heads != cache.c.kv_heads || kh.d != cache.c.head_dim)
    fail_assert("k has " + std::to_string(kh.heads) + " heads of " + std::to_string(kh.d) + ", the cache " +
                std::to_string(cache.c.kv_heads) + " of " + std::to_string(cache.c.head_dim));
  if (table.size(0) != kh.batch)
    fail_assert("page_table has " + std::to_string(table.size(0)) + " sequences, k " + std::to_string(kh.batch));
  if (has(positions) != has(inv_freq)) fail_assert("positions and inv_freq go together");
  if (has(q) && !has(inv_freq)) fail_assert("q is given to be rotated: positions and inv_freq are missing");
  Heads4 qh{};
  at::Tensor out;
  if (has(q)) {
    if (check_new("q", *q, cache, dev) != code) fail_assert("q, k and v must share a dtype");
    qh = heads4("q", *q, true);
    if (qh.batch != kh.batch || qh.tokens != kh.tokens || qh.d != kh.d)
      fail_assert("q " + shape_str(q->sizes()) + " does not fit k " + shape_str(k.sizes()));
    out = at::empty(q->sizes(), q->options());
  }
  const at::Tensor lens = lengths("seq_lens", seq_lens, kh.batch, dev);
  const at::Tensor fresh = has(new_lens) ? lengths("new_lens", *new_lens, kh.batch, dev) : at::Tensor();
  at::Tensor p, f;
  if (has(inv_freq)) {
    p = positions_of(*positions, kh.batch, kh.tokens, dev);
    f = frequencies(*inv_freq, kh.d, dev);
  }
  if (kh.batch && kh.tokens) {
    const int64_t strides[9] = {kh.strides[0], kh.strides[1], kh.strides[2], vh.strides[0], vh.strides[1],
                                vh.strides[2], qh.strides[0], qh.strides[1], qh.strides[2]};
    Launch l(dev);
    check("mi355_kv_cache_append_fwd",
          mi355_kv_cache_append_fwd(&cache.c, ptr(kh.t), ptr(vh.t), has(q) ? ptr(qh.t) : nullptr,
                                    has(q) ? ptr(out) : nullptr, ints(lens), ints(fresh),
                                    p.defined() ? static_cast<const int64_t*>(ptr(p)) : nullptr,
                                    f.defined() ? static_cast<const float*>(ptr(f)) : nullptr, kh.batch, kh.tokens,
                                    qh.heads, f.defined() ? 2 * f.size(0) : 0, strides,
                                    p.defined() ? p.stride(0) : 0, p.defined() ? p.stride(1) : 0,
                                    static_cast<float>(scale), interleaved, code, l.stream));
  }
  if (!has(q)) return c10::nullopt;
  return out;
}

std::tuple<at::Tensor, at::Tensor> kv_read(const at::Tensor& ck, const at::Tensor& cv, const at::Tensor& table,
                                           const OptTensor& ks, const OptTensor& vs, const at::Tensor& end,
                                           int64_t tokens, const OptTensor& start, at::ScalarType dtype) {
  const Cache cache = cache_of(ck, cv, table, ks, vs);
  const int dev = ck.get_device();
  if (dtype != at::kHalf && dtype != at::kBFloat16) fail_assert("dtype must be fp16 or bf16, got " + dtype_str(dtype));
  if (cache.c.format == MI355_KV_16BIT && dtype != cache.values)
    fail_assert("dtype is " + dtype_str(dtype) + ", the cache " + dtype_str(cache.values));
  if (tokens < 0) fail_assert("tokens must be >= 0");
  const int64_t batch = table.size(0);
  const at::Tensor e = lengths("end", end, batch, dev);
  const at::Tensor s = has(start) ? lengths("start", *start, batch, dev) : at::Tensor();
  const auto options = ck.options().dtype(dtype);
  at::Tensor k = at::empty({batch, cache.c.kv_heads, tokens, cache.c.head_dim}, options);
  at::Tensor v = at::empty(k.sizes(), options);
  if (batch && tokens) {
    Launch l(dev);
    check("mi355_kv_cache_read_fwd", mi355_kv_cache_read_fwd(&cache.c, ptr(k), ptr(v), ints(s), ints(e), batch, tokens,
                                                             code_of(dtype), l.stream));
  }
  return {k, v};
}

void kv_keep(const at::Tensor& ck, const at::Tensor& cv, const at::Tensor& table, const OptTensor& ks,
             const OptTensor& vs, const at::Tensor& seq_lens, const at::Tensor& kept, const OptTensor& kept_lens) {
  const Cache cache = cache_of(ck, cv, table, ks, vs);
  const int dev = ck.get_device();
  const int64_t batch = table.size(0);
  if (!(kept.is_cuda() && kept.get_device() == dev && kept.scalar_type() == at::kInt && kept.dim() == 2 &&
        kept.size(0) == batch))
    fail_assert("kept must be int32 [" + std::to_string(batch) + ", n] on the cache's device, got " +
                dtype_str(kept.scalar_type()) + " " + shape_str(kept.sizes()));
  const at::Tensor lens = lengths("seq_lens", seq_lens, batch, dev);
  const at::Tensor n = has(kept_lens) ? lengths("kept_lens", *kept_lens, batch, dev) : at::Tensor();
  const at::Tensor kc = kept.contiguous();
  if (batch && kept.size(1)) {
    Launch l(dev);
    check("mi355_kv_cache_keep_fwd", mi355_kv_cache_keep_fwd(&cache.c, ints(lens), ints(kc), ints(n), batch,
                                                             kc.size(1), kc.size(1), l.stream));
  }
}

at::Tensor tree_attention(const at::Tensor& q, const at::Tensor& ck, const at::Tensor& cv, const at::Tensor& table,
                          const OptTensor& ks, const OptTensor& vs, const at::Tensor& seq_lens,
                          const OptTensor& new_lens, const OptTensor& tree_mask, double scale) {
  const Cache cache = cache_of(ck, cv, table, ks, vs);
  const int dev = ck.get_device();
  const int code = check_new("q", q, cache, dev);
  const Heads4 h = heads4("q", q, true);
  if (h.d != cache.c.head_dim || h.heads % std::max<int64_t>(1, cache.c.kv_heads) != 0)
    fail_assert("q has " + std::to_string(h.heads) + " heads of " + std::to_string(h.d) + ", the cache " +
                std::to_string(cache.c.kv_heads) + " of " + std::to_string(cache.c.head_dim));
  if (table.size(0) != h.batch)
    fail_assert("page_table has " + std::to_string(table.size(0)) + " sequences, q " + std::to_string(h.batch));
  const at::Tensor lens = lengths("seq_lens", seq_lens, h.batch, dev);
  const at::Tensor fresh = has(new_lens) ? lengths("new_lens", *new_lens, h.batch, dev) : at::Tensor();
  at::Tensor mask;
  if (has(tree_mask)) {
    mask = *tree_mask;
    const bool fits = (mask.dim() == 2 || (mask.dim() == 3 && (mask.size(0) == h.batch || mask.size(0) == 1))) &&
                      mask.size(-1) == h.tokens && mask.size(-2) == h.tokens;
    if (!(mask.is_cuda() && mask.get_device() == dev && mask.scalar_type() == at::kBool && fits))
      fail_assert("tree_mask must be bool [tokens, tokens] or [batch, tokens, tokens] on q's device, got " +
                  dtype_str(mask.scalar_type()) + " " + shape_str(mask.sizes()));
    if (mask.dim() == 2) mask = mask.unsqueeze(0);
    if (mask.numel() && mask.stride(2) != 1 && mask.size(2) != 1) mask = mask.contiguous();
  }
  at::Tensor out = at::empty(q.sizes(), q.options());
  if (out.numel()) {
    Launch l(dev);
    const at::Tensor work = workspace(mi355_tree_attention_workspace(&cache.c, h.batch, h.tokens, h.heads), q);
    check("mi355_tree_attention_fwd",
          mi355_tree_attention_fwd(&cache.c, ptr(h.t), ptr(out), ints(lens), ints(fresh),
                                   mask.defined() ? static_cast<const uint8_t*>(ptr(mask)) : nullptr,
                                   mask.defined() && mask.size(0) > 1 ? mask.stride(0) : 0,
                                   mask.defined() && mask.size(1) > 1 ? mask.stride(1) : 0, h.batch, h.tokens, h.heads,
                                   h.strides, static_cast<float>(scale), code,
                                   work.defined() ? ptr(work) : nullptr, work.defined() ? work.numel() : 0, l.stream));
  }
  return out;
}

}  // namespace

PYBIND11_MODULE(_mi355_torch, m) {
  m.doc() = "Host-side launchers of the MI355X fused kernels (torch tensors -> the C ABI of libmi355_fused.so)";
  m.def("set_kernel_error", [](py::object cls) {
    if (g_kernel_error == nullptr) g_kernel_error = new py::object(cls);
    else *g_kernel_error = cls;
  });
  m.def("abi_version", []() { return mi355_abi_version(); });
  m.def("rmsnorm", &rmsnorm, py::arg("x"), py::arg("weight"), py::arg("eps"));
  m.def("add_rmsnorm", &add_rmsnorm, py::arg("x"), py::arg("residual"), py::arg("weight"), py::arg("eps"));
  m.def("silu_mul", &silu_mul, py::arg("gate"), py::arg("up"));
  m.def("gate_up_silu", &gate_up_silu, py::arg("x"), py::arg("w_gate"), py::arg("w_up"), py::arg("out_f32"));
  m.def("linear16", &linear16, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("out_f32"));
  m.def("w8a16_linear", &w8a16_linear, py::arg("x"), py::arg("w_q"), py::arg("scale"), py::arg("bias"),
        py::arg("out_f32"));
  m.def("gate_up_silu_w8a16", &gate_up_silu_w8a16, py::arg("x"), py::arg("wq_gate"), py::arg("scale_gate"),
        py::arg("wq_up"), py::arg("scale_up"), py::arg("out_f32"));
  m.def("rotary", &rotary, py::arg("x"), py::arg("positions"), py::arg("inv_freq"), py::arg("scale"),
        py::arg("interleaved"));
  m.def("kv_append", &kv_append, py::arg("cache_k"), py::arg("cache_v"), py::arg("page_table"), py::arg("k_scale"),
        py::arg("v_scale"), py::arg("k"), py::arg("v"), py::arg("seq_lens"), py::arg("new_lens"), py::arg("q"),
        py::arg("positions"), py::arg("inv_freq"), py::arg("scale"), py::arg("interleaved"));
  m.def("kv_read", &kv_read, py::arg("cache_k"), py::arg("cache_v"), py::arg("page_table"), py::arg("k_scale"),
        py::arg("v_scale"), py::arg("end"), py::arg("tokens"), py::arg("start"), py::arg("dtype"));
  m.def("kv_keep", &kv_keep, py::arg("cache_k"), py::arg("cache_v"), py::arg("page_table"), py::arg("k_scale"),
        py::arg("v_scale"), py::arg("seq_lens"), py::arg("kept"), py::arg("kept_lens"));
  m.def("tree_attention", &tree_attention, py::arg("q"), py::arg("cache_k"), py::arg("cache_v"),
        py::arg("page_table"), py::arg("k_scale"), py::arg("v_scale"), py::arg("seq_lens"), py::arg("new_lens"),
        py::arg("tree_mask"), py::arg("scale"));
}
