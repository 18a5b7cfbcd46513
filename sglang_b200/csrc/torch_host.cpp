// Native host path of the torch-facing functions (module sglang_b200._host).
//
// A decode-size linear is 10-20 us of device work; the Python-level sequence in front of it (argument checks, one
// torch.empty per intermediate, a ctypes call with a dozen arguments per kernel) took 60-80 us, a fused expert layer
// 240 us.  Each function here does the allocation and the C-ABI call(s) of one public function in one native call.
//
// Every function looks at its arguments first and returns None when they are not the plain case (CPU or non-contiguous
// tensors, another dtype, a size its caller would reject): the Python function then runs its own checks, which raise
// what they always raised.  Nothing is launched in that case.
//
// The functions from head_rows on have no Python twin: they check everything themselves and raise RuntimeError, shapes, types
// and strides before devices, so that a call on CPU tensors is refused for what is wrong with it first.
#include <Python.h>

#include <ATen/EmptyTensor.h>
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <initializer_list>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/b200_block_fp8.h"

namespace {

using at::Tensor;

int dt_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return B200_DT_F32;
    case at::kHalf: return B200_DT_F16;
    case at::kBFloat16: return B200_DT_BF16;
    default: return -1;
  }
}
bool is_16bit(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }

// A tensor whose memory this library may use directly: dense CUDA storage, no lazy negation or conjugation.
const Tensor* cuda_tensor(PyObject* o) {
  if (!THPVariable_Check(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.is_neg() || t.is_conj()) return nullptr;
  if (t.unsafeGetTensorImpl()->key_set().has(c10::DispatchKey::Python)) return nullptr;
  return &t;
}
const Tensor* cuda_tensor(PyObject* o, at::ScalarType dtype) {
  const Tensor* t = cuda_tensor(o);
  return t && t->scalar_type() == dtype ? t : nullptr;
}

Tensor empty(at::IntArrayRef sizes, at::ScalarType dtype, const at::Device& dev) {
  return at::detail::empty_cuda(sizes, dtype, dev, std::nullopt);
}
Tensor empty_strided(at::IntArrayRef sizes, at::IntArrayRef strides, at::ScalarType dtype, const at::Device& dev) {
  return at::detail::empty_strided_cuda(sizes, strides, dtype, dev);
}

void* stream_of(const at::Device& dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

PyObject* none() { Py_RETURN_NONE; }

// The interpreter lock is free while this lives.  Allocating may wait for the device and a launch for room in the queue;
// the process's other Python threads go on meanwhile, as they do under a ctypes call.  Everything that is read from a
// Python-owned tensor is read before; tensors held by value are fine.
struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  NoGil() = default;
  NoGil(const NoGil&) = delete;
  NoGil& operator=(const NoGil&) = delete;
  ~NoGil() { PyEval_RestoreThread(state); }
};

// Raises _lib.B200Error(fn, code, detail), the exception the Python functions raise.
PyObject* raise_status(const char* fn, int code) {
  PyObject* mod = PyImport_ImportModule("sglang_b200._lib");
  if (mod) {
    PyObject* r = PyObject_CallMethod(mod, "check", "si", fn, code);
    Py_XDECREF(r);
    Py_DECREF(mod);
    if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s failed (code %d)", fn, code);
  }
  return nullptr;
}

int64_t align4(int64_t v) { return (v + 3) / 4 * 4; }

// Scale tensor of sglang_per_token_group_quant_fp8 for x [..., K] of these sizes seen as [M, K]; `rs` and `gs` are its
// strides.
// Packed words are zero-filled where the quantiser may leave bytes alone (`partial`) or rows are padding.
Tensor scale_tensor(std::vector<int64_t> sizes, int64_t K, int64_t M, int64_t group, bool col_major, bool aligned, bool ue8m0,
                    bool partial, const at::Device& dev, int64_t& rs, int64_t& gs) {
  const int64_t G = K / group;
  if (ue8m0) {
    const int64_t W = (G + 3) / 4, ld = align4(M);
    rs = 1;
    gs = ld;
    Tensor whole = empty({W, ld}, at::kInt, dev);
    if (ld != M || (partial && G % 4 != 0))
      C10_CUDA_CHECK(cudaMemsetAsync(whole.data_ptr(), 0, W * ld * 4, static_cast<cudaStream_t>(stream_of(dev))));
    return whole.transpose(0, 1).narrow(0, 0, M);
  }
  if (col_major) {      // 2-D only (checked by the callers)
    const int64_t ld = aligned ? align4(M) : M;
    rs = 1;
    gs = ld;
    if (ld == M) return empty_strided({M, G}, {1, M}, at::kFloat, dev);
    return empty({G, ld}, at::kFloat, dev).transpose(0, 1).narrow(0, 0, M);
  }
  rs = G;
  gs = 1;
  sizes.back() = G;
  return empty(sizes, at::kFloat, dev);
}

PyObject* pair_of(Tensor a, Tensor b) {
  PyObject* pa = THPVariable_Wrap(std::move(a));
  PyObject* pb = THPVariable_Wrap(std::move(b));
  PyObject* r = PyTuple_Pack(2, pa, pb);
  Py_DECREF(pa);
  Py_DECREF(pb);
  return r;
}

#define HOST_FN(name) PyObject* name(PyObject*, PyObject* const* a, Py_ssize_t n) try
#define HOST_END                                        \
  catch (const std::exception& e) {                     \
    PyErr_SetString(PyExc_RuntimeError, e.what());      \
    return nullptr;                                     \
  }

// linear(x, weight, weight_scale, bias | None, out | None, scale_mode)
//   scale_mode 0: fp32 scales; 1: power-of-two activation scales; 2: power-of-two weight scales as well
HOST_FN(linear) {
  if (n != 6) return none();
  const Tensor *x = cuda_tensor(a[0]), *w = cuda_tensor(a[1], at::kFloat8_e4m3fn), *ws = cuda_tensor(a[2], at::kFloat);
  if (!x || !w || !ws || !is_16bit(x->scalar_type()) || x->dim() < 1 || w->dim() != 2 || ws->dim() != 2) return none();
  const int64_t K = w->size(1), N = w->size(0);
  long mode = PyLong_AsLong(a[5]);
  if (K <= 0 || N <= 0 || x->size(-1) != K || K % 128 != 0 || !x->is_contiguous() || !w->is_contiguous()) return none();
  if (ws->size(0) != (N + 127) / 128 || ws->size(1) != K / 128) return none();
  if (N % 128 == 0 && ws->stride(1) != 1) return none();
  if (N % 8 != 0 || w->device() != x->device() || ws->device() != x->device()) return none();
  if (mode != 0 && (x->scalar_type() != at::kBFloat16 || N % 128 != 0)) return none();
  const int64_t M = x->numel() / K;
  if (M == 0) return none();
  const Tensor* bias = nullptr;
  if (a[3] != Py_None) {
    bias = cuda_tensor(a[3], x->scalar_type());
    if (!bias || bias->dim() != 1 || bias->size(0) != N || !bias->is_contiguous() || bias->device() != x->device())
      return none();
  }
  const at::Device dev = x->device();
  const at::ScalarType xt = x->scalar_type();
  Tensor out;
  int64_t ldo = N;
  auto out_sizes = x->sizes().vec();
  out_sizes.back() = N;
  if (a[4] != Py_None) {
    const Tensor* o = cuda_tensor(a[4], xt);
    if (!o || o->dim() != 2 || o->size(0) != M || o->size(1) != N || o->stride(1) != 1 || o->stride(0) < N ||
        o->device() != dev || x->dim() != 2)
      return none();
    ldo = o->stride(0);
    out = *o;
  }
  const void *xp = x->data_ptr(), *wp = w->data_ptr(), *bp = bias ? bias->data_ptr() : nullptr;
  const float* wsp = static_cast<const float*>(ws->data_ptr());
  const int64_t ws_n = ws->stride(0), ws_g = ws->stride(1);
  int rc;
  {
    const NoGil no_gil;
    const c10::cuda::OptionalCUDAGuard guard(dev);
    if (!out.defined()) out = empty(out_sizes, xt, dev);
    const size_t bytes = b200_fp8_linear_workspace_bytes(M, N, K, static_cast<int>(mode));
    const Tensor work = empty({static_cast<int64_t>(bytes)}, at::kByte, dev);
    rc = b200_fp8_linear(xp, dt_of(xt), wp, K, wsp, ws_n, ws_g, bp, out.data_ptr(), ldo, M, N, K, static_cast<int>(mode),
                         work.data_ptr(), bytes, stream_of(dev));
  }
  if (rc != 0) return raise_status("fp8_linear", rc);
  return THPVariable_Wrap(std::move(out));
}
HOST_END

// quant(x, group_size, eps, column_major, aligned, ue8m0) -> (codes, scales)
HOST_FN(quant) {
  if (n != 6) return none();
  const Tensor* x = cuda_tensor(a[0]);
  if (!x || x->dim() < 1 || !x->is_contiguous() || x->numel() == 0) return none();
  const int dt = dt_of(x->scalar_type());
  const int64_t group = PyLong_AsLong(a[1]), K = x->size(-1);
  if (dt < 0 || (group != 64 && group != 128 && group != 256 && group != 512) || K % group != 0) return none();
  const double eps = PyFloat_AsDouble(a[2]);
  const bool col = PyObject_IsTrue(a[3]), aligned = PyObject_IsTrue(a[4]), ue8m0 = PyObject_IsTrue(a[5]);
  if (PyErr_Occurred()) return nullptr;
  if ((col || ue8m0) && x->dim() != 2) return none();
  if (ue8m0 && !(col && aligned && group == 128)) return none();
  const at::Device dev = x->device();
  const int64_t M = x->numel() / K;
  const auto sizes = x->sizes().vec();
  const void* xp = x->data_ptr();
  Tensor q, s;
  int rc;
  {
    const NoGil no_gil;
    const c10::cuda::OptionalCUDAGuard guard(dev);
    q = empty(sizes, at::kFloat8_e4m3fn, dev);
    int64_t rs, gs;
    s = scale_tensor(sizes, K, M, group, col, aligned, ue8m0, false, dev, rs, gs);
    void* st = stream_of(dev);
    rc = ue8m0 ? b200_per_token_group_quant_fp8_ue8m0(xp, dt, q.data_ptr(), static_cast<uint32_t*>(s.data_ptr()), M, K, gs,
                                                      static_cast<float>(eps), -448.0f, 448.0f, st)
               : b200_per_token_group_quant_fp8(xp, dt, q.data_ptr(), static_cast<float*>(s.data_ptr()), M, K, group, rs, gs,
                                                static_cast<float>(eps), -448.0f, 448.0f, st);
  }
  if (rc != 0) return raise_status("sgl_per_token_group_quant_fp8", rc);
  return pair_of(std::move(q), std::move(s));
}
HOST_END

// norm_quant(x, weight, norm_eps, residual | None, eps, column_major, aligned, ue8m0) -> (codes, scales)
HOST_FN(norm_quant) {
  if (n != 8) return none();
  const Tensor* x = cuda_tensor(a[0]);
  if (!x || !is_16bit(x->scalar_type()) || x->dim() < 1 || !x->is_contiguous() || x->numel() == 0) return none();
  const Tensor* w = cuda_tensor(a[1], x->scalar_type());
  const int64_t K = x->size(-1), M = x->numel() / K;
  if (!w || w->dim() != 1 || w->size(0) != K || !w->is_contiguous() || K % 128 != 0 || K > 16384) return none();
  const double norm_eps = PyFloat_AsDouble(a[2]), eps = PyFloat_AsDouble(a[4]);
  const Tensor* r = nullptr;
  if (a[3] != Py_None) {
    r = cuda_tensor(a[3], x->scalar_type());
    if (!r || r->sizes() != x->sizes() || !r->is_contiguous() || r->device() != x->device()) return none();
  }
  const bool col = PyObject_IsTrue(a[5]), aligned = PyObject_IsTrue(a[6]), ue8m0 = PyObject_IsTrue(a[7]);
  if (PyErr_Occurred()) return nullptr;
  if (x->dim() != 2 || (ue8m0 && !(col && aligned)) || w->device() != x->device()) return none();
  const at::Device dev = x->device();
  const auto sizes = x->sizes().vec();
  const int dt = dt_of(x->scalar_type());
  const void *xp = x->data_ptr(), *wp = w->data_ptr();
  void* rp = r ? r->data_ptr() : nullptr;
  Tensor q, s;
  int rc;
  {
    const NoGil no_gil;
    const c10::cuda::OptionalCUDAGuard guard(dev);
    q = empty(sizes, at::kFloat8_e4m3fn, dev);
    int64_t rs, gs;
    s = scale_tensor(sizes, K, M, 128, col, aligned, ue8m0, true, dev, rs, gs);
    rc = b200_rmsnorm_per_token_group_quant_fp8(xp, dt, rp, wp, static_cast<float>(norm_eps), nullptr, q.data_ptr(),
                                                s.data_ptr(), M, K, rs, gs, ue8m0 ? 1 : 0, static_cast<float>(eps), -448.0f,
                                                448.0f, stream_of(dev));
  }
  if (rc != 0) return raise_status("rmsnorm_per_token_group_quant_fp8", rc);
  return pair_of(std::move(q), std::move(s));
}
HOST_END

// silu_and_mul(x) -> out
HOST_FN(silu_and_mul) {
  if (n != 1) return none();
  const Tensor* x = cuda_tensor(a[0]);
  if (!x || !is_16bit(x->scalar_type()) || x->dim() < 1 || !x->is_contiguous() || x->numel() == 0) return none();
  const int64_t d2 = x->size(-1), d = d2 / 2;
  if (d2 % 16 != 0) return none();
  const at::Device dev = x->device();
  const at::ScalarType xt = x->scalar_type();
  auto sizes = x->sizes().vec();
  sizes.back() = d;
  const int64_t rows = x->numel() / d2;
  const void* xp = x->data_ptr();
  Tensor out;
  int rc;
  {
    const NoGil no_gil;
    const c10::cuda::OptionalCUDAGuard guard(dev);
    out = empty(sizes, xt, dev);
    rc = b200_silu_and_mul(xp, out.data_ptr(), rows, d, dt_of(xt), stream_of(dev));
  }
  if (rc != 0) return raise_status("silu_and_mul", rc);
  return THPVariable_Wrap(std::move(out));
}
HOST_END

// matmul(a [M, K], b [N, K], a_scale [M, K/128], b_scale [N/128, K/128], out_dtype) -> [M, N]: fp32 scales, any strides
HOST_FN(matmul) {
  if (n != 5) return none();
  const Tensor *x = cuda_tensor(a[0], at::kFloat8_e4m3fn), *w = cuda_tensor(a[1], at::kFloat8_e4m3fn),
               *xs = cuda_tensor(a[2], at::kFloat), *ws = cuda_tensor(a[3], at::kFloat);
  if (!x || !w || !xs || !ws || !THPDtype_Check(a[4])) return none();
  if (x->dim() != 2 || w->dim() != 2 || xs->dim() != 2 || ws->dim() != 2 || !x->is_contiguous() || !w->is_contiguous())
    return none();
  const at::ScalarType ot = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
  const int64_t M = x->size(0), K = x->size(1), N = w->size(0);
  if (dt_of(ot) < 0 || M == 0 || N == 0 || w->size(1) != K || K % 128 != 0 || N % 8 != 0) return none();
  if (xs->size(0) != M || xs->size(1) != K / 128 || ws->size(0) != (N + 127) / 128 || ws->size(1) != K / 128) return none();
  const at::Device dev = x->device();
  if (w->device() != dev || xs->device() != dev || ws->device() != dev) return none();
  const void *xp = x->data_ptr(), *wp = w->data_ptr();
  const float *xsp = static_cast<const float*>(xs->data_ptr()), *wsp = static_cast<const float*>(ws->data_ptr());
  const int64_t xs_m = xs->stride(0), xs_g = xs->stride(1), ws_n = ws->stride(0), ws_g = ws->stride(1);
  Tensor out;
  int rc;
  {
    const NoGil no_gil;
    const c10::cuda::OptionalCUDAGuard guard(dev);
    out = empty({M, N}, ot, dev);
    const size_t bytes = b200_fp8_blockwise_scaled_mm_workspace_bytes(M, N, K);
    Tensor work;
    if (bytes) work = empty({static_cast<int64_t>(bytes)}, at::kByte, dev);
    rc = b200_fp8_blockwise_scaled_mm_splitk(xp, K, wp, K, xsp, xs_m, xs_g, wsp, ws_n, ws_g, out.data_ptr(), N, dt_of(ot), M,
                                             N, K, 0, bytes ? work.data_ptr() : nullptr, bytes, stream_of(dev));
  }
  if (rc != 0) return raise_status("w8a8_block_fp8_matmul", rc);
  return THPVariable_Wrap(std::move(out));
}
HOST_END

// matmul_packed(a [M, K], b [N, K], a_words int32 [M, K/512], b_scale [N/128, K/128], weights_pow2) -> bf16 [M, N]
HOST_FN(matmul_packed) {
  if (n != 5) return none();
  const Tensor *x = cuda_tensor(a[0], at::kFloat8_e4m3fn), *w = cuda_tensor(a[1], at::kFloat8_e4m3fn),
               *xs = cuda_tensor(a[2], at::kInt), *ws = cuda_tensor(a[3], at::kFloat);
  if (!x || !w || !xs || !ws) return none();
  if (x->dim() != 2 || w->dim() != 2 || xs->dim() != 2 || ws->dim() != 2 || !x->is_contiguous() || !w->is_contiguous())
    return none();
  const int64_t M = x->size(0), K = x->size(1), N = w->size(0);
  if (M == 0 || N == 0 || w->size(1) != K || K % 128 != 0 || N % 128 != 0) return none();
  if (xs->size(0) != M || xs->size(1) != (K / 128 + 3) / 4 || (xs->stride(0) != 1 && M != 1)) return none();
  if (ws->size(0) != N / 128 || ws->size(1) != K / 128) return none();
  const at::Device dev = x->device();
  if (w->device() != dev || xs->device() != dev || ws->device() != dev) return none();
  const bool pow2 = PyObject_IsTrue(a[4]);
  const void *xp = x->data_ptr(), *wp = w->data_ptr();
  const uint32_t* xsp = static_cast<const uint32_t*>(xs->data_ptr());
  const float* wsp = static_cast<const float*>(ws->data_ptr());
  const int64_t xs_m = xs->stride(0), xs_g = xs->stride(1), ws_n = ws->stride(0), ws_g = ws->stride(1);
  Tensor out;
  int rc;
  {
    const NoGil no_gil;
    const c10::cuda::OptionalCUDAGuard guard(dev);
    out = empty({M, N}, at::kBFloat16, dev);
    rc = (pow2 ? b200_fp8_blockwise_scaled_mm_pow2 : b200_fp8_blockwise_scaled_mm_ue8m0)(
        xp, K, wp, K, xsp, xs_m, xs_g, wsp, ws_n, ws_g, out.data_ptr(), N, B200_DT_BF16, M, N, K, stream_of(dev));
  }
  if (rc != 0) return raise_status("w8a8_block_fp8_matmul_deepgemm", rc);
  return THPVariable_Wrap(std::move(out));
}
HOST_END

// gate_up_silu_quant(a [M, K], a_words, w [2n, K], w_scale [2n/128, K/128], mid_dtype) -> (codes [M, n], words)
HOST_FN(gate_up_silu_quant) {
  if (n != 5) return none();
  const Tensor *x = cuda_tensor(a[0], at::kFloat8_e4m3fn), *xs = cuda_tensor(a[1], at::kInt),
               *w = cuda_tensor(a[2], at::kFloat8_e4m3fn), *ws = cuda_tensor(a[3], at::kFloat);
  if (!x || !w || !xs || !ws || !THPDtype_Check(a[4])) return none();
  const at::ScalarType mid = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
  if (!is_16bit(mid) || x->dim() != 2 || w->dim() != 2 || xs->dim() != 2 || ws->dim() != 2 || !x->is_contiguous() ||
      !w->is_contiguous())
    return none();
  const int64_t M = x->size(0), K = x->size(1), n2 = w->size(0), N = n2 / 2;
  if (M == 0 || w->size(1) != K || K % 128 != 0 || n2 % 256 != 0 || n2 == 0) return none();
  if (xs->size(0) != M || xs->size(1) < (K / 128 + 3) / 4 || ws->size(0) != n2 / 128 || ws->size(1) != K / 128) return none();
  const at::Device dev = x->device();
  if (w->device() != dev || xs->device() != dev || ws->device() != dev) return none();
  const auto sizes = x->sizes().vec();
  const void *xp = x->data_ptr(), *wp = w->data_ptr();
  const uint32_t* xsp = static_cast<const uint32_t*>(xs->data_ptr());
  const float* wsp = static_cast<const float*>(ws->data_ptr());
  const int64_t xs_m = xs->stride(0), xs_g = xs->stride(1), ws_n = ws->stride(0), ws_g = ws->stride(1);
  Tensor q, s;
  int rc;
  {
    const NoGil no_gil;
    const c10::cuda::OptionalCUDAGuard guard(dev);
    q = empty({M, N}, at::kFloat8_e4m3fn, dev);
    int64_t rs, gs;
    s = scale_tensor(sizes, N, M, 128, true, true, true, true, dev, rs, gs);
    rc = b200_fp8_gate_up_silu_quant_pow2(xp, K, wp, K, xsp, xs_m, xs_g, wsp, ws_n, ws_g, q.data_ptr(), N,
                                          static_cast<uint32_t*>(s.data_ptr()), gs, dt_of(mid), M, N, K, stream_of(dev));
  }
  if (rc != 0) return raise_status("gate_up_silu_quant_pow2", rc);
  return pair_of(std::move(q), std::move(s));
}
HOST_END

// topk_softmax(logits [m, E], topk, renormalize) -> (weights fp32 [m, topk], ids int32 [m, topk])
HOST_FN(topk_softmax) {
  if (n != 3) return none();
  const Tensor* x = cuda_tensor(a[0]);
  if (!x || x->dim() != 2 || dt_of(x->scalar_type()) < 0 || x->stride(1) != 1) return none();
  const int64_t m = x->size(0), E = x->size(1), topk = PyLong_AsLong(a[1]);
  if (m == 0 || topk <= 0 || topk > E || topk > 32 || E > 1024 || x->stride(0) < E) return none();
  const at::Device dev = x->device();
  const int dt = dt_of(x->scalar_type()), renormalize = PyObject_IsTrue(a[2]) ? 1 : 0;
  const int64_t ld = x->stride(0);
  const void* xp = x->data_ptr();
  Tensor w, ids;
  int rc;
  {
    const NoGil no_gil;
    const c10::cuda::OptionalCUDAGuard guard(dev);
    w = empty({m, topk}, at::kFloat, dev);
    ids = empty({m, topk}, at::kInt, dev);
    rc = b200_topk_softmax(xp, dt, ld, static_cast<float*>(w.data_ptr()), static_cast<int32_t*>(ids.data_ptr()), m,
                           static_cast<int>(E), static_cast<int>(topk), renormalize, stream_of(dev));
  }
  if (rc != 0) return raise_status("topk_softmax", rc);
  return pair_of(std::move(w), std::move(ids));
}
HOST_END

// fused_gate(logits, bias, num_expert_group, topk_group, topk, num_fused_shared_experts, routed_scaling_factor)
HOST_FN(fused_gate) {
  if (n != 7) return none();
  const Tensor *x = cuda_tensor(a[0], at::kFloat), *b = cuda_tensor(a[1], at::kFloat);
  if (!x || !b || x->dim() != 2 || b->dim() != 1 || b->numel() != x->size(1) || x->stride(1) != 1 || !b->is_contiguous())
    return none();
  const int64_t m = x->size(0), E = x->size(1);
  const long groups = PyLong_AsLong(a[2]), tg = PyLong_AsLong(a[3]), topk = PyLong_AsLong(a[4]), shared = PyLong_AsLong(a[5]);
  const double factor = PyFloat_AsDouble(a[6]);
  if (PyErr_Occurred()) return nullptr;
  if (m == 0 || b->device() != x->device() || groups <= 0 || groups > 32 || E % groups != 0 || E / groups < 2 || E > 1024)
    return none();
  if (tg <= 0 || tg > groups || topk > 32 || shared < 0 || topk - shared <= 0 || topk - shared > tg * (E / groups) ||
      (shared > 0 && factor == 0.0) || x->stride(0) < E)
    return none();
  const at::Device dev = x->device();
  const int64_t ld = x->stride(0);
  const float *xp = static_cast<const float*>(x->data_ptr()), *bp = static_cast<const float*>(b->data_ptr());
  Tensor w, ids;
  int rc;
  {
    const NoGil no_gil;
    const c10::cuda::OptionalCUDAGuard guard(dev);
    w = empty({m, topk}, at::kFloat, dev);
    ids = empty({m, topk}, at::kInt, dev);
    rc = b200_moe_fused_gate_shared_experts(xp, ld, bp, static_cast<float*>(w.data_ptr()),
                                            static_cast<int32_t*>(ids.data_ptr()), m, static_cast<int>(E),
                                            static_cast<int>(groups), static_cast<int>(tg), static_cast<int>(topk),
                                            static_cast<int>(shared), shared ? factor : 1.0, stream_of(dev));
  }
  if (rc != 0) return raise_status("moe_fused_gate", rc);
  return pair_of(std::move(w), std::move(ids));
}
HOST_END

// experts(x [m, k], w13 [E, 2n, k], w2 [E, k, n], w13_scale, w2_scale, topk_weights, topk_ids, expert_offsets | None,
//         problem_sizes1 | None, problem_sizes2 | None, ue8m0) -> [m, k]
HOST_FN(experts) {
  if (n != 11) return none();
  const Tensor *x = cuda_tensor(a[0]), *w13 = cuda_tensor(a[1], at::kFloat8_e4m3fn), *w2 = cuda_tensor(a[2], at::kFloat8_e4m3fn),
               *s13 = cuda_tensor(a[3], at::kFloat), *s2 = cuda_tensor(a[4], at::kFloat), *tw = cuda_tensor(a[5], at::kFloat),
               *ti = cuda_tensor(a[6], at::kInt);
  if (!x || !w13 || !w2 || !s13 || !s2 || !tw || !ti || !is_16bit(x->scalar_type())) return none();
  if (x->dim() != 2 || w13->dim() != 3 || w2->dim() != 3 || s13->dim() != 3 || s2->dim() != 3 || tw->dim() != 2 || ti->dim() != 2)
    return none();
  const at::Device dev = x->device();
  for (const Tensor* t : {x, w13, w2, s13, s2, tw, ti})
    if (!t->is_contiguous() || t->device() != dev) return none();
  const int64_t m = x->size(0), k = x->size(1), E = w13->size(0), N = w2->size(2), topk = ti->size(1);
  if (m == 0 || E == 0 || topk == 0 || N == 0 || k == 0 || N % 128 != 0 || k % 128 != 0) return none();
  if (w13->size(1) != 2 * N || w13->size(2) != k || w2->size(0) != E || w2->size(1) != k || ti->size(0) != m ||
      tw->sizes() != ti->sizes())
    return none();
  if (s13->size(0) != E || s13->size(1) != 2 * N / 128 || s13->size(2) != k / 128 || s2->size(0) != E ||
      s2->size(1) != k / 128 || s2->size(2) != N / 128)
    return none();
  int32_t* tables[3] = {nullptr, nullptr, nullptr};
  for (int i = 0; i < 3; ++i) {
    if (a[7 + i] == Py_None) continue;
    const Tensor* t = cuda_tensor(a[7 + i], at::kInt);
    if (!t || !t->is_contiguous() || t->device() != dev || t->numel() != (i == 0 ? E + 1 : 3 * E)) return none();
    tables[i] = static_cast<int32_t*>(t->data_ptr());
  }
  const int ue8m0 = PyObject_IsTrue(a[10]) ? 1 : 0;
  const at::ScalarType xt = x->scalar_type();
  const void *xp = x->data_ptr(), *w13p = w13->data_ptr(), *w2p = w2->data_ptr();
  const float *s13p = static_cast<const float*>(s13->data_ptr()), *s2p = static_cast<const float*>(s2->data_ptr()),
              *twp = static_cast<const float*>(tw->data_ptr());
  const int32_t* tip = static_cast<const int32_t*>(ti->data_ptr());
  Tensor out;
  int rc;
  {
    const NoGil no_gil;
    const c10::cuda::OptionalCUDAGuard guard(dev);
    out = empty({m, k}, xt, dev);
    const size_t bytes = b200_fused_experts_fp8_workspace_bytes(m, k, N, static_cast<int>(topk), static_cast<int>(E), ue8m0);
    const Tensor work = empty({static_cast<int64_t>(bytes)}, at::kByte, dev);
    rc = b200_fused_experts_fp8(xp, dt_of(xt), w13p, w2p, s13p, s2p, twp, tip, m, k, N, static_cast<int>(topk),
                                static_cast<int>(E), tables[0], tables[1], tables[2], out.data_ptr(), ue8m0,
                                work.data_ptr(), bytes, stream_of(dev));
  }
  if (rc != 0) return raise_status("fused_experts_fp8", rc);
  return THPVariable_Wrap(std::move(out));
}
HOST_END

// ---- checked arguments of the functions below
// The message is put together only for a call that is refused: sixty strings a call took 4 us.
#define NEED(ok, message)                                        \
  do {                                                           \
    if (!(ok)) throw std::runtime_error(std::string() + message); \
  } while (0)
const Tensor& tensor_arg(PyObject* o, const char* name) {
  NEED(THPVariable_Check(o), std::string(name) + " must be a tensor");
  const Tensor& t = THPVariable_Unpack(o);
  NEED(t.defined() && t.layout() == at::kStrided && !t.is_neg() && !t.is_conj() &&
           !t.unsafeGetTensorImpl()->key_set().has(c10::DispatchKey::Python),
       std::string(name) + " must be a plain strided tensor");
  return t;
}
Tensor optional_arg(PyObject* o, const char* name) { return o == Py_None ? Tensor() : tensor_arg(o, name); }
void need_sizes(const Tensor& t, at::IntArrayRef sizes, const char* name) {
  if (t.sizes() == sizes) return;
  std::string want, got;
  for (const int64_t n : sizes) want += (want.empty() ? "" : ", ") + std::to_string(n);
  for (const int64_t n : t.sizes()) got += (got.empty() ? "" : ", ") + std::to_string(n);
  NEED(false, std::string(name) + " must have shape [" + want + "], got [" + got + "]");
}
void need_type(const Tensor& t, at::ScalarType type, const char* name, const char* what) {
  NEED(t.scalar_type() == type, std::string(name) + " must be " + what);
}
// The stride of a dimension; one that holds at most one element has none, nor has an empty tensor.
int64_t stride_of(const Tensor& t, int d) { return t.size(d) > 1 && t.numel() > 0 ? t.stride(d) : 0; }
// The leading dimension of a matrix whose rows do not overlap.
int64_t ld_of(const Tensor& t) { return stride_of(t, 0) != 0 ? t.stride(0) : t.size(1); }
void need_own_rows(const Tensor& t, const char* name) {       // a row broadcast over several is refused, too
  NEED(t.size(0) <= 1 || t.numel() == 0 || t.stride(0) >= t.size(1), std::string(name) + " must not overlap itself");
}
void need_rows(const Tensor& t, int64_t multiple, const char* name) {      // the last dimension dense, the others in whole vectors
  NEED(t.numel() == 0 || t.size(-1) == 1 || t.stride(-1) == 1, std::string(name) + " must be contiguous in its last dimension");
  for (int d = 0; d + 1 < t.dim(); ++d)
    NEED(stride_of(t, d) % multiple == 0,
         std::string(name) + ": strides must be multiples of " + std::to_string(multiple) + " elements");
}
void need_aligned(const Tensor& t, const char* name) {
  NEED(!t.defined() || (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15u) == 0, std::string(name) + " must be 16-byte aligned");
}
void need_writable(const Tensor& t, const char* name) {     // no two elements in one place
  for (int d = 0; d < t.dim(); ++d)
    NEED(t.size(d) <= 1 || t.stride(d) > 0, std::string(name) + " must not be an expanded tensor");
}
void need_index(const Tensor& t, int64_t n, const char* name) {
  NEED(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, std::string(name) + " must be int32 or int64");
  need_sizes(t, {n}, name);
  NEED(n <= 1 || t.stride(0) == 1, std::string(name) + " must be contiguous");
}
at::Device one_device(std::initializer_list<const Tensor*> all) {
  const at::Device dev = (*all.begin())->device();
  for (const Tensor* t : all) {
    if (!t->defined()) continue;
    NEED(t->is_cuda(), "all tensors must be CUDA tensors");
    NEED(t->device() == dev, "all tensors must be on the same device");
  }
  return dev;
}
// The bytes of a tensor: runs of `width` neighbouring ones, `count[d]` of them `step[d]` apart in each of n dimensions, the largest
// step first; `span[d]` is how far those of the dimensions from d on reach.  What is broadcast counts once.
struct Bytes {
  const char* at;
  int n = 0;
  int64_t count[8], step[8], span[9];
};
Bytes bytes_of(const Tensor& t) {
  Bytes b;
  b.at = static_cast<const char*>(t.const_data_ptr());
  int64_t width = static_cast<int64_t>(t.element_size());
  for (int d = 0; d < t.dim(); ++d) {
    if (t.size(d) <= 1 || t.stride(d) == 0) continue;
    const int64_t step = t.stride(d) * static_cast<int64_t>(t.element_size());
    int i = b.n++;
    for (; i > 0 && b.step[i - 1] < step; --i) b.step[i] = b.step[i - 1], b.count[i] = b.count[i - 1];
    b.step[i] = step, b.count[i] = t.size(d);
  }
  while (b.n > 0 && b.step[b.n - 1] == width) width *= b.count[--b.n];
  b.span[b.n] = width;
  for (int d = b.n - 1; d >= 0; --d) b.span[d] = b.span[d + 1] + (b.count[d] - 1) * b.step[d];
  return b;
}
// Whether the bytes of a from dimension i on and those of b from j on meet, b's beginning `off` bytes behind a's.  Two dimensions of one
// step are walked through together: only how many steps the two are apart matters.  Exact, unless there are more than 64
// places to look at in some dimension, which count as meeting.
bool meet(const Bytes& a, int i, const Bytes& b, int j, int64_t off) {
  if (off >= a.span[i] || -off >= b.span[j]) return false;
  if (i == a.n && j == b.n) return true;
  const bool in_a = i < a.n && (j == b.n || a.step[i] >= b.step[j]), in_b = j < b.n && (i == a.n || b.step[j] >= a.step[i]);
  const int64_t step = in_a ? a.step[i] : b.step[j];
  const int ni = i + in_a, nj = j + in_b;
  // by m steps a is ahead: -b.span[nj] < off - m step < a.span[ni]
  auto floor_div = [](int64_t x, int64_t y) { return x >= 0 ? x / y : -((-x + y - 1) / y); };
  int64_t from = floor_div(off - a.span[ni], step) + 1, to = -floor_div(-(off + b.span[nj]), step) - 1;
  from = std::max(from, in_b ? 1 - b.count[j] : 0);
  to = std::min(to, in_a ? a.count[i] - 1 : 0);
  if (to - from >= 64) return true;
  for (int64_t m = from; m <= to; ++m)
    if (meet(a, ni, b, nj, off - m * step)) return true;
  return false;
}
bool share_memory(const Tensor& t, const Tensor& u) {
  if (!t.defined() || !u.defined() || t.numel() == 0 || u.numel() == 0) return false;
  const Bytes a = bytes_of(t), b = bytes_of(u);
  return meet(a, 0, b, 0, b.at - a.at);
}
bool same_view(const Tensor& t, const Tensor& u) {
  if (!t.defined() || !u.defined() || t.const_data_ptr() != u.const_data_ptr() || t.sizes() != u.sizes()) return false;
  for (int d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1 && t.stride(d) != u.stride(d)) return false;
  return true;
}
// What a call writes must lie in places of its own: not overlap itself, nor, unless it is `in_place`, anything else that the call has.
// Nearly always the ranges of addresses settle it; only where two meet are the bytes looked at.
struct Held {
  Held(const Tensor& t, const char* name) : t(t), name(name), any(t.defined() && t.numel() > 0) {
    if (!any) return;
    dense = t.is_non_overlapping_and_dense();
    lo = static_cast<const char*>(t.const_data_ptr());
    int64_t last = t.numel() - 1;
    if (!dense) {
      last = 0;
      for (int d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    }
    hi = lo + (last + 1) * static_cast<int64_t>(t.element_size());
  }
  const Tensor& t;
  const char* name;
  bool any, dense = false;
  const char *lo = nullptr, *hi = nullptr;
};
void need_own_memory(const Held& out, const Held* in_place, at::ArrayRef<Held> all) {
  if (!out.any) return;
  if (!out.dense) {
    const Bytes b = bytes_of(out.t);
    for (int d = 0; d < b.n; ++d) NEED(b.step[d] >= b.span[d + 1], std::string(out.name) + " must not overlap itself");
  }
  for (const Held& o : all) {
    if (!o.any || &o == &out || out.hi <= o.lo || o.hi <= out.lo) continue;
    NEED((&o == in_place && same_view(out.t, o.t)) || !share_memory(out.t, o.t),
         std::string(out.name) + " must share no memory with " + o.name + (&o == in_place ? " or be it" : ""));
  }
}
b200_heads heads_of(const Tensor& t) { return {t.data_ptr(), stride_of(t, 0), stride_of(t, 1)}; }

struct CacheArgs {
  Tensor k, v, ks, vs;
  int64_t pages = 0, page = 0, heads = 0, dim = 0;
};
CacheArgs cache_args(PyObject* const* a) {
  CacheArgs c{tensor_arg(a[0], "k_cache"), tensor_arg(a[1], "v_cache"), tensor_arg(a[2], "k_scale"), tensor_arg(a[3], "v_scale")};
  NEED(c.k.dim() == 4, "k_cache must be [num_pages, page_size, num_kv_heads, head_dim]");
  c.pages = c.k.size(0), c.page = c.k.size(1), c.heads = c.k.size(2), c.dim = c.k.size(3);
  NEED(c.page > 0, "the pages of k_cache must hold at least one token");
  NEED(c.page < (1LL << 31) && c.pages < (1LL << 31) / c.page, "num_pages * page_size must be below 2^31");
  need_type(c.k, at::kFloat8_e4m3fn, "k_cache", "float8_e4m3fn");
  need_type(c.v, at::kFloat8_e4m3fn, "v_cache", "float8_e4m3fn");
  need_type(c.ks, at::kFloat, "k_scale", "float32");
  need_type(c.vs, at::kFloat, "v_scale", "float32");
  need_sizes(c.v, c.k.sizes(), "v_cache");
  need_sizes(c.ks, {c.pages, c.page, c.heads}, "k_scale");
  need_sizes(c.vs, {c.pages, c.page, c.heads}, "v_scale");
  need_rows(c.k, 16, "k_cache");
  need_rows(c.v, 16, "v_cache");
  need_aligned(c.k, "k_cache");
  need_aligned(c.v, "v_cache");
  return c;
}
b200_kv_cache cache_of(const CacheArgs& c) {
  b200_kv_cache r = {c.k.data_ptr(), c.v.data_ptr(), static_cast<float*>(c.ks.data_ptr()), static_cast<float*>(c.vs.data_ptr())};
  for (int d = 0; d < 3; ++d) {
    r.k_stride[d] = stride_of(c.k, d), r.v_stride[d] = stride_of(c.v, d);
    r.k_scale_stride[d] = stride_of(c.ks, d), r.v_scale_stride[d] = stride_of(c.vs, d);
  }
  r.num_pages = c.pages, r.page_size = c.page;
  return r;
}
void need_heads(const Tensor& t, const char* name) {
  NEED(t.dim() == 3, std::string(name) + " must be [num_tokens, num_heads, head_dim]");
  NEED(is_16bit(t.scalar_type()), std::string(name) + " must be bfloat16 or float16");
  NEED(t.size(2) > 0 && t.size(2) % 16 == 0 && t.size(2) <= 256, "head_dim must be a multiple of 16, at most 256");
  need_rows(t, 8, name);
  need_aligned(t, name);
}
// `t` as an output of the sizes and type of `like`, or a new tensor when there is none.
void need_out(const Tensor& t, const Tensor& like, const char* name) {
  need_heads(t, name);
  need_sizes(t, like.sizes(), name);
  NEED(t.scalar_type() == like.scalar_type(), std::string(name) + " must have the type of its input");
  need_writable(t, name);
}

// Tensors of the caller's that a kernel has written: autograd then knows that what it kept of them is no more.
void wrote(std::initializer_list<const Tensor*> all) {
  for (const Tensor* t : all)
    if (t->defined() && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

PyObject* wrap_or_none(Tensor t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(t));
}
PyObject* pair_or_none(Tensor a, Tensor b) {
  PyObject* pa = wrap_or_none(std::move(a));
  PyObject* pb = wrap_or_none(std::move(b));
  PyObject* r = PyTuple_Pack(2, pa, pb);
  Py_DECREF(pa);
  Py_DECREF(pb);
  return r;
}

// head_rows(name, q | None, k, v | None, positions | None, cos_sin | None, q_weight | None, k_weight | None, norm_eps, is_neox,
//           q_out | None, k_out | None, want_k, k_cache | None, v_cache, k_scale, v_scale, slots) -> (q_out | None, k_out | None)
HOST_FN(head_rows) {
  NEED(n == 18, "head_rows takes 18 arguments");
  const char* name = PyUnicode_AsUTF8(a[0]);
  if (!name) return nullptr;
  const Tensor q = optional_arg(a[1], "q"), k = tensor_arg(a[2], "k"), v = optional_arg(a[3], "v");
  const Tensor pos = optional_arg(a[4], "positions"), cs = optional_arg(a[5], "cos_sin_cache");
  const Tensor qw = optional_arg(a[6], "q_weight"), kw = optional_arg(a[7], "k_weight");
  const double eps = PyFloat_AsDouble(a[8]);
  if (PyErr_Occurred()) return nullptr;
  const bool neox = PyObject_IsTrue(a[9]), want_k = PyObject_IsTrue(a[12]);
  Tensor qo = optional_arg(a[10], "q_out"), ko = optional_arg(a[11], "k_out");
  need_heads(k, "k");
  const int64_t T = k.size(0), Hkv = k.size(1), D = k.size(2);
  const at::ScalarType type = k.scalar_type();
  if (q.defined()) {
    need_heads(q, "q");
    NEED(q.size(0) == T && q.size(2) == D, "q and k must have the same number of tokens and the same head_dim");
    NEED(q.scalar_type() == type, "q and k must have the same type");
  }
  const int64_t Hq = q.defined() ? q.size(1) : 0;
  if (v.defined()) {
    need_heads(v, "v");
    need_sizes(v, k.sizes(), "v");
    NEED(v.scalar_type() == type, "k and v must have the same type");
  }
  int64_t rot = 0, rows = 0;
  if (pos.defined()) need_index(pos, T, "positions");
  if (cs.defined()) {
    NEED(pos.defined(), "positions must be given with cos_sin_cache");
    need_type(cs, at::kFloat, "cos_sin_cache", "float32");
    NEED(cs.dim() == 2 && cs.is_contiguous(), "cos_sin_cache must be a contiguous [max_position, rotary_dim] tensor");
    rows = cs.size(0), rot = cs.size(1);
    NEED(rot > 0 && rot % 16 == 0 && rot <= D, "rotary_dim must be a multiple of 16, at most head_dim");
    need_aligned(cs, "cos_sin_cache");
  }
  for (const auto& [w, what] : {std::pair<const Tensor&, const char*>{qw, "q_weight"}, {kw, "k_weight"}}) {
    if (!w.defined()) continue;
    need_sizes(w, {D}, what);
    NEED(w.scalar_type() == type, std::string(what) + " must have the type of k");
    NEED(w.is_contiguous(), std::string(what) + " must be contiguous");
    need_aligned(w, what);
  }
  if (qo.defined()) {
    NEED(q.defined(), "q_out without q");
    need_out(qo, q, "q_out");
  }
  if (ko.defined()) need_out(ko, k, "k_out");
  CacheArgs cache;
  Tensor slots;
  const bool store = a[13] != Py_None;
  if (store) {
    cache = cache_args(a + 13);
    slots = tensor_arg(a[17], "slots");
    NEED(v.defined(), "v must be given with a cache");
    NEED(cache.heads == Hkv && cache.dim == D, "the cache must have the heads of k: [num_pages, page_size, num_kv_heads, head_dim]");
    need_index(slots, T, "slots");
    for (const auto& [t, what] : {std::pair<const Tensor&, const char*>{cache.k, "k_cache"}, {cache.v, "v_cache"}, {cache.ks, "k_scale"}, {cache.vs, "v_scale"}})
      need_writable(t, what);
  }
  if (store || qo.defined() || ko.defined()) {
    const Held all[] = {{q, "q"}, {k, "k"}, {qo, "q_out"}, {ko, "k_out"}, {cache.k, "k_cache"}, {cache.v, "v_cache"}, {cache.ks, "k_scale"},
                        {cache.vs, "v_scale"}, {v, "v"}, {pos, "positions"}, {cs, "cos_sin_cache"}, {qw, "q_weight"}, {kw, "k_weight"},
                        {slots, "slots"}};
    // keys and values that are the same data may go to one cache: both write the same bytes
    const bool one = store && !pos.defined() && !kw.defined() && same_view(k, v);
    need_own_memory(all[2], &all[0], all);
    need_own_memory(all[3], &all[1], all);
    for (int i = 4; i < 8; ++i) need_own_memory(all[i], one ? &all[i ^ 1] : nullptr, all);
  }
  const at::Device dev = one_device({&k, &q, &v, &pos, &cs, &qw, &kw, &qo, &ko, &cache.k, &cache.v, &cache.ks, &cache.vs, &slots});
  int rc = 0;
  {
    const NoGil no_gil;
    const c10::cuda::OptionalCUDAGuard guard(dev);
    if (q.defined() && !qo.defined()) qo = empty({T, Hq, D}, type, dev);
    if (want_k && !ko.defined()) ko = empty({T, Hkv, D}, type, dev);
    if (T > 0 && Hq + Hkv > 0) {
      const b200_heads qh = q.defined() ? heads_of(q) : b200_heads{}, kh = heads_of(k), vh = v.defined() ? heads_of(v) : b200_heads{};
      const b200_heads qoh = qo.defined() ? heads_of(qo) : b200_heads{}, koh = ko.defined() ? heads_of(ko) : b200_heads{};
      const void* pp = pos.defined() ? pos.data_ptr() : nullptr;
      // a table without rows has no address, but is not no table: any will do, as no position is read from it
      const float* cp = cs.defined() ? static_cast<const float*>(rows > 0 ? cs.data_ptr() : (Hkv > 0 ? k : q).data_ptr()) : nullptr;
      const int pos64 = pos.defined() && pos.scalar_type() == at::kLong;
      const void *qwp = qw.defined() ? qw.data_ptr() : nullptr, *kwp = kw.defined() ? kw.data_ptr() : nullptr;
      const int dt = dt_of(type);
      void* st = stream_of(dev);
      if (!store) {
        rc = b200_qk_norm_rope(q.defined() ? &qh : nullptr, &kh, qo.defined() ? &qoh : nullptr, &koh, dt, pp, pos64, cp, rows,
                               static_cast<int>(rot), neox, qwp, kwp, static_cast<float>(eps), T, static_cast<int>(Hq),
                               static_cast<int>(Hkv), static_cast<int>(D), st);
      } else {
        const b200_kv_cache ch = cache_of(cache);
        const int slots64 = slots.scalar_type() == at::kLong;
        rc = b200_qk_norm_rope_store_kv_fp8(q.defined() ? &qh : nullptr, &kh, &vh, qo.defined() ? &qoh : nullptr,
                                            ko.defined() ? &koh : nullptr, dt, pp, pos64, cp, rows, static_cast<int>(rot), neox, qwp,
                                            kwp, static_cast<float>(eps), &ch, slots.data_ptr(), slots64, T, static_cast<int>(Hq),
                                            static_cast<int>(Hkv), static_cast<int>(D), st);
      }
    }
  }
  if (rc != 0) return raise_status(name, rc);
  wrote({&qo, &ko, &cache.k, &cache.v, &cache.ks, &cache.vs});
  return pair_or_none(std::move(qo), std::move(ko));
}
HOST_END

// load_kv(k_cache, v_cache, k_scale, v_scale, page_table, indptr, starts | None, num_tokens, dtype, k_out | None, v_out | None)
HOST_FN(load_kv) {
  NEED(n == 11, "load_kv takes 11 arguments");
  const CacheArgs cache = cache_args(a);
  const Tensor table = tensor_arg(a[4], "page_table"), indptr = tensor_arg(a[5], "kv_indptr"), starts = optional_arg(a[6], "kv_start");
  const int64_t T = PyLong_AsLongLong(a[7]);
  if (PyErr_Occurred()) return nullptr;
  NEED(THPDtype_Check(a[8]), "out_dtype must be a torch.dtype");
  const at::ScalarType type = reinterpret_cast<THPDtype*>(a[8])->scalar_type;
  NEED(is_16bit(type), "out_dtype must be bfloat16 or float16");
  NEED(T >= 0, "num_tokens must not be negative");
  NEED(cache.dim > 0 && cache.dim % 16 == 0 && cache.dim <= 256, "head_dim must be a multiple of 16, at most 256");
  NEED(table.dim() == 2 && table.scalar_type() == at::kInt, "page_table must be an int32 [batch, max_pages] tensor");
  NEED(table.size(1) <= 1 || table.stride(1) == 1, "page_table must be contiguous in its last dimension");
  const int64_t batch = table.size(0);
  NEED(indptr.scalar_type() == at::kInt, "kv_indptr must be int32");
  need_index(indptr, batch + 1, "kv_indptr");
  if (starts.defined()) {
    NEED(starts.scalar_type() == at::kInt, "kv_start must be int32");
    need_index(starts, batch, "kv_start");
  }
  Tensor ko = optional_arg(a[9], "k_out"), vo = optional_arg(a[10], "v_out");
  for (const auto& [t, what] : {std::pair<const Tensor&, const char*>{ko, "k_out"}, {vo, "v_out"}}) {
    if (!t.defined()) continue;
    need_heads(t, what);
    need_sizes(t, {T, cache.heads, cache.dim}, what);
    NEED(t.scalar_type() == type, std::string(what) + " must be of out_dtype");
    need_writable(t, what);
  }
  if (ko.defined() || vo.defined()) {
    const Held all[] = {{ko, "k_out"}, {vo, "v_out"}, {cache.k, "k_cache"}, {cache.v, "v_cache"}, {cache.ks, "k_scale"}, {cache.vs, "v_scale"},
                        {table, "page_table"}, {indptr, "kv_indptr"}, {starts, "kv_start"}};
    for (int i = 0; i < 2; ++i) need_own_memory(all[i], nullptr, all);
  }
  const at::Device dev = one_device({&cache.k, &cache.v, &cache.ks, &cache.vs, &table, &indptr, &starts, &ko, &vo});
  int rc;
  {
    const NoGil no_gil;
    const c10::cuda::OptionalCUDAGuard guard(dev);
    if (!ko.defined()) ko = empty({T, cache.heads, cache.dim}, type, dev);
    if (!vo.defined()) vo = empty({T, cache.heads, cache.dim}, type, dev);
    const b200_kv_cache ch = cache_of(cache);
    const b200_heads kh = heads_of(ko), vh = heads_of(vo);
    rc = b200_load_kv_fp8(&ch, static_cast<const int32_t*>(table.data_ptr()), stride_of(table, 0), table.size(1),
                          static_cast<const int32_t*>(indptr.data_ptr()),
                          starts.defined() ? static_cast<const int32_t*>(starts.data_ptr()) : nullptr, batch, &kh, &vh, dt_of(type), T,
                          static_cast<int>(cache.heads), static_cast<int>(cache.dim), stream_of(dev));
  }
  if (rc != 0) return raise_status("load_kv_fp8", rc);
  wrote({&ko, &vo});
  return pair_or_none(std::move(ko), std::move(vo));
}
HOST_END

// lora_plan(token_adapters, ranks, plan | None) -> plan, written on the current stream
HOST_FN(lora_plan) {
  NEED(n == 3, "lora_plan takes 3 arguments");
  const Tensor ids = tensor_arg(a[0], "token_adapters"), ranks = tensor_arg(a[1], "lora_ranks");
  Tensor plan = optional_arg(a[2], "plan");
  NEED(ids.dim() == 1 && ids.scalar_type() == at::kInt, "token_adapters must be an int32 [num_tokens] tensor");
  NEED(ranks.dim() == 1 && ranks.scalar_type() == at::kInt, "lora_ranks must be an int32 [num_adapters] tensor");
  NEED(ids.is_contiguous() && ranks.is_contiguous(), "token_adapters and lora_ranks must be contiguous");
  const int64_t T = ids.size(0), L = ranks.size(0);
  NEED(L > 0 && L <= 1024, "between 1 and 1024 adapters");
  NEED(T <= 1000000, "at most 1000000 tokens");
  const int64_t bytes = static_cast<int64_t>(b200_lora_plan_bytes(T, static_cast<int>(L)));
  if (plan.defined()) {
    need_type(plan, at::kByte, "plan", "uint8");
    need_sizes(plan, {bytes}, "plan");
    NEED(plan.is_contiguous(), "plan must be contiguous");
  }
  const at::Device dev = one_device({&ids, &ranks, &plan});
  int rc;
  {
    const NoGil no_gil;
    const c10::cuda::OptionalCUDAGuard guard(dev);
    if (!plan.defined()) plan = empty({bytes}, at::kByte, dev);
    rc = b200_lora_plan(static_cast<const int32_t*>(ids.data_ptr()), T, static_cast<const int32_t*>(ranks.data_ptr()),
                        static_cast<int>(L), plan.data_ptr(), static_cast<size_t>(bytes), stream_of(dev));
  }
  if (rc != 0) return raise_status("lora_plan", rc);
  wrote({&plan});
  return THPVariable_Wrap(std::move(plan));
}
HOST_END

// lora(base | None, x [T, K] | None, h [T, S R] | None, lora_a [L, S R, K] | None, lora_b [L, N, R] | None, plan, num_adapters,
//      scalings, sizes (a tuple of S) | None, num_slices, out | None) -> out [T, N]: shrink and expand; without lora_b only the
// shrink, which returns h; without x only the expand.
HOST_FN(lora) {
  NEED(n == 11, "lora takes 11 arguments");
  const Tensor base = optional_arg(a[0], "base_output"), x = optional_arg(a[1], "x"), A = optional_arg(a[3], "lora_a"),
               B = optional_arg(a[4], "lora_b"), plan = tensor_arg(a[5], "plan"), scalings = tensor_arg(a[7], "scalings");
  Tensor h = optional_arg(a[2], "h"), out = optional_arg(a[10], "out");
  const int64_t L = PyLong_AsLongLong(a[6]);
  int64_t S = PyLong_AsLongLong(a[9]);
  if (PyErr_Occurred()) return nullptr;
  int64_t T, K = 0, R = 0, N = 0;
  at::ScalarType type;
  std::vector<int64_t> sizes;
  if (a[8] != Py_None) {
    NEED(PyTuple_Check(a[8]), "output_sizes must be a sequence of integers");
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(a[8]); ++i) {
      sizes.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(a[8], i)));
      if (PyErr_Occurred()) return nullptr;
      NEED(sizes.back() >= 0 && sizes.back() % 8 == 0, "output_sizes must be multiples of 8");
    }
    S = static_cast<int64_t>(sizes.size());
  }
  NEED(S >= 1 && S <= 8, "between 1 and 8 slices");
  if (B.defined()) {
    NEED(B.dim() == 3 && B.is_contiguous(), "lora_b must be a contiguous [num_adapters, N, R] tensor");
    NEED(B.size(0) == L, "lora_b must hold the adapters of the batch");
    N = B.size(1), R = B.size(2);
    if (sizes.empty()) sizes.push_back(N);
    int64_t sum = 0;
    for (const int64_t v : sizes) sum += v;
    NEED(sum == N && N % 8 == 0 && static_cast<int64_t>(sizes.size()) == S, "output_sizes must add up to the rows of lora_b, multiples of 8");
    need_aligned(B, "lora_b");
  }
  if (x.defined()) {
    NEED(x.dim() == 2 && A.defined(), "x must be [num_tokens, K]");
    T = x.size(0), K = x.size(1), type = x.scalar_type();
    NEED(A.dim() == 3 && A.is_contiguous(), "lora_a must be a contiguous [num_adapters, num_slices * R, K] tensor");
    NEED(A.size(0) == L, "lora_a must hold the adapters of the batch");
    if (!B.defined()) {
      NEED(A.size(1) % S == 0, "the rows of lora_a must be num_slices * R");
      R = A.size(1) / S;
    }
    NEED(A.size(1) == S * R && A.size(2) == K, "lora_a must be [num_adapters, num_slices * R, K]");
    NEED(K % 8 == 0, "K must be a multiple of 8");
    need_rows(x, 8, "x");
    need_own_rows(x, "x");
    need_aligned(x, "x");
    need_aligned(A, "lora_a");
    NEED(A.scalar_type() == type, "lora_a must have the type of x");
  } else {
    NEED(h.defined() && B.defined() && h.dim() == 2, "h must be [num_tokens, num_slices * R]");
    T = h.size(0), type = h.scalar_type();
    need_sizes(h, {T, S * R}, "h");
    need_rows(h, 8, "h");
    need_own_rows(h, "h");
    need_aligned(h, "h");
  }
  NEED(is_16bit(type), "x must be bfloat16 or float16");
  NEED(R > 0 && R % 8 == 0 && R <= 256, "R must be a multiple of 8, at most 256");
  NEED(!B.defined() || B.scalar_type() == type, "lora_b must have the type of x");
  const int64_t bytes = static_cast<int64_t>(b200_lora_plan_bytes(T, static_cast<int>(L)));
  NEED(plan.scalar_type() == at::kByte && plan.is_contiguous() && plan.numel() == bytes, "the batch was made for another number of tokens");
  need_type(scalings, at::kFloat, "scalings", "float32");
  need_sizes(scalings, {L}, "scalings");
  NEED(scalings.is_contiguous(), "scalings must be contiguous");
  for (const auto& [t, what] : {std::pair<const Tensor&, const char*>{base, "base_output"}, {out, "out"}}) {
    if (!t.defined()) continue;
    NEED(t.dim() == 2 && t.scalar_type() == type, std::string(what) + " must be [num_tokens, N] in the type of x");
    need_sizes(t, {T, N}, what);
    need_rows(t, 8, what);
    need_aligned(t, what);
    need_own_rows(t, what);
  }
  if (out.defined() && out.numel() > 0) {
    const bool same = base.defined() && base.data_ptr() == out.data_ptr() && stride_of(base, 0) == stride_of(out, 0);
    NEED(same || !share_memory(out, base), "out must be base_output itself or share no memory with it");
    NEED(!share_memory(out, x) && !share_memory(out, h), "out must share no memory with x or h");
  }
  const at::Device dev = one_device({&plan, &base, &x, &h, &A, &B, &scalings, &out});
  int rc = 0;
  {
    const NoGil no_gil;
    const c10::cuda::OptionalCUDAGuard guard(dev);
    void* st = stream_of(dev);
    const int dt = dt_of(type), iL = static_cast<int>(L), iR = static_cast<int>(R), iS = static_cast<int>(S);
    if (x.defined()) h = empty({T, S * R}, type, dev);
    if (B.defined() && !out.defined()) out = empty({T, N}, type, dev);
    const size_t pb = static_cast<size_t>(bytes);
    const float* sp = static_cast<const float*>(scalings.data_ptr());
    const void* base_p = base.defined() ? base.data_ptr() : nullptr;
    const int64_t base_ld = base.defined() ? ld_of(base) : N;
    if (T > 0 && !B.defined())
      rc = b200_lora_shrink(x.data_ptr(), ld_of(x), A.data_ptr(), dt, plan.data_ptr(), pb, T, iL, K, iR, iS, h.data_ptr(), S * R, st);
    else if (T > 0 && N > 0 && x.defined())
      rc = b200_lora_apply(x.data_ptr(), ld_of(x), A.data_ptr(), B.data_ptr(), dt, plan.data_ptr(), pb, sp, T, iL, K, iR, sizes.data(), iS,
                           base_p, base_ld, out.data_ptr(), ld_of(out), h.data_ptr(), st);
    else if (T > 0 && N > 0)
      rc = b200_lora_expand(h.data_ptr(), ld_of(h), B.data_ptr(), dt, plan.data_ptr(), pb, sp, T, iL, iR, sizes.data(), iS, base_p,
                            base_ld, out.data_ptr(), ld_of(out), st);
  }
  if (rc != 0) return raise_status("lora", rc);
  wrote({&out});
  return THPVariable_Wrap(B.defined() ? std::move(out) : std::move(h));
}
HOST_END

#define ENTRY(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(linear),        ENTRY(quant),         ENTRY(norm_quant),         ENTRY(silu_and_mul),
                         ENTRY(matmul),        ENTRY(matmul_packed), ENTRY(gate_up_silu_quant), ENTRY(topk_softmax),
                         ENTRY(fused_gate),    ENTRY(experts),       ENTRY(head_rows),          ENTRY(load_kv),
                         ENTRY(lora_plan),     ENTRY(lora),          {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module_def); }
