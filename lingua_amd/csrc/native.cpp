// The linear's host path for an interpreter that calls it per layer: checks, allocations and library calls of one forward or
// backward pass in one function.  Bound by the host: from Python a forward + backward of a small linear was some thirty
// crossings of the language boundary and eleven allocations at 1.5 to 2 us each around thirteen kernels that take 90 us.
// us per pass, [1021,2048].[2048,2048] with a bias, forward + backward 271 / 148; one token through a kept [2048,2048]
// weight 14.9 / 8.6.
//
// Every function returns None where its operands are not the plain ones (other types, devices, strides that need a copy,
// empty problems, a dispatch mode): the Python form in lingua_amd/float8.py then runs, with its error messages.  The memos
// and the weight cache stay there too; nothing is kept here between calls.
#include <ATen/ATen.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/lingua_fp8.h"

namespace {

using at::Tensor;

// The library's entries, taken from the handle that lingua_amd._lib loaded (bind): one copy of the library per process.
struct Library {
#define L8_ENTRY(name) decltype(&::name) name = nullptr;
#define L8_ENTRIES(X)                                                                                                        \
  X(l8_last_error) X(l8_linear_fwd_rows) X(l8_linear_fwd_rows_workspace) X(l8_cast_rowwise) X(l8_cast_rowwise_workspace)               \
  X(l8_cast_tensorwise) X(l8_cast_tensorwise_t_rows) X(l8_amax_reduce) X(l8_cast_colwise_transposed_pad) X(l8_cast_transposed_many) X(l8_col_amax) X(l8_col_sum) X(l8_col_sum_workspace) X(l8_gemm_nt) X(l8_linear_bwd_casts_bias) X(l8_linear_bwd_casts_pays)  \
  X(l8_cast_rowwise_many) X(l8_cast_rowwise_cols_many) X(l8_gemm_nt_multi) X(l8_gemm_nt_sum) X(l8_rmsnorm_cast_rowwise)            \
  X(l8_rmsnorm_workspace) X(l8_rmsnorm_bwd_as) X(l8_rmsnorm_bwd_workspace) X(l8_swiglu_cast_rowwise) X(l8_swiglu_workspace)        \
  X(l8_swiglu_bwd_cast_rowwise_q) X(l8_swiglu_bwd_cast_transposed) X(l8_add_rmsnorm_cast_rowwise) X(l8_add_rmsnorm_bwd) X(l8_rotary)     \
  X(l8_rotary_axes) X(l8_dropout) X(l8_norm_fwd) X(l8_norm_bwd) X(l8_norm_bwd_workspace) X(l8_lowrank_route) X(l8_lowrank_shrink) X(l8_lowrank_splits)   \
  X(l8_lowrank_expand) X(l8_lowrank_outer) X(l8_lowrank_outer_workspace) X(l8_lowrank_outer_shrink) X(l8_lowrank_outer_shrink_pays) X(l8_lowrank_outer_shrink_workspace) X(l8_lowrank_add) X(l8_lowrank_add_workspace)                   \
  X(l8_cast_mxfp4) X(l8_cast_mxfp4_two) X(l8_mxfp4_to_bf16) X(l8_gemm_mxfp4_nt) X(l8_gemm_mxfp4_workspace) X(l8_mxfp4_linear) X(l8_mxfp4_linear_workspace)
  L8_ENTRIES(L8_ENTRY)
#undef L8_ENTRY
} lib;

void check(int code, const char *what) {
  if (code != L8_OK) throw std::runtime_error(std::string(what) + " failed (" + std::to_string(code) + "): " + lib.l8_last_error());
}

// A bf16 matrix as the kernels take it: `rows` rows of `cols` elements, `ld` apart.
struct Rows {
  const void *p = nullptr;
  int64_t rows = 0, cols = 0, ld = 0;
};

bool plain_type(PyObject *o) {
  return THPVariable_CheckExact(o) || Py_TYPE(o) == reinterpret_cast<PyTypeObject *>(ParameterClass);
}

// Leading dimensions of a contiguous tensor count as one; a view that would need a copy is not taken.
bool as_rows(const Tensor &t, int device, Rows &m) {
  if (t.scalar_type() != at::kBFloat16 || t.layout() != at::kStrided || !t.is_cuda() || t.get_device() != device || t.dim() < 2) return false;
  m.cols = t.size(-1);
  if (t.dim() == 2) {
    m.rows = t.size(0);
    if (m.rows < 1 || m.cols < 1 || t.stride(1) != 1 || t.stride(0) < m.cols) return false;
    m.ld = m.rows > 1 ? t.stride(0) : m.cols;
  } else {
    if (t.numel() < 1 || !t.is_contiguous()) return false;
    m.rows = t.numel() / m.cols;
    m.ld = m.cols;
  }
  m.p = t.const_data_ptr();
  return true;
}

// Rows on 16-byte lines?
bool on_16_bytes(const Rows &m) { return ((uintptr_t)m.p % 16) == 0 && m.ld % 8 == 0 && m.cols % 8 == 0; }
// A dense tensor of `n` elements of one type (quantised copies, scales, amaxes, bias).
bool dense(const Tensor &t, at::ScalarType type, int64_t n, int device) {
  return t.defined() && t.scalar_type() == type && t.layout() == at::kStrided && t.is_cuda() && t.get_device() == device && t.numel() == n && t.is_contiguous();
}

// A quantised operand handed in: rows x cols bytes, rows any stride apart (0: not one).
int64_t fp8_rows(const Tensor &t, int64_t rows, int64_t cols, int device) {
  if (!t.defined() || t.scalar_type() != at::kFloat8_e4m3fn || t.layout() != at::kStrided || !t.is_cuda() || t.get_device() != device ||
      t.dim() != 2 || t.size(0) != rows || t.size(1) != cols || t.stride(1) != 1 || (rows > 1 && t.stride(0) < cols))
    return 0;
  return rows > 1 ? t.stride(0) : cols;
}
// A new one, its rows on 128-byte lines (figures in linear.cpp) or dense.
Tensor empty_fp8(int64_t rows, int64_t cols, const at::TensorOptions &o, bool on_lines = true) {
  return at::empty_strided({rows, cols}, {on_lines ? (cols + 127) / 128 * 128 : cols, 1}, o.dtype(at::kFloat8_e4m3fn));
}

Tensor arg(PyObject *o) { return o == Py_None ? Tensor() : THPVariable_Unpack(o); }
PyObject *wrap(const Tensor &t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
bool truth(PyObject *o) {  // as `if` takes it: a switch of the configuration may hold any number
  const int t = PyObject_IsTrue(o);
  if (t < 0) throw python_error();
  return t != 0;
}
bool tensors(PyObject *const *args, int n) {  // Tensor or Parameter with memory of its own (not a batch under vmap) or None, and no mode that wants to see what is done to them
  for (int i = 0; i < n; ++i)
    if (args[i] != Py_None && !(plain_type(args[i]) && THPVariable_Unpack(args[i]).has_storage())) return false;
  return !c10::impl::dispatch_mode_enabled();
}
PyObject *tuple_of(std::initializer_list<Tensor> ts) {
  PyObject *out = PyTuple_New((Py_ssize_t)ts.size());
  if (!out) throw python_error();
  Py_ssize_t i = 0;
  for (const Tensor &t : ts) PyTuple_SET_ITEM(out, i++, wrap(t));
  return out;
}

// Work space of one call: freed into the caching allocator on return, as a Python temporary's would be.
struct Space {
  Tensor t;
  Space(const Tensor &like, int64_t bytes) {
    if (bytes > 0) t = at::empty({bytes}, like.options().dtype(at::kByte));
  }
  void *p() const { return t.defined() ? t.mutable_data_ptr() : nullptr; }
};

// linear_fwd(x, w, bias, qx, sx, x_ready, want_qx, want_col, qw, sw, want_amax, algo) -> (y, qx, sx, col amax, w's row amax) or None.
// The casts and the product of l8_linear_fwd_rows.  qx / sx: x already quantised (x_ready); want_qx: hand the quantised x out.
PyObject *linear_fwd(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12) throw std::runtime_error("linear_fwd: 12 arguments");
  if (!tensors(args, 5) || !tensors(args + 8, 2) || args[0] == Py_None || args[1] == Py_None) Py_RETURN_NONE;
  const Tensor &x = THPVariable_Unpack(args[0]), &w = THPVariable_Unpack(args[1]);
  const Tensor bias = arg(args[2]), qx_in = arg(args[3]), sx_in = arg(args[4]), qw = arg(args[8]), sw = arg(args[9]);
  const bool x_ready = truth(args[5]), want_qx = truth(args[6]), want_col = truth(args[7]), want_amax = truth(args[10]);
  const int64_t algo = PyLong_AsLongLong(args[11]);
  if (!x.is_cuda()) Py_RETURN_NONE;
  const int device = x.get_device();
  Rows rx, rw;
  if (!as_rows(x, device, rx) || !as_rows(w, device, rw) || w.dim() != 2 || rx.cols != rw.cols || rx.cols % 16 || rw.rows % 16 ||
      c10::hip::current_device() != device)
    Py_RETURN_NONE;
  const int64_t M = rx.rows, N = rw.rows, K = rx.cols;
  int64_t ldqx = x_ready ? fp8_rows(qx_in, M, K, device) : K, ldqw = qw.defined() ? fp8_rows(qw, N, K, device) : K;
  if ((bias.defined() && !dense(bias, at::kBFloat16, N, device)) || !ldqx || !ldqw || (x_ready && !dense(sx_in, at::kFloat, M, device)) ||
      (qw.defined() && !dense(sw, at::kFloat, N, device)))
    Py_RETURN_NONE;
  Tensor y, qx, sx, col, amax;
  {
    pybind11::gil_scoped_release no_gil;
    const auto o = x.options();
    if (x.dim() == 2) {
      y = at::empty({M, N}, o);
    } else {
      at::DimVector shape(x.sizes().begin(), x.sizes().end());
      shape.back() = N;
      y = at::empty(shape, o);
    }
    qx = qx_in;
    sx = sx_in;
    if (!x_ready && want_qx) {
      qx = empty_fp8(M, K, o);
      ldqx = qx.stride(0);
      sx = at::empty({M, 1}, o.dtype(at::kFloat));
    }
    if (want_col) col = at::empty({K}, o.dtype(at::kFloat));
    if (want_amax) amax = at::empty({N, 1}, o);
    l8_linear_fwd_args a{};
    a.x = rx.p, a.M = M, a.K = K, a.ldx = rx.ld;
    a.w = rw.p, a.N = N, a.ldw = rw.ld;
    a.bias = bias.defined() ? bias.const_data_ptr() : nullptr;
    a.y = y.mutable_data_ptr(), a.ldy = N;
    if (qx.defined()) a.qx = qx.mutable_data_ptr(), a.sx = sx.mutable_data_ptr<float>(), a.x_ready = x_ready;
    if (col.defined()) a.col_amax_x = col.mutable_data_ptr<float>();
    if (qw.defined()) a.qw = qw.mutable_data_ptr(), a.sw = sw.mutable_data_ptr<float>(), a.w_ready = 1;
    if (amax.defined()) a.amax_w = amax.mutable_data_ptr();
    a.algo = algo;
    a.stream = c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream();
    const int64_t need = lib.l8_linear_fwd_rows_workspace(&a, ldqx, ldqw);
    const Space ws(x, need);  // a negative size is an error that the call below reports
    a.workspace = ws.p(), a.workspace_bytes = need > 0 ? need : 0;
    check(lib.l8_linear_fwd_rows(&a, ldqx, ldqw), "l8_linear_fwd");
  }
  return tuple_of({y, qx, sx, col, amax});
  END_HANDLE_TH_ERRORS
}

// A matrix quantised along its rows' direction, padded to 16 of them, in the layout that the weight gradient multiplies with.
void cast_colwise_t(const Tensor &like, const Rows &m, const Tensor &col, bool on_lines, Tensor &q, Tensor &s, void *stream) {
  const auto o = like.options();
  const int64_t padded = (m.rows + 15) / 16 * 16;
  q = empty_fp8(m.cols, padded, o, on_lines);
  s = at::empty({m.cols, 1}, o.dtype(at::kFloat));
  check(lib.l8_cast_colwise_transposed_pad(m.p, m.rows, m.cols, m.ld, col.const_data_ptr<float>(), q.mutable_data_ptr(), q.stride(0), padded,
                                           s.mutable_data_ptr<float>(), stream), "l8_cast_colwise_transposed_pad");
}

// linear_bwd(g, a, w, w's row amax, a's col amax, qat, sat, qwt, swt, need_a, need_b, need_bias, algo)
//   -> (grad a, grad w, grad bias, qat, sat) or None.  fp8 weight gradient.  qat / sat: a already quantised along the tokens
// (then a may be None); qwt / swt: w already quantised tensor-wise and transposed.
PyObject *linear_bwd(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 13) throw std::runtime_error("linear_bwd: 13 arguments");
  if (!tensors(args, 9) || args[0] == Py_None || args[2] == Py_None || args[3] == Py_None) Py_RETURN_NONE;
  const Tensor &g = THPVariable_Unpack(args[0]), &w = THPVariable_Unpack(args[2]), &amax = THPVariable_Unpack(args[3]);
  const Tensor a = arg(args[1]), a_col_in = arg(args[4]), qat_in = arg(args[5]), sat_in = arg(args[6]), qwt_in = arg(args[7]), swt_in = arg(args[8]);
  const bool need_a = truth(args[9]), need_b = truth(args[10]), need_bias = truth(args[11]);
  const int algo = (int)PyLong_AsLongLong(args[12]);
  if (!g.is_cuda()) Py_RETURN_NONE;
  const int device = g.get_device();
  Rows rg, rw, ra;
  if (g.dim() != 2 || w.dim() != 2 || !as_rows(g, device, rg) || !as_rows(w, device, rw) || c10::hip::current_device() != device) Py_RETURN_NONE;
  const int64_t M = rg.rows, N = rg.cols, K = rw.cols, padded = (M + 15) / 16 * 16;
  if (rw.rows != N || N % 16 || K % 16 || !dense(amax, at::kBFloat16, N, device) ||
      (need_bias && (rg.ld % 8 || reinterpret_cast<uintptr_t>(rg.p) % 16)))
    Py_RETURN_NONE;
  if (need_b && !qat_in.defined() && !(a.defined() && a.dim() == 2 && as_rows(a, device, ra) && ra.rows == M && ra.cols == K)) Py_RETURN_NONE;
  if ((qat_in.defined() && !(fp8_rows(qat_in, K, padded, device) && dense(sat_in, at::kFloat, K, device))) ||
      (qwt_in.defined() && !(fp8_rows(qwt_in, K, N, device) && dense(swt_in, at::kFloat, 1, device))) ||
      (a_col_in.defined() && !dense(a_col_in, at::kFloat, K, device)))
    Py_RETURN_NONE;
  Tensor ga, gb, gbias, qat = qat_in, sat = sat_in, qwt = qwt_in, swt = swt_in;
  {
    pybind11::gil_scoped_release no_gil;
    const auto o = g.options();
    void *stream = c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream();
    Tensor g_col, qg, sg, qgt, sgt;
    // the casts of a small pass in two launches
    const bool together = need_a && need_b && !(need_b && !qat.defined() && !a_col_in.defined()) &&
                          (reinterpret_cast<uintptr_t>(amax.const_data_ptr()) % 16) == 0 && lib.l8_linear_bwd_casts_pays(M, N, K);
    if (together) {
      l8_linear_bwd_casts_args c{};
      qg = empty_fp8(M, N, o), sg = at::empty({M, 1}, o.dtype(at::kFloat));
      qgt = empty_fp8(N, padded, o), sgt = at::empty({N, 1}, o.dtype(at::kFloat));
      c.g = rg.p, c.M = M, c.N = N, c.ldg = rg.ld, c.K = K, c.Mp = padded, c.stream = stream;
      c.qg = qg.mutable_data_ptr(), c.ldqg = qg.stride(0), c.sg = sg.mutable_data_ptr<float>();
      c.qgt = qgt.mutable_data_ptr(), c.ldqgt = qgt.stride(0), c.sgt = sgt.mutable_data_ptr<float>();
      if (!qat.defined()) {
        qat = empty_fp8(K, padded, o), sat = at::empty({K, 1}, o.dtype(at::kFloat));
        c.a = ra.p, c.lda = ra.ld, c.a_col = a_col_in.const_data_ptr<float>();
        c.qat = qat.mutable_data_ptr(), c.ldqat = qat.stride(0), c.sat = sat.mutable_data_ptr<float>();
      }
      if (!qwt.defined()) {
        qwt = empty_fp8(K, N, o), swt = at::empty({1, 1}, o.dtype(at::kFloat));
        c.w = rw.p, c.ldw = rw.ld, c.amax_w = amax.const_data_ptr();
        c.qwt = qwt.mutable_data_ptr(), c.ldqwt = qwt.stride(0), c.swt = swt.mutable_data_ptr<float>();
      }
      c.workspace_bytes = lib.l8_cast_rowwise_workspace(M, N);
      const Space ws(g, c.workspace_bytes);
      c.workspace = ws.p();
      if (need_bias) gbias = at::empty({N}, o);
      check(lib.l8_linear_bwd_casts_bias(&c, need_bias ? gbias.mutable_data_ptr() : nullptr), "l8_linear_bwd_casts");
    }
    if (need_b && !together) g_col = at::empty({N}, o.dtype(at::kFloat));
    if (need_a && !together) {
      qg = empty_fp8(M, N, o), sg = at::empty({M, 1}, o.dtype(at::kFloat));
      const int64_t ws_bytes = need_b ? lib.l8_cast_rowwise_workspace(M, N) : 0;
      const Space ws(g, ws_bytes);
      check(lib.l8_cast_rowwise(rg.p, M, N, rg.ld, qg.mutable_data_ptr(), qg.stride(0), sg.mutable_data_ptr<float>(), nullptr,
                                need_b ? g_col.mutable_data_ptr<float>() : nullptr, ws.p(), ws_bytes, stream), "l8_cast_rowwise");
      if (!qwt.defined()) {
        qwt = empty_fp8(K, N, o);
        swt = at::empty({1, 1}, o.dtype(at::kFloat));
        if (N % 8 == 0 && N <= 16384 && (reinterpret_cast<uintptr_t>(amax.const_data_ptr()) % 16) == 0) {
          check(lib.l8_cast_tensorwise_t_rows(rw.p, N, K, rw.ld, amax.const_data_ptr(), N, qwt.mutable_data_ptr(), qwt.stride(0), swt.mutable_data_ptr<float>(), stream),
                "l8_cast_tensorwise_t_rows");
        } else {
          Tensor whole = at::empty({1, 1}, o);
          check(lib.l8_amax_reduce(amax.const_data_ptr(), N, whole.mutable_data_ptr(), stream), "l8_amax_reduce");
          check(lib.l8_cast_tensorwise(rw.p, N, K, rw.ld, whole.const_data_ptr(), L8_AMAX_BF16, 1, qwt.mutable_data_ptr(), qwt.stride(0), swt.mutable_data_ptr<float>(), stream),
                "l8_cast_tensorwise");
        }
      }
    }
    if (need_a) {
      ga = at::empty({M, K}, o);
      check(lib.l8_gemm_nt(qg.const_data_ptr(), qwt.const_data_ptr(), M, K, N, qg.stride(0), qwt.stride(0), sg.const_data_ptr<float>(), L8_SCALE_ROW, swt.const_data_ptr<float>(),
                           L8_SCALE_SCALAR, nullptr, ga.mutable_data_ptr(), K, algo, stream), "l8_gemm_nt");
    } else if (need_b) {
      check(lib.l8_col_amax(rg.p, M, N, rg.ld, g_col.mutable_data_ptr<float>(), stream), "l8_col_amax");
    }
    if (need_b) {
      if (together) {   // made above
      } else if (qat.defined()) {
        cast_colwise_t(g, rg, g_col, true, qgt, sgt, stream);
      } else {
        Tensor a_col = a_col_in;
        if (!a_col.defined()) {
          a_col = at::empty({K}, o.dtype(at::kFloat));
          check(lib.l8_col_amax(ra.p, M, K, ra.ld, a_col.mutable_data_ptr<float>(), stream), "l8_col_amax");
        }
        qgt = empty_fp8(N, padded, o), sgt = at::empty({N, 1}, o.dtype(at::kFloat));
        qat = empty_fp8(K, padded, o), sat = at::empty({K, 1}, o.dtype(at::kFloat));
        const l8_cast_transposed_item both[2] = {
            {rg.p, M, N, rg.ld, g_col.const_data_ptr<float>(), nullptr, 0, qgt.mutable_data_ptr(), qgt.stride(0), padded, sgt.mutable_data_ptr<float>()},
            {ra.p, M, K, ra.ld, a_col.const_data_ptr<float>(), nullptr, 0, qat.mutable_data_ptr(), qat.stride(0), padded, sat.mutable_data_ptr<float>()}};
        check(lib.l8_cast_transposed_many(both, 2, stream), "l8_cast_transposed_many");
      }
      gb = at::empty({N, K}, o);
      check(lib.l8_gemm_nt(qgt.const_data_ptr(), qat.const_data_ptr(), N, K, padded, qgt.stride(0), qat.stride(0), sgt.const_data_ptr<float>(), L8_SCALE_ROW,
                           sat.const_data_ptr<float>(), L8_SCALE_ROW, nullptr, gb.mutable_data_ptr(), K, algo, stream), "l8_gemm_nt");
    }
    if (need_bias && !together) {
      gbias = at::empty({N}, o);
      const int64_t ws_bytes = lib.l8_col_sum_workspace(M, N);
      const Space ws(g, ws_bytes);
      check(lib.l8_col_sum(rg.p, M, N, rg.ld, gbias.mutable_data_ptr(), ws.p(), ws_bytes, stream), "l8_col_sum");
    }
  }
  return tuple_of({ga, gb, gbias, qat, sat});
  END_HANDLE_TH_ERRORS
}

// cast_colwise_transposed(a, col amax, on_lines) -> (q, s) or None, as in lingua_amd.ops
PyObject *cast_colwise_transposed(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3) throw std::runtime_error("cast_colwise_transposed: 3 arguments");
  if (!tensors(args, 2) || args[0] == Py_None || args[1] == Py_None) Py_RETURN_NONE;
  const Tensor &a = THPVariable_Unpack(args[0]), &col = THPVariable_Unpack(args[1]);
  if (!a.is_cuda()) Py_RETURN_NONE;
  const int device = a.get_device();
  Rows ra;
  if (a.dim() != 2 || !as_rows(a, device, ra) || !dense(col, at::kFloat, ra.cols, device) || c10::hip::current_device() != device) Py_RETURN_NONE;
  const bool on_lines = truth(args[2]);
  Tensor q, s;
  {
    pybind11::gil_scoped_release no_gil;
    cast_colwise_t(a, ra, col, on_lines, q, s, c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream());
  }
  return tuple_of({q, s});
  END_HANDLE_TH_ERRORS
}

// ---- fused blocks ----
// Attention projections, gated MLP and norm: one call per pass where the Python form (lingua_amd/qkv.py, swiglu.py, norm.py,
// float8.shared_input_backward) makes ten to fifteen and twice as many allocations.  us per pass, forward + backward, bound by
// the host, before / now: norm and projections [337,2624] 517 / 160, norm and MLP [400,1328] with 2688 hidden 554 / 234.

// Temporaries of one phase of a pass, in one allocation that is freed into the caching allocator behind the phase.
struct Arena {
  int64_t bytes = 0;
  Tensor t;
  int64_t add(int64_t n) {
    const int64_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  }
  void make(const Tensor &like) { t = at::empty({bytes > 0 ? bytes : 1}, like.options().dtype(at::kByte)); }
  uint8_t *p(int64_t at) const { return static_cast<uint8_t *>(t.mutable_data_ptr()) + at; }
  float *f(int64_t at) const { return reinterpret_cast<float *>(p(at)); }
};

int64_t on_lines(int64_t cols) { return (cols + 127) / 128 * 128; }

// A quantised operand in an arena: rows on 128-byte lines, and its scales.
struct Quantised {
  int64_t rows, cols, ld, q, s;
  Quantised(Arena &a, int64_t rows_, int64_t cols_, int64_t scales) : rows(rows_), cols(cols_), ld(on_lines(cols_)), q(a.add(rows_ * on_lines(cols_))), s(a.add(scales * 4)) {}
};

// Can a weight with these row amaxes be quantised tensor-wise from the list (as lingua_amd.ops asks)?
bool listed(const Tensor &amax, int64_t rows, int device) {
  return dense(amax, at::kBFloat16, rows, device) && rows % 8 == 0 && rows <= 16384 && reinterpret_cast<uintptr_t>(amax.const_data_ptr()) % 16 == 0;
}
l8_cast_transposed_item by_columns(const Rows &m, const float *col, const Arena &a, const Quantised &q) {
  return {m.p, m.rows, m.cols, m.ld, col, nullptr, 0, a.p(q.q), q.ld, q.cols, a.f(q.s)};
}
l8_cast_transposed_item by_tensor(const Rows &w, const Tensor &amax, const Arena &a, const Quantised &q) {
  return {w.p, w.rows, w.cols, w.ld, nullptr, amax.const_data_ptr(), w.rows, a.p(q.q), q.ld, w.rows, a.f(q.s)};
}
bool weight(const Tensor &w, int device, Rows &m) { return w.defined() && w.dim() == 2 && as_rows(w, device, m) && m.rows % 16 == 0 && m.cols % 16 == 0; }
void *stream_of(int device) { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream(); }
// the activation of a block: plain, on the current device
bool activation(const Tensor &x, Rows &m) {
  return x.defined() && x.is_cuda() && x.dim() == 2 && as_rows(x, x.get_device(), m) && m.cols % 16 == 0 && c10::hip::current_device() == x.get_device();
}

// rmsnorm_fwd(x, weight, eps, want_col) -> (y, q, scale, rstd, col amax) or None
PyObject *rmsnorm_fwd(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) throw std::runtime_error("rmsnorm_fwd: 4 arguments");
  if (!tensors(args, 2) || args[0] == Py_None || args[1] == Py_None) Py_RETURN_NONE;
  const Tensor &x = THPVariable_Unpack(args[0]), &w = THPVariable_Unpack(args[1]);
  const double eps = PyFloat_AsDouble(args[2]);
  if (eps == -1.0 && PyErr_Occurred()) throw python_error();
  const bool want_col = truth(args[3]);
  Rows rx;
  if (!activation(x, rx)) Py_RETURN_NONE;
  const int device = x.get_device();
  const int64_t R = rx.rows, C = rx.cols;
  const bool f32 = w.scalar_type() == at::kFloat;
  if (!dense(w, f32 ? at::kFloat : at::kBFloat16, C, device)) Py_RETURN_NONE;
  Tensor y, q, s, rstd, col;
  {
    pybind11::gil_scoped_release no_gil;
    const auto o = x.options();
    y = at::empty({R, C}, o);
    q = empty_fp8(R, C, o);
    s = at::empty({R, 1}, o.dtype(at::kFloat));
    rstd = at::empty({R, 1}, o.dtype(at::kFloat));
    if (want_col) col = at::empty({C}, o.dtype(at::kFloat));
    const int64_t ws_bytes = want_col ? lib.l8_rmsnorm_workspace(R, C) : 0;
    const Space ws(x, ws_bytes);
    check(lib.l8_rmsnorm_cast_rowwise(rx.p, w.const_data_ptr(), f32, R, C, rx.ld, (float)eps, y.mutable_data_ptr(), C, q.mutable_data_ptr(), q.stride(0),
                                      s.mutable_data_ptr<float>(), rstd.mutable_data_ptr<float>(), want_col ? col.mutable_data_ptr<float>() : nullptr, ws.p(),
                                      ws_bytes, stream_of(device)), "l8_rmsnorm_cast_rowwise");
  }
  return tuple_of({y, q, s, rstd, col});
  END_HANDLE_TH_ERRORS
}

// rmsnorm_bwd(gy, x, weight, rstd) -> (gx, gw of the weight's type) or None
PyObject *rmsnorm_bwd(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) throw std::runtime_error("rmsnorm_bwd: 4 arguments");
  if (!tensors(args, 4)) Py_RETURN_NONE;
  const Tensor gy = arg(args[0]), x = arg(args[1]), w = arg(args[2]), rstd = arg(args[3]);
  Rows rx, rg;
  if (!activation(x, rx) || !activation(gy, rg) || gy.get_device() != x.get_device() || rg.rows != rx.rows || rg.cols != rx.cols) Py_RETURN_NONE;
  const int device = x.get_device();
  const int64_t R = rx.rows, C = rx.cols;
  const bool f32 = w.defined() && w.scalar_type() == at::kFloat;
  if (!dense(w, f32 ? at::kFloat : at::kBFloat16, C, device) || !dense(rstd, at::kFloat, R, device)) Py_RETURN_NONE;
  Tensor gx, gw;
  {
    pybind11::gil_scoped_release no_gil;
    gx = at::empty({R, C}, x.options());
    gw = at::empty({C}, w.options());
    const int64_t ws_bytes = lib.l8_rmsnorm_bwd_workspace(R, C);
    const Space ws(x, ws_bytes > 16 ? ws_bytes : 16);
    check(lib.l8_rmsnorm_bwd_as(rg.p, rx.p, w.const_data_ptr(), f32, rstd.const_data_ptr<float>(), R, C, rg.ld, rx.ld, gx.mutable_data_ptr(), C,
                                gw.mutable_data_ptr(), f32, ws.p(), ws_bytes, stream_of(device)), "l8_rmsnorm_bwd");
  }
  return tuple_of({gx, gw});
  END_HANDLE_TH_ERRORS
}

// The activation quantised, if it is not yet, for a block's forward pass.
void cast_activation(const Tensor &x, const Rows &rx, bool want_col, void *q, int64_t ldq, float *s, Tensor &col, void *stream) {
  if (want_col) col = at::empty({rx.cols}, x.options().dtype(at::kFloat));
  const int64_t ws_bytes = want_col ? lib.l8_cast_rowwise_workspace(rx.rows, rx.cols) : 0;
  const Space ws(x, ws_bytes);
  check(lib.l8_cast_rowwise(rx.p, rx.rows, rx.cols, rx.ld, q, ldq, s, nullptr, want_col ? col.mutable_data_ptr<float>() : nullptr, ws.p(), ws_bytes, stream),
        "l8_cast_rowwise");
}

// qkv_fwd(x, wq, wk, wv, qx, sx, want_col, algo) -> (y, row amax of wq, of wk, of wv, qx, sx, col amax of x) or None.
// qx / sx: x already quantised (then want_col is not looked at).
PyObject *qkv_fwd(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) throw std::runtime_error("qkv_fwd: 8 arguments");
  if (!tensors(args, 6)) Py_RETURN_NONE;
  const Tensor x = arg(args[0]), w[3] = {arg(args[1]), arg(args[2]), arg(args[3])}, qx_in = arg(args[4]), sx_in = arg(args[5]);
  const bool want_col = truth(args[6]);
  const int algo = (int)PyLong_AsLongLong(args[7]);
  Rows rx, rw[3];
  if (!activation(x, rx)) Py_RETURN_NONE;
  const int device = x.get_device();
  const int64_t M = rx.rows, K = rx.cols;
  int64_t N = 0;
  for (int i = 0; i < 3; ++i) {
    if (!weight(w[i], device, rw[i]) || rw[i].cols != K) Py_RETURN_NONE;
    N += rw[i].rows;
  }
  int64_t ldqx = qx_in.defined() ? fp8_rows(qx_in, M, K, device) : on_lines(K);
  if (!ldqx || (qx_in.defined() && !dense(sx_in, at::kFloat, M, device))) Py_RETURN_NONE;
  Tensor y, qx = qx_in, sx = sx_in, col, amax[3];
  {
    pybind11::gil_scoped_release no_gil;
    const auto o = x.options();
    void *stream = stream_of(device);
    if (!qx.defined()) {
      qx = empty_fp8(M, K, o), sx = at::empty({M, 1}, o.dtype(at::kFloat));
      cast_activation(x, rx, want_col, qx.mutable_data_ptr(), ldqx, sx.mutable_data_ptr<float>(), col, stream);
    }
    Arena a;
    const Quantised qw(a, N, K, N);
    a.make(x);
    l8_cast_rowwise_item items[3];
    for (int64_t i = 0, row = 0; i < 3; row += rw[i++].rows) {
      amax[i] = at::empty({rw[i].rows, 1}, o);
      items[i] = {rw[i].p, rw[i].rows, rw[i].ld, a.p(qw.q) + row * qw.ld, qw.ld, a.f(qw.s) + row, amax[i].mutable_data_ptr()};
    }
    check(lib.l8_cast_rowwise_many(items, 3, K, stream), "l8_cast_rowwise_many");
    y = at::empty({M, N}, o);
    check(lib.l8_gemm_nt(qx.const_data_ptr(), a.p(qw.q), M, N, K, ldqx, qw.ld, sx.const_data_ptr<float>(), L8_SCALE_ROW, a.f(qw.s), L8_SCALE_ROW, nullptr,
                         y.mutable_data_ptr(), N, algo, stream), "l8_gemm_nt");
  }
  return tuple_of({y, amax[0], amax[1], amax[2], qx, sx, col});
  END_HANDLE_TH_ERRORS
}

// shared_bwd((grad ...), x, (w ...), (row amax of w ...), col amax of x, qxt, sxt, algo) -> (grad x, qxt, sxt, grad w ...) or None:
// float8.shared_input_backward of up to three linears that all learn.  qxt / sxt: x already quantised along the tokens.
PyObject *shared_bwd(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) throw std::runtime_error("shared_bwd: 8 arguments");
  constexpr int kMost = 3;
  const Py_ssize_t k = PyTuple_Check(args[0]) ? PyTuple_GET_SIZE(args[0]) : 0;
  if (k < 1 || k > kMost || !PyTuple_Check(args[2]) || !PyTuple_Check(args[3]) || PyTuple_GET_SIZE(args[2]) != k || PyTuple_GET_SIZE(args[3]) != k) Py_RETURN_NONE;
  for (int i : {0, 2, 3})
    if (!tensors(&PyTuple_GET_ITEM(args[i], 0), (int)k)) Py_RETURN_NONE;
  if (!tensors(args + 1, 1) || !tensors(args + 4, 3)) Py_RETURN_NONE;
  const Tensor x = arg(args[1]), x_col = arg(args[4]), qxt_in = arg(args[5]), sxt_in = arg(args[6]);
  const int algo = (int)PyLong_AsLongLong(args[7]);
  Rows rx, rg[kMost], rw[kMost];
  Tensor g[kMost], w[kMost], amax[kMost];
  if (!activation(x, rx)) Py_RETURN_NONE;
  const int device = x.get_device();
  const int64_t M = rx.rows, K = rx.cols, padded = (M + 15) / 16 * 16;
  for (Py_ssize_t i = 0; i < k; ++i) {
    g[i] = arg(PyTuple_GET_ITEM(args[0], i)), w[i] = arg(PyTuple_GET_ITEM(args[2], i)), amax[i] = arg(PyTuple_GET_ITEM(args[3], i));
    if (!activation(g[i], rg[i]) || g[i].get_device() != device || !weight(w[i], device, rw[i]) || rg[i].rows != M || rw[i].cols != K ||
        rw[i].rows != rg[i].cols || !amax[i].defined() || !listed(amax[i], rw[i].rows, device))
      Py_RETURN_NONE;
  }
  if (qxt_in.defined() ? !(fp8_rows(qxt_in, K, padded, device) && dense(sxt_in, at::kFloat, K, device)) : !(x_col.defined() && dense(x_col, at::kFloat, K, device)))
    Py_RETURN_NONE;
  Tensor gx, gw[kMost], qxt = qxt_in, sxt = sxt_in;
  {
    pybind11::gil_scoped_release no_gil;
    const auto o = x.options();
    void *stream = stream_of(device);
    Arena cols;  // column amaxes of the gradients: from the first phase to the second
    int64_t col[kMost];
    for (int i = 0; i < k; ++i) col[i] = cols.add(rg[i].cols * 4);
    cols.make(x);
    {
      Arena a;
      std::vector<Quantised> qg, qw;
      int64_t ws[kMost], ws_bytes[kMost];
      for (int i = 0; i < k; ++i) {
        qg.emplace_back(a, M, rg[i].cols, M);
        qw.emplace_back(a, K, rw[i].rows, 1);
        ws_bytes[i] = lib.l8_cast_rowwise_workspace(M, rg[i].cols);
        ws[i] = a.add(ws_bytes[i]);
      }
      a.make(x);
      l8_cast_rowwise_cols_item casts[kMost];
      l8_cast_transposed_item weights[kMost];
      l8_gemm_term terms[kMost];
      for (int i = 0; i < k; ++i) {
        casts[i] = {rg[i].p, M, rg[i].cols, rg[i].ld, a.p(qg[i].q), qg[i].ld, a.f(qg[i].s), nullptr, cols.f(col[i]), a.p(ws[i]), ws_bytes[i]};
        weights[i] = by_tensor(rw[i], amax[i], a, qw[i]);
        terms[i] = {a.p(qg[i].q), a.p(qw[i].q), rg[i].cols, qg[i].ld, qw[i].ld, a.f(qg[i].s), a.f(qw[i].s)};
      }
      check(lib.l8_cast_rowwise_cols_many(casts, k, stream), "l8_cast_rowwise_cols_many");
      check(lib.l8_cast_transposed_many(weights, k, stream), "l8_cast_transposed_many");
      gx = at::empty({M, K}, o);
      check(lib.l8_gemm_nt_sum(terms, k, M, K, gx.mutable_data_ptr(), K, algo, stream), "l8_gemm_nt_sum");
    }
    Arena a;
    std::vector<Quantised> qt;
    for (int i = 0; i < k; ++i) qt.emplace_back(a, rg[i].cols, padded, rg[i].cols);
    a.make(x);
    l8_cast_transposed_item casts[kMost + 1];
    l8_gemm_part parts[kMost];
    for (int i = 0; i < k; ++i) {
      gw[i] = at::empty({rw[i].rows, K}, o);
      casts[i] = by_columns(rg[i], cols.f(col[i]), a, qt[i]);
      parts[i] = {a.p(qt[i].q), rw[i].rows, a.f(qt[i].s), gw[i].mutable_data_ptr()};
    }
    int64_t n_casts = k;
    if (!qxt.defined()) {
      qxt = empty_fp8(K, padded, o), sxt = at::empty({K, 1}, o.dtype(at::kFloat));
      casts[n_casts++] = {rx.p, M, K, rx.ld, x_col.const_data_ptr<float>(), nullptr, 0, qxt.mutable_data_ptr(), qxt.stride(0), padded, sxt.mutable_data_ptr<float>()};
    }
    check(lib.l8_cast_transposed_many(casts, n_casts, stream), "l8_cast_transposed_many");
    check(lib.l8_gemm_nt_multi(parts, k, qxt.const_data_ptr(), K, padded, on_lines(padded), qxt.stride(0), sxt.const_data_ptr<float>(), L8_SCALE_ROW, K, algo, stream),
          "l8_gemm_nt_multi");
  }
  PyObject *out = PyTuple_New(3 + k);
  if (!out) throw python_error();
  PyTuple_SET_ITEM(out, 0, wrap(gx));
  PyTuple_SET_ITEM(out, 1, wrap(qxt));
  PyTuple_SET_ITEM(out, 2, wrap(sxt));
  for (Py_ssize_t i = 0; i < k; ++i) PyTuple_SET_ITEM(out, 3 + i, wrap(gw[i]));
  return out;
  END_HANDLE_TH_ERRORS
}

// swiglu_fwd(x, w1, w3, w2, qx, sx, want_x_col, want_h_col, want_h, algo)
//   -> (y, h1, h3, row amax of w1, of w3, of w2, h, col amax of x, of h) or None.  qx / sx: x already quantised (no col amax then).
PyObject *swiglu_fwd(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10) throw std::runtime_error("swiglu_fwd: 10 arguments");
  if (!tensors(args, 6)) Py_RETURN_NONE;
  const Tensor x = arg(args[0]), w1 = arg(args[1]), w3 = arg(args[2]), w2 = arg(args[3]), qx = arg(args[4]), sx = arg(args[5]);
  const bool want_x_col = truth(args[6]), want_h_col = truth(args[7]), want_h = truth(args[8]);
  const int algo = (int)PyLong_AsLongLong(args[9]);
  Rows rx, r1, r3, r2;
  if (!activation(x, rx)) Py_RETURN_NONE;
  const int device = x.get_device();
  if (!weight(w1, device, r1) || !weight(w3, device, r3) || !weight(w2, device, r2)) Py_RETURN_NONE;
  const int64_t M = rx.rows, K = rx.cols, F = r1.rows, D = r2.rows;
  if (r1.cols != K || r3.cols != K || r3.rows != F || r2.cols != F) Py_RETURN_NONE;
  const int64_t ldqx = qx.defined() ? fp8_rows(qx, M, K, device) : on_lines(K);
  if (!ldqx || (qx.defined() && !dense(sx, at::kFloat, M, device))) Py_RETURN_NONE;
  Tensor y, h1, h3, h, amax1, amax3, amax2, x_col, h_col;
  {
    pybind11::gil_scoped_release no_gil;
    const auto o = x.options();
    void *stream = stream_of(device);
    amax1 = at::empty({F, 1}, o), amax3 = at::empty({F, 1}, o), amax2 = at::empty({D, 1}, o);
    {
      Arena a;
      const Quantised q1(a, F, K, F), q3(a, F, K, F), q(a, qx.defined() ? 0 : M, K, M);
      a.make(x);
      if (!qx.defined()) cast_activation(x, rx, want_x_col, a.p(q.q), q.ld, a.f(q.s), x_col, stream);
      const void *at_x = qx.defined() ? qx.const_data_ptr() : a.p(q.q);
      const float *scale_x = qx.defined() ? sx.const_data_ptr<float>() : a.f(q.s);
      const l8_cast_rowwise_item items[2] = {{r1.p, F, r1.ld, a.p(q1.q), q1.ld, a.f(q1.s), amax1.mutable_data_ptr()},
                                             {r3.p, F, r3.ld, a.p(q3.q), q3.ld, a.f(q3.s), amax3.mutable_data_ptr()}};
      check(lib.l8_cast_rowwise_many(items, 2, K, stream), "l8_cast_rowwise_many");
      h1 = at::empty({M, F}, o), h3 = at::empty({M, F}, o);
      check(lib.l8_gemm_nt(at_x, a.p(q1.q), M, F, K, ldqx, q1.ld, scale_x, L8_SCALE_ROW, a.f(q1.s), L8_SCALE_ROW, nullptr, h1.mutable_data_ptr(), F, algo, stream), "l8_gemm_nt");
      check(lib.l8_gemm_nt(at_x, a.p(q3.q), M, F, K, ldqx, q3.ld, scale_x, L8_SCALE_ROW, a.f(q3.s), L8_SCALE_ROW, nullptr, h3.mutable_data_ptr(), F, algo, stream), "l8_gemm_nt");
    }
    if (want_h) h = at::empty({M, F}, o);
    if (want_h_col) h_col = at::empty({F}, o.dtype(at::kFloat));
    Arena a;
    const Quantised qh(a, M, F, M), q2(a, D, F, D);
    const int64_t amax_h = a.add(M * 2), ws_bytes = want_h_col ? lib.l8_swiglu_workspace(M, F) / 2 : 0, ws = a.add(ws_bytes);
    a.make(x);
    check(lib.l8_swiglu_cast_rowwise(h1.const_data_ptr(), h3.const_data_ptr(), M, F, F, F, want_h ? h.mutable_data_ptr() : nullptr, F, a.p(qh.q), qh.ld, a.f(qh.s),
                                     a.p(amax_h), want_h_col ? h_col.mutable_data_ptr<float>() : nullptr, ws_bytes ? a.p(ws) : nullptr, ws_bytes, stream), "l8_swiglu_cast_rowwise");
    check(lib.l8_cast_rowwise(r2.p, D, F, r2.ld, a.p(q2.q), q2.ld, a.f(q2.s), amax2.mutable_data_ptr(), nullptr, nullptr, 0, stream), "l8_cast_rowwise");
    y = at::empty({M, D}, o);
    check(lib.l8_gemm_nt(a.p(qh.q), a.p(q2.q), M, D, F, qh.ld, q2.ld, a.f(qh.s), L8_SCALE_ROW, a.f(q2.s), L8_SCALE_ROW, nullptr, y.mutable_data_ptr(), D, algo, stream), "l8_gemm_nt");
  }
  return tuple_of({y, h1, h3, amax1, amax3, amax2, h, x_col, h_col});
  END_HANDLE_TH_ERRORS
}

// swiglu_bwd(gy, x, w1, w3, w2, h1, h3, row amax of w1, of w3, of w2, col amax of x, of h, algo) -> (grad x, grad w1, grad w3, grad w2)
// or None: every weight and x learn, the operands of the weight gradients are made from the gate's inputs.
PyObject *swiglu_bwd(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 13) throw std::runtime_error("swiglu_bwd: 13 arguments");
  if (!tensors(args, 12)) Py_RETURN_NONE;
  const Tensor gy = arg(args[0]), x = arg(args[1]), w1 = arg(args[2]), w3 = arg(args[3]), w2 = arg(args[4]), h1 = arg(args[5]), h3 = arg(args[6]), amax1 = arg(args[7]),
               amax3 = arg(args[8]), amax2 = arg(args[9]), x_col = arg(args[10]), h_col = arg(args[11]);
  const int algo = (int)PyLong_AsLongLong(args[12]);
  Rows rx, rg, r1, r3, r2, rh1, rh3;
  if (!activation(x, rx) || !activation(gy, rg) || !activation(h1, rh1) || !activation(h3, rh3)) Py_RETURN_NONE;
  const int device = x.get_device();
  if (gy.get_device() != device || h1.get_device() != device || h3.get_device() != device || !weight(w1, device, r1) || !weight(w3, device, r3) || !weight(w2, device, r2))
    Py_RETURN_NONE;
  const int64_t M = rx.rows, K = rx.cols, F = r1.rows, D = r2.rows, padded = (M + 15) / 16 * 16;
  if (rg.rows != M || rg.cols != D || rh1.rows != M || rh1.cols != F || rh3.rows != M || rh3.cols != F || r1.cols != K || r3.cols != K || r3.rows != F || r2.cols != F ||
      !amax1.defined() || !amax3.defined() || !amax2.defined() || !listed(amax1, F, device) || !listed(amax3, F, device) || !listed(amax2, D, device) ||
      !dense(x_col, at::kFloat, K, device) || !dense(h_col, at::kFloat, F, device))
    Py_RETURN_NONE;
  Tensor gx, gw1, gw3, gw2;
  {
    pybind11::gil_scoped_release no_gil;
    const auto o = x.options();
    void *stream = stream_of(device);
    Arena cols, hidden;  // column amaxes and the gradient of h: kept through the phases
    const int64_t gy_col = cols.add(D * 4), g1_col = cols.add(F * 4), g3_col = cols.add(F * 4), dh = hidden.add(M * F * 2);
    cols.make(x);
    hidden.make(x);
    {
      Arena a;
      const Quantised qgy(a, M, D, M), qw2(a, F, D, 1);
      const int64_t ws_bytes = lib.l8_cast_rowwise_workspace(M, D), ws = a.add(ws_bytes);
      a.make(x);
      check(lib.l8_cast_rowwise(rg.p, M, D, rg.ld, a.p(qgy.q), qgy.ld, a.f(qgy.s), nullptr, cols.f(gy_col), a.p(ws), ws_bytes, stream), "l8_cast_rowwise");
      check(lib.l8_cast_tensorwise_t_rows(r2.p, D, F, r2.ld, amax2.const_data_ptr(), D, a.p(qw2.q), qw2.ld, a.f(qw2.s), stream), "l8_cast_tensorwise_t_rows");
      check(lib.l8_gemm_nt(a.p(qgy.q), a.p(qw2.q), M, F, D, qgy.ld, qw2.ld, a.f(qgy.s), L8_SCALE_ROW, a.f(qw2.s), L8_SCALE_SCALAR, nullptr, hidden.p(dh), F, algo, stream),
            "l8_gemm_nt");
    }
    {
      Arena a;
      const Quantised q1(a, M, F, M), q3(a, M, F, M), qw1(a, K, F, 1), qw3(a, K, F, 1);
      const int64_t ws_bytes = lib.l8_swiglu_workspace(M, F), ws = a.add(ws_bytes);
      a.make(x);
      check(lib.l8_swiglu_bwd_cast_rowwise_q(hidden.p(dh), rh1.p, rh3.p, M, F, F, rh1.ld, rh3.ld, a.p(q1.q), a.p(q3.q), q1.ld, a.f(q1.s), a.f(q3.s), cols.f(g1_col),
                                             cols.f(g3_col), a.p(ws), ws_bytes, stream), "l8_swiglu_bwd_cast_rowwise");
      const l8_cast_transposed_item weights[2] = {by_tensor(r1, amax1, a, qw1), by_tensor(r3, amax3, a, qw3)};
      check(lib.l8_cast_transposed_many(weights, 2, stream), "l8_cast_transposed_many");
      gx = at::empty({M, K}, o);
      const l8_gemm_term terms[2] = {{a.p(q1.q), a.p(qw1.q), F, q1.ld, qw1.ld, a.f(q1.s), a.f(qw1.s)}, {a.p(q3.q), a.p(qw3.q), F, q3.ld, qw3.ld, a.f(q3.s), a.f(qw3.s)}};
      check(lib.l8_gemm_nt_sum(terms, 2, M, K, gx.mutable_data_ptr(), K, algo, stream), "l8_gemm_nt_sum");
    }
    Arena a;
    const Quantised qx(a, K, padded, K), qgy(a, D, padded, D), q1(a, F, padded, F), q3(a, F, padded, F), qh(a, F, padded, F);
    a.make(x);
    const l8_cast_transposed_item casts[2] = {by_columns(rx, x_col.const_data_ptr<float>(), a, qx), by_columns(rg, cols.f(gy_col), a, qgy)};
    check(lib.l8_cast_transposed_many(casts, 2, stream), "l8_cast_transposed_many");
    check(lib.l8_swiglu_bwd_cast_transposed(hidden.p(dh), rh1.p, rh3.p, M, F, F, rh1.ld, rh3.ld, cols.f(g1_col), cols.f(g3_col), h_col.const_data_ptr<float>(), a.p(q1.q),
                                            a.p(q3.q), a.p(qh.q), q1.ld, padded, a.f(q1.s), a.f(q3.s), a.f(qh.s), stream), "l8_swiglu_bwd_cast_transposed");
    hidden.t = Tensor();
    gw1 = at::empty({F, K}, o), gw3 = at::empty({F, K}, o), gw2 = at::empty({D, F}, o);
    const l8_gemm_part parts[2] = {{a.p(q1.q), F, a.f(q1.s), gw1.mutable_data_ptr()}, {a.p(q3.q), F, a.f(q3.s), gw3.mutable_data_ptr()}};
    check(lib.l8_gemm_nt_multi(parts, 2, a.p(qx.q), K, padded, q1.ld, qx.ld, a.f(qx.s), L8_SCALE_ROW, K, algo, stream), "l8_gemm_nt_multi");
    check(lib.l8_gemm_nt(a.p(qgy.q), a.p(qh.q), D, F, padded, qgy.ld, qh.ld, a.f(qgy.s), L8_SCALE_ROW, a.f(qh.s), L8_SCALE_ROW, nullptr, gw2.mutable_data_ptr(), F, algo, stream),
          "l8_gemm_nt");
  }
  return tuple_of({gx, gw1, gw3, gw2});
  END_HANDLE_TH_ERRORS
}

// add_rmsnorm_fwd(x, residual, weight, eps, want_q, want_col, want_rstd, on_lines) -> (h, y, q, scale, rstd, col amax) or None
PyObject *add_rmsnorm_fwd(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) throw std::runtime_error("add_rmsnorm_fwd: 8 arguments");
  if (!tensors(args, 3) || args[0] == Py_None || args[1] == Py_None || args[2] == Py_None) Py_RETURN_NONE;
  const Tensor &x = THPVariable_Unpack(args[0]), &res = THPVariable_Unpack(args[1]), &w = THPVariable_Unpack(args[2]);
  const double eps = PyFloat_AsDouble(args[3]);
  if (eps == -1.0 && PyErr_Occurred()) throw python_error();
  const bool want_q = truth(args[4]), want_col = truth(args[5]), want_rstd = truth(args[6]), on_lines = truth(args[7]);
  if (!x.is_cuda() || x.dim() != 2 || res.dim() != 2 || (want_col && !want_q)) Py_RETURN_NONE;
  const int device = x.get_device();
  Rows rx, rr;
  if (!as_rows(x, device, rx) || !as_rows(res, device, rr) || rr.rows != rx.rows || rr.cols != rx.cols || !on_16_bytes(rx) || !on_16_bytes(rr) ||
      c10::hip::current_device() != device)
    Py_RETURN_NONE;
  const int64_t R = rx.rows, C = rx.cols;
  const bool f32 = w.scalar_type() == at::kFloat;
  if (!dense(w, f32 ? at::kFloat : at::kBFloat16, C, device)) Py_RETURN_NONE;
  Tensor h, y, q, s, rstd, col;
  {
    pybind11::gil_scoped_release no_gil;
    const auto o = x.options();
    h = at::empty({R, C}, o), y = at::empty({R, C}, o);
    if (want_q) q = empty_fp8(R, C, o, on_lines), s = at::empty({R, 1}, o.dtype(at::kFloat));
    if (want_rstd) rstd = at::empty({R, 1}, o.dtype(at::kFloat));
    if (want_col) col = at::empty({C}, o.dtype(at::kFloat));
    const int64_t ws_bytes = want_col ? lib.l8_rmsnorm_workspace(R, C) : 0;
    const Space ws(x, ws_bytes);
    check(lib.l8_add_rmsnorm_cast_rowwise(rx.p, rr.p, w.const_data_ptr(), f32, R, C, rx.ld, rr.ld, (float)eps, h.mutable_data_ptr(), C, y.mutable_data_ptr(), C,
                                          want_q ? q.mutable_data_ptr() : nullptr, want_q ? q.stride(0) : C, want_q ? s.mutable_data_ptr<float>() : nullptr,
                                          want_rstd ? rstd.mutable_data_ptr<float>() : nullptr, want_col ? col.mutable_data_ptr<float>() : nullptr, ws.p(), ws_bytes,
                                          stream_of(device)), "l8_add_rmsnorm_cast_rowwise");
  }
  return tuple_of({h, y, q, s, rstd, col});
  END_HANDLE_TH_ERRORS
}

// One MXFP4 copy: rows of codes and of scales, as lingua_amd.ops lays them out.
struct Mx {
  Tensor q, s;
  Mx() {}
  Mx(int64_t rows, int64_t cols, const at::TensorOptions &o, bool on_lines) {
    const int64_t blocks = (cols + 31) / 32, bytes = blocks * 16, padded = (bytes + 127) / 128 * 128;
    q = at::empty_strided({rows, bytes}, {on_lines && (padded - bytes) * 8 <= bytes ? padded : bytes, 1}, o.dtype(at::kFloat4_e2m1fn_x2));
    s = at::empty_strided({rows, blocks}, {(blocks + 15) / 16 * 16, 1}, o.dtype(at::kFloat8_e8m0fnu));
  }
  void *qp() const { return q.defined() ? q.mutable_data_ptr() : nullptr; }
  void *sp() const { return s.defined() ? s.mutable_data_ptr() : nullptr; }
  int64_t ldq() const { return q.defined() ? q.stride(0) : 0; }
  int64_t lds() const { return s.defined() ? s.stride(0) : 0; }
};
// One that is handed in: 16 bytes and a scale per block, each row dense.
struct MxRows {
  const void *q = nullptr, *s = nullptr;
  int64_t rows = 0, blocks = 0, ldq = 0, lds = 0;
};
bool as_mx(const Tensor &q, const Tensor &s, int device, MxRows &m) {
  if (!q.defined() || !s.defined() || (q.scalar_type() != at::kFloat4_e2m1fn_x2 && q.scalar_type() != at::kByte) ||
      (s.scalar_type() != at::kFloat8_e8m0fnu && s.scalar_type() != at::kByte) || q.layout() != at::kStrided || s.layout() != at::kStrided || !q.is_cuda() ||
      !s.is_cuda() || q.get_device() != device || s.get_device() != device || q.dim() != 2 || s.dim() != 2)
    return false;
  m.rows = q.size(0), m.blocks = s.size(1);
  if (m.rows < 1 || m.blocks < 1 || s.size(0) != m.rows || q.size(1) != 16 * m.blocks || q.stride(1) != 1 || s.stride(1) != 1) return false;
  m.ldq = m.rows > 1 ? q.stride(0) : 16 * m.blocks;
  m.lds = m.rows > 1 ? s.stride(0) : (m.blocks + 15) / 16 * 16;
  m.q = q.const_data_ptr(), m.s = s.const_data_ptr();
  return m.ldq >= 16 * m.blocks && m.ldq % 16 == 0 && m.lds >= m.blocks && ((uintptr_t)m.q % 16) == 0;
}
void cast_mx(const Rows &x, const Mx &rows, const Mx &cols, void *stream) {
  check(lib.l8_cast_mxfp4(x.p, x.rows, x.cols, x.ld, rows.qp(), rows.ldq(), rows.sp(), rows.lds(), cols.qp(), cols.ldq(), cols.sp(), cols.lds(), stream), "l8_cast_mxfp4");
}
void gemm_mx(const MxRows &a, const MxRows &b, const Tensor &bias, const Tensor &out, void *stream) {
  const int64_t K = a.blocks * 32, bytes = lib.l8_gemm_mxfp4_workspace(a.rows, b.rows, K);
  const Space ws(out, bytes);
  check(lib.l8_gemm_mxfp4_nt(a.q, a.s, b.q, b.s, a.rows, b.rows, K, a.ldq, a.lds, b.ldq, b.lds, bias.defined() ? bias.const_data_ptr() : nullptr, out.mutable_data_ptr(),
                             b.rows, ws.p(), bytes, stream), "l8_gemm_mxfp4_nt");
}
MxRows rows_of(const Mx &m) {
  MxRows r;
  as_mx(m.q, m.s, m.q.get_device(), r);
  return r;
}

// Rows of bytes that start on 16-byte lines, as the product wants them: `t` where they do, else a copy.  (Hooks on saved tensors hand a
// kept copy back in any layout.)
Tensor on_lines_of_16(const Tensor &t) {
  if (!t.defined() || t.dim() != 2 || !t.is_cuda() || (((uintptr_t)t.const_data_ptr() % 16) == 0 && t.stride(1) == 1 && (t.size(0) <= 1 || t.stride(0) % 16 == 0))) return t;
  return at::empty_strided(t.sizes(), {(t.size(1) + 15) / 16 * 16, 1}, t.options()).copy_(t);
}

// cast_mxfp4(x, rowwise, transposed, on_lines) -> (q, s, qt, st) or None
PyObject *cast_mxfp4(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) throw std::runtime_error("cast_mxfp4: 4 arguments");
  if (!tensors(args, 1) || args[0] == Py_None) Py_RETURN_NONE;
  const Tensor &x = THPVariable_Unpack(args[0]);
  const bool rowwise = truth(args[1]), transposed = truth(args[2]), on_lines = truth(args[3]);
  if (!x.is_cuda() || x.dim() != 2 || (!rowwise && !transposed)) Py_RETURN_NONE;
  const int device = x.get_device();
  Rows rx;
  if (!as_rows(x, device, rx) || !on_16_bytes(rx) || c10::hip::current_device() != device) Py_RETURN_NONE;
  Mx rows, cols;
  {
    pybind11::gil_scoped_release no_gil;
    if (rowwise) rows = Mx(rx.rows, rx.cols, x.options(), on_lines);
    if (transposed) cols = Mx(rx.cols, rx.rows, x.options(), on_lines);
    cast_mx(rx, rows, cols, stream_of(device));
  }
  return tuple_of({rows.q, rows.s, cols.q, cols.s});
  END_HANDLE_TH_ERRORS
}

// mxfp4_to_bf16(q, s, cols) -> y or None
PyObject *mxfp4_to_bf16(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3) throw std::runtime_error("mxfp4_to_bf16: 3 arguments");
  if (!tensors(args, 2) || args[0] == Py_None || args[1] == Py_None) Py_RETURN_NONE;
  const Tensor &q = THPVariable_Unpack(args[0]), &s = THPVariable_Unpack(args[1]);
  const int64_t cols = PyLong_AsLongLong(args[2]);
  if (cols == -1 && PyErr_Occurred()) throw python_error();
  if (!q.is_cuda()) Py_RETURN_NONE;
  const int device = q.get_device();
  MxRows m;
  if (!as_mx(q, s, device, m) || cols < 1 || cols > 32 * m.blocks || c10::hip::current_device() != device) Py_RETURN_NONE;
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    y = at::empty({m.rows, cols}, q.options().dtype(at::kBFloat16));
    check(lib.l8_mxfp4_to_bf16(m.q, m.ldq, m.s, m.lds, m.rows, cols, y.mutable_data_ptr(), cols, stream_of(device)), "l8_mxfp4_to_bf16");
  }
  return wrap(y);
  END_HANDLE_TH_ERRORS
}

// mxfp4_packed(x, qw, sw, bias) -> y or None: the product with a weight kept in MXFP4
PyObject *mxfp4_packed(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) throw std::runtime_error("mxfp4_packed: 4 arguments");
  if (!tensors(args, 4) || args[0] == Py_None || args[1] == Py_None || args[2] == Py_None) Py_RETURN_NONE;
  const Tensor &x = THPVariable_Unpack(args[0]), &qw = THPVariable_Unpack(args[1]), &sw = THPVariable_Unpack(args[2]);
  const Tensor bias = arg(args[3]);
  if (!x.is_cuda() || x.dim() != 2) Py_RETURN_NONE;
  const int device = x.get_device();
  Rows rx;
  MxRows w;
  if (!as_rows(x, device, rx) || !on_16_bytes(rx) || !as_mx(qw, sw, device, w) || (rx.cols + 31) / 32 != w.blocks || c10::hip::current_device() != device ||
      (bias.defined() && !dense(bias, at::kBFloat16, w.rows, device)))
    Py_RETURN_NONE;
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    y = at::empty({rx.rows, w.rows}, x.options());
    const int64_t bytes = lib.l8_mxfp4_linear_workspace(rx.rows, w.rows, rx.cols);
    const Space ws(x, bytes);
    check(lib.l8_mxfp4_linear(rx.p, rx.rows, rx.cols, rx.ld, w.q, w.ldq, w.s, w.lds, w.rows, bias.defined() ? bias.const_data_ptr() : nullptr, y.mutable_data_ptr(), w.rows,
                              ws.p(), bytes, stream_of(device)), "l8_mxfp4_linear");
  }
  return wrap(y);
  END_HANDLE_TH_ERRORS
}

// ---- differentiable forms ----
// The Python forms' backward passes take the interpreter from the thread that waits for them, at 20 to 30 us a node whatever the
// kernels take; as nodes of their own these need it neither way.  us, forward + backward of small operands, Python / here: residual
// norm 112 / 83, rotary 81 / 60, MXFP4 linear 111 / 93.  The Python forms run where operands need copies, under transforms and modes.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients as a pass that is itself differentiated hands them on: an error for whoever asks for the derivative of one that `varies` with
// something that learns.  (They come from kernels, which nothing records: each is made to ask for a gradient, so that the error is
// what it meets.  One that does not vary is a constant and stays one.)
variable_list once(variable_list grads, std::initializer_list<bool> varies, const char *what) {
  if (!at::GradMode::is_enabled()) return grads;
  size_t i = 0;
  for (const bool v : varies) {
    Tensor &g = grads[i++];
    if (v && g.defined()) g = torch::autograd::DelayedError(std::string(what) + " is not differentiable twice", 1)({g.detach().set_requires_grad(true)})[0];
  }
  return grads;
}
bool learns(const Tensor &t) { return t.defined() && t.requires_grad(); }
// Where an operand that says which elements or adapters a pass is about stood, and in which version.  A saved tensor's own check does not run
// under hooks, so a forward pass that is computed again (activation checkpointing) after the operand has changed would hand the backward pass the
// new contents: the same memory in another version.  (Hooks that kept a copy hand back other memory, with the contents of the forward pass.)
struct Stamp {
  int64_t at, version;
  explicit Stamp(const Tensor &t) : Stamp((int64_t)(uintptr_t)t.const_data_ptr(), t.is_inference() ? -1 : (int64_t)t._version()) {}
  Stamp(int64_t at, int64_t version) : at(at), version(version) {}
  void unchanged(const Tensor &now, const char *what, const char *name) const {
    TORCH_CHECK(version < 0 || now.is_inference() || at != (int64_t)(uintptr_t)now.const_data_ptr() || version == (int64_t)now._version(), what, ": ", name,
                " modified by an inplace operation between the forward pass and its recomputation");
  }
};
// A leaf's gradient is accumulated on the stream that its node was made on, and the node lives as long as a graph that holds it.  One
// made on the default stream cannot take part in a capture: the captured backward pass would end the process.
void refuse_captured(std::initializer_list<const Tensor *> inputs, const char *what) {
  bool capturing = false, asked = false;
  for (const Tensor *t : inputs) {
    if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (!node) continue;
    const auto stream = node->stream();
    if (!stream || stream->id() != 0) continue;
    if (!asked) capturing = c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None, asked = true;
    TORCH_CHECK(!capturing, what, ": captured while a graph of the same leaf, made on the default stream, is alive: release it first, or make it on another stream");
  }
}
PyObject *refuse_captured_py(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) throw std::runtime_error("refuse_captured: 4 arguments");
  Tensor t[3];
  for (int i = 0; i < 3; ++i)
    if (THPVariable_Check(args[i])) t[i] = THPVariable_Unpack(args[i]);
  if (at::GradMode::is_enabled()) refuse_captured({&t[0], &t[1], &t[2]}, PyUnicode_AsUTF8(args[3]));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
// A bf16 matrix as the kernels take it, or a dense copy.  (Hooks on saved tensors hand a kept one back in any layout, as gradients come.)
Tensor aligned_rows(const Tensor &t) {
  Rows r;
  return as_rows(t, t.get_device(), r) && on_16_bytes(r) ? t : t.clone(at::MemoryFormat::Contiguous);
}
Tensor gradient(const Tensor &g, const char *what) {
  TORCH_CHECK(g.scalar_type() == at::kBFloat16, what, " backward: bf16 gradients required, got ", g.scalar_type());
  return aligned_rows(g);
}
Rows rows_of(const Tensor &t) {
  Rows r;
  TORCH_CHECK(as_rows(t, t.get_device(), r), "gradient rows");
  return r;
}

struct AddRMSNorm : torch::autograd::Function<AddRMSNorm> {
  static constexpr const char *kName = "add_rmsnorm";
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &res, const Tensor &w, double eps, bool want_col) {
    const Rows rx = rows_of(x), rr = rows_of(res);
    const int64_t R = rx.rows, C = rx.cols;
    const int device = x.get_device();
    const auto o = x.options();
    const Tensor h = at::empty(x.sizes(), o), y = at::empty(x.sizes(), o), q = empty_fp8(R, C, o), s = at::empty({R, 1}, o.dtype(at::kFloat)),
                 rstd = at::empty({R, 1}, o.dtype(at::kFloat)), col = want_col ? at::empty({C}, o.dtype(at::kFloat)) : Tensor();
    const int64_t ws_bytes = want_col ? lib.l8_rmsnorm_workspace(R, C) : 0;
    const Space ws(x, ws_bytes);
    check(lib.l8_add_rmsnorm_cast_rowwise(rx.p, rr.p, w.const_data_ptr(), w.scalar_type() == at::kFloat, R, C, rx.ld, rr.ld, (float)eps, h.mutable_data_ptr(), C,
                                          y.mutable_data_ptr(), C, q.mutable_data_ptr(), q.stride(0), s.mutable_data_ptr<float>(), rstd.mutable_data_ptr<float>(),
                                          want_col ? col.mutable_data_ptr<float>() : nullptr, ws.p(), ws_bytes, stream_of(device)), "l8_add_rmsnorm_cast_rowwise");
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({h, w, rstd});
    ctx->saved_data["sum learns"] = learns(x) || learns(res);
    variable_list out = {h, y, q, s};
    if (want_col) out.push_back(col);
    ctx->mark_non_differentiable({out.begin() + 2, out.end()});
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    Tensor gx, gw;
    if (grads[1].defined()) {
      const Tensor h = aligned_rows(saved[0]), w = saved[1].contiguous(), rstd = saved[2].contiguous();
      const Tensor gy = gradient(grads[1], kName), gh = grads[0].defined() ? gradient(grads[0], kName) : Tensor();
      const Rows rg = rows_of(gy), rh = rows_of(h);
      const Rows ru = gh.defined() ? rows_of(gh) : Rows();
      const bool f32 = w.scalar_type() == at::kFloat;
      const int device = h.get_device();
      const c10::DeviceGuard guard(c10::Device(c10::DeviceType::CUDA, (c10::DeviceIndex)device));
      gx = at::empty(h.sizes(), h.options()), gw = at::empty({rh.cols}, w.options());
      const int64_t ws_bytes = lib.l8_rmsnorm_bwd_workspace(rh.rows, rh.cols);
      const Space ws(h, ws_bytes);
      if (gh.defined())
        check(lib.l8_add_rmsnorm_bwd(rg.p, ru.p, rh.p, w.const_data_ptr(), f32, rstd.const_data_ptr<float>(), rh.rows, rh.cols, rg.ld, ru.ld, rh.ld, gx.mutable_data_ptr(),
                                     rh.cols, gw.mutable_data_ptr(), f32, ws.p(), ws_bytes, stream_of(device)), "l8_add_rmsnorm_bwd");
      else
        check(lib.l8_rmsnorm_bwd_as(rg.p, rh.p, w.const_data_ptr(), f32, rstd.const_data_ptr<float>(), rh.rows, rh.cols, rg.ld, rh.ld, gx.mutable_data_ptr(), rh.cols,
                                    gw.mutable_data_ptr(), f32, ws.p(), ws_bytes, stream_of(device)), "l8_rmsnorm_bwd");
    } else if (grads[0].defined()) {   // only the sum was used
      TORCH_CHECK(grads[0].scalar_type() == at::kBFloat16, kName, " backward: bf16 gradients required, got ", grads[0].scalar_type());
      return {grads[0], grads[0], Tensor(), Tensor(), Tensor()};
    }
    const bool sum_learns = ctx->saved_data["sum learns"].toBool(), gx_varies = sum_learns || learns(saved[1]) || learns(grads[0]) || learns(grads[1]);
    return once({gx, gx, gw, Tensor(), Tensor()}, {gx_varies, gx_varies, sum_learns || learns(grads[1])}, kName);
  }
};

// add_rmsnorm(x, residual, weight, eps, want_col) -> (h, y, q, scale, col amax) or None
PyObject *add_rmsnorm(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) throw std::runtime_error("add_rmsnorm: 5 arguments");
  if (!tensors(args, 3) || args[0] == Py_None || args[1] == Py_None || args[2] == Py_None) Py_RETURN_NONE;
  const Tensor &x = THPVariable_Unpack(args[0]), &res = THPVariable_Unpack(args[1]), &w = THPVariable_Unpack(args[2]);
  const double eps = PyFloat_AsDouble(args[3]);
  if (eps == -1.0 && PyErr_Occurred()) throw python_error();
  const bool want_col = truth(args[4]);
  if (!x.is_cuda()) Py_RETURN_NONE;
  const int device = x.get_device();
  Rows rx, rr;
  if (!as_rows(x, device, rx) || !as_rows(res, device, rr) || x.sizes() != res.sizes() || !on_16_bytes(rx) || !on_16_bytes(rr) || c10::hip::current_device() != device ||
      !dense(w, w.scalar_type() == at::kFloat ? at::kFloat : at::kBFloat16, rx.cols, device))
    Py_RETURN_NONE;
  variable_list out;
  {
    pybind11::gil_scoped_release no_gil;
    if (at::GradMode::is_enabled()) refuse_captured({&x, &res, &w}, AddRMSNorm::kName);
    out = AddRMSNorm::apply(x, res, w, eps, want_col);
  }
  return tuple_of({out[0], out[1], out[2], out[3], want_col ? out[4] : Tensor()});
  END_HANDLE_TH_ERRORS
}

// Pairs that each axis of a position turns (none: one position a token), side by side or in turn.
struct Axes {
  std::vector<int64_t> sections;
  bool in_rounds = false;
};
// Both forms of a rotation: y of x, either of them possibly undefined.
void rotate(const Tensor (&x)[2], Tensor (&y)[2], const Tensor &cos, const Tensor &sin, const Tensor &pos, bool in_halves, bool inverse, const Axes &axes) {
  const Tensor &one = x[0].defined() ? x[0] : x[1];
  const int64_t B = one.size(0), S = one.size(1), D = one.size(3);
  int64_t at[3] = {0, 0, 0};   // strides of a position: axis, batch, token
  if (pos.defined())
    for (int64_t i = 0; i < pos.dim(); ++i) at[3 - pos.dim() + i] = pos.size(i) == 1 ? 0 : pos.stride(i);
  l8_rotary_operand two[2];
  for (int i = 0; i < 2; ++i) {
    two[i] = {nullptr, nullptr, 0, 0, 0, 0};
    if (!x[i].defined()) continue;
    y[i] = at::empty(x[i].sizes(), x[i].options());
    two[i] = {x[i].const_data_ptr(), y[i].mutable_data_ptr(), x[i].size(2), x[i].stride(0), x[i].stride(1), x[i].stride(2)};
  }
  const void *pos_p = pos.defined() ? pos.const_data_ptr() : nullptr;
  const bool i32 = pos.defined() && pos.scalar_type() == at::kInt;
  if (axes.sections.empty())
    check(lib.l8_rotary(two, B, S, D, 2 * cos.size(1), in_halves, inverse, cos.const_data_ptr<float>(), sin.const_data_ptr<float>(), cos.stride(0), cos.stride(1), cos.size(0),
                        pos_p, i32, at[1], at[2], stream_of(one.get_device())), "l8_rotary");
  else
    check(lib.l8_rotary_axes(two, B, S, D, axes.sections.data(), (int64_t)axes.sections.size(), axes.in_rounds, in_halves, inverse, cos.const_data_ptr<float>(),
                             sin.const_data_ptr<float>(), cos.stride(0), cos.stride(1), cos.size(0), pos_p, i32, at[0], at[1], at[2], stream_of(one.get_device())), "l8_rotary_axes");
}
// Dense heads, and for the interleaved layout pairs on 4-byte lines?
bool heads_fit(const Tensor &t, bool in_halves) {
  if (t.stride(3) != 1) return false;
  if (in_halves) return true;
  int64_t odd = (int64_t)((uintptr_t)t.const_data_ptr() >> 1);
  for (int i = 0; i < 3; ++i)
    if (t.size(i) > 1) odd |= t.stride(i);
  return (odd & 1) == 0;
}
// May the extension take these operands?
bool rotates(const Tensor (&x)[2], const Tensor &cos, const Tensor &sin, const Tensor &pos, bool in_halves, const Axes &axes) {
  const Tensor &one = x[0].defined() ? x[0] : x[1];
  if (!one.is_cuda() || one.dim() != 4) return false;
  const int device = one.get_device();
  const int64_t B = one.size(0), S = one.size(1), D = one.size(3);
  if (c10::hip::current_device() != device) return false;
  for (const Tensor &t : x)
    if (t.defined() && (t.scalar_type() != at::kBFloat16 || t.layout() != at::kStrided || !t.is_cuda() || t.get_device() != device || t.dim() != 4 || t.numel() < 1 ||
                        t.size(0) != B || t.size(1) != S || t.size(3) != D || !heads_fit(t, in_halves)))
      return false;
  for (const Tensor *t : {&cos, &sin})
    if (t->scalar_type() != at::kFloat || t->layout() != at::kStrided || !t->is_cuda() || t->get_device() != device || t->dim() != 2 || t->sizes() != cos.sizes() ||
        t->strides() != cos.strides())
      return false;
  const int64_t P = cos.size(0), rot = 2 * cos.size(1);
  if (rot < 2 || rot > D || (!pos.defined() && S > P)) return false;
  const int64_t count = (int64_t)axes.sections.size();
  if (count) {
    int64_t pairs = 0;
    for (const int64_t n : axes.sections) {
      if (n < 0 || n > 256) return false;
      pairs += n;
    }
    if (count > 4 || 2 * pairs != rot || !pos.defined()) return false;
  }
  if (pos.defined()) {   // broadcastable to [B,S], with axes to [axes,B,S]
    if ((pos.scalar_type() != at::kInt && pos.scalar_type() != at::kLong) || pos.layout() != at::kStrided || !pos.is_cuda() || pos.get_device() != device ||
        pos.dim() < 1 || pos.dim() > (count ? 3 : 2))
      return false;
    const int64_t whole[3] = {count, B, S};
    for (int64_t i = 0; i < pos.dim(); ++i)
      if (pos.size(i) != 1 && pos.size(i) != whole[3 - pos.dim() + i]) return false;
  }
  return true;
}

struct Rotary : torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext *ctx, const Tensor &xq, const Tensor &xk, const Tensor &cos, const Tensor &sin, const std::optional<Tensor> &at, bool in_halves,
                               std::vector<int64_t> sections, bool in_rounds) {
    const Tensor x[2] = {xq, xk}, pos = at.value_or(Tensor());
    Tensor y[2];
    rotate(x, y, cos, sin, pos, in_halves, false, Axes{sections, in_rounds});
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({cos, sin, pos});
    ctx->saved_data["half"] = in_halves;
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["rounds"] = in_rounds;
    return {y[0], y[1]};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    Tensor g[2], x[2];
    for (int i = 0; i < 2; ++i) {
      if (!grads[i].defined() || !ctx->needs_input_grad(i)) continue;
      TORCH_CHECK(grads[i].scalar_type() == at::kBFloat16, "rotary backward: bf16 gradients required, got ", grads[i].scalar_type());
      x[i] = heads_fit(grads[i], ctx->saved_data["half"].toBool()) ? grads[i] : grads[i].clone(at::MemoryFormat::Contiguous);
    }
    if (x[0].defined() || x[1].defined()) {
      const c10::DeviceGuard guard((x[0].defined() ? x[0] : x[1]).device());
      const Tensor in[2] = {x[0], x[1]};
      const bool alike = saved[0].strides() == saved[1].strides();   // (hooks may have handed one back in another layout)
      rotate(in, g, alike ? saved[0] : saved[0].contiguous(), alike ? saved[1] : saved[1].contiguous(), saved[2], ctx->saved_data["half"].toBool(), true,
             Axes{ctx->saved_data["sections"].toIntVector(), ctx->saved_data["rounds"].toBool()});
    }
    return once({g[0], g[1], Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()}, {learns(grads[0]), learns(grads[1])}, "rotary");
  }
};

// rotary(xq, xk, cos, sin, positions, in_halves, inverse) -> (yq, yk) or None; either of xq and xk may be None
PyObject *rotary(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) throw std::runtime_error("rotary: 7 arguments");
  if (!tensors(args, 5) || (args[0] == Py_None && args[1] == Py_None) || args[2] == Py_None || args[3] == Py_None) Py_RETURN_NONE;
  const Tensor x[2] = {arg(args[0]), arg(args[1])}, pos = arg(args[4]);
  const Tensor &cos = THPVariable_Unpack(args[2]), &sin = THPVariable_Unpack(args[3]);
  const bool in_halves = truth(args[5]), inverse = truth(args[6]);
  const Axes axes;
  if (!rotates(x, cos, sin, pos, in_halves, axes)) Py_RETURN_NONE;
  Tensor y[2];
  {
    pybind11::gil_scoped_release no_gil;
    rotate(x, y, cos, sin, pos, in_halves, inverse, axes);
  }
  return tuple_of({y[0], y[1]});
  END_HANDLE_TH_ERRORS
}

// rotary_pair(xq, xk, cos, sin, positions, in_halves[, sections, in_rounds]) -> (yq, yk), differentiable, or None
PyObject *rotary_pair(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 && n != 8) throw std::runtime_error("rotary_pair: 6 or 8 arguments");
  if (!tensors(args, 5) || args[0] == Py_None || args[1] == Py_None || args[2] == Py_None || args[3] == Py_None) Py_RETURN_NONE;
  const Tensor x[2] = {arg(args[0]), arg(args[1])}, pos = arg(args[4]);
  const Tensor &cos = THPVariable_Unpack(args[2]), &sin = THPVariable_Unpack(args[3]);
  const bool in_halves = truth(args[5]);
  Axes axes;
  if (n == 8) {
    if (!PyTuple_Check(args[6]) || PyTuple_GET_SIZE(args[6]) < 1) Py_RETURN_NONE;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[6]); ++i) {
      axes.sections.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(args[6], i)));
      if (axes.sections.back() == -1 && PyErr_Occurred()) throw python_error();
    }
    axes.in_rounds = truth(args[7]);
  }
  if (!rotates(x, cos, sin, pos, in_halves, axes)) Py_RETURN_NONE;
  variable_list y;
  {
    pybind11::gil_scoped_release no_gil;
    if (at::GradMode::is_enabled()) refuse_captured({&x[0], &x[1]}, n == 8 ? "rotary_axes" : "rotary");
    y = Rotary::apply(x[0], x[1], cos, sin, pos.defined() ? std::optional<Tensor>(pos) : std::nullopt, in_halves, axes.sections, axes.in_rounds);
  }
  return tuple_of({y[0], y[1]});
  END_HANDLE_TH_ERRORS
}

// ---- layer norm, dropout ----

// What is dropped of an operand: seed and step, and which call of the step.
struct Dropped {
  Tensor numbers;   // undefined: nothing
  int64_t site = 0, threshold = 0;
  const int64_t *p() const { return numbers.defined() ? numbers.const_data_ptr<int64_t>() : nullptr; }
};
std::optional<Tensor> maybe(const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
int64_t number(PyObject *o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
bool is_param(const Tensor &t, int64_t n, int device) { return !t.defined() || (t.dim() == 1 && dense(t, t.scalar_type() == at::kFloat ? at::kFloat : at::kBFloat16, n, device)); }
bool is_numbers(const Tensor &t, int device) { return !t.defined() || (t.dim() == 1 && dense(t, at::kLong, 2, device)); }
void *addr(const Tensor &t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
const void *caddr(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }

struct NormOut {
  Tensor h, y, q, s, stats, col;
};
NormOut norm_pass(const Tensor &x, const Tensor &res, const Tensor &w, const Tensor &b, const Dropped &drop, double eps, bool centred, bool want_q, bool want_col, bool want_stats,
                  bool on_lines) {
  const Rows rx = rows_of(x), rr = res.defined() ? rows_of(res) : Rows();
  const int64_t R = rx.rows, C = rx.cols;
  const auto o = x.options(), f32 = o.dtype(at::kFloat);
  NormOut out;
  if (res.defined()) out.h = at::empty(x.sizes(), o);
  out.y = at::empty(x.sizes(), o);
  if (want_q) out.q = empty_fp8(R, C, o, on_lines), out.s = at::empty({R, 1}, f32);
  if (want_stats) out.stats = at::empty({2, R}, f32);
  if (want_col) out.col = at::empty({C}, f32);
  const int64_t ws_bytes = want_col ? lib.l8_rmsnorm_workspace(R, C) : 0;
  const Space ws(x, ws_bytes);
  float *stats = want_stats ? out.stats.mutable_data_ptr<float>() : nullptr;
  const l8_norm_fwd_args a{rx.p, rr.p, caddr(w), caddr(b), w.defined() && w.scalar_type() == at::kFloat, b.defined() && b.scalar_type() == at::kFloat, centred, R, C, rx.ld, rr.ld, eps,
                           drop.p(), drop.site, drop.threshold, addr(out.h), C, addr(out.y), C, addr(out.q), want_q ? out.q.stride(0) : 0, (float *)addr(out.s), stats,
                           stats ? stats + R : nullptr, (float *)addr(out.col), ws.p(), ws_bytes, stream_of(x.get_device())};
  check(lib.l8_norm_fwd(&a), "l8_norm_fwd");
  return out;
}

constexpr const char *kNumbers = "the seed and step were";
struct Norm : torch::autograd::Function<Norm> {
  static const char *name(bool centred, bool added) { return !centred ? "add_rmsnorm" : added ? "add_layernorm" : "layernorm"; }
  // -> [h,] y[, q, scale[, col amax]]
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const std::optional<Tensor> &res, const std::optional<Tensor> &w, const std::optional<Tensor> &b,
                               const std::optional<Tensor> &numbers, int64_t site, int64_t threshold, double eps, bool centred, bool want_col, bool quantise) {
    const Tensor none;
    const Tensor &r = res ? *res : none, &wt = w ? *w : none, &bt = b ? *b : none, &n = numbers ? *numbers : none;
    const NormOut out = norm_pass(x, r, wt, bt, Dropped{n, site, threshold}, eps, centred, quantise, want_col, true, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({r.defined() ? out.h : x, wt, out.stats, n});
    ctx->saved_data["sum learns"] = learns(x) || learns(r);
    ctx->saved_data["centred"] = centred;
    ctx->saved_data["has"] = (int64_t)(r.defined() | (wt.defined() << 1) | (bt.defined() << 2));
    ctx->saved_data["b"] = bt.defined() ? (int64_t)bt.scalar_type() : (int64_t)0;
    ctx->saved_data["site"] = site;
    ctx->saved_data["threshold"] = threshold;
    if (n.defined()) {
      const Stamp s(n);
      ctx->saved_data["numbers"] = std::vector<int64_t>{s.at, s.version};
    }
    variable_list all;
    if (r.defined()) all.push_back(out.h);
    all.push_back(out.y);
    const size_t learn = all.size();
    if (quantise) all.insert(all.end(), {out.q, out.s});
    if (want_col) all.push_back(out.col);
    ctx->mark_non_differentiable({all.begin() + learn, all.end()});
    return all;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const int64_t has = ctx->saved_data["has"].toInt();
    const bool added = has & 1, has_w = has & 2, has_b = has & 4, centred = ctx->saved_data["centred"].toBool();
    const char *what = name(centred, added);
    const Tensor gh_in = added ? grads[0] : Tensor(), gy_in = grads[added ? 1 : 0];
    for (const Tensor *g : {&gh_in, &gy_in}) TORCH_CHECK(!g->defined() || g->scalar_type() == at::kBFloat16, what, " backward: bf16 gradients required, got ", g->scalar_type());
    // (asked for operand by operand, in the order in which those that are there were given)
    int at = 0;
    const bool need_x = ctx->needs_input_grad(at++), need_r = added && ctx->needs_input_grad(at++);
    const bool need_w = has_w && ctx->needs_input_grad(at++), need_b = has_b && ctx->needs_input_grad(at++);
    const Dropped drop{saved[3], ctx->saved_data["site"].toInt(), ctx->saved_data["threshold"].toInt()};
    if (saved[3].defined()) {
      const auto then = ctx->saved_data["numbers"].toIntVector();
      Stamp(then[0], then[1]).unchanged(saved[3], what, kNumbers);
    }
    Tensor gx, gres, gw, gb;
    auto all = [&](std::initializer_list<bool> varies) {
      return once({gx, gres, gw, gb, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()}, varies, what);
    };
    if (!gy_in.defined()) {   // only the sum was used, if anything
      if (!gh_in.defined()) return all({});
      gx = need_x ? gh_in : Tensor();
      if (gx.defined() && drop.numbers.defined()) {
        const c10::DeviceGuard guard(gh_in.device());
        const Tensor g = gh_in.contiguous(), numbers = drop.numbers.contiguous();
        gx = at::empty(g.sizes(), g.options());
        check(lib.l8_dropout(g.const_data_ptr(), nullptr, gx.mutable_data_ptr(), g.numel(), numbers.const_data_ptr<int64_t>(), drop.site, drop.threshold, stream_of(g.get_device())),
              "l8_dropout");
        variable_list one = once({gx}, {learns(gh_in)}, what);
        gx = one[0];
      }
      gres = need_r ? gh_in : Tensor();
      return {gx, gres, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
    const Tensor h = aligned_rows(saved[0]), w = saved[1].defined() ? saved[1].contiguous() : Tensor(), stats = saved[2].contiguous(),
                 numbers = saved[3].defined() ? saved[3].contiguous() : Tensor();
    const Tensor gy = gradient(gy_in, what), gh = gh_in.defined() ? gradient(gh_in, what) : Tensor();
    const Rows rh = rows_of(h), rg = rows_of(gy), ru = gh.defined() ? rows_of(gh) : Rows();
    const int64_t R = rh.rows, C = rh.cols;
    const int device = h.get_device();
    const c10::DeviceGuard guard(h.device());
    const auto o = h.options();
    gx = at::empty(h.sizes(), o);
    if (numbers.defined()) gres = at::empty(h.sizes(), o);
    if (need_w) gw = at::empty({C}, w.options());
    if (need_b) gb = at::empty({C}, o.dtype((at::ScalarType)ctx->saved_data["b"].toInt()));
    const int64_t ws_bytes = need_w || need_b ? lib.l8_norm_bwd_workspace(R, C, centred) : 0;
    const Space ws(h, ws_bytes);
    const float *st = stats.const_data_ptr<float>();
    const l8_norm_bwd_args a{rg.p, ru.p, rh.p, caddr(w), w.defined() && w.scalar_type() == at::kFloat, centred, R, C, rg.ld, ru.ld, rh.ld, st, st + R,
                             numbers.defined() ? numbers.const_data_ptr<int64_t>() : nullptr, drop.site, drop.threshold, addr(gx), C, addr(gres), C, addr(gw),
                             gw.defined() && gw.scalar_type() == at::kFloat, addr(gb), gb.defined() && gb.scalar_type() == at::kFloat, ws.p(), ws_bytes, stream_of(device)};
    check(lib.l8_norm_bwd(&a), "l8_norm_bwd");
    if (!numbers.defined()) gres = gx;
    if (!need_x) gx = Tensor();
    if (!need_r) gres = Tensor();
    const bool sum_learns = ctx->saved_data["sum learns"].toBool(), gy_learns = learns(gy_in), varies = sum_learns || learns(saved[1]) || learns(gh_in) || gy_learns;
    return all({varies, varies, sum_learns || gy_learns, gy_learns});
  }
};

bool norm_takes(const Tensor &x, const Tensor &res, const Tensor &w, const Tensor &b, const Tensor &numbers) {
  if (!x.is_cuda()) return false;
  const int device = x.get_device();
  Rows rx, rr;
  return as_rows(x, device, rx) && on_16_bytes(rx) && (!res.defined() || (as_rows(res, device, rr) && on_16_bytes(rr) && res.sizes() == x.sizes())) &&
         is_param(w, rx.cols, device) && is_param(b, rx.cols, device) && is_numbers(numbers, device) && c10::hip::current_device() == device;
}

// norm(x, residual, weight, bias, numbers, site, threshold, eps, centred, want_col, quantise) -> (h, y, q, scale, col amax), differentiable, or None
PyObject *norm(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11) throw std::runtime_error("norm: 11 arguments");
  if (!tensors(args, 5) || args[0] == Py_None) Py_RETURN_NONE;
  const Tensor &x = THPVariable_Unpack(args[0]);
  const Tensor res = arg(args[1]), w = arg(args[2]), b = arg(args[3]), numbers = arg(args[4]);
  const int64_t site = number(args[5]), threshold = number(args[6]);
  const double eps = PyFloat_AsDouble(args[7]);
  if (eps == -1.0 && PyErr_Occurred()) throw python_error();
  const bool centred = truth(args[8]), want_col = truth(args[9]), quantise = truth(args[10]);
  if (!norm_takes(x, res, w, b, numbers)) Py_RETURN_NONE;
  variable_list out;
  {
    pybind11::gil_scoped_release no_gil;
    if (at::GradMode::is_enabled()) refuse_captured({&x, &res, &w, &b}, Norm::name(centred, res.defined()));
    out = Norm::apply(x, maybe(res), maybe(w), maybe(b), maybe(numbers), site, threshold, eps, centred, want_col, quantise);
  }
  const size_t y = res.defined();
  return tuple_of({y ? out[0] : Tensor(), out[y], quantise ? out[y + 1] : Tensor(), quantise ? out[y + 2] : Tensor(), want_col ? out[y + 3] : Tensor()});
  END_HANDLE_TH_ERRORS
}

// norm_fwd(x, residual, weight, bias, numbers, site, threshold, eps, centred, want_q, want_stats, on_lines) -> (h, y, q, scale, stats) or None
PyObject *norm_fwd(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12) throw std::runtime_error("norm_fwd: 12 arguments");
  if (!tensors(args, 5) || args[0] == Py_None) Py_RETURN_NONE;
  const Tensor &x = THPVariable_Unpack(args[0]);
  const Tensor res = arg(args[1]), w = arg(args[2]), b = arg(args[3]), numbers = arg(args[4]);
  const int64_t site = number(args[5]), threshold = number(args[6]);
  const double eps = PyFloat_AsDouble(args[7]);
  if (eps == -1.0 && PyErr_Occurred()) throw python_error();
  const bool centred = truth(args[8]), want_q = truth(args[9]), want_stats = truth(args[10]), on_lines = truth(args[11]);
  if (x.dim() != 2 || !norm_takes(x, res, w, b, numbers)) Py_RETURN_NONE;
  NormOut out;
  {
    pybind11::gil_scoped_release no_gil;
    out = norm_pass(x, res, w, b, Dropped{numbers, site, threshold}, eps, centred, want_q, false, want_stats, on_lines);
  }
  return tuple_of({out.h, out.y, out.q, out.s, out.stats});
  END_HANDLE_TH_ERRORS
}

struct Dropout : torch::autograd::Function<Dropout> {
  struct Kept : torch::CustomClassHolder {   // of the forward pass: one entry of the context, where every one costs the host
    int64_t site, threshold;
    bool added;
    Stamp numbers;
    Kept(int64_t site, int64_t threshold, bool added, const Tensor &n) : site(site), threshold(threshold), added(added), numbers(n) {}
  };
  static Tensor pass(const Tensor &x, const Tensor &res, const Tensor &numbers, int64_t site, int64_t threshold) {
    const Tensor y = at::empty(x.sizes(), x.options());
    check(lib.l8_dropout(x.const_data_ptr(), caddr(res), y.mutable_data_ptr(), x.numel(), numbers.const_data_ptr<int64_t>(), site, threshold, stream_of(x.get_device())), "l8_dropout");
    return y;
  }
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const std::optional<Tensor> &res, const Tensor &numbers, int64_t site, int64_t threshold) {
    ctx->save_for_backward({numbers});
    ctx->saved_data["kept"] = c10::IValue::make_capsule(c10::make_intrusive<Kept>(site, threshold, res.has_value(), numbers));
    return pass(x, res.value_or(Tensor()), numbers, site, threshold);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const Tensor &g = grads[0];
    TORCH_CHECK(g.scalar_type() == at::kBFloat16, "dropout backward: bf16 gradients required, got ", g.scalar_type());
    const auto held = ctx->saved_data["kept"].toCapsule();
    const Kept &kept = static_cast<const Kept &>(*held);
    const Tensor saved = ctx->get_saved_variables()[0], numbers = saved.contiguous();
    kept.numbers.unchanged(saved, kept.added ? "dropout_add" : "dropout", kNumbers);
    Tensor gx;
    if (ctx->needs_input_grad(0)) {
      const c10::DeviceGuard guard(g.device());
      gx = once({pass(g.contiguous(), Tensor(), numbers, kept.site, kept.threshold)}, {learns(g)}, "dropout")[0];
    }
    return {gx, kept.added && ctx->needs_input_grad(1) ? g : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// dropout(x, residual, numbers, site, threshold) -> y, differentiable, or None
PyObject *dropout(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) throw std::runtime_error("dropout: 5 arguments");
  if (!tensors(args, 3) || args[0] == Py_None || args[2] == Py_None) Py_RETURN_NONE;
  const Tensor &x = THPVariable_Unpack(args[0]), &numbers = THPVariable_Unpack(args[2]);
  const Tensor res = arg(args[1]);
  const int64_t site = number(args[3]), threshold = number(args[4]);
  if (!x.is_cuda() || x.numel() < 1) Py_RETURN_NONE;
  const int device = x.get_device();
  if (!dense(x, at::kBFloat16, x.numel(), device) || (res.defined() && (!dense(res, at::kBFloat16, x.numel(), device) || res.sizes() != x.sizes())) || !is_numbers(numbers, device) ||
      c10::hip::current_device() != device)
    Py_RETURN_NONE;
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    if (at::GradMode::is_enabled()) refuse_captured({&x, &res}, res.defined() ? "dropout_add" : "dropout");
    y = Dropout::apply(x, maybe(res), numbers, site, threshold);
  }
  return wrap(y);
  END_HANDLE_TH_ERRORS
}

// ---- low-rank adapters ----

struct Bank {   // one factor, and whoever reads it
  const void *p;
  int64_t n, r, cols;
};
bool as_bank(const Tensor &t, int device, Bank &f) {
  if (!t.defined() || t.dim() != 3 || t.numel() < 1 || !dense(t, at::kBFloat16, t.numel(), device) || ((uintptr_t)t.const_data_ptr() % 16) != 0) return false;
  f = {t.const_data_ptr(), t.size(0), t.size(1), t.size(2)};
  return f.r % 8 == 0 && f.r >= 8 && f.r <= 128 && f.cols % 8 == 0;
}
// Factors as hooks on saved tensors may hand them back: dense and on 16-byte lines, or a copy that is.
Tensor bank_rows(const Tensor &t) {
  const Tensor c = t.contiguous();
  return ((uintptr_t)c.const_data_ptr() % 16) == 0 ? c : c.clone();
}
Tensor lowrank_h(const Rows &x, const Tensor &like, const Bank &f, const Tensor &order, const Tensor &starts, void *stream) {
  const int64_t splits = lib.l8_lowrank_splits(x.rows, f.n, f.r, f.cols);
  const Tensor h = at::empty({splits, x.rows, f.r}, like.options().dtype(at::kFloat));
  check(lib.l8_lowrank_shrink(x.p, x.rows, f.cols, x.ld, f.p, f.n, f.r, order.const_data_ptr<int>(), starts.const_data_ptr<int>(), h.mutable_data_ptr<float>(), splits, stream),
        "l8_lowrank_shrink");
  return h;
}
void lowrank_out(const Rows &y, const Tensor &h, const Tensor &scale, const Bank &f, const Tensor &order, const Tensor &starts, const Tensor &out, void *stream) {
  check(lib.l8_lowrank_expand(y.p, y.ld, h.const_data_ptr<float>(), h.size(0), scale.defined() ? scale.const_data_ptr<float>() : nullptr, f.p, h.size(1), f.cols, f.n, f.r,
                              order.const_data_ptr<int>(), starts.const_data_ptr<int>(), out.mutable_data_ptr(), f.cols, stream), "l8_lowrank_expand");
}

struct LowRank : torch::autograd::Function<LowRank> {
  static constexpr const char *kName = "add_lowrank";
  static Tensor forward(AutogradContext *ctx, const Tensor &y, const Tensor &x, const Tensor &a, const Tensor &b, const std::optional<Tensor> &scale, const Tensor &order,
                        const Tensor &starts, bool learn_x, bool learn_a, bool learn_b) {
    Bank fa, fb;
    TORCH_CHECK(as_bank(a, a.get_device(), fa) && as_bank(b, b.get_device(), fb), "add_lowrank: factors");
    void *stream = stream_of(x.get_device());
    const Tensor s = scale.value_or(Tensor()), h = lowrank_h(rows_of(x), x, fa, order, starts, stream), out = at::empty(y.sizes(), y.options());
    lowrank_out(rows_of(y), h, s, fb, order, starts, out, stream);
    ctx->save_for_backward({learn_a ? x : Tensor(), learn_x ? a : Tensor(), learn_x || learn_a ? b : Tensor(), learn_b ? h : Tensor(), s, order, starts});
    ctx->saved_data["like"] = x.sizes().vec();
    const Stamp stamp(order);
    ctx->saved_data["bank"] = std::vector<int64_t>{fa.n, fa.r, fa.cols, fb.cols, stamp.at, stamp.version};
    ctx->saved_data["learns"] = (int64_t)(learn_x | (learn_a << 1) | (learn_b << 2));
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto sizes = ctx->saved_data["bank"].toIntVector();
    Stamp(sizes[4], sizes[5]).unchanged(saved[5], kName, "the order of the tokens was");
    const Tensor gy = gradient(grads[0], kName);
    const int device = gy.get_device();
    const c10::DeviceGuard guard(gy.device());
    void *stream = stream_of(device);
    const int64_t n = sizes[0], r = sizes[1], K = sizes[2], N = sizes[3], learnt = ctx->saved_data["learns"].toInt();
    const bool need_y = ctx->needs_input_grad(0), need_x = ctx->needs_input_grad(1) && saved[1].defined(), need_a = ctx->needs_input_grad(2) && saved[0].defined(),
               need_b = ctx->needs_input_grad(3) && saved[3].defined();
    const Rows rg = rows_of(gy);
    const Tensor scale = saved[4].defined() ? saved[4].contiguous() : Tensor(), order = saved[5].contiguous(), starts = saved[6].contiguous();
    const Tensor x = need_a ? aligned_rows(saved[0]) : Tensor(), a = need_x ? bank_rows(saved[1]) : Tensor(), b = need_x || need_a ? bank_rows(saved[2]) : Tensor(),
                 h = need_b ? bank_rows(saved[3]) : Tensor();
    Tensor gh, gx, ga, gb;
    Bank f;
    const float *sp = scale.defined() ? scale.const_data_ptr<float>() : nullptr;
    const bool together = need_b && (need_x || need_a) && lib.l8_lowrank_outer_shrink_pays(rg.rows, r, N);
    if (need_x || need_a) {
      TORCH_CHECK(as_bank(b, device, f), "add_lowrank backward: factors");
      if (together) {
        gb = at::empty({n, r, N}, gy.options()), gh = at::empty({1, rg.rows, r}, gy.options().dtype(at::kFloat));
        const l8_lowrank_side one = {h.const_data_ptr<float>(), h.size(0), rg.p, rg.ld, N, gb.mutable_data_ptr()};
        const int64_t bytes = lib.l8_lowrank_outer_shrink_workspace(rg.rows, r, N);
        const Space ws(gy, bytes);
        check(lib.l8_lowrank_outer_shrink(&one, sp, f.p, gh.mutable_data_ptr<float>(), rg.rows, n, r, order.const_data_ptr<int>(), starts.const_data_ptr<int>(), ws.p(), bytes, stream),
              "l8_lowrank_outer_shrink");
      } else {
        gh = lowrank_h(rg, gy, f, order, starts, stream);
      }
    }
    if (need_x) {
      TORCH_CHECK(as_bank(a, device, f), "add_lowrank backward: factors");
      gx = at::empty(ctx->saved_data["like"].toIntVector(), gy.options());
      lowrank_out(Rows(), gh, scale, f, order, starts, gx, stream);
    }
    const bool side_b = need_b && !together;
    if (need_a || side_b) {
      l8_lowrank_side two[2] = {};
      if (need_a) {
        ga = at::empty({n, r, K}, gy.options());
        const Rows rx = rows_of(x);
        two[0] = {gh.const_data_ptr<float>(), gh.size(0), rx.p, rx.ld, K, ga.mutable_data_ptr()};
      }
      if (side_b) {
        gb = at::empty({n, r, N}, gy.options());
        two[1] = {h.const_data_ptr<float>(), h.size(0), rg.p, rg.ld, N, gb.mutable_data_ptr()};
      }
      const int64_t bytes = lib.l8_lowrank_outer_workspace(rg.rows, r, need_a ? K : 0, side_b ? N : 0);
      const Space ws(gy, bytes);
      check(lib.l8_lowrank_outer(two, sp, rg.rows, n, r, order.const_data_ptr<int>(), starts.const_data_ptr<int>(), ws.p(), bytes,
                                 stream), "l8_lowrank_outer");
    }
    const bool g = learns(grads[0]), lx = learnt & 1, la = learnt & 2, lb = learnt & 4;
    const variable_list made = once({gx, ga, gb}, {g || la || lb, g || lx || lb, g || lx || la}, kName);
    return {need_y ? grads[0] : Tensor(), made[0], made[1], made[2], Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// add_lowrank(y, x, a, b, scale, index, order, starts) -> out, differentiable, or None; order and starts (of one index): None where the index is to
// be looked at now
PyObject *add_lowrank(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) throw std::runtime_error("add_lowrank: 8 arguments");
  if (!tensors(args, 8) || args[0] == Py_None || args[1] == Py_None || args[2] == Py_None || args[3] == Py_None) Py_RETURN_NONE;
  const Tensor &y = THPVariable_Unpack(args[0]), &x = THPVariable_Unpack(args[1]), &a = THPVariable_Unpack(args[2]), &b = THPVariable_Unpack(args[3]);
  const Tensor scale = arg(args[4]), index = arg(args[5]);
  Tensor order = arg(args[6]), starts = arg(args[7]);
  if (!x.is_cuda()) Py_RETURN_NONE;
  const int device = x.get_device();
  Rows rx, ry;
  Bank fa, fb;
  if (!as_rows(x, device, rx) || !as_rows(y, device, ry) || !on_16_bytes(rx) || !on_16_bytes(ry) || rx.rows != ry.rows || !as_bank(a, device, fa) || !as_bank(b, device, fb) ||
      fa.n != fb.n || fa.r != fb.r || fa.cols != rx.cols || fb.cols != ry.cols || x.dim() != y.dim() || x.sizes().slice(0, x.dim() - 1) != y.sizes().slice(0, y.dim() - 1) ||
      (scale.defined() && (scale.dim() != 1 || !dense(scale, at::kFloat, fa.n, device) || (scale.requires_grad() && at::GradMode::is_enabled()))) || c10::hip::current_device() != device)
    Py_RETURN_NONE;
  const int64_t T = rx.rows;
  const bool planned = order.defined();
  if (planned ? !dense(order, at::kInt, T, device) || !starts.defined() || !dense(starts, at::kInt, fa.n + 3, device)
              : !index.defined() || !dense(index, index.scalar_type() == at::kLong ? at::kLong : at::kInt, T, device) || index.sizes() != x.sizes().slice(0, x.dim() - 1))
    Py_RETURN_NONE;
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    const bool grad = at::GradMode::is_enabled() && (learns(y) || learns(x) || learns(a) || learns(b));
    void *stream = stream_of(device);
    if (!grad && !planned) {
      out = at::empty(y.sizes(), y.options());
      const int64_t bytes = lib.l8_lowrank_add_workspace(T, fa.cols, fa.n, fa.r);
      const Space ws(x, bytes);
      check(lib.l8_lowrank_add(ry.p, ry.ld, rx.p, rx.ld, fa.p, fb.p, scale.defined() ? scale.const_data_ptr<float>() : nullptr, index.const_data_ptr(), index.scalar_type() == at::kLong,
                               T, fa.cols, fb.cols, fa.n, fa.r, out.mutable_data_ptr(), fb.cols, ws.p(), bytes, stream), "l8_lowrank_add");
    } else {
      if (grad) refuse_captured({&y, &x, &a, &b}, LowRank::kName);
      if (!planned) {
        order = at::empty({T}, x.options().dtype(at::kInt)), starts = at::empty({fa.n + 3}, x.options().dtype(at::kInt));
        check(lib.l8_lowrank_route(index.const_data_ptr(), index.scalar_type() == at::kLong, T, fa.n, order.mutable_data_ptr<int>(), starts.mutable_data_ptr<int>(), stream),
              "l8_lowrank_route");
      }
      out = LowRank::apply(y, x, a, b, maybe(scale), order, starts, grad && learns(x), grad && learns(a), grad && learns(b));
    }
  }
  return wrap(out);
  END_HANDLE_TH_ERRORS
}

// MXFP4 linear: what its two passes compute.
Tensor mx_forward(const Tensor &a, const Tensor &w, const Tensor &bias, bool need_a, bool need_w, Mx &at, Mx &wt) {
  const Rows ra = rows_of(a), rw = rows_of(w);
  const auto o = a.options();
  void *stream = stream_of(a.get_device());
  const Mx qa(ra.rows, ra.cols, o, true), qw(rw.rows, rw.cols, o, true);
  if (need_w) at = Mx(ra.cols, ra.rows, o, true);
  if (need_a) wt = Mx(rw.cols, rw.rows, o, true);
  const l8_mxfp4_cast two[2] = {{ra.p, ra.rows, ra.cols, ra.ld, qa.qp(), qa.ldq(), qa.sp(), qa.lds(), at.qp(), at.ldq(), at.sp(), at.lds()},
                                {rw.p, rw.rows, rw.cols, rw.ld, qw.qp(), qw.ldq(), qw.sp(), qw.lds(), wt.qp(), wt.ldq(), wt.sp(), wt.lds()}};
  check(lib.l8_cast_mxfp4_two(two, stream), "l8_cast_mxfp4_two");
  auto sizes = a.sizes().vec();
  sizes.back() = rw.rows;
  const Tensor y = at::empty(sizes, o);
  gemm_mx(rows_of(qa), rows_of(qw), bias, y, stream);
  return y;
}
bool mx_linear_takes(const Tensor &a, const Tensor &w, const Tensor &bias) {
  if (!a.is_cuda() || w.dim() != 2) return false;
  const int device = a.get_device();
  Rows ra, rw;
  return as_rows(a, device, ra) && as_rows(w, device, rw) && on_16_bytes(ra) && on_16_bytes(rw) && ra.cols == rw.cols && ra.cols % 16 == 0 && rw.rows % 16 == 0 &&
         c10::hip::current_device() == device && (!bias.defined() || dense(bias, at::kBFloat16, rw.rows, device));
}

struct Mxfp4Linear : torch::autograd::Function<Mxfp4Linear> {
  static Tensor forward(AutogradContext *ctx, const Tensor &a, const Tensor &w, const std::optional<Tensor> &bias, bool need_a, bool need_w) {
    Mx at, wt;
    const Tensor y = mx_forward(a, w, bias.value_or(Tensor()), need_a, need_w, at, wt);
    ctx->save_for_backward({at.q, at.s, wt.q, wt.s});
    ctx->saved_data["like"] = a.sizes().vec();
    ctx->saved_data["bias"] = bias.has_value();
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    auto saved = ctx->get_saved_variables();
    for (Tensor &t : saved) t = on_lines_of_16(t);
    const Tensor gy = gradient(grads[0], "mxfp4_linear");
    const int device = gy.get_device();
    const c10::DeviceGuard guard(c10::Device(c10::DeviceType::CUDA, (c10::DeviceIndex)device));
    const Rows rg = rows_of(gy);
    const auto o = gy.options();
    void *stream = stream_of(device);
    // (asked for when the graph was made, and again now: a part of the graph may be left out)
    const bool need_a = saved[2].defined() && ctx->needs_input_grad(0), need_w = saved[0].defined() && ctx->needs_input_grad(1);
    Mx rows, cols;
    MxRows a, w;
    TORCH_CHECK((!need_w || as_mx(saved[0], saved[1], device, a)) && (!need_a || as_mx(saved[2], saved[3], device, w)), "mxfp4_linear backward: saved copies");
    if (need_a) rows = Mx(rg.rows, rg.cols, o, true);
    if (need_w) cols = Mx(rg.cols, rg.rows, o, true);
    if (need_a || need_w) cast_mx(rg, rows, cols, stream);
    Tensor ga, gw, gbias;
    if (need_a) {
      ga = at::empty(ctx->saved_data["like"].toIntVector(), o);
      gemm_mx(rows_of(rows), w, Tensor(), ga, stream);
    }
    if (need_w) {
      gw = at::empty({rg.cols, a.rows}, o);
      gemm_mx(rows_of(cols), a, Tensor(), gw, stream);
    }
    if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2)) {
      gbias = at::empty({rg.cols}, o);
      const int64_t bytes = lib.l8_col_sum_workspace(rg.rows, rg.cols);
      const Space ws(gy, bytes);
      check(lib.l8_col_sum(rg.p, rg.rows, rg.cols, rg.ld, gbias.mutable_data_ptr(), ws.p(), bytes, stream), "l8_col_sum");
    }
    // (what was kept of the one operand says that the other learns)
    const bool gy_learns = learns(grads[0]);
    return once({ga, gw, gbias, Tensor(), Tensor()}, {gy_learns || saved[0].defined(), gy_learns || saved[2].defined(), gy_learns}, "mxfp4_linear");
  }
};

// mxfp4_linear(a, w, bias) -> y, differentiable, or None
PyObject *mxfp4_linear(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3) throw std::runtime_error("mxfp4_linear: 3 arguments");
  if (!tensors(args, 3) || args[0] == Py_None || args[1] == Py_None) Py_RETURN_NONE;
  const Tensor &a = THPVariable_Unpack(args[0]), &w = THPVariable_Unpack(args[1]);
  const Tensor bias = arg(args[2]);
  if (!mx_linear_takes(a, w, bias)) Py_RETURN_NONE;
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    const bool grad = at::GradMode::is_enabled();
    if (grad) refuse_captured({&a, &w, &bias}, "mxfp4_linear");
    y = Mxfp4Linear::apply(a, w, bias.defined() ? std::optional<Tensor>(bias) : std::nullopt, grad && a.requires_grad(), grad && w.requires_grad());
  }
  return wrap(y);
  END_HANDLE_TH_ERRORS
}

// key(tensor) -> bytes: equal for two tensors of the same memory, shape, strides, type, device and version, seen from the
// same current stream.
PyObject *key(PyObject *, PyObject *o) {
  HANDLE_TH_ERRORS
  const Tensor &t = THPVariable_Unpack(o);
  const int64_t dim = t.dim();
  c10::SmallVector<int64_t, 16> v;
  v.push_back(reinterpret_cast<int64_t>(t.const_data_ptr()));
  v.push_back((int64_t)t._version());
  v.push_back(((int64_t)t.scalar_type() << 32) | ((int64_t)t.device().type() << 16) | (uint16_t)t.device().index());
  v.push_back(t.is_cuda() ? reinterpret_cast<int64_t>(c10::hip::getCurrentHIPStream((c10::DeviceIndex)t.get_device()).stream()) : 0);
  for (int64_t i = 0; i < dim; ++i) {
    v.push_back(t.size(i));
    v.push_back(t.stride(i));
  }
  return PyBytes_FromStringAndSize(reinterpret_cast<const char *>(v.data()), (Py_ssize_t)(v.size() * sizeof(int64_t)));
  END_HANDLE_TH_ERRORS
}

// bind(handle of the loaded library, as ctypes holds it)
PyObject *bind(PyObject *, PyObject *o) {
  HANDLE_TH_ERRORS
  void *h = PyLong_AsVoidPtr(o);
  if (!h && PyErr_Occurred()) throw python_error();
#define L8_LOOK_UP(name)                                                   \
  lib.name = reinterpret_cast<decltype(lib.name)>(dlsym(h, #name));        \
  if (!lib.name) throw std::runtime_error("the library has no entry " #name);
  L8_ENTRIES(L8_LOOK_UP)
#undef L8_LOOK_UP
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", bind, METH_O, nullptr},
    {"key", key, METH_O, nullptr},
    {"linear_fwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear_fwd)), METH_FASTCALL, nullptr},
    {"linear_bwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear_bwd)), METH_FASTCALL, nullptr},
    {"cast_colwise_transposed", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cast_colwise_transposed)), METH_FASTCALL, nullptr},
    {"rmsnorm_fwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rmsnorm_fwd)), METH_FASTCALL, nullptr},
    {"rmsnorm_bwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rmsnorm_bwd)), METH_FASTCALL, nullptr},
    {"qkv_fwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(qkv_fwd)), METH_FASTCALL, nullptr},
    {"shared_bwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(shared_bwd)), METH_FASTCALL, nullptr},
    {"swiglu_fwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(swiglu_fwd)), METH_FASTCALL, nullptr},
    {"swiglu_bwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(swiglu_bwd)), METH_FASTCALL, nullptr},
    {"add_rmsnorm_fwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(add_rmsnorm_fwd)), METH_FASTCALL, nullptr},
    {"rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rotary)), METH_FASTCALL, nullptr},
    {"cast_mxfp4", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cast_mxfp4)), METH_FASTCALL, nullptr},
    {"mxfp4_to_bf16", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(mxfp4_to_bf16)), METH_FASTCALL, nullptr},
    {"add_rmsnorm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(add_rmsnorm)), METH_FASTCALL, nullptr},
    {"rotary_pair", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rotary_pair)), METH_FASTCALL, nullptr},
    {"norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(norm)), METH_FASTCALL, nullptr},
    {"norm_fwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(norm_fwd)), METH_FASTCALL, nullptr},
    {"dropout", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(dropout)), METH_FASTCALL, nullptr},
    {"add_lowrank", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(add_lowrank)), METH_FASTCALL, nullptr},
    {"refuse_captured", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(refuse_captured_py)), METH_FASTCALL, nullptr},
    {"mxfp4_packed", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(mxfp4_packed)), METH_FASTCALL, nullptr},
    {"mxfp4_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(mxfp4_linear)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() { return PyModule_Create(&module_def); }
