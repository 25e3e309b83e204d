// serving_ext.cpp — Python entry points of the serving operators.
//
// A call for a few new tokens takes the GPU 3 to 8 us, less than checking its
// tensors and passing two dozen arguments takes in Python (14 to 18 us a call).
// So the whole call is made here: checks, views, outputs, workspace, launch
// through the C ABI of libvmscan.so.  The documentation of the operators is at
// their Python functions (serving.py), which only forward here.
//
// Exceptions are the Python ones: TypeError, ValueError, RuntimeError.
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <nvtx3/nvToolsExt.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../include/vmscan.h"

namespace {

constexpr int64_t kMaxRows = int64_t(1) << 30;
constexpr int64_t kState = 16;

PyObject* g_batch_type = nullptr;     // RequestBatch
PyObject* g_adapters_type = nullptr;  // LoraAdapters

// Interned attribute and method names.
struct Names {
  PyObject *tokens, *index, *count, *max_slot, *max_adapter, *single_tokens, *table, *a, *b, *scale;
  PyObject *scan, *step, *conv, *lora;
};
Names g_names;

#define VALUE(cond, ...) TORCH_CHECK_VALUE(cond, where, ": ", __VA_ARGS__)
#define TYPE(cond, ...) TORCH_CHECK_TYPE(cond, where, ": ", __VA_ARGS__)
#define RUNTIME(cond, ...) TORCH_CHECK(cond, where, ": ", __VA_ARGS__)

struct Ref {  // owned Python reference
  PyObject* p;
  explicit Ref(PyObject* o) : p(o) {
    if (p == nullptr) throw python_error();
  }
  ~Ref() { Py_DECREF(p); }
  Ref(const Ref&) = delete;
  Ref& operator=(const Ref&) = delete;
};

int64_t int_attr(PyObject* o, PyObject* name) {
  Ref r(PyObject_GetAttr(o, name));
  const int64_t v = PyLong_AsLongLong(r.p);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

struct Range {  // profiler range of the entry point
  explicit Range(const char* name) { nvtxRangePushA(name); }
  ~Range() { nvtxRangePop(); }
};

std::string shape_of(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}

const at::Tensor& tensor(const char* where, const char* name, PyObject* o) {
  RUNTIME(THPVariable_Check(o), "`", name, "` must be a CUDA tensor (there is no CPU path)");
  return THPVariable_Unpack(o);
}

// A tensor on x's device.
const at::Tensor& beside(const char* where, const char* name, PyObject* o, int64_t index) {
  const at::Tensor& t = tensor(where, name, o);
  RUNTIME(t.is_cuda() && t.get_device() == index, "`", name,
          "` must be a CUDA tensor on x's device (there is no CPU path)");
  return t;
}

void shaped(const char* where, const char* name, const at::Tensor& t, int64_t rows, int64_t cols) {
  VALUE(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols, name, " must be (", rows, ", ", cols, "), got ",
        shape_of(t));
}

// Refuses inputs whose derivatives a caller asks for: reverse mode (off under
// no_grad) and forward mode (dual tensors; not off there).
void no_grad(const char* where, std::initializer_list<const at::Tensor*> ts) {
  const c10::AutogradState& on = c10::AutogradState::get_tls_state();
  for (const at::Tensor* t : ts) {
    if (t == nullptr) continue;
    RUNTIME(!on.get_grad_mode() || !t->requires_grad(),
            "a serving operator has no gradient; call it under torch.no_grad()");
    RUNTIME(!on.get_fw_grad_mode() || !t->_fw_grad(0).defined(), "a serving operator has no forward-mode derivative");
  }
}

// Notes for autograd that a kernel has written t: a graph that has saved it
// must not use the new values.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

struct Batch {
  PyObject* self;
  int64_t tokens, index;
};

Batch batch_of(const char* where, PyObject* o) {
  const int is = PyObject_IsInstance(o, g_batch_type);
  if (is < 0) throw python_error();
  TYPE(is, "`batch` must be a RequestBatch, got ", Py_TYPE(o)->tp_name);
  return {o, int_attr(o, g_names.tokens), int_attr(o, g_names.index)};
}

const at::Tensor& rows_of(const char* where, const Batch& b, PyObject* o) {
  const at::Tensor& x = tensor(where, "x", o);
  RUNTIME(x.is_cuda(), "inputs must be CUDA tensors (there is no CPU path)");
  VALUE(x.get_device() == b.index, "the batch is for device ", b.index, ", x is on ", x.device());
  VALUE(x.dim() == 2, "x must be (rows, channels), got ", shape_of(x));
  TYPE(x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16, "x must be fp32 or bf16, got ",
       x.scalar_type());
  VALUE(x.size(0) >= b.tokens, "x has ", x.size(0), " rows, the batch's requests have ", b.tokens);
  VALUE(x.size(0) <= kMaxRows, "x has ", x.size(0), " rows (at most ", kMaxRows, ")");
  return x;
}

void check_state(const char* where, const at::Tensor& s, const Batch& b, int64_t d1, int64_t d2, at::ScalarType dtype) {
  VALUE(s.dim() == 3 && s.size(1) == d1 && s.size(2) == d2 && s.scalar_type() == dtype, "state must be (slots, ", d1,
        ", ", d2, ") ", dtype, ", got ", shape_of(s), " ", s.scalar_type());
  const int64_t most = int_attr(b.self, g_names.max_slot);
  VALUE(most < s.size(0), "the batch uses slot ", most, ", the state has ", s.size(0), " slots");
  VALUE(s.is_contiguous() && reinterpret_cast<uintptr_t>(s.data_ptr()) % 16 == 0,
        "state must be contiguous and 16-byte aligned (it is updated in place)");
}

// t (rows, columns) in `dtype` with unit column stride: t itself when it is so,
// else a copy kept in `keep`.
const at::Tensor& as_rows(const at::Tensor& t, at::ScalarType dtype, at::Tensor& keep) {
  if (t.scalar_type() == dtype && (t.stride(1) == 1 || t.size(1) <= 1)) return t;
  keep = t.detach().to(dtype).contiguous();
  return keep;
}

// A parameter as contiguous, 16-byte aligned fp32.
const at::Tensor& as_param(const at::Tensor& t, at::Tensor& keep) {
  const auto aligned = [](const at::Tensor& v) { return reinterpret_cast<uintptr_t>(v.data_ptr()) % 16 == 0; };
  if (t.scalar_type() == at::kFloat && t.is_contiguous() && aligned(t)) return t;
  keep = t.detach().to(at::kFloat).contiguous();
  if (!aligned(keep)) keep = keep.clone();
  return keep;
}

// Output rows; those behind the last request are zero.
at::Tensor out_rows(const at::Tensor& x, const Batch& b) {
  at::Tensor y = at::empty({x.size(0), x.size(1)}, x.options().requires_grad(false));
  if (x.size(0) > b.tokens) y.narrow(0, b.tokens, x.size(0) - b.tokens).zero_();
  return y;
}

// The batch's device table of a kind for a stream: its address and up to six
// numbers (RequestBatch._table makes and keeps it).
struct Table {
  int64_t ptr;
  int64_t info[6];
};

Table table_of(const Batch& b, PyObject* kind, void* stream, int64_t arg, int64_t slots) {
  const bool capturing = c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
  Ref s(PyLong_FromVoidPtr(stream)), a(PyLong_FromLongLong(arg)), n(PyLong_FromLongLong(slots));
  PyObject* args[6] = {b.self, kind, s.p, a.p, capturing ? Py_True : Py_False, n.p};
  Ref r(PyObject_VectorcallMethod(g_names.table, args, 6, nullptr));
  TORCH_CHECK(PyTuple_Check(r.p) && PyTuple_GET_SIZE(r.p) <= 7, "RequestBatch._table returned no table");
  Table t{};
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(r.p); ++i) {
    const int64_t v = PyLong_AsLongLong(PyTuple_GET_ITEM(r.p, i));
    if (v == -1 && PyErr_Occurred()) throw python_error();
    (i == 0 ? t.ptr : t.info[i - 1]) = v;
  }
  return t;
}

const int32_t* i32(int64_t p) { return reinterpret_cast<const int32_t*>(p); }

void check(int rc, const char* where, const char* entry) {
  if (rc == VMSCAN_OK) return;
  const std::string detail = vmscan_last_error();
  RUNTIME(false, entry, ": vmscan status ", rc, ": ", vmscan_strerror(rc), detail.empty() ? "" : " (" + detail + ")");
}

vmscan_stream_t stream_of(const Batch& b) {
  return reinterpret_cast<vmscan_stream_t>(c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(b.index)).stream());
}

PyObject* scan(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const char* where = "selective_scan_cached_cuda";
  TYPE(nargs == 9, "takes 9 arguments");
  const Batch b = batch_of(where, args[7]);
  const at::Tensor& x = rows_of(where, b, args[0]);
  const int64_t rows = x.size(0), dn = x.size(1);
  const at::Tensor& delta = beside(where, "delta", args[1], b.index);
  const at::Tensor& A = beside(where, "A", args[2], b.index);
  const at::Tensor& B = beside(where, "B", args[3], b.index);
  const at::Tensor& C = beside(where, "C", args[4], b.index);
  const at::Tensor& D = beside(where, "D", args[5], b.index);
  const at::Tensor* z = args[8] == Py_None ? nullptr : &beside(where, "z", args[8], b.index);
  shaped(where, "delta", delta, rows, dn);
  shaped(where, "A", A, dn, kState);
  shaped(where, "B", B, rows, kState);
  shaped(where, "C", C, rows, kState);
  VALUE(D.dim() == 1 && D.size(0) == dn, "D must be (", dn, ",), got ", shape_of(D));
  if (z != nullptr) shaped(where, "z", *z, rows, dn);
  const at::Tensor& state = beside(where, "state", args[6], b.index);
  check_state(where, state, b, dn, kState, at::kFloat);
  no_grad(where, {&x, &delta, &A, &B, &C, &D, &state, z});
  if (dn == 0) return THPVariable_Wrap(at::zeros_like(x));
  const c10::cuda::OptionalCUDAGuard guard{c10::Device(c10::kCUDA, c10::DeviceIndex(b.index))};
  const at::ScalarType dt = x.scalar_type();
  const int bf16 = dt == at::kBFloat16;
  at::Tensor k0, k1, k2, k3, k4, k5, k6;
  const at::Tensor &x_ = as_rows(x, dt, k0), &d_ = as_rows(delta, dt, k1), &B_ = as_rows(B, dt, k2),
                   &C_ = as_rows(C, dt, k3), &A_ = as_param(A, k4), &D_ = as_param(D, k5);
  const at::Tensor* z_ = z == nullptr ? nullptr : &as_rows(*z, dt, k6);
  at::Tensor y = out_rows(x, b);
  vmscan_stream_t stream = stream_of(b);
  Range range(where);
  const void* zp = z_ == nullptr ? nullptr : z_->data_ptr();
  const int64_t ldz = z_ == nullptr ? 0 : z_->stride(0);
  Ref single(PyObject_GetAttr(b.self, g_names.single_tokens));
  if (single.p == Py_True) {
    const Table t = table_of(b, g_names.step, stream, 0, state.size(0));
    check(vmscan_cached_step(b.tokens, dn, kState, bf16, x_.data_ptr(), x_.stride(0), d_.data_ptr(), d_.stride(0),
                             static_cast<const float*>(A_.data_ptr()), B_.data_ptr(), B_.stride(0), C_.data_ptr(),
                             C_.stride(0), static_cast<const float*>(D_.data_ptr()), zp, ldz, y.data_ptr(), dn,
                             static_cast<float*>(state.data_ptr()), state.size(0), i32(t.ptr), i32(t.ptr) + t.info[0],
                             stream),
          where, "vmscan_cached_step");
    written(state);
    return THPVariable_Wrap(y);
  }
  const Table t = table_of(b, g_names.scan, stream, 2 * dn + bf16, state.size(0));
  const int64_t n = t.info[0], chains = t.info[2], carry_rows = t.info[3];
  at::Tensor ws;
  int64_t ws_bytes = 0;
  if (carry_rows > 0) {
    ws_bytes = vmscan_cached_scan_workspace_bytes(dn, carry_rows);
    if (ws_bytes < 0) check(int(-ws_bytes), where, "vmscan_cached_scan_workspace_bytes");
    ws = at::empty({ws_bytes}, x.options().dtype(at::kByte).requires_grad(false));
  }
  check(vmscan_cached_scan(rows, dn, kState, bf16, x_.data_ptr(), x_.stride(0), d_.data_ptr(), d_.stride(0),
                           static_cast<const float*>(A_.data_ptr()), B_.data_ptr(), B_.stride(0), C_.data_ptr(),
                           C_.stride(0), static_cast<const float*>(D_.data_ptr()), zp, ldz, y.data_ptr(), dn,
                           static_cast<float*>(state.data_ptr()), state.size(0), i32(t.ptr), n, t.info[1],
                           chains > 0 ? i32(t.ptr) + 8 * n : nullptr, chains, carry_rows, t.info[4], int(t.info[5]),
                           ws.defined() ? ws.data_ptr() : nullptr, size_t(ws_bytes), stream),
        where, "vmscan_cached_scan");
  written(state);
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

PyObject* conv(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const char* where = "conv1d_silu_cached_cuda";
  TYPE(nargs == 5, "takes 5 arguments");
  const Batch b = batch_of(where, args[4]);
  const at::Tensor& x = rows_of(where, b, args[0]);
  const int64_t rows = x.size(0), c = x.size(1);
  const at::Tensor& w = beside(where, "weight", args[1], b.index);
  const at::Tensor& bias = beside(where, "bias", args[2], b.index);
  VALUE(w.dim() == 3 && w.size(0) == c && w.size(2) == 1 && bias.dim() == 1 && bias.size(0) == c, "bad shapes x=",
        shape_of(x), " weight=", shape_of(w), " bias=", shape_of(bias));
  const int64_t k = w.size(1);
  VALUE(k >= 1 && k <= 8, "kernel size ", k, " (1 to 8)");
  const at::Tensor& state = beside(where, "state", args[3], b.index);
  check_state(where, state, b, k - 1, c, x.scalar_type());
  no_grad(where, {&x, &w, &bias, &state});
  if (c == 0) return THPVariable_Wrap(at::zeros_like(x));
  const c10::cuda::OptionalCUDAGuard guard{c10::Device(c10::kCUDA, c10::DeviceIndex(b.index))};
  at::Tensor k0, k1, k2;
  const at::Tensor &x_ = as_rows(x, x.scalar_type(), k0), &w_ = as_param(w, k1), &b_ = as_param(bias, k2);
  at::Tensor out = out_rows(x, b);
  vmscan_stream_t stream = stream_of(b);
  Range range(where);
  const Table t = table_of(b, g_names.conv, stream, c, state.size(0));
  check(vmscan_cached_conv1d_silu(rows, c, k, x.scalar_type() == at::kBFloat16, x_.data_ptr(), x_.stride(0),
                                  static_cast<const float*>(w_.data_ptr()), static_cast<const float*>(b_.data_ptr()),
                                  out.data_ptr(), c, state.data_ptr(), state.size(0), i32(t.ptr), t.info[0], stream),
        where, "vmscan_cached_conv1d_silu");
  written(state);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// Whether an element of `out` may also be one of t (both (rows, columns) with
// unit column stride; column slices of the same wider rows do not collide).
bool collide(const at::Tensor& out, const at::Tensor& t) {
  const auto span = [](const at::Tensor& v) {
    const char* p = static_cast<const char*>(v.data_ptr());
    return std::make_pair(p, p + ((v.size(0) - 1) * v.stride(0) + v.size(1)) * int64_t(v.element_size()));
  };
  const auto a = span(out), b = span(t);
  if (a.second <= b.first || b.second <= a.first) return false;
  const int64_t e = out.element_size(), ld = out.stride(0), off = b.first - a.first;
  if (int64_t(t.element_size()) == e && t.stride(0) == ld && ld > 0 && off % e == 0) {
    const int64_t shift = ((off / e) % ld + ld) % ld;  // columns between the two slices
    return !(out.size(1) <= shift && shift + t.size(1) <= ld);
  }
  return true;
}

PyObject* lora(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const char* where = "lora_add_cuda";
  TYPE(nargs == 5, "takes 5 arguments");
  const Batch b = batch_of(where, args[3]);
  const at::Tensor& x = rows_of(where, b, args[1]);
  const int is = PyObject_IsInstance(args[2], g_adapters_type);
  if (is < 0) throw python_error();
  TYPE(is, "`adapters` must be LoraAdapters, got ", Py_TYPE(args[2])->tp_name);
  Ref ra(PyObject_GetAttr(args[2], g_names.a)), rb(PyObject_GetAttr(args[2], g_names.b)),
      rs(PyObject_GetAttr(args[2], g_names.scale));
  const at::Tensor &a = tensor(where, "adapters", ra.p), &bb = tensor(where, "adapters", rb.p),
                   &scale = tensor(where, "adapters", rs.p);
  // padded storage: a (count, padded rank, lda), b (count, d_out, padded rank)
  VALUE(a.dim() == 3 && bb.dim() == 3 && scale.dim() == 1 && bb.size(0) == a.size(0) && scale.size(0) == a.size(0) &&
            bb.size(2) == a.size(1) && a.size(1) <= bb.stride(1) && a.size(2) <= a.stride(1) && a.stride(2) == 1 &&
            bb.stride(2) == 1 && a.stride(0) == bb.stride(1) * a.stride(1) && bb.stride(0) == bb.size(1) * bb.stride(1) &&
            a.storage_offset() == 0 && bb.storage_offset() == 0 &&
            int64_t(a.storage().nbytes()) >= a.size(0) * a.stride(0) * int64_t(a.element_size()) &&
            int64_t(bb.storage().nbytes()) >= bb.size(0) * bb.stride(0) * int64_t(bb.element_size()) &&
            scale.is_contiguous() && bb.scalar_type() == a.scalar_type() && scale.scalar_type() == at::kFloat &&
            a.is_cuda() && bb.device() == a.device() && scale.device() == a.device(),
        "the adapters' tensors are not as LoraAdapters made them");
  const int64_t rows = x.size(0), count = a.size(0), rank = bb.stride(1), d_in = a.size(2), d_out = bb.size(1);
  const at::Tensor& base = beside(where, "base", args[0], b.index);
  const at::Tensor* given = args[4] == Py_None ? nullptr : &beside(where, "out", args[4], b.index);
  shaped(where, "x", x, rows, d_in);
  shaped(where, "base", base, rows, d_out);
  if (given != nullptr) shaped(where, "out", *given, rows, d_out);
  const at::ScalarType dt = a.scalar_type();
  for (const auto& p : {std::make_pair("x", &x), std::make_pair("base", &base), std::make_pair("out", given)})
    TYPE(p.second == nullptr || p.second->scalar_type() == dt, p.first, " is ", p.second->scalar_type(),
         ", the adapters are ", dt);
  no_grad(where, {&x, &base, given});
  VALUE(a.get_device() == b.index, "the adapters are on ", a.device(), ", x is on ", x.device());
  const int64_t most = int_attr(b.self, g_names.max_adapter);
  VALUE(most >= -1, "the batch was made without adapters");
  VALUE(most < count, "the batch uses adapter ", most, ", there are ", count);
  const c10::cuda::OptionalCUDAGuard guard{c10::Device(c10::kCUDA, c10::DeviceIndex(b.index))};
  at::Tensor k0, k1;
  const at::Tensor& x_ = as_rows(x, dt, k0);
  bool in_place = false;
  if (given != nullptr && rows > 0) {
    in_place = given->data_ptr() == base.data_ptr() && given->strides() == base.strides();
    VALUE((given->stride(1) == 1 || d_out == 1) && (rows == 1 || given->stride(0) >= d_out),
          "out must have unit column stride and rows that do not overlap");
  }
  const at::Tensor& base_ = in_place ? base : as_rows(base, dt, k1);
  if (given != nullptr && rows > 0)
    VALUE(!collide(*given, x_) && (in_place || !collide(*given, base_)),
          "out overlaps x or base (it may only be base itself)");
  at::Tensor out = given != nullptr ? *given : at::empty({rows, d_out}, base.options().requires_grad(false));
  if (rows > b.tokens && !in_place)
    out.narrow(0, b.tokens, rows - b.tokens).copy_(base_.narrow(0, b.tokens, rows - b.tokens));
  if (b.tokens > 0) {
    vmscan_stream_t stream = stream_of(b);
    Range range(where);
    const Table t = table_of(b, g_names.lora, stream, count, 0);
    const int64_t tiles = t.info[0];
    check(vmscan_lora_add(rows, d_in, d_out, rank, count, dt == at::kBFloat16, x_.data_ptr(), x_.stride(0), a.data_ptr(),
                          a.stride(1), bb.data_ptr(), static_cast<const float*>(scale.data_ptr()), base_.data_ptr(), base_.stride(0),
                          out.data_ptr(), out.stride(0), i32(t.ptr) + 4 * tiles, b.tokens, i32(t.ptr), tiles, stream),
          where, "vmscan_lora_add");
    if (given != nullptr) written(out);
  }
  if (given != nullptr) {
    Py_INCREF(args[4]);
    return args[4];
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

PyObject* setup(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 2) {
    PyErr_SetString(PyExc_TypeError, "setup takes the RequestBatch and LoraAdapters types");
    return nullptr;
  }
  Py_INCREF(args[0]);
  Py_INCREF(args[1]);
  g_batch_type = args[0];
  g_adapters_type = args[1];
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"setup", reinterpret_cast<PyCFunction>(setup), METH_FASTCALL, "setup(RequestBatch, LoraAdapters)"},
    {"scan", reinterpret_cast<PyCFunction>(scan), METH_FASTCALL, "serving.selective_scan_cached_cuda"},
    {"conv", reinterpret_cast<PyCFunction>(conv), METH_FASTCALL, "serving.conv1d_silu_cached_cuda"},
    {"lora", reinterpret_cast<PyCFunction>(lora), METH_FASTCALL, "serving.lora_add_cuda"},
    {nullptr, nullptr, 0, nullptr}};

// The PyTorch and the interpreter that this was compiled for: build.py looks for
// it and compiles anew for others.
const char kBuiltFor[] = VMSCAN_BUILT_FOR;

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_serving_ext", "Calls of the serving operators.", -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__serving_ext(void) {
  struct {
    PyObject** at;
    const char* name;
  } const names[] = {{&g_names.tokens, "tokens"},         {&g_names.index, "index"},
                     {&g_names.count, "count"},           {&g_names.max_slot, "max_slot"},
                     {&g_names.max_adapter, "max_adapter"}, {&g_names.single_tokens, "single_tokens"},
                     {&g_names.table, "_table"},          {&g_names.a, "a"},
                     {&g_names.b, "b"},                   {&g_names.scale, "scale"},
                     {&g_names.scan, "scan"},             {&g_names.step, "step"},
                     {&g_names.conv, "conv"},             {&g_names.lora, "lora"}};
  for (const auto& n : names)
    if ((*n.at = PyUnicode_InternFromString(n.name)) == nullptr) return nullptr;
  PyObject* m = PyModule_Create(&g_module);
  if (m != nullptr && PyModule_AddStringConstant(m, "built_for", kBuiltFor) != 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
