// Python entry of the operators whose calls cost more on the host than on the GPU: label probabilities
// (ldm_label_log_probs, ldm_label_log_probs_bwd) and gradient norms over tensor lists (ldm_grad_norm).
//
// Checks of arguments, allocation of outputs and the walk over a list of tensors run here, in C++ on torch's
// tensors; the launches are the C ABI's, at the addresses that init() was given (the library that ctypes loaded).
// A call with 686 gradients takes about 30 us here and 400 us as Python loops over them; label_log_probs 3 us
// instead of 15.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/Functions.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <array>
#include <cmath>
#include <optional>
#include <vector>

#include "../../include/ldmseg_hip.h"

namespace {

size_t (*p_fwd_ws)(const ldm_label_probs_params*);
int (*p_fwd)(const ldm_label_probs_params*, ldm_stream_t);
int (*p_bwd)(const ldm_label_probs_bwd_params*, ldm_stream_t);
size_t (*p_norm_ws)(const int64_t*, int);
int (*p_norm)(const void* const*, const int64_t*, const uint8_t*, int, int, double, int, float*, void*, int64_t,
              ldm_stream_t);
const char* (*p_status)(int);

// The launches of a call go to its tensors' device, on that device's current stream.
struct OnDevice {
  c10::DeviceIndex was, now;
  explicit OnDevice(const at::Device& d) : was(c10::hip::current_device()), now(d.index()) {
    if (now != was) c10::hip::set_device(now);
  }
  ~OnDevice() {
    if (now != was) c10::hip::set_device(was);
  }
  ldm_stream_t stream() const { return reinterpret_cast<ldm_stream_t>(c10::hip::getCurrentHIPStream(now).stream()); }
};

void check_status(int rc, const char* what) {
  TORCH_CHECK(rc == LDM_OK, what, " failed: ", p_status(rc), " (status ", rc, ")");
}
int dtype_code(const at::Tensor& t, const char* what) {
  if (t.scalar_type() == at::kFloat) return LDM_F32;
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16, "unsupported ", what, " ", t.scalar_type(),
                   ": the HIP path computes in float32 or bfloat16");
  return LDM_BF16;
}
void check_gpu(const at::Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "ldmseg HIP ops take GPU tensors only (no CPU fallback); got a tensor on ", t.device());
}
const at::Tensor& tensor_of(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
  return THPVariable_Unpack(o);
}
int64_t int_of(PyObject* o, const char* name) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    TORCH_CHECK_TYPE(false, name, " must be an integer of 64 bits");
  }
  return v;
}
double double_of(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    TORCH_CHECK_TYPE(false, name, " must be a number");
  }
  return v;
}

// ------------------------------------------------------------------------------------ label probabilities
// Every dim of x but `dim` as three strided dims, merged on either side of the class dim and never across it; a
// tensor with more than three left is copied.  `out`, if any, is walked by the same sizes.
struct Positions {
  at::Tensor x;
  std::optional<at::Tensor> out;
  std::array<int64_t, 3> n{1, 1, 1}, s{0, 0, 0}, o{0, 0, 0};
  int64_t inner = 1;               // positions behind the class dim
};
Positions positions_of(const at::Tensor& x, int64_t dim, bool with_out) {
  Positions p;
  p.x = x;
  if (with_out) p.out = at::empty_like(x);
  for (int turn = 0;; ++turn) {
    std::vector<std::array<int64_t, 3>> d;          // size, stride, out's stride
    const auto sizes = p.x.sizes(), st = p.x.strides();
    p.inner = 1;
    auto side = [&](int64_t lo, int64_t hi) {
      const size_t first = d.size();
      for (int64_t i = lo; i < hi; ++i) {
        const int64_t n = sizes[i], s = st[i], o = with_out ? p.out->stride(i) : 0;
        if (n == 1) continue;
        if (d.size() > first && d.back()[1] == n * s && (!with_out || d.back()[2] == n * o))
          d.back() = {d.back()[0] * n, s, o};
        else
          d.push_back({n, s, o});
      }
    };
    side(0, dim);
    side(dim + 1, p.x.dim());
    for (int64_t i = dim + 1; i < p.x.dim(); ++i) p.inner *= sizes[i];
    if (d.size() > 3 && turn == 0) {
      p.x = x.contiguous();
      if (with_out) p.out = at::empty_like(p.x);
      continue;
    }
    for (size_t i = 0; i < d.size(); ++i) {
      const size_t at = 3 - d.size() + i;
      p.n[at] = d[i][0];
      p.s[at] = d[i][1];
      p.o[at] = d[i][2];
    }
    return p;
  }
}

// what a lazily negated view shows, not what its memory holds
at::Tensor logits_of(PyObject* o) { return tensor_of(o, "logits").resolve_neg(); }

int64_t class_dim(const at::Tensor& logits, int64_t dim) {
  const int64_t nd = logits.dim();
  TORCH_CHECK_VALUE(nd >= 2, "logits need a class dim and at least one position dim");
  TORCH_CHECK_VALUE(dim >= -nd && dim < nd, "class dim ", dim, " is outside logits of ", nd, " dims");
  if (dim < 0) dim += nd;
  TORCH_CHECK_VALUE(logits.size(dim) > 0, "logits have no classes");
  return dim;
}
float temperature_of(PyObject* o) {
  const double t = double_of(o, "temperature");
  TORCH_CHECK_VALUE(t >= 1e-4 && t <= 1e4, "temperature must be in [1e-4, 1e4], got ", t);
  return (float)t;
}
at::DimVector without(at::IntArrayRef sizes, int64_t dim) {
  at::DimVector v(sizes.begin(), sizes.end());
  v.erase(v.begin() + dim);
  return v;
}

// a class mask [C] or [logits.shape[0], C]: its row stride and the positions to a row
struct Mask {
  at::Tensor t;
  int64_t stride = 0, div = 1;
  const void* ptr() const { return t.defined() ? t.data_ptr() : nullptr; }
};
Mask mask_of(PyObject* o, const at::Tensor& logits, int64_t dim, int64_t positions) {
  Mask m;
  if (o == Py_None) return m;
  const at::Tensor& t = tensor_of(o, "class_mask");
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBool && t.device() == logits.device(),
                   "class_mask must be a bool tensor on the logits' device");
  const int64_t C = logits.size(dim), B = logits.size(0);
  const bool rows = dim != 0 && t.dim() == 2 && t.size(0) == B && t.size(1) == C;
  TORCH_CHECK_VALUE(rows || (t.dim() == 1 && t.size(0) == C), "class_mask must be [", C, "] or [", B, ", ", C,
                    "] (classes, or the logits' first dim by classes), got ", t.sizes());
  m.t = t.contiguous();
  m.stride = rows ? C : 0;
  m.div = std::max<int64_t>(1, rows ? positions / std::max<int64_t>(1, B) : positions);
  return m;
}

PyObject* wrap_or_none(const at::Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}

// (logits, labels | None, dim, topk, temperature, ignore_label | None, class_mask | None, want_stats)
//   -> (log_prob | None, entropy, top_log_probs | None, top_ids | None, stats | None)
PyObject* label_log_probs(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(nargs == 8 && p_fwd, "label_log_probs: 8 arguments after init()");
  const at::Tensor logits = logits_of(args[0]);
  const int code = dtype_code(logits, "dtype");
  const int64_t dim = class_dim(logits, int_of(args[2], "dim"));
  const int64_t topk = int_of(args[3], "topk"), C = logits.size(dim);
  const float temperature = temperature_of(args[4]);
  const int64_t most = std::min<int64_t>(C, LDM_LABEL_TOPK_MAX);
  TORCH_CHECK_VALUE(topk >= 0 && topk <= most, "topk must be in [0, ", most, "], got ", topk);
  const at::DimVector shape = without(logits.sizes(), dim);
  at::Tensor labels, log_prob, top_lp, top_id, stats, workspace;
  if (args[1] != Py_None) {
    labels = tensor_of(args[1], "labels");
    TORCH_CHECK_TYPE(labels.scalar_type() == at::kLong && labels.device() == logits.device(),
                     "labels must be an int64 tensor on the logits' device");
    TORCH_CHECK_VALUE(labels.sizes() == at::IntArrayRef(shape), "labels must be ", at::IntArrayRef(shape), ", got ",
                      labels.sizes());
    labels = labels.contiguous();
  }
  int64_t count = 1;
  for (int64_t n : shape) count *= n;
  const Mask mask = mask_of(args[6], logits, dim, count);
  const bool has_ignore = args[5] != Py_None;
  const int64_t ignore = has_ignore ? int_of(args[5], "ignore_label") : 0;
  const int want_stats = PyObject_IsTrue(args[7]);
  check_gpu(logits);
  const Positions pos = positions_of(logits, dim, false);
  const auto f32 = logits.options().dtype(at::kFloat).memory_format(std::nullopt).requires_grad(false);
  const at::Tensor entropy = at::empty(shape, f32);
  if (labels.defined()) log_prob = at::empty(shape, f32);
  if (topk) {
    at::DimVector top(logits.sizes().begin(), logits.sizes().end());
    top[dim] = topk;
    top_lp = at::empty(top, f32);
    top_id = at::empty(top, f32.dtype(at::kInt));
  }
  if (want_stats) {
    at::DimVector four(shape);
    four.insert(four.begin(), 4);
    stats = at::empty(four, f32);
  }
  if (count) {
    ldm_label_probs_params p = {};
    p.logits = pos.x.data_ptr();
    p.n0 = pos.n[0]; p.n1 = pos.n[1]; p.n2 = pos.n[2];
    p.s0 = pos.s[0]; p.s1 = pos.s[1]; p.s2 = pos.s[2];
    p.classes = C;
    p.sc = pos.x.stride(dim);
    if (labels.defined()) {
      p.labels = labels.const_data_ptr<int64_t>();
      p.log_prob = log_prob.data_ptr<float>();
    }
    p.ignore_label = ignore;
    p.has_ignore = has_ignore;
    p.class_mask = mask.ptr();
    p.mask_stride = mask.stride;
    p.mask_div = mask.div;
    p.inner = pos.inner;
    p.entropy = entropy.data_ptr<float>();
    if (topk) {
      p.top_log_probs = top_lp.data_ptr<float>();
      p.top_ids = top_id.data_ptr<int32_t>();
    }
    if (want_stats) p.stats = stats.data_ptr<float>();
    p.temperature = temperature;
    p.topk = (int)topk;
    p.dtype = code;
    const OnDevice on(logits.device());
    p.workspace_bytes = (int64_t)p_fwd_ws(&p);
    if (p.workspace_bytes) {
      workspace = at::empty({p.workspace_bytes}, f32.dtype(at::kByte));
      p.workspace = workspace.data_ptr();
    }
    check_status(p_fwd(&p, on.stream()), "ldm_label_log_probs");
  }
  PyObject* r = PyTuple_New(5);
  if (!r) return nullptr;
  const at::Tensor* all[5] = {&log_prob, &entropy, &top_lp, &top_id, &stats};
  for (int i = 0; i < 5; ++i) PyTuple_SET_ITEM(r, i, wrap_or_none(*all[i]));
  return r;
  END_HANDLE_TH_ERRORS
}

at::Tensor upstream(PyObject* o, const at::DimVector& shape, const at::Tensor& logits, const char* name) {
  if (o == Py_None) return {};
  const at::Tensor& g = tensor_of(o, name);
  TORCH_CHECK_VALUE(g.scalar_type() == at::kFloat && g.device() == logits.device() &&
                    g.sizes() == at::IntArrayRef(shape), name, " must be fp32 ", at::IntArrayRef(shape),
                    " on the logits' device");
  return g.resolve_neg().contiguous();
}

// (logits, stats, d_log_prob | None, d_entropy | None, dim, temperature, class_mask | None) -> d_logits
PyObject* label_log_probs_bwd(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(nargs == 7 && p_bwd, "label_log_probs_bwd: 7 arguments after init()");
  const at::Tensor logits = logits_of(args[0]);
  const int code = dtype_code(logits, "dtype");
  const int64_t dim = class_dim(logits, int_of(args[4], "dim"));
  const float temperature = temperature_of(args[5]);
  const at::DimVector shape = without(logits.sizes(), dim);
  const at::Tensor& stats = tensor_of(args[1], "stats");
  at::DimVector four(shape);
  four.insert(four.begin(), 4);
  TORCH_CHECK_VALUE(stats.scalar_type() == at::kFloat && stats.device() == logits.device() &&
                    stats.sizes() == at::IntArrayRef(four) && stats.is_contiguous(),
                    "stats must be label_log_probs' fp32 ", at::IntArrayRef(four));
  const at::Tensor gl = upstream(args[2], shape, logits, "d_log_prob"), ge = upstream(args[3], shape, logits, "d_entropy");
  int64_t count = 1;
  for (int64_t n : shape) count *= n;
  const Mask mask = mask_of(args[6], logits, dim, count);
  check_gpu(logits);
  const Positions pos = positions_of(logits.detach(), dim, true);
  if (count) {
    ldm_label_probs_bwd_params p = {};
    p.logits = pos.x.data_ptr();
    p.n0 = pos.n[0]; p.n1 = pos.n[1]; p.n2 = pos.n[2];
    p.s0 = pos.s[0]; p.s1 = pos.s[1]; p.s2 = pos.s[2];
    p.classes = logits.size(dim);
    p.sc = pos.x.stride(dim);
    p.class_mask = mask.ptr();
    p.mask_stride = mask.stride;
    p.mask_div = mask.div;
    p.stats = stats.data_ptr<float>();
    p.d_log_prob = gl.defined() ? gl.data_ptr<float>() : nullptr;
    p.d_entropy = ge.defined() ? ge.data_ptr<float>() : nullptr;
    p.d_logits = pos.out->data_ptr();
    p.o0 = pos.o[0]; p.o1 = pos.o[1]; p.o2 = pos.o[2];
    p.oc = pos.out->stride(dim);
    p.temperature = temperature;
    p.dtype = code;
    const OnDevice on(logits.device());
    check_status(p_bwd(&p, on.stream()), "ldm_label_log_probs_bwd");
  }
  return THPVariable_Wrap(*pos.out);
  END_HANDLE_TH_ERRORS
}

// (x, out | None, dim) -> (x walked, sizes, strides, positions behind the class dim, out walked, out strides): the
// address arithmetic of the two calls above, for tests without a GPU
PyObject* label_positions(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(nargs == 2, "label_positions: 2 arguments");
  const Positions p = positions_of(tensor_of(args[0], "x"), int_of(args[1], "dim"), true);
  return Py_BuildValue("N(LLL)(LLL)LN(LLL)", THPVariable_Wrap(p.x), (long long)p.n[0], (long long)p.n[1],
                       (long long)p.n[2], (long long)p.s[0], (long long)p.s[1], (long long)p.s[2], (long long)p.inner,
                       THPVariable_Wrap(*p.out), (long long)p.o[0], (long long)p.o[1], (long long)p.o[2]);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------ gradient norms
// The first n tensors of a list, or of a sequence, marked as modified while it is walked, unless what follows throws
// (in a walk of its own after the launches 700 gradients cost the host 20 us for 16, waiting for version counters).
struct Marks {
  const std::vector<at::Tensor>& list;
  PyObject* sequence;              // or null
  size_t n = 0;
  void add(const at::Tensor& t) {
    t.unsafeGetTensorImpl()->bump_version();       // throws at an inference tensor outside inference mode
    ++n;
  }
  ~Marks() {
    for (size_t i = 0; i < n; ++i) {
      const at::Tensor& t = sequence ? THPVariable_Unpack(PySequence_Fast_GET_ITEM(sequence, i)) : list[i];
      if (t.unsafeGetTensorImpl()->is_inference()) continue;               // has no version
      c10::VariableVersion v = t.unsafeGetTensorImpl()->version_counter();
      v.set_version((int64_t)v.current_version() - 1);
    }
  }
};

// (tensors, of_params, norm_type code, max_norm, clip, out | None): the norm and the factor of `tensors` (or, with
// of_params, of the gradients that they have), clip as in ldm_grad_norm -> the norm, or (norm, out) where clip is 0
// and out None; None without a gradient
PyObject* grad_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(nargs == 6 && p_norm, "grad_norm: 6 arguments after init()");
  const int of_params = PyObject_IsTrue(args[1]);
  const int64_t kind = int_of(args[2], "norm_type"), clip = int_of(args[4], "clip");
  const double max_norm = double_of(args[3], "max_norm");
  TORCH_CHECK_VALUE(max_norm >= 0, "max_norm must be a number >= 0, got ", max_norm);
  PyObject* items = PySequence_Fast(args[0], "an iterable of tensors is expected");
  if (!items) throw python_error();
  const THPObjectPtr hold(items);
  const Py_ssize_t given = PySequence_Fast_GET_SIZE(items);
  std::vector<const void*> ptrs;
  std::vector<int64_t> numel;
  std::vector<uint8_t> codes;
  ptrs.reserve(given);
  numel.reserve(given);
  codes.reserve(given);
  std::vector<at::Tensor> keep;    // gradients stay alive until the launches are queued
  keep.reserve(of_params ? given : 0);
  Marks marks{keep, of_params ? nullptr : items};
  at::Device device(at::kCPU);
  at::TensorOptions options;
  for (Py_ssize_t i = 0; i < given; ++i) {
    const at::Tensor& t = tensor_of(PySequence_Fast_GET_ITEM(items, i), "a parameter");
    if (of_params) {
      at::Tensor g = t.grad();
      if (!g.defined()) continue;
      keep.push_back(std::move(g));
    }
    const at::Tensor& g = of_params ? keep.back() : t;
    TORCH_CHECK_TYPE(g.layout() == at::kStrided, "sparse gradients are not supported");
    codes.push_back((uint8_t)dtype_code(g, "gradient dtype"));
    if (ptrs.empty()) {
      device = g.device();
      options = g.options();
    }
    TORCH_CHECK_VALUE(g.device() == device, "gradients on ", device, " and ", g.device(), ": one device per call");
    TORCH_CHECK_VALUE(g.is_non_overlapping_and_dense() || g.numel() == 0,
                      "a gradient is no dense memory (an expanded or strided view): make it contiguous");
    if (clip) marks.add(g);        // written in place: autograd sees it
    numel.push_back(g.numel());
    ptrs.push_back(g.numel() ? g.data_ptr() : nullptr);
  }
  if (ptrs.empty()) Py_RETURN_NONE;
  TORCH_CHECK(device.is_cuda(), "ldmseg HIP ops take GPU tensors only (no CPU fallback); got a tensor on ", device);
  const auto f32 = options.dtype(at::kFloat).memory_format(std::nullopt).requires_grad(false);
  const at::Tensor out = args[5] == Py_None ? at::empty({2}, f32) : tensor_of(args[5], "out");
  const int n = (int)ptrs.size();
  const OnDevice on(device);
  at::Tensor workspace;
  const size_t bytes = p_norm_ws(numel.data(), n);
  if (bytes) workspace = at::empty({(int64_t)bytes}, f32.dtype(at::kByte));
  const int rc = p_norm(ptrs.data(), numel.data(), codes.data(), n, (int)kind, max_norm, (int)clip,
                        out.data_ptr<float>(), bytes ? workspace.data_ptr() : nullptr, (int64_t)bytes, on.stream());
  TORCH_CHECK_VALUE(rc != LDM_ERR_OVERLAP,
                    "gradients overlap in memory (the same gradient twice, or views of one another)");
  check_status(rc, "ldm_grad_norm");
  marks.n = 0;                     // a refused call has not come here: its marks are taken back
  if (clip || args[5] != Py_None) return THPVariable_Wrap(out.select(0, 0));
  return Py_BuildValue("NN", THPVariable_Wrap(out.select(0, 0)), THPVariable_Wrap(out));
  END_HANDLE_TH_ERRORS
}

// init(addresses of the six C entries)
PyObject* init(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(nargs == 6, "init: 6 addresses");
  void* p[6];
  for (int i = 0; i < 6; ++i) p[i] = reinterpret_cast<void*>(int_of(args[i], "address"));
  p_fwd_ws = reinterpret_cast<decltype(p_fwd_ws)>(p[0]);
  p_fwd = reinterpret_cast<decltype(p_fwd)>(p[1]);
  p_bwd = reinterpret_cast<decltype(p_bwd)>(p[2]);
  p_norm_ws = reinterpret_cast<decltype(p_norm_ws)>(p[3]);
  p_norm = reinterpret_cast<decltype(p_norm)>(p[4]);
  p_status = reinterpret_cast<decltype(p_status)>(p[5]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)> PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
}
PyMethodDef methods[] = {
    {"init", fast<init>(), METH_FASTCALL, nullptr},
    {"label_log_probs", fast<label_log_probs>(), METH_FASTCALL, nullptr},
    {"label_log_probs_bwd", fast<label_log_probs_bwd>(), METH_FASTCALL, nullptr},
    {"label_positions", fast<label_positions>(), METH_FASTCALL, nullptr},
    {"grad_norm", fast<grad_norm>(), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "ldmseg_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_ldmseg_torch() { return PyModule_Create(&module); }
