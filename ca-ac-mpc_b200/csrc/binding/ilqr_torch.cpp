// ilqr_torch.cpp -- torch binding of the gradient norms and clipping.
//
// These calls take lists of up to thousands of tensors, whose addresses, sizes,
// types and strides are read here: the same reading through the Python
// interface costs 0.6 us a tensor and takes longer than the kernels for most
// lists (400 bf16 tensors of 600 MB: 246 us against 95 us of GPU time). The
// calls are documented in ilqr_native.py; everything but the reading goes through
// the C ABI in include/ilqr_b200.h.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/util/SmallVector.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <vector>

#include "../ilqr_overlap.h"
#include "ilqr_b200.h"

namespace {

struct Object {  // an owned reference
  PyObject* p;
  explicit Object(PyObject* o) : p(o) {
    if (p == nullptr) throw python_error();
  }
  ~Object() { Py_XDECREF(p); }
  Object(const Object&) = delete;
  Object& operator=(const Object&) = delete;
  PyObject* release() {
    PyObject* o = p;
    p = nullptr;
    return o;
  }
};

using Tensors = c10::SmallVector<at::Tensor, 16>;

template <typename T>
using Small = c10::SmallVector<T, 64>;

void check(int status, const char* what) {
  TORCH_CHECK(status == ILQR_OK, what, " failed: ", ilqr_b200_status_string(status), " (status ", status, ")");
}

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return ILQR_DTYPE_F32;
    case at::kHalf: return ILQR_DTYPE_F16;
    case at::kBFloat16: return ILQR_DTYPE_BF16;
    default: return -1;
  }
}

// The tensors of a Python list, checked: dense CUDA tensors of the three types
// on one device.
void read_list(PyObject* list, Tensors& out) {
  const Py_ssize_t n = PyList_GET_SIZE(list);
  out.reserve((size_t)n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PyList_GET_ITEM(list, i);
    TORCH_CHECK_TYPE(THPVariable_Check(o), "grads must hold tensors, not ", Py_TYPE(o)->tp_name);
    const at::Tensor& t = THPVariable_Unpack(o);
    TORCH_CHECK(t.is_cuda(), "grads must hold CUDA tensors (no CPU path)");
    TORCH_CHECK(t.layout() == at::kStrided, "grads must be dense tensors, got ", t.layout());
    TORCH_CHECK(code_of(t.scalar_type()) >= 0, "grads must be float32, float16 or bfloat16, got ", t.scalar_type());
    TORCH_CHECK(i == 0 || t.device() == out[0].device(), "grads must be on one device, got ", out[0].device(), " and ",
                t.device());
    out.push_back(t);
  }
}

// What a caller gave for a list of tensors, as a Python list.
PyObject* as_list(PyObject* given, const char* name) {
  TORCH_CHECK_TYPE(!THPVariable_Check(given), name, " must be a sequence of tensors, not one tensor");
  if (PyList_CheckExact(given)) {
    Py_INCREF(given);
    return given;
  }
  return PySequence_List(given);
}

// The outputs a caller gave as a new Python list; None stays.
PyObject* given_outputs(PyObject* given) {
  if (given == Py_None) return Py_NewRef(given);
  TORCH_CHECK_TYPE(!THPVariable_Check(given), "out must be a sequence of tensors, not one tensor");
  return PySequence_List(given);
}

bool truth(PyObject* o) {
  const int t = PyObject_IsTrue(o);
  if (t < 0) throw python_error();
  return t == 1;
}

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

int64_t dimension(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

int32_t norm_code(PyObject* norm_type) {
  const double p = number(norm_type);
  TORCH_CHECK_VALUE(p == 2.0 || p == INFINITY, "norm_type must be 2 or inf, not ", p);
  return p == 2.0 ? ILQR_NORM_L2 : ILQR_NORM_MAX;
}

struct Bound {
  double max_norm, eps;
  Bound(PyObject* m, PyObject* e) : max_norm(number(m)), eps(number(e)) {
    TORCH_CHECK_VALUE(max_norm >= 0.0, "max_norm must not be negative or NaN, got ", max_norm);
    TORCH_CHECK_VALUE(eps >= 0.0 && eps < INFINITY, "eps must be finite and not negative, got ", eps);
  }
};

struct Dim {
  int64_t size, stride;
};

// The dimensions of more than one value, by stride.
void by_stride(const at::Tensor& t, c10::SmallVector<Dim, 8>& d) {
  for (int64_t k = 0; k < t.dim(); ++k)
    if (t.size(k) != 1) d.push_back({t.size(k), t.stride(k)});
  std::sort(d.begin(), d.end(), [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
}

// Whether the values fill one run of memory, each in a place of its own.
bool without_gaps(const at::Tensor& t) {
  if (t.is_contiguous()) return true;
  c10::SmallVector<Dim, 8> d;
  by_stride(t, d);
  int64_t want = 1;
  for (const Dim& x : d) {
    if (x.stride != want) return false;
    want *= x.size;
  }
  return true;
}

// Whether each value has a place of its own: every stride steps over all that
// the smaller ones span.
bool one_to_a_place(const at::Tensor& t) {
  if (t.is_contiguous() || t.numel() == 0) return true;
  c10::SmallVector<Dim, 8> d;
  by_stride(t, d);
  int64_t span = 1;
  for (const Dim& x : d) {
    if (x.stride < span) return false;
    span += x.stride * (x.size - 1);
  }
  return true;
}

at::Tensor gathered(const at::Tensor& t) {
  at::Tensor flat = at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous));
  flat.copy_(t);
  return flat;
}

// The outputs: a Python list of new tensors, or `given` (of given_outputs)
// checked against the inputs.
PyObject* outputs(PyObject* given, PyObject* grads_list, const Tensors& grads, Tensors& out) {
  const Py_ssize_t n = (Py_ssize_t)grads.size();
  out.reserve((size_t)n);
  if (given == Py_None) {
    Object list(PyList_New(n));
    for (Py_ssize_t i = 0; i < n; ++i) {
      out.push_back(at::empty_like(grads[i]));
      PyObject* o = THPVariable_Wrap(out.back());
      if (o == nullptr) throw python_error();
      PyList_SET_ITEM(list.p, i, o);
    }
    return list.release();
  }
  TORCH_CHECK(PyList_GET_SIZE(given) == n, "out must hold ", n, " tensors, got ", PyList_GET_SIZE(given));
  const bool grad_mode = at::GradMode::is_enabled();
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PyList_GET_ITEM(given, i);
    TORCH_CHECK_TYPE(THPVariable_Check(o), "out must hold tensors, not ", Py_TYPE(o)->tp_name);
    const at::Tensor& t = THPVariable_Unpack(o);
    if (o != PyList_GET_ITEM(grads_list, i)) {
      const at::Tensor& g = grads[i];
      TORCH_CHECK(t.layout() == at::kStrided && t.sizes() == g.sizes() && t.scalar_type() == g.scalar_type() &&
                      t.device() == g.device(),
                  "out must have the gradients' shape, dtype and device: ", g.sizes(), " ", g.scalar_type(), " ",
                  g.device(), ", got ", t.sizes(), " ", t.scalar_type(), " ", t.device());
    }
    TORCH_CHECK(!(grad_mode && t.requires_grad()), "out must not require grad: clipping is not differentiable");
    TORCH_CHECK(one_to_a_place(t), "out must hold tensors whose values each have a place of their own");
    out.push_back(t);
  }
  return Py_NewRef(given);
}

using Gathered = c10::SmallVector<std::pair<size_t, at::Tensor>, 4>;

// A tensor of a call, as runs of bytes.
struct Place {
  c10::SmallVector<ilqr::Every, 8> dims;
  uintptr_t lo, hi;
  int64_t len;
  int64_t step = 0, at = 0;  // every run lies at `at` of `step` bytes; 0: not so
  bool is_out, is_gathered;
  Place(const at::Tensor& t, const void* p, bool o, bool g)
      : lo((uintptr_t)p), len(t.element_size()), is_out(o), is_gathered(g) {
    c10::SmallVector<Dim, 8> d;
    by_stride(t, d);
    for (const Dim& x : d) {
      const int64_t stride = x.stride * (int64_t)t.element_size();
      if (dims.empty() && stride == len) len *= x.size;
      else dims.push_back({x.size, stride});
    }
    hi = runs().hi();
    if (dims.empty() || dims[0].stride < len) return;
    for (const ilqr::Every& e : dims)
      if (e.stride % dims[0].stride != 0) return;
    step = dims[0].stride;
    at = (int64_t)(lo % (uintptr_t)step);
  }
  // Columns of one array, without a search.
  bool beside(const Place& x) const {
    return step > 0 && step == x.step && at + len <= step && x.at + x.len <= step &&
           (at + len <= x.at || x.at + x.len <= at);
  }
  ilqr::Strided runs() const { return {lo, len, dims.data(), (int)dims.size()}; }
  bool is(const Place& x) const {
    return lo == x.lo && len == x.len &&
           std::equal(dims.begin(), dims.end(), x.dims.begin(), x.dims.end(),
                      [](const ilqr::Every& a, const ilqr::Every& b) { return a.count == b.count && a.stride == b.stride; });
  }
};

// Whether all of them are columns of one array that end before the next begins.
bool all_beside(const std::vector<Place>& all) {
  std::vector<std::pair<int64_t, int64_t>> c;
  c.reserve(all.size() + 1);
  for (const Place& p : all) {
    if (p.step == 0 || p.step != all[0].step) return false;
    c.emplace_back(p.at, p.at + p.len);
  }
  std::sort(c.begin(), c.end());
  c.emplace_back(all[0].step, 0);
  for (size_t k = 1; k < c.size(); ++k)
    if (c[k - 1].second > c[k].first) return false;
  return true;
}

// The C ABI sees the copies of gathered tensors: whether what these write in the
// end is also written, or read, elsewhere in the call is found here.
bool gathered_overlap(const Tensors& grads, const Tensors& out, const Gathered& gathered, PyObject* total) {
  std::vector<Place> all;
  all.reserve(2 * grads.size() + 1);
  if (total != Py_None) {
    const at::Tensor& t = THPVariable_Unpack(total);
    all.emplace_back(t, t.const_data_ptr(), false, true);
  }
  for (size_t i = 0, k = 0; i < grads.size(); ++i) {
    const at::Tensor &g = grads[i], &o = out[i];
    const bool there = k < gathered.size() && gathered[k].first == i;
    if (there) ++k;
    if (g.numel() == 0) continue;
    all.emplace_back(o, o.mutable_data_ptr(), true, there);
    Place in(g, g.const_data_ptr(), false, there);
    if (!in.is(all.back())) all.push_back(std::move(in));
  }
  if (all.empty() || all_beside(all)) return false;
  std::sort(all.begin(), all.end(), [](const Place& a, const Place& b) { return a.lo < b.lo; });
  for (size_t a = 0; a < all.size(); ++a)
    for (size_t b = a + 1; b < all.size() && all[b].lo < all[a].hi; ++b)
      if ((all[a].is_out || all[b].is_out) && (all[a].is_gathered || all[b].is_gathered) &&
          !all[a].beside(all[b]) && ilqr::Meeting::of(all[a].runs(), all[b].runs()))
        return true;
  return false;
}

void written(const Tensors& out) {
  for (const at::Tensor& t : out)
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void device_ok(c10::DeviceIndex index) {
  static std::atomic<bool> fine[64];
  if (index < 64 && fine[index].load(std::memory_order_relaxed)) return;
  check(ilqr_b200_check_device(index), "device check");
  if (index < 64) fine[index].store(true, std::memory_order_relaxed);
}

struct Arrays {
  Small<const void*> in;
  Small<int64_t> numel;
  Small<int32_t> types;
  void add(const at::Tensor& t) {
    in.push_back(t.const_data_ptr());
    numel.push_back(t.numel());
    types.push_back(code_of(t.scalar_type()));
  }
};

at::Tensor new_tensor(at::IntArrayRef size, at::ScalarType type, c10::Device device) {
  return at::detail::empty_cuda(size, type, device, c10::nullopt);
}

at::Tensor workspace(int32_t n, c10::Device device, size_t* bytes) {
  check(ilqr_b200_grad_workspace_size(n, bytes), "workspace query");
  return new_tensor({(int64_t)*bytes}, at::kByte, device);
}

// grad_norm(grads, norm_type, norm?, norms?, total?) -> tuple of those asked for
PyObject* grad_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 5, "grad_norm takes five values");
  const int32_t code = norm_code(args[1]);
  bool want[3];
  for (int k = 0; k < 3; ++k) want[k] = truth(args[2 + k]);
  const Object given(as_list(args[0], "grads"));
  Tensors grads;
  read_list(given.p, grads);
  TORCH_CHECK(!grads.empty(), "grads is empty: there is no device to put its norm on");
  at::NoGradGuard no_grad;
  const c10::Device device = grads[0].device();
  const c10::cuda::OptionalCUDAGuard guard(device);
  device_ok(device.index());
  const int32_t n = (int32_t)grads.size();
  Arrays a;
  Tensors kept;
  for (const at::Tensor& g : grads) {
    if (without_gaps(g)) {
      a.add(g);
    } else {  // with gaps, or several values to a place
      kept.push_back(gathered(g));
      a.add(kept.back());
    }
  }
  at::Tensor out[3];
  if (want[0]) out[0] = new_tensor({}, at::kFloat, device);
  if (want[1]) out[1] = new_tensor({n}, at::kFloat, device);
  if (want[2]) out[2] = new_tensor({}, at::kDouble, device);
  size_t bytes = 0;
  const at::Tensor ws = workspace(n, device, &bytes);
  check(ilqr_b200_grad_norm(a.in.data(), a.numel.data(), a.types.data(), n, code,
                            want[0] ? out[0].mutable_data_ptr<float>() : nullptr,
                            want[1] ? out[1].mutable_data_ptr<float>() : nullptr,
                            want[2] ? out[2].mutable_data_ptr<double>() : nullptr, ws.mutable_data_ptr(), bytes,
                            c10::cuda::getCurrentCUDAStream(device.index()).stream()),
        "ilqr_b200_grad_norm");
  Object got(PyTuple_New(want[0] + want[1] + want[2]));
  for (int k = 0, at = 0; k < 3; ++k) {
    if (!want[k]) continue;
    PyObject* o = THPVariable_Wrap(out[k]);
    if (o == nullptr) throw python_error();
    PyTuple_SET_ITEM(got.p, at++, o);
  }
  return got.release();
  END_HANDLE_TH_ERRORS
}

// clip_grad_norm(grads, out or None, max_norm, norm_type, eps, total or None) -> (out, norm)
PyObject* clip_grad_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 6, "clip_grad_norm takes six values");
  const int32_t code = norm_code(args[3]);
  const Bound bound(args[2], args[4]);
  // all that may run the caller's code comes before the first tensor is read
  const Object given_out(given_outputs(args[1]));
  const Object given(as_list(args[0], "grads"));
  Tensors grads, out;
  read_list(given.p, grads);
  TORCH_CHECK(!grads.empty(), "grads is empty: there is no device to put its norm on");
  const c10::Device device = grads[0].device();
  const double* total = nullptr;
  if (args[5] != Py_None) {
    TORCH_CHECK_TYPE(THPVariable_Check(args[5]), "total must be a tensor");
    const at::Tensor& t = THPVariable_Unpack(args[5]);
    TORCH_CHECK(t.device() == device && t.scalar_type() == at::kDouble && t.dim() == 0,
                "total must be a 0-d float64 tensor on ", device, ", got ", t.sizes(), " ", t.scalar_type(), " on ",
                t.device());
    total = t.const_data_ptr<double>();
  }
  const c10::cuda::OptionalCUDAGuard guard(device);
  device_ok(device.index());
  Object list(outputs(given_out.p, given.p, grads, out));
  at::NoGradGuard no_grad;
  const int32_t n = (int32_t)grads.size();
  Arrays a;
  Small<void*> to;
  Gathered back;
  for (size_t i = 0; i < grads.size(); ++i) {
    const at::Tensor &g = grads[i], &o = out[i];
    if (without_gaps(g) && !g.is_neg() && !o.is_neg() && (g.is_same(o) || g.strides() == o.strides())) {
      a.add(g);
      to.push_back(o.mutable_data_ptr());
    } else {
      back.emplace_back(i, gathered(g));
      a.add(back.back().second);
      to.push_back(back.back().second.mutable_data_ptr());
    }
  }
  if (!back.empty() && args[1] != Py_None && gathered_overlap(grads, out, back, args[5]))
    check(ILQR_ERR_OVERLAP, "clip_grad_norm");
  const at::Tensor norm = new_tensor({}, at::kFloat, device);
  size_t bytes = 0;
  const at::Tensor ws = workspace(n, device, &bytes);
  check(ilqr_b200_grad_clip(a.in.data(), to.data(), a.numel.data(), a.types.data(), n, code, bound.max_norm, bound.eps,
                            total,
                            norm.mutable_data_ptr<float>(), ws.mutable_data_ptr(), bytes,
                            c10::cuda::getCurrentCUDAStream(device.index()).stream()),
        "ilqr_b200_grad_clip");
  for (const auto& b : back) out[b.first].copy_(b.second);
  if (args[1] != Py_None) written(out);
  Object got(PyTuple_New(2));
  PyTuple_SET_ITEM(got.p, 0, list.release());
  PyObject* o = THPVariable_Wrap(norm);
  if (o == nullptr) throw python_error();
  PyTuple_SET_ITEM(got.p, 1, o);
  return got.release();
  END_HANDLE_TH_ERRORS
}

// How the slices of g and o along dimension d lie in memory: segments, their
// length, strides of g's segments and slices, of o's. False where a slice is
// not evenly spaced segments of both.
bool segments(const at::Tensor& g, const at::Tensor& o, int64_t d, int64_t* lay) {
  struct Two {
    int64_t size, g, o;
  };
  c10::SmallVector<Two, 8> dims;  // innermost first, merged where both go on evenly
  for (int64_t k = g.dim() - 1; k >= 0; --k) {
    if (k == d || g.size(k) == 1) continue;
    const Two x{g.size(k), g.stride(k), o.stride(k)};
    if (!dims.empty() && x.g == dims.back().g * dims.back().size && x.o == dims.back().o * dims.back().size)
      dims.back().size *= x.size;
    else
      dims.push_back(x);
  }
  int64_t length = 1;
  size_t at = 0;
  if (!dims.empty() && dims[0].g == 1 && dims[0].o == 1) length = dims[at++].size;
  if (dims.size() - at > 1) return false;
  const Two s = dims.size() > at ? dims[at] : Two{1, 0, 0};
  const int64_t v[6] = {s.size, length, s.g, g.stride(d), s.o, o.stride(d)};
  std::copy(v, v + 6, lay);
  return true;
}

// clip_grad_elements(grads, out or None, batch dims: a number or a sequence, max_norm, eps, zero?) -> (out, norms)
PyObject* clip_grad_elements(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 6, "clip_grad_elements takes six values");
  const Bound bound(args[3], args[4]);
  const bool zero_nonfinite = truth(args[5]);
  // a number of any kind (NumPy's among them); tensors and arrays count as sequences
  const bool each = !PyIndex_Check(args[2]) || Py_TYPE(args[2])->tp_iter != nullptr;
  const Object given_out(given_outputs(args[1]));
  const Object given_dims(each ? PySequence_List(args[2]) : Py_NewRef(args[2]));
  c10::SmallVector<int64_t, ILQR_MAX_ELEMENT_TENSORS> dims;
  for (Py_ssize_t i = 0, k = each ? PyList_GET_SIZE(given_dims.p) : 1; i < k; ++i)
    dims.push_back(dimension(each ? PyList_GET_ITEM(given_dims.p, i) : given_dims.p));
  const Object given(as_list(args[0], "grads"));
  // all that may run the caller's code has come before the first tensor is read
  Tensors grads, out;
  read_list(given.p, grads);
  const size_t n = grads.size();
  TORCH_CHECK(n >= 1 && n <= ILQR_MAX_ELEMENT_TENSORS, "grads must hold 1 to ", ILQR_MAX_ELEMENT_TENSORS,
              " tensors, got ", n);
  TORCH_CHECK(!each || dims.size() == n, "batch_dims must hold ", n, " numbers, got ", dims.size());
  if (!each) dims.assign(n, dims[0]);
  int64_t B = 0;
  for (size_t i = 0; i < n; ++i) {
    TORCH_CHECK(dims[i] >= 0 && dims[i] < grads[i].dim(), "batch dimension ", dims[i], " of a tensor of shape ",
                grads[i].sizes());
    if (i == 0) B = grads[0].size(dims[0]);
    TORCH_CHECK(grads[i].size(dims[i]) == B, "grads must have one batch size, got ", B, " and ",
                grads[i].size(dims[i]));
  }
  const c10::Device device = grads[0].device();
  const c10::cuda::OptionalCUDAGuard guard(device);
  device_ok(device.index());
  Object list(outputs(given_out.p, given.p, grads, out));
  at::NoGradGuard no_grad;
  Arrays a;
  Small<void*> to;
  int64_t layout[6 * ILQR_MAX_ELEMENT_TENSORS] = {};
  Gathered back;
  for (size_t i = 0; i < n; ++i) {
    const at::Tensor &g = grads[i], &o = out[i];
    // a tensor without values has no segments
    if (g.numel() == 0 || (!g.is_neg() && !o.is_neg() && segments(g, o, dims[i], layout + 6 * i))) {
      a.add(g);
      to.push_back(o.mutable_data_ptr());
    } else {
      back.emplace_back(i, gathered(g));
      const at::Tensor& flat = back.back().second;
      a.add(flat);
      to.push_back(flat.mutable_data_ptr());
      TORCH_INTERNAL_ASSERT(segments(flat, flat, dims[i], layout + 6 * i));
    }
  }
  if (!back.empty() && args[1] != Py_None && gathered_overlap(grads, out, back, Py_None))
    check(ILQR_ERR_OVERLAP, "clip_grad_elements");
  const at::Tensor norms = new_tensor({B}, at::kFloat, device);
  check(ilqr_b200_grad_clip_elements(a.in.data(), to.data(), a.types.data(), layout, (int32_t)n, B, bound.max_norm,
                                     bound.eps, zero_nonfinite ? 1 : 0, norms.mutable_data_ptr<float>(),
                                     c10::cuda::getCurrentCUDAStream(device.index()).stream()),
        "ilqr_b200_grad_clip_elements");
  for (const auto& b : back) out[b.first].copy_(b.second);
  if (args[1] != Py_None) written(out);
  Object got(PyTuple_New(2));
  PyTuple_SET_ITEM(got.p, 0, list.release());
  PyObject* o = THPVariable_Wrap(norms);
  if (o == nullptr) throw python_error();
  PyTuple_SET_ITEM(got.p, 1, o);
  return got.release();
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"grad_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(grad_norm)), METH_FASTCALL, nullptr},
    {"clip_grad_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(clip_grad_norm)), METH_FASTCALL,
     nullptr},
    {"clip_grad_elements", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(clip_grad_elements)),
     METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "ilqr_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_ilqr_torch(void) { return PyModule_Create(&module_def); }
