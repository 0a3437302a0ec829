// Python binding of the calls whose kernels take a few microseconds: the norm, the appends,
// the calls on shared pages, the page copies and the runs of the paged prefill. It checks
// the tensors, allocates the outputs and fills the params structs of
// atflash_b200.h; the library itself is loaded by the package, which hands over the
// addresses of its functions (init).
//
// Why it is compiled: in Python these steps took 10 to 15 us of a call of 15 to 18 us, for
// kernels of 2 to 7 us (64 tokens' norm 18.3 -> 9.4 us, an append 15 -> 6.3, a fork with a
// free and copies 37 -> 20). Launches and allocations run without the GIL, which takes 0.2 us a
// call. The other entry points (plans, or longer work) stay on ctypes.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Device.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/headeronly/version.h>

#include <array>
#include <cmath>
#include <optional>
#include <string>

#include "../../include/atflash_b200.h"

namespace {

using at::Tensor;

// ------------------------------------------------------------------ what the package hands over

struct Library {
  decltype(&atf_qk_norm_rope) qk_norm_rope;
  decltype(&atf_paged_kv_append) append;
  decltype(&atf_paged_kv_append_e4m3) append_e4m3;
  decltype(&atf_paged_kv_append_norm) append_norm;
  decltype(&atf_fork_requests) fork;
  decltype(&atf_free_requests) free_;
  decltype(&atf_compact_pages) compact;
  decltype(&atf_copy_pages) copy;
  decltype(&atf_prefill_paged_fwd) paged;
} lib;
PyObject* g_check;    // check(name, status): raises
PyObject* g_runtime;  // the package's _runtime: _flags, error_flag, narrow_i32

struct ValueError : torch::PyTorchError {
  using PyTorchError::PyTorchError;
  PyObject* python_type() override { return PyExc_ValueError; }
};

// ------------------------------------------------------------------ arguments

const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw torch::TypeError(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}
const Tensor* tensor_or_none(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

// the two entries of a tuple or list
std::optional<std::array<PyObject*, 2>> pair(PyObject* o) {
  if (PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 2) return {{PyTuple_GET_ITEM(o, 0), PyTuple_GET_ITEM(o, 1)}};
  if (PyList_Check(o) && PyList_GET_SIZE(o) == 2) return {{PyList_GET_ITEM(o, 0), PyList_GET_ITEM(o, 1)}};
  return std::nullopt;
}

std::string on(c10::Device d) { return " on " + d.str(); }

constexpr const char* NO_CPU = "atflash kernels take CUDA tensors (there is no CPU path)";
constexpr const char* ONE_DEVICE = "all tensors must be on the same device";
c10::Device require_cuda(std::initializer_list<const Tensor*> ts) {
  const Tensor& first = **ts.begin();
  for (const Tensor* t : ts) {
    if (!t->is_cuda()) throw ValueError(NO_CPU);
    if (t->device() != first.device()) throw ValueError(ONE_DEVICE);
  }
  return first.device();
}

void refuse_gradients(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : ts)
    if (t != nullptr && t->requires_grad())
      throw std::runtime_error("atflash has no backward pass: call it under torch.no_grad() or with detached tensors");
}

bool is(PyObject* o, const char* text) { return PyUnicode_Check(o) && PyUnicode_CompareWithASCIIString(o, text) == 0; }
int pair_order(PyObject* o) {  // -1: neither
  return is(o, "sorted_pair") ? ATF_LAYOUT_SORTED_PAIR : is(o, "rotate_half") ? ATF_LAYOUT_ROTATE_HALF : -1;
}

// ------------------------------------------------------------------ calls

// Lets other Python threads run: over a launch, which waits where the queue of launches
// is full (perhaps for a host callback that needs Python), and over allocations.
struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

PyObject* device_object(c10::Device dev) {
  PyObject* r = THPDevice_New(dev);
  if (r == nullptr) throw python_error();
  return r;
}

// the device's error flag: the package's tensor for it, made when there is none yet
int* error_flag(c10::Device dev) {
  PyObject* flags = PyObject_GetAttrString(g_runtime, "_flags");
  PyObject* index = PyLong_FromLong(dev.index());
  PyObject* flag = flags != nullptr && index != nullptr ? Py_XNewRef(PyDict_GetItemWithError(flags, index)) : nullptr;
  Py_XDECREF(flags);
  Py_XDECREF(index);
  if (flag == nullptr) {
    if (PyErr_Occurred()) throw python_error();
    PyObject* d = device_object(dev);
    flag = PyObject_CallMethod(g_runtime, "error_flag", "N", d);
    if (flag == nullptr) throw python_error();
  }
  int* at = static_cast<int*>(tensor(flag, "the error flag").data_ptr());
  Py_DECREF(flag);  // (the package holds it)
  return at;
}

// fn(params ..., current stream) with the tensors' device current; raises on a non-zero status
template <typename F, typename... P>
void launch(const char* name, F fn, c10::Device dev, P... params) {
  int rc;
  {
    const NoGil no_gil;
    const c10::DeviceIndex idx = dev.index();
    c10::cuda::OptionalCUDAGuard guard;
    if (c10::cuda::current_device() != idx) guard.set_index(idx);
    rc = fn(params..., c10::cuda::getCurrentCUDAStream(idx).stream());
  }
  if (rc != ATF_OK) {
    PyObject* r = PyObject_CallFunction(g_check, "si", name, rc);
    Py_XDECREF(r);
    throw python_error();
  }
}

// An index list that a call reads, as contiguous int32 on `dev`. 64-bit values that do not
// fit become ones that the kernels report.
Tensor narrow(const Tensor& t, c10::Device dev, int64_t top = 0x7fffffff) {
  if (t.scalar_type() == at::kInt && t.device() == dev && t.is_contiguous()) return t;
  PyObject* r = PyObject_CallMethod(g_runtime, "narrow_i32", "NNL", THPVariable_Wrap(t), device_object(dev),
                                    static_cast<long long>(top));
  if (r == nullptr) throw python_error();
  Tensor out = THPVariable_Unpack(r);
  Py_DECREF(r);
  return out;
}

// an index list of the calls on shared pages
Tensor index_list(const Tensor& t, const char* name, c10::Device dev, int64_t n = -1) {
  if (t.dim() != 1 || (n >= 0 && t.size(0) != n) || (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong))
    throw ValueError(std::string(name) + " must be a 1-d integer tensor" +
                     (n >= 0 ? " of " + std::to_string(n) + " entries" : ""));
  if (t.device() != dev) throw ValueError(ONE_DEVICE);
  return narrow(t, dev);
}

// a tensor that a call changes in place, taken as it is; returns its number of entries
int32_t in_place(const Tensor& t, const char* name, c10::Device dev, int64_t least = 1) {
  if (t.dim() != 1 || t.size(0) < least || t.scalar_type() != at::kInt || !t.is_contiguous() || t.size(0) > 0x7fffffff)
    throw ValueError(std::string(name) + " must be a contiguous 1-d int32 tensor" +
                     (least > 1 ? " of " + std::to_string(least) + " entries or more" : ""));
  if (t.device() != dev) throw ValueError(ONE_DEVICE);
  return static_cast<int32_t>(t.size(0));
}

template <typename T>
T* data(const Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}

// ------------------------------------------------------------------ norm

int check_norm(const Tensor& w, double eps, c10::Device dev, const char* name) {
  const at::ScalarType t = w.scalar_type();
  if ((t != at::kBFloat16 && t != at::kFloat) || w.dim() != 1 || w.size(0) != 128 || w.stride(0) != 1 || w.device() != dev)
    throw ValueError(std::string(name) + " must be 128 contiguous bf16 or fp32 weights" + on(dev));
  // as the kernels take it: far enough from 0 for a root, and finite
  if (!(eps >= 1e-38 && static_cast<float>(eps) < INFINITY)) throw ValueError("the norm's eps must be a positive fp32 number");
  return t == at::kFloat ? ATF_DTYPE_F32 : ATF_DTYPE_BF16;
}

struct Heads {  // of a (B, S, H, 128) or (T, H, 128) tensor
  int64_t b, s, h, sb, ss, sh;
};
Heads heads(const Tensor& x, const std::string& name) {
  const int64_t n = x.dim();
  if (x.scalar_type() != at::kBFloat16 || (n != 3 && n != 4) || x.size(n - 1) != 128 || x.stride(n - 1) != 1)
    throw ValueError(name + " must be (B, S, H, 128) or (T, H, 128) bf16 with a contiguous last axis");
  if (n == 3) return {1, x.size(0), x.size(1), 0, x.stride(0), x.stride(1)};
  return {x.size(0), x.size(1), x.size(2), x.stride(0), x.stride(1), x.stride(2)};
}

Tensor output(const Tensor* out, const Tensor& x, const std::string& name) {
  if (out == nullptr) {
    const NoGil no_gil;
    return at::empty_like(x);
  }
  if (out->sizes() != x.sizes() || out->scalar_type() != at::kBFloat16 || out->device() != x.device() || out->stride(-1) != 1)
    throw ValueError(name + " must be a bf16 tensor of its input's shape and device with a contiguous last axis");
  for (int64_t i = 0; i < out->dim(); ++i)
    if (out->size(i) > 1 && out->stride(i) == 0) throw ValueError(name + " must not be expanded: its rows are written");
  if (out->numel() > 0 && out->data_ptr() == x.data_ptr() && out->strides() != x.strides())
    throw ValueError(name + " over its own input needs the input's strides");
  return *out;
}

struct Angles {
  const float *cos, *sin;
  int64_t stride, n_pos;
};
Angles angles(const Tensor& cos, const Tensor& sin, c10::Device dev, const char* what) {
  if (cos.scalar_type() != at::kFloat || sin.scalar_type() != at::kFloat || cos.dim() != 2 || cos.sizes() != sin.sizes() ||
      cos.size(0) < 1 || cos.size(1) < 64 || cos.strides() != sin.strides() || cos.stride(1) != 1 || cos.device() != dev ||
      sin.device() != dev)
    throw ValueError(what);
  return {data<float>(cos), data<float>(sin), cos.stride(0), cos.size(0)};
}

// (q, k, q_weight, k_weight, cos, sin, eps, pos_offset, positions, out_layout, q_out, k_out)
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12) throw torch::TypeError("12 arguments");
  const Tensor& q = tensor(a[0], "q");
  const Tensor* k = tensor_or_none(a[1], "k");
  const Tensor& qw = tensor(a[2], "q_weight");
  const Tensor* kw = tensor_or_none(a[3], "k_weight");
  const Tensor &cos = tensor(a[4], "cos"), &sin = tensor(a[5], "sin");
  const Tensor* positions = tensor_or_none(a[8], "positions");
  const Tensor *q_out = tensor_or_none(a[10], "q_out"), *k_out = tensor_or_none(a[11], "k_out");
  const double eps = PyFloat_AsDouble(a[6]);
  if (eps == -1.0 && PyErr_Occurred()) throw python_error();
  if ((k == nullptr) != (kw == nullptr) || (k == nullptr && k_out != nullptr))
    throw ValueError("k and k_weight go together");
  refuse_gradients({&q, k, &qw, kw});
  const c10::Device dev = require_cuda({&q, &cos, &sin});
  const Heads hq = heads(q, "q");
  AtfQkNormParams p = {};
  p.weight_dtype = check_norm(qw, eps, dev, "q_weight");
  p.out_layout = pair_order(a[9]);
  if (p.out_layout < 0) throw ValueError("out_layout must be one of ['rotate_half', 'sorted_pair']");
  const Angles t = angles(cos, sin, dev, "cos/sin must be matching fp32 (n_pos, >=64) tables with a contiguous last axis");
  const Tensor oq = output(q_out, q, "q_out");
  const Heads ho = heads(oq, "q_out");
  p.q = q.data_ptr();
  p.q_out = oq.data_ptr();
  p.q_weight = qw.data_ptr();
  p.batch = hq.b, p.seqlen = hq.s, p.num_heads_q = hq.h, p.head_dim = 128;
  p.q_stride_b = hq.sb, p.q_stride_s = hq.ss, p.q_stride_h = hq.sh;
  p.q_out_stride_b = ho.sb, p.q_out_stride_s = ho.ss, p.q_out_stride_h = ho.sh;
  Tensor ok;
  if (k != nullptr) {
    if (k->device() != dev) throw ValueError(ONE_DEVICE);
    const Heads hk = heads(*k, "k");
    if (k->dim() != q.dim() || hk.b != hq.b || hk.s != hq.s) throw ValueError("q and k must hold the same tokens");
    if (check_norm(*kw, eps, dev, "k_weight") != p.weight_dtype)
      throw ValueError("q_weight and k_weight must have the same type");
    ok = output(k_out, *k, "k_out");
    const Heads hko = heads(ok, "k_out");
    p.k = k->data_ptr();
    p.k_out = ok.data_ptr();
    p.k_weight = kw->data_ptr();
    p.num_heads_k = hk.h;
    p.k_stride_b = hk.sb, p.k_stride_s = hk.ss, p.k_stride_h = hk.sh;
    p.k_out_stride_b = hko.sb, p.k_out_stride_s = hko.ss, p.k_out_stride_h = hko.sh;
  }
  p.eps = static_cast<float>(eps);
  p.cos = t.cos, p.sin = t.sin, p.n_pos = t.n_pos;
  p.cs_stride_pos = t.n_pos > 1 ? t.stride : std::max<int64_t>(64, t.stride & ~int64_t{3});  // (the only row's is any)
  p.pos_offset = integer(a[7]);
  if (positions != nullptr) {
    const Tensor& x = *positions;
    const bool each = q.dim() == 4 && x.dim() == 2 && x.size(0) == hq.b && x.size(1) == hq.s;
    if ((x.scalar_type() != at::kInt && x.scalar_type() != at::kLong) || x.device() != dev ||
        !(each || (x.dim() == 1 && x.size(0) == hq.s)))
      throw ValueError("positions must be int32 or int64" + on(dev) + ", one per token");
    p.positions = x.data_ptr();
    p.positions_64 = x.scalar_type() == at::kLong ? 1 : 0;
    p.pos_stride_b = each ? x.stride(0) : 0;
    p.pos_stride_s = x.stride(each ? 1 : 0);
  }
  if (hq.b * hq.s > 0)  // (tensors without tokens have no address)
    launch("atf_qk_norm_rope", lib.qk_norm_rope, dev, &p);
  // an output that the caller gave is handed back as it is
  PyObject* rq = q_out != nullptr ? Py_NewRef(a[10]) : THPVariable_Wrap(oq);
  PyObject* rk = k == nullptr ? Py_NewRef(Py_None) : k_out != nullptr ? Py_NewRef(a[11]) : THPVariable_Wrap(ok);
  PyObject* both = rq != nullptr && rk != nullptr ? PyTuple_Pack(2, rq, rk) : nullptr;
  Py_XDECREF(rq);
  Py_XDECREF(rk);
  return both;
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------ appends

struct Pages {
  int64_t pages, page, heads, s_page, s_tok, s_head;
};
Pages pages_of(const Tensor& x, PyObject* layout) {
  if (is(layout, "NHD")) return {x.size(0), x.size(1), x.size(2), x.stride(0), x.stride(1), x.stride(2)};
  if (is(layout, "HND")) return {x.size(0), x.size(2), x.size(1), x.stride(0), x.stride(2), x.stride(1)};
  throw ValueError("kv_layout must be NHD or HND");
}

// Pages and scales of an e4m3 cache (the decode's checks are append.check_e4m3_cache)
Pages check_e4m3(const Tensor& kc, const Tensor& vc, PyObject* kv_scales, PyObject* layout, AtfKvScales* s) {
  if (kc.scalar_type() != at::kFloat8_e4m3fn || vc.scalar_type() != at::kFloat8_e4m3fn)
    throw ValueError("with kv_scales the cache pages must be float8_e4m3fn");
  if (kc.dim() != 4 || kc.sizes() != vc.sizes() || kc.strides() != vc.strides())
    throw ValueError("k and v pages must have the same 4-d shape and strides");
  if (kc.size(3) != 128 || kc.stride(3) != 1) throw ValueError("the cache pages must have a contiguous head_dim of 128");
  const Pages c = pages_of(kc, layout);
  const auto both = pair(kv_scales);
  if (!both) throw ValueError("kv_scales is (k_scales, v_scales)");
  const Tensor &ks = tensor((*both)[0], "k_scales"), &vs = tensor((*both)[1], "v_scales");
  for (const Tensor* t : {&ks, &vs})
    if (t->dim() != 2 || t->size(0) != c.pages || t->size(1) != c.heads || t->scalar_type() != at::kFloat ||
        t->device() != kc.device())
      throw ValueError("k_scales and v_scales must be float32 (" + std::to_string(c.pages) + ", " + std::to_string(c.heads) +
                       ") tensors (pages, kv heads)" + on(kc.device()));
  if (ks.strides() != vs.strides()) throw ValueError("k_scales and v_scales must have the same strides");
  *s = {data<float>(ks), data<float>(vs), ks.stride(0), ks.stride(1)};
  return c;
}

// (key, value, batch_indices, positions, k_pages, v_pages, kv_indices, kv_indptr, kv_layout, cos, sin, rope_positions,
//  out_layout, kv_scales, k_norm)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 15) throw torch::TypeError("15 arguments");
  PyObject *const layout_name = a[12], *const kv_scales = a[13], *const k_norm = a[14];
  const Tensor *cos = tensor_or_none(a[9], "cos"), *sin = tensor_or_none(a[10], "sin");
  const Tensor &key = tensor(a[0], "append_key"), &value = tensor(a[1], "append_value");
  const Tensor &batch = tensor(a[2], "batch_indices"), &pos = tensor(a[3], "positions");
  const Tensor &kc = tensor(a[4], "k pages"), &vc = tensor(a[5], "v pages");
  const Tensor &indices = tensor(a[6], "kv_indices"), &indptr = tensor(a[7], "kv_indptr");
  if ((cos == nullptr) != (sin == nullptr)) throw ValueError("rope is (cos, sin)");
  const bool e4m3 = kv_scales != Py_None;
  const c10::Device dev = require_cuda({&key, &value, &kc, &vc});
  AtfAppendParams p = {};
  AtfKvScales scales = {};
  Pages c = {};
  const bool level_major = !e4m3 && kc.dim() == 5;
  if (e4m3) {
    c = check_e4m3(kc, vc, kv_scales, a[8], &scales);
    if (key.dim() != 3 || key.size(2) != 128 || key.stride(2) != 1 || key.scalar_type() != at::kBFloat16 ||
        value.scalar_type() != at::kBFloat16)
      throw ValueError("keys and values must be (tokens, kv heads, 128) bf16 with a contiguous head_dim");
  } else {
    if (kc.scalar_type() == at::kFloat8_e4m3fn || vc.scalar_type() == at::kFloat8_e4m3fn)
      throw ValueError("float8_e4m3fn pages need kv_scales");
    for (const Tensor* t : {&key, &value, &vc, &kc})
      if (t->scalar_type() != at::kBFloat16 || t->dim() < 3 ||
          (!(level_major && t == &kc) && (t->size(-1) != 128 || t->stride(-1) != 1)))
        throw ValueError("keys, values and cache pages must be bf16 with a contiguous head_dim of 128");
  }
  if (key.sizes() != value.sizes() || key.strides() != value.strides())
    throw ValueError("append_key and append_value must have the same shape and strides");
  const int layout = pair_order(layout_name);
  if (!e4m3) {
    if (key.dim() != 3) throw ValueError("keys and values must be (tokens, kv heads, 128)");
    if (level_major) {
      // (P, Hkv, 8 levels, page, 16) sorted-pair K pages (see BatchDecodeWithPagedKVCacheWrapper.run)
      if (kc.size(2) != 8 || kc.size(4) != 16 || kc.stride(4) != 1 || kc.stride(3) != 16 || vc.dim() != 4 ||
          kc.size(0) != vc.size(0))
        throw ValueError("level-major k pages must be (P, Hkv, 8, page, 16) bf16 with 16-element rows");
      if (cos != nullptr && layout != ATF_LAYOUT_SORTED_PAIR) throw ValueError("level-major k pages hold sorted-pair K");
    } else if (kc.dim() != 4 || kc.sizes() != vc.sizes() || kc.strides() != vc.strides()) {
      throw ValueError("k and v pages must have the same 4-d shape and strides");
    }
    c = pages_of(vc, a[8]);
  }
  const int64_t nnz = key.size(0);
  if (key.size(1) != c.heads) throw ValueError("append_key heads do not match the cache");
  if (layout < 0) {
    PyErr_SetObject(PyExc_KeyError, layout_name);
    throw python_error();
  }
  if (level_major && (kc.size(1) != c.heads || kc.size(3) != c.page))
    throw ValueError("level-major k pages do not match the v pages");
  AtfKNorm norm = {};
  if (k_norm != Py_None) {
    const auto both = pair(k_norm);
    if (!both) throw ValueError("k_norm is (weight, eps)");
    if (cos == nullptr) throw ValueError("k_norm needs rope: the norm stands before the rotation");
    const Tensor& w = tensor((*both)[0], "k_norm's weight");
    const double eps = PyFloat_AsDouble((*both)[1]);
    if (eps == -1.0 && PyErr_Occurred()) throw python_error();
    refuse_gradients({&w, &key});
    norm = {w.data_ptr(), check_norm(w, eps, dev, "k_norm's weight"), static_cast<float>(eps)};
  }
  const Tensor bi = narrow(batch, dev), ps = narrow(pos, dev), ip = narrow(indptr, dev, indices.numel()),
               ix = narrow(indices, dev);
  if (bi.numel() != nnz || ps.numel() != nnz) throw ValueError("batch_indices and positions need one entry per appended token");
  if (nnz == 0) Py_RETURN_NONE;
  p.append_k = key.data_ptr();
  p.append_v = value.data_ptr();
  p.nnz = nnz, p.a_stride_n = key.stride(0), p.a_stride_h = key.stride(1);
  p.batch_indices = data<int32_t>(bi);
  p.positions = data<int32_t>(ps);
  p.k_cache = kc.data_ptr();
  p.v_cache = vc.data_ptr();
  p.num_pages = c.pages;
  p.kv_stride_page = c.s_page, p.kv_stride_token = c.s_tok, p.kv_stride_head = c.s_head;
  p.num_kv_heads = static_cast<int32_t>(c.heads), p.head_dim = 128, p.page_size = static_cast<int32_t>(c.page);
  p.batch_size = static_cast<int32_t>(ip.numel()) - 1;
  p.kv_indptr = data<int32_t>(ip);
  p.kv_indices = data<int32_t>(ix);
  Tensor rp;
  if (cos != nullptr) {
    const Angles t = angles(*cos, *sin, dev, "cos/sin must be matching fp32 (n_pos, >=64) tables");
    p.cos = t.cos, p.sin = t.sin, p.cs_stride_pos = t.stride, p.n_pos = t.n_pos;
    if (const Tensor* given = tensor_or_none(a[11], "rope_positions")) {
      {
        const NoGil no_gil;
        rp = given->to(dev, at::kLong).contiguous();
      }
      if (rp.numel() != nnz) throw ValueError("rope_positions needs one entry per appended token");
      p.rope_positions = data<int64_t>(rp);
    }
  }
  p.out_layout = layout;
  p.error_flag = error_flag(dev);
  if (level_major) {
    p.k_level_major = 1;
    p.k_stride_page = kc.stride(0), p.k_stride_head = kc.stride(1), p.k_stride_level = kc.stride(2);
  }
  if (norm.weight != nullptr)
    launch("atf_paged_kv_append_norm", lib.append_norm, dev, &p, e4m3 ? &scales : nullptr, &norm);
  else if (e4m3)
    launch("atf_paged_kv_append_e4m3", lib.append_e4m3, dev, &p, &scales);
  else
    launch("atf_paged_kv_append", lib.append, dev, &p);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------ shared pages

// Checks the request table and fills its fields of a params struct
template <typename P>
c10::Device request_table(P* p, const Tensor& t, int64_t batch, int64_t page_size) {
  const c10::Device dev = require_cuda({&t});
  if (t.dim() != 2 || t.scalar_type() != at::kInt || (t.size(1) > 1 && t.stride(1) != 1))
    throw ValueError("req_pages must be an int32 (rows, pages) tensor with contiguous rows");
  const int64_t rows = t.size(0), width = t.size(1);
  if (rows < 1 || width < 1 || rows > ATF_PAGES_MAX_ROWS)
    throw ValueError("req_pages must have between 1 and " + std::to_string(ATF_PAGES_MAX_ROWS) + " rows, of one page or more");
  if (rows > 1 && t.stride(0) < width) throw ValueError("the rows of req_pages must not overlap");
  if (batch < 1 || batch > ATF_TABLES_MAX_BATCH)
    throw ValueError("between 1 and " + std::to_string(ATF_TABLES_MAX_BATCH) + " requests");
  if (batch * width >= 1 << 30) throw ValueError("requests x pages must be under 2^30");
  if (page_size < 1 || page_size > 0x7fffffff) throw ValueError("page_size must be positive");
  p->batch = static_cast<int32_t>(batch), p->page_size = static_cast<int32_t>(page_size);
  p->req_pages = data<int32_t>(t);
  p->req_stride = rows > 1 ? t.stride(0) : width;
  p->num_rows = static_cast<int32_t>(rows), p->max_req_pages = static_cast<int32_t>(width);
  p->error_flag = error_flag(dev);
  return dev;
}
Tensor request_rows(const Tensor* rows, int64_t table_rows, int64_t batch, c10::Device dev) {
  if (rows != nullptr) return index_list(*rows, "req_rows", dev, batch);
  if (table_rows < batch) throw ValueError("req_pages needs a row for each request");
  return {};
}
Tensor empty(at::IntArrayRef sizes, at::ScalarType type, c10::Device dev) {
  const NoGil no_gil;
  return at::empty(sizes, at::TensorOptions().dtype(type).device(dev));
}
Tensor new_i32(int64_t n, c10::Device dev) { return empty({n}, at::kInt, dev); }

// (src, dst, head) of one buffer
PyObject* moves(const Tensor& buf, int64_t n) {
  PyObject* s = THPVariable_Wrap(buf.narrow(0, 0, n));
  PyObject* d = THPVariable_Wrap(buf.narrow(0, n, n));
  PyObject* h = THPVariable_Wrap(buf.narrow(0, 2 * n, 1));
  PyObject* r = s != nullptr && d != nullptr && h != nullptr ? PyTuple_Pack(3, s, d, h) : nullptr;
  Py_XDECREF(s);
  Py_XDECREF(d);
  Py_XDECREF(h);
  return r;
}

// (parents, children, kv_lens, req_pages, page_size, free_pages, free_head, shared) -> (src, dst, free_head)
PyObject* fork_requests(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 8) throw torch::TypeError("8 arguments");
  const Tensor& parents = tensor(a[0], "parents");
  const Tensor& shared = tensor(a[7], "shared");
  const int64_t n = parents.numel();
  AtfForkParams p = {};
  const c10::Device dev = request_table(&p, tensor(a[3], "req_pages"), n, integer(a[4]));
  const Tensor pa = index_list(parents, "parents", dev), ch = index_list(tensor(a[1], "children"), "children", dev, n),
               le = index_list(tensor(a[2], "kv_lens"), "kv_lens", dev, n);
  const Tensor fp = index_list(tensor(a[5], "free_pages"), "free_pages", dev),
               fh = index_list(tensor(a[6], "free_head"), "free_head", dev, 1);
  p.num_pages = in_place(shared, "shared", dev);
  const Tensor out = new_i32(2 * n + 1, dev);
  int32_t* o = data<int32_t>(out);
  p.parents = data<int32_t>(pa), p.children = data<int32_t>(ch), p.kv_lens = data<int32_t>(le);
  p.shared = data<int32_t>(shared);
  p.free_head = data<int32_t>(fh);
  // an empty list still has a head: any valid address will do for its pages
  p.free_pages = fp.numel() > 0 ? data<int32_t>(fp) : p.free_head;
  p.num_free = static_cast<int32_t>(fp.numel());
  p.src = o, p.dst = o + n, p.free_head_out = o + 2 * n;
  launch("atf_fork_requests", lib.fork, dev, &p);
  return moves(out, n);
  END_HANDLE_TH_ERRORS
}

// (req_rows, kv_lens, req_pages, page_size, free_pages, free_head, shared) -> free_head
PyObject* free_requests(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 7) throw torch::TypeError("7 arguments");
  const Tensor& lens = tensor(a[1], "kv_lens");
  const Tensor &free_pages = tensor(a[4], "free_pages"), *shared = tensor_or_none(a[6], "shared");
  const int64_t n = lens.numel();
  AtfFreeParams p = {};
  const c10::Device dev = request_table(&p, tensor(a[2], "req_pages"), n, integer(a[3]));
  const Tensor le = index_list(lens, "kv_lens", dev);
  const Tensor rows = request_rows(tensor_or_none(a[0], "req_rows"), p.num_rows, n, dev);
  p.num_free = in_place(free_pages, "free_pages", dev);
  const Tensor fh = index_list(tensor(a[5], "free_head"), "free_head", dev, 1);
  if (shared != nullptr) {
    p.num_pages = in_place(*shared, "shared", dev);
    p.shared = data<int32_t>(*shared);
  }
  const Tensor out = new_i32(1, dev);
  if (rows.defined()) p.req_rows = data<int32_t>(rows);
  p.kv_lens = data<int32_t>(le);
  p.free_pages = data<int32_t>(free_pages);
  p.free_head = data<int32_t>(fh);
  p.free_head_out = data<int32_t>(out);
  launch("atf_free_requests", lib.free_, dev, &p);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// (kv_lens, req_pages, page_size, num_pages, max_moves, free_pages, req_rows, shared) -> (src, dst, free_head)
PyObject* compact_pages(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 8) throw torch::TypeError("8 arguments");
  const Tensor& lens = tensor(a[0], "kv_lens");
  const Tensor &free_pages = tensor(a[5], "free_pages"), *shared = tensor_or_none(a[7], "shared");
  const int64_t n = lens.numel(), pages = integer(a[3]), most = integer(a[4]);
  AtfCompactParams p = {};
  const c10::Device dev = request_table(&p, tensor(a[1], "req_pages"), n, integer(a[2]));
  if (pages < 1 || pages > ATF_COMPACT_MAX_PAGES)
    throw ValueError("between 1 and " + std::to_string(ATF_COMPACT_MAX_PAGES) + " pages");
  if (most < 0 || most > pages) throw ValueError("max_moves must be between 0 and num_pages");
  const Tensor le = index_list(lens, "kv_lens", dev);
  const Tensor rows = request_rows(tensor_or_none(a[6], "req_rows"), p.num_rows, n, dev);
  p.num_free = in_place(free_pages, "free_pages", dev, pages);
  if (shared != nullptr) {
    in_place(*shared, "shared", dev, pages);
    p.shared = data<int32_t>(*shared);
  }
  const Tensor out = new_i32(2 * most + 1, dev);
  int32_t* o = data<int32_t>(out);
  if (rows.defined()) p.req_rows = data<int32_t>(rows);
  p.kv_lens = data<int32_t>(le);
  p.num_pages = static_cast<int32_t>(pages), p.max_moves = static_cast<int32_t>(most);
  p.free_pages = data<int32_t>(free_pages);
  p.src = o, p.dst = o + most, p.free_head_out = o + 2 * most;
  launch("atf_compact_pages", lib.compact, dev, &p);
  return moves(out, most);
  END_HANDLE_TH_ERRORS
}

// (descriptors' address, their number, pages, device index, src, dst)
PyObject* copy_pages(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 6) throw torch::TypeError("6 arguments");
  const c10::Device dev(c10::kCUDA, static_cast<c10::DeviceIndex>(integer(a[3])));
  const Tensor src = index_list(tensor(a[4], "src"), "src", dev);
  const Tensor dst = index_list(tensor(a[5], "dst"), "dst", dev, src.size(0));
  if (src.numel() == 0) Py_RETURN_NONE;
  if (src.numel() > 0x7fffffff) throw ValueError("fewer than 2^31 pairs");
  AtfCopyPagesParams p = {};
  p.tensors_host = reinterpret_cast<const AtfPageTensor*>(integer(a[0]));
  p.num_tensors = static_cast<int32_t>(integer(a[1]));
  p.num_pages = static_cast<int32_t>(integer(a[2]));
  p.src = data<int32_t>(src);
  p.dst = data<int32_t>(dst);
  p.num_pairs = static_cast<int32_t>(src.numel());
  p.error_flag = error_flag(dev);
  launch("atf_copy_pages", lib.copy, dev, &p);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------ paged prefill

// (the plan's params' address, its device index, nhd, q, k_pages, v_pages, out, lse, return_lse) -> out, or (out, lse)
PyObject* paged_run(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 9) throw torch::TypeError("9 arguments");
  AtfPrefillPagedParams p = *reinterpret_cast<const AtfPrefillPagedParams*>(integer(a[0]));
  const c10::Device planned(c10::kCUDA, static_cast<c10::DeviceIndex>(integer(a[1])));
  const bool nhd = PyObject_IsTrue(a[2]) == 1, return_lse = PyObject_IsTrue(a[8]) == 1;
  const Tensor &q = tensor(a[3], "q"), &kc = tensor(a[4], "k pages"), &vc = tensor(a[5], "v pages");
  const Tensor *out = tensor_or_none(a[6], "out"), *lse = tensor_or_none(a[7], "lse");
  const int64_t nq = p.total_q, hq = p.num_heads_q, hkv = p.num_heads_kv, page = p.page_size;
  const c10::Device dev = require_cuda({&q, &kc, &vc});
  if (dev != planned) throw ValueError("the plan is" + on(planned) + ", the tensors are" + on(dev));
  for (const Tensor* t : {&q, &kc, &vc})
    if (t->scalar_type() != at::kBFloat16) throw torch::TypeError("q and the KV cache must be bfloat16");
  const int tok = nhd ? 1 : 2, head = nhd ? 2 : 1;
  if (vc.dim() != 4 || kc.sizes() != vc.sizes() || vc.size(tok) != page || vc.size(head) != hkv || vc.size(3) != 128 ||
      vc.size(0) < 1)
    throw ValueError("planned for k and v pages of " + std::to_string(page) + " tokens and " + std::to_string(hkv) +
                     " kv heads of 128, " + (nhd ? "NHD" : "HND"));
  const std::string shape = "(" + std::to_string(nq) + ", " + std::to_string(hq) + ", 128)";
  if (q.dim() != 3 || q.size(0) != nq || q.size(1) != hq || q.size(2) != 128) throw ValueError("planned for q " + shape);
  if (q.stride(2) != 1 || kc.stride(3) != 1 || vc.stride(3) != 1) throw ValueError("the head_dim axis must be contiguous");
  if (out != nullptr && (out->sizes() != q.sizes() || out->scalar_type() != at::kBFloat16 || out->device() != dev ||
                         out->stride(2) != 1))
    throw ValueError("out must be a bf16 " + shape + " tensor" + on(dev) + " with a contiguous head_dim axis");
  for (int i = 0; out != nullptr && i < 2; ++i)
    if (out->size(i) > 1 && out->stride(i) == 0) throw ValueError("out must not be expanded: its rows are written");
  if (lse != nullptr && (lse->dim() != 2 || lse->size(0) != nq || lse->size(1) != hq || lse->scalar_type() != at::kFloat ||
                         lse->device() != dev || !lse->is_contiguous()))
    throw ValueError("lse must be a contiguous float32 (" + std::to_string(nq) + ", " + std::to_string(hq) + ") tensor" + on(dev));
  const Tensor o = out != nullptr ? *out : empty({nq, hq, 128}, at::kBFloat16, dev);
  Tensor l;
  if (lse != nullptr)
    l = *lse;
  else if (return_lse)
    l = empty({nq, hq}, at::kFloat, dev);
  if (nq > 0) {
    p.q = q.data_ptr();
    p.k_cache = kc.data_ptr();
    p.v_cache = vc.data_ptr();
    p.out = o.data_ptr();
    p.num_pages = vc.size(0);
    if (l.defined()) p.lse = data<float>(l);
    p.q_stride_s = q.stride(0), p.q_stride_h = q.stride(1);
    p.o_stride_s = o.stride(0), p.o_stride_h = o.stride(1);
    p.k_stride_page = kc.stride(0), p.k_stride_token = kc.stride(tok), p.k_stride_head = kc.stride(head);
    p.v_stride_page = vc.stride(0), p.v_stride_token = vc.stride(tok), p.v_stride_head = vc.stride(head);
    launch("atf_prefill_paged_fwd", lib.paged, dev, &p);
  }
  PyObject* ro = out != nullptr ? Py_NewRef(a[6]) : THPVariable_Wrap(o);
  if (!return_lse) return ro;
  PyObject* rl = lse != nullptr ? Py_NewRef(a[7]) : THPVariable_Wrap(l);
  PyObject* both = ro != nullptr && rl != nullptr ? PyTuple_Pack(2, ro, rl) : nullptr;
  Py_XDECREF(ro);
  Py_XDECREF(rl);
  return both;
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------ module

// ({function name: address}, check, the package's _runtime)
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3 || !PyDict_Check(a[0])) throw torch::TypeError("init(addresses, check, runtime)");
  auto address = [&](const char* name) -> void* {
    PyObject* v = PyDict_GetItemString(a[0], name);
    if (v == nullptr) throw ValueError(std::string("no address of ") + name);
    return PyLong_AsVoidPtr(v);
  };
  auto set = [&](auto& fn, const char* name) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>(address(name)); };
  set(lib.qk_norm_rope, "atf_qk_norm_rope");
  set(lib.append, "atf_paged_kv_append");
  set(lib.append_e4m3, "atf_paged_kv_append_e4m3");
  set(lib.append_norm, "atf_paged_kv_append_norm");
  set(lib.fork, "atf_fork_requests");
  set(lib.free_, "atf_free_requests");
  set(lib.compact, "atf_compact_pages");
  set(lib.copy, "atf_copy_pages");
  set(lib.paged, "atf_prefill_paged_fwd");
  if (PyErr_Occurred()) throw python_error();
  Py_XSETREF(g_check, Py_NewRef(a[1]));
  Py_XSETREF(g_runtime, Py_NewRef(a[2]));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define ATF_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ATF_METHOD(init),          ATF_METHOD(qk_norm_rope),  ATF_METHOD(append),     ATF_METHOD(fork_requests),
                         ATF_METHOD(free_requests), ATF_METHOD(compact_pages), ATF_METHOD(copy_pages), ATF_METHOD(paged_run),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() {
  PyObject* m = PyModule_Create(&module);
  if (m != nullptr && (PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0 ||
                       PyModule_AddIntConstant(m, "version", ATF_VERSION) < 0)) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
