// Native launcher of the common operator calls (module flash_sparse_attn._host): argument checks, result and workspace
// allocation through ATen and ONE call into the C ABI. The Python launchers (ops/triton/flash_dec.py, flash_fwd.py)
// do the same in Python, which took 36 us (decode) and 44 us (forward) per call on the build machine, several times
// what the kernels of a small call take; the functions here answer in a few microseconds.
//
// They take a call only when every argument is of the ordinary kind checked below and return None otherwise: the Python
// launcher then runs, raises the contract's errors, and serves the rest (gated kind, tensor subclasses, tensors on
// another device than the current one, default windows, debug outputs). Nothing is kept between calls but the function
// addresses of the library and the per-device status words.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <cmath>
#include <cstring>
#include <optional>
#include <vector>

#include "../../include/fsa_b200.h"

namespace {

decltype(&fsa_decode) g_decode = nullptr;
decltype(&fsa_fwd) g_fwd = nullptr;
decltype(&fsa_topk_indices) g_topk = nullptr;
decltype(&fsa_pack_scales) g_pack = nullptr;
decltype(&fsa_rotary) g_rotary = nullptr;
decltype(&fsa_kv_append_rotary_workspace_ints) g_append_ints = nullptr;
decltype(&fsa_kv_append_rotary) g_append = nullptr;
decltype(&fsa_shared_prefix_workspace_bytes) g_prefix_bytes = nullptr;
decltype(&fsa_decode_shared_prefix) g_prefix = nullptr;
decltype(&fsa_rotary_axes) g_axes = nullptr;
decltype(&fsa_kv_append_quantized_workspace_ints) g_qappend_ints = nullptr;
decltype(&fsa_kv_append_quantized) g_qappend = nullptr;
decltype(&fsa_kv_read_quantized) g_qread = nullptr;
decltype(&fsa_decode_quantized_workspace_bytes) g_qdecode_bytes = nullptr;
decltype(&fsa_decode_quantized) g_qdecode = nullptr;
constexpr int MAX_DEVICES = 64;
at::Tensor* g_status[MAX_DEVICES] = {};  // registered by the package, one int32 word per device, never replaced
int g_sms[MAX_DEVICES] = {};

using at::Tensor;

// Held around the allocations and the launch: an allocation may wait for the device, a launch for room in the stream's
// queue, and other Python threads (one of which may have to feed what is waited for) go on meanwhile.
struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

// Optional tensor argument: None -> undefined. Returns false for anything but None or an exact torch.Tensor.
bool opt_tensor(PyObject* o, Tensor* t) {
  if (o == Py_None) return true;
  if (!THPVariable_CheckExact(o)) return false;
  *t = THPVariable_Unpack(o);
  return true;
}
int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return FSA_DT_BF16;
    case at::kHalf: return FSA_DT_FP16;
    case at::kFloat8_e4m3fn: return FSA_DT_E4M3;
    case at::kFloat8_e5m2: return FSA_DT_E5M2;
    default: return -1;
  }
}
// The de-quantisation scales: None, one fp32 tensor of three, or a tuple of three tensors of one element and one type, which a
// kernel packs.
struct Scales {
  Tensor packed, one[3];
  bool defined() const { return packed.defined() || one[0].defined(); }
  bool get(PyObject* o) {
    if (!PyTuple_CheckExact(o)) return opt_tensor(o, &packed);
    if (PyTuple_GET_SIZE(o) != 3) return false;
    for (int i = 0; i < 3; ++i)
      if (PyTuple_GET_ITEM(o, i) == Py_None || !opt_tensor(PyTuple_GET_ITEM(o, i), &one[i])) return false;
    return true;
  }
  int type() const { return one[0].scalar_type() == at::kFloat ? FSA_DT_F32 : dtype_code(one[0].scalar_type()); }
  bool ok(const at::Device& dev) const {
    if (packed.defined())
      return packed.scalar_type() == at::kFloat && packed.numel() == 3 && packed.device() == dev && packed.is_contiguous();
    for (const Tensor& t : one)
      if (t.scalar_type() != one[0].scalar_type() || t.numel() != 1 || t.device() != dev) return false;
    return g_pack && type() >= 0 && type() != FSA_DT_E4M3 && type() != FSA_DT_E5M2;
  }
  int pack(cudaStream_t stream) {
    if (!one[0].defined()) return FSA_OK;
    packed = at::empty({3}, one[0].options().dtype(at::kFloat));
    return g_pack(one[0].data_ptr(), one[1].data_ptr(), one[2].data_ptr(), type(), packed.data_ptr<float>(), stream);
  }
};
bool opt_double(PyObject* o, double dflt, double* v) {
  if (o == Py_None) {
    *v = dflt;
    return true;
  }
  if (PyFloat_CheckExact(o)) {
    *v = PyFloat_AS_DOUBLE(o);
    return true;
  }
  if (PyLong_CheckExact(o)) {
    *v = PyLong_AsDouble(o);
    if (!PyErr_Occurred()) return true;
    PyErr_Clear();
  }
  return false;
}
bool get_int(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &overflow);
  return !overflow && *v >= 0 && *v <= INT32_MAX;
}

bool is_fp8(int code) { return code == FSA_DT_E4M3 || code == FSA_DT_E5M2; }

// An int32 vector / matrix on the device with unit inner stride (undefined passes).
bool int_ok(const Tensor& t, const at::Device& dev, int64_t ndim) {
  return !t.defined() || (t.scalar_type() == at::kInt && t.device() == dev && t.dim() == ndim &&
                          (t.size(ndim - 1) <= 1 || t.stride(ndim - 1) == 1));
}
template <typename T>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

// q, k, v and the scales: one device (the current one), one type the kernels take as it is, a head size they take.
// Returns the type code or -1.
int check_qkv(const Tensor& q, const Tensor& k, const Tensor& v, const Scales& scale, int64_t hq, int64_t hkv, int64_t d) {
  if (!q.is_cuda() || k.device() != q.device() || v.device() != q.device()) return -1;
  const int dev = q.device().index();
  if (dev < 0 || dev >= MAX_DEVICES || !g_status[dev] || c10::cuda::current_device() != dev) return -1;
  const int code = dtype_code(q.scalar_type());
  if (code < 0 || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) return -1;
  if (is_fp8(code) != scale.defined()) return -1;
  if (scale.defined() && (!scale.ok(q.device()) || d != 128)) return -1;
  if (hkv <= 0 || hq % hkv != 0 || d % 16 != 0 || d <= 0 || d > 256) return -1;
  if (q.stride(-1) != 1 || k.stride(-1) != 1 || k.sizes() != v.sizes() || k.strides() != v.strides()) return -1;
  return code;
}

// The rule of flash_dec.py::decode_num_splits.
int64_t decode_splits(int64_t batch, int64_t heads_kv, int64_t keys, int64_t sms) {
  const int64_t slots = 2 * std::max<int64_t>(sms, 1), ctas = std::max<int64_t>(batch * heads_kv, 1);
  const int64_t fill = std::min(slots / ctas, keys / 512);
  const int64_t balance = std::min<int64_t>({32, keys / 2048, (6 * slots + ctas - 1) / ctas});
  return std::max<int64_t>({1, fill, balance});
}

PyObject* none() { Py_RETURN_NONE; }

PyObject* pair(Tensor out, Tensor lse) {
  PyObject* a = THPVariable_Wrap(std::move(out));
  PyObject* b = a ? THPVariable_Wrap(std::move(lse)) : nullptr;
  PyObject* r = b ? PyTuple_Pack(2, a, b) : nullptr;
  Py_XDECREF(a);
  Py_XDECREF(b);
  return r;
}

// decode(kind, q, k, v, softmax_scale, window_sizes, softmax_threshold, is_local, num_splits, page_table, gather,
//        seqused_k, cu_seqlens_k, max_seqlen_k, out, lse, scales) -> (out, lse), an error code, or None
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 17 || !g_decode) return none();
  HANDLE_TH_ERRORS  // torch's own translation: an allocation that fails raises torch.OutOfMemoryError
    Tensor q, k, v, win, table, gather, used, cu, out, lse;
    Scales scale;
    if (a[1] == Py_None || a[2] == Py_None || a[3] == Py_None) return none();
    if (!opt_tensor(a[1], &q) || !opt_tensor(a[2], &k) || !opt_tensor(a[3], &v) || !opt_tensor(a[5], &win) ||
        !opt_tensor(a[9], &table) || !opt_tensor(a[10], &gather) || !opt_tensor(a[11], &used) ||
        !opt_tensor(a[12], &cu) || !opt_tensor(a[14], &out) || !opt_tensor(a[15], &lse) || !scale.get(a[16]))
      return none();
    int64_t kind, splits = 0, max_k = 0;
    if (!get_int(a[0], &kind)) return none();
    if (!PyBool_Check(a[7])) return none();
    const bool local = a[7] == Py_True;
    if (local != win.defined()) return none();
    const bool varlen = cu.defined();
    if (q.dim() != 3 || k.dim() != (varlen ? 3 : 4) || (varlen && (table.defined() || !get_int(a[13], &max_k)))) return none();
    const int64_t batch = q.size(0), hq = q.size(1), d = q.size(2), hkv = k.size(-2);
    if (batch <= 0 || hq <= 0 || k.size(-1) != d || v.dim() != k.dim()) return none();
    const int code = check_qkv(q, k, v, scale, hq, hkv, d);
    if (code < 0) return none();
    const at::Device dev = q.device();
    if (!int_ok(win, dev, 2) || !int_ok(table, dev, 2) || !int_ok(gather, dev, 2) || !int_ok(used, dev, 1) || !int_ok(cu, dev, 1))
      return none();
    if (win.defined() && (win.size(1) != 4 || win.size(0) < hkv)) return none();
    if (gather.defined() && gather.size(0) != batch) return none();
    if (used.defined() && used.size(0) < batch) return none();
    if (varlen && cu.size(0) != batch + 1) return none();
    int64_t page = 0, seqlen_k;
    if (table.defined()) {
      page = k.size(1);
      if ((page != 32 && page != 64 && page != 128 && page != 256) || table.size(0) != batch) return none();
      seqlen_k = table.size(1) * page;
    } else if (varlen) {
      seqlen_k = max_k;
    } else {
      if (k.size(0) != batch) return none();
      seqlen_k = k.size(1);
    }
    const auto out_type = is_fp8(code) ? at::kBFloat16 : q.scalar_type();
    if (out.defined() && (out.sizes() != q.sizes() || out.scalar_type() != out_type || out.device() != dev || out.stride(2) != 1))
      return none();
    if (lse.defined() && (lse.dim() != 2 || lse.size(0) != batch || lse.size(1) != hq || lse.scalar_type() != at::kFloat ||
                          lse.device() != dev || lse.stride(1) != 1))
      return none();
    double sm_scale, thr;
    if (!opt_double(a[4], 1.0 / std::sqrt((double)d), &sm_scale) || !opt_double(a[6], 1.0, &thr)) return none();
    const int64_t keys = gather.defined() ? gather.size(1) : seqlen_k;
    if (a[8] == Py_None)
      splits = decode_splits(batch, hkv, keys, g_sms[dev.index()]);
    else if (!get_int(a[8], &splits))
      return none();
    splits = std::max<int64_t>(splits, 1);
    int32_t* const status = ptr<int32_t>(*g_status[dev.index()]);
    std::optional<NoGil> no_gil(std::in_place);
    if (!out.defined()) out = at::empty(q.sizes(), q.options().dtype(out_type));
    if (!lse.defined()) lse = at::empty({batch, hq}, q.options().dtype(at::kFloat));

    FsaDecArgs x = {};
    Tensor partial;
    if (splits > 1) {
      partial = at::empty({splits * batch * hq * (d + 1)}, q.options().dtype(at::kFloat));
      x.out_partial = ptr<float>(partial);
      x.lse_partial = x.out_partial + splits * batch * hq * d;
    }
    x.q = q.data_ptr();
    x.k = k.data_ptr();
    x.v = v.data_ptr();
    x.out = out.data_ptr();
    x.lse = ptr<float>(lse);
    x.cu_seqlens_k = ptr<int32_t>(cu);
    x.seqused_k = ptr<int32_t>(used);
    x.page_table = ptr<int32_t>(table);
    x.gather_kv_indices = ptr<int32_t>(gather);
    x.window_sizes = ptr<int32_t>(win);
    x.status = status;
    x.q_stride_b = q.stride(0);
    x.q_stride_h = q.stride(1);
    x.k_stride_b = varlen ? 0 : k.stride(0);
    x.k_stride_s = k.stride(-3);
    x.k_stride_h = k.stride(-2);
    x.o_stride_b = out.stride(0);
    x.o_stride_h = out.stride(1);
    x.lse_stride_b = lse.stride(0);
    x.lse_stride_h = lse.stride(1);
    x.batch = (int)batch;
    x.seqlen_k = (int)seqlen_k;
    x.total_k = varlen ? (int)k.size(0) : 0;
    x.heads_q = (int)hq;
    x.heads_kv = (int)hkv;
    x.head_dim = (int)d;
    if (gather.defined()) {
      x.topk = (int)gather.size(1);
      x.gather_stride = (int)gather.stride(0);
    }
    if (table.defined()) {
      x.num_pages = (int)k.size(0);
      x.page_size = (int)page;
      x.page_table_stride = (int)table.stride(0);
    }
    x.window_stride = win.defined() ? (int)win.stride(0) : 0;
    x.num_splits = (int)splits;
    x.kind = (int)kind;
    x.dtype = code;
    x.flags = (local ? FSA_F_LOCAL : 0) | FSA_F_LOGSIGMOID | FSA_F_SCRATCH_PARTIALS;
    x.softmax_scale = (float)sm_scale;
    x.softmax_threshold = (float)thr;
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    int rc = scale.pack(stream);
    x.qkv_scale = ptr<float>(scale.packed);
    if (rc == FSA_OK) rc = g_decode(&x, stream);
    no_gil.reset();
    if (rc != FSA_OK) return PyLong_FromLong(rc);
    return pair(std::move(out), std::move(lse));
  END_HANDLE_TH_ERRORS
}

// forward(kind, q, k, v, is_causal, softmax_scale, window_sizes, softmax_threshold, is_local, num_splits, pack_gqa,
//         cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, page_table, seqused_q, seqused_k, out, lse, scales)
//         -> (out, lse), an error code, or None. num_splits: what the launcher settled on (1: unsplit).
PyObject* forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 21 || !g_fwd) return none();
  HANDLE_TH_ERRORS  // torch's own translation: an allocation that fails raises torch.OutOfMemoryError
    Tensor q, k, v, win, cu_q, cu_k, table, used_q, used_k, out, lse;
    Scales scale;
    if (a[1] == Py_None || a[2] == Py_None || a[3] == Py_None) return none();
    if (!opt_tensor(a[1], &q) || !opt_tensor(a[2], &k) || !opt_tensor(a[3], &v) || !opt_tensor(a[6], &win) ||
        !opt_tensor(a[11], &cu_q) || !opt_tensor(a[12], &cu_k) || !opt_tensor(a[15], &table) ||
        !opt_tensor(a[16], &used_q) || !opt_tensor(a[17], &used_k) || !opt_tensor(a[18], &out) ||
        !opt_tensor(a[19], &lse) || !scale.get(a[20]))
      return none();
    int64_t kind, splits, max_q = 0, max_k = 0;
    if (!get_int(a[0], &kind) || !get_int(a[9], &splits) || splits < 1) return none();
    if (!PyBool_Check(a[4]) || !PyBool_Check(a[8]) || !PyBool_Check(a[10])) return none();
    const bool causal = a[4] == Py_True, local = a[8] == Py_True, pack = a[10] == Py_True;
    if (local != win.defined()) return none();
    const bool varlen = cu_q.defined();
    if (varlen != cu_k.defined() || (varlen && (table.defined() || !get_int(a[13], &max_q) || !get_int(a[14], &max_k))))
      return none();
    if (q.dim() != (varlen ? 3 : 4) || k.dim() != q.dim() || v.dim() != k.dim()) return none();
    const int64_t hq = q.size(-2), d = q.size(-1), hkv = k.size(-2);
    if (hq <= 0 || k.size(-1) != d) return none();
    const int code = check_qkv(q, k, v, scale, hq, hkv, d);
    if (code < 0 || !q.is_contiguous() || !k.is_contiguous()) return none();
    const at::Device dev = q.device();
    if (!int_ok(win, dev, 2) || !int_ok(table, dev, 2) || !int_ok(used_q, dev, 1) || !int_ok(used_k, dev, 1) ||
        !int_ok(cu_q, dev, 1) || !int_ok(cu_k, dev, 1))
      return none();
    if (win.defined() && (win.size(1) != 4 || win.size(0) < hkv)) return none();
    int64_t batch, seqlen_q, seqlen_k, total_q = 0, total_k = 0, page = 0;
    if (varlen) {
      batch = cu_q.size(0) - 1;
      if (cu_k.size(0) != batch + 1) return none();
      seqlen_q = max_q;
      seqlen_k = max_k;
      total_q = q.size(0);
      total_k = k.size(0);
    } else {
      batch = q.size(0);
      seqlen_q = q.size(1);
      if (table.defined()) {
        page = k.size(1);
        if ((page != 32 && page != 64 && page != 128 && page != 256) || table.size(0) != batch) return none();
        seqlen_k = table.size(1) * page;
      } else {
        if (k.size(0) != batch) return none();
        seqlen_k = k.size(1);
      }
    }
    if (batch <= 0 || seqlen_q <= 0 || seqlen_k <= 0) return none();
    if ((used_q.defined() && used_q.size(0) < batch) || (used_k.defined() && used_k.size(0) < batch)) return none();
    if (splits > 1 && varlen && used_q.defined()) return none();  // the partials' unused rows want a fill there
    const auto out_type = is_fp8(code) ? at::kBFloat16 : q.scalar_type();
    if (out.defined() && (out.sizes() != q.sizes() || out.scalar_type() != out_type || out.device() != dev || out.stride(-1) != 1))
      return none();
    const int64_t l0 = varlen ? hq : batch, l1 = varlen ? total_q : hq;
    if (lse.defined() && (lse.dim() != (varlen ? 2 : 3) || lse.size(0) != l0 || lse.size(1) != l1 ||
                          (!varlen && lse.size(2) != seqlen_q) || lse.scalar_type() != at::kFloat || lse.device() != dev ||
                          lse.stride(-1) != 1))
      return none();
    double sm_scale, thr;
    if (!opt_double(a[5], 1.0 / std::sqrt((double)d), &sm_scale) || !opt_double(a[7], 1.0, &thr)) return none();
    int32_t* const status = ptr<int32_t>(*g_status[dev.index()]);
    std::optional<NoGil> no_gil(std::in_place);
    if (!out.defined()) out = at::empty(q.sizes(), q.options().dtype(out_type));
    if (!lse.defined())
      lse = varlen ? at::empty({hq, total_q}, q.options().dtype(at::kFloat))
                   : at::empty({batch, hq, seqlen_q}, q.options().dtype(at::kFloat));

    FsaFwdArgs x = {};
    Tensor partial;
    if (splits > 1) {
      const int64_t rows = varlen ? total_q : batch * seqlen_q;
      partial = at::empty({splits * rows * hq * (d + 1)}, q.options().dtype(at::kFloat));
      x.out_partial = ptr<float>(partial);
      x.lse_partial = x.out_partial + splits * rows * hq * d;
    }
    x.q = q.data_ptr();
    x.k = k.data_ptr();
    x.v = v.data_ptr();
    x.out = out.data_ptr();
    x.lse = ptr<float>(lse);
    x.cu_seqlens_q = ptr<int32_t>(cu_q);
    x.cu_seqlens_k = ptr<int32_t>(cu_k);
    x.seqused_q = ptr<int32_t>(used_q);
    x.seqused_k = ptr<int32_t>(used_k);
    x.page_table = ptr<int32_t>(table);
    x.window_sizes = ptr<int32_t>(win);
    x.status = status;
    x.q_stride_b = varlen ? 0 : q.stride(0);
    x.q_stride_s = q.stride(-3);
    x.q_stride_h = q.stride(-2);
    x.k_stride_b = x.v_stride_b = varlen ? 0 : k.stride(0);
    x.k_stride_s = x.v_stride_s = k.stride(-3);
    x.k_stride_h = x.v_stride_h = k.stride(-2);
    x.o_stride_b = varlen ? 0 : out.stride(0);
    x.o_stride_s = out.stride(-3);
    x.o_stride_h = out.stride(-2);
    x.lse_stride_b = varlen ? 0 : lse.stride(0);
    x.lse_stride_h = varlen ? lse.stride(0) : lse.stride(1);
    x.batch = (int)batch;
    x.seqlen_q = (int)seqlen_q;
    x.seqlen_k = (int)seqlen_k;
    x.total_q = (int)total_q;
    x.total_k = (int)total_k;
    x.heads_q = (int)hq;
    x.heads_kv = (int)hkv;
    x.head_dim = (int)d;
    if (table.defined()) {
      x.num_pages = (int)k.size(0);
      x.page_size = (int)page;
      x.page_table_stride = (int)table.stride(0);
    }
    x.window_stride = win.defined() ? (int)win.stride(0) : 0;
    x.num_splits = (int)splits;
    x.tile_m = x.tile_n = 128;
    x.kind = (int)kind;
    x.dtype = code;
    x.flags = (causal ? FSA_F_CAUSAL : 0) | (local ? FSA_F_LOCAL : 0) | (splits > 1 ? FSA_F_SPLIT : 0) |
              (pack && hq > hkv ? FSA_F_PACK_GQA : 0) | FSA_F_LOGSIGMOID | FSA_F_ADAPT_GATE;
    x.softmax_scale = (float)sm_scale;
    x.softmax_threshold = (float)thr;
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    int rc = scale.pack(stream);
    x.qkv_scale = ptr<float>(scale.packed);
    if (rc == FSA_OK) rc = g_fwd(&x, stream);
    no_gil.reset();
    if (rc != FSA_OK) return PyLong_FromLong(rc);
    return pair(std::move(out), std::move(lse));
  END_HANDLE_TH_ERRORS
}

// topk(scores, k, positions as int64) -> positions, an error code, or None. Scores of 16 or 32 bits whose rows are equally far apart.
PyObject* topk(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3 || !g_topk || !THPVariable_CheckExact(a[0]) || !PyBool_Check(a[2])) return none();
  HANDLE_TH_ERRORS
    int64_t k;
    const Tensor x = THPVariable_Unpack(a[0]);
    if (!get_int(a[1], &k) || !x.is_cuda() || x.dim() < 1) return none();
    const int dev = x.device().index();
    if (dev < 0 || dev >= MAX_DEVICES || c10::cuda::current_device() != dev) return none();
    const int type = x.scalar_type() == at::kFloat ? FSA_DT_F32 : dtype_code(x.scalar_type());
    const int64_t len = x.size(-1);
    if (type < 0 || is_fp8(type) || k <= 0 || k > len || len > INT32_MAX || x.numel() == 0) return none();
    if (!x.is_contiguous() && (x.dim() != 2 || x.stride(1) != 1 || x.stride(0) < len)) return none();
    const int64_t rows = x.numel() / len, pitch = x.is_contiguous() ? len : x.stride(0);
    if (rows > INT32_MAX) return none();
    auto shape = x.sizes().vec();
    shape.back() = k;
    const bool wide = a[2] == Py_True;
    std::optional<NoGil> no_gil(std::in_place);
    Tensor out = at::empty(shape, x.options().dtype(wide ? at::kLong : at::kInt));
    const int rc = g_topk(x.data_ptr(), type, (int)rows, (int)len, pitch, (int)k, out.data_ptr(), wide ? 1 : 0,
                          c10::cuda::getCurrentCUDAStream(dev).stream());
    no_gil.reset();
    if (rc != FSA_OK) return PyLong_FromLong(rc);
    return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---- rotary positions -------------------------------------------------------------------------------------------------

int table_code(at::ScalarType t) { return t == at::kFloat ? FSA_DT_F32 : (t == at::kBFloat16 ? FSA_DT_BF16 : (t == at::kHalf ? FSA_DT_FP16 : -1)); }

// The tables' contract (rotary.py::check_tables).
bool tables_ok(const Tensor& cos, const Tensor& sin, int64_t head_dim, const at::Device& dev) {
  return cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.strides() == sin.strides() && cos.scalar_type() == sin.scalar_type() &&
         table_code(cos.scalar_type()) >= 0 && cos.device() == dev && sin.device() == dev && cos.size(0) > 0 && cos.size(1) > 0 &&
         cos.size(0) <= INT32_MAX && 2 * cos.size(1) <= head_dim && (cos.size(1) == 1 || cos.stride(1) == 1) && !cos.requires_grad() &&
         !sin.requires_grad();
}

// None, an int, or an int32 tensor [batch].
bool get_offsets(PyObject* o, int64_t* value, Tensor* t) {
  *value = 0;
  if (o == Py_None || THPVariable_CheckExact(o)) return opt_tensor(o, t);
  int overflow = 0;
  if (!PyLong_CheckExact(o)) return false;
  *value = PyLong_AsLongLongAndOverflow(o, &overflow);
  return !overflow && *value >= INT32_MIN && *value <= INT32_MAX;
}
bool offsets_ok(const Tensor& t, int64_t batch, const at::Device& dev) {
  return !t.defined() || (t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == batch && t.is_contiguous() && t.device() == dev);
}

// What a rotation needs beside the tensors it turns. Those are checked before it is made.
struct RotaryCall {
  Tensor cos, sin, offsets, ids, cu;
  int64_t offset = 0;
  bool interleaved = false, transposed = false;
};

Tensor rows_of(const Tensor& t) { return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

// One launch for the tensors that are defined (one of them is).
void rotary_launch(const RotaryCall& c, const Tensor& q_in, const Tensor& k_in, Tensor* q_out, Tensor* k_out) {
  const Tensor& any = q_in.defined() ? q_in : k_in;
  const int dev = any.device().index();
  const Tensor q = q_in.defined() ? rows_of(q_in) : q_in, k = k_in.defined() ? rows_of(k_in) : k_in;
  FsaRotaryArgs x = {};
  auto put = [](const Tensor& t, int64_t* sb, int64_t* ss, int64_t* sh) {
    *sb = t.dim() == 3 ? 0 : t.stride(0);
    *ss = t.stride(-3);
    *sh = t.stride(-2);
  };
  if (q.defined()) {
    *q_out = at::empty(q.sizes(), q.options());
    x.q = q.data_ptr();
    x.q_out = q_out->data_ptr();
    x.heads_q = (int)q.size(-2);
    put(q, &x.q_stride_b, &x.q_stride_s, &x.q_stride_h);
    put(*q_out, &x.q_out_stride_b, &x.q_out_stride_s, &x.q_out_stride_h);
  }
  if (k.defined()) {
    *k_out = at::empty(k.sizes(), k.options());
    x.k = k.data_ptr();
    x.k_out = k_out->data_ptr();
    x.heads_k = (int)k.size(-2);
    put(k, &x.k_stride_b, &x.k_stride_s, &x.k_stride_h);
    put(*k_out, &x.k_out_stride_b, &x.k_out_stride_s, &x.k_out_stride_h);
  }
  if ((q.defined() ? q.numel() : 0) + (k.defined() ? k.numel() : 0) == 0) return;
  x.cos = c.cos.data_ptr();
  x.sin = c.sin.data_ptr();
  x.cu_seqlens = ptr<int32_t>(c.cu);
  x.seqlen_offsets = ptr<int32_t>(c.offsets);
  x.position_ids = ptr<void>(c.ids);
  x.status = ptr<int32_t>(*g_status[dev]);
  if (c.ids.defined()) {
    x.position_ids_int64 = c.ids.scalar_type() == at::kLong;
    x.position_stride_b = c.ids.dim() == 2 && c.ids.size(0) > 1 ? c.ids.stride(0) : 0;
    x.position_stride_s = c.ids.stride(-1);
  }
  x.table_stride = c.cos.stride(0);
  x.table_rows = (int)c.cos.size(0);
  x.rotary_dim = (int)(2 * c.cos.size(1));
  x.table_dtype = table_code(c.cos.scalar_type());
  if (c.cu.defined()) {
    x.batch = (int)c.cu.size(0) - 1;
    x.total = (int)any.size(0);
  } else {
    x.batch = any.dim() == 4 ? (int)any.size(0) : 1;
    x.seqlen = (int)any.size(-3);
  }
  x.head_dim = (int)any.size(-1);
  x.offset = (int)c.offset;
  x.dtype = dtype_code(any.scalar_type());
  x.interleaved = c.interleaved;
  x.transposed = c.transposed;
  const int rc = g_rotary(&x, c10::cuda::getCurrentCUDAStream(dev).stream());
  TORCH_CHECK(rc == FSA_OK, "fsa_rotary failed (code ", rc, ")");
}

// The rotation with its gradient, which is the transposed rotation of the gradients - a rotation again, so that it has a gradient too.
// Results are those of the tensors that are defined, in their order.
struct RotaryFn : torch::autograd::Function<RotaryFn> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const std::optional<Tensor>& q_in,
                                                const std::optional<Tensor>& k_in, const RotaryCall& c) {
    const Tensor q = q_in.value_or(Tensor()), k = k_in.value_or(Tensor());
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({c.cos, c.sin, c.offsets, c.ids, c.cu});
    ctx->saved_data["offset"] = c.offset;
    ctx->saved_data["form"] = int64_t(c.interleaved) | int64_t(c.transposed) << 1 | int64_t(q.defined()) << 2 | int64_t(k.defined()) << 3;
    return launch(q, k, c);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const int64_t form = ctx->saved_data["form"].toInt();
    const RotaryCall c{saved[0], saved[1], saved[2], saved[3], saved[4], ctx->saved_data["offset"].toInt(), (form & 1) != 0, (form & 2) == 0};
    Tensor in[2];
    size_t n = 0;
    for (int i = 0; i < 2; ++i)
      if (form & (4 << i)) {
        if (ctx->needs_input_grad(n)) in[i] = grads[n];  // (tensors that are left out have no edge)
        ++n;
      }
    torch::autograd::variable_list out(3);  // one entry for every argument of forward
    if (!in[0].defined() && !in[1].defined()) return out;
    const auto turned = turn(in[0], in[1], c);
    n = 0;
    for (int i = 0; i < 2; ++i)
      if (in[i].defined()) out[i] = turned[n++];
    return out;
  }
  static torch::autograd::variable_list launch(const Tensor& q, const Tensor& k, const RotaryCall& c) {
    Tensor q_out, k_out;
    rotary_launch(c, q, k, &q_out, &k_out);
    if (!k.defined()) return {q_out};
    if (!q.defined()) return {k_out};
    return {q_out, k_out};
  }
  static torch::autograd::variable_list turn(const Tensor& q, const Tensor& k, const RotaryCall& c) {
    // (a tangent is seen by the Function, which says that it has none for its results)
    auto seen = [](const Tensor& t) { return t.defined() && ((at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined()); };
    const bool records = seen(q) || seen(k);
    auto maybe = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
    return records ? apply(maybe(q), maybe(k), c) : launch(q, k, c);
  }
};

// rotary(q, k, cos, sin, seqlen_offsets, position_ids, cu_seqlens, interleaved) -> q or (q, k), or None. k may be None.
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8 || !g_rotary) return none();
  HANDLE_TH_ERRORS
    Tensor q, k;
    RotaryCall c;
    if (a[0] == Py_None || a[2] == Py_None || a[3] == Py_None || !opt_tensor(a[0], &q) || !opt_tensor(a[1], &k) || !opt_tensor(a[2], &c.cos) ||
        !opt_tensor(a[3], &c.sin) || !get_offsets(a[4], &c.offset, &c.offsets) || !opt_tensor(a[5], &c.ids) || !opt_tensor(a[6], &c.cu) ||
        !PyBool_Check(a[7]))
      return none();
    c.interleaved = a[7] == Py_True;
    const bool packed = c.cu.defined();
    if (!q.is_cuda() || (q.dim() != 3 && q.dim() != 4) || (packed && q.dim() != 3) || (!packed && q.dim() == 3 && !c.ids.defined())) return none();
    const at::Device dev = q.device();
    if (dev.index() < 0 || dev.index() >= MAX_DEVICES || !g_status[dev.index()] || c10::cuda::current_device() != dev.index()) return none();
    if (q.scalar_type() != at::kBFloat16 && q.scalar_type() != at::kHalf) return none();
    const int64_t d = q.size(-1), batch = packed ? c.cu.size(0) - 1 : (q.dim() == 4 ? q.size(0) : 1);
    if (batch <= 0 || q.numel() == 0 || q.numel() / (q.size(-2) * d) > INT32_MAX || !tables_ok(c.cos, c.sin, d, dev)) return none();
    if (k.defined()) {
      if (k.dim() != q.dim() || k.scalar_type() != q.scalar_type() || k.device() != dev || k.size(-1) != d || k.numel() == 0) return none();
      for (int64_t i = 0; i < q.dim() - 2; ++i)
        if (k.size(i) != q.size(i)) return none();
    }
    if (packed && (c.cu.scalar_type() != at::kInt || c.cu.dim() != 1 || !c.cu.is_contiguous() || c.cu.device() != dev)) return none();
    if (!offsets_ok(c.offsets, batch, dev)) return none();
    if (c.ids.defined()) {
      if (packed || a[4] != Py_None || (c.ids.scalar_type() != at::kInt && c.ids.scalar_type() != at::kLong) || c.ids.device() != dev ||
          c.ids.dim() != q.dim() - 2 || c.ids.size(-1) != q.size(-3) || (q.dim() == 4 && c.ids.size(0) != 1 && c.ids.size(0) != batch))
        return none();
    }
    std::optional<NoGil> no_gil(std::in_place);
    auto out = RotaryFn::turn(q, k, c);
    no_gil.reset();
    return k.defined() ? pair(std::move(out[0]), std::move(out[1])) : THPVariable_Wrap(std::move(out[0]));
  END_HANDLE_TH_ERRORS
}

// What a kernel wrote in place: a graph that kept it for its gradient has to notice (tensors of inference mode are in no graph).
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// append(q, k_new, v_new, k_cache, v_cache, seqused_k, cos, sin, page_table, free_pages, free_count, cu_seqlens_new, seqlen_offsets,
//        interleaved, q_scale, k_scale, v_scale, advance, out) -> the turned queries (True without queries), an error code, or None
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 19 || !g_append) return none();
  HANDLE_TH_ERRORS
    Tensor q, k, v, kc, vc, used, cos, sin, table, free, count, cu, offsets, qs, ks, vs, out;
    Tensor* const into[19] = {&q, &k, &v, &kc, &vc, &used, &cos, &sin, &table, &free, &count, &cu, nullptr, nullptr, &qs, &ks, &vs, nullptr, &out};
    for (int i = 0; i < 19; ++i)
      if (into[i] && !opt_tensor(a[i], into[i])) return none();
    for (int i = 1; i < 8; ++i)
      if (!into[i]->defined()) return none();
    int64_t offset;
    if (!get_offsets(a[12], &offset, &offsets) || !PyBool_Check(a[13]) || !PyBool_Check(a[17])) return none();
    const int64_t dims = cu.defined() ? 3 : 4;
    if (!k.is_cuda() || k.dim() != dims || k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type()) return none();
    const at::Device dev = k.device();
    if (dev.index() < 0 || dev.index() >= MAX_DEVICES || !g_status[dev.index()] || c10::cuda::current_device() != dev.index()) return none();
    for (int i = 0; i < 19; ++i)
      if (into[i] && into[i]->defined() && into[i]->device() != dev) return none();
    const auto type = k.scalar_type();
    if (type != at::kBFloat16 && type != at::kHalf) return none();
    const int64_t hkv = k.size(-2), d = k.size(-1), batch = used.numel();
    auto flat = [d](const Tensor& t) { return !t.defined() || t.size(-1) == 1 || t.stride(-1) == 1; };
    if (hkv <= 0 || d <= 0 || batch <= 0 || k.numel() == 0 || !flat(k) || !flat(v)) return none();
    for (const Tensor* t : {&kc, &vc, &used, &table, &free, &out})
      if (t->defined())
        for (int64_t i = 0; i < t->dim(); ++i)
          if (t->size(i) > 1 && t->stride(i) <= 0) return none();
    if (q.defined()) {
      if (q.dim() != dims || q.scalar_type() != type || q.size(-1) != d || q.size(-2) <= 0 || q.size(-2) % hkv || !flat(q)) return none();
      for (int64_t i = 0; i < dims - 2; ++i)
        if (q.size(i) != k.size(i)) return none();
    }
    if (kc.dim() != 4 || kc.sizes() != vc.sizes() || kc.scalar_type() != vc.scalar_type() || kc.size(2) != hkv || kc.size(3) != d || !flat(kc) ||
        !flat(vc))
      return none();
    const int cache_code = dtype_code(kc.scalar_type());
    const bool fp8 = is_fp8(cache_code);
    if (!fp8 && kc.scalar_type() != type) return none();
    for (const Tensor* t : {&qs, &ks, &vs})
      if (fp8 ? (t != &qs || q.defined()) && !(t->defined() && t->scalar_type() == at::kFloat && t->numel() == 1) : t->defined()) return none();
    if (used.scalar_type() != at::kInt || used.dim() != 1 || !used.is_contiguous()) return none();
    if (cu.defined() ? (cu.scalar_type() != at::kInt || cu.dim() != 1 || !cu.is_contiguous() || cu.size(0) != batch + 1) : k.size(0) != batch)
      return none();
    if (table.defined()) {
      if (!int_ok(table, dev, 2) || table.size(0) != batch || table.size(1) <= 0 || kc.size(0) <= 0 || kc.size(1) <= 0 || free.defined() != count.defined())
        return none();
      if (free.defined() && (free.scalar_type() != at::kInt || !free.is_contiguous() || count.scalar_type() != at::kInt || count.numel() != 1))
        return none();
    } else if (kc.size(0) != batch || kc.size(1) <= 0 || free.defined() || count.defined()) {
      return none();
    }
    if (!tables_ok(cos, sin, d, dev) || !offsets_ok(offsets, batch, dev)) return none();
    const auto out_type = fp8 ? kc.scalar_type() : type;
    if (out.defined() && (!q.defined() || out.sizes() != q.sizes() || out.scalar_type() != out_type || !flat(out))) return none();
    std::optional<NoGil> no_gil(std::in_place);
    if (q.defined() && !out.defined()) out = at::empty(q.sizes(), q.options().dtype(out_type));
    FsaKvAppendRotaryArgs x = {};
    auto put = [](const Tensor& t, int64_t* sb, int64_t* ss, int64_t* sh) {
      *sb = t.dim() == 3 ? 0 : t.stride(0);
      *ss = t.stride(-3);
      *sh = t.stride(-2);
    };
    if (q.defined()) {
      x.q = q.data_ptr();
      x.q_out = out.data_ptr();
      x.heads_q = (int)q.size(-2);
      put(q, &x.q_stride_b, &x.q_stride_s, &x.q_stride_h);
      put(out, &x.q_out_stride_b, &x.q_out_stride_s, &x.q_out_stride_h);
    }
    x.k_new = k.data_ptr();
    x.v_new = v.data_ptr();
    x.k_cache = kc.data_ptr();
    x.v_cache = vc.data_ptr();
    put(k, &x.k_stride_b, &x.k_stride_s, &x.k_stride_h);
    put(v, &x.v_stride_b, &x.v_stride_s, &x.v_stride_h);
    put(kc, &x.k_cache_stride_b, &x.k_cache_stride_s, &x.k_cache_stride_h);
    put(vc, &x.v_cache_stride_b, &x.v_cache_stride_s, &x.v_cache_stride_h);
    x.cos = cos.data_ptr();
    x.sin = sin.data_ptr();
    x.seqused_k = ptr<int32_t>(used);
    x.page_table = ptr<int32_t>(table);
    x.free_pages = ptr<int32_t>(free);
    x.free_count = ptr<int32_t>(count);
    x.cu_seqlens_new = ptr<int32_t>(cu);
    x.seqlen_offsets = ptr<int32_t>(offsets);
    if (fp8) {
      x.q_scale = ptr<float>(qs);
      x.k_scale = ptr<float>(ks);
      x.v_scale = ptr<float>(vs);
    }
    x.status = ptr<int32_t>(*g_status[dev.index()]);
    x.table_stride = cos.stride(0);
    x.table_rows = (int)cos.size(0);
    x.rotary_dim = (int)(2 * cos.size(1));
    x.table_dtype = table_code(cos.scalar_type());
    x.batch = (int)batch;
    if (cu.defined())
      x.total = (int)k.size(0);
    else
      x.new_tokens = (int)k.size(1);
    x.heads_kv = (int)hkv;
    x.head_dim = (int)d;
    x.offset = (int)offset;
    if (table.defined()) {
      x.num_pages = (int)kc.size(0);
      x.page_size = (int)kc.size(1);
      x.max_pages = (int)table.size(1);
      x.page_table_stride = table.stride(0);
    } else {
      x.capacity = (int)kc.size(1);
    }
    x.dtype = dtype_code(type);
    x.cache_dtype = cache_code;
    x.interleaved = a[13] == Py_True;
    x.advance = a[17] == Py_True;
    const int64_t ints = g_append_ints(&x);
    Tensor place;
    if (ints > 0) place = at::empty({ints}, used.options());
    x.place_ws = ptr<int32_t>(place);
    const int rc = g_append(&x, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
    if (rc == FSA_OK) {
      if (x.advance) written(used);
      if (a[18] != Py_None) written(out);
    }
    no_gil.reset();
    if (rc != FSA_OK) return PyLong_FromLong(rc);
    if (!q.defined()) Py_RETURN_TRUE;
    if (a[18] != Py_None) {
      Py_INCREF(a[18]);
      return a[18];
    }
    return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// shared_prefix(q, k, v, prefix_k, prefix_v, softmax_scale, page_table, seqused_k, prefix_page_table, prefix_seqused, out, lse)
//   -> (out, lse), an error code, or None
PyObject* shared_prefix(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 12 || !g_prefix || !g_prefix_bytes) return none();
  HANDLE_TH_ERRORS
    Tensor q, k, v, pk, pv, table, used, ptable, pused, out, lse;
    Tensor* const into[12] = {&q, &k, &v, &pk, &pv, nullptr, &table, &used, &ptable, &pused, &out, &lse};
    for (int i = 0; i < 12; ++i)
      if (into[i] && !opt_tensor(a[i], into[i])) return none();
    for (int i = 0; i < 5; ++i)
      if (!into[i]->defined()) return none();
    if (q.dim() != 3 || k.dim() != 4 || k.sizes() != v.sizes() || pk.sizes() != pv.sizes() || pk.dim() != (ptable.defined() ? 4 : 3)) return none();
    const int64_t batch = q.size(0), hq = q.size(1), d = q.size(2), hkv = k.size(2);
    if (batch <= 0 || hq <= 0 || hkv <= 0 || hq % hkv || k.size(3) != d || pk.size(-1) != d || pk.size(-2) != hkv || d <= 0 || d > 128 || d % 16)
      return none();
    const at::Device dev = q.device();
    if (!q.is_cuda() || dev.index() < 0 || dev.index() >= MAX_DEVICES || !g_status[dev.index()] || c10::cuda::current_device() != dev.index())
      return none();
    const auto type = q.scalar_type();
    if (type != at::kBFloat16 && type != at::kHalf) return none();
    auto rows_ok = [&](const Tensor& t) {  // the queries' type, on their device, rows on 16-byte boundaries
      if (t.scalar_type() != type || t.device() != dev) return false;
      if (t.numel() == 0) return true;
      if (t.stride(-1) != 1 || (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15)) return false;
      for (int64_t i = 0; i + 1 < t.dim(); ++i)
        if (t.size(i) != 1 && (t.stride(i) <= 0 || t.stride(i) % 8)) return false;
      return true;
    };
    for (const Tensor* t : {&q, &k, &v, &pk, &pv})
      if (!rows_ok(*t)) return none();
    auto page_ok = [](int64_t p) { return p == 32 || p == 64 || p == 128 || p == 256; };
    if (table.defined() ? !(int_ok(table, dev, 2) && table.is_contiguous() && table.size(0) == batch && table.size(1) > 0 && k.size(0) > 0 && page_ok(k.size(1)))
                        : k.size(0) != batch)
      return none();
    if (ptable.defined() && !(int_ok(ptable, dev, 1) && ptable.is_contiguous() && ptable.numel() > 0 && pk.size(0) > 0 && page_ok(pk.size(1)))) return none();
    if (!int_ok(used, dev, 1) || (used.defined() && (used.size(0) != batch || !used.is_contiguous()))) return none();
    if (pused.defined() && !(pused.scalar_type() == at::kInt && pused.device() == dev && pused.numel() == 1)) return none();
    if (out.defined() && (out.sizes() != q.sizes() || out.scalar_type() != type || out.device() != dev || out.stride(2) != 1)) return none();
    if (lse.defined() && (lse.dim() != 2 || lse.size(0) != batch || lse.size(1) != hq || lse.scalar_type() != at::kFloat || lse.device() != dev ||
                          lse.stride(1) != 1))
      return none();
    for (const Tensor* t : {&out, &lse})
      if (t->defined())
        for (int64_t i = 0; i < t->dim(); ++i)
          if (t->size(i) > 1 && t->stride(i) <= 0) return none();
    double scale;
    if (!opt_double(a[5], 1.0 / std::sqrt((double)d), &scale) || !(scale > 0.0) || std::isinf(scale)) return none();
    std::optional<NoGil> no_gil(std::in_place);
    if (!out.defined()) out = at::empty(q.sizes(), q.options());
    if (!lse.defined()) lse = at::empty({batch, hq}, q.options().dtype(at::kFloat));
    FsaSharedPrefixArgs x = {};
    x.q = q.data_ptr();
    x.k = k.data_ptr();
    x.v = v.data_ptr();
    x.prefix_k = pk.data_ptr();
    x.prefix_v = pv.data_ptr();
    x.out = out.data_ptr();
    x.lse = ptr<float>(lse);
    x.seqused_k = ptr<int32_t>(used);
    x.page_table = ptr<int32_t>(table);
    x.prefix_seqused = ptr<int32_t>(pused);
    x.prefix_page_table = ptr<int32_t>(ptable);
    x.status = ptr<int32_t>(*g_status[dev.index()]);
    x.q_stride_b = q.stride(0);
    x.q_stride_h = q.stride(1);
    x.o_stride_b = out.stride(0);
    x.o_stride_h = out.stride(1);
    x.lse_stride_b = lse.stride(0);
    x.lse_stride_h = lse.stride(1);
    x.k_stride_b = k.stride(0);
    x.k_stride_s = k.stride(1);
    x.k_stride_h = k.stride(2);
    x.v_stride_b = v.stride(0);
    x.v_stride_s = v.stride(1);
    x.v_stride_h = v.stride(2);
    x.prefix_k_stride_s = pk.stride(-3);
    x.prefix_k_stride_h = pk.stride(-2);
    x.prefix_v_stride_s = pv.stride(-3);
    x.prefix_v_stride_h = pv.stride(-2);
    x.batch = (int)batch;
    x.heads_q = (int)hq;
    x.heads_kv = (int)hkv;
    x.head_dim = (int)d;
    if (table.defined()) {
      x.num_pages = (int)k.size(0);
      x.page_size = (int)k.size(1);
      x.max_pages = (int)table.size(1);
    } else {
      x.seqlen_k = (int)k.size(1);
    }
    if (ptable.defined()) {
      x.prefix_k_stride_p = pk.stride(0);
      x.prefix_v_stride_p = pv.stride(0);
      x.prefix_num_pages = (int)pk.size(0);
      x.prefix_page_size = (int)pk.size(1);
      x.prefix_max_pages = (int)ptable.numel();
    } else {
      x.prefix_seqlen = (int)pk.size(0);
    }
    x.dtype = dtype_code(type);
    x.softmax_scale = (float)scale;
    FsaSharedPrefixWorkspace w;
    int rc = g_prefix_bytes(&x, &w);
    Tensor room;
    if (rc == FSA_OK) {
      room = at::empty({(int64_t)((w.out_partial + w.sum_partial + w.plan_ws) / 4)}, q.options().dtype(at::kFloat));
      x.out_partial = ptr<float>(room);
      x.sum_partial = x.out_partial + w.out_partial / 4;
      x.plan_ws = reinterpret_cast<int32_t*>(x.sum_partial + w.sum_partial / 4);
      rc = g_prefix(&x, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
    }
    no_gil.reset();
    if (rc != FSA_OK) return PyLong_FromLong(rc);
    if (a[10] == Py_None && a[11] == Py_None) return pair(std::move(out), std::move(lse));
    PyObject* o = a[10] != Py_None ? (Py_INCREF(a[10]), a[10]) : THPVariable_Wrap(std::move(out));
    PyObject* l = a[11] != Py_None ? (Py_INCREF(a[11]), a[11]) : THPVariable_Wrap(std::move(lse));
    PyObject* both = o && l ? PyTuple_Pack(2, o, l) : nullptr;
    Py_XDECREF(o);
    Py_XDECREF(l);
    return both;
  END_HANDLE_TH_ERRORS
}

// ---- rotary positions with several axes, caches with scales of their rows -----------------------------------------------

bool here(const at::Device& dev) {
  return dev.is_cuda() && dev.index() >= 0 && dev.index() < MAX_DEVICES && g_status[dev.index()] && c10::cuda::current_device() == dev.index();
}
bool is16(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }
// Rows on top of one another, backwards or without a stride.
bool expanded(const Tensor& t) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) <= 0) return true;
  return false;
}
// The axes of the pairs, as rotary_axes.py::axis_bits lays them out.
bool get_bits(PyObject* o, uint32_t* bits) {
  if (!PyBytes_CheckExact(o) || PyBytes_GET_SIZE(o) != 32) return false;
  std::memcpy(bits, PyBytes_AS_STRING(o), 32);
  return true;
}
// (axis, batch, token) strides of positions for rows of these leading sizes; false where they do not fit.
bool positions_ok(const Tensor& ids, int64_t axes, int64_t dims, at::IntArrayRef lead, const at::Device& dev, int64_t* sa, int64_t* sb, int64_t* ss) {
  if ((ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong) || ids.device() != dev || ids.dim() != dims + 1 || ids.size(0) != axes) return false;
  if (dims == 1) {
    if (ids.size(1) != lead[0]) return false;
    *sb = 0;
    *ss = ids.stride(1);
  } else {
    if ((ids.size(1) != 1 && ids.size(1) != lead[0]) || ids.size(2) != lead[1]) return false;
    *sb = ids.size(1) > 1 ? ids.stride(1) : 0;
    *ss = ids.stride(2);
  }
  *sa = ids.stride(0);
  return true;
}

struct AxesCall {
  Tensor cos, sin, ids;
  uint32_t bits[8];
  int64_t axes = 0;
  bool interleaved = false, transposed = false;
};

// One launch for the tensors that are defined (one of them is).
void axes_launch(const AxesCall& c, const Tensor& q_in, const Tensor& k_in, Tensor* q_out, Tensor* k_out) {
  const Tensor& any = q_in.defined() ? q_in : k_in;
  const int dev = any.device().index();
  const Tensor q = q_in.defined() ? rows_of(q_in) : q_in, k = k_in.defined() ? rows_of(k_in) : k_in;
  FsaRotaryAxesArgs x = {};
  auto put = [](const Tensor& t, int64_t* sb, int64_t* ss, int64_t* sh) {
    *sb = t.dim() == 3 ? 0 : t.stride(0);
    *ss = t.stride(-3);
    *sh = t.stride(-2);
  };
  if (q.defined()) {
    *q_out = at::empty(q.sizes(), q.options());
    x.q = q.data_ptr();
    x.q_out = q_out->data_ptr();
    x.heads_q = (int)q.size(-2);
    put(q, &x.q_stride_b, &x.q_stride_s, &x.q_stride_h);
    put(*q_out, &x.q_out_stride_b, &x.q_out_stride_s, &x.q_out_stride_h);
  }
  if (k.defined()) {
    *k_out = at::empty(k.sizes(), k.options());
    x.k = k.data_ptr();
    x.k_out = k_out->data_ptr();
    x.heads_k = (int)k.size(-2);
    put(k, &x.k_stride_b, &x.k_stride_s, &x.k_stride_h);
    put(*k_out, &x.k_out_stride_b, &x.k_out_stride_s, &x.k_out_stride_h);
  }
  if ((q.defined() ? q.numel() : 0) + (k.defined() ? k.numel() : 0) == 0) return;
  x.cos = c.cos.data_ptr();
  x.sin = c.sin.data_ptr();
  x.position_ids = c.ids.data_ptr();
  x.position_ids_int64 = c.ids.scalar_type() == at::kLong;
  TORCH_CHECK(positions_ok(c.ids, c.axes, any.dim() - 2, any.sizes(), any.device(), &x.position_stride_a, &x.position_stride_b, &x.position_stride_s),
              "position_ids must have one entry per axis and token");
  x.status = ptr<int32_t>(*g_status[dev]);
  x.table_stride = c.cos.stride(0);
  x.table_rows = (int)c.cos.size(0);
  x.rotary_dim = (int)(2 * c.cos.size(1));
  x.table_dtype = table_code(c.cos.scalar_type());
  std::memcpy(x.axis_bits, c.bits, 32);
  x.axes = (int)c.axes;
  x.batch = any.dim() == 4 ? (int)any.size(0) : 1;
  x.seqlen = (int)any.size(-3);
  x.head_dim = (int)any.size(-1);
  x.dtype = dtype_code(any.scalar_type());
  x.interleaved = c.interleaved;
  x.transposed = c.transposed;
  const int rc = g_axes(&x, c10::cuda::getCurrentCUDAStream(dev).stream());
  TORCH_CHECK(rc == FSA_OK, "fsa_rotary_axes failed (code ", rc, ")");
}

// As RotaryFn: the gradient is the transposed rotation, which is a rotation again.
struct AxesFn : torch::autograd::Function<AxesFn> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const std::optional<Tensor>& q_in,
                                                const std::optional<Tensor>& k_in, const AxesCall& c) {
    const Tensor q = q_in.value_or(Tensor()), k = k_in.value_or(Tensor());
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({c.cos, c.sin, c.ids});
    ctx->saved_data["form"] =
        int64_t(c.interleaved) | int64_t(c.transposed) << 1 | int64_t(q.defined()) << 2 | int64_t(k.defined()) << 3 | c.axes << 4;
    std::vector<int64_t> bits(c.bits, c.bits + 8);
    ctx->saved_data["bits"] = bits;
    return launch(q, k, c);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const int64_t form = ctx->saved_data["form"].toInt();
    const auto bits = ctx->saved_data["bits"].toIntVector();
    AxesCall c;
    c.cos = saved[0];
    c.sin = saved[1];
    c.ids = saved[2];
    for (int i = 0; i < 8; ++i) c.bits[i] = (uint32_t)bits[i];
    c.axes = form >> 4;
    c.interleaved = (form & 1) != 0;
    c.transposed = (form & 2) == 0;
    Tensor in[2];
    size_t n = 0;
    for (int i = 0; i < 2; ++i)
      if (form & (4 << i)) {
        if (ctx->needs_input_grad(n)) in[i] = grads[n];  // (tensors that are left out have no edge)
        ++n;
      }
    torch::autograd::variable_list out(3);  // one entry for every argument of forward
    if (!in[0].defined() && !in[1].defined()) return out;
    const auto turned = turn(in[0], in[1], c);
    n = 0;
    for (int i = 0; i < 2; ++i)
      if (in[i].defined()) out[i] = turned[n++];
    return out;
  }
  static torch::autograd::variable_list launch(const Tensor& q, const Tensor& k, const AxesCall& c) {
    Tensor q_out, k_out;
    axes_launch(c, q, k, &q_out, &k_out);
    if (!k.defined()) return {q_out};
    if (!q.defined()) return {k_out};
    return {q_out, k_out};
  }
  static torch::autograd::variable_list turn(const Tensor& q, const Tensor& k, const AxesCall& c) {
    auto seen = [](const Tensor& t) { return t.defined() && ((at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined()); };
    auto maybe = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
    return seen(q) || seen(k) ? apply(maybe(q), maybe(k), c) : launch(q, k, c);
  }
};

// rotary_axes(q, k, cos, sin, position_ids, axes of the pairs, number of axes, interleaved) -> q or (q, k), or None. k may be None.
PyObject* rotary_axes(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8 || !g_axes) return none();
  HANDLE_TH_ERRORS
    Tensor q, k;
    AxesCall c;
    if (a[0] == Py_None || a[2] == Py_None || a[3] == Py_None || a[4] == Py_None || !opt_tensor(a[0], &q) || !opt_tensor(a[1], &k) ||
        !opt_tensor(a[2], &c.cos) || !opt_tensor(a[3], &c.sin) || !opt_tensor(a[4], &c.ids) || !get_bits(a[5], c.bits) || !get_int(a[6], &c.axes) ||
        !PyBool_Check(a[7]))
      return none();
    c.interleaved = a[7] == Py_True;
    const at::Device dev = q.device();
    if ((q.dim() != 3 && q.dim() != 4) || !here(dev) || !is16(q.scalar_type())) return none();
    const int64_t d = q.size(-1);
    if (q.numel() == 0 || d > 256 || q.numel() / (q.size(-2) * d) > INT32_MAX || !tables_ok(c.cos, c.sin, d, dev)) return none();
    if (k.defined()) {
      if (k.dim() != q.dim() || k.scalar_type() != q.scalar_type() || k.device() != dev || k.size(-1) != d || k.numel() == 0) return none();
      for (int64_t i = 0; i < q.dim() - 2; ++i)
        if (k.size(i) != q.size(i)) return none();
    }
    int64_t sa, sb, ss;
    if (c.axes < 2 || !positions_ok(c.ids, c.axes, q.dim() - 2, q.sizes(), dev, &sa, &sb, &ss)) return none();
    std::optional<NoGil> no_gil(std::in_place);
    auto out = AxesFn::turn(q, k, c);
    no_gil.reset();
    return k.defined() ? pair(std::move(out[0]), std::move(out[1])) : THPVariable_Wrap(std::move(out[0]));
  END_HANDLE_TH_ERRORS
}

// The library's view of a cache (quantized_kvcache.py::check_quantized_cache, fill_quantized_cache); false where it is not an ordinary one.
bool quant_cache(const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs, const Tensor& table, int64_t batch, const at::Device& dev,
                 FsaQuantCache* c) {
  for (const Tensor* t : {&kc, &vc, &ks, &vs})
    if (!t->defined() || t->device() != dev || expanded(*t)) return false;
  if (kc.dim() != 4 || kc.sizes() != vc.sizes() || kc.scalar_type() != vc.scalar_type() || kc.numel() == 0) return false;
  const bool int4 = kc.scalar_type() == at::kByte;
  if (int4) c->format = FSA_QC_INT4;
  else if (kc.scalar_type() == at::kChar) c->format = FSA_QC_INT8;
  else if (kc.scalar_type() == at::kFloat8_e4m3fn) c->format = FSA_QC_E4M3;
  else return false;
  const int64_t d = kc.size(3) * (int4 ? 2 : 1);
  if (d > 128 || d % 16 || kc.size(0) > INT32_MAX || kc.size(1) > INT32_MAX || kc.size(2) > INT32_MAX) return false;
  if (ks.sizes() != vs.sizes() || ks.scalar_type() != vs.scalar_type() || ks.dim() != (int4 ? 5 : 4)) return false;
  for (int i = 0; i < 3; ++i)
    if (ks.size(i) != kc.size(i)) return false;
  const int64_t per = int4 ? 2 : 1;
  if (int4) {
    const int64_t groups = ks.size(3);
    if (ks.scalar_type() != at::kBFloat16 || ks.size(4) != 2 || groups <= 0 || d % groups || (d / groups != 32 && d / groups != 64)) return false;
    c->group = (int)(d / groups);
  } else if (ks.scalar_type() != at::kFloat || ks.size(3) != 1) {
    return false;
  }
  auto strides = [&](const Tensor& t, int64_t unit, int64_t divide, int64_t* sb, int64_t* ss, int64_t* sh) {
    int64_t* const to[3] = {sb, ss, sh};
    for (int i = 0; i < 3; ++i) {
      const int64_t s = t.size(i) == 1 ? 0 : t.stride(i);
      if (s % unit) return false;
      *to[i] = s / divide;
    }
    return true;
  };
  for (const Tensor* t : {&kc, &vc})
    if (t->stride(3) != 1 || (reinterpret_cast<uintptr_t>(t->data_ptr()) & 15)) return false;
  for (const Tensor* t : {&ks, &vs})
    if (int4 && (t->stride(4) != 1 || (t->size(3) > 1 && t->stride(3) != 2) || (reinterpret_cast<uintptr_t>(t->data_ptr()) & 3))) return false;
  if (!strides(kc, 16, 1, &c->k_stride_b, &c->k_stride_s, &c->k_stride_h) || !strides(vc, 16, 1, &c->v_stride_b, &c->v_stride_s, &c->v_stride_h) ||
      !strides(ks, per, per, &c->ks_stride_b, &c->ks_stride_s, &c->ks_stride_h) || !strides(vs, per, per, &c->vs_stride_b, &c->vs_stride_s, &c->vs_stride_h))
    return false;
  c->k = kc.data_ptr();
  c->v = vc.data_ptr();
  c->k_scales = ks.data_ptr();
  c->v_scales = vs.data_ptr();
  c->heads_kv = (int)kc.size(2);
  c->head_dim = (int)d;
  if (table.defined()) {
    if (!int_ok(table, dev, 2) || expanded(table) || table.size(0) != batch || table.size(1) <= 0 || (table.size(1) > 1 && table.stride(1) != 1)) return false;
    c->page_table = ptr<int32_t>(table);
    c->page_table_stride = table.stride(0);
    c->num_pages = (int)kc.size(0);
    c->page_size = (int)kc.size(1);
    c->max_pages = (int)table.size(1);
  } else {
    if (kc.size(0) != batch) return false;
    c->capacity = (int)kc.size(1);
  }
  return true;
}
// Rows of 16 bits on 16-byte boundaries (quantized_kvcache.py::rows_ok), and their strides, of dimensions of one none.
bool rows16(const Tensor& t, int64_t* sb, int64_t* ss, int64_t* sh) {
  if (t.stride(-1) != 1 || (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15)) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) % 8) return false;
  auto at = [&](int64_t i) { return t.size(i) == 1 ? 0 : t.stride(i); };
  *sb = t.dim() == 3 ? 0 : at(0);
  *ss = at(-3);
  *sh = at(-2);
  return true;
}

// append_quantized(q, k_new, v_new, k_cache, v_cache, k_scales, v_scales, seqused_k, cos, sin, page_table, free_pages, free_count, cu_seqlens_new,
//                  seqlen_offsets, position_ids, axes of the pairs, number of axes, interleaved, advance, out)
//   -> the turned queries (True without queries), an error code, or None
PyObject* append_quantized(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 21 || !g_qappend || !g_qappend_ints) return none();
  HANDLE_TH_ERRORS
    Tensor q, k, v, kc, vc, ks, vs, used, cos, sin, table, free, count, cu, offsets, ids, out;
    Tensor* const into[21] = {&q,     &k,    &v,     &kc, &vc,     &ks,  &vs,     &used,   &cos,    &sin, &table,
                              &free, &count, &cu, nullptr, &ids, nullptr, nullptr, nullptr, nullptr, &out};
    for (int i = 0; i < 21; ++i)
      if (into[i] && !opt_tensor(a[i], into[i])) return none();
    int64_t offset, axes = 0;
    if (!k.defined() || !v.defined() || !kc.defined() || !used.defined() || !get_offsets(a[14], &offset, &offsets) || !PyBool_Check(a[18]) ||
        !PyBool_Check(a[19]))
      return none();
    const int64_t dims = cu.defined() ? 3 : 4;
    if (k.dim() != dims || k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type() || !is16(k.scalar_type())) return none();
    const at::Device dev = k.device();
    if (!here(dev)) return none();
    for (int i = 0; i < 21; ++i)
      if (into[i] && into[i]->defined() && into[i]->device() != dev) return none();
    if (used.scalar_type() != at::kInt || used.dim() != 1 || !used.is_contiguous() || used.numel() == 0 || k.numel() == 0) return none();
    const int64_t batch = used.numel(), d = k.size(-1);
    FsaKvAppendQuantArgs x = {};
    if (!quant_cache(kc, vc, ks, vs, table, batch, dev, &x.cache) || x.cache.heads_kv != k.size(-2) || x.cache.head_dim != d) return none();
    if (cu.defined() ? (cu.scalar_type() != at::kInt || cu.dim() != 1 || !cu.is_contiguous() || cu.size(0) != batch + 1) : k.size(0) != batch) return none();
    if (cos.defined() != sin.defined()) return none();
    if (!cos.defined()) {
      if (q.defined() || a[14] != Py_None || ids.defined() || a[16] != Py_None) return none();
    } else {
      if (!tables_ok(cos, sin, d, dev) || cos.size(1) % 8) return none();
      const int64_t stride = cos.size(0) == 1 ? 0 : cos.stride(0);
      if (cos.scalar_type() == at::kFloat &&
          (((reinterpret_cast<uintptr_t>(cos.data_ptr()) | reinterpret_cast<uintptr_t>(sin.data_ptr())) & 15) || stride % 4))
        return none();
      x.cos = cos.data_ptr();
      x.sin = sin.data_ptr();
      x.table_rows = (int)cos.size(0);
      x.rotary_dim = (int)(2 * cos.size(1));
      x.table_stride = stride;
      x.table_dtype = table_code(cos.scalar_type());
    }
    if (ids.defined() != (a[16] != Py_None)) return none();
    if (ids.defined()) {
      if (a[14] != Py_None || !get_bits(a[16], x.axis_bits) || !get_int(a[17], &axes) ||
          !positions_ok(ids, axes, dims - 2, k.sizes(), dev, &x.position_stride_a, &x.position_stride_b, &x.position_stride_s))
        return none();
      x.position_ids = ids.data_ptr();
      x.position_ids_int64 = ids.scalar_type() == at::kLong;
      x.axes = (int)axes;
    }
    if (!offsets_ok(offsets, batch, dev)) return none();
    if (free.defined() != count.defined() || (free.defined() && (!table.defined() || free.scalar_type() != at::kInt || !free.is_contiguous() ||
                                                                   count.scalar_type() != at::kInt || count.numel() != 1)))
      return none();
    if (free.defined() && expanded(free)) return none();
    if (!rows16(k, &x.k_stride_b, &x.k_stride_s, &x.k_stride_h) || !rows16(v, &x.v_stride_b, &x.v_stride_s, &x.v_stride_h)) return none();
    if (q.defined()) {
      if (q.dim() != dims || q.scalar_type() != k.scalar_type() || q.size(-1) != d || q.size(-2) <= 0 || q.size(-2) % k.size(-2)) return none();
      for (int64_t i = 0; i < dims - 2; ++i)
        if (q.size(i) != k.size(i)) return none();
      if (!rows16(q, &x.q_stride_b, &x.q_stride_s, &x.q_stride_h)) return none();
    }
    if (out.defined() && (!q.defined() || out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type() || expanded(out))) return none();
    std::optional<NoGil> no_gil(std::in_place);
    if (q.defined()) {
      if (!out.defined()) out = at::empty(q.sizes(), q.options());
      if (!rows16(out, &x.q_out_stride_b, &x.q_out_stride_s, &x.q_out_stride_h)) {
        no_gil.reset();
        return none();
      }
      x.q = q.data_ptr();
      x.q_out = out.data_ptr();
      x.heads_q = (int)q.size(-2);
    }
    x.k_new = k.data_ptr();
    x.v_new = v.data_ptr();
    x.seqused_k = ptr<int32_t>(used);
    x.free_pages = ptr<int32_t>(free);
    x.free_count = ptr<int32_t>(count);
    x.cu_seqlens_new = ptr<int32_t>(cu);
    x.seqlen_offsets = ptr<int32_t>(offsets);
    x.status = ptr<int32_t>(*g_status[dev.index()]);
    x.batch = (int)batch;
    if (cu.defined())
      x.total = (int)k.size(0);
    else
      x.new_tokens = (int)k.size(1);
    x.offset = (int)offset;
    x.dtype = dtype_code(k.scalar_type());
    x.interleaved = a[18] == Py_True;
    x.advance = a[19] == Py_True;
    const int64_t ints = g_qappend_ints(&x);
    Tensor place;
    if (ints > 0) place = at::empty({ints}, used.options());
    x.place_ws = ptr<int32_t>(place);
    const int rc = g_qappend(&x, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
    if (rc == FSA_OK) {
      for (const Tensor* t : {&kc, &vc, &ks, &vs}) written(*t);
      if (x.advance) written(used);
      if (free.defined()) {
        written(table);
        written(count);
      }
      if (a[20] != Py_None) written(out);
    }
    no_gil.reset();
    if (rc != FSA_OK) return PyLong_FromLong(rc);
    if (!q.defined()) Py_RETURN_TRUE;
    if (a[20] != Py_None) {
      Py_INCREF(a[20]);
      return a[20];
    }
    return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// read_quantized(k_cache, v_cache, k_scales, v_scales, seqused_k, page_table, cu_seqlens, max_seqlen, total, bf16) -> (k, v), an error code, or None
PyObject* read_quantized(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 10 || !g_qread) return none();
  HANDLE_TH_ERRORS
    Tensor kc, vc, ks, vs, used, table, cu;
    Tensor* const into[7] = {&kc, &vc, &ks, &vs, &used, &table, &cu};
    for (int i = 0; i < 7; ++i)
      if (!opt_tensor(a[i], into[i])) return none();
    int64_t rows = 0;
    if (!kc.defined() || !PyBool_Check(a[9]) || cu.defined() != (a[7] == Py_None) || cu.defined() != (a[8] != Py_None) ||
        !get_int(cu.defined() ? a[8] : a[7], &rows) || rows <= 0)
      return none();
    const at::Device dev = kc.device();
    if (!here(dev)) return none();
    if (cu.defined() && (cu.scalar_type() != at::kInt || cu.dim() != 1 || cu.numel() < 2 || !cu.is_contiguous() || cu.device() != dev)) return none();
    if (kc.dim() != 4) return none();
    const int64_t batch = cu.defined() ? cu.numel() - 1 : (table.defined() && table.dim() > 0 ? table.size(0) : kc.size(0));
    FsaKvReadQuantArgs x = {};
    if (!quant_cache(kc, vc, ks, vs, table, batch, dev, &x.cache)) return none();
    if (used.defined() && (used.scalar_type() != at::kInt || used.dim() != 1 || used.size(0) != batch || !used.is_contiguous() || used.device() != dev)) return none();
    std::optional<NoGil> no_gil(std::in_place);
    const auto options = kc.options().dtype(a[9] == Py_True ? at::kBFloat16 : at::kHalf);
    const int64_t h = x.cache.heads_kv, d = x.cache.head_dim;
    const auto shape = cu.defined() ? std::vector<int64_t>{rows, h, d} : std::vector<int64_t>{batch, rows, h, d};
    Tensor k = at::empty(shape, options), v = at::empty(shape, options);
    x.k_out = k.data_ptr();
    x.v_out = v.data_ptr();
    if (!cu.defined()) x.k_out_stride_b = x.v_out_stride_b = rows * h * d;
    x.k_out_stride_s = x.v_out_stride_s = h * d;
    x.k_out_stride_h = x.v_out_stride_h = d;
    x.seqused_k = ptr<int32_t>(used);
    x.cu_seqlens = ptr<int32_t>(cu);
    x.status = ptr<int32_t>(*g_status[dev.index()]);
    x.batch = (int)batch;
    (cu.defined() ? x.total : x.seqlen) = (int)rows;
    x.dtype = a[9] == Py_True ? FSA_DT_BF16 : FSA_DT_FP16;
    const int rc = g_qread(&x, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
    no_gil.reset();
    if (rc != FSA_OK) return PyLong_FromLong(rc);
    return pair(std::move(k), std::move(v));
  END_HANDLE_TH_ERRORS
}

// decode_quantized(q, k, v, k_scales, v_scales, softmax_scale, page_table, gather_kv_indices, seqused_k, out, lse) -> (out, lse), an error code, or None
PyObject* decode_quantized(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 11 || !g_qdecode || !g_qdecode_bytes) return none();
  HANDLE_TH_ERRORS
    Tensor q, k, v, ks, vs, table, gather, used, out, lse;
    Tensor* const into[11] = {&q, &k, &v, &ks, &vs, nullptr, &table, &gather, &used, &out, &lse};
    for (int i = 0; i < 11; ++i)
      if (into[i] && !opt_tensor(a[i], into[i])) return none();
    if (!q.defined() || q.dim() != 3 || !is16(q.scalar_type())) return none();
    const at::Device dev = q.device();
    if (!here(dev)) return none();
    const int64_t batch = q.size(0), hq = q.size(1), d = q.size(2);
    FsaQuantDecodeArgs x = {};
    if (batch <= 0 || hq <= 0 || !quant_cache(k, v, ks, vs, table, batch, dev, &x.cache) || hq % x.cache.heads_kv || x.cache.head_dim != d) return none();
    const int page = x.cache.page_size;
    if (table.defined() && page != 32 && page != 64 && page != 128 && page != 256) return none();
    int64_t none_b;
    if (!rows16(q, &none_b, &x.q_stride_b, &x.q_stride_h)) return none();
    if (used.defined() && (used.scalar_type() != at::kInt || used.dim() != 1 || used.size(0) != batch || !used.is_contiguous() || used.device() != dev)) return none();
    if (gather.defined()) {
      if (gather.scalar_type() != at::kInt || gather.dim() != 2 || gather.size(0) != batch || gather.device() != dev || gather.size(1) <= 0 ||
          gather.size(1) > INT32_MAX || (gather.size(1) > 1 && gather.stride(1) != 1))
        return none();
      x.gather_kv_indices = ptr<int32_t>(gather);
      x.topk = (int)gather.size(1);
      x.gather_stride = gather.stride(0);
    }
    if (out.defined() && (out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type() || out.device() != dev || out.stride(2) != 1 || expanded(out) ||
                          (reinterpret_cast<uintptr_t>(out.data_ptr()) & 3) || (batch > 1 && out.stride(0) % 2) || (hq > 1 && out.stride(1) % 2)))
      return none();
    if (lse.defined() && (lse.dim() != 2 || lse.size(0) != batch || lse.size(1) != hq || lse.scalar_type() != at::kFloat || lse.device() != dev ||
                          (hq > 1 && lse.stride(1) != 1) || expanded(lse)))
      return none();
    double scale;
    if (!opt_double(a[5], 1.0 / std::sqrt((double)d), &scale) || !(scale > 0.0) || std::isinf(scale)) return none();
    std::optional<NoGil> no_gil(std::in_place);
    if (!out.defined()) out = at::empty({batch, hq, d}, q.options());
    if (!lse.defined()) lse = at::empty({batch, hq}, q.options().dtype(at::kFloat));
    x.q = q.data_ptr();
    x.out = out.data_ptr();
    x.lse = ptr<float>(lse);
    x.o_stride_b = batch > 1 ? out.stride(0) : 0;
    x.o_stride_h = hq > 1 ? out.stride(1) : 0;
    x.lse_stride_b = batch > 1 ? lse.stride(0) : 0;
    x.lse_stride_h = hq > 1 ? lse.stride(1) : 0;
    x.seqused_k = ptr<int32_t>(used);
    x.status = ptr<int32_t>(*g_status[dev.index()]);
    x.batch = (int)batch;
    x.heads_q = (int)hq;
    x.dtype = dtype_code(q.scalar_type());
    x.softmax_scale = (float)scale;
    int64_t bytes = g_qdecode_bytes(&x);
    int rc = bytes < 0 ? (int)bytes : FSA_OK;
    Tensor room;
    if (rc == FSA_OK) {
      room = at::empty({bytes / 4}, q.options().dtype(at::kFloat));
      x.ws = room.data_ptr();
      rc = g_qdecode(&x, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
    }
    if (rc == FSA_OK) {
      if (a[9] != Py_None) written(out);
      if (a[10] != Py_None) written(lse);
    }
    no_gil.reset();
    if (rc != FSA_OK) return PyLong_FromLong(rc);
    if (a[9] == Py_None && a[10] == Py_None) return pair(std::move(out), std::move(lse));
    PyObject* o = a[9] != Py_None ? (Py_INCREF(a[9]), a[9]) : THPVariable_Wrap(std::move(out));
    PyObject* l = a[10] != Py_None ? (Py_INCREF(a[10]), a[10]) : THPVariable_Wrap(std::move(lse));
    PyObject* both = o && l ? PyTuple_Pack(2, o, l) : nullptr;
    Py_XDECREF(o);
    Py_XDECREF(l);
    return both;
  END_HANDLE_TH_ERRORS
}

// init_quantized(addresses of fsa_rotary_axes, fsa_kv_append_quantized_workspace_ints, fsa_kv_append_quantized, fsa_kv_read_quantized,
//                fsa_decode_quantized_workspace_bytes, fsa_decode_quantized)
PyObject* init_quantized(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "init_quantized takes six addresses");
    return nullptr;
  }
  void* at[6] = {};
  for (Py_ssize_t i = 0; i < n && !PyErr_Occurred(); ++i) at[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) return nullptr;
  g_axes = reinterpret_cast<decltype(g_axes)>(at[0]);
  g_qappend_ints = reinterpret_cast<decltype(g_qappend_ints)>(at[1]);
  g_qappend = reinterpret_cast<decltype(g_qappend)>(at[2]);
  g_qread = reinterpret_cast<decltype(g_qread)>(at[3]);
  g_qdecode_bytes = reinterpret_cast<decltype(g_qdecode_bytes)>(at[4]);
  g_qdecode = reinterpret_cast<decltype(g_qdecode)>(at[5]);
  return none();
}

// init_cache(addresses of fsa_rotary, fsa_kv_append_rotary_workspace_ints, fsa_kv_append_rotary, fsa_shared_prefix_workspace_bytes,
//            fsa_decode_shared_prefix)
PyObject* init_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "init_cache takes five addresses");
    return nullptr;
  }
  void* at[5] = {};
  for (Py_ssize_t i = 0; i < n && !PyErr_Occurred(); ++i) at[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) return nullptr;
  g_rotary = reinterpret_cast<decltype(g_rotary)>(at[0]);
  g_append_ints = reinterpret_cast<decltype(g_append_ints)>(at[1]);
  g_append = reinterpret_cast<decltype(g_append)>(at[2]);
  g_prefix_bytes = reinterpret_cast<decltype(g_prefix_bytes)>(at[3]);
  g_prefix = reinterpret_cast<decltype(g_prefix)>(at[4]);
  return none();
}

// init(addresses of fsa_decode, fsa_fwd[, fsa_topk_indices, fsa_pack_scales])
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 2 && n != 4) {
    PyErr_SetString(PyExc_TypeError, "init takes two or four addresses");
    return nullptr;
  }
  void* at[4] = {};
  for (Py_ssize_t i = 0; i < n && !PyErr_Occurred(); ++i) at[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) return nullptr;
  if (n == 4) {
    g_topk = reinterpret_cast<decltype(g_topk)>(at[2]);
    g_pack = reinterpret_cast<decltype(g_pack)>(at[3]);
  }
  g_decode = reinterpret_cast<decltype(g_decode)>(at[0]);
  g_fwd = reinterpret_cast<decltype(g_fwd)>(at[1]);
  return none();
}

// set_status(device index, int32 status tensor, number of SMs)
PyObject* set_status(PyObject*, PyObject* const* a, Py_ssize_t n) {
  int64_t dev, sms;
  if (n != 3 || !get_int(a[0], &dev) || dev >= MAX_DEVICES || !THPVariable_CheckExact(a[1]) || !get_int(a[2], &sms)) {
    PyErr_SetString(PyExc_TypeError, "set_status takes a device index, a tensor and a number of SMs");
    return nullptr;
  }
  g_sms[dev] = (int)sms;
  if (!g_status[dev]) g_status[dev] = new Tensor(THPVariable_Unpack(a[1]));
  return none();
}

PyObject* decode_num_splits(PyObject*, PyObject* const* a, Py_ssize_t n) {
  int64_t v[4];
  for (int i = 0; i < 4; ++i)
    if (n != 4 || !get_int(a[i], &v[i])) {
      PyErr_SetString(PyExc_TypeError, "decode_num_splits takes four non-negative integers");
      return nullptr;
    }
  return PyLong_FromLongLong(decode_splits(v[0], v[1], v[2], v[3]));
}

PyMethodDef methods[] = {
    {"init", reinterpret_cast<PyCFunction>(init), METH_FASTCALL, nullptr},
    {"set_status", reinterpret_cast<PyCFunction>(set_status), METH_FASTCALL, nullptr},
    {"decode", reinterpret_cast<PyCFunction>(decode), METH_FASTCALL, nullptr},
    {"forward", reinterpret_cast<PyCFunction>(forward), METH_FASTCALL, nullptr},
    {"topk", reinterpret_cast<PyCFunction>(topk), METH_FASTCALL, nullptr},
    {"init_cache", reinterpret_cast<PyCFunction>(init_cache), METH_FASTCALL, nullptr},
    {"rotary", reinterpret_cast<PyCFunction>(rotary), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(append), METH_FASTCALL, nullptr},
    {"init_quantized", reinterpret_cast<PyCFunction>(init_quantized), METH_FASTCALL, nullptr},
    {"rotary_axes", reinterpret_cast<PyCFunction>(rotary_axes), METH_FASTCALL, nullptr},
    {"append_quantized", reinterpret_cast<PyCFunction>(append_quantized), METH_FASTCALL, nullptr},
    {"read_quantized", reinterpret_cast<PyCFunction>(read_quantized), METH_FASTCALL, nullptr},
    {"decode_quantized", reinterpret_cast<PyCFunction>(decode_quantized), METH_FASTCALL, nullptr},
    {"shared_prefix", reinterpret_cast<PyCFunction>(shared_prefix), METH_FASTCALL, nullptr},
    {"decode_num_splits", reinterpret_cast<PyCFunction>(decode_num_splits), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// ABI_VERSION and TORCH_VERSION: what this was compiled against (the argument blocks of the header, ATen's classes).
PyMODINIT_FUNC PyInit__host(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && (PyModule_AddIntConstant(m, "ABI_VERSION", FSA_ABI_VERSION) < 0 ||
            PyModule_AddStringConstant(m, "TORCH_VERSION", TORCH_VERSION) < 0)) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
