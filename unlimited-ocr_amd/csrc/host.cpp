// The host side of the 8-bit cache and page pool calls, without the interpreter's
// share: srswa/cache8.py and srswa/cache_pages.py hand a call here first.
//
// Reading a dozen tensors' pointers, strides and types from Python and packing
// them through ctypes takes 17 to 30 us, more than most serving steps' kernels
// (a reorder of 12 layers' caches: 185 us); here it takes 3 to 5.  A function
// checks that its call is an ordinary one -- plain tensors on the current GPU, the
// expected types, int32 tables with contiguous rows -- and answers NotImplemented
// to any other and to whatever the library refuses, with nothing launched: the
// Python path then converts what can be converted and raises what cannot be taken.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

#include "srswa.h"

namespace {

using at::Tensor;

PyObject* not_this() { Py_RETURN_NOTIMPLEMENTED; }

// The plain tensor behind an argument on GPU `dev` (-1: takes the first one's).
const Tensor* tensor(PyObject* o, int* dev) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.layout() != at::kStrided) return nullptr;
  const int d = t.get_device();
  if (*dev < 0) *dev = d;
  return d == *dev ? &t : nullptr;
}

bool as_long(PyObject* o, int64_t lo, int64_t hi, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &over);
  return !over && *v >= lo && *v <= hi;
}

bool i32_rows(const Tensor& t) {
  return t.scalar_type() == at::kInt && t.dim() == 2 && (t.stride(1) == 1 || t.size(1) <= 1);
}
bool i32_list(const Tensor& t) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && (t.stride(0) == 1 || t.size(0) <= 1);
}

int float_code(const Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? SRSWA_BF16 : t.scalar_type() == at::kHalf ? SRSWA_F16 : -1;
}

struct Cache {
  int64_t npages, page, heads, D;
  int code;
};

// The four tensors of a scaled cache; false where the Python path has to look.
bool cache(const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs, Cache* c) {
  if (kc.dim() != 4 || vc.sizes() != kc.sizes() || vc.scalar_type() != kc.scalar_type()) return false;
  if (kc.scalar_type() == at::kChar) c->code = SRSWA_I8;
  else if (kc.scalar_type() == at::kFloat8_e4m3fn) c->code = SRSWA_FP8_E4M3FN;
  else return false;
  c->npages = kc.size(0); c->page = kc.size(1); c->heads = kc.size(2); c->D = kc.size(3);
  if (c->npages < 1 || c->npages > INT32_MAX || c->page > 1024 || c->heads < 1 || kc.stride(3) != 1 || vc.stride(3) != 1)
    return false;
  for (const Tensor* s : {&ks, &vs})
    if (s->scalar_type() != at::kFloat || s->dim() != 2 || s->size(0) != c->npages || s->size(1) != c->heads) return false;
  return true;
}

void* stream_of(int dev) { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)dev).stream(); }

// attend(form, q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu | None, rows, scale, window, sinks,
//        out | None, return_lse, topk | None, bias | None): form 0 decode, 1 prefill; window 0 none
PyObject* attend(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 17) return not_this();
  int64_t form, rows, window, sinks;
  if (!as_long(args[0], 0, 1, &form) || !as_long(args[9], 1, INT32_MAX, &rows) || !as_long(args[11], 0, 1 << 30, &window) ||
      !as_long(args[12], 0, 1 << 30, &sinks) || !PyFloat_CheckExact(args[10]))
    return not_this();
  int dev = -1;
  const Tensor* t[7];
  for (int i = 0; i < 7; ++i)
    if (!(t[i] = tensor(args[1 + i], &dev))) return not_this();
  if (dev != c10::hip::current_device()) return not_this();
  const Tensor &q = *t[0], &kc = *t[1], &vc = *t[2], &ks = *t[3], &vs = *t[4], &bt = *t[5], &sl = *t[6];
  Cache c;
  if (!cache(kc, vc, ks, vs, &c) || !i32_rows(bt) || !i32_list(sl)) return not_this();
  const int code = float_code(q);
  if (code < 0 || q.dim() != 3 || q.size(2) != c.D || q.stride(2) != 1 || q.size(0) < 1 || q.size(0) > INT32_MAX)
    return not_this();
  const int64_t total = q.size(0), R = sl.size(0);
  if (R < 1 || bt.size(0) < R || bt.size(1) < 1 || bt.size(1) > INT32_MAX) return not_this();
  srswa_cache8_attend_args a{};
  const Tensor* cu = nullptr;
  if (args[8] != Py_None) {
    cu = tensor(args[8], &dev);
    if (!cu || !i32_list(*cu) || cu->size(0) != R + 1) return not_this();
    a.cu_seqlens_q = (const int32_t*)cu->const_data_ptr();
    rows = std::min(rows, total);
  } else if (total != R * rows) {
    return not_this();
  }
  if (args[15] != Py_None) {
    const Tensor* topk = tensor(args[15], &dev);
    if (!topk || topk->scalar_type() != at::kInt || topk->dim() != 3 || topk->size(0) != c.heads || topk->size(1) != total ||
        topk->size(2) < 1 || topk->size(2) > 1024)
      return not_this();
    a.topk = (const int32_t*)topk->const_data_ptr();
    a.t_sh = topk->stride(0); a.t_sn = topk->stride(1); a.t_sk = topk->stride(2);
    a.topk_n = (int32_t)topk->size(2);
    if (args[16] != Py_None) {
      const Tensor* bias = tensor(args[16], &dev);
      if (!bias || bias->scalar_type() != at::kFloat || bias->sizes() != topk->sizes() || bias->strides() != topk->strides())
        return not_this();
      a.bias = (const float*)bias->const_data_ptr();
    }
  }
  Tensor out, lse;
  if (args[13] != Py_None) {
    const Tensor* o = tensor(args[13], &dev);
    if (!o || o->sizes() != q.sizes() || o->scalar_type() != q.scalar_type() || o->stride(2) != 1) return not_this();
    out = *o;
  } else {
    out = at::empty(q.sizes(), q.options());
  }
  if (args[14] == Py_True) {
    lse = at::empty({total, q.size(1)}, q.options().dtype(at::kFloat));
    a.lse = (float*)lse.mutable_data_ptr();
    a.lse_sn = q.size(1);
    a.lse_sh = 1;
  }
  a.q = q.const_data_ptr(); a.q_sn = q.stride(0); a.q_sh = q.stride(1);
  a.k_cache = kc.const_data_ptr(); a.k_sp = kc.stride(0); a.k_st = kc.stride(1); a.k_sh = kc.stride(2);
  a.v_cache = vc.const_data_ptr(); a.v_sp = vc.stride(0); a.v_st = vc.stride(1); a.v_sh = vc.stride(2);
  a.k_scale = (const float*)ks.const_data_ptr(); a.ks_sp = ks.stride(0); a.ks_sh = ks.stride(1);
  a.v_scale = (const float*)vs.const_data_ptr(); a.vs_sp = vs.stride(0); a.vs_sh = vs.stride(1);
  a.block_table = (const int32_t*)bt.const_data_ptr(); a.bt_sr = bt.stride(0);
  a.seq_lens = (const int32_t*)sl.const_data_ptr();
  a.out = out.mutable_data_ptr(); a.o_sn = out.stride(0); a.o_sh = out.stride(1);
  a.R = (int32_t)R; a.total_q = (int32_t)total; a.max_query_len = (int32_t)rows;
  a.HQ = (int32_t)q.size(1); a.HKV = (int32_t)c.heads; a.D = (int32_t)c.D;
  a.max_blocks = (int32_t)bt.size(1); a.num_pages = (int32_t)c.npages; a.page_size = (int32_t)c.page;
  a.window = (int32_t)window; a.sinks = (int32_t)sinks;
  a.scale = (float)PyFloat_AS_DOUBLE(args[10]);
  a.dtype = code; a.kv_dtype = c.code;
  const size_t need = form ? srswa_cache8_prefill_workspace(&a) : srswa_cache8_decode_workspace(&a);
  Tensor ws;
  if (need) ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
  void* wp = need ? ws.mutable_data_ptr() : nullptr;
  const int rc = form ? srswa_cache8_prefill(&a, wp, need, stream_of(dev)) : srswa_cache8_decode(&a, wp, need, stream_of(dev));
  if (rc != SRSWA_OK) return not_this();
  PyObject* po;
  if (args[13] != Py_None) {
    po = args[13];
    Py_INCREF(po);
  } else {
    po = THPVariable_Wrap(out);
  }
  if (!lse.defined()) return po;
  PyObject* pl = THPVariable_Wrap(lse);
  PyObject* both = PyTuple_Pack(2, po, pl);
  Py_DECREF(po);
  Py_DECREF(pl);
  return both;
  END_HANDLE_TH_ERRORS
}

// append(k, v, k_cache, v_cache, k_scale, v_scale, block_table, start, cu | None, max_new_len | None)
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10) return not_this();
  int dev = -1;
  const Tensor* t[8];
  for (int i = 0; i < 8; ++i)
    if (!(t[i] = tensor(args[i], &dev))) return not_this();
  if (dev != c10::hip::current_device()) return not_this();
  const Tensor &k = *t[0], &v = *t[1], &kc = *t[2], &vc = *t[3], &ks = *t[4], &vs = *t[5], &bt = *t[6], &st = *t[7];
  Cache c;
  if (!cache(kc, vc, ks, vs, &c) || !i32_rows(bt) || !i32_list(st)) return not_this();
  const int code = float_code(k);
  if (code < 0 || k.dim() != 3 || k.size(1) != c.heads || k.size(2) != c.D || v.sizes() != k.sizes() ||
      v.scalar_type() != k.scalar_type() || k.stride(2) != 1 || v.stride(2) != 1)
    return not_this();
  const int64_t total = k.size(0), R = st.size(0);
  if (total < 1 || total > INT32_MAX || R < 1 || R > INT32_MAX || bt.size(0) < R || bt.size(1) < 1 ||
      bt.size(1) > INT32_MAX)
    return not_this();
  srswa_cache8_append_args a{};
  int64_t most;
  if (args[8] != Py_None) {
    const Tensor* cu = tensor(args[8], &dev);
    if (!cu || !i32_list(*cu) || cu->size(0) != R + 1 || !as_long(args[9], 0, INT32_MAX, &most)) return not_this();
    a.cu_seqlens = (const int32_t*)cu->const_data_ptr();
    most = std::min(most, total);
  } else {
    if (args[9] != Py_None || total % R) return not_this();
    most = total / R;
  }
  a.k = k.const_data_ptr(); a.k_sn = k.stride(0); a.k_sh = k.stride(1);
  a.v = v.const_data_ptr(); a.v_sn = v.stride(0); a.v_sh = v.stride(1);
  a.k_cache = kc.mutable_data_ptr(); a.kc_sp = kc.stride(0); a.kc_st = kc.stride(1); a.kc_sh = kc.stride(2);
  a.v_cache = vc.mutable_data_ptr(); a.vc_sp = vc.stride(0); a.vc_st = vc.stride(1); a.vc_sh = vc.stride(2);
  a.k_scale = (float*)ks.mutable_data_ptr(); a.ks_sp = ks.stride(0); a.ks_sh = ks.stride(1);
  a.v_scale = (float*)vs.mutable_data_ptr(); a.vs_sp = vs.stride(0); a.vs_sh = vs.stride(1);
  a.block_table = (const int32_t*)bt.const_data_ptr(); a.bt_sr = bt.stride(0);
  a.start = (const int32_t*)st.const_data_ptr();
  a.R = (int32_t)R; a.total = (int32_t)total; a.max_new_len = (int32_t)most;
  a.HKV = (int32_t)c.heads; a.D = (int32_t)c.D; a.max_blocks = (int32_t)bt.size(1);
  a.num_pages = (int32_t)c.npages; a.page_size = (int32_t)c.page;
  a.dtype = code; a.kv_dtype = c.code;
  if (srswa_cache8_append(&a, stream_of(dev)) != SRSWA_OK) return not_this();
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// pages(entry, block_table, seq_lens, ref, rows | None, caches tuple, page_size): entry 0 reserve, 1 reorder,
// 2 compact; returns (block_table, seq_lens, ref, count)
PyObject* pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t entry, page;
  if (n != 7 || !as_long(args[0], 0, 2, &entry) || !as_long(args[6], 1, INT32_MAX, &page) || !PyTuple_CheckExact(args[5]))
    return not_this();
  int dev = -1;
  const Tensor* t[3];
  for (int i = 0; i < 3; ++i)
    if (!(t[i] = tensor(args[1 + i], &dev))) return not_this();
  if (dev != c10::hip::current_device()) return not_this();
  const Tensor &bt = *t[0], &sl = *t[1], &ref = *t[2];
  if (!i32_rows(bt) || !i32_list(sl) || !i32_list(ref)) return not_this();
  const int64_t R = bt.size(0), W = bt.size(1), N = ref.size(0);
  if (R < 1 || W < 1 || N < 1 || R > INT32_MAX || W > INT32_MAX || N > INT32_MAX || sl.size(0) != R) return not_this();
  srswa_pages_args a{};
  if (args[4] != Py_None) {
    const Tensor* rows = tensor(args[4], &dev);
    if (!rows || !i32_list(*rows) || rows->size(0) != R) return not_this();
    a.rows = (const int32_t*)rows->const_data_ptr();
  } else if (entry != 2) {
    return not_this();
  }
  const Py_ssize_t nc = PyTuple_GET_SIZE(args[5]);
  std::vector<srswa_page_cache> list;
  list.reserve(nc);
  for (Py_ssize_t i = 0; i < nc; ++i) {
    const Tensor* x = tensor(PyTuple_GET_ITEM(args[5], i), &dev);
    if (!x || x->dim() < 1 || x->size(0) != N) return not_this();
    const int64_t m = x->numel() / N, e = (int64_t)x->element_size();
    if (m == 0) continue;
    int64_t want = 1;                          // each page contiguous
    for (int64_t d = x->dim() - 1; d > 0; --d) {
      if (x->size(d) != 1 && x->stride(d) != want) return not_this();
      want *= x->size(d);
    }
    if (N > 1 && x->stride(0) < m) return not_this();
    list.push_back({x->mutable_data_ptr(), (N > 1 ? x->stride(0) : m) * e, m * e});
  }
  const Tensor nt = at::empty({R, W}, bt.options()), ns = at::empty({R}, bt.options()), nr = at::empty({N}, bt.options());
  const Tensor count = at::empty({1}, bt.options());
  a.block_table = (const int32_t*)bt.const_data_ptr(); a.bt_sr = bt.stride(0);
  a.seq_lens = (const int32_t*)sl.const_data_ptr();
  a.ref = (const int32_t*)ref.const_data_ptr();
  a.block_table_out = (int32_t*)nt.mutable_data_ptr(); a.bto_sr = W;
  a.seq_lens_out = (int32_t*)ns.mutable_data_ptr();
  a.ref_out = (int32_t*)nr.mutable_data_ptr();
  a.count = (int32_t*)count.mutable_data_ptr();
  a.caches = list.data();
  a.ncaches = (int32_t)list.size();
  a.R = (int32_t)R; a.W = (int32_t)W; a.num_pages = (int32_t)N; a.page_size = (int32_t)page;
  const size_t need = srswa_pages_workspace(&a);
  const Tensor ws = at::empty({(int64_t)need}, bt.options().dtype(at::kByte));
  void* wp = ws.mutable_data_ptr();
  void* st = stream_of(dev);
  const int rc = entry == 0 ? srswa_pages_reserve(&a, wp, need, st)
                 : entry == 1 ? srswa_pages_reorder(&a, wp, need, st) : srswa_pages_compact(&a, wp, need, st);
  if (rc != SRSWA_OK) return not_this();
  PyObject* o[4] = {THPVariable_Wrap(nt), THPVariable_Wrap(ns), THPVariable_Wrap(nr), THPVariable_Wrap(count)};
  PyObject* all = PyTuple_Pack(4, o[0], o[1], o[2], o[3]);
  for (PyObject* x : o) Py_XDECREF(x);
  return all;
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attend)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, nullptr},
    {"pages", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(pages)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&kModule); }
