// Python binding of the operators that continue sequences from cached state: argument checks, output
// allocation, device and stream selection and the C call, without per-argument Python work.  A decoding
// step's kernels run a few microseconds each; checked in Python and called through ctypes, one call cost 24
// to 31 us of host time.  Functions take positional arguments (None for an absent tensor); ops.py holds
// the keyword signatures and the documentation.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <stdexcept>
#include <string>

#include "../../include/fdk.h"

namespace {

PyObject* g_fdk_error = nullptr;  // _lib.FdkError: launch and device failures

struct Bad : std::runtime_error {  // refused arguments
  using std::runtime_error::runtime_error;
};

[[noreturn]] void bad(const char* name, const char* why) { throw Bad(std::string(name) + ": " + why); }

const at::Tensor* tensor_or_null(PyObject* o) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) throw Bad("a tensor (or None) was expected");
  return &THPVariable_Unpack(o);
}
const at::Tensor& tensor(PyObject* o) {
  const at::Tensor* t = tensor_or_null(o);
  if (!t) throw Bad("a tensor was expected, not None");
  return *t;
}
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Bad("an integer was expected");
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Bad("a truth value was expected");
  return v == 1;
}

// The one CUDA device of all given tensors.
int device_of(std::initializer_list<const at::Tensor*> ts) {
  int dev = -1;
  for (const at::Tensor* t : ts) {
    if (!t) continue;
    if (!t->is_cuda()) throw Bad("fastdecisions_b200 ops run on CUDA tensors only (no CPU fallback)");
    const int d = t->get_device();
    if (dev >= 0 && d != dev) throw Bad("all tensors must share one CUDA device");
    dev = d;
  }
  return dev;
}

template <typename T = void>
T* ptr(const at::Tensor* t) { return t ? static_cast<T*>(t->data_ptr()) : nullptr; }

void status(const char* name, int st) {
  if (st == FDK_OK) return;
  const std::string msg = std::string(name) + ": " + fdk_get_last_error_string();
  if (st == FDK_ERR_INVALID_ARGUMENT || st == FDK_ERR_ALIGNMENT || st == FDK_ERR_UNSUPPORTED) throw Bad(msg);
  PyErr_SetString(g_fdk_error ? g_fdk_error : PyExc_RuntimeError, msg.c_str());
  throw std::logic_error("");  // the Python error is set
}

struct Launch {  // the tensors' device as the current one, and its current stream
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit Launch(int dev) : guard((c10::DeviceIndex)dev), stream(at::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream()) {}
};

void int32_vector(const char* name, const char* what, const at::Tensor& t, int64_t n) {
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != n || (n > 1 && t.stride(0) != 1))
    bad(name, (std::string(what) + " must be a contiguous int32 vector of " + std::to_string(n) + " elements").c_str());
}

bool is(const at::Tensor& t, at::ScalarType type, std::initializer_list<int64_t> shape) {
  return t.scalar_type() == type && t.sizes() == at::IntArrayRef(shape.begin(), shape.size());
}

// ------------------------------------------------------------------------------------------ paged KV cache
struct Paged {
  const at::Tensor &k, &v, &table, &cu, &lens;
  const at::Tensor *ks, *vs;
  int quant = 0;
  int64_t pages, hkv, page_size, d, segments, max_pages, ld_table;

  Paged(const char* name, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table, const at::Tensor& cu,
        const at::Tensor& lens, const at::Tensor* ks, const at::Tensor* vs)
      : k(k), v(v), table(table), cu(cu), lens(lens), ks(ks), vs(vs) {
    const auto type = k.scalar_type();
    quant = type == at::kFloat8_e4m3fn;
    if (k.dim() != 4 || v.sizes() != k.sizes() || v.scalar_type() != type || !(quant || type == at::kBFloat16))
      bad(name, "caches must be [pages, kv heads, page size, head_dim], both bf16 or both e4m3");
    pages = k.size(0);
    hkv = k.size(1);
    page_size = k.size(2);
    d = k.size(3);
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)) || (d != 128 && d != 256))
      bad(name, "page sizes 16, 32, 64, 128 and 256 and head_dim 128 or 256 supported");
    for (const at::Tensor* t : {&k, &v})
      if ((hkv > 1 && t->stride(1) != page_size * d) || t->stride(2) != d || t->stride(3) != 1)
        bad(name, "a cache page must be contiguous (only the page stride is free)");
    if (quant) {
      for (const at::Tensor* t : {ks, vs}) {
        if (!t || !is(*t, at::kByte, {pages, hkv, page_size}))
          bad(name, "an e4m3 cache needs uint8 k_scale and v_scale [pages, kv heads, page size]");
        if ((hkv > 1 && t->stride(1) != page_size) || t->stride(2) != 1)
          bad(name, "the scales of a page must be contiguous (only the page stride is free)");
      }
    } else if (ks || vs) {
      bad(name, "a bf16 cache has no scales");
    }
    segments = lens.numel();
    int32_vector(name, "kv_lens", lens, segments);
    int32_vector(name, "cu_seqlens", cu, segments + 1);
    if (segments < 1 || table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != segments ||
        table.size(1) < 1 || (table.size(1) > 1 && table.stride(1) != 1))
      bad(name, "page_table must be int32 [segments, pages] with unit column stride");
    max_pages = table.size(1);
    ld_table = segments > 1 ? table.stride(0) : max_pages;
  }
  // Page strides; a single page has none of its own.
  int64_t page_stride(const at::Tensor& t, int64_t elems) const { return pages > 1 ? t.stride(0) : elems; }
  int64_t ld_k() const { return page_stride(k, hkv * page_size * d); }
  int64_t ld_v() const { return page_stride(v, hkv * page_size * d); }
  int64_t ld_ks() const { return quant ? page_stride(*ks, hkv * page_size) : 0; }
  int64_t ld_vs() const { return quant ? page_stride(*vs, hkv * page_size) : 0; }
};

// Token stride of bf16 rows [tokens, heads, d].
int64_t token_rows(const char* name, const char* what, const at::Tensor& t, int64_t heads, int64_t d) {
  if (t.dim() != 3 || t.size(1) != heads || t.size(2) != d || t.scalar_type() != at::kBFloat16 || t.stride(2) != 1 ||
      (heads > 1 && t.stride(1) != d))
    bad(name, (std::string(what) + " must be bf16 [tokens, " + std::to_string(heads) + ", " + std::to_string(d) +
               "] with head stride " + std::to_string(d)).c_str());
  return t.size(0) > 1 ? t.stride(0) : heads * d;
}

PyObject* paged_kv_write(PyObject* const* a) {
  const char* name = "paged_kv_write";
  const at::Tensor &k = tensor(a[0]), &v = tensor(a[1]);
  const at::Tensor *ks = tensor_or_null(a[7]), *vs = tensor_or_null(a[8]);
  const at::Tensor &kc = tensor(a[2]), &vc = tensor(a[3]), &table = tensor(a[4]), &cu = tensor(a[5]), &lens = tensor(a[6]);
  const int dev = device_of({&k, &v, &kc, &vc, &table, &cu, &lens, ks, vs});
  const Paged c(name, kc, vc, table, cu, lens, ks, vs);
  const int64_t ldk = token_rows(name, "k", k, c.hkv, c.d), ldv = token_rows(name, "v", v, c.hkv, c.d);
  if (v.size(0) != k.size(0)) bad(name, "k and v must have the same tokens");
  Launch l(dev);
  status(name, fdk_paged_kv_write(k.data_ptr(), ldk, v.data_ptr(), ldv, kc.data_ptr(), c.ld_k(), vc.data_ptr(),
                                  c.ld_v(), c.quant, ptr(ks), c.ld_ks(), ptr(vs), c.ld_vs(), c.pages, c.page_size,
                                  ptr<int32_t>(&table), c.ld_table, c.max_pages, ptr<int32_t>(&cu), ptr<int32_t>(&lens),
                                  c.segments, k.size(0), c.hkv, c.d, l.stream));
  Py_RETURN_NONE;
}

PyObject* paged_kv_read(PyObject* const* a) {
  const char* name = "paged_kv_read";
  const at::Tensor &kc = tensor(a[0]), &vc = tensor(a[1]), &table = tensor(a[2]), &cu = tensor(a[3]), &lens = tensor(a[4]);
  const int64_t tokens = integer(a[5]);
  const at::Tensor *ks = tensor_or_null(a[6]), *vs = tensor_or_null(a[7]), *ko = tensor_or_null(a[8]), *vo = tensor_or_null(a[9]);
  const int dev = device_of({&kc, &vc, &table, &cu, &lens, ks, vs, ko, vo});
  const Paged c(name, kc, vc, table, cu, lens, ks, vs);
  if (tokens < 0) bad(name, "tokens must not be negative");
  for (const at::Tensor* t : {ko, vo})
    if (t && (!is(*t, at::kBFloat16, {tokens, c.hkv, c.d}) || !t->is_contiguous()))
      bad(name, "outputs must be contiguous bf16 [tokens, kv heads, head_dim]");
  Launch l(dev);
  const auto opt = kc.options().dtype(at::kBFloat16);
  const at::Tensor k = ko ? *ko : at::empty({tokens, c.hkv, c.d}, opt), v = vo ? *vo : at::empty({tokens, c.hkv, c.d}, opt);
  status(name, fdk_paged_kv_read(kc.data_ptr(), c.ld_k(), vc.data_ptr(), c.ld_v(), c.quant, ptr(ks), c.ld_ks(),
                                 ptr(vs), c.ld_vs(), c.pages, c.page_size, ptr<int32_t>(&table), c.ld_table, c.max_pages,
                                 ptr<int32_t>(&cu), ptr<int32_t>(&lens), c.segments, tokens, c.hkv, c.d, k.data_ptr(),
                                 v.data_ptr(), l.stream));
  PyObject *pk = THPVariable_Wrap(k), *pv = THPVariable_Wrap(v);
  PyObject* r = PyTuple_Pack(2, pk, pv);
  Py_XDECREF(pk);
  Py_XDECREF(pv);
  return r;
}

PyObject* paged_gqa_attention(PyObject* const* a) {
  const char* name = "paged_gqa_attention";
  const at::Tensor& q = tensor(a[0]);
  const at::Tensor &kc = tensor(a[1]), &vc = tensor(a[2]), &table = tensor(a[3]), &cu = tensor(a[4]), &lens = tensor(a[5]);
  const at::Tensor *ks = tensor_or_null(a[8]), *vs = tensor_or_null(a[9]), *gate = tensor_or_null(a[11]);
  const at::Tensor *out = tensor_or_null(a[13]), *ws = tensor_or_null(a[14]);
  const int dev = device_of({&q, &kc, &vc, &table, &cu, &lens, ks, vs, gate, out, ws});
  const Paged c(name, kc, vc, table, cu, lens, ks, vs);
  if (q.dim() != 3 || q.size(1) < 1 || q.size(1) % c.hkv)
    bad(name, "q must be [tokens, query heads, head_dim], whole groups of query heads");
  const int64_t T = q.size(0), hq = q.size(1), d = c.d;
  const int64_t ldq = token_rows(name, "q", q, hq, d);
  const bool inter = truth(a[12]);
  int64_t ldg = 0;
  if (gate) {
    const int64_t span = inter ? (2 * hq - 1) * d : hq * d;
    if (gate->dim() != 2 || gate->scalar_type() != at::kBFloat16 || gate->size(0) != T || gate->size(1) < span || gate->stride(1) != 1)
      bad(name, ("gate must be bf16 [tokens, >= " + std::to_string(span) + "] with unit column stride").c_str());
    ldg = T > 1 ? gate->stride(0) : (gate->size(1) + 7) / 8 * 8;
  }
  if (out && (!is(*out, at::kBFloat16, {T, hq, d}) || !out->is_contiguous())) bad(name, "out must be contiguous bf16 shaped like q");
  if (ws && !ws->is_contiguous()) bad(name, "workspace must be contiguous");
  // cut to what the library takes; to the table's reach only where no workspace was sized for the caller's own value
  const int64_t reach = c.max_pages * c.page_size, most = ws ? 0x7fffff00 : std::min<int64_t>(reach, 0x7fffff00);
  const int64_t max_seqlen = std::min<int64_t>(integer(a[6]), 0x7fffffff);
  const int64_t max_kv = std::min(a[7] == Py_None ? reach : integer(a[7]), most);
  if (max_seqlen < 0 || max_kv < 0) bad(name, "max_seqlen and max_kv_len must not be negative");
  double scale = 1.0 / std::sqrt((double)d);
  if (a[10] != Py_None) {
    scale = PyFloat_AsDouble(a[10]);
    if (scale == -1.0 && PyErr_Occurred()) throw Bad("paged_gqa_attention: scale must be a number");
  }
  Launch l(dev);
  const at::Tensor o = out ? *out : at::empty({T, hq, d}, q.options());
  at::Tensor scratch;
  if (!ws) {
    const size_t need = fdk_paged_gqa_workspace_size(c.segments, max_seqlen, max_kv, T, hq, c.hkv, d, c.quant);
    if (need) {
      scratch = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
      ws = &scratch;
    }
  }
  status(name, fdk_paged_gqa_fwd(q.data_ptr(), ldq, kc.data_ptr(), c.ld_k(), vc.data_ptr(), c.ld_v(), c.quant,
                                 ptr(ks), c.ld_ks(), ptr(vs), c.ld_vs(), c.pages, c.page_size, ptr<int32_t>(&table),
                                 c.ld_table, c.max_pages, ptr<int32_t>(&cu), ptr<int32_t>(&lens), c.segments, max_seqlen,
                                 max_kv, T, hq, c.hkv, d, (float)scale, ptr(gate), ldg, inter, o.data_ptr(), ptr(ws),
                                 ws ? (size_t)ws->nbytes() : 0, l.stream));
  return THPVariable_Wrap(o);
}

// ------------------------------------------------------------------------------------------ pools of states
// Segments of [B, T, ...] tokens: cu_seqlens' (B == 1), else the batch entries.
int64_t segments_of(const char* name, int64_t B, const at::Tensor* cu) {
  if (!cu) return B;
  if (B != 1) bad(name, "cu_seqlens needs batch size 1");
  const int64_t n = cu->numel();
  int32_vector(name, "cu_seqlens", *cu, n);
  if (n < 2) bad(name, "cu_seqlens must have at least two elements");
  return n - 1;
}

void slots(const char* name, const at::Tensor* pool, const at::Tensor* idx, int64_t S) {
  if (idx) int32_vector(name, "slot indices", *idx, S);
  else if (pool && pool->size(0) < S) bad(name, (std::to_string(S) + " segments need at least as many state slots").c_str());
}

// [B, T, H, D] as rows of one token stride (a copy when the layout has none).
at::Tensor rows_of(const char* name, const char* what, const at::Tensor& t, int64_t& ld) {
  if (t.scalar_type() != at::kBFloat16) bad(name, (std::string(what) + " must be bf16").c_str());
  const int64_t B = t.size(0), T = t.size(1), H = t.size(2), D = t.size(3);
  const bool fits = t.stride(3) == 1 && (H == 1 || t.stride(2) == D) && (B == 1 || T == 1 || t.stride(0) == T * t.stride(1));
  at::Tensor r = fits ? t : t.contiguous();
  ld = T > 1 ? r.stride(1) : B > 1 ? r.stride(0) : H * D;
  return r;
}

// name, query, key, value, g, beta, initial pool, its indices, final pool, its indices, cu_seqlens, l2norm, out
PyObject* recurrent_gated_delta_rule(PyObject* const* a) {
  const char* name = PyUnicode_AsUTF8(a[0]);
  if (!name) throw Bad("a name was expected");
  const at::Tensor &query = tensor(a[1]), &key = tensor(a[2]), &value = tensor(a[3]), &g = tensor(a[4]), &beta = tensor(a[5]);
  const at::Tensor *init = tensor_or_null(a[6]), *init_idx = tensor_or_null(a[7]), *fin = tensor_or_null(a[8]),
                   *fin_idx = tensor_or_null(a[9]), *cu = tensor_or_null(a[10]), *out = tensor_or_null(a[12]);
  const int dev = device_of({&query, &key, &value, &g, &beta, init, init_idx, fin, fin_idx, cu, out});
  if (query.dim() != 4 || key.sizes() != query.sizes() || value.dim() != 4) bad(name, "expected [B, T, H, D] query/key/value");
  const int64_t B = key.size(0), T = key.size(1), Hk = key.size(2), H = value.size(2);
  const int64_t like[3] = {B, T, H};
  if (value.size(0) != B || value.size(1) != T || g.sizes() != at::IntArrayRef(like) || beta.sizes() != at::IntArrayRef(like))
    bad(name, "shape mismatch between q/k/v/g/beta");
  if (key.size(3) != 128 || value.size(3) != 128) bad(name, "head dims must be 128");
  if (Hk < 1 || H < 1 || H % Hk) bad(name, "value heads must be a multiple of the key heads");
  const int64_t S = segments_of(name, B, cu);
  for (const at::Tensor* p : {init, fin})
    if (p && (p->dim() != 4 || !is(*p, at::kFloat, {p->size(0), H, 128, 128}) || !p->is_contiguous()))
      bad(name, "states must be contiguous float32 [slots, heads, 128, 128]");
  slots(name, init, init_idx, S);
  slots(name, fin, fin_idx, S);
  if (out && (!is(*out, at::kBFloat16, {B, T, H, 128}) || !out->is_contiguous()))
    bad(name, "out must be contiguous bf16 [B, T, H, 128]");
  Launch l(dev);
  const at::Tensor o = out ? *out : at::empty({B, T, H, 128}, value.options());
  if (S > 0) {
    int64_t ldq, ldk, ldv;
    const at::Tensor q = rows_of(name, "query", query, ldq), k = rows_of(name, "key", key, ldk), v = rows_of(name, "value", value, ldv);
    const at::Tensor gg = g.to(at::kFloat).contiguous(), bb = beta.to(at::kBFloat16).contiguous();
    status(name, fdk_recurrent_gated_delta_rule_fwd(
                     q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, ptr<float>(&gg), bb.data_ptr(), ptr<int32_t>(cu), S,
                     B * T, Hk, H, 128, 128, 1.f / std::sqrt(128.f), truth(a[11]), ptr<float>(init), ptr<int32_t>(init_idx),
                     init ? init->size(0) : 0, ptr<float>(fin), ptr<int32_t>(fin_idx), fin ? fin->size(0) : 0, o.data_ptr(),
                     l.stream));
  }
  return THPVariable_Wrap(o);
}

// x, weight, state, state_indices, final_indices, key_dim, value_dim, head_dim, cu_seqlens
PyObject* packed_conv_state(PyObject* const* a) {
  const char* name = "packed_conv_state_";
  const at::Tensor &x = tensor(a[0]), &w = tensor(a[1]), &state = tensor(a[2]);
  const at::Tensor *idx = tensor_or_null(a[3]), *fin = tensor_or_null(a[4]), *cu = tensor_or_null(a[8]);
  const int dev = device_of({&x, &w, &state, idx, fin, cu});
  if (x.dim() != 3 || x.scalar_type() != at::kBFloat16 || w.scalar_type() != at::kBFloat16) bad(name, "expected bf16 x [B, T, C] and weight");
  const int64_t B = x.size(0), T = x.size(1), C = x.size(2);
  if ((w.dim() != 2 && (w.dim() != 3 || w.size(1) != 1)) || w.size(0) != C || w.size(-1) < 2 || w.size(-1) > 4 || !w.is_contiguous())
    bad(name, "weight must be a contiguous [C, K] or [C, 1, K] tensor with K from 2 to 4");
  const int64_t K = w.size(-1), hd = integer(a[7]);
  const int64_t key_dim = a[5] == Py_None ? C / 3 : integer(a[5]);
  const int64_t value_dim = a[6] == Py_None ? C - 2 * key_dim : integer(a[6]);
  if (hd < 1 || key_dim < 1 || value_dim < 1 || 2 * key_dim + value_dim != C || key_dim % hd || value_dim % hd)
    bad(name, "C must equal 2*key_dim + value_dim with whole heads");
  if (state.dim() != 3 || !is(state, at::kBFloat16, {state.size(0), K - 1, C}) || !state.is_contiguous())
    bad(name, "state must be contiguous bf16 [slots, K - 1, C]");
  const int64_t S = segments_of(name, B, cu);
  if (!fin) fin = idx;
  slots(name, &state, idx, S);
  slots(name, &state, fin, S);
  Launch l(dev);
  const at::Tensor xc = x.stride(2) != 1 || (B > 1 && T > 1 && x.stride(0) != T * x.stride(1)) ? x.contiguous() : x;
  const int64_t ldx = T > 1 ? xc.stride(1) : B > 1 ? xc.stride(0) : C;
  const at::Tensor q = at::empty({B, T, key_dim / hd, hd}, x.options()), k = at::empty({B, T, key_dim / hd, hd}, x.options());
  const at::Tensor v = at::empty({B, T, value_dim / hd, hd}, x.options());
  if (S > 0)
    status(name, fdk_packed_conv_state(xc.data_ptr(), ldx, w.data_ptr(), ptr<int32_t>(cu), S, B * T, C, (int)K, key_dim, value_dim,
                                       state.data_ptr(), ptr<int32_t>(idx), state.size(0), state.data_ptr(), ptr<int32_t>(fin),
                                       state.size(0), q.data_ptr(), k.data_ptr(), v.data_ptr(), l.stream));
  PyObject *pq = THPVariable_Wrap(q), *pk = THPVariable_Wrap(k), *pv = THPVariable_Wrap(v);
  PyObject* r = PyTuple_Pack(3, pq, pk, pv);
  Py_XDECREF(pq);
  Py_XDECREF(pk);
  Py_XDECREF(pv);
  return r;
}

// No C++ exception leaves a function of the module.
template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  try {
    if (n != N) throw Bad(std::to_string(N) + " arguments expected");
    return F(args);
  } catch (const Bad& e) {
    PyErr_Clear();
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

PyObject* set_error_class(PyObject*, PyObject* cls) {
  Py_XINCREF(cls);
  Py_XDECREF(g_fdk_error);
  g_fdk_error = cls;
  Py_RETURN_NONE;
}

#define ENTRY(f, n) {#f, (PyCFunction)(void (*)(void))(PyObject * (*)(PyObject*, PyObject* const*, Py_ssize_t)) entry<f, n>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(paged_kv_write, 9),
                         ENTRY(paged_kv_read, 10),
                         ENTRY(paged_gqa_attention, 15),
                         ENTRY(recurrent_gated_delta_rule, 13),
                         ENTRY(packed_conv_state, 9),
                         {"set_error_class", set_error_class, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fdk_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fdk_torch() { return PyModule_Create(&module); }
