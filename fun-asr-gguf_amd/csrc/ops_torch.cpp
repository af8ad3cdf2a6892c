// torch binding of the drafted-token operators (fun_asr_gguf/ops.py): tensors are checked and unpacked here, so that a call on
// a few tokens costs a few microseconds of host time (filling the argument structures from Python took 12 to 15).
// The C entries are handed over as addresses by bind(): the library that fun_asr_gguf._native has loaded is the one used.
// ValueError before anything is enqueued for tensors that do not fit; RuntimeError with the library's message for what it
// refuses.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>

#include "funasr_hip.h"

namespace {

decltype(&fa_qk_norm_rope) norm_rope_fn;
decltype(&fa_kv_append) append_fn;
decltype(&fa_tree_attention) attention_fn;
decltype(&fa_tree_attention_workspace) attention_ws_fn;
decltype(&fa_sample_tokens) sample_fn;
decltype(&fa_sample_tokens_workspace) sample_ws_fn;
decltype(&fa_last_error) error_fn;

#define NEED(cond, msg) TORCH_CHECK_VALUE(cond, msg)

void check(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, " failed (", rc, "): ", error_fn());
}

// a tensor argument, nullptr for None
const at::Tensor* tensor(PyObject* o, const char* name) {
  if (o == Py_None) return nullptr;
  NEED(THPVariable_Check(o), c10::str(name, " must be a tensor"));
  const at::Tensor& t = THPVariable_Unpack(o);
  NEED(!t.requires_grad() || !c10::GradMode::is_enabled(), c10::str(name, " requires a gradient: call under torch.no_grad()"));
  NEED(!t.unsafeGetTensorImpl()->autograd_meta() || !t._fw_grad(0).defined(),
       c10::str(name, " has a tangent: there is no forward-mode gradient"));
  NEED(!t.is_neg(), c10::str(name, " is a negated view"));
  return &t;
}
const at::Tensor& gpu(PyObject* o, const char* name) {
  const at::Tensor* t = tensor(o, name);
  NEED(t && t->is_cuda(), c10::str(name, " must be a tensor on the GPU"));
  return *t;
}
// a tensor that is written: no two elements in one place
void written(const at::Tensor& t, const char* name) {
  NEED(at::has_internal_overlap(t) != at::MemOverlap::Yes, c10::str(name, " has elements that share memory"));
}
// a caller's tensor after the call: autograd notices that one it has saved is another now (an inference tensor has no version, nor
// is it saved)
void changed(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void changed(PyObject* o) {
  if (o != Py_None) changed(THPVariable_Unpack(o));
}
int type_of(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return FA_F32;
    case at::kHalf: return FA_F16;
    case at::kBFloat16: return FA_BF16;
    default: NEED(false, c10::str(name, ": type ", t.scalar_type()));
  }
  return -1;
}
void on(const at::Device& d, const at::Tensor* t, const char* name) {
  NEED(!t || t->device() == d, c10::str(name, " is on ", t->device(), ", not on ", d));
}
bool last_contiguous(const at::Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }
bool vector_of(const at::Tensor& t, int64_t n) { return t.dim() == 1 && t.size(0) == n && (n < 2 || t.stride(0) == 1); }
bool whole(const at::Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }
double number(PyObject* o, const char* name) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    NEED(false, c10::str(name, " must be a number"));
  }
  return x;
}
int truth(PyObject* o) {
  const int x = PyObject_IsTrue(o);
  if (x < 0) throw python_error();  // the object's own error (a tensor of several elements)
  return x;
}
at::Tensor fresh(at::IntArrayRef size, at::ScalarType type, const at::Device& d) {
  return at::Tensor(at::detail::empty_cuda(size, at::TensorOptions().dtype(type).device(d)));
}

// makes the tensors' device the current one where it is not
struct OnDevice {
  std::optional<c10::DeviceGuard> guard;
  void* stream;
  explicit OnDevice(const at::Device& d) {
    if (c10::hip::current_device() != d.index()) guard.emplace(d);
    stream = c10::hip::getCurrentHIPStream(d.index()).stream();
  }
};

template <typename A>
at::Tensor workspace(A& a, int (*query)(const A*, int64_t*), const char* what, const at::Device& d) {
  int64_t n = 0;
  check(query(&a, &n), what);
  if (!n) return {};
  at::Tensor ws = fresh({n}, at::kByte, d);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = n;
  return ws;
}

void arity(Py_ssize_t n, Py_ssize_t want) { TORCH_CHECK_TYPE(n == want, "expected ", want, " arguments, got ", n); }

// ------------------------------------------------------------------------------------------------------------- head rows
void head_args(fa_head_rows_args& a, const at::Tensor& k, const at::Tensor* q, const at::Tensor* cos, const at::Tensor* sin,
               const at::Tensor* positions, const at::Tensor* qw, const at::Tensor* kw, double eps, int interleaved) {
  const at::Device d = k.device();
  a.type = type_of(k, "k");
  NEED(k.dim() == 3 && last_contiguous(k), "k must be [tokens, kv_heads, head_dim] with contiguous heads");
  const int64_t T = k.size(0), KV = k.size(1), D = k.size(2);
  NEED(T < (1ll << 31) && KV < (1ll << 31) && D < (1ll << 31), "k: size");
  on(d, q, "q");
  on(d, cos, "cos");
  on(d, sin, "sin");
  on(d, positions, "positions");
  on(d, qw, "q_weight");
  on(d, kw, "k_weight");
  if (q) {
    NEED(q->dim() == 3 && q->size(0) == T && q->size(2) == D && q->scalar_type() == k.scalar_type() && last_contiguous(*q) &&
             q->size(1) < (1ll << 31),
         "q must be [tokens, heads, head_dim] of k's type with contiguous heads");
    a.q = q->data_ptr();
    a.q_token = q->stride(0);
    a.q_head = q->stride(1);
    a.heads = (int32_t)q->size(1);
  }
  for (const at::Tensor* w : {qw, kw})
    NEED(!w || (w->scalar_type() == at::kFloat && vector_of(*w, D)), "the norms' weights must be float32 [head_dim]");
  NEED(!cos == !sin && !cos == !positions, "cos, sin and positions come together");
  if (cos) {
    NEED(cos->scalar_type() == at::kFloat && sin->scalar_type() == at::kFloat && cos->dim() == 2 && cos->sizes() == sin->sizes() &&
             cos->is_contiguous() && sin->is_contiguous() && cos->size(0) < (1ll << 31) && cos->size(1) < (1ll << 30),
         "cos and sin must be contiguous float32 [table, rot_dim / 2]");
    NEED(whole(*positions) && vector_of(*positions, T), "positions must be int32 or int64 [tokens]");
    a.cos = cos->data_ptr<float>();
    a.sin = sin->data_ptr<float>();
    a.positions = positions->data_ptr();
    a.table_len = (int32_t)cos->size(0);
    a.rot_dim = 2 * (int32_t)cos->size(1);
    a.positions_64 = positions->scalar_type() == at::kLong;
  }
  a.q_weight = qw ? qw->data_ptr<float>() : nullptr;
  a.k_weight = kw ? kw->data_ptr<float>() : nullptr;
  a.k = k.data_ptr();
  a.k_token = k.stride(0);
  a.k_head = k.stride(1);
  a.tokens = (int32_t)T;
  a.kv_heads = (int32_t)KV;
  a.head_dim = (int32_t)D;
  a.interleaved = interleaved;
  a.eps = (float)eps;
}
at::Tensor rows_out(const at::Tensor& x, const at::Tensor* out, const char* name) {
  if (!out) return fresh(x.sizes(), x.scalar_type(), x.device());
  NEED(out->sizes() == x.sizes() && out->scalar_type() == x.scalar_type() && out->device() == x.device() && last_contiguous(*out),
       c10::str(name, " must be like its input, with contiguous heads"));
  written(*out, name);
  return *out;
}

PyObject* qk_norm_rope(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 11);
  const at::Tensor *q = tensor(v[0], "q"), *cos = tensor(v[2], "cos"), *sin = tensor(v[3], "sin"), *pos = tensor(v[4], "positions");
  const at::Tensor& k = gpu(v[1], "k");
  NEED(q, "q is missing (kv_append takes keys alone)");
  fa_head_rows_args a{};
  head_args(a, k, q, cos, sin, pos, tensor(v[5], "q_weight"), tensor(v[6], "k_weight"), number(v[7], "eps"), truth(v[8]));
  const at::Tensor oq = rows_out(*q, tensor(v[9], "out_q"), "out_q"), ok = rows_out(k, tensor(v[10], "out_k"), "out_k");
  a.q_out = oq.data_ptr();
  a.q_out_token = oq.stride(0);
  a.q_out_head = oq.stride(1);
  a.k_out = ok.data_ptr();
  a.k_out_token = ok.stride(0);
  a.k_out_head = ok.stride(1);
  OnDevice dev(k.device());
  check(norm_rope_fn(&a, dev.stream), "fa_qk_norm_rope");
  changed(v[9]);
  changed(v[10]);
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(oq));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(ok));
  return r;
  END_HANDLE_TH_ERRORS
}

// the caches' shape, type and strides
void cache_args(const at::Tensor& kc, const at::Tensor& vc, int64_t D) {
  NEED((kc.scalar_type() == at::kHalf || kc.scalar_type() == at::kBFloat16) && vc.scalar_type() == kc.scalar_type() && kc.dim() == 4 &&
           vc.sizes() == kc.sizes() && kc.size(3) == D && last_contiguous(kc) && last_contiguous(vc) && kc.size(0) < (1ll << 31) &&
           kc.size(1) < (1ll << 31) && kc.size(2) < (1ll << 31),
       "the caches must be float16 or bfloat16 [pages, kv_heads, page_size, head_dim] with contiguous rows");
}

PyObject* kv_append(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 14);
  const at::Tensor &k = gpu(p[0], "k"), &v = gpu(p[1], "v"), &kc = gpu(p[2], "k_cache"), &vc = gpu(p[3], "v_cache"),
                   &slots = gpu(p[4], "slots");
  const at::Tensor *cos = tensor(p[5], "cos"), *sin = tensor(p[6], "sin"), *pos = tensor(p[7], "positions"), *q = tensor(p[9], "q");
  NEED(q || p[10] == Py_None, "q_weight without q");
  NEED(q || p[13] == Py_None, "out_q without q");
  const at::Device d = k.device();
  fa_head_rows_args a{};
  head_args(a, k, q, cos, sin, pos, tensor(p[10], "q_weight"), tensor(p[8], "k_weight"), number(p[11], "eps"), truth(p[12]));
  on(d, &v, "v");
  on(d, &kc, "k_cache");
  on(d, &vc, "v_cache");
  on(d, &slots, "slots");
  NEED(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && last_contiguous(v), "v must be like k");
  cache_args(kc, vc, k.size(2));
  NEED(kc.size(1) == k.size(1), "the caches must have k's heads");
  written(kc, "k_cache");
  written(vc, "v_cache");
  NEED(whole(slots) && vector_of(slots, k.size(0)), "slots must be int32 or int64 [tokens]");
  at::Tensor oq;
  if (q) {
    oq = rows_out(*q, tensor(p[13], "out_q"), "out_q");
    a.q_out = oq.data_ptr();
    a.q_out_token = oq.stride(0);
    a.q_out_head = oq.stride(1);
  }
  a.v = v.data_ptr();
  a.v_token = v.stride(0);
  a.v_head = v.stride(1);
  a.k_out = kc.data_ptr();
  a.v_out = vc.data_ptr();
  a.k_out_page = kc.stride(0);
  a.k_out_head = kc.stride(1);
  a.k_out_token = kc.stride(2);
  a.v_out_page = vc.stride(0);
  a.v_out_head = vc.stride(1);
  a.v_out_token = vc.stride(2);
  a.pages = (int32_t)kc.size(0);
  a.page_size = (int32_t)kc.size(2);
  a.cache_type = type_of(kc, "k_cache");
  a.slots = slots.data_ptr();
  a.slots_64 = slots.scalar_type() == at::kLong;
  OnDevice dev(d);
  check(append_fn(&a, dev.stream), "fa_kv_append");
  changed(kc);
  changed(vc);
  if (!q) Py_RETURN_NONE;
  changed(p[13]);
  return THPVariable_Wrap(oq);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------------------------------- attention
PyObject* tree_attention(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 10);
  const at::Tensor &q = gpu(p[0], "q"), &kc = gpu(p[1], "k_cache"), &vc = gpu(p[2], "v_cache"), &table = gpu(p[3], "block_table"),
                   &ctx = gpu(p[4], "context_lens");
  const at::Tensor *mask = tensor(p[5], "mask"), *drafts = tensor(p[6], "draft_lens"), *given = tensor(p[9], "out");
  const at::Device d = q.device();
  fa_tree_attention_args a{};
  a.q_type = type_of(q, "q");
  NEED(q.dim() == 4 && last_contiguous(q), "q must be [seqs, nodes, heads, head_dim] with contiguous heads");
  const int64_t B = q.size(0), N = q.size(1), H = q.size(2), D = q.size(3);
  NEED(B < (1ll << 31) && N < (1ll << 31) && H < (1ll << 31) && D < (1ll << 31), "q: size");
  on(d, &kc, "k_cache");
  on(d, &vc, "v_cache");
  on(d, &table, "block_table");
  on(d, &ctx, "context_lens");
  on(d, mask, "mask");
  on(d, drafts, "draft_lens");
  on(d, given, "out");
  cache_args(kc, vc, D);
  NEED(table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == B && last_contiguous(table) &&
           table.size(1) < (1ll << 31),
       "block_table must be int32 [seqs, width]");
  NEED(ctx.scalar_type() == at::kInt && vector_of(ctx, B), "context_lens must be int32 [seqs]");
  NEED(!drafts || (drafts->scalar_type() == at::kInt && vector_of(*drafts, B)), "draft_lens must be int32 [seqs]");
  if (mask) {
    const int64_t m = mask->dim();
    NEED((mask->scalar_type() == at::kBool || mask->scalar_type() == at::kByte) && (m == 2 || m == 3) && mask->size(m - 1) == N &&
             mask->size(m - 2) == N && (m == 2 || mask->size(0) == B) && last_contiguous(*mask),
         "mask must be bool [nodes, nodes] or [seqs, nodes, nodes]");
    a.mask = reinterpret_cast<const uint8_t*>(mask->data_ptr());
    a.mask_row = mask->stride(m - 2);
    a.mask_seq = m == 3 ? mask->stride(0) : 0;
  }
  at::Tensor out;
  if (given) {
    NEED(given->sizes() == q.sizes() && given->scalar_type() == q.scalar_type() && last_contiguous(*given), "out must be like q");
    written(*given, "out");
    out = *given;
  } else {
    out = fresh(q.sizes(), q.scalar_type(), d);
  }
  a.q = q.data_ptr();
  a.out = out.data_ptr();
  a.k_cache = kc.data_ptr();
  a.v_cache = vc.data_ptr();
  a.block_table = table.data_ptr<int32_t>();
  a.context_lens = ctx.data_ptr<int32_t>();
  a.draft_lens = drafts ? drafts->data_ptr<int32_t>() : nullptr;
  a.q_seq = q.stride(0);
  a.q_node = q.stride(1);
  a.q_head = q.stride(2);
  a.out_seq = out.stride(0);
  a.out_node = out.stride(1);
  a.out_head = out.stride(2);
  a.k_page = kc.stride(0);
  a.k_head = kc.stride(1);
  a.k_slot = kc.stride(2);
  a.v_page = vc.stride(0);
  a.v_head = vc.stride(1);
  a.v_slot = vc.stride(2);
  a.table_seq = table.stride(0);
  a.table_len = (int32_t)table.size(1);
  a.seqs = (int32_t)B;
  a.nodes = (int32_t)N;
  a.heads = (int32_t)H;
  a.kv_heads = (int32_t)kc.size(1);
  a.head_dim = (int32_t)D;
  a.cache_type = type_of(kc, "k_cache");
  a.pages = (int32_t)kc.size(0);
  a.page_size = (int32_t)kc.size(2);
  a.scale = p[7] == Py_None ? (float)(1.0 / std::sqrt((double)D)) : (float)number(p[7], "scale");
  if (p[8] != Py_None) {
    const double m = number(p[8], "max_context");
    NEED(m >= 0 && m < 2147483648.0, "max_context must be a length");
    a.max_context = (int32_t)m;
  }
  OnDevice dev(d);
  const at::Tensor ws = workspace(a, attention_ws_fn, "fa_tree_attention", d);
  check(attention_fn(&a, dev.stream), "fa_tree_attention");
  changed(p[9]);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// -------------------------------------------------------------------------------------------------------------- sampling
PyObject* sample_tokens(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 8);
  const at::Tensor &x = gpu(p[0], "logits"), &u = gpu(p[1], "u");
  const at::Device d = x.device();
  fa_sample_args a{};
  a.type = type_of(x, "logits");
  NEED(x.dim() == 2 && last_contiguous(x) && x.size(0) < (1ll << 31) && x.size(1) < (1ll << 31),
       "logits must be [rows, vocab] with contiguous rows");
  const int64_t R = x.size(0);
  on(d, &u, "u");
  NEED(u.scalar_type() == at::kFloat && vector_of(u, R), "u must be float32 [rows]");
  auto setting = [&](PyObject* o, const char* name, float& one, const float*& each) {
    if (THPVariable_Check(o)) {
      const at::Tensor& t = *tensor(o, name);
      on(d, &t, name);
      NEED(t.scalar_type() == at::kFloat && vector_of(t, R), c10::str(name, " must be a number or float32 [rows]"));
      each = t.data_ptr<float>();
    } else {
      one = (float)number(o, name);
    }
  };
  setting(p[2], "temperature", a.temperature, a.temperatures);
  setting(p[4], "top_p", a.top_p, a.top_ps);
  setting(p[5], "min_p", a.min_p, a.min_ps);
  if (THPVariable_Check(p[3])) {
    const at::Tensor& t = *tensor(p[3], "top_k");
    on(d, &t, "top_k");
    NEED(t.scalar_type() == at::kInt && vector_of(t, R), "top_k must be a number or int32 [rows]");
    a.top_ks = t.data_ptr<int32_t>();
  } else {
    const double k = number(p[3], "top_k");
    NEED(k == k, "top_k must be a number");
    a.top_k = (int32_t)std::max(-1.0, std::min(k, 2147483647.0));
  }
  auto result = [&](PyObject* o, const char* name, at::ScalarType type) {
    const at::Tensor* t = tensor(o, name);
    if (!t) return fresh({R}, type, d);
    on(d, t, name);
    NEED(t->scalar_type() == type && vector_of(*t, R), "out must be int32 [rows], out_prob float32 [rows]");
    return *t;
  };
  const at::Tensor out = result(p[6], "out", at::kInt), prob = result(p[7], "out_prob", at::kFloat);
  a.logits = x.data_ptr();
  a.u = u.data_ptr<float>();
  a.token_out = out.data_ptr<int32_t>();
  a.prob_out = prob.data_ptr<float>();
  a.rows = (int32_t)R;
  a.vocab = (int32_t)x.size(1);
  a.row_stride = R > 1 ? x.stride(0) : x.size(1);
  OnDevice dev(d);
  const at::Tensor ws = workspace(a, sample_ws_fn, "fa_sample_tokens", d);
  check(sample_fn(&a, dev.stream), "fa_sample_tokens");
  changed(p[6]);
  changed(p[7]);
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(out));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(prob));
  return r;
  END_HANDLE_TH_ERRORS
}

PyObject* bind(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 7);
  void* f[7];
  for (int i = 0; i < 7; ++i) {
    f[i] = PyLong_AsVoidPtr(v[i]);
    if (!f[i]) return nullptr;
  }
  norm_rope_fn = reinterpret_cast<decltype(norm_rope_fn)>(f[0]);
  append_fn = reinterpret_cast<decltype(append_fn)>(f[1]);
  attention_fn = reinterpret_cast<decltype(attention_fn)>(f[2]);
  attention_ws_fn = reinterpret_cast<decltype(attention_ws_fn)>(f[3]);
  sample_fn = reinterpret_cast<decltype(sample_fn)>(f[4]);
  sample_ws_fn = reinterpret_cast<decltype(sample_ws_fn)>(f[5]);
  error_fn = reinterpret_cast<decltype(error_fn)>(f[6]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind),           METHOD(qk_norm_rope),  METHOD(kv_append),
                         METHOD(tree_attention), METHOD(sample_tokens), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "draft_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_draft_ops(void) { return PyModule_Create(&module_def); }
