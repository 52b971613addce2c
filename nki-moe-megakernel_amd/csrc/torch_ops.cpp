// The torch boundary of the paged-cache and sampling operators: checks of arguments,
// outputs and workspaces, and the call of the C ABI, natively.  Of the 5.3 us of host time
// that an append takes, the checks are 0.4, the output tensor 0.7 and the launch the rest; the
// same checks in Python took 12-15, more than a decode batch's kernels.
// The Python entry points (paged.py, sample.py) hold the documentation
// and pass their arguments on.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <initializer_list>
#include <sstream>
#include <string>
#include <utility>

#include "mkd.h"

namespace {

PyObject* g_error = nullptr;   // MkdError

using at::Tensor;
typedef std::pair<const char*, const Tensor*> Named;

std::string shape_of(const Tensor& t) {
  std::ostringstream s;
  s << t.scalar_type() << " " << t.sizes();
  return s.str();
}
Tensor tensor(PyObject* o, const char* name, bool optional = false) {
  if (optional && o == Py_None) return Tensor();
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
// The GPU that all the given tensors are on.
int one_gpu(std::initializer_list<Named> ts) {
  int dev = -1;
  for (const Named& n : ts) {
    if (!n.second->defined()) continue;
    TORCH_CHECK_VALUE(n.second->is_cuda(), "mkd operators take device (HIP) tensors; ", n.first, " is a CPU tensor");
    const int at = n.second->get_device();
    TORCH_CHECK_VALUE(dev < 0 || at == dev, n.first, " is on GPU ", at, ", the tensors before it on GPU ", dev);
    dev = at;
  }
  return dev;
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// Strides of the first n dimensions, 0 where there is nothing to step over.
void strides(const Tensor& t, int n, long long* out) {
  for (int i = 0; i < n; ++i) out[i] = t.size(i) == 1 ? 0 : t.stride(i);
}
bool rows_on(const Tensor& t, int64_t quantum) {   // rows contiguous, on multiples of `quantum` elements
  const int64_t n = t.dim() - 1;
  if (t.stride(n) != 1 && t.size(n) != 1) return false;
  for (int64_t i = 0; i < n; ++i)
    if (t.size(i) != 1 && t.stride(i) % quantum) return false;
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % (quantum * t.element_size()) == 0;
}
// t, or a copy whose rows lie as the kernels' loads need them.
Tensor readable(const Tensor& t, int64_t quantum) {
  return rows_on(t, quantum) ? t : t.clone(at::MemoryFormat::Contiguous);
}
Tensor flat(const Tensor& t, at::ScalarType type, int64_t quantum) {   // 1-D, contiguous, of that type
  Tensor r = t.scalar_type() == type ? t : t.to(type);
  if (r.dim() != 1) r = r.reshape({-1});
  return r.numel() == 0 ? r : readable(r, quantum);
}
void written(const Tensor& t, const char* name, int64_t quantum) {
  bool ok = t.numel() == 0 || rows_on(t, quantum);
  for (int64_t i = 0; ok && i < t.dim() - 1; ++i) ok = t.size(i) <= 1 || t.stride(i) > 0;
  TORCH_CHECK_VALUE(ok, name, " is used in place: its last dimension must be contiguous and its rows distinct, starting on "
                    "multiples of ", quantum, " elements");
}
void index_check(const Tensor& t, int64_t n, const char* name, bool i64) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt || (i64 && t.scalar_type() == at::kLong), name, " must be int32",
                    i64 ? " or int64" : "", ", got ", shape_of(t));
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n, name, " must be [", n, "], got ", shape_of(t));
}
double number(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    TORCH_CHECK_TYPE(false, name, " must be a number, got ", Py_TYPE(o)->tp_name);
  }
  return v;
}
Tensor out_tensor(at::IntArrayRef shape, at::ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(shape, type, like.device(), c10::nullopt));   // (as at::empty, without its dispatch)
}

// Runs call(stream) on the current stream of GPU dev, with that GPU current; raises its error.
template <typename F>
void launch(int dev, const char* what, F call) {
  const int now = c10::hip::current_device();
  if (now != dev) c10::hip::set_device(dev);
  const int rc = call(static_cast<void*>(c10::hip::getCurrentHIPStream(dev).stream()));
  if (now != dev) c10::hip::set_device(now);
  if (rc == MKD_OK) return;
  const std::string msg = std::string(what) + ": " + mkd_last_error();
  TORCH_CHECK_VALUE(rc != MKD_ERR_INVALID && rc != MKD_ERR_NULL && rc != MKD_ERR_WORKSPACE, msg);
  TORCH_CHECK_NOT_IMPLEMENTED(rc != MKD_ERR_UNSUPPORTED, msg);
  PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, msg.c_str());
  throw python_error();
}

struct Caches {
  int num_blocks, block_len, nkv;
  bool fp8;
};
Caches caches(const Tensor& K, const Tensor& V, int64_t d) {
  TORCH_CHECK_VALUE(K.dim() == 4 && K.sizes() == V.sizes(), "K_cache and V_cache must both be [num_blocks, block_len, "
                    "kv_heads, d], got ", shape_of(K), " and ", shape_of(V));
  TORCH_CHECK_VALUE(K.size(3) == d, "the caches hold heads of ", K.size(3), ", the inputs of ", d);
  TORCH_CHECK_NOT_IMPLEMENTED(d == 64 || d == 128, "d must be 64 or 128, got ", d);
  const auto type = K.scalar_type();
  TORCH_CHECK_VALUE(V.scalar_type() == type && (type == at::kBFloat16 || type == at::kFloat8_e4m3fn || type == at::kByte),
                    "the KV caches must both be bfloat16 or float8_e4m3, got ", shape_of(K), " and ", shape_of(V));
  TORCH_CHECK_VALUE(K.size(0) * K.size(1) < (1LL << 31) && K.size(0) > 0 && K.size(1) > 0 && K.size(2) > 0,
                    "a pool of ", K.size(0), " blocks of ", K.size(1), " rows");
  return {(int)K.size(0), (int)K.size(1), (int)K.size(2), type != at::kBFloat16};
}
Tensor scale_of(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(1) == 1 && t.size(0) >= 1, name, " must be (1, 1) or (PMAX, 1), got ", shape_of(t));
  const auto type = t.scalar_type();
  TORCH_CHECK_VALUE(type == at::kFloat || type == at::kHalf || type == at::kBFloat16, name,
                    " dtype must be float32 / float16 / bfloat16, got ", shape_of(t));
  return t;
}

// kv_append_rope(q, k, v, cos, sin, positions, K_cache, V_cache, slots, q_norm, k_norm, eps, k_scale, v_scale, output)
PyObject* kv_append_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 15, "kv_append_rope: ", n, " arguments");
  Tensor q = tensor(a[0], "q"), k = tensor(a[1], "k"), v = tensor(a[2], "v"), cos = tensor(a[3], "cos", true),
         sin = tensor(a[4], "sin", true), pos = tensor(a[5], "positions", true);
  const Tensor K = tensor(a[6], "K_cache"), V = tensor(a[7], "V_cache");
  Tensor slots = tensor(a[8], "slots"), qn = tensor(a[9], "q_norm", true), kn = tensor(a[10], "k_norm", true);
  const double eps = number(a[11], "eps");
  Tensor ks = tensor(a[12], "k_scale", true), vs = tensor(a[13], "v_scale", true), out = tensor(a[14], "output", true);
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(2) == q.size(2),
                    "q must be [T, q_heads, d], k and v [T, kv_heads, d], got ", shape_of(q), ", ", shape_of(k), ", ", shape_of(v));
  const int64_t T = q.size(0), nq = q.size(1), d = q.size(2);
  const Caches c = caches(K, V, d);
  TORCH_CHECK_VALUE(c.nkv == k.size(1), "the caches hold ", c.nkv, " kv heads, k and v ", k.size(1));
  TORCH_CHECK_VALUE(nq >= 1 && T * (nq + 2 * c.nkv) < (1LL << 28), T, " tokens of ", nq, " + 2 x ", c.nkv, " heads");
  const auto type = q.scalar_type();
  TORCH_CHECK_VALUE((type == at::kBFloat16 || type == at::kFloat) && k.scalar_type() == type && v.scalar_type() == type,
                    "q, k and v must all be bfloat16 or float32, got ", shape_of(q), ", ", shape_of(k), ", ", shape_of(v));
  TORCH_CHECK_VALUE(ks.defined() == vs.defined() && ks.defined() == c.fp8,
                    "float8_e4m3 caches need k_scale and v_scale, bfloat16 caches neither");
  TORCH_CHECK_VALUE(cos.defined() == sin.defined() && cos.defined() == pos.defined(),
                    "cos, sin and positions must be given together");
  int64_t rot = 0;
  if (cos.defined()) {
    TORCH_CHECK_VALUE(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.size(0) >= 1 && cos.size(0) < (1LL << 31),
                      "cos and sin must be [rows, r / 2], got ", shape_of(cos), " and ", shape_of(sin));
    rot = 2 * cos.size(1);
    TORCH_CHECK_VALUE(rot % 8 == 0 && rot >= 8 && rot <= d, "the rotated part must be a multiple of 8 from 8 to d = ", d,
                      ", got ", rot);
    for (const Tensor* t : {&cos, &sin})
      TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat || t->scalar_type() == at::kBFloat16,
                        "cos and sin must be float32 or bfloat16, got ", shape_of(*t));
    index_check(pos, T, "positions", true);
  }
  index_check(slots, T, "slots", true);
  for (const Named& x : {Named{"q_norm", &qn}, Named{"k_norm", &kn}})
    TORCH_CHECK_VALUE(!x.second->defined() || x.second->numel() == d, x.first, " must have ", d, " elements, got ",
                      shape_of(*x.second));
  if (c.fp8) {
    scale_of(ks, "k_scale");
    scale_of(vs, "v_scale");
  }
  if (out.defined())
    TORCH_CHECK_VALUE(out.sizes() == q.sizes() && out.scalar_type() == at::kBFloat16, "output must be bfloat16 ", q.sizes(),
                      ", got ", shape_of(out));
  const int dev = one_gpu({{"q", &q}, {"k", &k}, {"v", &v}, {"cos", &cos}, {"sin", &sin}, {"positions", &pos}, {"K_cache", &K},
                           {"V_cache", &V}, {"slots", &slots}, {"q_norm", &qn}, {"k_norm", &kn}, {"k_scale", &ks},
                           {"v_scale", &vs}, {"output", &out}});
  written(K, "K_cache", 4);
  written(V, "V_cache", 4);
  TORCH_CHECK_VALUE(T == 0 || ptr(K) != ptr(V), "K_cache and V_cache are used in place and must not be one tensor");
  if (out.defined()) written(out, "output", 4);
  else out = out_tensor(q.sizes(), at::kBFloat16, q);
  if (T > 0) {
    q = readable(q, 4);
    k = readable(k, 4);
    v = readable(v, 4);
    slots = slots.contiguous();
    if (rot) {
      cos = flat(cos.contiguous(), at::kFloat, 4);
      sin = flat(sin.contiguous(), at::kFloat, 4);
      pos = pos.contiguous();
    }
    if (qn.defined()) qn = flat(qn, at::kBFloat16, 4);
    if (kn.defined()) kn = flat(kn, at::kBFloat16, 4);
    if (c.fp8) {
      ks = ks.to(at::kFloat);
      vs = vs.to(at::kFloat);
    }
    mkd_kv_append_args g{};
    g.q = ptr(q);
    g.k = ptr(k);
    g.v = ptr(v);
    g.x_dtype = type == at::kFloat ? MKD_DT_F32 : MKD_DT_BF16;
    strides(q, 2, g.q_stride);
    strides(k, 2, g.k_stride);
    strides(v, 2, g.v_stride);
    g.q_out = ptr(out);
    strides(out, 2, g.q_out_stride);
    g.q_norm = ptr(qn);
    g.k_norm = ptr(kn);
    g.eps = (float)eps;
    g.cos = static_cast<const float*>(ptr(cos));
    g.sin = static_cast<const float*>(ptr(sin));
    g.table_rows = rot ? (int)(2 * cos.numel() / rot) : 0;
    g.rot = (int)rot;
    g.positions = ptr(pos);
    g.positions_i64 = rot && pos.scalar_type() == at::kLong;
    g.k_cache = ptr(K);
    g.v_cache = ptr(V);
    strides(K, 3, g.k_cache_stride);
    strides(V, 3, g.v_cache_stride);
    g.num_blocks = c.num_blocks;
    g.block_len = c.block_len;
    g.kv_format = c.fp8 ? MKD_KV_FP8 : 0;
    g.k_scale = static_cast<const float*>(ptr(ks));
    g.v_scale = static_cast<const float*>(ptr(vs));
    g.slots = ptr(slots);
    g.slots_i64 = slots.scalar_type() == at::kLong;
    g.T = (int)T;
    g.nq = (int)nq;
    g.nkv = c.nkv;
    g.d = (int)d;
    launch(dev, "kv_append_rope", [&](void* s) { return mkd_kv_append_rope(&g, s); });
  }
  PyObject* first = a[14] != Py_None ? (Py_INCREF(a[14]), a[14]) : THPVariable_Wrap(out);
  PyObject* r = PyTuple_Pack(3, first, a[6], a[7]);
  Py_DECREF(first);
  return r;
  END_HANDLE_TH_ERRORS
}

// attention_shared_prefix(q, K_cache, V_cache, prefix_tables, prefix_lens, prefix_starts, tables, lens, softmax_scale,
//                         sink, output)
PyObject* attention_shared_prefix(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 11, "attention_shared_prefix: ", n, " arguments");
  Tensor q = tensor(a[0], "q");
  const Tensor K = tensor(a[1], "K_cache"), V = tensor(a[2], "V_cache");
  Tensor pt = tensor(a[3], "prefix_tables", true), pl = tensor(a[4], "prefix_lens", true),
         ps = tensor(a[5], "prefix_starts", true), ot = tensor(a[6], "tables"), ol = tensor(a[7], "lens");
  Tensor sink = tensor(a[9], "sink", true), out = tensor(a[10], "output", true);
  TORCH_CHECK_VALUE((q.dim() == 3 || q.dim() == 4) && q.scalar_type() == at::kBFloat16,
                    "q must be bfloat16 [B, (S_tkg,) q_heads, d], got ", shape_of(q));
  const bool wide = q.dim() == 4;
  const int64_t B = q.size(0), S = wide ? q.size(1) : 1, nq = q.size(-2), d = q.size(-1);
  TORCH_CHECK_VALUE(S >= 1 && S <= 8, "S_tkg must be in [1, 8], got ", S);
  const Caches c = caches(K, V, d);
  TORCH_CHECK_VALUE(nq >= 1 && nq % c.nkv == 0 && nq <= 4096, nq, " query heads do not share ", c.nkv, " kv heads evenly");
  TORCH_CHECK_VALUE(B <= 65535, "B must be at most 65535, got ", B);
  auto table_check = [&](const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.dim() == 2 && t.scalar_type() == at::kInt && t.size(1) * c.block_len < (1LL << 30), name,
                      " must be int32 [", name[0] == 't' ? "B" : "G", ", blocks], got ", shape_of(t));
  };
  table_check(ot, "tables");
  TORCH_CHECK_VALUE(ot.size(0) == B, "tables must be int32 [B=", B, ", blocks], got ", shape_of(ot));
  index_check(ol, B, "lens", false);
  TORCH_CHECK_VALUE(pt.defined() == pl.defined() && pt.defined() == ps.defined(),
                    "prefix_tables, prefix_lens and prefix_starts must be given together");
  int64_t G = 0;
  if (pt.defined()) {
    table_check(pt, "prefix_tables");
    G = pt.size(0);
    TORCH_CHECK_VALUE(G <= 65535, "at most 65535 groups, got ", G);
    index_check(pl, G, "prefix_lens", false);
    index_check(ps, G + 1, "prefix_starts", false);
  }
  TORCH_CHECK_VALUE(!sink.defined() || sink.numel() == nq, "sink must have ", nq, " elements, got ",
                    sink.defined() ? shape_of(sink) : "");
  if (out.defined())
    TORCH_CHECK_VALUE(out.sizes() == q.sizes() && out.scalar_type() == at::kBFloat16, "output must be bfloat16 ", q.sizes(),
                      ", got ", shape_of(out));
  const double scale = a[8] == Py_None ? 1.0 / std::sqrt((double)d) : number(a[8], "softmax_scale");
  const int dev = one_gpu({{"q", &q}, {"K_cache", &K}, {"V_cache", &V}, {"prefix_tables", &pt}, {"prefix_lens", &pl},
                           {"prefix_starts", &ps}, {"tables", &ot}, {"lens", &ol}, {"sink", &sink}, {"output", &out}});
  const int64_t row = c.fp8 ? 16 : 8;             // 16 bytes
  written(K, "K_cache", row);
  written(V, "V_cache", row);
  if (out.defined()) written(out, "output", 2);
  else out = out_tensor(q.sizes(), at::kBFloat16, q);
  if (B > 0) {
    q = readable(q, 8);
    ot = ot.contiguous();
    ol = ol.contiguous();
    if (G) {
      pt = pt.contiguous();
      pl = pl.contiguous();
      ps = ps.contiguous();
    }
    if (sink.defined()) sink = flat(sink, at::kFloat, 1);
    mkd_shared_prefix_args g{};
    long long st[4];
    auto rows = [&](const Tensor& t, long long* to) {
      strides(t, (int)t.dim() - 1, st);
      to[0] = st[0];
      to[1] = wide ? st[1] : 0;
      to[2] = st[t.dim() - 2];
    };
    g.q = ptr(q);
    rows(q, g.q_stride);
    g.out = ptr(out);
    rows(out, g.out_stride);
    g.k_cache = ptr(K);
    g.v_cache = ptr(V);
    strides(K, 3, g.k_cache_stride);
    strides(V, 3, g.v_cache_stride);
    g.num_blocks = c.num_blocks;
    g.block_len = c.block_len;
    g.kv_format = c.fp8 ? MKD_KV_FP8 : 0;
    g.prefix_tables = static_cast<const int*>(ptr(pt));
    g.prefix_lens = static_cast<const int*>(ptr(pl));
    g.prefix_starts = static_cast<const int*>(ptr(ps));
    g.tables = static_cast<const int*>(ptr(ot));
    g.lens = static_cast<const int*>(ptr(ol));
    g.G = (int)G;
    g.prefix_blocks = G ? (int)pt.size(1) : 0;
    g.own_blocks = (int)ot.size(1);
    g.softmax_scale = (float)scale;
    g.sink = static_cast<const float*>(ptr(sink));
    g.B = (int)B;
    g.s_tkg = (int)S;
    g.nq = (int)nq;
    g.nkv = c.nkv;
    g.d = (int)d;
    const size_t need = mkd_shared_prefix_workspace_bytes(&g);
    const Tensor ws = need ? out_tensor({(int64_t)need}, at::kByte, q) : Tensor();
    launch(dev, "attention_shared_prefix", [&](void* s) { return mkd_attention_shared_prefix(&g, ptr(ws), need, s); });
  }
  if (a[10] != Py_None) return Py_INCREF(a[10]), a[10];
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// A setting: its value for all rows, or a [B] tensor of the kernels' type.
Tensor setting(PyObject* o, const char* name, int64_t B, double lo, double hi, at::ScalarType type, double* value) {
  if (!THPVariable_Check(o)) {
    *value = number(o, name);
    TORCH_CHECK_VALUE(*value >= lo && *value <= hi, name, " must be in [", lo, ", ", hi, "], got ", *value);   // (a NaN too)
    TORCH_CHECK_VALUE(type != at::kInt || *value == std::floor(*value), name, " must be a whole number, got ", *value);
    return Tensor();
  }
  const Tensor t = THPVariable_Unpack(o);
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == B, name, " must be a number or [B=", B, "], got ", shape_of(t));
  const bool whole = t.scalar_type() == at::kInt || t.scalar_type() == at::kLong;
  TORCH_CHECK_VALUE(type == at::kInt ? whole : t.is_floating_point(), name, " must be ",
                    type == at::kInt ? "int32 or int64" : "floating point", ", got ", shape_of(t));
  *value = 0;
  return t;
}
Tensor row_values(const Tensor& t, at::ScalarType type) {
  if (!t.defined()) return t;
  if (t.scalar_type() == type) return t.contiguous();
  return (type == at::kInt ? t.clamp(0, 0x7fffffff) : t).to(type).contiguous();
}

// sample_tokens(logits, uniforms, temperature, top_k, top_p, min_p, output)
PyObject* sample_tokens(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 7, "sample_tokens: ", n, " arguments");
  Tensor x = tensor(a[0], "logits"), u = tensor(a[1], "uniforms"), out = tensor(a[6], "output", true);
  const auto type = x.scalar_type();
  TORCH_CHECK_VALUE(x.dim() == 2 && (type == at::kBFloat16 || type == at::kFloat),
                    "logits must be bfloat16 or float32 [B, V], got ", shape_of(x));
  const int64_t B = x.size(0), V = x.size(1);
  TORCH_CHECK_VALUE(V >= 1 && V <= (1 << 20) && B <= 65535, "logits must be [B <= 65535, 1 <= V <= 2^20], got ", x.sizes());
  TORCH_CHECK_VALUE(u.scalar_type() == at::kFloat && u.dim() == 1 && u.size(0) == B, "uniforms must be float32 [B=", B,
                    "], got ", shape_of(u));
  double temp, top_k, top_p, min_p;
  Tensor t = setting(a[2], "temperature", B, 0.0, 3.4e38, at::kFloat, &temp);
  Tensor k = setting(a[3], "top_k", B, 0.0, INFINITY, at::kInt, &top_k);
  Tensor p = setting(a[4], "top_p", B, 0.0, 1.0, at::kFloat, &top_p);
  Tensor m = setting(a[5], "min_p", B, 0.0, 1.0, at::kFloat, &min_p);
  if (out.defined())
    TORCH_CHECK_VALUE(out.scalar_type() == at::kInt && out.dim() == 1 && out.size(0) == B && out.is_contiguous(),
                      "output must be a contiguous int32 [", B, "] tensor, got ", shape_of(out));
  const int dev = one_gpu({{"logits", &x}, {"uniforms", &u}, {"temperature", &t}, {"top_k", &k}, {"top_p", &p}, {"min_p", &m},
                           {"output", &out}});
  if (!out.defined()) out = out_tensor({B}, at::kInt, x);
  const Tensor lp = out_tensor({B}, at::kFloat, x);
  if (B > 0) {
    if (V > 1 && x.stride(1) != 1) x = x.contiguous();
    u = u.contiguous();
    t = row_values(t, at::kFloat);
    k = row_values(k, at::kInt);
    p = row_values(p, at::kFloat);
    m = row_values(m, at::kFloat);
    mkd_sample_args g{};
    g.logits = ptr(x);
    g.logits_dtype = type == at::kFloat ? MKD_DT_F32 : MKD_DT_BF16;
    g.row_stride = B > 1 ? x.stride(0) : 0;
    g.uniforms = static_cast<const float*>(ptr(u));
    g.temperature = (float)temp;
    g.top_p = (float)top_p;
    g.min_p = (float)min_p;
    g.top_k = top_k < 2147483647.0 ? (int)top_k : 2147483647;
    g.temperature_rows = static_cast<const float*>(ptr(t));
    g.top_p_rows = static_cast<const float*>(ptr(p));
    g.min_p_rows = static_cast<const float*>(ptr(m));
    g.top_k_rows = static_cast<const int*>(ptr(k));
    g.tokens = static_cast<int*>(ptr(out));
    g.logprobs = static_cast<float*>(ptr(lp));
    g.B = (int)B;
    g.V = (int)V;
    const size_t need = mkd_sample_workspace_bytes((int)B, (int)V);
    const Tensor ws = out_tensor({(int64_t)need}, at::kByte, x);
    launch(dev, "sample_tokens", [&](void* s) { return mkd_sample_tokens(&g, ws.data_ptr(), need, s); });
  }
  PyObject* first = a[6] != Py_None ? (Py_INCREF(a[6]), a[6]) : THPVariable_Wrap(out);
  PyObject* second = THPVariable_Wrap(lp);
  PyObject* r = PyTuple_Pack(2, first, second);
  Py_DECREF(first);
  Py_DECREF(second);
  return r;
  END_HANDLE_TH_ERRORS
}

PyObject* set_error(PyObject*, PyObject* cls) {
  Py_XINCREF(cls);
  g_error = cls;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"kv_append_rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(kv_append_rope)), METH_FASTCALL, nullptr},
    {"attention_shared_prefix", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(attention_shared_prefix)), METH_FASTCALL,
     nullptr},
    {"sample_tokens", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(sample_tokens)), METH_FASTCALL, nullptr},
    {"set_error", set_error, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mkd_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mkd_torch() { return PyModule_Create(&module); }
