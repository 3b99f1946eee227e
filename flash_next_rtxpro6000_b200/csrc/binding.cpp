// Python binding of the verify-step operators: argument checks, outputs and the call into the C ABI
// (include/fnx_gemv.h) in one native function per operator.  Through ctypes a call of rotary_append
// took 26 us on the host against 2 us on the GPU; the arguments' metadata is read here at a
// fraction of that.  Everything else of the package goes through ctypes.
//
// Functions take all arguments by place (the Python modules hold the signatures and the defaults)
// and raise ValueError, NotImplementedError or RuntimeError as the ctypes calls do.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdarg.h>

#include <stdexcept>
#include <string>

#include "../../include/fnx_gemv.h"

namespace {

// Other Python threads run while outputs are allocated and kernels launched: either may wait, for memory or
// for room in the launch queue.  What is inside reads no Python object.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

struct Refused {
  PyObject* type;
  std::string what;
};

[[noreturn]] void refuse(PyObject* type, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
void refuse(PyObject* type, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  throw Refused{type, buf};
}

void check(int rc, const char* what) {
  if (rc == FNX_OK) return;
  refuse(rc == FNX_EINVAL ? PyExc_ValueError : rc == FNX_EUNSUPPORTED ? PyExc_NotImplementedError : PyExc_RuntimeError,
         "%s: %s", what, fnx_last_error());
}

std::string sizes(const at::Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s must be a tensor", name);
  return THPVariable_Unpack(o);
}
bool given(PyObject* o) { return o != Py_None; }

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw std::bad_exception();
  return v;
}
int small(int64_t v, const char* name) {
  if (v < INT32_MIN || v > INT32_MAX) refuse(PyExc_NotImplementedError, "%s = %lld is too large", name, (long long)v);
  return (int)v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw std::bad_exception();
  return v != 0;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw std::bad_exception();
  return v;
}

// The type code of 16-bit activations.
int type16(const at::Tensor& t, const char* what) {
  if (t.scalar_type() == at::kBFloat16) return FNX_T_BF16;
  if (t.scalar_type() == at::kHalf) return FNX_T_F16;
  refuse(PyExc_NotImplementedError, "%s: bf16 or fp16, got %s", what, c10::toString(t.scalar_type()));
}

void on_gpu(const at::Tensor& t, const char* what) {
  if (!t.is_cuda()) refuse(PyExc_ValueError, "%s needs CUDA tensors", what);
}

// The current stream of the tensor's device, which has to be the current device.
cudaStream_t stream_of(const at::Tensor& t) {
  const auto now = c10::cuda::current_device();
  if (t.get_device() != now)
    refuse(PyExc_ValueError, "tensor on cuda:%d but the current device is cuda:%d", (int)t.get_device(), (int)now);
  return c10::cuda::getCurrentCUDAStream(now).stream();
}

// [tokens, heads, dim] of like's type and device, the elements of a head contiguous.
void heads(const at::Tensor& t, const char* name, int64_t tokens, int64_t dim, const at::Tensor& like) {
  if (t.dim() != 3 || t.size(0) != tokens || t.size(2) != dim)
    refuse(PyExc_ValueError, "%s must be [%lld, heads, %lld], got %s", name, (long long)tokens, (long long)dim,
           sizes(t).c_str());
  if (t.scalar_type() != like.scalar_type() || t.device() != like.device())
    refuse(PyExc_ValueError, "%s must be %s on %s, got %s on %s", name, c10::toString(like.scalar_type()),
           like.device().str().c_str(), c10::toString(t.scalar_type()), t.device().str().c_str());
  if (t.stride(2) != 1 && dim > 1)
    refuse(PyExc_ValueError, "the elements of a head of %s must be contiguous", name);
}

void index(const at::Tensor& t, const char* name, int64_t count, at::ScalarType type, const at::Tensor& like) {
  if (t.scalar_type() != type || t.device() != like.device() || t.dim() != 1 || t.size(0) != count ||
      !t.is_contiguous())
    refuse(PyExc_ValueError, "%s must be a contiguous %s [%lld] tensor on %s, got %s %s on %s", name,
           c10::toString(type), (long long)count, like.device().str().c_str(), c10::toString(t.scalar_type()),
           sizes(t).c_str(), t.device().str().c_str());
}

// A pair of paged caches [pages, page_size, kv_heads, dim] of q's type.
void caches(const at::Tensor& k, const at::Tensor& v, const at::Tensor& q) {
  if (k.dim() != 4 || v.sizes() != k.sizes())
    refuse(PyExc_ValueError, "k_cache and v_cache must be [pages, page_size, kv_heads, dim] of one shape; got %s and %s",
           sizes(k).c_str(), sizes(v).c_str());
  if (k.size(3) != q.size(2) || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() ||
      k.device() != q.device() || v.device() != q.device())
    refuse(PyExc_ValueError, "caches must be [pages, page_size, kv_heads, %lld] %s tensors on %s",
           (long long)q.size(2), c10::toString(q.scalar_type()), q.device().str().c_str());
  if ((k.stride(3) != 1 || v.stride(3) != 1) && k.size(3) > 1)
    refuse(PyExc_ValueError, "the elements of a cached head must be contiguous");
}

// The caller's destination, with as many heads, or null where a new one is wanted.
const at::Tensor* destination(PyObject* out, const at::Tensor& q) {
  if (!given(out)) return nullptr;
  const at::Tensor& t = tensor(out, "out");
  heads(t, "out", q.size(0), q.size(2), q);
  if (t.size(1) != q.size(1)) refuse(PyExc_ValueError, "out must have q's %lld heads", (long long)q.size(1));
  return &t;
}
const at::Tensor* lse_destination(PyObject* out, const at::Tensor& q) {
  if (!given(out)) return nullptr;
  const at::Tensor& lse = tensor(out, "lse");
  if (lse.dim() != 2 || lse.size(0) != q.size(0) || lse.size(1) != q.size(1) || lse.scalar_type() != at::kFloat ||
      lse.device() != q.device() || !lse.is_contiguous())
    refuse(PyExc_ValueError, "lse must be a contiguous fp32 [%lld, %lld] tensor on %s", (long long)q.size(0),
           (long long)q.size(1), q.device().str().c_str());
  return &lse;
}
at::Tensor like(const at::Tensor& q) { return at::empty({q.size(0), q.size(1), q.size(2)}, q.options()); }

// A pair of 8-bit paged caches [pages, page_size, kv_heads, dim] and their scales; the scales' block.
int64_t caches8(const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks, const at::Tensor& vs,
                const at::Tensor& like, int64_t lead) {
  const int64_t n = lead + 4;
  if (k.dim() != n || v.sizes() != k.sizes())
    refuse(PyExc_ValueError, "k_cache and v_cache must be [%spages, page_size, kv_heads, dim] of one shape; got %s and %s",
           lead ? "layers, " : "", sizes(k).c_str(), sizes(v).c_str());
  if (k.scalar_type() != at::kFloat8_e4m3fn || v.scalar_type() != at::kFloat8_e4m3fn || k.device() != like.device() ||
      v.device() != like.device())
    refuse(PyExc_ValueError, "caches must be float8_e4m3fn tensors on %s", like.device().str().c_str());
  if ((k.stride(n - 1) != 1 || v.stride(n - 1) != 1) && k.size(n - 1) > 1)
    refuse(PyExc_ValueError, "the elements of a cached head must be contiguous");
  const int64_t page = k.size(lead + 1), per = ks.dim() == lead + 3 ? ks.size(lead + 1) : 0;
  if (ks.dim() != lead + 3 || vs.sizes() != ks.sizes() || ks.size(0) != k.size(0) || ks.size(lead) != k.size(lead) ||
      ks.size(lead + 2) != k.size(lead + 2) || per < 1 || page % per)
    refuse(PyExc_ValueError, "k_scale and v_scale must be [%spages, page_size / block, kv_heads]; got %s and %s for caches %s",
           lead ? "layers, " : "", sizes(ks).c_str(), sizes(vs).c_str(), sizes(k).c_str());
  if (ks.scalar_type() != at::kFloat || vs.scalar_type() != at::kFloat || ks.device() != like.device() ||
      vs.device() != like.device())
    refuse(PyExc_ValueError, "scales must be fp32 tensors on %s", like.device().str().c_str());
  return page / per;
}

// A result: the caller's own object, or a new tensor's.
PyObject* result(PyObject* own, at::Tensor&& made) {
  if (!given(own)) return THPVariable_Wrap(std::move(made));
  Py_INCREF(own);
  return own;
}

void page_table(const at::Tensor& t, int64_t batch, const at::Tensor& like) {
  if (t.dim() != 2 || t.size(0) != batch || t.scalar_type() != at::kInt || t.device() != like.device() ||
      (t.stride(1) != 1 && t.size(1) > 1))
    refuse(PyExc_ValueError, "page_table must be a row-contiguous int32 [%lld, pages] tensor on %s", (long long)batch,
           like.device().str().c_str());
}

template <typename T> T* ptr(const at::Tensor& t) { return static_cast<T*>(t.data_ptr()); }

// q, k, v, positions, slots, table, k_cache, v_cache, interleaved, out, error_flag, pdl
PyObject* rotary_append(PyObject* const* a) {
  const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &v = tensor(a[2], "v"),
                   &pos = tensor(a[3], "positions"), &slots = tensor(a[4], "slots"), &table = tensor(a[5], "table"),
                   &kc = tensor(a[6], "k_cache"), &vc = tensor(a[7], "v_cache");
  if (q.dim() != 3) refuse(PyExc_ValueError, "q must be [tokens, heads, dim], got %s", sizes(q).c_str());
  const int type = type16(q, "rotary_append");
  on_gpu(q, "rotary_append");
  const int64_t T = q.size(0), D = q.size(2), Hk = k.dim() == 3 ? k.size(1) : 0;
  heads(q, "q", T, D, q);
  heads(k, "k", T, D, q);
  heads(v, "v", T, D, q);
  if (v.size(1) != Hk)
    refuse(PyExc_ValueError, "k and v must have one number of heads, got %lld and %lld", (long long)Hk,
           (long long)v.size(1));
  index(pos, "positions", T, at::kLong, q);
  index(slots, "slots", T, at::kLong, q);
  if (table.dim() != 2 || table.scalar_type() != at::kFloat || table.device() != q.device() ||
      (table.stride(1) != 1 && table.size(1) > 1))
    refuse(PyExc_ValueError, "table must be a row-contiguous fp32 [positions, rotated] tensor on %s",
           q.device().str().c_str());
  const int64_t R = table.size(1);
  if (R > D || R % 2)
    refuse(PyExc_ValueError, "the table's %lld columns must be even and at most dim = %lld", (long long)R, (long long)D);
  caches(kc, vc, q);
  if (kc.size(2) != Hk)
    refuse(PyExc_ValueError, "caches must have k's %lld heads, got %lld", (long long)Hk, (long long)kc.size(2));
  const cudaStream_t stream = stream_of(q);
  const at::Tensor* to = destination(a[9], q);
  const bool interleaved = truth(a[8]);
  int* flag = reinterpret_cast<int*>(integer(a[10]));
  const int pdl = (int)integer(a[11]);
  at::Tensor made;
  {
    Unlocked others;
    if (!to) made = like(q);
    const at::Tensor& out = to ? *to : made;
    check(fnx_rotary_append(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
                            v.data_ptr(), v.stride(0), v.stride(1), out.data_ptr(), out.stride(0), out.stride(1),
                            ptr<int64_t>(pos), ptr<int64_t>(slots), ptr<float>(table), table.stride(0), table.size(0),
                            kc.data_ptr(), kc.strides().data(), vc.data_ptr(), vc.strides().data(), kc.size(0),
                            small(kc.size(1), "page_size"), small(T, "tokens"), small(q.size(1), "q_heads"),
                            small(Hk, "kv_heads"), small(D, "dim"), (int)R, interleaved, type, flag, pdl, stream),
          "rotary_append");
  }
  return result(a[9], std::move(made));
}

// parents, node_offsets, context_lens, page_table, page_size, num_pages, error_flag, pdl
PyObject* tree_layout(PyObject* const* a) {
  const at::Tensor &parents = tensor(a[0], "parents"), &off = tensor(a[1], "node_offsets"),
                   &ctx = tensor(a[2], "context_lens"), &table = tensor(a[3], "page_table");
  on_gpu(parents, "tree_layout");
  const int64_t N = parents.numel(), B = ctx.numel();
  index(parents, "parents", N, at::kInt, parents);
  index(off, "node_offsets", B + 1, at::kInt, parents);
  index(ctx, "context_lens", B, at::kInt, parents);
  page_table(table, B, parents);
  const cudaStream_t stream = stream_of(parents);
  const int64_t page_size = integer(a[4]), num_pages = integer(a[5]);
  int* flag = reinterpret_cast<int*>(integer(a[6]));
  const int pdl = (int)integer(a[7]);
  at::Tensor out;
  {
    Unlocked others;
    out = at::empty({3, N}, parents.options().dtype(at::kLong));
    int64_t* to = ptr<int64_t>(out);
    check(fnx_tree_layout(ptr<int32_t>(parents), ptr<int32_t>(off), ptr<int32_t>(ctx), ptr<int32_t>(table),
                          table.stride(0), small(table.size(1), "pages"), num_pages, small(page_size, "page_size"),
                          small(B, "batch"), small(N, "nodes"), reinterpret_cast<uint64_t*>(to), to + N, to + 2 * N,
                          flag, pdl, stream),
          "tree_layout");
  }
  PyObject* t = PyTuple_New(3);
  for (int i = 0; i < 3; ++i) PyTuple_SET_ITEM(t, i, THPVariable_Wrap(out.select(0, i)));
  return t;
}

// q, k_cache, v_cache, page_table, context_lens, node_offsets, tree_mask, max_nodes, max_context, scale, out, lse,
// partials, error_flag, pdl
PyObject* tree_attention(PyObject* const* a) {
  const at::Tensor &q = tensor(a[0], "q"), &kc = tensor(a[1], "k_cache"), &vc = tensor(a[2], "v_cache"),
                   &table = tensor(a[3], "page_table"), &ctx = tensor(a[4], "context_lens"),
                   &off = tensor(a[5], "node_offsets");
  if (q.dim() != 3) refuse(PyExc_ValueError, "q must be [nodes, heads, dim], got %s", sizes(q).c_str());
  const int type = type16(q, "tree_attention");
  on_gpu(q, "tree_attention");
  const int64_t N = q.size(0), Hq = q.size(1), D = q.size(2), B = ctx.numel();
  heads(q, "q", N, D, q);
  caches(kc, vc, q);
  const int64_t Hk = kc.size(2);
  if (Hk < 1 || Hq % Hk)
    refuse(PyExc_ValueError, "%lld query heads must be a multiple of %lld kv heads", (long long)Hq, (long long)Hk);
  index(ctx, "context_lens", B, at::kInt, q);
  index(off, "node_offsets", B + 1, at::kInt, q);
  page_table(table, B, q);
  const uint64_t* mask = nullptr;
  if (given(a[6])) {
    const at::Tensor& m = tensor(a[6], "tree_mask");
    index(m, "tree_mask", N, at::kLong, q);
    mask = ptr<uint64_t>(m);
  }
  const cudaStream_t stream = stream_of(q);
  const at::Tensor *to = destination(a[10], q), *to_lse = lse_destination(a[11], q);
  const int max_nodes = small(integer(a[7]), "max_nodes");
  const int64_t max_context = given(a[8]) ? integer(a[8]) : table.size(1) * kc.size(1);
  const float scale = given(a[9]) ? (float)number(a[9]) : 1.0f / std::sqrt((float)D);
  float* partials = reinterpret_cast<float*>(integer(a[12]));
  int* flag = reinterpret_cast<int*>(integer(a[13]));
  const int pdl = (int)integer(a[14]);
  at::Tensor made, made_lse;
  {
    Unlocked others;
    if (!to) made = like(q);
    if (!to_lse) made_lse = at::empty({N, Hq}, q.options().dtype(at::kFloat));
    const at::Tensor &out = to ? *to : made, &lse = to_lse ? *to_lse : made_lse;
    check(fnx_tree_attention(q.data_ptr(), q.stride(0), q.stride(1), kc.data_ptr(), kc.strides().data(), vc.data_ptr(),
                             vc.strides().data(), kc.size(0), small(kc.size(1), "page_size"), ptr<int32_t>(table),
                             table.stride(0), small(table.size(1), "pages"), ptr<int32_t>(ctx), ptr<int32_t>(off), mask,
                             out.data_ptr(), out.stride(0), out.stride(1), ptr<float>(lse), small(B, "batch"),
                             small(N, "nodes"), small(Hq, "q_heads"), small(Hk, "kv_heads"), small(D, "dim"), max_nodes,
                             max_context, scale, type, partials, flag, pdl, stream),
          "tree_attention");
  }
  PyObject* t = PyTuple_New(2);
  PyTuple_SET_ITEM(t, 0, result(a[10], std::move(made)));
  PyTuple_SET_ITEM(t, 1, result(a[11], std::move(made_lse)));
  return t;
}

// logits, uniforms, temperature, top_k, top_p, min_p, pdl
PyObject* sample_tokens(PyObject* const* a) {
  const at::Tensor &x = tensor(a[0], "logits"), &u = tensor(a[1], "uniforms");
  if (x.dim() != 2 || (x.stride(1) != 1 && x.size(1) > 1))
    refuse(PyExc_ValueError, "logits must be row-contiguous [rows, vocab], got %s", sizes(x).c_str());
  const at::ScalarType st = x.scalar_type();
  if (st != at::kFloat && st != at::kBFloat16 && st != at::kHalf)
    refuse(PyExc_NotImplementedError, "sample_tokens: fp32, bf16 or fp16 logits, got %s", c10::toString(st));
  on_gpu(x, "sample_tokens");
  const int64_t M = x.size(0), V = x.size(1);
  index(u, "uniforms", M, at::kFloat, x);
  const char* names[4] = {"temperature", "top_k", "top_p", "min_p"};
  const void* p[4];
  for (int i = 0; i < 4; ++i) {
    p[i] = nullptr;
    if (!given(a[2 + i])) continue;
    const at::Tensor& t = tensor(a[2 + i], names[i]);
    index(t, names[i], M, i == 1 ? at::kInt : at::kFloat, x);
    p[i] = t.data_ptr();
  }
  const cudaStream_t stream = stream_of(x);
  const int pdl = (int)integer(a[6]);
  at::Tensor tokens, probs;
  {
    Unlocked others;
    tokens = at::empty({M}, x.options().dtype(at::kLong));
    probs = at::empty({M}, x.options().dtype(at::kFloat));
    check(fnx_sample(x.data_ptr(), M > 1 ? x.stride(0) : std::max(x.stride(0), V),
                     st == at::kFloat ? FNX_T_F32 : st == at::kHalf ? FNX_T_F16 : FNX_T_BF16, small(M, "rows"),
                     small(V, "vocab"), ptr<float>(u), static_cast<const float*>(p[0]),
                     static_cast<const int32_t*>(p[1]), static_cast<const float*>(p[2]), static_cast<const float*>(p[3]),
                     ptr<int64_t>(tokens), ptr<float>(probs), pdl, stream),
          "sample_tokens");
  }
  PyObject* t = PyTuple_New(2);
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(tokens)));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(probs)));
  return t;
}

// logits, temperature, top_k, top_p, min_p, out, pdl
PyObject* token_probs(PyObject* const* a) {
  const at::Tensor& x = tensor(a[0], "logits");
  if (x.dim() != 2 || (x.stride(1) != 1 && x.size(1) > 1))
    refuse(PyExc_ValueError, "logits must be row-contiguous [rows, vocab], got %s", sizes(x).c_str());
  const at::ScalarType st = x.scalar_type();
  if (st != at::kFloat && st != at::kBFloat16 && st != at::kHalf)
    refuse(PyExc_NotImplementedError, "token_probs: fp32, bf16 or fp16 logits, got %s", c10::toString(st));
  on_gpu(x, "token_probs");
  const int64_t M = x.size(0), V = x.size(1);
  const char* names[4] = {"temperature", "top_k", "top_p", "min_p"};
  const void* p[4];
  for (int i = 0; i < 4; ++i) {
    p[i] = nullptr;
    if (!given(a[1 + i])) continue;
    const at::Tensor& t = tensor(a[1 + i], names[i]);
    index(t, names[i], M, i == 1 ? at::kInt : at::kFloat, x);
    p[i] = t.data_ptr();
  }
  const at::Tensor* to = nullptr;
  if (given(a[5])) {
    to = &tensor(a[5], "out");
    if (to->dim() != 2 || to->size(0) != M || to->size(1) != V || to->scalar_type() != at::kFloat ||
        to->device() != x.device() || (to->stride(1) != 1 && V > 1) || (to->stride(0) < V && M > 1))
      refuse(PyExc_ValueError, "out must be a row-contiguous fp32 [%lld, %lld] tensor on %s", (long long)M, (long long)V,
             x.device().str().c_str());
    // a CTA reads its logits again while others write
    const char *l0 = static_cast<const char*>(x.data_ptr()), *o0 = static_cast<const char*>(to->data_ptr());
    const int64_t ln = M ? ((M - 1) * x.stride(0) + V) * x.element_size() : 0, on = M ? ((M - 1) * to->stride(0) + V) * 4 : 0;
    if (l0 < o0 + on && o0 < l0 + ln) refuse(PyExc_ValueError, "out must not overlap logits");
  }
  const cudaStream_t stream = stream_of(x);
  const int pdl = (int)integer(a[6]);
  at::Tensor made;
  {
    Unlocked others;
    if (!to) made = at::empty({M, V}, x.options().dtype(at::kFloat));
    const at::Tensor& out = to ? *to : made;
    const at::Tensor rows = at::empty({M, FNX_TOKEN_PROBS_SCRATCH / 8}, x.options().dtype(at::kLong));
    check(fnx_token_probs(x.data_ptr(), M > 1 ? x.stride(0) : std::max(x.stride(0), V),
                          st == at::kFloat ? FNX_T_F32 : st == at::kHalf ? FNX_T_F16 : FNX_T_BF16, small(M, "rows"),
                          small(V, "vocab"), static_cast<const float*>(p[0]), static_cast<const int32_t*>(p[1]),
                          static_cast<const float*>(p[2]), static_cast<const float*>(p[3]), ptr<float>(out),
                          M > 1 ? out.stride(0) : std::max(out.stride(0), V), rows.data_ptr(), pdl, stream),
          "token_probs");
  }
  return result(a[5], std::move(made));
}

// q, k, v, positions, context_lens, node_offsets, page_table, table, k_cache, v_cache, k_scale, v_scale, interleaved,
// out, error_flag, pdl
PyObject* rotary_append8(PyObject* const* a) {
  const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &v = tensor(a[2], "v"),
                   &pos = tensor(a[3], "positions"), &ctx = tensor(a[4], "context_lens"),
                   &off = tensor(a[5], "node_offsets"), &pages = tensor(a[6], "page_table"), &table = tensor(a[7], "table"),
                   &kc = tensor(a[8], "k_cache"), &vc = tensor(a[9], "v_cache"), &ks = tensor(a[10], "k_scale"),
                   &vs = tensor(a[11], "v_scale");
  if (q.dim() != 3) refuse(PyExc_ValueError, "q must be [tokens, heads, dim], got %s", sizes(q).c_str());
  const int type = type16(q, "rotary_append8");
  on_gpu(q, "rotary_append8");
  const int64_t T = q.size(0), D = q.size(2), Hk = k.dim() == 3 ? k.size(1) : 0, B = ctx.numel();
  heads(q, "q", T, D, q);
  heads(k, "k", T, D, q);
  heads(v, "v", T, D, q);
  if (v.size(1) != Hk)
    refuse(PyExc_ValueError, "k and v must have one number of heads, got %lld and %lld", (long long)Hk,
           (long long)v.size(1));
  index(pos, "positions", T, at::kLong, q);
  index(ctx, "context_lens", B, at::kInt, q);
  index(off, "node_offsets", B + 1, at::kInt, q);
  page_table(pages, B, q);
  if (table.dim() != 2 || table.scalar_type() != at::kFloat || table.device() != q.device() ||
      (table.stride(1) != 1 && table.size(1) > 1))
    refuse(PyExc_ValueError, "table must be a row-contiguous fp32 [positions, rotated] tensor on %s",
           q.device().str().c_str());
  const int64_t R = table.size(1);
  if (R > D || R % 2)
    refuse(PyExc_ValueError, "the table's %lld columns must be even and at most dim = %lld", (long long)R, (long long)D);
  const int64_t block = caches8(kc, vc, ks, vs, q, 0);
  if (kc.size(2) != Hk || kc.size(3) != D)
    refuse(PyExc_ValueError, "caches must have k's %lld heads of %lld, got %s", (long long)Hk, (long long)D, sizes(kc).c_str());
  const cudaStream_t stream = stream_of(q);
  const at::Tensor* to = destination(a[13], q);
  const bool interleaved = truth(a[12]);
  int* flag = reinterpret_cast<int*>(integer(a[14]));
  const int pdl = (int)integer(a[15]);
  at::Tensor made;
  {
    Unlocked others;
    if (!to) made = like(q);
    const at::Tensor& out = to ? *to : made;
    check(fnx_rotary_append8(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
                             v.data_ptr(), v.stride(0), v.stride(1), out.data_ptr(), out.stride(0), out.stride(1),
                             ptr<int64_t>(pos), ptr<int32_t>(ctx), ptr<int32_t>(off), ptr<int32_t>(pages), pages.stride(0),
                             small(pages.size(1), "pages"), ptr<float>(table), table.stride(0), table.size(0), kc.data_ptr(),
                             kc.strides().data(), vc.data_ptr(), vc.strides().data(), ptr<float>(ks), ks.strides().data(),
                             ptr<float>(vs), vs.strides().data(), kc.size(0), small(kc.size(1), "page_size"),
                             small(block, "block"), small(B, "batch"), small(T, "tokens"), small(q.size(1), "q_heads"),
                             small(Hk, "kv_heads"), small(D, "dim"), (int)R, interleaved, type, flag, pdl, stream),
          "rotary_append8");
  }
  return result(a[13], std::move(made));
}

// q, k_cache, v_cache, k_scale, v_scale, page_table, context_lens, node_offsets, tree_mask, max_nodes, max_context,
// scale, out, lse, partials, error_flag, pdl
PyObject* tree_attention8(PyObject* const* a) {
  const at::Tensor &q = tensor(a[0], "q"), &kc = tensor(a[1], "k_cache"), &vc = tensor(a[2], "v_cache"),
                   &ks = tensor(a[3], "k_scale"), &vs = tensor(a[4], "v_scale"), &table = tensor(a[5], "page_table"),
                   &ctx = tensor(a[6], "context_lens"), &off = tensor(a[7], "node_offsets");
  if (q.dim() != 3) refuse(PyExc_ValueError, "q must be [nodes, heads, dim], got %s", sizes(q).c_str());
  const int type = type16(q, "tree_attention8");
  on_gpu(q, "tree_attention8");
  const int64_t N = q.size(0), Hq = q.size(1), D = q.size(2), B = ctx.numel();
  heads(q, "q", N, D, q);
  const int64_t block = caches8(kc, vc, ks, vs, q, 0);
  const int64_t Hk = kc.size(2);
  if (kc.size(3) != D)
    refuse(PyExc_ValueError, "caches must have heads of q's %lld, got %s", (long long)D, sizes(kc).c_str());
  if (Hk < 1 || Hq % Hk)
    refuse(PyExc_ValueError, "%lld query heads must be a multiple of %lld kv heads", (long long)Hq, (long long)Hk);
  index(ctx, "context_lens", B, at::kInt, q);
  index(off, "node_offsets", B + 1, at::kInt, q);
  page_table(table, B, q);
  const uint64_t* mask = nullptr;
  if (given(a[8])) {
    const at::Tensor& m = tensor(a[8], "tree_mask");
    index(m, "tree_mask", N, at::kLong, q);
    mask = ptr<uint64_t>(m);
  }
  const cudaStream_t stream = stream_of(q);
  const at::Tensor *to = destination(a[12], q), *to_lse = lse_destination(a[13], q);
  const int max_nodes = small(integer(a[9]), "max_nodes");
  const int64_t max_context = given(a[10]) ? integer(a[10]) : table.size(1) * kc.size(1);
  const float scale = given(a[11]) ? (float)number(a[11]) : 1.0f / std::sqrt((float)D);
  float* partials = reinterpret_cast<float*>(integer(a[14]));
  int* flag = reinterpret_cast<int*>(integer(a[15]));
  const int pdl = (int)integer(a[16]);
  at::Tensor made, made_lse;
  {
    Unlocked others;
    if (!to) made = like(q);
    if (!to_lse) made_lse = at::empty({N, Hq}, q.options().dtype(at::kFloat));
    const at::Tensor &out = to ? *to : made, &lse = to_lse ? *to_lse : made_lse;
    check(fnx_tree_attention8(q.data_ptr(), q.stride(0), q.stride(1), kc.data_ptr(), kc.strides().data(), vc.data_ptr(),
                              vc.strides().data(), ptr<float>(ks), ks.strides().data(), ptr<float>(vs),
                              vs.strides().data(), kc.size(0), small(kc.size(1), "page_size"), small(block, "block"),
                              ptr<int32_t>(table), table.stride(0), small(table.size(1), "pages"), ptr<int32_t>(ctx),
                              ptr<int32_t>(off), mask, out.data_ptr(), out.stride(0), out.stride(1), ptr<float>(lse),
                              small(B, "batch"), small(N, "nodes"), small(Hq, "q_heads"), small(Hk, "kv_heads"),
                              small(D, "dim"), max_nodes, max_context, scale, type, partials, flag, pdl, stream),
          "tree_attention8");
  }
  PyObject* t = PyTuple_New(2);
  PyTuple_SET_ITEM(t, 0, result(a[12], std::move(made)));
  PyTuple_SET_ITEM(t, 1, result(a[13], std::move(made_lse)));
  return t;
}

// target_probs, draft_probs, tokens, parents, node_offsets, node_uniforms, draw_uniforms, max_nodes, error_flag, pdl
PyObject* verify_tokens(PyObject* const* a) {
  const at::Tensor &p = tensor(a[0], "target_probs"), &tokens = tensor(a[2], "tokens"), &parents = tensor(a[3], "parents"),
                   &off = tensor(a[4], "node_offsets"), &nu = tensor(a[5], "node_uniforms"),
                   &du = tensor(a[6], "draw_uniforms");
  on_gpu(p, "verify_tokens");
  const int64_t N = p.dim() == 2 ? p.size(0) : 0, V = p.dim() == 2 ? p.size(1) : 0, B = du.numel();
  auto rows = [&](const at::Tensor& t, const char* name) {
    if (t.dim() != 2 || t.size(0) != N || t.size(1) != V || t.scalar_type() != at::kFloat || t.device() != p.device() ||
        (t.stride(1) != 1 && V > 1))
      refuse(PyExc_ValueError, "%s must be a row-contiguous fp32 [%s, vocab] tensor on %s, got %s %s", name,
             std::to_string(N).c_str(), p.device().str().c_str(), c10::toString(t.scalar_type()), sizes(t).c_str());
    return N > 1 ? t.stride(0) : std::max(t.stride(0), V);
  };
  const int64_t ldt = rows(p, "target_probs");
  const float* draft = nullptr;
  int64_t ldd = 0;
  if (given(a[1])) {
    const at::Tensor& q = tensor(a[1], "draft_probs");
    ldd = rows(q, "draft_probs");
    draft = ptr<float>(q);
  }
  index(tokens, "tokens", N, at::kLong, p);
  index(parents, "parents", N, at::kInt, p);
  index(nu, "node_uniforms", N, at::kFloat, p);
  index(du, "draw_uniforms", B, at::kFloat, p);
  index(off, "node_offsets", B + 1, at::kInt, p);
  const cudaStream_t stream = stream_of(p);
  const int max_nodes = small(integer(a[7]), "max_nodes");
  int* flag = reinterpret_cast<int*>(integer(a[8]));
  const int pdl = (int)integer(a[9]);
  at::Tensor path, accepted, next;
  {
    Unlocked others;
    path = at::empty({B, max_nodes < 1 ? 0 : max_nodes}, p.options().dtype(at::kInt));
    accepted = at::empty({B}, p.options().dtype(at::kInt));
    next = at::empty({B}, p.options().dtype(at::kLong));
    check(fnx_verify_tokens(ptr<float>(p), ldt, draft, ldd, ptr<int64_t>(tokens), ptr<int32_t>(parents),
                            ptr<int32_t>(off), ptr<float>(nu), ptr<float>(du), small(B, "batch"), small(N, "nodes"),
                            small(V, "vocab"), max_nodes, ptr<int32_t>(path), ptr<int32_t>(accepted), ptr<int64_t>(next),
                            flag, pdl, stream),
          "verify_tokens");
  }
  PyObject* t = PyTuple_New(3);
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(path)));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(accepted)));
  PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(std::move(next)));
  return t;
}

// k_cache, v_cache, page_table, context_lens, path, accepted, k_scale, v_scale, error_flag, pdl
PyObject* compact_nodes(PyObject* const* a) {
  const at::Tensor &kc = tensor(a[0], "k_cache"), &vc = tensor(a[1], "v_cache"), &table = tensor(a[2], "page_table"),
                   &ctx = tensor(a[3], "context_lens"), &path = tensor(a[4], "path"), &acc = tensor(a[5], "accepted");
  on_gpu(kc, "compact_nodes");
  const int64_t lead = kc.dim() == 5 ? 1 : 0, B = ctx.numel(), n = lead + 4;
  int64_t block = 0;
  const at::Tensor *ks = nullptr, *vs = nullptr;
  if (given(a[6]) != given(a[7])) refuse(PyExc_ValueError, "k_scale and v_scale come together");
  if (given(a[6])) {
    ks = &tensor(a[6], "k_scale");
    vs = &tensor(a[7], "v_scale");
    block = caches8(kc, vc, *ks, *vs, kc, lead);
  } else {
    if (kc.dim() != n || vc.sizes() != kc.sizes())
      refuse(PyExc_ValueError, "k_cache and v_cache must be [pages, page_size, kv_heads, dim] of one shape, or with layers "
             "in front; got %s and %s", sizes(kc).c_str(), sizes(vc).c_str());
    if (kc.scalar_type() == at::kFloat8_e4m3fn) refuse(PyExc_ValueError, "an 8-bit cache needs k_scale and v_scale");
    type16(kc, "compact_nodes");
    if (vc.scalar_type() != kc.scalar_type() || vc.device() != kc.device())
      refuse(PyExc_ValueError, "v_cache must be %s on %s", c10::toString(kc.scalar_type()), kc.device().str().c_str());
    if ((kc.stride(n - 1) != 1 || vc.stride(n - 1) != 1) && kc.size(n - 1) > 1)
      refuse(PyExc_ValueError, "the elements of a cached head must be contiguous");
  }
  index(ctx, "context_lens", B, at::kInt, kc);
  index(acc, "accepted", B, at::kInt, kc);
  page_table(table, B, kc);
  if (path.dim() != 2 || path.size(0) != B || path.scalar_type() != at::kInt || path.device() != kc.device() ||
      (path.stride(1) != 1 && path.size(1) > 1))
    refuse(PyExc_ValueError, "path must be a row-contiguous int32 [%lld, nodes] tensor on %s", (long long)B,
           kc.device().str().c_str());
  const cudaStream_t stream = stream_of(kc);
  int* flag = reinterpret_cast<int*>(integer(a[8]));
  const int pdl = (int)integer(a[9]);
  const int64_t elem = kc.element_size();
  int64_t st[2][3];
  for (int i = 0; i < 3; ++i) st[0][i] = kc.stride(lead + i) * elem, st[1][i] = vc.stride(lead + i) * elem;
  at::Tensor lens;
  {
    Unlocked others;
    lens = at::empty({B}, ctx.options());
    check(fnx_compact_nodes(kc.data_ptr(), st[0], lead ? kc.stride(0) * elem : 0, vc.data_ptr(), st[1],
                            lead ? vc.stride(0) * elem : 0, ks ? ptr<float>(*ks) : nullptr,
                            ks ? ks->strides().data() + lead : nullptr, ks && lead ? ks->stride(0) : 0,
                            vs ? ptr<float>(*vs) : nullptr, vs ? vs->strides().data() + lead : nullptr,
                            vs && lead ? vs->stride(0) : 0, kc.size(lead), small(kc.size(lead + 1), "page_size"),
                            small(block, "block"), (int)elem, lead ? small(kc.size(0), "layers") : 1,
                            small(kc.size(lead + 2), "kv_heads"), small(kc.size(lead + 3), "dim"), ptr<int32_t>(table),
                            table.stride(0), small(table.size(1), "pages"), ptr<int32_t>(ctx), ptr<int32_t>(path),
                            B > 1 ? path.stride(0) : path.size(1), ptr<int32_t>(acc), small(B, "batch"),
                            small(path.size(1), "path's nodes"), ptr<int32_t>(lens), flag, pdl, stream),
          "compact_nodes");
  }
  return THPVariable_Wrap(std::move(lens));
}

// No C++ exception leaves a function that Python calls.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments wanted, %zd given", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refused& e) {
    PyErr_SetString(e.type, e.what.c_str());
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

template <PyObject* (*F)(PyObject* const*), int N>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<F, N>)), METH_FASTCALL, nullptr};
}

PyMethodDef kMethods[] = {
    method<rotary_append, 12>("rotary_append"), method<tree_layout, 8>("tree_layout"),
    method<tree_attention, 15>("tree_attention"), method<sample_tokens, 7>("sample_tokens"),
    method<token_probs, 7>("token_probs"), method<rotary_append8, 16>("rotary_append8"),
    method<tree_attention8, 17>("tree_attention8"), method<verify_tokens, 10>("verify_tokens"),
    method<compact_nodes, 10>("compact_nodes"),
    {nullptr, nullptr, 0, nullptr}};

// What the module was built for is its documentation, and looked for in the file before it is loaded.
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fnx_ops", FNX_BINDING_BUILD, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fnx_ops() { return PyModule_Create(&kModule); }
