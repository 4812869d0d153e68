// w4_torch.cpp - torch tensors to the C ABI, for the calls of a batched decoding
// step: argument checks, outputs and the call itself in one C function each.
//
// Such a step is a few kernels of 3 to 10 us a layer. Checking their ten or so
// tensors in Python and filling the C ABI's structures by ctypes took 15 to
// 20 us a call, longer than the kernels run. The Python functions that document
// these calls (kv8.py, kernels.py) pass their arguments on unchanged.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <string>

#include "../../include/w4b200.h"

namespace {

using at::Tensor;

struct Refused {
  std::string what;
};
struct PythonError {};  // the Python error is set already

PyObject* g_check = nullptr;          // _lib.check: raises for a status
PyObject* g_out_of_memory = nullptr;  // torch.OutOfMemoryError

std::string text(const std::string& s) { return s; }
std::string text(int64_t n) { return std::to_string(n); }
std::string text(at::ScalarType t) { return at::toString(t); }
std::string text(const at::Device& d) { return d.str(); }
std::string text(at::IntArrayRef v) {
  std::string s = "[";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + "]";
}
std::string text(const Tensor& t) {
  return text(t.scalar_type()) + " " + text(t.sizes()) + " on " + text(t.device());
}

// Plain strings, no streams: the message must not depend on which C++ runtime
// this module and torch share.
template <typename... A>
[[noreturn]] void refuse(const A&... a) {
  throw Refused{(text(a) + ...)};
}

void check_status(int status, const char* what) {
  if (status == W4_OK) return;
  PyObject* r = PyObject_CallFunction(g_check, "is", status, what);
  Py_XDECREF(r);
  if (r) PyErr_Format(PyExc_RuntimeError, "%s: status %d", what, status);
  throw PythonError{};
}

// ------------------------------------------------------------ arguments

struct Args {
  PyObject* const* v;
  const Tensor& tensor(int i, const char* name) const {
    if (!THPVariable_Check(v[i])) {
      PyErr_Format(PyExc_TypeError, "%s must be a tensor, got %s", name, Py_TYPE(v[i])->tp_name);
      throw PythonError{};
    }
    return THPVariable_Unpack(v[i]);
  }
  const Tensor* maybe(int i, const char* name) const {
    return v[i] == Py_None ? nullptr : &tensor(i, name);
  }
  double real(int i) const {
    const double x = PyFloat_AsDouble(v[i]);
    if (x == -1.0 && PyErr_Occurred()) throw PythonError{};
    return x;
  }
  int whole(int i) const {
    const long x = PyLong_AsLong(v[i]);
    if (x == -1 && PyErr_Occurred()) throw PythonError{};
    return (int)x;
  }
};

bool is16(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }
int code(at::ScalarType t) {
  return t == at::kHalf ? W4_F16 : t == at::kBFloat16 ? W4_BF16 : W4_F32;
}

void* ptr(const Tensor& t) { return t.numel() ? const_cast<void*>(t.const_data_ptr()) : nullptr; }
bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(ptr(t)) & 15) == 0; }

// t, or a copy of it that is contiguous and 16-byte aligned.
Tensor dense16(const Tensor& t) {
  return t.is_contiguous() && aligned(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}

Tensor empty(at::IntArrayRef shape, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(shape, like.scalar_type(), like.device(), std::nullopt));
}

// An output must not overlap what a call reads: some CTAs write while others still read.
// (Both contiguous.)
bool meet(const Tensor& out, const Tensor& in) {
  const auto a = reinterpret_cast<uintptr_t>(ptr(out)), b = reinterpret_cast<uintptr_t>(ptr(in));
  return a < b + in.numel() * in.element_size() && b < a + out.numel() * out.element_size();
}

// The tensors' device current for the call, and its current stream.
struct OnDevice {
  c10::cuda::OptionalCUDAGuard guard;
  void* stream;
  explicit OnDevice(const at::Device& d) {
    if (d.index() != c10::cuda::current_device()) guard.set_device(d);
    stream = c10::cuda::getCurrentCUDAStream(d.index()).stream();
  }
};

// ------------------------------------------------------------ rows of heads

// [rows, heads, dim] as the kernels read it: 16-byte aligned, a head's elements together.
bool readable(const Tensor& t) {
  const int64_t row = t.stride(0), head = t.stride(1);
  return t.stride(2) == 1 && ((row | head) & 7) == 0 && aligned(t) && row >= 0 &&
         (t.size(1) <= 1 || head >= t.size(2));
}
Tensor rows16(const Tensor& t) {
  return readable(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}
w4_heads heads(const Tensor& t) {
  return w4_heads{ptr(t), t.stride(0), t.stride(1), (int)t.size(1)};
}

void check_rows(const char* name, const Tensor& t, const Tensor& like, int64_t n_heads,
                int64_t dim) {
  if (t.dim() != 3 || t.size(0) != like.size(0) || t.size(2) != dim ||
      (n_heads >= 0 && t.size(1) != n_heads))
    refuse(name, " must be [", like.size(0), ", ",
           n_heads >= 0 ? text(n_heads) : text("heads"), ", ", dim, "], got ",
           t);
  if (t.scalar_type() != like.scalar_type() || t.device() != like.device())
    refuse(name, " must be ", like.scalar_type(), " on ", like.device(), ", got ", t);
}

// An output: `given`, checked, or a new tensor like x.
Tensor output(const char* name, const Tensor* given, const Tensor& x) {
  if (!given) return empty(x.sizes(), x);
  check_rows(name, *given, x, x.size(1), x.size(2));
  const int64_t rows = given->size(0), n = given->size(1), dim = given->size(2);
  const int64_t row = given->stride(0), head = given->stride(1);
  // rows apart by more than their heads span, or heads by more than their rows do
  if (!readable(*given) || (rows > 1 && n > 0 && row < (n - 1) * head + dim &&
                            (row < dim || head < (rows - 1) * row + dim)))
    refuse(name, " needs 16-byte aligned heads that do not overlap, got strides ",
           given->strides());
  return *given;
}

int64_t extent(const Tensor& t) {  // elements from the first to behind the last
  return (t.size(0) - 1) * t.stride(0) + (t.size(1) - 1) * t.stride(1) + t.size(2);
}

// Whether no head of one lies over a head of the other ([rows, heads, dim] of one dim
// and type, a head's elements together). Views into one buffer may interleave.
bool apart(const Tensor& a, const Tensor& b) {
  if (!a.numel() || !b.numel()) return true;
  const int64_t dim = a.size(2), na = a.size(1), nb = b.size(1);
  const int64_t off = (static_cast<const char*>(ptr(b)) - static_cast<const char*>(ptr(a))) /
                      (int64_t)a.element_size();  // exact: both are 16-byte aligned
  if (off >= extent(a) || -off >= extent(b)) return true;
  const int64_t ra = a.stride(0) ? a.size(0) : 1, rb = b.stride(0) ? b.size(0) : 1;
  const int64_t row = ra > 1 ? a.stride(0) : rb > 1 ? b.stride(0) : 0;
  if (ra > 1 && rb > 1 && a.stride(0) != b.stride(0)) return false;  // cannot tell
  const int64_t ha = a.stride(1), hb = b.stride(1), wide_a = (na - 1) * ha + dim,
                wide_b = (nb - 1) * hb + dim;
  if (row > 0) {  // a q|k|v buffer: each takes a part of its own of every row
    const int64_t at = ((off % row) + row) % row;
    if (at >= wide_a && at + wide_b <= row) return true;
  }
  for (int64_t i = 0; i < na; ++i)
    for (int64_t j = 0; j < nb; ++j) {
      // heads i of row r and j of row s are (s - r) row + d apart
      const int64_t d = off + j * hb - i * ha;
      // the least of it lies at the s - r next to -d / row
      const int64_t least = std::clamp(row > 0 ? -d / row : 0, 1 - ra, rb - 1);
      for (int64_t k = least - 1; k <= least + 1; ++k) {
        if (k < 1 - ra || k > rb - 1) continue;
        const int64_t gap = k * row + d;
        if (gap < dim && -gap < dim) return false;
      }
    }
  return true;
}
bool same(const Tensor& a, const Tensor& b) {  // of equal sizes
  return ptr(a) == ptr(b) && (a.size(0) <= 1 || a.stride(0) == b.stride(0)) &&
         (a.size(1) <= 1 || a.stride(1) == b.stride(1));
}
// An output of the call over what the call reads, or over its other output.
void check_apart(const char* out, const Tensor& to, const char* other, const Tensor& from) {
  if (!apart(to, from)) refuse(out, " must not overlap ", other);
}
void check_over(const char* out, const Tensor& to, const char* in, const Tensor& from) {
  if (!same(to, from) && !apart(to, from))
    refuse(out, " must not overlap ", in, ", but may be ", in, " itself");
}

// Tables, norm weights, and the copies that they may have needed.
struct RopeArgs {
  Tensor cos, sin, qn, kn;
  w4_rope rope;
  RopeArgs(const Tensor* c, const Tensor* s, const Tensor* q_norm, const Tensor* k_norm, double eps,
           int64_t dim, const Tensor& like) {
    rope = w4_rope{nullptr, nullptr, 0, 0, nullptr, nullptr, (float)eps};
    if (!c != !s) refuse("cos and sin come together");
    if (c) {
      if (c->dim() != 2 || c->size(1) != dim || c->size(0) == 0 || c->sizes() != s->sizes() ||
          c->size(0) > 0x7fffffff)
        refuse("cos and sin must be [positions, ", dim, "], got ", *c, " and ", *s);
      if ((!is16(c->scalar_type()) && c->scalar_type() != at::kFloat) ||
          s->scalar_type() != c->scalar_type() || c->device() != like.device() ||
          s->device() != like.device())
        refuse("cos and sin must be of one type (float16, bfloat16 or float32) on ", like.device(),
               ", got ", *c, " and ", *s);
      cos = dense16(*c);
      sin = dense16(*s);
      rope.cos_table = ptr(cos);
      rope.sin_table = ptr(sin);
      rope.table_dtype = code(cos.scalar_type());
      rope.max_pos = (int)cos.size(0);
    }
    weight("q_norm", q_norm, dim, like, qn, &rope.q_norm);
    weight("k_norm", k_norm, dim, like, kn, &rope.k_norm);
  }
  static void weight(const char* name, const Tensor* w, int64_t dim, const Tensor& like, Tensor& at,
                     const void** to) {
    if (!w) return;
    if (w->dim() != 1 || w->size(0) != dim || w->scalar_type() != like.scalar_type() ||
        w->device() != like.device())
      refuse(name, " must be ", like.scalar_type(), " [", dim, "] on ", like.device(), ", got ",
             *w);
    at = dense16(*w);
    *to = ptr(at);
  }
};

// ------------------------------------------------------------ cache and batch

w4_kv8_cache cache_desc(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs) {
  if (k.dim() != 4 || v.sizes() != k.sizes() || ks.dim() != 2 || ks.size(0) != k.size(0) ||
      ks.size(1) != k.size(1) || vs.sizes() != ks.sizes())
    refuse("cache must be k and v [pages, kv_heads, page_size, head_dim] with scales [pages, "
           "kv_heads], got ", k.sizes(), ", ", v.sizes(), ", ", ks.sizes(), ", ", vs.sizes());
  if (k.scalar_type() != at::kFloat8_e4m3fn || v.scalar_type() != at::kFloat8_e4m3fn ||
      ks.scalar_type() != at::kFloat || vs.scalar_type() != at::kFloat)
    refuse("cache must be float8_e4m3fn with float32 scales, got ", k.scalar_type(), ", ",
           v.scalar_type(), ", ", ks.scalar_type(), ", ", vs.scalar_type());
  if (!k.is_contiguous() || !v.is_contiguous() || !ks.is_contiguous() || !vs.is_contiguous())
    refuse("cache tensors must be contiguous");
  if (!k.is_cuda() || v.device() != k.device() || ks.device() != k.device() ||
      vs.device() != k.device())
    refuse("cache tensors must be on one CUDA device");
  if (k.size(0) > 0x7fffffff) refuse("cache has ", k.size(0), " pages");
  return w4_kv8_cache{ptr(k), ptr(v), static_cast<float*>(ptr(ks)), static_cast<float*>(ptr(vs)),
                      (int)k.size(0), (int)k.size(1), (int)k.size(2), (int)k.size(3)};
}

w4_kv_batch batch_desc(const Tensor& table, const Tensor& lengths, const Tensor& row_starts,
                       int64_t rows, const at::Device& device) {
  for (const Tensor* t : {&table, &lengths, &row_starts})
    if (t->scalar_type() != at::kInt || t->device() != device)
      refuse("page_table, lengths and row_starts must be int32 on ", device, ", got ", *t);
  if (table.dim() != 2 || lengths.dim() != 1 || row_starts.dim() != 1 ||
      table.size(0) != lengths.size(0) || row_starts.size(0) != lengths.size(0) + 1)
    refuse("page_table must be [seqs, pages], lengths [seqs] and row_starts [seqs + 1], got ",
           table.sizes(), ", ", lengths.sizes(), ", ", row_starts.sizes());
  if ((table.size(1) > 1 && table.stride(1) != 1) ||
      (lengths.size(0) > 1 && lengths.stride(0) != 1) ||
      (row_starts.size(0) > 1 && row_starts.stride(0) != 1))
    refuse("page_table's rows, lengths and row_starts must be contiguous");
  if (lengths.size(0) > 0x7ffffffe || table.size(1) > 0x7fffffff || rows > (1 << 24))
    refuse("a step takes at most 2^24 rows, got ", rows);
  return w4_kv_batch{static_cast<const int32_t*>(ptr(table)), table.stride(0), (int)table.size(1),
                     static_cast<const int32_t*>(ptr(lengths)),
                     static_cast<const int32_t*>(ptr(row_starts)), (int)lengths.size(0), (int)rows};
}

// ------------------------------------------------------------ the calls

PyObject* do_norm_rope(const Args& a) {
  const Tensor& q = a.tensor(0, "q");
  const Tensor& k = a.tensor(1, "k");
  if (q.dim() != 3 || !is16(q.scalar_type()) || !q.is_cuda())
    refuse("q must be float16 or bfloat16 [rows, heads, head_dim] on a CUDA device, got ", q);
  const int64_t rows = q.size(0), dim = q.size(2);
  if (rows > 0x7fffffff) refuse("q has ", rows, " rows");
  check_rows("k", k, q, -1, dim);
  const Tensor* cos = a.maybe(2, "cos");
  const RopeArgs r(cos, a.maybe(3, "sin"), a.maybe(5, "q_norm"), a.maybe(6, "k_norm"), a.real(7),
                   dim, q);
  Tensor pos;
  if (cos) {
    const Tensor* p = a.maybe(4, "positions");
    if (!p || p->dim() != 1 || p->size(0) != rows || p->scalar_type() != at::kLong ||
        p->device() != q.device())
      refuse("positions must be int64 [", rows, "] on ", q.device());
    pos = p->contiguous();
  }
  const Tensor qo = output("q_out", a.maybe(8, "q_out"), q), ko = output("k_out", a.maybe(9, "k_out"), k);
  const Tensor qs = rows16(q), ks = rows16(k);
  if (a.v[8] != Py_None) {
    check_over("q_out", qo, "q", qs);
    check_apart("q_out", qo, "k", ks);
  }
  if (a.v[9] != Py_None) {
    check_over("k_out", ko, "k", ks);
    check_apart("k_out", ko, "q", qs);
    if (a.v[8] != Py_None) check_apart("q_out", qo, "k_out", ko);
  }
  const w4_heads hq = heads(qs), hk = heads(ks), hqo = heads(qo), hko = heads(ko);
  const OnDevice on(q.device());
  check_status(w4_qk_norm_rope(&hq, &hk, &hqo, &hko, code(q.scalar_type()), (int)rows, (int)dim,
                               &r.rope, cos ? static_cast<const int64_t*>(ptr(pos)) : nullptr,
                               on.stream),
               "qk_norm_rope");
  PyObject* both = PyTuple_New(2);
  if (!both) throw PythonError{};
  PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(qo));
  PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(ko));
  return both;
}

PyObject* do_append(const Args& a) {
  const Tensor& kc = a.tensor(0, "cache.k");
  const w4_kv8_cache c = cache_desc(kc, a.tensor(1, "cache.v"), a.tensor(2, "cache.k_scale"),
                                    a.tensor(3, "cache.v_scale"));
  const Tensor& k = a.tensor(4, "k");
  const Tensor& v = a.tensor(5, "v");
  if (k.dim() != 3 || !is16(k.scalar_type()) || k.device() != kc.device())
    refuse("k must be float16 or bfloat16 [rows, ", c.kv_heads, ", ", c.head_dim, "] on ",
           kc.device(), ", got ", k);
  check_rows("k", k, k, c.kv_heads, c.head_dim);
  check_rows("v", v, k, c.kv_heads, c.head_dim);
  const w4_kv_batch b = batch_desc(a.tensor(6, "page_table"), a.tensor(7, "lengths"),
                                   a.tensor(8, "row_starts"), k.size(0), k.device());
  const RopeArgs r(a.maybe(9, "cos"), a.maybe(10, "sin"), a.maybe(12, "q_norm"),
                   a.maybe(13, "k_norm"), a.real(14), c.head_dim, k);
  const Tensor* q = a.maybe(11, "q");
  const Tensor* given = a.maybe(15, "out");
  Tensor qs, out;
  w4_heads hq{nullptr, 0, 0, 0}, ho = hq;
  if (q) {
    check_rows("q", *q, k, -1, c.head_dim);
    out = output("out", given, *q);
    qs = rows16(*q);
    hq = heads(qs);
    ho = heads(out);
  } else if (given) {
    refuse("out is for q");
  }
  const Tensor k16 = rows16(k), v16 = rows16(v);
  if (given) {
    check_over("out", out, "q", qs);
    check_apart("out", out, "k", k16);
    check_apart("out", out, "v", v16);
  }
  const w4_heads hk = heads(k16), hv = heads(v16);
  const OnDevice on(k.device());
  check_status(
      w4_kv8_append(&c, &b, &hk, &hv, &hq, &ho, code(k.scalar_type()), &r.rope, on.stream),
      "kv8_append");
  if (!q) Py_RETURN_NONE;
  return THPVariable_Wrap(out);
}

PyObject* do_attention(const Args& a) {
  const Tensor& q = a.tensor(0, "q");
  const Tensor& kc = a.tensor(1, "cache.k");
  const w4_kv8_cache c = cache_desc(kc, a.tensor(2, "cache.v"), a.tensor(3, "cache.k_scale"),
                                    a.tensor(4, "cache.v_scale"));
  if (q.dim() != 3 || !is16(q.scalar_type()) || q.device() != kc.device() ||
      q.size(2) != c.head_dim || c.kv_heads == 0 || q.size(1) % c.kv_heads != 0)
    refuse("q must be float16 or bfloat16 [rows, n * ", c.kv_heads, ", ", c.head_dim, "] on ",
           kc.device(), ", got ", q);
  const w4_kv_batch b = batch_desc(a.tensor(5, "page_table"), a.tensor(6, "lengths"),
                                   a.tensor(7, "row_starts"), q.size(0), q.device());
  const double scale = a.v[8] == Py_None ? 1.0 / std::sqrt((double)c.head_dim) : a.real(8);
  const Tensor* given = a.maybe(9, "out");
  const Tensor out = output("out", given, q);
  const Tensor qs = rows16(q);
  if (given) check_over("out", out, "q", qs);
  const size_t need = w4_kv8_attention_workspace_bytes(c.head_dim);
  // the workspace is this call's own: the allocator keeps it apart from other
  // streams' and, during capture, from other graphs'
  const Tensor ws(at::detail::empty_cuda({(int64_t)need}, at::kByte, q.device(), std::nullopt));
  const w4_heads hq = heads(qs), ho = heads(out);
  const OnDevice on(q.device());
  check_status(w4_kv8_attention(&c, &b, &hq, &ho, code(q.scalar_type()), (float)scale, ptr(ws),
                                need, on.stream),
               "kv8_attention");
  return THPVariable_Wrap(out);
}

PyObject* do_gemm(const Args& a) {
  const Tensor& x = a.tensor(0, "x");
  const Tensor& packed = a.tensor(1, "packed");
  const Tensor& scales = a.tensor(2, "scales");
  if (packed.dim() != 2 || packed.scalar_type() != at::kInt)
    refuse("packed must be int32 [K/8, N], got ", packed);
  const int64_t K = packed.size(0) * 8, N = packed.size(1);
  if (K == 0 || N == 0) refuse("packed must have K > 0 rows and N > 0 columns, got ", packed);
  if (K % 128 != 0 || scales.dim() != 2 || scales.scalar_type() != at::kHalf ||
      scales.size(0) != K / 128 || scales.size(1) != N)
    refuse("scales must be fp16 [", K / 128, ", ", N, "] for packed ", packed.sizes(),
           " (group size 128), got ", scales);
  if (!packed.is_cuda() || scales.device() != packed.device())
    refuse("packed and scales must be on the same CUDA device");
  if (N % 128 != 0) refuse("w4_gemm_fused needs N % 128 == 0, got N=", N);
  const int act = a.whole(4);
  if (!is16(x.scalar_type()) || x.device() != packed.device() || x.dim() < 1 || x.size(-1) != K)
    refuse("x must be float16 or bfloat16 [..., ", K, "] on ", packed.device(), ", got ", x);
  const int64_t M = K ? x.numel() / K : 0, wide = act == W4_ACT_SWIGLU ? N / 2 : N;
  if (M > 0x7fffffff || K > 0x7fffffff || N > 0x7fffffff) refuse("x is too large: ", x);
  at::ScalarType type = x.scalar_type();
  if (a.v[7] != Py_None) {
    if (!THPDtype_Check(a.v[7])) refuse("out_dtype must be a torch.dtype");
    type = reinterpret_cast<THPDtype*>(a.v[7])->scalar_type;
    if (!is16(type)) refuse("out_dtype must be float16 or bfloat16, got ", type);
  }
  const Tensor* bias = a.maybe(3, "bias");
  const Tensor* residual = a.maybe(5, "residual");
  const Tensor* given = a.maybe(6, "out");
  if (bias && (bias->scalar_type() != type || bias->device() != x.device() || bias->dim() != 1 ||
               bias->size(0) != N))
    refuse("bias must be ", type, " [", N, "] on ", x.device(), ", got ", *bias);
  if (residual && (residual->scalar_type() != type || residual->device() != x.device() ||
                   residual->dim() < 1 || residual->size(-1) != wide ||
                   residual->numel() != M * wide))
    refuse("residual must be ", type, " [", M, ", ", wide, "] on ", x.device(), ", got ",
           *residual);
  if (given && (given->scalar_type() != type || given->device() != x.device() ||
                given->numel() != M * wide || !given->is_contiguous()))
    refuse("out must be a contiguous ", type, " tensor of ", M, "x", wide, " elements on ",
           x.device(), ", got ", *given);
  const Tensor x2 = dense16(x), pk = packed.contiguous(), sc = scales.contiguous();
  const Tensor b = bias ? dense16(*bias) : Tensor(), r = residual ? dense16(*residual) : Tensor();
  Tensor y;
  if (given) {
    y = *given;
    if (meet(y, x2) || meet(y, pk) || meet(y, sc) || (bias && meet(y, b)) ||
        (residual && meet(y, r) && ptr(y) != ptr(r)))
      refuse("out must not overlap the inputs (it may be the residual itself)");
  } else {
    const int64_t two[2] = {M, wide};
    y = Tensor(at::detail::empty_cuda(x.dim() == 1 ? at::IntArrayRef(two + 1, 1)
                                                   : at::IntArrayRef(two, 2),
                                      type, x.device(), std::nullopt));
  }
  if (M > 0) {
    const w4_gemm_ops ops{act, bias ? ptr(b) : nullptr, residual ? ptr(r) : nullptr};
    const OnDevice on(x.device());
    check_status(w4_gemm_fused(ptr(x2), code(x.scalar_type()), static_cast<const int32_t*>(ptr(pk)),
                               ptr(sc), ptr(y), code(type), (int)M, (int)K, (int)N, &ops,
                               a.whole(8), on.stream),
                 "w4_gemm_fused");
  }
  return THPVariable_Wrap(y);
}

// No C++ exception leaves an entry point.
template <PyObject* (*F)(const Args&), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments needed, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(Args{args});
  } catch (const PythonError&) {
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what.c_str());
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(g_out_of_memory, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

PyObject* set_errors(PyObject*, PyObject* args) {
  PyObject *check, *out_of_memory;
  if (!PyArg_ParseTuple(args, "OO", &check, &out_of_memory)) return nullptr;
  Py_INCREF(check);
  Py_XSETREF(g_check, check);
  Py_INCREF(out_of_memory);
  Py_XSETREF(g_out_of_memory, out_of_memory);
  Py_RETURN_NONE;
}

template <PyObject* (*F)(const Args&), int N>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>)),
          METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {method<do_norm_rope, 10>("qk_norm_rope"),
                           method<do_append, 16>("kv8_append"),
                           method<do_attention, 10>("kv8_attention"),
                           method<do_gemm, 9>("w4_gemm_fused"),
                           {"set_errors", set_errors, METH_VARARGS, nullptr},
                           {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_w4torch",
                        "torch tensors to the C ABI of libw4b200.so", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__w4torch() {
  PyObject* module = PyModule_Create(&g_module);
  // The torch whose headers this was compiled against; another one's objects differ.
  if (module && PyModule_AddStringConstant(module, "torch_version", W4_TORCH_VERSION) < 0)
    Py_CLEAR(module);
  return module;
}
