// Python entry of the paged decode operators (simlingo_amd/paged.py): reads the tensors, checks the arguments and calls the
// C entries of libslx_hip.so (include/slx.h) on the current stream. One of these calls is a few small tensors many times a
// token, where reading them through Python costs more than the kernels: 6 - 9 us a call there, under 2 here.
// Host code only: the library's functions and torch's stream and device getters are handed in by setup().
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <exception>
#include <initializer_list>

#include "../../include/slx.h"

namespace {

using at::Tensor;

struct Raised : std::exception {};  // the Python error is set

[[noreturn]] void fail(PyObject* type, const char* who, const char* fmt, ...) {
  char msg[400];
  int n = snprintf(msg, sizeof msg, "%s: ", who);
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg + n, sizeof msg - n, fmt, ap);
  va_end(ap);
  PyErr_SetString(type, msg);
  throw Raised();
}
#define NEED(ok, ...)                                        \
  do {                                                       \
    if (!(ok)) fail(PyExc_ValueError, who, __VA_ARGS__);     \
  } while (0)

// ---- handed in by setup() --------------------------------------------------------------------------------------
struct Lib {
  int (*kv_append)(const slx_kv_append_desc*, slx_stream_t);
  int (*prefix_attn)(const slx_prefix_attn_desc*, slx_stream_t);
  int64_t (*prefix_attn_ws_floats)(const slx_prefix_attn_desc*);
  int (*beam_select)(const slx_beam_select_desc*, slx_stream_t);
  int64_t (*beam_select_ws_bytes)(const slx_beam_select_desc*);
  int (*beam_reorder)(const slx_beam_reorder_desc*, slx_stream_t);
  const char* (*last_error)();
} lib;
PyObject *get_stream, *get_device;

void check(int64_t rc, const char* name) {
  if (!rc) return;
  PyErr_Format(PyExc_RuntimeError, "%s failed (rc=%d): %s", name, (int)rc, lib.last_error());
  throw Raised();
}

// ---- arguments -------------------------------------------------------------------------------------------------
const Tensor& any_tensor(PyObject* o, const char* who, const char* name) {
  if (!THPVariable_Check(o)) fail(PyExc_TypeError, who, "%s must be a tensor", name);
  return THPVariable_Unpack(o);
}
const Tensor& tensor(PyObject* o, const char* who, const char* name) {
  const Tensor& t = any_tensor(o, who, name);
  NEED(!t.is_neg(), "%s is a lazily negated view (resolve_neg)", name);  // none of the types taken here can be conjugated
  return t;
}
const Tensor* maybe(PyObject* o, const char* who, const char* name) { return o == Py_None ? nullptr : &tensor(o, who, name); }
int64_t integer(PyObject* o, const char* who, const char* name) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    fail(PyExc_TypeError, who, "%s must be an integer", name);
  }
  return v;
}
constexpr int64_t kIntMax = 2147483647;

bool is_bool(const Tensor& t) { return t.scalar_type() == at::kBool || t.scalar_type() == at::kByte; }

struct Rows { void* p; int64_t ld; };
Rows rows_of(const char* who, const char* name, const Tensor& t, int64_t n, int64_t cols, bool written = false) {
  NEED(t.scalar_type() == at::kBFloat16 && t.dim() == 2, "%s must be a bf16 matrix", name);
  NEED(t.size(0) == n && t.size(1) >= cols, "%s must have %lld rows of at least %lld, got %lld x %lld", name, (long long)n,
       (long long)cols, (long long)t.size(0), (long long)t.size(1));
  const int64_t s0 = n > 1 ? t.stride(0) : t.size(1) / 8 * 8, s1 = t.stride(1);  // one row's stride says nothing
  NEED(s1 == 1 && s0 % 8 == 0 && ((uintptr_t)t.data_ptr() & 15) == 0, "rows of %s must be contiguous and 16-B aligned", name);
  NEED(!written || n <= 1 || s0 >= cols, "rows of %s overlap each other", name);
  return {t.data_ptr(), s0};
}

// Whether a call that reads x rows and writes y rows (n of them, wx and wy wide) may: apart, other columns of the same rows, or
// y in x's place.
bool may_write(const Rows& x, int64_t wx, const Rows& y, int64_t wy, int64_t n) {
  const int64_t delta = ((const char*)y.p - (const char*)x.p) / 2;  // both 16-B aligned
  if (n == 0 || delta >= (n - 1) * x.ld + wx || -delta >= (n - 1) * y.ld + wy) return true;
  if (x.ld != y.ld && n > 1) return false;
  if (delta == 0) return true;
  if (n == 1) return false;
  return delta > 0 ? delta >= wx && delta + wy <= x.ld : -delta >= wy && -delta + wx <= x.ld;
}

// ---- what is written lies apart ---------------------------------------------------------------------------------
// The memory of a strided array in bytes: runs of `run` bytes from p, ext[i] of them st[i] apart along each axis.
struct Box {
  const char* p;
  int64_t run;
  int n;
  int64_t ext[4], st[4];
  Box(const void* at, int64_t run_) : p((const char*)at), run(run_), n(0) {}
  Box& axis(int64_t e, int64_t s) {  // a run without elements stands for an empty array
    if (e == 0) run = 0;
    if (e > 1 && s != 0) { ext[n] = e; st[n++] = s; }
    return *this;
  }
  const char* end() const {
    const char* q = p + run;
    for (int i = 0; i < n; ++i) q += (ext[i] - 1) * st[i];
    return q;
  }
};
Box box_of(const Rows& r, int64_t n, int64_t cols) { return Box(r.p, 2 * cols).axis(n, 2 * r.ld); }
Box box_of(const slx_kv_pool& p, const void* at) {
  return Box(at, 2 * p.head_dim).axis(p.n_pages, 2 * p.page_stride).axis(p.page, 2 * p.slot_stride).axis(p.heads, 2 * p.head_stride);
}
Box box_of(const Tensor& t) {  // contiguous, or rows of a table
  const int64_t es = (int64_t)t.element_size();
  if (t.dim() == 2) return Box(t.data_ptr(), es * t.size(1)).axis(t.size(0), es * t.stride(0));
  return Box(t.data_ptr(), es * t.numel());
}

// Whether sum x_i s_i falls into [lo, hi] for whole x_i in [from_i, to_i], the largest s first: the x of an axis are those that leave
// what the axes after it can reach, one or two where an axis is longer than all after it together. An axis that another one's steps fill
// without a gap (pages of whole slots, slots that are another array's rows) is joined to it first. Arrays that take more than a few
// thousand trials are taken to meet.
struct Sum {
  int n = 0, tries = 4096;
  int64_t s[8], from[8], to[8], least[9], most[9];  // least, most: of the axes from i on
  void add(int64_t stride, int64_t f, int64_t t) {
    for (int i = 0; i < n; ++i)
      if (s[i] == stride) { from[i] += f; to[i] += t; return; }
    int i = n++;
    for (; i > 0 && s[i - 1] < stride; --i) { s[i] = s[i - 1]; from[i] = from[i - 1]; to[i] = to[i - 1]; }
    s[i] = stride; from[i] = f; to[i] = t;
  }
  static int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }
  bool reaches(int i, int64_t lo, int64_t hi) {
    if (i == n) return lo <= 0 && hi >= 0;
    const int64_t a = std::max(from[i], -floor_div(most[i + 1] - lo, s[i])), b = std::min(to[i], floor_div(hi - least[i + 1], s[i]));
    for (int64_t x = a; x <= b; ++x)
      if (--tries < 0 || reaches(i + 1, lo - x * s[i], hi - x * s[i])) return true;
    return false;
  }
  void join() {
    for (int j = 1; j < n; ++j)
      for (int i = j - 1; i >= 0; --i) {
        const int64_t q = s[i] / s[j];
        if (s[i] % s[j] || to[j] - from[j] + 1 < q) continue;
        from[j] += q * from[i];
        to[j] += q * to[i];
        --n;
        for (int m = i; m < n; ++m) { s[m] = s[m + 1]; from[m] = from[m + 1]; to[m] = to[m + 1]; }
        j = 0;  // from the start: a longer axis may be filled now
        break;
      }
  }
  bool reaches(int64_t lo, int64_t hi) {
    join();
    least[n] = most[n] = 0;
    for (int i = n - 1; i >= 0; --i) {
      least[i] = least[i + 1] + from[i] * s[i];
      most[i] = most[i + 1] + to[i] * s[i];
    }
    return reaches(0, lo, hi);
  }
};
bool meet(const Box& a, const Box& b) {
  if (!a.run || !b.run || a.end() <= b.p || b.end() <= a.p) return false;
  Sum s;
  for (int i = 0; i < a.n; ++i) s.add(a.st[i], 1 - a.ext[i], 0);
  for (int i = 0; i < b.n; ++i) s.add(b.st[i], 0, b.ext[i] - 1);
  const int64_t delta = b.p - a.p;
  return s.reaches(1 - b.run - delta, a.run - 1 - delta);
}
// Whether two runs of one array share memory: not where each axis steps over all that lies within it; else by the runs that differ
// along axis i first, by x_i > 0.
bool folds(const Box& a) {
  if (!a.run) return false;
  int64_t within = a.run;
  int left = a.n;
  for (unsigned done = 0; left; --left) {
    int least = -1;
    for (int i = 0; i < a.n; ++i)
      if (!(done >> i & 1) && (least < 0 || a.st[i] < a.st[least])) least = i;
    if (a.st[least] < within) break;
    within += (a.ext[least] - 1) * a.st[least];
    done |= 1u << least;
  }
  if (!left) return false;
  for (int i = 0; i < a.n; ++i) {
    Sum s;
    s.add(a.st[i], 1, a.ext[i] - 1);
    for (int j = i + 1; j < a.n; ++j) s.add(a.st[j], 1 - a.ext[j], a.ext[j] - 1);
    if (s.reaches(1 - a.run, a.run - 1)) return true;
  }
  return false;
}

slx_kv_pool pool_of(const char* who, const Tensor& k, const Tensor& v, bool written) {
  NEED(k.scalar_type() == at::kBFloat16 && v.scalar_type() == at::kBFloat16 && k.dim() == 4,
       "k and v must be bf16 [pages, page, heads, head size]");
  NEED(k.sizes() == v.sizes() && k.strides() == v.strides(), "k and v must have the same shape and strides");
  const auto sh = k.sizes();
  const auto st = k.strides();
  NEED(sh[0] > 0 && sh[0] <= kIntMax && sh[1] > 0 && sh[1] <= kIntMax && (sh[1] & (sh[1] - 1)) == 0 && sh[2] > 0 && sh[2] <= kIntMax &&
       (sh[3] == 64 || sh[3] == 128), "pages and heads > 0, page a power of two, head size 64 or 128 (got [%lld, %lld, %lld, %lld])",
       (long long)sh[0], (long long)sh[1], (long long)sh[2], (long long)sh[3]);
  NEED(st[3] == 1 && ((st[0] | st[1] | st[2]) & 7) == 0 && (((uintptr_t)k.data_ptr() | (uintptr_t)v.data_ptr()) & 15) == 0,
       "heads of k and v must be contiguous and 16-B aligned");
  NEED(!written || k.data_ptr() != v.data_ptr(), "k and v are the same memory");
  NEED(!written || ((st[0] || sh[0] == 1) && (st[1] || sh[1] == 1) && (st[2] || sh[2] == 1)), "k and v must not be expanded");
  slx_kv_pool p;
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.page_stride = st[0]; p.slot_stride = st[1]; p.head_stride = st[2];
  p.n_pages = (int)sh[0]; p.page = (int)sh[1]; p.heads = (int)sh[2]; p.head_dim = (int)sh[3];
  NEED(!written || !folds(box_of(p, p.k)), "heads of the cache overlap each other");
  NEED(!written || !meet(box_of(p, p.k), box_of(p, p.v)), "k and v overlap");
  return p;
}

struct Table { const int* p; int64_t ld; int n, cols; };
Table table_of(const char* who, const char* name, const Tensor& t) {
  NEED(t.scalar_type() == at::kInt && t.dim() == 2, "%s must be int32 [sequences, columns]", name);
  const int64_t n = t.size(0), cols = t.size(1), s0 = t.stride(0), s1 = t.stride(1);
  NEED(n <= kIntMax && cols > 0 && cols <= kIntMax && (s1 == 1 || cols == 1) && (s0 >= cols || n <= 1),
       "%s must have columns, its rows contiguous and apart", name);
  return {(const int*)t.data_ptr(), s0 > cols ? s0 : cols, (int)n, (int)cols};
}

const int* ints_of(const char* who, const char* name, const Tensor& t, int64_t n) {
  NEED(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous(), "%s must be contiguous int32 [%lld]", name,
       (long long)n);
  return (const int*)t.data_ptr();
}

// Every tensor on the current device, where the launch goes -> its current stream.
slx_stream_t stream_of(const char* who, std::initializer_list<const Tensor*> ts) {
  const Tensor* first = nullptr;
  for (const Tensor* t : ts) {
    if (!t) continue;
    if (!first) first = t;
    if (t->device() != first->device())
      fail(PyExc_RuntimeError, who, "tensors on %s and %s", first->device().str().c_str(), t->device().str().c_str());
  }
  if (!get_device) fail(PyExc_RuntimeError, who, "setup() was not called");
  if (!first->is_cuda()) fail(PyExc_RuntimeError, who, "SimLingo MI355X kernels need device tensors (no CPU fallback)");
  PyObject* cur = PyObject_CallNoArgs(get_device);
  if (!cur) throw Raised();
  const long dev = PyLong_AsLong(cur);
  if (first->device().index() != dev) {
    Py_DECREF(cur);
    fail(PyExc_RuntimeError, who, "tensors on %s, current device cuda:%ld", first->device().str().c_str(), dev);
  }
  PyObject* s = PyObject_CallOneArg(get_stream, cur);
  Py_DECREF(cur);
  if (!s) throw Raised();
  void* p = PyLong_AsVoidPtr(s);
  Py_DECREF(s);
  if (!p && PyErr_Occurred()) throw Raised();
  return (slx_stream_t)p;
}

// Runs a body; C++ exceptions become Python's.
template <typename F>
PyObject* guarded(const char* name, Py_ssize_t have, Py_ssize_t want, F&& body) {
  if (have != want) return PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, want, have);
  try {
    return body();
  } catch (const Raised&) {
  } catch (const std::exception& e) {
    PyErr_Format(PyExc_RuntimeError, "%s: %s", name, e.what());
  }
  return nullptr;
}
PyObject* none() { Py_RETURN_NONE; }

// (qkv, k, v, table, pos, q_out, n_heads, cos, sin, seq, rows_per_seq)
PyObject* kv_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded("kv_append", n, 11, [&] {
    const char* who = "kv_append";
    const Tensor &qkv = tensor(a[0], who, "qkv"), &k = tensor(a[1], who, "k"), &v = tensor(a[2], who, "v"), &table = tensor(a[3], who, "table"),
                 &pos = tensor(a[4], who, "pos");
    const Tensor *q = maybe(a[5], who, "q_out"), *cs = maybe(a[7], who, "cos"), *sn = maybe(a[8], who, "sin"), *seq = maybe(a[9], who, "seq");
    const int64_t heads = integer(a[6], who, "n_heads"), per = integer(a[10], who, "rows_per_seq");
    slx_kv_append_desc d{};
    d.pool = pool_of(who, k, v, true);
    const int64_t hkv = d.pool.heads, hd = d.pool.head_dim;
    NEED(heads >= 0 && heads <= (1 << 24) && (!q || heads > 0), "n_heads %lld", (long long)heads);
    NEED(qkv.dim() == 2, "qkv must be a bf16 matrix");
    d.rows = qkv.size(0);
    const Rows x = rows_of(who, "qkv", qkv, d.rows, (heads + 2 * hkv) * hd);
    d.qkv = x.p; d.ldqkv = x.ld;
    const Table t = table_of(who, "table", table);
    d.table = t.p; d.ldt = t.ld; d.n_seq = t.n; d.cols = t.cols;
    NEED(t.n > 0 && per > 0 && per <= kIntMax, "an empty table, or rows_per_seq < 1");
    d.rows_per_seq = (int)per;
    d.Hq = (int)heads;
    d.pos = ints_of(who, "pos", pos, d.rows);
    if (seq) d.seq = ints_of(who, "seq", *seq, d.rows);
    if (q) {
      const Rows y = rows_of(who, "q_out", *q, d.rows, heads * hd, true);
      NEED(may_write(x, (heads + 2 * hkv) * hd, y, heads * hd, d.rows), "q_out overlaps qkv other than in its own q columns");
      d.q_out = y.p; d.ldq = y.ld;
    }
    NEED(!cs == !sn, "cos and sin go together");
    if (cs) {
      NEED(cs->scalar_type() == at::kFloat && sn->scalar_type() == at::kFloat && cs->dim() == 2 && cs->sizes() == sn->sizes() &&
           cs->size(0) > 0 && cs->size(0) <= kIntMax && cs->size(1) == hd / 2 && cs->is_contiguous() && sn->is_contiguous() &&
           (((uintptr_t)cs->data_ptr() | (uintptr_t)sn->data_ptr()) & 15) == 0, "cos and sin must be contiguous f32 [positions, %lld]",
           (long long)(hd / 2));
      d.cos_tab = (const float*)cs->data_ptr(); d.sin_tab = (const float*)sn->data_ptr(); d.rope_rows = (int)cs->size(0);
    }
    const Box to[3] = {box_of(d.pool, d.pool.k), box_of(d.pool, d.pool.v), Box(d.q_out, 2 * heads * hd).axis(q ? d.rows : 0, 2 * d.ldq)};
    for (int i = 0; i < 3; ++i) {
      for (const Tensor* t : {&table, &pos, seq, cs, sn}) NEED(!t || !meet(to[i], box_of(*t)), "%s overlaps the table, positions, sequences or rotation", i < 2 ? "the cache" : "q_out");
      if (i < 2) NEED(!meet(to[i], box_of(x, d.rows, (heads + 2 * hkv) * hd)) && !meet(to[i], to[2]), "the cache overlaps qkv or q_out");
    }
    const slx_stream_t s = stream_of(who, {&qkv, &k, &v, &table, &pos, q, cs, sn, seq});
    check(lib.kv_append(&d, s), "slx_kv_append");
    return none();
  });
}

// (q, out, ok, ov, otab, olen, pk, pv, ptab, plen, n_heads, n_q, scale, max_own, max_prefix, lse) -> out; pk None: no prefix
PyObject* prefix_attn(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded("prefix_attn", n, 16, [&]() -> PyObject* {
    const char* who = "prefix_attn";
    const Tensor &q = tensor(a[0], who, "q"), &ok = tensor(a[2], who, "k"), &ov = tensor(a[3], who, "v"), &otab = tensor(a[4], who, "own table"),
                 &olen = tensor(a[5], who, "own lengths");
    const Tensor *pk = maybe(a[6], who, "k"), *pv = nullptr, *ptab = nullptr, *plen = nullptr, *lse = maybe(a[15], who, "lse");
    const int64_t heads = integer(a[10], who, "n_heads"), n_q = integer(a[11], who, "n_q");
    slx_prefix_attn_desc d{};
    d.own_pool = pool_of(who, ok, ov, false);
    const int64_t hd = d.own_pool.head_dim;
    const Table ot = table_of(who, "own table", otab);
    d.otab = ot.p; d.ldot = ot.ld; d.ocols = ot.cols;
    NEED(heads > 0 && heads <= (1 << 24) && heads % d.own_pool.heads == 0, "n_heads must be a multiple of the cache's %d heads", d.own_pool.heads);
    NEED(n_q > 0 && n_q <= kIntMax, "n_q %lld", (long long)n_q);
    d.Hq = (int)heads;
    d.n_q = (int)n_q;
    double scale = a[12] == Py_None ? 1.0 / std::sqrt((double)hd) : PyFloat_AsDouble(a[12]);
    if (PyErr_Occurred()) throw Raised();
    d.scale = (float)scale;
    NEED(d.scale > 0 && d.scale * 1.44269504088896341f < INFINITY, "scale must be positive and, times log2(e), finite in 32 bits");
    const int64_t rows = (int64_t)ot.n * n_q, cols = heads * hd;
    const Rows x = rows_of(who, "q", q, rows, cols);
    d.q = x.p; d.ldq = x.ld;
    d.olen = ints_of(who, "own lengths", olen, ot.n);
    d.groups = ot.n;
    auto bound = [&](PyObject* o, int64_t c, int page, const char* name) {
      const int64_t most = c * page < kIntMax ? c * page : kIntMax, b = o == Py_None ? most : integer(o, who, name);
      NEED(b >= 0 && b <= kIntMax, "bounds must be 0 .. 2^31 - 1");
      return (int)b;
    };
    d.max_own = bound(a[13], ot.cols, d.own_pool.page, "max_own");
    if (pk) {
      pv = &tensor(a[7], who, "v");
      ptab = &tensor(a[8], who, "prefix table");
      plen = &tensor(a[9], who, "prefix lengths");
      d.prefix_pool = pool_of(who, *pk, *pv, false);
      NEED(d.prefix_pool.heads == d.own_pool.heads && d.prefix_pool.head_dim == hd, "the two caches differ in heads or head size");
      const Table pt = table_of(who, "prefix table", *ptab);
      d.ptab = pt.p; d.ldpt = pt.ld; d.pcols = pt.cols;
      d.plen = ints_of(who, "prefix lengths", *plen, pt.n);
      NEED(pt.n > 0 && ot.n % pt.n == 0, "%d sequences do not make %d groups of one size", ot.n, pt.n);
      d.groups = pt.n;
      d.max_prefix = bound(a[14], pt.cols, d.prefix_pool.page, "max_prefix");
    } else if (a[14] != Py_None) {
      bound(a[14], 0, 1, "max_prefix");
    }
    d.width = d.groups ? ot.n / d.groups : 1;
    Tensor made;
    if (a[1] == Py_None) made = at::empty({rows, cols}, q.options());
    const Tensor& out = a[1] == Py_None ? made : tensor(a[1], who, "out");
    const Rows o = rows_of(who, "out", out, rows, cols, true);
    NEED(may_write(x, cols, o, cols, rows), "out overlaps q other than in its place");
    d.out = o.p; d.ldo = o.ld;
    if (lse) {
      NEED(lse->scalar_type() == at::kFloat && lse->dim() == 2 && lse->size(0) == rows && lse->size(1) == heads && lse->is_contiguous(),
           "lse must be contiguous f32 [%lld, %lld]", (long long)rows, (long long)heads);
      d.lse = (float*)lse->data_ptr();
      auto apart = [&](const Rows& r) {
        return !rows || (char*)(d.lse + rows * heads) <= (char*)r.p || (char*)r.p + 2 * ((rows - 1) * r.ld + cols) <= (char*)d.lse;
      };
      NEED(apart(x) && apart(o), "lse overlaps q or out");
    }
    const Box to[2] = {box_of(o, rows, cols), Box(d.lse, lse ? 4 * rows * heads : 0)};
    for (const Box& y : to) {
      for (const slx_kv_pool* p : {&d.own_pool, &d.prefix_pool}) {
        if (p->k) NEED(!meet(y, box_of(*p, p->k)) && !meet(y, box_of(*p, p->v)), "%s overlaps a cache", &y == to ? "out" : "lse");
      }
      for (const Tensor* t : {(const Tensor*)&otab, (const Tensor*)&olen, ptab, plen}) NEED(!t || !meet(y, box_of(*t)), "%s overlaps a table or lengths", &y == to ? "out" : "lse");
    }
    const slx_stream_t s = stream_of(who, {&q, &ok, &ov, &otab, &olen, &out, pk, pv, ptab, plen, lse});
    if (ot.n) {
      const int64_t need = lib.prefix_attn_ws_floats(&d);
      if (need < 0) check(need, "slx_prefix_attn");
      Tensor ws;  // of this call alone, from the current stream's memory
      if (need) {
        ws = at::empty({need}, q.options().dtype(at::kFloat));
        d.ws = (float*)ws.data_ptr();
        d.ws_floats = need;
      }
      check(lib.prefix_attn(&d, s), "slx_prefix_attn");
    }
    if (a[1] == Py_None) return THPVariable_Wrap(made);
    Py_INCREF(a[1]);
    return a[1];
  });
}

// (logits, scores, width, k, finished, pad_id, eos_id, out, finished_out) -> out
PyObject* beam_select(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded("beam_select", n, 9, [&]() -> PyObject* {
    const char* who = "beam_select";
    const Tensor &x = tensor(a[0], who, "logits"), &scores = tensor(a[1], who, "scores");
    const Tensor *fin = maybe(a[4], who, "finished"), *fout = maybe(a[8], who, "finished_out");
    const int64_t w = integer(a[2], who, "width"), k = a[3] == Py_None ? w : integer(a[3], who, "k");
    NEED(w > 0 && w <= 64 && k > 0 && k <= 64, "width and k must be 1 .. 64");
    const bool bf = x.scalar_type() == at::kBFloat16;
    NEED(x.dim() == 2 && (bf || x.scalar_type() == at::kFloat), "logits must be f32 or bf16 [rows, V]");
    const int64_t rows = x.size(0), vocab = x.size(1), ldx = x.stride(0);
    NEED((x.stride(1) == 1 || vocab <= 1) && (ldx >= vocab || rows <= 1), "rows of logits must be contiguous and apart");
    NEED(vocab > 0 && vocab <= 262144 && rows % w == 0 && k <= w * vocab,
         "1 .. 262144 logits a row, rows a multiple of width, k <= width * V");
    const int64_t b = rows / w;
    NEED(b <= kIntMax, "too many rows");
    NEED(scores.scalar_type() == at::kFloat && scores.numel() == rows && scores.is_contiguous(), "scores must be contiguous f32 [%lld]", (long long)rows);
    slx_beam_select_desc d{};
    if (fin) {
      NEED(is_bool(*fin) && fin->numel() == rows && fin->is_contiguous(), "finished must be contiguous bool [%lld]", (long long)rows);
      const int64_t pad = integer(a[5], who, "pad_id");
      NEED(pad >= 0 && pad < vocab, "pad_id outside the vocabulary");
      d.finished = (const unsigned char*)fin->data_ptr();
      d.pad = (int)pad;
    }
    if (fout) {
      NEED(is_bool(*fout) && fout->numel() == b * k && fout->is_contiguous(), "finished_out must be contiguous bool [%lld, %lld]", (long long)b, (long long)k);
      d.finished_out = (unsigned char*)fout->data_ptr();
    }
    d.eos = -1;
    if (a[6] != Py_None) {
      const int64_t e = integer(a[6], who, "eos_id");
      d.eos = e >= 0 && e < vocab ? (int)e : -1;
    }
    Tensor made[3];
    const Tensor* to[3];
    if (a[7] == Py_None) {
      made[0] = at::empty({b, k}, x.options().dtype(at::kFloat));
      made[1] = at::empty({b, k}, x.options().dtype(at::kInt));
      made[2] = at::empty({b, k}, x.options().dtype(at::kInt));
      for (int i = 0; i < 3; ++i) to[i] = &made[i];
    } else {
      NEED(PyTuple_Check(a[7]) && PyTuple_GET_SIZE(a[7]) == 3, "out must be three tensors");
      for (int i = 0; i < 3; ++i) to[i] = &tensor(PyTuple_GET_ITEM(a[7], i), who, "out");
    }
    for (int i = 0; i < 3; ++i)
      NEED(to[i]->scalar_type() == (i ? at::kInt : at::kFloat) && to[i]->numel() == b * k && to[i]->is_contiguous(),
           "out must be contiguous f32, int32, int32 [%lld, %lld]", (long long)b, (long long)k);
    d.logits = x.data_ptr(); d.ldx = ldx > vocab ? ldx : vocab; d.logits_bf16 = bf;
    d.batch = (int)b; d.width = (int)w; d.vocab = (int)vocab; d.k = (int)k;
    d.score = (const float*)scores.data_ptr();
    d.score_out = (float*)to[0]->data_ptr(); d.parent = (int*)to[1]->data_ptr(); d.token = (int*)to[2]->data_ptr();
    // batch entries run apart: what one writes, no other may read or write, but for scores and finished in place
    const struct { const void* p; int64_t n; } put[4] = {{d.score_out, 4 * b * k}, {d.parent, 4 * b * k}, {d.token, 4 * b * k}, {d.finished_out, b * k}},
                                               get[2] = {{d.score, 4 * rows}, {d.finished, rows}};
    auto apart = [](const auto& u, const auto& t) {
      return !u.p || !t.p || (const char*)u.p + u.n <= (const char*)t.p || (const char*)t.p + t.n <= (const char*)u.p;
    };
    for (int i = 0; i < 4; ++i) {
      for (int j = 0; j < 2; ++j) NEED(apart(put[i], get[j]) || (k == w && i == 3 * j && put[i].p == get[j].p), "scores or finished in place need k == width, and all of it");
      for (int j = 0; j < i; ++j) NEED(apart(put[i], put[j]), "outputs overlap");
    }
    const slx_stream_t s = stream_of(who, {&x, &scores, to[0], to[1], to[2], fin, fout});
    if (b) {
      const int64_t need = lib.beam_select_ws_bytes(&d);
      if (need < 0) check(need, "slx_beam_select");
      const Tensor ws = at::empty({need}, x.options().dtype(at::kByte));  // of this call alone, from the current stream's memory
      d.ws = ws.data_ptr();
      d.ws_bytes = need;
      check(lib.beam_select(&d, s), "slx_beam_select");
    }
    if (a[7] != Py_None) {
      Py_INCREF(a[7]);
      return a[7];
    }
    PyObject* r = PyTuple_New(3);
    if (!r) throw Raised();
    for (int i = 0; i < 3; ++i) {
      PyObject* t = THPVariable_Wrap(made[i]);
      if (!t) {
        Py_DECREF(r);
        throw Raised();
      }
      PyTuple_SET_ITEM(r, i, t);
    }
    return r;
  });
}

// (x, parent, dim, out) -> out
PyObject* beam_reorder(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded("beam_reorder", n, 4, [&]() -> PyObject* {
    const char* who = "beam_reorder";
    const Tensor &x = any_tensor(a[0], who, "x"), &parent = tensor(a[1], who, "parent");
    PyObject* back = a[3] == Py_None ? a[0] : a[3];
    const Tensor& out = any_tensor(back, who, "out");
    NEED(x.is_neg() == out.is_neg() && x.is_conj() == out.is_conj(), "x or out alone is lazily negated or conjugated");
    NEED(parent.scalar_type() == at::kInt && parent.dim() == 2 && parent.is_contiguous(), "parent must be contiguous int32 [batch, W]");
    const int64_t b = parent.size(0), w = parent.size(1), nd = x.dim();
    int64_t dim = integer(a[2], who, "dim");
    NEED(w > 0 && w <= 64 && b <= kIntMax, "W must be 1 .. 64");
    NEED(dim >= -nd && dim < nd && x.sizes() == out.sizes() && x.scalar_type() == out.scalar_type(), "dim, or out unlike x");
    if (dim < 0) dim += nd;
    NEED(x.size(dim) == b * w, "dimension %lld of x has %lld rows, parent %lld x %lld", (long long)dim, (long long)x.size(dim), (long long)b, (long long)w);
    const int64_t es = (int64_t)x.element_size();
    int64_t run = 1, m[2] = {1, 1}, s[2] = {0, 0}, t[2] = {0, 0};  // a row's contiguous elements; the outer dimensions, inner first
    int outer = 0;
    if (x.numel()) {
      for (int64_t i = nd - 1; i >= 0; --i) {
        const int64_t e = x.size(i), xs = x.stride(i), os = out.stride(i);
        if (i == dim || e == 1) continue;
        if (!outer && xs == run && os == run) {
          run *= e;
        } else if (outer && xs == m[outer - 1] * s[outer - 1] && os == m[outer - 1] * t[outer - 1]) {
          m[outer - 1] *= e;
        } else {
          NEED(outer < 2, "the state's strides make more than two runs of rows");
          NEED(os, "out must not be expanded");
          m[outer] = e; s[outer] = xs; t[outer] = os;
          ++outer;
        }
      }
      NEED(out.stride(dim) || b * w == 1, "out must not be expanded");
      NEED(m[0] <= kIntMax && m[1] <= kIntMax, "dimensions too long");
      const auto box = [&](const Tensor& u, const int64_t* st) {
        return Box(u.data_ptr(), run * es).axis(m[1], st[1] * es).axis(m[0], st[0] * es).axis(b * w, u.stride(dim) * es);
      };
      const Box to = box(out, t);
      const bool same = x.data_ptr() == out.data_ptr() && s[0] == t[0] && s[1] == t[1] && (x.stride(dim) == out.stride(dim) || b * w == 1);
      NEED(same || !meet(box(x, s), to), "out overlaps x");
      NEED(!folds(to), "rows of out overlap each other");
      NEED(!meet(to, box_of(parent)), "out overlaps parent");
    }
    const slx_stream_t st = stream_of(who, {&x, &out, &parent});
    if (x.numel()) {
      slx_beam_reorder_desc d{};
      d.src = x.data_ptr(); d.dst = out.data_ptr();
      const bool one = b * w == 1;  // its stride says nothing
      d.s0 = s[1] * es; d.s1 = s[0] * es; d.src_row = one ? 0 : x.stride(dim) * es;
      d.d0 = t[1] * es; d.d1 = t[0] * es; d.dst_row = one ? 0 : out.stride(dim) * es;
      d.row_bytes = run * es;
      d.n0 = (int)m[1]; d.n1 = (int)m[0]; d.batch = (int)b; d.width = (int)w;
      d.parent = (const int*)parent.data_ptr();
      check(lib.beam_reorder(&d, st), "slx_beam_reorder");
    }
    Py_INCREF(back);
    return back;
  });
}

// (addresses of the C entries in Lib's order, current_raw_stream(device), current_device())
PyObject* setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded("setup", n, 3, [&] {
    void* p[7];
    if (!PyTuple_Check(a[0]) || PyTuple_GET_SIZE(a[0]) != 7) fail(PyExc_TypeError, "setup", "seven addresses");
    for (int i = 0; i < 7; ++i) {
      p[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(a[0], i));
      if (!p[i]) fail(PyExc_TypeError, "setup", "seven addresses");
    }
    lib.kv_append = (decltype(lib.kv_append))p[0];
    lib.prefix_attn = (decltype(lib.prefix_attn))p[1];
    lib.prefix_attn_ws_floats = (decltype(lib.prefix_attn_ws_floats))p[2];
    lib.beam_select = (decltype(lib.beam_select))p[3];
    lib.beam_select_ws_bytes = (decltype(lib.beam_select_ws_bytes))p[4];
    lib.beam_reorder = (decltype(lib.beam_reorder))p[5];
    lib.last_error = (decltype(lib.last_error))p[6];
    Py_INCREF(a[1]);
    Py_INCREF(a[2]);
    Py_XDECREF(get_stream);
    Py_XDECREF(get_device);
    get_stream = a[1];
    get_device = a[2];
    return none();
  });
}

#define FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(setup), FAST(kv_append), FAST(prefix_attn), FAST(beam_select), FAST(beam_reorder), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged() { return PyModule_Create(&module); }
