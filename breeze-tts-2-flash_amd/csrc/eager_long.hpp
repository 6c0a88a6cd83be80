// The long-cache operators of the native eager binding (include/bz_long_cache.h), part of eager_ext.cpp: argument checks,
// output allocation, device switch, stream and workspace lookup and the C ABI call in one call from Python. An attention
// call whose stream has no workspace yet returns what it needs (a tuple); the Python side makes it (outside any graph
// memory pool), registers it and calls again.
#pragma once

#include <array>

#include "bz_long_cache.h"

namespace {

using WindowFn = int (*)(const bz_gqa_window_args*, hipStream_t);
using Kv4Fn = int (*)(const bz_gqa_kv4_args*, hipStream_t);
using TrackedFn = int (*)(const bz_gqa_tracked_args*, hipStream_t);
using LongSizeFn = int (*)(int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
                           size_t*);
using StoreFn = int (*)(const void*, const void*, int64_t, int64_t, int64_t, int32_t, const int32_t*, const int32_t*,
                        const bz_kv4_cache*, hipStream_t);
using LoadFn = int (*)(const bz_kv4_cache*, const int32_t*, int32_t, void*, void*, int64_t, int64_t, int64_t, hipStream_t);
using SelectFn = int (*)(const bz_kv_select_args*, hipStream_t);
using CompactFn = int (*)(const bz_kv_tensor*, int32_t, const int32_t*, const int32_t*, int32_t, int32_t, int32_t, int32_t,
                          hipStream_t);

WindowFn g_window = nullptr;
Kv4Fn g_kv4 = nullptr;
TrackedFn g_tracked = nullptr;
LongSizeFn g_long_size = nullptr;
StoreFn g_store = nullptr;
LoadFn g_load = nullptr;
SelectFn g_select = nullptr;
CompactFn g_compact = nullptr;

// (device, raw stream, kind, sharing) -> workspace. Sharing: calls that find the counters of a workspace where others leave them
// zero (sharing_of).
using LongKey = std::array<int64_t, 4>;
std::map<LongKey, at::Tensor> g_long_ws;
std::map<std::array<int64_t, 12>, size_t> g_long_bytes;

// check() for messages that need no building: nothing is allocated where the condition holds.
inline void require(bool cond, const char* msg) {
  if (__builtin_expect(!cond, 0)) throw Error{msg};
}

// An int32 argument (window, sinks, ...), not negative.
int32_t int_arg(PyObject* o, const char* name, bool zero = true) {
  const long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Error{std::string(name) + " must be an int"};
  }
  if (x < (zero ? 0 : 1) || x > INT32_MAX) throw Error{std::string(name) + " is out of range, got " + std::to_string(x)};
  return (int32_t)x;
}
float float_arg(PyObject* o, const char* name) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Error{std::string(name) + " must be a number"};
  }
  return (float)x;
}

const int32_t* rows_arg(PyObject* o, int64_t B, const char* name, const at::Device& dev) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != at::kInt || t.device() != dev || t.numel() != B || !t.is_contiguous())
    throw Error{std::string(name) + " must be a contiguous int32 device tensor of " + std::to_string(B) + " elements"};
  return t.data_ptr<int32_t>();
}
const int32_t* rows_or_null(PyObject* o, int64_t B, const char* name, const at::Device& dev) {
  return o == Py_None ? nullptr : rows_arg(o, B, name, dev);
}

// Whether K and V have one shape and the same steps in every dim of more than one element (a single token's keys, rotated, and
// values, as the projection left them, differ in the step between tokens, which no access uses).
bool alike(const at::Tensor& k, const at::Tensor& v) {
  const auto sz = k.sizes(), a = k.strides(), b = v.strides();
  if (v.sizes() != sz) return false;
  for (size_t i = 0; i < sz.size(); ++i)
    if (sz[i] > 1 && a[i] != b[i]) return false;
  return true;
}

// Whether no two elements of t share a place because of a broadcast dim.
bool one_place_each(const at::Tensor& t) {
  const auto sz = t.sizes(), st = t.strides();
  for (size_t i = 0; i < sz.size(); ++i)
    if (st[i] == 0 && sz[i] > 1) return false;
  return true;
}

// The query's, ranges' and output's part of a call's arguments. out: the caller's or nullptr (then out_shape is what to
// allocate).
void fill_query(const at::Tensor& q, const at::Tensor* out, PyObject* seq_lens, PyObject* kv_start, PyObject* scale,
                PyObject* num_splits, PyObject* max_seq_len, bz_gqa_decode_args& a, std::array<int64_t, 4>& out_shape,
                int& out_dims) {
  require(q.is_cuda(), "query must be a device tensor");
  require(q.scalar_type() == at::kBFloat16, "query must be bf16");
  const int nd = (int)q.dim();
  if (nd != 3 && nd != 4) throw Error{"query must be [B, NH, D] or [B, NH, T, D], got shape " + shape_str(q)};
  const auto sz = q.sizes(), st = q.strides();
  require(st[nd - 1] == 1, "query's head_dim must be contiguous");
  const int64_t B = sz[0], NH = sz[1], T = nd == 4 ? sz[2] : 1, D = sz[nd - 1];
  require(B > 0 && NH > 0 && T > 0 && B <= INT32_MAX && NH <= INT32_MAX && T <= INT32_MAX && D <= INT32_MAX,
          "query must not be empty");
  a.q = q.data_ptr();
  a.q_stride_b = st[0], a.q_stride_h = st[1], a.q_stride_t = nd == 4 ? st[2] : 0;
  a.batch = (int32_t)B, a.num_q_heads = (int32_t)NH, a.tokens_per_row = (int32_t)T, a.head_dim = (int32_t)D;
  if (out == nullptr) {
    out_dims = T == 1 ? 3 : 4;
    out_shape = T == 1 ? std::array<int64_t, 4>{B, NH, D, 1} : std::array<int64_t, 4>{B, T, NH, D};
    a.out_stride_b = T * NH * D, a.out_stride_t = NH * D, a.out_stride_h = D;
  } else {
    const at::Tensor& o = *out;
    require(o.device() == q.device(), "out must be on the query's device");
    require(o.scalar_type() == at::kBFloat16, "out must be bf16");
    require(o.dim() >= 1 && o.stride(-1) == 1, "out's last dimension must be contiguous");
    if (o.dim() == 4 && o.size(0) == B && o.size(1) == T && o.size(2) == NH && o.size(3) == D) {
      a.out_stride_b = o.stride(0), a.out_stride_h = o.stride(2), a.out_stride_t = o.stride(1);
    } else if (o.dim() == 4 && o.size(0) == B && o.size(1) == NH && o.size(2) == T && o.size(3) == D) {
      a.out_stride_b = o.stride(0), a.out_stride_h = o.stride(1), a.out_stride_t = o.stride(2);
    } else if (T == 1 && o.dim() == 3 && o.size(0) == B && o.size(1) == NH && o.size(2) == D) {
      a.out_stride_b = o.stride(0), a.out_stride_h = o.stride(1), a.out_stride_t = 0;
    } else {
      throw Error{"out must be [B, T, NH, D], [B, NH, T, D] or (T = 1) [B, NH, D] with B=" + std::to_string(B) +
                  ", T=" + std::to_string(T) + ", NH=" + std::to_string(NH) + ", D=" + std::to_string(D)};
    }
    require(one_place_each(o), "out must not be a broadcast view");
    a.out = o.data_ptr();
  }
  a.seq_lens = rows_arg(seq_lens, B, "seq_lens", q.device());
  a.kv_start = rows_or_null(kv_start, B, "kv_start", q.device());
  a.scale = float_arg(scale, "scale");
  a.num_splits = int_arg(num_splits, "num_splits");
  a.max_seq_len = int_arg(max_seq_len, "max_seq_len");
}

void fill_bf16_cache(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, bz_gqa_decode_args& a) {
  require(k.scalar_type() == at::kBFloat16 && v.scalar_type() == at::kBFloat16, "k_cache and v_cache must be bf16");
  require(k.device() == q.device() && v.device() == q.device(), "all tensors must be on one device");
  require(k.dim() == 4 && alike(k, v),
          "k_cache and v_cache must be [B, NKV, capacity, D] with equal shapes and strides");
  const auto sz = k.sizes(), st = k.strides();
  if (sz[0] != a.batch || sz[3] != a.head_dim || st[3] != 1)
    throw Error{"k_cache " + shape_str(k) + " does not match query " + shape_str(q)};
  require(sz[1] <= INT32_MAX && sz[2] <= INT32_MAX, "k_cache is too large");
  a.k_cache = k.data_ptr(), a.v_cache = v.data_ptr();
  a.kv_stride_b = st[0], a.kv_stride_h = st[1], a.kv_stride_s = st[2];
  a.num_kv_heads = (int32_t)sz[1], a.capacity = (int32_t)sz[2];
}

// bz_kv4_cache of the four tensors k, v, k_scale, v_scale; their device.
at::Device fill_kv4(PyObject* const* t, bz_kv4_cache& c) {
  const at::Tensor &k = tensor(t[0], "k"), &v = tensor(t[1], "v"), &ks = tensor(t[2], "k_scale"), &vs = tensor(t[3], "v_scale");
  const at::Device dev = k.device();
  for (const at::Tensor* x : {&k, &v, &ks, &vs})
    require(x->is_cuda() && x->scalar_type() == at::kByte && x->dim() == 4 && x->device() == dev,
            "a 4-bit cache is four uint8 device tensors [B, NKV, capacity, ..] on one device");
  const auto sz = k.sizes(), st = k.strides(), zs = ks.sizes(), ts = ks.strides();
  const int64_t D = 2 * sz[3];
  require(alike(k, v) && st[3] == 1,
          "codes k and v must have equal shapes and strides and a contiguous last dim");
  require(zs[0] == sz[0] && zs[1] == sz[1] && zs[2] == sz[2] && zs[3] == D / 32 && alike(ks, vs),
          "scales must be [B, NKV, capacity, D / 32] with equal strides");
  require(ts[3] == 1 && ts[2] == D / 32, "the last two dims of the scales must be contiguous");
  for (int i = 0; i < 4; ++i) require(sz[i] <= INT32_MAX / 2, "the 4-bit cache is too large");
  c.k = k.data_ptr(), c.v = v.data_ptr(), c.k_scale = ks.data_ptr(), c.v_scale = vs.data_ptr();
  c.stride_b = st[0], c.stride_h = st[1], c.stride_s = st[2];
  c.scale_stride_b = ts[0], c.scale_stride_h = ts[1];
  c.batch = (int32_t)sz[0], c.num_kv_heads = (int32_t)sz[1], c.capacity = (int32_t)sz[2], c.head_dim = (int32_t)D;
  return dev;
}

// 0 for calls of few units, whose counters have one room for all; 1 for the chunks of bz_gqa_window beyond (more units than the
// device has CUs: the chunk kernel, which has no counters and writes what it reads); else the room, a power of two of units.
int64_t sharing_of(int kind, const bz_gqa_decode_args& a) {
  const int64_t group = a.num_q_heads / std::max(a.num_kv_heads, 1), T = a.tokens_per_row;
  const int64_t tpt = std::min<int64_t>(T, 16 / std::max<int64_t>(std::min<int64_t>(group, 16), 1)), tiles = (T + tpt - 1) / tpt;
  const int64_t units = a.batch * tiles * a.num_kv_heads;
  if (units <= BZ_LONG_SHARED_UNITS) return 0;
  if (kind == BZ_LONG_WINDOW && tiles > 1) return 1;
  int64_t room = BZ_LONG_SHARED_UNITS;
  while (room < units) room *= 2;
  return room;
}

// The workspace of an attention call into a; true if there is one or none is needed. Otherwise `need` is the tuple the
// Python side makes one from (a call under capture raises instead: nothing is allocated then).
bool long_workspace(int kind, int idx, hipStream_t stream, int window, int sinks, const at::Tensor* given, const at::Device& dev,
                    bz_gqa_decode_args& a, PyObject** need) {
  if (given != nullptr) {
    require(given->device() == dev && given->is_contiguous(), "workspace must be a contiguous tensor on the query's device");
    a.workspace = given->data_ptr();
    a.workspace_bytes = (size_t)given->numel() * given->element_size();
    return true;
  }
  const std::array<int64_t, 12> sizes{idx,        kind,   a.batch, a.num_q_heads, a.num_kv_heads, a.head_dim, a.capacity,
                                      a.tokens_per_row, window, sinks,   a.num_splits,  a.max_seq_len};
  auto it = g_long_bytes.find(sizes);
  if (it == g_long_bytes.end()) {
    size_t n = 0;
    check_status(g_long_size(kind, a.batch, a.num_q_heads, a.num_kv_heads, a.head_dim, a.capacity, a.tokens_per_row, window,
                             sinks, a.num_splits, a.max_seq_len, &n),
                 "bz_long_workspace_size");
    if (g_long_bytes.size() >= 4096) g_long_bytes.clear();
    it = g_long_bytes.emplace(sizes, n).first;
  }
  if (it->second == 0) return true;
  if (capturing(stream))
    throw Error{"a call being captured into a graph needs workspace= (long_workspace(...), made before the capture; " +
                std::to_string(it->second) + " bytes): graphs that shared the stream's own could not run at the same time"};
  const LongKey key{idx, (int64_t)reinterpret_cast<uintptr_t>(stream), kind, sharing_of(kind, a)};
  auto ws = g_long_ws.find(key);
  if (ws != g_long_ws.end() && (size_t)ws->second.numel() >= it->second) {
    a.workspace = ws->second.data_ptr();
    a.workspace_bytes = (size_t)ws->second.numel();
    return true;
  }
  *need = Py_BuildValue("(LLLLn)", (long long)key[0], (long long)key[1], (long long)key[2], (long long)key[3],
                        (Py_ssize_t)it->second);
  return false;
}

// register_long_workspace(device, stream, kind, sharing, workspace)
PyObject* register_long_workspace(PyObject*, PyObject* args) {
  long long k[4];
  PyObject* o;
  if (!PyArg_ParseTuple(args, "LLLLO", &k[0], &k[1], &k[2], &k[3], &o)) return nullptr;
  if (!THPVariable_Check(o)) {
    PyErr_SetString(PyExc_TypeError, "register_long_workspace: a tensor expected");
    return nullptr;
  }
  g_long_ws[LongKey{k[0], k[1], k[2], k[3]}] = THPVariable_Unpack(o);
  Py_RETURN_NONE;
}

at::Tensor make_out(const at::Tensor* out, const std::array<int64_t, 4>& shape, int dims, const at::Tensor& q,
                    bz_gqa_decode_args& a) {
  if (out != nullptr) return *out;
  at::Tensor t = at::empty(at::IntArrayRef(shape.data(), dims), q.options());
  a.out = t.data_ptr();
  return t;
}

// Runs body, turning errors into RuntimeError.
template <class F>
PyObject* guarded(const char* name, Py_ssize_t nargs, Py_ssize_t want, F body) {
  if (!bound()) return nullptr;
  if (nargs != want) {
    PyErr_Format(PyExc_TypeError, "%s() takes %zd arguments", name, want);
    return nullptr;
  }
  try {
    return body();
  } catch (const Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.msg.c_str());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// window(q, k_cache, v_cache, seq_lens, scale, window, out, sinks, kv_start, num_splits, max_seq_len, workspace) -> out, or
// the tuple of long_workspace
PyObject* window(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("window", nargs, 12, [&]() -> PyObject* {
    const at::Tensor &q = tensor(args[0], "query"), &k = tensor(args[1], "k_cache"), &v = tensor(args[2], "v_cache");
    const at::Tensor* out = tensor_or_none(args[6], "out");
    const at::Tensor* ws = tensor_or_none(args[11], "workspace");
    bz_gqa_window_args w{};
    std::array<int64_t, 4> shape;
    int dims = 0;
    fill_query(q, out, args[3], args[8], args[4], args[9], args[10], w.base, shape, dims);
    fill_bf16_cache(q, k, v, w.base);
    w.window = int_arg(args[5], "window"), w.sinks = int_arg(args[7], "sinks");
    const int idx = q.device().index();
    DeviceScope scope(idx);
    hipStream_t stream = c10::hip::getCurrentHIPStream(idx).stream();
    PyObject* need = nullptr;
    if (!long_workspace(BZ_LONG_WINDOW, idx, stream, w.window, w.sinks, ws, q.device(), w.base, &need)) return need;
    at::Tensor t = make_out(out, shape, dims, q, w.base);
    check_status(g_window(&w, stream), "bz_gqa_window");
    return result(args[6], t);
  });
}

// kv4(q, k, v, k_scale, v_scale, seq_lens, scale, out, kv_start, window, sinks, num_splits, max_seq_len, workspace) -> out,
// or the tuple of long_workspace
PyObject* kv4(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("kv4", nargs, 14, [&]() -> PyObject* {
    const at::Tensor& q = tensor(args[0], "query");
    const at::Tensor* out = tensor_or_none(args[7], "out");
    const at::Tensor* ws = tensor_or_none(args[13], "workspace");
    bz_gqa_kv4_args ka{};
    std::array<int64_t, 4> shape;
    int dims = 0;
    fill_query(q, out, args[5], args[8], args[6], args[11], args[12], ka.base, shape, dims);
    require(fill_kv4(args + 1, ka.cache) == q.device(), "all tensors must be on one device");
    if (ka.cache.batch != ka.base.batch || ka.cache.head_dim != ka.base.head_dim)
      throw Error{"a cache of batch " + std::to_string(ka.cache.batch) + " and head_dim " + std::to_string(ka.cache.head_dim) +
                  " does not match query " + shape_str(q)};
    ka.base.num_kv_heads = ka.cache.num_kv_heads, ka.base.capacity = ka.cache.capacity;
    ka.window = int_arg(args[9], "window"), ka.sinks = int_arg(args[10], "sinks");
    const int idx = q.device().index();
    DeviceScope scope(idx);
    hipStream_t stream = c10::hip::getCurrentHIPStream(idx).stream();
    PyObject* need = nullptr;
    if (!long_workspace(BZ_LONG_KV4, idx, stream, ka.window, ka.sinks, ws, q.device(), ka.base, &need)) return need;
    at::Tensor t = make_out(out, shape, dims, q, ka.base);
    check_status(g_kv4(&ka, stream), "bz_gqa_decode_kv4");
    return result(args[7], t);
  });
}

// First and one-past-last byte of a tensor's elements.
std::pair<uintptr_t, uintptr_t> span_of(const at::Tensor& t) {
  const auto sz = t.sizes(), st = t.strides();
  int64_t last = 0;
  for (size_t i = 0; i < sz.size(); ++i) {
    if (sz[i] == 0) return {0, 0};
    last += (sz[i] - 1) * st[i];
  }
  const uintptr_t p = reinterpret_cast<uintptr_t>(t.data_ptr());
  return {p, p + (uintptr_t)((last + 1) * (int64_t)t.element_size())};
}

// One dim of two tensors whose steps in it are alike: the step in bytes and the sizes.
struct SharedDim {
  int64_t step, nx, ny;
};
// Whether a block of x and one of y meet, for some indices of the dims from `d` on: y's lies diff + sum (j_y - j_x) step bytes
// behind x's, and they hold ex and ey bytes.
bool blocks_meet(const SharedDim* d, int dims, int64_t diff, int64_t ex, int64_t ey) {
  if (dims == 0) return diff < ex && diff > -ey;
  if (d->step == 0) return blocks_meet(d + 1, dims - 1, diff, ex, ey);
  int64_t below = ey, above = ex;  // what the inner dims can still move the blocks by
  for (int i = 1; i < dims; ++i) below += (d[i].ny - 1) * d[i].step, above += (d[i].nx - 1) * d[i].step;
  const auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
  const int64_t lo = std::max(1 - d->nx, floor_div(-below - diff, d->step) + 1);
  const int64_t hi = std::min(d->ny - 1, -floor_div(diff - above, d->step) - 1);
  if (hi - lo > 8) return true;  // steps that do not nest: taken to meet
  for (int64_t j = lo; j <= hi; ++j)
    if (blocks_meet(d + 1, dims - 1, diff + j * d->step, ex, ey)) return true;
  return false;
}

// Whether two tensors share no memory: their spans lie apart, or they are views of one tensor side by side in one of its dims (a
// cache that holds K and V in turns by batch row, head or position). Their largest steps, as far as both have the same ones, run
// over blocks that the smaller ones fill; no two of those may meet. Where that cannot be shown they are taken to share some.
bool apart(const at::Tensor& x, const at::Tensor& y) {
  const auto a = span_of(x), b = span_of(y);
  if (a.second <= b.first || b.second <= a.first) return true;
  if (x.dim() != y.dim() || x.dim() > 8) return false;
  const int64_t sx = x.element_size(), sy = y.element_size();
  int order[8], dims = 0;
  for (int i = 0; i < x.dim(); ++i)
    if (x.size(i) > 1 || y.size(i) > 1) order[dims++] = i;
  std::stable_sort(order, order + dims, [&](int i, int j) { return x.stride(i) * sx > x.stride(j) * sx; });
  SharedDim outer[8];
  for (int n = 0; n < dims; ++n) {
    const int i = order[n];
    if (x.stride(i) * sx != y.stride(i) * sy) return false;
    outer[n] = {x.stride(i) * sx, x.size(i), y.size(i)};
    int64_t ex = sx, ey = sy;
    for (int m = n + 1; m < dims; ++m) {
      ex += (x.size(order[m]) - 1) * x.stride(order[m]) * sx;
      ey += (y.size(order[m]) - 1) * y.stride(order[m]) * sy;
    }
    if (!blocks_meet(outer, n + 1, (int64_t)(b.first - a.first), ex, ey)) return true;
  }
  return false;
}

// apart(x, y) for tests, on tensors of any device
PyObject* apart_py(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("apart", nargs, 2, [&]() -> PyObject* {
    return PyBool_FromLong(apart(tensor(args[0], "x"), tensor(args[1], "y")));
  });
}

// dst is src itself (the same elements), or shares none of its memory; every element has a place of its own.
void check_destination(const at::Tensor& src, const at::Tensor& dst, const char* name) {
  for (int64_t i = 0; i < dst.dim(); ++i)
    if (dst.stride(i) <= 0 && dst.size(i) != 1) throw Error{std::string(name) + " must not be a broadcast view"};
  if (dst.data_ptr() == src.data_ptr() && dst.strides() == src.strides()) return;
  if (!apart(src, dst)) throw Error{std::string(name) + " must be its source itself or not overlap it"};
}

void weights_view(const at::Tensor& t, int64_t B, int64_t NKV, int64_t cap, const char* name, const at::Device& dev) {
  if (t.scalar_type() != at::kFloat || t.device() != dev || t.dim() != 3 || t.size(0) != B || t.size(1) != NKV ||
      t.size(2) != cap || t.stride(2) != 1)
    throw Error{std::string(name) + " must be float32 [B, NKV, capacity] = (" + std::to_string(B) + ", " + std::to_string(NKV) +
                ", " + std::to_string(cap) + ") on the cache's device, its last dim contiguous"};
}

// tracked(q, k_cache, v_cache, seq_lens, scale, weights, out, decay, weights_out, kv_start, num_splits, max_seq_len, workspace)
// -> out, or the tuple of long_workspace
PyObject* tracked(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("tracked", nargs, 13, [&]() -> PyObject* {
    const at::Tensor &q = tensor(args[0], "query"), &k = tensor(args[1], "k_cache"), &v = tensor(args[2], "v_cache"),
                     &w = tensor(args[5], "weights"), &wo = tensor(args[8], "weights_out");
    const at::Tensor* out = tensor_or_none(args[6], "out");
    const at::Tensor* ws = tensor_or_none(args[12], "workspace");
    bz_gqa_tracked_args ta{};
    bz_gqa_decode_args& a = ta.base;
    std::array<int64_t, 4> shape;
    int dims = 0;
    fill_query(q, out, args[3], args[9], args[4], args[10], args[11], a, shape, dims);
    require(a.tokens_per_row == 1, "gqa_decode_tracked takes one query token per row");
    fill_bf16_cache(q, k, v, a);
    weights_view(w, a.batch, a.num_kv_heads, a.capacity, "weights", q.device());
    weights_view(wo, a.batch, a.num_kv_heads, a.capacity, "weights_out", q.device());
    check_destination(w, wo, "weights_out");
    ta.weights = w.data_ptr<float>(), ta.w_stride_b = w.stride(0), ta.w_stride_h = w.stride(1);
    ta.weights_out = wo.data_ptr<float>(), ta.wo_stride_b = wo.stride(0), ta.wo_stride_h = wo.stride(1);
    ta.decay = float_arg(args[7], "decay");
    const int idx = q.device().index();
    DeviceScope scope(idx);
    hipStream_t stream = c10::hip::getCurrentHIPStream(idx).stream();
    PyObject* need = nullptr;
    if (!long_workspace(BZ_LONG_TRACKED, idx, stream, 0, 0, ws, q.device(), a, &need)) return need;
    at::Tensor t = make_out(out, shape, dims, q, a);
    check_status(g_tracked(&ta, stream), "bz_gqa_decode_tracked");
    return result(args[6], t);
  });
}

void check_kv(const at::Tensor& k, const at::Tensor& v, const bz_kv4_cache& c, const at::Device& dev) {
  require(k.scalar_type() == at::kBFloat16 && v.scalar_type() == at::kBFloat16 && k.device() == dev && v.device() == dev,
          "k and v must be bf16 on the cache's device");
  require(k.dim() == 4 && alike(k, v) && k.stride(3) == 1,
          "k and v must be [B, NKV, T, D] with equal shapes and strides and a contiguous last dim");
  if (k.size(0) != c.batch || k.size(1) != c.num_kv_heads || k.size(3) != c.head_dim)
    throw Error{"k " + shape_str(k) + " does not match a cache of batch " + std::to_string(c.batch) + ", " +
                std::to_string(c.num_kv_heads) + " heads, head_dim " + std::to_string(c.head_dim)};
  require(k.size(2) <= INT32_MAX, "too many tokens");
}

// kv4_store(k, v, ck, cv, k_scale, v_scale, slots, counts)
PyObject* kv4_store(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("kv4_store", nargs, 8, [&]() -> PyObject* {
    const at::Tensor &k = tensor(args[0], "k"), &v = tensor(args[1], "v");
    bz_kv4_cache c{};
    const at::Device dev = fill_kv4(args + 2, c);
    check_kv(k, v, c, dev);
    std::pair<uintptr_t, uintptr_t> span[4];  // (each worked out once: six calls of apart cost a decode step 0.4 us)
    for (int i = 0; i < 4; ++i) {
      const at::Tensor& t = THPVariable_Unpack(args[2 + i]);
      require(one_place_each(t), "a cache that is written must not be a broadcast view");
      span[i] = span_of(t);
      for (int j = 0; j < i; ++j)
        require(span[i].second <= span[j].first || span[j].second <= span[i].first || apart(t, THPVariable_Unpack(args[2 + j])),
                "the tensors of a cache that is written must not overlap one another");
    }
    const int32_t *slots = rows_arg(args[6], c.batch, "slots", dev), *counts = rows_or_null(args[7], c.batch, "counts", dev);
    const int idx = dev.index();
    DeviceScope scope(idx);
    check_status(g_store(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), (int32_t)k.size(2), slots, counts,
                         &c, c10::hip::getCurrentHIPStream(idx).stream()),
                 "bz_kv4_store");
    Py_RETURN_NONE;
  });
}

// kv4_load(ck, cv, k_scale, v_scale, slots, tokens, k, v) -> (k, v); k, v None: allocated
PyObject* kv4_load(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("kv4_load", nargs, 8, [&]() -> PyObject* {
    bz_kv4_cache c{};
    const at::Device dev = fill_kv4(args, c);
    const int32_t* slots = rows_arg(args[4], c.batch, "slots", dev);
    const int32_t tokens = int_arg(args[5], "tokens", false);
    const at::Tensor *kg = tensor_or_none(args[6], "k"), *vg = tensor_or_none(args[7], "v");
    require((kg == nullptr) == (vg == nullptr), "kv4_load takes both outputs or neither");
    const int idx = dev.index();
    DeviceScope scope(idx);
    const auto options = at::TensorOptions().dtype(at::kBFloat16).device(dev);
    at::Tensor k = kg ? *kg : at::empty({c.batch, c.num_kv_heads, tokens, c.head_dim}, options);
    at::Tensor v = vg ? *vg : at::empty({c.batch, c.num_kv_heads, tokens, c.head_dim}, options);
    check_kv(k, v, c, dev);
    require(k.size(2) == tokens, "the outputs must hold as many tokens as are asked for");
    if (kg != nullptr) {
      require(one_place_each(k) && one_place_each(v), "an output must not be a broadcast view");
      require(apart(k, v), "the outputs must not overlap one another");
    }
    check_status(g_load(&c, slots, tokens, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2),
                        c10::hip::getCurrentHIPStream(idx).stream()),
                 "bz_kv4_load");
    PyObject *pk = result(args[6], k), *pv = result(args[7], v);
    PyObject* r = pk && pv ? PyTuple_Pack(2, pk, pv) : nullptr;
    Py_XDECREF(pk);
    Py_XDECREF(pv);
    return r;
  });
}

// The select part of an eviction into a; index and lens: the caller's, or allocated here.
void fill_select(PyObject* const* args, bz_kv_select_args& a, at::Tensor& index, at::Tensor& lens) {
  const at::Tensor& w = tensor(args[0], "weights");
  require(w.is_cuda() && w.dim() == 3, "weights must be a device tensor [B, NKV, capacity]");
  const at::Device dev = w.device();
  const int64_t B = w.size(0), NKV = w.size(1), cap = w.size(2);
  require(B <= INT32_MAX && NKV <= INT32_MAX && cap <= INT32_MAX, "weights is too large");
  weights_view(w, B, NKV, cap, "weights", dev);
  a.weights = w.data_ptr<float>(), a.w_stride_b = w.stride(0), a.w_stride_h = w.stride(1);
  a.seq_lens = rows_arg(args[1], B, "seq_lens", dev);
  a.keep = int_arg(args[2], "keep"), a.sinks = int_arg(args[3], "sinks"), a.recent = int_arg(args[4], "recent");
  if (a.keep < 1 || a.keep > cap || (int64_t)a.sinks + a.recent > a.keep)
    throw Error{"keep must be 1 to the capacity and at least sinks + recent, got " + std::to_string(a.keep)};
  a.kv_start = rows_or_null(args[5], B, "kv_start", dev);
  const at::Tensor *ig = tensor_or_none(args[6], "index"), *lg = tensor_or_none(args[7], "lens");
  const auto options = at::TensorOptions().dtype(at::kInt).device(dev);
  index = ig ? *ig : at::empty({B, NKV, a.keep}, options);
  lens = lg ? *lg : at::empty({B}, options);
  if (index.scalar_type() != at::kInt || index.device() != dev || index.dim() != 3 || index.size(0) != B ||
      index.size(1) != NKV || index.size(2) != a.keep || !index.is_contiguous())
    throw Error{"index must be a contiguous int32 [B, NKV, keep] = (" + std::to_string(B) + ", " + std::to_string(NKV) + ", " +
                std::to_string(a.keep) + ") device tensor"};
  if (lg) rows_arg(args[7], B, "lens", dev);
  a.index = index.data_ptr<int32_t>(), a.lens = lens.data_ptr<int32_t>();
  if (const at::Tensor* wo = tensor_or_none(args[8], "weights_out")) {
    weights_view(*wo, B, NKV, cap, "weights_out", dev);
    check_destination(w, *wo, "weights_out");
    a.weights_out = wo->data_ptr<float>(), a.wo_stride_b = wo->stride(0), a.wo_stride_h = wo->stride(1);
  }
  a.batch = (int32_t)B, a.num_kv_heads = (int32_t)NKV, a.capacity = (int32_t)cap;
}

struct Tensors {
  int num = 0;
  at::Tensor src[BZ_KV_TENSORS], dst[BZ_KV_TENSORS];
  bz_kv_tensor t[BZ_KV_TENSORS] = {};
};

// The compaction of a sequence of tensors (outs None: in place).
void fill_compact(PyObject* tensors, PyObject* outs, int64_t B, int64_t NKV, int64_t cap, const at::Device& dev, Tensors& m) {
  PyObject* ts = PySequence_Fast(tensors, "tensors must be a sequence");
  PyObject* os = outs == Py_None ? ts : PySequence_Fast(outs, "outs must be a sequence");
  const Py_ssize_t n = ts ? PySequence_Fast_GET_SIZE(ts) : 0;
  const bool ok = ts && os && n > 0 && n <= BZ_KV_TENSORS && PySequence_Fast_GET_SIZE(os) == n;
  bool all = ok;
  if (ok) {
    m.num = (int)n;
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject *s = PySequence_Fast_GET_ITEM(ts, i), *d = PySequence_Fast_GET_ITEM(os, i);
      if (!THPVariable_Check(s) || !THPVariable_Check(d)) {
        all = false;
        break;
      }
      m.src[i] = THPVariable_Unpack(s), m.dst[i] = THPVariable_Unpack(d);
    }
  }
  if (os != ts) Py_XDECREF(os);
  Py_XDECREF(ts);
  PyErr_Clear();
  require(all, "kv_compact takes one to 4 tensors and as many outputs");
  for (int i = 0; i < m.num; ++i) {
    const at::Tensor &s = m.src[i], &d = m.dst[i];
    require(s.is_cuda() && s.dim() == 4 && s.size(0) == B && s.size(1) == NKV && s.size(2) == cap && s.device() == dev &&
                s.stride(3) == 1 && s.size(3) > 0,
            "tensors must be [B, NKV, capacity, X] on one device with a contiguous last dim");
    require(d.sizes() == s.sizes() && d.scalar_type() == s.scalar_type() && d.device() == dev && d.stride(3) == 1,
            "an output must match its tensor");
    check_destination(s, d, "an output");
    for (int j = 0; j < m.num; ++j)
      if (j != i) require(apart(m.src[j], d) && apart(m.dst[j], d), "an output must not overlap another tensor");
    const int64_t e = s.element_size();
    require(s.size(3) * e <= INT32_MAX, "a row is too large");
    bz_kv_tensor& t = m.t[i];
    t.src = s.data_ptr(), t.dst = d.data_ptr(), t.row_bytes = (int32_t)(s.size(3) * e);
    t.src_stride_b = e * s.stride(0), t.src_stride_h = e * s.stride(1), t.src_stride_s = e * s.stride(2);
    t.dst_stride_b = e * d.stride(0), t.dst_stride_h = e * d.stride(1), t.dst_stride_s = e * d.stride(2);
  }
}

PyObject* index_and_lens(PyObject* const* args, const at::Tensor& index, const at::Tensor& lens) {
  PyObject *pi = result(args[6], index), *pl = result(args[7], lens);
  PyObject* r = pi && pl ? PyTuple_Pack(2, pi, pl) : nullptr;
  Py_XDECREF(pi);
  Py_XDECREF(pl);
  return r;
}

// select(weights, seq_lens, keep, sinks, recent, kv_start, index, lens, weights_out) -> (index, lens)
PyObject* select(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("select", nargs, 9, [&]() -> PyObject* {
    bz_kv_select_args a{};
    at::Tensor index, lens;
    fill_select(args, a, index, lens);
    const int idx = index.device().index();
    DeviceScope scope(idx);
    check_status(g_select(&a, c10::hip::getCurrentHIPStream(idx).stream()), "bz_kv_select");
    return index_and_lens(args, index, lens);
  });
}

// compact(tensors, index, lens, outs)
PyObject* compact(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("compact", nargs, 4, [&]() -> PyObject* {
    const at::Tensor& index = tensor(args[1], "index");
    require(index.is_cuda() && index.scalar_type() == at::kInt && index.dim() == 3 && index.is_contiguous(),
            "index must be a contiguous int32 [B, NKV, keep] device tensor");
    const at::Device dev = index.device();
    const int64_t B = index.size(0), NKV = index.size(1), keep = index.size(2);
    require(B <= INT32_MAX && NKV <= INT32_MAX && keep <= INT32_MAX, "index is too large");
    const int32_t* lens = rows_arg(args[2], B, "lens", dev);
    PyObject* first = PySequence_Check(args[0]) && PySequence_Size(args[0]) > 0 ? PySequence_GetItem(args[0], 0) : nullptr;
    PyErr_Clear();
    const int64_t cap = first && THPVariable_Check(first) && THPVariable_Unpack(first).dim() == 4
                            ? THPVariable_Unpack(first).size(2)
                            : -1;
    Py_XDECREF(first);
    require(cap >= 0 && cap <= INT32_MAX, "kv_compact takes one to 4 tensors [B, NKV, capacity, X]");
    Tensors m;
    fill_compact(args[0], args[3], B, NKV, cap, dev, m);
    const int idx = dev.index();
    DeviceScope scope(idx);
    check_status(g_compact(m.t, m.num, index.data_ptr<int32_t>(), lens, (int32_t)B, (int32_t)NKV, (int32_t)cap, (int32_t)keep,
                           c10::hip::getCurrentHIPStream(idx).stream()),
                 "bz_kv_compact");
    Py_RETURN_NONE;
  });
}

// evict(weights, seq_lens, keep, sinks, recent, kv_start, index, lens, weights_out, tensors, outs) -> (index, lens): both of
// the above, everything checked before anything runs
PyObject* evict(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("evict", nargs, 11, [&]() -> PyObject* {
    bz_kv_select_args a{};
    at::Tensor index, lens;
    fill_select(args, a, index, lens);
    Tensors m;
    fill_compact(args[9], args[10], a.batch, a.num_kv_heads, a.capacity, index.device(), m);
    if (const at::Tensor* wo = tensor_or_none(args[8], "weights_out")) {  // written by the selection, before the tensors move
      const auto span = span_of(*wo);
      const auto clear = [&](const at::Tensor& t) {  // (the view only where the spans meet: 0.2 us of host time)
        const auto other = span_of(t);
        return other.second <= span.first || span.second <= other.first || apart(t, wo->unsqueeze(-1));
      };
      for (int i = 0; i < m.num; ++i)
        require(clear(m.src[i]) && clear(m.dst[i]), "weights_out is compacted with the tensors and must not overlap one of them");
    }
    const int idx = index.device().index();
    DeviceScope scope(idx);
    hipStream_t stream = c10::hip::getCurrentHIPStream(idx).stream();
    check_status(g_select(&a, stream), "bz_kv_select");
    check_status(g_compact(m.t, m.num, a.index, a.lens, a.batch, a.num_kv_heads, a.capacity, a.keep, stream), "bz_kv_compact");
    return index_and_lens(args, index, lens);
  });
}

// bind_long(window, kv4, tracked, workspace_size, store, load, select, compact): the C ABI functions' addresses
PyObject* bind_long(PyObject*, PyObject* args) {
  unsigned long long f[8];
  if (!PyArg_ParseTuple(args, "KKKKKKKK", &f[0], &f[1], &f[2], &f[3], &f[4], &f[5], &f[6], &f[7])) return nullptr;
  g_window = reinterpret_cast<WindowFn>(f[0]);
  g_kv4 = reinterpret_cast<Kv4Fn>(f[1]);
  g_tracked = reinterpret_cast<TrackedFn>(f[2]);
  g_long_size = reinterpret_cast<LongSizeFn>(f[3]);
  g_store = reinterpret_cast<StoreFn>(f[4]);
  g_load = reinterpret_cast<LoadFn>(f[5]);
  g_select = reinterpret_cast<SelectFn>(f[6]);
  g_compact = reinterpret_cast<CompactFn>(f[7]);
  Py_RETURN_NONE;
}

}  // namespace
