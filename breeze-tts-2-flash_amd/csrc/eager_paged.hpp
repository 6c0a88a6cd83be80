// The paged cache's operators of the native eager binding (include/bz_paged_cache.h), part of eager_ext.cpp: argument checks, output
// allocation, device switch, stream and workspace lookup and the C ABI call in one call from Python, as eager_long.hpp does for the
// long cache (whose helpers and workspaces it shares).
#pragma once

#include "bz_paged_cache.h"
#include "eager_long.hpp"

namespace {

using RopeFn = int (*)(const bz_rope_args*, hipStream_t);
using PagedStoreFn = int (*)(const bz_paged_store_args*, hipStream_t);
using PagedLoadFn = int (*)(const bz_paged_cache*, const int32_t*, int32_t, void*, void*, int64_t, int64_t, int64_t, hipStream_t);
using PagedFn = int (*)(const bz_gqa_paged_args*, hipStream_t);
using PagedSizeFn = int (*)(int32_t, int32_t, int32_t, size_t*);

RopeFn g_rope = nullptr;
PagedStoreFn g_paged_store = nullptr;
PagedLoadFn g_paged_load = nullptr;
PagedFn g_paged = nullptr;
PagedSizeFn g_paged_size = nullptr;

constexpr int kPagedKind = 3;  // the kind of its workspaces, next to bz_long_kind's

// The step of a dim, 0 where it has one element (whose step no access uses).
int64_t step_of(const at::Tensor& t, int dim) { return t.size(dim) == 1 ? 0 : t.stride(dim); }

// Tensors that a call writes, and those it reads: each written one shares no memory with any other (but with `same`, where a
// result may take its input's place).
struct Touched {
  const at::Tensor* t[24];
  std::pair<uintptr_t, uintptr_t> span[24];
  const char* name[24];
  int n = 0, written = 0;
  void write(const at::Tensor* x, const char* what) {  // all writes before the first read
    if (x == nullptr) return;
    if (!one_place_each(*x)) throw Error{std::string(what) + " must not be a broadcast view"};
    read(x, what);
    written = n;
  }
  void read(const at::Tensor* x, const char* what) {
    if (x == nullptr || x->numel() == 0) return;
    t[n] = x, span[n] = span_of(*x), name[n] = what;
    ++n;
  }
  void check(const at::Tensor* result = nullptr, const at::Tensor* source = nullptr) const {
    for (int i = 0; i < written; ++i)
      for (int j = i + 1; j < n; ++j) {
        if (span[i].second <= span[j].first || span[j].second <= span[i].first) continue;
        if (t[i] == result && t[j] == source && t[i]->data_ptr() == t[j]->data_ptr() && alike(*t[i], *t[j]) &&
            t[i]->scalar_type() == t[j]->scalar_type())
          continue;
        at::Tensor x = *t[i], y = *t[j];  // (a head's codes and scales side by side differ in their dims)
        while (x.dim() < y.dim()) x = x.unsqueeze(-1);
        while (y.dim() < x.dim()) y = y.unsqueeze(-1);
        if (!apart(x, y)) throw Error{std::string(name[i]) + " must not overlap " + name[j]};
      }
  }
};

// Heads of the batch's tokens: bf16 [N, H, D].
void check_heads(const at::Tensor& x, const char* name, const at::Device& dev) {
  if (x.scalar_type() != at::kBFloat16 || x.device() != dev || x.dim() != 3 || x.size(2) == 0 || x.stride(2) != 1 ||
      x.size(0) > INT32_MAX || x.size(1) > INT32_MAX || x.size(2) > INT32_MAX)
    throw Error{std::string(name) + " must be a bf16 [tokens, heads, head_dim] tensor on the cache's device, head_dim contiguous, got " +
                shape_str(x)};
}
void like_heads(const at::Tensor& x, const char* name, int64_t N, int64_t H, int64_t D, const at::Device& dev) {
  check_heads(x, name, dev);
  if (x.size(0) != N || x.size(1) != H || x.size(2) != D)
    throw Error{std::string(name) + " must be [" + std::to_string(N) + ", " + std::to_string(H) + ", " + std::to_string(D) +
                "], got " + shape_str(x)};
}

// The cache k, v, k_scale, v_scale (args[0 .. 3]) and its page table (args[4]).
at::Device fill_paged(PyObject* const* args, bz_paged_cache& c) {
  const at::Tensor &k = tensor(args[0], "the cache's k"), &v = tensor(args[1], "the cache's v");
  const at::Tensor *ks = tensor_or_none(args[2], "k_scale"), *vs = tensor_or_none(args[3], "v_scale");
  const at::Tensor& table = tensor(args[4], "page_table");
  require(k.is_cuda() && v.device() == k.device(), "the cache's tensors must be on one device");
  const at::Device dev = k.device();
  const bool f8 = k.scalar_type() == at::kFloat8_e4m3fn;
  require((f8 || k.scalar_type() == at::kBFloat16) && v.scalar_type() == k.scalar_type(),
          "the cache's k and v must both be bf16 or float8_e4m3fn");
  require(k.dim() == 4 && alike(k, v) && k.stride(3) == 1 && k.numel() > 0,
          "the cache's k and v must be [pages, NKV, page_size, D] with equal shapes and strides and a contiguous last dim");
  for (int i = 0; i < 4; ++i) require(k.size(i) <= INT32_MAX, "the cache is too large");
  const int64_t e = k.element_size();
  c.k = k.data_ptr(), c.v = v.data_ptr();
  c.stride_page = e * step_of(k, 0), c.stride_h = e * step_of(k, 1), c.stride_s = e * k.stride(2);
  c.pages = (int32_t)k.size(0), c.num_kv_heads = (int32_t)k.size(1), c.page_size = (int32_t)k.size(2);
  c.head_dim = (int32_t)k.size(3), c.bits = f8 ? 8 : 16;
  if (f8) {
    require(ks != nullptr && vs != nullptr, "a cache of 8 bits has k_scale and v_scale");
    for (const at::Tensor* s : {ks, vs})
      require(s->scalar_type() == at::kByte && s->device() == dev && s->dim() == 3 && s->size(0) == c.pages &&
                  s->size(1) == c.num_kv_heads && s->size(2) == c.page_size && s->stride(2) == 1,
              "scales must be uint8 [pages, NKV, page_size] on the cache's device, the last dim contiguous");
    require(alike(*ks, *vs), "k_scale and v_scale must have equal strides");
    c.k_scale = ks->data_ptr(), c.v_scale = vs->data_ptr();
    c.scale_stride_page = step_of(*ks, 0), c.scale_stride_h = step_of(*ks, 1);
  } else {
    require(ks == nullptr && vs == nullptr, "a cache of bf16 has no scales");
  }
  require(table.scalar_type() == at::kInt && table.device() == dev && table.dim() == 2 && table.size(0) > 0 && table.size(1) > 0 &&
              (table.stride(1) == 1 || table.size(1) == 1) && table.size(0) < INT32_MAX && table.size(1) <= INT32_MAX,
          "page_table must be int32 [batch, pages a row] on the cache's device, its last dim contiguous");
  c.page_table = table.data_ptr<int32_t>(), c.table_stride = step_of(table, 0);
  c.batch = (int32_t)table.size(0), c.max_pages = (int32_t)table.size(1);
  return dev;
}

// The batch's rows and tokens.
void fill_rows(PyObject* seq_lens, PyObject* q_start, int64_t N, const at::Device& dev, bz_paged_cache& c) {
  c.seq_lens = rows_arg(seq_lens, c.batch, "seq_lens", dev);
  c.q_start = q_start == Py_None ? nullptr : rows_arg(q_start, (int64_t)c.batch + 1, "q_start", dev);
  if (c.q_start == nullptr && N != c.batch)
    throw Error{"without q_start there is one token a row: " + std::to_string(c.batch) + " rows, got " + std::to_string(N) + " tokens"};
  c.tokens = (int32_t)N;
}

// True or False (or the ints 1 and 0): not whatever has a truth value, as texts do, and tensors at the price of a synchronisation.
bool flag_arg(PyObject* o, const char* name) {
  if (o == Py_True || o == Py_False) return o == Py_True;
  const long x = PyLong_CheckExact(o) ? PyLong_AsLong(o) : -1;
  if (x != 0 && x != 1) {
    PyErr_Clear();
    throw Error{std::string(name) + " must be a bool"};
  }
  return x == 1;
}

// A Rope's inv_freq, factor and interleaved.
void fill_rope(PyObject* const* args, const at::Device& dev, bz_rope& r) {
  const at::Tensor& f = tensor(args[0], "inv_freq");
  require(f.scalar_type() == at::kDouble && f.device() == dev && f.dim() == 1 && f.is_contiguous() && f.numel() > 0 &&
              f.numel() <= INT32_MAX / 2,
          "inv_freq must be a contiguous float64 tensor [rotary_dim / 2] on the tokens' device");
  r.inv_freq = f.data_ptr<double>(), r.rotary_dim = (int32_t)(2 * f.numel());
  r.factor = float_arg(args[1], "factor");
  require(std::isfinite(r.factor) && r.factor != 0.f, "factor must be finite and not 0");
  r.interleaved = flag_arg(args[2], "interleaved");
}

const void* positions_arg(PyObject* o, int64_t N, const at::Device& dev, int32_t& is64) {
  const at::Tensor& t = tensor(o, "positions");
  if ((t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) || t.device() != dev || t.dim() != 1 || t.numel() != N ||
      !t.is_contiguous())
    throw Error{"positions must be a contiguous int32 or int64 tensor of " + std::to_string(N) + " elements on the tokens' device"};
  is64 = t.scalar_type() == at::kLong;
  return t.data_ptr();
}

at::Tensor heads_like(const at::Tensor& x) { return at::empty({x.size(0), x.size(1), x.size(2)}, x.options()); }

// rope(x, positions, inv_freq, factor, interleaved, inverse, out) -> out
PyObject* rope(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("rope", nargs, 7, [&]() -> PyObject* {
    const at::Tensor& x = tensor(args[0], "x");
    require(x.is_cuda(), "x must be a device tensor");
    const at::Device dev = x.device();
    check_heads(x, "x", dev);
    bz_rope_args a{};
    a.positions = positions_arg(args[1], x.size(0), dev, a.positions_64);
    fill_rope(args + 2, dev, a.rope);
    a.inverse = flag_arg(args[5], "inverse");
    const at::Tensor* given = tensor_or_none(args[6], "out");
    if (given != nullptr) {
      like_heads(*given, "out", x.size(0), x.size(1), x.size(2), dev);
      Touched all;
      all.write(given, "out");
      all.read(&x, "x");
      all.read(&tensor(args[1], "positions"), "positions");
      all.read(&tensor(args[2], "inv_freq"), "inv_freq");
      all.check(given, &x);
    }
    const int idx = dev.index();
    DeviceScope scope(idx);
    at::Tensor out = given != nullptr ? *given : heads_like(x);
    if (x.numel() == 0) return result(args[6], out);
    a.x = x.data_ptr(), a.x_stride_t = step_of(x, 0), a.x_stride_h = step_of(x, 1);
    a.out = out.data_ptr(), a.out_stride_t = step_of(out, 0), a.out_stride_h = step_of(out, 1);
    a.tokens = (int32_t)x.size(0), a.heads = (int32_t)x.size(1), a.head_dim = (int32_t)x.size(2);
    check_status(g_rope(&a, c10::hip::getCurrentHIPStream(idx).stream()), "bz_rope_apply");
    return result(args[6], out);
  });
}

// The new keys and values of a store, and the cache as args[0 .. 4].
at::Device fill_new(PyObject* const* cache, PyObject* k, PyObject* v, bz_paged_store_args& a, Touched& all) {
  const at::Device dev = fill_paged(cache, a.cache);
  const at::Tensor &xk = tensor(k, "k"), &xv = tensor(v, "v");
  check_heads(xk, "k", dev);
  like_heads(xk, "k", xk.size(0), a.cache.num_kv_heads, a.cache.head_dim, dev);
  like_heads(xv, "v", xk.size(0), a.cache.num_kv_heads, a.cache.head_dim, dev);
  a.k = xk.data_ptr(), a.k_stride_t = step_of(xk, 0), a.k_stride_h = step_of(xk, 1);
  a.v = xv.data_ptr(), a.v_stride_t = step_of(xv, 0), a.v_stride_h = step_of(xv, 1);
  const char* const names[4] = {"the cache's k", "the cache's v", "k_scale", "v_scale"};
  for (int i = 0; i < 4; ++i) all.write(tensor_or_none(cache[i], names[i]), names[i]);
  return dev;
}
void read_rows(PyObject* k, PyObject* v, PyObject* table, PyObject* seq_lens, PyObject* q_start, Touched& all) {
  all.read(&tensor(k, "k"), "k");
  all.read(&tensor(v, "v"), "v");
  all.read(&tensor(table, "page_table"), "page_table");
  all.read(&tensor(seq_lens, "seq_lens"), "seq_lens");
  all.read(tensor_or_none(q_start, "q_start"), "q_start");
}

// paged_store(k, v, ck, cv, k_scale, v_scale, page_table, seq_lens, q_start)
PyObject* paged_store(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("paged_store", nargs, 9, [&]() -> PyObject* {
    bz_paged_store_args a{};
    Touched all;
    const at::Device dev = fill_new(args + 2, args[0], args[1], a, all);
    const int64_t N = tensor(args[0], "k").size(0);
    fill_rows(args[7], args[8], N, dev, a.cache);
    read_rows(args[0], args[1], args[6], args[7], args[8], all);
    all.check();
    if (N == 0) Py_RETURN_NONE;
    const int idx = dev.index();
    DeviceScope scope(idx);
    check_status(g_paged_store(&a, c10::hip::getCurrentHIPStream(idx).stream()), "bz_paged_store");
    Py_RETURN_NONE;
  });
}

const void* weight_arg(PyObject* o, const char* name, int64_t D, const at::Device& dev) {
  const at::Tensor* w = tensor_or_none(o, name);
  if (w == nullptr) return nullptr;
  if (w->scalar_type() != at::kBFloat16 || w->device() != dev || w->numel() != D || !w->is_contiguous())
    throw Error{std::string(name) + " must be a contiguous bf16 tensor of " + std::to_string(D) + " elements on the cache's device"};
  return w->data_ptr();
}

// rope_store(q, k, v, ck, cv, k_scale, v_scale, page_table, seq_lens, inv_freq, factor, interleaved, q_start, out, positions,
// q_norm_weight, k_norm_weight, eps) -> out
PyObject* rope_store(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("rope_store", nargs, 18, [&]() -> PyObject* {
    bz_paged_store_args a{};
    Touched all;
    const at::Device dev = fill_new(args + 3, args[1], args[2], a, all);
    const at::Tensor& q = tensor(args[0], "q");
    const int64_t N = tensor(args[1], "k").size(0), D = a.cache.head_dim;
    check_heads(q, "q", dev);
    like_heads(q, "q", N, q.size(1), D, dev);
    require(q.size(1) > 0, "q must have heads");
    fill_rows(args[8], args[12], N, dev, a.cache);
    fill_rope(args + 9, dev, a.rope);
    if (args[14] != Py_None) a.positions = positions_arg(args[14], N, dev, a.positions_64);
    a.q_norm_weight = weight_arg(args[15], "q_norm_weight", D, dev);
    a.k_norm_weight = weight_arg(args[16], "k_norm_weight", D, dev);
    a.eps = float_arg(args[17], "eps");
    const at::Tensor* given = tensor_or_none(args[13], "out");
    if (given != nullptr) {
      like_heads(*given, "out", N, q.size(1), D, dev);
      all.write(given, "out");
    }
    all.read(&q, "q");
    read_rows(args[1], args[2], args[7], args[8], args[12], all);
    all.read(&tensor(args[9], "inv_freq"), "inv_freq");
    all.read(tensor_or_none(args[14], "positions"), "positions");
    all.read(tensor_or_none(args[15], "q_norm_weight"), "q_norm_weight");
    all.read(tensor_or_none(args[16], "k_norm_weight"), "k_norm_weight");
    all.check(given, &q);
    const int idx = dev.index();
    DeviceScope scope(idx);
    at::Tensor out = given != nullptr ? *given : heads_like(q);
    if (N == 0) return result(args[13], out);
    a.q = q.data_ptr(), a.q_stride_t = step_of(q, 0), a.q_stride_h = step_of(q, 1);
    a.q_out = out.data_ptr(), a.q_out_stride_t = step_of(out, 0), a.q_out_stride_h = step_of(out, 1);
    a.num_q_heads = (int32_t)q.size(1);
    check_status(g_paged_store(&a, c10::hip::getCurrentHIPStream(idx).stream()), "bz_paged_store");
    return result(args[13], out);
  });
}

// paged_load(ck, cv, k_scale, v_scale, page_table, starts, tokens, k, v) -> (k, v); k, v None: allocated
PyObject* paged_load(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("paged_load", nargs, 9, [&]() -> PyObject* {
    bz_paged_cache c{};
    const at::Device dev = fill_paged(args, c);
    const int32_t* starts = rows_arg(args[5], c.batch, "starts", dev);
    const int32_t tokens = int_arg(args[6], "tokens");
    const at::Tensor *kg = tensor_or_none(args[7], "k"), *vg = tensor_or_none(args[8], "v");
    require((kg == nullptr) == (vg == nullptr), "paged_load takes both outputs or neither");
    const int idx = dev.index();
    DeviceScope scope(idx);
    const auto options = at::TensorOptions().dtype(at::kBFloat16).device(dev);
    at::Tensor k = kg ? *kg : at::empty({c.batch, c.num_kv_heads, tokens, c.head_dim}, options);
    at::Tensor v = vg ? *vg : at::empty({c.batch, c.num_kv_heads, tokens, c.head_dim}, options);
    if (kg != nullptr) {
      for (const at::Tensor* x : {kg, vg})
        if (x->scalar_type() != at::kBFloat16 || x->device() != dev || x->dim() != 4 || x->size(0) != c.batch ||
            x->size(1) != c.num_kv_heads || x->size(2) != tokens || x->size(3) != c.head_dim || x->stride(3) != 1)
          throw Error{"outputs must be bf16 [batch, NKV, tokens, D] on the cache's device, the last dim contiguous, got " +
                      shape_str(*x)};
      require(alike(k, v), "the outputs must have equal strides");
      Touched all;
      all.write(kg, "k");
      all.write(vg, "v");
      const char* const names[4] = {"the cache's k", "the cache's v", "k_scale", "v_scale"};
      for (int i = 0; i < 4; ++i) all.read(tensor_or_none(args[i], names[i]), names[i]);
      all.read(&tensor(args[4], "page_table"), "page_table");
      all.read(&tensor(args[5], "starts"), "starts");
      all.check();
    }
    if (tokens > 0)
      check_status(g_paged_load(&c, starts, tokens, k.data_ptr(), v.data_ptr(), step_of(k, 0), step_of(k, 1), step_of(k, 2),
                                c10::hip::getCurrentHIPStream(idx).stream()),
                   "bz_paged_load");
    PyObject *pk = result(args[7], k), *pv = result(args[8], v);
    PyObject* r = pk && pv ? PyTuple_Pack(2, pk, pv) : nullptr;
    Py_XDECREF(pk);
    Py_XDECREF(pv);
    return r;
  });
}

// paged(q, ck, cv, k_scale, v_scale, page_table, seq_lens, scale, q_start, out, max_tokens, max_seq_len, workspace) -> out, or the
// tuple of long_workspace
PyObject* paged(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded("paged", nargs, 13, [&]() -> PyObject* {
    const at::Tensor& q = tensor(args[0], "query");
    bz_gqa_paged_args a{};
    bz_paged_cache& c = a.cache;
    const at::Device dev = fill_paged(args + 1, c);
    check_heads(q, "query", dev);
    const int64_t N = q.size(0), NH = q.size(1);
    if (q.size(2) != c.head_dim || NH == 0 || NH % c.num_kv_heads != 0)
      throw Error{"query " + shape_str(q) + " does not match a cache of " + std::to_string(c.num_kv_heads) + " heads, head_dim " +
                  std::to_string(c.head_dim)};
    fill_rows(args[6], args[8], N, dev, c);
    a.scale = float_arg(args[7], "scale");
    a.max_tokens = int_arg(args[10], "max_tokens"), a.max_seq_len = int_arg(args[11], "max_seq_len");
    const at::Tensor *given = tensor_or_none(args[9], "out"), *ws = tensor_or_none(args[12], "workspace");
    if (given != nullptr) {
      like_heads(*given, "out", N, NH, c.head_dim, dev);
      Touched all;
      all.write(given, "out");
      all.read(&q, "query");
      const char* const names[4] = {"the cache's k", "the cache's v", "k_scale", "v_scale"};
      for (int i = 0; i < 4; ++i) all.read(tensor_or_none(args[1 + i], names[i]), names[i]);
      all.read(&tensor(args[5], "page_table"), "page_table");
      all.read(&tensor(args[6], "seq_lens"), "seq_lens");
      all.read(tensor_or_none(args[8], "q_start"), "q_start");
      all.read(ws, "workspace");
      all.check();
    }
    const int idx = dev.index();
    DeviceScope scope(idx);
    if (N == 0) return result(args[9], given != nullptr ? *given : heads_like(q));
    hipStream_t stream = c10::hip::getCurrentHIPStream(idx).stream();
    if (ws != nullptr) {
      require(ws->device() == dev && ws->is_contiguous(), "workspace must be a contiguous tensor on the query's device");
      a.workspace = ws->data_ptr();
      a.workspace_bytes = (size_t)ws->numel() * ws->element_size();
    } else {
      const int64_t most = c.q_start == nullptr ? 1 : a.max_tokens > 0 ? std::min<int64_t>(a.max_tokens, N) : N;
      size_t need = 0;
      check_status(g_paged_size(c.head_dim, (int32_t)(NH / c.num_kv_heads), (int32_t)most, &need), "bz_paged_workspace_size");
      if (capturing(stream))
        throw Error{"a call being captured into a graph needs workspace= (paged_workspace(...), made before the capture; " +
                    std::to_string(need) + " bytes): graphs that shared the stream's own could not run at the same time"};
      const LongKey key{idx, (int64_t)reinterpret_cast<uintptr_t>(stream), kPagedKind, 0};
      auto it = g_long_ws.find(key);
      if (it == g_long_ws.end() || (size_t)it->second.numel() < need)
        return Py_BuildValue("(LLLLn)", (long long)key[0], (long long)key[1], (long long)key[2], (long long)key[3], (Py_ssize_t)need);
      a.workspace = it->second.data_ptr();
      a.workspace_bytes = (size_t)it->second.numel();
    }
    at::Tensor out = given != nullptr ? *given : heads_like(q);
    a.q = q.data_ptr(), a.q_stride_t = step_of(q, 0), a.q_stride_h = step_of(q, 1);
    a.out = out.data_ptr(), a.out_stride_t = step_of(out, 0), a.out_stride_h = step_of(out, 1);
    a.num_q_heads = (int32_t)NH;
    check_status(g_paged(&a, stream), "bz_gqa_paged");
    return result(args[9], out);
  });
}

// bind_paged(rope, store, load, paged, workspace_size): the C ABI functions' addresses
PyObject* bind_paged(PyObject*, PyObject* args) {
  unsigned long long f[5];
  if (!PyArg_ParseTuple(args, "KKKKK", &f[0], &f[1], &f[2], &f[3], &f[4])) return nullptr;
  g_rope = reinterpret_cast<RopeFn>(f[0]);
  g_paged_store = reinterpret_cast<PagedStoreFn>(f[1]);
  g_paged_load = reinterpret_cast<PagedLoadFn>(f[2]);
  g_paged = reinterpret_cast<PagedFn>(f[3]);
  g_paged_size = reinterpret_cast<PagedSizeFn>(f[4]);
  Py_RETURN_NONE;
}

}  // namespace
