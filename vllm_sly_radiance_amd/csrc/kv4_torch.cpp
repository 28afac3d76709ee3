// The 4-bit cache's ops on torch tensors: argument checks, outputs, workspaces and the current stream,
// then one call of the C ABI (kv4_attn.h). A CPython module without the dispatcher in front: a decode
// step's ops are a few microseconds of GPU work each, and the host has to keep up with them. One
// token through qk_norm_rope takes 6.4 us a call from Python, 2.7 of them the launch, where the
// same checks in Python and a ctypes call took 13.
#include "kv4_attn.h"

#define BINDING_TAG "[radiance.kv4] "
#define BINDING_ERROR kv4_last_error
#include "torch_args.h"

namespace {

bool head_size(long d) { return d == 64 || d == 128 || d == 256; }

// bf16 [T, heads, d] whose heads are 16-byte aligned runs, other layouts copied; the stride of an axis
// of one, which may be anything, as 0.
struct Heads {
  Tensor x;
  int T, H, d;
  long ts, hs;
};
Heads heads(const Args& a, const char* name, Tensor x) {
  if (x.scalar_type() != at::kBFloat16 || x.dim() != 3)
    fail(a.op, std::string(name) + " must be bf16 [tokens, heads, head size], got " + str(x));
  Heads h = {x, a.to_int(x.size(0), "tokens"), a.to_int(x.size(1), "heads"), 0, 0, 0};
  if (!head_size(x.size(2)))
    fail(a.op, "head size " + str(x.size(2)) + " of " + name + " is none of 64, 128, 256");
  h.d = (int)x.size(2);
  h.ts = h.T > 1 ? x.stride(0) : 0, h.hs = h.H > 1 ? x.stride(1) : 0;
  if (h.T && (x.stride(2) != 1 || ((h.ts | h.hs) & 7) || ((uintptr_t)address(x) & 15))) {
    h.x = x.clone(at::MemoryFormat::Contiguous);
    h.ts = h.T > 1 ? h.x.stride(0) : 0, h.hs = h.H > 1 ? h.x.stride(1) : 0;
  }
  return h;
}
void matches(const Args& a, const char* name, const Heads& h, const Heads& q, int H) {
  if (h.T != q.T || h.d != q.d || h.H != H)
    fail(a.op, std::string(name) + " " + str(h.x) + " does not match [" + str(q.T) + ", " + str(H) +
                   ", " + str(q.d) + "]");
}

struct Cache {
  uint8_t* p;
  long pages, stride;
  int H, page, d;
  size_t bytes;             // of a page
};
// A layer's cache, in `t`'s last four axes.
Cache cache_of(const Args& a, const Tensor& t, int d = 0, int H = 0) {
  const long n = t.dim(), b = n < 4 ? 0 : t.size(n - 1), groups = n < 4 ? 0 : t.size(n - 2);
  if (t.scalar_type() != at::kByte || n < 4 || b % 17 || !head_size(b / 17) || groups <= 0 ||
      groups > 16 || (groups & (groups - 1)))
    fail(a.op, "cache must be uint8 [pages, kv heads, page / 16, 17 * head size], got " + str(t));
  Cache c = {address_as<uint8_t>(t), t.size(n - 4), 0, a.to_int(t.size(n - 3), "kv heads"),
             (int)groups * 16, (int)(b / 17), (size_t)(t.size(n - 3) * groups * b)};
  if (t.numel() && (t.stride(n - 1) != 1 || (groups > 1 && t.stride(n - 2) != b) ||
                    (c.H > 1 && t.stride(n - 3) != groups * b) || ((uintptr_t)c.p & 15)))
    fail(a.op, "a page of the cache must be contiguous and 16-byte aligned");
  if (d && c.d != d) fail(a.op, "cache of head size " + str(c.d) + " against " + str(d));
  if (H && c.H != H) fail(a.op, "cache of " + str(c.H) + " kv heads against " + str(H));
  c.stride = c.pages > 1 ? t.stride(n - 4) : (long)c.bytes;
  return c;
}

// ---- norm and rotation --------------------------------------------------------------------------
struct Turn {
  Tensor qw, kw, table, pos, axis;
  long rows = 0, pos_stride = 0;
  int rot = 0, axes = 1, flags = 0;
};
Turn turn_of(const Args& a, int T, int d, const Tensor& qw, const Tensor& kw, const Tensor& table,
             const Tensor& pos, const Tensor& axis, bool plus_one, bool adjacent) {
  Turn r;
  r.flags = (plus_one ? KV4_PLUS_ONE : 0) | (adjacent ? KV4_ADJACENT : 0);
  auto weight = [&](const char* name, const Tensor& w) {
    if (!w.defined()) return w;
    if (w.scalar_type() != at::kBFloat16 || w.dim() != 1 || w.size(0) != d)
      fail(a.op, std::string(name) + " must be bf16 [" + str(d) + "], got " + str(w));
    return w.stride(0) != 1 || ((uintptr_t)address(w) & 15) ? w.clone(at::MemoryFormat::Contiguous) : w;
  };
  r.qw = weight("q_weight", qw), r.kw = weight("k_weight", kw);
  if (!table.defined()) return r;
  const bool bf16 = table.scalar_type() == at::kBFloat16;
  if ((!bf16 && table.scalar_type() != at::kFloat) || table.dim() != 2)
    fail(a.op, "cos_sin must be fp32 or bf16 [positions, rotated channels], got " + str(table));
  const long rot = table.size(1);
  if (rot == 0 || rot > d || rot % 16)
    fail(a.op, str(rot) + " rotated channels: need a multiple of 16 up to the head size " + str(d));
  r.rows = table.size(0), r.rot = (int)rot, r.table = table.contiguous();
  const long dims = pos.defined() ? pos.dim() : 0;
  const bool i32 = dims && pos.scalar_type() == at::kInt;
  if (dims < 1 || dims > 2 || (!i32 && pos.scalar_type() != at::kLong) || pos.size(dims - 1) != T ||
      (dims == 2 && pos.size(0) == 0))
    fail(a.op, "positions must be int64 or int32 [" + str(T) + "] or [axes, " + str(T) + "], got " +
                   str(pos));
  r.axes = dims == 2 ? a.to_int(pos.size(0), "axes") : 1;
  if (r.axes > 1 && !axis.defined())
    fail(a.op, "positions on " + str(r.axes) + " axes need the axis of each pair (rotary_axes)");
  if (axis.defined()) r.axis = ints(a, "axis", axis, at::kInt, rot / 2, "int32");
  r.pos = pos.stride(dims - 1) != 1 || (r.axes > 1 && pos.stride(0) < T) ? pos.contiguous() : pos;
  r.pos_stride = r.axes > 1 ? r.pos.stride(0) : T;
  r.flags |= (bf16 ? KV4_TABLE_BF16 : 0) | (i32 ? KV4_POS_I32 : 0);
  return r;
}

PyObject* qk_norm_rope(const Args& a) {
  const Tensor q0 = a.tensor(0), k0 = a.tensor(1), qw = a.optional(2), kw = a.optional(3),
               table = a.optional(4), pos = a.optional(5), axis = a.optional(6);
  const c10::Device dev = device_of(a.op, {&q0, &k0, &qw, &kw, &table, &pos, &axis});
  const c10::DeviceGuard guard(dev);
  const Heads q = heads(a, "q", q0), k = heads(a, "k", k0);
  matches(a, "k", k, q, k.H);
  const Turn r = turn_of(a, q.T, q.d, qw, kw, table, pos, axis, a.flag(8), a.flag(9));
  const float eps = (float)a.real(7);
  const Tensor qo = new_bf16(dev, {q.T, q.H, q.d}), ko = new_bf16(dev, {k.T, k.H, k.d});
  launch(dev, [&](void* stream) {
    return kv4_qk_norm_rope(address(q.x), q.ts, q.hs, address(k.x), k.ts, k.hs, address(r.qw),
                            address(r.kw), address(r.table), r.rows, r.rot, address(r.pos),
                            r.pos_stride, r.axes, address_as<const int>(r.axis), address_as<void>(qo),
                            address_as<void>(ko), q.T, q.H, k.H, q.d, eps, r.flags, stream);
  });
  PyObject* out = PyTuple_New(2);
  if (!out) throw python_error();
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(qo));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(ko));
  return out;
}

PyObject* qk_norm_rope_append(const Args& a) {
  const Tensor q0 = a.tensor(0), k0 = a.tensor(1), v0 = a.tensor(2), qw = a.optional(3),
               kw = a.optional(4), table = a.optional(5), pos = a.optional(6), cache = a.tensor(7),
               slots0 = a.tensor(8), axis = a.optional(9);
  const c10::Device dev =
      device_of(a.op, {&q0, &k0, &v0, &qw, &kw, &table, &pos, &cache, &slots0, &axis});
  const c10::DeviceGuard guard(dev);
  const Heads q = heads(a, "q", q0), k = heads(a, "k", k0), v = heads(a, "v", v0);
  matches(a, "k", k, q, k.H), matches(a, "v", v, q, k.H);
  const Turn r = turn_of(a, q.T, q.d, qw, kw, table, pos, axis, a.flag(11), a.flag(12));
  const float eps = (float)a.real(10);
  if (cache.dim() != 4) fail(a.op, "cache must be one layer's, got " + str(cache));
  const Cache c = cache_of(a, cache, q.d, k.H);
  const Tensor slots = ints(a, "slots", slots0, at::kLong, q.T, "int64");
  const Tensor qo = new_bf16(dev, {q.T, q.H, q.d});
  launch(dev, [&](void* stream) {
    return kv4_qk_norm_rope_append(
        address(q.x), q.ts, q.hs, address(k.x), k.ts, k.hs, address(v.x), v.ts, v.hs, address(r.qw),
        address(r.kw), address(r.table), r.rows, r.rot, address(r.pos), r.pos_stride, r.axes,
        address_as<const int>(r.axis), address_as<void>(qo), c.p, c.pages, c.stride, c.page,
        address_as<const int64_t>(slots), q.T, q.H, k.H, q.d, eps, r.flags, stream);
  });
  written(cache);
  return THPVariable_Wrap(qo);
}

// ---- reading back -------------------------------------------------------------------------------
PyObject* gather(const Args& a) {
  const Tensor cache = a.tensor(0), slots0 = a.tensor(1);
  const c10::Device dev = device_of(a.op, {&cache, &slots0});
  const c10::DeviceGuard guard(dev);
  if (cache.dim() != 4) fail(a.op, "cache must be one layer's, got " + str(cache));
  const Cache c = cache_of(a, cache);
  const int T = a.to_int(slots0.dim() ? slots0.size(0) : 0, "slots");
  const Tensor slots = ints(a, "slots", slots0, at::kLong, T, "int64");
  const Tensor k = new_bf16(dev, {T, c.H, c.d}), v = new_bf16(dev, {T, c.H, c.d});
  launch(dev, [&](void* stream) {
    return kv4_gather(c.p, c.pages, c.stride, c.page, address_as<const int64_t>(slots),
                      address_as<void>(k), address_as<void>(v), T, c.H, c.d, stream);
  });
  PyObject* out = PyTuple_New(2);
  if (!out) throw python_error();
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(k));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(v));
  return out;
}

// ---- attention ----------------------------------------------------------------------------------
PyObject* attention(const Args& a) {
  const Tensor q0 = a.tensor(0), cache = a.tensor(1), table0 = a.tensor(2), lens0 = a.tensor(3),
               starts0 = a.tensor(4);
  const int max_q = a.integer(5, "max_q"), max_len = a.integer(6, "max_len");
  const float scale = (float)a.real(7);
  const bool causal = a.flag(8);
  const int window = a.integer(9, "window");
  const c10::Device dev = device_of(a.op, {&q0, &cache, &table0, &lens0, &starts0});
  const c10::DeviceGuard guard(dev);
  const Heads q = heads(a, "q", q0);
  if (cache.dim() != 4) fail(a.op, "cache must be one layer's, got " + str(cache));
  const Cache c = cache_of(a, cache, q.d);
  if (lens0.dim() != 1) fail(a.op, "seq_lens must be int32 [batch], got " + str(lens0));
  const int B = a.to_int(lens0.size(0), "batch");
  const Tensor lens = ints(a, "seq_lens", lens0, at::kInt, B, "int32");
  const Tensor starts = ints(a, "q_starts", starts0, at::kInt, (long)B + 1, "int32");
  if (table0.scalar_type() != at::kInt || table0.dim() != 2 || table0.size(0) != B)
    fail(a.op, "page_table must be int32 [" + str(B) + ", pages of a sequence], got " + str(table0));
  const Tensor table = table0.stride(1) != 1 ? table0.contiguous() : table0;
  const int cols = a.to_int(table.size(1), "pages of a sequence");
  const Tensor out = new_bf16(dev, {q.T, q.H, q.d});
  if (q.T && B) {
    size_t need = 0;
    check(kv4_attention_workspace(q.T, B, max_q, max_len, q.H, c.H, q.d, window, &need));
    Tensor space;
    if (need) space = at::empty({(long)need}, at::TensorOptions().dtype(at::kByte).device(dev));
    // (the workspace, and inputs that are copies, are freed stream-ordered: reused after the launch)
    launch(dev, [&](void* stream) {
      return kv4_attention(address(q.x), q.ts, q.hs, c.p, c.pages, c.stride, c.page,
                           address_as<const int>(table), B > 1 ? table.stride(0) : 0, cols,
                           address_as<const int>(lens), address_as<const int>(starts),
                           address_as<void>(out), address_as<void>(space), need, q.T, B, max_q,
                           max_len, q.H, c.H, q.d, scale, window, causal ? KV4_CAUSAL : 0, stream);
    });
  }
  return THPVariable_Wrap(out);
}

// ---- pages --------------------------------------------------------------------------------------
PyObject* move_pages(const Args& a) {
  const Tensor cache = a.tensor(0), pairs0 = a.tensor(1), table = a.optional(2);
  const c10::Device dev = device_of(a.op, {&cache, &table});
  const c10::DeviceGuard guard(dev);
  const Cache c = cache_of(a, cache);
  if (cache.dim() > 5) fail(a.op, "cache of one layer or of layers, got " + str(cache));
  if (!pairs0.device().is_cpu() || pairs0.scalar_type() != at::kInt || pairs0.dim() != 2 ||
      pairs0.size(1) != 2)
    fail(a.op, "pairs must be int32 [n, 2] (from, to) on the host, got " + str(pairs0) + " on " +
                   pairs0.device().str());
  const Tensor pairs = pairs0.contiguous();
  const int n = a.to_int(pairs.size(0), "pairs");
  const int layers = cache.dim() == 5 ? a.to_int(cache.size(0), "layers") : 1;
  int rows = 0, cols = 0;
  long row = 0;
  if (table.defined()) {
    if (table.scalar_type() != at::kInt || table.dim() != 2 ||
        (table.numel() && table.size(1) > 1 && table.stride(1) != 1))
      fail(a.op, "page_table must be int32 [sequences, pages] with contiguous rows, got " + str(table));
    rows = a.to_int(table.size(0), "sequences"), cols = a.to_int(table.size(1), "pages");
    row = rows > 1 ? table.stride(0) : cols;
  }
  if (layers)
    launch(dev, [&](void* stream) {
      return kv4_move_pages(c.p, layers, layers > 1 ? cache.stride(0) : 0, c.pages, c.stride, c.bytes,
                            address_as<const int>(pairs), n,
                            rows && cols ? address_as<int>(table) : nullptr, rows, cols, row, stream);
    });
  written(cache), written(table);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {ENTRIES(qk_norm_rope, 10), ENTRIES(qk_norm_rope_append, 13), ENTRIES(gather, 2),
                         ENTRIES(attention, 10),    ENTRIES(move_pages, 3),           METHOD("is_plain", is_plain),
                         {}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kv4_torch", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__kv4_torch() {
  if (kv4_abi_version() != KV4_ABI_VERSION) {
    PyErr_SetString(PyExc_RuntimeError, "libkv4_attn.so is of another ABI than _kv4_torch.so");
    return nullptr;
  }
  return PyModule_Create(&module);
}
