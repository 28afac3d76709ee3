// The operators of decode_ops.h on torch tensors: argument checks, outputs, workspaces and the current
// stream, then one call of the C ABI.
#include "decode_ops.h"

#define BINDING_TAG "[radiance.decode] "
#define BINDING_ERROR dec_last_error
#include "torch_args.h"

namespace {

Tensor new_bytes(c10::Device dev, size_t n) {
  return n ? at::empty({(long)n}, at::TensorOptions().dtype(at::kByte).device(dev)) : Tensor();
}

// A batch's starts and slots, and the strides of its states' slots.
struct Batch {
  Tensor starts, read, write;
  long slots, slot_stride, write_stride;
  int batch, cols;
};
Batch batch_of(const Args& a, const Tensor& state, const Tensor& starts, const Tensor& read, const Tensor& write) {
  if (read.dim() != 1) fail(a.op, "read_slots must be int32 [batch], got " + str(read));
  Batch r;
  r.batch = a.to_int(read.size(0), "batch");
  r.read = ints(a, "read_slots", read, at::kInt, r.batch, "int32");
  r.starts = ints(a, "q_starts", starts, at::kInt, (long)r.batch + 1, "int32");
  if (write.scalar_type() != at::kInt || write.dim() < 1 || write.dim() > 2 || write.size(0) != r.batch)
    fail(a.op, "write_slots must be int32 [" + str(r.batch) + "] or [" + str(r.batch) + ", tokens], got " + str(write));
  r.write = write.contiguous();
  r.cols = write.dim() == 2 ? a.to_int(write.size(1), "write slots") : 0;
  if (write.dim() == 2 && !r.cols) fail(a.op, "write_slots has no columns");
  r.write_stride = write.dim() == 2 ? r.cols : 1;
  const long n = state.dim();
  long size = 1;
  for (long i = n - 1; i > 0; --i) {
    if (state.numel() && state.size(i) > 1 && state.stride(i) != size)
      fail(a.op, "a slot of the state must be contiguous");
    size *= state.size(i);
  }
  r.slots = state.size(0);
  r.slot_stride = r.slots > 1 ? state.stride(0) : size;
  return r;
}

// bf16 [T, ...] as 16-byte aligned rows, other layouts copied.
bool rows_fit(const Tensor& x) {
  if (!x.numel()) return true;
  const long n = x.dim();
  if (x.stride(n - 1) != 1 || ((uintptr_t)address(x) & 15)) return false;
  for (long i = 0; i < n - 1; ++i)
    if (x.size(i) > 1 && ((x.stride(i) & 7) || x.stride(i) < 0 || (i == 0 && x.stride(i) > 1 << 23))) return false;
  return true;
}
Tensor rows(const Args& a, const char* name, const Tensor& x, at::IntArrayRef shape) {
  if (x.scalar_type() != at::kBFloat16 || !x.sizes().equals(shape)) {
    std::string s;
    for (long n : shape) s += (s.empty() ? "" : ", ") + str(n);
    fail(a.op, std::string(name) + " must be bf16 [" + s + "], got " + str(x));
  }
  return rows_fit(x) ? x : x.clone(at::MemoryFormat::Contiguous);
}
long stride(const Tensor& x, int i) { return x.size(i) > 1 ? x.stride(i) : 0; }

PyObject* causal_conv(const Args& a) {
  const Tensor x0 = a.tensor(0), w0 = a.tensor(1), bias0 = a.optional(2), state = a.tensor(3), starts = a.tensor(4),
               read = a.tensor(5), write = a.tensor(6);
  const int max_q = a.integer(7, "max_q");
  const bool silu = a.flag(8);
  const c10::Device dev = device_of(a.op, {&x0, &w0, &bias0, &state, &starts, &read, &write});
  const c10::DeviceGuard guard(dev);
  if (x0.dim() != 2 || w0.dim() != 2) fail(a.op, "x must be bf16 [tokens, channels] and weight [channels, width], got " + str(x0) + " and " + str(w0));
  const int T = a.to_int(x0.size(0), "tokens"), C = a.to_int(x0.size(1), "channels"), W = a.to_int(w0.size(1), "width");
  if (C <= 0 || C % 8) fail(a.op, str(C) + " channels: need a multiple of 8");
  const Tensor x = rows(a, "x", x0, {T, C});
  if (w0.scalar_type() != at::kBFloat16 || w0.size(0) != C)
    fail(a.op, "weight must be bf16 [" + str(C) + ", width], got " + str(w0));
  const Tensor w = w0.is_contiguous() && !((uintptr_t)address(w0) & 15) ? w0 : w0.clone(at::MemoryFormat::Contiguous);
  const Tensor bias = bias0.defined() ? rows(a, "bias", bias0, {C}) : bias0;
  if (state.scalar_type() != at::kBFloat16 || state.dim() != 3 || state.size(1) != W - 1 || state.size(2) != C)
    fail(a.op, "state must be bf16 [slots, " + str(W - 1) + ", " + str(C) + "], got " + str(state));
  const Batch s = batch_of(a, state, starts, read, write);
  const Tensor out = new_bf16(dev, {T, C});
  launch(dev, [&](void* stream) {
    return dec_causal_conv(address(x), stride(x, 0), address(w), address(bias), address_as<void>(state), s.slots,
                           s.slot_stride, address_as<const int>(s.starts), address_as<const int>(s.read),
                           address_as<const int>(s.write), s.write_stride, s.cols, address_as<void>(out), T,
                           s.batch, max_q, C, W, silu ? DEC_SILU : 0, stream);
  });
  written(state);
  return THPVariable_Wrap(out);
}

PyObject* gated_delta_rule(const Args& a) {
  const Tensor q0 = a.tensor(0), k0 = a.tensor(1), v0 = a.tensor(2), a0 = a.tensor(3), b0 = a.tensor(4),
               a_log = a.tensor(5), dt_bias = a.tensor(6), state = a.tensor(7), starts = a.tensor(8),
               read = a.tensor(9), write = a.tensor(10);
  const int max_q = a.integer(11, "max_q");
  const c10::Device dev =
      device_of(a.op, {&q0, &k0, &v0, &a0, &b0, &a_log, &dt_bias, &state, &starts, &read, &write});
  const c10::DeviceGuard guard(dev);
  if (q0.dim() != 3 || v0.dim() != 3) fail(a.op, "q, k and v must be bf16 [tokens, heads, channels], got " + str(q0) + " and " + str(v0));
  const int T = a.to_int(q0.size(0), "tokens"), Hk = a.to_int(q0.size(1), "key heads"),
            dk = a.to_int(q0.size(2), "key channels"), Hv = a.to_int(v0.size(1), "value heads"),
            dv = a.to_int(v0.size(2), "value channels");
  const float scale = a.at[12] == Py_None ? (float)(1.0 / std::sqrt((double)std::max(dk, 1))) : (float)a.real(12);
  const float eps = (float)a.real(13);
  const Tensor q = rows(a, "q", q0, {T, Hk, dk}), k = rows(a, "k", k0, {T, Hk, dk}), v = rows(a, "v", v0, {T, Hv, dv});
  const auto gate = [&](const char* name, const Tensor& x) {
    if (x.scalar_type() != at::kBFloat16 || x.dim() != 2 || x.size(0) != T || x.size(1) != Hv)
      fail(a.op, std::string(name) + " must be bf16 [" + str(T) + ", " + str(Hv) + "], got " + str(x));
    return x.size(1) > 1 && x.stride(1) != 1 ? x.contiguous() : x;     // (one number for all heads: stride 0)
  };
  const Tensor ga = gate("a", a0), gb = gate("b", b0);
  const auto per_head = [&](const char* name, const Tensor& x) {
    return ints(a, name, x, at::kFloat, Hv, "fp32");
  };
  const Tensor al = per_head("a_log", a_log), db = per_head("dt_bias", dt_bias);
  if (state.scalar_type() != at::kFloat || state.dim() != 4 || state.size(1) != Hv || state.size(2) != dk || state.size(3) != dv)
    fail(a.op, "state must be fp32 [slots, " + str(Hv) + ", " + str(dk) + ", " + str(dv) + "], got " + str(state));
  const Batch s = batch_of(a, state, starts, read, write);
  const Tensor out = new_bf16(dev, {T, Hv, dv});
  size_t need = 0;
  check(dec_gated_delta_workspace(T, s.batch, max_q, s.cols, Hk, Hv, dk, dv, &need));
  const Tensor space = new_bytes(dev, need);
  // (the workspace, and inputs that are copies, are freed stream-ordered: reused after the launch)
  launch(dev, [&](void* stream) {
    return dec_gated_delta(address(q), stride(q, 0), stride(q, 1), address(k), stride(k, 0), stride(k, 1),
                           address(v), stride(v, 0), stride(v, 1), address(ga), stride(ga, 0), address(gb),
                           stride(gb, 0), address_as<const float>(al), address_as<const float>(db),
                           address_as<float>(state), s.slots, s.slot_stride, address_as<const int>(s.starts),
                           address_as<const int>(s.read), address_as<const int>(s.write), s.write_stride, s.cols,
                           address_as<void>(out), address_as<void>(space), need, T, s.batch, max_q, Hk, Hv, dk, dv,
                           scale, eps, stream);
  });
  written(state);
  return THPVariable_Wrap(out);
}

PyObject* sample(const Args& a) {
  const Tensor x0 = a.tensor(0), u0 = a.tensor(1), t0 = a.optional(2), k0 = a.optional(3), p0 = a.optional(4),
               mp0 = a.optional(5);
  const float t_all = (float)a.real(6), p_all = (float)a.real(8), mp_all = (float)a.real(9);
  const int k_all = a.integer(7, "top_k");
  const bool logprobs = a.flag(10);
  const c10::Device dev = device_of(a.op, {&x0, &u0, &t0, &k0, &p0, &mp0});
  const c10::DeviceGuard guard(dev);
  const bool bf16 = x0.scalar_type() == at::kBFloat16;
  if ((!bf16 && x0.scalar_type() != at::kFloat) || x0.dim() != 2)
    fail(a.op, "logits must be fp32 or bf16 [rows, vocabulary], got " + str(x0));
  const int rows = a.to_int(x0.size(0), "rows"), V = a.to_int(x0.size(1), "vocabulary");
  if (!V) fail(a.op, "logits of no vocabulary");
  const Tensor x = rows && (stride(x0, 1) != (V > 1) || (rows > 1 && x0.stride(0) < V)) ? x0.clone(at::MemoryFormat::Contiguous) : x0;
  const auto per_row = [&](const char* name, const Tensor& t, at::ScalarType type, const char* what) {
    return t.defined() ? ints(a, name, t, type, rows, what) : t;
  };
  const Tensor u = per_row("uniform", u0, at::kFloat, "fp32"), t = per_row("temperature", t0, at::kFloat, "fp32"),
               k = per_row("top_k", k0, at::kInt, "int32"), p = per_row("top_p", p0, at::kFloat, "fp32"),
               mp = per_row("min_p", mp0, at::kFloat, "fp32");
  const Tensor tokens = at::empty({rows}, at::TensorOptions().dtype(at::kLong).device(dev));
  const Tensor lp = at::empty({logprobs ? rows : 0}, at::TensorOptions().dtype(at::kFloat).device(dev));
  const int flags = (bf16 ? DEC_BF16 : 0) | (logprobs ? DEC_LOGPROBS : 0);
  size_t need = 0;
  check(dec_sample_workspace(rows, V, k.defined() ? 1 : k_all, flags, &need));
  const Tensor space = new_bytes(dev, need);
  launch(dev, [&](void* stream) {
    return dec_sample(address(x), rows > 1 ? x.stride(0) : V, address_as<const float>(u),
                      address_as<const float>(t), t_all, address_as<const int>(k), k_all,
                      address_as<const float>(p), p_all, address_as<const float>(mp), mp_all,
                      address_as<int64_t>(tokens), address_as<float>(lp), address_as<void>(space), need, rows, V,
                      flags, stream);
  });
  PyObject* out = PyTuple_New(2);
  if (!out) throw python_error();
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(tokens));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(lp));
  return out;
}

PyMethodDef methods[] = {ENTRIES(causal_conv, 9), ENTRIES(gated_delta_rule, 14), ENTRIES(sample, 11),
                         METHOD("is_plain", is_plain), {}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_decode_torch", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__decode_torch() {
  if (dec_abi_version() != DEC_ABI_VERSION) {
    PyErr_SetString(PyExc_RuntimeError, "libdecode_ops.so is of another ABI than _decode_torch.so");
    return nullptr;
  }
  return PyModule_Create(&module);
}
