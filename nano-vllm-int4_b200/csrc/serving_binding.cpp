// Python binding of the 4-bit cache, step table and log-probability entry points
// (nanovllm/kernels/{kv4_cache,step_tables,token_logprobs}.py), whose kernels
// take 3 to 15 us: the checks of the arguments, the outputs' allocation and the
// call itself.  The same through Python and ctypes took 17 to 22 us of host time
// a call, most of it in new tensors (2.5 us each there, 0.9 us here) and checks;
// here it is 4 to 8 us in a loop of one call (x.add_(1) takes 4.4), 6 to 12 among others.
// Every output has storage of its own: parts of one allocation would save 3 us of
// the step tables' 9, but could not be saved together and would keep one another alive.
// The calls go to the C ABI of include/nv4.h.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../include/nv4.h"

namespace {

constexpr int64_t kD = 128, kPage = 256, kCodeBytes = 64, kGroups = 4;

struct Refused {  // a Python exception to raise
  PyObject* type;
  std::string text;
};
[[noreturn]] void refuse(const char* text) { throw Refused{PyExc_ValueError, text}; }
[[noreturn]] void refuse_type(const char* text) { throw Refused{PyExc_TypeError, text}; }
struct Raised {};  // one is set already

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw Refused{PyExc_TypeError, std::string("Expected a tensor for ") + name};
  return THPVariable_Unpack(o);
}
const at::Tensor* optional(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised{};
  return v;
}
bool shaped(const at::Tensor& t, at::ScalarType type, std::initializer_list<int64_t> sizes) {
  return t.scalar_type() == type && t.sizes() == at::IntArrayRef(sizes.begin(), sizes.size());
}
void* address(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }

// The device of the first tensor, when all are contiguous there.
class Device {
 public:
  explicit Device(const at::Tensor& t) : index_(t.is_cuda() ? t.get_device() : -1) { add(&t); }
  void add(const at::Tensor* t) {
    if (t) ok_ = ok_ && t->is_cuda() && t->get_device() == index_ && t->is_contiguous();
  }
  void check() const {
    if (index_ < 0 || !ok_) refuse("All tensors must be contiguous on one CUDA device");
  }
  int index() const { return index_; }

 private:
  int index_;
  bool ok_ = true;
};

// Runs `call(stream)` on the current stream of the device; a status other than
// NV4_OK becomes the exception that nanovllm._native.check makes of it.
template <typename Call>
void launch(int device, const char* name, const Call& call) {
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
  const int status = call(static_cast<void*>(c10::cuda::getCurrentCUDAStream(device).stream()));
  if (status == NV4_OK) return;
  PyObject* module = PyImport_ImportModule("nanovllm._native");
  PyObject* result = module ? PyObject_CallMethod(module, "check", "is", status, name) : nullptr;
  Py_XDECREF(result);
  Py_XDECREF(module);
  throw Raised{};
}

at::Tensor fresh(const at::Tensor& like, at::IntArrayRef sizes, at::ScalarType type) {
  return at::empty(sizes, like.options().dtype(type).memory_format(c10::nullopt));
}

// KV heads of a well-formed cache (k_codes, k_scales, v_codes, v_scales).
int64_t check_cache(const at::Tensor* const (&c)[4]) {
  const auto s = c[0]->sizes();
  if (s.size() != 4 || s[0] < 1 || s[1] < 1 || s[2] != kPage || s[3] != kCodeBytes)
    refuse("Expected codes[pages,Hkv,256,64]");
  const int64_t scales[4] = {s[0], s[1], kPage, kGroups};
  if (c[2]->sizes() != s || c[1]->sizes() != at::IntArrayRef(scales) || c[3]->sizes() != at::IntArrayRef(scales))
    refuse("Expected K and V codes[pages,Hkv,256,64] and scales[pages,Hkv,256,4]");
  if (c[0]->scalar_type() != at::kByte || c[2]->scalar_type() != at::kByte) refuse_type("Codes must be UINT8");
  if (c[1]->scalar_type() != at::kBFloat16 || c[3]->scalar_type() != at::kBFloat16)
    refuse_type("Cache scales must be BF16");
  return s[1];
}

void expect_args(Py_ssize_t n, Py_ssize_t wanted) {
  if (n != wanted) throw Refused{PyExc_TypeError, "wrong number of arguments"};
}

template <typename Body>
PyObject* guarded(const Body& body) {
  try {
    return body();
  } catch (const Refused& e) {
    PyErr_SetString(e.type, e.text.c_str());
  } catch (const Raised&) {
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    PyErr_SetString(type ? type : PyExc_RuntimeError, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// check_cache(k_codes, k_scales, v_codes, v_scales) -> KV heads
PyObject* py_check_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect_args(n, 4);
    const at::Tensor* const cache[4] = {&tensor(a[0], "k_codes"), &tensor(a[1], "k_scales"),
                                        &tensor(a[2], "v_codes"), &tensor(a[3], "v_scales")};
    return PyLong_FromLongLong(check_cache(cache));
  });
}

// attention(q, k_codes, k_scales, v_codes, v_scales, block_tables, context_lens, out, workspace, scale) -> out
PyObject* py_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect_args(n, 10);
    const at::Tensor& q = tensor(a[0], "q");
    const at::Tensor* const cache[4] = {&tensor(a[1], "k_codes"), &tensor(a[2], "k_scales"),
                                        &tensor(a[3], "v_codes"), &tensor(a[4], "v_scales")};
    const at::Tensor &tables = tensor(a[5], "block_tables"), &lens = tensor(a[6], "context_lens");
    const at::Tensor *out_in = optional(a[7], "out"), *ws_in = optional(a[8], "workspace");
    const double scale = real(a[9]);
    if (q.dim() != 3 || q.scalar_type() != at::kBFloat16 || q.size(0) < 1 || q.size(2) != kD)
      refuse("Expected BF16 q[B,Hq,128], B>0");
    const int64_t b = q.size(0), hq = q.size(1), hkv = check_cache(cache);
    if (hq < hkv || hq % hkv || hq / hkv > 8) refuse("Expected query heads to be 1 to 8 times the KV heads");
    if (tables.dim() != 2 || tables.size(0) != b || tables.size(1) < 1 || tables.scalar_type() != at::kInt)
      refuse("Expected INT32 block_tables[B,max_pages]");
    if (!shaped(lens, at::kInt, {b})) refuse("Expected INT32 context_lens[B]");
    if (!(scale > 0)) refuse("scale must be positive");
    if (out_in && !shaped(*out_in, at::kBFloat16, {b, hq, kD})) refuse("Expected BF16 out[B,Hq,128]");
    Device device(q);
    for (const at::Tensor* t : {&tables, &lens, cache[0], cache[1], cache[2], cache[3], out_in, ws_in}) device.add(t);
    device.check();
    const at::Tensor out = out_in ? *out_in : fresh(q, q.sizes(), at::kBFloat16);
    const at::Tensor ws =
        ws_in ? *ws_in : fresh(q, {nv4_paged_attention_kv4_workspace_bytes(b, hq, tables.size(1))}, at::kByte);
    launch(device.index(), "nv4_paged_decode_attention_kv4", [&](void* stream) {
      return nv4_paged_decode_attention_kv4(
          q.data_ptr(), cache[0]->data_ptr(), cache[1]->data_ptr(), cache[2]->data_ptr(), cache[3]->data_ptr(),
          static_cast<const int32_t*>(tables.data_ptr()), static_cast<const int32_t*>(lens.data_ptr()),
          out.data_ptr(), ws.data_ptr(), static_cast<int64_t>(ws.nbytes()), b, hq, hkv, kD, kPage, cache[0]->size(0),
          tables.size(1), static_cast<float>(scale), stream);
    });
    return THPVariable_Wrap(out);
  });
}

// store(qkv, q_weight, k_weight, cos_sin, positions, slot_mapping, k_codes, k_scales, v_codes, v_scales, num_heads,
//       num_kv_heads, eps, q_out, return_values) -> q, or (q, k, v); slot_mapping and the cache may be None
PyObject* py_store(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect_args(n, 15);
    const at::Tensor &qkv = tensor(a[0], "qkv"), &qw = tensor(a[1], "q_weight"), &kw = tensor(a[2], "k_weight");
    const at::Tensor &cos_sin = tensor(a[3], "cos_sin"), &positions = tensor(a[4], "positions");
    const at::Tensor* slots = optional(a[5], "slot_mapping");
    const at::Tensor* const cache[4] = {optional(a[6], "k_codes"), optional(a[7], "k_scales"),
                                        optional(a[8], "v_codes"), optional(a[9], "v_scales")};
    const int64_t hq = integer(a[10]), hkv = integer(a[11]);
    const double eps = real(a[12]);
    const at::Tensor* q_in = optional(a[13], "q_out");
    const int values = PyObject_IsTrue(a[14]);
    if (values < 0) throw Raised{};
    if (hq < 1 || hkv < 1) refuse("Expected at least one query head and one KV head");
    if (qkv.dim() != 2 || qkv.scalar_type() != at::kBFloat16 || qkv.size(0) < 1 || qkv.size(1) != (hq + 2 * hkv) * kD)
      refuse("Expected BF16 qkv[T,(Hq+2Hkv)*128], T>0");
    const int64_t t = qkv.size(0);
    if (!shaped(qw, at::kBFloat16, {kD}) || !shaped(kw, at::kBFloat16, {kD}))
      refuse("Expected BF16 q_weight[128] and k_weight[128]");
    if (cos_sin.dim() != 2 || cos_sin.size(0) < 1 || cos_sin.size(1) != kD || cos_sin.scalar_type() != at::kFloat)
      refuse("Expected FP32 cos_sin[max_position,128]");
    if (!shaped(positions, at::kLong, {t})) refuse("Expected INT64 positions[T]");
    for (const at::Tensor* x : cache)
      if (!slots != !x) refuse("slot_mapping and cache go together");
    if (slots && !shaped(*slots, at::kInt, {t})) refuse("Expected INT32 slot_mapping[T]");
    if (cache[0] && check_cache(cache) != hkv) refuse("The cache has another number of KV heads");
    if (q_in && !shaped(*q_in, at::kBFloat16, {t, hq, kD})) refuse("Expected BF16 q_out[T,Hq,128]");
    Device device(qkv);
    for (const at::Tensor* x : {&qw, &kw, &cos_sin, &positions, slots, cache[0], cache[1], cache[2], cache[3], q_in})
      device.add(x);
    device.check();
    const at::Tensor q = q_in ? *q_in : fresh(qkv, {t, hq, kD}, at::kBFloat16);
    at::Tensor k, v;
    if (values) k = fresh(qkv, {t, hkv, kD}, at::kBFloat16), v = fresh(qkv, {t, hkv, kD}, at::kBFloat16);
    launch(device.index(), "nv4_qk_norm_rope_store_kv4", [&](void* stream) {
      return nv4_qk_norm_rope_store_kv4(
          qkv.data_ptr(), qw.data_ptr(), kw.data_ptr(), static_cast<const float*>(cos_sin.data_ptr()),
          static_cast<const int64_t*>(positions.data_ptr()), static_cast<const int32_t*>(address(slots)), q.data_ptr(),
          values ? k.data_ptr() : nullptr, values ? v.data_ptr() : nullptr, address(cache[0]), address(cache[1]),
          address(cache[2]), address(cache[3]), t, hq, hkv, kD, kPage, cache[0] ? cache[0]->size(0) : 0,
          cos_sin.size(0), eps, stream);
    });
    if (!values) return THPVariable_Wrap(q);
    return Py_BuildValue("(NNN)", THPVariable_Wrap(q), THPVariable_Wrap(k), THPVariable_Wrap(v));
  });
}

// step_tables(cached_lens, new_lens, pages, num_tokens, max_pages, page_size[, block_tables, context_lens,
//             slot_mapping, positions, query_starts]) -> those five
PyObject* py_step_tables(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 6) expect_args(n, 11);
    const at::Tensor &cached = tensor(a[0], "cached_lens"), &news = tensor(a[1], "new_lens");
    const at::Tensor& pages = tensor(a[2], "pages");
    const int64_t tokens = integer(a[3]), max_pages = integer(a[4]), page_size = integer(a[5]);
    if (cached.dim() != 1 || cached.size(0) < 1 || cached.scalar_type() != at::kInt ||
        !shaped(news, at::kInt, {cached.size(0)}))
      refuse("Expected INT32 cached_lens[B] and new_lens[B], B>0");
    const int64_t b = cached.size(0);
    if (b > NV4_STEP_MAX_BATCH) {
      const std::string text = "Expected at most " + std::to_string(NV4_STEP_MAX_BATCH) + " requests";
      refuse(text.c_str());
    }
    if (pages.dim() != 1 || pages.scalar_type() != at::kInt) refuse("Expected INT32 pages[P]");
    if (tokens < 0 || max_pages < 1 || page_size < 1) refuse("Expected num_tokens>=0, max_pages>0, page_size>0");
    Device device(cached);
    device.add(&news);
    device.add(&pages);
    at::Tensor out[5];
    if (n == 11) {
      for (int i = 0; i < 5; ++i) out[i] = tensor(a[6 + i], "out");
      const int64_t rows = out[0].dim() == 2 ? out[0].size(0) : -1;
      if (rows < b || out[0].size(1) != max_pages || out[1].sizes() != at::IntArrayRef({rows}) ||
          out[4].sizes() != at::IntArrayRef({rows + 1}) || out[2].dim() != 1 || out[2].size(0) < tokens ||
          out[3].sizes() != out[2].sizes())
        refuse("Expected out with block_tables[rows>=B,max_pages], context_lens[rows], query_starts[rows+1], "
               "slot_mapping and positions[tokens>=num_tokens]");
      for (int i = 0; i < 5; ++i) {
        if (out[i].scalar_type() != (i == 3 ? at::kLong : at::kInt))
          refuse_type("Expected INT64 positions and INT32 other outputs");
        device.add(&out[i]);
      }
      device.check();
    } else {
      device.check();
      if (max_pages > int64_t(1) << 24 || tokens > int64_t(1) << 30)
        refuse("Expected num_tokens<=2^30 and max_pages<=2^24");
      out[0] = fresh(cached, {b, max_pages}, at::kInt);
      out[1] = fresh(cached, {b}, at::kInt);
      out[2] = fresh(cached, {tokens}, at::kInt);
      out[3] = fresh(cached, {tokens}, at::kLong);
      out[4] = fresh(cached, {b + 1}, at::kInt);
    }
    const auto i32 = [](const at::Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); };
    launch(device.index(), "nv4_step_tables", [&](void* stream) {
      return nv4_step_tables(i32(cached), i32(news), i32(pages), i32(out[0]), i32(out[1]), i32(out[4]), i32(out[2]),
                             static_cast<int64_t*>(out[3].data_ptr()), b, out[0].size(0), pages.size(0),
                             out[2].size(0), max_pages, page_size, stream);
    });
    return Py_BuildValue("(NNNNN)", THPVariable_Wrap(out[0]), THPVariable_Wrap(out[1]), THPVariable_Wrap(out[2]),
                         THPVariable_Wrap(out[3]), THPVariable_Wrap(out[4]));
  });
}

// logprobs(logits, targets, top_k) -> logprobs, ranks, entropy, top_logprobs, top_ids (the last two None for top_k 0)
PyObject* py_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect_args(n, 3);
    const at::Tensor &logits = tensor(a[0], "logits"), &targets = tensor(a[1], "targets");
    const int64_t k = integer(a[2]);
    const bool fp32 = logits.scalar_type() == at::kFloat;
    if (logits.dim() != 2 || logits.size(1) < 1 || (!fp32 && logits.scalar_type() != at::kBFloat16))
      refuse("Expected BF16 or FP32 logits[T,V], V>0");
    const int64_t t = logits.size(0), v = logits.size(1);
    if (v > NV4_LOGPROB_MAX_VOCAB) {
      const std::string text = "Expected a vocabulary of at most " + std::to_string(NV4_LOGPROB_MAX_VOCAB);
      refuse(text.c_str());
    }
    if (!shaped(targets, at::kLong, {t})) refuse("Expected INT64 targets[T]");
    if (k < 0 || k > NV4_LOGPROB_MAX_TOP) {
      const std::string text = "top_k must be in 0.." + std::to_string(NV4_LOGPROB_MAX_TOP);
      refuse(text.c_str());
    }
    if (!logits.is_cuda() || !targets.is_cuda() || targets.get_device() != logits.get_device() ||
        !targets.is_contiguous())
      refuse("All tensors must be on one CUDA device, targets contiguous");
    if ((v > 1 && logits.stride(1) != 1) || (t > 1 && logits.stride(0) < v))
      refuse("The logits of a row must be contiguous, and rows must not overlap");
    at::Tensor out[5] = {fresh(logits, {t}, at::kFloat), fresh(logits, {t}, at::kLong), fresh(logits, {t}, at::kFloat)};
    if (k) out[3] = fresh(logits, {t, k}, at::kFloat), out[4] = fresh(logits, {t, k}, at::kLong);
    if (t) {
      const int64_t nbytes = nv4_token_logprobs_workspace_bytes(t, v, k);
      at::Tensor ws;
      if (nbytes) ws = fresh(logits, {nbytes}, at::kByte);
      launch(logits.get_device(), "nv4_token_logprobs", [&](void* stream) {
        return nv4_token_logprobs(
            logits.data_ptr(), fp32, static_cast<const int64_t*>(targets.data_ptr()),
            static_cast<float*>(out[0].data_ptr()), static_cast<int64_t*>(out[1].data_ptr()),
            static_cast<float*>(out[2].data_ptr()), k ? static_cast<float*>(out[3].data_ptr()) : nullptr,
            k ? static_cast<int64_t*>(out[4].data_ptr()) : nullptr, nbytes ? ws.data_ptr() : nullptr, nbytes, t, v,
            logits.stride(0), k, stream);
      });
    }
    PyObject* none = Py_None;
    return Py_BuildValue("(NNNNN)", THPVariable_Wrap(out[0]), THPVariable_Wrap(out[1]), THPVariable_Wrap(out[2]),
                         k ? THPVariable_Wrap(out[3]) : Py_NewRef(none), k ? THPVariable_Wrap(out[4]) : Py_NewRef(none));
  });
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
constexpr PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}

PyMethodDef kMethods[] = {method<py_check_cache>("check_cache"), method<py_attention>("attention"),
                          method<py_store>("store"), method<py_step_tables>("step_tables"),
                          method<py_logprobs>("logprobs"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_nv4_serving", nullptr, -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__nv4_serving(void) { return PyModule_Create(&kModule); }
