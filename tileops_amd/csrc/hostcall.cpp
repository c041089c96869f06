// Host side of the serving-step calls on plain tensors: checks, output allocation and the C entry point in one native call.
//
// A decode step's bookkeeping runs 3 to 6 us on the device; checks, allocations and argument conversions in the interpreter made the
// host, not the device, set the pace of small steps.  Host time of a call, interpreter and operator registry / here: page allocation for
// 64 sequences 16.8 / 5.9 us (7.5 with an allocation per output), release 12.8 / 5.5 us, append + rows read back 36.8 / 12 us, attention over
// 300 tokens 17.8 / 6.3 us (less than its kernel takes).
//
// Every function here returns None when a call is not for it -- a tensor that is not a plain one on the current device, a gradient, a
// tracer, a dispatch mode or a function mode in force, a check that does not hold -- and has then done nothing: the op's Python path takes the call and says what
// is wrong with it.  Otherwise it returns the outputs, or the C entry point's negative error code.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/PyInterpreter.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <utility>

#include "../../include/mi355_tileops.h"

namespace {

using at::IntArrayRef;
using at::ScalarType;
using at::Tensor;

const c10::DispatchKeySet kNotPlain({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot, c10::DispatchKey::Conjugate, c10::DispatchKey::Negative,
                                     c10::DispatchKey::ZeroTensor, c10::DispatchKey::Functionalize, c10::DispatchKey::FuncTorchBatched,
                                     c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::FuncTorchVmapMode, c10::DispatchKey::Batched,
                                     c10::DispatchKey::FuncTorchDynamicLayerFrontMode, c10::DispatchKey::FuncTorchDynamicLayerBackMode,
                                     c10::DispatchKey::Tracer});

// Modes on the level of torch's functions want to see the call, all but the one that a default device sets: it only fills in the device
// of factory functions, and programs keep it set.
PyTypeObject* g_default_device_mode = nullptr;
bool function_modes() {
  using Stack = at::impl::PythonTorchFunctionTLS;
  if (!at::impl::torch_function_mode_enabled()) return false;
  for (int64_t i = 0; i < Stack::stack_len(); i++)
    if (Py_TYPE(Stack::get_stack_at(i)->ptr(getPyInterpreter())) != g_default_device_mode) return true;
  return false;
}

// The conditions of one call: a device index that is the current one, and no mode that wants to see the call.
struct Call {
  c10::Device device;
  bool ok, grad;
  explicit Call(long index) : device(c10::DeviceType::CUDA, (c10::DeviceIndex)index), grad(at::GradMode::is_enabled()) {
    ok = !c10::impl::TorchDispatchModeTLS::any_modes_set() && !function_modes() && !c10::impl::tls_local_dispatch_key_set().included_.has_any(kNotPlain) &&
         c10::impl::VirtualGuardImpl(c10::DeviceType::CUDA).getDevice() == device;
  }
  const Tensor* plain(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return fail();
    const Tensor& t = THPVariable_Unpack(o);
    if (t.device() != device || t.layout() != c10::kStrided || t.key_set().has_any(kNotPlain) || (grad && t.requires_grad())) return fail();
    return &t;
  }
  // A contiguous tensor of this type and shape.
  const Tensor* dense(PyObject* o, ScalarType type, IntArrayRef shape) {
    const Tensor* t = plain(o);
    if (!t || t->scalar_type() != type || t->sizes() != shape || !t->is_contiguous()) return fail();
    return t;
  }
  const Tensor* optional(PyObject* o, ScalarType type, IntArrayRef shape) { return o == Py_None ? nullptr : dense(o, type, shape); }
  // Block-table rows that do not overlap; width < 0: any.
  const Tensor* table(PyObject* o, int64_t batch, int64_t width, int64_t* stride) {
    const Tensor* t = plain(o);
    if (!t || t->scalar_type() != ScalarType::Int || t->dim() != 2 || t->size(0) != batch || t->size(1) < 1 || (width >= 0 && t->size(1) != width) ||
        t->stride(1) != 1 || (batch > 1 && t->stride(0) < t->size(1)))
      return fail();
    *stride = batch > 1 ? t->stride(0) : t->size(1);
    return t;
  }
  // The function behind at::empty on this device, without the dispatcher before it.
  Tensor empty(IntArrayRef shape, ScalarType type) const { return Tensor(at::detail::empty_cuda(shape, type, device, std::nullopt)); }
  // Several small outputs of a call in one allocation (each 64-byte aligned; freed with the last of them).
  template <size_t N> std::array<Tensor, N> empties(const std::pair<int64_t, ScalarType> (&of)[N]) const {
    int64_t at[N], bytes = 0;
    for (size_t i = 0; i < N; i++) {
      at[i] = bytes;
      bytes += (of[i].first * (int64_t)c10::elementSize(of[i].second) + 63) / 64 * 64;
    }
    const Tensor block = empty({bytes}, ScalarType::Byte);
    std::array<Tensor, N> out;
    for (size_t i = 0; i < N; i++) {
      out[i] = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(block.storage()), block.key_set(), c10::scalarTypeToTypeMeta(of[i].second));
      c10::TensorImpl* t = out[i].unsafeGetTensorImpl();
      t->set_storage_offset(at[i] / (int64_t)c10::elementSize(of[i].second));
      t->set_sizes_contiguous({of[i].first});
    }
    return out;
  }
  const Tensor* fail() {
    ok = false;
    return nullptr;
  }
};

void* ptr(const Tensor* t) { return t ? t->data_ptr() : nullptr; }
int code16(ScalarType t) { return t == ScalarType::BFloat16 ? MI355_DT_BF16 : t == ScalarType::Half ? MI355_DT_FP16 : -1; }
int side_code(ScalarType t) { return t == ScalarType::Float ? MI355_DT_FP32 : code16(t); }

// Integer arguments behind the tensors.
struct Ints {
  PyObject* const* args;
  bool ok = true;
  int64_t operator()(int i) {
    const int64_t v = PyLong_AsLongLong(args[i]);
    if (v == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return v;
  }
};

PyObject* none() { Py_RETURN_NONE; }

// What a call writes in place counts as a new version of the tensor, as it does through the registered operator.
void written(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

PyObject* result(int rc, std::initializer_list<const Tensor*> outs) {
  if (rc != MI355_OK) return PyLong_FromLong(rc);
  if (outs.size() == 1) return THPVariable_Wrap(**outs.begin());
  PyObject* tuple = PyTuple_New((Py_ssize_t)outs.size());
  if (!tuple) return nullptr;
  Py_ssize_t i = 0;
  for (const Tensor* t : outs) {
    PyObject* o = THPVariable_Wrap(*t);
    if (!o) {
      Py_DECREF(tuple);
      return nullptr;
    }
    PyTuple_SET_ITEM(tuple, i++, o);
  }
  return tuple;
}

// (cache_seqlens, block_table, free_pages, free_count, cu_seqlens_q, total_q, batch, max_pages, num_pages, page_size, device, stream)
PyObject* kv_alloc(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12) return none();
  Ints v{a};
  const int64_t batch = v(6), width = v(7), pages = v(8), page = v(9), index = v(10), stream = v(11);
  const int64_t total = a[5] == Py_None ? (a[4] == Py_None ? batch : -1) : v(5);
  if (!v.ok || total < 0 || total > INT32_MAX || (a[4] == Py_None && total != batch)) return none();
  Call c(index);
  int64_t stride = 0;
  const Tensor* table = c.table(a[1], batch, width, &stride);
  const Tensor *cached = c.dense(a[0], ScalarType::Int, {batch}), *list = c.dense(a[2], ScalarType::Int, {pages}),
               *count = c.dense(a[3], ScalarType::Int, {1}), *cu = c.optional(a[4], ScalarType::Int, {batch + 1});
  if (!c.ok) return none();
  const auto [slots, positions, lens, refused, left] = c.empties<5>(
      {{total, ScalarType::Long}, {total, ScalarType::Int}, {batch, ScalarType::Int}, {batch, ScalarType::Bool}, {1, ScalarType::Int}});
  const int rc = mi355_kv_alloc((const int32_t*)ptr(cached), (const int32_t*)ptr(cu), (int32_t*)ptr(table), stride, (int)width, (const int32_t*)ptr(list),
                                (const int32_t*)ptr(count), (int64_t*)slots.data_ptr(), (int32_t*)positions.data_ptr(), (int32_t*)lens.data_ptr(),
                                (uint8_t*)refused.data_ptr(), (int32_t*)left.data_ptr(), (int)batch, (int)total, (int)page, (int)pages, (void*)stream);
  written({table});
  return result(rc, {&slots, &positions, &lens, &refused, &left});
  END_HANDLE_TH_ERRORS
}

// (finished, seqlens, block_table, free_pages, free_count, batch, max_pages, num_pages, page_size, device, stream)
PyObject* kv_release(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11) return none();
  Ints v{a};
  const int64_t batch = v(5), width = v(6), pages = v(7), page = v(8), index = v(9), stream = v(10);
  if (!v.ok) return none();
  Call c(index);
  int64_t stride = 0;
  const Tensor* table = c.table(a[2], batch, width, &stride);
  const Tensor *finished = c.dense(a[0], ScalarType::Bool, {batch}), *lens = c.dense(a[1], ScalarType::Int, {batch}),
               *list = c.dense(a[3], ScalarType::Int, {pages}), *count = c.dense(a[4], ScalarType::Int, {1});
  if (!c.ok) return none();
  const auto [lens_out, count_out] = c.empties<2>({{batch, ScalarType::Int}, {1, ScalarType::Int}});
  const int rc = mi355_kv_release((const uint8_t*)ptr(finished), (const int32_t*)ptr(lens), (const int32_t*)ptr(table), stride, (int)width, (int32_t*)ptr(list),
                                  (const int32_t*)ptr(count), (int32_t*)lens_out.data_ptr(), (int32_t*)count_out.data_ptr(), (int)batch, (int)page, (int)pages,
                                  (void*)stream);
  written({list});
  return result(rc, {&lens_out, &count_out});
  END_HANDLE_TH_ERRORS
}

// Rows [tokens, heads, dim] with contiguous heads and an even token stride.
const Tensor* rows(Call& c, PyObject* o, ScalarType type, int64_t tokens, int64_t heads, int64_t dim) {
  const Tensor* t = c.plain(o);
  if (!t || t->scalar_type() != type || t->dim() != 3 || t->size(0) != tokens || t->size(1) != heads || t->size(2) != dim) return c.fail();
  if (tokens > 0 && (t->stride(2) != 1 || (heads > 1 && t->stride(1) != dim) || t->stride(0) % 2 != 0)) return c.fail();
  return t;
}

// (q, k, v, q_weight, k_weight, cos_table, sin_table, positions, slot_mapping, k_cache, v_cache, k_scale, v_scale,
//  heads, heads_kv, dim, page_size, rotary_dim, interleaved, cache (0: as q, else a type code), eps, device, stream)
PyObject* qk_norm_rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 23) return none();
  Ints v{a};
  const int64_t heads = v(13), heads_kv = v(14), dim = v(15), page = v(16), rotary = v(17), interleaved = v(18), kind = v(19), index = v(21), stream = v(22);
  const double eps = PyFloat_AsDouble(a[20]);
  if (!v.ok || PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  Call c(index);
  const Tensor* q = c.plain(a[0]);
  if (!q || q->dim() != 3) return none();
  const ScalarType type = q->scalar_type();
  const int x_code = code16(type);
  const int64_t tokens = q->size(0);
  if (x_code < 0 || tokens > INT32_MAX) return none();
  q = rows(c, a[0], type, tokens, heads, dim);
  const Tensor *k = rows(c, a[1], type, tokens, heads_kv, dim), *val = rows(c, a[2], type, tokens, heads_kv, dim);
  const Tensor* slots = c.dense(a[8], ScalarType::Long, {tokens});
  const Tensor *weights[2] = {nullptr, nullptr}, *cos = nullptr, *sin = nullptr, *positions = nullptr;
  ScalarType weight_type = type, table_type = type;
  for (int i = 0; i < 2; i++) {
    if (a[3 + i] == Py_None) continue;
    weights[i] = c.plain(a[3 + i]);
    if (!weights[i]) return none();
    if (i == 1 && weights[0] && weights[1]->scalar_type() != weight_type) return none();
    weight_type = weights[i]->scalar_type();
    if (weight_type != type && weight_type != ScalarType::Float) return none();
    weights[i] = c.dense(a[3 + i], weight_type, {dim});
  }
  if (rotary > 0) {
    cos = c.plain(a[5]);
    if (!cos || cos->dim() != 2 || cos->size(0) < 1) return none();
    table_type = cos->scalar_type();
    if (table_type != type && table_type != ScalarType::Float) return none();
    const int64_t shape[2] = {cos->size(0), rotary / 2};
    cos = c.dense(a[5], table_type, shape);
    sin = c.dense(a[6], table_type, shape);
    positions = c.dense(a[7], ScalarType::Int, {tokens});
  } else if (a[5] != Py_None || a[6] != Py_None) {
    return none();
  }
  const Tensor* kc = c.plain(a[9]);
  if (!kc || kc->dim() < 1 || kc->size(0) < 1 || !c.ok) return none();
  const int64_t first = kc->size(0);
  const Tensor *vc, *ks = nullptr, *vs = nullptr;
  int64_t pool = first;
  if (kind == MI355_DT_FP4_E2M1) {
    const int64_t codes[4] = {first, heads_kv, page, dim / 2}, scales[4] = {first, heads_kv, page, dim / 32};
    kc = c.dense(a[9], ScalarType::Byte, codes);
    vc = c.dense(a[10], ScalarType::Byte, codes);
    ks = c.dense(a[11], ScalarType::Byte, scales);
    vs = c.dense(a[12], ScalarType::Byte, scales);
    pool = first * page;
  } else {
    const bool fp8 = kind == MI355_DT_FP8_E4M3FN;
    const int64_t shape[3] = {first, heads_kv, dim}, scales[2] = {first, heads_kv};
    if (first % page != 0) return none();
    kc = c.dense(a[9], fp8 ? ScalarType::Float8_e4m3fn : type, shape);
    vc = c.dense(a[10], fp8 ? ScalarType::Float8_e4m3fn : type, shape);
    if (fp8) {
      ks = c.dense(a[11], ScalarType::Float, scales);
      vs = c.dense(a[12], ScalarType::Float, scales);
    } else if (a[11] != Py_None || a[12] != Py_None) {
      return none();
    }
  }
  if (!c.ok || (((uintptr_t)ptr(q) | (uintptr_t)ptr(k) | (uintptr_t)ptr(val)) & 3)) return none();
  const Tensor out = c.empty({tokens, heads, dim}, type);
  const int rc = mi355_qk_norm_rope_append(ptr(q), ptr(k), ptr(val), q->stride(0), k->stride(0), val->stride(0), ptr(weights[0]), ptr(weights[1]),
                                           side_code(weight_type), ptr(cos), ptr(sin), side_code(table_type), cos ? cos->size(0) : 0,
                                           (const int32_t*)ptr(positions), (const int64_t*)ptr(slots), out.data_ptr(), ptr(kc), ptr(vc), ptr(ks), ptr(vs),
                                           (int)tokens, (int)heads, (int)heads_kv, (int)dim, (int)rotary, (int)interleaved, eps, (int)page, pool, x_code,
                                           kind == 0 ? x_code : (int)kind, (void*)stream);
  written({kc, vc, ks, vs});
  return result(rc, {&out});
  END_HANDLE_TH_ERRORS
}

struct Fp4Cache {
  const Tensor *k, *v, *ks, *vs;
  Fp4Cache(Call& c, PyObject* const* a, int64_t pages, int64_t heads_kv, int64_t page, int64_t dim) {
    const int64_t codes[4] = {pages, heads_kv, page, dim / 2}, scales[4] = {pages, heads_kv, page, dim / 32};
    k = c.dense(a[0], ScalarType::Byte, codes);
    v = c.dense(a[1], ScalarType::Byte, codes);
    ks = c.dense(a[2], ScalarType::Byte, scales);
    vs = c.dense(a[3], ScalarType::Byte, scales);
  }
};

// (k, v, k_scale, v_scale, slot_mapping, heads_kv, dim, page_size, type code, device, stream)
PyObject* kv_gather_fp4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11) return none();
  Ints v{a};
  const int64_t heads_kv = v(5), dim = v(6), page = v(7), type = v(8), index = v(9), stream = v(10);
  if (!v.ok) return none();
  Call c(index);
  const Tensor *k = c.plain(a[0]), *slots = c.plain(a[4]);
  if (!c.ok || k->dim() != 4 || k->size(0) < 1 || slots->dim() != 1 || slots->size(0) > INT32_MAX) return none();
  const int64_t pages = k->size(0), tokens = slots->size(0);
  const Fp4Cache cache(c, a, pages, heads_kv, page, dim);
  slots = c.dense(a[4], ScalarType::Long, {tokens});
  if (!c.ok) return none();
  const ScalarType out_type = type == MI355_DT_BF16 ? ScalarType::BFloat16 : ScalarType::Half;
  const Tensor ko = c.empty({tokens, heads_kv, dim}, out_type), vo = c.empty({tokens, heads_kv, dim}, out_type);
  const int rc = mi355_kv_gather_fp4(ptr(cache.k), ptr(cache.v), ptr(cache.ks), ptr(cache.vs), (const int64_t*)ptr(slots), ko.data_ptr(), vo.data_ptr(),
                                     (int)tokens, (int)heads_kv, (int)dim, (int)page, pages * page, (int)type, (void*)stream);
  return result(rc, {&ko, &vo});
  END_HANDLE_TH_ERRORS
}

// (k, v, k_scale, v_scale, q, real_seqlen_kv, block_table, batch, q_len, heads, heads_kv, pages, dim, page_size, is_causal, sm_scale, softcap,
//  workspace bytes, type code of q that they are for, device, stream)
PyObject* decode_fp4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 21) return none();
  Ints v{a};
  const int64_t batch = v(7), q_len = v(8), heads = v(9), heads_kv = v(10), pages = v(11), dim = v(12), page = v(13), causal = v(14), bytes = v(17),
                type = v(18), index = v(19), stream = v(20);
  const double sm_scale = PyFloat_AsDouble(a[15]), softcap = PyFloat_AsDouble(a[16]);
  if (!v.ok || PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  Call c(index);
  const ScalarType q_type = type == MI355_DT_BF16 ? ScalarType::BFloat16 : ScalarType::Half;
  const int64_t shape[4] = {batch, q_len, heads, dim}, shape1[3] = {batch, heads, dim};
  const Tensor* q = q_len == 1 ? c.dense(a[4], q_type, shape1) : c.dense(a[4], q_type, shape);
  const Fp4Cache cache(c, a, pages, heads_kv, page, dim);
  int64_t stride = 0;
  const Tensor *lens = c.dense(a[5], ScalarType::Int, {batch}), *table = c.table(a[6], batch, -1, &stride);
  if (!c.ok || table->size(1) > INT32_MAX) return none();
  const Tensor out = c.empty(q->sizes(), q_type), workspace = c.empty({bytes}, ScalarType::Byte);
  const int rc = mi355_gqa_paged_decode_fp4(ptr(q), ptr(cache.k), ptr(cache.v), ptr(cache.ks), ptr(cache.vs), (const int32_t*)ptr(lens),
                                            (const int32_t*)ptr(table), stride, (int)table->size(1), out.data_ptr(), workspace.data_ptr(), (size_t)bytes,
                                            (int)batch, (int)q_len, (int)heads, (int)heads_kv, (int)dim, (int)page, pages * page, (int)type, (float)sm_scale,
                                            (float)softcap, (int)causal, (void*)stream);
  return result(rc, {&out});
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"kv_alloc", (PyCFunction)(void (*)(void))kv_alloc, METH_FASTCALL, nullptr},
    {"kv_release", (PyCFunction)(void (*)(void))kv_release, METH_FASTCALL, nullptr},
    {"qk_norm_rope_append", (PyCFunction)(void (*)(void))qk_norm_rope_append, METH_FASTCALL, nullptr},
    {"kv_gather_fp4", (PyCFunction)(void (*)(void))kv_gather_fp4, METH_FASTCALL, nullptr},
    {"decode_fp4", (PyCFunction)(void (*)(void))decode_fp4, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_hostcall", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__hostcall(void) {
  PyObject* device = PyImport_ImportModule("torch.utils._device");
  if (!device) return nullptr;
  g_default_device_mode = (PyTypeObject*)PyObject_GetAttrString(device, "DeviceContext");  // (kept for the life of the process)
  Py_DECREF(device);
  return g_default_device_mode ? PyModule_Create(&kModule) : nullptr;
}
