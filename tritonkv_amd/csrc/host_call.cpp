// Host side of a repeated decode call, as a CPython module (_hostcall).
//
// A decode loop calls the same entry point with the same caches, buffers and
// options every step; only q, the new token's rows and the output may be other
// tensors of the same form.  The Python wrapper checks and plans such a call
// once and hands its argument block here; later calls compare each tensor
// (storage, shape, dtype, device, layout) with the form that was checked, refresh the
// pointers that may move and launch.  Doing the comparison in Python took most
// of the 9.7 us an eager Qwen2.5-1.5B-shape step (B = 1, ctx 512) spent on the
// host; with it here such steps run back to back at the GPU's 6.0 us.
//
// Nothing is cached by a tensor object's identity: every property is read from
// the tensors passed, on every call.  A tensor without plain storage
// (functorch wrappers, fake tensors) never matches, and the caller takes the full
// path.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <cstring>
#include <vector>

#include "../../include/tkv.h"

namespace {

typedef int (*EntryFn)(const void*, tkv_stream_t);  // any entry that takes an argument block and a stream
typedef int (*ChannelFn)(const tkv_decode_args*, const void*, const void*, const int32_t*, int32_t,
                         tkv_stream_t);

constexpr const char* kName = "tritonkv_amd.prepared_call";
constexpr int kFixed = -1;  // offset of a slot whose storage must be the same

// The form a tensor argument must have.
struct Slot {
  bool present;
  int offset;  // of its pointer in the argument block, or kFixed
  uintptr_t align_mask;
  const void* ptr;
  c10::ScalarType dtype;
  c10::Device device{c10::kCPU};
  std::vector<int64_t> sizes;
  std::vector<int64_t> strides;  // of a tensor that is used as it is strided; else empty: contiguous
  std::vector<int64_t> layout;   // its strides in bytes, whichever form it has
  int64_t entry;                 // bytes of an entry
  uintptr_t span;                // bytes from its first entry to the end of its last
  bool apart, written;           // shares no memory with other such slots if one of the two is written
};

constexpr int kStrided = 1, kApart = 2, kWritten = 4;  // a slot's flags
constexpr size_t kMaxApart = 16;                       // such slots of a call

constexpr size_t kMaxArgs = 2048;  // bytes of an argument block

struct Call {
  size_t size;
  alignas(16) char args[kMaxArgs];
  void* entry;
  c10::DeviceIndex device;
  std::vector<Slot> slots;
  bool channel;  // tkv_channel_decode_attention with:
  const void *k_res, *v_res;
  const int32_t* res_lens;
  int32_t res_cap;
};

// The tensor's storage if it is an ordinary tensor, contiguous or of these strides, else null.
void* plain_pointer(const at::Tensor& t, const std::vector<int64_t>& strides) {
  const auto* impl = t.unsafeGetTensorImpl();
  if (!impl->has_storage() || impl->is_python_dispatch() || t.layout() != c10::kStrided ||
      impl->key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::Functionalize,
                                                   c10::DispatchKey::FuncTorchBatched,
                                                   c10::DispatchKey::FuncTorchGradWrapper})) ||
      !(strides.empty() ? t.is_contiguous() : t.strides() == c10::IntArrayRef(strides)))
    return nullptr;
  return t.mutable_data_ptr();
}

// Bytes from a slot's first entry to the end of its last over the axes of smaller strides than `below`.
int64_t extent(const Slot& s, int64_t below) {
  int64_t n = s.entry;
  for (size_t d = 0; d < s.sizes.size(); ++d)
    if (s.layout[d] < below) n += (s.sizes[d] - 1) * s.layout[d];
  return n;
}

// Whether two slots' tensors, `between` bytes apart, lie in turn over a stride that both have (queries and
// keys of one projection's output), and so share nothing although their spans do.
bool in_turn(const Slot& a, const Slot& b, int64_t between) {
  auto steps = [](const Slot& s, int64_t period) {  // every wider stride is a multiple of the period
    for (size_t d = 0; d < s.sizes.size(); ++d)
      if (s.sizes[d] > 1 && s.layout[d] > period && s.layout[d] % period) return false;
    return true;
  };
  for (size_t d = 0; d < a.sizes.size(); ++d) {
    const int64_t period = a.layout[d];
    if (a.sizes[d] < 2 || period <= 0) continue;
    for (size_t x = 0; x < b.sizes.size(); ++x) {
      if (b.sizes[x] < 2 || b.layout[x] != period || !steps(a, period) || !steps(b, period)) continue;
      const int64_t at = (between % period + period) % period;
      if (extent(a, period) <= at && at + extent(b, period) <= period) return true;
      break;
    }
  }
  return false;
}

void free_call(PyObject* capsule) {
  delete static_cast<Call*>(PyCapsule_GetPointer(capsule, kName));
}

// prepare(args: bytes, entry: int, device: int, slots: tuple of (tensor or None,
//   offset or -1, alignment[, flags: 1 the argument block holds its strides, 2 it must
//   not share memory with a slot of flag 4, 4 it is written]),
//   window: None or (k_res, v_res, res_lens, res_cap))
PyObject* prepare(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    char* bytes;
    Py_ssize_t len;
    if (n != 5 || PyBytes_AsStringAndSize(a[0], &bytes, &len) || len > (Py_ssize_t)kMaxArgs ||
        (a[4] != Py_None && len != sizeof(tkv_decode_args)) || !PyTuple_Check(a[3])) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "prepare: wrong arguments");
      return nullptr;
    }
    auto call = std::make_unique<Call>();
    call->size = len;
    std::memcpy(call->args, bytes, len);
    call->entry = PyLong_AsVoidPtr(a[1]);
    call->device = (c10::DeviceIndex)PyLong_AsLong(a[2]);
    size_t apart = 0;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(a[3]); ++i) {
      PyObject *t;
      int offset, align, flags = 0;
      if (!PyArg_ParseTuple(PyTuple_GET_ITEM(a[3], i), "Oii|i", &t, &offset, &align, &flags)) return nullptr;
      if (offset != kFixed && (offset < 0 || offset + (Py_ssize_t)sizeof(void*) > len)) {
        PyErr_SetString(PyExc_ValueError, "prepare: an offset past the argument block");
        return nullptr;
      }
      Slot s{};
      s.present = t != Py_None;
      s.offset = offset;
      s.align_mask = (uintptr_t)align - 1;
      if (s.present) {
        if (!THPVariable_Check(t)) {
          PyErr_SetString(PyExc_TypeError, "prepare: a slot holds no tensor");
          return nullptr;
        }
        const at::Tensor& v = THPVariable_Unpack(t);
        if (flags & kStrided && !v.is_contiguous()) s.strides = v.strides().vec();
        s.ptr = plain_pointer(v, s.strides);
        if (!s.ptr || ((uintptr_t)s.ptr & s.align_mask)) Py_RETURN_NONE;  // not a call to keep
        s.dtype = v.scalar_type();
        s.device = v.device();
        s.sizes = v.sizes().vec();
        s.written = flags & kWritten;
        s.apart = s.written || flags & kApart;
        s.entry = v.element_size();
        for (int64_t d = 0; d < v.dim(); ++d) s.layout.push_back(s.entry * v.stride(d));
        s.span = extent(s, INT64_MAX);
        if (s.apart && ++apart > kMaxApart) {
          PyErr_SetString(PyExc_ValueError, "prepare: too many slots that must lie apart");
          return nullptr;
        }
      }
      call->slots.push_back(std::move(s));
    }
    call->channel = a[4] != Py_None;
    if (call->channel) {
      call->k_res = PyLong_AsVoidPtr(PyTuple_GetItem(a[4], 0));
      call->v_res = PyLong_AsVoidPtr(PyTuple_GetItem(a[4], 1));
      PyObject* lens = PyTuple_GetItem(a[4], 2);
      call->res_lens = lens == Py_None ? nullptr : static_cast<const int32_t*>(PyLong_AsVoidPtr(lens));
      call->res_cap = (int32_t)PyLong_AsLong(PyTuple_GetItem(a[4], 3));
    }
    if (PyErr_Occurred()) return nullptr;
    PyObject* capsule = PyCapsule_New(call.get(), kName, free_call);
    if (capsule) call.release();
    return capsule;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// run(call, *tensors): the entry's status, or None when a tensor does not have
// the form that was prepared (nothing was launched).
PyObject* run(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n < 1) {
    PyErr_SetString(PyExc_TypeError, "run: no call");
    return nullptr;
  }
  const Call* call = static_cast<const Call*>(PyCapsule_GetPointer(a[0], kName));
  if (!call) return nullptr;
  try {
    if ((size_t)(n - 1) != call->slots.size()) Py_RETURN_NONE;
    alignas(16) char args[kMaxArgs];
    std::memcpy(args, call->args, call->size);
    struct {
      uintptr_t begin, end;
      const Slot* slot;
    } apart[kMaxApart];
    size_t spans = 0;
    for (size_t i = 0; i < call->slots.size(); ++i) {
      const Slot& s = call->slots[i];
      PyObject* o = a[i + 1];
      if (o == Py_None) {
        if (s.present) Py_RETURN_NONE;
        continue;
      }
      if (!s.present || !THPVariable_Check(o)) Py_RETURN_NONE;
      const at::Tensor& t = THPVariable_Unpack(o);
      if (t.scalar_type() != s.dtype || t.device() != s.device || t.sizes() != c10::IntArrayRef(s.sizes))
        Py_RETURN_NONE;
      void* p = plain_pointer(t, s.strides);
      if (!p || ((uintptr_t)p & s.align_mask) || (s.offset == kFixed && p != s.ptr)) Py_RETURN_NONE;
      if (s.offset != kFixed) std::memcpy(args + s.offset, &p, sizeof p);
      if (s.apart) {
        const uintptr_t begin = (uintptr_t)p, end = begin + s.span;
        for (size_t x = 0; x < spans; ++x)
          if ((s.written || apart[x].slot->written) && begin < apart[x].end && apart[x].begin < end &&
              !in_turn(*apart[x].slot, s, (int64_t)(begin - apart[x].begin)))
            Py_RETURN_NONE;
        apart[spans++] = {begin, end, &s};
      }
    }
    c10::hip::OptionalHIPGuard guard;
    if (c10::hip::current_device() != call->device) guard.set_index(call->device);
    tkv_stream_t st = reinterpret_cast<tkv_stream_t>(c10::hip::getCurrentHIPStream(call->device).stream());
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = call->channel
             ? reinterpret_cast<ChannelFn>(call->entry)(reinterpret_cast<const tkv_decode_args*>(args), call->k_res, call->v_res, call->res_lens,
                                                        call->res_cap, st)
             : reinterpret_cast<EntryFn>(call->entry)(args, st);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// raw_stream(device): torch's current stream there as an integer, or None when
// the device is not the calling thread's current one.
PyObject* raw_stream(PyObject*, PyObject* arg) {
  const long device = PyLong_AsLong(arg);
  if (device == -1 && PyErr_Occurred()) return nullptr;
  try {
    if (c10::hip::current_device() != (c10::DeviceIndex)device) Py_RETURN_NONE;
    return PyLong_FromVoidPtr(c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyMethodDef methods[] = {
    {"prepare", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(prepare)), METH_FASTCALL, nullptr},
    {"run", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(run)), METH_FASTCALL, nullptr},
    {"raw_stream", raw_stream, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hostcall", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__hostcall() { return PyModule_Create(&module); }
