// The token operators' host path in ppo_amd._native.
#include "native.hpp"

#include <hip/hip_runtime.h>

namespace ppo_native {
namespace {

// The capture that the current stream of a device (its index) is in, 0 if none.
PyObject* capture_id(PyObject*, PyObject* index) {
  const long device = PyLong_AsLong(index);
  if (device == -1 && PyErr_Occurred()) return nullptr;
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  const hipError_t e = hipStreamGetCaptureInfo(
      c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream(), &status, &id);
  if (e != hipSuccess) {
    PyErr_SetString(PyExc_RuntimeError, hipGetErrorString(e));
    return nullptr;
  }
  return PyLong_FromUnsignedLongLong(status == hipStreamCaptureStatusNone ? 0 : id);
}

}  // namespace

PyMethodDef kTokenMethods[] = {{"capture_id", capture_id, METH_O, nullptr},
                               {nullptr, nullptr, 0, nullptr}};

}  // namespace ppo_native
