// abi_checks.h — what the device-pointer entries of the C-ABI that allocate
// nothing check before any launch: ranges, alignment, overlap, the device.
#pragma once

#include <hip/hip_runtime.h>

#include <initializer_list>
#include <string>

#include "../../include/seeml_hip.h"
#include "kernels.h"

namespace seeml_hip {

inline size_t ElemSize(int dtype) { return dtype == kF32 ? 4 : 2; }

// A byte range that a call reads or writes.
struct Span {
  const char* name;
  const void* p;
  uint64_t bytes;
  bool write;
  size_t align;
  uintptr_t lo() const { return reinterpret_cast<uintptr_t>(p); }
};

struct AbiCall {
  const char* name;
  Status Fail(const std::string& what) const {
    return Status::Fail(kUnitEngine, std::string(name) + ": " + what);
  }

  // Nulls are the caller's business (a null span is skipped). Written ranges
  // overlap nothing.
  Status Ranges(std::initializer_list<Span> spans) const {
    for (const Span& s : spans) {
      if (!s.p) continue;
      if (s.lo() % s.align) return Fail(std::string(s.name) + " is not aligned to its elements");
      if (s.bytes > UINTPTR_MAX - s.lo())
        return Fail(std::string(s.name) + " passes the end of memory");
    }
    for (const Span& s : spans) {
      if (!s.p || !s.write) continue;
      for (const Span& o : spans) {
        if (&o == &s || !o.p) continue;
        if (s.lo() < o.lo() + o.bytes && o.lo() < s.lo() + s.bytes)
          return Fail(std::string(s.name) + " overlaps " + o.name);
      }
    }
    return Status::Ok();
  }

  // The data's device is the current one, where the launch goes: on another
  // the kernels would fault.
  Status OnDevice(const void* p, void* stream, const char* what) const {
    int dev = 0;
    if (const hipError_t e = hipGetDevice(&dev); e != hipSuccess)
      return Fail(std::string("hipGetDevice: ") + hipGetErrorString(e));
    hipPointerAttribute_t at{};
    if (hipPointerGetAttributes(&at, p) != hipSuccess) {
      (void)hipGetLastError();
      return Fail(std::string(what) + " is not device memory");
    }
    if (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged)
      return Fail(std::string(what) + " is not device memory");
    if (at.type == hipMemoryTypeDevice && at.device != dev)
      return Fail(std::string(what) + " is on device " + std::to_string(at.device) +
                  ", the current one is " + std::to_string(dev));
    // hipStreamLegacy and hipStreamPerThread are the current device's.
    if (reinterpret_cast<uintptr_t>(stream) > 2) {
      int sdev = dev;
      if (hipStreamGetDevice(static_cast<hipStream_t>(stream), &sdev) != hipSuccess) {
        (void)hipGetLastError();
        return Fail("not a stream");
      }
      if (sdev != dev) return Fail("the stream is on another device than the current one");
    }
    return Status::Ok();
  }

  Status Scratch(const void* p, uint64_t bytes, uint64_t need) const {
    if (need == 0) return Status::Ok();
    if (!p || bytes < need)
      return Fail("scratch of " + std::to_string(bytes) + " bytes, " + std::to_string(need) +
                  " needed");
    return Status::Ok();
  }
};

// No exception leaves a C entry.
template <typename F>
int Entry(F&& f) {
  try {
    return ReportStandalone(f());
  } catch (...) {
    return SEEML_HIP_ERROR;
  }
}

inline Ctx On(void* stream) {
  Ctx c;
  c.stream = static_cast<hipStream_t>(stream);
  return c;
}

}  // namespace seeml_hip
