/*
 * op_checks.h -- what the ops of ops_batch.cpp and ops_packed.cpp check and take
 * before they launch: refusals, alignment, extents, the GPU that holds the
 * operands, and the workspace.
 */
#ifndef VX_AMD_OP_CHECKS_H
#define VX_AMD_OP_CHECKS_H

#include "../../include/vx_hip_ops.h"
#include "op_space.h"
#include "vx_hip_common.h"
#include "vx_ops_internal.h"

#include <initializer_list>

namespace vxops {
namespace {

int32_t refuse(int32_t code, const char *op, const char *why) {
  fprintf(stderr, "[Vx HIP] %s: %s\n", op, why);
  return code;
}

bool aligned16(std::initializer_list<const void *> ptrs) {
  for (const void *p : ptrs) {
    if (reinterpret_cast<uintptr_t>(p) & 15) {
      return false;
    }
  }
  return true;
}

bool aligned4(std::initializer_list<const void *> ptrs) {
  for (const void *p : ptrs) {
    if (reinterpret_cast<uintptr_t>(p) & 3) {
      return false;
    }
  }
  return true;
}

/* Makes the GPU that holds every (non-NULL) operand the current one for the
 * scope; `code` says why it cannot. */
class OnDeviceOf {
public:
  OnDeviceOf(const char *op, std::initializer_list<const void *> ptrs) {
    if (!vxops::device_present()) {
      code = refuse(VX_OP_ENODEV, op, "no GPU; this op has no host copy");
      return;
    }
    int device = -1;
    for (const void *p : ptrs) {
      if (!p) {
        continue;
      }
      const int d = vxops::device_of(p);
      if (d < 0) {
        code = refuse(VX_OP_ENOTDEV, op, "every operand must be GPU memory");
        return;
      }
      if (device >= 0 && d != device) {
        code = refuse(VX_OP_EINVAL, op, "operands of different GPUs");
        return;
      }
      device = d;
    }
    VX_HIP_CHECK(hipGetDevice(&before_));
    if (vxops::stream() && vxk::one_stream(vxops::stream())) {
      hipDevice_t of = device;
      if (hipStreamGetDevice(vxops::stream(), &of) != hipSuccess) {
        (void)hipGetLastError();
      } else if (of != device) {
        code = refuse(VX_OP_EINVAL, op, "the stream belongs to another GPU than the operands");
        return;
      }
    }
    if (device != before_) {
      VX_HIP_CHECK(hipSetDevice(device));
      moved_ = true;
    }
  }
  ~OnDeviceOf() {
    if (moved_) {
      (void)hipSetDevice(before_);
    }
  }
  OnDeviceOf(const OnDeviceOf &) = delete;
  OnDeviceOf &operator=(const OnDeviceOf &) = delete;

  int32_t code = VX_OP_OK;

private:
  int before_ = 0;
  bool moved_ = false;
};

/* A launch's workspace: the caller's, or the one kept for the stream, or (more
 * than is kept) one for this call, held through the scope. A stream that is
 * capturing a graph, or a handle of several streams, has none of the library's. */
class Space {
public:
  Space(void *given, int64_t bytes) {
    if (bytes == 0 || given) {
      base = static_cast<char *>(given);
      enough = true;
    } else if (vxk::one_stream(vxops::stream()) && !vxops::capturing()) {
      once_ = bytes > vxk::kOpSpaceKept;
      if (once_) {
        base = vxk::op_space_once((size_t)bytes, vxops::stream());
      } else {
        hold_ = vxk::op_space_lock();
        base = vxk::op_space((size_t)bytes, vxops::stream());
      }
      enough = base != nullptr;
    }
  }
  ~Space() {
    if (once_ && base) {
      vxk::op_space_once_free(base, vxops::stream());
    }
  }
  Space(const Space &) = delete;
  Space &operator=(const Space &) = delete;

  char *base = nullptr;
  bool enough = false;

private:
  bool once_ = false;
  std::unique_lock<std::mutex> hold_;
};

/* The product of extents that are each at most 2^40, or -1 past 2^62. */
int64_t product(std::initializer_list<int64_t> extents) {
  int64_t p = 1;
  for (int64_t e : extents) {
    if (e > 0 && p > (int64_t(1) << 62) / e) {
      return -1;
    }
    p *= e;
  }
  return p;
}

constexpr int64_t kMaxExtent = int64_t(1) << 40;

bool within(std::initializer_list<int64_t> extents, int64_t least) {
  for (int64_t e : extents) {
    if (e < least || e > kMaxExtent) {
      return false;
    }
  }
  return true;
}

} // namespace
} // namespace vxops

#endif /* VX_AMD_OP_CHECKS_H */
