/*
 * op_space.cpp -- see op_space.h.
 */
#include "op_space.h"
#include "vx_hip_common.h"

#include <map>
#include <new>
#include <utility>

namespace vxk {
namespace {

struct Block {
  char *base = nullptr;
  size_t bytes = 0;
};
std::mutex blocks_mutex;
std::map<std::pair<int, hipStream_t>, Block> &blocks() {
  static auto *m = new std::map<std::pair<int, hipStream_t>, Block>();
  return *m;
}

} // namespace

std::unique_lock<std::mutex> op_space_lock() {
  return std::unique_lock<std::mutex>(blocks_mutex);
}

char *op_space(size_t bytes, hipStream_t stream) {
  int device = 0;
  VX_HIP_CHECK(hipGetDevice(&device));
  Block *b = nullptr;
  try {
    b = &blocks()[{device, stream}];
  } catch (const std::bad_alloc &) {
    return nullptr;
  }
  if (b->base && bytes <= b->bytes) {
    return b->base;
  }
  char *fresh = op_space_once(bytes, stream);
  if (!fresh) {
    return nullptr;
  }
  if (b->base) {
    VX_HIP_CHECK(hipFreeAsync(b->base, stream));
  }
  b->base = fresh;
  b->bytes = bytes;
  return b->base;
}

char *op_space_once(size_t bytes, hipStream_t stream) {
  void *fresh = nullptr;
  if (hipMallocAsync(&fresh, bytes, stream) != hipSuccess) {
    (void)hipGetLastError();
    return nullptr;
  }
  return static_cast<char *>(fresh);
}

void op_space_once_free(char *base, hipStream_t stream) {
  VX_HIP_CHECK(hipFreeAsync(base, stream));
}

int op_space_release_stream(hipStream_t stream) {
  if (!stream) {
    return 0;
  }
  /* A stream that is capturing would record the free into its graph: its
   * blocks stay until a later release finds it idle. */
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream, &status) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  if (status != hipStreamCaptureStatusNone) {
    return 0;
  }
  std::lock_guard<std::mutex> hold(blocks_mutex);
  int freed = 0;
  auto &m = blocks();
  for (auto it = m.begin(); it != m.end();) {
    if (it->first.second != stream) {
      ++it;
      continue;
    }
    if (it->second.base) {
      VX_HIP_CHECK(hipFreeAsync(it->second.base, stream));
      ++freed;
    }
    it = m.erase(it);
  }
  return freed;
}

void op_space_stats(int64_t *held, int64_t *bytes) {
  std::lock_guard<std::mutex> hold(blocks_mutex);
  *held = 0;
  *bytes = 0;
  for (const auto &e : blocks()) {
    *held += e.second.base != nullptr;
    *bytes += (int64_t)e.second.bytes;
  }
}

} // namespace vxk
