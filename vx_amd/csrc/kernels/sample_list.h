/*
 * sample_list.h -- the list that a workgroup's threads fill together
 * (sample.hip), written once for the kernels and for the CPU check that runs
 * it on threads (tests/native/sample_list_test.cpp). Plain C++ apart from the
 * host/device qualifier.
 */
#ifndef VX_AMD_SAMPLE_LIST_H
#define VX_AMD_SAMPLE_LIST_H

#include <cstdint>

#if defined(__HIPCC__)
#define VX_LIST_FN __host__ __device__ __forceinline__
#else
#define VX_LIST_FN inline
#endif

namespace vxk {

/* `each` hands entries to its callback, on every thread of `group`; the first
 * kCap to come go into the list. How many came, the same for every thread:
 * nobody clears the count, in a next call, before all have read it. */
template <typename Group, int kCap, typename Each>
VX_LIST_FN int fill_list(const Group &group, uint32_t &count, unsigned long long (&list)[kCap],
                         Each each) {
  if (group.thread() == 0) {
    count = 0;
  }
  group.sync();
  each([&](unsigned long long entry) {
    const uint32_t at = group.add(count);
    if (at < (uint32_t)kCap) {
      list[at] = entry;
    }
  });
  group.sync();
  const int n = (int)count;
  group.sync();
  return n;
}

} // namespace vxk

#endif /* VX_AMD_SAMPLE_LIST_H */
