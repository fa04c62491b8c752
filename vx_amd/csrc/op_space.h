/*
 * op_space.h -- the workspaces that the library keeps for the ops of
 * ops_batch.cpp and ops_packed.cpp: one block per (device, stream), shared by the
 * launches on that stream, which run in order. A block grows as it is asked for (the old
 * one freed in the stream's order) and is freed, in that order, when the
 * calling thread's stream is set to another one; the default stream's stays.
 * A call that needs more than kOpSpaceKept has it for itself.
 */
#ifndef VX_AMD_OP_SPACE_H
#define VX_AMD_OP_SPACE_H

#include <hip/hip_runtime.h>

#include <cstdint>
#include <mutex>

namespace vxk {

/* The most that is kept for a stream, as for the GEMM's. 4096 sequences of 32
 * heads on 8 of 128 over 2048 keys take 130 MiB; for itself such a call takes 585
 * us for 565, and 930 for 576 where the GPU was waited for before it, which gives
 * the memory back. The caller's workspace costs neither. */
constexpr int64_t kOpSpaceKept = (int64_t)128 << 20;

/* Held from op_space through the launches that use the block, so that a growth
 * on one thread cannot free a block another is about to use. */
std::unique_lock<std::mutex> op_space_lock();

/* At least `bytes` for launches on `stream` of the current device, or NULL
 * when the memory cannot be had. The caller holds the lock. */
char *op_space(size_t bytes, hipStream_t stream);

/* The same for one call, which gives it back after its launches; no lock. */
char *op_space_once(size_t bytes, hipStream_t stream);
void op_space_once_free(char *base, hipStream_t stream);

/* Frees the blocks kept for `stream` (nothing for the default stream or one
 * that is capturing); returns how many. The stream must still exist. */
int op_space_release_stream(hipStream_t stream);

/* Blocks held, and their bytes. */
void op_space_stats(int64_t *blocks, int64_t *bytes);

} // namespace vxk

#endif /* VX_AMD_OP_SPACE_H */
