// status.hip — the host's one look at a launch: whether any row's status bit is set, and whether
// any id lies outside its range.
//
// The sampler and scoring calls raise the reference's ValueErrors (dsv41_train/rl/rollout.py:145-146,
// models/dsv4/model.py:725-727), so every checked call ends with this question.  Asked with
// tensor operations it took a compare, a reduction and a copy back behind the launch, and the
// host's wake-up from its wait: 15 us of the 75 us of an 8-row call.  Here one workgroup answers
// into pinned memory that the host watches.  (An empty launch and hipStreamSynchronize take
// 11.4 us on this machine, a launch and a watched word 6.0.)  Bound by its loads' latency up to a
// few thousand values, then by what one CU reads: 1000000 statuses 38 us a call with four 16-byte
// loads in flight per thread (114 with single ones), 30 by tensor operations, which the Python
// calls use above 2^18.

#include "status.h"

namespace dsv41 {
namespace status {

// flags[0]: 1 + (1 if some status is set) + (2 if some id lies outside [0, limit)).
__global__ __launch_bounds__(NT) void check_kernel(const int32_t* st, int64_t n, const int64_t* ids, int64_t n_ids,
                                                   int64_t limit, int32_t* flags) {
  const int set = __syncthreads_or(any_of(st, n, [](int32_t s) { return s != 0; }));
  const int outside =
      __syncthreads_or(any_of(ids, n_ids, [=](int64_t t) { return (uint64_t)t >= (uint64_t)max(limit, (int64_t)0); }));
  if (threadIdx.x == 0)
    __hip_atomic_store(flags, 1 + (set ? 1 : 0) + (outside ? 2 : 0), __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_SYSTEM);
}

}  // namespace status
}  // namespace dsv41

using namespace dsv41;

extern "C" int dsv41_check_wait(const int32_t* st, int64_t n, const int64_t* ids, int64_t n_ids, int64_t limit,
                                int32_t* flags, void* stream) {
  if (n < 0 || n_ids < 0 || (n > 0 && !st) || (n_ids > 0 && !ids) || !flags)
    return fail(DSV41_E_INVALID, "check: statuses, ids and flags are required");
  hipStream_t s = static_cast<hipStream_t>(stream);
  __atomic_store_n(flags, 0, __ATOMIC_RELAXED);
  hipLaunchKernelGGL(status::check_kernel, dim3(1), dim3(status::NT), 0, s, st, n, ids, n_ids, limit, flags);
  DSV41_HIP_CHECK(hipGetLastError());
  int got;
  if (int rc = status::watch(flags, s, got)) return rc;
  return got - 1;
}
