// status.h — one workgroup's look at many values, and the host's wait for what it found.
#pragma once

#include <chrono>

#include "common.h"

namespace dsv41 {
namespace status {

constexpr int NT = 1024;
// how long the host watches before it waits on the stream (and learns of a failed launch)
constexpr std::chrono::microseconds WATCH{2000};

// Whether pred holds for some a[i] of the n values: 16-byte loads, four in flight per thread, with
// single ones before the first 16-byte boundary and behind the last.
template <typename T, class Pred>
__device__ __forceinline__ bool any_of(const T* a, int64_t n, Pred pred) {
  constexpr int G = 16 / (int)sizeof(T), U = 4;
  struct alignas(16) Group {
    T v[G];
  };
  if (n <= NT) return threadIdx.x < n && pred(a[threadIdx.x]);  // 2.4 us, 2.7 the general way
  bool hit = false;
  const int64_t head = min(n, (int64_t)((16 - ((uintptr_t)a & 15)) & 15) / (int)sizeof(T));
  if (threadIdx.x < head) hit |= pred(a[threadIdx.x]);
  const Group* g = reinterpret_cast<const Group*>(a + head);
  const int64_t groups = (n - head) / G;
  int64_t i = threadIdx.x;
  for (; i + (U - 1) * NT < groups; i += U * NT) {
    Group x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = g[i + u * NT];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < G; ++k) hit |= pred(x[u].v[k]);
  }
  for (; i < groups; i += NT) {
    const Group x = g[i];
#pragma unroll
    for (int k = 0; k < G; ++k) hit |= pred(x.v[k]);
  }
  const int64_t tail = head + groups * G + threadIdx.x;
  if (tail < n) hit |= pred(a[tail]);
  return hit;
}

// What a kernel on `s` left in the word of pinned memory, which was 0 before its launch.
inline int watch(int32_t* word, hipStream_t s, int& got) {
  const auto until = std::chrono::steady_clock::now() + WATCH;
  got = 0;
  do {
    for (int i = 0; i < 64 && got == 0; ++i) got = __atomic_load_n(word, __ATOMIC_ACQUIRE);
  } while (got == 0 && std::chrono::steady_clock::now() < until);
  if (got == 0) {
    DSV41_HIP_CHECK(hipStreamSynchronize(s));
    got = __atomic_load_n(word, __ATOMIC_ACQUIRE);
    if (got == 0) return fail(DSV41_E_HIP, "check: the launch left no answer");
  }
  return DSV41_OK;
}

}  // namespace status
}  // namespace dsv41
