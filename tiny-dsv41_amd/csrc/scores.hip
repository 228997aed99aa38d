// scores.hip — log-probs of given tokens from their logits, with rank, entropy and the top
// alternatives, and the gradient of all of them with respect to the logits.
//
// For one row x [V] with p = softmax(x / T), m = max x and S = sum exp((x - m) / T):
//   log p_i = (x_i - m) / T - log S,   H = log S - (1 / S) sum exp((x - m) / T) (x - m) / T
// so one pass over the row (row_scan.h) gives everything but the alternatives.
//
// Alternatives.  The pass also leaves the maximum of each 32 consecutive elements in LDS.  Order the
// elements by (logit desc, index asc) and the groups by (maximum desc, index asc): every element of the
// top k lies in one of the first k groups.  For if its group G were not among them, k groups would come
// before G, and each holds an element that comes before it: a larger one, or an equal one of a lower
// index, since groups are index ranges.  So after the pass k groups at most are read again, whatever the
// logits are, and those of their elements that reach the k-th group's maximum are sorted.
//
// A row of few is cut into slices, which leave their sums and their sorted lists in the workspace for a
// second kernel.
//
// What bounds it.  4096 fp32 rows of 151936 with 64 alternatives take 379-383 us, 6.5 TB/s (7.0 is what
// nontemporal reads reach): memory, and the selections, which fall together on the workgroups of a CU.
// 1000 bf16 rows of 129280 with ranks take 50 us, 5.2 TB/s: 10.8 vector instructions an element, of which
// the exponential counts twice.  A single row, 7.3 us and 4.6 to join, is a chain of latencies.
#include <limits.h>
#include <math.h>

#include "row_scan.h"

namespace dsv41 {
namespace scores {

using rows::bf16_t;
using rows::Cut;
using rows::Elem;
using rows::GROUP;
using rows::NT;
using rows::Scale;
using rows::State;
using rows::WAVES;

constexpr int MAX_K = 1024;
constexpr int MAX_GROUPS = 5120;                  // of one slice
constexpr int MAX_LEN = MAX_GROUPS * GROUP - rows::MOST_SKEW;  // elements of one slice
constexpr int LIST = MAX_K + MAX_K / 4 + 64;      // groups that are read again
constexpr int BATCH = 2048;                       // elements or keys that one step may add to the buffer
constexpr int BUF = 2 * BATCH;
constexpr int BUCKETS = NT;                       // of a sort
constexpr int CROWD = 256;                        // keys of one bucket that are placed by counting
static_assert(BUF >= BATCH + MAX_K, "a compressed buffer takes a batch");
static_assert(BUF * sizeof(uint64_t) >= MAX_GROUPS * sizeof(float), "the buffer stands over the group maxima");

struct Params {
  const void* logits;
  int64_t stride;
  const int64_t* targets;
  int rows, V, K, slices, len;
  Scale sc;
  float* out_logprob;
  int64_t* out_rank;
  float* out_entropy;
  int64_t* out_top_ids;
  float* out_top_logprob;
  int32_t* out_status;
  double* out_stats;
  State* states;   // [rows, slices]
  uint64_t* keys;  // [rows, slices, K]
};

// A logit as an integer of the same order (-0 as +0), and back.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
constexpr uint32_t ABOVE_MASKED = 0x00800000u;  // order_of(-inf) + 1
// Element i of a row in (logit desc, index asc): larger keys come first.  0 is no element.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) { return (uint64_t)order_of(x) << 32 | (0xFFFFFFFFu - i); }

struct Shared {
  union {
    uint64_t buf[BUF];
    float group_max[MAX_GROUPS];
  };
  uint16_t list[LIST];
  int bucket[BUCKETS];
  double red[4 * WAVES];
  int counts[2][7 * WAVES];
  uint64_t least;
  State state;
  int64_t target;
  float xt, bound;
  int n, listed;
};

// Descending bitonic sort of buf[0, n), over the next power of two, padded with zeros.  Threads 64 w to
// 64 w + 63 take the pairs of 128 elements that no other wave touches while the pairs are at most 64
// apart: those steps need no barrier.
__device__ __forceinline__ void sort_bitonic(uint64_t* buf, int n) {
  const int tid = threadIdx.x;
  int P = 256;
  while (P < n) P <<= 1;
  for (int i = n + tid; i < P; i += NT) buf[i] = 0;
  int last = P;
  for (int k = 2; k <= P; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      if (j > 64 || last > 64) {
        __syncthreads();
      } else {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
      last = j;
      for (int q = tid; q < P / 2; q += NT) {
        const int i = 2 * q - (q & (j - 1));
        const uint64_t a = buf[i], b = buf[i + j];
        if ((a < b) == ((i & k) == 0)) {
          buf[i] = b;
          buf[i + j] = a;
        }
      }
    }
  __syncthreads();
}

// Descending order of s.buf[0, n), n <= BUF, of logits in [low, m].  Every thread calls it, behind a
// barrier.  Up to 128 keys are placed by counting the larger ones.  More are dealt into BUCKETS intervals of
// the logits, and placed by counting within their bucket: 710 keys of a row's tail in 4.6 us beside three
// other workgroups, 15 by the bitonic sort, which is left for logits that crowd into few buckets.
__device__ __forceinline__ void sort_desc(Shared& s, int n, float low, float m) {
  const int tid = threadIdx.x;
  uint64_t* buf = s.buf;
  if (n <= 128) {
    // four threads a key
    const int i = tid >> 2;
    const uint64_t key = i < n ? buf[i] : 0;
    int before = 0;
    for (int q = tid & 3; q < n; q += 4) before += buf[q] > key;
    before += __shfl_xor(before, 1);
    before += __shfl_xor(before, 2);
    __syncthreads();
    if (i < n && (tid & 3) == 0) buf[before] = key;
    __syncthreads();
    return;
  }
  static_assert(BUCKETS == NT, "a bucket for every thread");
  constexpr int EACH = BUF / NT;
  const float scale = BUCKETS / (m - low);
  const auto bucket_of = [&](uint64_t key) {  // 0 holds the largest; monotone, as each rounding is
    const float at = (m - logit_of((uint32_t)(key >> 32))) * scale;
    return at < (float)(BUCKETS - 1) ? (int)at : BUCKETS - 1;
  };
  s.bucket[tid] = 0;
  __syncthreads();
  uint64_t key[EACH];
  int slot[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    if (e * NT >= n) break;
    key[e] = e * NT + tid < n ? buf[e * NT + tid] : 0;
    slot[e] = key[e] ? atomicAdd(&s.bucket[bucket_of(key[e])], 1) : 0;
  }
  __syncthreads();
  const int size = s.bucket[tid];
  if (__syncthreads_or(size > CROWD || !(scale < INFINITY))) {
    sort_bitonic(buf, n);
    return;
  }
  const int up_to = (int)wave_incl_scan_u32((uint32_t)size);
  if ((tid & 63) == 63) s.counts[0][tid >> 6] = up_to;
  __syncthreads();
  int begin = up_to - size;
  for (int w = 0; w < tid >> 6; ++w) begin += s.counts[0][w];
  s.bucket[tid] = begin | size << 16;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    if (e * NT >= n) break;
    if (key[e]) buf[(s.bucket[bucket_of(key[e])] & 0xFFFF) + slot[e]] = key[e];
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    if (e * NT >= n) break;
    if (!key[e]) continue;
    const int b = s.bucket[bucket_of(key[e])], first = b & 0xFFFF, end = first + (b >> 16);
    int at = first;
#pragma unroll 4
    for (int q = first; q < end; ++q) at += buf[q] > key[e];
    slot[e] = at;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    if (e * NT >= n) break;
    if (key[e]) buf[slot[e]] = key[e];
  }
  __syncthreads();
}

// Room for another batch: past BUF - BATCH keys, the first K in order are kept, and what follows has
// to come before the last of them.  Every thread calls it behind a barrier.
__device__ __forceinline__ void make_room(Shared& s, int K, uint64_t& floor_key) {
  const int n = s.n;
  __syncthreads();
  if (n <= BUF - BATCH) return;
  sort_bitonic(s.buf, n);
  floor_key = s.buf[K - 1];
  __syncthreads();
  if (threadIdx.x == 0) s.n = K;
  __syncthreads();
}

__device__ __forceinline__ void push(Shared& s, uint64_t key) { s.buf[atomicAdd(&s.n, 1)] = key; }

template <int CTRL>
__device__ __forceinline__ int dpp_i(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, true);
}

// c[w] summed over the workgroup's waves.
template <int W>
__device__ __forceinline__ void join_counts(int (&c)[W], int* counts) {
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int w = 0; w < W; ++w) counts[w * WAVES + (threadIdx.x >> 6)] = c[w];
  __syncthreads();
  // lane 8 w + i takes wave i's count of at[w]
  static_assert(WAVES == 8 && W <= 8, "a lane for every count");
  const int lane = threadIdx.x & 63;
  int v = lane < W * WAVES ? counts[lane] : 0;
  v += dpp_i<0xB1>(v);   // quad_perm [1,0,3,2]
  v += dpp_i<0x4E>(v);   // quad_perm [2,3,0,1]
  v += dpp_i<0x141>(v);  // row_half_mirror
#pragma unroll
  for (int w = 0; w < W; ++w) c[w] = __builtin_amdgcn_readlane(v, 8 * w);
}

// Raises `lo`, an order that c >= K values reach, until at most `most` do, as far as ties let it; `hi`
// is an order that fewer than K reach.  W + 1 intervals at a time, three times of the logits between the
// two, then of their orders; count(at, got) gives how many reach each at[w].
template <int W, class Count>
__device__ __forceinline__ void search(uint32_t& lo, uint32_t& hi, int& c, int K, int most, Count count) {
  for (int turn = 0; c > most && hi - lo > 1u; ++turn) {
    uint32_t at[W];
    float value[W];
    int got[W];
    const float from = logit_of(lo), part = (logit_of(hi - 1u) - from) / (W + 1);
    const uint32_t step = (hi - lo) / (W + 1);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      at[w] = lo + (step ? step * (w + 1) : 1u);
      if (turn < 3 && part < INFINITY) at[w] = min(max(order_of(from + part * (w + 1)), lo + 1u), hi - 1u);
      value[w] = logit_of(at[w]);
    }
    count(value, got);
    uint32_t above = hi;
#pragma unroll
    for (int w = W - 1; w >= 0; --w) {
      if (at[w] >= above) continue;
      if (got[w] >= K) {
        lo = at[w];
        c = got[w];
        break;
      }
      above = at[w];
    }
    hi = above;
  }
}

// The selection begins within the pass: what the threads met bounds the row's K-th element.  The K-th
// largest of the shares' maxima is such a bound, and few more groups than K reach it where K is at most
// half of the shares: in rows of no special order, 68 groups the 64th of 512, 710 the 512th of 1024.
// Up to K = 256 one wave searches among the 512 threads' maxima by itself, without a barrier, while the
// others join their sums (both launches of one row's top 5: 11.3 us instead of 13.9; of 48 rows' top 20: 15.9 instead
// of 19.3; 4096 bf16 rows' top 64: 225 instead of 231); above, all search among 1024 or 2048 (search_shares).
constexpr int ALONE = NT / 2;
__device__ __forceinline__ void met_shares(Shared& s, const float (&own)[4], int K) {
  if (K <= ALONE) s.bucket[threadIdx.x] = __float_as_int(fmaxf(fmaxf(own[0], own[1]), fmaxf(own[2], own[3])));
}
__device__ __forceinline__ void search_alone(Shared& s, int K, float m) {
  if (threadIdx.x >= 64) return;
  constexpr int EACH = NT / 64, W = 3;
  float v[EACH], least = INFINITY;
  int c = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    v[e] = __int_as_float(s.bucket[e * 64 + threadIdx.x]);
    c += __popcll(__ballot(v[e] > -INFINITY));
    least = fminf(least, v[e] > -INFINITY ? v[e] : INFINITY);
  }
  uint32_t lo = ABOVE_MASKED;
  if (c >= K) {
    // (the smallest: a maximum with the signs turned)
    lo = max(order_of(-wave_max_dpp(-least)), ABOVE_MASKED);
    uint32_t hi = order_of(m) + 1u;
    search<W>(lo, hi, c, K, K + max(16, K / 4), [&](const float(&at)[W], int(&got)[W]) {
#pragma unroll
      for (int w = 0; w < W; ++w) {
        got[w] = 0;
#pragma unroll
        for (int e = 0; e < EACH; ++e) got[w] += __popcll(__ballot(v[e] >= at[w]));
      }
    });
  }
  if (threadIdx.x == 0) {
    s.bound = logit_of(lo);
    s.listed = s.n = 0;
  }
}
__device__ __forceinline__ void search_shares(Shared& s, const float (&own)[4], int K, float m) {
  constexpr int W = 7;
  const float a = fmaxf(own[0], own[1]), b = fmaxf(own[2], own[3]);
  int turn = 0;
  const auto count = [&](const float(&at)[W], int(&got)[W]) {
#pragma unroll
    for (int w = 0; w < W; ++w)
      got[w] = K <= NT ? __popcll(__ballot(a >= at[w])) + __popcll(__ballot(b >= at[w]))
                       : __popcll(__ballot(own[0] >= at[w])) + __popcll(__ballot(own[1] >= at[w])) +
                             __popcll(__ballot(own[2] >= at[w])) + __popcll(__ballot(own[3] >= at[w]));
    join_counts(got, s.counts[turn]);
    turn ^= 1;
  };
  float least = INFINITY;
#pragma unroll
  for (int u = 0; u < 4; ++u) least = fminf(least, own[u] > -INFINITY ? own[u] : INFINITY);
  const uint32_t first = max(order_of(-rows::block_max(-least, s.red)), ABOVE_MASKED);
  const float at[W] = {logit_of(first), INFINITY, INFINITY, INFINITY, INFINITY, INFINITY, INFINITY};
  int got[W];
  count(at, got);
  int c = got[0];
  uint32_t lo = ABOVE_MASKED, hi = order_of(m) + 1u;
  if (c >= K) {
    lo = first;
    search<W>(lo, hi, c, K, K + K / 4, count);
  }
  if (threadIdx.x == 0) {
    s.bound = logit_of(lo);
    s.listed = s.n = 0;
  }
  __syncthreads();
}

// Appends the groups whose maximum is at least `bound` to s.list, from s.listed = 0 on, as many as it
// holds, and returns their number.
__device__ __forceinline__ int list_groups(Shared& s, int n, float bound) {
  for (int j = threadIdx.x; j < n; j += NT)
    if (s.group_max[j] >= bound) {
      const int at = atomicAdd(&s.listed, 1);
      if (at < LIST) s.list[at] = (uint16_t)j;
    }
  __syncthreads();
  return s.listed;
}

// s.list = at least the first K groups in (maximum desc, index asc) of those that hold an unmasked
// element, or all of them; returns their number, and in `bound` a logit that the row's K-th element
// reaches, which comes as s.bound.
__device__ __forceinline__ int select_groups(Shared& s, int n, int K, float m, float& bound) {
  constexpr int W = 7;
  const int tid = threadIdx.x, most = K + max(16, K / 4);
  bound = s.bound;
  int c = list_groups(s, n, bound);
  if (c <= (bound > logit_of(ABOVE_MASKED) ? min(2 * most, LIST) : most)) return c;

  // too many: the bound is searched among the groups' maxima, and what is left at the end are ties
  uint32_t lo = order_of(bound), hi = order_of(m) + 1u;
  int turn = 0;
  search<W>(lo, hi, c, K, most, [&](const float(&at)[W], int(&got)[W]) {
#pragma unroll
    for (int w = 0; w < W; ++w) got[w] = 0;
    for (int j = 0; j < n; j += NT) {
      const float v = j + tid < n ? s.group_max[j + tid] : -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) got[w] += __popcll(__ballot(v >= at[w]));
    }
    join_counts(got, s.counts[turn]);
    turn ^= 1;
  });
  bound = logit_of(lo);
  // those above `lo` in any order, and at most as many at `lo` as are wanted, from the lowest index
  const bool all = c <= most;
  __syncthreads();
  if (tid == 0) s.listed = 0;
  __syncthreads();
  int taken = min(list_groups(s, n, all ? bound : logit_of(hi)), LIST);
  if (!all) {
    const int wave = tid >> 6, lane = tid & 63;
    for (int j = 0; j < n && taken < K; j += NT) {
      const bool tie = j + tid < n && s.group_max[j + tid] == bound;
      const uint64_t b = __ballot(tie);
      __syncthreads();
      if (lane == 0) s.counts[0][wave] = __popcll(b);
      __syncthreads();
      int before = taken, total = 0;
      for (int w = 0; w < WAVES; ++w) {
        if (w < wave) before += s.counts[0][w];
        total += s.counts[0][w];
      }
      before += __popcll(b & ((1ull << lane) - 1ull));
      if (tie && before < K) s.list[before] = (uint16_t)(j + tid);
      taken = min(K, taken + total);
    }
  }
  __syncthreads();
  return taken;
}

// s.buf = the first K elements of x[from, len) in order (or as many as are not masked); returns their
// number.  `first`: the index of x[0] in its row (below 0 where x[from] is the row's first).
template <typename T>
__device__ __forceinline__ int top_of(Shared& s, const T* x, int from, int len, int first, int K, float m) {
  constexpr int VEC = Elem<T>::VEC, LANES = GROUP / VEC, AT_ONCE = BATCH / GROUP;
  float bound;
  const int n_groups = (len + GROUP - 1) / GROUP;
  const int groups = select_groups(s, n_groups, K, m, bound);
  // calls f(w, at) for the 16 bytes w at chunk `at` of each listed group, or masked ones; every thread of a
  // wave as often as the others
  const int lane = (int)threadIdx.x % LANES;
  const auto each_chunk = [&](auto&& f) {
    constexpr int AHEAD = 4;  // loads in flight at once
    for (int b = 0; b < groups; b += AHEAD * (NT / LANES)) {
      uint32_t w[AHEAD][4];
      int at[AHEAD];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int g = b + a * (NT / LANES) + (int)threadIdx.x / LANES;
        at[a] = g < groups ? (int)s.list[g] * LANES + lane : -1;
        rows::load_some<false>(x, from, len, at[a], w[a]);
      }
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) f(w[a], at[a]);
    }
  };
  const auto element_key = [&](float v, int at, int j) { return key_of(v, (uint32_t)(first + at * VEC + j)); };
  const auto gather = [&](float least) {
    each_chunk([&](const uint32_t(&w)[4], int at) {
      float v[VEC];
      Elem<T>::unpack(w, v);
      // the wave's elements one after the other: one addition for all of them
      uint64_t pass[VEC];
      int total = 0;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        pass[j] = __ballot(v[j] >= least);
        total += __popcll(pass[j]);
      }
      if (total == 0) return;
      int to = 0;
      if ((threadIdx.x & 63) == 0) to = atomicAdd(&s.n, total);
      to = __builtin_amdgcn_readfirstlane(to);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int mine = to + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(pass[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)pass[j], 0));
        if (v[j] >= least && mine < BUF) s.buf[mine] = element_key(v[j], at, j);
        to += __popcll(pass[j]);
      }
    });
    __syncthreads();
    const int n = s.n;
    __syncthreads();
    return n;
  };
  int n = gather(bound);
  if (n > BUF) {
    // few groups for many alternatives: the bound is searched among their elements
    constexpr int W = 7;
    uint32_t lo = order_of(bound), hi = order_of(m) + 1u;
    int turn = 0;
    search<W>(lo, hi, n, K, BUF, [&](const float(&at)[W], int(&got)[W]) {
#pragma unroll
      for (int q = 0; q < W; ++q) got[q] = 0;
      each_chunk([&](const uint32_t(&w)[4], int) {
        float v[VEC];
        Elem<T>::unpack(w, v);
#pragma unroll
        for (int q = 0; q < W; ++q)
#pragma unroll
          for (int j = 0; j < VEC; ++j) got[q] += __popcll(__ballot(v[j] >= at[q]));
      });
      join_counts(got, s.counts[turn]);
      turn ^= 1;
    });
    bound = logit_of(lo);
    __syncthreads();
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
    n = gather(bound);
  }
  if (n > BUF) {
    // more ties at the bound than the buffer holds: a batch at a time
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
    uint64_t floor_key = 0;
    for (int b = 0; b < groups; b += AT_ONCE) {
      make_room(s, K, floor_key);
      const int g = b + (int)threadIdx.x / LANES;
      if ((int)threadIdx.x < AT_ONCE * LANES && g < groups) {
        const int at = (int)s.list[g] * LANES + lane;
        uint32_t w[4];
        float v[VEC];
        rows::load_some<false>(x, from, len, at, w);
        Elem<T>::unpack(w, v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const uint64_t key = element_key(v[j], at, j);
          if (v[j] >= bound && key > floor_key) push(s, key);
        }
      }
      __syncthreads();
    }
    n = s.n;
  }
  sort_desc(s, n, bound, m);
  return min(n, K);
}

// The row's outputs from its sums and its sorted list.
__device__ __forceinline__ void write_row(const Params& p, int row, const Shared& s, int n_top) {
  if ((int)(threadIdx.x & ~63u) > p.K) return;  // waves without an alternative to write
  const State st = s.state;
  const uint64_t* top = s.buf;
  const double S = st.S + p.sc.kappa * st.U;
  const bool bad = !(S > 0.0 && S < INFINITY);
  const double m = st.m, ln_s = log(S);
  const double entropy = bad ? (double)NAN : fmax(ln_s - st.U * (p.sc.inv_t / p.sc.cd) / S, 0.0);
  for (int i = threadIdx.x; i < p.K; i += NT) {
    const uint64_t key = i < n_top ? top[i] : 0;
    const int64_t at = (int64_t)row * p.K + i;
    const bool none = bad || key == 0;
    p.out_top_ids[at] = none ? -1 : (int64_t)(0xFFFFFFFFu - (uint32_t)key);
    p.out_top_logprob[at] =
        bad ? NAN : none ? -INFINITY : (float)(((double)logit_of((uint32_t)(key >> 32)) - m) * p.sc.inv_t - ln_s);
  }
  if (threadIdx.x) return;
  int status = bad ? DSV41_STATUS_NONFINITE : 0;
  if (p.targets) {
    const int64_t target = s.target;
    const float xt = s.xt;
    const bool outside = target < 0 || target >= p.V;
    if (outside) status |= DSV41_STATUS_BAD_TARGET;
    p.out_logprob[row] = bad || outside ? NAN : (float)(((double)xt - m) * p.sc.inv_t - ln_s);
    p.out_rank[row] = bad || outside ? 0 : 1 + (int64_t)st.before;
  }
  p.out_entropy[row] = (float)entropy;
  p.out_status[row] = status;
  if (p.out_stats) {
    double* o = p.out_stats + (int64_t)row * 4;
    o[0] = m;
    o[1] = bad ? (double)NAN : S;
    o[2] = ln_s;
    o[3] = entropy;
  }
}

template <typename T, bool ONCE, bool TOP>
__global__ __launch_bounds__(NT, 8) void scores_kernel(Params p) {
  __shared__ Shared s;
  const int row = blockIdx.x / p.slices, slice = blockIdx.x % p.slices;
  const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.stride;
  const int skew = rows::skew_of(x + slice * p.len), begin = slice * p.len - skew, len = min(p.len, p.V - slice * p.len) + skew;
  int64_t target = -1;
  float at_target = INFINITY;
  const auto before = [&](float& xt, int& t) {
    if (p.targets) {
      target = p.targets[row];
      if (target >= 0 && target < p.V) {
        xt = at_target = Elem<T>::one(x + target);
        t = (int)target - begin;
      }
    }
    return true;
  };
  float own[4];
  const auto met = [&](const float(&o)[4]) {
    if constexpr (TOP) {
      met_shares(s, o, p.K);
#pragma unroll
      for (int u = 0; u < 4; ++u) own[u] = o[u];
    }
  };
  const auto found = [&](float m) {
    if constexpr (TOP)
      if (p.K <= ALONE) search_alone(s, p.K, m);
  };
  const State st =
      rows::scan<T, ONCE, TOP, false>(x + begin, skew, len, p.sc, s.group_max, nullptr, s.red, before, met, found);
  if constexpr (TOP)
    if (p.K > ALONE) search_shares(s, own, p.K, st.m);
  if (threadIdx.x == 0) {  // (registers that would be kept over the selection)
    s.state = st;
    s.target = target;
    s.xt = at_target;
  }
  int n = 0;
  if constexpr (TOP)
    n = top_of(s, x + begin, skew, len, begin, p.K, st.m);
  else
    __syncthreads();
  if (p.slices == 1) {
    write_row(p, row, s, n);
    return;
  }
  const int64_t at = (int64_t)row * p.slices + slice;
  if (threadIdx.x == 0) p.states[at] = s.state;
  for (int i = threadIdx.x; i < p.K; i += NT) p.keys[at * p.K + i] = i < n ? s.buf[i] : 0;
}

// Joins the slices of a row, at most 64.
template <typename T>
__global__ __launch_bounds__(NT) void scores_join_kernel(Params p) {
  __shared__ Shared s;
  const int row = blockIdx.x, tid = threadIdx.x;
  // the lists' first keys before their second ones and so on, so that what is left below the bound need
  // not be read
  const uint64_t* keys = p.keys + (int64_t)row * p.slices * p.K;
  const int total = p.slices * p.K;
  const auto key_at = [&](int i) { return i < total ? keys[(int64_t)(i % p.slices) * p.K + i / p.slices] : 0; };
  constexpr int EACH = BATCH / NT;
  uint64_t key[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) key[e] = key_at(e * NT + tid);
  int64_t target = -1;
  float xt = INFINITY;
  if (p.targets) {
    target = p.targets[row];
    if (target >= 0 && target < p.V) xt = Elem<T>::one(static_cast<const T*>(p.logits) + (int64_t)row * p.stride + target);
  }
  if (tid < 64) {
    State st{0.0, 0.0, -INFINITY, 0};
    // Two bounds of the row's K-th key.  Each list holds K keys that come no later than its last; and
    // all hold ceil(K / slices) that come no later than the last of these.
    uint64_t last = 1, share = ~0ull;
    if (tid < p.slices) {
      st = p.states[(int64_t)row * p.slices + tid];
      if (p.K) {
        last = max(last, keys[(int64_t)tid * p.K + p.K - 1]);
        share = keys[(int64_t)tid * p.K + (p.K + p.slices - 1) / p.slices - 1];
      }
    }
    const float m = wave_max_dpp(st.m);
    if (st.S == 0.0)
      st.U = 0.0;
    else
      rows::rebase(st.S, st.U, ((double)st.m - (double)m) * p.sc.cd);
    const double S = wave_total_d(st.S), U = wave_total_d(st.U);
    const int before = wave_sum_i(st.before);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      last = max(last, (uint64_t)__shfl_xor((unsigned long long)last, o));
      share = min(share, (uint64_t)__shfl_xor((unsigned long long)share, o));
    }
    if (tid == 0) {
      s.state = State{S, U, m, before};
      s.target = target;
      s.xt = xt;
      s.least = max(last, share);
      s.n = 0;
    }
  }
  __syncthreads();
  int n = 0;
  if (p.K) {
    const uint64_t least = s.least;
    uint64_t floor_key = 0;
    for (int b = 0; b < total; b += BATCH) {
      if (b) {
        make_room(s, p.K, floor_key);
#pragma unroll
        for (int e = 0; e < EACH; ++e) key[e] = key_at(b + e * NT + tid);
      }
      bool any = false;
#pragma unroll
      for (int e = 0; e < EACH; ++e)
        if (key[e] >= least && key[e] > floor_key) {
          push(s, key[e]);
          any = true;
        }
      if (!__syncthreads_or(any)) break;
    }
    n = s.n;
    sort_desc(s, n, logit_of((uint32_t)(least >> 32)), s.state.m);
    n = min(n, p.K);
  }
  write_row(p, row, s, n);
}

// ------------------------------------------------------------------------------------ gradient
struct GradParams {
  const void* logits;
  int64_t stride;
  const int64_t* targets;
  const int64_t* top_ids;
  int rows, V, K, slices, len;
  Scale sc;
  const double* stats;
  const float* g_logprob;
  const float* g_entropy;
  const float* g_top;
  void* out;  // [rows, V], rows V apart
};

// dx_i = (1 / T) (-(G + g_H (log p_i + H)) p_i + g_lp [i = t] + sum_k g_k [i = id_k]),  G = g_lp + sum_k g_k,
// as e_i (A + B d_i) with e_i = 2^d_i and d_i = (x_i - m) c: one read and one write of the row.  The
// tokens that have a gradient of their own are written again by the waves that wrote them.  Bound by memory:
// 1000 bf16 rows of 151851 in 95-107 us, 5.7-6.4 TB/s of read and write.  The last rows come first: the
// forward read them last, and the caches may still hold them.
template <typename T>
__global__ __launch_bounds__(NT, 8) void scores_grad_kernel(GradParams p) {
  __shared__ double red[3 * WAVES];
  const int row = p.rows - 1 - (int)(blockIdx.x / p.slices), slice = blockIdx.x % p.slices;
  const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.stride;
  const int begin = slice * p.len, len = min(p.len, p.V - begin);
  T* out = static_cast<T*>(p.out) + (int64_t)row * p.V + begin;
  const int tid = threadIdx.x;
  const int64_t t = p.targets && p.g_logprob ? p.targets[row] : -1;
  const double g_lp = p.targets && p.g_logprob ? p.g_logprob[row] : 0.0, g_h = p.g_entropy ? p.g_entropy[row] : 0.0;
  const int64_t* ids = p.g_top ? p.top_ids + (int64_t)row * p.K : nullptr;
  const float* g_top = p.g_top ? p.g_top + (int64_t)row * p.K : nullptr;
  double G = 0.0;
  int any = g_lp != 0.0 || g_h != 0.0;
  if (p.g_top) {
    for (int k = tid; k < p.K; k += NT)
      if (ids[k] >= 0) {
        G += g_top[k];
        any |= g_top[k] != 0.f;
      }
    double sum[1] = {G};
    rows::block_sums(sum, red);
    G = sum[0];
    any = __syncthreads_or(any);
  }
  G += g_lp != 0.0 && (t < 0 || t >= p.V) ? (double)NAN : g_lp;
  if (!any) {
    rows::fill_zero(out, len);
    return;
  }
  const double* st = p.stats + (int64_t)row * 4;
  const float m = (float)st[0];
  const double S = st[1];
  const double a = -(G + g_h * (st[3] - st[2])) * p.sc.inv_t / S, b = -g_h * p.sc.inv_t * p.sc.inv_t / (p.sc.c * S);
  const rows::Lift lift(fabs(a) + fabs(b));
  const float A = (float)(a * lift.down), B = (float)(b * lift.down), c = p.sc.c;
  auto dense = [&](float v) {
    const float d = v - m;
    return lift.exp2(d, c) * __builtin_fmaf(B, fmaxf(d * c, -1000.f), A);
  };
  // the tokens with a gradient of their own, in fp64, since 1 - p_t is what is left of a likely target's
  const auto value = [&](int64_t id, double g) {
    const double d = ((double)Elem<T>::one(x + id) - st[0]) * p.sc.inv_t;
    // (b goes with exponents of 2; a masked token has a power of 0, and a row without sums NaN)
    const double e = d > -INFINITY ? exp(d) * (a + b * d * (p.sc.c / p.sc.inv_t)) : 0.0 * S;
    return (float)(e + g * p.sc.inv_t);
  };
  const auto place = [&](int64_t id) { return id >= begin && id < begin + len ? (int)(id - begin) : -1; };
  if (!p.g_top) {
    rows::map(x + begin, out, len, dense);
    rows::own_stores_in_order();
    const int i = place(t);
    if (i >= 0 && rows::wrote(x + begin, i, len) && (tid & 63) == 0) rows::store_one(out + i, value(t, g_lp));
    return;
  }
  // the alternatives, and the target where it is none of them
  __shared__ rows::Again again;
  int listed = 0;
  const auto entry = [&](int k) {
    const int64_t id = k < p.K ? ids[k] : -1;
    listed |= id >= 0 && id == t;
    const int i = place(id);
    if (i >= 0) again.v[tid] = value(id, (double)g_top[k] + (id == t ? g_lp : 0.0));
    again.at[tid] = i;
  };
  entry(tid);
  rows::map(x + begin, out, len, dense);
  rows::own_stores_in_order();
  rows::lds_barrier();
  rows::store_again(again, min(p.K, NT), x + begin, out, len);
  for (int k = NT; k < p.K; k += NT) {
    rows::lds_barrier();
    entry(k + tid);
    rows::lds_barrier();
    rows::store_again(again, min(p.K - k, NT), x + begin, out, len);
  }
  listed = __syncthreads_or(listed);
  const int i = place(t);
  if (!listed && i >= 0 && rows::wrote(x + begin, i, len) && (tid & 63) == 0) rows::store_one(out + i, value(t, g_lp));
}

// ---------------------------------------------------------------------------------------- host
// More than 256 alternatives take slices whose threads meet four chunks each, whose maxima bound them.
Cut cut_of(int rows, int V, int K, int esize) {
  return rows::cut_rows(rows, V, K, esize, K > ALONE ? 4 * NT * (16 / esize) : 6144, MAX_LEN);
}

size_t workspace_of(int rows, int K, const Cut& c) {
  return c.slices == 1 ? 0 : (size_t)rows * c.slices * (sizeof(State) + (size_t)K * sizeof(uint64_t));
}

template <typename T, bool ONCE>
void launch(const Params& p, hipStream_t s) {
  const dim3 grid((unsigned)p.rows * (unsigned)p.slices);
  if (p.K)
    hipLaunchKernelGGL((scores_kernel<T, ONCE, true>), grid, dim3(NT), 0, s, p);
  else
    hipLaunchKernelGGL((scores_kernel<T, ONCE, false>), grid, dim3(NT), 0, s, p);
  if (p.slices > 1) hipLaunchKernelGGL(scores_join_kernel<T>, dim3(p.rows), dim3(NT), 0, s, p);
}
template <typename T>
void launch(const Params& p, hipStream_t s) {
  if (rows::read_once(p.rows, p.V, sizeof(T)))
    launch<T, true>(p, s);
  else
    launch<T, false>(p, s);
}

int check_desc(const dsv41_scores_desc* d) {
  if (!d) return fail(DSV41_E_INVALID, "scores descriptor is NULL");
  if (d->struct_size != sizeof(dsv41_scores_desc))
    return fail(DSV41_E_ABI, "dsv41_scores_desc size mismatch (rebuild the binding)");
  if (int rc = rows::check_rows(d->rows, d->vocab, d->logits_dtype, d->logits_row_stride, d->logits, d->temperature)) return rc;
  if (d->top_k < 0 || d->top_k > d->vocab) return fail(DSV41_E_INVALID, "top_k must lie in [0, vocabulary_size]");
  if (d->top_k > MAX_K) return fail(DSV41_E_UNSUPPORTED, "top_k above 1024 is not supported");
  if (!d->out_entropy || !d->out_status) return fail(DSV41_E_INVALID, "out_entropy and out_status are required");
  if (d->targets && (!d->out_logprob || !d->out_rank))
    return fail(DSV41_E_INVALID, "targets need out_logprob and out_rank");
  if (d->top_k && (!d->out_top_ids || !d->out_top_logprob))
    return fail(DSV41_E_INVALID, "top_k needs out_top_ids and out_top_logprob");
  return rows::check_grid(d->rows, cut_of(d->rows, d->vocab, d->top_k, d->logits_dtype == DSV41_DTYPE_F32 ? 4 : 2));
}

}  // namespace scores
}  // namespace dsv41

using namespace dsv41;

extern "C" size_t dsv41_scores_workspace_bytes(const dsv41_scores_desc* d) {
  if (scores::check_desc(d)) return 0;
  return scores::workspace_of(d->rows, d->top_k, scores::cut_of(d->rows, d->vocab, d->top_k, d->logits_dtype == DSV41_DTYPE_F32 ? 4 : 2));
}

extern "C" int dsv41_scores_run(const dsv41_scores_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = scores::check_desc(d)) return rc;
  const rows::Cut c = scores::cut_of(d->rows, d->vocab, d->top_k, d->logits_dtype == DSV41_DTYPE_F32 ? 4 : 2);
  const size_t need = scores::workspace_of(d->rows, d->top_k, c);
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 8))
    return fail(DSV41_E_WORKSPACE, "scores workspace is missing, too small or not 8-byte aligned");
  scores::Params p{};
  p.logits = d->logits;
  p.stride = d->logits_row_stride;
  p.targets = d->targets;
  p.rows = d->rows;
  p.V = d->vocab;
  p.K = d->top_k;
  p.slices = c.slices;
  p.len = c.len;
  p.sc = rows::scale_of(d->temperature, false);
  p.out_logprob = d->out_logprob;
  p.out_rank = d->out_rank;
  p.out_entropy = d->out_entropy;
  p.out_top_ids = d->out_top_ids;
  p.out_top_logprob = d->out_top_logprob;
  p.out_status = d->out_status;
  p.out_stats = d->out_stats;
  p.states = static_cast<rows::State*>(workspace);
  p.keys = reinterpret_cast<uint64_t*>(p.states + (c.slices > 1 ? (int64_t)d->rows * c.slices : 0));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (d->logits_dtype == DSV41_DTYPE_F32)
    scores::launch<float>(p, s);
  else
    scores::launch<rows::bf16_t>(p, s);
  DSV41_HIP_CHECK(hipGetLastError());
  return DSV41_OK;
}

extern "C" int dsv41_scores_grad_run(const dsv41_scores_grad_desc* d, void* stream) {
  if (!d) return fail(DSV41_E_INVALID, "scores gradient descriptor is NULL");
  if (d->struct_size != sizeof(dsv41_scores_grad_desc))
    return fail(DSV41_E_ABI, "dsv41_scores_grad_desc size mismatch (rebuild the binding)");
  if (int rc = rows::check_rows(d->rows, d->vocab, d->logits_dtype, d->logits_row_stride, d->logits, d->temperature))
    return rc;
  if (!d->stats || !d->out) return fail(DSV41_E_INVALID, "stats and out are required");
  if ((uintptr_t)d->out % (d->logits_dtype == DSV41_DTYPE_F32 ? 4 : 2))
    return fail(DSV41_E_INVALID, "out is not aligned to its type");
  if (d->grad_logprob && !d->targets) return fail(DSV41_E_INVALID, "grad_logprob needs targets");
  if (d->grad_top && (!d->top_ids || d->top_k <= 0)) return fail(DSV41_E_INVALID, "grad_top needs top_ids and top_k");
  const rows::Cut c = rows::grad_cut(d->rows, d->vocab, d->logits_dtype == DSV41_DTYPE_F32 ? 4 : 2);
  if (int rc = rows::check_grid(d->rows, c)) return rc;
  scores::GradParams p{};
  p.logits = d->logits;
  p.stride = d->logits_row_stride;
  p.targets = d->targets;
  p.top_ids = d->top_ids;
  p.rows = d->rows;
  p.V = d->vocab;
  p.K = d->grad_top ? d->top_k : 0;
  p.slices = c.slices;
  p.len = c.len;
  p.sc = rows::scale_of(d->temperature, false);
  p.stats = d->stats;
  p.g_logprob = d->grad_logprob;
  p.g_entropy = d->grad_entropy;
  p.g_top = d->grad_top;
  p.out = d->out;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)p.rows * (unsigned)p.slices);
  if (d->logits_dtype == DSV41_DTYPE_F32)
    hipLaunchKernelGGL(scores::scores_grad_kernel<float>, grid, dim3(rows::NT), 0, s, p);
  else
    hipLaunchKernelGGL(scores::scores_grad_kernel<rows::bf16_t>, grid, dim3(rows::NT), 0, s, p);
  DSV41_HIP_CHECK(hipGetLastError());
  return DSV41_OK;
}
