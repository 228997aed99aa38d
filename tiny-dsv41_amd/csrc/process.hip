// process.hip — biases, penalties for repeated tokens and token masks on rows of logits, and their
// gradient.
//
// Row r, token i, fp32, every step rounded as the sampler rounds its own penalties:
//   v = x + b_i                                     (a bias list of the row names i)
//   v = v > 0 ? v / rp : v * rp                     (i is in the row's history)
//   v = v - freq c                                  (c: how often, past the prompt)
//   v = v - pres                                    (c > 0)
//   v = fill                                        (the row's mask leaves i out)
// and, for a gradient g of the outputs: 0 where the mask leaves i out, g / rp or g rp in the history by the
// sign of x + b_i, g elsewhere.
//
// One pass: a workgroup takes a slice of 8192 ids of a row.  What the lists say of the slice's ids goes into
// one LDS word each, by integer atomics, so in any order to the same words.  The slice's elements are on their way
// meanwhile, and most words are 0 then: such groups of 16 bytes go out as they came.  Every slice reads all of its
// row's lists, which therefore stay on one XCD (whose L2 serves all but the first).  A mask's words come before the
// elements: groups without an allowed one are not read.
// In place, nothing is read but groups that a list names or that are masked in part, and written but those and what is masked.
// The gradient needs two bits an id: whether the history has it, and the sign of x + b, from single logits that are
// read for the history's ids while the gradient's own are on their way.
//
// Slices begin at memory lines of the result, so rows of an odd vocabulary are written by whole lines: 500 bf16 rows of
// 151851 copied in 51 us (5.9 TB/s of read and write), as many of 151936 in 50.  2048 fp32 rows of 151936: 432 us (5.8
// TB/s), with masks 441, with histories of 2048 and 4096 440 and 464 (452 where they are ragged, three quarters of that); bf16 213,
// 218, 239 and 265.  256 to 1024 threads and slices of 8192 to 16384 ids, timed before the loads of a slice went together:
// 512 and 8192 the best or within 3% (2048 fp32 rows with ragged histories 477; 1024 and 16384: 506, 256 and 8192: 778).
// The gradient: 500 fp32 rows of 151851 111 us, with masks 114, with histories of 2048 146, with both 150; bf16 56, 63, 90
// and 91; 1000 fp32 rows of 151936 214 us (5.7 TB/s), with masks 219, with histories of 4096 334.
// What bounds it: memory, and beside long histories the instructions of reading the lists, once a slice (2048 ids cost
// 500 bf16 rows 16 to 18 us), in the gradient the single logits, too.

#include <math.h>

#include "row_scan.h"

namespace dsv41 {
namespace process {

using rows::bf16_t;
using rows::Elem;

constexpr int NT = 512;
// ids of a slice: 32 KB of words, four workgroups a CU
constexpr int SLICE = 8192, SHORT_SLICE = 16384;
constexpr int MAX_HISTORY = (1 << 19) - 1, MAX_BIAS = (1 << 12) - 1;  // entries of a row's lists
constexpr int SHORT_HISTORY = (1 << 14) - 1, SHORT_BIAS = 64;         // those that words of 16 bits take
constexpr int AHEAD = 8;                                              // history entries of a thread in flight

struct Params {
  const void* x;
  int64_t xs;
  void* out;
  int64_t os;
  const void* grad;
  int64_t gs;
  int rows, V, slices;
  const int64_t* history;
  int64_t hs;
  int hist_len;
  const int32_t* lens;
  const int32_t* prompt_lens;
  float rp, pres, freq;
  const float *rps, *press, *freqs;
  const int64_t* bias_ids;
  const float* bias;
  int64_t bs;
  int n_bias;
  const uint32_t* mask;
  int64_t ms;
  int masks;
  const int32_t* mask_rows;
  float fill;
  int32_t* status;
  bool knobs_of_rows() const { return rps || press || freqs; }
};

// What the lists say of an element: how often it was said, whether it is in the history at all, and its entry of the
// bias list (-1: none).
struct Said {
  uint32_t count;
  bool listed;
  int entry;
};

// What the row's knobs make of it.
struct Knobs {
  float rp, pres, freq;
  __device__ __forceinline__ float apply(float x, Said s, const float* bias) const {
    if (s.entry >= 0) x = x + bias[s.entry];
    if (s.listed) {
      x = x > 0.0f ? x / rp : x * rp;
      const float f = freq * (float)s.count;
      x = x - f;
      if (s.count > 0) x = x - pres;
    }
    return x;
  }
};

// The words of a slice.  Of 32 bits: count (19), in the history (1), bias entry + 1 (12).
template <typename T, bool SHORT>
struct Words {
  static constexpr int IDS = SLICE, G = Elem<T>::VEC;
  uint32_t* w;
  // a thread's group of 8 bf16 elements lies in two planes, so that either half of it is read without bank conflicts
  static __device__ __forceinline__ int place(int at) {
    return G == 4 ? at : ((at >> 2 & 1) * (IDS / 2)) + (at >> 3 << 2) + (at & 3);
  }
  __device__ __forceinline__ void say(int at) const { atomicAdd(&w[place(at)], 1u); }
  __device__ __forceinline__ void list(int at) const { atomicOr(&w[place(at)], 1u << 19); }
  __device__ __forceinline__ void bias(int at, int entry) const { atomicMax(&w[place(at)], (uint32_t)(entry + 1) << 20); }
  // the elements at .. at + G - 1 that anything is said of
  __device__ __forceinline__ uint32_t marked(int at) const {
    uint32_t m = 0;
#pragma unroll
    for (int q = 0; q < G; q += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(w + place(at + q));
      m |= (min(v.x, 1u) | min(v.y, 1u) << 1 | min(v.z, 1u) << 2 | min(v.w, 1u) << 3) << q;
    }
    return m;
  }
  __device__ __forceinline__ Said read(int at, const int*, int) const {
    const uint32_t v = w[place(at)];
    return {v & MAX_HISTORY, (v & 0xFFFFF) != 0, (int)(v >> 20) - 1};
  }
};
// Of 16 bits: count (14), in the history (1), biased (1), for slices twice as long, whose lists are read half as often;
// a biased element looks for its entry among the list's places.
template <typename T>
struct Words<T, true> {
  static constexpr int IDS = SHORT_SLICE, G = Elem<T>::VEC;
  uint32_t* w;
  __device__ __forceinline__ void say(int at) const { atomicAdd(&w[at >> 1], 1u << (16 * (at & 1))); }
  __device__ __forceinline__ void list(int at) const { atomicOr(&w[at >> 1], 0x4000u << (16 * (at & 1))); }
  __device__ __forceinline__ void bias(int at, int) const { atomicOr(&w[at >> 1], 0x8000u << (16 * (at & 1))); }
  __device__ __forceinline__ uint32_t marked(int at) const {
    static_assert(G == 8, "a group's words are 16 bytes");
    const uint4 v = *reinterpret_cast<const uint4*>(w + (at >> 1));
    const uint32_t d[4] = {v.x, v.y, v.z, v.w};
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m |= (min(d[i] & 0xFFFFu, 1u) | min(d[i] >> 16, 1u) << 1) << (2 * i);
    return m;
  }
  __device__ __forceinline__ Said read(int at, const int* places, int n) const {
    const uint32_t v = w[at >> 1] >> (16 * (at & 1)) & 0xFFFFu;
    int entry = -1;
    if (v & 0x8000u)
      for (entry = n - 1; entry > 0 && places[entry] != at; --entry) {}
    return {v & SHORT_HISTORY, (v & 0x7FFFu) != 0, entry};
  }
};

// A group of 16 bytes, kept as they are in memory: most groups go out as they came.
struct Group {
  uint32_t w[4];
};
template <typename T>
constexpr uint32_t ALL = (1u << Elem<T>::VEC) - 1;
// Element j, which differs from lane to lane (selections: registers have no addresses).
__device__ __forceinline__ uint32_t pick(const Group& g, int i) {
  const uint32_t lo = i & 1 ? g.w[1] : g.w[0], hi = i & 1 ? g.w[3] : g.w[2];
  return i & 2 ? hi : lo;
}
__device__ __forceinline__ void place(Group& g, int i, uint32_t w) {
#pragma unroll
  for (int k = 0; k < 4; ++k) g.w[k] = i == k ? w : g.w[k];
}
// The elements j with bit j of `there`, from p (the others come as 0), and to it.  (Straight code: around a loop the
// compiler waits for all loads in flight.)
template <typename T>
__device__ __forceinline__ void load_group(const T* p, uint32_t there, Group& g) {
  if (there == ALL<T>) {
    rows::load16<false>(p, g.w);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) g.w[i] = 0;
#pragma unroll
    for (int j = 0; j < Elem<T>::VEC; ++j)
      if (there >> j & 1) Elem<T>::put(g.w, j, p[j]);
  }
}
__device__ __forceinline__ void store_element(float* p, const Group& g, int j) { *p = __uint_as_float(g.w[j]); }
__device__ __forceinline__ void store_element(bf16_t* p, const Group& g, int j) {
  p->v = (uint16_t)(g.w[j >> 1] >> (16 * (j & 1)));
}
template <typename T>
__device__ __forceinline__ void store_group(T* p, uint32_t there, const Group& g) {
  if (there == ALL<T>) {
    typename Elem<T>::Raw r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = g.w[i];
    *reinterpret_cast<typename Elem<T>::Raw*>(p) = r;
  } else {
#pragma unroll
    for (int j = 0; j < Elem<T>::VEC; ++j)
      if (there >> j & 1) store_element(p + j, g, j);
  }
}
__device__ __forceinline__ float get(const Group& g, int j, float) { return __uint_as_float(pick(g, j)); }
__device__ __forceinline__ float get(const Group& g, int j, bf16_t) {
  const uint32_t w = pick(g, j >> 1);
  return j & 1 ? bf16_hi(w) : bf16_lo(w);
}
__device__ __forceinline__ void set(Group& g, int j, float v, float) { place(g, j, __float_as_uint(v)); }
__device__ __forceinline__ void set(Group& g, int j, float v, bf16_t) {
  const uint32_t w = pick(g, j >> 1), b = pack_bf16(v, v);
  place(g, j >> 1, j & 1 ? (w & 0xFFFFu) | (b & 0xFFFF0000u) : (w & 0xFFFF0000u) | (b & 0xFFFFu));
}
// `instead` (of every element, in the type) where bit j of `allowed` is 0
__device__ __forceinline__ void drop(Group& g, uint32_t allowed, uint32_t instead, float) {
#pragma unroll
  for (int k = 0; k < 4; ++k) g.w[k] = allowed >> k & 1 ? g.w[k] : instead;
}
__device__ __forceinline__ void drop(Group& g, uint32_t allowed, uint32_t instead, bf16_t) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t lo = (uint32_t)((int)(allowed << (31 - 2 * k)) >> 31), hi = (uint32_t)((int)(allowed << (30 - 2 * k)) >> 31);
    const uint32_t keep = (lo & 0xFFFFu) | (hi & 0xFFFF0000u);
    g.w[k] = (g.w[k] & keep) | (instead & ~keep);
  }
}
// A workgroup's slice: ids [begin, begin + IDS) of a row, those of them that exist from `first` on, `count` of them.
struct Slice {
  int row, number, begin;
  uint32_t first, count;
  // the slice's place of an id (any 64 bits), where that is below `count` when `first` is taken off
  __device__ __forceinline__ bool place_of(uint2 id, uint32_t& at) const {
    at = id.x - (uint32_t)begin;
    return id.y == 0 && at - first < count;
  }
};
// false: none.  A row's slices go one after another to one XCD (workgroups go round-robin over the eight), and begin at
// memory lines of the result.
template <typename T, int IDS>
__device__ __forceinline__ bool slice_of(const Params& p, Slice& s) {
  const uint32_t item = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  s.row = (int)(item / (uint32_t)p.slices), s.number = (int)(item % (uint32_t)p.slices);
  if (s.row >= p.rows) return false;
  s.begin = s.number * IDS - rows::skew_of(static_cast<const T*>(p.out) + s.row * p.os);
  if (s.begin >= p.V) return false;
  s.first = (uint32_t)max(-s.begin, 0), s.count = (uint32_t)min(IDS, p.V - s.begin) - s.first;
  return true;
}

// The row's own values.
struct Row {
  Knobs knobs{1.f, 0.f, 0.f};
  bool bad = false;  // the row holds NaN
  int bits = 0;      // the status bit that says why
  const uint32_t* mask = nullptr;
  const uint2* h = nullptr;  // the history, where the knobs ask for it
  int len = 0, prompt = 0;
};
template <bool LISTS, bool MASK, bool GRADIENT>
__device__ __forceinline__ Row row_of(const Params& p, int row) {
  // all on their way at once: arrays that are not given are read at the arguments' begin
  typedef const __attribute__((address_space(4))) int32_t* constant_t;
  const uintptr_t nowhere = (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
  auto value_of = [&](const void* a) { return *(constant_t)(a ? (uintptr_t)a + 4 * (int64_t)row : nowhere); };
  const int m_row = MASK ? value_of(p.mask_rows) : 0;
  const int rp_row = LISTS ? value_of(p.rps) : 0, pres_row = LISTS ? value_of(p.press) : 0, freq_row = LISTS ? value_of(p.freqs) : 0;
  const int len_row = LISTS ? value_of(p.lens) : 0, prompt_row = LISTS ? value_of(p.prompt_lens) : 0;
  Row r;
  if constexpr (MASK) {
    const int m = p.mask_rows ? m_row : p.masks == 1 ? 0 : row;
    r.bad = m >= p.masks;
    if (r.bad) r.bits |= DSV41_STATUS_BAD_MASK;
    r.mask = m >= 0 && !r.bad ? p.mask + m * p.ms : nullptr;
  }
  if constexpr (LISTS) {
    Knobs& k = r.knobs;
    k.rp = p.rps ? __int_as_float(rp_row) : p.rp;
    k.pres = p.press ? __int_as_float(pres_row) : p.pres;
    k.freq = p.freqs ? __int_as_float(freq_row) : p.freq;
    if (!(isfinite(k.rp) && k.rp > 0.f) || !isfinite(k.pres) || !isfinite(k.freq)) {
      r.bad = true;
      r.bits |= DSV41_STATUS_BAD_PENALTY;
    }
    // (a gradient asks for the repetition penalty alone)
    if (p.history && !(k.rp == 1.f && (GRADIENT || (k.pres == 0.f && k.freq == 0.f)))) {
      r.h = reinterpret_cast<const uint2*>(p.history + row * p.hs);
      r.len = p.lens ? min(max(len_row, 0), p.hist_len) : p.hist_len;
      r.prompt = p.prompt_lens ? prompt_row : 0;
    }
  }
  return r;
}

// Which elements of a group at id i there are, and which of them the row's mask allows.
template <typename T, bool MASK>
__device__ __forceinline__ void group_at(const Params& p, const Row& r, int i, uint32_t& there, uint32_t& allowed) {
  constexpr int G = Elem<T>::VEC;
  const int lo = max(-i, 0), hi = min(p.V - i, G);  // elements [lo, hi)
  there = lo < hi ? (ALL<T> << lo) & (ALL<T> >> (G - hi)) : 0u;
  allowed = r.bad ? 0u : there;
  if (MASK && r.mask && there) {
    const int k = max(i, 0) >> 5, last = (p.V - 1) >> 5;
    const uint64_t both = (uint64_t)r.mask[min(k + 1, last)] << 32 | r.mask[k];
    allowed &= i >= 0 ? (uint32_t)(both >> (i & 31)) : (uint32_t)(both << -i);
  }
}
// The same for a thread's groups from id i on.  `inside`: all of the slice's ids exist.  Its loads go together then, here and in
// load_groups: a condition that differs from lane to lane has the wave wait for the loads under it.
template <typename T, bool MASK, int U>
__device__ __forceinline__ void groups_at(const Params& p, const Row& r, int i, bool inside, uint32_t (&there)[U], uint32_t (&allowed)[U]) {
  constexpr int STEP = NT * Elem<T>::VEC;
  if (!inside) {
#pragma unroll
    for (int u = 0; u < U; ++u) group_at<T, MASK>(p, r, i + u * STEP, there[u], allowed[u]);
    return;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) there[u] = ALL<T>, allowed[u] = r.bad ? 0u : ALL<T>;
  if (MASK && r.mask) {
    uint32_t lo[U], hi[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (i + u * STEP) >> 5;
      lo[u] = r.mask[k], hi[u] = r.mask[min(k + 1, (p.V - 1) >> 5)];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) allowed[u] &= (uint32_t)(((uint64_t)hi[u] << 32 | lo[u]) >> ((i + u * STEP) & 31));
  }
}
// A thread's groups that are wanted, from x at the slice's begin (others hold anything).
template <typename T, int U>
__device__ __forceinline__ void load_groups(const T* x, bool inside, const uint32_t (&there)[U], const uint32_t (&want)[U], Group (&v)[U]) {
  constexpr int G = Elem<T>::VEC;
  if (inside) {
#pragma unroll
    for (int u = 0; u < U; ++u) rows::load16<false>(x + (want[u] ? (u * NT + (int)threadIdx.x) * G : 0), v[u].w);
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (want[u]) load_group(x + (u * NT + (int)threadIdx.x) * G, there[u], v[u]);
  }
}

// `batch(first, ids)` for every AHEAD entries of a thread; the first ones were loaded ahead of the slice itself, as loads come back
// in order.
// (EACH: loads that wait for one another.  In the gradient and with short words they are better so, 500 bf16 rows by 2 us
// each; 2048 fp32 rows with ragged histories take 459 us that way and 452 with all of them together.)
template <bool EACH>
__device__ __forceinline__ void load_ahead(const Row& r, int j0, uint2 (&ids)[AHEAD]) {
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int j = j0 + k * NT + (int)threadIdx.x;
    if (EACH ? j < r.len : j0 + k * NT < r.len) ids[k] = r.h[min(j, r.len - 1)];
  }
}
template <bool EACH, class F>
__device__ __forceinline__ void for_history(const Row& r, uint2 (&ahead)[AHEAD], F batch) {
  batch((int)threadIdx.x, ahead);
  for (int j0 = AHEAD * NT; j0 < r.len; j0 += AHEAD * NT) {
    load_ahead<EACH>(r, j0, ahead);
    batch(j0 + (int)threadIdx.x, ahead);
  }
}
__device__ __forceinline__ bool past(uint2 id, int V) { return (int)id.y >= 0 && (id.y > 0 || id.x >= (uint32_t)V); }

template <typename T, bool LISTS, bool MASK, bool INPLACE, bool SHORT>
__global__ __launch_bounds__(NT, 8) void process_kernel(Params p) {
  using W = Words<T, SHORT>;
  constexpr int IDS = W::IDS, G = Elem<T>::VEC, U = IDS / (NT * G), DWORDS = IDS / (SHORT ? 2 : 1);
  extern __shared__ uint32_t shared[];  // the words, then the row's biases and (short words) their places in the slice
  const W words{shared};
  float* biases = reinterpret_cast<float*>(shared + DWORDS);
  int* places = reinterpret_cast<int*>(biases + p.n_bias);
  const int tid = threadIdx.x;
  Slice s;
  if (!slice_of<T, IDS>(p, s)) return;
  const Row r = row_of<LISTS, MASK, false>(p, s.row);
  const T* x = static_cast<const T*>(p.x) + s.row * p.xs + s.begin;
  T* out = static_cast<T*>(p.out) + s.row * p.os + s.begin;
  const bool listed = LISTS && (r.len > 0 || p.n_bias > 0), inside = s.begin >= 0 && s.begin + IDS <= p.V;
  int bits = r.bits;  // status bits that this thread met

  uint2 ahead[AHEAD];
  if (LISTS) load_ahead<SHORT>(r, 0, ahead);
  uint32_t there[U], allowed[U];
  groups_at<T, MASK, U>(p, r, s.begin + tid * G, inside, there, allowed);
  if (listed) {
    uint4* w4 = reinterpret_cast<uint4*>(shared);
#pragma unroll
    for (int i = 0; i < DWORDS / 4 / NT; ++i) w4[i * NT + tid] = make_uint4(0, 0, 0, 0);
    rows::lds_barrier();
  }
  // what is read: the groups with an allowed element
  Group v[U];
  if constexpr (!INPLACE) load_groups<T, U>(x, inside, there, allowed, v);

  if (listed) {
    const bool report = p.status && s.number == 0;
    if (p.n_bias) {
      const uint2* ids = reinterpret_cast<const uint2*>(p.bias_ids + s.row * p.bs);
      const float* b = p.bias + s.row * p.bs;
      for (int e = tid; e < p.n_bias; e += NT) {
        const uint2 id = ids[e];
        biases[e] = b[e];
        uint32_t at;
        const bool here = s.place_of(id, at);
        if (SHORT) places[e] = here ? (int)at : -1;
        if (here) words.bias(at, e);
        if (report && past(id, p.V)) bits |= DSV41_STATUS_BAD_BIAS;
      }
      rows::lds_barrier();
    }
    for_history<SHORT>(r, ahead, [&](int j0, const uint2 (&ids)[AHEAD]) {
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int j = j0 + k * NT;
        if (j >= r.len) continue;
        uint32_t at;
        if (s.place_of(ids[k], at)) {
          if (j < r.prompt) words.list(at);
          else words.say(at);
        }
        if (report && past(ids[k], p.V)) bits |= DSV41_STATUS_BAD_HISTORY;
      }
    });
    rows::lds_barrier();
  }

  const float value = r.bad ? __builtin_nanf("") : p.fill;
  const uint32_t instead = sizeof(T) == 4 ? __float_as_uint(value) : pack_bf16(value, value);
  uint32_t marked[U];  // elements whose word is not 0
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = (u * NT + tid) * G;
    marked[u] = listed ? words.marked(at) & allowed[u] : 0u;
    // in place, groups that stay as they are are neither read nor written
    if (INPLACE && allowed[u] && (marked[u] || allowed[u] != there[u])) load_group(x + at, there[u], v[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = (u * NT + tid) * G;
    if (INPLACE && !marked[u] && allowed[u] == there[u]) continue;
    if (LISTS) {
      // (few: a wave takes as many turns as its lane with the most of them)
#pragma unroll 1
      for (uint32_t m = marked[u]; m; m &= m - 1) {
        const int j = __builtin_ctz(m);
        set(v[u], j, r.knobs.apply(get(v[u], j, T{}), words.read(at + j, places, p.n_bias), biases), T{});
      }
    }
    if (allowed[u] != there[u]) drop(v[u], allowed[u], instead, T{});
    if (there[u]) store_group(out + at, there[u], v[u]);
  }

  // the first slice reports for its row
  if (p.status && s.number == 0) {
    bool some = true;
    if (MASK && r.mask) {
      some = false;
      const int full = p.V / 32;
      for (int k = tid; k < full; k += NT) some = some || r.mask[k] != 0;
      if (tid == 0 && p.V % 32) some = some || (r.mask[full] & ((1u << (p.V % 32)) - 1)) != 0;
    }
    if (!__syncthreads_or(some)) bits |= DSV41_STATUS_NO_TOKEN;
    if (__syncthreads_or(bits & DSV41_STATUS_BAD_HISTORY)) bits |= DSV41_STATUS_BAD_HISTORY;
    if (__syncthreads_or(bits & DSV41_STATUS_BAD_BIAS)) bits |= DSV41_STATUS_BAD_BIAS;
    if (tid == 0) p.status[s.row] = bits;
  }
}

template <typename T, bool LISTS, bool MASK>
__global__ __launch_bounds__(NT, 8) void process_grad_kernel(Params p) {
  constexpr int IDS = sizeof(T) == 4 ? SLICE : SHORT_SLICE, G = Elem<T>::VEC, U = IDS / (NT * G);
  __shared__ uint32_t in_history[IDS / 32], positive[IDS / 32];  // of an id that is in the history: whether x + b > 0
  extern __shared__ int places[];                                // the bias entries' places in the slice
  const int tid = threadIdx.x;
  Slice s;
  if (!slice_of<T, IDS>(p, s)) return;
  const Row r = row_of<LISTS, MASK, true>(p, s.row);
  const T* x = static_cast<const T*>(p.x) + s.row * p.xs + s.begin;
  const T* g = static_cast<const T*>(p.grad) + s.row * p.gs + s.begin;
  T* out = static_cast<T*>(p.out) + s.row * p.os + s.begin;
  const bool listed = LISTS && r.len > 0, inside = s.begin >= 0 && s.begin + IDS <= p.V;

  uint2 ahead[AHEAD];
  if (LISTS) load_ahead<true>(r, 0, ahead);
  uint32_t there[U], allowed[U];
  groups_at<T, MASK, U>(p, r, s.begin + tid * G, inside, there, allowed);
  if (listed) {
    static_assert(IDS / 32 <= NT);
    if (tid < IDS / 32) in_history[tid] = positive[tid] = 0;
    rows::lds_barrier();
  }
  Group v[U];
  load_groups<T, U>(g, inside, there, allowed, v);

  if (listed) {
    for_history<true>(r, ahead, [&](int j0, const uint2 (&ids)[AHEAD]) {
      float logit[AHEAD];
      uint32_t at[AHEAD];
      bool here[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        here[k] = j0 + k * NT < r.len && s.place_of(ids[k], at[k]);
        if (here[k]) logit[k] = Elem<T>::one(x + at[k]);
      }
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        if (!here[k]) continue;
        atomicOr(&in_history[at[k] >> 5], 1u << (at[k] & 31));
        if (logit[k] > 0.f) atomicOr(&positive[at[k] >> 5], 1u << (at[k] & 31));
      }
    });
    if (p.n_bias) {
      const uint2* ids = reinterpret_cast<const uint2*>(p.bias_ids + s.row * p.bs);
      const float* b = p.bias + s.row * p.bs;
      for (int e = tid; e < p.n_bias; e += NT) {
        uint32_t at;
        places[e] = s.place_of(ids[e], at) ? (int)at : -1;
      }
      rows::lds_barrier();
      // the last entry of an id in the history says its sign anew
      for (int e = tid; e < p.n_bias; e += NT) {
        const int at = places[e];
        if (at < 0 || !(in_history[at >> 5] >> (at & 31) & 1)) continue;
        int later = e + 1;
        while (later < p.n_bias && places[later] != at) ++later;
        if (later < p.n_bias) continue;
        const float sum = Elem<T>::one(x + at) + b[e];
        if (sum > 0.f) atomicOr(&positive[at >> 5], 1u << (at & 31));
        else atomicAnd(&positive[at >> 5], ~(1u << (at & 31)));
      }
    }
    rows::lds_barrier();
  }

  const float value = r.bad ? __builtin_nanf("") : 0.f, rp = r.knobs.rp;
  const uint32_t instead = sizeof(T) == 4 ? __float_as_uint(value) : pack_bf16(value, value);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = (u * NT + tid) * G;
    if (listed) {
      const uint32_t sign = positive[at >> 5] >> (at & 31);
#pragma unroll 1
      for (uint32_t m = in_history[at >> 5] >> (at & 31) & allowed[u]; m; m &= m - 1) {
        const int j = __builtin_ctz(m);
        const float y = get(v[u], j, T{});
        set(v[u], j, sign >> j & 1 ? y / rp : y * rp, T{});
      }
    }
    if (allowed[u] != there[u]) drop(v[u], allowed[u], instead, T{});
    if (there[u]) store_group(out + at, there[u], v[u]);
  }
}

// ---------------------------------------------------------------------------------------- host
// (the last slice of a row that begins at a memory line may have nothing)
int slices_of(int V, int ids) { return (V + rows::MOST_SKEW - 1 + ids - 1) / ids; }
dim3 grid_of(Params& p, int ids) {
  p.slices = slices_of(p.V, ids);
  return dim3((unsigned)(((int64_t)p.rows * p.slices + 7) / 8 * 8));
}

template <typename T, bool LISTS, bool MASK, bool INPLACE, bool SHORT>
void launch(Params p, hipStream_t s) {
  const dim3 grid = grid_of(p, Words<T, SHORT>::IDS);
  const size_t lds = LISTS ? SLICE * sizeof(uint32_t) + (size_t)p.n_bias * (SHORT ? 8 : 4) : 0;
  hipLaunchKernelGGL((process_kernel<T, LISTS, MASK, INPLACE, SHORT>), grid, dim3(NT), lds, s, p);
}
// Words of 16 bits take what they hold of bf16 rows' lists, in batches that fill the GPU with the longer slices too.  With
// histories of 2048 and 4096 and in place with 2048, us, 32 and 16 bits: 2048 rows 244 and 238, 288 and 264, 257 and 227; 500
// rows 68 and 66, 80 and 74, 57 and 50; 200 rows 26.3 and 26.5, 31.0 and 29.5, 26.4 and 23.9.
template <typename T, bool MASK, bool INPLACE>
void launch_lists(const Params& p, hipStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (p.hist_len <= SHORT_HISTORY && p.n_bias <= SHORT_BIAS && (int64_t)p.rows * slices_of(p.V, SHORT_SLICE) >= 1024)
      return launch<T, true, MASK, INPLACE, true>(p, s);
  launch<T, true, MASK, INPLACE, false>(p, s);
}
template <typename T, bool INPLACE>
void launch(const Params& p, hipStream_t s) {
  const bool lists = p.n_bias || p.history || p.knobs_of_rows();
  if (lists && p.mask) launch_lists<T, true, INPLACE>(p, s);
  else if (lists) launch_lists<T, false, INPLACE>(p, s);
  else if (p.mask) launch<T, false, true, INPLACE, false>(p, s);
  else launch<T, false, false, INPLACE, false>(p, s);
}
template <typename T>
void launch_grad(Params p, hipStream_t s) {
  const dim3 grid = grid_of(p, sizeof(T) == 4 ? SLICE : SHORT_SLICE);
  const size_t lds = (size_t)p.n_bias * sizeof(int);
  const bool lists = p.history || p.knobs_of_rows();
  if (lists && p.mask) hipLaunchKernelGGL((process_grad_kernel<T, true, true>), grid, dim3(NT), lds, s, p);
  else if (lists) hipLaunchKernelGGL((process_grad_kernel<T, true, false>), grid, dim3(NT), lds, s, p);
  else if (p.mask) hipLaunchKernelGGL((process_grad_kernel<T, false, true>), grid, dim3(NT), lds, s, p);
  else hipLaunchKernelGGL((process_grad_kernel<T, false, false>), grid, dim3(NT), lds, s, p);
}

constexpr int64_t MAX_GRID = (1 << 22) - 8;  // workgroups of 512 threads: HIP's grids stop short of 2^32 threads

int check_desc(const dsv41_process_desc* d, bool grad) {
  if (!d) return fail(DSV41_E_INVALID, "process descriptor is NULL");
  if (d->struct_size != sizeof(dsv41_process_desc))
    return fail(DSV41_E_ABI, "dsv41_process_desc size mismatch (rebuild the binding)");
  const int unit = d->logits_dtype == DSV41_DTYPE_F32 ? 4 : 2;
  if (int rc = rows::check_rows(d->rows, d->vocab, d->logits_dtype, d->logits_row_stride, d->logits, 1.f)) return rc;
  if (!d->out) return fail(DSV41_E_INVALID, "out is required");
  if (d->out_row_stride < d->vocab) return fail(DSV41_E_INVALID, "out row stride is smaller than the vocabulary");
  if ((uintptr_t)d->out % unit) return fail(DSV41_E_INVALID, "out is not aligned to its type");
  if (grad) {
    if (!d->grad) return fail(DSV41_E_INVALID, "grad is required");
    if ((uintptr_t)d->grad % unit) return fail(DSV41_E_INVALID, "grad is not aligned to its type");
    if (d->grad_row_stride < 0 || (d->grad_row_stride != 0 && d->grad_row_stride < d->vocab))
      return fail(DSV41_E_INVALID, "grad row stride is smaller than the vocabulary");
    if (d->out == d->logits || d->out == d->grad) return fail(DSV41_E_INVALID, "the gradient is not written in place");
  } else if (d->out == d->logits && d->rows > 1 && d->out_row_stride != d->logits_row_stride) {
    return fail(DSV41_E_INVALID, "in place, out has the row stride of the logits");
  }
  if (!(isfinite(d->repetition_penalty) && d->repetition_penalty > 0.f))
    return fail(DSV41_E_INVALID, "repetition_penalty must be finite and positive");
  if (!isfinite(d->presence_penalty) || !isfinite(d->frequency_penalty))
    return fail(DSV41_E_INVALID, "presence_penalty and frequency_penalty must be finite");
  if (d->hist_len < 0 || (d->hist_len > 0 && !d->history)) return fail(DSV41_E_INVALID, "hist_len needs a history");
  if (d->hist_len > 0 && d->history_row_stride < 0) return fail(DSV41_E_INVALID, "history row stride is negative");
  if (d->hist_len > MAX_HISTORY) return fail(DSV41_E_UNSUPPORTED, "histories above 524287 tokens are not supported");
  if (d->bias_len < 0 || (d->bias_len > 0 && (!d->bias_ids || !d->bias)))
    return fail(DSV41_E_INVALID, "bias_len needs bias_ids and bias");
  if (d->bias_len > 0 && d->bias_row_stride < 0) return fail(DSV41_E_INVALID, "bias row stride is negative");
  if (d->bias_len > MAX_BIAS) return fail(DSV41_E_UNSUPPORTED, "more than 4095 biased tokens a row are not supported");
  if (d->mask) {
    if (d->masks <= 0 || (!d->mask_rows && d->masks != 1 && d->masks != d->rows))
      return fail(DSV41_E_INVALID, "without mask_rows there is one mask, or one per row");
    if (d->mask_row_stride < 0) return fail(DSV41_E_INVALID, "mask row stride is negative");
  }
  if (isnan(d->fill)) return fail(DSV41_E_INVALID, "fill must be a number");
  if ((int64_t)d->rows * slices_of(d->vocab, SLICE) > MAX_GRID)
    return fail(DSV41_E_UNSUPPORTED, "more than 2^22 row slices are not supported");
  return DSV41_OK;
}

int run(const dsv41_process_desc* d, bool grad, void* stream) {
  if (int rc = check_desc(d, grad)) return rc;
  Params p{};
  p.x = d->logits;
  p.xs = d->logits_row_stride;
  p.out = d->out;
  p.os = d->out_row_stride;
  p.grad = d->grad;
  p.gs = d->grad_row_stride;
  p.rows = d->rows;
  p.V = d->vocab;
  const bool neutral = !d->repetition_penalties && !d->presence_penalties && !d->frequency_penalties &&
                       d->repetition_penalty == 1.f && d->presence_penalty == 0.f && d->frequency_penalty == 0.f;
  if (d->hist_len > 0 && !neutral) {
    p.history = d->history;
    p.hs = d->history_row_stride;
    p.hist_len = d->hist_len;
    p.lens = d->history_lens;
    p.prompt_lens = d->history_prompt_lens;
  }
  // (rows' knobs are looked at without a history, too)
  p.rps = d->repetition_penalties;
  p.press = d->presence_penalties;
  p.freqs = d->frequency_penalties;
  p.rp = d->repetition_penalty;
  p.pres = d->presence_penalty;
  p.freq = d->frequency_penalty;
  // (a bias alone shifts: its gradient is the identity)
  if (d->bias_len > 0 && (!grad || p.history)) {
    p.bias_ids = d->bias_ids;
    p.bias = d->bias;
    p.bs = d->bias_row_stride;
    p.n_bias = d->bias_len;
  }
  if (d->mask) {
    p.mask = reinterpret_cast<const uint32_t*>(d->mask);
    p.ms = d->mask_row_stride;
    p.masks = d->masks;
    p.mask_rows = d->mask_rows;
  }
  p.fill = d->fill;
  p.status = d->out_status;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool f32 = d->logits_dtype == DSV41_DTYPE_F32;
  if (grad) f32 ? launch_grad<float>(p, s) : launch_grad<bf16_t>(p, s);
  else if (d->out == d->logits) f32 ? launch<float, true>(p, s) : launch<bf16_t, true>(p, s);
  else f32 ? launch<float, false>(p, s) : launch<bf16_t, false>(p, s);
  DSV41_HIP_CHECK(hipGetLastError());
  return DSV41_OK;
}

}  // namespace process
}  // namespace dsv41

extern "C" int dsv41_process_run(const dsv41_process_desc* d, void* stream) {
  return dsv41::process::run(d, false, stream);
}

extern "C" int dsv41_process_grad_run(const dsv41_process_desc* d, void* stream) {
  return dsv41::process::run(d, true, stream);
}
