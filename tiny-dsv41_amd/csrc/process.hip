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
// One pass: a workgroup takes a slice of SLICE ids of a row.  What the lists say of the slice's ids goes into
// one LDS word each, by integer atomics, so in any order to the same words: 12 bits the last bias entry that
// names the id (+ 1), one bit "in the history", 19 bits its count.  The slice's elements are on their way
// meanwhile, and most words are 0 then: such elements go out as they came.  Every slice reads all of its
// row's lists, which therefore stay on one XCD (whose L2 serves all but the first).
// In place nothing is read but what a list names, and nothing written but that and what is masked.

#include <math.h>

#include "row_scan.h"

namespace dsv41 {
namespace process {

using rows::bf16_t;
using rows::Elem;

constexpr int NT = 512;
constexpr int SLICE = 8192;  // ids; 32 KB of words: four workgroups a CU
constexpr int COUNT_BITS = 19;
constexpr uint32_t COUNT = (1u << COUNT_BITS) - 1, SEEN = 1u << COUNT_BITS;
constexpr int ENTRY_SHIFT = COUNT_BITS + 1;
constexpr int MAX_BIAS = (1 << (32 - ENTRY_SHIFT)) - 1;  // entries of a row's list

constexpr int COPY = 0, INPLACE = 1, GRAD = 2;

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
};

// What the row's knobs and lists make of an element whose word is not 0.
struct Knobs {
  float rp, pres, freq;
  __device__ __forceinline__ float apply(float x, uint32_t word, const float* bias) const {
    if (word >> ENTRY_SHIFT) x = x + bias[(word >> ENTRY_SHIFT) - 1];
    const uint32_t c = word & COUNT;
    if (word & (SEEN | COUNT)) {
      x = x > 0.0f ? x / rp : x * rp;
      const float f = freq * (float)c;
      x = x - f;
      if (c > 0) x = x - pres;
    }
    return x;
  }
  // the gradient's factor is 1 / rp or rp, of ids that are not only biased
  __device__ __forceinline__ float slope(float g, float x, uint32_t word, const float* bias) const {
    if (!(word & (SEEN | COUNT))) return g;
    if (word >> ENTRY_SHIFT) x = x + bias[(word >> ENTRY_SHIFT) - 1];
    return x > 0.0f ? g / rp : g * rp;
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
// The word of element `at` of a slice: a thread's group of 8 bf16 elements lies in two planes, so that either
// half of it is read without bank conflicts.
template <typename T>
__device__ __forceinline__ int word_at(int at) {
  return Elem<T>::VEC == 4 ? at : ((at >> 2 & 1) * (SLICE / 2)) + (at >> 3 << 2) + (at & 3);
}

template <typename T, bool LISTS, bool MASK, int MODE>
__global__ __launch_bounds__(NT, 8) void process_kernel(Params p) {
  constexpr int G = Elem<T>::VEC, U = SLICE / (NT * G), AHEAD = 8;
  extern __shared__ uint32_t words[];  // SLICE words, then the row's biases
  float* biases = reinterpret_cast<float*>(words + SLICE);
  const int tid = threadIdx.x;
  // a row's slices one after another on one XCD (workgroups go round-robin over the eight)
  const uint32_t item = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  const int row = (int)(item / (uint32_t)p.slices), slice = (int)(item % (uint32_t)p.slices);
  if (row >= p.rows) return;
  const T* x = static_cast<const T*>(p.x) + row * p.xs;
  T* out = static_cast<T*>(p.out) + row * p.os;
  // slices begin at memory lines of the result
  const int begin = slice * SLICE - rows::skew_of(out);
  if (begin >= p.V) return;
  const T* from = MODE == GRAD ? static_cast<const T*>(p.grad) + row * p.gs : x;

  // the row's own values, all on their way at once: arrays that are not given are read at the arguments' begin
  typedef const __attribute__((address_space(4))) int32_t* constant_t;
  const uintptr_t nowhere = (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
  auto value_of = [&](const void* a) { return *(constant_t)(a ? (uintptr_t)a + 4 * (int64_t)row : nowhere); };
  const int m_row = MASK ? value_of(p.mask_rows) : 0;
  const int rp_row = LISTS ? value_of(p.rps) : 0, pres_row = LISTS ? value_of(p.press) : 0, freq_row = LISTS ? value_of(p.freqs) : 0;
  const int len_row = LISTS ? value_of(p.lens) : 0, prompt_row = LISTS ? value_of(p.prompt_lens) : 0;
  Knobs knobs{1.f, 0.f, 0.f};
  bool bad = false;
  int bits = 0;  // status bits that this thread met
  const uint32_t* mask = nullptr;
  if constexpr (MASK) {
    const int m = p.mask_rows ? m_row : p.masks == 1 ? 0 : row;
    bad = m >= p.masks;
    if (bad) bits |= DSV41_STATUS_BAD_MASK;
    mask = m >= 0 && !bad ? p.mask + m * p.ms : nullptr;
  }
  bool listed = false;
  int len = 0, prompt = 0;
  const int64_t* h = nullptr;
  if constexpr (LISTS) {
    knobs.rp = p.rps ? __int_as_float(rp_row) : p.rp;
    knobs.pres = p.press ? __int_as_float(pres_row) : p.pres;
    knobs.freq = p.freqs ? __int_as_float(freq_row) : p.freq;
    if (!(isfinite(knobs.rp) && knobs.rp > 0.f) || !isfinite(knobs.pres) || !isfinite(knobs.freq)) {
      bad = true;
      bits |= DSV41_STATUS_BAD_PENALTY;
    }
    // (a gradient asks for the repetition penalty alone)
    if (p.history && !(knobs.rp == 1.f && (MODE == GRAD || (knobs.pres == 0.f && knobs.freq == 0.f)))) {
      h = p.history + row * p.hs;
      len = p.lens ? min(max(len_row, 0), p.hist_len) : p.hist_len;
      prompt = p.prompt_lens ? prompt_row : 0;
    }
    listed = len > 0 || (p.n_bias > 0 && (MODE != GRAD || h));
  }

  // the history's first entries, ahead of the slice itself: loads come back in order
  uint2 ahead[AHEAD];
  const uint2* h2 = reinterpret_cast<const uint2*>(h);
  if (LISTS) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (tid + k * NT < len) ahead[k] = h2[tid + k * NT];
  }
  // which elements of the thread's groups there are, and which of them the mask allows
  const bool inside = begin >= 0 && begin + SLICE <= p.V;  // (all of them)
  uint32_t there[U], allowed[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = begin + (u * NT + tid) * G;
    there[u] = ALL<T>;
    if (!inside) {
      const int lo = max(-i, 0), hi = min(p.V - i, G);  // elements [lo, hi)
      there[u] = lo < hi ? (ALL<T> << lo) & (ALL<T> >> (G - hi)) : 0u;
    }
    allowed[u] = bad ? 0u : there[u];
    if (MASK && mask && there[u]) {
      const int k = max(i, 0) >> 5, last = (p.V - 1) >> 5;
      const uint64_t both = (uint64_t)mask[min(k + 1, last)] << 32 | mask[k];
      allowed[u] &= i >= 0 ? (uint32_t)(both >> (i & 31)) : (uint32_t)(both << -i);
    }
  }
  if (LISTS && listed) {
    uint4* w4 = reinterpret_cast<uint4*>(words);
#pragma unroll
    for (int i = 0; i < SLICE / 4 / NT; ++i) w4[i * NT + tid] = make_uint4(0, 0, 0, 0);
    rows::lds_barrier();
  }
  // what is read: the groups with an allowed element
  Group v[U];
  if constexpr (MODE != INPLACE) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (allowed[u]) load_group(from + begin + (u * NT + tid) * G, there[u], v[u]);
  }

  if constexpr (LISTS) {
    if (listed) {
      // ids in [max(begin, 0), begin + SLICE) and below V, as unsigned offsets of the slice
      const uint32_t first = (uint32_t)max(-begin, 0), count = (uint32_t)min(SLICE, p.V - begin) - first;
      const bool report = MODE != GRAD && p.status && slice == 0;
      if (p.n_bias) {
        const uint2* ids = reinterpret_cast<const uint2*>(p.bias_ids + row * p.bs);
        const float* b = p.bias + row * p.bs;
        for (int e = tid; e < p.n_bias; e += NT) {
          const uint2 id = ids[e];
          biases[e] = b[e];
          const uint32_t at = id.x - (uint32_t)begin;
          if (id.y == 0 && at - first < count) atomicMax(&words[word_at<T>(at)], (uint32_t)(e + 1) << ENTRY_SHIFT);
          if (report && (int)id.y >= 0 && (id.y > 0 || id.x >= (uint32_t)p.V)) bits |= DSV41_STATUS_BAD_BIAS;
        }
        rows::lds_barrier();
      }
      auto mark = [&](int j, uint2 id) {
        const uint32_t at = id.x - (uint32_t)begin;
        if (id.y == 0 && at - first < count) {
          if (j < prompt) atomicOr(&words[word_at<T>(at)], SEEN);
          else atomicAdd(&words[word_at<T>(at)], 1u);
        }
        if (report && (int)id.y >= 0 && (id.y > 0 || id.x >= (uint32_t)p.V)) bits |= DSV41_STATUS_BAD_HISTORY;
      };
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (tid + k * NT < len) mark(tid + k * NT, ahead[k]);
      for (int j0 = AHEAD * NT; j0 < len; j0 += AHEAD * NT) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
          if (j0 + tid + k * NT < len) ahead[k] = h2[j0 + tid + k * NT];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
          if (j0 + tid + k * NT < len) mark(j0 + tid + k * NT, ahead[k]);
      }
      rows::lds_barrier();
    }
  }

  const float value = bad ? __builtin_nanf("") : MODE == GRAD ? 0.f : p.fill;
  const uint32_t instead = sizeof(T) == 4 ? __float_as_uint(value) : pack_bf16(value, value);
  uint32_t marked[U];  // elements whose word is not 0
  Group xs[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    marked[u] = 0;
    const int at = (u * NT + tid) * G;
    if (LISTS && listed) {
#pragma unroll
      for (int q = 0; q < G; q += 4) {
        const uint4 w = *reinterpret_cast<const uint4*>(words + word_at<T>(at + q));
        marked[u] |= (min(w.x, 1u) | min(w.y, 1u) << 1 | min(w.z, 1u) << 2 | min(w.w, 1u) << 3) << q;
      }
      marked[u] &= allowed[u];
    }
    // in place, groups that stay as they are are neither read nor written; of a gradient, the logits are
    // read where a sign is asked for
    if (MODE == INPLACE && allowed[u] && (marked[u] || allowed[u] != there[u])) load_group(x + begin + at, there[u], v[u]);
    if (MODE == GRAD && marked[u]) load_group(x + begin + at, there[u], xs[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = (u * NT + tid) * G;
    if (MODE == INPLACE && !marked[u] && allowed[u] == there[u]) continue;
    if (LISTS) {
      // (few: a wave takes as many turns as its lane with the most of them)
#pragma unroll 1
      for (uint32_t m = marked[u]; m; m &= m - 1) {
        const int j = __builtin_ctz(m);
        const uint32_t word = words[word_at<T>(at + j)];
        const float y = MODE == GRAD ? knobs.slope(get(v[u], j, T{}), get(xs[u], j, T{}), word, biases)
                                     : knobs.apply(get(v[u], j, T{}), word, biases);
        set(v[u], j, y, T{});
      }
    }
    if (allowed[u] != there[u]) drop(v[u], allowed[u], instead, T{});
    if (there[u]) store_group(out + begin + at, there[u], v[u]);
  }

  // the first slice reports for its row
  if (MODE != GRAD && p.status && slice == 0) {
    bool some = true;
    if (MASK && mask) {
      some = false;
      const int full = p.V / 32;
      for (int k = tid; k < full; k += NT) some = some || mask[k] != 0;
      if (tid == 0 && p.V % 32) some = some || (mask[full] & ((1u << (p.V % 32)) - 1)) != 0;
    }
    if (!__syncthreads_or(some)) bits |= DSV41_STATUS_NO_TOKEN;
    if (__syncthreads_or(bits & DSV41_STATUS_BAD_HISTORY)) bits |= DSV41_STATUS_BAD_HISTORY;
    if (__syncthreads_or(bits & DSV41_STATUS_BAD_BIAS)) bits |= DSV41_STATUS_BAD_BIAS;
    if (tid == 0) p.status[row] = bits;
  }
}

template <typename T, bool LISTS, bool MASK, int MODE>
void launch(const Params& p, hipStream_t s) {
  const int64_t items = (int64_t)p.rows * p.slices;
  const size_t lds = LISTS ? SLICE * sizeof(uint32_t) + p.n_bias * sizeof(float) : 0;
  hipLaunchKernelGGL((process_kernel<T, LISTS, MASK, MODE>), dim3((unsigned)((items + 7) / 8 * 8)), dim3(NT), lds, s, p);
}
template <typename T, int MODE>
void launch(const Params& p, hipStream_t s) {
  const bool lists = p.n_bias || p.history;
  if (lists && p.mask) launch<T, true, true, MODE>(p, s);
  else if (lists) launch<T, true, false, MODE>(p, s);
  else if (p.mask) launch<T, false, true, MODE>(p, s);
  else launch<T, false, false, MODE>(p, s);
}

constexpr int64_t MAX_GRID = (1 << 22) - 8;  // workgroups of 512 threads: HIP's grids stop short of 2^32 threads

// (the last slice of a row that begins at a memory line may have nothing)
int slices_of(int V) { return (V + rows::MOST_SKEW - 1 + SLICE - 1) / SLICE; }

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
  if (d->hist_len > (int)COUNT) return fail(DSV41_E_UNSUPPORTED, "histories above 524287 tokens are not supported");
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
  if ((int64_t)d->rows * slices_of(d->vocab) > MAX_GRID)
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
  p.slices = slices_of(d->vocab);
  const bool neutral = !d->repetition_penalties && !d->presence_penalties && !d->frequency_penalties &&
                       d->repetition_penalty == 1.f && d->presence_penalty == 0.f && d->frequency_penalty == 0.f;
  if (d->hist_len > 0 && !neutral) {
    p.history = d->history;
    p.hs = d->history_row_stride;
    p.hist_len = d->hist_len;
    p.lens = d->history_lens;
    p.prompt_lens = d->history_prompt_lens;
    p.rps = d->repetition_penalties;
    p.press = d->presence_penalties;
    p.freqs = d->frequency_penalties;
  }
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
  if (grad) f32 ? launch<float, GRAD>(p, s) : launch<bf16_t, GRAD>(p, s);
  else if (d->out == d->logits) f32 ? launch<float, INPLACE>(p, s) : launch<bf16_t, INPLACE>(p, s);
  else f32 ? launch<float, COPY>(p, s) : launch<bf16_t, COPY>(p, s);
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
