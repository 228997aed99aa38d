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
static_assert(SLICE % 32 == 0, "a slice begins at a word of a mask");

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
  // the gradient's factor is 1 / rp or rp
  __device__ __forceinline__ float slope(float g, float x, uint32_t word, const float* bias) const {
    if (word >> ENTRY_SHIFT) x = x + bias[(word >> ENTRY_SHIFT) - 1];
    return x > 0.0f ? g / rp : g * rp;
  }
};

// G elements from p of which the first n exist (the others come as 0)
template <typename T>
__device__ __forceinline__ void load_group(const T* p, int n, float (&v)[Elem<T>::VEC]) {
  constexpr int G = Elem<T>::VEC;
  uint32_t w[4] = {0, 0, 0, 0};
  if (n >= G) {
    rows::load16<false>(p, w);
  } else {
#pragma unroll
    for (int j = 0; j < G; ++j)
      if (j < n) Elem<T>::put(w, j, p[j]);
  }
  Elem<T>::unpack(w, v);
}
template <typename T>
__device__ __forceinline__ void store_group(T* p, int n, const float (&v)[Elem<T>::VEC]) {
  constexpr int G = Elem<T>::VEC;
  if (n >= G) {
    rows::store_full(p, 0, v);
  } else {
#pragma unroll
    for (int j = 0; j < G; ++j)
      if (j < n) rows::store_one(p + j, v[j]);
  }
}

template <typename T, bool LISTS, bool MASK, int MODE>
__global__ __launch_bounds__(NT) void process_kernel(Params p) {
  constexpr int G = Elem<T>::VEC, U = SLICE / (NT * G);
  extern __shared__ uint32_t words[];  // SLICE words, then the row's biases
  float* biases = reinterpret_cast<float*>(words + SLICE);
  const int tid = threadIdx.x;
  // a row's slices one after another on one XCD (workgroups go round-robin over the eight)
  const int64_t items = (int64_t)p.rows * p.slices, per = (items + 7) / 8;
  const int64_t item = (int64_t)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int64_t)(blockIdx.x >> 3) >= per || item >= items) return;
  const int row = (int)(item / p.slices), slice = (int)(item % p.slices);
  const int s0 = slice * SLICE, n = min(SLICE, p.V - s0);
  const T* x = static_cast<const T*>(p.x) + row * p.xs + s0;
  T* out = static_cast<T*>(p.out) + row * p.os + s0;

  float v[U][G];
  if constexpr (MODE != INPLACE) {
    const T* from = MODE == GRAD ? static_cast<const T*>(p.grad) + row * p.gs + s0 : x;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = (u * NT + tid) * G;
      if (i < n) load_group(from + i, n - i, v[u]);
    }
  }

  Knobs knobs{1.f, 0.f, 0.f};
  bool bad = false;
  int bits = 0;  // status bits that this thread met
  if constexpr (LISTS) {
    knobs.rp = p.rps ? p.rps[row] : p.rp;
    knobs.pres = p.press ? p.press[row] : p.pres;
    knobs.freq = p.freqs ? p.freqs[row] : p.freq;
    if (!(isfinite(knobs.rp) && knobs.rp > 0.f) || !isfinite(knobs.pres) || !isfinite(knobs.freq)) {
      bad = true;
      bits |= DSV41_STATUS_BAD_PENALTY;
    }
    uint4* w4 = reinterpret_cast<uint4*>(words);
#pragma unroll
    for (int i = 0; i < SLICE / 4 / NT; ++i) w4[i * NT + tid] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (p.n_bias) {
      const int64_t* ids = p.bias_ids + row * p.bs;
      const float* b = p.bias + row * p.bs;
      for (int e = tid; e < p.n_bias; e += NT) {
        const int64_t id = ids[e];
        biases[e] = b[e];
        const uint64_t at = (uint64_t)(id - s0);
        if (id >= 0 && at < (uint64_t)n) atomicMax(&words[at], (uint32_t)(e + 1) << ENTRY_SHIFT);
        if (id >= p.V) bits |= DSV41_STATUS_BAD_BIAS;
      }
      __syncthreads();
    }
    if (p.history && !(knobs.rp == 1.f && knobs.pres == 0.f && knobs.freq == 0.f)) {
      const int64_t* h = p.history + row * p.hs;
      const int len = p.lens ? min(max(p.lens[row], 0), p.hist_len) : p.hist_len;
      const int prompt = p.prompt_lens ? p.prompt_lens[row] : 0;
      for (int j = tid; j < len; j += NT) {
        const int64_t id = h[j];
        const uint64_t at = (uint64_t)(id - s0);
        if (id >= 0 && at < (uint64_t)n) {
          if (j < prompt) atomicOr(&words[at], SEEN);
          else atomicAdd(&words[at], 1u);
        }
        if (id >= p.V) bits |= DSV41_STATUS_BAD_HISTORY;
      }
    }
    __syncthreads();
  }
  const uint32_t* mask = nullptr;
  if constexpr (MASK) {
    const int m = p.mask_rows ? p.mask_rows[row] : p.masks == 1 ? 0 : row;
    if (m >= p.masks) {
      bad = true;
      bits |= DSV41_STATUS_BAD_MASK;
    } else if (m >= 0) {
      mask = p.mask + m * p.ms;
    }
  }

  const float nan = __builtin_nanf("");
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = (u * NT + tid) * G;
    if (i >= n) continue;
    uint32_t w[G];
#pragma unroll
    for (int j = 0; j < G; ++j) w[j] = LISTS ? words[i + j] : 0;
    uint32_t allowed = (1u << G) - 1;
    if (MASK && mask) allowed &= mask[(s0 + i) >> 5] >> ((s0 + i) & 31);
    if constexpr (MODE == INPLACE) {
      bool all = true;
      float o[G];
#pragma unroll
      for (int j = 0; j < G; ++j) {
        o[j] = bad ? nan : p.fill;
        all = all && (bad || !(allowed >> j & 1));
      }
      if (all) {
        store_group(out + i, n - i, o);
      } else {
#pragma unroll
        for (int j = 0; j < G; ++j) {
          if (i + j >= n) continue;
          if (!(allowed >> j & 1)) rows::store_one(out + i + j, p.fill);
          else if (w[j]) rows::store_one(out + i + j, knobs.apply(Elem<T>::one(x + i + j), w[j], biases));
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < G; ++j) {
        if (MODE == GRAD) {
          if (w[j] & (SEEN | COUNT) && knobs.rp != 1.f && i + j < n)
            v[u][j] = knobs.slope(v[u][j], Elem<T>::one(x + i + j), w[j], biases);
          if (!(allowed >> j & 1)) v[u][j] = 0.f;
        } else {
          if (w[j]) v[u][j] = knobs.apply(v[u][j], w[j], biases);
          if (!(allowed >> j & 1)) v[u][j] = p.fill;
        }
        if (bad) v[u][j] = nan;
      }
      store_group(out + i, n - i, v[u]);
    }
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
  if ((int64_t)d->rows * ((d->vocab + SLICE - 1) / SLICE) > MAX_GRID)
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
  p.slices = (d->vocab + SLICE - 1) / SLICE;
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
