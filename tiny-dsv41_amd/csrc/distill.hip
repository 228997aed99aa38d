// distill.hip — divergence of a student's rows of logits from a teacher's top tokens, and its gradient.
//
// One row: student logits x [V], p = softmax(x / T); the teacher's list of tokens with log-probs lq
// (entries with a negative id are none).  With m = max x, d_i = (x_i - m) / T, S = sum exp(d_i), and
// S_rest the part of S outside the list:
//   renormalize: q = softmax(lq) over the list;  L = sum_k q_k (log q_k - log p_k)
//   rest: q_k = exp(lq_k), q_rest = 1 - sum q_k, p_rest = S_rest / S;
//         L = sum_k q_k (lq_k - log p_k) + q_rest (log q_rest - log p_rest)
//   dL/dx_k = (Q p_k - q_k) / T in the list, dL/dx_i = p_i (Q - q_rest / p_rest) / T outside,
//   Q = sum q + q_rest (1, and q_rest 0, when renormalized).
// p_rest may be many orders below 1, so S_rest is summed by itself: the list's tokens are bits of a map
// in LDS that the pass over the row treats as masked.  What is left of nearly cancelling terms, the
// divergence, is formed in fp64 from the list's logits.  fp32 log-probs do not carry a rest mass below
// 2^-20, which counts as none.  Where no logit outside the list is above its type's lowest value and the list's
// are, that value is a mask like -inf: the student has no mass for the teacher's rest.
//
// Forward: one read of the row, 4096 bf16 rows of 151936 with 64 entries (a tenth of them without) in
// 201 us, 5.6 TB/s of what is read: vector instructions, 10 an element; 512 fp32 rows in 56 us, 5.5 TB/s.
// Backward: one read, one write, 409 us for the same 4096 rows, 5.8 TB/s.
#include <math.h>

#include "row_scan.h"

namespace dsv41 {
namespace distill {

using rows::bf16_t;
using rows::Cut;
using rows::Elem;
using rows::GROUP;
using rows::NT;
using rows::Scale;
using rows::State;
using rows::WAVES;

constexpr int MAP = 5120 * 32;                     // bits of the map: 20 KB
constexpr int MAX_LEN = MAP - rows::MOST_SKEW;  // elements of one slice
constexpr double REST_FLOOR = 0x1p-20;
constexpr double MOST_MASS = 1.01;  // log-probs rounded to bf16 may add up to 1 + 2^-8 |lq| or so
constexpr int STATS = 7;            // per row, see write_row

struct SliceState {
  State s;
  int32_t flags, pad;
};

struct Params {
  const void* logits;
  int64_t stride;
  const int64_t* ids;
  const float* lq;
  int rows, V, K, slices, len, rest;
  Scale sc;
  float* out_loss;
  int32_t* out_status;
  double* out_stats;
  SliceState* states;  // [rows, slices]
};

struct Shared {
  alignas(16) uint32_t named[MAP / 32];  // whole 16 bytes
  double red[4 * WAVES];
  int flags;
};
template <typename T>
constexpr float lowest() {
  return sizeof(T) == 4 ? -0x1.fffffep127f : -0x1.fep127f;
}
constexpr int LIVE = 1 << 16;  // the list has an entry (above the status bits)

// What the gradient needs of a row: p_k = exp((x_k - m) / T) / S in its list; p_i (Q - q_rest / p_rest) =
// others exp((x_i - base) / T) outside, with the largest of these logits as base, since p_rest may lie
// below what fp32 holds; Q; q_k = share exp(lq_k - top), with the list's largest lq apart, to which the logarithm of
// the list's sum may be too small to be added; share is 0 where there is nothing to do.
struct Stats {
  double m, S, base, others, Q, top, share;
};
static_assert(sizeof(Stats) == STATS * sizeof(double), "the layout of out_stats");
__device__ __forceinline__ void write_row(const Params& p, int row, float loss, int status, const Stats& st) {
  if (threadIdx.x) return;
  p.out_loss[row] = loss;
  p.out_status[row] = status;
  if (p.out_stats) reinterpret_cast<Stats*>(p.out_stats)[row] = st;
}

// A thread's first entry of a list: read ahead of the pass over the row, whose loads hide its own.
struct Entry {
  int64_t id;
  float x, lq;
};
template <typename T>
__device__ __forceinline__ Entry entry_of(const Params& p, int row, int k) {
  Entry e{-1, -INFINITY, 0.f};
  if (k < p.K) {
    e.id = p.ids[(int64_t)row * p.K + k];
    e.lq = p.lq[(int64_t)row * p.K + k];
    if (e.id >= 0 && e.id < p.V) e.x = Elem<T>::one(static_cast<const T*>(p.logits) + (int64_t)row * p.stride + e.id);
  }
  return e;
}

// The sum outside the list again, as 2^((x - m) c) against its own largest logit m, where the pass could not form
// it.  What is above m is the list's; what the list has at or below m is added as the row's, and the very same
// terms are taken off again in fp64.  Only rows whose rest is all beyond FAR are read twice (finite masks: 331 bf16 rows of
// 129280 in 58 us instead of 26); slices of masks beside others add nothing and cost nothing.
template <typename T>
__device__ __forceinline__ double sum_again(const Params& p, int row, float m, const Entry& mine, double* red) {
  constexpr int VEC = Elem<T>::VEC, AHEAD = 4;
  const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.stride;
  const auto term = [&](float v) -> double {
    const float d = v - m;
    return v > m ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(d, p.sc.c_lo, d * p.sc.c));
  };
  double sum[1] = {0.0};
  for (int base = 0; base <= p.V / VEC; base += AHEAD * NT) {
    uint32_t w[AHEAD][4];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) rows::load_some<false>(x, 0, p.V, base + u * NT + (int)threadIdx.x, w[u]);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      float v[VEC];
      Elem<T>::unpack(w[u], v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[0] += term(v[j]);
    }
  }
  if (mine.id >= 0) sum[0] -= term(mine.x);
  for (int k = threadIdx.x + NT; k < p.K; k += NT) {
    const Entry e = entry_of<T>(p, row, k);
    if (e.id >= 0) sum[0] -= term(e.x);
  }
  rows::block_sums(sum, red);
  return sum[0];
}

// The row's divergence from the sums outside its list and the list itself.
template <typename T>
__device__ __forceinline__ void finish(const Params& p, int row, State st, int flags, const Entry& mine, double* red) {
  if (!(flags & LIVE)) {
    write_row(p, row, 0.f, 0, Stats{0.0, 1.0, 0.0, 0.0, 0.0, 0.0, 0.0});
    return;
  }
  if (flags != LIVE) {
    write_row(p, row, NAN, flags & ~LIVE, Stats{NAN, NAN, NAN, NAN, NAN, 0.0, 1.0});
    return;
  }
  // (a list of more than NT entries is read again here; the first entries stay in registers, and the
  // code for them apart, which the constants of a loop would push into memory)
  float mf = st.m, top = -INFINITY;
  int bad = 0;
  const auto meet = [&](const Entry& e) {
    if (e.id < 0) return;
    mf = fmaxf(mf, e.x);
    top = fmaxf(top, e.lq);
    bad |= !(e.lq < INFINITY);
  };
  meet(mine);
  for (int k = threadIdx.x + NT; k < p.K; k += NT) meet(entry_of<T>(p, row, k));
  const double m = rows::block_max(mf, red);
  if (st.U != 0.0) {
    // the sum is needed where the rest is asked for or not negligible, and to find a NaN among positive logits, whose
    // sum of the pass may be one by itself
    const double d = ((double)st.m - m) * p.sc.cd;
    if (p.rest || !(d < -2000.0) || st.m > 0.f)
      st.S = sum_again<T>(p, row, st.m, mine, red);
    else
      st.S = st.S == st.S ? 0.0 : st.S;
  }
  top = p.rest ? 0.f : rows::block_max(top, red);
  bad = __syncthreads_or(bad || !(top > -INFINITY));
  double sum[4] = {0.0, 0.0, 0.0, 0.0};
  const auto add = [&](const Entry& e) {
    if (e.id < 0) return;
    const double d = ((double)e.x - m) * p.sc.inv_t, l = (double)e.lq - top, w = exp(l);
    sum[0] += exp(d);
    if (w > 0.0) {
      sum[1] += w;
      sum[2] += w * l;
      sum[3] += w * d;
    }
  };
  if (!bad) {
    add(mine);
    for (int k = threadIdx.x + NT; k < p.K; k += NT) add(entry_of<T>(p, row, k));
  }
  rows::block_sums(sum, red);
  if (threadIdx.x >= 64) return;  // (one thread writes)
  const double Sn = sum[0], W = sum[1], WL = sum[2], WD = sum[3];
  // S_rest against m, by `down` from the sum against its own largest logit
  const double down = st.S != 0.0 ? exp2(fmax(((double)st.m - m) * p.sc.cd, -2000.0)) : 0.0;
  const double S_rest = st.S * down, S = S_rest + Sn, ln_s = log(S);
  const bool nonfinite = !(S > 0.0 && S < INFINITY);
  if (bad || (p.rest && W > MOST_MASS)) {
    write_row(p, row, NAN, DSV41_STATUS_BAD_TEACHER, Stats{NAN, NAN, NAN, NAN, NAN, 0.0, 1.0});
    return;
  }
  double loss, rest = 0.0, Q = 1.0, share = 1.0;
  if (p.rest) {
    rest = 1.0 - W;
    if (rest < REST_FLOOR) rest = 0.0;
    // (the sum against its own largest logit, whose distance from m counts in full, also where fp64 does not
    // hold the mass; a NaN is none above 0, and makes S one)
    const bool masked = !(st.S > 0.0) || ((double)st.m == (double)lowest<T>() && m > (double)st.m);
    const double log_rest = masked ? -(double)INFINITY : log(st.S) + ((double)st.m - m) * p.sc.inv_t - ln_s;
    loss = WL - WD + W * ln_s + (rest > 0.0 ? rest * (log(rest) - log_rest) : 0.0);
    Q = W + rest;
  } else {
    share = 1.0 / W;
    loss = (WL - WD) / W - log(W) + ln_s;
  }
  const float l = nonfinite ? NAN : (float)loss;
  Stats out{m, nonfinite ? (double)NAN : S, m, 0.0, Q, top, share};
  if (st.S != 0.0) {
    out.base = st.m;
    out.others = Q * down / S - (rest > 0.0 ? rest / st.S : 0.0);
  }
  write_row(p, row, l, nonfinite || !isfinite(l) ? DSV41_STATUS_NONFINITE : 0, out);
}

template <typename T, bool ONCE>
__global__ __launch_bounds__(NT, 8) void distill_kernel(Params p) {
  __shared__ Shared s;
  const int row = blockIdx.x / p.slices, slice = blockIdx.x % p.slices, tid = threadIdx.x;
  const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.stride;
  const int skew = rows::skew_of(x + slice * p.len), begin = slice * p.len - skew, len = min(p.len, p.V - slice * p.len) + skew;
  Entry mine;
  int flags;
  const auto before = [&](float&, int&) {
    mine = entry_of<T>(p, row, tid);
    for (int i = 4 * tid; i < (len + 31) / 32; i += 4 * NT) *reinterpret_cast<uint4*>(s.named + i) = make_uint4(0, 0, 0, 0);
    if (tid == 0) s.flags = 0;
    __syncthreads();
    int f = 0;
    for (int k = tid; k < p.K; k += NT) {
      const int64_t id = k < NT ? mine.id : p.ids[(int64_t)row * p.K + k];
      if (id < 0) continue;
      f |= LIVE;
      if (id >= p.V) f |= DSV41_STATUS_BAD_TARGET;
      if (id >= begin + skew && id < begin + len) {
        const uint32_t i = (uint32_t)(id - begin), bit = 1u << (i & 31);
        if (atomicOr(&s.named[i >> 5], bit) & bit) f |= DSV41_STATUS_REPEATED;
      }
    }
    if (f) atomicOr(&s.flags, f);
    __syncthreads();
    flags = s.flags;
    return flags == LIVE;
  };
  const State st = rows::scan<T, ONCE, false, true>(
      x + begin, skew, len, p.sc, nullptr, s.named, s.red, before, [](const float(&)[4]) {}, [](float) {});
  if (p.slices == 1) {
    finish<T>(p, row, st, flags, mine, s.red);
  } else if (tid == 0) {
    SliceState* o = p.states + (int64_t)row * p.slices + slice;
    o->s = st;
    o->flags = flags;
  }
}

template <typename T>
__global__ __launch_bounds__(NT) void distill_join_kernel(Params p) {
  __shared__ double red[4 * WAVES];
  __shared__ int flags;
  const int row = blockIdx.x, tid = threadIdx.x;
  const Entry mine = entry_of<T>(p, row, tid);
  SliceState in{{0.0, 0.0, -INFINITY, 0}, 0, 0};
  if (tid == 0) flags = 0;
  __syncthreads();
  if (tid < p.slices) in = p.states[(int64_t)row * p.slices + tid];
  if (in.flags) atomicOr(&flags, in.flags);
  State st = in.s;
  const float m = rows::block_max(st.m, red);
  // a slice whose sum was not formed adds nothing far below the others; else it is the row's that is formed again
  const double d = ((double)st.m - (double)m) * p.sc.cd;
  const bool far = st.U != 0.0;
  if (far)
    st.S = st.S == st.S ? 0.0 : st.S;
  else if (st.S != 0.0)
    rows::rebase(st.S, st.U, d);
  double sum[2] = {st.S, far && !(d < -2000.0) ? 1.0 : 0.0};
  rows::block_sums(sum, red);
  finish<T>(p, row, State{sum[0], sum[1], m, 0}, flags, mine, red);
}

struct GradParams {
  const void* logits;
  int64_t stride;
  const int64_t* ids;
  const float* lq;
  int rows, V, K, slices, len;
  Scale sc;
  const double* stats;
  const float* g;
  void* out;  // [rows, V], rows V apart
};

// One read and one write of the row; then the list's tokens are written again, with values that the threads
// form first, while the other waves already read.  Rows whose list is empty or whose gradient is zero are
// zeros and are not read.
template <typename T>
__global__ __launch_bounds__(NT) void distill_grad_kernel(GradParams p) {
  const int row = p.rows - 1 - (int)(blockIdx.x / p.slices), slice = blockIdx.x % p.slices;
  const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.stride;
  const int begin = slice * p.len, len = min(p.len, p.V - begin);
  T* out = static_cast<T*>(p.out) + (int64_t)row * p.V + begin;
  const Stats st = reinterpret_cast<const Stats*>(p.stats)[row];
  const double g = (double)p.g[row] * p.sc.inv_t;
  if (g == 0.0 || st.share == 0.0) {
    rows::fill_zero(out, len);
    return;
  }
  // entry k's place in the slice (below 0: none of this slice's) and gradient
  const auto entry = [&](int k, float& v) {
    const int64_t id = p.ids[(int64_t)row * p.K + k], i = id - begin;
    if (id < 0 || i < 0 || i >= len) return -1;
    const double e = exp(((double)Elem<T>::one(x + id) - st.m) * p.sc.inv_t);
    v = (float)(g * (st.Q * e / st.S - st.share * exp((double)p.lq[(int64_t)row * p.K + k] - st.top)));
    return (int)i;
  };
  __shared__ rows::Again again;
  const int tid = threadIdx.x;
  again.at[tid] = tid < p.K ? entry(tid, again.v[tid]) : -1;
  const rows::Lift lift(g * st.others);
  const float base = (float)st.base, A = (float)(g * st.others * lift.down);
  // (a row whose sums are NaN has NaN for S: its gradient is, too)
  const float bad = st.S == st.S ? 0.f : NAN;
  rows::map(x + begin, out, len, [&](float v) { return __builtin_fmaf(A, lift.exp2(v - base, p.sc.c), bad); });
  rows::own_stores_in_order();
  rows::lds_barrier();
  rows::store_again(again, min(p.K, NT), x + begin, out, len);
  for (int k = NT; k < p.K; k += NT) {
    rows::lds_barrier();
    again.at[tid] = k + tid < p.K ? entry(k + tid, again.v[tid]) : -1;
    rows::lds_barrier();
    rows::store_again(again, min(p.K - k, NT), x + begin, out, len);
  }
}

template <typename T>
void launch(const Params& p, hipStream_t s) {
  const dim3 grid((unsigned)p.rows * (unsigned)p.slices);
  if (rows::read_once(p.rows, p.V, sizeof(T)))
    hipLaunchKernelGGL((distill_kernel<T, true>), grid, dim3(NT), 0, s, p);
  else
    hipLaunchKernelGGL((distill_kernel<T, false>), grid, dim3(NT), 0, s, p);
  if (p.slices > 1) hipLaunchKernelGGL(distill_join_kernel<T>, dim3(p.rows), dim3(NT), 0, s, p);
}

Cut cut_of(int rows, int V, int esize) { return rows::cut_rows(rows, V, 0, esize, 6144, MAX_LEN); }
int esize_of(const dsv41_distill_desc* d) { return d->logits_dtype == DSV41_DTYPE_F32 ? 4 : 2; }

int check_desc(const dsv41_distill_desc* d) {
  if (!d) return fail(DSV41_E_INVALID, "distillation descriptor is NULL");
  if (d->struct_size != sizeof(dsv41_distill_desc))
    return fail(DSV41_E_ABI, "dsv41_distill_desc size mismatch (rebuild the binding)");
  if (int rc = rows::check_rows(d->rows, d->vocab, d->logits_dtype, d->logits_row_stride, d->logits, d->temperature)) return rc;
  if (d->top_k <= 0) return fail(DSV41_E_INVALID, "teacher lists must have at least one entry");
  if (!d->teacher_ids || !d->teacher_logprob) return fail(DSV41_E_INVALID, "teacher_ids and teacher_logprob are required");
  if (d->tail != DSV41_TAIL_RENORMALIZE && d->tail != DSV41_TAIL_REST)
    return fail(DSV41_E_INVALID, "tail must be DSV41_TAIL_RENORMALIZE or DSV41_TAIL_REST");
  if (!d->out_loss || !d->out_status) return fail(DSV41_E_INVALID, "out_loss and out_status are required");
  return rows::check_grid(d->rows, cut_of(d->rows, d->vocab, esize_of(d)));
}

size_t workspace_of(int rows, const Cut& c) { return c.slices == 1 ? 0 : (size_t)rows * c.slices * sizeof(SliceState); }

}  // namespace distill
}  // namespace dsv41

using namespace dsv41;

extern "C" size_t dsv41_distill_workspace_bytes(const dsv41_distill_desc* d) {
  if (distill::check_desc(d)) return 0;
  return distill::workspace_of(d->rows, distill::cut_of(d->rows, d->vocab, distill::esize_of(d)));
}

extern "C" int dsv41_distill_run(const dsv41_distill_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = distill::check_desc(d)) return rc;
  const rows::Cut c = distill::cut_of(d->rows, d->vocab, distill::esize_of(d));
  const size_t need = distill::workspace_of(d->rows, c);
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 8))
    return fail(DSV41_E_WORKSPACE, "distillation workspace is missing, too small or not 8-byte aligned");
  distill::Params p{};
  p.logits = d->logits;
  p.stride = d->logits_row_stride;
  p.ids = d->teacher_ids;
  p.lq = d->teacher_logprob;
  p.rows = d->rows;
  p.V = d->vocab;
  p.K = d->top_k;
  p.slices = c.slices;
  p.len = c.len;
  p.rest = d->tail == DSV41_TAIL_REST;
  p.sc = rows::scale_of(d->temperature, true);
  p.out_loss = d->out_loss;
  p.out_status = d->out_status;
  p.out_stats = d->out_stats;
  p.states = static_cast<distill::SliceState*>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (d->logits_dtype == DSV41_DTYPE_F32)
    distill::launch<float>(p, s);
  else
    distill::launch<rows::bf16_t>(p, s);
  DSV41_HIP_CHECK(hipGetLastError());
  return DSV41_OK;
}

extern "C" int dsv41_distill_grad_run(const dsv41_distill_grad_desc* d, void* stream) {
  if (!d) return fail(DSV41_E_INVALID, "distillation gradient descriptor is NULL");
  if (d->struct_size != sizeof(dsv41_distill_grad_desc))
    return fail(DSV41_E_ABI, "dsv41_distill_grad_desc size mismatch (rebuild the binding)");
  if (int rc = rows::check_rows(d->rows, d->vocab, d->logits_dtype, d->logits_row_stride, d->logits, d->temperature))
    return rc;
  if (d->top_k <= 0 || !d->teacher_ids || !d->teacher_logprob || !d->stats || !d->grad_loss || !d->out)
    return fail(DSV41_E_INVALID, "teacher_ids, teacher_logprob, stats, grad_loss and out are required");
  if ((uintptr_t)d->out % (d->logits_dtype == DSV41_DTYPE_F32 ? 4 : 2))
    return fail(DSV41_E_INVALID, "out is not aligned to its type");
  const rows::Cut c = rows::grad_cut(d->rows, d->vocab, d->logits_dtype == DSV41_DTYPE_F32 ? 4 : 2);
  if (int rc = rows::check_grid(d->rows, c)) return rc;
  distill::GradParams p{};
  p.logits = d->logits;
  p.stride = d->logits_row_stride;
  p.ids = d->teacher_ids;
  p.lq = d->teacher_logprob;
  p.rows = d->rows;
  p.V = d->vocab;
  p.K = d->top_k;
  p.slices = c.slices;
  p.len = c.len;
  p.sc = rows::scale_of(d->temperature, false);
  p.stats = d->stats;
  p.g = d->grad_loss;
  p.out = d->out;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)p.rows * (unsigned)p.slices), block(rows::NT);
  if (d->logits_dtype == DSV41_DTYPE_F32)
    hipLaunchKernelGGL(distill::distill_grad_kernel<float>, grid, block, 0, s, p);
  else
    hipLaunchKernelGGL(distill::distill_grad_kernel<rows::bf16_t>, grid, block, 0, s, p);
  DSV41_HIP_CHECK(hipGetLastError());
  return DSV41_OK;
}
