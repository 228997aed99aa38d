// row_scan.h — what the kernels over rows of logits share (scores.hip, distill.hip): 16-byte loads of
// rows of any alignment, the pass over a row (or a slice of it) with its running softmax sums, and
// sums over a workgroup.
//
// Sums.  With c = log2(e) / T and a reference that a thread raises when it meets a larger logit, a pass
// keeps sums of exponentials in fp32 over the thread's few hundred elements; the threads' sums are
// brought to the largest logit and added in fp64.
//   For scores, S = sum 2^d and U = sum 2^d d with d = (x - r) c.  The difference is what lets a certain token
// score 0: its term is 1 and S is 1, whatever its logit.  Beside a likely token's 1 a thread's two sums, of n / 1024
// elements each in a row or slice of n, keep the other terms to half a step of 1, so S, and S - 1 with it, is off
// by n / 1024 times 2^-24 at most: 9e-6 for an uncut row of 151936.  (One token 18 nats above all the others, at
// -2.3e-3: 2.2e-6.  Sums that are emptied into fp64 ones every two steps have a tenth of that, and cost bf16
// passes 3 to 4%: 4096 rows 210 us instead of 203.)  c is rounded to fp32, which puts the same relative error
// into every exponent; to first order it is made up for by kappa U, kappa = ln 2 (c - fp32(c)) / fp32(c), which
// S takes in the end.
//   For the mass outside a list, S = sum 2^(x c - r) alone: c as a sum of two and one multiply-add for
// each, so there is nothing to make up for.  r is a rounded x c, and what is left of x c - r for that x itself
// is up to half a step of r and what the second part of c adds: powers of two that the sums bear up to |r| =
// FAR, and not beyond.  So r begins at -FAR: what lies further down, a mask of any finite size, adds
// nothing.  Where the largest x c is not within FAR, U says so, and S is no sum; below it, S is still NaN for a NaN.
//   x = -inf is a masked token: it adds nothing to any sum.  A NaN or +inf makes S NaN.
#pragma once

#include <math.h>
#include <stdint.h>

#include "common.h"

namespace dsv41 {
namespace rows {

constexpr int NT = 512;       // threads of a workgroup
constexpr int WAVES = NT / 64;
constexpr int GROUP = 32;     // elements whose maximum the top-k selection keeps
constexpr float LOWEST = -3.402823466e38f;

struct bf16_t {
  uint16_t v;
};

// 16 bytes of a row; rows begin at any element, so the loads assume the element's alignment only
// (global_load_dwordx4 takes any).
template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int VEC = 4;
  typedef uint32_t Raw __attribute__((ext_vector_type(4), aligned(4)));
  static constexpr uint32_t MASKED = 0xFF800000u;  // -inf
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ void put(uint32_t (&w)[4], int j, float v) { w[j] = __float_as_uint(v); }
  static __device__ __forceinline__ void unpack(const uint32_t (&w)[4], float (&x)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(w[j]);
  }
};
template <>
struct Elem<bf16_t> {
  static constexpr int VEC = 8;
  typedef uint32_t Raw __attribute__((ext_vector_type(4), aligned(2)));
  static constexpr uint32_t MASKED = 0xFF80FF80u;  // twice -inf
  static __device__ __forceinline__ float one(const bf16_t* p) { return bf16_to_f32(p->v); }
  static __device__ __forceinline__ void put(uint32_t (&w)[4], int j, bf16_t v) {
    w[j >> 1] = j & 1 ? (w[j >> 1] & 0xFFFFu) | (uint32_t)v.v << 16 : (w[j >> 1] & 0xFFFF0000u) | v.v;
  }
  static __device__ __forceinline__ void unpack(const uint32_t (&w)[4], float (&x)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = bf16_lo(w[j]);
      x[2 * j + 1] = bf16_hi(w[j]);
    }
  }
};

// 16 bytes at p.  ONCE: nontemporal, for rows that are read once and do not stay in a cache.
template <bool ONCE, typename T>
__device__ __forceinline__ void load16(const T* p, uint32_t (&w)[4]) {
  using Raw = typename Elem<T>::Raw;
  Raw r;
  if constexpr (ONCE)
    r = __builtin_nontemporal_load(reinterpret_cast<const Raw*>(p));
  else
    r = *reinterpret_cast<const Raw*>(p);
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = r[j];
}
// Elements between the memory line (128 bytes) that holds *x and x.  A pass counts its 16 bytes from the line's
// begin, and takes the elements before x for masked ones: 4096 bf16 rows of an odd vocabulary, which begin
// at odd elements, in 205 us instead of 265, fp32 ones in 378 instead of 415.
constexpr int MOST_SKEW = 64;
template <typename T>
__device__ __forceinline__ int skew_of(const T* x) {
  return (int)((uintptr_t)x % 128 / sizeof(T));
}
// The elements [i VEC, i VEC + VEC) of x[from, len) as 16 bytes, -inf where they lie outside; i < 0: none.
template <bool ONCE, typename T>
__device__ __forceinline__ void load_some(const T* x, int from, int len, int i, uint32_t (&w)[4]) {
  constexpr int VEC = Elem<T>::VEC;
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = Elem<T>::MASKED;
  if (i * VEC >= from && i >= 0 && i < len / VEC) {
    load16<ONCE>(x + (int64_t)i * VEC, w);
  } else if (i >= 0 && i <= len / VEC) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int at = i * VEC + j;
      if (at >= from && at < len) Elem<T>::put(w, j, x[at]);
    }
  }
}
template <bool ONCE = false, typename T>
__device__ __forceinline__ void load_full(const T* x, int i, float (&v)[Elem<T>::VEC]) {
  uint32_t w[4];
  load16<ONCE>(x + (int64_t)i * Elem<T>::VEC, w);
  Elem<T>::unpack(w, v);
}

// ---- a row written: out[0, len) = f(x[0, len)), or zeros.  Ordinary stores: nontemporal ones are no faster (331 bf16
// rows of distillation's gradient 28.9 us with either, 1000 fp32 rows 225 instead of 202, 4096 bf16 rows 408 instead
// of 406), and what reads the gradient next finds it in no cache (with a multiplication in place behind it 58 us
// instead of 54, 412 instead of 398, and 817 instead of 825).
__device__ __forceinline__ void store_one(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_one(bf16_t* p, float v) { p->v = (uint16_t)pack_bf16(v, 0.f); }
__device__ __forceinline__ void store_full(float* out, int i, const float (&v)[4]) {
  Elem<float>::Raw r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = __float_as_uint(v[j]);
  *reinterpret_cast<Elem<float>::Raw*>(out + (int64_t)i * 4) = r;
}
__device__ __forceinline__ void store_full(bf16_t* out, int i, const float (&v)[8]) {
  Elem<bf16_t>::Raw r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
  *reinterpret_cast<Elem<bf16_t>::Raw*>(out + (int64_t)i * 8) = r;
}
// A factor times 2^(d c), d c <= 0.  v_exp_f32 returns zero below 2^-126, where fp32 and bf16 still hold
// values; a factor that brings such a power back above them gives 2^32 of its size to the exponent.
struct Lift {
  float up, down;  // what the exponent takes, and 2^-up
  __device__ __forceinline__ explicit Lift(double factor) {
    const bool large = fabs(factor) >= 0x1p-60;
    up = large ? 32.f : 0.f;
    down = large ? 0x1p-32f : 1.f;
  }
  __device__ __forceinline__ float exp2(float d, float c) const { return __builtin_amdgcn_exp2f(__builtin_fmaf(d, c, up)); }
};
// U chunks a thread from `base` on, the loads of all of them in flight; of the last U only `rest` threads'.
template <int U, typename T, class F>
__device__ __forceinline__ void map_some(const T* x, T* out, int base, int rest, F f) {
  constexpr int VEC = Elem<T>::VEC;
  const int tid = threadIdx.x;
  float v[U][VEC];
#pragma unroll
  for (int u = 0; u < U; ++u) load_full(x, base + u * NT + (u + 1 < U ? tid : min(tid, rest - 1)), v[u]);
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[u][j] = f(v[u][j]);
    if (u + 1 < U || tid < rest) store_full(out, base + u * NT + tid, v[u]);
  }
}
// Elements before the first that 16-byte loads take: one of a row of 2-byte elements that begins between two words.
// (4096 such rows of distillation's gradient 426 us instead of 469.)
template <typename T>
__device__ __forceinline__ int odd_of(const T* x) {
  return (uintptr_t)x % 4 != 0;
}
template <typename T, class F>
__device__ __forceinline__ void map(const T* x, T* out, int len, F f) {
  constexpr int VEC = Elem<T>::VEC, U = 4;
  const int tid = threadIdx.x, odd = odd_of(x);
  if (odd && tid == 0) store_one(out, f(Elem<T>::one(x)));
  x += odd, out += odd, len -= odd;
  const int full = len / VEC;
  int base = 0;
  for (; base + U * NT <= full; base += U * NT) map_some<U>(x, out, base, NT, f);
  const int left = full - base;
  if (left > 3 * NT) map_some<4>(x, out, base, left - 3 * NT, f);
  else if (left > 2 * NT) map_some<3>(x, out, base, left - 2 * NT, f);
  else if (left > NT) map_some<2>(x, out, base, left - NT, f);
  else if (left > 0) map_some<1>(x, out, base, left, f);
  for (int i = full * VEC + tid; i < len; i += NT) store_one(out + i, f(Elem<T>::one(x + i)));
}
// Some elements of a row that `map` wrote are written again, by the wave that wrote them: its stores to one
// address stay in order, so no wave waits for those of the others, nor for its own, which a barrier of
// all memory would have it do.  `wrote` says whether element i of out[0, len) is this wave's.
template <typename T>
__device__ __forceinline__ bool wrote(const T* x, int i, int len) {
  constexpr int VEC = Elem<T>::VEC;
  i -= odd_of(x), len -= odd_of(x);
  const int at = i >= 0 && i < len / VEC * VEC ? i / VEC % NT : 0;  // (those beside the chunks are the first wave's)
  return at >> 6 == (int)threadIdx.x >> 6;
}
__device__ __forceinline__ void own_stores_in_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
// A barrier for what the threads wrote to LDS, with stores to memory left in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
// Values for the elements at[k] (below 0: none) of out[0, len), k < n: a thread's entry is formed before the row
// is mapped, then each wave stores those of its own elements.
struct Again {
  int at[NT];
  float v[NT];
};
template <typename T>
__device__ __forceinline__ void store_again(const Again& a, int n, const T* x, T* out, int len) {
  for (int k = (int)threadIdx.x & 63; k < n; k += 64) {
    const int i = a.at[k];
    if (i >= 0 && wrote(x, i, len)) store_one(out + i, a.v[k]);
  }
}
template <typename T>
__device__ __forceinline__ void fill_zero(T* out, int len) {
  constexpr int VEC = Elem<T>::VEC;
  const int full = len / VEC;
  const float zero[VEC] = {};
  for (int i = threadIdx.x; i < full; i += NT) store_full(out, i, zero);
  for (int i = full * VEC + (int)threadIdx.x; i < len; i += NT) store_one(out + i, 0.f);
}

// ---- sums and maxima over the workgroup, the same value in every thread, in scalar registers.  `s`: LDS,
// WAVES values for each value that is joined.  Eight lanes take the waves' values of each.
static_assert(WAVES == 8, "a lane for every wave's value");
template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xF, 0xF, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lane_d(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// FRESH: `s` has not been read since the last barrier, so none is needed before it is written.
template <bool FRESH = false, int N>
__device__ __forceinline__ void block_sums(double (&v)[N], double* s) {
  static_assert(N <= 8, "a lane for every value");
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_total_d(v[i]);
  if (!FRESH) __syncthreads();
  const int lane = threadIdx.x & 63;
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) s[i * WAVES + (threadIdx.x >> 6)] = v[i];
  __syncthreads();
  double a = lane < N * WAVES ? s[lane] : 0.0;
  a += dpp_d<0xB1>(a);   // quad_perm [1,0,3,2]
  a += dpp_d<0x4E>(a);   // quad_perm [2,3,0,1]
  a += dpp_d<0x141>(a);  // row_half_mirror
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lane_d(a, 8 * i);
}
template <bool FRESH = false>
__device__ __forceinline__ float block_max(float v, double* s) {
  v = wave_max_dpp(v);
  if (!FRESH) __syncthreads();
  const int lane = threadIdx.x & 63;
  if (lane == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  const float w = wave_max_dpp((float)s[lane & (WAVES - 1)]);
  return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(w)));
}

// The scale of a temperature, computed on the host.
struct Scale {
  float c, c_lo;  // log2(e) / T in fp32, or as a sum of two
  float margin;   // how far a logit may exceed the reference: two powers of two
  double cd;      // what c and c_lo say
  double inv_t;   // 1 / T
  double kappa;   // ln 2 (log2(e) / T - cd) / cd
};
inline Scale scale_of(float temperature, bool split) {
  Scale s;
  const double c = 1.4426950408889634 / (double)temperature;
  s.c = (float)c;
  s.c_lo = 0.f;
  if (split) {
    // c_lo above zero, so that -inf stays -inf in both products
    while ((double)s.c >= c || (float)(c - (double)s.c) == 0.f) s.c = nextafterf(s.c, 0.f);
    s.c_lo = (float)(c - (double)s.c);
  }
  s.cd = (double)s.c + (double)s.c_lo;
  s.margin = (float)(2.0 / c);
  s.inv_t = 1.0 / (double)temperature;
  s.kappa = 0.6931471805599453 * (c - s.cd) / s.cd;
  return s;
}
// Temperatures whose c or c_lo leave fp32's range are refused.
inline bool scale_ok(float temperature) { return temperature >= 1e-30f && temperature <= 1e30f; }

// What a slice of a row (or the whole row) adds up to: its largest logit, S and U against it (outside a list, U
// whether m c is beyond FAR), and how many of its elements come before the target in (logit desc, index asc).
struct State {
  double S, U;
  float m;
  int32_t before;
};
// S and U from one reference to another, d = the first less the second as an exponent.
__device__ __forceinline__ void rebase(double& S, double& U, double d) {
  d = fmax(d, -2000.0);
  const double f = exp2(d);
  U = f * (U + d * S);
  S = f * S;
}

// Largest of a chunk.  v_max3_f32 by itself: fmaxf would first quiet each operand.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float m;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(a), "v"(b), "v"(c));
  return m;
}
__device__ __forceinline__ float max_of(const float (&x)[4]) {
  const float m = max3(x[0], x[1], x[2]);
  return max3(m, x[3], x[3]);
}
__device__ __forceinline__ float max_of(const float (&x)[8]) {
  const float a = max3(x[0], x[1], x[2]), b = max3(x[3], x[4], x[5]);
  return max3(max3(a, x[6], x[7]), b, b);
}

// Two chunk maxima become the maxima of their groups of LANES lanes (8 or 4), in every lane of them.  A
// DPP read needs two wait states after the instruction that wrote its register.
template <int LANES>
__device__ __forceinline__ void group_max2(float& g, float& h) {
#define DSV41_DPP2(ctrl)                                                                        \
  "s_nop 0\n\t"                                                                                 \
  "v_max_f32_dpp %0, %0, %0 " ctrl " row_mask:0xf bank_mask:0xf bound_ctrl:1\n\t"               \
  "v_max_f32_dpp %1, %1, %1 " ctrl " row_mask:0xf bank_mask:0xf bound_ctrl:1\n\t"
  asm("s_nop 1\n\t" DSV41_DPP2("quad_perm:[1,0,3,2]") DSV41_DPP2("quad_perm:[2,3,0,1]") "s_nop 1" : "+v"(g), "+v"(h));
  if constexpr (LANES == 8) asm("s_nop 1\n\t" DSV41_DPP2("row_half_mirror") "s_nop 1" : "+v"(g), "+v"(h));
#undef DSV41_DPP2
}

// The largest number below x that is not equal to it (-0 equals +0); NaN, which no number is at most,
// below -inf.
__device__ __forceinline__ float next_below(float x) {
  const uint32_t b = __float_as_uint(x);
  if (x == 0.f) return __uint_as_float(0x80000001u);
  return __uint_as_float(x > 0.f ? b - 1u : b + 1u);
}

// The largest |r| that x c - r is formed with.  At 2^24, half a step is 1, and the second part of c, at most a step
// of the first, adds 2: exponents up to 5, with the 2 that a logit may exceed its reference by.
constexpr float FAR = 0x1p24f;

// One pass over x[from, len) by the workgroup, whose threads take 16 bytes in turn; x is a line's begin, and
// from below MOST_SKEW.
//   TOP: group_max[g] = the largest of the elements [32 g, 32 g + 32).
//   NAMED: the sum outside a list: elements whose bit in `named` (from x on) is set count as masked.
//   before(xt, t): called once, with the first loads in flight; it may use barriers, gives the target's
//     logit (+inf: no target) and index, from x on, and says whether there is a pass to make.
//   met(own): called with the largest elements of the thread's four shares, before a barrier; found(m)
//     with the largest of all, behind it and before the last one.
//   red: LDS of 4 WAVES values that nothing else uses in the meantime.
template <typename T, bool ONCE, bool TOP, bool NAMED, class Before, class Met, class Found>
__device__ __forceinline__ State scan(const T* x, int from, int len, const Scale& sc, float* group_max, const uint32_t* named,
                                      double* red, Before before, Met met, Found found) {
  constexpr int VEC = Elem<T>::VEC, LANES = GROUP / VEC;
  const int full = len / VEC, n = (len + VEC - 1) / VEC;
  const int tid = threadIdx.x;
  float own[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  float r = NAMED ? -FAR : LOWEST, S[2] = {0.f, 0.f}, Us[2] = {0.f, 0.f}, margin = NAMED ? 2.f : sc.margin;
  asm("" : "+v"(margin));  // (a scalar register short, the compiler would load it in every step)
  int ahead = 0, t = 0;  // (ahead: the wave's count)
  float xt = INFINITY;

  int target_chunk = 0;
  float below = INFINITY;
  using Tile = uint32_t[2][4];  // two chunks a thread
  constexpr int STEP = 2 * NT;
  auto load = [&](Tile& w, int base) {
#pragma unroll
    for (int u = 0; u < 2; ++u) load16<ONCE>(x + (int64_t)(base + u * NT + tid) * VEC, w[u]);
  };
  auto take = [&](const Tile& w, int base, float& own0, float& own1) {
    float v[2][VEC], cm[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      Elem<T>::unpack(w[u], v[u]);
      if constexpr (NAMED) {
        const int i = base + u * NT + tid;
        const uint32_t bits = i < n ? (named[(i * VEC) >> 5] >> ((i * VEC) & 31)) & ((1u << VEC) - 1u) : 0u;
        if (bits) {
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if (bits >> j & 1) v[u][j] = -INFINITY;
        }
      }
      cm[u] = max_of(v[u]);
    }
    own0 = fmaxf(own0, cm[0]);
    own1 = fmaxf(own1, cm[1]);
    const float tm = max3(cm[0], cm[1], cm[1]);
    // elements before the target: those above its logit, and in chunks before its own also the equal
    // ones, which are above the next smaller number
    if (!NAMED && __ballot(tm >= xt)) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float at_most = base + u * NT + tid < target_chunk ? below : xt;
#pragma unroll
        for (int j = 0; j < VEC; ++j) ahead += __popcll(__ballot(!(v[u][j] <= at_most)));
      }
    }
    if constexpr (TOP) {
      group_max2<LANES>(cm[0], cm[1]);
      if ((tid & (LANES - 1)) == 0) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int i = base + u * NT + tid;
          if (i < n) group_max[i / LANES] = cm[u];
        }
      }
    }
    if constexpr (NAMED) {
      // (the rounded product in both places: r - tm c in one step would bring the sums to another reference than the
      // one that is kept, half a step of it apart)
#pragma clang fp contract(off)
      const float mc = tm * sc.c;
      if (mc > r + margin) {
        const float f = __builtin_amdgcn_exp2f(r - mc);
        S[0] *= f;
        S[1] *= f;
        r = mc;
      }
    } else if (tm > r + margin) {
      const float d = fmaxf((r - tm) * sc.c, -1000.f), f = __builtin_amdgcn_exp2f(d);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        Us[q] = f * (Us[q] + d * S[q]);
        S[q] = f * S[q];
      }
      r = tm;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if constexpr (NAMED) {
          const float d = __builtin_fmaf(v[u][j], sc.c_lo, __builtin_fmaf(v[u][j], sc.c, -r));
          S[j & 1] += __builtin_amdgcn_exp2f(d);
        } else {
          const float d = (v[u][j] - r) * sc.c, e = __builtin_amdgcn_exp2f(d);
          S[j & 1] += e;
          Us[j & 1] = __builtin_fmaf(e, fmaxf(d, -1000.f), Us[j & 1]);
        }
      }
  };
  // the whole steps, each one's loads in flight while the one before it is taken
  Tile a, b;
  const int steps = full / STEP;
  if (steps > 0 && tid * VEC >= from) {
    load(a, 0);
  } else {
#pragma unroll
    for (int u = 0; u < 2; ++u) load_some<ONCE>(x, from, len, u * NT + tid, a[u]);
  }
  if (!before(xt, t)) return State{0.0, 0.0, -INFINITY, 0};
  if constexpr (!NAMED) {
    target_chunk = t < from ? 0 : t < len ? t / VEC : n;  // (behind the slice: all of its chunks, and none past them)
    below = next_below(xt);
    if (t >= from && t < len && xt < INFINITY) {
      const int at = target_chunk * VEC + tid;  // equal ones of the target's own chunk
      ahead += __popcll(__ballot(at >= from && at < t && Elem<T>::one(x + min(max(at, from), t)) == xt));
    }
    // (a masked target's `below` counts all of the chunks before its own, and with them what lies outside the slice)
    if (xt == -INFINITY && tid < 64) ahead -= min(from, target_chunk * VEC) + (t >= len ? n * VEC - len : 0);
  }
  for (int i = 0; i < steps; i += 2) {
    if (i + 1 < steps) load(b, (i + 1) * STEP);
    take(a, i * STEP, own[0], own[1]);
    if (i + 1 == steps) break;
    if (i + 2 < steps) load(a, (i + 2) * STEP);
    take(b, (i + 1) * STEP, own[2], own[3]);
  }
  if (steps * STEP < n) {
    if (steps > 0) {
#pragma unroll
      for (int u = 0; u < 2; ++u) load_some<ONCE>(x, 0, len, steps * STEP + u * NT + tid, a[u]);
    }
    take(a, steps * STEP, own[2], own[3]);
  }

  // to the largest logit of all threads
  State s;
  met(own);
  s.m = block_max<true>(fmaxf(fmaxf(own[0], own[1]), fmaxf(own[2], own[3])), red);
  double sum[3] = {(double)S[0] + S[1], (double)Us[0] + Us[1], (tid & 63) == 0 ? (double)ahead : 0.0};
  if (sum[0] == 0.0) {
    sum[1] = 0.0;  // nothing met: its reference means nothing
  } else {
    // as rebase, with v_exp_f32: off by 2^-23 of the thread's share, and exact for the one that holds m
    const double d = fmax(NAMED ? (double)r - (double)s.m * sc.cd : ((double)r - (double)s.m) * sc.cd, -1000.0);
    const float near = (float)d;
    const double f = (double)__builtin_amdgcn_exp2f(near) * (1.0 + 0.6931471805599453 * (d - (double)near));
    sum[1] = f * (sum[1] + d * sum[0]);
    sum[0] *= f;
  }
  found(s.m);
  block_sums<true>(sum, red + WAVES);
  s.S = sum[0];
  s.U = NAMED ? (fabsf(s.m * sc.c) > FAR && s.m > -INFINITY) : sum[1];
  s.before = (int32_t)sum[2];
  return s;
}

// ---- host: whether a pass reads its rows with nontemporal loads, which leave the caches as they are.
// Entropies alone, fp32 rows of 151936: 4096 rows 371 us, 442 otherwise; 331 rows (201 MB) just written
// 45 and 42, but 43 and 72 behind other work that filled the 256 MB cache with what has to be written
// back.  Pass and gradient in turn, whose second read the caches serve: 600 rows 218 and 239, bf16 124 and
// 132; 100 bf16 rows of 129280 (26 MB) 36 and 32.
inline bool read_once(int rows, int V, int esize) { return (double)rows * V * esize > 64e6; }

// ---- host: how a batch of rows is cut, and what every call checks
struct Cut {
  int slices, len;  // slices a row, of `len` elements (the last one less)
};

// One workgroup of NT threads per slice: HIP's grids stop short of 2^32 threads.
constexpr int64_t MAX_GRID = 1 << 22;

// Rows of a forward are cut where there are too few of them to occupy the GPU, into slices of at least
// `least` elements.  The time of a pass is that of the CU with the most workgroups, in elements: each of
// them its slice, and 10000 + 100 top_k for its latencies and its selection; fp32 slices a fifth more where a
// CU has one workgroup, which does not keep enough loads in flight; and 16000 for the second kernel of rows
// that are cut at all.  Workgroups that do not fit on the GPU together are not made.  Measured on 348
// batches of 16 to 1000 rows of 50000 and 151936, fp32 and bf16, up to 512 alternatives, as GPU time of
// calls in a graph: within 0.9% of the best number of slices on average and 15% at worst; ceil(512 / rows)
// slices are 10% behind on average, 512 / rows 5%.
constexpr int CUS = 256, PER_CU = 4, MAX_SLICES = 64;
inline Cut cut_rows(int rows, int V, int top_k, int esize, int least, int max_len) {
  int64_t best = INT64_MAX;
  int slices = 1;
  for (int s = 1; s <= MAX_SLICES; ++s) {
    if (s > 1 && ((int64_t)rows * s > CUS * PER_CU || s > V / least)) break;
    const int64_t each = ((int64_t)rows * s + CUS - 1) / CUS, len = (V + s - 1) / s;
    const int64_t cost = each * (len + (each == 1 && esize == 4 ? len / 5 : 0) + 10000 + 100 * top_k) + (s > 1 ? 16000 : 0);
    if (cost < best) {
      best = cost;
      slices = s;
    }
  }
  int len = ((V + slices - 1) / slices + GROUP - 1) / GROUP * GROUP;
  if (len > max_len) len = max_len;
  return {(V + len - 1) / len, len};
}

// A gradient writes each element by itself, so its rows are cut freely: into slices of 32 KB, four chunks a
// thread, whose loads are all in flight at once and whose workgroup ends with its stores; and into smaller ones
// for 512 workgroups, of 4096 elements at least.  Distillation, rows of 151936, GPU time of calls in a graph:
// 1000 in fp32 202 us, 240 with 2048 workgroups of any length, 247 uncut, 230 in slices of 16 KB (5632
// elements 206); 4096 in bf16 415, 488 uncut; 48 in bf16 7.6, and 9.9 with 2048 workgroups.
inline Cut grad_cut(int rows, int V, int esize) {
  int64_t want = ((int64_t)V * esize + 32767) / 32768, few = (512 + rows - 1) / rows;
  if (few > V / 4096) few = V / 4096;
  if (want < few) want = few;
  if (want > MAX_GRID / rows) want = MAX_GRID / rows > 1 ? MAX_GRID / rows : 1;
  const int len = (int)(((V + want - 1) / want + GROUP - 1) / GROUP * GROUP);
  return {(V + len - 1) / len, len};
}

inline int check_grid(int rows, const Cut& c) {
  if ((int64_t)rows * c.slices > MAX_GRID) return fail(DSV41_E_UNSUPPORTED, "more than 2^22 row slices are not supported");
  return DSV41_OK;
}

inline int check_rows(int rows, int V, int dtype, int64_t stride, const void* logits, float temperature) {
  if (rows <= 0 || V <= 0) return fail(DSV41_E_INVALID, "logits must have shape [rows, vocabulary_size]");
  if (!logits) return fail(DSV41_E_INVALID, "logits are required");
  if (dtype != DSV41_DTYPE_F32 && dtype != DSV41_DTYPE_BF16) return fail(DSV41_E_INVALID, "logits must be fp32 or bf16");
  if (stride < 0 || (stride != 0 && stride < V)) return fail(DSV41_E_INVALID, "logits row stride is smaller than the vocabulary");
  if ((uintptr_t)logits % (dtype == DSV41_DTYPE_F32 ? 4 : 2)) return fail(DSV41_E_INVALID, "logits are not aligned to their type");
  if (!isfinite(temperature) || !(temperature > 0.f)) return fail(DSV41_E_INVALID, "temperature must be finite and positive");
  if (!scale_ok(temperature)) return fail(DSV41_E_INVALID, "temperature must lie in [1e-30, 1e30]");
  if (V > (1 << 21)) return fail(DSV41_E_UNSUPPORTED, "vocabularies above 2^21 are not supported");
  return DSV41_OK;
}

}  // namespace rows
}  // namespace dsv41
