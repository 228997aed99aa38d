// row_scan.h — what the kernels over rows of logits share (scores.hip, distill.hip): 16-byte loads of
// rows of any alignment, the pass over a row (or a slice of it) with its running softmax sums, and
// sums over a workgroup.
//
// Sums.  With c = log2(e) / T and a reference r that a thread raises when it meets a larger logit, the
// pass keeps
//   S = sum 2^((x - r) c)   and   U = sum 2^((x - r) c) (x - r) c
// in fp32 over the thread's few hundred elements; the threads' sums are brought to the row's maximum
// and added in fp64.  c itself is rounded to fp32, which would put the same relative error into every
// exponent; to first order that is S (1 + kappa U / S) with kappa = ln 2 (c - fp32(c)) / fp32(c), so the
// joined S takes kappa U more.  x = -inf is a masked token: it adds nothing to either sum.  A NaN or
// +inf makes S NaN.
#pragma once

#include <math.h>

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
struct Raw;
template <>
struct __attribute__((packed, aligned(4))) Raw<float> {
  uint32_t w[4];
};
template <>
struct __attribute__((packed, aligned(2))) Raw<bf16_t> {
  uint32_t w[4];
};

template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int VEC = 4;
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ void unpack(const uint32_t (&w)[4], float (&x)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(w[j]);
  }
};
template <>
struct Elem<bf16_t> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float one(const bf16_t* p) { return bf16_to_f32(p->v); }
  static __device__ __forceinline__ void unpack(const uint32_t (&w)[4], float (&x)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = bf16_lo(w[j]);
      x[2 * j + 1] = bf16_hi(w[j]);
    }
  }
};

// The elements [i VEC, i VEC + VEC) of x[0, len), -inf where they lie outside.
template <typename T>
__device__ __forceinline__ void load_edge(const T* x, int len, int i, float (&v)[Elem<T>::VEC]) {
  constexpr int VEC = Elem<T>::VEC;
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const int64_t at = (int64_t)i * VEC + j;
    v[j] = at < len ? Elem<T>::one(x + at) : -INFINITY;
  }
}
template <typename T>
__device__ __forceinline__ void load_full(const T* x, int i, float (&v)[Elem<T>::VEC]) {
  const Raw<T> r = *reinterpret_cast<const Raw<T>*>(x + (int64_t)i * Elem<T>::VEC);
  const uint32_t w[4] = {r.w[0], r.w[1], r.w[2], r.w[3]};
  Elem<T>::unpack(w, v);
}

// ---- a row written: out[0, len) = f(x[0, len)), or zeros.
__device__ __forceinline__ void store_one(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_one(bf16_t* p, float v) { p->v = (uint16_t)pack_bf16(v, 0.f); }
__device__ __forceinline__ void store_full(float* out, int i, const float (&v)[4]) {
  Raw<float> r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r.w[j] = __float_as_uint(v[j]);
  *reinterpret_cast<Raw<float>*>(out + (int64_t)i * 4) = r;
}
__device__ __forceinline__ void store_full(bf16_t* out, int i, const float (&v)[8]) {
  Raw<bf16_t> r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r.w[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
  *reinterpret_cast<Raw<bf16_t>*>(out + (int64_t)i * 8) = r;
}
template <typename T, class F>
__device__ __forceinline__ void map(const T* x, T* out, int len, F f) {
  constexpr int VEC = Elem<T>::VEC, U = 4;
  const int full = len / VEC, tid = threadIdx.x;
  int base = 0;
  for (; base + U * NT <= full; base += U * NT) {
    float v[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) load_full(x, base + u * NT + tid, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[u][j] = f(v[u][j]);
      store_full(out, base + u * NT + tid, v[u]);
    }
  }
  for (int i = base + tid; i < full; i += NT) {
    float v[VEC];
    load_full(x, i, v);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = f(v[j]);
    store_full(out, i, v);
  }
  for (int i = full * VEC + tid; i < len; i += NT) store_one(out + i, f(Elem<T>::one(x + i)));
}
template <typename T>
__device__ __forceinline__ void fill_zero(T* out, int len) {
  constexpr int VEC = Elem<T>::VEC;
  const int full = len / VEC;
  const float zero[VEC] = {};
  for (int i = threadIdx.x; i < full; i += NT) store_full(out, i, zero);
  for (int i = full * VEC + (int)threadIdx.x; i < len; i += NT) store_one(out + i, 0.f);
}

// ---- sums and maxima over the workgroup, the same value in every thread.  `s`: WAVES values of LDS.
template <int W>
__device__ __forceinline__ double block_sum(double v, double* s) {
  v = wave_total_d(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < W; ++w) v += s[w];
  return v;
}
template <int W>
__device__ __forceinline__ double block_max(double v, double* s) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s[0];
#pragma unroll
  for (int w = 1; w < W; ++w) v = fmax(v, s[w]);
  return v;
}

// The scale of a temperature, computed on the host.
struct Scale {
  float c;       // log2(e) / T in fp32
  float margin;  // how far a logit may exceed the reference: two powers of two
  double inv_t;  // 1 / T
  double kappa;  // ln 2 (log2(e) / T - c) / c
};
inline Scale scale_of(float temperature) {
  Scale s;
  const double c = 1.4426950408889634 / (double)temperature;
  s.c = (float)c;
  s.margin = (float)(2.0 / c);
  s.inv_t = 1.0 / (double)temperature;
  s.kappa = 0.6931471805599453 * (c - (double)s.c) / (double)s.c;
  return s;
}
// Temperatures whose c or margin leave fp32's normal numbers are refused.
inline bool scale_ok(float temperature) { return temperature >= 1e-30f && temperature <= 1e30f; }

// What a slice of a row (or the whole row) adds up to: its largest logit, S and U against it, and how
// many of its elements come before the target in (logit desc, index asc).
struct State {
  double S, U;
  float m;
  int32_t before;
};
// The join of two: S and U against the larger maximum.
__device__ __forceinline__ void rebase(double& S, double& U, float from, double to, const Scale& sc) {
  const double d = fmax(((double)from - to) * sc.c, -2000.0);
  const double f = exp2(d);
  U = f * (U + d * S);
  S = f * S;
}

// Largest of N values and a running one.  v_max3_f32 by itself: fmaxf would first quiet each operand.
template <int N>
__device__ __forceinline__ float max_of(const float (&x)[N]) {
  float m;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(x[0]), "v"(x[1]), "v"(x[2]));
  if constexpr (N == 4) {
    asm("v_max_f32 %0, %1, %2\n\ts_nop 1" : "=v"(m) : "v"(m), "v"(x[3]));
  } else {
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(m), "v"(x[3]), "v"(x[4]));
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(m), "v"(x[5]), "v"(x[6]));
    asm("v_max_f32 %0, %1, %2\n\ts_nop 1" : "=v"(m) : "v"(m), "v"(x[7]));
  }
  return m;
}

template <int CTRL>
__device__ __forceinline__ float max_dpp(float v) {
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true)));
}

struct Thread {
  float r, m, S, U;
  int before;
};

// One pass over x[0, len) by the workgroup, whose threads take 16 bytes in turn.
//   TOP: group_max[g] = the largest of the elements [32 g, 32 g + 32).
//   NAMED: elements whose bit in `named` is set count as masked.
//   xt, t: the target's logit (+inf: no target) and index, from x's begin.
template <typename T, bool TOP, bool NAMED>
__device__ __forceinline__ State scan(const T* x, int len, const Scale& sc, float xt, int64_t t, float* group_max,
                                      const uint32_t* named, double* red) {
  constexpr int VEC = Elem<T>::VEC, U = 4, LANES = GROUP / VEC;
  const int full = len / VEC, n = (len + VEC - 1) / VEC;
  const int tid = threadIdx.x;
  Thread a{LOWEST, -INFINITY, 0.f, 0.f, 0};

  auto take = [&](float(&v)[VEC], int i) {
    if constexpr (NAMED) {
      const uint32_t bits = i < n ? (named[(i * VEC) >> 5] >> ((i * VEC) & 31)) & ((1u << VEC) - 1u) : 0u;
      if (bits) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (bits >> j & 1) v[j] = -INFINITY;
      }
    }
    const float cm = max_of(v);
    if constexpr (TOP) {
      float g = max_dpp<0xB1>(cm);                   // quad_perm [1,0,3,2]
      g = max_dpp<0x4E>(g);                          // quad_perm [2,3,0,1]
      if constexpr (LANES == 8) g = max_dpp<0x141>(g);  // row_half_mirror
      if ((tid & (LANES - 1)) == 0 && i < n) group_max[i / LANES] = g;
    }
    if (cm >= xt) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int64_t at = (int64_t)i * VEC + j;
        a.before += (v[j] > xt || (v[j] == xt && at < t)) ? 1 : 0;
      }
    }
    a.m = fmaxf(a.m, cm);
    if (cm > a.r + sc.margin) {
      const float d = fmaxf((a.r - cm) * sc.c, -1000.f);
      const float f = __builtin_amdgcn_exp2f(d);
      a.U = f * (a.U + d * a.S);
      a.S = f * a.S;
      a.r = cm;
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float d = (v[j] - a.r) * sc.c;
      const float e = __builtin_amdgcn_exp2f(d);
      a.S += e;
      a.U = __builtin_fmaf(e, fmaxf(d, -1000.f), a.U);
    }
  };

  int base = 0;
  for (; base + U * NT <= full; base += U * NT) {
    float v[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) load_full(x, base + u * NT + tid, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) take(v[u], base + u * NT + tid);
  }
  for (; base < n; base += NT) {
    const int i = base + tid;
    float v[VEC];
    if (i < full)
      load_full(x, i, v);
    else
      load_edge(x, i < n ? len : 0, i, v);
    take(v, i);
  }

  // to the largest logit of all threads
  State s;
  const double m = block_max<WAVES>((double)a.m, red);
  s.m = (float)m;
  double S = a.S, Ud = a.U;
  rebase(S, Ud, a.r, m, sc);
  if (a.S == 0.f) S = Ud = 0.0;  // nothing met (its reference means nothing); a NaN stays
  s.S = block_sum<WAVES>(S, red);
  s.U = block_sum<WAVES>(Ud, red);
  s.before = (int32_t)block_sum<WAVES>((double)a.before, red);
  return s;
}

// ---- host: how a batch of rows is cut, and what every call checks
struct Cut {
  int slices, len;  // slices a row, of `len` elements (the last one less)
};

// A gradient writes each element by itself, so its rows are cut wherever there are few.
inline Cut grad_cut(int rows, int V) {
  int64_t want = (2048 + rows - 1) / rows;
  if (want > V / 4096) want = V / 4096;
  if (want < 1) want = 1;
  const int len = (int)(((V + want - 1) / want + GROUP - 1) / GROUP * GROUP);
  return {(V + len - 1) / len, len};
}

// One workgroup of NT threads per slice: HIP's grids stop short of 2^32 threads.
inline int check_grid(int rows, const Cut& c) {
  if ((int64_t)rows * c.slices > (1 << 22)) return fail(DSV41_E_UNSUPPORTED, "more than 2^22 row slices are not supported");
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
