// inthead.hip — logits of an 8-bit head: rows quantized to integers, and their product with the head's
// rows on the integer matrix cores.
//
// A row x of bf16 becomes q_k = rint(127 x_k / a) with a = max |x| and the scale a / 127 (fp32); the
// head's rows w are kept that way.  127 x_k and a have 15 and 8 bits, so their quotient is a half or at
// least 2^-9 of its size away from one: the fp32 division decides as the exact one.  With s, t the scales,
//   out[n, v] = (sum_k q[n, k] w[v, k]) s[n] t[v],
// the sum exact in 32-bit integers (up to 2^31 / 127^2 = 133152 columns), then two fp32 products.
//
// The columns are padded to a multiple of 128 (one cache line of a row), those of q with zeros.
//
// head_kernel, up to 64 tokens, is bound by reading w once.  A workgroup takes 64 rows of w, its eight waves
// every eighth line of their columns; fragments go from memory to registers with no LDS between, and
// the waves' integer sums meet in LDS (atomics whose order does not matter to integers).
// gemm_kernel, above, has the schedule of the bf16 products (mfma_tile.h): 256 x 256 tiles, eight waves
// whose pairs multiply and read in turns, stages of 128 bytes a row loaded straight to LDS.  An integer
// fragment (16 rows x 64) lies in a row's bytes exactly as a bf16 one (16 x 32).

#include <algorithm>
#include <type_traits>

#include "mfma_tile.h"
#include "row_scan.h"

namespace dsv41 {
namespace inthead {

using TL = Tile<SQUARE>;
using rows::bf16_t;
constexpr int BM = TL::BV, BN = TL::BT;
constexpr int LINE = ROWB;            // columns are padded to whole lines
constexpr int MAX_COLUMNS = 133120;   // 2^31 / 127^2 = 133152, in whole lines
constexpr int QUANT_NT = 256;
constexpr int FEW = 64;               // tokens of head_kernel
constexpr int HEAD_ROWS = 64;         // rows of w of its workgroup

typedef int intx4 __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------------------- quantization
__global__ __launch_bounds__(QUANT_NT) void quantize_kernel(const bf16_t* x, int64_t xs, int cols, int8_t* q, int64_t qs,
                                                            int padded, float* scales, int32_t* status) {
  constexpr int G = 8;
  __shared__ float tops[QUANT_NT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  x += (int64_t)blockIdx.x * xs;
  q += (int64_t)blockIdx.x * qs;
  float top = 0.f;
  int odd = 0;  // a NaN or an infinity
  for (int i = tid * G; i < cols; i += QUANT_NT * G) {
    uint32_t w[4];
    rows::load_some<false>(x, 0, cols, i / G, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float lo = bf16_lo(w[j]), hi = bf16_hi(w[j]);
      if (i + 2 * j < cols) odd |= !isfinite(lo), top = fmaxf(top, fabsf(lo));
      if (i + 2 * j + 1 < cols) odd |= !isfinite(hi), top = fmaxf(top, fabsf(hi));
    }
  }
  top = wave_max(top);
  if (lane == 0) tops[wave] = top;
  odd = __syncthreads_or(odd);
  for (int w = 0; w < QUANT_NT / 64; ++w) top = fmaxf(top, tops[w]);
  if (tid == 0) {
    scales[blockIdx.x] = odd ? __builtin_nanf("") : top / 127.f;
    if (status) status[blockIdx.x] = odd ? DSV41_STATUS_NONFINITE : 0;
  }
  const bool none = odd || top == 0.f;
  const float lift = top > 1e30f ? 0x1p-64f : 1.f;  // (127 x is finite; what it takes from small x is far below a half)
  top *= lift;
  for (int i = tid * G; i < padded; i += QUANT_NT * G) {
    uint32_t w[4];
    rows::load_some<false>(x, 0, cols, i / G, w);
    uint32_t o[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const float v = j & 1 ? bf16_hi(w[j >> 1]) : bf16_lo(w[j >> 1]);
      const int k = none || i + j >= cols ? 0 : (int)rintf(127.f * (v * lift) / top);
      o[j >> 2] |= (uint32_t)(k & 0xFF) << (8 * (j & 3));
    }
    *reinterpret_cast<uint2*>(q + i) = make_uint2(o[0], o[1]);
  }
}

// -------------------------------------------------------------------------------- few tokens
struct Params {
  const int8_t* w;
  int64_t ws;
  const float* ts;  // scales of w's rows
  const int8_t* q;  // [N rounded up to 16, K] (the rows past N are read, and their sums left out)
  const float* ss;
  int N, V, K;      // K: a multiple of 128
  void* out;
  int64_t os;
  int n_tb, ranges;
};

template <typename T>
__device__ __forceinline__ float logit(int sum, float s, float t) {
  return (float)sum * s * t;
}

template <typename T, int NB>  // NB blocks of 16 tokens
__global__ __launch_bounds__(NT) void head_kernel(Params p) {
  __shared__ int sums[NB * 16][HEAD_ROWS + 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, quad = lane >> 4;
  const int v0 = blockIdx.x * HEAD_ROWS;
  for (int i = tid; i < NB * 16 * (HEAD_ROWS + 4); i += NT) (&sums[0][0])[i] = 0;
  __syncthreads();
  intx4 acc[4][NB];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[i][b] = intx4{0, 0, 0, 0};
  const int8_t* w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = p.w + (int64_t)min(v0 + 16 * i + r16, p.V - 1) * p.ws + 16 * quad;
  const int8_t* q = p.q + (int64_t)r16 * p.K + 16 * quad;
  for (int k = wave * LINE; k < p.K; k += NWAVES * LINE) {
    intx4 a[4][2], b[NB][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i][h] = *reinterpret_cast<const intx4*>(w[i] + k + 64 * h);
#pragma unroll
      for (int i = 0; i < NB; ++i) b[i][h] = *reinterpret_cast<const intx4*>(q + (int64_t)16 * i * p.K + k + 64 * h);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[i][h], b[j][h], acc[i][j], 0, 0, 0);
  }
  // lane: rows 4 quad .. + 3 of w, token r16
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) atomicAdd(&sums[16 * j + r16][16 * i + 4 * quad + r], acc[i][j][r]);
  __syncthreads();
  T* out = static_cast<T*>(p.out);
  for (int i = tid; i < NB * 16 * HEAD_ROWS; i += NT) {
    const int n = i / HEAD_ROWS, v = i % HEAD_ROWS;
    if (n < p.N && v0 + v < p.V)
      rows::store_one(out + n * p.os + v0 + v, logit<T>(sums[n][v], p.ss[n], p.ts[v0 + v]));
  }
}

// ------------------------------------------------------------------------------- many tokens
template <typename T, bool WIDE>  // WIDE: rows of the output take 4 elements at once
__global__ __launch_bounds__(NT, 1) __attribute__((amdgpu_waves_per_eu(2, 2))) void gemm_kernel(Params p) {
  __shared__ __align__(1024) unsigned char lds[2 * TL::STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wv = wid % SQUARE, wt = wid / SQUARE;
  int tb, range;
  if (!xcd_item(blockIdx.x, p.n_tb, p.ranges, tb, range)) return;
  const int n_mb = (p.V + BM - 1) / BM, nst = p.K / LINE;
  const int mb0 = (int)((int64_t)range * n_mb / p.ranges), mb1 = (int)((int64_t)(range + 1) * n_mb / p.ranges);
  const int total = (mb1 - mb0) * nst;
  const int t0 = tb * BN;

  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr_t)lds;
  uint32_t wvo[2], xvo[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = wid * 16 + 8 * i + (lane >> 3), c = (lane & 7) ^ swz(r);
    wvo[i] = (uint32_t)(r * p.ws) + 16 * c;
    xvo[i] = (uint32_t)(r * p.K) + 16 * c;
  }
  const uint32_t whalf = (uint32_t)(128 * p.ws), xhalf = (uint32_t)(128 * p.K);
  int ld = 0, ld_k = 0, ld_m = mb0 * BM;  // the stage being loaded
  auto rows_of_w = [&](int r0) { return rsrc(p.w + (int64_t)r0 * p.ws, (uint32_t)(min(BM, p.V - r0) * p.ws)); };
  v4i wrs = rows_of_w(ld_m);
  const v4i xrs = rsrc(p.q + (int64_t)t0 * p.K, (uint32_t)(min(BN, p.N - t0) * p.K));
  auto load_region = [&](int reg) {
    const uint32_t dst = lds0 + (uint32_t)((ld & 1) * TL::STAGE + reg * TL::REGION_W + wid * 2048);
    const uint32_t past = ld >= total ? 1u << 31 : 0u;
    const uint32_t off = (uint32_t)(ld_k * LINE) + (reg & 1) * (reg < B0 ? whalf : xhalf) + past;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (reg < B0) load_lds(wrs, wvo[i] + off, dst + i * 1024);
      else load_lds(xrs, xvo[i] + off, dst + i * 1024);
    }
  };
  auto next_load_stage = [&]() {
    ++ld;
    if (++ld_k == nst) {
      ld_k = 0;
      ld_m = min(ld_m + BM, (mb1 - 1) * BM);  // (past the last stage nothing is read)
      wrs = rows_of_w(ld_m);
    }
  };

  const int r16 = lane & 15, quad = lane >> 4;
  uint32_t ra[KS], rb[KS];
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    ra[i] = (uint32_t)((wv * 64 + r16) * ROWB + (((4 * i + quad) ^ swz(r16)) << 4));
    rb[i] = 2 * TL::REGION_W + (uint32_t)((wt * 32 + r16) * ROWB + (((4 * i + quad) ^ swz(r16)) << 4));
  }
  intx4 acc[WV][WT];
  intx4 fa[4][KS], fb0[2][KS], fb1[2][KS];
  auto frag = [&](uint32_t off) { return *reinterpret_cast<const intx4*>(lds + off); };
  auto read_w = [&](int h) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i) fa[i][ks] = frag(ra[ks] + h * TL::REGION_W + i * 16 * ROWB);
  };
  auto read_x = [&](intx4 (&fb)[2][KS], int ks, int h) {
#pragma unroll
    for (int i = 0; i < 2; ++i) fb[i][ks] = frag(rb[ks] + h * TL::REGION_X + i * 16 * ROWB);
  };
  auto multiply = [&](auto first, int h, int j, const intx4 (&fb)[2][KS], auto&& after) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          intx4& c = acc[4 * h + i][2 * j + q];
          const intx4 c0 = first && ks == 0 ? intx4{} : c;
          c = __builtin_amdgcn_mfma_i32_16x16x64_i8(fa[i][ks], fb[q][ks], c0, 0, 0, 0);
        }
      after(ks);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
  };
  auto nothing = [](int) {};
  auto stage = [&](auto first) {
    read_w(0);
    load_region(B1);
    wait_loads<TL::AHEAD>();
    barrier();
    multiply(first, 0, 0, fb0, nothing);
    barrier();

#pragma unroll
    for (int ks = 0; ks < KS; ++ks) read_x(fb1, ks, 1);
    load_region(A1);
    next_load_stage();
    wait_loads<TL::AHEAD>();
    barrier();
    multiply(first, 0, 1, fb1, nothing);
    barrier();

    read_w(1);
    load_region(B0);
    wait_loads<TL::AHEAD>();
    barrier();
    multiply(first, 1, 1, fb1, nothing);
    barrier();

#pragma unroll
    for (int i = 0; i < KS; ++i) {
      ra[i] ^= TL::STAGE;
      rb[i] ^= TL::STAGE;
      asm volatile("" : "+v"(ra[i]), "+v"(rb[i]));  // here, not among the multiplies
    }
    load_region(A0);
    wait_loads<TL::AHEAD>();
    barrier();
    multiply(first, 1, 0, fb0, [&](int ks) { read_x(fb0, ks, 0); });
  };

  load_region(B0);
  load_region(A0);
  load_region(B1);
  load_region(A1);
  next_load_stage();
  load_region(B0);
  load_region(A0);
  wait_loads<TL::AHEAD>();
  barrier();
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) read_x(fb0, ks, 0);
  if (wid >= NWAVES / 2) barrier();

  T* out = static_cast<T*>(p.out);
  for (int mb = mb0; mb < mb1; ++mb) {
    stage(std::true_type{});
    for (int k = 1; k < nst; ++k) {
      barrier();
      stage(std::false_type{});
    }
    // lane: four consecutive rows of w and one token of each block
#pragma unroll
    for (int j = 0; j < WT; ++j) {
      int n = t0 + wt * 32 + col_off<TL>(j) + r16;
      asm volatile("" : "+v"(n));  // addresses are formed here, not kept across the blocks
      if (n >= p.N) continue;
      const float s = p.ss[n];
#pragma unroll
      for (int i = 0; i < WV; ++i) {
        const int m = mb * BM + wv * 64 + row_off<TL>(i, 0) + 4 * quad;
        const intx4 c = acc[i][j];
        T* o = out + (int64_t)n * p.os + m;
        if (WIDE && m + 4 <= p.V) {
          const float4 t = *reinterpret_cast<const float4*>(p.ts + m);
          const float r[4] = {logit<T>(c[0], s, t.x), logit<T>(c[1], s, t.y), logit<T>(c[2], s, t.z), logit<T>(c[3], s, t.w)};
          if constexpr (sizeof(T) == 4)
            *reinterpret_cast<float4*>(o) = make_float4(r[0], r[1], r[2], r[3]);
          else
            *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16(r[0], r[1]), pack_bf16(r[2], r[3]));
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (m + r < p.V) rows::store_one(o + r, logit<T>(c[r], s, p.ts[m + r]));
        }
      }
    }
    barrier();
  }
  if (wid < NWAVES / 2) barrier();
  wait_loads<0>();  // no load to LDS outlives the loop
}

// ---------------------------------------------------------------------------------------- host
constexpr int64_t MAX_GRID = 1 << 22;

int padded_of(int cols) { return (cols + LINE - 1) / LINE * LINE; }

int check_cols(int cols) {
  if (cols <= 0) return fail(DSV41_E_INVALID, "rows need columns");
  if (cols > MAX_COLUMNS) return fail(DSV41_E_UNSUPPORTED, "more than 133120 columns overflow a 32-bit sum");
  return DSV41_OK;
}

int check_head(const dsv41_int_head_desc* d) {
  if (!d) return fail(DSV41_E_INVALID, "8-bit head descriptor is NULL");
  if (d->struct_size != sizeof(dsv41_int_head_desc))
    return fail(DSV41_E_ABI, "dsv41_int_head_desc size mismatch (rebuild the binding)");
  if (d->n_tokens < 0 || d->vocab <= 0) return fail(DSV41_E_INVALID, "hidden must be [tokens, hidden] and the head [vocab, hidden]");
  if (int rc = check_cols(d->hidden)) return rc;
  if (!d->w || !d->scales || (d->n_tokens > 0 && (!d->x || !d->out))) return fail(DSV41_E_INVALID, "x, w, scales and out are required");
  if (d->out_dtype != DSV41_DTYPE_F32 && d->out_dtype != DSV41_DTYPE_BF16) return fail(DSV41_E_INVALID, "logits must be fp32 or bf16");
  if (d->x_row_stride < d->hidden || d->out_row_stride < d->vocab)
    return fail(DSV41_E_INVALID, "8-bit head: row strides must cover the rows");
  if (d->w_row_stride < padded_of(d->hidden) || d->w_row_stride % LINE || (uintptr_t)d->w % 16)
    return fail(DSV41_E_INVALID, "8-bit head: rows of w are 16-byte aligned, and padded to a multiple of 128 columns");
  if ((uintptr_t)d->x % 2 || (uintptr_t)d->scales % 16 || (uintptr_t)d->out % (d->out_dtype == DSV41_DTYPE_F32 ? 4 : 2))
    return fail(DSV41_E_INVALID, "8-bit head: operands are not aligned to their type, or the scales not to 16 bytes");
  if (256 * d->w_row_stride >= (1ll << 31)) return fail(DSV41_E_UNSUPPORTED, "row stride too large for 32-bit block offsets");
  if ((int64_t)d->n_tokens > MAX_GRID) return fail(DSV41_E_UNSUPPORTED, "8-bit head: the batch is too large for one call");
  return DSV41_OK;
}

size_t scales_at(const dsv41_int_head_desc* d) { return (size_t)((d->n_tokens + 15) / 16 * 16) * padded_of(d->hidden); }

template <typename T>
void launch(const Params& p, hipStream_t s) {
  const dim3 few((p.V + HEAD_ROWS - 1) / HEAD_ROWS);
  if (p.N <= 16) hipLaunchKernelGGL((head_kernel<T, 1>), few, dim3(NT), 0, s, p);
  else if (p.N <= 32) hipLaunchKernelGGL((head_kernel<T, 2>), few, dim3(NT), 0, s, p);
  else if (p.N <= 48) hipLaunchKernelGGL((head_kernel<T, 3>), few, dim3(NT), 0, s, p);
  else if (p.N <= FEW) hipLaunchKernelGGL((head_kernel<T, 4>), few, dim3(NT), 0, s, p);
  else {
    const dim3 grid((p.n_tb * p.ranges + 7) / 8 * 8);
    const bool wide = p.os % 4 == 0 && (uintptr_t)p.out % (4 * sizeof(T)) == 0;
    if (wide) hipLaunchKernelGGL((gemm_kernel<T, true>), grid, dim3(NT), 0, s, p);
    else hipLaunchKernelGGL((gemm_kernel<T, false>), grid, dim3(NT), 0, s, p);
  }
}

}  // namespace inthead
}  // namespace dsv41

using namespace dsv41;
using namespace dsv41::inthead;

extern "C" int dsv41_quantize_rows_run(const void* x, int64_t xs, int rows, int cols, int8_t* q, int64_t qs, float* scales,
                                       int32_t* status, void* stream) {
  if (int rc = check_cols(cols)) return rc;
  if (rows < 0 || xs < cols || qs < padded_of(cols) || qs % 16)
    return fail(DSV41_E_INVALID, "quantize: row strides must cover the rows, padded to a multiple of 128 columns");
  if (rows > 0 && (!x || !q || !scales)) return fail(DSV41_E_INVALID, "quantize: x, q and scales are required");
  if ((uintptr_t)x % 2 || (uintptr_t)q % 16 || (uintptr_t)scales % 4)
    return fail(DSV41_E_INVALID, "quantize: operands are not aligned");
  if (rows > MAX_GRID) return fail(DSV41_E_UNSUPPORTED, "quantize: too many rows for one call");
  if (rows == 0) return DSV41_OK;
  hipLaunchKernelGGL(quantize_kernel, dim3(rows), dim3(QUANT_NT), 0, static_cast<hipStream_t>(stream),
                     static_cast<const bf16_t*>(x), xs, cols, q, qs, padded_of(cols), scales, status);
  DSV41_HIP_CHECK(hipGetLastError());
  return DSV41_OK;
}

extern "C" size_t dsv41_int_head_workspace_bytes(const dsv41_int_head_desc* d) {
  return check_head(d) ? 0 : scales_at(d) + (size_t)d->n_tokens * sizeof(float);
}

extern "C" int dsv41_int_head_run(const dsv41_int_head_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_head(d)) return rc;
  if (d->n_tokens == 0) return DSV41_OK;
  const size_t at = scales_at(d);
  if (!workspace || workspace_bytes < at + (size_t)d->n_tokens * sizeof(float) || (uintptr_t)workspace % 16)
    return fail(DSV41_E_WORKSPACE, "8-bit head workspace is missing, too small or not 16-byte aligned");
  int8_t* q = static_cast<int8_t*>(workspace);
  float* ss = reinterpret_cast<float*>(q + at);
  const int K = padded_of(d->hidden);
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(quantize_kernel, dim3(d->n_tokens), dim3(QUANT_NT), 0, s, static_cast<const bf16_t*>(d->x),
                     d->x_row_stride, d->hidden, q, (int64_t)K, K, ss, d->out_status);
  Params p{};
  p.w = d->w;
  p.ws = d->w_row_stride;
  p.ts = d->scales;
  p.q = q;
  p.ss = ss;
  p.N = d->n_tokens;
  p.V = d->vocab;
  p.K = K;
  p.out = d->out;
  p.os = d->out_row_stride;
  p.n_tb = (p.N + BN - 1) / BN;
  p.ranges = std::max(1, std::min((p.V + BM - 1) / BM, CU_COUNT / p.n_tb));
  if (d->out_dtype == DSV41_DTYPE_F32) launch<float>(p, s);
  else launch<bf16_t>(p, s);
  DSV41_HIP_CHECK(hipGetLastError());
  return DSV41_OK;
}
