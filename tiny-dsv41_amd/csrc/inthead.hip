// inthead.hip — logits of an 8-bit head: rows quantized to integers, and their product with the head's
// rows on the integer matrix cores.
//
// A row x of bf16 becomes q_k = rint(127 x_k / a) with a = max |x| and the scale a / 127 (fp32); the
// head's rows w are kept that way.  x_k and a have 8 bits, so 127 x_k / a is a half or at least 2^-16 of its
// size away from one (254 X - (2 k + 1) A 2^s is an integer): a quotient good to a last place decides as the exact one.  With s, t the scales,
//   out[n, v] = (sum_k q[n, k] w[v, k]) s[n] t[v],
// the sum exact in 32-bit integers (up to 2^31 / 127^2 = 133144 columns), then two fp32 products.
//
// The columns are padded to a multiple of 128 (one cache line of a row), those of q with zeros.
//
// Times below are of calls, the quantization's launch (3 to 12 us) included, unless they say "kernel".
//
// head_kernel, up to 16 tokens, is bound by reading w once: one token, 7168 -> 129280, kernel 130 us (7.1 TB/s, what a
// nontemporal read reaches), call 135.  A workgroup takes 64 rows of w, its four waves every fourth k-step of their columns;
// fragments go from memory to registers with no LDS between, so the rows lie in memory as tiles of a fragment's lanes.
// (Row-major, each load of a wave met 16 lines, and the loads' rate was the bound: 203 us.)  The waves' integer sums
// meet in LDS.
// ring_kernel, up to 128 tokens, shares the tokens' tiles among up to 256 rows of w, by LDS: 64 tokens of 7168 -> 129280 164
// us, of 2048 -> 151936 67.  Earlier, head_kernel took them, with the tokens' tiles read from L2 for every 64 rows: 205 and
// 73, and for every 128 of long rows 178 to 185.
// gemm_kernel, above, has the schedule of the bf16 products (mfma_tile.h): eight waves whose pairs multiply and read in
// turns, stages of 128 columns loaded straight to LDS, tiles of 256 rows x 192, 256 or 320 tokens.  4096 tokens of 7168 ->
// 129280: bf16 2.61 ms, 2.9 POP/s, fp32 2.90; of 2048 -> 151936 bf16 1.10, 2.3 POP/s, fp32 1.35.  Power bounds the long rows
// (300 tokens in tiles of 256: the matrix cores busy 71% of the cycles at 1.73 GHz).  Of 2048 columns a tile has 16 stages,
// and a fifth of its time is the conversion and stores of its logits; of 1024 columns that is nearly half, of fewer more: 4096
// tokens of 1024, 512 and 256 columns -> 151936 take 712, 555 and 457 us in bf16, 944, 777 and 690 in fp32.

#include <algorithm>
#include <iterator>
#include <type_traits>

#include "mfma_tile.h"
#include "ring_rule.h"
#include "row_scan.h"

namespace dsv41 {
namespace inthead {

using TL = Tile<SQUARE>;
using rows::bf16_t;
constexpr int BM = TL::BV;
constexpr int LINE = ROWB;            // columns are padded to whole lines
constexpr int MAX_COLUMNS = 133120;   // 2^31 / 127^2 = 133144, in whole lines (132104 where the head holds -128)
constexpr int QUANT_NT = 256;
// Tokens of head_kernel (a fragment's, at most), and of ring_kernel.  By the first and the second, fp32: 16 tokens of 7168 ->
// 129280 149 and 150 us, 8 141 and 144, one 135 and 140; of 2048 -> 151936 55 and 58, 53 and 55, 51 and 53.  By the second and
// gemm_kernel: 17 tokens of 7168 149 and 155, 128 183 and 184; of 2048 57 and 71, 80 and 88.
constexpr int FEW = 16, RING_TOKENS = 128;

typedef int intx4 __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------------------------ layout
// Tiles of 16 rows x 64 columns, in the order of a fragment's lanes: 16 columns of each row, row after row, four
// times.  The tiles of 16 rows follow one another along the columns.
constexpr int TILE = 1024;
constexpr int GROUP = 64;  // rows of a head that share four tiles' rows
// Row m of a head's tile i is row 16 (m / 4) + 4 i + m % 4 of its group of 64: a lane, which holds sums of four rows of
// a tile, holds 16 neighbouring logits of four tiles.
__device__ __forceinline__ int64_t head_row(int64_t v) {  // -> the row's place among the tiles' rows
  const int r = (int)(v % GROUP);
  return v - r + (r >> 2 & 3) * 16 + (r >> 4) * 4 + (r & 3);
}
// Byte of column c (a multiple of 8) of the row at place m.
__device__ __forceinline__ int64_t byte_of(int64_t m, int c, int padded) {
  return (m / 16 * (padded / 64) + c / 64) * TILE + (c / 16 % 4) * 256 + m % 16 * 16 + c % 16;
}

// ------------------------------------------------------------------------------- quantization
// One workgroup a row; the first KEPT chunks of a thread stay in registers between the two passes.
constexpr int KEPT = 4;

// 8 elements of x[0, cols) from i on, zeros where it ends
__device__ __forceinline__ void load_chunk(const bf16_t* x, int cols, int i, uint32_t (&w)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = 0;
  if (i + 8 <= cols) {
    rows::load16<false>(x + i, w);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < cols) rows::Elem<bf16_t>::put(w, j, x[i + j]);
  }
}
// Chunks of x[0, cols), c STEP + i for c < C: those of rows of whole chunks are on their way together (a condition around
// a load has the wave wait for it); ones past the end hold anything until cut() makes them zeros.
template <int C, int STEP>
__device__ __forceinline__ void load_chunks(const bf16_t* x, int cols, int i, uint32_t (&w)[C][4]) {
  if (cols % 8 == 0) {
#pragma unroll
    for (int c = 0; c < C; ++c) rows::load16<false>(x + min(c * STEP + i, cols - 8), w[c]);
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c) load_chunk(x, cols, c * STEP + i, w[c]);
  }
}
__device__ __forceinline__ void cut(uint32_t (&w)[4], bool there) {
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = there ? w[j] : 0;
}
// The largest magnitude's bits, of which those of infinities and NaNs are the largest.
__device__ __forceinline__ uint32_t top_of(const uint32_t (&w)[4], uint32_t top) {
#pragma unroll
  for (int j = 0; j < 4; ++j) top = max(top, max((w[j] << 16) & 0x7FFF0000u, w[j] & 0x7FFF0000u));
  return top;
}
// What the largest magnitude of a row makes of it.
struct Span {
  bool odd, none;
  float lift, most, over, scale;  // over: about 1 / most
};
__device__ __forceinline__ Span span_of(uint32_t top) {
  const float most = __uint_as_float(top);
  Span r;
  r.odd = top >= 0x7F800000u, r.none = r.odd || top == 0;
  r.scale = r.odd ? __builtin_nanf("") : most / 127.f;
  // (127 x and 1 / most are finite and normal; what it takes from small x is far below a half)
  r.lift = most > 1e30f ? 0x1p-64f : most < 1e-30f ? 0x1p64f : 1.f;
  r.most = most * r.lift;
  r.over = __builtin_amdgcn_rcpf(r.most);
  return r;
}
// The quotient's first guess is off by a few last places at most, so what is left of the dividend (of 15 bits, where guess
// times divisor has 32) is exact, and one step with it (Markstein's) gives a half or an integer exactly and others to a
// last place, far nearer than 2^-16.
__device__ __forceinline__ uint2 quantize(const uint32_t (&w)[4], const Span& r) {
  uint32_t o[2] = {0, 0};
  if (r.none) return make_uint2(0, 0);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float v = j & 1 ? bf16_hi(w[j >> 1]) : bf16_lo(w[j >> 1]);
    const float x = 127.f * (v * r.lift), guess = x * r.over;
    const float q = __builtin_fmaf(__builtin_fmaf(-guess, r.most, x), r.over, guess);
    o[j >> 2] |= (uint32_t)((int)rintf(q) & 0xFF) << (8 * (j & 3));
  }
  return make_uint2(o[0], o[1]);
}

template <bool HEAD>
__global__ __launch_bounds__(QUANT_NT) void quantize_kernel(const bf16_t* x, int64_t xs, int rows, int cols, int8_t* q,
                                                            int padded, float* scales, int32_t* status) {
  constexpr int STEP = QUANT_NT * 8;
  __shared__ uint32_t tops[QUANT_NT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // the rows of a tile on one XCD, whose L2 puts their lines together (workgroups go round-robin over the eight): a head of
  // 7168 x 129280 in 897 us, 1111 with rows in turn
  const int64_t row = (int64_t)(blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  if (row >= rows) return;
  x += row * xs;
  const int64_t place = HEAD ? head_row(row) : row;
  uint32_t kept[KEPT][4], top = 0;
  load_chunks<KEPT, STEP>(x, cols, tid * 8, kept);
#pragma unroll
  for (int c = 0; c < KEPT; ++c) {
    cut(kept[c], c * STEP + tid * 8 < cols);
    top = top_of(kept[c], top);
  }
  for (int i = KEPT * STEP + tid * 8; i < cols; i += STEP) {
    uint32_t w[4];
    load_chunk(x, cols, i, w);
    top = top_of(w, top);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
  for (int w = 0; w < QUANT_NT / 64; ++w) top = max(top, tops[w]);
  const Span span = span_of(top);
  if (tid == 0) {
    scales[row] = span.scale;
    if (status) status[row] = span.odd ? DSV41_STATUS_NONFINITE : 0;
  }
#pragma unroll
  for (int c = 0; c < KEPT; ++c) {
    const int i = c * STEP + tid * 8;
    if (i < padded) *reinterpret_cast<uint2*>(q + byte_of(place, i, padded)) = quantize(kept[c], span);
  }
  for (int i = KEPT * STEP + tid * 8; i < padded; i += STEP) {
    uint32_t w[4];
    load_chunk(x, cols, i, w);
    *reinterpret_cast<uint2*>(q + byte_of(place, i, padded)) = quantize(w, span);
  }
}

// -------------------------------------------------------------------------------- few tokens
// waves of a workgroup, steps of theirs in registers, workgroups of a CU: of one token, 2048 -> 151936 and 7168 -> 129280,
// quantized by a launch before it, 51 and 135 us; eight waves (one workgroup) 51 and 138, two (four workgroups) 57 and 138,
// five steps ahead 53 and 137.
constexpr int SPLIT = 4, DEPTH = 4, PER_CU = 2;
// tokens that head_kernel quantizes itself (with room for eight, one token took 48.9 us instead of 47.7), their columns,
// LDS bytes that shift banks
constexpr int OWN = 4, OWN_COLUMNS = 64 * SPLIT * 8, OWN_PAD = 64;

struct Params {
  const int8_t* w;  // tiles of the head
  const float* ts;  // scales of its rows
  const int8_t* q;  // tiles of the tokens (rows past N are read, and their sums left out)
  const float* ss;
  int N, V, K;      // K: a multiple of 128
  void* out;
  int64_t os;
  const bf16_t* x;  // the tokens themselves, which head_kernel quantizes where they are few
  int64_t xs;
  int cols;
  int32_t* status;
  int n_tb, ranges, w1;  // gemm_kernel's blocks of tokens, the parts its rows are cut into, and its W1
};

template <typename T>
__device__ __forceinline__ float logit(int sum, float s, float t) {
  return (float)sum * s * t;
}

// The four rows of 16 lanes of b and a's, transposed as 2 x 2 blocks: a keeps its even rows and takes b's even rows for its
// odd ones (permlane16), its lower half and b's lower half for its upper one (permlane32).
__device__ __forceinline__ void swap_rows(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0], b = r[1];
}
__device__ __forceinline__ void swap_halves(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0], b = r[1];
}
// 64 neighbouring logits, from column v on, of each of 16 tokens: lane (quad, token) has columns 16 quad .. + 15 in
// c0 .. c3.  The quads exchange theirs, so that a store of 16 bytes a lane writes 64 neighbouring bytes of a token's row
// (4096 tokens, 2048 -> 151936, fp32: 1331 us, 1573 without).  All lanes take part; those of tokens that do not
// exist (there == false) store nothing.  `wide`: rows begin at multiples of 16 bytes.
template <typename T>
__device__ __forceinline__ void store_logits(T* row, int v, int V, bool there, bool wide, const intx4& c0, const intx4& c1,
                                             const intx4& c2, const intx4& c3, float s, const float* ts) {
  const intx4 c[4] = {c0, c1, c2, c3};
  const int quad = (threadIdx.x & 63) >> 4;
  constexpr int E = 16 / sizeof(T), PARTS = 16 / E;  // elements of a store, stores
  uint32_t w[PARTS][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 t = *reinterpret_cast<const float4*>(ts + 4 * i);
    const float r0 = logit<T>(c[i][0], s, t.x), r1 = logit<T>(c[i][1], s, t.y);
    const float r2 = logit<T>(c[i][2], s, t.z), r3 = logit<T>(c[i][3], s, t.w);
    if constexpr (sizeof(T) == 4) {
      w[i][0] = __float_as_uint(r0), w[i][1] = __float_as_uint(r1), w[i][2] = __float_as_uint(r2), w[i][3] = __float_as_uint(r3);
    } else {
      w[i / 2][i % 2 * 2] = pack_bf16(r0, r1), w[i / 2][i % 2 * 2 + 1] = pack_bf16(r2, r3);
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
#pragma unroll
    for (int i = 0; i < PARTS; i += 2) swap_rows(w[i][k], w[i + 1][k]);
    if constexpr (PARTS == 4) {
      swap_halves(w[0][k], w[2][k]);
      swap_halves(w[1][k], w[3][k]);
    } else {
      swap_halves(w[0][k], w[1][k]);
    }
  }
  if (!there) return;
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    const int at = v + (4 * i + quad) * E, left = V - at;
    if (wide && left >= E) {
      *reinterpret_cast<uint4*>(row + at) = make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (j < left) {
          if constexpr (sizeof(T) == 4) row[at + j] = __uint_as_float(w[i][j]);
          else row[at + j].v = (uint16_t)(w[i][j / 2] >> (16 * (j % 2)));
        }
    }
  }
}

// The fragments of one k-step: of a group of 64 rows and of the tokens.
struct Step {
  intx4 a[4], b;
};

// SPLIT waves share the columns of a group, every SPLIT-th k-step each; a workgroup takes group after group, with
// DEPTH - 1 steps of each wave on their way from memory throughout.
// SELF: every workgroup quantizes the tokens itself, into LDS, while its first weights are on their way.
template <typename T, bool SELF>
__global__ __launch_bounds__(64 * SPLIT, SPLIT * PER_CU / 4) void head_kernel(Params p, bool wide) {
  __shared__ intx4 parts[SPLIT - 1][4][64];
  __shared__ float scales[GROUP];
  __shared__ __align__(16) int8_t own[SELF ? OWN * (OWN_COLUMNS + OWN_PAD) : 16];
  __shared__ uint32_t tops[OWN][SPLIT];
  __shared__ float own_scales[OWN];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, quad = lane >> 4;
  const int steps = p.K / 64, turns = (steps + SPLIT * DEPTH - 1) / (SPLIT * DEPTH) * DEPTH, groups = (p.V + GROUP - 1) / GROUP;
  T* out = static_cast<T*>(p.out) + r16 * p.os;
  intx4 acc[4] = {};
  Step f[DEPTH];
  int at = wave, left = turns, ahead = blockIdx.x;  // the step to load, those left of its group, the group
  const int8_t* w = p.w + (int64_t)ahead * GROUP * p.K;  // (the same in all lanes, which add theirs in 32 bits)
  // (a step that is none reads the first bytes of w, which caches hold: loads under a condition cost registers)
  auto load = [&](Step& s) {
    const bool some = ahead < groups && at < steps;
    const int8_t* wa = some ? w + at * TILE : p.w;
    const int64_t tile_row = some ? (int64_t)16 * p.K : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) s.a[i] = __builtin_nontemporal_load(reinterpret_cast<const intx4*>(wa + i * tile_row) + lane);
    if (!SELF) s.b = reinterpret_cast<const intx4*>(p.q + (some ? at * TILE : 0))[lane];
    at += SPLIT;
    if (--left == 0) {
      at = wave, left = turns, ahead += gridDim.x;
      w += (int64_t)gridDim.x * GROUP * p.K;
    }
  };
  // a thread has 8 columns of each token (those past the last token are its again)
  const int token = min(r16, p.N - 1);
  uint32_t kept[OWN][4];
  if (SELF) {
#pragma unroll
    for (int n = 0; n < OWN; ++n) rows::load16<false>(p.x + min(n, p.N - 1) * p.xs + min(tid * 8, p.cols - 8), kept[n]);
  }
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d) load(f[d]);
  if (SELF) {
    uint32_t top[OWN];
#pragma unroll
    for (int n = 0; n < OWN; ++n) {
      cut(kept[n], tid * 8 < p.cols);
      top[n] = top_of(kept[n], 0);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
#pragma unroll
      for (int n = 0; n < OWN; ++n) top[n] = max(top[n], (uint32_t)__shfl_xor((int)top[n], o));
    if (lane == 0) {
#pragma unroll
      for (int n = 0; n < OWN; ++n) tops[n][wave] = top[n];
    }
    rows::lds_barrier();
#pragma unroll
    for (int n = 0; n < OWN; ++n) {
      const Span span = span_of(max(max(tops[n][0], tops[n][1]), max(tops[n][2], tops[n][3])));
      if (tid * 8 < p.K) *reinterpret_cast<uint2*>(own + n * (OWN_COLUMNS + OWN_PAD) + tid * 8) = quantize(kept[n], span);
      if (tid == 0) {
        own_scales[n] = span.scale;
        if (p.status && blockIdx.x == 0 && n < p.N) p.status[n] = span.odd ? DSV41_STATUS_NONFINITE : 0;
      }
    }
    rows::lds_barrier();
  }
  const float ss = SELF ? own_scales[token] : p.ss[token];
  for (int group = blockIdx.x; group < groups; group += gridDim.x) {
    // (read at the end, it would have the wave wait for all steps on their way)
    const float t = p.ts[min(group * GROUP + lane, p.V - 1)];
    for (int turn = 0; turn < turns; turn += DEPTH) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        load(f[(d + DEPTH - 1) % DEPTH]);
        const int step = wave + (turn + d) * SPLIT;
        if (step < steps) {
          const intx4 b = SELF ? *reinterpret_cast<const intx4*>(own + token * (OWN_COLUMNS + OWN_PAD) + step * 64 + quad * 16) : f[d].b;
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[d].a[i], b, acc[i], 0, 0, 0);
        }
      }
    }
    // the waves' sums meet in the first one
    if (wave > 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) parts[wave - 1][i][lane] = acc[i];
    } else {
      scales[lane] = t;
    }
    rows::lds_barrier();
    if (wave == 0) {
#pragma unroll
      for (int s = 0; s < SPLIT - 1; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] += parts[s][i][lane];
      store_logits(out, group * GROUP, p.V, r16 < p.N, wide, acc[0], acc[1], acc[2], acc[3], ss, scales + 16 * quad);
    }
    rows::lds_barrier();
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = intx4{0, 0, 0, 0};
  }
}

// ---------------------------------------------------------------------------- up to 128 tokens
// A workgroup takes a run of groups, up to four at a time, against all tokens, 32 NB at most: wave (wv, wt) group wv's 64 rows
// and half of the tokens.  Stages of 128 columns go straight to a ring of RING in LDS, RING - 1 of them on their way from
// memory throughout; one barrier a stage says that it has come and that the one before it is free.
// load_lds of what is read once: 7168 -> 129280, 128 tokens 208 us without the hint, 183 with it; 64 tokens 189 and 164
__device__ __forceinline__ void load_lds_once(v4i rs, uint32_t voff, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen nt lds" ::"v"(voff), "s"(rs),
               "s"(lds_addr)
               : "memory");
}
template <typename T, int NB>
__global__ __launch_bounds__(NT, 1) __attribute__((amdgpu_waves_per_eu(2, 2))) void ring_kernel(Params p, bool wide) {
  constexpr int STAGE = (32 + 4 * NB) * TILE, LOADS = 4 + NB / 2;  // loads of a wave a stage
  __shared__ __align__(1024) unsigned char lds[RING * STAGE + NWAVES * BM * 4];  // for each wave the block's scales, too
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, quad = lane >> 4;
  const int wv = wid & 3, wt = wid >> 2;
  const int groups = (p.V + GROUP - 1) / GROUP, nst = p.K / LINE;
  const int g0 = (int)((int64_t)blockIdx.x * groups / p.ranges), g1 = (int)((int64_t)(blockIdx.x + 1) * groups / p.ranges);
  const int blocks = (g1 - g0 + 3) / 4, total = blocks * nst;
  auto first_of = [&](int b) { return g0 + (g1 - g0) * b / blocks; };

  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr_t)lds;
  const uint32_t bytes = (uint32_t)(16 * p.K);  // of 16 rows
  auto rows_of_w = [&](int b) {
    const int g = first_of(b);
    return rsrc(p.w + (int64_t)g * GROUP * p.K, (uint32_t)(first_of(b + 1) - g) * 4 * bytes);
  };
  v4i wrs = rows_of_w(0);
  const v4i xrs = rsrc(p.q, (uint32_t)(p.N + 15) / 16 * bytes);
  const v4i srs = rsrc(p.ts, (uint32_t)p.V * 4);
  float* scales = reinterpret_cast<float*>(lds + RING * STAGE) + wid * BM;
  int ld = 0, ld_k = 0, ld_b = 0;  // the stage being loaded
  uint32_t ld_at = 0;
  auto load_stage = [&]() {
    const uint32_t off = (uint32_t)(lane * 16 + ld_k * 2 * TILE) + (ld >= total ? 1u << 31 : 0u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = 2 * wid + i / 2;
      load_lds_once(wrs, off + m * bytes + (i & 1) * TILE, lds0 + ld_at + (2 * m + (i & 1)) * TILE);
    }
#pragma unroll
    for (int i = 0; i < NB / 2; ++i) {
      const int tile = wid * (NB / 2) + i;
      load_lds(xrs, off + (tile >> 1) * bytes + (tile & 1) * TILE, lds0 + ld_at + (32 + tile) * TILE);
    }
    ++ld;
    ld_at = ld_at == (RING - 1) * STAGE ? 0 : ld_at + STAGE;
    if (++ld_k == nst) {
      ld_k = 0;
      ld_b = min(ld_b + 1, blocks - 1);  // (past the last stage nothing is read)
      wrs = rows_of_w(ld_b);
    }
  };
  float ss[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) ss[j] = p.ss[min((wt * NB + j) * 16 + r16, p.N - 1)];
#pragma unroll
  for (int j = 0; j < NB; ++j) asm volatile("" ::"v"(ss[j]));  // here, with no load behind them yet
#pragma unroll
  for (int i = 0; i < RING - 1; ++i) load_stage();

  T* out = static_cast<T*>(p.out);
  uint32_t at = 0;
  for (int b = 0; b < blocks; ++b) {
    const int g = first_of(b);
    const bool some = wv < first_of(b + 1) - g;
    intx4 acc[4][NB];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = intx4{0, 0, 0, 0};
    for (int k = 0; k < nst; ++k) {
      wait_loads<stage_wait(LOADS)>();
      barrier();
      if (k == 0) load_lds(srs, (uint32_t)(g * GROUP * 4 + lane * 16), lds0 + (uint32_t)(RING * STAGE + wid * BM * 4));
      load_stage();
      if (some) {
        const unsigned char* from = lds + at + lane * 16;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          intx4 fa[4], fb[NB];
#pragma unroll
          for (int i = 0; i < 4; ++i) fa[i] = *reinterpret_cast<const intx4*>(from + (2 * (4 * wv + i) + ks) * TILE);
#pragma unroll
          for (int j = 0; j < NB; ++j) fb[j] = *reinterpret_cast<const intx4*>(from + (32 + 2 * (NB * wt + j) + ks) * TILE);
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fa[i], fb[j], acc[i][j], 0, 0, 0);
        }
      }
      at = at == (RING - 1) * STAGE ? 0 : at + STAGE;
    }
    // (longer rows have waited for the scales by now)
    static_assert(scales_wait(2, LOADS) < 0);
    if (nst == 1) wait_loads<scales_wait(1, LOADS)>();
    if (some) {
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const int n = (wt * NB + j) * 16 + r16;
        store_logits(out + (int64_t)n * p.os, (g + wv) * GROUP, p.V, n < p.N, wide, acc[0][j], acc[1][j], acc[2][j], acc[3][j],
                     ss[j], scales + wv * GROUP + 16 * quad);
      }
    }
  }
  wait_loads<0>();  // no load to LDS outlives the loop
}

// ------------------------------------------------------------------------------- many tokens
// W1: blocks of 16 tokens of a wave beyond its first two: tiles of 192 tokens (1), 256 (2) or 320 (3).  ONCE: one tile has all
// tokens, so that no other reads the weights again (256 tokens of 7168 -> 129280 250 us without the hint, 224 with it).
template <typename T, int W1, bool ONCE>
__global__ __launch_bounds__(NT, 1) __attribute__((amdgpu_waves_per_eu(2, 2))) void gemm_kernel(Params p, bool wide) {
  constexpr int WT = 2 + W1, BN = 64 * WT, AHEAD = 6 + W1;  // loads of a wave's four regions
  constexpr int STAGE = 2 * TL::REGION_W + TL::REGION_X + W1 * 8 * TILE;
  // two stages, and for each wave the scales of the block's rows: read from memory between the multiplies, they would
  // have the wave wait for its stores
  __shared__ __align__(1024) unsigned char lds[2 * STAGE + NWAVES * BM * 4];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wv = wid % SQUARE, wt = wid / SQUARE;
  int tb, range;
  if (!xcd_item(blockIdx.x, p.n_tb, p.ranges, tb, range)) return;
  const int n_mb = (p.V + BM - 1) / BM, nst = p.K / LINE;
  const int mb0 = (int)((int64_t)range * n_mb / p.ranges), mb1 = (int)((int64_t)(range + 1) * n_mb / p.ranges);
  const int total = (mb1 - mb0) * nst;
  const int t0 = tb * BN;

  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr_t)lds;
  const int bytes = 16 * p.K;  // of 16 rows
  const uint32_t mine = (uint32_t)(wid * bytes + lane * 16), half = (uint32_t)(8 * bytes);
  int ld = 0, ld_k = 0, ld_m = mb0 * BM;  // the stage being loaded
  auto rows_of_w = [&](int r0) {
    return rsrc(p.w + (int64_t)r0 * p.K, (uint32_t)((min(BM, p.V - r0) + GROUP - 1) / GROUP * GROUP * p.K));
  };
  v4i wrs = rows_of_w(ld_m);
  const v4i xrs = rsrc(p.q + (int64_t)t0 * p.K, (uint32_t)((min(BN, p.N - t0) + 15) / 16 * bytes));
  const v4i srs = rsrc(p.ts, (uint32_t)p.V * 4);
  float* scales = reinterpret_cast<float*>(lds + 2 * STAGE) + wid * BM;
  auto load_scales = [&](int mb) {
    load_lds(srs, (uint32_t)(mb * BM * 4 + lane * 16), lds0 + (uint32_t)(2 * STAGE + wid * BM * 4));
  };
  auto load_region = [&](int reg) {
    const uint32_t dst = lds0 + (uint32_t)((ld & 1) * STAGE + reg * TL::REGION_W + wid * 2 * TILE);
    const uint32_t off = mine + (uint32_t)(ld_k * 2 * TILE) + (reg & 1) * half + (ld >= total ? 1u << 31 : 0u);
    if (W1 != 2 && reg == B1) {  // not two tiles a wave, a row block's, but one or three
#pragma unroll
      for (int i = 0; i < W1; ++i) {
        const int tile = wid * W1 + i;
        load_lds(xrs, (uint32_t)((8 + (tile >> 1)) * bytes + (tile & 1) * TILE + ld_k * 2 * TILE) + (ld >= total ? 1u << 31 : 0u) +
                          (uint32_t)(lane * 16), dst + (tile - 2 * wid) * TILE);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (ONCE && reg < B0) load_lds_once(wrs, off + i * TILE, dst + i * TILE);
      else load_lds(reg < B0 ? wrs : xrs, off + i * TILE, dst + i * TILE);
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
  // a region's tiles: those of a row block's two k-steps side by side
  uint32_t ra = (uint32_t)(wv * 8 * TILE + lane * 16), rb = 2 * TL::REGION_W + (uint32_t)(wt * 4 * TILE + lane * 16);
  uint32_t rb1 = 2 * TL::REGION_W + TL::REGION_X + (uint32_t)(wt * 2 * W1 * TILE + lane * 16);
  int other = STAGE;  // from this stage's place to the other one's
  intx4 acc[WV][WT];
  intx4 fa[4][KS], fb0[2][KS], fb1[W1][KS];
  auto frag = [&](uint32_t off) { return *reinterpret_cast<const intx4*>(lds + off); };
  auto read_w = [&](int h) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i) fa[i][ks] = frag(ra + h * TL::REGION_W + (2 * i + ks) * TILE);
  };
  auto read_x = [&](auto& fb, int ks, uint32_t r) {
#pragma unroll
    for (int i = 0; i < (int)std::size(fb); ++i) fb[i][ks] = frag(r + (2 * i + ks) * TILE);
  };
  auto multiply = [&](auto first, int h, int j, const auto& fb, auto&& after) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < (int)std::size(fb); ++q) {
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
    wait_loads<AHEAD>();
    barrier();
    multiply(first, 0, 0, fb0, nothing);
    barrier();

#pragma unroll
    for (int ks = 0; ks < KS; ++ks) read_x(fb1, ks, rb1);
    load_region(A1);
    next_load_stage();
    wait_loads<AHEAD>();
    barrier();
    multiply(first, 0, 1, fb1, nothing);
    barrier();

    read_w(1);
    load_region(B0);
    wait_loads<AHEAD>();
    barrier();
    multiply(first, 1, 1, fb1, nothing);
    barrier();

    ra += other;
    rb += other;
    rb1 += other;
    other = -other;
    asm volatile("" : "+v"(ra), "+v"(rb), "+v"(rb1));  // here, not among the multiplies
    load_region(A0);
    wait_loads<AHEAD>();
    barrier();
    multiply(first, 1, 0, fb0, [&](int ks) { read_x(fb0, ks, rb); });
  };

  auto token_of = [&](int j) { return j < 2 ? wt * 32 + 16 * j : 128 + wt * 16 * W1 + 16 * (j - 2); };  // of block j, first
  float ss[WT];  // scales of the lane's tokens
#pragma unroll
  for (int j = 0; j < WT; ++j) ss[j] = p.ss[min(t0 + token_of(j) + r16, p.N - 1)];
#pragma unroll
  for (int j = 0; j < WT; ++j) asm volatile("" ::"v"(ss[j]));  // here, with no load behind them yet

  load_region(B0);
  load_region(A0);
  load_region(B1);
  load_region(A1);
  next_load_stage();
  load_region(B0);
  load_region(A0);
  wait_loads<AHEAD>();
  barrier();
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) read_x(fb0, ks, rb);
  if (wid >= NWAVES / 2) barrier();

  T* out = static_cast<T*>(p.out);
  for (int mb = mb0; mb < mb1; ++mb) {
    load_scales(mb);  // here by the end of the next stage, whose loads are all younger
    stage(std::true_type{});
    for (int k = 1; k < nst; ++k) {
      barrier();
      stage(std::false_type{});
    }
    // lane: 16 neighbouring logits of one token of each block, in either half of the rows
#pragma unroll
    for (int j = 0; j < WT; ++j) {
      int n = t0 + token_of(j) + r16;
      asm volatile("" : "+v"(n));  // addresses are formed here, not kept across the blocks
#pragma unroll
      for (int i = 0; i < WV; i += 4) {
        const int m = wv * 64 + row_off<TL>(i, 0);
        store_logits(out + (int64_t)n * p.os, mb * BM + m, p.V, n < p.N, wide, acc[i][j], acc[i + 1][j], acc[i + 2][j],
                     acc[i + 3][j], ss[j], scales + m + 16 * quad);
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

// Workgroups of a quantization: eight XCDs' runs of whole groups of rows.
dim3 quantize_grid(int rows) { return dim3((unsigned)(((int64_t)rows + 8 * GROUP - 1) / (8 * GROUP) * (8 * GROUP))); }

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
  if ((uintptr_t)d->w % 16) return fail(DSV41_E_INVALID, "8-bit head: the tiles must be 16-byte aligned");
  if ((uintptr_t)d->x % 2 || (uintptr_t)d->scales % 16 || (uintptr_t)d->out % (d->out_dtype == DSV41_DTYPE_F32 ? 4 : 2))
    return fail(DSV41_E_INVALID, "8-bit head: operands are not aligned to their type, or the scales not to 16 bytes");
  if ((int64_t)d->n_tokens > MAX_GRID || d->vocab > 1 << 28)
    return fail(DSV41_E_UNSUPPORTED, "8-bit head: the batch or the vocabulary is too large for one call");
  return DSV41_OK;
}

size_t scales_at(const dsv41_int_head_desc* d) { return (size_t)((d->n_tokens + 15) / 16 * 16) * padded_of(d->hidden); }

// What a block of rows costs against a tile of 128 + 64 W1 tokens, 256 tokens' being 1.  Tiles of 192, 256 and 320, us: 256
// tokens of 7168 -> 129280 (fp32) 299, 226 and 247, 300 tokens 313, 352 and 256, 600 570, 519 and 468, 4096 3192, 2903 and
// 2900; of 2048 -> 151936 256 tokens (bf16) 105, 93 and 102, 300 (fp32) 129, 162 and 129, 576 (bf16) 174, 195 and 176, 600
// (fp32) 248, 221 and 209, 1100 (bf16) 345, 311 and 327, 4096 (bf16) 1220, 1096 and 1087.  The stores of short rows' logits
// have no part in it: 4096 tokens of 256, 512 and 1024 columns (bf16) take the tiles of 256, 458, 555 and 709, where those
// of 320 take 427, 516 and 678.
constexpr double TILE_COST[4] = {0, 0.85, 1.0, 1.2};

// Whether head_kernel quantizes the tokens: 2048 -> 151936, one and four tokens 48.6 and 49.5 us, 51.3 and 51.9 by a launch
// before it; of 7168 -> 129280 one token, whose parts a thread then has to hold together, 136.4 and 134.9.
bool own_quantization(int n, int cols) { return n <= OWN && cols <= OWN_COLUMNS && cols % 8 == 0; }

// As many workgroups as fit on the GPU together take the same number of groups each.
template <typename T>
void launch_few(const Params& p, bool wide, hipStream_t s) {
  const int groups = (p.V + GROUP - 1) / GROUP, slots = PER_CU * CU_COUNT, rounds = (groups + slots - 1) / slots;
  const dim3 grid((groups + rounds - 1) / rounds);
  if (own_quantization(p.N, p.cols)) hipLaunchKernelGGL((head_kernel<T, true>), grid, dim3(64 * SPLIT), 0, s, p, wide);
  else hipLaunchKernelGGL((head_kernel<T, false>), grid, dim3(64 * SPLIT), 0, s, p, wide);
}
template <typename T, int NB>
void launch_ring(Params p, bool wide, hipStream_t s) {
  p.ranges = std::min((p.V + GROUP - 1) / GROUP, CU_COUNT);
  hipLaunchKernelGGL((ring_kernel<T, NB>), dim3(p.ranges), dim3(NT), 0, s, p, wide);
}
template <typename T, int W1>
void launch_tiles(const Params& p, bool wide, hipStream_t s) {
  const dim3 grid((p.n_tb * p.ranges + 7) / 8 * 8);
  if (p.n_tb == 1) hipLaunchKernelGGL((gemm_kernel<T, W1, true>), grid, dim3(NT), 0, s, p, wide);
  else hipLaunchKernelGGL((gemm_kernel<T, W1, false>), grid, dim3(NT), 0, s, p, wide);
}
template <typename T>
void launch(const Params& p, hipStream_t s) {
  const bool wide = p.os * sizeof(T) % 16 == 0 && (uintptr_t)p.out % 16 == 0;
  if (p.N <= FEW) {
    launch_few<T>(p, wide, s);
  } else if (p.N <= 64) {
    launch_ring<T, 2>(p, wide, s);
  } else if (p.N <= RING_TOKENS) {
    launch_ring<T, 4>(p, wide, s);
  } else {
    p.w1 == 1 ? launch_tiles<T, 1>(p, wide, s) : p.w1 == 2 ? launch_tiles<T, 2>(p, wide, s) : launch_tiles<T, 3>(p, wide, s);
  }
}

// The tile of the shorter estimate: rounds of workgroups, each of as many blocks of rows as the longest range has.
void plan_tiles(Params& p) {
  const int n_mb = (p.V + BM - 1) / BM;
  double best = 1e300;
  for (int w1 : {2, 1, 3}) {
    const int bn = 128 + 64 * w1, n_tb = (p.N + bn - 1) / bn, ranges = std::max(1, std::min(n_mb, CU_COUNT / n_tb));
    const double cost = (double)((n_tb * ranges + CU_COUNT - 1) / CU_COUNT) * ((n_mb + ranges - 1) / ranges) * TILE_COST[w1];
    if (cost < best) best = cost, p.n_tb = n_tb, p.ranges = ranges, p.w1 = w1;
  }
}

}  // namespace inthead
}  // namespace dsv41

using namespace dsv41;
using namespace dsv41::inthead;

extern "C" int dsv41_quantize_rows_run(const void* x, int64_t xs, int rows, int cols, int8_t* q, float* scales, int32_t* status,
                                       void* stream) {
  if (int rc = check_cols(cols)) return rc;
  if (rows < 0 || xs < cols) return fail(DSV41_E_INVALID, "quantize: the row stride must cover the rows");
  if (rows > 0 && (!x || !q || !scales)) return fail(DSV41_E_INVALID, "quantize: x, q and scales are required");
  if ((uintptr_t)x % 2 || (uintptr_t)q % 16 || (uintptr_t)scales % 4)
    return fail(DSV41_E_INVALID, "quantize: operands are not aligned");
  if (rows > MAX_GRID) return fail(DSV41_E_UNSUPPORTED, "quantize: too many rows for one call");
  if (rows == 0) return DSV41_OK;
  hipLaunchKernelGGL(quantize_kernel<true>, quantize_grid(rows), dim3(QUANT_NT), 0, static_cast<hipStream_t>(stream),
                     static_cast<const bf16_t*>(x), xs, rows, cols, q, padded_of(cols), scales, status);
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
  if (!own_quantization(d->n_tokens, d->hidden))
    hipLaunchKernelGGL(quantize_kernel<false>, quantize_grid(d->n_tokens), dim3(QUANT_NT), 0, s,
                       static_cast<const bf16_t*>(d->x), d->x_row_stride, d->n_tokens, d->hidden, q, K, ss, d->out_status);
  Params p{};
  p.w = d->w;
  p.ts = d->scales;
  p.q = q;
  p.ss = ss;
  p.x = static_cast<const bf16_t*>(d->x);
  p.xs = d->x_row_stride;
  p.cols = d->hidden;
  p.status = d->out_status;
  p.N = d->n_tokens;
  p.V = d->vocab;
  p.K = K;
  p.out = d->out;
  p.os = d->out_row_stride;
  plan_tiles(p);
  if (d->out_dtype == DSV41_DTYPE_F32) launch<float>(p, s);
  else launch<bf16_t>(p, s);
  DSV41_HIP_CHECK(hipGetLastError());
  return DSV41_OK;
}
