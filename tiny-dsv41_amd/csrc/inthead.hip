// inthead.hip — logits of an 8-bit head: rows quantized to integers, and their product with the head's
// rows on the integer matrix cores.
//
// A row x of bf16 becomes q_k = rint(127 x_k / a) with a = max |x| and the scale a / 127 (fp32); the
// head's rows w are kept that way.  x_k and a have 8 bits, so 127 x_k / a is a half or at least 2^-16 of its
// size away from one (254 X - (2 k + 1) A 2^s is an integer): the fp32 division decides as the exact one.  With s, t the scales,
//   out[n, v] = (sum_k q[n, k] w[v, k]) s[n] t[v],
// the sum exact in 32-bit integers (up to 2^31 / 127^2 = 133144 columns), then two fp32 products.
//
// The columns are padded to a multiple of 128 (one cache line of a row), those of q with zeros.
//
// head_kernel, up to 64 tokens, is bound by reading w once: one token, 7168 -> 129280, 130 us (7.1 TB/s, what a
// nontemporal read reaches); 48 tokens of 2048 -> 151936 55 us.  A workgroup takes 64 rows of w, its four
// waves every fourth k-step of their columns; fragments go from memory to registers with no LDS between, so the rows lie
// in memory as tiles of a fragment's lanes.  (Row-major, each load of a wave met 16 lines, and the loads' rate was the
// bound: 203 us, and 316 with 48 tokens of 7168 -> 129280 where tiles take 182.)  The waves' integer sums meet in LDS.
// What more tokens cost is their own tiles, read from L2 by every workgroup.
// gemm_kernel, above, has the schedule of the bf16 products (mfma_tile.h): eight waves whose pairs multiply and read in
// turns, stages of 128 columns loaded straight to LDS, tiles of 256 rows x 256 or 192 tokens.  4096 tokens of 7168 ->
// 129280: 2.69 ms, 2.8 POP/s, the matrix cores busy 71% of the cycles at 1.75 GHz (power); of 2048 -> 151936 1.11 ms,
// 2.3 POP/s: a tile there has 16 stages, and a fifth of its time is the conversion and stores of its logits.

#include <algorithm>
#include <iterator>
#include <type_traits>

#include "mfma_tile.h"
#include "row_scan.h"

namespace dsv41 {
namespace inthead {

using TL = Tile<SQUARE>;
using rows::bf16_t;
constexpr int BM = TL::BV;
constexpr int LINE = ROWB;            // columns are padded to whole lines
constexpr int MAX_COLUMNS = 133120;   // 2^31 / 127^2 = 133144, in whole lines
constexpr int QUANT_NT = 256;
// Tokens of head_kernel.  64 and 65, the first of gemm_kernel: 2048 -> 151936 68 and 81 us, 7168 -> 129280 187 and 189.
constexpr int FEW = 64;

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
// The largest magnitude's bits, of which those of infinities and NaNs are the largest.
__device__ __forceinline__ uint32_t top_of(const uint32_t (&w)[4], uint32_t top) {
#pragma unroll
  for (int j = 0; j < 4; ++j) top = max(top, max((w[j] << 16) & 0x7FFF0000u, w[j] & 0x7FFF0000u));
  return top;
}
__device__ __forceinline__ uint2 quantize(const uint32_t (&w)[4], float lift, float top) {
  uint32_t o[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float v = j & 1 ? bf16_hi(w[j >> 1]) : bf16_lo(w[j >> 1]);
    o[j >> 2] |= (uint32_t)((int)rintf(127.f * (v * lift) / top) & 0xFF) << (8 * (j & 3));
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
#pragma unroll
  for (int c = 0; c < KEPT; ++c) load_chunk(x, cols, c * STEP + tid * 8, kept[c]);
#pragma unroll
  for (int c = 0; c < KEPT; ++c) top = top_of(kept[c], top);
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
  const bool odd = top >= 0x7F800000u;
  float most = __uint_as_float(top);
  if (tid == 0) {
    scales[row] = odd ? __builtin_nanf("") : most / 127.f;
    if (status) status[row] = odd ? DSV41_STATUS_NONFINITE : 0;
  }
  const bool none = odd || top == 0;
  const float lift = most > 1e30f ? 0x1p-64f : 1.f;  // (127 x is finite; what it takes from small x is far below a half)
  most *= lift;
#pragma unroll
  for (int c = 0; c < KEPT; ++c) {
    const int i = c * STEP + tid * 8;
    if (i < padded) *reinterpret_cast<uint2*>(q + byte_of(place, i, padded)) = none ? make_uint2(0, 0) : quantize(kept[c], lift, most);
  }
  for (int i = KEPT * STEP + tid * 8; i < padded; i += STEP) {
    uint32_t w[4];
    load_chunk(x, cols, i, w);
    *reinterpret_cast<uint2*>(q + byte_of(place, i, padded)) = none ? make_uint2(0, 0) : quantize(w, lift, most);
  }
}

// -------------------------------------------------------------------------------- few tokens
constexpr int SPLIT = 4, PER_CU = 2;  // waves of a workgroup, workgroups of a CU

struct Params {
  const int8_t* w;  // tiles of the head
  const float* ts;  // scales of its rows
  const int8_t* q;  // tiles of the tokens (rows past N are read, and their sums left out)
  const float* ss;
  int N, V, K;      // K: a multiple of 128
  void* out;
  int64_t os;
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
// (4096 tokens, 2048 -> 151936: fp32 1573 us without, bf16 1133).  All lanes take part; those of tokens that do not
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

// The fragments of one k-step: of GB groups of 64 rows and of NB blocks of 16 tokens.
template <int NB, int GB>
struct Step {
  intx4 a[4 * GB], b[NB];
};

// SPLIT waves share the columns of GB groups, every SPLIT-th k-step each; a workgroup takes item after item of GB groups, with
// DEPTH - 1 steps of each wave on their way from memory throughout.
template <typename T, int NB, int GB, int DEPTH>
__global__ __launch_bounds__(64 * SPLIT, SPLIT * PER_CU / 4) void head_kernel(Params p, bool wide) {
  __shared__ intx4 parts[SPLIT][4 * NB][64];
  __shared__ float scales[SPLIT][GB * GROUP];  // each wave's copy of the groups'
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, quad = lane >> 4;
  const int steps = p.K / 64, turns = (steps + SPLIT * DEPTH - 1) / (SPLIT * DEPTH) * DEPTH, groups = (p.V + GROUP - 1) / GROUP;
  const int items = (groups + GB - 1) / GB;
  T* out = static_cast<T*>(p.out);
  intx4 acc[4 * GB][NB];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < 4 * GB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = intx4{0, 0, 0, 0};
  };
  clear();
  Step<NB, GB> f[DEPTH];
  int at = wave, left = turns, ahead = blockIdx.x;  // the step to load, those left of its item, the item
  // (addresses are the same in all lanes, which add theirs in 32 bits; a step that is none reads the first bytes of q, which
  // all caches hold, as loads under a condition cost registers; a group past the last is the last one again)
  auto load = [&](Step<NB, GB>& s) {
    const bool some = ahead < items && at < steps;
    const int8_t* qa = p.q + (some ? at * TILE : 0);
    const int64_t tile_row = some ? (int64_t)16 * p.K : 0;
#pragma unroll
    for (int g = 0; g < GB; ++g) {
      const int8_t* wa = some ? p.w + (int64_t)min(ahead * GB + g, groups - 1) * GROUP * p.K + at * TILE : p.q;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s.a[4 * g + i] = __builtin_nontemporal_load(reinterpret_cast<const intx4*>(wa + i * tile_row) + lane);
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) s.b[j] = reinterpret_cast<const intx4*>(qa + j * tile_row)[lane];
    at += SPLIT;
    if (--left == 0) at = wave, left = turns, ahead += gridDim.x;
  };
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d) load(f[d]);
  float ss[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) ss[j] = p.ss[min(16 * j + r16, p.N - 1)];
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    // (read at the end, they would have the wave wait for all steps on their way)
    float t[GB];
#pragma unroll
    for (int g = 0; g < GB; ++g) t[g] = p.ts[min((item * GB + g) * GROUP + lane, p.V - 1)];
    for (int turn = 0; turn < turns; turn += DEPTH) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        load(f[(d + DEPTH - 1) % DEPTH]);
        if (wave + (turn + d) * SPLIT < steps) {
#pragma unroll
          for (int i = 0; i < 4 * GB; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[d].a[i], f[d].b[j], acc[i][j], 0, 0, 0);
        }
      }
    }
    // the waves' sums meet, a group at a time: token block j is wave j % SPLIT's to finish
#pragma unroll
    for (int g = 0; g < GB; ++g) scales[wave][g * GROUP + lane] = t[g];
#pragma unroll
    for (int g = 0; g < GB; ++g) {
#pragma unroll
      for (int j = 0; j < NB; ++j)
        if (j % SPLIT != wave) {
#pragma unroll
          for (int i = 0; i < 4; ++i) parts[wave][4 * j + i][lane] = acc[4 * g + i][j];
        }
      rows::lds_barrier();
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        if (j % SPLIT != wave) continue;
        intx4 c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = acc[4 * g + i][j];
#pragma unroll
        for (int s = 0; s < SPLIT; ++s)
          if (s != wave) {
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] += parts[s][4 * j + i][lane];
          }
        const int n = 16 * j + r16;
        store_logits(out + n * p.os, (item * GB + g) * GROUP, p.V, n < p.N, wide, c[0], c[1], c[2], c[3], ss[j],
                     scales[wave] + g * GROUP + 16 * quad);
      }
      rows::lds_barrier();
    }
    clear();
  }
}

// ------------------------------------------------------------------------------- many tokens
// W1: blocks of 16 tokens of a wave beyond its first two: tiles of 192 tokens (1), 256 (2) or 320 (3).
template <typename T, int W1>
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
    for (int i = 0; i < 2; ++i) load_lds(reg < B0 ? wrs : xrs, off + i * TILE, dst + i * TILE);
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

// A block of rows against 192 tokens costs this of one against 256.  256 and 192 wide, us: 300 tokens of 7168 ->
// 129280 (fp32) 370 and 322, of 2048 -> 151936 (bf16) 133 and 111, 576 tokens 195 and 167; but 256 tokens 99 and 110,
// 1100 tokens 330 and 344, 4096 tokens 1136 and 1221.
constexpr double TILE_COST[4] = {0, 0.85, 1.0, 1.2};

// As many workgroups as fit on the GPU together take the same number of groups each.  Four waves with three
// steps ahead, two workgroups a CU: 2048 -> 151936, 1, 17, 48 and 64 tokens 52, 57, 64 and 68 us, 7168 -> 129280 151,
// 164, 182 and 199.  Eight waves: 54, 59, 68, 72 and 155, 174, 193, 208; two (four workgroups): 57, 63, 70, 75 and 153,
// 162, 177, 193; five steps ahead 60, 69, 77, 89 and 152, 167, 186, 222.
constexpr int rounds_of(int items) { return (items + PER_CU * CU_COUNT - 1) / (PER_CU * CU_COUNT); }
template <typename T, int NB, int GB, int DEPTH>
void launch_few(const Params& p, bool wide, hipStream_t s) {
  const int items = ((p.V + GROUP - 1) / GROUP + GB - 1) / GB, rounds = rounds_of(items);
  hipLaunchKernelGGL((head_kernel<T, NB, GB, DEPTH>), dim3((items + rounds - 1) / rounds), dim3(64 * SPLIT), 0, s, p, wide);
}
template <typename T>
void launch(const Params& p, hipStream_t s) {
  const bool wide = p.os * sizeof(T) % 16 == 0 && (uintptr_t)p.out % 16 == 0;
  const int groups = (p.V + GROUP - 1) / GROUP;
  // Groups of 64 rows by twos read the tokens' tiles half as often, if no workgroup gets more of them by it: 7168 -> 129280,
  // 48 tokens 198 -> 184 us, 64 tokens 210 -> 185 (bf16: 182 -> 173, 195 -> 177); 8192 -> 65536, 64 tokens 123 -> 110.  In short rows the
  // meeting of the waves' sums, two groups' at once, costs more: 2048 -> 129280, 48 tokens 57 -> 61.
  const bool pairs = p.K >= 4096 && 2 * rounds_of((groups + 1) / 2) <= rounds_of(groups);
  if (p.N <= 16) launch_few<T, 1, 1, 4>(p, wide, s);
  else if (p.N <= 32) launch_few<T, 2, 1, 4>(p, wide, s);
  else if (p.N <= 48) pairs ? launch_few<T, 3, 2, 3>(p, wide, s) : launch_few<T, 3, 1, 4>(p, wide, s);
  else if (p.N <= FEW) pairs ? launch_few<T, 4, 2, 2>(p, wide, s) : launch_few<T, 4, 1, 4>(p, wide, s);
  else {
    const dim3 grid((p.n_tb * p.ranges + 7) / 8 * 8);
    if (p.w1 == 1) hipLaunchKernelGGL((gemm_kernel<T, 1>), grid, dim3(NT), 0, s, p, wide);
    else if (p.w1 == 2) hipLaunchKernelGGL((gemm_kernel<T, 2>), grid, dim3(NT), 0, s, p, wide);
    else hipLaunchKernelGGL((gemm_kernel<T, 3>), grid, dim3(NT), 0, s, p, wide);
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
  hipLaunchKernelGGL(quantize_kernel<false>, quantize_grid(d->n_tokens), dim3(QUANT_NT), 0, s,
                     static_cast<const bf16_t*>(d->x), d->x_row_stride, d->n_tokens, d->hidden, q, K, ss, d->out_status);
  Params p{};
  p.w = d->w;
  p.ts = d->scales;
  p.q = q;
  p.ss = ss;
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
