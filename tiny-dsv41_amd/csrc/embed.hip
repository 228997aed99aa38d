// embed.hip — rows of a table by token ids, scaled, and the gradient of the table.
//
//   out[n, :] = scale w[ids[n], :]                        (fp32 product, rounded once)
//   dw[v, :]  = scale sum over n with ids[n] = v of g[n, :]   (fp32 sums in the order of the batch)
//
// Negative ids are padding: rows of zeros, and no part in the gradient.
//
// The gradient in three kernels, none of which adds into memory that another writes, so its bits do not
// depend on the order in which workgroups run:
//   sort_kernel   the batch's positions ordered by (id, position).  A workgroup owns `range` ids and reads all
//                 ids of the batch (from its L2): it counts its own, wave by wave, and how many lie below
//                 its range, so it knows where its part of the sorted list begins without hearing from the
//                 others; then each wave places its tokens in their order.
//   sum_kernel    a wave takes a chunk of CHUNK positions of the sorted list and a strip of the columns: rows of
//                 g summed while the id stays the same.  An id whose tokens all lie within the chunk is
//                 finished there; one that reaches over its ends leaves a partial row.  Other workgroups
//                 of the same launch write zeros where no token is, which is most of a dense gradient's time.
//   join_kernel   the partial rows of an id that reaches over chunks, in their order.
// Bound by memory: a gradient of 151851 x 2048 in fp32 from 1000 tokens takes 7 + 177 + 4 us, 7.0 TB/s of zeros
// (by torch's fill 6.9); 129280 x 7168 in bf16 from 16384 tokens 14 + 342 + 11, 6.0 TB/s of zeros, gradients and partial
// rows.  Rows of the table, 16384 x 7168 in bf16, take 59 us: 7.9 TB/s of result and rows, of which frequent tokens' come
// from caches.

#include <math.h>

#include <algorithm>
#include <type_traits>

#include "row_scan.h"
#include "status.h"

namespace dsv41 {
namespace embed {

using rows::bf16_t;
using rows::Elem;

constexpr int COPY_NT = 256;
constexpr int SORT_NT = 1024, SORT_WAVES = SORT_NT / 64;
constexpr int RANGE_BITS = 9, RANGE = 1 << RANGE_BITS;  // ids of a sorting workgroup, at most
constexpr int ONE_BY_ONE = 3;  // of the ids among 64 tokens, of which few are the range's
constexpr int SUM_NT = 256, SUM_WAVES = SUM_NT / 64;
constexpr int CHUNK = 32;     // sorted positions of a summing wave
// A zeroing workgroup has about this many bytes, and those of an XCD a contiguous part of the table: 1.2 GB in 191 us,
// 195 and 206 with spans of 8, 16 and 32 KB, 219, 212 and 231 where the XCDs take spans in turn, 232 and 219 at 1 MB.
constexpr int ZERO_BYTES = 16384;
constexpr int JOIN_NT = 128;
constexpr int64_t MAX_GRID = 1 << 22;
constexpr int MAX_HIDDEN = 1 << 24;  // columns are counted in 32 bits, steps beyond the last one included

// 16 bytes of a row from p on, of which n elements exist (zeros beyond).
template <typename T>
__device__ __forceinline__ void load_raw(const T* p, int n, uint32_t (&w)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = 0;
  if (n >= Elem<T>::VEC) {
    rows::load16<false>(p, w);
  } else {
#pragma unroll
    for (int j = 0; j < Elem<T>::VEC; ++j)
      if (j < n) Elem<T>::put(w, j, p[j]);
  }
}
template <typename T>
__device__ __forceinline__ void load_group(const T* p, int n, float (&v)[Elem<T>::VEC]) {
  uint32_t w[4];
  load_raw(p, n, w);
  Elem<T>::unpack(w, v);
}

struct CopyParams {
  const void* w;
  int64_t ws;
  const int64_t* ids;
  int n, H, V;
  float scale;
  void* out;
  int64_t os;
  int32_t* status;
  int lanes;  // threads of a row, a power of two
};

template <typename T>
__global__ __launch_bounds__(COPY_NT) void copy_kernel(CopyParams p) {
  constexpr int G = Elem<T>::VEC;
  const int per = COPY_NT / p.lanes, lane = threadIdx.x % p.lanes;
  const int64_t n = (int64_t)blockIdx.x * per + threadIdx.x / p.lanes;
  if (n >= p.n) return;
  const int64_t id = p.ids[n];
  const bool bad = id >= p.V;
  if (p.status && lane == 0) p.status[n] = bad ? DSV41_STATUS_BAD_TARGET : 0;
  const float instead = bad ? __builtin_nanf("") : 0.f;
  const bool some = id >= 0 && !bad;
  const T* w = static_cast<const T*>(p.w) + (some ? id * p.ws : 0);
  T* out = static_cast<T*>(p.out) + n * p.os;
  constexpr int U = 4;
  if (p.H % G == 0) {  // U loads on their way together: a condition around a load has the wave wait for it
    for (int i0 = lane * G; i0 < p.H; i0 += U * p.lanes * G) {
      uint32_t raw[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) rows::load16<false>(w + min(i0 + u * p.lanes * G, p.H - G), raw[u]);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * p.lanes * G;
        float v[G];
        Elem<T>::unpack(raw[u], v);
#pragma unroll
        for (int j = 0; j < G; ++j) v[j] = some ? v[j] * p.scale : instead;
        if (i < p.H) rows::store_full(out + i, 0, v);
      }
    }
    return;
  }
  for (int i0 = lane * G; i0 < p.H; i0 += U * p.lanes * G) {
    float v[U][G];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * p.lanes * G;
      if (some && i < p.H) load_group(w + i, p.H - i, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * p.lanes * G;
      if (i >= p.H) break;
#pragma unroll
      for (int j = 0; j < G; ++j) v[u][j] = some ? v[u][j] * p.scale : instead;
      if (p.H - i >= G) {
        rows::store_full(out + i, 0, v[u]);
      } else {
#pragma unroll
        for (int j = 0; j < G; ++j)
          if (i + j < p.H) rows::store_one(out + i + j, v[u][j]);
      }
    }
  }
}

// word: 1, or 2 if some id is at or above V.
__global__ __launch_bounds__(status::NT) void check_ids_kernel(const int64_t* ids, int n, int V, int32_t* word) {
  const int bad = __syncthreads_or(status::any_of(ids, n, [=](int64_t id) { return id >= V; }));
  if (threadIdx.x == 0) __hip_atomic_store(word, bad ? 2 : 1, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_SYSTEM);
}

struct GradParams {
  const int64_t* ids;
  int n, H, V;
  const void* g;
  int64_t gs;
  float scale;
  void* out;
  int64_t os;
  int range, chunks, strips;
  int zero_rows;      // rows of the table of a zeroing workgroup: 1 .. 16, a power of two
  int64_t zero_grid;  // zeroing workgroups, a multiple of 8
  int32_t* total;     // [1] tokens with a row
  int32_t* place;     // [n] positions sorted by (id, position)
  int32_t* name;      // [n] their ids
  uint32_t* present;  // [(V + 31) / 32] ids that some token has
  float* part;        // [chunks, 2, H]: of the id that reaches into the chunk, and of the one that reaches beyond
};

// n elements from p on become 0: 16-byte stores from the first of their boundaries on, by the workgroup.
template <typename T>
__device__ __forceinline__ void clear_row(T* p, int64_t n) {
  constexpr int G = 16 / sizeof(T);
  const int tid = threadIdx.x, head = (int)min(n, (int64_t)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(T));
  if (tid < head) rows::store_one(p + tid, 0.f);
  uint4* q = reinterpret_cast<uint4*>(p + head);
  const int64_t groups = (n - head) / G;
  for (int64_t i = tid; i < groups; i += SUM_NT) q[i] = make_uint4(0, 0, 0, 0);
  const int64_t tail = head + groups * G + tid;
  if (tid < G && tail < n) rows::store_one(p + tail, 0.f);
}

__global__ __launch_bounds__(SORT_NT) void sort_kernel(GradParams p) {
  __shared__ uint32_t hist[SORT_WAVES][RANGE];
  __shared__ uint32_t sums[SORT_WAVES];
  constexpr int AHEAD = 8;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r0 = (int64_t)blockIdx.x * p.range;
  const uint64_t width = (uint64_t)min((int64_t)p.range, p.V - r0);
  const int per = ((p.n + SORT_WAVES - 1) / SORT_WAVES + 63) / 64 * 64;
  const int from = min(p.n, wave * per), to = min(p.n, from + per);
  for (int i = tid; i < SORT_WAVES * RANGE; i += SORT_NT) (&hist[0][0])[i] = 0;
  __syncthreads();
  uint32_t below = 0;
  for (int b = from; b < to; b += AHEAD * 64) {
    int64_t id[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) id[k] = b + k * 64 + lane < to ? p.ids[b + k * 64 + lane] : -1;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const uint64_t at = (uint64_t)(id[k] - r0);
      if (id[k] >= 0 && id[k] < r0) ++below;
      if (id[k] >= 0 && at < width) atomicAdd(&hist[wave][at], 1u);
    }
  }
  below = (uint32_t)wave_sum_i((int)below);
  if (lane == 0) sums[wave] = below;
  __syncthreads();
  uint32_t base = 0;
  for (int w = 0; w < SORT_WAVES; ++w) base += sums[w];
  __syncthreads();
  // starts: exclusive over (id, wave)
  uint32_t mine = 0;
  if (tid < RANGE)
    for (int w = 0; w < SORT_WAVES; ++w) mine += hist[w][tid];
  const uint32_t upto = wave_incl_scan_u32(mine);
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  uint32_t start = base + upto - mine;
  for (int w = 0; w < wave; ++w) start += sums[w];
  if (tid < RANGE) {
    uint32_t s = start;
    for (int w = 0; w < SORT_WAVES; ++w) {
      const uint32_t c = hist[w][tid];
      hist[w][tid] = s;
      s += c;
    }
    const uint64_t some = __ballot(mine != 0);
    const int64_t word = r0 / 32 + tid / 32;
    if ((tid & 31) == 0 && tid < p.range && word < ((int64_t)p.V + 31) / 32) p.present[word] = (uint32_t)(some >> (tid & 32));
    if (tid == RANGE - 1 && blockIdx.x == gridDim.x - 1) *p.total = (int32_t)s;
  }
  __syncthreads();
  for (int b0 = from; b0 < to; b0 += AHEAD * 64) {
    int64_t ids[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) ids[k] = b0 + k * 64 + lane < to ? p.ids[b0 + k * 64 + lane] : -1;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = b0 + k * 64 + lane;
      const uint64_t at = (uint64_t)(ids[k] - r0);
      const bool in = ids[k] >= 0 && at < width;
      uint64_t left = __ballot(in);
      // the tokens of these 64 that share an id take consecutive places: the first few ids one by one, as most ranges have
      // few tokens, or many of one
      const int turns = __popcll(left) > 16 ? 1 : ONE_BY_ONE;
      for (int t = 0; t < turns && left; ++t) {
        const int first = __builtin_ctzll(left);
        const uint32_t which = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)at, first);
        const uint64_t same = __ballot(in && (uint32_t)at == which) & left;
        uint32_t s = 0;
        if (lane == first) s = atomicAdd(&hist[wave][which], (uint32_t)__popcll(same));
        s = (uint32_t)__builtin_amdgcn_readlane((int)s, first);
        if (same >> lane & 1) {
          const uint32_t to_place = s + (uint32_t)__popcll(same & ((1ull << lane) - 1));
          p.place[to_place] = i;
          p.name[to_place] = (int32_t)ids[k];
        }
        left &= ~same;
      }
      if (left == 0) continue;
      // the others at once, found bit by bit of their id's place: a range of frequent tokens' ids, which often are the lowest,
      // has half of a batch (16384 tokens, ids log-uniform below 129280: 84 us one by one, about 20 so; alike in all ranges
      // 14, and 20 without any one by one)
      const bool mine = left >> lane & 1;
      uint64_t same = left;
#pragma unroll
      for (int bit = 0; bit < RANGE_BITS; ++bit) {
        const uint64_t set = __ballot(mine && (at >> bit & 1));
        same &= at >> bit & 1 ? set : ~set;
      }
      const int rank = __popcll(same & ((1ull << lane) - 1)), first = mine ? __builtin_ctzll(same) : lane;
      uint32_t s = 0;
      if (mine && rank == 0) s = atomicAdd(&hist[wave][at], (uint32_t)__popcll(same));
      s = (uint32_t)__shfl((int)s, first);
      if (mine) {
        p.place[s + rank] = i;
        p.name[s + rank] = (int32_t)ids[k];
      }
    }
  }
}

// G columns of a finished row, of which the first n exist; EARLY: `old` holds what was there.
template <typename T, bool ONTO, bool EARLY, int G>
__device__ __forceinline__ void finish(T* out, int n, const float (&s)[G], float scale, const uint32_t (&old)[4]) {
  constexpr int GO = Elem<T>::VEC;
  n = min(n, G);
#pragma unroll
  for (int b = 0; b < G; b += GO) {
    float v[GO];
    if (EARLY) Elem<T>::unpack(old, v);
    else if (ONTO) load_group(out + b, n - b, v);
#pragma unroll
    for (int j = 0; j < GO; ++j) {
      const float sum = b + j < G ? s[b + j < G ? b + j : 0] * scale : 0.f;
      v[j] = ONTO ? v[j] + sum : sum;
    }
    if (n - b >= GO) {
      rows::store_full(out + b, 0, v);
    } else {
#pragma unroll
      for (int j = 0; j < GO; ++j)
        if (b + j < n) rows::store_one(out + b + j, v[j]);
    }
  }
}

template <typename TG, typename TO, bool ONTO>
__global__ __launch_bounds__(SUM_NT) void sum_kernel(GradParams p) {
  constexpr int G = Elem<TG>::VEC;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  TO* out = static_cast<TO*>(p.out);
  const int64_t items = (int64_t)p.chunks * p.strips, sums = (items + SUM_WAVES - 1) / SUM_WAVES;
  if ((int64_t)blockIdx.x >= sums) {
    const int64_t z = (int64_t)blockIdx.x - sums, v0 = ((z & 7) * (p.zero_grid / 8) + (z >> 3)) * p.zero_rows;
    if (v0 >= p.V) return;
    const int rows_here = (int)min((int64_t)p.zero_rows, p.V - v0);
    const uint32_t there = p.present[v0 >> 5] >> (v0 & 31) & ((1u << p.zero_rows) - 1);
    if (there == 0 && p.os == p.H) {
      clear_row(out + v0 * p.os, (int64_t)rows_here * p.H);
    } else {
      for (int r = 0; r < rows_here; ++r)
        if (!(there >> r & 1)) clear_row(out + (v0 + r) * p.os, p.H);
    }
    return;
  }
  const int64_t item = (int64_t)blockIdx.x * SUM_WAVES + wave;
  const int total = *p.total;
  const int chunk = (int)(item / p.strips), strip = (int)(item % p.strips);
  const int c0 = chunk * CHUNK, count = min(CHUNK, total - c0);
  if (item >= items || count <= 0) return;
  // lane l: position and id of entry l; where its id ends, and whether the first one's began before
  const int at = min(c0 + lane, total - 1);
  const int place = p.place[at], name = p.name[at], after = p.name[min(at + 1, total - 1)];
  const bool last = name != after || at + 1 == total;
  const uint32_t ends = (uint32_t)__ballot(last);
  bool reaches_in = c0 > 0 && p.name[max(c0 - 1, 0)] == __builtin_amdgcn_readfirstlane(name);
  const int col = (strip * 64 + lane) * G, n = p.H - col;
  const TG* g = static_cast<const TG*>(p.g) + col;
  float s[G];
#pragma unroll
  for (int j = 0; j < G; ++j) s[j] = 0.f;
  constexpr int U = 16;  // rows in flight
  // Onto a gradient of the same type, finished ids' rows are read beside them: 16384 bf16 rows of 7168, all three kernels,
  // 111 us, 121 where each waits for its own (7027 ids, log-uniform and spread over 129280); uniform ids 158 and 170.
  constexpr bool EARLY = ONTO && std::is_same<TG, TO>::value;
#pragma unroll
  for (int c = 0; c < CHUNK; c += U) {
    uint32_t raw[U][4], old[EARLY ? U : 1][4];
    if (c >= count) break;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = __builtin_amdgcn_readlane(place, min(c + u, count - 1));
      if (n > 0) load_raw(g + row * p.gs, n, raw[u]);
    }
    if constexpr (EARLY) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c + u < count && (ends >> (c + u) & 1)) {
          const int64_t id = __builtin_amdgcn_readlane(name, c + u);
          if (n > 0) load_raw(out + id * p.os + col, n, old[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c + u >= count) break;
      float v[G];
      Elem<TG>::unpack(raw[u], v);
#pragma unroll
      for (int j = 0; j < G; ++j) s[j] += v[j];
      const bool done = ends >> (c + u) & 1;
      if (!done && c + u + 1 < count) continue;
      if (n > 0) {
        if (reaches_in || !done) {
          float* part = p.part + ((int64_t)chunk * 2 + (reaches_in ? 0 : 1)) * p.H + col;
#pragma unroll
          for (int j = 0; j < G; ++j)
            if (j < n) part[j] = s[j];
        } else {
          const int64_t id = __builtin_amdgcn_readlane(name, c + u);
          finish<TO, ONTO, EARLY>(out + id * p.os + col, n, s, p.scale, old[EARLY ? u : 0]);
        }
      }
      reaches_in = false;
#pragma unroll
      for (int j = 0; j < G; ++j) s[j] = 0.f;
    }
  }
}

template <typename TO, bool ONTO>
__global__ __launch_bounds__(JOIN_NT) void join_kernel(GradParams p) {
  constexpr int G = 4;
  const int total = *p.total;
  const int chunk = (int)(blockIdx.x / p.strips), strip = (int)(blockIdx.x % p.strips);
  const int c1 = (chunk + 1) * CHUNK;
  if (c1 >= total) return;
  const int id = p.name[c1];
  if (p.name[c1 - 1] != id) return;                                   // nothing reaches beyond this chunk,
  if (chunk > 0 && p.name[chunk * CHUNK] == id && p.name[chunk * CHUNK - 1] == id) return;  // or not from here
  const int col = (strip * JOIN_NT + threadIdx.x) * G;
  if (col >= p.H) return;
  const int n = min(G, p.H - col);
  const bool whole = p.H % G == 0;  // groups of 16 bytes, all of them
  auto row = [&](int64_t r, float (&v)[G]) {
    const float* part = p.part + r * p.H + col;
    if (whole) {
      const float4 w = *reinterpret_cast<const float4*>(part);
      v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
    } else {
#pragma unroll
      for (int j = 0; j < G; ++j) v[j] = part[min(j, n - 1)];
    }
  };
  float s[G];
  row((int64_t)chunk * 2 + 1, s);
  // the chunks that the id reaches into: names and rows of U of them at a time
  constexpr int U = 16;
  for (int c = chunk + 1;; c += U) {
    int name[U], more = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) name[u] = p.name[min((c + u) * CHUNK, total - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) more += more == u && (c + u) * CHUNK < total && name[u] == id;
    float v[U][G];
    // (most ids reach into few)
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u < more) row((int64_t)(c + u) * 2, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u < more) {
#pragma unroll
        for (int j = 0; j < G; ++j) s[j] += v[u][j];
      }
    if (more < U) break;
  }
  TO* out = static_cast<TO*>(p.out) + id * p.os + col;
#pragma unroll
  for (int j = 0; j < G; ++j)
    if (j < n) rows::store_one(out + j, ONTO ? Elem<TO>::one(out + j) + s[j] * p.scale : s[j] * p.scale);
}

int check_sizes(int dtype, int n, int h, int v) {
  if (n < 0 || h <= 0 || v <= 0) return fail(DSV41_E_INVALID, "the table must have shape [vocabulary_size, hidden]");
  if (dtype != DSV41_DTYPE_F32 && dtype != DSV41_DTYPE_BF16) return fail(DSV41_E_INVALID, "the table must be fp32 or bf16");
  if (h > MAX_HIDDEN) return fail(DSV41_E_UNSUPPORTED, "hidden sizes above 2^24 are not supported");
  return DSV41_OK;
}

struct Plan {
  int64_t range, ranges, chunks, strips, join_strips, zero_rows, zero_grid, sum_grid;
  size_t place, name, present, part, bytes;  // offsets into the workspace (the total is at its begin)
};

Plan plan(const dsv41_embed_grad_desc* d) {
  Plan q{};
  const int g = d->grad_dtype == DSV41_DTYPE_F32 ? 4 : 8;
  // a small vocabulary is cut finer, for as many workgroups as there are CUs
  q.range = RANGE;
  while (q.range > 32 && d->vocab < q.range * 256) q.range /= 2;
  q.ranges = (d->vocab + q.range - 1) / q.range;
  q.chunks = ((int64_t)d->n_tokens + CHUNK - 1) / CHUNK;
  q.strips = ((int64_t)d->hidden + 64 * g - 1) / (64 * g);
  q.join_strips = ((int64_t)d->hidden + JOIN_NT * 4 - 1) / (JOIN_NT * 4);
  q.zero_rows = 1;
  while (q.zero_rows < 16 && q.zero_rows * 2 * d->hidden * (d->out_dtype == DSV41_DTYPE_F32 ? 4 : 2) <= ZERO_BYTES) q.zero_rows *= 2;
  q.zero_grid = d->accumulate ? 0 : ((d->vocab + q.zero_rows - 1) / q.zero_rows + 7) / 8 * 8;
  q.sum_grid = (q.chunks * q.strips + SUM_WAVES - 1) / SUM_WAVES + q.zero_grid;
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  q.place = 256;
  q.name = q.place + up((size_t)d->n_tokens * 4);
  q.present = q.name + up((size_t)d->n_tokens * 4);
  q.part = q.present + up(((size_t)d->vocab + 31) / 32 * 4);
  q.bytes = q.part + (size_t)q.chunks * 2 * d->hidden * 4;
  return q;
}

int check_grad(const dsv41_embed_grad_desc* d) {
  if (!d) return fail(DSV41_E_INVALID, "embedding gradient descriptor is NULL");
  if (d->struct_size != sizeof(dsv41_embed_grad_desc))
    return fail(DSV41_E_ABI, "dsv41_embed_grad_desc size mismatch (rebuild the binding)");
  if (int rc = check_sizes(d->out_dtype, d->n_tokens, d->hidden, d->vocab)) return rc;
  if (int rc = check_sizes(d->grad_dtype, d->n_tokens, d->hidden, d->vocab)) return rc;
  if (!d->out || (d->n_tokens > 0 && (!d->ids || !d->grad))) return fail(DSV41_E_INVALID, "ids, grad and out are required");
  if (d->out_row_stride < d->hidden || (d->grad_row_stride != 0 && d->grad_row_stride < d->hidden))
    return fail(DSV41_E_INVALID, "embedding gradient: row strides must cover the rows");
  if ((uintptr_t)d->grad % (d->grad_dtype == DSV41_DTYPE_F32 ? 4 : 2) || (uintptr_t)d->out % (d->out_dtype == DSV41_DTYPE_F32 ? 4 : 2))
    return fail(DSV41_E_INVALID, "embedding gradient: operands are not aligned to their type");
  const Plan q = plan(d);
  if (q.chunks * q.join_strips > MAX_GRID || q.sum_grid > MAX_GRID || q.ranges >= MAX_GRID)
    return fail(DSV41_E_UNSUPPORTED, "embedding gradient: the batch is too large for one call");
  return DSV41_OK;
}

template <typename TG, typename TO, bool ONTO>
void launch(GradParams p, const Plan& q, hipStream_t s) {
  hipLaunchKernelGGL((sum_kernel<TG, TO, ONTO>), dim3((unsigned)q.sum_grid), dim3(SUM_NT), 0, s, p);
  if (q.chunks > 1) {
    p.strips = (int)q.join_strips;
    hipLaunchKernelGGL((join_kernel<TO, ONTO>), dim3((unsigned)((q.chunks - 1) * q.join_strips)), dim3(JOIN_NT), 0, s, p);
  }
}
template <typename TG, typename TO>
void launch(const GradParams& p, const Plan& q, bool onto, hipStream_t s) {
  onto ? launch<TG, TO, true>(p, q, s) : launch<TG, TO, false>(p, q, s);
}

}  // namespace embed
}  // namespace dsv41

using namespace dsv41;
using namespace dsv41::embed;

namespace {
int copy_params(const dsv41_embed_desc* d, CopyParams& p, int64_t& grid) {
  if (!d) return fail(DSV41_E_INVALID, "embedding descriptor is NULL");
  if (d->struct_size != sizeof(dsv41_embed_desc))
    return fail(DSV41_E_ABI, "dsv41_embed_desc size mismatch (rebuild the binding)");
  if (int rc = check_sizes(d->dtype, d->n_tokens, d->hidden, d->vocab)) return rc;
  const int unit = d->dtype == DSV41_DTYPE_F32 ? 4 : 2;
  if (!d->weight || (d->n_tokens > 0 && (!d->ids || !d->out))) return fail(DSV41_E_INVALID, "weight, ids and out are required");
  if (d->weight_row_stride < d->hidden || d->out_row_stride < d->hidden)
    return fail(DSV41_E_INVALID, "embedding: row strides must cover the rows");
  if ((uintptr_t)d->weight % unit || (uintptr_t)d->out % unit)
    return fail(DSV41_E_INVALID, "embedding: operands are not aligned to their type");
  p.w = d->weight;
  p.ws = d->weight_row_stride;
  p.ids = d->ids;
  p.n = d->n_tokens;
  p.H = d->hidden;
  p.V = d->vocab;
  p.scale = d->scale;
  p.out = d->out;
  p.os = d->out_row_stride;
  p.status = d->out_status;
  p.lanes = 1;
  while (p.lanes < COPY_NT && p.lanes * (16 / unit) < p.H) p.lanes *= 2;
  grid = ((int64_t)p.n * p.lanes + COPY_NT - 1) / COPY_NT;
  if (grid > MAX_GRID * 2) return fail(DSV41_E_UNSUPPORTED, "embedding: the batch is too large for one call");
  return DSV41_OK;
}
int copy(const CopyParams& p, int64_t grid, int dtype, hipStream_t s) {
  if (grid == 0) return DSV41_OK;
  if (dtype == DSV41_DTYPE_F32) hipLaunchKernelGGL(copy_kernel<float>, dim3((unsigned)grid), dim3(COPY_NT), 0, s, p);
  else hipLaunchKernelGGL(copy_kernel<rows::bf16_t>, dim3((unsigned)grid), dim3(COPY_NT), 0, s, p);
  DSV41_HIP_CHECK(hipGetLastError());
  return DSV41_OK;
}
}  // namespace

extern "C" int dsv41_embed_run(const dsv41_embed_desc* d, void* stream) {
  CopyParams p{};
  int64_t grid;
  if (int rc = copy_params(d, p, grid)) return rc;
  return copy(p, grid, d->dtype, static_cast<hipStream_t>(stream));
}

// The ids are looked at by a launch of its own before the rows, so that the host goes on while they are copied: with its
// gradient, 16384 rows of 7168 (bf16) take 471 us, and 518 where the host waits for the rows' statuses.
extern "C" int dsv41_embed_checked_run(const dsv41_embed_desc* d, int32_t* flags, void* stream) {
  CopyParams p{};
  int64_t grid;
  if (int rc = copy_params(d, p, grid)) return rc;
  if (!flags) return fail(DSV41_E_INVALID, "embedding: flags are required");
  if (grid == 0) return 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  __atomic_store_n(flags, 0, __ATOMIC_RELAXED);
  hipLaunchKernelGGL(check_ids_kernel, dim3(1), dim3(status::NT), 0, s, p.ids, p.n, p.V, flags);
  DSV41_HIP_CHECK(hipGetLastError());
  if (int rc = copy(p, grid, d->dtype, s)) return rc;
  int got;
  if (int rc = status::watch(flags, s, got)) return rc;
  return got - 1;
}

extern "C" size_t dsv41_embed_grad_workspace_bytes(const dsv41_embed_grad_desc* d) {
  return check_grad(d) ? 0 : plan(d).bytes;
}

extern "C" int dsv41_embed_grad_run(const dsv41_embed_grad_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_grad(d)) return rc;
  const Plan q = plan(d);
  if (!workspace || workspace_bytes < q.bytes || (uintptr_t)workspace % 16)
    return fail(DSV41_E_WORKSPACE, "embedding gradient workspace is missing, too small or not 16-byte aligned");
  char* ws = static_cast<char*>(workspace);
  GradParams p{};
  p.ids = d->ids;
  p.n = d->n_tokens;
  p.H = d->hidden;
  p.V = d->vocab;
  p.g = d->grad;
  p.gs = d->grad_row_stride;
  p.scale = d->scale;
  p.out = d->out;
  p.os = d->out_row_stride;
  p.range = (int)q.range;
  p.chunks = (int)q.chunks;
  p.strips = (int)q.strips;
  p.zero_rows = (int)q.zero_rows;
  p.zero_grid = q.zero_grid;
  p.total = reinterpret_cast<int32_t*>(ws);
  p.place = reinterpret_cast<int32_t*>(ws + q.place);
  p.name = reinterpret_cast<int32_t*>(ws + q.name);
  p.present = reinterpret_cast<uint32_t*>(ws + q.present);
  p.part = reinterpret_cast<float*>(ws + q.part);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool gf = d->grad_dtype == DSV41_DTYPE_F32, of = d->out_dtype == DSV41_DTYPE_F32, onto = d->accumulate != 0;
  hipLaunchKernelGGL(sort_kernel, dim3((unsigned)q.ranges), dim3(SORT_NT), 0, s, p);
  if (q.sum_grid > 0) {
    if (gf && of) launch<float, float>(p, q, onto, s);
    else if (gf) launch<float, rows::bf16_t>(p, q, onto, s);
    else if (of) launch<rows::bf16_t, float>(p, q, onto, s);
    else launch<rows::bf16_t, rows::bf16_t>(p, q, onto, s);
  }
  DSV41_HIP_CHECK(hipGetLastError());
  return DSV41_OK;
}
