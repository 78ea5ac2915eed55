// The gradient of an embedding table: out[v] = scale * sum of g[t] over the t with index v.
//
// The rows of the table that no token names are most of what has to be written, so the first launch clears the table
// while some of its workgroups sort the tokens (clearing is bound by memory, sorting by arithmetic and latency); the
// others add up the rows of g.  The launches:
//
//   sort   32 tokens a workgroup; a token's place among the up to 8192 of its tile is the number of smaller keys
//          (index, then position), counted by comparing with all of them from LDS: no passes, no exchange between
//          workgroups, and the same place every time.  Four tokens a lane, so that reading the keys does not take the
//          longest.
//   merge  (more than one tile) 8 or 16 sorted runs become one: the same count in the other runs, by bisection.
//   sum    one wavefront per 512 columns of a window of places, added in float32 in their order.  A row whose tokens
//          lie in one window is done; what reaches beyond it is kept as a piece.
//   join   the pieces of rows that reach over several windows, in their order.
//
// Few tokens are not sorted but compared with each other where they are added up.
//
// 8192 tokens of a text in 50257x1024 (bf16): 16.6 + 11 + 5 us, where clearing alone takes 15 (6.8 TB/s); 32768:
// 19 + 8 + 22 + 9.6; 2048 in 128256x4096: 167 + 15 + 5 us, bound by clearing.  Windows of 8 places instead of 16: 9 us
// for the sums, 10 to join.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "nz_operators.h"

namespace {

constexpr uint32_t kTile = 8192;      // tokens that are compared with each other, at most
constexpr uint32_t kTileBits = 13;
constexpr uint32_t kSorted = 32;      // tokens that a workgroup places
constexpr uint32_t kClear = 1 << 14;  // bytes a workgroup clears
constexpr uint32_t kBatch = 16;       // rows of g that a wavefront has on their way at a time
constexpr uint32_t kJoin = 4;         // wavefronts that join a row's pieces
constexpr uint32_t kFew = 2048;       // tokens that may go unsorted
constexpr uint32_t kFewWaves = 8;     // wavefronts that look for them: 2048 in 30000x512 13 us, by 4 14.5, by 16 19

// A sorted token: its index (the number of rows if it takes no part) and where it stands.
struct Place {
  uint32_t row, token;
};

template <class Key, uint32_t TILE>
__global__ __launch_bounds__(512) void nz_embedding_sort_kernel(const long long* index, uint32_t count, uint32_t rows,
                                                                long long skip, Place* places, uint32_t sorters,
                                                                uint8_t* out, uint64_t bytes) {
  if (blockIdx.x >= sorters) {  // clear
    typedef uint32_t word4 __attribute__((ext_vector_type(4)));
    const uint64_t head = min(bytes, (uint64_t)(-(uintptr_t)out & 15)), body = (bytes - head) / 16 * 16;
    const uint64_t from = (uint64_t)(blockIdx.x - sorters) * kClear;
    word4* q = (word4*)(out + head);
#pragma unroll
    for (uint32_t i = 0; i < kClear / (512 * 16); ++i) {
      const uint64_t at = from + (i * 512 + threadIdx.x) * 16;
      if (at < body) q[at / 16] = word4{0, 0, 0, 0};
    }
    if (from == 0 && threadIdx.x < 32) {  // what does not lie in whole words
      const uint64_t at = threadIdx.x < 16 ? threadIdx.x : head + body + threadIdx.x - 16;
      if (threadIdx.x < 16 ? at < head : at < bytes) out[at] = 0;
    }
    return;
  }
  typedef Key key4 __attribute__((ext_vector_type(4)));
  __shared__ __attribute__((aligned(32))) Key keys[TILE];
  __shared__ uint32_t smaller[8][kSorted];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  const uint32_t block = blockIdx.x % (TILE / kSorted), base = blockIdx.x / (TILE / kSorted) * TILE;
  const uint32_t here = min(TILE, count - base), rounds = (here + 255) / 256;
  long long value[TILE / 512];
#pragma unroll
  for (uint32_t j = 0; j < TILE / 512; ++j)  // all on their way at once
    if (j * 512 < here) value[j] = index[base + min(j * 512 + threadIdx.x, here - 1)];
#pragma unroll
  for (uint32_t j = 0; j < TILE / 512; ++j) {
    const uint32_t i = j * 512 + threadIdx.x;
    const long long v = i < here ? value[j] : -1;
    const uint32_t row = v >= 0 && v < (long long)rows && v != skip ? (uint32_t)v : rows;
    if (j * 512 < here) keys[i] = (Key)row << kTileBits | i;
  }
  __syncthreads();
  // a lane holds four of the tokens; eight lanes hold them all, and look at every 64th four of the keys
  key4 mine = *(const key4*)(keys + block * kSorted + lane % 8 * 4);
  uint32_t less[4] = {};
  for (uint32_t r = 0; r < rounds; ++r) {
    const key4 k = *(const key4*)(keys + r * 256 + wave * 32 + lane / 8 * 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) less[e] += (k.x < mine[e]) + (k.y < mine[e]) + (k.z < mine[e]) + (k.w < mine[e]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    less[e] += __shfl_xor(less[e], 8);
    less[e] += __shfl_xor(less[e], 16);
    less[e] += __shfl_xor(less[e], 32);
    if (lane < 8) smaller[wave][lane * 4 + e] = less[e];
  }
  __syncthreads();
  const uint32_t i = block * kSorted + threadIdx.x;
  if (threadIdx.x >= kSorted || i >= here) return;
  uint32_t at = 0;
#pragma unroll
  for (uint32_t w = 0; w < 8; ++w) at += smaller[w][threadIdx.x];
  places[base + at] = Place{(uint32_t)(keys[i] >> kTileBits), base + i};
}

// tokens of a sorted tile whose index is less than `row`
__device__ inline uint32_t below(const Place* tile, uint32_t n, uint64_t row) {
  uint32_t lo = 0;
  while (n) {
    const uint32_t half = n / 2;
    if (tile[lo + half].row < row)
      lo += half + 1, n -= half + 1;
    else
      n = half;
  }
  return lo;
}

// `fan` sorted runs of `run` places each become one: a place moves up by the number of places of the other runs that
// stand before it.  Eight lanes a place, each for every eighth run: a bisection is a chain of loads.
__global__ __launch_bounds__(256) void nz_embedding_merge_kernel(const Place* from, uint32_t count, uint32_t run,
                                                                 uint32_t fan, Place* to) {
  const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint32_t i = (uint32_t)min(id / 8, (uint64_t)count - 1), part = threadIdx.x & 7;
  const Place p = from[i];
  const uint64_t own = i / run * run, first = i / run / fan * fan * (uint64_t)run;
  const uint64_t end = min((uint64_t)count, first + fan * (uint64_t)run);
  uint32_t at = 0;
  for (uint64_t base = first + part * (uint64_t)run; base < end; base += 8 * (uint64_t)run)
    if (base != own)  // equal ones of the runs before stand before
      at += below(from + base, (uint32_t)min((uint64_t)run, count - base), (uint64_t)p.row + (base < own));
  at += __shfl_xor(at, 1);
  at += __shfl_xor(at, 2);
  at += __shfl_xor(at, 4);
  if (part == 0 && id / 8 < count) to[first + (i - own) + at] = p;
}

template <class T>
struct Pack {
  typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

// The 8 columns a lane works on: from `c` as loaded (all inside the row, or the row has fewer than 8), of which those
// from `from` on, `n` of them, are its own.  The last lane of a row whose width is no multiple of 8 begins earlier
// than its own columns do, so that every load is a whole one.
struct Columns {
  uint32_t c, from, n;
  bool whole;
};
__device__ inline Columns columns_of(uint32_t slice, uint32_t lane, uint32_t cols) {
  const uint32_t own = slice * 512 + lane * 8;
  Columns k;
  k.whole = cols >= 8;
  k.c = k.whole ? min(own, cols - 8) : 0;
  k.from = own - k.c;
  k.n = own < cols ? min(8u, cols - own) : 0;
  return k;
}

template <class T>
__device__ inline void load8(const T* row, const Columns& k, uint32_t cols, float (&v)[8]) {
  if (k.whole) {
    const typename Pack<T>::type a = *(const typename Pack<T>::type*)(row + k.c);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (uint32_t)i < cols ? (float)row[i] : 0.0f;
  }
}

template <class T>
__device__ inline void store8(T* row, const Columns& k, const float (&v)[8]) {
  if (k.n == 8) {
    typename Pack<T>::type a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = (T)v[i];
    *(typename Pack<T>::type*)(row + k.c) = a;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i >= (int)k.from && i < (int)(k.from + k.n)) row[k.c + i] = (T)v[i];
  }
}

// 8 sums of a row with `tokens` tokens into the table
template <class T>
__device__ inline void put8(T* row, const Columns& k, uint32_t cols, const float (&sum)[8], uint32_t tokens,
                            float scale, uint32_t flags) {
  const float f = flags & NZ_GRAD_BY_FREQUENCY ? scale / (float)tokens : scale;
  float v[8], old[8] = {};
  if (flags & NZ_GRAD_ACCUMULATE) load8(row, k, cols, old);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = old[i] + sum[i] * f;
  store8(row, k, v);
}

// Of a window, at most one row began before it (piece 0) and one begins in it and goes on behind it (piece 1).
__device__ inline uint64_t piece_at(uint64_t window, uint32_t which, uint32_t cols) {
  return (window * 2 + which) * cols;
}

template <class T>
__global__ __launch_bounds__(256) void nz_embedding_sum_kernel(const Place* places, uint32_t count, uint32_t rows,
                                                               uint32_t size, const T* g, uint64_t stride,
                                                               uint32_t cols, uint32_t slices, float scale,
                                                               uint32_t flags, T* out, float* pieces) {
  const uint64_t id = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64;
  const uint64_t window = id / slices, first = window * size;
  if (first >= count) return;
  const uint32_t lane = threadIdx.x & 63, end = (uint32_t)min((uint64_t)count, first + size);
  const Columns k = columns_of((uint32_t)(id - window * slices), lane, cols);
  float sum[8] = {};
  uint32_t tokens = 0;
  bool begun = first == 0 || places[first - 1].row != places[first].row;  // the row being added up: in this window
  for (uint32_t at = (uint32_t)first; at < end; at += kBatch) {
    // lanes 0 .. 15: the places of the batch; lanes 1 .. 16 look at the one behind each
    const Place mine = places[min(at + lane, count - 1)];
    typename Pack<T>::type v[kBatch];  // raw, for all to be on their way before the first is used
    if (k.whole) {
#pragma unroll
      for (uint32_t j = 0; j < kBatch; ++j)
        v[j] = *(const typename Pack<T>::type*)(g + __builtin_amdgcn_readlane(mine.token, j) * stride + k.c);
    } else {  // narrower than a load
#pragma unroll
      for (uint32_t j = 0; j < kBatch; ++j)
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e)
          v[j][e] = e < cols ? g[__builtin_amdgcn_readlane(mine.token, j) * stride + e] : (T)0;
    }
#pragma unroll
    for (uint32_t j = 0; j < kBatch; ++j) {
      if (at + j >= end) break;
      const uint32_t row = __builtin_amdgcn_readlane(mine.row, j);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += (float)v[j][e];
      ++tokens;
      const bool ends = at + j + 1 == count || __builtin_amdgcn_readlane(mine.row, j + 1) != row;
      if (!ends && at + j + 1 < end) continue;
      if (row != rows && k.n) {
        if (begun && ends)
          put8(out + row * (uint64_t)cols, k, cols, sum, tokens, scale, flags);
        else
          store8(pieces + piece_at(window, begun, cols), k, sum);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] = 0;
      tokens = 0;
      begun = true;
    }
  }
}

// One workgroup per 512 columns and window: the row that begins in it and goes on behind it, if there is one.  Its
// pieces are many where a row has many tokens (those that fill up a batch): the wavefronts take a part each.  32768
// tokens, half of them the same: 18 us, 57 by one wavefront; eight are faster there, but take 13 instead of
// 9.6 us for a text.
template <class T>
__global__ __launch_bounds__(64 * kJoin) void nz_embedding_join_kernel(const Place* places, uint32_t count,
                                                                       uint32_t rows, uint32_t size, uint32_t cols,
                                                                       uint32_t slices, float scale, uint32_t flags,
                                                                       T* out, const float* pieces) {
  __shared__ float sums[kJoin - 1][64][9];  // a ninth: lanes apart in their banks
  const uint32_t window = blockIdx.x / slices, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint64_t first = (uint64_t)window * size, next = first + size;
  if (next >= count) return;
  // the places around the window's borders, asked for together
  const uint32_t lane = threadIdx.x & 63, row = places[next - 1].row, behind = places[next].row;
  const uint32_t begin = places[first].row, before = places[first ? first - 1 : 0].row;
  if (row == rows || behind != row) return;
  if (first && begin == row && before == row) return;  // it began before
  uint32_t more = 0;  // windows that it goes on in
  for (;;) {
    const uint64_t at = next + (uint64_t)(more + lane) * size;
    const uint64_t other = __ballot(at >= count || places[min(at, (uint64_t)count - 1)].row != row);
    if (other) {
      more += __builtin_ctzll(other);
      break;
    }
    more += 64;
  }
  uint32_t tokens = 1;
  if (flags & NZ_GRAD_BY_FREQUENCY) {
    tokens = (more - 1) * size;
    for (uint32_t i = 0; i < size; i += 64) {  // of the first window and of the last one
      tokens += __popcll(__ballot(i + lane < size && places[first + min(i + lane, size - 1)].row == row));
      const uint64_t at = next + (uint64_t)(more - 1) * size + i + lane;
      tokens += __popcll(__ballot(i + lane < size && at < count && places[min(at, (uint64_t)count - 1)].row == row));
    }
  }
  const Columns k = columns_of(blockIdx.x - window * slices, lane, cols);
  const uint32_t share = more <= 16 ? 16 : (more + kJoin - 1) / kJoin, begins = 1 + wave * share;
  const uint32_t last = min(more, begins + share - 1);
  float sum[8] = {};
  if (wave == 0) load8(pieces + piece_at(window, 1, cols), k, cols, sum);
  for (uint32_t q = begins; q <= last; q += 16) {
    Pack<float>::type v[16];
    const auto piece = [&](uint32_t j) {  // the last one again where there are fewer
      return pieces + piece_at(window + min(q + j, last), 0, cols);
    };
    if (k.whole) {
#pragma unroll
      for (uint32_t j = 0; j < 16; ++j) v[j] = *(const Pack<float>::type*)(piece(j) + k.c);
    } else {
#pragma unroll
      for (uint32_t j = 0; j < 16; ++j)
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) v[j][e] = e < cols ? piece(j)[e] : 0.0f;
    }
#pragma unroll
    for (uint32_t j = 0; j < 16; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] = q + j <= last ? sum[e] + v[j][e] : sum[e];
  }
  if (more > 16) {
    if (wave)
#pragma unroll
      for (int e = 0; e < 8; ++e) sums[wave - 1][lane][e] = sum[e];
    __syncthreads();
    if (wave == 0)
#pragma unroll
      for (uint32_t w = 0; w < kJoin - 1; ++w)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += sums[w][lane][e];
  }
  if (wave == 0 && k.n) put8(out + row * (uint64_t)cols, k, cols, sum, tokens, scale, flags);
}

// Few tokens, without sorting them: one workgroup per 512 columns of a token looks for the token's index among all of
// them, a part a wavefront.  Where it is the first of its row it adds up the row, again a part a wavefront if there are
// many, in their order; else it is done.
template <class T>
__global__ __launch_bounds__(64 * kFewWaves) void nz_embedding_few_kernel(const long long* index, uint32_t count,
                                                                          uint32_t rows, long long skip, const T* g,
                                                                          uint64_t stride, uint32_t cols,
                                                                          uint32_t slices, float scale, uint32_t flags,
                                                                          T* out) {
  constexpr uint32_t W = kFewWaves, kPart = kFew / W;
  __shared__ uint32_t found[W];
  __shared__ uint16_t list[kFew];
  __shared__ float sums[W - 1][64][9];  // a ninth: lanes apart in their banks
  const uint32_t token = blockIdx.x / slices, lane = threadIdx.x & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const long long row = index[token];
  if (row < 0 || row >= (long long)rows || row == skip) return;
  bool hit[kPart / 64];
#pragma unroll
  for (uint32_t j = 0; j < kPart / 64; ++j) {
    const uint32_t at = wave * kPart + j * 64 + lane;
    hit[j] = index[min(at, count - 1)] == row && at < count;
  }
  uint32_t n = 0;
  bool earlier = false;
#pragma unroll
  for (uint32_t j = 0; j < kPart / 64; ++j) {
    const uint64_t mask = __ballot(hit[j]);
    earlier |= mask && wave * kPart + j * 64 + __builtin_ctzll(mask) < token;
    n += __popcll(mask);
  }
  if (lane == 0) found[wave] = earlier ? ~0u : n;
  __syncthreads();
  uint32_t to = 0;
  n = 0;
#pragma unroll
  for (uint32_t w = 0; w < W; ++w) {
    const uint32_t of = __builtin_amdgcn_readfirstlane(found[w]);
    if (of == ~0u) return;
    if (w == wave) to = n;
    n += of;
  }
#pragma unroll
  for (uint32_t j = 0; j < kPart / 64; ++j) {
    const uint64_t mask = __ballot(hit[j]);
    if (hit[j]) list[to + __popcll(mask & ((1ull << lane) - 1))] = (uint16_t)(wave * kPart + j * 64 + lane);
    to += __popcll(mask);
  }
  __syncthreads();
  const uint32_t share = n <= 16 ? 16 : (n + W - 1) / W, first = min(n, wave * share), last = min(n, first + share);
  const Columns k = columns_of(blockIdx.x - token * slices, lane, cols);
  float sum[8] = {};
  const auto row_at = [&](uint32_t i) {
    return g + (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)list[min(i, last - 1)]) * stride;
  };
  const auto add = [&](uint32_t i, auto size) {  // `size` tokens from i on, all on their way before the first is used
    constexpr uint32_t N = decltype(size)::value;
    typename Pack<T>::type v[N];
#pragma unroll
    for (uint32_t j = 0; j < N; ++j) v[j] = *(const typename Pack<T>::type*)(row_at(i + j) + k.c);
#pragma unroll
    for (uint32_t j = 0; j < N; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] = i + j < last ? sum[e] + (float)v[j][e] : sum[e];
    return i + N;
  };
  for (uint32_t i = first; i < last && !k.whole; ++i) {  // narrower than a load
    float v[8];
    load8(row_at(i), k, cols, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += v[e];
  }
  for (uint32_t i = first; i < last && k.whole;) {
    if (last - i > 4)
      i = add(i, std::integral_constant<uint32_t, 16>());
    else if (last - i > 1)
      i = add(i, std::integral_constant<uint32_t, 4>());
    else
      i = add(i, std::integral_constant<uint32_t, 1>());
  }
  if (n > 16) {
    if (wave)
#pragma unroll
      for (int e = 0; e < 8; ++e) sums[wave - 1][lane][e] = sum[e];
    __syncthreads();
    if (wave == 0)
#pragma unroll
      for (uint32_t w = 0; w < W - 1; ++w)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += sums[w][lane][e];
  }
  if (wave == 0 && k.n) put8(out + (uint64_t)row * cols, k, cols, sum, n, scale, flags);
}

uint64_t align256(uint64_t v) { return (v + 255) / 256 * 256; }

// Places a window holds: few while there are few tokens, for the sake of many wavefronts, more for the sake of fewer
// pieces.  50257x1024, windows of 16, 32 and 64: 8192 tokens 33, 37, 49 us; 24000 68, 61, 69; 50000 117, 108, 103.
uint32_t window_of(uint64_t count) {
  return count <= 16384 ? kBatch : count <= 32768 ? 2 * kBatch : 4 * kBatch;
}

// Whether tokens are few enough to be compared with each other for each 512 columns; what that reads is 8 count^2
// slices bytes.  (On the device, bf16, against sorting: 30000x512, 1440 tokens 12 and 19 us, 2048 13 and 20, 4096 21
// and 21; 8000x256, 2048 9 and 17; where half of 2048 tokens are the same 26 and 22; 32000x4096, 1440 73 and 50.)
bool unsorted(uint64_t count, uint64_t cols) {
  return count <= kFew && count * count * nz_ceil_div(cols, 512) <= (uint64_t)kFew * kFew;
}

// Tokens that are sorted among each other: up to 8192 need no second launch; above, comparing takes count x tile steps.
uint32_t tile_of(uint64_t count) { return count <= kTile ? kTile : kTile / 4; }

// Where the workspace holds what: places, once more (if runs of them are merged), pieces.
struct Room {
  uint64_t again, pieces, bytes;
};
Room room_of(uint64_t count, uint64_t cols) {
  const uint64_t window = window_of(count);
  Room r = {};
  if (unsorted(count, cols)) return r;
  r.again = align256(count * sizeof(Place));
  r.pieces = count > kTile ? 2 * r.again : r.again;
  r.bytes = r.pieces + nz_mul(nz_ceil_div(count, window) * 2 * 4, cols);
  return r;
}

}  // namespace

extern "C" {

uint64_t nz_embedding_gradient_workspace_bytes(uint64_t count, uint64_t cols) {
  return count && cols ? room_of(count, cols).bytes : 0;
}

int nz_embedding_gradient(const void* dev_indices, uint64_t count, const void* dev_g, int dtype, uint64_t stride,
                          uint64_t rows, uint64_t cols, float scale, int64_t padding_idx, uint32_t flags,
                          void* dev_out, void* dev_workspace, uint64_t workspace_bytes, void* stream) {
  const uint32_t size = nz_dtype_bytes(dtype);
  if (!size) return nz_fail(NZ_ERR_DTYPE, "Unsupported data type");
  if (flags & ~(NZ_GRAD_BY_FREQUENCY | NZ_GRAD_ACCUMULATE)) return nz_fail(NZ_ERR_ARG, "unknown flags");
  if (rows == 0 || cols == 0) return NZ_OK;
  const uint64_t slices = nz_ceil_div(cols, 512);
  // of the last two launches, which are counted in pieces of windows, and of the sort
  if (cols > 1u << 24 || rows > 0x7FFFFFFFull || count > nz_most_groups(512) * kSorted ||
      (!unsorted(count, cols) && nz_ceil_div(count, window_of(count)) * slices > nz_most_groups(64 * kJoin)))
    return nz_fail(NZ_ERR_ARG, "too many rows, columns or indices");
  if (!dev_out || (count && (!dev_indices || !dev_g))) return nz_fail(NZ_ERR_ARG, "null indices, gradient or output");
  if ((uintptr_t)dev_indices % 8 || (uintptr_t)dev_g % size || (uintptr_t)dev_out % size)
    return nz_fail(NZ_ERR_ALIGN, "pointers must be aligned to their elements");
  const Room room = room_of(count, cols);
  if (room.bytes) {
    if (workspace_bytes < room.bytes) return nz_fail(NZ_ERR_CAPACITY, "workspace too small");
    if (!dev_workspace || (uintptr_t)dev_workspace % 16) return nz_fail(NZ_ERR_ALIGN, "misaligned workspace");
  }
  const uint64_t bytes = flags & NZ_GRAD_ACCUMULATE ? 0 : rows * cols * size;
  const bool few = unsorted(count, cols);
  const uint32_t sorters = few ? 0 : (uint32_t)nz_ceil_div(count, kSorted);
  const hipStream_t st = (hipStream_t)stream;
  uint8_t* ws = (uint8_t*)dev_workspace;
  Place *places = (Place*)ws, *other = (Place*)(ws + room.again);
  const uint32_t tile = tile_of(count);
  const auto sort = [&](auto key, auto size) {
    constexpr uint32_t TILE = decltype(size)::value;
    // the sort and what a launch holds of the clearing besides; the rest of tables beyond 137 GB in further launches
    uint64_t done = 0;
    for (uint32_t sorting = sorters; sorting || done < bytes; sorting = 0) {
      const uint64_t clearers = std::min(nz_ceil_div(bytes - done, kClear), nz_most_groups(512) - sorting);
      const uint64_t now = std::min(bytes - done, clearers * kClear);
      nz_embedding_sort_kernel<decltype(key), TILE><<<(uint32_t)clearers + sorting, 512, 0, st>>>(
          (const long long*)dev_indices, (uint32_t)count, (uint32_t)rows, padding_idx, places, sorting,
          (uint8_t*)dev_out + done, now);
      done += now;
    }
  };
  const auto sort_by = [&](auto key) {
    if (tile == kTile)
      sort(key, std::integral_constant<uint32_t, kTile>());
    else
      sort(key, std::integral_constant<uint32_t, kTile / 4>());
  };
  if (rows < 1u << (32 - kTileBits)) {
    sort_by(uint32_t());
  } else {
    sort_by(uint64_t());
  }
  // 16 runs at a time if that ends it: 51 us for 262144 places, 28 + 28 in two passes of 8 and 2
  for (uint64_t run = tile; !few && run < count;) {
    const uint32_t fan = nz_ceil_div(count, run) <= 16 ? 16 : 8;
    nz_embedding_merge_kernel<<<(uint32_t)nz_ceil_div(count, 32), 256, 0, st>>>(places, (uint32_t)count, (uint32_t)run,
                                                                               fan, other);
    std::swap(places, other);
    run *= fan;
  }
  const auto add_up = [&](auto type) {
    using T = decltype(type);
    const T* g = (const T*)dev_g;
    T* out = (T*)dev_out;
    if (few) {
      nz_embedding_few_kernel<T><<<(uint32_t)(count * slices), 64 * kFewWaves, 0, st>>>(
          (const long long*)dev_indices, (uint32_t)count, (uint32_t)rows, padding_idx, g, stride, (uint32_t)cols,
          (uint32_t)slices, scale, flags, out);
      return;
    }
    float* pieces = (float*)(ws + room.pieces);
    const uint32_t window = window_of(count);
    const uint32_t waves = (uint32_t)nz_ceil_div(nz_ceil_div(count, window) * slices, 4);
    nz_embedding_sum_kernel<T><<<waves, 256, 0, st>>>(places, (uint32_t)count, (uint32_t)rows, window, g, stride,
                                                      (uint32_t)cols, (uint32_t)slices, scale, flags, out, pieces);
    nz_embedding_join_kernel<T><<<(uint32_t)(nz_ceil_div(count, window) * slices), 64 * kJoin, 0, st>>>(
        places, (uint32_t)count, (uint32_t)rows, window, (uint32_t)cols, (uint32_t)slices, scale, flags, out, pieces);
  };
  if (count == 0) {
  } else if (dtype == NZ_DTYPE_BF16) {
    add_up(nz_bf16());
  } else if (dtype == NZ_DTYPE_F16) {
    add_up(nz_f16());
  } else {
    add_up(float());
  }
  return nz_launched();
}

}  // extern "C"
