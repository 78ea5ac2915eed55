// The gradient of an embedding table: out[v] = scale * sum of g[t] over the t with index v.
//
// The rows of the table that no token names are most of what has to be written, so the first launch clears the table
// while some of its workgroups sort the tokens (clearing is bound by memory, sorting by arithmetic and latency); the
// others add up the rows of g.  The launches:
//
//   sort   32 tokens a workgroup; a token's place among the 8192 of its tile is the number of smaller keys (index, then
//          position), counted by comparing with all of them from LDS: no passes, no exchange between workgroups, and
//          the same place every time.
//   merge  (more than one tile) the place among all tokens: the same count in the other tiles, by bisection.
//   sum    one wavefront per 512 columns of a window of places, added in float32 in their order.  A row whose tokens
//          lie in one window is done; what reaches beyond it is kept as a piece.
//   join   (more than one window) the pieces of rows that reach over several windows, in their order.
//
// 8192 tokens of a text in 50257x1024 (bf16): 21 + 11.5 + 6 us, where clearing alone takes 15 (6.8 TB/s) and sorting 12;
// 2048 in 128256x4096: 170 + 11 us, bound by clearing.  Windows of 8 places instead of 16: 9 us for the sums, 10 to join.
#include "nz_operators.h"

namespace {

constexpr uint32_t kTile = 8192;      // tokens that are compared with each other
constexpr uint32_t kTileBits = 13;
constexpr uint32_t kSorted = 32;      // tokens that a workgroup places
constexpr uint32_t kClear = 1 << 14;  // bytes a workgroup clears
constexpr uint32_t kBatch = 16;      // rows of g that a wavefront has on their way at a time

// A sorted token: its index (the number of rows if it takes no part) and where it stands.
struct Place {
  uint32_t row, token;
};

template <class Key>
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
  __shared__ __attribute__((aligned(32))) Key keys[kTile];
  __shared__ uint32_t smaller[8][64];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  const uint32_t block = blockIdx.x % (kTile / kSorted), base = blockIdx.x / (kTile / kSorted) * kTile;
  const uint32_t here = min(kTile, count - base), blocks = (here + 31) / 32;
  for (uint32_t i = threadIdx.x; i < blocks * 32; i += 512) {
    const long long v = i < here ? index[base + i] : -1;
    const uint32_t row = v >= 0 && v < (long long)rows && v != skip ? (uint32_t)v : rows;
    keys[i] = (Key)row << kTileBits | i;
  }
  __syncthreads();
  // the two halves of a wavefront hold the same tokens and look at another sixteenth of the keys each
  const uint32_t i = block * kSorted + lane % kSorted, part = wave * 2 + lane / kSorted;
  const Key mine = keys[i];
  uint32_t less = 0;
  const uint32_t first = blocks * part / 16, last = blocks * (part + 1) / 16;
  for (uint32_t b = first; b < last; ++b) {
#pragma unroll
    for (uint32_t j = 0; j < 32; j += 4) {
      const key4 k = *(const key4*)(keys + b * 32 + j);
      less += (k.x < mine) + (k.y < mine) + (k.z < mine) + (k.w < mine);
    }
  }
  smaller[wave][lane] = less;
  __syncthreads();
  if (threadIdx.x >= kSorted || i >= here) return;
  less = 0;
#pragma unroll
  for (uint32_t w = 0; w < 8; ++w) less += smaller[w][lane] + smaller[w][lane + kSorted];
  places[base + less] = Place{(uint32_t)(mine >> kTileBits), base + i};
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

__global__ __launch_bounds__(256) void nz_embedding_merge_kernel(const Place* tiles, uint32_t count, Place* places) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= count) return;
  const Place p = tiles[i];
  const uint32_t own = i / kTile * kTile;
  uint32_t at = i - own;
  for (uint32_t base = 0; base < count; base += kTile)  // equal ones of the tiles before stand before
    if (base != own) at += below(tiles + base, min(kTile, count - base), (uint64_t)p.row + (base < own));
  places[at] = p;
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
    typename Pack<T>::type v[kBatch];
    float w[kBatch][8];
#pragma unroll
    for (uint32_t j = 0; j < kBatch; ++j) {
      const T* row = g + __builtin_amdgcn_readlane(mine.token, j) * stride;
      if (k.whole)
        v[j] = *(const typename Pack<T>::type*)(row + k.c);
      else
        load8(row, k, cols, w[j]);
    }
#pragma unroll
    for (uint32_t j = 0; j < kBatch; ++j) {
      if (at + j >= end) break;
      const uint32_t row = __builtin_amdgcn_readlane(mine.row, j);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += k.whole ? (float)v[j][e] : w[j][e];
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

// One wavefront per 512 columns and window: the row that begins in it and goes on behind it, if there is one.
template <class T>
__global__ __launch_bounds__(256) void nz_embedding_join_kernel(const Place* places, uint32_t count, uint32_t rows,
                                                                uint32_t size, uint32_t cols, uint32_t slices,
                                                                float scale, uint32_t flags, T* out,
                                                                const float* pieces) {
  const uint64_t id = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64;
  const uint64_t window = id / slices, first = window * size, next = first + size;
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
  const Columns k = columns_of((uint32_t)(id - window * slices), lane, cols);
  float sum[8];
  load8(pieces + piece_at(window, 1, cols), k, cols, sum);
  for (uint32_t q = 1; q <= more; q += 16) {
    float v[16][8];
#pragma unroll
    for (uint32_t j = 0; j < 16; ++j)  // the last piece again where there are fewer
      load8(pieces + piece_at(window + min(q + j, more), 0, cols), k, cols, v[j]);
#pragma unroll
    for (uint32_t j = 0; j < 16; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] = q + j <= more ? sum[e] + v[j][e] : sum[e];
  }
  if (k.n) put8(out + row * (uint64_t)cols, k, cols, sum, tokens, scale, flags);
}

uint64_t align256(uint64_t v) { return (v + 255) / 256 * 256; }

// Places a window holds: few while there are few tokens, for the sake of many wavefronts.
uint32_t window_of(uint64_t count) { return count <= 32768 ? kBatch : 4 * kBatch; }

// Where the workspace holds what: sorted tiles (more than one), places, pieces.
struct Room {
  uint64_t places, pieces, bytes;
};
Room room_of(uint64_t count, uint64_t cols) {
  const uint64_t window = window_of(count);
  Room r;
  r.places = count > kTile ? align256(count * sizeof(Place)) : 0;
  r.pieces = r.places + align256(count * sizeof(Place));
  r.bytes = r.pieces + (count > window ? nz_mul(nz_ceil_div(count, window) * 2 * 4, cols) : 0);
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
  if (cols > 1u << 24 || rows > 0x7FFFFFFFull || count > 1u << 28 || count * slices > 1ull << 32)
    return nz_fail(NZ_ERR_ARG, "too many rows, columns or indices");
  if (!dev_out || (count && (!dev_indices || !dev_g))) return nz_fail(NZ_ERR_ARG, "null indices, gradient or output");
  if ((uintptr_t)dev_indices % 8 || (uintptr_t)dev_g % size || (uintptr_t)dev_out % size)
    return nz_fail(NZ_ERR_ALIGN, "pointers must be aligned to their elements");
  const Room room = room_of(count, cols);
  if (count) {
    if (workspace_bytes < room.bytes) return nz_fail(NZ_ERR_CAPACITY, "workspace too small");
    if (!dev_workspace || (uintptr_t)dev_workspace % 16) return nz_fail(NZ_ERR_ALIGN, "misaligned workspace");
  }
  const uint64_t bytes = flags & NZ_GRAD_ACCUMULATE ? 0 : rows * cols * size, clearers = nz_ceil_div(bytes, kClear);
  const uint32_t sorters = (uint32_t)nz_ceil_div(count, kSorted);
  if (clearers + sorters > 0x7FFFFFFFull) return nz_fail(NZ_ERR_ARG, "table too large for one launch");
  if (clearers + sorters == 0) return NZ_OK;
  const hipStream_t st = (hipStream_t)stream;
  uint8_t* ws = (uint8_t*)dev_workspace;
  Place *places = (Place*)(ws + room.places), *tiles = (Place*)ws;
  Place* sorted = count > kTile ? tiles : places;
  const dim3 grid((uint32_t)clearers + sorters);
  if (rows < 1u << (32 - kTileBits))
    nz_embedding_sort_kernel<uint32_t><<<grid, 512, 0, st>>>((const long long*)dev_indices, (uint32_t)count,
                                                             (uint32_t)rows, padding_idx, sorted, sorters,
                                                             (uint8_t*)dev_out, bytes);
  else
    nz_embedding_sort_kernel<uint64_t><<<grid, 512, 0, st>>>((const long long*)dev_indices, (uint32_t)count,
                                                             (uint32_t)rows, padding_idx, sorted, sorters,
                                                             (uint8_t*)dev_out, bytes);
  if (count > kTile)
    nz_embedding_merge_kernel<<<(uint32_t)nz_ceil_div(count, 256), 256, 0, st>>>(tiles, (uint32_t)count, places);
  if (count) {
    float* pieces = (float*)(ws + room.pieces);
    const uint32_t window = window_of(count);
    const uint32_t waves = (uint32_t)nz_ceil_div(nz_ceil_div(count, window) * slices, 4);
#define NZ_GRADIENT(T)                                                                                               \
  nz_embedding_sum_kernel<T><<<waves, 256, 0, st>>>(places, (uint32_t)count, (uint32_t)rows, window, (const T*)dev_g, \
                                                    stride, (uint32_t)cols, (uint32_t)slices, scale, flags,          \
                                                    (T*)dev_out, pieces);                                            \
  if (count > window)                                                                                                \
  nz_embedding_join_kernel<T><<<waves, 256, 0, st>>>(places, (uint32_t)count, (uint32_t)rows, window, (uint32_t)cols, \
                                                     (uint32_t)slices, scale, flags, (T*)dev_out, pieces)
    if (dtype == NZ_DTYPE_BF16) {
      NZ_GRADIENT(nz_bf16);
    } else if (dtype == NZ_DTYPE_F16) {
      NZ_GRADIENT(nz_f16);
    } else {
      NZ_GRADIENT(float);
    }
#undef NZ_GRADIENT
  }
  return nz_launched();
}

}  // extern "C"
