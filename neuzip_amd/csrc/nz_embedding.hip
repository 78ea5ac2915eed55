// The gradient of an embedding table: out[v] = scale * sum of g[t] over the t with index v.
//
// The rows of the table that no token names are most of what has to be written, so the first launch clears the table
// while some of its workgroups sort the tokens (clearing is bound by memory, sorting by arithmetic and latency); the
// second adds up the rows of g.  Its launches:
//
//   sort   64 tokens a workgroup; a token's place among the 8192 of its tile is the number of smaller indices plus that
//          of equal ones before it, counted by comparing with all of them from LDS: no passes, no exchange between
//          workgroups, and the same place every time.
//   merge  (more than one tile) the place among all tokens: the same counts in the other tiles, by bisection.
//   sum    one wavefront per 512 columns of up to 64 tokens of a row, in their order, in float32.
//   join   (more than 64 tokens) the pieces of rows with more than 64 tokens, in their order.
#include "nz_operators.h"

namespace {

constexpr uint32_t kTile = 8192;     // tokens that are compared with each other
constexpr uint32_t kPiece = 64;      // tokens that one wavefront adds up
constexpr uint32_t kNone = ~0u;      // the index of a token that takes no part
constexpr uint32_t kClear = 1 << 16; // bytes a workgroup clears

// A token in its place: index, token, tokens of the same index before it, tokens of this index.
typedef uint32_t Place __attribute__((ext_vector_type(4)));

__global__ __launch_bounds__(512) void nz_embedding_sort_kernel(const long long* index, uint32_t count, uint64_t rows,
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
      if (at < body) __builtin_nontemporal_store(word4{0, 0, 0, 0}, q + at / 16);
    }
    if (from == 0 && threadIdx.x < 32) {  // what does not lie in whole words
      const uint64_t at = threadIdx.x < 16 ? threadIdx.x : head + body + threadIdx.x - 16;
      if (threadIdx.x < 16 ? at < head : at < bytes) out[at] = 0;
    }
    return;
  }
  __shared__ __attribute__((aligned(16))) uint32_t keys[kTile];
  __shared__ uint32_t smaller[8][64], equal[8][64], before[8][64];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  const uint32_t block = blockIdx.x % (kTile / 64), base = blockIdx.x / (kTile / 64) * kTile;
  const uint32_t here = min(kTile, count - base), blocks = (here + 63) / 64;
  for (uint32_t i = threadIdx.x; i < blocks * 64; i += 512) {
    const long long v = i < here ? index[base + i] : -1;
    keys[i] = v >= 0 && (uint64_t)v < rows && v != skip ? (uint32_t)v : kNone;
  }
  __syncthreads();
  const uint32_t mine = keys[block * 64 + lane];
  uint32_t lt = 0, eq = 0, eqb = 0;
  const uint32_t first = blocks * wave / 8, last = blocks * (wave + 1) / 8;
  for (uint32_t b = first; b < last; ++b) {
    const uint32_t* p = keys + b * 64;
    if (b == block) {
      eqb = eq;
      for (uint32_t j = 0; j < 64; ++j) {
        const bool e = p[j] == mine;
        lt += p[j] < mine;
        eq += e;
        eqb += e && j < lane;
      }
    } else {
#pragma unroll
      for (uint32_t j = 0; j < 64; j += 4) {
        const Place k = *(const Place*)(p + j);
        lt += (k.x < mine) + (k.y < mine) + (k.z < mine) + (k.w < mine);
        eq += (k.x == mine) + (k.y == mine) + (k.z == mine) + (k.w == mine);
      }
    }
  }
  if (last <= block) eqb = eq;
  smaller[wave][lane] = lt, equal[wave][lane] = eq, before[wave][lane] = eqb;
  __syncthreads();
  if (wave || block * 64 + lane >= here) return;
  lt = eq = eqb = 0;
  for (uint32_t w = 0; w < 8; ++w) lt += smaller[w][lane], eq += equal[w][lane], eqb += before[w][lane];
  places[base + lt + eqb] = Place{mine, base + block * 64 + lane, eqb, eq};
}

// tokens of a sorted tile whose index is less than `key`
__device__ inline uint32_t below(const Place* tile, uint32_t n, uint64_t key) {
  uint32_t lo = 0;
  while (n) {
    const uint32_t half = n / 2;
    if (tile[lo + half].x < key)
      lo += half + 1, n -= half + 1;
    else
      n = half;
  }
  return lo;
}

__global__ __launch_bounds__(256) void nz_embedding_merge_kernel(const Place* tiles, uint32_t count, Place* places) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= count) return;
  Place p = tiles[i];
  uint32_t at = i % kTile;
  for (uint32_t base = 0; base < count; base += kTile) {
    if (base == i / kTile * kTile) continue;
    const uint32_t n = min(kTile, count - base);
    const uint32_t lt = below(tiles + base, n, p.x), eq = below(tiles + base, n, (uint64_t)p.x + 1) - lt;
    at += lt;
    p.w += eq;
    if (base < i) at += eq, p.z += eq;
  }
  places[at] = p;
}

template <class T>
struct Pack {
  typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

template <class T>
__device__ inline void add8(const T* p, uint32_t n, float (&sum)[8]) {
  if (n >= 8) {
    const typename Pack<T>::type v = *(const typename Pack<T>::type*)p;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += (float)v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((uint32_t)i < n) sum[i] += (float)p[i];
  }
}

// 8 sums of a row with `tokens` tokens into the table
template <class T>
__device__ inline void put8(T* q, uint32_t n, const float (&sum)[8], uint32_t tokens, float scale, uint32_t flags) {
  const float f = flags & NZ_GRAD_BY_FREQUENCY ? scale / (float)tokens : scale;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = sum[i] * f;
  if (flags & NZ_GRAD_ACCUMULATE) add8(q, n, v);
  if (n >= 8) {
    typename Pack<T>::type a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = (T)v[i];
    *(typename Pack<T>::type*)q = a;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((uint32_t)i < n) q[i] = (T)v[i];
  }
}

// Where a piece that begins at place i is kept: of the places i / 64 * 64 .. + 63, at most one begins a row of more
// than 64 tokens, and at most one a later piece of such a row.
__device__ inline uint64_t piece_at(uint32_t i, uint32_t before) { return (uint64_t)(i / kPiece) * 2 + (before == 0); }

template <class T>
__global__ __launch_bounds__(256) void nz_embedding_sum_kernel(const Place* places, uint32_t count, const T* g,
                                                               uint64_t stride, uint32_t cols, uint32_t slices,
                                                               float scale, uint32_t flags, T* out, float* pieces) {
  const uint64_t id = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64;
  const uint32_t i = (uint32_t)(id / slices), lane = threadIdx.x & 63;
  if (i >= count) return;
  const Place p = places[i];
  if (p.x == kNone || p.z % kPiece) return;
  const uint32_t c = (uint32_t)(id % slices) * 512 + lane * 8;
  const uint32_t n = c < cols ? cols - c : 0, tokens = min(kPiece, p.w - p.z);
  const uint32_t token = places[min(i + lane, count - 1)].y;
  float sum[8] = {};
  uint32_t t = 0;
  for (; t + 8 <= tokens; t += 8) {  // eight rows on their way at a time, added one after the other
    float v[8][8] = {};
#pragma unroll
    for (int j = 0; j < 8; ++j) add8(g + __builtin_amdgcn_readlane(token, t + j) * stride + c, n, v[j]);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += v[j][e];
  }
  for (; t < tokens; ++t) add8(g + __builtin_amdgcn_readlane(token, t) * stride + c, n, sum);
  if (p.w <= kPiece) {
    if (n) put8(out + p.x * (uint64_t)cols + c, n, sum, p.w, scale, flags);
  } else {
    float* q = pieces + piece_at(i, p.z) * cols + c;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if ((uint32_t)e < n) q[e] = sum[e];
  }
}

// One wavefront per 512 columns and 64 places: at most one row of more than 64 tokens begins there.
template <class T>
__global__ __launch_bounds__(256) void nz_embedding_join_kernel(const Place* places, uint32_t count, uint32_t cols,
                                                                uint32_t slices, float scale, uint32_t flags, T* out,
                                                                const float* pieces) {
  const uint64_t id = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64;
  const uint64_t from = id / slices * kPiece;
  const uint32_t lane = threadIdx.x & 63;
  if (from >= count) return;
  const Place mine = places[min((uint32_t)from + lane, count - 1)];
  const uint64_t heads = __ballot(from + lane < count && mine.x != kNone && mine.z == 0 && mine.w > kPiece);
  if (!heads) return;
  const uint32_t i = (uint32_t)from + __builtin_ctzll(heads);
  const Place p = places[i];
  const uint32_t c = (uint32_t)(id % slices) * 512 + lane * 8;
  if (c >= cols) return;
  float sum[8] = {};
  for (uint32_t t = 0; t < p.w; t += kPiece) add8(pieces + piece_at(i + t, t) * cols + c, cols - c, sum);
  put8(out + p.x * (uint64_t)cols + c, cols - c, sum, p.w, scale, flags);
}

uint64_t align256(uint64_t v) { return (v + 255) / 256 * 256; }

// Where the workspace holds what: sorted tiles (more than one), places, pieces.
struct Room {
  uint64_t places, pieces, bytes;
};
Room room_of(uint64_t count, uint64_t cols) {
  Room r;
  r.places = count > kTile ? align256(count * sizeof(Place)) : 0;
  r.pieces = r.places + align256(count * sizeof(Place));
  r.bytes = r.pieces + (count > kPiece ? nz_mul(nz_ceil_div(count, kPiece) * 2 * 4, cols) : 0);
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
  const uint32_t sorters = (uint32_t)nz_ceil_div(count, 64);
  if (clearers + sorters > 0x7FFFFFFFull) return nz_fail(NZ_ERR_ARG, "table too large for one launch");
  if (clearers + sorters == 0) return NZ_OK;
  const hipStream_t st = (hipStream_t)stream;
  uint8_t* ws = (uint8_t*)dev_workspace;
  Place *places = (Place*)(ws + room.places), *tiles = (Place*)ws;
  nz_embedding_sort_kernel<<<(uint32_t)clearers + sorters, 512, 0, st>>>(
      (const long long*)dev_indices, (uint32_t)count, rows, padding_idx, count > kTile ? tiles : places, sorters,
      (uint8_t*)dev_out, bytes);
  if (count > kTile)
    nz_embedding_merge_kernel<<<(uint32_t)nz_ceil_div(count, 256), 256, 0, st>>>(tiles, (uint32_t)count, places);
  if (count) {
    float* pieces = (float*)(ws + room.pieces);
    const uint32_t sums = (uint32_t)nz_ceil_div(count * slices, 4);
    const uint32_t joins = (uint32_t)nz_ceil_div(nz_ceil_div(count, kPiece) * slices, 4);
#define NZ_GRADIENT(T)                                                                                            \
  nz_embedding_sum_kernel<T><<<sums, 256, 0, st>>>(places, (uint32_t)count, (const T*)dev_g, stride, (uint32_t)cols, \
                                                   (uint32_t)slices, scale, flags, (T*)dev_out, pieces);          \
  if (count > kPiece)                                                                                             \
  nz_embedding_join_kernel<T><<<joins, 256, 0, st>>>(places, (uint32_t)count, (uint32_t)cols, (uint32_t)slices,   \
                                                     scale, flags, (T*)dev_out, pieces)
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
