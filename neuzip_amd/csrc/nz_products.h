// What the products of weights that are held in few bits share (nz_mx.hip, nz_fp8.hip): loads and stores of rows, the
// way of a tile through LDS, the join of parts, and the choice of tiles and parts.
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "nz_operators.h"

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef int i8v __attribute__((ext_vector_type(8)));
typedef int i4v __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef nz_bf16 b8v __attribute__((ext_vector_type(8)));
typedef nz_bf16 b2v __attribute__((ext_vector_type(2)));
typedef short s4v __attribute__((ext_vector_type(4)));

// ---- elements --------------------------------------------------------------------------------------------------

// Rows begin wherever their elements may: a vector of 8 is as aligned as one of them, which the memory allows.
template <class T>
struct Pack {
  typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

// 8 values of which the first `n` count, zeros behind them
template <class T>
__device__ inline void load8_upto(const T* p, uint32_t n, float (&v)[8]) {
  if (n >= 8) {
    const typename Pack<T>::type a = *reinterpret_cast<const typename Pack<T>::type*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (uint32_t)i < n ? (float)p[i] : 0.0f;
  }
}

// 8 values to a place that is aligned for vectors
template <class T>
__device__ inline void store8(T* p, const float (&v)[8]) {
  typedef T whole __attribute__((ext_vector_type(8)));
  whole a;
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = (T)v[i];
  *reinterpret_cast<whole*>(p) = a;
}

template <class T>
__device__ inline void store8_upto(T* p, uint32_t n, const float (&v)[8]) {
  if (n >= 8) {
    typename Pack<T>::type a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = (T)v[i];
    *reinterpret_cast<typename Pack<T>::type*>(p) = a;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((uint32_t)i < n) p[i] = (T)v[i];
  }
}

// 2^(127 - s) for a scale byte that scale_byte gives (at most 252); zero for 255
__device__ inline float up_factor(uint32_t s) { return s == 255 ? 0.0f : __uint_as_float((254u - s) << 23); }

// 2^(s - 127), a subnormal for s = 0; NaN for 255
__device__ inline float down_factor(uint32_t s) {
  return __uint_as_float(s == 255 ? 0x7FC00000u : s == 0 ? 0x00400000u : s << 23);
}

// codes of 8 values that share the factor `up`; larger ones become 448 (the conversion gives NaN above 464)
__device__ inline uint2 codes8(const float (&v)[8], float up) {
  float c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = __builtin_amdgcn_fmed3f(v[i] * up, -448.0f, 448.0f);
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[4], c[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[6], c[7], hi, true);
  return make_uint2((uint32_t)lo, (uint32_t)hi);
}

__device__ inline void values8(uint2 codes, float factor, float (&v)[8]) {
  const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.x, false);
  const f2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.x, true);
  const f2 c = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.y, false);
  const f2 d = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.y, true);
  v[0] = a.x * factor, v[1] = a.y * factor, v[2] = b.x * factor, v[3] = b.y * factor;
  v[4] = c.x * factor, v[5] = c.y * factor, v[6] = d.x * factor, v[7] = d.y * factor;
}

// ---- tiles -----------------------------------------------------------------------------------------------------

// 16 (4) bytes of every lane to LDS: lane l's to `to` (an LDS address, the same for all lanes) + 16 l (4 l), from
// `from`, the same for all lanes, + `offset`.  In assembly because the compiler, where it knows of such loads, waits
// for all of them in front of other reads of LDS, the next steps' loads among them.  It has no register to give to
// anything else too early, and the kernels count these loads themselves (wait_loads).  The address goes in through m0
// as an operand, so the compiler knows what is in that register; s_nop stands between its write and the load.
__device__ inline void to_lds16(const uint8_t* from, uint32_t offset, uint32_t to) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(to), "v"(offset), "s"(from) : "memory");
}
__device__ inline void to_lds4(const uint8_t* from, uint32_t offset, uint32_t to) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %1, %2" ::"{m0}"(to), "v"(offset), "s"(from) : "memory");
}

__device__ inline uint32_t lds_address(uint8_t* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)p;
}

// Wait until all but the last N loads of this wavefront have arrived.
template <int N>
__device__ inline void wait_loads() {
  static_assert(N < 64, "what the counter holds");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ inline void block_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Tile of the workgroup.  Workgroups go to the eight dies in turn: a die takes a run of consecutive tiles, and
// tiles are numbered through columns of eight tiles along m, so that what a die has in work at a time shares rows of
// both sides in its L2.
__device__ inline void tile_of(uint32_t id, uint32_t mt, uint32_t nt, uint32_t& tm, uint32_t& tn) {
  const uint32_t total = mt * nt, per = total / 8, rest = total % 8, die = id % 8;
  id = die * per + min(die, rest) + id / 8;
  const uint32_t column = id / (8 * nt), at = id - column * (8 * nt), high = min(mt - column * 8, 8u);
  tm = column * 8 + at % high;
  tn = at / high;
}

// Store a workgroup's tile in y, plus the bias (ADD: what y holds).  A lane (r, g) of wavefront (wm, wn) holds rows
// m0 + (wm TM + i) 16 + r and, from acc[i][0] to acc[i][TN - 1], 4 TN consecutive columns.
//
// It goes through LDS once more, so that a wavefront stores whole lines: straight from the lanes, which hold pieces of
// 16 rows, 8192 x (4096x1024) takes 53 us in tiles of 128x256 instead of 37, 8192 x (14336x4096) 434 instead of 409. (In
// tiles of 128x128 39 instead of 37 and 462 instead of 466.)
template <int WM, int WN, int TM, int TN, int LDS, bool ADD, class T>
__device__ inline void store_tile(f4 (&acc)[TM][TN], uint8_t* lds, uint32_t m, uint32_t n, uint32_t m0, uint32_t n0,
                                  const T* bias, T* y) {
  constexpr int W = WM * WN, BM = WM * TM * 16, BN = WN * TN * 16;
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64, r = lane & 15, g = lane / 16;
  const uint32_t wm = wave % WM, wn = wave / WM, c0 = wn * TN * 16 + g * TN * 4;
  constexpr int PITCH = BN * sizeof(T) + 16;  // eight lanes in turn write to all banks
  static_assert(BM * PITCH <= LDS, "a tile of the result");
  block_barrier();
#pragma unroll
  for (int j = 0; j < TN; j += 2) {
    float b[8] = {};
    const uint32_t c = n0 + c0 + j * 4;
    if (bias && c < n) load8_upto(bias + c, n - c, b);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      if constexpr (ADD) {
        const uint32_t row = m0 + (wm * TM + i) * 16 + r;
        if (row < m && c < n) load8_upto(y + (uint64_t)row * n + c, n - c, b);
      }
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = acc[i][j + e / 4][e % 4] + b[e];
      store8(reinterpret_cast<T*>(lds + ((wm * TM + i) * 16 + r) * PITCH) + c0 + j * 4, v);
    }
  }
  __syncthreads();
  constexpr int V = 16 / sizeof(T), ACROSS = BN / V;
  typedef T whole __attribute__((ext_vector_type(V)));
  typedef T piece __attribute__((ext_vector_type(V), aligned(sizeof(T))));
#pragma unroll
  for (int i = 0; i < BM * ACROSS / (64 * W); ++i) {
    const uint32_t at = i * (64 * W) + threadIdx.x, row = at / ACROSS, c = at % ACROSS * V;
    const whole v = *(const whole*)(lds + row * PITCH + c * sizeof(T));
    if (m0 + row >= m || n0 + c >= n) continue;
    T* q = y + (uint64_t)(m0 + row) * n + n0 + c;
    if (n0 + c + V <= n)
      *(piece*)q = v;
    else
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (n0 + c + e < n) q[e] = v[e];
  }
}

// The end of a tile: to y as above, or as it is to its place among the parts.  A part goes through LDS too where
// PARTS_TOO: of the gradient of a weight, two parts of 4096x1024, 75 us instead of 81.5.
template <int WM, int WN, int TM, int TN, int LDS, bool ADD = false, bool PARTS_TOO = false, class T>
__device__ inline void finish_tile(f4 (&acc)[TM][TN], uint8_t* lds, uint32_t m, uint32_t n, uint32_t m0, uint32_t n0,
                                   const T* bias, T* y, float* part) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64, r = lane & 15, g = lane / 16;
  const uint32_t wm = wave % WM, wn = wave / WM, c0 = wn * TN * 16 + g * TN * 4;
  if (part) {
    part += (uint64_t)blockIdx.y * m * n;
    if constexpr (PARTS_TOO) {
      store_tile<WM, WN, TM, TN, LDS, false>(acc, lds, m, n, m0, n0, (const float*)nullptr, part);
      return;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const uint32_t row = m0 + (wm * TM + i) * 16 + r;
      if (row >= m) break;
#pragma unroll
      for (int j = 0; j < TN; j += 2) {
        const uint32_t c = n0 + c0 + j * 4;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = acc[i][j + e / 4][e % 4];
        if (c < n) store8_upto(part + (uint64_t)row * n + c, n - c, v);
      }
    }
    return;
  }
  store_tile<WM, WN, TM, TN, LDS, ADD>(acc, lds, m, n, m0, n0, bias, y);
}

// The parts of a product whose rows were cut, added in their order (ADD: to what y holds).
template <bool ADD, class T>
__global__ __launch_bounds__(256) void nz_join_kernel(const float* part, uint32_t parts, uint64_t size, uint32_t n,
                                                      const T* bias, T* y) {
  const uint64_t at = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= size) return;
  if (size % 4 == 0) {
    f4 sum = *(const f4*)(part + at);
    for (uint32_t i = 1; i < parts; ++i) sum += *(const f4*)(part + i * size + at);
    const uint32_t col = (uint32_t)(at % n);
    typedef T pack __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    pack v;
    if constexpr (ADD) v = *(const pack*)(y + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (ADD)
        v[e] = (T)(sum[e] + (float)v[e]);
      else
        v[e] = (T)(bias ? sum[e] + (float)bias[(col + e) % n] : sum[e]);
    }
    *(pack*)(y + at) = v;
    return;
  }
  for (uint64_t i = at; i < min(at + 4, size); ++i) {
    float sum = part[i];
    for (uint32_t p = 1; p < parts; ++p) sum += part[p * size + i];
    if constexpr (ADD)
      y[i] = (T)(sum + (float)y[i]);
    else
      y[i] = (T)(bias ? sum + (float)bias[i % n] : sum);
  }
}

// Rows cut into P bf16 planes, [m][P][padded]: each plane takes the 8 leading bits that the planes before it left, so
// three hold all 24 bits of a float32 (of one below 2^-110 those down to 2^-133) and two the 11 of a float16.  What is not
// finite stays in the first.
template <int P, class T>
__global__ __launch_bounds__(256) void nz_planes_kernel(const T* g, uint64_t stride, uint64_t m, uint32_t n,
                                                           uint32_t padded, nz_bf16* out) {
  const uint64_t at = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  const uint64_t row = at / padded;
  const uint32_t c = (uint32_t)(at - row * padded);
  if (row >= m) return;
  float v[8];
  load8_upto(g + row * stride + c, c < n ? n - c : 0, v);
  nz_bf16* q = out + row * P * padded + c;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    b8v b;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t u = __float_as_uint(v[i]), hi = (u >> 23 & 255) == 255 && (u & 0x7FFFFF) ? u | 0x400000 : u;
      const float first = __uint_as_float(hi & 0xFFFF0000u);
      b[i] = __builtin_bit_cast(nz_bf16, (unsigned short)(hi >> 16));
      v[i] = (u >> 23 & 255) == 255 ? 0.0f : v[i] - first;
    }
    *(b8v*)(q + (uint64_t)p * padded) = b;
  }
}

// ---- host side -------------------------------------------------------------------------------------------------

bool aligned(const void* p, uint64_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

int check_dtype(int dtype, const void* a, const void* b, const void* c) {
  const uint32_t size = nz_dtype_bytes(dtype);
  if (!size) return nz_fail(NZ_ERR_DTYPE, "Unsupported data type");
  if (!aligned(a, size) || !aligned(b, size) || !aligned(c, size))
    return nz_fail(NZ_ERR_ALIGN, "dense pointers must be aligned to their elements");
  return NZ_OK;
}

template <class F>
void by_dtype(int dtype, F f) {
  if (dtype == NZ_DTYPE_BF16)
    f(nz_bf16());
  else if (dtype == NZ_DTYPE_F16)
    f(nz_f16());
  else
    f(float());
}

uint64_t align256(uint64_t v) { return (v + 255) / 256 * 256; }

// How a product is cut: the kernel's tile, and the parts the summed axis is cut into.
struct Cut {
  uint32_t bm, bn, parts, part_length, mt, nt;
  uint64_t part_bytes(uint64_t m, uint64_t cols) const { return parts > 1 ? align256(parts * m * cols * 4) : 0; }
};

// What a step takes (us) of a kernel with this tile while `slots` workgroups run, and while half of them or fewer do,
// on 256 compute units; the begin and end of a round of workgroups, which others do not cover; and whether it takes whole
// products of whole steps only.
struct Tile {
  uint32_t bm, bn, slots;
  float full, half, ends = 1.0f;
  bool whole = false;
};

// The cut that takes the least time by these figures.  Rounds of workgroups follow each other; parts cost a launch of
// 4 us and are written, read and joined at 5 TB/s.  `whole`: the product is one of whole steps.
// From rows in 8 bits, 64 x (4096x14336) takes 24 us in 64 tiles of 64x64 and 12.5 in four parts of them; 17 x
// (128256x4096) 71 us in tiles of 128x256, 51 in 64x128.  Where the figures are off: 5366 x (576x12736) takes 64 us in
// the 420 tiles of 64x128 that are chosen, 60 in two parts of 210 tiles of 128x128.
template <int N>
Cut cut_product(const Tile (&kinds)[N], uint64_t m, uint64_t cols, uint64_t units_of, uint64_t steps_per_unit,
                uint64_t least, bool whole = false) {
  const uint32_t cus = nz_compute_units();
  const float scale = cus ? cus / 256.0f : 1.0f;
  Cut best = {};
  float best_time = 0;
  for (const Tile& t : kinds) {
    if (t.whole && !whole) continue;
    const uint64_t mt = nz_ceil_div(m, t.bm), nt = nz_ceil_div(cols, t.bn);
    const float slots = t.slots * scale;
    const uint32_t units = (uint32_t)std::min<uint64_t>(units_of, 1u << 30);
    for (uint32_t want = 1; want <= std::min<uint64_t>(units_of, 16); ++want) {
      if (want > 1 && (t.whole || (float)(mt * nt * want) > 4 * slots)) break;  // enough without parts
      const uint32_t length = (units + want - 1) / want, parts = (units + length - 1) / length;
      if (parts != want || (parts > 1 && length < least)) continue;
      const float groups = (float)(mt * nt * parts), rounds = floorf(groups / slots), rest = groups - rounds * slots;
      float time = (rounds * t.full + (rest == 0 ? 0.0f : rest <= slots / 2 ? t.half : t.full)) *
                       (float)(length * steps_per_unit) +
                   t.ends * rounds + t.ends * (rest > 0);
      if (parts > 1) time += 4.0f + (float)parts * (float)m * (float)cols * 2.8e-6f;
      if (best.parts == 0 || time < best_time) {
        best = Cut{t.bm, t.bn, (uint32_t)parts, (uint32_t)length, (uint32_t)mt, (uint32_t)nt};
        best_time = time;
      }
    }
  }
  return best;
}

template <bool ADD = false>
void launch_join(const float* part, const Cut& c, uint64_t m, uint64_t n, const void* bias, void* y, int dtype,
                 hipStream_t st) {
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    nz_join_kernel<ADD, T><<<(uint32_t)nz_ceil_div(m * n, 1024), 256, 0, st>>>(part, c.parts, m * n, (uint32_t)n,
                                                                              (const T*)bias, (T*)y);
  });
}

// Tiles of the largest products are counted by the grid: workgroups have up to 512 threads.
int check_cut(const Cut& c) {
  return (uint64_t)c.mt * c.nt <= nz_most_groups(512) ? NZ_OK : nz_fail(NZ_ERR_ARG, "too many rows for one launch");
}

int check_workspace(const void* workspace, uint64_t bytes, uint64_t need) {
  if (bytes < need) return nz_fail(NZ_ERR_CAPACITY, "workspace too small");
  if (need && (!workspace || !aligned(workspace, 16))) return nz_fail(NZ_ERR_ALIGN, "misaligned workspace");
  return NZ_OK;
}

// The gradient's rows as planes of bf16, or as they are.
struct Planes {
  uint32_t count;
  uint64_t padded, bytes;
};
Planes planes_of(const void* g, int dtype, uint64_t m, uint64_t n, uint64_t stride) {
  Planes p;
  p.count = dtype == NZ_DTYPE_BF16 ? 1 : dtype == NZ_DTYPE_F16 ? 2 : 3;
  p.padded = nz_ceil_div(n, 64) * 64;
  const bool as_is = dtype == NZ_DTYPE_BF16 && n % 64 == 0 && stride % 8 == 0 && stride <= 1ull << 22 && aligned(g, 16);
  p.bytes = as_is ? 0 : align256(nz_mul(m, p.padded * p.count * 2));
  return p;
}

}  // namespace
