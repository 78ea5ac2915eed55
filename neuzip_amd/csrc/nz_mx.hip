// Weights in microscaled 4 bits: quantisation, values, row lookup, and the products with activation rows.
//
// The format is stated in include/neuzip_hip.h.  A row's codes lie in order and are filled up to 128 values, so
// that a step of the matrix instruction (128 values of a row) never ends inside one; its block scales lie in
// groups of 16 (512 values) with the four bytes that a lane needs in four successive steps next to each other.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "nz_operators.h"

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef int i8v __attribute__((ext_vector_type(8)));
typedef int i4v __attribute__((ext_vector_type(4)));

constexpr uint32_t kStep = 128;   // values of a row that one matrix instruction takes
constexpr uint32_t kGroup = 512;  // values of a row whose scales are 16 consecutive bytes

template <int BITS>
struct Element;
template <>
struct Element<4> {
  static constexpr int kTop = 2;  // exponent of the largest binade
};
template <>
struct Element<8> {
  static constexpr int kTop = 8;
};

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

// scale byte of a block from the bits of its largest magnitude: a subnormal has exponent bits 0, which the clamp
// takes to the smallest scale as well
template <int BITS>
__device__ inline uint32_t scale_byte(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23);
  return e == 255 ? 255u : (uint32_t)max(e - Element<BITS>::kTop, 0);
}

// 2^(127 - s) for a scale byte that scale_byte gives (at most 252); zero for 255
__device__ inline float up_factor(uint32_t s) { return s == 255 ? 0.0f : __uint_as_float((254u - s) << 23); }

// 2^(s - 127), a subnormal for s = 0; NaN for 255
__device__ inline float down_factor(uint32_t s) {
  return __uint_as_float(s == 255 ? 0x7FC00000u : s == 0 ? 0x00400000u : s << 23);
}

// codes of 8 values that share the factor `up`.  Multiplying by a power of two is exact (a product that leaves the
// normal range is far below half of the smallest code).  The 4-bit conversion clamps by itself, the 8-bit one gives
// NaN above 464.
__device__ inline uint32_t codes4(const float (&v)[8], float up) {
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0] * up, v[1] * up, 1.0f, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2] * up, v[3] * up, 1.0f, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4] * up, v[5] * up, 1.0f, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6] * up, v[7] * up, 1.0f, 3);
  return r;
}
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

typedef float f2 __attribute__((ext_vector_type(2)));

__device__ inline void values4(uint32_t codes, float factor, float (&v)[8]) {
  const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 0);
  const f2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 1);
  const f2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 2);
  const f2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 3);
  v[0] = a.x * factor, v[1] = a.y * factor, v[2] = b.x * factor, v[3] = b.y * factor;
  v[4] = c.x * factor, v[5] = c.y * factor, v[6] = d.x * factor, v[7] = d.y * factor;
}
__device__ inline void values8(uint2 codes, float factor, float (&v)[8]) {
  const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.x, false);
  const f2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.x, true);
  const f2 c = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.y, false);
  const f2 d = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.y, true);
  v[0] = a.x * factor, v[1] = a.y * factor, v[2] = b.x * factor, v[3] = b.y * factor;
  v[4] = c.x * factor, v[5] = c.y * factor, v[6] = d.x * factor, v[7] = d.y * factor;
}

// Scale byte of a block that four lanes share, 8 values each; a block that reads as NaN is cleared.
template <int BITS>
__device__ inline uint32_t block_scale(float (&v)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xB1, 0xF, 0xF, true));  // lane ^ 1
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4E, 0xF, 0xF, true));  // lane ^ 2
  const uint32_t s = scale_byte<BITS>(top);
  if (s == 255)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
  return s;
}

// place of block b (of a row) among the row's scale bytes
__device__ inline uint32_t scale_at(uint32_t b) { return (b & ~15u) + 4 * (b & 3) + ((b >> 2) & 3); }

// ---- quantisation and values -----------------------------------------------------------------------------------
//
// One wavefront per 512 values of a row: 8 values a lane, four lanes a block, so that loads and stores of a
// wavefront are consecutive and the block's maximum takes two exchanges inside a quad.  Both are bound by memory:
// 16384x4096 bf16 values to 4 bits in 35.5 us (4.8 TB/s; a copy reaches 5.1), back in 26.6 us.  (Two groups a
// wavefront, for twice the loads on their way, took 37.9.)

template <int BITS, class T>
__global__ __launch_bounds__(256) void nz_mx_quantize_kernel(const T* x, uint64_t stride, uint32_t cols,
                                                             uint64_t waves, uint32_t groups, uint8_t* data,
                                                             uint8_t* scales) {
  const uint64_t wave = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64;
  if (wave >= waves) return;
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t row = wave / groups;
  const uint32_t group = (uint32_t)(wave - row * groups);
  const uint32_t at = group * kGroup + lane * 8;
  const T* p = x + row * stride + at;
  float v[8];
  load8_upto(p, at < cols ? cols - at : 0, v);
  const uint32_t s = block_scale<BITS>(v);
  const float up = up_factor(s);
  const uint32_t filled = (cols + kStep - 1) / kStep * kStep;
  if (at < filled) {
    uint8_t* out = data + row * (uint64_t)(filled / 8 * BITS) + at / 8 * BITS;
    if constexpr (BITS == 4)
      *reinterpret_cast<uint32_t*>(out) = codes4(v, up);
    else
      *reinterpret_cast<uint2*>(out) = codes8(v, up);
  }
  if ((lane & 3) == 0) scales[(row * groups + group) * 16 + scale_at(lane / 4)] = (uint8_t)s;
}

// Values of the rows `index` names (or of all rows), times `scale`.
template <int BITS, class T>
__global__ __launch_bounds__(256) void nz_mx_values_kernel(const uint8_t* data, const uint8_t* scales, uint64_t rows,
                                                           uint32_t cols, const long long* index, uint64_t waves,
                                                           uint32_t groups, float scale, T* out, uint32_t* status) {
  const uint64_t wave = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64;
  if (wave >= waves) return;
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t to = wave / groups;
  const uint32_t group = (uint32_t)(wave - to * groups);
  const uint32_t at = group * kGroup + lane * 8;
  if (at >= cols) return;
  float v[8];
  const uint64_t row = index ? (uint64_t)index[to] : to;
  if (row < rows) {
    const float f = down_factor(scales[(row * groups + group) * 16 + scale_at(lane / 4)]);
    const uint32_t filled = (cols + kStep - 1) / kStep * kStep;
    const uint8_t* p = data + row * (uint64_t)(filled / 8 * BITS) + at / 8 * BITS;
    if constexpr (BITS == 4)
      values4(*reinterpret_cast<const uint32_t*>(p), f, v);
    else
      values8(*reinterpret_cast<const uint2*>(p), f, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= scale;
  } else {
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    if (status && at == 0) atomicOr(status, 1u);
  }
  store8_upto(out + to * (uint64_t)cols + at, cols - at, v);
}

// ---- product ---------------------------------------------------------------------------------------------------
//
// The matrix instruction takes 16 rows of each side and 128 values of a row.  A lane (r = lane % 16, g = lane / 16)
// holds, of row r: 4-bit values 32 g .. 32 g + 31; 8-bit values 16 g .. 16 g + 15 and 64 + 16 g .. 64 + 16 g + 15;
// and, on both sides, the scale of block g.  Of the result it holds weight rows 4 g .. 4 g + 3 against activation
// row r.
//
// The instruction adds eight consecutive products at a time behind the largest exponent E of the eight: a product is
// cut, toward zero, to a multiple of 2^(E - 13); what it adds after that it holds in 32 bits. (As its results show: all
// pairs of the 128 places, both signs, subnormal and zero elements.) A product has 5 bits behind its leading one at
// most, so only those are cut that are some 2^9 smaller than a neighbour, whose activation was rounded to 4 bits
// before: 1.5e-5 of a sum of normal values, and one 16-bit result in 100 (bf16, 4096 values) rounded the other way.
// That is the price of its rate. The same products by bf16 instructions on values converted first, which keep 32 bits,
// take 8.8 and 13.7 us for one row (14336x4096, rows in 8 bits), 12.6 and 30 for 64 (4096x14336), 399 and 990 for 8192
// rows: this is what a float32 result is made with, and a caller who needs those bits asks for one.

__device__ inline f4 step(i4v w, i4v x0, i4v x1, f4 acc, uint32_t sw, uint32_t sx, int byte) {
  const i8v a = {w.x, w.y, w.z, w.w, 0, 0, 0, 0};
  const i8v b = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
  switch (byte) {  // a constant where this is inlined
    case 0: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 0, 0, (int)sw, 0, (int)sx);
    case 1: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 0, 1, (int)sw, 1, (int)sx);
    case 2: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 0, 2, (int)sw, 2, (int)sx);
    default: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 0, 3, (int)sw, 3, (int)sx);
  }
}

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

// Add the bias to a workgroup's tile and store it, or store it as it is among the parts.  A lane (r, g) of wavefront
// (wm, wn) holds rows m0 + (wm TM + i) 16 + r and, from acc[i][0] to acc[i][TN - 1], 4 TN consecutive columns.
//
// The tile goes through LDS once more, so that a wavefront stores whole lines: straight from the lanes, which hold
// pieces of 16 rows, 8192 x (4096x1024) takes 53 us in tiles of 128x256 instead of 37, 8192 x (14336x4096) 434 instead
// of 409. (In tiles of 128x128 39 instead of 37 and 462 instead of 466.)
template <int WM, int WN, int TM, int TN, int LDS, class T>
__device__ inline void finish_tile(f4 (&acc)[TM][TN], uint8_t* lds, uint32_t m, uint32_t n, uint32_t m0, uint32_t n0,
                                   const T* bias, T* y, float* part) {
  constexpr int W = WM * WN, BM = WM * TM * 16, BN = WN * TN * 16;
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64, r = lane & 15, g = lane / 16;
  const uint32_t wm = wave % WM, wn = wave / WM, c0 = wn * TN * 16 + g * TN * 4;
  if (part) {
    part += (uint64_t)blockIdx.y * m * n;
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

// A tile of WM TM x WN TN matrix instructions' results, WM x WN wavefronts with TM x TN each.
//
// The rows of both sides are staged through LDS in steps of 128 values, NS stages deep, by loads that go to LDS
// without registers; a wavefront counts its own loads down, and one barrier a step tells that everybody's have
// arrived and that the stage before is used up.  Staged rows are exchanged in chunks of 16 bytes (x: chunk c of row
// r at c ^ (r & 7); w: at c ^ ((r >> 1) & 3)) so that eight lanes in turn read from all banks, and the weight rows of
// a wavefront are staged in an order that leaves each lane 4 TN consecutive columns of the result.  Scales are
// staged once per 512 values.
//
// 8192 x (14336x4096) takes 400 us, 2.4 PFLOP/s, in runs of ten; a library's 8-bit product of 8192^3 reaches 2.7. Those
// are 800000 cycles, at 2.0 GHz: the matrix units, busy for 60 % of them (48 % where a row has 1024 values only), draw
// the clock down, the more the longer such passes follow each other without a pause (465 to 493 us). The LDS is in use
// for 19 %, hardly any of it in conflicts; 281 MB come from memory, and 90 % of the reads of L2 hit. What the matrix
// units wait for is the begin and end of a tile and the barrier of a step: two workgroups a compute unit, with two
// stages each, cover each other's; a 256x256 tile, which leaves room for one, took 423 us where this took 380. Reading
// operands ahead across the barrier, or 32x32x64 instructions, do not pay.
template <int WM, int WN, int TM, int TN, int NS, class T>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(2, 2))) void nz_mx_tiles_kernel(
    const uint8_t* xd, const uint8_t* xs, uint32_t m, const uint8_t* wd, const uint8_t* ws, uint32_t n, uint32_t k,
    const T* bias, T* y, uint32_t mt, uint32_t nt, uint32_t part_groups, float* part) {
  constexpr int W = WM * WN, BM = WM * TM * 16, BN = WN * TN * 16;
  constexpr int XB = BM * 128, WB = BN * 64, STAGE = XB + WB;
  constexpr int XI = BM / 8 / W, WI = BN / 16 / W, LOADS = XI + WI;
  constexpr int SI = (BM + BN + 63) / 64, SB = SI * 1024;  // scales: 64 rows of 16 bytes a load
  constexpr int SL = (SI + W - 1) / W;                     // of a wavefront
  static_assert(XI * 8 * W == BM && WI * 16 * W == BN, "loads per wavefront");
  static_assert(NS >= 2 && NS <= 4, "a group's scales are asked for when the last group's have been read");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[NS * STAGE + SB];
  const uint32_t base = lds_address(lds);
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t r = lane & 15, g = lane / 16;
  const uint32_t all_steps = (k + kStep - 1) / kStep, groups = (k + kGroup - 1) / kGroup;
  const uint32_t from = blockIdx.y * part_groups, steps = min(all_steps - from * 4, part_groups * 4);
  uint32_t tm, tn;
  tile_of(blockIdx.x, mt, nt, tm, tn);
  const uint32_t m0 = tm * BM, n0 = tn * BN;
  const uint32_t m_last = min((uint32_t)BM, m - m0) - 1, n_last = min((uint32_t)BN, n - n0) - 1;

  // Where this lane loads from: a base of the workgroup and an offset.  Rows behind the last one are read as the last.
  const uint8_t* xb = xd + (uint64_t)m0 * (all_steps * 128ull) + from * 512ull;
  const uint8_t* wb = wd + (uint64_t)n0 * (all_steps * 64ull) + from * 256ull;
  const auto column = [](uint32_t row) {  // of the tile, for a staged weight row
    return row / (TN * 16) * (TN * 16) + row % 16 / 4 * (TN * 4) + row / 16 % TN * 4 + row % 4;
  };
  uint32_t xo[XI], wo[WI];
#pragma unroll
  for (int i = 0; i < XI; ++i)
    xo[i] = min((wave * XI + i) * 8 + lane / 8, m_last) * (all_steps * 128) + ((lane & 7) ^ (lane / 8)) * 16;
#pragma unroll
  for (int i = 0; i < WI; ++i)
    wo[i] = min(column((wave * WI + i) * 16 + lane / 4), n_last) * (all_steps * 64) +
            ((lane & 3) ^ ((lane >> 3) & 3)) * 16;
  // where wavefronts and loads of scales do not match, some load the same
  const uint8_t* sb[SL];
  uint32_t so[SL], si[SL];
#pragma unroll
  for (int i = 0; i < SL; ++i) {
    si[i] = (i * W + wave) % SI;
    const uint32_t row = min(si[i] * 64 + lane, BM + BN - 1u);
    sb[i] = (si[i] * 64 < BM ? xs + (uint64_t)m0 * (groups * 16ull) : ws + (uint64_t)n0 * (groups * 16ull)) + from * 16;
    so[i] = (row < BM ? min(row, m_last) : min(column(row - BM), n_last)) * (groups * 16);
  }
  static_assert(BM % 64 == 0, "a load takes scales of one side");
  const auto load_stage = [&](uint32_t s, uint32_t buf, bool scales) {
    s = min(s, steps - 1);  // past the end the last stage is loaded again, into a buffer that is not read
    const uint32_t to = base + buf * STAGE;
#pragma unroll
    for (int i = 0; i < XI; ++i) to_lds16(xb + s * 128ull, xo[i], to + (wave * XI + i) * 1024);
#pragma unroll
    for (int i = 0; i < WI; ++i) to_lds16(wb + s * 64ull, wo[i], to + XB + (wave * WI + i) * 1024);
    if (scales) {
#pragma unroll
      for (int i = 0; i < SL; ++i)
        to_lds16(sb[i] + (s >> 2) * 16, so[i], base + NS * STAGE + si[i] * 1024);
    }
  };

  const uint32_t wm = wave % WM, wn = wave / WM;
  f4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f4{0, 0, 0, 0};
  uint32_t sx[TM], sw[TN];
  const uint32_t xr = (wm * TM * 16 + r) * 128, x0c = (g ^ (r & 7)) * 16, x1c = x0c ^ 64;
  const uint32_t wr = XB + (wn * TN * 16 + r) * 64 + (g ^ ((r >> 1) & 3)) * 16;

#pragma unroll
  for (int i = 0; i < NS - 1; ++i) load_stage(i, i, i % 4 == 0);
  uint32_t buf = 0;
  const auto body = [&](uint32_t s, auto b4) {
    constexpr int byte = decltype(b4)::value;  // s % 4
    // loads behind those of stage s: NS - 2 stages, with scales where a stage begins a group
    constexpr int starts = (byte + NS - 2) / 4;
    wait_loads<(NS - 2) * LOADS + starts * SL>();
    block_barrier();  // stage s is there, stage s - 1 is used up
    const uint8_t* b = lds + buf * STAGE;
    if (byte == 0) {
      const uint8_t* st = lds + NS * STAGE;
#pragma unroll
      for (int i = 0; i < TM; ++i) sx[i] = *(const uint32_t*)(st + (wm * TM * 16 + i * 16 + r) * 16 + g * 4);
#pragma unroll
      for (int j = 0; j < TN; ++j) sw[j] = *(const uint32_t*)(st + (BM + wn * TN * 16 + j * 16 + r) * 16 + g * 4);
    }
    i4v x0[TM], x1[TM], w[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      x0[i] = *(const i4v*)(b + xr + i * 2048 + x0c);
      x1[i] = *(const i4v*)(b + xr + i * 2048 + x1c);
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) w[j] = *(const i4v*)(b + wr + j * 1024);
    load_stage(s + NS - 1, buf == 0 ? NS - 1 : buf - 1, (byte + NS - 1) % 4 == 0);
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i) acc[i][j] = step(w[j], x0[i], x1[i], acc[i][j], sw[j], sx[i], byte);
    buf = buf == NS - 1 ? 0 : buf + 1;
    __builtin_amdgcn_sched_barrier(0);  // matrix instructions stay inside their step
  };
  using B0 = std::integral_constant<int, 0>;
  using B1 = std::integral_constant<int, 1>;
  using B2 = std::integral_constant<int, 2>;
  using B3 = std::integral_constant<int, 3>;
  uint32_t s = 0;
  for (; s + 4 <= steps; s += 4) {
    body(s, B0());
    body(s + 1, B1());
    body(s + 2, B2());
    body(s + 3, B3());
  }
  if (s < steps) body(s, B0());
  if (s + 1 < steps) body(s + 1, B1());
  if (s + 2 < steps) body(s + 2, B2());
  wait_loads<0>();  // nothing may arrive in this memory once it is another workgroup's

  finish_tile<WM, WN, TM, TN, NS * STAGE + SB>(acc, lds, m, n, m0, n0, bias, y, part);
}

// The parts of a product whose rows were cut, added in their order.
template <class T>
__global__ __launch_bounds__(256) void nz_mx_join_kernel(const float* part, uint32_t parts, uint64_t size, uint32_t n,
                                                         const T* bias, T* y) {
  const uint64_t at = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= size) return;
  if (size % 4 == 0) {
    f4 sum = *(const f4*)(part + at);
    for (uint32_t i = 1; i < parts; ++i) sum += *(const f4*)(part + i * size + at);
    const uint32_t col = (uint32_t)(at % n);
    typedef T pack __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    pack v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (T)(bias ? sum[e] + (float)bias[(col + e) % n] : sum[e]);
    *(pack*)(y + at) = v;
    return;
  }
  for (uint64_t i = at; i < min(at + 4, size); ++i) {
    float sum = part[i];
    for (uint32_t p = 1; p < parts; ++p) sum += part[p * size + i];
    y[i] = (T)(bias ? sum + (float)bias[i % n] : sum);
  }
}

typedef nz_bf16 b8v __attribute__((ext_vector_type(8)));
typedef nz_bf16 b2v __attribute__((ext_vector_type(2)));
typedef short s4v __attribute__((ext_vector_type(4)));

// 8 codes as bf16 numbers.  The conversion takes the exponent field of its scale: a scale byte there is what it means.
__device__ inline b8v bf16_of_codes(uint32_t codes, uint32_t s) {
  const float scale = __uint_as_float(s << 23);
  const b2v a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
  const b2v b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  const b2v c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
  const b2v d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return b8v{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Up to 16 rows, where reading the weight is all that counts: no staging and no barrier in the way of it.  The eight
// wavefronts are kw that share the values of a row (512 at a time, in turn) times 8 / kw with 16 weight rows each;
// a lane loads its operand of the matrix instruction straight from memory.  The rows come in 8 bits, or
// (QUANTIZE) as they are: then every workgroup brings them to 8 bits in LDS while its first weights are on their way.
// Results in float32 are summed by bf16 instructions (why, see `step`), for which a lane takes both sides to bf16: of
// the 128 values of a step those of its block, 8 at a time (both sides in the same order, which is all that counts).
// One row against 14336x4096: 8.2 us, 3.8 TB/s of codes and scales, of which 2 are the launch.
template <bool QUANTIZE, class T>
__global__ __launch_bounds__(512) void nz_mx_few_kernel(const void* x, uint64_t stride, const uint8_t* xs,
                                                        uint32_t m, const uint8_t* wd, const uint8_t* ws, uint32_t n,
                                                        uint32_t k, const T* bias, T* y, uint32_t kw) {
  extern __shared__ __attribute__((aligned(16))) uint8_t few_lds[];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64, r = lane & 15, g = lane / 16;
  const uint32_t steps = (k + kStep - 1) / kStep, groups = (k + kGroup - 1) / kGroup;
  const uint32_t kwave = wave % kw, tile = blockIdx.x * (8 / kw) + wave / kw;
  const uint64_t w_row = min(tile * 16 + r, n - 1);
  const uint8_t* wp = wd + w_row * (steps * 64ull) + g * 16;
  const uint8_t* sp = ws + w_row * (groups * 16ull) + g * 4;
  struct Held {
    i4v w[4];
    uint32_t s;
  } a, b;
  const auto load = [&](Held& h, uint32_t group) {
    h.s = *(const uint32_t*)(sp + group * 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) h.w[i] = *(const i4v*)(wp + (uint64_t)min(group * 4 + i, steps - 1) * 64);
  };
  if (kwave < groups) load(a, kwave);

  constexpr bool kWide = std::is_same<T, float>::value;
  const uint32_t row = min(r, m - 1), xg = g * (kWide ? 32 : 16);
  const uint8_t *xp, *xsp;
  if constexpr (QUANTIZE) {
    // rows of groups * 528 bytes: 512 values and their scales per group
    const T* xt = (const T*)x;
    const auto quantise = [&](uint32_t i, auto size) {  // every eighth from i on, all on their way at once
      constexpr uint32_t N = decltype(size)::value;
      typename Pack<T>::type raw[N];
#pragma unroll
      for (uint32_t j = 0; j < N; ++j) {
        const uint32_t to = (i + 8 * j) / groups, at = (i + 8 * j - to * groups) * kGroup + lane * 8;
        raw[j] = {};
        if (at + 8 <= k) raw[j] = *(const typename Pack<T>::type*)(xt + to * stride + at);
      }
#pragma unroll
      for (uint32_t j = 0; j < N; ++j) {
        const uint32_t to = (i + 8 * j) / groups, at = (i + 8 * j - to * groups) * kGroup + lane * 8;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)raw[j][e];
        if (at < k && at + 8 > k) load8_upto(xt + to * stride + at, k - at, v);
        const uint32_t s = block_scale<8>(v);
        uint8_t* q = few_lds + (i + 8 * j) * 528u;
        *(uint2*)(q + lane * 8) = codes8(v, up_factor(s));
        if ((lane & 3) == 0) q[512 + scale_at(lane / 4)] = (uint8_t)s;
      }
    };
    uint32_t i = wave;
    for (; i + 24 < m * groups; i += 32) quantise(i, std::integral_constant<uint32_t, 4>());
    for (; i < m * groups; i += 8) quantise(i, std::integral_constant<uint32_t, 1>());
    __syncthreads();
    xp = few_lds + row * groups * 528u + xg;
    xsp = few_lds + row * groups * 528u + 512 + g * 4;
  } else {
    xp = (const uint8_t*)x + row * (steps * 128ull) + xg;
    xsp = xs + row * (groups * 16ull) + g * 4;
  }
  f4 acc = {0, 0, 0, 0};
  const auto multiply = [&](const Held& h, uint32_t group) {
    const uint32_t sx = *(const uint32_t*)(xsp + group * (QUANTIZE ? 528 : 16));
    const auto one = [&](auto b4) {
      constexpr int i = decltype(b4)::value;
      if (group * 4 + i >= steps) return;
      const uint8_t* p = xp + (QUANTIZE ? group * 528 : (uint64_t)group * 512) + i * 128;
      if constexpr (kWide) {
        const float f = down_factor(sx >> (8 * i) & 255);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[8];
          values8(*(const uint2*)(p + 8 * q), f, v);
          b8v xv;
#pragma unroll
          for (int e = 0; e < 8; ++e) xv[e] = (nz_bf16)v[e];
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf16_of_codes(h.w[i][q], h.s >> (8 * i) & 255), xv, acc, 0, 0,
                                                        0);
        }
      } else {
        const i4v x0 = *(const i4v*)p, x1 = *(const i4v*)(p + 64);
        acc = step(h.w[i], x0, x1, acc, h.s, sx, i);
      }
    };
    one(std::integral_constant<int, 0>());
    one(std::integral_constant<int, 1>());
    one(std::integral_constant<int, 2>());
    one(std::integral_constant<int, 3>());
  };
  for (uint32_t group = kwave; group < groups; group += 2 * kw) {  // one group is on its way while one is multiplied
    if (group + kw < groups) load(b, group + kw);
    multiply(a, group);
    if (group + kw >= groups) break;
    if (group + 2 * kw < groups) load(a, group + 2 * kw);
    multiply(b, group + kw);
  }
  // the wavefronts that share rows add up in their order
  __syncthreads();
  float* part = (float*)few_lds;
  *(f4*)(part + (wave * 16 + r) * 16 + g * 4) = acc;
  __syncthreads();
  const uint32_t tiles = 8 / kw;
  for (uint32_t i = threadIdx.x; i < m * tiles * 16; i += 512) {
    const uint32_t to = i / (tiles * 16), c = i - to * (tiles * 16), t = c / 16;
    const uint32_t col = blockIdx.x * tiles * 16 + c;
    if (col >= n) continue;
    float sum = 0;
    for (uint32_t q = 0; q < kw; ++q) sum += part[((t * kw + q) * 16 + to) * 16 + c % 16];
    if (bias) sum += (float)bias[col];
    y[(uint64_t)to * n + col] = (T)sum;
  }
}

// ---- products of 16-bit rows -----------------------------------------------------------------------------------
//
// What the scaled instruction cannot do: the gradient of the rows, whose sums run over the weight's rows (a lane
// would need a scale per value), and results in float32 (it cuts products as stated at `step`: 1.5e-5 of a sum,
// measured, against 6e-8 of this one).  A weight's values are exact in
// bf16, and so is an activation of 8 bits; a gradient of 16 or 32 bits is the sum of two or three bf16 numbers, laid
// side by side along the summed axis.

// Rows cut into P bf16 planes, [m][P][padded]: each plane takes the 8 leading bits that the planes before it left, so
// three hold all 24 bits of a float32 (of one below 2^-110 those down to 2^-133) and two the 11 of a float16.  What is not
// finite stays in the first.
template <int P, class T>
__global__ __launch_bounds__(256) void nz_mx_planes_kernel(const T* g, uint64_t stride, uint64_t m, uint32_t n,
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

// What the 8 bits of float32 rows stand for, as bf16 numbers, rows filled up to whole steps: the rows' side of a
// product with a float32 result.
__global__ __launch_bounds__(256) void nz_mx_rounded_kernel(const float* x, uint64_t stride, uint32_t cols,
                                                            uint64_t waves, uint32_t groups, nz_bf16* out) {
  const uint64_t wave = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64;
  if (wave >= waves) return;
  const uint64_t row = wave / groups;
  const uint32_t at = (uint32_t)(wave - row * groups) * kGroup + (threadIdx.x & 63) * 8;
  float v[8];
  load8_upto(x + row * stride + at, at < cols ? cols - at : 0, v);
  const uint32_t s = block_scale<8>(v);
  const uint2 codes = codes8(v, up_factor(s));
  values8(codes, down_factor(s), v);
  const uint32_t filled = (cols + kStep - 1) / kStep * kStep;
  if (at < filled) store8(out + row * filled + at, v);
}

// A tile of C[m][cols] = sum over c of A[m][c] B(c, col), c running `planes` times through the summed axis.
// ROWS: B(c, col) = w[c][col], the gradient; else w[col][c], the product itself.
//
// Steps of 64 values.  Rows of A, codes and scales go to LDS without registers two steps ahead (16-byte chunk c of a
// row of A at c ^ (row & 7)); a step ahead, the codes are written to LDS once more as bf16, once for all wavefronts.
// Where the sums run over the weight's rows that tile lies as in memory, and the operand is read by the instruction
// that transposes 4 x 16 values on the way.  A lane ends with 4 TN consecutive columns, as in nz_mx_tiles_kernel.
//
// 8192 rows of gradients against 4096x1024: 66 us, 1.04 PFLOP/s; a library's bf16 product of 8192^3 reaches 1.26 and
// the instructions of this loop without the rest 1.65.  Reads of operands, conversion and loads cost some 10 us each:
// all of them go through LDS, which is in use for 53 % of the time (15 % in conflicts), the matrix units for 56 %.
// Tiles of 128x128, two workgroups a compute unit, took 78 us.
template <int WM, int WN, int TM, int TN, bool ROWS, class T>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(2, 2))) void nz_mx_tiles16_kernel(
    const nz_bf16* a, uint64_t a_stride, uint32_t m, const uint8_t* wd, const uint8_t* ws, uint32_t w_rows,
    uint32_t w_cols, uint32_t steps_1, uint32_t planes, uint32_t cols, const T* bias, T* y, uint32_t mt, uint32_t nt,
    uint32_t part_steps, float* part) {
  constexpr int W = WM * WN, BM = WM * TM * 16, BN = WN * TN * 16, XI = BM / 8 / W, ROW = ROWS ? BN : 64;
  constexpr int AB = BM * 128, BB = BN * 128, CB = BN * 32, SB = BN * 8;  // bytes a step: A, bf16, codes, scales
  constexpr int B_AT = 3 * AB, C_AT = B_AT + 2 * BB, S_AT = C_AT + 3 * CB, LOADS = XI + 2;
  static_assert(XI * 8 * W == BM && BN * 64 == 16 * 64 * W, "16 rows of A and 16 codes per lane");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[S_AT + 3 * SB];
  const uint32_t base = lds_address(lds);
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t r = lane & 15, g = lane / 16;
  const uint32_t from = blockIdx.y * part_steps, steps = min(steps_1 * planes - from, part_steps);
  const uint32_t w_steps = (w_cols + kStep - 1) / kStep, w_groups = (w_cols + kGroup - 1) / kGroup;
  const uint32_t w_bytes = w_steps * 64, s_bytes = w_groups * 16;
  uint32_t tm, tn;
  tile_of(blockIdx.x, mt, nt, tm, tn);
  const uint32_t m0 = tm * BM, n0 = tn * BN, m_last = min((uint32_t)BM, m - m0) - 1;

  // Loads: a base of the workgroup, moved from step to step, and an offset of the lane.
  const uint8_t* ab = (const uint8_t*)(a + (uint64_t)m0 * a_stride) + from * 128ull;
  uint32_t ao[XI];
#pragma unroll
  for (int i = 0; i < XI; ++i)
    ao[i] = min((wave * XI + i) * 8 + lane / 8, m_last) * (uint32_t)(a_stride * 2) + ((lane & 7) ^ (lane / 8)) * 16;
  const auto load_a = [&](uint32_t s, uint32_t buf, int i) {  // the i-th of XI
    // past the end the last stage is loaded again, into a buffer that is not read
    to_lds16(ab + min(s, steps - 1) * 128ull, ao[i], base + buf * AB + (wave * XI + i) * 1024);
  };
  // Codes: 16 bytes, a block of 32, of a lane; scales: the four bytes that hold that block's.  The first 2 BN lanes'
  // are all; the others load the same again.  The last rows of a weight have offsets of their own, so that none
  // behind the last is read.
  const uint32_t id = threadIdx.x % (2 * BN), id_row = id / (ROW / 32), id_block = id % (ROW / 32);
  uint32_t co, so, co_last, so_last;
  if constexpr (ROWS) {
    const uint32_t block = min(n0 / 32 + id_block, w_steps * 4 - 1), last = min(id_row, (w_rows - 1) % 64);
    const uint32_t group = block / 16 * 16 + block % 4 * 4;
    co = id_row * w_bytes + block * 16, co_last = last * w_bytes + block * 16;
    so = id_row * s_bytes + group, so_last = last * s_bytes + group;
  } else {
    const uint32_t col =
        id_row / (TN * 16) * (TN * 16) + id_row % 16 / 4 * (TN * 4) + id_row / 16 % TN * 4 + id_row % 4;
    const uint32_t row = min(n0 + col, w_rows - 1) - n0;
    co = co_last = row * w_bytes + id_block * 16;
    so = so_last = row * s_bytes + id_block * 4;
    wd += (uint64_t)n0 * w_bytes, ws += (uint64_t)n0 * s_bytes;
  }
  uint32_t w_step = from % steps_1;  // of the codes that are loaded next
  const auto load_w = [&](uint32_t buf) {
    const bool last = ROWS && w_step + 1 == steps_1;
    const uint8_t* c = wd + (ROWS ? (uint64_t)w_step * 64 * w_bytes : w_step * 32ull);
    const uint8_t* s = ws + (ROWS ? (uint64_t)w_step * 64 * s_bytes : w_step / 8 * 16ull + (w_step & 1) * 8);
    to_lds16(c, last ? co_last : co, base + C_AT + buf * CB + wave % (BN / 32) * 1024);
    to_lds4(s, last ? so_last : so, base + S_AT + buf * SB + wave % (BN / 32) * 256);
    w_step = w_step + 1 == steps_1 ? 0 : w_step + 1;
  };
  // To bf16: 16 codes of a lane, neighbours' from eight rows.  Rows exchange 16-byte pieces (piece c of row r at
  // c ^ (r & 7)) so that eight lanes write to all banks; ROWS: in rows 2 and 3 of four, 8-byte halves of a piece as
  // well, so that the four rows of a transposing read do not meet.
  constexpr uint32_t ACROSS = ROW / 16;
  const uint32_t l_row = threadIdx.x / (8 * ACROSS) * 8 + threadIdx.x % 8, l_at = threadIdx.x / 8 % ACROSS * 16;
  const uint32_t swap = ROWS && (l_row & 2) ? 16 : 0;
  const uint32_t c_at = C_AT + l_row * (ROW / 2) + l_at / 2, s_at = S_AT + l_row * (ROW / 8) + l_at / 32 * 4;
  uint32_t to[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) to[j] = B_AT + l_row * (ROW * 2) + ((l_at / 8 + j) ^ (l_row & 7)) * 16;
  uint32_t c_step = from % steps_1;  // of the codes that are written next
  const auto convert = [&](uint32_t buf, uint32_t half) {
    const uint2 codes = *(const uint2*)(lds + c_at + buf * CB);
    const uint32_t scale = lds[s_at + buf * SB + (ROWS ? n0 / 128 & 3 : c_step / 2 & 3)];
    const uint32_t word[2] = {codes.x, codes.y};
#pragma unroll
    for (int j = 0; j < 2; ++j)
      *(b8v*)(lds + to[j] + half * BB) =
          bf16_of_codes(ROWS ? __builtin_amdgcn_alignbit(word[j], word[j], swap) : word[j], scale);
    c_step = c_step + 1 == steps_1 ? 0 : c_step + 1;
  };

  const uint32_t wm = wave % WM, wn = wave / WM;
  f4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f4{0, 0, 0, 0};
  // operand addresses; the halves of a step lie at constant distances
  uint32_t ra[2], rb[TN * 2];
#pragma unroll
  for (int h = 0; h < 2; ++h) ra[h] = (wm * TM * 16 + r) * 128 + ((h * 4 + g) ^ (r & 7)) * 16;
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint32_t row = g * 8 + q * 4 + r / 4, slot = wn * TN * 4 + r % 4 * TN + j;
      rb[j * 2 + q] = base + B_AT + row * (BN * 2) + (slot ^ (row & 7) * 2 ^ (row >> 1 & 1)) * 8;
    }
  const uint32_t rw = B_AT + (wn * TN * 16 + r) * 128;

  load_w(0);
#pragma unroll
  for (int i = 0; i < XI; ++i) load_a(0, 0, i);
  load_w(1);
#pragma unroll
  for (int i = 0; i < XI; ++i) load_a(1, 1, i);
  load_w(2);
  wait_loads<2 * LOADS>();  // codes of step 0
  block_barrier();
  convert(0, 0);
  wait_loads<LOADS>();  // rows of step 0, codes of step 1
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  block_barrier();

  // Operands of a half step are read while the other half's are multiplied, across the barrier as well: behind it
  // the first half of step s + 1 while the second of step s is multiplied.
  struct Operands {
    b8v a[TM], b[TN];
  } first, second;
  constexpr int READS = TN + TM;
  const auto read = [&](Operands& o, uint32_t buf, uint32_t odd, int h, int q) {  // the q-th of READS
    if (q >= TN) {
      o.a[q - TN] = *(const b8v*)(lds + buf * AB + ra[h] + (q - TN) * 2048);
    } else if constexpr (ROWS) {
      s4v part[2];
#pragma unroll
      for (int p = 0; p < 2; ++p)
        part[p] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s4v*)(uintptr_t)(rb[q * 2 + p] + odd * BB + h * 64 * BN));
      o.b[q] = __builtin_bit_cast(b8v, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      o.b[q] = *(const b8v*)(lds + odd * BB + rw + q * 2048 + ((h * 4 + g) ^ (r & 7)) * 16);
    }
  };
  uint32_t buf = 0;  // s % 3
#pragma unroll
  for (int q = 0; q < READS; ++q) read(first, 0, 0, 0, q);
  const auto body = [&](uint32_t s, auto odd) {
    constexpr uint32_t here = decltype(odd)::value;  // s % 2
    // reads and loads stand between the instructions, in an order that the barriers of scheduling keep
    constexpr int M = TM * TN, EARLY = M - M / 4;
    const auto multiply = [&](const Operands& o, auto beside) {
#pragma unroll
      for (int t = 0; t < M; ++t) {
        const int i = t % TM, j = t / TM;
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(o.b[j], o.a[i], acc[i][j], 0, 0, 0);
        beside(t);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    const uint32_t after = buf == 2 ? 0 : buf + 1, free = buf == 0 ? 2 : buf - 1;
    multiply(first, [&](int t) {
      if (t == 0) convert(after, here ^ 1);
#pragma unroll
      for (int q = 0; q < READS; ++q)
        if (q * EARLY / READS == t) read(second, buf, here, 1, q);
#pragma unroll
      for (int i = 0; i < XI; ++i)
        if (i * M / XI == t) load_a(s + 2, free, i);
      if (t == M - 1) load_w(buf);
    });
    // behind the rows of step s + 1 and the codes of step s + 2: what has just been asked for
    wait_loads<LOADS>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    block_barrier();  // step s + 1 is in LDS, step s is used up
    multiply(second, [&](int t) {
#pragma unroll
      for (int q = 0; q < READS; ++q)
        if (q * EARLY / READS == t) read(first, after, here ^ 1, 0, q);
    });
    buf = after;
  };
  uint32_t s = 0;
  for (; s + 2 <= steps; s += 2) {
    body(s, std::integral_constant<uint32_t, 0>());
    body(s + 1, std::integral_constant<uint32_t, 1>());
  }
  if (s < steps) body(s, std::integral_constant<uint32_t, 0>());
  wait_loads<0>();  // nothing may arrive in this memory once it is another workgroup's
  finish_tile<WM, WN, TM, TN, S_AT + 3 * SB>(acc, lds, m, cols, m0, n0, bias, y, part);
}

// ---- host side -------------------------------------------------------------------------------------------------

uint64_t filled(uint64_t cols) { return nz_ceil_div(cols, kStep) * kStep; }

// rows are counted in 64 bits, the values of one row in 31
bool cols_ok(uint64_t cols) { return cols <= 0x40000000ull; }

// Sums over rows, the gradient of a bias: 512 columns a workgroup, every fourth of its rows a wavefront, eight of them
// on their way at a time; the wavefronts' sums are added in their order.  Many rows are cut into parts, whose sums are
// summed by the same kernel: no atomics, so the order of additions is that of the sizes, and nothing has to be cleared.
// 8192 x 4096 bf16 values take 18 us, 3.7 TB/s; 8192 x 1021 12.6.
template <class T, class R>
__global__ __launch_bounds__(256) void nz_mx_column_sums_kernel(const T* x, uint64_t stride, uint32_t m, uint32_t n,
                                                                uint32_t rows, R* out) {
  constexpr uint32_t kRows = 8;
  __shared__ float sums[3][64][9];  // a ninth: lanes apart in their banks
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  // the last columns of a width that is no multiple of 8 are loaded with some before them
  const uint32_t own = blockIdx.x * 512 + lane * 8, mine = own < n ? min(8u, n - own) : 0;
  const uint32_t c = n < 8 ? 0 : min(own, n - 8);
  const uint32_t first = blockIdx.y * rows, last = min(m, first + rows);
  float sum[8] = {};
  if (n >= 8) {
    for (uint32_t row = first + wave; row < last; row += 4 * kRows) {
      typename Pack<T>::type v[kRows];
#pragma unroll
      for (uint32_t j = 0; j < kRows; ++j)
        v[j] = *(const typename Pack<T>::type*)(x + min(row + 4 * j, last - 1) * stride + c);
#pragma unroll
      for (uint32_t j = 0; j < kRows; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] = row + 4 * j < last ? sum[e] + (float)v[j][e] : sum[e];
    }
  } else {
    for (uint32_t row = first + wave; row < last; row += 4) {
      float v[8];
      load8_upto(x + row * stride, n, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += v[e];
    }
  }
  if (wave)
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[wave - 1][lane][e] = sum[e];
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 0; w < 3; ++w)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += sums[w][lane][e];
  R* to = out + (uint64_t)blockIdx.y * n;
  if (mine == 8) {
    store8_upto(to + own, 8, sum);
  } else {
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e)
      if (c + e >= own && c + e < own + mine) to[c + e] = (R)sum[e];
  }
}

bool aligned(const void* p, uint64_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

int check_dtype(int dtype, const void* a, const void* b, const void* c) {
  const uint32_t size = nz_dtype_bytes(dtype);
  if (!size) return nz_fail(NZ_ERR_DTYPE, "Unsupported data type");
  if (!aligned(a, size) || !aligned(b, size) || !aligned(c, size))
    return nz_fail(NZ_ERR_ALIGN, "dense pointers must be aligned to their elements");
  return NZ_OK;
}

int check_mx(const void* data, const void* scales) {
  if (!data || !scales) return nz_fail(NZ_ERR_ARG, "null data or scales");
  if (!aligned(data, 16) || !aligned(scales, 16))
    return nz_fail(NZ_ERR_ALIGN, "microscaled data and scales must be 16-byte aligned");
  return NZ_OK;
}

int check_bits(int bits) {
  return bits == 4 || bits == 8 ? NZ_OK : nz_fail(NZ_ERR_ARG, "bits must be 4 or 8");
}

// groups of 512 values in all rows, beyond any memory
int check_groups(uint64_t rows, uint64_t groups) {
  return nz_mul(rows, groups) <= 1ull << 33 ? NZ_OK : nz_fail(NZ_ERR_ARG, "too many rows");
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

int launch_quantize(const void* x, int dtype, uint64_t rows, uint32_t cols, uint64_t stride, int bits, void* data,
                    void* scales, hipStream_t st) {
  const uint32_t groups = (cols + kGroup - 1) / kGroup;
  if (int rc = check_groups(rows, groups)) return rc;
  const uint64_t row_bytes = nz_mx_row_bytes(cols, bits);
  nz_in_pieces(rows, groups * 64ull, [&](uint64_t first, uint64_t count) {
    const uint64_t waves = count * groups;
    const dim3 grid((uint32_t)nz_ceil_div(waves, 4));
    uint8_t* d = (uint8_t*)data + first * row_bytes;
    uint8_t* s = (uint8_t*)scales + first * groups * 16;
    by_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      const T* from = (const T*)x + first * stride;
      if (bits == 4)
        nz_mx_quantize_kernel<4, T><<<grid, 256, 0, st>>>(from, stride, cols, waves, groups, d, s);
      else
        nz_mx_quantize_kernel<8, T><<<grid, 256, 0, st>>>(from, stride, cols, waves, groups, d, s);
    });
  });
  return nz_launched();
}

int launch_values(const void* data, const void* scales, uint64_t rows, uint64_t cols, int bits, const void* index,
                  uint64_t count, float scale, void* out, int dtype, void* status, hipStream_t st) {
  const uint32_t groups = (uint32_t)nz_ceil_div(cols, kGroup);
  if (int rc = check_groups(count, groups)) return rc;
  const uint64_t row_bytes = nz_mx_row_bytes(cols, bits);
  nz_in_pieces(count, groups * 64ull, [&](uint64_t first, uint64_t piece) {
    const uint64_t waves = piece * groups;
    const dim3 grid((uint32_t)nz_ceil_div(waves, 4));
    // rows that no index names begin at the piece's first
    const uint64_t skip = index ? 0 : first;
    const uint8_t* d = (const uint8_t*)data + skip * row_bytes;
    const uint8_t* s = (const uint8_t*)scales + skip * groups * 16;
    const long long* ids = index ? (const long long*)index + first : nullptr;
    by_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      T* to = (T*)out + first * cols;
      if (bits == 4)
        nz_mx_values_kernel<4, T><<<grid, 256, 0, st>>>(d, s, rows - skip, (uint32_t)cols, ids, waves, groups, scale,
                                                        to, (uint32_t*)status);
      else
        nz_mx_values_kernel<8, T><<<grid, 256, 0, st>>>(d, s, rows - skip, (uint32_t)cols, ids, waves, groups, scale,
                                                        to, (uint32_t*)status);
    });
  });
  return nz_launched();
}

uint64_t align256(uint64_t v) { return (v + 255) / 256 * 256; }

// How a product is cut: the kernel's tile, and the parts the summed axis is cut into.
struct Cut {
  uint32_t bm, bn, parts, part_length, mt, nt;
  uint64_t part_bytes(uint64_t m, uint64_t cols) const { return parts > 1 ? align256(parts * m * cols * 4) : 0; }
};

// What a step takes (us) of a kernel with this tile while `slots` workgroups run, and while half of them or fewer do,
// on 256 compute units.  These and the figures of cut_product are fitted to times of 150 products of 17 to 8192 rows
// with weights of 256 to 16384 rows and columns, each in all tiles and up to 16 parts: the cut chosen by them takes
// 1.2 % more than the fastest one in the mean (of 16-bit rows 1.4 %), at most 17 %.
struct Tile {
  uint32_t bm, bn, slots;
  float full, half;
};
// Products of 8-bit rows, 128 values a step: 8192 x (14336x4096) at 2.3, 2.1, 1.7 and 1.4 PFLOP/s.
constexpr Tile kTiles[] = {{128, 256, 512, 1.70f, 1.40f},
                           {128, 128, 512, 1.00f, 1.00f},
                           {64, 128, 256, 0.36f, 0.38f},
                           {64, 64, 256, 0.25f, 0.28f}};
// Products of 16-bit rows, 64 values a step: 8192 x (4096x4096) at 1.0 and 0.5 PFLOP/s.
constexpr Tile kTiles16[] = {{256, 128, 256, 0.95f, 0.86f}, {64, 64, 256, 0.31f, 0.31f}};

// The cut that takes the least time by these figures.  Rounds of workgroups follow each other and begin and end in 1 us
// that others do not cover; parts cost a launch of 4 us and are written, read and joined at 5 TB/s.
// From rows in 8 bits, 64 x (4096x14336) takes 24 us in 64 tiles of 64x64 and 12.5 in four parts of them; 17 x
// (128256x4096) 71 us in tiles of 128x256, 51 in 64x128.  Where the figures are off: 5366 x (576x12736) takes 64 us in
// the 420 tiles of 64x128 that are chosen, 60 in two parts of 210 tiles of 128x128.
template <int N>
Cut cut_product(const Tile (&kinds)[N], uint64_t m, uint64_t cols, uint64_t units_of, uint64_t steps_per_unit,
                uint64_t least) {
  const uint32_t cus = nz_compute_units();
  const float scale = cus ? cus / 256.0f : 1.0f;
  Cut best = {};
  float best_time = 0;
  for (const Tile& t : kinds) {
    const uint64_t mt = nz_ceil_div(m, t.bm), nt = nz_ceil_div(cols, t.bn);
    const float slots = t.slots * scale;
    const uint32_t units = (uint32_t)std::min<uint64_t>(units_of, 1u << 30);
    for (uint32_t want = 1; want <= std::min<uint64_t>(units_of, 16); ++want) {
      if (want > 1 && (float)(mt * nt * want) > 4 * slots) break;  // enough without parts
      const uint32_t length = (units + want - 1) / want, parts = (units + length - 1) / length;
      if (parts != want || (parts > 1 && length < least)) continue;
      const float groups = (float)(mt * nt * parts), rounds = floorf(groups / slots), rest = groups - rounds * slots;
      float time = (rounds * t.full + (rest == 0 ? 0.0f : rest <= slots / 2 ? t.half : t.full)) *
                       (float)(length * steps_per_unit) +
                   rounds + (rest > 0);
      if (parts > 1) time += 4.0f + (float)parts * (float)m * (float)cols * 2.8e-6f;
      if (best.parts == 0 || time < best_time) {
        best = Cut{t.bm, t.bn, (uint32_t)parts, (uint32_t)length, (uint32_t)mt, (uint32_t)nt};
        best_time = time;
      }
    }
  }
  return best;
}

// The product of 8-bit rows, cut along k by groups of four steps, two at least.
Cut cut_product8(uint64_t m, uint64_t n, uint64_t k) {
  return cut_product(kTiles, m, n, nz_ceil_div(k, kGroup), 4, 2);
}

// The products of 16-bit rows, in steps of 64.
Cut cut_product16(uint64_t m, uint64_t cols, uint64_t steps) {
  return cut_product(kTiles16, m, cols, steps, 1, 8);
}

void launch_join(const float* part, const Cut& c, uint64_t m, uint64_t n, const void* bias, void* y, int dtype,
                 hipStream_t st) {
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    nz_mx_join_kernel<T><<<(uint32_t)nz_ceil_div(m * n, 1024), 256, 0, st>>>(part, c.parts, m * n, (uint32_t)n,
                                                                            (const T*)bias, (T*)y);
  });
}

template <bool ROWS>
int launch_tiles16(const Cut& c, const void* a, uint64_t a_stride, uint64_t m, const void* wd, const void* ws,
                   uint64_t w_rows, uint64_t w_cols, uint64_t steps_1, uint32_t planes, uint64_t cols,
                   const void* bias, void* y, int dtype, void* part, hipStream_t st) {
  const dim3 grid(c.mt * c.nt, c.parts);
  float* p = c.parts > 1 ? (float*)part : nullptr;
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if constexpr (!ROWS && !std::is_same<T, float>::value) {
      return;  // the product itself has results of 16 bits from the scaled instruction
    } else {
#define NZ_TILES16(WM, WN, TM, TN)                                                                                     \
  nz_mx_tiles16_kernel<WM, WN, TM, TN, ROWS, T><<<grid, 64 * WM * WN, 0, st>>>(                                        \
      (const nz_bf16*)a, a_stride, (uint32_t)m, (const uint8_t*)wd, (const uint8_t*)ws, (uint32_t)w_rows,              \
      (uint32_t)w_cols, (uint32_t)steps_1, planes, (uint32_t)cols, (const T*)bias, (T*)y, c.mt, c.nt, c.part_length, p)
      if (c.bm == 256)
        NZ_TILES16(4, 2, 4, 4);
      else
        NZ_TILES16(2, 2, 2, 2);
#undef NZ_TILES16
    }
  });
  if (p) launch_join(p, c, m, cols, bias, y, dtype, st);
  return nz_launched();
}

// Rows that go to the kernel for few (one tile of the instruction), and those that are brought to 8 bits inside it:
// every workgroup does that again, which costs more the longer and the more the rows are and the more workgroups there
// are (`groups` of 512 values in all rows).  Times on the device of quantising inside, before it, and before tiles
// (with the join of their parts, if any); a launch less is 4 us less for the caller, who often is what takes longest:
//    2 rows of 12421x14421, 58 groups   21.8 26.7 24.9      8 rows of 50257x4096, 64 groups   28.4 43.8 22.5
//    8 of 9505x3706, 64                  9.9 12.4  9.4      4 of 128256x1024, 8               15.1 23.7 21.9
//    6 of 1735x7471, 90                    -  8.8 12.3     16 of 9498x3995, 128                  - 17.6 10.1
//    7 of 5003x3001, 42                  7.0  8.8  9.2      8 of 14336x4096, 64               10.3 14.4  9.9
// The rule loses 3 us at the first of these.  Results in float32, whose tiles are slower, are better off in this kernel
// always: 16 rows of 12886x8431 31 us (quantised before it) against 46, one of 14336x4096 11 (inside) against 25.
bool few_inside(uint64_t m, uint64_t n, uint64_t k, int dtype) {
  const uint64_t groups = m * nz_ceil_div(k, kGroup);
  return m <= 16 && groups <= 64 && (groups <= 32 || n * k <= 1ull << 26 || dtype == NZ_DTYPE_F32);
}
bool few_rows(uint64_t m, uint64_t n, uint64_t k, int dtype) {
  return few_inside(m, n, k, dtype) || (m <= 16 && (n * k <= 1ull << 25 || dtype == NZ_DTYPE_F32));
}

template <bool QUANTIZE, class T>
void launch_few(const void* x, uint64_t stride, const void* xs, uint64_t m, const void* wd, const void* ws, uint64_t n,
                uint32_t k, const T* bias, T* y, hipStream_t st) {
  const uint32_t groups = (k + kGroup - 1) / kGroup;
  uint32_t kw = groups >= 8 ? 8 : groups >= 4 ? 4 : groups >= 2 ? 2 : 1;
  const uint64_t t = nz_ceil_div(n, 16);
  // weights that fill the device with fewer wavefronts to a row: fewer workgroups that each bring the rows to 8 bits.
  // 14336x4096, with 2, 4, 8 wavefronts to a row: one row 8.1, 7.5, 8.7 us; four 8.9, 9.2, 11.2
  const uint32_t cus = nz_compute_units();
  if (t > 2 * (cus ? cus : 256)) kw = kw < 4 ? kw : m >= 4 ? 2 : 4;
  const uint32_t lds = QUANTIZE ? (uint32_t)m * groups * 528 : 0;
  nz_mx_few_kernel<QUANTIZE, T><<<(uint32_t)nz_ceil_div(t, 8 / kw), 512, lds > 8192 ? lds : 8192, st>>>(
      x, stride, (const uint8_t*)xs, (uint32_t)m, (const uint8_t*)wd, (const uint8_t*)ws, (uint32_t)n, k, bias, y, kw);
}

template <class T>
void launch_tiles(const Cut& c, const void* xd, const void* xs, uint64_t m, const void* wd, const void* ws, uint64_t n,
                  uint32_t k, const T* bias, T* y, float* part, hipStream_t st) {
  const dim3 grid(c.mt * c.nt, c.parts);
#define NZ_TILES(WM, WN, TM, TN, NS)                                                                               \
  nz_mx_tiles_kernel<WM, WN, TM, TN, NS, T><<<grid, 64 * WM * WN, 0, st>>>(                                        \
      (const uint8_t*)xd, (const uint8_t*)xs, (uint32_t)m, (const uint8_t*)wd, (const uint8_t*)ws, (uint32_t)n, k, \
      bias, y, c.mt, c.nt, c.part_length, part)
  if (c.bn == 256)
    NZ_TILES(2, 2, 4, 8, 2);
  else if (c.bm == 128)
    NZ_TILES(2, 2, 4, 4, 2);
  else if (c.bn == 128)
    NZ_TILES(2, 2, 2, 4, 4);
  else
    NZ_TILES(2, 2, 2, 2, 4);
#undef NZ_TILES
}

// Parts that the rows of a column sum are cut into: workgroups for the whole device, each with 32 rows at least; one
// where few rows do not pay for a second launch (64 x 4096: 2.8 us).
uint32_t sum_parts(uint64_t m, uint64_t n) {
  if (m <= 128) return 1;
  const uint64_t slices = nz_ceil_div(n, 512);
  return (uint32_t)std::max<uint64_t>(1, std::min(nz_ceil_div(m, 32), nz_ceil_div(1024, slices)));
}

// Where a product's workspace holds what: rows in 8 bits, their values for a float32 result, parts.
struct Room {
  uint64_t xd, xs, values, parts, bytes;
  Cut cut;  // of rows that go to tiles
};
Room product_room(uint64_t m, uint64_t n, uint64_t k, int dtype) {
  Room r = {};
  if (few_inside(m, n, k, dtype)) return r;
  r.xd = 0;
  r.xs = align256(nz_mul(m, nz_mx_row_bytes(k, 8)));
  r.values = align256(r.xs + nz_mul(m, nz_mx_scale_bytes(k)));
  r.bytes = r.values;
  if (few_rows(m, n, k, dtype)) return r;
  const uint64_t pad = filled(k);
  if (dtype == NZ_DTYPE_F32) {
    r.cut = cut_product16(m, n, pad / 64);
    r.values = 0;  // the rows' 8 bits are not kept
    r.parts = align256(nz_mul(m, pad * 2));
  } else {
    r.cut = cut_product8(m, n, k);
    r.parts = r.values;
  }
  r.bytes = r.parts + r.cut.part_bytes(m, n);
  return r;
}

// A float32 result of rows whose values lie in the workspace.
int launch_wide(uint64_t m, const void* wd, const void* ws, uint64_t n, uint32_t k, const void* bias, void* y,
                const Room& room, uint8_t* workspace, hipStream_t st) {
  return launch_tiles16<false>(room.cut, workspace + room.values, filled(k), m, wd, ws, n, k, filled(k) / 64, 1, n,
                               bias, y, NZ_DTYPE_F32, workspace + room.parts, st);
}

int launch_product(const void* xd, const void* xs, uint64_t m, const void* wd, const void* ws, uint64_t n, uint32_t k,
                   const void* bias, void* y, int dtype, const Room& room, uint8_t* workspace, hipStream_t st) {
  if (few_rows(m, n, k, dtype)) {
    by_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      launch_few<false>(xd, 0, xs, m, wd, ws, n, k, (const T*)bias, (T*)y, st);
    });
    return nz_launched();
  }
  if (dtype == NZ_DTYPE_F32) {
    if (int rc = launch_values(xd, xs, m, filled(k), 8, nullptr, m, 1.0f, workspace + room.values, NZ_DTYPE_BF16,
                               nullptr, st))
      return rc;
    return launch_wide(m, wd, ws, n, k, bias, y, room, workspace, st);
  }
  const Cut& c = room.cut;
  float* part = c.parts > 1 ? (float*)(workspace + room.parts) : nullptr;
  if (dtype == NZ_DTYPE_BF16)
    launch_tiles(c, xd, xs, m, wd, ws, n, k, (const nz_bf16*)bias, (nz_bf16*)y, part, st);
  else
    launch_tiles(c, xd, xs, m, wd, ws, n, k, (const nz_f16*)bias, (nz_f16*)y, part, st);
  if (part) launch_join(part, c, m, n, bias, y, dtype, st);
  return nz_launched();
}

// What the products ask of the weight and the counts: an offset inside a tile has 32 bits.
int check_product(uint64_t m, uint64_t n, uint64_t k, const void* wd, const void* ws) {
  if (k == 0 || k > 1ull << 22 || n > 1ull << 21)
    return nz_fail(NZ_ERR_ARG, "a weight must have 1 to 2^22 columns and up to 2^21 rows");
  if (m > 1ull << 24) return nz_fail(NZ_ERR_ARG, "too many rows");
  return check_mx(wd, ws);
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

extern "C" {

uint64_t nz_mx_row_bytes(uint64_t cols, int bits) { return bits == 4 || bits == 8 ? filled(cols) / 8 * bits : 0; }

uint64_t nz_mx_scale_bytes(uint64_t cols) { return nz_ceil_div(cols, kGroup) * 16; }

int nz_mx_quantize(const void* dev_x, int dtype, uint64_t rows, uint64_t cols, uint64_t stride, int bits,
                   void* dev_data, void* dev_scales, void* stream) {
  if (int rc = check_bits(bits)) return rc;
  if (int rc = check_dtype(dtype, dev_x, nullptr, nullptr)) return rc;
  if (rows == 0 || cols == 0) return NZ_OK;
  if (!cols_ok(cols)) return nz_fail(NZ_ERR_ARG, "rows must hold 1 to 2^30 values");
  if (!dev_x) return nz_fail(NZ_ERR_ARG, "null input");
  if (int rc = check_mx(dev_data, dev_scales)) return rc;
  return launch_quantize(dev_x, dtype, rows, (uint32_t)cols, stride, bits, dev_data, dev_scales, (hipStream_t)stream);
}

int nz_mx_dequantize(const void* dev_data, const void* dev_scales, uint64_t rows, uint64_t cols, int bits,
                     void* dev_out, int dtype, void* stream) {
  return nz_mx_lookup(dev_data, dev_scales, rows, cols, bits, nullptr, rows, 1.0f, dev_out, dtype, nullptr, stream);
}

int nz_mx_lookup(const void* dev_data, const void* dev_scales, uint64_t rows, uint64_t cols, int bits,
                 const void* dev_indices, uint64_t count, float scale, void* dev_out, int dtype, void* dev_status,
                 void* stream) {
  if (int rc = check_bits(bits)) return rc;
  if (int rc = check_dtype(dtype, dev_out, nullptr, nullptr)) return rc;
  if (count == 0 || cols == 0) return NZ_OK;
  if (!cols_ok(cols)) return nz_fail(NZ_ERR_ARG, "rows must hold 1 to 2^30 values");
  if (!dev_out) return nz_fail(NZ_ERR_ARG, "null output");
  if (!dev_indices && count != rows) return nz_fail(NZ_ERR_ARG, "null indices");
  if (!aligned(dev_indices, 8) || !aligned(dev_status, 4)) return nz_fail(NZ_ERR_ALIGN, "misaligned indices or status");
  if (rows)  // a table without rows is never read
    if (int rc = check_mx(dev_data, dev_scales)) return rc;
  return launch_values(dev_data, dev_scales, rows, cols, bits, dev_indices, count, scale, dev_out, dtype, dev_status,
                       (hipStream_t)stream);
}

uint64_t nz_mx_linear_workspace_bytes(uint64_t m, uint64_t n, uint64_t k, int dtype) {
  if (m == 0 || n == 0 || k == 0) return 0;
  return product_room(m, n, k, dtype).bytes;
}

int nz_mx_linear(const void* dev_x, int dtype, uint64_t m, uint64_t k, uint64_t stride, const void* dev_w_data,
                 const void* dev_w_scales, uint64_t n, const void* dev_bias, void* dev_y, void* dev_workspace,
                 uint64_t workspace_bytes, void* stream) {
  if (int rc = check_dtype(dtype, dev_x, dev_bias, dev_y)) return rc;
  if (m == 0 || n == 0) return NZ_OK;
  if (int rc = check_product(m, n, k, dev_w_data, dev_w_scales)) return rc;
  if (!dev_x || !dev_y) return nz_fail(NZ_ERR_ARG, "null rows or output");
  const Room room = product_room(m, n, k, dtype);
  if (int rc = check_cut(room.cut)) return rc;
  if (int rc = check_workspace(dev_workspace, workspace_bytes, room.bytes)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  if (few_inside(m, n, k, dtype)) {
    by_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      launch_few<true>(dev_x, stride, nullptr, m, dev_w_data, dev_w_scales, n, (uint32_t)k, (const T*)dev_bias,
                       (T*)dev_y, st);
    });
    return nz_launched();
  }
  uint8_t* base = (uint8_t*)dev_workspace;
  if (dtype == NZ_DTYPE_F32 && !few_rows(m, n, k, dtype)) {
    const uint64_t groups = nz_ceil_div(k, kGroup);
    nz_in_pieces(m, groups * 64, [&](uint64_t first, uint64_t count) {
      nz_mx_rounded_kernel<<<(uint32_t)nz_ceil_div(count * groups, 4), 256, 0, st>>>(
          (const float*)dev_x + first * stride, stride, (uint32_t)k, count * groups, (uint32_t)groups,
          (nz_bf16*)(base + room.values) + first * filled(k));
    });
    return launch_wide(m, dev_w_data, dev_w_scales, n, (uint32_t)k, dev_bias, dev_y, room, base, st);
  }
  if (int rc = launch_quantize(dev_x, dtype, m, (uint32_t)k, stride, 8, base + room.xd, base + room.xs, st)) return rc;
  return launch_product(base + room.xd, base + room.xs, m, dev_w_data, dev_w_scales, n, (uint32_t)k, dev_bias, dev_y,
                        dtype, room, base, st);
}

int nz_mx_linear_rows8(const void* dev_x_data, const void* dev_x_scales, uint64_t m, uint64_t k,
                       const void* dev_w_data, const void* dev_w_scales, uint64_t n, const void* dev_bias, void* dev_y,
                       int dtype, void* dev_workspace, uint64_t workspace_bytes, void* stream) {
  if (int rc = check_dtype(dtype, dev_bias, dev_y, nullptr)) return rc;
  if (m == 0 || n == 0) return NZ_OK;
  if (int rc = check_product(m, n, k, dev_w_data, dev_w_scales)) return rc;
  if (int rc = check_mx(dev_x_data, dev_x_scales)) return rc;
  if (!dev_y) return nz_fail(NZ_ERR_ARG, "null output");
  const Room room = product_room(m, n, k, dtype);
  if (int rc = check_cut(room.cut)) return rc;
  if (int rc = check_workspace(dev_workspace, workspace_bytes, room.bytes)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  return launch_product(dev_x_data, dev_x_scales, m, dev_w_data, dev_w_scales, n, (uint32_t)k, dev_bias, dev_y, dtype,
                        room, (uint8_t*)dev_workspace, st);
}

uint64_t nz_mx_linear_grad_workspace_bytes(const void* dev_g, int dtype, uint64_t m, uint64_t n, uint64_t stride,
                                           uint64_t k) {
  if (m == 0 || n == 0 || k == 0) return 0;
  const Planes p = planes_of(dev_g, dtype, m, n, stride);
  return p.bytes + cut_product16(m, k, p.padded / 64 * p.count).part_bytes(m, k);
}

int nz_mx_linear_grad(const void* dev_g, int dtype, uint64_t m, uint64_t n, uint64_t stride, const void* dev_w_data,
                      const void* dev_w_scales, uint64_t k, void* dev_dx, void* dev_workspace,
                      uint64_t workspace_bytes, void* stream) {
  if (int rc = check_dtype(dtype, dev_g, dev_dx, nullptr)) return rc;
  if (m == 0 || k == 0) return NZ_OK;
  if (!dev_dx || !dev_g) return nz_fail(NZ_ERR_ARG, "null gradient or output");
  if (n == 0) return nz_fail(NZ_ERR_ARG, "a weight without rows has no gradient to pass on");
  if (int rc = check_product(m, n, k, dev_w_data, dev_w_scales)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  const Planes p = planes_of(dev_g, dtype, m, n, stride);
  const uint64_t steps = p.padded / 64;
  const Cut cut = cut_product16(m, k, steps * p.count);
  if (int rc = check_cut(cut)) return rc;
  if (int rc = check_workspace(dev_workspace, workspace_bytes, p.bytes + cut.part_bytes(m, k))) return rc;
  const void* a = dev_g;
  uint64_t a_stride = stride;
  if (p.bytes) {
    a = dev_workspace, a_stride = p.padded * p.count;
#define NZ_PLANES(P, T)                                                                                           \
  nz_in_pieces(m, p.padded / 8, [&](uint64_t first, uint64_t count) {                                             \
    nz_mx_planes_kernel<P, T><<<(uint32_t)nz_ceil_div(count * (p.padded / 8), 256), 256, 0, st>>>(                \
        (const T*)dev_g + first * stride, stride, count, (uint32_t)n, (uint32_t)p.padded,                         \
        (nz_bf16*)dev_workspace + first * a_stride);                                                              \
  })
    if (dtype == NZ_DTYPE_BF16)
      NZ_PLANES(1, nz_bf16);
    else if (dtype == NZ_DTYPE_F16)
      NZ_PLANES(2, nz_f16);
    else
      NZ_PLANES(3, float);
#undef NZ_PLANES
  }
  return launch_tiles16<true>(cut, a, a_stride, m, dev_w_data, dev_w_scales, n, k,
                              steps, p.count, k, nullptr, dev_dx, dtype, (uint8_t*)dev_workspace + p.bytes, st);
}

uint64_t nz_column_sums_workspace_bytes(uint64_t m, uint64_t n) {
  const uint32_t parts = sum_parts(m, n);
  return parts > 1 ? nz_mul(parts, nz_mul(n, 4)) : 0;
}

int nz_column_sums(const void* dev_x, int dtype, uint64_t m, uint64_t n, uint64_t stride, void* dev_out,
                   void* dev_workspace, uint64_t workspace_bytes, void* stream) {
  if (int rc = check_dtype(dtype, dev_x, dev_out, nullptr)) return rc;
  if (n == 0) return NZ_OK;
  if (!dev_out || (m && !dev_x)) return nz_fail(NZ_ERR_ARG, "null input or output");
  if (m > 1u << 30 || n > 1u << 30) return nz_fail(NZ_ERR_ARG, "too many rows or columns");
  if (int rc = check_workspace(dev_workspace, workspace_bytes, nz_column_sums_workspace_bytes(m, n))) return rc;
  const hipStream_t st = (hipStream_t)stream;
  const uint32_t parts = sum_parts(m, n), slices = (uint32_t)nz_ceil_div(n, 512);
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const T* x = (const T*)dev_x;
    T* out = (T*)dev_out;
    float* part = (float*)dev_workspace;
    if (parts == 1) {
      nz_mx_column_sums_kernel<T, T><<<slices, 256, 0, st>>>(x, stride, (uint32_t)m, (uint32_t)n, (uint32_t)m, out);
    } else {
      nz_mx_column_sums_kernel<T, float><<<dim3(slices, parts), 256, 0, st>>>(
          x, stride, (uint32_t)m, (uint32_t)n, (uint32_t)nz_ceil_div(m, parts), part);
      nz_mx_column_sums_kernel<float, T><<<slices, 256, 0, st>>>(part, n, parts, (uint32_t)n, parts, out);
    }
  });
  return nz_launched();
}

}  // extern "C"
