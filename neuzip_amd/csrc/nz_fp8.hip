// Tensors in 8 bits with a scale for each block of 128: quantisation, values, products with activation rows and their
// gradients, the gradient of a dense weight from rows that were kept in 8 bits, activation functions that keep theirs.
//
// The format is stated in include/neuzip_hip.h.  A row's codes lie in order and are filled up to 128 values, one step
// of the scaled matrix instruction, which takes the scale of a block as it is: powers of two, one a step and row.  The
// scales of four successive blocks of a row are 4 bytes, what a lane loads for four steps.  Weights have one scale for
// 128 rows (`shift` = 7) or one for each (0); which, costs the kernels nothing.
#include "nz_products.h"

namespace {

constexpr uint32_t kStep = 128;   // values of a row that one matrix instruction takes, and that share a scale
constexpr uint32_t kGroup = 512;  // values of a row whose scales are 4 consecutive bytes

// Scale byte of a block from the bits of its largest magnitude: the exponent, one more where it is beyond 1.75 (448 is
// 1.75 * 2^8), less 8.  A subnormal has exponent bits 0, which the clamp takes to the smallest scale as well.
__device__ inline uint32_t scale_byte(uint32_t amax_bits) {
  return amax_bits >= 0x7F800000u ? 255u : (uint32_t)max((int)((amax_bits + 0x1FFFFFu) >> 23) - 8, 0);
}

__device__ inline uint32_t top8(const float (&v)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  return top;
}

// the largest among 16 lanes
__device__ inline uint32_t max16(uint32_t top) {
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xB1, 0xF, 0xF, true));   // lane ^ 1
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4E, 0xF, 0xF, true));   // lane ^ 2
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x141, 0xF, 0xF, true));  // 7 - lane of 8
  return max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x140, 0xF, 0xF, true));  // 15 - lane of 16
}

// Scale byte of a block that 16 lanes share, 8 values each; a block that reads as NaN is cleared.
__device__ inline uint32_t block_scale(float (&v)[8]) {
  const uint32_t s = scale_byte(max16(top8(v)));
  if (s == 255)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
  return s;
}

// With the largest scale byte that finite values have, what is 31/32 of 2^128 or more is held as 256 times 2^120.  No 32
// bits hold that; where it goes into sums (and would make infinity times zero of a masked place) it counts as the largest
// bf16 number.  (The look for that byte costs the gradient of a weight 1 to 2 %, one row of 14336x4096 in float32 0.6 of
// 16.6 us.)
constexpr uint32_t kTopScale = 247;
__device__ inline void below_infinity(float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = __float_as_uint(v[i]);
    if ((u & 0x7FFFFFFFu) == 0x7F800000u) v[i] = __uint_as_float(u - 0x10000u);
  }
}
__device__ inline void below_infinity(b8v& v) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint16_t u = __builtin_bit_cast(uint16_t, (nz_bf16)v[i]);
    if ((u & 0x7FFF) == 0x7F80) v[i] = __builtin_bit_cast(nz_bf16, (uint16_t)(u - 1));
  }
}

// Values of 8 codes, 2^128 as it is (infinity) or, FINITE, as above.  The conversion takes the exponent field of its
// scale: a scale byte there is what it means.
template <bool FINITE = true>
__device__ inline void values_of(uint2 codes, uint32_t s, float (&v)[8]) {
  const float scale = __uint_as_float(s << 23);
  const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes.x, scale, false);
  const f2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes.x, scale, true);
  const f2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes.y, scale, false);
  const f2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes.y, scale, true);
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
  if (FINITE && s == kTopScale) below_infinity(v);
}

// ---- quantisation and values -----------------------------------------------------------------------------------
//
// One wavefront per 512 values of a row: 8 values a lane, 16 lanes a block.  Memory bounds them: 8192x4096 of bf16 to
// rows in 8 bits 22 to 24 us (4.3 TB/s), 16384x4096 to values 29.8 (6.8 TB/s, written and read; a fill reaches 6.8).

// Division of the number of a wavefront, below 2^26 in one launch, by the groups of 512 values in a row: n / d is
// n mul >> shift with mul = floor(2^shift / d) + 1 and 2^shift >= 2^26 d, for then n (mul d - 2^shift) < 2^shift.
// (In 64 bits as it is, it takes more instructions than what follows.)
struct Groups {
  uint32_t count, mul, shift;
};
struct Place {
  uint64_t row;
  uint32_t at;  // column of the lane's first value
};
__device__ inline Place place_of(uint32_t wave, const Groups& g) {
  const uint32_t n = __builtin_amdgcn_readfirstlane(wave);
  const uint32_t row = (uint32_t)((uint64_t)n * g.mul >> g.shift);
  return Place{row, (n - row * g.count) * kGroup + (threadIdx.x & 63) * 8};
}

// Codes and scale of 8 values of a row (`at` its first one's column, a multiple of 8) by a lane of such a wavefront.
__device__ inline void hold(float (&v)[8], Place at, uint32_t cols, uint32_t groups, uint8_t* data, uint8_t* scales) {
  const uint32_t s = block_scale(v), filled = (cols + kStep - 1) / kStep * kStep;
  if (at.at < filled) *reinterpret_cast<uint2*>(data + at.row * filled + at.at) = codes8(v, up_factor(s));
  if (at.at % kStep == 0) scales[at.row * (groups * 4ull) + at.at / kStep] = (uint8_t)s;
}

template <class T>
__global__ __launch_bounds__(256) void nz_fp8_quantize_kernel(const T* x, uint64_t stride, uint32_t cols,
                                                              uint32_t waves, Groups groups, uint8_t* data,
                                                              uint8_t* scales) {
  const uint32_t wave = blockIdx.x * 4 + threadIdx.x / 64;
  if (wave >= waves) return;
  const Place p = place_of(wave, groups);
  float v[8];
  load8_upto(x + p.row * stride + p.at, p.at < cols ? cols - p.at : 0, v);
  hold(v, p, cols, groups.count, data, scales);
}

// A workgroup per block of 128 x 128 values, which stay in registers between the search for the largest and the
// rounding: 16 lanes a row, 16 rows at a time.  16384x4096 of bf16: 42.5 us, 4.7 TB/s read and written (a large copy:
// 5.15).
template <class T>
__global__ __launch_bounds__(256) void nz_fp8_quantize_blocks_kernel(const T* x, uint64_t stride, uint64_t rows,
                                                                     uint32_t cols, uint32_t blocks, uint32_t pitch,
                                                                     uint8_t* data, uint8_t* scales) {
  const uint32_t down = blockIdx.x / blocks, across = blockIdx.x - down * blocks;
  const uint32_t at = across * kStep + threadIdx.x % 16 * 8, n = at < cols ? cols - at : 0;
  const uint64_t first = down * 128ull + threadIdx.x / 16;
  typename Pack<T>::type raw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const T* p = x + min(first + i * 16, rows - 1) * stride + at;
    if (n >= 8) {
      raw[i] = *(const typename Pack<T>::type*)p;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) raw[i][e] = (uint32_t)e < n ? p[e] : (T)0.0f;
    }
  }
  uint32_t top = 0;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)raw[i][e];
    top = max(top, top8(v));  // a row behind the last is the last one once more
  }
  top = max16(top);
  top = max(top, (uint32_t)__shfl_xor((int)top, 16));
  top = max(top, (uint32_t)__shfl_xor((int)top, 32));
  __shared__ uint32_t tops[4];
  if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
  __syncthreads();
  const uint32_t s = scale_byte(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
  const float up = up_factor(s);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint64_t row = first + i * 16;
    asm volatile("" : "+v"(raw[i]));  // converted again instead of kept in 32 bits: twice the wavefronts
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = s == 255 ? 0.0f : (float)raw[i][e];
    if (row < rows) *reinterpret_cast<uint2*>(data + row * (blocks * 128ull) + at) = codes8(v, up);
  }
  uint8_t* to = scales + (uint64_t)down * pitch + across;
  if (threadIdx.x == 0) *to = (uint8_t)s;
  if (across + 1 == blocks && threadIdx.x > 0 && across + threadIdx.x < pitch) to[threadIdx.x] = 0;
}

template <bool FINITE, class T>
__global__ __launch_bounds__(256) void nz_fp8_values_kernel(const uint8_t* data, const uint8_t* scales, uint32_t shift,
                                                            uint64_t first, uint32_t cols, uint32_t waves,
                                                            Groups groups, T* out) {
  const uint32_t wave = blockIdx.x * 4 + threadIdx.x / 64;
  if (wave >= waves) return;
  const Place p = place_of(wave, groups);
  const uint64_t row = first + p.row;
  const uint32_t at = p.at;
  if (at >= cols) return;
  const uint32_t filled = (cols + kStep - 1) / kStep * kStep;
  float v[8];
  values_of<FINITE>(*reinterpret_cast<const uint2*>(data + row * filled + at),
                    scales[(row >> shift) * (groups.count * 4ull) + at / kStep], v);
  store8_upto(out + row * cols + at, cols - at, v);
}

// ---- activation functions --------------------------------------------------------------------------------------
//
// f(x) = x p(x) with p between 0 and 1; p and f' from one exponential and one reciprocal.

constexpr float kLog2E = 1.44269504f, kLog2ERest = 1.92596299e-8f, kLn2 = 0.693147181f;

// exp(x), x finite or not.  For float32 the rounding of the exponent (its magnitude times 2^-24) counts: what it
// loses is put back as a factor.
template <bool FINE>
__device__ inline float exp_of(float x) {
  const float h = x * kLog2E;
  const float e = __builtin_amdgcn_exp2f(h);
  if constexpr (!FINE) return e;
  const float l = __builtin_fmaf(x, kLog2ERest, __builtin_fmaf(x, kLog2E, -h));
  return fabsf(h) < 126.0f ? __builtin_fmaf(e, l * kLn2, e) : e;
}

// p(x), and f'(x) where SLOPE.  The slope is asked for of what is held in 8 bits, which is finite or NaN.
template <int KIND, bool FINE, bool SLOPE>
__device__ inline float gate(float x, float& slope) {
  if constexpr (KIND == NZ_ACTIVATION_GELU) {
    // p is the normal distribution's integral.  Below zero it is exp(-x^2 / 2) r(t), r(t) = t times a polynomial in
    // t = 1 / (1 + c |x|), fitted to the least relative error from 0 to -14 (3.2e-8, for results of 16 bits 1.5e-07; the
    // integral is below 2^-126 from -13 on).
    constexpr float k[9] = {0.139621407f,  0.139861897f,  0.119832724f, 0.105508536f, -0.0231109783f,
                            0.159175649f, -0.25571543f, 0.143972203f, -0.0291460212f};
    constexpr float k16[8] = {0.119629294f, 0.120754004f, 0.0999131426f, 0.128562927f,
                              -0.0536863729f, 0.206356779f, -0.15720515f, 0.0356753133f};
    // (FINE subtracts squares, which must not overflow)
    const float a = FINE ? fminf(fabsf(x), 30.0f) : fabsf(x);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(FINE ? 0.35f : 0.3f, a, 1.0f));
    float r = FINE ? k[8] : k16[7];
#pragma unroll
    for (int i = FINE ? 7 : 6; i >= 0; --i) r = __builtin_fmaf(r, t, FINE ? k[i] : k16[i]);
    const float square = a * a;
    float e;
    if constexpr (FINE) {
      e = exp_of<true>(-0.5f * square);
      e = __builtin_fmaf(e, -0.5f * __builtin_fmaf(a, a, -square), e);
    } else {
      e = __builtin_amdgcn_exp2f(square * (-0.5f * kLog2E));
    }
    const float tail = e * (r * t), p = x > 0.0f ? 1.0f - tail : tail;
    if constexpr (SLOPE) slope = __builtin_fmaf(x * e, 0.398942280f, p);
    return p;
  } else {
    // p = 1 / (1 + exp(-u)); u = x, or 2 sqrt(2 / pi) (x + 0.044715 x^3).  With t = exp(-|u|), which does not overflow,
    // p is 1 / (1 + t) or t / (1 + t), and p (1 - p) is t / (1 + t)^2.
    constexpr float c = 1.59576912f;
    const float square = x * x;
    const float u = KIND == NZ_ACTIVATION_SILU ? x : c * x * __builtin_fmaf(0.044715f, square, 1.0f);
    const float t = exp_of<FINE>(-fabsf(u)), q = __builtin_amdgcn_rcpf(1.0f + t), r = t * q, p = u >= 0.0f ? q : r;
    if constexpr (SLOPE) {
      const float du = KIND == NZ_ACTIVATION_SILU ? 1.0f : c * __builtin_fmaf(3 * 0.044715f, square, 1.0f);
      // x du, which may overflow, is below 3 |u|, and t is zero where that is above 1000
      slope = __builtin_fmaf(__builtin_amdgcn_fmed3f(x * du, -1000.0f, 1000.0f), r * q, p);
    }
    return p;
  }
}

// y = f(x), times `up` where GATED; x (and `up`) in 8 bits, where they are to be kept.  A wavefront per 512 values of a
// row, as above.
//
// Instructions bound gelu (8192x4096 of bf16: 35.5 to 37 us, 4.5 to 4.7 TB/s, and 35.4 to 37.7 back), memory silu with
// a second factor (2048x14336: 43 and 39.7 us, 5.5 and 5.9 TB/s; a large copy: 5.2).
template <int KIND, bool GATED, class T>
__global__ __launch_bounds__(256) void nz_fp8_activation_kernel(const T* x, uint64_t stride, const T* up,
                                                                uint64_t up_stride, uint32_t cols, uint32_t waves,
                                                                Groups groups, T* y, uint8_t* x_data,
                                                                uint8_t* x_scales, uint8_t* up_data,
                                                                uint8_t* up_scales) {
  const uint32_t wave = blockIdx.x * 4 + threadIdx.x / 64;
  if (wave >= waves) return;
  const Place p = place_of(wave, groups);
  const uint64_t row = p.row;
  const uint32_t at = p.at, n = at < cols ? cols - at : 0;
  float v[8], u[8], f[8], none;
  load8_upto(x + row * stride + at, n, v);
  if constexpr (GATED) load8_upto(up + row * up_stride + at, n, u);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f[i] = v[i] * gate<KIND, std::is_same<T, float>::value, false>(v[i], none);
    if constexpr (GATED) f[i] *= u[i];
  }
  if (n) store8_upto(y + row * cols + at, n, f);
  if (!x_data) return;
  hold(v, p, cols, groups.count, x_data, x_scales);
  if constexpr (GATED) hold(u, p, cols, groups.count, up_data, up_scales);
}

// dx = g f'(x), times `up` where GATED, and dup = g f(x).
template <int KIND, bool GATED, class T>
__global__ __launch_bounds__(256) void nz_fp8_activation_grad_kernel(const T* g, uint64_t stride, uint32_t cols,
                                                                     uint32_t waves, Groups groups,
                                                                     const uint8_t* x_data, const uint8_t* x_scales,
                                                                     const uint8_t* up_data, const uint8_t* up_scales,
                                                                     T* dx, T* dup) {
  const uint32_t wave = blockIdx.x * 4 + threadIdx.x / 64;
  if (wave >= waves) return;
  const Place p = place_of(wave, groups);
  const uint64_t row = p.row;
  const uint32_t at = p.at;
  if (at >= cols) return;
  const uint32_t n = cols - at, filled = (cols + kStep - 1) / kStep * kStep;
  const uint64_t code = row * filled + at, scale = row * (groups.count * 4ull) + at / kStep;
  float v[8], u[8], d[8], a[8], b[8];
  load8_upto(g + row * stride + at, n, d);
  const uint32_t sx = x_scales[scale], su = GATED ? up_scales[scale] : 0;
  values_of<false>(*reinterpret_cast<const uint2*>(x_data + code), sx, v);
  if constexpr (GATED) values_of<false>(*reinterpret_cast<const uint2*>(up_data + code), su, u);
  if (sx == kTopScale || su == kTopScale) {  // (one look for both)
    below_infinity(v);
    if constexpr (GATED) below_infinity(u);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float slope;
    const float f = gate<KIND, std::is_same<T, float>::value, true>(v[i], slope);
    if constexpr (GATED) {
      a[i] = d[i] * slope * u[i];  // d u may overflow where the slope is zero
      b[i] = d[i] * (v[i] * f);
    } else {
      a[i] = d[i] * slope;
    }
  }
  store8_upto(dx + row * cols + at, n, a);
  if constexpr (GATED) store8_upto(dup + row * cols + at, n, b);
}

// ---- product ---------------------------------------------------------------------------------------------------
//
// The matrix instruction takes 16 rows of each side and 128 values of a row.  A lane (r = lane % 16, g = lane / 16)
// holds, of row r, values 16 g .. 16 g + 15 and 64 + 16 g .. 64 + 16 g + 15, and on both sides the row's scale.  Of the
// result it holds weight rows 4 g .. 4 g + 3 against activation row r.
//
// The instruction adds eight consecutive products at a time, each cut, toward zero, 13 places behind the largest
// exponent of the eight; 32 bits hold the rest.  Results of 16 bits are made with it for its rate; results in float32
// by bf16 instructions on the same values, which bf16 holds exactly.

__device__ inline f4 step(i4v w0, i4v w1, i4v x0, i4v x1, f4 acc, uint32_t sw, uint32_t sx, int byte) {
  const i8v a = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
  const i8v b = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
  switch (byte) {  // a constant where this is inlined
    case 0: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 0, 0, 0, (int)sw, 0, (int)sx);
    case 1: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 0, 0, 1, (int)sw, 1, (int)sx);
    case 2: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 0, 0, 2, (int)sw, 2, (int)sx);
    default: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 0, 0, 3, (int)sw, 3, (int)sx);
  }
}

// 8 codes as bf16 numbers, by such a conversion too (2^128 as infinity: below_infinity).
__device__ inline b8v bf16_of_codes(uint2 codes, uint32_t s) {
  const float scale = __uint_as_float(s << 23);
  const b2v a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes.x, scale, false);
  const b2v b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes.x, scale, true);
  const b2v c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes.y, scale, false);
  const b2v d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes.y, scale, true);
  return b8v{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// A tile of WM TM x WN TN matrix instructions' results, WM x WN wavefronts with TM x TN each.
//
// The rows of both sides are staged through LDS in steps of 128 values, NS stages deep, by loads that go to LDS
// without registers; a wavefront counts its own loads down, and one barrier a step tells that everybody's have
// arrived and that the stage before is used up.  Staged rows are exchanged in chunks of 16 bytes (chunk c of row r at
// c ^ (r & 7)) so that eight lanes in turn read from all banks, and the weight rows of a wavefront are staged in an
// order that leaves each lane 4 TN consecutive columns of the result.  Scales are staged once per 512 values.
//
// 64 x (4096x14336) in tiles of 64x64 and 4 parts: 12.2 to 13.6 us, the weight at 4.3 to 4.8 TB/s (3.1 more for the rows,
// 2.2 to 4 for the join).  Of larger products 256x256 (below) gives more where k is a multiple of 512; the figures at
// `kTiles` decide.
template <int WM, int WN, int TM, int TN, int NS, int EU, class T>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(EU, EU))) void nz_fp8_tiles_kernel(
    const uint8_t* xd, const uint8_t* xs, uint32_t m, const uint8_t* wd, const uint8_t* ws, uint32_t shift, uint32_t n,
    uint32_t k, const T* bias, T* y, uint32_t mt, uint32_t nt, uint32_t part_groups, float* part) {
  constexpr int W = WM * WN, BM = WM * TM * 16, BN = WN * TN * 16;
  constexpr int XB = BM * 128, STAGE = (BM + BN) * 128;
  constexpr int XI = BM / 8 / W, WI = BN / 8 / W, LOADS = XI + WI;
  constexpr int SI = (BM + BN) / 64, SB = SI * 256;  // scales: 64 rows of 4 bytes a load
  constexpr int SL = (SI + W - 1) / W;               // of a wavefront
  static_assert(XI * 8 * W == BM && WI * 8 * W == BN, "loads per wavefront");
  static_assert(BM % 64 == 0 && BN % 64 == 0, "a load takes scales of one side");
  static_assert(NS >= 2 && NS <= 4, "a group's scales are asked for when the last group's have been read");
  constexpr int STAGES = NS * STAGE + SB, OUT = BM * (BN * (int)sizeof(T) + 16), LDS = STAGES > OUT ? STAGES : OUT;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[LDS];
  const uint32_t base = lds_address(lds);
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t r = lane & 15, g = lane / 16;
  const uint32_t all_steps = (k + kStep - 1) / kStep, pitch = (k + kGroup - 1) / kGroup * 4;
  const uint32_t from = blockIdx.y * part_groups, steps = min(all_steps - from * 4, part_groups * 4);
  uint32_t tm, tn;
  tile_of(blockIdx.x, mt, nt, tm, tn);
  const uint32_t m0 = tm * BM, n0 = tn * BN;
  const uint32_t m_last = min((uint32_t)BM, m - m0) - 1, n_last = min((uint32_t)BN, n - n0) - 1;

  // Where this lane loads from: a base of the workgroup and an offset.  Rows behind the last one are read as the last.
  const uint8_t* xb = xd + (uint64_t)m0 * (all_steps * 128ull) + from * 512ull;
  const uint8_t* wb = wd + (uint64_t)n0 * (all_steps * 128ull) + from * 512ull;
  const auto column = [](uint32_t row) {  // of the tile, for a staged weight row
    return row / (TN * 16) * (TN * 16) + row % 16 / 4 * (TN * 4) + row / 16 % TN * 4 + row % 4;
  };
  uint32_t xo[XI], wo[WI];
#pragma unroll
  for (int i = 0; i < XI; ++i)
    xo[i] = min((wave * XI + i) * 8 + lane / 8, m_last) * (all_steps * 128) + ((lane & 7) ^ (lane / 8)) * 16;
#pragma unroll
  for (int i = 0; i < WI; ++i)
    wo[i] = min(column((wave * WI + i) * 8 + lane / 8), n_last) * (all_steps * 128) + ((lane & 7) ^ (lane / 8)) * 16;
  // where wavefronts and loads of scales do not match, some load the same
  const uint8_t* sb[SL];
  uint32_t so[SL], si[SL];
#pragma unroll
  for (int i = 0; i < SL; ++i) {
    si[i] = (i * W + wave) % SI;
    const uint32_t row = si[i] * 64 + lane, of_w = min(column(row - BM), n_last) + n0;
    sb[i] = si[i] * 64 < BM ? xs + (uint64_t)m0 * pitch + from * 4 : ws + (uint64_t)(n0 >> shift) * pitch + from * 4;
    so[i] = (si[i] * 64 < BM ? min(row, m_last) : (of_w >> shift) - (n0 >> shift)) * pitch;
  }
  const auto load_stage = [&](uint32_t s, uint32_t buf, bool scales) {
    s = min(s, steps - 1);  // past the end the last stage is loaded again, into a buffer that is not read
    const uint32_t to = base + buf * STAGE;
#pragma unroll
    for (int i = 0; i < XI; ++i) to_lds16(xb + s * 128ull, xo[i], to + (wave * XI + i) * 1024);
#pragma unroll
    for (int i = 0; i < WI; ++i) to_lds16(wb + s * 128ull, wo[i], to + XB + (wave * WI + i) * 1024);
    if (scales) {
#pragma unroll
      for (int i = 0; i < SL; ++i) to_lds4(sb[i] + (s >> 2) * 4, so[i], base + NS * STAGE + si[i] * 256);
    }
  };

  const uint32_t wm = wave % WM, wn = wave / WM;
  f4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f4{0, 0, 0, 0};
  uint32_t sx[TM], sw[TN];
  const uint32_t c0 = (g ^ (r & 7)) * 16, c1 = c0 ^ 64;
  const uint32_t xr = (wm * TM * 16 + r) * 128, wr = XB + (wn * TN * 16 + r) * 128;

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
      for (int i = 0; i < TM; ++i) sx[i] = *(const uint32_t*)(st + (wm * TM * 16 + i * 16 + r) * 4);
#pragma unroll
      for (int j = 0; j < TN; ++j) sw[j] = *(const uint32_t*)(st + (BM + wn * TN * 16 + j * 16 + r) * 4);
    }
    i4v x0[TM], x1[TM], w0[TN], w1[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      x0[i] = *(const i4v*)(b + xr + i * 2048 + c0);
      x1[i] = *(const i4v*)(b + xr + i * 2048 + c1);
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      w0[j] = *(const i4v*)(b + wr + j * 2048 + c0);
      w1[j] = *(const i4v*)(b + wr + j * 2048 + c1);
    }
    load_stage(s + NS - 1, buf == 0 ? NS - 1 : buf - 1, (byte + NS - 1) % 4 == 0);
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i) acc[i][j] = step(w0[j], w1[j], x0[i], x1[i], acc[i][j], sw[j], sx[i], byte);
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

  finish_tile<WM, WN, TM, TN, LDS>(acc, lds, m, n, m0, n0, bias, y, part);
}

__device__ inline i8v both(i4v a, i4v b) { return i8v{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}; }

// `step` in assembly: the sum stays in the registers it is in, of the kind that only such instructions use.  (Where sums
// fill half of all registers the compiler, which may choose others for each instruction's result, moves them about.)
// What reads a sum, and the first instruction behind a write of its registers, has to wait: `settle`.
template <int BYTE>
__device__ inline void step_in_place(i8v w, i8v x, f4& acc, uint32_t sw, uint32_t sx) {
  asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%5,0] op_sel_hi:[%6,%6,0]"
               : "+a"(acc)
               : "v"(w), "v"(x), "v"(sw), "v"(sx), "n"(BYTE & 1), "n"(BYTE >> 1));
}
__device__ inline void settle() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

// The same for the largest products, whose results are of 16 bits: tiles of 256x256, four wavefronts of 128x128 each, a
// compute unit's own, and every workgroup goes through several of them.  k is a multiple of 512.
//
// What a wavefront reads of LDS for its matrix instructions is the less the larger its tile: 32 KB a step for 64
// instructions (2048 cycles), where 64x64 take 16 KB for 16.  A step's 64 squares are multiplied a row of x at a time, in
// four places that are read again as soon as they are used up; w's eight follow beside the last row.  From the sixth row
// on what is read is of the next step: before it is the step's only barrier, which tells that the stage behind has
// arrived and that this one has been read, so that the loads of the stage after the next go there.  Steps follow each
// other across tiles: the loads run ahead into the next tile, whose first operands are there when the result has been
// stored.  It goes through a part of LDS that is each wavefront's own, 16 rows at a time.
//
// 8192 x (14336x4096): 360 to 376 us where passes go on without a pause, 2.56 to 2.67 PFLOP/s (a library's 8-bit product
// of these sizes 315 to 329; k = 4000 in the tiles of 128x256 above 416).  One by itself takes 374 to 384, and of passes
// that begin behind a pause the first fifty up to 510, while the card settles its clock (the library's first twenty 415).
// Of that some 50 are the stores of the results, in which all compute units meet seven times; letting them start apart by
// up to half a tile gained nothing.
template <class T>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void nz_fp8_wide_kernel(
    const uint8_t* xd, const uint8_t* xs, uint32_t m, const uint8_t* wd, const uint8_t* ws, uint32_t shift, uint32_t n,
    uint32_t k, const T* bias, T* y, uint32_t mt, uint32_t nt) {
  constexpr int SIDE = 256, XB = SIDE * 128, STAGE = 2 * XB, S_AT = 2 * STAGE, OUT_AT = S_AT + 2 * SIDE * 4;
  constexpr int PITCH = 128 * (int)sizeof(T) + 16;  // a row of a wavefront's part of the result
  static_assert(sizeof(T) == 2 && OUT_AT + 4 * 16 * PITCH <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[OUT_AT + 4 * 16 * PITCH];
  const uint32_t base = lds_address(lds);
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t r = lane & 15, g = lane / 16, wm = wave & 1, wn = wave / 2;
  const uint32_t groups = k / kGroup, pitch = groups * 4, tiles = mt * nt;

  // Where a lane loads a tile from: bases of the workgroup, moved from step to step, and offsets.  Rows behind the last
  // one are read as the last.
  const uint8_t *xb, *wb, *sb;
  uint32_t xo[8], wo[8], so[2];
  const auto column = [](uint32_t row) {  // of the tile, for a staged weight row: a lane ends with 32 consecutive ones
    return row / 128 * 128 + row % 16 / 4 * 32 + row / 16 % 8 * 4 + row % 4;
  };
  const auto aim = [&](uint32_t tile, uint32_t group) {
    uint32_t tm, tn;
    tile_of(tile, mt, nt, tm, tn);
    const uint32_t m0 = tm * SIDE, n0 = tn * SIDE;
    const uint32_t m_last = min((uint32_t)SIDE, m - m0) - 1, n_last = min((uint32_t)SIDE, n - n0) - 1;
    xb = xd + (uint64_t)m0 * k + group * kGroup, wb = wd + (uint64_t)n0 * k + group * kGroup;
    const uint32_t chunk = ((lane & 7) ^ (lane / 8)) * 16;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t row = (wave * 8 + i) * 8 + lane / 8;
      xo[i] = __umul24(min(row, m_last), k) + chunk;
      wo[i] = __umul24(min(column(row), n_last), k) + chunk;
    }
    // wavefronts 0 and 1 load the scales of x, the others those of w
    sb = wave < 2 ? xs + (uint64_t)m0 * pitch : ws + (uint64_t)(n0 >> shift) * pitch;
    sb += group * 4;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t row = (wave % 2 * 2 + i) * 64 + lane;
      so[i] = (wave < 2 ? min(row, m_last) : ((min(column(row), n_last) + n0) >> shift) - (n0 >> shift)) * pitch;
    }
  };
  const auto load_x = [&](uint32_t buf, int i) { to_lds16(xb, xo[i], base + buf * STAGE + (wave * 8 + i) * 1024); };
  const auto load_w = [&](uint32_t buf, int i) { to_lds16(wb, wo[i], base + buf * STAGE + XB + (wave * 8 + i) * 1024); };
  const auto load_scales = [&]() {
#pragma unroll
    for (int i = 0; i < 2; ++i) to_lds4(sb, so[i], base + S_AT + (wave * 2 + i) * 256);
  };

  f4 acc[8][8];
  i8v x[4], w[8];
  uint32_t sx[8], sw[8];
  const uint32_t c0 = (g ^ (r & 7)) * 16, c1 = c0 ^ 64;
  const uint32_t xr = (wm * 128 + r) * 128, wr = XB + (wn * 128 + r) * 128;
  const auto read_x = [&](uint32_t buf, int i) {
    x[i % 4] = both(*(const i4v*)(lds + buf * STAGE + xr + i * 2048 + c0),
                    *(const i4v*)(lds + buf * STAGE + xr + i * 2048 + c1));
  };
  const auto read_w = [&](uint32_t buf, int j) {
    w[j] = both(*(const i4v*)(lds + buf * STAGE + wr + j * 2048 + c0),
                *(const i4v*)(lds + buf * STAGE + wr + j * 2048 + c1));
  };
  const auto read_scales = [&]() {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sx[i] = *(const uint32_t*)(lds + S_AT + (wm * 128 + i * 16 + r) * 4);
      sw[i] = *(const uint32_t*)(lds + S_AT + SIDE * 4 + (wn * 128 + i * 16 + r) * 4);
    }
  };

  uint32_t tile = blockIdx.x;
  aim(tile, 0);
#pragma unroll
  for (int i = 0; i < 8; ++i) load_x(0, i), load_w(0, i);
  load_scales();
  xb += 128, wb += 128;
  wait_loads<0>();
  block_barrier();
#pragma unroll
  for (int i = 0; i < 8; ++i) read_w(0, i);
#pragma unroll
  for (int i = 0; i < 4; ++i) read_x(0, i);
  read_scales();
#pragma unroll
  for (int i = 0; i < 8; ++i) load_x(1, i), load_w(1, i);
  xb += 128, wb += 128;

  // A step, s % 4 of a tile; stage s is in buffer s % 2.  An empty statement that could change a result holds each
  // instruction in its place among the reads and loads.
  const auto body = [&](auto b4) {
    constexpr int byte = decltype(b4)::value, buf = byte % 2;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i == 5) {
        wait_loads<0>();  // the next stage
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        block_barrier();
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        step_in_place<byte>(w[j], x[i % 4], acc[i][j], sw[j], sx[i]);
        if (i == 7) read_w(buf ^ 1, j);
        if (i == 5 || i == 6) {
          if (i == 5) load_x(buf, j);
          else load_w(buf, j);
        }
        if (j == 7 && i < 4) read_x(buf, i + 4);
        if (j == 7 && i == 5) read_x(buf ^ 1, 0), read_x(buf ^ 1, 1);
        if (j == 7 && i > 5) read_x(buf ^ 1, i - 4);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (byte == 2) load_scales();
    if (byte == 3) read_scales();
    xb += 128, wb += 128;
  };
  using B0 = std::integral_constant<int, 0>;
  using B1 = std::integral_constant<int, 1>;
  using B2 = std::integral_constant<int, 2>;
  using B3 = std::integral_constant<int, 3>;
  for (;;) {
    uint32_t tm, tn;
    tile_of(tile, mt, nt, tm, tn);
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc[i][j] = f4{0, 0, 0, 0};
        asm volatile("" : "+a"(acc[i][j]));
      }
    settle();
    const bool more = tile + gridDim.x < tiles;
    const uint32_t next = more ? tile + gridDim.x : tile;  // behind the last tile its own begin, which is not used
    uint32_t i = 0;
    do {
      body(B0());
      body(B1());
      ++i;
      aim(i == groups ? next : tile, i == groups ? 0 : i);
      body(B2());
      body(B3());
    } while (i != groups);
    tile = next;
    settle();

    const uint32_t row0 = tm * SIDE + wm * 128, col0 = tn * SIDE + wn * 128;
    uint8_t* mine = lds + OUT_AT + wave * 16 * PITCH;
    typedef T whole __attribute__((ext_vector_type(8)));
    typedef T piece __attribute__((ext_vector_type(8), aligned(sizeof(T))));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) asm volatile("" : "+a"(acc[i][j]));  // they stay in their registers until here
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        float v[8], b[8] = {};
        const uint32_t c = col0 + g * 32 + j * 4;
        if (bias && c < n) load8_upto(bias + c, n - c, b);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = acc[i][j + e / 4][e % 4] + b[e];
        store8((T*)(mine + r * PITCH) + g * 32 + j * 4, v);
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t at = q * 4 + lane / 16, row = row0 + i * 16 + at, c = col0 + lane % 16 * 8;
        const whole v = *(const whole*)(mine + at * PITCH + lane % 16 * 16);
        if (row >= m || c >= n) continue;
        T* to = y + (uint64_t)row * n + c;
        if (c + 8 <= n)
          *(piece*)to = v;
        else
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c + e < n) to[e] = v[e];
      }
      __builtin_amdgcn_wave_barrier();
    }
    if (!more) break;
  }
  wait_loads<0>();  // nothing may arrive in this memory once it is another workgroup's
}

// Up to 16 rows, where reading the weight is all that counts: no staging and no barrier in the way of it.  The eight
// wavefronts are kw that share the values of a row (512 at a time, in turn) times 8 / kw with 16 weight rows each;
// a lane loads its operand of the matrix instruction straight from memory.  The rows come in 8 bits (N = 0), or
// as they are, at most 8 N groups of 512 values: then every workgroup brings them to 8 bits in LDS while its first weights
// are on their way.
// Results in float32 are summed by bf16 instructions (why, see `step`), for which a lane takes both sides to bf16: of
// the 128 values of a step those it holds, 8 at a time (both sides in the same order, which is all that counts).
//
// What bounds it is memory's way to few lines at a time: one row of 14336x4096 13.8 to 14.4 us (4.1 to 4.3 TB/s of the
// weight), 7 of 5003x3001 8.8 to 9.2, launches in a row (in a kernel trace, which adds to short ones, up to 15.3 and 10.6).
constexpr uint32_t kHeld = 528;  // bytes of 512 values of a row and their scales in LDS

template <int N, class T>
__global__ __launch_bounds__(512) void nz_fp8_few_kernel(const void* x, uint64_t stride, const uint8_t* xs, uint32_t m,
                                                         const uint8_t* wd, const uint8_t* ws, uint32_t shift,
                                                         uint32_t n, uint32_t k, const T* bias, T* y, uint32_t kw) {
  extern __shared__ __attribute__((aligned(16))) uint8_t few_lds[];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64, r = lane & 15, g = lane / 16;
  const uint32_t steps = (k + kStep - 1) / kStep, groups = (k + kGroup - 1) / kGroup;
  const uint32_t kwave = wave % kw, tile = blockIdx.x * (8 / kw) + wave / kw;
  const uint64_t w_row = min(tile * 16 + r, n - 1);
  const uint8_t* wp = wd + w_row * (steps * 128ull) + g * 16;
  const uint8_t* sp = ws + (w_row >> shift) * (groups * 4ull);
  struct Held {
    i4v w[4][2];
    uint32_t s;
  } a, b;
  const auto load = [&](Held& h, uint32_t group) {
    h.s = *(const uint32_t*)(sp + group * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* p = wp + (uint64_t)min(group * 4 + i, steps - 1) * 128;
      h.w[i][0] = *(const i4v*)p, h.w[i][1] = *(const i4v*)(p + 64);
    }
  };
  if (kwave < groups) load(a, kwave);

  constexpr bool kWide = std::is_same<T, float>::value;
  const uint32_t row = min(r, m - 1);
  const uint8_t *xp, *xsp;
  if constexpr (N > 0) {
    const T* xt = (const T*)x;
    typename Pack<T>::type raw[N];  // every eighth group of values of a wavefront, all on their way at once
#pragma unroll
    for (uint32_t j = 0; j < N; ++j) {
      const uint32_t i = wave + 8 * j, to = i / groups, at = (i - to * groups) * kGroup + lane * 8;
      raw[j] = {};
      if (i < m * groups && at + 8 <= k) raw[j] = *(const typename Pack<T>::type*)(xt + to * stride + at);
    }
#pragma unroll
    for (uint32_t j = 0; j < N; ++j) {
      const uint32_t i = wave + 8 * j, to = i / groups, at = (i - to * groups) * kGroup + lane * 8;
      if (i >= m * groups) break;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (float)raw[j][e];
      if (at < k && at + 8 > k) load8_upto(xt + to * stride + at, k - at, v);
      const uint32_t s = block_scale(v);
      uint8_t* q = few_lds + i * kHeld;
      *(uint2*)(q + lane * 8) = codes8(v, up_factor(s));
      if ((lane & 15) == 0) q[kGroup + lane / 16] = (uint8_t)s;
    }
    __syncthreads();
    xp = few_lds + row * groups * kHeld + g * 16;
    xsp = few_lds + row * groups * kHeld + kGroup;
  } else {
    xp = (const uint8_t*)x + row * (steps * 128ull) + g * 16;
    xsp = xs + row * (groups * 4ull);
  }
  f4 acc = {0, 0, 0, 0};
  const auto multiply = [&](const Held& h, uint32_t group) {
    const uint32_t sx = *(const uint32_t*)(xsp + group * (N ? kHeld : 4));
    const auto one = [&](auto b4) {
      constexpr int i = decltype(b4)::value;
      if (group * 4 + i >= steps) return;
      const uint8_t* p = xp + (N ? group * kHeld : (uint64_t)group * 512) + i * 128;
      const i4v x0 = *(const i4v*)p, x1 = *(const i4v*)(p + 64);
      if constexpr (kWide) {
        const uint32_t s = sx >> (8 * i) & 255, sw = h.s >> (8 * i) & 255;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const i4v xq = q < 2 ? x0 : x1, wq = h.w[i][q / 2];
          const uint2 xc = make_uint2(xq[q % 2 * 2], xq[q % 2 * 2 + 1]), wc = make_uint2(wq[q % 2 * 2], wq[q % 2 * 2 + 1]);
          b8v xv = bf16_of_codes(xc, s);
          if (s == kTopScale) below_infinity(xv);
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf16_of_codes(wc, sw), xv, acc, 0, 0, 0);
        }
      } else {
        acc = step(h.w[i][0], h.w[i][1], x0, x1, acc, h.s, sx, i);
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
// What the scaled instruction cannot do: the gradients, one of whose sides is not in 8 bits, and results in float32.
// What is held in 8 bits is exact in bf16; a gradient of 16 or 32 bits is the sum of two or three bf16 numbers, laid
// side by side along the summed axis.  (A float16 gradient does not go to float16 instructions as it is: they would take
// the codes, but not with their scales, which reach from 2^-127 to 2^125.)
//
// 8192 rows, 4096x1024, calls without a pause: the rows' gradient in bf16, float16 and float32 57 to 60, 130 and 224 us,
// the weight's 76 to 78, 157 and 233, a float32 result 90.

// What 8 bits of float32 rows stand for, as bf16 numbers, rows filled up to whole steps: the rows' side of a product
// with a float32 result.
__global__ __launch_bounds__(256) void nz_fp8_rounded_kernel(const float* x, uint64_t stride, uint32_t cols,
                                                             uint32_t waves, Groups groups, nz_bf16* out) {
  const uint32_t wave = blockIdx.x * 4 + threadIdx.x / 64;
  if (wave >= waves) return;
  const Place p = place_of(wave, groups);
  const uint32_t at = p.at;
  float v[8];
  load8_upto(x + p.row * stride + at, at < cols ? cols - at : 0, v);
  const uint32_t s = block_scale(v);
  values_of(codes8(v, up_factor(s)), s, v);
  const uint32_t filled = (cols + kStep - 1) / kStep * kStep;
  if (at < filled) store8(out + p.row * filled + at, v);
}

// Which product: x wT (a float32 result), g w (the gradient of the rows), gT x (the gradient of a weight).
enum Product { kForward, kInput, kWeight };

// A tile of C[m][cols] = sum over c of A(m, c) B(c, col), c running `planes` times through the summed axis.  B is held
// in 8 bits: kForward, b[col][c]; else b[c][col].  A is bf16: a[m][c], kWeight: a[c][m].
//
// Steps of 64 values.  A, codes and scales go to LDS without registers two steps ahead (16-byte chunk c of a row of A at
// c ^ (row & 7)); a step ahead, the codes are written to LDS once more as bf16, once for all wavefronts.  Where rows
// run along the summed axis the tile lies as in memory, and the operand is read by the instruction that transposes
// 4 x 16 values on the way.  A lane ends with 4 TN consecutive columns.
//
// The gradient of a 4096x1024 weight from 8192 rows, tiles of 256x128 in two parts: 76.5 to 80 us, 0.86 to 0.90 PFLOP/s
// (a library's bf16 product of the same sizes 85), and 7.3 for the join.  Matrix units are busy for 45 % of it, LDS for 43
// (11 of conflicts), and the wavefronts wait for a third of their time at the one barrier of a step.  Neither LDS nor memory
// alone bounds it: without conflicts (rows exchanging halves in every other eight), with half of what is fetched (tiles
// numbered two high) and with codes read half a step before they are converted it took 74 to 78.  Four wavefronts of
// 128x64, which read 96 KB of LDS a step instead of 128, took 82 (nothing covers what each waits for); tiles of 256x256 8 %
// less at 4096x4096, but four parts and so more at 4096x1024.
template <int WM, int WN, int TM, int TN, Product P, bool ADD, class T>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(2, 2))) void nz_fp8_tiles16_kernel(
    const nz_bf16* a, uint64_t a_stride, uint32_t a_width, uint64_t a_plane, uint32_t m, const uint8_t* bd,
    const uint8_t* bs, uint32_t shift, uint32_t b_rows, uint32_t b_cols, uint32_t steps_1, uint32_t planes,
    uint32_t cols, const T* bias, T* y, uint32_t mt, uint32_t nt, uint32_t part_steps, float* part) {
  constexpr bool ROWS = P != kForward, TURN = P == kWeight;
  constexpr int W = WM * WN, BM = WM * TM * 16, BN = WN * TN * 16, XI = BM / 8 / W, ROW = ROWS ? BN : 64;
  constexpr int CROWS = BN * 64 / ROW, OWN = CROWS / W;       // rows of codes a step, those of a wavefront
  constexpr int AB = BM * 128, BB = BN * 128, CB = BN * 64, SB = W * 256;  // bytes a step: A, bf16, codes, scales
  constexpr int B_AT = 3 * AB, C_AT = B_AT + 2 * BB, S_AT = C_AT + 3 * CB, LOADS = XI + 2;
  static_assert(XI * 8 * W == BM && BN * 64 == 16 * 64 * W, "16 rows of A and 16 codes per lane");
  static_assert(S_AT + 3 * SB <= 160 * 1024, "LDS");
  static_assert(OWN * W == CROWS && OWN % 8 == 0, "a wavefront writes the rows whose codes and scales it loads");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[S_AT + 3 * SB];
  const uint32_t base = lds_address(lds);
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t r = lane & 15, g = lane / 16;
  const uint32_t from = blockIdx.y * part_steps, steps = min(steps_1 * planes - from, part_steps);
  const uint32_t b_steps = (b_cols + kStep - 1) / kStep, b_bytes = b_steps * 128;
  const uint32_t pitch = (b_cols + kGroup - 1) / kGroup * 4;
  uint32_t tm, tn;
  tile_of(blockIdx.x, mt, nt, tm, tn);
  const uint32_t m0 = tm * BM, n0 = tn * BN, m_last = min((uint32_t)BM, m - m0) - 1;
  // ROWS: the last step of a plane may have fewer than 64 rows of its own.  TURN: it begins earlier, so that it has 64, of
  // which those that the step before had count as zeros.
  const uint32_t last_rows = b_rows - (steps_1 - 1) * 64, last_at = b_rows > 64 ? b_rows - 64 : 0;

  // Loads: a base of the workgroup, moved from step to step, and an offset of the lane.
  const auto turned = [](uint32_t row) { return ((row & 3) | (row >> 1 & 4)) * 2 % (BM / 8); };
  const uint8_t* ab = (const uint8_t*)a;
  if constexpr (!TURN) ab += (uint64_t)m0 * a_stride * 2 + from * 128ull;
  uint32_t ao[XI];
#pragma unroll
  for (int i = 0; i < XI; ++i) {
    if constexpr (TURN) {
      const uint32_t id = (wave * XI + i) * 64 + lane, row = id / (BM / 8), c = id % (BM / 8) ^ turned(row);
      const uint32_t col = min(m0 + c * 8, a_width - 8);
      ao[i] = (min(row, b_rows - 1) * (uint32_t)a_stride + col) * 2;
    } else {
      ao[i] = min((wave * XI + i) * 8 + lane / 8, m_last) * (uint32_t)(a_stride * 2) + ((lane & 7) ^ (lane / 8)) * 16;
    }
  }
  uint32_t a_step = from % steps_1, plane = from / steps_1;  // TURN: of the stage that is loaded next
  const auto a_base = [&]() { return ab + (plane * a_plane + min(a_step * 64, last_at) * a_stride) * 2; };
  const uint8_t* a_at = TURN ? a_base() : nullptr;
  const auto load_a = [&](uint32_t s, uint32_t buf, int i) {  // the i-th of XI
    const uint32_t to = base + buf * AB + (wave * XI + i) * 1024;
    // past the end the last stage is loaded again, into a buffer that is not read
    if constexpr (TURN) {
      to_lds16(a_at, ao[i], to);
      if (i == XI - 1 && s + 1 < steps) {
        const bool turn = a_step + 1 == steps_1;
        a_step = turn ? 0 : a_step + 1, plane += turn;
        a_at = a_base();
      }
    } else {
      to_lds16(ab + min(s, steps - 1) * 128ull, ao[i], to);
    }
  };
  // Codes: 16 bytes of a lane.  Scales: the four bytes that hold a row's, of the rows whose codes the wavefront loads;
  // lanes behind them load the last of these again.  A row's 16-byte chunks are exchanged (chunk c at c ^ mixed(row)) so
  // that eight lanes with eight rows read from all banks.
  const auto mixed = [](uint32_t row) { return ROW == 128 ? row & 7 : row >> 2 & 1; };
  uint32_t co, so, co_last, so_last;
  {
    const uint32_t row = threadIdx.x / (ROW / 16), c = threadIdx.x % (ROW / 16) ^ mixed(row);
    const uint32_t s_row = wave * OWN + min(lane, OWN - 1u);
    if constexpr (ROWS) {
      const uint32_t chunk = min(n0 / 16 + c, b_steps * 8 - 1), group = n0 / kGroup * 4;
      const uint32_t end = TURN ? b_rows : last_rows;
      co = (TURN ? min(row, end - 1) : row) * b_bytes + chunk * 16, co_last = min(row, end - 1) * b_bytes + chunk * 16;
      so = (s_row >> shift) * pitch + group, so_last = (min(s_row, end - 1) >> shift) * pitch + group;
      if constexpr (TURN) so = min(s_row, end - 1), so_last = group;
    } else {
      const auto place = [&](uint32_t id) {
        const uint32_t col = id / (TN * 16) * (TN * 16) + id % 16 / 4 * (TN * 4) + id / 16 % TN * 4 + id % 4;
        return min(n0 + col, b_rows - 1);
      };
      co = co_last = (place(row) - n0) * b_bytes + c * 16;
      so = so_last = ((place(s_row) >> shift) - (n0 >> shift)) * pitch;
      bd += (uint64_t)n0 * b_bytes, bs += (uint64_t)(n0 >> shift) * pitch;
    }
  }
  uint32_t w_step = from % steps_1;  // of the codes that are loaded next
  const auto load_b = [&](uint32_t buf) {
    const uint32_t row = TURN ? min(w_step * 64, last_at) : w_step * 64;
    const uint8_t* c = bd + (ROWS ? (uint64_t)row * b_bytes : w_step * 64ull);
    // steps begin at multiples of 64, so with a scale for 128 rows all of one have the same; TURN: not the last
    const uint8_t* s = bs + (ROWS ? (uint64_t)(row >> shift) * pitch : w_step / 8 * 4ull);
    const bool last = ROWS && w_step + 1 == steps_1;
    to_lds16(c, !TURN && last ? co_last : co, base + C_AT + buf * CB + wave * 1024);
    to_lds4(s, TURN ? (((row + so) >> shift) - (row >> shift)) * pitch + so_last : last ? so_last : so,
            base + S_AT + buf * SB + wave * 256);
    w_step = w_step + 1 == steps_1 ? 0 : w_step + 1;
  };
  // To bf16: 16 codes of a lane, neighbours' from eight rows.  Rows exchange 16-byte pieces (piece c of row r at
  // c ^ (r & 7)) so that eight lanes write to all banks; ROWS: in rows 2 and 3 of four, 8-byte halves of a piece as
  // well, so that the four rows of a transposing read do not meet.
  constexpr uint32_t ACROSS = ROW / 16;
  const uint32_t l_row = threadIdx.x / (8 * ACROSS) * 8 + threadIdx.x % 8, l_at = threadIdx.x / 8 % ACROSS;
  const bool swap = ROWS && (l_row & 2);
  const uint32_t c_at = C_AT + l_row * ROW + (l_at ^ mixed(l_row)) * 16;
  const uint32_t s_at = S_AT + wave * 256 + (l_row - wave * OWN) * 4;
  uint32_t to[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) to[j] = B_AT + l_row * (ROW * 2) + ((l_at * 2 + j) ^ (l_row & 7)) * 16;
  uint32_t c_step = from % steps_1;  // of the codes that are written next
  const auto convert = [&](uint32_t buf, uint32_t half) {
    const uint4 codes = *(const uint4*)(lds + c_at + buf * CB);
    const uint32_t scale = lds[s_at + buf * SB + (ROWS ? n0 / kStep & 3 : c_step / 2 & 3)];
    b8v first = bf16_of_codes(swap ? make_uint2(codes.y, codes.x) : make_uint2(codes.x, codes.y), scale);
    b8v second = bf16_of_codes(swap ? make_uint2(codes.w, codes.z) : make_uint2(codes.z, codes.w), scale);
    if (TURN && scale == kTopScale) below_infinity(first), below_infinity(second);  // rows; else a weight
    *(b8v*)(lds + to[0] + half * BB) = first;
    *(b8v*)(lds + to[1] + half * BB) = second;
    c_step = c_step + 1 == steps_1 ? 0 : c_step + 1;
  };
  // TURN: rows of A that a plane's last step has once more count as zeros.
  uint32_t z_step = from % steps_1;  // of the rows that are looked at next
  const auto clear = [&](uint32_t buf) {
    if constexpr (TURN) {
      if (z_step + 1 == steps_1 && last_rows < 64) {
        const uint32_t begin = b_rows < 64 ? b_rows : 0, end = b_rows < 64 ? 64 : 64 - last_rows;
        for (uint32_t at = begin * (BM * 2) + threadIdx.x * 16; at < end * (BM * 2); at += 64 * W * 16)
          *(i4v*)(lds + buf * AB + at) = i4v{0, 0, 0, 0};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        block_barrier();
      }
      z_step = z_step + 1 == steps_1 ? 0 : z_step + 1;
    }
  };

  const uint32_t wm = wave % WM, wn = wave / WM;
  f4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f4{0, 0, 0, 0};
  // operand addresses; the halves of a step lie at constant distances
  uint32_t ra[TURN ? TM * 2 : 2], rb[TN * 2];
  if constexpr (TURN) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint32_t row = g * 8 + q * 4 + r / 4, slot = (wm * TM + i) * 4 + r % 4;
        ra[i * 2 + q] = base + row * (BM * 2) + (slot ^ turned(row) * 2) * 8;
      }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) ra[h] = (wm * TM * 16 + r) * 128 + ((h * 4 + g) ^ (r & 7)) * 16;
  }
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint32_t row = g * 8 + q * 4 + r / 4, slot = wn * TN * 4 + r % 4 * TN + j;
      rb[j * 2 + q] = base + B_AT + row * (BN * 2) + (slot ^ (row & 7) * 2 ^ (row >> 1 & 1)) * 8;
    }
  const uint32_t rw = B_AT + (wn * TN * 16 + r) * 128;

  load_b(0);
#pragma unroll
  for (int i = 0; i < XI; ++i) load_a(0, 0, i);
  load_b(1);
#pragma unroll
  for (int i = 0; i < XI; ++i) load_a(1, 1, i);
  load_b(2);
  wait_loads<2 * LOADS>();  // codes of step 0
  block_barrier();
  convert(0, 0);
  wait_loads<LOADS>();  // rows of step 0, codes of step 1
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  block_barrier();
  clear(0);

  // Operands of a half step are read while the other half's are multiplied, across the barrier as well: behind it
  // the first half of step s + 1 while the second of step s is multiplied.
  struct Operands {
    b8v a[TM], b[TN];
  } first, second;
  constexpr int READS = TN + TM;
  const auto transposed = [&](const uint32_t* at, uint32_t more) {
    s4v part[2];
#pragma unroll
    for (int p = 0; p < 2; ++p)
      part[p] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s4v*)(uintptr_t)(at[p] + more));
    return __builtin_bit_cast(b8v, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
  };
  const auto read = [&](Operands& o, uint32_t buf, uint32_t odd, int h, int q) {  // the q-th of READS
    if (q >= TN) {
      if constexpr (TURN)
        o.a[q - TN] = transposed(ra + (q - TN) * 2, buf * AB + h * 64 * BM);
      else
        o.a[q - TN] = *(const b8v*)(lds + buf * AB + ra[h] + (q - TN) * 2048);
    } else if constexpr (ROWS) {
      o.b[q] = transposed(rb + q * 2, odd * BB + h * 64 * BN);
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
      if (t == M - 1) load_b(buf);
    });
    // behind the rows of step s + 1 and the codes of step s + 2: what has just been asked for
    wait_loads<LOADS>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    block_barrier();  // step s + 1 is in LDS, step s is used up
    clear(after);
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
  finish_tile<WM, WN, TM, TN, S_AT + 3 * SB, ADD, true>(acc, lds, m, cols, m0, n0, bias, y, part);
}

// `mfma` of bf16 in assembly, as step_in_place.
__device__ inline void step16_in_place(b8v b, b8v a, f4& acc) {
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(b), "v"(a));
}

// The gradient of the rows where 128 rows of the weight share a scale: tiles of 256 x 32 TN, four wavefronts of 128 x
// 16 TN each, a compute unit's own.
//
// In the kernel above much passes LDS: its wavefronts' tiles of 64x64 read 128 KB a step, and the codes go through it twice
// more.  Here a wavefront's tile is as large as its registers allow
// (96 KB a step of 256x128, 128 KB of 256x256), and codes are read as they are, eight of a column by the instruction that
// transposes 8 x 16 bytes on the way, and converted in the wavefront that multiplies them: a step has one scale.
//
// Steps of 64 values in two halves, whose operands are read while the other half's are multiplied.  In the middle is the
// step's barrier: the next step has arrived and this one has been read, so that the third behind it goes there, two steps
// ahead of its use.
//
// 8192 rows: 4096x1024 in tiles of 256x128 62 to 65 us, 1.08 PFLOP/s (68.5 by the kernel above), 4096x4096 in tiles of
// 256x256 191 us, 1.43 PFLOP/s (258).
template <int TN, class T>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void nz_fp8_input_kernel(
    const nz_bf16* a, uint64_t a_stride, uint32_t m, const uint8_t* bd, const uint8_t* bs, uint32_t b_rows,
    uint32_t b_cols, uint32_t steps_1, uint32_t planes, T* y, uint32_t mt, uint32_t nt, uint32_t part_steps,
    float* part) {
  constexpr int TM = 8, BM = 256, BN = TN * 32, M = TM * TN, CI = TN / 2;
  constexpr int AB = BM * 128, CB = BN * 64, S_AT = AB + CB, STAGE = S_AT + 1024, NS = 3, LOADS = 8 + CI + 1;
  static_assert(NS * STAGE <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[NS * STAGE];
  const uint32_t base = lds_address(lds);
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t r = lane & 15, g = lane / 16, wm = wave & 1, wn = wave / 2;
  const uint32_t from = blockIdx.y * part_steps, steps = min(steps_1 * planes - from, part_steps);
  const uint32_t b_bytes = (b_cols + kStep - 1) / kStep * 128, pitch = (b_cols + kGroup - 1) / kGroup * 4;
  uint32_t tm, tn;
  tile_of(blockIdx.x, mt, nt, tm, tn);
  const uint32_t m0 = tm * BM, n0 = tn * BN;

  // Loads: a base of the workgroup, moved from step to step, and offsets of the lane.  Rows and columns behind the last
  // are read as that; the last rows along the summed axis, beside which A has zeros, have offsets of their own.  16-byte
  // chunk c of a row of A lies at c ^ (row & 7), of a row of codes at c ^ mixed(row): what 32 lanes read is in all banks.
  const auto mixed = [](uint32_t row) { return BN == 256 ? row & 15 : row >> 1 & 7; };
  const uint8_t* ab = (const uint8_t*)a + (uint64_t)m0 * a_stride * 2 + from * 128ull;
  uint32_t ao[8], co[CI], co_last[CI];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t row = min((wave * 8 + i) * 8 + lane / 8, m - m0 - 1);
    ao[i] = row * (uint32_t)(a_stride * 2) + ((lane & 7) ^ (lane / 8)) * 16;
  }
  const uint32_t last_rows = b_rows - (steps_1 - 1) * 64;
#pragma unroll
  for (int i = 0; i < CI; ++i) {
    const uint32_t id = (wave * CI + i) * 64 + lane, row = id / (BN / 16), c = id % (BN / 16) ^ mixed(row);
    const uint32_t at = min(n0 + c * 16, b_bytes - 16);
    co[i] = row * b_bytes + at, co_last[i] = min(row, last_rows - 1) * b_bytes + at;
  }
  // the block of columns that the wavefront has, among four of which a load takes the scales
  const uint32_t block = min((n0 + wn * TN * 16) / kStep, pitch - 1);
  uint32_t left = steps, b_step = from % steps_1;
  const auto load = [&](uint32_t at, int i) {  // the i-th of LOADS; `at`: the stage's place in LDS
    if (i < 8) {
      to_lds16(ab, ao[i], base + at + (wave * 8 + i) * 1024);
    } else if (i < 8 + CI) {
      to_lds16(bd + (uint64_t)b_step * 64 * b_bytes, b_step + 1 == steps_1 ? co_last[i - 8] : co[i - 8],
               base + at + AB + (wave * CI + i - 8) * 1024);
    } else {
      to_lds4(bs + (uint64_t)(b_step / 2) * pitch + (block & ~3u), 0, base + at + S_AT + wave * 256);
      const uint32_t more = left > 1;  // behind the last step it is loaded again, into a place that is not read
      left -= more, ab += more * 128;
      b_step = more ? (b_step + 1 == steps_1 ? 0 : b_step + 1) : b_step;
    }
  };

  uint32_t ra[2], rc[TN];
#pragma unroll
  for (int h = 0; h < 2; ++h) ra[h] = (wm * 128 + r) * 128 + ((h * 4 + g) ^ (r & 7)) * 16;
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const uint32_t row = g * 8 + r / 2;
    rc[j] = base + AB + row * BN + (wn * TN + j ^ mixed(row)) * 16 + r % 2 * 8;
  }
  b8v x[2][TM], w[2][TN];
  typedef int i2v __attribute__((ext_vector_type(2)));
  i2v codes[TN];
  uint32_t scale;
  const auto read_x = [&](uint32_t at, int h, int i) { x[h][i] = *(const b8v*)(lds + at + ra[h] + i * 2048); };
  const auto read_codes = [&](uint32_t at, int h, int j) {
    codes[j] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
        (__attribute__((address_space(3))) i2v*)(uintptr_t)(rc[j] + at + h * 32 * BN));
  };
  const auto read_scale = [&](uint32_t at) {
    scale = *(const uint32_t*)(lds + at + S_AT + wave * 256) >> (block & 3) * 8 & 255;
  };
  const auto convert = [&](int h, int j) {
    w[h][j] = bf16_of_codes(make_uint2((uint32_t)codes[j].x, (uint32_t)codes[j].y), scale);
  };

  f4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      acc[i][j] = f4{0, 0, 0, 0};
      asm volatile("" : "+a"(acc[i][j]));
    }
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load(s * STAGE, i);
  wait_loads<(NS - 1) * LOADS>();
  block_barrier();
  read_scale(0);
#pragma unroll
  for (int j = 0; j < TN; ++j) read_codes(0, 0, j);
#pragma unroll
  for (int i = 0; i < TM; ++i) read_x(0, 0, i);
#pragma unroll
  for (int j = 0; j < TN; ++j) convert(0, j);
  settle();

  const auto multiply = [&](int h, auto beside) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        step16_in_place(w[h][j], x[h][i], acc[i][j]);
        beside(i * TN + j);
        __builtin_amdgcn_sched_barrier(0);
      }
  };
  // half h of the stage at `at` is read beside the other's instructions: its codes first, which are converted later
  const auto read_beside = [&](uint32_t at, int h, int t) {
    constexpr int C = M / 2 / TN;  // instructions between two conversions
    if (t < TN) read_codes(at, h, t);
    if (t >= TN && t < TN + 2 * TM && (t - TN) % 2 == 0) read_x(at, h, (t - TN) / 2);
    if (t >= M / 2 && (t - M / 2) % C == 0) convert(h, (t - M / 2) / C);
  };
  uint32_t at = 0;
  for (uint32_t s = 0; s < steps; ++s) {
    const uint32_t next = at == (NS - 1) * STAGE ? 0 : at + STAGE;
    multiply(0, [&](int t) { read_beside(at, 1, t); });
    // a stage is asked for in the second half of a step: one is on its way, that of the step before
    wait_loads<LOADS>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    block_barrier();
    read_scale(next);
    multiply(1, [&](int t) {
      read_beside(next, 0, t);
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
        if (i * M / LOADS == t) load(at, i);
    });
    at = next;
  }
  wait_loads<0>();  // nothing may arrive in this memory once it is used for something else
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  block_barrier();
  settle();

  // The result through a part of LDS of the wavefront's own, 16 rows at a time.
  const uint32_t row0 = m0 + wm * 128, col0 = n0 + wn * TN * 16;
  const auto finish = [&](auto* out) {
    using O = std::remove_reference_t<decltype(*out)>;
    constexpr int PITCH = TN * 16 * (int)sizeof(O) + 16, V = 16 / sizeof(O), ACROSS = TN * 16 / V;
    static_assert(4 * 16 * PITCH <= (int)sizeof(lds), "four parts");
    typedef O four __attribute__((ext_vector_type(4)));
    typedef O whole __attribute__((ext_vector_type(V)));
    typedef O piece __attribute__((ext_vector_type(V), aligned(sizeof(O))));
    uint8_t* mine = lds + wave * 16 * PITCH;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        asm volatile("" : "+a"(acc[i][j]));  // it stays where it is until here
        four v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (O)acc[i][j][e];
        *(four*)(mine + r * PITCH + (j * 16 + g * 4) * sizeof(O)) = v;
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int q = 0; q < 16 * ACROSS / 64; ++q) {
        const uint32_t id = q * 64 + lane, row = row0 + i * 16 + id / ACROSS, c = col0 + id % ACROSS * V;
        const whole v = *(const whole*)(mine + id / ACROSS * PITCH + id % ACROSS * 16);
        if (row >= m || c >= b_cols) continue;
        O* p = out + (uint64_t)row * b_cols + c;
        if (c + V <= b_cols)
          *(piece*)p = v;
        else
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (c + e < b_cols) p[e] = v[e];
      }
      __builtin_amdgcn_wave_barrier();
    }
  };
  if (part)
    finish(part + (uint64_t)blockIdx.y * m * b_cols);
  else
    finish(y);
}

// ---- host side -------------------------------------------------------------------------------------------------

uint64_t filled(uint64_t cols) { return nz_ceil_div(cols, kStep) * kStep; }

// rows are counted in 64 bits, the values of one row in 31
bool cols_ok(uint64_t cols) { return cols <= 0x40000000ull; }

// groups of 512 values in all rows, beyond any memory
int check_groups(uint64_t rows, uint64_t groups) {
  return nz_mul(rows, groups) <= 1ull << 33 ? NZ_OK : nz_fail(NZ_ERR_ARG, "too many rows");
}

Groups groups_of(uint64_t cols) {
  Groups g;
  g.count = (uint32_t)nz_ceil_div(cols, kGroup);
  uint32_t up = 0;  // 2^up is d at least
  while ((1ull << up) < g.count) ++up;
  g.shift = 26 + up;
  g.mul = (uint32_t)((1ull << g.shift) / g.count + 1);
  return g;
}

int check_fp8(const void* data, const void* scales) {
  if (!data || !scales) return nz_fail(NZ_ERR_ARG, "null data or scales");
  if (!aligned(data, 16) || !aligned(scales, 16))
    return nz_fail(NZ_ERR_ALIGN, "8-bit data and scales must be 16-byte aligned");
  return NZ_OK;
}

int check_block(int block_rows) {
  return block_rows == 1 || block_rows == 128 ? NZ_OK : nz_fail(NZ_ERR_ARG, "block_rows must be 1 or 128");
}
uint32_t shift_of(int block_rows) { return block_rows == 128 ? 7 : 0; }

int check_rows(uint64_t rows, uint64_t cols) {
  if (!cols_ok(cols)) return nz_fail(NZ_ERR_ARG, "rows must hold 1 to 2^30 values");
  return check_groups(rows, nz_ceil_div(cols, kGroup));
}

int launch_quantize(const void* x, int dtype, uint64_t rows, uint32_t cols, uint64_t stride, int block_rows,
                    void* data, void* scales, hipStream_t st) {
  const Groups g = groups_of(cols);
  const uint32_t groups = g.count, blocks = (cols + kStep - 1) / kStep;
  if (block_rows == 1) {
    nz_in_pieces(rows, groups * 64ull, [&](uint64_t first, uint64_t count) {
      const uint64_t waves = count * groups;
      by_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        nz_fp8_quantize_kernel<T><<<(uint32_t)nz_ceil_div(waves, 4), 256, 0, st>>>(
            (const T*)x + first * stride, stride, cols, (uint32_t)waves, g, (uint8_t*)data + first * filled(cols),
            (uint8_t*)scales + first * groups * 4);
      });
    });
  } else {
    nz_in_pieces(nz_ceil_div(rows, 128), blocks * 256ull, [&](uint64_t first, uint64_t count) {
      by_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        nz_fp8_quantize_blocks_kernel<T><<<(uint32_t)(count * blocks), 256, 0, st>>>(
            (const T*)x + first * 128 * stride, stride, rows - first * 128, cols, blocks, groups * 4,
            (uint8_t*)data + first * 128 * filled(cols), (uint8_t*)scales + first * groups * 4);
      });
    });
  }
  return nz_launched();
}

template <bool FINITE, class T>
int launch_values(const void* data, const void* scales, uint32_t shift, uint64_t rows, uint64_t cols, T* out,
                  hipStream_t st) {
  const Groups groups = groups_of(cols);
  nz_in_pieces(rows, groups.count * 64ull, [&](uint64_t first, uint64_t count) {
    const uint32_t waves = (uint32_t)(count * groups.count);
    nz_fp8_values_kernel<FINITE><<<(uint32_t)nz_ceil_div(waves, 4), 256, 0, st>>>(
        (const uint8_t*)data, (const uint8_t*)scales, shift, first, (uint32_t)cols, waves, groups, out);
  });
  return nz_launched();
}

// Figures of the tiles, fitted to times of 60 products of 17 to 8192 rows with weights of 256 to 16384 rows and columns,
// each in all tiles and up to 16 parts, and of 45 gradients of either kind.  The cut chosen by them takes 1.2 % more than
// the fastest one in the mean (of gradients of rows 2.3 %, of a weight 0.2 %).
// Products of 8-bit rows, 128 values a step.
constexpr Tile kTiles[] = {{256, 256, 256, 1.31f, 0.94f, 4.0f, true},
                           {128, 256, 256, 0.72f, 0.74f, 3.2f},
                           {128, 128, 512, 0.78f, 0.76f, 2.4f},
                           {64, 128, 256, 0.30f, 0.28f, 1.1f},
                           {64, 64, 256, 0.21f, 0.15f, 0.8f}};
// Products of 16-bit rows, 64 values a step.
constexpr Tile kTiles16[] = {{256, 128, 256, 0.86f, 0.94f, 0.9f}, {64, 64, 256, 0.40f, 0.44f, 0.5f}};
// The gradient of the rows where 128 rows of the weight share a scale.
constexpr Tile kTilesInput[] = {{256, 256, 256, 1.07f, 0.92f, 3.9f},
                                {256, 128, 256, 0.80f, 0.83f, 1.1f},
                                {64, 64, 256, 0.34f, 0.33f, 0.9f}};

// The product of 8-bit rows, cut along k by groups of four steps, two at least.
Cut cut_product8(uint64_t m, uint64_t n, uint64_t k) {
  return cut_product(kTiles, m, n, nz_ceil_div(k, kGroup), 4, 2, k % kGroup == 0);
}

// The products of 16-bit rows, in steps of 64.
Cut cut_product16(uint64_t m, uint64_t cols, uint64_t steps) {
  return cut_product(kTiles16, m, cols, steps, 1, 8);
}
Cut cut_input(uint64_t m, uint64_t cols, uint64_t steps, uint32_t shift) {
  return shift ? cut_product(kTilesInput, m, cols, steps, 1, 8) : cut_product16(m, cols, steps);
}

template <class T>
void launch_tiles(const Cut& c, const void* xd, const void* xs, uint64_t m, const void* wd, const void* ws,
                  uint32_t shift, uint64_t n, uint32_t k, const T* bias, T* y, float* part, hipStream_t st) {
  const dim3 grid(c.mt * c.nt, c.parts);
#define NZ_TILES(WM, WN, TM, TN, NS, EU)                                                                           \
  nz_fp8_tiles_kernel<WM, WN, TM, TN, NS, EU, T><<<grid, 64 * WM * WN, 0, st>>>(                                   \
      (const uint8_t*)xd, (const uint8_t*)xs, (uint32_t)m, (const uint8_t*)wd, (const uint8_t*)ws, shift,          \
      (uint32_t)n, k, bias, y, c.mt, c.nt, c.part_length, part)
  const uint32_t cus = nz_compute_units();
  if (c.bm == 256)
    nz_fp8_wide_kernel<T><<<std::min(c.mt * c.nt, cus ? cus : 256), 256, 0, st>>>(
        (const uint8_t*)xd, (const uint8_t*)xs, (uint32_t)m, (const uint8_t*)wd, (const uint8_t*)ws, shift, (uint32_t)n,
        k, bias, y, c.mt, c.nt);
  else if (c.bn == 256)
    NZ_TILES(2, 4, 4, 4, 3, 2);
  else if (c.bm == 128)
    NZ_TILES(2, 2, 4, 4, 2, 2);
  else if (c.bn == 128)
    NZ_TILES(2, 2, 2, 4, 3, 2);
  else
    NZ_TILES(2, 2, 2, 2, 4, 2);
#undef NZ_TILES
}

// The operands of a product of 16-bit rows.
struct Rows16 {
  const void* data;
  uint64_t stride, width, plane;  // elements
  uint32_t planes;
};
struct Held8 {
  const void *data, *scales;
  uint32_t shift;
  uint64_t rows, cols;
};

template <Product P, bool ADD = false>
int launch_tiles16(const Cut& c, const Rows16& a, uint64_t m, const Held8& b, uint64_t steps_1, uint64_t cols,
                   const void* bias, void* y, int dtype, void* part, hipStream_t st) {
  const dim3 grid(c.mt * c.nt, c.parts);
  float* p = c.parts > 1 ? (float*)part : nullptr;
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if constexpr (P == kForward && !std::is_same<T, float>::value) {
      return;  // results of 16 bits come from the scaled instruction
    } else {
#define NZ_TILES16(WM, WN, TM, TN)                                                                                  \
  nz_fp8_tiles16_kernel<WM, WN, TM, TN, P, ADD, T><<<grid, 64 * WM * WN, 0, st>>>(                                  \
      (const nz_bf16*)a.data, a.stride, (uint32_t)a.width, a.plane, (uint32_t)m, (const uint8_t*)b.data,            \
      (const uint8_t*)b.scales, b.shift, (uint32_t)b.rows, (uint32_t)b.cols, (uint32_t)steps_1, a.planes,           \
      (uint32_t)cols, (const T*)bias, (T*)y, c.mt, c.nt, c.part_length, p)
#define NZ_INPUT(TN)                                                                                                \
  nz_fp8_input_kernel<TN, T><<<grid, 256, 0, st>>>((const nz_bf16*)a.data, a.stride, (uint32_t)m,                   \
                                                   (const uint8_t*)b.data, (const uint8_t*)b.scales,                \
                                                   (uint32_t)b.rows, (uint32_t)b.cols, (uint32_t)steps_1, a.planes, \
                                                   (T*)y, c.mt, c.nt, c.part_length, p)
      if constexpr (P == kInput) {
        if (b.shift && c.bm == 256) {
          if (c.bn == 256)
            NZ_INPUT(8);
          else
            NZ_INPUT(4);
          return;
        }
      }
      if (c.bm == 256)
        NZ_TILES16(4, 2, 4, 4);
      else
        NZ_TILES16(2, 2, 2, 2);
#undef NZ_TILES16
#undef NZ_INPUT
    }
  });
  if (p) launch_join<ADD>(p, c, m, cols, bias, y, dtype, st);
  return nz_launched();
}

// Rows that go to the kernel for few (one tile of the instruction), and those that are brought to 8 bits inside it.
// The others go to tiles where the weight is large, for those read it in longer runs and their further launches count
// less.  us a call in a captured graph, weights from memory, rows as they are, the kernel for few against tiles (of 17
// rows): 8x4096x4096 9.9, 12.6; 4x4096x4096 8.1, 12.6; 16x4096x4096 (rows brought to 8 bits before) 9.7, 12.7;
// 1x4096x14336 15.2, 19.1; 8x14336x4096 18.5, 17.2; 8x50257x4096 51 (rows in 8 bits, two wavefronts for each), 43.3.  Of
// small k and many rows the few lose up to 2.5 us: 16x4096x1024 6.7, 6.0; 16x14336x2048 12.7, 10.2.
bool few_inside(uint64_t m, uint64_t n, uint64_t k, int dtype) {
  const uint64_t groups = m * nz_ceil_div(k, kGroup);
  return m <= 16 && groups <= 64 && (groups <= 32 || n * k <= 1ull << 26 || dtype == NZ_DTYPE_F32);
}
bool few_rows(uint64_t m, uint64_t n, uint64_t k, int dtype) {
  return few_inside(m, n, k, dtype) || (m <= 16 && (n * k <= 1ull << 25 || dtype == NZ_DTYPE_F32));
}

template <int N, class T>
void launch_few(const void* x, uint64_t stride, const void* xs, uint64_t m, const void* wd, const void* ws,
                uint32_t shift, uint64_t n, uint32_t k, const T* bias, T* y, hipStream_t st) {
  const uint32_t groups = (k + kGroup - 1) / kGroup;
  // As many wavefronts for a row as it has groups for, while there are not enough rows of the weight to fill the card;
  // beyond that two for many rows of x, else four.  us with 1, 2, 4, 8 of them, launches in a row, weights from memory:
  // 1x4096x14336 54, 30, 18, 13.4; 7x5003x3001 16.6, 11.3, 8.8, 10.6; 1x14336x4096 18.9, 14.0, 14.4, 14.2; 8x14336x4096
  // 22.5, 17.6, 18.7, 23.7; 4x128256x1024 23.0, 22.8, 27.3, 38.6.
  uint32_t kw = groups >= 8 ? 8 : groups >= 4 ? 4 : groups >= 2 ? 2 : 1;
  const uint64_t t = nz_ceil_div(n, 16);
  const uint32_t cus = nz_compute_units();
  if (t > 2 * (cus ? cus : 256)) kw = kw < 4 ? kw : m >= 4 ? 2 : 4;
  const uint32_t lds = N ? (uint32_t)m * groups * kHeld : 0;
  nz_fp8_few_kernel<N, T><<<(uint32_t)nz_ceil_div(t, 8 / kw), 512, lds > 8192 ? lds : 8192, st>>>(
      x, stride, (const uint8_t*)xs, (uint32_t)m, (const uint8_t*)wd, (const uint8_t*)ws, shift, (uint32_t)n, k, bias,
      y, kw);
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
  r.xs = align256(nz_mul(m, nz_fp8_row_bytes(k)));
  r.values = align256(r.xs + nz_mul(m, nz_fp8_scale_bytes(k)));
  r.bytes = r.values;
  if (few_rows(m, n, k, dtype)) return r;
  if (dtype == NZ_DTYPE_F32) {
    r.cut = cut_product16(m, n, filled(k) / 64);
    r.values = 0;  // the rows' 8 bits are not kept
    r.parts = align256(nz_mul(m, filled(k) * 2));
  } else {
    r.cut = cut_product8(m, n, k);
    r.parts = r.values;
  }
  r.bytes = r.parts + r.cut.part_bytes(m, n);
  return r;
}

// A float32 result of rows whose values lie in the workspace.
int launch_wide(uint64_t m, const Held8& w, const void* bias, void* y, const Room& room, uint8_t* workspace,
                hipStream_t st) {
  const uint64_t pad = filled(w.cols);
  return launch_tiles16<kForward>(room.cut, Rows16{workspace + room.values, pad, pad, 0, 1}, m, w, pad / 64, w.rows,
                                  bias, y, NZ_DTYPE_F32, workspace + room.parts, st);
}

int launch_product(const void* xd, const void* xs, uint64_t m, const Held8& w, const void* bias, void* y, int dtype,
                   const Room& room, uint8_t* workspace, hipStream_t st) {
  const uint64_t n = w.rows;
  const uint32_t k = (uint32_t)w.cols;
  if (few_rows(m, n, k, dtype)) {
    by_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      launch_few<0>(xd, 0, xs, m, w.data, w.scales, w.shift, n, k, (const T*)bias, (T*)y, st);
    });
    return nz_launched();
  }
  if (dtype == NZ_DTYPE_F32) {
    if (int rc = launch_values<true>(xd, xs, 0, m, filled(k), (nz_bf16*)(workspace + room.values), st)) return rc;
    return launch_wide(m, w, bias, y, room, workspace, st);
  }
  const Cut& c = room.cut;
  float* part = c.parts > 1 ? (float*)(workspace + room.parts) : nullptr;
  if (dtype == NZ_DTYPE_BF16)
    launch_tiles(c, xd, xs, m, w.data, w.scales, w.shift, n, k, (const nz_bf16*)bias, (nz_bf16*)y, part, st);
  else
    launch_tiles(c, xd, xs, m, w.data, w.scales, w.shift, n, k, (const nz_f16*)bias, (nz_f16*)y, part, st);
  if (part) launch_join(part, c, m, n, bias, y, dtype, st);
  return nz_launched();
}

// What the products ask of the counts: an offset inside a tile has 32 bits.
int check_product(uint64_t m, uint64_t n, uint64_t k, int block_rows, const void* wd, const void* ws) {
  if (int rc = check_block(block_rows)) return rc;
  if (k == 0 || k > 1ull << 22 || n > 1ull << 21)
    return nz_fail(NZ_ERR_ARG, "a weight must have 1 to 2^22 columns and up to 2^21 rows");
  if (m > 1ull << 24) return nz_fail(NZ_ERR_ARG, "too many rows");
  return check_fp8(wd, ws);
}

// A gradient's rows as bf16: as they are, or as planes at `room`.
Rows16 launch_planes(const void* g, int dtype, uint64_t m, uint64_t n, uint64_t stride, const Planes& p, void* room,
                     hipStream_t st) {
  if (!p.bytes) return Rows16{g, stride, n, 0, 1};
  const uint64_t pitch = p.padded * p.count;
#define NZ_PLANES(P, T)                                                                                           \
  nz_in_pieces(m, p.padded / 8, [&](uint64_t first, uint64_t count) {                                             \
    nz_planes_kernel<P, T><<<(uint32_t)nz_ceil_div(count * (p.padded / 8), 256), 256, 0, st>>>(                   \
        (const T*)g + first * stride, stride, count, (uint32_t)n, (uint32_t)p.padded, (nz_bf16*)room + first * pitch); \
  })
  if (dtype == NZ_DTYPE_BF16)
    NZ_PLANES(1, nz_bf16);
  else if (dtype == NZ_DTYPE_F16)
    NZ_PLANES(2, nz_f16);
  else
    NZ_PLANES(3, float);
#undef NZ_PLANES
  return Rows16{room, pitch, p.padded, p.padded, p.count};
}

// The gradient's rows where they run along the summed axis: their ends need no zeros.
Planes planes_of_rows(const void* g, int dtype, uint64_t m, uint64_t n, uint64_t stride) {
  Planes p = planes_of(g, dtype, m, n, stride);
  if (dtype == NZ_DTYPE_BF16 && n % 8 == 0 && stride % 8 == 0 && stride <= 1ull << 22 && aligned(g, 16)) p.bytes = 0;
  return p;
}

int check_kind(int kind) {
  return kind >= NZ_ACTIVATION_GELU && kind <= NZ_ACTIVATION_SILU ? NZ_OK
                                                                  : nz_fail(NZ_ERR_ARG, "unknown activation function");
}

template <class F>
void by_kind(int kind, bool gated, F f) {
  using Gelu = std::integral_constant<int, NZ_ACTIVATION_GELU>;
  using GeluTanh = std::integral_constant<int, NZ_ACTIVATION_GELU_TANH>;
  using Silu = std::integral_constant<int, NZ_ACTIVATION_SILU>;
  const auto with = [&](auto k) {
    if (gated)
      f(k, std::true_type());
    else
      f(k, std::false_type());
  };
  if (kind == NZ_ACTIVATION_GELU)
    with(Gelu());
  else if (kind == NZ_ACTIVATION_GELU_TANH)
    with(GeluTanh());
  else
    with(Silu());
}

}  // namespace

extern "C" {

uint64_t nz_fp8_row_bytes(uint64_t cols) { return filled(cols); }

uint64_t nz_fp8_scale_bytes(uint64_t cols) { return nz_ceil_div(cols, kGroup) * 4; }

int nz_fp8_quantize(const void* dev_x, int dtype, uint64_t rows, uint64_t cols, uint64_t stride, int block_rows,
                    void* dev_data, void* dev_scales, void* stream) {
  if (int rc = check_block(block_rows)) return rc;
  if (int rc = check_dtype(dtype, dev_x, nullptr, nullptr)) return rc;
  if (rows == 0 || cols == 0) return NZ_OK;
  if (int rc = check_rows(rows, cols)) return rc;
  if (!dev_x) return nz_fail(NZ_ERR_ARG, "null input");
  if (int rc = check_fp8(dev_data, dev_scales)) return rc;
  return launch_quantize(dev_x, dtype, rows, (uint32_t)cols, stride, block_rows, dev_data, dev_scales,
                         (hipStream_t)stream);
}

int nz_fp8_dequantize(const void* dev_data, const void* dev_scales, uint64_t rows, uint64_t cols, int block_rows,
                      void* dev_out, int dtype, void* stream) {
  if (int rc = check_block(block_rows)) return rc;
  if (int rc = check_dtype(dtype, dev_out, nullptr, nullptr)) return rc;
  if (rows == 0 || cols == 0) return NZ_OK;
  if (int rc = check_rows(rows, cols)) return rc;
  if (!dev_out) return nz_fail(NZ_ERR_ARG, "null output");
  if (int rc = check_fp8(dev_data, dev_scales)) return rc;
  int rc = NZ_OK;
  by_dtype(dtype, [&](auto t) {
    rc = launch_values<false>(dev_data, dev_scales, shift_of(block_rows), rows, cols, (decltype(t)*)dev_out,
                              (hipStream_t)stream);
  });
  return rc;
}

uint64_t nz_fp8_linear_workspace_bytes(uint64_t m, uint64_t n, uint64_t k, int dtype) {
  if (m == 0 || n == 0 || k == 0) return 0;
  return product_room(m, n, k, dtype).bytes;
}

int nz_fp8_linear(const void* dev_x, int dtype, uint64_t m, uint64_t k, uint64_t stride, const void* dev_w_data,
                  const void* dev_w_scales, uint64_t n, int block_rows, const void* dev_bias, void* dev_y,
                  void* dev_workspace, uint64_t workspace_bytes, void* stream) {
  if (int rc = check_dtype(dtype, dev_x, dev_bias, dev_y)) return rc;
  if (m == 0 || n == 0) return NZ_OK;
  if (int rc = check_product(m, n, k, block_rows, dev_w_data, dev_w_scales)) return rc;
  if (!dev_x || !dev_y) return nz_fail(NZ_ERR_ARG, "null rows or output");
  const Room room = product_room(m, n, k, dtype);
  if (int rc = check_cut(room.cut)) return rc;
  if (int rc = check_workspace(dev_workspace, workspace_bytes, room.bytes)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  const Held8 w = {dev_w_data, dev_w_scales, shift_of(block_rows), n, k};
  if (few_inside(m, n, k, dtype)) {
    by_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      const auto launch = [&](auto held) {
        launch_few<decltype(held)::value>(dev_x, stride, nullptr, m, w.data, w.scales, w.shift, n, (uint32_t)k,
                                          (const T*)dev_bias, (T*)dev_y, st);
      };
      const uint64_t groups = m * nz_ceil_div(k, kGroup);
      if (groups <= 8)
        launch(std::integral_constant<int, 1>());
      else if (groups <= 32)
        launch(std::integral_constant<int, 4>());
      else
        launch(std::integral_constant<int, 8>());
    });
    return nz_launched();
  }
  uint8_t* base = (uint8_t*)dev_workspace;
  if (dtype == NZ_DTYPE_F32 && !few_rows(m, n, k, dtype)) {
    const Groups groups = groups_of(k);
    nz_in_pieces(m, groups.count * 64ull, [&](uint64_t first, uint64_t count) {
      const uint32_t waves = (uint32_t)(count * groups.count);
      nz_fp8_rounded_kernel<<<(uint32_t)nz_ceil_div(waves, 4), 256, 0, st>>>(
          (const float*)dev_x + first * stride, stride, (uint32_t)k, waves, groups,
          (nz_bf16*)(base + room.values) + first * filled(k));
    });
    return launch_wide(m, w, dev_bias, dev_y, room, base, st);
  }
  if (int rc = launch_quantize(dev_x, dtype, m, (uint32_t)k, stride, 1, base + room.xd, base + room.xs, st)) return rc;
  return launch_product(base + room.xd, base + room.xs, m, w, dev_bias, dev_y, dtype, room, base, st);
}

int nz_fp8_linear_rows8(const void* dev_x_data, const void* dev_x_scales, uint64_t m, uint64_t k,
                        const void* dev_w_data, const void* dev_w_scales, uint64_t n, int block_rows,
                        const void* dev_bias, void* dev_y, int dtype, void* dev_workspace, uint64_t workspace_bytes,
                        void* stream) {
  if (int rc = check_dtype(dtype, dev_bias, dev_y, nullptr)) return rc;
  if (m == 0 || n == 0) return NZ_OK;
  if (int rc = check_product(m, n, k, block_rows, dev_w_data, dev_w_scales)) return rc;
  if (int rc = check_fp8(dev_x_data, dev_x_scales)) return rc;
  if (!dev_y) return nz_fail(NZ_ERR_ARG, "null output");
  const Room room = product_room(m, n, k, dtype);
  if (int rc = check_cut(room.cut)) return rc;
  if (int rc = check_workspace(dev_workspace, workspace_bytes, room.bytes)) return rc;
  return launch_product(dev_x_data, dev_x_scales, m, Held8{dev_w_data, dev_w_scales, shift_of(block_rows), n, k},
                        dev_bias, dev_y, dtype, room, (uint8_t*)dev_workspace, (hipStream_t)stream);
}

uint64_t nz_fp8_linear_grad_workspace_bytes(const void* dev_g, int dtype, uint64_t m, uint64_t n, uint64_t stride,
                                            uint64_t k, int block_rows) {
  if (m == 0 || n == 0 || k == 0) return 0;
  const Planes p = planes_of(dev_g, dtype, m, n, stride);
  return p.bytes + cut_input(m, k, p.padded / 64 * p.count, shift_of(block_rows)).part_bytes(m, k);
}

int nz_fp8_linear_grad(const void* dev_g, int dtype, uint64_t m, uint64_t n, uint64_t stride, const void* dev_w_data,
                       const void* dev_w_scales, uint64_t k, int block_rows, void* dev_dx, void* dev_workspace,
                       uint64_t workspace_bytes, void* stream) {
  if (int rc = check_dtype(dtype, dev_g, dev_dx, nullptr)) return rc;
  if (m == 0 || k == 0) return NZ_OK;
  if (!dev_dx || !dev_g) return nz_fail(NZ_ERR_ARG, "null gradient or output");
  if (n == 0) return nz_fail(NZ_ERR_ARG, "a weight without rows has no gradient to pass on");
  if (int rc = check_product(m, n, k, block_rows, dev_w_data, dev_w_scales)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  const Planes p = planes_of(dev_g, dtype, m, n, stride);
  const uint64_t steps = p.padded / 64;
  const Cut cut = cut_input(m, k, steps * p.count, shift_of(block_rows));
  if (int rc = check_cut(cut)) return rc;
  if (int rc = check_workspace(dev_workspace, workspace_bytes, p.bytes + cut.part_bytes(m, k))) return rc;
  const Rows16 a = launch_planes(dev_g, dtype, m, n, stride, p, dev_workspace, st);
  return launch_tiles16<kInput>(cut, a, m, Held8{dev_w_data, dev_w_scales, shift_of(block_rows), n, k}, steps, k,
                                nullptr, dev_dx, dtype, (uint8_t*)dev_workspace + p.bytes, st);
}

uint64_t nz_fp8_weight_grad_workspace_bytes(const void* dev_g, int dtype, uint64_t m, uint64_t n, uint64_t stride,
                                            uint64_t k) {
  if (m == 0 || n == 0 || k == 0) return 0;
  const Planes p = planes_of_rows(dev_g, dtype, m, n, stride);
  return p.bytes + cut_product16(n, k, nz_ceil_div(m, 64) * p.count).part_bytes(n, k);
}

int nz_fp8_weight_grad(const void* dev_g, int dtype, uint64_t m, uint64_t n, uint64_t stride, const void* dev_x_data,
                       const void* dev_x_scales, uint64_t k, int block_rows, uint32_t flags, void* dev_out,
                       void* dev_workspace, uint64_t workspace_bytes, void* stream) {
  if (flags & ~NZ_GRAD_ACCUMULATE) return nz_fail(NZ_ERR_ARG, "unknown flags");
  if (int rc = check_dtype(dtype, dev_g, dev_out, nullptr)) return rc;
  if (n == 0 || k == 0) return NZ_OK;
  if (m == 0) return nz_fail(NZ_ERR_ARG, "a gradient without rows is zero");
  if (!dev_out || !dev_g) return nz_fail(NZ_ERR_ARG, "null gradient or output");
  if (int rc = check_product(m, n, k, block_rows, dev_x_data, dev_x_scales)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  const Planes p = planes_of_rows(dev_g, dtype, m, n, stride);
  const uint64_t steps = nz_ceil_div(m, 64);
  const Cut cut = cut_product16(n, k, steps * p.count);
  if (int rc = check_cut(cut)) return rc;
  if (int rc = check_workspace(dev_workspace, workspace_bytes, p.bytes + cut.part_bytes(n, k))) return rc;
  const Rows16 a = launch_planes(dev_g, dtype, m, n, stride, p, dev_workspace, st);
  const Held8 x = {dev_x_data, dev_x_scales, shift_of(block_rows), m, k};
  void* part = (uint8_t*)dev_workspace + p.bytes;
  if (flags & NZ_GRAD_ACCUMULATE)
    return launch_tiles16<kWeight, true>(cut, a, n, x, steps, k, nullptr, dev_out, dtype, part, st);
  return launch_tiles16<kWeight>(cut, a, n, x, steps, k, nullptr, dev_out, dtype, part, st);
}

int nz_fp8_activation(int kind, const void* dev_x, int dtype, uint64_t rows, uint64_t cols, uint64_t stride,
                      const void* dev_up, uint64_t up_stride, void* dev_y, void* dev_x_data, void* dev_x_scales,
                      void* dev_up_data, void* dev_up_scales, void* stream) {
  if (int rc = check_kind(kind)) return rc;
  if (int rc = check_dtype(dtype, dev_x, dev_up, dev_y)) return rc;
  if (rows == 0 || cols == 0) return NZ_OK;
  if (int rc = check_rows(rows, cols)) return rc;
  if (!dev_x || !dev_y) return nz_fail(NZ_ERR_ARG, "null input or output");
  const bool keep = dev_x_data != nullptr;
  if (keep)
    if (int rc = check_fp8(dev_x_data, dev_x_scales)) return rc;
  if (keep && dev_up)
    if (int rc = check_fp8(dev_up_data, dev_up_scales)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  const Groups groups = groups_of(cols);
  nz_in_pieces(rows, groups.count * 64ull, [&](uint64_t first, uint64_t count) {
    const uint32_t waves = (uint32_t)(count * groups.count);
    const uint64_t d = first * filled(cols), s = first * groups.count * 4;
    by_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      by_kind(kind, dev_up != nullptr, [&](auto k, auto gated) {
        nz_fp8_activation_kernel<decltype(k)::value, decltype(gated)::value, T>
            <<<(uint32_t)nz_ceil_div(waves, 4), 256, 0, st>>>(
                (const T*)dev_x + first * stride, stride, gated ? (const T*)dev_up + first * up_stride : nullptr,
                up_stride, (uint32_t)cols, waves, groups, (T*)dev_y + first * cols,
                keep ? (uint8_t*)dev_x_data + d : nullptr, (uint8_t*)dev_x_scales + s, (uint8_t*)dev_up_data + d,
                (uint8_t*)dev_up_scales + s);
      });
    });
  });
  return nz_launched();
}

int nz_fp8_activation_grad(int kind, const void* dev_g, int dtype, uint64_t rows, uint64_t cols, uint64_t stride,
                           const void* dev_x_data, const void* dev_x_scales, const void* dev_up_data,
                           const void* dev_up_scales, void* dev_dx, void* dev_dup, void* stream) {
  if (int rc = check_kind(kind)) return rc;
  if (int rc = check_dtype(dtype, dev_g, dev_dx, dev_dup)) return rc;
  if (rows == 0 || cols == 0) return NZ_OK;
  if (int rc = check_rows(rows, cols)) return rc;
  if (!dev_g || !dev_dx) return nz_fail(NZ_ERR_ARG, "null gradient or output");
  if (int rc = check_fp8(dev_x_data, dev_x_scales)) return rc;
  if (dev_up_data) {
    if (int rc = check_fp8(dev_up_data, dev_up_scales)) return rc;
    if (!dev_dup) return nz_fail(NZ_ERR_ARG, "null output");
  }
  const hipStream_t st = (hipStream_t)stream;
  const Groups groups = groups_of(cols);
  nz_in_pieces(rows, groups.count * 64ull, [&](uint64_t first, uint64_t count) {
    const uint32_t waves = (uint32_t)(count * groups.count);
    const uint64_t d = first * filled(cols), s = first * groups.count * 4;
    by_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      by_kind(kind, dev_up_data != nullptr, [&](auto k, auto gated) {
        nz_fp8_activation_grad_kernel<decltype(k)::value, decltype(gated)::value, T>
            <<<(uint32_t)nz_ceil_div(waves, 4), 256, 0, st>>>(
                (const T*)dev_g + first * stride, stride, (uint32_t)cols, waves, groups,
                (const uint8_t*)dev_x_data + d, (const uint8_t*)dev_x_scales + s,
                gated ? (const uint8_t*)dev_up_data + d : nullptr, gated ? (const uint8_t*)dev_up_scales + s : nullptr,
                (T*)dev_dx + first * cols, gated ? (T*)dev_dup + first * cols : nullptr);
      });
    });
  });
  return nz_launched();
}

}  // extern "C"
