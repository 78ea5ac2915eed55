// Weights in microscaled 4 bits: quantisation, values, row lookup, and the products with activation rows.
//
// The format is stated in include/neuzip_hip.h.  A row's codes lie in order and are filled up to 128 values, so
// that a step of the matrix instruction (128 values of a row) never ends inside one; its block scales lie in
// groups of 16 (512 values) with the four bytes that a lane needs in four successive steps next to each other.
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

template <class T>
__device__ inline void load8(const T* p, float (&v)[8]) {
  typedef T pack __attribute__((ext_vector_type(8)));
  const pack a = *reinterpret_cast<const pack*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
}

// the first `n` of 8 values, zeros behind them
template <class T>
__device__ inline void load8_part(const T* p, long long n, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? (float)p[i] : 0.0f;
}

template <class T>
__device__ inline void store8(T* p, const float (&v)[8]) {
  typedef T pack __attribute__((ext_vector_type(8)));
  pack a;
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = (T)v[i];
  *reinterpret_cast<pack*>(p) = a;
}

template <class T>
__device__ inline void store8_part(T* p, long long n, const float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = (T)v[i];
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

// place of block b (of a row) among the row's scale bytes
__device__ inline uint32_t scale_at(uint32_t b) { return (b & ~15u) + 4 * (b & 3) + ((b >> 2) & 3); }

// ---- quantisation and values -----------------------------------------------------------------------------------
//
// One wavefront per 512 values of a row: 8 values a lane, four lanes a block, so that loads and stores of a
// wavefront are consecutive and the block's maximum takes two exchanges inside a quad.

template <int BITS, class T>
__global__ __launch_bounds__(256) void nz_mx_quantize_kernel(const T* x, uint64_t stride, uint32_t cols,
                                                             uint64_t waves, uint32_t groups, uint32_t wide,
                                                             uint8_t* data, uint8_t* scales) {
  const uint64_t wave = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64;
  if (wave >= waves) return;
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t row = wave / groups;
  const uint32_t group = (uint32_t)(wave - row * groups);
  const uint32_t at = group * kGroup + lane * 8;
  const T* p = x + row * stride + at;
  float v[8];
  if (wide && at + 8 <= cols)
    load8(p, v);
  else
    load8_part(p, (long long)cols - at, v);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xB1, 0xF, 0xF, true));  // lane ^ 1
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4E, 0xF, 0xF, true));  // lane ^ 2
  const uint32_t s = scale_byte<BITS>(top);
  if (s == 255)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
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
                                                           uint32_t groups, uint32_t wide, float scale, T* out,
                                                           uint32_t* status) {
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
  T* q = out + to * (uint64_t)cols + at;
  if (wide && at + 8 <= cols)
    store8(q, v);
  else
    store8_part(q, (long long)cols - at, v);
}

// ---- product ---------------------------------------------------------------------------------------------------
//
// The matrix instruction takes 16 rows of each side and 128 values of a row.  A lane (r = lane % 16, g = lane / 16)
// holds, of row r: 4-bit values 32 g .. 32 g + 31; 8-bit values 16 g .. 16 g + 15 and 64 + 16 g .. 64 + 16 g + 15;
// and, on both sides, the scale of block g.  Of the result it holds weight rows 4 g .. 4 g + 3 against activation
// row r.

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

// 16 weight rows against 16 MT activation rows; the wavefronts of a workgroup share the values of a row.
template <int MT, class T>
__global__ __launch_bounds__(512) void nz_mx_product_kernel(const uint8_t* xd, const uint8_t* xs, uint64_t m,
                                                            const uint8_t* wd, const uint8_t* ws, uint64_t n,
                                                            uint32_t k, const T* bias, T* y) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64, r = lane & 15, g = lane / 16;
  const uint32_t steps = (k + kStep - 1) / kStep, groups = (k + kGroup - 1) / kGroup;
  const uint64_t n0 = (uint64_t)blockIdx.x * 16, m0 = (uint64_t)blockIdx.y * (16 * MT);
  const uint64_t wrow = min(n0 + r, n - 1);
  const uint8_t* wp = wd + wrow * (steps * 64ull) + g * 16;
  const uint8_t* wsp = ws + wrow * (groups * 16ull) + g * 4;
  const uint8_t* xp[MT];
  const uint8_t* xsp[MT];
  f4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const uint64_t xrow = min(m0 + t * 16 + r, m - 1);
    xp[t] = xd + xrow * (steps * 128ull) + g * 16;
    xsp[t] = xs + xrow * (groups * 16ull) + g * 4;
    acc[t] = f4{0, 0, 0, 0};
  }
  for (uint32_t group = wave; group < groups; group += 8) {
    const uint32_t sw = *reinterpret_cast<const uint32_t*>(wsp + group * 16);
    uint32_t sx[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) sx[t] = *reinterpret_cast<const uint32_t*>(xsp[t] + group * 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t s = group * 4 + j;
      if (s < steps) {
        const i4v w = *reinterpret_cast<const i4v*>(wp + s * 64ull);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const i4v x0 = *reinterpret_cast<const i4v*>(xp[t] + s * 128ull);
          const i4v x1 = *reinterpret_cast<const i4v*>(xp[t] + s * 128ull + 64);
          acc[t] = step(w, x0, x1, acc[t], sw, sx[t], j);
        }
      }
    }
  }
  __shared__ float part[8][MT * 256];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) part[wave][t * 256 + r * 16 + g * 4 + j] = acc[t][j];
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < MT * 256; i += 512) {
    float sum = part[0][i];
#pragma unroll
    for (int w = 1; w < 8; ++w) sum += part[w][i];
    const uint64_t row = m0 + i / 16, col = n0 + i % 16;
    if (row < m && col < n) {
      if (bias) sum += (float)bias[col];
      y[row * n + col] = (T)sum;
    }
  }
}

// ---- gradient of the rows --------------------------------------------------------------------------------------

template <class T>
__global__ __launch_bounds__(256) void nz_mx_grad_kernel(const T* g, uint64_t stride, uint64_t m, uint64_t n,
                                                         const uint8_t* wd, const uint8_t* ws, uint32_t k, T* dx) {
  __shared__ float sg[32][65], sw[32][64];
  const uint32_t steps = (k + kStep - 1) / kStep, groups = (k + kGroup - 1) / kGroup;
  const uint32_t k0 = blockIdx.x * 64;
  const uint64_t m0 = (uint64_t)blockIdx.y * 64;
  const uint32_t tx = threadIdx.x & 15, ty = threadIdx.x / 16;
  float acc[4][4] = {};
  for (uint64_t n0 = 0; n0 < n; n0 += 32) {
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 64 * 32; i += 256) {
      const uint64_t row = m0 + i / 32, col = n0 + i % 32;
      sg[i % 32][i / 32] = row < m && col < n ? (float)g[row * stride + col] : 0.0f;
    }
    {
      const uint32_t i = threadIdx.x;  // 32 rows of 64 values, 8 a lane
      const uint64_t row = n0 + i / 8;
      const uint32_t at = k0 + (i % 8) * 8;
      float v[8] = {};
      if (row < n && at < steps * kStep)
        values4(*reinterpret_cast<const uint32_t*>(wd + row * (steps * 64ull) + at / 2),
                down_factor(ws[row * (groups * 16ull) + scale_at(at / 32)]), v);
#pragma unroll
      for (int j = 0; j < 8; ++j) sw[i / 8][(i % 8) * 8 + j] = v[j];
    }
    __syncthreads();
    for (int j = 0; j < 32; ++j) {
#pragma unroll
      for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) acc[a][b] += sg[j][ty * 4 + a] * sw[j][tx * 4 + b];
    }
  }
  for (int a = 0; a < 4; ++a)
    for (int b = 0; b < 4; ++b) {
      const uint64_t row = m0 + ty * 4 + a;
      const uint32_t col = k0 + tx * 4 + b;
      if (row < m && col < k) dx[row * k + col] = (T)acc[a][b];
    }
}

// ---- host side -------------------------------------------------------------------------------------------------

uint64_t filled(uint64_t cols) { return nz_ceil_div(cols, kStep) * kStep; }

// rows are counted in 64 bits, the values of one row in 31
bool cols_ok(uint64_t cols) { return cols <= 0x40000000ull; }

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

int check_grid(uint64_t blocks) {
  return blocks <= 0x7FFFFFFFull ? NZ_OK : nz_fail(NZ_ERR_ARG, "too many rows for one launch");
}

// rows of `stride` elements that all start 16-byte aligned
bool wide_rows(const void* p, uint64_t stride, uint32_t size) { return aligned(p, 16) && stride * size % 16 == 0; }

template <class F>
void by_dtype(int dtype, F f) {
  if (dtype == NZ_DTYPE_BF16)
    f(nz_bf16());
  else if (dtype == NZ_DTYPE_F16)
    f(nz_f16());
  else
    f(float());
}

void launch_quantize(const void* x, int dtype, uint64_t rows, uint32_t cols, uint64_t stride, int bits, void* data,
                     void* scales, hipStream_t st) {
  const uint32_t groups = (cols + kGroup - 1) / kGroup;
  const uint64_t waves = rows * groups;
  const dim3 grid((uint32_t)nz_ceil_div(waves, 4));
  const uint32_t wide = wide_rows(x, stride, nz_dtype_bytes(dtype));
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (bits == 4)
      nz_mx_quantize_kernel<4, T><<<grid, 256, 0, st>>>((const T*)x, stride, cols, waves, groups, wide,
                                                        (uint8_t*)data, (uint8_t*)scales);
    else
      nz_mx_quantize_kernel<8, T><<<grid, 256, 0, st>>>((const T*)x, stride, cols, waves, groups, wide,
                                                        (uint8_t*)data, (uint8_t*)scales);
  });
}

int launch_values(const void* data, const void* scales, uint64_t rows, uint64_t cols, int bits, const void* index,
                  uint64_t count, float scale, void* out, int dtype, void* status, hipStream_t st) {
  const uint32_t groups = (uint32_t)nz_ceil_div(cols, kGroup);
  const uint64_t waves = nz_mul(count, groups);
  if (int rc = check_grid(nz_ceil_div(waves, 4))) return rc;
  const dim3 grid((uint32_t)nz_ceil_div(waves, 4));
  const uint32_t wide = wide_rows(out, cols, nz_dtype_bytes(dtype));
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (bits == 4)
      nz_mx_values_kernel<4, T><<<grid, 256, 0, st>>>((const uint8_t*)data, (const uint8_t*)scales, rows,
                                                      (uint32_t)cols, (const long long*)index, waves, groups, wide,
                                                      scale, (T*)out, (uint32_t*)status);
    else
      nz_mx_values_kernel<8, T><<<grid, 256, 0, st>>>((const uint8_t*)data, (const uint8_t*)scales, rows,
                                                      (uint32_t)cols, (const long long*)index, waves, groups, wide,
                                                      scale, (T*)out, (uint32_t*)status);
  });
  return nz_launched();
}

int launch_product(const void* xd, const void* xs, uint64_t m, const void* wd, const void* ws, uint64_t n, uint32_t k,
                   const void* bias, void* y, int dtype, hipStream_t st) {
  const uint64_t mt = m <= 16 ? 1 : m <= 32 ? 2 : 4;
  const dim3 grid((uint32_t)nz_ceil_div(n, 16), (uint32_t)nz_ceil_div(m, 16 * mt));
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
#define NZ_MX_PRODUCT(MT)                                                                                        \
  nz_mx_product_kernel<MT, T><<<grid, 512, 0, st>>>((const uint8_t*)xd, (const uint8_t*)xs, m, (const uint8_t*)wd, \
                                                    (const uint8_t*)ws, n, k, (const T*)bias, (T*)y)
    if (mt == 1)
      NZ_MX_PRODUCT(1);
    else if (mt == 2)
      NZ_MX_PRODUCT(2);
    else
      NZ_MX_PRODUCT(4);
#undef NZ_MX_PRODUCT
  });
  return nz_launched();
}

// what both forms of the product, and its gradient, ask of the weight and the counts
int check_product(uint64_t m, uint64_t n, uint64_t k, const void* wd, const void* ws) {
  if (k == 0 || !cols_ok(k)) return nz_fail(NZ_ERR_ARG, "rows must hold 1 to 2^30 values");
  if (m > 65535ull * 64 || n > 0x7FFFFFFFull) return nz_fail(NZ_ERR_ARG, "too many rows for one launch");
  return check_mx(wd, ws);
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
  if (int rc = check_grid(nz_ceil_div(nz_mul(rows, nz_ceil_div(cols, kGroup)), 4))) return rc;
  launch_quantize(dev_x, dtype, rows, (uint32_t)cols, stride, bits, dev_data, dev_scales, (hipStream_t)stream);
  return nz_launched();
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

uint64_t nz_mx_linear_workspace_bytes(uint64_t m, uint64_t n, uint64_t k) {
  (void)n;
  return (m * nz_mx_row_bytes(k, 8) + 255) / 256 * 256 + m * nz_mx_scale_bytes(k);
}

int nz_mx_linear(const void* dev_x, int dtype, uint64_t m, uint64_t k, uint64_t stride, const void* dev_w_data,
                 const void* dev_w_scales, uint64_t n, const void* dev_bias, void* dev_y, void* dev_workspace,
                 uint64_t workspace_bytes, void* stream) {
  if (int rc = check_dtype(dtype, dev_x, dev_bias, dev_y)) return rc;
  if (m == 0 || n == 0) return NZ_OK;
  if (int rc = check_product(m, n, k, dev_w_data, dev_w_scales)) return rc;
  if (!dev_x || !dev_y) return nz_fail(NZ_ERR_ARG, "null rows or output");
  if (workspace_bytes < nz_mx_linear_workspace_bytes(m, n, k)) return nz_fail(NZ_ERR_CAPACITY, "workspace too small");
  if (!dev_workspace || !aligned(dev_workspace, 16)) return nz_fail(NZ_ERR_ALIGN, "misaligned workspace");
  uint8_t* xd = (uint8_t*)dev_workspace;
  uint8_t* xs = xd + (m * nz_mx_row_bytes(k, 8) + 255) / 256 * 256;
  launch_quantize(dev_x, dtype, m, (uint32_t)k, stride, 8, xd, xs, (hipStream_t)stream);
  return launch_product(xd, xs, m, dev_w_data, dev_w_scales, n, (uint32_t)k, dev_bias, dev_y, dtype,
                        (hipStream_t)stream);
}

int nz_mx_linear_rows8(const void* dev_x_data, const void* dev_x_scales, uint64_t m, uint64_t k,
                       const void* dev_w_data, const void* dev_w_scales, uint64_t n, const void* dev_bias, void* dev_y,
                       int dtype, void* dev_workspace, uint64_t workspace_bytes, void* stream) {
  (void)dev_workspace, (void)workspace_bytes;
  if (int rc = check_dtype(dtype, dev_bias, dev_y, nullptr)) return rc;
  if (m == 0 || n == 0) return NZ_OK;
  if (int rc = check_product(m, n, k, dev_w_data, dev_w_scales)) return rc;
  if (int rc = check_mx(dev_x_data, dev_x_scales)) return rc;
  if (!dev_y) return nz_fail(NZ_ERR_ARG, "null output");
  return launch_product(dev_x_data, dev_x_scales, m, dev_w_data, dev_w_scales, n, (uint32_t)k, dev_bias, dev_y, dtype,
                        (hipStream_t)stream);
}

int nz_mx_linear_grad(const void* dev_g, int dtype, uint64_t m, uint64_t n, uint64_t stride, const void* dev_w_data,
                      const void* dev_w_scales, uint64_t k, void* dev_dx, void* stream) {
  if (int rc = check_dtype(dtype, dev_g, dev_dx, nullptr)) return rc;
  if (m == 0 || k == 0) return NZ_OK;
  if (!dev_dx) return nz_fail(NZ_ERR_ARG, "null output");
  if (n) {
    if (int rc = check_product(m, n, k, dev_w_data, dev_w_scales)) return rc;
    if (!dev_g) return nz_fail(NZ_ERR_ARG, "null gradient");
  }
  const dim3 grid((uint32_t)nz_ceil_div(k, 64), (uint32_t)nz_ceil_div(m, 64));
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    nz_mx_grad_kernel<T><<<grid, 256, 0, (hipStream_t)stream>>>((const T*)dev_g, stride, m, n,
                                                                (const uint8_t*)dev_w_data,
                                                                (const uint8_t*)dev_w_scales, (uint32_t)k, (T*)dev_dx);
  });
  return nz_launched();
}

}  // extern "C"
