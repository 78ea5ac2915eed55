// What the operators beside the codec (nz_mx.hip, nz_fp8.hip, nz_embedding.hip) share.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/neuzip_hip.h"

// Set the calling thread's message (nz_last_error) and hand the code back (nz_api.hip).
__attribute__((visibility("hidden"))) int nz_fail(int code, const char* msg);

// Compute units of the device in use (nz_api.hip).
__attribute__((visibility("hidden"))) uint32_t nz_compute_units();

// NZ_OK, or what the launches since the last look have failed with.
inline int nz_launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? NZ_OK : nz_fail(NZ_ERR_HIP, hipGetErrorString(e));
}

inline uint64_t nz_ceil_div(uint64_t a, uint64_t b) { return a / b + (a % b != 0); }

inline uint32_t nz_dtype_bytes(int dtype) {
  return dtype == NZ_DTYPE_F32 ? 4u : dtype == NZ_DTYPE_BF16 || dtype == NZ_DTYPE_F16 ? 2u : 0u;
}

// a * b, or 2^64 - 1 where that is too large
inline uint64_t nz_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  return __builtin_mul_overflow(a, b, &r) ? ~0ull : r;
}

// Workgroups of `threads` threads that one launch may have along an axis: its threads are counted in 32 bits.  (Beyond
// that a launch is no error here, it leaves workgroups out.)
inline uint64_t nz_most_groups(uint32_t threads) { return 0xFFFFFFFFull / threads; }

// f(first, count) for pieces of `rows` rows, each as many as a launch of workgroups of 256 threads takes with `threads`
// threads to a row: one piece, but for tens of millions of rows.
template <class F>
inline void nz_in_pieces(uint64_t rows, uint64_t threads, F f) {
  const uint64_t most = nz_most_groups(256) * 256 / threads;
  for (uint64_t first = 0; first < rows; first += most) f(first, rows - first < most ? rows - first : most);
}

using nz_bf16 = __bf16;
using nz_f16 = _Float16;
