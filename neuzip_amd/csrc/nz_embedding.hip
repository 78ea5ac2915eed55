// The gradient of an embedding table.
#include "nz_operators.h"

namespace {

// One wavefront per row of the table and 512 of its columns: it looks through all indices for its row and adds the
// gradients of those it finds, in their order.
template <class T>
__global__ __launch_bounds__(256) void nz_embedding_gradient_kernel(const long long* index, uint32_t count,
                                                                    const T* g, uint64_t stride, uint64_t rows,
                                                                    uint32_t cols, uint32_t slices, float scale,
                                                                    long long skip, uint32_t flags, T* out) {
  const uint64_t wave = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64;
  const uint64_t row = wave / slices;
  if (row >= rows) return;
  const uint32_t lane = threadIdx.x & 63, c0 = (uint32_t)(wave - row * slices) * 512 + lane;
  float sum[8] = {};
  uint32_t found = 0;
  if ((long long)row != skip)
    for (uint32_t at = 0; at < count; at += 64) {
      uint64_t hits = __ballot(at + lane < count && index[at + lane] == (long long)row);
      found += __popcll(hits);
      for (; hits; hits &= hits - 1) {
        const T* p = g + (at + __builtin_ctzll(hits)) * stride;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c0 + i * 64 < cols) sum[i] += (float)p[c0 + i * 64];
      }
    }
  if (!found && (flags & NZ_GRAD_ACCUMULATE)) return;
  const float f = flags & NZ_GRAD_BY_FREQUENCY && found ? scale / (float)found : scale;
  T* q = out + row * cols;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c0 + i * 64 < cols) {
      float v = sum[i] * f;
      if (flags & NZ_GRAD_ACCUMULATE) v += (float)q[c0 + i * 64];
      q[c0 + i * 64] = (T)v;
    }
}

}  // namespace

extern "C" {

uint64_t nz_embedding_gradient_workspace_bytes(uint64_t count, uint64_t rows, uint64_t cols) {
  (void)count, (void)rows, (void)cols;
  return 0;
}

int nz_embedding_gradient(const void* dev_indices, uint64_t count, const void* dev_g, int dtype, uint64_t stride,
                          uint64_t rows, uint64_t cols, float scale, int64_t padding_idx, uint32_t flags,
                          void* dev_out, void* dev_workspace, uint64_t workspace_bytes, void* stream) {
  (void)dev_workspace;
  const uint32_t size = nz_dtype_bytes(dtype);
  if (!size) return nz_fail(NZ_ERR_DTYPE, "Unsupported data type");
  if (flags & ~(NZ_GRAD_BY_FREQUENCY | NZ_GRAD_ACCUMULATE)) return nz_fail(NZ_ERR_ARG, "unknown flags");
  if (rows == 0 || cols == 0) return NZ_OK;
  if (cols > 0x40000000ull || rows > 0x7FFFFFFFull || count > 0x7FFFFFFFull)
    return nz_fail(NZ_ERR_ARG, "too many rows, columns or indices");
  if (!dev_out || (count && (!dev_indices || !dev_g))) return nz_fail(NZ_ERR_ARG, "null indices, gradient or output");
  if ((uintptr_t)dev_indices % 8 || (uintptr_t)dev_g % size || (uintptr_t)dev_out % size)
    return nz_fail(NZ_ERR_ALIGN, "pointers must be aligned to their elements");
  if (workspace_bytes < nz_embedding_gradient_workspace_bytes(count, rows, cols))
    return nz_fail(NZ_ERR_CAPACITY, "workspace too small");
  const uint32_t slices = (uint32_t)nz_ceil_div(cols, 512);
  const uint64_t blocks = nz_ceil_div(rows * slices, 4);
  if (blocks > 0x7FFFFFFFull) return nz_fail(NZ_ERR_ARG, "too many rows for one launch");
  const hipStream_t st = (hipStream_t)stream;
  const dim3 grid((uint32_t)blocks);
#define NZ_GRADIENT(T)                                                                                               \
  nz_embedding_gradient_kernel<T><<<grid, 256, 0, st>>>((const long long*)dev_indices, (uint32_t)count,              \
                                                        (const T*)dev_g, stride, rows, (uint32_t)cols, slices, scale, \
                                                        padding_idx, flags, (T*)dev_out)
  if (dtype == NZ_DTYPE_BF16)
    NZ_GRADIENT(nz_bf16);
  else if (dtype == NZ_DTYPE_F16)
    NZ_GRADIENT(nz_f16);
  else
    NZ_GRADIENT(float);
#undef NZ_GRADIENT
  return nz_launched();
}

}  // extern "C"
