// Operands of the matrix products as their callers give them: copies of those
// that the loads to LDS cannot take, and the bytes of a product's workspace.
#pragma once

#include "mhc_gemm.hpp"

namespace mhc {
namespace gemm {

// rows of `width` elements, `ld` apart, into rows of whole chunks of 16 bytes, with zeros after the last element
template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(const T* src, int64_t ld, T* dst, int64_t rows, int64_t width, int64_t chunks) {
  constexpr int kE = 16 / (int)sizeof(T);
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < rows * chunks; at += (int64_t)gridDim.x * 256) {
    const int64_t row = at / chunks, k = at % chunks * kE;
    const T* const p = src + row * ld + k;
    u32x4 v = {0, 0, 0, 0};
    if (k + kE <= width) {
      __builtin_memcpy(&v, p, 16);
    } else {
      T e[kE];
#pragma unroll
      for (int j = 0; j < kE; ++j) e[j] = k + j < width ? p[j] : (T)0;
      __builtin_memcpy(&v, e, 16);
    }
    reinterpret_cast<u32x4*>(dst)[at] = v;
  }
}

// bytes of the sums of an M x N product whose reduction is split
inline size_t part_bytes(const Cut& c, int64_t M, int64_t N) { return c.splits > 1 ? (size_t)(c.splits * M * N) * sizeof(float) : 0; }

inline size_t up256(size_t b) { return (b + 255) / 256 * 256; }

// a row's length in a copy: a multiple of eight elements, and of sixteen bytes
inline int64_t padded(int64_t width, int dtype) { return dtype == kI8 ? (width + 15) / 16 * 16 : (width + 7) / 8 * 8; }

// bytes of an operand's copy in rows of whole chunks; 0: it is read as it is
inline size_t pack_bytes(const void* p, int64_t rows, int64_t ld, int64_t width, int dtype) {
  if (in_words(p, ld, width, elem_bytes(dtype))) return 0;
  return up256((size_t)(rows * padded(width, dtype)) * elem_bytes(dtype));
}

template <typename T>
int run_pack(const void* p, int64_t ld, void* to, int64_t rows, int64_t width, int64_t wide, hipStream_t s) {
  const int64_t chunks = wide * (int64_t)sizeof(T) / 16;
  const int64_t blocks = std::min(ceil_div(rows * chunks, 256), (int64_t)device_cu_count() * 16);
  hipLaunchKernelGGL((pack_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, s, static_cast<const T*>(p), ld,
                     static_cast<T*>(to), rows, width, chunks);
  MHC_CHECK_LAUNCH("pack_kernel");
  return MHC_OK;
}

// The operand, copied to `ws` first (which moves on) where its rows are no whole words.
inline int operand(Operand& o, const void* p, int64_t rows, int64_t ld, int64_t width, int dtype, char*& ws, hipStream_t s) {
  const size_t bytes = pack_bytes(p, rows, ld, width, dtype);
  if (bytes == 0) {
    o = Operand{p, ld, width};
    return MHC_OK;
  }
  const int64_t wide = padded(width, dtype);
  o = Operand{ws, wide, wide};
  const int rc = dtype == kF32  ? run_pack<float>(p, ld, ws, rows, width, wide, s)
                 : dtype == kI8 ? run_pack<uint8_t>(p, ld, ws, rows, width, wide, s)
                                : run_pack<uint16_t>(p, ld, ws, rows, width, wide, s);
  ws += bytes;
  return rc;
}

}  // namespace gemm
}  // namespace mhc
