// Rows of 8-bit (e4m3) or 4-bit (e2m1) codes with one power-of-two scale (e8m0:
// 2^(byte - 127), 255 for NaN) per 32 values, the operands of gfx950's scaled
// MFMA, shared by the quantisation (mx_quantize.hip) and the product
// (mx_gemm.hip). A row's codes are consecutive, 4-bit ones two to a byte with
// the first in the low half; its k / 32 scales are a row of their own.
#pragma once
#include "common.h"

namespace yuear {
namespace mx {

constexpr int kBlock = 32;            // values of a scale
constexpr int kMaxK = 1 << 20;        // values of a row
constexpr int64_t kMaxStride = 1 << 22;  // bytes from row to row: 256 rows count in 32 bits

// The workgroup's barrier after a wave's LDS operations. (__syncthreads() would wait for its
// global memory operations too, loads into LDS and stores.)
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ---- host-side checks ----
inline bool aligned(const void *p, int bytes) {
  return p && (reinterpret_cast<uintptr_t>(p) & uintptr_t(bytes - 1)) == 0;
}
// A row array in memory: `rows` rows of `bytes` bytes, `stride` bytes apart.
struct Span {
  const void *base;
  int64_t rows, bytes, stride;
};
// Whether two row arrays share a byte. Rows of one stride may lie between each
// other (columns of one wide array); of unlike strides they count as sharing
// where their address ranges meet.
inline bool overlap(const Span &x, const Span &y) {
  if (!x.base || !y.base || x.rows < 1 || y.rows < 1)
    return false;
  const uintptr_t a = reinterpret_cast<uintptr_t>(x.base), b = reinterpret_cast<uintptr_t>(y.base);
  const uintptr_t ae = a + uintptr_t((x.rows - 1) * x.stride + x.bytes),
                  be = b + uintptr_t((y.rows - 1) * y.stride + y.bytes);
  if (ae <= b || be <= a)
    return false;
  if (x.stride != y.stride)
    return true;
  const uintptr_t s = uintptr_t(x.stride);
  const uintptr_t d = b >= a ? (b - a) % s : (s - (a - b) % s) % s;  // y's column in x's rows
  return d < uintptr_t(x.bytes) || d + uintptr_t(y.bytes) > s;
}
// Codes and scales of `rows` rows of k values that a call is given.
inline bool rows_ok(const uint8_t *codes, int64_t stride, const uint8_t *scales,
                    int64_t scale_stride, int k, int bits) {
  return (bits == 4 || bits == 8) && k >= kBlock && k <= kMaxK && k % kBlock == 0 &&
         aligned(codes, 16) && stride >= int64_t(k) * bits / 8 && stride % 16 == 0 &&
         stride <= kMaxStride && scales && scale_stride >= k / kBlock && scale_stride <= kMaxStride;
}
// bf16 rows that are read or written 16 bytes a lane.
inline bool wide_ok(const uint16_t *p, int64_t stride, int k) {
  return aligned(p, 16) && stride >= k && stride % 8 == 0 && stride <= kMaxStride;
}
inline Span codes_span(const uint8_t *codes, int64_t stride, int64_t rows, int k, int bits) {
  return Span{codes, rows, int64_t(k) * bits / 8, stride};
}
inline Span scales_span(const uint8_t *scales, int64_t stride, int64_t rows, int k) {
  return Span{scales, rows, k / kBlock, stride};
}
inline Span bf16_span(const uint16_t *p, int64_t stride, int64_t rows, int64_t n) {
  return Span{p, rows, 2 * n, 2 * stride};
}

}  // namespace mx
}  // namespace yuear
