// bf16 rows into 8- or 4-bit codes with a scale per 32 values, the same behind a
// residual addition and RMSNorm, and codes back into bf16 (mx.h has the layout).
//
// Of 32 values with the largest magnitude t the scale is 2^e,
//   e = max(floor(log2 t) - E, -127), E = 8 (e4m3, largest 448) or 2 (e2m1, 6),
// read from t's exponent bits, and the codes are the values / 2^e rounded to the
// nearest (ties to even) by gfx950's scaled conversions, which divide exactly.
// Quotients are below 512 or 8; past the largest code they become that code (the
// e2m1 conversion saturates, the e4m3 one gives NaN from 464 on, so values are
// clamped to 448 * 2^e first). 32 values with an infinity or NaN among them get
// the scale NaN and codes of zero: all of them stand for NaN.
//
// All three are bound by memory: a lane moves 8 values, 16 bytes of bf16, so a
// wave reads whole KiB, and four lanes share a scale (two DPP steps).
#include "kernels.h"
#include "mx.h"

namespace yuear {
namespace mx {
namespace {

typedef short i16x2 __attribute__((ext_vector_type(2)));

// Largest of four neighbouring lanes.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, uint32_t(__builtin_amdgcn_mov_dpp(int(v), 0xB1, 0xF, 0xF, false)));
  return max(v, uint32_t(__builtin_amdgcn_mov_dpp(int(v), 0x4E, 0xF, 0xF, false)));
}

// A lane's 8 values of a block held by four lanes: its codes (4 or 8 bytes) and
// the block's scale byte. Magnitudes are compared as integers, where infinities
// and NaNs are the largest.
template <int BITS>
__device__ __forceinline__ void encode(const float (&v)[8], uint32_t (&codes)[BITS / 4],
                                       uint32_t &scale) {
  constexpr int E = BITS == 8 ? 8 : 2;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    top = max(top, f32_bits(v[i]) & 0x7fffffffu);
  const int exponent = int(quad_max(top) >> 23);
  const bool finite = exponent < 255;
  scale = finite ? uint32_t(max(exponent - E, 0)) : 255u;
  const float s = bits_f32(scale ? scale << 23 : 0x00400000u);  // 2^-127 is subnormal
  if (BITS == 4) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
    codes[0] = finite ? w : 0u;
  } else {
    const float most = 448.f * s;
    auto in = [&](float x) { return __builtin_amdgcn_fmed3f(x, -most, most); };
#pragma unroll
    for (int i = 0; i < BITS / 4; ++i) {
      i16x2 w = {0, 0};
      w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, in(v[4 * i]), in(v[4 * i + 1]), s, false);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, in(v[4 * i + 2]), in(v[4 * i + 3]), s, true);
      codes[i] = finite ? __builtin_bit_cast(uint32_t, w) : 0u;
    }
  }
}

__device__ __forceinline__ void unpack8(u32x4 x, float (&v)[8]) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = bflo(w[i]);
    v[2 * i + 1] = bfhi(w[i]);
  }
}

template <int BITS>
__device__ __forceinline__ void store_codes(uint8_t *p, const uint32_t (&w)[BITS / 4]) {
  if (BITS == 8)
    *reinterpret_cast<uint2 *>(p) = uint2{w[0], w[BITS / 4 - 1]};
  else
    *reinterpret_cast<uint32_t *>(p) = w[0];
}

// Chunk of 8 values: row and place in it of chunk `first + t` of rows of `per`
// chunks, first in chunk `at0` of row `row0`.
struct Place {
  int64_t row;
  uint32_t chunk;
};
__device__ __forceinline__ Place place(int64_t row0, uint32_t at0, uint32_t t, uint32_t per) {
  const uint32_t i = at0 + t, down = i / per;
  return Place{row0 + down, i - down * per};
}

constexpr int kThreads = 256;
constexpr int kLoads = 4;  // chunks of a thread, all read before the first is used

template <int BITS>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const uint16_t *x, int64_t x_stride,
                                                            int64_t chunks, uint32_t per,
                                                            uint8_t *codes, int64_t stride,
                                                            uint8_t *scales, int64_t scale_stride) {
  const int64_t first = int64_t(blockIdx.x) * (kThreads * kLoads);
  const int64_t row0 = first / per;
  const uint32_t at0 = uint32_t(first - row0 * per);
  const uint32_t left = uint32_t(min(chunks - first, int64_t(kThreads * kLoads)));
  u32x4 in[kLoads];
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    const uint32_t t = u * kThreads + threadIdx.x;
    if (t < left) {
      const Place at = place(row0, at0, t, per);
      in[u] = *reinterpret_cast<const u32x4 *>(x + at.row * x_stride + at.chunk * 8);
    }
  }
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    const uint32_t t = u * kThreads + threadIdx.x;
    if (t < left) {  // whole blocks: four lanes agree
      const Place at = place(row0, at0, t, per);
      float v[8];
      unpack8(in[u], v);
      uint32_t w[BITS / 4], scale;
      encode<BITS>(v, w, scale);
      store_codes<BITS>(codes + at.row * stride + at.chunk * BITS, w);
      if ((threadIdx.x & 3) == 0)
        scales[at.row * scale_stride + (at.chunk >> 2)] = uint8_t(scale);
    }
  }
}

// code * 2^(scale - 127) in 32 bits, which hold it exactly (the smallest is
// 2^-9 * 2^-127, a subnormal), then one rounding to bf16.
template <int BITS>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(const uint8_t *codes, int64_t stride,
                                                              const uint8_t *scales,
                                                              int64_t scale_stride, int64_t chunks,
                                                              uint32_t per, uint16_t *out,
                                                              int64_t out_stride) {
  const int64_t first = int64_t(blockIdx.x) * (kThreads * kLoads);
  const int64_t row0 = first / per;
  const uint32_t at0 = uint32_t(first - row0 * per);
  const uint32_t left = uint32_t(min(chunks - first, int64_t(kThreads * kLoads)));
  uint32_t in[kLoads][BITS / 4], scale[kLoads];
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    const uint32_t t = u * kThreads + threadIdx.x;
    if (t < left) {
      const Place at = place(row0, at0, t, per);
      const uint8_t *p = codes + at.row * stride + at.chunk * BITS;
      scale[u] = scales[at.row * scale_stride + (at.chunk >> 2)];
      if (BITS == 8) {
        const uint2 w = *reinterpret_cast<const uint2 *>(p);
        in[u][0] = w.x;
        in[u][BITS / 4 - 1] = w.y;
      } else {
        in[u][0] = *reinterpret_cast<const uint32_t *>(p);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    const uint32_t t = u * kThreads + threadIdx.x;
    if (t < left) {
      const Place at = place(row0, at0, t, per);
      const float s = scale[u] == 255u ? __builtin_nanf("")
                                       : bits_f32(scale[u] ? scale[u] << 23 : 0x00400000u);
      uint32_t w[4];
      auto two = [&](auto pair) {
        return uint32_t(f2bf(pair[0])) | uint32_t(f2bf(pair[1])) << 16;
      };
      if (BITS == 8) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          w[2 * i] = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp8(in[u][i % (BITS / 4)], s, false));
          w[2 * i + 1] = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp8(in[u][i % (BITS / 4)], s, true));
        }
      } else {
        w[0] = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(in[u][0], s, 0));
        w[1] = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(in[u][0], s, 1));
        w[2] = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(in[u][0], s, 2));
        w[3] = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(in[u][0], s, 3));
      }
      if (scale[u] == 255u)
        w[0] = w[1] = w[2] = w[3] = 0x7fc07fc0u;
      *reinterpret_cast<u32x4 *>(out + at.row * out_stride + at.chunk * 8) =
          u32x4{w[0], w[1], w[2], w[3]};
    }
  }
}

struct NormArgs {
  const uint16_t *x, *residual, *gain;
  uint16_t *sum;
  uint8_t *codes, *scales;
  int64_t x_stride, residual_stride, sum_stride, stride, scale_stride;
  int rows, k;
  float eps;
};

// h = bf16(x + residual) (or x), y = h / sqrt(mean h^2 + eps) * gain in 32 bits,
// y quantised without a rounding in between. WPR waves have a row, each lane C
// chunks of 8 in registers from the read to the codes, so a row is read once.
template <int BITS, int WPR, int C>
__global__ __launch_bounds__(256) void norm_kernel(NormArgs p) {
  constexpr int kRows = 4 / WPR;  // rows of a workgroup
  __shared__ float part[4];
  const int wave = threadIdx.x >> 6;
  const int row = int(blockIdx.x) * kRows + wave / WPR;
  const int t = threadIdx.x & (WPR * 64 - 1);
  const int chunks = p.k >> 3;
  const bool in_row = row < p.rows;
  u32x4 x[C], r[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = c * WPR * 64 + t;
    if (in_row && i < chunks) {
      x[c] = *reinterpret_cast<const u32x4 *>(p.x + row * p.x_stride + i * 8);
      if (p.residual)
        r[c] = *reinterpret_cast<const u32x4 *>(p.residual + row * p.residual_stride + i * 8);
    }
  }
  float v[C][8], squares = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = c * WPR * 64 + t;
    if (!(in_row && i < chunks))
      continue;
    unpack8(x[c], v[c]);
    if (p.residual) {
      float a[8];
      unpack8(r[c], a);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[c][e] = rbf(v[c][e] + a[e]);
      u32x4 h;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        h[e] = (f32_bits(v[c][2 * e]) >> 16) | (f32_bits(v[c][2 * e + 1]) & 0xffff0000u);
      *reinterpret_cast<u32x4 *>(p.sum + row * p.sum_stride + i * 8) = h;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      squares = fmaf(v[c][e], v[c][e], squares);
  }
  float total = wave_sum(squares);
  if (WPR > 1) {
    if ((threadIdx.x & 63) == 0)
      part[wave] = total;
    __syncthreads();
    total = (part[0] + part[1]) + (part[2] + part[3]);
  }
  const float scale = 1.0f / __builtin_sqrtf(total / float(p.k) + p.eps);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = c * WPR * 64 + t;
    if (!(in_row && i < chunks))
      continue;
    float g[8];
    unpack8(*reinterpret_cast<const u32x4 *>(p.gain + i * 8), g);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      v[c][e] = v[c][e] * g[e] * scale;  // the first product, of two bf16 values, is exact
    uint32_t w[BITS / 4], s;
    encode<BITS>(v[c], w, s);
    store_codes<BITS>(p.codes + row * p.stride + i * BITS, w);
    if ((threadIdx.x & 3) == 0)
      p.scales[row * p.scale_stride + (i >> 2)] = uint8_t(s);
  }
}

constexpr int kMaxNormK = 16384;

template <int BITS>
hipError_t launch_norm(const NormArgs &p, hipStream_t s) {
  auto go = [&](auto kernel, int rows) {
    hipLaunchKernelGGL(kernel, dim3(unsigned((p.rows + rows - 1) / rows)), dim3(256), 0, s, p);
    return hipGetLastError();
  };
  if (p.k <= 512)
    return go(norm_kernel<BITS, 1, 1>, 4);
  if (p.k <= 2048)
    return go(norm_kernel<BITS, 4, 1>, 1);
  if (p.k <= 4096)
    return go(norm_kernel<BITS, 4, 2>, 1);
  if (p.k <= 8192)
    return go(norm_kernel<BITS, 4, 4>, 1);
  return go(norm_kernel<BITS, 4, 8>, 1);
}

// Workgroups of a call over `chunks` chunks, 0 where the grid cannot hold them.
unsigned groups(int64_t chunks) {
  const int64_t n = (chunks + kThreads * kLoads - 1) / (kThreads * kLoads);
  return n < (int64_t(1) << 31) / kThreads ? unsigned(n) : 0u;
}

}  // namespace
}  // namespace mx
}  // namespace yuear

using namespace yuear;

extern "C" {

int32_t yuear_op_mx_quantize(const uint16_t *x, int64_t x_stride, int32_t rows, int32_t k,
                             int32_t bits, uint8_t *codes, int64_t codes_stride, uint8_t *scales,
                             int64_t scales_stride, void *stream) {
  if (rows == 0)
    return 0;
  if (rows < 0 || !mx::rows_ok(codes, codes_stride, scales, scales_stride, k, bits) ||
      !mx::wide_ok(x, x_stride, k))
    return int32_t(hipErrorInvalidValue);
  const mx::Span in = mx::bf16_span(x, x_stride, rows, k),
                 c = mx::codes_span(codes, codes_stride, rows, k, bits),
                 s = mx::scales_span(scales, scales_stride, rows, k);
  const unsigned grid = mx::groups(int64_t(rows) * (k / 8));
  if (mx::overlap(in, c) || mx::overlap(in, s) || mx::overlap(c, s) || !grid)
    return int32_t(hipErrorInvalidValue);
  hipLaunchKernelGGL(bits == 8 ? mx::quantize_kernel<8> : mx::quantize_kernel<4>, dim3(grid),
                     dim3(mx::kThreads), 0, static_cast<hipStream_t>(stream), x, x_stride,
                     int64_t(rows) * (k / 8), uint32_t(k / 8), codes, codes_stride, scales,
                     scales_stride);
  return int32_t(hipGetLastError());
}

int32_t yuear_op_mx_dequantize(const uint8_t *codes, int64_t codes_stride, const uint8_t *scales,
                               int64_t scales_stride, int32_t rows, int32_t k, int32_t bits,
                               uint16_t *out, int64_t out_stride, void *stream) {
  if (rows == 0)
    return 0;
  if (rows < 0 || !mx::rows_ok(codes, codes_stride, scales, scales_stride, k, bits) ||
      !mx::wide_ok(out, out_stride, k))
    return int32_t(hipErrorInvalidValue);
  const mx::Span o = mx::bf16_span(out, out_stride, rows, k);
  const unsigned grid = mx::groups(int64_t(rows) * (k / 8));
  if (mx::overlap(o, mx::codes_span(codes, codes_stride, rows, k, bits)) ||
      mx::overlap(o, mx::scales_span(scales, scales_stride, rows, k)) || !grid)
    return int32_t(hipErrorInvalidValue);
  hipLaunchKernelGGL(bits == 8 ? mx::dequantize_kernel<8> : mx::dequantize_kernel<4>, dim3(grid),
                     dim3(mx::kThreads), 0, static_cast<hipStream_t>(stream), codes, codes_stride,
                     scales, scales_stride, int64_t(rows) * (k / 8), uint32_t(k / 8), out,
                     out_stride);
  return int32_t(hipGetLastError());
}

int32_t yuear_op_mx_rms_norm(const uint16_t *x, int64_t x_stride, const uint16_t *residual,
                             int64_t residual_stride, const uint16_t *gain, float eps,
                             int32_t rows, int32_t k, int32_t bits, uint8_t *codes,
                             int64_t codes_stride, uint8_t *scales, int64_t scales_stride,
                             uint16_t *sum, int64_t sum_stride, void *stream) {
  if (rows == 0)
    return 0;
  if (rows < 0 || rows >= 1 << 23 || k > mx::kMaxNormK ||
      !mx::rows_ok(codes, codes_stride, scales, scales_stride, k, bits) ||
      !mx::wide_ok(x, x_stride, k) || !mx::aligned(gain, 16) || !residual != !sum ||
      (residual &&
       (!mx::wide_ok(residual, residual_stride, k) || !mx::wide_ok(sum, sum_stride, k))))
    return int32_t(hipErrorInvalidValue);
  const mx::Span in = mx::bf16_span(x, x_stride, rows, k),
                 res = mx::bf16_span(residual, residual_stride, rows, k),
                 h = mx::bf16_span(sum, sum_stride, rows, k),
                 g = mx::bf16_span(gain, k, 1, k),
                 c = mx::codes_span(codes, codes_stride, rows, k, bits),
                 s = mx::scales_span(scales, scales_stride, rows, k);
  // the sum may replace either of its parts: a lane reads its values before it writes them
  auto apart = [&](const uint16_t *part, int64_t stride, const mx::Span &span) {
    return (part == sum && stride == sum_stride) || !mx::overlap(span, h);
  };
  for (const mx::Span &from : {in, res, g, h})
    if (mx::overlap(from, c) || mx::overlap(from, s))
      return int32_t(hipErrorInvalidValue);
  if (mx::overlap(c, s) || mx::overlap(g, h) || !apart(x, x_stride, in) ||
      !apart(residual, residual_stride, res))
    return int32_t(hipErrorInvalidValue);
  const mx::NormArgs p{x,        residual,        gain,       sum,          codes,
                       scales,   x_stride,        residual_stride, sum_stride, codes_stride,
                       scales_stride, rows,       k,          eps};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return int32_t(bits == 8 ? mx::launch_norm<8>(p, st) : mx::launch_norm<4>(p, st));
}

}  // extern "C"
