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
// wave reads whole KiB, and four lanes share a scale (two DPP steps). MI355X, where a
// plain copy reaches 4.7 TB/s, from memory (from the last-level cache): quantising 3000 x 8192
// in 8 bits 17.9 us (13.5 to 15.2), 4.2 TB/s; 16384 x 3072 in 4 bits and back 52, 4.9 TB/s; the
// norm of 3000 x 3072 with its residual 17.2 (12.6 to 14.4), 3.8 TB/s. One row of 3072: 1.8 and
// 2.6 us, a launch.
#include <algorithm>

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

// The rows' chunks of 8 values, `per` a row, in one sequence. A thread has one, and a
// workgroup 256 of them: with four a thread, all read before the first is used, 3000 x
// 8192 values in 8 bits take 15.8 us instead of 13.5, and 517 x 2048 in 4 bits and back
// 6.7 instead of 4.8. (Past the grid's limit a thread goes on to the chunk that lies
// all threads further.)
struct Place {
  int64_t row;
  uint32_t chunk;
};
__device__ __forceinline__ Place place(int64_t i, uint32_t per) {
  const int64_t row = i / per;
  return Place{row, uint32_t(i - row * per)};
}

constexpr int kThreads = 256;
constexpr int64_t kMaxValues = int64_t(1) << 40;  // of a call: more than memory holds

template <int BITS>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const uint16_t *x, int64_t x_stride,
                                                            int64_t chunks, uint32_t per,
                                                            uint8_t *codes, int64_t stride,
                                                            uint8_t *scales, int64_t scale_stride) {
  for (int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x; i < chunks;
       i += int64_t(gridDim.x) * kThreads) {  // whole blocks: four lanes agree
    const Place at = place(i, per);
    float v[8];
    unpack8(*reinterpret_cast<const u32x4 *>(x + at.row * x_stride + at.chunk * 8), v);
    uint32_t w[BITS / 4], scale;
    encode<BITS>(v, w, scale);
    store_codes<BITS>(codes + at.row * stride + at.chunk * BITS, w);
    if ((threadIdx.x & 3) == 0)
      scales[at.row * scale_stride + (at.chunk >> 2)] = uint8_t(scale);
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
  for (int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x; i < chunks;
       i += int64_t(gridDim.x) * kThreads) {
    const Place at = place(i, per);
    const uint8_t *p = codes + at.row * stride + at.chunk * BITS;
    const uint32_t scale = scales[at.row * scale_stride + (at.chunk >> 2)];
    const float s = bits_f32(scale ? scale << 23 : 0x00400000u);
    auto two = [&](auto pair) {
      return uint32_t(f2bf(pair[0])) | uint32_t(f2bf(pair[1])) << 16;
    };
    u32x4 w;
    if (BITS == 8) {
      const uint2 in = *reinterpret_cast<const uint2 *>(p);
      w[0] = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp8(in.x, s, false));
      w[1] = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp8(in.x, s, true));
      w[2] = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp8(in.y, s, false));
      w[3] = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp8(in.y, s, true));
    } else {
      const uint32_t in = *reinterpret_cast<const uint32_t *>(p);
      w[0] = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(in, s, 0));
      w[1] = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(in, s, 1));
      w[2] = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(in, s, 2));
      w[3] = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(in, s, 3));
    }
    if (scale == 255u)
      w = u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
    *reinterpret_cast<u32x4 *>(out + at.row * out_stride + at.chunk * 8) = w;
  }
}

struct NormArgs {
  const uint16_t *x, *residual, *gain;
  uint16_t *sum;
  uint8_t *codes, *scales;
  int64_t x_stride, residual_stride, sum_stride, stride, scale_stride;
  int rows, k;
  float eps;
  double inverse_k;
};

// Sum over the wave's lanes.
template <int CTRL> __device__ __forceinline__ double dpp64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = uint32_t(__builtin_amdgcn_mov_dpp(int(b), CTRL, 0xF, 0xF, false));
  const uint32_t hi = uint32_t(__builtin_amdgcn_mov_dpp(int(b >> 32), CTRL, 0xF, 0xF, false));
  return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_sum64(double v) {
  v += dpp64<0xB1>(v);   // lane ^ 1
  v += dpp64<0x4E>(v);   // lane ^ 2
  v += dpp64<0x141>(v);  // the other quad of the half-row
  v += dpp64<0x140>(v);  // the other half of the row of 16
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  auto row = [&](int lane) {
    const uint32_t lo = uint32_t(__builtin_amdgcn_readlane(int(b), lane));
    const uint32_t hi = uint32_t(__builtin_amdgcn_readlane(int(b >> 32), lane));
    return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
  };
  return (row(0) + row(16)) + (row(32) + row(48));
}

// The edges of the codes, their ties, and the powers of two, where a block's scale changes, end in
// 19 zeros. y = p scale in 32 bits is less than 4 units of its last place off (3.5 roundings: half
// a one in the mean's root, the root's, the quotient's, the product's), so where its last 19 bits
// are more than 4 away from zeros it lies on the side that it would lie on exactly. A wave's 512
// values have one nearer in 1 of 100 cases. (Zeros, two in a row of a sum's 3072, are none, or
// the branch cost 0.2 us a row: what is added, 5 units, leaves products from 2^-122 on.)
__device__ __forceinline__ bool near_an_edge(const float (&p)[8], float scale) {
  uint32_t least = ~0u;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    least = min(least, (f32_bits(fmaf(p[e], scale, bits_f32(5u))) << 13) + (4u << 13));
  return least < 9u << 13;
}

// The same in 64 bits, scale with a Newton step (none where it is 0 or infinite): 1.5 times the
// square of scale's 2.5 roundings of 2^-24 is left, 2^-44.7. Products may lie on an edge itself
// though their factor is no float (rows of one magnitude: 3 gain / 3), so what is within 2^-43 of
// one may be taken for it; the rest is rounded to odd, towards zero and the last bit set, which keeps
// its side.
__device__ __forceinline__ void settle8(const float (&p)[8], double mean, float scale, float (&y)[8]) {
  asm volatile("" : "+v"(scale));  // or the step is taken ahead of the branch
  const double s = scale, off = fma(-mean * s, s, 1.0), factor = fabs(off) < 1e-6 ? fma(0.5 * s, off, s) : s;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint64_t b = (__builtin_bit_cast(uint64_t, double(p[e]) * factor) + 0x200u) & ~uint64_t(0x3ff);
    const uint64_t top = b & ~((uint64_t(1) << 29) - 1);
    y[e] = bits_f32(f32_bits(float(__builtin_bit_cast(double, top))) | uint32_t(b != top));
  }
}

// h = bf16(x + residual) (or x), y = h * gain / sqrt(mean h^2 + eps), y quantised without a
// rounding in between. A workgroup has a row, each lane C chunks of 8 in registers from
// the read to the codes, so a row is read once. The squares are added in 64 bits, and products
// whose side of a code's edge is in doubt are taken again in 64 bits, which makes the codes those of
// 64-bit arithmetic: a row's values all carry its factor's error, and one that it takes past a
// code's edge is off by a whole step of the code (7 in 9 million with all of it in 32 bits, and
// one in 30 of a row of one magnitude).
template <int BITS, int C>
__global__ __launch_bounds__(1024) void norm_kernel(NormArgs p) {
  __shared__ double part[16];
  const int waves = int(blockDim.x) >> 6, chunks = p.k >> 3;
  const int64_t row = blockIdx.x;
  u32x4 x[C], r[C], gain[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = c * int(blockDim.x) + int(threadIdx.x);
    if (i < chunks) {
      x[c] = *reinterpret_cast<const u32x4 *>(p.x + row * p.x_stride + i * 8);
      if (p.residual)
        r[c] = *reinterpret_cast<const u32x4 *>(p.residual + row * p.residual_stride + i * 8);
      gain[c] = *reinterpret_cast<const u32x4 *>(p.gain + i * 8);
    }
  }
  float v[C][8];
  double squares = 0.0;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = c * int(blockDim.x) + int(threadIdx.x);
    if (i >= chunks)
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
      squares = fma(double(v[c][e]), double(v[c][e]), squares);
  }
  double total = wave_sum64(squares);
  if (waves > 1) {
    if ((threadIdx.x & 63) == 0)
      part[threadIdx.x >> 6] = total;
    lds_barrier();  // the stores of h go on
    total = part[0];
    for (int w = 1; w < waves; ++w)
      total += part[w];
  }
  const double mean = fma(total, p.inverse_k, double(p.eps));
  const float scale = 1.0f / __builtin_sqrtf(float(mean));
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = c * int(blockDim.x) + int(threadIdx.x);
    if (i >= chunks)
      continue;
    float g[8], y[8];
    unpack8(gain[c], g);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      y[e] = (g[e] *= v[c][e]) * scale;  // the first product, of two bf16 values, is exact
    if (__builtin_expect(near_an_edge(g, scale), 0))
      settle8(g, mean, scale, y);
    uint32_t w[BITS / 4], s;
    encode<BITS>(y, w, s);
    store_codes<BITS>(p.codes + row * p.stride + i * BITS, w);
    if ((threadIdx.x & 3) == 0)
      p.scales[row * p.scale_stride + (i >> 2)] = uint8_t(s);
  }
}

constexpr int kMaxNormK = 16384;

// One chunk a lane and k / 512 waves are the quickest for few rows, two no slower for many long
// ones, whose workgroups they halve (us, with a residual, rows from memory):
//    1 x 3072: 2.43, 2.62    8000 x 3072: 35.2, 35.0    8000 x 2048: 23.6, 24.5
//    1 x 2048: 2.14, 2.52    3000 x 8192: 35.0, 35.0    8000 x 1024: 15.1, 14.8
// The choice goes by k alone, so that a row's sum has one order however many rows there are.
template <int BITS> hipError_t launch_norm(NormArgs p, hipStream_t s) {
  const int each = p.k <= 2048 ? 1 : 2, threads = (p.k / 8 + 64 * each - 1) / (64 * each) * 64;
  constexpr int kMost = 1 << 21;  // of a launch, whose threads count in 32 bits
  for (int left = p.rows; left > 0; left -= kMost) {
    p.rows = std::min(left, kMost);
    hipLaunchKernelGGL((each == 1 ? norm_kernel<BITS, 1> : norm_kernel<BITS, 2>),
                       dim3(unsigned(p.rows)), dim3(unsigned(threads)), 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
      return e;
    p.x += p.rows * p.x_stride;
    if (p.residual) {
      p.residual += p.rows * p.residual_stride;
      p.sum += p.rows * p.sum_stride;
    }
    p.codes += p.rows * p.stride;
    p.scales += p.rows * p.scale_stride;
  }
  return hipSuccess;
}

// Workgroups of a call over `chunks` chunks.
unsigned groups(int64_t chunks) {
  return unsigned(std::min<int64_t>((chunks + kThreads - 1) / kThreads, 1 << 23));
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
  if (rows < 0 || int64_t(rows) * k > mx::kMaxValues ||
      !mx::rows_ok(codes, codes_stride, scales, scales_stride, k, bits) ||
      !mx::wide_ok(x, x_stride, k))
    return int32_t(hipErrorInvalidValue);
  const mx::Span in = mx::bf16_span(x, x_stride, rows, k),
                 c = mx::codes_span(codes, codes_stride, rows, k, bits),
                 s = mx::scales_span(scales, scales_stride, rows, k);
  if (mx::overlap(in, c) || mx::overlap(in, s) || mx::overlap(c, s))
    return int32_t(hipErrorInvalidValue);
  hipLaunchKernelGGL(bits == 8 ? mx::quantize_kernel<8> : mx::quantize_kernel<4>,
                     dim3(mx::groups(int64_t(rows) * (k / 8))), dim3(mx::kThreads), 0,
                     static_cast<hipStream_t>(stream), x, x_stride,
                     int64_t(rows) * (k / 8), uint32_t(k / 8), codes, codes_stride, scales,
                     scales_stride);
  return int32_t(hipGetLastError());
}

int32_t yuear_op_mx_dequantize(const uint8_t *codes, int64_t codes_stride, const uint8_t *scales,
                               int64_t scales_stride, int32_t rows, int32_t k, int32_t bits,
                               uint16_t *out, int64_t out_stride, void *stream) {
  if (rows == 0)
    return 0;
  if (rows < 0 || int64_t(rows) * k > mx::kMaxValues ||
      !mx::rows_ok(codes, codes_stride, scales, scales_stride, k, bits) ||
      !mx::wide_ok(out, out_stride, k))
    return int32_t(hipErrorInvalidValue);
  const mx::Span o = mx::bf16_span(out, out_stride, rows, k);
  if (mx::overlap(o, mx::codes_span(codes, codes_stride, rows, k, bits)) ||
      mx::overlap(o, mx::scales_span(scales, scales_stride, rows, k)))
    return int32_t(hipErrorInvalidValue);
  hipLaunchKernelGGL(bits == 8 ? mx::dequantize_kernel<8> : mx::dequantize_kernel<4>,
                     dim3(mx::groups(int64_t(rows) * (k / 8))), dim3(mx::kThreads), 0,
                     static_cast<hipStream_t>(stream), codes, codes_stride,
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
  if (rows < 0 || k > mx::kMaxNormK ||
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
                       scales_stride, rows,       k,          eps, 1.0 / k};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return int32_t(bits == 8 ? mx::launch_norm<8>(p, st) : mx::launch_norm<4>(p, st));
}

}  // extern "C"
