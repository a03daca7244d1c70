// C[m][n] = bf16(epilogue(sum_k A[m][k] W[n][k])) of rows with a scale per 32
// values (mx.h): activations in 8 or 4 bits, weights in 4, on gfx950's scaled
// MFMA, 128 of K at a time with sums in fp32.
#include "kernels.h"
#include "mx.h"

namespace yuear {
namespace mx {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

enum Epilogue : int { kStore = 0, kResidual = 1, kSwiglu = 2 };

struct GemmArgs {
  const uint8_t *a, *a_scales, *w, *w_scales;
  int64_t a_stride, a_scale_stride, w_stride, w_scale_stride;
  int m, n, k;
  const uint16_t *residual;
  uint16_t *c;
  int64_t residual_stride, ldc;
  int epilogue;
};

constexpr int kStep = 128;  // K of an MFMA

// Range of a tile's `rows` rows (at most 256) from `base`, of which the last ends
// with its data: what lies past it reads as zero.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const uint8_t *base, int64_t stride,
                                                            int rows, int bytes) {
  const int64_t n = (rows - 1) * stride + bytes;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, int(n), 0x00020000);
}

__device__ __forceinline__ float silu_times(float gate, float up) {
  return gate / (1.0f + expf(-gate)) * up;
}

// A lane's features n .. n + 3 (n a multiple of 4) of token row m < p.m.
__device__ __forceinline__ void finish4(const GemmArgs &p, int m, int n, const float (&v)[4]) {
  if (n >= p.n)
    return;
  if (p.epilogue == kSwiglu) {
    uint16_t *c = p.c + m * p.ldc + (n >> 1);
    c[0] = f2bf(silu_times(v[0], v[1]));
    if (n + 2 < p.n)
      c[1] = f2bf(silu_times(v[2], v[3]));
    return;
  }
  uint16_t *c = p.c + m * p.ldc + n;
  const uint16_t *r = p.residual + m * p.residual_stride + n;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < p.n)
      c[e] = f2bf(p.epilogue == kResidual ? bf2f(r[e]) + v[e] : v[e]);
}

// Few token rows: a workgroup computes 16 FT features of 16 MT tokens, its KW
// waves a part of K each with all operands straight from memory into registers,
// then adds the waves' sums in order.
//
// MFMA operands, lane l = 16 g + r: W (4 bits) row r, k 32 g .. 32 g + 31 of the
// step, the same of A in 4 bits; A in 8 bits k 16 g .. 16 g + 15 and 64 + 16 g ..;
// the scale of k-block g of row r in either case. D: features 4 g .. 4 g + 3 of
// token r.
template <int ABITS, int MT, int FT, int KW>
__global__ __launch_bounds__(KW * 64) void rows_kernel(GemmArgs p) {
  constexpr int AQ = ABITS / 4;  // 16-byte pieces of A of a lane and step
  constexpr int kBatch = 4;      // steps whose loads go out together
  __shared__ f32x4 sums[KW][FT * MT][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int n0 = int(blockIdx.x) * (16 * FT), m0 = int(blockIdx.y) * (16 * MT);
  const auto ra = rows_rsrc(p.a + m0 * p.a_stride, p.a_stride, min(p.m - m0, 16 * MT), p.k * ABITS / 8);
  const auto rw = rows_rsrc(p.w + n0 * p.w_stride, p.w_stride, min(p.n - n0, 16 * FT), p.k / 2);
  const auto rsa =
      rows_rsrc(p.a_scales + m0 * p.a_scale_stride, p.a_scale_stride,
                             min(p.m - m0, 16 * MT), p.k / 32);
  const auto rsw =
      rows_rsrc(p.w_scales + n0 * p.w_scale_stride, p.w_scale_stride,
                             min(p.n - n0, 16 * FT), p.k / 32);
  const int steps = p.k / kStep;
  const int begin = steps * wave / KW, end = steps * (wave + 1) / KW;
  f32x4 acc[FT][MT];
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t)
      acc[f][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = begin; s < end; s += kBatch) {
    u32x4 w[FT][kBatch], a[MT][kBatch][AQ], ws[FT], as[MT];
#pragma unroll
    for (int f = 0; f < FT; ++f) {
      const int row = 16 * f + r;
      ws[f] = __builtin_amdgcn_raw_buffer_load_b128(rsw, row * int(p.w_scale_stride) + 4 * s, 0, 0);
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        w[f][j] = __builtin_amdgcn_raw_buffer_load_b128(
            rw, row * int(p.w_stride) + (s + j) * (kStep / 2) + 16 * g, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int row = 16 * t + r;
      as[t] = __builtin_amdgcn_raw_buffer_load_b128(rsa, row * int(p.a_scale_stride) + 4 * s, 0, 0);
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
#pragma unroll
        for (int q = 0; q < AQ; ++q)
          a[t][j][q] = __builtin_amdgcn_raw_buffer_load_b128(
              ra, row * int(p.a_stride) + (s + j) * (kStep * ABITS / 8) + 64 * q + 16 * g, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (s + j >= end)  // what was read past the wave's part counts for nothing
        break;
#pragma unroll
      for (int f = 0; f < FT; ++f)
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const u32x4 lo = a[t][j][0], hi = a[t][j][AQ - 1];
          const i32x8 wv = {int(w[f][j].x), int(w[f][j].y), int(w[f][j].z), int(w[f][j].w), 0, 0, 0, 0};
          const i32x8 av = {int(lo.x), int(lo.y), int(lo.z), int(lo.w),
                            int(hi.x), int(hi.y), int(hi.z), int(hi.w)};
          acc[f][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
              wv, av, acc[f][t], 4, ABITS == 8 ? 0 : 4, 0, int(ws[f][j] >> (8 * g)), 0,
              int(as[t][j] >> (8 * g)));
        }
    }
  }
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t)
      sums[wave][f * MT + t][lane] = acc[f][t];
  __syncthreads();
  for (int i = threadIdx.x; i < FT * MT * 64; i += KW * 64) {
    const int tile = i >> 6, l = i & 63;
    f32x4 sum = sums[0][tile][l];
#pragma unroll
    for (int q = 1; q < KW; ++q)
      sum += sums[q][tile][l];
    const int m = m0 + 16 * (tile % MT) + (l & 15), n = n0 + 16 * (tile / MT) + 4 * (l >> 4);
    const float v[4] = {sum[0], sum[1], sum[2], sum[3]};
    if (m < p.m)
      finish4(p, m, n, v);
  }
}

template <int ABITS> hipError_t launch(const GemmArgs &p, hipStream_t s) {
  auto go = [&](auto kernel, int mt, int ft, int kw) {
    const int64_t x = (int64_t(p.n) + 16 * ft - 1) / (16 * ft), y = (int64_t(p.m) + 16 * mt - 1) / (16 * mt);
    if (x * kw * 64 >= int64_t(1) << 32 || y > 65535)
      return hipErrorInvalidValue;
    hipLaunchKernelGGL(kernel, dim3(unsigned(x), unsigned(y)), dim3(unsigned(kw * 64)), 0, s, p);
    return hipGetLastError();
  };
  if (p.m <= 16)
    return go(rows_kernel<ABITS, 1, 1, 4>, 1, 1, 4);
  return go(rows_kernel<ABITS, 4, 4, 4>, 4, 4, 4);
}

}  // namespace
}  // namespace mx
}  // namespace yuear

extern "C" int32_t yuear_op_mx_gemm(const uint8_t *a, int64_t a_stride, const uint8_t *a_scales,
                                    int64_t a_scales_stride, int32_t a_bits, const uint8_t *w,
                                    int64_t w_stride, const uint8_t *w_scales,
                                    int64_t w_scales_stride, int32_t m, int32_t n, int32_t k,
                                    const uint16_t *residual, int64_t residual_stride, uint16_t *c,
                                    int64_t ldc, int32_t swiglu, void *stream) {
  using namespace yuear;
  if (m == 0 || n == 0)
    return 0;
  if (m < 0 || n < 0 || k % mx::kStep || (swiglu != 0 && swiglu != 1) || (swiglu && (n % 2 || residual)) ||
      !mx::rows_ok(a, a_stride, a_scales, a_scales_stride, k, a_bits) ||
      !mx::rows_ok(w, w_stride, w_scales, w_scales_stride, k, 4) || !mx::aligned(a_scales, 4) ||
      !mx::aligned(w_scales, 4) || a_scales_stride % 4 || w_scales_stride % 4 || !mx::aligned(c, 2))
    return int32_t(hipErrorInvalidValue);
  const int width = swiglu ? n / 2 : n;
  constexpr int64_t kMostLd = int64_t(1) << 31;
  if (ldc < width || ldc >= kMostLd ||
      (residual && (!mx::aligned(residual, 2) || residual_stride < width || residual_stride >= kMostLd)))
    return int32_t(hipErrorInvalidValue);
  const mx::Span out = mx::bf16_span(c, ldc, m, width);
  for (const mx::Span &in : {mx::codes_span(a, a_stride, m, k, a_bits), mx::scales_span(a_scales, a_scales_stride, m, k),
                             mx::codes_span(w, w_stride, n, k, 4), mx::scales_span(w_scales, w_scales_stride, n, k)})
    if (mx::overlap(in, out))
      return int32_t(hipErrorInvalidValue);
  // the output may replace the residual: a lane reads its values before it writes them
  if (residual && !(residual == c && residual_stride == ldc) &&
      mx::overlap(mx::bf16_span(residual, residual_stride, m, width), out))
    return int32_t(hipErrorInvalidValue);
  const mx::GemmArgs p{a,      a_scales, w, w_scales, a_stride, a_scales_stride, w_stride, w_scales_stride, m, n, k,
                       residual, c, residual_stride, ldc,
                       swiglu ? mx::kSwiglu : residual ? mx::kResidual : mx::kStore};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return int32_t(a_bits == 8 ? mx::launch<8>(p, st) : mx::launch<4>(p, st));
}
