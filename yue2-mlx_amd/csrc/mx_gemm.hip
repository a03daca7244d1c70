// C[m][n] = bf16(epilogue(sum_k A[m][k] W[n][k])) of rows with a scale per 32
// values (mx.h): activations in 8 or 4 bits, weights in 4, on gfx950's scaled
// MFMA, 128 of K at a time with sums in fp32.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kernels.h"
#include "mx.h"

namespace yuear {
namespace mx {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

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

// Outputs and residuals lie at any even address: the hardware takes loads and stores of 4 to 16
// bytes there, and the type tells the compiler that this is one.
template <class T> struct __attribute__((packed, aligned(2))) AtHalves { T v; };
template <class T> __device__ __forceinline__ T load_at(const uint16_t *p) {
  return reinterpret_cast<const AtHalves<T> *>(p)->v;
}
template <class T> __device__ __forceinline__ void store_at(uint16_t *p, T v) {
  reinterpret_cast<AtHalves<T> *>(p)->v = v;
}

constexpr int kStep = 128;           // K of an MFMA
constexpr int kMaxRows = 1 << 30;    // tokens, features

// Range of a tile's `rows` rows (at most 256) from `base`, of which the last ends
// with its data: what lies past it reads as zero.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const uint8_t *base, int64_t stride,
                                                            int rows, int bytes) {
  const int64_t n = (rows - 1) * stride + bytes;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, int(n), 0x00020000);
}

// silu(gate) * up with e^-gate as 2^t. Rounding t = -gate log2 e moves the result by up to
// |gate| 7.3e-8 of it, no more than half a step of gate, a 32-bit sum, does (|gate| 6e-8). A
// quarter of the quotient's parts: 1 / (1 + e^-gate) itself would be subnormal, which the
// reciprocal takes for zero, from gate = -87.3 on, where the result need not be. Eight operations a
// value and half a one for far gates, two of them of quarter rate: with expf and a division they were a third of the SwiGLU
// tiles' time past the last product.
__device__ __forceinline__ float silu_times(float gate, float up) {
  const float r = __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_exp2f(gate * -1.44269502f), 0.25f, 0.25f));
  return gate * 0.25f * r * up;
}
// The same below kFarGate, where e^-gate goes out of 32 bits (at -88.7) while a large up brings the
// result back: 1 / (1 + e^-gate) is e^gate there, to 2^-125 of it, and the cube of a third of it
// is multiplied in one by one, so that nothing is lost that the result has.
constexpr float kFarGate = -87.f;
__device__ __forceinline__ float far_silu_times(float gate, float up) {
  const float third = __builtin_amdgcn_exp2f(gate * 0.480898347f);
  return gate * third * up * third * third;
}
// N values of interleaved gates and ups. (Negative numbers compare by their bits the other way.)
template <int N> __device__ __forceinline__ void swiglu(const float (&v)[2 * N], float (&y)[N]) {
  uint32_t far = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    y[i] = silu_times(v[2 * i], v[2 * i + 1]);
    far = max(far, f32_bits(v[2 * i]));
  }
  if (__builtin_expect(far > f32_bits(kFarGate), 0))
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (v[2 * i] < kFarGate)
        y[i] = far_silu_times(v[2 * i], v[2 * i + 1]);
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
}

// A lane's features n .. n + 3 (n a multiple of 4) of token row m < p.m.
template <int EPI>
__device__ __forceinline__ void finish4(const GemmArgs &p, int m, int n, const float (&v)[4]) {
  const bool whole = n + 4 <= p.n;
  if (EPI == kSwiglu) {
    uint16_t *c = p.c + m * p.ldc + (n >> 1);
    float y[2];
    swiglu<2>(v, y);
    const uint32_t out = pack2(y[0], y[1]);
    if (whole)
      store_at(c, out);
    else if (n < p.n)
      c[0] = uint16_t(out);
    return;
  }
  uint16_t *c = p.c + m * p.ldc + n;
  const uint16_t *r = p.residual + m * p.residual_stride + n;
  if (whole) {
    float x[4] = {v[0], v[1], v[2], v[3]};
    if (EPI == kResidual) {
      const u32x2 add = load_at<u32x2>(r);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        x[2 * e] += bflo(add[e]);
        x[2 * e + 1] += bfhi(add[e]);
      }
    }
    store_at(c, u32x2{pack2(x[0], x[1]), pack2(x[2], x[3])});
    return;
  }
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (n + e < p.n)
      c[e] = f2bf(EPI == kResidual ? bf2f(r[e]) + v[e] : v[e]);
}

// What finish32() adds, read ahead of it.
__device__ __forceinline__ void residual32(const GemmArgs &p, int m, int n, int h,
                                           u32x4 (&residual)[2]) {
  if (n + 32 > p.n || m >= p.m)
    return;
  const uint16_t *r = p.residual + m * p.residual_stride + n + 16 * h;
  residual[0] = load_at<u32x4>(r);
  residual[1] = load_at<u32x4>(r + 8);
}

// A 32 x 32 MFMA tile, lane 32 h + r with features n + 8 q + 4 h + [0, 4) of token m
// at v[4 q ..]. Where all features exist the lanes of a token trade halves first, so
// that each stores 16 bytes: h = 0 the features (SwiGLU outputs) below 16 (8), h = 1
// the others.
template <int EPI>
__device__ __forceinline__ void finish32(const GemmArgs &p, int m, int n, int h,
                                         const float (&v)[16], const u32x4 (&residual)[2]) {
  if (n + 32 > p.n) {
    if (m < p.m)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float f[4] = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
        finish4<EPI>(p, m, n + 8 * q + 4 * h, f);
      }
    return;
  }
  if (EPI == kSwiglu) {
    float y[8];
    swiglu<8>(v, y);
    uint32_t w[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      w[q] = pack2(y[2 * q], y[2 * q + 1]);
    permlane32_swap(w[0], w[2]);
    permlane32_swap(w[1], w[3]);
    if (m < p.m)
      store_at(p.c + m * p.ldc + (n >> 1) + 8 * h, u32x4{w[0], w[2], w[1], w[3]});
    return;
  }
  uint32_t f[16];
#pragma unroll
  for (int e = 0; e < 16; ++e)
    f[e] = f32_bits(v[e]);
#pragma unroll
  for (int e = 0; e < 8; ++e)  // q 0 with q 2, q 1 with q 3: features 8 q + e and 8 q + 4 + e of one lane
    permlane32_swap(f[e], f[8 + e]);
  if (m >= p.m)
    return;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int at = n + 16 * h + 8 * q;
    float x[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = bits_f32(f[4 * q + e]);
      x[4 + e] = bits_f32(f[8 + 4 * q + e]);
    }
    if (EPI == kResidual) {
      const u32x4 r = residual[q];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] += bflo(r[e]);
        x[2 * e + 1] += bfhi(r[e]);
      }
    }
    store_at(p.c + m * p.ldc + at,
             u32x4{pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7])});
  }
}

// ---- few token rows ----
//
// A workgroup computes 16 FT features of up to 16 MT tokens, its waves 512 of K each
// (and the next 512 that no wave has, where K is longer), then adds the waves' sums in
// order. A wave brings its rows into an LDS region of its own by direct-to-LDS loads,
// 1 KiB of whole 256- or 512-byte row pieces an instruction, and reads them back as
// MFMA operands: no barrier before the sums. (Operands loaded straight into registers
// have neighbouring lanes in different rows: some 55 cycles a load instead of 16, and
// 137 MB of weights in 35 to 45 us instead of 29.) Bound by a launch and one or two
// trips to memory (here to the last-level cache): 1 x 5120 x 3072 3.8 us, 8 x 16384 x 3072 (27 MB) 7.7 to 8.2, 24 x 5120 x 3072 by
// 32 x 32 4.7, 64 x 5120 x 3072 8.2.
//
// 16 x 16 x 128 MFMAs, lane l = 16 g + r: row r; W and 4-bit A k 32 g .. 32 g + 31 of the
// 128, 8-bit A k 16 g .. 16 g + 15 and 64 + 16 g ..; the scale of k-block g. D: features
// 4 g .. 4 g + 3 of token r. Rows of A past m are not loaded: what the region holds there
// reaches only their own, unwritten, tokens.
//
// The 16-byte chunk c of a row is at slot c ^ (row & 15) within 256 bytes: the 16 rows
// that a ds_read_b128 serves at a time, with one chunk of two neighbours, lie in 16
// different slots.
typedef __attribute__((address_space(3))) void *lds_ptr_t;

// The kernels' only LDS object, so that the compiler tells the loads into one
// place from the reads of another.
extern __shared__ __attribute__((aligned(1024))) char mx_lds[];

constexpr int kSliceK = 512;
constexpr int kNonTemporal = 2;  // of a load: what it brings goes from the caches first
// Bytes of a wave's region: pieces of W and A, then their scales.
template <int ABITS, int FT> constexpr int region(int a_rows) {
  return 16 * FT * (kSliceK / 2 + 16) + a_rows * (kSliceK * ABITS / 8 + 16);
}

constexpr int kWPiece = kSliceK / 2;
template <int ABITS> constexpr int a_piece() { return kSliceK * ABITS / 8; }

// 512 of K from k0 on of 16 FT rows of W and of A's rows, with their scales, into LDS at the
// places given. (What lies past K in a piece belongs to other rows, and is not used.)
template <int FT, bool ONCE = false>
__device__ __forceinline__ void load_w(const GemmArgs &p, __amdgpu_buffer_rsrc_t rw,
                                       __amdgpu_buffer_rsrc_t rsw, char *w, char *scales, int k0) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < 4 * FT; ++i) {
    const int row = 4 * i + (lane >> 4);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        rw, (lds_ptr_t)(w + i * 1024), 16,
        row * int(p.w_stride) + k0 / 2 + ((lane & 15) ^ (row & 15)) * 16, 0, 0, ONCE ? kNonTemporal : 0);
  }
  if (lane < 16 * FT)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsw, (lds_ptr_t)scales, 16,
                                             lane * int(p.w_scale_stride) + k0 / 32, 0, 0, 0);
}
template <int ABITS>
__device__ __forceinline__ void load_a(const GemmArgs &p, __amdgpu_buffer_rsrc_t ra,
                                       __amdgpu_buffer_rsrc_t rsa, char *a, char *scales, int k0,
                                       int a_rows) {
  constexpr int kSlots = a_piece<ABITS>() / 16;
  const int lane = threadIdx.x & 63;
  for (int i = 0; i < a_rows * a_piece<ABITS>() / 1024; ++i) {
    const int row = 64 / kSlots * i + lane / kSlots, slot = lane % kSlots;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        ra, (lds_ptr_t)(a + i * 1024), 16,
        row * int(p.a_stride) + k0 * ABITS / 8 + (slot ^ (row & 15)) * 16, 0, 0, 0);
  }
  if (lane < a_rows)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsa, (lds_ptr_t)scales, 16,
                                             lane * int(p.a_scale_stride) + k0 / 32, 0, 0, 0);
}

// acc += W A^T over the 512 of K from k0 on that those loads brought.
template <int ABITS, int MT, int FT>
__device__ __forceinline__ void multiply_slice(const GemmArgs &p, const char *w_at,
                                               const char *w_scales, const char *a_at,
                                               const char *a_scales, int k0, int a_rows,
                                               f32x4 (&acc)[FT][MT]) {
  constexpr int AQ = ABITS / 4;  // 16-byte pieces of A of a lane and MFMA
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  u32x4 ws[FT], as[MT];
#pragma unroll
  for (int f = 0; f < FT; ++f)
    ws[f] = *reinterpret_cast<const u32x4 *>(w_scales + (16 * f + r) * 16);
#pragma unroll
  for (int t = 0; t < MT; ++t)
    as[t] = *reinterpret_cast<const u32x4 *>(a_scales + min(16 * t + r, a_rows - 1) * 16);
#pragma unroll
  for (int s = 0; s < kSliceK / kStep; ++s) {
    if (k0 + s * kStep >= p.k)
      break;
    u32x4 w[FT], a[MT][AQ];
#pragma unroll
    for (int f = 0; f < FT; ++f)
      w[f] = *reinterpret_cast<const u32x4 *>(w_at + (16 * f + r) * kWPiece + ((4 * s + g) ^ r) * 16);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int q = 0; q < AQ; ++q)
        a[t][q] = *reinterpret_cast<const u32x4 *>(
            a_at + min(16 * t + r, a_rows - 1) * a_piece<ABITS>() +
            ((ABITS == 8 ? 8 * s + 4 * q + g : 4 * s + g) ^ r) * 16);
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const u32x4 lo = a[t][0], hi = a[t][AQ - 1];
        const i32x8 wv = {int(w[f].x), int(w[f].y), int(w[f].z), int(w[f].w), 0, 0, 0, 0};
        const i32x8 av = {int(lo.x), int(lo.y), int(lo.z), int(lo.w),
                          int(hi.x), int(hi.y), int(hi.z), int(hi.w)};
        acc[f][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            wv, av, acc[f][t], 4, ABITS == 8 ? 0 : 4, 0, int(ws[f][s] >> (8 * g)), 0,
            int(as[t][s] >> (8 * g)));
      }
  }
}

// Sums of all waves at `sums` (a wave's `stride` bytes apart) to memory.
template <int EPI, int MT, int FT>
__device__ __forceinline__ void add_and_finish(const GemmArgs &p, const char *sums, int stride,
                                               int m0, int n0) {
  const int waves = int(blockDim.x) >> 6;
  for (int i = threadIdx.x; i < FT * MT * 64; i += int(blockDim.x)) {
    const int tile = i >> 6, l = i & 63;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int q = 0; q < waves; ++q)
      sum += *reinterpret_cast<const f32x4 *>(sums + q * stride + i * 16);
    const int m = m0 + 16 * (tile % MT) + (l & 15), n = n0 + 16 * (tile / MT) + 4 * (l >> 4);
    const float v[4] = {sum[0], sum[1], sum[2], sum[3]};
    if (m < p.m)
      finish4<EPI>(p, m, n, v);
  }
}

// s_waitcnt for all but the last `loads` vector memory operations.
template <int LOADS> __device__ __forceinline__ void wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((LOADS & 15) | (LOADS >> 4) << 14 | 0x0f70);
  asm volatile("" ::: "memory");
}

template <int ABITS, int EPI, int MT, int FT>
__global__ __launch_bounds__(1024) void rows_kernel(GemmArgs p, int a_rows) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = int(blockDim.x) >> 6;
  const int n0 = int(blockIdx.x) * (16 * FT), m0 = int(blockIdx.y) * (16 * MT);
  const int rows_a = min(p.m - m0, a_rows), rows_w = min(p.n - n0, 16 * FT);
  const auto ra = rows_rsrc(p.a + m0 * p.a_stride, p.a_stride, rows_a, p.k * ABITS / 8);
  const auto rw = rows_rsrc(p.w + n0 * p.w_stride, p.w_stride, rows_w, p.k / 2);
  const auto rsa = rows_rsrc(p.a_scales + m0 * p.a_scale_stride, p.a_scale_stride, rows_a, p.k / 32);
  const auto rsw = rows_rsrc(p.w_scales + n0 * p.w_scale_stride, p.w_scale_stride, rows_w, p.k / 32);
  char *const w = mx_lds + wave * region<ABITS, FT>(a_rows), *const a = w + 16 * FT * kWPiece;
  char *const w_scales = a + a_rows * a_piece<ABITS>(), *const a_scales = w_scales + 16 * FT * 16;

  f32x4 acc[FT][MT];
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t)
      acc[f][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int k0 = wave * kSliceK; k0 < p.k; k0 += waves * kSliceK) {
    load_w<FT>(p, rw, rsw, w, w_scales, k0);
    load_a<ABITS>(p, ra, rsa, a, a_scales, k0, a_rows);
    wait_loads<0>();  // the wave's own: nobody else reads them
    multiply_slice<ABITS, MT, FT>(p, w, w_scales, a, a_scales, k0, a_rows, acc);
    __builtin_amdgcn_s_waitcnt(0xc07f);  // every read, before the next loads
    asm volatile("" ::: "memory");
  }
  f32x4 *const sums = reinterpret_cast<f32x4 *>(w);  // the region's pieces are used up
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t)
      sums[(f * MT + t) * 64 + lane] = acc[f][t];
  __syncthreads();
  add_and_finish<EPI, MT, FT>(p, mx_lds, region<ABITS, FT>(a_rows), m0, n0);
}

// The same for weights of many features, k up to 512 a wave: a workgroup keeps A and goes
// from one 16 FT features to another, the next ones' weights on their way under the products
// and sums of these. (A workgroup for each 16 or 32 features spends half of its time on its
// start and end. 5 x 83968 x 3072 in 8 bits, weights from HBM: 30.5 and 29.3 us, this 26.7;
// 8 x 16384 x 3072: 8.2, 7.7, this 7.4.)
//
// ONCE: weights of more than 64 MiB, which the last-level cache (256 MB) does not keep until
// the next token's turn, are loaded past it: 5 x 83968 x 3072 26.7 -> 24.5 us (5.6 TB/s), 5 x
// 200000 x 3072 57 -> 52; kept in the cache by calls of them alone 22.2 -> 23.6. 61 MB 12.9
// either way, 25 MB from the cache 5.1 -> 5.4.
template <int ABITS, int FT> constexpr int stream_region(int a_rows) {
  return 2 * (16 * FT * (kWPiece + 16) + FT * 1024) + a_rows * (a_piece<ABITS>() + 16);
}
template <int ABITS, int EPI, int FT, bool ONCE>
__global__ __launch_bounds__(1024) void stream_kernel(GemmArgs p, int a_rows) {
  constexpr int kW = 16 * FT * (kWPiece + 16);  // a buffer's rows and scales
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int k0 = wave * kSliceK, stride = stream_region<ABITS, FT>(a_rows);
  const auto ra = rows_rsrc(p.a, p.a_stride, min(p.m, a_rows), p.k * ABITS / 8);
  const auto rsa = rows_rsrc(p.a_scales, p.a_scale_stride, min(p.m, a_rows), p.k / 32);
  char *const mine = mx_lds + wave * stride;  // two buffers of W, two of sums, A
  char *const a = mine + 2 * (kW + FT * 1024), *const a_scales = a + a_rows * a_piece<ABITS>();
  auto load = [&](int n0, int buffer) {
    const int rows = min(p.n - n0, 16 * FT);
    char *const w = mine + buffer * kW;
    load_w<FT, ONCE>(p, rows_rsrc(p.w + n0 * p.w_stride, p.w_stride, rows, p.k / 2),
                     rows_rsrc(p.w_scales + n0 * p.w_scale_stride, p.w_scale_stride, rows, p.k / 32), w,
                     w + 16 * FT * kWPiece, k0);
  };
  load_a<ABITS>(p, ra, rsa, a, a_scales, k0, a_rows);
  const int tiles = (p.n + 16 * FT - 1) / (16 * FT);
  load(int(blockIdx.x) * (16 * FT), 0);
  int buffer = 0;
  for (int tile = int(blockIdx.x); tile < tiles; tile += int(gridDim.x), buffer ^= 1) {
    const int next = tile + int(gridDim.x);
    if (next < tiles) {
      load(next * (16 * FT), buffer ^ 1);
      wait_loads<4 * FT + 1>();
    } else {
      wait_loads<0>();
    }
    f32x4 acc[FT][1];
#pragma unroll
    for (int f = 0; f < FT; ++f)
      acc[f][0] = f32x4{0.f, 0.f, 0.f, 0.f};
    const char *const w = mine + buffer * kW;
    multiply_slice<ABITS, 1, FT>(p, w, w + 16 * FT * kWPiece, a, a_scales, k0, a_rows, acc);
    f32x4 *const sums = reinterpret_cast<f32x4 *>(mine + 2 * kW + buffer * FT * 1024);
#pragma unroll
    for (int f = 0; f < FT; ++f)
      sums[f * 64 + lane] = acc[f][0];
    // Sums and the weights just read are written again after the next barrier but this one.
    lds_barrier();  // the next weights' loads go on
    add_and_finish<EPI, 1, FT>(p, mx_lds + 2 * kW + buffer * FT * 1024, stride, 0, tile * (16 * FT));
  }
}

// ---- many token rows: tiles through LDS ----
//
// A workgroup of WM x WN waves computes BM x BN tiles of C, each wave BM / WM tokens
// by BN / WN features as 32 x 32 MFMA tiles, 64 of K at a time. K advances by steps
// of KSTEP through a ring of LDS stages that direct-to-LDS loads fill (1 KiB an
// instruction). The operands of the next 64 of K are read from LDS under the MFMAs
// of these. One barrier a step, before its last 64: past it every wave has read all
// of the stage, which takes the step that the ring has room for, and the next step's
// loads have landed.
//
// There is a workgroup for each CU, which takes one tile after another, and the ring
// does not stop between them: the last steps of a tile load the first ones of the
// next, whose products go on while this one's results are on their way to memory.
//
// Scales come 512 of K (a group) at a time, 16 bytes a row, into two buffers behind
// the ring, a group in use and the one after it; a lane reads the bytes of its row
// and step and shifts them so that k-block h of each 64 is at byte 0 or 2.
//
// us of stores, operands from
// the last-level cache:         64x64  64x128  128x128  192x192  256x256
//   8 bits, 100 x 5120 x 3072      8.5    10.5     13.2
//   8 bits, 300 x 5120 x 3072     15.8    11.6     14.1     24.5
//   8 bits, 1000 x 5120 x 3072    36.6    29.1     25.5     26.0     33.7
//   8 bits, 3000 x 3072 x 8192             109     86.8     64.7     74.5
//   8 bits, 3000 x 16384 x 3072            207      149      141      117
//   4 bits, 6001 x 12288 x 2048            165      124      104       95
// The largest run at 2.6 PFLOP/s (8 bits, 2.9 at K 8192) and 3.4 (4 bits, 4.2): matrix
// cores busy 62 and 37% of the cycles at the 2.0 GHz that the power limit leaves (operands of
// zeros run 27-30% faster), in 4 bits SwiGLU a sixth of the time (K 2048).
// The smallest are bound by LDS: 64 x 64 tiles of 197 x 3072 x 8192 bring 768 KiB a CU at 70
// KB/us of the 66 (rows of 64 bytes) to 120 (128) that loads into LDS reach, 15.6 us.
//
// MFMA operands, lane l = 32 h + r: in 4 bits row r, k 32 h .. 32 h + 31 of the 64;
// in 8 bits k 16 h .. 16 h + 15 and 32 + 16 h ..; the scale of k-block h of row r.
// D: features 8 q + 4 h + [0, 4) of token r.
//
// LDS rows of 128 bytes keep their 16-byte chunk c at slot c ^ (row >> 1 & 7), rows
// of 64 bytes at c ^ (bit 2 of the row | bit 4 << 1). A ds_read_b128 is served 16
// lanes at a time (bit 5 of the lane, and bit 3 ^ bit 4): rows 0-7 and 24-31, or
// 8-23, with one chunk, which either layout spreads over all 16 slots of 256 bytes.
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kGroupK = 512;  // K of a group of scales

template <int ABITS, int BM, int BN, int WM, int WN, int KS, int KSTEP, int STAGES> struct Tile {
  static constexpr int kTeam = WM * WN, kWaves = kTeam * KS, kBM = BM, kBN = BN;
  static constexpr int kARow = KSTEP * ABITS / 8, kWRow = KSTEP / 2;  // bytes of a row a step
  static constexpr int kStage = BM * kARow + BN * kWRow;
  static constexpr int kScales = (BM + BN) * 16;
  static constexpr int kStages = STAGES;
  static constexpr int kRing = kStages * kStage + 2 * kScales;  // of a team
  static constexpr int kLds = KS * kRing;
  static constexpr bool kOnward = KS == 1 && STAGES <= 3;  // takes one tile after another
  static_assert(kLds <= 160 * 1024, "LDS");
};

// Tiles of workgroup b of `grid` (a multiple of 8): the n-th, counted from 0. Workgroups
// go to the 8 XCDs in turn, each with its own L2: XCD x takes one contiguous range of
// an order in columns of four tile rows, so that the tiles that share an L2 form a
// compact block of A and W rows.
__device__ __forceinline__ bool tile_of(int b, int grid, int n, int tiles_m, int tiles_n, int &tm,
                                        int &tn) {
  constexpr int kXcds = 8, kGroup = 4;
  const int total = tiles_m * tiles_n, each = total / kXcds, more = total % kXcds;
  const int x = b % kXcds, at = b / kXcds + n * (grid / kXcds);
  if (at >= each + (x < more))
    return false;
  const int t = x * each + min(x, more) + at;
  const int per = kGroup * tiles_n, first = t / per * kGroup;
  const int rows = min(tiles_m - first, kGroup), r = t % per;
  tm = first + r % rows;
  tn = r / rows;
  return true;
}

__device__ __forceinline__ int slot_of(int bytes, int row, int chunk) {
  return bytes == 128 ? chunk ^ ((row >> 1) & 7) : chunk ^ (((row >> 2) & 1) | ((row >> 3) & 2));
}

// s_waitcnt for all but the last `loads` vector memory operations, and every LDS read.
constexpr int waitcnt(int loads) { return (loads & 15) | (loads >> 4) << 14 | 0x0070; }
// The workgroup's barrier, after the wave's LDS reads and, from step FROM on, all but the last
// LOADS of its vector memory operations. (__syncthreads() would wait for every load into LDS,
// those of the steps ahead too. The branch is in the assembly so that a step stays one block for
// the scheduler.)
template <int LOADS, int FROM, bool MEET> __device__ __forceinline__ void wait_and_meet(int step) {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_cmp_lt_i32 %0, %2\n\t"
               "s_cbranch_scc1 .Lmeet%=\n\t"
               "s_waitcnt vmcnt(%1)\n"
               ".Lmeet%=:" ::"s"(__builtin_amdgcn_readfirstlane(step)), "n"(LOADS), "n"(FROM)
               : "scc", "memory");
  __builtin_amdgcn_s_waitcnt(waitcnt(63));
  if constexpr (MEET)
    __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// What a wave loads of a tile: its rows of A, of W, and its blocks of scales.
template <int SPW> struct Source {
  const uint8_t *a, *w, *s[SPW];
  int a_bytes, w_bytes, s_bytes[SPW];  // past which nothing is read
};
__device__ __forceinline__ int range(int64_t stride, int rows, int bytes) {
  return int((rows - 1) * stride + bytes);
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const uint8_t *base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, bytes, 0x00020000);
}

// With k up to 512 (fewer than two groups of scales) loads could reach past the next
// tile: the launch gives each workgroup one tile then, and they read nothing.
//
// KS > 1: one wave has the whole tile, and KS of them a part of K and a ring each, with
// no barrier before their sums are added.
template <int ABITS, int EPI, int BM, int BN, int WM, int WN, int KS, int KSTEP, int STAGES>
__device__ __forceinline__ void tile(const GemmArgs &p) {
  using T = Tile<ABITS, BM, BN, WM, WN, KS, KSTEP, STAGES>;
  constexpr int TM = BM / WM / 32, TN = BN / WN / 32, PARTS = KSTEP / 64;
  constexpr int kGroupSteps = kGroupK / KSTEP;
  constexpr int AQ = ABITS / 4;  // 16-byte pieces of A of a lane and 64 of K
  constexpr int APW = BM * T::kARow / 1024 / T::kTeam, WPW = BN * T::kWRow / 1024 / T::kTeam;
  constexpr int SB = (BM + BN) / 64, SPW = (SB + T::kTeam - 1) / T::kTeam;  // blocks of scales
  // A group of scales is asked for at the end of the group before the last one, so kGroupSteps
  // steps ahead, and waited for with the loads of STAGES - 2 steps later.
  static_assert(APW * T::kTeam * 1024 == BM * T::kARow && WPW * T::kTeam * 1024 == BN * T::kWRow &&
                    TM * 32 * WM == BM && TN * 32 * WN == BN && BM % 64 == 0 && BN % 64 == 0 &&
                    STAGES >= 2 && STAGES - 2 <= kGroupSteps && kGroupSteps >= 2 &&
                    (KS == 1 || (T::kTeam == 1 && TM * TN == KS)),
                "tile");
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave_id = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int team = KS == 1 ? 0 : wave_id / T::kTeam, wave = KS == 1 ? wave_id : wave_id % T::kTeam;
  const int ring = team * T::kRing;
  const int k_begin = p.k / KSTEP * team / KS * KSTEP;  // this team's K
  const int k_len = p.k / KSTEP * (team + 1) / KS * KSTEP - k_begin;
  const int wm = wave / WN, wn = wave % WN;
  const int r = lane & 31, h = lane >> 5;
  const int tiles_m = (p.m + BM - 1) / BM, tiles_n = (p.n + BN - 1) / BN;

  // this wave's KiB blocks of a stage's A and W: lane l fills slot l
  // (the slots repeat after 16 rows, of 64 bytes after 32: blocks that far apart share an offset)
  constexpr int kARows = 1024 / T::kARow, kWRows = 1024 / T::kWRow;  // of a block
  constexpr int AP = APW % 2 ? APW : 2, WP = WPW % 2 ? WPW : 2;
  static_assert(kARows >= 8 && kWRows >= 8, "blocks");
  uint32_t from_a[AP], from_w[WP], from_s[SPW];
#pragma unroll
  for (int i = 0; i < AP; ++i) {
    const int row = kARows * (wave * APW + i) + lane / (64 / kARows);
    from_a[i] = uint32_t(row * int(p.a_stride) + slot_of(T::kARow, row, lane % (64 / kARows)) * 16);
  }
#pragma unroll
  for (int i = 0; i < WP; ++i) {
    const int row = kWRows * (wave * WPW + i) + lane / (64 / kWRows);
    from_w[i] = uint32_t(row * int(p.w_stride) + slot_of(T::kWRow, row, lane % (64 / kWRows)) * 16);
  }
  // 64 rows of scales a block, A's first; waves past the last block repeat it
  auto block = [&](int i) { return min(wave + i * T::kTeam, SB - 1); };
#pragma unroll
  for (int i = 0; i < SPW; ++i) {
    const bool is_a = block(i) < BM / 64;
    from_s[i] = uint32_t((64 * (is_a ? block(i) : block(i) - BM / 64) + lane) *
                         int(is_a ? p.a_scale_stride : p.w_scale_stride));
  }
  auto source = [&](int m0, int n0) {
    const int rows_a = min(p.m - m0, BM), rows_w = min(p.n - n0, BN);
    Source<SPW> s;
    s.a = p.a + m0 * p.a_stride + k_begin * ABITS / 8;
    s.w = p.w + n0 * p.w_stride + k_begin / 2;
    s.a_bytes = range(p.a_stride, rows_a, (p.k - k_begin) * ABITS / 8);
    s.w_bytes = range(p.w_stride, rows_w, (p.k - k_begin) / 2);
#pragma unroll
    for (int i = 0; i < SPW; ++i) {
      const bool is_a = block(i) < BM / 64;
      s.s[i] = (is_a ? p.a_scales + m0 * p.a_scale_stride : p.w_scales + n0 * p.w_scale_stride) +
               k_begin / 32;
      s.s_bytes[i] = is_a ? range(p.a_scale_stride, rows_a, (p.k - k_begin) / 32)
                          : range(p.w_scale_stride, rows_w, (p.k - k_begin) / 32);
    }
    return s;
  };

  int tm, tn;
  if (!tile_of(int(blockIdx.x), int(gridDim.x), 0, tiles_m, tiles_n, tm, tn))
    return;
  int m0 = tm * BM, n0 = tn * BN;
  Source<SPW> now = source(m0, n0), then = now;

  const int steps = k_len / KSTEP, groups = (k_len + kGroupK - 1) / kGroupK;
  // step `step` of this tile, or step - steps of the next, into the stage that begins at `stage`
  auto load = [&](int stage, int step) {
    const bool here = step < steps;
    const int at = here ? step : step - steps;
    const auto ra = rsrc(here ? now.a : then.a, here ? now.a_bytes : then.a_bytes);
    const auto rw = rsrc(here ? now.w : then.w, here ? now.w_bytes : then.w_bytes);
#pragma unroll
    for (int i = 0; i < APW; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          ra, (lds_ptr_t)(mx_lds + stage + (wave * APW + i) * 1024), 16,
          from_a[i % AP] + (at * T::kARow + i / AP * AP * kARows * int(p.a_stride)), 0, 0, 0);
#pragma unroll
    for (int i = 0; i < WPW; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rw, (lds_ptr_t)(mx_lds + stage + BM * T::kARow + (wave * WPW + i) * 1024), 16,
          from_w[i % WP] + (at * T::kWRow + i / WP * WP * kWRows * int(p.w_stride)), 0, 0, 0);
  };
  const int scales_at = ring + T::kStages * T::kStage;
  int odd = 0;  // the buffer of this tile's first group
  auto load_scales = [&](int group) {
    const bool here = group < groups;
    const int at = here ? group : group - groups;
#pragma unroll
    for (int i = 0; i < SPW; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc(here ? now.s[i] : then.s[i], here ? now.s_bytes[i] : then.s_bytes[i]),
          (lds_ptr_t)(mx_lds + scales_at + ((group + odd) & 1) * T::kScales + block(i) * 1024), 16,
          from_s[i] + at * 16, 0, 0, 0);
  };

  const int a_row = wm * (BM / WM) + r, w_row = wn * (BN / WN) + r;  // of the first MFMA tiles
  f32x16 acc[TM][TN];
  u32x4 af[2][TM][AQ], wf[2][TN];
  constexpr int SW = PARTS / 2;  // 4-byte words of a row's scales a step
  int as[SW][TM], ws[SW][TN], as_next[SW][TM], ws_next[SW][TN];
  // operands of part s of a step from its stage
  auto read = [&](int stage, int s) {
    const char *a = mx_lds + stage + a_row * T::kARow;
    const char *w = mx_lds + stage + BM * T::kARow + w_row * T::kWRow;
#pragma unroll
    for (int x = 0; x < (TM > TN ? TM : TN); ++x) {
      if (x < TN)
        wf[s & 1][x] = *reinterpret_cast<const u32x4 *>(w + x * 32 * T::kWRow +
                                                        slot_of(T::kWRow, r, 2 * s + h) * 16);
      if (x < TM)
#pragma unroll
        for (int q = 0; q < AQ; ++q)
          af[s & 1][x][q] = *reinterpret_cast<const u32x4 *>(
              a + x * 32 * T::kARow +
              slot_of(T::kARow, r, (ABITS == 8 ? 4 * s + 2 * q : 2 * s) + h) * 16);
    }
  };
  // scales of step `at` of the group in buffer `buffer`
  auto read_scales = [&](int buffer, int at) {
    const char *sc = mx_lds + scales_at + buffer * T::kScales + at * (KSTEP / 32);
#pragma unroll
    for (int x = 0; x < TN; ++x)
#pragma unroll
      for (int e = 0; e < SW; ++e)
        ws_next[e][x] = *reinterpret_cast<const int *>(sc + (BM + w_row + 32 * x) * 16 + 4 * e);
#pragma unroll
    for (int x = 0; x < TM; ++x)
#pragma unroll
      for (int e = 0; e < SW; ++e)
        as_next[e][x] = *reinterpret_cast<const int *>(sc + (a_row + 32 * x) * 16 + 4 * e);
  };
  auto take_scales = [&] {
#pragma unroll
    for (int e = 0; e < SW; ++e) {
#pragma unroll
      for (int x = 0; x < TN; ++x)
        ws[e][x] = int(uint32_t(ws_next[e][x]) >> (8 * h));
#pragma unroll
      for (int x = 0; x < TM; ++x)
        as[e][x] = int(uint32_t(as_next[e][x]) >> (8 * h));
    }
  };
  auto multiply = [&](auto part) {
    constexpr int s = decltype(part)::value, e = s / 2, byte = 2 * (s & 1);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const u32x4 w = wf[s & 1][j], lo = af[s & 1][i][0], hi = af[s & 1][i][AQ - 1];
        const i32x8 wv = {int(w.x), int(w.y), int(w.z), int(w.w), 0, 0, 0, 0};
        const i32x8 av = {int(lo.x), int(lo.y), int(lo.z), int(lo.w),
                          int(hi.x), int(hi.y), int(hi.z), int(hi.w)};
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
            wv, av, acc[i][j], 4, ABITS == 8 ? 0 : 4, byte, ws[e][j], byte, as[e][i]);
      }
  };

  // A step, with the next one's stage at `next` and scales at (buffer, at). Past its barrier the
  // ring takes step + STAGES, and, where the step ends a group, that group's buffer the group
  // after the next. Reads and loads go between the MFMAs.
  constexpr int kReads = TN + TM * AQ, kScaleReads = SW * (TM + TN), kMfmas = TM * TN,
                kLoads = APW + WPW, kHalf = (kMfmas + 1) / 2;
  int ahead = STAGES;  // the first tile's loads are in order from its first step on
  auto advance = [&](auto ends, int stage, int next, int step, int buffer, int at, int group) {
    auto part = [&](auto s) {
      read(stage, s + 1);
      multiply(s);
#pragma unroll
      for (int x = 0; x < kMfmas; ++x) {
        __builtin_amdgcn_sched_group_barrier(0x100, (kReads + kMfmas - 1) / kMfmas, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    part(std::integral_constant<int, 0>());
    if constexpr (PARTS == 4) {
      part(std::integral_constant<int, 1>());
      part(std::integral_constant<int, 2>());
    }
    // (the first steps of a later tile find theirs waited for before the last one's stores)
    wait_and_meet<(STAGES - 2) * kLoads, STAGES - 1, (T::kTeam > 1)>(step + ahead);
    read(next, 0);
    read_scales(buffer, at);
    if constexpr (decltype(ends)::value)
      load_scales(group + 2);
    load(stage, step + STAGES);
    multiply(std::integral_constant<int, PARTS - 1>());
#pragma unroll
    for (int x = 0; x < kMfmas; ++x) {
      if (x < kHalf)
        __builtin_amdgcn_sched_group_barrier(0x100, (kReads + kScaleReads + kHalf - 1) / kHalf, 0);
      else
        __builtin_amdgcn_sched_group_barrier(0x020, (kLoads + SPW + kHalf - 1) / kHalf, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    take_scales();
  };
  using Ends = std::true_type;
  using Goes = std::false_type;

  load_scales(0);
  load_scales(1);
#pragma unroll
  for (int s = 0; s < STAGES; ++s)
    load(ring + s * T::kStage, s);
  wait_and_meet<(STAGES - 1) * kLoads, 0, (T::kTeam > 1)>(0);
  read(ring, 0);
  read_scales(0, 0);
  take_scales();
  int stage = ring;
  auto after = [&](int at) {
    return at + T::kStage == ring + STAGES * T::kStage ? ring : at + T::kStage;
  };

  for (int turn = 1;; ++turn) {
    const bool more =
        T::kOnward && tile_of(int(blockIdx.x), int(gridDim.x), turn, tiles_m, tiles_n, tm, tn);
    then = source(more ? tm * BM : m0, more ? tn * BN : n0);
    if (!more) {
      then.a_bytes = then.w_bytes = 0;
#pragma unroll
      for (int i = 0; i < SPW; ++i)
        then.s_bytes[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          acc[i][j][e] = 0.f;

    auto one = [&](auto ends, int step, int s, int g) {  // step s of group g
      const int next = after(stage);
      const bool last = s == kGroupSteps - 1 || step == steps - 1;
      advance(ends, stage, next, step, (last ? g + 1 + odd : g + odd) & 1, last ? 0 : s + 1, g);
      stage = next;
    };
    int step = 0, g = 0;
    for (; step + kGroupSteps <= steps; step += kGroupSteps, ++g)
#pragma unroll
      for (int s = 0; s < kGroupSteps; ++s) {
        if (s == kGroupSteps - 1)
          one(Ends(), step + s, s, g);
        else
          one(Goes(), step + s, s, g);
      }
    if (step < steps) {
      int s = 0;
      for (; step + 1 < steps; ++step, ++s)
        one(Goes(), step, s, g);
      one(Ends(), step, s, g);
    }

    // the loads of the next tile's first steps, before this one's stores queue up behind them
    __builtin_amdgcn_s_waitcnt(waitcnt(0) | 0x0f00);
    if constexpr (KS > 1) {  // team t finishes MFMA tile t, from everybody's sums in order
      f32x4 *const sums = reinterpret_cast<f32x4 *>(mx_lds) + lane;
      static_assert(KS * BM * BN * 4 <= T::kLds, "sums");
      __syncthreads();
#pragma unroll
      for (int t = 0; t < KS; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x16 &a = acc[t / TN][t % TN];
          sums[((team * KS + t) * 4 + q) * 64] = f32x4{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
        }
      __syncthreads();
      float v[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x4 sum = sums[(team * 4 + q) * 64];
#pragma unroll
        for (int t = 1; t < KS; ++t)
          sum += sums[((t * KS + team) * 4 + q) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[4 * q + e] = sum[e];
      }
      const int m = m0 + r + team / TN * 32, n = n0 + team % TN * 32;
      u32x4 residual[2];
      if (EPI == kResidual)
        residual32(p, m, n, h, residual);
      finish32<EPI>(p, m, n, h, v, residual);
      return;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int m = m0 + a_row + 32 * i, n = n0 + wn * (BN / WN);
      u32x4 residual[2][2];  // of this tile and the next
      if (EPI == kResidual)
        residual32(p, m, n, h, residual[0]);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        if (EPI == kResidual && j + 1 < TN)
          residual32(p, m, n + 32 * (j + 1), h, residual[(j + 1) & 1]);
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e)
          v[e] = acc[i][j][e];
        finish32<EPI>(p, m, n + 32 * j, h, v, residual[j & 1]);
      }
    }
    if (!more)
      break;
    ahead = 0;
    odd = (odd + groups) & 1;
    m0 = tm * BM;
    n0 = tn * BN;
    now = then;
  }
}

template <int ABITS, int EPI, int BM, int BN, int WM, int WN, int KS, int KSTEP, int STAGES>
__global__ __launch_bounds__(WM * WN * KS * 64, BM * BN > WM * WN * 8192 ? 1 : 2) void tile_kernel(GemmArgs p) {
  tile<ABITS, EPI, BM, BN, WM, WN, KS, KSTEP, STAGES>(p);
}

template <class T>
hipError_t launch_tile(void (*kernel)(GemmArgs), const GemmArgs &p, hipStream_t s) {
  const int64_t tiles = ((int64_t(p.m) + T::kBM - 1) / T::kBM) * ((int64_t(p.n) + T::kBN - 1) / T::kBN);
  const int64_t all = (tiles + 7) / 8 * 8, cus = std::max(gemm_cus() / 8 * 8, 8);
  const int64_t grid = T::kOnward && p.k > kGroupK ? std::min(cus, all) : all;
  // threads of the grid count in 32 bits, tiles in 31 (the largest ones of what memory holds do)
  if (grid * T::kWaves * 64 >= int64_t(1) << 32 || tiles > int64_t(1) << 30)
    return hipErrorInvalidValue;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, T::kLds);
  if (e != hipSuccess)
    return e;
  hipLaunchKernelGGL(kernel, dim3(unsigned(grid)), dim3(T::kWaves * 64), T::kLds, s, p);
  return hipGetLastError();
}

template <int ABITS, int MT, int FT>
hipError_t launch_rows(void (*kernel)(GemmArgs, int), const GemmArgs &p, hipStream_t s) {
  const int64_t x = (int64_t(p.n) + 16 * FT - 1) / (16 * FT), y = (int64_t(p.m) + 16 * MT - 1) / (16 * MT);
  if (x >= int64_t(1) << 22 || y > 65535)  // threads of the grid count in 32 bits
    return hipErrorInvalidValue;
  // whole KiB of A's rows; at least the sums fit a region
  const int per_kib = 1024 / (kSliceK * ABITS / 8), rows = std::min(p.m, 16 * MT);
  const int a_rows = (rows + per_kib - 1) / per_kib * per_kib;
  const int bytes = region<ABITS, FT>(a_rows);
  static_assert(16 * FT * (kSliceK / 2) >= 1024 * FT * MT, "sums");
  const int waves = std::min({(p.k + kSliceK - 1) / kSliceK, 160 * 1024 / bytes, 16});
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
  if (e != hipSuccess)
    return e;
  hipLaunchKernelGGL(kernel, dim3(unsigned(x), unsigned(y)), dim3(unsigned(waves * 64)), waves * bytes, s, p,
                     a_rows);
  return hipGetLastError();
}

// ---- the forms, and which one a call takes ----

enum Form : int {
  kRows16,
  kRows32,
  kRows32x32,
  kTile64,
  kTile64x128,
  kTile128,
  kTile192,
  kTile256,
  kStream16,
  kStream32,
  kForms
};

// k up to 512 a wave, m up to 16.
template <int ABITS, int EPI, int FT> hipError_t launch_stream(const GemmArgs &p, hipStream_t s) {
  const int per_kib = 1024 / (kSliceK * ABITS / 8);
  const int a_rows = (p.m + per_kib - 1) / per_kib * per_kib;
  const int waves = (p.k + kSliceK - 1) / kSliceK, bytes = waves * stream_region<ABITS, FT>(a_rows);
  if (p.m > 16 || waves > 16 || bytes > 160 * 1024)
    return hipErrorInvalidValue;
  void (*const kernel)(GemmArgs, int) = int64_t(p.n) * (p.k / 2) > int64_t(64) << 20
                                            ? stream_kernel<ABITS, EPI, FT, true>
                                            : stream_kernel<ABITS, EPI, FT, false>;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
  if (e != hipSuccess)
    return e;
  const int64_t tiles = (int64_t(p.n) + 16 * FT - 1) / (16 * FT);
  const int per_cu = std::max(1, std::min(160 * 1024 / bytes, 32 / waves));
  hipLaunchKernelGGL(kernel, dim3(unsigned(std::min<int64_t>(tiles, int64_t(gemm_cus()) * per_cu))),
                     dim3(unsigned(waves * 64)), bytes, s, p, a_rows);
  return hipGetLastError();
}

template <int ABITS, int EPI> hipError_t launch_form(int form, const GemmArgs &p, hipStream_t s) {
#define YUEAR_MX_ROWS(MT, FT) launch_rows<ABITS, MT, FT>(rows_kernel<ABITS, EPI, MT, FT>, p, s)
#define YUEAR_MX_TILE(...)                                                                 \
  launch_tile<Tile<ABITS, __VA_ARGS__>>(tile_kernel<ABITS, EPI, __VA_ARGS__>, p, s)
  switch (form) {
  case kRows16: return YUEAR_MX_ROWS(1, 1);
  case kRows32: return YUEAR_MX_ROWS(1, 2);
  case kRows32x32: return YUEAR_MX_ROWS(2, 2);
  case kTile64: return YUEAR_MX_TILE(64, 64, 1, 1, 4, 128, (ABITS == 8 ? 3 : 4));
  case kTile64x128: return YUEAR_MX_TILE(64, 128, 1, 4, 1, 128, 6);
  case kTile128: return YUEAR_MX_TILE(128, 128, 2, 2, 1, 128, 3);
  // 4 bits: rows of 128 bytes (256 of K) a load where K has them; 64 bytes ask L2 as often
  case kTile192:
    if constexpr (ABITS == 4)
      if (p.k % 256 == 0)
        return YUEAR_MX_TILE(192, 192, 2, 2, 1, 256, 3);
    return YUEAR_MX_TILE(192, 192, 2, 2, 1, 128, 3);
  case kTile256:
    if constexpr (ABITS == 4)
      if (p.k % 256 == 0)
        return YUEAR_MX_TILE(256, 256, 4, 2, 1, 256, 2);
    return YUEAR_MX_TILE(256, 256, 4, 2, 1, 128, 3);
  case kStream16: return launch_stream<ABITS, EPI, 1>(p, s);
  case kStream32: return launch_stream<ABITS, EPI, 2>(p, s);
  }
#undef YUEAR_MX_ROWS
#undef YUEAR_MX_TILE
  return hipErrorInvalidValue;
}

template <int ABITS> hipError_t launch(int form, const GemmArgs &p, hipStream_t s) {
  switch (p.epilogue) {
  case kSwiglu: return launch_form<ABITS, kSwiglu>(form, p, s);
  case kResidual: return launch_form<ABITS, kResidual>(form, p, s);
  default: return launch_form<ABITS, kStore>(form, p, s);
  }
}

// Estimated us of m x n x k by a form, infinite where it cannot run; fitted on MI355X to 4400
// shapes of stores in all forms (to 6000 tokens, 84000 features, K 128-8192; 6-13% rms where a form
// is within 1.6 of the fastest). Over 450 other shapes what it picks takes 1.9% more than the
// fastest form for stores and SwiGLU of 8-bit rows, 3.3% with a residual, 1.4 to 2.5% for 4-bit rows.
double form_time(int form, int bits, int m, int n, int k, int cus) {
  const bool a8 = bits == 8;
  const double kk = k / 1024.0;
  auto tiles = [&](int bm, int bn) { return double((m + bm - 1) / bm) * double((n + bn - 1) / bn); };
  if (form <= kRows32x32 || form >= kStream16) {
    const bool stream = form >= kStream16;
    const int bm = form == kRows32x32 ? 32 : 16, bn = form == kRows16 || form == kStream16 ? 16 : 32;
    const int per_kib = a8 ? 2 : 4, rows = (std::min(m, bm) + per_kib - 1) / per_kib * per_kib;
    const int a_bytes = rows * (kSliceK * bits / 8 + 16), w_bytes = bn * (kSliceK / 2 + 16);
    const int slices = (k + kSliceK - 1) / kSliceK;
    const double t = tiles(bm, bn);
    if (!stream) {
      if (n / bn >= (1 << 22) - 1 || m / bm >= 65535)  // past a launch's grid
        return __builtin_inf();
      // the launch, each 512 of K that a wave takes after another, each round of the workgroups
      // that the CUs hold, the bytes of W, each workgroup
      const int waves = std::min({slices, 160 * 1024 / (w_bytes + a_bytes), 16});
      const int held = std::max(1, std::min(160 * 1024 / (waves * (w_bytes + a_bytes)), 32 / waves));
      static const double fit[2][3][5] = {
          {{0.254, 1.274, 1.444, 0.0203, 0.0},
           {0.681, 1.135, 1.365, 0.0189, 0.0},
           {0.541, 1.268, 1.818, 0.0193, 0.0501}},
          {{0.0, 1.708, 1.174, 0.0188, 0.0},
           {0.697, 1.11, 1.303, 0.0182, 0.0},
           {1.274, 1.147, 1.076, 0.0173, 0.0918}}};
      const double *c = fit[a8 ? 0 : 1][form];
      return c[0] + c[1] * ((slices + waves - 1) / waves) + c[2] * std::ceil(t / (double(cus) * held)) +
             t / cus * (c[3] * kk * bn + c[4]);
    }
    // the launch, each 16 or 32 features of a workgroup, the bytes of W and once those of A
    const int bytes = slices * (2 * (w_bytes + bn * 64) + a_bytes);
    if (m > 16 || slices > 16 || bytes > 160 * 1024)
      return __builtin_inf();
    const double grid = std::min(t, double(cus) * std::max(1, std::min(160 * 1024 / bytes, 32 / slices)));
    static const double fit[2][2][5] = {{{1.926, 0.757, 0.0138, 0.002, 0.0997}, {1.626, 1.285, 0.0088, 0.0101, 0.0998}},
                                        {{1.901, 0.741, 0.0142, 0.0, 0.0663}, {1.506, 1.274, 0.0087, 0.0204, 0.0766}}};
    const double *c = fit[a8 ? 0 : 1][form - kStream16];
    return c[0] + c[1] * std::ceil(t / grid) + c[2] * t / cus * kk * bn + c[3] * grid / cus * kk * rows * bits / 8 +
           c[4] * kk;
  }
  // the launch, full rounds of tiles, and a last one by how many CUs it has work for
  static const int shape[5][3] = {{64, 64, 1}, {64, 128, 1}, {128, 128, 2}, {192, 192, 1}, {256, 256, 1}};
  static const double fit[2][5][7] = {{{1.957, 3.111, 1.389, 2.548, 0.748, 0.18, 0.795},
                                       {1.234, 2.978, 2.319, 2.314, 1.868, 0.776, 0.654},
                                       {1.634, 5.877, 6.484, 3.391, 2.459, 0.488, 2.216},
                                       {3.525, 6.613, 6.164, 2.594, 5.338, 5.195, 0.645},
                                       {0.591, 10.876, 9.663, 5.976, 7.548, 8.132, 1.331}},
                                      {{1.35, 2.936, 1.339, 2.938, 0.478, 0.0, 0.971},
                                       {2.87, 1.481, 1.862, 0.528, 1.506, 0.809, 0.599},
                                       {2.423, 4.764, 5.324, 2.061, 2.014, 1.129, 1.981},
                                       {5.728, 5.124, 4.198, 0.0, 3.757, 5.692, 0.15},
                                       {3.142, 8.015, 6.513, 2.969, 4.77, 8.5, 0.893}}};
  const int *of = shape[form - kTile64];
  if (form != kTile256 && tiles(of[0], of[1]) >= (1 << 22))
    return __builtin_inf();
  const double *c = fit[a8 ? 0 : 1][form - kTile64];
  const double slots = double(cus) * of[2], t = tiles(of[0], of[1]);
  double full = std::floor(t / slots), rest = t / slots - full;
  if (of[2] == 2 && rest > 0.5) {  // some CU has both of its tiles again
    full += 1;
    rest = 0;
  }
  return c[0] + full * (c[1] + c[2] * kk) + (rest > 0 ? c[3] + c[4] * kk + rest * (c[5] + c[6] * kk) : 0.0);
}

// The form of least estimated time: for few tokens rows, streamed where a workgroup can keep
// A, the larger tiles the more there are to fill the CUs with. The sum over K is split as the
// form is (by waves, in order), so the form decides the order of the sums.
int pick_form(int bits, int m, int n, int k) {
  const int cus = gemm_cus();
  int best = 0;
  double least = __builtin_inf();
  for (int form = 0; form < kForms; ++form) {
    const double t = form_time(form, bits, m, n, k, cus);
    if (t < least) {
      least = t;
      best = form;
    }
  }
  return best;
}

}  // namespace
}  // namespace mx
}  // namespace yuear

extern "C" {

int32_t yuear_op_mx_gemm_form(const uint8_t *a, int64_t a_stride, const uint8_t *a_scales,
                              int64_t a_scales_stride, int32_t a_bits, const uint8_t *w,
                              int64_t w_stride, const uint8_t *w_scales, int64_t w_scales_stride,
                              int32_t m, int32_t n, int32_t k, const uint16_t *residual,
                              int64_t residual_stride, uint16_t *c, int64_t ldc, int32_t swiglu,
                              int32_t form, void *stream) {
  using namespace yuear;
  if (m == 0 || n == 0)
    return 0;
  if (m < 0 || n < 0 || m > mx::kMaxRows || n > mx::kMaxRows || k % mx::kStep ||
      (swiglu != 0 && swiglu != 1) || (swiglu && (n % 2 || residual)) ||
      !mx::rows_ok(a, a_stride, a_scales, a_scales_stride, k, a_bits) ||
      !mx::rows_ok(w, w_stride, w_scales, w_scales_stride, k, 4) || !mx::aligned(a_scales, 4) ||
      !mx::aligned(w_scales, 4) || a_scales_stride % 4 || w_scales_stride % 4 || !mx::aligned(c, 2) || form < -1 ||
      form >= mx::kForms)
    return int32_t(hipErrorInvalidValue);
  const int width = swiglu ? n / 2 : n;
  constexpr int64_t kMostLd = int64_t(1) << 31;
  if (ldc < width || ldc >= kMostLd ||
      (residual && (!mx::aligned(residual, 2) || residual_stride < width || residual_stride >= kMostLd)))
    return int32_t(hipErrorInvalidValue);
  const mx::Span out = mx::bf16_span(c, ldc, m, width);
  for (const mx::Span &in :
       {mx::codes_span(a, a_stride, m, k, a_bits), mx::scales_span(a_scales, a_scales_stride, m, k),
        mx::codes_span(w, w_stride, n, k, 4), mx::scales_span(w_scales, w_scales_stride, n, k)})
    if (mx::overlap(in, out))
      return int32_t(hipErrorInvalidValue);
  // the output may replace the residual: a lane reads its values before it writes them
  if (residual && !(residual == c && residual_stride == ldc) &&
      mx::overlap(mx::bf16_span(residual, residual_stride, m, width), out))
    return int32_t(hipErrorInvalidValue);
  const mx::GemmArgs p{a, a_scales, w, w_scales, a_stride, a_scales_stride, w_stride, w_scales_stride, m, n, k,
                       residual, c, residual_stride, ldc,
                       swiglu ? mx::kSwiglu : residual ? mx::kResidual : mx::kStore};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (form < 0)
    form = mx::pick_form(a_bits, m, n, k);
  return int32_t(a_bits == 8 ? mx::launch<8>(form, p, st) : mx::launch<4>(form, p, st));
}

int32_t yuear_op_mx_gemm(const uint8_t *a, int64_t a_stride, const uint8_t *a_scales,
                         int64_t a_scales_stride, int32_t a_bits, const uint8_t *w, int64_t w_stride,
                         const uint8_t *w_scales, int64_t w_scales_stride, int32_t m, int32_t n,
                         int32_t k, const uint16_t *residual, int64_t residual_stride, uint16_t *c,
                         int64_t ldc, int32_t swiglu, void *stream) {
  return yuear_op_mx_gemm_form(a, a_stride, a_scales, a_scales_stride, a_bits, w, w_stride, w_scales,
                               w_scales_stride, m, n, k, residual, residual_stride, c, ldc, swiglu, -1, stream);
}

}  // extern "C"
