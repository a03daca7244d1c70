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
  int wide;  // 16-byte stores (and residual loads) where a tile is whole
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
template <int EPI>
__device__ __forceinline__ void finish4(const GemmArgs &p, int m, int n, const float (&v)[4]) {
  if (n >= p.n)
    return;
  if (EPI == kSwiglu) {
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
      c[e] = f2bf(EPI == kResidual ? bf2f(r[e]) + v[e] : v[e]);
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return uint32_t(f2bf(lo)) | uint32_t(f2bf(hi)) << 16;
}

// A 32 x 32 MFMA tile, lane 32 h + r with features n + 8 q + 4 h + [0, 4) of token m
// at v[4 q ..]. Where the rows allow it (p.wide, whole tile) the lanes of a token
// trade halves first, so that each stores 16 bytes: h = 0 the features (SwiGLU
// outputs) below 16 (8), h = 1 the others.
template <int EPI>
__device__ __forceinline__ void finish32(const GemmArgs &p, int m, int n, int h,
                                         const float (&v)[16]) {
  if (!p.wide || n + 32 > p.n) {
    if (m < p.m)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float f[4] = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
        finish4<EPI>(p, m, n + 8 * q + 4 * h, f);
      }
    return;
  }
  if (EPI == kSwiglu) {
    uint32_t w[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      w[q] = pack2(silu_times(v[4 * q], v[4 * q + 1]), silu_times(v[4 * q + 2], v[4 * q + 3]));
    permlane32_swap(w[0], w[2]);
    permlane32_swap(w[1], w[3]);
    if (m < p.m)
      *reinterpret_cast<u32x4 *>(p.c + m * p.ldc + (n >> 1) + 8 * h) = u32x4{w[0], w[2], w[1], w[3]};
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
      const u32x4 r = *reinterpret_cast<const u32x4 *>(p.residual + m * p.residual_stride + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] += bflo(r[e]);
        x[2 * e + 1] += bfhi(r[e]);
      }
    }
    *reinterpret_cast<u32x4 *>(p.c + m * p.ldc + at) =
        u32x4{pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7])};
  }
}

// Few token rows: a workgroup computes 16 FT features of 16 MT tokens, its KW
// waves a part of K each with all operands straight from memory into registers,
// then adds the waves' sums in order.
//
// MFMA operands, lane l = 16 g + r: W (4 bits) row r, k 32 g .. 32 g + 31 of the
// step, the same of A in 4 bits; A in 8 bits k 16 g .. 16 g + 15 and 64 + 16 g ..;
// the scale of k-block g of row r in either case. D: features 4 g .. 4 g + 3 of
// token r.
template <int ABITS, int EPI, int MT, int FT, int KW>
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
      finish4<EPI>(p, m, n, v);
  }
}

// ---- many token rows: tiles through LDS ----
//
// A workgroup of WM x WN waves computes a BM x BN tile of C, each wave BM / WM
// tokens by BN / WN features as 32 x 32 MFMA tiles, 64 of K at a time. K advances
// by steps of 128 bytes of each A row (128 of K in 8 bits, 256 in 4) through a
// two-stage LDS ring that direct-to-LDS loads fill (1 KiB an instruction). The
// operands of the next 64 of K are read from LDS under the MFMAs of these. One
// barrier a step, before its last 64: past it every wave has read all of the
// stage, which takes the step after the next, and the next step's loads have
// landed.
//
// Scales come 512 of K at a time, 16 bytes a row, into two buffers behind the
// ring; a lane reads the byte of its row and k-block.
//
// MFMA operands, lane l = 32 h + r: W (4 bits) row r, k 32 h .. 32 h + 31 of the
// 64, the same of A in 4 bits; A in 8 bits k 16 h .. 16 h + 15 and 32 + 16 h ..; the
// scale of k-block h of row r. D: features 8 q + 4 h + [0, 4) of token r.
//
// LDS rows of 128 bytes (A, and W beside 4-bit A) keep their 16-byte chunk c at
// slot c ^ (row >> 1 & 7); rows of 64 bytes (W beside 8-bit A) at c ^ (bit 2 of the
// row | bit 4 << 1). A ds_read_b128 is served 16 lanes at a time (bit 5 of the
// lane, and bit 3 ^ bit 4): rows 0-7 and 24-31, or 8-23, with one chunk, which
// either layout spreads over all 16 slots of 256 bytes.
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void *lds_ptr_t;

// The kernel's only LDS object, so that the compiler tells the loads into one
// stage from the reads of the other.
extern __shared__ __attribute__((aligned(1024))) char mx_lds[];

template <int ABITS, int BM, int BN, int WM, int WN> struct Tile {
  static constexpr int kWaves = WM * WN;
  static constexpr int kWRow = ABITS == 8 ? 64 : 128;    // bytes of a W row a step
  static constexpr int kStepK = ABITS == 8 ? 128 : 256;  // K of a step
  static constexpr int kStage = BM * 128 + BN * kWRow;
  static constexpr int kScales = (BM + BN) * 16;         // of 512 of K
  static constexpr int kLds = 2 * kStage + 2 * kScales;
};

// Tile of workgroup b. Workgroups go to the 8 XCDs in turn, each with its own L2:
// XCD x takes one contiguous range of an order in columns of four tile rows, so
// that the tiles that share an L2 form a compact block of A and W rows.
__device__ __forceinline__ void tile_of(int b, int tiles_m, int tiles_n, int &tm, int &tn) {
  constexpr int kXcds = 8, kGroup = 4;
  const int total = tiles_m * tiles_n, each = total / kXcds, more = total % kXcds;
  const int x = b % kXcds;
  const int t = x * each + min(x, more) + b / kXcds;
  const int per = kGroup * tiles_n, first = t / per * kGroup;
  const int rows = min(tiles_m - first, kGroup), r = t % per;
  tm = first + r % rows;
  tn = r / rows;
}

__device__ __forceinline__ int slot128(int row, int chunk) { return chunk ^ ((row >> 1) & 7); }
__device__ __forceinline__ int slot64(int row, int chunk) {
  return chunk ^ (((row >> 2) & 1) | ((row >> 3) & 2));
}

template <int ABITS, int EPI, int BM, int BN, int WM, int WN>
__device__ __forceinline__ void tile(const GemmArgs &p) {
  using T = Tile<ABITS, BM, BN, WM, WN>;
  constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
  constexpr int AQ = ABITS / 4;            // 16-byte pieces of A of a lane and 64 of K
  constexpr int PARTS = T::kStepK / 64;
  constexpr int APW = BM / 8 / T::kWaves, WPW = BN * T::kWRow / 1024 / T::kWaves;
  constexpr int kGroupSteps = 512 / T::kStepK;
  static_assert(APW * T::kWaves * 8 == BM && WPW * T::kWaves * 1024 == BN * T::kWRow &&
                    TM * 32 * WM == BM && TN * 32 * WN == BN,
                "tile");
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int r = lane & 31, h = lane >> 5;
  int tm, tn;
  tile_of(int(blockIdx.x), (p.m + BM - 1) / BM, (p.n + BN - 1) / BN, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const int rows_a = min(p.m - m0, BM), rows_w = min(p.n - n0, BN);
  const auto ra = rows_rsrc(p.a + m0 * p.a_stride, p.a_stride, rows_a, p.k * ABITS / 8);
  const auto rw = rows_rsrc(p.w + n0 * p.w_stride, p.w_stride, rows_w, p.k / 2);

  // this wave's KiB blocks of A and of W: lane l fills slot l
  uint32_t from_a[APW], from_w[WPW];
#pragma unroll
  for (int i = 0; i < APW; ++i) {
    const int row = 8 * (wave * APW + i) + (lane >> 3);
    from_a[i] = uint32_t(row * int(p.a_stride) + slot128(row, lane & 7) * 16);
  }
#pragma unroll
  for (int i = 0; i < WPW; ++i) {
    constexpr int kRows = 1024 / T::kWRow;
    const int row = kRows * (wave * WPW + i) + lane / (64 / kRows);
    from_w[i] = uint32_t(row * int(p.w_stride) +
                         (T::kWRow == 64 ? slot64(row, lane & 3) : slot128(row, lane & 7)) * 16);
  }
  auto load = [&](int step) {
    char *stage = mx_lds + (step & 1) * T::kStage;
#pragma unroll
    for (int i = 0; i < APW; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_ptr_t)(stage + (wave * APW + i) * 1024), 16,
                                               from_a[i] + step * 128, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < WPW; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rw, (lds_ptr_t)(stage + BM * 128 + (wave * WPW + i) * 1024), 16,
          from_w[i] + step * T::kWRow, 0, 0, 0);
  };
  // 64 rows of scales a wave, A's first; waves past the last block repeat it
  constexpr int SB = (BM + BN) / 64;
  static_assert(SB <= T::kWaves && BM % 64 == 0, "scale blocks");
  const int sb = min(wave, SB - 1);
  const bool sb_a = sb < BM / 64;
  const auto rs = rows_rsrc(sb_a ? p.a_scales + m0 * p.a_scale_stride : p.w_scales + n0 * p.w_scale_stride,
                            sb_a ? p.a_scale_stride : p.w_scale_stride, sb_a ? rows_a : rows_w, p.k / 32);
  const uint32_t from_s = uint32_t((64 * (sb_a ? sb : sb - BM / 64) + lane) *
                                   int(sb_a ? p.a_scale_stride : p.w_scale_stride));
  auto load_scales = [&](int group) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        rs, (lds_ptr_t)(mx_lds + 2 * T::kStage + (group & 1) * T::kScales + sb * 1024), 16,
        from_s + group * 16, 0, 0, 0);
  };

  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        acc[i][j][e] = 0.f;

  const int a_row = wm * (BM / WM) + r, w_row = wn * (BN / WN) + r;  // of the first tiles
  u32x4 af[2][TM][AQ], wf[2][TN];
  int as[2][TM], ws[2][TN];
  // operands of part s of a step (64 of K), from the stage and scale buffers that hold it
  auto read = [&](int buf, int step, int s) {
    const char *a = mx_lds + (step & 1) * T::kStage + a_row * 128;
    const char *w = mx_lds + (step & 1) * T::kStage + BM * 128 + w_row * T::kWRow;
    const int at = PARTS * step + s;
    const uint8_t *sc = reinterpret_cast<const uint8_t *>(mx_lds) + 2 * T::kStage +
                        (at >> 3 & 1) * T::kScales + 2 * (at & 7) + h;
#pragma unroll
    for (int x = 0; x < (TM > TN ? TM : TN); ++x) {
      if (x < TN) {
        wf[buf][x] = *reinterpret_cast<const u32x4 *>(
            w + x * 32 * T::kWRow +
            (T::kWRow == 64 ? slot64(r, 2 * s + h) : slot128(r, 2 * s + h)) * 16);
        ws[buf][x] = sc[(BM + w_row + 32 * x) * 16];
      }
      if (x < TM) {
#pragma unroll
        for (int q = 0; q < AQ; ++q)
          af[buf][x][q] = *reinterpret_cast<const u32x4 *>(
              a + x * 32 * 128 + slot128(r, (ABITS == 8 ? 4 * s + 2 * q : 2 * s) + h) * 16);
        as[buf][x] = sc[(a_row + 32 * x) * 16];
      }
    }
  };
  auto multiply = [&](int buf) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const u32x4 w = wf[buf][j], lo = af[buf][i][0], hi = af[buf][i][AQ - 1];
        const i32x8 wv = {int(w.x), int(w.y), int(w.z), int(w.w), 0, 0, 0, 0};
        const i32x8 av = {int(lo.x), int(lo.y), int(lo.z), int(lo.w),
                          int(hi.x), int(hi.y), int(hi.z), int(hi.w)};
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
            wv, av, acc[i][j], 4, ABITS == 8 ? 0 : 4, 0, ws[buf][j], 0, as[buf][i]);
      }
  };

  // Step `step`, whose last barrier lets the ring take step + 2 and, at the end of a group of
  // scales, their buffer the next but one. Reads and loads go between the MFMAs.
  constexpr int kReads = TN + TM * AQ + TM + TN, kMfmas = TM * TN;
  auto advance = [&](int step, int s_last) {
#pragma unroll
    for (int s = 0; s + 1 < PARTS; ++s) {
      read((s + 1) & 1, step, s + 1);
      multiply(s & 1);
#pragma unroll
      for (int x = 0; x < kMfmas; ++x) {
        __builtin_amdgcn_sched_group_barrier(0x100, (kReads + kMfmas - 1) / kMfmas, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
    read(0, step + 1, 0);
    load(step + 2);
    if (s_last)
      load_scales(step / kGroupSteps + 2);
    multiply(1);
#pragma unroll
    for (int x = 0; x < kMfmas; ++x) {
      if (x < kMfmas / 2)
        __builtin_amdgcn_sched_group_barrier(0x100, (kReads + kMfmas / 2 - 1) / (kMfmas / 2), 0);
      else
        __builtin_amdgcn_sched_group_barrier(0x020, (APW + WPW + 1 + kMfmas / 2 - 1) / (kMfmas / 2), 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  const int steps = p.k / T::kStepK;
  load(0);
  load_scales(0);
  load_scales(1);
  __builtin_amdgcn_s_waitcnt(0);  // (a barrier waits for no global load)
  load(1);                        // past K, here and below: read by nobody
  __syncthreads();
  read(0, 0, 0);
  int step = 0;
  for (; step + kGroupSteps <= steps; step += kGroupSteps)
#pragma unroll
    for (int s = 0; s < kGroupSteps; ++s)
      advance(step + s, s == kGroupSteps - 1);
  for (; step < steps; ++step)
    advance(step, 0);
  if (p.k % T::kStepK) {  // 4 bits: an odd number of 128s leaves half of a step
    read(1, step, 1);
    multiply(0);
    multiply(1);
  }
  __builtin_amdgcn_s_waitcnt(0);  // loads past K still in flight

#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e)
        v[e] = acc[i][j][e];
      finish32<EPI>(p, m0 + a_row + 32 * i, n0 + wn * (BN / WN) + 32 * j, h, v);
    }
}

template <int ABITS, int EPI, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void tile_kernel(GemmArgs p) {
  tile<ABITS, EPI, BM, BN, WM, WN>(p);
}

template <class T>
hipError_t launch_tile(void (*kernel)(GemmArgs), int bm, int bn, const GemmArgs &p, hipStream_t s) {
  const int64_t tiles = ((int64_t(p.m) + bm - 1) / bm) * ((int64_t(p.n) + bn - 1) / bn);
  if (tiles * T::kWaves * 64 >= int64_t(1) << 32)
    return hipErrorInvalidValue;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, T::kLds);
  if (e != hipSuccess)
    return e;
  hipLaunchKernelGGL(kernel, dim3(unsigned(tiles)), dim3(T::kWaves * 64), T::kLds, s, p);
  return hipGetLastError();
}

template <int ABITS, int EPI> hipError_t launch_form(const GemmArgs &p, hipStream_t s) {
  auto go = [&](auto kernel, int mt, int ft, int kw) {
    const int64_t x = (int64_t(p.n) + 16 * ft - 1) / (16 * ft), y = (int64_t(p.m) + 16 * mt - 1) / (16 * mt);
    if (x * kw * 64 >= int64_t(1) << 32 || y > 65535)
      return hipErrorInvalidValue;
    hipLaunchKernelGGL(kernel, dim3(unsigned(x), unsigned(y)), dim3(unsigned(kw * 64)), 0, s, p);
    return hipGetLastError();
  };
  if (p.m <= 16)
    return go(rows_kernel<ABITS, EPI, 1, 1, 4>, 1, 1, 4);
  if (p.m <= 512)
    return go(rows_kernel<ABITS, EPI, 4, 4, 4>, 4, 4, 4);
  return launch_tile<Tile<ABITS, 256, 256, 4, 2>>(tile_kernel<ABITS, EPI, 256, 256, 4, 2>, 256, 256, p, s);
}

template <int ABITS> hipError_t launch(const GemmArgs &p, hipStream_t s) {
  switch (p.epilogue) {
  case kSwiglu: return launch_form<ABITS, kSwiglu>(p, s);
  case kResidual: return launch_form<ABITS, kResidual>(p, s);
  default: return launch_form<ABITS, kStore>(p, s);
  }
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
                       swiglu ? mx::kSwiglu : residual ? mx::kResidual : mx::kStore,
                       mx::aligned(c, 16) && ldc % 8 == 0 &&
                           (!residual || (mx::aligned(residual, 16) && residual_stride % 8 == 0))};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return int32_t(a_bits == 8 ? mx::launch<8>(p, st) : mx::launch<4>(p, st));
}
