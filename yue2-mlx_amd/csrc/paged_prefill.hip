// Causal attention of prompt rows over pages of keys and values (paged.h,
// head_dim 128), for several sequences in one launch, with an optional window:
// row i of sequence b sits at position p = pos0[b] + i and
//
//   out[h] = sum_t softmax_t(q[h] . K[t] / sqrt(128)) V[t]
//
// over t <= p with p - t < window or t < sinks (window 0: all t), in pages that
// the table has; a row that sees nothing gives zeros. Bound by the two matrix
// products (4 * 128 operations a query head, row and visible key).
//
// A workgroup takes a tile of 32 rows a wave of one kv head: its "rows" are
// the (token, query head) pairs of the kv head's group, token by token, so all
// heads of a group share the K and V that the workgroup stages, and a tile spans
// few tokens, so little of its causal edge is computed for nothing. It walks the
// 64-key blocks that any of its rows sees. Both products run on
// v_mfma_f32_32x32x16_bf16:
//
//   S^T[key][row] = K[key][:] . q[row][:]      O^T[dim][row] += V^T[dim][key] . P^T[key][row]
//
// A lane holds one row's scores (column lane % 32), so the softmax needs one
// exchange with lane ^ 32 a block, and a rescale multiplies its own sums. The rows
// of the K operand are permuted (key_of) so that the scores a lane ends up with
// are its operand of the second product.
//
// The running maximum m of a row enters S as the accumulator's start (-m), so
// the difference is taken before the scale. It is raised only when a block's
// score passes it by more than kSlack (weights up to 2^8, exact in 32 bits as
// smaller ones are), which saves almost every rescale of the 64 sums. P is
// rounded to bf16, 2^-9 of each weight at most, as the output is: one MFMA per
// operand instead of two or three; the denominator sums the rounded weights.
#include <algorithm>
#include <cmath>

#include "../../include/yuear.h"
#include "attn_core.h"
#include "common.h"
#include "paged.h"
#include "paged_workspace.h"

namespace yuear {
namespace {

using attn::as_bf16x8;
using paged::Cache;
using paged::D;
using paged::kBlock;
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void *lds_ptr_t;

constexpr int kKeys = 64;  // keys of a step

struct PrefillParams {
  const uint16_t *q = nullptr;
  long long q_stride = 0;
  Cache cache;
  const int32_t *starts = nullptr, *pos0 = nullptr;
  int batch = 0, rows = 0, heads = 0, window = 0, sinks = 0;
  uint16_t *out = nullptr;
  long long out_stride = 0;
};

// [stage][32-key half][K | V][16-byte pieces]: 8 KiB each. K: the chunk c of
// key R in slot c ^ (R % 16) of its 256 bytes. V: chunk c (8 keys) of dim d in
// slot c ^ (d / 4 % 4) of its 64. Either way the 16 lanes that a ds_read_b128
// serves at once read 16 different 16-byte slots (gemm.hip).
struct Stage {
  u32x4 kv[2][2][512];
};

// Key of a 32-key block in row r of the K operand: lane l of the result then
// holds, in element j, the key 16 (j / 8) + 8 (l / 32) + j % 8.
__device__ __forceinline__ int key_of(int r) {
  return 16 * (r >> 4) + 8 * ((r >> 2) & 1) + 4 * ((r >> 3) & 1) + (r & 3);
}

__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}

template <int G, int W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(2, 2))) void
paged_prefill_kernel(PrefillParams p, float qscale, int max_tiles) {
  constexpr int kRows = 32 * W;
  __shared__ Stage ring[2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int kvh = blockIdx.x;

  // the tile: the last ones, which see the most keys, first
  auto rows_of = [&](int b) {
    return paged::sequence_rows(p.starts, p.pos0, b, p.rows, p.cache.capacity);
  };
  int b, tile;
  if (!paged::find_item(p.batch, max_tiles - 1 - int(blockIdx.y),
                        [&](int s) { return (rows_of(s).n * G + kRows - 1) / kRows; }, b, tile))
    return;
  const paged::Rows rs = rows_of(b);
  const int pos0 = rs.pos0;
  // packed rows of this tile, and of this wave's lane
  const int first_row = tile * kRows, end_row = min(rs.n * G, first_row + kRows);
  const int p0 = pos0 + first_row / G, p1 = pos0 + (end_row - 1) / G;
  const int my_row = first_row + 32 * wave + col;
  const bool valid = my_row < end_row;
  const int token = min(my_row, end_row - 1) / G, head = min(my_row, end_row - 1) % G;
  const int my_pos = pos0 + token;

  // 64-key blocks [0, lead) and [first, p1 / 64]
  int first = 0, lead = 0;
  if (p.window > 0) {
    first = max(0, p0 - p.window + 1) / kKeys;
    lead = min((p.sinks - 1) / kKeys + (p.sinks > 0), first);
  }
  const int steps = lead + p1 / kKeys - first + 1;
  auto block_of = [&](int x) { return x < lead ? x : first + x - lead; };

  // pages of the 32-key halves: lane 2 j + h the one of step base + j, half h
  const int32_t *table = p.cache.table + size_t(b) * p.cache.table_stride;
  int pages = 0, page_base = 0;
  auto load_pages = [&](int x0) {
    const int t = block_of(min(x0 + (lane >> 1), steps - 1)) * kKeys + kBlock * (lane & 1);
    pages = t < p.cache.capacity ? table[t >> p.cache.shift] : -1;
    page_base = x0;
  };
  load_pages(0);
  auto page_at = [&](int x, int h) {
    return __builtin_amdgcn_readlane(pages, 2 * (x - page_base) + h);
  };
  // this wave's part of step x: pieces of 1 KiB, 8 a half of K or V
  auto fetch = [&](int x, int stage) {
    if (x - page_base >= 32)
      load_pages(x);
    const int t0 = block_of(x) * kKeys;
#pragma unroll
    for (int j = 0; j < 32 / W; ++j) {
      const int piece = wave * (32 / W) + j;  // [half][K | V][8]
      const int h = piece >> 4, is_v = (piece >> 3) & 1, q = piece & 7;
      const int page = page_at(x, h);
      const size_t at = p.cache.at(p.cache.has(page) ? page : 0, kvh,
                                   (t0 + kBlock * h) & ((1 << p.cache.shift) - 1));
      const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(
          (is_v ? p.cache.v : p.cache.k) + at, 0, kBlock * D * 2, 0x00020000);
      const uint32_t off =
          is_v ? uint32_t(q * 1024 + (lane >> 2) * 64 + ((lane & 3) ^ (lane >> 4)) * 16)
               : uint32_t(q * 1024 + (lane >> 4) * 256 +
                          ((lane & 15) ^ ((4 * q + (lane >> 4)) & 15)) * 16);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)&ring[stage].kv[h][is_v][64 * q],
                                               16, off, 0, 0, 0);
    }
  };
  fetch(0, 0);

  // q operands: row `col`, dims 16 s + 8 half + [0, 8)
  u32x4 qb[8];
  {
    const u32x4 *src = reinterpret_cast<const u32x4 *>(
        p.q + (size_t(rs.first) + token) * p.q_stride + size_t(kvh * G + head) * D);
#pragma unroll
    for (int s = 0; s < 8; ++s)
      qb[s] = src[2 * s + half];
  }
  const float slack = 8.f / qscale;
  f32x16 start;  // -m in every element
#pragma unroll
  for (int j = 0; j < 16; ++j)
    start[j] = 0.f;
  bool set = false;  // m is a score of this row
  float l_run = 0.f;
  f32x16 o[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int j = 0; j < 16; ++j)
      o[dt][j] = 0.f;
  const int key_row = key_of(col);

  for (int x = 0; x < steps; ++x) {
    const int stage = x & 1, t0 = block_of(x) * kKeys;
    const bool held[2] = {p.cache.has(page_at(x, 0)), p.cache.has(page_at(x, 1))};
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's part has landed
    __syncthreads();                     // ... and everyone's; the other stage is free
    if (x + 1 < steps)
      fetch(x + 1, stage ^ 1);
    const int low = p.window > 0 ? my_pos - p.window : -1;  // visible: t > low or t < sinks
    // keys that some row of the tile does not see
    const bool part = !held[0] || !held[1] || t0 + kKeys - 1 > p0 ||
                      (p.window > 0 && t0 <= p1 - p.window && t0 + kKeys > p.sinks);
    f32x16 st[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      st[h] = start;
      const u32x4 *ks = ring[stage].kv[h][0] + key_row * 16;
#pragma unroll
      for (int s = 0; s < 8; ++s)
        st[h] = mfma32(ks[(2 * s + half) ^ (key_row & 15)], qb[s], st[h]);
    }
    if (part) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int t = t0 + kBlock * h + 16 * (j >> 3) + 8 * half + (j & 7);
          if (!held[h] || t > my_pos || (t <= low && t >= p.sinks))
            st[h][j] = -__builtin_inff();
        }
    }
    float mx = st[0][0];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 16; ++j)
        mx = fmaxf(mx, st[h][j]);
    mx = max_halves(mx);
    const bool raise = mx > slack || (!set && mx > -__builtin_inff());
    if (__any(raise)) {
      const float d = raise ? mx : 0.f;
      const float corr = __builtin_amdgcn_exp2f(-d * qscale);
      const float f = set ? corr : 1.f;  // (all sums are zero before the first score)
      l_run *= f;
      set = set || raise;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        start[j] -= d;
        st[0][j] -= d;
        st[1][j] -= d;
      }
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int j = 0; j < 16; ++j)
          o[dt][j] *= f;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t pw[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float a = __builtin_amdgcn_exp2f(st[h][2 * j] * qscale);
        const float c = __builtin_amdgcn_exp2f(st[h][2 * j + 1] * qscale);
        pw[j] = uint32_t(f2bf(a)) | (uint32_t(f2bf(c)) << 16);
        l_run = __builtin_amdgcn_fdot2_f32_bf16(as_bf16x2(pw[j]), as_bf16x2(0x3f803f80u), l_run,
                                                false);
      }
      uint32_t keep[8];  // values of keys that no row of the tile sees become zeros
      if (part) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          keep[j] = 0u;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int t = t0 + kBlock * h + 16 * (j >> 2) + 8 * half + 2 * (j & 3) + e;
            if (held[h] && t <= p1 && (p.window <= 0 || t > p0 - p.window || t < p.sinks))
              keep[j] |= 0xffffu << (16 * e);
          }
        }
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const u32x4 pb = u32x4{pw[4 * s], pw[4 * s + 1], pw[4 * s + 2], pw[4 * s + 3]};
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) {
          u32x4 v = ring[stage].kv[h][1][(32 * dt + col) * 4 + ((2 * s + half) ^ ((col >> 2) & 3))];
          if (part)
            v = u32x4{v.x & keep[4 * s], v.y & keep[4 * s + 1], v.z & keep[4 * s + 2],
                      v.w & keep[4 * s + 3]};
          o[dt] = mfma32(v, pb, o[dt]);
        }
      }
    }
  }
  const float l = sum_halves(l_run);
  if (!valid)
    return;
  const float inv = set ? 1.f / l : 0.f;
  // element j of tile dt: dim 32 dt + 8 (j / 4) + 4 half + j % 4
  uint16_t *dst = p.out + (size_t(rs.first) + token) * p.out_stride + size_t(kvh * G + head) * D;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const uint32_t lo = uint32_t(f2bf(o[dt][4 * a] * inv)) |
                          (uint32_t(f2bf(o[dt][4 * a + 1] * inv)) << 16);
      const uint32_t hi = uint32_t(f2bf(o[dt][4 * a + 2] * inv)) |
                          (uint32_t(f2bf(o[dt][4 * a + 3] * inv)) << 16);
      *reinterpret_cast<uint2 *>(dst + 32 * dt + 8 * a + 4 * half) = uint2{lo, hi};
    }
}

template <int G> hipError_t launch_g(const PrefillParams &p, hipStream_t s) {
  constexpr int W = 4;
  const float qscale = float(std::pow(double(D), -0.5)) * attn::kLog2e;
  // sequences of n rows take at most n G / 128 + 1 tiles each
  const long long tiles =
      (long long)p.rows * G / (32 * W) + std::min(p.batch, p.rows);
  if (tiles > 65535)
    return hipErrorInvalidValue;
  hipLaunchKernelGGL((paged_prefill_kernel<G, W>), dim3(p.cache.kv_heads, unsigned(tiles)),
                     dim3(64 * W), 0, s, p, qscale, int(tiles));
  return hipGetLastError();
}

}  // namespace
}  // namespace yuear

extern "C" {

int64_t yuear_op_paged_workspace_bytes(int32_t batch, int32_t heads, int32_t kv_heads,
                                       int32_t rows) {
  using namespace yuear;
  if (batch < 0 || rows < 0 || !paged::group_ok(heads, kv_heads))
    return 0;
  const int64_t group = heads / kv_heads;
  return int64_t(paged::kCounterBytes) + int64_t(2 * paged::kDecodeGroups) * group * (paged::D + 2) * 4;
}

int32_t yuear_op_paged_attention_prefill(
    const uint16_t *q, int64_t q_stride, const uint16_t *k_pages, const uint16_t *v_pages,
    int32_t pages, int32_t page_slots, const int32_t *table, int32_t table_width,
    int32_t table_stride, const int32_t *starts, const int32_t *pos0, int32_t batch, int32_t rows,
    int32_t heads, int32_t kv_heads, int32_t window, int32_t sinks, void *workspace,
    int64_t workspace_bytes, uint16_t *out, int64_t out_stride, void *stream) {
  using namespace yuear;
  if (batch < 0 || rows < 0 || window < 0 || sinks < 0 || !paged::group_ok(heads, kv_heads))
    return int32_t(hipErrorInvalidValue);
  if (!batch || !rows)
    return int32_t(hipSuccess);
  PrefillParams p;
  if (!paged::make_cache(p.cache, k_pages, v_pages, pages, page_slots, table, table_width,
                         table_stride, kv_heads) ||
      !paged::aligned16(q) || !paged::aligned16(out) || !starts || !pos0 || q_stride % 8 ||
      q_stride < int64_t(heads) * paged::D || out_stride % 8 ||
      out_stride < int64_t(heads) * paged::D || !paged::aligned16(workspace) ||
      workspace_bytes < yuear_op_paged_workspace_bytes(batch, heads, kv_heads, rows) ||
      (long long)rows * (heads / kv_heads) > 0x3fffffffLL)
    return int32_t(hipErrorInvalidValue);
  p.q = q;
  p.q_stride = q_stride;
  p.starts = starts;
  p.pos0 = pos0;
  p.batch = batch;
  p.rows = rows;
  p.heads = heads;
  p.window = window;
  p.sinks = sinks;
  p.out = out;
  p.out_stride = out_stride;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (heads / kv_heads) {
  case 1: return int32_t(launch_g<1>(p, s));
  case 2: return int32_t(launch_g<2>(p, s));
  case 3: return int32_t(launch_g<3>(p, s));
  case 4: return int32_t(launch_g<4>(p, s));
  case 6: return int32_t(launch_g<6>(p, s));
  case 8: return int32_t(launch_g<8>(p, s));
  }
  return int32_t(hipErrorInvalidValue);
}

}  // extern "C"
