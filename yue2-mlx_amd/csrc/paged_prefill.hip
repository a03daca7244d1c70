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
// A workgroup of 4 waves takes a tile of 128 rows of one kv head, 32 a wave: its
// "rows" are the (token, query head) pairs of the kv head's group, token by token,
// so all heads of a group share the K and V that the workgroup stages, and a tile
// spans few tokens, so little of its causal edge is computed for nothing. It
// walks the 64-key steps that any of its rows sees. Both products run on
// v_mfma_f32_32x32x16_bf16:
//
//   S^T[key][row] = K[key][:] . q[row][:]      O^T[dim][row] += V^T[dim][key] . P^T[key][row]
//
// A lane holds one row's scores (column lane % 32), so the softmax needs one
// exchange with lane ^ 32 a step, and a rescale multiplies its own sums. The rows
// of the K operand are permuted (key_of) so that the scores a lane ends up with
// are its operand of the second product: P never passes through LDS.
//
// K and V go from HBM to LDS without registers, two steps of each in 64 KiB, so
// two workgroups share a CU and one's products run beside the other's barriers.
// A step computes S of the step after it beside its own exponentials, and P V
// beside the scaling of those scores; K is therefore loaded a step ahead of V.
// Measured, 24 heads of 8 at 3000 rows / 16 of 8 and a window of 1024, 5 sequences of
// 411 to 5003 (us): this form 73 / 111 (760 / 640 TFLOP/s; 12000 rows 1080); 64 rows a
// wave, one wave a SIMD, 106 / 155; 8 waves and four steps of LDS, one workgroup a CU,
// 88 / 130; S and P V of the same step one after the other 103 / 155.
//
// The running maximum m of a row is a raw score, taken off the others before the
// scale: equal keys weigh the same in every step, whatever their score is (off as
// they are scaled, fma(score, scale, -m), weights of scores past 2^24 are wrong; as
// fast). It is raised only when a score passes it by more than kSlack (the weights,
// up to 2^20, are as exact in 32 bits and in bf16 as smaller ones), so almost no
// step rescales the 64 sums.
//
// P is rounded to bf16, half a step of 2^-8 of each weight, as the output is; the
// denominator sums the rounded weights. Whole calls are off by 0.0020-0.0022 of 64
// bits' (2-norm), of which the output's rounding is 0.0017. P in two pieces leaves
// that alone and takes 16 more products a step: 3000 rows 75 -> 95 us, 12000 rows
// 821 -> 1101, the windowed prompts 108 -> 133, 97 rows after 4000 keys 28 -> 29.
//
// A prompt piece of few rows behind many keys has fewer tiles than CUs (runs_of):
// there the workgroups take equal runs of all tiles' steps, leave the sums of tiles
// that they share, and a second kernel joins them.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/yuear.h"
#include "attn_core.h"
#include "common.h"
#include "paged.h"
#include "paged_workspace.h"

namespace yuear {
namespace {

using attn::as_bf16x8;
using attn::f32x4;
using paged::Cache;
using paged::D;
using paged::kBlock;
using paged::pack_bf16;
using paged::wave_scan;
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void *lds_ptr_t;

constexpr int kKeys = 64;                 // keys of a step
constexpr int kWaves = 4, kRows = 32 * kWaves;  // of a tile
constexpr float kSlack = 20.f;  // log2 of the largest weight

struct PrefillParams {
  const uint16_t *q = nullptr;
  long long q_stride = 0;
  Cache cache;
  const int32_t *starts = nullptr, *pos0 = nullptr;
  int batch = 0, rows = 0, heads = 0, window = 0, sinks = 0;
  uint16_t *out = nullptr;
  long long out_stride = 0;
  int tiles = 0;  // of a kv head, at most
  int runs = 0;   // workgroups of a dealt launch
  // dealt launches: records of the tiles (head: their number) and partials
  int32_t *info = nullptr;
  float *part = nullptr;
};

constexpr int kRuns = 512;  // workgroups of a dealt launch, at most
// Steps that beginning a tile costs (97 rows after 4000 keys / 400 after 3000: 27.2 /
// 40.3 us; 1: 29.4 / 42.7, 5: 27.5 / 40.4).
constexpr int kTileCost = 3;
// Sequences of a dealt launch, at most: every workgroup walks them all. Short pieces
// after 2000 and 3000 keys (us), dealt / whole tiles: 32 sequences 30.7 / 35.0 and
// 46.5 / 60.3, 60 sequences 46.6 / 35.3 and 70.8 / 66.0.
constexpr int kDealSequences = 32;
// A piece's sums as the lanes hold them, then its rows' maxima and denominators.
constexpr size_t kPartFloats = size_t(kRows) * D + 2 * kRows;
constexpr int kInfo = 8;  // words of a tile's record: first and last run, rows

// A step's K or V: [32-key half][16-byte pieces], 16 KiB. K: the chunk c of key
// R in slot c ^ (R % 16) of its 256 bytes. V: chunk c (8 keys) of dim d in slot
// c ^ (d / 4 % 4) of its 64. Either way the 16 lanes that a ds_read_b128 serves
// at once read 16 different 16-byte slots (gemm.hip).
struct Ring {
  u32x4 k[2][2][512], v[2][2][512];  // [step % 2]
};

// Key of a 32-key block in row r of the K operand: lane l of the result then
// holds, in element j, the key 16 (j / 8) + 8 (l / 32) + j % 8.
__device__ __forceinline__ int key_of(int r) {
  return 16 * (r >> 4) + 8 * ((r >> 2) & 1) + 4 * ((r >> 3) & 1) + (r & 3);
}

__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}

// A tile of kRows rows of one kv head: its sequence's rows, its own, and the
// 64-key blocks that it walks, [0, lead) and [first, ...).
struct Tile {
  paged::Rows rows;
  int seq, index;               // index: in the sequence
  int first_row, end_row;       // of the sequence's packed rows
  int p0, p1;                   // positions of the first and the last
  int first, lead, steps;
  __device__ __forceinline__ int block(int x) const { return x < lead ? x : first + x - lead; }
};
template <int G> __device__ __forceinline__ int tiles_of(const paged::Rows &r) {
  return (r.n * G + kRows - 1) / kRows;
}
template <int G>
__device__ __forceinline__ Tile tile_of(const PrefillParams &p, const paged::Rows &rows, int seq,
                                        int index) {
  Tile t;
  t.rows = rows;
  t.seq = seq;
  t.index = index;
  t.first_row = index * kRows;
  t.end_row = min(rows.n * G, t.first_row + kRows);
  t.p0 = rows.pos0 + t.first_row / G;
  t.p1 = rows.pos0 + (t.end_row - 1) / G;
  t.first = t.lead = 0;
  if (p.window > 0) {
    t.first = max(0, t.p0 - p.window + 1) / kKeys;
    t.lead = min((p.sinks - 1) / kKeys + (p.sinks > 0), t.first);
  }
  t.steps = t.lead + t.p1 / kKeys - t.first + 1;
  return t;
}

// The work of a dealt launch in units, a step each and kTileCost for beginning a
// tile: the units of a kv head are those of its tiles, sequence by sequence. Every
// wave holds the (at most kDealSequences) sequences, one a lane, and walks their
// tiles 64 at a time.
template <int G> struct Deal {
  const PrefillParams &p;
  paged::Rows mine;  // of the lane's sequence
  int total = 0, tiles = 0;
  __device__ __forceinline__ explicit Deal(const PrefillParams &params) : p(params) {
    const int lane = threadIdx.x & 63;
    mine = paged::Rows{0, 0, 0};
    if (lane < p.batch)
      mine = paged::sequence_rows(p.starts, p.pos0, lane, p.rows, p.cache.capacity);
    for (int b = 0; b < p.batch; ++b) {
      const paged::Rows r = rows(b);
      const int n = tiles_of<G>(r);
      for (int t0 = 0; t0 < n; t0 += 64)
        total += __builtin_amdgcn_readlane(wave_scan(units(r, b, t0 + lane, n)), 63);
      tiles += n;
    }
  }
  __device__ __forceinline__ paged::Rows rows(int b) const {
    return paged::Rows{__builtin_amdgcn_readlane(mine.first, b), __builtin_amdgcn_readlane(mine.n, b),
                       __builtin_amdgcn_readlane(mine.pos0, b)};
  }
  __device__ __forceinline__ int units(const paged::Rows &r, int b, int t, int n) const {
    return t < n ? tile_of<G>(p, r, b, t).steps + kTileCost : 0;
  }
  // The tile of unit u < total, its number among a head's tiles, and the unit's
  // place in it.
  __device__ __forceinline__ Tile find(int u, int &number, int &place) const {
    const int lane = threadIdx.x & 63;
    number = 0;
    for (int b = 0;; ++b) {
      const paged::Rows r = rows(b);
      const int n = tiles_of<G>(r);
      for (int t0 = 0; t0 < n; t0 += 64) {
        const int mine_ = units(r, b, t0 + lane, n), incl = wave_scan(mine_);
        const int all = __builtin_amdgcn_readlane(incl, 63);
        if (u < all) {
          const int at = __builtin_popcountll(__ballot(incl <= u));
          place = u - __builtin_amdgcn_readlane(incl - mine_, at);
          number += t0 + at;
          return tile_of<G>(p, r, b, t0 + at);
        }
        u -= all;
      }
      number += n;
    }
  }
  // The tile after t of the same head; false past its last.
  __device__ __forceinline__ bool next(Tile &t) const {
    if (t.index + 1 < tiles_of<G>(t.rows)) {
      t = tile_of<G>(p, t.rows, t.seq, t.index + 1);
      return true;
    }
    for (int b = t.seq + 1; b < p.batch; ++b) {
      const paged::Rows r = rows(b);
      if (r.n) {
        t = tile_of<G>(p, r, b, 0);
        return true;
      }
    }
    return false;
  }
};

// Whether the row at pos sees a key of steps [x_begin, x_end).
__device__ __forceinline__ bool sees_any(const PrefillParams &p, const Tile &tl, const int32_t *table,
                                         int pos, int low, int x_begin, int x_end) {
#pragma unroll 1
  for (int x = 2 * x_begin; x < 2 * x_end; ++x) {  // 32-key halves
    const int t = tl.block(x >> 1) * kKeys + kBlock * (x & 1);
    if (t <= pos && (min(t + kBlock - 1, pos) > low || t < p.sinks) && p.cache.has(table[t >> p.cache.shift]))
      return true;
  }
  return false;
}

// Steps [x_begin, x_end) of a tile of kv head kvh; part_of: where a piece of the
// tile leaves its sums (null: the whole tile). False, with nothing written, where
// walk_odd() has to do it.
template <int G>
__device__ __forceinline__ bool walk_tile(const PrefillParams &p, float qscale, const Tile &tl, int kvh,
                                          int x_begin, int x_end, float *part_of,
                                          Ring &ring) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  // the packed row of this lane
  const int my_row = tl.first_row + 32 * wave + col;
  const bool valid = my_row < tl.end_row;
  const int token = min(my_row, tl.end_row - 1) / G, head = min(my_row, tl.end_row - 1) % G;
  const int my_pos = tl.rows.pos0 + token;

  const int low = p.window > 0 ? my_pos - p.window : -1;  // visible: t > low or t < sinks
  const int x_last = x_end - 1;

  // ---- what the steps of [base, base + 32) need, lane 2 j + h for half h of
  // step base + j: its page's element (of this kv head; page 0 where the table
  // has none) and which steps have no page (absent), keys that some row of the
  // wave does not see (partial), some row
  // of the tile does not see (edge) or no row of the tile sees (dead) ----
  const int32_t *table = p.cache.table + size_t(tl.seq) * p.cache.table_stride;
  int base = 0;
  uint32_t at_lo = 0, at_hi = 0;
  unsigned long long absent = 0, partial = 0, edge = 0, dead = 0;
  const int w0 = tl.rows.pos0 + min(tl.first_row + 32 * wave, tl.end_row - 1) / G;
  const int w1 = tl.rows.pos0 + min(tl.first_row + 32 * wave + 31, tl.end_row - 1) / G;
  auto load_steps = [&](int x0) __attribute__((always_inline)) {
    const int t0 = tl.block(min(x0 + (lane >> 1), x_last)) * kKeys, t = t0 + kBlock * (lane & 1);
    const int page = t < p.cache.capacity ? table[t >> p.cache.shift] : -1;
    const bool has = p.cache.has(page);
    const size_t at = p.cache.at(has ? page : 0, kvh, t & ((1 << p.cache.shift) - 1));
    at_lo = uint32_t(at);
    at_hi = uint32_t(at >> 32);
    absent = __ballot(!has);
    auto unseen = [&](int last, int first) {  // by rows at first .. last
      return t0 + kKeys - 1 > first ||
             (p.window > 0 && t0 <= last - p.window && t0 + kKeys > p.sinks);
    };
    partial = absent | __ballot(unseen(w1, w0));
    edge = absent | __ballot(unseen(tl.p1, tl.p0));
    dead = absent | __ballot(unseen(tl.p0, tl.p1));
    base = x0;
  };
  auto bits = [&](unsigned long long of, int x) __attribute__((always_inline)) { return int(of >> (2 * (x - base))) & 3; };

  // ---- loads: a wave's part of a step's K and V is 4 pieces of 1 KiB of
  // one half. Past the last step it is taken again (nobody reads it), so every
  // step issues as many loads and the waits count them. ----
  constexpr int kPieces = 16 / kWaves;
  const int my_half = wave >> 1, piece0 = (wave & 1) * kPieces;
  uint32_t k_off[kPieces];
#pragma unroll
  for (int j = 0; j < kPieces; ++j)
    k_off[j] = uint32_t((piece0 + j) * 1024 + (lane >> 4) * 256 +
                        ((lane & 15) ^ ((4 * (piece0 + j) + (lane >> 4)) & 15)) * 16);
  const uint32_t v_off = uint32_t(piece0 * 1024 + (lane >> 2) * 64 + ((lane & 3) ^ (lane >> 4)) * 16);
  auto at_of = [&](int x) __attribute__((always_inline)) {
    const int from = 2 * (min(x, x_last) - base) + my_half;
    return (unsigned long long)(uint32_t(__builtin_amdgcn_readlane(at_hi, from))) << 32 |
           uint32_t(__builtin_amdgcn_readlane(at_lo, from));
  };
  auto load = [&](const uint16_t *from, size_t at, u32x4 *to, uint32_t off, int piece) __attribute__((always_inline)) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(from) + at, 0, kBlock * D * 2,
                                          0x00020000),
        (lds_ptr_t)(to + 64 * piece), 16, off, 0, 0, 0);
  };
  auto load_k = [&](size_t at, int x, int j) __attribute__((always_inline)) {
    load(p.cache.k, at, ring.k[x & 1][my_half], k_off[j], piece0 + j);
  };
  auto load_v = [&](size_t at, int x, int j) __attribute__((always_inline)) {
    load(p.cache.v, at, ring.v[x & 1][my_half], v_off + 1024 * j, piece0 + j);
  };

  // q operands: row `col`, dims 16 s + 8 half + [0, 8)
  u32x4 qb[8];
  {
    const u32x4 *src = reinterpret_cast<const u32x4 *>(
        p.q + (size_t(tl.rows.first) + token) * p.q_stride + size_t(kvh * G + head) * D);
#pragma unroll
    for (int s = 0; s < 8; ++s)
      qb[s] = src[2 * s + half];
  }
  load_steps(x_begin);
  size_t v_at = at_of(x_begin);  // of the step whose V is loaded next
#pragma unroll
  for (int j = 0; j < kPieces; ++j)
    load_k(v_at, x_begin, j);
  const size_t second_at = at_of(x_begin + 1);
#pragma unroll
  for (int j = 0; j < kPieces; ++j)
    load_v(v_at, x_begin, j);
#pragma unroll
  for (int j = 0; j < kPieces; ++j)
    load_k(second_at, x_begin + 1, j);
  v_at = second_at;

  float m_run = 0.f;  // what is taken off the row's scores: the largest at some step
  bool set = false;   // m_run is from a score of this row
  float l_run[2] = {0.f, 0.f};
  f32x16 o[4], e[2];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int j = 0; j < 16; ++j)
      o[dt][j] = 0.f;
  const int key_row = key_of(col);
  const int k_read = key_row * 16, k_xor = (key_row & 15) ^ half;  // chunk 2 s + half: 2 s ^ k_xor
  const int v_read = col * 4, v_xor = ((col >> 2) & 3) ^ half;
  auto k_operand = [&](int x, int n) __attribute__((always_inline)) {  // of product n: half n % 2, dims 16 (n / 2)
    return ring.k[x & 1][n & 1][k_read + ((n & ~1) ^ k_xor)];
  };

  // The exponents of a step's weights from its scores st, where its keys are not all
  // seen or its largest score passed the running maximum by kSlack: -inf for keys
  // that the lane's row does not see, and a raised maximum.
  f32x16 st[2];
  auto settle = [&](int x) __attribute__((always_inline)) {
    const int t0 = tl.block(x) * kKeys;
    if (bits(partial, x)) {
      const bool cut = p.window > 0 && t0 <= w1 - p.window;  // (uniform)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // element j is the key at + 16 (j / 8) + j % 8; unseen: past `last`, or
        // `many` keys from `from` on
        const int at = t0 + kBlock * h + 8 * half, from = p.sinks - at;
        const int last = (bits(absent, x) >> h) & 1 ? -1 : my_pos - at;
        const uint32_t many = uint32_t(max(low - p.sinks + 1, 0));
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (16 * (j >> 3) + (j & 7) > last)
            st[h][j] = -__builtin_inff();
        if (cut)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (uint32_t(16 * (j >> 3) + (j & 7) - from) < many)
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
    const bool raise = set ? (mx - m_run) * qscale > kSlack : mx > -__builtin_inff();
    if (__any(raise)) {
      const float m_new = raise ? mx : m_run;
      const float f = set ? __builtin_amdgcn_exp2f((m_run - m_new) * qscale) : 1.f;  // (no sums before the first score)
      l_run[0] *= f;
      l_run[1] *= f;
      m_run = m_new;
      set = set || raise;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int j = 0; j < 16; ++j)
          o[dt][j] *= f;
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      e[0][j] = (st[0][j] - m_run) * qscale;
      e[1][j] = (st[1][j] - m_run) * qscale;
    }
  };
  // what every wave does at the start of a step
  auto begin_step = [&](int x) __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // V of step x and K of step x + 1
    __syncthreads();  // everyone's part; V's slot of step x - 1 and K's of x are free
    if (__builtin_expect(x + 2 - base >= 32, 0))
      load_steps(x);
  };
  // An unseen key weighs 0, but 0 times an infinity or a NaN would count. So in a
  // step with keys that not all rows of the tile see, the values of those that
  // none sees become zeros here (a wave takes 8 keys of all dims at a time, a lane
  // two dims), and infinities or NaNs that remain are noticed: walk_odd() then does
  // the tile again.
  uint32_t odd = 0;
  auto odd_halves = [&](uint32_t w) __attribute__((always_inline)) {
    return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
  };
  // (the lane's number anew, so that what this computes from it stays here)
  auto rare = [&](int v) __attribute__((always_inline)) {
    asm volatile("" : "+v"(v));
    return v;
  };
  auto bury = [&](int x) __attribute__((always_inline)) {
    const int me = rare(lane);
    if (bits(dead, x)) {
      const int t0 = tl.block(x) * kKeys;
      for (int n = wave; n < kKeys / 8; n += kWaves) {
        const int t = t0 + 8 * n;
        uint32_t keep[4] = {0u, 0u, 0u, 0u};
        if (!((bits(absent, x) >> (n >> 2)) & 1)) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (t + k <= tl.p1 && (p.window <= 0 || t + k > tl.p0 - p.window || t + k < p.sinks))
              keep[k >> 1] |= 0xffffu << (16 * (k & 1));
        }
        if ((keep[0] & keep[1] & keep[2] & keep[3]) == 0xffffffffu)
          continue;
#pragma unroll
        for (int d0 = 0; d0 < D; d0 += 64) {
          const int d = d0 + me;
          u32x4 &v = ring.v[x & 1][n >> 2][d * (kBlock / 8) + ((n & 3) ^ ((d >> 2) & 3))];
          v = u32x4{v.x & keep[0], v.y & keep[1], v.z & keep[2], v.w & keep[3]};
        }
      }
      __syncthreads();  // (all waves agree: the tile's keys and pages are the same)
    }
    const u32x4 *v = ring.v[x & 1][0] + 256 * wave + me;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x4 w = v[64 * i];
      odd |= odd_halves(w.x) | odd_halves(w.y) | odd_halves(w.z) | odd_halves(w.w);
    }
  };
  // At the tile's end: whether any wave noticed some. Through K's slot of the last
  // step, which nothing is loaded into any more.
  auto any_odd = [&]() __attribute__((always_inline)) {
    const uint32_t mine = __any(odd != 0);
    u32x4 &slot = ring.k[x_last & 1][0][0];
    if (lane == 0)
      reinterpret_cast<uint32_t *>(&slot)[wave] = mine;
    __syncthreads();
    const u32x4 all = slot;
    return __builtin_amdgcn_readfirstlane(all.x | all.y | all.z | all.w) != 0;
  };

  __builtin_amdgcn_s_waitcnt(0x0F70 | 2 * kPieces);  // Q and K of the first step
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int j = 0; j < 16; ++j)
      st[h][j] = 0.f;
#pragma unroll
  for (int n = 0; n < 16; ++n)
    st[n & 1] = mfma32(k_operand(x_begin, n), qb[n >> 1], st[n & 1]);

  if (tl.first_row + 32 * wave >= tl.end_row) {  // no row of the wave's: it only loads
    for (int x = x_begin; x < x_end; ++x) {
      begin_step(x);
      if (bits(edge, x))
        bury(x);
      if (x == x_last)
        break;
      const size_t k_at = at_of(x + 2);
#pragma unroll
      for (int j = 0; j < kPieces; ++j)
        load_v(v_at, x + 1, j);
#pragma unroll
      for (int j = 0; j < kPieces; ++j)
        load_k(k_at, x + 2, j);
      v_at = k_at;
    }
    return !any_odd();
  }
  settle(x_begin);
  auto step = [&](int x, auto more_tag) __attribute__((always_inline)) {
    constexpr bool more = decltype(more_tag)::value;  // not the last one
    begin_step(x);
    if (__builtin_expect(bits(edge, x), 0))
      bury(x);
    u32x4(&vs)[2][512] = ring.v[x & 1];
    uint32_t pw[2][8];
    auto weights = [&](int w) __attribute__((always_inline)) {  // words 2 w, 2 w + 1 of P's 16, rounded, and their sum
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int h = w >> 2, j = (2 * w + k) & 7;
        pw[h][j] = pack_bf16(__builtin_amdgcn_exp2f(e[h][2 * j]),
                             __builtin_amdgcn_exp2f(e[h][2 * j + 1]));
        l_run[k] = __builtin_amdgcn_fdot2_f32_bf16(as_bf16x2(pw[h][j]), as_bf16x2(0x3f803f80u),
                                                   l_run[k], false);
      }
    };
    auto values = [&](int n) __attribute__((always_inline)) {  // the 16 products of P and V
      const int h = n >> 3, s = (n >> 2) & 1, dt = n & 3;
      o[dt] = mfma32(vs[h][v_read + 128 * dt + ((2 * s) ^ v_xor)],
                     u32x4{pw[h][4 * s], pw[h][4 * s + 1], pw[h][4 * s + 2], pw[h][4 * s + 3]},
                     o[dt]);
    };
    if constexpr (more) {
      const size_t k_at = at_of(x + 2);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 16; ++j)
          st[h][j] = 0.f;
      // S of the next step beside P of this one
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        st[n & 1] = mfma32(k_operand(x + 1, n), qb[n >> 1], st[n & 1]);
        if (n % (16 / kPieces) == 0)
          load_v(v_at, x + 1, n / (16 / kPieces));
        if (n & 1)
          weights(n >> 1);
      }
      // P V beside the scaling of the next step's scores
      float mx[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        mx[k] = -__builtin_inff();
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        values(n);
        if (n % (16 / kPieces) == 0)
          load_k(k_at, x + 2, n / (16 / kPieces));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int h = n >> 3, j = (2 * n + k) & 15;
          e[h][j] = (st[h][j] - m_run) * qscale;
          mx[n & 3] = fmaxf(mx[n & 3], e[h][j]);
        }
      }
      v_at = k_at;
      // LDS reads a few products ahead of their use
      constexpr int kAhead = 4;
      __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
      for (int n = 0; n < 32 - kAhead; ++n) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
      const bool due = bool(
          int(bits(partial, x + 1) != 0) |
          int(__ballot(!set | (fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) > kSlack)) != 0));
      if (__builtin_expect(due, 0))
        settle(x + 1);
    } else {
#pragma unroll
      for (int w = 0; w < 8; ++w)
        weights(w);
#pragma unroll
      for (int n = 0; n < 16; ++n)
        values(n);
    }
  };
  for (int x = x_begin; x < x_last; ++x)
    step(x, std::true_type{});
  step(x_last, std::false_type{});
  if (any_odd())
    return false;
  float l = sum_halves(l_run[0] + l_run[1]);
  // No weight: the lane's row sees no key, or scores of -inf alone (rare: not a
  // number, but in a piece only where the others have none either).
  const bool none = l == 0.f;
  if (__builtin_expect(__any(none), 0))
    l = none && sees_any(p, tl, table, my_pos, low, x_begin, x_end) ? __builtin_nanf("") : l;
  if (part_of) {
    f32x4 *to = reinterpret_cast<f32x4 *>(part_of) + wave * (16 * 64) + lane;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int a = 0; a < 4; ++a)
        to[(4 * dt + a) * 64] =
            f32x4{o[dt][4 * a], o[dt][4 * a + 1], o[dt][4 * a + 2], o[dt][4 * a + 3]};
    if (half == 0)
      reinterpret_cast<float2 *>(part_of + kRows * D)[32 * wave + col] =
          float2{none ? -__builtin_inff() : m_run, l};
    return true;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // (0: the row sees nothing)
  // element j of tile dt: dim 32 dt + 8 (j / 4) + 4 half + j % 4
  uint16_t *dst = p.out + (size_t(tl.rows.first) + token) * p.out_stride + size_t(kvh * G + head) * D;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int a = 0; a < 4; a += 2) {  // the halves trade pieces: 16 bytes a lane
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        w[k] = pack_bf16(o[dt][4 * a + 2 * k] * inv, o[dt][4 * a + 2 * k + 1] * inv);
        w[k + 2] = pack_bf16(o[dt][4 * a + 2 * k + 4] * inv, o[dt][4 * a + 2 * k + 5] * inv);
        permlane32_swap(w[k], w[k + 2]);
      }
      if (valid)
        *reinterpret_cast<u32x4 *>(dst + 32 * dt + 8 * (a + half)) = u32x4{w[0], w[1], w[2], w[3]};
    }
  return true;
}

// walk_tile() where a value that some rows of the tile see and others do not is
// not finite: row by row, a lane per key for the scores and per two dims for the
// sums, over the keys that the row sees alone. Rare, so plain.
template <int G>
__device__ __forceinline__ void walk_odd(const PrefillParams &p, float qscale, const Tile &tl, int kvh,
                                         int x_begin, int x_end, float *part_of) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int32_t *table = p.cache.table + size_t(tl.seq) * p.cache.table_stride;
  const int last = min(tl.first_row + 32 * (wave + 1), tl.end_row);
#pragma unroll 1
  for (int r = tl.first_row + 32 * wave; r < last; ++r) {
    const int token = r / G, head = kvh * G + r % G, pos = tl.rows.pos0 + token;
    const uint32_t *q = reinterpret_cast<const uint32_t *>(
        p.q + (size_t(tl.rows.first) + token) * p.q_stride + size_t(head) * D);
    float M = -__builtin_inff(), l = 0.f, o[2] = {0.f, 0.f};  // of dims lane and lane + 64
    bool any = false;  // a key is seen
#pragma unroll 1
    for (int x = x_begin; x < x_end; ++x) {
      const int t0 = tl.block(x) * kKeys, t = t0 + lane;
      const int page = t < p.cache.capacity ? table[t >> p.cache.shift] : -1;
      const bool sees = p.cache.has(page) && t <= pos &&
                        (p.window <= 0 || t > pos - p.window || t < p.sinks);
      const size_t at = p.cache.at(p.cache.has(page) ? page : 0, kvh,
                                   (t & ~(kBlock - 1)) & ((1 << p.cache.shift) - 1));
      const uint32_t *k = reinterpret_cast<const uint32_t *>(p.cache.k + at) + (lane & 31) * (D / 2);
      float score = 0.f;
#pragma unroll 8
      for (int d = 0; d < D / 2; ++d)
        score = __builtin_amdgcn_fdot2_f32_bf16(as_bf16x2(k[d]), as_bf16x2(q[d]), score, false);
      score = sees ? score : -__builtin_inff();
      float top = score;
#pragma unroll
      for (int b = 1; b < 64; b <<= 1)
        top = fmaxf(top, __shfl_xor(top, b));
      top = fmaxf(M, top);
      unsigned long long left = __ballot(sees);
      any = any || left;
      if (top == -__builtin_inff()) {
        if (!__any(sees && score != score))
          continue;
        top = 0.f;
      }
      const float f = M == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f((M - top) * qscale);
      const float w = sees ? __builtin_amdgcn_exp2f((score - top) * qscale) : 0.f;
      M = top;
      l *= f;
      o[0] *= f;
      o[1] *= f;
      for (; left; left &= left - 1) {
        const int n = __builtin_ctzll(left);
        const float wn = __shfl(w, n);
        const uint16_t *v = p.cache.v + __shfl((long long)at, n) + (n & 31);
        l += wn;
        o[0] += wn * __uint_as_float(uint32_t(v[lane * kBlock]) << 16);
        o[1] += wn * __uint_as_float(uint32_t(v[(lane + 64) * kBlock]) << 16);
      }
    }
    if (M == -__builtin_inff() && any)
      l = __builtin_nanf("");
    if (part_of) {  // as walk_tile() leaves it
      const int col = r - tl.first_row - 32 * wave;
      for (int k = 0; k < 2; ++k) {
        const int d = lane + 64 * k;
        part_of[4 * (wave * (16 * 64) + (d >> 3) * 64 + (d >> 2 & 1) * 32 + col) + (d & 3)] = o[k];
      }
      if (lane == 0)
        reinterpret_cast<float2 *>(part_of + kRows * D)[32 * wave + col] = float2{M, l};
      continue;
    }
    uint16_t *dst = p.out + (size_t(tl.rows.first) + token) * p.out_stride + size_t(head) * D;
    for (int k = 0; k < 2; ++k)
      dst[lane + 64 * k] = uint16_t(pack_bf16(M == -__builtin_inff() ? l : o[k] / l, 0.f));
  }
}

// One tile a workgroup, those of a sequence's end, which see the most keys, first
// (several sequences: the last one's).
template <int G>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) void
paged_prefill_kernel(PrefillParams p, float qscale) {
  __shared__ Ring ring;
  const int kv_heads = p.cache.kv_heads, kvh = int(blockIdx.x) % kv_heads;
  int seq, index;
  paged::Rows rows;
  if (!paged::find_rows(
          p.starts, p.pos0, p.batch, p.rows, p.cache.capacity,
          p.tiles - 1 - int(blockIdx.x) / kv_heads,
          [](const paged::Rows &of) { return tiles_of<G>(of); }, seq, index, rows))
    return;
  const Tile t = tile_of<G>(p, rows, seq, index);
  if (!walk_tile<G>(p, qscale, t, kvh, 0, t.steps, nullptr, ring))
    walk_odd<G>(p, qscale, t, kvh, 0, t.steps, nullptr);
}

// Dealt: every workgroup takes an equal run of the units of all heads.
template <int G>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) void
paged_prefill_deal_kernel(PrefillParams p, float qscale) {
  __shared__ Ring ring;
  const Deal<G> deal(p);
  const int total = deal.total * p.cache.kv_heads, each = total / p.runs, more = total % p.runs;
  auto run_begin = [&](int g) { return g * each + min(g, more); };
  auto run_of = [&](int u) {
    return u < more * (each + 1) ? u / (each + 1) : more + (u - more * (each + 1)) / each;
  };
  // dispatch goes round the 8 XCDs: each takes neighbouring runs, whose tiles
  // share K and V in its L2
  const int run = int(blockIdx.x % 8) * (p.runs / 8) + int(blockIdx.x / 8);
  // (more tiles than rows: `starts` decreases, and the workspace has no records for them)
  const bool valid = deal.tiles <= p.tiles;
  if (run == 0 && threadIdx.x == 0)
    p.info[0] = valid ? deal.tiles : 0;
  if (!valid)
    return;
  int u = run_begin(run);
  const int u1 = run_begin(run + 1);
  if (u >= u1)
    return;
  int kvh = u / deal.total, number, place;
  Tile t = deal.find(u - kvh * deal.total, number, place);
  while (true) {
    const int first = u - place + kTileCost;  // unit of the tile's first step
    const int x0 = max(place - kTileCost, 0), x1 = min(t.steps, u1 - first);
    if (x1 <= 0)
      return;  // not one step of the run's last tile
    const int r0 = run_of(first), r1 = run_of(first + t.steps - 1);
    if (x0 == 0 && threadIdx.x == 0) {
      int32_t *info = p.info + kInfo * (1 + size_t(kvh) * p.tiles + number);
      info[0] = r0;
      info[1] = r1;
      info[2] = t.rows.first;
      info[3] = t.first_row;
      info[4] = t.end_row;
    }
    // slot 2 run + 1: the tile begins in this run (its last one); 2 run: before it
    float *part_of = r0 == r1 ? nullptr : p.part + size_t(2 * run + (run == r0)) * kPartFloats;
    if (!walk_tile<G>(p, qscale, t, kvh, x0, x1, part_of, ring))
      walk_odd<G>(p, qscale, t, kvh, x0, x1, part_of);
    u = first + x1;
    if (u >= u1)
      return;
    __syncthreads();  // the ring is free
    place = 0;
    ++number;
    if (!deal.next(t)) {
      ++kvh;
      t = deal.find(0, number, place);
    }
  }
}

// Rows of tiles that several runs hold, joined in order of the keys: a workgroup
// per 32 rows and 32 dims, a wave per quarter of the pieces, its lanes as the
// tile's held them. Every load of a round of pieces is issued before the first is
// used: what costs here is the latency of one round after the other (a wave for
// all pieces: one row after 4000 keys 22.8 us in all, else 18.3).
template <int G>
__global__ __launch_bounds__(256) void paged_prefill_join_kernel(PrefillParams p, float qscale) {
  __shared__ f32x4 sums[kWaves][4][64];
  __shared__ float2 tops[kWaves][32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 31, half = lane >> 5, kvh = blockIdx.x;
  const int group = blockIdx.y >> 2, dt = blockIdx.y & 3;
  if (int(blockIdx.z) >= p.info[0])
    return;
  const int32_t *info = p.info + kInfo * (1 + size_t(kvh) * p.tiles + blockIdx.z);
  const int r0 = info[0], r1 = info[1], first = info[2], first_row = info[3], end_row = info[4];
  if (r0 == r1 || first_row + 32 * group >= end_row)
    return;
  const int pieces = r1 - r0 + 1, row = first_row + 32 * group + col;
  constexpr int kRound = 2;
  float M = -__builtin_inff(), l = 0.f, none = 0.f;  // none: of pieces without a weight, 0 or a NaN
  f32x4 o[4] = {};
  for (int j0 = wave; j0 < pieces; j0 += kRound * kWaves) {
    float2 ml[kRound];
    f32x4 v[kRound][4];
#pragma unroll
    for (int j = 0; j < kRound; ++j) {  // (past the last piece: that one, with weight 0)
      const int g = min(j0 + kWaves * j, pieces - 1);
      const float *from = p.part + size_t(2 * (r0 + g) + (g == 0)) * kPartFloats;
      ml[j] = reinterpret_cast<const float2 *>(from + kRows * D)[32 * group + col];
#pragma unroll
      for (int a = 0; a < 4; ++a)
        v[j][a] = reinterpret_cast<const f32x4 *>(from)[group * (16 * 64) + (4 * dt + a) * 64 + lane];
    }
    float top = M;
#pragma unroll
    for (int j = 0; j < kRound; ++j)
      top = fmaxf(top, ml[j].x);
    const float f = M == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((M - top) * qscale);
    l *= f;
#pragma unroll
    for (int a = 0; a < 4; ++a)
      o[a] *= f;
#pragma unroll
    for (int j = 0; j < kRound; ++j) {
      const bool out = j0 + kWaves * j >= pieces || ml[j].x == -__builtin_inff();
      none += ml[j].x == -__builtin_inff() ? ml[j].y : 0.f;
      const float w = out ? 0.f : __builtin_amdgcn_exp2f((ml[j].x - top) * qscale);
      l += out ? 0.f : w * ml[j].y;
#pragma unroll
      for (int a = 0; a < 4; ++a)
        o[a] += out ? f32x4{0.f, 0.f, 0.f, 0.f} : w * v[j][a];
    }
    M = top;
  }
#pragma unroll
  for (int a = 0; a < 4; ++a)
    sums[wave][a][lane] = o[a];
  if (half == 0)
    tops[wave][col] = float2{M, M == -__builtin_inff() ? none : l};
  __syncthreads();
  if (row >= end_row)
    return;
  // wave a: dims 8 a + [0, 8) of the 32
  M = tops[0][col].x;
#pragma unroll
  for (int w = 1; w < kWaves; ++w)
    M = fmaxf(M, tops[w][col].x);
  f32x4 all = {};
  l = none = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float2 ml = tops[w][col];
    if (ml.x == -__builtin_inff()) {
      none += ml.y;
      continue;
    }
    const float f = __builtin_amdgcn_exp2f((ml.x - M) * qscale);
    l += f * ml.y;
    all += f * sums[w][wave][lane];
  }
  if (M == -__builtin_inff())
    all = f32x4{none, none, none, none};
  else
    all *= 1.f / l;
  uint16_t *dst = p.out + (size_t(first) + row / G) * p.out_stride +
                  size_t(kvh * G + row % G) * D + 32 * dt + 8 * wave + 4 * half;
  *reinterpret_cast<uint2 *>(dst) = uint2{pack_bf16(all[0], all[1]), pack_bf16(all[2], all[3])};
}

// Tiles of a kv head that `rows` rows of `batch` sequences take at most.
long long tiles_at_most(int batch, int rows, int group) {
  return (long long)rows * group / kRows + std::min(batch, rows);
}

// Workgroups to deal the steps out over; 0: one tile a workgroup. To deal them
// costs about 8 steps' time (every piece begins anew, and a second kernel joins
// them), and is worth it where whole tiles would leave compute units idle for
// longer: a launch of them takes as long as one that sees all the keys that the
// tables hold, at most. A workgroup that shares its CU does a step in two thirds of
// the time, but shares more tiles: two a CU from 8 steps a workgroup on. 24 heads of
// 8, time of whole tiles / dealt over 256 / over 512 (us):
//   200 rows after 0 keys 11.0 / 14.7 / 16.7    97 after 4000   61.6 / 25.7 / 25.8
//   700 after 0           17.4 / 23.5 / 25.7    400 after 3000  55.9 / 41.0 / 37.2
//   1000 after 0          23.0 / 31.0 / 29.8    1000 after 3000 68.7 / 82.3 / 66.3
// The tables' width stands for the keys, which the host does not know: in a table of
// 24576 slots, 64 / 200 / 700 / 1000 rows from position 0 are dealt, and take 12.6 /
// 17.1 / 26.1 / 30.3 instead of 8.0 / 11.2 / 17.9 / 23.2.
int runs_of(const PrefillParams &p, long long tiles) {
  constexpr int kDealTiles = 256, kDealSteps = 8;
  if (p.batch > kDealSequences || tiles >= kDealTiles)
    return 0;
  long long keys = p.cache.capacity;
  if (p.window > 0)
    keys = std::min(keys, (long long)p.window + p.sinks + 2 * kKeys);
  const long long steps = keys / kKeys;
  // (steps are counted in 31 bits)
  if (steps >= (1 << 20) || steps * (kDealTiles - tiles) <= kDealSteps * kDealTiles)
    return 0;
  return steps * tiles < 8 * kRuns ? kRuns / 2 : kRuns;
}

template <int G> hipError_t launch_g(PrefillParams p, hipStream_t s) {
  const float qscale = float(std::pow(double(D), -0.5)) * attn::kLog2e;
  const int kv_heads = p.cache.kv_heads;
  const long long tiles = tiles_at_most(p.batch, p.rows, G);
  if (tiles * kv_heads > 0xffffff)  // workgroups of a launch
    return hipErrorInvalidValue;
  p.tiles = int(tiles);
  p.runs = runs_of(p, tiles * kv_heads);
  if (!p.runs) {
    hipLaunchKernelGGL(paged_prefill_kernel<G>, dim3(unsigned(p.tiles * kv_heads)), dim3(64 * kWaves), 0, s,
                       p, qscale);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(paged_prefill_deal_kernel<G>, dim3(p.runs), dim3(64 * kWaves), 0, s, p, qscale);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return e;
  hipLaunchKernelGGL(paged_prefill_join_kernel<G>, dim3(kv_heads, 4 * kWaves, p.tiles), dim3(256), 0, s,
                     p, qscale);
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
  // enough for every call of no more sequences, rows and heads
  const int64_t decode = int64_t(2 * paged::kDecodeGroups) * paged::kMaxGroup * (paged::D + 2) * 4;
  const int64_t tiles = tiles_at_most(batch, rows, paged::kMaxGroup) * kv_heads;
  const int64_t prefill =
      rows ? (1 + tiles) * int64_t(kInfo * 4) + 2 * kRuns * int64_t(kPartFloats * 4) : 0;
  return int64_t(paged::kCounterBytes) + std::max(decode, prefill);
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
  p.part = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + paged::kCounterBytes);
  p.info = reinterpret_cast<int32_t *>(p.part + 2 * kRuns * kPartFloats);
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
