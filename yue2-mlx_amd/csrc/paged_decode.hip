// Attention of one new token per sequence over pages of keys and values, with
// the token's q/k RMSNorm, RoPE and append (paged.h, head_dim 128).
//
//   K[pos] = bf16(rope(norm(k))), V[pos] = v
//   out[h] = sum_t softmax_t(rope(norm(q))[h] . K[t] / sqrt(128)) V[t]
//
// over t <= pos with pos - t < window or t < sinks (window 0: all t), in pages
// that the table has. The bytes of the visible K and V bound it; the arithmetic
// is G multiply-adds a byte.
//
// The work of a launch is the list of the visible 32-key blocks of every
// (sequence, kv head) item. The positions are read on the device, so one captured
// launch serves every length. Two ways to cut the list into workgroups:
//
// - up to 64 sequences, 512 items and 24 blocks a workgroup: each item into equal
//   chunks, one workgroup each, as many as 512 workgroups and 64 parts an item allow,
//   of at least a block a wave (one sequence of 4096 keys: 12.3 us, 15.9 cut the
//   other way, 14 with two blocks a wave; one kv head of 20000: 21 and 65). The
//   sequences are a wave's lanes, so the 65th changes the plan: 64 of 30 to 100 keys
//   11.8 us, 65 in runs 19.3; of 200 to 700 keys 27.7 and 31.0. Not where so many
//   items take one chunk each that the rest would be cut into more than twice the
//   blocks of equal shares (63 sequences of 370 keys and one of 24570: 414 us, in
//   runs 43);
// - else into equal runs, whatever the lengths of the sequences, and a workgroup
//   walks the items of its run (45 sequences of 150 to 24500 keys: 155 us, 189 in
//   chunks). To begin an item (positions, page, q, the joining of the waves) costs
//   a workgroup about as much as 8 blocks, which the runs count (2: 172 us).
//
// Short caches are bound by a chain of dependent loads, 8.2 us for one block a
// wave: positions, page numbers, K and V, each in turn, then what the waves leave in
// LDS; the joining of parts adds 2.8 us (333 keys: 10.9).
//
// A part that is a whole item is finished there; else the workgroup leaves its
// running maximum, sum and weighted values in its slots of the workspace, and
// the one that arrives last joins the item's parts in order of the keys.
//
// A wave takes every fourth block of its workgroup's. The block's K and V go to
// an LDS stage of the wave's own in whole KiB (buffer_load lds) and from there to
// registers, when the next block's loads are issued: 16 KiB a wave are always in
// flight, 32 MB over the chip. The loads are non-temporal: caches larger than the
// last-level cache pass through it 10% slower otherwise (45 sequences 176 us).
//
// Both products run on v_mfma_f32_16x16x32_bf16 as in attn_core.h (S^T = K q,
// O^T = V^T P^T, K rows permuted so that a lane's scores are its operand of the
// second product), with the G <= 8 heads in columns 0-7 as the leading bf16 piece
// of q and in columns 8-15 as the rest, so that q counts to 16 bits and P, split
// the same way, too: 2^-17 of each weight, at no more MFMAs than one piece each.
// Sums that are not finite are formed once more without pieces (walk_odd; 0.2 us of
// every call go into its being there and into looking at the sums).
#include <algorithm>
#include <cmath>

#include "../../include/yuear.h"
#include "attn_block.h"
#include "attn_core.h"
#include "common.h"
#include "kernels.h"
#include "paged.h"
#include "paged_workspace.h"

namespace yuear {
namespace {

using attn::f32x4;
using paged::Cache;
using paged::D;
using paged::kBlock;
using paged::pack_bf16;
using paged::wave_scan;

constexpr int kWaves = 4;
constexpr int kChunks = 512, kChunkBlocks = 24 * kChunks, kParts = 64;
typedef __attribute__((address_space(3))) void *lds_ptr_t;
constexpr int kLoadAux = 2;  // nt
constexpr int kItemCost = 8;  // blocks

struct DecodeParams {
  const uint16_t *qkv = nullptr;
  long long qkv_stride = 0;
  const uint16_t *q_norm = nullptr, *k_norm = nullptr;
  float eps = 0.f;
  const uint16_t *cos = nullptr, *sin = nullptr;
  Cache cache;
  const int32_t *pos = nullptr;
  int batch = 0, heads = 0, limit = 0, window = 0, sinks = 0, groups = 0;
  int32_t *counters = nullptr;
  float *part = nullptr;
  uint16_t *out = nullptr;
  long long out_stride = 0;
};

// The 32-key blocks that position pos sees: [0, lead) and [first, pos / 32].
struct Span {
  int lead = 0, first = 0, blocks = 0;
  __device__ __forceinline__ int block(int v) const { return v < lead ? v : first + v - lead; }
};
__device__ __forceinline__ Span span_of(int pos, int window, int sinks) {
  Span s;
  if (window > 0 && pos >= window) {
    s.first = (pos - window + 1) / kBlock;
    s.lead = min((sinks - 1) / kBlock + (sinks > 0), s.first);
  }
  s.blocks = s.lead + pos / kBlock - s.first + 1;
  return s;
}
__device__ __forceinline__ int blocks_at(const DecodeParams &p, int pos) {
  return pos < 0 || pos >= p.limit ? 0 : span_of(pos, p.window, p.sinks).blocks;
}
__device__ __forceinline__ int blocks_of(const DecodeParams &p, int b) {
  return blocks_at(p, p.pos[b]);
}

// m (running maximum of the raw scores), l, and o of one head of a
// workgroup's part of an item.
constexpr int kPartFloats = D + 2;
// parts that a joining thread has in flight (more heads: more of its registers are taken)
template <int G> constexpr int kRoundOf = G > 4 ? 16 : 32;

template <int G> struct Shared {
  union {
    u32x4 stage[kWaves][2][512];  // a wave's 32 keys: K, V; then its o over K
    float w[2][G][paged::kDecodeGroups];  // joining parts: m then weights, l
  };
  float q[G][D];
  uint16_t kv_new[2][D];
  float m[kWaves][G], l[kWaves][G];
  int is_last;
};

// Parts of an item that runs r0 .. r1 share, joined in order into the output of
// its G heads. Every load that a thread needs is issued before the first is
// used, kRound parts at a time: one after the other, 32 parts took 20 us.
template <int G>
__device__ __forceinline__ void join_parts(const DecodeParams &p, float qscale, int r0, int r1,
                                           int step, uint16_t *out, Shared<G> &sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = (r1 - r0) / step + 1;
  constexpr int kRound = kRoundOf<G>, kPairs = G * D / 2, kThreads = 64 * kWaves;
  // slot 2 r0 + 1, then 2 g: kSlot floats apart but for the first
  const int kSlot = 2 * G * kPartFloats * step;
  const float *first = p.part + size_t(2 * r0 + 1) * (G * kPartFloats);
  const float *rest = p.part + size_t(2 * r0) * (G * kPartFloats);
  const auto part = [&](int t) { return (t ? rest + size_t(t) * kSlot : first); };
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const auto load2 = [&](const float *at) {
    const unsigned long long v =
        __hip_atomic_load(reinterpret_cast<const unsigned long long *>(at), __ATOMIC_RELAXED,
                          __HIP_MEMORY_SCOPE_AGENT);
    return f32x2{__builtin_bit_cast(float, uint32_t(v)), __builtin_bit_cast(float, uint32_t(v >> 32))};
  };
  f32x2 o[kRound];
  auto load_round = [&](int q, int t0) {
    const int h = q / (D / 2), d = 2 * (q % (D / 2));
#pragma unroll
    for (int j = 0; j < kRound; ++j)  // (past the last part: that one, with weight 0)
      o[j] = load2(part(min(t0 + j, n - 1)) + h * kPartFloats + d);
  };
  const int q0 = min(int(threadIdx.x), kPairs - 1);
  const auto load_ml = [&](int at) { return load2(part(at / G) + (at % G) * kPartFloats + D); };
  const auto keep_ml = [&](int at, f32x2 ml) {
    sh.w[0][at % G][at / G] = ml.x;
    sh.w[1][at % G][at / G] = ml.y;
  };
  const f32x2 ml0 = load_ml(min(int(threadIdx.x), G * n - 1));
  load_round(q0, 0);
  if (int(threadIdx.x) < G * n)
    keep_ml(threadIdx.x, ml0);
  for (int at = threadIdx.x + kThreads; at < G * n; at += kThreads)
    keep_ml(at, load_ml(at));
  __syncthreads();
  for (int h = wave; h < G; h += kWaves) {
    float M = -__builtin_inff();
    for (int t = lane; t < n; t += 64)
      M = fmaxf(M, sh.w[0][h][t]);
    M = wave_max(M);
    float den = 0.f;
    for (int t = lane; t < n; t += 64) {
      const float m = sh.w[0][h][t];
      const float f = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((m - M) * qscale);
      den += f * sh.w[1][h][t];
      sh.w[0][h][t] = f;
    }
    const float inv = 1.f / wave_sum(den);
    for (int t = lane; t < (n + kRound - 1) / kRound * kRound; t += 64)
      sh.w[0][h][t] = t < n ? sh.w[0][h][t] * inv : 0.f;
  }
  __syncthreads();
  for (int q = threadIdx.x; q < kPairs; q += kThreads) {
    if (q != q0)
      load_round(q, 0);
    const int h = q / (D / 2);
    float a0 = 0.f, a1 = 0.f;
    for (int t0 = 0; t0 < n; t0 += kRound) {
      if (t0)
        load_round(q, t0);
#pragma unroll
      for (int j = 0; j < kRound; ++j) {
        const float w = sh.w[0][h][t0 + j];
        a0 = fmaf(w, o[j].x, a0);
        a1 = fmaf(w, o[j].y, a1);
      }
    }
    if (__builtin_expect(fmaf(a0, 0.f, a1 * 0.f) != 0.f, 0)) {
      // not finite: maybe only by 0 times an infinity of what is past the last part
      const int d = 2 * (q % (D / 2));
      a0 = a1 = 0.f;
#pragma unroll 1
      for (int t = 0; t < n; ++t) {
        const f32x2 v = load2(part(t) + h * kPartFloats + d);
        a0 = fmaf(sh.w[0][h][t], v.x, a0);
        a1 = fmaf(sh.w[0][h][t], v.y, a1);
      }
    }
    reinterpret_cast<uint32_t *>(out)[q] = pack_bf16(a0, a1);
  }
}

// A wave's blocks x, x + kWaves, ... < x1 of an item once more, where its sums are
// not finite: of an infinity the pieces of P and q can make a NaN (a second piece
// of 0 or of the other sign), so here q and the weights keep their 32 bits. Head by
// head, lanes n and n + 32 half a key each for the scores, a lane two dims for the
// sums. Rare, so plain.
template <int G>
__device__ __forceinline__ void walk_odd(const DecodeParams &p, float qscale, const Span &span,
                                         const int32_t *table, int kvh, int pos, int x, int x1,
                                         int wave, Shared<G> &sh) {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // (anew, so that what this computes from it stays here)
  const int low = p.window > 0 ? pos - p.window : -1;
  float *to = reinterpret_cast<float *>(sh.stage[wave][0]);
#pragma unroll 1
  for (int h = 0; h < G; ++h) {
    float M = -__builtin_inff(), l = 0.f, o[2] = {0.f, 0.f};  // of dims lane and lane + 64
    const float2 *q = reinterpret_cast<const float2 *>(sh.q[h]) + (lane >> 5) * (D / 4);
#pragma unroll 1
    for (int v = x; v < x1; v += kWaves) {
      const int t0 = span.block(v) * kBlock, t = t0 + (lane & 31);
      const int page = table[t0 >> p.cache.shift];
      const bool held = p.cache.has(page);
      const size_t at = p.cache.at(held ? page : 0, kvh, t0 & ((1 << p.cache.shift) - 1));
      const bool sees = t == pos || (held && t < pos && (t > low || t < p.sinks));
      const uint32_t *k = reinterpret_cast<const uint32_t *>(p.cache.k + at) + lane % 32 * (D / 2) +
                          (lane >> 5) * (D / 4);
      const uint32_t *own = reinterpret_cast<const uint32_t *>(sh.kv_new[0]) + (lane >> 5) * (D / 4);
      float score = 0.f;
#pragma unroll 4
      for (int d = 0; d < D / 4; ++d) {
        const uint32_t w = t == pos ? own[d] : k[d];
        score = fmaf(q[d].x, bflo(w), score);
        score = fmaf(q[d].y, bfhi(w), score);
      }
      score += xor32(score, lane);
      if (!sees)
        score = -__builtin_inff();
      const float top = fmaxf(M, wave_max(score));
      const float m_use = top == -__builtin_inff() ? 0.f : top;
      const float f = M == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f((M - m_use) * qscale);
      const float weight = sees ? __builtin_amdgcn_exp2f((score - m_use) * qscale) : 0.f;
      M = top;
      l *= f;
      o[0] *= f;
      o[1] *= f;
      for (uint32_t left = uint32_t(__ballot(sees)); left; left &= left - 1) {
        const int n = __builtin_ctz(left);
        const float w = __shfl(weight, n);
        l += w;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int d = lane + 64 * j;
          const uint16_t value = t0 + n == pos ? sh.kv_new[1][d] : p.cache.v[at + d * kBlock + n];
          o[j] = fmaf(w, bflo(value), o[j]);
        }
      }
    }
    to[h * D + lane] = o[0];
    to[h * D + lane + 64] = o[1];
    if (lane == 0) {
      sh.m[wave][h] = M;
      sh.l[wave][h] = l;
    }
  }
}

template <int G>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) void
paged_decode_kernel(DecodeParams p, float qscale) {
  __shared__ Shared<G> sh;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane >> 4, i = lane & 15;
  const int hkv = p.cache.kv_heads;

  // ---- which blocks are this workgroup's ----
  const int my_pos = lane < p.batch ? p.pos[lane] : -1;  // of the first 64 sequences
  const int my_blocks = blocks_at(p, my_pos);
  int total = __builtin_amdgcn_readlane(wave_scan(my_blocks), 63);
  int sequences = __builtin_popcountll(__ballot(my_blocks > 0));
  for (int b0 = 64; b0 < p.batch; b0 += 64) {
    const int n = b0 + lane < p.batch ? blocks_of(p, b0 + lane) : 0;
    total += __builtin_amdgcn_readlane(wave_scan(n), 63);
    sequences += __builtin_popcountll(__ballot(n > 0));
  }
  const int items = sequences * hkv;
  total *= hkv;
  // dispatch goes round the 8 XCDs: each takes neighbouring runs
  int run = int(blockIdx.x % 8) * (p.groups / 8) + int(blockIdx.x / 8);
  int b, place, nb, kvh, x, u, u1, each = 0, more = 0, r0 = 0, r1 = 0, step = 1;
  bool chunks = p.batch <= 64 && total <= kChunkBlocks && items <= kChunks;
  auto run_begin = [&](int g) { return g * each + min(g, more); };
  auto run_of = [&](int v) {
    return v < more * (each + 1) ? v / (each + 1) : more + (v - more * (each + 1)) / each;
  };
  // blocks of a chunk, at most: one a wave, kChunks chunks, kParts of a sequence
  int size = 0, count = 0;
  auto cut = [&](int blocks) { return (blocks + size - 1) / size; };
  auto chunks_of = [&](int blocks) {
    size = blocks;
    return count = __builtin_amdgcn_readlane(wave_scan(cut(my_blocks)), 63) * hkv;
  };
  if (chunks) {
    const int longest = int(wave_max(float(my_blocks)));
    const int least = max(max(kWaves, (longest + kParts - 1) / kParts), (total + kChunks - 1) / kChunks);
    // many short items leave a long one few chunks: runs share it out (at 2 * least
    // blocks a chunk, up to kChunks / 2 items always fit)
    if (items > kChunks / 2)
      chunks = chunks_of(2 * least) <= kChunks;
    for (int s = least; chunks && chunks_of(s) > kChunks; ++s) {
    }
  }
  if (chunks) {
    const int n = my_blocks;
    const int per = (count + 7) / 8;
    run = int(blockIdx.x % 8) * per + int(blockIdx.x / 8);
    if (int(blockIdx.x / 8) >= per ||
        !paged::find_item(p.batch, run, [&](int) { return cut(n) * hkv; }, b, place))
      return;
    nb = __builtin_amdgcn_readlane(n, b);
    const int of = cut(nb), j = place / hkv;
    kvh = place % hkv;
    step = hkv;
    r0 = run - j * hkv;
    r1 = r0 + (of - 1) * hkv;
    x = j * nb / of;
    u = x;
    u1 = (j + 1) * nb / of;
  } else {
    // units: an item's first kItemCost stand for what it takes to begin one
    total += items * kItemCost;
    each = total / p.groups;
    more = total % p.groups;  // the first `more` runs take one more
    u = run_begin(run);
    u1 = run_begin(run + 1);
    if (u >= u1)
      return;
    paged::find_item(
        p.batch, u,
        [&](int s) {
          const int n = blocks_of(p, s);
          return n ? (n + kItemCost) * hkv : 0;
        },
        b, place);
    nb = blocks_of(p, b);
    kvh = place / (nb + kItemCost);
    x = place - kvh * (nb + kItemCost) - kItemCost;  // (negative: begins an item)
  }

  while (true) {
    const int first = u - x, x1 = min(nb, x + u1 - u);  // blocks [x, x1) of item (b, kvh)
    if (x1 <= 0)
      return;  // not one block of the run's last item
    x = max(x, 0);
    const int pos = b < 64 ? __builtin_amdgcn_readlane(my_pos, b) : p.pos[b];
    const Span span = span_of(pos, p.window, p.sinks);
    const bool whole = x == 0 && x1 == nb;
    if (!chunks) {  // the runs that share the item
      r0 = run_of(first);
      r1 = run_of(first + nb - 1);
    }
    const int low = p.window > 0 ? pos - p.window : -1;  // visible: t > low or t < sinks

    // pages of this wave's blocks: lane j the one of block base + 4 j
    const int32_t *table = p.cache.table + size_t(b) * p.cache.table_stride;
    int v = x + wave, pages = 0, page_base = v;
    auto load_pages = [&](int v0) {
      const int vb = min(v0 + kWaves * lane, span.blocks - 1);
      pages = table[(span.block(vb) * kBlock) >> p.cache.shift];
      page_base = v0;
    };
    load_pages(v);

    // ---- the token's heads h = wave + 4 j: h < G query, G key, G + 1 value;
    // their inputs are on the way before K and V ----
    constexpr int kHeads = (G + 2 + kWaves - 1) / kWaves;
    const uint16_t *row = p.qkv + size_t(b) * p.qkv_stride;
    uint32_t pair[kHeads], gain2[kHeads];
    NormRope nr;
    load_rope(nr, p.cos + size_t(pos) * (D / 2), p.sin + size_t(pos) * (D / 2), lane);
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      const int h = min(wave + kWaves * j, G + 1);
      const size_t col = h < G ? size_t(kvh * G + h) * D : size_t(p.heads + (h - G) * hkv + kvh) * D;
      pair[j] = reinterpret_cast<const uint32_t *>(row + col)[lane];
      const uint16_t *gain = h < G ? p.q_norm : p.k_norm;
      gain2[j] = reinterpret_cast<const uint32_t *>(gain ? gain : row + col)[lane];
    }
    __builtin_amdgcn_sched_barrier(0);

    // A block's K and V go straight to LDS in whole KiB, into the wave's own
    // stage: K's 16-byte chunk c of key R to slot c ^ (4 (R / 8) + R % 4) of its
    // 256 bytes, V's chunk c of dim d to slot c ^ (d / 4 % 4) of its 64 (the
    // operand reads below then meet no bank twice, attn_tile.h).
    u32x4 *ks = sh.stage[wave][0], *vs = sh.stage[wave][1];
    int t0 = 0;
    bool held = false;
    auto fetch = [&](int vb) {
      if (vb - page_base >= 64 * kWaves)
        load_pages(vb);
      const int page = __builtin_amdgcn_readlane(pages, (vb - page_base) / kWaves);
      t0 = span.block(vb) * kBlock;
      held = p.cache.has(page);
      const size_t at = p.cache.at(held ? page : 0, kvh, t0 & ((1 << p.cache.shift) - 1));
      const auto rk = __builtin_amdgcn_make_buffer_rsrc(p.cache.k + at, 0, kBlock * D * 2, 0x00020000);
      const auto rv = __builtin_amdgcn_make_buffer_rsrc(p.cache.v + at, 0, kBlock * D * 2, 0x00020000);
#pragma unroll
      for (int q = 0; q < 8; ++q)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rk, (lds_ptr_t)(ks + 64 * q), 16,
            uint32_t((4 * q + r) * (D * 2) + (i ^ (4 * (q >> 1) + r)) * 16), 0, 0, kLoadAux);
#pragma unroll
      for (int q = 0; q < 8; ++q)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_ptr_t)(vs + 64 * q), 16,
                                                 uint32_t(q * 1024 + (lane >> 2) * 64 +
                                                          ((lane & 3) ^ (lane >> 4)) * 16),
                                                 0, 0, kLoadAux);
    };
    if (v < x1)
      fetch(v);

    // every head's chain side by side; the value's is not used
    float y0[kHeads], y1[kHeads];
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      y0[j] = bflo(pair[j]);
      y1[j] = bfhi(pair[j]);
      const bool normed = wave + kWaves * j < G ? p.q_norm : p.k_norm;
      const float scale =
          __builtin_amdgcn_rsqf(wave_sum(y0[j] * y0[j] + y1[j] * y1[j]) * (1.f / D) + p.eps);
      y0[j] *= normed ? scale * bflo(gain2[j]) : 1.f;
      y1[j] *= normed ? scale * bfhi(gain2[j]) : 1.f;
    }
    const float sgn = lane < 32 ? -1.f : 1.f;
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      const float a = sgn * xor32(y0[j], lane), c = sgn * xor32(y1[j], lane);
      y0[j] = fmaf(a, nr.s0, y0[j] * nr.c0);
      y1[j] = fmaf(c, nr.s1, y1[j] * nr.c1);
      const int h = wave + kWaves * j;
      if (h < G)
        reinterpret_cast<float2 *>(sh.q[h])[lane] = float2{y0[j], y1[j]};
      else if (h < G + 2)
        reinterpret_cast<uint32_t *>(sh.kv_new[h - G])[lane] =
            h == G ? pack_bf16(y0[j], y1[j]) : pair[j];
    }
    __syncthreads();
    // q operands: columns 0-7 the leading pieces of the heads, 8-15 the rests
    u32x4 qb[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 q2 = reinterpret_cast<const float2 *>(sh.q[min(i & 7, G - 1)])[16 * s + 4 * r + e];
        const uint32_t lead = pack_bf16(q2.x, q2.y);
        const uint32_t rest = pack_bf16(q2.x - bflo(lead), q2.y - bfhi(lead));
        w[e] = (i & 7) < G ? (i < 8 ? lead : rest) : 0u;
      }
      qb[s] = u32x4{w[0], w[1], w[2], w[3]};
    }

    // ---- the wave's blocks: one in registers, the next on its way to LDS ----
    float m_run = -__builtin_inff(), l_run = 0.f;
    f32x4 o[8];
#pragma unroll
    for (int dt = 0; dt < 8; ++dt)
      o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (; v < x1; v += kWaves) {
      wait_vmem();  // the block has landed
      __builtin_amdgcn_sched_barrier(0);
      u32x4 kr[8], vr[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        kr[j] = ks[attn::key_ofs(j >> 2, i) * 16 + ((4 * (j & 3) + r) ^ i)];
#pragma unroll
      for (int dt = 0; dt < 8; ++dt)
        vr[dt] = vs[64 * dt + 4 * i + (r ^ (i >> 2))];
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): it is in registers
      __builtin_amdgcn_sched_barrier(0);
      const int key0 = t0;
      // a block that holds the token's own slot, keys it does not see, or no page
      const bool part = !held || key0 + kBlock > pos || (key0 <= low && key0 + kBlock > p.sinks);
      uint32_t seen = 0xffu;  // bit e: key key0 + 8 r + e
      if (part) {
        seen = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int t = key0 + 8 * r + e;
          if (t == pos || (held && t < pos && (t > low || t < p.sinks)))
            seen |= 1u << e;
        }
#pragma unroll
        for (int T = 0; T < 2; ++T)
          if (key0 + attn::key_ofs(T, i) == pos)
#pragma unroll
            for (int s = 0; s < 4; ++s)
              kr[4 * T + s] = reinterpret_cast<const u32x4 *>(sh.kv_new[0])[4 * s + r];
        // values of keys that are not seen become zeros (their weights are: but
        // 0 times an infinity or NaN would count), the token's own come from LDS
        const int ep = pos - (key0 + 8 * r);
        uint32_t keep[4];
#pragma unroll
        for (int w = 0; w < 4; ++w)
          keep[w] = ((seen >> (2 * w)) & 1u ? 0x0000ffffu : 0u) |
                    ((seen >> (2 * w + 1)) & 1u ? 0xffff0000u : 0u);
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
          vr[dt] = u32x4{vr[dt].x & keep[0], vr[dt].y & keep[1], vr[dt].z & keep[2],
                         vr[dt].w & keep[3]};
          if (ep >= 0 && ep < 8)
            vr[dt] = attn::with_elem(vr[dt], ep, sh.kv_new[1][16 * dt + i]);
        }
      }
      if (v + kWaves < x1)
        fetch(v + kWaves);
      f32x4 st[2];
#pragma unroll
      for (int T = 0; T < 2; ++T)
        st[T] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int T = 0; T < 2; ++T)
          st[T] = attn::mfma(kr[4 * T + s], qb[s], st[T]);
      float sc[8], mx = -__builtin_inff();
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float raw = st[e >> 2][e & 3];
        sc[e] = (seen >> e) & 1u ? raw + paged::xor8(raw) : -__builtin_inff();
        mx = fmaxf(mx, sc[e]);
      }
      mx = max_halves(max_row_pairs(mx));
      const float m_new = fmaxf(m_run, mx);
      const float m_use = m_new == -__builtin_inff() ? 0.f : m_new;
      const float corr = __builtin_amdgcn_exp2f((m_run - m_use) * qscale);
      float ps = 0.f;
      uint32_t pw[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float p0 = __builtin_amdgcn_exp2f((sc[2 * q] - m_use) * qscale);
        const float p1 = __builtin_amdgcn_exp2f((sc[2 * q + 1] - m_use) * qscale);
        ps += p0;
        ps += p1;
        const uint32_t lead = pack_bf16(p0, p1);
        pw[q] = i < 8 ? lead : pack_bf16(p0 - bflo(lead), p1 - bfhi(lead));
      }
      l_run = l_run * corr + ps;
      m_run = m_new;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        o[dt] *= corr;
        o[dt] = attn::mfma(vr[dt], u32x4{pw[0], pw[1], pw[2], pw[3]}, o[dt]);
      }
    }
    u = first + x1;

    // ---- join the waves: each leaves its result in its own stage ----
    const float l_all = sum_halves(sum_row_pairs(l_run));
    f32x4 finite = {l_all * 0.f, 0.f, 0.f, 0.f};  // a NaN where some sum is not
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      f32x4 s;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[e] = o[dt][e] + paged::xor8(o[dt][e]);  // the pieces of P
        finite[e] = fmaf(s[e], 0.f, finite[e]);
      }
      if (i < G)
        reinterpret_cast<f32x4 *>(ks)[i * (D / 4) + 4 * dt + r] = s;
    }
    if (i < G && r == 0) {
      sh.m[wave][i] = m_run;
      sh.l[wave][i] = l_all;
    }
    if (__builtin_expect(__any(i < G && finite[0] + finite[1] + (finite[2] + finite[3]) != 0.f), 0))
      walk_odd<G>(p, qscale, span, table, kvh, pos, x + wave, x1, wave, sh);
    __syncthreads();
    uint16_t *out = p.out + size_t(b) * p.out_stride + size_t(kvh * G) * D;
    // slot 2 run + 1: the item begins in this run (its last one); 2 run: before it
    float *part = p.part + size_t(2 * run + (run == r0)) * (G * kPartFloats);
    if (threadIdx.x < G * D / 4) {  // one thread per head and 4 dims
      const int h = threadIdx.x / (D / 4), d = 4 * (threadIdx.x % (D / 4));
      float M = sh.m[0][h];
#pragma unroll
      for (int w = 1; w < kWaves; ++w)
        M = fmaxf(M, sh.m[w][h]);
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      float l = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = sh.m[w][h] == -__builtin_inff()
                            ? 0.f
                            : __builtin_amdgcn_exp2f((sh.m[w][h] - M) * qscale);
        acc += f * *reinterpret_cast<const f32x4 *>(
                       reinterpret_cast<const float *>(sh.stage[w][0]) + h * D + d);
        l = fmaf(f, sh.l[w][h], l);
      }
      if (whole) {
        acc *= 1.f / l;
        *reinterpret_cast<uint2 *>(out + h * D + d) =
            uint2{pack_bf16(acc[0], acc[1]), pack_bf16(acc[2], acc[3])};
      } else {
        // write-through (agent-scope) stores: visible to every XCD once complete
        const auto put = [&](int at, float lo, float hi) {
          __hip_atomic_store(reinterpret_cast<unsigned long long *>(part + h * kPartFloats + at),
                             (unsigned long long)f32_bits(hi) << 32 | f32_bits(lo),
                             __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        };
        put(d, acc[0], acc[1]);
        put(d + 2, acc[2], acc[3]);
        if (d == 0)
          put(D, M, l);
      }
    }
    // ---- append, by the workgroup that holds the last pass (the one that read
    // the block) ----
    if (x1 == nb) {
      const int page = table[pos >> p.cache.shift];
      const int slot = pos & ((1 << p.cache.shift) - 1);
      if (p.cache.has(page) && threadIdx.x < D / 8 + D) {
        if (threadIdx.x < D / 8) {
          reinterpret_cast<u32x4 *>(p.cache.k + p.cache.at(page, kvh, slot))[threadIdx.x] =
              reinterpret_cast<const u32x4 *>(sh.kv_new[0])[threadIdx.x];
        } else {
          const int d = threadIdx.x - D / 8;
          p.cache.v[p.cache.at(page, kvh, slot & ~(kBlock - 1)) + d * kBlock +
                    (slot & (kBlock - 1))] = sh.kv_new[1][d];
        }
      }
    }
    if (!whole) {
      // Arrival: every wave's stores have completed, then one increment. The
      // counter is the one of the run that holds the item's first pass; no other
      // shared item begins in that run. The last workgroup joins the parts.
      wait_vmem();
      __syncthreads();
      if (threadIdx.x == 0) {
        const int prev = __hip_atomic_fetch_add(&p.counters[r0 * kCounterStride], 1,
                                                __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sh.is_last = prev == (r1 - r0) / step;
      }
      __syncthreads();
      if (sh.is_last) {
        join_parts<G>(p, qscale, r0, r1, step, out, sh);
        if (threadIdx.x == 0)
          __hip_atomic_store(&p.counters[r0 * kCounterStride], 0, __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    if (u >= u1)
      return;
    __syncthreads();  // what the join read is written by the next item
    x = -kItemCost;
    if (++kvh == hkv) {
      kvh = 0;
      do
        nb = blocks_of(p, ++b);
      while (nb == 0);
    }
  }
}

template <int G> hipError_t launch_g(const DecodeParams &p, float qscale, hipStream_t s) {
  hipLaunchKernelGGL(paged_decode_kernel<G>, dim3(p.groups), dim3(64 * kWaves), 0, s, p, qscale);
  return hipGetLastError();
}

}  // namespace
}  // namespace yuear

extern "C" int32_t yuear_op_paged_attention_decode(
    const uint16_t *qkv, int64_t qkv_stride, const uint16_t *q_norm, const uint16_t *k_norm,
    float eps, const uint16_t *rope_cos, const uint16_t *rope_sin, int32_t positions,
    uint16_t *k_pages, uint16_t *v_pages, int32_t pages, int32_t page_slots, const int32_t *table,
    int32_t table_width, int32_t table_stride, const int32_t *pos, int32_t batch, int32_t heads,
    int32_t kv_heads, int32_t window, int32_t sinks, void *workspace, int64_t workspace_bytes,
    uint16_t *out, int64_t out_stride, void *stream) {
  using namespace yuear;
  if (batch < 0 || window < 0 || sinks < 0 || !paged::group_ok(heads, kv_heads))
    return int32_t(hipErrorInvalidValue);
  if (!batch)
    return int32_t(hipSuccess);
  DecodeParams p;
  if (!paged::make_cache(p.cache, k_pages, v_pages, pages, page_slots, table, table_width,
                         table_stride, kv_heads) ||
      !paged::aligned16(qkv) || !paged::aligned16(out) || !paged::aligned16(rope_cos) ||
      !paged::aligned16(rope_sin) || (q_norm && !paged::aligned16(q_norm)) ||
      (k_norm && !paged::aligned16(k_norm)) || !pos || positions < 1 || qkv_stride % 8 ||
      qkv_stride < int64_t(heads + 2 * kv_heads) * paged::D || out_stride % 8 ||
      out_stride < int64_t(heads) * paged::D || !paged::aligned16(workspace) ||
      workspace_bytes < yuear_op_paged_workspace_bytes(batch, heads, kv_heads, 0))
    return int32_t(hipErrorInvalidValue);
  p.limit = std::min(p.cache.capacity, positions);
  // blocks, and what begins items, are counted in 31 bits
  if ((long long)batch * kv_heads * (p.limit / paged::kBlock + 1 + kItemCost) > 0x3fffffffLL)
    return int32_t(hipErrorInvalidValue);
  p.qkv = qkv;
  p.qkv_stride = qkv_stride;
  p.q_norm = q_norm;
  p.k_norm = k_norm;
  p.eps = eps;
  p.cos = rope_cos;
  p.sin = rope_sin;
  p.pos = pos;
  p.batch = batch;
  p.heads = heads;
  p.window = window;
  p.sinks = sinks;
  p.groups = paged::kDecodeGroups;
  p.counters = static_cast<int32_t *>(workspace);
  p.part = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + paged::kCounterBytes);
  p.out = out;
  p.out_stride = out_stride;
  const float qscale = float(std::pow(double(paged::D), -0.5)) * attn::kLog2e;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (heads / kv_heads) {
  case 1: return int32_t(launch_g<1>(p, qscale, s));
  case 2: return int32_t(launch_g<2>(p, qscale, s));
  case 3: return int32_t(launch_g<3>(p, qscale, s));
  case 4: return int32_t(launch_g<4>(p, qscale, s));
  case 6: return int32_t(launch_g<6>(p, qscale, s));
  case 8: return int32_t(launch_g<8>(p, qscale, s));
  }
  return int32_t(hipErrorInvalidValue);
}
