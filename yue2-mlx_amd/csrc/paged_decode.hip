// Attention of one new token per sequence over pages of keys and values, with
// the token's q/k RMSNorm, RoPE and append (paged.h, head_dim 128).
//
//   K[pos] = bf16(rope(norm(k))), V[pos] = v
//   out[h] = sum_t softmax_t(rope(norm(q))[h] . K[t] / sqrt(128)) V[t]
//
// over t <= pos with pos - t < window or t < sinks (window 0: all t), in pages
// that the table has. The bytes of the visible K and V bound it; the arithmetic
// is 2 G multiply-adds a byte.
//
// The work of a launch is the list of (sequence, kv head, pass), a pass being
// the next 4 visible 32-key blocks, one a wave. It is cut into equal runs, one
// per workgroup, whatever the lengths of the sequences: the positions are read
// on the device, so a captured launch serves every length. A workgroup walks the
// (sequence, kv head) items of its run one by one. An item that lies in one
// run is finished there; of one that several runs share, each workgroup leaves
// its running maximum, sum and weighted values in its slots of the workspace,
// and the one that arrives last joins them in order of the keys.
//
// Both products run on v_mfma_f32_16x16x32_bf16 as in attn_core.h (S^T = K q,
// O^T = V^T P^T, K rows permuted so that a lane's scores are its operand of the
// second product), with the G <= 8 heads in columns 0-7 as the leading bf16 piece
// of q and in columns 8-15 as the rest, so that q counts to 16 bits and P, split
// the same way, too: 2^-17 of each weight, at no more MFMAs than one piece each.
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

constexpr int kWaves = 4;

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
__device__ __forceinline__ int passes_of(const DecodeParams &p, int b) {
  const int pos = p.pos[b];
  if (pos < 0 || pos >= p.limit)
    return 0;
  return (span_of(pos, p.window, p.sinks).blocks + kWaves - 1) / kWaves;
}

template <int G> struct Shared {
  float q[G][D];
  uint16_t kv_new[2][D];
  float m[kWaves][G], l[kWaves][G], o[kWaves][G][D];
  int is_last;
};

// m (running maximum, in units of qscale * score), l, and o of one head of a
// workgroup's part of an item.
constexpr int kPartFloats = D + 2;

template <int G>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) void
paged_decode_kernel(DecodeParams p, float qscale) {
  __shared__ Shared<G> sh;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane >> 4, i = lane & 15;
  const int hkv = p.cache.kv_heads;

  // this workgroup's run [u0, u1) of the passes of all (sequence, kv head)
  int total = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    int n = b0 + lane < p.batch ? passes_of(p, b0 + lane) : 0;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1)
      n += __shfl_xor(n, s);
    total += __builtin_amdgcn_readfirstlane(n);
  }
  total *= hkv;
  const int each = total / p.groups, more = total % p.groups;  // the first `more` take one more
  auto run_begin = [&](int g) { return g * each + min(g, more); };
  auto run_of = [&](int u) {
    return u < more * (each + 1) ? u / (each + 1) : more + (u - more * (each + 1)) / each;
  };
  const int run = blockIdx.x;
  int u = run_begin(run);
  const int u1 = run_begin(run + 1);
  if (u >= u1)
    return;
  int b, place;
  paged::find_item(p.batch, u, [&](int s) { return passes_of(p, s) * hkv; }, b, place);
  int np = passes_of(p, b), kvh = place / np, x = place - kvh * np;

  while (true) {
    const int x1 = min(np, x + u1 - u);  // passes [x, x1) of item (b, kvh)
    const int pos = p.pos[b];
    const Span span = span_of(pos, p.window, p.sinks);
    const int item = u - x;  // first unit of the item
    const bool whole = x == 0 && x1 == np;

    // pages of this wave's blocks: lane j the one of pass x + j
    const int32_t *table = p.cache.table + size_t(b) * p.cache.table_stride;
    int pages = 0, page_base = x;
    auto load_pages = [&](int x0) {
      const int v = min(kWaves * (x0 + lane) + wave, span.blocks - 1);
      pages = table[(span.block(v) * kBlock) >> p.cache.shift];
      page_base = x0;
    };
    load_pages(x);

    // ---- the token's heads: h < G query head, G key, G + 1 value ----
    const uint16_t *row = p.qkv + size_t(b) * p.qkv_stride;
    for (int h = wave; h < G + 2; h += kWaves) {
      const size_t col = h < G ? size_t(kvh * G + h) * D : size_t(p.heads + (h - G) * hkv + kvh) * D;
      const uint32_t pair = reinterpret_cast<const uint32_t *>(row + col)[lane];
      if (h == G + 1) {
        reinterpret_cast<uint32_t *>(sh.kv_new[1])[lane] = pair;
        continue;
      }
      NormRope nr;
      load_rope(nr, p.cos + size_t(pos) * (D / 2), p.sin + size_t(pos) * (D / 2), lane);
      const uint16_t *gain = h < G ? p.q_norm : p.k_norm;
      float x0 = bflo(pair), x1 = bfhi(pair);
      if (gain) {
        load_gain(nr, gain, lane);
        const float scale = 1.0f / __builtin_sqrtf(wave_sum(x0 * x0 + x1 * x1) / float(D) + p.eps);
        x0 = x0 * scale * nr.g0;
        x1 = x1 * scale * nr.g1;
      }
      const float sgn = lane < 32 ? -1.f : 1.f;
      const float y0 = fmaf(sgn * xor32(x0, lane), nr.s0, x0 * nr.c0);
      const float y1 = fmaf(sgn * xor32(x1, lane), nr.s1, x1 * nr.c1);
      if (h < G)
        reinterpret_cast<float2 *>(sh.q[h])[lane] = float2{y0, y1};
      else
        reinterpret_cast<uint32_t *>(sh.kv_new[0])[lane] =
            uint32_t(f2bf(y0)) | (uint32_t(f2bf(y1)) << 16);
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
        uint16_t a = f2bf(q2.x), c = f2bf(q2.y);
        if (i >= 8) {
          a = f2bf(q2.x - bf2f(a));
          c = f2bf(q2.y - bf2f(c));
        }
        w[e] = (i & 7) < G ? uint32_t(a) | (uint32_t(c) << 16) : 0u;
      }
      qb[s] = u32x4{w[0], w[1], w[2], w[3]};
    }

    // ---- passes ----
    float m_run = -__builtin_inff(), l_run = 0.f;
    f32x4 o[8];
#pragma unroll
    for (int dt = 0; dt < 8; ++dt)
      o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (; x < x1; ++x, ++u) {
      const int v = kWaves * x + wave;
      if (v >= span.blocks)  // uniform in the wave
        continue;
      if (x - page_base >= 64)
        load_pages(x);
      const int page = __builtin_amdgcn_readlane(pages, x - page_base);
      const bool held = p.cache.has(page);
      const int t0 = span.block(v) * kBlock;
      const size_t at = p.cache.at(held ? page : 0, kvh, t0 & ((1 << p.cache.shift) - 1));
      const u32x4 *kc = reinterpret_cast<const u32x4 *>(p.cache.k + at);
      const u32x4 *vc = reinterpret_cast<const u32x4 *>(p.cache.v + at);
      u32x4 kr[8], vr[8];
#pragma unroll
      for (int T = 0; T < 2; ++T)
#pragma unroll
        for (int s = 0; s < 4; ++s)
          kr[4 * T + s] = kc[attn::key_ofs(T, i) * (D / 8) + 4 * s + r];
#pragma unroll
      for (int dt = 0; dt < 8; ++dt)
        vr[dt] = vc[(16 * dt + i) * (kBlock / 8) + r];
      // a block that holds the token's own slot, keys it does not see, or no page
      const int low = p.window > 0 ? pos - p.window : -1;  // visible: t > low or t < sinks
      const bool part = !held || t0 + kBlock > pos || (t0 <= low && t0 + kBlock > p.sinks);
      uint32_t seen = 0xffu;  // bit e: key t0 + 8 r + e
      if (part) {
        seen = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int t = t0 + 8 * r + e;
          if (t == pos || (held && t < pos && (t > low || t < p.sinks)))
            seen |= 1u << e;
        }
#pragma unroll
        for (int T = 0; T < 2; ++T)
          if (t0 + attn::key_ofs(T, i) == pos)
#pragma unroll
            for (int s = 0; s < 4; ++s)
              kr[4 * T + s] = reinterpret_cast<const u32x4 *>(sh.kv_new[0])[4 * s + r];
        // values of keys that are not seen become zeros (their weights are: but
        // 0 times an infinity or NaN would count), the token's own come from LDS
        const int ep = pos - (t0 + 8 * r);
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
      f32x4 st[2];
#pragma unroll
      for (int T = 0; T < 2; ++T) {
        st[T] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 4; ++s)
          st[T] = attn::mfma(kr[4 * T + s], qb[s], st[T]);
      }
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
        uint16_t a = f2bf(p0), c = f2bf(p1);
        if (i >= 8) {
          a = f2bf(p0 - bf2f(a));
          c = f2bf(p1 - bf2f(c));
        }
        pw[q] = uint32_t(a) | (uint32_t(c) << 16);
      }
      l_run = l_run * corr + ps;
      m_run = m_new;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        o[dt] *= corr;
        o[dt] = attn::mfma(vr[dt], u32x4{pw[0], pw[1], pw[2], pw[3]}, o[dt]);
      }
    }

    // ---- join the waves ----
    const float l_all = sum_halves(sum_row_pairs(l_run));
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      f32x4 s;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s[e] = o[dt][e] + paged::xor8(o[dt][e]);  // the pieces of P
      if (i < G)
        *reinterpret_cast<f32x4 *>(&sh.o[wave][i][16 * dt + 4 * r]) = s;
    }
    if (i < G && r == 0) {
      sh.m[wave][i] = m_run;
      sh.l[wave][i] = l_all;
    }
    __syncthreads();
    // slot 2 run + 1: the item begins in this run (its last one); 2 run: before it
    float *part = p.part + size_t(2 * run + (item >= run_begin(run))) * (G * kPartFloats);
    for (int e = threadIdx.x; e < G * D; e += 64 * kWaves) {
      const int h = e / D;
      float M = sh.m[0][h];
#pragma unroll
      for (int w = 1; w < kWaves; ++w)
        M = fmaxf(M, sh.m[w][h]);
      float acc = 0.f, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = sh.m[w][h] == -__builtin_inff()
                            ? 0.f
                            : __builtin_amdgcn_exp2f((sh.m[w][h] - M) * qscale);
        acc = fmaf(f, sh.o[w][h][e % D], acc);
        l = fmaf(f, sh.l[w][h], l);
      }
      if (whole) {
        p.out[size_t(b) * p.out_stride + size_t(kvh * G) * D + e] = f2bf(acc / l);
        continue;
      }
      // write-through (agent-scope) stores: visible to every XCD once complete
      __hip_atomic_store(&part[h * kPartFloats + e % D], acc, __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
      if (e % D == 0) {
        __hip_atomic_store(&part[h * kPartFloats + D], M, __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(&part[h * kPartFloats + D + 1], l, __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    // ---- append, by the workgroup that holds the last pass (the one that read
    // the block) ----
    if (x1 == np) {
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
      const int r0 = run_of(item), r1 = run_of(item + np - 1);
      wait_vmem();
      __syncthreads();
      if (threadIdx.x == 0) {
        const int prev = __hip_atomic_fetch_add(&p.counters[r0 * kCounterStride], 1,
                                                __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sh.is_last = prev == r1 - r0;
      }
      __syncthreads();
      if (sh.is_last) {
        const auto slot_of = [&](int g) { return size_t(2 * g + (g == r0)) * (G * kPartFloats); };
        for (int e = threadIdx.x; e < G * D; e += 64 * kWaves) {
          const int h = e / D;
          const auto load = [&](int g, int f) {
            return __hip_atomic_load(&p.part[slot_of(g) + h * kPartFloats + f], __ATOMIC_RELAXED,
                                     __HIP_MEMORY_SCOPE_AGENT);
          };
          float M = -__builtin_inff(), acc = 0.f, l = 0.f;
          for (int g = r0; g <= r1; ++g) {
            const float m = load(g, D), lg = load(g, D + 1), og = load(g, e % D);
            if (m == -__builtin_inff())
              continue;
            const float top = fmaxf(M, m);
            const float f0 = M == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((M - top) * qscale);
            const float f1 = __builtin_amdgcn_exp2f((m - top) * qscale);
            acc = fmaf(f1, og, acc * f0);
            l = fmaf(f1, lg, l * f0);
            M = top;
          }
          p.out[size_t(b) * p.out_stride + size_t(kvh * G) * D + e] = f2bf(acc / l);
        }
        if (threadIdx.x == 0)
          __hip_atomic_store(&p.counters[r0 * kCounterStride], 0, __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    if (u >= u1)
      return;
    __syncthreads();  // the join has read what the next item writes
    x = 0;
    if (++kvh == hkv) {
      kvh = 0;
      do
        np = passes_of(p, ++b);
      while (np == 0);
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
  // passes are counted in 31 bits
  if ((long long)batch * kv_heads * (p.limit / (paged::kBlock * kWaves) + 1) > 0x3fffffffLL)
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
