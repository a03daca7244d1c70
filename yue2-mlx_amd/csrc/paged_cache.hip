// Pages of a key-value cache: the append of prompt rows, page copies, and the
// host bookkeeping of which sequence holds which page.
#include <algorithm>
#include <cstring>
#include <map>
#include <memory>
#include <mutex>
#include <set>
#include <vector>

#include "../../include/yuear.h"
#include "abi_util.h"
#include "attn_core.h"
#include "common.h"
#include "paged.h"

namespace yuear {
namespace {

using paged::Cache;
using paged::D;
using paged::kBlock;

struct AppendParams {
  const uint16_t *qkv = nullptr;
  long long qkv_stride = 0;
  const uint16_t *q_norm = nullptr, *k_norm = nullptr;
  float eps = 0.f;
  const uint16_t *cos = nullptr, *sin = nullptr;
  Cache cache;
  const int32_t *starts = nullptr, *pos0 = nullptr;
  int batch = 0, rows = 0, heads = 0, limit = 0;
  uint16_t *q = nullptr;
  long long q_stride = 0;
};

constexpr int kHeadsPerGroup = 3;

__device__ __forceinline__ void unpack8(u32x4 w, float (&x)[8]) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bflo(v[i]);
    x[2 * i + 1] = bfhi(v[i]);
  }
}
__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  return u32x4{paged::pack_bf16(x[0], x[1]), paged::pack_bf16(x[2], x[3]),
               paged::pack_bf16(x[4], x[5]), paged::pack_bf16(x[6], x[7])};
}

// q/k RMSNorm + RoPE of prompt rows, q out, K and V into their pages. A
// workgroup takes one 32-slot block of one sequence and 3 of the qkv heads; a
// wave takes 8 of the block's rows, 16 lanes a row with 8 dims each (dims 8 c of
// chunk c, whose rotation partner 8 c +- 64 lies in lane ^ 8). All arithmetic is
// in 32 bits and each value is rounded to bf16 once, where it is stored. The 8
// keys of a wave are one 16-byte piece of V per dim, turned through LDS. Bound by
// latency where there are few rows and by HBM where there are many. Rows of 40
// heads, 3000 of them / 7 sequences of 19 to 301 with 32 heads (us): 2 heads a
// workgroup 17.5 / 7.3, 3 heads 15.3 / 7.6 (62 MB at 4.1 TB/s), 4 heads 15.8 / 8.6;
// 8 heads, each loaded after the one before it, 17.4 / 12.5.
__global__ __launch_bounds__(256) void paged_append_kernel(AppendParams p) {
  __shared__ uint32_t turn[4][8][D / 2 + 1];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int b, place;
  paged::Rows r;
  if (!paged::find_rows(
          p.starts, p.pos0, p.batch, p.rows, p.limit, blockIdx.x,
          [](const paged::Rows &of) {
            return of.n ? (of.pos0 + of.n - 1) / kBlock - of.pos0 / kBlock + 1 : 0;
          },
          b, place, r))
    return;
  const int block = r.pos0 / kBlock + place;
  const int lo = max(block * kBlock, r.pos0);
  const int hi = min(block * kBlock + kBlock, r.pos0 + r.n);  // positions [lo, hi)
  const int first = block * kBlock + 8 * wave;
  if (first >= hi || first + 8 <= lo)
    return;  // (no barrier below)
  const int kv = p.cache.kv_heads, h0 = blockIdx.y * kHeadsPerGroup;
  const int h1 = min(h0 + kHeadsPerGroup, p.heads + 2 * kv);
  const int slot = (block * kBlock) & ((1 << p.cache.shift) - 1);
  const int chunk = lane & 15;
  u32x4 all[kHeadsPerGroup][2];  // every load is on its way before the first use
  int pos[2];
  float c[2][8], s[2][8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    pos[i] = first + 4 * i + (lane >> 4);
    const int in = min(max(pos[i], lo), hi - 1);
    const uint16_t *row =
        p.qkv + (size_t(r.first) + (in - r.pos0)) * p.qkv_stride + size_t(h0) * D + 8 * chunk;
#pragma unroll
    for (int h = 0; h < kHeadsPerGroup; ++h)
      if (h0 + h < h1)
        all[h][i] = *reinterpret_cast<const u32x4 *>(row + h * D);
    unpack8(*reinterpret_cast<const u32x4 *>(p.cos + size_t(in) * (D / 2) + 8 * (chunk & 7)), c[i]);
    unpack8(*reinterpret_cast<const u32x4 *>(p.sin + size_t(in) * (D / 2) + 8 * (chunk & 7)), s[i]);
    if (chunk < 8)  // first half: x c - partner s; second half: x c + partner s
#pragma unroll
      for (int e = 0; e < 8; ++e)
        s[i][e] = -s[i][e];
  }
  const int page = p.cache.table[size_t(b) * p.cache.table_stride +
                                 ((block * kBlock) >> p.cache.shift)];
  const bool held = p.cache.has(page);
#pragma unroll
  for (int n = 0; n < kHeadsPerGroup; ++n) {
    const int h = h0 + n;
    if (h >= h1)
      break;
    const u32x4(&w)[2] = all[n];
    if (h < p.heads + kv) {
      const bool is_q = h < p.heads;
      const uint16_t *gain = is_q ? p.q_norm : p.k_norm;
      float g[8];
      if (gain)
        unpack8(*reinterpret_cast<const u32x4 *>(gain + 8 * chunk), g);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x[8];
        unpack8(w[i], x);
        if (gain) {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            ss += x[e] * x[e];
          const float scale = __builtin_amdgcn_rsqf(row_sum16(ss) * (1.f / D) + p.eps);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            x[e] = x[e] * scale * g[e];
        }
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          y[e] = fmaf(paged::xor8(x[e]), s[i][e], x[e] * c[i][e]);
        if (pos[i] < lo || pos[i] >= hi)
          continue;
        if (is_q)
          *reinterpret_cast<u32x4 *>(p.q + (size_t(r.first) + (pos[i] - r.pos0)) * p.q_stride +
                                     h * D + 8 * chunk) = pack8(y);
        else if (held)
          *reinterpret_cast<u32x4 *>(p.cache.k + p.cache.at(page, h - p.heads, slot) +
                                     size_t(pos[i] - block * kBlock) * D + 8 * chunk) = pack8(y);
      }
      continue;
    }
    if (!held)
      break;
    // V: rows of 8 keys -> per dim a piece of 8 keys. The wave's own rows only,
    // so its LDS accesses, which stay in order, need no barrier.
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t *to = &turn[wave][4 * i + (lane >> 4)][4 * chunk];
      to[0] = w[i].x;
      to[1] = w[i].y;
      to[2] = w[i].z;
      to[3] = w[i].w;
    }
    __builtin_amdgcn_wave_barrier();
    uint32_t t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      t[e] = turn[wave][e][lane];  // dims 2 lane, 2 lane + 1 of key e
    __builtin_amdgcn_wave_barrier();
    uint16_t *to = p.cache.v + p.cache.at(page, h - p.heads - kv, slot) + 2 * lane * kBlock +
                   8 * wave;
    if (first >= lo && first + 8 <= hi) {
      uint32_t a[4], b2[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = __builtin_amdgcn_perm(t[2 * e + 1], t[2 * e], 0x05040100u);
        b2[e] = __builtin_amdgcn_perm(t[2 * e + 1], t[2 * e], 0x07060302u);
      }
      *reinterpret_cast<u32x4 *>(to) = u32x4{a[0], a[1], a[2], a[3]};
      *reinterpret_cast<u32x4 *>(to + kBlock) = u32x4{b2[0], b2[1], b2[2], b2[3]};
    } else {  // the other slots of the piece keep their contents
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (first + e >= lo && first + e < hi) {
          to[e] = uint16_t(t[e]);
          to[kBlock + e] = uint16_t(t[e] >> 16);
        }
    }
  }
}

// ---- page copies ----
// A thread copies one 16-byte chunk of a page of one layer's K or V. Bound by HBM;
// what hides its latency is many short workgroups, and stores that do not stay in
// L2. One page of 128 KiB to 7 others / 90 pages to 90, in 28 layers (59 MB / 1.3 GB;
// us): 9.8 / 215 (6.1 TB/s); with ordinary stores 12.8 / 222, with those and four
// chunks a thread 13.7 / 256.
constexpr int kPairs = 240;  // (source, destination) pairs of a launch, in its arguments
struct CopyParams {
  uint16_t *k = nullptr, *v = nullptr;
  long long layer_stride = 0, page_elems = 0;
  int32_t src[kPairs], dst[kPairs];
};
__global__ __launch_bounds__(256) void pages_copy_kernel(CopyParams p) {
  uint16_t *base = (blockIdx.z & 1 ? p.v : p.k) + size_t(blockIdx.z >> 1) * p.layer_stride;
  const u32x4 *from =
      reinterpret_cast<const u32x4 *>(base + size_t(p.src[blockIdx.y]) * p.page_elems);
  u32x4 *to = reinterpret_cast<u32x4 *>(base + size_t(p.dst[blockIdx.y]) * p.page_elems);
  const long long c = (long long)blockIdx.x * 256 + threadIdx.x;
  if (c < p.page_elems / 8)
    __builtin_nontemporal_store(from[c], to + c);
}

hipError_t copy_pages(uint16_t *k, uint16_t *v, int layers, long long layer_stride, int pages,
                      int kv_heads, int slots, const int32_t *src, const int32_t *dst, int n,
                      hipStream_t s) {
  const long long page_elems = (long long)kv_heads * slots * D;
  if (layers < 1 || layers > 32767 || pages < 1 || kv_heads < 1 || !paged::slots_ok(slots) ||
      n < 0 || !paged::aligned16(k) || !paged::aligned16(v) || (n && (!src || !dst)) ||
      layer_stride % 8 || (layers > 1 && layer_stride < page_elems * pages))
    return hipErrorInvalidValue;
  if (!n)
    return hipSuccess;
  // every copy reads what was there before the call: no page is written twice,
  // and none that is read is written
  std::vector<int32_t> to(dst, dst + n);
  std::sort(to.begin(), to.end());
  if (to.front() < 0 || to.back() >= pages ||
      std::adjacent_find(to.begin(), to.end()) != to.end())
    return hipErrorInvalidValue;
  for (int i = 0; i < n; ++i)
    if (src[i] < 0 || src[i] >= pages || std::binary_search(to.begin(), to.end(), src[i]))
      return hipErrorInvalidValue;
  CopyParams p;
  p.k = k;
  p.v = v;
  p.layer_stride = layer_stride;
  p.page_elems = page_elems;
  const long long chunks = (page_elems / 8 + 255) / 256;
  if (chunks > 0x7fffffffLL)
    return hipErrorInvalidValue;
  for (int i = 0; i < n; i += kPairs) {
    const int m = std::min(kPairs, n - i);
    std::memcpy(p.src, src + i, m * sizeof(int32_t));
    std::memcpy(p.dst, dst + i, m * sizeof(int32_t));
    hipLaunchKernelGGL(pages_copy_kernel, dim3(unsigned(chunks), m, 2 * layers), dim3(256), 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
      return e;
  }
  return hipSuccess;
}

}  // namespace
}  // namespace yuear

// Pages of a pool at most: one layer's smallest ones (16 KiB) would take 512 GiB. The
// bookkeeping of 2^31 would take all of the host's memory.
constexpr int32_t kMaxPages = 1 << 25;

// Host bookkeeping of a pool of pages. Pages are handed out lowest first, so
// the same calls give the same pages.
struct yuear_pages {
  struct Sequence {
    std::vector<int32_t> pages;  // -1: given back by trim
    int32_t length = 0, trimmed = 0;  // trimmed: the length when pages were last given back
  };
  std::mutex busy;
  int32_t slots = 0;
  std::vector<int32_t> holders;  // sequences that hold each page
  std::set<int32_t> unused;
  std::map<int32_t, Sequence> sequences;
  int32_t next = 0;

  Sequence &at(int32_t id) {
    auto it = sequences.find(id);
    if (it == sequences.end())
      yuear::invalid("no such sequence");
    return it->second;
  }
  int32_t take() {
    const int32_t page = *unused.begin();
    unused.erase(unused.begin());
    holders[page] = 1;
    return page;
  }
  void give(int32_t page) {
    if (page >= 0 && --holders[page] == 0)
      unused.insert(page);
  }
};

namespace {
template <class F> yuear_status with_pool(yuear_pages *pool, char **error_json, F &&f) {
  return yuear::guarded(error_json, [&] {
    if (!pool)
      yuear::invalid("pool is required");
    std::lock_guard<std::mutex> lock(pool->busy);
    f();
  });
}
}  // namespace

extern "C" {

yuear_status yuear_pages_create(int32_t pages, int32_t page_slots, yuear_pages **out,
                                char **error_json) {
  if (out)
    *out = nullptr;
  return yuear::guarded(error_json, [&] {
    if (!out)
      yuear::invalid("output pointer is required");
    if (pages < 1)
      yuear::invalid("a pool needs at least one page");
    if (pages > kMaxPages)
      yuear::invalid("a pool holds at most 2^25 pages");
    if (!yuear::paged::slots_ok(page_slots))
      yuear::invalid("page slots must be a power of two of at least 32");
    auto pool = std::make_unique<yuear_pages>();
    pool->slots = page_slots;
    pool->holders.assign(pages, 0);
    for (int32_t p = 0; p < pages; ++p)
      pool->unused.insert(pool->unused.end(), p);
    *out = pool.release();
  });
}

void yuear_pages_destroy(yuear_pages *pool) { delete pool; }

yuear_status yuear_pages_open(yuear_pages *pool, int32_t *sequence, char **error_json) {
  return with_pool(pool, error_json, [&] {
    if (!sequence)
      yuear::invalid("output pointer is required");
    if (pool->next == INT32_MAX)
      throw yuear::Error("RuntimeError", "out of sequence ids");
    pool->sequences[pool->next];
    *sequence = pool->next++;
  });
}

yuear_status yuear_pages_fork(yuear_pages *pool, int32_t sequence, int32_t *fork,
                              char **error_json) {
  return with_pool(pool, error_json, [&] {
    if (!fork)
      yuear::invalid("output pointer is required");
    if (pool->next == INT32_MAX)
      throw yuear::Error("RuntimeError", "out of sequence ids");
    yuear_pages::Sequence copy = pool->at(sequence);
    auto &held = pool->sequences[pool->next] = std::move(copy);
    for (int32_t page : held.pages)
      if (page >= 0)
        ++pool->holders[page];
    *fork = pool->next++;
  });
}

yuear_status yuear_pages_extend(yuear_pages *pool, int32_t sequence, int32_t tokens,
                                int32_t *copy_src, int32_t *copy_dst, char **error_json) {
  return with_pool(pool, error_json, [&] {
    if (!copy_src || !copy_dst)
      yuear::invalid("output pointers are required");
    *copy_src = *copy_dst = -1;
    auto &s = pool->at(sequence);
    if (tokens < 0)
      yuear::invalid("tokens must not be negative");
    if (tokens > INT32_MAX - pool->slots - s.length)
      yuear::invalid("the sequence would pass 2^31 positions");
    if (!tokens)
      return;
    // the last page takes the first new tokens: its own copy where others hold it
    const bool own = s.length % pool->slots && pool->holders[s.pages.back()] > 1;
    const size_t need = size_t(s.length + tokens + pool->slots - 1) / pool->slots;
    const size_t more = need - s.pages.size() + (own ? 1 : 0);
    if (more > pool->unused.size())
      throw yuear::Error("MemoryError", "out of pages");
    s.pages.reserve(need);
    if (own) {
      *copy_src = s.pages.back();
      *copy_dst = pool->take();
      pool->give(*copy_src);
      s.pages.back() = *copy_dst;
    }
    while (s.pages.size() < need)
      s.pages.push_back(pool->take());
    s.length += tokens;
  });
}

yuear_status yuear_pages_truncate(yuear_pages *pool, int32_t sequence, int32_t length,
                                  char **error_json) {
  return with_pool(pool, error_json, [&] {
    auto &s = pool->at(sequence);
    if (length < 0 || length > s.length)
      yuear::invalid("length must be in [0, the sequence's length]");
    if (length < s.trimmed)
      yuear::invalid("pages before this length were given back by trim");
    const size_t keep = size_t(length + pool->slots - 1) / pool->slots;
    while (s.pages.size() > keep) {
      pool->give(s.pages.back());
      s.pages.pop_back();
    }
    s.length = length;
  });
}

yuear_status yuear_pages_trim(yuear_pages *pool, int32_t sequence, int32_t window, int32_t sinks,
                              char **error_json) {
  return with_pool(pool, error_json, [&] {
    auto &s = pool->at(sequence);
    if (window < 1 || sinks < 0)
      yuear::invalid("window must be positive and sinks must not be negative");
    // the next token, at position `length`, sees no key before length - window + 1
    const long long low = (long long)s.length - window + 1;
    bool gave = false;
    for (size_t j = 0; (long long)(j + 1) * pool->slots <= low; ++j)
      if ((long long)j * pool->slots >= sinks && s.pages[j] >= 0) {
        pool->give(s.pages[j]);
        s.pages[j] = -1;
        gave = true;
      }
    if (gave)
      s.trimmed = s.length;
  });
}

yuear_status yuear_pages_close(yuear_pages *pool, int32_t sequence, char **error_json) {
  return with_pool(pool, error_json, [&] {
    auto &s = pool->at(sequence);
    for (int32_t page : s.pages)
      pool->give(page);
    pool->sequences.erase(sequence);
  });
}

yuear_status yuear_pages_compact(yuear_pages *pool, int32_t *copy_src, int32_t *copy_dst,
                                 int32_t *n, char **error_json) {
  if (n)
    *n = 0;
  return with_pool(pool, error_json, [&] {
    if (!copy_src || !copy_dst || !n)
      yuear::invalid("output pointers are required");
    const int32_t pages = int32_t(pool->holders.size());
    const int32_t live = pages - int32_t(pool->unused.size());
    std::vector<int32_t> to(pages);
    for (int32_t p = 0; p < pages; ++p)
      to[p] = p;
    auto hole = pool->unused.begin();
    int32_t moved = 0;
    for (int32_t p = live; p < pages; ++p)
      if (pool->holders[p]) {  // as many as there are unused pages below `live`
        copy_src[moved] = p;
        copy_dst[moved] = to[p] = *hole++;
        ++moved;
      }
    std::set<int32_t> unused;
    for (int32_t p = live; p < pages; ++p)
      unused.insert(unused.end(), p);
    for (int32_t i = 0; i < moved; ++i) {
      pool->holders[copy_dst[i]] = pool->holders[copy_src[i]];
      pool->holders[copy_src[i]] = 0;
    }
    pool->unused.swap(unused);
    for (auto &s : pool->sequences)
      for (int32_t &page : s.second.pages)
        if (page >= 0)
          page = to[page];
    *n = moved;
  });
}

yuear_status yuear_pages_table(yuear_pages *pool, const int32_t *sequences, int32_t n,
                               int32_t width, int32_t *table, char **error_json) {
  return with_pool(pool, error_json, [&] {
    if (n < 0 || width < 0 || (n && (!sequences || (width && !table))))
      yuear::invalid("sequences and a table are required");
    for (int32_t i = 0; i < n; ++i)
      if (pool->at(sequences[i]).pages.size() > size_t(width))
        yuear::invalid("a sequence has more pages than the table is wide");
    for (int32_t i = 0; i < n; ++i) {
      const auto &pages = pool->at(sequences[i]).pages;
      int32_t *row = table + size_t(i) * width;
      std::copy(pages.begin(), pages.end(), row);
      std::fill(row + pages.size(), row + width, -1);
    }
  });
}

int32_t yuear_pages_length(yuear_pages *pool, int32_t sequence) {
  if (!pool)
    return -1;
  std::lock_guard<std::mutex> lock(pool->busy);
  auto it = pool->sequences.find(sequence);
  return it == pool->sequences.end() ? -1 : it->second.length;
}

int32_t yuear_pages_unused(yuear_pages *pool) {
  if (!pool)
    return -1;
  std::lock_guard<std::mutex> lock(pool->busy);
  return int32_t(pool->unused.size());
}

int32_t yuear_op_pages_copy(uint16_t *k, uint16_t *v, int32_t layers, int64_t layer_stride,
                            int32_t pages, int32_t kv_heads, int32_t page_slots,
                            const int32_t *src, const int32_t *dst, int32_t n, void *stream) {
  try {
    return int32_t(yuear::copy_pages(k, v, layers, layer_stride, pages, kv_heads, page_slots, src,
                                     dst, n, static_cast<hipStream_t>(stream)));
  } catch (...) {  // the check's list of pages
    return int32_t(hipErrorOutOfMemory);
  }
}

int32_t yuear_op_paged_append(const uint16_t *qkv, int64_t qkv_stride, const uint16_t *q_norm,
                              const uint16_t *k_norm, float eps, const uint16_t *rope_cos,
                              const uint16_t *rope_sin, int32_t positions, uint16_t *k_pages,
                              uint16_t *v_pages, int32_t pages, int32_t page_slots,
                              const int32_t *table, int32_t table_width, int32_t table_stride,
                              const int32_t *starts, const int32_t *pos0, int32_t batch,
                              int32_t rows, int32_t heads, int32_t kv_heads, uint16_t *q_out,
                              int64_t q_stride, void *stream) {
  using namespace yuear;
  AppendParams p;
  if (batch < 0 || rows < 0 || !paged::group_ok(heads, kv_heads))
    return int32_t(hipErrorInvalidValue);
  if (!batch || !rows)
    return int32_t(hipSuccess);
  if (!paged::make_cache(p.cache, k_pages, v_pages, pages, page_slots, table, table_width,
                         table_stride, kv_heads) ||
      !paged::aligned16(qkv) || !paged::aligned16(q_out) || !paged::aligned16(rope_cos) ||
      !paged::aligned16(rope_sin) || (q_norm && !paged::aligned16(q_norm)) ||
      (k_norm && !paged::aligned16(k_norm)) || !starts || !pos0 || positions < 1 ||
      qkv_stride % 8 || qkv_stride < int64_t(heads + 2 * kv_heads) * paged::D || q_stride % 8 ||
      q_stride < int64_t(heads) * paged::D)
    return int32_t(hipErrorInvalidValue);
  p.qkv = qkv;
  p.qkv_stride = qkv_stride;
  p.q_norm = q_norm;
  p.k_norm = k_norm;
  p.eps = eps;
  p.cos = rope_cos;
  p.sin = rope_sin;
  p.starts = starts;
  p.pos0 = pos0;
  p.batch = batch;
  p.rows = rows;
  p.heads = heads;
  p.limit = std::min(p.cache.capacity, positions);
  p.q = q_out;
  p.q_stride = q_stride;
  // n rows from any position cover at most (n - 2) / 32 + 2 blocks
  const long long blocks = (long long)rows / paged::kBlock + 2LL * std::min(batch, rows);
  const int groups = (heads + 2 * kv_heads + kHeadsPerGroup - 1) / kHeadsPerGroup;
  if (groups > 65535)
    return int32_t(hipErrorInvalidValue);
  hipLaunchKernelGGL(paged_append_kernel, dim3(unsigned(blocks), groups), dim3(256), 0,
                     static_cast<hipStream_t>(stream), p);
  return int32_t(hipGetLastError());
}

}  // extern "C"
