// Pages of a key-value cache, shared by the append (paged_cache.hip) and the
// attention kernels (paged_decode.hip, paged_prefill.hip).
//
// A page holds 2^shift slots of every kv head of one layer: K as rows
// [kv head][slot][128], V as the framework's 32-slot blocks
// [kv head][slot / 32][128][32] (attn_core.h). Slot s of a page and kv head
// starts at the same element of either array when s is a multiple of 32. Key t
// of a sequence lies in page table[t >> shift] of the sequence's table row; an
// entry outside [0, pages) stands for keys that are not there.
#pragma once
#include "common.h"

namespace yuear {
namespace paged {

constexpr int D = 128;
constexpr int kBlock = 32;
constexpr int kMaxGroup = 8;  // query heads of a kv head

struct Cache {
  uint16_t *k = nullptr, *v = nullptr;
  int pages = 0, shift = 0, kv_heads = 0;
  const int32_t *table = nullptr;  // [batch][table_stride]
  int table_stride = 0;
  int capacity = 0;  // positions of a table row (its width * slots, at most 2^31 - 256)
  __device__ __forceinline__ bool has(int page) const { return unsigned(page) < unsigned(pages); }
  // Element of slot `slot` (a multiple of 32 for V) of a page's kv head.
  __device__ __forceinline__ size_t at(int page, int kvh, int slot) const {
    return (((size_t(page) * kv_heads + kvh) << shift) + slot) * D;
  }
};

// Inclusive sums over the lanes of a wave (DPP: shifts inside the 16-lane rows,
// then the last lane of each row into the rows after it).
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15: rows 1, 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast 31: rows 2, 3
  return v;
}

// Item `target` of items numbered through the sequences, count(b) of them for
// sequence b: its sequence and place there; false past the last item. Every
// wave walks 64 sequences at a time, one per lane.
template <class F>
__device__ __forceinline__ bool find_item(int batch, int target, F &&count, int &seq, int &place) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int b0 = 0; b0 < batch; b0 += 64) {
    const int n = b0 + lane < batch ? count(b0 + lane) : 0;
    const int incl = wave_scan(n);
    const int total = __builtin_amdgcn_readlane(incl, 63);
    if (target < before + total) {
      const int at = __builtin_popcountll(__ballot(before + incl <= target));
      seq = b0 + at;
      place = target - before - __builtin_amdgcn_readlane(incl - n, at);
      return true;
    }
    before += total;
  }
  return false;
}

// Rows [first, first + n) of a prompt call that belong to sequence b, at
// positions from pos0 on; n is 0 for one that starts outside [0, limit), and
// rows at or past `limit` are left out.
struct Rows {
  int first, n, pos0;
};
__device__ __forceinline__ Rows sequence_rows(const int32_t *starts, const int32_t *pos0, int b,
                                              int rows, int limit) {
  const int s0 = min(max(starts[b], 0), rows), s1 = min(max(starts[b + 1], s0), rows);
  const int p = pos0[b];
  const bool in = p >= 0 && p < limit;
  return Rows{s0, in ? min(s1 - s0, limit - p) : 0, in ? p : 0};
}

// find_item() of items that each sequence's rows count: with the rows of the one found.
template <class F>
__device__ __forceinline__ bool find_rows(const int32_t *starts, const int32_t *pos0, int batch,
                                          int rows, int limit, int target, F &&count, int &seq,
                                          int &place, Rows &of) {
  Rows mine{0, 0, 0};  // of the lane's sequence of the last 64 looked at
  if (!find_item(
          batch, target,
          [&](int b) {
            mine = sequence_rows(starts, pos0, b, rows, limit);
            return count(mine);
          },
          seq, place))
    return false;
  const int lane = seq & 63;
  of = Rows{__builtin_amdgcn_readlane(mine.first, lane), __builtin_amdgcn_readlane(mine.n, lane),
            __builtin_amdgcn_readlane(mine.pos0, lane)};
  return true;
}

// Two values as bf16, rounded to the nearest (ties to even).
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2_t));
}

// Value of lane ^ 8 (lanes of a 16-lane row turned by half a row).
__device__ __forceinline__ float xor8(float v) { return dpp<0x128>(v); }

// ---- host-side checks ----
inline bool aligned16(const void *p) { return p && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline bool group_ok(int heads, int kv_heads) {
  if (kv_heads < 1 || heads < kv_heads || heads % kv_heads)
    return false;
  const int g = heads / kv_heads;
  return g == 1 || g == 2 || g == 3 || g == 4 || g == 6 || g == 8;
}
inline bool slots_ok(int slots) { return slots >= kBlock && (slots & (slots - 1)) == 0; }
// Fills the cache arguments; false where they are not valid.
inline bool make_cache(Cache &c, const uint16_t *k, const uint16_t *v, int pages, int slots,
                       const int32_t *table, int width, int stride, int kv_heads) {
  if (!aligned16(k) || !aligned16(v) || !table || pages < 1 || !slots_ok(slots) || width < 1 ||
      stride < width || kv_heads < 1)
    return false;
  c.k = const_cast<uint16_t *>(k);
  c.v = const_cast<uint16_t *>(v);
  c.pages = pages;
  c.shift = __builtin_ctz(unsigned(slots));
  c.kv_heads = kv_heads;
  c.table = table;
  c.table_stride = stride;
  const long long cap = (long long)width * slots;
  c.capacity = int(cap < 0x7fffff00LL ? cap : 0x7fffff00LL);  // a block past it counts in 31 bits
  return true;
}

}  // namespace paged
}  // namespace yuear
