// The caller's workspace of the paged attention: arrival counters of the decode
// form, one for each of its workgroups (zero between calls), then partials. One
// offset for every call, so that calls of unlike shapes may take turns on it.
#pragma once
#include <cstddef>

#include "../../include/yuear.h"
#include "kernels.h"

namespace yuear {
namespace paged {

constexpr int kDecodeGroups = 512;  // workgroups of a decode launch
constexpr size_t kCounterBytes = size_t(kDecodeGroups) * kCounterStride * 4;
static_assert(kCounterBytes == YUEAR_PAGED_COUNTER_BYTES, "what the caller zeroes");

}  // namespace paged
}  // namespace yuear
