// offsets.hpp — which arrays kernels reach by 32-bit byte offsets, decided on the
// host from their sizes alone.
#pragma once

#include <cstdint>

namespace nerf_hip {
namespace grouped {

// Whether `count` rows of 16-bit values, `ld` apart, are within 32-bit offsets from
// the first: an offset of 2^31 or more is taken for one beyond the array.
constexpr bool near(uint64_t count, uint64_t ld) { return count * ld * 2u < 1ull << 31; }

// Positions whose rows k_adapter_stream looks up at a time.
constexpr uint32_t kStreamChunk = 1024u;

// Whether k_adapter_stream reaches its outputs, whose widest rows are `widest` 16-bit
// values apart: an index names any of `count` rows, counted from the array's first;
// without one rows are counted from the chunk's first.
constexpr bool stream_outputs_near(bool index, uint64_t count, uint64_t widest) { return near(index ? count : kStreamChunk, widest); }

}  // namespace grouped
}  // namespace nerf_hip
