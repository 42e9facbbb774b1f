// Where a wave's lanes find their channels of a sequence tensor (glr_kernels.hip). Plain arithmetic, so that it can be
// checked without a device.
//
// A lane's bytes are at a base that is the same for the whole wave plus a 32-bit offset of its own, which the load
// extends without a sign: no offset may be negative.
#pragma once
#include <cstdint>

namespace fhc {
namespace seq {

// Whether a wave's columns may run from one sequence into the next, bs elements away: 63 sequences and one row of
// channels have to fit the offset. Sequences may overlap, or be one and the same (bs 0).
constexpr bool near_sequences(uint32_t b, uint32_t d, int64_t bs, uint32_t elem) {
    return b <= 1 || (bs >= 0 && bs < (1 << 30) / 64 / (int64_t)elem && (uint64_t)d * elem < 1ull << 31);
}
// The channel that the base is at, of the first lane's sequence. A wave that may run into the next sequence comes to
// channels before its first one there, so its base is the sequence's channel 0.
constexpr uint32_t base_channel(bool straddles, uint32_t first) { return straddles ? 0 : first; }
// bs in bytes
constexpr uint32_t lane_offset(uint32_t b, uint32_t ch, uint32_t b0, uint32_t c0, int64_t bs, uint32_t elem) {
    return (b - b0) * (uint32_t)bs + (ch - c0) * elem;
}

}  // namespace seq
}  // namespace fhc
