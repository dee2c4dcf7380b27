// Host-side rules of the decode-attention launches: plain C++, no CUDA.
#pragma once
#include <stdint.h>

namespace kvmb {

constexpr uint32_t kAttendMaxSplits = 256;

// Fewest key chunks with which no chunk of the tcgen05 tree kernel has more than `most` page tiles, the room of its
// table of page boxes (0: more than kAttendMaxSplits). A chunk has no more page tiles than the list, however long the
// tail is. Longer lists are cut with the tail: chunks are even shares of all tiles.
inline uint32_t attend_least_chunks(uint64_t list_tiles, uint64_t tail_tiles, uint64_t most) {
    if (list_tiles <= most) return 1;
    const uint64_t all = list_tiles + tail_tiles;
    return all / most >= kAttendMaxSplits ? 0 : uint32_t(all / most + 1);
}

// Registers per thread that the warps of the tcgen05 kernel take (setmaxnreg). Narrow shape: 4 warps for copies and
// MMAs, 4 of softmax. Quantised pages: 4, 8 of softmax, 8 that decode.
constexpr int kAcNarrowIssue = 72, kAcNarrowSoftmax = 184;
constexpr int kAcQuantIssue = 64, kAcQuantSoftmax = 136, kAcQuantDecode = 72;

// Whether a kernel compiled to `regs` registers per thread can make that split: warps that ask for more than the launch
// brought would wait for ever.
constexpr bool ac_registers_fit(bool quant, int regs) {
    return quant ? regs <= kAcQuantSoftmax &&
                       640 * regs >= 128 * kAcQuantIssue + 256 * kAcQuantSoftmax + 256 * kAcQuantDecode
                 : regs <= kAcNarrowSoftmax && 256 * regs >= 128 * kAcNarrowIssue + 128 * kAcNarrowSoftmax;
}

}  // namespace kvmb
