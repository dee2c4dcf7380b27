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

}  // namespace kvmb
