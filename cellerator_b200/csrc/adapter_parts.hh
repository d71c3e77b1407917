// How a row's entries are shared out to the warps of a block in the adapters' kernel: by its length alone.  Plain C++, so that a test on
// the host can look it over for rows that are too long to try.  Places in a row are unsigned: the end of a row of almost 2^31 entries
// rounded up to whole parts is past 2^31.
#pragma once

#if defined(__CUDACC__)
#define CB200_BOTH_SIDES __host__ __device__ __forceinline__
#else
#define CB200_BOTH_SIDES inline
#endif

namespace cb200 {

constexpr int kRuns = 4;                // runs of 32 entries that a warp decodes at a time
constexpr int kSegment = 32 * kRuns;
constexpr int kMostParts = 32;          // of a row

// Entries of a part of a row of `len` entries, below 2^31: a multiple of a warp's segment.
CB200_BOTH_SIDES unsigned part_entries(unsigned len) {
    const unsigned even = (len + kMostParts - 1) / kMostParts, whole = (even + kSegment - 1) / kSegment * kSegment;
    return whole > 0u ? whole : kSegment;
}
// `share`: part_entries(len)
CB200_BOTH_SIDES unsigned parts_of(unsigned len, unsigned share) { return (len + share - 1) / share; }
CB200_BOTH_SIDES unsigned part_end(unsigned begin, unsigned len, unsigned share) { return begin + share < len ? begin + share : len; }

} // namespace cb200
