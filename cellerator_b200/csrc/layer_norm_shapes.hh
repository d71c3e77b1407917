// How the rows of a block kernel of the layer norm's forward pass lie over its threads.  Plain C++: the rule is looked over for every
// width where it is compiled and by a test on the host.
#pragma once

namespace cb200 {

constexpr int kWarpColumns = 8 * 32 * 4;             // 1,024: rows of up to so many belong to a group of lanes of a warp
constexpr int kRowThreads = 1024;                    // of a block, at most
constexpr int kRowColumns = 9 * 4 * kRowThreads;     // 36,864: rows of up to so many stay in a block's registers

// Quads of a thread, a block's width apart.  All but a thread's last are loaded and stored without a look at the row's end, so that they
// have to lie in the row.
constexpr int row_quads_of(int columns) { return columns <= 2048 ? 2 : columns <= 4 * 4 * kRowThreads ? 4 : columns <= 6 * 4 * kRowThreads ? 6 : 9; }
constexpr int row_threads_of(int columns) { return ((columns + 3) / 4 + row_quads_of(columns) * 32 - 1) / (row_quads_of(columns) * 32) * 32; }

// whether the row has room for all quads but each thread's last, and the threads room for the row
constexpr bool row_fits(int columns) {
    const int width = row_threads_of(columns) * 4, quads = row_quads_of(columns);
    return row_threads_of(columns) <= kRowThreads && (quads - 1) * width <= columns && columns <= quads * width;
}
constexpr bool rows_fit(int from, int to) {
    for (int columns = from; columns <= to; ++columns)
        if (!row_fits(columns)) return false;
    return true;
}
// With blocks of whole warps that holds for rows of more than 32 quads with two to a thread, 288 with four, 800 with six and 2,048 with
// nine; the rule above begins behind 256, 512, 4,096 and 6,144.
static_assert(rows_fit(kWarpColumns + 1, kRowColumns), "a thread's inner quads reach past the end of a row");

} // namespace cb200
