// Layer norm over the rows of a dense matrix, with the activation and the dropout that follow it in the same pass:
//     u = (x - mean) / sqrt(var + eps),  y = drop(act(gamma u + beta)).
// Mean and variance are sums in fp32 over values that stay in registers, of what the values differ from a number next to their mean, so
// that a row far from zero loses what its mean's own rounding takes, and a row of one value is beta.
#include "layer_norm.cuh"
#include "layer_norm_shapes.hh"

#include <atomic>

namespace cb200 {
namespace {

constexpr int kNarrowItems[] = {4, 3, 2, 6, 8}; // quads of a row that a lane can hold, four by preference (32 columns: 65 us, eight 111)
// Blocks that are resident on an SM.
constexpr int narrow_blocks(int items) { return items <= 4 ? 3 : 2; }

// What a thread's distances are taken from, next to the value given.  Values too large for that (an infinity among them) keep their distance
// from zero: 65,536 distances from 10^33 add up to a number of fp32 where the values do.
__device__ __forceinline__ float centre_at(float v) { return fabsf(v) < 1e33f ? v : 0.0f; }
// The sums of a thread's distances from its centre and of their squares, a quad at a time.
struct thread_statistics {
    pair minus, moved, spread;
    __device__ __forceinline__ explicit thread_statistics(float centre) : minus(-centre), moved(0.0f), spread(0.0f) {}
    __device__ __forceinline__ void add(const float (&v)[4]) {
        const pair d = pair(v[0], v[1]) + minus, e = pair(v[2], v[3]) + minus;
        moved = moved + d;
        spread = fma(d, d, spread);
        moved = moved + e;
        spread = fma(e, e, spread);
    }
};
// Columns from n on, of a quad that starts at column `at`, count as the centre.
__device__ __forceinline__ void cut_off(float (&v)[4], int at, int n, float centre) {
    if (at + 4 <= n) return;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (at + k >= n) v[k] = centre;
}

// A group of p.lanes lanes per row; the next rows' values are on their way while these are worked on.  gamma and beta come out of
// shared memory: a lane's columns of them would take a third of its registers.  1,000,000 x 64 fp32 to bf16 with relu: 71 us, 5.5 TB/s,
// 84 % of a copy, bound by HBM (74 us with a choice of activation and alignment for every quad, 86 with a row's loads waited for at
// once).  GELU and dropout are bound by instructions, 63 % of the issue slots with the FMA pipe half full: 48 million values of 512 columns
// 93 us.  So are 16-bit rows without either, 73 % of the slots: 43 us, 69 % of a copy.
// Of fp32 rows a lane sums up distances from its first value, and the lanes' sums meet as distances from the first lane's: all of them zero in
// a row of one value.  The sum of the values themselves is rounded, which such a row, if its value is large, shows as that rounding over
// sqrt(epsilon).  Rows of 16-bit values need it not: the sum of 1,024 equal ones is a number of fp32.
template<int SIZE, bool HALVES, int ITEMS>
__global__ void __launch_bounds__(kNarrowThreads, ITEMS <= 4 ? 3 : 2) layer_norm_narrow_kernel(const layer_norm_params p) {
    constexpr int kColumns = ITEMS * 32 * 4 + 4;
    constexpr bool kCentred = SIZE == 4;
    __shared__ __align__(16) float parameters[2][kColumns];
    const int lane = threadIdx.x & 31, in_row = lane & (p.lanes - 1), group = lane / p.lanes, rows_per_warp = 32 / p.lanes;
    const bool half = p.x.dtype == CB200_DTYPE_F16;
    const std::uint64_t sequence = sequence_of(p.drop);
    int col[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) col[i] = min((i * p.lanes + in_row) * 4, (p.columns + 3) & ~3);
    const float count = static_cast<float>(p.columns), inverse = 1.0f / count;
    const std::int64_t step = static_cast<std::int64_t>(gridDim.x) * (kNarrowThreads / 32) * rows_per_warp;
    std::int64_t row = (static_cast<std::int64_t>(blockIdx.x) * (kNarrowThreads / 32) + (threadIdx.x >> 5)) * rows_per_warp + group;
    raw_quad<SIZE> raw[ITEMS];
    if (row < p.rows) load_quads(p.x.base + row * p.x.pitch, col, p.columns, p.per_access, raw);
    for (int c = threadIdx.x; c < kColumns; c += kNarrowThreads) {
        parameters[0][c] = p.gamma != nullptr && c < p.columns ? __ldg(p.gamma + c) : 1.0f;
        parameters[1][c] = p.beta != nullptr && c < p.columns ? __ldg(p.beta + c) : 0.0f;
    }
    __syncthreads();
    float own = 0.0f; // columns of the lane
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) own += static_cast<float>(min(max(p.columns - col[i], 0), 4));
    const float own_inverse = own > 0.0f ? 1.0f / own : 0.0f;
    for (; row - group < p.rows; row += step) {
        float v[ITEMS][4], mean, rstd;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) raw[i].template widen<HALVES>(half, v[i]);
        if (row + step < p.rows) load_quads(p.x.base + (row + step) * p.x.pitch, col, p.columns, p.per_access, raw);
        if constexpr (kCentred) {
            const float centre = centre_at(v[0][0]);
            thread_statistics sums(centre);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                cut_off(v[i], col[i], p.columns, centre);
                sums.add(v[i]);
            }
            const float first = __shfl_sync(0xffffffffu, centre, lane - in_row), moved = sums.moved.sum(), off = moved * own_inverse;
            float t[1] = {fmaf(own, centre - first, moved)};
            lane_sums(t, p.lanes);
            mean = fmaf(t[0], inverse, first);
            const float differs = (centre - mean) + off;
            t[0] = fmaf(own * differs, differs, fmaf(-moved, off, sums.spread.sum()));
            lane_sums(t, p.lanes);
            rstd = rsqrtf(fmaf(t[0], inverse, p.epsilon));
            const pair minus_mean(-mean);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
                for (int k = 0; k < 4; k += 2) (pair(v[i][k], v[i][k + 1]) + minus_mean).get(v[i][k], v[i][k + 1]);
            }
        } else {
            pair all(0.0f);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) all = all + (pair(v[i][0], v[i][1]) + pair(v[i][2], v[i][3]));
            float sum[1] = {all.sum()};
            lane_sums(sum, p.lanes);
            mean = sum[0] / count; // a division: exact for rows of one value
            const pair minus_mean(-mean);
            all = pair(0.0f);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
                for (int k = 0; k < 4; k += 2) (pair(v[i][k], v[i][k + 1]) + minus_mean).get(v[i][k], v[i][k + 1]);
                cut_off(v[i], col[i], p.columns, 0.0f);
#pragma unroll
                for (int k = 0; k < 4; k += 2) {
                    const pair d(v[i][k], v[i][k + 1]);
                    all = fma(d, d, all);
                }
            }
            sum[0] = all.sum();
            lane_sums(sum, p.lanes);
            rstd = rsqrtf(fmaf(sum[0], inverse, p.epsilon));
        }
        if (row >= p.rows) continue;
        const pair scale(rstd);
        if (p.stats != nullptr && in_row == 0) *reinterpret_cast<float2 *>(p.stats + 2 * row) = make_float2(mean, rstd);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) { // past the row's end there is room in the shared memory, and nothing is stored
            const float4 g = *reinterpret_cast<const float4 *>(parameters[0] + col[i]), b = *reinterpret_cast<const float4 *>(parameters[1] + col[i]);
            fma(pair(v[i][0], v[i][1]) * scale, pair(g.x, g.y), pair(b.x, b.y)).get(v[i][0], v[i][1]);
            fma(pair(v[i][2], v[i][3]) * scale, pair(g.z, g.w), pair(b.z, b.w)).get(v[i][2], v[i][3]);
        }
        activate(p.epilogue, v);
        drop_quads(p.drop, sequence, static_cast<std::uint32_t>(row), col, v);
        store_quads<HALVES>(p.y.base + row * p.y.pitch, col, p.columns, p.per_access, p.y.dtype, v);
    }
}

// Mean and variance of a row that a block's threads hold, in one walk over the values and with one barrier.  Each thread sums up
// its columns' distances from a centre of its own, the mean of its first quad, and their squares: the square of how far that is
// from the mean of all its columns is at most the number of its quads times their variance, so no digits are lost to the difference
// in the end.  From the sum of each thread's distances and their squares about its mean come those of the warps, and from these
//     mean = m0 + sum over warps of n (warp's mean - m0) / N,  N var = sum over warps of (squares + n (warp's mean - mean)^2),
// m0 the first warp's mean; a warp's mean comes from its threads in the same way, from its first thread's centre on.  So what is summed up
// are differences, all of them zero in a row of one value, and the mean of a row far from zero is off by roundings of itself alone.
struct block_statistics {
    float notes[2][2][32], sizes[32], inverses[32]; // of the warps: of two rows in turn, {mean, squares about it}; columns

    // before the first row; own: columns of the thread
    __device__ __forceinline__ void begin(float own) {
        float size[1] = {own};
        warp_sums(size);
        if ((threadIdx.x & 31) == 0) {
            sizes[threadIdx.x >> 5] = size[0];
            inverses[threadIdx.x >> 5] = size[0] > 0.0f ? 1.0f / size[0] : 0.0f;
        }
        __syncwarp();
    }
    // {mean, 1 / sqrt(var + epsilon)}.  moved, spread: sums of the thread's distances from `centre` and of their squares.
    __device__ __forceinline__ float2 of_row(int set, float own, float own_inverse, float centre, float moved, float spread, float count, float epsilon) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
        const float first = __shfl_sync(0xffffffffu, centre, 0);
        float t[1] = {fmaf(own, centre - first, moved)};
        const float off = moved * own_inverse; // of the thread's mean from its centre
        warp_sums(t);
        const float of_mine = fmaf(t[0], inverses[warp], first);
        if (lane == 0) notes[set][0][warp] = of_mine;
        const float differs = (centre - of_mine) + off;
        t[0] = fmaf(own * differs, differs, fmaf(-moved, off, spread));
        warp_sums(t);
        if (lane == 0) notes[set][1][warp] = t[0];
        __syncthreads();
        const float m0 = notes[set][0][0];
        float from = lane < warps ? notes[set][0][lane] - m0 : 0.0f;
        t[0] = lane < warps ? sizes[lane] / count * from : 0.0f; // shares, whose sum is a number of fp32 where the means are
        warp_sums(t);
        const float mean = m0 + t[0];
        from -= t[0];
        t[0] = lane < warps ? fmaf(sizes[lane] * from, from, notes[set][1][lane]) : 0.0f;
        warp_sums(t);
        return make_float2(mean, rsqrtf(fmaf(t[0], 1.0f / count, epsilon)));
    }
};

// A block per row, the row in registers, its next row on the way where two fit and asked for in L2 where not; gamma and beta stay in
// shared memory from row to row, as many columns of them as it holds (the rest of beta comes out of L2).
// 4,099 x 33,538 bf16: 160 us, 52 % of a copy.  Half of the issue slots are taken (54 %, some 22 instructions a value; 41 with branches for each
// quad, 277 us), and 30 warps, all at the same step of the same row, wait for loads in the others (4.7 of them for each instruction).  Measured against it: a cluster of eight blocks
// per row, whose threads kept gamma and beta of their columns, 373 us, waiting for its barriers; 512 threads with twice the quads 260;
// the next row's quads loaded as soon as these are stored 173; two-wide products 183 (registers); the choices of activation and
// dropout in the loop 180; three quads at a time 169; the columns walked twice as below 212.
constexpr std::size_t kRowShared = 220 * 1024; // of parameters, at most

// The quads of a thread lie a block's width apart; only the last of them can reach past the row's end (layer_norm_shapes.hh).
// PLAIN: neither activation nor dropout.
template<int SIZE, bool HALVES, int QT, bool PLAIN>
__global__ void __launch_bounds__(kRowThreads, 1) layer_norm_row_kernel(const layer_norm_params p, int beta_quads) {
    constexpr bool kAhead = QT * SIZE <= 16; // registers for two rows
    extern __shared__ __align__(16) float parameters[]; // gamma, then beta of each thread's first beta_quads quads
    __shared__ block_statistics statistics;
    const int n = p.columns, width = static_cast<int>(blockDim.x) * 4;
    const bool half = p.x.dtype == CB200_DTYPE_F16;
    const std::uint64_t sequence = PLAIN ? 0u : sequence_of(p.drop);
    const int padded = (n + 3) & ~3;
    const float *beta_at = parameters + padded + 4; // behind each there is room for a quad past the row's end
    const bool beta_vectors = p.beta != nullptr && reinterpret_cast<std::uintptr_t>(p.beta) % 16u == 0u;
    int col[QT];
#pragma unroll
    for (int i = 0; i < QT; ++i) col[i] = i * width + static_cast<int>(threadIdx.x) * 4;
    col[QT - 1] = min(col[QT - 1], padded);
    std::int64_t row = blockIdx.x;
    raw_quad<SIZE> now[QT], next[kAhead ? QT : 1];
    load_quads<QT - 1>(p.x.base + row * p.x.pitch, col, n, p.per_access, now);
    for (int c = threadIdx.x; c < padded + 4; c += blockDim.x) {
        parameters[c] = p.gamma != nullptr && c < n ? __ldg(p.gamma + c) : 1.0f;
        if (c < beta_quads * width) parameters[padded + 4 + c] = p.beta != nullptr && c < n ? __ldg(p.beta + c) : 0.0f;
    }
    const float own_columns = static_cast<float>(4 * (QT - 1) + min(max(n - col[QT - 1], 0), 4)), own_inverse = 1.0f / own_columns;
    statistics.begin(own_columns);
    int set = 0;
    const std::int64_t ahead = kAhead ? 2 : 1; // rows, of this block's, that L2 is asked for in advance
    for (; row < p.rows; row += gridDim.x, set ^= 1) {
        if (threadIdx.x == 0 && row + ahead * gridDim.x < p.rows)
            prefetch_bytes(p.x.base + (row + ahead * gridDim.x) * p.x.pitch, static_cast<std::uint32_t>(n) * SIZE);
        if constexpr (kAhead) {
            if (row + gridDim.x < p.rows) load_quads<QT - 1>(p.x.base + (row + gridDim.x) * p.x.pitch, col, n, p.per_access, next);
        }
        float v[4];
        now[0].template widen<HALVES>(half, v);
        const float centre = centre_at(0.25f * ((v[0] + v[1]) + (v[2] + v[3])));
        thread_statistics sums(centre);
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            now[i].template widen<HALVES>(half, v);
            if (i == QT - 1) cut_off(v, col[i], n, centre);
            sums.add(v);
        }
        const float2 s = statistics.of_row(set, own_columns, own_inverse, centre, sums.moved.sum(), sums.spread.sum(), static_cast<float>(n), p.epsilon);
        const float mean = s.x, rstd = s.y;
        if (p.stats != nullptr && threadIdx.x == 0) *reinterpret_cast<float2 *>(p.stats + 2 * row) = s;
        // a few quads at a time, so that one choice of activation serves them, where the registers hold them besides the row (48 million
        // values of 33,538 columns, fp32 with GELU and dropout: 146 us, three at a time 157)
        constexpr int B = PLAIN || QT == 9 ? 1 : QT % 3 == 0 ? 3 : 2;
        unsigned char *y = p.y.base + row * p.y.pitch;
#pragma unroll
        for (int first = 0; first < QT; first += B) {
            float v[B][4];
            int at[B];
#pragma unroll
            for (int j = 0; j < B; ++j) {
                const int i = first + j;
                at[j] = col[i];
                now[i].template widen<HALVES>(half, v[j]);
                const float4 g = *reinterpret_cast<const float4 *>(parameters + at[j]);
                float b[4];
                if (i < beta_quads) *reinterpret_cast<float4 *>(b) = *reinterpret_cast<const float4 *>(beta_at + at[j]);
                else if (i < QT - 1 && beta_vectors) *reinterpret_cast<float4 *>(b) = __ldg(reinterpret_cast<const float4 *>(p.beta + at[j]));
                else load_parameters(p.beta, at[j], n, 0.0f, b);
                v[j][0] = fmaf((v[j][0] - mean) * rstd, g.x, b[0]);
                v[j][1] = fmaf((v[j][1] - mean) * rstd, g.y, b[1]);
                v[j][2] = fmaf((v[j][2] - mean) * rstd, g.z, b[2]);
                v[j][3] = fmaf((v[j][3] - mean) * rstd, g.w, b[3]);
            }
            if constexpr (!PLAIN) {
                activate(p.epilogue, v);
                drop_quads(p.drop, sequence, static_cast<std::uint32_t>(row), at, v);
            }
            if (first + B < QT) store_quads<HALVES, B>(y, at, n, p.per_access, p.y.dtype, v);
            else store_quads<HALVES, B - 1>(y, at, n, p.per_access, p.y.dtype, v);
        }
        if constexpr (kAhead) {
#pragma unroll
            for (int i = 0; i < QT; ++i) now[i] = next[i];
        } else {
            if (row + gridDim.x < p.rows) load_quads<QT - 1>(p.x.base + (row + gridDim.x) * p.x.pitch, col, n, p.per_access, now);
        }
    }
}

template<int SIZE, bool HALVES, int QT, bool PLAIN>
cb200_status launch_rows(const layer_norm_params &p, int device, cudaStream_t stream) {
    constexpr auto kernel = layer_norm_row_kernel<SIZE, HALVES, QT, PLAIN>;
    const int quads = (p.columns + 3) / 4, threads = row_threads_of(p.columns);
    const std::size_t gamma_bytes = static_cast<std::size_t>(quads + 1) * 16u, width = static_cast<std::size_t>(threads) * 16u;
    const std::size_t beta_quads = std::min<std::size_t>(QT, (kRowShared - gamma_bytes) / width), beta_bytes = beta_quads == QT ? gamma_bytes : beta_quads * width;
    // more than the default 48 KB is asked for once per kernel and device
    static std::atomic<bool> asked[64];
    if (gamma_bytes + beta_bytes > 40 * 1024 && !(device < 64 && asked[device].load(std::memory_order_relaxed))) {
        CB200_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kRowShared)));
        if (device < 64) asked[device].store(true, std::memory_order_relaxed);
    }
    const std::int64_t by_shared = kRowShared / (gamma_bytes + beta_bytes + 1024), resident = std::max<std::int64_t>(1, std::min<std::int64_t>({kRowThreads / threads, by_shared, 32}));
    const unsigned grid = static_cast<unsigned>(std::min<std::int64_t>(p.rows, 148 * resident));
    kernel<<<grid, threads, gamma_bytes + beta_bytes, stream>>>(p, static_cast<int>(beta_quads));
    count_launch();
    CB200_CUDA_OK(cudaGetLastError());
    return CB200_STATUS_SUCCESS;
}

// Rows that do not fit the registers: a block walks along its row twice, the second time out of L2.  40,000 columns, 48 million values:
// fp32 96 us, bf16 67 us, bound by the wait for what L2 delivers (the row twice, gamma and beta; 7.8 warps an instruction; 116 and 94 with
// one column of these to a load);
// clusters of eight blocks that held a row took 183 and 122.
constexpr int kLongThreads = 512, kLongQuads = 4; // quads that a thread has in flight

template<int SIZE, bool HALVES>
__global__ void __launch_bounds__(kLongThreads, 2) layer_norm_long_kernel(const layer_norm_params p) {
    __shared__ block_statistics statistics;
    constexpr int kStep = kLongThreads * 4;
    const int n = p.columns, first = static_cast<int>(threadIdx.x) * 4;
    const bool half = p.x.dtype == CB200_DTYPE_F16;
    const std::uint64_t sequence = sequence_of(p.drop);
    const bool vectors = on_16_bytes(p.gamma) && on_16_bytes(p.beta);
    float own = 0.0f;
    for (int at = first; at < n; at += kStep) own += static_cast<float>(min(4, n - at));
    const float own_inverse = 1.0f / own; // a thread has columns: there are more than 2,048 of them
    statistics.begin(own);
    int set = 0;
    for (std::int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, set ^= 1) {
        const unsigned char *x = p.x.base + row * p.x.pitch;
        unsigned char *y = p.y.base + row * p.y.pitch;
        float centre = 0.0f;
        thread_statistics sums(0.0f);
        for (int at = first; at < n; at += kLongQuads * kStep) {
            raw_quad<SIZE> raw[kLongQuads];
            int col[kLongQuads];
#pragma unroll
            for (int i = 0; i < kLongQuads; ++i) col[i] = min(at + i * kStep, (n + 3) & ~3);
            load_quads(x, col, n, p.per_access, raw);
#pragma unroll
            for (int i = 0; i < kLongQuads; ++i) {
                float v[4];
                raw[i].template widen<HALVES>(half, v);
                if (i == 0 && at == first) {
                    centre = centre_at(0.25f * ((v[0] + v[1]) + (v[2] + v[3])));
                    sums.minus = pair(-centre);
                }
                cut_off(v, col[i], n, centre);
                sums.add(v);
            }
        }
        const float2 s = statistics.of_row(set, own, own_inverse, centre, sums.moved.sum(), sums.spread.sum(), static_cast<float>(n), p.epsilon);
        if (p.stats != nullptr && threadIdx.x == 0) *reinterpret_cast<float2 *>(p.stats + 2 * row) = s;
        for (int at = first; at < n; at += kLongQuads * kStep) {
            raw_quad<SIZE> raw[kLongQuads];
            int col[kLongQuads];
            float v[kLongQuads][4];
#pragma unroll
            for (int i = 0; i < kLongQuads; ++i) col[i] = min(at + i * kStep, (n + 3) & ~3);
            load_quads(x, col, n, p.per_access, raw);
            float4 g[kLongQuads], b[kLongQuads];
#pragma unroll
            for (int i = 0; i < kLongQuads; ++i) {
                g[i] = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
                b[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (p.gamma != nullptr) g[i] = load_parameter_quad(p.gamma, col[i], n, vectors);
                if (p.beta != nullptr) b[i] = load_parameter_quad(p.beta, col[i], n, vectors);
            }
#pragma unroll
            for (int i = 0; i < kLongQuads; ++i) {
                raw[i].template widen<HALVES>(half, v[i]);
                v[i][0] = fmaf((v[i][0] - s.x) * s.y, g[i].x, b[i].x);
                v[i][1] = fmaf((v[i][1] - s.x) * s.y, g[i].y, b[i].y);
                v[i][2] = fmaf((v[i][2] - s.x) * s.y, g[i].z, b[i].z);
                v[i][3] = fmaf((v[i][3] - s.x) * s.y, g[i].w, b[i].w);
            }
            activate(p.epilogue, v);
            drop_quads(p.drop, sequence, static_cast<std::uint32_t>(row), col, v);
            store_quads<HALVES>(y, col, n, p.per_access, p.y.dtype, v);
        }
    }
}

template<int SIZE, bool HALVES, int ITEMS>
cb200_status launch_narrow(const layer_norm_params &p, cudaStream_t stream) {
    const std::int64_t per_block = kNarrowThreads / p.lanes, blocks = (p.rows + per_block - 1) / per_block;
    layer_norm_narrow_kernel<SIZE, HALVES, ITEMS><<<static_cast<unsigned>(std::min<std::int64_t>(blocks, 148 * narrow_blocks(ITEMS))), kNarrowThreads, 0, stream>>>(p);
    count_launch();
    CB200_CUDA_OK(cudaGetLastError());
    return CB200_STATUS_SUCCESS;
}

template<int SIZE, bool HALVES, int QT>
cb200_status launch_rows(const layer_norm_params &p, int device, cudaStream_t stream) {
    return p.epilogue == CB200_EPILOGUE_NONE && !p.drop.on ? launch_rows<SIZE, HALVES, QT, true>(p, device, stream) : launch_rows<SIZE, HALVES, QT, false>(p, device, stream);
}

template<int SIZE, bool HALVES>
cb200_status launch_forward(layer_norm_params p, int device, cudaStream_t stream) {
    if (p.columns <= kWarpColumns) {
        const narrow_shape narrow = narrow_shape_of(p.columns, kNarrowItems, 5);
        p.lanes = narrow.lanes;
        switch (narrow.items) {
        case 2: return launch_narrow<SIZE, HALVES, 2>(p, stream);
        case 3: return launch_narrow<SIZE, HALVES, 3>(p, stream);
        case 4: return launch_narrow<SIZE, HALVES, 4>(p, stream);
        case 6: return launch_narrow<SIZE, HALVES, 6>(p, stream);
        default: return launch_narrow<SIZE, HALVES, 8>(p, stream);
        }
    }
    if (p.columns <= kRowColumns) {
        switch (row_quads_of(p.columns)) {
        case 2: return launch_rows<SIZE, HALVES, 2>(p, device, stream);
        case 4: return launch_rows<SIZE, HALVES, 4>(p, device, stream);
        case 6: return launch_rows<SIZE, HALVES, 6>(p, device, stream);
        default: return launch_rows<SIZE, HALVES, 9>(p, device, stream);
        }
    }
    layer_norm_long_kernel<SIZE, HALVES><<<static_cast<unsigned>(std::min<std::int64_t>(p.rows, 148 * 2)), kLongThreads, 0, stream>>>(p);
    count_launch();
    CB200_CUDA_OK(cudaGetLastError());
    return CB200_STATUS_SUCCESS;
}

} // namespace
} // namespace cb200

extern "C" cb200_status cb200_layer_norm_forward(const cb200_layer_norm *d, void *stream) {
    using namespace cb200;
    clear_error();
    layer_norm_params p{};
    cb200_status st = layer_norm_checked(d, false, &p);
    if (st == CB200_STATUS_SUCCESS) st = row_matrix_of(d->y, d->y_ld, d->y_dtype, d->rows, d->columns, "y", &p.y);
    if (st != CB200_STATUS_SUCCESS) return st;
    if (!rows_compatible(p.y, p.x, p.rows, p.columns)) return fail(CB200_STATUS_INVALID_ARGUMENT, "y overlaps x without being x");
    p.per_access = columns_per_access(p.y, p.per_access);
    device_scope scope(d->device);
    CB200_CUDA_OK(scope.status);
    if (p.rows == 0) return CB200_STATUS_SUCCESS;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool halves = p.x.dtype == CB200_DTYPE_F16 || p.y.dtype == CB200_DTYPE_F16;
    if (element_bytes(p.x.dtype) == 4) return halves ? launch_forward<4, true>(p, d->device, s) : launch_forward<4, false>(p, d->device, s);
    return halves ? launch_forward<2, true>(p, d->device, s) : launch_forward<2, false>(p, d->device, s);
}
