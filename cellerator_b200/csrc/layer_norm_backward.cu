// Gradients of the layer norm with its activation and dropout.  With u = (x - mean) rstd and z = gamma u + beta,
//     dz = drop(dy) act'(z),  dbeta = sum over rows of dz,  dgamma = sum over rows of dz u,  h = gamma dz,
//     dx = rstd (h - mean over columns of h - u mean over columns of (h u)).
// One pass reads x and dy, keeps a row in registers between its sums and its dx, and adds dz and dz u up per column in the
// threads that own the columns; a block leaves its sums in the workspace, and a second launch adds these up in order.
#include "dependent_launch.cuh"
#include "layer_norm.cuh"

namespace cb200 {
namespace {

constexpr int kNarrowItems[] = {2, 4, 3}; // quads of a row that a lane can hold, two by preference (64 columns: 97 us, four 122)
constexpr std::int64_t kNarrowColumns = 4 * 32 * 4;
// Blocks that are resident on an SM: with two quads to a lane, which keeps two sums for each of its columns, 24 warps fit.
constexpr int narrow_blocks(int items) { return items == 2 ? 3 : 2; }

// u and h in place of x and dy of some quads of a row; dz u and dz added to what the thread keeps of their columns, h and h u to the
// row's sums.  at: where the quads' gamma (and, beta_at further, beta) stand in shared memory.
template<int KIND, int Q>
__device__ __forceinline__ void row_terms(float mean, float rstd, const float *gamma_at, int beta_at, const int (&at)[Q], float (&x)[Q][4], float (&dy)[Q][4],
                                          float (&dgamma)[Q][4], float (&dbeta)[Q][4], float (&sums)[2]) {
    float4 gamma[Q];
    const pair minus_mean(-mean), scale(rstd);
    pair sum_h(0.0f), sum_hu(0.0f);
#pragma unroll
    for (int i = 0; i < Q; ++i) {
        gamma[i] = *reinterpret_cast<const float4 *>(gamma_at + at[i]);
#pragma unroll
        for (int k = 0; k < 4; k += 2) ((pair(x[i][k], x[i][k + 1]) + minus_mean) * scale).get(x[i][k], x[i][k + 1]);
    }
    if constexpr (KIND != CB200_EPILOGUE_NONE) {
        float4 beta[Q];
#pragma unroll
        for (int i = 0; i < Q; ++i) beta[i] = *reinterpret_cast<const float4 *>(gamma_at + beta_at + at[i]);
        through_as<KIND>(dy, x, gamma, beta);
    }
#pragma unroll
    for (int i = 0; i < Q; ++i) {
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
            const pair u(x[i][k], x[i][k + 1]), dz(dy[i][k], dy[i][k + 1]);
            (pair(dbeta[i][k], dbeta[i][k + 1]) + dz).get(dbeta[i][k], dbeta[i][k + 1]);
            fma(dz, u, pair(dgamma[i][k], dgamma[i][k + 1])).get(dgamma[i][k], dgamma[i][k + 1]);
            const pair h = dz * (k == 0 ? pair(gamma[i].x, gamma[i].y) : pair(gamma[i].z, gamma[i].w));
            sum_h = sum_h + h;
            sum_hu = fma(h, u, sum_hu);
            h.get(dy[i][k], dy[i][k + 1]);
        }
    }
    sums[0] = sum_h.sum();
    sums[1] = sum_hu.sum();
}

// A group of p.lanes lanes per row; the next rows' values are on their way while these are worked on.  Columns past the last hold
// zeros in dy, so that they add nothing.  1,000,000 x 64, fp32 and a bf16 dy, GELU (tanh) and dropout: 169 us, 58 % of a copy, bound by
// instructions (the random words and the slope; 62 % of the issue slots, ALU and FMA pipes 44 %; 175 us with one column at a time, 212 with an activation chosen per quad, 182 before the slope was rearranged);
// without either 101 us for 48 million values (87 %).
template<int SX, int SG, bool HALVES, int ITEMS>
__global__ void __launch_bounds__(kNarrowThreads, ITEMS == 2 ? 3 : 2) layer_norm_back_narrow_kernel(const layer_norm_params p) {
    __shared__ float meet[kNarrowThreads / 32][ITEMS * 4 * 32];
    constexpr int kParameters = ITEMS * 4 * 32 + 4;
    __shared__ __align__(16) float parameters[2][kParameters]; // gamma and beta: registers are short here
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, in_row = lane & (p.lanes - 1), group = lane / p.lanes, rows_per_warp = 32 / p.lanes;
    const bool half = p.x.dtype == CB200_DTYPE_F16, half_dy = p.dy.dtype == CB200_DTYPE_F16;
    const std::uint64_t sequence = sequence_of(p.drop);
    for (int c = threadIdx.x; c < kParameters; c += kNarrowThreads) {
        parameters[0][c] = p.gamma != nullptr && c < p.columns ? __ldg(p.gamma + c) : 1.0f;
        parameters[1][c] = p.beta != nullptr && c < p.columns ? __ldg(p.beta + c) : 0.0f;
    }
    __syncthreads();
    float dgamma[ITEMS][4], dbeta[ITEMS][4];
    int col[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        col[i] = min((i * p.lanes + in_row) * 4, (p.columns + 3) & ~3);
#pragma unroll
        for (int k = 0; k < 4; ++k) dgamma[i][k] = dbeta[i][k] = 0.0f;
    }
    const float inverse = 1.0f / static_cast<float>(p.columns);
    const std::int64_t step = static_cast<std::int64_t>(gridDim.x) * (kNarrowThreads / 32) * rows_per_warp;
    std::int64_t row = (static_cast<std::int64_t>(blockIdx.x) * (kNarrowThreads / 32) + warp) * rows_per_warp + group;
    raw_quad<SX> raw_x[ITEMS];
    raw_quad<SG> raw_dy[ITEMS];
    float2 stats = make_float2(0.0f, 0.0f);
    const auto fetch = [&](std::int64_t at) {
        if (at >= p.rows) return;
        stats = *reinterpret_cast<const float2 *>(p.stats + 2 * at);
        load_quads(p.x.base + at * p.x.pitch, col, p.columns, p.per_access, raw_x);
        load_quads(p.dy.base + at * p.dy.pitch, col, p.columns, p.per_access, raw_dy);
    };
    fetch(row);
    for (; row - group < p.rows; row += step) {
        const bool active = row < p.rows;
        const float mean = stats.x, rstd = stats.y;
        float x[ITEMS][4], dy[ITEMS][4], sums[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            raw_x[i].template widen<HALVES>(half, x[i]);
            raw_dy[i].template widen<HALVES>(half_dy, dy[i]);
        }
        fetch(row + step);
        if (active) {
            drop_quads(p.drop, sequence, static_cast<std::uint32_t>(row), col, dy);
            with_epilogue(p.epilogue, [&](auto kind) { row_terms<decltype(kind)::value>(mean, rstd, parameters[0], kParameters, col, x, dy, dgamma, dbeta, sums); });
        }
        lane_sums(sums, p.lanes);
        sums[0] *= inverse;
        sums[1] *= inverse;
        if (!active || p.dx.base == nullptr) continue;
        const pair scale(rstd), minus_h(-sums[0]), minus_hu(-sums[1]);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
            for (int k = 0; k < 4; k += 2)
                (scale * fma(pair(x[i][k], x[i][k + 1]), minus_hu, pair(dy[i][k], dy[i][k + 1]) + minus_h)).get(x[i][k], x[i][k + 1]);
        }
        store_quads<HALVES>(p.dx.base + row * p.dx.pitch, col, p.columns, p.per_access, p.dx.dtype, x);
    }
    let_next_launch_start();
    if (p.partials == nullptr) return;
    // the groups of a warp, then the warps of the block, one of the two sums after the other
#pragma unroll
    for (int which = 0; which < 2; ++which) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float v = which == 0 ? dgamma[i][k] : dbeta[i][k];
                for (int off = p.lanes; off < 32; off <<= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
                if (group == 0) meet[warp][(i * p.lanes + in_row) * 4 + k] = v; // columns past the row's end hold nothing that is read
            }
        }
        __syncthreads();
        float *out = p.partials + (static_cast<std::int64_t>(blockIdx.x) * 2 + which) * p.columns;
        for (int c = threadIdx.x; c < p.columns; c += kNarrowThreads) {
            float v = meet[0][c];
#pragma unroll
            for (int w = 1; w < kNarrowThreads / 32; ++w) v += meet[w][c];
            out[c] = v;
        }
        __syncthreads();
    }
}

constexpr int kBlockQuads = 2, kBlockThreads = kBlockColumns / (4 * kBlockQuads); // of a thread; of a block, at most

// A block per row; a thread keeps the sums of its columns from row to row.  gamma and beta are in shared memory: the sums, a row and
// the next one's values take the registers.  48 million values of 4,000 columns: fp32 132 us (66 % of a copy), bf16 97 us (45 %), one
// barrier a row and half of the issue slots; with GELU and dropout 183 and 149, bound by instructions.
template<int SX, int SG, bool HALVES>
__global__ void __launch_bounds__(kBlockThreads) layer_norm_back_block_kernel(const layer_norm_params p) {
    constexpr int QT = kBlockQuads;
    __shared__ float notes[2][2][kBlockThreads / 32]; // of two rows in turn: each warp's sums
    extern __shared__ __align__(16) float parameters[]; // gamma and beta, and a quad each for threads without columns
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, n = p.columns, beta_at = ((n + 3) & ~3) + 4;
    const bool half = p.x.dtype == CB200_DTYPE_F16, half_dy = p.dy.dtype == CB200_DTYPE_F16;
    const std::uint64_t sequence = sequence_of(p.drop);
    for (int c = threadIdx.x; c < beta_at; c += blockDim.x) {
        parameters[c] = p.gamma != nullptr && c < n ? __ldg(p.gamma + c) : 1.0f;
        parameters[beta_at + c] = p.beta != nullptr && c < n ? __ldg(p.beta + c) : 0.0f;
    }
    float dgamma[QT][4], dbeta[QT][4];
    int col[QT];
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        col[i] = min((i * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * 4, (n + 3) & ~3);
#pragma unroll
        for (int k = 0; k < 4; ++k) dgamma[i][k] = dbeta[i][k] = 0.0f;
    }
    const float inverse = 1.0f / static_cast<float>(n);
    raw_quad<SX> raw_x[QT];
    raw_quad<SG> raw_dy[QT];
    float2 stats;
    const auto fetch = [&](std::int64_t row) {
        if (row >= p.rows) return;
        stats = *reinterpret_cast<const float2 *>(p.stats + 2 * row);
        load_quads(p.x.base + row * p.x.pitch, col, n, p.per_access, raw_x);
        load_quads(p.dy.base + row * p.dy.pitch, col, n, p.per_access, raw_dy);
    };
    fetch(blockIdx.x);
    __syncthreads();
    int set = 0;
    for (std::int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, set ^= 1) {
        float x[QT][4], dy[QT][4], sums[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            raw_x[i].template widen<HALVES>(half, x[i]);
            raw_dy[i].template widen<HALVES>(half_dy, dy[i]);
        }
        const float mean = stats.x, rstd = stats.y;
        fetch(row + gridDim.x);
        drop_quads(p.drop, sequence, static_cast<std::uint32_t>(row), col, dy);
        with_epilogue(p.epilogue, [&](auto kind) { row_terms<decltype(kind)::value>(mean, rstd, parameters, beta_at, col, x, dy, dgamma, dbeta, sums); });
        if (p.dx.base == nullptr) continue;
        warp_sums(sums);
        if (lane == 0) {
            notes[set][0][warp] = sums[0];
            notes[set][1][warp] = sums[1];
        }
        __syncthreads();
        sums[0] = lane < warps ? notes[set][0][lane] : 0.0f;
        sums[1] = lane < warps ? notes[set][1][lane] : 0.0f;
        warp_sums(sums);
        const pair scale(rstd), minus_h(-sums[0] * inverse), minus_hu(-sums[1] * inverse);
#pragma unroll
        for (int i = 0; i < QT; ++i) {
#pragma unroll
            for (int k = 0; k < 4; k += 2)
                (scale * fma(pair(x[i][k], x[i][k + 1]), minus_hu, pair(dy[i][k], dy[i][k + 1]) + minus_h)).get(x[i][k], x[i][k + 1]);
        }
        store_quads<HALVES>(p.dx.base + row * p.dx.pitch, col, n, p.per_access, p.dx.dtype, x);
    }
    let_next_launch_start();
    if (p.partials == nullptr) return;
    float *out = p.partials + static_cast<std::int64_t>(blockIdx.x) * 2 * n;
#pragma unroll
    for (int i = 0; i < QT; ++i) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (col[i] + k >= n) continue;
            out[col[i] + k] = dgamma[i][k];
            out[n + col[i] + k] = dbeta[i][k];
        }
    }
}

constexpr int kMeetWarps = 32; // most warps of a block

// dgamma and dbeta from the parts' sums: of 32 columns, each warp adds up every so many parts, then the warps' sums in order.
__global__ void __launch_bounds__(kMeetWarps * 32) layer_norm_meet_kernel(const float *partials, int parts, int columns, float *dgamma, float *dbeta) {
    __shared__ float meet[kMeetWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, c = blockIdx.x * 32 + lane;
    wait_for_previous_launch();
    float v = 0.0f;
    if (c < 2 * columns) {
#pragma unroll 16
        for (int part = warp; part < parts; part += warps) v += partials[static_cast<std::int64_t>(part) * 2 * columns + c];
    }
    meet[warp][lane] = v;
    __syncthreads();
    if (warp != 0 || c >= 2 * columns) return;
    for (int w = 1; w < warps; ++w) v += meet[w][lane];
    float *out = c < columns ? dgamma : dbeta;
    if (out != nullptr) out[c < columns ? c : c - columns] = v;
}
// Warps of a block: about twelve parts for each, so that a thread has its loads in flight at once.
int meet_warps(std::int64_t parts) { return static_cast<int>(std::min<std::int64_t>(kMeetWarps, (parts + 11) / 12)); }

// Blocks of a launch over narrow rows.
std::int64_t narrow_parts(std::int64_t rows, std::int64_t columns) {
    const narrow_shape narrow = narrow_shape_of(columns, kNarrowItems, 3);
    const std::int64_t per_block = kNarrowThreads / narrow.lanes;
    return std::min<std::int64_t>((rows + per_block - 1) / per_block, 148 * narrow_blocks(narrow.items));
}

// Threads of a block of a row that it holds, and blocks of a launch: those that are resident with 96 registers a thread.
int block_threads(std::int64_t columns) { return static_cast<int>((columns + 4 * kBlockQuads * 32 - 1) / (4 * kBlockQuads * 32) * 32); }
std::int64_t block_parts(std::int64_t rows, std::int64_t columns) { return std::min<std::int64_t>(rows, 148 * std::max(1, 640 / block_threads(columns))); }

struct backward_launch {
    layer_norm_params p;
    float *dgamma, *dbeta;
    cudaStream_t stream;

    cb200_status finish(std::int64_t parts) const {
        count_launch();
        CB200_CUDA_OK(cudaGetLastError());
        return meet(parts);
    }
    cb200_status meet(std::int64_t parts) const {
        if (p.partials == nullptr) return CB200_STATUS_SUCCESS;
        CB200_CUDA_OK(launch_kernel(true, layer_norm_meet_kernel, dim3(static_cast<unsigned>((2 * p.columns + 31) / 32)), meet_warps(parts) * 32, 0, stream,
                                    static_cast<const float *>(p.partials), static_cast<int>(parts), p.columns, dgamma, dbeta));
        count_launch();
        return CB200_STATUS_SUCCESS;
    }
    template<int SX, int SG, bool HALVES>
    cb200_status run() {
        if (p.columns <= kNarrowColumns) {
            const std::int64_t parts = narrow_parts(p.rows, p.columns);
            const narrow_shape narrow = narrow_shape_of(p.columns, kNarrowItems, 3);
            p.lanes = narrow.lanes;
            if (narrow.items == 2) layer_norm_back_narrow_kernel<SX, SG, HALVES, 2><<<static_cast<unsigned>(parts), kNarrowThreads, 0, stream>>>(p);
            else if (narrow.items == 3) layer_norm_back_narrow_kernel<SX, SG, HALVES, 3><<<static_cast<unsigned>(parts), kNarrowThreads, 0, stream>>>(p);
            else layer_norm_back_narrow_kernel<SX, SG, HALVES, 4><<<static_cast<unsigned>(parts), kNarrowThreads, 0, stream>>>(p);
            return finish(parts);
        }
        const std::int64_t parts = block_parts(p.rows, p.columns);
        const std::size_t smem = static_cast<std::size_t>((p.columns + 3) / 4 + 1) * 32u;
        layer_norm_back_block_kernel<SX, SG, HALVES><<<static_cast<unsigned>(parts), block_threads(p.columns), smem, stream>>>(p);
        return finish(parts);
    }
};

std::uint64_t partial_bytes(std::int64_t rows, std::int64_t columns) {
    const std::int64_t parts = columns <= kNarrowColumns ? narrow_parts(rows, columns)
                               : columns <= kBlockColumns ? block_parts(rows, columns)
                                                          : layer_norm_columns_parts(rows, columns);
    return static_cast<std::uint64_t>(parts) * 2u * static_cast<std::uint64_t>(columns) * sizeof(float);
}
std::uint64_t sums_bytes(std::int64_t rows, std::int64_t columns) { return columns <= kBlockColumns ? 0u : layer_norm_columns_sums_bytes(rows, columns); }

} // namespace
} // namespace cb200

extern "C" cb200_status cb200_layer_norm_backward_workspace(int64_t rows, int64_t columns, uint64_t *bytes) {
    using namespace cb200;
    clear_error();
    if (bytes == nullptr) return fail(CB200_STATUS_INVALID_ARGUMENT, "workspace needs an output");
    if (rows < 0 || columns < 1 || columns > kMostColumns || rows >= (1ll << 32))
        return fail(CB200_STATUS_INVALID_SHAPE, "the layer norm takes fewer than 2^32 rows of 1 to %lld columns, got %lld x %lld", (long long)kMostColumns, (long long)rows, (long long)columns);
    *bytes = rows == 0 ? 0u : partial_bytes(rows, columns) + sums_bytes(rows, columns);
    return CB200_STATUS_SUCCESS;
}

extern "C" cb200_status cb200_layer_norm_backward(const cb200_layer_norm *d, void *stream) {
    using namespace cb200;
    clear_error();
    backward_launch b{};
    layer_norm_params &p = b.p;
    cb200_status st = layer_norm_checked(d, true, &p);
    if (st == CB200_STATUS_SUCCESS) st = row_matrix_of(d->dy, d->dy_ld, d->dy_dtype, d->rows, d->columns, "dy", &p.dy);
    if (st == CB200_STATUS_SUCCESS && d->dx != nullptr) st = row_matrix_of(d->dx, d->dx_ld, d->dx_dtype, d->rows, d->columns, "dx", &p.dx);
    if (st != CB200_STATUS_SUCCESS) return st;
    if (d->stats == nullptr && p.rows > 0) return fail(CB200_STATUS_INVALID_ARGUMENT, "the backward pass needs the statistics of the forward pass");
    if (!rows_compatible(p.dx, p.x, p.rows, p.columns) || !rows_compatible(p.dx, p.dy, p.rows, p.columns))
        return fail(CB200_STATUS_INVALID_ARGUMENT, "dx overlaps x or dy without being it");
    if (d->dgamma != nullptr && d->dbeta != nullptr) {
        const auto g = reinterpret_cast<std::uintptr_t>(d->dgamma), b = reinterpret_cast<std::uintptr_t>(d->dbeta);
        if ((g > b ? g - b : b - g) < static_cast<std::uintptr_t>(d->columns) * sizeof(float)) return fail(CB200_STATUS_INVALID_ARGUMENT, "dgamma and dbeta overlap");
    }
    const bool sums = d->dgamma != nullptr || d->dbeta != nullptr;
    const bool two_passes = p.columns > kBlockColumns && p.dx.base != nullptr;
    float *row_sums = nullptr;
    if ((sums || two_passes) && p.rows > 0) {
        const std::uint64_t partial = sums ? partial_bytes(p.rows, p.columns) : 0u, need = partial + (two_passes ? sums_bytes(p.rows, p.columns) : 0u);
        if (d->workspace == nullptr || d->workspace_bytes < need || reinterpret_cast<std::uintptr_t>(d->workspace) % 4u != 0u)
            return fail(CB200_STATUS_INSUFFICIENT_WORKSPACE, "workspace of %llu bytes needed, %llu given", (unsigned long long)need,
                        (unsigned long long)(d->workspace == nullptr ? 0u : d->workspace_bytes));
        if (sums) p.partials = static_cast<float *>(d->workspace);
        row_sums = reinterpret_cast<float *>(static_cast<unsigned char *>(d->workspace) + partial);
    }
    p.per_access = columns_per_access(p.dy, p.per_access);
    if (p.dx.base != nullptr) p.per_access = columns_per_access(p.dx, p.per_access);
    b.dgamma = d->dgamma;
    b.dbeta = d->dbeta;
    b.stream = static_cast<cudaStream_t>(stream);
    device_scope scope(d->device);
    CB200_CUDA_OK(scope.status);
    if (p.rows == 0) { // sums over nothing
        if (b.dgamma != nullptr) CB200_CUDA_OK(cudaMemsetAsync(b.dgamma, 0, static_cast<std::size_t>(p.columns) * sizeof(float), b.stream));
        if (b.dbeta != nullptr) CB200_CUDA_OK(cudaMemsetAsync(b.dbeta, 0, static_cast<std::size_t>(p.columns) * sizeof(float), b.stream));
        return CB200_STATUS_SUCCESS;
    }
    if (!sums && p.dx.base == nullptr) return CB200_STATUS_SUCCESS;
    if (p.columns > kBlockColumns) {
        st = launch_layer_norm_columns(p, row_sums, b.stream);
        return st == CB200_STATUS_SUCCESS ? b.meet(layer_norm_columns_parts(p.rows, p.columns)) : st;
    }
    const bool wide_x = element_bytes(p.x.dtype) == 4, wide_dy = element_bytes(p.dy.dtype) == 4;
    const auto of_sizes = [&](auto halves) {
        constexpr bool H = decltype(halves)::value;
        if (wide_x) return wide_dy ? b.run<4, 4, H>() : b.run<4, 2, H>();
        return wide_dy ? b.run<2, 4, H>() : b.run<2, 2, H>();
    };
    return p.x.dtype == CB200_DTYPE_F16 || p.dy.dtype == CB200_DTYPE_F16 || (p.dx.base != nullptr && p.dx.dtype == CB200_DTYPE_F16) ? of_sizes(std::true_type{})
                                                                                                                                    : of_sizes(std::false_type{});
}
