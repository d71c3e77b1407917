// Gradients of the layer norm with its activation and dropout.  With u = (x - mean) rstd and z = gamma u + beta,
//     dz = drop(dy) act'(z),  dbeta = sum over rows of dz,  dgamma = sum over rows of dz u,  h = gamma dz,
//     dx = rstd (h - mean over columns of h - u mean over columns of (h u)).
// One pass reads x and dy, keeps a row in registers between its sums and its dx, and adds dz and dz u up per column in the
// threads that own the columns; a block or cluster leaves its sums in the workspace, and a second launch adds these up in order.
#include "dependent_launch.cuh"
#include "layer_norm.cuh"

namespace cb200 {
namespace {

// Most blocks (narrow) or clusters (wide) of a launch: each leaves 2 x columns sums.
constexpr int kNarrowParts = 148 * 2;
constexpr int kWideParts = 148 * 4;

// dz and u of a quad in place of dy and x; h u added to sums[1], h to sums[0]
struct quad_terms {
    float mean, rstd;
    int epilogue;

    __device__ __forceinline__ void apply(float (&x)[4], float (&dy)[4], const float (&gamma)[4], const float (&beta)[4], float (&dgamma)[4],
                                          float (&dbeta)[4], float (&sums)[2]) const {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            x[k] = (x[k] - mean) * rstd;
            if (epilogue != CB200_EPILOGUE_NONE) dy[k] = through_activation(dy[k], fmaf(x[k], gamma[k], beta[k]), epilogue);
            dbeta[k] += dy[k];
            dgamma[k] = fmaf(dy[k], x[k], dgamma[k]);
            dy[k] *= gamma[k];
            sums[0] += dy[k];
            sums[1] = fmaf(dy[k], x[k], sums[1]);
        }
    }
};

// A group of p.lanes lanes per row.  Columns past the last hold zeros in x and dy, so that u there is not zero but dz is.
template<int SX, int SG>
__global__ void __launch_bounds__(kNarrowThreads) layer_norm_back_narrow_kernel(const layer_norm_params p) {
    __shared__ float meet[kNarrowThreads / 32][kNarrowItems * 4 * 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, in_row = lane & (p.lanes - 1), group = lane / p.lanes, rows_per_warp = 32 / p.lanes;
    const bool half = p.x.dtype == CB200_DTYPE_F16, half_dy = p.dy.dtype == CB200_DTYPE_F16;
    const std::uint64_t sequence = sequence_of(p.drop);
    float gamma[kNarrowItems][4], beta[kNarrowItems][4], dgamma[kNarrowItems][4], dbeta[kNarrowItems][4];
    int col[kNarrowItems];
#pragma unroll
    for (int i = 0; i < kNarrowItems; ++i) {
        col[i] = min((i * p.lanes + in_row) * 4, p.columns);
        load_parameters(p.gamma, col[i], p.columns, 1.0f, gamma[i]);
        load_parameters(p.beta, col[i], p.columns, 0.0f, beta[i]);
#pragma unroll
        for (int k = 0; k < 4; ++k) dgamma[i][k] = dbeta[i][k] = 0.0f;
    }
    const float inverse = 1.0f / static_cast<float>(p.columns);
    const std::int64_t step = static_cast<std::int64_t>(gridDim.x) * (kNarrowThreads / 32) * rows_per_warp;
    for (std::int64_t base = (static_cast<std::int64_t>(blockIdx.x) * (kNarrowThreads / 32) + warp) * rows_per_warp; base < p.rows; base += step) {
        const std::int64_t row = base + group;
        const bool active = row < p.rows;
        raw_quad<SX> raw_x[kNarrowItems];
        raw_quad<SG> raw_dy[kNarrowItems];
        quad_terms terms{0.0f, 0.0f, p.epilogue};
        if (active) {
            const float2 s = *reinterpret_cast<const float2 *>(p.stats + 2 * row);
            terms.mean = s.x;
            terms.rstd = s.y;
        }
#pragma unroll
        for (int i = 0; i < kNarrowItems; ++i) {
            raw_x[i].clear();
            raw_dy[i].clear();
            if (active) {
                raw_x[i].load(p.x.base + row * p.x.pitch, col[i], p.columns, p.per_access);
                raw_dy[i].load(p.dy.base + row * p.dy.pitch, col[i], p.columns, p.per_access);
            }
        }
        float x[kNarrowItems][4], dy[kNarrowItems][4], sums[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kNarrowItems; ++i) {
            raw_x[i].widen(half, x[i]);
            raw_dy[i].widen(half_dy, dy[i]);
            if (!active || col[i] >= p.columns) continue;
            if (p.drop.on) drop_quad(p.drop, sequence, static_cast<std::uint32_t>(row), static_cast<std::uint32_t>(col[i] >> 2), dy[i]);
            terms.apply(x[i], dy[i], gamma[i], beta[i], dgamma[i], dbeta[i], sums);
        }
        sums[0] = lane_sum(sums[0], p.lanes) * inverse;
        sums[1] = lane_sum(sums[1], p.lanes) * inverse;
        if (!active || p.dx.base == nullptr) continue;
#pragma unroll
        for (int i = 0; i < kNarrowItems; ++i) {
            if (col[i] >= p.columns) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k) x[i][k] = terms.rstd * (dy[i][k] - sums[0] - x[i][k] * sums[1]);
            store_quad(p.dx.base + row * p.dx.pitch, col[i], p.columns, p.per_access, p.dx.dtype, x[i]);
        }
    }
    let_next_launch_start();
    if (p.partials == nullptr) return;
    // the groups of a warp, then the warps of the block, one of the two sums after the other
#pragma unroll
    for (int which = 0; which < 2; ++which) {
#pragma unroll
        for (int i = 0; i < kNarrowItems; ++i) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float v = which == 0 ? dgamma[i][k] : dbeta[i][k];
                for (int off = p.lanes; off < 32; off <<= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
                if (group == 0) meet[warp][(i * p.lanes + in_row) * 4 + k] = v;
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

// A block or a cluster of blocks per row, each block with a slice of the columns, whose sums its threads keep from row to row.
template<int SX, int SG, int QT, bool CLUSTER>
__global__ void __launch_bounds__(kWideThreads) layer_norm_back_wide_kernel(const layer_norm_params p) {
    __shared__ wide_sums<2, CLUSTER> around;
    const int rank = CLUSTER ? static_cast<int>(blockIdx.x) % p.cluster : 0;
    const std::int64_t first = CLUSTER ? blockIdx.x / p.cluster : blockIdx.x, step = CLUSTER ? gridDim.x / p.cluster : gridDim.x;
    const bool half = p.x.dtype == CB200_DTYPE_F16, half_dy = p.dy.dtype == CB200_DTYPE_F16;
    const std::uint64_t sequence = sequence_of(p.drop);
    float gamma[QT][4], beta[QT][4], dgamma[QT][4], dbeta[QT][4];
    int col[QT];
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        const int quad = i * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x);
        col[i] = quad < p.slice_quads ? min((rank * p.slice_quads + quad) * 4, p.columns) : p.columns;
        load_parameters(p.gamma, col[i], p.columns, 1.0f, gamma[i]);
        load_parameters(p.beta, col[i], p.columns, 0.0f, beta[i]);
#pragma unroll
        for (int k = 0; k < 4; ++k) dgamma[i][k] = dbeta[i][k] = 0.0f;
    }
    const float inverse = 1.0f / static_cast<float>(p.columns);
    raw_quad<SX> raw_x[QT];
    raw_quad<SG> raw_dy[QT];
    float2 stats = *reinterpret_cast<const float2 *>(p.stats + 2 * first);
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        raw_x[i].load(p.x.base + first * p.x.pitch, col[i], p.columns, p.per_access);
        raw_dy[i].load(p.dy.base + first * p.dy.pitch, col[i], p.columns, p.per_access);
    }
    if constexpr (CLUSTER) cluster_barrier(); // every block of the cluster has begun
    int turn = 0;
    for (std::int64_t row = first; row < p.rows; row += step, turn ^= 1) {
        const quad_terms terms{stats.x, stats.y, p.epilogue};
        float x[QT][4], dy[QT][4], sums[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            raw_x[i].widen(half, x[i]);
            raw_dy[i].widen(half_dy, dy[i]);
        }
        if (row + step < p.rows) {
            stats = *reinterpret_cast<const float2 *>(p.stats + 2 * (row + step));
#pragma unroll
            for (int i = 0; i < QT; ++i) {
                raw_x[i].load(p.x.base + (row + step) * p.x.pitch, col[i], p.columns, p.per_access);
                raw_dy[i].load(p.dy.base + (row + step) * p.dy.pitch, col[i], p.columns, p.per_access);
            }
        }
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            if (col[i] >= p.columns) continue;
            if (p.drop.on) drop_quad(p.drop, sequence, static_cast<std::uint32_t>(row), static_cast<std::uint32_t>(col[i] >> 2), dy[i]);
            terms.apply(x[i], dy[i], gamma[i], beta[i], dgamma[i], dbeta[i], sums);
        }
        around.add_up(sums, turn, rank, p.cluster);
        if (p.dx.base == nullptr) continue;
        sums[0] *= inverse;
        sums[1] *= inverse;
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            if (col[i] >= p.columns) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k) x[i][k] = terms.rstd * (dy[i][k] - sums[0] - x[i][k] * sums[1]);
            store_quad(p.dx.base + row * p.dx.pitch, col[i], p.columns, p.per_access, p.dx.dtype, x[i]);
        }
    }
    let_next_launch_start();
    if (p.partials == nullptr) return;
    float *out = p.partials + first * 2 * p.columns;
#pragma unroll
    for (int i = 0; i < QT; ++i) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (col[i] + k >= p.columns) continue;
            out[col[i] + k] = dgamma[i][k];
            out[p.columns + col[i] + k] = dbeta[i][k];
        }
    }
}

constexpr int kMeetWarps = 16;

// dgamma and dbeta from the parts' sums: a warp adds up every sixteenth part of 32 columns, then the warps' sums in order.
__global__ void __launch_bounds__(kMeetWarps * 32) layer_norm_meet_kernel(const float *partials, int parts, int columns, float *dgamma, float *dbeta) {
    __shared__ float meet[kMeetWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    wait_for_previous_launch();
    float v = 0.0f;
    if (c < 2 * columns) {
#pragma unroll 4
        for (int part = warp; part < parts; part += kMeetWarps) v += partials[static_cast<std::int64_t>(part) * 2 * columns + c];
    }
    meet[warp][lane] = v;
    __syncthreads();
    if (warp != 0 || c >= 2 * columns) return;
#pragma unroll
    for (int w = 1; w < kMeetWarps; ++w) v += meet[w][lane];
    float *out = c < columns ? dgamma : dbeta;
    if (out != nullptr) out[c < columns ? c : c - columns] = v;
}

struct backward_launch {
    layer_norm_params p;
    float *dgamma, *dbeta;
    int device;
    cudaStream_t stream;

    cb200_status finish(std::int64_t parts) const {
        count_launch();
        CB200_CUDA_OK(cudaGetLastError());
        if (p.partials == nullptr) return CB200_STATUS_SUCCESS;
        CB200_CUDA_OK(launch_kernel(true, layer_norm_meet_kernel, dim3(static_cast<unsigned>((2 * p.columns + 31) / 32)), kMeetWarps * 32, 0, stream,
                                    static_cast<const float *>(p.partials), static_cast<int>(parts), p.columns, dgamma, dbeta));
        count_launch();
        return CB200_STATUS_SUCCESS;
    }
    template<auto kernel>
    cb200_status wide(const wide_shape &shape) const {
        const std::int64_t parts = std::min<std::int64_t>({p.rows, kWideParts / shape.cluster, resident_clusters<kernel>(shape, device)});
        CB200_CUDA_OK(launch_wide(kernel, p, shape, static_cast<unsigned>(parts), stream));
        return finish(parts);
    }
    template<int SX, int SG>
    cb200_status run() {
        if (p.columns <= kNarrowColumns) {
            const std::int64_t per_block = kNarrowThreads / p.lanes, parts = std::min<std::int64_t>((p.rows + per_block - 1) / per_block, kNarrowParts);
            layer_norm_back_narrow_kernel<SX, SG><<<static_cast<unsigned>(parts), kNarrowThreads, 0, stream>>>(p);
            return finish(parts);
        }
        const wide_shape shape = wide_shape_of(p.columns);
        p.cluster = shape.cluster;
        p.slice_quads = shape.slice_quads;
        if (shape.cluster == 1) return wide<layer_norm_back_wide_kernel<SX, SG, 2, false>>(shape);
        if (shape.quads_per_thread == 2) return wide<layer_norm_back_wide_kernel<SX, SG, 2, true>>(shape);
        return wide<layer_norm_back_wide_kernel<SX, SG, 4, true>>(shape);
    }
};

std::uint64_t partial_bytes(std::int64_t rows, std::int64_t columns) {
    const std::int64_t parts = columns <= kNarrowColumns ? std::min<std::int64_t>((rows + kNarrowThreads / narrow_lanes(columns) - 1) / (kNarrowThreads / narrow_lanes(columns)), kNarrowParts)
                                                         : std::min<std::int64_t>(rows, kWideParts / wide_shape_of(columns).cluster);
    return static_cast<std::uint64_t>(parts) * 2u * static_cast<std::uint64_t>(columns) * sizeof(float);
}

} // namespace
} // namespace cb200

extern "C" cb200_status cb200_layer_norm_backward_workspace(int64_t rows, int64_t columns, uint64_t *bytes) {
    using namespace cb200;
    clear_error();
    if (bytes == nullptr) return fail(CB200_STATUS_INVALID_ARGUMENT, "workspace needs an output");
    if (rows < 0 || columns < 1 || columns > kMostColumns || rows > (1ll << 32))
        return fail(CB200_STATUS_INVALID_SHAPE, "the layer norm takes up to 2^32 rows of 1 to %lld columns, got %lld x %lld", (long long)kMostColumns, (long long)rows, (long long)columns);
    *bytes = partial_bytes(rows, columns);
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
    if (d->dgamma != nullptr && d->dgamma == d->dbeta) return fail(CB200_STATUS_INVALID_ARGUMENT, "dgamma and dbeta are the same vector");
    const bool sums = d->dgamma != nullptr || d->dbeta != nullptr;
    if (sums && p.rows > 0) {
        const std::uint64_t need = partial_bytes(p.rows, p.columns);
        if (d->workspace == nullptr || d->workspace_bytes < need || reinterpret_cast<std::uintptr_t>(d->workspace) % 4u != 0u)
            return fail(CB200_STATUS_INSUFFICIENT_WORKSPACE, "workspace of %llu bytes needed, %llu given", (unsigned long long)need,
                        (unsigned long long)(d->workspace == nullptr ? 0u : d->workspace_bytes));
        p.partials = static_cast<float *>(d->workspace);
    }
    p.per_access = columns_per_access(p.dy, p.per_access);
    if (p.dx.base != nullptr) p.per_access = columns_per_access(p.dx, p.per_access);
    b.dgamma = d->dgamma;
    b.dbeta = d->dbeta;
    b.device = d->device;
    b.stream = static_cast<cudaStream_t>(stream);
    device_scope scope(d->device);
    CB200_CUDA_OK(scope.status);
    if (p.rows == 0) { // sums over nothing
        if (b.dgamma != nullptr) CB200_CUDA_OK(cudaMemsetAsync(b.dgamma, 0, static_cast<std::size_t>(p.columns) * sizeof(float), b.stream));
        if (b.dbeta != nullptr) CB200_CUDA_OK(cudaMemsetAsync(b.dbeta, 0, static_cast<std::size_t>(p.columns) * sizeof(float), b.stream));
        return CB200_STATUS_SUCCESS;
    }
    if (!sums && p.dx.base == nullptr) return CB200_STATUS_SUCCESS;
    const bool wide_x = element_bytes(p.x.dtype) == 4, wide_dy = element_bytes(p.dy.dtype) == 4;
    if (wide_x) return wide_dy ? b.run<4, 4>() : b.run<4, 2>();
    return wide_dy ? b.run<2, 4>() : b.run<2, 2>();
}
