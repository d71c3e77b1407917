// Layer norm over the rows of a dense matrix, with the activation and the dropout that follow it in the same pass:
//     u = (x - mean) / sqrt(var + eps),  y = drop(act(gamma u + beta)).
// Mean and variance are sums in fp32 over values that stay in registers: the mean first, then the squares of what differs
// from it, so that a row far from zero loses nothing.
#include "layer_norm.cuh"

namespace cb200 {
namespace {

__device__ __forceinline__ bool held(int col, int k, int n, bool tail) { return tail ? col + k < n : col < n; }

// A group of p.lanes lanes per row.
template<int SIZE, bool TAIL>
__global__ void __launch_bounds__(kNarrowThreads) layer_norm_narrow_kernel(const layer_norm_params p) {
    const int lane = threadIdx.x & 31, in_row = lane & (p.lanes - 1), group = lane / p.lanes, rows_per_warp = 32 / p.lanes;
    const bool half = p.x.dtype == CB200_DTYPE_F16;
    const std::uint64_t sequence = sequence_of(p.drop);
    float gamma[kNarrowItems][4], beta[kNarrowItems][4];
    int col[kNarrowItems];
#pragma unroll
    for (int i = 0; i < kNarrowItems; ++i) {
        col[i] = (i * p.lanes + in_row) * 4;
        load_parameters(p.gamma, col[i], p.columns, 1.0f, gamma[i]);
        load_parameters(p.beta, col[i], p.columns, 0.0f, beta[i]);
    }
    const float inverse = 1.0f / static_cast<float>(p.columns);
    const std::int64_t warps = static_cast<std::int64_t>(gridDim.x) * (kNarrowThreads / 32);
    for (std::int64_t base = (static_cast<std::int64_t>(blockIdx.x) * (kNarrowThreads / 32) + (threadIdx.x >> 5)) * rows_per_warp; base < p.rows;
         base += warps * rows_per_warp) {
        const std::int64_t row = base + group;
        const bool active = row < p.rows;
        raw_quad<SIZE> raw[kNarrowItems];
#pragma unroll
        for (int i = 0; i < kNarrowItems; ++i) {
            raw[i].clear();
            if (active) raw[i].load(p.x.base + row * p.x.pitch, col[i], p.columns, p.per_access);
        }
        float v[kNarrowItems][4], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kNarrowItems; ++i) {
            raw[i].widen(half, v[i]);
            sum += (v[i][0] + v[i][1]) + (v[i][2] + v[i][3]);
        }
        const float mean = lane_sum(sum, p.lanes) / static_cast<float>(p.columns); // a division: exact for rows of one value
        float squares = 0.0f;
#pragma unroll
        for (int i = 0; i < kNarrowItems; ++i) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[i][k] -= mean;
                if (held(col[i], k, p.columns, TAIL)) squares = fmaf(v[i][k], v[i][k], squares);
            }
        }
        const float rstd = rsqrtf(lane_sum(squares, p.lanes) * inverse + p.epsilon);
        if (!active) continue;
        if (p.stats != nullptr && in_row == 0) *reinterpret_cast<float2 *>(p.stats + 2 * row) = make_float2(mean, rstd);
#pragma unroll
        for (int i = 0; i < kNarrowItems; ++i) {
            if (col[i] >= p.columns) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[i][k] = activation(fmaf(v[i][k] * rstd, gamma[i][k], beta[i][k]), p.epilogue);
            if (p.drop.on) drop_quad(p.drop, sequence, static_cast<std::uint32_t>(row), static_cast<std::uint32_t>(col[i] >> 2), v[i]);
            store_quad(p.y.base + row * p.y.pitch, col[i], p.columns, p.per_access, p.y.dtype, v[i]);
        }
    }
}

// A block or a cluster of blocks per row, each block with a slice of the columns; the next row's values are on their way while
// this one's sums go round.
template<int SIZE, int QT, bool CLUSTER>
__global__ void __launch_bounds__(kWideThreads) layer_norm_wide_kernel(const layer_norm_params p) {
    __shared__ wide_sums<1, CLUSTER> sums;
    const int rank = CLUSTER ? static_cast<int>(blockIdx.x) % p.cluster : 0;
    const std::int64_t first = CLUSTER ? blockIdx.x / p.cluster : blockIdx.x, step = CLUSTER ? gridDim.x / p.cluster : gridDim.x;
    const bool half = p.x.dtype == CB200_DTYPE_F16;
    const std::uint64_t sequence = sequence_of(p.drop);
    float gamma[QT][4], beta[QT][4];
    int col[QT];
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        const int quad = i * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x);
        col[i] = quad < p.slice_quads ? min((rank * p.slice_quads + quad) * 4, p.columns) : p.columns;
        load_parameters(p.gamma, col[i], p.columns, 1.0f, gamma[i]);
        load_parameters(p.beta, col[i], p.columns, 0.0f, beta[i]);
    }
    const float inverse = 1.0f / static_cast<float>(p.columns);
    raw_quad<SIZE> raw[QT];
#pragma unroll
    for (int i = 0; i < QT; ++i) raw[i].load(p.x.base + first * p.x.pitch, col[i], p.columns, p.per_access);
    if constexpr (CLUSTER) cluster_barrier(); // every block of the cluster has begun
    for (std::int64_t row = first; row < p.rows; row += step) {
        float v[QT][4], sum[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            raw[i].widen(half, v[i]);
            sum[0] += (v[i][0] + v[i][1]) + (v[i][2] + v[i][3]);
        }
        if (row + step < p.rows) {
#pragma unroll
            for (int i = 0; i < QT; ++i) raw[i].load(p.x.base + (row + step) * p.x.pitch, col[i], p.columns, p.per_access);
        }
        sums.add_up(sum, 0, rank, p.cluster);
        const float mean = sum[0] / static_cast<float>(p.columns);
        sum[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < QT; ++i) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[i][k] -= mean;
                if (col[i] + k < p.columns) sum[0] = fmaf(v[i][k], v[i][k], sum[0]);
            }
        }
        sums.add_up(sum, 1, rank, p.cluster);
        const float rstd = rsqrtf(sum[0] * inverse + p.epsilon);
        if (p.stats != nullptr && rank == 0 && threadIdx.x == 0) *reinterpret_cast<float2 *>(p.stats + 2 * row) = make_float2(mean, rstd);
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            if (col[i] >= p.columns) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[i][k] = activation(fmaf(v[i][k] * rstd, gamma[i][k], beta[i][k]), p.epilogue);
            if (p.drop.on) drop_quad(p.drop, sequence, static_cast<std::uint32_t>(row), static_cast<std::uint32_t>(col[i] >> 2), v[i]);
            store_quad(p.y.base + row * p.y.pitch, col[i], p.columns, p.per_access, p.y.dtype, v[i]);
        }
    }
}

template<auto kernel>
cb200_status launch_wide_forward(const layer_norm_params &p, const wide_shape &shape, int device, cudaStream_t stream) {
    const std::int64_t clusters = std::min<std::int64_t>(p.rows, resident_clusters<kernel>(shape, device));
    CB200_CUDA_OK(launch_wide(kernel, p, shape, static_cast<unsigned>(clusters), stream));
    count_launch();
    return CB200_STATUS_SUCCESS;
}

template<int SIZE>
cb200_status launch_forward(layer_norm_params p, int device, cudaStream_t stream) {
    if (p.columns <= kNarrowColumns) {
        const std::int64_t per_block = kNarrowThreads / p.lanes;
        const unsigned grid = static_cast<unsigned>(std::min<std::int64_t>((p.rows + per_block - 1) / per_block, 148 * 4));
        if (p.columns % 4 != 0) layer_norm_narrow_kernel<SIZE, true><<<grid, kNarrowThreads, 0, stream>>>(p);
        else layer_norm_narrow_kernel<SIZE, false><<<grid, kNarrowThreads, 0, stream>>>(p);
        count_launch();
        CB200_CUDA_OK(cudaGetLastError());
        return CB200_STATUS_SUCCESS;
    }
    const wide_shape shape = wide_shape_of(p.columns);
    p.cluster = shape.cluster;
    p.slice_quads = shape.slice_quads;
    if (shape.cluster == 1) return launch_wide_forward<layer_norm_wide_kernel<SIZE, 2, false>>(p, shape, device, stream);
    if (shape.quads_per_thread == 2) return launch_wide_forward<layer_norm_wide_kernel<SIZE, 2, true>>(p, shape, device, stream);
    return launch_wide_forward<layer_norm_wide_kernel<SIZE, 4, true>>(p, shape, device, stream);
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
    return element_bytes(p.x.dtype) == 4 ? launch_forward<4>(p, d->device, s) : launch_forward<2>(p, d->device, s);
}
