// Layer norm over the rows of a dense matrix, with the activation and the dropout that follow it in the same pass:
//     u = (x - mean) / sqrt(var + eps),  y = drop(act(gamma u + beta)).
// Mean and variance are sums in fp32 over values that stay in registers: the mean first, then the squares of what differs
// from it, so that a row far from zero loses nothing.
#include "layer_norm.cuh"

namespace cb200 {
namespace {

constexpr int kNarrowBlocks = 3; // resident on an SM

// A group of p.lanes lanes per row; the next rows' values are on their way while these are worked on.  gamma and beta come out of
// shared memory: a lane's sixteen columns of them would take a third of its registers.
template<int SIZE, int KIND>
__global__ void __launch_bounds__(kNarrowThreads, kNarrowBlocks) layer_norm_narrow_kernel(const layer_norm_params p) {
    __shared__ __align__(16) float parameters[2][kNarrowColumns];
    const int lane = threadIdx.x & 31, in_row = lane & (p.lanes - 1), group = lane / p.lanes, rows_per_warp = 32 / p.lanes;
    const bool half = p.x.dtype == CB200_DTYPE_F16, affine = p.gamma != nullptr || p.beta != nullptr;
    const std::uint64_t sequence = sequence_of(p.drop);
    int col[kNarrowItems];
#pragma unroll
    for (int i = 0; i < kNarrowItems; ++i) col[i] = min((i * p.lanes + in_row) * 4, p.columns);
    const float count = static_cast<float>(p.columns), inverse = 1.0f / count;
    const std::int64_t step = static_cast<std::int64_t>(gridDim.x) * (kNarrowThreads / 32) * rows_per_warp;
    std::int64_t row = (static_cast<std::int64_t>(blockIdx.x) * (kNarrowThreads / 32) + (threadIdx.x >> 5)) * rows_per_warp + group;
    raw_quad<SIZE> raw[kNarrowItems];
    if (row < p.rows) load_quads(p.x.base + row * p.x.pitch, col, p.columns, p.per_access, raw);
    if (affine) {
        for (int c = threadIdx.x; c < kNarrowColumns; c += kNarrowThreads) {
            parameters[0][c] = p.gamma != nullptr && c < p.columns ? __ldg(p.gamma + c) : 1.0f;
            parameters[1][c] = p.beta != nullptr && c < p.columns ? __ldg(p.beta + c) : 0.0f;
        }
        __syncthreads();
    }
    for (; row - group < p.rows; row += step) {
        float v[kNarrowItems][4], sum[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < kNarrowItems; ++i) {
            raw[i].widen(half, v[i]);
            sum[0] += (v[i][0] + v[i][1]) + (v[i][2] + v[i][3]);
        }
        if (row + step < p.rows) load_quads(p.x.base + (row + step) * p.x.pitch, col, p.columns, p.per_access, raw);
        lane_sums(sum, p.lanes);
        const float mean = sum[0] / count; // a division: exact for rows of one value
        sum[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < kNarrowItems; ++i) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[i][k] -= mean;
            if (col[i] + 4 > p.columns) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (col[i] + k >= p.columns) v[i][k] = 0.0f;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[0] = fmaf(v[i][k], v[i][k], sum[0]);
        }
        lane_sums(sum, p.lanes);
        const float rstd = rsqrtf(fmaf(sum[0], inverse, p.epsilon));
        if (row >= p.rows) continue;
        if (p.stats != nullptr && in_row == 0) *reinterpret_cast<float2 *>(p.stats + 2 * row) = make_float2(mean, rstd);
#pragma unroll
        for (int i = 0; i < kNarrowItems; ++i) {
            if (col[i] >= p.columns) continue;
            if (affine) {
                const float4 g = *reinterpret_cast<const float4 *>(parameters[0] + col[i]), b = *reinterpret_cast<const float4 *>(parameters[1] + col[i]);
                v[i][0] = activation<KIND>(fmaf(v[i][0] * rstd, g.x, b.x));
                v[i][1] = activation<KIND>(fmaf(v[i][1] * rstd, g.y, b.y));
                v[i][2] = activation<KIND>(fmaf(v[i][2] * rstd, g.z, b.z));
                v[i][3] = activation<KIND>(fmaf(v[i][3] * rstd, g.w, b.w));
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[i][k] = activation<KIND>(v[i][k] * rstd);
            }
            if (p.drop.on) drop_quad(p.drop, sequence, static_cast<std::uint32_t>(row), static_cast<std::uint32_t>(col[i] >> 2), v[i]);
        }
        store_quads(p.y.base + row * p.y.pitch, col, p.columns, p.per_access, p.y.dtype, v);
    }
}

// Rows of a step of a wide kernel.
template<int SIZE, int QT>
constexpr int kWideRows = (QT == 3 ? 8 : 4) / SIZE;

// A block, or a cluster of blocks that take a slice of the columns each, works on R rows at a time.  Each warp takes the mean of
// its columns and the squares of what differs from that; from all warps' numbers come the row's mean and variance,
//     mean = sum of sums / N,  N var = sum over warps of (squares + n (warp's mean - mean)^2),
// with one exchange between them.  In a cluster the exchange of one step of rows goes round while the step before is written
// and the one behind it is summed.
template<int SIZE, int KIND, int QT, bool CLUSTER>
__global__ void __launch_bounds__(wide_threads(QT)) layer_norm_wide_kernel(const layer_norm_params p) {
    constexpr int R = kWideRows<SIZE, QT>;
    __shared__ wide_notes<2 * R, CLUSTER> notes;
    __shared__ float sizes[(CLUSTER ? kMostCluster : 1) * kMostWarps]; // columns of each warp
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, all_warps = p.cluster * warps;
    const int rank = CLUSTER ? static_cast<int>(blockIdx.x) % p.cluster : 0;
    const std::int64_t first = (CLUSTER ? blockIdx.x / p.cluster : blockIdx.x) * static_cast<std::int64_t>(R);
    const std::int64_t stride = (CLUSTER ? gridDim.x / p.cluster : gridDim.x) * static_cast<std::int64_t>(R);
    const bool half = p.x.dtype == CB200_DTYPE_F16;
    const std::uint64_t sequence = sequence_of(p.drop);
    float gamma[QT][4], beta[QT][4];
    int col[QT];
    wide_columns<QT>(p, rank, col);
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        load_parameters(p.gamma, col[i], p.columns, 1.0f, gamma[i]);
        load_parameters(p.beta, col[i], p.columns, 0.0f, beta[i]);
    }
    const auto columns_of = [&](int w) { // of warp w of the block with this rank
        return [&, w](int of_rank) {
            int n = 0;
            for (int i = 0; i < QT; ++i) {
                const int begin = i * static_cast<int>(blockDim.x) + w * 32, end = min(begin + 32, p.slice_quads);
                if (begin < end) n += max(0, min((of_rank * p.slice_quads + end) * 4, p.columns) - min((of_rank * p.slice_quads + begin) * 4, p.columns));
            }
            return n;
        };
    };
    for (int i = threadIdx.x; i < all_warps; i += blockDim.x) sizes[i] = static_cast<float>(columns_of(i % warps)(i / warps));
    const float size = static_cast<float>(columns_of(warp)(rank)), inverse_size = size > 0.0f ? 1.0f / size : 0.0f;
    const float count = static_cast<float>(p.columns), inverse = 1.0f / count;

    raw_quad<SIZE> now[R][QT], next[R][QT], before[R][QT];
    const auto fetch = [&](raw_quad<SIZE> (&raw)[R][QT], std::int64_t at) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (at + r < p.rows) load_quads(p.x.base + (at + r) * p.x.pitch, col, p.columns, p.per_access, raw[r]);
        }
    };
    // {sum, squares of what differs from the warp's mean} of each row
    const auto summed = [&](float (&v)[2 * R]) {
        float t[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            t[r] = 0.0f;
#pragma unroll
            for (int i = 0; i < QT; ++i) {
                float x[4];
                now[r][i].widen(half, x);
                t[r] += (x[0] + x[1]) + (x[2] + x[3]);
            }
        }
        warp_sums<R>(t);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            v[r] = t[r];
            const float mean = t[r] * inverse_size;
            t[r] = 0.0f;
#pragma unroll
            for (int i = 0; i < QT; ++i) {
                float x[4];
                now[r][i].widen(half, x);
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] -= mean;
                if (col[i] + 4 > p.columns) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (col[i] + k >= p.columns) x[k] = 0.0f;
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) t[r] = fmaf(x[k], x[k], t[r]);
            }
        }
        warp_sums<R>(t);
#pragma unroll
        for (int r = 0; r < R; ++r) v[R + r] = t[r];
    };
    const auto finish = [&](const raw_quad<SIZE> (&raw)[R][QT], std::int64_t at, int set) {
        float mean[R], var[R];
#pragma unroll
        for (int r = 0; r < R; ++r) mean[r] = var[r] = 0.0f;
        for (int w = lane; w < all_warps; w += 32) {
#pragma unroll
            for (int r = 0; r < R; ++r) mean[r] += notes.note[set][w][r];
        }
        warp_sums<R>(mean);
#pragma unroll
        for (int r = 0; r < R; ++r) mean[r] /= count; // exact for rows of one value
        for (int w = lane; w < all_warps; w += 32) {
            const float n = sizes[w], over = n > 0.0f ? 1.0f / n : 0.0f;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float off = fmaf(notes.note[set][w][r], over, -mean[r]);
                var[r] += fmaf(n * off, off, notes.note[set][w][R + r]);
            }
        }
        warp_sums<R>(var);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const std::int64_t row = at + r;
            if (row >= p.rows) break;
            const float rstd = rsqrtf(var[r] * inverse + p.epsilon);
            if (p.stats != nullptr && rank == 0 && threadIdx.x == 0) *reinterpret_cast<float2 *>(p.stats + 2 * row) = make_float2(mean[r], rstd);
            float v[QT][4];
#pragma unroll
            for (int i = 0; i < QT; ++i) {
                raw[r][i].widen(half, v[i]);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[i][k] = activation<KIND>(fmaf((v[i][k] - mean[r]) * rstd, gamma[i][k], beta[i][k]));
                if (p.drop.on) drop_quad(p.drop, sequence, static_cast<std::uint32_t>(row), static_cast<std::uint32_t>(col[i] >> 2), v[i]);
            }
            store_quads(p.y.base + row * p.y.pitch, col, p.columns, p.per_access, p.y.dtype, v);
        }
    };

    fetch(now, first);
    int set = 0;
    if constexpr (CLUSTER) {
        cluster_arrive(); // every block of the cluster has begun
        std::int64_t row = first;
        for (; row < p.rows; row += stride) {
            float v[2 * R];
            summed(v);
            cluster_wait();
            notes.leave(v, set, rank, p.cluster);
            cluster_arrive();
            fetch(next, row + stride);
            if (row != first) finish(before, row - stride, set == 0 ? 2 : set - 1);
            set = next_set(set, 3);
#pragma unroll
            for (int r = 0; r < R; ++r) {
#pragma unroll
                for (int i = 0; i < QT; ++i) {
                    before[r][i] = now[r][i];
                    now[r][i] = next[r][i];
                }
            }
        }
        cluster_wait();
        if (row != first) finish(before, row - stride, set == 0 ? 2 : set - 1);
    } else {
        for (std::int64_t row = first; row < p.rows; row += stride, set ^= 1) {
            float v[2 * R];
            summed(v);
            notes.leave(v, set, rank, p.cluster);
            fetch(next, row + stride);
            __syncthreads();
            finish(now, row, set);
#pragma unroll
            for (int r = 0; r < R; ++r) {
#pragma unroll
                for (int i = 0; i < QT; ++i) now[r][i] = next[r][i];
            }
        }
    }
}

template<int SIZE, int KIND, int QT, bool CLUSTER>
cb200_status launch_wide_forward(const layer_norm_params &p, const wide_shape &shape, int device, cudaStream_t stream) {
    constexpr auto kernel = layer_norm_wide_kernel<SIZE, KIND, QT, CLUSTER>;
    constexpr int step = kWideRows<SIZE, QT>;
    const std::int64_t clusters = std::min<std::int64_t>((p.rows + step - 1) / step, resident_clusters<kernel>(shape, device));
    CB200_CUDA_OK(launch_wide(kernel, p, shape, static_cast<unsigned>(clusters), stream));
    count_launch();
    return CB200_STATUS_SUCCESS;
}

template<int SIZE, int KIND>
cb200_status launch_forward(layer_norm_params p, int device, cudaStream_t stream) {
    if (p.columns <= kNarrowColumns) {
        const std::int64_t per_block = kNarrowThreads / p.lanes, blocks = (p.rows + per_block - 1) / per_block;
        layer_norm_narrow_kernel<SIZE, KIND><<<static_cast<unsigned>(std::min<std::int64_t>(blocks, 148 * kNarrowBlocks)), kNarrowThreads, 0, stream>>>(p);
        count_launch();
        CB200_CUDA_OK(cudaGetLastError());
        return CB200_STATUS_SUCCESS;
    }
    const wide_shape shape = wide_shape_of(p.columns);
    p.cluster = shape.cluster;
    p.slice_quads = shape.slice_quads;
    if (shape.cluster == 1) return launch_wide_forward<SIZE, KIND, 3, false>(p, shape, device, stream);
    if (shape.quads_per_thread == 3) return launch_wide_forward<SIZE, KIND, 3, true>(p, shape, device, stream);
    return launch_wide_forward<SIZE, KIND, 4, true>(p, shape, device, stream);
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
    return with_epilogue(p.epilogue, [&](auto kind) {
        return element_bytes(p.x.dtype) == 4 ? launch_forward<4, kind()>(p, d->device, s) : launch_forward<2, kind()>(p, d->device, s);
    });
}
