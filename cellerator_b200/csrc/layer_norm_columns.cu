// Gradients of the layer norm over rows that no block can hold (more than 4,608 columns), in two passes: the first adds up h and h u
// of each row, piece by piece of its columns; the second, whose threads own columns, reads x and dy again, writes dx, adds up
// dgamma and dbeta, and waits for nobody.  It begins with the rows that the first read last, which are in L2 still.
//
// Bound by HBM: five values a place, where one pass would move three.  1,025 x 33,538 fp32: 141 us, 74 % of a copy.  A cluster of eight blocks per row,
// each holding a slice of it and passing its sums round, moved three and took 162 to 170 us: a barrier of the cluster for every row
// (its release waits for the stores in front of it), with one block of 17 warps on an SM.  Both passes over 40, 80 or 120 MB of x and
// dy at a time, so that the second finds them in L2, took 195, 176 and 170 us where all rows at once took 145: launches too short.
#include "dependent_launch.cuh"
#include "layer_norm.cuh"

namespace cb200 {
namespace {

constexpr int kSumThreads = 256, kSumRows = 4, kPiece = 4 * 4 * kSumThreads; // rows of a block, columns of a piece
constexpr int kColumnThreads = 128, kTileRows = 64, kRowsAhead = 4;
constexpr std::int64_t kMostParts = 128, kColumnBlocks = 148 * 16; // of a launch, about

struct columns_params {
    layer_norm_params p;
    float *sums; // [rows][pieces][2]
    int pieces;
    std::int64_t part_rows;
};

// h and h u of a quad, added up
template<int KIND>
__device__ __forceinline__ void add_terms(const float (&u)[1][4], float (&dz)[1][4], const float4 (&gamma)[1], const float4 (&beta)[1], float &h, float &hu) {
    if constexpr (KIND != CB200_EPILOGUE_NONE) through_as<KIND>(dz, u, gamma, beta);
    const pair s = pair(dz[0][0], dz[0][1]) * pair(gamma[0].x, gamma[0].y), t = pair(dz[0][2], dz[0][3]) * pair(gamma[0].z, gamma[0].w);
    h += (s + t).sum();
    hu += fma(t, pair(u[0][2], u[0][3]), s * pair(u[0][0], u[0][1])).sum();
}
// u in place of x
__device__ __forceinline__ void normalise(float (&x)[1][4], float mean, float rstd) {
    const pair minus_mean(-mean), scale(rstd);
#pragma unroll
    for (int k = 0; k < 4; k += 2) ((pair(x[0][k], x[0][k + 1]) + minus_mean) * scale).get(x[0][k], x[0][k + 1]);
}

// A block: four rows of a piece of 4,096 columns; gamma and beta of a thread's columns serve all four.
template<int SX, int SG, bool HALVES>
__global__ void __launch_bounds__(kSumThreads, 3) layer_norm_sums_kernel(const columns_params c) {
    __shared__ float meet[kSumThreads / 32][2 * kSumRows];
    const layer_norm_params &p = c.p;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = p.columns;
    const bool half = p.x.dtype == CB200_DTYPE_F16, half_dy = p.dy.dtype == CB200_DTYPE_F16;
    const int piece = static_cast<int>(blockIdx.x % static_cast<unsigned>(c.pieces));
    const std::int64_t row0 = static_cast<std::int64_t>(blockIdx.x / static_cast<unsigned>(c.pieces)) * kSumRows;
    const std::uint64_t sequence = sequence_of(p.drop);
    float mean[kSumRows], rstd[kSumRows], sums[2 * kSumRows];
#pragma unroll
    for (int r = 0; r < kSumRows; ++r) {
        const std::int64_t row = min(row0 + r, p.rows - 1);
        mean[r] = __ldg(p.stats + 2 * row);
        rstd[r] = __ldg(p.stats + 2 * row + 1);
        sums[2 * r] = sums[2 * r + 1] = 0.0f;
    }
    const int end = min(n, (piece + 1) * kPiece);
    for (int at = piece * kPiece + static_cast<int>(threadIdx.x) * 4; at < end; at += 4 * kSumThreads) {
        const int col[1] = {at};
        raw_quad<SX> raw_x[kSumRows][1];
        raw_quad<SG> raw_dy[kSumRows][1];
#pragma unroll
        for (int r = 0; r < kSumRows; ++r) {
            const std::int64_t row = min(row0 + r, p.rows - 1);
            load_quads(p.x.base + row * p.x.pitch, col, n, p.per_access, raw_x[r]);
            load_quads(p.dy.base + row * p.dy.pitch, col, n, p.per_access, raw_dy[r]);
        }
        float g[4], b[4];
        load_parameters(p.gamma, at, n, 1.0f, g);
        load_parameters(p.beta, at, n, 0.0f, b);
        const float4 gamma[1] = {make_float4(g[0], g[1], g[2], g[3])}, beta[1] = {make_float4(b[0], b[1], b[2], b[3])};
        const auto rows = [&](auto kind) {
#pragma unroll
            for (int r = 0; r < kSumRows; ++r) {
                float u[1][4], dz[1][4];
                raw_x[r][0].template widen<HALVES>(half, u[0]);
                raw_dy[r][0].template widen<HALVES>(half_dy, dz[0]);
                drop_quads(p.drop, sequence, static_cast<std::uint32_t>(row0 + r), col, dz);
                normalise(u, mean[r], rstd[r]);
                add_terms<decltype(kind)::value>(u, dz, gamma, beta, sums[2 * r], sums[2 * r + 1]);
            }
        };
        with_epilogue(p.epilogue, rows);
    }
    let_next_launch_start();
    warp_sums(sums);
    if (lane == 0) {
#pragma unroll
        for (int k = 0; k < 2 * kSumRows; ++k) meet[warp][k] = sums[k];
    }
    __syncthreads();
    if (threadIdx.x < 2 * kSumRows) {
        const int r = threadIdx.x >> 1;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kSumThreads / 32; ++w) v += meet[w][threadIdx.x];
        if (row0 + r < p.rows) c.sums[((row0 + r) * c.pieces + piece) * 2 + (threadIdx.x & 1)] = v;
    }
}

// A block: 512 columns, a quad to a thread, of a part of the rows, 64 at a time.  Blocks of an SM by registers: with five, GELU and
// dropout over 48 million values of 33,538 columns took 256 us (fp32) and 237 (bf16), with six and seven 243 and 225.
template<int SX, int SG, bool HALVES>
__global__ void __launch_bounds__(kColumnThreads, SX + SG == 4 ? 7 : 6) layer_norm_columns_kernel(const columns_params c) {
    __shared__ float4 of_row[kTileRows]; // mean, 1 / standard deviation, mean of h, mean of h u
    const layer_norm_params &p = c.p;
    const int n = p.columns, col[1] = {min((static_cast<int>(blockIdx.x) * kColumnThreads + static_cast<int>(threadIdx.x)) * 4, (n + 3) & ~3)};
    const bool half = p.x.dtype == CB200_DTYPE_F16, half_dy = p.dy.dtype == CB200_DTYPE_F16;
    const std::int64_t part = gridDim.y - 1 - blockIdx.y, part_end = min(p.rows, (part + 1) * c.part_rows);
    const std::uint64_t sequence = sequence_of(p.drop);
    float g[4], b[4];
    load_parameters(p.gamma, col[0], n, 1.0f, g);
    load_parameters(p.beta, col[0], n, 0.0f, b);
    const float4 gamma[1] = {make_float4(g[0], g[1], g[2], g[3])}, beta[1] = {make_float4(b[0], b[1], b[2], b[3])};
    const float inverse = 1.0f / static_cast<float>(n);
    pair dgamma_sum[2] = {pair(0.0f), pair(0.0f)}, dbeta_sum[2] = {pair(0.0f), pair(0.0f)};
    wait_for_previous_launch();
    for (std::int64_t row0 = part * c.part_rows; row0 < part_end; row0 += kTileRows) {
        const int rows = static_cast<int>(min(static_cast<std::int64_t>(kTileRows), part_end - row0));
        if (threadIdx.x < rows) {
            float h = 0.0f, hu = 0.0f;
            if (p.dx.base != nullptr) {
                const float *sums = c.sums + (row0 + threadIdx.x) * c.pieces * 2;
                for (int i = 0; i < c.pieces; ++i) {
                    h += sums[2 * i];
                    hu += sums[2 * i + 1];
                }
            }
            const float2 s = *reinterpret_cast<const float2 *>(p.stats + 2 * (row0 + threadIdx.x));
            of_row[threadIdx.x] = make_float4(s.x, s.y, h * inverse, hu * inverse);
        }
        __syncthreads();
        pair tile_dgamma[2] = {pair(0.0f), pair(0.0f)}, tile_dbeta[2] = {pair(0.0f), pair(0.0f)};
        for (int first = 0; first < rows; first += kRowsAhead) {
            raw_quad<SX> raw_x[kRowsAhead][1];
            raw_quad<SG> raw_dy[kRowsAhead][1];
#pragma unroll
            for (int r = 0; r < kRowsAhead; ++r) {
                const std::int64_t row = row0 + min(first + r, rows - 1);
                load_quads(p.x.base + row * p.x.pitch, col, n, p.per_access, raw_x[r]);
                load_quads(p.dy.base + row * p.dy.pitch, col, n, p.per_access, raw_dy[r]);
            }
            const auto some = [&](auto kind) {
#pragma unroll
                for (int r = 0; r < kRowsAhead; ++r) {
                    if (first + r >= rows) break;
                    const float4 s = of_row[first + r];
                    float u[1][4], dz[1][4];
                    raw_x[r][0].template widen<HALVES>(half, u[0]);
                    raw_dy[r][0].template widen<HALVES>(half_dy, dz[0]);
                    drop_quads(p.drop, sequence, static_cast<std::uint32_t>(row0 + first + r), col, dz);
                    normalise(u, s.x, s.y);
                    if constexpr (decltype(kind)::value != CB200_EPILOGUE_NONE) through_as<decltype(kind)::value>(dz, u, gamma, beta);
                    float dx[1][4];
                    const pair scale(s.y), minus_h(-s.z), minus_hu(-s.w);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const pair z(dz[0][2 * k], dz[0][2 * k + 1]), v(u[0][2 * k], u[0][2 * k + 1]);
                        tile_dbeta[k] = tile_dbeta[k] + z;
                        tile_dgamma[k] = fma(z, v, tile_dgamma[k]);
                        (scale * fma(v, minus_hu, fma(z, pair(g[2 * k], g[2 * k + 1]), minus_h))).get(dx[0][2 * k], dx[0][2 * k + 1]);
                    }
                    if (p.dx.base != nullptr) store_quads<HALVES>(p.dx.base + (row0 + first + r) * p.dx.pitch, col, n, p.per_access, p.dx.dtype, dx);
                }
            };
            with_epilogue(p.epilogue, some);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            dgamma_sum[k] = dgamma_sum[k] + tile_dgamma[k];
            dbeta_sum[k] = dbeta_sum[k] + tile_dbeta[k];
        }
        __syncthreads();
    }
    let_next_launch_start();
    if (p.partials == nullptr) return;
    float dgamma[4], dbeta[4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        dgamma_sum[k].get(dgamma[2 * k], dgamma[2 * k + 1]);
        dbeta_sum[k].get(dbeta[2 * k], dbeta[2 * k + 1]);
    }
    float *out = p.partials + part * 2 * n;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (col[0] + k >= n) continue;
        out[col[0] + k] = dgamma[k];
        out[n + col[0] + k] = dbeta[k];
    }
}

std::int64_t pieces_of(std::int64_t columns) { return (columns + kPiece - 1) / kPiece; }
unsigned column_blocks(std::int64_t columns) { return static_cast<unsigned>((columns + 4 * kColumnThreads - 1) / (4 * kColumnThreads)); }
// Rows of a part: as many parts as give every SM 16 blocks, but 16 rows in each.
std::int64_t part_rows(std::int64_t rows, std::int64_t columns) {
    const std::int64_t parts = std::min(kMostParts, std::max<std::int64_t>(1, kColumnBlocks / column_blocks(columns)));
    return std::max<std::int64_t>(16, (rows + parts - 1) / parts);
}

template<int SX, int SG, bool HALVES>
cb200_status run_passes(const columns_params &c, cudaStream_t stream) {
    const bool first = c.p.dx.base != nullptr;
    if (first) {
        const std::int64_t blocks = (c.p.rows + kSumRows - 1) / kSumRows * c.pieces;
        if (blocks > 0x7fffffffll) return fail(CB200_STATUS_INVALID_SHAPE, "too many rows of so many columns for one launch");
        layer_norm_sums_kernel<SX, SG, HALVES><<<static_cast<unsigned>(blocks), kSumThreads, 0, stream>>>(c);
        count_launch();
        CB200_CUDA_OK(cudaGetLastError());
    }
    CB200_CUDA_OK(launch_kernel(first, layer_norm_columns_kernel<SX, SG, HALVES>, dim3(column_blocks(c.p.columns), static_cast<unsigned>((c.p.rows + c.part_rows - 1) / c.part_rows)),
                                kColumnThreads, 0, stream, c));
    count_launch();
    return CB200_STATUS_SUCCESS;
}

} // namespace

std::int64_t layer_norm_columns_parts(std::int64_t rows, std::int64_t columns) {
    const std::int64_t of_part = part_rows(rows, columns);
    return (rows + of_part - 1) / of_part;
}
std::uint64_t layer_norm_columns_sums_bytes(std::int64_t rows, std::int64_t columns) { return static_cast<std::uint64_t>(rows * pieces_of(columns) * 2) * sizeof(float); }

cb200_status launch_layer_norm_columns(const layer_norm_params &p, float *sums, cudaStream_t stream) {
    columns_params c{};
    c.p = p;
    c.sums = sums;
    c.pieces = static_cast<int>(pieces_of(p.columns));
    c.part_rows = part_rows(p.rows, p.columns);
    const bool wide_x = element_bytes(p.x.dtype) == 4, wide_dy = element_bytes(p.dy.dtype) == 4;
    const auto of_sizes = [&](auto halves) {
        constexpr bool H = decltype(halves)::value;
        if (wide_x) return wide_dy ? run_passes<4, 4, H>(c, stream) : run_passes<4, 2, H>(c, stream);
        return wide_dy ? run_passes<2, 4, H>(c, stream) : run_passes<2, 2, H>(c, stream);
    };
    return p.x.dtype == CB200_DTYPE_F16 || p.dy.dtype == CB200_DTYPE_F16 || (p.dx.base != nullptr && p.dx.dtype == CB200_DTYPE_F16) ? of_sizes(std::true_type{}) : of_sizes(std::false_type{});
}

} // namespace cb200
