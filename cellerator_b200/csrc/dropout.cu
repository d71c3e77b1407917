// Dropout of a dense matrix with a mask that is never stored: y = x / (1 - p) where the value's random word keeps it, else 0.
// The gradient is the same call on the gradient of y.
#include "counter_random.cuh"
#include "row_quads.cuh"

#include <algorithm>
#include <type_traits>

namespace cb200 {
namespace {

constexpr int kThreads = 256, kInFlight = 4, kBlocks = 3; // resident on an SM

struct dropout_params {
    row_matrix x, y;
    dropout_args drop;
    std::uint32_t rows;
    std::uint32_t pieces;                 // of a row: of Q quads each
    std::uint32_t step_rows, step_pieces; // from one piece of a thread to its next
    int columns, per_access;
};

// A thread works on pieces of Q quads that lie a launch's width apart; it goes from one to the next by adding rows and pieces,
// with no division.  Q = 2 for two-byte elements in rows of whole 16-byte pieces, where a piece is one load and one store.
// WHOLE: rows are whole pieces and every access is aligned.
//
// Bound by integer work: ten rounds are 20 products of 32 x 32 bits and 20 xors for four values, whatever the type; the ALU pipe is busy 54 % of
// the cycles, the FMA pipe, which multiplies, 37 %, and warps wait for one of them or to be dispatched to it.  500,000 x 128
// bf16 64 us (4.0 TB/s, 61 % of a copy; 68 with 8-byte pieces, 89 before loads and stores lost their branches); 48 million values of
// fp32 70 us (84 %), of bf16 49 us (59 %).  The rounds' keys come out of the launch's constants: worked out by each thread, they were
// 20 more additions.
template<int SIZE, bool HALVES, int Q, bool WHOLE>
__global__ void __launch_bounds__(kThreads, kBlocks) dropout_kernel(const dropout_params p) {
    const std::uint64_t first = static_cast<std::uint64_t>(blockIdx.x) * kThreads + threadIdx.x;
    const std::uint64_t sequence = sequence_of(p.drop);
    const bool half = p.x.dtype == CB200_DTYPE_F16;
    std::uint64_t row = first / p.pieces;
    std::uint32_t piece = static_cast<std::uint32_t>(first - row * p.pieces);
    while (row < p.rows) {
        raw_quad<SIZE> raw[kInFlight][Q];
        std::uint32_t r[kInFlight], at[kInFlight];
        bool in[kInFlight];
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) {
            r[i] = static_cast<std::uint32_t>(row);
            at[i] = piece;
            in[i] = row < p.rows;
            row += p.step_rows;
            piece += p.step_pieces;
            if (piece >= p.pieces) {
                piece -= p.pieces;
                ++row;
            }
            if (!in[i]) continue;
            const unsigned char *x = p.x.base + r[i] * p.x.pitch;
            if constexpr (WHOLE && Q == 2) {
                const uint4 v = *reinterpret_cast<const uint4 *>(x + static_cast<std::uint64_t>(at[i]) * 16u);
                raw[i][0].w[0] = v.x; raw[i][0].w[1] = v.y; raw[i][1].w[0] = v.z; raw[i][1].w[1] = v.w;
            } else if constexpr (WHOLE) {
                raw[i][0].template load<4>(x + static_cast<std::uint64_t>(at[i]) * (4u * SIZE), 4);
            } else {
                const int col[1] = {static_cast<int>(at[i]) * 4};
                load_quads(x, col, p.columns, p.per_access, raw[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) {
            if (!in[i]) break;
            float v[Q][4];
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                raw[i][q].template widen<HALVES>(half, v[q]);
                if (p.drop.on) drop_quad(p.drop, sequence, r[i], at[i] * Q + q, v[q]);
            }
            unsigned char *y = p.y.base + r[i] * p.y.pitch;
            if constexpr (WHOLE && Q == 2) { // a result of two bytes as well
                const bool y_half = HALVES && p.y.dtype == CB200_DTYPE_F16;
                *reinterpret_cast<uint4 *>(y + static_cast<std::uint64_t>(at[i]) * 16u) =
                    make_uint4(pack_pair(v[0][0], v[0][1], y_half), pack_pair(v[0][2], v[0][3], y_half), pack_pair(v[1][0], v[1][1], y_half),
                               pack_pair(v[1][2], v[1][3], y_half));
            } else {
                const int col[1] = {static_cast<int>(at[i]) * 4};
                store_quads<HALVES>(y, col, p.columns, WHOLE ? 4 : p.per_access, p.y.dtype, v);
            }
        }
    }
}

template<int SIZE, bool HALVES, int Q, bool WHOLE>
cb200_status launch(dropout_params p, std::int64_t rows, cudaStream_t stream) {
    p.rows = static_cast<std::uint32_t>(rows);
    p.pieces = static_cast<std::uint32_t>((p.columns + 4ll * Q - 1) / (4 * Q));
    const std::int64_t threads = (rows * static_cast<std::int64_t>(p.pieces) + kInFlight - 1) / kInFlight;
    const unsigned grid = static_cast<unsigned>(std::min<std::int64_t>((threads + kThreads - 1) / kThreads, 148 * kBlocks));
    const std::int64_t step = static_cast<std::int64_t>(grid) * kThreads;
    p.step_rows = static_cast<std::uint32_t>(step / p.pieces);
    p.step_pieces = static_cast<std::uint32_t>(step % p.pieces);
    dropout_kernel<SIZE, HALVES, Q, WHOLE><<<grid, kThreads, 0, stream>>>(p);
    count_launch();
    CB200_CUDA_OK(cudaGetLastError());
    return CB200_STATUS_SUCCESS;
}

} // namespace
} // namespace cb200

extern "C" cb200_status cb200_dropout_rows(const cb200_dropout_matrix *m, void *stream) {
    using namespace cb200;
    clear_error();
    if (m == nullptr || m->version != CB200_ABI_VERSION || m->size < sizeof(cb200_dropout_matrix))
        return fail(CB200_STATUS_INVALID_ARGUMENT, "bad cb200_dropout_matrix header");
    if (m->rows < 0 || m->columns < 0 || m->columns > (1ll << 30) || m->rows >= (1ll << 32)) // a place in a row is a 32-bit number of bytes
        return fail(CB200_STATUS_INVALID_SHAPE, "dropout takes fewer than 2^32 rows of up to 2^30 columns, got %lld x %lld", (long long)m->rows, (long long)m->columns);
    dropout_params p{};
    cb200_status st = row_matrix_of(m->x, m->x_ld, m->x_dtype, m->rows, m->columns, "x", &p.x);
    if (st == CB200_STATUS_SUCCESS) st = row_matrix_of(m->y, m->y_ld, m->y_dtype, m->rows, m->columns, "y", &p.y);
    if (st == CB200_STATUS_SUCCESS) st = dropout_of(&m->dropout, m->rows, &p.drop);
    if (st != CB200_STATUS_SUCCESS) return st;
    if (!rows_compatible(p.y, p.x, m->rows, m->columns)) return fail(CB200_STATUS_INVALID_ARGUMENT, "y overlaps x without being x");
    device_scope scope(m->device);
    CB200_CUDA_OK(scope.status);
    if (m->rows == 0 || m->columns == 0) return CB200_STATUS_SUCCESS;
    p.columns = static_cast<int>(m->columns);
    p.per_access = columns_per_access(p.y, columns_per_access(p.x, columns_of_access(m->columns)));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool whole = p.per_access == 4;
    const auto run = [&](auto halves) {
        constexpr bool H = decltype(halves)::value;
        if (element_bytes(p.x.dtype) == 4) return whole ? launch<4, H, 1, true>(p, m->rows, s) : launch<4, H, 1, false>(p, m->rows, s);
        if (whole && element_bytes(p.y.dtype) == 2 && p.columns % 8 == 0 && columns_per_access(p.x, 8) == 8 && columns_per_access(p.y, 8) == 8)
            return launch<2, H, 2, true>(p, m->rows, s);
        return whole ? launch<2, H, 1, true>(p, m->rows, s) : launch<2, H, 1, false>(p, m->rows, s);
    };
    return p.x.dtype == CB200_DTYPE_F16 || p.y.dtype == CB200_DTYPE_F16 ? run(std::true_type{}) : run(std::false_type{});
}
