// Dropout of a dense matrix with a mask that is never stored: y = x / (1 - p) where the value's random word keeps it, else 0.
// The gradient is the same call on the gradient of y.
#include "counter_random.cuh"
#include "row_quads.cuh"

#include <algorithm>

namespace cb200 {
namespace {

constexpr int kThreads = 256, kInFlight = 4;

struct dropout_params {
    row_matrix x, y;
    dropout_args drop;
    std::uint32_t rows;
    std::uint32_t quads;                 // of a row
    std::uint32_t step_rows, step_quads; // from one quad of a thread to its next
    int columns, per_access;
};

// A thread's quads lie a launch's width apart; it goes from one to the next by adding rows and quads, with no division.
template<int SIZE>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const dropout_params p) {
    const std::uint64_t first = static_cast<std::uint64_t>(blockIdx.x) * kThreads + threadIdx.x;
    const std::uint64_t sequence = sequence_of(p.drop);
    const bool half = p.x.dtype == CB200_DTYPE_F16;
    std::uint64_t row = first / p.quads;
    std::uint32_t quad = static_cast<std::uint32_t>(first - row * p.quads);
    while (row < p.rows) {
        raw_quad<SIZE> raw[kInFlight];
        std::uint32_t r[kInFlight], q[kInFlight];
        bool in[kInFlight];
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) {
            r[i] = static_cast<std::uint32_t>(row);
            q[i] = quad;
            in[i] = row < p.rows;
            row += p.step_rows;
            quad += p.step_quads;
            if (quad >= p.quads) {
                quad -= p.quads;
                ++row;
            }
            if (in[i]) raw[i].load(p.x.base + r[i] * p.x.pitch, static_cast<int>(q[i]) * 4, p.columns, p.per_access);
        }
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) {
            if (!in[i]) break;
            float v[4];
            raw[i].widen(half, v);
            if (p.drop.on) drop_quad(p.drop, sequence, r[i], q[i], v);
            store_quad(p.y.base + r[i] * p.y.pitch, static_cast<int>(q[i]) * 4, p.columns, p.per_access, p.y.dtype, v);
        }
    }
}

} // namespace
} // namespace cb200

extern "C" cb200_status cb200_dropout_rows(const cb200_dropout_matrix *m, void *stream) {
    using namespace cb200;
    clear_error();
    if (m == nullptr || m->version != CB200_ABI_VERSION || m->size < sizeof(cb200_dropout_matrix))
        return fail(CB200_STATUS_INVALID_ARGUMENT, "bad cb200_dropout_matrix header");
    if (m->rows < 0 || m->columns < 0 || m->columns > 0x7ffffff0ll || m->rows >= (1ll << 32))
        return fail(CB200_STATUS_INVALID_SHAPE, "dropout takes fewer than 2^32 rows of fewer than 2^31 columns, got %lld x %lld", (long long)m->rows, (long long)m->columns);
    dropout_params p{};
    cb200_status st = row_matrix_of(m->x, m->x_ld, m->x_dtype, m->rows, m->columns, "x", &p.x);
    if (st == CB200_STATUS_SUCCESS) st = row_matrix_of(m->y, m->y_ld, m->y_dtype, m->rows, m->columns, "y", &p.y);
    if (st == CB200_STATUS_SUCCESS) st = dropout_of(&m->dropout, m->rows, &p.drop);
    if (st != CB200_STATUS_SUCCESS) return st;
    if (!rows_compatible(p.y, p.x, m->rows, m->columns)) return fail(CB200_STATUS_INVALID_ARGUMENT, "y overlaps x without being x");
    device_scope scope(m->device);
    CB200_CUDA_OK(scope.status);
    if (m->rows == 0 || m->columns == 0) return CB200_STATUS_SUCCESS;
    p.rows = static_cast<std::uint32_t>(m->rows);
    p.columns = static_cast<int>(m->columns);
    p.quads = static_cast<std::uint32_t>((m->columns + 3) / 4);
    p.per_access = columns_per_access(p.y, columns_per_access(p.x, 4));
    const std::int64_t threads = (m->rows * static_cast<std::int64_t>(p.quads) + kInFlight - 1) / kInFlight;
    const unsigned grid = static_cast<unsigned>(std::min<std::int64_t>((threads + kThreads - 1) / kThreads, 148 * 8));
    const std::int64_t step = static_cast<std::int64_t>(grid) * kThreads;
    p.step_rows = static_cast<std::uint32_t>(step / p.quads);
    p.step_quads = static_cast<std::uint32_t>(step % p.quads);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (element_bytes(p.x.dtype) == 4) dropout_kernel<4><<<grid, kThreads, 0, s>>>(p);
    else dropout_kernel<2><<<grid, kThreads, 0, s>>>(p);
    count_launch();
    CB200_CUDA_OK(cudaGetLastError());
    return CB200_STATUS_SUCCESS;
}
