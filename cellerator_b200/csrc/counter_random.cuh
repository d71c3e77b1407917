// Random words from a counter, for dropout without a stored mask: Philox4x32 with ten rounds (J. K. Salmon, M. A. Moraes,
// R. O. Dror, D. E. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC'11).  One call makes four 32-bit words; value
// (row, column) of a matrix takes word column % 4 of counter {column / 4, row, sequence}, so that its word does not depend on
// how the matrix is stored, cut into shards or shared out to threads, and the backward pass makes it again.
#pragma once

#include "common.cuh"

#include <cmath>

namespace cb200 {

// What a kernel needs of a cb200_dropout.  threshold: a value whose word is below it is dropped.
struct dropout_args {
    std::uint32_t threshold = 0u;
    float scale = 1.0f;
    std::uint32_t key[10][2] = {}; // of the rounds: the same for every value, so they are operands out of the launch's constants
    std::uint64_t sequence = 0u;
    const std::uint64_t *device_sequence = nullptr;
    std::uint32_t first_row = 0u;
    int on = 0;
};

// d null: no dropout.  rows: of the call.
inline cb200_status dropout_of(const cb200_dropout *d, std::int64_t rows, dropout_args *out) {
    *out = dropout_args{};
    if (d == nullptr) return CB200_STATUS_SUCCESS;
    if (!(d->probability >= 0.0 && d->probability < 1.0))
        return fail(CB200_STATUS_INVALID_ARGUMENT, "dropout probability %g outside [0, 1)", d->probability);
    if (d->first_row < 0 || d->first_row > (1ll << 32) - rows)
        return fail(CB200_STATUS_INVALID_SHAPE, "dropout numbers rows below 2^32, got %lld from %lld", (long long)rows, (long long)d->first_row);
    if (reinterpret_cast<std::uintptr_t>(d->device_sequence) % 8u != 0u)
        return fail(CB200_STATUS_INVALID_ARGUMENT, "device_sequence is not aligned to 8 bytes");
    const double threshold = std::floor(d->probability * 4294967296.0 + 0.5);
    out->threshold = threshold >= 4294967295.0 ? 0xffffffffu : static_cast<std::uint32_t>(threshold);
    out->scale = static_cast<float>(1.0 / (1.0 - d->probability));
    for (std::uint32_t round = 0; round < 10; ++round) {
        out->key[round][0] = static_cast<std::uint32_t>(d->seed) + round * 0x9E3779B9u;
        out->key[round][1] = static_cast<std::uint32_t>(d->seed >> 32) + round * 0xBB67AE85u;
    }
    out->sequence = d->sequence;
    out->device_sequence = d->device_sequence;
    out->first_row = static_cast<std::uint32_t>(d->first_row);
    out->on = d->probability > 0.0 ? 1 : 0;
    return CB200_STATUS_SUCCESS;
}

#if defined(__CUDACC__)
__device__ __forceinline__ std::uint64_t sequence_of(const dropout_args &d) {
    return d.sequence + (d.device_sequence != nullptr ? *d.device_sequence : 0u);
}

// The words of columns 4 * quad ... 4 * quad + 3 of a row.  A round is two 32 x 32 -> 64-bit products and two three-way xors.
__device__ __forceinline__ void random_words(const dropout_args &d, std::uint64_t sequence, std::uint32_t row, std::uint32_t quad,
                                             std::uint32_t (&word)[4]) {
    std::uint32_t a = quad, b = row, c = static_cast<std::uint32_t>(sequence), e = static_cast<std::uint32_t>(sequence >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const std::uint64_t p = static_cast<std::uint64_t>(a) * 0xD2511F53u, q = static_cast<std::uint64_t>(c) * 0xCD9E8D57u;
        a = static_cast<std::uint32_t>(q >> 32) ^ b ^ d.key[round][0];
        b = static_cast<std::uint32_t>(q);
        c = static_cast<std::uint32_t>(p >> 32) ^ e ^ d.key[round][1];
        e = static_cast<std::uint32_t>(p);
    }
    word[0] = a; word[1] = b; word[2] = c; word[3] = e;
}

// v of columns 4 * quad ... of a row: dropped values become zero whatever they were, the others are scaled
__device__ __forceinline__ void drop_quad(const dropout_args &d, std::uint64_t sequence, std::uint32_t row, std::uint32_t quad, float (&v)[4]) {
    std::uint32_t word[4];
    random_words(d, sequence, d.first_row + row, quad, word);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = word[k] >= d.threshold ? v[k] * d.scale : 0.0f;
}
#endif

} // namespace cb200
