// What the forward and the backward pass of the layer norm share: the checks of a call, how narrow rows lie in a warp, activations,
// and sums over lanes.
#pragma once

#include "counter_random.cuh"
#include "row_quads.cuh"

#include <algorithm>
#include <type_traits>

namespace cb200 {

// Widths.  Up to 1,024 columns (backward 512) a row belongs to a group of lanes of one warp, wider ones to a block; backward, rows that
// no block holds are taken in two passes.
constexpr int kBlockColumns = 4608; // of a row that one block holds, backward
constexpr std::int64_t kMostColumns = 65536;
constexpr int kNarrowThreads = 256;

struct layer_norm_params {
    row_matrix x, y, dy, dx;
    const float *gamma, *beta;
    float *stats;          // [rows][2]: mean, 1 / standard deviation
    float *partials;       // backward: [parts][2][columns]
    std::int64_t rows;
    int columns;
    int per_access;        // columns that a load or store of every one of the matrices can take
    int lanes;             // narrow: lanes of a row, a power of two
    int epilogue;
    float epsilon;
    dropout_args drop;
};

// Backward pass of rows that no block holds (layer_norm_columns.cu): parts of the sums of dgamma and dbeta, bytes of the rows' sums,
// launch.  p.partials (for the parts) and `sums` are the caller's; sums is needed where p.dx is.
std::int64_t layer_norm_columns_parts(std::int64_t rows, std::int64_t columns);
std::uint64_t layer_norm_columns_sums_bytes(std::int64_t rows, std::int64_t columns);
cb200_status launch_layer_norm_columns(const layer_norm_params &p, float *sums, cudaStream_t stream);

// How a narrow row is laid over the lanes of a warp: a power of two of them, with so many quads each that few are left empty (an
// empty quad costs what a full one does: 8 columns with GELU and dropout took 211 us with four quads to a lane, 112 with two), and
// of equal choices the first of `items`.
struct narrow_shape {
    int items, lanes;
};
inline narrow_shape narrow_shape_of(std::int64_t columns, const int *items, int choices) {
    const std::int64_t quads = (columns + 3) / 4;
    narrow_shape best{0, 0};
    for (int i = 0; i < choices; ++i) {
        int lanes = 1;
        while (lanes < 32 && lanes * items[i] < quads) lanes *= 2;
        if (lanes * items[i] >= quads && (best.lanes == 0 || lanes * items[i] < best.lanes * best.items)) best = narrow_shape{items[i], lanes};
    }
    return best;
}

inline cb200_status layer_norm_checked(const cb200_layer_norm *d, bool backward, layer_norm_params *p) {
    if (d == nullptr || d->version != CB200_ABI_VERSION || d->size < sizeof(cb200_layer_norm))
        return fail(CB200_STATUS_INVALID_ARGUMENT, "bad cb200_layer_norm header");
    if (d->rows < 0 || d->columns < 1 || d->columns > kMostColumns || d->rows >= (1ll << 32))
        return fail(CB200_STATUS_INVALID_SHAPE, "the layer norm takes fewer than 2^32 rows of 1 to %lld columns, got %lld x %lld", (long long)kMostColumns,
                    (long long)d->rows, (long long)d->columns);
    if (d->epilogue != CB200_EPILOGUE_NONE && d->epilogue != CB200_EPILOGUE_RELU && d->epilogue != CB200_EPILOGUE_GELU_ERF &&
        d->epilogue != CB200_EPILOGUE_GELU_TANH)
        return fail(CB200_STATUS_UNSUPPORTED, "the layer norm's epilogue is none, relu, gelu_erf or gelu_tanh (its bias is beta), got kind %d", d->epilogue);
    cb200_status st = row_matrix_of(d->x, d->x_ld, d->x_dtype, d->rows, d->columns, "x", &p->x);
    if (st == CB200_STATUS_SUCCESS) st = dropout_of(&d->dropout, d->rows, &p->drop);
    if (st != CB200_STATUS_SUCCESS) return st;
    const float *vectors[] = {d->gamma, d->beta, d->dgamma, d->dbeta};
    for (const float *v : vectors)
        if (reinterpret_cast<std::uintptr_t>(v) % 4u != 0u) return fail(CB200_STATUS_INVALID_ARGUMENT, "a vector of parameters is not aligned to its elements");
    if (reinterpret_cast<std::uintptr_t>(d->stats) % 8u != 0u) return fail(CB200_STATUS_INVALID_ARGUMENT, "stats is not aligned to 8 bytes");
    p->gamma = d->gamma;
    p->beta = d->beta;
    p->stats = d->stats;
    p->rows = d->rows;
    p->columns = static_cast<int>(d->columns);
    p->epilogue = d->epilogue;
    p->epsilon = d->epsilon;
    p->per_access = columns_per_access(p->x, columns_of_access(d->columns));
    if (!backward && !(d->epsilon >= 0.0f && d->epsilon < 3.4e38f)) return fail(CB200_STATUS_INVALID_ARGUMENT, "epsilon %g is no number from 0 on", d->epsilon);
    return CB200_STATUS_SUCCESS;
}

#if defined(__CUDACC__)
// A quad of a parameter vector; `otherwise` where there is no vector or no column.
__device__ __forceinline__ void load_parameters(const float *v, int col, int n, float otherwise, float (&out)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) out[k] = v != nullptr && col + k < n ? __ldg(v + col + k) : otherwise;
}

// The same where the vector is known to be there, in one load where `vectors` says that it lies on a 16-byte boundary and the quad
// lies in it.
__device__ __forceinline__ float4 load_parameter_quad(const float *v, int col, int n, bool vectors) {
    if (vectors && col + 4 <= n) return __ldg(reinterpret_cast<const float4 *>(v + col));
    float w[4];
    load_parameters(v, col, n, 0.0f, w);
    return make_float4(w[0], w[1], w[2], w[3]);
}
inline __host__ __device__ bool on_16_bytes(const void *p) { return reinterpret_cast<std::uintptr_t>(p) % 16u == 0u; }

// 2^t and 1 / t by the hardware's approximations, within 2 units and 1 unit of the last place; what is too small for a normal number
// is 0.
__device__ __forceinline__ float fast_exp2(float t) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    return e;
}
__device__ __forceinline__ float fast_reciprocal(float t) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
    return r;
}
__device__ __forceinline__ pair fast_exp2(pair t) {
    float lo, hi;
    t.get(lo, hi);
    return pair(fast_exp2(lo), fast_exp2(hi));
}
__device__ __forceinline__ pair fast_reciprocal(pair t) {
    float lo, hi;
    t.get(lo, hi);
    return pair(fast_reciprocal(lo), fast_reciprocal(hi));
}
// z^2, cut off above 10^6, where the tanh form's factor is 0 or 1 long since
__device__ __forceinline__ pair square(pair z) {
    float lo, hi;
    (z * z).get(lo, hi);
    return pair(fminf(lo, 1e6f), fminf(hi, 1e6f));
}
// The factor of the tanh form of GELU, (1 + tanh(c (z + 0.044715 z^3))) / 2 with c = sqrt(2 / pi): the logistic function of twice that
// argument, within a few units of the last place of 1.  zz: square(z).
__device__ __forceinline__ pair tanh_gate(pair z, pair zz) {
    // -2 c / ln 2 and 0.044715 of it
    return fast_reciprocal(fast_exp2(z * fma(pair(-0.10294324f), zz, pair(-2.3022082f))) + pair(1.0f));
}

// Phi(z) = (1 + erf(z / sqrt 2)) / 2 by formula 7.1.26 of Abramowitz and Stegun (C. Hastings, 1955): off by 0.75e-7 itself, by 4.5e-7 at most
// with fp32's roundings and what the two approximations are granted (3.5e-7 seen, next to 0), at z = -3 by 1e-4 of itself, at -5 by 2e-3, and
// smoothly 0 and 1 far out.  erff, whose branches a warp takes both, made the forward pass of 48 million values with dropout 112 us.  tail:
// e^(-z z / 2), which the slope needs as well.
__device__ __forceinline__ pair normal_integral(pair z, pair &tail) {
    float lo, hi;
    z.get(lo, hi);
    const pair t = fast_reciprocal(fma(pair(fabsf(lo), fabsf(hi)), pair(0.23164189f), pair(1.0f))); // 0.3275911 / sqrt 2
    pair poly = fma(t, pair(0.5307027145f), pair(-0.7265760135f));
    poly = fma(t, poly, pair(0.7107068705f));
    poly = fma(t, poly, pair(-0.142248368f));
    poly = t * fma(t, poly, pair(0.127414796f));
    tail = fast_exp2(z * pair(-0.72134752f) * z);
    float outside_lo, outside_hi;
    (poly * tail).get(outside_lo, outside_hi);
    return pair(lo >= 0.0f ? 1.0f - outside_lo : outside_lo, hi >= 0.0f ? 1.0f - outside_hi : outside_hi);
}

// act(z)
template<int KIND>
__device__ __forceinline__ pair activation(pair z) {
    if constexpr (KIND == CB200_EPILOGUE_RELU) {
        float lo, hi;
        z.get(lo, hi);
        return pair(lo < 0.0f ? 0.0f : lo, hi < 0.0f ? 0.0f : hi); // NaN stays
    }
    if constexpr (KIND == CB200_EPILOGUE_GELU_ERF) {
        pair tail(0.0f);
        return normal_integral(z, tail) * z;
    }
    if constexpr (KIND == CB200_EPILOGUE_GELU_TANH) return tanh_gate(z, square(z)) * z;
    return z;
}

// dy act'(z); relu's slope is 0 at 0, and lets nothing of dy through there
template<int KIND>
__device__ __forceinline__ pair through_activation(pair dy, pair z) {
    if constexpr (KIND == CB200_EPILOGUE_RELU) {
        float lo, hi, dy_lo, dy_hi;
        z.get(lo, hi);
        dy.get(dy_lo, dy_hi);
        return pair(lo <= 0.0f ? 0.0f : dy_lo, hi <= 0.0f ? 0.0f : dy_hi);
    }
    if constexpr (KIND == CB200_EPILOGUE_GELU_ERF) {
        pair tail(0.0f);
        const pair integral = normal_integral(z, tail);
        return fma(z * pair(0.39894228f), tail, integral) * dy;
    }
    if constexpr (KIND == CB200_EPILOGUE_GELU_TANH) {
        const pair zz = square(z), gate = tanh_gate(z, zz);
        // 0 far from 0, times finite numbers; for z from 3 to 6 the rounding of 1 - gate, times z (1.6 + 0.2 z^2), is up to 2e-6 of a slope of 1
        const pair steep = fma(gate, pair(-1.0f), pair(1.0f)) * gate;
        return fma(z * steep, fma(pair(0.21406445f), zz, pair(1.5957691f)), gate) * dy; // 2 c and 3 times 0.044715 of it
    }
    return dy;
}

// Some quads at once: the choices are made once for all of them, as a branch for each costs a quarter of the instructions.
template<int KIND, int Q>
__device__ __forceinline__ void activate_as(float (&v)[Q][4]) {
#pragma unroll
    for (int i = 0; i < Q; ++i) {
#pragma unroll
        for (int k = 0; k < 4; k += 2) activation<KIND>(pair(v[i][k], v[i][k + 1])).get(v[i][k], v[i][k + 1]);
    }
}
template<int Q>
__device__ __forceinline__ void activate(int kind, float (&v)[Q][4]) {
    if (kind == CB200_EPILOGUE_NONE) return;
    if (kind == CB200_EPILOGUE_RELU) activate_as<CB200_EPILOGUE_RELU>(v);
    else if (kind == CB200_EPILOGUE_GELU_ERF) activate_as<CB200_EPILOGUE_GELU_ERF>(v);
    else activate_as<CB200_EPILOGUE_GELU_TANH>(v);
}
// dz in place of dy, from u
template<int KIND, int Q>
__device__ __forceinline__ void through_as(float (&dy)[Q][4], const float (&u)[Q][4], const float4 (&gamma)[Q], const float4 (&beta)[Q]) {
#pragma unroll
    for (int i = 0; i < Q; ++i) {
        through_activation<KIND>(pair(dy[i][0], dy[i][1]), fma(pair(u[i][0], u[i][1]), pair(gamma[i].x, gamma[i].y), pair(beta[i].x, beta[i].y))).get(dy[i][0], dy[i][1]);
        through_activation<KIND>(pair(dy[i][2], dy[i][3]), fma(pair(u[i][2], u[i][3]), pair(gamma[i].z, gamma[i].w), pair(beta[i].z, beta[i].w))).get(dy[i][2], dy[i][3]);
    }
}
// Calls f with the epilogue as a constant: one branch for all that f does.
template<typename F>
__device__ __forceinline__ void with_epilogue(int kind, F f) {
    if (kind == CB200_EPILOGUE_NONE) f(std::integral_constant<int, CB200_EPILOGUE_NONE>{});
    else if (kind == CB200_EPILOGUE_RELU) f(std::integral_constant<int, CB200_EPILOGUE_RELU>{});
    else if (kind == CB200_EPILOGUE_GELU_ERF) f(std::integral_constant<int, CB200_EPILOGUE_GELU_ERF>{});
    else f(std::integral_constant<int, CB200_EPILOGUE_GELU_TANH>{});
}
template<int Q>
__device__ __forceinline__ void drop_quads(const dropout_args &d, std::uint64_t sequence, std::uint32_t row, const int (&col)[Q], float (&v)[Q][4]) {
    if (!d.on) return;
#pragma unroll
    for (int i = 0; i < Q; ++i) drop_quad(d, sequence, row, static_cast<std::uint32_t>(col[i]) >> 2, v[i]);
}

// Brings `bytes` bytes at p on their way to L2, whole pieces of 16 bytes from the one that p lies in; p is not the start of its
// allocation (a row behind the first), so that the bytes in front of it are there.
__device__ __forceinline__ void prefetch_bytes(const unsigned char *p, std::uint32_t bytes) {
    const std::uint64_t from = reinterpret_cast<std::uint64_t>(p) & ~std::uint64_t{15}, to = (reinterpret_cast<std::uint64_t>(p) + bytes) & ~std::uint64_t{15};
    if (to > from) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from), "r"(static_cast<std::uint32_t>(to - from)) : "memory");
}

// Sums over groups of `lanes` neighbouring lanes (a power of two), in each of them.
template<int N>
__device__ __forceinline__ void lane_sums(float (&v)[N], int lanes) {
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        if (off >= lanes) break;
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
    }
}

template<int N>
__device__ __forceinline__ void warp_sums(float (&v)[N]) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
    }
}
#endif

} // namespace cb200
