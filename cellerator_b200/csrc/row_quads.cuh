// Rows of dense fp32, bf16 or fp16 matrices, four neighbouring columns ("a quad") at a time, and what the row operators
// check of them.
#pragma once

#include "common.cuh"

#include <cuda_fp16.h>

namespace cb200 {

// Rows of a dense matrix, of any leading dimension.
struct row_matrix {
    unsigned char *base = nullptr;
    std::int64_t pitch = 0; // bytes
    int dtype = CB200_DTYPE_F32;
};

inline int element_bytes(int dtype) { return dtype == CB200_DTYPE_F32 ? 4 : dtype == CB200_DTYPE_BF16 || dtype == CB200_DTYPE_F16 ? 2 : 0; }

// rows x columns at `data`, `ld` elements from row to row
inline cb200_status row_matrix_of(const void *data, std::int64_t ld, int dtype, std::int64_t rows, std::int64_t columns, const char *name, row_matrix *out) {
    const int bytes = element_bytes(dtype);
    if (bytes == 0) return fail(CB200_STATUS_UNSUPPORTED, "%s: type %d is none of fp32, bf16, fp16", name, dtype);
    if (data == nullptr && rows > 0 && columns > 0) return fail(CB200_STATUS_INVALID_ARGUMENT, "%s is null", name);
    if (reinterpret_cast<std::uintptr_t>(data) % static_cast<unsigned>(bytes) != 0u)
        return fail(CB200_STATUS_INVALID_ARGUMENT, "%s is not aligned to its %d-byte elements", name, bytes);
    if (rows > 1 && ld < columns) return fail(CB200_STATUS_INVALID_SHAPE, "%s: leading dimension %lld smaller than %lld columns", name, (long long)ld, (long long)columns);
    if (rows > 1 && ld > (1ll << 58) / rows) return fail(CB200_STATUS_INVALID_SHAPE, "%s: leading dimension %lld", name, (long long)ld);
    out->base = static_cast<unsigned char *>(const_cast<void *>(data));
    out->pitch = rows > 1 ? ld * bytes : columns * bytes;
    out->dtype = dtype;
    return CB200_STATUS_SUCCESS;
}

// Whether a result may be written over an operand: they are the same rows, element for element, or share no byte.
inline bool rows_compatible(const row_matrix &out, const row_matrix &in, std::int64_t rows, std::int64_t columns) {
    if (out.base == nullptr || in.base == nullptr || rows <= 0 || columns <= 0) return true;
    const std::int64_t out_width = columns * element_bytes(out.dtype), in_width = columns * element_bytes(in.dtype);
    if (out.base == in.base && out.pitch == in.pitch && out_width == in_width) return true;
    const auto o = reinterpret_cast<std::uintptr_t>(out.base), i = reinterpret_cast<std::uintptr_t>(in.base);
    if (o + static_cast<std::uintptr_t>((rows - 1) * out.pitch + out_width) <= i || i + static_cast<std::uintptr_t>((rows - 1) * in.pitch + in_width) <= o) return true;
    if (out.pitch != in.pitch) return false;
    // columns side by side in the same rows
    const std::int64_t apart = static_cast<std::int64_t>(o > i ? (o - i) % static_cast<std::uintptr_t>(in.pitch)
                                                               : (in.pitch - static_cast<std::int64_t>((i - o) % static_cast<std::uintptr_t>(in.pitch))) % in.pitch);
    return apart >= in_width && apart + out_width <= in.pitch;
}

// Columns that one load or store takes: 4, 2 or 1, by the alignment of every row.
inline int columns_per_access(const row_matrix &m, int most) {
    const int bytes = element_bytes(m.dtype);
    while (most > 1 && (reinterpret_cast<std::uintptr_t>(m.base) % static_cast<unsigned>(most * bytes) != 0u || m.pitch % (most * bytes) != 0)) most /= 2;
    return most;
}

#if defined(__CUDACC__)
// The bits of a quad of elements of SIZE bytes.
template<int SIZE>
struct raw_quad {
    std::uint32_t w[SIZE];

    // columns col ... col + 3 of the row at `row`; those from n on are zero
    __device__ __forceinline__ void load(const unsigned char *row, int col, int n, int per_access) {
        const unsigned char *p = row + static_cast<std::int64_t>(col) * SIZE;
        if (col + 4 <= n) {
            if (per_access == 4) {
                if constexpr (SIZE == 4) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(p);
                    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
                } else {
                    const uint2 v = *reinterpret_cast<const uint2 *>(p);
                    w[0] = v.x; w[1] = v.y;
                }
            } else if (per_access == 2) {
                if constexpr (SIZE == 4) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(p), u = *reinterpret_cast<const uint2 *>(p + 8);
                    w[0] = v.x; w[1] = v.y; w[2] = u.x; w[3] = u.y;
                } else {
                    w[0] = *reinterpret_cast<const std::uint32_t *>(p);
                    w[1] = *reinterpret_cast<const std::uint32_t *>(p + 4);
                }
            } else {
                if constexpr (SIZE == 4) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) w[k] = reinterpret_cast<const std::uint32_t *>(p)[k];
                } else {
                    const unsigned short *h = reinterpret_cast<const unsigned short *>(p);
                    const std::uint32_t h0 = h[0], h1 = h[1], h2 = h[2], h3 = h[3];
                    w[0] = h0 | h1 << 16;
                    w[1] = h2 | h3 << 16;
                }
            }
            return;
        }
#pragma unroll
        for (int k = 0; k < SIZE; ++k) w[k] = 0u;
        if (col < n) {
            if constexpr (SIZE == 4) {
#pragma unroll
                for (int k = 0; k < 3; ++k)
                    if (col + k < n) w[k] = reinterpret_cast<const std::uint32_t *>(p)[k];
            } else {
                const unsigned short *h = reinterpret_cast<const unsigned short *>(p);
                w[0] = h[0];
                if (col + 1 < n) w[0] |= static_cast<std::uint32_t>(h[1]) << 16;
                if (col + 2 < n) w[1] = h[2];
            }
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int k = 0; k < SIZE; ++k) w[k] = 0u;
    }
    // half: fp16 and not bf16, of two-byte elements
    __device__ __forceinline__ void widen(bool half, float (&v)[4]) const {
        if constexpr (SIZE == 4) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = __uint_as_float(w[k]);
        } else if (half) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                __half2 h;
                memcpy(&h, &w[k], 4);
                const float2 f = __half22float2(h);
                v[2 * k] = f.x;
                v[2 * k + 1] = f.y;
            }
        } else {
            bf16x2_to_f32(w[0], v[0], v[1]);
            bf16x2_to_f32(w[1], v[2], v[3]);
        }
    }
};

__device__ __forceinline__ std::uint32_t pack_pair(float lo, float hi, bool half) {
    std::uint32_t w;
    if (half) {
        const __half2 h = __floats2half2_rn(lo, hi);
        memcpy(&w, &h, 4);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        memcpy(&w, &h, 4);
    }
    return w;
}

// One rounding, to nearest, where the type has fewer bits than fp32.
__device__ __forceinline__ void store_quad(unsigned char *row, int col, int n, int per_access, int dtype, const float (&v)[4]) {
    if (col >= n) return;
    if (dtype == CB200_DTYPE_F32) {
        float *p = reinterpret_cast<float *>(row) + col;
        if (col + 4 <= n && per_access == 4) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
        else if (col + 4 <= n && per_access == 2) {
            reinterpret_cast<float2 *>(p)[0] = make_float2(v[0], v[1]);
            reinterpret_cast<float2 *>(p)[1] = make_float2(v[2], v[3]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (col + k < n) p[k] = v[k];
        }
        return;
    }
    const bool half = dtype == CB200_DTYPE_F16;
    unsigned short *p = reinterpret_cast<unsigned short *>(row) + col;
    const std::uint32_t lo = pack_pair(v[0], v[1], half), hi = pack_pair(v[2], v[3], half);
    if (col + 4 <= n && per_access == 4) *reinterpret_cast<uint2 *>(p) = make_uint2(lo, hi);
    else if (col + 4 <= n && per_access == 2) {
        reinterpret_cast<std::uint32_t *>(p)[0] = lo;
        reinterpret_cast<std::uint32_t *>(p)[1] = hi;
    } else {
        const unsigned short e[4] = {static_cast<unsigned short>(lo), static_cast<unsigned short>(lo >> 16), static_cast<unsigned short>(hi),
                                     static_cast<unsigned short>(hi >> 16)};
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (col + k < n) p[k] = e[k];
    }
}
#endif

} // namespace cb200
