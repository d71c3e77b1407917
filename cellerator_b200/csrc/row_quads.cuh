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

// Columns that one load or store takes: 4, 2 or 1, so that every row is whole accesses, each of them aligned.
inline int columns_of_access(std::int64_t columns) { return columns % 4 == 0 ? 4 : columns % 2 == 0 ? 2 : 1; }
inline int columns_per_access(const row_matrix &m, int most) {
    const int bytes = element_bytes(m.dtype);
    while (most > 1 && (reinterpret_cast<std::uintptr_t>(m.base) % static_cast<unsigned>(most * bytes) != 0u || m.pitch % (most * bytes) != 0)) most /= 2;
    return most;
}

#if defined(__CUDACC__)
// Two fp32 operations in one instruction: half the issue slots where a kernel is short of them.
struct pair {
    unsigned long long bits;
    __device__ __forceinline__ pair(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(lo), "f"(hi)); }
    __device__ __forceinline__ explicit pair(float both) : pair(both, both) {}
    __device__ __forceinline__ void get(float &lo, float &hi) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(bits)); }
    __device__ __forceinline__ float sum() const {
        float lo, hi;
        get(lo, hi);
        return lo + hi;
    }
};
__device__ __forceinline__ pair operator+(pair a, pair b) {
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a.bits) : "l"(b.bits));
    return a;
}
__device__ __forceinline__ pair operator*(pair a, pair b) {
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a.bits) : "l"(b.bits));
    return a;
}
__device__ __forceinline__ pair fma(pair a, pair b, pair c) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c.bits) : "l"(a.bits), "l"(b.bits));
    return c;
}

// The bits of a quad of elements of SIZE bytes.
template<int SIZE>
struct raw_quad {
    std::uint32_t w[SIZE];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int k = 0; k < SIZE; ++k) w[k] = 0u;
    }
    // those of its columns at p that are among the `count` left of the row, in loads of PER_ACCESS elements; the others are zero
    template<int PER_ACCESS>
    __device__ __forceinline__ void load(const unsigned char *p, int count) {
        clear();
        if constexpr (SIZE == 4 && PER_ACCESS == 4) {
            if (count <= 0) return;
            const uint4 v = *reinterpret_cast<const uint4 *>(p);
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else if constexpr (SIZE * PER_ACCESS == 8) {
#pragma unroll
            for (int k = 0; k < SIZE; k += 2) {
                if (k * 4 / SIZE >= count) continue;
                const uint2 v = *reinterpret_cast<const uint2 *>(p + 4 * k);
                w[k] = v.x;
                w[k + 1] = v.y;
            }
        } else if constexpr (SIZE * PER_ACCESS == 4) {
#pragma unroll
            for (int k = 0; k < SIZE; ++k)
                if (k * 4 / SIZE < count) w[k] = *reinterpret_cast<const std::uint32_t *>(p + 4 * k);
        } else {
            std::uint32_t h[4] = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < count) h[k] = reinterpret_cast<const unsigned short *>(p)[k];
            w[0] = h[0] | h[1] << 16;
            w[1] = h[2] | h[3] << 16;
        }
    }
    // half: fp16 and not bf16, of two-byte elements.  HALVES: whether they can be at all; a choice at run time would convert both ways.
    template<bool HALVES>
    __device__ __forceinline__ void widen(bool half, float (&v)[4]) const {
        if constexpr (SIZE == 4) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = __uint_as_float(w[k]);
        } else if (HALVES && half) {
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

template<int WHOLE, int PER_ACCESS, int SIZE, int Q>
__device__ __forceinline__ void load_quads_by(const unsigned char *row, const int (&col)[Q], int n, raw_quad<SIZE> (&raw)[Q]) {
#pragma unroll
    for (int i = 0; i < Q; ++i) raw[i].template load<PER_ACCESS>(row + static_cast<std::uint32_t>(col[i]) * SIZE, i < WHOLE ? 4 : n - col[i]);
}
// Quads of a row of n columns, starting at columns col[i]; columns from n on are zero.  Nothing waits for a load here, but for
// two-byte elements one by one, which are put together.  WHOLE: so many of the quads, the first ones, are known to lie in the row.
template<int WHOLE = 0, int SIZE, int Q>
__device__ __forceinline__ void load_quads(const unsigned char *row, const int (&col)[Q], int n, int per_access, raw_quad<SIZE> (&raw)[Q]) {
    if (per_access == 4) load_quads_by<WHOLE, 4>(row, col, n, raw);
    else if (per_access == 2) load_quads_by<WHOLE, 2>(row, col, n, raw);
    else load_quads_by<WHOLE, 1>(row, col, n, raw);
}

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

// A quad's elements of SIZE bytes, packed: those among the `count` left of the row.
template<int PER_ACCESS, int SIZE>
__device__ __forceinline__ void store_quad(unsigned char *p, int count, const std::uint32_t (&w)[SIZE]) {
    if constexpr (SIZE == 4 && PER_ACCESS == 4) {
        if (count > 0) *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else if constexpr (SIZE * PER_ACCESS == 8) {
#pragma unroll
        for (int k = 0; k < SIZE; k += 2)
            if (k * 4 / SIZE < count) *reinterpret_cast<uint2 *>(p + 4 * k) = make_uint2(w[k], w[k + 1]);
    } else if constexpr (SIZE * PER_ACCESS == 4) {
#pragma unroll
        for (int k = 0; k < SIZE; ++k)
            if (k * 4 / SIZE < count) *reinterpret_cast<std::uint32_t *>(p + 4 * k) = w[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < count) reinterpret_cast<unsigned short *>(p)[k] = static_cast<unsigned short>(w[k / 2] >> (16 * (k & 1)));
    }
}
template<int WHOLE, int SIZE, int Q>
__device__ __forceinline__ void store_packed(unsigned char *row, const int (&col)[Q], int n, int per_access, const std::uint32_t (&w)[Q][SIZE]) {
    if (per_access == 4) {
#pragma unroll
        for (int i = 0; i < Q; ++i) store_quad<4>(row + static_cast<std::uint32_t>(col[i]) * SIZE, i < WHOLE ? 4 : n - col[i], w[i]);
    } else if (per_access == 2) {
#pragma unroll
        for (int i = 0; i < Q; ++i) store_quad<2>(row + static_cast<std::uint32_t>(col[i]) * SIZE, i < WHOLE ? 4 : n - col[i], w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < Q; ++i) store_quad<1>(row + static_cast<std::uint32_t>(col[i]) * SIZE, i < WHOLE ? 4 : n - col[i], w[i]);
    }
}
// Values of quads into a row of n columns.  One rounding, to nearest, where the type has fewer bits than fp32.  HALVES as for widen,
// WHOLE as for load_quads.
template<bool HALVES, int WHOLE = 0, int Q>
__device__ __forceinline__ void store_quads(unsigned char *row, const int (&col)[Q], int n, int per_access, int dtype, const float (&v)[Q][4]) {
    if (dtype == CB200_DTYPE_F32) {
        std::uint32_t w[Q][4];
#pragma unroll
        for (int i = 0; i < Q; ++i) {
#pragma unroll
            for (int k = 0; k < 4; ++k) w[i][k] = __float_as_uint(v[i][k]);
        }
        store_packed<WHOLE>(row, col, n, per_access, w);
        return;
    }
    const bool half = HALVES && dtype == CB200_DTYPE_F16;
    std::uint32_t w[Q][2];
#pragma unroll
    for (int i = 0; i < Q; ++i) {
        w[i][0] = pack_pair(v[i][0], v[i][1], half);
        w[i][1] = pack_pair(v[i][2], v[i][3], half);
    }
    store_packed<WHOLE>(row, col, n, per_access, w);
}
#endif

} // namespace cb200
