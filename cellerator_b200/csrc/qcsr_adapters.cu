// Low-rank adapters of many requests beside the shared projection of a quantized CSR batch:
//     out[r] = act(alpha s_a (deq(X)[r] A_a) B_a + beta out[r] + bias),  a = adapter[r].
// The same walk over the row's entries as the projection, with a narrow operand that changes from row to row, and the second
// product while the first is still in shared memory.
#include "kernels.cuh"

#include <algorithm>
#include <type_traits>

namespace cb200 {
namespace {

constexpr int kSegment = 128;   // entries that a warp decodes at a time
constexpr int kMostParts = 32;  // of a row
constexpr int kMostWarps = 8;
constexpr int kMostRank = 256;

struct adapter_params {
    const std::int64_t *row_ptr, *packed_row_ptr;
    const std::int32_t *col_idx;
    const std::uint8_t *packed;
    const float *scales, *offsets;
    const std::int32_t *adapter;
    const unsigned char *down;
    const void *up;
    const float *scale;
    float *out;
    const float *bias;
    std::int64_t row_begin, cols, adapters, out_ld, n;
    float alpha, beta;
    int rank, policy, epilogue;
    int lanes; // that serve an entry: a power of two
};

// Entries of a part of a row of `len` entries, a multiple of a warp's segment: by the length alone.
__device__ __forceinline__ std::int64_t part_entries(std::int64_t len) {
    const std::int64_t even = (len + kMostParts - 1) / kMostParts;
    return max(static_cast<std::int64_t>(kSegment), (even + kSegment - 1) / kSegment * kSegment);
}

// V neighbouring elements of a row of A.
template<typename WT, int V>
struct slice {
    static constexpr int bytes = V * static_cast<int>(sizeof(WT));
    std::uint32_t w[bytes >= 4 ? bytes / 4 : 1];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < (bytes >= 4 ? bytes / 4 : 1); ++i) w[i] = 0u;
    }
    __device__ __forceinline__ void load(const unsigned char *p) {
        if constexpr (bytes == 16) {
            const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p));
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else if constexpr (bytes == 8) {
            const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
            w[0] = v.x; w[1] = v.y;
        } else if constexpr (bytes == 4) {
            w[0] = __ldg(reinterpret_cast<const unsigned *>(p));
        } else {
            w[0] = __ldg(reinterpret_cast<const unsigned short *>(p));
        }
    }
    __device__ __forceinline__ void add_to(float (&acc)[V], float v) const {
        if constexpr (V == 1) {
            acc[0] = fmaf(v, __uint_as_float(sizeof(WT) == 2 ? w[0] << 16 : w[0]), acc[0]);
        } else {
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                float a, b;
                if constexpr (sizeof(WT) == 2) bf16x2_to_f32(w[i / 2], a, b);
                else { a = __uint_as_float(w[i]); b = __uint_as_float(w[i + 1]); }
                acc[i] = fmaf(v, a, acc[i]);
                acc[i + 1] = fmaf(v, b, acc[i + 1]);
            }
        }
    }
};

// A block per row.  Its warps take the row's parts in turn; a warp decodes 128 entries at a time into shared memory, {gene,
// value}, and then `lanes` lanes serve an entry, V columns of A each.
template<int BITS, typename WT, int V>
__global__ void __launch_bounds__(kMostWarps * 32) qcsr_adapter_kernel(const adapter_params p) {
    __shared__ __align__(16) int2 staged[kMostWarps][kSegment];
    __shared__ float hidden[kMostRank];
    extern __shared__ float sums[]; // [parts][rank]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const std::int64_t row = p.row_begin + blockIdx.x;
    const int a = __ldg(p.adapter + row);
    const bool has = a >= 0 && a < p.adapters;
    if (has) {
        const std::int64_t start = __ldg(p.row_ptr + row), len = __ldg(p.row_ptr + row + 1) - start;
        const std::int64_t share = part_entries(len);
        const int parts = static_cast<int>((len + share - 1) / share);
        const std::int32_t *cols = p.col_idx + start;
        const std::uint8_t *codes = p.packed + (p.packed_row_ptr != nullptr ? __ldg(p.packed_row_ptr + row) : start);
        const bool row_policy = p.policy == CB200_DECODE_COLUMN_SCALE_ROW_OFFSET;
        const float row_offset = row_policy && p.offsets != nullptr ? __ldg(p.offsets + row) : 0.0f;
        const int lanes = p.lanes, groups = 32 / lanes, group = lane / lanes, in_row = lane & (lanes - 1);
        const unsigned row_bytes = static_cast<unsigned>(p.rank) * sizeof(WT);
        const unsigned char *down = p.down + static_cast<std::int64_t>(a) * p.cols * row_bytes;
        for (int part = warp; part < parts; part += warps) {
            for (int first = 0; first < p.rank; first += lanes * V) { // columns of A; one turn but for wide ranks of narrow slices
                const int col = first + in_row * V;
                const bool holds = col < p.rank;
                float acc[V];
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] = 0.0f;
                const std::int64_t to = min(len, (part + 1) * share);
                for (std::int64_t at = part * share; at < to; at += kSegment) {
#pragma unroll
                    for (int i = 0; i < kSegment / 32; ++i) {
                        const std::int64_t e = at + i * 32 + lane;
                        int2 entry = make_int2(-1, 0);
                        if (e < to) {
                            const std::int32_t gene = __ldg(cols + e);
                            unsigned code;
                            if constexpr (BITS == 8) code = __ldg(codes + e);
                            else code = (__ldg(codes + (e >> 1)) >> (4 * (e & 1))) & 15u;
                            if (gene >= 0 && gene < p.cols) {
                                const float scale = p.scales != nullptr ? __ldg(p.scales + gene) : 1.0f;
                                const float offset = row_policy ? row_offset : p.offsets != nullptr ? __ldg(p.offsets + gene) : 0.0f;
                                entry = make_int2(gene, __float_as_int(fmaf(static_cast<float>(code), scale, offset)));
                            }
                        }
                        staged[warp][i * 32 + lane] = entry;
                    }
                    __syncwarp();
                    const int count = static_cast<int>(min(static_cast<std::int64_t>(kSegment), to - at));
                    for (int e = group; e < count + group; e += 4 * groups) {
                        slice<WT, V> w[4];
                        float v[4];
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const int2 entry = e + u * groups < kSegment ? staged[warp][e + u * groups] : make_int2(-1, 0);
                            v[u] = __int_as_float(entry.y);
                            w[u].clear();
                            if (entry.x >= 0 && holds) w[u].load(down + static_cast<std::uint64_t>(entry.x) * row_bytes + col * sizeof(WT));
                        }
#pragma unroll
                        for (int u = 0; u < 4; ++u) w[u].add_to(acc, v[u]);
                    }
                    __syncwarp();
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    for (int off = lanes; off < 32; off <<= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], off);
                    if (group == 0 && col + i < p.rank) sums[part * p.rank + col + i] = acc[i];
                }
            }
        }
        __syncthreads();
        for (int k = threadIdx.x; k < p.rank; k += blockDim.x) {
            float h = 0.0f;
            for (int part = 0; part < parts; ++part) h += sums[part * p.rank + k];
            hidden[k] = h;
        }
        __syncthreads();
    }
    const float factor = has ? p.alpha * (p.scale != nullptr ? __ldg(p.scale + a) : 1.0f) : 0.0f;
    const WT *up = static_cast<const WT *>(p.up) + static_cast<std::int64_t>(has ? a : 0) * p.rank * p.n;
    for (std::int64_t c = threadIdx.x; c < p.n; c += blockDim.x) {
        float v = 0.0f;
        if (has) {
#pragma unroll 8
            for (int k = 0; k < p.rank; ++k) v = fmaf(hidden[k], load1(up + k * p.n + c), v);
            v *= factor;
        }
        float *out = p.out + row * p.out_ld + c;
        if (p.beta != 0.0f) v = fmaf(p.beta, *out, v);
        *out = p.epilogue == CB200_EPILOGUE_NONE ? v : apply_epilogue(v, epilogue_has_bias(p.epilogue) ? __ldg(p.bias + c) : 0.0f, p.epilogue);
    }
}

template<int BITS, typename WT, int V>
cb200_status launch(adapter_params p, std::int64_t rows, int warps, cudaStream_t stream) {
    p.lanes = 1;
    while (p.lanes < 32 && p.lanes * V < p.rank) p.lanes *= 2;
    const std::size_t smem = static_cast<std::size_t>(kMostParts) * p.rank * sizeof(float);
    qcsr_adapter_kernel<BITS, WT, V><<<static_cast<unsigned>(rows), warps * 32, smem, stream>>>(p);
    count_launch();
    CB200_CUDA_OK(cudaGetLastError());
    return CB200_STATUS_SUCCESS;
}

// Elements of a lane's slice of A: 16 bytes where every row starts on such a boundary, else 8, else one element.
template<int BITS, typename WT>
cb200_status dispatch(const adapter_params &p, std::int64_t rows, int warps, cudaStream_t stream) {
    constexpr int widest = 16 / static_cast<int>(sizeof(WT));
    const std::uintptr_t base = reinterpret_cast<std::uintptr_t>(p.down);
    if (p.rank % widest == 0 && base % 16u == 0u) return launch<BITS, WT, widest>(p, rows, warps, stream);
    if (p.rank % (widest / 2) == 0 && base % 8u == 0u) return launch<BITS, WT, widest / 2>(p, rows, warps, stream);
    return launch<BITS, WT, 1>(p, rows, warps, stream);
}

} // namespace
} // namespace cb200

extern "C" cb200_status cb200_qcsr_adapters(const cb200_adapters *d, void *stream) {
    using namespace cb200;
    clear_error();
    if (d == nullptr || d->version != CB200_ABI_VERSION || d->size < sizeof(cb200_adapters))
        return fail(CB200_STATUS_INVALID_ARGUMENT, "bad cb200_adapters header");
    const cb200_qcsr *x = d->csr;
    if (x == nullptr || x->version != CB200_ABI_VERSION || x->size < sizeof(cb200_qcsr))
        return fail(CB200_STATUS_INVALID_ARGUMENT, "bad cb200_qcsr header");
    if (x->bits != 8 && x->bits != 4) return fail(CB200_STATUS_UNSUPPORTED, "adapters take 8-bit and 4-bit codes, got %d", x->bits);
    if (x->policy != CB200_DECODE_PER_GENE_AFFINE && x->policy != CB200_DECODE_COLUMN_SCALE_ROW_OFFSET)
        return fail(CB200_STATUS_UNSUPPORTED, "unknown decode policy %d", x->policy);
    if (d->weight_dtype != CB200_DTYPE_F32 && d->weight_dtype != CB200_DTYPE_BF16)
        return fail(CB200_STATUS_UNSUPPORTED, "adapters are fp32 or bf16, got type %d", d->weight_dtype);
    if (d->epilogue < CB200_EPILOGUE_NONE || d->epilogue > CB200_EPILOGUE_BIAS_GELU_TANH)
        return fail(CB200_STATUS_UNSUPPORTED, "unknown epilogue kind %d", d->epilogue);
    const bool bias_kind = d->epilogue == CB200_EPILOGUE_BIAS || d->epilogue >= CB200_EPILOGUE_BIAS_RELU;
    if (d->rank < 1 || d->rank > kMostRank) return fail(CB200_STATUS_UNSUPPORTED, "rank %lld outside 1 .. %d", (long long)d->rank, kMostRank);
    if (d->n < 0 || d->adapters < 0 || x->rows < 0 || x->cols < 0 || x->cols > 0x7fffffffll || x->nnz < 0 || d->n > 0x7fffffffll || d->adapters > 0x7fffffffll)
        return fail(CB200_STATUS_INVALID_SHAPE, "a size is negative or above 2^31");
    if (d->out_ld < d->n) return fail(CB200_STATUS_INVALID_SHAPE, "leading dimension smaller than n");
    const std::int64_t begin = d->row_begin, end = d->row_end == CB200_ALL_ROWS ? x->rows : d->row_end;
    if (begin < 0 || end > x->rows || begin > end)
        return fail(CB200_STATUS_INVALID_SHAPE, "row range [%lld,%lld) outside 0..%lld", (long long)begin, (long long)end, (long long)x->rows);
    if (end - begin > 0x7fffffffll) return fail(CB200_STATUS_INVALID_SHAPE, "row range too large for one launch");
    const bool nothing = begin == end || d->n == 0;
    if (!nothing) {
        if (d->adapter == nullptr || d->out == nullptr || x->row_ptr == nullptr || (x->nnz != 0 && (x->col_idx == nullptr || x->packed_values == nullptr)) ||
            (d->adapters > 0 && (d->up == nullptr || (d->down == nullptr && x->cols > 0))) || (bias_kind && d->bias == nullptr))
            return fail(CB200_STATUS_INVALID_ARGUMENT, "adapters: an array is null");
        if (x->bits == 4 && x->packed_row_ptr == nullptr) return fail(CB200_STATUS_INVALID_ARGUMENT, "4-bit codes need packed_row_ptr");
        const std::uintptr_t element = d->weight_dtype == CB200_DTYPE_BF16 ? 2u : 4u;
        if (reinterpret_cast<std::uintptr_t>(d->down) % element != 0u || reinterpret_cast<std::uintptr_t>(d->up) % element != 0u ||
            reinterpret_cast<std::uintptr_t>(d->out) % 4u != 0u || reinterpret_cast<std::uintptr_t>(d->adapter) % 4u != 0u)
            return fail(CB200_STATUS_INVALID_ARGUMENT, "adapters: an array is not aligned to its elements");
    }
    device_scope scope(d->device);
    CB200_CUDA_OK(scope.status);
    if (nothing) return CB200_STATUS_SUCCESS;
    adapter_params p{};
    p.row_ptr = x->row_ptr; p.packed_row_ptr = x->packed_row_ptr; p.col_idx = x->col_idx; p.packed = x->packed_values;
    p.scales = x->scales; p.offsets = x->offsets; p.adapter = d->adapter;
    p.down = static_cast<const unsigned char *>(d->down); p.up = d->up; p.scale = d->scale; p.out = d->out;
    p.bias = bias_kind ? d->bias : nullptr;
    p.row_begin = begin; p.cols = x->cols; p.adapters = d->adapters; p.out_ld = d->out_ld; p.n = d->n;
    p.alpha = d->alpha; p.beta = d->beta;
    p.rank = static_cast<int>(d->rank); p.policy = x->policy; p.epilogue = d->epilogue;
    const std::int64_t mean = x->nnz / std::max<std::int64_t>(x->rows, 1);
    const int warps = static_cast<int>(std::min<std::int64_t>(kMostWarps, std::max<std::int64_t>(2, (mean + kSegment - 1) / kSegment)));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool bf16 = d->weight_dtype == CB200_DTYPE_BF16;
    if (x->bits == 8) return bf16 ? dispatch<8, __nv_bfloat16>(p, end - begin, warps, s) : dispatch<8, float>(p, end - begin, warps, s);
    return bf16 ? dispatch<4, __nv_bfloat16>(p, end - begin, warps, s) : dispatch<4, float>(p, end - begin, warps, s);
}
