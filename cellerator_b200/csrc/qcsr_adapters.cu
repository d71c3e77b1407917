// Low-rank adapters of many requests beside the shared projection of a quantized CSR batch:
//     out[r] = act(alpha s_a (deq(X)[r] A_a) B_a + beta out[r] + bias),  a = adapter[r].
// The same walk over the row's entries as the projection, with a narrow operand that changes from row to row, and the second
// product while the first is still in shared memory.
#include "adapter_parts.hh"
#include "kernels.cuh"

#include <algorithm>
#include <cstring>
#include <type_traits>

namespace cb200 {
namespace {

constexpr int kWarps = 8;
constexpr int kMostRows = 8;            // of a block
constexpr int kMostRank = 256;
constexpr int kSumsBytes = 32 * 1024;   // of parts' sums in shared memory, or one row's

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
    std::int64_t row_begin, row_end, cols, adapters, out_ld, n;
    float alpha, beta;
    int rank, policy, epilogue;
    int lanes;      // that serve an entry: a power of two
    int up_quads;   // B in columns of four
    int block_rows; // rows of a block
};

// V neighbouring elements of a row of A.
template<typename WT, int V>
struct slice {
    static constexpr int bytes = V * static_cast<int>(sizeof(WT));
    static constexpr int words = bytes >= 4 ? bytes / 4 : 1;
    std::uint32_t w[words];
    __device__ __forceinline__ void load(const unsigned char *p) {
        // volatile: a batch of loads is issued before the first of its products
        if constexpr (bytes == 16)
            asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
        else if constexpr (bytes == 8) asm volatile("ld.global.nc.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
        else if constexpr (bytes == 4) asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(w[0]) : "l"(p));
        else {
            unsigned short h;
            asm volatile("ld.global.nc.b16 %0, [%1];" : "=h"(h) : "l"(p));
            w[0] = h;
        }
    }
    __device__ __forceinline__ void keep_if(bool held) {
#pragma unroll
        for (int i = 0; i < words; ++i) w[i] = held ? w[i] : 0u;
    }
    // acc += v * w; pairs of columns with the two-wide fp32 FMA
    __device__ __forceinline__ void add_to(float (&acc)[V], float v) const {
        if constexpr (V == 1) {
            acc[0] = fmaf(v, __uint_as_float(sizeof(WT) == 2 ? w[0] << 16 : w[0]), acc[0]);
        } else {
            const float2 vv = make_float2(v, v);
            unsigned long long vp;
            memcpy(&vp, &vv, 8);
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                float2 f;
                if constexpr (sizeof(WT) == 2) bf16x2_to_f32(w[i / 2], f.x, f.y);
                else f = make_float2(__uint_as_float(w[i]), __uint_as_float(w[i + 1]));
                float2 a = make_float2(acc[i], acc[i + 1]);
                unsigned long long ap, fp;
                memcpy(&ap, &a, 8);
                memcpy(&fp, &f, 8);
                asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(ap) : "l"(vp), "l"(fp));
                memcpy(&a, &ap, 8);
                acc[i] = a.x;
                acc[i + 1] = a.y;
            }
        }
    }
};

// Columns of the second product that a thread works out at a time: four, where B's rows are whole groups of them on their boundaries.
template<typename WT>
__device__ __forceinline__ void load4(const WT *p, float (&w)[4]) {
    if constexpr (sizeof(WT) == 4) {
        const float4 v = __ldg(reinterpret_cast<const float4 *>(p));
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
        bf16x2_to_f32(v.x, w[0], w[1]);
        bf16x2_to_f32(v.y, w[2], w[3]);
    }
}

// A block takes p.block_rows rows, cut into parts by their lengths alone, and deals the parts to its warps, so that a long row
// does not hold up the others.  A warp decodes 128 entries at a time into shared memory, {gene, value}, the next ones' indices and
// codes being on their way meanwhile; then `lanes` lanes serve an entry, V columns of A each, 8 rows of A in flight.  A part's sum is
// that of 32 / lanes classes of its entries, a row's that of its parts in order, and the product with B follows from shared memory.
// Lanes past a part's end read its last entry again, and genes outside the matrix row 0 of A: both are staged as gene -1, whose row
// counts as zeros whatever it holds.  Segments without such genes, up to the last whole piece of 8 entries a class, take the branch that
// does not look, where every lane holds columns: of ranks that are no power of two times a slice some lanes hold none, and all segments
// take the branch that looks (4,099 x 33,538, bf16: rank 12 95 us where rank 16 takes 76; rank 24 94, rank 32 90).  Ranks that are no multiple
// of half a 16-byte slice go column by column, and rank 50 twice along the row (525 us).
//
// 4,099 x 33,538, 8 bits, rank 16 bf16: 75 us, bound by what the SMs get out of L2 in pieces of 32 bytes at random places (a row of A, a
// scale and a zero-point for each entry; L1 and texture 70 %, issue 42 %).  50,000 x 4,000, 4 bits, rank 32: 292 us, bound by L1's wavefronts
// (71 %, two for an entry) and instructions (66 % of the slots, six for an entry in its share of a warp).  Before loads lost their branches 104 and 437.  Measured
// against it: scales and zero-points in shared memory, with fewer blocks an SM, 112 and 430 us; a third stage of loads under way 84; rows
// of A kept in L1 79 and 298; scales and zero-points side by side, laid so in a launch before, 77 and 305; parts of 256 entries 86 and
// 369; four blocks an SM by launch bounds 93, and with four rows of A in flight instead of eight 85 and
// 320; two blocks and sixteen rows 105 and 382; every part's sum by a butterfly over all columns, and partial segments wholly in the
// branch that looks, 78 and 298.
template<int BITS, typename WT, int V>
__global__ void __launch_bounds__(kWarps * 32) qcsr_adapter_kernel(const adapter_params p) {
    __shared__ __align__(16) int2 staged[kWarps][kSegment];
    __shared__ std::int64_t row_start[kMostRows], code_start[kMostRows];
    __shared__ unsigned row_len[kMostRows], row_share[kMostRows];
    __shared__ int row_adapter[kMostRows], first_part[kMostRows + 1];
    extern __shared__ float sums[]; // [parts][rank]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const std::int64_t row0 = p.row_begin + static_cast<std::int64_t>(blockIdx.x) * p.block_rows;
    const int rows = static_cast<int>(min(static_cast<std::int64_t>(p.block_rows), p.row_end - row0));
    if (warp == 0) {
        int upto = 0;
        if (lane < rows) {
            const int a = __ldg(p.adapter + row0 + lane);
            const bool has = a >= 0 && a < p.adapters && p.cols > 0;
            const std::int64_t start = __ldg(p.row_ptr + row0 + lane);
            const unsigned len = has ? static_cast<unsigned>(__ldg(p.row_ptr + row0 + lane + 1) - start) : 0u, share = part_entries(len);
            row_adapter[lane] = has ? a : -1;
            row_start[lane] = start;
            row_len[lane] = len;
            row_share[lane] = share;
            code_start[lane] = p.packed_row_ptr != nullptr ? __ldg(p.packed_row_ptr + row0 + lane) : start;
            upto = static_cast<int>(parts_of(len, share));
        }
#pragma unroll
        for (int off = 1; off < kMostRows; off <<= 1) {
            const int below = __shfl_up_sync(0xffffffffu, upto, off);
            if (lane >= off) upto += below;
        }
        if (lane == 0) first_part[0] = 0;
        if (lane < rows) first_part[lane + 1] = upto;
    }
    __syncthreads();
    const int parts = first_part[rows];
    const unsigned genes = static_cast<unsigned>(p.cols);
    const bool row_policy = p.policy == CB200_DECODE_COLUMN_SCALE_ROW_OFFSET, by_gene = p.scales != nullptr && p.offsets != nullptr && !row_policy;
    const int lanes = p.lanes, groups = 32 / lanes, group = lane / lanes, in_row = lane & (lanes - 1);
    const unsigned row_bytes = static_cast<unsigned>(p.rank) * sizeof(WT);
    int2 *stage = staged[warp];
    for (int column0 = 0; column0 < p.rank; column0 += lanes * V) { // of A; one turn but for wide ranks of narrow slices
        const int col = column0 + in_row * V;
        const bool holds = col < p.rank;
        int part = warp, r = 0;
        unsigned at = 0, to = 0; // entries of row r: those of the segment start at `at`
        int gene[kRuns];
        unsigned code[kRuns];
        const auto fetch = [&]() {
            const std::int32_t *cols = p.col_idx + row_start[r] + at;
            const std::uint8_t *codes = p.packed + code_start[r] + (BITS == 8 ? at : at >> 1); // `at` is even
            const int last = static_cast<int>(to - at) - 1;
#pragma unroll
            for (int i = 0; i < kRuns; ++i) {
                const int e = min(i * 32 + lane, last);
                asm volatile("ld.global.nc.L1::no_allocate.b32 %0, [%1];" : "=r"(gene[i]) : "l"(cols + e));
                if constexpr (BITS == 8) code[i] = __ldg(codes + e);
                else code[i] = __ldg(codes + (e >> 1)) >> (4 * (e & 1)) & 15u;
            }
        };
        const auto open = [&]() {
            if (part >= parts) return;
            r = __popc(__ballot_sync(0xffffffffu, lane < rows && first_part[min(lane, kMostRows)] <= part)) - 1;
            at = static_cast<unsigned>(part - first_part[r]) * row_share[r];
            to = part_end(at, row_len[r], row_share[r]);
            fetch();
        };
        open();
        float acc[V];
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.0f;
        while (part < parts) {
            const int count = static_cast<int>(min(static_cast<unsigned>(kSegment), to - at)), part_now = part;
            const unsigned char *down = p.down + static_cast<std::int64_t>(row_adapter[r]) * p.cols * row_bytes + (holds ? col : 0) * sizeof(WT);
            float scale[kRuns], offset[kRuns];
            bool fine = holds;
            unsigned at_gene[kRuns];
#pragma unroll
            for (int i = 0; i < kRuns; ++i) {
                const bool inside = static_cast<unsigned>(gene[i]) < genes;
                fine = fine && inside;
                at_gene[i] = inside ? static_cast<unsigned>(gene[i]) : 0u;
                if (!inside || i * 32 + lane >= count) gene[i] = -1;
            }
            if (by_gene) {
#pragma unroll
                for (int i = 0; i < kRuns; ++i) {
                    scale[i] = __ldg(p.scales + at_gene[i]);
                    offset[i] = __ldg(p.offsets + at_gene[i]);
                }
            } else {
                const float row_offset = row_policy && p.offsets != nullptr ? __ldg(p.offsets + row0 + r) : 0.0f;
#pragma unroll
                for (int i = 0; i < kRuns; ++i) {
                    scale[i] = p.scales != nullptr ? __ldg(p.scales + at_gene[i]) : 1.0f;
                    offset[i] = !row_policy && p.offsets != nullptr ? __ldg(p.offsets + at_gene[i]) : row_offset;
                }
            }
            fine = __all_sync(0xffffffffu, fine);
#pragma unroll
            for (int i = 0; i < kRuns; ++i)
                stage[i * 32 + lane] = make_int2(gene[i], __float_as_int(fmaf(static_cast<float>(code[i]), scale[i], offset[i])));
            __syncwarp();
            at += kSegment;
            const bool ends = at >= to;
            if (ends) {
                part += kWarps;
                open();
            } else {
                fetch();
            }
            const int2 *mine = stage + group;
            int e = 0;
            if (fine) {
                const auto add = [&](auto unrolled, int first) {
                    constexpr int U = decltype(unrolled)::value;
                    slice<WT, V> w[U];
                    float v[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int2 entry = mine[first + u * groups];
                        v[u] = __int_as_float(entry.y);
                        w[u].load(down + static_cast<std::uint64_t>(static_cast<std::uint32_t>(entry.x)) * row_bytes);
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u) w[u].add_to(acc, v[u]);
                };
                if (groups == 32) { // one entry to a lane
                    if (count == kSegment) {
                        add(std::integral_constant<int, 4>{}, 0);
                        e = kSegment;
                    }
                } else {
                    for (; e + 8 * groups <= count; e += 8 * groups) add(std::integral_constant<int, 8>{}, e);
                }
            }
            for (; e < count; e += 4 * groups) {
                slice<WT, V> w[4];
                float v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int2 entry = mine[e + u * groups];
                    const bool held = entry.x >= 0 && holds;
                    v[u] = held ? __int_as_float(entry.y) : 0.0f;
                    w[u].load(down + static_cast<std::uint64_t>(static_cast<std::uint32_t>(max(entry.x, 0))) * row_bytes);
                    w[u].keep_if(held);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) w[u].add_to(acc, v[u]);
            }
            __syncwarp();
            if (!ends) continue;
            // the classes' sums: in each step a lane gives half of its columns away and keeps the sums of the other half
            int kept = V, from = 0;
#pragma unroll
            for (int step = 0; step < 5; ++step) {
                const int off = lanes << step;
                if (off >= 32) break;
                if ((V >> step) > 1) {
                    const int w = (V >> step) / 2;
                    const bool upper = (lane & off) != 0;
#pragma unroll
                    for (int i = 0; i < w; ++i) {
                        const float given = upper ? acc[i] : acc[i + w];
                        acc[i] = (upper ? acc[i + w] : acc[i]) + __shfl_xor_sync(0xffffffffu, given, off);
                    }
                    kept = w;
                    from += upper ? w : 0;
                } else {
                    acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], off);
                }
            }
            if (group < V && holds) {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (i < kept) sums[part_now * p.rank + col + from + i] = acc[i];
            }
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = 0.0f;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * p.rank; i += kWarps * 32) {
        const int r = i / p.rank, k = i - r * p.rank, last = first_part[r + 1];
        if (first_part[r] == last) continue;
        float *sum = sums + first_part[r] * p.rank + k, h = *sum;
        for (int part = first_part[r] + 1; part < last; ++part) h += sums[part * p.rank + k];
        *sum = h;
    }
    __syncthreads();
    const int n = static_cast<int>(p.n), per_row = p.up_quads ? n >> 2 : n;
    for (int i = threadIdx.x; i < rows * per_row; i += kWarps * 32) {
        const int r = i / per_row, a = row_adapter[r];
        const bool has = first_part[r] < first_part[r + 1];
        const float *hidden = sums + first_part[r] * p.rank;
        const float factor = has ? p.alpha * (p.scale != nullptr ? __ldg(p.scale + a) : 1.0f) : 0.0f;
        const int c = p.up_quads ? i % per_row * 4 : i % per_row;
        const WT *up = static_cast<const WT *>(p.up) + static_cast<std::int64_t>(has ? a : 0) * p.rank * n + c;
        float *out = p.out + (row0 + r) * p.out_ld + c;
        if (p.up_quads) {
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (has) {
#pragma unroll 8
                for (int k = 0; k < p.rank; ++k, up += n) {
                    float w[4];
                    load4(up, w);
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = fmaf(hidden[k], w[j], v[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[j] *= factor;
                if (p.beta != 0.0f) v[j] = fmaf(p.beta, out[j], v[j]);
                out[j] = finish_output(v[j], p.bias, c + j, p.epilogue);
            }
        } else {
            float v = 0.0f;
            if (has) {
#pragma unroll 8
                for (int k = 0; k < p.rank; ++k, up += n) v = fmaf(hidden[k], load1(up), v);
            }
            v *= factor;
            if (p.beta != 0.0f) v = fmaf(p.beta, *out, v);
            *out = finish_output(v, p.bias, c, p.epilogue);
        }
    }
}

template<int BITS, typename WT, int V>
cb200_status launch(adapter_params p, std::int64_t rows, cudaStream_t stream) {
    p.lanes = 1;
    while (p.lanes < 32 && p.lanes * V < p.rank) p.lanes *= 2;
    const std::size_t smem = static_cast<std::size_t>(p.block_rows) * kMostParts * p.rank * sizeof(float);
    qcsr_adapter_kernel<BITS, WT, V><<<static_cast<unsigned>((rows + p.block_rows - 1) / p.block_rows), kWarps * 32, smem, stream>>>(p);
    count_launch();
    CB200_CUDA_OK(cudaGetLastError());
    return CB200_STATUS_SUCCESS;
}

// Elements of a lane's slice of A: 16 bytes where every row starts on such a boundary, else 8, else one element.
template<int BITS, typename WT>
cb200_status dispatch(const adapter_params &p, std::int64_t rows, cudaStream_t stream) {
    constexpr int widest = 16 / static_cast<int>(sizeof(WT));
    const std::uintptr_t base = reinterpret_cast<std::uintptr_t>(p.down);
    if (p.rank % widest == 0 && base % 16u == 0u) return launch<BITS, WT, widest>(p, rows, stream);
    if (p.rank % (widest / 2) == 0 && base % 8u == 0u) return launch<BITS, WT, widest / 2>(p, rows, stream);
    return launch<BITS, WT, 1>(p, rows, stream);
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
    if (d->n < 0 || d->adapters < 0 || x->rows < 0 || x->cols < 0 || x->cols > 0x7fffffffll || x->nnz < 0 || d->n > (1ll << 27) || d->adapters > 0x7fffffffll)
        return fail(CB200_STATUS_INVALID_SHAPE, "a size is negative or too large (n up to 2^27, the others below 2^31)");
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
        const auto odd = [](const void *a, std::uintptr_t bytes) { return reinterpret_cast<std::uintptr_t>(a) % bytes != 0u; };
        if (odd(d->down, element) || odd(d->up, element) ||
            odd(d->out, 4) || odd(d->adapter, 4) || odd(d->scale, 4) || odd(d->bias, 4) || odd(x->row_ptr, 8) || odd(x->packed_row_ptr, 8) ||
            odd(x->col_idx, 4) || odd(x->scales, 4) || odd(x->offsets, 4))
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
    p.row_end = end;
    // Rows of a block: about 8,192 entries, so that blocks are long enough to hide their start and end, but blocks enough for every SM,
    // and no more parts than the shared memory holds.
    const double mean = static_cast<double>(x->nnz) / static_cast<double>(std::max<std::int64_t>(x->rows, 1));
    p.block_rows = 1;
    while (2 * p.block_rows <= kMostRows && 2 * p.block_rows * mean <= 8192.0 && end - begin >= 4ll * 148 * p.block_rows &&
           2 * p.block_rows * kMostParts * p.rank * static_cast<int>(sizeof(float)) <= kSumsBytes)
        p.block_rows *= 2;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool bf16 = d->weight_dtype == CB200_DTYPE_BF16;
    const std::uintptr_t quad = bf16 ? 8u : 16u;
    p.up_quads = d->n % 4 == 0 && reinterpret_cast<std::uintptr_t>(d->up) % quad == 0u ? 1 : 0;
    if (x->bits == 8) return bf16 ? dispatch<8, __nv_bfloat16>(p, end - begin, s) : dispatch<8, float>(p, end - begin, s);
    return bf16 ? dispatch<4, __nv_bfloat16>(p, end - begin, s) : dispatch<4, float>(p, end - begin, s);
}
