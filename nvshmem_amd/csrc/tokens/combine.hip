// What a token's copies come back as: their sum weighted with the router's gates, and its gradients.
//
//   out@p[t] = sum_k gate@p[t, k] * recv@d[r]      d = dest_pe@p[t, k], r = dest_row@p[t, k], k ascending in fp32, rounded once
//   drecv@d[r] = gate@p[t, k] * dout@p[t]          dgate@p[t, k] = <dout@p[t], recv@d[r]> in fp32
//
// The tables are those of the dispatch; an entry outside [0, npes) x [0, recv_cap_rows) is a copy that was dropped: it adds
// nothing, and its dgate is 0.
#include "token_common.hpp"

namespace nvshmem_amd {
namespace tokens {
namespace {

template <int SIZE>
struct same_size {
    typedef uint16_t type;
};
template <>
struct same_size<4> {
    typedef uint32_t type;
};

// Most copies of a token whose loads are in flight together.
constexpr int kCopies = 8;

// One wavefront per piece of 64 chunks of a token's row, or rows of fewer chunks that share a wavefront, 2^lanes_log lanes each.
// Reads every copy once and writes a row: bound by memory.  All K loads of a lane leave before the first is used, so neither their
// addresses nor whether a copy was dropped may be waited for in between: a dropped copy's load goes to the row to be written.
// Where a wavefront has one token, its entries are scalar loads and its rows scalar addresses.
// us for 8 x 4096 rows of 7168 bf16, top-8 (4.23 GB): 706 are 6.0 TB/s; with each entry loaded in front of its row 828, loads that stay in
// the caches 743, two chunks of each copy a lane 852 (159 registers).  8 x 64 rows, which the Infinity Cache holds: 13.4.
template <typename T, int K, int MODE>
__global__ __launch_bounds__(64) void combine_sum_kernel(T *__restrict__ out, const T *__restrict__ recv, const float *__restrict__ gate,
                                                         const int32_t *__restrict__ dest_pe, const int64_t *__restrict__ dest_row,
                                                         uint64_t stride, uint64_t cap, unsigned tokens, unsigned topk, unsigned dim,
                                                         unsigned npes, unsigned lanes_log) {
    const unsigned lane = threadIdx.x, pe = blockIdx.z, log = MODE == kWhole ? 6 : lanes_log, per_wave = kLanes >> log;
    const unsigned c = blockIdx.x * kLanes + (lane & ((1u << log) - 1));
    if (c * Chunk<T>::N >= dim) return;
    const unsigned first = chunk_first<T>(c, dim);
    const int32_t *my_pe = copy_of(dest_pe, pe, stride);
    const int64_t *my_row = copy_of(dest_row, pe, stride);
    const float *my_gate = gate ? copy_of(gate, pe, stride) : nullptr;
    T *my_out = copy_of(out, pe, stride);
    for (uint64_t t = (uint64_t)blockIdx.y * per_wave + (MODE == kWhole ? 0 : lane >> log); t < tokens;
         t += (uint64_t)gridDim.y * per_wave) {
        T *dst = my_out + t * dim;
        typename Chunk<T>::facc sum = {};
        for (unsigned k0 = 0; k0 < topk; k0 += K) {
            // the entries first, all of them; behind the last copy (K is topk where that is less than kCopies) it stands in
            unsigned d[K];
            uint64_t r[K];
            float w[K];
            uint32_t bits[K];
#pragma unroll
            for (unsigned k = 0; k < K; ++k) {
                const uint64_t e = t * topk + (K < kCopies || k0 + k < topk ? k0 + k : topk - 1);
                d[k] = (unsigned)my_pe[e];
                r[k] = (uint64_t)my_row[e];
                w[k] = 1.0f;
            }
            if (my_gate) {
#pragma unroll
                for (unsigned k = 0; k < K; ++k) w[k] = my_gate[t * topk + (K < kCopies || k0 + k < topk ? k0 + k : topk - 1)];
            }
            const T *src[K];
#pragma unroll
            for (unsigned k = 0; k < K; ++k) {
                const bool ok = (K < kCopies | k0 + k < topk) & (d[k] < npes) & (r[k] < cap);
                const T *from = copy_of(recv, d[k], stride) + r[k] * dim;
                src[k] = ok ? from : dst;
                bits[k] = ok ? ~0u : 0u;
                w[k] = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, w[k]) & bits[k]);  // (it may be infinite or a NaN)
            }
            typename Chunk<T>::vec x[K];
#pragma unroll
            for (unsigned k = 0; k < K; ++k) x[k] = MODE == kTiny ? chunk_load_part(src[k], dim) : chunk_load_stream(src[k] + first);
#pragma unroll
            for (unsigned k = 0; k < K; ++k) {
                // (a selection would become a branch around the load, with a wait behind it)
                const nvshmemi_v4u v = __builtin_bit_cast(nvshmemi_v4u, x[k]) & bits[k];
                sum += chunk_to_float<T>(__builtin_bit_cast(typename Chunk<T>::vec, v)) * w[k];
            }
        }
        const typename Chunk<T>::vec y = chunk_from_float<T>(sum);
        if (MODE == kTiny) chunk_store_part(dst, y, dim);
        else chunk_store_stream(dst + first, y);
    }
}

// The sum of one copy.  kTokens tokens for each row's lanes, as wavefronts of one piece of two rows start too slowly to keep memory busy.
// us for 8 x t rows of d bf16, one token / four: 6000 of 512 23.1 / 17.4, 6000 of 2048 85 / 63 (6.2 TB/s), 4096 of 7168 148 / 147, 600 of
// 512 (4800 wavefronts of one) 5.0 / 4.5, 64 of 512 (512) 2.5 / 3.0; 8000 of 64 (8000) 7.2 / 6.4, 2100 of 64 (2104) 4.1 / 4.3.
constexpr uint64_t kManyPieces = 4096;
constexpr unsigned kTokens = 4;

template <typename T, int MODE>
__global__ __launch_bounds__(64) void combine_one_kernel(T *__restrict__ out, const T *__restrict__ recv, const float *__restrict__ gate,
                                                         const int32_t *__restrict__ dest_pe, const int64_t *__restrict__ dest_row,
                                                         uint64_t stride, uint64_t cap, unsigned tokens, unsigned dim, unsigned npes,
                                                         unsigned lanes_log) {
    typedef typename Chunk<T>::facc facc;
    const unsigned lane = threadIdx.x, pe = blockIdx.z, log = MODE == kWhole ? 6 : lanes_log, per_wave = kLanes >> log;
    const unsigned c = blockIdx.x * kLanes + (lane & ((1u << log) - 1));
    if (c * Chunk<T>::N >= dim) return;
    const unsigned first = chunk_first<T>(c, dim);
    const int32_t *my_pe = copy_of(dest_pe, pe, stride);
    const int64_t *my_row = copy_of(dest_row, pe, stride);
    const float *my_gate = gate ? copy_of(gate, pe, stride) : nullptr;
    T *my_out = copy_of(out, pe, stride);
    for (uint64_t t0 = (uint64_t)blockIdx.y * per_wave * kTokens + (MODE == kWhole ? 0 : lane >> log); t0 < tokens;
         t0 += (uint64_t)gridDim.y * per_wave * kTokens) {
        unsigned d[kTokens];
        uint64_t r[kTokens];
        float w[kTokens];
#pragma unroll
        for (unsigned i = 0; i < kTokens; ++i) {
            const uint64_t t = t0 + i * per_wave < tokens ? t0 + i * per_wave : t0;
            d[i] = (unsigned)my_pe[t], r[i] = (uint64_t)my_row[t], w[i] = 1.0f;
        }
        if (my_gate) {
#pragma unroll
            for (unsigned i = 0; i < kTokens; ++i) w[i] = my_gate[t0 + i * per_wave < tokens ? t0 + i * per_wave : t0];
        }
        typename Chunk<T>::vec x[kTokens] = {};
#pragma unroll
        for (unsigned i = 0; i < kTokens; ++i)
            if (d[i] < npes && r[i] < cap) x[i] = chunk_load_stream(copy_of(recv, d[i], stride) + r[i] * dim + first);
            else w[i] = 0.0f;
#pragma unroll
        for (unsigned i = 0; i < kTokens; ++i) {
            facc sum = {};
            sum += chunk_to_float<T>(x[i]) * w[i];
            if (t0 + i * per_wave < tokens) chunk_store_stream(my_out + (t0 + i * per_wave) * dim + first, chunk_from_float<T>(sum));
        }
    }
}

// A block of up to 8 wavefronts per token.  A lane loads a chunk of all K copies before it uses the first or stores any (drecv may be
// recv), and keeps the products for the K gates in registers; they are added up lane by lane and then wavefront by wavefront.
// Bound by memory: 8 x 2048 rows of 7168 bf16, top-8 (3.99 GB) take 651 us, 6.1 TB/s; one copy after the other 674 to 696.  4 x 501 rows of
// 1029 halves, top-2: 7.0, with the elements of a last partial chunk one by one 12.6.
constexpr unsigned kGradWaves = 8;

template <typename T, int K, bool TINY>
__global__ __launch_bounds__(kGradWaves *kLanes) void combine_grad_kernel(T *drecv, float *__restrict__ dgate, const T *__restrict__ dout,
                                                                          const T *recv, const float *__restrict__ gate,
                                                                          const int32_t *__restrict__ dest_pe,
                                                                          const int64_t *__restrict__ dest_row, uint64_t stride,
                                                                          uint64_t cap, unsigned tokens, unsigned topk, unsigned dim,
                                                                          unsigned npes) {
    constexpr unsigned N = Chunk<T>::N;
    typedef typename Chunk<T>::vec vec;
    typedef typename Chunk<T>::facc facc;
    __shared__ float partial[kGradWaves][K];
    const unsigned pe = blockIdx.z, wave = wave_of_block(), waves = blockDim.x / kLanes, lane = threadIdx.x % kLanes;
    const int32_t *my_pe = copy_of(dest_pe, pe, stride);
    const int64_t *my_row = copy_of(dest_row, pe, stride);
    const float *my_gate = copy_of(gate, pe, stride);
    const T *my_dout = copy_of(dout, pe, stride);
    float *my_dgate = copy_of(dgate, pe, stride);
    for (uint64_t t = blockIdx.x; t < tokens; t += gridDim.x) {
        const T *from = my_dout + t * dim;
        for (unsigned k0 = 0; k0 < topk; k0 += K) {
            // the entries; behind the last copy (K is topk where that is less than kCopies) it stands in
            unsigned d[K];
            uint64_t r[K];
            float w[K];
#pragma unroll
            for (unsigned k = 0; k < K; ++k) {
                const uint64_t e = t * topk + (K < kCopies || k0 + k < topk ? k0 + k : topk - 1);
                d[k] = (unsigned)my_pe[e];
                r[k] = (uint64_t)my_row[e];
                w[k] = my_gate[e];
            }
            const T *src[K];
            T *dst[K];
            unsigned ok = 0;
#pragma unroll
            for (unsigned k = 0; k < K; ++k) {
                const bool there = (K < kCopies | k0 + k < topk) & (d[k] < npes) & (r[k] < cap);
                const T *x = copy_of(recv, d[k], stride) + r[k] * dim;
                src[k] = there ? x : from;
                dst[k] = copy_of(drecv, d[k], stride) + r[k] * dim;
                ok |= there ? 1u << k : 0u;
            }
            float dot[K] = {};
            for (unsigned c = wave * kLanes + lane; c * N < dim; c += waves * kLanes) {
                const unsigned first = chunk_first<T>(c, dim), shared = c * N - first;
                vec x[K];
#pragma unroll
                for (unsigned k = 0; k < K; ++k) x[k] = TINY ? chunk_load_part(src[k], dim) : chunk_load_stream(src[k] + first);
                const vec raw = TINY ? chunk_load_part(from, dim) : chunk_load(from + first);
                // elements that the chunk in front has too are its: zeros here, of both (in place, a copy's values may be gone by now, and an
                // infinity of dout's times a zero is a NaN)
                vec mask;
#pragma unroll
                for (unsigned i = 0; i < N; ++i) {
                    typedef typename same_size<sizeof(T)>::type bits;
                    mask[i] = __builtin_bit_cast(T, (bits)(i < shared ? 0 : ~(bits)0));
                }
                const facc g = chunk_to_float<T>(__builtin_bit_cast(vec, __builtin_bit_cast(nvshmemi_v4u, raw) & __builtin_bit_cast(nvshmemi_v4u, mask)));
#pragma unroll
                for (unsigned k = 0; k < K; ++k) {
                    const facc v = chunk_to_float<T>(__builtin_bit_cast(vec, __builtin_bit_cast(nvshmemi_v4u, x[k]) & __builtin_bit_cast(nvshmemi_v4u, mask)));
#pragma unroll
                    for (unsigned i = 0; i < N; ++i) dot[k] = __builtin_fmaf(v[i], g[i], dot[k]);
                }
#pragma unroll
                for (unsigned k = 0; k < K; ++k) {
                    if (!(ok >> k & 1)) continue;
                    const vec y = chunk_from_float<T>(g * w[k]);
                    // (the elements shared with the chunk in front are stored by its lane, which may still have to read them)
                    if (TINY) chunk_store_part(dst[k], y, dim);
                    else if (shared == 0) chunk_store_stream(dst[k] + first, y);
                    else chunk_store_behind(dst[k] + first, y, shared);
                }
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                dot[k] = group_sum<64>(dot[k]);
                if (lane == 0) partial[wave][k] = dot[k];
            }
            __syncthreads();
            if (threadIdx.x < K && k0 + threadIdx.x < topk) {
                float sum = 0.0f;
                for (unsigned i = 0; i < waves; ++i) sum += partial[i][threadIdx.x];
                my_dgate[t * topk + k0 + threadIdx.x] = ok >> threadIdx.x & 1 ? sum : 0.0f;
            }
            __syncthreads();
        }
    }
}

int check_sizes(Runtime &rt, const char *what, size_t tokens, int topk, size_t dim) {
    NVSHMEM_AMD_REFUSE(topk < 1 || topk > 1024, "%s: %d copies of a token, outside [1, 1024]", what, topk);
    NVSHMEM_AMD_REFUSE(tokens > ((size_t)1 << 31) / (size_t)rt.npes, "%s: %zu tokens on %d PEs, at most 2^31 in all", what, tokens, rt.npes);
    NVSHMEM_AMD_REFUSE(dim < 1 || dim > (1u << 24), "%s: rows of %zu elements, outside [1, 2^24]", what, dim);
    return 0;
}

template <typename API>
int combine_sum_on_stream(API *out, const API *recv, size_t recv_cap_rows, const float *gate, const int32_t *dest_pe,
                          const int64_t *dest_row, size_t tokens, int topk, size_t dim, hipStream_t stream) {
    typedef typename element<API>::type T;
    Runtime &rt = Runtime::get();
    std::lock_guard<std::recursive_mutex> lock(rt.mu);
    if (!ready(rt, "moe_combine_sum")) return NVSHMEMX_ERROR_INVALID_VALUE;
    if (int rc = check_sizes(rt, "moe_combine_sum", tokens, topk, dim)) return rc;
    NVSHMEM_AMD_REFUSE(recv_cap_rows > rt.heap_size / (dim * sizeof(T)), "moe_combine_sum recv: %zu rows leave the PE's heap slice", recv_cap_rows);
    const uint64_t copies = (uint64_t)tokens * topk;
    Operands ops(rt, "moe_combine_sum");
    const T *src = (const T *)ops.in("recv", recv, (uint64_t)recv_cap_rows * dim);
    const int32_t *to = ops.in("dest_pe", dest_pe, copies);
    const int64_t *at = ops.in("dest_row", dest_row, copies);
    const float *w = gate ? ops.in("gate", gate, copies) : nullptr;
    T *dst = (T *)ops.out("out", out, (uint64_t)tokens * dim);
    if (!ops.ok()) return NVSHMEMX_ERROR_INVALID_VALUE;
    if (tokens == 0) return 0;
    const size_t chunks = (dim + Chunk<T>::N - 1) / Chunk<T>::N;
    const unsigned log = row_lanes_log2(chunks), groups = div_up(tokens, kLanes >> log);
    const unsigned rows = groups < 65535 ? groups : 65535;
#define NVSHMEM_AMD_LAUNCH_SUM(K, MODE)                                                                                             \
    launch_kernel((combine_sum_kernel<T, K, MODE>), dim3(div_up(chunks, kLanes), rows, rt.npes), dim3(kLanes), 0, stream, dst, src, \
                  w, to, at, rt.heap_size, (uint64_t)recv_cap_rows, (unsigned)tokens, (unsigned)topk, (unsigned)dim,                \
                  (unsigned)rt.npes, log)
#define NVSHMEM_AMD_LAUNCH_SUM_OF(MODE)                 \
    switch (topk) {                                     \
        case 1: NVSHMEM_AMD_LAUNCH_SUM(1, MODE); break; \
        case 2: NVSHMEM_AMD_LAUNCH_SUM(2, MODE); break; \
        case 3: NVSHMEM_AMD_LAUNCH_SUM(3, MODE); break; \
        case 4: NVSHMEM_AMD_LAUNCH_SUM(4, MODE); break; \
        case 5: NVSHMEM_AMD_LAUNCH_SUM(5, MODE); break; \
        case 6: NVSHMEM_AMD_LAUNCH_SUM(6, MODE); break; \
        case 7: NVSHMEM_AMD_LAUNCH_SUM(7, MODE); break; \
        default: NVSHMEM_AMD_LAUNCH_SUM(8, MODE);       \
    }
    if (dim < (size_t)Chunk<T>::N) NVSHMEM_AMD_LAUNCH_SUM(8, kTiny);
    else if (topk == 1 && (uint64_t)tokens * rt.npes / (kLanes >> log) * div_up(chunks, kLanes) >= kManyPieces) {
        const unsigned fours = div_up(tokens, (kLanes >> log) * kTokens);
        const dim3 grid(div_up(chunks, kLanes), fours < 65535 ? fours : 65535, rt.npes);
        if (log == 6)
            launch_kernel((combine_one_kernel<T, kWhole>), grid, dim3(kLanes), 0, stream, dst, src, w, to, at, rt.heap_size,
                          (uint64_t)recv_cap_rows, (unsigned)tokens, (unsigned)dim, (unsigned)rt.npes, log);
        else
            launch_kernel((combine_one_kernel<T, kShared>), grid, dim3(kLanes), 0, stream, dst, src, w, to, at, rt.heap_size,
                          (uint64_t)recv_cap_rows, (unsigned)tokens, (unsigned)dim, (unsigned)rt.npes, log);
    }
    else if (log == 6) NVSHMEM_AMD_LAUNCH_SUM_OF(kWhole)
    else NVSHMEM_AMD_LAUNCH_SUM_OF(kShared)
#undef NVSHMEM_AMD_LAUNCH_SUM_OF
#undef NVSHMEM_AMD_LAUNCH_SUM
    return launched("moe_combine_sum");
}

template <typename API>
int combine_grad_on_stream(API *drecv, float *dgate, const API *dout, const API *recv, size_t recv_cap_rows, const float *gate,
                           const int32_t *dest_pe, const int64_t *dest_row, size_t tokens, int topk, size_t dim, hipStream_t stream) {
    typedef typename element<API>::type T;
    Runtime &rt = Runtime::get();
    std::lock_guard<std::recursive_mutex> lock(rt.mu);
    if (!ready(rt, "moe_combine_grad")) return NVSHMEMX_ERROR_INVALID_VALUE;
    if (int rc = check_sizes(rt, "moe_combine_grad", tokens, topk, dim)) return rc;
    NVSHMEM_AMD_REFUSE(recv_cap_rows > rt.heap_size / (dim * sizeof(T)), "moe_combine_grad recv: %zu rows leave the PE's heap slice", recv_cap_rows);
    const uint64_t copies = (uint64_t)tokens * topk;
    Operands ops(rt, "moe_combine_grad");
    const T *src = (const T *)ops.in("recv", recv, (uint64_t)recv_cap_rows * dim);
    const T *from = (const T *)ops.in("dout", dout, (uint64_t)tokens * dim);
    const int32_t *to = ops.in("dest_pe", dest_pe, copies);
    const int64_t *at = ops.in("dest_row", dest_row, copies);
    const float *w = ops.in("gate", gate, copies);
    float *dw = ops.out("dgate", dgate, copies);
    ops.may_be(src);
    T *dst = (T *)ops.out("drecv", drecv, (uint64_t)recv_cap_rows * dim);
    if (!ops.ok()) return NVSHMEMX_ERROR_INVALID_VALUE;
    if (tokens == 0) return 0;
    // as many wavefronts as make the last of their steps through a row a full one, more or less
    const unsigned chunks = div_up(dim, Chunk<T>::N), steps = div_up(chunks, kGradWaves * kLanes), waves = div_up(chunks, steps * kLanes);
#define NVSHMEM_AMD_LAUNCH_GRAD(K, TINY)                                                                                             \
    launch_kernel((combine_grad_kernel<T, K, TINY>), dim3((unsigned)(tokens < (1u << 20) ? tokens : 1u << 20), 1, rt.npes),          \
                  dim3(waves * kLanes), 0, stream, dst, dw, from, src, w, to, at, rt.heap_size, (uint64_t)recv_cap_rows,             \
                  (unsigned)tokens, (unsigned)topk, (unsigned)dim, (unsigned)rt.npes)
    if (dim < (size_t)Chunk<T>::N) {
        NVSHMEM_AMD_LAUNCH_GRAD(8, true);
    } else {
        switch (topk) {
            case 1: NVSHMEM_AMD_LAUNCH_GRAD(1, false); break;
            case 2: NVSHMEM_AMD_LAUNCH_GRAD(2, false); break;
            case 3: NVSHMEM_AMD_LAUNCH_GRAD(3, false); break;
            case 4: NVSHMEM_AMD_LAUNCH_GRAD(4, false); break;
            case 5: NVSHMEM_AMD_LAUNCH_GRAD(5, false); break;
            case 6: NVSHMEM_AMD_LAUNCH_GRAD(6, false); break;
            case 7: NVSHMEM_AMD_LAUNCH_GRAD(7, false); break;
            default: NVSHMEM_AMD_LAUNCH_GRAD(8, false);
        }
    }
#undef NVSHMEM_AMD_LAUNCH_GRAD
    return launched("moe_combine_grad");
}

}  // namespace
}  // namespace tokens
}  // namespace nvshmem_amd

using namespace nvshmem_amd;

extern "C" {

#define NVSHMEM_AMD_COMBINE(NAME, TYPE)                                                                                            \
    int nvshmemx_amd_##NAME##_moe_combine_sum_on_stream(TYPE *out, const TYPE *recv, size_t recv_cap_rows, const float *gate,      \
                                                        const int32_t *dest_pe, const int64_t *dest_row, size_t tokens, int topk,  \
                                                        size_t dim, nvshmemx_stream_t stream) {                                    \
        return tokens::combine_sum_on_stream(out, recv, recv_cap_rows, gate, dest_pe, dest_row, tokens, topk, dim,                 \
                                             (hipStream_t)stream);                                                                 \
    }                                                                                                                              \
    int nvshmemx_amd_##NAME##_moe_combine_grad_on_stream(TYPE *drecv, float *dgate, const TYPE *dout, const TYPE *recv,            \
                                                         size_t recv_cap_rows, const float *gate, const int32_t *dest_pe,          \
                                                         const int64_t *dest_row, size_t tokens, int topk, size_t dim,             \
                                                         nvshmemx_stream_t stream) {                                               \
        return tokens::combine_grad_on_stream(drecv, dgate, dout, recv, recv_cap_rows, gate, dest_pe, dest_row, tokens, topk, dim, \
                                              (hipStream_t)stream);                                                                \
    }
NVSHMEMI_AMD_REPT_FOR_TOKEN_TYPES(NVSHMEM_AMD_COMBINE)
#undef NVSHMEM_AMD_COMBINE

}  // extern "C"
