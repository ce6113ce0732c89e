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

// Most copies of a token whose loads are in flight together.
constexpr int kCopies = 8;

// One wavefront per piece of 64 chunks of a token's row, or rows of fewer chunks that share a wavefront, 2^lanes_log lanes each.
// Reads every copy once and writes a row: bound by memory.  All K loads of a lane leave before the first is used, so neither their
// addresses nor whether a copy was dropped may be waited for in between: a dropped copy's load goes to the row to be written.
// Where a wavefront has one token, its entries are scalar loads and its rows scalar addresses.
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

// A block per token.  A thread keeps the products of its chunks for up to kCopies gates in registers; the block adds them up at
// the end, lane by lane and then wavefront by wavefront.
template <typename T>
__global__ __launch_bounds__(256) void combine_grad_kernel(T *drecv, float *dgate, const T *dout, const T *recv, const float *gate,
                                                           const int32_t *dest_pe, const int64_t *dest_row, uint64_t stride,
                                                           uint64_t cap, unsigned tokens, unsigned topk, unsigned dim,
                                                           unsigned npes) {
    constexpr unsigned N = Chunk<T>::N;
    __shared__ float partial[4][kCopies];
    const unsigned pe = blockIdx.z;
    const int32_t *my_pe = copy_of(dest_pe, pe, stride);
    const int64_t *my_row = copy_of(dest_row, pe, stride);
    const float *my_gate = copy_of(gate, pe, stride);
    const T *my_dout = copy_of(dout, pe, stride);
    float *my_dgate = copy_of(dgate, pe, stride);
    for (uint64_t t = (uint64_t)blockIdx.y * gridDim.x + blockIdx.x; t < tokens; t += (uint64_t)gridDim.y * gridDim.x) {
        for (unsigned k0 = 0; k0 < topk; k0 += kCopies) {
            float dot[kCopies] = {};
            for (unsigned first = threadIdx.x * N; first < dim; first += 256 * N) {
                const unsigned left = dim - first;
                const T *from = my_dout + t * dim + first;
                const typename Chunk<T>::facc g = chunk_to_float<T>(left >= N ? chunk_load(from) : chunk_load_part(from, left));
#pragma unroll
                for (unsigned k = 0; k < kCopies; ++k) {
                    if (k0 + k >= topk) continue;
                    const uint64_t c = t * topk + k0 + k;
                    const unsigned d = (unsigned)my_pe[c];
                    const uint64_t r = (uint64_t)my_row[c];
                    if (d >= npes || r >= cap) continue;
                    const uint64_t at = r * dim + first;
                    const T *src = copy_of(recv, d, stride) + at;
                    const typename Chunk<T>::facc x = chunk_to_float<T>(left >= N ? chunk_load(src) : chunk_load_part(src, left));
#pragma unroll
                    for (unsigned i = 0; i < N; ++i) dot[k] = __builtin_fmaf(x[i], g[i], dot[k]);
                    T *dst = copy_of(drecv, d, stride) + at;
                    const typename Chunk<T>::vec y = chunk_from_float<T>(g * my_gate[c]);
                    if (left >= N) chunk_store_stream(dst, y);
                    else chunk_store_part(dst, y, left);
                }
            }
#pragma unroll
            for (int k = 0; k < kCopies; ++k) {
                for (int m = 32; m; m >>= 1) dot[k] += __shfl_xor(dot[k], m);
                if (threadIdx.x % kLanes == 0) partial[threadIdx.x / kLanes][k] = dot[k];
            }
            __syncthreads();
            if (threadIdx.x < kCopies && k0 + threadIdx.x < topk)
                my_dgate[t * topk + k0 + threadIdx.x] = (partial[0][threadIdx.x] + partial[1][threadIdx.x]) +
                                                        (partial[2][threadIdx.x] + partial[3][threadIdx.x]);
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
    launch_kernel(combine_grad_kernel<T>, dim3((unsigned)(tokens < (1u << 20) ? tokens : 1u << 20), 1, rt.npes), dim3(256), 0, stream,
                  dst, dw, from, src, w, to, at, rt.heap_size, (uint64_t)recv_cap_rows, (unsigned)tokens, (unsigned)topk,
                  (unsigned)dim, (unsigned)rt.npes);
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
