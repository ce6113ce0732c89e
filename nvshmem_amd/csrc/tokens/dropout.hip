// Rows of tokens with elements dropped, added to a residual; which ones stay follows from a counter and is stored nowhere.
//
//   out@p[e] = residual@p[e] + (keep(p, e) ? rows@p[e] / (1 - P) : 0)      e = t * dim + i,  P = limit / 2^16,  limit = round(2^16 p)
//
// keep(p, e): 16 bits of Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers, as easy as 1, 2, 3; 2011) are not below
// the limit.  Element e has the bits [16 (e % 8), + 16) of block e / 8, whose counter is {e / 8 (48 bits), PE (16 bits), seed[1]} and
// whose key is seed[0].  So the mask is a function of (seed, PE, e) alone, whatever the launch; the gradient is the same call on dout.
#include "token_common.hpp"

namespace nvshmem_amd {
namespace tokens {
namespace {

typedef unsigned v4u __attribute__((ext_vector_type(4)));

__device__ __forceinline__ v4u philox(uint64_t block, uint64_t second, uint64_t key) {
    unsigned c0 = (unsigned)block, c1 = (unsigned)(block >> 32), c2 = (unsigned)second, c3 = (unsigned)(second >> 32);
    unsigned k0 = (unsigned)key, k1 = (unsigned)(key >> 32);
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
        c0 = (unsigned)(p1 >> 32) ^ c1 ^ k0, c1 = (unsigned)p1;
        c2 = (unsigned)(p0 >> 32) ^ c3 ^ k1, c3 = (unsigned)p0;
        k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
    }
    return v4u{c0, c1, c2, c3};
}

// A lane has eight elements, one block of the generator, in one or two chunks of 16 bytes.  16 bits an element, as 32 would have the generator run
// twice as often (ten rounds of two products, 28 operations an element): the vector unit, not memory, would bound it.  Bound by memory: 8 x 4096 rows
// of 7168 bf16 and a residual (1.41 GB) take 217 us, 6.5 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(T *out, const T *rows, const T *residual, const uint64_t *seed, uint64_t stride,
                                                      uint64_t elems, unsigned limit, float scale) {
    constexpr unsigned kChunks = 8 / Chunk<T>::N, N = Chunk<T>::N;
    typedef typename Chunk<T>::facc facc;
    const unsigned pe = blockIdx.z;
    const uint64_t *my_seed = copy_of(seed, pe, stride);
    const uint64_t key = my_seed[0], second = my_seed[1];
    const T *x = copy_of(rows, pe, stride);
    const T *r = residual ? copy_of(residual, pe, stride) : nullptr;
    T *y = copy_of(out, pe, stride);
    const uint64_t blocks = (elems + 7) / 8;
    for (uint64_t b = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; b < blocks; b += (uint64_t)gridDim.x * blockDim.x) {
        const uint64_t e = b * 8;
        const bool whole = elems - e >= 8;
        typename Chunk<T>::vec v[kChunks], w[kChunks] = {};
#pragma unroll
        for (unsigned c = 0; c < kChunks; ++c) {
            const uint64_t at = e + c * N;
            const unsigned n = at < elems ? (elems - at < N ? (unsigned)(elems - at) : N) : 0;
            v[c] = whole ? chunk_load_stream(x + at) : chunk_load_part(x + at, n);
            if (r) w[c] = whole ? chunk_load_stream(r + at) : chunk_load_part(r + at, n);
        }
        const v4u bits = philox(b | (uint64_t)pe << 48, second, key);
#pragma unroll
        for (unsigned c = 0; c < kChunks; ++c) {
            const uint64_t at = e + c * N;
            facc f = chunk_to_float<T>(v[c]);
            const facc add = chunk_to_float<T>(w[c]);
#pragma unroll
            for (unsigned i = 0; i < N; ++i) {
                const unsigned j = c * N + i, mine = bits[j / 2] >> j % 2 * 16 & 0xffff;
                // (a selection, not a product: a dropped element may be infinite or a NaN)
                f[i] = mine >= limit ? f[i] * scale : 0.0f;
                if (r) f[i] += add[i];
            }
            if (whole) chunk_store_stream(y + at, chunk_from_float<T>(f));
            else chunk_store_part(y + at, chunk_from_float<T>(f), at < elems ? (elems - at < N ? (unsigned)(elems - at) : N) : 0);
        }
    }
}

template <typename API>
int dropout_on_stream(API *out, const API *rows, const API *residual, const uint64_t *seed, size_t tokens, size_t dim, float p,
                      hipStream_t stream) {
    typedef typename element<API>::type T;
    Runtime &rt = Runtime::get();
    std::lock_guard<std::recursive_mutex> lock(rt.mu);
    if (!ready(rt, "dropout")) return NVSHMEMX_ERROR_INVALID_VALUE;
    NVSHMEM_AMD_REFUSE(!(p >= 0.0f && p < 1.0f), "dropout: a probability of %g, outside [0, 1)", (double)p);
    const unsigned limit = (unsigned)__builtin_rint((double)p * 65536.0);
    NVSHMEM_AMD_REFUSE(limit >= 65536, "dropout: a probability of %g, which is 1 in steps of 2^-16", (double)p);
    NVSHMEM_AMD_REFUSE(dim < 1 || dim > (1u << 24), "dropout: rows of %zu elements, outside [1, 2^24]", dim);
    NVSHMEM_AMD_REFUSE(tokens > rt.heap_size / (dim * sizeof(T)), "dropout: %zu tokens leave the PE's heap slice", tokens);
    const uint64_t elems = (uint64_t)tokens * dim;
    Operands ops(rt, "dropout");
    const T *x = (const T *)ops.in("rows", rows, elems);
    const uint64_t *s = ops.in("seed", seed, 2);
    const T *r = residual ? (const T *)ops.in("residual", residual, elems) : nullptr;
    ops.may_be(residual ? (const void *)r : (const void *)x);
    T *y = (T *)ops.out("out", out, elems);
    if (!ops.ok()) return NVSHMEMX_ERROR_INVALID_VALUE;
    if (elems == 0) return 0;
    const uint64_t blocks = (elems + 8 * 256 - 1) / (8 * 256), most = (1u << 23) / (unsigned)rt.npes;  // (a launch holds fewer than 2^32 threads)
    launch_kernel(dropout_kernel<T>, dim3((unsigned)(blocks < most ? blocks : most), 1, rt.npes), dim3(256), 0, stream, y, x, r, s,
                  rt.heap_size, elems, limit, (float)(65536.0 / (65536.0 - limit)));
    return launched("dropout");
}

}  // namespace
}  // namespace tokens
}  // namespace nvshmem_amd

using namespace nvshmem_amd;

extern "C" {

#define NVSHMEM_AMD_DROPOUT(NAME, TYPE)                                                                                        \
    int nvshmemx_amd_##NAME##_dropout_on_stream(TYPE *out, const TYPE *rows, const TYPE *residual, const uint64_t *seed,       \
                                                size_t tokens, size_t dim, float p, nvshmemx_stream_t stream) {                \
        return tokens::dropout_on_stream(out, rows, residual, seed, tokens, dim, p, (hipStream_t)stream);                      \
    }
NVSHMEMI_AMD_REPT_FOR_TOKEN_TYPES(NVSHMEM_AMD_DROPOUT)
#undef NVSHMEM_AMD_DROPOUT

}  // extern "C"
