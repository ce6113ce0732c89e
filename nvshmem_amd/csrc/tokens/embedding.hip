// Embedding lookup with scaling from a table that is cut by rows over the PEs, and the table's gradient.
//
//   out@p[t] = scale * table@(v / R)[v % R]           v = ids@p[t], R = ceil(vocab / npes) rows of the table on each PE
//   dtable@(v / R)[v % R] = scale * sum dout@p[t]     over all (p, t) with ids@p[t] = v, in the order of (p, t)
//
// An id outside [0, vocab) is padding: a row of zeros, no gradient.
#include "token_common.hpp"

namespace nvshmem_amd {
namespace tokens {
namespace {

// One wavefront per piece of 64 chunks of a row; a row of fewer chunks takes the next power of two lanes and shares its
// wavefront with others (2^lanes_log lanes a row).  Reads T x dim elements of the table and writes as many: bound by memory.
template <typename T>
__global__ __launch_bounds__(64) void embedding_kernel(T *out, const T *table, const int64_t *ids, uint64_t stride,
                                                       unsigned tokens, unsigned vocab, unsigned rows, unsigned dim,
                                                       unsigned lanes_log, float scale) {
    constexpr unsigned N = Chunk<T>::N;
    const unsigned lane = threadIdx.x, pe = blockIdx.z;
    const unsigned first = (blockIdx.x * kLanes + (lane & ((1u << lanes_log) - 1))) * N;
    if (first >= dim) return;
    const unsigned left = dim - first;
    const int64_t *my_ids = copy_of(ids, pe, stride);
    T *my_out = copy_of(out, pe, stride);
    const unsigned per_wave = kLanes >> lanes_log;
    for (uint64_t t = (uint64_t)blockIdx.y * per_wave + (lane >> lanes_log); t < tokens; t += (uint64_t)gridDim.y * per_wave) {
        const uint64_t id = (uint64_t)my_ids[t];
        typename Chunk<T>::facc x = {};
        if (id < vocab) {
            const unsigned owner = (unsigned)id / rows, row = (unsigned)id % rows;
            const T *src = copy_of(table, owner, stride) + (uint64_t)row * dim + first;
            x = chunk_to_float<T>(left >= N ? chunk_load(src) : chunk_load_part(src, left));
        }
        const typename Chunk<T>::vec y = chunk_from_float<T>(x * scale);
        T *dst = my_out + t * dim + first;
        if (left >= N) chunk_store_stream(dst, y);
        else chunk_store_part(dst, y, left);
    }
}

// ---- gradient ----
// The tokens of all PEs are sorted by id, stable; a wavefront adds up kPart consecutive ones of a piece of a row, in order, and
// writes the sums of the ids that lie in its part as a whole.  A sum that goes on into the next part leaves a partial sum in fp32
// (`carry`), and a kernel behind it adds those up, in order: nothing depends on which block comes first.
constexpr unsigned kPart = 32;

// Place of every token in the sorted order, by counting the smaller ones.
__global__ __launch_bounds__(256) void embedding_rank_kernel(uint32_t *key_out, uint32_t *pos_out, const int64_t *ids,
                                                             uint64_t stride, unsigned tokens, unsigned n, unsigned vocab) {
    __shared__ uint32_t tile[256];
    const unsigned i = blockIdx.x * 256 + threadIdx.x;
    auto key_of = [&](unsigned j) -> uint32_t {
        if (j >= n) return 0xffffffffu;
        const uint64_t id = (uint64_t)copy_of(ids, j / tokens, stride)[j % tokens];
        return id < vocab ? (uint32_t)id : vocab;
    };
    const uint32_t mine = key_of(i);
    unsigned rank = 0;
    for (unsigned base = 0; base < n; base += 256) {
        __syncthreads();
        tile[threadIdx.x] = key_of(base + threadIdx.x);
        __syncthreads();
        for (unsigned j = 0; j < 256 && base + j < n; ++j)
            rank += (tile[j] < mine || (tile[j] == mine && base + j < i)) ? 1u : 0u;
    }
    if (i < n) {
        key_out[rank] = mine;
        pos_out[rank] = i;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void embedding_zero_kernel(T *dtable, uint64_t stride, unsigned vocab, unsigned rows,
                                                             unsigned dim) {
    const unsigned owner = blockIdx.z;
    const uint64_t first = (uint64_t)owner * rows;
    if (first >= vocab) return;
    const uint64_t elems = (uint64_t)(vocab - first < rows ? vocab - first : rows) * dim;
    T *mine = copy_of(dtable, owner, stride);
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < elems; i += (uint64_t)gridDim.x * 256) mine[i] = (T)0.0f;
}

template <typename T>
__device__ __forceinline__ void write_row(T *dtable, uint64_t stride, uint32_t key, unsigned rows, unsigned dim, unsigned first,
                                          unsigned left, typename Chunk<T>::facc sum, float scale) {
    T *dst = copy_of(dtable, key / rows, stride) + (uint64_t)(key % rows) * dim + first;
    const typename Chunk<T>::vec y = chunk_from_float<T>(sum * scale);
    if (left >= (unsigned)Chunk<T>::N) chunk_store_stream(dst, y);
    else chunk_store_part(dst, y, left);
}

template <typename T>
__global__ __launch_bounds__(64) void embedding_sum_kernel(T *dtable, float *carry, const T *dout, const uint32_t *key,
                                                           const uint32_t *pos, uint64_t stride, unsigned tokens, unsigned n,
                                                           unsigned vocab, unsigned rows, unsigned dim, unsigned pitch,
                                                           float scale) {
    constexpr unsigned N = Chunk<T>::N;
    typedef typename Chunk<T>::facc facc;
    const unsigned first = (blockIdx.x * kLanes + threadIdx.x) * N, left = first < dim ? dim - first : 0;
    for (unsigned part = blockIdx.y; (uint64_t)part * kPart < n; part += gridDim.y) {
    const unsigned begin = part * kPart, end = n - begin > kPart ? begin + kPart : n;
    facc sum = {};
    unsigned run = begin;  // where the run being added up begins, or begins in this part
    for (unsigned j = begin; j < end; ++j) {
        const uint32_t k = key[j];
        if (k >= vocab) break;
        if (left) {
            const uint32_t i = pos[j];
            const T *src = copy_of(dout, i / tokens, stride) + (uint64_t)(i % tokens) * dim + first;
            sum += chunk_to_float<T>(left >= N ? chunk_load(src) : chunk_load_part(src, left));
        }
        const bool last = j + 1 == end;
        if (!last && key[j + 1] == k) continue;
        const bool from_before = run == begin && begin > 0 && key[begin - 1] == k;
        const bool goes_on = last && end < n && key[end] == k;
        if (left) {
            if (!from_before && !goes_on) {
                write_row(dtable, stride, k, rows, dim, first, left, sum, scale);
            } else {
                // slot 0: a sum that came from the part before, slot 1: one that begins here
                float *c = carry + ((uint64_t)part * 2 + (from_before ? 0 : 1)) * pitch + first;
                *(facc *)c = sum;
            }
        }
        sum = facc{};
        run = j + 1;
    }
    }
}

template <typename T>
__global__ __launch_bounds__(64) void embedding_join_kernel(T *dtable, const float *carry, const uint32_t *key, uint64_t stride,
                                                            unsigned n, unsigned vocab, unsigned rows, unsigned dim,
                                                            unsigned pitch, float scale) {
    constexpr unsigned N = Chunk<T>::N;
    typedef typename Chunk<T>::facc facc;
    const unsigned first = (blockIdx.x * kLanes + threadIdx.x) * N;
    if (first >= dim) return;
    for (unsigned part = blockIdx.y; ((uint64_t)part + 1) * kPart < n; part += gridDim.y) {
    const unsigned begin = part * kPart, end = begin + kPart;
    const uint32_t k = key[end - 1];
    // a run that begins in this part and goes on
    if (k >= vocab || key[end] != k || (begin > 0 && key[begin - 1] == k)) continue;
    facc sum = *(const facc *)(carry + ((uint64_t)part * 2 + 1) * pitch + first);
    for (unsigned q = part + 1; (uint64_t)q * kPart < n && key[q * kPart] == k; ++q)
        sum += *(const facc *)(carry + (uint64_t)q * 2 * pitch + first);
    write_row(dtable, stride, k, rows, dim, first, dim - first, sum, scale);
    }
}

unsigned lanes_log2(size_t chunks) {
    unsigned l = 0;
    while (l < 6 && ((size_t)1 << l) < chunks) ++l;
    return l;
}

constexpr size_t kMostTokens = (size_t)1 << 31;

int check_sizes(Runtime &rt, const char *what, size_t tokens, size_t vocab, size_t dim, float scale) {
    NVSHMEM_AMD_REFUSE(tokens > kMostTokens / (size_t)rt.npes, "%s: %zu tokens on %d PEs, at most 2^31 in all", what, tokens, rt.npes);
    NVSHMEM_AMD_REFUSE(vocab < 1 || vocab > 0x7fffffffu, "%s: a table of %zu rows, outside [1, 2^31)", what, vocab);
    NVSHMEM_AMD_REFUSE(dim < 1 || dim > (1u << 24), "%s: rows of %zu elements, outside [1, 2^24]", what, dim);
    NVSHMEM_AMD_REFUSE(!(scale - scale == 0.0f), "%s: the scale must be finite", what);
    return 0;
}

template <typename API>
int embedding_on_stream(API *out, const API *table, const int64_t *ids, size_t tokens, size_t vocab, size_t dim, float scale,
                        hipStream_t stream) {
    typedef typename element<API>::type T;
    Runtime &rt = Runtime::get();
    std::lock_guard<std::recursive_mutex> lock(rt.mu);
    if (!ready(rt, "embedding")) return NVSHMEMX_ERROR_INVALID_VALUE;
    if (int rc = check_sizes(rt, "embedding", tokens, vocab, dim, scale)) return rc;
    const size_t rows = (vocab + rt.npes - 1) / rt.npes;
    Operands ops(rt, "embedding");
    const T *tab = (const T *)ops.in("table", table, (uint64_t)rows * dim);
    const int64_t *id = ops.in("ids", ids, tokens);
    T *dst = (T *)ops.out("out", out, (uint64_t)tokens * dim);
    if (!ops.ok()) return NVSHMEMX_ERROR_INVALID_VALUE;
    if (tokens == 0) return 0;
    const size_t chunks = (dim + Chunk<T>::N - 1) / Chunk<T>::N;
    const unsigned log = lanes_log2(chunks), groups = div_up(tokens, kLanes >> log);
    launch_kernel(embedding_kernel<T>, dim3(div_up(chunks, kLanes), groups < 65535 ? groups : 65535, rt.npes), dim3(kLanes), 0,
                  stream, dst, tab, id, rt.heap_size, (unsigned)tokens, (unsigned)vocab, (unsigned)rows, (unsigned)dim, log, scale);
    return launched("embedding");
}

// The gradient's workspace, in PE 0's copy: keys and positions in sorted order, and two partial sums for every part.
struct GradSpace {
    uint64_t key, pos, carry, bytes;
    unsigned pitch;
    GradSpace(uint64_t n, uint64_t dim) {
        const uint64_t list = (n * 4 + 63) / 64 * 64;
        pitch = (unsigned)((dim + 7) / 8 * 8);
        key = 0;
        pos = list;
        carry = 2 * list;
        bytes = carry + (n + kPart - 1) / kPart * 2 * pitch * sizeof(float);
    }
};

template <typename API>
int embedding_grad_on_stream(API *dtable, const API *dout, const int64_t *ids, void *workspace, size_t tokens, size_t vocab,
                             size_t dim, float scale, hipStream_t stream) {
    typedef typename element<API>::type T;
    Runtime &rt = Runtime::get();
    std::lock_guard<std::recursive_mutex> lock(rt.mu);
    if (!ready(rt, "embedding_grad")) return NVSHMEMX_ERROR_INVALID_VALUE;
    if (int rc = check_sizes(rt, "embedding_grad", tokens, vocab, dim, scale)) return rc;
    const size_t rows = (vocab + rt.npes - 1) / rt.npes, n = tokens * rt.npes;
    const GradSpace space(n, dim);
    Operands ops(rt, "embedding_grad");
    const T *src = (const T *)ops.in("dout", dout, (uint64_t)tokens * dim);
    const int64_t *id = ops.in("ids", ids, tokens);
    T *tab = (T *)ops.out("dtable", dtable, (uint64_t)rows * dim);
    char *ws = ops.out("workspace", (char *)workspace, n ? space.bytes : 0, 64);
    if (!ops.ok()) return NVSHMEMX_ERROR_INVALID_VALUE;
    launch_kernel(embedding_zero_kernel<T>, dim3(1024, 1, rt.npes), dim3(256), 0, stream, tab, rt.heap_size, (unsigned)vocab,
                  (unsigned)rows, (unsigned)dim);
    if (n) {
        uint32_t *key = (uint32_t *)(ws + space.key), *pos = (uint32_t *)(ws + space.pos);
        float *carry = (float *)(ws + space.carry);
        const unsigned pieces = div_up(dim, Chunk<T>::N * kLanes), parts = div_up(n, kPart) < 65535 ? div_up(n, kPart) : 65535;
        launch_kernel(embedding_rank_kernel, dim3(div_up(n, 256)), dim3(256), 0, stream, key, pos, id, rt.heap_size,
                      (unsigned)tokens, (unsigned)n, (unsigned)vocab);
        launch_kernel(embedding_sum_kernel<T>, dim3(pieces, parts), dim3(kLanes), 0, stream, tab, carry, src, key, pos,
                      rt.heap_size, (unsigned)tokens, (unsigned)n, (unsigned)vocab, (unsigned)rows, (unsigned)dim, space.pitch, scale);
        launch_kernel(embedding_join_kernel<T>, dim3(pieces, parts), dim3(kLanes), 0, stream, tab, carry, key, rt.heap_size,
                      (unsigned)n, (unsigned)vocab, (unsigned)rows, (unsigned)dim, space.pitch, scale);
    }
    return launched("embedding_grad");
}

}  // namespace
}  // namespace tokens
}  // namespace nvshmem_amd

using namespace nvshmem_amd;

extern "C" {

#define NVSHMEM_AMD_EMBEDDING(NAME, TYPE)                                                                                       \
    int nvshmemx_amd_##NAME##_embedding_on_stream(TYPE *out, const TYPE *table, const int64_t *ids, size_t tokens, size_t vocab, \
                                                  size_t dim, float scale, nvshmemx_stream_t stream) {                          \
        return tokens::embedding_on_stream(out, table, ids, tokens, vocab, dim, scale, (hipStream_t)stream);                    \
    }                                                                                                                           \
    int nvshmemx_amd_##NAME##_embedding_grad_on_stream(TYPE *dtable, const TYPE *dout, const int64_t *ids, void *workspace,     \
                                                       size_t tokens, size_t vocab, size_t dim, float scale,                    \
                                                       nvshmemx_stream_t stream) {                                              \
        return tokens::embedding_grad_on_stream(dtable, dout, ids, workspace, tokens, vocab, dim, scale, (hipStream_t)stream);  \
    }
NVSHMEMI_AMD_REPT_FOR_TOKEN_TYPES(NVSHMEM_AMD_EMBEDDING)
#undef NVSHMEM_AMD_EMBEDDING

size_t nvshmemx_amd_embedding_grad_workspace(size_t tokens, size_t vocab, size_t dim) {
    (void)vocab;
    const int npes = Runtime::get().npes;
    return npes < 1 ? 0 : tokens::GradSpace((uint64_t)tokens * npes, dim).bytes;
}

}  // extern "C"
