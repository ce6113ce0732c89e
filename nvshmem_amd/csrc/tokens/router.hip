// The router in front of the token shuffle: top-k experts of every token with their gates, counts per expert, the balance loss
// over all PEs, the gradient of gates and loss, and the shuffle's tables.
//
//   a logit of -inf or NaN masks an expert out;  m = max l, z = sum exp(l - m), p = exp(l - m) / z   (0 where masked)
//   S = the topk largest logits that are not masked, ties to the lowest expert; expert = -1 and gate = 0 where there are fewer
//   gate = scale * p / (normalise ? sum of p over S : 1)
//   counts@p[e] = copies that PE p sends to expert e;  c_e = sum of them over the PEs, C = sum of c_e, N = tokens with an expert
//   loss = E / (C N) sum_e c_e sum_t p[t, e],   balance[e] = d loss / d p[t, e] = E c_e / (C N)
//
// Backward, for upstream dgate and dloss:  q_e = dloss balance_e + (normalise ? 0 : scale dgate_e on S)
//   dl = p (q - sum q p) + (normalise ? w scale (dgate - sum_S w dgate) on S, w = p / sum_S p : 0)
#include "counting_sort.hpp"
#include "token_common.hpp"

namespace nvshmem_amd {
namespace tokens {
namespace {

constexpr int kMostExperts = 1024, kMostTopk = 16;

// ---- keys: a logit and its expert in one word, larger for the larger logit and then for the lower expert ----
// A logit is cleaned first: NaN becomes -inf, -0.0 becomes 0.0.  Its bits are then put in ascending order, in front of the
// expert's complement: 16-bit logits in an unsigned word, fp32 logits in the 52 mantissa bits of a double in [1, 2), which v_max_f64
// and v_min_f64 compare.  A key whose logit is -inf (or that is `none`, whose logit reads as NaN) is a masked expert's.
__device__ __forceinline__ uint32_t ascending(uint32_t b) { return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u); }
__device__ __forceinline__ uint32_t ascending_back(uint32_t s) { return s ^ (~(uint32_t)((int32_t)s >> 31) | 0x80000000u); }
// (the sum first: it quiets a signalling NaN, which a maximum would return; widening a bf16 leaves it one, whatever the compiler
// takes that for)
__device__ __forceinline__ float clean(float x) { return fmaxf(x + 0.0f, -__builtin_inff()); }

template <typename T>
struct Key {  // _Float16, __bf16
    typedef uint32_t type;
    static __device__ __forceinline__ type none() { return 0; }
    static __device__ __forceinline__ type make(float x, uint32_t e) {
        return (ascending((uint32_t)__builtin_bit_cast(uint16_t, (T)x) << 16) & 0xffff0000u) | (0xffffu - e);
    }
    static __device__ __forceinline__ uint32_t expert(type k) { return 0xffffu - (k & 0xffffu); }
    static __device__ __forceinline__ float logit(type k) {
        return (float)__builtin_bit_cast(T, (uint16_t)(ascending_back(k) >> 16));
    }
    static __device__ __forceinline__ type larger(type a, type b) { return a > b ? a : b; }
    static __device__ __forceinline__ type smaller(type a, type b) { return a < b ? a : b; }
};
template <>
struct Key<float> {
    typedef double type;
    static __device__ __forceinline__ type none() { return 1.0; }
    static __device__ __forceinline__ type make(float x, uint32_t e) {
        const uint32_t s = ascending(__float_as_uint(x));
        return __longlong_as_double((long long)((uint64_t)__builtin_amdgcn_alignbit(0x3ffu, s, 12) << 32 | (s << 20 | (0xfffffu - e))));
    }
    static __device__ __forceinline__ uint32_t expert(type k) { return 0xfffffu - ((uint32_t)__double_as_longlong(k) & 0xfffffu); }
    static __device__ __forceinline__ float logit(type k) {
        return __uint_as_float(ascending_back((uint32_t)((uint64_t)__double_as_longlong(k) >> 20)));
    }
    // (the instructions themselves: around fmax and fmin the compiler quiets NaNs that no key is)
    static __device__ __forceinline__ type larger(type a, type b) {
        type r;
        asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
        return r;
    }
    static __device__ __forceinline__ type smaller(type a, type b) {
        type r;
        asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
        return r;
    }
};

// Batcher's odd-even merge sort, largest first, all indices known at compile time.
template <typename K, int N>
__device__ __forceinline__ void sort_largest_first(typename K::type *a) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const typename K::type x = a[i + j], y = a[i + j + k];
                        a[i + j] = K::larger(x, y);
                        a[i + j + k] = K::smaller(x, y);
                    }
}
// The N largest of two sorted lists, sorted: one list against the other backwards leaves them, rising and then falling.
template <typename K, int N>
__device__ __forceinline__ void keep_largest(typename K::type *a, const typename K::type *b) {
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = K::larger(a[i], b[N - 1 - i]);
#pragma unroll
    for (int s = N / 2; s >= 1; s /= 2)
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (!(i & s)) {
                const typename K::type x = a[i], y = a[i + s];
                a[i] = K::larger(x, y);
                a[i + s] = K::smaller(x, y);
            }
}
template <typename K, int N, int STEP>
__device__ __forceinline__ void keep_largest_of_pair(typename K::type *a) {
    typename K::type b[N];
#pragma unroll
    for (int i = 0; i < N; ++i) b[i] = partner<STEP>(a[i]);
    keep_largest<K, N>(a, b);
}

// ---- a lane's V logits of a token: loads of W neighbouring ones, G lanes side by side ----
template <typename T, int G, int V>
struct Slots {
    static constexpr int W = V < chunk_elems<T>() ? V : chunk_elems<T>();
    typedef T vec __attribute__((ext_vector_type(W)));
    typedef vec vec_unaligned __attribute__((aligned(sizeof(T))));
    static __device__ __forceinline__ unsigned expert(int u, unsigned sub) { return (unsigned)(u / W * G + sub) * W + u % W; }
    static __device__ __forceinline__ void load(T *x, const T *row, unsigned experts, unsigned sub) {
#pragma unroll
        for (int u = 0; u < V; u += W) {
            const unsigned e = expert(u, sub);
            if (e + W <= experts) {
                const vec v = *reinterpret_cast<const vec_unaligned *>(row + e);
#pragma unroll
                for (int i = 0; i < W; ++i) x[u + i] = v[i];
            } else {
#pragma unroll
                for (int i = 0; i < W; ++i) x[u + i] = e + i < experts ? row[e + i] : (T)-__builtin_inff();
            }
        }
    }
    static __device__ __forceinline__ void store(T *row, const T *x, unsigned experts, unsigned sub) {
#pragma unroll
        for (int u = 0; u < V; u += W) {
            const unsigned e = expert(u, sub);
            if (e + W <= experts) {
                vec v;
#pragma unroll
                for (int i = 0; i < W; ++i) v[i] = x[u + i];
                __builtin_nontemporal_store(v, reinterpret_cast<vec_unaligned *>(row + e));
            } else {
#pragma unroll
                for (int i = 0; i < W; ++i)
                    if (e + i < experts) row[e + i] = x[u + i];
            }
        }
    }
};

// exp(l - m) for l <= m; two infinities of a sign differ by nothing.
__device__ __forceinline__ float exp_below(float l, float m) { return __expf(l == m ? 0.0f : l - m); }

struct RouteArgs {
    uint64_t stride;
    int32_t *expert;
    float *gate;
    int64_t *counts;  // written by the blocks themselves where a PE has one block, and no loss is asked for
    char *work;
    uint64_t hist, psum, rows, ticket;
    unsigned tokens, threads, per_block, blocks, experts, topk;
    int normalise, loss;
    float scale;
};

// Threads of a block: few for few tokens, which then spread over more compute units, many for many, whose second kernel then has
// fewer rows to read.  us with 256 / 1024, 256 experts, bf16: 1024 tokens in all 6.4 / 9.2, 8192 8.2 / 10.4; from 16384 on 1024 are ahead,
// with 65536 tokens by what the second kernel saves (14.0 with 1024 blocks, 9.6 with 256).
//
// What bounds it in large batches is the vector unit, busy for 78 % of the time: 642 instructions for 4 tokens of 256 experts, of which
// 236 compare keys, 64 carry them to other lanes, 96 make them and 100 are the softmax.  65536 tokens of 256 fp32 logits: 26.5 us (the
// 67 MB alone would take 10.5); bf16 23.  8 lanes a token with twice the keys each take as long.  Four tokens to a group, merged
// so that each quad of lanes ends up with one (5 merges for 4 tokens instead of 16), spill and take 35 us; the next tokens' logits
// loaded ahead change nothing.
constexpr unsigned kRouteThreads = 256, kRouteMostThreads = 1024;

template <typename T, int G, int V, int KP>
__global__ __launch_bounds__(kRouteMostThreads) void route_kernel(const T *logits, RouteArgs a) {
    typedef Key<T> K;
    const unsigned threads = a.threads, waves = threads / kLanes, groups = threads / G;
    extern __shared__ uint32_t lds[];  // hist[experts], float psum[waves][experts], rows
    uint32_t *hist = lds;
    float *psum = (float *)(lds + a.experts);
    uint32_t *rows = lds + a.experts * (1 + (a.loss ? waves : 0));
    const unsigned pe = blockIdx.z, sub = threadIdx.x % G, group = threadIdx.x / G;
    for (unsigned e = threadIdx.x; e < a.experts; e += threads) hist[e] = 0;
    if (threadIdx.x == 0) rows[0] = 0;
    __syncthreads();
    if (a.loss && blockIdx.x == 0 && pe == 0 && threadIdx.x == 0) *(uint32_t *)(a.work + a.ticket) = 0;

    const T *my_logits = copy_of(logits, pe, a.stride);
    int32_t *my_expert = copy_of(a.expert, pe, a.stride);
    float *my_gate = copy_of(a.gate, pe, a.stride);
    const unsigned begin = blockIdx.x * a.per_block, end = a.tokens - begin > a.per_block ? begin + a.per_block : a.tokens;
    float mass[V] = {};
    unsigned live = 0;
    for (unsigned t0 = begin; t0 < end; t0 += groups) {  // (all lanes take part in every exchange)
        const unsigned t = t0 + group;
        T raw[V];
        Slots<T, G, V>::load(raw, my_logits + (uint64_t)(t < end ? t : begin) * a.experts, a.experts, sub);
        float x[V];
        typename K::type key[V < KP ? KP : V];
#pragma unroll
        for (int u = 0; u < V; ++u) {
            x[u] = clean((float)raw[u]);
            key[u] = K::make(x[u], Slots<T, G, V>::expert(u, sub));
        }
        if (V < KP) {
            sort_largest_first<K, V>(key);
#pragma unroll
            for (int u = V; u < KP; ++u) key[u] = K::none();
        } else {
#pragma unroll
            for (int u = 0; u < V; u += KP) {
                sort_largest_first<K, KP>(key + u);
                if (u) keep_largest<K, KP>(key, key + u);
            }
        }
        keep_largest_of_pair<K, KP, 0>(key);
        keep_largest_of_pair<K, KP, 1>(key);
        keep_largest_of_pair<K, KP, 2>(key);
        keep_largest_of_pair<K, KP, 3>(key);
        if (G == 64) {
            keep_largest_of_pair<K, KP, 4>(key);
            keep_largest_of_pair<K, KP, 5>(key);
        }
        const float m = K::logit(key[0]);
        const bool some = m > -__builtin_inff();
        float z = 1.0f;
        if (a.loss || !a.normalise) {
            // weights against the largest logit; where that is inf, those that are inf weigh 1 and the others nothing
            const bool endless = m == __builtin_inff();
            if (__builtin_amdgcn_ballot_w64(endless)) {
#pragma unroll
                for (int u = 0; u < V; ++u) x[u] = endless ? (x[u] == m ? 0.0f : -__builtin_inff()) : x[u];
            }
            const float top = some && !endless ? m : 0.0f;
            float sum = 0.0f;
#pragma unroll
            for (int u = 0; u < V; ++u) {
                x[u] = __expf(x[u] - top);
                sum += x[u];
            }
            z = group_sum<G>(sum);
            const float r = some && t < end ? 1.0f / z : 0.0f;
#pragma unroll
            for (int u = 0; u < V; ++u) mass[u] = __builtin_fmaf(x[u], r, mass[u]);
        }
        typename K::type own = K::none();
#pragma unroll
        for (int k = 0; k < KP; ++k)
            if (sub == (unsigned)k) own = key[k];
        const float l = K::logit(own);
        const bool chosen = sub < a.topk && l > -__builtin_inff();
        const float p = chosen ? exp_below(l, m) : 0.0f;
        const float s = group_sum<G>(p);
        if (t < end) {
            live += some && sub == 0;
            if (sub < a.topk) {
                const uint32_t e = K::expert(own);
                my_expert[(uint64_t)t * a.topk + sub] = chosen ? (int32_t)e : -1;
                my_gate[(uint64_t)t * a.topk + sub] = chosen ? a.scale * (p / (a.normalise ? s : z)) : 0.0f;
                if (chosen) atomicAdd(&hist[e], 1u);
            }
        }
    }
    if (live) atomicAdd(rows, live);
    if (a.loss) {
#pragma unroll
        for (int u = 0; u < V; ++u) {
            if (G == 16) {
                mass[u] += partner<4>(mass[u]);
                mass[u] += partner<5>(mass[u]);
            }
            const unsigned e = Slots<T, G, V>::expert(u, sub);
            if (threadIdx.x % kLanes < G && e < a.experts) psum[threadIdx.x / kLanes * a.experts + e] = mass[u];
        }
    }
    __syncthreads();
    char *work = copy_of(a.work, pe, a.stride);
    for (unsigned e = threadIdx.x; e < a.experts; e += threads) {
        if (a.counts) copy_of(a.counts, pe, a.stride)[e] = hist[e];
        else ((uint32_t *)(work + a.hist))[(uint64_t)blockIdx.x * a.experts + e] = hist[e];
        if (a.loss) {
            float s = 0.0f;
            for (unsigned w = 0; w < waves; ++w) s += psum[w * a.experts + e];
            ((float *)(work + a.psum))[(uint64_t)blockIdx.x * a.experts + e] = s;
        }
    }
    if (a.loss) {
        if (threadIdx.x == 0) ((uint32_t *)(work + a.rows))[2 * blockIdx.x] = rows[0];
        // copies of this block
        __syncthreads();
        if (threadIdx.x < kLanes) {
            uint32_t n = 0;
            for (unsigned e = threadIdx.x; e < a.experts; e += kLanes) n += hist[e];
            for (int s = 32; s; s >>= 1) n += __shfl_xor((int)n, s);
            if (threadIdx.x == 0) ((uint32_t *)(work + a.rows))[2 * blockIdx.x + 1] = n;
        }
    }
}

// Counts, loss and its derivative from what the blocks of all PEs left.  A block has 8 experts, a wavefront 8 rows of a PE's at a
// time, so that no wavefront waits for another until all PEs are added up (32 experts a block, waiting after each PE: 25 us, so
// 9.6, for 256 rows of 256 experts).  It waits for memory four times in a row: rows, own result, ticket, all results.
constexpr unsigned kFinishExperts = 8, kFinishWaves = 16;

__global__ __launch_bounds__(kFinishWaves *kLanes) void route_finish_kernel(int64_t *counts, float *loss, float *balance, char *work,
                                                                            uint64_t stride, uint64_t hist, uint64_t psum,
                                                                            uint64_t rows, uint64_t ticket, unsigned blocks,
                                                                            unsigned experts, unsigned npes) {
    __shared__ double value[kFinishWaves][kFinishExperts];
    __shared__ unsigned long long copies[kFinishExperts], totals[2];
    __shared__ unsigned last;
    const unsigned wave = wave_of_block(), x = threadIdx.x % kFinishExperts, y = threadIdx.x % kLanes / kFinishExperts;
    const unsigned e = blockIdx.x * kFinishExperts + x;
    if (threadIdx.x < kFinishExperts) copies[threadIdx.x] = 0;
    if (threadIdx.x < 2) totals[threadIdx.x] = 0;
    __syncthreads();
    double mass = 0.0;
    // tokens and copies of all PEs
    unsigned long long tokens_here = 0, copies_here = 0;
    if (loss) {
        for (unsigned i = threadIdx.x; i < npes * blocks; i += kFinishWaves * kLanes) {
            const uint32_t *r = (const uint32_t *)(copy_of(work, i / blocks, stride) + rows) + 2 * (i % blocks);
            tokens_here += r[0];
            copies_here += r[1];
        }
    }
    for (unsigned pe = wave; pe < npes; pe += kFinishWaves) {
        const char *w = copy_of(work, pe, stride);
        const uint32_t *h = (const uint32_t *)(w + hist) + e;
        const float *s = (const float *)(w + psum) + e;
        uint32_t c = 0;
        if (e < experts) {
            if (loss) {
#pragma unroll 8
                for (unsigned r = y; r < blocks; r += kLanes / kFinishExperts) {
                    c += h[(uint64_t)r * experts];
                    mass += s[(uint64_t)r * experts];
                }
            } else {
#pragma unroll 8
                for (unsigned r = y; r < blocks; r += kLanes / kFinishExperts) c += h[(uint64_t)r * experts];
            }
        }
        c += dpp<0x128>(c);  // row_ror:8
        c += partner<4>(c);
        c += partner<5>(c);
        if (y == 0 && e < experts) {
            copy_of(counts, pe, stride)[e] = c;
            atomicAdd(&copies[x], (unsigned long long)c);
        }
    }
    if (!loss) return;
    for (int s = kFinishExperts; s < kLanes; s <<= 1) mass += __shfl_xor(mass, s);
    if (y == 0) value[wave][x] = mass;
    if (tokens_here) atomicAdd(&totals[0], tokens_here);
    if (copies_here) atomicAdd(&totals[1], copies_here);
    __syncthreads();
    double *found = (double *)(work + ticket + 64);
    if (wave == 0) {
        double v = 0.0;
        if (y == 0 && e < experts) {
            const double b = totals[1] ? (double)experts * (double)copies[x] / ((double)totals[1] * (double)totals[0]) : 0.0;
            for (unsigned w = 0; w < kFinishWaves; ++w) v += value[w][x];
            v *= b;
            for (unsigned pe = 0; pe < npes; ++pe) copy_of(balance, pe, stride)[e] = (float)b;
        }
        for (int s = 1; s < (int)kFinishExperts; s <<= 1) v += __shfl_xor(v, s);
        // the block that comes last adds up what each block found, in their order
        if (threadIdx.x == 0) {
            __hip_atomic_store(found + blockIdx.x, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            // (agent-scope stores and loads pass the L2s by: that the store has arrived is all that the ticket has to wait for,
            // and no L2 has to be written back for it)
            nvshmemi_amd_wait_vm();
            last = __hip_atomic_fetch_add((uint32_t *)(work + ticket), 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == gridDim.x;
        }
    }
    __syncthreads();
    if (!last || wave != 0) return;
    double v = 0.0;
    for (unsigned i = threadIdx.x; i < gridDim.x; i += kLanes) v += __hip_atomic_load(found + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int s = 1; s < kLanes; s <<= 1) v += __shfl_xor(v, s);
    if (threadIdx.x < npes) copy_of(loss, threadIdx.x, stride)[0] = (float)v;
}

// Bound by memory: logits read once, their gradient written once.  us for 65536 tokens of 256 fp32 logits (138 MB): 27.5 are 5.0 TB/s;
// with stores that stay in the caches 33.7.  Blocks of all PEs: 4096 (a step each) 32.5, 2048 29.3, 1024 27.5.
constexpr int kGradThreads = 256;
constexpr unsigned kGradBlocks = 1024;

template <typename T, int G, int V>
__global__ __launch_bounds__(kGradThreads) void route_grad_kernel(T *dlogits, const T *logits, const int32_t *expert,
                                                                   const float *dgate, const float *balance, const float *dloss,
                                                                   uint64_t stride, unsigned tokens, unsigned experts, unsigned topk,
                                                                   int normalise, float scale) {
    constexpr int kGroups = kGradThreads / G;
    __shared__ float chosen_part[kGroups][G * V];  // what only the chosen experts get, by expert
    const unsigned pe = blockIdx.z, sub = threadIdx.x % G, group = threadIdx.x / G;
    const T *my_logits = copy_of(logits, pe, stride);
    T *my_dlogits = copy_of(dlogits, pe, stride);
    const int32_t *my_expert = copy_of(expert, pe, stride);
    const float *my_dgate = copy_of(dgate, pe, stride);
    float *part = chosen_part[group];
#pragma unroll
    for (int u = 0; u < V; ++u) part[u * G + sub] = 0.0f;
    float b[V];
    const float up = balance ? copy_of(dloss, pe, stride)[0] : 0.0f;
#pragma unroll
    for (int u = 0; u < V; ++u) {
        const unsigned e = Slots<T, G, V>::expert(u, sub);
        b[u] = balance && e < experts ? up * copy_of(balance, pe, stride)[e] : 0.0f;
    }
    for (unsigned t0 = blockIdx.x * kGroups; t0 < tokens; t0 += gridDim.x * kGroups) {
        const bool here = t0 + group < tokens;
        const unsigned t = here ? t0 + group : t0;
        const T *row = my_logits + (uint64_t)t * experts;
        T x[V];
        Slots<T, G, V>::load(x, row, experts, sub);
        int32_t e = -1;
        float g = 0.0f, l = -__builtin_inff();
        if (sub < topk) {
            e = my_expert[(uint64_t)t * topk + sub];
            if ((unsigned)e < experts) {
                g = scale * my_dgate[(uint64_t)t * topk + sub];
                l = (float)row[e];
            }
        }
        const bool chosen = (unsigned)e < experts && l > -__builtin_inff();
        float p[V], m = -__builtin_inff();
#pragma unroll
        for (int u = 0; u < V; ++u) {
            p[u] = clean((float)x[u]);
            m = fmaxf(m, p[u]);
        }
        m = group_max<G>(m);
        float z = 0.0f, bp = 0.0f;
#pragma unroll
        for (int u = 0; u < V; ++u) {
            p[u] = p[u] > -__builtin_inff() ? exp_below(p[u], m) : -0.0f;  // (the sign says that it is masked)
            z += p[u];
            bp = __builtin_fmaf(p[u], b[u], bp);
        }
        z = group_sum<G>(z);
        const float r = z > 0.0f ? 1.0f / z : 0.0f;
        bp = group_sum<G>(bp) * r;
        if (!chosen) g = 0.0f;
        // the gates' own softmax is taken against the largest chosen logit, whatever else the row holds
        const float top = normalise ? group_max<G>(chosen ? l : -__builtin_inff()) : m;
        const float pk = chosen ? exp_below(l, top) * (normalise ? 1.0f : r) : 0.0f;
        const float s = group_sum<G>(pk), gs = group_sum<G>(pk * g);
        if (chosen) part[e] = normalise ? pk / s * (g - gs / s) : g;
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        T d[V];
#pragma unroll
        for (int u = 0; u < V; ++u) {
            const unsigned at = Slots<T, G, V>::expert(u, sub);
            const float c = part[at], pr = p[u] * r;
            const float v = normalise ? __builtin_fmaf(pr, b[u] - bp, c) : pr * (b[u] + c - (bp + gs));
            d[u] = (T)(__builtin_bit_cast(uint32_t, p[u]) != 0x80000000u ? v : 0.0f);  // (a NaN or infinity upstream leaves it at 0, too)
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (chosen) part[e] = 0.0f;
        if (here) Slots<T, G, V>::store(my_dlogits + (uint64_t)t * experts, d, experts, sub);
    }
}

// ---- the shuffle's tables ----
// A stable counting sort of the copies by expert: rows of a destination PE lie in the order (expert, source PE, token, k).  Nothing
// here is much data; what it costs is waiting, so a block asks for all that it needs from memory at once, at its start.
// Copies of a thread: one where a block has room for all of a PE's, two for fewer than kPlaceSpread of them, which then spread over
// more compute units, eight beyond, as each block adds up what the blocks in front of it counted.  us with 1 | 2 | 8, 8 PEs, 256 experts:
// 512 copies a PE 5.4 | 6.2 | 10.7, 65536 11.5 | 8.6 | 11.8, 131072 27.5 | 14.1 | 13.4, 262144 61.7 | 31.0 | 15.7 (and 4.9 for the counts in
// front of it, from two blocks on).
constexpr uint64_t kPlaceSpread = 1 << 17;
unsigned place_rounds(uint64_t copies) { return copies <= kSortThreads ? 1 : copies < kPlaceSpread ? 2 : 8; }
// The most blocks of a PE for as many copies or fewer: just below kPlaceSpread there are more than just above.
uint64_t place_most_blocks(uint64_t copies) {
    const uint64_t spread = ((copies < kPlaceSpread ? copies : kPlaceSpread) + 2 * kSortThreads - 1) / (2 * kSortThreads);
    const uint64_t rounds_8 = (copies + 8 * kSortThreads - 1) / (8 * kSortThreads);
    return spread > rounds_8 ? spread : rounds_8;
}

template <unsigned ROUNDS>
__global__ __launch_bounds__(kSortThreads) void place_count_kernel(uint32_t *hist, const int32_t *expert, uint64_t stride,
                                                                   unsigned copies, unsigned experts) {
    __shared__ uint32_t count[kMostExperts];
    const unsigned pe = blockIdx.z;
    const int32_t *mine = copy_of(expert, pe, stride);
    unsigned to[ROUNDS];
#pragma unroll
    for (unsigned i = 0; i < ROUNDS; ++i) {
        const unsigned c = blockIdx.x * (kSortThreads * ROUNDS) + i * kSortThreads + threadIdx.x;
        to[i] = c < copies ? (unsigned)mine[c] : ~0u;
    }
    count[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (unsigned i = 0; i < ROUNDS; ++i)
        if (to[i] < experts) atomicAdd(&count[to[i]], 1u);
    __syncthreads();
    if (threadIdx.x < experts) copy_of(hist, pe, stride)[(uint64_t)blockIdx.x * experts + threadIdx.x] = count[threadIdx.x];
}

template <unsigned ROUNDS>
__global__ __launch_bounds__(kSortThreads) void place_kernel(int32_t *dest_pe, int64_t *dest_row, uint64_t *expected,
                                                             int64_t *expert_row, const uint32_t *hist, const int32_t *expert,
                                                             const int64_t *counts, uint64_t stride, unsigned copies,
                                                             unsigned experts, unsigned npes, uint64_t cap, unsigned column_log) {
    extern __shared__ uint32_t lds[];  // stable_places' counts
    __shared__ uint32_t total[kMostExperts], before[kMostExperts], run[kMostExperts], scan[kMostExperts + 1], wave_sum[kSortWaves];
    __shared__ uint32_t arriving[NVSHMEMI_AMD_MAX_PES], from[kMostExperts];
    const unsigned pe = blockIdx.z, per_pe = experts / npes;
    const int32_t *mine = copy_of(expert, pe, stride);
    const unsigned c0 = blockIdx.x * (kSortThreads * ROUNDS) + threadIdx.x / kLanes * (ROUNDS * kLanes) + threadIdx.x % kLanes;
    uint32_t to[ROUNDS], place[ROUNDS];
#pragma unroll
    for (unsigned i = 0; i < ROUNDS; ++i) to[i] = c0 + i * kLanes < copies ? (uint32_t)mine[c0 + i * kLanes] : ~0u;
    // (own expert, source PE), what arrives from there: one pair a thread
    const unsigned own = threadIdx.x / npes, source = threadIdx.x % npes;
    const bool pair = blockIdx.x == 0 && own < per_pe;
    if (pair) from[threadIdx.x] = (uint32_t)copy_of(counts, source, stride)[pe * per_pe + own];
    // copies to every expert from all sources, and from the sources and blocks in front of this one; threads beyond the experts
    // share the sources and blocks with those below (column_log: log2 of the experts, rounded up)
    const unsigned e = threadIdx.x & ((1u << column_log) - 1), share = threadIdx.x >> column_log, shares = kSortThreads >> column_log;
    uint32_t all = 0, ahead = 0;
    if (e < experts) {
#pragma unroll 8
        for (unsigned src = share; src < npes; src += shares) {
            const uint32_t c = (uint32_t)copy_of(counts, src, stride)[e];
            ahead += src < pe ? c : 0;
            all += c;
        }
        const uint32_t *h = copy_of(hist, pe, stride) + e;
#pragma unroll 8
        for (unsigned b = share; b < blockIdx.x; b += shares) ahead += h[(uint64_t)b * experts];
    }
    total[threadIdx.x] = before[threadIdx.x] = 0;
    if (threadIdx.x < NVSHMEMI_AMD_MAX_PES) arriving[threadIdx.x] = 0;
    __syncthreads();
    if (e < experts) {
        atomicAdd(&total[e], all);
        atomicAdd(&before[e], ahead);
    }
    __syncthreads();
    const uint32_t in_front = scan_block(total[threadIdx.x], wave_sum);
    scan[threadIdx.x] = in_front;
    if (threadIdx.x == kSortThreads - 1) scan[kSortThreads] = in_front + total[threadIdx.x];
    __syncthreads();
    if (threadIdx.x < experts) run[threadIdx.x] = in_front - scan[threadIdx.x / per_pe * per_pe] + before[threadIdx.x];
    if (pair) {
        uint32_t at = scan[pe * per_pe + own] - scan[pe * per_pe];
        if (source == 0) copy_of(expert_row, pe, stride)[own] = at < cap ? at : (int64_t)cap;
        for (unsigned s = 0; s < source; ++s) at += from[own * npes + s];
        const uint32_t n = from[threadIdx.x];
        const uint64_t room = at < cap ? cap - at : 0;
        atomicAdd(&arriving[source], n < room ? n : (uint32_t)room);
        if (threadIdx.x == 0) {
            const uint32_t rows = scan[(pe + 1) * per_pe] - scan[pe * per_pe];
            copy_of(expert_row, pe, stride)[per_pe] = rows < cap ? rows : (int64_t)cap;
        }
    }
    __syncthreads();
    if (blockIdx.x == 0 && threadIdx.x < npes) copy_of(expected, pe, stride)[threadIdx.x] = arriving[threadIdx.x];
    stable_places<ROUNDS>(place, to, experts, run, lds);
    int32_t *out_pe = copy_of(dest_pe, pe, stride);
    int64_t *out_row = copy_of(dest_row, pe, stride);
#pragma unroll
    for (unsigned i = 0; i < ROUNDS; ++i) {
        const unsigned c = c0 + i * kLanes;
        if (c >= copies) continue;
        const bool kept = to[i] < experts && place[i] < cap;
        out_pe[c] = kept ? (int32_t)(to[i] / per_pe) : -1;
        out_row[c] = kept ? (int64_t)place[i] : -1;
    }
}

// ---- host ----
// (a lane adds up at most kMostSteps shares in fp32)
constexpr unsigned kFewBlocks = 512, kManyBlocks = 256, kMostSteps = 64;
// Blocks of a PE: enough of them over all PEs to fill the GPU, and no more, as the second kernel reads what each one leaves.
struct RouteShape {
    unsigned threads, per_block, blocks;
    uint64_t hist, psum, rows, ticket, bytes;
    RouteShape(size_t tokens, int experts, int npes, bool loss) {
        const unsigned group = experts > 256 ? kLanes : 16;
        // Without a loss, few tokens go to one block, whose counts are the PE's: a call of 8 x 64 tokens with its tables 11.3 us (router
        // 6.2), in four blocks and with the second kernel 12.4 (4.2 and 2.7).
        if (!loss && tokens * group <= kRouteMostThreads) {
            threads = tokens * group <= kLanes ? kLanes : (unsigned)((tokens * group + kLanes - 1) / kLanes * kLanes);
            per_block = threads / group;
            blocks = 1;
            hist = psum = rows = ticket = bytes = 0;
            return;
        }
        const uint64_t all = (uint64_t)tokens * npes;
        threads = all * group <= kFewBlocks * kRouteThreads ? kRouteThreads : kRouteMostThreads;
        const unsigned groups = threads / group, most = threads == kRouteThreads ? kFewBlocks : kManyBlocks;
        const uint64_t steps = (all + groups - 1) / groups, each = (steps + most - 1) / most;
        per_block = groups * (unsigned)(each < 1 ? 1 : each < kMostSteps ? each : kMostSteps);
        blocks = tokens ? div_up(tokens, per_block) : 1;
        lay_out(experts);
    }
    void lay_out(int experts) {
        const uint64_t table = ((uint64_t)blocks * experts * 4 + 63) / 64 * 64;
        hist = 0;
        psum = table;
        rows = 2 * table;
        ticket = rows + ((uint64_t)blocks * 8 + 63) / 64 * 64;
        bytes = ticket + 64 + (kMostExperts / kFinishExperts) * sizeof(double);
    }
    // What a program allocates: enough for these sizes and for all that are no larger, of which some have more blocks (8 PEs, 256 experts:
    // 64 a PE for 1024 tokens, 32 for 8192).  A block takes at least one step of the smaller one, and there are at most kFewBlocks of
    // them over all PEs, unless each takes all of its kMostSteps.
    static uint64_t space(uint64_t tokens, int experts, int npes) {
        const unsigned group = experts > 256 ? kLanes : 16;
        const uint64_t least = kRouteThreads / group, full = kRouteMostThreads / group * kMostSteps;
        const uint64_t one_step = (tokens + least - 1) / least, all_steps = (tokens + full - 1) / full, few = div_up(kFewBlocks, npes);
        const uint64_t most = few > all_steps ? few : all_steps;
        RouteShape shape(0, experts, npes, true);
        if (tokens) shape.blocks = (unsigned)(one_step < most ? one_step : most);
        shape.lay_out(experts);
        return shape.bytes;
    }
};

int check_routing(Runtime &rt, const char *what, size_t tokens, int experts, int topk) {
    NVSHMEM_AMD_REFUSE(experts < 1 || experts > kMostExperts, "%s: %d experts, outside [1, %d]", what, experts, kMostExperts);
    NVSHMEM_AMD_REFUSE(topk < 1 || topk > kMostTopk || topk > experts, "%s: top-%d of %d experts, outside [1, %d]", what, topk, experts,
                       kMostTopk < experts ? kMostTopk : experts);
    NVSHMEM_AMD_REFUSE(tokens > 0x7fffffffull / (size_t)rt.npes / (size_t)topk, "%s: %zu tokens x %d copies on %d PEs, at most 2^31 - 1 in all",
                       what, tokens, topk, rt.npes);
    return 0;
}

template <typename T, int G, int V>
void launch_route(const T *logits, const RouteArgs &a, unsigned npes, hipStream_t stream) {
    const dim3 grid(a.blocks, 1, npes);
    const size_t lds = ((size_t)a.experts * (1 + (a.loss ? a.threads / kLanes : 0)) + 1) * 4;
    if (a.topk <= 2) launch_kernel(route_kernel<T, G, V, 2>, grid, dim3(a.threads), lds, stream, logits, a);
    else if (a.topk <= 8) launch_kernel(route_kernel<T, G, V, 8>, grid, dim3(a.threads), lds, stream, logits, a);
    else launch_kernel(route_kernel<T, G, V, 16>, grid, dim3(a.threads), lds, stream, logits, a);
}

template <typename API>
int route_on_stream(int32_t *expert, float *gate, int64_t *counts, float *loss, float *balance, void *workspace, const API *logits,
                    size_t tokens, int experts, int topk, int normalise, float scale, hipStream_t stream) {
    typedef typename element<API>::type T;
    Runtime &rt = Runtime::get();
    std::lock_guard<std::recursive_mutex> lock(rt.mu);
    if (!ready(rt, "moe_route")) return NVSHMEMX_ERROR_INVALID_VALUE;
    if (int rc = check_routing(rt, "moe_route", tokens, experts, topk)) return rc;
    NVSHMEM_AMD_REFUSE(!loss != !balance, "moe_route: loss and balance come together");
    NVSHMEM_AMD_REFUSE(!(scale - scale == 0.0f), "moe_route: the scale must be finite");
    const RouteShape shape(tokens, experts, rt.npes, loss != nullptr);
    const uint64_t copies = (uint64_t)tokens * topk;
    Operands ops(rt, "moe_route");
    const T *in = (const T *)ops.in("logits", logits, (uint64_t)tokens * experts);
    RouteArgs a{};
    a.stride = rt.heap_size;
    a.expert = ops.out("expert", expert, copies);
    a.gate = ops.out("gate", gate, copies);
    int64_t *count = ops.out("counts", counts, (uint64_t)experts);
    float *l = loss ? ops.out("loss", loss, 1) : nullptr, *b = loss ? ops.out("balance", balance, (uint64_t)experts) : nullptr;
    a.work = ops.out("workspace", (char *)workspace, RouteShape(tokens, experts, rt.npes, true).bytes, 64);
    if (!ops.ok()) return NVSHMEMX_ERROR_INVALID_VALUE;
    const bool alone = shape.blocks == 1 && !loss;
    a.counts = alone ? count : nullptr;
    a.hist = shape.hist, a.psum = shape.psum, a.rows = shape.rows, a.ticket = shape.ticket;
    a.tokens = (unsigned)tokens, a.threads = shape.threads, a.per_block = shape.per_block, a.blocks = shape.blocks;
    a.experts = (unsigned)experts, a.topk = (unsigned)topk;
    a.normalise = normalise != 0, a.loss = loss != nullptr, a.scale = scale;
    if (experts <= 64) launch_route<T, 16, 4>(in, a, rt.npes, stream);
    else if (experts <= 256) launch_route<T, 16, 16>(in, a, rt.npes, stream);
    else launch_route<T, 64, 16>(in, a, rt.npes, stream);
    if (!alone)
        launch_kernel(route_finish_kernel, dim3(div_up(experts, kFinishExperts)), dim3(kFinishWaves * kLanes), 0, stream, count, l,
                      b, a.work, a.stride, a.hist, a.psum, a.rows, a.ticket, a.blocks, a.experts, (unsigned)rt.npes);
    return launched("moe_route");
}

template <typename API>
int route_grad_on_stream(API *dlogits, const API *logits, const int32_t *expert, const float *dgate, const float *balance,
                         const float *dloss, size_t tokens, int experts, int topk, int normalise, float scale, hipStream_t stream) {
    typedef typename element<API>::type T;
    Runtime &rt = Runtime::get();
    std::lock_guard<std::recursive_mutex> lock(rt.mu);
    if (!ready(rt, "moe_route_grad")) return NVSHMEMX_ERROR_INVALID_VALUE;
    if (int rc = check_routing(rt, "moe_route_grad", tokens, experts, topk)) return rc;
    NVSHMEM_AMD_REFUSE(!dloss != !balance, "moe_route_grad: dloss and balance come together");
    NVSHMEM_AMD_REFUSE(!(scale - scale == 0.0f), "moe_route_grad: the scale must be finite");
    const uint64_t copies = (uint64_t)tokens * topk, values = (uint64_t)tokens * experts;
    Operands ops(rt, "moe_route_grad");
    const T *in = (const T *)ops.in("logits", logits, values);
    const int32_t *to = ops.in("expert", expert, copies);
    const float *dg = ops.in("dgate", dgate, copies);
    const float *b = balance ? ops.in("balance", balance, (uint64_t)experts) : nullptr;
    const float *dl = balance ? ops.in("dloss", dloss, 1) : nullptr;
    T *out = (T *)ops.out("dlogits", dlogits, values);
    if (!ops.ok()) return NVSHMEMX_ERROR_INVALID_VALUE;
    if (tokens == 0) return 0;
#define NVSHMEM_AMD_LAUNCH_GRAD(G, V)                                                                                             \
    {                                                                                                                             \
        const unsigned steps = div_up(tokens, kGradThreads / G), most = kGradBlocks / (unsigned)rt.npes;                                \
        launch_kernel(route_grad_kernel<T, G, V>, dim3(steps < most ? steps : most, 1, rt.npes), dim3(kGradThreads), 0, stream,  \
                      out, in, to, dg, b, dl, rt.heap_size, (unsigned)tokens, (unsigned)experts, (unsigned)topk, normalise != 0, scale); \
    }
    if (experts <= 64) NVSHMEM_AMD_LAUNCH_GRAD(16, 4)
    else if (experts <= 256) NVSHMEM_AMD_LAUNCH_GRAD(16, 16)
    else NVSHMEM_AMD_LAUNCH_GRAD(64, 16)
#undef NVSHMEM_AMD_LAUNCH_GRAD
    return launched("moe_route_grad");
}

int place_on_stream(int32_t *dest_pe, int64_t *dest_row, uint64_t *expected, int64_t *expert_row, void *workspace,
                    const int32_t *expert, const int64_t *counts, size_t tokens, int topk, int experts, size_t recv_cap_rows,
                    hipStream_t stream) {
    Runtime &rt = Runtime::get();
    std::lock_guard<std::recursive_mutex> lock(rt.mu);
    if (!ready(rt, "moe_place")) return NVSHMEMX_ERROR_INVALID_VALUE;
    if (int rc = check_routing(rt, "moe_place", tokens, experts, topk)) return rc;
    NVSHMEM_AMD_REFUSE(experts % rt.npes, "moe_place: %d experts on %d PEs, not the same number on each", experts, rt.npes);
    const uint64_t copies = (uint64_t)tokens * topk;
    const unsigned rounds = place_rounds(copies), blocks = copies ? div_up(copies, kSortThreads * rounds) : 1;
    Operands ops(rt, "moe_place");
    const int32_t *in = ops.in("expert", expert, copies);
    const int64_t *count = ops.in("counts", counts, (uint64_t)experts);
    int32_t *to = ops.out("dest_pe", dest_pe, copies);
    int64_t *row = ops.out("dest_row", dest_row, copies);
    uint64_t *exp = ops.out("expected", expected, (uint64_t)rt.npes);
    int64_t *first = ops.out("expert_row", expert_row, (uint64_t)(experts / rt.npes + 1));
    uint32_t *hist = blocks > 1 ? ops.out("workspace", (uint32_t *)workspace, (uint64_t)blocks * experts, 64) : nullptr;
    if (!ops.ok()) return NVSHMEMX_ERROR_INVALID_VALUE;
    unsigned column_log = 0;
    while ((1u << column_log) < (unsigned)experts) ++column_log;
#define NVSHMEM_AMD_LAUNCH_PLACE(ROUNDS)                                                                                               \
    {                                                                                                                                \
        if (blocks > 1)                                                                                                              \
            launch_kernel(place_count_kernel<ROUNDS>, dim3(blocks, 1, rt.npes), dim3(kSortThreads), 0, stream, hist, in,             \
                          rt.heap_size, (unsigned)copies, (unsigned)experts);                                                        \
        launch_kernel(place_kernel<ROUNDS>, dim3(blocks, 1, rt.npes), dim3(kSortThreads), (size_t)kSortWaves * experts * 4, stream, \
                      to, row, exp, first, hist, in, count, rt.heap_size, (unsigned)copies, (unsigned)experts, (unsigned)rt.npes,    \
                      (uint64_t)recv_cap_rows, column_log);                                                                          \
    }
    if (rounds == 1) NVSHMEM_AMD_LAUNCH_PLACE(1)
    else if (rounds == 2) NVSHMEM_AMD_LAUNCH_PLACE(2)
    else NVSHMEM_AMD_LAUNCH_PLACE(8)
#undef NVSHMEM_AMD_LAUNCH_PLACE
    return launched("moe_place");
}

}  // namespace
}  // namespace tokens
}  // namespace nvshmem_amd

using namespace nvshmem_amd;

extern "C" {

#define NVSHMEM_AMD_ROUTE(NAME, TYPE)                                                                                              \
    int nvshmemx_amd_##NAME##_moe_route_on_stream(int32_t *expert, float *gate, int64_t *counts, float *loss, float *balance,      \
                                                  void *workspace, const TYPE *logits, size_t tokens, int experts, int topk,       \
                                                  int normalise, float scale, nvshmemx_stream_t stream) {                          \
        return tokens::route_on_stream(expert, gate, counts, loss, balance, workspace, logits, tokens, experts, topk, normalise,   \
                                       scale, (hipStream_t)stream);                                                                \
    }                                                                                                                              \
    int nvshmemx_amd_##NAME##_moe_route_grad_on_stream(TYPE *dlogits, const TYPE *logits, const int32_t *expert,                   \
                                                       const float *dgate, const float *balance, const float *dloss,               \
                                                       size_t tokens, int experts, int topk, int normalise, float scale,           \
                                                       nvshmemx_stream_t stream) {                                                 \
        return tokens::route_grad_on_stream(dlogits, logits, expert, dgate, balance, dloss, tokens, experts, topk, normalise,      \
                                            scale, (hipStream_t)stream);                                                           \
    }
NVSHMEMI_AMD_REPT_FOR_TOKEN_TYPES(NVSHMEM_AMD_ROUTE)
#undef NVSHMEM_AMD_ROUTE

size_t nvshmemx_amd_moe_route_workspace(size_t tokens, int experts) {
    const int npes = Runtime::get().npes;
    if (npes < 1 || experts < 1 || experts > tokens::kMostExperts) return 0;
    return tokens::RouteShape::space(tokens, experts, npes);  // (what a call without a loss takes is less)
}

int nvshmemx_amd_moe_place_on_stream(int32_t *dest_pe, int64_t *dest_row, uint64_t *expected, int64_t *expert_row, void *workspace,
                                     const int32_t *expert, const int64_t *counts, size_t tokens, int topk, int experts,
                                     size_t recv_cap_rows, nvshmemx_stream_t stream) {
    return tokens::place_on_stream(dest_pe, dest_row, expected, expert_row, workspace, expert, counts, tokens, topk, experts,
                                   recv_cap_rows, (hipStream_t)stream);
}
size_t nvshmemx_amd_moe_place_workspace(size_t tokens, int topk, int experts) {
    if (Runtime::get().npes < 1 || topk < 1 || experts < 1) return 0;
    return tokens::place_most_blocks((uint64_t)tokens * topk) * (uint64_t)experts * sizeof(uint32_t);
}

}  // extern "C"
