// The experts' gated feed-forward block with weights of 4 bits: (q - 8) * scale, one scale for each `group` consecutive k of a row.
//
//   pre = [gate | up] = x W_in^T      h = gate * sigmoid(gate) * up      out = h W_out^T
//
// The matrix cores get x and the whole numbers q exactly; what a group adds up to is multiplied with its scale in fp32.
#include "expert_few.hpp"

namespace nvshmem_amd {
namespace tokens {
namespace {

template <typename T>
struct W4Args {
    ExpertArgs<T> e;
    const unsigned char *w_in, *w_out;
    const T *s_in, *s_out;
    unsigned group;
};

// ---- experts of few rows ----

// The two halves of a word that an element of x and a weight become for the matrix cores.  A weight is 16 + q, whose bits are those of
// 16 with q in the mantissa; what that is too much, 24 times the sum of x, goes into the sums first as a product with -24.
template <typename T>
struct Nibble;
template <>
struct Nibble<__bf16> {
    static constexpr unsigned kSixteen = 0x41804180u, kMinus24 = 0xC1C0C1C0u, kShift = 3;
    typedef __bf16 type;
};
template <>
struct Nibble<_Float16> {
    static constexpr unsigned kSixteen = 0x4C004C00u, kMinus24 = 0xCE00CE00u, kShift = 6;
    typedef _Float16 type;
};
template <>
struct Nibble<float> : Nibble<__bf16> {};  // an fp32 number is the sum of three bf16 ones, of 8 bits of its mantissa each

// Eight weights, k in the order 0 4 1 5 2 6 3 7.
template <typename T>
__device__ __forceinline__ v4u eight_weights(unsigned q) {
    constexpr unsigned s = Nibble<T>::kShift, mask = 0x000F000Fu << s;
    v4u v;
#pragma unroll
    for (unsigned j = 0; j < 4; ++j) {
        const unsigned at = j * 4;
        v[j] = ((at <= s ? q << (s - at) : q >> (at - s)) & mask) | Nibble<T>::kSixteen;
    }
    return v;
}
// Eight elements of x in that order.
__device__ __forceinline__ v4u reorder_eight(v4u x) {
    return v4u{__builtin_amdgcn_perm(x[2], x[0], 0x05040100u), __builtin_amdgcn_perm(x[2], x[0], 0x07060302u),
               __builtin_amdgcn_perm(x[3], x[1], 0x05040100u), __builtin_amdgcn_perm(x[3], x[1], 0x07060302u)};
}
// Eight fp32 numbers in that order as three bf16 parts: the highest 8 bits of the mantissa, the next, the last.  Each difference is exact.
// (An infinity or a NaN is its own first part and leaves 0.)
__device__ __forceinline__ void split_eight(v4f lo, v4f hi, v4u (&part)[3]) {
    unsigned bits[3][8];
#pragma unroll
    for (unsigned i = 0; i < 8; ++i) {
        float v = i < 4 ? lo[i] : hi[i - 4];
        const bool finite = (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u;
#pragma unroll
        for (unsigned p = 0; p < 3; ++p) {
            // (a NaN stays one: its highest mantissa bit is set)
            bits[p][i] = p == 0 && !finite && v != v ? 0x7fc00000u : __float_as_uint(v) & 0xffff0000u;
            v = finite ? v - __uint_as_float(bits[p][i]) : 0.0f;
        }
    }
#pragma unroll
    for (unsigned p = 0; p < 3; ++p)
#pragma unroll
        for (unsigned j = 0; j < 4; ++j) part[p][j] = __builtin_amdgcn_perm(bits[p][j + 4], bits[p][j], 0x07060302u);
}

template <unsigned N>
struct words;
template <>
struct words<1> {
    typedef unsigned type;
};
template <>
struct words<2> {
    typedef v2u type;
};
template <>
struct words<4> {
    typedef v4u type;
};

// A wavefront takes 64 rows and 32 * WORDS k at a time, all of one group: lane (r, g) has of each of four groups of 16 rows 4 * WORDS bytes,
// 8 * WORDS consecutive k of row r.  WORDS is 4 where the group is a multiple of 128, else 2 or 1.
template <typename T, unsigned WORDS>
struct FourBitWeights {
    static constexpr unsigned kStepK = 32 * WORDS, kParts = sizeof(T) == 4 ? 3 : 1;
    typedef typename words<WORDS>::type raw;
    typedef raw raw_unaligned __attribute__((aligned(1)));
    typedef typename Nibble<T>::type M;
    const unsigned char *base[2];
    const T *scale[2];
    unsigned row_bytes, row_scales, k_all, group;
    unsigned row[4];

    raw w[4];
    float s[4];
    __device__ __forceinline__ void load(unsigned k, unsigned lane, bool whole) {
        const unsigned at = k + lane / 16 * 8 * WORDS;
#pragma unroll
        for (unsigned ni = 0; ni < 4; ++ni) {
            const unsigned char *p = base[ni / 2] + (uint64_t)row[ni] * row_bytes + at / 2;
            if (whole) {
                w[ni] = __builtin_nontemporal_load((const raw_unaligned *)p);
            } else {
                unsigned v[WORDS] = {};
                const unsigned n = at < k_all ? (k_all - at + 1) / 2 : 0;
#pragma unroll
                for (unsigned i = 0; i < 4 * WORDS; ++i)
                    if (i < n) v[i / 4] |= (unsigned)p[i] << i % 4 * 8;
                __builtin_memcpy(&w[ni], v, sizeof v);
            }
            s[ni] = (float)scale[ni / 2][(uint64_t)row[ni] * row_scales + k / group];
        }
    }
    template <int MT>
    __device__ __forceinline__ void multiply(const T *const (&x)[MT], unsigned k, unsigned lane, bool whole, v4f (&acc)[MT][4]) const {
        const unsigned at = k + lane / 16 * 8 * WORDS;
        v4u a[MT][WORDS][kParts];
        v4f sum[MT] = {};
        const unsigned c = Nibble<T>::kMinus24;
#pragma unroll
        for (int mi = 0; mi < MT; ++mi)
#pragma unroll
            for (unsigned j = 0; j < WORDS; ++j) {
                const T *p = x[mi] + at + j * 8;
                const unsigned from = at + j * 8, n = whole ? 8 : from < k_all ? (k_all - from < 8 ? k_all - from : 8) : 0;
                if constexpr (sizeof(T) == 2) {
                    a[mi][j][0] = reorder_eight(__builtin_bit_cast(v4u, whole ? chunk_load(p) : chunk_load_part(p, n)));
                } else {
                    const v4f lo = whole ? chunk_load(p) : chunk_load_part(p, n < 4 ? n : 4);
                    const v4f hi = whole ? chunk_load(p + 4) : chunk_load_part(p + 4, n < 4 ? 0 : n - 4);
                    split_eight(lo, hi, a[mi][j]);
                }
#pragma unroll
                for (unsigned q = 0; q < kParts; ++q) sum[mi] = Mma<M>::step(a[mi][j][q], v4u{c, c, c, c}, sum[mi]);
            }
#pragma unroll
        for (unsigned ni = 0; ni < 4; ++ni) {
            v4f d[MT];
#pragma unroll
            for (int mi = 0; mi < MT; ++mi) d[mi] = sum[mi];
#pragma unroll
            for (unsigned j = 0; j < WORDS; ++j) {
                unsigned word;
                if constexpr (WORDS == 1) word = w[ni];
                else word = w[ni][j];
                const v4u b = eight_weights<T>(word);
#pragma unroll
                for (int mi = 0; mi < MT; ++mi)
#pragma unroll
                    for (unsigned q = 0; q < kParts; ++q) d[mi] = Mma<M>::step(a[mi][j][q], b, d[mi]);
            }
#pragma unroll
            for (int mi = 0; mi < MT; ++mi)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[mi][ni][i] = __builtin_fmaf(s[ni], d[mi][i], acc[mi][ni][i]);
        }
    }
};

template <typename T, int OP, unsigned WORDS>
__global__ __launch_bounds__(kFewThreads) void expert_few_w4_kernel(const W4Args<T> args) {
    typedef FourBitWeights<T, WORDS> W;
    few_rows_block<W, T, OP>(args.e, [&](W &w, unsigned pe, unsigned e, unsigned n0) {
        const ExpertArgs<T> &a = args.e;
        const unsigned n_all = OP == kIn ? a.hidden : a.dim, k_all = OP == kIn ? a.dim : a.hidden;
        const uint64_t before = (uint64_t)e * (OP == kIn ? 2 * n_all : n_all) + n0;
        w.k_all = k_all, w.group = args.group, w.row_bytes = (k_all + 1) / 2, w.row_scales = (k_all + args.group - 1) / args.group;
        w.base[0] = copy_of(OP == kIn ? args.w_in : args.w_out, pe, a.stride) + before * w.row_bytes;
        w.scale[0] = copy_of(OP == kIn ? args.s_in : args.s_out, pe, a.stride) + before * w.row_scales;
        w.base[1] = OP == kIn ? w.base[0] + (uint64_t)n_all * w.row_bytes : w.base[0];
        w.scale[1] = OP == kIn ? w.scale[0] + (uint64_t)n_all * w.row_scales : w.scale[0];
        for (unsigned ni = 0; ni < 4; ++ni) w.row[ni] = few_rows_row<OP>(ni, threadIdx.x % kLanes, n_all - n0);
    });
}

// ---- experts of more rows: tiles ----

// B's way into LDS: 256 rows of packed weights, half a step's k of a row for each thread, as q - 8 in T (exact) where TileSide<T, 256, false>
// reads them.  Their scales go beside them, one for each half of each row.
template <typename T>
struct FourBitSide {
    static constexpr unsigned kStepK = kStepBytes / sizeof(T), kHalfK = kStepK / 2, kWords = kHalfK / 8;
    typedef typename words<kWords>::type raw;
    typedef raw raw_unaligned __attribute__((aligned(1)));
    const unsigned char *row;  // this thread's; where it has none, a row that exists
    const T *scale;
    unsigned k_all, group;
    raw held;
    float held_scale;

    __device__ __forceinline__ void fetch(uint64_t k) {
        const unsigned at = (unsigned)k + threadIdx.x % 2 * kHalfK;
        const unsigned char *p = row + at / 2;
        const unsigned n = at < k_all ? (k_all - at + 1) / 2 : 0;
        if (n >= kHalfK / 2) {
            held = *(const raw_unaligned *)p;
        } else {
            unsigned v[kWords] = {};
#pragma unroll
            for (unsigned i = 0; i < 4 * kWords; ++i)
                if (i < n) v[i / 4] |= (unsigned)p[i] << i % 4 * 8;
            __builtin_memcpy(&held, v, sizeof v);
        }
        held_scale = n ? (float)scale[at / group] : 0.0f;
    }
    __device__ __forceinline__ void land(NVSHMEM_AMD_LDS char *lds, float *scales) const {
        const unsigned r = threadIdx.x / 2, half = threadIdx.x % 2;
        scales[half * kTileN + r] = held_scale;
#pragma unroll
        for (unsigned j = 0; j < 4; ++j) {
            typename Chunk<T>::vec v;
#pragma unroll
            for (unsigned i = 0; i < (unsigned)Chunk<T>::N; ++i) {
                const unsigned at = j * Chunk<T>::N + i;
                v[i] = (T)((float)(held[at / 8] >> at % 8 * 4 & 15) - 8.0f);
            }
            *(NVSHMEM_AMD_LDS v4u *)(lds + r * kStepBytes + (((half * 4 + j) ^ (r & 7)) * 16)) = __builtin_bit_cast(v4u, v);
        }
    }
};

constexpr unsigned kW4TileRows = 128;

template <typename T, int OP, bool DMA>
__global__ __launch_bounds__(kTileThreads, 2) void expert_tile_w4_kernel(const W4Args<T> args4) {
    constexpr unsigned BM = kW4TileRows, kMi = BM / 32, kNi = 4;
    typedef TileSide<T, BM, false, DMA> A;
    typedef TileSide<T, kTileN, false, true> B;  // (its layout in LDS)
    typedef FourBitSide<T> Q;
    constexpr unsigned kStepK = A::kStepK;
    __shared__ __attribute__((aligned(1024))) char lds_a[2][A::kBytes];
    __shared__ __attribute__((aligned(1024))) char lds_b[2][B::kBytes];
    __shared__ __attribute__((aligned(16))) float lds_s[2][2 * kTileN];
    const ExpertArgs<T> &args = args4.e;
    const unsigned pe = blockIdx.z, wave = wave_of_block(), lane = threadIdx.x % kLanes;
    const int64_t *expert_row = copy_of(args.expert_row, pe, args.stride);
    const unsigned n_all = OP == kIn ? args.hidden : args.dim, k_all = OP == kIn ? args.dim : args.hidden;
    const unsigned n_tile = OP == kIn ? kTileN / 2 : kTileN, wide = (n_all + n_tile - 1) / n_tile;
    const TileList list = {expert_row, args.cap, args.experts, BM, wide, args.more_than};
    const uint64_t total = list.total(), chunk = (total + 7) / 8;
    for (uint64_t i = blockIdx.x / 8; i < chunk; i += gridDim.x / 8) {
        uint64_t t = blockIdx.x % 8 * chunk + i;
        if (t >= total) return;
        const unsigned e = list.find(t);
        uint64_t first, rows;
        expert_range(expert_row, e, args.cap, first, rows);
        first = scalar64(first), rows = scalar64(rows);
        unsigned tm, tn;
        tile_place((unsigned)t, (unsigned)((rows + BM - 1) / BM), wide, tm, tn);
        const uint64_t m0 = (uint64_t)tm * BM;
        const unsigned n0 = tn * n_tile, m_here = rows - m0 < BM ? (unsigned)(rows - m0) : BM;
        const unsigned n_here = n_all - n0 < n_tile ? n_all - n0 : n_tile;
        const T *a = copy_of(OP == kIn ? args.rows : (const T *)args.h, pe, args.stride) + (first + m0) * k_all;
        A side_a;
        side_a.begin(wave, lane, m_here, k_all, [](unsigned r) { return r; });
        Q side_b;
        {
            const unsigned r = threadIdx.x / 2, at = OP == kIn ? r / 64 * 32 + r % 32 : r;
            const uint64_t n = (uint64_t)e * (OP == kIn ? 2 : 1) * n_all + (OP == kIn && r % 64 >= 32 ? n_all : 0) + n0 + (at < n_here ? at : n_here - 1);
            side_b.k_all = k_all, side_b.group = args4.group;
            side_b.row = copy_of(OP == kIn ? args4.w_in : args4.w_out, pe, args.stride) + n * ((k_all + 1) / 2);
            side_b.scale = copy_of(OP == kIn ? args4.s_in : args4.s_out, pe, args.stride) + n * ((k_all + args4.group - 1) / args4.group);
        }
        const auto fetch = [&](unsigned buffer, unsigned k) {
            const unsigned left = k_all - k < kStepK ? k_all - k : kStepK;
            side_a.fetch((NVSHMEM_AMD_LDS char *)lds_a[buffer], wave, left, [&](unsigned) { return a + k; });
            side_b.fetch(k);
        };
        v4f acc[kMi][kNi] = {};
        const unsigned wm = wave / 4, wn = wave % 4;
        fetch(0, 0);
        unsigned buffer = 0;
        const bool halves = args4.group % kStepK != 0;  // (then the halves of a step may be of two groups)
        for (unsigned k = 0; k < k_all; k += kStepK, buffer ^= 1) {
            side_a.land((NVSHMEM_AMD_LDS char *)lds_a[buffer], wave, lane);
            side_b.land((NVSHMEM_AMD_LDS char *)lds_b[buffer], lds_s[buffer]);
            asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
            __syncthreads();
            if (k + kStepK < k_all) fetch(buffer ^ 1, k + kStepK);
            v4u fa[2][kMi], fb[2][kNi];
#pragma unroll
            for (unsigned s = 0; s < 2; ++s) {
#pragma unroll
                for (unsigned ni = 0; ni < kNi; ++ni) fb[s][ni] = B::read((NVSHMEM_AMD_LDS const char *)lds_b[buffer], wn * 4 + ni, s, lane);
#pragma unroll
                for (unsigned mi = 0; mi < kMi; ++mi) fa[s][mi] = A::read((NVSHMEM_AMD_LDS const char *)lds_a[buffer], wm * kMi + mi, s, lane);
            }
#pragma unroll
            for (unsigned ni = 0; ni < kNi; ++ni) {
                const float *s = &lds_s[buffer][wn * 64 + ni * 16 + lane / 16 * 4];
                const v4f s0 = *(const v4f *)s, s1 = *(const v4f *)(s + kTileN);
#pragma unroll
                for (unsigned mi = 0; mi < kMi; ++mi) {
                    v4f d = Mma<T>::step(fb[0][ni], fa[0][mi], v4f{});
                    if (halves) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[mi][ni][j] = __builtin_fmaf(s0[j], d[j], acc[mi][ni][j]);
                        d = v4f{};
                    }
                    d = Mma<T>::step(fb[1][ni], fa[1][mi], d);
                    const v4f scale = halves ? s1 : s0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[mi][ni][j] = __builtin_fmaf(scale[j], d[j], acc[mi][ni][j]);
                }
            }
        }
        __syncthreads();
        const unsigned r = lane % 16, g = lane / 16;
#pragma unroll
        for (unsigned mi = 0; mi < kMi; ++mi) {
            const unsigned m = (wm * kMi + mi) * 16 + r;
            if (m >= m_here) continue;
            const uint64_t row = first + m0 + m;
            if (OP == kIn) {
#pragma unroll
                for (unsigned ni = 0; ni < 2; ++ni) {
                    const unsigned c = wn * 32 + ni * 16 + g * 4;
                    if (c >= n_here) continue;
                    v4f h;
#pragma unroll
                    for (int j = 0; j < 4; ++j) h[j] = acc[mi][ni][j] * sigmoid(acc[mi][ni][j]) * acc[mi][ni + 2][j];
                    store_four(copy_of(args.h, pe, args.stride) + row * args.hidden + n0 + c, h, n_here - c);
                }
            } else {
#pragma unroll
                for (unsigned ni = 0; ni < kNi; ++ni) {
                    const unsigned c = wn * 64 + ni * 16 + g * 4;
                    if (c < n_here) store_four(copy_of(args.out, pe, args.stride) + row * args.dim + n0 + c, acc[mi][ni], n_here - c);
                }
            }
        }
    }
}

template <typename T, int OP>
void launch_w4(const W4Args<T> &args, bool whole, int npes, hipStream_t stream) {
    const dim3 few = few_rows_grid<OP>(args.e, npes);
    if (args.group % 128 == 0) launch_kernel((expert_few_w4_kernel<T, OP, 4>), few, dim3(kFewThreads), 0, stream, args);
    else if (args.group % 64 == 0) launch_kernel((expert_few_w4_kernel<T, OP, 2>), few, dim3(kFewThreads), 0, stream, args);
    else launch_kernel((expert_few_w4_kernel<T, OP, 1>), few, dim3(kFewThreads), 0, stream, args);
    if (args.e.cap <= kFewRows) return;
    const uint64_t wide = div_up(OP == kIn ? args.e.hidden : args.e.dim, OP == kIn ? kTileN / 2 : kTileN);
    const uint64_t tiles = (args.e.cap / kW4TileRows + (args.e.experts < args.e.cap ? args.e.experts : args.e.cap)) * wide;
    if (whole) launch_kernel((expert_tile_w4_kernel<T, OP, true>), tile_grid(tiles, npes), dim3(kTileThreads), 0, stream, args);
    else launch_kernel((expert_tile_w4_kernel<T, OP, false>), tile_grid(tiles, npes), dim3(kTileThreads), 0, stream, args);
}

template <typename API>
int experts_w4_on_stream(API *out, void *workspace, const API *rows, const uint8_t *w_in, const API *w_in_scale, const uint8_t *w_out,
                         const API *w_out_scale, const int64_t *expert_row, size_t recv_cap_rows, int experts, size_t dim,
                         size_t hidden, int group, hipStream_t stream) {
    typedef typename element<API>::type T;
    Runtime &rt = Runtime::get();
    std::lock_guard<std::recursive_mutex> lock(rt.mu);
    if (!ready(rt, "moe_experts_w4")) return NVSHMEMX_ERROR_INVALID_VALUE;
    if (int rc = check_expert_sizes(rt, "moe_experts_w4", experts, dim, hidden)) return rc;
    NVSHMEM_AMD_REFUSE(group < 32 || group % 32 || group > 65536, "moe_experts_w4: groups of %d, not a multiple of 32 up to 65536", group);
    const uint64_t cap = recv_cap_rows, mine = (uint64_t)(experts / rt.npes);
    NVSHMEM_AMD_REFUSE(cap > rt.heap_size / (dim * sizeof(T)) || cap > rt.heap_size / (hidden * sizeof(T)),
                       "moe_experts_w4: %zu rows leave the PE's heap slice", recv_cap_rows);
    Operands ops(rt, "moe_experts_w4");
    W4Args<T> args = {};
    ExpertArgs<T> &a = args.e;
    a.rows = (const T *)ops.in("rows", rows, cap * dim);
    args.w_in = ops.in("w_in", w_in, mine * 2 * hidden * ((dim + 1) / 2));
    args.s_in = (const T *)ops.in("w_in_scale", w_in_scale, mine * 2 * hidden * ((dim + group - 1) / group));
    args.w_out = ops.in("w_out", w_out, mine * dim * ((hidden + 1) / 2));
    args.s_out = (const T *)ops.in("w_out_scale", w_out_scale, mine * dim * ((hidden + group - 1) / group));
    a.expert_row = ops.in("expert_row", expert_row, mine + 1);
    a.out = (T *)ops.out("out", out, cap * dim);
    a.h = (T *)ops.out("workspace", (char *)workspace, cap * hidden * sizeof(T), 64);
    if (!ops.ok()) return NVSHMEMX_ERROR_INVALID_VALUE;
    if (cap == 0) return 0;
    args.group = (unsigned)group;
    a.stride = rt.heap_size, a.cap = cap, a.experts = (unsigned)mine, a.dim = (unsigned)dim, a.hidden = (unsigned)hidden;
    a.more_than = kFewRows;
    const bool whole = dim * sizeof(T) % 16 == 0 && hidden * sizeof(T) % 16 == 0 && aligned16(a.rows);
    launch_w4<T, kIn>(args, whole, rt.npes, stream);
    launch_w4<T, kOut>(args, whole, rt.npes, stream);
    return launched("moe_experts_w4");
}

}  // namespace
}  // namespace tokens
}  // namespace nvshmem_amd

using namespace nvshmem_amd;

extern "C" {

#define NVSHMEM_AMD_EXPERTS_W4(NAME, TYPE)                                                                                         \
    int nvshmemx_amd_##NAME##_moe_experts_w4_on_stream(TYPE *out, void *workspace, const TYPE *rows, const uint8_t *w_in,          \
                                                       const TYPE *w_in_scale, const uint8_t *w_out, const TYPE *w_out_scale,      \
                                                       const int64_t *expert_row, size_t recv_cap_rows, int experts, size_t dim,   \
                                                       size_t hidden, int group, nvshmemx_stream_t stream) {                       \
        return tokens::experts_w4_on_stream(out, workspace, rows, w_in, w_in_scale, w_out, w_out_scale, expert_row, recv_cap_rows, \
                                            experts, dim, hidden, group, (hipStream_t)stream);                                     \
    }
NVSHMEMI_AMD_REPT_FOR_TOKEN_TYPES(NVSHMEM_AMD_EXPERTS_W4)
#undef NVSHMEM_AMD_EXPERTS_W4

}  // extern "C"
