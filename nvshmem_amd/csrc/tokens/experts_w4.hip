// The experts' gated feed-forward block with weights of 4 bits: (q - 8) * scale, one scale for each `group` consecutive k of a row.
//
//   pre = [gate | up] = x W_in^T      h = gate * sigmoid(gate) * up      out = h W_out^T
//
// The matrix cores get x and the whole numbers q exactly; what a group adds up to is multiplied with its scale in fp32.
#include "expert_tiles.hpp"

namespace nvshmem_amd {
namespace tokens {
namespace {

template <typename T>
struct W4Args {
    ExpertArgs<T> e;
    const unsigned char *w_in, *w_out;
    const T *s_in, *s_out;
    unsigned group, per_group;  // per_group: 2^31 / (group / 32), rounded up: k / group is k / 32 times that, over 2^31 (k is at most 2^16)
};

// ---- experts of few rows ----

// What x and a weight become for the matrix cores.  Of bfloat16 elements a weight is 128 + q, whose bits are those of 128 with q in the
// mantissa: one operation for two weights.  The 136 that this is too much, times the sum of x, goes into the sums first, as a product with
// too_much().  What the sums, in fp32, lose by it is some 2^-17 of the sum of |x|, which x's own rounding to 2^-8 has long lost; 2^-16 of the result
// where a row's elements are of one sign.  For a half, which is rounded to 2^-11 and whose bits would need 1024 in 128's place, that does not
// hold: 1024 + q (64 + q of the next four bits) loses the 1032 (72) by one more operation for two weights, exactly.  An fp32 element is the sum of
// three bf16 ones, of 8 bits of its mantissa each, and weights are (q - 8) / 16: nothing of it above 2^-133, bf16's least number, is lost in front
// of the sum.
// us of 64 tokens on each of 8 PEs, halves, 256 experts of 7168 x 2048, groups of 64, by products with the 1032 and 72 and now: 1618 / 1641.
template <typename T>
struct Nibble;
template <>
struct Nibble<__bf16> {
    typedef __bf16 type;
    static __device__ __forceinline__ v4u too_much() { return v4u{0xC308C308u, 0xC308C308u, 0xC308C308u, 0xC308C308u}; }
};
template <>
struct Nibble<_Float16> {
    typedef _Float16 type;
};
template <>
struct Nibble<float> : Nibble<__bf16> {};

// Eight weights, k in the order 0 4 1 5 2 6 3 7.  SIXTEENTHS: (q - 8) / 16, as the tiles take them, so that sums of 128 elements under 2^121 stay in fp32.
template <typename T, bool SIXTEENTHS>
__device__ __forceinline__ v4u eight_weights(unsigned q) {
    v4u v;
    if (SIXTEENTHS) {
        const unsigned even = q ^ 0x88888888u, odd = even >> 4;
#pragma unroll
        for (unsigned j = 0; j < 4; ++j) {
            const unsigned from = j % 2 ? odd : even;
            const float a = __builtin_amdgcn_cvt_off_f32_i4((int)(from >> j / 2 * 8)), b = __builtin_amdgcn_cvt_off_f32_i4((int)(from >> (j / 2 * 8 + 16)));
            v[j] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);  // (few bits: bf16 is their upper half)
        }
        return v;
    }
    // (constants that the compiler does not see through stay in registers, where an "and" and an "or" are one instruction)
    unsigned low = 0x000F000Fu, next = 0x00F000F0u, base = __is_same(T, _Float16) ? 0x64006400u : 0x43004300u, base_next = 0x54005400u;
    asm("" : "+v"(base), "+v"(base_next));
    if (__is_same(T, _Float16)) {
        typedef _Float16 two __attribute__((ext_vector_type(2)));
        const unsigned upper = q >> 8;
        const auto less = [](unsigned w, float by) { return __builtin_bit_cast(unsigned, __builtin_bit_cast(two, w) - two{(_Float16)by, (_Float16)by}); };
        return v4u{less((q & low) | base, 1032), less((q & next) | base_next, 72), less((upper & low) | base, 1032), less((upper & next) | base_next, 72)};
    }
#pragma unroll
    for (unsigned j = 0; j < 4; ++j) v[j] = (q >> j * 4 & low) | base;
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

// A block has 32 rows of one expert's weights for each of its wavefronts, and up to 32 rows of x (fp32: 16).  It goes over k in chunks of 256:
// weights go to LDS as they are, whole lines of memory (128 bytes of a row) at a time; x goes there in the order that the matrix cores take
// (fp32: as three parts), and the rows' scales.  While a chunk is multiplied the next is on its way.
// Within a chunk a step is 32 * WORDS k, all of one group: lane (r, g) has of each of two groups of 16 rows 4 * WORDS bytes, 8 * WORDS
// consecutive k of row r.  WORDS is 4 where the group is a multiple of 128, else 2 or 1.
// Bound by reading the weights, at 5 TB/s, and by what the vector unit does for them.  us for one token on each of 8 PEs, 256 experts of 7168 x 2048,
// bf16, groups of 128 (1.3 GB), and for 64 tokens a PE (5.9 GB): 225 and 1440; with weights read into registers, 16 to 64 bytes of a row at a time, 564
// and 3900 (the lines came from memory up to four times); with two blocks a compute unit and x of two chunks in LDS 238 and 1530, with blocks of
// eight wavefronts 307 and 1730; with three operations for two weights instead of one 253 and 1690.
// Wavefronts of a block.  A few small blocks to a compute unit wait for memory apart from each other; only of fp32 elements, whose three
// parts fill LDS, eight wavefronts share one x.
template <typename T>
constexpr unsigned few_w4_waves() {
    return sizeof(T) == 4 ? 8 : 4;
}

template <typename T, unsigned WORDS, bool DMA>
struct FewFourBits {
    static constexpr unsigned kWaves = few_w4_waves<T>(), kThreads = kWaves * kLanes, kColumns = kWaves * 32;
    static constexpr bool kTwo = sizeof(T) == 4;  // x and scales of two chunks in LDS
    typedef TileSide<unsigned char, kColumns, false, DMA, kWaves> Side;
    static constexpr unsigned kChunk = 256, kParts = sizeof(T) == 4 ? 3 : 1, kStep = 32 * WORDS, kSteps = kChunk / kStep;
    static constexpr unsigned kRowBytes = kChunk * 2;  // of x in LDS
    typedef typename words<WORDS>::type raw;
    typedef typename Nibble<T>::type M;
    template <int MT>
    struct Held {
        static constexpr unsigned kPieces = MT * 16 * kChunk / 8 / kThreads;  // of eight elements of x, a thread's
        v4u x[kPieces][8 / Chunk<T>::N];
        T scale[kSteps / 2 ? kSteps / 2 : 1];  // two threads have a row's
    };
    Side side;
    const unsigned char *w, *w_up;  // the block's first row
    const T *scale;                 // this thread's row's
    const T *x;
    unsigned k_all, rows, per_group;

    template <int MT>
    __device__ __forceinline__ void fetch(Held<MT> &h, NVSHMEM_AMD_LDS char *lds_w, unsigned k, bool in) {
        constexpr unsigned N = Chunk<T>::N, kPerRow = kChunk / 8;
        const bool whole = k + kChunk <= k_all;
#pragma unroll
        for (unsigned i = 0; i < Held<MT>::kPieces; ++i) {
            const unsigned piece = i * kThreads + threadIdx.x, m = piece / kPerRow, at = k + piece % kPerRow * 8;
            const T *p = x + (uint64_t)(m < rows ? m : rows - 1) * k_all + at;  // (the last row's products stand in for rows behind it)
#pragma unroll
            for (unsigned c = 0; c < 8 / N; ++c) h.x[i][c] = __builtin_bit_cast(v4u, chunk_load(p + c * N));
            if (whole) continue;
            const unsigned left = at < k_all ? k_all - at : 0;
#pragma unroll
            for (unsigned c = 0; c < 8 / N; ++c) h.x[i][c] = chunk_load_front(p + c * N, left > c * N ? left - c * N : 0);
        }
#pragma unroll
        for (unsigned j = 0; j < kSteps / 2; ++j) {
            const unsigned at = k + (threadIdx.x / kColumns * (kSteps / 2) + j) * kStep;
            h.scale[j] = scale[__umulhi((at < k_all ? at : k) / 16, per_group)];
        }
        const unsigned wave = wave_of_block(), left = (k_all - k + 1) / 2;
        side.fetch(lds_w, wave, left < kStepBytes ? left : kStepBytes, [&](unsigned j) {
            return (in && (wave * Side::kMoves + j) * 8 % 32 >= 16 ? w_up : w) + k / 2;
        });
    }
    template <int MT>
    __device__ __forceinline__ void land(const Held<MT> &h, NVSHMEM_AMD_LDS char *lds_x, NVSHMEM_AMD_LDS float *lds_s) const {
        constexpr unsigned kPerRow = kChunk / 8;
#pragma unroll
        for (unsigned i = 0; i < Held<MT>::kPieces; ++i) {
            const unsigned piece = i * kThreads + threadIdx.x, m = piece / kPerRow, c = piece % kPerRow;
            v4u a[kParts];
            if constexpr (sizeof(T) == 2) a[0] = reorder_eight(h.x[i][0]);
            else split_eight(__builtin_bit_cast(v4f, h.x[i][0]), __builtin_bit_cast(v4f, h.x[i][1]), a);
#pragma unroll
            for (unsigned q = 0; q < kParts; ++q)
                *(NVSHMEM_AMD_LDS v4u *)(lds_x + (q * MT * 16 + m) * kRowBytes + (c ^ (m & 7)) * 16) = a[q];
        }
#pragma unroll
        for (unsigned j = 0; j < kSteps / 2; ++j)
            lds_s[(threadIdx.x / kColumns * (kSteps / 2) + j) * kColumns + threadIdx.x % kColumns] = (float)h.scale[j];
    }
    // D = w x^T: element i of a lane is row lane / 16 * 4 + i of the weights' 16, column lane % 16: a row of x.
    template <bool SIXTEENTHS, int MT>
    __device__ __forceinline__ void multiply(unsigned j, NVSHMEM_AMD_LDS const char *lds_w, NVSHMEM_AMD_LDS const char *lds_x,
                                             NVSHMEM_AMD_LDS const float *lds_s, unsigned wave, unsigned lane, v4f (&acc)[MT][2]) const {
        const unsigned r = lane % 16, g = lane / 16;
        v4u a[MT][WORDS][kParts];
        v4f sum[MT] = {};
#pragma unroll
        for (int mi = 0; mi < MT; ++mi)
#pragma unroll
            for (unsigned i = 0; i < WORDS; ++i)
#pragma unroll
                for (unsigned q = 0; q < kParts; ++q) {
                    const unsigned chunk = (j * 4 + g) * WORDS + i;
                    a[mi][i][q] = *(NVSHMEM_AMD_LDS const v4u *)(lds_x + ((q * MT + mi) * 16 + r) * kRowBytes + (chunk ^ (r & 7)) * 16);
                    if constexpr (__is_same(T, __bf16) && !SIXTEENTHS) sum[mi] = Mma<M>::step(Nibble<T>::too_much(), a[mi][i][q], sum[mi]);
                }
#pragma unroll
        for (unsigned ni = 0; ni < 2; ++ni) {
            const unsigned byte = (j * 4 + g) * 4 * WORDS, row = wave * 32 + ni * 16;
            const raw held = *(NVSHMEM_AMD_LDS const raw *)(lds_w + (row + r) * kStepBytes + ((byte / 16) ^ (r & 7)) * 16 + byte % 16);
            v4f d[MT];
#pragma unroll
            for (int mi = 0; mi < MT; ++mi) d[mi] = sum[mi];
#pragma unroll
            for (unsigned i = 0; i < WORDS; ++i) {
                unsigned word;
                if constexpr (WORDS == 1) word = held;
                else word = held[i];
                const v4u b = eight_weights<T, SIXTEENTHS>(word);
#pragma unroll
                for (int mi = 0; mi < MT; ++mi)
#pragma unroll
                    for (unsigned q = 0; q < kParts; ++q) d[mi] = Mma<M>::step(b, a[mi][i][q], d[mi]);
            }
            const v4f s = *(NVSHMEM_AMD_LDS const v4f *)(lds_s + j * kColumns + row + g * 4);
#pragma unroll
            for (int mi = 0; mi < MT; ++mi)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[mi][ni][i] = __builtin_fmaf(s[i], d[mi][i], acc[mi][ni][i]);
        }
    }
    template <bool SIXTEENTHS, int MT>
    __device__ __forceinline__ void sum_as(char *lds_w, char *lds_x, float *lds_s, bool in, v4f (&acc)[MT][2]) {
        constexpr unsigned kXBytes = kParts * MT * 16 * kRowBytes, kScales = kSteps * kColumns;
        const unsigned wave = wave_of_block(), lane = threadIdx.x % kLanes;
        Held<MT> next;
        fetch(next, (NVSHMEM_AMD_LDS char *)lds_w, 0, in);
        unsigned buffer = 0;
        for (unsigned k = 0; k < k_all; k += kChunk, buffer ^= 1) {
            NVSHMEM_AMD_LDS char *lw = (NVSHMEM_AMD_LDS char *)lds_w + buffer * Side::kBytes;
            NVSHMEM_AMD_LDS char *lx = (NVSHMEM_AMD_LDS char *)lds_x + (kTwo ? buffer : 0) * kXBytes;
            NVSHMEM_AMD_LDS float *ls = (NVSHMEM_AMD_LDS float *)lds_s + (kTwo ? buffer : 0) * kScales;
            if (!kTwo && k) __syncthreads();  // (all have multiplied the last chunk)
            side.land(lw, wave, lane);
            land(next, lx, ls);
            asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
            __syncthreads();
            if (k + kChunk < k_all) fetch(next, (NVSHMEM_AMD_LDS char *)lds_w + (buffer ^ 1) * Side::kBytes, k + kChunk, in);
#pragma unroll
            for (unsigned j = 0; j < kSteps; ++j) {
                multiply<SIXTEENTHS, MT>(j, lw, lx, ls, wave, lane, acc);
                __builtin_amdgcn_sched_barrier(0);  // (the compiler would gather all steps' reads, in registers for all)
            }
        }
    }
    // Sums over 128 + q leave fp32 before those over q - 8 do (128 elements of one sign from 2^114 on), and an infinity meets its negative in
    // them.  Once one has, it stays an infinity or a NaN.  So a block that has such a sum makes all of its sums again, of sixteenths, and takes
    // those in place of what was not finite: an element's result is the same whatever rows it came with.
    // us of one token on each of 8 PEs, 256 experts of 7168 x 2048, without / with: 225 / 227.
    template <int MT>
    __device__ __forceinline__ void sum(char *lds_w, char *lds_x, float *lds_s, bool in, v4f (&acc)[MT][2]) {
        constexpr bool kSixteenths = sizeof(T) == 4;
        sum_as<kSixteenths, MT>(lds_w, lds_x, lds_s, in, acc);
        if constexpr (__is_same(T, __bf16)) {
            float zero = 0.0f;  // (or a NaN)
#pragma unroll
            for (int mi = 0; mi < MT; ++mi)
#pragma unroll
                for (unsigned ni = 0; ni < 2; ++ni)
#pragma unroll
                    for (int i = 0; i < 4; ++i) zero = __builtin_fmaf(acc[mi][ni][i], 0.0f, zero);
            const bool any = __any(zero != 0.0f);
            __syncthreads();  // (all have multiplied the last chunk)
            if (threadIdx.x % kLanes == 0) lds_s[wave_of_block()] = any ? 1.0f : 0.0f;
            __syncthreads();
            float blocks = 0.0f;
#pragma unroll
            for (unsigned w = 0; w < kWaves; ++w) blocks += lds_s[w];
            if (__builtin_amdgcn_readfirstlane(__float_as_uint(blocks)) == 0) return;
            __syncthreads();  // (all have read it)
            v4f again[MT][2] = {};
            sum_as<true, MT>(lds_w, lds_x, lds_s, in, again);
#pragma unroll
            for (int mi = 0; mi < MT; ++mi)
#pragma unroll
                for (unsigned ni = 0; ni < 2; ++ni)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[mi][ni][i] = acc[mi][ni][i] * 0.0f == 0.0f ? acc[mi][ni][i] : again[mi][ni][i] * 16.0f;
        }
        if constexpr (kSixteenths) {
#pragma unroll
            for (int mi = 0; mi < MT; ++mi)
#pragma unroll
                for (unsigned ni = 0; ni < 2; ++ni) acc[mi][ni] *= 16.0f;
        }
    }
};

template <typename T, int OP, int MT>
__device__ __forceinline__ void few_w4_store(const ExpertArgs<T> &args, const v4f (&acc)[MT][2], unsigned pe, uint64_t first, unsigned rows,
                                             unsigned n0) {
    const unsigned wave = wave_of_block(), lane = threadIdx.x % kLanes, g = lane / 16;
    const unsigned n_all = OP == kIn ? args.hidden : args.dim;
#pragma unroll
    for (int mi = 0; mi < MT; ++mi) {
        const unsigned m = mi * 16 + lane % 16;
        if (m >= rows) continue;
        const uint64_t row = first + m;
#pragma unroll
        for (unsigned ni = 0; ni < (OP == kIn ? 1 : 2); ++ni) {
            const unsigned n = n0 + wave * (OP == kIn ? 16 : 32) + ni * 16 + g * 4;
            if (n >= n_all) continue;
            if (OP == kIn) {
                v4f h;
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = acc[mi][0][i] * sigmoid(acc[mi][0][i]) * acc[mi][1][i];
                store_four(copy_of(args.h, pe, args.stride) + row * n_all + n, h, n_all - n);
            } else {
                store_four(copy_of(args.out, pe, args.stride) + row * n_all + n, acc[mi][ni], n_all - n);
            }
        }
    }
}

// An expert of up to `more_than` rows has a block for each 32 (16) of them, which reads the weights again.
template <typename T, int OP, unsigned WORDS, bool DMA>
__global__ __launch_bounds__(few_w4_waves<T>() * kLanes, sizeof(T) == 4 ? 2 : 3) void expert_few_w4_kernel(const W4Args<T> args4) {
    typedef FewFourBits<T, WORDS, DMA> W;
    constexpr unsigned kMost = sizeof(T) == 4 ? 16 : 32;  // rows of x at a time
    __shared__ __attribute__((aligned(1024))) char lds_w[2 * W::Side::kBytes];
    __shared__ __attribute__((aligned(16))) char lds_x[(W::kTwo ? 2 : 1) * W::kParts * kMost * W::kRowBytes];
    __shared__ __attribute__((aligned(16))) float lds_s[(W::kTwo ? 2 : 1) * W::kSteps * W::kColumns];
    const ExpertArgs<T> &args = args4.e;
    const unsigned pe = blockIdx.z, lane = threadIdx.x % kLanes, part = blockIdx.y / args.experts, e = blockIdx.y % args.experts;
    const unsigned n0 = blockIdx.x * (OP == kIn ? W::kColumns / 2 : W::kColumns);
    uint64_t first, rows;
    expert_range(copy_of(args.expert_row, pe, args.stride), e, args.cap, first, rows);
    if (rows <= part * kMost || rows > args.more_than) return;
    first = scalar64(first + part * kMost);
    const unsigned mine = rows - part * kMost < kMost ? (unsigned)(rows - part * kMost) : kMost;
    const unsigned n_all = OP == kIn ? args.hidden : args.dim, k_all = OP == kIn ? args.dim : args.hidden;
    const unsigned row_bytes = (k_all + 1) / 2, n_here = n_all - n0;
    const uint64_t before = (uint64_t)e * (OP == kIn ? 2 : 1) * n_all + n0;
    // Row r of the block's weights, from its first: kIn's wavefronts have 16 of gate and the same 16 of up.
    const auto place = [](unsigned r) { return OP == kIn ? r / 32 * 16 + r % 16 : r; };
    W w;
    w.side.begin(wave_of_block(), lane, n_here, row_bytes, place);
    w.w = copy_of(OP == kIn ? args4.w_in : args4.w_out, pe, args.stride) + before * row_bytes;
    w.w_up = w.w + (uint64_t)n_all * row_bytes;
    const unsigned r = threadIdx.x % W::kColumns, at = place(r) < n_here ? place(r) : n_here - 1;
    w.scale = copy_of(OP == kIn ? args4.s_in : args4.s_out, pe, args.stride) +
              (before + (OP == kIn && r % 32 >= 16 ? n_all : 0) + at) * ((k_all + args4.group - 1) / args4.group);
    w.x = copy_of(OP == kIn ? args.rows : (const T *)args.h, pe, args.stride) + first * k_all;
    w.k_all = k_all, w.rows = mine, w.per_group = args4.per_group;
    if (kMost == 16 || mine <= 16) {
        v4f acc[1][2] = {};
        w.template sum<1>(lds_w, lds_x, lds_s, OP == kIn, acc);
        few_w4_store<T, OP, 1>(args, acc, pe, first, mine, n0);
    } else if constexpr (kMost > 16) {
        v4f acc[2][2] = {};
        w.template sum<2>(lds_w, lds_x, lds_s, OP == kIn, acc);
        few_w4_store<T, OP, 2>(args, acc, pe, first, mine, n0);
    }
}

// ---- experts of more rows: tiles ----

constexpr unsigned kTileN = 256;

// B's way into LDS: 256 rows of packed weights, half a step's k of a row for each thread, as (q - 8) / 16 in T (exact) where TileSide<T, 256, false>
// reads them.  Their scales go beside them, one for each half of each row.
template <typename T>
struct FourBitSide {
    static constexpr unsigned kStepK = kStepBytes / sizeof(T), kHalfK = kStepK / 2, kWords = kHalfK / 8;
    typedef typename words<kWords>::type raw;
    typedef raw raw_unaligned __attribute__((aligned(1)));
    const unsigned char *row;  // this thread's; where it has none, a row that exists
    const T *scale;
    unsigned k_all, per_group;
    struct Held {
        raw q;
        T scale;
    };

    __device__ __forceinline__ Held fetch(unsigned k) const {
        Held h;
        const unsigned at = k + threadIdx.x % 2 * kHalfK;
        const unsigned char *p = row + at / 2;
        h.scale = scale[__umulhi((at < k_all ? at : k) / 16, per_group)];
        h.q = *(const raw_unaligned *)p;  // (behind the row's end: what lies there, times zeros of A)
        return h;
    }
    __device__ __forceinline__ void land(const Held &h, NVSHMEM_AMD_LDS char *lds, NVSHMEM_AMD_LDS float *scales) const {
        const unsigned r = threadIdx.x / 2, half = threadIdx.x % 2;
        scales[half * kTileN + r] = (float)h.scale;
#pragma unroll
        for (unsigned j = 0; j < 4; ++j) {
            typename Chunk<T>::vec v;
#pragma unroll
            for (unsigned i = 0; i < (unsigned)Chunk<T>::N; ++i) {
                // (the instruction takes four bits with a sign and gives a sixteenth of them: q - 8 with its highest bit turned over)
                const unsigned at = j * Chunk<T>::N + i, word = h.q[at / 8] ^ 0x88888888u;
                v[i] = (T)__builtin_amdgcn_cvt_off_f32_i4((int)((at % 2 ? word >> 4 : word) >> at % 8 / 2 * 8));
            }
            *(NVSHMEM_AMD_LDS v4u *)(lds + r * kStepBytes + (((half * 4 + j) ^ (r & 7)) * 16)) = __builtin_bit_cast(v4u, v);
        }
    }
};

// HALVES: the halves of a step may be of two groups.  Bound by the vector unit: it makes q - 8 of a block's weights once for BM rows, and for each
// product of the matrix cores multiplies four sums with their scales (HALVES; two otherwise), which takes as long as the product.  us for 32768 rows of 64
// experts of 7168 x 2048, groups of 32: 3970 with BM of 256 (0.73 PFLOP/s); with weights fetched behind the products' start 5040, with BM of 128
// before that 7780.
template <typename T, int OP, unsigned BM, bool HALVES, bool DMA>
__global__ __launch_bounds__(kTileThreads, 2) void expert_tile_w4_kernel(const W4Args<T> args4) {
    constexpr unsigned kMi = BM / 32, kNi = 4;
    typedef TileSide<T, BM, false, DMA> A;
    typedef TileSide<T, kTileN, false, true> B;  // (its layout in LDS)
    typedef FourBitSide<T> Q;
    constexpr unsigned kStepK = A::kStepK;
    constexpr bool kAhead = BM == 128 && DMA;
    __shared__ __attribute__((aligned(1024))) char lds_a[2 * A::kBytes];
    __shared__ __attribute__((aligned(1024))) char lds_b[2 * B::kBytes];
    __shared__ __attribute__((aligned(16))) float lds_s[2 * 2 * kTileN];
    __shared__ TileList list;
    const ExpertArgs<T> &args = args4.e;
    const unsigned wave = wave_of_block(), lane = threadIdx.x % kLanes;
    const unsigned n_all = OP == kIn ? args.hidden : args.dim, k_all = OP == kIn ? args.dim : args.hidden;
    const unsigned n_tile = OP == kIn ? kTileN / 2 : kTileN, wide = (n_all + n_tile - 1) / n_tile;
    list.make(args.expert_row, args.stride, args.cap, args.experts, args.npes, BM, wide, args.more_than);
    const unsigned total = list.total();
    for (unsigned i = 0;; ++i) {
        unsigned t = tile_of_block(i, total);
        if (t >= total) return;
        unsigned e = list.find(t);
        const unsigned pe = e / args.experts;
        e -= pe * args.experts;
        uint64_t first, rows;
        expert_range(copy_of(args.expert_row, pe, args.stride), e, args.cap, first, rows);
        first = scalar64(first), rows = scalar64(rows);
        unsigned tm, tn;
        const uint64_t high = (rows + BM - 1) / BM;
        if (t >= high * wide) continue;  // (a table whose ranges overlap many times over may count past 2^32)
        tile_place(t, (unsigned)high, wide, tm, tn);
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
            side_b.k_all = k_all, side_b.per_group = args4.per_group;
            side_b.row = copy_of(OP == kIn ? args4.w_in : args4.w_out, pe, args.stride) + n * ((k_all + 1) / 2);
            side_b.scale = copy_of(OP == kIn ? args4.s_in : args4.s_out, pe, args.stride) + n * ((k_all + args4.group - 1) / args4.group);
        }
        const auto fetch_a = [&](unsigned buffer, unsigned k) {
            const unsigned left = k_all - k < kStepK ? k_all - k : kStepK;
            side_a.fetch((NVSHMEM_AMD_LDS char *)lds_a + buffer * A::kBytes, wave, left, [&](unsigned) { return a + k; });
        };
        v4f acc[kMi][kNi] = {};
        const unsigned wm = wave / 4, wn = wave % 4;
        typename Q::Held held = side_b.fetch(0), next = {};
        fetch_a(0, 0);
        // (tiles of 128 rows, of which there are few: weights are fetched two steps ahead)
        if (kAhead && kStepK < k_all) next = side_b.fetch(kStepK);
        unsigned buffer = 0;
        for (unsigned k = 0; k < k_all; k += kStepK, buffer ^= 1) {
            NVSHMEM_AMD_LDS char *la = (NVSHMEM_AMD_LDS char *)lds_a + buffer * A::kBytes, *lb = (NVSHMEM_AMD_LDS char *)lds_b + buffer * B::kBytes;
            NVSHMEM_AMD_LDS float *ls = (NVSHMEM_AMD_LDS float *)lds_s + buffer * 2 * kTileN;
            side_a.land(la, wave, lane);
            side_b.land(held, lb, ls);
            // what of A is on its way to LDS was asked for in front of the weights two steps ahead, whose last load may go on
            if (kAhead && k + kStepK < k_all) asm volatile("s_waitcnt vmcnt(1)" : : : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
            __syncthreads();
            if (k + kStepK < k_all) {
                fetch_a(buffer ^ 1, k + kStepK);
                if (!kAhead) held = side_b.fetch(k + kStepK);
                else held = next;
                if (kAhead && k + 2 * kStepK < k_all) next = side_b.fetch(k + 2 * kStepK);
                __builtin_amdgcn_sched_barrier(0);
            }
            v4u fb[2][kNi], fa[2][2];
            v4f s[HALVES ? 2 : 1][kNi];
#pragma unroll
            for (unsigned ni = 0; ni < kNi; ++ni) {
                fb[0][ni] = B::read(lb, wn * 4 + ni, 0, lane), fb[1][ni] = B::read(lb, wn * 4 + ni, 1, lane);
                s[0][ni] = *(NVSHMEM_AMD_LDS const v4f *)(ls + wn * 64 + ni * 16 + lane / 16 * 4);
                if (HALVES) s[HALVES][ni] = *(NVSHMEM_AMD_LDS const v4f *)(ls + kTileN + wn * 64 + ni * 16 + lane / 16 * 4);
            }
            fa[0][0] = A::read(la, wm * kMi, 0, lane), fa[0][1] = A::read(la, wm * kMi, 1, lane);
#pragma unroll
            for (unsigned mi = 0; mi < kMi; ++mi) {
                if (mi + 1 < kMi) fa[(mi + 1) % 2][0] = A::read(la, wm * kMi + mi + 1, 0, lane), fa[(mi + 1) % 2][1] = A::read(la, wm * kMi + mi + 1, 1, lane);
#pragma unroll
                for (unsigned n = 0; n < kNi; n += 2) {
                    v4f d[2][2];
#pragma unroll
                    for (unsigned ni = 0; ni < 2; ++ni) d[0][ni] = Mma<T>::step(fb[0][n + ni], fa[mi % 2][0], v4f{});
#pragma unroll
                    for (unsigned ni = 0; ni < 2; ++ni) d[1][ni] = Mma<T>::step(fb[1][n + ni], fa[mi % 2][1], HALVES ? v4f{} : d[0][ni]);
#pragma unroll
                    for (unsigned ni = 0; ni < 2; ++ni)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (HALVES) acc[mi][n + ni][j] = __builtin_fmaf(s[0][n + ni][j], d[0][ni][j], acc[mi][n + ni][j]);
                            acc[mi][n + ni][j] = __builtin_fmaf(s[HALVES][n + ni][j], d[1][ni][j], acc[mi][n + ni][j]);
                        }
                }
                if (BM == 256) __builtin_amdgcn_sched_barrier(0);  // (or products of several rows wait for their sums in registers that are not there)
            }
        }
        __syncthreads();
        const unsigned r = lane % 16;
#pragma unroll
        for (unsigned mi = 0; mi < kMi; ++mi) {
            const unsigned m = (wm * kMi + mi) * 16 + r;
            if (m >= m_here) continue;
            const uint64_t row = first + m0 + m;
            v4f v[kNi];
#pragma unroll
            for (unsigned ni = 0; ni < kNi; ++ni) v[ni] = acc[mi][ni] * 16.0f;  // (weights were sixteenths)
            if (OP == kIn) {
#pragma unroll
                for (unsigned ni = 0; ni < 2; ++ni)
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[ni][j] = v[ni][j] * sigmoid(v[ni][j]) * v[ni + 2][j];
                store_32(copy_of(args.h, pe, args.stride) + row * args.hidden + n0, wn * 32, v[0], v[1], n_here, lane);
            } else {
#pragma unroll
                for (unsigned ni = 0; ni < kNi; ni += 2)
                    store_32(copy_of(args.out, pe, args.stride) + row * args.dim + n0, wn * 64 + ni * 16, v[ni], v[ni + 1], n_here, lane);
            }
        }
    }
}

// Experts of more rows are the tiles'.  us with 64 / 128 here: 64 tokens on each of 8 PEs, 256 experts of 7168 x 2048, 1560 / 1660; 128 rows each for 64
// experts of 4096 x 1536 820 / 780; a step of four tokens that no expert can have more than 74 rows of 16.4 / 11.3 (no launch of tiles).
constexpr unsigned kW4FewRows = 64;
// ... and those of 256 rows where experts have more than this on average at most: weights are made ready half as often.  us with 128 / 256 rows, 64
// experts of 4096 x 1536 with 100 rows each 531 / -, 200: 883 / 869, 400: 1512 / 1276, 800: 2665 / 2303.
constexpr unsigned kW4LargeRows = 256;

template <typename T, int OP, bool DMA>
void launch_few_w4(const W4Args<T> &args, int npes, hipStream_t stream) {
    const uint64_t rows = args.e.cap < kW4FewRows ? args.e.cap : kW4FewRows;
    constexpr unsigned threads = few_w4_waves<T>() * kLanes, columns = few_w4_waves<T>() * 32;
    const dim3 grid(div_up(OP == kIn ? args.e.hidden : args.e.dim, OP == kIn ? columns / 2 : columns),
                    args.e.experts * div_up(rows, sizeof(T) == 4 ? 16 : 32), npes);
    if (args.group % 128 == 0) launch_kernel((expert_few_w4_kernel<T, OP, 4, DMA>), grid, dim3(threads), 0, stream, args);
    else if (args.group % 64 == 0) launch_kernel((expert_few_w4_kernel<T, OP, 2, DMA>), grid, dim3(threads), 0, stream, args);
    else launch_kernel((expert_few_w4_kernel<T, OP, 1, DMA>), grid, dim3(threads), 0, stream, args);
}
template <typename T, int OP, unsigned BM, bool HALVES, bool DMA>
void launch_tiles_w4_as(const W4Args<T> &args, int npes, hipStream_t stream) {
    const uint64_t wide = div_up(OP == kIn ? args.e.hidden : args.e.dim, OP == kIn ? kTileN / 2 : kTileN);
    const uint64_t tiles = (args.e.cap / BM + (args.e.experts < args.e.cap ? args.e.experts : args.e.cap)) * wide * npes;
    launch_kernel((expert_tile_w4_kernel<T, OP, BM, HALVES, DMA>), dim3(tile_blocks(tiles, 1)), dim3(kTileThreads), 0, stream, args);
}
template <typename T, int OP, bool HALVES>
void launch_tiles_w4(const W4Args<T> &args, bool whole, int npes, hipStream_t stream) {
    const uint64_t rows = (args.e.cap + args.e.experts - 1) / args.e.experts;
    if (!whole) return launch_tiles_w4_as<T, OP, 128, HALVES, false>(args, npes, stream);
    if constexpr (sizeof(T) == 2)
        if (rows > kW4LargeRows) return launch_tiles_w4_as<T, OP, 256, HALVES, true>(args, npes, stream);
    launch_tiles_w4_as<T, OP, 128, HALVES, true>(args, npes, stream);
}
template <typename T, int OP>
void launch_w4(const W4Args<T> &args, bool whole, int npes, hipStream_t stream) {
    const unsigned row_bytes = ((OP == kIn ? args.e.dim : args.e.hidden) + 1) / 2;
    if (row_bytes % 16 == 0 && aligned16(OP == kIn ? args.w_in : args.w_out)) launch_few_w4<T, OP, true>(args, npes, stream);
    else launch_few_w4<T, OP, false>(args, npes, stream);
    if (args.e.cap <= kW4FewRows) return;
    if constexpr (sizeof(T) == 2)
        if (args.group % 64) return launch_tiles_w4<T, OP, true>(args, whole, npes, stream);
    launch_tiles_w4<T, OP, false>(args, whole, npes, stream);
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
    args.per_group = (unsigned)((((uint64_t)1 << 31) + group / 32 - 1) / (group / 32));
    a.stride = rt.heap_size, a.cap = cap, a.experts = (unsigned)mine, a.npes = (unsigned)rt.npes, a.dim = (unsigned)dim, a.hidden = (unsigned)hidden;
    a.more_than = kW4FewRows;
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
