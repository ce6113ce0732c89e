// The experts' products in tiles of the matrix cores: D[m, n] = sum over k of A(m, k) B(n, k) for one expert at a time.
//
//            A(m, k)            B(n, k)               D
//   kIn      rows[m][k]         w_in[n][k], two n     pre, h = silu(gate) * up    one tile has BN/2 columns of gate and the same of up
//   kOut     h[m][k]            w_out[n][k]           out
//   kDh      dout[m][k]         w_out[k][n]           dh, and from it with pre: dpre and h
//   kDx      dpre[m][k]         w_in[k][n]            drows
//   kDwIn    dpre[k][m]         rows[k][n]            dw_in                       k runs over the expert's rows
//   kDwOut   dout[k][m]         h[k][n]               dw_out
//
// A tile of D is BM x BN, a block has one: eight wavefronts in two rows of four (four in one row, of tiles of 32 rows), each with BM/2 (32) x
// BN/4 of it in its accumulators (fp32).  A and B pass through LDS in steps of 128 bytes of k, two or three in turn: while one is
// multiplied the others are on their way.
//
// Large products are bound by the matrix cores, at the clock that the power limit leaves them: 131072 rows of 64 experts of 7168 x 2048 bf16 (kIn)
// run at 1.86 GHz with the matrix cores busy for 64 % of the time, 1.2 PFLOP/s with the tiles' ragged ends, and a library's product of 8192^3
// at 1.49 GHz and 87 %, 1.33 to 1.39.  Small ones are bound by reading the weights, or by the chain of steps of one tile.
#pragma once

#include "token_common.hpp"

namespace nvshmem_amd {
namespace tokens {

enum ExpertProduct { kIn, kOut, kDh, kDx, kDwIn, kDwOut };

typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));

#define NVSHMEM_AMD_LDS __attribute__((address_space(3)))

// What a lane holds of 16 rows for the matrix cores: 16 bytes of consecutive k of row lane % 16, the (lane / 16)-th such piece of 64
// bytes.  D has a's row lane / 16 * 4 + i and b's row lane % 16 in element i.
template <typename T>
struct Mma;
template <>
struct Mma<__bf16> {
    typedef __bf16 vec __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ v4f step(v4u a, v4u b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
    }
};
template <>
struct Mma<_Float16> {
    typedef _Float16 vec __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ v4f step(v4u a, v4u b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
    }
};
template <>
struct Mma<float> {
    static __device__ __forceinline__ v4f step(v4u a, v4u b, v4f c) {
#pragma unroll
        for (int i = 0; i < 4; ++i)  // (k in another order than it lies in memory, the same for both)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
        return c;
    }
};

// The first n (at most N) elements at p, and zeros behind them.  All of a chunk is read: no operand ends less than
// NVSHMEMI_AMD_INTERNAL_BYTES in front of its PE's slice, so that what lies behind it can be read, whatever it is.
template <typename T>
__device__ __forceinline__ v4u chunk_load_front(const T *p, unsigned n) {
    const v4u v = __builtin_bit_cast(v4u, chunk_load(p));
    v4u mask;
#pragma unroll
    for (unsigned i = 0; i < 4; ++i) {
        const int bytes = (int)(n * sizeof(T)) - (int)i * 4;  // of this word
        mask[i] = bytes >= 4 ? ~0u : bytes <= 0 ? 0u : (1u << bytes * 8) - 1;
    }
    return v & mask;
}

// One call's operands, PE 0's copies.  Which of them a product reads and writes is in the table above.
template <typename T>
struct ExpertArgs {
    const int64_t *expert_row;
    const T *rows, *w_in, *w_out, *dout, *pre_in;
    T *out, *pre, *h, *dpre, *drows, *dw_in, *dw_out;
    uint64_t stride, cap;
    unsigned experts, npes;  // experts of a PE
    unsigned dim, hidden;
    unsigned more_than;  // experts of at most so many rows are another kernel's (of the weights of 4 bits)
};

// Expert e's rows, whatever the table holds: never outside [0, cap).
__device__ __forceinline__ void expert_range(const int64_t *expert_row, unsigned e, uint64_t cap, uint64_t &first, uint64_t &rows) {
    const int64_t a = expert_row[e], b = expert_row[e + 1];
    const uint64_t lo = a < 0 ? 0 : (uint64_t)a < cap ? (uint64_t)a : cap, hi = b < 0 ? 0 : (uint64_t)b < cap ? (uint64_t)b : cap;
    first = lo;
    rows = hi > lo ? hi - lo : 0;
}

__device__ __forceinline__ uint64_t scalar64(uint64_t x) {
    return (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)x);
}

constexpr unsigned kTileThreads = 512, kTileWaves = kTileThreads / kLanes;
constexpr unsigned kMostExperts = 1024;

// The tiles of all PEs' experts in a row: expert by expert, `columns` tiles wide and as many high as its rows need.  first[e] is where
// those of expert e (the e-th of all) begin.
struct TileList {
    unsigned first[kMostExperts + 1];
    unsigned wave_sum[kTileWaves];

    // By a whole block of WAVES wavefronts; two experts a thread, or four.
    template <unsigned WAVES = kTileWaves>
    __device__ __forceinline__ void make(const int64_t *expert_row, uint64_t stride, uint64_t cap, unsigned per_pe, unsigned npes, unsigned tile_rows,
                                         unsigned columns, unsigned more_than) {
        const unsigned wave = wave_of_block(), lane = threadIdx.x % kLanes, all = per_pe * npes;
        constexpr unsigned kEach = kMostExperts / (WAVES * kLanes);
        unsigned own[kEach], sum = 0;
#pragma unroll
        for (unsigned i = 0; i < kEach; ++i) {
            const unsigned e = threadIdx.x * kEach + i;
            uint64_t at = 0, rows = 0;
            if (e < all) expert_range(copy_of(expert_row, e / per_pe, stride), e % per_pe, cap, at, rows);
            own[i] = rows > more_than ? (unsigned)((rows + tile_rows - 1) / tile_rows) * columns : 0;
            sum += own[i];
        }
        if (!__syncthreads_or(sum)) {  // as in a step of single tokens: none of this kernel's experts has rows
            if (threadIdx.x == 0) first[kMostExperts] = 0;
            __syncthreads();
            return;
        }
        unsigned before = sum;
#pragma unroll
        for (int d = 1; d < kLanes; d *= 2) {
            const unsigned up = __shfl_up(before, d);
            if (lane >= (unsigned)d) before += up;
        }
        if (lane == kLanes - 1) wave_sum[wave] = before;
        __syncthreads();
        for (unsigned w = 0; w < wave; ++w) before += wave_sum[w];
        before -= sum;
#pragma unroll
        for (unsigned i = 0; i < kEach; ++i) {
            first[threadIdx.x * kEach + i] = before;
            before += own[i];
        }
        if (threadIdx.x == WAVES * kLanes - 1) first[kMostExperts] = before;
        __syncthreads();
    }
    __device__ __forceinline__ unsigned total() const { return __builtin_amdgcn_readfirstlane(first[kMostExperts]); }
    // The expert of tile t < total(), which becomes the number among that expert's.
    __device__ __forceinline__ unsigned find(unsigned &t) const {
        unsigned lo = 0;  // first[lo] <= t < first[lo + 2 * step]
#pragma unroll
        for (unsigned step = kMostExperts / 2; step; step /= 2)
            if (first[lo + step] <= t) lo += step;
        lo = __builtin_amdgcn_readfirstlane(lo);
        t = __builtin_amdgcn_readfirstlane(t - first[lo]);
        return lo;
    }
};

// The tiles of a launch go to its blocks in turn, groups of up to 32 consecutive ones to an XCD (a block runs on XCD blockIdx.x % 8, which
// has 32 compute units; 64 where two blocks share one): what such a group shares is read into one L2.  The i-th tile of this block, or
// a number that no tile has.
__device__ __forceinline__ unsigned tile_of_block(unsigned i, unsigned total) {
    const unsigned slots = gridDim.x / 8, even = (total + 7) / 8, group = even < slots ? even : slots;
    const unsigned slot = blockIdx.x / 8;
    return slot < group ? (i * 8 + blockIdx.x % 8) * group + slot : ~0u;
}

// Where tile number i of `high` x `wide` tiles lies: columns of four tiles are gone through from top to bottom, so that the 32 tiles
// that an XCD works on at a time share 8 strips of A and 4 of B in its L2.
__device__ __forceinline__ void tile_place(unsigned i, unsigned high, unsigned wide, unsigned &m, unsigned &n) {
    const unsigned per = high * 4, strip = i / per, left = wide - strip * 4, width = left < 4 ? left : 4, rest = i - strip * per;
    m = rest / width;
    n = strip * 4 + rest % width;
}

constexpr unsigned kStepBytes = 128;        // of k
constexpr unsigned kNowhere = 0x80000000u;  // an offset behind every buffer: reads zeros

// One operand's way into LDS: R rows of a step.
//   KM false: k is contiguous in memory.  LDS holds R rows of 128 bytes, chunk c of row r (16 bytes) at place c ^ (r & 7): what 16 lanes
//     read together, one chunk of 16 rows, then lies in 8 different groups of banks.
//   KM true: k is the row in memory.  LDS holds the step's k one after the other, R elements each, whose blocks of 16 elements change
//     places with k (block b at b ^ swap(k)) for the same reason; ds_read_b64_tr_b16 turns them over on the way to the registers.
// A wavefront moves 1 KiB at a time, which lands in LDS as it goes over its lanes; so the lanes pick the chunks that belong there.
template <typename T, unsigned R, bool KM, bool DMA, unsigned WAVES = kTileWaves>
struct TileSide {
    static constexpr unsigned N = 16 / sizeof(T), kMoves = R / 8 / WAVES, kBytes = R * kStepBytes, kStepK = kStepBytes / sizeof(T);
    unsigned off[kMoves];   // from the step's base, kNowhere where nothing is to be read whatever k is
    unsigned along[kMoves]; // KM: the step's k of this lane's chunk; else its first k
    unsigned width[kMoves]; // KM: elements of the chunk that are inside; else N
    v4u held[DMA ? 1 : kMoves];

    static __device__ __forceinline__ unsigned swap(unsigned k) { return sizeof(T) == 2 ? (k & 3) | (k >> 1 & 4) : k >> 2 & 3; }

    // `extent`: rows (KM: columns) that exist from the tile's first on; ld in elements.  Tile row r is row place(r) of the operand.
    template <typename PLACE>
    __device__ __forceinline__ void begin(unsigned wave, unsigned lane, unsigned extent, unsigned ld, PLACE place) {
#pragma unroll
        for (unsigned j = 0; j < kMoves; ++j) {
            const unsigned move = wave * kMoves + j;
            if (!KM) {
                const unsigned r = move * 8 + lane / 8, c = lane % 8 ^ (r & 7), at = place(r);
                along[j] = c * N;
                width[j] = N;
                off[j] = at < extent ? at * ld * (unsigned)sizeof(T) + c * 16 : kNowhere;
            } else {
                constexpr unsigned kPer = R * sizeof(T) / 16, kBlock = sizeof(T);  // chunks of a k, chunks of 16 elements
                const unsigned chunk = move * kLanes + lane, k = chunk / kPer, c = chunk % kPer;
                const unsigned from = ((c / kBlock) ^ swap(k)) * kBlock + c % kBlock, col = from * N;
                along[j] = k;
                width[j] = col < extent ? (extent - col < N ? extent - col : N) : 0;
                off[j] = col < extent ? k * ld * (unsigned)sizeof(T) + from * 16 : kNowhere;
            }
        }
    }
    // Starts the way of a step whose first k is at `base` (per move) and that has `left` k.
    template <typename BASE>
    __device__ __forceinline__ void fetch(NVSHMEM_AMD_LDS char *lds, unsigned wave, unsigned left, BASE base) {
#pragma unroll
        for (unsigned j = 0; j < kMoves; ++j) {
            const char *p = (const char *)base(j);
            if (DMA) {
                const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, 0x7fffffff, 0x00020000);
                const unsigned o = along[j] < left ? off[j] : kNowhere;
                // Not the builtin: behind that, the compiler waits for all loads on their way to LDS in front of every read of it.
                // The step's barrier waits for them instead.  (Five wait states: the buffer's words may come from v_readfirstlane.  m0 is
                // named as changed: the compiler gives it to no variable, and says so, but may keep an address there for LDS.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                             :
                             : "s"((unsigned)(uintptr_t)(lds + (wave * kMoves + j) * 1024)), "v"(o), "s"(rsrc)
                             : "memory", "m0");
#pragma clang diagnostic pop
            } else {
                const unsigned n = off[j] == kNowhere || along[j] >= left ? 0 : KM ? width[j] : (left - along[j] < N ? left - along[j] : N);
                held[j] = chunk_load_front((const T *)(p + (n ? off[j] : 0)), n);
            }
        }
    }
    __device__ __forceinline__ void land(NVSHMEM_AMD_LDS char *lds, unsigned wave, unsigned lane) {
        if (DMA) return;
#pragma unroll
        for (unsigned j = 0; j < kMoves; ++j) *(NVSHMEM_AMD_LDS v4u *)(lds + (wave * kMoves + j) * 1024 + lane * 16) = held[j];
    }
    // Rows [16 block, 16 block + 16) of 64 bytes of k, the s-th of a step's two, as the matrix cores take them.
    static __device__ __forceinline__ v4u read(NVSHMEM_AMD_LDS const char *lds, unsigned block, unsigned s, unsigned lane) {
        const unsigned r = lane % 16, g = lane / 16;
        if (!KM) return *(NVSHMEM_AMD_LDS const v4u *)(lds + (block * 16 + r) * kStepBytes + (((s * 4 + g) ^ (r & 7)) * 16));
        if (sizeof(T) == 2) {
            // (what a wavefront reads at once, k of g * 8 + 0..3 and four k further, is spread over all eight places of a block among eight)
            const unsigned k = s * 32 + g * 8 + r / 4;
            const char NVSHMEM_AMD_LDS *p = lds + k * R * 2 + ((block ^ (r / 4 | (g & 1) * 4)) * 32) + r % 4 * 8, *q = p + 4 * R * 2;
            const v2u lo = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((NVSHMEM_AMD_LDS v4s *)p));
            const v2u hi = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((NVSHMEM_AMD_LDS v4s *)q));
            return v4u{lo[0], lo[1], hi[0], hi[1]};
        }
        v4u v;
#pragma unroll
        for (unsigned i = 0; i < 4; ++i)
            v[i] = *(NVSHMEM_AMD_LDS const unsigned *)(lds + (s * 16 + g * 4 + i) * R * 4 + ((block ^ g) * 64) + r * 4);
        return v;
    }
};

// Four consecutive elements of a row, of which `n` exist.
template <typename T>
__device__ __forceinline__ void store_four(T *p, v4f v, unsigned n) {
    typedef T four __attribute__((ext_vector_type(4)));
    typedef four four_unaligned __attribute__((aligned(sizeof(T))));
    const four y = __builtin_convertvector(v, four);
    if (n >= 4) {
        *(four_unaligned *)p = y;
    } else {
#pragma unroll
        for (unsigned i = 0; i < 3; ++i)
            if (i < n) p[i] = y[i];
    }
}
// Columns [c, c + 32) of a row, of which a lane has c + 4 (lane / 16) + i in lo and 16 further in hi; `n` of them exist.  Of 16-bit elements,
// rows of 16 lanes exchange halves first, so that each lane stores eight consecutive ones: half as many stores of twice the length.  us
// without / with: forward pass of 131072 rows 9660 / 9370, gradients of 76 rows an expert 838 / 716.
template <typename T>
__device__ __forceinline__ void store_32(T *row, unsigned c, v4f lo, v4f hi, unsigned n, unsigned lane) {
    const unsigned g = lane / 16;
    if constexpr (sizeof(T) == 4) {
        if (c + g * 4 < n) store_four(row + c + g * 4, lo, n - c - g * 4);
        if (c + 16 + g * 4 < n) store_four(row + c + 16 + g * 4, hi, n - c - 16 - g * 4);
    } else {
        typedef T four __attribute__((ext_vector_type(4)));
        const v2u a = __builtin_bit_cast(v2u, __builtin_convertvector(lo, four)), b = __builtin_bit_cast(v2u, __builtin_convertvector(hi, four));
        // (the second and fourth row of the first operand change places with the first and third of the second)
        const auto x = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), y = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
        const unsigned at = c + (g & 1) * 16 + (g >> 1) * 8;
        if (at >= n) return;
        const typename Chunk<T>::vec v = __builtin_bit_cast(typename Chunk<T>::vec, v4u{x[0], y[0], x[1], y[1]});
        if (n - at >= 8) *(typename Chunk<T>::vec_unaligned *)(row + at) = v;
        else chunk_store_part(row + at, v, n - at);
    }
}
template <typename T>
struct Four {
    typedef T vec __attribute__((ext_vector_type(4)));
    typedef vec vec_unaligned __attribute__((aligned(sizeof(T))));
};
template <typename T>
__device__ __forceinline__ v4f as_float(typename Four<T>::vec v) {
    return __builtin_convertvector(v, v4f);
}
// 1 / (1 + exp(-x)); exp overflows to an infinity, whose reciprocal is 0.
__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }

template <int OP>
constexpr bool a_by_k() { return OP == kDwIn || OP == kDwOut; }
template <int OP>
constexpr bool b_by_k() { return OP != kIn && OP != kOut; }

// The multiplication of a tile, once its first STAGES steps are on their way (start()).  A wavefront goes through a step in groups of one
// piece of A with all of its pieces of B, kAhead groups after it read the piece, so that reads of LDS and products overlap.  All of a
// step's pieces are in registers kAhead groups before its end: there the block meets, the step STAGES further takes the step's place in
// LDS, and what is read from there on is of the next step.  us for 131072 rows of 64 experts (7168 x 2048 bf16, kIn / kOut) with the reads left to
// the compiler, which waits for each pair of them, and now: 6473 / 3637, 6382 / 3524.  kAhead of 4, a branch around pieces of A without rows, and
// a higher priority for wavefronts at products were not faster; nor was it to start the next tile's way in front of a tile's stores.
template <typename T, typename A, typename B, unsigned kMi, unsigned kNi, unsigned STAGES>
struct TileProduct {
    static constexpr unsigned kGroups = 2 * kMi, kAhead = kMi < 4 ? 1 : 2, kMoves = A::kMoves + B::kMoves;
    static constexpr unsigned kAlone = 256 / A::kStepK;  // steps
    NVSHMEM_AMD_LDS char *lds_a, *lds_b;  // STAGES steps of each
    unsigned wave, lane;

    // fetch(buffer, step): starts the step's way; land(buffer): ends it where it leads through registers.
    template <bool DMA, typename FETCH, typename LAND>
    __device__ __forceinline__ void start(unsigned steps, FETCH fetch, LAND land) const {
        if (steps == 0) return;
        fetch(0, 0);
        land(0);
#pragma unroll
        for (unsigned i = 1; i < STAGES; ++i)
            if (i < steps) fetch(i, i);
    }
    // Until no more than `later` steps' loads are on their way (a barrier alone does not wait for what goes to LDS); all of them where
    // the last steps' were not asked for.
    __device__ __forceinline__ void wait(bool all_there, unsigned later) const {
        if (STAGES > 2 && all_there && later == STAGES - 1) asm volatile("s_waitcnt vmcnt(%0)" : : "n"((STAGES - 1) * kMoves) : "memory");
        else if (STAGES > 2 && all_there) asm volatile("s_waitcnt vmcnt(%0)" : : "n"((STAGES - 2) * kMoves) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    }
    template <bool DMA, typename FETCH, typename LAND>
    __device__ __forceinline__ void run(unsigned steps, FETCH fetch, LAND land, v4f (&acc)[kMi][kNi]) const {
        if (steps == 0) return;
        wait(steps >= STAGES, STAGES - 1);
        __syncthreads();
        const unsigned wm = wave / 4, wn = wave % 4;
        v4u fa[2 * kAhead], fb[2][kNi];
        const auto read_a = [&](unsigned buffer, unsigned g) {
            fa[g % (2 * kAhead)] = A::read(lds_a + buffer * A::kBytes, wm * kMi + g % kMi, g / kMi, lane);
        };
        const auto read_b = [&](unsigned buffer, unsigned s, unsigned ni) { fb[s][ni] = B::read(lds_b + buffer * B::kBytes, wn * kNi + ni, s, lane); };
#pragma unroll
        for (unsigned ni = 0; ni < kNi; ++ni) read_b(0, 0, ni);
#pragma unroll
        for (unsigned g = 0; g < kAhead; ++g) read_a(0, g);
        unsigned buffer = 0, other = 1;
        // Of fp32 elements, whose results are rounded no further, products of 256 k are added up by themselves: a sum of thousands in a row
        // would lose a bit or two more (relative to 64 bits, of 3918: 1.3e-6 in a row, 5e-7 so; and 7.5e-7 in PyTorch).
        v4f all[sizeof(T) == 4 ? kMi : 1][kNi] = {};
        for (unsigned step = 0; step < steps; ++step, buffer = other, other = other + 1 == STAGES ? 0 : other + 1) {
            if (sizeof(T) == 4 && step && step % kAlone == 0) {
#pragma unroll
                for (unsigned mi = 0; mi < kMi; ++mi)
#pragma unroll
                    for (unsigned ni = 0; ni < kNi; ++ni) all[mi % (sizeof(T) == 4 ? kMi : 1)][ni] += acc[mi][ni], acc[mi][ni] = v4f{};
            }
#pragma unroll
            for (unsigned g = 0; g < kGroups; ++g) {
                if (g == kGroups - kAhead) {
                    land(other);
                    wait(step + STAGES <= steps, STAGES - 2);
                    __syncthreads();
                    if (step + STAGES < steps) fetch(buffer, step + STAGES);
                    __builtin_amdgcn_sched_barrier(0);
                }
                // (behind the last step: what LDS happens to hold, unused)
                const unsigned from = g < kGroups - kAhead ? buffer : other;
                read_a(from, (g + kAhead) % kGroups);
                // the other half step's pieces of B, spread over the groups in front of it
                if (g < kMi) {
#pragma unroll
                    for (unsigned ni = 0; ni < kNi; ++ni)
                        if (kMi - kAhead <= g && ni * kAhead / kNi == g - (kMi - kAhead)) read_b(buffer, 1, ni);
                } else if (g >= kGroups - kAhead) {
#pragma unroll
                    for (unsigned ni = 0; ni < kNi; ++ni)
                        if (ni * kAhead / kNi == g - (kGroups - kAhead)) read_b(other, 0, ni);
                }
#pragma unroll
                for (unsigned ni = 0; ni < kNi; ++ni) acc[g % kMi][ni] = Mma<T>::step(fb[g / kMi][ni], fa[g % (2 * kAhead)], acc[g % kMi][ni]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (sizeof(T) == 4) {
#pragma unroll
            for (unsigned mi = 0; mi < kMi; ++mi)
#pragma unroll
                for (unsigned ni = 0; ni < kNi; ++ni) acc[mi][ni] += all[mi % (sizeof(T) == 4 ? kMi : 1)][ni];
        }
    }
};

// Wavefronts of a block lie in one or two rows of four.
template <unsigned BM>
constexpr unsigned tile_wave_rows() {
    return BM == 32 ? 1 : 2;
}

// Steps of a tile in LDS.
template <unsigned BM>
constexpr unsigned tile_stages() {
    return BM <= 64 ? 3 : 2;
}

template <typename T, int OP, unsigned BM, unsigned BN, bool DMA>
__global__ __launch_bounds__(tile_wave_rows<BM>() * 256, tile_wave_rows<BM>() * (sizeof(T) == 4 && BM == 128 && DMA ? 2 : 1)) void expert_tile_kernel(const ExpertArgs<T> args) {
    constexpr unsigned kWaveRows = tile_wave_rows<BM>();
    typedef TileSide<T, BM, a_by_k<OP>(), DMA, kWaveRows * 4> A;
    typedef TileSide<T, BN, b_by_k<OP>(), DMA, kWaveRows * 4> B;
    constexpr unsigned kMi = BM / 16 / kWaveRows, kNi = BN / 64, kStepK = A::kStepK;
    constexpr bool kWeights = OP == kDwIn || OP == kDwOut;  // D is a weight's gradient: k runs over rows
    constexpr unsigned kStages = DMA ? tile_stages<BM>() : 2;
    __shared__ __attribute__((aligned(1024))) char lds_a[kStages * A::kBytes];
    __shared__ __attribute__((aligned(1024))) char lds_b[kStages * B::kBytes];
    __shared__ TileList list;
    const unsigned wave = wave_of_block(), lane = threadIdx.x % kLanes;
    const unsigned dim = args.dim, hidden = args.hidden;
    const unsigned n_all = OP == kIn || OP == kDh || OP == kDwOut ? hidden : dim, n_tile = OP == kIn ? BN / 2 : BN;
    const unsigned wide = (n_all + n_tile - 1) / n_tile;
    const unsigned m_all = OP == kDwIn ? 2 * hidden : dim;  // of a weight's gradient
    const unsigned lda = OP == kIn || OP == kDh || OP == kDwOut ? dim : OP == kOut ? hidden : 2 * hidden;
    const unsigned ldb = OP == kIn || OP == kDx || OP == kDwIn ? dim : hidden;
    const unsigned high_w = (m_all + BM - 1) / BM;
    if (!kWeights) list.template make<kWaveRows * 4>(args.expert_row, args.stride, args.cap, args.experts, args.npes, BM, wide, args.more_than);
    const unsigned total = kWeights ? args.experts * args.npes * high_w * wide : list.total();
    const TileProduct<T, A, B, kMi, kNi, kStages> product = {(NVSHMEM_AMD_LDS char *)lds_a, (NVSHMEM_AMD_LDS char *)lds_b, wave, lane};
    A side_a;
    B side_b;
    for (unsigned i = 0;; ++i) {
        unsigned t = tile_of_block(i, total);
        if (t >= total) return;
        unsigned e;
        if (kWeights) {
            e = t / (high_w * wide);
            t -= e * high_w * wide;
        } else {
            e = list.find(t);
        }
        const unsigned pe = e / args.experts;
        e -= pe * args.experts;
        uint64_t first, rows;
        expert_range(copy_of(args.expert_row, pe, args.stride), e, args.cap, first, rows);
        first = scalar64(first), rows = scalar64(rows);
        unsigned tm, tn;
        const uint64_t high = kWeights ? high_w : (rows + BM - 1) / BM;
        if (t >= high * wide) continue;  // (a table whose ranges overlap many times over may count past 2^32)
        tile_place(t, (unsigned)high, wide, tm, tn);
        const uint64_t m0 = (uint64_t)tm * BM;
        const unsigned n0 = tn * n_tile;
        const uint64_t k_all = kWeights ? rows : OP == kOut ? hidden : OP == kDx ? 2 * hidden : dim;
        const uint64_t m_left = (kWeights ? m_all : rows) - m0;
        const unsigned m_here = m_left < BM ? (unsigned)m_left : BM, n_here = n_all - n0 < n_tile ? n_all - n0 : n_tile;
        // the operands' corners
        const T *a = OP == kIn ? args.rows : OP == kOut ? args.h : OP == kDh || OP == kDwOut ? args.dout : args.dpre;
        a = copy_of(a, pe, args.stride) + first * lda + (kWeights ? m0 : m0 * lda);
        const T *b = OP == kIn || OP == kDx ? args.w_in : OP == kOut || OP == kDh ? args.w_out : OP == kDwIn ? args.rows : args.h;
        b = copy_of(b, pe, args.stride);
        if (OP == kIn || OP == kDx) b += (uint64_t)e * 2 * hidden * dim;
        if (OP == kOut || OP == kDh) b += (uint64_t)e * hidden * dim;
        if (kWeights) b += first * ldb;
        b += b_by_k<OP>() ? (uint64_t)n0 : (uint64_t)n0 * ldb;
        const T *b_up = b + (uint64_t)hidden * dim;  // kIn: the same columns of up
        side_a.begin(wave, lane, m_here, lda, [](unsigned r) { return r; });
        // kIn: the first half of a wavefront's columns are gate's, the second half the same of up
        side_b.begin(wave, lane, n_here, ldb, [](unsigned r) { return OP == kIn ? r / (BN / 4) * (BN / 8) + r % (BN / 8) : r; });
        const auto fetch = [&](unsigned buffer, unsigned step) {
            const uint64_t k = (uint64_t)step * kStepK;
            const unsigned left = k_all - k < kStepK ? (unsigned)(k_all - k) : kStepK;
            side_a.fetch((NVSHMEM_AMD_LDS char *)lds_a + buffer * A::kBytes, wave, left, [&](unsigned) { return a + (a_by_k<OP>() ? k * lda : k); });
            side_b.fetch((NVSHMEM_AMD_LDS char *)lds_b + buffer * B::kBytes, wave, left, [&](unsigned j) {
                const bool up = OP == kIn && (wave * B::kMoves + j) * 8 % (BN / 4) >= BN / 8;
                return (up ? b_up : b) + (b_by_k<OP>() ? k * ldb : k);
            });
        };
        const auto land = [&](unsigned buffer) {
            side_a.land((NVSHMEM_AMD_LDS char *)lds_a + buffer * A::kBytes, wave, lane);
            side_b.land((NVSHMEM_AMD_LDS char *)lds_b + buffer * B::kBytes, wave, lane);
        };
        v4f acc[kMi][kNi] = {};
        const unsigned wm = wave / 4, wn = wave % 4, steps = (unsigned)((k_all + kStepK - 1) / kStepK);
        product.template start<DMA>(steps, fetch, land);
        product.template run<DMA>(steps, fetch, land, acc);
        // A lane has four consecutive columns of row lane % 16 of each 16 x 16 piece.
        const unsigned r = lane % 16, g = lane / 16;
        // kDh: gate and up of the next 16 rows are on their way while these are worked on
        typename Four<T>::vec kept[2][2][kNi];
        const auto load_kept = [&](unsigned mi) {
            const unsigned m = (wm * kMi + mi) * 16 + r;
            const T *from = copy_of(args.pre_in, pe, args.stride) + (first + m0 + (m < m_here ? m : m_here - 1)) * 2 * hidden + n0;
#pragma unroll
            for (unsigned ni = 0; ni < kNi; ++ni) {
                // (behind the last column: what lies there, unused)
                const unsigned at = wn * (BN / 4) + ni * 16 + g * 4, there = at < n_here ? at : n_here - 1;
                kept[mi % 2][0][ni] = *(const typename Four<T>::vec_unaligned *)(from + there);
                kept[mi % 2][1][ni] = *(const typename Four<T>::vec_unaligned *)(from + hidden + there);
            }
        };
        if (OP == kDh) load_kept(0);
#pragma unroll
        for (unsigned mi = 0; mi < kMi; ++mi) {
            const unsigned m = (wm * kMi + mi) * 16 + r;
            if (OP == kDh && mi + 1 < kMi) load_kept(mi + 1);
            if (m >= m_here) continue;
            const uint64_t row = kWeights ? m0 + m : first + m0 + m;
            if (OP == kIn) {
                v4f h[kNi / 2];
#pragma unroll
                for (unsigned ni = 0; ni < kNi / 2; ++ni) {
                    const v4f gate = acc[mi][ni], up = acc[mi][ni + kNi / 2];
#pragma unroll
                    for (int i = 0; i < 4; ++i) h[ni][i] = gate[i] * sigmoid(gate[i]) * up[i];
                }
                const unsigned c = wn * (BN / 8);
                T *to = copy_of(args.h, pe, args.stride) + row * hidden + n0, *pre = copy_of(args.pre, pe, args.stride) + row * 2 * hidden + n0;
                if constexpr (kNi == 4) {
                    store_32(to, c, h[0], h[1], n_here, lane);
                    if (args.pre) {
                        store_32(pre, c, acc[mi][0], acc[mi][1], n_here, lane);
                        store_32(pre + hidden, c, acc[mi][2], acc[mi][3], n_here, lane);
                    }
                } else if (c + g * 4 < n_here) {
                    store_four(to + c + g * 4, h[0], n_here - c - g * 4);
                    if (args.pre) {
                        store_four(pre + c + g * 4, acc[mi][0], n_here - c - g * 4);
                        store_four(pre + hidden + c + g * 4, acc[mi][1], n_here - c - g * 4);
                    }
                }
                continue;
            }
#pragma unroll
            for (unsigned ni = 0; ni < kNi; ni += 2) {
                const unsigned c = wn * (BN / 4) + ni * 16;
                if (OP == kDh) {
                    v4f dgate[2], dup[2], h[2];
#pragma unroll
                    for (unsigned half = 0; half < 2; ++half) {
                        const v4f gate = as_float<T>(kept[mi % 2][0][ni + half]), up = as_float<T>(kept[mi % 2][1][ni + half]), dh = acc[mi][ni + half];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float s = sigmoid(gate[i]), silu = gate[i] * s;
                            h[half][i] = silu * up[i];
                            dup[half][i] = dh[i] * silu;
                            dgate[half][i] = dh[i] * up[i] * (s + silu * (1.0f - s));
                        }
                    }
                    T *dpre = copy_of(args.dpre, pe, args.stride) + row * 2 * hidden + n0;
                    store_32(dpre, c, dgate[0], dgate[1], n_here, lane);
                    store_32(dpre + hidden, c, dup[0], dup[1], n_here, lane);
                    store_32(copy_of(args.h, pe, args.stride) + row * hidden + n0, c, h[0], h[1], n_here, lane);
                } else {
                    T *to = OP == kDwIn ? copy_of(args.dw_in, pe, args.stride) + ((uint64_t)e * 2 * hidden + row) * dim
                          : OP == kDwOut ? copy_of(args.dw_out, pe, args.stride) + ((uint64_t)e * dim + row) * hidden
                                         : copy_of(OP == kOut ? args.out : args.drows, pe, args.stride) + row * dim;
                    store_32(to + n0, c, acc[mi][ni], acc[mi][ni + 1], n_here, lane);
                }
            }
        }
    }
}

// As many blocks as have room on a compute unit take tiles as long as there are any.
inline unsigned tile_blocks(uint64_t tiles, unsigned blocks_per_cu) {
    const uint64_t most = 256 * blocks_per_cu;
    return (unsigned)((tiles < most ? tiles : most) + 7) / 8 * 8;
}

// Tiles of a product, if each expert had as many rows as any could at most on average.
template <typename T, int OP>
inline uint64_t tiles_of(const ExpertArgs<T> &args, uint64_t bm, uint64_t bn) {
    const uint64_t n_all = OP == kIn || OP == kDh || OP == kDwOut ? args.hidden : args.dim;
    const uint64_t m_all = OP == kDwIn ? 2 * (uint64_t)args.hidden : OP == kDwOut ? args.dim : (args.cap + args.experts - 1) / args.experts;
    return (uint64_t)args.experts * args.npes * ((m_all + bm - 1) / bm) * ((n_all * (OP == kIn ? 2 : 1) + bn - 1) / bn);
}

template <typename T, int OP, unsigned BM, unsigned BN, bool DMA>
inline void launch_tiles_as(const ExpertArgs<T> &args, hipStream_t stream) {
    // (of `cap` rows in all, every expert has at most one tile that is not full)
    const uint64_t n_all = OP == kIn || OP == kDh || OP == kDwOut ? args.hidden : args.dim, wide = div_up(n_all, OP == kIn ? BN / 2 : BN);
    const uint64_t high = OP == kDwIn || OP == kDwOut ? args.experts * (uint64_t)div_up(OP == kDwIn ? 2 * (uint64_t)args.hidden : args.dim, BM)
                                                      : args.cap / BM + (args.experts < args.cap ? args.experts : args.cap);
    const uint64_t tiles = high * wide * args.npes;
    if (tiles) launch_kernel((expert_tile_kernel<T, OP, BM, BN, DMA>), dim3(tile_blocks(tiles, BN == 256 ? 1 : DMA || BM == 128 ? 2 : 3)), dim3(tile_wave_rows<BM>() * 256), 0, stream, args);
}
// Large tiles read the least, small ones waste less on experts of few rows, have more steps on their way to LDS at a time, and two blocks of
// a compute unit, of which one multiplies while the other stores.  What an expert may have on average by the buffers' capacity, `rows`, is all
// that the host knows of the rows, and what the limits are in.  In the following the rows are those that came; there is room for a quarter more
// and for 64 a PE (of 12: 23, of 57 in all: 10 each, of 300: 383).  us of the forward pass, 256 x 256 / 128 x 128 / 64 x 128 / 32 x 128:
//   bf16, 64 experts of 4096 x 1536 with 12 rows each - / 436 / 414 / 454, 40: - / 461 / 468 / 548; 57 rows for 64 experts of 7168 x 2048 - / 652 / 630 / 612;
//   8 rows for 8 experts of 2048 x 1408, too few for the larger tiles to fill the GPU: - / 41.8 / 28.2 / 26.9;
//   64 experts of 2048 x 1408 with 300 rows each 504 / 519, 600: 754 / 821; 32 of 7168 x 2048 with 180: 880 / 862, 600: 1776 / 1971.
//   fp32, 16 rows for 64 experts of 4096 x 1536 - / 671 / 370 / 218; 16 of 2048 x 1408 with 180 rows each 831 / 672 / 572, 600: 1648 / 1494 / 1401.
// A kernel without LDS for few rows, whose wavefronts split k, took 39 in the smallest of these and 501 in the first.
template <typename T, int OP, bool DMA>
inline void launch_expert_tiles(const ExpertArgs<T> &args, hipStream_t stream) {
    constexpr bool kWeights = OP == kDwIn || OP == kDwOut;
    const uint64_t rows = (args.cap + args.experts - 1) / args.experts;
    if constexpr (DMA && sizeof(T) == 2)
        if (rows > 448 && tiles_of<T, OP>(args, 256, 256) >= 256) return launch_tiles_as<T, OP, 256, 256, DMA>(args, stream);
    if constexpr (!kWeights) {
        const bool many = tiles_of<T, OP>(args, 128, 128) >= 256;
        if (rows <= 12 || ((sizeof(T) == 4 || !many) && (rows <= 40 || tiles_of<T, OP>(args, 64, 128) < 256)))
            return launch_tiles_as<T, OP, 32, 128, DMA>(args, stream);
        if (sizeof(T) == 4 || !many || rows <= 32) return launch_tiles_as<T, OP, 64, 128, DMA>(args, stream);
    }
    if constexpr (kWeights || sizeof(T) == 2) launch_tiles_as<T, OP, 128, 128, DMA>(args, stream);
}

// Products of one PE's experts may be at most so wide and high; their offsets inside a tile stay under 2^31 bytes.
constexpr size_t kMostFeatures = 65536;

inline int check_expert_sizes(Runtime &rt, const char *what, int experts, size_t dim, size_t hidden) {
    NVSHMEM_AMD_REFUSE(experts < 1 || experts > (int)kMostExperts, "%s: %d experts, outside [1, %u]", what, experts, kMostExperts);
    NVSHMEM_AMD_REFUSE(experts % rt.npes, "%s: %d experts on %d PEs, which have to have the same number each", what, experts, rt.npes);
    NVSHMEM_AMD_REFUSE(dim < 1 || dim > kMostFeatures, "%s: rows of %zu elements, outside [1, %zu]", what, dim, kMostFeatures);
    NVSHMEM_AMD_REFUSE(hidden < 1 || hidden > kMostFeatures, "%s: %zu hidden elements, outside [1, %zu]", what, hidden, kMostFeatures);
    return 0;
}
inline bool aligned16(const void *p) { return (uintptr_t)p % 16 == 0; }
inline uint64_t align_up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

}  // namespace tokens
}  // namespace nvshmem_amd
