// The experts' two products for experts that have few rows, as in steps of single tokens: weights are read once, straight into
// registers, and are what bounds them.
#pragma once

#include "expert_tiles.hpp"

namespace nvshmem_amd {
namespace tokens {

// Experts of more rows are the tiles'.
constexpr unsigned kFewRows = 32;
constexpr unsigned kFewWaves = 4, kFewThreads = kFewWaves * kLanes;
constexpr unsigned kFewColumns = 64;  // rows of weights that a block reads: kIn: 32 of gate and the same 32 of up

// Weights of T: a wavefront takes 64 of their rows and 128 bytes of k at a time.  Lane (r, g) has of each of four groups of 16 rows the
// g-th and the (g + 4)-th piece of 16 bytes of row r, and the same of x.
template <typename T>
struct PlainWeights {
    static constexpr unsigned kN = 16 / sizeof(T), kStepK = kStepBytes / sizeof(T);
    const T *base[2];  // the first of the block's rows: gate (or all), up
    unsigned ld, k_all;
    unsigned row[4];   // this lane's of each group, from its base

    template <int MT>
    struct Stage {
        v4u w[4][2], x[MT][2];
    };
    template <bool WHOLE, int MT>
    __device__ __forceinline__ void load(Stage<MT> &s, const T *const (&x)[MT], unsigned k, unsigned lane) const {
        const unsigned g = lane / 16;
#pragma unroll
        for (unsigned h = 0; h < 2; ++h) {
            const unsigned at = k + (h * 4 + g) * kN, n = at < k_all ? (k_all - at < kN ? k_all - at : kN) : 0;
#pragma unroll
            for (unsigned ni = 0; ni < 4; ++ni) {
                const T *p = base[ni / 2] + row[ni] * ld + at;
                s.w[ni][h] = WHOLE ? __builtin_bit_cast(v4u, chunk_load_stream(p)) : chunk_load_front(p, n);
            }
#pragma unroll
            for (int mi = 0; mi < MT; ++mi) s.x[mi][h] = WHOLE ? __builtin_bit_cast(v4u, chunk_load(x[mi] + at)) : chunk_load_front(x[mi] + at, n);
        }
    }
    template <int MT>
    __device__ __forceinline__ void multiply(const Stage<MT> &s, v4f (&acc)[MT][4]) const {
#pragma unroll
        for (unsigned h = 0; h < 2; ++h)
#pragma unroll
            for (int mi = 0; mi < MT; ++mi)
#pragma unroll
                for (unsigned ni = 0; ni < 4; ++ni) acc[mi][ni] = Mma<T>::step(s.x[mi][h], s.w[ni][h], acc[mi][ni]);
    }
};

// One block has 64 rows of one expert's weights; its four wavefronts take steps of k in turn, each with the loads of its next step on
// their way while it multiplies, and their sums are added up in their order.
// D = x w^T: element i of a lane is row lane / 16 * 4 + i of x, column lane % 16.
template <typename W, typename T, int MT>
__device__ __forceinline__ void few_rows_sum(const W &weights, const T *x, unsigned ldx, unsigned rows, float (*part)[MT * 16][kFewColumns + 4]) {
    const unsigned wave = wave_of_block(), lane = threadIdx.x % kLanes;
    const T *from[MT];
#pragma unroll
    for (int mi = 0; mi < MT; ++mi) {
        const unsigned m = mi * 16 + lane % 16;
        from[mi] = x + (uint64_t)(m < rows ? m : rows - 1) * ldx;  // (what the last row gives in other rows' places goes nowhere)
    }
    v4f acc[MT][4] = {};
    const unsigned whole = weights.k_all / W::kStepK;
    typename W::template Stage<MT> even, odd;
    if (wave < whole) weights.template load<true>(even, from, wave * W::kStepK, lane);
    for (unsigned i = wave; i < whole; i += 2 * kFewWaves) {
        if (i + kFewWaves < whole) weights.template load<true>(odd, from, (i + kFewWaves) * W::kStepK, lane);
        weights.multiply(even, acc);
        if (i + kFewWaves >= whole) break;
        if (i + 2 * kFewWaves < whole) weights.template load<true>(even, from, (i + 2 * kFewWaves) * W::kStepK, lane);
        weights.multiply(odd, acc);
    }
    if (weights.k_all % W::kStepK && wave == whole % kFewWaves) {
        weights.template load<false>(even, from, whole * W::kStepK, lane);
        weights.multiply(even, acc);
    }
#pragma unroll
    for (int mi = 0; mi < MT; ++mi)
#pragma unroll
        for (unsigned ni = 0; ni < 4; ++ni)
#pragma unroll
            for (unsigned i = 0; i < 4; ++i) part[wave][mi * 16 + lane / 16 * 4 + i][ni * 16 + lane % 16] = acc[mi][ni][i];
    __syncthreads();
}
template <int MT>
__device__ __forceinline__ v4f few_rows_total(float (*part)[MT * 16][kFewColumns + 4], unsigned m, unsigned c) {
    v4f sum = *(const v4f *)&part[0][m][c];
#pragma unroll
    for (unsigned w = 1; w < kFewWaves; ++w) sum += *(const v4f *)&part[w][m][c];
    return sum;
}

// What a block does with the sums: kIn's activation, or kOut's rows.
template <typename T, int OP, int MT>
__device__ __forceinline__ void few_rows_store(const ExpertArgs<T> &args, float (*part)[MT * 16][kFewColumns + 4], unsigned pe, uint64_t first,
                                               unsigned rows, unsigned n0) {
    const unsigned hidden = args.hidden;
    constexpr unsigned kFours = OP == kIn ? 8 : 16;
    const unsigned n_all = OP == kIn ? hidden : args.dim;
    for (unsigned i = threadIdx.x; i < rows * kFours; i += kFewThreads) {
        const unsigned m = i / kFours, c = i % kFours * 4, n = n0 + c;
        if (n >= n_all) continue;
        const uint64_t row = first + m;
        if (OP == kIn) {
            const v4f gate = few_rows_total<MT>(part, m, c), up = few_rows_total<MT>(part, m, c + 32);
            v4f h;
#pragma unroll
            for (int j = 0; j < 4; ++j) h[j] = gate[j] * sigmoid(gate[j]) * up[j];
            store_four(copy_of(args.h, pe, args.stride) + row * hidden + n, h, n_all - n);
            if (args.pre) {
                T *pre = copy_of(args.pre, pe, args.stride) + row * 2 * hidden + n;
                store_four(pre, gate, n_all - n);
                store_four(pre + hidden, up, n_all - n);
            }
        } else {
            store_four(copy_of(args.out, pe, args.stride) + row * args.dim + n, few_rows_total<MT>(part, m, c), n_all - n);
        }
    }
}

// SETUP makes the block's weights: setup(e, n0) -> W.
template <typename W, typename T, int OP, typename SETUP>
__device__ __forceinline__ void few_rows_block(const ExpertArgs<T> &args, SETUP setup) {
    __shared__ __attribute__((aligned(16))) float part[kFewWaves][kFewRows][kFewColumns + 4];
    const unsigned pe = blockIdx.z, e = blockIdx.y, n0 = blockIdx.x * (OP == kIn ? kFewColumns / 2 : kFewColumns);
    uint64_t first, rows;
    expert_range(copy_of(args.expert_row, pe, args.stride), e, args.cap, first, rows);
    if (rows == 0 || rows > kFewRows) return;
    const unsigned ldx = OP == kIn ? args.dim : args.hidden;
    const T *x = copy_of(OP == kIn ? args.rows : (const T *)args.h, pe, args.stride) + first * ldx;
    W weights;
    setup(weights, pe, e, n0);
    if (rows <= 16) {
        float(*p)[16][kFewColumns + 4] = (float(*)[16][kFewColumns + 4])part;
        few_rows_sum<W, T, 1>(weights, x, ldx, (unsigned)rows, p);
        few_rows_store<T, OP, 1>(args, p, pe, first, (unsigned)rows, n0);
    } else {
        few_rows_sum<W, T, 2>(weights, x, ldx, (unsigned)rows, part);
        few_rows_store<T, OP, 2>(args, part, pe, first, (unsigned)rows, n0);
    }
}

// Row of the weights that lane % 16 has of group ni, from the block's first; rows behind the last are the last one again.
template <int OP>
__device__ __forceinline__ unsigned few_rows_row(unsigned ni, unsigned lane, unsigned n_left) {
    const unsigned r = (OP == kIn ? ni % 2 : ni) * 16 + lane % 16;
    return r < n_left ? r : n_left - 1;
}

template <typename T, int OP>
__global__ __launch_bounds__(kFewThreads) void expert_few_kernel(const ExpertArgs<T> args) {
    few_rows_block<PlainWeights<T>, T, OP>(args, [&](PlainWeights<T> &w, unsigned pe, unsigned e, unsigned n0) {
        const unsigned n_all = OP == kIn ? args.hidden : args.dim, ld = OP == kIn ? args.dim : args.hidden;
        const T *p = copy_of(OP == kIn ? args.w_in : args.w_out, pe, args.stride) + (uint64_t)e * (OP == kIn ? 2 : 1) * args.hidden * args.dim;
        w.base[0] = p + (uint64_t)n0 * ld;
        w.base[1] = OP == kIn ? w.base[0] + (uint64_t)args.hidden * args.dim : w.base[0];
        w.ld = ld, w.k_all = ld;
        for (unsigned ni = 0; ni < 4; ++ni) w.row[ni] = few_rows_row<OP>(ni, threadIdx.x % kLanes, n_all - n0);
    });
}

template <int OP, typename T>
inline dim3 few_rows_grid(const ExpertArgs<T> &args, int npes) {
    return dim3(div_up(OP == kIn ? args.hidden : args.dim, OP == kIn ? kFewColumns / 2 : kFewColumns), args.experts, npes);
}

}  // namespace tokens
}  // namespace nvshmem_amd
