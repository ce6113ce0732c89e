// A block's part of a stable counting sort: where each of its items goes, items of one bin in their order.
#pragma once

#include "token_common.hpp"

namespace nvshmem_amd {
namespace tokens {

constexpr unsigned kSortThreads = 1024, kSortWaves = kSortThreads / kLanes;

// Inclusive sum over the lanes of a wavefront.
__device__ __forceinline__ uint32_t scan_lanes(uint32_t x) {
    const unsigned lane = threadIdx.x % kLanes;
#pragma unroll
    for (int s = 1; s < kLanes; s <<= 1) {
        const uint32_t up = (uint32_t)__shfl_up((int)x, s);
        if (lane >= (unsigned)s) x += up;
    }
    return x;
}
// Sum over the threads in front of this one, of kSortThreads; wave_sum: kSortWaves words of LDS.  Ends behind a barrier.
__device__ __forceinline__ uint32_t scan_block(uint32_t x, uint32_t *wave_sum) {
    const unsigned wave = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
    const uint32_t upto = scan_lanes(x);
    if (lane == kLanes - 1) wave_sum[wave] = upto;
    __syncthreads();
    uint32_t before = 0;
#pragma unroll
    for (unsigned w = 0; w < kSortWaves; ++w)
        if (w < wave) before += wave_sum[w];
    return before + upto - x;
}

// Item i of a thread is number wave * ROUNDS * 64 + i * 64 + lane of the block's; bin[i] >= bins: no item.  On entry run[b] (LDS) is
// the place of the block's first item of bin b, on return of the first behind the block's.  count: kSortWaves x bins words of LDS.
// A wavefront ranks 64 items at a time by ballots over the bits of their bins, so nothing depends on the order of atomics.
// Begins behind a barrier of the caller's, ends without one.
template <unsigned ROUNDS>
__device__ __forceinline__ void stable_places(uint32_t (&place)[ROUNDS], const uint32_t (&bin)[ROUNDS], unsigned bins, uint32_t *run,
                                              uint32_t *count) {
    const unsigned wave = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
    uint32_t *mine = count + wave * bins;
    for (unsigned i = lane; i < bins; i += kLanes) mine[i] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (unsigned i = 0; i < ROUNDS; ++i)
        if (bin[i] < bins) atomicAdd(&mine[bin[i]], 1u);
    __syncthreads();
    for (unsigned b = threadIdx.x; b < bins; b += kSortThreads) {
        uint32_t n[kSortWaves], at = run[b];
#pragma unroll
        for (unsigned w = 0; w < kSortWaves; ++w) n[w] = count[w * bins + b];
#pragma unroll
        for (unsigned w = 0; w < kSortWaves; ++w) {
            count[w * bins + b] = at;
            at += n[w];
        }
        run[b] = at;
    }
    __syncthreads();
    const unsigned bits = 32 - __builtin_clz(bins);
#pragma unroll
    for (unsigned i = 0; i < ROUNDS; ++i) {
        const bool some = bin[i] < bins;
        uint64_t same = __builtin_amdgcn_ballot_w64(some);  // the lanes with an item of this lane's bin
        for (unsigned b = 0; b < bits; ++b) {
            const bool bit = bin[i] >> b & 1;
            const uint64_t set = __builtin_amdgcn_ballot_w64(bit);
            same &= bit ? set : ~set;
        }
        const unsigned rank = (unsigned)__builtin_popcountll(same & ((1ull << lane) - 1)), n = (unsigned)__builtin_popcountll(same);
        if (some) place[i] = mine[bin[i]] + rank;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (some && rank + 1 == n) mine[bin[i]] = place[i] + 1;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

}  // namespace tokens
}  // namespace nvshmem_amd
