// Embedding lookup with scaling from a table that is cut by rows over the PEs, and the table's gradient.
//
//   out@p[t] = scale * table@(v / R)[v % R]           v = ids@p[t], R = ceil(vocab / npes) rows of the table on each PE
//   dtable@(v / R)[v % R] = scale * sum dout@p[t]     over all (p, t) with ids@p[t] = v
//
// The sum's terms are taken in the order of (p, t), but added up in partial sums whose ends follow from the ids of the whole batch.
// An id outside [0, vocab) is padding: a row of zeros, no gradient.
#include "counting_sort.hpp"
#include "token_common.hpp"

namespace nvshmem_amd {
namespace tokens {
namespace {

// One wavefront per piece of V x 64 chunks of a row; a row of fewer chunks than a wavefront has lanes takes the next power of two of
// them and shares the wavefront with others (2^lanes_log lanes a row).  Reads a row of the table and writes one: bound by memory, and
// for short rows by the rate at which wavefronts start, so there one has TOKENS tokens (or TOKENS for each row's lanes).
// Where a wavefront has whole tokens, their ids are scalar loads and their rows scalar addresses.
// us, bf16, of 100003 rows by a Zipf distribution.  8 x 4096 rows of 7168 (0.47 GB written, 0.16 GB of distinct rows: 113 us are 5.6 TB/s of
// what is needed; 0.29 GB are read, as every XCD's L2 fetches a popular row for itself, which makes 6.7 of what is moved): one chunk a lane
// 141, two 120, four (of 14) 130, seven 116; two, written through to memory 113.  8 x 64 rows: 4.4, written through 4.0.
// Rows of up to four pieces of 64 chunks are one wavefront's, against two pieces each: 8 x 20000 rows of 1152 92 / 137, of 2048 177 / 167;
// of 16000 rows, which the Infinity Cache holds, 71 / 139 and 127 / 150.
// One / four tokens a wavefront: 8 x 5970 rows of 512 (47760 wavefronts of one) 22.0 / 12.2, 8 x 600 (4800) 4.0 / 3.5, 8 x 64 (512)
// 2.3 / 2.7; 8 x 5970 rows of 64 (5976) 5.0 / 3.9, 8 x 2100 (2104) 3.3 / 3.4.  Two tokens for rows of 900: 14.6 / 15.1, not taken.
constexpr uint64_t kManyWaves = 4096;
template <typename T, int V, int TOKENS, int MODE>
__global__ __launch_bounds__(64) void embedding_kernel(T *__restrict__ out, const T *__restrict__ table, const int64_t *__restrict__ ids,
                                                       uint64_t stride, unsigned tokens, unsigned vocab, unsigned rows, unsigned dim,
                                                       unsigned lanes_log, float scale) {
    typedef typename Chunk<T>::vec vec;
    const unsigned lane = threadIdx.x, pe = blockIdx.z, log = MODE == kWhole ? 6 : lanes_log, per_wave = kLanes >> log;
    unsigned first[V];
    bool mine[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const unsigned c = (blockIdx.x * V + v) * kLanes + (lane & ((1u << log) - 1));
        first[v] = chunk_first<T>(c, dim), mine[v] = c * Chunk<T>::N < dim;
    }
    if (!mine[0]) return;
    const int64_t *my_ids = copy_of(ids, pe, stride);
    T *my_out = copy_of(out, pe, stride);
    for (uint64_t t0 = (uint64_t)blockIdx.y * per_wave * TOKENS + (MODE == kWhole ? 0 : lane >> log); t0 < tokens;
         t0 += (uint64_t)gridDim.y * per_wave * TOKENS) {
        uint64_t id[TOKENS];
#pragma unroll
        for (int i = 0; i < TOKENS; ++i) id[i] = (uint64_t)my_ids[t0 + i * per_wave < tokens ? t0 + i * per_wave : t0];
        vec x[TOKENS][V] = {};
#pragma unroll
        for (int i = 0; i < TOKENS; ++i) {
            if (id[i] >= vocab) continue;
            const unsigned owner = (unsigned)id[i] / rows, row = (unsigned)id[i] % rows;
            const T *src = copy_of(table, owner, stride) + (uint64_t)row * dim;
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (MODE == kTiny) x[i][v] = chunk_load_part(src, dim);
                else if (v == 0 || mine[v]) x[i][v] = chunk_load(src + first[v]);
        }
#pragma unroll
        for (int i = 0; i < TOKENS; ++i) {
            const uint64_t t = t0 + i * per_wave;
            if (t >= tokens) break;
            T *dst = my_out + t * dim;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const vec y = chunk_from_float<T>(chunk_to_float<T>(x[i][v]) * (id[i] < vocab ? scale : 0.0f));
                if (MODE == kTiny) chunk_store_part(dst, y, dim);
                else if (v == 0 || mine[v]) chunk_store_through(dst + first[v], y);
            }
        }
    }
}

// ---- gradient ----
// The tokens of all PEs are sorted by id, stable; a wavefront adds up a part of consecutive ones, of a piece of a row, in order, and
// writes the sums of the ids that lie in its part as a whole.  A sum that goes on into the next part leaves a partial sum in fp32
// (`carry`), and a kernel behind it adds those up, in order: nothing depends on which block comes first.
// Parts are short where there are few wavefronts, long where there are many, as sums that go on cost a partial sum per part.  us
// for sums | partial sums joined, parts of 8 / 32 / 64: 608 tokens of 515 fp32 13.5 / 19.7 / 29.0 | 4; 32768 of 7168 bf16 - / 330 / 330 | - /
// 16.8 / 10.4; 8192 of 64 bf16 7.6 / 21.0 / - | 4.
constexpr unsigned kLeastPart = 8, kMostPart = kLanes, kPiece = 512, kPartPieces = 4096;
unsigned part_of(uint64_t n, uint64_t dim) {
    const uint64_t pieces = (dim + kPiece - 1) / kPiece;
    unsigned part = kLeastPart;
    while (part < kMostPart && n * pieces / kPartPieces > part) part *= 2;
    return part;
}

// A token: its id (vocab: padding, sorted behind all ids) and its number pe * tokens + t.
struct Item {
    uint32_t key, pos;
};
__device__ __forceinline__ uint32_t key_of(const int64_t *ids, uint64_t stride, unsigned tokens, unsigned vocab, unsigned i) {
    const uint64_t id = (uint64_t)copy_of(ids, i / tokens, stride)[i % tokens];
    return id < vocab ? (uint32_t)id : vocab;
}

// Up to kRankTokens tokens: a token's place in the sorted order is the number of smaller ones.  A block of 16 wavefronts counts it for
// 32 tokens, two lanes each; a lane goes through a thirty-second of all tokens, four at a time.  Quadratic, but one launch; what bounds
// it is LDS, which half the keys to a block, in twice the blocks, halves.  us here / by digits: 608 tokens 3.6 / -, 8192 10.9 / about 20,
// 16384 26.8 / 20.8 (and three more launches).
constexpr unsigned kRankTokens = 12288, kRankKeys = kLanes / 2;

__global__ __launch_bounds__(kSortThreads) void embedding_rank_kernel(Item *sorted, const int64_t *ids, uint64_t stride,
                                                                      unsigned tokens, unsigned n, unsigned vocab) {
    extern __shared__ __align__(16) uint32_t all[];  // n, rounded up to 64
    __shared__ uint32_t smaller[kRankKeys];
    const unsigned wave = threadIdx.x / kLanes, lane = threadIdx.x % kRankKeys, half = threadIdx.x % kLanes / kRankKeys;
    const unsigned padded = (n + 63) / 64 * 64, block = blockIdx.x * kRankKeys;
#pragma unroll 8
    for (unsigned i = threadIdx.x; i < padded; i += kSortThreads) all[i] = i < n ? key_of(ids, stride, tokens, vocab, i) : 0xffffffffu;
    if (threadIdx.x < kRankKeys) smaller[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t mine = all[block + lane];
    unsigned rank = 0;
    // 32 keys at a time; those in front of this block's count when they are equal
    for (unsigned j0 = wave * kLanes + half * kRankKeys; j0 < padded; j0 += kSortThreads) {
        if (j0 == block) {
            for (unsigned j = 0; j < kRankKeys; ++j) rank += all[block + j] < mine + (j < lane);
            continue;
        }
        const uint32_t limit = mine + (j0 < block);
#pragma unroll
        for (unsigned j = 0; j < kRankKeys; j += 4) {
            const uint4 k = *(const uint4 *)(all + j0 + j);
            rank += (k.x < limit) + (k.y < limit) + (k.z < limit) + (k.w < limit);
        }
    }
    atomicAdd(&smaller[lane], rank);
    __syncthreads();
    if (threadIdx.x < kRankKeys && block + lane < n) sorted[smaller[lane]] = {mine, block + lane};
}

// More tokens: counting sorts by kDigit bits of the id at a time, lowest first, of at most kSortBlocks blocks of consecutive tokens.
// Not much data, all waiting: 32768 tokens, 17 bits: counts 4.6 and 4.8 us, sorts 7.9 and 8.4.
constexpr unsigned kDigit = 9, kBins = 1u << kDigit, kSortBlocks = 64, kSortRounds = 2, kSortTile = kSortThreads * kSortRounds;

template <bool FIRST>
__device__ __forceinline__ Item item_of(const Item *in, const int64_t *ids, uint64_t stride, unsigned tokens, unsigned vocab,
                                        unsigned i) {
    if (FIRST) return {key_of(ids, stride, tokens, vocab, i), i};
    return in[i];
}

template <bool FIRST>
__global__ __launch_bounds__(kSortThreads) void embedding_count_kernel(uint32_t *hist, const Item *in, const int64_t *ids,
                                                                       uint64_t stride, unsigned tokens, unsigned n, unsigned vocab,
                                                                       unsigned per_block, unsigned shift) {
    __shared__ uint32_t count[kBins];
    if (threadIdx.x < kBins) count[threadIdx.x] = 0;
    __syncthreads();
    const uint64_t begin = (uint64_t)blockIdx.x * per_block, end = begin + per_block < n ? begin + per_block : n;
    for (uint64_t i = begin + threadIdx.x; i < end; i += kSortThreads)
        atomicAdd(&count[item_of<FIRST>(in, ids, stride, tokens, vocab, (unsigned)i).key >> shift & (kBins - 1)], 1u);
    __syncthreads();
    if (threadIdx.x < kBins) hist[blockIdx.x * kBins + threadIdx.x] = count[threadIdx.x];
}

template <bool FIRST>
__global__ __launch_bounds__(kSortThreads) void embedding_sort_kernel(Item *out, const uint32_t *hist, const Item *in,
                                                                      const int64_t *ids, uint64_t stride, unsigned tokens, unsigned n,
                                                                      unsigned vocab, unsigned per_block, unsigned shift) {
    __shared__ uint32_t count[kSortWaves * kBins], run[kBins], wave_sum[kSortWaves], half[2][kBins];
    const uint64_t begin = (uint64_t)blockIdx.x * per_block, end = begin + per_block < n ? begin + per_block : n;
    Item item[kSortRounds];
    uint32_t to[kSortRounds], place[kSortRounds];
    auto fetch = [&](uint64_t tile) {
#pragma unroll
        for (unsigned r = 0; r < kSortRounds; ++r) {
            const uint64_t i = tile + threadIdx.x / kLanes * (kSortRounds * kLanes) + r * kLanes + threadIdx.x % kLanes;
            item[r] = i < end ? item_of<FIRST>(in, ids, stride, tokens, vocab, (unsigned)i) : Item{0, 0};
            to[r] = i < end ? item[r].key >> shift & (kBins - 1) : kBins;
        }
    };
    fetch(begin);  // (in flight while the counts are)
    // items of each bin in all blocks, and in those before this one: two threads a bin
    const unsigned bin = threadIdx.x % kBins;
    uint32_t total = 0, before = 0;
#pragma unroll 16
    for (unsigned b = threadIdx.x / kBins; b < gridDim.x; b += kSortThreads / kBins) {
        const uint32_t c = hist[b * kBins + bin];
        total += c;
        before += b < blockIdx.x ? c : 0;
    }
    if (threadIdx.x >= kBins) {
        half[0][bin] = total;
        half[1][bin] = before;
    }
    __syncthreads();
    const bool first = threadIdx.x < kBins;
    total = first ? total + half[0][bin] : 0;
    const uint32_t start = scan_block(total, wave_sum);
    if (first) run[bin] = start + before + half[1][bin];
    for (uint64_t tile = begin; tile < end; tile += kSortTile) {
        if (tile != begin) fetch(tile);
        __syncthreads();
        stable_places<kSortRounds>(place, to, kBins, run, count);
#pragma unroll
        for (unsigned r = 0; r < kSortRounds; ++r)
            if (to[r] < kBins) out[place[r]] = item[r];
        __syncthreads();
    }
}

template <typename T>
__device__ __forceinline__ void write_row(T *dtable, uint64_t stride, uint32_t key, unsigned rows, unsigned dim, unsigned first,
                                          typename Chunk<T>::facc sum, float scale) {
    T *dst = copy_of(dtable, key / rows, stride) + (uint64_t)(key % rows) * dim + first;
    const typename Chunk<T>::vec y = chunk_from_float<T>(sum * scale);
    if (dim < (unsigned)Chunk<T>::N) chunk_store_part(dst, y, dim);
    else chunk_store_stream(dst, y);
}
// A partial sum's chunk, at any element.
template <typename T>
struct Partial {
    typedef typename Chunk<T>::facc type __attribute__((aligned(4)));
};

struct SumArgs {
    const Item *sorted;
    float *carry;
    uint64_t stride;
    unsigned tokens, n, part, parts, vocab, rows, dim, pitch, pieces, sum_blocks;
    float scale;
};

// `elems` zeros at p by a wavefront: elements up to a 16-byte boundary, vectors, elements.
template <typename T>
__device__ __forceinline__ void zero_fill(T *p, uint64_t elems) {
    const unsigned lane = threadIdx.x;
    const uint64_t head = ((16 - (uintptr_t)p % 16) % 16) / sizeof(T);
    if (elems < head + Chunk<T>::N) {
        for (uint64_t i = lane; i < elems; i += kLanes) p[i] = (T)0.0f;
        return;
    }
    if (lane < head) p[lane] = (T)0.0f;
    typedef typename Chunk<T>::vec vec;
    vec *v = (vec *)(p + head);
    const uint64_t n = (elems - head) / Chunk<T>::N, tail = head + n * Chunk<T>::N;
    for (uint64_t i = lane; i < n; i += kLanes) v[i] = vec{};
    if (lane < elems - tail) p[tail + lane] = (T)0.0f;
}

// Loads of a wavefront's rows that are in flight together.  us of the kernel below with eight / sixteen: 8 x 4096 tokens of 7168 bf16, 100003
// rows, 307 to 320 / 306, 8 x 6081 of 1088 62.0 to 63.4 / 60.6, 8 x 500 of 8000, 1000 rows, 33 / 32, 608 of 515 fp32 13.2 / 13.0: the spread
// between processes and little more, and sixteen take 100 registers, eight 68.  (Four: 335 where eight took 330.)
constexpr unsigned kAhead = 8;

template <typename T>
__device__ __forceinline__ void embedding_sum_part(T *dtable, const T *dout, const SumArgs &a, unsigned part, unsigned piece) {
    constexpr unsigned N = Chunk<T>::N;
    typedef typename Chunk<T>::facc facc;
    const unsigned lane = threadIdx.x, c = piece * kLanes + lane, first = chunk_first<T>(c, a.dim);
    const bool mine = c * N < a.dim, row_part = a.dim < N;
    const unsigned begin = part * a.part, here = a.n - begin < a.part ? a.n - begin : a.part;
    // lane j looks at item j: where its row is, and whether it is the last of its id
    Item item = {a.vocab, 0};
    uint32_t after = a.vocab, prior = a.vocab;
    if (lane < here) item = a.sorted[begin + lane];
    if (begin + here < a.n) after = a.sorted[begin + here].key;  // the item behind the part, and the one in front
    if (begin > 0) prior = a.sorted[begin - 1].key;
    const uint64_t off = (uint64_t)(item.pos / a.tokens) * a.stride + (uint64_t)(item.pos % a.tokens) * a.dim * sizeof(T);
    const uint32_t next = (uint32_t)__shfl_down((int)item.key, 1);
    const bool padding = item.key >= a.vocab;
    const uint64_t last = __builtin_amdgcn_ballot_w64(!padding && (lane + 1 >= here || next != item.key));
    const unsigned count = kLanes - __builtin_clzll(last | 1);  // items up to the last that is no padding
    if (!last) return;
    const bool goes_on = count == here && after == (uint32_t)__builtin_amdgcn_readlane((int)item.key, here - 1);
    const bool came = prior == (uint32_t)__builtin_amdgcn_readlane((int)item.key, 0);
    facc sum = {};
    bool from_before = came;
    for (unsigned j0 = 0; j0 < count; j0 += kAhead) {
        typename Chunk<T>::vec x[kAhead];
#pragma unroll
        for (unsigned u = 0; u < kAhead; ++u) {
            if (j0 + u >= count) break;
            const uint64_t o = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(off >> 32), j0 + u) << 32 |
                               (uint32_t)__builtin_amdgcn_readlane((int)off, j0 + u);
            const T *src = (const T *)((const char *)dout + o) + first;
            x[u] = row_part ? chunk_load_part(src, a.dim) : chunk_load_stream(src);
        }
#pragma unroll
        for (unsigned u = 0; u < kAhead; ++u) {
            if (j0 + u >= count) break;
            sum += chunk_to_float<T>(x[u]);
            if (!(last >> (j0 + u) & 1)) continue;
            const uint32_t key = (uint32_t)__builtin_amdgcn_readlane((int)item.key, j0 + u);
            if (from_before || (goes_on && j0 + u + 1 == count)) {
                // slot 0: a sum that came from the part before, slot 1: one that begins here
                if (mine) *(typename Partial<T>::type *)(a.carry + ((uint64_t)part * 2 + (from_before ? 0 : 1)) * a.pitch + first) = sum;
            } else if (mine) {
                write_row(dtable, a.stride, key, a.rows, a.dim, first, sum, a.scale);
            }
            sum = facc{};
            from_before = false;
        }
    }
}

// The number of items whose key is less than `key`, by a wavefront that looks at 64 places at a time.
__device__ __forceinline__ unsigned items_below(const Item *sorted, unsigned n, uint64_t key) {
    const unsigned lane = threadIdx.x % kLanes;
    unsigned low = 0;  // all items in front of low are less, all from low + left on are not
    for (unsigned left = n; left;) {
        const unsigned step = (left + kLanes - 1) / kLanes;
        // lane l looks at the last item of its `step` ones: if that is less, so are the others
        const uint64_t at = (uint64_t)(lane + 1) * step - 1;
        const bool less = at < left && sorted[low + at].key < key;
        const unsigned steps = __builtin_popcountll(__builtin_amdgcn_ballot_w64(less));
        low += steps * step;
        left -= steps * step;
        // the item that ends the next ones is not less
        left = left < step - 1 ? left : step - 1;
    }
    return low;
}

// Zeros for those of kZeroRows (at most 64) rows that no token names.
constexpr unsigned kZeroRows = kLanes;

template <typename T>
__device__ __forceinline__ void embedding_zero_rows(T *dtable, const SumArgs &a, unsigned group) {
    const unsigned lane = threadIdx.x;
    const uint64_t base = (uint64_t)group * kZeroRows;
    const unsigned rows = a.vocab - base < kZeroRows ? (unsigned)(a.vocab - base) : kZeroRows;
    const unsigned begin = items_below(a.sorted, a.n, base);
    const uint64_t key = begin + lane < a.n ? a.sorted[begin + lane].key : a.vocab;
    uint64_t named = 0;
    if (__builtin_amdgcn_ballot_w64(key >= base + rows)) {  // all of these rows' items are in sight
        const uint32_t prior = (uint32_t)__shfl_up((int)(uint32_t)key, 1);
        uint64_t heads = __builtin_amdgcn_ballot_w64(key < base + rows && (lane == 0 || prior != key));
        for (; heads; heads &= heads - 1)
            named |= 1ull << ((uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)key, __builtin_ctzll(heads)) - (uint32_t)base);
    } else {  // many tokens to a row: each lane looks for one row
        unsigned low = begin, high = a.n;
        while (low < high) {
            const unsigned mid = low + (high - low) / 2;
            if (a.sorted[mid].key < base + lane) low = mid + 1;
            else high = mid;
        }
        named = __builtin_amdgcn_ballot_w64(low < a.n && a.sorted[low].key == base + lane);
    }
    uint64_t todo = ~named & (rows < 64 ? (1ull << rows) - 1 : ~0ull);
    while (todo) {
        const unsigned first = __builtin_ctzll(todo);
        const uint64_t rest = ~(todo >> first);
        unsigned run = rest ? __builtin_ctzll(rest) : kLanes;
        // a PE's rows end where the next one's begin
        const uint64_t v = base + first;
        const unsigned owner = (unsigned)(v / a.rows), at = (unsigned)(v % a.rows);
        if (run > a.rows - at) run = a.rows - at;
        zero_fill(copy_of(dtable, owner, a.stride) + (uint64_t)at * a.dim, (uint64_t)run * a.dim);
        todo &= run >= kLanes ? 0 : ~(((1ull << run) - 1) << first);
    }
}

// The first sum_blocks blocks add up, the others fill with zeros: bound by memory.  8 x 4096 tokens of 7168 bf16, 100003 rows (0.47 GB read,
// 1.43 written): 307 to 320 us by process are 6.0 to 6.2 TB/s; where this form took 319, zeros as streaming stores 330, written through 330,
// zeros first 331, in turn with the sums 349.  Zeros for 64 / 16 rows a wavefront: there 307 to 320 / 328, 8 x 500 tokens of 8000 and 1000
// rows, of which 16 wavefronts are few, 33 / 20.
template <typename T>
__global__ __launch_bounds__(64) void embedding_sum_kernel(T *dtable, const T *dout, SumArgs a) {
    if (blockIdx.x < a.sum_blocks) {
        const uint64_t items = (uint64_t)a.parts * a.pieces;
        for (uint64_t i = blockIdx.x; i < items; i += a.sum_blocks)
            embedding_sum_part<T>(dtable, dout, a, (unsigned)(i / a.pieces), (unsigned)(i % a.pieces));
    } else {
        embedding_zero_rows<T>(dtable, a, blockIdx.x - a.sum_blocks);
    }
}

// A block per part in which a sum begins that goes on behind it; its wavefronts share the parts that the sum goes through.
constexpr unsigned kJoinWaves = 4;

template <typename T>
__global__ __launch_bounds__(kJoinWaves *kLanes) void embedding_join_kernel(T *dtable, SumArgs a) {
    typedef typename Chunk<T>::facc facc;
    typedef typename Partial<T>::type stored;
    __shared__ facc partial[kJoinWaves - 1][kLanes];
    const unsigned wave = wave_of_block(), lane = threadIdx.x % kLanes;
    const unsigned c = blockIdx.x * kLanes + lane, first = chunk_first<T>(c, a.dim);
    const bool mine = c * Chunk<T>::N < a.dim;
    for (unsigned part = blockIdx.y; part + 1 < a.parts; part += gridDim.y) {
        const unsigned begin = part * a.part, end = begin + a.part;
        const uint32_t k = a.sorted[end - 1].key, after = a.sorted[end].key, prior = a.sorted[begin > 0 ? begin - 1 : 0].key;
        if (k >= a.vocab || after != k || (begin > 0 && prior == k)) continue;
        unsigned stop = part + 1;  // the first part that does not begin with k
        for (;;) {
            const unsigned q = stop + lane;
            const uint64_t other = __builtin_amdgcn_ballot_w64(q >= a.parts || a.sorted[(uint64_t)q * a.part].key != k);
            if (other) {
                stop += __builtin_ctzll(other);
                break;
            }
            stop += kLanes;
        }
        const unsigned share = (stop - part - 1 + kJoinWaves - 1) / kJoinWaves;
        const unsigned from = part + 1 + wave * share, to = from + share < stop ? from + share : stop;
        facc sum = {};
        if (mine) {
            if (wave == 0) sum = *(const stored *)(a.carry + ((uint64_t)part * 2 + 1) * a.pitch + first);
#pragma unroll 8
            for (unsigned q = from; q < to; ++q) sum += *(const stored *)(a.carry + (uint64_t)q * 2 * a.pitch + first);
        }
        if (wave) partial[wave - 1][lane] = sum;
        __syncthreads();
        if (wave == 0 && mine) {
#pragma unroll
            for (unsigned w = 0; w < kJoinWaves - 1; ++w) sum += partial[w][lane];
            write_row(dtable, a.stride, k, a.rows, a.dim, first, sum, a.scale);
        }
        __syncthreads();
    }
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
    const unsigned log = row_lanes_log2(chunks), per_wave = kLanes >> log;
    const bool many = (uint64_t)tokens * rt.npes / per_wave >= kManyWaves;
#define NVSHMEM_AMD_LAUNCH_EMBEDDING(V, TOKENS, MODE)                                                                                  \
    {                                                                                                                                  \
        const unsigned groups = div_up(tokens, per_wave * TOKENS);                                                                     \
        launch_kernel((embedding_kernel<T, V, TOKENS, MODE>), dim3(div_up(chunks, kLanes * V), groups < 65535 ? groups : 65535, rt.npes), \
                      dim3(kLanes), 0, stream, dst, tab, id, rt.heap_size, (unsigned)tokens, (unsigned)vocab, (unsigned)rows,          \
                      (unsigned)dim, log, scale);                                                                                      \
    }
    if (dim < (size_t)Chunk<T>::N) NVSHMEM_AMD_LAUNCH_EMBEDDING(1, 1, kTiny)
    else if (chunks > 4 * kLanes) NVSHMEM_AMD_LAUNCH_EMBEDDING(2, 1, kWhole)
    else if (chunks > 3 * kLanes) NVSHMEM_AMD_LAUNCH_EMBEDDING(4, 1, kWhole)
    else if (chunks > 2 * kLanes) NVSHMEM_AMD_LAUNCH_EMBEDDING(3, 1, kWhole)
    else if (chunks > kLanes) NVSHMEM_AMD_LAUNCH_EMBEDDING(2, 1, kWhole)
    else if (log == 6 && many) NVSHMEM_AMD_LAUNCH_EMBEDDING(1, 4, kWhole)
    else if (log == 6) NVSHMEM_AMD_LAUNCH_EMBEDDING(1, 1, kWhole)
    else if (many) NVSHMEM_AMD_LAUNCH_EMBEDDING(1, 4, kShared)
    else NVSHMEM_AMD_LAUNCH_EMBEDDING(1, 1, kShared)
#undef NVSHMEM_AMD_LAUNCH_EMBEDDING
    return launched("embedding");
}

// The gradient's workspace, in PE 0's copy: the sorted items, twice where they are sorted digit by digit, with the blocks' counts,
// and two partial sums for every part.
struct GradSpace {
    uint64_t items, hist, carry, bytes;
    unsigned pitch, passes, part;
    GradSpace(uint64_t n, uint64_t vocab, uint64_t dim) {
        unsigned bits = 1;
        while (bits < 32 && vocab >> bits) ++bits;  // (vocab itself is the key of padding)
        passes = n <= kRankTokens ? 0 : (bits + kDigit - 1) / kDigit;
        const uint64_t list = (n * sizeof(Item) + 63) / 64 * 64;
        pitch = (unsigned)((dim + 7) / 8 * 8);
        part = part_of(n, dim);
        items = list;
        hist = passes > 1 ? 2 * list : list;
        carry = hist + (passes ? kSortBlocks * kBins * sizeof(uint32_t) : 0);
        bytes = carry + (n + part - 1) / part * 2 * pitch * sizeof(float);
    }
    // What a program allocates: enough for these sizes and for all that are no larger, of which some have shorter parts and so more partial
    // sums (8 PEs, rows of 7168: 329 tokens take 18.9 MB, 1207 take 8.7).  Parts of P < kMostPart items are for n * pieces < kPartPieces *
    // (P + 1), and rows have at most pieces * kPiece elements: partial sums of that many elements over P, and of one row for the last
    // part.  That is the most where P is the least.
    uint64_t space(uint64_t n) const {
        const uint64_t short_parts = (n + kLeastPart - 1) / kLeastPart * pitch, long_parts = (n + kMostPart - 1) / kMostPart * pitch;
        const uint64_t shorter = (uint64_t)kPartPieces * (kLeastPart + 1) * kPiece / kLeastPart + pitch;
        const uint64_t most = long_parts > shorter ? long_parts : shorter;
        return carry + (short_parts < most ? short_parts : most) * 2 * sizeof(float);
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
    const GradSpace space(n, vocab, dim);
    Operands ops(rt, "embedding_grad");
    const T *src = (const T *)ops.in("dout", dout, (uint64_t)tokens * dim);
    const int64_t *id = ops.in("ids", ids, tokens);
    T *tab = (T *)ops.out("dtable", dtable, (uint64_t)rows * dim);
    char *ws = ops.out("workspace", (char *)workspace, n ? space.bytes : 0, 64);
    if (!ops.ok()) return NVSHMEMX_ERROR_INVALID_VALUE;
    Item *sorted = (Item *)ws, *other = (Item *)(ws + space.items);
    if (n && !space.passes) {
        launch_kernel(embedding_rank_kernel, dim3(div_up(n, kRankKeys)), dim3(kSortThreads), (n + 63) / 64 * 256, stream, sorted, id, rt.heap_size,
                      (unsigned)tokens, (unsigned)n, (unsigned)vocab);
    } else if (n) {
        uint32_t *hist = (uint32_t *)(ws + space.hist);
        const uint64_t tiles = div_up(n, kSortTile);
        const unsigned per_block = (unsigned)((tiles + kSortBlocks - 1) / kSortBlocks) * kSortTile;
        const dim3 grid(div_up(n, per_block));
        Item *out = space.passes % 2 ? sorted : other, *in = space.passes % 2 ? other : sorted;
        for (unsigned p = 0; p < space.passes; ++p) {
#define NVSHMEM_AMD_SORT(FIRST)                                                                                                       \
    launch_kernel(embedding_count_kernel<FIRST>, grid, dim3(kSortThreads), 0, stream, hist, in, id, rt.heap_size, (unsigned)tokens,  \
                  (unsigned)n, (unsigned)vocab, per_block, p * kDigit);                                                              \
    launch_kernel(embedding_sort_kernel<FIRST>, grid, dim3(kSortThreads), 0, stream, out, hist, in, id, rt.heap_size,                \
                  (unsigned)tokens, (unsigned)n, (unsigned)vocab, per_block, p * kDigit)
            if (p == 0) {
                NVSHMEM_AMD_SORT(true);
            } else {
                NVSHMEM_AMD_SORT(false);
            }
#undef NVSHMEM_AMD_SORT
            Item *swap = in;
            in = out, out = swap;
        }
    }
    SumArgs a{};
    a.sorted = sorted, a.carry = (float *)(ws + space.carry), a.stride = rt.heap_size;
    a.tokens = (unsigned)tokens, a.n = (unsigned)n, a.vocab = (unsigned)vocab, a.rows = (unsigned)rows, a.dim = (unsigned)dim;
    a.pitch = space.pitch, a.pieces = div_up(dim, Chunk<T>::N * kLanes), a.scale = scale;
    a.part = space.part, a.parts = div_up(n, space.part);
    const uint64_t items = (uint64_t)a.parts * a.pieces;
    a.sum_blocks = (unsigned)(items < (1u << 22) ? items : 1u << 22);
    launch_kernel(embedding_sum_kernel<T>, dim3(a.sum_blocks + div_up(vocab, kZeroRows)), dim3(kLanes), 0, stream, tab, src, a);
    if (a.parts > 1)
        launch_kernel(embedding_join_kernel<T>, dim3(a.pieces, a.parts < 65535 ? a.parts : 65535), dim3(kJoinWaves * kLanes), 0, stream,
                      tab, a);
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
    const int npes = Runtime::get().npes;
    if (npes < 1) return 0;
    const uint64_t n = (uint64_t)tokens * npes;
    return tokens::GradSpace(n, vocab, dim).space(n);
}

}  // extern "C"
