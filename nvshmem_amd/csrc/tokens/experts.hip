// The experts of a model, on the rows that were dispatched to them: a gated feed-forward block each.
//
//   pre = [gate | up] = x W_in^T      h = gate * sigmoid(gate) * up      out = h W_out^T
//
// for the rows [expert_row[i], expert_row[i + 1]) of expert i.  Both input projections, the activation and the product are one
// kernel; h goes through memory in the rows' type, rounded once, and is what the second kernel reads: the matrix cores take it in no
// other (a half beyond 65504 becomes an infinity there).  us for bf16, 64 experts of 7168 x 2048: 131072 rows 9250 to 9800
// by board (1.18 to 1.25 PFLOP/s), 64 rows (3.7 GB of weights) 580 to 600 (6.1 to 6.4 TB/s).
#include "expert_tiles.hpp"

namespace nvshmem_amd {
namespace tokens {
namespace {

template <typename API>
int experts_on_stream(API *out, API *pre, void *workspace, const API *rows, const API *w_in, const API *w_out,
                      const int64_t *expert_row, size_t recv_cap_rows, int experts, size_t dim, size_t hidden, hipStream_t stream) {
    typedef typename element<API>::type T;
    Runtime &rt = Runtime::get();
    std::lock_guard<std::recursive_mutex> lock(rt.mu);
    if (!ready(rt, "moe_experts")) return NVSHMEMX_ERROR_INVALID_VALUE;
    if (int rc = check_expert_sizes(rt, "moe_experts", experts, dim, hidden)) return rc;
    const uint64_t cap = recv_cap_rows, mine = (uint64_t)(experts / rt.npes);
    NVSHMEM_AMD_REFUSE(cap > rt.heap_size / (dim * sizeof(T)) || cap > rt.heap_size / (hidden * sizeof(T)),
                       "moe_experts: %zu rows leave the PE's heap slice", recv_cap_rows);
    Operands ops(rt, "moe_experts");
    ExpertArgs<T> args = {};
    args.rows = (const T *)ops.in("rows", rows, cap * dim);
    args.w_in = (const T *)ops.in("w_in", w_in, mine * 2 * hidden * dim);
    args.w_out = (const T *)ops.in("w_out", w_out, mine * dim * hidden);
    args.expert_row = ops.in("expert_row", expert_row, mine + 1);
    args.out = (T *)ops.out("out", out, cap * dim);
    if (pre) args.pre = (T *)ops.out("pre", pre, cap * 2 * hidden);
    args.h = (T *)ops.out("workspace", (char *)workspace, cap * hidden * sizeof(T), 64);
    if (!ops.ok()) return NVSHMEMX_ERROR_INVALID_VALUE;
    if (cap == 0) return 0;
    args.stride = rt.heap_size, args.cap = cap, args.experts = (unsigned)mine, args.npes = (unsigned)rt.npes, args.dim = (unsigned)dim, args.hidden = (unsigned)hidden;
    // (the slices' stride is a multiple of 2 MiB, so that every PE's copies are aligned like PE 0's)
    const bool whole = dim * sizeof(T) % 16 == 0 && hidden * sizeof(T) % 16 == 0 && aligned16(args.rows) && aligned16(args.w_in) &&
                       aligned16(args.w_out);
    if (whole) {
        launch_expert_tiles<T, kIn, true>(args, stream);
        launch_expert_tiles<T, kOut, true>(args, stream);
    } else {
        launch_expert_tiles<T, kIn, false>(args, stream);
        launch_expert_tiles<T, kOut, false>(args, stream);
    }
    return launched("moe_experts");
}

}  // namespace
}  // namespace tokens
}  // namespace nvshmem_amd

using namespace nvshmem_amd;

extern "C" {

#define NVSHMEM_AMD_EXPERTS(NAME, TYPE)                                                                                           \
    int nvshmemx_amd_##NAME##_moe_experts_on_stream(TYPE *out, TYPE *pre, void *workspace, const TYPE *rows, const TYPE *w_in,    \
                                                    const TYPE *w_out, const int64_t *expert_row, size_t recv_cap_rows,           \
                                                    int experts, size_t dim, size_t hidden, nvshmemx_stream_t stream) {           \
        return tokens::experts_on_stream(out, pre, workspace, rows, w_in, w_out, expert_row, recv_cap_rows, experts, dim, hidden, \
                                         (hipStream_t)stream);                                                                    \
    }
NVSHMEMI_AMD_REPT_FOR_TOKEN_TYPES(NVSHMEM_AMD_EXPERTS)
#undef NVSHMEM_AMD_EXPERTS

size_t nvshmemx_amd_moe_experts_workspace(size_t recv_cap_rows, int experts, size_t dim, size_t hidden) {
    (void)dim;
    Runtime &rt = Runtime::get();
    std::lock_guard<std::recursive_mutex> lock(rt.mu);
    if (!rt.initialized || experts < 1 || hidden > tokens::kMostFeatures || recv_cap_rows > ((uint64_t)1 << 40)) return 0;
    return recv_cap_rows * hidden * sizeof(float);
}

}  // extern "C"
