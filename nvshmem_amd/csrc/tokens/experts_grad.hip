// The gradients of the experts' gated feed-forward block, from dout and the projections [gate | up] that the forward pass kept.
//
//   s = sigmoid(gate)   h = gate s up   dh = dout W_out
//   dup = dh gate s     dgate = dh up (s + gate s (1 - s))
//   drows = [dgate | dup] W_in      dW_in = [dgate | dup]^T x      dW_out = dout^T h
//
// The first kernel makes dh in its accumulators and stores [dgate | dup] and h, in the rows' type, rounded once each: the matrix cores
// take them in no other.  An expert without rows gets weights' gradients of zeros.  us for bf16, 65536 rows of 32 experts of 7168 x 2048: 10050 to 10800
// by board (1.07 to 1.15 PFLOP/s; dh 1980, drows 3280 to 3350, dw_in 3640, dw_out 1840).
#include "expert_tiles.hpp"

namespace nvshmem_amd {
namespace tokens {
namespace {

uint64_t dpre_bytes(uint64_t cap, uint64_t hidden, uint64_t size) { return align_up(cap * 2 * hidden * size, 64); }

template <typename API>
int experts_grad_on_stream(API *drows, API *dw_in, API *dw_out, void *workspace, const API *dout, const API *rows, const API *pre,
                           const API *w_in, const API *w_out, const int64_t *expert_row, size_t recv_cap_rows, int experts, size_t dim,
                           size_t hidden, hipStream_t stream) {
    typedef typename element<API>::type T;
    Runtime &rt = Runtime::get();
    std::lock_guard<std::recursive_mutex> lock(rt.mu);
    if (!ready(rt, "moe_experts_grad")) return NVSHMEMX_ERROR_INVALID_VALUE;
    if (int rc = check_expert_sizes(rt, "moe_experts_grad", experts, dim, hidden)) return rc;
    const uint64_t cap = recv_cap_rows, mine = (uint64_t)(experts / rt.npes);
    NVSHMEM_AMD_REFUSE(cap > rt.heap_size / (dim * sizeof(T)) || cap > rt.heap_size / (3 * hidden * sizeof(T)),
                       "moe_experts_grad: %zu rows leave the PE's heap slice", recv_cap_rows);
    Operands ops(rt, "moe_experts_grad");
    ExpertArgs<T> args = {};
    args.dout = (const T *)ops.in("dout", dout, cap * dim);
    args.rows = (const T *)ops.in("rows", rows, cap * dim);
    args.pre_in = (const T *)ops.in("pre", pre, cap * 2 * hidden);
    args.w_in = (const T *)ops.in("w_in", w_in, mine * 2 * hidden * dim);
    args.w_out = (const T *)ops.in("w_out", w_out, mine * dim * hidden);
    args.expert_row = ops.in("expert_row", expert_row, mine + 1);
    args.drows = (T *)ops.out("drows", drows, cap * dim);
    args.dw_in = (T *)ops.out("dw_in", dw_in, mine * 2 * hidden * dim);
    args.dw_out = (T *)ops.out("dw_out", dw_out, mine * dim * hidden);
    const uint64_t h_at = dpre_bytes(cap, hidden, sizeof(T));
    char *ws = ops.out("workspace", (char *)workspace, cap ? h_at + cap * hidden * sizeof(T) : 0, 64);
    if (!ops.ok()) return NVSHMEMX_ERROR_INVALID_VALUE;
    args.dpre = (T *)ws, args.h = (T *)(ws + h_at);
    args.stride = rt.heap_size, args.cap = cap, args.experts = (unsigned)mine, args.npes = (unsigned)rt.npes, args.dim = (unsigned)dim, args.hidden = (unsigned)hidden;
    const bool whole = dim * sizeof(T) % 16 == 0 && hidden * sizeof(T) % 16 == 0 && aligned16(args.rows) && aligned16(args.w_in) &&
                       aligned16(args.w_out) && aligned16(args.dout);
    if (whole) {
        launch_expert_tiles<T, kDh, true>(args, stream);
        launch_expert_tiles<T, kDx, true>(args, stream);
        launch_expert_tiles<T, kDwIn, true>(args, stream);
        launch_expert_tiles<T, kDwOut, true>(args, stream);
    } else {
        launch_expert_tiles<T, kDh, false>(args, stream);
        launch_expert_tiles<T, kDx, false>(args, stream);
        launch_expert_tiles<T, kDwIn, false>(args, stream);
        launch_expert_tiles<T, kDwOut, false>(args, stream);
    }
    return launched("moe_experts_grad");
}

}  // namespace
}  // namespace tokens
}  // namespace nvshmem_amd

using namespace nvshmem_amd;

extern "C" {

#define NVSHMEM_AMD_EXPERTS_GRAD(NAME, TYPE)                                                                                          \
    int nvshmemx_amd_##NAME##_moe_experts_grad_on_stream(TYPE *drows, TYPE *dw_in, TYPE *dw_out, void *workspace, const TYPE *dout,   \
                                                         const TYPE *rows, const TYPE *pre, const TYPE *w_in, const TYPE *w_out,      \
                                                         const int64_t *expert_row, size_t recv_cap_rows, int experts, size_t dim,    \
                                                         size_t hidden, nvshmemx_stream_t stream) {                                   \
        return tokens::experts_grad_on_stream(drows, dw_in, dw_out, workspace, dout, rows, pre, w_in, w_out, expert_row,              \
                                              recv_cap_rows, experts, dim, hidden, (hipStream_t)stream);                              \
    }
NVSHMEMI_AMD_REPT_FOR_TOKEN_TYPES(NVSHMEM_AMD_EXPERTS_GRAD)
#undef NVSHMEM_AMD_EXPERTS_GRAD

size_t nvshmemx_amd_moe_experts_grad_workspace(size_t recv_cap_rows, int experts, size_t dim, size_t hidden) {
    (void)dim;
    Runtime &rt = Runtime::get();
    std::lock_guard<std::recursive_mutex> lock(rt.mu);
    if (!rt.initialized || experts < 1 || hidden > tokens::kMostFeatures || recv_cap_rows > ((uint64_t)1 << 40)) return 0;
    return tokens::dpre_bytes(recv_cap_rows, hidden, sizeof(float)) + recv_cap_rows * hidden * sizeof(float);
}

}  // extern "C"
