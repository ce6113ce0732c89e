// What the operators on rows of tokens share: element types, 16-byte chunks of rows, checks of operands.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <mutex>

#include "launch.hpp"
#include "nvshmem.h"
#include "runtime.hpp"

namespace nvshmem_amd {
namespace tokens {

// The storage of the typed entry points' elements in kernels.  Arithmetic is in fp32; a result is rounded to its type once, to
// the nearest, ties to even (v_cvt_pk_bf16_f32, v_cvt_f16_f32).
template <typename API>
struct element;
template <>
struct element<float> {
    typedef float type;
};
template <>
struct element<nvshmem_half_t> {
    typedef _Float16 type;
};
template <>
struct element<nvshmem_bfloat16_t> {
    typedef __bf16 type;
};

constexpr int kLanes = 64;

// How a row's chunks lie on lanes: a wavefront and more to a row, rows that share a wavefront, rows of less than a chunk (which
// share one as well).
enum { kWhole, kShared, kTiny };

// A row is handled in chunks of 16 bytes, counted from its first element whatever that is aligned to: gfx950 takes 16-byte
// accesses at any address (one global_load_dwordx4 either way), so rows of an odd number of elements need no kernel of their own.
template <typename T>
constexpr int chunk_elems() {
    return 16 / (int)sizeof(T);
}
template <typename T>
struct Chunk {
    static constexpr int N = chunk_elems<T>();
    typedef T vec __attribute__((ext_vector_type(N)));
    typedef vec vec_unaligned __attribute__((aligned(sizeof(T))));
    typedef float facc __attribute__((ext_vector_type(N)));
};
template <typename T>
__device__ __forceinline__ typename Chunk<T>::vec chunk_load(const T *p) {
    return *reinterpret_cast<const typename Chunk<T>::vec_unaligned *>(p);
}
template <typename T>
__device__ __forceinline__ typename Chunk<T>::vec chunk_load_stream(const T *p) {
    return __builtin_nontemporal_load(reinterpret_cast<const typename Chunk<T>::vec_unaligned *>(p));
}
template <typename T>
__device__ __forceinline__ void chunk_store_stream(T *p, typename Chunk<T>::vec v) {
    __builtin_nontemporal_store(v, reinterpret_cast<typename Chunk<T>::vec_unaligned *>(p));
}
// ... and written through to memory, past the L2.
template <typename T>
__device__ __forceinline__ void chunk_store_through(T *p, typename Chunk<T>::vec v) {
    asm volatile("global_store_dwordx4 %0, %1, off sc1 nt\n\ts_nop 1" : : "v"(p), "v"(v) : "memory");
}
// Where chunk c of a row begins.  The last one ends with the row and so may share elements with the one in front of it: what is
// computed for an element depends on the element alone, so both store the same bits, and every access is a whole vector.
// Rows of less than a chunk have one, of `dim` elements, which the _part functions move.
template <typename T>
__device__ __forceinline__ unsigned chunk_first(unsigned c, unsigned dim) {
    const unsigned first = c * Chunk<T>::N, most = dim < (unsigned)Chunk<T>::N ? 0 : dim - Chunk<T>::N;
    return first < most ? first : most;
}
template <typename T>
__device__ __forceinline__ typename Chunk<T>::vec chunk_load_part(const T *p, unsigned n) {
    typename Chunk<T>::vec v;
#pragma unroll
    for (int i = 0; i < Chunk<T>::N; ++i) v[i] = i < (int)n ? p[i] : (T)0.0f;
    return v;
}
template <typename T>
__device__ __forceinline__ void chunk_store_part(T *p, typename Chunk<T>::vec v, unsigned n) {
#pragma unroll
    for (int i = 0; i < Chunk<T>::N; ++i)
        if (i < (int)n) p[i] = v[i];
}
// All but the first `n` elements.
template <typename T>
__device__ __forceinline__ void chunk_store_behind(T *p, typename Chunk<T>::vec v, unsigned n) {
#pragma unroll
    for (int i = 0; i < Chunk<T>::N; ++i)
        if (i >= (int)n) p[i] = v[i];
}
template <typename T>
__device__ __forceinline__ typename Chunk<T>::facc chunk_to_float(typename Chunk<T>::vec v) {
    return __builtin_convertvector(v, typename Chunk<T>::facc);
}
template <typename T>
__device__ __forceinline__ typename Chunk<T>::vec chunk_from_float(typename Chunk<T>::facc v) {
    return __builtin_convertvector(v, typename Chunk<T>::vec);
}

// PE pe's copy of a symmetric object of which `p` is PE 0's.
template <typename T>
__device__ __forceinline__ T *copy_of(T *p, unsigned pe, uint64_t stride) {
    return (T *)((char *)p + pe * stride);  // (pointer arithmetic all the way, or loads become flat ones)
}
// ---- lanes that exchange values: groups of G (16, or the wavefront) ----
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xf, 0xf, true);
}
// The value of the lane that step STEP of a reduction over a group pairs with.  Steps 2 and 3 mirror 8 and 16 lanes: after the
// steps before, all lanes of a quad (a half of the row) hold the same.
template <int STEP>
__device__ __forceinline__ uint32_t partner(uint32_t x) {
    if (STEP == 0) return dpp<0xB1>(x);   // quad_perm [1,0,3,2]
    if (STEP == 1) return dpp<0x4E>(x);   // quad_perm [2,3,0,1]
    if (STEP == 2) return dpp<0x141>(x);  // row_half_mirror
    if (STEP == 3) return dpp<0x140>(x);  // row_mirror
    return (uint32_t)__shfl_xor((int)x, STEP == 4 ? 16 : 32);
}
template <int STEP>
__device__ __forceinline__ float partner(float x) {
    return __uint_as_float(partner<STEP>(__float_as_uint(x)));
}
template <int STEP>
__device__ __forceinline__ double partner(double x) {
    const uint64_t b = (uint64_t)__double_as_longlong(x);
    return __longlong_as_double((long long)((uint64_t)partner<STEP>((uint32_t)(b >> 32)) << 32 | partner<STEP>((uint32_t)b)));
}
template <int G>
__device__ __forceinline__ float group_sum(float x) {
    x += partner<0>(x);
    x += partner<1>(x);
    x += partner<2>(x);
    x += partner<3>(x);
    if (G == 64) {
        x += partner<4>(x);
        x += partner<5>(x);
    }
    return x;
}
template <int G>
__device__ __forceinline__ float group_max(float x) {
    x = fmaxf(x, partner<0>(x));
    x = fmaxf(x, partner<1>(x));
    x = fmaxf(x, partner<2>(x));
    x = fmaxf(x, partner<3>(x));
    if (G == 64) {
        x = fmaxf(x, partner<4>(x));
        x = fmaxf(x, partner<5>(x));
    }
    return x;
}
// The wavefront's index in its block as a scalar.
__device__ __forceinline__ unsigned wave_of_block() { return __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes); }

// Operands of a call: each has to lie in one PE's part of the heap, and what is written may overlap nothing else.
class Operands {
  public:
    Operands(Runtime &rt, const char *what) : rt_(rt), what_(what) {}
    // PE 0's copy of the object; nullptr (and not ok()) when it does not fit.  An object of no bytes is not looked at.
    template <typename T>
    T *in(const char *name, const T *p, uint64_t elems, uint64_t align = sizeof(T)) {
        return (T *)add(name, p, elems, sizeof(T), align, false);
    }
    template <typename T>
    T *out(const char *name, T *p, uint64_t elems, uint64_t align = sizeof(T)) {
        return (T *)add(name, p, elems, sizeof(T), align, true);
    }
    // Lets the last operand named be the very buffer of an earlier one.
    void may_be(const void *other) { may_be_ = other; }
    bool ok() const { return ok_; }

  private:
    void *add(const char *name, const void *p, uint64_t elems, uint64_t size, uint64_t align, bool written) {
        if (!ok_ || elems == 0) return nullptr;
        uint64_t off = 0;
        const bool fits = elems <= rt_.heap_size / size;
        if (!fits || !rt_.usable(p, elems * size, &off) || off % align) return refuse(name, p, fits, elems, size, align);
        const uint64_t end = off + elems * size;
        for (int i = 0; i < n_; ++i) {
            if (!written && !op_[i].written) continue;
            if (off >= op_[i].end || op_[i].off >= end) continue;
            if (may_be_ && off == op_[i].off && end == op_[i].end && may_be_ == rt_.base + off) continue;
            set_error("%s %s: overlaps %s", what_, name, op_[i].name);
            return fail();
        }
        if (n_ < kMost) op_[n_++] = {name, off, end, written};
        return rt_.base + off;
    }
    // (a call that is fine makes no text)
    void *refuse(const char *name, const void *p, bool fits, uint64_t elems, uint64_t size, uint64_t align) {
        char label[96];
        snprintf(label, sizeof label, "%s %s", what_, name);
        uint64_t off = 0;
        if (!fits) set_error("%s: %llu elements leave the PE's heap slice", label, (unsigned long long)elems);
        else if (check_symmetric_range(rt_, label, p, elems * size, &off)) set_error("%s: must be aligned to %llu bytes", label, (unsigned long long)align);
        return fail();
    }
    void *fail() {
        ok_ = false;
        return nullptr;
    }
    static constexpr int kMost = 16;
    struct {
        const char *name;
        uint64_t off, end;
        bool written;
    } op_[kMost];
    Runtime &rt_;
    const char *what_;
    const void *may_be_ = nullptr;
    int n_ = 0;
    bool ok_ = true;
};

// Initialised, and on the heap's GPU: kernels go to the calling thread's current device.
inline bool ready(Runtime &rt, const char *what) {
    if (!rt.initialized) {
        set_error("%s called before nvshmem_init", what);
        return false;
    }
    int device = -1;
    if (hipGetDevice(&device) != hipSuccess || device != rt.device) {
        set_error("%s: the current device is %d, the symmetric heap's %d", what, device, rt.device);
        return false;
    }
    return true;
}
inline int launched(const char *what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    set_error("%s: kernel launch failed: %s", what, hipGetErrorString(e));
    return NVSHMEMX_ERROR_INTERNAL;
}
#define NVSHMEM_AMD_REFUSE(cond, ...)                \
    do {                                             \
        if (cond) {                                  \
            set_error(__VA_ARGS__);                  \
            return NVSHMEMX_ERROR_INVALID_VALUE;     \
        }                                            \
    } while (0)

// The least power of two of lanes (its logarithm, at most a wavefront) that a row of so many chunks fills.
inline unsigned row_lanes_log2(size_t chunks) {
    unsigned l = 0;
    while (l < 6 && ((size_t)1 << l) < chunks) ++l;
    return l;
}
inline unsigned div_up(uint64_t a, uint64_t b) { return (unsigned)((a + b - 1) / b); }

}  // namespace tokens
}  // namespace nvshmem_amd
