// Shared by the operators on rows of channels (include/fhc_seq.h): the three element types, vector loads at any
// alignment, and the host-side checks.
#pragma once
#include <hip/hip_runtime.h>

#include <cmath>

#include "common.h"
#include "fhc_seq.h"

namespace fhc {
namespace seq {

struct F16 {
    using Raw = uint16_t;
    static constexpr uint32_t id = FHC_F16;
};
struct BF16 {
    using Raw = uint16_t;
    static constexpr uint32_t id = FHC_BF16;
};
struct F32 {
    using Raw = float;
    static constexpr uint32_t id = FHC_F32;
};

__device__ __forceinline__ float widen(F16, uint16_t b) { return (float)__builtin_bit_cast(_Float16, b); }
__device__ __forceinline__ float widen(BF16, uint16_t b) { return __builtin_bit_cast(float, (uint32_t)b << 16); }
__device__ __forceinline__ float widen(F32, float v) { return v; }
// Round to nearest even. f16's is written as its instruction: the compiler otherwise fuses it with the operation before
// it in some places and not in others (a mixed-precision FMA that rounds once), and the same row then gives other bits
// in another variant of a kernel.
__device__ __forceinline__ uint16_t narrow(F16, float v) {
    uint32_t r;
    asm("v_cvt_f16_f32 %0, %1" : "=v"(r) : "v"(v));
    return (uint16_t)r;
}
__device__ __forceinline__ uint16_t narrow(BF16, float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
__device__ __forceinline__ float narrow(F32, float v) { return v; }

// N consecutive elements as one load (16-bit pairs and quads, f32 pairs; 8 elements as one or two 16-byte loads).
// AL: the address is a multiple of the vector's size (16 bytes at most), else of the element's: the hardware reads and
// writes dwords at any byte address, only slower, and the compiler is told the smaller alignment.
template <class R, int N, bool AL>
struct Pack {
    static constexpr int kBytes = N * (int)sizeof(R);
    static constexpr int kAlign = AL ? (kBytes < 16 ? kBytes : 16) : (int)sizeof(R);
    typedef R Vec __attribute__((ext_vector_type(N)));
    typedef Vec Mem __attribute__((aligned(kAlign)));
};
template <class R, int N, bool AL>
__device__ __forceinline__ void load_raw(const R* p, R (&o)[N]) {
    if constexpr (N == 1) {
        o[0] = *p;
    } else {
        using Mem = typename Pack<R, N, AL>::Mem;
        const auto v = *reinterpret_cast<const Mem*>(p);
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = v[i];
    }
}
template <class R, int N, bool AL>
__device__ __forceinline__ void store_raw(R* p, const R (&o)[N]) {
    if constexpr (N == 1) {
        *p = o[0];
    } else {
        using Mem = typename Pack<R, N, AL>::Mem;
        typename Pack<R, N, AL>::Vec v;
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = o[i];
        *reinterpret_cast<Mem*>(p) = v;
    }
}

inline uint32_t elem_bytes(uint32_t dtype) { return dtype == FHC_F32 ? 4 : 2; }
inline bool aligned(const void* p, uint32_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
inline uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

inline int launched(const char* op) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(-2, "%s: launch failed: %s", op, hipGetErrorString(e));
    return 0;
}

// a launch has fewer than 2^32 threads
inline int check_grid(const char* op, uint64_t blocks, uint32_t threads) {
    if (blocks >= (1ull << 32) / threads) return fail(-1, "%s: too many workgroups (%llu)", op, (unsigned long long)blocks);
    return 0;
}

inline int check_workspace(const char* op, size_t need, const void* ws, size_t have) {
    if (!need) return 0;
    if (!ws) return fail(-1, "%s: null workspace (%zu bytes needed)", op, need);
    if (have < need) return fail(-1, "%s: workspace of %zu bytes, %zu needed", op, have, need);
    if (!aligned(ws, 256)) return fail(-1, "%s: the workspace is not 256-byte aligned", op);
    return 0;
}

#define FHC_TRY(x)               \
    do {                         \
        const int rc_ = (x);     \
        if (rc_ < 0) return rc_; \
    } while (0)

}  // namespace seq
}  // namespace fhc
