// Shared by the short convolution and the state space scan: sequence tensors as kernels take them, the checks of them,
// and the sum of partial rows that closes a weight's gradient.
#pragma once
#include <cstdlib>

#include "seq_common.h"

namespace fhc {
namespace seq {

template <class R>
struct Seq {  // strides in elements
    R* p;
    int64_t bs, ts;
    __device__ __forceinline__ R* at(uint32_t b, int64_t t) const { return p + (int64_t)b * bs + t * ts; }
};

template <class R>
Seq<R> seq_of(const fhc_seq* s) {
    return s ? Seq<R>{static_cast<R*>(s->p), s->bs, s->ts} : Seq<R>{nullptr, 0, 0};
}

template <class F>
void with_type(uint32_t dtype, F&& f) {
    if (dtype == FHC_F16) f(F16{});
    else if (dtype == FHC_BF16) f(BF16{});
    else f(F32{});
}

inline int check_shape(const char* op, uint32_t dtype, uint32_t b, uint32_t t, uint32_t d) {
    if (dtype > FHC_F32) return fail(-1, "%s: dtype %u is none of f16, bf16, f32", op, dtype);
    if ((uint64_t)b * d >= 1ull << 31) return fail(-1, "%s: %u x %u columns, at most 2^31 - 1", op, b, d);
    if (t > 0x7FFFFF00u) return fail(-1, "%s: %u steps", op, t);
    return 0;
}

// a tensor of b sequences of t steps
inline int check_in(const char* op, const char* name, const fhc_seq* s, uint32_t dtype, uint32_t t) {
    if (!s) return fail(-1, "%s: null %s", op, name);
    if (t && !s->p) return fail(-1, "%s: null pointer of %s", op, name);
    if (!aligned(s->p, elem_bytes(dtype))) return fail(-1, "%s: %s is not aligned to its elements", op, name);
    return 0;
}
// an output's elements are distinct addresses where its strides leave room for a row of `width` channels
inline int check_out(const char* op, const char* name, const fhc_seq* s, uint32_t dtype, uint32_t b, uint32_t t,
                     uint32_t width) {
    FHC_TRY(check_in(op, name, s, dtype, t));
    if (t > 1 && (uint64_t)std::llabs(s->ts) < width)
        return fail(-1, "%s: %s: steps %lld apart overlap", op, name, (long long)s->ts);
    if (b > 1 && t > 0 && (uint64_t)std::llabs(s->bs) < width)
        return fail(-1, "%s: %s: sequences %lld apart overlap", op, name, (long long)s->bs);
    return 0;
}
inline int check_array(const char* op, const char* name, const void* p, uint32_t bytes, bool needed) {
    if (!p) return needed ? fail(-1, "%s: null %s", op, name) : 0;
    if (!aligned(p, bytes)) return fail(-1, "%s: %s is not aligned to its elements", op, name);
    return 0;
}

namespace {  // a kernel of this unit: another one's is registered apart

// The sums over rows of part[row][.] in f64, its columns dealt to up to three outputs one after another (null: not
// wanted): of each of COLS columns, ROWS threads take every ROWS-th row, and their sums are added in their order.
struct Sums {
    float* out[3];
    uint64_t cols[3];
};
template <int COLS>
__global__ __launch_bounds__(1024) void column_sums(const float* part, uint32_t rows, Sums o) {
    constexpr uint32_t ROWS = 1024 / COLS;
    __shared__ double s[ROWS][COLS];
    const uint32_t x = threadIdx.x % COLS, y = threadIdx.x / COLS;
    uint64_t c = (uint64_t)blockIdx.x * COLS + x;
    const uint64_t pitch = o.cols[0] + o.cols[1] + o.cols[2];
    const bool live = c < pitch;
    double sum = 0.0;
    if (live) {
#pragma unroll 4
        for (uint64_t r = y; r < rows; r += ROWS) sum += part[r * pitch + c];
    }
    s[y][x] = sum;
    __syncthreads();
    if (y > 0 || !live) return;
#pragma unroll
    for (uint32_t k = 1; k < ROWS; k++) sum += s[k][x];
#pragma unroll
    for (int k = 0; k < 3; k++) {
        if (c < o.cols[k]) {
            if (o.out[k]) o.out[k][c] = (float)sum;
            return;
        }
        c -= o.cols[k];
    }
}
inline int close_sums(const char* op, const float* part, uint32_t rows, const Sums& o, hipStream_t st) {
    const uint64_t columns = o.cols[0] + o.cols[1] + o.cols[2];
    if (!columns || (!o.out[0] && !o.out[1] && !o.out[2])) return 0;
    // Few columns over many rows have a whole workgroup's threads to 8 columns, else to 64. us of a backward pass with 64 and with
    // 8: 16384 rows of 1152 5275, 5190; 8192 of 320 1424, 1404; 4096 of 1152 1347, 1337; 1024 of 1280 350, 359.
    const bool few = columns <= 2048 && rows >= 4096;
    const uint64_t blocks = ceil_div(columns, few ? 8 : 64);
    FHC_TRY(check_grid(op, blocks, 1024));
    if (few) hipLaunchKernelGGL(column_sums<8>, dim3((uint32_t)blocks), dim3(1024), 0, st, part, rows, o);
    else hipLaunchKernelGGL(column_sums<64>, dim3((uint32_t)blocks), dim3(1024), 0, st, part, rows, o);
    return launched(op);
}

}  // namespace

// sigmoid(v); the exponential is inf for v far below 0, and its reciprocal 0
__device__ __forceinline__ float sigmoid1(float v) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.44269504088896340736f));
}
// v sigmoid(v) and its slope, p + v p (1 - p). What 1 - p multiplies is held finite: where p is 0 or 1 an infinity times 0
// is not 0.
__device__ __forceinline__ void silu_grad(float v, float& value, float& slope) {
    const float e = __builtin_amdgcn_exp2f(v * -1.44269504088896340736f), p = __builtin_amdgcn_rcpf(1.0f + e);
    const float q = __builtin_fminf(e * p, 1.0f);  // 1 - p; inf * 0 where e overflows
    value = v * p;
    slope = p * __builtin_fmaf(__builtin_amdgcn_fmed3f(v, -1e12f, 1e12f), q, 1.0f);
}

}  // namespace seq
}  // namespace fhc
