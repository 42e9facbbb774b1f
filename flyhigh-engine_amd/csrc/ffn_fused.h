// The gated feed-forward block over few channels (c <= 256) and many rows, in one kernel a direction
// (include/fhc_seq.h). Its products between rows and features are f / c times larger than its input, so nothing of them
// leaves the chip: forward, y = (act(x wg^T) * (x wu^T)) wd^T; backward, dx, with x wg^T and x wu^T computed again (two of
// its five products) rather than read, and h, dL/dgate and dL/dup written once in 16 bits for the weights' gradients.
//
// - A wave has 16 MB rows of x (and dy) as fragments in registers and walks the features, 32 at a time. The sums of a
//   slice come out of the MFMA with 4 adjacent features of one row a lane; two such blocks are the second operand of the
//   next product as they are, in an order of K (features 4 g .. 4 g + 3 and 16 + 4 g .. of lane group g) that the
//   weights' fragments are read in too. So they never pass through LDS.
// - The slices of wg, wu ([32 features][c]) and wd ([c][32 features]) come by LDS DMA, three buffers in turn, shared by
//   the workgroup's waves. dx reads wg and wu along the features and dL/dh reads wd along the channels: the transposing
//   LDS read, from the same buffers. 16-byte chunks are permuted within a row so that neither read meets a bank twice:
//   wg, wu: chunk ^ 2 (row & 7) (c <= 64, whose rows are half as long: ^ 2 (row >> 1 & 3)); wd: chunk ^ (row >> 2 & 3).
//
// Bound by the chain of a slice (fragments from LDS, products, activation, products) at two waves a SIMD, which its
// registers allow. MI355X, 51840 x 128, f 512, f16: forward 38 us (20 GFLOP, 540 TFLOP/s), backward 84 (34 GFLOP, 405
// TFLOP/s). Backward spills, bytes a lane: c > 64 104 (f16) and 72 (bf16), c > 128 144 and 136.
#pragma once
#include "ffn_gemm.h"

namespace fhc {
namespace seq {

struct FusedArgs {
    const uint16_t *x, *wg, *wu, *wd, *dy;  // widths in multiples of 8, zeros from c (f) on
    int64_t ldx, ldg, ldd, ldy;
    int rows, c, f;
    uint16_t* out;  // y or dx; null: not wanted
    int64_t ldo;
    uint16_t *h, *dg, *du;  // backward: [rows][up8(f)]
    uint32_t act;
};

// the transposing read at byte `at` of a buffer (one opaque offset: see Operand::frag)
__device__ __forceinline__ uint2 read_tr(const uint4* lds, int at) {
    asm volatile("" : "+v"(at));  // volatile: made anew for each slice rather than kept, registers are short
#if defined(__HIP_DEVICE_COMPILE__)
    typedef __attribute__((address_space(3))) s4_t* lds_s4;
    const char* p = reinterpret_cast<const char*>(lds) + at;
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p)));
#else
    return uint2{};
#endif
}

template <class T, int CP, int MB, int NW, bool BWD>
__global__ __launch_bounds__(64 * NW, 2) void ffn_fused(FusedArgs g) {
    constexpr int KS = CP / 32, NB = CP / 16, ROW = CP * 2;     // ROW: bytes of a feature's row of wg, wu
    constexpr int IU = CP / 16 / NW, ID = CP / 16 / NW, NI = 2 * IU + ID;  // DMA instructions a wave: of wg, of wd
    constexpr int U4 = 32 * ROW / 16;                           // 16-byte units of a slice, of any of the three
    __shared__ __align__(1024) uint4 g0[U4], u0[U4], d0[U4], g1[U4], u1[U4], d1[U4], g2[U4], u2[U4], d2[U4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lo = lane & 15, hi = lane >> 4;
    const int m0 = (blockIdx.x * NW + wave) * 16 * MB;
    auto turn = [](int row) { return CP == 64 ? (row >> 1 & 3) << 1 : (row & 7) << 1; };

    // ---- fetching slices, in order
    uint32_t offg[IU], offd[ID];
    int fd[ID];
#pragma unroll
    for (int q = 0; q < IU; q++) {
        constexpr int LPR = ROW / 16;  // lanes of a row
        const int row = (wave * IU + q) * (64 / LPR) + lane / LPR, k = (lane % LPR ^ turn(row)) * 8;
        offg[q] = k < g.c ? (uint32_t)(row * (int)g.ldg + k) * 2u : kFar;
    }
#pragma unroll
    for (int q = 0; q < ID; q++) {
        const int row = (wave * ID + q) * 16 + (lane >> 2);
        fd[q] = ((lane & 3) ^ (row >> 2 & 3)) * 8;
        offd[q] = row < g.c ? (uint32_t)(row * (int)g.ldd + fd[q]) * 2u : kFar;
    }
    const char *pg = reinterpret_cast<const char*>(g.wg), *pu = reinterpret_cast<const char*>(g.wu);
    const char* pd = reinterpret_cast<const char*>(g.wd);
    const int64_t step = 32 * g.ldg * 2;
    int64_t left = ((g.f - 1) * g.ldg + up8(g.c)) * 2;  // bytes to wg's end
    int fleft = g.f;
    auto resource = [](const char* p, int64_t bytes) {
        const int top = (int)(bytes >> 32), n = top < 0 ? 0 : top > 0 || (int)bytes < 0 ? 0x7FFFFFFF : (int)bytes;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), (short)0, n, 0x00020000);
    };
    auto fetch = [&](uint4* bg, uint4* bu, uint4* bd) __attribute__((always_inline)) {
        const auto rg = resource(uniform(pg), left), ru = resource(uniform(pu), left);
        const auto rd = resource(uniform(pd), 0x7FFFFFFF);
#pragma unroll
        for (int q = 0; q < IU; q++) {
            lds_dma16(rg, bg + (wave * IU + q) * 64, offg[q]);
            lds_dma16(ru, bu + (wave * IU + q) * 64, offg[q]);
        }
#pragma unroll
        for (int q = 0; q < ID; q++) lds_dma16(rd, bd + (wave * ID + q) * 64, fd[q] < fleft ? offd[q] : kFar);
        pg += step, pu += step, pd += 64, left -= step, fleft -= 32;
    };
    auto fence = [] { asm volatile("" ::: "memory"); };
    fetch(g0, u0, d0);
    fetch(g1, u1, d1);

    // ---- the rows' fragments
    u4_t xf[MB][KS], yf[BWD ? MB : 1][BWD ? KS : 1];
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const int m = m0 + i * 16 + lo, k = ks * 32 + hi * 8;
            const bool in = m < g.rows && k < g.c;
            xf[i][ks] = in ? load_some(g.x + m * g.ldx + k, 8) : u4_t{0, 0, 0, 0};
            if constexpr (BWD) yf[i][ks] = in ? load_some(g.dy + m * g.ldy + k, 8) : u4_t{0, 0, 0, 0};
        }
    f4 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
        for (int n = 0; n < NB; n++) acc[i][n] = f4{0.0f, 0.0f, 0.0f, 0.0f};

    const int64_t fp = up8(g.f);
    // the wave's rows of h, dL/dgate and dL/dup
    const int64_t first = BWD ? m0 * fp * 2 : 0;
    const auto og = resource(uniform(reinterpret_cast<const char*>(g.dg) + first), 0x7FFFFFFF);
    const auto ou = resource(uniform(reinterpret_cast<const char*>(g.du) + first), 0x7FFFFFFF);
    const auto oh = resource(uniform(reinterpret_cast<const char*>(g.h) + first), 0x7FFFFFFF);
    auto multiply = [&](int f0, const uint4* bg, const uint4* bu, const uint4* bd) __attribute__((always_inline)) {
        f4 ga[MB][2], up[MB][2], dh[BWD ? MB : 1][2];
#pragma unroll
        for (int i = 0; i < MB; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                ga[i][j] = up[i][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (BWD) dh[i][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
            }
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int row = j * 16 + lo, at = row * ROW + (((ks * 4 + hi) ^ turn(row)) << 4);
                const u4_t fg = *reinterpret_cast<const u4_t*>(reinterpret_cast<const char*>(bg) + at);
                const u4_t fu = *reinterpret_cast<const u4_t*>(reinterpret_cast<const char*>(bu) + at);
                u4_t fd;
                if constexpr (BWD) {
                    const int k = ks * 32 + hi * 8 + (lo >> 2), ch = j * 2 + (lo >> 1 & 1);
                    const uint2 a = read_tr(bd, k * 64 + ((ch ^ (k >> 2 & 3)) << 4) + (lo & 1) * 8);
                    const uint2 b = read_tr(bd, (k + 4) * 64 + ((ch ^ ((k + 4) >> 2 & 3)) << 4) + (lo & 1) * 8);
                    fd = u4_t{a.x, a.y, b.x, b.y};
                }
#pragma unroll
                for (int i = 0; i < MB; i++) {
                    ga[i][j] = mfma16(T{}, fg, xf[i][ks], ga[i][j]);
                    up[i][j] = mfma16(T{}, fu, xf[i][ks], up[i][j]);
                    if constexpr (BWD) dh[i][j] = mfma16(T{}, fd, yf[i][ks], dh[i][j]);
                }
            }
        }
        u4_t v0[MB], v1[BWD ? MB : 1];  // h; or dL/dgate and dL/dup
#pragma unroll
        for (int i = 0; i < MB; i++) {
            const int m = m0 + i * 16 + lo;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                uint16_t q0[4], q1[4], q2[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if constexpr (BWD) {
                        float value, slope;
                        act_grad(g.act, ga[i][j][r], value, slope);
                        q0[r] = narrow(T{}, dh[i][j][r] * up[i][j][r] * slope);
                        q1[r] = narrow(T{}, dh[i][j][r] * value);
                        q2[r] = narrow(T{}, value * up[i][j][r]);
                    } else {
                        q0[r] = narrow(T{}, act_of(g.act, ga[i][j][r]) * up[i][j][r]);
                    }
                }
                v0[i][2 * j] = q0[0] | (uint32_t)q0[1] << 16, v0[i][2 * j + 1] = q0[2] | (uint32_t)q0[3] << 16;
                if constexpr (BWD) {
                    v1[i][2 * j] = q1[0] | (uint32_t)q1[1] << 16, v1[i][2 * j + 1] = q1[2] | (uint32_t)q1[3] << 16;
                    // always a store each, out of range where there is no such row or feature: the waits count them
                    const int f = f0 + j * 16 + hi * 4;
                    const uint32_t at = m < g.rows && f < (int)fp ? (uint32_t)((i * 16 + lo) * (int)fp + f) * 2u : kFar;
                    put8(og, uint2{v0[i][2 * j], v0[i][2 * j + 1]}, at);
                    put8(ou, uint2{v1[i][2 * j], v1[i][2 * j + 1]}, at);
                    put8(oh, uint2{q2[0] | (uint32_t)q2[1] << 16, q2[2] | (uint32_t)q2[3] << 16}, at);
                }
            }
        }
#pragma unroll
        for (int n = 0; n < NB; n++) {
            if constexpr (BWD) {
                const int k = hi * 4 + (lo >> 2), ch = n * 2 + (lo >> 1 & 1);
                const int a = k * ROW + ((ch ^ turn(k)) << 4) + (lo & 1) * 8;
                const int b = (k + 16) * ROW + ((ch ^ turn(k + 16)) << 4) + (lo & 1) * 8;
                const uint2 ga0 = read_tr(bg, a), ga1 = read_tr(bg, b), up0 = read_tr(bu, a), up1 = read_tr(bu, b);
                const u4_t fg = {ga0.x, ga0.y, ga1.x, ga1.y}, fu = {up0.x, up0.y, up1.x, up1.y};
#pragma unroll
                for (int i = 0; i < MB; i++) {
                    acc[i][n] = mfma16(T{}, fg, v0[i], acc[i][n]);
                    acc[i][n] = mfma16(T{}, fu, v1[i], acc[i][n]);
                }
            } else {
                const int row = n * 16 + lo, s = row >> 2 & 3;
                const char* p = reinterpret_cast<const char*>(bd) + row * 64 + (hi & 1) * 8;
                const uint2 a = *reinterpret_cast<const uint2*>(p + (((hi >> 1) ^ s) << 4));
                const uint2 b = *reinterpret_cast<const uint2*>(p + (((2 + (hi >> 1)) ^ s) << 4));
                const u4_t fw = {a.x, a.y, b.x, b.y};
#pragma unroll
                for (int i = 0; i < MB; i++) acc[i][n] = mfma16(T{}, fw, v0[i], acc[i][n]);
            }
        }
    };
    // Slice s has landed, and every wave is done with slice s - 1, whose buffers slice s + 2 takes (see ffn_gemm). Behind
    // the fetch of s a wave has started the stores of step s - 2, the fetch of s + 1 and the stores of s - 1.
    constexpr int STORES = BWD ? 6 * MB : 0;
    auto one = [&](int s, const uint4* bg, const uint4* bu, const uint4* bd, uint4* ng, uint4* nu,
                   uint4* nd) __attribute__((always_inline)) {
        wait_vm<NI + 2 * STORES>();
        __builtin_amdgcn_s_barrier();
        fence();
        fetch(ng, nu, nd);
        multiply(s * 32, bg, bu, bd);
        fence();
    };
    wait_vm<0>();
    const int slices = (g.f + 31) / 32;
    int s = 0;
    for (; s + 3 <= slices; s += 3) {
        one(s, g0, u0, d0, g2, u2, d2);
        one(s + 1, g1, u1, d1, g0, u0, d0);
        one(s + 2, g2, u2, d2, g1, u1, d1);
    }
    if (s < slices) one(s, g0, u0, d0, g2, u2, d2);
    if (s + 1 < slices) one(s + 1, g1, u1, d1, g0, u0, d0);
    wait_vm<0>();

#pragma unroll
    for (int i = 0; i < MB; i++) {
        const int m = m0 + i * 16 + lo;
        if (m >= g.rows || !g.out) continue;
#pragma unroll
        for (int n = 0; n < NB; n++) {
            const int c = n * 16 + hi * 4;
            if (c >= g.c) continue;
            uint16_t q[4];
#pragma unroll
            for (int r = 0; r < 4; r++) q[r] = narrow(T{}, acc[i][n][r]);
            store4(g.out + m * g.ldo + c, g.c - c, q);
        }
    }
}

}  // namespace seq
}  // namespace fhc
