// The matrix products of the gated feed-forward block (include/fhc_seq.h): one tiled kernel over 16-bit operands with
// f32 accumulation, in the layouts and with the epilogues that the block's forward and backward passes need.
//
// out[m][n] = sum over k of A(m, k) B(n, k). An operand is stored either with k adjacent ("rows": A's row m at
// a + m * ld) or with m (n) adjacent ("columns": A's column k at a + k * ld), so no product needs a transposed copy.
//
// - A workgroup computes a BM x BN tile, wave (wm, wn) a 16 MB x 64 part of it, K in slabs of 64. Both operands' slabs
//   go from global memory straight into LDS (LDS DMA, 16 bytes a lane), two buffers in turn: slab s + 1 loads while
//   slab s computes, one barrier a slab.
// - Rows: an LDS row holds 64 k (128 bytes), its 16-byte chunk c at position c ^ (row & 7), so that the 16 rows of a
//   fragment read (16 bytes a lane) spread over all banks. Columns: an LDS row holds the tile's m (n) of one k, its
//   32-byte blocks permuted by f(k) = k & 3 | (k >> 3 & 1) << 2; fragments come from the transposing LDS read (16 lanes
//   read 4 k x 16 m and receive 4 k of one m each), whose 32 lanes at once then spread over all banks too.
// - The MFMA takes B's fragment as its first operand: a lane's 4 results are 4 adjacent n of one m.
// - Workgroups go round-robin to the 8 XCDs, each with its own L2: the tile index is permuted so that an XCD works on
//   neighbouring tiles, in groups of 8 tile rows.
// - DMA needs 4-byte aligned chunks: even widths and strides. Odd ones go through registers (element-aligned loads).
// - Past an operand's end the buffer's range check gives zeros; a k group of 8 that the end of K cuts is zeroed in LDS
//   (both operands: what lies past a row's end may be anything, NaN included).
#pragma once
#include "seq_common.h"
#include "wave_impl.h"

namespace fhc {
namespace seq {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef short s4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f4 mfma16(F16, u4_t a, u4_t b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f4 mfma16(BF16, u4_t a, u4_t b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

enum Epi {
    kStore,  // out, 16 bits
    kPart,   // f32 partial sums of a split K
    kGlu,    // N counts gate and up rows: h = act(gate) * up, and both in f32 where they are kept
    kGrad,   // dh -> dL/dgate, dL/dup
};

struct GemmArgs {
    const uint16_t *a0, *a1, *b0, *b1;
    int64_t lda, ldb;
    int m, n, k;        // kGlu: n is the features, each a gate row of b0 and an up row of b1
    int segments;       // 2: a0 b0 and then a1 b1 along K (kStore, kPart)
    int pairs;          // 2: a0 -> o0 and a1 -> o1, both with b0 (kStore, kPart)
    int slabs, per_split, splits;  // slabs of 64 over all segments, an even number of each; per_split even
    int tiles_m, tiles_n;
    uint16_t *o0, *o1;
    int64_t ldo;
    float *pre_g, *pre_u;  // [m][ldpre]
    int64_t ldpre;
    float* part;           // [pair][split][m][ldpart]
    int64_t ldpart;
    uint32_t act;
};

// act(v) = v sigmoid(k(v)), k(v) = v (silu) or 2 sqrt(2 / pi) (v + 0.044715 v^3) (gelu, tanh form)
__device__ __forceinline__ float sigmoid_of(float v) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.44269504088896340736f));
}
constexpr float kGelu1 = 1.59576912160573071176f, kGelu3 = kGelu1 * 0.044715f;
__device__ __forceinline__ float act_of(uint32_t act, float v) {
    const float k = act == FHC_ACT_SILU ? v : v * __builtin_fmaf(kGelu3 * v, v, kGelu1);
    return v * sigmoid_of(k);
}
__device__ __forceinline__ void act_grad(uint32_t act, float v, float& value, float& slope) {
    const bool silu = act == FHC_ACT_SILU;
    const float k = silu ? v : v * __builtin_fmaf(kGelu3 * v, v, kGelu1);
    const float dk = silu ? 1.0f : __builtin_fmaf(3.0f * kGelu3 * v, v, kGelu1);
    const float p = sigmoid_of(k), q = sigmoid_of(-k);
    value = v * p;
    slope = p * __builtin_fmaf(v * dk, q, 1.0f);
}

// up to 8 elements at p, `valid` of them inside
__device__ __forceinline__ u4_t load_some(const uint16_t* p, int valid) {
    if (valid >= 8) {
        uint16_t q[8];
        load_raw<uint16_t, 8, false>(p, q);
        u4_t r;
#pragma unroll
        for (int i = 0; i < 4; i++) r[i] = q[2 * i] | (uint32_t)q[2 * i + 1] << 16;
        return r;
    }
    u4_t r = {0, 0, 0, 0};
    for (int i = 0; i < valid; i++) r[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
    return r;
}

__device__ __forceinline__ void store4(uint16_t* p, int valid, const uint16_t (&q)[4]) {
    if (valid >= 4) {
        store_raw<uint16_t, 4, false>(p, q);
    } else {
        for (int i = 0; i < valid; i++) p[i] = q[i];
    }
}

// One operand's part of a tile: R rows (or columns) of it, a slab of 64 k in LDS, 1 KB (one DMA instruction) per 8 rows
// of 128 bytes, or per 512 / R columns.
template <bool COLS, int R, int NW>
struct Operand {
    static constexpr int NI = R * 128 / 1024 / NW;  // DMA instructions a wave
    static constexpr int CPI = 512 / R;             // COLS: k of an instruction
    // the k and the first m (n) of lane `lane`'s 16 bytes of instruction q, relative to the tile and slab
    static __device__ __forceinline__ void place(int inst, int lane, int& r, int& k) {
        if constexpr (COLS) {
            k = inst * CPI + lane / (64 / CPI);
            const int pos = lane % (64 / CPI);
            const int f = (k & 3) | (k >> 3 & 1) << 2;
            r = (((pos >> 1) ^ f) << 4) + ((pos & 1) << 3);
        } else {
            r = inst * 8 + (lane >> 3);
            k = ((lane & 7) ^ (lane >> 3)) * 8;
        }
    }
    // the fragment of rows base .. base + 15, k step ks of 32: lane l has row l & 15, k 8 (l >> 4) .. + 7
    static __device__ __forceinline__ u4_t frag(const uint4* lds, int base, int ks, int lane) {
        const char* p = reinterpret_cast<const char*>(lds);
        if constexpr (COLS) {
            const int j = (lane & 15) >> 2, g = lane >> 4;
            const int f = j | (g & 1) << 2;
            [[maybe_unused]] const char* at =
                p + (ks * 32 + g * 8 + j) * (R * 2) + (((base >> 4) ^ f) << 5) + (lane & 3) * 8;
#if defined(__HIP_DEVICE_COMPILE__)
            typedef __attribute__((address_space(3))) s4_t* lds_s4;
            const s4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)at);
            const s4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(at + 4 * (R * 2)));
            typedef short s8_t __attribute__((ext_vector_type(8)));
            return __builtin_bit_cast(u4_t, (s8_t)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#else
            return u4_t{};
#endif
        } else {
            const int row = base + (lane & 15);
            return *reinterpret_cast<const u4_t*>(p + row * 128 + (((ks * 4 + (lane >> 4)) ^ (lane & 7)) << 4));
        }
    }
};

constexpr uint32_t kFar = 0x80000000u;  // an offset out of every buffer's range

// WM x WN waves of 16 MB x 64; GLU interleaves B's tile by waves: 32 gate rows, then the same features' 32 up rows
template <class T, bool AC, bool BC, Epi E, int MB, int WM, int WN, bool DMA>
__global__ __launch_bounds__(64 * WM * WN) void ffn_gemm(GemmArgs g) {
    constexpr int NW = WM * WN, BM = 16 * MB * WM, BN = 64 * WN;
    constexpr int FN = E == kGlu ? BN / 2 : BN;  // features of a tile
    using OA = Operand<AC, BM, NW>;
    using OB = Operand<BC, BN, NW>;
    // one object per buffer: the compiler's wait for a DMA then covers only reads of the buffer it fills
    __shared__ __align__(1024) uint4 as0[BM * 8], as1[BM * 8], bs0[BN * 8], bs1[BN * 8];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave % WN, wm = wave / WN;
    int tm, tn;
    {
        const int tiles = g.tiles_m * g.tiles_n, q = tiles / 8, r = tiles % 8;
        const int x = blockIdx.x % 8, at = x * q + min(x, r) + blockIdx.x / 8;
        const int wide = 8 * g.tiles_n, gr = at / wide, in = at - gr * wide;
        const int rows = min(g.tiles_m - gr * 8, 8);
        tm = gr * 8 + in % rows, tn = in / rows;
    }
    const int m0 = tm * BM, n0 = tn * FN;
    const int pair = g.pairs > 1 ? blockIdx.z / g.splits : 0, split = blockIdx.z - pair * g.splits;
    const int s0 = split * g.per_split, s1 = min(g.slabs, s0 + g.per_split);
    const int seg_slabs = g.slabs / g.segments;

    // per-lane offsets of the DMA (bytes from the tile's first element), and k within the slab of a row's chunk
    uint32_t offa[OA::NI], offb[OB::NI];
    int ka[OA::NI], kb[OB::NI], ra[OA::NI], rb[OB::NI];
#pragma unroll
    for (int q = 0; q < OA::NI; q++) {
        OA::place(wave * OA::NI + q, lane, ra[q], ka[q]);
        offa[q] = (uint32_t)(AC ? ka[q] * (int)g.lda + ra[q] : ra[q] * (int)g.lda + ka[q]) * 2u;
    }
#pragma unroll
    for (int q = 0; q < OB::NI; q++) {
        OB::place(wave * OB::NI + q, lane, rb[q], kb[q]);
        if constexpr (E == kGlu) rb[q] = (rb[q] >> 6) * 32 + (rb[q] & 31);  // the feature; gate or up is the wave's
        offb[q] = (uint32_t)(BC ? kb[q] * (int)g.ldb + rb[q] : rb[q] * (int)g.ldb + kb[q]) * 2u;
    }

    auto range = [](int64_t bytes) { return (int)(bytes < 0 ? 0 : bytes > 0x7FFFFFFF ? 0x7FFFFFFF : bytes); };
    u4_t rega[DMA ? 1 : OA::NI], regb[DMA ? 1 : OB::NI];
    // starts slab s's way into the buffers (into registers on the odd path)
    auto fetch = [&](int s, uint4* la, uint4* lb) {
        const int seg = s >= seg_slabs ? 1 : 0;
        const int k0 = (s - seg * seg_slabs) * 64;
        const uint16_t* a = seg + pair ? g.a1 : g.a0;
        const uint16_t* b = seg ? g.b1 : g.b0;
        if constexpr (DMA) {
            const int64_t ea = AC ? (int64_t)k0 * g.lda + m0 : (int64_t)m0 * g.lda;
            const int64_t eb = BC ? (int64_t)k0 * g.ldb + n0 : (int64_t)n0 * g.ldb;
            const int64_t enda = AC ? (int64_t)(g.k - 1) * g.lda + g.m : (int64_t)(g.m - 1) * g.lda + g.k;
            const int64_t endb = BC ? (int64_t)(g.k - 1) * g.ldb + g.n : (int64_t)(g.n - 1) * g.ldb + g.k;
            const auto rsa = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a + ea), (short)0,
                                                               range((enda - ea) * 2), 0x00020000);
            const auto rsb = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(b + eb), (short)0,
                                                               range((endb - eb) * 2), 0x00020000);
            const auto rsu = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<uint16_t*>((E == kGlu ? g.b1 : b) + eb), (short)0, range((endb - eb) * 2), 0x00020000);
#pragma unroll
            for (int q = 0; q < OA::NI; q++) {
                uint32_t off = offa[q];
                if constexpr (!AC) off = k0 + ka[q] < g.k ? off + 2u * k0 : kFar;
                lds_dma16(rsa, la + (wave * OA::NI + q) * 64, off);
            }
#pragma unroll
            for (int q = 0; q < OB::NI; q++) {
                const int inst = wave * OB::NI + q;
                uint32_t off = offb[q];
                if constexpr (!BC) off = k0 + kb[q] < g.k ? off + 2u * k0 : kFar;
                lds_dma16(E == kGlu && (inst & 4) ? rsu : rsb, lb + inst * 64, off);
            }
        } else {
#pragma unroll
            for (int q = 0; q < OA::NI; q++) {
                const int r = m0 + ra[q], k = k0 + ka[q];
                const int valid = AC ? (k < g.k ? g.m - r : 0) : (r < g.m ? g.k - k : 0);
                rega[q] = load_some(a + (AC ? (int64_t)k * g.lda + r : (int64_t)r * g.lda + k), valid);
            }
#pragma unroll
            for (int q = 0; q < OB::NI; q++) {
                const int r = n0 + rb[q], k = k0 + kb[q];
                const int valid = BC ? (k < g.k ? g.n - r : 0) : (r < g.n ? g.k - k : 0);
                const uint16_t* p = E == kGlu && (wave * OB::NI + q & 4) ? g.b1 : b;
                regb[q] = load_some(p + (BC ? (int64_t)k * g.ldb + r : (int64_t)r * g.ldb + k), valid);
            }
        }
    };
    auto land = [&](uint4* la, uint4* lb) {
        if constexpr (!DMA) {
#pragma unroll
            for (int q = 0; q < OA::NI; q++)
                *reinterpret_cast<u4_t*>(la + (wave * OA::NI + q) * 64 + lane) = rega[q];
#pragma unroll
            for (int q = 0; q < OB::NI; q++)
                *reinterpret_cast<u4_t*>(lb + (wave * OB::NI + q) * 64 + lane) = regb[q];
        }
    };
    // zeroes the end of the 8-group that the end of K cuts in slab s
    auto trim = [&](int s, uint4* la, uint4* lb) {
        if constexpr (DMA) {
            const int left = g.k - (s >= seg_slabs ? s - seg_slabs : s) * 64;
            if (left >= 64 || left <= 0 || !(left & 7)) return;
            auto cut = [&](uint4* p, int rows) {
                for (int r = tid; r < rows; r += 64 * NW) {
                    uint16_t* e = reinterpret_cast<uint16_t*>(p + r * 8 + ((left >> 3) ^ (r & 7)));
                    for (int i = left & 7; i < 8; i++) e[i] = 0;
                }
            };
            if constexpr (!AC) cut(la, BM);
            if constexpr (!BC) cut(lb, BN);
            __syncthreads();
        }
    };

    f4 acc[MB][4];
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    auto compute = [&](const uint4* la, const uint4* lb) {
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            u4_t fb[4], fa[MB];
#pragma unroll
            for (int j = 0; j < 4; j++) fb[j] = OB::frag(lb, wn * 64 + j * 16, ks, lane);
#pragma unroll
            for (int i = 0; i < MB; i++) fa[i] = OA::frag(la, wm * 16 * MB + i * 16, ks, lane);
#pragma unroll
            for (int i = 0; i < MB; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = mfma16(T{}, fb[j], fa[i], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);  // no fragment of the next step is read early: registers
        }
    };

    // slabs come in pairs (the host rounds up; one past the end of K is all zeros): a loop left in its middle would
    // need a second copy of the accumulators
    fetch(s0, as0, bs0);
    land(as0, bs0);
    __syncthreads();
    for (int s = s0; s < s1; s += 2) {
        trim(s, as0, bs0);
        fetch(s + 1, as1, bs1);
        compute(as0, bs0);
        land(as1, bs1);
        __syncthreads();
        trim(s + 1, as1, bs1);
        if (s + 2 < s1) fetch(s + 2, as0, bs0);
        compute(as1, bs1);
        if (s + 2 < s1) land(as0, bs0);
        __syncthreads();
    }

    const int mw = m0 + wm * 16 * MB + (lane & 15), quad = 4 * (lane >> 4);
#pragma unroll
    for (int i = 0; i < MB; i++) {
        const int m = mw + i * 16;
        if (m >= g.m) continue;
        if constexpr (E == kGlu) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int f = n0 + wn * 32 + j * 16 + quad;
                if (f >= g.n) continue;
                const f4 ga = acc[i][j], up = acc[i][j + 2];
                uint16_t q[4];
#pragma unroll
                for (int r = 0; r < 4; r++) q[r] = narrow(T{}, act_of(g.act, ga[r]) * up[r]);
                store4(g.o0 + m * g.ldo + f, g.n - f, q);
                if (g.pre_g) {  // rows padded to 8: a whole vector always fits
                    *reinterpret_cast<f4*>(g.pre_g + m * g.ldpre + f) = ga;
                    *reinterpret_cast<f4*>(g.pre_u + m * g.ldpre + f) = up;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int n = n0 + wn * 64 + j * 16 + quad;
                if (n >= g.n) continue;
                const f4 v = acc[i][j];
                if constexpr (E == kPart) {
                    *reinterpret_cast<f4*>(g.part + ((int64_t)(pair * g.splits + split) * g.m + m) * g.ldpart + n) = v;
                } else if constexpr (E == kGrad) {
                    const f4 ga = *reinterpret_cast<const f4*>(g.pre_g + m * g.ldpre + n);
                    const f4 up = *reinterpret_cast<const f4*>(g.pre_u + m * g.ldpre + n);
                    uint16_t qg[4], qu[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        float value, slope;
                        act_grad(g.act, ga[r], value, slope);
                        qg[r] = narrow(T{}, v[r] * up[r] * slope);
                        qu[r] = narrow(T{}, v[r] * value);
                    }
                    store4(g.o0 + m * g.ldo + n, g.n - n, qg);
                    store4(g.o1 + m * g.ldo + n, g.n - n, qu);
                } else {
                    uint16_t q[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) q[r] = narrow(T{}, v[r]);
                    store4((pair ? g.o1 : g.o0) + m * g.ldo + n, g.n - n, q);
                }
            }
        }
    }
}

}  // namespace seq
}  // namespace fhc
