// The matrix products of the gated feed-forward block and of the product with bias, activation and residual
// (include/fhc_seq.h): one tiled kernel over 16-bit operands with f32 accumulation, in the layouts and with the epilogues
// that their forward and backward passes need.
//
// out[m][n] = sum over k of A(m, k) B(n, k). An operand is stored either with k adjacent ("rows": A's row m at
// a + m * ld) or with m (n) adjacent ("columns": A's column k at a + k * ld), so no product needs a transposed copy.
//
// - A workgroup of WM x WN waves computes a BM x BN tile, a wave 16 MB x 16 NB of it, K in slabs of 32. Both operands'
//   slabs go from global memory straight into LDS (LDS DMA, 16 bytes a lane), the next slabs on their way while one
//   computes. Tiles of 128 x 64 and 128 x 128 have four waves and three buffers in turn, one barrier a slab, and several
//   workgroups a CU, whose epilogues and waits lie under each other's products. Tiles of 256 x 256 have eight waves and
//   four buffers; a CU holds one such workgroup, so its halves take turns: while one reads fragments the other
//   multiplies. Measured on the way, TFLOP/s: three buffers and one barrier a slab for all eight waves 990; turns 984
//   with 64-bit lane addresses, 1230 once a row's address is scalar; 128 x 256 tiles, two workgroups a CU, 924 (their LDS
//   traffic). At that rate the matrix units are busy 64% of the cycles and the card's power holds the clock at 1.8 GHz.
//   8192 rows, 2048 channels, 8192 features, bf16: weights' gradients 1270-1350 over three runs, dx 1250-1320, y
//   1140-1155, GLU 890-910 and dL/dh 620-640, whose f32 states pass through the epilogue; a large library product
//   reaches 1307.
// - Rows: an LDS row holds 32 k (64 bytes), its 16-byte chunk c at position c ^ (row >> 2 & 2): a fragment read (16
//   bytes a lane) goes by lanes 0-3, 12-15, 20-23, 24-27 and the like, 16 at once, which so fall on all 64 banks (other
//   permutations of the chunks, by row >> 2 or by 8 neighbours, measured a conflict for every read). Columns: an LDS row
//   holds the tile's m (n) of one k, its 32-byte blocks permuted by f(k) = k & 3 | (k >> 3 & 1) << 2 (64 wide:
//   k >> 1 & 1 | (k >> 3 & 1) << 1); fragments come from the transposing LDS read (16 lanes read 4 k x 16 m and receive
//   4 k of one m each), whose 32 lanes at once then spread over all banks too.
// - The MFMA takes B's fragment as its first operand: a lane's 4 results are 4 adjacent n of one m.
// - Workgroups go round-robin to the 8 XCDs, each with its own L2: the tile index is permuted so that an XCD works on
//   neighbouring tiles, in groups of 8 tile rows.
// - DMA needs 4-byte aligned chunks, and a rows operand's K a multiple of 8 or padded to one with zeros. What the caller
//   gives otherwise is copied into such a form first (ffn_pack). Past an operand's end the buffer's range check gives
//   zeros.
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
    kLinear,  // act(v + bias) + residual; v + bias in f32 too where it is kept (pre_g)
};

struct GemmArgs {
    const uint16_t *a0, *a1, *b0, *b1;
    int64_t lda, ldb;
    int m, n, k;        // kGlu: n is the features, each a gate row of b0 and an up row of b1
    int wide_m, wide_n;  // the columns that a column operand's last row is read to: m (n), to whole 4 bytes
    int segments;       // 2: a0 b0 and then a1 b1 along K (kStore, kPart)
    int pairs;          // 2: a0 -> o0 and a1 -> o1, both with b0 (kStore, kPart)
    int slabs, per_split, splits;  // slabs of 32 over all segments
    int tiles_m, tiles_n;
    uint16_t *o0, *o1;
    int64_t ldo;
    bool dwords;  // kLinear: residual and output of whole, 4-byte aligned pairs
    bool quads;  // kStore: outputs of whole, 8-byte aligned quads, whose offsets in a tile fit 32 bits
    float *pre_g, *pre_u;  // [m][ldpre]
    int64_t ldpre;
    float* part;           // [pair][split][m][ldpart]
    int64_t ldpart;
    uint32_t act;
    const uint16_t *bias, *res;  // kLinear, either may be null
    int64_t ldr;
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
// Far from 0 p is 0 or 1 and the slope is p. w, v held to where gelu's cube is finite, keeps what p multiplies finite: an
// infinity times 0 is not 0. (A NaN comes through p.) This form costs 0 to 1.4% of a training step; those that hold the
// product v k'(v) instead cost up to 4%, by the registers of the one-kernel form.
__device__ __forceinline__ void act_grad(uint32_t act, float v, float& value, float& slope) {
    const bool silu = act == FHC_ACT_SILU;
    const float w = __builtin_amdgcn_fmed3f(v, -1e12f, 1e12f);
    const float k = silu ? v : v * __builtin_fmaf(kGelu3 * v, v, kGelu1);
    const float dk = silu ? 1.0f : __builtin_fmaf(3.0f * kGelu3 * w, w, kGelu1);
    const float e = __builtin_amdgcn_exp2f(k * -1.44269504088896340736f), p = __builtin_amdgcn_rcpf(1.0f + e);
    const float q = __builtin_fminf(e * p, 1.0f);  // 1 - p; inf * 0 where e overflows
    value = v * p;
    slope = p * __builtin_fmaf(w * dk, q, 1.0f);
}

// What kLinear adds to a sum, for up to 4 adjacent columns: pre's rows are whole quads.
struct Tail {
    const uint16_t *bias, *res;
    int64_t ldr;
    float* pre;
    int64_t ldpre;
    uint32_t act;
};
template <class T>
__device__ __forceinline__ void tail4(const Tail& e, int64_t row, int col, int valid, f4 v, uint16_t (&q)[4]) {
#pragma unroll
    for (int r = 0; r < 4; r++)
        if (e.bias && r < valid) v[r] += widen(T{}, e.bias[col + r]);
    if (e.pre) *reinterpret_cast<f4*>(e.pre + row * e.ldpre + col) = v;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        float y = e.act == FHC_ACT_IDENTITY ? v[r] : act_of(e.act, v[r]);
        if (e.res && r < valid) y += widen(T{}, e.res[row * e.ldr + col + r]);
        q[r] = narrow(T{}, y);
    }
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

// One operand's part of a tile: R rows (or columns) of it, a slab of 32 k in LDS, 1 KB (one DMA instruction) per 16 rows
// of 64 bytes, or per 512 / R columns.
template <bool COLS, int R, int NW>
struct Operand {
    static constexpr int NI = R * 64 / 1024 / NW;  // DMA instructions a wave
    static constexpr int CPI = 512 / R;            // COLS: k of an instruction
    static constexpr int U4 = R * 4;               // 16-byte units of a slab
    // COLS: the permutation of a row's 32-byte blocks (4 of them in 64 columns); k and k + 4 have the same
    static __device__ __forceinline__ int blocks_turn(int k) {
        return R == 64 ? (k >> 1 & 1) | (k >> 3 & 1) << 1 : (k & 3) | (k >> 3 & 1) << 2;
    }
    static __device__ __forceinline__ int turn(int row) { return row >> 2 & 2; }
    // the k and the first m (n) of lane `lane`'s 16 bytes of instruction q, relative to the tile and slab
    static __device__ __forceinline__ void place(int inst, int lane, int& r, int& k) {
        if constexpr (COLS) {
            k = inst * CPI + lane / (64 / CPI);
            const int pos = lane % (64 / CPI);
            const int f = blocks_turn(k);
            r = (((pos >> 1) ^ f) << 4) + ((pos & 1) << 3);
        } else {
            r = inst * 16 + (lane >> 2);
            k = ((lane & 3) ^ turn(r)) * 8;
        }
    }
    // the fragment of rows base .. base + 15: lane l has row l & 15, k 8 (l >> 4) .. + 7
    static __device__ __forceinline__ u4_t frag(const uint4* lds, int base, int lane) {
        const char* p = reinterpret_cast<const char*>(lds);
        if constexpr (COLS) {
            const int j = (lane & 15) >> 2, g = lane >> 4;
            const int f = blocks_turn(g * 8 + j);
            // Each address one opaque offset from the buffer: of a sum with a constant the compiler makes a chain, behind
            // which it no longer knows the buffer that is read, and it then waits for the DMA of all.
            [[maybe_unused]] int lo_at = (g * 8 + j) * (R * 2) + (((base >> 4) ^ f) << 5) + (lane & 3) * 8;
            [[maybe_unused]] int hi_at = lo_at + 4 * (R * 2);
            asm("" : "+v"(hi_at));
#if defined(__HIP_DEVICE_COMPILE__)
            typedef __attribute__((address_space(3))) s4_t* lds_s4;
            const s4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p + lo_at));
            const s4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p + hi_at));
            typedef short s8_t __attribute__((ext_vector_type(8)));
            return __builtin_bit_cast(u4_t, (s8_t)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#else
            return u4_t{};
#endif
        } else {
            const int row = base + (lane & 15);
            return *reinterpret_cast<const u4_t*>(p + row * 64 + (((lane >> 4) ^ turn(row)) << 4));
        }
    }
};

constexpr uint32_t kFar = 0x80000000u;  // an offset out of every buffer's range

__host__ __device__ constexpr int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }
template <class P>
__device__ __forceinline__ P* uniform(P* p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return reinterpret_cast<P*>((uint64_t)hi << 32 | lo);
}
template <class R>
__device__ __forceinline__ void put8(R rsrc, uint2 v, uint32_t at) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
    __builtin_amdgcn_raw_buffer_store_b64(u2_t{v.x, v.y}, rsrc, at, 0, 0);
#endif
}
template <class R>
__device__ __forceinline__ uint2 get8(R rsrc, uint32_t at) {
#if defined(__HIP_DEVICE_COMPILE__)
    const auto v = __builtin_amdgcn_raw_buffer_load_b64(rsrc, at, 0, 0);
    return uint2{v[0], v[1]};
#else
    return uint2{};
#endif
}
template <class R>
__device__ __forceinline__ uint32_t get4(R rsrc, uint32_t at) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_raw_buffer_load_b32(rsrc, at, 0, 0);
#else
    return 0;
#endif
}
template <class R>
__device__ __forceinline__ void put4(R rsrc, uint32_t v, uint32_t at) {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_raw_buffer_store_b32(v, rsrc, at, 0, 0);
#endif
}
template <class R>
__device__ __forceinline__ void put16(R rsrc, f4 v, uint32_t at) {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, v), rsrc, at, 0, 0);
#endif
}
// waits until at most N of the wave's vector memory operations are under way, and its LDS reads have arrived
template <int N>
__device__ __forceinline__ void wait_vm() {
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);
}

namespace {  // a kernel of this unit: another one's is registered apart

// WM x WN waves of 16 MB x 16 NB; GLU interleaves B's tile by waves: 8 NB gate rows, then the same features' up rows
template <class T, bool AC, bool BC, Epi E, int MB, int NB, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void ffn_gemm(GemmArgs g) {
    constexpr int NW = WM * WN, BM = 16 * MB * WM, BN = 16 * NB * WN;
    constexpr int FW = E == kGlu ? 8 * NB : 16 * NB, FN = FW * WN;  // features of a wave, of a tile
    using OA = Operand<AC, BM, NW>;
    using OB = Operand<BC, BN, NW>;
    constexpr int NI = OA::NI + OB::NI;
    constexpr bool TURNS = NW == 8;
    // one object per buffer: the compiler's wait for a DMA then covers only reads of the buffer it fills
    __shared__ __align__(1024) uint4 as0[OA::U4], bs0[OB::U4], as1[OA::U4], bs1[OB::U4], as2[OA::U4], bs2[OB::U4];
    __shared__ __align__(1024) uint4 as3[TURNS ? OA::U4 : 1], bs3[TURNS ? OB::U4 : 1];

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
    int ka[OA::NI], kb[OB::NI];
#pragma unroll
    for (int q = 0; q < OA::NI; q++) {
        int r;
        OA::place(wave * OA::NI + q, lane, r, ka[q]);
        offa[q] = (uint32_t)(AC ? ka[q] * (int)g.lda + r : r * (int)g.lda + ka[q]) * 2u;
    }
#pragma unroll
    for (int q = 0; q < OB::NI; q++) {
        int r;
        OB::place(wave * OB::NI + q, lane, r, kb[q]);
        if constexpr (E == kGlu) r = r / (2 * FW) * FW + r % FW;  // the feature; gate or up is the instruction's
        offb[q] = (uint32_t)(BC ? kb[q] * (int)g.ldb + r : r * (int)g.ldb + kb[q]) * 2u;
    }

    // The fetches run through the slabs in order. Of each operand: the address of the tile's part of the next slab, and
    // the bytes from there to its end, behind which the range check gives zeros.
    const int64_t step_a = (AC ? 32 * g.lda : 32) * 2, step_b = (BC ? 32 * g.ldb : 32) * 2;
    const char *pa, *pb, *pu;
    int64_t ra, rb;
    int kleft, switch_at = g.segments > 1 && s0 < seg_slabs ? seg_slabs - s0 : -1;  // fetches until the second segment
    auto start = [&](int seg, int slab) {
        const int64_t k0 = slab * 32;
        const int64_t ea = AC ? k0 * g.lda + m0 : m0 * g.lda + k0, eb = BC ? k0 * g.ldb + n0 : n0 * g.ldb + k0;
        const int64_t enda = AC ? (g.k - 1) * g.lda + g.wide_m : (g.m - 1) * g.lda + up8(g.k);
        const int64_t endb = BC ? (g.k - 1) * g.ldb + g.wide_n : (g.n - 1) * g.ldb + up8(g.k);
        pa = uniform(reinterpret_cast<const char*>((seg + pair ? g.a1 : g.a0) + ea));
        pb = uniform(reinterpret_cast<const char*>((seg ? g.b1 : g.b0) + eb));
        if constexpr (E == kGlu) pu = uniform(reinterpret_cast<const char*>(g.b1 + eb));
        ra = (enda - ea) * 2, rb = (endb - eb) * 2, kleft = g.k - (int)k0;
    };
    start(g.segments > 1 && s0 >= seg_slabs, g.segments > 1 && s0 >= seg_slabs ? s0 - seg_slabs : s0);
    auto resource = [](const char* p, int64_t bytes) {
        const int hi = (int)(bytes >> 32), n = hi < 0 ? 0 : hi > 0 || (int)bytes < 0 ? 0x7FFFFFFF : (int)bytes;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), (short)0, n, 0x00020000);
    };
    // starts the next slab's way into the buffers
    auto fetch = [&](uint4* la, uint4* lb) {
        if (switch_at-- == 0) start(1, 0);
        const auto rsa = resource(pa, ra), rsb = resource(pb, rb), rsu = resource(E == kGlu ? pu : pb, rb);
        const bool whole = kleft >= 32;  // else a row's chunk past the end of K lies in the next row
#pragma unroll
        for (int q = 0; q < OA::NI; q++)
            lds_dma16(rsa, la + (wave * OA::NI + q) * 64, AC || whole || ka[q] < kleft ? offa[q] : kFar);
#pragma unroll
        for (int q = 0; q < OB::NI; q++) {
            const int inst = wave * OB::NI + q;
            const bool up = E == kGlu && (inst * 16 & FW);
            lds_dma16(up ? rsu : rsb, lb + inst * 64, BC || whole || kb[q] < kleft ? offb[q] : kFar);
        }
        pa += step_a, pb += step_b, ra -= step_a, rb -= step_b, kleft -= 32;
        if constexpr (E == kGlu) pu += step_b;
    };

    f4 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
        for (int j = 0; j < NB; j++) acc[i][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    u4_t fb[NB], fa[MB];
    auto read = [&](const uint4* la, const uint4* lb) {
        int at = lane;
#pragma unroll
        for (int j = 0; j < NB; j++) fb[j] = OB::frag(lb, (wn * NB + j) * 16, at);
#pragma unroll
        for (int i = 0; i < MB; i++) fa[i] = OA::frag(la, (wm * MB + i) * 16, at);
    };
    auto multiply = [&] {
#pragma unroll
        for (int i = 0; i < MB; i++)
#pragma unroll
            for (int j = 0; j < NB; j++) acc[i][j] = mfma16(T{}, fb[j], fa[i], acc[i][j]);
    };
    // What would follow the last slab is fetched too, so that the number under way is known at every wait; no kernel may
    // end before it has landed. The fetches stay in this order: the waits count them.
    auto fence = [] { asm volatile("" ::: "memory"); };
    fetch(as0, bs0);
    fence();
    fetch(as1, bs1);
    fence();
    int s = s0;
    // (what is left over is not an exit from the loop's middle: the compiler would join it with the loop's head, and its
    // own waits would then be for both)
    if constexpr (TURNS) {
        // The two halves of the workgroup, one wave of each on every SIMD, take turns: while one reads a slab's
        // fragments and starts the fetch of slab s + 3, the other multiplies. A barrier ends every phase; the second
        // half enters one phase late and leaves one late.
        //   A half's phase of reading s: slab s has landed in all waves (each waits for its share of slab s + 1 at the
        //   end of its reading of s, two phases before anyone reads that), and slab s - 1, whose buffers s + 3 takes, was
        //   last read one phase ago, with its reads waited for before the barrier.
        auto phase_end = [&] {
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            fence();
        };
        auto step = [&](const uint4* la, const uint4* lb, uint4* na, uint4* nb) {
            fetch(na, nb);
            read(la, lb);
            wait_vm<2 * NI>();
            phase_end();
            __builtin_amdgcn_s_setprio(1);
            multiply();
            __builtin_amdgcn_s_setprio(0);
            phase_end();
        };
        fetch(as2, bs2);
        wait_vm<2 * NI>();
        phase_end();
        if (wave >= NW / 2) phase_end();
        for (; s + 4 <= s1; s += 4) {
            step(as0, bs0, as3, bs3);
            step(as1, bs1, as0, bs0);
            step(as2, bs2, as1, bs1);
            step(as3, bs3, as2, bs2);
        }
        if (s < s1) step(as0, bs0, as3, bs3);
        if (s + 1 < s1) step(as1, bs1, as0, bs0);
        if (s + 2 < s1) step(as2, bs2, as1, bs1);
        if (wave < NW / 2) phase_end();
    } else {
        // Slab s has landed, and every wave is done with slab s - 1, whose buffers slab s + 2 takes while s computes.
        auto step = [&](const uint4* la, const uint4* lb, uint4* na, uint4* nb) {
            wait_vm<NI>();
            __builtin_amdgcn_s_barrier();
            fence();
            fetch(na, nb);
            read(la, lb);
            multiply();
            fence();
        };
        for (; s + 3 <= s1; s += 3) {
            step(as0, bs0, as2, bs2);
            step(as1, bs1, as0, bs0);
            step(as2, bs2, as1, bs1);
        }
        if (s < s1) step(as0, bs0, as2, bs2);
        if (s + 1 < s1) step(as1, bs1, as0, bs0);
    }
    wait_vm<0>();

    // ---- The epilogue: rows m0 + .., columns n0 + .. of the outputs, by buffer stores whose offsets are out of range
    // where there is no such row or column (no branches: they would be most of the code, which a short launch fetches
    // for the first time).
    const int mr = wm * 16 * MB + (lane & 15), nr = wn * FW + 4 * (lane >> 4);  // in the tile, with 16 i and 16 j
    auto place = [&](int i, int j, int64_t ld, int cols, uint32_t elem) -> uint32_t {
        const int m = mr + i * 16, n = nr + j * 16;
        return m0 + m < g.m && n0 + n < cols ? (uint32_t)(m * (int)ld + n) * elem : kFar;
    };
    auto at_tile = [&](auto* p, int64_t ld) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(uniform(reinterpret_cast<const char*>(p + m0 * ld + n0))),
                                                 (short)0, 0x7FFFFFFF, 0x00020000);
    };
    auto pack = [](const uint16_t (&q)[4]) { return uint2{q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16}; };
    if constexpr (E == kGrad) {  // o0 and o1 have rows of up8(n), whose ends are zeros
        const auto t0 = at_tile(g.o0, g.ldo), t1 = at_tile(g.o1, g.ldo);
        // both products of the next 16 rows are on their way while 16 rows are worked on; past the edge, the last ones
        f4 ga[2][NB], up[2][NB];
        auto load = [&](int i) {
            const int64_t row = min(m0 + mr + i * 16, g.m - 1) * g.ldpre;
#pragma unroll
            for (int j = 0; j < NB; j++) {
                const int64_t at = row + min(n0 + nr + j * 16, (int)g.ldpre - 4);
                ga[i & 1][j] = *reinterpret_cast<const f4*>(g.pre_g + at);
                up[i & 1][j] = *reinterpret_cast<const f4*>(g.pre_u + at);
            }
        };
        load(0);
#pragma unroll
        for (int i = 0; i < MB; i++) {
            if (i + 1 < MB) load(i + 1);
#pragma unroll
            for (int j = 0; j < NB; j++) {
                const int n = n0 + nr + j * 16;
                const f4 v = acc[i][j];
                uint16_t qg[4], qu[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float value, slope;
                    act_grad(g.act, ga[i & 1][j][r], value, slope);
                    qg[r] = n + r < g.n ? narrow(T{}, v[r] * up[i & 1][j][r] * slope) : (uint16_t)0;
                    qu[r] = n + r < g.n ? narrow(T{}, v[r] * value) : (uint16_t)0;
                }
                const uint32_t at = place(i, j, g.ldo, (int)g.ldo, 2);
                put8(t0, pack(qg), at);
                put8(t1, pack(qu), at);
            }
        }
    } else if constexpr (E == kGlu) {  // as have o0, pre_g and pre_u
        const auto th = at_tile(g.o0, g.ldo), tg = at_tile(g.pre_g, g.ldpre), tu = at_tile(g.pre_u, g.ldpre);
#pragma unroll
        for (int i = 0; i < MB; i++) {
#pragma unroll
            for (int j = 0; j < NB / 2; j++) {
                const f4 ga = acc[i][j], up = acc[i][j + NB / 2];
                uint16_t q[4];
#pragma unroll
                for (int r = 0; r < 4; r++) q[r] = narrow(T{}, act_of(g.act, ga[r]) * up[r]);  // 0 past n: both are 0
                put8(th, pack(q), place(i, j, g.ldo, (int)g.ldo, 2));
                if (g.pre_g) {
                    const uint32_t at = place(i, j, g.ldpre, (int)g.ldpre, 4);
                    put16(tg, ga, at);
                    put16(tu, up, at);
                }
            }
        }
    } else if constexpr (E == kLinear) {
        const Tail tail{g.bias, g.res, g.ldr, g.pre_g, g.ldpre, g.act};
        // PAIRS: a lane's 4 columns as two dwords, each inside or out as a whole
        auto rows = [&](auto pairs) __attribute__((always_inline)) {
            constexpr bool PAIRS = pairs;
            const auto ty = at_tile(g.o0, g.ldo), tr = at_tile(g.res ? g.res : g.o0, g.res ? g.ldr : g.ldo);
            const auto tp = at_tile(g.pre_g, g.ldpre);
            f4 bias[NB];
#pragma unroll
            for (int j = 0; j < NB; j++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    bias[j][r] = g.bias ? widen(T{}, g.bias[min(n0 + nr + j * 16 + r, g.n - 1)]) : 0.0f;
            // of a quad the second dword, out of range where its columns are
            auto second = [&](int j, uint32_t at) { return n0 + nr + j * 16 + 2 < g.n ? at + 4 : kFar; };
            // the residual's next 16 rows are on their way while 16 rows are worked on (y may lie over it: an element is
            // read before it is written, by the same lane)
            uint2 rr[2][NB];
            auto load = [&](int i) {
#pragma unroll
                for (int j = 0; j < NB; j++) {
                    const uint32_t at = place(i, j, g.ldr, g.n, 2);
                    rr[i & 1][j] = PAIRS ? uint2{get4(tr, at), get4(tr, second(j, at))} : get8(tr, at);
                }
            };
            if (g.res) load(0);
#pragma unroll
            for (int i = 0; i < MB; i++) {
                if (g.res && i + 1 < MB) load(i + 1);
#pragma unroll
                for (int j = 0; j < NB; j++) {
                    f4 v = acc[i][j] + bias[j];
                    if (g.pre_g) put16(tp, v, place(i, j, g.ldpre, (int)g.ldpre, 4));
                    if (g.act != FHC_ACT_IDENTITY) {
#pragma unroll
                        for (int r = 0; r < 4; r++) v[r] = act_of(g.act, v[r]);
                    }
                    if (g.res) {
                        const uint2 e = rr[i & 1][j];
                        const uint16_t h[4] = {(uint16_t)e.x, (uint16_t)(e.x >> 16), (uint16_t)e.y, (uint16_t)(e.y >> 16)};
#pragma unroll
                        for (int r = 0; r < 4; r++) v[r] += widen(T{}, h[r]);
                    }
                    uint16_t q[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) q[r] = narrow(T{}, v[r]);
                    const uint2 o = pack(q);
                    const uint32_t at = place(i, j, g.ldo, g.n, 2);
                    if (PAIRS) put4(ty, o.x, at), put4(ty, o.y, second(j, at));
                    else put8(ty, o, at);
                }
            }
        };
        if (g.quads) {
            rows(std::false_type{});
        } else if (g.dwords) {
            rows(std::true_type{});
        } else {
#pragma unroll
            for (int i = 0; i < MB; i++) {
                const int m = m0 + mr + i * 16;
                if (m >= g.m) continue;
#pragma unroll
                for (int j = 0; j < NB; j++) {
                    const int n = n0 + nr + j * 16;
                    if (n >= g.n) continue;
                    uint16_t q[4];
                    tail4<T>(tail, m, n, g.n - n, acc[i][j], q);
                    store4(g.o0 + m * g.ldo + n, g.n - n, q);
                }
            }
        }
    } else if constexpr (E == kPart) {
        const auto t = at_tile(g.part + (int64_t)(pair * g.splits + split) * g.m * g.ldpart, g.ldpart);
#pragma unroll
        for (int i = 0; i < MB; i++)
#pragma unroll
            for (int j = 0; j < NB; j++) put16(t, acc[i][j], place(i, j, g.ldpart, g.n, 4));
    } else if (g.quads) {
        const auto t = at_tile(pair ? g.o1 : g.o0, g.ldo);
#pragma unroll
        for (int i = 0; i < MB; i++) {
#pragma unroll
            for (int j = 0; j < NB; j++) {
                uint16_t q[4];
#pragma unroll
                for (int r = 0; r < 4; r++) q[r] = narrow(T{}, acc[i][j][r]);
                put8(t, pack(q), place(i, j, g.ldo, g.n, 2));
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < MB; i++) {
            const int m = m0 + mr + i * 16;
            if (m >= g.m) continue;
#pragma unroll
            for (int j = 0; j < NB; j++) {
                const int n = n0 + nr + j * 16;
                if (n >= g.n) continue;
                uint16_t q[4];
#pragma unroll
                for (int r = 0; r < 4; r++) q[r] = narrow(T{}, acc[i][j][r]);
                store4((pair ? g.o1 : g.o0) + m * g.ldo + n, g.n - n, q);
            }
        }
    }
}

}  // namespace
}  // namespace seq
}  // namespace fhc
