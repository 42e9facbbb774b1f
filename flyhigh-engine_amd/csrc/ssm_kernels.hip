// The selective state space scan (include/fhc_seq.h), forward and backward.
//
// A workgroup has 64 channels of one sequence and group, a lane one channel; its W waves share out the states, 2, 4 or 8 of
// them a wave, in registers. Time goes in tiles of 16 steps: the waves first prepare 16 / W steps each (D = softplus,
// D x), which then lie in LDS for all of them; every wave runs its states through the 16 steps and leaves its part of
// sum C h a step in LDS; the waves add the parts of their steps, apply skip and gate, and store. B and C are the same for
// all lanes: a register holds them for 4 steps x 4 states in every row of 16 lanes, and a fused multiply-add takes a lane
// of its row for an operand (DPP).
//
// Where the columns are too few for the chip, time is cut into segments: a first launch folds each to the state that it
// leaves from zeros, and its sum of D (its decay is exp(a sum D), so one number a channel composes all of them); the
// second launch starts each segment from the fold of those before it.
//
// Backward, with q = dy silu(z) and c the gradient that reaches a step's state from behind:
//     g_t = C_t q_t + c,   c <- a_t g_t,   s1 = sum B g,   s2 = sum a[k] a_t h_(t-1) g
//     dx = D s1 + skip q,   ddt = (s2 + x s1) sigmoid(dt + bias),   dz = dy p silu'(z)
//     da[k] = sum of D a_t h_(t-1) g,   dB = sum over channels of D x g,   dC = sum over channels of q h
// The forward pass keeps every tile's first state; a tile's 16 states and decays are computed again into registers and
// walked backwards. The sums over a wave's 64 channels for dB and dC go through LDS; a closing launch adds the channel
// blocks, in their order.
#include "seq_args.h"

namespace fhc {
namespace seq {
namespace {

constexpr int kTile = 16;
constexpr uint32_t kStretch = 16;  // tiles whose terms of a weight's gradient are added in f32; the closing sum is f64
typedef float f4 __attribute__((ext_vector_type(4)));
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

template <class R>
struct SsmArgs {
    Seq<R> x, dt, bm, cm, z, y, dy, dx, ddt, dz;
    const float *a, *bias, *skip;
    const int32_t* lengths;
    const float* h0;
    float* ht;
    f4* states;    // [b][tile][quad][d]
    const float* dht;
    float* dh0;
    f4* ends;     // segments: [segment + 1][b][quad][d], forward's slot 0 is h0
    float* lasts;   // and their sums of D, [segment][b][d]
    float* part;    // [segment][walk][stretch][d * n + 2 d]: da, dskip, ddt_bias
    float* bc;      // [group and block][b][t][2][quad * 4]
    uint32_t b, t, d, n, groups;
    uint32_t width, blocks, quads;    // channels of a group, its blocks of 64, quads of states
    uint32_t tiles, segs, seg_tiles;  // tiles of 16 steps; segments and theirs
    uint32_t walks;                   // backward: workgroups that the sequences are dealt to
    uint32_t stretches;               // and the stretches of kStretch tiles that a workgroup has at most
};

// softplus(v) = max(v, 0) + log1p(e), e = exp(-|v|): a polynomial of degree 9 in e for log1p(e) / e on [0, 1], the least
// squares of its relative error, which is 1.6e-8 at most (1.3e-7 as f32 evaluates it): small steps keep their digits.
__device__ __forceinline__ float softplus(float v, float& e) {
    e = __builtin_amdgcn_exp2f(__builtin_fabsf(v) * -kLog2e);
    float p = -0.0031640392262488604f;
    p = __builtin_fmaf(p, e, 0.019487930461764336f);
    p = __builtin_fmaf(p, e, -0.05627012997865677f);
    p = __builtin_fmaf(p, e, 0.10533029586076736f);
    p = __builtin_fmaf(p, e, -0.15263333916664124f);
    p = __builtin_fmaf(p, e, 0.1966104507446289f);
    p = __builtin_fmaf(p, e, -0.2495117485523224f);
    p = __builtin_fmaf(p, e, 0.33329665660858154f);
    p = __builtin_fmaf(p, e, -0.49999889731407166f);
    p = __builtin_fmaf(p, e, 1.0f);
    return __builtin_fmaf(p, e, v > 0.0f ? v : 0.0f);
}
// a state's rate for exp2, finite: times a step of 0 it is 0
__device__ __forceinline__ float rate_of(float a) {
    const float k = a * kLog2e;
    return k < -3.4e38f ? -3.4e38f : k > 3.4e38f ? 3.4e38f : k;
}

// NS states of a lane.
template <int NS>
struct States {
    float v[NS];
};

// h[k] += B_k u, then the sum of C_k h[k], B_k and C_k from lane FROM + k of the own row of 16 lanes. In assembly: the
// compiler spends a move on each such operand. The instructions in front may have written b or c (a DPP operand's two wait
// states). What an instruction writes before the last input is read is an early clobber, here and below: an input of the
// same value would otherwise be given the same register.
template <int FROM>
__device__ __forceinline__ float step_states(States<4>& h, float b, float u, float c) {
    float p = 0.0f;
#if defined(__HIP_DEVICE_COMPILE__)
    asm("s_nop 1\n"
        "v_fmac_f32_dpp %1, %5, %6 row_newbcast:%8 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %2, %5, %6 row_newbcast:%9 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %3, %5, %6 row_newbcast:%10 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %4, %5, %6 row_newbcast:%11 row_mask:0xf bank_mask:0xf\n"
        "v_mul_f32_dpp %0, %7, %1 row_newbcast:%8 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %0, %7, %2 row_newbcast:%9 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %0, %7, %3 row_newbcast:%10 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %0, %7, %4 row_newbcast:%11 row_mask:0xf bank_mask:0xf"
        : "=&v"(p), "+&v"(h.v[0]), "+&v"(h.v[1]), "+&v"(h.v[2]), "+&v"(h.v[3])
        : "v"(b), "v"(u), "v"(c), "n"(FROM), "n"(FROM + 1), "n"(FROM + 2), "n"(FROM + 3));
#endif
    return p;
}
template <int FROM>
__device__ __forceinline__ float step_states(States<2>& h, float b, float u, float c) {
    float p = 0.0f;
#if defined(__HIP_DEVICE_COMPILE__)
    asm("s_nop 1\n"
        "v_fmac_f32_dpp %1, %3, %4 row_newbcast:%6 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %2, %3, %4 row_newbcast:%7 row_mask:0xf bank_mask:0xf\n"
        "v_mul_f32_dpp %0, %5, %1 row_newbcast:%6 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %0, %5, %2 row_newbcast:%7 row_mask:0xf bank_mask:0xf"
        : "=&v"(p), "+&v"(h.v[0]), "+&v"(h.v[1])
        : "v"(b), "v"(u), "v"(c), "n"(FROM), "n"(FROM + 1));
#endif
    return p;
}
// h[k] += B_k u
template <int FROM>
__device__ __forceinline__ void add_outer(f4& h, float b, float u) {
#if defined(__HIP_DEVICE_COMPILE__)
    float h0 = h[0], h1 = h[1], h2 = h[2], h3 = h[3];
    asm("s_nop 1\n"
        "v_fmac_f32_dpp %0, %4, %5 row_newbcast:%6 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %1, %4, %5 row_newbcast:%7 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %2, %4, %5 row_newbcast:%8 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %3, %4, %5 row_newbcast:%9 row_mask:0xf bank_mask:0xf"
        : "+&v"(h0), "+&v"(h1), "+&v"(h2), "+&v"(h3)
        : "v"(b), "v"(u), "n"(FROM), "n"(FROM + 1), "n"(FROM + 2), "n"(FROM + 3));
    h = f4{h0, h1, h2, h3};
#endif
}
// g[k] += C_k q, then s1 = the sum of B_k g[k] and p = the sum of C_k h[k]
template <int FROM>
__device__ __forceinline__ void step_back(f4& g, f4 h, float b, float c, float q, float& p, float& s1) {
#if defined(__HIP_DEVICE_COMPILE__)
    float g0 = g[0], g1 = g[1], g2 = g[2], g3 = g[3];
    asm("s_nop 1\n"
        "v_fmac_f32_dpp %2, %11, %12 row_newbcast:%13 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %3, %11, %12 row_newbcast:%14 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %4, %11, %12 row_newbcast:%15 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %5, %11, %12 row_newbcast:%16 row_mask:0xf bank_mask:0xf\n"
        "v_mul_f32_dpp %0, %11, %6 row_newbcast:%13 row_mask:0xf bank_mask:0xf\n"
        "v_mul_f32_dpp %1, %10, %2 row_newbcast:%13 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %0, %11, %7 row_newbcast:%14 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %1, %10, %3 row_newbcast:%14 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %0, %11, %8 row_newbcast:%15 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %1, %10, %4 row_newbcast:%15 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %0, %11, %9 row_newbcast:%16 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %1, %10, %5 row_newbcast:%16 row_mask:0xf bank_mask:0xf"
        : "=&v"(p), "=&v"(s1), "+&v"(g0), "+&v"(g1), "+&v"(g2), "+&v"(g3)
        : "v"(h[0]), "v"(h[1]), "v"(h[2]), "v"(h[3]), "v"(b), "v"(c), "v"(q), "n"(FROM), "n"(FROM + 1), "n"(FROM + 2),
          "n"(FROM + 3));
    g = f4{g0, g1, g2, g3};
#endif
}
__device__ __forceinline__ void fence() { asm volatile("" ::: "memory"); }
// and nothing is scheduled across, so that registers hold the work of one group of steps at a time
__device__ __forceinline__ void group() {
    fence();
    __builtin_amdgcn_sched_barrier(0);
}
// A barrier for what lies in LDS: __syncthreads would also wait for the next tile's loads, which are under way.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
// The values are in registers from here on: what they come from has been waited for.
template <int N>
__device__ __forceinline__ void settle(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) asm volatile("" : "+v"(v[i]));
}

template <class F, int... I>
__device__ __forceinline__ void each_of(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
// f(0) .. f(N - 1) with constants for arguments
template <int N, class F>
__device__ __forceinline__ void each(F&& f) {
    each_of(f, std::make_integer_sequence<int, N>{});
}

// Where a workgroup is. Channel blocks come first in the index and segments last, so every XCD (workgroups go round-robin to
// the 8) has a share of every sequence and segment: lengths may leave the late ones empty.
struct Spot {
    uint32_t seg, walk, group, block, ch;
    bool live;
    template <class R>
    __device__ __forceinline__ Spot(const SsmArgs<R>& g, uint32_t lane) {
        uint32_t q = blockIdx.x;
        block = q % g.blocks, q /= g.blocks;
        group = q % g.groups, q /= g.groups;
        walk = q % g.walks, seg = q / g.walks;
        const uint32_t at = block * 64 + lane;
        live = at < g.width;
        ch = group * g.width + (live ? at : g.width - 1);  // a lane without a channel repeats the last one's work
    }
};

__device__ __forceinline__ void swap32(float& a, float& b) {  // {a0 a1 b0 b1}, {a2 a3 b2 b3} by rows of 16 lanes
#if defined(__HIP_DEVICE_COMPILE__)
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false, false);
    const uint32_t p = r[0], q = r[1];  // (a cast of a vector's element itself takes the first one's bits for every index)
    a = __builtin_bit_cast(float, p), b = __builtin_bit_cast(float, q);
#endif
}
__device__ __forceinline__ void swap16(float& a, float& b) {  // {a0 b0 a2 b2}, {a1 b1 a3 b3}
#if defined(__HIP_DEVICE_COMPILE__)
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false, false);
    const uint32_t p = r[0], q = r[1];
    a = __builtin_bit_cast(float, p), b = __builtin_bit_cast(float, q);
#endif
}
// A tile's B or C of NS states: lane l reads step l / NS and state l % NS, one load, and rows of lanes are then spread over
// the wave: register j has the 16 / NS steps of row j in every row.
template <class R, int NS>
struct Vectors {
    const R* p;
    int64_t ts;
    uint32_t step;
    bool has;
    __device__ __forceinline__ Vectors(const Seq<R>& m, uint32_t b, uint32_t t, uint32_t group, uint32_t n, uint32_t q,
                                       uint32_t lane)
        : ts(m.ts), step(lane / NS % kTile) {
        const uint32_t k = NS * q + lane % NS;
        has = k < n;
        p = m.at(b, t + step) + (group * n + (has ? k : 0));
    }
    // the tile that p is at, `left` steps of it there
    __device__ __forceinline__ R load(uint32_t left) const { return has && step < left ? *p : R(0); }
    __device__ __forceinline__ void move(int steps) { p += steps * ts; }
};
template <int NS>
__device__ __forceinline__ void spread(float v, float (&o)[NS]) {
    if constexpr (NS == 4) {
        o[0] = o[2] = v;
        swap32(o[0], o[2]);
        o[1] = o[0], o[3] = o[2];
        swap16(o[0], o[1]);
        swap16(o[2], o[3]);
    } else {  // lanes 32 up have the same values as those below
        o[0] = o[1] = v;
        swap16(o[0], o[1]);
    }
}

// A wave's part of a tile outside the states: 16 / W steps, wave * K + row, each on 64 / K lanes of K adjacent channels
// (one wide load a tensor).
template <class R, int W>
struct Part {
    static constexpr int K = kTile / W;
    uint32_t step, c0;  // of the tile; of the block's channels
    int valid;          // channels there
    __device__ __forceinline__ Part(uint32_t lane, uint32_t wave, uint32_t width, uint32_t block)
        : step(wave * K + lane / (64 / K)), c0(lane % (64 / K) * K) {
        const uint32_t c = block * 64 + c0;
        valid = c < width ? min(K, (int)(width - c)) : 0;
    }
    __device__ __forceinline__ R* at(const Seq<R>& s, uint32_t b, uint32_t t, uint32_t ch) const {
        return s.p ? s.at(b, t + step) + ch : nullptr;
    }
    // the channels as they lie, in dwords: taking a dword apart would wait for it
    static constexpr int kWords = K * sizeof(R) / 4;
    __device__ __forceinline__ void load(const R* p, bool there, uint32_t (&o)[kWords]) const {
        constexpr int M = kWords < 4 ? kWords : 4;
        typedef uint32_t Vec __attribute__((ext_vector_type(M)));
        typedef Vec Mem __attribute__((aligned(sizeof(R))));
        if (there && valid == K) {
#pragma unroll
            for (int i = 0; i < kWords; i += M) {
                const Vec q = *reinterpret_cast<const Mem*>(reinterpret_cast<const uint32_t*>(p) + i);
#pragma unroll
                for (int j = 0; j < M; j++) {
                    if constexpr (M == 1) o[i] = q[0];
                    else o[i + j] = q[j];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kWords; i++) o[i] = 0;
            if (!there) return;
#pragma unroll
            for (int i = 0; i < K; i++) {
                if (i >= valid) continue;
                if constexpr (sizeof(R) == 2) o[i / 2] |= (uint32_t)p[i] << (16 * (i & 1));
                else o[i] = __builtin_bit_cast(uint32_t, p[i]);
            }
        }
    }
    __device__ __forceinline__ void store(R* p, bool there, const R (&o)[K]) const {
        constexpr int M = sizeof(R) == 2 ? (K < 8 ? K : 8) : (K < 4 ? K : 4);
        if (!there) return;
        if (valid == K) {
#pragma unroll
            for (int i = 0; i < K; i += M) {
                R q[M];
#pragma unroll
                for (int j = 0; j < M; j++) q[j] = o[i + j];
                store_raw<R, M, false>(p + i, q);
            }
        } else {
#pragma unroll
            for (int i = 0; i < K; i++)
                if (i < valid) p[i] = o[i];
        }
    }
    // per-channel weights (zeros where there are none)
    __device__ __forceinline__ void weights(const float* p, uint32_t ch, float (&o)[K]) const {
#pragma unroll
        for (int i = 0; i < K; i++) o[i] = p && i < valid ? p[ch + i] : 0.0f;
    }
};
// element i of such dwords
template <class T, int N>
__device__ __forceinline__ float element(const uint32_t (&w)[N], int i) {
    if constexpr (sizeof(typename T::Raw) == 2) return widen(T{}, (uint16_t)(w[i / 2] >> (16 * (i & 1))));
    else return __builtin_bit_cast(float, w[i]);
}
// K adjacent values of an LDS row
template <int K>
__device__ __forceinline__ void read_row(const float* p, float (&o)[K]) {
    constexpr int M = K < 4 ? K : 4;
#pragma unroll
    for (int i = 0; i < K; i += M) {
        float q[M];
        load_raw<float, M, true>(p + i, q);
#pragma unroll
        for (int j = 0; j < M; j++) o[i + j] = q[j];
    }
}
template <int K>
__device__ __forceinline__ void write_row(float* p, const float (&o)[K]) {
    constexpr int M = K < 4 ? K : 4;
#pragma unroll
    for (int i = 0; i < K; i += M) {
        float q[M];
#pragma unroll
        for (int j = 0; j < M; j++) q[j] = o[i + j];
        store_raw<float, M, true>(p + i, q);
    }
}

// states from s on of a [b][d][n] tensor, zeros past the last one: one wide load or store where all are there (a lane's are n
// apart from its neighbour's, so each narrow one would touch a cache line a lane)
template <int NS>
__device__ __forceinline__ void load_states(const float* p, uint64_t at, uint32_t n, uint32_t s, float (&h)[NS]) {
#pragma unroll
    for (int k = 0; k < NS; k++) h[k] = 0.0f;
    if (!p) return;
    if (s + NS <= n) {
        load_raw<float, NS, false>(p + at * n + s, h);
    } else {
#pragma unroll
        for (int k = 0; k < NS; k++)
            if (s + k < n) h[k] = p[at * n + s + k];
    }
}
template <int NS>
__device__ __forceinline__ void store_states(float* p, uint64_t at, uint32_t n, uint32_t s, const float (&h)[NS]) {
    if (s + NS <= n) {
        store_raw<float, NS, false>(p + at * n + s, h);
    } else {
#pragma unroll
        for (int k = 0; k < NS; k++)
            if (s + k < n) p[at * n + s + k] = h[k];
    }
}
// the same of quad q
__device__ __forceinline__ f4 load_states(const float* p, uint64_t at, uint32_t n, uint32_t q) {
    float h[4];
    load_states<4>(p, at, n, 4 * q, h);
    return f4{h[0], h[1], h[2], h[3]};
}
__device__ __forceinline__ void store_states(float* p, uint64_t at, uint32_t n, uint32_t q, f4 v) {
    const float h[4] = {v[0], v[1], v[2], v[3]};
    store_states<4>(p, at, n, 4 * q, h);
}
__device__ __forceinline__ f4 rates_of(const float* a, uint32_t ch, uint32_t n, uint32_t q) {
    f4 h = load_states(a, ch, n, q);
#pragma unroll
    for (int k = 0; k < 4; k++) h[k] = rate_of(h[k]);
    return h;
}
__device__ __forceinline__ f4 decay(float step, f4 rate) {
    f4 a;
#pragma unroll
    for (int k = 0; k < 4; k++) a[k] = __builtin_amdgcn_exp2f(step * rate[k]);
    return a;
}
// The ends of segments from zeros: W waves, NQ quads of states each. What bounds it (MI355X): the vector units, as below, 109
// cycles a step of four states; 32768 steps of 2048 channels of 16 states, bf16, in 64 segments, 205 us, 99% of them issue.
template <class T, int W, int NQ>
__global__ __launch_bounds__(64 * W, 2) void ssm_fold(SsmArgs<typename T::Raw> g) {
    using R = typename T::Raw;
    using P = Part<R, W>;
    constexpr int K = P::K;
    __shared__ __align__(16) float steps[2][kTile][128];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Spot at(g, lane);
    const P part(lane, wave, g.width, at.block);
    const uint32_t b = at.walk, ch = at.ch, base = at.group * g.width + at.block * 64 + part.c0;
    const uint64_t flat = (uint64_t)b * g.d + ch, slots = (uint64_t)g.b * g.quads * g.d;
    const uint32_t n = g.lengths ? (uint32_t)min(max(g.lengths[b], 0), (int32_t)g.t) : g.t;
    const uint32_t first = at.seg * g.seg_tiles, last = min(first + g.seg_tiles, g.tiles);
    const uint32_t busy = min(last, (n + kTile - 1) / kTile);
    float bias[K];
    part.weights(g.bias, base, bias);
    f4 rate[NQ], h[NQ];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        const uint32_t q = wave + W * i;
        rate[i] = rates_of(g.a, ch, g.n, q);
        h[i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        // the second launch reads the first state here: the last one may lie over h0
        if (at.seg == 0 && q < g.quads && at.live) g.ends[((uint64_t)b * g.quads + q) * g.d + ch] = load_states(g.h0, flat, g.n, q);
    }
    const uint32_t from = first * kTile;
    const R *px = part.at(g.x, b, from, base), *pt = part.at(g.dt, b, from, base);
    Vectors<R, 4> vec[2] = {{g.bm, b, from, at.group, g.n, wave, lane}, {g.bm, b, from, at.group, g.n, wave + W * (NQ - 1), lane}};
    uint32_t x[P::kWords], dt[P::kWords];
    R bm[NQ];
    auto load = [&](uint32_t left) __attribute__((always_inline)) {
        part.load(px, part.step < left, x), part.load(pt, part.step < left, dt);
        px += kTile * g.x.ts, pt += kTile * g.dt.ts;
#pragma unroll
        for (int i = 0; i < NQ; i++) bm[i] = vec[i].load(left), vec[i].move(kTile);
    };
    uint32_t left = first < busy ? n - from : 0;  // steps of the sequence from the tile on
    if (left) load(left);
    for (uint32_t tile = first; tile < busy; tile++, left -= kTile) {
        float* rows = steps[(tile - first) & 1][0];  // the other one may still be read
        float o[2 * K], bv[NQ][4];
#pragma unroll
        for (int j = 0; j < K; j++) {
            float e;
            const float d = softplus(element<T>(dt, j) + bias[j], e);
            o[2 * j] = part.step < left && j < part.valid ? d : 0.0f, o[2 * j + 1] = o[2 * j] * element<T>(x, j);
        }
        write_row<2 * K>(rows + part.step * 128 + part.c0 * 2, o);
#pragma unroll
        for (int i = 0; i < NQ; i++) spread<4>(widen(T{}, bm[i]), bv[i]), settle(bv[i]);  // before the next tile's loads start
        if (tile + 1 < busy) load(left - kTile);
        lds_barrier();
        float2 st[2][4];  // four steps' LDS reads are on their way while four steps run
        auto read = [&](int m) __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < 4; r++) st[m & 1][r] = *reinterpret_cast<const float2*>(rows + (4 * m + r) * 128 + lane * 2);
        };
        read(0);
        each<4>([&](auto mc) {
            constexpr int m = mc;
            if constexpr (m < 3) read(m + 1);
            fence();
            each<4>([&](auto rc) {
                constexpr int r = rc;
                sum += st[m & 1][r].x;
                each<NQ>([&](auto i) {
                    h[i] *= decay(st[m & 1][r].x, rate[i]);
                    add_outer<r * 4>(h[i], bv[i][m], st[m & 1][r].y);
                });
            });
        });
    }
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        const uint32_t q = wave + W * i;
        if (q < g.quads && at.live) g.ends[(at.seg + 1) * slots + ((uint64_t)b * g.quads + q) * g.d + ch] = h[i];
    }
    if (wave == 0 && at.live) g.lasts[(uint64_t)at.seg * g.b * g.d + flat] = sum;
}

// h through the folds of `count` segments, `step` slots apart from p on: eight segments' loads are under way together. A
// segment that is not there is one that changes nothing. A segment's decay goes in as its square root, twice: from states to
// states that f32 holds it may itself be out of range. The root is finite, so that a state of 0 stays 0 (any other normal one
// that 2^255 multiplies is past the range with it).
template <int NS>
__device__ __forceinline__ void through(const float* p, int64_t step, const float* total, int64_t tstep, uint32_t count,
                                        const float (&rate)[NS], float (&h)[NS]) {
    for (uint32_t s = 0; s < count; s += 8) {
        float end[8][NS], sum[8];
#pragma unroll
        for (int u = 0; u < 8; u++) {
            sum[u] = 0.0f;
#pragma unroll
            for (int k = 0; k < NS; k++) end[u][k] = 0.0f;
            if (s + u < count) {
                sum[u] = total[(s + u) * tstep];
                load_raw<float, NS, false>(p + (s + u) * step, end[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < 8; u++)
#pragma unroll
            for (int k = 0; k < NS; k++) {
                const float half = rate[k] * sum[u] * 0.5f, root = __builtin_amdgcn_exp2f(half > 127.5f ? 127.5f : half);
                h[k] = __builtin_fmaf(root, root * h[k], end[u][k]);
            }
    }
}

// W waves, NQ times NS states each. What bounds it (MI355X): the vector units. By the issue counters a step of four states of 64
// channels takes 154 cycles of a SIMD, with its share of the tile's preparation and end: four exponentials (8 cycles each), eight
// products and eight multiply-adds (4 each) are 96 of them. 2^30 steps of a state are 630,000 cycles on 1024 SIMDs, 290 us at the
// 2.16 GHz that the chip then runs at; HBM would take 104. 32768 steps of 2048 channels of 16 states, bf16 with a gate, in
// segments: 300 us, 97% of them issue, after the fold's 205. 4 x 4096 steps of 4096 channels: 390 us a call, 430 under the
// profiler, 64% of them issue (256 workgroups of 8 waves: two waves a SIMD, whose waits at a tile's two barriers nothing fills).
// 1620 x 24 steps of 256 channels, f16, 64 us for 135 MB (2.1 TB/s: two tiles a workgroup, whose first loads nothing covers). f32
// takes as long: 391 us for 4 x 4096 x 4096, 476 for the long sequence.
// Tried without gain: one barrier a tile with two buffers; outer products on the matrix units, which do not run beside the
// vector unit's exponentials; a workgroup order by XCD.
template <class T, int W, int NQ, int NS>
__global__ __launch_bounds__(64 * W, 2) void ssm_fwd(SsmArgs<typename T::Raw> g) {
    using R = typename T::Raw;
    using P = Part<R, W>;
    constexpr int K = P::K, SPR = 16 / NS;  // steps a register of vectors
    __shared__ __align__(16) float steps[2][kTile][128];
    __shared__ __align__(16) float parts[W][kTile][64];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Spot at(g, lane);
    const P part(lane, wave, g.width, at.block);
    const uint32_t b = at.walk, ch = at.ch, base = at.group * g.width + at.block * 64 + part.c0;
    const uint64_t flat = (uint64_t)b * g.d + ch, slots = (uint64_t)g.b * g.quads * g.d;
    const uint32_t n = g.lengths ? (uint32_t)min(max(g.lengths[b], 0), (int32_t)g.t) : g.t;
    const uint32_t first = at.seg * g.seg_tiles, last = min(first + g.seg_tiles, g.tiles);
    const uint32_t busy = min(last, (n + kTile - 1) / kTile);
    float bias[K], skip[K];
    part.weights(g.bias, base, bias), part.weights(g.skip, base, skip);
    // state k of the wave's part i: number NS * (wave + W * i) + k
    auto number = [&](int i, int k) __attribute__((always_inline)) { return NS * (wave + W * i) + k; };
    // its place in a buffer of quads [quad][d] of 4
    auto in_quads = [&](int i, int k) __attribute__((always_inline)) {
        const uint32_t s = number(i, k);
        return ((uint64_t)(s >> 2) * g.d + ch) * 4 + (s & 3);
    };
    States<NS> rate[NQ], h[NQ];
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        load_states<NS>(g.a, ch, g.n, number(i, 0), rate[i].v);
        load_states<NS>(g.segs == 1 ? g.h0 : nullptr, flat, g.n, number(i, 0), h[i].v);
#pragma unroll
        for (int k = 0; k < NS; k++) rate[i].v[k] = rate_of(rate[i].v[k]);
        if (g.segs > 1 && number(i, 0) < g.n) {
            const float* p = reinterpret_cast<const float*>(g.ends + (uint64_t)b * g.quads * g.d) + in_quads(i, 0);
            load_raw<float, NS, false>(p, h[i].v);
            through<NS>(p + slots * 4, slots * 4, g.lasts + flat, (int64_t)g.b * g.d, at.seg, rate[i].v, h[i].v);
        }
    }
    const uint32_t from = first * kTile;
    const R *px = part.at(g.x, b, from, base), *pt = part.at(g.dt, b, from, base), *pz = part.at(g.z, b, from, base);
    R* py = part.at(g.y, b, from, base);
    Vectors<R, NS> vb[2] = {{g.bm, b, from, at.group, g.n, wave, lane}, {g.bm, b, from, at.group, g.n, wave + W * (NQ - 1), lane}};
    Vectors<R, NS> vc[2] = {{g.cm, b, from, at.group, g.n, wave, lane}, {g.cm, b, from, at.group, g.n, wave + W * (NQ - 1), lane}};
    // the inputs of the two tiles to come (a tile takes about as long as its loads from memory); x and z of the tile that runs
    uint32_t x[2][P::kWords], dt[2][P::kWords], z[2][P::kWords], xs[P::kWords], zs[P::kWords];
    R bm[2][NQ], cm[2][NQ];
    auto load = [&](uint32_t left, auto slot) __attribute__((always_inline)) {
        const bool there = part.step < left;
        part.load(px, there, x[slot]), part.load(pt, there, dt[slot]);
        if (g.z.p) part.load(pz, there, z[slot]), pz += kTile * g.z.ts;
        px += kTile * g.x.ts, pt += kTile * g.dt.ts;
#pragma unroll
        for (int i = 0; i < NQ; i++) {
            bm[slot][i] = vb[i].load(left), cm[slot][i] = vc[i].load(left);
            vb[i].move(kTile), vc[i].move(kTile);
        }
    };
    auto prepare = [&](uint32_t left, auto slot) __attribute__((always_inline)) {
        float o[2 * K];
#pragma unroll
        for (int j = 0; j < K; j++) {
            float e;
            const float d = softplus(element<T>(dt[slot], j) + bias[j], e);
            o[2 * j] = part.step < left && j < part.valid ? d : 0.0f, o[2 * j + 1] = o[2 * j] * element<T>(x[slot], j);
        }
        write_row<2 * K>(steps[slot][part.step] + part.c0 * 2, o);
    };
    float bv[NQ][NS], cv[NQ][NS];
    auto vectors = [&](auto slot) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NQ; i++) {  // settled before their registers are loaded again
            spread<NS>(widen(T{}, bm[slot][i]), bv[i]), spread<NS>(widen(T{}, cm[slot][i]), cv[i]);
            settle(bv[i]), settle(cv[i]);
        }
    };
    auto keep = [&](auto slot) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < P::kWords; j++) {
            xs[j] = x[slot][j], zs[j] = z[slot][j];
            asm volatile("" : "+v"(xs[j]), "+v"(zs[j]));
        }
    };
    auto states = [&](uint32_t tile) __attribute__((always_inline)) {
        if (!g.states || !at.live) return;
        float* to = reinterpret_cast<float*>(g.states + ((uint64_t)b * g.tiles + tile) * g.quads * g.d);
#pragma unroll
        for (int i = 0; i < NQ; i++) {
            if (number(i, 0) >= 4 * g.quads) continue;
            if constexpr (NS == 4) *reinterpret_cast<f4*>(to + in_quads(i, 0)) = f4{h[i].v[0], h[i].v[1], h[i].v[2], h[i].v[3]};
            else *reinterpret_cast<float2*>(to + in_quads(i, 0)) = float2{h[i].v[0], h[i].v[1]};
        }
    };
    auto run = [&](int buf) __attribute__((always_inline)) {
        float2 st[2][4];  // four steps' LDS reads are on their way while four steps run
        auto read = [&](int m) __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < 4; r++) st[m & 1][r] = *reinterpret_cast<const float2*>(steps[buf][4 * m + r] + lane * 2);
        };
        read(0);
        each<4>([&](auto mc) {
            constexpr int m = mc;
            if constexpr (m < 3) read(m + 1);
            fence();
            each<4>([&](auto rc) {
                constexpr int r = rc, s = 4 * m + r;
                float p = 0.0f;
                each<NQ>([&](auto ic) {
                    constexpr int i = ic;
                    each<NS>([&](auto kc) { h[i].v[kc] *= __builtin_amdgcn_exp2f(st[m & 1][r].x * rate[i].v[kc]); });
                    const float q = step_states<s % SPR * NS>(h[i], bv[i][s / SPR], st[m & 1][r].y, cv[i][s / SPR]);
                    p = i ? p + q : q;
                });
                parts[wave][s][lane] = p;
            });
        });
    };
    // left: of the tile's steps those inside the length; there: those inside the tensor
    auto finish = [&](uint32_t left, uint32_t there) __attribute__((always_inline)) {
        float p[K];
        R out[K];
#pragma unroll
        for (int j = 0; j < K; j++) p[j] = skip[j] * element<T>(xs, j);
#pragma unroll
        for (int w = 0; w < W; w++) {
            float q[K];
            read_row<K>(parts[w][part.step] + part.c0, q);
#pragma unroll
            for (int j = 0; j < K; j++) p[j] += q[j];
        }
#pragma unroll
        for (int j = 0; j < K; j++) {
            if (g.z.p) {
                const float v = element<T>(zs, j);
                p[j] *= v * sigmoid1(v);
            }
            out[j] = part.step < left ? narrow(T{}, p[j]) : R(0);
        }
        part.store(py, part.step < there, out);
        py += kTile * g.y.ts;
    };
    using Zero = std::integral_constant<int, 0>;
    using One = std::integral_constant<int, 1>;
    uint32_t left = first < busy ? n - from : 0;  // steps of the sequence from the tile on
    if (left) {
        load(left, Zero{});
        if (left > kTile) load(left - kTile, One{});
    }
    auto body = [&](auto slot, uint32_t tile) __attribute__((always_inline)) {
        prepare(left, slot);
        keep(slot);
        vectors(slot);
        if (left > 2 * kTile) load(left - 2 * kTile, slot);
        states(tile);
        lds_barrier();
        run(slot);
        lds_barrier();
        finish(left, g.t - tile * kTile);
        left -= kTile;
    };
    for (uint32_t tile = first; tile < busy; tile += 2) {
        body(Zero{}, tile);
        if (tile + 1 < busy) body(One{}, tile + 1);
    }
    for (uint32_t t = max(busy, first) * kTile; t < min(last * kTile, g.t); t += kTile) {
        R out[K];
#pragma unroll
        for (int j = 0; j < K; j++) out[j] = R(0);
        part.store(py, t + part.step < g.t, out);
        py += kTile * g.y.ts;
    }
    if (g.ht && at.live && last == g.tiles) {
#pragma unroll
        for (int i = 0; i < NQ; i++) store_states<NS>(g.ht, flat, g.n, number(i, 0), h[i].v);
    }
}

// Few steps: a thread has one quad of one channel's states, LP threads side by side a channel, so a wave reads and writes
// the states as they lie, 16 bytes a lane; the steps follow one another. WHOLE: n is a multiple of 4.
// What bounds it (MI355X): HBM, which the states are read from and written to. One step of 64 x 4096 channels of 16
// states, bf16: 9.9 us for 36 MB (11 under the profiler); each step more is 2 to 4 us, of its narrow loads.
template <class T, int LP, bool WHOLE>
__global__ __launch_bounds__(256) void ssm_step(SsmArgs<typename T::Raw> g) {
    using R = typename T::Raw;
    const uint64_t k = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const bool live = k < (uint64_t)g.d * LP;
    const uint32_t q = k % LP, ch = live ? (uint32_t)(k / LP) : 0, group = g.groups > 1 ? ch / g.width : 0;
    const uint32_t here = live && 4 * q < g.n ? min(4u, g.n - 4 * q) : 0, col = group * g.n + 4 * q;
    auto states = [&](const float* p, uint64_t at) __attribute__((always_inline)) {
        float h[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (WHOLE && here) load_raw<float, 4, false>(p + at * g.n + 4 * q, h);
#pragma unroll
        for (int i = 0; i < 4 && !WHOLE; i++)
            if (i < (int)here) h[i] = p[at * g.n + 4 * q + i];
        return States<4>{{h[0], h[1], h[2], h[3]}};
    };
    auto vector = [&](const R* p, R (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = R(0);
        if (WHOLE && here) load_raw<R, 4, false>(p + col, v);
#pragma unroll
        for (int i = 0; i < 4 && !WHOLE; i++)
            if (i < (int)here) v[i] = p[col + i];
    };
    States<4> rate = states(g.a, ch);
#pragma unroll
    for (int i = 0; i < 4; i++) rate.v[i] = rate_of(rate.v[i]);
    const float bias = g.bias ? g.bias[ch] : 0.0f, skip = g.skip ? g.skip[ch] : 0.0f;
    for (uint32_t b = blockIdx.y; b < g.b; b += gridDim.y) {
        const uint32_t n = g.lengths ? (uint32_t)min(max(g.lengths[b], 0), (int32_t)g.t) : g.t;
        const uint64_t flat = (uint64_t)b * g.d + ch;
        States<4> h{{0.0f, 0.0f, 0.0f, 0.0f}};
        if (g.h0) h = states(g.h0, flat);
        for (uint32_t t = 0; t < g.t; t++) {
            if (g.states && here && t % kTile == 0)
                g.states[(((uint64_t)b * g.tiles + t / kTile) * g.quads + q) * g.d + ch] = f4{h.v[0], h.v[1], h.v[2], h.v[3]};
            float p = 0.0f, x = 0.0f, gate = 1.0f;
            if (t < n) {
                float e;
                R bv[4], cv[4];
                vector(g.bm.at(b, t), bv), vector(g.cm.at(b, t), cv);
                x = widen(T{}, g.x.at(b, t)[ch]);
                if (g.z.p) {
                    const float z = widen(T{}, g.z.at(b, t)[ch]);
                    gate = z * sigmoid1(z);
                }
                const float step = softplus(widen(T{}, g.dt.at(b, t)[ch]) + bias, e), u = step * x;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    h.v[i] = __builtin_fmaf(widen(T{}, bv[i]), u, __builtin_amdgcn_exp2f(step * rate.v[i]) * h.v[i]);
                    p = __builtin_fmaf(widen(T{}, cv[i]), h.v[i], p);
                }
            }
#pragma unroll
            for (int m = 1; m < LP; m *= 2) p += __shfl_xor(p, m);
            if (live && q == 0) {
                p = __builtin_fmaf(skip, x, p) * gate;
                g.y.at(b, t)[ch] = t < n ? narrow(T{}, p) : R(0);
            }
        }
        if (here && g.ht) {
            if (WHOLE) store_raw<float, 4, false>(g.ht + flat * g.n + 4 * q, h.v);
#pragma unroll
            for (int i = 0; i < 4 && !WHOLE; i++)
                if (i < (int)here) g.ht[flat * g.n + 4 * q + i] = h.v[i];
        }
    }
}

// The sums over a wave's 64 lanes of 16 values: each lane's values lie in LDS, 68 floats a value, four lanes take a value's 64
// floats in 16-byte reads (whose 16 lanes at once fall on all 64 banks) and add their sums. A halving exchange in
// registers takes 87 cycles of the vector unit for 8 values, this 30.
constexpr int kPitch = 68;
// lane + 1, lane + 2 of a quad of lanes
__device__ __forceinline__ float add_quad(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
    int i = __builtin_bit_cast(int, v);
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, 0xB1, 0xF, 0xF, true));
    i = __builtin_bit_cast(int, v);
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, 0x4E, 0xF, 0xF, true));
#endif
    return v;
}

// FOLD: the gradients that reach the states before a segment, from zeros behind it.
// What bounds it (MI355X): waits beside the vector units. A step of a state and 64 channels takes 96 cycles of a SIMD's issue with
// 64 states a channel and 119 with 16 and lengths; that is 66% and 60% of the kernel's time, 75% while a CU has work. The rest
// are waits at barriers and for LDS, at two waves a SIMD, which LDS and the 64 registers of a tile's states set. 6 x 2051 steps at
// most of 1532 channels of 16 states, bf16: 256 us, after its fold's 61; 4 x 512 of 1024 channels of 64 states, f32: 128 and 31.
// With all its columns side by side, 4 x 4096 of 4096 channels of 16 states: 1230 us a call in bf16 and in f32.
template <class T, int W, int NQ, bool FOLD>
__global__ __launch_bounds__(64 * W, 2) void ssm_bwd(SsmArgs<typename T::Raw> g) {
    using R = typename T::Raw;
    using P = Part<R, W>;
    constexpr int K = P::K;
    __shared__ __align__(16) float steps[kTile][128];                  // D, D x
    __shared__ __align__(16) float ups[kTile][64];                     // q
    __shared__ __align__(16) float parts[FOLD ? 1 : 3][FOLD ? 1 : W][kTile][64];  // sum C h, s1, s2 of a wave's states
    __shared__ float vectors[FOLD ? 1 : kTile][2][W * NQ * 4];         // dB, dC over the workgroup's channels
    __shared__ __align__(16) float lanes[FOLD ? 1 : W][16][kPitch];    // dB, dC of two steps, lane by lane
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Spot at(g, lane);
    const P part(lane, wave, g.width, at.block);
    const uint32_t ch = at.ch, base = at.group * g.width + at.block * 64 + part.c0;
    const uint32_t first = at.seg * g.seg_tiles, last = min(first + g.seg_tiles, g.tiles);
    const uint64_t slots = (uint64_t)g.b * g.quads * g.d;
    float bias[K], skip[K], dskip[K], dbias[K];
    part.weights(g.bias, base, bias), part.weights(g.skip, base, skip);
#pragma unroll
    for (int j = 0; j < K; j++) dskip[j] = dbias[j] = 0.0f;
    f4 rate[NQ], da[NQ];
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        rate[i] = rates_of(g.a, ch, g.n, wave + W * i);
        da[i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // The sums of the weights' gradients so far become a row of partial sums, and start again.
    const uint64_t part_row = (uint64_t)g.d * (g.n + 2);
    float* to = g.part + ((uint64_t)at.seg * g.walks + at.walk) * g.stretches * part_row;
    uint32_t stretch = 0, added = 0;  // rows written; tiles in the sums
    auto close_stretch = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NQ; i++) {
            if (at.live) store_states(to, ch, g.n, wave + W * i, da[i]);
            da[i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        lds_barrier();
        write_row<K>(parts[0][0][part.step] + part.c0, dskip), write_row<K>(parts[FOLD ? 0 : 1][0][part.step] + part.c0, dbias);
#pragma unroll
        for (int j = 0; j < K; j++) dskip[j] = dbias[j] = 0.0f;
        lds_barrier();
        if (wave == 0 && at.live) {  // read before the next tile's parts are written, a barrier further on
            float s = 0.0f, u = 0.0f;
#pragma unroll
            for (int r = 0; r < kTile; r++) s += parts[0][0][r][lane], u += parts[FOLD ? 0 : 1][0][r][lane];
            to[(uint64_t)g.d * g.n + ch] = s, to[(uint64_t)g.d * (g.n + 1) + ch] = u;
        }
        to += part_row, stretch++, added = 0;
    };
    for (uint32_t b = at.walk; b < g.b; b += g.walks) {
        const uint64_t flat = (uint64_t)b * g.d + ch;
        const uint32_t n = g.lengths ? (uint32_t)min(max(g.lengths[b], 0), (int32_t)g.t) : g.t;
        const uint32_t busy = min(last, (n + kTile - 1) / kTile);
        f4 c[NQ];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NQ; i++) {
            const uint32_t q = wave + W * i;
            const uint64_t slot = ((uint64_t)b * g.quads + q) * g.d + ch;
            c[i] = load_states(FOLD || !at.live ? nullptr : g.dht, flat, g.n, q);
            if (!FOLD && g.segs > 1 && q < g.quads && at.live) {
                float r[4] = {rate[i][0], rate[i][1], rate[i][2], rate[i][3]}, h[4] = {c[i][0], c[i][1], c[i][2], c[i][3]};
                const uint32_t behind = g.segs - 1;  // from the last segment to the one behind this
                through<4>(reinterpret_cast<const float*>(g.ends + behind * slots + slot), -(int64_t)slots * 4,
                           g.lasts + (uint64_t)behind * g.b * g.d + flat, -(int64_t)g.b * g.d, behind - at.seg, r, h);
                c[i] = f4{h[0], h[1], h[2], h[3]};
            }
        }
        const uint32_t from = busy > first ? (busy - 1) * kTile : 0;  // tiles go from the last to the first
        const R *px = part.at(g.x, b, from, base), *pt = part.at(g.dt, b, from, base), *pz = part.at(g.z, b, from, base);
        const R* py = part.at(g.dy, b, from, base);
        R *pdx = part.at(g.dx, b, from, base), *pdt = part.at(g.ddt, b, from, base), *pdz = part.at(g.dz, b, from, base);
        Vectors<R, 4> vb[2] = {{g.bm, b, from, at.group, g.n, wave, lane}, {g.bm, b, from, at.group, g.n, wave + W * (NQ - 1), lane}};
        Vectors<R, 4> vc[2] = {{g.cm, b, from, at.group, g.n, wave, lane}, {g.cm, b, from, at.group, g.n, wave + W * (NQ - 1), lane}};
        uint32_t x[P::kWords], dt[P::kWords], z[P::kWords], dy[P::kWords];
        R bm[NQ], cm[NQ];
        f4 start[NQ];
        auto load = [&](uint32_t tile) __attribute__((always_inline)) {
            const uint32_t left = n - tile * kTile;
            const bool there = part.step < left;
            if (!FOLD) part.load(px, there, x), px -= kTile * g.x.ts;
            part.load(pt, there, dt), part.load(py, there, dy);
            if (g.z.p) part.load(pz, there, z), pz -= kTile * g.z.ts;
            pt -= kTile * g.dt.ts, py -= kTile * g.dy.ts;
#pragma unroll
            for (int i = 0; i < NQ; i++) {
                const uint32_t q = wave + W * i;
                cm[i] = vc[i].load(left), vc[i].move(-kTile);
                if constexpr (!FOLD) {
                    bm[i] = vb[i].load(left), vb[i].move(-kTile);
                    start[i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
                    if (q < g.quads && at.live) start[i] = g.states[(((uint64_t)b * g.tiles + tile) * g.quads + q) * g.d + ch];
                }
            }
        };
        if (first < busy) load(busy - 1);
        for (uint32_t end = busy; end > first; end--) {
            const uint32_t tile = end - 1, left = n - tile * kTile;
            const bool on = part.step < left;
            float xs[K], slope[K], zg[K], bv[NQ][4], cv[NQ][4];  // the step's slope; dy silu'(z)
            {
                float o[2 * K], q[K];
#pragma unroll
                for (int j = 0; j < K; j++) {
                    const float v = element<T>(dt, j) + bias[j], up = element<T>(dy, j);
                    float e, gate = 1.0f, dgate = 0.0f;
                    const float d = softplus(v, e);
                    if (g.z.p) silu_grad(element<T>(z, j), gate, dgate);
                    o[2 * j] = on && j < part.valid ? d : 0.0f, o[2 * j + 1] = 0.0f;
                    q[j] = on ? up * gate : 0.0f;
                    if constexpr (!FOLD) {
                        const float r = __builtin_amdgcn_rcpf(1.0f + e);
                        xs[j] = element<T>(x, j), slope[j] = v >= 0.0f ? r : e * r, zg[j] = up * dgate;
                        o[2 * j + 1] = o[2 * j] * xs[j];
                    }
                }
                write_row<2 * K>(steps[part.step] + part.c0 * 2, o);
                write_row<K>(ups[part.step] + part.c0, q);
            }
            f4 h0[NQ];
#pragma unroll
            for (int i = 0; i < NQ; i++) {
                spread<4>(widen(T{}, cm[i]), cv[i]), settle(cv[i]);
                if constexpr (!FOLD) spread<4>(widen(T{}, bm[i]), bv[i]), settle(bv[i]), h0[i] = start[i];
            }
            lds_barrier();
            if (tile > first) load(tile - 1);
            auto step_of = [&](int s) __attribute__((always_inline)) { return *reinterpret_cast<const float2*>(steps[s] + lane * 2); };
            if constexpr (FOLD) {
                each<4>([&](auto mc) {
                    constexpr int m = 3 - mc;
                    float2 st[4];
                    float q[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) st[r] = step_of(4 * m + r), q[r] = ups[4 * m + r][lane];
                    group();
                    each<4>([&](auto rc) {
                        constexpr int r = 3 - rc;
                        sum += st[r].x;
                        each<NQ>([&](auto i) {
                            add_outer<r * 4>(c[i], cv[i][m], q[r]);
                            c[i] *= decay(st[r].x, rate[i]);
                        });
                    });
                });
            } else {
                each<NQ>([&](auto ic) {
                    constexpr int i = ic;
                    // The states of the tile; the decays are computed again on the way back: kept, their 64 registers would not
                    // fit beside them, and a register that lies in memory meanwhile makes its load wait for all that is
                    // under way.
                    f4 h[kTile];
                    each<4>([&](auto mc) {  // four steps' LDS reads at once, no more: registers
                        constexpr int m = mc;
                        float2 st[4];
#pragma unroll
                        for (int r = 0; r < 4; r++) st[r] = step_of(4 * m + r);
                        group();
                        each<4>([&](auto rc) {
                            constexpr int s = 4 * m + rc;
                            h[s] = decay(st[rc].x, rate[i]) * (s ? h[s ? s - 1 : 0] : h0[i]);
                            add_outer<rc * 4>(h[s], bv[i][m], st[rc].y);
                        });
                    });
                    float sums[16];  // a lane's share of the sums of the two steps before
                    // the sums of steps s and s + 1, whose products are in LDS: value 8 (step) + 4 (dC) + state, a quad each
                    auto close = [&](int s) __attribute__((always_inline)) {
                        float v = sums[0];
#pragma unroll
                        for (int k = 1; k < 16; k++) v += sums[k];
                        v = add_quad(v);
                        const uint32_t at = lane >> 2;
                        if ((lane & 3) == 0) vectors[s + (at >> 3)][at >> 2 & 1][(wave + W * i) * 4 + (at & 3)] = v;
                    };
                    each<4>([&](auto mc) {
                        constexpr int m = 3 - mc;
                        float2 st[4];
                        float q[4];
#pragma unroll
                        for (int r = 0; r < 4; r++) st[r] = step_of(4 * m + r), q[r] = ups[4 * m + r][lane];
                        group();
                        each<4>([&](auto rc) {
                            constexpr int r = 3 - rc, s = 4 * m + r;
                            float p, s1, s2 = 0.0f;
                            step_back<r * 4>(c[i], h[s], bv[i][m], cv[i][m], q[r], p, s1);
                            float* to = lanes[wave][(s & 1) * 8] + lane;
#pragma unroll
                            for (int k = 0; k < 4; k++) to[k * kPitch] = c[i][k] * st[r].y, to[(4 + k) * kPitch] = h[s][k] * q[r];
                            c[i] *= decay(st[r].x, rate[i]);
                            const f4 past = c[i] * (s ? h[s ? s - 1 : 0] : h0[i]);
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                da[i][k] = __builtin_fmaf(past[k], st[r].x, da[i][k]);
                                s2 = __builtin_fmaf(past[k], rate[i][k], s2);
                                // added here: moved behind the tile's steps, as the compiler does, the sums would hold the 64
                                // products of a quad in registers until then
                                asm volatile("" : "+v"(da[i][k]));
                            }
                            if (i > 0) {
                                p += parts[0][wave][s][lane], s1 += parts[1][wave][s][lane];
                                s2 += parts[2][wave][s][lane];
                            }
                            parts[0][wave][s][lane] = p, parts[1][wave][s][lane] = s1, parts[2][wave][s][lane] = s2;
                            if constexpr ((s & 1) == 0) {
                                // a wave's LDS accesses stay in order: the reads see the writes before them, and the next
                                // steps' writes come after
                                if constexpr (s < kTile - 2) close(s + 2);
                                fence();
                                read_row<16>(lanes[wave][lane >> 2] + (lane & 3) * 16, sums);
                                fence();
                            }
                            __builtin_amdgcn_sched_barrier(0);
                        });
                    });
                    close(0);
                });
            }
            lds_barrier();
            if constexpr (!FOLD) {
                const uint32_t there = g.t - tile * kTile;
                float p[K], s1[K], s2[K], q[K], st[2 * K];
#pragma unroll
                for (int j = 0; j < K; j++) p[j] = s1[j] = s2[j] = 0.0f;
#pragma unroll
                for (int w = 0; w < W; w++) {
                    float u[K];
                    auto add = [&](int of, float(&to)[K]) {
                        read_row<K>(parts[of][w][part.step] + part.c0, u);
#pragma unroll
                        for (int j = 0; j < K; j++) to[j] += u[j];
                    };
                    add(0, p), add(1, s1), add(2, s2);
                }
                read_row<2 * K>(steps[part.step] + part.c0 * 2, st), read_row<K>(ups[part.step] + part.c0, q);
                R ox[K], ot[K], oz[K];
#pragma unroll
                for (int j = 0; j < K; j++) {
                    const float dd = __builtin_fmaf(xs[j], s1[j], s2[j] * kLn2) * slope[j];
                    if (on && j < part.valid) dskip[j] = __builtin_fmaf(q[j], xs[j], dskip[j]), dbias[j] += dd;
                    ox[j] = on ? narrow(T{}, __builtin_fmaf(st[2 * j], s1[j], skip[j] * q[j])) : R(0);
                    ot[j] = on ? narrow(T{}, dd) : R(0);
                    oz[j] = on ? narrow(T{}, zg[j] * __builtin_fmaf(skip[j], xs[j], p[j])) : R(0);
                }
                part.store(pdx, part.step < there, ox), part.store(pdt, part.step < there, ot);
                if (g.z.p) part.store(pdz, part.step < there, oz), pdz -= kTile * g.dz.ts;
                pdx -= kTile * g.dx.ts, pdt -= kTile * g.ddt.ts;
                // the tile's dB and dC of this block, as they lie
                const uint32_t row = 8 * g.quads, steps_here = min((uint32_t)kTile, there);
                float* vec = g.bc + (((uint64_t)(at.group * g.blocks + at.block) * g.b + b) * g.t + tile * kTile) * row;
                for (uint32_t k = threadIdx.x; k < steps_here * row; k += 64 * W) {
                    const uint32_t s = k / row, v = k - s * row, half = v >= 4 * g.quads;
                    vec[k] = vectors[s][half][v - half * 4 * g.quads];
                }
                lds_barrier();
                if (__builtin_expect(++added == kStretch, 0)) close_stretch();
            }
        }
        if constexpr (FOLD) {
#pragma unroll
            for (int i = 0; i < NQ; i++) {
                const uint32_t q = wave + W * i;
                if (q < g.quads && at.live) g.ends[at.seg * slots + ((uint64_t)b * g.quads + q) * g.d + ch] = c[i];
            }
            if (wave == 0 && at.live) g.lasts[(uint64_t)at.seg * g.b * g.d + flat] = sum;
        } else {
            const uint32_t past = max(busy, first) * kTile;
            R none[K];
#pragma unroll
            for (int j = 0; j < K; j++) none[j] = R(0);
            R *ex = part.at(g.dx, b, past, base), *et = part.at(g.ddt, b, past, base), *ez = part.at(g.dz, b, past, base);
            for (uint32_t t = past; t < min(last * kTile, g.t); t += kTile) {
                const bool there = t + part.step < g.t;
                part.store(ex, there, none), part.store(et, there, none);
                if (g.z.p) part.store(ez, there, none), ez += kTile * g.dz.ts;
                ex += kTile * g.dx.ts, et += kTile * g.ddt.ts;
            }
            if (g.dh0 && at.live && at.seg == 0) {
#pragma unroll
                for (int i = 0; i < NQ; i++) store_states(g.dh0, flat, g.n, wave + W * i, c[i]);
            }
        }
    }
    if constexpr (!FOLD) {
        while (stretch < g.stretches) close_stretch();  // behind the last one zeros, where lengths left tiles out
    }
}

// dB and dC from the channel blocks' sums, those past a length 0
template <class R>
struct VectorArgs {
    const float* bc;
    Seq<R> dbm, dcm;
    const int32_t* lengths;
    uint32_t b, t, n, groups, blocks, quads;
};
template <class T>
__global__ __launch_bounds__(256) void ssm_vectors(VectorArgs<typename T::Raw> g) {
    const uint64_t rows = (uint64_t)g.b * g.t, all = rows * g.groups * 2 * g.n;
    for (uint64_t k = (uint64_t)blockIdx.x * 256 + threadIdx.x; k < all; k += (uint64_t)gridDim.x * 256) {
        const uint32_t v = k % g.n;
        uint64_t q = k / g.n;
        const uint32_t half = q & 1;
        q >>= 1;
        const uint64_t row = q % rows;
        const uint32_t group = (uint32_t)(q / rows), b = (uint32_t)(row / g.t), t = (uint32_t)(row - (uint64_t)b * g.t);
        const uint32_t n = g.lengths ? (uint32_t)min(max(g.lengths[b], 0), (int32_t)g.t) : g.t;
        float sum = 0.0f;
        if (t < n) {
            const float* p = g.bc + ((uint64_t)group * g.blocks * rows + row) * 8 * g.quads + half * 4 * g.quads + v;
#pragma unroll 4
            for (uint32_t i = 0; i < g.blocks; i++) sum += p[i * rows * 8 * g.quads];
        }
        (half ? g.dcm : g.dbm).at(b, t)[group * g.n + v] = narrow(T{}, sum);
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------

template <class T>
int close_vectors(const char* op, const fhc_ssm_desc* g, const float* bc, const fhc_seq* dbm, const fhc_seq* dcm,
                  uint32_t blocks, hipStream_t st) {
    using R = typename T::Raw;
    const uint64_t all = (uint64_t)g->b * g->t * g->groups * 2 * g->n;
    if (!all) return 0;
    const VectorArgs<R> v{bc, seq_of<R>(dbm), seq_of<R>(dcm), g->lengths, g->b, g->t, g->n, g->groups, blocks,
                          (g->n + 3) / 4};
    const uint64_t wgs = ceil_div(all, 256);
    hipLaunchKernelGGL((ssm_vectors<T>), dim3((uint32_t)(wgs < 1u << 16 ? wgs : 1u << 16)), dim3(256), 0, st, v);
    return launched(op);
}

// Up to here steps, then tiles. bf16, us from cold caches, by steps 1, 2, 3, 4, 6, 8: 64 x 4096 channels of 16 states 17, 21,
// 24, 28, 35, 44, by tiles 5, 8: 32, 32; 64 x 1024 of 64 states 17, 20, 24, 27, 34, 41 and 29, 29; 64 x 2048 of 8 states 8, 9,
// 11, 12 and 17, 17. A step's five loads, which the lanes of a channel repeat, are most of it.
constexpr uint32_t kFewSteps = 4;

struct Plan {
    uint32_t width, blocks, quads, tiles, segs, seg_tiles, walks, stretches;
    bool halves;  // forward: two states a lane
    uint64_t wgs;
    size_t ends_bytes, lasts_bytes, part_bytes, bc_bytes;
};
size_t up256(size_t n) { return (n + 255) / 256 * 256; }
Plan plan_of(const fhc_ssm_desc* g, bool backward, bool ragged) {
    Plan p{};
    p.width = g->d / g->groups, p.blocks = (uint32_t)ceil_div(p.width, 64), p.quads = (g->n + 3) / 4;
    p.tiles = (uint32_t)ceil_div(g->t, kTile);
    const uint64_t cols = (uint64_t)g->groups * p.blocks;
    const uint64_t one = g->b * cols;
    // Segments, of at least four tiles, where the columns alone leave CUs idle. Forward as many as keep the vector units busy
    // (the fold is half as much work again, so not more than that takes), and two states a lane instead of four where there
    // are columns for every CU but not for every SIMD. us, bf16, n 16, by workgroups:
    //   forward             one a column block, four states   two states   segments
    //    16  (1024 steps)   118                               -            4: 57, 8: 34, 16: 23, 32: 24
    //    64  (128 steps)    20                                18           2: 22, 4: 20
    //   128  (2048 steps)   228                               198          8: 141, 16: 143
    //   192  (2048)         232                               205          4: 211, 8: 202
    //   256  (4096)         453                               398          2: 530
    //   512  (2048)         339                               336
    //   768  (1024)         244                               252
    // Backward the number whose rounds of workgroups (as many at once as LDS holds) take the least, a round the tiles of a
    // segment and two for its start, with segments 1.3 times that for the fold; with lengths, which leave some empty, as many
    // as even that out. A training step in segments of
    //    64  (1024)         4: 196, 8: 156, 12: 174, 16: 163
    //   144  (512)          1: 244, 2: 249, 3: 189, 4: 208, 7: 182, 8: 191
    //   256  (1024)         1: 473, 2: 450, 3: 461, 4: 440, 8: 451
    //   512  (1024)         1: 671, 2: 772
    //   128  (1024, n 64)   1: 1094, 2: 769, 3: 959, 4: 771, 8: 790
    //   144  (lengths of 0 to 2051)   4: 597, 8: 506, 11: 484, 14: 480, 18: 475, 22: 488
    p.segs = 1;
    const uint64_t most = p.tiles / 4 < 64 ? p.tiles / 4 : 64;
    auto at_most = [&](uint64_t want) { return (uint32_t)(want < most ? want : most < 1 ? 1 : most); };
    if (!backward && one < 192 && p.tiles >= 16) p.segs = at_most(ceil_div(2048, one));
    if (backward && one < 512 && ragged) {
        p.segs = at_most(ceil_div(2048, one));
    } else if (backward && one < 512) {
        const uint64_t at_once = p.quads <= 2 ? 768 : p.quads <= 4 ? 512 : 256;
        uint64_t best = 0;
        for (uint32_t s = 1; s == 1 || s <= most; s++) {
            const uint64_t time = ceil_div(one * s, at_once) * (ceil_div(p.tiles, s) + 2) * (s > 1 ? 13 : 10);
            if (s == 1 || time < best) best = time, p.segs = s;
        }
    }
    p.halves = !backward && p.segs == 1 && one <= 512 && p.quads <= 4;
    p.seg_tiles = p.tiles ? (uint32_t)ceil_div(p.tiles, p.segs) : 1;
    p.segs = p.tiles ? (uint32_t)ceil_div(p.tiles, p.seg_tiles) : 1;
    p.walks = g->b;
    if (backward && one > 2048) {
        const uint64_t w = ceil_div(2048, cols);
        p.walks = (uint32_t)(w < g->b ? w : g->b);
    }
    p.wgs = p.walks * cols * p.segs;
    const uint64_t flat = (uint64_t)g->b * g->d;
    if (p.segs > 1) {
        p.ends_bytes = up256((size_t)(p.segs + 1) * flat * p.quads * 16);
        p.lasts_bytes = up256((size_t)p.segs * flat * 4);
    }
    if (backward) {
        const uint64_t stretches = ceil_div(ceil_div(g->b, p.walks ? p.walks : 1) * p.seg_tiles, kStretch);
        p.stretches = (uint32_t)(stretches ? stretches : 1);
        p.part_bytes = up256((size_t)p.segs * p.walks * p.stretches * g->d * (g->n + 2) * 4);
        p.bc_bytes = up256((size_t)cols * g->b * g->t * 8 * p.quads * 4);
    }
    return p;
}
size_t workspace_of(const Plan& p) { return p.ends_bytes + p.lasts_bytes + p.part_bytes + p.bc_bytes; }
// one size for a shape, with and without lengths
size_t workspace_of(const fhc_ssm_desc* g, bool backward) {
    const size_t n = workspace_of(plan_of(g, backward, false)), m = workspace_of(plan_of(g, backward, true));
    return n > m ? n : m;
}

int check_desc(const char* op, const fhc_ssm_desc* g) {
    if (!g) return fail(-1, "%s: null descriptor", op);
    FHC_TRY(check_shape(op, g->dtype, g->b, g->t, g->d));
    if (g->n < 1 || g->n > 64) return fail(-1, "%s: %u states a channel, 1 to 64 are possible", op, g->n);
    if (g->groups < 1 || g->d % g->groups) return fail(-1, "%s: %u groups of %u channels", op, g->groups, g->d);
    if ((uint64_t)g->groups * g->n >= 1ull << 31)
        return fail(-1, "%s: %u groups of %u states, at most 2^31 - 1 values a step", op, g->groups, g->n);
    FHC_TRY(check_array(op, "a", g->a, 4, g->b && g->d));
    FHC_TRY(check_array(op, "dt_bias", g->dt_bias, 4, false));
    FHC_TRY(check_array(op, "skip", g->skip, 4, false));
    return check_array(op, "lengths", g->lengths, 4, false);
}

template <class T>
SsmArgs<typename T::Raw> args_of(const fhc_ssm_desc* g, const Plan& p, const fhc_seq* x, const fhc_seq* dt,
                                 const fhc_seq* bm, const fhc_seq* cm, const fhc_seq* z, void* ws) {
    using R = typename T::Raw;
    SsmArgs<R> a{};
    a.x = seq_of<R>(x), a.dt = seq_of<R>(dt), a.bm = seq_of<R>(bm), a.cm = seq_of<R>(cm), a.z = seq_of<R>(z);
    a.a = g->a, a.bias = g->dt_bias, a.skip = g->skip, a.lengths = g->lengths;
    a.b = g->b, a.t = g->t, a.d = g->d, a.n = g->n, a.groups = g->groups;
    a.width = p.width, a.blocks = p.blocks, a.quads = p.quads, a.tiles = p.tiles, a.segs = p.segs;
    a.seg_tiles = p.seg_tiles, a.walks = p.walks, a.stretches = p.stretches;
    char* w = static_cast<char*>(ws);
    a.ends = reinterpret_cast<f4*>(w), w += p.ends_bytes;
    a.lasts = reinterpret_cast<float*>(w), w += p.lasts_bytes;
    a.part = reinterpret_cast<float*>(w), w += p.part_bytes;
    a.bc = reinterpret_cast<float*>(w);
    return a;
}

// waves of a workgroup of the tile kernels (with two states a lane up to 8, but of few workgroups)
uint32_t waves_of(const Plan& p) { return p.quads <= 2 ? 2 : p.quads <= 4 ? 4 : 8; }

enum Kernel { kFold, kForward, kFoldBack, kBackward };
template <class T, Kernel KERNEL>
int launch(const char* op, const Plan& p, const SsmArgs<typename T::Raw>& a, hipStream_t st) {
    const dim3 grid((uint32_t)p.wgs);
#define SSM(W, NQ, NS)                                                                                             \
    do {                                                                                                           \
        if constexpr (KERNEL == kFold) hipLaunchKernelGGL((ssm_fold<T, W, NQ>), grid, dim3(64 * W), 0, st, a);     \
        else if constexpr (KERNEL == kForward)                                                                     \
            hipLaunchKernelGGL((ssm_fwd<T, W, NQ, NS>), grid, dim3(64 * W), 0, st, a);                             \
        else if constexpr (KERNEL == kFoldBack)                                                                    \
            hipLaunchKernelGGL((ssm_bwd<T, W, NQ, true>), grid, dim3(64 * W), 0, st, a);                           \
        else hipLaunchKernelGGL((ssm_bwd<T, W, NQ, false>), grid, dim3(64 * W), 0, st, a);                         \
    } while (0)
    if constexpr (KERNEL == kForward) {
        if (p.halves) {
            if (p.quads == 1) SSM(2, 1, 2);
            else if (p.quads == 2) SSM(4, 1, 2);
            else SSM(8, 1, 2);
            return launched(op);
        }
    }
    if (p.quads <= 2) SSM(2, 1, 4);
    else if (p.quads <= 4) SSM(4, 1, 4);
    else if (p.quads <= 8) SSM(8, 1, 4);
    else SSM(8, 2, 4);
#undef SSM
    return launched(op);
}

template <class T>
int launch_step(const char* op, const Plan& p, const SsmArgs<typename T::Raw>& a, hipStream_t st) {
    uint32_t lp = 1;
    while (lp < p.quads) lp *= 2;
    // as many sequences side by side as one launch has workgroups for
    const uint64_t wide = ceil_div((uint64_t)a.d * lp, 256), room = ((1ull << 32) / 256 - 1) / wide;
    FHC_TRY(check_grid(op, wide, 256));
    const uint64_t rows = room < 65535 ? room : 65535;
    const dim3 grid((uint32_t)wide, a.b < rows ? a.b : (uint32_t)rows);
#define STEP(LP)                                                                                           \
    do {                                                                                                   \
        if (a.n % 4 == 0) hipLaunchKernelGGL((ssm_step<T, LP, true>), grid, dim3(256), 0, st, a);          \
        else hipLaunchKernelGGL((ssm_step<T, LP, false>), grid, dim3(256), 0, st, a);                      \
    } while (0)
    if (lp == 1) STEP(1);
    else if (lp == 2) STEP(2);
    else if (lp == 4) STEP(4);
    else if (lp == 8) STEP(8);
    else STEP(16);
#undef STEP
    return launched(op);
}

int check_inputs(const char* op, const fhc_ssm_desc* g, const Plan& p, const fhc_seq* x, const fhc_seq* dt,
                 const fhc_seq* bm, const fhc_seq* cm, const fhc_seq* z, bool few_steps) {
    FHC_TRY(check_in(op, "x", x, g->dtype, g->t));
    FHC_TRY(check_in(op, "dt", dt, g->dtype, g->t));
    FHC_TRY(check_in(op, "bm", bm, g->dtype, g->t));
    FHC_TRY(check_in(op, "cm", cm, g->dtype, g->t));
    if (z) FHC_TRY(check_in(op, "z", z, g->dtype, g->t));
    return few_steps ? 0 : check_grid(op, p.wgs, 64 * waves_of(p));  // the step kernel's grid is checked where it is made
}

}  // namespace
}  // namespace seq
}  // namespace fhc

using namespace fhc;
using namespace fhc::seq;

extern "C" size_t fhc_ssm_states_bytes(const fhc_ssm_desc* g) {
    return guard((size_t)0, [&]() -> size_t {
        clear_error();
        if (check_desc("ssm_states_bytes", g) < 0) return 0;
        return (size_t)g->b * ceil_div(g->t, kTile) * ((g->n + 3) / 4) * g->d * 16;
    });
}

extern "C" size_t fhc_ssm_workspace_bytes(const fhc_ssm_desc* g, int backward) {
    return guard((size_t)0, [&]() -> size_t {
        clear_error();
        if (check_desc("ssm_workspace_bytes", g) < 0 || (uint64_t)g->b * g->d == 0) return 0;
        return workspace_of(g, backward != 0);
    });
}

extern "C" int fhc_ssm_forward(const fhc_ssm_desc* g, const fhc_seq* x, const fhc_seq* dt, const fhc_seq* bm,
                               const fhc_seq* cm, const fhc_seq* z, const float* h0, const fhc_seq* y, float* ht,
                               float* states, void* ws, size_t ws_bytes, void* stream) {
    return guard(-3, [&]() -> int {
        clear_error();
        const char* op = "ssm_forward";
        FHC_TRY(check_desc(op, g));
        if ((uint64_t)g->b * g->d == 0) return 0;
        const Plan p = plan_of(g, false, g->lengths != nullptr);
        FHC_TRY(check_inputs(op, g, p, x, dt, bm, cm, z, g->t <= kFewSteps));
        FHC_TRY(check_out(op, "y", y, g->dtype, g->b, g->t, g->d));
        FHC_TRY(check_array(op, "h0", h0, 4, false));
        FHC_TRY(check_array(op, "ht", ht, 4, false));
        if (!aligned(states, 256)) return fail(-1, "%s: states is not 256-byte aligned", op);
        FHC_TRY(check_workspace(op, workspace_of(g, false), ws, ws_bytes));
        const hipStream_t st = (hipStream_t)stream;
        int rc = 0;
        with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            auto a = args_of<T>(g, p, x, dt, bm, cm, z, ws);
            a.h0 = h0, a.y = seq_of<typename T::Raw>(y), a.ht = ht, a.states = reinterpret_cast<f4*>(states);
            if (g->t <= kFewSteps) {
                rc = launch_step<T>(op, p, a, st);
                return;
            }
            if (p.segs > 1) rc = launch<T, kFold>(op, p, a, st);
            if (rc == 0) rc = launch<T, kForward>(op, p, a, st);
        });
        return rc;
    });
}

extern "C" int fhc_ssm_backward(const fhc_ssm_desc* g, const fhc_seq* x, const fhc_seq* dt, const fhc_seq* bm,
                                const fhc_seq* cm, const fhc_seq* z, const float* states, const fhc_seq* dy,
                                const float* dht, const fhc_seq* dx, const fhc_seq* ddt, const fhc_seq* dbm,
                                const fhc_seq* dcm, const fhc_seq* dz, float* da, float* ddt_bias, float* dskip,
                                float* dh0, void* ws, size_t ws_bytes, void* stream) {
    return guard(-3, [&]() -> int {
        clear_error();
        const char* op = "ssm_backward";
        FHC_TRY(check_desc(op, g));
        const hipStream_t st = (hipStream_t)stream;
        FHC_TRY(check_array(op, "da", da, 4, false));
        FHC_TRY(check_array(op, "ddt_bias", ddt_bias, 4, false));
        FHC_TRY(check_array(op, "dskip", dskip, 4, false));
        FHC_TRY(check_array(op, "dh0", dh0, 4, false));
        FHC_TRY(check_array(op, "dht", dht, 4, false));
        const Sums sums{{da, dskip, ddt_bias}, {(uint64_t)g->d * g->n, g->d, g->d}};
        if (g->b == 0) return close_sums(op, nullptr, 0, sums, st);  // empty ones
        FHC_TRY(check_out(op, "dbm", dbm, g->dtype, g->b, g->t, g->groups * g->n));
        FHC_TRY(check_out(op, "dcm", dcm, g->dtype, g->b, g->t, g->groups * g->n));
        int rc = 0;
        if (g->d == 0) {  // no channels that B and C act on
            with_type(g->dtype, [&](auto t) { rc = close_vectors<decltype(t)>(op, g, nullptr, dbm, dcm, 0, st); });
            return rc;
        }
        const Plan p = plan_of(g, true, g->lengths != nullptr);
        FHC_TRY(check_inputs(op, g, p, x, dt, bm, cm, z, false));
        FHC_TRY(check_in(op, "dy", dy, g->dtype, g->t));
        FHC_TRY(check_out(op, "dx", dx, g->dtype, g->b, g->t, g->d));
        FHC_TRY(check_out(op, "ddt", ddt, g->dtype, g->b, g->t, g->d));
        if (z) FHC_TRY(check_out(op, "dz", dz, g->dtype, g->b, g->t, g->d));
        else if (dz) return fail(-1, "%s: dz without z", op);
        if (g->t && !states) return fail(-1, "%s: null states", op);
        if (!aligned(states, 256)) return fail(-1, "%s: states is not 256-byte aligned", op);
        FHC_TRY(check_workspace(op, workspace_of(g, true), ws, ws_bytes));
        with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            using R = typename T::Raw;
            auto a = args_of<T>(g, p, x, dt, bm, cm, z, ws);
            a.states = reinterpret_cast<f4*>(const_cast<float*>(states)), a.dy = seq_of<R>(dy), a.dht = dht;
            a.dx = seq_of<R>(dx), a.ddt = seq_of<R>(ddt), a.dz = seq_of<R>(dz), a.dh0 = dh0;
            if (p.segs > 1) rc = launch<T, kFoldBack>(op, p, a, st);
            if (rc == 0) rc = launch<T, kBackward>(op, p, a, st);
            if (rc == 0) rc = close_vectors<T>(op, g, a.bc, dbm, dcm, p.blocks, st);
        });
        if (rc < 0) return rc;
        const float* part = reinterpret_cast<const float*>(static_cast<char*>(ws) + p.ends_bytes + p.lasts_bytes);
        return close_sums(op, part, p.segs * p.walks * p.stretches, sums, st);
    });
}
