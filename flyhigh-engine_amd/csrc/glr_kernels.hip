// The gated linear recurrence (include/fhc_seq.h), forward and backward.
//
// h_t = a_t h_(t-1) + b_t composes: a stretch of steps is the map h -> A h + S, and two stretches' maps compose to a
// third. So a stretch is read once into registers, folded to its (A, S), and swept again from the state that reaches
// it. The backward pass runs the same way over c -> a_t (dy_t + c), whose stretches have the same A.
//
// A lane holds V channels of one sequence ("column group") for L consecutive steps; W waves of a workgroup hold W
// consecutive stretches of the same columns and exchange their maps through LDS, so a chunk of W * L steps costs one
// barrier. Columns run over sequences and channels together, so narrow maps of many sequences (pixels) fill a wave as
// well as wide rows of one. Chunks follow one another in one of two ways:
//   stream   a workgroup walks all chunks of its columns, the state in registers (many columns, or few steps);
//   chain    a workgroup takes one chunk and publishes its map (few columns, many steps: the time axis is what fills
//            the chip). 8 chunks form a group, 8 groups a run; the state that reaches a chunk is the one at the head of
//            its run folded through the maps of groups and chunks before it (chain_find), and the run's last chunk
//            publishes the next head: a step of the serial chain is a run long, not a chunk.
// In the chain, the chunks of a column block are taken in order by its ticket, so every chunk waited for is held by a
// workgroup that already runs and itself waits for earlier tickets only: every wait ends. What is published is one
// 8-byte word (A, S), or (0, state), written once and read by atomic accesses of the whole word, so no fence orders
// anything; its A is -1 until then (decays are >= 0). Only the first chunk reads the initial state (it publishes it as
// the first head), so the last one may write the final state over it.
//
// What bounds it (MI355X): forward moves 4 elements an element and takes 38 vector instructions, 6 of them
// transcendental, at a quarter of the rate: 65536 x 2048 bf16 need 213 us of HBM and about 200 us of the vector units,
// and take 282. Hence the short polynomial and sigmoids without clamps (138 issue slots an element before), scalar row
// addresses, and 16 steps a lane (half the exchanges of 8). Backward holds six values a step, so registers (occupancy)
// bound it: 1000 x 64 x 512 bf16 about 135 us for 92 us of HBM. Many short sequences are near HBM's rate: 1000 x 64 x 512
// forward 52 us (5.0 TB/s); 1620 x 24 x 128 f16 12.2 us. One long narrow sequence is bound by the chain's tickets and
// words: 65536 x 32 30 us.
#include "glr_place.h"
#include "seq_common.h"

namespace fhc {
namespace seq {
namespace {

struct Col {  // a sequence tensor, strides in bytes
    char* p;
    int64_t bs, ts;
};
// A wave's view of it: the step t of its first lane at p + t * ts, the same for all lanes, and a lane's own 32-bit
// offset from there (no vector arithmetic for an address).
struct Wave {
    char* p;
    int64_t ts;
    uint32_t lane;
    __device__ __forceinline__ Wave(const Col& c, uint32_t b, uint32_t ch, uint32_t elem, bool straddles) : ts(c.ts) {
        const uint32_t b0 = __builtin_amdgcn_readfirstlane(b);
        const uint32_t c0 = base_channel(straddles, __builtin_amdgcn_readfirstlane(ch));
        p = c.p + b0 * c.bs + (uint64_t)c0 * elem;
        lane = lane_offset(b, ch, b0, c0, c.bs, elem);
    }
    // the step's address is made scalar in so many words: the lane's offset is else folded into a vector product
    __device__ __forceinline__ __attribute__((address_space(1))) char* row(uint32_t t) const {
        const uint64_t at = reinterpret_cast<uint64_t>(p) + (uint64_t)((int64_t)t * ts);
        const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)at);
        const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(at >> 32));
        uint32_t own = lane;  // opaque: its extension to 64 bits stays here, where a load takes it for nothing
        asm("" : "+v"(own));
        return (__attribute__((address_space(1))) char*)((uint64_t)hi << 32 | lo) + own;
    }
    template <class C>
    __device__ __forceinline__ C load(uint32_t t) const {
        return __builtin_bit_cast(C, *(__attribute__((address_space(1))) const typename C::Mem*)row(t));
    }
    template <class C>
    __device__ __forceinline__ void store(uint32_t t, C c) const {
        *(__attribute__((address_space(1))) typename C::Mem*)row(t) = __builtin_bit_cast(typename C::Mem, c);
    }
};

struct GlrArgs {
    Col x, r, i, y, dy, dx, dr, di;
    const float* lam;
    const int32_t* lengths;
    const float* h0;
    float* ht;
    float* states;
    const float* dht;
    float* dh0;
    float* part;      // dlam's partial sums, [part rows][d]
    uint64_t* agg;    // chain: published maps [chunk][b * d],
    uint64_t* group_maps;  // those of whole groups [group][b * d],
    uint64_t* heads;       // and the first states of the runs [run][b * d]
    uint32_t* tickets;
    uint32_t b, t, d, groups;  // groups: lanes that a sequence's channels take
    uint32_t nchunk, colblocks, nstates;
    uint32_t spacing;  // log2 of the steps from one kept state to the next: the backward pass's chunk
    bool straddles;    // a wave's columns may run over sequences
    float rate;
};

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

// 1 - 2^(2z) for z <= 0, a2 = 2^(2z). Near 0 the difference cancels, so a polynomial there: (1 - 2^(2z)) / -z
// interpolated at the 4 Chebyshev nodes of [-0.18, 0], off by 2.8e-7 of it, which is what the difference loses at the
// border. A NaN z goes the second way and stays.
__device__ __forceinline__ float one_minus_square(float z, float a) {
    float p = __builtin_fmaf(0.1393723995578612f, z, 0.4424283742923703f);
    p = __builtin_fmaf(p, z, 0.9608486733131862f);
    p = __builtin_fmaf(p, z, 1.3862940389244018f);
    return z > -0.18f ? -z * p : __builtin_fmaf(-a, a, 1.0f);
}

// One step of one channel. Logits of -inf shut their gates: the exponential is inf, its reciprocal 0. A step that is not
// there (past a length) is read as x = 0, r = i = -inf, which leaves the state as it is (a = 1, no input).
struct Gates {
    float er, ei, sr, si, z, a, v;  // e^-r, e^-i; the sigmoids; log2 a; a; 1 - a^2
};
// k2 = -rate * softplus(lam) * log2(e)
__device__ __forceinline__ Gates gates_of(float k2, float r, float i) {
    Gates g;
    g.er = __builtin_amdgcn_exp2f(r * -kLog2e), g.ei = __builtin_amdgcn_exp2f(i * -kLog2e);
    g.sr = __builtin_amdgcn_rcpf(1.0f + g.er), g.si = __builtin_amdgcn_rcpf(1.0f + g.ei);
    g.z = k2 * g.sr;
    g.a = __builtin_amdgcn_exp2f(g.z);
    g.v = one_minus_square(g.z, g.a);
    return g;
}
// 1 - sigmoid(u) = e^-u sigmoid(u), accurate where it is small; inf * 0 where e^-u overflows, and 1 then (a NaN u's is 1
// too, but everything that it multiplies is NaN)
__device__ __forceinline__ float shut(float e, float s) { return __builtin_fminf(e * s, 1.0f); }

// The V channels of a lane as they lie in memory: a pair of 16-bit elements stays one register until it is used.
template <class T, int V>
struct Cell {
    typedef typename T::Raw Mem __attribute__((ext_vector_type(V)));
    typename T::Raw e[V];
    static constexpr float kLow = -__builtin_inff();
    __device__ __forceinline__ float at(int v) const { return widen(T{}, e[v]); }
    static __device__ __forceinline__ Cell of(const float (&f)[V]) {
        Cell c;
#pragma unroll
        for (int v = 0; v < V; v++) c.e[v] = narrow(T{}, f[v]);
        return c;
    }
    __device__ __forceinline__ Cell where(bool on) const {
        Cell c;
#pragma unroll
        for (int v = 0; v < V; v++) c.e[v] = on ? e[v] : typename T::Raw(0);
        return c;
    }
    __device__ __forceinline__ void forget() {
#pragma unroll
        for (int v = 0; v < V; v++) asm volatile("" : "+v"(e[v]));
    }
    static __device__ __forceinline__ Cell zero() { return Cell{}; }
    static __device__ __forceinline__ Cell lowest() {
        float f[V];
#pragma unroll
        for (int v = 0; v < V; v++) f[v] = kLow;
        return of(f);
    }
};
template <class T>
struct Pair {
    using Mem = uint32_t;
    uint32_t e;
    __device__ __forceinline__ float at(int v) const { return widen(T{}, (uint16_t)(v ? e >> 16 : e)); }
    static __device__ __forceinline__ Pair of(const float (&f)[2]) {
        return {(uint32_t)narrow(T{}, f[0]) | (uint32_t)narrow(T{}, f[1]) << 16};
    }
    __device__ __forceinline__ Pair where(bool on) const { return {on ? e : 0u}; }
    __device__ __forceinline__ void forget() { asm volatile("" : "+v"(e)); }
    static __device__ __forceinline__ Pair zero() { return {0u}; }
    static __device__ __forceinline__ Pair lowest() {
        return {T::id == FHC_F16 ? 0xFC00FC00u : 0xFF80FF80u};
    }
};
template <>
struct Cell<F16, 2> : Pair<F16> {
    __device__ Cell() = default;
    __device__ __forceinline__ Cell(Pair<F16> p) : Pair<F16>(p) {}
};
template <>
struct Cell<BF16, 2> : Pair<BF16> {
    __device__ Cell() = default;
    __device__ __forceinline__ Cell(Pair<BF16> p) : Pair<BF16>(p) {}
};

// L steps from t0 on of the lane's channels, those at and past n as `absent`. Where no lane of the wave has such a
// step, the loads stand without a branch.
template <class C, int L>
__device__ __forceinline__ void load_steps(const Wave& w, uint32_t t0, uint32_t n, bool full, C absent, C (&o)[L]) {
    if (full) {
#pragma unroll
        for (int l = 0; l < L; l++) o[l] = w.load<C>(t0 + l);
    } else {
#pragma unroll
        for (int l = 0; l < L; l++) {
            o[l] = absent;
            if (t0 + l < n) o[l] = w.load<C>(t0 + l);
        }
    }
}

// log2 of the decay of an open gate: -rate * softplus(lam) * log2(e), softplus = max(lam, 0) + log1p(e^-|lam|).
// Short, since a lane may use it for few steps: e^-|lam| with its argument's rounding put back, and log1p(e) = 2 atanh(s),
// s = e / (2 + e) <= 1/3, whose series' 7 terms leave 1.4e-8 of it.
__device__ __forceinline__ float decay_rate(float rate, float lam) {
    const float u = -__builtin_fabsf(lam), t = u * kLog2e;
    const float lost = __builtin_fmaf(u, kLog2e, -t) + u * 1.92596299e-8f;  // log2(e) - kLog2e
    float e = __builtin_amdgcn_exp2f(t);
    e = e > 0.0f ? __builtin_fmaf(e * kLn2, lost, e) : lam == lam ? 0.0f : lam;  // of 0 and -inf: no correction
    const float s = e * __builtin_amdgcn_rcpf(2.0f + e), q = s * s;
    float p = __builtin_fmaf(q, 1.0f / 13.0f, 1.0f / 11.0f);
    p = __builtin_fmaf(p, q, 1.0f / 9.0f);
    p = __builtin_fmaf(p, q, 1.0f / 7.0f);
    p = __builtin_fmaf(p, q, 1.0f / 5.0f);
    p = __builtin_fmaf(p, q, 1.0f / 3.0f);
    p = __builtin_fmaf(p, q, 1.0f);
    const float sp = (lam > 0.0f ? lam : 0.0f) + 2.0f * s * p;
    const float k = -rate * sp * kLog2e;
    return k < -3.4e38f ? -3.4e38f : k;  // finite: times a shut gate's 0 it is 0
}

__device__ __forceinline__ uint64_t word_of(float a, float s) {
    return (uint64_t)__builtin_bit_cast(uint32_t, a) | (uint64_t)__builtin_bit_cast(uint32_t, s) << 32;
}
constexpr uint64_t kUnpublished = 0xBF800000ull;  // (-1, 0)
__device__ __forceinline__ void publish(uint64_t* p, float a, float s) {
    __hip_atomic_store(p, word_of(a, s), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
constexpr uint32_t kGroup = 8, kRun = kGroup * kGroup;  // chunks of a group; of a run

constexpr uint32_t kTicketStep = 32;  // a column block's ticket has 128 bytes of its own

__global__ __launch_bounds__(256) void glr_clear(uint64_t* agg, uint64_t n, uint32_t* tickets, uint32_t colblocks) {
    const uint64_t k = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (k < n) agg[k] = kUnpublished;
    if (k < colblocks) tickets[k * kTicketStep] = 0;
}

// The chain's search: the state that reaches this lane's columns of a chunk, the k-th of its run (k = 8 group + j): the
// run's first state through the maps of the groups before the chunk's and of the j chunks before it in its group. A
// chunk so reads 15 words a column at most, and a run is 64 chunks (runs of 32 without groups: one sequence of 65536 x 32
// bf16 took 43 us, with groups 30). The W waves fetch the words together, a wave all
// of its own at once, and again until they are all there; the folds are in the chunks' order whatever the order of their
// arrival, so results repeat bit for bit.
//   agg, groups, heads: the run's first words of this column block's lane, `flats` words from one to the next
//   a, s: the chunk's own map. The last chunk of a group publishes the group's before it looks for anything else.
template <int V, int W>
__device__ __forceinline__ void chain_find(uint32_t k, bool first_run, bool more, uint32_t tw, uint32_t slot, bool live,
                                           float2 (*lds)[64 * V], const uint64_t* agg, uint64_t* groups,
                                           const uint64_t* head, uint64_t flats, const float (&a)[V], const float (&s)[V],
                                           float (&h)[V]) {
    constexpr uint32_t N = 16 / W;  // entries of a wave: 0-6 chunks, 7-13 groups, 15 the head
    const uint32_t group = k / kGroup, j = k % kGroup;
    const bool has_head = !first_run || k > 0;
    auto fetch = [&](uint32_t from, uint32_t to) {
        if (live) {
            uint64_t w[N][V];
            bool missing;
            do {
#pragma unroll
                for (uint32_t n = 0; n < N; n++) {
                    const uint32_t e = n * W + tw;
                    const uint64_t* p = nullptr;
                    if (e >= from && e < to) {
                        if (e < 7) p = e < j ? agg + (group * kGroup + e) * flats : nullptr;
                        else if (e < 14) p = e - 7 < group ? groups + (e - 7) * flats : nullptr;
                        else p = e == 15 && has_head ? head : nullptr;
                    }
#pragma unroll
                    for (int v = 0; v < V; v++) {
                        w[n][v] = 0;
                        if (p) w[n][v] = __hip_atomic_load(p + v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    }
                }
                missing = false;
#pragma unroll
                for (uint32_t n = 0; n < N; n++)
#pragma unroll
                    for (int v = 0; v < V; v++) missing |= (uint32_t)w[n][v] == (uint32_t)kUnpublished;
            } while (missing);
#pragma unroll
            for (uint32_t n = 0; n < N; n++) {
                const uint32_t e = n * W + tw;
                if (e < from || e >= to) continue;
#pragma unroll
                for (int v = 0; v < V; v++)
                    lds[e][slot * V + v] = float2{__builtin_bit_cast(float, (uint32_t)w[n][v]),
                                                 __builtin_bit_cast(float, (uint32_t)(w[n][v] >> 32))};
            }
        }
        __syncthreads();
    };
    const bool closes = j == kGroup - 1 && group < kGroup - 1 && more;  // the same for the whole workgroup
    if (closes) {
        fetch(0, 7);
        if (live && tw == 0) {
#pragma unroll
            for (int v = 0; v < V; v++) {
                float ga = 1.0f, gs = 0.0f;
#pragma unroll
                for (uint32_t e = 0; e < 7; e++) {
                    const float2 q = lds[e][slot * V + v];
                    gs = __builtin_fmaf(q.x, gs, q.y);
                    ga *= q.x;
                }
                publish(groups + group * flats + v, a[v] * ga, __builtin_fmaf(a[v], gs, s[v]));
            }
        }
    }
    fetch(closes ? 7 : 0, 16);
    if (!live) return;
    if (has_head) {
#pragma unroll
        for (int v = 0; v < V; v++) h[v] = lds[15][slot * V + v].y;
    }
    for (uint32_t e = 0; e < group; e++) {
#pragma unroll
        for (int v = 0; v < V; v++) {
            const float2 q = lds[7 + e][slot * V + v];
            h[v] = __builtin_fmaf(q.x, h[v], q.y);
        }
    }
    for (uint32_t e = 0; e < j; e++) {
#pragma unroll
        for (int v = 0; v < V; v++) {
            const float2 q = lds[e][slot * V + v];
            h[v] = __builtin_fmaf(q.x, h[v], q.y);
        }
    }
}

// Which columns and chunk a workgroup has. Every column block has a ticket of its own: its chunks are taken in order.
template <bool CHAIN>
__device__ __forceinline__ uint32_t take_chunk(const GlrArgs& g, uint32_t& cb) {
    if constexpr (!CHAIN) return 0;
    __shared__ uint32_t taken;
    cb = blockIdx.x % g.colblocks;
    if (threadIdx.x == 0) taken = atomicAdd(g.tickets + cb * kTicketStep, 1u);
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(taken);
}

// W waves of consecutive stretches x CW waves of column groups
template <class T, int V, int L, int W, int CW, bool CHAIN>
__global__ __launch_bounds__(64 * W * CW, L > 8 ? (CHAIN && sizeof(typename T::Raw) == 2 ? 4 : 3) : 1) void glr_fwd(GlrArgs g) {
    using R = typename T::Raw;
    using C = Cell<T, V>;
    constexpr int CL = W * L;
    constexpr bool ONE = W > 1 && W < 8;  // these chunks hold whole sequences
    __shared__ float2 maps[W > 1 ? W : 1][W > 1 ? CW * 64 * V : 1];
    __shared__ float2 far[CHAIN ? 16 : 1][CHAIN ? 64 * V : 1];
    static_assert(!CHAIN || CW == 1, "a chained chunk's columns are one wave wide");
    uint32_t cb = blockIdx.x, chunk = take_chunk<CHAIN>(g, cb);
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tw = W > 1 ? wave % W : 0, slot = (W > 1 ? wave / W : wave) * 64 + lane;
    const uint32_t col = cb * (CW * 64) + slot;
    uint32_t b = col / g.groups, ch = (col - b * g.groups) * V;
    const bool live = b < g.b && ch < g.d;
    if (!live) b = ch = 0;
    const uint64_t flat = (uint64_t)b * g.d + ch;
    const uint32_t n = live ? (g.lengths ? (uint32_t)min(max(g.lengths[b], 0), (int32_t)g.t) : g.t) : 0;

    float k[V], h[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
        k[v] = live ? decay_rate(g.rate, g.lam[ch + v]) : 0.0f;
        h[v] = live && g.h0 && (!CHAIN || chunk == 0) ? g.h0[flat + v] : 0.0f;
    }
    auto wave_of = [&](const Col& c) { return Wave(c, b, ch, sizeof(R), g.straddles); };
    const Wave wx = wave_of(g.x), wr = wave_of(g.r), wi = wave_of(g.i), wy = wave_of(g.y);

    const uint32_t last = CHAIN ? chunk + 1 : ONE ? 1 : g.nchunk;
    for (; chunk < last; chunk++) {
        const uint32_t t0 = chunk * CL + tw * L;
        const bool full = __all(t0 + L <= n), some = __any(t0 < n);
        float a[L][V], in[L][V], A[V], S[V];
#pragma unroll
        for (int v = 0; v < V; v++) A[v] = 1.0f, S[v] = 0.0f;
        if (some) {
            C xr[L], rr[L], ir[L];
            load_steps(wr, t0, n, full, C(C::lowest()), rr);
            load_steps(wi, t0, n, full, C(C::lowest()), ir);
            load_steps(wx, t0, n, full, C(C::zero()), xr);
#pragma unroll
            for (int l = 0; l < L; l++) {
#pragma unroll
                for (int v = 0; v < V; v++) {
                    const Gates q = gates_of(k[v], rr[l].at(v), ir[l].at(v));
                    a[l][v] = q.a, in[l][v] = __builtin_amdgcn_sqrtf(q.v) * (q.si * xr[l].at(v));
                    if constexpr (W > 1) {
                        S[v] = __builtin_fmaf(a[l][v], S[v], in[l][v]);
                        A[v] *= a[l][v];
                    }
                }
            }
        }
        float end[V];  // the state after the chunk
        if constexpr (W > 1) {
#pragma unroll
            for (int v = 0; v < V; v++) maps[tw][slot * V + v] = float2{A[v], S[v]};
            __syncthreads();
            float pa[V], ps[V], ta[V], ts[V];  // the maps of the stretches before this one, and of the whole chunk
#pragma unroll
            for (int v = 0; v < V; v++) pa[v] = ta[v] = 1.0f, ps[v] = ts[v] = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++) {
                if (w == (int)tw) {
#pragma unroll
                    for (int v = 0; v < V; v++) pa[v] = ta[v], ps[v] = ts[v];
                }
#pragma unroll
                for (int v = 0; v < V; v++) {
                    const float2 q = maps[w][slot * V + v];
                    ts[v] = __builtin_fmaf(q.x, ts[v], q.y);
                    ta[v] *= q.x;
                }
            }
            if constexpr (CHAIN) {
                const uint64_t flats = (uint64_t)g.b * g.d;
                const uint32_t run = chunk / kRun, k = chunk - run * kRun;
                const bool more = chunk + 1 < g.nchunk;
                if (tw == 0 && live && k % kGroup < kGroup - 1 && more) {
#pragma unroll
                    for (int v = 0; v < V; v++) publish(g.agg + chunk * flats + flat + v, ta[v], ts[v]);
                }
                if (tw == 0 && live && chunk == 0 && more) {
#pragma unroll
                    for (int v = 0; v < V; v++) publish(g.heads + flat + v, 0.0f, h[v]);
                }
                chain_find<V, W>(k, run == 0, more, tw, slot, live, far, g.agg + run * kRun * flats + flat,
                                 g.group_maps + run * kGroup * flats + flat, g.heads + run * flats + flat, flats, ta, ts, h);
#pragma unroll
                for (int v = 0; v < V; v++) end[v] = __builtin_fmaf(ta[v], h[v], ts[v]);
                if (tw == 0 && live && k + 1 == kRun && chunk + 1 < g.nchunk) {
#pragma unroll
                    for (int v = 0; v < V; v++) publish(g.heads + (run + 1) * flats + flat + v, 0.0f, end[v]);
                }
            } else {
#pragma unroll
                for (int v = 0; v < V; v++) end[v] = __builtin_fmaf(ta[v], h[v], ts[v]);
                __syncthreads();  // the maps are read before the next chunk's are written
            }
#pragma unroll
            for (int v = 0; v < V; v++) h[v] = __builtin_fmaf(pa[v], h[v], ps[v]);
        }
        // the states that the backward pass starts its chunks from
        if (g.states && live && (t0 & ((1u << g.spacing) - 1)) == 0 && t0 < g.t) {
#pragma unroll
            for (int v = 0; v < V; v++) g.states[((uint64_t)b * g.nstates + (t0 >> g.spacing)) * g.d + ch + v] = h[v];
        }
        if (some) {
#pragma unroll
            for (int l = 0; l < L; l++) {
#pragma unroll
                for (int v = 0; v < V; v++) h[v] = __builtin_fmaf(a[l][v], h[v], in[l][v]);
                const C out = C::of(h);
                if (full || (live && t0 + l < g.t)) wy.store(t0 + l, C(out.where(full || t0 + l < n)));
            }
        } else {
            for (int l = 0; l < L; l++)
                if (live && t0 + l < g.t) wy.store(t0 + l, C(C::zero()));
        }
        if constexpr (W > 1) {
#pragma unroll
            for (int v = 0; v < V; v++) h[v] = end[v];
        }
    }
    if (live && g.ht && tw == 0 && last == g.nchunk) {
#pragma unroll
        for (int v = 0; v < V; v++) g.ht[flat + v] = h[v];
    }
}

// Backward. With g_t = dy_t + c_t, c_(t-1) = a_t g_t the gradient that reaches the state before a step:
//     dx = g m si,   di = g m si x (1 - si),   d/d(log a) = a g (h_(t-1) - a w / m),   w = si x, m = sqrt(1 - a^2)
//     dr = d/d(log a) log a (1 - sr),   dlam = sum of d/d(log a) sr * -rate sigmoid(lam)
// A lane keeps six values a step while the chunk's maps are exchanged (and x and dy as they were read): more registers
// would cost the waves that hide the loads.
template <class T, int V, int L, int W, int CW, bool CHAIN>
__global__ __launch_bounds__(64 * W * CW, L == 1 ? 1 : L == 4 ? 4 : 3) void glr_bwd(GlrArgs g) {
    using R = typename T::Raw;
    using C = Cell<T, V>;
    constexpr int CL = W * L;
    constexpr bool ONE = W > 1 && W < 8;  // these chunks hold whole sequences
    __shared__ float2 maps[W > 1 ? W : 1][W > 1 ? CW * 64 * V : 1];  // (A, S) forward
    __shared__ float back[W > 1 ? W : 1][W > 1 ? CW * 64 * V : 1];   // the R of c -> A c + R
    __shared__ float2 far[CHAIN ? 16 : 1][CHAIN ? 64 * V : 1];
    static_assert(!CHAIN || CW == 1, "a chained chunk's columns are one wave wide");
    uint32_t cb = blockIdx.x, done = take_chunk<CHAIN>(g, cb);  // chunks go from the last to the first
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tw = W > 1 ? wave % W : 0, slot = (W > 1 ? wave / W : wave) * 64 + lane;
    const uint32_t col = cb * (CW * 64) + slot;
    uint32_t b = col / g.groups, ch = (col - b * g.groups) * V;
    const bool live = b < g.b && ch < g.d;
    if (!live) b = ch = 0;
    const uint64_t flat = (uint64_t)b * g.d + ch;
    const uint32_t n = live ? (g.lengths ? (uint32_t)min(max(g.lengths[b], 0), (int32_t)g.t) : g.t) : 0;

    float k[V], c[V], lam_sum[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
        k[v] = live ? decay_rate(g.rate, g.lam[ch + v]) : 0.0f;
        c[v] = live && g.dht && (!CHAIN || done == 0) ? g.dht[flat + v] : 0.0f;
        lam_sum[v] = 0.0f;
    }
    auto wave_of = [&](const Col& c) { return Wave(c, b, ch, sizeof(R), g.straddles); };
    const Wave wx = wave_of(g.x), wr = wave_of(g.r), wi = wave_of(g.i), wdy = wave_of(g.dy), wdx = wave_of(g.dx),
               wdr = wave_of(g.dr), wdi = wave_of(g.di);

    const uint32_t last = CHAIN ? done + 1 : ONE ? 1 : g.nchunk;
    for (; done < last; done++) {
        const uint32_t chunk = g.nchunk - 1 - done, t0 = chunk * CL + tw * L;
        C xr[L], gr[L];
        const bool full = __all(t0 + L <= n), some = __any(t0 < n);
        float h[V];
#pragma unroll
        for (int v = 0; v < V; v++)
            h[v] = live && chunk < g.nstates ? g.states[((uint64_t)b * g.nstates + chunk) * g.d + ch + v] : 0.0f;
        // p = m si; q = a w / m, later h_(t-1) - q
        float a[L][V], p[L][V], q[L][V], sr[L][V], lr[L][V], ni[L][V], A[V], S[V], B[V];
#pragma unroll
        for (int v = 0; v < V; v++) A[v] = 1.0f, S[v] = 0.0f, B[v] = 0.0f;
        if (some) {
            C rr[L], ir[L];
            load_steps(wr, t0, n, full, C(C::lowest()), rr);
            load_steps(wi, t0, n, full, C(C::lowest()), ir);
            load_steps(wx, t0, n, full, C(C::zero()), xr);
            load_steps(wdy, t0, n, full, C(C::zero()), gr);
#pragma unroll
            for (int l = 0; l < L; l++) {
                // one step after the other: with every step's exponentials taken first, as the compiler would, the gates of
                // all steps are alive together
                rr[l].forget(), ir[l].forget();
#pragma unroll
                for (int v = 0; v < V; v++) {
                    const Gates s = gates_of(k[v], rr[l].at(v), ir[l].at(v));
                    const float x = xr[l].at(v), dy = gr[l].at(v);
                    // 1 - a^2 is 0 where nothing decays, and no larger than log a: the gradient that passes through m's
                    // root, log a / m, is 0 at this limit (times a finite value)
                    const float rm = __builtin_amdgcn_rsqf(__builtin_fmaxf(s.v, 1.17549435e-38f));
                    a[l][v] = s.a, sr[l][v] = s.sr;
                    lr[l][v] = s.z * kLn2 * shut(s.er, s.sr);
                    ni[l][v] = shut(s.ei, s.si);
                    p[l][v] = s.v * rm * s.si;
                    q[l][v] = s.a * rm * (s.si * x);
                    if constexpr (W > 1) {
                        S[v] = __builtin_fmaf(s.a, S[v], p[l][v] * x);
                        A[v] *= s.a;
                        B[v] = __builtin_fmaf(A[v], dy, B[v]);  // dy_l reaches the front through a_1 .. a_l
                    }
                    asm volatile("" : "+v"(p[l][v]), "+v"(q[l][v]), "+v"(lr[l][v]), "+v"(ni[l][v]));
                }
            }
        }
        float end[V];  // what the chunk hands to the chunk before it
        if constexpr (W > 1) {
#pragma unroll
            for (int v = 0; v < V; v++) {
                maps[tw][slot * V + v] = float2{A[v], S[v]};
                back[tw][slot * V + v] = B[v];
            }
            __syncthreads();
            float pa[V], ps[V], ta[V], ts[V];  // c of this stretch, and of the whole chunk, from the chunk's c
#pragma unroll
            for (int v = 0; v < V; v++) pa[v] = ta[v] = 1.0f, ps[v] = ts[v] = 0.0f;
            for (int w = 0; w < (int)tw; w++) {  // the state that reaches the stretch
#pragma unroll
                for (int v = 0; v < V; v++) {
                    const float2 m = maps[w][slot * V + v];
                    h[v] = __builtin_fmaf(m.x, h[v], m.y);
                }
            }
#pragma unroll
            for (int w = W - 1; w >= 0; w--) {
                if (w == (int)tw) {
#pragma unroll
                    for (int v = 0; v < V; v++) pa[v] = ta[v], ps[v] = ts[v];
                }
#pragma unroll
                for (int v = 0; v < V; v++) {
                    const float m = maps[w][slot * V + v].x;
                    ts[v] = __builtin_fmaf(m, ts[v], back[w][slot * V + v]);
                    ta[v] *= m;
                }
            }
            if constexpr (CHAIN) {
                const uint64_t flats = (uint64_t)g.b * g.d;
                const uint32_t run = done / kRun, k = done - run * kRun;
                const bool more = chunk > 0;
                if (tw == 0 && live && k % kGroup < kGroup - 1 && more) {
#pragma unroll
                    for (int v = 0; v < V; v++) publish(g.agg + done * flats + flat + v, ta[v], ts[v]);
                }
                if (tw == 0 && live && done == 0 && more) {
#pragma unroll
                    for (int v = 0; v < V; v++) publish(g.heads + flat + v, 0.0f, c[v]);
                }
                chain_find<V, W>(k, run == 0, more, tw, slot, live, far, g.agg + run * kRun * flats + flat,
                                 g.group_maps + run * kGroup * flats + flat, g.heads + run * flats + flat, flats, ta, ts, c);
#pragma unroll
                for (int v = 0; v < V; v++) end[v] = __builtin_fmaf(ta[v], c[v], ts[v]);
                if (tw == 0 && live && k + 1 == kRun && chunk > 0) {
#pragma unroll
                    for (int v = 0; v < V; v++) publish(g.heads + (run + 1) * flats + flat + v, 0.0f, end[v]);
                }
            } else {
#pragma unroll
                for (int v = 0; v < V; v++) end[v] = __builtin_fmaf(ta[v], c[v], ts[v]);
                __syncthreads();
            }
#pragma unroll
            for (int v = 0; v < V; v++) c[v] = __builtin_fmaf(pa[v], c[v], ps[v]);
        }
        if (some) {
            // what was derived from x and dy is derived again: the compiler would keep it in registers across the exchange
#pragma unroll
            for (int l = 0; l < L; l++) xr[l].forget(), gr[l].forget();
#pragma unroll
            for (int l = 0; l < L; l++) {
#pragma unroll
                for (int v = 0; v < V; v++) {
                    q[l][v] = h[v] - q[l][v];
                    h[v] = __builtin_fmaf(a[l][v], h[v], p[l][v] * xr[l].at(v));
                }
            }
#pragma unroll
            for (int l = L - 1; l >= 0; l--) {
                const bool on = full || t0 + l < n;
                float ox[V], orr[V], oi[V];
#pragma unroll
                for (int v = 0; v < V; v++) {
                    const float gt = gr[l].at(v) + c[v];
                    c[v] = a[l][v] * gt;
                    const float dla = on ? c[v] * q[l][v] : 0.0f;
                    ox[v] = gt * p[l][v];
                    orr[v] = dla * lr[l][v];
                    oi[v] = ox[v] * xr[l].at(v) * ni[l][v];
                    lam_sum[v] = __builtin_fmaf(dla, sr[l][v], lam_sum[v]);
                }
                if (full || (live && t0 + l < g.t)) {
                    wdx.store(t0 + l, C(C(C::of(ox)).where(on)));
                    wdr.store(t0 + l, C(C::of(orr)));
                    wdi.store(t0 + l, C(C(C::of(oi)).where(on)));
                }
            }
        } else {
            for (int l = 0; l < L; l++) {
                if (!live || t0 + l >= g.t) continue;
                wdx.store(t0 + l, C(C::zero()));
                wdr.store(t0 + l, C(C::zero()));
                wdi.store(t0 + l, C(C::zero()));
            }
        }
        if constexpr (W > 1) {
#pragma unroll
            for (int v = 0; v < V; v++) c[v] = end[v];
        }
    }
    if (live && g.dh0 && tw == 0 && last == g.nchunk) {
#pragma unroll
        for (int v = 0; v < V; v++) g.dh0[flat + v] = c[v];
    }
    if constexpr (W > 1) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; v++) back[tw][slot * V + v] = lam_sum[v];
        __syncthreads();
        if (tw == 0) {
#pragma unroll
            for (int v = 0; v < V; v++) {
#pragma unroll
                for (int w = 1; w < W; w++) lam_sum[v] += back[w][slot * V + v];
            }
        }
    }
    if (live && tw == 0) {
        const uint64_t row = (uint64_t)(CHAIN ? last - 1 : 0) * g.b + b;
#pragma unroll
        for (int v = 0; v < V; v++) g.part[row * g.d + ch + v] = lam_sum[v];
    }
}

// Column sums of the partial rows: 16 columns x 64 row lanes a workgroup, rows y, y + gridDim.y * 64, ...; a second
// launch with one row block finishes. In f64: millions of terms of either sign meet here. `first`: the launch's first 16
// columns.
template <class In, bool LAST>
__global__ __launch_bounds__(1024) void glr_sum(const In* part, uint64_t rows, uint32_t d, double* out, float* dlam,
                                                const float* lam, float rate, uint32_t first) {
    __shared__ double s[64][17];
    const uint32_t c0 = (first + blockIdx.x) * 16, x = threadIdx.x & 15, ch = c0 + x, y = threadIdx.x >> 4;
    double acc = 0.0;
    if (ch < d) {
#pragma unroll 8
        for (uint64_t r = (uint64_t)blockIdx.y * 64 + y; r < rows; r += (uint64_t)gridDim.y * 64)
            acc += (double)part[r * d + ch];
    }
    s[y][x] = acc;
    __syncthreads();
    if (threadIdx.x < 64) {  // 4 lanes a column, 16 rows each
        const uint32_t col = threadIdx.x >> 2, q = threadIdx.x & 3, c = c0 + col;
        acc = 0.0;
#pragma unroll
        for (int k = 0; k < 16; k++) acc += s[q * 16 + k][col];
        acc += __shfl_xor(acc, 1);
        acc += __shfl_xor(acc, 2);
        if (q == 0 && c < d) {
            if constexpr (LAST) {
                const float e = expf(-fabsf(lam[c]));  // d softplus / d lam = sigmoid(lam)
                const float sg = (lam[c] >= 0.0f ? 1.0f : e) / (1.0f + e);
                dlam[c] = (float)(acc * -(double)rate * (double)sg);
            } else {
                out[(uint64_t)blockIdx.y * d + c] = acc;
            }
        }
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------

constexpr int kL = 8;              // steps a lane holds
constexpr uint32_t kOneSum = 512;  // partial rows up to which one launch adds them
constexpr uint32_t kSumRows = 64;  // row blocks of the first sum otherwise

struct Plan {
    int l, w;    // steps of a stretch; stretches (waves) of a chunk
    bool chain, straddles;
    uint32_t v, groups, nchunk, colblocks, nstates, spacing;
    uint64_t words;      // of the chain: maps, then heads
    uint64_t part_rows;  // of dlam's partial sums
    size_t agg_bytes, part_bytes, sum_bytes;
};

// One wave per column group walks kL steps at a time (one, for a single token) where that alone fills the chip or
// there is little to split; else up to 8 waves share a chunk, and chunks are chained where the columns give fewer than
// two workgroups a CU. Measured, bf16, rows of 512 channels, us forward and a training step, at both sides of the lines:
//   columns  steps   one wave   eight waves         columns  steps   eight waves in a stream   chained
//   2^17        64    24   63     17   50           2^14       128    10   32                   13   35
//              256    98  263     79  206                     1024    57  209                   37  129
//   2^18        64    31   95     27  100           2^15       128    12   37                   15   41
//              256   127  351    151  399                     1024    73  239                   68  240
//   2^19        64    55  180     53  193                     4096   267  929                  255  897
//              256   225  670    282  737           2^16      1024   138  363                  128  451
// (2^18 columns of long sequences would be ahead with one wave, chains of few steps in a stream.) v: the channels a lane takes; near: a wave's columns may run over sequences, since the offsets
// between them fit a lane's 32 bits; else each sequence starts a wave of its own.
Plan plan_of(const fhc_glr_desc* g, bool backward, uint32_t v, bool near) {
    Plan p{};
    p.v = v, p.straddles = near && g->b > 1;
    p.groups = near ? g->d / v : (uint32_t)ceil_div(g->d / v, 64) * 64;
    const uint64_t cols = (uint64_t)g->b * p.groups;
    const uint64_t flat = (uint64_t)g->b * g->d;
    p.l = g->t == 1 ? 1 : kL;
    p.w = flat >= (1u << 19) || g->t <= kL ? 1 : g->t <= 2 * kL ? 2 : g->t <= 4 * kL ? 4 : 8;
    p.chain = g->t > 8 * kL && p.w == 8 && flat < (1u << 16);
    // backward, whose steps take twice the registers: half as many a lane where chunks follow one another in a workgroup
    // (two workgroups a CU instead of one: 1000 x 64 x 512 bf16 222 -> 191 us a training step), and one channel a lane
    // where they are chained, whose number should not grow
    const bool half = p.w == 8 && !p.chain;
    p.spacing = p.w == 1 ? 3 : p.w == 2 ? 4 : p.w == 4 || half ? 5 : 6;
    if (backward) p.l = half ? kL / 2 : p.l;
    else if (g->t >= 16 * kL && p.w == 8) p.l = 2 * kL;
    p.nchunk = (uint32_t)(g->t ? ceil_div(g->t, p.l * p.w) : 1);
    p.nstates = (uint32_t)ceil_div(g->t, 1u << p.spacing);
    p.colblocks = (uint32_t)ceil_div(cols, p.w >= 4 ? 64 : p.w == 2 ? 128 : 256);
    p.words = p.chain ? (p.nchunk + ceil_div(p.nchunk, kGroup) + ceil_div(p.nchunk, kRun)) * flat : 0;
    p.agg_bytes = p.chain ? p.words * 8 + (size_t)g->b * ceil_div(g->d, 64) * kTicketStep * 4 : 0;
    p.part_bytes = (size_t)ceil_div((p.chain ? p.nchunk : 1) * flat * 4, 256) * 256;
    p.part_rows = (uint64_t)(p.chain ? p.nchunk : 1) * g->b;
    p.sum_bytes = p.part_rows > kOneSum ? (size_t)kSumRows * g->d * 8 : 0;
    return p;
}

int check_desc(const char* op, const fhc_glr_desc* g) {
    if (!g) return fail(-1, "%s: null descriptor", op);
    if (g->dtype > FHC_F32) return fail(-1, "%s: dtype %u is none of f16, bf16, f32", op, g->dtype);
    if (!(g->rate >= 0.0f) || !std::isfinite(g->rate)) return fail(-1, "%s: rate %g", op, (double)g->rate);
    if ((uint64_t)g->b * g->d >= 1ull << 31) return fail(-1, "%s: %u x %u columns, at most 2^31 - 1", op, g->b, g->d);
    if (g->t > 0x7FFFFF00u) return fail(-1, "%s: %u steps", op, g->t);
    if (g->b && g->d && !g->lam) return fail(-1, "%s: null lam", op);
    return 0;
}
int check_seq(const char* op, const char* name, const fhc_seq* s, const fhc_glr_desc* g) {
    if (!s) return fail(-1, "%s: null %s", op, name);
    if (g->t && !s->p) return fail(-1, "%s: null pointer of %s", op, name);
    if (!aligned(s->p, elem_bytes(g->dtype))) return fail(-1, "%s: %s is not aligned to its elements", op, name);
    return 0;
}
int check_out(const char* op, const char* name, const fhc_seq* s, const fhc_glr_desc* g) {
    FHC_TRY(check_seq(op, name, s, g));
    // an output's elements are distinct addresses where its strides leave room for a row of channels
    if (g->t > 1 && (uint64_t)std::llabs(s->ts) < g->d)
        return fail(-1, "%s: %s: steps %lld apart overlap", op, name, (long long)s->ts);
    if (g->b > 1 && (uint64_t)std::llabs(s->bs) < g->d)
        return fail(-1, "%s: %s: sequences %lld apart overlap", op, name, (long long)s->bs);
    return 0;
}

Col col(const fhc_seq* s, uint32_t dtype) {
    const int64_t e = elem_bytes(dtype);
    return Col{static_cast<char*>(s->p), s->bs * e, s->ts * e};
}

// the plan for these tensors: pairs of channels as one load, waves over several sequences, where every one allows it
Plan plan_for(const fhc_glr_desc* g, bool backward, std::initializer_list<const fhc_seq*> all) {
    bool pairs = g->d % 2 == 0, near = true;
    const int64_t e = elem_bytes(g->dtype);
    for (const fhc_seq* s : all) {
        if ((g->b > 1 && s->bs % 2) || (g->t > 1 && s->ts % 2) || !aligned(s->p, 2 * (uint32_t)e)) pairs = false;
        if (!near_sequences(g->b, g->d, s->bs, (uint32_t)e)) near = false;
    }
    if (backward && plan_of(g, true, 1, near).chain) pairs = false;
    return plan_of(g, backward, pairs ? 2 : 1, near);
}

template <class F>
void with_type(uint32_t dtype, F&& f) {
    if (dtype == FHC_F16) f(F16{});
    else if (dtype == FHC_BF16) f(BF16{});
    else f(F32{});
}

template <bool BWD, class T, int V>
void launch(const Plan& p, const GlrArgs& a, hipStream_t s) {
#define GLR(L, W, CW, CHAIN, GRID)                                                                          \
    do {                                                                                                    \
        if constexpr (BWD)                                                                                  \
            hipLaunchKernelGGL((glr_bwd<T, V, L, W, CW, CHAIN>), dim3(GRID), dim3(64 * W * CW), 0, s, a);   \
        else                                                                                                \
            hipLaunchKernelGGL((glr_fwd<T, V, L, W, CW, CHAIN>), dim3(GRID), dim3(64 * W * CW), 0, s, a);   \
    } while (0)
    if constexpr (!BWD) {
        if (p.l > kL) {
            if (p.chain) GLR(2 * kL, 8, 1, true, p.colblocks * p.nchunk);
            else GLR(2 * kL, 8, 1, false, p.colblocks);
            return;
        }
    }
    if constexpr (BWD) {
        if (p.l == kL / 2) {
            GLR(kL / 2, 8, 1, false, p.colblocks);
            return;
        }
    }
    if constexpr (!BWD || V == 1) {
        if (p.chain) {
            GLR(kL, 8, 1, true, p.colblocks * p.nchunk);
            return;
        }
    }
    if constexpr (!BWD) {
        if (p.w == 8) {
            GLR(kL, 8, 1, false, p.colblocks);
            return;
        }
    }
    if (p.w == 4) GLR(kL, 4, 1, false, p.colblocks);
    else if (p.w == 2) GLR(kL, 2, 2, false, p.colblocks);
    else if (p.l == 1) GLR(1, 1, 4, false, p.colblocks);
    else GLR(kL, 1, 4, false, p.colblocks);
#undef GLR
}

// a launch has fewer than 2^32 threads: wide rows take several
template <class In, bool LAST>
int sum(const char* op, const In* part, uint64_t rows, uint32_t d, uint32_t row_blocks, double* out, float* dlam,
        const float* lam, float rate, hipStream_t s) {
    const uint32_t blocks = (uint32_t)ceil_div(d, 16), most = (1u << 21) / row_blocks;
    for (uint32_t first = 0; first < blocks; first += most) {
        const dim3 grid(blocks - first < most ? blocks - first : most, row_blocks);
        hipLaunchKernelGGL((glr_sum<In, LAST>), grid, dim3(1024), 0, s, part, rows, d, out, dlam, lam, rate, first);
        FHC_TRY(launched(op));
    }
    return 0;
}

template <bool BWD>
int run(const char* op, const Plan& p, GlrArgs& a, uint32_t dtype, void* ws, hipStream_t s) {
    if ((uint64_t)p.colblocks * p.nchunk >= 1ull << 31 || (uint64_t)a.b * p.groups >= 1ull << 31)
        return fail(-1, "%s: too many chunks", op);
    FHC_TRY(check_grid(op, (uint64_t)p.colblocks * (p.chain ? p.nchunk : 1), p.w == 8 ? 512 : 256));
    FHC_TRY(check_grid(op, ceil_div(p.words, 256), 256));
    a.groups = p.groups, a.nchunk = p.nchunk, a.colblocks = p.colblocks, a.nstates = p.nstates;
    a.spacing = p.spacing, a.straddles = p.straddles;
    char* w = static_cast<char*>(ws);
    if (p.chain) {
        a.agg = reinterpret_cast<uint64_t*>(w);
        a.group_maps = a.agg + (uint64_t)p.nchunk * a.b * a.d;
        a.heads = a.group_maps + ceil_div(p.nchunk, kGroup) * a.b * a.d;
        a.tickets = reinterpret_cast<uint32_t*>(a.agg + p.words);
        hipLaunchKernelGGL(glr_clear, dim3((uint32_t)ceil_div(p.words, 256)), dim3(256), 0, s, a.agg, p.words,
                           a.tickets, p.colblocks);
        FHC_TRY(launched(op));
    }
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (p.v == 2) launch<BWD, T, 2>(p, a, s);
        else launch<BWD, T, 1>(p, a, s);
    });
    return launched(op);
}

size_t workspace_of(const Plan& p, bool backward) {
    const size_t agg = (p.agg_bytes + 255) / 256 * 256;
    return backward ? agg + p.part_bytes + p.sum_bytes : agg;
}

}  // namespace
}  // namespace seq
}  // namespace fhc

using namespace fhc;
using namespace fhc::seq;

extern "C" size_t fhc_glr_states_bytes(const fhc_glr_desc* g) {
    return guard((size_t)0, [&]() -> size_t {
        clear_error();
        if (check_desc("glr_states_bytes", g) < 0) return 0;
        return (size_t)g->b * plan_of(g, true, 1, true).nstates * g->d * 4;
    });
}

extern "C" size_t fhc_glr_workspace_bytes(const fhc_glr_desc* g, int backward) {
    return guard((size_t)0, [&]() -> size_t {
        clear_error();
        if (check_desc("glr_workspace_bytes", g) < 0 || (uint64_t)g->b * g->d == 0) return 0;
        return workspace_of(plan_of(g, backward != 0, 1, true), backward != 0);
    });
}

extern "C" int fhc_glr_forward(const fhc_glr_desc* g, const fhc_seq* x, const fhc_seq* r, const fhc_seq* i,
                               const float* h0, const fhc_seq* y, float* ht, float* states, void* ws, size_t ws_bytes,
                               void* stream) {
    return guard(-3, [&]() -> int {
        clear_error();
        const char* op = "glr_forward";
        FHC_TRY(check_desc(op, g));
        if ((uint64_t)g->b * g->d == 0) return 0;
        FHC_TRY(check_seq(op, "x", x, g));
        FHC_TRY(check_seq(op, "r", r, g));
        FHC_TRY(check_seq(op, "i", i, g));
        FHC_TRY(check_out(op, "y", y, g));
        const Plan p = plan_for(g, false, {x, r, i, y});
        FHC_TRY(check_workspace(op, workspace_of(p, false), ws, ws_bytes));
        GlrArgs a{};
        a.x = col(x, g->dtype), a.r = col(r, g->dtype), a.i = col(i, g->dtype), a.y = col(y, g->dtype);
        a.lam = g->lam, a.lengths = g->lengths, a.h0 = h0, a.ht = ht, a.states = states;
        a.b = g->b, a.t = g->t, a.d = g->d, a.rate = g->rate;
        return run<false>(op, p, a, g->dtype, ws, (hipStream_t)stream);
    });
}

extern "C" int fhc_glr_backward(const fhc_glr_desc* g, const fhc_seq* x, const fhc_seq* r, const fhc_seq* i,
                                const float* states, const fhc_seq* dy, const float* dht, const fhc_seq* dx,
                                const fhc_seq* dr, const fhc_seq* di, float* dlam, float* dh0, void* ws,
                                size_t ws_bytes, void* stream) {
    return guard(-3, [&]() -> int {
        clear_error();
        const char* op = "glr_backward";
        FHC_TRY(check_desc(op, g));
        if (g->d == 0) return 0;
        if (!dlam) return fail(-1, "%s: null dlam", op);
        const hipStream_t s = (hipStream_t)stream;
        if (g->b == 0) {  // an empty sum
            if (!g->lam) return fail(-1, "%s: null lam", op);
            return sum<float, true>(op, nullptr, 0, g->d, 1, nullptr, dlam, g->lam, g->rate, s);
        }
        FHC_TRY(check_seq(op, "x", x, g));
        FHC_TRY(check_seq(op, "r", r, g));
        FHC_TRY(check_seq(op, "i", i, g));
        FHC_TRY(check_seq(op, "dy", dy, g));
        FHC_TRY(check_out(op, "dx", dx, g));
        FHC_TRY(check_out(op, "dr", dr, g));
        FHC_TRY(check_out(op, "di", di, g));
        if (g->t && !states) return fail(-1, "%s: null states", op);
        const Plan p = plan_for(g, true, {x, r, i, dy, dx, dr, di});
        FHC_TRY(check_workspace(op, workspace_of(p, true), ws, ws_bytes));
        GlrArgs a{};
        a.x = col(x, g->dtype), a.r = col(r, g->dtype), a.i = col(i, g->dtype), a.dy = col(dy, g->dtype);
        a.dx = col(dx, g->dtype), a.dr = col(dr, g->dtype), a.di = col(di, g->dtype);
        a.lam = g->lam, a.lengths = g->lengths, a.states = const_cast<float*>(states), a.dht = dht, a.dh0 = dh0;
        a.b = g->b, a.t = g->t, a.d = g->d, a.rate = g->rate;
        char* w = static_cast<char*>(ws) + (p.agg_bytes + 255) / 256 * 256;
        a.part = reinterpret_cast<float*>(w);
        FHC_TRY(run<true>(op, p, a, g->dtype, ws, s));
        if (!p.sum_bytes)
            return sum<float, true>(op, a.part, p.part_rows, g->d, 1, nullptr, dlam, g->lam, g->rate, s);
        double* sums = reinterpret_cast<double*>(w + p.part_bytes);
        FHC_TRY((sum<float, false>(op, a.part, p.part_rows, g->d, kSumRows, sums, nullptr, nullptr, 0.0f, s)));
        return sum<double, true>(op, sums, kSumRows, g->d, 1, nullptr, dlam, g->lam, g->rate, s);
    });
}
