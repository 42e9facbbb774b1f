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
//            the chip). Chunks form runs of kRun; the state that reaches a chunk is the one at the head of its run
//            folded through the maps of the run's chunks before it, and the run's last chunk publishes the next head:
//            a step of the serial chain is a run long, not a chunk.
// In the chain, chunks are taken in order by a ticket, so every chunk waited for is held by a workgroup that already
// runs and itself waits for earlier tickets only: every wait ends. What is published is one 8-byte word (A, S), or
// (0, state), written once and read by atomic accesses of the whole word, so no fence orders anything; its A is -1
// until then (decays are >= 0). Only the first chunk reads the initial state (it publishes it as the first head), so
// the last one may write the final state over it.
#include "seq_common.h"

namespace fhc {
namespace seq {
namespace {

struct Col {  // a sequence tensor in elements
    char* p;
    int64_t bs, ts;
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
    uint64_t* heads;  // and the first states of the runs [run][b * d]
    uint32_t* ticket;
    uint32_t b, t, d, groups, cols;  // groups: column groups of a sequence; cols = b * groups
    uint32_t nchunk, colblocks, nstates;
    float rate;
};

constexpr float kLog2e = 1.44269504088896340736f;

// e^-v, at most 1e37: its reciprocal and the product with it stay normal, so sigmoid(v) -> 0 and 1 - sigmoid(v) -> 1
// for the largest negative v (a NaN stays: fminf would drop it, the select keeps it)
__device__ __forceinline__ float exp_neg(float v) {
    const float e = __builtin_amdgcn_exp2f(v * -kLog2e);
    return e > 1e37f ? 1e37f : e;
}

// 1 - e^z for z <= 0. Near 0 the difference cancels, so -expm1's series there: 8 terms at z > -1/2 leave 2^-24 of it
__device__ __forceinline__ float one_minus_exp(float z, float ez) {
    float p = 1.0f / 40320.0f;
    p = __builtin_fmaf(p, z, 1.0f / 5040.0f);
    p = __builtin_fmaf(p, z, 1.0f / 720.0f);
    p = __builtin_fmaf(p, z, 1.0f / 120.0f);
    p = __builtin_fmaf(p, z, 1.0f / 24.0f);
    p = __builtin_fmaf(p, z, 1.0f / 6.0f);
    p = __builtin_fmaf(p, z, 0.5f);
    p = __builtin_fmaf(p, z, 1.0f);
    return z > -0.5f ? -z * p : 1.0f - ez;
}

struct Step {  // one step of one channel
    float a, sr, nr, si, ni, m, w, la, rm;  // nr, ni: 1 - sr, 1 - si; w = si * x; rm = 1 / m
};

// k = -rate * softplus(lam)
template <bool GRAD>
__device__ __forceinline__ Step step_of(float k, float x, float r, float i) {
    Step s;
    const float er = exp_neg(r), ei = exp_neg(i);
    s.sr = __builtin_amdgcn_rcpf(1.0f + er), s.si = __builtin_amdgcn_rcpf(1.0f + ei);
    s.la = k * s.sr;
    s.a = __builtin_amdgcn_exp2f(s.la * kLog2e);
    const float v = one_minus_exp(2.0f * s.la, s.a * s.a);
    s.w = s.si * x;
    if constexpr (GRAD) {
        s.nr = er * s.sr, s.ni = ei * s.si;
        // v is 0 where nothing decays (a = 1): no input either, and the gradient through m is taken at its limit 0 (a
        // subnormal v, which the instruction takes for 0, the same)
        s.rm = v >= 1.17549435e-38f ? __builtin_amdgcn_rsqf(v) : 0.0f * v;
        s.m = v * s.rm;
    } else {
        s.m = __builtin_amdgcn_sqrtf(v);
    }
    return s;
}

__device__ __forceinline__ float decay_rate(float rate, float lam) {
    // softplus without overflow: max(lam, 0) + log1p(e^-|lam|)
    const float sp = (lam > 0.0f ? lam : lam < 0.0f ? 0.0f : lam) + log1pf(expf(-fabsf(lam)));
    return -rate * sp;
}

__device__ __forceinline__ uint64_t word_of(float a, float s) {
    return (uint64_t)__builtin_bit_cast(uint32_t, a) | (uint64_t)__builtin_bit_cast(uint32_t, s) << 32;
}
constexpr uint64_t kUnpublished = 0xBF800000ull;  // (-1, 0)
__device__ __forceinline__ void publish(uint64_t* p, float a, float s) {
    __hip_atomic_store(p, word_of(a, s), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
constexpr uint32_t kRun = 16;  // chunks of a run

__global__ __launch_bounds__(256) void glr_clear(uint64_t* agg, uint64_t n, uint32_t* ticket) {
    const uint64_t k = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (k < n) agg[k] = kUnpublished;
    if (k == 0) *ticket = 0;
}

// The chain's search: the state that reaches this lane's columns of a chunk, `k` chunks after the head of its run.
// word(j) is the published map of the run's j-th chunk, head the run's first state. The W waves fetch the words
// together; the fold is in the chunks' order whatever the order of their arrival, so results repeat bit for bit.
template <int V, int W, class Word>
__device__ __forceinline__ void chain_find(uint32_t k, uint32_t tw, uint32_t slot, bool live, float2 (*lds)[64 * V],
                                           const uint64_t* head, Word word, float (&h)[V]) {
    auto wait_for = [](const uint64_t* p) {
        uint64_t w;
        do {
            w = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        } while ((uint32_t)w == (uint32_t)kUnpublished);
        return float2{__builtin_bit_cast(float, (uint32_t)w), __builtin_bit_cast(float, (uint32_t)(w >> 32))};
    };
    if (live) {
        for (uint32_t j = tw; j < k; j += W) {
#pragma unroll
            for (int v = 0; v < V; v++) lds[j][slot * V + v] = wait_for(word(j) + v);
        }
        if (tw == W - 1 && head) {  // the wave with the fewest words of chunks
#pragma unroll
            for (int v = 0; v < V; v++) lds[kRun - 1][slot * V + v] = wait_for(head + v);
        }
    }
    __syncthreads();
    if (!live) return;
    if (head) {
#pragma unroll
        for (int v = 0; v < V; v++) h[v] = lds[kRun - 1][slot * V + v].y;
    }
    for (uint32_t j = 0; j < k; j++) {
#pragma unroll
        for (int v = 0; v < V; v++) {
            const float2 q = lds[j][slot * V + v];
            h[v] = __builtin_fmaf(q.x, h[v], q.y);
        }
    }
}

// W waves of consecutive stretches x CW waves of column groups
template <class T, int V, int L, int W, int CW, bool CHAIN>
__global__ __launch_bounds__(64 * W * CW) void glr_fwd(GlrArgs g) {
    using R = typename T::Raw;
    constexpr int CL = W * L;
    __shared__ float2 maps[W > 1 ? W : 1][W > 1 ? CW * 64 * V : 1];
    __shared__ float2 far[CHAIN ? kRun : 1][CHAIN ? 64 * V : 1];
    static_assert(!CHAIN || CW == 1, "a chained chunk's columns are one wave wide");
    __shared__ uint32_t taken;
    uint32_t cb = blockIdx.x, chunk = 0;
    if constexpr (CHAIN) {
        if (threadIdx.x == 0) taken = atomicAdd(g.ticket, 1u);
        __syncthreads();
        chunk = taken / g.colblocks, cb = taken - chunk * g.colblocks;
    }
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t tw = W > 1 ? wave % W : 0, slot = (W > 1 ? wave / W : wave) * 64 + lane;
    const uint32_t col = cb * (CW * 64) + slot;
    const bool live = col < g.cols;
    const uint32_t b = live ? col / g.groups : 0, ch = live ? (col - b * g.groups) * V : 0;
    const uint64_t flat = (uint64_t)b * g.d + ch;
    const uint32_t n = live ? (g.lengths ? (uint32_t)min(max(g.lengths[b], 0), (int32_t)g.t) : g.t) : 0;

    float k[V], h[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
        k[v] = live ? decay_rate(g.rate, g.lam[ch + v]) : 0.0f;
        h[v] = live && g.h0 && (!CHAIN || chunk == 0) ? g.h0[flat + v] : 0.0f;
    }
    const R* xp = reinterpret_cast<const R*>(g.x.p) + b * g.x.bs + ch;
    const R* rp = reinterpret_cast<const R*>(g.r.p) + b * g.r.bs + ch;
    const R* ip = reinterpret_cast<const R*>(g.i.p) + b * g.i.bs + ch;
    R* yp = reinterpret_cast<R*>(g.y.p) + b * g.y.bs + ch;

    const uint32_t last = CHAIN ? chunk + 1 : g.nchunk;
    for (; chunk < last; chunk++) {
        const uint32_t t0 = chunk * CL + tw * L;
        R xr[L][V] = {}, rr[L][V] = {}, ir[L][V] = {};
#pragma unroll
        for (int l = 0; l < L; l++) {
            if (t0 + l < n) {
                load_raw<R, V, true>(xp + (int64_t)(t0 + l) * g.x.ts, xr[l]);
                load_raw<R, V, true>(rp + (int64_t)(t0 + l) * g.r.ts, rr[l]);
                load_raw<R, V, true>(ip + (int64_t)(t0 + l) * g.i.ts, ir[l]);
            }
        }
        float a[L][V], in[L][V], A[V], S[V];
#pragma unroll
        for (int v = 0; v < V; v++) A[v] = 1.0f, S[v] = 0.0f;
#pragma unroll
        for (int l = 0; l < L; l++) {
            const bool on = t0 + l < n;
#pragma unroll
            for (int v = 0; v < V; v++) {
                const Step s = step_of<false>(k[v], widen(T{}, xr[l][v]), widen(T{}, rr[l][v]), widen(T{}, ir[l][v]));
                a[l][v] = on ? s.a : 1.0f, in[l][v] = on ? s.m * s.w : 0.0f;
                if constexpr (W > 1) {
                    S[v] = __builtin_fmaf(a[l][v], S[v], in[l][v]);
                    A[v] *= a[l][v];
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
            for (int v = 0; v < V; v++) {
                ta[v] = 1.0f, ts[v] = 0.0f;
#pragma unroll
                for (int w = 0; w < W; w++) {
                    if (w == (int)tw) pa[v] = ta[v], ps[v] = ts[v];
                    const float2 q = maps[w][slot * V + v];
                    ts[v] = __builtin_fmaf(q.x, ts[v], q.y);
                    ta[v] *= q.x;
                }
            }
            if constexpr (CHAIN) {
                const uint64_t flats = (uint64_t)g.b * g.d;
                const uint32_t run = chunk / kRun, k = chunk - run * kRun;
                if (tw == 0 && live && k + 1 < kRun && chunk + 1 < g.nchunk) {
#pragma unroll
                    for (int v = 0; v < V; v++) {
                        publish(g.agg + chunk * flats + flat + v, ta[v], ts[v]);
                        if (chunk == 0) publish(g.heads + flat + v, 0.0f, h[v]);
                    }
                }
                chain_find<V, W>(
                    k, tw, slot, live, far, chunk ? g.heads + run * flats + flat : nullptr,
                    [&](uint32_t j) { return g.agg + (uint64_t)(run * kRun + j) * flats + flat; }, h);
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
        if (live && g.states && tw == 0 && t0 < g.t) {
#pragma unroll
            for (int v = 0; v < V; v++) g.states[((uint64_t)b * g.nstates + chunk) * g.d + ch + v] = h[v];
        }
#pragma unroll
        for (int l = 0; l < L; l++) {
            R out[V];
#pragma unroll
            for (int v = 0; v < V; v++) {
                h[v] = __builtin_fmaf(a[l][v], h[v], in[l][v]);
                out[v] = narrow(T{}, t0 + l < n ? h[v] : 0.0f);
            }
            if (live && t0 + l < g.t) store_raw<R, V, true>(yp + (int64_t)(t0 + l) * g.y.ts, out);
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

template <class T, int V, int L, int W, int CW, bool CHAIN>
__global__ __launch_bounds__(64 * W * CW) void glr_bwd(GlrArgs g) {
    using R = typename T::Raw;
    constexpr int CL = W * L;
    __shared__ float2 maps[W > 1 ? W : 1][W > 1 ? CW * 64 * V : 1];  // (A, S) forward
    __shared__ float back[W > 1 ? W : 1][W > 1 ? CW * 64 * V : 1];   // the R of c -> A c + R
    __shared__ float2 far[CHAIN ? kRun : 1][CHAIN ? 64 * V : 1];
    static_assert(!CHAIN || CW == 1, "a chained chunk's columns are one wave wide");
    __shared__ uint32_t taken;
    uint32_t cb = blockIdx.x, done = 0;  // chunks go from the last to the first; done: those already passed
    if constexpr (CHAIN) {
        if (threadIdx.x == 0) taken = atomicAdd(g.ticket, 1u);
        __syncthreads();
        done = taken / g.colblocks, cb = taken - done * g.colblocks;
    }
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t tw = W > 1 ? wave % W : 0, slot = (W > 1 ? wave / W : wave) * 64 + lane;
    const uint32_t col = cb * (CW * 64) + slot;
    const bool live = col < g.cols;
    const uint32_t b = live ? col / g.groups : 0, ch = live ? (col - b * g.groups) * V : 0;
    const uint64_t flat = (uint64_t)b * g.d + ch;
    const uint32_t n = live ? (g.lengths ? (uint32_t)min(max(g.lengths[b], 0), (int32_t)g.t) : g.t) : 0;

    float k[V], c[V], lam_sum[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
        k[v] = live ? decay_rate(g.rate, g.lam[ch + v]) : 0.0f;
        c[v] = live && g.dht && (!CHAIN || done == 0) ? g.dht[flat + v] : 0.0f;
        lam_sum[v] = 0.0f;
    }
    const R* xp = reinterpret_cast<const R*>(g.x.p) + b * g.x.bs + ch;
    const R* rp = reinterpret_cast<const R*>(g.r.p) + b * g.r.bs + ch;
    const R* ip = reinterpret_cast<const R*>(g.i.p) + b * g.i.bs + ch;
    const R* dyp = reinterpret_cast<const R*>(g.dy.p) + b * g.dy.bs + ch;
    R* dxp = reinterpret_cast<R*>(g.dx.p) + b * g.dx.bs + ch;
    R* drp = reinterpret_cast<R*>(g.dr.p) + b * g.dr.bs + ch;
    R* dip = reinterpret_cast<R*>(g.di.p) + b * g.di.bs + ch;

    const uint32_t last = CHAIN ? done + 1 : g.nchunk;
    for (; done < last; done++) {
        const uint32_t chunk = g.nchunk - 1 - done, t0 = chunk * CL + tw * L;
        R xr[L][V] = {}, rr[L][V] = {}, ir[L][V] = {}, gr[L][V] = {};
        float h[V];
#pragma unroll
        for (int v = 0; v < V; v++)
            h[v] = live && chunk < g.nstates ? g.states[((uint64_t)b * g.nstates + chunk) * g.d + ch + v] : 0.0f;
#pragma unroll
        for (int l = 0; l < L; l++) {
            if (t0 + l < n) {
                load_raw<R, V, true>(xp + (int64_t)(t0 + l) * g.x.ts, xr[l]);
                load_raw<R, V, true>(rp + (int64_t)(t0 + l) * g.r.ts, rr[l]);
                load_raw<R, V, true>(ip + (int64_t)(t0 + l) * g.i.ts, ir[l]);
                load_raw<R, V, true>(dyp + (int64_t)(t0 + l) * g.dy.ts, gr[l]);
            }
        }
        Step s[L][V];
        float dy[L][V], A[V], S[V], B[V];
#pragma unroll
        for (int v = 0; v < V; v++) A[v] = 1.0f, S[v] = 0.0f, B[v] = 0.0f;
#pragma unroll
        for (int l = 0; l < L; l++) {
            const bool on = t0 + l < n;
#pragma unroll
            for (int v = 0; v < V; v++) {
                s[l][v] = step_of<true>(k[v], widen(T{}, xr[l][v]), widen(T{}, rr[l][v]), widen(T{}, ir[l][v]));
                dy[l][v] = on ? widen(T{}, gr[l][v]) : 0.0f;
                if (!on) s[l][v].a = 1.0f, s[l][v].m = 0.0f, s[l][v].w = 0.0f;
                if constexpr (W > 1) {
                    S[v] = __builtin_fmaf(s[l][v].a, S[v], s[l][v].m * s[l][v].w);
                    A[v] *= s[l][v].a;
                    B[v] = __builtin_fmaf(A[v], dy[l][v], B[v]);  // dy_l reaches the front through a_1 .. a_l
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
            for (int v = 0; v < V; v++) {
#pragma unroll
                for (int w = 0; w < W; w++) {  // the state that reaches the stretch
                    const float2 q = maps[w][slot * V + v];
                    if (w < (int)tw) h[v] = __builtin_fmaf(q.x, h[v], q.y);
                }
                ta[v] = 1.0f, ts[v] = 0.0f;
#pragma unroll
                for (int w = W - 1; w >= 0; w--) {
                    if (w == (int)tw) pa[v] = ta[v], ps[v] = ts[v];
                    const float qa = maps[w][slot * V + v].x;
                    ts[v] = __builtin_fmaf(qa, ts[v], back[w][slot * V + v]);
                    ta[v] *= qa;
                }
            }
            if constexpr (CHAIN) {
                const uint64_t flats = (uint64_t)g.b * g.d;
                const uint32_t run = done / kRun, k = done - run * kRun;
                if (tw == 0 && live && k + 1 < kRun && chunk > 0) {
#pragma unroll
                    for (int v = 0; v < V; v++) {
                        publish(g.agg + done * flats + flat + v, ta[v], ts[v]);
                        if (done == 0) publish(g.heads + flat + v, 0.0f, c[v]);
                    }
                }
                chain_find<V, W>(
                    k, tw, slot, live, far, done ? g.heads + run * flats + flat : nullptr,
                    [&](uint32_t j) { return g.agg + (uint64_t)(run * kRun + j) * flats + flat; }, c);
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
        float hp[L][V];  // the state before each step
#pragma unroll
        for (int l = 0; l < L; l++) {
#pragma unroll
            for (int v = 0; v < V; v++) {
                hp[l][v] = h[v];
                h[v] = __builtin_fmaf(s[l][v].a, h[v], s[l][v].m * s[l][v].w);
            }
        }
#pragma unroll
        for (int l = L - 1; l >= 0; l--) {
            const bool on = t0 + l < n;
            R ox[V], orr[V], oi[V];
#pragma unroll
            for (int v = 0; v < V; v++) {
                const Step& q = s[l][v];
                const float gt = dy[l][v] + c[v];
                c[v] = q.a * gt;
                // d/d(log a): a h_(t-1) from the decay, -(a^2 / m) w from the input's normalisation
                const float dla = c[v] * (hp[l][v] - q.a * q.rm * q.w);
                const float gm = gt * q.m;
                ox[v] = narrow(T{}, on ? gm * q.si : 0.0f);
                orr[v] = narrow(T{}, on ? dla * q.la * q.nr : 0.0f);
                oi[v] = narrow(T{}, on ? gm * q.w * q.ni : 0.0f);
                lam_sum[v] += on ? dla * q.sr : 0.0f;
            }
            if (live && t0 + l < g.t) {
                store_raw<R, V, true>(dxp + (int64_t)(t0 + l) * g.dx.ts, ox);
                store_raw<R, V, true>(drp + (int64_t)(t0 + l) * g.dr.ts, orr);
                store_raw<R, V, true>(dip + (int64_t)(t0 + l) * g.di.ts, oi);
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

// Column sums of the partial rows: 64 columns x 16 row lanes a workgroup, rows y, y + gridDim.y * 16, ...; a second
// launch with one row block finishes. In f64: millions of terms of either sign meet here.
template <class In, bool LAST>
__global__ __launch_bounds__(1024) void glr_sum(const In* part, uint64_t rows, uint32_t d, double* out, float* dlam,
                                                const float* lam, float rate) {
    __shared__ double s[16][64];
    const uint32_t ch = blockIdx.x * 64 + (threadIdx.x & 63), y = threadIdx.x >> 6;
    double acc = 0.0;
    if (ch < d) {
#pragma unroll 4
        for (uint64_t r = (uint64_t)blockIdx.y * 16 + y; r < rows; r += (uint64_t)gridDim.y * 16)
            acc += (double)part[r * d + ch];
    }
    s[y][threadIdx.x & 63] = acc;
    __syncthreads();
    if (y == 0 && ch < d) {
#pragma unroll
        for (int k = 1; k < 16; k++) acc += s[k][threadIdx.x];
        if constexpr (LAST) {
            const float e = expf(-fabsf(lam[ch]));  // d softplus / d lam = sigmoid(lam)
            const float sg = (lam[ch] >= 0.0f ? 1.0f : e) / (1.0f + e);
            dlam[ch] = (float)(acc * -(double)rate * (double)sg);
        } else {
            out[(uint64_t)blockIdx.y * d + ch] = acc;
        }
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------

constexpr int kL = 8;         // steps a lane holds
constexpr int kW = 8;         // waves of a chunk, where a chunk has more than one
constexpr int kChunk = kL * kW;
constexpr uint32_t kSumRows = 64;  // row blocks of the first sum

struct Plan {
    bool split, chain;  // split: chunks of kW waves
    uint32_t v, groups, cols, chunk, nchunk, colblocks, nstates;
    uint64_t words;  // of the chain: maps, then heads
    size_t agg_bytes, part_bytes, sum_bytes;
};

// One wave per column group walks kL steps at a time where that alone fills the chip or there is little to split;
// else kW waves share a chunk, and chunks are chained where the columns give fewer than two workgroups a CU. v: the
// channels a lane takes.
Plan plan_of(const fhc_glr_desc* g, uint32_t v) {
    Plan p{};
    p.v = v;
    p.groups = g->d / v;
    p.cols = g->b * p.groups;
    const uint64_t flat = (uint64_t)g->b * g->d;
    p.split = g->t > 2 * kL && flat < (1u << 19);
    p.chunk = p.split ? kChunk : kL;
    p.nchunk = (uint32_t)(g->t ? ceil_div(g->t, p.chunk) : 1);
    p.nstates = (uint32_t)ceil_div(g->t, p.chunk);
    p.colblocks = (uint32_t)ceil_div(p.cols, p.split ? 64 : 256);
    p.chain = p.split && p.nchunk > 1 && flat < (1u << 16);
    p.words = p.chain ? (p.nchunk + ceil_div(p.nchunk, kRun)) * flat : 0;
    p.agg_bytes = p.chain ? p.words * 8 + 256 : 0;
    p.part_bytes = (size_t)ceil_div((p.chain ? p.nchunk : 1) * flat * 4, 256) * 256;
    p.sum_bytes = (size_t)kSumRows * g->d * 8;
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
    if (g->t > 1 && (uint64_t)std::llabs(s->ts) < g->d) return fail(-1, "%s: %s: steps %lld apart overlap", op, name, (long long)s->ts);
    if (g->b > 1 && (uint64_t)std::llabs(s->bs) < g->d) return fail(-1, "%s: %s: sequences %lld apart overlap", op, name, (long long)s->bs);
    return 0;
}

Col col(const fhc_seq* s) { return Col{static_cast<char*>(s->p), s->bs, s->ts}; }

// pairs of channels as one load where every tensor allows it
bool pairs(const fhc_glr_desc* g, std::initializer_list<const fhc_seq*> all) {
    if (g->d % 2) return false;
    for (const fhc_seq* s : all)
        if ((g->b > 1 && s->bs % 2) || (g->t > 1 && s->ts % 2) || !aligned(s->p, 2 * elem_bytes(g->dtype)))
            return false;
    return true;
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
    if (p.chain) GLR(kL, kW, 1, true, p.colblocks * p.nchunk);
    else if (p.split) GLR(kL, kW, 1, false, p.colblocks);
    else GLR(kL, 1, 4, false, p.colblocks);
#undef GLR
}

template <bool BWD>
int run(const char* op, const Plan& p, GlrArgs& a, uint32_t dtype, void* ws, hipStream_t s) {
    if ((uint64_t)p.colblocks * p.nchunk >= 1ull << 31) return fail(-1, "%s: too many chunks", op);
    a.groups = p.groups, a.cols = p.cols, a.nchunk = p.nchunk, a.colblocks = p.colblocks, a.nstates = p.nstates;
    char* w = static_cast<char*>(ws);
    if (p.chain) {
        a.ticket = reinterpret_cast<uint32_t*>(w);
        a.agg = reinterpret_cast<uint64_t*>(w + 256);
        a.heads = a.agg + (uint64_t)p.nchunk * a.b * a.d;
        hipLaunchKernelGGL(glr_clear, dim3((uint32_t)ceil_div(p.words, 256)), dim3(256), 0, s, a.agg, p.words, a.ticket);
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
        return (size_t)g->b * plan_of(g, 1).nstates * g->d * 4;
    });
}

extern "C" size_t fhc_glr_workspace_bytes(const fhc_glr_desc* g, int backward) {
    return guard((size_t)0, [&]() -> size_t {
        clear_error();
        if (check_desc("glr_workspace_bytes", g) < 0 || (uint64_t)g->b * g->d == 0) return 0;
        return workspace_of(plan_of(g, 1), backward != 0);
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
        const Plan p = plan_of(g, pairs(g, {x, r, i, y}) ? 2 : 1);
        FHC_TRY(check_workspace(op, workspace_of(p, false), ws, ws_bytes));
        GlrArgs a{};
        a.x = col(x), a.r = col(r), a.i = col(i), a.y = col(y);
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
        Plan p = plan_of(g, 1);
        const uint32_t dblocks = (uint32_t)ceil_div(g->d, 64);
        if (g->b == 0) {  // an empty sum
            if (!g->lam) return fail(-1, "%s: null lam", op);
            hipLaunchKernelGGL((glr_sum<float, true>), dim3(dblocks), dim3(1024), 0, s, (const float*)nullptr,
                               (uint64_t)0, g->d, (double*)nullptr, dlam, g->lam, g->rate);
            return launched(op);
        }
        FHC_TRY(check_seq(op, "x", x, g));
        FHC_TRY(check_seq(op, "r", r, g));
        FHC_TRY(check_seq(op, "i", i, g));
        FHC_TRY(check_seq(op, "dy", dy, g));
        FHC_TRY(check_out(op, "dx", dx, g));
        FHC_TRY(check_out(op, "dr", dr, g));
        FHC_TRY(check_out(op, "di", di, g));
        if (g->t && !states) return fail(-1, "%s: null states", op);
        if (pairs(g, {x, r, i, dy, dx, dr, di})) p = plan_of(g, 2);
        FHC_TRY(check_workspace(op, workspace_of(p, true), ws, ws_bytes));
        GlrArgs a{};
        a.x = col(x), a.r = col(r), a.i = col(i), a.dy = col(dy), a.dx = col(dx), a.dr = col(dr), a.di = col(di);
        a.lam = g->lam, a.lengths = g->lengths, a.states = const_cast<float*>(states), a.dht = dht, a.dh0 = dh0;
        a.b = g->b, a.t = g->t, a.d = g->d, a.rate = g->rate;
        char* w = static_cast<char*>(ws) + (p.agg_bytes + 255) / 256 * 256;
        a.part = reinterpret_cast<float*>(w);
        FHC_TRY(run<true>(op, p, a, g->dtype, ws, s));
        const uint64_t rows = (uint64_t)(p.chain ? p.nchunk : 1) * g->b;
        if (rows <= 512) {
            hipLaunchKernelGGL((glr_sum<float, true>), dim3(dblocks), dim3(1024), 0, s, a.part, rows, g->d,
                               (double*)nullptr, dlam, g->lam, g->rate);
            return launched(op);
        }
        double* sums = reinterpret_cast<double*>(w + p.part_bytes);
        hipLaunchKernelGGL((glr_sum<float, false>), dim3(dblocks, kSumRows), dim3(1024), 0, s, a.part, rows, g->d, sums,
                           (float*)nullptr, (const float*)nullptr, 0.0f);
        FHC_TRY(launched(op));
        hipLaunchKernelGGL((glr_sum<double, true>), dim3(dblocks), dim3(1024), 0, s, sums, (uint64_t)kSumRows, g->d,
                           (double*)nullptr, dlam, g->lam, g->rate);
        return launched(op);
    });
}
