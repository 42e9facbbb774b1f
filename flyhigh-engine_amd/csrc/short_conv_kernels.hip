// The short causal convolution along a sequence (include/fhc_seq.h), forward and backward.
//
// A thread has V adjacent channels of one sequence and walks a chunk of steps with the last k - 1 inputs in registers,
// so every input is read once, bar the k - 1 rows in front of a chunk (which the caches hold: a workgroup has
// neighbouring chunks of the same channels). Lanes run over channels; a map of few channels gives a wave's other lanes
// further chunks or sequences. The first chunk of a sequence also moves the state on: it alone reads the old one, so the
// new one may lie over it.
//
// Backward, with dv = dy act'(v) (v computed again) and e the state's rows and then the sequence's:
//     de_i = sum over j of w[j] dv_(i - j),   dw[j] = sum over t of dv_t e_(t + j),   dbias = sum over t of dv_t
// A thread walks its chunk and k - 1 steps more, whose dv it needs for its last inputs, and adds its weights' gradients
// in registers, over 256 steps at most; a workgroup's chunks of the same channels are added in LDS and the workgroups' sums
// in f64 by column_sums, all in a fixed order.
#include "seq_args.h"

namespace fhc {
namespace seq {
namespace {

template <class R>
struct ConvArgs {
    Seq<R> x, y, dy, dx;
    const R *w, *bias, *state, *dend;
    R *end, *dstate;
    float* part;  // [workgroup rows][d * k + d]
    const int32_t* lengths;
    uint32_t b, t, d, groups;       // groups: threads that a row of channels takes
    uint32_t lanes, colblocks;      // log2 of the threads of a workgroup side by side; their blocks
    uint32_t chunks, steps, items;  // chunks of `steps` a sequence; b * chunks
    uint32_t walks;                 // backward: workgroups that a column block's items are dealt to
    bool silu;
    bool whole;  // the last thread of a row takes its last V channels, some of them twice: the same bytes are stored twice
};

constexpr uint32_t kThreads = 256;

// V elements at p, `valid` of them there
template <class R, int V>
__device__ __forceinline__ void load_v(const R* p, int valid, R (&o)[V]) {
    if (valid >= V) {
        load_raw<R, V, false>(p, o);
    } else {
#pragma unroll
        for (int v = 0; v < V; v++) o[v] = v < valid ? p[v] : R(0);
    }
}
template <class R, int V>
__device__ __forceinline__ void store_v(R* p, int valid, const R (&o)[V]) {
    if (valid >= V) {
        store_raw<R, V, false>(p, o);
    } else {
#pragma unroll
        for (int v = 0; v < V; v++)
            if (v < valid) p[v] = o[v];
    }
}

// A thread's channels and weights.
template <class T, int K, int V>
struct Taps {
    using R = typename T::Raw;
    float w[K][V], bias[V];
    __device__ __forceinline__ Taps(const ConvArgs<R>& g, uint32_t ch, int valid) {
        R q[K * V];
#pragma unroll
        for (int k = 0; k < K; k++) {
            R part[V];
            load_v<R, V>(g.w + (uint64_t)ch * K + k * V, valid * K - k * V, part);
#pragma unroll
            for (int v = 0; v < V; v++) q[k * V + v] = part[v];
        }
        R z[V];
#pragma unroll
        for (int v = 0; v < V; v++) z[v] = R(0);
        if (g.bias) load_v<R, V>(g.bias + ch, valid, z);
#pragma unroll
        for (int v = 0; v < V; v++) {
            bias[v] = widen(T{}, z[v]);
#pragma unroll
            for (int k = 0; k < K; k++) w[k][v] = widen(T{}, q[v * K + k]);
        }
    }
};

// Which channels and chunk a thread has: item `item` of column block `cb`.
template <int V>
struct Place {
    uint32_t ch, b, t0, n;
    int valid, twice;  // channels there; those of them, from the first on, that the lane before has too
    bool live;
    template <class R>
    __device__ __forceinline__ Place(const ConvArgs<R>& g, uint32_t cb, uint32_t item) {
        const uint32_t cg = (cb << g.lanes) + (threadIdx.x & ((1u << g.lanes) - 1));
        live = cg < g.groups && item < g.items;
        ch = live ? cg * V : 0, twice = 0;
        if (g.whole && live && ch + V > g.d) twice = ch + V - g.d, ch = g.d - V;
        valid = live ? min(V, (int)(g.d - ch)) : 0;
        const uint32_t k = live ? item : 0;
        b = k / g.chunks;
        t0 = (k - b * g.chunks) * g.steps;
        n = g.lengths ? (uint32_t)min(max(g.lengths[b], 0), (int32_t)g.t) : g.t;
    }
};

// The k - 1 rows in front of step t0, as values.
template <class T, int K, int V>
__device__ __forceinline__ void rows_before(const ConvArgs<typename T::Raw>& g, const Place<V>& p, float (&win)[K][V]) {
    using R = typename T::Raw;
#pragma unroll
    for (int j = 0; j < K - 1; j++) {
        R q[V];
#pragma unroll
        for (int v = 0; v < V; v++) q[v] = R(0);
        if (p.t0 == 0) {
            if (g.state) load_v<R, V>(g.state + ((uint64_t)p.b * (K - 1) + j) * g.d + p.ch, p.valid, q);
        } else if (p.t0 - (K - 1) + j < p.n) {
            load_v<R, V>(g.x.at(p.b, (int64_t)p.t0 - (K - 1) + j) + p.ch, p.valid, q);
        }
#pragma unroll
        for (int v = 0; v < V; v++) win[j][v] = widen(T{}, q[v]);
    }
}

// What bounds it (MI355X): HBM. 4 x 4096 x 4096, 4 taps: bf16 53 us, 5.1 TB/s of the 5.2 that a large copy reaches; f32 107,
// 5.0 TB/s.
template <class T, int K, int V>
__global__ __launch_bounds__(kThreads) void short_conv_fwd(ConvArgs<typename T::Raw> g) {
    using R = typename T::Raw;
    constexpr int U = 4;  // steps whose loads are under way together
    const uint32_t ib = blockIdx.x / g.colblocks, cb = blockIdx.x - ib * g.colblocks;
    const Place<V> p(g, cb, (ib << (8 - g.lanes)) + (threadIdx.x >> g.lanes));
    if (!p.live) return;
    const Taps<T, K, V> taps(g, p.ch, p.valid);
    float win[K][V];
    rows_before<T, K, V>(g, p, win);
    if (p.t0 == 0 && g.end) {  // the state's rows are in registers: the new ones may lie over them
        R q[K - 1][V];
#pragma unroll
        for (int j = 0; j < K - 1; j++) {
            const uint32_t i = p.n + j;
            if (i >= K - 1) {
                load_v<R, V>(g.x.at(p.b, i - (K - 1)) + p.ch, p.valid, q[j]);
            } else {
#pragma unroll
                for (int v = 0; v < V; v++) {
                    float f = win[0][v];
#pragma unroll
                    for (int m = 1; m < K - 1; m++) f = i == (uint32_t)m ? win[m][v] : f;
                    q[j][v] = narrow(T{}, f);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < K - 1; j++)
            store_v<R, V>(g.end + ((uint64_t)p.b * (K - 1) + j) * g.d + p.ch, p.valid, q[j]);
    }
    const uint32_t t1 = min(p.t0 + g.steps, g.t), last = min(t1, p.n);
    const R* px = g.x.at(p.b, p.t0) + p.ch;
    R* py = g.y.at(p.b, p.t0) + p.ch;
    for (uint32_t t = p.t0; t < t1; t += U) {
        R in[U][V];
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (t + u < last) load_v<R, V>(px + u * g.x.ts, p.valid, in[u]);
            else
#pragma unroll
                for (int v = 0; v < V; v++) in[u][v] = R(0);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            R out[V];
#pragma unroll
            for (int v = 0; v < V; v++) {
                win[K - 1][v] = widen(T{}, in[u][v]);
                float s = taps.bias[v];
#pragma unroll
                for (int k = 0; k < K; k++) s = __builtin_fmaf(taps.w[k][v], win[k][v], s);
                if (g.silu) s *= sigmoid1(s);
                out[v] = t + u < last ? narrow(T{}, s) : R(0);
#pragma unroll
                for (int k = 0; k < K - 1; k++) win[k][v] = win[k + 1][v];
            }
            if (t + u < t1) store_v<R, V>(py + u * g.y.ts, p.valid, out);
        }
        px += U * g.x.ts, py += U * g.y.ts;
    }
}

// What bounds it (MI355X): HBM beside the vector units, at four waves a SIMD. 4 x 4096 x 4096 bf16, 4 taps, 101 us for 403 MB,
// 4.0 TB/s, and 5 for the closing sums; f32 185 with them, 4.3 TB/s.
template <class T, int K, int V>
__global__ __launch_bounds__(kThreads) void short_conv_bwd(ConvArgs<typename T::Raw> g) {
    using R = typename T::Raw;
    constexpr int U = 4;
    __shared__ float sums[V][kThreads];
    const uint32_t walk = blockIdx.x / g.colblocks, cb = blockIdx.x - walk * g.colblocks;
    const uint32_t rows = kThreads >> g.lanes, row = threadIdx.x >> g.lanes;
    float dw[K][V], db[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
        db[v] = 0.0f;
#pragma unroll
        for (int k = 0; k < K; k++) dw[k][v] = 0.0f;
    }
    const Place<V> mine(g, cb, 0);  // the channels are the same for every item
    const Taps<T, K, V> taps(g, mine.ch, mine.valid);
    for (uint64_t item = (uint64_t)walk * rows + row; item < g.items; item += (uint64_t)g.walks * rows) {
        const Place<V> p(g, cb, (uint32_t)item);
        if (!p.live) break;
        float win[K][V], dv[K][V];  // e_t .. e_(t + k - 1); dv_(t - k + 1) .. dv_t
        rows_before<T, K, V>(g, p, win);
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int v = 0; v < V; v++) dv[k][v] = 0.0f;
        const uint32_t t1 = min(p.t0 + g.steps, g.t), most = t1 + K - 1, there = min(most, p.n);
        const R *px = g.x.at(p.b, p.t0) + p.ch, *py = g.dy.at(p.b, p.t0) + p.ch;
        R* pd = g.dx.at(p.b, p.t0) + p.ch;
        // M steps' rows from step i on; those past the length or the chunk as zeros
        auto load = [&](auto m, uint32_t i, R(*in)[V], R(*up)[V]) {
            constexpr int M = m;
            if (i + M <= there && p.valid >= V) {
#pragma unroll
                for (int u = 0; u < M; u++) {
                    load_raw<R, V, false>(px + u * g.x.ts, in[u]);
                    load_raw<R, V, false>(py + u * g.dy.ts, up[u]);
                }
            } else {
#pragma unroll
                for (int u = 0; u < M; u++) {
#pragma unroll
                    for (int v = 0; v < V; v++) in[u][v] = up[u][v] = R(0);
                    if (i + u < there) {
                        load_v<R, V>(px + u * g.x.ts, p.valid, in[u]);
                        load_v<R, V>(py + u * g.dy.ts, p.valid, up[u]);
                    }
                }
            }
            px += M * g.x.ts, py += M * g.dy.ts;
        };
        // Step i: dv_i, the weights' gradients (INNER: certainly a step of this chunk inside the length), and de_i.
        auto step = [&](auto inner, uint32_t i, const R(&in)[V], const R(&up)[V], float(&de)[V]) {
            constexpr bool INNER = inner;
            const bool own = INNER || (i < t1 && i < p.n);  // steps behind are the next chunk's, and so their terms
#pragma unroll
            for (int v = 0; v < V; v++) {
                win[K - 1][v] = widen(T{}, in[v]);
                float s = taps.bias[v], slope = 1.0f, value;
#pragma unroll
                for (int k = 0; k < K; k++) s = __builtin_fmaf(taps.w[k][v], win[k][v], s);
                if (g.silu) silu_grad(s, value, slope);
                const float q = INNER || i < p.n ? widen(T{}, up[v]) * slope : 0.0f;
                dv[K - 1][v] = q;
                if (own) {
                    db[v] += q;
#pragma unroll
                    for (int k = 0; k < K; k++) dw[k][v] = __builtin_fmaf(q, win[k][v], dw[k][v]);
                }
                de[v] = 0.0f;
#pragma unroll
                for (int k = 0; k < K; k++) de[v] = __builtin_fmaf(taps.w[k][v], dv[K - 1 - k][v], de[v]);
#pragma unroll
                for (int k = 0; k < K - 1; k++) win[k][v] = win[k + 1][v], dv[k][v] = dv[k + 1][v];
            }
            if (!INNER && i >= p.n && i < p.n + K - 1 && g.dend) {  // e_i is also a row of the state that is left
                R end[V];
                load_v<R, V>(g.dend + ((uint64_t)p.b * (K - 1) + (i - p.n)) * g.d + p.ch, p.valid, end);
#pragma unroll
                for (int v = 0; v < V; v++) de[v] += widen(T{}, end[v]);
            }
        };
        {  // the first k - 1 steps complete rows in front of the chunk: the state's, or the chunk's before
            R in[K - 1][V], up[K - 1][V], out[V];
            load(std::integral_constant<int, K - 1>{}, p.t0, in, up);
#pragma unroll
            for (int u = 0; u < K - 1; u++) {
                float de[V];
                step(std::false_type{}, p.t0 + u, in[u], up[u], de);
#pragma unroll
                for (int v = 0; v < V; v++) out[v] = narrow(T{}, de[v]);
                if (p.t0 == 0 && g.dstate)
                    store_v<R, V>(g.dstate + ((uint64_t)p.b * (K - 1) + u) * g.d + p.ch, p.valid, out);
            }
        }
        R in[U][V], up[U][V];
        const std::integral_constant<int, U> block{};
        load(block, p.t0 + K - 1, in, up);
        for (uint32_t i = p.t0 + K - 1; i < most; i += U) {
            R now[U][V], dnow[U][V];
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int v = 0; v < V; v++) now[u][v] = in[u][v], dnow[u][v] = up[u][v];
            if (i + U < most) load(block, i + U, in, up);
            const bool inner = i + U <= min(t1, p.n) && p.valid >= V && g.dx.p;
            if (inner) {
#pragma unroll
                for (int u = 0; u < U; u++) {
                    float de[V];
                    R out[V];
                    step(std::true_type{}, i + u, now[u], dnow[u], de);
#pragma unroll
                    for (int v = 0; v < V; v++) out[v] = narrow(T{}, de[v]);
                    store_raw<R, V, false>(pd + u * g.dx.ts, out);
                }
            } else {
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (i + u >= most) break;
                    float de[V];
                    R out[V];
                    step(std::false_type{}, i + u, now[u], dnow[u], de);
#pragma unroll
                    for (int v = 0; v < V; v++) out[v] = i + u - (K - 1) < p.n ? narrow(T{}, de[v]) : R(0);
                    if (g.dx.p) store_v<R, V>(pd + u * g.dx.ts, p.valid, out);
                }
            }
            pd += U * g.dx.ts;
        }
    }
    float* part = g.part + (uint64_t)walk * g.d * (K + 1);
#pragma unroll
    for (int k = 0; k <= K; k++) {
#pragma unroll
        for (int v = 0; v < V; v++) sums[v][threadIdx.x] = k < K ? dw[k < K ? k : 0][v] : db[v];
        __syncthreads();
        if (row == 0) {
#pragma unroll
            for (int v = 0; v < V; v++) {
                float s = 0.0f;
                for (uint32_t r = 0; r < rows; r++) s += sums[v][(r << g.lanes) + threadIdx.x];
                if (v < mine.valid && v >= mine.twice) part[k < K ? (uint64_t)(mine.ch + v) * K + k : (uint64_t)g.d * K + mine.ch + v] = s;
            }
        }
        __syncthreads();
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------

// Channels of a thread: 16 bytes forward (8-byte loads take 72 us where these take 58, 4 x 4096 x 4096 bf16); backward two
// channels, since their windows and sums decide how many waves a SIMD has (4 with two, 2 with eight: 108 us and 320).
constexpr int kBackV = 2;
constexpr uint32_t kForwardV(uint32_t dtype) { return dtype == FHC_F32 ? 4 : 8; }
constexpr uint32_t kMostItems = 8;  // of up to 32 steps each; the sums over workgroups are f64
struct Plan {
    uint32_t v, groups, lanes, colblocks, chunks, steps, items, blocks, walks;
};
Plan plan_of(const fhc_short_conv_desc* g, bool backward) {
    Plan p{};
    p.v = backward ? kBackV : kForwardV(g->dtype);
    p.groups = (uint32_t)ceil_div(g->d, p.v);
    while (p.lanes < 6 && (1u << p.lanes) < p.groups) p.lanes++;
    p.colblocks = (uint32_t)ceil_div(p.groups, 1u << p.lanes);
    // The longest chunks that leave enough threads; shorter ones read more rows twice. us with chunks of 8, 16, 32 steps,
    // 4 taps, forward: 1 x 4096 x 1024 bf16 12, 15, 25; 2 x 4096 x 2048 20, 24, 27 (2^18 threads with 8); 4 x 4096 x 4096
    // 67, 62, 58 (2^18 with 32). Backward: 19, 19, 20 (2^16 with 32); 44, 37, 29.
    p.steps = 32;
    const uint64_t enough = backward ? 1u << 16 : 1u << 18;
    while (p.steps > 8 && (uint64_t)g->b * ceil_div(g->t, p.steps) * p.groups < enough) p.steps /= 2;
    p.chunks = g->t ? (uint32_t)ceil_div(g->t, p.steps) : 1;
    const uint64_t items = (uint64_t)g->b * p.chunks;
    p.items = items >= 1ull << 32 ? 0 : (uint32_t)items;
    const uint64_t blocks = ceil_div(items, kThreads >> p.lanes);
    p.blocks = blocks >= 1ull << 32 ? 0 : (uint32_t)blocks;
    // workgroups of a column block: 2048 over all, and as many (of one launch's) as leave a thread kMostItems chunks' terms
    const uint64_t few = ceil_div(2048, p.colblocks), room = ((1ull << 32) / kThreads - 1) / p.colblocks;
    uint64_t walks = ceil_div(blocks, kMostItems);
    if (walks > room) walks = room;
    if (walks < few) walks = few;
    p.walks = (uint32_t)(walks < blocks ? walks : blocks);
    return p;
}
size_t workspace_of(const fhc_short_conv_desc* g) {
    return (size_t)plan_of(g, true).walks * g->d * (g->k + 1) * 4;
}

int check_desc(const char* op, const fhc_short_conv_desc* g) {
    if (!g) return fail(-1, "%s: null descriptor", op);
    FHC_TRY(check_shape(op, g->dtype, g->b, g->t, g->d));
    if (g->k < 2 || g->k > 4) return fail(-1, "%s: %u taps, 2 to 4 are possible", op, g->k);
    if (g->act != FHC_ACT_SILU && g->act != FHC_ACT_IDENTITY) return fail(-1, "%s: act %u", op, g->act);
    const uint32_t e = elem_bytes(g->dtype);
    FHC_TRY(check_array(op, "w", g->w, e, g->b && g->d));
    FHC_TRY(check_array(op, "bias", g->bias, e, false));
    return check_array(op, "lengths", g->lengths, 4, false);
}

template <class T>
ConvArgs<typename T::Raw> args_of(const fhc_short_conv_desc* g, const Plan& p, const fhc_seq* x, const void* state) {
    using R = typename T::Raw;
    ConvArgs<R> a{};
    a.x = seq_of<R>(x), a.w = static_cast<const R*>(g->w), a.bias = static_cast<const R*>(g->bias);
    a.state = static_cast<const R*>(state), a.lengths = g->lengths;
    a.b = g->b, a.t = g->t, a.d = g->d, a.groups = p.groups, a.lanes = p.lanes, a.colblocks = p.colblocks;
    a.chunks = p.chunks, a.steps = p.steps, a.items = p.items, a.walks = p.walks;
    a.silu = g->act == FHC_ACT_SILU, a.whole = g->d >= p.v;
    return a;
}

template <class T, bool BWD>
void launch(uint32_t k, uint32_t blocks, const ConvArgs<typename T::Raw>& a, hipStream_t st) {
    constexpr int V = BWD ? kBackV : kForwardV(T::id);
#define CONV(K)                                                                                              \
    do {                                                                                                     \
        if constexpr (BWD) hipLaunchKernelGGL((short_conv_bwd<T, K, V>), dim3(blocks), dim3(kThreads), 0, st, a); \
        else hipLaunchKernelGGL((short_conv_fwd<T, K, V>), dim3(blocks), dim3(kThreads), 0, st, a);          \
    } while (0)
    if (k == 2) CONV(2);
    else if (k == 3) CONV(3);
    else CONV(4);
#undef CONV
}

}  // namespace
}  // namespace seq
}  // namespace fhc

using namespace fhc;
using namespace fhc::seq;

extern "C" int fhc_short_conv_forward(const fhc_short_conv_desc* g, const fhc_seq* x, const void* state,
                                      const fhc_seq* y, void* state_out, void* stream) {
    return guard(-3, [&]() -> int {
        clear_error();
        const char* op = "short_conv_forward";
        FHC_TRY(check_desc(op, g));
        if ((uint64_t)g->b * g->d == 0) return 0;
        FHC_TRY(check_in(op, "x", x, g->dtype, g->t));
        FHC_TRY(check_out(op, "y", y, g->dtype, g->b, g->t, g->d));
        FHC_TRY(check_array(op, "state", state, elem_bytes(g->dtype), false));
        FHC_TRY(check_array(op, "state_out", state_out, elem_bytes(g->dtype), false));
        const Plan p = plan_of(g, false);
        const uint64_t grid = (uint64_t)p.blocks * p.colblocks;
        if (!p.items || !p.blocks) return fail(-1, "%s: too many workgroups", op);
        FHC_TRY(check_grid(op, grid, kThreads));
        with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            using R = typename T::Raw;
            auto a = args_of<T>(g, p, x, state);
            a.y = seq_of<R>(y), a.end = static_cast<R*>(state_out);
            // over the old state, both threads of a channel have to read it before either writes: the same wave's do
            if (state && state == state_out && p.groups % (1u << p.lanes) == 1) a.whole = false;
            launch<T, false>(g->k, (uint32_t)grid, a, (hipStream_t)stream);
        });
        return launched(op);
    });
}

extern "C" size_t fhc_short_conv_workspace_bytes(const fhc_short_conv_desc* g) {
    return guard((size_t)0, [&]() -> size_t {
        clear_error();
        if (check_desc("short_conv_workspace_bytes", g) < 0 || (uint64_t)g->b * g->d == 0) return 0;
        return workspace_of(g);
    });
}

extern "C" int fhc_short_conv_backward(const fhc_short_conv_desc* g, const fhc_seq* x, const void* state,
                                       const fhc_seq* dy, const void* dstate_out, const fhc_seq* dx, float* dw,
                                       float* dbias, void* dstate, void* ws, size_t ws_bytes, void* stream) {
    return guard(-3, [&]() -> int {
        clear_error();
        const char* op = "short_conv_backward";
        FHC_TRY(check_desc(op, g));
        if (g->d == 0) return 0;
        const hipStream_t st = (hipStream_t)stream;
        FHC_TRY(check_array(op, "dw", dw, 4, false));
        FHC_TRY(check_array(op, "dbias", dbias, 4, false));
        const Sums sums{{dw, dbias, nullptr}, {(uint64_t)g->d * g->k, g->d, 0}};
        if (g->b == 0) return close_sums(op, nullptr, 0, sums, st);  // empty ones
        const uint32_t e = elem_bytes(g->dtype);
        FHC_TRY(check_in(op, "x", x, g->dtype, g->t));
        FHC_TRY(check_in(op, "dy", dy, g->dtype, g->t));
        if (dx) FHC_TRY(check_out(op, "dx", dx, g->dtype, g->b, g->t, g->d));
        FHC_TRY(check_array(op, "state", state, e, false));
        FHC_TRY(check_array(op, "dstate_out", dstate_out, e, false));
        FHC_TRY(check_array(op, "dstate", dstate, e, false));
        const Plan p = plan_of(g, true);
        if (!p.items || !p.blocks) return fail(-1, "%s: too many workgroups", op);
        FHC_TRY(check_grid(op, (uint64_t)p.walks * p.colblocks, kThreads));
        FHC_TRY(check_workspace(op, workspace_of(g), ws, ws_bytes));
        with_type(g->dtype, [&](auto t) {
            using T = decltype(t);
            using R = typename T::Raw;
            auto a = args_of<T>(g, p, x, state);
            a.dy = seq_of<R>(dy), a.dx = seq_of<R>(dx), a.dend = static_cast<const R*>(dstate_out);
            a.dstate = static_cast<R*>(dstate), a.part = static_cast<float*>(ws);
            launch<T, true>(g->k, p.walks * p.colblocks, a, st);
        });
        FHC_TRY(launched(op));
        return close_sums(op, static_cast<const float*>(ws), p.walks, sums, st);
    });
}
