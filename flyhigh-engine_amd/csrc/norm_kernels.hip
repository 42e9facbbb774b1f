// The norms around a block with its gate and the scaled residual (include/fhc_seq.h), forward and backward.
//
// Both directions are bound by HBM: x and o in, y and u out; x, o, dy, du in, dx and do out. So a row is read once into
// registers, every statistic comes from there, and y (which u and its statistics need unrounded) is never read back:
// the backward pass computes it again from x and o in place of reading it. A row is held by threads of 8 channels each
// (K such groups for the widest rows): a part of a wave for narrow rows, so that a wave takes several pixels, as many
// waves as it needs (up to 16) for wide ones.
//
// MI355X, where a large copy moves 5.0 TB/s: forward of 16384 x 4096 bf16 95 us (537 MB, 5.7 TB/s), of
// 15009 x 1931 f16, whose rows lie at any 2-byte address, 51 (4.6). Backward of the former 174 us (805 MB, 4.6 TB/s; the
// first form, which did not have the next row's loads under way, 289), its closing sums 10 us more. Two shapes are far
// from that: above 8192 channels, 16 a thread, a backward pass spills 330 to 940 bytes a lane (4000 x 8192 bf16 105 us,
// 4000 x 8200 325); and norm_sum walks groups 64 at a time (262144 x 128 bf16, backward, in 64 groups 95 us, in 4096 158).
#include "seq_common.h"

namespace fhc {
namespace seq {
namespace {

struct Rows {
    char* p;
    int64_t ld;
};

struct NormArgs {
    Rows x, o, y, u, dy, du, dx, dout;
    const void *w_post, *w_pre, *gate;
    float *dgate, *part_post, *part_pre;  // see norm_bwd
    uint32_t rows, c, rpg, groups;
    uint32_t first;  // the launch's first row (forward)
    uint32_t per_group, part_rows;  // parts of a group, rows of a part; per_group 0: a workgroup takes whole groups
    uint32_t wg_groups;             // groups of a workgroup, where per_group is 0
    float alpha, eps;
};

// 8 adjacent channels of a row as they lie in memory, held in registers until they are used: all of a row's loads are
// then under way together.
template <class T>
struct Chunk {
    typedef uint32_t Vec __attribute__((ext_vector_type(4)));
    Vec w;
    __device__ __forceinline__ float at(int i) const { return widen(T{}, (uint16_t)(i & 1 ? w[i >> 1] >> 16 : w[i >> 1])); }
    __device__ __forceinline__ void set(int i, uint16_t v) {
        w[i >> 1] = i & 1 ? (w[i >> 1] & 0xFFFFu) | (uint32_t)v << 16 : (w[i >> 1] & 0xFFFF0000u) | v;
    }
};
template <>
struct Chunk<F32> {
    typedef float Vec __attribute__((ext_vector_type(8)));
    Vec w;
    __device__ __forceinline__ float at(int i) const { return w[i]; }
    __device__ __forceinline__ void set(int i, float v) { w[i] = v; }
};

// Where a thread's 8 channels are. AL: c is a multiple of 8 and every address one of 16 bytes. Otherwise the last
// thread of a row takes the row's last 8 channels, of which the first `skip` belong to the thread before it: they are
// read again, count for nothing and are not stored (c < 8: one thread, element by element).
struct Place {
    uint32_t ch, skip;
    bool in;
};
template <bool AL>
__device__ __forceinline__ Place place_of(uint32_t thread, uint32_t c) {
    const uint32_t ch = thread * 8;
    if (AL || c < 8) return {ch, 0, ch < c};
    const uint32_t at = ch + 8 <= c ? ch : c - 8;
    return {at, ch < c ? ch - at : 8, ch < c};
}
template <class T, bool AL>
__device__ __forceinline__ Chunk<T> load8(const void* base, int64_t at, Place p, uint32_t c) {
    using R = typename T::Raw;
    typedef typename Chunk<T>::Vec Mem __attribute__((aligned(AL ? 16 : sizeof(R))));
    const R* q = reinterpret_cast<const R*>(base) + at + p.ch;
    Chunk<T> v{};
    if (AL || c >= 8) {
        if (p.in) v.w = *reinterpret_cast<const Mem*>(q);
    } else if (p.in) {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < (int)c) v.set(i, q[i]);
    }
    return v;
}
// the values, 0 where they are another thread's (weights and gates too: 0 times an infinite one is not 0)
template <class T, bool AL>
__device__ __forceinline__ float own(const Chunk<T>& v, Place p, int i) {
    return AL || i >= (int)p.skip ? v.at(i) : 0.0f;
}
template <class T, bool AL>
__device__ __forceinline__ void widen8(const Chunk<T>& v, Place p, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = own<T, AL>(v, p, i);
}
template <class T, bool AL>
__device__ __forceinline__ void store8(void* base, int64_t at, Place p, uint32_t c, const float (&f)[8]) {
    using R = typename T::Raw;
    typedef typename Chunk<T>::Vec Mem __attribute__((aligned(AL ? 16 : sizeof(R))));
    R* q = reinterpret_cast<R*>(base) + at + p.ch;
    Chunk<T> v{};
#pragma unroll
    for (int i = 0; i < 8; i++) v.set(i, narrow(T{}, f[i]));
    if (AL || (p.skip == 0 && c >= 8)) {
        if (p.in) *reinterpret_cast<Mem*>(q) = v.w;
    } else if (p.in) {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i >= (int)p.skip && i < (int)c) q[i] = narrow(T{}, f[i]);
    }
}
// 8 weights, 1 where there are none
template <class T, bool AL>
__device__ __forceinline__ Chunk<T> weight8(const void* base, int64_t at, Place p, uint32_t c) {
    if (base) return load8<T, AL>(base, at, p, c);
    Chunk<T> v{};
#pragma unroll
    for (int i = 0; i < 8; i++) v.set(i, narrow(T{}, 1.0f));
    return v;
}

template <int CTRL>
__device__ __forceinline__ float dpp_plus(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
// the sum over TPR <= 64 lanes, in each of them: within 16 lanes by the adder's own lane selection (neighbours, pairs,
// mirrored halves), then by exchanging rows of 16 and of 32
template <int TPR>
__device__ __forceinline__ float lane_sum(float v) {
    v = dpp_plus<0xB1>(v);
    v = dpp_plus<0x4E>(v);
    v = dpp_plus<0x141>(v);
    v = dpp_plus<0x140>(v);
    if constexpr (TPR >= 32) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v);
        const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        const uint32_t a = s[0], b = s[1];  // (a bit cast of an element itself reads the first one)
        v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
    }
    if constexpr (TPR >= 64) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v);
        const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        const uint32_t a = s[0], b = s[1];
        v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
    }
    return v;
}
// 1 / sqrt(mean + eps). The instruction takes f32's subnormal numbers for 0, which only an eps that small leads to (a row
// of zeros is still a row of zeros then). A NaN stays.
__device__ __forceinline__ float inv_rms(float sum, float inv_c, float eps) {
    const float v = __builtin_fmaf(sum, inv_c, eps);
    if (eps < 0x1p-126f && v < 0x1p-126f) return __builtin_amdgcn_rsqf(v * 0x1p64f) * 0x1p32f;
    return __builtin_amdgcn_rsqf(v);
}
constexpr int kWide = 1024;  // TPR of rows that a whole workgroup of up to 16 waves holds
// Sums of N values over the threads of a row. Rows of several waves go through LDS, the buffers of successive sums in
// turn so that one barrier a sum is enough; each wave adds all waves' sums.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*lds)[N][16], uint32_t waves) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = lane_sum<TPR>(v[i]);
    if constexpr (TPR == kWide) {
        const uint32_t lane = threadIdx.x & 63;
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < N; i++) (*lds)[i][threadIdx.x >> 6] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float q = (*lds)[i][lane & 15];
            v[i] = lane_sum<16>((lane & 15) < waves ? q : 0.0f);
        }
    }
}

// threads of a workgroup: several narrow rows, or one wide one
template <int TPR>
constexpr int kBlock = TPR <= 64 ? 256 : TPR;

template <class T, int TPR, int K, bool AL>
__global__ __launch_bounds__(kBlock<TPR>) void norm_fwd(NormArgs g) {
    __shared__ float lds[2][1][16];
    const uint32_t tpr = TPR == kWide ? blockDim.x : TPR, waves = blockDim.x / 64;
    const uint32_t lane = TPR == kWide ? threadIdx.x : threadIdx.x % TPR;
    const uint32_t row = g.first + (TPR == kWide ? blockIdx.x : blockIdx.x * (kBlock<TPR> / TPR) + threadIdx.x / TPR);
    const bool live = row < g.rows;  // a row past the end keeps pace
    const int64_t group = g.gate && live ? row / g.rpg : 0;
    const float inv_c = 1.0f / (float)g.c;
    Place at[K];
    Chunk<T> xr[K], orr[K], wp[K], ga[K], wn[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        at[k] = place_of<AL>(k * tpr + lane, g.c);
        at[k].in &= live;
        xr[k] = load8<T, AL>(g.x.p, row * g.x.ld, at[k], g.c);
        orr[k] = Chunk<T>{};
        if (g.o.p) {
            orr[k] = load8<T, AL>(g.o.p, row * g.o.ld, at[k], g.c);
            wp[k] = weight8<T, AL>(g.w_post, 0, at[k], g.c);
            ga[k] = weight8<T, AL>(g.gate, group * g.c, at[k], g.c);
        }
        wn[k] = weight8<T, AL>(g.w_pre, 0, at[k], g.c);
    }
    float x[K][8], o[K][8], s[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < K; k++) widen8<T, AL>(orr[k], at[k], o[k]);
    if (g.o.p) {
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int i = 0; i < 8; i++) s[0] = __builtin_fmaf(o[k][i], o[k][i], s[0]);
        row_sum<TPR, 1>(s, &lds[0], waves);
        const float ro = inv_rms(s[0], inv_c, g.eps);
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int i = 0; i < 8; i++) o[k][i] *= ro * own<T, AL>(wp[k], at[k], i) * own<T, AL>(ga[k], at[k], i);
    }
    s[0] = 0.0f;
#pragma unroll
    for (int k = 0; k < K; k++) {
        widen8<T, AL>(xr[k], at[k], x[k]);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[k][i] = __builtin_fmaf(g.alpha, x[k][i], o[k][i]);
            s[0] = __builtin_fmaf(x[k][i], x[k][i], s[0]);
        }
        if (g.y.p) store8<T, AL>(g.y.p, row * g.y.ld, at[k], g.c, x[k]);
    }
    if (!g.u.p) return;
    row_sum<TPR, 1>(s, &lds[1], waves);
    const float ry = inv_rms(s[0], inv_c, g.eps);
#pragma unroll
    for (int k = 0; k < K; k++) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[k][i] *= ry * own<T, AL>(wn[k], at[k], i);
        store8<T, AL>(g.u.p, row * g.u.ld, at[k], g.c, x[k]);
    }
}

// Backward. With n_o = o / rms(o), n_y = y / rms(y), z = gate * w_post * dY:
//     dY = dy + (w_pre du - n_y mean(w_pre du n_y)) / rms(y)
//     dx = alpha dY,   do = (z - n_o mean(z n_o)) / rms(o)
//     dgate = w_post * sum dY n_o,   dw_post = sum gate dY n_o,   dw_pre = sum du n_y
// mean(z n_o) is linear in dY, so its sum splits into three that need only o and y; they are taken together with
// those of y, and a row costs two exchanges in place of four. The next row's loads are under way while a row is worked
// on (without that the loads' latency was half of the time).
//
// A workgroup (one wide row or RPB narrow ones at a time) owns the sums of its rows in registers. PARTS: groups are
// long, a workgroup takes a part of one group (group = part / per_group), and its dY n_o sum is a partial sum of dgate
// and, times the gate, of dw_post. Otherwise every RPB-th group of a run of wg_groups is one slot's, which writes dgate
// itself and leaves a partial sum of dw_post. norm_sum adds the partial rows in their order.
// waves a SIMD that the registers are held to; the narrow rows' larger variants spill at 4
template <int TPR, int ELEM, bool PARTS>
constexpr int kWaves = TPR == kWide || (PARTS && ELEM == 2) ? 4 : 3;

template <class T, int TPR, int K, bool AL, bool PARTS>
__global__ __launch_bounds__(kBlock<TPR>, (kWaves<TPR, sizeof(typename T::Raw), PARTS>)) void norm_bwd(NormArgs g) {
    constexpr int RPB = kBlock<TPR> / TPR;
    __shared__ float lds1[2][1][16];
    __shared__ float lds5[2][5][16];
    __shared__ float fold[RPB > 1 ? RPB * TPR * 8 : 1];
    const uint32_t tpr = TPR == kWide ? blockDim.x : TPR, waves = blockDim.x / 64;
    const uint32_t lane = TPR == kWide ? threadIdx.x : threadIdx.x % TPR;
    const uint32_t slot = TPR == kWide ? 0 : threadIdx.x / TPR;
    const float inv_c = 1.0f / (float)g.c;
    const bool has_o = g.o.p != nullptr;
    // the groups and rows of this slot: group gr, gr + gstep, ... below g1; rows r, r + rstep, ... below hi of each
    uint32_t gr, g1, r, lo = 0, hi;
    constexpr uint32_t gstep = RPB, rstep = PARTS ? RPB : 1;
    auto rows_of = [&](uint32_t group) {
        const uint64_t base = (uint64_t)group * g.rpg;
        return (uint32_t)min((uint64_t)g.rpg, g.rows - base);
    };
    if constexpr (PARTS) {
        gr = blockIdx.x / g.per_group, g1 = gr + 1;
        const uint32_t part = blockIdx.x - gr * g.per_group;
        lo = part * g.part_rows, hi = min(lo + g.part_rows, rows_of(gr));
        lo += slot;
    } else {
        gr = blockIdx.x * g.wg_groups + slot, g1 = min((blockIdx.x + 1) * g.wg_groups, g.groups);
        hi = gr < g1 ? rows_of(gr) : 0;
    }
    r = lo;
    bool more = gr < g1 && r < hi;

    Place at[K];
    float wn[K][8], gw[K][8], q[K][8], pre[K][8], post[PARTS ? 1 : K][8];
    Chunk<T> wp[PARTS ? 1 : K], xr[K], orr[K], dyr[K], dur[K], gar[PARTS ? 1 : K];
    auto fetch = [&](bool ok) {
        const int64_t row = (int64_t)((uint64_t)gr * g.rpg + r);
#pragma unroll
        for (int k = 0; k < K; k++) {
            Place p = at[k];
            p.in &= ok;
            xr[k] = load8<T, AL>(g.x.p, row * g.x.ld, p, g.c);
            if (has_o) orr[k] = load8<T, AL>(g.o.p, row * g.o.ld, p, g.c);
            if (g.dy.p) dyr[k] = load8<T, AL>(g.dy.p, row * g.dy.ld, p, g.c);
            if (g.du.p) dur[k] = load8<T, AL>(g.du.p, row * g.du.ld, p, g.c);
            if constexpr (!PARTS) gar[k] = weight8<T, AL>(g.gate, (int64_t)gr * g.c, p, g.c);
        }
    };
#pragma unroll
    for (int k = 0; k < K; k++) {
        at[k] = place_of<AL>(k * tpr + lane, g.c);
        orr[k] = dyr[k] = dur[k] = Chunk<T>{};
    }
    fetch(more);
#pragma unroll
    for (int k = 0; k < K; k++) {
        const Chunk<T> pw = weight8<T, AL>(g.w_post, 0, at[k], g.c), nw = weight8<T, AL>(g.w_pre, 0, at[k], g.c);
        widen8<T, AL>(nw, at[k], wn[k]);
        if constexpr (PARTS) {
            const Chunk<T> ga = weight8<T, AL>(g.gate, (int64_t)gr * g.c, at[k], g.c);
#pragma unroll
            for (int i = 0; i < 8; i++) gw[k][i] = own<T, AL>(pw, at[k], i) * own<T, AL>(ga, at[k], i);
        } else {
            wp[k] = pw;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) q[k][i] = pre[k][i] = post[PARTS ? 0 : k][i] = 0.0f;
    }

    uint32_t turn = 0;
    while (more) {
        const int64_t row = (int64_t)((uint64_t)gr * g.rpg + r);
        const uint32_t group = gr;
        float x[K][8], o[K][8], dy[K][8], du[K][8];
        Chunk<T> ga[PARTS ? 1 : K];
        float s1[1] = {0.0f}, s5[5] = {};
#pragma unroll
        for (int k = 0; k < K; k++) {
            widen8<T, AL>(xr[k], at[k], x[k]);
            widen8<T, AL>(orr[k], at[k], o[k]);
            widen8<T, AL>(dyr[k], at[k], dy[k]);
            widen8<T, AL>(dur[k], at[k], du[k]);
            if constexpr (!PARTS) {
                ga[k] = gar[k];
#pragma unroll
                for (int i = 0; i < 8; i++) gw[k][i] = own<T, AL>(ga[k], at[k], i) * own<T, AL>(wp[k], at[k], i);
            }
        }
        r += rstep;
        if (r >= hi) {
            gr += gstep, r = lo;
            more = !PARTS && gr < g1;
            if (more) hi = rows_of(gr);
        }
        if (more) fetch(true);
        float ro = 0.0f;
        if (has_o) {
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int i = 0; i < 8; i++) s1[0] = __builtin_fmaf(o[k][i], o[k][i], s1[0]);
            row_sum<TPR, 1>(s1, &lds1[turn], waves);
            ro = inv_rms(s1[0], inv_c, g.eps);
        }
#pragma unroll
        for (int k = 0; k < K; k++) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                o[k][i] *= ro;  // n_o
                const float zo = gw[k][i] * o[k][i], w = wn[k][i] * du[k][i];
                x[k][i] = __builtin_fmaf(g.alpha, x[k][i], zo);  // y
                s5[0] = __builtin_fmaf(x[k][i], x[k][i], s5[0]);
                s5[1] = __builtin_fmaf(w, x[k][i], s5[1]);
                s5[2] = __builtin_fmaf(zo, dy[k][i], s5[2]);
                s5[3] = __builtin_fmaf(zo, w, s5[3]);
                s5[4] = __builtin_fmaf(zo, x[k][i], s5[4]);
            }
        }
        row_sum<TPR, 5>(s5, &lds5[turn], waves);
        turn ^= 1;
        const float ry = inv_rms(s5[0], inv_c, g.eps);
        const float my = s5[1] * inv_c * ry * ry;                          // mean(w_pre du n_y) / rms(y)
        const float mo = (s5[2] + ry * s5[3] - ry * my * s5[4]) * inv_c;    // mean(z n_o)
#pragma unroll
        for (int k = 0; k < K; k++) {
            float dx[8], dv[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float ny = x[k][i] * ry;
                const float d = __builtin_fmaf(-my, ny, __builtin_fmaf(ry, wn[k][i] * du[k][i], dy[k][i]));  // dY
                dx[i] = g.alpha * d;
                dv[i] = ro * __builtin_fmaf(-mo, o[k][i], gw[k][i] * d);
                q[k][i] = __builtin_fmaf(d, o[k][i], q[k][i]);
                pre[k][i] = __builtin_fmaf(du[k][i], ny, pre[k][i]);
            }
            store8<T, AL>(g.dx.p, row * g.dx.ld, at[k], g.c, dx);
            if (has_o) store8<T, AL>(g.dout.p, row * g.dout.ld, at[k], g.c, dv);
        }
        if constexpr (!PARTS) {
            if (gr != group) {  // the group is done
#pragma unroll
                for (int k = 0; k < K; k++) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        post[k][i] = __builtin_fmaf(ga[k].at(i), q[k][i], post[k][i]);
                        if (g.dgate && at[k].in && i >= (int)at[k].skip && at[k].ch + i < g.c)
                            g.dgate[(uint64_t)group * g.c + at[k].ch + i] = wp[k].at(i) * q[k][i];
                        q[k][i] = 0.0f;
                    }
                }
            }
        }
    }
    // the slots' sums of one workgroup, added in the slots' order by slot 0
    auto leave = [&](float (*v)[8], float* out) {
        if (!out) return;
#pragma unroll
        for (int k = 0; k < K; k++) {
            if constexpr (RPB > 1) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 8; i++) fold[(slot * 8 + i) * TPR + lane] = v[k][i];
                __syncthreads();
                if (slot == 0) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
#pragma unroll
                        for (int t = 1; t < RPB; t++) v[k][i] += fold[(t * 8 + i) * TPR + lane];
                    }
                }
            }
            if (slot == 0 && at[k].in) {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i >= (int)at[k].skip && at[k].ch + i < g.c)
                        out[(uint64_t)blockIdx.x * g.c + at[k].ch + i] = v[k][i];
            }
        }
    };
    leave(pre, g.part_pre);
    leave(PARTS ? q : post, g.part_post);
}

// The partial rows' sums, 16 columns x 64 row lanes a workgroup, in f64. z 0: dw_pre, the sum of all `wgs` rows of
// `pre`. z 1: the sum Q of `parts` rows of `post` for each group; dgate = w_post * Q, dw_post = the sum of gate * Q over
// the groups. The 64 lanes are as many groups as there are (up to 64) times the lanes that are left for a group's parts.
template <class T>
__global__ __launch_bounds__(1024) void norm_sum(const float* pre, float* dw_pre, uint32_t wgs, const float* post,
                                                 float* dw_post, float* dgate, const void* gate, const void* w_post,
                                                 uint32_t groups, uint32_t parts, uint32_t part_lanes, uint32_t c) {
    __shared__ double s[64][17];
    using R = typename T::Raw;
    const uint32_t x = threadIdx.x & 15, y = threadIdx.x >> 4, ch = blockIdx.x * 16 + x;
    const bool first = blockIdx.z == 0;
    if (first ? !dw_pre : !post) return;
    const float* in = first ? pre : post;
    const uint32_t rows = first ? wgs : parts, pl = first ? 64 : part_lanes, p = y % pl, gl = 64 / pl;
    const uint32_t n = first ? 1 : groups;
    double total = 0.0;
    for (uint32_t g0 = 0; g0 < n; g0 += gl) {
        const uint32_t g = g0 + y / pl;
        double acc = 0.0;
        if (ch < c && g < n) {
#pragma unroll 8
            for (uint32_t r = p; r < rows; r += pl) acc += (double)in[((uint64_t)g * rows + r) * c + ch];
        }
        if (pl > 1) {
            __syncthreads();
            s[y][x] = acc;
            __syncthreads();
            if (p == 0) {
                for (uint32_t k = 1; k < pl; k++) acc += s[y + k][x];
            }
        }
        if (p == 0 && ch < c && g < n) {
            if (first) {
                total = acc;
            } else {
                if (dgate) {
                    const double w = w_post ? (double)widen(T{}, reinterpret_cast<const R*>(w_post)[ch]) : 1.0;
                    dgate[(uint64_t)g * c + ch] = (float)(acc * w);
                }
                total += gate ? acc * (double)widen(T{}, reinterpret_cast<const R*>(gate)[(uint64_t)g * c + ch]) : acc;
            }
        }
    }
    float* out = first ? dw_pre : dw_post;
    if (!out) return;
    __syncthreads();
    s[y][x] = total;  // 0 in lanes that are not a group's first
    __syncthreads();
    if (y == 0 && ch < c) {
        for (uint32_t k = pl; k < 64; k += pl) total += s[k][x];
        out[ch] = (float)total;
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------

int check_desc(const char* op, const fhc_norm_desc* n) {
    if (!n) return fail(-1, "%s: null descriptor", op);
    if (n->dtype > FHC_F32) return fail(-1, "%s: dtype %u is none of f16, bf16, f32", op, n->dtype);
    if (n->c > 16384) return fail(-1, "%s: %u channels, at most 16384", op, n->c);
    if (n->rows > 0x7FFFFFFFu) return fail(-1, "%s: %u rows, at most 2^31 - 1", op, n->rows);
    if (n->gate && n->rows_per_group == 0) return fail(-1, "%s: rows_per_group is 0", op);
    if (!std::isfinite(n->alpha)) return fail(-1, "%s: alpha %g", op, (double)n->alpha);
    if (!(n->eps > 0.0f) || !std::isfinite(n->eps)) return fail(-1, "%s: eps %g", op, (double)n->eps);
    const uint32_t e = elem_bytes(n->dtype);
    if (!aligned(n->w_post, e) || !aligned(n->w_pre, e) || !aligned(n->gate, e))
        return fail(-1, "%s: a weight or the gate is not aligned to its elements", op);
    return 0;
}
int check_rows(const char* op, const char* name, const fhc_rows* r, const fhc_norm_desc* n, bool needed) {
    if (!r) return needed ? fail(-1, "%s: null %s", op, name) : 0;
    if (!r->p) return fail(-1, "%s: null pointer of %s", op, name);
    if (r->ld < (int64_t)n->c)
        return fail(-1, "%s: rows of %s are %lld apart, below %u channels", op, name, (long long)r->ld, n->c);
    if (!aligned(r->p, elem_bytes(n->dtype))) return fail(-1, "%s: %s is not aligned to its elements", op, name);
    return 0;
}

Rows rows_of(const fhc_rows* r) { return r ? Rows{static_cast<char*>(r->p), r->ld} : Rows{nullptr, 0}; }

// whole 8-channel groups at 16-byte (f32: 32-byte) steps everywhere
bool whole(const fhc_norm_desc* n, std::initializer_list<const fhc_rows*> all) {
    if (n->c % 8 || !aligned(n->w_post, 16) || !aligned(n->w_pre, 16) || !aligned(n->gate, 16)) return false;
    for (const fhc_rows* r : all)
        if (r && (r->ld % 8 || !aligned(r->p, 16))) return false;
    return true;
}

// threads of a row, 8 channels each, 16 each above 8192: a part of a wave, or whole waves
uint32_t threads_of_row(uint32_t c) {
    if (c <= 128) return 16;
    if (c <= 256) return 32;
    return (uint32_t)ceil_div(c, c > 8192 ? 1024 : 512) * 64;
}

// f(T, TPR, K, AL)
template <class F>
void with_shape(uint32_t dtype, uint32_t tpr, uint32_t c, bool al, F&& f) {
    auto by_al = [&](auto t, auto n, auto k) {
        if (al) f(t, n, k, std::true_type{});
        else f(t, n, k, std::false_type{});
    };
    auto by_rows = [&](auto t) {
        using std::integral_constant;
        if (c > 8192) by_al(t, integral_constant<int, kWide>{}, integral_constant<int, 2>{});
        else if (tpr > 64) by_al(t, integral_constant<int, kWide>{}, integral_constant<int, 1>{});
        else if (tpr == 64) by_al(t, integral_constant<int, 64>{}, integral_constant<int, 1>{});
        else if (tpr == 32) by_al(t, integral_constant<int, 32>{}, integral_constant<int, 1>{});
        else by_al(t, integral_constant<int, 16>{}, integral_constant<int, 1>{});
    };
    if (dtype == FHC_F16) by_rows(F16{});
    else if (dtype == FHC_BF16) by_rows(BF16{});
    else by_rows(F32{});
}

struct Split {
    uint32_t tpr, rpb, block, groups, rpg, per_group, part_rows, wg_groups, wgs;
    size_t post_at, bytes;
};
// The backward pass's workgroups: as many as its registers let the CUs hold at once, at least 4 rows a slot where there
// are so many. Groups of at least 4 passes are cut into parts; shorter ones are taken whole.
Split split_of(const fhc_norm_desc* n) {
    Split s{};
    s.tpr = threads_of_row(n->c);
    s.block = s.tpr <= 64 ? 256 : s.tpr;
    s.rpb = s.block / s.tpr;
    s.rpg = n->gate ? n->rows_per_group : n->rows;
    if (s.rpg > n->rows) s.rpg = n->rows;
    if (s.rpg == 0) s.rpg = 1;
    s.groups = (uint32_t)ceil_div(n->rows, s.rpg);
    const bool parts = s.groups && s.rpg >= 4 * s.rpb;
    const uint32_t waves = s.tpr > 64 || (parts && n->dtype != FHC_F32) ? 16 : 12;  // a CU's, see kWaves
    const uint32_t most = 256 * (waves * 64 / s.block);
    if (parts) {
        uint64_t per = s.groups >= most ? 1 : most / s.groups;
        const uint64_t cap = ceil_div(s.rpg, 4 * s.rpb);
        if (per > cap) per = cap;
        s.part_rows = (uint32_t)ceil_div(s.rpg, per);
        s.per_group = (uint32_t)ceil_div(s.rpg, s.part_rows);
        s.wgs = s.groups * s.per_group;
    } else {
        s.wg_groups = (uint32_t)ceil_div(ceil_div(s.groups, most), s.rpb) * s.rpb;
        s.wgs = s.groups ? (uint32_t)ceil_div(s.groups, s.wg_groups) : 0;
    }
    s.post_at = (size_t)ceil_div((uint64_t)s.wgs * n->c * 4, 256) * 256;
    s.bytes = 2 * s.post_at;
    return s;
}

}  // namespace
}  // namespace seq
}  // namespace fhc

using namespace fhc;
using namespace fhc::seq;

extern "C" int fhc_norm_block(const fhc_norm_desc* n, const fhc_rows* x, const fhc_rows* o, const fhc_rows* y,
                              const fhc_rows* u, void* stream) {
    return guard(-3, [&]() -> int {
        clear_error();
        const char* op = "norm_block";
        FHC_TRY(check_desc(op, n));
        if (n->rows == 0 || n->c == 0) return 0;
        FHC_TRY(check_rows(op, "x", x, n, true));
        FHC_TRY(check_rows(op, "o", o, n, false));
        FHC_TRY(check_rows(op, "y", y, n, false));
        FHC_TRY(check_rows(op, "u", u, n, false));
        if (!y && !u) return fail(-1, "%s: neither y nor u is wanted", op);
        if (!o && (n->w_post || n->gate)) return fail(-1, "%s: a weight or gate without o", op);
        NormArgs a{};
        a.x = rows_of(x), a.o = rows_of(o), a.y = rows_of(y), a.u = rows_of(u);
        a.w_post = n->w_post, a.w_pre = n->w_pre, a.gate = n->gate;
        a.rows = n->rows, a.c = n->c, a.rpg = n->rows_per_group, a.alpha = n->alpha, a.eps = n->eps;
        const uint32_t tpr = threads_of_row(n->c);
        with_shape(n->dtype, tpr, n->c, whole(n, {x, o, y, u}), [&](auto t, auto w, auto k, auto al) {
            constexpr int TPR = decltype(w)::value;
            const uint32_t block = TPR == kWide ? tpr : kBlock<TPR>;
            const uint32_t most = (1u << 31) / block * (block / tpr);  // rows of a launch
            for (uint64_t first = 0; first < n->rows; first += most) {
                a.first = (uint32_t)first;
                const uint32_t count = n->rows - a.first < most ? n->rows - a.first : most;
                hipLaunchKernelGGL((norm_fwd<decltype(t), TPR, decltype(k)::value, decltype(al)::value>),
                                   dim3((uint32_t)ceil_div(count, block / tpr)), dim3(block), 0, (hipStream_t)stream, a);
            }
        });
        return launched(op);
    });
}

extern "C" size_t fhc_norm_block_workspace_bytes(const fhc_norm_desc* n) {
    return guard((size_t)0, [&]() -> size_t {
        clear_error();
        if (check_desc("norm_block_workspace_bytes", n) < 0) return 0;
        return split_of(n).bytes;
    });
}

extern "C" int fhc_norm_block_backward(const fhc_norm_desc* n, const fhc_rows* x, const fhc_rows* o,
                                       const fhc_rows* dy, const fhc_rows* du, const fhc_rows* dx,
                                       const fhc_rows* dout, float* dw_post, float* dgate, float* dw_pre, void* ws,
                                       size_t ws_bytes, void* stream) {
    return guard(-3, [&]() -> int {
        clear_error();
        const char* op = "norm_block_backward";
        FHC_TRY(check_desc(op, n));
        if (n->c == 0) return 0;
        if (!o && (n->w_post || n->gate || dout || dw_post || dgate))
            return fail(-1, "%s: a weight, gate or gradient of the block without o", op);
        if (dgate && !n->gate) return fail(-1, "%s: dgate without a gate", op);
        const Split s = split_of(n);
        FHC_TRY(check_grid(op, s.wgs, s.block));
        NormArgs a{};
        if (n->rows) {
            FHC_TRY(check_rows(op, "x", x, n, true));
            FHC_TRY(check_rows(op, "o", o, n, false));
            FHC_TRY(check_rows(op, "dy", dy, n, false));
            FHC_TRY(check_rows(op, "du", du, n, false));
            FHC_TRY(check_rows(op, "dx", dx, n, true));
            FHC_TRY(check_rows(op, "dout", dout, n, o != nullptr));
            if (!dy && !du) return fail(-1, "%s: neither dy nor du is given", op);
            FHC_TRY(check_workspace(op, s.bytes, ws, ws_bytes));
        }
        char* w = static_cast<char*>(ws);
        a.x = rows_of(x), a.o = rows_of(o), a.dy = rows_of(dy), a.du = rows_of(du), a.dx = rows_of(dx);
        a.dout = rows_of(dout);
        a.w_post = n->w_post, a.w_pre = n->w_pre, a.gate = n->gate;
        a.rows = n->rows, a.c = n->c, a.rpg = s.rpg, a.groups = s.groups, a.alpha = n->alpha, a.eps = n->eps;
        a.per_group = s.per_group, a.part_rows = s.part_rows, a.wg_groups = s.wg_groups;
        a.dgate = dgate;
        const bool parts = s.per_group != 0;
        a.part_pre = dw_pre ? reinterpret_cast<float*>(w) : nullptr;
        a.part_post = dw_post || (dgate && parts) ? reinterpret_cast<float*>(w + s.post_at) : nullptr;
        const hipStream_t st = (hipStream_t)stream;
        if (s.wgs) {
            with_shape(n->dtype, s.tpr, n->c, whole(n, {x, o, dy, du, dx, dout}), [&](auto t, auto tpr, auto k, auto al) {
                constexpr int TPR = decltype(tpr)::value, K = decltype(k)::value;
                using T = decltype(t);
                if (parts)
                    hipLaunchKernelGGL((norm_bwd<T, TPR, K, decltype(al)::value, true>), dim3(s.wgs), dim3(s.block), 0, st, a);
                else
                    hipLaunchKernelGGL((norm_bwd<T, TPR, K, decltype(al)::value, false>), dim3(s.wgs), dim3(s.block), 0, st, a);
            });
            FHC_TRY(launched(op));
        }
        if (dw_pre || dw_post || (dgate && parts)) {
            // of whole groups, dgate is written, and what is left for dw_post is one sum of all rows
            const uint32_t groups = parts ? s.groups : 1, rows = parts ? s.per_group : s.wgs;
            uint32_t lanes = 64;
            while (lanes > 1 && (uint64_t)lanes * groups > 64) lanes /= 2;
            auto sum = n->dtype == FHC_F16 ? norm_sum<F16> : n->dtype == FHC_BF16 ? norm_sum<BF16> : norm_sum<F32>;
            // without rows there are no partial sums, but dw_post is still written: any pointer will do
            const float* post = a.part_post || !dw_post ? a.part_post : dw_post;
            hipLaunchKernelGGL(sum, dim3((uint32_t)ceil_div(n->c, 16), 1, 2), dim3(1024), 0, st, a.part_pre, dw_pre,
                               s.wgs, post, dw_post, parts ? dgate : nullptr, parts ? n->gate : nullptr, n->w_post,
                               groups, rows, lanes, n->c);
            FHC_TRY(launched(op));
        }
        return 0;
    });
}
