// The norms around a block with its gate and the scaled residual (include/fhc_seq.h), forward and backward.
//
// Both directions are bound by HBM: x and o in, y and u out; x, o, dy, du in, dx and do out. So a row is read once into
// registers, every statistic comes from there, and y (which u and its statistics need unrounded) is never read back:
// the backward pass computes it again from x and o in place of reading it. A row is held by `tpr` threads, 8 channels
// each (K such groups for the widest rows): a part of a wave for narrow rows, so that a wave takes several pixels, up
// to a workgroup for wide ones.
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
    float *dgate, *part_post, *part_pre, *part_gate;  // see norm_bwd
    uint32_t rows, c, rpg, groups;
    uint32_t per_group, part_rows;  // parts of a group, rows of a part; per_group 0: a workgroup takes whole groups
    uint32_t wg_groups;             // groups of a workgroup, where per_group is 0
    float alpha, eps;
};

template <class T, bool AL>
__device__ __forceinline__ void load8(const void* base, int64_t at, uint32_t ch, uint32_t c, float (&f)[8]) {
    using R = typename T::Raw;
    const R* p = reinterpret_cast<const R*>(base) + at + ch;
    if (AL || ch + 8 <= c) {
        R q[8];
        load_raw<R, 8, AL>(p, q);
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = widen(T{}, q[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const R q = p[(ch + i < c ? i : 0)];
            f[i] = ch + i < c ? widen(T{}, q) : 0.0f;
        }
    }
}
template <class T, bool AL>
__device__ __forceinline__ void store8(void* base, int64_t at, uint32_t ch, uint32_t c, const float (&f)[8]) {
    using R = typename T::Raw;
    R* p = reinterpret_cast<R*>(base) + at + ch;
    R q[8];
#pragma unroll
    for (int i = 0; i < 8; i++) q[i] = narrow(T{}, f[i]);
    if (AL || ch + 8 <= c) {
        store_raw<R, 8, AL>(p, q);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (ch + i < c) p[i] = q[i];
    }
}
// 8 weights, 1 where there are none
template <class T, bool AL>
__device__ __forceinline__ void weight8(const void* base, int64_t at, uint32_t ch, uint32_t c, float (&f)[8]) {
    if (base) {
        load8<T, AL>(base, at, ch, c, f);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = 1.0f;
    }
}

// Sums of N values over the TPR threads of a row. Within a wave by lane exchange; a row of several waves goes through
// LDS, two buffers in turn so that one barrier a sum is enough.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*lds)[N][TPR > 64 ? TPR / 64 : 1]) {
#pragma unroll
    for (int m = 1; m < (TPR < 64 ? TPR : 64); m *= 2) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] += __shfl_xor(v[i], m);
    }
    if constexpr (TPR > 64) {
        constexpr int NW = TPR / 64;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; i++) (*lds)[i][threadIdx.x >> 6] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            v[i] = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; w++) v[i] += (*lds)[i][w];
        }
    }
}

template <int TPR>
constexpr int kBlock = TPR <= 64 ? 256 : TPR;  // rows of several waves have a workgroup each: its barriers are theirs

template <class T, int TPR, int K, bool AL>
__global__ __launch_bounds__(kBlock<TPR>) void norm_fwd(NormArgs g) {
    constexpr int RPB = kBlock<TPR> / TPR, NW = TPR > 64 ? TPR / 64 : 1;
    __shared__ float lds[2][1][NW];
    const uint32_t lane = threadIdx.x % TPR, row = blockIdx.x * RPB + threadIdx.x / TPR;
    const bool live = row < g.rows;  // a row past the end keeps pace with the barriers
    const int64_t group = g.gate && live ? row / g.rpg : 0;
    const float inv_c = 1.0f / (float)g.c;
    float x[K][8], o[K][8], s[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < K; k++) {
        const uint32_t ch = (k * TPR + lane) * 8;
#pragma unroll
        for (int i = 0; i < 8; i++) x[k][i] = o[k][i] = 0.0f;
        if (live && ch < g.c) {
            load8<T, AL>(g.x.p, row * g.x.ld, ch, g.c, x[k]);
            if (g.o.p) load8<T, AL>(g.o.p, row * g.o.ld, ch, g.c, o[k]);
        }
    }
    if (g.o.p) {
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int i = 0; i < 8; i++) s[0] = __builtin_fmaf(o[k][i], o[k][i], s[0]);
        row_sum<TPR, 1>(s, &lds[0]);
        const float ro = __builtin_amdgcn_rsqf(__builtin_fmaf(s[0], inv_c, g.eps));
#pragma unroll
        for (int k = 0; k < K; k++) {
            const uint32_t ch = (k * TPR + lane) * 8;
            if (!live || ch >= g.c) continue;
            float w[8], ga[8];
            weight8<T, AL>(g.w_post, 0, ch, g.c, w);
            weight8<T, AL>(g.gate, group * g.c, ch, g.c, ga);
#pragma unroll
            for (int i = 0; i < 8; i++) o[k][i] *= ro * w[i] * ga[i];
        }
    }
    s[0] = 0.0f;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const uint32_t ch = (k * TPR + lane) * 8;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[k][i] = __builtin_fmaf(g.alpha, x[k][i], o[k][i]);
            s[0] = __builtin_fmaf(x[k][i], x[k][i], s[0]);
        }
        if (g.y.p && live && ch < g.c) store8<T, AL>(g.y.p, row * g.y.ld, ch, g.c, x[k]);
    }
    if (!g.u.p) return;
    row_sum<TPR, 1>(s, &lds[1]);
    const float ry = __builtin_amdgcn_rsqf(__builtin_fmaf(s[0], inv_c, g.eps));
#pragma unroll
    for (int k = 0; k < K; k++) {
        const uint32_t ch = (k * TPR + lane) * 8;
        if (!live || ch >= g.c) continue;
        float w[8];
        weight8<T, AL>(g.w_pre, 0, ch, g.c, w);
#pragma unroll
        for (int i = 0; i < 8; i++) x[k][i] *= ry * w[i];
        store8<T, AL>(g.u.p, row * g.u.ld, ch, g.c, x[k]);
    }
}

// Backward. With n_o = o / rms(o), n_y = y / rms(y), z = gate * w_post * dY:
//     dY = dy + (w_pre du - n_y mean(w_pre du n_y)) / rms(y)
//     dx = alpha dY,   do = (z - n_o mean(z n_o)) / rms(o)
//     dgate = w_post * sum dY n_o,   dw_post = sum gate dY n_o,   dw_pre = sum du n_y
// mean(z n_o) is linear in dY, so its sum splits into three that need only o and y; they are taken together with
// those of y, and a row costs two exchanges in place of four.
//
// A workgroup (tpr threads a row, RPB rows at a time) owns the sums of its rows in registers. Where groups are long, a
// workgroup takes a part of one group (group = part / per_group), and its dY n_o sum is a partial sum of dgate; where
// they are short, every RPB-th group of a run of wg_groups is one slot's, which then writes dgate itself. dw_post and
// dw_pre leave one partial row a workgroup. norm_sum adds the partial rows in their order.
template <class T, int TPR, int K, bool AL>
__global__ __launch_bounds__(kBlock<TPR>) void norm_bwd(NormArgs g) {
    constexpr int RPB = kBlock<TPR> / TPR, NW = TPR > 64 ? TPR / 64 : 1;
    __shared__ float lds1[2][1][NW];
    __shared__ float lds5[2][5][NW];
    __shared__ float fold[RPB > 1 ? RPB * TPR * 8 : 1];
    const uint32_t lane = threadIdx.x % TPR, slot = threadIdx.x / TPR;
    const float inv_c = 1.0f / (float)g.c;
    const bool has_o = g.o.p != nullptr;
    float wp[K][8], wn[K][8], q[K][8], post[K][8], pre[K][8];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const uint32_t ch = (k * TPR + lane) * 8;
#pragma unroll
        for (int i = 0; i < 8; i++) wp[k][i] = wn[k][i] = q[k][i] = post[k][i] = pre[k][i] = 0.0f;
        if (ch < g.c) {
            weight8<T, AL>(g.w_post, 0, ch, g.c, wp[k]);
            weight8<T, AL>(g.w_pre, 0, ch, g.c, wn[k]);
        }
    }
    // the groups and rows of this slot: group g0, g0 + gstep, ... below g1; rows r0 + slot offset, + rstep, ... of each
    uint32_t g0, g1, gstep, first, rstep;
    uint32_t part = 0;
    if (g.per_group) {
        g0 = blockIdx.x / g.per_group, g1 = g0 + 1, gstep = 1;
        part = blockIdx.x - g0 * g.per_group;
        first = slot, rstep = RPB;
    } else {
        g0 = blockIdx.x * g.wg_groups + slot, g1 = min((blockIdx.x + 1) * g.wg_groups, g.groups), gstep = RPB;
        first = 0, rstep = 1;
    }
    // all slots of a workgroup make the same number of passes, so that barriers meet (rows of several waves have one
    // slot; the passes of slots within a wave may differ, and their lane exchanges stay inside the slot)
    uint32_t turn = 0;
    for (uint32_t gr = g0; gr < g1; gr += gstep) {
        float ga[K][8];
#pragma unroll
        for (int k = 0; k < K; k++) {
            const uint32_t ch = (k * TPR + lane) * 8;
#pragma unroll
            for (int i = 0; i < 8; i++) ga[k][i] = 0.0f;
            if (ch < g.c) weight8<T, AL>(g.gate, (int64_t)gr * g.c, ch, g.c, ga[k]);
        }
        const uint64_t base = (uint64_t)gr * g.rpg;
        const uint32_t in_group = (uint32_t)min((uint64_t)g.rpg, g.rows - base);
        const uint32_t lo = g.per_group ? part * g.part_rows : 0;
        const uint32_t hi = g.per_group ? min(lo + g.part_rows, in_group) : in_group;
        for (uint32_t r = lo + first; r < hi; r += rstep, turn ^= 1) {
            const int64_t row = (int64_t)(base + r);
            float x[K][8], o[K][8], dy[K][8], dn[K][8];
            float s1[1] = {0.0f}, s5[5] = {};
#pragma unroll
            for (int k = 0; k < K; k++) {
                const uint32_t ch = (k * TPR + lane) * 8;
#pragma unroll
                for (int i = 0; i < 8; i++) x[k][i] = o[k][i] = dy[k][i] = dn[k][i] = 0.0f;
                if (ch < g.c) {
                    load8<T, AL>(g.x.p, row * g.x.ld, ch, g.c, x[k]);
                    if (has_o) load8<T, AL>(g.o.p, row * g.o.ld, ch, g.c, o[k]);
                    if (g.dy.p) load8<T, AL>(g.dy.p, row * g.dy.ld, ch, g.c, dy[k]);
                    if (g.du.p) load8<T, AL>(g.du.p, row * g.du.ld, ch, g.c, dn[k]);
                }
            }
            float ro = 0.0f;
            if (has_o) {
#pragma unroll
                for (int k = 0; k < K; k++)
#pragma unroll
                    for (int i = 0; i < 8; i++) s1[0] = __builtin_fmaf(o[k][i], o[k][i], s1[0]);
                row_sum<TPR, 1>(s1, &lds1[turn]);
                ro = __builtin_amdgcn_rsqf(__builtin_fmaf(s1[0], inv_c, g.eps));
            }
#pragma unroll
            for (int k = 0; k < K; k++) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    o[k][i] *= ro;  // n_o
                    const float zo = ga[k][i] * wp[k][i] * o[k][i], w = wn[k][i] * dn[k][i];
                    x[k][i] = __builtin_fmaf(g.alpha, x[k][i], zo);  // y
                    s5[0] = __builtin_fmaf(x[k][i], x[k][i], s5[0]);
                    s5[1] = __builtin_fmaf(w, x[k][i], s5[1]);
                    s5[2] = __builtin_fmaf(zo, dy[k][i], s5[2]);
                    s5[3] = __builtin_fmaf(zo, w, s5[3]);
                    s5[4] = __builtin_fmaf(zo, x[k][i], s5[4]);
                }
            }
            row_sum<TPR, 5>(s5, &lds5[turn]);
            const float ry = __builtin_amdgcn_rsqf(__builtin_fmaf(s5[0], inv_c, g.eps));
            const float my = s5[1] * inv_c * ry * ry;                                      // mean(w du n_y) / rms(y)
            const float mo = (s5[2] + ry * s5[3] - ry * my * s5[4]) * inv_c;                // mean(z n_o)
#pragma unroll
            for (int k = 0; k < K; k++) {
                const uint32_t ch = (k * TPR + lane) * 8;
                float dx[8], dv[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float ny = x[k][i] * ry;
                    const float d = __builtin_fmaf(ry, wn[k][i] * dn[k][i], dy[k][i]) - ny * my;  // dY
                    dx[i] = g.alpha * d;
                    dv[i] = ro * (ga[k][i] * wp[k][i] * d - o[k][i] * mo);
                    q[k][i] = __builtin_fmaf(d, o[k][i], q[k][i]);
                    pre[k][i] = __builtin_fmaf(dn[k][i], ny, pre[k][i]);
                }
                if (ch < g.c) {
                    store8<T, AL>(g.dx.p, row * g.dx.ld, ch, g.c, dx);
                    if (has_o) store8<T, AL>(g.dout.p, row * g.dout.ld, ch, g.c, dv);
                }
            }
        }
        // a group (or this part of it) is done
#pragma unroll
        for (int k = 0; k < K; k++) {
            const uint32_t ch = (k * TPR + lane) * 8;
#pragma unroll
            for (int i = 0; i < 8; i++) post[k][i] = __builtin_fmaf(ga[k][i], q[k][i], post[k][i]);
            if (!g.per_group) {
                if (g.dgate && ch < g.c) {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (ch + i < g.c) g.dgate[(uint64_t)gr * g.c + ch + i] = wp[k][i] * q[k][i];
                }
#pragma unroll
                for (int i = 0; i < 8; i++) q[k][i] = 0.0f;
            }
        }
    }
    // the slots' sums of one workgroup, added in the slots' order by slot 0
    auto leave = [&](float (&v)[K][8], float* out) {
        if (!out) return;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const uint32_t ch = (k * TPR + lane) * 8;
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
            if (slot == 0 && ch < g.c) {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (ch + i < g.c) out[(uint64_t)blockIdx.x * g.c + ch + i] = v[k][i];
            }
        }
    };
    leave(pre, g.part_pre);
    leave(post, g.part_post);
    leave(q, g.part_gate);
}

// out[group][ch] = scale[ch] * the sum of `parts` partial rows of the group; 64 columns x 16 row lanes a workgroup
template <class T>
__global__ __launch_bounds__(1024) void norm_sum(const float* a, float* out_a, const float* b, float* out_b,
                                                 uint32_t parts, uint32_t c, const void* scale) {
    __shared__ double s[16][64];
    const uint32_t ch = blockIdx.x * 64 + (threadIdx.x & 63), y = threadIdx.x >> 6;
    const float* part = blockIdx.z ? b : a;
    float* out = blockIdx.z ? out_b : out_a;
    if (!out) return;
    double acc = 0.0;
    if (ch < c) {
#pragma unroll 8
        for (uint32_t r = y; r < parts; r += 16) acc += (double)part[((uint64_t)blockIdx.y * parts + r) * c + ch];
    }
    s[y][threadIdx.x & 63] = acc;
    __syncthreads();
    if (y == 0 && ch < c) {
#pragma unroll
        for (int k = 1; k < 16; k++) acc += s[k][threadIdx.x];
        if (scale) acc *= (double)widen(T{}, reinterpret_cast<const typename T::Raw*>(scale)[ch]);
        out[(uint64_t)blockIdx.y * c + ch] = (float)acc;
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
    if (r->ld < (int64_t)n->c) return fail(-1, "%s: rows of %s are %lld apart, below %u channels", op, name, (long long)r->ld, n->c);
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

uint32_t threads_of_row(uint32_t c) {  // 8 channels a thread, 16 a thread above 8192
    uint32_t t = 16;
    while (t < 1024 && t * 8 < c) t *= 2;
    return t;
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
        if (c > 8192) by_al(t, integral_constant<int, 1024>{}, integral_constant<int, 2>{});
        else if (tpr == 1024) by_al(t, integral_constant<int, 1024>{}, integral_constant<int, 1>{});
        else if (tpr == 512) by_al(t, integral_constant<int, 512>{}, integral_constant<int, 1>{});
        else if (tpr == 256) by_al(t, integral_constant<int, 256>{}, integral_constant<int, 1>{});
        else if (tpr == 128) by_al(t, integral_constant<int, 128>{}, integral_constant<int, 1>{});
        else if (tpr == 64) by_al(t, integral_constant<int, 64>{}, integral_constant<int, 1>{});
        else if (tpr == 32) by_al(t, integral_constant<int, 32>{}, integral_constant<int, 1>{});
        else by_al(t, integral_constant<int, 16>{}, integral_constant<int, 1>{});
    };
    if (dtype == FHC_F16) by_rows(F16{});
    else if (dtype == FHC_BF16) by_rows(BF16{});
    else by_rows(F32{});
}

struct Split {
    uint32_t tpr, rpb, groups, rpg, per_group, part_rows, wg_groups, wgs;
    size_t pre_at, post_at, gate_at, bytes;
};
// The backward pass's workgroups: about 4 rounds of 1024 threads a CU, at least 4 rows a slot where there are so many.
// Groups of at least 4 passes are cut into parts; shorter ones are taken whole.
Split split_of(const fhc_norm_desc* n) {
    Split s{};
    s.tpr = threads_of_row(n->c);
    const uint32_t block = s.tpr <= 64 ? 256 : s.tpr;
    s.rpb = block / s.tpr;
    s.rpg = n->gate ? n->rows_per_group : n->rows;
    if (s.rpg > n->rows) s.rpg = n->rows;
    if (s.rpg == 0) s.rpg = 1;
    s.groups = (uint32_t)ceil_div(n->rows, s.rpg);
    const uint32_t most = 256 * 1024 / block;
    if (s.groups && s.rpg >= 4 * s.rpb) {
        uint64_t per = ceil_div(most, s.groups);
        const uint64_t cap = ceil_div(s.rpg, 4 * s.rpb);
        if (per > cap) per = cap;
        s.part_rows = (uint32_t)ceil_div(s.rpg, per);
        s.per_group = (uint32_t)ceil_div(s.rpg, s.part_rows);
        s.wgs = s.groups * s.per_group;
    } else {
        s.wg_groups = (uint32_t)ceil_div(ceil_div(s.groups, most), s.rpb) * s.rpb;
        s.wgs = s.groups ? (uint32_t)ceil_div(s.groups, s.wg_groups) : 0;
    }
    const size_t one = (size_t)ceil_div((uint64_t)s.wgs * n->c * 4, 256) * 256;
    s.pre_at = 0, s.post_at = one, s.gate_at = 2 * one;
    s.bytes = (s.per_group ? 3 : 2) * one;
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
            constexpr int TPR = decltype(w)::value, block = kBlock<TPR>;
            hipLaunchKernelGGL((norm_fwd<decltype(t), TPR, decltype(k)::value, decltype(al)::value>),
                               dim3((uint32_t)ceil_div(n->rows, block / TPR)), dim3(block), 0, (hipStream_t)stream, a);
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
        a.part_pre = dw_pre ? reinterpret_cast<float*>(w + s.pre_at) : nullptr;
        a.part_post = dw_post ? reinterpret_cast<float*>(w + s.post_at) : nullptr;
        a.part_gate = dgate && s.per_group ? reinterpret_cast<float*>(w + s.gate_at) : nullptr;
        const hipStream_t st = (hipStream_t)stream;
        if (s.wgs) {
            with_shape(n->dtype, s.tpr, n->c, whole(n, {x, o, dy, du, dx, dout}), [&](auto t, auto tpr, auto k, auto al) {
                constexpr int TPR = decltype(tpr)::value, block = kBlock<TPR>;
                hipLaunchKernelGGL((norm_bwd<decltype(t), TPR, decltype(k)::value, decltype(al)::value>), dim3(s.wgs),
                                   dim3(block), 0, st, a);
            });
            FHC_TRY(launched(op));
        }
        const uint32_t blocks = (uint32_t)ceil_div(n->c, 64);
        if (dw_pre || dw_post) {
            hipLaunchKernelGGL((norm_sum<F32>), dim3(blocks, 1, 2), dim3(1024), 0, st, a.part_pre, dw_pre, a.part_post,
                               dw_post, s.wgs, n->c, (const void*)nullptr);
            FHC_TRY(launched(op));
        }
        if (a.part_gate && s.groups) {
            auto sum = n->dtype == FHC_F16 ? norm_sum<F16> : n->dtype == FHC_BF16 ? norm_sum<BF16> : norm_sum<F32>;
            for (uint32_t g = 0; g < s.groups; g += 65535) {  // the grid's limit
                const uint32_t m = s.groups - g < 65535 ? s.groups - g : 65535;
                hipLaunchKernelGGL(sum, dim3(blocks, m, 1), dim3(1024), 0, st,
                                   a.part_gate + (uint64_t)g * s.per_group * n->c, dgate + (uint64_t)g * n->c,
                                   (const float*)nullptr, (float*)nullptr, s.per_group, n->c, n->w_post);
                FHC_TRY(launched(op));
            }
        }
        return 0;
    });
}
