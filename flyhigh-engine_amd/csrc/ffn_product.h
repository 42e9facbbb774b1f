// The launches around the products of ffn_gemm.h, shared by the feed-forward block and the product with its epilogue
// (include/fhc_seq.h): the join of a split K, copies of operands that cannot be fetched as they lie, the products of few
// rows, and the choice of tiles.
#pragma once
#include "ffn_gemm.h"

namespace fhc {
namespace seq {
namespace {

// out = the sum of the splits' partial sums (LIN: with the product's tail); LANES threads take every LANES-th split of a quad
// of columns each, and their sums are added in order
template <class T, int LANES, bool LIN>
__global__ __launch_bounds__(256) void ffn_join(const float* part, int splits, int m, int n, int64_t ldpart,
                                                uint16_t* o0, uint16_t* o1, int64_t ldo, Tail tail) {
    constexpr int Q = 256 / LANES;
    __shared__ f4 s[LANES > 1 ? LANES : 1][LANES > 1 ? Q : 1];
    const int quads = (n + 3) / 4, x = threadIdx.x % Q, y = threadIdx.x / Q;
    const int64_t at = (int64_t)blockIdx.x * Q + x;
    const bool live = at < (int64_t)m * quads;
    const int64_t row = live ? at / quads : 0;
    const int c = live ? (int)(at - row * quads) * 4 : 0;
    const float* p = part + ((int64_t)blockIdx.y * splits * m + row) * ldpart + c;
    f4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (live) {
#pragma unroll 4
        for (int z = y; z < splits; z += LANES) sum += *reinterpret_cast<const f4*>(p + (int64_t)z * m * ldpart);
    }
    if constexpr (LANES > 1) {
        s[y][x] = sum;
        __syncthreads();
        if (y > 0) return;
#pragma unroll
        for (int k = 1; k < LANES; k++) sum += s[k][x];
    }
    if (!live) return;
    uint16_t q[4];
    if constexpr (LIN) {
        tail4<T>(tail, row, c, n - c, sum, q);
    } else {
#pragma unroll
        for (int r = 0; r < 4; r++) q[r] = narrow(T{}, sum[r]);
    }
    store4((blockIdx.y ? o1 : o0) + row * ldo + c, n - c, q);
}

// Copies of up to five matrices with rows of up8(width) elements, the last ones zeros: 8 elements a thread.
struct PackArgs {
    const uint16_t* in[5];
    uint16_t* out[5];
    int64_t ld[5];
    int rows[5], width[5];
};
__global__ __launch_bounds__(256) void ffn_pack(PackArgs g) {
    const uint16_t* in = g.in[blockIdx.y];
    uint16_t* out = g.out[blockIdx.y];
    const int width = g.width[blockIdx.y], groups = (width + 7) / 8;
    const int64_t items = (int64_t)g.rows[blockIdx.y] * groups, ld = g.ld[blockIdx.y];
    for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < items; k += (int64_t)gridDim.x * 256) {
        const int64_t row = k / groups;
        const int c = (int)(k - row * groups) * 8;
        *reinterpret_cast<u4_t*>(out + k * 8) = load_some(in + row * ld + c, width - c);
    }
}

// ---- few rows: a wave streams weight rows past the matrix unit straight from global memory (each weight is used once,
// so LDS would only add a step), NB blocks of 16 token rows as the other operand; the NW waves of a workgroup split K and
// add their sums in LDS in the waves' order. GLU: 16 rows of wg and of wu. Else the 16 rows that the unit takes are 8
// weight rows twice, at the two halves of K, each half with its own token fragment (the other half's result is left):
// twice the workgroups and half the steps, where the second product has few columns to spread over the chip.
struct SkinnyArgs {
    const uint16_t *x, *w0, *w1;
    int64_t ldx, ldw;
    int rows, n, k;
    uint16_t* out;
    int64_t ldo;
    int width;  // columns of out that are written, zeros from n on
    float *pre_g, *pre_u;  // GLU: both products, rows of ldo, or null
    uint32_t act;
    Tail tail;  // LIN
};

// 8 elements from k on, all of them inside
template <bool AL>
__device__ __forceinline__ u4_t load_k(const uint16_t* row, int k) {
    if constexpr (AL) return *reinterpret_cast<const u4_t*>(row + k);
    else return load_some(row + k, 8);
}

template <class T, bool GLU, int NB, int NW, bool AL, bool LIN>
__global__ __launch_bounds__(64 * NW) void ffn_skinny(SkinnyArgs g) {
    constexpr int ROWS = GLU ? 16 : 8;
    __shared__ f4 sums[NW][2 * NB][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int f0 = blockIdx.x * ROWS, f = min(f0 + (lane & (ROWS - 1)), g.n - 1);  // a row past the end: the last one again
    const int kl = 8 * (lane >> 4);
    const int all = (g.k + 31) / 32, steps = GLU ? all : (all + 1) / 2, per = (steps + NW - 1) / NW;
    const int s0 = wave * per, s1 = min(steps, s0 + per);
    const int half = steps * 32, wk = kl + (GLU ? 0 : (lane >> 3 & 1) * half);  // the lane's k of step 0, weights
    const uint16_t* w0 = g.w0 + (int64_t)f * g.ldw;
    const uint16_t* w1 = GLU ? g.w1 + (int64_t)f * g.ldw : nullptr;
    const uint16_t* x[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) x[b] = g.x + (int64_t)min(b * 16 + (lane & 15), g.rows - 1) * g.ldx;
    f4 acc[2][NB];  // gate and up; or the halves of K
#pragma unroll
    for (int p = 0; p < 2; p++)
#pragma unroll
        for (int b = 0; b < NB; b++) acc[p][b] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int U = 8;  // steps whose loads are in flight together
    auto multiply = [&](u4_t wa, u4_t wb, const u4_t (&v)[NB], const u4_t (&v2)[NB]) {
#pragma unroll
        for (int b = 0; b < NB; b++) {
            acc[0][b] = mfma16(T{}, wa, v[b], acc[0][b]);
            acc[1][b] = mfma16(T{}, wb, v2[b], acc[1][b]);
        }
    };
    const int full = (g.k - (GLU ? 0 : half)) / 32;  // the last steps may be cut, and of the second half missing
    int s = s0;
    for (; s + U <= min(s1, full); s += U) {
        u4_t w[U][2], v[U][NB], v2[U][GLU ? 1 : NB];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k = (s + u) * 32;
            w[u][0] = load_k<AL>(w0, k + wk);
            if constexpr (GLU) w[u][1] = load_k<AL>(w1, k + wk);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                v[u][b] = load_k<AL>(x[b], k + kl);
                if constexpr (!GLU) v2[u][b] = load_k<AL>(x[b], k + half + kl);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if constexpr (GLU) multiply(w[u][0], w[u][1], v[u], v[u]);
            else multiply(w[u][0], w[u][0], v[u], v2[u]);
        }
    }
    for (; s < s1; s++) {
        const int k = s * 32;
        u4_t wa = load_some(w0 + k + wk, g.k - k - wk), wb, v[NB], v2[NB];
        if constexpr (GLU) wb = load_some(w1 + k + wk, g.k - k - wk);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            v[b] = load_some(x[b] + k + kl, g.k - k - kl);
            if constexpr (!GLU) v2[b] = load_some(x[b] + k + half + kl, g.k - k - half - kl);
        }
        if constexpr (GLU) multiply(wa, wb, v, v);
        else multiply(wa, wa, v, v2);
    }
#pragma unroll
    for (int p = 0; p < 2; p++)
#pragma unroll
        for (int b = 0; b < NB; b++) sums[wave][p * NB + b][lane] = acc[p][b];
    __syncthreads();
    // wave b finishes token block b (f0 + 4 (lane >> 4) + r of row b * 16 + (lane & 15))
    for (int b = wave; b < NB; b += NW) {
        f4 t[2] = {f4{0.0f, 0.0f, 0.0f, 0.0f}, f4{0.0f, 0.0f, 0.0f, 0.0f}};
        for (int w = 0; w < NW; w++) {
            t[0] += sums[w][b][lane];
            t[1] += sums[w][NB + b][GLU ? lane : (lane + 32) & 63];  // the second half's rows are the unit's 8 to 15
        }
        const int row = b * 16 + (lane & 15), at = f0 + 4 * (lane >> 4);
        if (row >= g.rows || at >= g.width || (!GLU && lane >= 32)) continue;
        uint16_t q[4];
        if constexpr (LIN) {
            tail4<T>(g.tail, row, at, g.width - at, t[0] + t[1], q);
            store4(g.out + row * g.ldo + at, g.width - at, q);
            continue;
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
            if (GLU && at + r >= g.n) t[0][r] = t[1][r] = 0.0f;
            q[r] = narrow(T{}, GLU ? act_of(g.act, t[0][r]) * t[1][r] : t[0][r] + t[1][r]);
        }
        store4(g.out + row * g.ldo + at, g.width - at, q);
        if (GLU && g.pre_g) {
            *reinterpret_cast<f4*>(g.pre_g + row * g.ldo + at) = t[0];
            *reinterpret_cast<f4*>(g.pre_u + row * g.ldo + at) = t[1];
        }
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------

constexpr uint32_t kSkinnyRows = 32;  // up to here the weights' bytes are all that counts

inline int check_rows(const char* op, const char* name, const fhc_rows* r, uint32_t c) {
    if (!r) return fail(-1, "%s: null %s", op, name);
    if (!r->p) return fail(-1, "%s: null pointer of %s", op, name);
    if (r->ld < (int64_t)c)
        return fail(-1, "%s: rows of %s are %lld apart, below %u channels", op, name, (long long)r->ld, c);
    if (!aligned(r->p, 2)) return fail(-1, "%s: %s is not aligned to its elements", op, name);
    return 0;
}
inline int check_weight(const char* op, const char* name, const void* p) {
    if (!p) return fail(-1, "%s: null %s", op, name);
    if (!aligned(p, 2)) return fail(-1, "%s: %s is not aligned to its elements", op, name);
    return 0;
}

inline size_t up256(size_t n) { return (n + 255) / 256 * 256; }

enum Tile { kNarrow, kMedium, kLarge };  // 128 x 64, 128 x 128, 256 x 256
struct Shape {  // a product's tiles and splits
    Tile tile;
    int tiles_m, tiles_n, slabs, per_split, splits;
    size_t part_bytes;
};
// The tile whose workgroups, a round of 256 at a time, take the least: a medium tile's slab counts 100, a narrow one's 75
// and a large one's 270 (of 50 and 400 by area: the wider the tile, the less LDS traffic a product). Where K may be split
// and there are at most 128 medium tiles, it is split to one workgroup a CU, at least 8 slabs each. Training steps, us,
// bf16, with narrow, medium, large tiles for every product that is not split, and by the rule:
//   8192 x 2048, f 8192   4401  3074  2234  large throughout
//   4096 x 1024, f 4096    546   470   629   458
//   1024 x 1024, f 4096    150   143   202   141
inline Shape shape_of(int64_t m, int64_t n, int64_t k, int segments, int pairs, bool glu, bool may_split) {
    Shape s{};
    const int unit = glu ? 2 : 1;
    const int64_t bm[3] = {128, 128, 256}, bn[3] = {64, 128, 256}, cost[3] = {75, 100, 270};
    auto count = [&](int t) { return (int64_t)(ceil_div(m, bm[t]) * ceil_div(n, bn[t] / unit)) * pairs; };
    s.tile = kMedium;
    const int64_t medium = count(kMedium);  // none where there are no rows or no columns
    const bool split = may_split && medium > 0 && medium <= 128 && ceil_div(k, 32) * segments >= 16;
    if (!split) {
        int64_t best = 0;
        for (int t = 0; t < 3; t++) {
            const int64_t time = (int64_t)ceil_div(count(t), 256) * cost[t];
            if (t == 0 || time < best) best = time, s.tile = (Tile)t;
        }
    }
    s.tiles_m = (int)ceil_div(m, bm[s.tile]), s.tiles_n = (int)ceil_div(n, bn[s.tile] / unit);
    s.slabs = (int)ceil_div(k, 32) * segments;
    s.splits = 1;
    const int64_t wgs = (int64_t)s.tiles_m * s.tiles_n * pairs;
    if (split) {
        int64_t z = 256 / wgs;
        if (z > s.slabs / 8) z = s.slabs / 8;
        s.splits = z < 1 ? 1 : (int)z;
    }
    s.per_split = (int)ceil_div(s.slabs, s.splits);
    s.splits = s.slabs ? (int)ceil_div(s.slabs, s.per_split) : 1;
    s.part_bytes = s.splits > 1 ? up256((size_t)pairs * s.splits * m * ((n + 3) / 4 * 4) * 4) : 0;
    return s;
}

// A matrix of a product as it can be fetched: itself, or a copy with padded rows.
struct Operands {
    PackArgs args;
    int count;
    char* at;  // the workspace's next byte
    // rows x width elements ld apart; k: the width is a product's K
    bool direct(const void* p, int64_t ld, int64_t width, bool k) const {
        return ld % 2 == 0 && width % (k ? 8 : 2) == 0 && ld <= 1 << 20 && aligned(p, 4);
    }
    const uint16_t* take(const void* p, int64_t& ld, uint32_t rows, uint32_t width, bool k, bool copied = false) {
        const uint16_t* q = static_cast<const uint16_t*>(p);
        if (!copied && direct(p, ld, width, k)) return q;
        args.in[count] = q, args.ld[count] = ld, args.rows[count] = (int)rows, args.width[count] = (int)width;
        args.out[count] = reinterpret_cast<uint16_t*>(at);
        at += pack_bytes(rows, width);
        ld = up8(width);
        return args.out[count++];
    }
    // two matrices of one shape, which a product reads with one stride: both as they are or both copied
    void take_two(const void* p, const void* q, int64_t& ld, uint32_t rows, uint32_t width, bool k, const uint16_t*& a,
                  const uint16_t*& b) {
        const bool copied = !direct(p, ld, width, k) || !direct(q, ld, width, k);
        int64_t other = ld;
        a = take(p, other, rows, width, k, copied), b = take(q, ld, rows, width, k, copied);
    }
    static size_t pack_bytes(uint32_t rows, uint32_t width) { return up256((size_t)rows * up8(width) * 2); }
    int copy(const char* op, hipStream_t st) const {
        if (!count) return 0;
        uint64_t items = 1;
        for (int i = 0; i < count; i++) {
            const uint64_t n = (uint64_t)args.rows[i] * ((args.width[i] + 7) / 8);
            items = n > items ? n : items;
        }
        const uint64_t blocks = ceil_div(items, 256);
        hipLaunchKernelGGL(ffn_pack, dim3((uint32_t)(blocks < 4096 ? blocks : 4096), count), dim3(256), 0, st, args);
        return launched(op);
    }
};

template <class T, bool AC, bool BC, Epi E>
void launch_tiles(const Shape& s, const GemmArgs& g, hipStream_t st) {
    const dim3 grid(s.tiles_m * s.tiles_n, 1, s.splits * g.pairs);
    if constexpr (E != kPart) {  // a split K has medium tiles
        if (s.tile == kLarge) {
            hipLaunchKernelGGL((ffn_gemm<T, AC, BC, E, 8, 4, 2, 4>), grid, dim3(512), 0, st, g);
            return;
        }
        if (s.tile == kNarrow) {
            hipLaunchKernelGGL((ffn_gemm<T, AC, BC, E, 4, 2, 2, 2>), grid, dim3(256), 0, st, g);
            return;
        }
    }
    hipLaunchKernelGGL((ffn_gemm<T, AC, BC, E, 4, 4, 2, 2>), grid, dim3(256), 0, st, g);
}

// g without tiles and splits
template <class T, bool AC, bool BC, Epi E>
int product(const char* op, GemmArgs g, float* part, hipStream_t st) {
    if (g.m == 0 || g.n == 0) return 0;
    g.segments = g.segments ? g.segments : 1, g.pairs = g.pairs ? g.pairs : 1;
    const Shape s = shape_of(g.m, g.n, g.k, g.segments, g.pairs, E == kGlu, E == kStore || E == kLinear);
    g.tiles_m = s.tiles_m, g.tiles_n = s.tiles_n, g.slabs = s.slabs, g.per_split = s.per_split, g.splits = s.splits;
    // The columns that the last row of a column operand is read to. The range check goes by 4 bytes, so an odd width needs
    // one more: an operand of odd width has padded rows (Operands::direct). An even one may be a caller's view that ends
    // with its buffer, whatever its stride: not an element more.
    g.wide_m = g.m + (g.m & 1), g.wide_n = g.n + (g.n & 1);
    if ((int64_t)s.tiles_m * s.tiles_n >= 1ll << 31) return fail(-1, "%s: too many tiles", op);
    g.quads = g.n % 4 == 0 && g.ldo % 4 == 0 && g.ldo <= 1 << 21 && aligned(g.o0, 8) && aligned(g.o1, 8) &&
              g.ldr % 4 == 0 && g.ldr <= 1 << 21 && aligned(g.res, 8);
    g.dwords = g.n % 2 == 0 && g.ldo % 2 == 0 && g.ldo <= 1 << 21 && aligned(g.o0, 4) && g.ldr % 2 == 0 &&
               g.ldr <= 1 << 21 && aligned(g.res, 4);
    if constexpr (E == kStore || E == kLinear) {
        constexpr bool LIN = E == kLinear;
        const Tail tail{g.bias, g.res, g.ldr, g.pre_g, g.ldpre, g.act};
        if (s.splits > 1) {
            g.part = part, g.ldpart = ((int64_t)g.n + 3) / 4 * 4;
            launch_tiles<T, AC, BC, kPart>(s, g, st);
            FHC_TRY(launched(op));
            const uint64_t items = (uint64_t)g.m * ((g.n + 3) / 4);
            if (s.splits >= 16)
                hipLaunchKernelGGL((ffn_join<T, 8, LIN>), dim3((uint32_t)ceil_div(items, 32), g.pairs), dim3(256), 0, st,
                                   g.part, s.splits, g.m, g.n, g.ldpart, g.o0, g.o1, g.ldo, tail);
            else
                hipLaunchKernelGGL((ffn_join<T, 1, LIN>), dim3((uint32_t)ceil_div(items, 256), g.pairs), dim3(256), 0, st,
                                   g.part, s.splits, g.m, g.n, g.ldpart, g.o0, g.o1, g.ldo, tail);
            return launched(op);
        }
    }
    launch_tiles<T, AC, BC, E>(s, g, st);
    return launched(op);
}

template <class T, bool GLU, bool LIN>
int skinny(const char* op, const SkinnyArgs& a, hipStream_t st) {
    if (a.n == 0) return 0;
    const dim3 grid((uint32_t)ceil_div(a.n, GLU ? 16 : 8));
    // a whole step's loads are 16-byte aligned (the second half of K starts at a multiple of 32)
    const bool al = a.k % 8 == 0 && a.ldx % 8 == 0 && a.ldw % 8 == 0 && aligned(a.x, 16) && aligned(a.w0, 16) &&
                    aligned(a.w1, 16);
#define SKINNY_OF(NB, NW)                                                                                       \
    do {                                                                                                        \
        if (al) hipLaunchKernelGGL((ffn_skinny<T, GLU, NB, NW, true, LIN>), grid, dim3(64 * NW), 0, st, a);     \
        else hipLaunchKernelGGL((ffn_skinny<T, GLU, NB, NW, false, LIN>), grid, dim3(64 * NW), 0, st, a);       \
    } while (0)
// Few waves a workgroup where there are many of them, which then all run at once: LIN, bf16, us with 16 and with 4 waves:
// 4 x 2048 -> 8192 (1024 workgroups) 15, 11; 32 x 2048 -> 8192 30, 23; 4 x 4096 -> 4096 (512) 14, 12; 4 x 8192 -> 4096
// 21, 22; 4 x 8192 -> 2048 (256) 12, 14.
#define SKINNY(NB)                                                \
    do {                                                          \
        if constexpr (GLU) SKINNY_OF(NB, 4);                      \
        else if constexpr (!LIN) SKINNY_OF(NB, 16);               \
        else if (grid.x >= 512) SKINNY_OF(NB, 4);                 \
        else SKINNY_OF(NB, 16);                                   \
    } while (0)
    if (a.rows <= 16) SKINNY(1);
    else SKINNY(2);
#undef SKINNY
#undef SKINNY_OF
    return launched(op);
}

inline size_t part_of(int64_t m, int64_t n, int64_t k, int segments, int pairs) {
    return shape_of(m, n, k, segments, pairs, false, true).part_bytes;
}

}  // namespace
}  // namespace seq
}  // namespace fhc
