// The gated feed-forward block (include/fhc_seq.h): the launches around the products of ffn_gemm.h, and the products
// of few rows.
//
// Forward: one product with gate and up rows side by side whose epilogue is the activation and the product, one with
// wd. Backward: dh = dy wd with dL/dgate, dL/dup in its epilogue; dx = [dL/dgate dL/dup] [wg; wu] as one product over
// both halves of K; dwg and dwu (one launch), dwd, with the rows as K.
#include "ffn_fused.h"

namespace fhc {
namespace seq {
namespace {

// out = the sum of the splits' partial sums; LANES threads take every LANES-th split of a quad of columns each, and their
// sums are added in order
template <class T, int LANES>
__global__ __launch_bounds__(256) void ffn_join(const float* part, int splits, int m, int n, int64_t ldpart,
                                                uint16_t* o0, uint16_t* o1, int64_t ldo) {
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
#pragma unroll
    for (int r = 0; r < 4; r++) q[r] = narrow(T{}, sum[r]);
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
};

// 8 elements from k on, all of them inside
template <bool AL>
__device__ __forceinline__ u4_t load_k(const uint16_t* row, int k) {
    if constexpr (AL) return *reinterpret_cast<const u4_t*>(row + k);
    else return load_some(row + k, 8);
}

template <class T, bool GLU, int NB, int NW, bool AL>
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

// One kernel a direction (ffn_fused.h) where the channels fit its registers and the rows give it work for the chip: a
// workgroup has 128 rows and walks all features, so the time hardly changes until the rows fill the CUs, where the
// products of ffn_gemm.h spread few rows over features too. Measured, f16, us of one kernel, of products:
//                     rows  forward   training step
//   c  64, f  512     3000   16,  15    75,  58
//                     6000   16,  18    76,  67
//                    12000   16,  25    76,  85
//   c 128, f  512     6000   22,  20    93,  75
//                    11500   22,  30    97,  96
//                    20000   23,  25   105, 121
//   c 256, f 1024    10000   65,  35   242, 149
//                    19500   67,  62   273, 286
//                    32768   72,  81   339, 448
//                    40000  131, 103   550, 532
//                   131072  275, 312  1481, 1523
// Above 128 channels a CU holds one workgroup, so 32768 rows are a round and a few rows more cost another one: from 26000
// rows up, steps of c 160 to 256 and f 512 to 2048 took 0.72 to 1.04 of the products' time, bar 40000 rows with f 2048,
// 1.12 to 1.19; forward 0.86 to 1.23, and 1.2 to 1.68 at 40000. There the step without a hidden layer in memory is what
// the rule is for. f moves the crossing: c 32, f 128 is ahead from below 3000 rows (9, 12 and 37, 42); a forward of
// c 128, f 2048 from 20000 (75, 77), its step from 11500 (276, 291). One rule for both passes and with or without states
// kept, so that serving gives a training forward's bits; it follows the step.
bool fused(const fhc_ffn_desc* d) {
    return d->c > 0 && d->f > 0 && d->c <= 256 && d->rows >= (d->c <= 64 ? 6000u : d->c <= 128 ? 11500u : 19500u);
}

int check_desc(const char* op, const fhc_ffn_desc* d) {
    if (!d) return fail(-1, "%s: null descriptor", op);
    if (d->dtype > FHC_BF16) return fail(-1, "%s: dtype %u is neither f16 nor bf16", op, d->dtype);
    if (d->act > FHC_ACT_GELU) return fail(-1, "%s: act %u", op, d->act);
    if (d->c > 1u << 20 || d->f > 1u << 20) return fail(-1, "%s: %u x %u channels, at most 2^20", op, d->c, d->f);
    if (d->rows > 0x7FFFFF00u) return fail(-1, "%s: %u rows", op, d->rows);
    return 0;
}
int check_rows(const char* op, const char* name, const fhc_rows* r, uint32_t c) {
    if (!r) return fail(-1, "%s: null %s", op, name);
    if (!r->p) return fail(-1, "%s: null pointer of %s", op, name);
    if (r->ld < (int64_t)c)
        return fail(-1, "%s: rows of %s are %lld apart, below %u channels", op, name, (long long)r->ld, c);
    if (!aligned(r->p, 2)) return fail(-1, "%s: %s is not aligned to its elements", op, name);
    return 0;
}
int check_weight(const char* op, const char* name, const void* p) {
    if (!p) return fail(-1, "%s: null %s", op, name);
    if (!aligned(p, 2)) return fail(-1, "%s: %s is not aligned to its elements", op, name);
    return 0;
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }
size_t hidden_bytes(const fhc_ffn_desc* d) { return up256((size_t)d->rows * up8(d->f) * 2); }
size_t pre_bytes(const fhc_ffn_desc* d) { return up256((size_t)d->rows * up8(d->f) * 4); }

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
Shape shape_of(int64_t m, int64_t n, int64_t k, int segments, int pairs, bool glu, bool may_split) {
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
    const Shape s = shape_of(g.m, g.n, g.k, g.segments, g.pairs, E == kGlu, E == kStore);
    g.tiles_m = s.tiles_m, g.tiles_n = s.tiles_n, g.slabs = s.slabs, g.per_split = s.per_split, g.splits = s.splits;
    // The columns that the last row of a column operand is read to. The range check goes by 4 bytes, so an odd width needs
    // one more: an operand of odd width has padded rows (Operands::direct). An even one may be a caller's view that ends
    // with its buffer, whatever its stride: not an element more.
    g.wide_m = g.m + (g.m & 1), g.wide_n = g.n + (g.n & 1);
    if ((int64_t)s.tiles_m * s.tiles_n >= 1ll << 31) return fail(-1, "%s: too many tiles", op);
    g.quads = g.n % 4 == 0 && g.ldo % 4 == 0 && g.ldo <= 1 << 21 && aligned(g.o0, 8) && aligned(g.o1, 8);
    if constexpr (E == kStore) {
        if (s.splits > 1) {
            g.part = part, g.ldpart = ((int64_t)g.n + 3) / 4 * 4;
            launch_tiles<T, AC, BC, kPart>(s, g, st);
            FHC_TRY(launched(op));
            const uint64_t items = (uint64_t)g.m * ((g.n + 3) / 4);
            if (s.splits >= 16)
                hipLaunchKernelGGL((ffn_join<T, 8>), dim3((uint32_t)ceil_div(items, 32), g.pairs), dim3(256), 0, st,
                                   g.part, s.splits, g.m, g.n, g.ldpart, g.o0, g.o1, g.ldo);
            else
                hipLaunchKernelGGL((ffn_join<T, 1>), dim3((uint32_t)ceil_div(items, 256), g.pairs), dim3(256), 0, st,
                                   g.part, s.splits, g.m, g.n, g.ldpart, g.o0, g.o1, g.ldo);
            return launched(op);
        }
    }
    launch_tiles<T, AC, BC, E>(s, g, st);
    return launched(op);
}

template <class T, bool GLU>
int skinny(const char* op, const SkinnyArgs& a, hipStream_t st) {
    if (a.n == 0) return 0;
    constexpr int NW = GLU ? 4 : 16;
    const dim3 grid((uint32_t)ceil_div(a.n, GLU ? 16 : 8));
    // a whole step's loads are 16-byte aligned (the second half of K starts at a multiple of 32)
    const bool al = a.k % 8 == 0 && a.ldx % 8 == 0 && a.ldw % 8 == 0 && aligned(a.x, 16) && aligned(a.w0, 16) &&
                    aligned(a.w1, 16);
#define SKINNY(NB)                                                                                              \
    do {                                                                                                        \
        if (al) hipLaunchKernelGGL((ffn_skinny<T, GLU, NB, NW, true>), grid, dim3(64 * NW), 0, st, a);          \
        else hipLaunchKernelGGL((ffn_skinny<T, GLU, NB, NW, false>), grid, dim3(64 * NW), 0, st, a);            \
    } while (0)
    if (a.rows <= 16) SKINNY(1);
    else SKINNY(2);
#undef SKINNY
    return launched(op);
}

template <class T, bool BWD>
int run_fused(const char* op, const FusedArgs& a, hipStream_t st) {
#define FUSED(CP, MB, NW)                                                                                    \
    hipLaunchKernelGGL((ffn_fused<T, CP, MB, NW, BWD>), dim3((uint32_t)ceil_div(a.rows, 16 * MB * NW)), dim3(64 * NW), \
                       0, st, a)
    if (a.c <= 64) FUSED(64, 2, 4);
    else if (a.c <= 128) FUSED(128, 2, 4);
    else FUSED(256, 1, 8);
#undef FUSED
    return launched(op);
}

size_t part_of(int64_t m, int64_t n, int64_t k, int segments, int pairs) {
    return shape_of(m, n, k, segments, pairs, false, true).part_bytes;
}

// Copies of the operands are counted whether a call makes them or not: that depends on its pointers and strides.
size_t workspace(const fhc_ffn_desc* d, bool backward) {
    const size_t rows = Operands::pack_bytes(d->rows, d->c), up = Operands::pack_bytes(d->f, d->c),
                 down = Operands::pack_bytes(d->c, d->f);
    if (!backward) {  // h, where nothing is kept, and the second product's partial sums; in one kernel neither is made
        const size_t copies = d->rows > kSkinnyRows ? rows + 2 * up + down : 0;
        if (fused(d)) return copies;
        return hidden_bytes(d) + part_of(d->rows, d->c, d->f, 1, 1) + copies;
    }
    size_t part = 0;
    for (const size_t n : {part_of(d->rows, d->c, d->f, 2, 1), part_of(d->f, d->c, d->rows, 1, 2),
                           part_of(d->f, d->c, d->rows, 1, 1), part_of(d->c, d->f, d->rows, 1, 1)})
        part = n > part ? n : part;
    return (fused(d) ? 3 : 2) * hidden_bytes(d) + part + 2 * rows + 2 * up + down;
}

template <class T>
int forward(const char* op, const fhc_ffn_desc* d, const fhc_rows* x, const void* wg, const void* wu, const void* wd,
            const fhc_rows* y, void* saved, void* ws, hipStream_t st) {
    const int64_t fp = up8(d->f);
    char* keep = static_cast<char*>(saved);
    char* w = static_cast<char*>(ws);
    uint16_t* h = reinterpret_cast<uint16_t*>(saved ? keep : w);
    auto u16 = [](const void* p) { return static_cast<const uint16_t*>(p); };
    float* pre_g = saved ? reinterpret_cast<float*>(keep + hidden_bytes(d)) : nullptr;
    float* pre_u = saved ? reinterpret_cast<float*>(keep + hidden_bytes(d) + pre_bytes(d)) : nullptr;
    if (d->rows <= kSkinnyRows) {
        SkinnyArgs a{u16(x->p), u16(wg), u16(wu), x->ld, (int64_t)d->c, (int)d->rows, (int)d->f, (int)d->c, h, fp, (int)fp,
                     pre_g, pre_u, d->act};
        FHC_TRY((skinny<T, true>(op, a, st)));
        SkinnyArgs b{h, u16(wd), nullptr, fp, (int64_t)d->f, (int)d->rows, (int)d->c, (int)d->f,
                     static_cast<uint16_t*>(y->p), y->ld, (int)d->c, nullptr, nullptr, d->act};
        return skinny<T, false>(op, b, st);
    }
    if (fused(d)) {
        Operands o{{}, 0, w};
        FusedArgs a{};
        a.ldx = x->ld, a.ldg = d->c, a.ldd = d->f, a.rows = (int)d->rows, a.c = (int)d->c, a.f = (int)d->f, a.act = d->act;
        a.x = o.take(x->p, a.ldx, d->rows, d->c, true);
        o.take_two(wg, wu, a.ldg, d->f, d->c, true, a.wg, a.wu);
        a.wd = o.take(wd, a.ldd, d->c, d->f, true);
        FHC_TRY(o.copy(op, st));
        a.out = static_cast<uint16_t*>(y->p), a.ldo = y->ld;
        return run_fused<T, false>(op, a, st);
    }
    char* part = w + hidden_bytes(d);
    Operands o{{}, 0, part + part_of(d->rows, d->c, d->f, 1, 1)};
    GemmArgs g{}, p{};
    g.lda = x->ld, g.ldb = d->c, p.ldb = d->f;
    g.a0 = o.take(x->p, g.lda, d->rows, d->c, true);
    o.take_two(wg, wu, g.ldb, d->f, d->c, true, g.b0, g.b1);
    p.b0 = o.take(wd, p.ldb, d->c, d->f, true);
    FHC_TRY(o.copy(op, st));
    g.m = d->rows, g.n = d->f, g.k = d->c, g.o0 = h, g.ldo = fp, g.ldpre = fp, g.act = d->act;
    g.pre_g = pre_g, g.pre_u = pre_u;
    FHC_TRY((product<T, false, false, kGlu>(op, g, nullptr, st)));
    p.a0 = h, p.lda = fp, p.m = d->rows, p.n = d->c, p.k = d->f;
    p.o0 = static_cast<uint16_t*>(y->p), p.ldo = y->ld;
    return product<T, false, false, kStore>(op, p, reinterpret_cast<float*>(part), st);
}

template <class T>
int backward(const char* op, const fhc_ffn_desc* d, const fhc_rows* x, const void* wg, const void* wu, const void* wd,
             const void* saved, const fhc_rows* dy, const fhc_rows* dx, void* dwg, void* dwu, void* dwd, void* ws,
             hipStream_t st) {
    const int64_t fp = up8(d->f);
    char* keep = const_cast<char*>(static_cast<const char*>(saved));
    char* w = static_cast<char*>(ws);
    auto out = [](void* p) { return static_cast<uint16_t*>(p); };
    const bool one = fused(d);
    uint16_t *dg = out(w), *du = out(w + hidden_bytes(d));
    const uint16_t* h = reinterpret_cast<const uint16_t*>(one ? w + 2 * hidden_bytes(d) : keep);
    float* part = reinterpret_cast<float*>(w + (one ? 3 : 2) * hidden_bytes(d));
    Operands o{{}, 0, w + workspace(d, true) - 2 * Operands::pack_bytes(d->rows, d->c) -
                          2 * Operands::pack_bytes(d->f, d->c) - Operands::pack_bytes(d->c, d->f)};
    int64_t ldx = x->ld, ldy = dy->ld, ldd = d->f, ldg = d->c;
    const bool hidden = one || dx || dwg || dwu;
    // dy is a product's rows for dL/dh (K its channels) and columns for dwd
    const uint16_t* vdy = hidden || dwd ? o.take(dy->p, ldy, d->rows, d->c, hidden) : nullptr;
    const uint16_t* vx = one || dwg || dwu ? o.take(x->p, ldx, d->rows, d->c, one) : nullptr;
    const uint16_t* vwd = hidden ? o.take(wd, ldd, d->c, d->f, one) : nullptr;
    const uint16_t *vwg = nullptr, *vwu = nullptr;
    if (one || dx) o.take_two(wg, wu, ldg, d->f, d->c, one, vwg, vwu);
    FHC_TRY(o.copy(op, st));
    if (one) {
        FusedArgs a{};
        a.x = vx, a.wg = vwg, a.wu = vwu, a.wd = vwd, a.dy = vdy, a.ldx = ldx, a.ldg = ldg, a.ldd = ldd, a.ldy = ldy;
        a.rows = (int)d->rows, a.c = (int)d->c, a.f = (int)d->f, a.act = d->act;
        a.out = dx ? out(dx->p) : nullptr, a.ldo = dx ? dx->ld : 0, a.dg = dg, a.du = du, a.h = out(w + 2 * hidden_bytes(d));
        FHC_TRY((run_fused<T, true>(op, a, st)));
    } else if (hidden) {
        GemmArgs g{};
        g.a0 = vdy, g.b0 = vwd, g.lda = ldy, g.ldb = ldd, g.m = d->rows, g.n = d->f, g.k = d->c;
        g.o0 = dg, g.o1 = du, g.ldo = fp, g.ldpre = fp, g.act = d->act;
        g.pre_g = reinterpret_cast<float*>(keep + hidden_bytes(d));
        g.pre_u = reinterpret_cast<float*>(keep + hidden_bytes(d) + pre_bytes(d));
        FHC_TRY((product<T, false, true, kGrad>(op, g, nullptr, st)));
    }
    if (dx && !one) {
        GemmArgs g{};
        g.a0 = dg, g.a1 = du, g.b0 = vwg, g.b1 = vwu, g.lda = fp, g.ldb = ldg, g.segments = 2;
        g.m = d->rows, g.n = d->c, g.k = d->f, g.o0 = out(dx->p), g.ldo = dx->ld;
        FHC_TRY((product<T, false, true, kStore>(op, g, part, st)));
    }
    if (dwg || dwu) {
        GemmArgs g{};
        g.a0 = dwg ? dg : du, g.a1 = du, g.b0 = vx, g.lda = fp, g.ldb = ldx, g.pairs = dwg && dwu ? 2 : 1;
        g.m = d->f, g.n = d->c, g.k = d->rows, g.o0 = out(dwg ? dwg : dwu), g.o1 = out(dwu), g.ldo = d->c;
        FHC_TRY((product<T, true, true, kStore>(op, g, part, st)));
    }
    if (dwd) {
        GemmArgs g{};
        g.a0 = vdy, g.b0 = h, g.lda = ldy, g.ldb = fp;
        g.m = d->c, g.n = d->f, g.k = d->rows, g.o0 = out(dwd), g.ldo = d->f;
        FHC_TRY((product<T, true, true, kStore>(op, g, part, st)));
    }
    return 0;
}

}  // namespace
}  // namespace seq
}  // namespace fhc

using namespace fhc;
using namespace fhc::seq;

extern "C" size_t fhc_ffn_saved_bytes(const fhc_ffn_desc* d) {
    return guard((size_t)0, [&]() -> size_t {
        clear_error();
        if (check_desc("ffn_saved_bytes", d) < 0) return 0;
        return fused(d) ? 256 : hidden_bytes(d) + 2 * pre_bytes(d);
    });
}

extern "C" size_t fhc_ffn_workspace_bytes(const fhc_ffn_desc* d, int back) {
    return guard((size_t)0, [&]() -> size_t {
        clear_error();
        if (check_desc("ffn_workspace_bytes", d) < 0) return 0;
        return workspace(d, back != 0);
    });
}

extern "C" int fhc_ffn_forward(const fhc_ffn_desc* d, const fhc_rows* x, const void* wg, const void* wu,
                               const void* wd, const fhc_rows* y, void* saved, void* ws, size_t ws_bytes,
                               void* stream) {
    return guard(-3, [&]() -> int {
        clear_error();
        const char* op = "ffn_forward";
        FHC_TRY(check_desc(op, d));
        if (d->rows == 0 || d->c == 0) return 0;
        FHC_TRY(check_rows(op, "x", x, d->c));
        FHC_TRY(check_rows(op, "y", y, d->c));
        if (d->f) {
            FHC_TRY(check_weight(op, "wg", wg));
            FHC_TRY(check_weight(op, "wu", wu));
            FHC_TRY(check_weight(op, "wd", wd));
        }
        if (saved && !aligned(saved, 256)) return fail(-1, "%s: saved is not 256-byte aligned", op);
        FHC_TRY(check_workspace(op, workspace(d, false), ws, ws_bytes));
        const hipStream_t st = (hipStream_t)stream;
        return d->dtype == FHC_F16 ? forward<F16>(op, d, x, wg, wu, wd, y, saved, ws, st)
                                   : forward<BF16>(op, d, x, wg, wu, wd, y, saved, ws, st);
    });
}

extern "C" int fhc_ffn_backward(const fhc_ffn_desc* d, const fhc_rows* x, const void* wg, const void* wu,
                                const void* wd, const void* saved, const fhc_rows* dy, const fhc_rows* dx, void* dwg,
                                void* dwu, void* dwd, void* ws, size_t ws_bytes, void* stream) {
    return guard(-3, [&]() -> int {
        clear_error();
        const char* op = "ffn_backward";
        FHC_TRY(check_desc(op, d));
        if (d->c == 0) return 0;
        if (d->rows) {
            FHC_TRY(check_rows(op, "x", x, d->c));
            FHC_TRY(check_rows(op, "dy", dy, d->c));
            if (dx) FHC_TRY(check_rows(op, "dx", dx, d->c));
            if (d->f) {
                FHC_TRY(check_weight(op, "wg", wg));
                FHC_TRY(check_weight(op, "wu", wu));
                FHC_TRY(check_weight(op, "wd", wd));
                if (!saved) return fail(-1, "%s: null saved", op);
                if (!aligned(saved, 256)) return fail(-1, "%s: saved is not 256-byte aligned", op);
            }
        }
        // without rows there is nothing behind x, dy and dx, and they may be null; dense, the products' ranges are empty
        const fhc_rows none{nullptr, (int64_t)d->c};
        if (!d->rows) x = dy = &none, dx = nullptr;
        if (!aligned(dwg, 2) || !aligned(dwu, 2) || !aligned(dwd, 2))
            return fail(-1, "%s: a weight's gradient is not aligned to its elements", op);
        FHC_TRY(check_workspace(op, workspace(d, true), ws, ws_bytes));
        const hipStream_t st = (hipStream_t)stream;
        return d->dtype == FHC_F16 ? backward<F16>(op, d, x, wg, wu, wd, saved, dy, dx, dwg, dwu, dwd, ws, st)
                                   : backward<BF16>(op, d, x, wg, wu, wd, saved, dy, dx, dwg, dwu, dwd, ws, st);
    });
}
