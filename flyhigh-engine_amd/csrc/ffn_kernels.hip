// The gated feed-forward block (include/fhc_seq.h): the launches around the products of ffn_gemm.h, and the products
// of few rows.
//
// Forward: one product with gate and up rows side by side whose epilogue is the activation and the product, one with
// wd. Backward: dh = dy wd with dL/dgate, dL/dup in its epilogue; dx = [dL/dgate dL/dup] [wg; wu] as one product over
// both halves of K; dwg and dwu (one launch), dwd, with the rows as K.
#include "ffn_fused.h"
#include "ffn_product.h"

namespace fhc {
namespace seq {
namespace {

// ---- host side ----------------------------------------------------------------------------------------------------

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
size_t hidden_bytes(const fhc_ffn_desc* d) { return up256((size_t)d->rows * up8(d->f) * 2); }
size_t pre_bytes(const fhc_ffn_desc* d) { return up256((size_t)d->rows * up8(d->f) * 4); }

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
                     pre_g, pre_u, d->act, {}};
        FHC_TRY((skinny<T, true, false>(op, a, st)));
        SkinnyArgs b{h, u16(wd), nullptr, fp, (int64_t)d->f, (int)d->rows, (int)d->c, (int)d->f,
                     static_cast<uint16_t*>(y->p), y->ld, (int)d->c, nullptr, nullptr, d->act, {}};
        return skinny<T, false, false>(op, b, st);
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
