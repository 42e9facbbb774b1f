// The matrix product with bias, activation and residual in its epilogue (include/fhc_seq.h), forward and backward, on the
// products of ffn_gemm.h and, for few rows, of ffn_product.h.
//
// Forward: one product, whose epilogue adds the bias in f32, keeps the sum where the backward pass needs it, applies the
// activation and adds the residual. Backward: dv = dy act'(v), with its sums over rows for the bias, in one pass (without an
// activation dv is dy itself, and only the bias needs a pass); dx = dv w, dw = dv^T x. The matrix units take operands of 16
// bits, so dv goes in as two numbers of the operands' type, its rounding and that rounding's remainder, one behind the other
// along K: what is lost is half a step of the remainder, 2^-16 (bf16) or 2^-22 (f16) of dv. FHC_LINEAR_ROUND_DV leaves the
// remainder out: half the work, and dx and dw carry dv's rounding beside their own (of random terms 1.4 times the error).
//
// What bounds it (MI355X): matrix units for large calls, HBM for few rows. 8192 x 2048 -> 8192 bf16 with silu, bias and
// residual: 320 us forward, 390 where v is kept (its f32 passes through the epilogue), a training step 1300: dv and its
// remainder 155 for 671 MB (4.3 TB/s), dx and dw 446 and 449 (1230 TFLOP/s over both parts; a large library product reaches
// 1344). With a rounded dv the step takes 910: dv 130, dx and dw 240 each. 4 x 2048 -> 8192: 11 us for 34 MB.
#include "ffn_product.h"
#include "seq_args.h"

namespace fhc {
namespace seq {
namespace {

// dv = dy act'(v) and its rounding's remainder in rows of up8(n), whose ends are zeros (dv null: dy is dv), and its sums over
// this workgroup's rows: 64 threads side by side take 8 columns each, 4 rows at once.
struct SlopeArgs {
    const uint16_t* dy;
    int64_t ldy;
    const float* pre;
    int64_t ldpre;
    uint16_t *dv, *rest;  // rest: dv's remainder, or null
    float* part;  // [workgroup rows][n], or null
    int rows, n, walks;
    uint32_t colblocks;  // of 512 columns; they come first in the workgroup's index
    uint32_t act;
};
template <class T>
__global__ __launch_bounds__(256) void linear_slope(SlopeArgs g) {
    __shared__ float sums[3][8][64];
    const uint32_t walk = blockIdx.x / g.colblocks, cb = blockIdx.x - walk * g.colblocks;
    const int lane = threadIdx.x & 63, row = threadIdx.x >> 6, c = (cb * 64 + lane) * 8, valid = g.n - c;
    float db[8];
#pragma unroll
    for (int v = 0; v < 8; v++) db[v] = 0.0f;
    if (valid > 0) {
        for (int64_t m = (int64_t)walk * 4 + row; m < g.rows; m += (int64_t)g.walks * 4) {
            const u4_t q = load_some(g.dy + m * g.ldy + c, valid);
            uint16_t out[8], rest[8];
            f4 pre[2] = {};
            if (g.pre) {
                pre[0] = *reinterpret_cast<const f4*>(g.pre + m * g.ldpre + c);
                pre[1] = *reinterpret_cast<const f4*>(g.pre + m * g.ldpre + c + 4);
            }
#pragma unroll
            for (int v = 0; v < 8; v++) {
                float d = widen(T{}, (uint16_t)(q[v >> 1] >> (16 * (v & 1)))), value, slope = 1.0f;
                if (g.pre) act_grad(g.act, pre[v >> 2][v & 3], value, slope);
                d = v < valid ? d * slope : 0.0f;
                db[v] += d;
                out[v] = narrow(T{}, d);
                const float held = widen(T{}, out[v]);  // past the type's range it is inf, and has no remainder
                rest[v] = narrow(T{}, __builtin_fabsf(held) < __builtin_inff() ? d - held : 0.0f);
            }
            if (g.dv) store_raw<uint16_t, 8, true>(g.dv + m * g.ldpre + c, out);
            if (g.rest) store_raw<uint16_t, 8, true>(g.rest + m * g.ldpre + c, rest);
        }
    }
    if (!g.part) return;
    if (row > 0) {
#pragma unroll
        for (int v = 0; v < 8; v++) sums[row - 1][v][lane] = db[v];
    }
    __syncthreads();
    if (row > 0) return;
#pragma unroll
    for (int v = 0; v < 8; v++) {
#pragma unroll
        for (int r = 0; r < 3; r++) db[v] += sums[r][v][lane];
        if (v < valid) g.part[(int64_t)walk * g.n + c + v] = db[v];
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------

uint32_t act(const fhc_linear_desc* d) { return d->act & ~FHC_LINEAR_ROUND_DV; }
int check_desc(const char* op, const fhc_linear_desc* d) {
    if (!d) return fail(-1, "%s: null descriptor", op);
    if (d->dtype > FHC_BF16) return fail(-1, "%s: dtype %u is neither f16 nor bf16", op, d->dtype);
    if (act(d) > FHC_ACT_IDENTITY) return fail(-1, "%s: act %u", op, d->act);
    if (d->c > 1u << 20 || d->f > 1u << 20) return fail(-1, "%s: %u x %u channels, at most 2^20", op, d->c, d->f);
    if (d->rows > 0x7FFFFF00u) return fail(-1, "%s: %u rows", op, d->rows);
    return 0;
}

bool keeps(const fhc_linear_desc* d) { return act(d) != FHC_ACT_IDENTITY; }
size_t pre_bytes(const fhc_linear_desc* d) { return keeps(d) ? up256((size_t)d->rows * up8(d->f) * 4) : 0; }
// products of the backward pass that dv takes along K
int parts_of(const fhc_linear_desc* d) { return keeps(d) && !(d->act & FHC_LINEAR_ROUND_DV) ? 2 : 1; }
// workgroups that a column block's rows are dealt to: four a CU over all columns, and as many (of one launch's) as leave a
// thread kMostTerms rows, whose sum for the bias is f32; the sums over workgroups are f64
constexpr uint32_t kMostTerms = 256;
uint32_t walks_of(const fhc_linear_desc* d) {
    const uint64_t cols = ceil_div(d->f, 512), most = ceil_div(d->rows, 4);
    if (!cols) return 0;
    const uint64_t few = ceil_div(1024, cols), room = ((1ull << 32) / 256 - 1) / cols;
    uint64_t want = ceil_div(most, kMostTerms);
    if (want > room) want = room;
    if (want < few) want = few;
    return (uint32_t)(want < most ? want : most);
}
size_t sums_bytes(const fhc_linear_desc* d) { return up256((size_t)walks_of(d) * d->f * 4); }

// Copies of the operands are counted whether a call makes them or not: that depends on its pointers and strides.
size_t workspace(const fhc_linear_desc* d, bool backward) {
    const size_t rows = Operands::pack_bytes(d->rows, d->c), w = Operands::pack_bytes(d->f, d->c);
    if (!backward) return d->rows > kSkinnyRows ? part_of(d->rows, d->f, d->c, 1, 1) + rows + w : 0;
    const int parts = parts_of(d);
    const size_t dx = part_of(d->rows, d->c, d->f, parts, 1), dw = part_of(d->f, d->c, d->rows, parts, 1);
    return parts * Operands::pack_bytes(d->rows, d->f) + sums_bytes(d) + (dx > dw ? dx : dw) + rows + w;
}

const uint16_t* u16(const void* p) { return static_cast<const uint16_t*>(p); }

template <class T>
int forward(const char* op, const fhc_linear_desc* d, const fhc_rows* x, const void* w, const void* bias,
            const fhc_rows* res, const fhc_rows* y, void* saved, void* ws, hipStream_t st) {
    float* pre = keeps(d) ? static_cast<float*>(saved) : nullptr;
    const Tail tail{u16(bias), res ? u16(res->p) : nullptr, res ? res->ld : 0, pre, up8(d->f), act(d)};
    uint16_t* out = static_cast<uint16_t*>(y->p);
    if (d->rows <= kSkinnyRows) {
        const SkinnyArgs a{u16(x->p), u16(w), nullptr, x->ld, (int64_t)d->c, (int)d->rows, (int)d->f, (int)d->c, out, y->ld,
                           (int)d->f, nullptr, nullptr, tail.act, tail};
        return skinny<T, false, true>(op, a, st);
    }
    char* at = static_cast<char*>(ws);
    Operands o{{}, 0, at + part_of(d->rows, d->f, d->c, 1, 1)};
    GemmArgs g{};
    g.lda = x->ld, g.ldb = d->c;
    g.a0 = o.take(x->p, g.lda, d->rows, d->c, true);
    g.b0 = o.take(w, g.ldb, d->f, d->c, true);
    FHC_TRY(o.copy(op, st));
    g.m = d->rows, g.n = d->f, g.k = d->c, g.o0 = out, g.ldo = y->ld;
    g.pre_g = pre, g.ldpre = tail.ldpre, g.act = tail.act, g.bias = tail.bias, g.res = tail.res, g.ldr = tail.ldr;
    return product<T, false, false, kLinear>(op, g, reinterpret_cast<float*>(at), st);
}

template <class T>
int backward(const char* op, const fhc_linear_desc* d, const fhc_rows* x, const void* w, const void* saved,
             const fhc_rows* dy, const fhc_rows* dx, void* dw, float* dbias, void* ws, hipStream_t st) {
    char* at = static_cast<char*>(ws);
    uint16_t* dv = reinterpret_cast<uint16_t*>(at);  // dL/dv, or a copy of dy that can be fetched
    at += Operands::pack_bytes(d->rows, d->f);
    const int parts = parts_of(d);
    uint16_t* rest = parts > 1 ? reinterpret_cast<uint16_t*>(at) : nullptr;
    at += (parts - 1) * Operands::pack_bytes(d->rows, d->f);
    float* sums = reinterpret_cast<float*>(at);
    at += sums_bytes(d);
    const size_t part_dx = part_of(d->rows, d->c, d->f, parts, 1), part_dw = part_of(d->f, d->c, d->rows, parts, 1);
    float* part = reinterpret_cast<float*>(at);
    at += part_dx > part_dw ? part_dx : part_dw;
    const uint32_t walks = walks_of(d);
    const bool slope = keeps(d) && (dx || dw || dbias);
    if (d->rows && d->f && (slope || dbias)) {
        SlopeArgs s{u16(dy->p), dy->ld, slope ? static_cast<const float*>(saved) : nullptr, up8(d->f),
                    slope ? dv : nullptr, slope ? rest : nullptr, dbias ? sums : nullptr, (int)d->rows, (int)d->f, (int)walks, (uint32_t)ceil_div(d->f, 512), act(d)};
        hipLaunchKernelGGL((linear_slope<T>), dim3(walks * s.colblocks), dim3(256), 0, st, s);
        FHC_TRY(launched(op));
    }
    if (dbias) FHC_TRY(close_sums(op, sums, walks, Sums{{dbias, nullptr, nullptr}, {d->f, 0, 0}}, st));
    int64_t ldv = up8(d->f), ldx = x->ld, ldw = d->c;
    const uint16_t* v = dv;
    if (!slope && (dx || dw)) {
        Operands o{{}, 0, reinterpret_cast<char*>(dv)};
        ldv = dy->ld;
        v = o.take(dy->p, ldv, d->rows, d->f, dx != nullptr);
        FHC_TRY(o.copy(op, st));
    }
    Operands o{{}, 0, at};
    const uint16_t* vx = dw ? o.take(x->p, ldx, d->rows, d->c, false) : nullptr;
    const uint16_t* vw = dx ? o.take(w, ldw, d->f, d->c, false) : nullptr;
    FHC_TRY(o.copy(op, st));
    if (dx) {
        GemmArgs g{};
        g.a0 = v, g.a1 = rest, g.b0 = g.b1 = vw, g.segments = parts, g.lda = ldv, g.ldb = ldw, g.m = d->rows, g.n = d->c, g.k = d->f;
        g.o0 = static_cast<uint16_t*>(dx->p), g.ldo = dx->ld;
        FHC_TRY((product<T, false, true, kStore>(op, g, part, st)));
    }
    if (dw) {
        GemmArgs g{};
        g.a0 = v, g.a1 = rest, g.b0 = g.b1 = vx, g.segments = parts, g.lda = ldv, g.ldb = ldx, g.m = d->f, g.n = d->c, g.k = d->rows;
        g.o0 = static_cast<uint16_t*>(dw), g.ldo = d->c;
        FHC_TRY((product<T, true, true, kStore>(op, g, part, st)));
    }
    return 0;
}

}  // namespace
}  // namespace seq
}  // namespace fhc

using namespace fhc;
using namespace fhc::seq;

extern "C" size_t fhc_linear_saved_bytes(const fhc_linear_desc* d) {
    return guard((size_t)0, [&]() -> size_t {
        clear_error();
        return check_desc("linear_saved_bytes", d) < 0 ? 0 : pre_bytes(d);
    });
}

extern "C" size_t fhc_linear_workspace_bytes(const fhc_linear_desc* d, int back) {
    return guard((size_t)0, [&]() -> size_t {
        clear_error();
        return check_desc("linear_workspace_bytes", d) < 0 ? 0 : workspace(d, back != 0);
    });
}

extern "C" int fhc_linear_forward(const fhc_linear_desc* d, const fhc_rows* x, const void* w, const void* bias,
                                  const fhc_rows* residual, const fhc_rows* y, void* saved, void* ws, size_t ws_bytes,
                                  void* stream) {
    return guard(-3, [&]() -> int {
        clear_error();
        const char* op = "linear_forward";
        FHC_TRY(check_desc(op, d));
        if (d->rows == 0 || d->f == 0) return 0;
        const fhc_rows none{nullptr, 0};
        if (d->c) {
            FHC_TRY(check_rows(op, "x", x, d->c));
            FHC_TRY(check_weight(op, "w", w));
        } else {
            x = &none;
        }
        FHC_TRY(check_rows(op, "y", y, d->f));
        if (residual) FHC_TRY(check_rows(op, "residual", residual, d->f));
        FHC_TRY(check_array(op, "bias", bias, 2, false));
        if (saved && !aligned(saved, 256)) return fail(-1, "%s: saved is not 256-byte aligned", op);
        FHC_TRY(check_workspace(op, workspace(d, false), ws, ws_bytes));
        const hipStream_t st = (hipStream_t)stream;
        return d->dtype == FHC_F16 ? forward<F16>(op, d, x, w, bias, residual, y, saved, ws, st)
                                   : forward<BF16>(op, d, x, w, bias, residual, y, saved, ws, st);
    });
}

extern "C" int fhc_linear_backward(const fhc_linear_desc* d, const fhc_rows* x, const void* w, const void* saved,
                                   const fhc_rows* dy, const fhc_rows* dx, void* dw, float* dbias, void* ws,
                                   size_t ws_bytes, void* stream) {
    return guard(-3, [&]() -> int {
        clear_error();
        const char* op = "linear_backward";
        FHC_TRY(check_desc(op, d));
        if (d->rows) {
            if (d->c && dw) FHC_TRY(check_rows(op, "x", x, d->c));
            if (d->c && dx) FHC_TRY(check_rows(op, "dx", dx, d->c));
            if (d->f) {
                FHC_TRY(check_rows(op, "dy", dy, d->f));
                if (d->c && dx) FHC_TRY(check_weight(op, "w", w));
                if (keeps(d) && !saved) return fail(-1, "%s: null saved", op);
                if (!aligned(saved, 256)) return fail(-1, "%s: saved is not 256-byte aligned", op);
            }
        }
        // without rows, channels or features there is nothing behind these, and the products' ranges are empty
        const fhc_rows none_x{nullptr, (int64_t)d->c}, none_y{nullptr, (int64_t)d->f};
        if (!d->rows) x = &none_x, dy = &none_y, dx = nullptr;
        if (!d->c) x = &none_x, dx = nullptr, dw = nullptr;
        if (!dw) x = &none_x;
        if (!d->f) dy = &none_y, dw = nullptr;
        if (!aligned(dw, 2)) return fail(-1, "%s: dw is not aligned to its elements", op);
        FHC_TRY(check_array(op, "dbias", dbias, 4, false));
        FHC_TRY(check_workspace(op, workspace(d, true), ws, ws_bytes));
        const hipStream_t st = (hipStream_t)stream;
        return d->dtype == FHC_F16 ? backward<F16>(op, d, x, w, saved, dy, dx, dw, dbias, ws, st)
                                   : backward<BF16>(op, d, x, w, saved, dy, dx, dw, dbias, ws, st);
    });
}
