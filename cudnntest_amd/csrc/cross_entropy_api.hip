// C entry points of the softmax cross entropy (include/wino_amd.h).
#include "cross_entropy.hpp"
#include "host.hpp"

using namespace wino;

namespace {

bool valid_dtype(int d) { return d == WINO_F32 || d == WINO_F16 || d == WINO_BF16; }
bool misaligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

constexpr int kMaxCols = 1 << 21;                     // the kernels' 32-bit offsets inside a tile rest on it
constexpr long kMaxTiles = 1L << 27;                  // of 128 x 128
// dl of one piece of the vocabulary: half of the last-level cache (2048 x 32000 x 2048 bf16 with 64 / 128 / 256 MB: 1635 /
// 1567 / 1566 us)
constexpr size_t kPieceBytes = 128u << 20;
// Rows of a backward call in 16 bits: dl of the smallest piece (128 classes, two values) is then 256 GB.  Twice as many are
// the length of dw's reduction, an int.
constexpr int kMaxTwinRows = 1 << 29;

// Where everything is in the workspace, and how the problem is cut.  The same function sizes the workspace and drives
// the calls.
struct Plan {
    bool pad_x, pad_w;                  // copied to 16-byte aligned rows first (odd lengths or bases); backward copies x for dw anyway
    int pitch_x, pitch_w;               // elements
    bool small;                         // too few tiles for the chip: logits as partial sums of a cut reduction
    TilePick logit, dx_cut, dw_cut;     // how the three products are cut
    int rows;                           // of dl: T rounded up to a stage
    int piece;                          // classes per piece (backward)
    bool together;                      // dx, dw and dbias in one launch
    size_t x, w, logits, stats, picked, scale, dl, dx, dw, total;
};

size_t place(size_t& at, size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
}

constexpr int kMostParts = 64;
constexpr int kTogetherTiles = 8;

template <typename E> Plan plan_as(int dtype, int T, int D, int V, const void* x, const void* w, bool backward) {
    Plan p = {};
    const size_t e = dtype_size(dtype);
    const int cus = device_cus();
    const bool odd = (size_t)D * e % 16 != 0;
    p.pad_x = odd || misaligned(x, 16);
    p.pad_w = odd || misaligned(w, 16);
    const int padded = (int)round_up(D, 8);
    p.pitch_x = p.pad_x ? padded : D;
    p.pitch_w = p.pad_w ? padded : D;
    p.logit = tile_pick<E>(V, T, D, kMostParts, cus);
    p.rows = (int)round_up(T, 64);
    constexpr int two = kValues<E>;
    p.small = p.logit.parts > 1 && (!backward || (size_t)p.rows * round_up(V, 128) * e * two <= kPieceBytes);
    size_t at = 0;
    if (p.pad_x || backward) p.x = place(at, (size_t)T * p.pitch_x * e);
    if (p.pad_w) p.w = place(at, (size_t)V * p.pitch_w * e);
    if (p.small) p.logits = place(at, part_bytes(V, T, p.logit.parts));
    else p.logit = tile_pick<E>(V, T, D, 1, cus);
    if (!backward) {
        if (!p.small) {
            p.stats = place(at, (size_t)ceil_div(V, p.logit.rows) * T * sizeof(float2));
            p.picked = place(at, (size_t)T * sizeof(float));
        }
    } else {
        p.scale = place(at, 2 * sizeof(float));
        const size_t fit = kPieceBytes / ((size_t)p.rows * e * two) / 256 * 256;
        p.piece = p.small ? V : (int)std::min<size_t>(V, std::max<size_t>(fit, 256));
        p.dl = place(at, (size_t)p.rows * round_up(p.piece, 128) * e * two);
        if (!p.small) p.logit = tile_pick<E>(p.piece, T, D, 1, cus);
        // the reductions as they run: twice over whole stages where dl is two values (the join adds as many parts as the cut has)
        p.dx_cut = tile_pick<E>(D, T, two > 1 ? two * (int)round_up(p.piece, kStageOf<E>) : p.piece, kMostParts, cus);
        p.dw_cut = tile_pick<E>(D, p.piece, two > 1 ? two * p.rows : T, kMostParts, cus);
        // one launch for the gradients while 64 x 64 tiles of both are a few to a CU, and whole sums are the better cut
        p.together = p.piece == V && p.dx_cut.parts == 1 && p.dw_cut.parts == 1 &&
                     (long)ceil_div(D, 64) * (ceil_div(T, 64) + ceil_div(V, 64)) <= kTogetherTiles * (long)cus;
        if (p.dx_cut.parts > 1 || p.piece < V) p.dx = place(at, part_bytes(D, T, p.dx_cut.parts));
        if (p.dw_cut.parts > 1) p.dw = place(at, part_bytes(D, p.piece, p.dw_cut.parts));
    }
    p.total = at;
    return p;
}
Plan plan(int dtype, int T, int D, int V, const void* x, const void* w, bool backward) {
    return dtype == WINO_F32   ? plan_as<float>(dtype, T, D, V, x, w, backward)
           : dtype == WINO_F16 ? plan_as<f16_t>(dtype, T, D, V, x, w, backward)
                               : plan_as<bf16_t>(dtype, T, D, V, x, w, backward);
}

int check(const char* what, int dtype, int T, int D, int V, const void* x, const void* w, const void* bias, const void* target) {
    if (!valid_dtype(dtype)) return fail(WINO_ERR_INVALID, "%s: bad dtype %d", what, dtype);
    if (T <= 0 || D <= 0 || V <= 0) return fail(WINO_ERR_INVALID, "%s: sizes must be positive (T %d, D %d, V %d)", what, T, D, V);
    if (D > kMaxCols) return fail(WINO_ERR_UNSUPPORTED, "%s: D = %d, at most %d", what, D, kMaxCols);
    if (V > (1 << 24)) return fail(WINO_ERR_UNSUPPORTED, "%s: V = %d, at most %d", what, V, 1 << 24);
    if ((long)ceil_div(T, kTile) * ceil_div(V, kTile) > kMaxTiles || (long)ceil_div(T, kTile) * ceil_div(D, kTile) > kMaxTiles)
        return fail(WINO_ERR_UNSUPPORTED, "%s: T = %d is too large", what, T);
    if (!x || !w || !target) return fail(WINO_ERR_INVALID, "%s: null x, w or target", what);
    const size_t e = dtype_size(dtype);
    if (misaligned(x, e) || misaligned(w, e) || (bias && misaligned(bias, e)) || misaligned(target, 8))
        return fail(WINO_ERR_INVALID, "%s: tensors must be aligned to their element type", what);
    return WINO_OK;
}

int check_backward(const char* what, int dtype, int T) {
    if (dtype != WINO_F32 && T > kMaxTwinRows) return fail(WINO_ERR_UNSUPPORTED, "%s: T = %d, at most %d in 16 bits", what, T, kMaxTwinRows);
    return WINO_OK;
}

template <typename T> TileOperand inner(const T* p, long pitch, int rows) {
    const long b = pitch * (long)sizeof(T);
    return {reinterpret_cast<const char*>(p), nullptr, b, 0, rows, 0};
}
template <typename T> TileOperand outer(const T* p, long pitch, int k_rows) {
    const long b = pitch * (long)sizeof(T);
    return {reinterpret_cast<const char*>(p), nullptr, b, 0, k_rows, (int)(b / 16)};
}

template <typename T> int row_copy(const RowCopy<T>& c, hipStream_t s) {
    if (c.blocks() > 0x7ffffff0L) return fail(WINO_ERR_UNSUPPORTED, "row copy: %ld rows of %d", c.rows, c.cols);
    hipLaunchKernelGGL((row_copy_kernel<T>), dim3((unsigned)c.blocks()), dim3(256), 0, s, c);
    LAUNCH_CHECK("row_copy");
    return WINO_OK;
}

template <typename T> struct Call {
    int T_, D, V;
    const T *x, *w, *bias;
    CeRows rows;
    Plan p;
    char* ws;
    hipStream_t s;

    // backward: without what ignored rows hold
    RowCopy<T> copy_of_x(bool backward) const {
        return {x, reinterpret_cast<T*>(ws + p.x), T_, D, p.pitch_x, backward ? rows.target : nullptr, rows.ignore};
    }
    int operands(bool backward) {
        if (p.pad_x) {
            const RowCopy<T> c = copy_of_x(backward);
            const int rc = row_copy<T>(c, s);
            if (rc) return rc;
            x = c.y;
        }
        if (p.pad_w) {
            const RowCopy<T> c = {w, reinterpret_cast<T*>(ws + p.w), V, D, p.pitch_w, nullptr, 0};
            const int rc = row_copy<T>(c, s);
            if (rc) return rc;
            w = c.y;
        }
        return WINO_OK;
    }
    TileArgs logits(int v0, int n) const {
        TileArgs g = {};
        g.a = inner<T>(w + (long)v0 * p.pitch_w, p.pitch_w, n);
        g.b = inner<T>(x, p.pitch_x, T_);
        g.M = n;
        g.N = T_;
        g.K = D;
        return g;
    }
    int partial_logits(CeParts<T>* parts) {
        float* to = reinterpret_cast<float*>(ws + p.logits);
        const long pitch = round_up(V, 4);
        const int made = tile_launch<T, K_INNER, K_INNER>(logits(0, V), TilePart{to, pitch, 0}, p.logit, T_, s);
        LAUNCH_CHECK("logits in parts");
        if (made != p.logit.parts) return fail(WINO_ERR_HIP, "logits: %d parts for %d", made, p.logit.parts);
        *parts = {to, p.logit.parts, pitch, pitch * T_, bias};
        return WINO_OK;
    }

    int forward(float* loss, float* lse) {
        int rc = operands(false);
        if (rc) return rc;
        if (p.small) {
            CeParts<T> parts;
            if ((rc = partial_logits(&parts))) return rc;
            hipLaunchKernelGGL((ce_rows_kernel<T>), dim3(T_), dim3(1024), 0, s, parts, rows, loss, lse);
            LAUNCH_CHECK("ce_rows");
            return WINO_OK;
        }
        float2* stats = reinterpret_cast<float2*>(ws + p.stats);
        float* picked = reinterpret_cast<float*>(ws + p.picked);
        tile_launch<T, K_INNER, K_INNER>(logits(0, V), CeStats<T>{bias, rows, stats, picked}, p.logit, T_, s);
        LAUNCH_CHECK("ce_stats");
        hipLaunchKernelGGL(ce_join_kernel, dim3(ceil_div(T_, 32)), dim3(256), 0, s, stats, picked, rows, T_, ceil_div(V, p.logit.rows), loss, lse);
        LAUNCH_CHECK("ce_join");
        return WINO_OK;
    }

    int backward(const float* grad, const float* lse, T* dx, T* dw, T* dbias) {
        int rc = operands(true);
        if (rc) return rc;
        // x for dw: copied with the operands, by the kernel that writes a small problem's dl, or here
        RowCopy<T> copy = copy_of_x(true);
        const bool copy_inside = p.small && dw && !p.pad_x && copy.blocks() < (1 << 20);
        if (dw && !p.pad_x && !copy_inside && (rc = row_copy<T>(copy, s))) return rc;
        const T* xw = copy.y;
        float* scale = nullptr;
        const float top = std::is_same<T, f16_t>::value ? 32768.f : 1.f;
        const bool scale_inside = p.small && T_ <= 1024;      // the kernel that writes dl finds the factor itself
        if (sizeof(T) == 2) {
            scale = reinterpret_cast<float*>(ws + p.scale);
            if (!scale_inside) {
                hipLaunchKernelGGL(ce_scale_kernel, dim3(1), dim3(1024), 0, s, grad, rows, T_, top, scale);
                LAUNCH_CHECK("ce_scale");
            }
        }
        const float* back = scale ? scale + 1 : nullptr;
        T* dl = reinterpret_cast<T*>(ws + p.dl);
        float* dx_part = reinterpret_cast<float*>(ws + p.dx);
        float* dw_part = reinterpret_cast<float*>(ws + p.dw);
        const bool dx_direct = p.dx_cut.parts == 1 && p.piece >= V;
        const long d4 = round_up(D, 4);
        const TileStore<T> dx_store = {dx, D, nullptr, back, 0};
        for (int v0 = 0; v0 < V; v0 += p.piece) {
            const int n = std::min(p.piece, V - v0);
            const int width = (int)round_up(n, 128);
            const long pitch = (long)kValues<T> * width;
            const CeDl<T> out = {bias ? bias + v0 : nullptr, rows, lse, grad, scale_inside ? nullptr : scale, v0, dl, pitch, width, p.rows};
            if (p.small) {
                CeParts<T> parts;
                if ((rc = partial_logits(&parts))) return rc;
                const int blocks = ceil_div((long)p.rows * (width / 4), 256);
                hipLaunchKernelGGL((ce_dl_kernel<T>), dim3(blocks + (copy_inside ? (int)copy.blocks() : 0)), dim3(256), 0, s, parts, out, T_, top,
                                   scale_inside ? scale : nullptr, blocks, copy);
            } else {
                tile_launch<T, K_INNER, K_INNER>(logits(v0, n), out, p.logit, p.rows, s);
            }
            LAUNCH_CHECK("ce_dl");
            // dx[t][d] (+)= sum_v w[v][d] dl[t][v]
            TileArgs gx = {};
            gx.a = outer<T>(w + (long)v0 * p.pitch_w, p.pitch_w, n);
            gx.b = inner<T>(dl, pitch, T_);
            gx.M = D;
            gx.N = T_;
            gx.K = n;
            if (kValues<T> == 2) {      // over dl, then over what it leaves; w from its start again
                gx.K = (int)round_up(n, kStageOf<T>);
                gx.passes = 2;
                gx.a_turn = -(long)gx.K * gx.a.pitch;
                gx.b_turn = (width - gx.K) * (long)sizeof(T);
            }
            // dw[v][d] = sum_t x[t][d] dl[t][v]
            TileArgs gw = {};
            gw.a = outer<T>(xw, p.pitch_x, T_);
            gw.b = outer<T>(dl, pitch, p.rows);
            gw.b.pieces = width * (int)sizeof(T) / 16;     // of one value: the second pass starts `width` elements into the row
            gw.M = D;
            gw.N = n;
            gw.K = T_;
            if (kValues<T> == 2) {
                gw.K = p.rows;
                gw.passes = 2;
                gw.a_turn = -(long)gw.K * gw.a.pitch;
                gw.b_turn = -(long)gw.K * gw.b.pitch + width * (long)sizeof(T);
            }
            const TileStore<T> dw_store = {dw ? dw + (long)v0 * D : nullptr, D, nullptr, back, 0};
            const CeBias<T> bias_sum = {dl, pitch, width, T_, n, back, dbias ? dbias + v0 : nullptr};
            if (p.together && dx && dw) {
                tile_prepare<T, K_OUTER, K_INNER, 64, 64, 128>(gx, 1, T_);
                tile_prepare<T, K_OUTER, K_OUTER, 64, 64, 128>(gw, 1, n);
                const int nx = tile_grid(gx.mt, gx.nt), nw = tile_grid(gw.mt, gw.nt);
                const int nb = dbias ? (ceil_div(n, 64) + 7) / 8 * 8 : 0;      // (the tiles keep their XCDs)
                hipLaunchKernelGGL((ce_gradients_kernel<T>), dim3(nb + nx + nw), dim3(256), 0, s, bias_sum, nb, gx, dx_store, nx, gw, dw_store);
                LAUNCH_CHECK("ce_gradients");
                return WINO_OK;
            }
            if (dx) {
                int made = p.dx_cut.parts;
                if (dx_direct) tile_launch<T, K_OUTER, K_INNER>(gx, dx_store, p.dx_cut, T_, s);
                else made = tile_launch<T, K_OUTER, K_INNER>(gx, TilePart{dx_part, d4, v0 > 0}, p.dx_cut, T_, s);
                LAUNCH_CHECK("ce_dx");
                // (a shorter last piece may make fewer; the others' sums stay)
                if (v0 == 0 && made != p.dx_cut.parts) return fail(WINO_ERR_HIP, "dx: %d parts for %d", made, p.dx_cut.parts);
            }
            if (dw) {
                if (p.dw_cut.parts == 1) {
                    tile_launch<T, K_OUTER, K_OUTER>(gw, dw_store, p.dw_cut, n, s);
                } else {
                    const int made = tile_launch<T, K_OUTER, K_OUTER>(gw, TilePart{dw_part, d4, 0}, p.dw_cut, n, s);
                    LAUNCH_CHECK("ce_dw");
                    if (made != p.dw_cut.parts) return fail(WINO_ERR_HIP, "dw: %d parts for %d", made, p.dw_cut.parts);
                    hipLaunchKernelGGL((tile_join_kernel<T>), dim3(ceil_div((long)ceil_div(D, 4) * n, 256)), dim3(256), 0, s,
                                       dw_part, p.dw_cut.parts, d4, D, n, dw_store);
                }
                LAUNCH_CHECK("ce_dw");
            }
            if (dbias) {
                hipLaunchKernelGGL((ce_bias_kernel<T>), dim3(ceil_div(n, 64)), dim3(1024), 0, s, bias_sum);
                LAUNCH_CHECK("ce_bias");
            }
        }
        if (dx && !dx_direct) {
            hipLaunchKernelGGL((tile_join_kernel<T>), dim3(ceil_div((long)ceil_div(D, 4) * T_, 256)), dim3(256), 0, s, dx_part, p.dx_cut.parts, d4, D, T_, dx_store);
            LAUNCH_CHECK("ce_dx join");
        }
        return WINO_OK;
    }
};

template <typename T>
Call<T> make_call(int T_, int D, int V, const void* x, const void* w, const void* bias, const long long* target, long long ignore,
                  const Plan& p, void* ws, void* stream) {
    return {T_, D, V, static_cast<const T*>(x), static_cast<const T*>(w), static_cast<const T*>(bias), {target, ignore, V}, p,
            static_cast<char*>(ws), (hipStream_t)stream};
}

int check_workspace(const char* what, const Plan& p, const void* ws, size_t bytes) {
    if (p.total == 0) return WINO_OK;
    if (!ws || bytes < p.total) return fail(WINO_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, ws ? bytes : 0, p.total);
    if (misaligned(ws, 256)) return fail(WINO_ERR_INVALID, "%s: the workspace must be 256-byte aligned", what);
    return WINO_OK;
}

}  // namespace

extern "C" {

size_t wino_linear_cross_entropy_workspace_bytes(int dtype, int T, int D, int V, const void* x, const void* w, int backward) {
    static const long long any = 0;
    if (check("wino_linear_cross_entropy_workspace_bytes", dtype, T, D, V, x, w, nullptr, &any)) return 0;
    if (backward && check_backward("wino_linear_cross_entropy_workspace_bytes", dtype, T)) return 0;
    return plan(dtype, T, D, V, x, w, backward != 0).total;
}

int wino_linear_cross_entropy(int dtype, int T, int D, int V, const void* x, const void* w, const void* bias, const long long* target,
                              long long ignore_index, float* loss, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check("wino_linear_cross_entropy", dtype, T, D, V, x, w, bias, target);
    if (rc) return rc;
    if (!loss || !lse) return fail(WINO_ERR_INVALID, "wino_linear_cross_entropy: null loss or lse");
    if (misaligned(loss, 4) || misaligned(lse, 4)) return fail(WINO_ERR_INVALID, "wino_linear_cross_entropy: loss and lse must be 4-byte aligned");
    const Plan p = plan(dtype, T, D, V, x, w, false);
    if ((rc = check_workspace("wino_linear_cross_entropy", p, workspace, workspace_bytes))) return rc;
    if (dtype == WINO_F32) return make_call<float>(T, D, V, x, w, bias, target, ignore_index, p, workspace, stream).forward(loss, lse);
    if (dtype == WINO_F16) return make_call<f16_t>(T, D, V, x, w, bias, target, ignore_index, p, workspace, stream).forward(loss, lse);
    return make_call<bf16_t>(T, D, V, x, w, bias, target, ignore_index, p, workspace, stream).forward(loss, lse);
}

int wino_linear_cross_entropy_backward(int dtype, int T, int D, int V, const void* x, const void* w, const void* bias,
                                       const long long* target, long long ignore_index, const float* grad, const float* lse, void* dx,
                                       void* dw, void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check("wino_linear_cross_entropy_backward", dtype, T, D, V, x, w, bias, target);
    if (!rc) rc = check_backward("wino_linear_cross_entropy_backward", dtype, T);
    if (rc) return rc;
    if (!grad || !lse) return fail(WINO_ERR_INVALID, "wino_linear_cross_entropy_backward: null grad or lse");
    if (!dx && !dw && !dbias) return fail(WINO_ERR_INVALID, "wino_linear_cross_entropy_backward: no gradient asked for");
    const size_t e = dtype_size(dtype);
    if (misaligned(grad, 4) || misaligned(lse, 4) || misaligned(dx, e) || misaligned(dw, e) || misaligned(dbias, e))
        return fail(WINO_ERR_INVALID, "wino_linear_cross_entropy_backward: tensors must be aligned to their element type");
    const Plan p = plan(dtype, T, D, V, x, w, true);
    if ((rc = check_workspace("wino_linear_cross_entropy_backward", p, workspace, workspace_bytes))) return rc;
    if (dtype == WINO_F32)
        return make_call<float>(T, D, V, x, w, bias, target, ignore_index, p, workspace, stream)
            .backward(grad, lse, static_cast<float*>(dx), static_cast<float*>(dw), static_cast<float*>(dbias));
    if (dtype == WINO_F16)
        return make_call<f16_t>(T, D, V, x, w, bias, target, ignore_index, p, workspace, stream)
            .backward(grad, lse, static_cast<f16_t*>(dx), static_cast<f16_t*>(dw), static_cast<f16_t*>(dbias));
    return make_call<bf16_t>(T, D, V, x, w, bias, target, ignore_index, p, workspace, stream)
        .backward(grad, lse, static_cast<bf16_t*>(dx), static_cast<bf16_t*>(dw), static_cast<bf16_t*>(dbias));
}

}  // extern "C"
