// C entry points of the 4-bit layers (include/wino_amd.h).
#include "host.hpp"
#include "mx4.hpp"

using namespace wino;

namespace {

bool valid_dtype(int d) { return d == WINO_F32 || d == WINO_F16 || d == WINO_BF16; }
bool misaligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

bool overlap(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
    return p < q + nb && q < p + na;
}

// limits that the kernels' 32-bit offsets inside a tile rest on
constexpr int kMaxCols = 1 << 21;
constexpr long kMaxTiles = 1L << 27;            // of 128 x 128

int check_shape(const char* what, long rows, int K) {
    if (rows <= 0 || K <= 0) return fail(WINO_ERR_INVALID, "%s: sizes must be positive (rows %ld, K %d)", what, rows, K);
    if (K > kMaxCols) return fail(WINO_ERR_UNSUPPORTED, "%s: K = %d, at most %d", what, K, kMaxCols);
    if (mx4_grid<float>(rows, K) > 0x7fffffffL) return fail(WINO_ERR_UNSUPPORTED, "%s: %ld rows of %d", what, rows, K);
    return WINO_OK;
}
int check_operand(const char* what, const void* codes, const void* scales) {
    if (!codes || !scales) return fail(WINO_ERR_INVALID, "%s: null codes or scales", what);
    if (misaligned(codes, 16) || misaligned(scales, 16)) return fail(WINO_ERR_INVALID, "%s: codes and scales must be 16-byte aligned", what);
    return WINO_OK;
}

template <typename T> int quantize(int rows, int K, const void* x, void* codes, void* scales, hipStream_t s) {
    const int vec = !misaligned(x, 16) && (size_t)K * sizeof(T) % 16 == 0;
    hipLaunchKernelGGL((mx4_quantize_kernel<T>), dim3(mx4_grid<T>(rows, K)), dim3(256), 0, s,
                       static_cast<const T*>(x), rows, K, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), vec,
                       (size_t)rows * K * sizeof(T) > kMxStream);
    LAUNCH_CHECK("mx4_quantize");
    return WINO_OK;
}
int quantize_any(int dtype, int rows, int K, const void* x, void* codes, void* scales, hipStream_t s) {
    return dtype == WINO_F32   ? quantize<float>(rows, K, x, codes, scales, s)
           : dtype == WINO_F16 ? quantize<f16_t>(rows, K, x, codes, scales, s)
                               : quantize<bf16_t>(rows, K, x, codes, scales, s);
}

template <typename T> int dequantize(int rows, int K, const void* codes, const void* scales, void* x, hipStream_t s) {
    const int vec = !misaligned(x, 16) && (size_t)K * sizeof(T) % 16 == 0;
    hipLaunchKernelGGL((mx4_dequantize_kernel<T>), dim3(mx4_grid<T>(rows, K)), dim3(256), 0, s,
                       static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), rows, K, static_cast<T*>(x), vec);
    LAUNCH_CHECK("mx4_dequantize");
    return WINO_OK;
}

TileOperand mx4_operand(const void* codes, const void* scales, int rows) {
    return {static_cast<const char*>(codes), static_cast<const char*>(scales), kMxCols / 2, 0, rows, 0};
}

constexpr int kMostParts = 64;

TilePick pick_product(int M, int N, int K) { return tile_pick<mx4_t>(N, M, mx4_cols(K), kMostParts, device_cus()); }
// Up to 16 rows always (one column block of the multiply), up to 32 while the reduction is short: 32 x 1000 x 4096 takes
// 5.0 us against 7.3 through the tiles, 32 x 4096 x 25088 20.8 us against 15.3 -- x's codes are then read by every
// workgroup in as many bytes as w's.
bool few_rows(int M, int K) { return M <= 16 || (M <= kFewRows && K <= 8192); }
bool few_quant(int M, int K) { return few_rows(M, K) && (long)M * mx4_cols(K) <= kFewQuant; }

// x (in T) or its codes, whichever is not null
template <typename T>
int few_rows_product(unsigned flags, int M, int N, int K, const void* x, const void* xc, const void* xs, const void* wc, const void* ws,
                     const void* bias, void* y, hipStream_t s) {
    const int waves = std::min(kFewWaves, std::max(4, mx4_cols(K) / kMxCols));
    const int vec = x && !misaligned(x, 16) && (size_t)K * sizeof(T) % 16 == 0;
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(ceil_div(N, 16)), dim3(64 * waves), 0, s, static_cast<const T*>(x), static_cast<const uint8_t*>(xc),
                           static_cast<const uint8_t*>(xs), static_cast<const uint8_t*>(wc), static_cast<const uint8_t*>(ws),
                           static_cast<const T*>(bias), static_cast<T*>(y), M, N, K, (flags & WINO_FLAG_RELU) != 0, vec);
    };
    if (x && M <= 16) launch(mx4_few_rows_kernel<T, 1, true>);
    else if (x) launch(mx4_few_rows_kernel<T, 2, true>);
    else if (M <= 16) launch(mx4_few_rows_kernel<T, 1, false>);
    else launch(mx4_few_rows_kernel<T, 2, false>);
    LAUNCH_CHECK("mx4 product of few rows");
    return WINO_OK;
}
int few_rows_any(int dtype, unsigned flags, int M, int N, int K, const void* x, const void* xc, const void* xs, const void* wc,
                 const void* ws, const void* bias, void* y, hipStream_t s) {
    return dtype == WINO_F32   ? few_rows_product<float>(flags, M, N, K, x, xc, xs, wc, ws, bias, y, s)
           : dtype == WINO_F16 ? few_rows_product<f16_t>(flags, M, N, K, x, xc, xs, wc, ws, bias, y, s)
                               : few_rows_product<bf16_t>(flags, M, N, K, x, xc, xs, wc, ws, bias, y, s);
}

size_t product_bytes(int M, int N, int K) {
    if (few_rows(M, K)) return 0;
    const int parts = pick_product(M, N, K).parts;
    return parts > 1 ? part_bytes(N, M, parts) : 0;
}

// y[m][n] = relu?(sum_k x[m][k] w[n][k] + bias[n]): the weights' rows are the tile's m side, so that a lane stores
// neighbouring n
template <typename T>
int product(unsigned flags, int M, int N, int K, const void* xc, const void* xs, const void* wc, const void* ws, const void* bias,
            void* y, void* work, size_t work_bytes, hipStream_t s) {
    TileArgs g = {};
    g.a = mx4_operand(wc, ws, N);
    g.b = mx4_operand(xc, xs, M);
    g.M = N;
    g.N = M;
    g.K = mx4_cols(K);
    const TilePick pick = pick_product(M, N, K);
    const TileStore<T> store = {static_cast<T*>(y), N, static_cast<const T*>(bias), nullptr, (flags & WINO_FLAG_RELU) != 0};
    if (pick.parts == 1) {
        tile_launch<mx4_t, K_INNER, K_INNER>(g, store, pick, M, s);
        LAUNCH_CHECK("mx4 product");
        return WINO_OK;
    }
    const size_t need = part_bytes(N, M, pick.parts);
    if (!work || work_bytes < need) return fail(WINO_ERR_WORKSPACE, "mx4 product: workspace of %zu bytes, %zu needed", work ? work_bytes : 0, need);
    const long pitch = round_up(N, 4);
    const int made = tile_launch<mx4_t, K_INNER, K_INNER>(g, TilePart{static_cast<float*>(work), pitch, 0}, pick, M, s);
    LAUNCH_CHECK("mx4 product in parts");
    if (made != pick.parts) return fail(WINO_ERR_HIP, "mx4 product: %d parts for %d", made, pick.parts);
    hipLaunchKernelGGL((tile_join_kernel<T>), dim3(ceil_div((long)ceil_div(N, 4) * M, 256)), dim3(256), 0, s,
                       static_cast<const float*>(work), pick.parts, pitch, N, M, store);
    LAUNCH_CHECK("mx4 join");
    return WINO_OK;
}
int product_any(int dtype, unsigned flags, int M, int N, int K, const void* xc, const void* xs, const void* wc, const void* ws,
                const void* bias, void* y, void* work, size_t work_bytes, hipStream_t s) {
    if (few_rows(M, K)) return few_rows_any(dtype, flags, M, N, K, nullptr, xc, xs, wc, ws, bias, y, s);
    return dtype == WINO_F32   ? product<float>(flags, M, N, K, xc, xs, wc, ws, bias, y, work, work_bytes, s)
           : dtype == WINO_F16 ? product<f16_t>(flags, M, N, K, xc, xs, wc, ws, bias, y, work, work_bytes, s)
                               : product<bf16_t>(flags, M, N, K, xc, xs, wc, ws, bias, y, work, work_bytes, s);
}

int check_product(const char* what, int dtype, unsigned flags, int M, int N, int K, const void* wc, const void* ws, const void* bias,
                  const void* y, const void* work) {
    if (!valid_dtype(dtype)) return fail(WINO_ERR_INVALID, "%s: bad dtype %d", what, dtype);
    if (flags & ~WINO_FLAG_RELU) return fail(WINO_ERR_INVALID, "%s: flags 0x%x (only WINO_FLAG_RELU)", what, flags);
    int rc = check_shape(what, M, K);
    if (!rc) rc = check_shape(what, N, K);
    if (!rc) rc = check_operand(what, wc, ws);
    if (rc) return rc;
    if ((long)ceil_div(M, kTile) * ceil_div(N, kTile) > kMaxTiles) return fail(WINO_ERR_UNSUPPORTED, "%s: %d x %d outputs", what, M, N);
    if (!y) return fail(WINO_ERR_INVALID, "%s: null output", what);
    const size_t e = dtype_size(dtype);
    if (misaligned(y, e) || (bias && misaligned(bias, e))) return fail(WINO_ERR_INVALID, "%s: bias and y must be aligned to their element type", what);
    if (work && misaligned(work, 256)) return fail(WINO_ERR_INVALID, "%s: the workspace must be 256-byte aligned", what);
    return WINO_OK;
}

}  // namespace

extern "C" {

int wino_mx4_geometry(int rows, int K, int* Kp, size_t* code_bytes, size_t* scale_bytes) {
    const int rc = check_shape("wino_mx4_geometry", rows, K);
    if (rc) return rc;
    if (Kp) *Kp = mx4_cols(K);
    if (code_bytes) *code_bytes = mx4_code_bytes(rows, K);
    if (scale_bytes) *scale_bytes = mx4_scale_bytes(rows, K);
    return WINO_OK;
}

int wino_mx4_quantize(int dtype, int rows, int K, const void* x, void* codes, void* scales, void* stream) {
    if (!valid_dtype(dtype)) return fail(WINO_ERR_INVALID, "wino_mx4_quantize: bad dtype %d", dtype);
    int rc = check_shape("wino_mx4_quantize", rows, K);
    if (!rc) rc = check_operand("wino_mx4_quantize", codes, scales);
    if (rc) return rc;
    if (!x) return fail(WINO_ERR_INVALID, "wino_mx4_quantize: null input");
    if (misaligned(x, dtype_size(dtype))) return fail(WINO_ERR_INVALID, "wino_mx4_quantize: x must be aligned to its element type");
    return quantize_any(dtype, rows, K, x, codes, scales, (hipStream_t)stream);
}

int wino_mx4_dequantize(int dtype, int rows, int K, const void* codes, const void* scales, void* x, void* stream) {
    if (!valid_dtype(dtype)) return fail(WINO_ERR_INVALID, "wino_mx4_dequantize: bad dtype %d", dtype);
    int rc = check_shape("wino_mx4_dequantize", rows, K);
    if (!rc) rc = check_operand("wino_mx4_dequantize", codes, scales);
    if (rc) return rc;
    if (!x) return fail(WINO_ERR_INVALID, "wino_mx4_dequantize: null output");
    if (misaligned(x, dtype_size(dtype))) return fail(WINO_ERR_INVALID, "wino_mx4_dequantize: x must be aligned to its element type");
    hipStream_t s = (hipStream_t)stream;
    return dtype == WINO_F32   ? dequantize<float>(rows, K, codes, scales, x, s)
           : dtype == WINO_F16 ? dequantize<f16_t>(rows, K, codes, scales, x, s)
                               : dequantize<bf16_t>(rows, K, codes, scales, x, s);
}

size_t wino_mx4_workspace_bytes(int M, int N, int K) {
    if (check_shape("wino_mx4_workspace_bytes", M, K) || check_shape("wino_mx4_workspace_bytes", N, K)) return 0;
    if (few_quant(M, K)) return 0;
    return round_up(mx4_code_bytes(M, K), 256) + round_up(mx4_scale_bytes(M, K), 256) + round_up(product_bytes(M, N, K), 256);
}

int wino_mx4_gemm(int dtype, unsigned flags, int M, int N, int K, const void* xcodes, const void* xscales, const void* wcodes,
                  const void* wscales, const void* bias, void* y, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_product("wino_mx4_gemm", dtype, flags, M, N, K, wcodes, wscales, bias, y, workspace);
    if (!rc) rc = check_operand("wino_mx4_gemm", xcodes, xscales);
    if (rc) return rc;
    return product_any(dtype, flags, M, N, K, xcodes, xscales, wcodes, wscales, bias, y, workspace, workspace_bytes, (hipStream_t)stream);
}

int wino_mx4_linear(int dtype, unsigned flags, int M, int N, int K, const void* x, const void* wcodes, const void* wscales,
                    const void* bias, void* y, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = check_product("wino_mx4_linear", dtype, flags, M, N, K, wcodes, wscales, bias, y, workspace);
    if (rc) return rc;
    if (!x) return fail(WINO_ERR_INVALID, "wino_mx4_linear: null input");
    if (misaligned(x, dtype_size(dtype))) return fail(WINO_ERR_INVALID, "wino_mx4_linear: x must be aligned to its element type");
    // this kernel's workgroups all read x, and store their columns of y when they are done: one may still read what another
    // has written over
    if (few_quant(M, K) && overlap(x, (size_t)M * K * dtype_size(dtype), y, (size_t)M * N * dtype_size(dtype)))
        return fail(WINO_ERR_INVALID, "wino_mx4_linear: y must not overlap x in a call without a workspace (quantise x first)");
    if (few_quant(M, K)) return few_rows_any(dtype, flags, M, N, K, x, nullptr, nullptr, wcodes, wscales, bias, y, (hipStream_t)stream);
    const size_t need = wino_mx4_workspace_bytes(M, N, K);
    if (!workspace || workspace_bytes < need)
        return fail(WINO_ERR_WORKSPACE, "wino_mx4_linear: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, need);
    char* w = static_cast<char*>(workspace);
    char* xc = w;
    char* xs = xc + round_up(mx4_code_bytes(M, K), 256);
    char* part = xs + round_up(mx4_scale_bytes(M, K), 256);
    const int rq = quantize_any(dtype, M, K, x, xc, xs, (hipStream_t)stream);
    if (rq) return rq;
    return product_any(dtype, flags, M, N, K, xc, xs, wcodes, wscales, bias, y, part, need - (part - w), (hipStream_t)stream);
}

}  // extern "C"
