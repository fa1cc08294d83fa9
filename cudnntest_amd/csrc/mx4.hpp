// Microscaled 4-bit floating point (the OCP MX format with e2m1 elements): quantisation and reading back.
//
// Along a row, blocks of 32 values share a scale 2^(b - 127), b one byte; an element is sign, two exponent bits and one
// mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6.  A block with largest magnitude a gets
//     b = clamp(floor(log2 a) - 2 + 127, 0, 254),        element = round(x / 2^(b - 127))
// to nearest, ties to even, saturating at 6 (the MX specification's conversion: the scale is the largest power of two
// that keeps the block's top binade on the grid, at the price of saturation between 6 and 8).  A block that holds a NaN or
// an infinity gets b = 255, the format's NaN, so that it stays visible in every product.
//
// A quantised matrix of R rows and K columns is kept as the product kernels read it, Kp = K rounded up to 128:
//     codes  [Kp/128][R][64]              two codes per byte, the lower column in the low half
//     scales [Kp/128][R rounded up to 4][4]
// i.e. one stage of a tile's rows is one contiguous run.  Columns past K are zeros.
#pragma once
#include "common.hpp"
#include "tile_gemm.hpp"

namespace wino {

constexpr int kMxCols = 128;             // columns of a stage
inline int mx4_cols(int K) { return (int)round_up(K, kMxCols); }
inline size_t mx4_code_bytes(long rows, int K) { return (size_t)rows * (mx4_cols(K) / 2); }
inline size_t mx4_scale_bytes(long rows, int K) { return (size_t)round_up(rows, 4) * (mx4_cols(K) / 32); }

// eight consecutive elements of a row as fp32; left: how many of them exist
template <typename T> __device__ __forceinline__ void load8(const T* x, int left, bool vec, float (&v)[8]) {
    if (vec && left >= 8) {
        constexpr int n = 16 / (int)sizeof(T);
#pragma unroll
        for (int p = 0; p < 8 / n; ++p) {
            const Pack16<T> pk = reinterpret_cast<const Pack16<T>*>(x)[p];
#pragma unroll
            for (int e = 0; e < n; ++e) v[p * n + e] = to_f32(pk.e[e]);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < left ? to_f32(x[e]) : 0.f;
}

// the scale byte of a block whose largest magnitude has these bits (NaN and infinity sort above every number)
__device__ __forceinline__ unsigned mx4_scale_byte(unsigned top_bits) {
    const unsigned e = top_bits >> 23;
    return e == 255 ? 255u : e < 2 ? 0u : e - 2;
}
// 2^(b - 127) as a float; b = 0 is a subnormal
__device__ __forceinline__ float mx4_scale_value(unsigned b) { return __uint_as_float(b == 0 ? 0x00400000u : b << 23); }

// eight values as eight codes; the conversion instruction divides by the scale, rounds to nearest even and saturates
__device__ __forceinline__ unsigned mx4_encode8(const float (&v)[8], float scale) {
    unsigned c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
    return c;
}

// largest of the values of four neighbouring lanes
__device__ __forceinline__ unsigned quad_max(unsigned v) {
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));
    return max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));
}

// Both conversions move 16 bytes of the wide side per lane, so that a wave's access is one run of 1 KB per two rows (fp32)
// or four: E = 4 or 8 columns, 32 / E neighbouring lanes to a block.  A workgroup takes kMxStages stages of 128 columns
// of 8 or 16 rows, all of a thread's loads in flight before the first is used (4096 x 25088 fp32, 1 / 2 / 4 stages: quantise
// 91 / 81 / 77 us, one row of 4096 2.9 / 3.1 / 3.4 us).  The wide side is read or written past the caches' replacement order
// (non-temporal): always when it is written (the same matrix 128 -> 66 us, 4096 x 8192 bf16 17.7 -> 15.7: 7 TB/s), when it is
// read only if it could not have been in the 256 MB last-level cache (93 -> 81 us; 134 MB in that cache 23 -> 26 us).
constexpr size_t kMxStream = 256u << 20;
constexpr int kMxStages = 2;
template <typename T> constexpr int kMxPer = 16 / (int)sizeof(T);      // columns per thread
template <typename T> constexpr int kMxRows = 256 * kMxPer<T> / kMxCols;   // rows per workgroup
template <typename T> inline long mx4_grid(int rows, int K) {
    return (long)ceil_div(mx4_cols(K) / kMxCols, kMxStages) * ceil_div(rows, kMxRows<T>);
}

template <typename T>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const T* __restrict__ x, int rows, int K, uint8_t* __restrict__ codes,
                                                           uint8_t* __restrict__ scales, int vec, int stream) {
    constexpr int E = kMxPer<T>, LANES = kMxCols / E;                  // threads per row and stage
    const unsigned kbs = (K + kMxCols - 1) / kMxCols, groups = (kbs + kMxStages - 1) / kMxStages;
    const int row = blockIdx.x / groups * kMxRows<T> + threadIdx.x / LANES, t = threadIdx.x % LANES;
    const int kb0 = blockIdx.x % groups * kMxStages;
    if (row >= rows) return;
    float v[kMxStages][E];
#pragma unroll
    for (int u = 0; u < kMxStages; ++u) {
        const int k = (kb0 + u) * kMxCols + t * E, left = K - k;
        const T* at = x + (long)row * K + k;
        if (vec && left >= E) {
            const uintx4* from = reinterpret_cast<const uintx4*>(at);
            const Pack16<T> pk = __builtin_bit_cast(Pack16<T>, stream ? __builtin_nontemporal_load(from) : *from);
#pragma unroll
            for (int e = 0; e < E; ++e) v[u][e] = to_f32(pk.e[e]);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) v[u][e] = e < left ? to_f32(at[e]) : 0.f;
        }
    }
#pragma unroll
    for (int u = 0; u < kMxStages; ++u) {
        const int kb = kb0 + u;
        if (kb >= (int)kbs) return;
        unsigned top = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) top = max(top, __float_as_uint(v[u][e]) & 0x7fffffffu);
        top = quad_max(top);
        if (E == 4) top = max(top, (unsigned)__builtin_amdgcn_mov_dpp((int)top, 0x141, 0xF, 0xF, true));   // the other four of eight lanes
        const unsigned b = mx4_scale_byte(top);
        const float s = mx4_scale_value(b);
        const long at = (long)kb * rows + row;
        if constexpr (E == 8) {
            reinterpret_cast<unsigned*>(codes)[at * 16 + t] = b == 255 ? 0u : mx4_encode8(v[u], s);
        } else {
            unsigned c = 0;
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[u][0], v[u][1], s, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[u][2], v[u][3], s, 1);
            reinterpret_cast<unsigned short*>(codes)[at * 32 + t] = b == 255 ? 0 : (unsigned short)c;
        }
        if (t % (32 / E) == 0) {
            uint8_t* sp = scales + ((long)kb * ((rows + 3) & ~3) + row) * 4 + t / (32 / E);
            *sp = (uint8_t)b;
            if (row == rows - 1)                                       // the rows that pad the count to four
                for (int r = rows; r & 3; ++r) sp[4 * (r - row)] = 0;
        }
    }
}

// code (low four bits) * 2^(b - 127), exact in fp32
__device__ __forceinline__ float mx4_value(unsigned code, int b) {
    const unsigned e = (code >> 1) & 3, m = code & 1;
    const float mag = e ? __uint_as_float(((126 + e) << 23) | (m << 22)) : 0.5f * (float)m;
    const float v = b == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(mag, b - 127);
    return code & 8 ? -v : v;
}

template <typename T>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                             int rows, int K, T* __restrict__ x, int vec) {
    constexpr int E = kMxPer<T>, LANES = kMxCols / E;
    const unsigned kbs = (K + kMxCols - 1) / kMxCols, groups = (kbs + kMxStages - 1) / kMxStages;
    const int row = blockIdx.x / groups * kMxRows<T> + threadIdx.x / LANES, t = threadIdx.x % LANES;
    const int kb0 = blockIdx.x % groups * kMxStages;
    if (row >= rows) return;
    unsigned c[kMxStages], b[kMxStages];
#pragma unroll
    for (int u = 0; u < kMxStages; ++u) {
        const long kb = min(kb0 + u, (int)kbs - 1), at = kb * rows + row;
        c[u] = E == 8 ? reinterpret_cast<const unsigned*>(codes)[at * 16 + t] : reinterpret_cast<const unsigned short*>(codes)[at * 32 + t];
        b[u] = scales[(kb * ((rows + 3) & ~3) + row) * 4 + t / (32 / E)];
    }
#pragma unroll
    for (int u = 0; u < kMxStages; ++u) {
        const int k = (kb0 + u) * kMxCols + t * E;
        if (k >= K) return;
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = mx4_value(c[u] >> (4 * e), b[u]);
        T* to = x + (long)row * K + k;
        if (vec && K - k >= E) {
            Pack16<T> pk;
#pragma unroll
            for (int e = 0; e < E; ++e) pk.e[e] = from_f32<T>(v[e]);
            __builtin_nontemporal_store(__builtin_bit_cast(uintx4, pk), reinterpret_cast<uintx4*>(to));
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (k + e < K) to[e] = from_f32<T>(v[e]);
        }
    }
}

// ---- few rows ------------------------------------------------------------------------------------
// y = relu?(x w^T + bias) for up to 32 rows of x: bound by reading w once.  A workgroup owns 16 rows of w (for 4096 rows
// one workgroup per CU) and its waves share the reduction, stage by stage; a wave's load of w is 1 KB of consecutive
// memory (16 rows x 64 bytes), the operand of one v_mfma_scale_f32_16x16x128 per 16 rows of x, and the loads of
// kFlight stages are in flight.  The partial sums meet in LDS and are added in wave order.
// QUANT: x arrives in T and every workgroup quantises all of it into LDS while its first loads of w travel, which saves
// a launch and the codes' way through memory (while x is small: the work is repeated by every workgroup); otherwise x's
// codes come from memory.  Both give the same bits: the same codes, multiplied and added in the same order.
constexpr int kFewRows = 32;             // rows of x that this kernel takes
constexpr int kFewQuant = 32768;         // elements of x (columns rounded up) that it quantises itself
constexpr int kFewWaves = 16;

template <typename T, int NT, bool QUANT>
__global__ __launch_bounds__(64 * kFewWaves) void mx4_few_rows_kernel(const T* __restrict__ x, const uint8_t* __restrict__ xc,
                                                                      const uint8_t* __restrict__ xs, const uint8_t* __restrict__ wc,
                                                                      const uint8_t* __restrict__ ws, const T* __restrict__ bias,
                                                                      T* __restrict__ y, int M, int N, int K, int relu, int vec) {
    __shared__ __align__(16) uint8_t qc[QUANT ? kFewQuant / 2 : 16];
    __shared__ uint8_t qs[QUANT ? kFewQuant / 32 : 4];
    __shared__ floatx4 part[kFewWaves][NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int r = lane & 15, q = lane >> 4;
    const int kbs = (K + kMxCols - 1) / kMxCols;
    const int n0 = blockIdx.x * 16, row = min(n0 + r, N - 1);
    const long rows4 = (N + 3) & ~3;
    // stage kb of this lane's row of w: 16 bytes of codes and the scale of those 32
    const uint8_t* wp = wc + (long)row * 64 + q * 16;
    const uint8_t* sp = ws + (long)row * 4 + q;
    constexpr int kFlight = 4;                                         // (8 and 13: 14.3 and 16.3 us for 14.2)
    constexpr int kX = QUANT ? 0 : NT;
    const long xrows4 = (M + 3) & ~3;
    uintx4 fw[kFlight], fx[kFlight][kX + 1];
    unsigned sw[kFlight], sx[kFlight][kX + 1];
    auto fetch = [&](int u, int kb) {
        if (kb >= kbs) return;                                         // (wave-uniform)
        const int k = kb;
        fw[u] = *reinterpret_cast<const uintx4*>(wp + (long)k * N * 64);
        sw[u] = sp[k * rows4 * 4];
#pragma unroll
        for (int t = 0; t < kX; ++t) {
            const int m = min(16 * t + r, M - 1);
            fx[u][t] = *reinterpret_cast<const uintx4*>(xc + ((long)k * M + m) * 64 + q * 16);
            sx[u][t] = xs[(k * xrows4 + m) * 4 + q];
        }
    };
#pragma unroll
    for (int u = 0; u < kFlight; ++u) fetch(u, wave + u * waves);
    if constexpr (QUANT) {
        // eight columns per thread, four neighbouring threads a block; rows of x one after the other
        const int threads = blockDim.x, per_row = kbs * 16;
        for (int i = threadIdx.x; i < M * per_row; i += threads) {     // (a whole number of quads: per_row and threads are)
            const int m = i / per_row, t = i - m * per_row, k = t * 8;
            float v[8];
            load8(x + (long)m * K + k, K - k, vec, v);
            unsigned top = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
            const unsigned b = mx4_scale_byte(quad_max(top));
            const int at = (t >> 4) * M + m;                           // [kb][row]
            reinterpret_cast<unsigned*>(qc)[at * 16 + (t & 15)] = b == 255 ? 0u : mx4_encode8(v, mx4_scale_value(b));
            if ((t & 3) == 0) qs[at * 4 + ((t >> 2) & 3)] = (uint8_t)b;
        }
        __syncthreads();
    }
    floatx4 acc[NT] = {};
    for (int kb = wave; kb < kbs; kb += waves * kFlight) {
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
            const int k = kb + u * waves;
            const uintx4 a = fw[u];
            const unsigned sa = sw[u];
            uintx4 bx[kX + 1];
            unsigned sbx[kX + 1];
#pragma unroll
            for (int t = 0; t < kX; ++t) { bx[t] = fx[u][t]; sbx[t] = sx[u][t]; }
            fetch(u, k + waves * kFlight);
            if (k >= kbs) continue;
            const intx8 a8 = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                uintx4 b;
                unsigned sb;
                if constexpr (QUANT) {
                    const int m = min(16 * t + r, M - 1);
                    b = *reinterpret_cast<const uintx4*>(qc + ((long)k * M + m) * 64 + q * 16);
                    sb = qs[(k * M + m) * 4 + q];
                } else {
                    b = bx[t];
                    sb = sbx[t];
                }
                const intx8 b8 = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
                acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b8, acc[t], 4, 4, 0, (int)sa, 0, (int)sb);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) part[wave][t][lane] = acc[t];
    __syncthreads();
    if (wave >= NT) return;
    const int t = wave;                                                // (NT <= waves)
    floatx4 s = part[0][t][lane];
    for (int z = 1; z < waves; ++z) s += part[z][t][lane];
    const int m = 16 * t + r, n = n0 + 4 * q;
    if (m >= M || n >= N) return;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] = s[e] + (bias && n + e < N ? to_f32(bias[n + e]) : 0.f);
        if (relu) v[e] = v[e] > 0.f || v[e] != v[e] ? v[e] : 0.f;
    }
    store4<T>(y + (long)m * N + n, v, N - n, N % 4 == 0 && (reinterpret_cast<uintptr_t>(y) & (4 * sizeof(T) - 1)) == 0);
}

}  // namespace wino
