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

// A workgroup takes 16 rows x 128 columns: a thread eight columns, four neighbouring threads a block.
template <typename T>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const T* __restrict__ x, int rows, int K, uint8_t* __restrict__ codes,
                                                           uint8_t* __restrict__ scales, int vec) {
    const unsigned kbs = (K + kMxCols - 1) / kMxCols;
    const int row = blockIdx.x / kbs * 16 + (threadIdx.x >> 4), t = threadIdx.x & 15;
    const int kb = blockIdx.x % kbs;
    if (row >= rows) return;
    const int k = kb * kMxCols + t * 8;
    float v[8];
    load8(x + (long)row * K + k, K - k, vec, v);
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    const unsigned b = mx4_scale_byte(quad_max(top));
    const unsigned c = b == 255 ? 0u : mx4_encode8(v, mx4_scale_value(b));
    reinterpret_cast<unsigned*>(codes)[((long)kb * rows + row) * 16 + t] = c;
    if ((t & 3) == 0) {
        uint8_t* s = scales + ((long)kb * ((rows + 3) & ~3) + row) * 4 + (t >> 2);
        *s = (uint8_t)b;
        if (row == rows - 1)                                     // the rows that pad the count to four
            for (int r = rows; r & 3; ++r) s[4 * (r - row)] = 0;
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
    const unsigned kbs = (K + kMxCols - 1) / kMxCols;
    const int row = blockIdx.x / kbs * 16 + (threadIdx.x >> 4), t = threadIdx.x & 15;
    const int kb = blockIdx.x % kbs;
    const int k = kb * kMxCols + t * 8;
    if (row >= rows || k >= K) return;
    const unsigned c = reinterpret_cast<const unsigned*>(codes)[((long)kb * rows + row) * 16 + t];
    const int b = scales[((long)kb * ((rows + 3) & ~3) + row) * 4 + (t >> 2)];
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = mx4_value(c >> (4 * e), b);
    T* to = x + (long)row * K + k;
    constexpr int n = 16 / (int)sizeof(T);
    if (vec && K - k >= 8) {
#pragma unroll
        for (int p = 0; p < 8 / n; ++p) store_chan_vec<T>(to + p * n, v + p * n);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (k + e < K) to[e] = from_f32<T>(v[e]);
}

}  // namespace wino
