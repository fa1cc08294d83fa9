// Softmax cross entropy of linear logits, and its gradient, without the logits in memory.
//
//   l[t][v] = sum_d x[t][d] w[v][d] + bias[v]
//   lse[t]  = log sum_v exp l[t][v]                loss[t] = lse[t] - l[t][target[t]]   (0 for an ignored row)
//   dl[t][v] = grad[t] * (exp(l[t][v] - lse[t]) - [v == target[t]])                     (0 for an ignored row)
//   dx = dl w        dw = dl^T x        dbias[v] = sum_t dl[t][v]
//
// The products run on tile_gemm_kernel with the vocabulary on the tile's m side: a lane then holds one row t and up to
// 64 of its logits in registers, so the softmax statistics of a tile need no exchange between lanes but one.
// Forward: every tile leaves (max, sum of exp) per row, 8 bytes for 128 logits, and one kernel joins them.  Backward:
// the vocabulary is taken in pieces; a piece's dl goes to scratch and feeds the two products and dbias.  In fp32 it is kept
// as it is; in 16 bits as two values, what the type holds and what that leaves over (16 bits of significand in bf16, 22 in
// f16), and the products run over both, their reduction twice as long.  One value would not do, at any number of rows: its
// rounding makes the gradients' error 1.3 to 1.4 of their own rounding where the terms of their sums do not cancel, and 4.4 of
// it in dx where the classes' rows of w share a component five times as long as what tells them apart.  It would be a third
// faster where the multiplies bound the call (2048 rows, 32000 classes, D = 2048 in bf16: 1010 us for 1500).
//
// What bounds it: the multiplies.  That problem: the logits, twice, at 240 us and, with dl's two stores, 300 us; dx and dw
// over two values 2 x 237 and 2 x 232 us in two pieces of the vocabulary (1.13 to 1.15 PFLOP/s); 10 us for the statistics and
// the row weights, 13 us to join dx's parts.  In fp32 (777 x 10007 x 1003) the matrix pipe is busy for 0.8 of the products'
// time.  Small problems are bound by their launches: 250 rows, 1000 classes, D = 4096 in f16 take 47 us in five kernels, none
// above 23.
#pragma once
#include "common.hpp"
#include "tile_gemm.hpp"

namespace wino {

template <typename T> constexpr int kValues = sizeof(T) == 2 ? 2 : 1;  // that dl is kept as

constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// exp(l - ref) for many l and one ref.  16-bit tensors: one multiply-add, l log2(e) - (ref log2(e) rounded), whose error is
// |ref| 2^-24 at most and the same for every l, far below the rounding of their gradients; fp32 subtracts first.
template <typename T> struct ExpFrom {
    float ref;
    __device__ __forceinline__ explicit ExpFrom(float r) : ref(sizeof(T) == 4 ? r : r * kLog2e) {}
    __device__ __forceinline__ float operator()(float l) const {
        return sizeof(T) == 4 ? exp_of(l - ref) : __builtin_amdgcn_exp2f(__builtin_fmaf(l, kLog2e, -ref));
    }
};

// (max, sum of exp(l - max)) of the union of two sets of logits; the empty set is (-inf, 0)
__device__ __forceinline__ void stats_join(float& mx, float& sum, float mx2, float sum2) {
    const float m = fmaxf(mx, mx2);
    // both empty, or both all -inf: no exp(-inf + inf).  A NaN sum stays one: fmaxf drops the NaN of a maximum.
    const float a = mx == m ? sum : sum * exp_of(mx - m), b = mx2 == m ? sum2 : sum2 * exp_of(mx2 - m);
    sum = a + b;
    mx = m;
}

// a target outside the vocabulary that is not `ignore` makes its row's loss and gradient NaN
struct CeRows {
    const long long* target;
    long long ignore;
    int V;
};

// ---- epilogues ---------------------------------------------------------------------------------

// stats[tile][t] = (max, sum) over the tile's logits; picked[t] = the target's logit
template <typename T> struct CeStats {
    const T* bias;
    CeRows rows;
    float2* stats;
    float* picked;
    template <int BM, int BN, int WM, int WN, int MI, int NI>
    __device__ __forceinline__ void run(floatx16 (&acc)[MI][NI], const TileArgs& g, int m0, int n0, int wm, int wn, int l32, int lh, char* lds) const {
        float mx[NI], sum[NI];
#pragma unroll
        for (int n = 0; n < NI; ++n) mx[n] = -INFINITY;
        // a tile inside the vocabulary and without a bias (the epilogue's vector work is a good part of a short
        // reduction's time: T = 4096, V = 50257, D = 1024 takes 456 us with the checks everywhere, 418 without)
        auto finish = [&](auto checked) {
            constexpr bool CHECKED = decltype(checked)::value;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    if constexpr (CHECKED) {
                        const int m = m0 + (wm * MI + i) * 32 + 8 * (r >> 2) + 4 * lh + (r & 3);
                        const float b = bias && m < g.M ? to_f32(bias[m]) : 0.f;
#pragma unroll
                        for (int n = 0; n < NI; ++n) acc[i][n][r] = m < g.M ? acc[i][n][r] + b : -INFINITY;
                    }
#pragma unroll
                    for (int n = 0; n < NI; ++n) mx[n] = fmaxf(mx[n], acc[i][n][r]);
                }
        };
        if (!bias && m0 + BM <= g.M) finish(std::false_type{});
        else finish(std::true_type{});
#pragma unroll
        for (int n = 0; n < NI; ++n) {
            const int t = n0 + (wn * NI + n) * 32 + l32;
            const long long at = t < g.N ? rows.target[t] - (m0 + wm * MI * 32) : -1;
            const int want = at >= 0 && at < min(MI * 32, g.M - (m0 + wm * MI * 32)) ? (int)at : -1;
            float s = 0.f;
            const ExpFrom<T> term(mx[n] == -INFINITY ? 0.f : mx[n]);  // all -inf: exp(-inf) = 0 each
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) s += term(acc[i][n][r]);
            if (__any(want >= 0)) {                                    // few blocks hold a target
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (want == i * 32 + 8 * (r >> 2) + 4 * lh + (r & 3)) picked[t] = acc[i][n][r];
            }
            sum[n] = s;
            const float mo = __shfl_xor(mx[n], 32), so = __shfl_xor(sum[n], 32);
            stats_join(mx[n], sum[n], mo, so);
        }
        __builtin_amdgcn_s_barrier();                                  // every wave is done with the last stage
        asm volatile("" ::: "memory");
        float2* ex = reinterpret_cast<float2*>(lds);                   // [WM][BN]
        if (lh == 0) {
#pragma unroll
            for (int n = 0; n < NI; ++n) ex[wm * BN + (wn * NI + n) * 32 + l32] = make_float2(mx[n], sum[n]);
        }
        __syncthreads();
        for (int c = threadIdx.x; c < BN; c += 64 * WM * WN) {
            if (n0 + c >= g.N) continue;
            float2 a = ex[c];
#pragma unroll
            for (int k = 1; k < WM; ++k) stats_join(a.x, a.y, ex[k * BN + c].x, ex[k * BN + c].y);
            stats[(long)(m0 / BM) * g.N + n0 + c] = a;
        }
    }
};

// the weight of a row's gradient: 0 for an ignored row, NaN where the target is outside the vocabulary
__device__ __forceinline__ float row_weight(const CeRows& rows, long long target, float grad) {
    if (target == rows.ignore) return 0.f;
    return target < 0 || target >= rows.V ? NAN : grad;
}
template <typename T> __device__ __forceinline__ float dl_of(float l, const ExpFrom<T>& p, bool hit, float weight, bool ignored) {
    return ignored ? 0.f : (p(l) - (hit ? 1.f : 0.f)) * weight;
}

// what rounding to T leaves of a value (0 where there is nothing finite to leave)
template <typename T> __device__ __forceinline__ float left_over(float v) {
    const float d = v - to_f32(from_f32<T>(v));
    return d - d == 0.f ? d : 0.f;
}

// dl[t][v - v0] of a piece of the vocabulary, zeros around it (rows up to row_end, columns up to pitch)
template <typename T> struct CeDl {
    const T* bias;          // of the piece
    CeRows rows;
    const float* lse;
    const float* grad;
    const float* scale;     // one factor in device memory, or null
    int v0;                 // first class of the piece
    T* dl;
    long pitch;             // elements from row to row
    int width;              // of a row, a multiple of 8; two values: followed by `width` elements of what rounding left over
    int row_end;
    template <int BM, int BN, int WM, int WN, int MI, int NI>
    __device__ __forceinline__ void run(floatx16 (&acc)[MI][NI], const TileArgs& g, int m0, int n0, int wm, int wn, int l32, int lh, char* lds) const {
        const float f = scale ? *scale : 1.f;
        float weight[NI], z[NI];
        const bool plain = !bias && m0 + BM <= g.M;                    // no bias, inside the vocabulary
        bool none[NI];                                                 // no target in this wave's block
        int hit[NI];
        bool ignored[NI];
#pragma unroll
        for (int n = 0; n < NI; ++n) {
            const int t = n0 + (wn * NI + n) * 32 + l32;
            const bool in = t < g.N;
            const long long target = in ? rows.target[t] : rows.ignore;
            ignored[n] = !in || target == rows.ignore;
            weight[n] = in ? row_weight(rows, target, grad[t]) * f : 0.f;
            z[n] = in ? lse[t] : 0.f;
            hit[n] = target >= v0 && target - v0 < g.M ? (int)(target - v0) : -1;
            const int first = m0 + wm * MI * 32;
            none[n] = !__any(hit[n] >= first && hit[n] < first + MI * 32);
        }
        // logits to dl where they are, once for both stores
#pragma unroll
        for (int n = 0; n < NI; ++n) {
            const ExpFrom<T> p(z[n]);
            if (plain && none[n]) {
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[i][n][r] = ignored[n] ? 0.f : p(acc[i][n][r]) * weight[n];
                continue;
            }
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int m = m0 + (wm * MI + i) * 32 + 8 * (r >> 2) + 4 * lh + (r & 3);
                    const float b = bias && m < g.M ? to_f32(bias[m]) : 0.f;
                    acc[i][n][r] = m < g.M ? dl_of(acc[i][n][r] + b, p, hit[n] == m, weight[n], ignored[n]) : 0.f;
                }
        }
        tile_store<T, WM, WN, MI, NI>(dl, pitch, m0, n0, row_end, width, wm, wn, l32, lh, lds, false, [&](int i, int q, int n, float (&v)[4]) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = acc[i][n][4 * q + e];
        });
        if constexpr (kValues<T> == 2)
            tile_store<T, WM, WN, MI, NI>(dl + width, pitch, m0, n0, row_end, width, wm, wn, l32, lh, lds, false, [&](int i, int q, int n, float (&v)[4]) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = left_over<T>(acc[i][n][4 * q + e]);
            });
    }
};

// ---- kernels -----------------------------------------------------------------------------------

// loss and lse from the tiles' statistics: 32 rows x 8 parts of the tile list per workgroup
__global__ __launch_bounds__(256) static void ce_join_kernel(const float2* __restrict__ stats, const float* __restrict__ picked, CeRows rows,
                                                             int T, int tiles, float* __restrict__ loss, float* __restrict__ lse) {
    __shared__ float2 ex[8][32];
    const int c = threadIdx.x & 31, part = threadIdx.x >> 5;
    const int t = blockIdx.x * 32 + c;
    float mx = -INFINITY, sum = 0.f;
    if (t < T) {
        int k = part;
        for (; k + 24 < tiles; k += 32) {                              // four loads in flight
            float2 a[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) a[u] = stats[(long)(k + 8 * u) * T + t];
#pragma unroll
            for (int u = 0; u < 4; ++u) stats_join(mx, sum, a[u].x, a[u].y);
        }
        for (; k < tiles; k += 8) {
            const float2 a = stats[(long)k * T + t];
            stats_join(mx, sum, a.x, a.y);
        }
    }
    ex[part][c] = make_float2(mx, sum);
    __syncthreads();
    if (part != 0 || t >= T) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) stats_join(mx, sum, ex[k][c].x, ex[k][c].y);
    const float z = mx + logf(sum);
    const long long target = rows.target[t];
    lse[t] = z;
    loss[t] = target == rows.ignore ? 0.f : target < 0 || target >= rows.V ? NAN : z - picked[t];
}

// the partial sums of a cut reduction of the logits
template <typename T> struct CeParts {
    const float* part;
    int parts;
    long pitch, plane;      // elements per row, per part
    const T* bias;
};

// small problems: loss and lse of one row per workgroup from the partial sums: 256 threads of four classes each, times
// four quarters of the parts (up to 64 parts: a thread alone would wait for eight batches of loads one after the other)
template <typename T>
__global__ __launch_bounds__(1024) void ce_rows_kernel(CeParts<T> p, CeRows rows, float* __restrict__ loss, float* __restrict__ lse) {
    __shared__ floatx4 quarter[3][256];
    __shared__ float2 ex[256];
    __shared__ float picked;
    const int t = blockIdx.x, c = threadIdx.x & 255, part = threadIdx.x >> 8;
    const int per = (p.parts + 3) / 4, z0 = min(part * per, p.parts), z1 = min(z0 + per, p.parts);
    const long long target = rows.target[t];
    float mx = -INFINITY, sum = 0.f;
    for (int v0 = 0; v0 < rows.V; v0 += 1024) {
        const int v = v0 + 4 * c;
        floatx4 s = {0.f, 0.f, 0.f, 0.f};
        if (v < rows.V) s = sum_parts<floatx4>(p.part + t * p.pitch + v + z0 * p.plane, z1 - z0, p.plane);   // v + 3 < pitch
        if (part) quarter[part - 1][c] = s;
        __syncthreads();
        if (part == 0) {
#pragma unroll
            for (int k = 0; k < 3; ++k) s += quarter[k][c];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (v + e >= rows.V) continue;
                const float l = s[e] + (p.bias ? to_f32(p.bias[v + e]) : 0.f);
                if (target == v + e) picked = l;
                stats_join(mx, sum, l, l == -INFINITY ? 0.f : 1.f + (l - l));      // +inf and NaN make the row NaN
            }
        }
        __syncthreads();
    }
    if (part == 0) ex[c] = make_float2(mx, sum);
    __syncthreads();
    for (int k = 128; k > 0; k >>= 1) {
        if ((int)threadIdx.x < k) {
            stats_join(mx, sum, ex[threadIdx.x + k].x, ex[threadIdx.x + k].y);
            ex[threadIdx.x] = make_float2(mx, sum);
        }
        __syncthreads();
    }
    if (threadIdx.x != 0) return;
    const float z = mx + logf(sum);
    lse[t] = z;
    loss[t] = target == rows.ignore ? 0.f : target < 0 || target >= rows.V ? NAN : z - picked;
}

// 16-bit dl is stored relative to the largest weight: with equal weights (a mean over the rows) the targets' entries are
// then close to -1, which the type holds well, instead of all sharing the rounding error of the weight.  f16 in addition
// has only five exponent bits: times 2^15 (|exp(l - lse) - hit| <= 1, so nothing overflows), which keeps values down to
// 2^-39 of the largest weight.  `top` is 1 or 2^15; the factor is top / weight_top(), its inverse is applied to the fp32
// sums.  Called by a whole workgroup; ex holds one float per wave.
__device__ __forceinline__ float weight_top(const float* grad, const CeRows& rows, int T, float top, float* ex) {
    float mx = 0.f;
#pragma unroll 8
    for (int t = threadIdx.x; t < T; t += blockDim.x) {
        const float a = fabsf(grad[t]);                                // (read whether it counts or not: no load waits for another)
        // an infinite weight spoils its row of dx and all of dw, not the scale of the other rows of dx
        mx = fmaxf(mx, rows.target[t] != rows.ignore && a <= 3.4028235e38f ? a : 0.f);
    }
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor(mx, k));
    if ((threadIdx.x & 63) == 0) ex[threadIdx.x >> 6] = mx;
    __syncthreads();
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) mx = fmaxf(mx, ex[w]);
    return mx > 0.f ? fmaxf(mx, 1e-30f) : top;                         // no weight at all: factor 1
}
// out[0] = the factor, out[1] = its inverse
__global__ __launch_bounds__(1024) static void ce_scale_kernel(const float* __restrict__ grad, CeRows rows, int T, float top, float* __restrict__ out) {
    __shared__ float ex[16];
    const float g = weight_top(grad, rows, T, top, ex);
    if (threadIdx.x != 0) return;
    out[0] = top / g;
    out[1] = g / top;
}

// Rows copied to a 16-byte aligned pitch, zeros behind them, and in place of rows whose target is `ignore` (target null:
// none).  Backward reads x through such a copy: an ignored row's dl is zero, but zero times what an unused row of a padded
// batch may hold (a NaN, an infinity) would still reach every class's dw.
template <typename T> struct RowCopy {
    const T* x;
    T* y;
    long rows;
    int cols, pitch;                    // elements; y's pitch is a multiple of 16 bytes
    const long long* target;
    long long ignore;
    static constexpr int kPer = 16 / (int)sizeof(T);
    long blocks() const { return (rows * (pitch / kPer) + 255) / 256; }
    __device__ __forceinline__ void run(long block) const {
        const long i = block * 256 + threadIdx.x;
        const int pieces = pitch / kPer;
        const long row = i / pieces;
        if (row >= rows) return;
        const int c = (int)(i - row * pieces) * kPer;
        const T* from = x + row * cols + c;
        Pack16<T> pk;
        const bool keep = !target || target[row] != ignore;
        if (cols == pitch && (reinterpret_cast<uintptr_t>(x) & 15) == 0) {
            pk = *reinterpret_cast<const Pack16<T>*>(from);
            if (!keep) pk = __builtin_bit_cast(Pack16<T>, uintx4{0, 0, 0, 0});
        } else {
#pragma unroll
            for (int e = 0; e < kPer; ++e) pk.e[e] = keep && c + e < cols ? from[e] : from_f32<T>(0.f);
        }
        *reinterpret_cast<Pack16<T>*>(y + row * pitch + c) = pk;
    }
};
template <typename T> __global__ __launch_bounds__(256) void row_copy_kernel(RowCopy<T> c) { c.run(blockIdx.x); }

// small problems: dl from the partial sums, four classes per thread.  scale: null, or where the factor and its inverse go
// (every workgroup finds them itself, which saves a launch)
template <typename T>
__global__ __launch_bounds__(256) void ce_dl_kernel(CeParts<T> p, CeDl<T> o, int T_rows, float top, float* __restrict__ scale, int blocks,
                                                    RowCopy<T> copy) {
    __shared__ float ex[4];
    if ((int)blockIdx.x >= blocks) return copy.run(blockIdx.x - blocks);        // beside dl: x for dw
    float f = o.scale ? *o.scale : 1.f;
    if (scale) {
        const float g = weight_top(o.grad, o.rows, T_rows, top, ex);
        f = top / g;
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            scale[0] = f;
            scale[1] = g / top;
        }
    }
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    const int quads = o.width / 4;
    const int t = (int)(i / quads), m = (int)(i - (long)t * quads) * 4;
    if (t >= o.row_end) return;
    const bool in = t < T_rows;
    const long long target = in ? o.rows.target[t] : o.rows.ignore;
    const bool ignored = !in || target == o.rows.ignore;
    const float weight = in ? row_weight(o.rows, target, o.grad[t]) * f : 0.f;
    const float z = in ? o.lse[t] : 0.f;
    floatx4 l = {0.f, 0.f, 0.f, 0.f};
    if (in && m < o.rows.V) l = sum_parts<floatx4>(p.part + t * p.pitch + m, p.parts, p.plane);              // m + 3 < pitch of the parts
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float b = p.bias && m + e < o.rows.V ? to_f32(p.bias[m + e]) : 0.f;
        v[e] = in && m + e < o.rows.V ? dl_of(l[e] + b, ExpFrom<T>(z), target == m + e, weight, ignored) : 0.f;
    }
    store4<T>(o.dl + (long)t * o.pitch + m, v, 4, true);
    if constexpr (kValues<T> == 2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = left_over<T>(v[e]);
        store4<T>(o.dl + (long)t * o.pitch + o.width + m, v, 4, true);
    }
}

// dbias[v] = scale * sum_t dl[t][v], fp32: 64 classes per workgroup, 16 groups of rows shared by its waves and added in order
template <typename T> struct CeBias {
    const T* dl;
    long pitch;
    int width, rows, V;
    const float* scale;
    T* dbias;
    __device__ __forceinline__ void run(int block, float* ex) const {  // ex [16][64]
        const int c = threadIdx.x & 63, v = block * 64 + c, waves = blockDim.x >> 6;
        for (int g = threadIdx.x >> 6; g < 16; g += waves) {
            float s = 0.f;
            for (int two = 0; v < V && two < kValues<T>; ++two) {
                const T* at = dl + two * width + v;
                int t = g;
                for (; t + 112 < rows; t += 128) {                     // eight loads in flight
                    float a[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u) a[u] = to_f32(at[(long)(t + 16 * u) * pitch]);
#pragma unroll
                    for (int u = 0; u < 8; ++u) s += a[u];
                }
                for (; t < rows; t += 16) s += to_f32(at[(long)t * pitch]);
            }
            ex[g * 64 + c] = s;
        }
        __syncthreads();
        if (threadIdx.x >= 64 || v >= V) return;
        float s = ex[c];
#pragma unroll
        for (int g = 1; g < 16; ++g) s += ex[g * 64 + c];
        dbias[v] = from_f32<T>(s * (scale ? *scale : 1.f));
    }
};
template <typename T> __global__ __launch_bounds__(1024) void ce_bias_kernel(CeBias<T> b) {
    __shared__ float ex[1024];
    b.run(blockIdx.x, ex);
}

// Small problems: dx, dw and dbias in one launch.  Each alone leaves most of the chip idle and waits for its own loads (250
// rows, 1000 classes, D = 4096 in f16: 15.6 + 12.9 + 4.2 us one after the other, 21.7 together).
template <typename T>
__global__ __launch_bounds__(256, 2) void ce_gradients_kernel(CeBias<T> bias, int nb, TileArgs gx, TileStore<T> x, int nx, TileArgs gw, TileStore<T> w) {
    __shared__ __align__(1024) char lds[kSmallRing<T> * kTileSlot<T, 64, 64, 128>];
    const int b = blockIdx.x;
    if (b < nb) bias.run(b, reinterpret_cast<float*>(lds));            // (the longest wait first)
    else if (b < nb + nx) tile_gemm<T, K_OUTER, K_INNER, 64, 64, 2, 2, 128, kSmallRing<T>>(gx, x, b - nb, 0, lds);
    else tile_gemm<T, K_OUTER, K_OUTER, 64, 64, 2, 2, 128, kSmallRing<T>>(gw, w, b - nb - nx, 0, lds);
}

}  // namespace wino
