// Matrix product on MFMA for row-major operands (the fully connected layers and the softmax cross entropy):
//
//   out[n][m] = sum_k A[m][k] * B[n][k]
//
// An operand is stored either with its reduction index contiguous (K_INNER: rows of k) or with it outermost (K_OUTER:
// one row per k); the four products of a linear layer and its gradients need both.  Types: fp32, f16, bf16, and
// microscaled 4-bit values (mx4_t, K_INNER only).
//
// All types share one shape in BYTES: a stage is 128 bytes of k per operand row (32 fp32, 64 16-bit, 256 4-bit
// elements), and a 16-byte piece of a row is one multiply's share of a lane (v_mfma_f32_32x32x16_{f16,bf16},
// v_mfma_scale_f32_32x32x64_f8f6f4, or four v_mfma_f32_32x32x2_f32).  Lane half lh takes the pieces 4*lh + j,
// j = 0..3: the sum does not care which half takes which k as long as both operands agree, and this way the block
// scales of a lane's four 4-bit pieces are the four bytes of one dword, picked by the instruction's byte selector.
//
// Operands move HBM -> LDS by direct 16-byte loads into a ring of stages; rows past the end are clamped to the last
// one (their results are never stored).  LDS holds K_INNER rows of 128 bytes with their pieces exchanged by the row's
// low bits, so that the 16-byte reads of 32 rows spread over the banks; K_OUTER tiles keep the k rows, and 16-bit
// fragments are read through the transposing LDS read (ds_read_b64_tr_b16: the 16 lanes of a group supply four k rows
// of 16 elements and each receives one column), fp32 ones element by element.
//
// The accumulator of a 32x32 block has its n index on the lanes and four consecutive m in consecutive registers, so
// every output with m contiguous in memory is written in vectors of four.
#pragma once
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "mma.hpp"

namespace wino {

typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

struct mx4_t {};          // 32 values per 16-byte piece, with a power-of-two scale byte per piece

enum { K_INNER = 0, K_OUTER = 1 };

// elements of k per 16-byte piece and per stage
template <typename T> struct TileElem { static constexpr int piece = 16 / (int)sizeof(T), stage = 8 * piece, bytes = (int)sizeof(T); };
template <> struct TileElem<mx4_t> { static constexpr int piece = 32, stage = 256, bytes = 0; };

struct TileOperand {
    const char* p;          // first byte of the operand
    const char* scale;      // mx4: [k stage][rows rounded up to 2][8] scale bytes
    long pitch;             // K_INNER: bytes from row to row; K_OUTER: bytes from one k row to the next
    long step;              // bytes from stage to stage
    int rows;               // K_INNER: rows (m or n); K_OUTER: k rows that may be read
    int pieces;             // K_OUTER: 16-byte pieces per k row that may be read
};

struct TileArgs {
    TileOperand a, b;
    int M, N, K;            // K in elements
    int mt, nt;             // tiles along m and n
    int stages, split;      // stages in all, stages per part of the reduction (grid.y parts)
};

// the j-th of a lane's four scale bytes: a compile-time operand of the instruction
template <typename T, int J> __device__ __forceinline__ void tile_mma(const uintx4& a, const uintx4& b, floatx16& c, unsigned sa, unsigned sb) {
    if constexpr (std::is_same<T, mx4_t>::value) {
        const intx8 a8 = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
        const intx8 b8 = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
        c = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, 4, 4, J, (int)sa, J, (int)sb);
    } else {
        typedef typename Mma<T>::vec vec;
        Mma<T>::run(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c);
    }
}

__device__ __forceinline__ unsigned lds_addr(const void* p) {
    return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// 1 KB HBM -> LDS: lane l moves the 16 bytes at sbase + off to dst + 16*l (dma_row with an LDS address)
__device__ __forceinline__ void dma_piece(uint64_t sbase, unsigned off, unsigned dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(dst)), "v"(off), "s"(sbase) : "memory");
}

template <int N> __device__ __forceinline__ void wait_loads() {      // at most N loads in flight, every LDS read returned
    static_assert(N < 64, "six bits of vmcnt");
    __builtin_amdgcn_s_waitcnt((N & 0xF) | (0x7 << 4) | (0x0 << 8) | ((N >> 4) << 14));
}

// One operand's side of a workgroup's tile: EXT rows (or columns) of it starting at org.
template <typename T, int ORDER, int EXT, int WAVES> struct TileSide {
    static constexpr int kBytes = EXT * 128;                           // of a stage in LDS, either order
    static constexpr int kLoads = kBytes / 1024 / WAVES;               // 1 KB loads per wave and stage
    static constexpr int kRow = EXT * TileElem<T>::bytes;              // K_OUTER: bytes of a k row in LDS
    static constexpr bool kOuter = ORDER == K_OUTER;
    static constexpr bool kMx4 = std::is_same<T, mx4_t>::value;
    static_assert(kBytes % (1024 * WAVES) == 0, "whole loads per wave");

    uint64_t base;            // of the stage to load next
    unsigned off[kLoads];
    unsigned rd[4];           // K_INNER: a lane's LDS offsets of its pieces j = 0..3 (of 32-row block 0)

    // position in a k row (in pieces) that holds piece c; an involution
    static __device__ __forceinline__ int outer_swap(int krow, int c) {
        constexpr int inside = kRow / 16 - 1;                           // narrow tiles: as far as their rows reach
        return TileElem<T>::bytes == 4 ? c ^ ((((krow >> 4) & 1) * 8) & inside) : c ^ (((krow & 3) * 4) & inside);
    }
    static __device__ __forceinline__ int inner_swap(int row) { return (row >> 1) & 7; }

    // byte offset, from the tile's origin in the stage at hand, of what this lane loads with load q of its wave;
    // k_left: k pieces (K_INNER) or k rows (K_OUTER) of the stage that exist
    static __device__ __forceinline__ unsigned source(const TileOperand& op, int org, int q, int wave, int lane, int k_left) {
        const int at = (wave * kLoads + q) * 1024 + lane * 16;
        if constexpr (!kOuter) {
            const int row = at >> 7;
            const int c = min((lane & 7) ^ inner_swap(row), k_left - 1);
            return (unsigned)((long)max(min(row, op.rows - 1 - org), 0) * op.pitch) + c * 16;
        } else {
            const int krow = at / kRow;
            const int org_piece = org / TileElem<T>::piece;
            const int c = min(outer_swap(krow, (at % kRow) >> 4), op.pieces - 1 - org_piece);
            return (unsigned)((long)min(krow, k_left - 1) * op.pitch) + c * 16;
        }
    }
    // what exists of a stage that starts at element k0 of the reduction
    static __device__ __forceinline__ int left(const TileOperand& op, int K, int k0) {
        if constexpr (!kOuter) return min(8, (K - k0 + TileElem<T>::piece - 1) / TileElem<T>::piece);
        return op.rows - k0;
    }

    __device__ __forceinline__ void init(const TileOperand& op, int org, int stage0, int wave, int lane) {
        // a tile may lie wholly behind the last row (an epilogue's cover): it then reads the last row
        const uint64_t origin = kOuter ? (uint64_t)org * TileElem<T>::bytes : (uint64_t)min(org, op.rows - 1) * (uint64_t)op.pitch;
        base = uniform64((uint64_t)op.p + origin + (uint64_t)stage0 * (uint64_t)op.step);
        const int whole = kOuter ? 1 << 30 : 8;
#pragma unroll
        for (int q = 0; q < kLoads; ++q) off[q] = source(op, org, q, wave, lane, whole);
        if constexpr (!kOuter) {
            const int l32 = lane & 31, lh = lane >> 5;
#pragma unroll
            for (int j = 0; j < 4; ++j) rd[j] = l32 * 128 + (((4 * lh + j) ^ inner_swap(l32)) << 4);
        }
    }
    __device__ __forceinline__ void load(const TileOperand& op, unsigned dst, int wave) {
#pragma unroll
        for (int q = 0; q < kLoads; ++q) dma_piece(base, off[q], dst + (wave * kLoads + q) * 1024);
        base += (uint64_t)op.step;
    }
    // the last stage of a reduction that does not fill it
    __device__ __forceinline__ void load_tail(const TileOperand& op, int org, int k_left, unsigned dst, int wave, int lane) {
#pragma unroll
        for (int q = 0; q < kLoads; ++q)
            dma_piece(base, source(op, org, q, wave, lane, k_left), dst + (wave * kLoads + q) * 1024);
    }
    // piece j of block `blk` (32 rows or columns) for this lane
    __device__ __forceinline__ uintx4 fragment(const char* st, int blk, int j, int lane) const {
        if constexpr (!kOuter) {
            return *reinterpret_cast<const uintx4*>(st + rd[j] + blk * 4096);
        } else if constexpr (TileElem<T>::bytes == 2) {
            const int row = 8 * (4 * (lane >> 5) + j) + ((lane >> 2) & 3);            // row & 3 == (lane >> 2) & 3
            const int piece = outer_swap(row, blk * 4 + ((lane >> 4) & 1) * 2) * 16 + (lane & 3) * 8;
            typedef __attribute__((address_space(3))) shortx4* ldsp;
            const char* at = st + row * kRow + piece;
            const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ldsp)(at));
            const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ldsp)(at + 4 * kRow));
            typedef unsigned uintx2 __attribute__((ext_vector_type(2)));
            const uintx2 l = __builtin_bit_cast(uintx2, lo), h = __builtin_bit_cast(uintx2, hi);
            return uintx4{l[0], l[1], h[0], h[1]};
        } else {
            const int row = 4 * (4 * (lane >> 5) + j);
            const int col = outer_swap(row, blk * 8 + ((lane & 31) >> 2)) * 16 + (lane & 3) * 4;
            uintx4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const unsigned*>(st + (row + e) * kRow + col);
            return v;
        }
    }
};

// Workgroup id -> tile.  Ids go round-robin to the 8 XCDs: an XCD takes a contiguous run of the tile sequence, and the
// sequence walks groups of 8 n tiles so that the tiles an XCD works on at once share their operands in its L2.
__device__ __forceinline__ bool tile_of(int id, int mt, int nt, int& tm, int& tn) {
    const int total = mt * nt, per = (total + 7) / 8;
    const int t = (id & 7) * per + (id >> 3);
    if ((id >> 3) >= per || t >= total) return false;
    constexpr int G = 8;
    const int group = t / (G * mt), first = group * G, width = min(G, nt - first), r = t - group * G * mt;
    tn = first + r % width;
    tm = r / width;
    return true;
}
inline int tile_grid(int mt, int nt) { return (mt * nt + 7) / 8 * 8; }

// WM x WN waves; a wave owns BM/WM x BN/WN of the tile.  RING stages of LDS, RING - 1 of them in flight.
template <typename T, int AO, int BO, int BM, int BN, int WM, int WN, int RING, class Epi>
__global__ __launch_bounds__(64 * WM * WN, WM * WN > 4 ? 1 : 2) void tile_gemm_kernel(TileArgs g, Epi epi) {
    constexpr int WAVES = WM * WN, MI = BM / WM / 32, NI = BN / WN / 32;
    constexpr bool MX4 = std::is_same<T, mx4_t>::value;
    typedef TileSide<T, AO, BM, WAVES> SA;
    typedef TileSide<T, BO, BN, WAVES> SB;
    // scale bytes of a stage: 8 per row, loaded 1 KB (128 rows) at a time
    constexpr int SCA = (BM + 127) / 128, SCB = (BN + 127) / 128;
    constexpr int SC = MX4 ? (SCA + SCB) * 1024 : 0;
    constexpr int SLOT = SA::kBytes + SB::kBytes + SC;
    __shared__ __align__(1024) char lds[RING * SLOT];

    int tm, tn;
    if (!tile_of(blockIdx.x, g.mt, g.nt, tm, tn)) return;
    const int m0 = tm * BM, n0 = tn * BN;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int l32 = lane & 31, lh = lane >> 5;
    const int first = blockIdx.y * g.split, last = min(first + g.split, g.stages);
    const bool ragged = last == g.stages && g.K % TileElem<T>::stage != 0;   // the last stage is a part of one

    SA sa;
    SB sb;
    sa.init(g.a, m0, first, wave, lane);
    sb.init(g.b, n0, first, wave, lane);
    const unsigned lds0 = lds_addr(lds);
    // mx4: scale bytes as 16-byte pieces (two rows), one load each by the first waves
    uint64_t sc_base = 0;
    unsigned sc_off = 0, sc_dst = 0;
    long sc_step = 0;
    static_assert(!MX4 || SCA + SCB <= WAVES, "a scale load per wave at most");
    if constexpr (MX4) {
        if (wave < SCA + SCB) {
            const bool isa = wave < SCA;
            const TileOperand& op = isa ? g.a : g.b;
            const int part = isa ? wave : wave - SCA, org = isa ? m0 : n0;
            const int rows2 = (op.rows + 1) >> 1;                                   // 16-byte pieces per stage
            sc_step = (long)rows2 * 16;
            sc_base = uniform64((uint64_t)op.scale + (uint64_t)first * (uint64_t)sc_step);
            sc_off = (unsigned)min(org / 2 + part * 64 + lane, rows2 - 1) * 16u;
            sc_dst = SA::kBytes + SB::kBytes + wave * 1024;
        }
    }

    floatx16 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int n = 0; n < NI; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][n][r] = 0.f;

    auto issue = [&](int s, int slot) {
        const unsigned dst = lds0 + slot * SLOT;
        if (ragged && s == last - 1) {
            const int k0 = s * TileElem<T>::stage;
            sa.load_tail(g.a, m0, SA::left(g.a, g.K, k0), dst, wave, lane);
            sb.load_tail(g.b, n0, SB::left(g.b, g.K, k0), dst + SA::kBytes, wave, lane);
        } else {
            sa.load(g.a, dst, wave);
            sb.load(g.b, dst + SA::kBytes, wave);
        }
        if constexpr (MX4) {
            if (wave < SCA + SCB) {
                dma_piece(sc_base, sc_off, dst + sc_dst);
                sc_base += (uint64_t)sc_step;
            }
        }
    };
    // Two sets of fragments: while one step's are multiplied the next step's are on their way from LDS, across the stage
    // border too.  The border sits before a stage's last multiplies: by then every wave holds the stage's last fragments,
    // so its slot can be refilled, and the multiplies cover the barrier, the requests and the first reads of the next stage.
    uintx4 fa[2][MI], fb[2][NI];
    unsigned qa[2][MI] = {}, qb[2][NI] = {};
    auto read = [&](int slot, auto jc) {
        constexpr int J = decltype(jc)::value;
        const char* sta = lds + slot * SLOT;
        const char* stb = sta + SA::kBytes;
#pragma unroll
        for (int i = 0; i < MI; ++i) fa[J & 1][i] = sa.fragment(sta, wm * MI + i, J, lane);
#pragma unroll
        for (int n = 0; n < NI; ++n) fb[J & 1][n] = sb.fragment(stb, wn * NI + n, J, lane);
    };
    auto read_scales = [&](int slot, int set) {
        if constexpr (MX4) {
            const char* sca = lds + slot * SLOT + SA::kBytes + SB::kBytes;
#pragma unroll
            for (int i = 0; i < MI; ++i) qa[set][i] = *reinterpret_cast<const unsigned*>(sca + ((wm * MI + i) * 32 + l32) * 8 + lh * 4);
#pragma unroll
            for (int n = 0; n < NI; ++n) qb[set][n] = *reinterpret_cast<const unsigned*>(sca + SCA * 1024 + ((wn * NI + n) * 32 + l32) * 8 + lh * 4);
        }
    };
    auto multiply = [&](int s, auto jc, auto tail) {
        constexpr int J = decltype(jc)::value;
        if constexpr (decltype(tail)::value && !MX4) {
            // pieces past the end of the reduction: zero wherever k is inner (they were read from elsewhere in the
            // row).  A k-outer operand needs no mask beside a k-inner one; where both are k-outer, the rows past
            // the end exist and one of the two holds zeros in them.
            const bool in = 4 * lh + J < (g.K - s * TileElem<T>::stage + TileElem<T>::piece - 1) / TileElem<T>::piece;
#pragma unroll
            for (int i = 0; i < MI; ++i)
                if (AO == K_INNER && !in) fa[J & 1][i] = uintx4{0, 0, 0, 0};
#pragma unroll
            for (int n = 0; n < NI; ++n)
                if (BO == K_INNER && !in) fb[J & 1][n] = uintx4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int n = 0; n < NI; ++n) tile_mma<T, J>(fa[J & 1][i], fb[J & 1][n], acc[i][n], qa[0][i], qb[0][n]);
    };
    const std::integral_constant<int, 0> j0;
    const std::integral_constant<int, 1> j1;
    const std::integral_constant<int, 2> j2;
    const std::integral_constant<int, 3> j3;
    constexpr int LPW = SA::kLoads + SB::kLoads;

    const int ahead = min(first + RING, last);
    for (int s = first; s < ahead; ++s) issue(s, s - first);
    if (ahead - first == RING) wait_loads<(RING - 1) * LPW>();
    else wait_loads<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(0, j0);
    read_scales(0, 0);
    int slot = 0;
    for (int s = first; s < last - 1; ++s) {
        read(slot, j1);
        __builtin_amdgcn_sched_barrier(0);
        multiply(s, j0, std::false_type{});
        __builtin_amdgcn_sched_barrier(0);
        read(slot, j2);
        __builtin_amdgcn_sched_barrier(0);
        multiply(s, j1, std::false_type{});
        __builtin_amdgcn_sched_barrier(0);
        read(slot, j3);
        __builtin_amdgcn_sched_barrier(0);
        multiply(s, j2, std::false_type{});
        __builtin_amdgcn_sched_barrier(0);
        // stage s + 1 has landed (the RING - 2 behind it may still be in flight, fewer near the end) and this wave has read
        // all of stage s; behind the barrier that holds for every wave
        asm volatile("" ::: "memory");
        if (RING > 2 && s + RING <= last) wait_loads<(RING - 2) * LPW>();
        else wait_loads<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (s + RING < last) issue(s + RING, slot);
        slot = slot + 1 == RING ? 0 : slot + 1;
        read(slot, j0);
        read_scales(slot, 1);
        __builtin_amdgcn_sched_barrier(0);
        multiply(s, j3, std::false_type{});
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (MX4) {
#pragma unroll
            for (int i = 0; i < MI; ++i) qa[0][i] = qa[1][i];
#pragma unroll
            for (int n = 0; n < NI; ++n) qb[0][n] = qb[1][n];
        }
    }
    read(slot, j1);
    multiply(last - 1, j0, std::true_type{});
    read(slot, j2);
    multiply(last - 1, j1, std::true_type{});
    read(slot, j3);
    multiply(last - 1, j2, std::true_type{});
    multiply(last - 1, j3, std::true_type{});
    wait_loads<0>();
    epi.template run<BM, BN, WM, WN, MI, NI>(acc, g, m0, n0, wm, wn, l32, lh, lds);
}

// ---- epilogues ---------------------------------------------------------------------------------

// four consecutive elements of an output row; vec: the row and its base allow one store
template <typename T> __device__ __forceinline__ void store4(T* y, const float (&v)[4], int left, bool vec) {
    if (vec && left >= 4) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<floatx4*>(y) = floatx4{v[0], v[1], v[2], v[3]};
        } else {
            typedef unsigned uintx2 __attribute__((ext_vector_type(2)));
            *reinterpret_cast<uintx2*>(y) = uintx2{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < left) y[e] = from_f32<T>(v[e]);
}

// out[n][m] = relu?( scale * acc + bias[m] ), rounded to T once
template <typename T> struct TileStore {
    T* out;
    long pitch;             // elements
    const T* bias;          // or null
    const float* scale;     // one factor in device memory, or null
    int relu;
    template <int BM, int BN, int WM, int WN, int MI, int NI>
    __device__ __forceinline__ void run(floatx16 (&acc)[MI][NI], const TileArgs& g, int m0, int n0, int wm, int wn, int l32, int lh, char*) const {
        const bool vec = pitch % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & (4 * sizeof(T) - 1)) == 0;
        const float f = scale ? *scale : 1.f;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int m = m0 + (wm * MI + i) * 32 + 8 * q + 4 * lh;
                if (m >= g.M) continue;
                float b[4] = {0.f, 0.f, 0.f, 0.f};
                if (bias) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (m + e < g.M) b[e] = to_f32(bias[m + e]);
                }
#pragma unroll
                for (int n = 0; n < NI; ++n) {
                    const int row = n0 + (wn * NI + n) * 32 + l32;
                    if (row >= g.N) continue;
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v[e] = acc[i][n][4 * q + e] * f + b[e];
                        if (relu) v[e] = v[e] > 0.f || v[e] != v[e] ? v[e] : 0.f;      // a NaN stays one
                    }
                    store4<T>(out + row * pitch + m, v, g.M - m, vec);
                }
            }
    }
};

// part[z][n][m] (fp32) = acc, or += where `add` is set (a tile is owned by one workgroup: the order is fixed)
struct TilePart {
    float* part;
    long pitch;             // elements, a multiple of 4; part is 16-byte aligned
    int add;
    template <int BM, int BN, int WM, int WN, int MI, int NI>
    __device__ __forceinline__ void run(floatx16 (&acc)[MI][NI], const TileArgs& g, int m0, int n0, int wm, int wn, int l32, int lh, char*) const {
        float* to = part + (long)blockIdx.y * g.N * pitch;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int m = m0 + (wm * MI + i) * 32 + 8 * q + 4 * lh;
                if (m >= g.M) continue;
#pragma unroll
                for (int n = 0; n < NI; ++n) {
                    const int row = n0 + (wn * NI + n) * 32 + l32;
                    if (row >= g.N) continue;
                    floatx4* at = reinterpret_cast<floatx4*>(to + row * pitch + m);    // m + 3 < pitch
                    floatx4 v = {acc[i][n][4 * q], acc[i][n][4 * q + 1], acc[i][n][4 * q + 2], acc[i][n][4 * q + 3]};
                    if (add) v += *at;
                    *at = v;
                }
            }
    }
};

// at[0] + at[plane] + ... in order, eight loads in flight
template <typename V> __device__ __forceinline__ V sum_parts(const float* at, int parts, long plane) {
    V s = {};
    int z = 0;
    for (; z + 8 <= parts; z += 8) {
        V a[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) a[u] = *reinterpret_cast<const V*>(at + (z + u) * plane);
#pragma unroll
        for (int u = 0; u < 8; ++u) s += a[u];
    }
    for (; z < parts; ++z) s += *reinterpret_cast<const V*>(at + z * plane);
    return s;
}

// out[n][m] = relu?( scale * sum_z part[z][n][m] + bias[m] ): four m per thread, parts added in order
template <typename T>
__global__ __launch_bounds__(256) void tile_join_kernel(const float* __restrict__ part, int parts, long part_pitch, int M, int N,
                                                        TileStore<T> o) {
    const int quads = (M + 3) / 4;
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long)quads * N) return;
    const long row = i / quads;
    const int m = (int)(i - row * quads) * 4;
    const floatx4 s = sum_parts<floatx4>(part + row * part_pitch + m, parts, (long)N * part_pitch);
    const bool vec = o.pitch % 4 == 0 && (reinterpret_cast<uintptr_t>(o.out) & (4 * sizeof(T) - 1)) == 0;
    const float f = o.scale ? *o.scale : 1.f;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] = s[e] * f + (o.bias && m + e < M ? to_f32(o.bias[m + e]) : 0.f);
        if (o.relu) v[e] = v[e] > 0.f || v[e] != v[e] ? v[e] : 0.f;
    }
    store4<T>(o.out + row * o.pitch + m, v, M - m, vec);
}

// ---- host side -----------------------------------------------------------------------------------

constexpr int kTile = 128;               // edge of a tile

inline int ceil_div(long a, long b) { return (int)((a + b - 1) / b); }

template <typename T, int AO, int BO, int BM, int BN, int WM, int WN, int RING, class Epi>
inline void tile_launch_as(TileArgs g, const Epi& epi, int parts, int cover, hipStream_t s) {
    g.mt = ceil_div(g.M, BM);
    g.nt = ceil_div(cover, BN);
    g.stages = ceil_div(g.K, TileElem<T>::stage);
    g.split = ceil_div(g.stages, parts);
    parts = ceil_div(g.stages, g.split);
    hipLaunchKernelGGL((tile_gemm_kernel<T, AO, BO, BM, BN, WM, WN, RING, Epi>), dim3(tile_grid(g.mt, g.nt), parts), dim3(64 * WM * WN), 0, s, g, epi);
}

// How a product is cut: the tile (256 x 256, or 128 x cols) and the parts of its reduction.
struct TilePick {
    int big, cols, parts;
    int edge() const { return big ? 256 : kTile; }      // m extent of a tile
};

// The cut with the smallest estimated time.  A CU works through its share of the (tile, part) items; an item takes the
// longer of its multiplies and its operands' way into LDS; parts are written and read back once in fp32 by one more
// launch.  `most` bounds the parts (1: the epilogue needs whole sums).  Rates in products / bytes per microsecond and CU,
// fitted to the measured products of the classifier's sizes.
template <typename T> inline TilePick tile_pick(int M, int N, int K, int most, int cus) {
    constexpr bool F32 = std::is_same<T, float>::value, MX4 = std::is_same<T, mx4_t>::value;
    const double rate = F32 ? 0.28e6 : MX4 ? 6.5e6 : 2.1e6, rate_big = F32 ? 0.28e6 : MX4 ? 8.0e6 : 2.8e6, bytes = 45e3;
    const int stages = ceil_div(K, TileElem<T>::stage);
    TilePick best = {0, kTile, 1};
    double least = 1e30;
    for (int kind = 0; kind < 2; ++kind) {
        const int cols = kind ? 256 : N <= 32 ? 32 : N <= 64 ? 64 : kTile, rows = kind ? 256 : kTile;
        const long tiles = (long)ceil_div(M, rows) * ceil_div(N, cols);
        if (kind && (M <= kTile || N <= kTile)) continue;
        for (int parts = 1; parts <= most && parts <= std::max(1, stages / 2); parts += parts < 8 ? 1 : parts / 4) {
            const int split = ceil_div(stages, parts);
            if (ceil_div(stages, split) != parts) continue;
            const long items = tiles * parts;
            if (parts > 1 && (items > 4L * cus || (size_t)parts * M * N * 4 > (64u << 20))) break;
            const double k = (double)split * TileElem<T>::stage;
            const double mul = (double)rows * cols * k / (kind ? rate_big : rate);
            const double move = (double)(rows + cols) * split * 128 / bytes;
            // one small tile alone on its CU waits for its own loads
            const double item = std::max(mul, move) * (!kind && items <= cus ? 1.25 : 1.0);
            const double t = ceil_div(items, cus) * item + (parts > 1 ? 4.0 + (double)parts * M * N * 8 / 4e6 : 0.0);
            if (t < least) {
                least = t;
                best = {kind, cols, parts};
            }
        }
    }
    return best;
}

// `cover`: rows of n that the epilogue has to reach (N or a little more)
template <typename T, int AO, int BO, class Epi>
inline void tile_launch(const TileArgs& g, const Epi& epi, const TilePick& pick, int cover, hipStream_t s) {
    if (pick.big) return tile_launch_as<T, AO, BO, 256, 256, 2, 4, 2>(g, epi, pick.parts, cover, s);
    switch (pick.cols) {
    case 32: return tile_launch_as<T, AO, BO, kTile, 32, 4, 1, std::is_same<T, mx4_t>::value ? 3 : 4>(g, epi, pick.parts, cover, s);
    case 64: return tile_launch_as<T, AO, BO, kTile, 64, 4, 1, 3>(g, epi, pick.parts, cover, s);
    default: return tile_launch_as<T, AO, BO, kTile, kTile, 2, 2, 2>(g, epi, pick.parts, cover, s);
    }
}

inline size_t part_bytes(int M, int N, int parts) { return (size_t)parts * N * round_up(M, 4) * sizeof(float); }

}  // namespace wino
