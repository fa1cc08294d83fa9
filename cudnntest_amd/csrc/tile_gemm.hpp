// Matrix product on MFMA for row-major operands (the fully connected layers and the softmax cross entropy):
//
//   out[n][m] = sum_k A[m][k] * B[n][k]
//
// An operand is stored either with its reduction index contiguous (K_INNER: rows of k) or with it outermost (K_OUTER:
// one row per k); the four products of a linear layer and its gradients need both.  Types: fp32, f16, bf16, and
// microscaled 4-bit values (mx4_t, K_INNER only).
//
// All types share one shape in BYTES: a stage is RB = 128 bytes of k per operand row (32 fp32, 64 16-bit elements; 64 bytes =
// 128 elements of 4-bit operands, as they are stored), and a 16-byte piece of a row is one multiply's share of a lane
// (v_mfma_f32_32x32x16_{f16,bf16}, v_mfma_scale_f32_32x32x64_f8f6f4, or four v_mfma_f32_32x32x2_f32).  Of a row's 2 S pieces
// lane half lh takes S*lh + j, j = 0 .. S - 1: the sum does not care which half takes which k as long as both operands agree,
// and this way the block scales of a lane's 4-bit pieces are neighbouring bytes, read at once and picked by the instruction's
// byte selector.
//
// Operands move HBM -> LDS by direct 16-byte loads into a ring of stages; rows past the end are clamped to the last
// one (their results are never stored).  LDS holds K_INNER rows of RB bytes with their pieces exchanged by the row's
// low bits, so that the 16-byte reads of 32 rows spread over the banks; K_OUTER tiles keep the k rows, and 16-bit
// fragments are read through the transposing LDS read (ds_read_b64_tr_b16: the 16 lanes of a group supply four k rows
// of 16 elements and each receives one column), fp32 ones element by element.
//
// The accumulator of a 32x32 block has its n index on the lanes and four consecutive m in consecutive registers, so
// every output with m contiguous in memory is written in vectors of four.
#pragma once
#include <algorithm>
#include <type_traits>
#include <utility>

#include "common.hpp"
#include "mma.hpp"

namespace wino {

typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

struct mx4_t {};          // 32 values per 16-byte piece, with a power-of-two scale byte per piece

enum { K_INNER = 0, K_OUTER = 1 };

// elements of k per 16-byte piece
template <typename T> struct TileElem { static constexpr int piece = 16 / (int)sizeof(T), bytes = (int)sizeof(T); };
template <> struct TileElem<mx4_t> { static constexpr int piece = 32, bytes = 0; };

struct TileOperand {
    const char* p;          // first byte of the operand
    const char* scale;      // mx4: [k stage][rows rounded up to 4][4] scale bytes
    long pitch;             // K_INNER: bytes from row to row; K_OUTER: bytes from one k row to the next
    long step;              // bytes from stage to stage (set by the launch)
    int rows;               // K_INNER: rows (m or n); K_OUTER: k rows that may be read
    int pieces;             // K_OUTER: 16-byte pieces per k row that may be read
};

struct TileArgs {
    TileOperand a, b;
    int M, N, K;            // K in elements (of one pass)
    int passes;             // 2: the reduction runs twice, the operands starting over at a_turn / b_turn (0 counts as 1)
    long a_turn, b_turn;    // bytes added behind a pass's last stage
    int mt, nt;             // tiles along m and n
    int stages, split;      // stages in all, stages per part of the reduction (grid.y parts)
    int pass, tail_at;      // stages of a pass; the one of them that does not exist in full, or -1 (set by the launch)
};

// J: which of a lane's scale bytes, a compile-time operand of the instruction
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

template <int... S, class F> __device__ __forceinline__ void for_each_step(std::integer_sequence<int, S...>, F&& f) {
    (f(std::integral_constant<int, S>{}), ...);
}

template <int N> __device__ __forceinline__ void wait_loads() {      // at most N loads in flight, every LDS read returned
    static_assert(N < 64, "six bits of vmcnt");
    __builtin_amdgcn_s_waitcnt((N & 0xF) | (0x7 << 4) | (0x0 << 8) | ((N >> 4) << 14));
}

// One operand's side of a workgroup's tile: EXT rows (or columns) of it starting at org.
template <typename T, int ORDER, int EXT, int WAVES, int RB> struct TileSide {
    static constexpr int kPieces = RB / 16, kSteps = kPieces / 2;      // of a row and stage, of a lane half
    static constexpr int kBytes = EXT * RB;                            // of a stage in LDS, either order
    static constexpr int kLoads = kBytes / 1024 / WAVES;               // 1 KB loads per wave and stage
    static constexpr int kRow = EXT * TileElem<T>::bytes;              // K_OUTER: bytes of a k row in LDS
    static constexpr bool kOuter = ORDER == K_OUTER;
    static_assert(kBytes % (1024 * WAVES) == 0, "whole loads per wave");

    uint64_t base;            // of the stage to load next
    unsigned off[kLoads];
    unsigned rd[kSteps];      // K_INNER: a lane's LDS offsets of its pieces j (of 32-row block 0)

    // position in a k row (in pieces) that holds piece c; an involution
    static __device__ __forceinline__ int outer_swap(int krow, int c) {
        constexpr int inside = kRow / 16 - 1;                           // narrow tiles: as far as their rows reach
        return TileElem<T>::bytes == 4 ? c ^ ((krow / (4 * kSteps) & 1) * 8 & inside) : c ^ (((krow & 3) * 4) & inside);
    }
    // 16 neighbouring rows of one piece: spread over the 16 pieces of 256 bytes, a sweep of the banks
    static __device__ __forceinline__ int inner_swap(int row) { return row / (16 / kPieces) & (kPieces - 1); }

    // byte offset, from the tile's origin in the stage at hand, of what this lane loads with load q of its wave;
    // k_left: k pieces (K_INNER) or k rows (K_OUTER) of the stage that exist
    static __device__ __forceinline__ unsigned source(const TileOperand& op, int org, int q, int wave, int lane, int k_left) {
        const int at = (wave * kLoads + q) * 1024 + lane * 16;
        if constexpr (!kOuter) {
            const int row = at / RB;
            const int c = min((lane % kPieces) ^ inner_swap(row), k_left - 1);
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
        if constexpr (!kOuter) return min(kPieces, (K - k0 + TileElem<T>::piece - 1) / TileElem<T>::piece);
        return op.rows - k0;
    }

    __device__ __forceinline__ void init(const TileOperand& op, int org, int stage0, int wave, int lane) {
        // a tile may lie wholly behind the last row (an epilogue's cover): it then reads the last row
        const uint64_t origin = kOuter ? (uint64_t)org * TileElem<T>::bytes : (uint64_t)min(org, op.rows - 1) * (uint64_t)op.pitch;
        base = uniform64((uint64_t)op.p + origin + (uint64_t)stage0 * (uint64_t)op.step);
        const int whole = kOuter ? 1 << 30 : kPieces;
#pragma unroll
        for (int q = 0; q < kLoads; ++q) off[q] = source(op, org, q, wave, lane, whole);
        if constexpr (!kOuter) {
            const int l32 = lane & 31, lh = lane >> 5;
#pragma unroll
            for (int j = 0; j < kSteps; ++j) rd[j] = l32 * RB + (((kSteps * lh + j) ^ inner_swap(l32)) << 4);
        }
    }
    __device__ __forceinline__ void load(const TileOperand& op, unsigned dst, int wave) {
#pragma unroll
        for (int q = 0; q < kLoads; ++q) dma_piece(base, off[q], dst + (wave * kLoads + q) * 1024);
        base += (uint64_t)op.step;
    }
    template <int P, int OF> __device__ __forceinline__ void load_part(const TileOperand& op, unsigned dst, int wave) {
#pragma unroll
        for (int q = kLoads * P / OF; q < kLoads * (P + 1) / OF; ++q) dma_piece(base, off[q], dst + (wave * kLoads + q) * 1024);
        if (P == OF - 1) base += (uint64_t)op.step;
    }
    // a stage that does not exist in full
    __device__ __forceinline__ void load_tail(const TileOperand& op, int org, int k_left, unsigned dst, int wave, int lane) {
#pragma unroll
        for (int q = 0; q < kLoads; ++q)
            dma_piece(base, source(op, org, q, wave, lane, k_left), dst + (wave * kLoads + q) * 1024);
        base += (uint64_t)op.step;
    }
    // piece j of block `blk` (32 rows or columns) for this lane
    __device__ __forceinline__ uintx4 fragment(const char* st, int blk, int j, int lane) const {
        if constexpr (!kOuter) {
            return *reinterpret_cast<const uintx4*>(st + rd[j] + blk * 32 * RB);
        } else if constexpr (TileElem<T>::bytes == 2) {
            const int row = 8 * (kSteps * (lane >> 5) + j) + ((lane >> 2) & 3);            // row & 3 == (lane >> 2) & 3
            const int piece = outer_swap(row, blk * 4 + ((lane >> 4) & 1) * 2) * 16 + (lane & 3) * 8;
            typedef __attribute__((address_space(3))) shortx4* ldsp;
            const char* at = st + row * kRow + piece;
            const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ldsp)(at));
            const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ldsp)(at + 4 * kRow));
            typedef unsigned uintx2 __attribute__((ext_vector_type(2)));
            const uintx2 l = __builtin_bit_cast(uintx2, lo), h = __builtin_bit_cast(uintx2, hi);
            return uintx4{l[0], l[1], h[0], h[1]};
        } else {
            const int row = 4 * (kSteps * (lane >> 5) + j);
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
//
// What bounds it (256 x 256, bf16 of random values, 8192 x 4096 outputs): K = 8192 takes 419 us, 1.31 PFLOP/s, K = 2048 in
// two rounds 126 us: 14 us of a round are its first loads and its stores.  Without the loads the first takes about a
// seventh less, without the LDS reads as well, without the multiplies (loads and LDS reads alone) 165 of 265 us at
// K = 4096: the CU's request path (64 KB of operands per 2048 clocks of multiplies), LDS and the matrix pipe are each
// busy for more than half of the time, and on zeros instead of random values the same launch runs a quarter faster (the
// clock follows the data).  4-bit 4096 x 8192 x 8192: 155 us, 3.5 PFLOP/s, the same bytes per clock.  Tried without gain: stages
// of 64 bytes in a deeper ring, four waves of 128 x 128, two workgroups of 256 x 128 per CU, wave priorities, a workgroup
// per CU that walks the tiles and requests the next one's first stages before it stores.
template <typename T, int BM, int BN, int RB> constexpr int kTileSlot =       // LDS of a stage; 4-bit scales 1 KB at a time
    (BM + BN) * RB + (std::is_same<T, mx4_t>::value ? ((BM * RB / 16 + 1023) / 1024 + (BN * RB / 16 + 1023) / 1024) * 1024 : 0);

// one tile (or part `part` of its reduction): `id` counts the tiles, lds holds RING stages
template <typename T, int AO, int BO, int BM, int BN, int WM, int WN, int RB, int RING, class Epi>
__device__ __forceinline__ void tile_gemm(const TileArgs& g, const Epi& epi, int id, int part, char* lds) {
    constexpr int WAVES = WM * WN, MI = BM / WM / 32, NI = BN / WN / 32;
    constexpr bool MX4 = std::is_same<T, mx4_t>::value;
    constexpr int STAGE = RB / 16 * TileElem<T>::piece, STEPS = RB / 32;   // elements of k, multiplies of a lane half
    typedef TileSide<T, AO, BM, WAVES, RB> SA;
    typedef TileSide<T, BO, BN, WAVES, RB> SB;
    constexpr int SROW = RB / 16, SCA = (BM * SROW + 1023) / 1024, SCB = (BN * SROW + 1023) / 1024;      // scale bytes, loads
    constexpr int SLOT = kTileSlot<T, BM, BN, RB>;
    constexpr bool TWO = AO == K_OUTER && sizeof(T) == 2;              // the products that run in two passes

    int tm, tn;
    if (!tile_of(id, g.mt, g.nt, tm, tn)) return;
    const int m0 = tm * BM, n0 = tn * BN;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int l32 = lane & 31, lh = lane >> 5;
    const int first = part * g.split, last = min(first + g.split, g.stages);

    SA sa;
    SB sb;
    sa.init(g.a, m0, first, wave, lane);
    sb.init(g.b, n0, first, wave, lane);
    if (TWO && first >= g.pass) {
        sa.base += (uint64_t)g.a_turn;
        sb.base += (uint64_t)g.b_turn;
    }
    const unsigned lds0 = lds_addr(lds);
    // mx4: scale bytes as 16-byte pieces (16 / SROW rows), one load each by the first waves
    uint64_t sc_base = 0;
    unsigned sc_off = 0, sc_dst = 0;
    long sc_step = 0;
    static_assert(!MX4 || SCA + SCB <= WAVES, "a scale load per wave at most");
    if constexpr (MX4) {
        if (wave < SCA + SCB) {
            const bool isa = wave < SCA;
            const TileOperand& op = isa ? g.a : g.b;
            const int part = isa ? wave : wave - SCA, org = isa ? m0 : n0;
            constexpr int R = 16 / SROW;
            const int rows16 = (op.rows + R - 1) / R;                               // 16-byte pieces per stage
            sc_step = (long)rows16 * 16;
            sc_base = uniform64((uint64_t)op.scale + (uint64_t)first * (uint64_t)sc_step);
            sc_off = (unsigned)min(org / R + part * 64 + lane, rows16 - 1) * 16u;
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
        const int local = TWO && s >= g.pass ? s - g.pass : s;
        if (local == g.tail_at) {
            sa.load_tail(g.a, m0, SA::left(g.a, g.K, local * STAGE), dst, wave, lane);
            sb.load_tail(g.b, n0, SB::left(g.b, g.K, local * STAGE), dst + SA::kBytes, wave, lane);
        } else {
            sa.load(g.a, dst, wave);
            sb.load(g.b, dst + SA::kBytes, wave);
        }
        if (TWO && local == g.pass - 1) {
            sa.base += (uint64_t)g.a_turn;
            sb.base += (uint64_t)g.b_turn;
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
            typedef unsigned short SW;                                 // a lane's scale bytes of a stage
            static_assert(STEPS == (int)sizeof(SW), "a scale byte per step");
            const char* sca = lds + slot * SLOT + SA::kBytes + SB::kBytes;
#pragma unroll
            for (int i = 0; i < MI; ++i) qa[set][i] = *reinterpret_cast<const SW*>(sca + ((wm * MI + i) * 32 + l32) * SROW + lh * STEPS);
#pragma unroll
            for (int n = 0; n < NI; ++n) qb[set][n] = *reinterpret_cast<const SW*>(sca + SCA * 1024 + ((wn * NI + n) * 32 + l32) * SROW + lh * STEPS);
        }
    };
    auto multiply = [&](int s, auto jc, auto tail) {
        constexpr int J = decltype(jc)::value;
        if constexpr (decltype(tail)::value && !MX4) {
            // pieces past the end of the reduction (two passes: whole stages): zero wherever k is inner (they were read
            // from elsewhere in the row).  A k-outer operand needs no mask beside a k-inner one; where both are k-outer, the rows past
            // the end exist and one of the two holds zeros in them.
            const bool in = (TWO && g.passes > 1) || STEPS * lh + J < (g.K - s * STAGE + TileElem<T>::piece - 1) / TileElem<T>::piece;
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
    const std::integral_constant<int, STEPS - 1> j_last;
    // A full stage's requests, one share per step so that no step waits long for the CU's request path: with four steps A's
    // in the first two and B's in the last two (16-bit 8192 x 4096 x 16384: 943 -> 902 us), with two all of them at once
    // (4-bit: a split there gains nothing).
    constexpr bool SPREAD = STEPS == 4;
    auto plain_stage = [&](int s) {                                    // (the others go in one piece)
        const int local = TWO && s >= g.pass ? s - g.pass : s;
        return local != g.tail_at && (!TWO || local != g.pass - 1);
    };
    bool pending = false;
    int refill = 0;
    auto share = [&](auto pc) {
        constexpr int P = decltype(pc)::value;
        const unsigned dst = lds0 + refill * SLOT;
        if constexpr (P < 2) sa.template load_part<P, 2>(g.a, dst, wave);
        else sb.template load_part<P - 2, 2>(g.b, dst + SA::kBytes, wave);
    };
    // steps 0 .. STEPS - 2 of stage s, each behind the request for the fragments of the next
    auto all_but_last = [&](int s, int slot, auto tail) {
        for_each_step(std::make_integer_sequence<int, STEPS - 1>{}, [&](auto jc) {
            read(slot, std::integral_constant<int, decltype(jc)::value + 1>{});
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (SPREAD) {
                if (pending) share(std::integral_constant<int, decltype(jc)::value + 1>{});
                __builtin_amdgcn_sched_barrier(0);
            }
            multiply(s, jc, tail);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
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
        all_but_last(s, slot, std::false_type{});
        // stage s + 1 has landed (the RING - 2 behind it may still be in flight, fewer near the end) and this wave has read
        // all of stage s; behind the barrier that holds for every wave
        asm volatile("" ::: "memory");
        if (RING > 2 && s + RING <= last) wait_loads<(RING - 2) * LPW>();
        else wait_loads<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        refill = slot;
        slot = slot + 1 == RING ? 0 : slot + 1;
        read(slot, j0);
        read_scales(slot, 1);
        __builtin_amdgcn_sched_barrier(0);
        pending = SPREAD && !MX4 && s + RING < last && plain_stage(s + RING);
        if (pending) share(j0);
        else if (s + RING < last) issue(s + RING, refill);
        __builtin_amdgcn_sched_barrier(0);
        multiply(s, j_last, std::false_type{});
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (MX4) {
#pragma unroll
            for (int i = 0; i < MI; ++i) qa[0][i] = qa[1][i];
#pragma unroll
            for (int n = 0; n < NI; ++n) qb[0][n] = qb[1][n];
        }
    }
    all_but_last(last - 1, slot, std::true_type{});
    multiply(last - 1, j_last, std::true_type{});
    asm volatile("" ::: "memory");                                    // (the last reads stay above the epilogue's barrier)
    wait_loads<0>();
    epi.template run<BM, BN, WM, WN, MI, NI>(acc, g, m0, n0, wm, wn, l32, lh, lds);
}

template <typename T, int AO, int BO, int BM, int BN, int WM, int WN, int RB, int RING, class Epi>
__global__ __launch_bounds__(64 * WM * WN, WM * WN > 4 ? 1 : 2) void tile_gemm_kernel(TileArgs g, Epi epi) {
    __shared__ __align__(1024) char lds[RING * kTileSlot<T, BM, BN, RB>];
    tile_gemm<T, AO, BO, BM, BN, WM, WN, RB, RING>(g, epi, blockIdx.x, blockIdx.y, lds);
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

// What a wave's accumulators become, written to out[n][m]: value(i, q, n, v) gives the four results at block i, quad q of
// column block n.  A lane holds four of them per row, 8 or 16 bytes, which would touch 32 rows per store; so a wave turns
// one 32-row block at a time in LDS of its own and stores rows in runs of MI * 32 elements, 16 bytes per lane (pieces
// exchanged by row for the banks), or an element per lane where the output's rows are not 16-byte aligned.
// rows past row_end and columns past col_end are not written; add: += (fp32).
template <typename T, int WM, int WN, int MI, int NI, class F>
__device__ __forceinline__ void tile_store(T* out, long pitch, int m0, int n0, int row_end, int col_end, int wm, int wn, int l32, int lh,
                                           char* lds, bool add, F&& value) {
    constexpr int CH = MI * 32 * (int)sizeof(T) / 16;                  // 16-byte pieces of a row of the block
    const bool wide = (pitch * (long)sizeof(T)) % 16 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    const int mb = m0 + wm * MI * 32;
    __builtin_amdgcn_s_barrier();                                      // every wave is done with the last stage
    asm volatile("" ::: "memory");
    char* own = lds + (wm * WN + wn) * (32 * CH * 16);
    auto swap = [](int row) { return CH >= 16 ? row & (CH - 1) : row / (16 / CH) & (CH - 1); };
#pragma unroll
    for (int n = 0; n < NI; ++n) {
        const int nb = n0 + (wn * NI + n) * 32;
        if (nb >= row_end) continue;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float v[4];
                value(i, q, n, v);
                const int at = (i * 32 + 8 * q + 4 * lh) * (int)sizeof(T);
                store4<T>(reinterpret_cast<T*>(own + l32 * CH * 16 + (((at >> 4) ^ swap(l32)) << 4) + (at & 15)), v, 4, true);
            }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        if (wide) {
#pragma unroll
            for (int k = 0; k < CH / 2; ++k) {
                const int idx = k * 64 + lh * 32 + l32, row = idx / CH, c = idx % CH;
                const uintx4 v = *reinterpret_cast<const uintx4*>(own + row * CH * 16 + ((c ^ swap(row)) << 4));
                constexpr int E = 16 / (int)sizeof(T);
                const int m = mb + c * E;
                if (nb + row >= row_end || m >= col_end) continue;
                T* to = out + (long)(nb + row) * pitch + m;
                if (m + E <= col_end) {
                    if constexpr (sizeof(T) == 4) {
                        floatx4 f = __builtin_bit_cast(floatx4, v);
                        if (add) f += *reinterpret_cast<const floatx4*>(to);
                        *reinterpret_cast<floatx4*>(to) = f;
                    } else {
                        *reinterpret_cast<uintx4*>(to) = v;
                    }
                } else {
                    const Pack16<T> pk = __builtin_bit_cast(Pack16<T>, v);
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (m + e < col_end) to[e] = pk.e[e];
                }
            }
        } else {
            const int lane = lh * 32 + l32;
            for (int k = 0; k < MI * 16; ++k) {
                const int idx = k * 64 + lane, row = idx / (MI * 32), c = idx % (MI * 32), at = c * (int)sizeof(T);
                const T v = *reinterpret_cast<const T*>(own + row * CH * 16 + (((at >> 4) ^ swap(row)) << 4) + (at & 15));
                if (nb + row < row_end && mb + c < col_end) out[(long)(nb + row) * pitch + mb + c] = v;
            }
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
    }
}

// out[n][m] = relu?( scale * acc + bias[m] ), rounded to T once
template <typename T> struct TileStore {
    T* out;
    long pitch;             // elements
    const T* bias;          // or null
    const float* scale;     // one factor in device memory, or null
    int relu;
    template <int BM, int BN, int WM, int WN, int MI, int NI>
    __device__ __forceinline__ void run(floatx16 (&acc)[MI][NI], const TileArgs& g, int m0, int n0, int wm, int wn, int l32, int lh, char* lds) const {
        const float f = scale ? *scale : 1.f;
        tile_store<T, WM, WN, MI, NI>(out, pitch, m0, n0, g.N, g.M, wm, wn, l32, lh, lds, false, [&](int i, int q, int n, float (&v)[4]) {
            const int m = m0 + (wm * MI + i) * 32 + 8 * q + 4 * lh;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float b = bias && m + e < g.M ? to_f32(bias[m + e]) : 0.f;
                v[e] = acc[i][n][4 * q + e] * f + b;
                if (relu) v[e] = v[e] > 0.f || v[e] != v[e] ? v[e] : 0.f;              // a NaN stays one
            }
        });
    }
};

// part[z][n][m] (fp32) = acc, or += where `add` is set (a tile is owned by one workgroup: the order is fixed)
struct TilePart {
    float* part;
    long pitch;             // elements, a multiple of 4; part is 16-byte aligned
    int add;
    template <int BM, int BN, int WM, int WN, int MI, int NI>
    __device__ __forceinline__ void run(floatx16 (&acc)[MI][NI], const TileArgs& g, int m0, int n0, int wm, int wn, int l32, int lh, char* lds) const {
        tile_store<float, WM, WN, MI, NI>(part + (long)blockIdx.y * g.N * pitch, pitch, m0, n0, g.N, (int)pitch, wm, wn, l32, lh, lds, add != 0,
                                          [&](int i, int q, int n, float (&v)[4]) {
#pragma unroll
                                              for (int e = 0; e < 4; ++e) v[e] = acc[i][n][4 * q + e];
                                          });
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

constexpr int kTile = 128;               // edge of the usual tile

inline int ceil_div(long a, long b) { return (int)((a + b - 1) / b); }

// the parts that are not empty when `stages` are cut into `parts`
inline int parts_of(int stages, int parts) { return ceil_div(stages, ceil_div(stages, parts)); }

template <typename T> constexpr int kStageBytes = std::is_same<T, mx4_t>::value ? 64 : 128;   // of an operand row
template <typename T> constexpr int kStageOf = kStageBytes<T> / 16 * TileElem<T>::piece;      // elements of k

// the fields of g that follow from the tile and the parts; returns the parts that are not empty
template <typename T, int AO, int BO, int BM, int BN, int RB> inline int tile_prepare(TileArgs& g, int parts, int cover) {
    g.mt = ceil_div(g.M, BM);
    g.nt = ceil_div(cover, BN);
    constexpr int stage = RB / 16 * TileElem<T>::piece;
    const bool mx4 = std::is_same<T, mx4_t>::value;
    g.a.step = mx4 ? g.a.rows * (long)RB : AO == K_INNER ? RB : g.a.pitch * stage;
    g.b.step = mx4 ? g.b.rows * (long)RB : BO == K_INNER ? RB : g.b.pitch * stage;
    g.passes = std::max(g.passes, 1);
    g.pass = ceil_div(g.K, stage);
    // with two passes K is a whole number of stages, of which a k-outer A may hold a little less
    g.tail_at = g.passes > 1 ? (AO == K_OUTER && g.a.rows < g.K ? g.pass - 1 : -1) : g.K % stage ? g.pass - 1 : -1;
    g.stages = g.passes * g.pass;
    g.split = ceil_div(g.stages, parts);
    return parts_of(g.stages, parts);
}

template <typename T, int AO, int BO, int BM, int BN, int WM, int WN, int RB, int RING, class Epi>
inline int tile_launch_as(TileArgs g, const Epi& epi, int parts, int cover, hipStream_t s) {
    parts = tile_prepare<T, AO, BO, BM, BN, RB>(g, parts, cover);
    hipLaunchKernelGGL((tile_gemm_kernel<T, AO, BO, BM, BN, WM, WN, RB, RING, Epi>), dim3(tile_grid(g.mt, g.nt), parts), dim3(64 * WM * WN), 0, s, g, epi);
    return parts;
}

// stages in LDS of a 64 x 64 tile: fp32 is bound by its multiplies and takes more workgroups to a CU instead
template <typename T> constexpr int kSmallRing = std::is_same<T, mx4_t>::value ? 5 : sizeof(T) == 4 ? 2 : 3;

struct TilePick {
    int rows, cols, parts;      // m and n extent of a tile, parts of the reduction
};

// The cut with the smallest estimated time.  A CU works through its share of the (tile, part) items; an item takes the
// longer of its multiplies and its operands' way into LDS; parts are written and read back once in fp32 by one more
// launch.  `most` bounds the parts (1: the epilogue needs whole sums).  Rates in products / bytes per microsecond and CU,
// fitted to 24 products in all three kinds of type, each timed with every tile and 1 to 64 parts: the cut it takes is at
// most 1.2 times the fastest (once 1.33), 1.0 in the middle.  Some of those, us, 256 x 256 / 128 x 128 / 128 x 64 / 64 x 64,
// whole sums, M x N x K: 16-bit 4096 x 250 x 1000 28 / 15 / 11 / 9, 2048 x 2048 x 2048 52 / 31 / 24 / 29, 2048 x 700 x
// 32000 in 10 parts 98 (128 x 128: 116 in 4); fp32 10007 x 777 x 1004 250 / 196 / 175 / 138; 4-bit 4096 x 4096 x 4096
// 43 / 47 / 64 / 72, 500 x 200 x 512 13 / 8 / 6 / 5.
template <typename T> inline TilePick tile_pick(int M, int N, int K, int most, int cus) {
    constexpr bool F32 = std::is_same<T, float>::value, MX4 = std::is_same<T, mx4_t>::value;
    const double rate = F32 ? 0.28e6 : MX4 ? 6.5e6 : 2.1e6, bytes = 45e3;
    // relative to 128 x 128: the large tile draws half the bytes per product, the small ones more
    const struct { int rows, cols; double factor; } kinds[] = {
        {256, 256, F32 ? 1.0 : MX4 ? 1.23 : 1.33}, {kTile, kTile, 1.0}, {kTile, 64, F32 ? 0.9 : 0.8}, {kTile, 32, F32 ? 1.05 : 0.5}, {64, 64, F32 ? 1.0 : MX4 ? 0.8 : 0.6}};
    // the rates were fitted with cuts of 128 bytes of a row, two stages of 4-bit operands
    constexpr int kUnit = 8 * TileElem<T>::piece;
    const int stages = ceil_div(K, kUnit), launched = ceil_div(K, kStageOf<T>);
    TilePick best = {kTile, kTile, 1};
    double least = 1e30;
    for (const auto& kind : kinds) {
        const int rows = kind.rows, cols = kind.cols;
        if ((rows == 256 && (M <= kTile || N <= kTile)) || (cols == 32 && (MX4 || N > 64))) continue;
        const long tiles = (long)ceil_div(M, rows) * ceil_div(N, cols);
        for (int parts = 1; parts <= most && parts <= std::max(1, stages / 2); parts += parts < 8 ? 1 : parts / 4) {
            const int split = ceil_div(stages, parts);
            if (parts_of(stages, parts) != parts || parts_of(launched, parts) != parts) continue;
            const long items = tiles * parts;
            if (parts > 1 && (items > (rows == 64 ? 8L : 4L) * cus || (size_t)parts * M * N * 4 > (64u << 20))) break;
            const double k = (double)split * kUnit;
            const double mul = (double)rows * cols * k / (rate * kind.factor);
            const double move = (double)(rows + cols) * split * 128 / bytes;
            // one small tile alone on its CU waits for its own loads
            const double item = std::max(mul, move) * (rows < 256 && items <= cus ? (rows == kTile ? 1.4 : 1.25) : 1.0);
            const double t = ceil_div(items, cus) * item + (parts > 1 ? 4.0 + (double)parts * M * N * 8 / 4e6 : 0.0);
            if (t < least) {
                least = t;
                best = {rows, cols, parts};
            }
        }
    }
    return best;
}

// `cover`: rows of n that the epilogue has to reach (N or a little more).  Returns the parts that were launched: those of
// the cut if it was picked for this reduction.
template <typename T, int AO, int BO, class Epi>
inline int tile_launch(const TileArgs& g, const Epi& epi, const TilePick& pick, int cover, hipStream_t s) {
    constexpr int RB = kStageBytes<T>;
    if (pick.rows == 256) return tile_launch_as<T, AO, BO, 256, 256, 2, 4, RB, RB == 64 ? 4 : 2>(g, epi, pick.parts, cover, s);
    if (pick.rows == 64) return tile_launch_as<T, AO, BO, 64, 64, 2, 2, RB, kSmallRing<T>>(g, epi, pick.parts, cover, s);
    if constexpr (RB == 128)            // (a 4-bit stage of 32 rows is less than a load per wave)
        if (pick.cols == 32) return tile_launch_as<T, AO, BO, kTile, 32, 4, 1, RB, 4>(g, epi, pick.parts, cover, s);
    if (pick.cols == 64) return tile_launch_as<T, AO, BO, kTile, 64, 4, 1, RB, RB == 64 ? 5 : 3>(g, epi, pick.parts, cover, s);
    return tile_launch_as<T, AO, BO, kTile, kTile, 2, 2, RB, RB == 64 ? 4 : 2>(g, epi, pick.parts, cover, s);
}

inline size_t part_bytes(int M, int N, int parts) { return (size_t)parts * N * round_up(M, 4) * sizeof(float); }

}  // namespace wino
