// One BN x BM tile of a microscaled 4-bit product on the matrix cores: BN weight rows times BM activation rows over all of K.
//
// K goes by in stages of eight blocks (128 bytes and 8 scale bytes a row), NST of them in LDS at once.  Both arrive there by LDS
// DMA, no register between: 16 bytes a lane of the values (a wave's instruction brings eight rows), 4 of the scales (32 rows).
// A row's eight blocks lie permuted (block c of row r in slot c ^ (r & 7)), so that lanes that read one block of eight rows
// meet no bank twice.  Waves hold WN x WM of the tile as 32 x 32 sums.  A matrix instruction takes two blocks of each row, one
// from either half of the stage (4 h + s for the lanes' half h at step s): a lane then has its four steps' scales in one word,
// which the instruction picks its byte from.  Each step's fragments are read during the step before.  At the last step of a
// stage every wave has its fragments in registers: one barrier there hands the stage's LDS to the rows NST stages on
// and opens the next stage.
#pragma once

#include "i8tile.hpp"
#include "mx4.hpp"

namespace trk {

// C += A B, 32 x 32 x two blocks: lane l holds a block of A's row l % 32 and of B's column l % 32, the two halves a block each,
// its scale in byte S of sa, sb; element e of C's column l % 32: row 8 (e / 4) + 4 (l / 32) + e % 4.
template <int S>
__device__ __forceinline__ f32x16 mfma_mx4_32(i32x4 a, uint32_t sa, i32x4 b, uint32_t sb, f32x16 c) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(a), mx_operand(b), c, MX_FP4, MX_FP4, S, (int)sa, S, (int)sb);
}

// 4 bytes a lane to the 256 bytes of LDS at `lds`, as lds_dma's 16
__device__ __forceinline__ void lds_dma4(i32x4 rsrc, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(rsrc)
                 : "memory", "m0");
}

template <int BN_, int BM_, int WN_, int WM_, int NST_>
struct Mx4Tile {
    static constexpr int BN = BN_, BM = BM_, WN = WN_, WM = WM_, NST = NST_, BK = 128, BS = 8;  // a stage's bytes of a row
    static constexpr int NW = BN / WN * (BM / WM), T = NW * WAVE;
    static constexpr int FN = WN / 32, FM = WM / 32;
    static constexpr int NA = BN / 8 / NW, NB = BM / 8 / NW, NSC = (BN + BM) / 32, NS = (NSC + NW - 1) / NW;  // a wave's loads of a stage
    static constexpr int NL = NA + NB + NS;
    static constexpr int SCALES = (BN + BM) * BK, STAGE = SCALES + (BN + BM) * BS, LDS = STAGE * NST;
    static_assert(BN % (8 * NW) == 0 && BM % (8 * NW) == 0 && BN % 32 == 0 && BM % 32 == 0 && LDS <= 160 * 1024, "tile");

    f32x16 acc[FN][FM];
    uint32_t lane, wv, wn, wm;  // this wave's first weight and activation row in the tile

    __device__ __forceinline__ Mx4Tile() {
        wv = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
        wn = wv % (BN / WN) * WN, wm = wv / (BN / WN) * WM;
#pragma unroll
        for (int i = 0; i < FN; i++)
#pragma unroll
            for (int j = 0; j < FM; j++)
#pragma unroll
                for (int e = 0; e < 16; e++) acc[i][j][e] = 0.0f;
    }
    // the tile row that this lane loads of its wave's i-th piece of weights (activations: the same with NB)
    __device__ __forceinline__ uint32_t load_row(int i) const { return (i * NW + wv) * 8 + lane / 8; }
    // its wave's i-th piece of scales, 32 rows, the weights' before the activations' (the last may be taken by several waves)
    __device__ __forceinline__ uint32_t scale_piece(int i) const {
        const uint32_t n = i * NW + wv;
        return n < NSC ? n : NSC - 1;
    }

    // rw[i], wo[i]: buffer and this lane's row offset for its i-th eight weight rows; rx, xo: the activations'.  rs[i], so[i]: its
    // i-th scales', lanes 2 n and 2 n + 1 a row's.
    // a0: the LDS row of this lane's weight row of the wave's first 32 (a place in eight as lane % 8 has); the i-th's: a0 + i * astep.
    // live: this wave's 32-row groups of activations that hold any (PART: the others' products are left out).
    // ONCE: the weight rows are this workgroup's alone.
    template <bool PART, bool ONCE>
    __device__ __forceinline__ void run(uint8_t* lds, const i32x4 (&rw)[NA], const uint32_t (&wo)[NA], i32x4 rx,
                                        const uint32_t (&xo)[NB], const i32x4 (&rs)[NS], const uint32_t (&so)[NS], uint32_t nb,
                                        uint32_t live, uint32_t a0, uint32_t astep) {
        const uint32_t l0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
        const uint32_t S = (nb + 7) / 8, bytes = 16 * nb, words = (nb + 3) / 4 * 4;
        const uint32_t piece = 16 * (lane % 8 ^ lane / 8);  // where in a row this lane loads
        uint32_t sat[NS];
#pragma unroll
        for (int i = 0; i < NS; i++) sat[i] = SCALES + scale_piece(i) * 256;
        // the n-th of a wave's loads of stage s; past the row's end anything, it multiplies zeros by 1
        auto load1 = [&](uint32_t s, uint32_t at, int n) {
            const uint32_t o = s * BK + piece, oc = o < bytes ? o : 0, q = s * BS + 4 * (lane % 2), qc = q < words ? q : 0;
            if (n < NA)
                lds_dma<ONCE>(rw[n < NA ? n : 0], wo[n < NA ? n : 0] + oc, at + (n * NW + wv) * 1024);
            else if (n < NA + NB)
                lds_dma<false>(rx, xo[n < NA + NB ? n - NA : 0] + oc, at + (n * NW + wv) * 1024);  // the activations' rows follow the weights'
            else
                lds_dma4(rs[n - NA - NB], so[n - NA - NB] + qc, at + sat[n - NA - NB]);
        };
        auto load_at = [&](uint32_t s) { return l0 + s % NST * STAGE; };
        i32x4 a[2][FN], b[2][FM];
        uint32_t sa[2][FN], sb[2][FM];
        const uint32_t row = lane % 32, half = lane / 32, slot = 16 * (4 * half ^ row % 8), b0 = BN + wm + row;
        auto read = [&](uint32_t at, int s, int to) {
#pragma unroll
            for (int i = 0; i < FN; i++) a[to][i] = *reinterpret_cast<const i32x4*>(lds + at + (a0 + i * astep) * BK + (slot ^ (16 * s)));
#pragma unroll
            for (int j = 0; j < FM; j++)
                if (!PART || j < (int)live)
                    b[to][j] = *reinterpret_cast<const i32x4*>(lds + at + (b0 + j * 32) * BK + (slot ^ (16 * s)));
        };
        auto read_scales = [&](uint32_t at, int to) {
#pragma unroll
            for (int i = 0; i < FN; i++)
                sa[to][i] = *reinterpret_cast<const uint32_t*>(lds + at + SCALES + (a0 + i * astep) * BS + 4 * half);
#pragma unroll
            for (int j = 0; j < FM; j++)
                if (!PART || j < (int)live)
                    sb[to][j] = *reinterpret_cast<const uint32_t*>(lds + at + SCALES + (b0 + j * 32) * BS + 4 * half);
        };
        // a step's products, with the loads of a stage between them
        auto mul = [&](auto step, int from, int sc, bool loads, uint32_t s, uint32_t at) {
            constexpr int ST = decltype(step)::value;
#pragma unroll
            for (int j = 0; j < FM; j++) {
                if (!PART || j < (int)live) {
#pragma unroll
                    for (int i = 0; i < FN; i++)
                        acc[i][j] = mfma_mx4_32<ST>(a[from][i], sa[sc][i], b[from][j], sb[sc][j], acc[i][j]);
                    // the products stay where they are: on their side of the barrier, and before any branch that lanes part at
                    // (their operands would be made in the lanes that take it alone)
#pragma unroll
                    for (int i = 0; i < FN; i++) asm volatile("" : "+v"(acc[i][j]));
                }
                if (loads)
#pragma unroll
                    for (int n = j * NL / FM; n < (j + 1) * NL / FM; n++) load1(s, at, n);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (uint32_t s = 0; s < NST; s++)
            if (s < S)
#pragma unroll
                for (int n = 0; n < NL; n++) load1(s, load_at(s), n);
        if (S >= NST)
            wait_dma<(NST - 1) * NL>();
        else
            wait_dma<0>();
        wg_barrier();
        read(0, 0, 0);
        read_scales(0, 0);
        uint32_t cur = 0;
        for (uint32_t s = 0; s + 1 < S; s++) {
            const uint32_t nxt = cur + STAGE == LDS ? 0 : cur + STAGE;
            read(cur, 1, 1);
            mul(std::integral_constant<int, 0>{}, 0, 0, false, 0, 0);
            read(cur, 2, 0);
            mul(std::integral_constant<int, 1>{}, 1, 0, false, 0, 0);
            read(cur, 3, 1);
            mul(std::integral_constant<int, 2>{}, 0, 0, false, 0, 0);
            if (s + NST <= S)
                wait_dma<(NST - 2) * NL>();
            else
                wait_dma<0>();
            wg_barrier();
            read(nxt, 0, 0);
            read_scales(nxt, 1);
            mul(std::integral_constant<int, 3>{}, 1, 0, s + NST < S, s + NST, load_at(s + NST));
#pragma unroll
            for (int i = 0; i < FN; i++) sa[0][i] = sa[1][i];
#pragma unroll
            for (int j = 0; j < FM; j++) sb[0][j] = sb[1][j];
            cur = nxt;
        }
        // the last stage: past the row's end zeros, by 1
        const uint32_t first = 8 * (S - 1) + 4 * half, in = first < nb ? (nb - first < 4 ? nb - first : 4u) : 0u;
        const uint32_t keep = in >= 4 ? 0xffffffffu : (1u << (8 * in)) - 1u, one = MX_ONE * 0x01010101u & ~keep;
#pragma unroll
        for (int i = 0; i < FN; i++) sa[0][i] = (sa[0][i] & keep) | one;
#pragma unroll
        for (int j = 0; j < FM; j++) sb[0][j] = (sb[0][j] & keep) | one;
        auto cut = [&](uint32_t s, int to) {
            if (s >= in)
#pragma unroll
                for (int j = 0; j < FM; j++) b[to][j] = i32x4{0, 0, 0, 0};
        };
        read(cur, 1, 1);
        cut(0, 0);
        mul(std::integral_constant<int, 0>{}, 0, 0, false, 0, 0);
        read(cur, 2, 0);
        cut(1, 1);
        mul(std::integral_constant<int, 1>{}, 1, 0, false, 0, 0);
        read(cur, 3, 1);
        cut(2, 0);
        mul(std::integral_constant<int, 2>{}, 0, 0, false, 0, 0);
        cut(3, 1);
        mul(std::integral_constant<int, 3>{}, 1, 0, false, 0, 0);
    }
};

}  // namespace trk
