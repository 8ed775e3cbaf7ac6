// One BN x BM tile of a microscaled 4-bit product on the matrix cores: BN weight rows times BM activation rows over all of K.
//
// K goes by in stages of eight blocks (128 bytes a row), NST of them in LDS at once, and their scales by GS stages (8 GS bytes a
// row), for a row's eight bytes of one stage are a cache line's trip by themselves.  Both arrive by LDS DMA, no register between: 16
// bytes a lane of the values (a wave's instruction brings eight rows), 4 of the scales (32 / GS rows).  A row's blocks lie permuted
// (block c of row r in slot c ^ (r & 7) ^ (r >> 3 & 1)), and its words of scales, so that neither read meets a bank twice.  Waves hold WN x
// WM of the tile as 32 x 32 sums.  A matrix instruction takes two blocks of each row, one from either half of the stage (4 h + s for
// the lanes' half h at step s): a lane then has its four steps' scales in one word, which the instruction picks its byte from.
// Each step's fragments are read during the step before.  At the last step of a stage every wave has its fragments in
// registers: one barrier there hands the stage's LDS to the rows NST stages on and opens the next stage.  The scales' LDS is
// handed on one stage before their last (that stage's are read before the barrier), which leaves the next ones a stage to arrive.
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

// Four neighbouring values of a row of type DT at any address, `left` of them there
template <uint32_t DT>
__device__ __forceinline__ void store4_any(typename Elem<DT>::T* y, f32x4 v, uint32_t left) {
    if (left >= 4) {
        if constexpr (DT == TRK_DT_F32) {
            typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
            *reinterpret_cast<f32x4_any*>(y) = v;
        } else {
            typedef float f32x2 __attribute__((ext_vector_type(2)));
            typedef uint32_t u32x2_h __attribute__((ext_vector_type(2), aligned(2)));
            typedef typename std::conditional<DT == TRK_DT_BF16, __bf16, _Float16>::type E;
            typedef E e16x2 __attribute__((ext_vector_type(2)));
            *reinterpret_cast<u32x2_h*>(y) =
                u32x2_h{__builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[0], v[1]}), e16x2)),
                        __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[2], v[3]}), e16x2))};
        }
        return;
    }
#pragma unroll
    for (uint32_t c = 0; c < 4; c++)
        if (c < left) y[c] = Elem<DT>::put(v[c]);
}

template <int BN_, int BM_, int WN_, int WM_, int NST_, int GS_ = 4>
struct Mx4Tile {
    static constexpr int BN = BN_, BM = BM_, WN = WN_, WM = WM_, NST = NST_, GS = GS_, BK = 128;  // BK: a stage's bytes of a row
    static constexpr int NW = BN / WN * (BM / WM), T = NW * WAVE;
    static constexpr int FN = WN / 32, FM = WM / 32;
    static constexpr int NA = BN / 8 / NW, NB = BM / 8 / NW, NL = NA + NB;  // a wave's loads of a stage
    static constexpr int SW = 2 * GS, SR = WAVE / SW;                           // words of scales a row and group, rows a load
    static constexpr int NSC = (BN + BM) / SR, NS = (NSC + NW - 1) / NW;        // loads of a group's scales, a wave's
    static constexpr int STAGE = (BN + BM) * BK, SCALES = STAGE * NST, LDS = SCALES + (BN + BM) * SW * 4;
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
    // of its wave's i-th load of scales (the last may be taken by several waves)
    __device__ __forceinline__ uint32_t scale_load(int i) const {
        const uint32_t n = i * NW + wv;
        return n < NSC ? n : NSC - 1;
    }
    __device__ __forceinline__ uint32_t scale_row(int i) const { return scale_load(i) * SR + lane / SW; }

    // rw[i], wo[i]: buffer and this lane's row offset for its i-th eight weight rows; rx, xo: the activations'.  scales(i, rs, so) gives the
    // buffer and this lane's row offset for its i-th scales.
    // a0: the LDS row of this lane's weight row of the wave's first 32 (its place in sixteen is the lane's); the i-th's: a0 + i * astep.
    // live: this wave's 32-row groups of activations that hold any (PART: the others' products are left out).
    // ONCE: the weight rows are this workgroup's alone.
    template <bool PART, bool ONCE, typename Scales>
    __device__ __forceinline__ void run(uint8_t* lds, const i32x4 (&rw)[NA], const uint32_t (&wo)[NA], i32x4 rx,
                                        const uint32_t (&xo)[NB], Scales&& scales, uint32_t nb, uint32_t live, uint32_t a0, uint32_t astep) {
        const uint32_t l0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
        const uint32_t S = (nb + 7) / 8, bytes = 16 * nb, words = (nb + 3) / 4 * 4;
        static_assert(NW % 2 == 0, "a wave's eight rows are all even ones of their sixteen, or all odd");
        const uint32_t piece = 16 * (lane % 8 ^ lane / 8 ^ wv % 2);  // where in a row this lane loads
        // the n-th of a wave's loads of stage s; past the row's end anything, it multiplies zeros by 1
        auto load1 = [&](uint32_t s, uint32_t at, int n) {
            const uint32_t o = s * BK + piece, oc = o < bytes ? o : 0;
            if (n < NA)
                lds_dma<ONCE>(rw[n < NA ? n : 0], wo[n < NA ? n : 0] + oc, at + (n * NW + wv) * 1024);
            else
                lds_dma<false>(rx, xo[n < NA ? 0 : n - NA] + oc, at + (n * NW + wv) * 1024);  // the activations' rows follow the weights'
        };
        // the scales of GS stages from s on
        auto load_scales = [&](uint32_t s) {
#pragma unroll
            for (int i = 0; i < NS; i++) {
                const uint32_t n = scale_load(i), q = 8 * s + 4 * (lane % SW ^ 2 * (n % GS));
                i32x4 rs;
                uint32_t so;
                scales(i, rs, so);
                lds_dma4(rs, so + (q < words ? q : 0), l0 + SCALES + n * 256);
            }
        };
        i32x4 a[2][FN], b[2][FM];
        uint32_t sa[2][FN], sb[2][FM];
        const uint32_t row = lane % 32, half = lane / 32, slot = 16 * (4 * half ^ row % 8 ^ row / 8 % 2), b0 = BN + wm + row;
        auto read = [&](uint32_t at, int s, int to) {
#pragma unroll
            for (int i = 0; i < FN; i++) a[to][i] = *reinterpret_cast<const i32x4*>(lds + at + (a0 + i * astep) * BK + (slot ^ (16 * s)));
#pragma unroll
            for (int j = 0; j < FM; j++)
                if (!PART || j < (int)live)
                    b[to][j] = *reinterpret_cast<const i32x4*>(lds + at + (b0 + j * 32) * BK + (slot ^ (16 * s)));
        };
        auto read_scales = [&](uint32_t s, int to) {
            auto word = [&](uint32_t r) {  // row r's of this lane's half
                return *reinterpret_cast<const uint32_t*>(lds + SCALES + r * (4 * SW) + 4 * ((2 * (s % GS) + half) ^ (2 * (r / SR % GS))));
            };
#pragma unroll
            for (int i = 0; i < FN; i++) sa[to][i] = word(a0 + i * astep);
#pragma unroll
            for (int j = 0; j < FM; j++)
                if (!PART || j < (int)live) sb[to][j] = word(b0 + j * 32);
        };
        // a step's products, with the loads of a stage between them
        auto mul = [&](auto step, int from, auto loads, uint32_t s, uint32_t at) {
            constexpr int ST = decltype(step)::value;
#pragma unroll
            for (int j = 0; j < FM; j++) {
                if (!PART || j < (int)live) {
#pragma unroll
                    for (int i = 0; i < FN; i++)
                        acc[i][j] = mfma_mx4_32<ST>(a[from][i], sa[0][i], b[from][j], sb[0][j], acc[i][j]);
                    // the products stay where they are: on their side of the barrier, and before any branch that lanes part at
                    // (their operands would be made in the lanes that take it alone)
#pragma unroll
                    for (int i = 0; i < FN; i++) asm volatile("" : "+v"(acc[i][j]));
                }
                if constexpr (decltype(loads)::value)
#pragma unroll
                    for (int n = j * NL / FM; n < (j + 1) * NL / FM; n++) load1(s, at, n);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        constexpr std::integral_constant<int, 0> S0{};
        constexpr std::integral_constant<int, 1> S1{};
        constexpr std::integral_constant<int, 2> S2{};
        constexpr std::integral_constant<int, 3> S3{};
        constexpr std::false_type NO{};
        load_scales(0);
#pragma unroll
        for (uint32_t s = 0; s < NST; s++)
            if (s < S)
#pragma unroll
                for (int n = 0; n < NL; n++) load1(s, l0 + s * STAGE, n);
        if (S >= NST)
            wait_dma<(NST - 1) * NL>();
        else
            wait_dma<0>();
        wg_barrier();
        read(0, 0, 0);
        read_scales(0, 0);
        uint32_t cur = 0;
        // a stage that is not the last; `loads`: the stage NST on comes in its place
        auto stage = [&](uint32_t s, auto loads) {
            const uint32_t nxt = cur + STAGE == SCALES ? 0 : cur + STAGE;
            const bool group = (s + 1) % GS == 0;  // the next stage begins one
            read(cur, 1, 1);
            mul(S0, 0, NO, 0, 0);
            read(cur, 2, 0);
            mul(S1, 1, NO, 0, 0);
            read(cur, 3, 1);
            if (!group) read_scales(s + 1, 1);
            mul(S2, 0, NO, 0, 0);
            // the next stage's rows are there; before a group its scales, which no more than one stage's loads follow
            if (!(decltype(loads)::value || s + NST <= S))
                wait_dma<0>();
            else if (NST > 3 && group)
                wait_dma<NL>();
            else
                wait_dma<(NST - 2) * NL>();
            wg_barrier();
            read(nxt, 0, 0);
            if (group)
                read_scales(s + 1, 1);
            else if ((s + 2) % GS == 0 && s + 2 < S)
                load_scales(s + 2);
            mul(S3, 1, loads, s + NST, l0 + cur);
#pragma unroll
            for (int i = 0; i < FN; i++) sa[0][i] = sa[1][i];
#pragma unroll
            for (int j = 0; j < FM; j++) sb[0][j] = sb[1][j];
            cur = nxt;
        };
        uint32_t s = 0;
        for (; s + NST < S; s++) stage(s, std::true_type{});
        for (; s + 1 < S; s++) stage(s, NO);
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
        mul(S0, 0, NO, 0, 0);
        read(cur, 2, 0);
        cut(1, 1);
        mul(S1, 1, NO, 0, 0);
        read(cur, 3, 1);
        cut(2, 0);
        mul(S2, 0, NO, 0, 0);
        cut(3, 1);
        mul(S3, 1, NO, 0, 0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        wg_barrier();  // the stages' LDS is the outputs' from here on
    }

    // A wave's outputs of 32 activation rows by CW weight rows, turned in its part of LDS so that what lies next to another in
    // memory is written together: lane l has row l % 32, v[g] its columns 8 g + 4 (l / 32) .. + 3; out(r, c, x) is given four columns of
    // a row, neighbouring lanes neighbouring ones.
    template <int CW, typename Out>
    __device__ __forceinline__ void turn(uint8_t* lds, const float (&v)[CW / 8][4], Out&& out) const {
        constexpr uint32_t PITCH = CW * 4 + 16, LPR = CW / 4;
        static_assert(NW * 32 * PITCH <= LDS, "the outputs' LDS");
        uint8_t* buf = lds + wv * (32 * PITCH);
        wave_sync();  // the turn before has been read
#pragma unroll
        for (int g = 0; g < CW / 8; g++)
            *reinterpret_cast<f32x4*>(buf + lane % 32 * PITCH + 32 * g + 16 * (lane / 32)) = f32x4{v[g][0], v[g][1], v[g][2], v[g][3]};
        wave_sync();
        f32x4 x[32 * LPR / WAVE];  // all of them before the first goes on
#pragma unroll
        for (uint32_t n = 0; n < 32 * LPR / WAVE; n++)
            x[n] = *reinterpret_cast<const f32x4*>(buf + (n * WAVE + lane) / LPR * PITCH + lane % LPR * 16);
#pragma unroll
        for (uint32_t n = 0; n < 32 * LPR / WAVE; n++) out((n * WAVE + lane) / LPR, lane % LPR * 4, x[n]);
    }
};

}  // namespace trk
