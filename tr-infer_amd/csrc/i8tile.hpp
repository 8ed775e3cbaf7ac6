// One BN x BM tile of an int8 product on the matrix cores: BN weight rows times BM activation rows over all of K.
//
// K goes by in stages of 128 bytes a row, NST of them in LDS at once.  Rows arrive there by LDS DMA, 16 bytes a lane, no
// register between: a wave's instruction brings eight rows' 128 bytes.  A row's eight pieces lie permuted (piece c of row r
// in slot c ^ (r & 7)), so that the 64 lanes of a fragment's ds_read_b128 (16 rows x 4 pieces) meet no bank twice.  Waves
// hold WN x WM of the tile as 16 x 16 sums and walk a stage in phases, each phase's fragments read during the phase
// before it.  At the last phase of a stage every wave has its fragments in registers: one barrier there hands the
// stage's LDS to the rows NST stages on and opens the next stage, so that rows have (NST - 1) stages' time to arrive.
#pragma once

#include "i8.hpp"

namespace trk {

// 16 bytes a lane from base + off (per lane) to the 1024 bytes of LDS at `lds`; vmcnt counts it.  In asm, because the
// compiler would hold every later LDS read until it has arrived.  m0 is named as overwritten: the compiler has uses for it too.
// ONCE: nobody reads these bytes again, and they are the first that the caches drop.
template <bool ONCE>
__device__ __forceinline__ void lds_dma(i32x4 rsrc, uint32_t off, uint32_t lds) {
    if constexpr (ONCE)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds" ::"s"(lds), "v"(off), "s"(rsrc)
                     : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(rsrc)
                     : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_dma() {  // all but the last N, and this wave's LDS reads
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wg_barrier() {
    asm volatile("s_barrier" ::: "memory");
}

// a raw buffer of any length from p: accesses are in bounds by their offsets
__device__ __forceinline__ i32x4 buffer_at(const int8_t* p) {
    const uint64_t a = (uint64_t)p;
    return i32x4{(int)__builtin_amdgcn_readfirstlane((uint32_t)a),
                 (int)(__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32)) & 0xffffu), -1, 0x00027000};
}

template <int BN_, int BM_, int WN_, int WM_, int NST_>
struct I8Tile {
    static constexpr int BN = BN_, BM = BM_, WN = WN_, WM = WM_, NST = NST_, BK = 128;
    static constexpr int NW = BN / WN * (BM / WM), T = NW * WAVE;
    static constexpr int FN = WN / 16, FM = WM / 16;
    static constexpr int NA = BN / 8 / NW, NB = BM / 8 / NW;  // a wave's loads of a stage
    static constexpr int STAGE = (BN + BM) * BK, LDS = STAGE * NST;
    static constexpr int H = FN * FM > 16 ? 2 : 1, FH = FM / H, P = 2 * H;  // phases of a half stage, of a stage
    static_assert(BN % (8 * NW) == 0 && BM % (8 * NW) == 0 && FM % H == 0 && LDS <= 160 * 1024, "tile");

    i32x4 acc[FN][FM];
    uint32_t lane, wv, wn, wm;  // this wave's first weight and activation row in the tile

    __device__ __forceinline__ I8Tile() {
        wv = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
        wn = wv % (BN / WN) * WN, wm = wv / (BN / WN) * WM;
#pragma unroll
        for (int i = 0; i < FN; i++)
#pragma unroll
            for (int j = 0; j < FM; j++) acc[i][j] = i32x4{0, 0, 0, 0};
    }
    // the tile row that this lane loads of its wave's i-th piece of weights (activations: the same with NB)
    __device__ __forceinline__ uint32_t load_row(int i) const { return (i * NW + wv) * 8 + lane / 8; }

    // rw[i], wo[i]: buffer and this lane's row offset for its i-th eight weight rows; rx, xo: the activations'.
    // lrow(i): the LDS row of the wave's i-th 16 weight rows.
    // live: this wave's 16-row groups of activations that hold any (PART: the others' products are left out).
    // ONCE: the weight rows are this workgroup's alone.
    template <bool PART, bool ONCE, typename Frag>
    __device__ __forceinline__ void run(uint8_t* lds, const i32x4 (&rw)[NA], const uint32_t (&wo)[NA], i32x4 rx,
                                        const uint32_t (&xo)[NB], uint32_t k, uint32_t live, Frag&& lrow) {
        const uint32_t l0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
        const uint32_t S = (k + BK - 1) / BK;
        const uint32_t piece = 16 * (lane % 8 ^ lane / 8);  // where in a row this lane loads
        // the n-th of a wave's loads of stage s
        auto load1 = [&](uint32_t o, uint32_t at, int n) {
            if (n < NA)
                lds_dma<ONCE>(rw[n < NA ? n : 0], wo[n < NA ? n : 0] + o, at + n * NW * 1024);
            else
                lds_dma<false>(rx, xo[n < NA ? 0 : n - NA] + o, at + n * NW * 1024);  // the activations' rows follow the weights'
        };
        auto load_off = [&](uint32_t s) {
            const uint32_t o = s * BK + piece;
            return o < k ? o : 0;  // a piece past the row's end: any, it multiplies zeros
        };
        auto load_at = [&](uint32_t s) { return l0 + s % NST * STAGE + wv * 1024; };
        i32x4 a[2][FN], b[2][FH];
        const uint32_t la = lane % 16 * BK + 16 * (lane / 16 ^ lane % 8);
        auto read_a = [&](uint32_t at, int kk) {
#pragma unroll
            for (int i = 0; i < FN; i++)
                a[kk][i] = *reinterpret_cast<const i32x4*>(lds + at + lrow(i) * BK + (la ^ (64 * kk)));
        };
        auto read_b = [&](uint32_t at, int kk, int h, int to) {
#pragma unroll
            for (int j = 0; j < FH; j++)
                if (!PART || h * FH + j < (int)live)
                    b[to][j] = *reinterpret_cast<const i32x4*>(lds + at + (BN + wm + (h * FH + j) * 16) * BK + (la ^ (64 * kk)));
        };
        // a phase's products, with the loads of a stage between them: all at once they would hold up every wave for as
        // long as the memory pipe takes to accept them
        auto mul = [&](int kk, int h, int from, bool loads, uint32_t o, uint32_t at) {
            if constexpr (PART) {
#pragma unroll
                for (int j = 0; j < FH; j++) {
                    if (h * FH + j < (int)live) {
#pragma unroll
                        for (int i = 0; i < FN; i++) acc[i][h * FH + j] = mfma_i8(a[kk][i], b[from][j], acc[i][h * FH + j]);
#pragma unroll
                        for (int i = 0; i < FN; i++) asm volatile("" : "+v"(acc[i][h * FH + j]));
                    }
                    if (loads)
#pragma unroll
                        for (int n = j * (NA + NB) / FH; n < (j + 1) * (NA + NB) / FH; n++) load1(o, at, n);
                }
            } else {
#pragma unroll
                for (int i = 0; i < FN; i++) {
#pragma unroll
                    for (int j = 0; j < FH; j++) acc[i][h * FH + j] = mfma_i8(a[kk][i], b[from][j], acc[i][h * FH + j]);
                    // the products stay where they are, on their side of the barrier
#pragma unroll
                    for (int j = 0; j < FH; j++) asm volatile("" : "+v"(acc[i][h * FH + j]));
                    if (loads)
#pragma unroll
                        for (int n = i * (NA + NB) / FN; n < (i + 1) * (NA + NB) / FN; n++) load1(o, at, n);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (uint32_t s = 0; s < NST; s++)
            if (s < S)
#pragma unroll
                for (int n = 0; n < NA + NB; n++) load1(load_off(s), load_at(s), n);
        if (S >= NST)
            wait_dma<(NST - 1) * (NA + NB)>();
        else
            wait_dma<0>();
        wg_barrier();
        read_a(0, 0);
        read_b(0, 0, 0, 0);
        uint32_t cur = 0;
        for (uint32_t s = 0; s + 1 < S; s++) {
            const uint32_t nxt = cur + STAGE == LDS ? 0 : cur + STAGE;
#pragma unroll
            for (int p = 0; p < P; p++) {
                if (p == P - 1) {
                    if (s + NST <= S)
                        wait_dma<(NST - 2) * (NA + NB)>();
                    else
                        wait_dma<0>();
                    wg_barrier();
                }
                const int n = (p + 1) % P;
                if (n % H == 0) read_a(n ? cur : nxt, n / H);
                read_b(n ? cur : nxt, n / H, n % H, n & 1);
                mul(p / H, p % H, p & 1, p == P - 1 && s + NST < S, load_off(s + NST), load_at(s + NST));
            }
            cur = nxt;
        }
#pragma unroll
        for (int p = 0; p < P; p++) {  // the last stage, its end past the row's masked
            if (p && p % H == 0) read_a(cur, p / H);
            if (p) read_b(cur, p / H, p % H, p & 1);
            if (k % BK) {
                const uint32_t o = (S - 1) * BK + 64 * (p / H) + 16 * (lane / 16);
                const uint32_t n = o < k ? (k - o < 16 ? k - o : 16) : 0;
#pragma unroll
                for (int j = 0; j < FH; j++) b[p & 1][j] = first_bytes(b[p & 1][j], n);
            }
            mul(p / H, p % H, p & 1, false, 0, 0);
        }
    }
};

// Four neighbouring values of a row of type DT, n of them there (`vec`: all four may be stored as one)
template <uint32_t DT>
__device__ __forceinline__ void store4(typename Elem<DT>::T* y, const float (&v)[4], uint32_t n, bool vec) {
    if (n >= 4 && vec) {
        if constexpr (DT == TRK_DT_F32)
            *reinterpret_cast<float4*>(y) = make_float4(v[0], v[1], v[2], v[3]);
        else
            *reinterpret_cast<ushort4*>(y) = make_ushort4(Elem<DT>::put(v[0]), Elem<DT>::put(v[1]), Elem<DT>::put(v[2]),
                                                          Elem<DT>::put(v[3]));
        return;
    }
#pragma unroll
    for (uint32_t c = 0; c < 4; c++)
        if (c < n) y[c] = Elem<DT>::put(v[c]);
}

}  // namespace trk
