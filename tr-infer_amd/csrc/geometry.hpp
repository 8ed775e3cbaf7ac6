// Launch geometry and workspace extents of the MoE kernels, as plain host arithmetic (no HIP
// types), shared by the launchers, the workspace sizing of trk_create and a CPU-only check that
// sweeps shapes (tests/geometry_check.cpp).  Every grid a launcher builds and every workspace
// extent a kernel indexes is computed here, so a grid that addresses strips past F or a buffer
// sized below what a dispatch writes shows up on the host, without a GPU.  The rules that choose between
// two kernels by size are here too (tests/dispatch_rules_check.cpp: at sizes where both were timed).
#pragma once

#include <stdint.h>

#include <initializer_list>

namespace trk {
namespace geo {

constexpr uint32_t KMAX = 32;      // router.rs:6 MOE_K_MAX: stride of the per-token id / weight rows
constexpr uint32_t ITEM_ROWS = 16; // rows of a grouped work item (one 16-row MFMA tile)
constexpr uint32_t CHUNK = 64;     // tokens per dispatch chunk (one wave's lane mask)
constexpr uint32_t DN_R = 4;       // output rows per decode down workgroup

struct Caps {  // what trk_create sizes for (m_max rows, k_cap selections per token)
    uint32_t H, E, F, m_max, k_cap;
};

inline uint64_t ent_cap(const Caps& c) { return (uint64_t)c.m_max * c.k_cap; }
// work items: every non-empty expert's entries in items of <= 16 rows (at most E + entries / 16 of
// them), then the shared expert's tokens in items of <= 16
inline uint64_t item_cap(const Caps& c) {
    return c.E + (ent_cap(c) + ITEM_ROWS - 1) / ITEM_ROWS + (c.m_max + ITEM_ROWS - 1) / ITEM_ROWS + 1;
}
inline uint64_t items_max(uint32_t E, uint32_t m, uint32_t kcap) {
    const uint64_t ent = (uint64_t)m * kcap;
    const uint64_t nonempty = ent < E ? ent : E;
    return nonempty + ent / ITEM_ROWS + (m + ITEM_ROWS - 1) / ITEM_ROWS;
}
// activation rows of the down input: one per entry and one per token (shared), the decode slots
// (K_MAX routed + the shared one, two levels each), and a TQ batch of up to 16 tokens run as
// per-token decodes (k_cap + 1 slots of two rows per token)
inline uint64_t act_rows(const Caps& c) {
    const uint64_t a = ent_cap(c) + c.m_max, d = (uint64_t)(KMAX + 1) * 2;
    const uint64_t t = 2ull * (c.m_max < 16 ? c.m_max : 16) * (c.k_cap + 1);
    const uint64_t ad = a > d ? a : d;
    return ad > t ? ad : t;
}
inline uint64_t yent_rows(const Caps& c) { return ent_cap(c) + c.m_max; }
// dispatch chunks of 64 tokens, and the per-(chunk, expert) offsets the split dispatch writes
inline uint32_t chunks(uint32_t m) { return (m + CHUNK - 1) / CHUNK; }
inline uint64_t doff_elems(uint32_t m, uint32_t E) { return (uint64_t)chunks(m) * E; }
inline bool dispatch_split(uint32_t m) { return m >= 256; }

// MFMA gate/up: grid.x column blocks of F / 16 / grid.x strips, four waves taking every fourth.
// A wave's strips run one after another, so with few items (one or two rounds of workgroups on
// the GPU) the kernel time is a wave's chain of strips: 128-wide blocks below 2048 rows (M = 512:
// gate/up 210 -> 197 us), 256-wide from 2048 (config 4: 507 against 512 us with 128), 64-wide for
// small batches.
inline uint32_t mfma_gateup_cols(uint32_t m, uint32_t F) {
    return m >= 2048 && F % 256 == 0 ? F / 256 : m >= 64 && F % 128 == 0 ? F / 128 : F / 64;
}
inline uint32_t mfma_gateup_strips(uint32_t m, uint32_t F) { return F / 16 / mfma_gateup_cols(m, F); }
// MFMA gate/up over item pairs from 2048 rows: two items of one expert run as one 32-row tile
// (v_mfma_i32_32x32x32_i8) in a workgroup of eight waves, each taking every eighth strip of the
// column block.  The pair's activations and scales take 40 H bytes of LDS, which leaves room for
// two workgroups per CU up to H = 2048.
inline bool gateup_pairs(uint32_t m, uint32_t H) { return m >= 2048 && H <= 2048; }
inline uint64_t gateup_pair_lds(uint32_t H) { return (uint64_t)H * 40; }
// a pair's workgroup takes 32 strips (four per wave) where F allows: the 80 KB of staged
// activations then serve twice the weights (config 4 gate/up 500 -> 483 us against 16 strips)
inline uint32_t gateup_pair_cols(uint32_t m, uint32_t F) { return F % 512 == 0 ? F / 512 : mfma_gateup_cols(m, F); }
inline uint32_t gateup_pair_strips(uint32_t m, uint32_t F) { return F / 16 / gateup_pair_cols(m, F); }
// MFMA down: grid.x blocks of 256 or 64 output rows, four waves of 16-row strips
inline uint32_t mfma_down_cols(uint32_t m, uint32_t H) { return m >= 64 ? H / 256 : H / 64; }
inline uint32_t mfma_down_rows(uint32_t m, uint32_t H) { return H / mfma_down_cols(m, H); }
// MFMA down over item pairs (two items of one expert share each weight load, unpack and scale
// decode) from 256 rows: config 4's Q6_K down 457 -> 416 us, M = 512's Q4_K down 123 -> 120 us
inline bool down_pairs(uint32_t m) { return m >= 256; }
// streaming down: 4 waves of 64 / (2 NSB) units of 2 NSB lanes (half a superblock each)
inline uint32_t stream_down_rows_per_wg(uint32_t F) { return 4 * (64 / (2 * (F / 256))); }
inline uint32_t stream_down_cols(uint32_t H, uint32_t F) {
    const uint32_t r = stream_down_rows_per_wg(F);
    return (H + r - 1) / r;
}
// decode: gate/up (F / 16 strips, kcap + 1 slots), down H / 4 workgroups
inline uint32_t decode_gateup_strips(uint32_t F) { return F / 16; }
inline uint32_t decode_down_wgs(uint32_t H) { return H / DN_R; }

// TQ layer (k_tq.hip): gate/up strips of 16 over F twice (gate, up), down strips of 16 over H;
// grid.y: the decode slots (kcap + 1) or the work items
inline uint32_t tq_gateup_tiles(uint32_t F) { return 2 * F / 16; }
inline uint32_t tq_down_tiles(uint32_t H) { return H / 16; }

// A launch's workgroups over x and y: a launch holds less than 2^32 threads in x, and a kernel that numbers its
// workgroups in one run takes the rest as rows of y (x * y >= n; multiples of 8 in x keep id % 8 the XCD).
struct Grid2 {
    uint32_t x, y;
};
inline Grid2 grid_run(uint64_t n, uint32_t threads) {
    const uint64_t most = 0xffffffffull / threads / 8 * 8;
    if (n <= most) return Grid2{(uint32_t)n, 1};
    return Grid2{(uint32_t)most, (uint32_t)((n + most - 1) / most)};
}

// Router logits in gemm order (k_router.hip) from 64 rows: VALU tiles of 16 rows x 8 experts (x 2 where
// H is no multiple of 256), or matrix-core tiles of 32 x 32.
inline uint64_t router_valu_wgs(uint32_t m, uint32_t E, uint32_t H) {
    const uint64_t te = H % 256 == 0 ? 8 : 2;
    return (E + te - 1) / te * ((m + 15) / 16);
}
// A matrix-core tile takes as long however few they are (the walk of one workgroup: 16 us at H = 2048),
// while the VALU tiles' time goes with their workgroups per CU.  us, VALU / matrix cores, the kernel alone
// and in a layer (x quantised beside it), H = 2048:
//   up to a workgroup per CU: E = 64 x 200 rows 11.6 / 16.0 and 12.6 / 16.1, E = 16 x 800 11.7 / 16.0
//   and 15 / 18, E = 64 x 500 13.2 / 16.0 and 15.2 / 18.2;
//   up to two, from a few hundred rows on beside as many quantising workgroups: E = 128 x 400 (400 of
//   them) 14.3 / 15.9 and 16.9 / 17.8, E = 384 x 160 (480) 14.3 / 16.0 and 15.0 / 16.0, but E = 128 x 500
//   (512) 15.4 / 16.0 and 19.5 / 18.0, E = 256 x 256 (512) 14.6 / 16.0 and 18.5 / 16.8;
//   beyond: E = 512 x 160 (640) 18.2 / 15.9, x 300 27.7 / 18.5.
// H = 640, 320 and 192 (K-split slices): E = 64 x 500 (1024) 7.3 / 7.6, 5.1 / 5.8 and 4.1 / 4.7, E = 128 x
// 300 (1216) 9.6 / 7.6, 6.9 / 5.9 and 5.3 / 4.7.
inline bool router_on_mfma(uint32_t m, uint32_t E, uint32_t H) {
    if (m < 160 || H % 64) return false;
    const uint64_t valu = router_valu_wgs(m, E, H);
    if (H % 256) return valu > 1024;
    return valu > (m <= 400 ? 480u : m <= 1024 ? 256u : 0u);
}

// The matrix-core tiles walk 256-wide chunks (133 KB of LDS: a CU each) while they and what runs beside them
// have CUs of their own, else 128-wide ones (two tiles per CU).  In a layer the quantising workgroups carry
// the tiles' LDS too, in a few turns on the CUs that the tiles leave: an eighth of the GPU is enough, none
// is not.  us in a layer, 256 / 128 wide: E = 512, H = 2048 x 300 rows (160 tiles) 19.1 / 21.9, x 400
// (208) 18.9 / 22.1, x 500 (256) 26.4 / 21.9; the tiles alone x 500 18.9 / 21.9, x 640 (320) 33.7 / 29.2.
inline bool router_wide_chunks(uint64_t tiles, bool aux) { return tiles + (aux ? 32 : 0) <= 256; }

// trk_gemv tiles (k_gemm.hip) of 128 weight rows (rb blocks of them) x 32 activation rows (t32 blocks) or x 64.
// A 64-row workgroup serves two tiles from one unpacking and takes half as long again as a 32-row one (a
// third at kb 16); up to three per CU the 32-row form is ahead however they divide, beyond it where the
// 64-row form has empty halves.  us, 32 / 64 rows a workgroup:
//   2 and 1 per CU: [12288][2560] TQ5_32 x 128 rows 40 / 53; 3 and 2: x 256 53 / 65, [4096][4096] TQ5_16 x 768
//   147 / 154 and Q6_K 167 / 166 (kb 16: two resident, the third a second round, as dear as the 64-row form);
//   6 and 3: [12288][2560] TQ5_32 x 512 93 / 82, [24576][2048] Q4_K x 256 79 / 63, TQ5_16 x 256 137 / 105;
//   4 and 3: [24576][2048] Q4_K x 160 55 / 60, TQ5_16 x 160 95 / 103; 12 and 8: [131072][768] Q6_K x 96 125 / 112;
//   one block: [150016][2048] Q4_K x 8 (5 and 5) 62 / 93, [248320][2560] TQ8_32 x 8 (8 and 8) 162 / 233.
inline bool gemm_narrow(uint64_t rb, uint64_t t32, uint32_t kb) {
    const uint64_t c32 = (rb * t32 + 255) / 256, c64 = (rb * ((t32 + 1) / 2) + 255) / 256;
    return c32 <= 3 || (kb == 16 ? 3 * c32 <= 4 * c64 : 2 * c32 <= 3 * c64);
}

// trk_gemv on TQ strips of few rows: four rows a workgroup (gemv_quad_kernel) or a strip's sixteen.  Row quads put
// four times the workgroups on the GPU, two per CU at 2048 (row, pass) pairs, for staging that a strip does once:
// they are ahead where a row has enough blocks, earlier while each has a CU of its own and with more activation
// rows (more chains to share), later with 8 bits (the bytes summed besides).  us, strips / quads, at blocks:
//   a CU each, 1024 rows x 1: TQ4_32 10 3.2 / 3.4, 20 3.6 / 3.6, 40 4.1 / 3.8, 80 5.8 / 4.5; TQ8_32 20 3.6 / 3.8, 40
//   4.2 / 4.2, 64 5.0 / 4.6; 320 x 4: TQ8_32 10 4.1 / 4.7, 20 5.3 / 5.0, 40 6.6 / 5.3;
//   two per CU, 2048 rows x 1: TQ5_32 20 3.7 / 4.4, 64 5.3 / 5.2, 128 8.1 / 6.7; TQ8_32 64 5.1 / 5.5, 128 7.9 / 7.3;
//   x 4: TQ4_32 20 5.2 / 5.3, 40 6.5 / 5.7.  [320][10240] TQ8_32 at 1 / 2 / 4 rows 18.3 / 22.9 / 31.8 strips, 11.2 / 12.7
//   / 15.5 quads; beyond 2048, [12288][2560] TQ5_32 x 2 11.3 / 28.5.
// na: activation rows a pass (1, 2, 4).
inline bool gemv_quads(uint64_t row_passes, uint32_t na, uint32_t bits, uint32_t blocks) {
    if (row_passes > 2048) return false;
    if (row_passes <= 1024) return blocks >= (bits == 8 && na < 4 ? 40u : 20u);
    return blocks >= (na == 4 ? 40u : bits != 8 ? 64u : na == 2 ? 80u : 96u);
}

// trk_gemv of many activation rows: its passes of four rows x strips are so many GEMV workgroups, four resident
// per CU, so that it takes whole rounds of 1024; the tiles take as long for one row as for thirty-two.  The
// tiles take over in the third round, before it where they beat two rounds: GGUF formats, whose GEMV decodes
// more, and short columns, where the tiles' unpacking (dearer with more bits) is a smaller part.  us, GEMV /
// tiles, at workgroups:
//   GGUF from 1792: [4096][4096] Q6_K x 28 rows (1792) 89 / 76, [2560][2560] Q4_K x 48 (1920) 41 / 26;
//   TQ [4096][3072] 1792 / 2048 / 2304: TQ4_32 26.5 / 28.8, 29.1 / 28.7, 33.7 / 29.0; TQ5_32 28.1 / 33.3, 30.5 /
//   33.2, 35.1 / 33.3; TQ8_32 27.3 / 33.8, 30.1 / 33.6, 34.9 / 33.9; TQ5_16 48.7 / 52.9, 53.7 / 53.1, 61.0 / 53.0;
//   [256][k] at 1792: TQ4_32 k = 1024 11.6 / 11.5, 1536 15.4 / 15.9; TQ5_32 768 10.8 / 10.4, 1024 12.1 / 13.0;
//   TQ8_32 768 10.8 / 10.5, TQ8_16 512 11.3 / 11.5, 768 14.5 / 15.7;
//   longer ones: [320][10240] TQ4_32 1920 82 / 89, 2080 101 / 89; TQ5_32 1920 87 / 104, 2320 113 / 104; TQ8_32 2060
//   100 / 107, 2320 111 / 106.
inline bool gemv_tiles(uint64_t workgroups, uint32_t tq, uint32_t k) {  // tq: 0 for GGUF, else bits << 8 | kb
    const uint32_t bits = tq >> 8;
    if (tq == 0 || k <= (bits == 4 ? 1024u : tq == 0x810 ? 512u : 768u)) return workgroups >= 1792;
    if (bits == 4 && k <= 3072) return workgroups >= 1920;
    return workgroups > (bits == 8 && k > 3072 ? 2303u : 2048u);
}

// trk_gemm_i8 (k_i8.hip): 16-row strips whose waves share K, or tiles of weight rows x tokens through LDS (256 x 256,
// 128 x 128, 64 x 64, 64 x 32).
enum I8Form { I8_STRIP, I8_TILE_32, I8_TILE_64, I8_TILE_128, I8_TILE_256 };
inline uint64_t i8_tiles(uint64_t rows, uint64_t m, uint32_t bn, uint32_t bm) {
    return (rows + bn - 1) / bn * ((m + bm - 1) / bm);
}
// Strips have every wave's share of K in flight at once and win while each has a CU of its own; beyond it the weights come
// faster through LDS.  us, strips / 64 x 32 tiles, k = 512 and 2560: [1024] x 16 rows (64 strips) 2.6 / 3.1 and 4.2 / 6.2,
// [2560] x 16 (160) 2.7 / 3.1 and 4.8 / 6.4, [5000] x 1 (313) 2.6 / 3.0 and 5.4 / 6.5, x 16 3.1 / 3.1 and 7.1 / 6.5,
// [12288] x 1 (768) 3.5 / 3.6 and 7.2 / 7.0, x 16 4.0 / 3.8 and 9.3 / 7.1.  At long k, weights from memory: k = 8192 [2048] x 1
// 9.4 / 18.6, x 16 12.3 / 18.9; k = 12288 [1024] x 1 12.2 / 25.9, [2560] x 1 13.1 / 25.1, x 16 17.6 / 25.6, [4096] x 16 19.6 / 26.9.
inline bool i8_strips(uint32_t m, uint32_t rows) {
    const uint64_t wgs = i8_tiles(rows, m, 16, 16);
    return wgs <= 256 || (m <= 4 && wgs <= 512);
}
// A tile's time in ns: what it takes to begin and end, and each of its stages (128 bytes of k); n tiles of a CU share it.
// Fitted to, us at 256 x 256 / 128 x 128 / 64 x 64 / 64 x 32: [512] x 48, k = 512 9.0 / 5.9 / 3.9 / 3.4 and k = 4096
// 42 / 23 / 10.4 / 8.7; [2560] x 400, k = 4096 49 / 27 / 13.7 / 17.5; [12288] x 512, k = 2560 41 / 26 / 33 / 43; [6000] x
// 1600, k = 512 15.9 / 15.7 / 18.4 / 26 and k = 4096 49 / 57 / 65 / 89; [12288] x 1024, k = 2560 42 / 47 / 59 / 83,
// x 4096 125 / 148 / 219 / 315; 8192 cubed 423 / 506 / 824 / 1162.
inline uint64_t i8_tile_ns(I8Form f, uint32_t m, uint32_t rows, uint32_t k) {
    const uint64_t S = (k + 127) / 128;
    auto per_cu = [&](uint32_t bn, uint32_t bm) { return (i8_tiles(rows, m, bn, bm) + 255) / 256; };
    if (f == I8_TILE_256) return per_cu(256, 256) * (10000 + 1450 * S);
    if (f == I8_TILE_128) {  // two resident on a CU
        const uint64_t n = per_cu(128, 128);
        return 1500 + n / 2 * (5500 + 850 * S) + n % 2 * (2500 + 660 * S);
    }
    if (f == I8_TILE_64) return 2000 + per_cu(64, 64) * (900 + 190 * S);
    return 2000 + per_cu(64, 32) * (500 + 155 * S);
}
inline I8Form gemm_i8_form(uint32_t m, uint32_t rows, uint32_t k, uint64_t ldw, uint64_t ldq) {
    // the tiles address their rows by 32-bit offsets from the first
    if (ldw >= 1u << 23 || ldq >= 1u << 23 || i8_strips(m, rows)) return I8_STRIP;
    I8Form best = I8_TILE_32;
    for (I8Form f : {I8_TILE_64, I8_TILE_128, I8_TILE_256})
        if (i8_tile_ns(f, m, rows, k) < i8_tile_ns(best, m, rows, k)) best = f;
    return best;
}

// The int8 experts' products (k_i8x.hip): up to eight tokens each entry by itself, beyond it by a plan: entries sorted
// by expert and cut into tiles of at most plan_rows entries of one expert.
// us, up and down by themselves / planned (the plan included; H = 2048): 8 tokens of 10 in 512 experts of F = 512 52 / 58, of 8
// in 128 of 768 60 / 67, of 2 in 8 of 1024 22 / 24; 16 tokens 90 / 89, 105 / 91 and 36 / 24.  By tokens alone: that is wrong for
// many entries an expert, each of which reads its weights (a plan for each product, F = 1024): 8 tokens of 4 in 8 33 / 25, of 8 in
// 8 57 / 26, of 8 in 16 62 / 33; right for few: 4 of 4 in 8 20 / 24, 2 of 8 in 8 21 / 25, 8 of 1 in 1 13 / 20.
constexpr uint32_t DIRECT_M = 8;  // TRK_EXPERTS_DIRECT_M
inline bool plan_used(uint32_t m) { return m > DIRECT_M; }
// us, up at 32 / 64 / 128 rows: 2 entries an expert (4 of 16 x 100 tokens: 25) 7.1 / 7.3 / 8.1, 62 (8 of 128 x 1000) 110 / 94
// / 91, 80 (10 of 512 x 4096) 309 / 270 / 245; down at 10 entries (10 of 512 x 512) 134 / 139 / 154, at 62 93 / 88 / 89.
inline uint32_t plan_rows(uint32_t m, uint32_t slots, uint32_t E) {
    const uint64_t avg = (uint64_t)m * slots / E;
    return avg <= 24 ? 32 : avg <= 48 ? 64 : 128;
}
// An expert's entries seldom need a second tile: its weights are then loaded past the caches' replacement order, so that
// what does come again stays there (down's work rows, the entries' own).  Tiles below 128 rows: always; of 128: up to 64
// entries an expert on average for up, 128 for down.  us, without / with: up, 10 entries (10 of 512 x 512) 199 / 178, 4 (8
// of 128 x 64) 71 / 61, 62 (x 1000) 88 / 83, 80 (10 of 512 x 4096) 232 / 234, 125 (8 of 128 x 2000) 115 / 123, 250 (2 of 8
// x 1000) 25 / 31; down, 39 (10 of 512 x 2000) 189 / 178, 80 294 / 282, 125 135 / 132, 160 (10 of 512 x 8192) 543 / 548, 256
// (4 of 64 x 4096) 262 / 282.
inline bool experts_once(uint32_t m, uint32_t slots, uint32_t E, uint32_t most) { return (uint64_t)m * slots / E <= most; }
// The tiles address weight rows from their block's first, activation rows from the first of all, by 32 bits.
inline bool i8_tile_addresses(uint64_t ldw, uint64_t ldq, uint64_t rows) {
    return ldw < 1u << 23 && ldq <= 0xffffffffull / rows;
}
// Weight rows of an experts' tile (up: of gate and up together): 128, 64 where those leave CUs without a second tile, and
// (up, of 128 entries) 256 from three tiles per CU on.  us: up, 64 / 128 rows, 100 tokens of 4 in 16 experts (H = 1024, F
// = 512) at 32 / 64 / 128 entries a tile 7.1 / 7.5, 7.3 / 10.0, 8.1 / 11.2; down 9.5 / 9.6, 9.2 / 10.1, 9.7 / 11.2; 2000 tokens
// of 8 in 128 (2048, 768) 138 / 124.  Up, 128 / 256: 4096 of 10 in 512 256 / 245, 1000 of 8 in 128 94 / 91, 3000 of 2 in 8 24 / 28.
enum ExpertsWidth { X_NARROW, X_128, X_WIDE };
inline ExpertsWidth experts_width(uint32_t rows, uint64_t tiles, bool wide) {
    const uint64_t wgs = (rows + 127) / 128 * tiles;
    return wgs < 512 ? X_NARROW : wide && wgs >= 1536 ? X_WIDE : X_128;
}
// The plan's words: {tiles, m, slots, E}, ent [m * slots], (16-byte aligned) four words per tile, then the counts of each of
// plan_workgroups' entries [workgroups][E].
inline uint64_t plan_tiles(uint32_t m, uint32_t slots, uint32_t E, uint32_t rows) {  // no call has more
    const uint64_t n = (uint64_t)m * slots;
    return (n < E ? n : E) + n / rows;
}
inline uint64_t plan_tile_at(uint32_t m, uint32_t slots) { return 4 + ((uint64_t)m * slots + 3) / 4 * 4; }
inline uint64_t plan_counts_at(uint32_t m, uint32_t slots, uint32_t E) {
    return plan_tile_at(m, slots) + 4 * plan_tiles(m, slots, E, plan_rows(m, slots, E));
}
// One workgroup sorts up to 4096 entries by itself (us, 1 / several: 3000 entries 6.1 / 7.5, 5120 8.2 / 7.1, 40960 42 / 9.3).
inline uint32_t plan_workgroups(uint32_t m, uint32_t slots) {
    const uint64_t n = (uint64_t)m * slots;
    return n <= 4096 ? 1u : n > 65536 ? 64u : (uint32_t)((n + 1023) / 1024);
}
inline uint64_t plan_words(uint32_t m, uint32_t slots, uint32_t E) {
    const uint32_t wgs = plan_workgroups(m, slots);
    return plan_counts_at(m, slots, E) + (wgs > 1 ? (uint64_t)wgs * E : 0);
}

// trk_gemm_mx4 (k_mx4.hip): the int8 product's forms for 4-bit rows of nb blocks.  A form's time in ns, S stages of eight blocks,
// fitted to 129 sizes; what it chooses there is 0.8 % slower than the best of each (us, strips / 64 x 32 / 64 x 64 / 128 x 128 /
// 256 x 256): k = 512: [512] x 400 3.2 / 3.5 / 3.6 / 4.4 / 10, [5003] x 33 3.2 / 3.9 / 3.8 / 4.6 / 9.2, [12288] x 400 30 / 11.8 / 10.0 / 7.5 / 12,
// x 4096 - / 81 / 66 / 36 / 34; k = 2560: [12288] x 1 4.3 / 5.7 / 6.0 / 8.2 / 20, x 64 16.5 / 7.1 / 6.0 / 8.5 / 20, x 800 - / 40 / 34 / 23 / 27,
// x 4096 - / 190 / 152 / 87 / 81; k = 8192: [2560] x 33 10.8 / 11.8 / 12.0 / 17.5 / 45, x 800 - / 29 / 28 / 25 / 49, [12288] x 800 - / 100 / 79 / 63 / 61.
inline uint64_t mx4_form_ns(I8Form f, uint32_t m, uint32_t rows, uint64_t S) {
    if (f == I8_STRIP) {
        const uint64_t n = i8_tiles(rows, m, 16, 16);  // one to four tokens' rows come from a cache
        return 2200 + 60 * S + (m <= 4 ? n * 70 * S : n * (200 + 110 * S)) / 256;
    }
    auto per_cu = [&](uint32_t bn, uint32_t bm) { return (i8_tiles(rows, m, bn, bm) + 255) / 256; };
    if (f == I8_TILE_32) {
        const uint64_t n = i8_tiles(rows, m, 64, 32);
        return 2900 + 270 * S + (n > 256 ? n - 256 : 0) * (550 + 142 * S) / 256;
    }
    if (f == I8_TILE_64) return 2900 + 272 * S + (per_cu(64, 64) - 1) * (900 + 219 * S);
    if (f == I8_TILE_128) {  // two resident on a CU
        const uint64_t n = per_cu(128, 128);
        return 1200 + n / 2 * (4050 + 830 * S) + n % 2 * (2650 + 490 * S);
    }
    return per_cu(256, 256) * (8050 + 1310 * S);
}
inline I8Form gemm_mx4_form(uint32_t m, uint32_t rows, uint32_t nb, uint64_t ldw, uint64_t ldx, uint64_t sldw, uint64_t sldx) {
    // the tiles address their rows by 32-bit offsets from the first
    if ((ldw | ldx | sldw | sldx) >= 1u << 23) return I8_STRIP;
    I8Form best = I8_STRIP;
    for (I8Form f : {I8_TILE_32, I8_TILE_64, I8_TILE_128, I8_TILE_256})
        if (mx4_form_ns(f, m, rows, (nb + 7ull) / 8) < mx4_form_ns(best, m, rows, (nb + 7ull) / 8)) best = f;
    return best;
}

// trk_moe_mx4 (k_mx4l.hip): the choice by a launch of its own, or by each workgroup of the gate and up launch (`wgs` of them: 32
// rows of an entry each).  us a layer, inside / apart, bf16 x, one shared expert: H = 2048, F = 512, 10 of 512: 1 token (176
// workgroups) 18.8 / 20.4, 2 23.2 / 25.4, 4 (704) 32.8 / 34.7, 8 (1408) 52.9 / 50.7; 8 of 256, F = 768, 8 tokens (1728) 62.3 / 57.5;
// 2 of 8, F = 1024, 8 (768) 22.9 / 24.9; 8 of 8 (2304) 50.0 / 46.0.
inline bool layer_routes_apart(uint64_t wgs) { return wgs > 1024; }
// Waves of a workgroup of its down launch, a slot at a time each: 4 or 12 of 16 rows of a token (`wgs` such workgroups), 8 of 32.  us a
// layer, 4 / 8 / 12: the same layers' 1 token (128 workgroups) 19.8 / 20.3 / 18.7, 2 24.4 / 26.2 / 23.1, 4 (512) 32.8 / 31.6 / 31.4, 8
// (1024) 46.5 / 45.7 / 47.5; F = 768, 8 52.6 / 51.5 / 53.6; 8 of 8, 8 45.8 / 43.9 / -; few slots: 2 of 8, 8 21.0 / 21.0 / 23.0, 2 of 10
// 13.7 / 14.1 / -.  The eight hold 32 slots' sums in LDS.
inline uint32_t layer_down_waves(uint64_t wgs, uint32_t slots) {
    if (slots <= 4) return 4;
    return wgs <= 512 ? 12 : slots <= 32 ? 8 : 4;
}

// Every invariant a call of m rows with kcap selections per token relies on; returns nullptr when
// they hold, else what failed.  tq: the experts are TQ strips (k_tq.hip), not GGUF superblocks.
inline const char* check_call(const Caps& c, uint32_t m, uint32_t kcap, bool tq = false) {
    if (c.H == 0 || c.H % 256) return "H must be a multiple of 256";
    if (c.F == 0 || c.F % (tq ? 16 : 256)) return tq ? "F must be a multiple of 16" : "F must be a multiple of 256";
    if (m == 0 || m > c.m_max) return "m outside 1..m_max";
    if (kcap == 0 || kcap > c.k_cap || kcap > KMAX) return "kcap outside 1..k_cap";
    if ((uint64_t)m * kcap > ent_cap(c)) return "entries above the entry capacity";
    if (items_max(c.E, m, kcap) > item_cap(c)) return "work items above the item capacity";
    if ((uint64_t)m * kcap + m > act_rows(c) || (uint64_t)m * kcap + m > yent_rows(c))
        return "activation rows above capacity";
    if (doff_elems(m, c.E) > doff_elems(c.m_max, c.E)) return "dispatch offsets above capacity";
    if (tq) {
        if (tq_gateup_tiles(c.F) * 16 != 2 * c.F || tq_down_tiles(c.H) * 16 != c.H) return "TQ strips do not tile F / H";
        // decode: slots 0..kcap (the shared one last) in h / yent rows and in the [33][2] act rows
        if (m == 1 && ((uint64_t)kcap + 1 > yent_rows(c) || (uint64_t)(KMAX + 1) * 2 > act_rows(c)))
            return "decode slots above capacity";
        return nullptr;
    }
    {  // MFMA gate/up: the column blocks tile F's strips exactly, four waves each
        const uint32_t cols = mfma_gateup_cols(m, c.F), s = mfma_gateup_strips(m, c.F);
        if (cols == 0 || cols * s * 16 != c.F || s % 4) return "MFMA gate/up grid does not tile F";
        // the pairs' workgroups: eight waves over the block's strips (the launcher runs every item
        // on the 16-row path otherwise), and two workgroups' LDS per CU
        if (gateup_pairs(m, c.H) && gateup_pair_strips(m, c.F) % 8 == 0 && 2 * gateup_pair_lds(c.H) > 160 * 1024)
            return "MFMA gate/up pair LDS above 80 KiB";
    }
    {  // MFMA down: the row blocks tile H exactly, 16-row strips over four waves
        const uint32_t cols = mfma_down_cols(m, c.H), r = mfma_down_rows(m, c.H);
        if (cols == 0 || cols * r != c.H || r % 64) return "MFMA down grid does not tile H";
    }
    {  // streaming down: the row blocks cover H (the kernel guards rows past H)
        const uint32_t r = stream_down_rows_per_wg(c.F);
        if (r == 0 || (uint64_t)stream_down_cols(c.H, c.F) * r < c.H) return "stream down grid does not cover H";
    }
    if (m == 1) {  // decode: slots 0..kcap-1 and the shared slot, strips of F, rows of H
        if (decode_gateup_strips(c.F) * 16 != c.F) return "decode gate/up strips do not tile F";
        if (decode_down_wgs(c.H) * DN_R != c.H) return "decode down workgroups do not tile H";
        if ((uint64_t)(KMAX + 1) * 2 > act_rows(c)) return "decode activation slots above capacity";
    }
    return nullptr;
}

}  // namespace geo
}  // namespace trk
