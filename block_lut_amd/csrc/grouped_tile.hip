// Products of rows sorted by expert, tiles: C[r][c] = sum_k A(r, k) B(c, k) with
//   forward  r a group's rows, c the rows of W[e], k columns: both operands k-contiguous
//   dgrad    r a group's rows, c columns of W[e], k rows of W[e]: W transposed on its way
//   wgrad    r rows of dW[e], c its columns, k the group's rows: both transposed
// on MFMA (16 x 16 x 32, 16-bit operands; forward with both operands in MXFP4: the scaled
// 16 x 16 x 128, four times the columns in the same bytes).
//
// A CTA is 4 waves (2 x 2) on a tile of 256 x 256, a wave 128 x 128 in 256 accumulation registers.  A product
// takes a quarter of a fragment from LDS there; on the 128 x 64 of 8 waves half as much again, and LDS, which takes the
// loads too, held those back (60% of the matrix rate).  Where such tiles leave CUs without one: 128 x 128, two
// CTAs a CU.  K goes in stages of 128 bytes a row (64
// columns, MXFP4: 256; whole cache lines, half lines cost a quarter of the time), two substeps each, through
// rings of stages filled by 16-byte LDS DMA: two of the r operand, three (MXFP4: two) of
// the c operand, whose first touch of a matrix comes from HBM.  A substep's fragments are
// read while the one before is multiplied, a read or a load behind every second product: a wave alone on its SIMD
// loses whatever is issued in a row (loads in one half of a stage only: 66% of the matrix rate in a long
// reduction, spread out 75%).  One barrier a stage: behind the first products of its second substep, when its last
// fragments are in registers; it frees the stage's slots and hands over the next stage.
// Layouts of a stage (reads without bank conflicts):
//   k-contiguous  128-byte rows, 16-byte chunk q of row r at q ^ (r / 2 % 8)
//   transposed    rows of the tile's columns (chunk q of row r at q ^ (2 (r % 4) + 8 (r / 8 % 2))), read
//                 by the transposing LDS read (ds_read_b64_tr_b16: 4 rows x 16 columns -> 4
//                 elements of a column a lane)
// CTAs stay for further tiles: the next tile's first loads go out in front of a tile's stores (64
// matrices' gradients, 2816 x 2048 from 192 rows each: 308 us, a CTA a tile 318; with every LDS read of
// the results waited for 408).
// Ragged groups: a group's last tile computes 64, 128 or 192 rows where that is enough (the
// two waves of a column block take alternate 16-row fragments).
// Measured: bf16 8192 rows of 8 matrices 28672 x 4096 1670 us (1150 TFLOP/s; the clock falls to 1.6 GHz
// under it), 12288 rows of 64 matrices 2816 x 2048 190 us (4.5 TB/s), MXFP4 rows 700 us and 78 us; the gradients of
// those rows 1970 and 185 us (dgrad), 1890 and 248 us (wgrad, 738 MB written).
#include "grouped.h"
#include <utility>

using namespace lutmoe;

namespace {

typedef __attribute__((__vector_size__(4 * sizeof(short)))) short s16x4_t;
typedef __attribute__((address_space(3))) s16x4_t* lds_tr_t;
typedef __attribute__((address_space(3))) f32x4_t* lds_f32x4_t;

// A tile of 32 N x 32 N, type kT.  kSD: dwords of MXFP4 scales a row and stage (2, or 3 where they
// start at any byte).
template <int kT, int kSD, int N>
struct Tile {
    static constexpr int kSize = 32 * N;                      // rows, columns
    static constexpr int kSub = kT == kF4 ? 128 : 32;         // columns of a substep
    static constexpr int kOperand = kSize * 128;              // stage bytes of an operand
    static constexpr int kSC = kT == kF4 ? 2 : 3;             // stages of the c operand; of the r operand 2
    static constexpr int kC = 2 * kOperand;                   // LDS: r stages, c stages,
    static constexpr int kScales = kC + kSC * kOperand;       // two stages of scales (r rows, c rows,
    static constexpr int kPlane = 8 * kSize;                  // a dword each, in kSD planes)
    static constexpr int kBytes = kScales + 2 * kSD * kPlane;
};

// 8 elements k of one column: two transposing reads 4 rows (of kRow bytes) apart
template <int kRow>
__device__ __forceinline__ u32x4_t lds_tr(uint32_t a) {
    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_t)a);
    const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_t)(a + 4u * kRow));
    const u32x2_t l = __builtin_bit_cast(u32x2_t, lo), h = __builtin_bit_cast(u32x2_t, hi);
    return u32x4_t{l[0], l[1], h[0], h[1]};
}

// The same with this wave's LDS reads done too (before the barrier that frees a stage).
template <int kAfter>
__device__ __forceinline__ void stage_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kAfter) : "memory");
}

// The tiles of an operation: of every group, or (wgrad) of every matrix, in eighths alike.
template <int kOp, int kSize>
struct Work {
    Tiles<kSize> tiles;
    __device__ __forceinline__ Work(const GroupedArgs& g, int nct) : tiles(g, nct) {}
    __device__ __forceinline__ bool at(const GroupedArgs& g, int b, TileAt& t) {
        if constexpr (kOp != kGroupedWgrad) {
            if (!tiles.at(g, b, t)) return false;
        } else {
            const int nct = tiles.nct, each = (g.M + kSize - 1) / kSize * nct, total = g.E * each, per = (total + 7) / 8;
            const int i = (b & 7) * per + (b >> 3);
            if ((b >> 3) >= per || i >= total) return false;
            t.e = i / each;
            const int in = i - t.e * each, rt = in / nct;
            t.r0 = rt * kSize;
            t.ct = in - rt * nct;
            if (tiles.groups <= 64) {
                t.p0 = __builtin_amdgcn_readlane(tiles.p0, t.e);
                t.n = __builtin_amdgcn_readlane(tiles.n, t.e);
            } else {
                group_rows(g, t.e, t.p0, t.n);
            }
        }
        t.e = __builtin_amdgcn_readfirstlane(t.e);   // (the loads' buffers are in scalar registers)
        t.p0 = __builtin_amdgcn_readfirstlane(t.p0);
        t.n = __builtin_amdgcn_readfirstlane(t.n);
        t.r0 = __builtin_amdgcn_readfirstlane(t.r0);
        t.ct = __builtin_amdgcn_readfirstlane(t.ct);
        return true;
    }
};

template <int MF, int N>
__device__ __forceinline__ void settle(f32x4_t (&acc)[MF][N]) {
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
    for (int m = 0; m < MF; ++m)
#pragma unroll
        for (int f = 0; f < N; f += 2) asm volatile("" : "+a"(acc[m][f]), "+a"(acc[m][f + 1]));
}

// What a wave loads of one operand: its n DMAs of a stage, out of a buffer that ends with the tile's last
// valid row (kTr, transposed: the reduction's last row); what lies past it arrives as zeros, and so
// does a whole stage behind the last.
template <bool kTr, int N, int n>
struct Source {
    static constexpr int kLanes = 4 * N;   // kTr: lanes a row
    const uint8_t* base;
    int rows;                // (kTr: of the reduction)
    uint32_t row, before;    // bytes of a row, and of it in front of base
    uint32_t off[n];         // the lane's offset in each DMA
    u32x4_t src;             // of the stage that is loaded
    uint32_t soff;

    __device__ __forceinline__ static int q(int j) { return (((int)threadIdx.x & 7) ^ ((int)threadIdx.x >> 4 & 3)) ^ (4 * (j & 1)); }
    // first: the wave's row in DMA 0; a lane's further one, and DMA j's, by `lane_row` and `dma_row`
    template <typename L, typename D>
    __device__ __forceinline__ void start(int first, L lane_row, D dma_row) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < n; ++j) {
            const int r = first + lane_row(lane) + dma_row(j);
            const int chunk = kTr ? (lane % kLanes) ^ (((r & 3) << 1) | (r & 8)) : q(j);
            off[j] = (uint32_t)r * row + 16u * (uint32_t)chunk;
        }
        if constexpr (!kTr) src = lds_source(base, (uint32_t)rows * row);
    }
    // before the loads of stage p of np, kStage columns each; the last one's chunks from `valid` on go
    // behind the buffer (valid: 8 where it is whole)
    template <int kStage>
    __device__ __forceinline__ void stage(int p, int np, int valid) {
        asm volatile("" : "+s"(p));   // (no copies of the loop for the last stages)
        if constexpr (kTr) {
            const int left = min(max(rows - p * kStage, 0), kStage);
            src = lds_source(base + (int64_t)p * kStage * row, left ? (uint32_t)left * row - before : 0u);
            soff = 0;
        } else {
            soff = p < np ? 128u * (uint32_t)p : 0x7ffffff0u;
            if (p == np - 1 && valid < 8) {
#pragma unroll
                for (int j = 0; j < n; ++j) off[j] = q(j) < valid ? off[j] : 0x80000000u;
                asm volatile("" : "+v"(off[0]));   // (a branch: no instructions in the other stages)
            }
        }
    }
};

// acc += c x r, in accumulation registers and in place: left to the compiler, 256 of them are split and
// spilled, and the scaled form's result gets registers of its own.  What it does between instructions that
// it knows is done by hand: accumulators settle between products and anything else (settle).  (Operands come
// out of LDS, and scale words are made pairs of products before they are used.)  MXFP4: the scales are
// bytes b / 4 of sc and b % 4 of sr.
template <int b>
__device__ __forceinline__ void mma_f4(f32x4_t& acc, const u32x4_t& c, const u32x4_t& r, uint32_t sc, uint32_t sr) {
    asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0] cbsz:4 blgp:4"
        : "+a"(acc)
        : "v"(c), "v"(r), "v"(sc), "v"(sr), "n"(b >> 2 & 1), "n"(b & 1), "n"(b >> 3), "n"(b >> 1 & 1));
}
template <int kT, int b>
__device__ __forceinline__ void mma_to(f32x4_t& acc, const u32x4_t& c, const u32x4_t& r, uint32_t sc, uint32_t sr) {
    if constexpr (kT == kF4) mma_f4<b>(acc, c, r, sc, sr);
    else if constexpr (kT == kHF) asm("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(acc) : "v"(c), "v"(r));
    else asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(c), "v"(r));
}

// f(0) .. f(n - 1), constants
template <typename F, int... k>
__device__ __forceinline__ void each(std::integer_sequence<int, k...>, F&& f) {
    (f(std::integral_constant<int, k>{}), ...);
}
template <int n, typename F>
__device__ __forceinline__ void each(F&& f) {
    each(std::make_integer_sequence<int, n>{}, f);
}

// A wave's loads of a tile.
template <int kOp, int kT, int kSD, int N>
struct Loads {
    using Tl = Tile<kT, kSD, N>;
    static constexpr int kStage = 2 * Tl::kSub, kChunk = Tl::kSub / 4;   // columns of a stage, a 16-byte chunk
    static constexpr bool kRtr = kOp == kGroupedWgrad, kCtr = kOp != kGroupedFwd, kThree = Tl::kSC == 3;
    static constexpr int L = N, LS = N / 4 * kSD;   // loads of a stage: of each operand, of scales
    uint32_t l0;
    int wv, np, valid;   // stages, chunks of the last one
    int K, rows, cols;   // columns of the reduction, valid rows and columns
    Source<kRtr, N, L> r;
    Source<kCtr, N, L> c;
    uint32_t so[2];      // MXFP4 scales: 64 rows of an operand at a time, a row a lane, the dwords that hold
    u32x4_t ssrc[2];     // the stage's eight bytes, from the tile's aligned base to its last row's last dword

    __device__ __forceinline__ void start(const GroupedArgs& g, const TileAt& t) {
        const int lane = threadIdx.x & 63, C = kOp == kGroupedFwd ? g.M : g.K, c0 = t.ct * Tl::kSize;
        rows = min(Tl::kSize, (kRtr ? g.M : t.n) - t.r0);
        cols = min(Tl::kSize, C - c0);
        K = t.e >= g.E ? 0 : kOp == kGroupedFwd ? g.K : kOp == kGroupedDgrad ? g.M : t.n;
        np = (K + kStage - 1) / kStage;
        const int rem = K - (np - 1) * kStage;
        valid = rem < kStage ? (rem + kChunk - 1) / kChunk : 8;
        const int row_bytes = kT == kF4 ? g.K / 2 : 2 * (kOp == kGroupedDgrad ? g.M : g.K);   // k-contiguous
        auto tr_lane = [](int l) __attribute__((always_inline)) { return l / (4 * N); };
        auto tr_dma = [](int j) __attribute__((always_inline)) { return j * (16 / N); };
        if constexpr (kRtr) {
            r.row = 2 * g.M;
            r.before = 2 * t.r0;
            r.base = (const uint8_t*)g.x + (int64_t)t.p0 * r.row + r.before;
            r.rows = K;
            r.start(16 * wv, tr_lane, tr_dma);
        } else {
            r.row = row_bytes;
            r.base = (const uint8_t*)g.x + (int64_t)(t.p0 + t.r0) * r.row;
            r.rows = rows;
            r.start(8 * L * wv, [](int l) { return l >> 3; }, [](int j) { return 8 * j; });
        }
        if constexpr (kCtr) {
            c.row = 2 * C;
            c.before = 2 * c0;
            c.base = (const uint8_t*)g.w + (kOp == kGroupedDgrad ? (int64_t)t.e * g.M : (int64_t)t.p0) * c.row + c.before;
            c.rows = K;
            c.start(16 * wv, tr_lane, tr_dma);
        } else {
            c.row = row_bytes;
            c.base = (const uint8_t*)g.w + ((int64_t)t.e * g.M + c0) * c.row;
            c.rows = cols;
            // (of 64 columns, row i of fragment f is column 16 (i / 4) + 4 f + i % 4; DMA j: fragment j / 2, i = 8 (j % 2) + lane / 8)
            c.start(N == 8 ? 64 * wv : 64 * (wv >> 1) + 8 * (wv & 1), [](int l) { return 16 * (l >> 5) + ((l >> 3) & 3); },
                    [](int j) { return 32 * (j & 1) + 4 * (j >> 1); });
        }
        if constexpr (kSD > 0) {
            const int kb = g.K / 32;
#pragma unroll
            for (int u = 0; u < N / 4; ++u) {
                const int b = wv + 4 * u, first = 64 * (b % (N / 2));
                const bool is_r = b < N / 2;
                const int64_t row0 = is_r ? (int64_t)(t.p0 + t.r0) : (int64_t)t.e * g.M + c0;
                const uint8_t* s0 = (const uint8_t*)(is_r ? g.x_scales : g.w_scales) + row0 * kb;
                const uint32_t d = kSD == 3 ? (uint32_t)((uintptr_t)s0 & 3) : 0u, n = (uint32_t)(is_r ? rows : cols);
                so[u] = (d + min((uint32_t)(first + lane), n - 1) * (uint32_t)kb) & ~3u;
                ssrc[u] = lds_source(s0 - d, (n * (uint32_t)kb + d + 3u) & ~3u);
            }
        }
    }
    // DMA j of a stage into a slot
    __device__ __forceinline__ void load_r(uint32_t slot, int j) const { lds_dma16(r.off[j], r.src, r.soff, l0 + slot + (uint32_t)(L * wv + j) * 1024u); }
    __device__ __forceinline__ void load_c(uint32_t slot, int j) const {
        lds_dma16(c.off[j], c.src, c.soff, l0 + (uint32_t)Tl::kC + slot + (uint32_t)(L * wv + j) * 1024u);
    }
    __device__ __forceinline__ void load_s(int p) const {
        if constexpr (kSD > 0)
#pragma unroll
            for (int u = 0; u < N / 4; ++u) {
                const uint32_t to = l0 + Tl::kScales + (uint32_t)(p & 1) * (kSD * Tl::kPlane) + 256u * (uint32_t)(wv + 4 * u);
#pragma unroll
                for (int d = 0; d < kSD; ++d) lds_dma4(so[u] + 4 * d, ssrc[u], p < np ? 8u * (uint32_t)p : 0x7ffffff0u, to + Tl::kPlane * d);
            }
    }
    __device__ __forceinline__ void stage_r(int p) { r.template stage<kStage>(p, np, valid); }
    __device__ __forceinline__ void stage_c(int p) { c.template stage<kStage>(p, np, valid); }
    // The first two stages (behind the last one: zeros, here and later, so that counts stay)
    static constexpr int kBehind = (kThree ? L : 0) + LS + L;   // of the loads, those behind stage 0
    __device__ __forceinline__ void first() {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            if (kThree || p == 0) {
                stage_r(p);
#pragma unroll
                for (int j = 0; j < L; ++j) load_r((uint32_t)(p * Tl::kOperand), j);
            }
            load_s(p);
            stage_c(p);
#pragma unroll
            for (int j = 0; j < L; ++j) load_c((uint32_t)(p * Tl::kOperand), j);
        }
    }
};

// One tile, whose first loads are on their way, and behind its products those of the next (more).
// MF: 16-row fragments of a wave that are computed (32 MF of the tile's rows).  `stores`: of the tile before,
// this wave's stores behind those loads if known, else -1; returns this tile's.
template <int kOp, int kT, int kSD, int N, int MF>
__device__ __forceinline__ int run_tile(const GroupedArgs& g, const TileAt& t, const TileAt& tn, bool more, int stores, Loads<kOp, kT, kSD, N>& ld) {
    using Tl = Tile<kT, kSD, N>;
    using Ld = Loads<kOp, kT, kSD, N>;
    constexpr int kSub = Tl::kSub, kStage = Ld::kStage;
    constexpr bool kRtr = Ld::kRtr, kCtr = Ld::kCtr, kThree = Ld::kThree;
    constexpr int kRow = 64 * N;          // bytes of a transposed stage row
    constexpr int kStores = N * N / 2;    // 16-byte stores of a whole tile's 16-bit results, a wave
    const int lane = threadIdx.x & 63, wv = ld.wv;
    const int C = kOp == kGroupedFwd ? g.M : g.K, c0 = t.ct * Tl::kSize;
    const int nrows = ld.rows, Kt = ld.K, np = ld.np;
    const bool whole = MF == N && nrows == Tl::kSize && ld.cols == Tl::kSize && g.out_vec && g.out_dtype != LUTMOE_DTYPE_F32;
    const uint32_t l0 = ld.l0;

    // ---- products
    const int i = lane & 15, gq = lane >> 4, wm = wv >> 1, wn = wv & 1;
    const int iq = i >> 2, ib = i & 3;
    uint32_t ar, ac;
    // (transposed: rows 8 gq + 4 s + iq, 8 bytes of them at column 4 ib of a fragment's 16)
    const uint32_t at_tr = (uint32_t)((8 * gq + iq) * kRow + 8 * (ib & 1)), h_tr = (uint32_t)((iq << 1) | ((gq & 1) << 3));
    if constexpr (kRtr) ar = at_tr + 16u * ((uint32_t)(2 * wm + (ib >> 1)) ^ h_tr);
    else ar = (uint32_t)((16 * wm + i) * 128 + 16 * (gq ^ (i >> 1)));
    if constexpr (kCtr) ac = at_tr + 16u * ((uint32_t)(2 * N * wn + (ib >> 1)) ^ h_tr);
    else ac = (uint32_t)((16 * N * wn + i) * 128 + 16 * (gq ^ (i >> 1)));
    ar += l0;
    ac += l0 + (uint32_t)Tl::kC;
    // MXFP4 scales: lane group q the words (4 blocks) of r fragments 4 h + q and of c fragments 4 h + q
    constexpr int kRH = (MF + 3) / 4, kCH = N / 4;
    uint32_t asr = 0, asc = 0, shift_r = 0, shift_c = 0;
    const uint32_t pick = 0x0c0c0000u | (uint32_t)(4 + gq) << 8 | (uint32_t)gq;
    if constexpr (kSD > 0) {
        const int rr = 32 * gq + 16 * wm + i, cc = 16 * N * wn + 16 * iq + 4 * gq + ib;
        asr = l0 + Tl::kScales + 4u * (uint32_t)rr;
        asc = l0 + Tl::kScales + 4u * (uint32_t)(Tl::kSize + cc);
        if constexpr (kSD == 3) {   // where in its first dword a row's window starts (rows 64 further alike)
            shift_r = ((uint32_t)((uintptr_t)g.x_scales & 3) + (uint32_t)((t.p0 + t.r0 + rr) & 3) * (uint32_t)((g.K / 32) & 3)) & 3u;
            shift_c = ((uint32_t)((uintptr_t)g.w_scales & 3) + (uint32_t)(((int64_t)t.e * g.M + c0 + cc) & 3) * (uint32_t)((g.K / 32) & 3)) & 3u;
        }
    }
    // A substep's fragments are read while the one before is multiplied
    u32x4_t fc[2][N], fr[2][MF];
    struct Words {
        uint32_t c[kCH][2], r[kRH][2];
    };
    Words sw;                             // the next substep's
    uint32_t bc[2][kCH] = {}, br[2][kRH] = {};   // substep s's, a byte a fragment
    // substep s of a stage, into fragments s
    auto read_c = [&](uint32_t slot, int s, int f) __attribute__((always_inline)) {
        if constexpr (kCtr) fc[s][f] = lds_tr<kRow>(((ac + slot) ^ (uint32_t)(32 * f)) + 32 * kRow * s);
        else fc[s][f] = lds_quad(((ac + slot) ^ (uint32_t)(64 * s)) + 2048 * f);
    };
    auto read_r = [&](uint32_t slot, int s, int m) __attribute__((always_inline)) {
        if constexpr (kRtr) fr[s][m] = lds_tr<kRow>(((ar + slot) ^ (uint32_t)(64 * (m & 3))) + 256 * (m >> 2) + 32 * kRow * s);
        else fr[s][m] = lds_quad(((ar + slot) ^ (uint32_t)(64 * s)) + 4096 * m);
    };
    auto read_s = [&](uint32_t slot, int s) __attribute__((always_inline)) {
        if constexpr (kSD > 0)
#pragma unroll
            for (int d = 0; d < kSD - 1; ++d) {
                const uint32_t o = slot + (uint32_t)((s + d) * Tl::kPlane);
#pragma unroll
                for (int h = 0; h < kCH; ++h) sw.c[h][d] = lds_ld32(asc + o + 256 * h);
#pragma unroll
                for (int h = 0; h < kRH; ++h) sw.r[h][d] = lds_ld32(asr + o + 512 * h);
            }
    };
    // word w of substep s, c's first (left: columns from the substep's first on; scales past a row's
    // end are another's)
    constexpr int kWords = kSD > 0 ? kCH + kRH : 0;
    auto use_s = [&](int s, int left, int w) __attribute__((always_inline)) {
        if constexpr (kSD > 0) {
            const uint32_t(&v)[2] = w < kCH ? sw.c[w] : sw.r[w - kCH];
            const uint32_t u = bytes4(kSD == 3 ? __builtin_amdgcn_alignbyte(v[kSD - 2], v[0], w < kCH ? shift_c : shift_r) : v[0], pick);
            (w < kCH ? bc[s][w] : br[s][w - kCH]) = 32 * gq >= left ? 0u : u;
        }
    };
    f32x4_t acc[MF][N];
#pragma unroll
    for (int m = 0; m < MF; ++m)
#pragma unroll
        for (int f = 0; f < N; ++f) acc[m][f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    settle(acc);
    // A substep of S pairs of products; behind each pair what is due there, and nothing moves across:
    // the matrix unit runs while that is issued
    constexpr int S = MF * N / 2, kReads = MF + N;
    auto pair = [&](auto s, auto k) __attribute__((always_inline)) {
        each<2>([&](auto x) __attribute__((always_inline)) {
            constexpr int m = (2 * k + x) / N, f = (2 * k + x) % N;
            mma_to<kT, 4 * (f & 3) + (m & 3)>(acc[m][f], fc[s][f], fr[s][m], bc[s][f >> 2], br[s][m >> 2]);
        });
    };
    constexpr std::integral_constant<int, 0> kFirst;
    constexpr std::integral_constant<int, 1> kSecond;
    // read o of a substep, in the order of their use
    auto read = [&](uint32_t slot_r, uint32_t slot_c, int s, int o) __attribute__((always_inline)) {
        if (o == 0 || o > N) read_r(slot_r, s, o == 0 ? 0 : o - N);
        else read_c(slot_c, s, o - 1);
    };
    // stage 0 has landed (loads and stores are counted together, in order)
    if (stores == 0) stage_barrier<Ld::kBehind>();
    else if (stores == kStores) stage_barrier<Ld::kBehind + kStores>();
    else stage_barrier<0>();
    // Loads are spread over a whole stage, half of them in a substep (more in a row than the address unit
    // takes, and the wave stands still): stage p + 2 of the operand with three slots in the first substep of
    // stage p, that of the other in the second, whose barrier frees its slot.  MXFP4, two slots
    // each: c in the second substep, r (from the L2) in the first one after it.
    if (np > 0) {
        read_s(0, 0);
#pragma unroll
        for (int o = 0; o < kReads; ++o) read(0, 0, 0, o);
#pragma unroll
        for (int w = 0; w < kWords; ++w) use_s(0, Kt, w);
        uint32_t slot_r = 0, slot_c = 0, slot_s = 0;   // of stage p
        uint32_t last_c = (uint32_t)((Tl::kSC - 1) * Tl::kOperand);   // .. of stage p - 1
        for (int p = 0; p < np; ++p) {
            // (addresses are made from these in every stage: hoisted, they take registers)
            asm volatile("" : "+v"(ar), "+v"(ac));
            const int left = Kt - p * kStage;
            const uint32_t next_r = (uint32_t)Tl::kOperand - slot_r, next_s = (uint32_t)(kSD * Tl::kPlane) - slot_s;
            const uint32_t next_c = slot_c == (uint32_t)((Tl::kSC - 1) * Tl::kOperand) ? 0u : slot_c + (uint32_t)Tl::kOperand;
            each<S>([&](auto k) __attribute__((always_inline)) {
                constexpr int Q = (2 * S + 2) / 3;   // (the last third: for the reads to arrive)
                constexpr int L = Ld::L;
                pair(kFirst, k);
                if (k == 0) {
                    if (kThree) ld.stage_c(p + 2);
                    else ld.stage_r(p + 1);
                    read_s(slot_s, 1);
                }
#pragma unroll
                for (int o = k * kReads / Q; o < (k + 1) * kReads / Q && o < kReads; ++o) read(slot_r, slot_c, 1, o);
#pragma unroll
                for (int j = k * L / S; j < (k + 1) * L / S; ++j) {
                    if (kThree) ld.load_c(last_c, j);
                    else ld.load_r(next_r, j);
                }
#pragma unroll
                for (int w = 0; w < kWords; ++w)
                    if (k == S / 2 + w * (S / 2 - 1) / 4) use_s(1, left - kSub, w);
                __builtin_amdgcn_sched_barrier(0);
            });
            // in front of the barrier, which frees the stage's slots and hands over the next one
            constexpr int B = (S + 7) / 8, R = S - B, Q = (2 * R + 2) / 3;
            each<B>([&](auto k) __attribute__((always_inline)) {
                pair(kSecond, k);
                if (k == 0) {
                    if (kThree) ld.stage_r(p + 2);
                    else ld.stage_c(p + 2);
                }
                __builtin_amdgcn_sched_barrier(0);
            });
            stage_barrier<kThree ? Ld::L : 0>();
            each<R>([&](auto k) __attribute__((always_inline)) {
                constexpr int L = Ld::L;
                pair(kSecond, std::integral_constant<int, B + k>{});
                if (k == 0) read_s(next_s, 0);
                if (k == 1) ld.load_s(p + 2);
#pragma unroll
                for (int o = k * kReads / Q; o < (k + 1) * kReads / Q && o < kReads; ++o) read(next_r, next_c, 0, o);
#pragma unroll
                for (int w = 0; w < kWords; ++w)
                    if (k == R / 2 + w * (R / 2 - 1) / 4) use_s(0, left - kStage, w);
#pragma unroll
                for (int j = k * L / R; j < (k + 1) * L / R; ++j) {
                    if (kThree) ld.load_r(slot_r, j);
                    else ld.load_c(slot_c, j);
                }
                __builtin_amdgcn_sched_barrier(0);
            });
            last_c = slot_c;
            slot_r = next_r;
            slot_c = next_c;
            slot_s = next_s;
        }
    }
    stage_barrier<0>();   // every slot is free, and nothing is on its way into LDS
    if (more) {
        ld.start(g, tn);
        ld.first();
    }
    settle(acc);
    // Results leave through LDS, 16 rows of the wave's at a time (every wave its own part of the slot that
    // the next tile's first loads leave free; 16-byte chunks swizzled by the row): whole lines are stored.
    // A wave's LDS accesses are done in order: the next rows are written while these are stored.
    const int64_t out0 = kRtr ? (int64_t)t.e * g.M + t.r0 : t.p0 + t.r0;
    const uint32_t mine = l0 + (uint32_t)(kThree ? Tl::kC + 2 * Tl::kOperand : Tl::kOperand) + (uint32_t)(wv * 16 * kRow);
    constexpr int kAt = 2 * N, kEach = N / 2;   // lanes a row, 8 columns each; rows of a lane
    int el = lane;
    asm volatile("" : "+v"(el));   // (what is made of it is not kept in registers all along)
    const int lc = el % kAt, lr = el / kAt, c = c0 + 16 * N * wn + 8 * lc, ei = el & 15, eq = el >> 4;
    auto put = [&](int m) __attribute__((always_inline)) {
#pragma unroll
        for (int f = 0; f < N; ++f) {
            const int chunk = kCtr ? 4 * f + eq : 16 * (f >> 2) + 4 * eq + (f & 3);
            *(lds_f32x4_t)(mine + (uint32_t)(ei * kRow) + 16u * (uint32_t)(chunk ^ ei)) = acc[m][f];
        }
        asm volatile("" ::: "memory");
    };
    auto get = [&](int rr, f32x4_t (&v)[2]) __attribute__((always_inline)) {
        const uint32_t a = mine + (uint32_t)(rr * kRow);
        v[0] = *(lds_f32x4_t)(a + 16u * (uint32_t)((2 * lc) ^ rr));
        v[1] = *(lds_f32x4_t)(a + 16u * (uint32_t)((2 * lc + 1) ^ rr));
    };
    auto rows16 = [&](auto pack) __attribute__((always_inline)) {
        const uint32_t at = 2u * ((uint32_t)(16 * wm + lr) * (uint32_t)C + (uint32_t)(c - c0));
        uint8_t* base = (uint8_t*)g.out + 2 * (out0 * C + c0);
        put(0);
#pragma unroll
        for (int m = 0; m < MF; ++m) {
            f32x4_t v[kEach][2];
#pragma unroll
            for (int u = 0; u < kEach; ++u) get(lr + 64 / kAt * u, v[u]);
            asm volatile("" ::: "memory");
            if (m + 1 < MF) put(m + 1);
#pragma unroll
            for (int u = 0; u < kEach; ++u) {
                const int r = 32 * m + 64 / kAt * u;
                u32x4_t* to = (u32x4_t*)(base + 2 * (int64_t)r * C + at);
                // (wgrad past the caches, whose results are many times their size: 310 -> 248 us for 738 MB; the others'
                // gain 1 to 3%, and are read next)
                if (16 * wm + lr + r < nrows && c < C) {
                    if constexpr (kRtr) __builtin_nontemporal_store(pack(v[u]), to);
                    else *to = pack(v[u]);
                }
            }
        }
    };
    if (g.out_vec && g.out_dtype == LUTMOE_DTYPE_BF16) {
        rows16([](const f32x4_t(&v)[2]) __attribute__((always_inline)) {
            return u32x4_t{f32x2_to_bf16x2(v[0][0], v[0][1]), f32x2_to_bf16x2(v[0][2], v[0][3]), f32x2_to_bf16x2(v[1][0], v[1][1]), f32x2_to_bf16x2(v[1][2], v[1][3])};
        });
    } else if (g.out_vec && g.out_dtype == LUTMOE_DTYPE_F16) {
        rows16([](const f32x4_t(&v)[2]) __attribute__((always_inline)) {
            u32x4_t u;
#pragma unroll
            for (int d = 0; d < 4; ++d) u[d] = f32_to_f16(v[d >> 1][2 * (d & 1)]) | f32_to_f16(v[d >> 1][2 * (d & 1) + 1]) << 16;
            return u;
        });
    } else {
#pragma unroll
        for (int m = 0; m < MF; ++m) {
            put(m);
#pragma unroll 1
            for (int rr = lr; rr < 16; rr += 64 / kAt) {
                f32x4_t v[2];
                get(rr, v);
                if (32 * m + 16 * wm + rr < nrows) store_row(g, out0 + 32 * m + 16 * wm + rr, c, C, v);
            }
            asm volatile("" ::: "memory");
        }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (before a load into that slot)
    return whole ? kStores : -1;
}

template <int kOp, int kT, int kSD, int N>
__global__ __launch_bounds__(256, N == 8 ? 1 : 2) void tile_kernel(GroupedArgs g, int nct, int end) {
    using Tl = Tile<kT, kSD, N>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Tl::kBytes];
    Work<kOp, Tl::kSize> work(g, nct);
    int b = blockIdx.x, stores = 0;
    auto next = [&](TileAt& t) __attribute__((always_inline)) {
        for (; b < end; b += gridDim.x)
            if (work.at(g, b, t)) {
                b += gridDim.x;
                return true;
            }
        return false;
    };
    TileAt t, tn;
    if (!next(t)) return;
    Loads<kOp, kT, kSD, N> ld;
    ld.l0 = lds_addr(lds);
    ld.wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    ld.start(g, t);
    ld.first();
    for (;;) {
        const bool more = next(tn);
        const int rows = ld.rows;
        if (N == 8 && rows > 192) stores = run_tile<kOp, kT, kSD, N, N>(g, t, tn, more, stores, ld);
        else if (N == 8 && rows > 128) stores = run_tile<kOp, kT, kSD, N, N - N / 4>(g, t, tn, more, stores, ld);
        else if (rows > 64) stores = run_tile<kOp, kT, kSD, N, 4>(g, t, tn, more, stores, ld);
        else stores = run_tile<kOp, kT, kSD, N, 2>(g, t, tn, more, stores, ld);
        if (!more) return;
        t = tn;
    }
}

template <int kOp, int kT, int kSD, int N>
int tile_launch(const GroupedArgs& g, hipStream_t s) {
    using Tl = Tile<kT, kSD, N>;
    const int C = kOp == kGroupedFwd ? g.M : g.K, nct = (C + Tl::kSize - 1) / Tl::kSize;
    // row tiles: a group's last one may be short
    const int64_t groups = g.E + (g.zero_rest ? 1 : 0);
    const int64_t rt = kOp == kGroupedWgrad ? (int64_t)g.E * ((g.M + Tl::kSize - 1) / Tl::kSize)
                                            : g.P / Tl::kSize + (g.P < groups ? g.P : groups);
    const int64_t tiles = 8 * ((rt * nct + 7) / 8);
    if (tiles >= (int64_t(1) << 31) - 512) return LUTMOE_EUNSUPPORTED;
    const int at_once = N == 8 ? 256 : 512;   // CTAs that the 256 CUs hold (a multiple of the 8 XCDs)
    hipLaunchKernelGGL((tile_kernel<kOp, kT, kSD, N>), dim3((uint32_t)(tiles < at_once ? tiles : at_once)), dim3(256), 0, s, g, nct, (int)tiles);
    return lutmoe_host::check_launch();
}

// 128 x 128 where 256 x 256 would be at most about half a tile a CU (every group's last tile counted half):
// 4096 x 4096, 512 rows (32 tiles) 82 -> 37 us, 2048 rows (128) 86 -> 67, 3000 rows (192) 95 -> 104; 8 matrices
// 2816 x 2048 with 256 rows each (88) 52 -> 45, 512 each (176) 54 -> 65; MXFP4 rows, dgrad alike.
template <int kOp, int kT, int kSD>
int tile_size(const GroupedArgs& g, hipStream_t s) {
    const int64_t nct = ((kOp == kGroupedFwd ? g.M : g.K) + 255) / 256;
    const int64_t twice = kOp == kGroupedWgrad ? 2 * (int64_t)g.E * ((g.M + 255) / 256) : g.P / 128 + (g.P < g.E ? g.P : g.E);
    return twice * nct <= 2 * 144 ? tile_launch<kOp, kT, kSD, 4>(g, s) : tile_launch<kOp, kT, kSD, 8>(g, s);
}

}  // namespace

namespace lutmoe_host {

int launch_grouped_tile(const GroupedArgs& g, hipStream_t s) {
    const bool f16 = g.x_dtype == kHF;
    switch (g.op) {
        case kGroupedFwd:
            if (g.x_dtype == kF4) {
                const bool whole = g.K % 128 == 0 && (uintptr_t)g.x_scales % 4 == 0 && (uintptr_t)g.w_scales % 4 == 0;
                return whole ? tile_size<kGroupedFwd, kF4, 2>(g, s) : tile_size<kGroupedFwd, kF4, 3>(g, s);
            }
            return f16 ? tile_size<kGroupedFwd, kHF, 0>(g, s) : tile_size<kGroupedFwd, kBF, 0>(g, s);
        case kGroupedDgrad:
            return f16 ? tile_size<kGroupedDgrad, kHF, 0>(g, s) : tile_size<kGroupedDgrad, kBF, 0>(g, s);
        default:
            return f16 ? tile_size<kGroupedWgrad, kHF, 0>(g, s) : tile_size<kGroupedWgrad, kBF, 0>(g, s);
    }
}

}  // namespace lutmoe_host
