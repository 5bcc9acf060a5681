// Products of rows sorted by expert, tiles: C[r][c] = sum_k A(r, k) B(c, k) with
//   forward  r a group's rows, c the rows of W[e], k columns: both operands k-contiguous
//   dgrad    r a group's rows, c columns of W[e], k rows of W[e]: W transposed on its way
//   wgrad    r rows of dW[e], c its columns, k the group's rows: both transposed
// on MFMA (16 x 16 x 32, 16-bit operands; forward with both operands in MXFP4: the scaled
// 16 x 16 x 128, four times the columns in the same bytes).
//
// A CTA is 8 waves (2 along r x 4 along c, a wave 128 x 64) on a tile of up to 256 x 256.
// K goes in steps of 64 bytes a row (32 columns, MXFP4: 128) through a ring of stages of 32 KB,
// filled by 16-byte LDS DMA; a step's fragments are read while the one before is multiplied.
// Layouts of a stage (reads without bank conflicts):
//   k-contiguous  64-byte rows, 16-byte chunk q of row r at q ^ (-(r / 4) % 4)
//   transposed    512-byte rows of 256 columns (chunk q of row r at q ^ (2 (r % 4) + 8 (r / 8 % 2))), read
//                 by the transposing LDS read (ds_read_b64_tr_b16: 4 rows x 16 columns -> 4
//                 elements of a column a lane)
// A lane's accumulators become 16 consecutive results of one row, whole 16-byte stores: a
// k-contiguous c operand's rows are put in that order on their way to LDS, a transposed one's
// results exchanged between the lane groups at the end.
// Ragged groups: a group's last tile computes 64, 128 or 192 rows where that is enough (the
// two waves of a column block take alternate 16-row fragments).
#include "grouped.h"

using namespace lutmoe;

namespace {

typedef __attribute__((__vector_size__(4 * sizeof(short)))) short s16x4_t;

constexpr int kTile = 256;
constexpr int kOperand = 16384;   // stage bytes of an operand

template <int kT, int kSD>
struct Ring {
    static constexpr int kStage = 2 * kOperand + 2048 * kSD;   // MXFP4: 512 rows' scales, kSD dwords each
    static constexpr int kStages = kT == kF4 ? 4 : 5;
    static constexpr int kStep = kT == kF4 ? 128 : 32;         // columns
};

typedef __attribute__((address_space(3))) s16x4_t* lds_tr_t;
// 8 elements k of one column: two transposing reads 4 rows (2 KB) apart
__device__ __forceinline__ u32x4_t lds_tr(uint32_t a) {
    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_t)a);
    const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_t)(a + 2048u));
    const u32x2_t l = __builtin_bit_cast(u32x2_t, lo), h = __builtin_bit_cast(u32x2_t, hi);
    return u32x4_t{l[0], l[1], h[0], h[1]};
}

// wgrad: every tile of every matrix, in eighths as find_tile's.
__device__ __forceinline__ bool find_wgrad_tile(const GroupedArgs& g, int nct, TileAt& t) {
    const int nrt = (g.M + kTile - 1) / kTile, each = nrt * nct, total = g.E * each, per = (total + 7) / 8;
    const int b = blockIdx.x, i = (b & 7) * per + (b >> 3);
    if ((b >> 3) >= per || i >= total) return false;
    t.e = i / each;
    const int in = i - t.e * each;
    t.r0 = in / nct * kTile;
    t.ct = in - in / nct * nct;
    group_rows(g, t.e, t.p0, t.n);
    t.p0 = __builtin_amdgcn_readfirstlane(t.p0);
    t.n = __builtin_amdgcn_readfirstlane(t.n);
    return true;
}

// MF: 16-row fragments of a wave (the tile has 32 MF rows).
template <int kOp, int kT, int kSD, int MF>
__device__ __forceinline__ void run_tile(const GroupedArgs& g, const TileAt& t, uint8_t* ring) {
    using Rg = Ring<kT, kSD>;
    constexpr int S = Rg::kStages, kStep = Rg::kStep, kChunk = kStep / 4;   // columns of a 16-byte chunk
    constexpr bool kRtr = kOp == kGroupedWgrad, kCtr = kOp != kGroupedFwd;
    constexpr int LR = kRtr ? 4 : MF / 2;   // DMAs of a wave that loads rows (the others: 4)
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int C = kOp == kGroupedFwd ? g.M : g.K, c0 = t.ct * kTile;
    const int nrows = min(32 * MF, (kRtr ? g.M : t.n) - t.r0);   // valid rows of the tile
    const int Kt = t.e >= g.E ? 0 : kOp == kGroupedFwd ? g.K : kOp == kGroupedDgrad ? g.M : t.n;
    const int nk = (Kt + kStep - 1) / kStep, rem = Kt - (nk - 1) * kStep;   // columns of the last step

    // ---- loader: waves 0 .. 3 the r operand, 4 .. 7 the c operand
    const bool is_r = wv < 4;
    const int lw = wv & 3, row_bytes_k = kT == kF4 ? g.K / 2 : 2 * (kOp == kGroupedDgrad ? g.M : g.K);
    const uint8_t* base;
    int64_t advance = 64;
    uint32_t off[4];
    if ((is_r && !kRtr) || (!is_r && !kCtr)) {
        const int valid = is_r ? nrows : min(kTile, C - c0);
        base = is_r ? (const uint8_t*)g.x + (int64_t)(t.p0 + t.r0) * row_bytes_k
                    : (const uint8_t*)g.w + ((int64_t)t.e * g.M + c0) * row_bytes_k;
        const int nl = is_r ? LR : 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // (a c fragment's row i is column 16 (i / 4) + 4 j + i % 4 of the wave's 64)
            const int row = min(is_r ? 16 * (nl * lw + j) + (lane >> 2) : 64 * lw + 16 * (lane >> 4) + 4 * j + ((lane >> 2) & 3), valid - 1);
            const int chunk = (lane & 3) ^ quad_order(lane >> 2);
            off[j] = (uint32_t)row * (uint32_t)row_bytes_k + 16u * (uint32_t)chunk;
        }
    } else {
        // 512-byte rows of 256 columns: two rows a DMA
        const int cols = is_r ? g.M : C, first = is_r ? t.r0 : c0, ld = 2 * cols;
        base = is_r ? (const uint8_t*)g.x + (int64_t)t.p0 * ld
                    : (const uint8_t*)g.w + (kOp == kGroupedDgrad ? (int64_t)t.e * g.M : (int64_t)t.p0) * ld;
        advance = (int64_t)kStep * ld;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int row = 2 * (4 * lw + j) + (lane >> 5);
            const int chunk = min(first / 8 + ((lane & 31) ^ (((row & 3) << 1) | (row & 8))), cols / 8 - 1);
            off[j] = (uint32_t)row * (uint32_t)ld + 16u * (uint32_t)chunk;
        }
    }
    // MXFP4: the scale bytes of row `lane` of the wave's 64: the dword that holds the step's four
    // (kSD 2: the two, at any alignment), `so` from the wave's aligned base
    const uint8_t* sbase = nullptr;
    uint32_t so = 0;
    int64_t slast = 0;
    if constexpr (kSD > 0) {
        const int kb = g.K / 32, valid = is_r ? nrows : min(kTile, C - c0);
        const uint8_t* s0 = is_r ? (const uint8_t*)g.x_scales + (int64_t)(t.p0 + t.r0) * kb
                                 : (const uint8_t*)g.w_scales + ((int64_t)t.e * g.M + c0) * kb;
        const uint8_t* end = is_r ? (const uint8_t*)g.x_scales + (int64_t)g.P * kb
                                  : (const uint8_t*)g.w_scales + (int64_t)g.E * g.M * kb;
        const uint32_t d = kSD == 2 ? (uint32_t)((uintptr_t)s0 & 3) : 0u;
        sbase = s0 - d;
        so = (d + (uint32_t)min(64 * lw + lane, valid - 1) * (uint32_t)kb) & ~3u;
        slast = (int64_t)((((uintptr_t)end - 1) & ~(uintptr_t)3) - (uintptr_t)sbase);
    }
    const uint32_t l_ring = lds_addr(ring);
    // the last step's offsets, where it is short: what lies past the end is read from the
    // step's first chunk (row) instead
    auto tail_off = [&](int j) __attribute__((always_inline)) {
        if ((is_r && !kRtr) || (!is_r && !kCtr)) {
            const int chunk = (lane & 3) ^ quad_order(lane >> 2);
            return off[j] - (chunk * kChunk >= rem ? 16u * (uint32_t)chunk : 0u);
        }
        const int row = 2 * (4 * lw + j) + (lane >> 5);
        return off[j] - (row >= rem ? (uint32_t)row * (uint32_t)(2 * (is_r ? g.M : C)) : 0u);
    };
    // part j of stage k's loads
    auto issue_part = [&](int k, uint32_t slot, int j) __attribute__((always_inline)) {
        const uint8_t* b = base + (int64_t)k * advance;
        const uint32_t l0 = l_ring + slot + (is_r ? (uint32_t)(LR * lw) * 1024u : (uint32_t)kOperand + (uint32_t)lw * 4096u);
        if (!is_r || j < LR) lds_dma16(kSD != 1 && k == nk - 1 && rem < kStep ? tail_off(j) : off[j], b, l0 + 1024u * j);   // (kSD 1: whole steps)
        if (kSD > 0 && j == 0) {
            const uint32_t ls = l_ring + slot + 2 * kOperand + (is_r ? 0u : 1024u) + 256u * (uint32_t)lw;
            lds_dma4(so, sbase + 4 * (int64_t)k, ls);
            if constexpr (kSD == 2) {
                const int64_t last = slast - 4 * (int64_t)k;   // (the last dword of the array)
                lds_dma4((uint32_t)min((int64_t)so + 4, last), sbase + 4 * (int64_t)k, ls + 2048u);
            }
        }
    };

    // ---- compute side
    const int i = lane & 15, gq = lane >> 4, wm = wv >> 2, wn = wv & 3;
    const int iq = i >> 2, ib = i & 3;
    uint32_t ar, ac;
    // (transposed: rows 8 gq + 4 s + iq, 8 bytes of them at column 4 ib of a fragment's 16)
    const uint32_t at_tr = (uint32_t)((8 * gq + iq) * 512 + 8 * (ib & 1)), h_tr = (uint32_t)((iq << 1) | ((gq & 1) << 3));
    if constexpr (kRtr) ar = at_tr + 16u * ((uint32_t)(2 * wm + (ib >> 1)) ^ h_tr);
    else ar = (uint32_t)((16 * wm + i) * 64 + 16 * (gq ^ quad_order(i)));
    if constexpr (kCtr) ac = at_tr + 16u * ((uint32_t)(8 * wn + (ib >> 1)) ^ h_tr);
    else ac = (uint32_t)((64 * wn + i) * 64 + 16 * (gq ^ quad_order(i)));
    ar += l_ring;
    ac += l_ring + kOperand;
    uint32_t asr = 0, asc = 0;   // MXFP4: scale byte addresses
    if constexpr (kSD > 0) {
        auto at = [&](const void* s, int64_t row0, int row) __attribute__((always_inline)) {
            uint32_t q = (uint32_t)gq;
            if constexpr (kSD == 2) q += ((uint32_t)((uintptr_t)s & 3) + (uint32_t)((row0 + row) & 3) * (uint32_t)((g.K / 32) & 3)) & 3u;
            return (uint32_t)(row * 4) + (q >> 2) * 2048u + (q & 3u);
        };
        asr = l_ring + 2 * kOperand + at(g.x_scales, t.p0 + t.r0, 16 * wm + i);
        asc = l_ring + 2 * kOperand + 1024 + at(g.w_scales, (int64_t)t.e * g.M + c0, 64 * wn + 16 * iq + ib);
    }
    // A step's c fragments are read while the one before is multiplied, an r fragment right
    // after the last product of the one that it replaces: a read has most of a step to arrive
    struct ColFrags {
        u32x4_t v[4];
        int s[4];
    };
    ColFrags fc[2];
    u32x4_t fr[MF];
    int sr[MF];
    auto read_c = [&](uint32_t slot, ColFrags& F, int f) __attribute__((always_inline)) {
        if constexpr (kCtr) F.v[f] = lds_tr((ac + slot) ^ (uint32_t)(32 * f));
        else F.v[f] = lds_quad(ac + slot + 1024 * f);
        F.s[f] = 0;
        if constexpr (kSD > 0) F.s[f] = *(lds_byte_t)(asc + slot + 16 * f);
    };
    auto read_r = [&](uint32_t slot, int m) __attribute__((always_inline)) {
        if constexpr (kRtr) fr[m] = lds_tr(((ar + slot) ^ (uint32_t)(64 * (m & 3))) + 256 * (m >> 2));
        else fr[m] = lds_quad(ar + slot + 2048 * m);
        sr[m] = 0;
        if constexpr (kSD > 0) sr[m] = *(lds_byte_t)(asr + slot + 128 * m);
    };
    // columns past the end of the last step: zero in both operands (what was loaded
    // there belongs to something else)
    auto mask = [&](ColFrags& F) __attribute__((always_inline)) {
        uint32_t keep[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const int k = kRtr ? 8 * gq + 2 * d : kChunk * gq;   // (wgrad: single rows end, else whole chunks)
            keep[d] = !kRtr ? (k < rem ? 0xffffffffu : 0u) : k + 1 < rem ? 0xffffffffu : k < rem ? 0xffffu : 0u;
        }
#pragma unroll
        for (int f = 0; f < 4; ++f) {
#pragma unroll
            for (int d = 0; d < 4; ++d) F.v[f][d] &= keep[d];
            if constexpr (kSD > 0) F.s[f] &= keep[0];
        }
#pragma unroll
        for (int m = 0; m < MF; ++m) {
#pragma unroll
            for (int d = 0; d < 4; ++d) fr[m][d] &= keep[d];
            if constexpr (kSD > 0) sr[m] &= keep[0];
        }
    };
    f32x4_t acc[MF][4];
#pragma unroll
    for (int m = 0; m < MF; ++m)
#pragma unroll
        for (int f = 0; f < 4; ++f) acc[m][f] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    // at most `after` stages issued later than the one needed may be in flight
    auto wait_stage = [&](int after) __attribute__((always_inline)) {
        if (is_r) {
            constexpr int L = LR + kSD;
            if (after >= S - 3) loads_barrier<(S - 3) * L>();
            else if (after == 1) loads_barrier<L>();
            else loads_barrier<0>();
        } else {
            constexpr int L = 4 + kSD;
            if (after >= S - 3) loads_barrier<(S - 3) * L>();
            else if (after == 1) loads_barrier<L>();
            else loads_barrier<0>();
        }
    };
    if (nk > 0) {
        for (int k = 0; k < min(S - 1, nk); ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) issue_part(k, (uint32_t)k * Rg::kStage, j);
        wait_stage(min(S - 2, nk - 1));   // stage 0 has landed (the count of S - 3 stages waits for one more)
#pragma unroll
        for (int f = 0; f < 4; ++f) read_c(0, fc[0], f);
#pragma unroll
        for (int m = 0; m < MF; ++m) read_r(0, m);
        // slots of the steps k - 1 (refilled: every wave has multiplied it when step k's
        // barrier is behind it) and k + 1
        uint32_t prev = (uint32_t)(S - 1) * Rg::kStage, next = Rg::kStage;
        auto after_slot = [&](uint32_t s) __attribute__((always_inline)) {
            return s == (uint32_t)(S - 1) * Rg::kStage ? 0u : s + (uint32_t)Rg::kStage;
        };
        auto step = [&](ColFrags& F0, ColFrags& F1, int k) __attribute__((always_inline)) {
            wait_stage(min(S - 3, nk - 2 - k));
            const bool refill = k - 1 + S < nk;
            // (what is loaded and read goes behind products, which hide its issue)
#pragma unroll
            for (int m = 0; m < MF; ++m) {
#pragma unroll
                for (int f = 0; f < 4; ++f) acc[m][f] = mma<kT>(F0.v[f], fr[m], acc[m][f], F0.s[f], sr[m]);
                read_r(next, m);
                constexpr int kPer = MF < 4 ? 2 : 1;   // parts of the rest behind a fragment's products
                if (kPer * m < 4) {
#pragma unroll
                    for (int j = 0; j < kPer; ++j) {
                        read_c(next, F1, kPer * m + j);
                        if (refill) issue_part(k - 1 + S, prev, kPer * m + j);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);   // (a read hoisted higher takes registers that are not there)
            }
            prev = after_slot(prev);
            next = after_slot(next);
        };
        for (int k = 0; k + 1 < nk; k += 2) {
            step(fc[0], fc[1], k);
            if (k + 2 < nk) step(fc[1], fc[0], k + 1);
            else fc[0] = fc[1];
        }
        if (kSD != 1 && rem < kStep) mask(fc[0]);
#pragma unroll
        for (int m = 0; m < MF; ++m)
#pragma unroll
            for (int f = 0; f < 4; ++f) acc[m][f] = mma<kT>(fc[0].v[f], fr[m], acc[m][f], fc[0].s[f], sr[m]);
    }
    const int64_t row0 = kRtr ? (int64_t)t.e * g.M + t.r0 : t.p0 + t.r0;
    const int c = c0 + 64 * wn + 16 * gq;
#pragma unroll
    for (int m = 0; m < MF; ++m) {
        const int r = 32 * m + 16 * wm + i;
        // (transposed c fragments are 16 columns each: a lane's results made consecutive)
        if constexpr (kCtr)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                float v0 = acc[m][0][d], v1 = acc[m][1][d], v2 = acc[m][2][d], v3 = acc[m][3][d];
                transpose4(v0, v1, v2, v3);
                acc[m][0][d] = v0;
                acc[m][1][d] = v1;
                acc[m][2][d] = v2;
                acc[m][3][d] = v3;
            }
        if (r < nrows) store_row(g, row0 + r, c, C, acc[m]);
    }
}

template <int kOp, int kT, int kSD>
__global__ __launch_bounds__(512, 2) void tile_kernel(GroupedArgs g, int nct) {
    __shared__ __attribute__((aligned(1024))) uint8_t ring[Ring<kT, kSD>::kStages * Ring<kT, kSD>::kStage];
    TileAt t;
    if (!(kOp == kGroupedWgrad ? find_wgrad_tile(g, nct, t) : find_tile<kTile>(g, nct, t))) return;
    const int rows = (kOp == kGroupedWgrad ? g.M : t.n) - t.r0;
    if (rows > 192) run_tile<kOp, kT, kSD, 8>(g, t, ring);
    else if (rows > 128) run_tile<kOp, kT, kSD, 6>(g, t, ring);
    else if (rows > 64) run_tile<kOp, kT, kSD, 4>(g, t, ring);
    else run_tile<kOp, kT, kSD, 2>(g, t, ring);
}

template <int kOp, int kT, int kSD>
int tile_launch(const GroupedArgs& g, hipStream_t s) {
    const int C = kOp == kGroupedFwd ? g.M : g.K, nct = (C + kTile - 1) / kTile;
    // row tiles: a group's last one may be short
    const int64_t groups = g.E + (g.zero_rest ? 1 : 0);
    const int64_t rt = kOp == kGroupedWgrad ? (int64_t)g.E * ((g.M + kTile - 1) / kTile)
                                            : g.P / kTile + (g.P < groups ? g.P : groups);
    const int64_t ctas = 8 * ((rt * nct + 7) / 8);
    if (ctas >= (int64_t(1) << 31)) return LUTMOE_EUNSUPPORTED;
    hipLaunchKernelGGL((tile_kernel<kOp, kT, kSD>), dim3((uint32_t)ctas), dim3(512), 0, s, g, nct);
    return lutmoe_host::check_launch();
}

}  // namespace

namespace lutmoe_host {

int launch_grouped_tile(const GroupedArgs& g, hipStream_t s) {
    const bool f16 = g.x_dtype == LUTMOE_DTYPE_F16;
    switch (g.op) {
        case kGroupedFwd:
            if (g.x_dtype == LUTMOE_DTYPE_MXFP4) {
                const bool whole = g.K % 128 == 0 && (uintptr_t)g.x_scales % 4 == 0 && (uintptr_t)g.w_scales % 4 == 0;
                return whole ? tile_launch<kGroupedFwd, kF4, 1>(g, s) : tile_launch<kGroupedFwd, kF4, 2>(g, s);
            }
            return f16 ? tile_launch<kGroupedFwd, LUTMOE_DTYPE_F16, 0>(g, s) : tile_launch<kGroupedFwd, LUTMOE_DTYPE_BF16, 0>(g, s);
        case kGroupedDgrad:
            return f16 ? tile_launch<kGroupedDgrad, LUTMOE_DTYPE_F16, 0>(g, s) : tile_launch<kGroupedDgrad, LUTMOE_DTYPE_BF16, 0>(g, s);
        default:
            return f16 ? tile_launch<kGroupedWgrad, LUTMOE_DTYPE_F16, 0>(g, s) : tile_launch<kGroupedWgrad, LUTMOE_DTYPE_BF16, 0>(g, s);
    }
}

}  // namespace lutmoe_host
