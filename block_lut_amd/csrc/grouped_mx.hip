// Products of rows sorted by expert, MXFP4 matrices with bf16 rows: the weights stay codes until
// the wave that multiplies them widens them in its registers (exactly, four conversions for
// 8 weights).
//
// A CTA is 8 waves on 256 columns and up to 128 rows of one group, a wave 32 columns of all
// rows.  K steps of 128 columns through a ring of stages filled by LDS DMA: each wave's codes
// and scales (32 matrix rows of 64 bytes, 16-byte piece p of row r at p ^ (-(r / 4) % 4); two
// dwords of scales a row, so that they may start anywhere), and the rows that all waves share
// (256 bytes each, chunk c of row r at c ^ swz(r)): reads without bank conflicts.  Lane (i, q)
// holds block 4 s + q of its two matrix rows, and the rows' fragment j of the step is their
// columns 32 q + 8 j .. + 7 (the same permutation of k on both sides).  A fragment is read
// right after the last product of the one that it replaces.
#include "grouped.h"

using namespace lutmoe;

namespace {

constexpr int kCols = 256;

// A stage of a tile of 16 RF rows, and the stages that fit (up to 32 rows: two CTAs a CU).
template <int RF>
struct Ring {
    static constexpr int kLoadF = RF < 2 ? 2 : RF;        // row fragments loaded
    static constexpr int kWave = 2048 + 256;              // codes, scales
    static constexpr int kX = 8 * kWave;                  // the rows behind them
    static constexpr int kStage = kX + kLoadF * 4096;
    static constexpr int kStages = 3;
    static constexpr int kLoads = 3 + kLoadF / 2;         // DMAs a wave and stage
};

__device__ __forceinline__ int swz(int r) { return 4 * quad_order(r & 15) | (r & 3); }

template <int RF>
__device__ __forceinline__ void run_tile(const GroupedArgs& g, const TileAt& t, uint8_t* ring) {
    using Rg = Ring<RF>;
    constexpr int S = Rg::kStages, L = Rg::kLoads, LX = Rg::kLoadF / 2;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, q = lane >> 4;
    const int nrows = min(16 * RF, t.n - t.r0), nb = g.K / 32;
    const int nk = t.e >= g.E ? 0 : (nb + 3) / 4, rem = nb - 4 * (nk - 1);   // blocks of the last step
    const int cw = kCols * t.ct + 32 * wv;
    f32x4_t acc[RF][2];
#pragma unroll
    for (int m = 0; m < RF; ++m) acc[m][0] = acc[m][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    if (nk > 0) {
        const uint32_t l_ring = lds_addr(ring);
        const uint32_t row_b = (uint32_t)(g.K / 2);
        // ---- weights: row r of the wave's 32 is column 8 (r / 4 % 4) + 4 (r / 16) + r % 4 (fragment r / 16;
        // a lane's results lie side by side); columns past the matrix: its last row
        const int c_first = min(cw, g.M - 1);
        const int64_t wrow0 = (int64_t)t.e * g.M + c_first;
        auto column = [&](int r) __attribute__((always_inline)) {
            return (uint32_t)min(8 * ((r >> 2) & 3) + 4 * (r >> 4) + (r & 3), g.M - 1 - c_first);
        };
        const uint8_t* wbase = (const uint8_t*)g.w + wrow0 * row_b;
        const int wpiece = (lane & 3) ^ quad_order(lane >> 2);
        uint32_t wo[2];
#pragma unroll
        for (int d = 0; d < 2; ++d) wo[d] = column(16 * d + (lane >> 2)) * row_b + 16u * (uint32_t)wpiece;
        // scales: lane l dword l % 2 of row l / 2's window, from the aligned base, never past the last dword
        const uint8_t* s0 = (const uint8_t*)g.w_scales + wrow0 * nb;
        const uint32_t first = (uint32_t)((uintptr_t)s0 & 3);
        const uint8_t* sbase = s0 - first;
        const int64_t slast = (int64_t)((((uintptr_t)g.w_scales + (uintptr_t)((int64_t)g.E * g.M * nb) - 1) & ~(uintptr_t)3) -
                                        (uintptr_t)sbase);
        const uint32_t so = ((first + column(lane >> 1) * (uint32_t)nb) & ~3u) + 4u * (uint32_t)(lane & 1);
        // ---- rows: DMA j of the wave covers rows 4 (LX wv + j) .. + 3, lane l chunk l % 16 of row l / 16
        const uint8_t* xbase = (const uint8_t*)g.x + (int64_t)(t.p0 + t.r0) * (2 * (int64_t)g.K);
        uint32_t xo[LX];
#pragma unroll
        for (int j = 0; j < LX; ++j) {
            const int r = 4 * (LX * wv + j) + q;
            xo[j] = (uint32_t)min(r, nrows - 1) * (uint32_t)(2 * g.K) + 16u * (uint32_t)(i ^ swz(r));
        }
        auto issue = [&](int k, uint32_t slot) __attribute__((always_inline)) {
            const bool tail = k == nk - 1;   // pieces past the row's end: the step's first piece again
            const uint32_t lw = l_ring + slot + (uint32_t)(wv * Rg::kWave);
#pragma unroll
            for (int d = 0; d < 2; ++d)
                lds_dma16(wo[d] - (tail && wpiece >= rem ? 16u * (uint32_t)wpiece : 0u), wbase + 64 * (int64_t)k, lw + 1024u * d);
            lds_dma4((uint32_t)min((int64_t)so, slast - 4 * (int64_t)k), sbase + 4 * (int64_t)k, lw + 2048u);
            const uint32_t lx = l_ring + slot + Rg::kX + (uint32_t)(LX * wv) * 1024u;
#pragma unroll
            for (int j = 0; j < LX; ++j) {
                const int c = i ^ swz(4 * (LX * wv + j) + q);
                lds_dma16(xo[j] - (tail && c >= 4 * rem ? 16u * (uint32_t)c : 0u), xbase + 256 * (int64_t)k, lx + 1024u * j);
            }
        };
        // ---- reads
        const uint32_t ar = l_ring + Rg::kX + (uint32_t)(i * 256 + 16 * ((4 * q) ^ swz(i)));
        const uint32_t aw = l_ring + (uint32_t)(wv * Rg::kWave + i * 64 + 16 * (q ^ quad_order(i)));
        uint32_t as[2];
#pragma unroll
        for (int f = 0; f < 2; ++f)
            as[f] = l_ring + (uint32_t)(wv * Rg::kWave + 2048 + 8 * (16 * f + i) + q) + ((first + column(16 * f + i) * (uint32_t)nb) & 3u);
        struct Weights {
            u32x4_t c[2];
            uint32_t s[2];
        };
        Weights w[2];
        u32x4_t fr[RF];
        auto read_w = [&](Weights& v, uint32_t slot) __attribute__((always_inline)) {
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                v.c[f] = lds_quad(aw + slot + 1024 * f);
                v.s[f] = *(lds_byte_t)(as[f] + slot);
            }
        };
        auto read_r = [&](uint32_t slot, int j, int m) __attribute__((always_inline)) {
            fr[m] = lds_quad(((ar + slot) ^ (uint32_t)(16 * j)) + 4096 * m);
        };
        for (int k = 0; k < min(S - 1, nk); ++k) issue(k, (uint32_t)(k * Rg::kStage));
        if (nk > 1) loads_barrier<L>();
        else loads_barrier<0>();
        read_w(w[0], 0);
#pragma unroll
        for (int m = 0; m < RF; ++m) read_r(0, 0, m);
        // slots of the steps k - 1 (refilled: every wave has multiplied it when step k's barrier is
        // behind it), k and k + 1
        uint32_t prev = (uint32_t)((S - 1) * Rg::kStage), slot = 0, next = Rg::kStage;
        auto step = [&](Weights& v, Weights& vn, int k) __attribute__((always_inline)) {
            loads_barrier<0>();   // (S - 3 = 0 stages may be behind step k + 1's)
            if (k - 1 + S < nk) issue(k - 1 + S, prev);
            read_w(vn, next);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const u32x4_t c0 = widen(v.c[0][j], v.s[0]), c1 = widen(v.c[1][j], v.s[1]);
#pragma unroll
                for (int m = 0; m < RF; ++m) {
                    acc[m][0] = mma<kBF>(c0, fr[m], acc[m][0], 0, 0);
                    acc[m][1] = mma<kBF>(c1, fr[m], acc[m][1], 0, 0);
                    read_r(j == 3 ? next : slot, (j + 1) & 3, m);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            const uint32_t p = prev;
            prev = slot;
            slot = next;
            next = p;
        };
        static_assert(S == 3, "three slots rotate");
        for (int k = 0; k + 1 < nk; k += 2) {
            step(w[0], w[1], k);
            if (k + 2 < nk) step(w[1], w[0], k + 1);
            else w[0] = w[1];
        }
        // the last step: blocks past the end are zero on both sides
        const uint32_t keep = q >= rem ? 0u : 0xffffffffu;
        const u32x4_t keep4 = {keep, keep, keep, keep};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const u32x4_t c0 = widen(w[0].c[0][j], w[0].s[0]) & keep4, c1 = widen(w[0].c[1][j], w[0].s[1]) & keep4;
#pragma unroll
            for (int m = 0; m < RF; ++m) {
                const u32x4_t r = fr[m] & keep4;
                acc[m][0] = mma<kBF>(c0, r, acc[m][0], 0, 0);
                acc[m][1] = mma<kBF>(c1, r, acc[m][1], 0, 0);
                if (j < 3) read_r(slot, j + 1, m);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < RF; ++m) {
        const int r = 16 * m + i;
        if (r < nrows) store_row(g, (int64_t)t.p0 + t.r0 + r, cw + 8 * q, g.M, acc[m]);
    }
}

// kTall: tiles of up to 128 rows, else up to 32.
template <bool kTall>
__global__ __launch_bounds__(512, kTall ? 2 : 4) void mx_kernel(GroupedArgs g, int nct) {
    constexpr int kHeight = kTall ? 128 : 32;
    __shared__ __attribute__((aligned(1024))) uint8_t ring[Ring<kHeight / 16>::kStages * Ring<kHeight / 16>::kStage];
    TileAt t;
    if (!find_tile<kHeight>(g, nct, t)) return;
    const int rows = t.n - t.r0;
    if constexpr (kTall) {
        if (rows > 64) run_tile<8>(g, t, ring);
        else if (rows > 32) run_tile<4>(g, t, ring);
        else run_tile<2>(g, t, ring);
    } else {
        if (rows > 16) run_tile<2>(g, t, ring);
        else run_tile<1>(g, t, ring);
    }
}

template <bool kTall>
int mx_launch(const GroupedArgs& g, hipStream_t s) {
    const int nct = (g.M + kCols - 1) / kCols, height = kTall ? 128 : 32;
    const int64_t groups = g.E + (g.zero_rest ? 1 : 0);
    const int64_t ctas = 8 * (((g.P / height + (g.P < groups ? g.P : groups)) * nct + 7) / 8);
    if (ctas >= (int64_t(1) << 31)) return LUTMOE_EUNSUPPORTED;
    hipLaunchKernelGGL((mx_kernel<kTall>), dim3((uint32_t)ctas), dim3(512), 0, s, g, nct);
    return lutmoe_host::check_launch();
}

}  // namespace

namespace lutmoe_host {

int launch_grouped_mx(const GroupedArgs& g, hipStream_t s) {
    // by the average rows of a group that can have any; us, tiles of up to 32 / 128 rows: 60 matrices
    // 2816 x 2048 with 22 / 34 / 205 rows each 53 / 64, 71 / 68, 215 / 185; 8 matrices 28672 x 4096 with 16 / 32 rows
    // 140 / 149, 184 / 166
    const int64_t active = g.P < g.E ? g.P : g.E;
    return g.P > 28 * active ? mx_launch<true>(g, s) : mx_launch<false>(g, s);
}

}  // namespace lutmoe_host
