// Products of rows sorted by expert, few rows an expert: every matrix is read once, and what
// counts is that its bytes are always under way.  A CTA computes 16 CR columns of up to 16
// rows of one group, its waves split K (steps of 128 bytes of a matrix row, wave w the steps
// w, w + waves, ..); their partial sums meet in LDS and are added in wave order.  Lane (i, q)
// holds a quarter of row i's step in both operands: a permutation of k that is common to the
// two.
//
// few_kernel     16-bit matrices straight to registers: 5.9 to 6.2 TB/s (60 matrices 2816 x 2048 with 16 rows
//                26 us, 8 matrices 28672 x 4096 with 32 rows 270 us), what streaming reads reach here.
// few_mx_kernel  MXFP4 matrices through LDS that each wave has to itself: the 60 matrices with 128 bf16
//                rows 31.9 us (4.7 TB/s; operands straight to registers 46), MXFP4 rows 30.5.
#include "grouped.h"

using namespace lutmoe;

namespace {


constexpr int kWaves = 4;   // (16-bit matrices)

// 16-bit matrices, D steps of 64 columns of each wave in flight.
template <int kT, int CR, int D>
__global__ __launch_bounds__(64 * kWaves) void few_kernel(GroupedArgs g, int nct) {
    __shared__ f32x4_t s_p[kWaves][CR][64];
    TileAt t;
    if (!find_tile<16>(g, nct, t)) return;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, q = lane >> 4, c0 = 16 * CR * t.ct;
    const int nrows = min(16, t.n - t.r0);
    const int nsteps = t.e >= g.E ? 0 : (g.K + 63) / 64;
    // fragment f's row i is column 4 CR (i / 4) + 4 f + i % 4 (a lane's results lie side by side)
    const uint16_t* wp[CR];
#pragma unroll
    for (int f = 0; f < CR; ++f)
        wp[f] = (const uint16_t*)g.w + ((int64_t)t.e * g.M + min(c0 + 4 * CR * (i >> 2) + 4 * f + (i & 3), g.M - 1)) * g.K;
    const uint16_t* xp = (const uint16_t*)g.x + (int64_t)(t.p0 + t.r0 + min(i, nrows - 1)) * g.K;
    struct Step {
        u32x4_t w[CR][2], x[2];
    };
    // step s: what lies past the row's end is read from its last piece (and masked later)
    auto load = [&](Step& f, int s) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = min(64 * s + 16 * q + 8 * h, g.K - 8);
#pragma unroll
            for (int r = 0; r < CR; ++r) f.w[r][h] = *(const u32x4_t*)(wp[r] + c);
            f.x[h] = *(const u32x4_t*)(xp + c);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    f32x4_t acc[CR];
#pragma unroll
    for (int r = 0; r < CR; ++r) acc[r] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    auto use = [&](Step& f, int s) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (s == nsteps - 1) {   // columns past the end: zero in both operands
                const uint32_t keep = 64 * s + 16 * q + 8 * h < g.K ? 0xffffffffu : 0u;
                const u32x4_t keep4 = {keep, keep, keep, keep};
#pragma unroll
                for (int r = 0; r < CR; ++r) f.w[r][h] &= keep4;
                f.x[h] &= keep4;
            }
#pragma unroll
            for (int r = 0; r < CR; ++r) acc[r] = mma<kT>(f.w[r][h], f.x[h], acc[r], 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // loads without conditions (the compiler's wait counts keep them in flight)
    const int mine = wv < nsteps ? (nsteps - wv + kWaves - 1) / kWaves : 0;   // steps of this wave
    if (mine > 0) {
        Step f[D];
        auto at = [&](int j) __attribute__((always_inline)) { return wv + kWaves * min(j, mine - 1); };
#pragma unroll
        for (int d = 0; d < D; ++d) load(f[d], at(d));
        int j = 0;
        for (; j + D < mine; j += D)
#pragma unroll
            for (int d = 0; d < D; ++d) {
                use(f[d], at(j + d));
                load(f[d], at(j + d + D));
            }
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (j + d < mine) use(f[d], at(j + d));
    }
#pragma unroll
    for (int r = 0; r < CR; ++r) s_p[wv][r][lane] = acc[r];
    __syncthreads();
    if (wv) return;
    // D: lane (row i, q), element d of fragment f -> column 4 CR q + 4 f + d
    f32x4_t sum[CR];
#pragma unroll
    for (int r = 0; r < CR; ++r) {
        sum[r] = s_p[0][r][lane];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) sum[r] += s_p[w][r][lane];
    }
    if (i < nrows) store_row(g, (int64_t)t.p0 + t.r0 + i, c0 + 4 * CR * q, g.M, sum);
}

// CTAs of tiles of `height` rows by `columns`: a group's last row tile may be short.
int64_t few_ctas(const GroupedArgs& g, int height, int columns, int& nct) {
    const int64_t groups = g.E + (g.zero_rest ? 1 : 0);
    nct = (g.M + columns - 1) / columns;
    return 8 * (((g.P / height + (g.P < groups ? g.P : groups)) * nct + 7) / 8);
}

template <int kT, int CR, int D>
int few_launch(const GroupedArgs& g, hipStream_t s) {
    int nct;
    const int64_t ctas = few_ctas(g, 16, 16 * CR, nct);
    if (ctas >= (int64_t(1) << 31)) return LUTMOE_EUNSUPPORTED;
    hipLaunchKernelGGL((few_kernel<kT, CR, D>), dim3((uint32_t)ctas), dim3(64 * kWaves), 0, s, g, nct);
    return lutmoe_host::check_launch();
}

// One wave's K steps of MXFP4 (256 columns): LDS that the wave has to itself, filled by DMA.  Rows
// of the matrix as 8 16-byte pieces on consecutive lanes (a load of 16 bytes from 16 rows on
// consecutive lanes takes the address unit a line a lane, which bounds it: 3.3 TB/s at 14 loads
// per 4 KB), piece p of row r at p ^ swz(r); 16 bytes of scales a row from the dword that holds
// the step's first one; bf16 rows as 32 chunks, chunk c of row r at c ^ xswz(r), MXFP4 ones as the
// matrix.
__device__ __forceinline__ int swz(int r) { return 2 * quad_order(r & 15) | ((r >> 1) & 1); }
__device__ __forceinline__ int xswz(int r) { return ((r >> 1) & 4) | (r & 3); }

template <bool kX4, int CR, int kRows>
struct MxStage {
    static constexpr int kXLoads = kX4 ? (kRows + 7) / 8 : (kRows + 1) / 2;
    static constexpr int kW = 0, kWs = CR * 2048, kX = kWs + CR * 256, kXs = kX + kXLoads * 1024;
    static constexpr int kBytes = kXs + (kX4 ? 256 : 0);
    static constexpr int kLoads = 3 * CR + kXLoads + (kX4 ? 1 : 0);
};

// kRows: rows of a work item (at most 16), S: stages of a wave.
template <bool kX4, int CR, int kRows, int W, int S>
__global__ __launch_bounds__(64 * W) void few_mx_kernel(GroupedArgs g, int nct) {
    using St = MxStage<kX4, CR, kRows>;
    constexpr int L = St::kLoads;
    __shared__ __attribute__((aligned(1024))) uint8_t s_ring[W * S * St::kBytes];
    static_assert(St::kBytes >= CR * 1024, "a wave's partial sums take its stages' place");
    TileAt t;
    if (!find_tile<kRows>(g, nct, t)) return;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, q = lane >> 4, c0 = 16 * CR * t.ct;
    const int nrows = min(kRows, t.n - t.r0), nb = g.K / 32;
    const int nsteps = t.e >= g.E ? 0 : (nb + 7) / 8, rem = nb - 8 * (nsteps - 1);   // blocks of the last step
    const uint32_t ring = lds_addr(s_ring) + (uint32_t)(wv * S * St::kBytes);
    const uint32_t row_b = (uint32_t)(g.K / 2);

    // ---- loads.  Matrix fragment f's row r is column 4 CR (r / 4) + 4 f + r % 4 (a lane's results lie
    // side by side); DMA d of it rows 8 d .. + 7
    const int64_t wrow0 = (int64_t)t.e * g.M + c0, xrow0 = (int64_t)t.p0 + t.r0;
    const uint8_t* wbase = (const uint8_t*)g.w + wrow0 * row_b;
    const uint8_t* xbase = (const uint8_t*)g.x + xrow0 * (kX4 ? row_b : 4 * row_b);
    auto column = [&](int f, int r) __attribute__((always_inline)) {
        return min(4 * CR * (r >> 2) + 4 * f + (r & 3), g.M - 1 - c0);
    };
    auto pieces = [&](int r) __attribute__((always_inline)) { return (lane & 7) ^ swz(r); };
    uint32_t wo[CR][2], xo[St::kXLoads];
#pragma unroll
    for (int f = 0; f < CR; ++f)
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            const int r = 8 * d + (lane >> 3);
            wo[f][d] = (uint32_t)column(f, r) * row_b + 16u * (uint32_t)pieces(r);
        }
#pragma unroll
    for (int d = 0; d < St::kXLoads; ++d) {
        const int r = kX4 ? 8 * d + (lane >> 3) : 2 * d + (lane >> 5);
        const uint32_t row = (uint32_t)min(r, nrows - 1);
        xo[d] = kX4 ? row * row_b + 16u * (uint32_t)pieces(r) : row * 4 * row_b + 16u * (uint32_t)((lane & 31) ^ xswz(r));
    }
    // scales: lane l dword l % 4 of row l / 4's window, which starts at the dword that holds the step's
    // first byte; `so` from the aligned base, never past the array's last dword
    struct Scales {
        const uint8_t* base;
        int64_t last;
        uint32_t first;   // the base's distance from the aligned one
    };
    auto scales = [&](const void* p, int64_t row0, int64_t rows) __attribute__((always_inline)) {
        const uint8_t* b = (const uint8_t*)p + row0 * nb;
        const uint32_t d = (uint32_t)((uintptr_t)b & 3);
        const uint8_t* end = (const uint8_t*)p + rows * nb;
        return Scales{b - d, (int64_t)((((uintptr_t)end - 1) & ~(uintptr_t)3) - (uintptr_t)(b - d)), d};
    };
    const Scales ws = scales(g.w_scales, wrow0, (int64_t)g.E * g.M);
    const Scales xs = kX4 ? scales(g.x_scales, xrow0, g.P) : ws;
    uint32_t wso[CR], xso = 0;
#pragma unroll
    for (int f = 0; f < CR; ++f)
        wso[f] = ((ws.first + (uint32_t)column(f, lane >> 2) * (uint32_t)nb) & ~3u) + 4u * (uint32_t)(lane & 3);
    if constexpr (kX4) xso = ((xs.first + (uint32_t)min(lane >> 2, nrows - 1) * (uint32_t)nb) & ~3u) + 4u * (uint32_t)(lane & 3);
    auto scale_dma = [&](const Scales& c, uint32_t o, int s, uint32_t to) __attribute__((always_inline)) {
        const int64_t last = c.last - 8 * (int64_t)s;
        lds_dma4((uint32_t)min((int64_t)o, last), c.base + 8 * (int64_t)s, to);
    };
    auto issue = [&](int s, uint32_t slot) __attribute__((always_inline)) {
        const uint32_t l0 = ring + slot;
        const bool tail = s == nsteps - 1;
        // pieces past the row's end: the step's first piece again
        auto in_row = [&](uint32_t o, int piece, int per) __attribute__((always_inline)) {
            return o - (tail && piece >= per * rem ? 16u * (uint32_t)piece : 0u);
        };
#pragma unroll
        for (int f = 0; f < CR; ++f) {
#pragma unroll
            for (int d = 0; d < 2; ++d)
                lds_dma16(in_row(wo[f][d], pieces(8 * d + (lane >> 3)), 1), wbase + 128 * (int64_t)s, l0 + St::kW + 2048 * f + 1024 * d);
            scale_dma(ws, wso[f], s, l0 + St::kWs + 256 * f);
        }
#pragma unroll
        for (int d = 0; d < St::kXLoads; ++d) {
            if constexpr (kX4) lds_dma16(in_row(xo[d], pieces(8 * d + (lane >> 3)), 1), xbase + 128 * (int64_t)s, l0 + St::kX + 1024 * d);
            else lds_dma16(in_row(xo[d], (lane & 31) ^ xswz(2 * d + (lane >> 5)), 4), xbase + 512 * (int64_t)s, l0 + St::kX + 1024 * d);
        }
        if constexpr (kX4) scale_dma(xs, xso, s, l0 + St::kXs);
    };

    // ---- reads: lane (i, q) blocks 2 q, 2 q + 1 of row i (rows past the item's: its last loaded one)
    const int xi = min(i, St::kXLoads * (kX4 ? 8 : 2) - 1);
    const uint32_t wr = ring + (uint32_t)(i * 128 + 16 * ((2 * q) ^ swz(i)));
    const uint32_t xr = ring + St::kX + (kX4 ? (uint32_t)(xi * 128 + 16 * ((2 * q) ^ swz(xi)))
                                             : (uint32_t)(xi * 512 + 16 * ((8 * q) ^ xswz(xi))));
    uint32_t wsr[CR];
#pragma unroll
    for (int f = 0; f < CR; ++f)
        wsr[f] = ring + St::kWs + (uint32_t)(256 * f + 16 * i + 2 * q) + ((ws.first + (uint32_t)column(f, i) * (uint32_t)nb) & 3u);
    const uint32_t xsr = ring + St::kXs + (uint32_t)(16 * i + 2 * q) + ((xs.first + (uint32_t)min(i, nrows - 1) * (uint32_t)nb) & 3u);
    f32x4_t acc[CR];
#pragma unroll
    for (int f = 0; f < CR; ++f) acc[f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    auto use = [&](int s, uint32_t slot) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            // blocks past the end: zero on both sides
            const uint32_t keep = s == nsteps - 1 && 2 * q + h >= rem ? 0u : 0xffffffffu;
            const u32x4_t keep4 = {keep, keep, keep, keep};
            u32x4_t w[CR];
            uint32_t wb[CR];
#pragma unroll
            for (int f = 0; f < CR; ++f) {
                w[f] = lds_quad(((wr + slot) ^ (16u * h)) + 2048 * f) & keep4;
                wb[f] = *(lds_byte_t)(wsr[f] + slot + h) & keep;
            }
            if constexpr (kX4) {
                const u32x4_t x = lds_quad((xr + slot) ^ (16u * h)) & keep4;
                const uint32_t xb = *(lds_byte_t)(xsr + slot + h) & keep;
#pragma unroll
                for (int f = 0; f < CR; ++f) acc[f] = mma<kF4>(w[f], x, acc[f], (int)wb[f], (int)xb);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const u32x4_t x = lds_quad((xr + slot) ^ (uint32_t)(64 * h + 16 * j)) & keep4;
#pragma unroll
                    for (int f = 0; f < CR; ++f) acc[f] = mma<kBF>(widen(w[f][j], wb[f]), x, acc[f], 0, 0);
                }
            }
        }
    };
    const int mine = wv < nsteps ? (nsteps - wv + W - 1) / W : 0;   // steps of this wave
#pragma unroll
    for (int d = 0; d < S; ++d)
        if (d < mine) issue(wv + W * d, (uint32_t)(d * St::kBytes));
    uint32_t slot = 0;
    for (int j = 0; j < mine; ++j) {
        // step j has landed: the later stages may be in flight
        const int after = min(S - 1, mine - 1 - j);
        if (after >= 3) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S > 3 ? 3 : 0) * L) : "memory");
        else if (after == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S > 2 ? 2 : 0) * L) : "memory");
        else if (after == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S > 1 ? 1 : 0) * L) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        use(wv + W * j, slot);
        if (j + S < mine) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the stage is read
            issue(wv + W * (j + S), slot);
        }
        slot = slot == (uint32_t)((S - 1) * St::kBytes) ? 0u : slot + (uint32_t)St::kBytes;
    }
    f32x4_t* s_p = (f32x4_t*)s_ring;   // [wave][CR][64] at the waves' first stages
    constexpr int kWaveP = S * St::kBytes / 16;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int f = 0; f < CR; ++f) s_p[wv * kWaveP + 64 * f + lane] = acc[f];
    __syncthreads();
    if (wv) return;
    // D: lane (row i, q), element d of fragment f -> column 4 CR q + 4 f + d
    f32x4_t sum[CR];
#pragma unroll
    for (int f = 0; f < CR; ++f) {
        sum[f] = s_p[64 * f + lane];
#pragma unroll
        for (int w = 1; w < W; ++w) sum[f] += s_p[w * kWaveP + 64 * f + lane];
    }
    if (i < nrows) store_row(g, xrow0 + i, c0 + 4 * CR * q, g.M, sum);
}

template <bool kX4, int CR, int kRows, int W, int S>
int few_mx_launch(const GroupedArgs& g, hipStream_t s) {
    int nct;
    const int64_t ctas = few_ctas(g, kRows, 16 * CR, nct);
    if (ctas >= (int64_t(1) << 31)) return LUTMOE_EUNSUPPORTED;
    hipLaunchKernelGGL((few_mx_kernel<kX4, CR, kRows, W, S>), dim3((uint32_t)ctas), dim3(64 * W), 0, s, g, nct);
    return lutmoe_host::check_launch();
}

// Work items of 16 rows by 16 columns, by the average rows of a group that can have any: what a
// variant is chosen by (the host does not see the groups).
struct Items {
    int64_t rows;    // average, rounded up
    int64_t count;
};
Items items_of(const GroupedArgs& g) {
    const int64_t active = g.P < g.E ? g.P : g.E, rows = (g.P + active - 1) / active;
    return Items{rows, active * ((rows + 15) / 16) * ((g.M + 15) / 16)};
}

// MXFP4 matrices.  A wave's LDS holds its stages, so the rows of an item set how many CTAs a CU
// holds: the fewest rows that the groups fill, wide items where there are plenty, narrow ones
// with more waves along K where CUs would idle.  us, columns x waves x rows a CTA (one stage a
// wave unless said), MI355X:
//   bf16 rows, up to 3 rows a group: 1 matrix 4096 x 14336, 1 row: 16 x 8 x 4 with two stages 9.2, 16 x 4 x 4
//     15.4, 32 x 4 x 4 18; 4 of 60 matrices 2816 x 2048, 1 row: 16 x 4 x 4 5.4, 32 x 4 x 4 6.3, 16 x 8 x 4 6.8;
//     the 60 with 128 rows: 32 x 4 x 4 31.9, 16 x 4 x 4 37.3, 64 x 4 x 8 35.1
//   up to 8 rows, 8 matrices 28672 x 4096 with 4 rows each: 64 x 4 x 8 83.9, 32 x 4 x 8 89.2, 32 x 4 x 16 98.2
//   16 rows, 1 matrix 4096 x 14336 with 16 / 32 / 64 / 128 rows: 16 x 8 12.9 / 22 / 40 / 79, 16 x 4 18 / 18.9 / 36 /
//     57, 32 x 4 20 / 20.6 / 23 / 43, 64 x 4 28 / 28 / 28 / 31
// MXFP4 rows take little LDS at any number: always 16 (60 matrices 2816 x 2048 with 512 rows, 32 x 4 x 16
// / x 8: 38 / 42; with 128 rows 30.5 / 30.0).
template <bool kX4>
int few_mx(const GroupedArgs& g, hipStream_t s) {
    const Items it = items_of(g);
    if constexpr (!kX4) {
        if (it.rows <= 3) {
            if (it.count <= 512) return few_mx_launch<kX4, 1, 4, 8, 2>(g, s);
            if (it.count <= 2048) return few_mx_launch<kX4, 1, 4, 4, 1>(g, s);
            return few_mx_launch<kX4, 2, 4, 4, 1>(g, s);
        }
        if (it.rows <= 8 && it.count > 2048) return few_mx_launch<kX4, 4, 8, 4, 1>(g, s);
    }
    if (it.count <= 256) return few_mx_launch<kX4, 1, 16, 8, 1>(g, s);
    if (it.count <= 768) return few_mx_launch<kX4, 1, 16, 4, 1>(g, s);
    if (it.count <= 1536 || (kX4 && it.rows <= 16)) return few_mx_launch<kX4, 2, 16, 4, 1>(g, s);
    return few_mx_launch<kX4, 4, 16, 4, 1>(g, s);
}

// 16-bit matrices: the wider item where there are plenty, more steps in flight where there are
// few (1 matrix 4096 x 14336 with 1 / 32 rows: 16 columns 25 / 52 us, 32 columns 32 / 41).
template <int kT>
int few_rows(const GroupedArgs& g, hipStream_t s) {
    return items_of(g).count <= 384 ? few_launch<kT, 1, 4>(g, s) : few_launch<kT, 2, 2>(g, s);
}

}  // namespace

namespace lutmoe_host {

// Up to how many rows a group the kernels here are taken (the tiles read a matrix once for up to
// 32, 128 or 256 rows): while its groups are short, or their tiles would leave most CUs
// without one.  us, these / the tiles: 60 matrices 2816 x 2048, bf16 with 240 (960) rows 125 / 146 (191 / 145),
// MXFP4 rows 1200 (1920) 50 / 56 (60 / 57), MXFP4 and bf16 rows 512 (1024) 50.6 / 49.9 (71 / 52); one matrix
// 4096 x 4096, bf16 64 (128) rows 25 / 32 (46 / 36), MXFP4 rows 256 16 / 21; 8 matrices 2816 x 2048, bf16 128
// rows 35 / 27, MXFP4 rows 512 16 / 13.
bool grouped_few_rows(const GroupedArgs& g) {
    const Items it = items_of(g);
    const int rows = !g.w_scales ? 10 : g.x_scales ? 28 : 8;
    return it.rows <= rows || it.count <= (g.w_scales ? 4096 : 1280);
}

int launch_grouped_few(const GroupedArgs& g, hipStream_t s) {
    if (g.w_scales) return g.x_scales ? few_mx<true>(g, s) : few_mx<false>(g, s);
    return g.x_dtype == LUTMOE_DTYPE_F16 ? few_rows<kHF>(g, s) : few_rows<kBF>(g, s);
}

}  // namespace lutmoe_host
