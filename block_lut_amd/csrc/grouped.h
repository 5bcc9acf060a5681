// Shared by the grouped products' kernels: groups, the tile of a CTA, stores of results.
#pragma once
#include "common.h"
#include "kernels.h"
#include "lut_core.h"

namespace lutmoe {

using lutmoe_host::GroupedArgs;

typedef __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16 f16x8_t;
typedef __attribute__((__vector_size__(8 * sizeof(int)))) int i32x8_t;

constexpr int kF4 = LUTMOE_DTYPE_MXFP4;   // (kernel template arguments)
constexpr int kBF = LUTMOE_DTYPE_BF16, kHF = LUTMOE_DTYPE_F16;

// Group e's rows, clamped into [0, P] (the first starts at row 0); e = E: the rows behind,
// e > E: none.
__device__ __forceinline__ void group_rows(const GroupedArgs& g, int e, int& p0, int& n) {
    const int a = e <= 0 || !g.offsets ? 0 : min(max(g.offsets[min(e, g.E)], 0), g.P);
    const int b = e >= g.E || !g.offsets ? g.P : min(max(g.offsets[e + 1], 0), g.P);
    p0 = a;
    n = e > g.E ? 0 : max(b - a, 0);
}

struct TileAt {
    int e, p0, n;   // group (E: the rows behind), its first row, rows
    int r0, ct;     // first row of the tile in the group, column tile
};

// Inclusive sum over the wave's lanes (row shifts within 16 lanes, then the rows' totals).
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // row_bcast:31 into rows 2 and 3
    return v;
}

// The tile of a CTA among tiles of kHeight rows of a group by nct columns.  Each eighth of the
// tiles runs on one XCD (a CTA's index modulo 8), group by group; in a group up to 8 row
// tiles go along with a column tile.  Every wave finds it by itself: the tiles of 64 groups
// at a time summed up across its lanes (up to 64 groups: one load of the offsets, one sum).
template <int kHeight>
struct Tiles {
    int nct, groups, total, p0, n, mine, upto;

    __device__ __forceinline__ int sums(const GroupedArgs& g, int e0) {
        const int lane = threadIdx.x & 63;
        group_rows(g, e0 + lane, p0, n);
        if (e0 + lane >= groups) n = 0;
        mine = (n + kHeight - 1) / kHeight;
        upto = wave_scan(mine);
        return __builtin_amdgcn_readlane(upto, 63);
    }
    __device__ __forceinline__ Tiles(const GroupedArgs& g, int nct_) : nct(nct_), groups(g.E + (g.zero_rest ? 1 : 0)), total(0) {
        for (int e0 = 0; e0 < groups; e0 += 64) total += sums(g, e0);
        total *= nct;
    }
    // the tile of CTA b
    __device__ __forceinline__ bool at(const GroupedArgs& g, int b, TileAt& t) {
        const int per = (total + 7) / 8, i = (b & 7) * per + (b >> 3);
        if ((b >> 3) >= per || i >= total) return false;
        int before = 0;
        for (int e0 = 0; e0 < groups; e0 += 64) {
            if (groups > 64) sums(g, e0);
            const uint64_t m = __ballot(i < before + upto * nct);
            if (m) {
                const int l = __builtin_ctzll(m);
                t.e = e0 + l;
                t.p0 = __builtin_amdgcn_readlane(p0, l);
                t.n = __builtin_amdgcn_readlane(n, l);
                const int mt = __builtin_amdgcn_readlane(mine, l);
                const int in = i - before - (__builtin_amdgcn_readlane(upto, l) - mt) * nct;
                if (mt == 1) {
                    t.ct = in;
                    t.r0 = 0;
                } else {
                    const int grp = in / (8 * nct), size = min(8, mt - 8 * grp), rem = in - grp * 8 * nct;
                    t.ct = rem / size;
                    t.r0 = (8 * grp + rem - t.ct * size) * kHeight;
                }
                // (decreasing offsets can count more tiles than an int holds)
                return (uint32_t)t.r0 < (uint32_t)t.n && (uint32_t)t.ct < (uint32_t)nct;
            }
            before += __builtin_amdgcn_readlane(upto, 63) * nct;
        }
        return false;
    }
};
template <int kHeight>
__device__ __forceinline__ bool find_tile(const GroupedArgs& g, int nct, TileAt& t) {
    return Tiles<kHeight>(g, nct).at(g, blockIdx.x, t);
}

// 4 Q results of one row from its column c on (C columns in all): whole vectors where the
// rows are aligned, else one by one.
template <int Q>
__device__ __forceinline__ void store_row(const GroupedArgs& g, int64_t row, int c, int C, const f32x4_t (&v)[Q]) {
    if (c >= C) return;
    const int64_t o = row * C + c;
    if (g.out_dtype == LUTMOE_DTYPE_F32) {
        float* p = (float*)g.out + o;
        if (g.out_vec) {
#pragma unroll
            for (int q = 0; q < Q; ++q)
                if (c + 4 * q < C) *(f32x4_t*)(p + 4 * q) = v[q];
        } else {
#pragma unroll
            for (int q = 0; q < 4 * Q; ++q)
                if (c + q < C) p[q] = v[q >> 2][q & 3];
        }
        return;
    }
    uint32_t u[2 * Q];
#pragma unroll
    for (int q = 0; q < 2 * Q; ++q) {
        const float a = v[q >> 1][2 * (q & 1)], b = v[q >> 1][2 * (q & 1) + 1];
        u[q] = g.out_dtype == LUTMOE_DTYPE_F16 ? f32_to_f16(a) | f32_to_f16(b) << 16 : f32x2_to_bf16x2(a, b);
    }
    uint16_t* p = (uint16_t*)g.out + o;
    if (g.out_vec) {
        if constexpr (Q == 1) {
            *(u32x2_t*)p = u32x2_t{u[0], u[1]};
        } else {
#pragma unroll
            for (int q = 0; q < Q / 2; ++q)
                if (c + 8 * q < C) *(u32x4_t*)(p + 8 * q) = u32x4_t{u[4 * q], u[4 * q + 1], u[4 * q + 2], u[4 * q + 3]};
        }
    } else {
#pragma unroll
        for (int q = 0; q < 4 * Q; ++q)
            if (c + q < C) p[q] = (uint16_t)(u[q >> 1] >> (16 * (q & 1)));
    }
}

// acc + (columns c) x (rows r): the weights are the MFMA's A operand, so that a lane's results
// are of one row.
template <int kT>
__device__ __forceinline__ f32x4_t mma(u32x4_t c, u32x4_t r, f32x4_t acc, int sc, int sr) {
    if constexpr (kT == kF4) {
        const i32x8_t a = {(int)c[0], (int)c[1], (int)c[2], (int)c[3], 0, 0, 0, 0};
        const i32x8_t b = {(int)r[0], (int)r[1], (int)r[2], (int)r[3], 0, 0, 0, 0};
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, 0, sc, 0, sr);
    } else if constexpr (kT == kHF) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, c), __builtin_bit_cast(f16x8_t, r), acc, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, c), __builtin_bit_cast(bf16x8_t, r), acc, 0, 0, 0);
    }
}

// Eight MXFP4 codes and their scale byte -> bf16 (exact).
__device__ __forceinline__ u32x4_t widen(uint32_t codes, uint32_t byte) {
    const float s = __uint_as_float(byte == 255u ? 0x7fc00000u : byte << 23);
    return u32x4_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 0)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 1)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 2)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 3))};
}

// LDS DMA: 16 (4) bytes a lane from sbase + voff to m0 + 16 (4) x lane.  The loads are written in
// asm, so they carry the 5 wait states themselves that a vector instruction's write of their scalar operands
// needs (the compiler reloads those from vector registers where it runs short).
__device__ __forceinline__ void lds_dma16(uint32_t voff, const void* sbase, uint32_t m0) {
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(voff), "s"(sbase), "{m0}"(m0) : "memory");
}
__device__ __forceinline__ void lds_dma4(uint32_t voff, const void* sbase, uint32_t m0) {
    asm volatile("s_nop 4\n\tglobal_load_lds_dword %0, %1" : : "v"(voff), "s"(sbase), "{m0}"(m0) : "memory");
}
// The same from a buffer, at voff + soff; at and beyond its end (descriptor: the bytes from `base`
// on): zeros.
__device__ __forceinline__ u32x4_t lds_source(const uint8_t* base, uint32_t bytes) {
    const uint64_t a = (uint64_t)(uintptr_t)base;
    u32x4_t d = {(uint32_t)__builtin_amdgcn_readfirstlane((int)a), (uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32)) & 0xffffu,
                 (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), (uint32_t)kBufWord3};
    asm volatile("" : "+s"(d));   // (not in vector registers)
    return d;
}
__device__ __forceinline__ void lds_dma16(uint32_t voff, const u32x4_t& src, uint32_t soff, uint32_t m0) {
    asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" : : "v"(voff), "s"(src), "s"(soff), "{m0}"(m0) : "memory");
}
__device__ __forceinline__ void lds_dma4(uint32_t voff, const u32x4_t& src, uint32_t soff, uint32_t m0) {
    asm volatile("s_nop 4\n\tbuffer_load_dword %0, %1, %2 offen lds" : : "v"(voff), "s"(src), "s"(soff), "{m0}"(m0) : "memory");
}
// At most kAfter of the wave's loads still in flight, then barrier.  Every wave has waited for
// the LDS reads of what it multiplied before.
template <int kAfter>
__device__ __forceinline__ void loads_barrier() {
    static_assert(kAfter >= 0 && kAfter <= 63, "vmcnt range");
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(kAfter) : "memory");
}

// A 16-byte LDS read of a wave is served 16 lanes at a time, but not in lane order: of lanes
// 0 .. 31 first 0 - 3, 12 - 15 and 20 - 27, then the others (32 .. 63 alike).  Where lane (i, q) =
// (l % 16, l / 16) reads row i, that is every i once, with two neighbouring q; a row's swizzle
// is made of this.
__device__ __forceinline__ int quad_order(int i) { return (-(i >> 2)) & 3; }

// Four bytes of each of four rows' words -> one byte of each: lane group f holds the word of row f,
// group q gets byte q of the words 0 .. 3 (`pick`: 0x0c0c0000 | (4 + q) << 8 | q).
__device__ __forceinline__ uint32_t bytes4(uint32_t v, uint32_t pick) {
    const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);          // words 0 1 0 1, 2 3 2 3
    const auto a = __builtin_amdgcn_permlane16_swap(h[0], h[0], false, false);    // 0 everywhere, 1
    const auto b = __builtin_amdgcn_permlane16_swap(h[1], h[1], false, false);    // 2, 3
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[1], b[0], pick), __builtin_amdgcn_perm(a[1], a[0], pick), 0x05040100u);
}

typedef __attribute__((address_space(3))) const u32x4_t* lds_quad_t;
typedef __attribute__((address_space(3))) const uint8_t* lds_byte_t;
__device__ __forceinline__ u32x4_t lds_quad(uint32_t a) { return *(lds_quad_t)a; }

}  // namespace lutmoe
