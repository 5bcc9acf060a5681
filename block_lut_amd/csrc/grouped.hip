// Products of rows sorted by expert: group e = rows [off[e], off[e + 1]) of x, and matrix
// e of a stack.
//   forward  y[p] = x[p] . W[e]^T              sum over the K columns
//   dgrad    dx[p] = dy[p] . W[e]              sum over the M rows of W[e]
//   wgrad    dW[e] = sum over the group's rows p of dy[p]^T x[p]
// W bf16 or fp16, or (forward) MXFP4 with bf16 or MXFP4 rows.  fp32 accumulation on MFMA
// (16 x 16 x 32), one rounding of the result.
//
// All three are C[r][c] = sum_k A(r, k) B(c, k): r positions (wgrad: rows of W), c outputs.
// A CTA computes 64 x 64 of C; the operands go through LDS by single elements, any layout
// into k-contiguous rows.
#include "common.h"
#include "kernels.h"

using namespace lutmoe;
using lutmoe_host::GroupedArgs;

namespace {

typedef __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16 f16x8_t;

constexpr int kB = 64, kBK = 32, kPad = 8;

__device__ __forceinline__ uint32_t e2m1_bf16(uint32_t code, uint32_t byte) {
    const float s = __uint_as_float(byte == 255u ? 0x7fc00000u : byte << 23);
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, s, 0)) & 0xffffu;
}

// Element (row, col) of a row-major matrix of `cols` columns, as 16 bits.
template <bool kFp4>
__device__ __forceinline__ uint32_t element(const void* p, const void* scales, int64_t row, int col, int cols) {
    const int64_t i = row * cols + col;
    if constexpr (kFp4) {
        const uint32_t b = ((const uint8_t*)p)[i >> 1];
        return e2m1_bf16((b >> (4 * (col & 1))) & 15u, ((const uint8_t*)scales)[i >> 5]);
    } else {
        return ((const uint16_t*)p)[i];
    }
}

// Group e's rows, clamped into [0, P] (the first starts at row 0); e = E: the rows behind.
__device__ __forceinline__ void group_rows(const int32_t* off, int E, int P, int e, int& p0, int& n) {
    const int a = e == 0 || !off ? 0 : min(max(off[e], 0), P);
    const int b = e == E || !off ? P : min(max(off[e + 1], 0), P);
    p0 = a;
    n = max(b - a, 0);
}

template <int kOp, bool kF16, bool kXFp4, bool kWFp4>
__global__ __launch_bounds__(256) void simple_kernel(GroupedArgs g) {
    __shared__ __attribute__((aligned(16))) uint16_t s_r[kB][kBK + kPad], s_c[kB][kBK + kPad];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int C = kOp == kGroupedFwd ? g.M : g.K;
    int e, p0 = 0, n = 0, r0 = 0;
    if constexpr (kOp == kGroupedWgrad) {
        e = blockIdx.z;
        group_rows(g.offsets, g.E, g.P, e, p0, n);
        r0 = blockIdx.x * kB;
    } else {
        int t = blockIdx.x;
        for (e = 0;; ++e) {
            if (e > g.E - (g.zero_rest ? 0 : 1)) return;
            group_rows(g.offsets, g.E, g.P, e, p0, n);
            const int tiles = (n + kB - 1) / kB;
            if (t < tiles) break;
            t -= tiles;
        }
        r0 = t * kB;
    }
    const bool rest = e == g.E;   // rows of no group: zeros
    const int c0 = blockIdx.y * kB;
    const int R = kOp == kGroupedWgrad ? g.M : n, Kt = rest ? 0 : kOp == kGroupedFwd ? g.K : kOp == kGroupedDgrad ? g.M : n;
    const int64_t wrow = (int64_t)e * g.M;
    f32x4_t acc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < Kt; k0 += kBK) {
        __syncthreads();
        for (int i = tid; i < kB * kBK; i += 256) {
            const int kk = kOp == kGroupedFwd ? i % kBK : i / kB, q = kOp == kGroupedFwd ? i / kBK : i % kB;
            const int k = k0 + kk;
            uint32_t a = 0, b = 0;
            if (k < Kt && r0 + q < R) {
                if constexpr (kOp == kGroupedFwd) a = element<kXFp4>(g.x, g.x_scales, p0 + r0 + q, k, g.K);
                else if constexpr (kOp == kGroupedDgrad) a = element<false>(g.x, nullptr, p0 + r0 + q, k, g.M);
                else a = element<false>(g.x, nullptr, p0 + k, r0 + q, g.M);
            }
            if (k < Kt && c0 + q < C) {
                if constexpr (kOp == kGroupedFwd) b = element<kWFp4>(g.w, g.w_scales, wrow + c0 + q, k, g.K);
                else if constexpr (kOp == kGroupedDgrad) b = element<false>(g.w, nullptr, wrow + k, c0 + q, g.K);
                else b = element<false>(g.w, nullptr, p0 + k, c0 + q, g.K);
            }
            s_r[q][kk] = (uint16_t)a;
            s_c[q][kk] = (uint16_t)b;
        }
        __syncthreads();
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const u32x4_t a = *(const u32x4_t*)&s_r[16 * wv + (lane & 15)][8 * (lane >> 4)];
            const u32x4_t b = *(const u32x4_t*)&s_c[16 * f + (lane & 15)][8 * (lane >> 4)];
            if constexpr (kF16)
                acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), acc[f], 0, 0, 0);
            else
                acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), acc[f], 0, 0, 0);
        }
    }
    const int64_t out0 = kOp == kGroupedWgrad ? wrow : p0;
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + 16 * wv + 4 * (lane >> 4) + i, c = c0 + 16 * f + (lane & 15);
            if (r >= R || c >= C) continue;
            const int64_t o = (out0 + r) * C + c;
            const float v = acc[f][i];
            if (g.out_dtype == LUTMOE_DTYPE_F32) ((float*)g.out)[o] = v;
            else ((uint16_t*)g.out)[o] = (uint16_t)(g.out_dtype == LUTMOE_DTYPE_F16 ? f32_to_f16(v) : f32_to_bf16(v));
        }
}

}  // namespace

namespace lutmoe_host {

int launch_grouped(const GroupedArgs& g, hipStream_t s) {
    if (!g.w_scales || g.x_scales) return launch_grouped_tile(g, s);
    const int C = g.op == kGroupedFwd ? g.M : g.K;
    const int64_t rows = g.op == kGroupedWgrad ? (g.M + kB - 1) / kB : g.P / kB + (g.P < g.E + 1 ? g.P : g.E + 1);
    const dim3 grid((uint32_t)rows, (C + kB - 1) / kB, g.op == kGroupedWgrad ? g.E : 1), block(256);
    const bool f16 = g.x_dtype == LUTMOE_DTYPE_F16;
#define LUTMOE_GROUPED(OP, F16, X4, W4) hipLaunchKernelGGL((simple_kernel<OP, F16, X4, W4>), grid, block, 0, s, g)
    if (g.op == kGroupedFwd) {
        if (g.w_scales) {
            if (g.x_scales) LUTMOE_GROUPED(kGroupedFwd, false, true, true);
            else LUTMOE_GROUPED(kGroupedFwd, false, false, true);
        } else if (f16) LUTMOE_GROUPED(kGroupedFwd, true, false, false);
        else LUTMOE_GROUPED(kGroupedFwd, false, false, false);
    } else if (g.op == kGroupedDgrad) {
        if (f16) LUTMOE_GROUPED(kGroupedDgrad, true, false, false);
        else LUTMOE_GROUPED(kGroupedDgrad, false, false, false);
    } else {
        if (f16) LUTMOE_GROUPED(kGroupedWgrad, true, false, false);
        else LUTMOE_GROUPED(kGroupedWgrad, false, false, false);
    }
#undef LUTMOE_GROUPED
    return check_launch();
}

}  // namespace lutmoe_host
