// MXFP4: blocks of 32 values along a row, one power-of-two scale a block (E8M0 byte b:
// 2^(b - 127), 255: NaN) and 4-bit E2M1 elements (0, .5, 1, 1.5, 2, 3, 4, 6 and their
// negatives; two a byte, the even element in the low four bits).
//
//   encode  e = floor(log2(max |x|)) - 2 (the largest element lands in [4, 8)), byte =
//           max(e + 127, 0), code = x / 2^e to the nearest element, ties to the even code,
//           past 6 to 6.  A block with an infinity or NaN: byte 255, codes 0.
//   dequant bf16 values (a product of an E2M1 element and a power of two has two
//           significant bits: exact in bf16 wherever it is in range).
//
// Both are bound by memory: 16 bytes of 16-bit values a lane are loaded at once, the four
// lanes of a block meet in two cross-lane maxima, and the conversions are the hardware's
// (v_cvt_scalef32_*, round to nearest even, a scale of which it takes the exponent byte
// alone, so that byte 0 is 2^-127 there too).
#include "common.h"
#include "kernels.h"

using namespace lutmoe;

namespace {

typedef __attribute__((__vector_size__(2 * sizeof(_Float16)))) _Float16 f16x2_t;

// (By value: a bit cast of a vector's element itself takes the vector's first bytes.)
template <class V>
__device__ __forceinline__ V pair_of(uint32_t u) {
    return __builtin_bit_cast(V, u);
}

// The float whose exponent byte is the scale's (255: a NaN).
__device__ __forceinline__ float scale_f32(uint32_t byte) {
    return __uint_as_float(byte == 255u ? 0x7fc00000u : byte << 23);
}

// Eight values of one row, 16 or 32 bytes.
template <int kType>
struct Values {
    u32x4_t v[kType == LUTMOE_DTYPE_F32 ? 2 : 1];
    __device__ __forceinline__ void load(const void* x, int64_t i) {
        const u32x4_t* p = (const u32x4_t*)((const uint8_t*)x + i * (kType == LUTMOE_DTYPE_F32 ? 32 : 16));
        v[0] = p[0];
        if constexpr (kType == LUTMOE_DTYPE_F32) v[1] = p[1];
    }
    // the largest magnitude's fp32 bits (NaN and infinity at or above 0x7f800000)
    __device__ __forceinline__ uint32_t amax() const {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (kType == LUTMOE_DTYPE_F32) {
                m = max(m, max(v[0][j] & 0x7fffffffu, v[1][j] & 0x7fffffffu));
            } else if constexpr (kType == LUTMOE_DTYPE_BF16) {
                m = max(m, max((v[0][j] << 16) & 0x7fff0000u, v[0][j] & 0x7fff0000u));
            } else {   // (the 16-bit patterns order as the values do)
                m = max(m, max(v[0][j] & 0x7fffu, (v[0][j] >> 16) & 0x7fffu));
            }
        }
        if constexpr (kType == LUTMOE_DTYPE_F16) m = __float_as_uint(f16_to_f32(m));
        return m;
    }
    __device__ __forceinline__ uint32_t codes(float scale) const {
        uint32_t c = 0;
        if constexpr (kType == LUTMOE_DTYPE_F32) {
            const float* f0 = (const float*)&v[0];
            const float* f1 = (const float*)&v[1];
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f0[0], f0[1], scale, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f0[2], f0[3], scale, 1);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f1[0], f1[1], scale, 2);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f1[2], f1[3], scale, 3);
        } else if constexpr (kType == LUTMOE_DTYPE_BF16) {
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, pair_of<bf16x2_t>(v[0][0]), scale, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, pair_of<bf16x2_t>(v[0][1]), scale, 1);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, pair_of<bf16x2_t>(v[0][2]), scale, 2);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, pair_of<bf16x2_t>(v[0][3]), scale, 3);
        } else {
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, pair_of<f16x2_t>(v[0][0]), scale, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, pair_of<f16x2_t>(v[0][1]), scale, 1);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, pair_of<f16x2_t>(v[0][2]), scale, 2);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, pair_of<f16x2_t>(v[0][3]), scale, 3);
        }
        return c;
    }
};

// n8: groups of eight values, four a block.
template <int kType>
__global__ __launch_bounds__(256) void encode_kernel(const void* __restrict__ x, int64_t n8,
                                                     uint32_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n8) return;   // (whole blocks: the four lanes of one stay together)
    Values<kType> v;
    v.load(x, i);
    uint32_t m = v.amax();
    m = max(m, (uint32_t)__shfl_xor((int)m, 1, kWave));
    m = max(m, (uint32_t)__shfl_xor((int)m, 2, kWave));
    const uint32_t field = m >> 23;
    const bool bad = field == 255u;
    const uint32_t byte = bad ? 255u : field > 2u ? field - 2u : 0u;
    const uint32_t c = v.codes(__uint_as_float(bad ? 0x3f800000u : byte << 23));
    codes[i] = bad ? 0u : c;
    if ((threadIdx.x & 3) == 0) scales[i >> 2] = (uint8_t)byte;
}

__global__ __launch_bounds__(256) void dequant_kernel(const uint32_t* __restrict__ codes,
                                                      const uint8_t* __restrict__ scales, int64_t n8,
                                                      u32x4_t* __restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n8) return;
    const uint32_t c = codes[i];
    const float s = scale_f32(scales[i >> 2]);
    out[i] = u32x4_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3))};
}

}  // namespace

namespace lutmoe_host {

int launch_mxfp4_encode(const void* x, int dtype, int64_t nblocks, uint8_t* codes, uint8_t* scales, hipStream_t s) {
    const int64_t n8 = nblocks * 4;
    const dim3 grid((uint32_t)((n8 + 255) / 256)), block(256);
    switch (dtype) {
        case LUTMOE_DTYPE_F32: hipLaunchKernelGGL((encode_kernel<LUTMOE_DTYPE_F32>), grid, block, 0, s, x, n8, (uint32_t*)codes, scales); break;
        case LUTMOE_DTYPE_F16: hipLaunchKernelGGL((encode_kernel<LUTMOE_DTYPE_F16>), grid, block, 0, s, x, n8, (uint32_t*)codes, scales); break;
        default: hipLaunchKernelGGL((encode_kernel<LUTMOE_DTYPE_BF16>), grid, block, 0, s, x, n8, (uint32_t*)codes, scales); break;
    }
    return check_launch();
}

int launch_mxfp4_dequant(uint16_t* out, const uint8_t* codes, const uint8_t* scales, int64_t nblocks, hipStream_t s) {
    const int64_t n8 = nblocks * 4;
    hipLaunchKernelGGL(dequant_kernel, dim3((uint32_t)((n8 + 255) / 256)), dim3(256), 0, s, (const uint32_t*)codes, scales,
                       n8, (u32x4_t*)out);
    return check_launch();
}

}  // namespace lutmoe_host
