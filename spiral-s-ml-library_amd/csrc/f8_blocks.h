// Eight-bit numbers in blocks that share an f32 scale: what the kernels that write and read them have in common.
#pragma once
#include "vec_io.h"

namespace sp {

constexpr int QB = 128;                       // elements of a block
constexpr float SCALE_LEAST = 0x1p-126f;      // the smallest normal f32: 1 / scale stays finite, and a block of zeros has a scale

template <int F8>
constexpr float F8_MOST = F8 == SP_F8_E4M3 ? 448.f : 57344.f;

// Four numbers as four bytes.
template <int F8>
__device__ __forceinline__ unsigned pack_f8(float a, float b, float c, float d) {
    int v = 0;
    if constexpr (F8 == SP_F8_E4M3) {
        v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, v, false);
        v = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
    } else {
        v = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, v, false);
        v = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, v, true);
    }
    return (unsigned)v;
}

// The first `left` of four bytes, and zeros: what lies behind a row is zeros whatever its block's scale is (0 / inf and 0 / NaN are NaNs).
__device__ __forceinline__ unsigned first_bytes(unsigned v, long left) { return left >= 4 ? v : left <= 0 ? 0u : v & ((1u << (8 * (int)left)) - 1u); }

struct BlockScale {
    float scale, inv;
    template <int F8>
    __device__ __forceinline__ void set(unsigned magnitude) {
        scale = __uint_as_float(magnitude) / F8_MOST<F8>;
        scale = scale < SCALE_LEAST ? SCALE_LEAST : scale;               // (a NaN stays)
        inv = 1.f / scale;
    }
    __device__ __forceinline__ float operator()(float x) const {
        const float q = x * inv;
        return __builtin_fmaf(__builtin_fmaf(-q, scale, x), inv, q);
    }
};

__device__ __forceinline__ unsigned max_u32(unsigned a, unsigned b) { return a > b ? a : b; }

}  // namespace sp
