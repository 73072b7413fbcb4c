// Sixteen bytes of a row as f32 values, for kernels whose rows may begin at any element.
#pragma once
#include "gemm_common.h"

namespace sp {

template <int DT>
constexpr int ELEM_BYTES = DT == SP_F32 ? 4 : 2;
template <int DT>
constexpr int PER16 = 16 / ELEM_BYTES<DT>;     // elements of one 16-byte access

// The bits of PER16 elements from element `at` on; where only `left` of them exist, those one by one and zeros behind them.
template <int DT>
__device__ __forceinline__ u32x4 load_each(const void* p, long at, long left) {
    constexpr int E = ELEM_BYTES<DT>;
    const unsigned char* q = (const unsigned char*)p + at * E;
    if (left >= PER16<DT>) return load_aligned<E, u32x4>(q);
    u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < PER16<DT> - 1; ++i)
        if (i < left) {
            if constexpr (E == 4) v[i] = ((const unsigned*)q)[i];
            else v[i >> 1] |= (unsigned)((const unsigned short*)q)[i] << (16 * (i & 1));
        }
    return v;
}

// The same, for tensors p whose elements in front of `at` may be read as well.
template <int DT>
__device__ __forceinline__ u32x4 load16(const void* p, long at, long left) {
    constexpr int E = ELEM_BYTES<DT>, N = PER16<DT>;
    const unsigned char* q = (const unsigned char*)p + at * E;
    if (left >= N) return load_aligned<E, u32x4>(q);
    u32x4 v = {0u, 0u, 0u, 0u};
    if (left <= 0) return v;
    if (at + left < N) return load_each<DT>(p, at, left);
    // the 16 bytes that end with them, moved down: one load, where one by one would wait N - 1 times (378 x 235 bf16 in 8-bit blocks both ways 9.4 us, 8.2)
    const int up = N - (int)left, words = E == 4 ? up : up >> 1;
    v = load_aligned<E, u32x4>(q - up * E);
    if (words & 2) v = u32x4{v[2], v[3], 0u, 0u};
    if (words & 1) v = u32x4{v[1], v[2], v[3], 0u};
    if (E == 2 && (up & 1) != 0) v = u32x4{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
    return v;
}

template <int DT>
__device__ __forceinline__ float element(const u32x4& v, int i) {
    if constexpr (DT == SP_F32) return __uint_as_float(v[i]);
    else return half_bits_to_f32<DT>(i & 1 ? v[i >> 1] >> 16 : v[i >> 1] & 0xffffu);
}

template <int DT, int POLICY = ST_PLAIN>
__device__ __forceinline__ void store16(void* p, long at, long left, const float (&v)[PER16<DT>]) {
    constexpr int E = ELEM_BYTES<DT>, N = PER16<DT>;
    unsigned char* q = (unsigned char*)p + at * E;
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (E == 4) o[i] = __float_as_uint(v[i]);
        else o[i] = pack_halves<DT>(v[2 * i], v[2 * i + 1]);
    }
    if (left >= N) {
        store_c<POLICY, E>(q, o);
        return;
    }
#pragma unroll
    for (int i = 0; i < N - 1; ++i)
        if (i < left) {
            if constexpr (E == 4) ((unsigned*)q)[i] = o[i];
            else ((unsigned short*)q)[i] = (unsigned short)(o[i >> 1] >> (16 * (i & 1)));
        }
}

}  // namespace sp
