// C = A . B^T of 8-bit operands with a scale for each block of 128 along K: per row of A, per row of B or per 128 of its rows.
//
// A block of 128 is 128 bytes of a row: one MFMA of K = 128, or four of K = 32, which start from zero.  The vector ALU multiplies their sum by
// the block's two scales and adds it to the accumulators (so the sum over the blocks is rounded to nearest f32): four multiply-adds
// of 4 cycles per 16 x 16 block, against 32 or 64 cycles on the matrix pipe.
//
// The B fragment is the MFMA's first operand: register r of lane l of a 16 x 16 fragment holds C[m = l % 16][n = 4 (l / 16) + r], so a lane
// needs one scale of A per fragment and stores four consecutive columns.
//
// Two kernels.  gemm_scaled_tile_kernel: workgroup tiles in LDS, for outputs that fill the chip.  gemm_scaled_split_kernel: few rows, or
// few tiles; the waves of a workgroup share one small tile, take the blocks of K in turn straight from global memory, and add up in LDS, in a fixed order.
#include "gemm_common.h"

namespace sp {

typedef int i32x8 __attribute__((ext_vector_type(8)));

struct ScaledArgs {
    const unsigned char *A, *B;
    const float *scale_a, *scale_b;
    void* C;
    const float* bias;
    long M, N, K;
    long blocks;                  // of K
    float beta;
    int relu, out_dtype;
    int tiles_m, tiles_n, group_m;
};

// A lane's 32 numbers of a block of one row.  A and B agree on which 16-byte chunks of the block they are; in which order does not matter.
template <int F8, bool FAST>
struct Fragment;

template <int F8>
struct Fragment<F8, true> {
    i32x8 v;
    __device__ __forceinline__ void set(const u32x4 (&c)[2]) {
        struct Pair { u32x4 v[2]; };
        v = __builtin_bit_cast(i32x8, Pair{{c[0], c[1]}});
    }
};

// As f16, which holds every number of both types.
template <int F8>
struct Fragment<F8, false> {
    f16x8 v[4];
    __device__ __forceinline__ void set(const u32x4 (&c)[2]) {
#pragma unroll
        for (int h = 0; h < 8; ++h) {
            const unsigned four = c[h >> 2][h & 3];
            f16x2 lo, hi;
            if constexpr (F8 == SP_F8_E4M3) {
                lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(four, 1.f, false);
                hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(four, 1.f, true);
            } else {
                lo = __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(four, 1.f, false);
                hi = __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(four, 1.f, true);
            }
            const int at = 4 * (h & 1);
            v[h >> 1][at] = lo[0], v[h >> 1][at + 1] = lo[1], v[h >> 1][at + 2] = hi[0], v[h >> 1][at + 3] = hi[1];
        }
    }
};

// The sum of one block.  The 8-bit MFMAs add eight products at a time and cut off what lies below 2^-13 of the largest's power of two before they go on in f32 (measured:
// 2^16 + 8 is exact, 2^16 + 4 is 2^16 with both in one group of eight, and exact otherwise; sums of 4096 N(0, 1) products are 1.5e-5 off in the 2-norm).  FAST
// takes them, for C of 16 bits, whose own rounding is 1.7e-3 (bf16) or 2.1e-4 (f16).  C of f32 takes the f16 MFMAs, at half their rate,
// where products are exact and sums f32.
template <int F8A, int F8B, bool FAST>
__device__ __forceinline__ f32x4 block_sum(const Fragment<F8B, FAST>& b, const Fragment<F8A, FAST>& a) {
    f32x4 t = {0.f, 0.f, 0.f, 0.f};
    if constexpr (FAST) {
        constexpr int FA = F8A == SP_F8_E4M3 ? 0 : 1, FB = F8B == SP_F8_E4M3 ? 0 : 1;
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.v, a.v, t, FB, FA, 0, 0, 0, 0);
    } else {
#pragma unroll
        for (int h = 0; h < 4; ++h) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(b.v[h], a.v[h], t, 0, 0, 0);
        return t;
    }
}

// Four columns of a row of C from col on.
__device__ __forceinline__ void put_quad(const ScaledArgs& g, long row, long col, f32x4 v) {
    if (row >= g.M || col >= g.N) return;
    const long idx = row * g.N + col;
    if (col + 3 < g.N) {
        f32x4 old = {0.f, 0.f, 0.f, 0.f}, bias = old;
        if (g.beta != 0.f) {
            if (g.out_dtype == SP_F32) {
                old = *reinterpret_cast<const f32x4_unaligned*>((const float*)g.C + idx);
            } else {
                const u32x2 o = *reinterpret_cast<const u32x2_unaligned*>((const unsigned short*)g.C + idx);
                const unsigned h[4] = {o.x & 0xffffu, o.x >> 16, o.y & 0xffffu, o.y >> 16};
#pragma unroll
                for (int e = 0; e < 4; ++e) old[e] = g.out_dtype == SP_BF16 ? half_bits_to_f32<SP_BF16>(h[e]) : half_bits_to_f32<SP_F16>(h[e]);
            }
        }
        if (g.bias) bias = *reinterpret_cast<const f32x4_unaligned*>(g.bias + col);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (g.beta != 0.f) v[e] += g.beta * old[e];
            v[e] += bias[e];
            if (g.relu) v[e] = fmaxf(v[e], 0.f);
        }
        if (g.out_dtype == SP_F32) {
            *reinterpret_cast<f32x4_unaligned*>((float*)g.C + idx) = v;
        } else {
            u32x2 o;
            o.x = g.out_dtype == SP_BF16 ? pack_halves<SP_BF16>(v[0], v[1]) : pack_halves<SP_F16>(v[0], v[1]);
            o.y = g.out_dtype == SP_BF16 ? pack_halves<SP_BF16>(v[2], v[3]) : pack_halves<SP_F16>(v[2], v[3]);
            *reinterpret_cast<u32x2_unaligned*>((unsigned short*)g.C + idx) = o;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (col + e < g.N) store_element((unsigned char*)g.C, g.out_dtype, idx + e, v[e], g.beta, g.bias ? g.bias[col + e] : 0.f, g.relu);
    }
}

__device__ __forceinline__ void scaled_tile_of_block(int pid, int tiles_m, int tiles_n, int group_m, int& tm, int& tn) {
    // workgroups are dealt round-robin to the 8 XCDs: each gets a contiguous range of a walk in groups of group_m tile rows
    const int n = tiles_m * tiles_n, xcd = pid & 7, base = n >> 3, rem = n & 7;
    const int t = xcd * base + (xcd < rem ? xcd : rem) + (pid >> 3);
    const int group_size = group_m * tiles_n, g = t / group_size, first = g * group_m;
    const int rows = tiles_m - first < group_m ? tiles_m - first : group_m, in = t - g * group_size;
    tm = first + in % rows;
    tn = in / rows;
}

// 64 scales, four bytes a lane, like dma_to_lds.
__device__ __forceinline__ void dma4_to_lds(const unsigned char* base, unsigned lane_offset, unsigned lds_addr) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" : : "v"(lane_offset), "s"(base), "s"(lds_addr) : "memory", "m0");
}

// Tiles of BM x BN on WM x WN waves, two stages of LDS: tile kt + 1 comes in while tile kt is multiplied.  SHIFT: 7 where a scale of B
// holds for 128 rows, else 0.
template <int F8A, int F8B, bool FAST, int SHIFT, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM* WN * 64) void gemm_scaled_tile_kernel(const ScaledArgs g) {
    constexpr int NW = WM * WN, WTM = BM / WM, WTN = BN / WN, TM = WTM / 16, TN = WTN / 16;
    constexpr int NIA = BM / 8 / NW, NI = (BM + BN) / 8 / NW;       // DMA instructions of 8 rows per wave and K-tile; A's first
    constexpr int SCALES = (BM + BN) / 64;                          // and of 64 scales per workgroup
    static_assert(SCALES == NW, "one instruction of scales per wave");
    constexpr int TILE_BYTES = (BM + BN) * ROW_BYTES, STAGE = TILE_BYTES + (BM + BN) * 4;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN, fi = lane & 15, fq = lane >> 4;
    int tm, tn;
    scaled_tile_of_block(blockIdx.x, g.tiles_m, g.tiles_n, g.group_m, tm, tn);
    const long m0 = (long)tm * BM, n0 = (long)tn * BN;
    const int nk = (int)g.blocks;
    const bool k_tail = (g.K & 127) != 0;

    // operands: rows past the end are the last row again, chunks past the end of a row zeros
    const unsigned char* pA = uniform_ptr(g.A + m0 * g.K);
    const unsigned char* pB = uniform_ptr(g.B + n0 * g.K);
    const unsigned lds_base = (unsigned)(size_t)lds;
    unsigned voff[NI], dst[NI], tail_in = 0;
#pragma unroll
    for (int q = 0; q < NI; ++q) {
        const bool is_a = q < NIA;
        const int blk = (is_a ? q : q - NIA) * NW + wave, r = lane >> 3, kc = (lane & 7) ^ ((r ^ blk) & 7);
        const long left = (is_a ? g.M - m0 : g.N - n0) - 1, row = blk * 8 + r < left ? blk * 8 + r : left;
        voff[q] = (unsigned)(row * g.K) + kc * 16;
        if ((long)(nk - 1) * ROW_BYTES + kc * 16 < g.K) tail_in |= 1u << q;
        dst[q] = __builtin_amdgcn_readfirstlane(lds_base + ((is_a ? 0 : BM) + blk * 8) * ROW_BYTES);
    }
    // scales: position p of A's is row 16 (p % TM) + p / TM of a wave's rows, so that a lane reads its TM side by side
    const bool scales_of_a = wave < BM / 64;
    const int pos = (scales_of_a ? wave : wave - BM / 64) * 64 + lane;
    const long left = (scales_of_a ? g.M - m0 : g.N - n0) - 1;
    long srow = scales_of_a ? (long)(pos / WTM) * WTM + 16 * (pos % TM) + pos % WTM / TM : (long)pos;
    srow = srow < left ? srow : left;
    const unsigned char* pS;
    unsigned soff;
    if (scales_of_a) {
        pS = uniform_ptr((const unsigned char*)(g.scale_a + m0 * g.blocks));
        soff = (unsigned)(srow * g.blocks * 4);
    } else {
        pS = uniform_ptr((const unsigned char*)(g.scale_b + (n0 >> SHIFT) * g.blocks));
        soff = (unsigned)((((n0 + srow) >> SHIFT) - (n0 >> SHIFT)) * g.blocks * 4);
    }
    const unsigned sdst = __builtin_amdgcn_readfirstlane(lds_base + TILE_BYTES + wave * 256);
    auto fetch = [&](int kt) {
        const unsigned stage = (kt & 1) * STAGE;
        const unsigned char *a = pA + (long)kt * ROW_BYTES, *b = pB + (long)kt * ROW_BYTES;
        if (k_tail && kt == nk - 1) {
#pragma unroll
            for (int q = 0; q < NI; ++q) {
                const unsigned char* inside = (q < NIA ? a : b) + voff[q];
                dma_to_lds_addr((tail_in >> q) & 1u ? inside : (const unsigned char*)kZeroChunk, dst[q] + stage);
            }
        } else {
#pragma unroll
            for (int q = 0; q < NI; ++q) dma_to_lds(q < NIA ? a : b, voff[q], dst[q] + stage);
        }
        dma4_to_lds(pS + (long)kt * 4, soff, sdst + stage);
    };

    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    fetch(0);
    for (int kt = 0; kt < nk; ++kt) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();                       // tile kt is there, and everybody has read tile kt - 1
        if (kt + 1 < nk) fetch(kt + 1);
        const unsigned char* at = lds + (kt & 1) * STAGE;
        const float* scales = reinterpret_cast<const float*>(at + TILE_BYTES);
        auto fragment = [&](auto& f, int row) {
            u32x4 c[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) c[h] = *reinterpret_cast<const u32x4*>(at + lds_offset(row, 2 * fq + h));
            f.set(c);
        };
        Fragment<F8B, FAST> b[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) fragment(b[j], BM + wn * WTN + 16 * j + fi);
        float sa[TM];
#pragma unroll
        for (int i = 0; i < TM; ++i) sa[i] = scales[wm * WTM + fi * TM + i];
        f32x4 sb[TN];
        if constexpr (SHIFT == 7) {
            const float s = scales[BM + wn * WTN];
#pragma unroll
            for (int i = 0; i < TM; ++i) sa[i] *= s;
        } else {
#pragma unroll
            for (int j = 0; j < TN; ++j) sb[j] = *reinterpret_cast<const f32x4*>(scales + BM + wn * WTN + 16 * j + 4 * fq);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            Fragment<F8A, FAST> a;
            fragment(a, wm * WTM + 16 * i + fi);
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const f32x4 t = block_sum<F8A, F8B, FAST>(b[j], a);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(t[e], SHIFT == 7 ? sa[i] : sa[i] * sb[j][e], acc[i][j][e]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) put_quad(g, m0 + wm * WTM + 16 * i + fi, n0 + wn * WTN + 16 * j + 4 * fq, acc[i][j]);
}

// One tile of (16 TM) x (16 TN) on KS waves; wave w takes blocks w, w + KS, ... of K, U of them at a time under way.
template <int F8A, int F8B, bool FAST, int SHIFT, int TM, int TN, int KS, int U>
__global__ __launch_bounds__(KS * 64) void gemm_scaled_split_kernel(const ScaledArgs g) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fi = lane & 15, fq = lane >> 4;
    int tm, tn;
    scaled_tile_of_block(blockIdx.x, g.tiles_m, g.tiles_n, g.group_m, tm, tn);
    const long m0 = (long)tm * (16 * TM), n0 = (long)tn * (16 * TN);
    const unsigned char *rowA[TM], *rowB[TN];
    const float *rowSA[TM], *rowSB[TN][SHIFT == 7 ? 1 : 4];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const long row = m0 + 16 * i + fi < g.M ? m0 + 16 * i + fi : g.M - 1;
        rowA[i] = g.A + row * g.K + fq * 32;
        rowSA[i] = g.scale_a + row * g.blocks;
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const long row = n0 + 16 * j + fi < g.N ? n0 + 16 * j + fi : g.N - 1;
        rowB[j] = g.B + row * g.K + fq * 32;
#pragma unroll
        for (int e = 0; e < (SHIFT == 7 ? 1 : 4); ++e) {
            const long mine = SHIFT == 7 ? n0 + 16 * j : n0 + 16 * j + 4 * fq + e;
            rowSB[j][e] = g.scale_b + ((mine < g.N ? mine : g.N - 1) >> SHIFT) * g.blocks;
        }
    }
    const int nk = (int)g.blocks;
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const u32x4 none = {0u, 0u, 0u, 0u};
    auto blocks = [&](int first, auto WHOLE_) {
        constexpr bool WHOLE = decltype(WHOLE_)::value;         // all U blocks exist and are whole
        u32x4 a[U][TM][2], b[U][TN][2];
        float sa[U][TM], sb[U][TN][SHIFT == 7 ? 1 : 4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kt = first + u * KS;
            const bool in = WHOLE || kt < nk;
            const long k = (long)kt * ROW_BYTES;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bool there = WHOLE || (in && k + fq * 32 + h * 16 < g.K);
#pragma unroll
                for (int j = 0; j < TN; ++j) b[u][j][h] = there ? *reinterpret_cast<const u32x4*>(rowB[j] + k + h * 16) : none;
#pragma unroll
                for (int i = 0; i < TM; ++i) a[u][i][h] = there ? *reinterpret_cast<const u32x4*>(rowA[i] + k + h * 16) : none;
            }
#pragma unroll
            for (int i = 0; i < TM; ++i) sa[u][i] = in ? rowSA[i][kt] : 0.f;
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int e = 0; e < (SHIFT == 7 ? 1 : 4); ++e) sb[u][j][e] = in ? rowSB[j][e][kt] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            Fragment<F8B, FAST> fb[TN];
#pragma unroll
            for (int j = 0; j < TN; ++j) fb[j].set(b[u][j]);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                Fragment<F8A, FAST> fa;
                fa.set(a[u][i]);
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    const f32x4 t = block_sum<F8A, F8B, FAST>(fb[j], fa);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(t[e], sa[u][i] * sb[u][j][SHIFT == 7 ? 0 : e], acc[i][j][e]);
                }
            }
        }
    };
    const int whole = (int)(g.K >> 7);
    int kt = wave;
    for (; kt + (U - 1) * KS < whole; kt += U * KS) blocks(kt, std::true_type{});
    for (; kt < nk; kt += U * KS) blocks(kt, std::false_type{});
    // fragment f of wave w at (f * KS + w) * 1 KiB; fragment f is then finished by wave f % KS
    f32x4* part = reinterpret_cast<f32x4*>(lds);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) part[((i * TN + j) * KS + wave) * 64 + lane] = acc[i][j];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int f = i * TN + j;
            if (f % KS != wave) continue;
            const f32x4* p = part + f * KS * 64 + lane;
            f32x4 s = p[0];
#pragma unroll
            for (int w = 1; w < KS; ++w) s += p[w * 64];
            put_quad(g, m0 + 16 * i + fi, n0 + 16 * j + 4 * fq, s);
        }
}

// ---- host side -------------------------------------------------------------------------------

static int check_tiles(ScaledArgs& g, int bm, int bn, int threads) {
    const long tm = (g.M + bm - 1) / bm, tn = (g.N + bn - 1) / bn;
    if (tm * tn * threads >= 1l << 32 || tm * tn >= 1l << 31) return fail(SP_ERR_SHAPE, "sp_gemm_abt_scaled: too large");
    g.tiles_m = (int)tm;
    g.tiles_n = (int)tn;
    return SP_OK;
}

template <int F8A, int F8B, bool FAST, int SHIFT, int BM, int BN, int WM, int WN>
static int launch_tile(ScaledArgs g, hipStream_t stream) {
    auto kernel = gemm_scaled_tile_kernel<F8A, F8B, FAST, SHIFT, BM, BN, WM, WN>;
    constexpr int lds_bytes = 2 * (BM + BN) * (ROW_BYTES + 4);
    if (const int rc = check_tiles(g, BM, BN, WM * WN * 64); rc != SP_OK) return rc;
    if (const int rc = ensure_dynamic_lds((const void*)kernel, lds_bytes); rc != SP_OK) return rc;
    g.group_m = 4;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(g.tiles_m * g.tiles_n)), dim3(WM * WN * 64), lds_bytes, stream, g);
    return check_launch("sp_gemm_abt_scaled");
}

template <int F8A, int F8B, bool FAST, int SHIFT, int TM, int TN, int KS, int U>
static int launch_split(ScaledArgs g, hipStream_t stream) {
    auto kernel = gemm_scaled_split_kernel<F8A, F8B, FAST, SHIFT, TM, TN, KS, U>;
    constexpr int lds_bytes = KS * TM * TN * 1024;
    if (const int rc = check_tiles(g, 16 * TM, 16 * TN, KS * 64); rc != SP_OK) return rc;
    if (const int rc = ensure_dynamic_lds((const void*)kernel, lds_bytes); rc != SP_OK) return rc;
    g.group_m = g.tiles_m;        // the tiles of one panel of B stand side by side
    hipLaunchKernelGGL(kernel, dim3((unsigned)(g.tiles_m * g.tiles_n)), dim3(KS * 64), lds_bytes, stream, g);
    return check_launch("sp_gemm_abt_scaled");
}

template <int F8A, int F8B, bool FAST, int SHIFT>
static int multiply(const ScaledArgs& g, hipStream_t stream) {
    const long cus = device_cu_count();
    const long tiles128 = ((g.M + 127) / 128) * ((g.N + 127) / 128);
    if (g.M > 64 && tiles128 * 2 > cus) return launch_tile<F8A, F8B, FAST, SHIFT, 128, 128, 2, 2>(g, stream);
    if (g.M <= 16) return launch_split<F8A, F8B, FAST, SHIFT, 1, 1, 8, 4>(g, stream);
    if (g.M <= 32) return launch_split<F8A, F8B, FAST, SHIFT, 2, 2, 8, 2>(g, stream);
    return launch_split<F8A, F8B, FAST, SHIFT, 4, 2, 4, 2>(g, stream);
}

namespace {
struct GemmScaledKernelNames {
    GemmScaledKernelNames() {
        register_kernel("gemm_scaled_128x128", (const void*)gemm_scaled_tile_kernel<SP_F8_E4M3, SP_F8_E4M3, true, 7, 128, 128, 2, 2>, 256);
        register_kernel("gemm_scaled_split_16x16", (const void*)gemm_scaled_split_kernel<SP_F8_E4M3, SP_F8_E4M3, true, 7, 1, 1, 8, 4>, 512);
    }
} gemm_scaled_kernel_names;
}  // namespace

}  // namespace sp

using namespace sp;

extern "C" int sp_gemm_abt_scaled(int f8_a, int f8_b, int dtype_out, const void* A, const float* scale_a, const void* B, const float* scale_b,
                                  int32_t block_n, void* C, const float* bias, int64_t M, int64_t N, int64_t K, float beta, uint32_t flags,
                                  void* stream) {
    SP_REQUIRE_PTR(A);
    SP_REQUIRE_PTR(scale_a);
    SP_REQUIRE_PTR(B);
    SP_REQUIRE_PTR(scale_b);
    SP_REQUIRE_PTR(C);
    SP_OPTIONAL_PTR(bias);
    if ((f8_a != SP_F8_E4M3 && f8_a != SP_F8_E5M2) || (f8_b != SP_F8_E4M3 && f8_b != SP_F8_E5M2))
        return fail(SP_ERR_DTYPE, "sp_gemm_abt_scaled: operands must be e4m3 or e5m2, got %d and %d", f8_a, f8_b);
    if (dtype_out != SP_F32 && dtype_out != SP_F16 && dtype_out != SP_BF16)
        return fail(SP_ERR_DTYPE, "sp_gemm_abt_scaled: C must be f32, f16 or bf16, got %d", dtype_out);
    if (block_n != 1 && block_n != 128) return fail(SP_ERR_ARG, "sp_gemm_abt_scaled: a scale of B holds for 1 or 128 rows, got %d", block_n);
    if (flags & ~SP_GEMM_RELU) return fail(SP_ERR_ARG, "sp_gemm_abt_scaled: unknown flags 0x%x", flags);
    if (M <= 0 || N <= 0 || K <= 0) return fail(SP_ERR_SHAPE, "sp_gemm_abt_scaled: M, N, K must be positive (got %lld, %lld, %lld)", (long long)M, (long long)N, (long long)K);
    if (K % 16 != 0) return fail(SP_ERR_SHAPE, "sp_gemm_abt_scaled: K must be a multiple of 16 (16-byte rows), got %lld", (long long)K);
    // a tile's rows are addressed by 32-bit offsets
    if (K > (int64_t)1 << 23 || M >= (int64_t)1 << 31 || N >= (int64_t)1 << 31) return fail(SP_ERR_SHAPE, "sp_gemm_abt_scaled: too large");
    const int rc = require_gfx950(__func__);
    if (rc != SP_OK) return rc;
    ScaledArgs g{};
    g.A = (const unsigned char*)A; g.B = (const unsigned char*)B; g.scale_a = scale_a; g.scale_b = scale_b; g.C = C; g.bias = bias;
    g.M = M; g.N = N; g.K = K; g.blocks = (K + 127) / 128; g.beta = beta; g.relu = (flags & SP_GEMM_RELU) != 0; g.out_dtype = dtype_out;
    auto by_block = [&](auto fa, auto fb) {
        constexpr int FA = decltype(fa)::value, FB = decltype(fb)::value;
        const hipStream_t st = (hipStream_t)stream;
        if (dtype_out == SP_F32) return block_n == 128 ? multiply<FA, FB, false, 7>(g, st) : multiply<FA, FB, false, 0>(g, st);
        return block_n == 128 ? multiply<FA, FB, true, 7>(g, st) : multiply<FA, FB, true, 0>(g, st);
    };
    typedef std::integral_constant<int, SP_F8_E4M3> e4m3;
    typedef std::integral_constant<int, SP_F8_E5M2> e5m2;
    if (f8_a == SP_F8_E4M3) return f8_b == SP_F8_E4M3 ? by_block(e4m3{}, e4m3{}) : by_block(e4m3{}, e5m2{});
    return f8_b == SP_F8_E4M3 ? by_block(e5m2{}, e4m3{}) : by_block(e5m2{}, e5m2{});
}
