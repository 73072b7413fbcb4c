// C = A . B^T of 8-bit operands with a scale for each block of 128 along K: per row of A, per row of B or per 128 of its rows.
//
// A block of 128 is 128 bytes of a row: four f16 MFMAs of K = 32, which start from zero.  The vector ALU multiplies their sum by
// the block's two scales and adds it to the accumulators (so the sum over the blocks is rounded to nearest f32): four multiply-adds
// of 4 cycles per 16 x 16 block, against 64 cycles on the matrix pipe.
//
// The B fragment is the MFMA's first operand: register r of lane l of a 16 x 16 fragment holds C[m = l % 16][n = 4 (l / 16) + r], so a lane
// needs one scale of A per fragment and stores four consecutive columns.
//
// Two kernels.  gemm_scaled_tile_kernel: workgroup tiles in LDS, for outputs that fill the chip.  gemm_scaled_split_kernel: few rows, or
// few tiles; the waves of a workgroup share one small tile, take the blocks of K in turn straight from global memory, and add up in LDS, in a fixed order.
#include "vec_io.h"

namespace sp {

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
    int stream;                   // C does not stay in the caches
};

// A lane's 32 numbers of a block of one row, as f16, which holds every number of both types.  A and B agree on which 16-byte chunks of the block they
// are; in which order does not matter.
template <int F8>
struct Fragment {
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

// The sum of one block.  The f16 MFMAs have exact products and keep 24 bits below the largest of a sum (measured: 128 N(0, 1) products are 0.5 U of the sum of their magnitudes off at
// most, numbers of every exponent 4 U, U = 2^-24).  The 8-bit MFMAs, of K = 128 at twice the rate and of K = 32 at the same, add eight products at a time and cut off what
// lies below 2^-13 of the largest's power of two before they go on in f32 (2^16 + 4 - 2^16 is 0; 280 to 3000 U off): no type of C takes them.
template <int F8A, int F8B>
__device__ __forceinline__ f32x4 block_sum(const Fragment<F8B>& b, const Fragment<F8A>& a) {
    f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 4; ++h) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(b.v[h], a.v[h], t, 0, 0, 0);
    return t;
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

// Eight (16-bit C) or four columns of a row of C from col on, all of which exist if WHOLE.
template <int OT, bool HAS_BETA, bool WHOLE, int POLICY>
__device__ __forceinline__ void put_piece(const ScaledArgs& g, long row, long col, float (&v)[PER16<OT>], const float (&bias)[PER16<OT>]) {
    constexpr int P = PER16<OT>;
    if (!WHOLE && (row >= g.M || col >= g.N)) return;
    const long idx = row * g.N + col, left = WHOLE ? P : g.N - col;
    if constexpr (HAS_BETA) {
        const u32x4 old = load16<OT>(g.C, idx, left);
#pragma unroll
        for (int e = 0; e < P; ++e) v[e] += g.beta * element<OT>(old, e);
    }
#pragma unroll
    for (int e = 0; e < P; ++e) {
        v[e] += bias[e];
        v[e] = g.relu ? fmaxf(v[e], 0.f) : v[e];
    }
    store16<OT, POLICY>(g.C, idx, left, v);
}

// A wave's accumulators to C: two rows of fragments at a time go through a strip of LDS of its own, so that whole 16-byte pieces of C leave, side by
// side along its rows (as 16 rows of 32 bytes per instruction, straight from the registers, 8192 x 4096 x 4096 bf16 takes 248 us against 235, 8192 x 8192 x 2048 280 against 253).
template <int TN>
constexpr int STRIP_ROW = 16 * TN * 4 + 16;                // bytes; the pad spreads a column over the banks
template <int OT, bool HAS_BETA, bool WHOLE, int POLICY, int TM, int TN>
__device__ __forceinline__ void put_rows(const ScaledArgs& g, const f32x4 (&acc)[TM][TN], unsigned char* strip, long row0, long col0, int lane) {
    constexpr int P = PER16<OT>, LANES = 16 * TN / P, ROWS = 64 / LANES;       // lanes per row of C, rows per pass
    static_assert(ROWS >= 1 && 32 % ROWS == 0, "a strip of 32 rows in whole passes");
    const int fi = lane & 15, fq = lane >> 4, er = lane / LANES, ec = lane % LANES * P;
    const long col = col0 + ec;
    float bias[P] = {};
    if (g.bias != nullptr)
#pragma unroll
        for (int e = 0; e < P; ++e)
            if (WHOLE || col + e < g.N) bias[e] = g.bias[col + e];
#pragma unroll
    for (int i = 0; i < TM; i += 2) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int j = 0; j < TN; ++j) *reinterpret_cast<f32x4*>(strip + (16 * k + fi) * STRIP_ROW<TN> + (16 * j + 4 * fq) * 4) = acc[i + k][j];
#pragma unroll
        for (int p = 0; p < 32 / ROWS; ++p) {
            float v[P];
#pragma unroll
            for (int h = 0; h < P; h += 4) {
                const f32x4 q = *reinterpret_cast<const f32x4*>(strip + (p * ROWS + er) * STRIP_ROW<TN> + (ec + h) * 4);
                v[h] = q[0], v[h + 1] = q[1], v[h + 2] = q[2], v[h + 3] = q[3];
            }
            put_piece<OT, HAS_BETA, WHOLE, POLICY>(g, row0 + 16 * i + p * ROWS + er, col, v, bias);
        }
    }
}
template <int TM, int TN>
__device__ __forceinline__ void put_tile(const ScaledArgs& g, const f32x4 (&acc)[TM][TN], unsigned char* strip, long row0, long col0, int lane) {
    // a C that does not stay in the caches anyway is streamed past them where its tiles are whole: 8192 x 8192 x 2048 bf16 260 -> 254 us, 8192 x 4096 x 4096 bf16
    // 245 -> 239
    const bool whole = row0 + 16 * TM <= g.M && col0 + 16 * TN <= g.N;
    auto put = [&](auto ot) {
        constexpr int OT = decltype(ot)::value;
        if (g.beta != 0.f) put_rows<OT, true, false, ST_PLAIN>(g, acc, strip, row0, col0, lane);
        else if (whole && g.stream) put_rows<OT, false, true, ST_STREAM>(g, acc, strip, row0, col0, lane);
        else if (whole) put_rows<OT, false, true, ST_PLAIN>(g, acc, strip, row0, col0, lane);
        else put_rows<OT, false, false, ST_PLAIN>(g, acc, strip, row0, col0, lane);
    };
    if (g.out_dtype == SP_F32) put(std::integral_constant<int, SP_F32>{});
    else if (g.out_dtype == SP_BF16) put(std::integral_constant<int, SP_BF16>{});
    else put(std::integral_constant<int, SP_F16>{});
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

// Scales come in for several blocks of K at a time, a chunk: SB = 8 of them of eight rows, or 4 of sixteen, per instruction.  The scales of a row's blocks lie side
// by side, so that a load asks for eight or sixteen lines of memory and not for 64, as many as the operands of a whole block.
constexpr int SCALE_BLOCKS = 8, SPLIT_BLOCKS = 4;

// Lane l's scale is that of row l / SB and block l % SB of what `row` and `first` say; to LDS bytes lds_addr + 4 l.
template <int SB>
__device__ __forceinline__ void dma_scales(const float* scales, long row, long last_row, long first, long blocks, int lane, unsigned lds_addr) {
    const long r = row + lane / SB < last_row ? row + lane / SB : last_row, k = first + lane % SB < blocks ? first + lane % SB : blocks - 1;
    const float* at = scales + r * blocks + k;
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(at), "s"(lds_addr) : "memory", "m0");
}

// 16-byte chunk kc of row `row` of a tile in LDS stands in slot kc ^ f(row) of the row: the 16 rows that one read of a fragment touches lie in
// different banks, and every fragment has the same pattern, so fragments of an operand are apart by immediates.
__device__ __forceinline__ int tile_slot(int row, int kc) { return (kc ^ row ^ (row >> 3 & 1)) & 7; }

// Tiles of BM x BN on WM x WN waves, two stages of LDS.  SHIFT: 7 where a scale of B holds for 128 rows, else 0.
//
// A wave walks its TM rows of fragments.  While row i is on the matrix pipe, the vector ALU adds the scaled sums of row i - 1 and the fragment of row i + 1 comes
// in from LDS.  The boundary between two blocks of K stands in front of a block's last row: by then everything of the
// block is in registers, and the next block has landed.  Behind each MFMA of the last row the next block's fragment of B takes the place of the one just
// used; then the block after that is asked for.  A wave waits where it asks (the unit takes an instruction of 1 KiB every 16 cycles), so it does that with MFMAs under way: in front of the last row
// 4096 x 2048 x 5008 took 95 us, behind it 89, half there and half a row later 90.
template <int F8A, int F8B, int SHIFT, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM* WN * 64, 2) void gemm_scaled_tile_kernel(const ScaledArgs g) {
    constexpr int NW = WM * WN, WTM = BM / WM, WTN = BN / WN, TM = WTM / 16, TN = WTN / 16;
    constexpr int NIA = BM / 8 / NW, NI = (BM + BN) / 8 / NW;       // DMA instructions of 8 rows per wave and block; A's first
    constexpr int GROUPS_A = BM / 8, GROUPS = GROUPS_A + (SHIFT == 7 ? 1 : BN / 8);      // of eight rows of scales; B's behind A's
    static_assert(GROUPS <= SCALE_BLOCKS * NW && NW % 2 == 0 && TM % 2 == 0, "one instruction of scales per wave and block");
    constexpr int STAGE = (BM + BN) * ROW_BYTES, SCALE_STAGE = GROUPS * 256;
    static_assert(2 * (STAGE + SCALE_STAGE) <= 160 * 1024 && NW * 32 * STRIP_ROW<TN> <= 2 * STAGE, "LDS");
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN, fi = lane & 15, fq = lane >> 4;
    int tm, tn;
    scaled_tile_of_block(blockIdx.x, g.tiles_m, g.tiles_n, g.group_m, tm, tn);
    const long m0 = (long)tm * BM, n0 = (long)tn * BN;
    const int nk = (int)g.blocks;
    const bool k_tail = (g.K & 127) != 0;

    // operands: instruction q of a wave takes rows (q NW + wave) 8 ... of A's or B's part of the tile, a lane 16 bytes of one of them.  Rows past the
    // end are the last row again: the offset of a row stops at that row's.  Chunks past the end of a row are zeros.
    const unsigned char* pA = uniform_ptr(g.A + m0 * g.K);
    const unsigned char* pB = uniform_ptr(g.B + n0 * g.K);
    const unsigned K = (unsigned)g.K, lds_base = (unsigned)(size_t)lds;
    const int r = lane >> 3, kc = tile_slot((wave & 1) * 8 + r, lane & 7);
    const unsigned voff = (unsigned)(wave * 8 + r) * K + kc * 16;
    const long left_a = g.M - m0 - 1, left_b = g.N - n0 - 1;
    const unsigned last_a = (unsigned)(left_a < BM ? left_a : BM) * K + kc * 16, last_b = (unsigned)(left_b < BN ? left_b : BN) * K + kc * 16;
    const bool tail_in = (long)(nk - 1) * ROW_BYTES + kc * 16 < g.K;
    const unsigned dst = __builtin_amdgcn_readfirstlane(lds_base + wave * 8 * ROW_BYTES);
    // scales: of the eight blocks from 8 c on, in stage c % 2; wave w brings its share (group `part` NW + w) once per block, a chunk ahead
    const unsigned scale_lds = __builtin_amdgcn_readfirstlane(lds_base + 2 * STAGE);
    const long last_sb = SHIFT == 7 ? (g.N - 1) >> 7 : g.N - 1;
    auto fetch_scales = [&](int chunk, int part) {
        const int group = part * NW + wave;
        if (group >= GROUPS || chunk * SCALE_BLOCKS >= nk) return;
        const bool of_a = group < GROUPS_A;
        const unsigned to = scale_lds + (chunk & 1) * SCALE_STAGE + group * 256;
        dma_scales<SCALE_BLOCKS>(of_a ? g.scale_a : g.scale_b, of_a ? m0 + group * 8 : (n0 >> SHIFT) + (group - GROUPS_A) * 8, of_a ? g.M - 1 : last_sb,
                   (long)chunk * SCALE_BLOCKS, nk, lane, to);
    };
    auto fetch = [&](int kt, unsigned stage) {
        const unsigned char *a = pA + (long)kt * ROW_BYTES, *b = pB + (long)kt * ROW_BYTES;
        auto offset = [&](int q) {
            const unsigned at = voff + (unsigned)(q < NIA ? q : q - NIA) * (NW * 8) * K, last = q < NIA ? last_a : last_b;
            return at < last ? at : last;
        };
        auto to = [&](int q) { return dst + stage + (q < NIA ? q * NW * 8 : BM + (q - NIA) * NW * 8) * ROW_BYTES; };
        if (k_tail && kt == nk - 1) {
#pragma unroll
            for (int q = 0; q < NI; ++q) {
                const unsigned char* inside = (q < NIA ? a : b) + offset(q);
                dma_to_lds_addr(tail_in ? inside : (const unsigned char*)kZeroChunk, to(q));
            }
        } else {
#pragma unroll
            for (int q = 0; q < NI; ++q) dma_to_lds(q < NIA ? a : b, offset(q), to(q));
        }
    };
    // fragments: chunks 2 fq and 2 fq + 1 of a row
    int at_a[2], at_b[2];
    const int at_sa = 2 * STAGE + (wm * WTM + fi) * 32, at_sb = 2 * STAGE + GROUPS_A * 256 + (SHIFT == 7 ? (wn * WTN) >> 7 : wn * WTN + 4 * fq) * 32;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int in = fi * ROW_BYTES + (tile_slot(fi, 2 * fq + h) << 4);
        at_a[h] = wm * WTM * ROW_BYTES + in;
        at_b[h] = (BM + wn * WTN) * ROW_BYTES + in;
    }
    u32x4 ra[2][2], rb[TN][2];
    auto load_a = [&](int i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) ra[i & 1][h] = *reinterpret_cast<const u32x4*>(lds + at_a[h] + i * 16 * ROW_BYTES);
    };
    auto load_b = [&](int j) {
#pragma unroll
        for (int h = 0; h < 2; ++h) rb[j][h] = *reinterpret_cast<const u32x4*>(lds + at_b[h] + j * 16 * ROW_BYTES);
    };
    float sa[TM], pending = 0.f;                       // pending: the scale of the row whose sums are still to be added
    f32x4 sb[SHIFT == 7 ? 1 : TN], sb_pending[SHIFT == 7 ? 1 : TN];
    auto load_scales = [&](int kt) {
        const unsigned char* at = lds + (kt >> 3 & 1) * SCALE_STAGE + (kt & 7) * 4;
#pragma unroll
        for (int i = 0; i < TM; ++i) sa[i] = *reinterpret_cast<const float*>(at + at_sa + i * 512);
        if constexpr (SHIFT == 7) {
            sb[0][0] = *reinterpret_cast<const float*>(at + at_sb);
        } else {
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) sb[j][e] = *reinterpret_cast<const float*>(at + at_sb + (16 * j + e) * 32);
        }
    };
    f32x4 acc[TM][TN], sums[2][TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        sums[1][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (SHIFT != 7) sb_pending[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    auto add = [&](int i, int j, float scale, const f32x4& scale_n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            // (the scales first, as in the other kernel: the sum times one of them may be no f32 where the product of both is)
            acc[i][j][e] = __builtin_fmaf(sums[i & 1][j][e], SHIFT == 7 ? scale : scale * scale_n[e], acc[i][j][e]);
        }
        asm volatile("" : "+v"(acc[i][j]));            // here, not where the loop ends: that is where the compiler would gather them
    };

    for (int part = 0; part < SCALE_BLOCKS; ++part) fetch_scales(0, part);
    fetch(0, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    fetch_scales(1, 0);
    fetch(nk > 1 ? 1 : 0, STAGE);                      // (past the last block the last one comes again, into a stage that is not read: no branch)
#pragma unroll
    for (int j = 0; j < TN; ++j) load_b(j);
    load_a(0);
    load_scales(0);
    int step = STAGE;
    Fragment<F8B> fb[TN];
    for (int kt = 0; kt < nk; ++kt) {
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const bool boundary = i == TM - 1;
            if (!boundary) {
                load_a(i + 1);
            } else {
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                __syncthreads();
#pragma unroll
                for (int h = 0; h < 2; ++h) at_a[h] += step, at_b[h] += step;
                step = -step;
                load_a(0);
            }
            __builtin_amdgcn_sched_barrier(0);
            Fragment<F8A> fa;
            fa.set(ra[i & 1]);
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                if (i == 0) fb[j].set(rb[j]);
                sums[i & 1][j] = block_sum<F8A, F8B>(fb[j], fa);
                if (i == 0) add(TM - 1, j, pending, sb_pending[SHIFT == 7 ? 0 : j]);
                else add(i - 1, j, sa[i - 1], sb[SHIFT == 7 ? 0 : j]);
                if (boundary) load_b(j);
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (SHIFT == 7)
                if (i == 0)
#pragma unroll
                    for (int k = 0; k < TM; ++k) sa[k] *= sb[0][0];
            if (boundary) {
                fetch_scales((kt + 1) / SCALE_BLOCKS + 1, (kt + 1) % SCALE_BLOCKS);
                fetch(kt + 2 < nk ? kt + 2 : nk - 1, step > 0 ? STAGE : 0);
                pending = sa[TM - 1];
                if constexpr (SHIFT != 7)
#pragma unroll
                    for (int j = 0; j < TN; ++j) sb_pending[j] = sb[j];
                load_scales(kt + 1);
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int j = 0; j < TN; ++j) add(TM - 1, j, pending, sb_pending[SHIFT == 7 ? 0 : j]);
    __syncthreads();                                       // the stages are not read any more
    put_tile(g, acc, lds + wave * (32 * STRIP_ROW<TN>), m0 + wm * WTM, n0 + wn * WTN, lane);
}

// One tile of (16 TM) x (16 TN) outputs on four waves: each takes a quarter of K through an LDS ring of NS stages of its own, so no
// wave waits for another inside the loop, and the four partial sums meet in LDS at the end.  All that is read comes in by DMA, the scales too.
template <int F8A, int F8B, int SHIFT, int TM, int TN, int NS>
__global__ __launch_bounds__(256) void gemm_scaled_split_kernel(const ScaledArgs g) {
    constexpr int KS = 4;
    constexpr int NIA = 2 * TM, ND = 2 * (TM + TN);     // DMA instructions per block
    constexpr int GROUPS_A = TM, GROUPS = GROUPS_A + (SHIFT == 7 ? 1 : TN);               // of sixteen rows of scales
    constexpr int STAGE = ND * 8 * ROW_BYTES, WAVE_LDS = NS * STAGE + 2 * GROUPS * 256;
    static_assert((NS - 1) * ND < 64 && NS <= SPLIT_BLOCKS, "vmcnt counts to 63; scales are asked for a chunk ahead of their operands");
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fi = lane & 15, fq = lane >> 4;
    int tm, tn;
    scaled_tile_of_block(blockIdx.x, g.tiles_m, g.tiles_n, g.group_m, tm, tn);
    const long m0 = (long)tm * (16 * TM), n0 = (long)tn * (16 * TN);
    const int nk = (int)g.blocks;
    const bool k_tail = (g.K & 127) != 0;
    const unsigned char* pA = uniform_ptr(g.A + m0 * g.K);
    const unsigned char* pB = uniform_ptr(g.B + n0 * g.K);
    const unsigned my_lds = __builtin_amdgcn_readfirstlane((unsigned)(size_t)lds + wave * WAVE_LDS);
    const int r = lane >> 3;
    unsigned voff[ND], tail_in = 0;
#pragma unroll
    for (int q = 0; q < ND; ++q) {
        const int blk = q < NIA ? q : q - NIA, kc = (lane & 7) ^ ((r ^ blk) & 7);
        const long left = (q < NIA ? g.M - m0 : g.N - n0) - 1, row = blk * 8 + r < left ? blk * 8 + r : left;
        voff[q] = (unsigned)(row * g.K) + kc * 16;
        if ((long)(nk - 1) * ROW_BYTES + kc * 16 < g.K) tail_in |= 1u << q;
    }
    // this wave's blocks: an even share, one after the other
    const int first = (int)((long)nk * wave / KS), mine = (int)((long)nk * (wave + 1) / KS) - first;
    const long last_sb = SHIFT == 7 ? (g.N - 1) >> 7 : g.N - 1;
    auto fetch_scales = [&](int chunk) {
#pragma unroll
        for (int q = 0; q < GROUPS; ++q) {
            const bool of_a = q < GROUPS_A;
            dma_scales<SPLIT_BLOCKS>(of_a ? g.scale_a : g.scale_b, of_a ? m0 + q * 16 : (n0 >> SHIFT) + (q - GROUPS_A) * 16, of_a ? g.M - 1 : last_sb,
                       (long)first + chunk * SPLIT_BLOCKS, nk, lane, my_lds + NS * STAGE + ((chunk & 1) * GROUPS + q) * 256);
        }
    };
    auto fetch = [&](int kt, unsigned stage) {
        const unsigned char *a = pA + (long)kt * ROW_BYTES, *b = pB + (long)kt * ROW_BYTES;
        const unsigned dst = my_lds + stage * STAGE;
        if (k_tail && kt == nk - 1) {
#pragma unroll
            for (int q = 0; q < ND; ++q) {
                const unsigned char* inside = (q < NIA ? a : b) + voff[q];
                dma_to_lds_addr((tail_in >> q) & 1u ? inside : (const unsigned char*)kZeroChunk, dst + q * 8 * ROW_BYTES);
            }
        } else {
#pragma unroll
            for (int q = 0; q < ND; ++q) dma_to_lds(q < NIA ? a : b, voff[q], dst + q * 8 * ROW_BYTES);
        }
    };

    if (mine > 0) fetch_scales(0);
#pragma unroll
    for (int s = 0; s < NS; ++s)
        if (s < mine) fetch(first + s, s);
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const unsigned char* ring = lds + wave * WAVE_LDS;
    int stage = 0;
    for (int t = 0; t < mine; ++t) {
        // block t has landed, and the scales, which were asked for before it: with NS of them under way that leaves NS - 1 behind it, near the end only "none" says it
        if (t + NS <= mine) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 1) * ND) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const unsigned char* at = ring + stage * STAGE;
        const float* scales = reinterpret_cast<const float*>(ring + NS * STAGE + (t / SPLIT_BLOCKS & 1) * (GROUPS * 256)) + t % SPLIT_BLOCKS;
        u32x4 ra[TM][2], rb[TN][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < TM; ++i) ra[i][h] = *reinterpret_cast<const u32x4*>(at + lds_offset(16 * i + fi, 2 * fq + h));
#pragma unroll
            for (int j = 0; j < TN; ++j) rb[j][h] = *reinterpret_cast<const u32x4*>(at + NIA * 8 * ROW_BYTES + lds_offset(16 * j + fi, 2 * fq + h));
        }
        float sa[TM];
        f32x4 sb[TN];
#pragma unroll
        for (int i = 0; i < TM; ++i) sa[i] = scales[(16 * i + fi) * SPLIT_BLOCKS];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            if constexpr (SHIFT == 7) {
                sb[j][0] = scales[GROUPS_A * 64];             // (a tile lies inside one block of 128 rows of B)
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) sb[j][e] = scales[(16 * (TM + j) + 4 * fq + e) * SPLIT_BLOCKS];
            }
        }
        if (t + NS < mine) {
            // the stage is free once all of it is in registers, and so is, with the first block of a chunk, the chunk before it
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (t % SPLIT_BLOCKS == 0 && t + SPLIT_BLOCKS < mine) fetch_scales(t / SPLIT_BLOCKS + 1);
            fetch(first + t + NS, stage);
            __builtin_amdgcn_sched_barrier(0);
        }
        stage = stage + 1 == NS ? 0 : stage + 1;
        Fragment<F8A> fa[TM];
#pragma unroll
        for (int i = 0; i < TM; ++i) fa[i].set(ra[i]);
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            Fragment<F8B> fb;
            fb.set(rb[j]);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const f32x4 v = block_sum<F8A, F8B>(fb, fa[i]);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(v[e], sa[i] * sb[j][SHIFT == 7 ? 0 : e], acc[i][j][e]);
            }
        }
    }
    // partial tiles: fragment f of wave w at (f * 4 + w) * 1 KiB; fragment f is then finished by wave f % 4
    __syncthreads();                                       // the rings are not read any more
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
            put_quad(g, m0 + 16 * i + fi, n0 + 16 * j + 4 * fq, (p[0] + p[64]) + (p[128] + p[192]));
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

template <int F8A, int F8B, int SHIFT, int BM, int BN, int WM, int WN>
static int launch_tile(ScaledArgs g, hipStream_t stream) {
    auto kernel = gemm_scaled_tile_kernel<F8A, F8B, SHIFT, BM, BN, WM, WN>;
    constexpr int lds_bytes = 2 * ((BM + BN) * ROW_BYTES + (BM / 8 + (SHIFT == 7 ? 1 : BN / 8)) * 256);
    if (const int rc = check_tiles(g, BM, BN, WM * WN * 64); rc != SP_OK) return rc;
    if (const int rc = ensure_dynamic_lds((const void*)kernel, lds_bytes); rc != SP_OK) return rc;
    g.group_m = 4;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(g.tiles_m * g.tiles_n)), dim3(WM * WN * 64), lds_bytes, stream, g);
    return check_launch("sp_gemm_abt_scaled");
}

template <int F8A, int F8B, int SHIFT, int TM, int TN, int NS>
static int launch_split(ScaledArgs g, hipStream_t stream) {
    auto kernel = gemm_scaled_split_kernel<F8A, F8B, SHIFT, TM, TN, NS>;
    constexpr int ring = 4 * (NS * 2 * (TM + TN) * 8 * ROW_BYTES + 2 * (TM + (SHIFT == 7 ? 1 : TN)) * 256), partial = TM * TN * 4096;
    constexpr int lds_bytes = ring > partial ? ring : partial;
    if (const int rc = check_tiles(g, 16 * TM, 16 * TN, 256); rc != SP_OK) return rc;
    if (const int rc = ensure_dynamic_lds((const void*)kernel, lds_bytes); rc != SP_OK) return rc;
    g.group_m = g.tiles_m;        // the tiles of one panel of B stand side by side
    hipLaunchKernelGGL(kernel, dim3((unsigned)(g.tiles_m * g.tiles_n)), dim3(256), lds_bytes, stream, g);
    return check_launch("sp_gemm_abt_scaled");
}

// Which kernel: the largest tile that still gives every compute unit one (and half of them for 128 x 128); else the split ones.
// Measured (us), bf16 C, scales of 128 x 128 of B, N = K = 4096: 4096 rows 128 x 256 122, 128 x 128 129; 2048 rows 61, 65.5; 1024 rows 54, 42, split 64 x 64 46; 512 rows
// 128 x 128 41, split 64 x 64 25, 32 x 32 34.5; 256 rows 40.5, 18.4, 19.7; 128 rows split 64 x 64 17.3, 32 x 32 11.3, 16 x 16 19.9; 64 rows 16.9, 8.0, 11.9; 16 rows
// split 32 x 32 7.6, 16 x 16 6.3; one row 7.6, 6.0.  49 x 32003 x 4096 split 64 x 64 35.4, 32 x 32 42.9 (f32 C 35.6, 43.1); 32 x 32003 x 4096 33.3, 32.2; 1 x 16384 x 16384
// split 32 x 32 64, 16 x 16 55; 4096 x 2048 x 5008, f32 C and scales per row of B: 128 x 256 95.7, 128 x 128 99.
template <int F8A, int F8B, int SHIFT>
static int multiply(const ScaledArgs& g, hipStream_t stream) {
    const long cus = device_cu_count();
    auto tiles = [&](long bm, long bn) { return ((g.M + bm - 1) / bm) * ((g.N + bn - 1) / bn); };
    if (g.M > 64) {
        if (tiles(128, 256) >= cus) return launch_tile<F8A, F8B, SHIFT, 128, 256, 2, 4>(g, stream);
        if (tiles(128, 128) * 2 > cus) return launch_tile<F8A, F8B, SHIFT, 128, 128, 2, 2>(g, stream);
    }
    if (g.M <= 16) return launch_split<F8A, F8B, SHIFT, 1, 1, 4>(g, stream);
    if (g.M <= 32 || tiles(32, 32) <= 3 * cus) return launch_split<F8A, F8B, SHIFT, 2, 2, 2>(g, stream);
    return launch_split<F8A, F8B, SHIFT, 4, 4, 1>(g, stream);
}

namespace {
struct GemmScaledKernelNames {
    GemmScaledKernelNames() {
        register_kernel("gemm_scaled_128x256", (const void*)gemm_scaled_tile_kernel<SP_F8_E4M3, SP_F8_E4M3, 7, 128, 256, 2, 4>, 512);
        register_kernel("gemm_scaled_128x128", (const void*)gemm_scaled_tile_kernel<SP_F8_E4M3, SP_F8_E4M3, 7, 128, 128, 2, 2>, 256);
        register_kernel("gemm_scaled_split_16x16", (const void*)gemm_scaled_split_kernel<SP_F8_E4M3, SP_F8_E4M3, 7, 1, 1, 4>, 256);
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
    g.stream = M * N * (dtype_out == SP_F32 ? 4 : 2) > (int64_t)32 << 20;
    auto by_block = [&](auto fa, auto fb) {
        constexpr int FA = decltype(fa)::value, FB = decltype(fb)::value;
        const hipStream_t st = (hipStream_t)stream;
        return block_n == 128 ? multiply<FA, FB, 7>(g, st) : multiply<FA, FB, 0>(g, st);
    };
    typedef std::integral_constant<int, SP_F8_E4M3> e4m3;
    typedef std::integral_constant<int, SP_F8_E5M2> e5m2;
    if (f8_a == SP_F8_E4M3) return f8_b == SP_F8_E4M3 ? by_block(e4m3{}, e4m3{}) : by_block(e4m3{}, e5m2{});
    return f8_b == SP_F8_E4M3 ? by_block(e5m2{}, e4m3{}) : by_block(e5m2{}, e5m2{});
}
