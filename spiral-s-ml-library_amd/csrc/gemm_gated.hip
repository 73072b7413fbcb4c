// The gated feed-forward block and its gradients: C = act(A . G^T) * (A . U^T), the two projections G (gate) and U (up) of N x K.
//
// Forward: one product of A with rows of G and of U in turn, 16 of one and 16 of the other, so that a lane's accumulators hold both factors of its
// outputs; activation and product are the epilogue, and the factors leave only where a backward pass wants them (kept), whole or as 8-bit blocks.
// Backward, from g and u as they were kept:  dg = dC u act'(g), du = dC act(g), rounded to the type of A, side by side in a workspace of M x 2 N';
//   dA = dg . G + du . U     sums over N: one product over both halves of the workspace, one behind the other
//   dG = dg^T . A, dU = du^T . A     sums over M
// G, U, A and the workspace are then read across their rows: tiles of K rows go to LDS as they lie in memory, and a fragment is read transposed
// (ds_read_b64_tr_b16: 16 lanes take 4 x 16 numbers, each lane a column's four; f32: four reads of 4 bytes).
//
// All products: tiles of LDS in two stages that DMA fills, 128 bytes of K (of a row, or of K rows) a stage.  A wave walks its TM rows of fragments; the fragment of a
// row is replaced by the next half stage's once its MFMAs are issued, the B fragments have two sets.  The boundary between two stages stands in the middle: everything
// of a stage is in registers then, and the next one has landed.
// K may end anywhere: what is missing of the last K-tile comes from zeros, and that tile goes first, so that the loop has whole ones only.
#include "f8_blocks.h"

namespace sp {

enum { MM_FORWARD, MM_INPUT, MM_WEIGHTS };
enum { KEEP_NONE, KEEP_WHOLE, KEEP_F8 };

struct GatedArgs {
    // forward: A, G, U; gradient of A: workspace, G, U; of the weights: workspace, A
    const unsigned char *A, *B0, *B1;
    void *C0, *C1;                // C; dA; dG, dU
    void *gate, *up;              // kept
    float *gate_scale, *up_scale;
    long M, N, K;                 // of the forward product
    long half;                    // N': columns of either half of the workspace, N rounded up to a whole K-tile, zeros behind N
    int activation, keep;
    int tiles_m, tiles_n, group_m;
    int stream;                   // C does not stay in the caches
};

__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504088896340736f)); }
__device__ __forceinline__ float gated_activation(float g, int kind) {
    if (kind == SP_ACT_SILU) return g * sigmoid(g);
    if (kind == SP_ACT_GELU) return 0.5f * g * (1.f + erff(g * 0.70710678118654752440f));
    return g < 0.f ? 0.f : g;                              // (a NaN stays)
}
// act(g) and act'(g).
__device__ __forceinline__ void activation_and_slope(float g, int kind, float& act, float& slope) {
    if (kind == SP_ACT_SILU) {
        const float s = sigmoid(g);
        act = g * s;
        slope = s * __builtin_fmaf(g, 1.f - s, 1.f);
    } else if (kind == SP_ACT_GELU) {
        const float below = 0.5f * (1.f + erff(g * 0.70710678118654752440f));
        act = g * below;
        slope = __builtin_fmaf(g * 0.39894228040143267794f, __builtin_amdgcn_exp2f(g * g * -0.72134752044448170368f), below);
    } else {
        act = g < 0.f ? 0.f : g;
        slope = g > 0.f ? 1.f : 0.f;
    }
}

// One K-step of a 16 x 16 fragment: 16 bytes of K per lane from either operand, B first (a lane then holds four consecutive columns of a row).
template <int DT>
__device__ __forceinline__ f32x4 gated_mma(const u32x4& b, const u32x4& a, f32x4 c) {
    if constexpr (DT == SP_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), c, 0, 0, 0);
    } else if constexpr (DT == SP_F16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, b), __builtin_bit_cast(f16x8, a), c, 0, 0, 0);
    } else {
        const f32x4 vb = __builtin_bit_cast(f32x4, b), va = __builtin_bit_cast(f32x4, a);
#pragma unroll
        for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(vb[s], va[s], c, 0, 0, 0);
        return c;
    }
}

// Workgroups are dealt round-robin to the 8 XCDs: each gets a contiguous range of a walk in groups of group_m tile rows.
__device__ __forceinline__ void gated_tile_of_block(int pid, int tiles_m, int tiles_n, int group_m, int& tm, int& tn) {
    const int n = tiles_m * tiles_n, xcd = pid & 7, base = n >> 3, rem = n & 7;
    const int t = xcd * base + (xcd < rem ? xcd : rem) + (pid >> 3);
    const int group_size = group_m * tiles_n, g = t / group_size, first = g * group_m;
    const int rows = tiles_m - first < group_m ? tiles_m - first : group_m, in = t - g * group_size;
    tm = first + in % rows;
    tn = in / rows;
}

// ---- an operand's tile in LDS ----
// Along K: R rows of 128 bytes; 16-byte chunk kc of row `row` in slot kc ^ row ^ (row >> 3 & 1).
// Across: the K rows of W columns; what 16 lanes read at once (16 columns, 32 or 64 bytes, of four K rows or of one) is a unit, and units are
// swizzled over the 256 bytes of the banks so that the four rows, and two groups of lanes, or the four groups, have different ones.
__device__ __forceinline__ int along_slot(int row, int kc) { return (kc ^ row ^ (row >> 3 & 1)) & 7; }
template <int ES, int W>
__device__ __forceinline__ int across_swizzle(int k) {
    if constexpr (ES == 4) return k >> 3 & 3;
    else if constexpr (W >= 128) return (k & 3) | (k >> 4 & 1) << 2;
    else return (k >> 1 & 1) | (k >> 4 & 1) << 1;
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// R: rows (columns) of the tile, TF: fragments of a wave, from row (column) `first` on.
template <int ES, bool ACROSS, int R, int TF>
struct Fragments {
    static constexpr int ROW = R * ES;                     // bytes of a K row, ACROSS
    int at[ACROSS ? TF : 2];
    __device__ __forceinline__ Fragments(int base, int first, int fi, int fq) {
        if constexpr (ACROSS) {
            const int k = ES == 4 ? 8 * fq : 16 * fq + (fi >> 2);
            const int in = ES == 4 ? fi * 4 : (fi & 3) * 8;
#pragma unroll
            for (int t = 0; t < TF; ++t) at[t] = base + k * ROW + (((first >> 4) + t) ^ across_swizzle<ES, R>(k)) * (16 * ES) + in;
        } else {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) at[ks] = base + (first + fi) * ROW_BYTES + along_slot(fi, 2 * fq + ks) * 16;
        }
    }
    __device__ __forceinline__ void step(int bytes) {
#pragma unroll
        for (int t = 0; t < (ACROSS ? TF : 2); ++t) at[t] += bytes;
    }
    // The chunk 2 fq + ks of K of row 16 t + fi.
    __device__ __forceinline__ u32x4 load(unsigned char* lds, int ks, int t) const {
        if constexpr (!ACROSS) {
            return *reinterpret_cast<const u32x4*>(lds + at[ks] + t * 16 * ROW_BYTES);
        } else if constexpr (ES == 2) {
            const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds + at[t] + (8 * ks) * ROW)));
            const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds + at[t] + (8 * ks + 4) * ROW)));
            return u32x4{lo.x, lo.y, hi.x, hi.y};
        } else {
            u32x4 v;
#pragma unroll
            for (int s = 0; s < 4; ++s) v[s] = *reinterpret_cast<const unsigned*>(lds + at[t] + (4 * ks + s) * ROW);
            return v;
        }
    }
};

// A wave's share of the DMA of an operand's tile: instruction q takes 1 KiB, block q NW + wave.
template <int ES, bool ACROSS, int R, int NW>
struct Loader {
    static constexpr int NI = R / 8 / NW;
    static_assert(R / 8 % NW == 0 && NW % 4 == 0, "blocks split evenly over the waves");
    unsigned off[NI];
    unsigned tail_in = 0;                                  // bit q: this lane's 16 bytes of the partial K-tile exist
    // pitch: bytes from row to row; left: rows (along) or 16-byte chunks of columns (across) from the tile's first one to the last; tail: K of the partial tile.
    // PAIR: rows of two matrices in turn, 16 and 16; a wave's blocks are all of one of them.
    template <bool PAIR>
    __device__ __forceinline__ void set(int lane, int wave, long pitch, long left, int tail) {
#pragma unroll
        for (int q = 0; q < NI; ++q) {
            const int blk = q * NW + wave;
            if constexpr (ACROSS) {
                constexpr int LANES = R * ES / 16, PER_UNIT = ES;
                const int k = blk * (64 / LANES) + lane / LANES, slot = lane % LANES;
                const long chunk = ((slot / PER_UNIT) ^ across_swizzle<ES, R>(k)) * PER_UNIT + slot % PER_UNIT;
                off[q] = (unsigned)(k * pitch + (chunk < left ? chunk : left - 1) * 16);
                if (k < tail) tail_in |= 1u << q;
            } else {
                const int r = lane >> 3, kc = along_slot((blk & 1) * 8 + r, lane & 7);
                const long row = PAIR ? (blk >> 2) * 16 + (blk & 1) * 8 + r : blk * 8 + r;
                off[q] = (unsigned)((row < left ? row : left - 1) * pitch) + kc * 16;
                if (kc * 16 < tail * ES) tail_in |= 1u << q;
            }
        }
    }
};

template <int TN>
constexpr int GATED_STRIP_ROW = 16 * TN * 4 + 16;          // bytes; the pad spreads a column over the banks

// COLS columns of 32 rows that stand in a strip of LDS leave as 16-byte pieces, side by side along the rows.
template <int DT, int COLS, int STRIDE, int POLICY>
__device__ __forceinline__ void put_strip(const unsigned char* strip, void* C, long pitch, long row0, long rows, long col0, long cols, int lane) {
    constexpr int P = PER16<DT>, LANES = COLS / P, ROWS = 64 / LANES;
    static_assert(32 % ROWS == 0, "a strip in whole passes");
    const int er = lane / LANES, ec = lane % LANES * P;
#pragma unroll
    for (int p = 0; p < 32 / ROWS; ++p) {
        float v[P];
#pragma unroll
        for (int h = 0; h < P; h += 4) {
            const f32x4 q = *reinterpret_cast<const f32x4*>(strip + (p * ROWS + er) * STRIDE + (ec + h) * 4);
            v[h] = q[0], v[h + 1] = q[1], v[h + 2] = q[2], v[h + 3] = q[3];
        }
        const long row = row0 + p * ROWS + er, left = cols - col0 - ec;
        if (row < rows && left > 0) store16<DT, POLICY>(C, row * pitch + col0 + ec, left, v);
    }
}

template <int DT, int MODE, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM* WN * 64, 2) void gated_mm_kernel(const GatedArgs g) {
    constexpr int ES = ELEM_BYTES<DT>, BK = ROW_BYTES / ES, NW = WM * WN, WTM = BM / WM, WTN = BN / WN, TM = WTM / 16, TN = WTN / 16;
    constexpr bool A_ACROSS = MODE == MM_WEIGHTS, B_ACROSS = MODE != MM_FORWARD;
    constexpr int A_BYTES = BM * ROW_BYTES, STAGE = (BM + BN) * ROW_BYTES;
    static_assert(TM % 2 == 0 && TN % 2 == 0, "strips of two rows of fragments; a gate's fragment and an up's");
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN, fi = lane & 15, fq = lane >> 4;
    int tm, tn;
    gated_tile_of_block(blockIdx.x, g.tiles_m, g.tiles_n, g.group_m, tm, tn);

    // where the tile lies, and the operands' first rows or columns of it
    const int of_up = MODE == MM_WEIGHTS && tm >= g.tiles_m / 2 ? 1 : 0;
    const long m0 = (long)(tm - of_up * (g.tiles_m / 2)) * BM, n0 = (long)tn * (MODE == MM_FORWARD ? BN / 2 : BN);
    const long pitch_a = (MODE == MM_FORWARD ? g.K : 2 * g.half) * ES, pitch_b = g.K * ES;
    const long inner = MODE == MM_FORWARD ? g.K : MODE == MM_INPUT ? g.N : g.M;          // of one half of K, MM_INPUT
    const int tail = (int)(inner % BK);
    Loader<ES, A_ACROSS, BM, NW> la;
    Loader<ES, B_ACROSS, BN, NW> lb;
    la.template set<false>(lane, wave, pitch_a, A_ACROSS ? (g.half - m0) * ES / 16 : g.M - m0, MODE == MM_INPUT ? BK : tail);
    lb.template set<MODE == MM_FORWARD>(lane, wave, pitch_b, B_ACROSS ? (g.K - n0) * ES / 16 : g.N - n0, tail);
    const unsigned char* const pA = uniform_ptr(g.A + (A_ACROSS ? (of_up * g.half + m0) * ES : m0 * pitch_a));
    const unsigned char* const pB = uniform_ptr(MODE == MM_FORWARD ? ((wave >> 1 & 1) != 0 ? g.B1 : g.B0) + n0 * pitch_b : g.B0 + n0 * ES);
    const long to_up = MODE == MM_INPUT ? g.B1 - g.B0 : 0;

    // the K-tiles in their order, partial ones first: where number s begins in A and in B
    const int whole = (int)(inner / BK), partial = tail != 0 ? (MODE == MM_INPUT ? 2 : 1) : 0, nk = whole * (MODE == MM_INPUT ? 2 : 1) + partial;
    const unsigned char *at_a, *at_b;
    auto locate = [&](int s) {
        long t;
        if constexpr (MODE == MM_INPUT) {
            const bool second = s < partial ? s == 1 : s - partial >= whole;
            t = s < partial ? whole : s - partial - (second ? whole : 0);
            at_a = pA + (t + (second ? g.half / BK : 0)) * ROW_BYTES;
            at_b = pB + (second ? to_up : 0) + t * BK * pitch_b;
        } else {
            t = s < partial ? whole : s - partial;
            at_a = pA + t * (A_ACROSS ? BK * pitch_a : (long)ROW_BYTES);
            at_b = pB + t * (B_ACROSS ? BK * pitch_b : (long)ROW_BYTES);
        }
        at_a = uniform_ptr(at_a);
        at_b = uniform_ptr(at_b);
    };
    const unsigned lds_base = __builtin_amdgcn_readfirstlane((unsigned)(size_t)lds + wave * 1024);
    constexpr int NIA = la.NI, NI = la.NI + lb.NI;
    auto to = [&](int q) { return lds_base + (q < NIA ? q * NW * 1024 : A_BYTES + (q - NIA) * NW * 1024); };
    auto fetch_first = [&](int s) {                        // K-tile s into stage s, whole or not
        locate(s);
#pragma unroll
        for (int q = 0; q < NI; ++q) {
            const unsigned char* inside = q < NIA ? at_a + la.off[q < NIA ? q : 0] : at_b + lb.off[q < NIA ? 0 : q - NIA];
            const bool exists = s >= partial || ((q < NIA ? la.tail_in >> q : lb.tail_in >> (q - NIA)) & 1u) != 0;
            dma_to_lds_addr(exists ? inside : (const unsigned char*)kZeroChunk, to(q) + s * STAGE);
        }
    };
    auto fetch = [&](int q, unsigned stage) {
        if (q < NIA) dma_to_lds(at_a, la.off[q < NIA ? q : 0], to(q) + stage);
        else dma_to_lds(at_b, lb.off[q < NIA ? 0 : q - NIA], to(q) + stage);
    };

    Fragments<ES, A_ACROSS, BM, TM> ra(0, wm * WTM, fi, fq);
    Fragments<ES, B_ACROSS, BN, TN> rb(A_BYTES, wn * WTN, fi, fq);
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    u32x4 fa[TM], fb[2][TN];

    fetch_first(0);
    if (nk > 1) {
        fetch_first(1);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NI) : "memory");
    } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[0][j] = rb.load(lds, 0, j);
#pragma unroll
    for (int i = 0; i < TM; ++i) fa[i] = ra.load(lds, 0, i);
    int step = STAGE;
    // One K-tile: its first half's MFMAs while the second half's fragments come in, the boundary, its second half's while the next tile's come in (behind the last
    // tile they are of a stage that is not looked at any more) and, with MORE, the one after that is asked for.
    auto tile = [&](int kt, auto more) {
        constexpr bool MORE = decltype(more)::value;
        const unsigned stage = step > 0 ? 0 : STAGE;
        if constexpr (MORE) locate(kt + 2);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
            for (int i = 0; i < TM; ++i) {
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = gated_mma<DT>(fb[ks][j], fa[i], acc[i][j]);
                __builtin_amdgcn_sched_barrier(0);
                fa[i] = ra.load(lds, ks ^ 1, i);
#pragma unroll
                for (int j = i * TN / TM; j < (i + 1) * TN / TM; ++j) fb[ks ^ 1][j] = rb.load(lds, ks ^ 1, j);
                if (MORE && ks == 1)
#pragma unroll
                    for (int q = i * NI / TM; q < (i + 1) * NI / TM; ++q) fetch(q, stage);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (ks == 0) {
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                __syncthreads();
                ra.step(step);
                rb.step(step);
                step = -step;
            }
        }
    };
    int kt = 0;
    for (; kt + 2 < nk; ++kt) tile(kt, std::true_type{});
    for (; kt < nk; ++kt) tile(kt, std::false_type{});
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();                                       // the stages are not read any more

    const long row0 = m0 + wm * WTM;
    if constexpr (MODE != MM_FORWARD) {
        constexpr int STRIDE = GATED_STRIP_ROW<TN>;
        static_assert(NW * 32 * STRIDE <= 2 * STAGE, "strips");
        unsigned char* strip = lds + wave * (32 * STRIDE);
        void* const C = of_up != 0 ? g.C1 : g.C0;
        const long rows = MODE == MM_INPUT ? g.M : g.N, col0 = n0 + wn * WTN;
#pragma unroll
        for (int i = 0; i < TM; i += 2) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int j = 0; j < TN; ++j) *reinterpret_cast<f32x4*>(strip + (16 * k + fi) * STRIDE + (16 * j + 4 * fq) * 4) = acc[i + k][j];
            if (g.stream) put_strip<DT, 16 * TN, STRIDE, ST_STREAM>(strip, C, g.K, row0 + 16 * i, rows, col0, g.K, lane);
            else put_strip<DT, 16 * TN, STRIDE, ST_PLAIN>(strip, C, g.K, row0 + 16 * i, rows, col0, g.K, lane);
        }
    } else {
        constexpr int PAIRS = TN / 2, STRIDE = GATED_STRIP_ROW<PAIRS>;
        constexpr int STRIPS = NW * 32 * STRIDE;
        static_assert(STRIPS + 2 * WN * BM * 4 <= 2 * STAGE, "strips, and the largest magnitudes of rows");
        unsigned char* strip = lds + wave * (32 * STRIDE);
        const long col0 = n0 + wn * (WTN / 2);
        // 32 rows of what f(accumulators of a gate, of an up) gives, through the strip
        auto put = [&](void* C, int i, const auto& f) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int p = 0; p < PAIRS; ++p) {
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = f(acc[i + k][2 * p][e], acc[i + k][2 * p + 1][e]);
                    *reinterpret_cast<f32x4*>(strip + (16 * k + fi) * STRIDE + (16 * p + 4 * fq) * 4) = v;
                }
            if (g.stream) put_strip<DT, 16 * PAIRS, STRIDE, ST_STREAM>(strip, C, g.N, row0 + 16 * i, g.M, col0, g.N, lane);
            else put_strip<DT, 16 * PAIRS, STRIDE, ST_PLAIN>(strip, C, g.N, row0 + 16 * i, g.M, col0, g.N, lane);
        };
#pragma unroll
        for (int i = 0; i < TM; i += 2) {
            if (g.activation == SP_ACT_SILU) put(g.C0, i, [](float a, float u) { return gated_activation(a, SP_ACT_SILU) * u; });
            else if (g.activation == SP_ACT_GELU) put(g.C0, i, [](float a, float u) { return gated_activation(a, SP_ACT_GELU) * u; });
            else put(g.C0, i, [](float a, float u) { return gated_activation(a, SP_ACT_RELU) * u; });
            if (g.keep == KEEP_WHOLE) {
                put(g.gate, i, [](float a, float) { return a; });
                put(g.up, i, [](float, float u) { return u; });
            }
        }
        if constexpr (BN == 256) {
            if (g.keep != KEEP_F8) return;
            // blocks of one row and 128 columns, which are the tile's: the largest magnitudes of a row, as bits, from all lanes and waves that have some of it
            unsigned* const most = reinterpret_cast<unsigned*>(lds + STRIPS);            // [gate, up][wn][row]
            const long pitch = (g.N + 15) / 16 * 16, blocks = (g.N + QB - 1) / QB;
            const long left = g.N - col0 - 4 * fq;         // of this lane's columns 16 p .. 16 p + 3: those that exist
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int of = 0; of < 2; ++of) {
                    unsigned m = 0;
#pragma unroll
                    for (int p = 0; p < PAIRS; ++p)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (16 * p + e < left) m = max_u32(m, __float_as_uint(acc[i][2 * p + of][e]) & 0x7fffffffu);
                    m = max_u32(m, __shfl_xor(m, 16, WAVE));
                    m = max_u32(m, __shfl_xor(m, 32, WAVE));
                    if (fq == 0) most[(of * WN + wn) * BM + wm * WTM + 16 * i + fi] = m;
                }
            __syncthreads();
            constexpr int BYTES = 16 * PAIRS, LANES = BYTES / 16, ROWS = 64 / LANES, STRIDE8 = BYTES + 16;     // of a strip of bytes
            static_assert(32 % ROWS == 0 || ROWS > 32, "a strip in whole passes");
#pragma unroll
            for (int i = 0; i < TM; i += 2)
#pragma unroll
                for (int of = 0; of < 2; ++of) {
                    unsigned char* const q = (unsigned char*)(of != 0 ? g.up : g.gate);
                    float* const scales = of != 0 ? g.up_scale : g.gate_scale;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const int row = wm * WTM + 16 * (i + k) + fi;
                        unsigned m = most[of * WN * BM + row];
#pragma unroll
                        for (int w = 1; w < WN; ++w) m = max_u32(m, most[(of * WN + w) * BM + row]);
                        BlockScale s;
                        s.set<SP_F8_E4M3>(m);
                        if (wn == 0 && fq == 0 && m0 + row < g.M) scales[(m0 + row) * blocks + tn] = s.scale;
#pragma unroll
                        for (int p = 0; p < PAIRS; ++p) {
                            const f32x4& v = acc[i + k][2 * p + of];
                            const unsigned bytes = first_bytes(pack_f8<SP_F8_E4M3>(s(v[0]), s(v[1]), s(v[2]), s(v[3])), left - 16 * p);
                            *reinterpret_cast<unsigned*>(strip + (16 * k + fi) * STRIDE8 + 16 * p + 4 * fq) = bytes;
                        }
                    }
                    const int er = lane / LANES, ec = lane % LANES * 16;
#pragma unroll
                    for (int r = er; r < 32; r += ROWS) {
                        const u32x4 v = *reinterpret_cast<const u32x4*>(strip + r * STRIDE8 + ec);
                        const long row = row0 + 16 * i + r;
                        if (row < g.M && col0 + ec < pitch) *reinterpret_cast<u32x4*>(q + row * pitch + col0 + ec) = v;
                    }
                }
        }
    }
}

// ---- dg and du ----
struct GatedGradArgs {
    const void *dC, *gate, *up;
    const float *gate_scale, *up_scale;
    void* out;                    // M x 2 half
    long M, N, half;
    int activation;
};

// Eight columns of a row a lane.  F8: gate and up are e4m3 blocks.
template <int DT, bool F8>
__global__ __launch_bounds__(256) void gated_grad_kernel(const GatedGradArgs g) {
    constexpr int P = PER16<DT>, PIECES = 8 / P;
    const unsigned per_row = (unsigned)(g.half / 8), at = blockIdx.x * 256u + threadIdx.x, row_ = at / per_row;
    const long row = row_, col = (long)(at - row_ * per_row) * 8, left = g.N - col;
    if (row >= g.M) return;
    float dg[8], du[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) dg[e] = du[e] = 0.f;
    if (left > 0) {
        u32x4 raw[PIECES];
#pragma unroll
        for (int p = 0; p < PIECES; ++p) raw[p] = load16<DT>(g.dC, row * g.N + col + p * P, left - p * P);
        float a[8], u[8];
        if constexpr (F8) {
            const long pitch = (g.N + 15) / 16 * 16, blocks = (g.N + QB - 1) / QB;
            const u32x2 qa = *reinterpret_cast<const u32x2*>((const unsigned char*)g.gate + row * pitch + col);
            const u32x2 qu = *reinterpret_cast<const u32x2*>((const unsigned char*)g.up + row * pitch + col);
            const float sa = g.gate_scale[row * blocks + col / QB], su = g.up_scale[row * blocks + col / QB];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x2 a0 = __builtin_amdgcn_cvt_pk_f32_fp8(qa[h], false), a1 = __builtin_amdgcn_cvt_pk_f32_fp8(qa[h], true);
                const f32x2 u0 = __builtin_amdgcn_cvt_pk_f32_fp8(qu[h], false), u1 = __builtin_amdgcn_cvt_pk_f32_fp8(qu[h], true);
                a[4 * h] = a0.x * sa, a[4 * h + 1] = a0.y * sa, a[4 * h + 2] = a1.x * sa, a[4 * h + 3] = a1.y * sa;
                u[4 * h] = u0.x * su, u[4 * h + 1] = u0.y * su, u[4 * h + 2] = u1.x * su, u[4 * h + 3] = u1.y * su;
            }
        } else {
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                const u32x4 ra = load16<DT>(g.gate, row * g.N + col + p * P, left - p * P), ru = load16<DT>(g.up, row * g.N + col + p * P, left - p * P);
#pragma unroll
                for (int e = 0; e < P; ++e) a[p * P + e] = element<DT>(ra, e), u[p * P + e] = element<DT>(ru, e);
            }
        }
        auto each = [&](int kind) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float act, slope;
                activation_and_slope(a[e], kind, act, slope);
                const float d = element<DT>(raw[e / P], e % P);
                dg[e] = e < left ? d * u[e] * slope : 0.f;
                du[e] = e < left ? d * act : 0.f;
            }
        };
        if (g.activation == SP_ACT_SILU) each(SP_ACT_SILU);
        else if (g.activation == SP_ACT_GELU) each(SP_ACT_GELU);
        else each(SP_ACT_RELU);
    }
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        float v[P], w[P];
#pragma unroll
        for (int e = 0; e < P; ++e) v[e] = dg[p * P + e], w[e] = du[p * P + e];
        store16<DT>(g.out, row * 2 * g.half + col + p * P, P, v);
        store16<DT>(g.out, row * 2 * g.half + g.half + col + p * P, P, w);
    }
}

// ---- host side -------------------------------------------------------------------------------

static long gated_ceil(long a, long b) { return (a + b - 1) / b; }

template <int DT, int MODE, int BM, int BN, int WM, int WN>
static int launch_mm(const char* what, GatedArgs g, hipStream_t stream) {
    auto kernel = gated_mm_kernel<DT, MODE, BM, BN, WM, WN>;
    constexpr int lds_bytes = 2 * (BM + BN) * ROW_BYTES;
    const long tiles_m = MODE == MM_WEIGHTS ? 2 * gated_ceil(g.N, BM) : gated_ceil(g.M, BM);
    const long tiles_n = MODE == MM_FORWARD ? gated_ceil(g.N, BN / 2) : gated_ceil(g.K, BN);
    if (tiles_m >= 1l << 31 || tiles_n >= 1l << 31 || tiles_m * tiles_n >= 1l << 31 || tiles_m * tiles_n * (WM * WN * 64) >= 1l << 32) return fail(SP_ERR_SHAPE, "%s: too large", what);
    if (const int rc = ensure_dynamic_lds((const void*)kernel, lds_bytes); rc != SP_OK) return rc;
    g.tiles_m = (int)tiles_m;
    g.tiles_n = (int)tiles_n;
    g.group_m = 4;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles_m * tiles_n)), dim3(WM * WN * 64), lds_bytes, stream, g);
    return check_launch(what);
}

template <int DT>
static int gated_forward(const GatedArgs& g, hipStream_t stream) {
    const long cus = device_cu_count();
    auto tiles = [&](long bm) { return gated_ceil(g.M, bm) * gated_ceil(g.N, 128); };
    if (tiles(256) * 5 >= cus * 4) return launch_mm<DT, MM_FORWARD, 256, 256, 4, 2>("sp_gemm_abt_gated", g, stream);
    if (tiles(128) * 5 >= cus * 4) return launch_mm<DT, MM_FORWARD, 128, 256, 4, 2>("sp_gemm_abt_gated", g, stream);
    return launch_mm<DT, MM_FORWARD, 64, 256, 2, 2>("sp_gemm_abt_gated", g, stream);
}

template <int DT, int MODE>
static int gated_backward_product(const GatedArgs& g, hipStream_t stream) {
    const long cus = device_cu_count(), rows = MODE == MM_INPUT ? g.M : g.N;
    auto tiles = [&](long b) { return gated_ceil(rows, b) * (MODE == MM_WEIGHTS ? 2 : 1) * gated_ceil(g.K, b); };
    if (tiles(256) * 5 >= cus * 4) return launch_mm<DT, MODE, 256, 256, 2, 4>("sp_gemm_abt_gated_backward", g, stream);
    if (tiles(128) * 5 >= cus * 4) return launch_mm<DT, MODE, 128, 128, 2, 2>("sp_gemm_abt_gated_backward", g, stream);
    return launch_mm<DT, MODE, 64, 64, 2, 2>("sp_gemm_abt_gated_backward", g, stream);
}

template <int DT>
static int gated_backward(const GatedArgs& input, const GatedArgs& weights, const GatedGradArgs& grad, bool f8, hipStream_t stream) {
    const long pieces = grad.M * (grad.half / 8);
    const dim3 blocks((unsigned)gated_ceil(pieces, 256));
    if (f8) hipLaunchKernelGGL((gated_grad_kernel<DT, true>), blocks, dim3(256), 0, stream, grad);
    else hipLaunchKernelGGL((gated_grad_kernel<DT, false>), blocks, dim3(256), 0, stream, grad);
    if (const int rc = check_launch("sp_gemm_abt_gated_backward"); rc != SP_OK) return rc;
    if (input.C0 != nullptr)
        if (const int rc = gated_backward_product<DT, MM_INPUT>(input, stream); rc != SP_OK) return rc;
    return weights.C0 != nullptr ? gated_backward_product<DT, MM_WEIGHTS>(weights, stream) : SP_OK;
}

namespace {
struct GatedKernelNames {
    GatedKernelNames() {
        register_kernel("gated_forward_256x256", (const void*)gated_mm_kernel<SP_BF16, MM_FORWARD, 256, 256, 4, 2>, 512);
        register_kernel("gated_input_256x256", (const void*)gated_mm_kernel<SP_BF16, MM_INPUT, 256, 256, 2, 4>, 512);
        register_kernel("gated_weights_256x256", (const void*)gated_mm_kernel<SP_BF16, MM_WEIGHTS, 256, 256, 2, 4>, 512);
    }
} gated_kernel_names;
}  // namespace

}  // namespace sp

using namespace sp;

// Columns of either half of the backward pass's workspace: whole K-tiles, of 64 numbers of 16 bits (two of f32).
static int64_t gated_half(int64_t N) { return (N + 63) / 64 * 64; }

static int gated_sizes(const char* fn, int dtype, int activation, int kept, bool keeps, int64_t M, int64_t N, int64_t K) {
    if (dtype != SP_F32 && dtype != SP_F16 && dtype != SP_BF16) return fail(SP_ERR_DTYPE, "%s: dtype must be f32, f16 or bf16, got %d", fn, dtype);
    if (keeps && kept != dtype && kept != SP_F8_E4M3) return fail(SP_ERR_DTYPE, "%s: gate and up are kept in the operands' type or in e4m3, got %d", fn, kept);
    if (activation != SP_ACT_SILU && activation != SP_ACT_GELU && activation != SP_ACT_RELU) return fail(SP_ERR_ARG, "%s: unknown activation %d", fn, activation);
    if (M <= 0 || N <= 0 || K <= 0) return fail(SP_ERR_SHAPE, "%s: M, N, K must be positive (got %lld, %lld, %lld)", fn, (long long)M, (long long)N, (long long)K);
    const int per = dtype == SP_F32 ? 4 : 8;
    if (K % per != 0) return fail(SP_ERR_SHAPE, "%s: K must be a multiple of %d (16-byte rows), got %lld", fn, per, (long long)K);
    // a tile's rows (256, or 64 across) are addressed by 32-bit offsets
    const int64_t most = ((int64_t)1 << 24) / (dtype == SP_F32 ? 4 : 2);
    if (K > most / 2 || N > most / 4 || M > INT32_MAX) return fail(SP_ERR_SHAPE, "%s: too large", fn);
    return SP_OK;
}

extern "C" int sp_gemm_abt_gated(int dtype, int activation, const void* A, const void* B_gate, const void* B_up, void* C, int kept_dtype, void* gate, float* gate_scale, void* up,
                                 float* up_scale, int64_t M, int64_t N, int64_t K, void* stream) {
    SP_REQUIRE_PTR(A);
    SP_REQUIRE_PTR(B_gate);
    SP_REQUIRE_PTR(B_up);
    SP_REQUIRE_PTR(C);
    SP_OPTIONAL_PTR(gate);
    SP_OPTIONAL_PTR(gate_scale);
    SP_OPTIONAL_PTR(up);
    SP_OPTIONAL_PTR(up_scale);
    const bool keeps = gate != nullptr || up != nullptr;
    if (const int rc = gated_sizes(__func__, dtype, activation, kept_dtype, keeps, M, N, K); rc != SP_OK) return rc;
    const bool f8 = keeps && kept_dtype == SP_F8_E4M3;
    if (keeps && (gate == nullptr || up == nullptr)) return fail(SP_ERR_NULL, "sp_gemm_abt_gated: gate and up go together");
    if (f8 && (gate_scale == nullptr || up_scale == nullptr)) return fail(SP_ERR_NULL, "sp_gemm_abt_gated: numbers and their scales go together");
    if (const int rc = require_gfx950(__func__); rc != SP_OK) return rc;
    GatedArgs g{};
    g.A = (const unsigned char*)A; g.B0 = (const unsigned char*)B_gate; g.B1 = (const unsigned char*)B_up; g.C0 = C; g.gate = gate; g.up = up;
    g.gate_scale = gate_scale; g.up_scale = up_scale; g.M = M; g.N = N; g.K = K; g.activation = activation; g.keep = f8 ? KEEP_F8 : keeps ? KEEP_WHOLE : KEEP_NONE;
    g.stream = M * N * (dtype == SP_F32 ? 4 : 2) > (int64_t)32 << 20;
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == SP_F32) return gated_forward<SP_F32>(g, st);
    if (dtype == SP_F16) return gated_forward<SP_F16>(g, st);
    return gated_forward<SP_BF16>(g, st);
}

extern "C" int64_t sp_gemm_abt_gated_backward_workspace_bytes(int dtype, int64_t M, int64_t N) {
    if (M <= 0 || N <= 0 || M > INT32_MAX || N > (int64_t)1 << 24) return 0;
    return M * 2 * gated_half(N) * (dtype == SP_F32 ? 4 : 2);
}

extern "C" int sp_gemm_abt_gated_backward(int dtype, int activation, const void* dC, const void* A, const void* B_gate, const void* B_up, int kept_dtype, const void* gate,
                                          const float* gate_scale, const void* up, const float* up_scale, void* dA, void* dB_gate, void* dB_up, int64_t M, int64_t N, int64_t K,
                                          void* workspace, int64_t workspace_bytes, void* stream) {
    SP_REQUIRE_PTR(dC);
    SP_REQUIRE_PTR(A);
    SP_REQUIRE_PTR(B_gate);
    SP_REQUIRE_PTR(B_up);
    SP_REQUIRE_PTR(gate);
    SP_REQUIRE_PTR(up);
    SP_OPTIONAL_PTR(gate_scale);
    SP_OPTIONAL_PTR(up_scale);
    SP_OPTIONAL_PTR(dA);
    SP_OPTIONAL_PTR(dB_gate);
    SP_OPTIONAL_PTR(dB_up);
    SP_REQUIRE_PTR(workspace);
    if (const int rc = gated_sizes(__func__, dtype, activation, kept_dtype, true, M, N, K); rc != SP_OK) return rc;
    const bool f8 = kept_dtype == SP_F8_E4M3;
    if (f8 && (gate_scale == nullptr || up_scale == nullptr)) return fail(SP_ERR_NULL, "sp_gemm_abt_gated_backward: numbers and their scales go together");
    if ((dB_gate == nullptr) != (dB_up == nullptr)) return fail(SP_ERR_ARG, "sp_gemm_abt_gated_backward: dB_gate and dB_up: both or neither");
    if (dA == nullptr && dB_gate == nullptr) return fail(SP_ERR_NULL, "sp_gemm_abt_gated_backward: no gradient is wanted");
    const int64_t half = gated_half(N);
    if (M * (half / 8) > ((int64_t)1 << 32) - 256) return fail(SP_ERR_SHAPE, "sp_gemm_abt_gated_backward: too large");
    if (workspace_bytes < sp_gemm_abt_gated_backward_workspace_bytes(dtype, M, N))
        return fail(SP_ERR_ARG, "sp_gemm_abt_gated_backward: workspace of %lld bytes, %lld are needed", (long long)workspace_bytes,
                    (long long)sp_gemm_abt_gated_backward_workspace_bytes(dtype, M, N));
    if (const int rc = require_gfx950(__func__); rc != SP_OK) return rc;
    GatedGradArgs grad{};
    grad.dC = dC; grad.gate = gate; grad.up = up; grad.gate_scale = gate_scale; grad.up_scale = up_scale; grad.out = workspace; grad.M = M; grad.N = N; grad.half = half;
    grad.activation = activation;
    const int es = dtype == SP_F32 ? 4 : 2;
    GatedArgs input{}, weights{};
    input.A = (const unsigned char*)workspace; input.B0 = (const unsigned char*)B_gate; input.B1 = (const unsigned char*)B_up; input.C0 = dA; input.M = M; input.N = N; input.K = K;
    input.half = half; input.stream = M * K * es > (int64_t)32 << 20;
    weights = input;
    weights.B0 = (const unsigned char*)A; weights.B1 = nullptr; weights.C0 = dB_gate; weights.C1 = dB_up; weights.stream = 2 * N * K * es > (int64_t)32 << 20;
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == SP_F32) return gated_backward<SP_F32>(input, weights, grad, f8, st);
    if (dtype == SP_F16) return gated_backward<SP_F16>(input, weights, grad, f8, st);
    return gated_backward<SP_BF16>(input, weights, grad, f8, st);
}
