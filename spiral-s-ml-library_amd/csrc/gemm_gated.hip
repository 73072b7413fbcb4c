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
// All products: tiles of LDS in a ring of stages that DMA fills, 128 bytes of K (of a row, or of K rows) a stage.  A wave walks its TM rows of fragments; the fragment of a
// row is replaced by the next half stage's once its MFMAs are issued, the B fragments have two sets.  The boundary between two stages stands in the middle: everything
// of a stage is in registers then, and the next one has landed.
// K may end anywhere: what is missing of the last K-tile comes from zeros, and that tile goes first, so that the loop has whole ones only.
#include "f8_blocks.h"
#include "overlap.h"

namespace sp {

enum { MM_FORWARD, MM_INPUT, MM_WEIGHTS };
enum { KEEP_NONE, KEEP_WHOLE, KEEP_F8 };
template <int DT>
constexpr int STAGES_64 = DT == SP_F32 ? 2 : 4;            // of tiles of 64 x 64: of f32, whose MFMAs take longest, five workgroups to a unit
constexpr unsigned ROTATE = 7;      // odd: it meets every one of a power of two of K-tiles

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
    int stream;                   // C does not stay in the caches; bit 1: nor do gate and up
    float* parts;                 // backward: partial sums of several workgroups, all of a result (of both weights' gradients) each
};

__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504088896340736f)); }
// Phi(g) of the normal distribution, and e^(-g^2 / 2).  Not (1 + erf(g / sqrt 2)) / 2, which loses the lower tail: half a percent of GELU at -4.5 and the whole of it at -5.6.
// Phi(-a) e^(a^2 / 2) is t times a polynomial of t = 1 / (1 + 0.35 a), fitted by weighted least squares to a relative error of 3.2e-8 where Phi is a f32 (a to 13.3); in f32, with the
// exponential, (1.3 g^2 + 11) roundings off at most.  It has no branch: 8192 x 2048 x 8192 bf16 forward with GELU takes 415 us, 440 with erff, 460 with erfcf.
__device__ __forceinline__ float below_normal(float g, float& bell) {
    constexpr float C[9] = {0.13962166f, 0.13985756f, 0.119863085f, 0.105392143f, -0.0228434224f, 0.158796564f, -0.255391002f, 0.143818408f, -0.0291150156f};
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(fabsf(g), 0.35f, 1.f));
    float v = C[8];
#pragma unroll
    for (int i = 7; i >= 0; --i) v = __builtin_fmaf(v, t, C[i]);
    bell = __builtin_amdgcn_exp2f(g * g * -0.72134752044448170368f);
    const float tail = bell * (v * t);
    return g < 0.f ? tail : 1.f - tail;
}
__device__ __forceinline__ float gated_activation(float g, int kind) {
    if (kind == SP_ACT_SILU) return g * sigmoid(g);
    if (kind == SP_ACT_GELU) {
        float bell;
        return g * below_normal(g, bell);
    }
    return g < 0.f ? 0.f : g;                              // (a NaN stays)
}
// act(g) and act'(g).
__device__ __forceinline__ void activation_and_slope(float g, int kind, float& act, float& slope) {
    if (kind == SP_ACT_SILU) {
        const float s = sigmoid(g);
        act = g * s;
        slope = s * __builtin_fmaf(g, 1.f - s, 1.f);
    } else if (kind == SP_ACT_GELU) {
        float bell;
        const float below = below_normal(g, bell);
        act = g * below;
        slope = __builtin_fmaf(g * 0.39894228040143267794f, bell, below);
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
    static_assert(W >= 64, "four units a row");
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
    static_assert(R / 8 % NW == 0, "blocks split evenly over the waves");
    unsigned off[NI];
    unsigned tail_in = 0;                                  // bit q: this lane's 16 bytes of the partial K-tile exist
    // pitch: bytes from row to row; left: rows (along) or 16-byte chunks of columns (across) from the tile's first one to the last; tail: K of the partial tile.
    // PAIR: rows of two matrices in turn, 16 and 16; block b is of number b / 2 % 2 (a wave's blocks are all of one of them where NW is a multiple of 4).
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

// A wave's strip of LDS through which sixteen rows of COLS columns leave as 16-byte pieces, side by side along the rows; the pad spreads a column over the banks.
template <int DT, int COLS>
struct Strip {
    static constexpr int E = ELEM_BYTES<DT>, P = PER16<DT>, ROW = COLS * E + 16, BYTES = 16 * ROW, LANES = COLS / P, ROWS = 64 / LANES;
    // four columns of row fi
    static __device__ __forceinline__ void set(unsigned char* strip, int fi, int col, const f32x4& v) {
        if constexpr (E == 4) *reinterpret_cast<f32x4*>(strip + fi * ROW + col * 4) = v;
        else *reinterpret_cast<u32x2*>(strip + fi * ROW + col * 2) = u32x2{pack_halves<DT>(v[0], v[1]), pack_halves<DT>(v[2], v[3])};
    }
    template <int POLICY>
    static __device__ __forceinline__ void put(const unsigned char* strip, void* C, long pitch, long row0, long rows, long col0, long cols, int lane) {
        const int er = lane / LANES, ec = lane % LANES * P;
#pragma unroll
        for (int r = 0; r < 16; r += ROWS) {
            if (ROWS > 16 && er >= 16) break;
            const u32x4 v = *reinterpret_cast<const u32x4*>(strip + (r + er) * ROW + ec * E);
            const long row = row0 + r + er, left = cols - col0 - ec;
            unsigned char* q = (unsigned char*)C + (row * pitch + col0 + ec) * E;
            if (row >= rows || left <= 0) continue;
            if (left >= P) {
                store_c<POLICY, E>(q, v);
                continue;
            }
#pragma unroll
            for (int i = 0; i < P - 1; ++i)
                if (i < left) {
                    if constexpr (E == 4) ((unsigned*)q)[i] = v[i];
                    else ((unsigned short*)q)[i] = (unsigned short)(v[i >> 1] >> (16 * (i & 1)));
                }
        }
    }
};

// Bound by the matrix pipe and, in large products, by the part's power: 8192 x 4096 x 8192 bf16 takes 812 us, 1.35 PFLOP/s with the pipe busy 70 % of all cycles, and the gradients of
// 8192 x 2048 x 8192 782 us, 1.41 PFLOP/s; f32, 4096 x 2048 x 4096, 955 us, 144 TFLOP/s.  Large tiles for the few bytes from LDS and L2 to an MFMA, eight waves for two on a SIMD; four waves on 256 x 256,
// loads between a row's MFMAs, raised wave priorities and other groups of the walk gave nothing, a workgroup that goes on to a next tile while its results leave spilled.  So results leave bare:
// both factors of 8192 x 2048 x 8192 kept whole cost 36 us beside 375, in 8-bit blocks (5008 x 2048 x 5461) 21 beside 171.
// One tile, or this workgroup's share of its K-tiles: with parts > 1 the sums go to a workspace in f32 (gated_join_kernel adds them up).
template <int DT, int MODE, int BM, int BN, int WM, int WN, int NS>
__device__ __forceinline__ void gated_mm(const GatedArgs& g, unsigned block, unsigned part, unsigned parts) {
    constexpr int ES = ELEM_BYTES<DT>, BK = ROW_BYTES / ES, NW = WM * WN, WTM = BM / WM, WTN = BN / WN, TM = WTM / 16, TN = WTN / 16;
    constexpr bool A_ACROSS = MODE == MM_WEIGHTS, B_ACROSS = MODE != MM_FORWARD;
    constexpr int A_BYTES = BM * ROW_BYTES, STAGE = (BM + BN) * ROW_BYTES;
    static_assert(TN % 2 == 0, "a gate's fragment and an up's");
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN, fi = lane & 15, fq = lane >> 4;
    int tm, tn;
    gated_tile_of_block(block, g.tiles_m, g.tiles_n, g.group_m, tm, tn);

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
    const int whole = (int)(inner / BK), partial = tail != 0 ? (MODE == MM_INPUT ? 2 : 1) : 0, all = whole * (MODE == MM_INPUT ? 2 : 1) + partial;
    const int first = (int)((unsigned)all * part / parts), nk = (int)((unsigned)all * (part + 1) / parts) - first;
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
    // from one whole K-tile to number s
    const long step_a = A_ACROSS ? BK * pitch_a : (long)ROW_BYTES, step_b = B_ACROSS ? BK * pitch_b : (long)ROW_BYTES;
    auto advance = [&](int s) {
        at_a += step_a;
        at_b += step_b;
        if (MODE == MM_INPUT && s == partial + whole) locate(s);
    };
    const unsigned lds_base = __builtin_amdgcn_readfirstlane((unsigned)(size_t)lds + wave * 1024);
    constexpr int NIA = la.NI, NI = la.NI + lb.NI;
    auto to = [&](int q) { return lds_base + (q < NIA ? q * NW * 1024 : A_BYTES + (q - NIA) * NW * 1024); };
    auto fetch_first = [&](int st) {                       // K-tile `st` of this workgroup into stage st, whole or not
        const int s = first + st;
        locate(s);
#pragma unroll
        for (int q = 0; q < NI; ++q) {
            const unsigned char* inside = q < NIA ? at_a + la.off[q < NIA ? q : 0] : at_b + lb.off[q < NIA ? 0 : q - NIA];
            const bool exists = s >= partial || ((q < NIA ? la.tail_in >> q : lb.tail_in >> (q - NIA)) & 1u) != 0;
            dma_to_lds_addr(exists ? inside : (const unsigned char*)kZeroChunk, to(q) + st * STAGE);
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

#pragma unroll
    for (int st = 0; st < NS; ++st)
        if (st < nk) fetch_first(st);
    if (nk >= NS) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 1) * NI) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[0][j] = rb.load(lds, 0, j);
#pragma unroll
    for (int i = 0; i < TM; ++i) fa[i] = ra.load(lds, 0, i);
    unsigned stage = 0;                                    // where the K-tile that is being multiplied begins
    // One K-tile: its first half's MFMAs while the second half's fragments come in, the boundary, its second half's while the next tile's come in (behind the last
    // tile they are of a stage that is not looked at any more) and, with MORE, the one NS tiles on is asked for.
    auto tile = [&](int kt, auto more) {
        constexpr bool MORE = decltype(more)::value;
        const unsigned released = stage;
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
                    for (int q = i * NI / TM; q < (i + 1) * NI / TM; ++q) fetch(q, released);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (ks == 0) {
                // tile kt + 1 has landed: the NS - 2 behind it may be on their way; near the end only "none" says it
                if constexpr (MORE) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NS - 2) * NI) : "memory");
                else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                __syncthreads();
                const int step = stage == (NS - 1) * STAGE ? -(NS - 1) * STAGE : STAGE;
                ra.step(step);
                rb.step(step);
                stage += step;
            }
        }
        if constexpr (MORE) advance(first + kt + NS + 1);
    };
    int kt = 0;
    if (nk > NS) locate(first + NS);                       // (whole: partial tiles are two at most)
    for (; kt + NS < nk; ++kt) tile(kt, std::true_type{});
    for (; kt < nk; ++kt) tile(kt, std::false_type{});
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();                                       // the stages are not read any more

    const long row0 = m0 + wm * WTM;
    if constexpr (MODE != MM_FORWARD) {
        static_assert(NW * Strip<SP_F32, 16 * TN>::BYTES <= 2 * STAGE, "strips");
        const long rows = MODE == MM_INPUT ? g.M : g.N, col0 = n0 + wn * WTN;
        auto put = [&](void* C, auto type, auto policy) {
            typedef Strip<decltype(type)::value, 16 * TN> S;
            unsigned char* strip = lds + wave * S::BYTES;
#pragma unroll
            for (int i = 0; i < TM; ++i) {
#pragma unroll
                for (int j = 0; j < TN; ++j) S::set(strip, fi, 16 * j + 4 * fq, acc[i][j]);
                S::template put<decltype(policy)::value>(strip, C, g.K, row0 + 16 * i, rows, col0, g.K, lane);
            }
        };
        if (parts > 1) put(g.parts + ((MODE == MM_INPUT ? part : 2 * part + of_up) * rows) * g.K, std::integral_constant<int, SP_F32>{}, std::integral_constant<int, ST_PLAIN>{});
        else if (g.stream) put(of_up != 0 ? g.C1 : g.C0, std::integral_constant<int, DT>{}, std::integral_constant<int, ST_STREAM>{});
        else put(of_up != 0 ? g.C1 : g.C0, std::integral_constant<int, DT>{}, std::integral_constant<int, ST_PLAIN>{});
    } else {
        constexpr int PAIRS = TN / 2;
        typedef Strip<DT, 16 * PAIRS> S;
        constexpr int STRIPS = NW * S::BYTES;
        static_assert(STRIPS + 2 * WN * BM * 4 <= 2 * STAGE, "strips, and the largest magnitudes of rows");
        unsigned char* strip = lds + wave * S::BYTES;
        const long col0 = n0 + wn * (WTN / 2);
        // sixteen rows of what f(accumulators of a gate, of an up) gives, through the strip
        auto put = [&](void* C, int stream, int i, const auto& f) {
#pragma unroll
            for (int p = 0; p < PAIRS; ++p) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = f(acc[i][2 * p][e], acc[i][2 * p + 1][e]);
                S::set(strip, fi, 16 * p + 4 * fq, v);
            }
            if (stream) S::template put<ST_STREAM>(strip, C, g.N, row0 + 16 * i, g.M, col0, g.N, lane);
            else S::template put<ST_PLAIN>(strip, C, g.N, row0 + 16 * i, g.M, col0, g.N, lane);
        };
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            if (g.activation == SP_ACT_SILU) put(g.C0, g.stream, i, [](float a, float u) { return gated_activation(a, SP_ACT_SILU) * u; });
            else if (g.activation == SP_ACT_GELU) put(g.C0, g.stream, i, [](float a, float u) { return gated_activation(a, SP_ACT_GELU) * u; });
            else put(g.C0, g.stream, i, [](float a, float u) { return gated_activation(a, SP_ACT_RELU) * u; });
            if (g.keep == KEEP_WHOLE) {
                put(g.gate, g.stream & 2, i, [](float a, float) { return a; });
                put(g.up, g.stream & 2, i, [](float, float u) { return u; });
            }
        }
        if (BN == 256 && g.keep == KEEP_F8) {
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
            constexpr int LANES = PAIRS, ROWS = 64 / LANES, STRIDE8 = 16 * PAIRS + 16;     // of a strip of bytes, 16 a lane
            static_assert(16 * STRIDE8 <= S::BYTES, "a strip of bytes");
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int of = 0; of < 2; ++of) {
                    unsigned char* const q = (unsigned char*)(of != 0 ? g.up : g.gate);
                    const int in_tile = wm * WTM + 16 * i + fi;
                    unsigned m = most[of * WN * BM + in_tile];
#pragma unroll
                    for (int w = 1; w < WN; ++w) m = max_u32(m, most[(of * WN + w) * BM + in_tile]);
                    BlockScale s;
                    s.set<SP_F8_E4M3>(m);
                    if (wn == 0 && fq == 0 && m0 + in_tile < g.M) (of != 0 ? g.up_scale : g.gate_scale)[(m0 + in_tile) * blocks + tn] = s.scale;
#pragma unroll
                    for (int p = 0; p < PAIRS; ++p) {
                        const f32x4& v = acc[i][2 * p + of];
                        *reinterpret_cast<unsigned*>(strip + fi * STRIDE8 + 16 * p + 4 * fq) = first_bytes(pack_f8<SP_F8_E4M3>(s(v[0]), s(v[1]), s(v[2]), s(v[3])), left - 16 * p);
                    }
                    const int er = lane / LANES, ec = lane % LANES * 16;
#pragma unroll
                    for (int r = 0; r < 16; r += ROWS) {
                        if (ROWS > 16 && er >= 16) break;
                        const u32x4 v = *reinterpret_cast<const u32x4*>(strip + (r + er) * STRIDE8 + ec);
                        const long row = row0 + 16 * i + r + er;
                        if (row < g.M && col0 + ec < pitch) *reinterpret_cast<u32x4*>(q + row * pitch + col0 + ec) = v;
                    }
                }
        }
    }
}

template <int DT, int BM, int BN, int WM, int WN, int NS>
__global__ __launch_bounds__(WM* WN * 64, 2) void gated_forward_kernel(const GatedArgs g) {
    gated_mm<DT, MM_FORWARD, BM, BN, WM, WN, NS>(g, blockIdx.x, 0, 1);
}

// Tiles of 256 x 256 and, below them, of 128 x 256: the last round of the large ones is seldom a full one, and the small ones fill the units that it leaves.
struct GatedRows {
    GatedArgs large, small;
    unsigned large_blocks;
};
template <int DT>
__global__ __launch_bounds__(512, 2) void gated_forward_rows_kernel(const GatedRows p) {
    if (blockIdx.x < p.large_blocks) gated_mm<DT, MM_FORWARD, 256, 256, 4, 2, 2>(p.large, blockIdx.x, 0, 1);
    else gated_mm<DT, MM_FORWARD, 128, 256, 4, 2, 3>(p.small, blockIdx.x - p.large_blocks, 0, 1);
}

// Both products of the backward pass in one launch, or one of them: neither waits for the other, and the tiles of one fill the units that the other's leave.
struct GatedPair {
    GatedArgs input, weights;
    unsigned first_blocks;        // of those that begin first
    int input_first;
    unsigned input_parts, weights_parts;
};
template <typename Input, typename Weights>
__device__ __forceinline__ void gated_pair(const GatedPair& p, const Input& input, const Weights& weights) {
    const bool first = blockIdx.x < p.first_blocks;
    const unsigned at = first ? blockIdx.x : blockIdx.x - p.first_blocks;
    if (first == (p.input_first != 0)) {
        const unsigned tiles = (unsigned)(p.input.tiles_m * p.input.tiles_n), part = p.input_parts > 1 ? at / tiles : 0;
        input(p.input, at - part * tiles, part, p.input_parts);
    } else {
        const unsigned tiles = (unsigned)(p.weights.tiles_m * p.weights.tiles_n), part = p.weights_parts > 1 ? at / tiles : 0;
        weights(p.weights, at - part * tiles, part, p.weights_parts);
    }
}
template <int DT, int BM, int BN, int WM, int WN, int NS>
__global__ __launch_bounds__(WM* WN * 64, 2) void gated_backward_kernel(const GatedPair p) {
    gated_pair(p, [](const GatedArgs& g, unsigned block, unsigned part, unsigned parts) { gated_mm<DT, MM_INPUT, BM, BN, WM, WN, NS>(g, block, part, parts); },
               [](const GatedArgs& g, unsigned block, unsigned part, unsigned parts) { gated_mm<DT, MM_WEIGHTS, BM, BN, WM, WN, NS>(g, block, part, parts); });
}

// ---- few rows, or few tiles ----
// One tile of (16 TM) x (16 TN) sums on four waves: wave w takes K-tiles w, w + 4, ... through an LDS ring of NS stages of its own, so no wave waits for another inside the loop, and the four
// partial sums meet in LDS, in a fixed order.  Forward and the gradient of A; of the weights there are always many.
// Bound by the weights' way from HBM: 1 x 4096 x 8192 bf16, 134 MB, 24.2 us (5.5 TB/s); few K-tiles, 49 x 1000 x 2667 f16: 6.0 us, launch and latency.
// Several workgroups may share the K-tiles, too, as above.
template <int DT, int MODE, int TM, int TN, int NS>
__device__ __forceinline__ void gated_split(const GatedArgs& g, unsigned block, unsigned share, unsigned parts) {
    constexpr int KS = 4, ES = ELEM_BYTES<DT>, BK = ROW_BYTES / ES, BM = 16 * TM, BN = 16 * TN;
    constexpr bool B_ACROSS = MODE == MM_INPUT;
    constexpr int A_BYTES = BM * ROW_BYTES, STAGE = (BM + BN) * ROW_BYTES;
    static_assert(MODE == MM_FORWARD ? TN % 2 == 0 : MODE == MM_INPUT, "a gate's fragment and an up's");
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fi = lane & 15, fq = lane >> 4;
    int tm, tn;
    gated_tile_of_block(block, g.tiles_m, g.tiles_n, g.group_m, tm, tn);
    const long m0 = (long)tm * BM, n0 = (long)tn * (MODE == MM_FORWARD ? BN / 2 : BN);
    const long pitch_a = (MODE == MM_FORWARD ? g.K : 2 * g.half) * ES, pitch_b = g.K * ES;
    const long inner = MODE == MM_FORWARD ? g.K : g.N;
    const int tail = (int)(inner % BK), per_half = (int)((inner + BK - 1) / BK), all = per_half * (MODE == MM_INPUT ? 2 : 1);
    const int first = (int)((unsigned)all * share / parts), nk = (int)((unsigned)all * (share + 1) / parts) - first;
    Loader<ES, false, BM, 1> la;
    Loader<ES, B_ACROSS, BN, 1> lb;
    la.template set<false>(lane, 0, pitch_a, g.M - m0, MODE == MM_INPUT ? BK : tail);
    lb.template set<MODE == MM_FORWARD>(lane, 0, pitch_b, B_ACROSS ? (g.K - n0) * ES / 16 : g.N - n0, tail);
    constexpr int NIA = la.NI, NI = la.NI + lb.NI;
    static_assert((NS - 1) * NI < 64, "vmcnt counts to 63");
    const unsigned char* const pA = uniform_ptr(g.A + m0 * pitch_a);
    const unsigned char* const pB = uniform_ptr(g.B0 + n0 * (MODE == MM_FORWARD ? pitch_b : ES));
    const long to_up = g.B1 - g.B0;
    const unsigned my_lds = __builtin_amdgcn_readfirstlane((unsigned)(size_t)lds + wave * (NS * STAGE));
    auto fetch = [&](int t, unsigned stage) {
        const int second = MODE == MM_INPUT && t >= per_half ? 1 : 0, in_half = t - second * per_half;
        const unsigned char* const a = uniform_ptr(pA + (MODE == MM_INPUT ? in_half + second * (g.half / BK) : t) * ROW_BYTES);
        const unsigned char* const b = uniform_ptr(pB + (MODE == MM_INPUT ? second * to_up + in_half * (BK * pitch_b) : t * (long)ROW_BYTES));
        const unsigned char* const b_up = MODE == MM_FORWARD ? uniform_ptr(b + to_up) : b;
        const unsigned dst = my_lds + stage * STAGE;
        if (tail != 0 && in_half == per_half - 1) {
#pragma unroll
            for (int q = 0; q < NI; ++q) {
                const unsigned char* inside = q < NIA ? a + la.off[q < NIA ? q : 0] : ((q - NIA) >> 1 & 1 ? b_up : b) + lb.off[q < NIA ? 0 : q - NIA];
                const bool exists = ((q < NIA ? la.tail_in >> q : lb.tail_in >> (q - NIA)) & 1u) != 0;
                dma_to_lds_addr(exists ? inside : (const unsigned char*)kZeroChunk, dst + q * 1024);
            }
        } else {
#pragma unroll
            for (int q = 0; q < NI; ++q) dma_to_lds(q < NIA ? a : (q - NIA) >> 1 & 1 ? b_up : b, q < NIA ? la.off[q < NIA ? q : 0] : lb.off[q < NIA ? 0 : q - NIA], dst + q * 1024);
        }
    };
    // this wave's K-tiles: wave, wave + KS, ...; where only the weights count, from another one on in every workgroup: if all began with the first, they would ask the memory system for
    // the same columns of all rows at a time (1 x 4096 x 8192 bf16 30.3 us, so 24.8; with more rows, whose panels of A the workgroups share, 32 x 4096 x 8192 25.0 and 26.6)
    const int mine = (nk - wave + KS - 1) / KS;
    int next = MODE == MM_FORWARD && TM == 1 && mine > 0 ? (int)(block * ROTATE % (unsigned)mine) : 0;
    auto fetch_next = [&](unsigned stage) {
        fetch(first + wave + next * KS, stage);
        next = next + 1 == mine ? 0 : next + 1;
    };
#pragma unroll
    for (int s = 0; s < NS; ++s)
        if (s < mine) fetch_next(s);
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const Fragments<ES, false, BM, TM> ra(wave * (NS * STAGE), 0, fi, fq);
    const Fragments<ES, B_ACROSS, BN, TN> rb(wave * (NS * STAGE) + A_BYTES, 0, fi, fq);
    int stage = 0;
    for (int t = 0; t < mine; ++t) {
        // tile t has landed: with NS tiles under way that leaves NS - 1 behind it, near the end only "none" says it
        if (t + NS <= mine) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 1) * NI) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        unsigned char* const at = lds + stage * STAGE;
        u32x4 fa[2][TM], fb[2][TN];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
            for (int i = 0; i < TM; ++i) fa[ks][i] = ra.load(at, ks, i);
#pragma unroll
            for (int j = 0; j < TN; ++j) fb[ks][j] = rb.load(at, ks, j);
        }
        if (t + NS < mine) {
            // the stage is free once its fragments are in registers
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            fetch_next(stage);
            __builtin_amdgcn_sched_barrier(0);
        }
        stage = stage + 1 == NS ? 0 : stage + 1;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = gated_mma<DT>(fb[ks][j], fa[ks][i], acc[i][j]);
    }
    // partial tiles: fragment f of wave w at (f KS + w) KiB; a fragment, or a pair of them, is then finished by one wave
    __syncthreads();                                       // the rings are not read any more
    f32x4* const part = reinterpret_cast<f32x4*>(lds);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) part[((i * TN + j) * KS + wave) * 64 + lane] = acc[i][j];
    __syncthreads();
    auto sum = [&](int f) {
        const f32x4* p = part + f * KS * 64 + lane;
        return (p[0] + p[64]) + (p[128] + p[192]);
    };
    auto put = [&](void* C, long pitch, long row, long col, const f32x4& v) {
        if (row >= g.M || col >= pitch) return;
        const long at = row * pitch + col;
        if (col + 3 < pitch) {
            if constexpr (DT == SP_F32) store_c<ST_PLAIN, 4>((float*)C + at, v);
            else store_c<ST_PLAIN, 2>((unsigned short*)C + at, u32x2{pack_halves<DT>(v[0], v[1]), pack_halves<DT>(v[2], v[3])});
        } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (col + e < pitch) {
                    if constexpr (DT == SP_F32) ((float*)C)[at + e] = v[e];
                    else ((unsigned short*)C)[at + e] = (unsigned short)pack_halves<DT>(v[e], 0.f);
                }
        }
    };
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const long row = m0 + 16 * i + fi;
        if constexpr (MODE == MM_FORWARD) {
#pragma unroll
            for (int p = 0; p < TN / 2; ++p) {
                if ((i * (TN / 2) + p) % KS != wave) continue;
                const f32x4 a = sum(i * TN + 2 * p), u = sum(i * TN + 2 * p + 1);
                const long col = n0 + 16 * p + 4 * fq;
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = gated_activation(a[e], g.activation) * u[e];
                put(g.C0, g.N, row, col, v);
                if (g.keep == KEEP_WHOLE) {
                    put(g.gate, g.N, row, col, a);
                    put(g.up, g.N, row, col, u);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < TN; ++j)
                if ((i * TN + j) % KS == wave) {
                    const long col = n0 + 16 * j + 4 * fq;
                    if (parts > 1) {                       // (K is a multiple of four)
                        if (row < g.M && col < g.K) *reinterpret_cast<f32x4*>(g.parts + ((long)share * g.M + row) * g.K + col) = sum(i * TN + j);
                    } else {
                        put(g.C0, g.K, row, col, sum(i * TN + j));
                    }
                }
        }
    }
}

template <int DT, int TM, int TN, int NS>
__global__ __launch_bounds__(256) void gated_forward_split_kernel(const GatedArgs g) {
    gated_split<DT, MM_FORWARD, TM, TN, NS>(g, blockIdx.x, 0, 1);
}
// The gradient of A so, those of the weights in tiles of 64 x 64.
template <int DT>
__global__ __launch_bounds__(256) void gated_backward_split_kernel(const GatedPair p) {
    gated_pair(p, [](const GatedArgs& g, unsigned block, unsigned part, unsigned parts) { gated_split<DT, MM_INPUT, 2, 4, 2>(g, block, part, parts); },
               [](const GatedArgs& g, unsigned block, unsigned part, unsigned parts) { gated_mm<DT, MM_WEIGHTS, 64, 64, 2, 2, STAGES_64<DT>>(g, block, part, parts); });
}

// The partial sums of several workgroups, in their order: dA, of `of_input` numbers, dG and dU, of half of `of_weights` each (0: nothing to add up); four numbers a lane.
struct GatedJoin {
    const float *input, *weights;
    int input_parts, weights_parts;
    long of_input, of_weights;
    void *dA, *dG, *dU;
};
template <int DT>
__global__ __launch_bounds__(256) void gated_join_kernel(const GatedJoin a) {
    long at = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (at >= a.of_input + a.of_weights) return;
    const bool input = at < a.of_input;
    at -= input ? 0 : a.of_input;
    const float* const from = input ? a.input : a.weights;
    const long all = input ? a.of_input : a.of_weights;
    const int n = input ? a.input_parts : a.weights_parts;
    f32x4 v = *reinterpret_cast<const f32x4*>(from + at);
    for (int p = 1; p < n; ++p) v += *reinterpret_cast<const f32x4*>(from + p * all + at);
    const bool of_up = !input && at >= all / 2;
    void* const C = input ? a.dA : of_up ? a.dU : a.dG;
    at -= of_up ? all / 2 : 0;
    if constexpr (DT == SP_F32) *reinterpret_cast<f32x4*>((float*)C + at) = v;
    else *reinterpret_cast<u32x2*>((unsigned short*)C + at) = u32x2{pack_halves<DT>(v[0], v[1]), pack_halves<DT>(v[2], v[3])};
}

// ---- dg and du ----
struct GatedGradArgs {
    const void *dC, *gate, *up;
    const float *gate_scale, *up_scale;
    void* out;                    // M x 2 half
    long M, N, half;
    int activation;
};

// Bound by HBM: 8192 x 8192 bf16, 671 MB, 101 us (6.6 TB/s); from 8-bit blocks, 5008 x 5461, 228 MB, 35.6 us (6.4).  A kernel of its own: in the products' loads dg and du would be computed
// again for every tile of columns.  dg and du are rounded to the operands' type, as the matrix instructions take both of one: gradients in 16 bits have sqrt 2 of the error that the rounding of the results alone
// would leave (bf16 0.0024 of the norm, 0.0017), where two parts of each would be twice the products; and f16's range.  Eight columns of a row a lane.  F8: gate and up are e4m3 blocks.
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

constexpr double MOST_ITEMS = 4294967296.0;     // a launch holds fewer than 2^32 work items
template <int MODE, int BM, int BN>
static bool set_tiles(GatedArgs& g, int group_m) {
    const long tiles_m = MODE == MM_WEIGHTS ? 2 * gated_ceil(g.N, BM) : gated_ceil(g.M, BM), tiles_n = MODE == MM_FORWARD ? gated_ceil(g.N, BN / 2) : gated_ceil(g.K, BN);
    if (tiles_m * tiles_n >= 1l << 24) return false;
    g.tiles_m = (int)tiles_m;
    g.tiles_n = (int)tiles_n;
    g.group_m = group_m == 0 ? g.tiles_m : group_m;        // 0: the tiles of one panel of weights stand side by side
    return true;
}
template <typename Kernel, typename Args>
static int launch_lds(const char* what, Kernel kernel, unsigned blocks, unsigned threads, int lds_bytes, const Args& args, hipStream_t stream) {
    if ((double)blocks * threads >= MOST_ITEMS) return fail(SP_ERR_SHAPE, "%s: too large", what);
    if (const int rc = ensure_dynamic_lds((const void*)kernel, lds_bytes); rc != SP_OK) return rc;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(threads), lds_bytes, stream, args);
    return check_launch(what);
}
constexpr int larger(int a, int b) { return a > b ? a : b; }
constexpr int split_lds(int TM, int TN, int NS) { return larger(4 * NS * 16 * (TM + TN) * ROW_BYTES, TM * TN * 4096); }
constexpr int mm_lds(int BM, int BN, int NS) { return NS * (BM + BN) * ROW_BYTES; }

template <int DT, int BM, int BN, int WM, int WN, int NS>
static int launch_forward(const char* what, GatedArgs g, hipStream_t stream) {
    if (!set_tiles<MM_FORWARD, BM, BN>(g, 4)) return fail(SP_ERR_SHAPE, "%s: too large", what);
    return launch_lds(what, gated_forward_kernel<DT, BM, BN, WM, WN, NS>, (unsigned)(g.tiles_m * g.tiles_n), WM * WN * 64, mm_lds(BM, BN, NS), g, stream);
}
template <int DT, int TM, int TN, int NS>
static int launch_forward_split(const char* what, GatedArgs g, hipStream_t stream) {
    if (!set_tiles<MM_FORWARD, 16 * TM, 16 * TN>(g, 0)) return fail(SP_ERR_SHAPE, "%s: too large", what);
    return launch_lds(what, gated_forward_split_kernel<DT, TM, TN, NS>, (unsigned)(g.tiles_m * g.tiles_n), 256, split_lds(TM, TN, NS), g, stream);
}

// The first `rows` rows in tiles of 256 x 256, the others in tiles of 128 x 256.
template <int DT>
static int launch_forward_rows(const char* what, const GatedArgs& g, long rows, hipStream_t stream) {
    constexpr long ES = ELEM_BYTES<DT>;
    GatedRows p{g, g, 0};
    p.large.M = rows;
    p.small.M = g.M - rows;
    p.small.A = g.A + rows * g.K * ES;
    p.small.C0 = (unsigned char*)g.C0 + rows * g.N * ES;
    if (g.keep != KEEP_NONE) {
        const long bytes = rows * (g.keep == KEEP_F8 ? (g.N + 15) / 16 * 16 : g.N * ES);
        p.small.gate = (unsigned char*)g.gate + bytes;
        p.small.up = (unsigned char*)g.up + bytes;
    }
    if (g.keep == KEEP_F8) {
        const long blocks = rows * ((g.N + QB - 1) / QB);
        p.small.gate_scale = g.gate_scale + blocks;
        p.small.up_scale = g.up_scale + blocks;
    }
    if (!set_tiles<MM_FORWARD, 256, 256>(p.large, 4) || !set_tiles<MM_FORWARD, 128, 256>(p.small, 4)) return fail(SP_ERR_SHAPE, "%s: too large", what);
    p.large_blocks = (unsigned)(p.large.tiles_m * p.large.tiles_n);
    const unsigned blocks = p.large_blocks + (unsigned)(p.small.tiles_m * p.small.tiles_n);
    return launch_lds(what, gated_forward_rows_kernel<DT>, blocks, 512, larger(mm_lds(256, 256, 2), mm_lds(128, 256, 3)), p, stream);
}

// Those of the two products that have parts; the longer ones' workgroups first.
static unsigned set_pair(GatedPair& p, bool input_first) {
    const unsigned input = p.input_parts * (unsigned)(p.input.tiles_m * p.input.tiles_n), weights = p.weights_parts * (unsigned)(p.weights.tiles_m * p.weights.tiles_n);
    p.input_first = input_first;
    p.first_blocks = input_first ? input : weights;
    return input + weights;
}
template <int DT, int BM, int BN, int WM, int WN, int NS>
static int launch_backward(const char* what, GatedPair p, bool input_first, hipStream_t stream) {
    if (!set_tiles<MM_INPUT, BM, BN>(p.input, 4) || !set_tiles<MM_WEIGHTS, BM, BN>(p.weights, 4)) return fail(SP_ERR_SHAPE, "%s: too large", what);
    const unsigned blocks = set_pair(p, input_first);
    return launch_lds(what, gated_backward_kernel<DT, BM, BN, WM, WN, NS>, blocks, WM * WN * 64, mm_lds(BM, BN, NS), p, stream);
}
template <int DT>
static int launch_backward_split(const char* what, GatedPair p, bool input_first, hipStream_t stream) {
    if (!set_tiles<MM_INPUT, 32, 64>(p.input, 0) || !set_tiles<MM_WEIGHTS, 64, 64>(p.weights, 4)) return fail(SP_ERR_SHAPE, "%s: too large", what);
    const unsigned blocks = set_pair(p, input_first);
    return launch_lds(what, gated_backward_split_kernel<DT>, blocks, 256, larger(split_lds(2, 4, 2), mm_lds(64, 64, STAGES_64<DT>)), p, stream);
}

// ---- which kernel ----
// Estimated times in us, without the launch: workgroups in rounds of as many as a unit's LDS holds at a time, each nk K-tiles (a quarter of them, where four waves share
// them) plus an overhead; n workgroups on a unit take n times the work of a K-tile, and never less than what a lone one waits for.
// Forward: fitted on what every kernel took on 99 shapes, from 1 x 512 x 1365 to 16384 x 4096 x 512; the one it picks is on the mean 2 % behind the fastest (3 with 8-bit blocks).
// Factors that are kept whole are in no menu: their results come on top, whatever the tile (8192 x 1024 x 2736 bf16 85 us with them, 76 without).
// More tiles (64 x 128, 128 x 256 in two stages, 16 x 64 and 64 x 64 in four parts) were worth less than a hundredth.
struct MmCost {
    int id, bm, bn;               // bn: columns of the result
    int per_unit;
    bool split;
    float lone, work, overhead;
};
enum { SPLIT_16, SPLIT_32, TILE_32_BLOCKS, TILE_64, TILE_64_BLOCKS, TILE_128, TILE_128_WIDE, TILE_256 };
static int threads_of(int id) { return id <= TILE_64 ? 256 : 512; }
static const MmCost kForward16[] = {{SPLIT_16, 16, 16, 3, true, 0.156f, 0.278f, 2.55f}, {SPLIT_32, 32, 16, 2, true, 0.336f, 0.387f, 2.65f}, {TILE_64, 64, 32, 2, false, 0.227f, 0.183f, 2.57f},
                                    {TILE_128, 128, 64, 1, false, 0.437f, 0.386f, 3.84f}, {TILE_128_WIDE, 128, 128, 1, false, 0.716f, 0.4f, 4.67f}, {TILE_256, 256, 128, 1, false, 1.2f, 0.1f, 5.95f}};
static const MmCost kForward32[] = {{SPLIT_16, 16, 16, 3, true, 0.587f, 0.354f, 2.47f}, {SPLIT_32, 32, 16, 2, true, 0.587f, 0.632f, 3.2f}, {TILE_64, 64, 32, 5, false, 0.633f, 0.54f, 2.4f}};
// tiles that hold whole blocks of 128 columns of both factors
static const MmCost kBlocks16[] = {{TILE_32_BLOCKS, 32, 128, 1, false, 0.41f, 0.41f, 4.8f}, {TILE_64_BLOCKS, 64, 128, 1, false, 0.46f, 0.46f, 5.3f}, {TILE_128_WIDE, 128, 128, 1, false, 0.716f, 0.4f, 6.7f},
                                   {TILE_256, 256, 128, 1, false, 1.2f, 0.1f, 8.f}};
static const MmCost kBlocks32[] = {{TILE_32_BLOCKS, 32, 128, 1, false, 1.05f, 1.05f, 5.f}, {TILE_64_BLOCKS, 64, 128, 1, false, 1.972f, 1.039f, 6.f}};
// Backward, both products in one launch (the input's tile first in a pair, the weights' beside it): fitted on 2,700 timings of 150 shapes from 55 x 1720 x 1674 to 9344 x 2304 x 768 with
// every tile and numbers of parts; what it picks is on the mean 4 % behind the fastest of them.  (us, each in a launch of its own with its best tile / together: 1341 x 1536 x 2992 bf16
// 84.4 / 64.5, 1003 x 512 x 1365 29.3 / 22.8, 9344 x 896 x 1664 164 / 154, 1003 x 512 x 1365 f32 74.2 / 61.2.)  per_unit 0: as many as there is room for, which share the unit's rate.
static const MmCost kInput16[] = {{SPLIT_32, 32, 64, 1, true, 0.585f, 0.109f, 4.213f}, {TILE_64, 64, 64, 2, false, 0.248f, 0.083f, 3.684f}, {TILE_128, 128, 128, 1, false, 0.428f, 0.424f, 2.987f},
                                  {TILE_128_WIDE, 128, 256, 1, false, 0.695f, 0.704f, 3.237f}, {TILE_256, 256, 256, 1, false, 1.265f, 0.329f, 4.056f}};
static const MmCost kWeights16[] = {{TILE_64, 64, 64, 1, false, 0.107f, 0.498f, 1.264f}, {TILE_64, 64, 64, 2, false, 0.262f, 0.258f, 1.686f}, {TILE_128, 128, 128, 1, false, 0.405f, 0.45f, 3.003f},
                                    {TILE_128_WIDE, 128, 256, 1, false, 0.667f, 0.134f, 4.458f}, {TILE_256, 256, 256, 1, false, 1.45f, 0.134f, 0.053f}};
static const MmCost kInput32[] = {{SPLIT_32, 32, 64, 1, true, 1.228f, 0.474f, 3.027f}, {TILE_64, 64, 64, 0, false, 0.778f, 0.487f, 1.19f}};
static const MmCost kWeights32[] = {{TILE_64, 64, 64, 1, false, 0.607f, 0.609f, 2.227f}, {TILE_64, 64, 64, 0, false, 0.826f, 0.454f, 1.19f}};

// What a product of rows x cols asks of a tile.
struct MmWork {
    double tiles;
    long nk;                      // K-tiles of one
    double sums;                  // numbers of the result
};
static MmWork work_of(const MmCost& c, int mode, bool f32, long M, long N, long K) {
    const long bk = f32 ? 32 : 64, rows = mode == MM_WEIGHTS ? N : M, cols = mode == MM_FORWARD ? N : K, twice = mode == MM_WEIGHTS ? 2 : 1;
    return {(double)gated_ceil(rows, c.bm) * (double)gated_ceil(cols, c.bn) * twice, mode == MM_FORWARD ? gated_ceil(K, bk) : mode == MM_INPUT ? 2 * gated_ceil(N, bk) : gated_ceil(M, bk),
            (double)rows * cols * twice};
}
static long tiles_of_k(const MmCost& c, long nk, int parts) { return gated_ceil(gated_ceil(nk, parts), c.split ? 4 : 1); }
static double group_us(const MmCost& c, long k_tiles, double on_unit) { return k_tiles * (on_unit * c.work > c.lone ? on_unit * c.work : (double)c.lone) + c.overhead; }
constexpr double JOIN_US = 5, SHARED_US = 1.9;
static double join_us(const MmWork& w, int parts, bool f32) { return parts > 1 ? w.sums * (8.0 * parts + (f32 ? 4 : 2)) * 1e-6 / 8 : 0; }
static bool may_split(const MmWork& w, int parts) { return parts == 1 || (w.tiles * parts <= 2.0 * device_cu_count() && w.nk >= 4l * parts); }

template <size_t N>
static int cheapest(const MmCost (&menu)[N], bool f32, long M, long N_, long K, double& best_us) {
    const long cus = device_cu_count();
    int best = -1;
    for (const MmCost& c : menu) {
        const MmWork w = work_of(c, MM_FORWARD, f32, M, N_, K);
        if (w.tiles * threads_of(c.id) >= MOST_ITEMS) continue;
        const double round = (double)cus * c.per_unit, full = (double)(int64_t)(w.tiles / round), rest = w.tiles - full * round;
        const long k_tiles = tiles_of_k(c, w.nk, 1);
        const double us = full * group_us(c, k_tiles, c.per_unit) + (rest > 0 ? group_us(c, k_tiles, (double)(int64_t)((rest + cus - 1) / cus)) : 0);
        if (best < 0 || us < best_us) {
            best = c.id;
            best_us = us;
        }
    }
    return best;
}

// Estimated time of n1 workgroups of t1 us, the longer ones, and then n2 of t2, each to the slot that is free first.
static double both_us(double slots, double n1, double t1, double n2, double t2) {
    const double rounds = (double)(int64_t)(n1 / slots), late = n1 - rounds * slots;        // `late` slots have one round more of the first
    if (n1 + n2 > 64 * slots) {                            // (many rounds: the last one is not looked at)
        const double all = (n1 * t1 + n2 * t2) / slots + t2, first = (late > 0 ? rounds + 1 : rounds) * t1;
        return all > first ? all : first;
    }
    double count[2] = {late, slots - late}, at[2] = {(rounds + 1) * t1, rounds * t1};
    while (n2 > 0) {
        const int next = count[0] > 0 && at[0] < at[1] ? 0 : 1;
        at[next] += t2;
        n2 -= count[next];
    }
    return count[0] > 0 && at[0] > at[1] ? at[0] : at[1];
}
// How many rows to take in tiles of 256 x 256 where the others take 128 x 256: all of them, unless less than `us` comes out.
// (us, all in large ones / so: 3000 x 2048 x 5461 bf16 136 / 123, 5008 x 2048 x 5461 with 8-bit blocks 210 / 201; steps of both directions, which the part's power limits, 404 / 393 and 606 / 600.)
template <size_t N>
static long rows_of_large(const MmCost (&menu)[N], long M, long N_, long K, double us) {
    const MmCost &small = menu[N - 2], &large = menu[N - 1];
    const long cus = device_cu_count(), nk = gated_ceil(K, 64), tiles_n = gated_ceil(N_, large.bn), tiles_m = gated_ceil(M, large.bm);
    const long tail = 2 * gated_ceil(cus, tiles_n), fewest = tiles_m - 1 < tail ? 1 : tiles_m - tail;        // what two rounds take, and a bound for the search
    const double t1 = group_us(large, nk, 1), t2 = group_us(small, nk, 1);
    long best = M;
    for (long rows = tiles_m - 1; rows >= fewest && rows >= tiles_m - 64; --rows) {
        const double one = both_us((double)cus, (double)(rows * tiles_n), t1, (double)(gated_ceil(M - rows * large.bm, small.bm) * tiles_n), t2);
        if (one < us) {
            us = one;
            best = rows * large.bm;
        }
    }
    return best;
}
// Long products are limited by the part's power, of which smaller tiles take more.
static double of_power(double us, int id, bool f32) { return !f32 && id != TILE_256 && us > 100 ? us + 0.2 * (us - 100) : us; }

// The tile and the parts of both products of the backward pass, and the tiles of one alone.  Tiles add up a K-tile after the other, all in the same order, so with the same parts a gradient has
// the same bits whether the other is wanted or not; where four waves share K, the kernel is the same, too.  (A lone gradient, us, on the tile of both / on its own: of the input,
// 2048 x 2048 x 5461 bf16 149 / 114, 4096 x 1024 x 4096 134 / 109; of the weights, 2048 x 1024 x 2736 45 / 37; the wrong way, 2048 x 1024 x 2736, input, 46 / 51.)
struct BackwardPlan {
    int id, input_parts, weights_parts;
    bool input_first;
    int input_id, weights_id;
};
template <size_t N_>
static int tile_alone(const MmCost (&menu)[N_], int mode, bool f32, int parts, long M, long N, long K, int otherwise) {
    const long cus = device_cu_count();
    double best_us = 0;
    int best = otherwise;
    for (size_t i = 1; i < N_; ++i) {                      // (behind the one whose waves share K)
        const MmCost& c = menu[i];
        const MmWork w = work_of(c, mode, f32, M, N, K);
        if (c.per_unit == 0 || w.tiles * parts * threads_of(c.id) >= MOST_ITEMS) continue;
        const double alone = both_us((double)cus * c.per_unit, w.tiles * parts, group_us(c, tiles_of_k(c, w.nk, parts), c.per_unit), 0, 1), us = of_power(alone, c.id, f32);
        if (best_us == 0 || us < best_us) {
            best_us = us;
            best = c.id;
        }
    }
    return best;
}
template <size_t N_>
static BackwardPlan plan_of(const MmCost (&inputs)[N_], const MmCost (&weights)[N_], bool f32, long M, long N, long K) {
    const long cus = device_cu_count();
    BackwardPlan best{-1, 1, 1, true, -1, -1};
    double best_us = 0;
    for (size_t i = 0; i < N_; ++i) {
        const MmCost &ci = inputs[i], &cw = weights[i];
        const MmWork wi = work_of(ci, MM_INPUT, f32, M, N, K), ww = work_of(cw, MM_WEIGHTS, f32, M, N, K);
        if ((wi.tiles + ww.tiles) * threads_of(ci.id) >= MOST_ITEMS) continue;
        // shares of K about as long as one another's
        const double li = wi.nk * (ci.split ? 0.25 : 1.0) * ci.work, lw = ww.nk * cw.work;
        for (int n = 1; n <= 16; ++n) {
            const int other = (int)(n * (li > lw ? lw / li : li / lw) + 0.5), fewer = other > 1 ? other : 1;
            const int pi = li > lw ? n : fewer, pw = li > lw ? fewer : n;
            if (!may_split(wi, pi) || !may_split(ww, pw)) break;
            const double ni = wi.tiles * pi, nw = ww.tiles * pw, all = (double)(int64_t)((ni + nw + cus - 1) / cus);
            const long ki = tiles_of_k(ci, wi.nk, pi), kw = tiles_of_k(cw, ww.nk, pw);
            double ti, tw, us;
            if (ci.per_unit == 0) {                        // those on a unit share its rate
                ti = ki * ci.work + ci.overhead;
                tw = kw * cw.work + cw.overhead;
                us = ti > tw ? both_us(cus, ni, ti, nw, tw) : both_us(cus, nw, tw, ni, ti);
                const double longest = ki * ci.lone > kw * cw.lone ? ki * ci.lone : kw * cw.lone;
                us = (us > longest ? us : longest) + SHARED_US;
            } else {
                const double on_unit = all < ci.per_unit ? all : ci.per_unit;
                ti = group_us(ci, ki, on_unit);
                tw = group_us(cw, kw, on_unit);
                us = ti > tw ? both_us(cus * on_unit, ni, ti, nw, tw) : both_us(cus * on_unit, nw, tw, ni, ti);
            }
            us = of_power(us, ci.id, f32);
            if (pi > 1 || pw > 1) us += JOIN_US + join_us(wi, pi, f32) + join_us(ww, pw, f32);
            if (best.id < 0 || us < best_us) {
                best = {ci.id, pi, pw, ti > tw, ci.id, ci.id};
                best_us = us;
            }
        }
    }
    if (best.id > SPLIT_32) {
        best.input_id = tile_alone(inputs, MM_INPUT, f32, best.input_parts, M, N, K, best.id);
        best.weights_id = tile_alone(weights, MM_WEIGHTS, f32, best.weights_parts, M, N, K, best.id);
    }
    return best;
}
// The plans of the sizes that this thread asked for last: they follow from the sizes alone, and a short call would take as long to make one as its kernels run.
static BackwardPlan choose_backward(bool f32, long M, long N, long K) {
    struct Known {
        bool f32;
        int cus;
        long M, N, K;
        BackwardPlan plan;
    };
    constexpr unsigned PLACES = 16;
    static thread_local Known known[PLACES];
    const int cus = device_cu_count();
    Known& at = known[(unsigned)((unsigned long)(M * 31 + N * 17 + K) * 0x9e3779b97f4a7c15ul >> 32) % PLACES];
    if (at.f32 != f32 || at.cus != cus || at.M != M || at.N != N || at.K != K)
        at = {f32, cus, M, N, K, f32 ? plan_of(kInput32, kWeights32, f32, M, N, K) : plan_of(kInput16, kWeights16, f32, M, N, K)};
    return at.plan;
}

template <int DT>
static int gated_forward(const GatedArgs& g, hipStream_t stream) {
    constexpr bool F32 = DT == SP_F32;
    const char* const what = "sp_gemm_abt_gated";
    double us = 0;
    int id;
    if (g.keep == KEEP_F8) id = F32 ? cheapest(kBlocks32, F32, g.M, g.N, g.K, us) : cheapest(kBlocks16, F32, g.M, g.N, g.K, us);
    else id = F32 ? cheapest(kForward32, F32, g.M, g.N, g.K, us) : cheapest(kForward16, F32, g.M, g.N, g.K, us);
    switch (id) {
        case SPLIT_16: return launch_forward_split<DT, 1, 2, 2>(what, g, stream);
        case SPLIT_32: return launch_forward_split<DT, 2, 2, 2>(what, g, stream);
        case TILE_64: return launch_forward<DT, 64, 64, 2, 2, STAGES_64<DT>>(what, g, stream);
        case TILE_32_BLOCKS: return launch_forward<DT, 32, 256, 1, 4, 3>(what, g, stream);
        case TILE_64_BLOCKS: return launch_forward<DT, 64, 256, 2, 4, 3>(what, g, stream);
    }
    if constexpr (!F32) {
        if (id == TILE_128) return launch_forward<DT, 128, 128, 2, 4, 4>(what, g, stream);
        const long rows = g.keep == KEEP_F8 ? rows_of_large(kBlocks16, g.M, g.N, g.K, us) : rows_of_large(kForward16, g.M, g.N, g.K, us);
        if (rows < g.M) return launch_forward_rows<DT>(what, g, rows, stream);
        if (id == TILE_128_WIDE) return launch_forward<DT, 128, 256, 4, 2, 3>(what, g, stream);
        return launch_forward<DT, 256, 256, 4, 2, 2>(what, g, stream);
    }
    return fail(SP_ERR_SHAPE, "%s: too large", what);
}

template <int DT>
static int backward_products(int id, const GatedPair& p, bool input_first, hipStream_t stream) {
    constexpr bool F32 = DT == SP_F32;
    const char* const what = "sp_gemm_abt_gated_backward";
    if (id == SPLIT_32) return launch_backward_split<DT>(what, p, input_first, stream);
    if (id == TILE_64) return launch_backward<DT, 64, 64, 2, 2, STAGES_64<DT>>(what, p, input_first, stream);
    if constexpr (!F32) {
        if (id == TILE_128) return launch_backward<DT, 128, 128, 2, 4, 4>(what, p, input_first, stream);
        if (id == TILE_128_WIDE) return launch_backward<DT, 128, 256, 2, 4, 3>(what, p, input_first, stream);
        return launch_backward<DT, 256, 256, 2, 4, 2>(what, p, input_first, stream);
    }
    return fail(SP_ERR_SHAPE, "%s: too large", what);
}

template <int DT>
static int gated_backward(GatedArgs input, GatedArgs weights, const GatedGradArgs& grad, bool f8, hipStream_t stream) {
    const long pieces = grad.M * (grad.half / 8);
    const dim3 blocks((unsigned)gated_ceil(pieces, 256));
    if (f8) hipLaunchKernelGGL((gated_grad_kernel<DT, true>), blocks, dim3(256), 0, stream, grad);
    else hipLaunchKernelGGL((gated_grad_kernel<DT, false>), blocks, dim3(256), 0, stream, grad);
    if (const int rc = check_launch("sp_gemm_abt_gated_backward"); rc != SP_OK) return rc;
    const BackwardPlan plan = choose_backward(DT == SP_F32, grad.M, grad.N, input.K);
    const unsigned input_parts = input.C0 != nullptr ? plan.input_parts : 0, weights_parts = weights.C0 != nullptr ? plan.weights_parts : 0;
    if (plan.input_parts > 1) weights.parts = input.parts + (long)plan.input_parts * input.M * input.K;
    const int id = weights_parts == 0 ? plan.input_id : input_parts == 0 ? plan.weights_id : plan.id;
    if (const int rc = backward_products<DT>(id, GatedPair{input, weights, 0, 0, input_parts, weights_parts}, plan.input_first, stream); rc != SP_OK) return rc;
    if (input_parts <= 1 && weights_parts <= 1) return SP_OK;
    GatedJoin join{input.parts, weights.parts, (int)input_parts, (int)weights_parts, input_parts > 1 ? input.M * input.K : 0, weights_parts > 1 ? 2 * weights.N * weights.K : 0,
                   input.C0, weights.C0, weights.C1};
    hipLaunchKernelGGL(gated_join_kernel<DT>, dim3((unsigned)gated_ceil(join.of_input + join.of_weights, 1024)), dim3(256), 0, stream, join);
    return check_launch("sp_gemm_abt_gated_backward");
}

namespace {
struct GatedKernelNames {
    GatedKernelNames() {
        register_kernel("gated_forward_256x256", (const void*)gated_forward_kernel<SP_BF16, 256, 256, 4, 2, 2>, 512);
        register_kernel("gated_backward_256x256", (const void*)gated_backward_kernel<SP_BF16, 256, 256, 2, 4, 2>, 512);
    }
} gated_kernel_names;
}  // namespace

}  // namespace sp

using namespace sp;

// Columns of either half of the backward pass's workspace: whole K-tiles, of 64 numbers of 16 bits (two of f32).
static int64_t gated_half(int64_t N) { return (N + 63) / 64 * 64; }
// Bytes of either kept factor, and of its scales.
static int64_t gated_kept_bytes(bool f8, int es, int64_t M, int64_t N) { return M * (f8 ? (N + 15) / 16 * 16 : N * es); }
static int64_t gated_scale_bytes(bool f8, int64_t M, int64_t N) { return f8 ? M * ((N + QB - 1) / QB) * 4 : 0; }

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
    const int es = dtype == SP_F32 ? 4 : 2;
    const int64_t kept_bytes = gated_kept_bytes(f8, es, M, N), scale_bytes = gated_scale_bytes(f8, M, N);
    if (const int rc = lie_apart(__func__, {{"C", C, M * N * es}, {"gate", gate, kept_bytes}, {"up", up, kept_bytes},
                                  {"gate_scale", f8 ? gate_scale : nullptr, scale_bytes}, {"up_scale", f8 ? up_scale : nullptr, scale_bytes}},
                                 {{"A", A, M * K * es}, {"B_gate", B_gate, N * K * es}, {"B_up", B_up, N * K * es}});
        rc != SP_OK)
        return rc;
    if (const int rc = require_gfx950(__func__); rc != SP_OK) return rc;
    GatedArgs g{};
    g.A = (const unsigned char*)A; g.B0 = (const unsigned char*)B_gate; g.B1 = (const unsigned char*)B_up; g.C0 = C; g.gate = gate; g.up = up;
    g.gate_scale = gate_scale; g.up_scale = up_scale; g.M = M; g.N = N; g.K = K; g.activation = activation; g.keep = f8 ? KEEP_F8 : keeps ? KEEP_WHOLE : KEEP_NONE;
    // what does not stay in the caches (32 MiB of L2) is streamed past them, gate and up only where a row is of whole lines (5008 x 2048 x 5461 bf16: 188 us, 216 streamed)
    const int64_t pitch = N * es;
    g.stream = M * pitch <= (int64_t)32 << 20 ? 0 : pitch % 128 == 0 ? 3 : 1;
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == SP_F32) return gated_forward<SP_F32>(g, st);
    if (dtype == SP_F16) return gated_forward<SP_F16>(g, st);
    return gated_forward<SP_BF16>(g, st);
}

// Partial sums of the backward products, side by side.
static int64_t gated_parts_bytes(int dtype, int64_t M, int64_t N, int64_t K) {
    const BackwardPlan plan = choose_backward(dtype == SP_F32, M, N, K);
    return (plan.input_parts > 1 ? plan.input_parts * M * K * 4 : 0) + (plan.weights_parts > 1 ? plan.weights_parts * 2 * N * K * 4 : 0);
}
static int64_t gated_halves_bytes(int dtype, int64_t M, int64_t N) { return M * 2 * gated_half(N) * (dtype == SP_F32 ? 4 : 2); }

extern "C" int64_t sp_gemm_abt_gated_backward_workspace_bytes(int dtype, int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || M > INT32_MAX || N > (int64_t)1 << 24 || K > (int64_t)1 << 24) return 0;
    return gated_halves_bytes(dtype, M, N) + gated_parts_bytes(dtype, M, N, K);
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
    const int64_t need = sp_gemm_abt_gated_backward_workspace_bytes(dtype, M, N, K);
    if (workspace_bytes < need)
        return fail(SP_ERR_ARG, "sp_gemm_abt_gated_backward: workspace of %lld bytes, %lld are needed", (long long)workspace_bytes, (long long)need);
    // (dC, gate and up are read by the first launch alone, before any gradient is written: a gradient may take their place)
    const int es = dtype == SP_F32 ? 4 : 2;
    const int64_t kept_bytes = gated_kept_bytes(f8, es, M, N), scale_bytes = gated_scale_bytes(f8, M, N);
    if (const int rc = lie_apart(__func__, {{"dA", dA, M * K * es}, {"dB_gate", dB_gate, N * K * es}, {"dB_up", dB_up, N * K * es}, {"workspace", workspace, need}},
                                 {{"A", A, M * K * es}, {"B_gate", B_gate, N * K * es}, {"B_up", B_up, N * K * es}});
        rc != SP_OK)
        return rc;
    if (const int rc = lie_apart(__func__, {{"workspace", workspace, need}},
                                 {{"dC", dC, M * N * es}, {"gate", gate, kept_bytes}, {"up", up, kept_bytes},
                                  {"gate_scale", f8 ? gate_scale : nullptr, scale_bytes}, {"up_scale", f8 ? up_scale : nullptr, scale_bytes}});
        rc != SP_OK)
        return rc;
    if (const int rc = require_gfx950(__func__); rc != SP_OK) return rc;
    GatedGradArgs grad{};
    grad.dC = dC; grad.gate = gate; grad.up = up; grad.gate_scale = gate_scale; grad.up_scale = up_scale; grad.out = workspace; grad.M = M; grad.N = N; grad.half = half;
    grad.activation = activation;
    GatedArgs input{}, weights{};
    input.A = (const unsigned char*)workspace; input.B0 = (const unsigned char*)B_gate; input.B1 = (const unsigned char*)B_up; input.C0 = dA; input.M = M; input.N = N; input.K = K;
    input.half = half; input.parts = (float*)((unsigned char*)workspace + gated_halves_bytes(dtype, M, N)); input.stream = M * K * es > (int64_t)32 << 20;
    weights = input;
    weights.B0 = (const unsigned char*)A; weights.B1 = nullptr; weights.C0 = dB_gate; weights.C1 = dB_up; weights.stream = 2 * N * K * es > (int64_t)32 << 20;
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == SP_F32) return gated_backward<SP_F32>(input, weights, grad, f8, st);
    if (dtype == SP_F16) return gated_backward<SP_F16>(input, weights, grad, f8, st);
    return gated_backward<SP_BF16>(input, weights, grad, f8, st);
}
