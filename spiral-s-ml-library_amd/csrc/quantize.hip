// Rows and columns of a matrix in 8-bit blocks of 128 with a scale each: the operands of gemm_scaled.hip.
//
// A workgroup takes a tile of 128 x 128 (16 x 128 where only rows are wanted in blocks of one, 128 x 64 for few blocks of one column), so every block along either direction lies inside
// one tile, and x is read once whatever is wanted of it.  A lane holds 1, 4 or 8 rows of 8 columns.  A row's 16 lanes are a DPP row, so the
// largest magnitude of a row's block takes four DPP steps; a column's takes two or three cross-lane steps and, over the waves, LDS.
// Magnitudes are compared as bits: an infinity is larger than every number and a NaN larger than that, so neither is lost.  The transposed
// numbers go through LDS so that both forms leave in 128-byte rows.
//
// x / scale costs three operations: q = x * (1 / scale) and one step q + (x - q * scale) * (1 / scale), whose remainder is exact (Markstein's
// correction).  That is x / scale rounded to f32, but for ties of f32, before the 8-bit rounding.
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

struct QuantArgs {
    const void* x;
    unsigned char *q, *q_t;
    float *scale, *scale_t;
    long rows, cols;
    long pitch, pitch_t;          // of q and q_t: cols and rows rounded up to a multiple of 16
    long blocks_c, blocks_r;      // blocks of 128 along cols and rows: the widths of scale and scale_t
};

__device__ __forceinline__ unsigned max_u32(unsigned a, unsigned b) { return a > b ? a : b; }

// WIDE: blocks of 128 x 128.  OUT: 1 = q, 2 = q_t, 3 = both.  R: rows per lane, ROWS: of the tile, LANES: of 8 columns, its width.  POLICY: of the stores (a branch at each
// store, the compiler folds both sides into a plain one).
template <int DT, int F8, bool WIDE, int OUT, int R, int ROWS, int LANES, int POLICY>
__global__ __launch_bounds__(ROWS / R * LANES) void quantize_kernel(const void* x_first, long rows_first, long cols_first, const QuantArgs args) {
    constexpr int E = ELEM_BYTES<DT>, PIECES = 8 / PER16<DT>;
    constexpr bool ROW = (OUT & 1) != 0, COL = (OUT & 2) != 0;
    constexpr int COLS = LANES * 8, THREADS = ROWS / R * LANES, WAVES = THREADS / 64;
    static_assert(ROWS == QB || (!COL && !WIDE), "tiles of fewer rows hold blocks of one row only");
    static_assert(LANES == 16 || (!ROW && !WIDE), "tiles of fewer columns hold blocks of one column only");
    static_assert(!COL || R == 8 || R == 4, "a lane's rows of a column are one store");
    constexpr int PITCH = QB + 16;            // bytes of a transposed row in LDS
    __shared__ __attribute__((aligned(16))) unsigned char turned[COL ? COLS * PITCH : 16];
    __shared__ unsigned most[COL && !WIDE ? WAVES * COLS : WAVES];
    const long rows = rows_first, cols = cols_first;
    const int tid = threadIdx.x, cg = tid % LANES, rg = tid / LANES, wave = tid >> 6;
    const long tiles_c = (cols + COLS - 1) / COLS;
    const long tile_r = blockIdx.x / tiles_c, tile_c = blockIdx.x - tile_r * tiles_c;
    const long r0 = tile_r * ROWS + rg * R, c0 = tile_c * COLS + cg * 8;
    u32x4 raw[R][PIECES];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const long col = c0 + p * PER16<DT>;
            raw[i][p] = load16<DT>(x_first, (r0 + i) * cols + col, r0 + i < rows ? cols - col : 0);
        }
    auto put = [&](auto* to, auto v) { store_c<POLICY, sizeof(v)>(to, v); };
    auto value = [&](int i, int j) { return element<DT>(raw[i][j / PER16<DT>], j % PER16<DT>); };
    auto magnitude = [&](int i, int j) { return __float_as_uint(value(i, j)) & 0x7fffffffu; };
    auto across_row = [](unsigned v) { return group_allreduce<16>(v, max_u32); };      // over the 16 lanes of a row
    auto across_wave = [](unsigned v) {                                                  // over the row groups of a wave
#pragma unroll
        for (int d = LANES; d < WAVE; d *= 2) v = max_u32(v, __shfl_xor(v, d, WAVE));
        return v;
    };
    BlockScale one;                           // WIDE: of the tile
    if constexpr (WIDE) {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max_u32(m, magnitude(i, j));
        m = across_wave(across_row(m));
        if ((tid & 63) == 0) most[wave] = m;
        __syncthreads();
        m = most[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) m = max_u32(m, most[w]);
        one.template set<F8>(m);
        if (tid == 0) {
            if constexpr (ROW) args.scale[tile_r * args.blocks_c + tile_c] = one.scale;
            if constexpr (COL) args.scale_t[tile_c * args.blocks_r + tile_r] = one.scale;
        }
    }
    if constexpr (ROW) {
        const bool ends = ((int)cols & 15) != 0 && (tile_c + 1) * COLS > cols;             // the rows end inside this tile, with padding behind them
#pragma unroll
        for (int i = 0; i < R; ++i) {
            BlockScale s = one;
            if constexpr (!WIDE) {
                unsigned m = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) m = max_u32(m, magnitude(i, j));
                s.template set<F8>(across_row(m));
                if (cg == 0 && r0 + i < rows) args.scale[(r0 + i) * args.blocks_c + tile_c] = s.scale;
            }
            u32x2 o;
            o.x = pack_f8<F8>(s(value(i, 0)), s(value(i, 1)), s(value(i, 2)), s(value(i, 3)));
            o.y = pack_f8<F8>(s(value(i, 4)), s(value(i, 5)), s(value(i, 6)), s(value(i, 7)));
            if (ends) {
                o.x = first_bytes(o.x, cols - c0);
                o.y = first_bytes(o.y, cols - c0 - 4);
            }
            if (r0 + i < rows && c0 < args.pitch) put(args.q + (r0 + i) * args.pitch + c0, o);
        }
    }
    if constexpr (COL) {
        const bool ends = ((int)rows & 15) != 0 && (tile_r + 1) * ROWS > rows;
        unsigned column[8];                   // !WIDE: the largest magnitude of each of this lane's columns
        if constexpr (!WIDE) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                unsigned m = 0;
#pragma unroll
                for (int i = 0; i < R; ++i) m = max_u32(m, magnitude(i, j));
                m = across_wave(m);
                if ((tid & 63) < LANES) most[wave * COLS + cg * 8 + j] = m;
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                column[j] = most[cg * 8 + j];
#pragma unroll
                for (int w = 1; w < WAVES; ++w) column[j] = max_u32(column[j], most[w * COLS + cg * 8 + j]);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            BlockScale s = one;
            if constexpr (!WIDE) {
                s.template set<F8>(column[j]);
                if (rg == 0 && c0 + j < cols) args.scale_t[(c0 + j) * args.blocks_r + tile_r] = s.scale;
            }
#pragma unroll
            for (int i = 0; i < R; i += 4) {
                unsigned o = pack_f8<F8>(s(value(i, j)), s(value(i + 1, j)), s(value(i + 2, j)), s(value(i + 3, j)));
                if (ends) o = first_bytes(o, rows - r0 - i);
                *reinterpret_cast<unsigned*>(turned + (cg * 8 + j) * PITCH + rg * R + i) = o;
            }
        }
        __syncthreads();
        // 16 bytes per lane: eight lanes a row of 128 bytes
        const long at = tile_r * QB + (tid & 7) * 16;
#pragma unroll
        for (int k = 0; k < COLS * 8 / THREADS; ++k) {
            const int c = k * (THREADS / 8) + (tid >> 3);
            const u32x4 v = *reinterpret_cast<const u32x4*>(turned + c * PITCH + (tid & 7) * 16);
            if (tile_c * COLS + c < cols && at < args.pitch_t) put(args.q_t + (tile_c * COLS + c) * args.pitch_t + at, v);
        }
    }
}

// ---- host side -------------------------------------------------------------------------------

template <int DT, int F8, bool WIDE, int OUT, int R, int ROWS, int LANES, int POLICY>
static int launch_quantize(const QuantArgs& a, hipStream_t stream) {
    constexpr int THREADS = ROWS / R * LANES, COLS = LANES * 8;
    const long tiles = ((a.rows + ROWS - 1) / ROWS) * ((a.cols + COLS - 1) / COLS);
    if (tiles * THREADS >= 1l << 32) return fail(SP_ERR_SHAPE, "sp_quantize_blocks: too large");
    hipLaunchKernelGGL((quantize_kernel<DT, F8, WIDE, OUT, R, ROWS, LANES, POLICY>), dim3((unsigned)tiles), dim3(THREADS), 0, stream, a.x, a.rows, a.cols, a);
    return check_launch("sp_quantize_blocks");
}

// Rows per lane of the 128 x 128 tiles: 4 (eight waves) where a tile has one scale, 8 where every row or column has its own, whose steps across
// lanes count then.  (us, 8 / 4 rows: 8192 x 4096 bf16 both ways in 128 x 128 blocks 22.6 / 22.2; 16384 x 4096 both ways in rows of 128
// 60.1 / 69.5, transposed alone 43.8 / 50.2.  Written back instead of streamed 27.5 / 25.8, 62.8 / 67.7, 44.9 / 49.)
// Where the chip has less than two tiles a unit the way through one counts, 4 rows per lane: 16 x 4096 bf16 both ways in rows of 128 7.4 / 6.5,
// 512 x 1024 7.3 / 6.7, 2047 x 3000 12.7 / 12.4; 2048 x 4096, two a unit, is on 8.
// Transposed alone, in tiles of 64 columns and 4 rows per lane there: 5001 x 1003 f32 11.1 / 10.1,
// 512 x 1024 bf16 5.6 / 4.8; 2048 x 4096 bf16, two a unit, 9.0 / 9.15, 8192 x 4096 21.6 / 22.8.
template <int DT, int F8, int POLICY>
static int quantize(const QuantArgs& a, bool wide, hipStream_t stream) {
    const int out = (a.q != nullptr ? 1 : 0) | (a.q_t != nullptr ? 2 : 0);
    if (wide) {
        if (out == 1) return launch_quantize<DT, F8, true, 1, 4, QB, 16, POLICY>(a, stream);
        if (out == 2) return launch_quantize<DT, F8, true, 2, 4, QB, 16, POLICY>(a, stream);
        return launch_quantize<DT, F8, true, 3, 4, QB, 16, POLICY>(a, stream);
    }
    if (out == 1) return launch_quantize<DT, F8, false, 1, 1, 16, 16, POLICY>(a, stream);
    if (out == 2) {
        if constexpr (POLICY == ST_PLAIN)
            if (a.blocks_r * a.blocks_c < 2 * device_cu_count()) return launch_quantize<DT, F8, false, 2, 4, QB, 8, POLICY>(a, stream);
        return launch_quantize<DT, F8, false, 2, 8, QB, 16, POLICY>(a, stream);
    }
    if constexpr (POLICY == ST_PLAIN)
        if (a.blocks_r * a.blocks_c < 2 * device_cu_count()) return launch_quantize<DT, F8, false, 3, 4, QB, 16, POLICY>(a, stream);
    return launch_quantize<DT, F8, false, 3, 8, QB, 16, POLICY>(a, stream);
}

namespace {
struct QuantizeKernelNames {
    QuantizeKernelNames() {
        register_kernel("quantize_rows", (const void*)quantize_kernel<SP_BF16, SP_F8_E4M3, false, 1, 1, 16, 16, ST_STREAM>, 256);
        register_kernel("quantize_both", (const void*)quantize_kernel<SP_BF16, SP_F8_E4M3, false, 3, 8, QB, 16, ST_STREAM>, 256);
        register_kernel("quantize_both_128", (const void*)quantize_kernel<SP_BF16, SP_F8_E4M3, true, 3, 4, QB, 16, ST_STREAM>, 512);
    }
} quantize_kernel_names;
}  // namespace

}  // namespace sp

using namespace sp;

extern "C" int sp_quantize_blocks(int dtype, int f8, int32_t block_rows, const void* x, void* q, float* scale, void* q_t, float* scale_t,
                                  int64_t rows, int64_t cols, void* stream) {
    SP_REQUIRE_PTR(x);
    SP_OPTIONAL_PTR(q);
    SP_OPTIONAL_PTR(scale);
    SP_OPTIONAL_PTR(q_t);
    SP_OPTIONAL_PTR(scale_t);
    if (q == nullptr && q_t == nullptr) return fail(SP_ERR_NULL, "sp_quantize_blocks: q and q_t are NULL");
    if ((q == nullptr) != (scale == nullptr) || (q_t == nullptr) != (scale_t == nullptr))
        return fail(SP_ERR_NULL, "sp_quantize_blocks: numbers and their scales go together");
    if (dtype != SP_F32 && dtype != SP_F16 && dtype != SP_BF16) return fail(SP_ERR_DTYPE, "sp_quantize_blocks: dtype must be f32, f16 or bf16, got %d", dtype);
    if (f8 != SP_F8_E4M3 && f8 != SP_F8_E5M2) return fail(SP_ERR_DTYPE, "sp_quantize_blocks: f8 must be e4m3 or e5m2, got %d", f8);
    if (block_rows != 1 && block_rows != QB) return fail(SP_ERR_ARG, "sp_quantize_blocks: blocks have 1 or 128 rows, got %d", block_rows);
    if (rows <= 0 || cols <= 0) return fail(SP_ERR_SHAPE, "sp_quantize_blocks: rows and cols must be positive (got %lld, %lld)", (long long)rows, (long long)cols);
    if (rows > (int64_t)1 << 31 || cols > (int64_t)1 << 31) return fail(SP_ERR_SHAPE, "sp_quantize_blocks: too large");
    const int rc = require_gfx950(__func__);
    if (rc != SP_OK) return rc;
    QuantArgs a{};
    a.x = x; a.q = (unsigned char*)q; a.q_t = (unsigned char*)q_t; a.scale = scale; a.scale_t = scale_t; a.rows = rows; a.cols = cols;
    a.pitch = (cols + 15) / 16 * 16; a.pitch_t = (rows + 15) / 16 * 16;
    a.blocks_c = (cols + QB - 1) / QB; a.blocks_r = (rows + QB - 1) / QB;
    // results that do not stay in the caches (32 MiB of L2) are streamed past them
    const bool large = ((q != nullptr ? rows * a.pitch : 0) + (q_t != nullptr ? cols * a.pitch_t : 0)) > (int64_t)32 << 20;
    const bool wide = block_rows == QB;
    auto by_policy = [&](auto dt, auto type) {
        constexpr int DT = decltype(dt)::value, F8 = decltype(type)::value;
        return large ? quantize<DT, F8, ST_STREAM>(a, wide, (hipStream_t)stream) : quantize<DT, F8, ST_PLAIN>(a, wide, (hipStream_t)stream);
    };
    auto by_f8 = [&](auto dt) {
        return f8 == SP_F8_E4M3 ? by_policy(dt, std::integral_constant<int, SP_F8_E4M3>{}) : by_policy(dt, std::integral_constant<int, SP_F8_E5M2>{});
    };
    if (dtype == SP_F32) return by_f8(std::integral_constant<int, SP_F32>{});
    if (dtype == SP_F16) return by_f8(std::integral_constant<int, SP_F16>{});
    return by_f8(std::integral_constant<int, SP_BF16>{});
}
