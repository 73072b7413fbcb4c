// Layer norm of rows, and its gradients.
//
// Forward: a row stays in the registers of its T lanes, so it is read once: mean, then the mean of the squares of what is left of it (no
// difference of large sums), then the results.  Bound by memory: 2 rows of traffic per row.
//
// Backward: with h = (x - mean) rstd and g = dy w, dx = rstd (g - mean(g) - h mean(g h)) needs two sums over the row, and
// dw = sum of dy h, db = sum of dy over all rows two per column.  A lane has the same columns of every row that its group of T lanes takes,
// so both of a column's sums stay in its registers until the rows are done; the groups of a workgroup then add theirs up in
// LDS, and the workgroups' sums, one row each in the workspace, are added by a second launch, always in the same order.
#include "vec_io.h"

#include <algorithm>

namespace sp {

constexpr int NORM_MOST_COLS = 16384;

// Results that do not stay in the caches anyway (32 MiB of L2) are streamed past them: 16384 x 4096 bf16, forward and backward, 146 -> 133 us.
__device__ __forceinline__ bool streamed(long rows, int cols, int bytes) { return rows * cols * bytes > 32l << 20; }
template <int DT>
__device__ __forceinline__ void put16(bool stream, void* p, long at, long left, const float (&v)[PER16<DT>]) {
    if (stream) store16<DT, ST_STREAM>(p, at, left, v);
    else store16<DT>(p, at, left, v);
}

// The sums of v over a group of T lanes, a power of two.  A group wider than a wave goes through `slots` (T / 64 floats per sum of LDS of this group) and
// is joined by a barrier of the whole workgroup; `slots` must not be used again before another one.
template <int T, int N>
__device__ __forceinline__ void group_sums(float (&v)[N], float* slots) {
    constexpr int W = T / 64;
    auto add = [](float a, float b) { return a + b; };
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = group_reduce<T < 64 ? T : 64>(v[i], add);
    if constexpr (W > 1) {
        const int wave = (threadIdx.x % T) >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) slots[i * W + wave] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = slots[i * W];
#pragma unroll
            for (int w = 1; w < W; ++w) s += slots[i * W + w];
            v[i] = s;
        }
    }
}

// The N columns that piece `at` of a row stands for: from `col` on, of which the first `skip` are its neighbour's.  The last piece of a row that is no
// multiple of N begins where its 16 bytes end with the row, so that it is one load and one store like the others (element by
// element 33554432 / 2500 rows of 2500 bf16, forward and backward, took 143 us, whole 70): what it has twice counts once, and is stored twice with
// the same bits.  A row of fewer than N columns is one piece, loaded element by element.
// WHOLE: rows are a multiple of N, and there is none of that to keep track of (16384 x 4096 bf16, forward and backward, 134 us without it, 129 with).
template <int N, bool WHOLE>
struct Piece {
    int col, skip;
    __device__ __forceinline__ Piece(int at, int cols) {
        const int wanted = at * N, last = cols - N;
        if constexpr (WHOLE) {
            col = wanted;
            skip = wanted < cols ? 0 : N;
        } else {
            col = wanted <= last || cols < N ? wanted : last;
            skip = wanted < cols ? wanted - col : N;
            col = skip < N ? col : 0;
        }
    }
    __device__ __forceinline__ bool mine() const { return skip < N; }
    // Whether element i is a column that this piece counts.
    __device__ __forceinline__ bool counts(int i, int cols) const { return WHOLE ? mine() : i >= skip && col + i < cols; }
    template <int DT>
    __device__ __forceinline__ u32x4 load(const void* p, long row_at, int cols, bool ok) const {
        u32x4 v = {0u, 0u, 0u, 0u};
        if (!WHOLE && cols < N) v = load_each<DT>(p, row_at + col, ok && mine() ? cols - col : 0);
        else if (ok && mine()) v = load_aligned<WHOLE ? 16 : ELEM_BYTES<DT>, u32x4>((const unsigned char*)p + (row_at + col) * ELEM_BYTES<DT>);
        return v;
    }
};
// N weights from column `col` on (all of them exist where the row has N columns).
template <int WT, int N, bool WHOLE>
__device__ __forceinline__ void load_weights(const void* weight, float otherwise, const Piece<N, WHOLE>& piece, int cols, float (&w)[N]) {
    const int col = piece.col;
#pragma unroll
    for (int h = 0; h < N; h += PER16<WT>) {
        u32x4 v = {0u, 0u, 0u, 0u};
        if (weight != nullptr && (!WHOLE || piece.mine())) {
            if (!WHOLE && cols < N) v = load_each<WT>(weight, col + h, cols - col - h);
            else v = load_aligned<WHOLE ? 16 : ELEM_BYTES<WT>, u32x4>((const unsigned char*)weight + (col + h) * ELEM_BYTES<WT>);
        }
#pragma unroll
        for (int i = 0; i < PER16<WT>; ++i) w[h + i] = weight != nullptr ? element<WT>(v, i) : otherwise;
    }
}

// T lanes per row, C 16-byte pieces of it per lane; a workgroup takes ROWS rows at a time.
template <int DT, int WT, int T, int C, bool WHOLE>
__global__ __launch_bounds__(T < 256 ? 256 : T) void layer_norm_kernel(const void* x, const void* weight, const void* bias, void* y, long rows,
                                                                      int cols, float eps, float* mean_out, float* rstd_out) {
    constexpr int N = PER16<DT>, ROWS = T < 256 ? 256 / T : 1;
    __shared__ float slots[2][T < 64 ? 1 : T / 64 * ROWS];
    const int t = threadIdx.x % T, group = threadIdx.x / T;
    const float count = (float)cols;
    const bool stream = streamed(rows, cols, ELEM_BYTES<DT>);
    for (long first = (long)blockIdx.x * ROWS; first < rows; first += (long)gridDim.x * ROWS) {
        const long row = first + group;
        const bool ok = row < rows;                        // (one row per workgroup: always)
        u32x4 raw[C];
#pragma unroll
        for (int c = 0; c < C; ++c) raw[c] = Piece<N, WHOLE>(c * T + t, cols).template load<DT>(x, row * cols, cols, ok);
        float s[1] = {0.f};
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const Piece<N, WHOLE> piece(c * T + t, cols);
#pragma unroll
            for (int i = 0; i < N; ++i) s[0] += piece.counts(i, cols) ? element<DT>(raw[c], i) : 0.f;
        }
        group_sums<T>(s, slots[0] + group * (T / 64));
        // (equal numbers have themselves as their mean where their sums are exact: in bf16, in f16 up to 8192 columns; in f32 it may be the roundings of the sum off)
        const float mean = s[0] / count;
        float q[1] = {0.f};
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const Piece<N, WHOLE> piece(c * T + t, cols);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float d = element<DT>(raw[c], i) - mean;
                q[0] += piece.counts(i, cols) ? d * d : 0.f;
            }
        }
        group_sums<T>(q, slots[1] + group * (T / 64));
        const float rstd = 1.f / sqrtf(q[0] / count + eps);
        if (ok && t == 0) {
            if (mean_out != nullptr) mean_out[row] = mean;
            if (rstd_out != nullptr) rstd_out[row] = rstd;
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const Piece<N, WHOLE> piece(c * T + t, cols);
            if (!ok || !piece.mine()) continue;
            float w[N], b[N], o[N];
            load_weights<WT>(weight, 1.f, piece, cols, w);
            load_weights<WT>(bias, 0.f, piece, cols, b);
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] = (element<DT>(raw[c], i) - mean) * rstd * w[i] + b[i];
            put16<DT>(stream, y, row * cols + piece.col, cols - piece.col, o);
        }
    }
}

// T lanes per row, C pieces of it per lane, 1024 / T rows at a time in a workgroup; SUMS: dweight and dbias are wanted.
// With 8 columns per lane the weights and the next row fit its 128 registers as well; with 16 (rows of more than 8192) they do not, and the
// sums over rows, which would not either, are in LDS, every lane's own (in registers,
// spilled: 2048 x 16384 bf16, forward and backward, 103 us, in LDS 93; 37 x 12887 30, 18).
template <int DT, int WT, int T, int C, bool SUMS, bool WHOLE>
__global__ __launch_bounds__(1024) void layer_norm_backward_kernel(const void* dy, const void* x, const float* mean, const float* rstd, long rows,
                                                                  int cols, const void* weight, void* dx, float* partial) {
    constexpr int N = PER16<DT>, GROUPS = 1024 / T, W = T < 64 ? 1 : T / 64;
    constexpr bool AHEAD = C * N <= 8, IN_LDS = SUMS && !AHEAD;
    static_assert(AHEAD || GROUPS == 1, "nothing to join where the sums are in LDS");
    extern __shared__ __attribute__((aligned(16))) float sums[];          // SUMS: 512 lanes x C N floats; IN_LDS: 1024 lanes x 2 C N
    __shared__ float slots[2][GROUPS * 2 * W];
    const int t = threadIdx.x % T, group = threadIdx.x / T;
    const float count = (float)cols;
    const bool stream = streamed(rows, cols, ELEM_BYTES<DT>);
    auto load_weight = [&](int c, float(&w)[N]) { load_weights<WT>(weight, 1.f, Piece<N, WHOLE>(c * T + t, cols), cols, w); };
    float kept[AHEAD ? C : 1][N], dw[C][N], db[C][N];
    f32x4* const mine = reinterpret_cast<f32x4*>(sums) + threadIdx.x;     // IN_LDS: 4 of dw at mine[1024 (c N / 4 + i / 4)], db behind them
#pragma unroll
    for (int c = 0; c < C; ++c) {
        if constexpr (AHEAD) load_weight(c, kept[c]);
#pragma unroll
        for (int i = 0; i < N; ++i) dw[c][i] = db[c][i] = 0.f;
    }
    if constexpr (IN_LDS)
#pragma unroll
        for (int q = 0; q < C * N / 2; ++q) mine[1024 * q] = f32x4{0.f, 0.f, 0.f, 0.f};
    // what is in LDS of a piece's sums, into registers and back
    auto bring = [&](int c, bool back) {
        if constexpr (IN_LDS)
#pragma unroll
            for (int h = 0; h < N; h += 4)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    f32x4* at = mine + 1024 * (((k * C + c) * N + h) / 4);
                    float* v = (k == 0 ? dw[c] : db[c]) + h;
                    if (back) *at = f32x4{v[0], v[1], v[2], v[3]};
                    else {
                        const f32x4 q = *at;
                        v[0] = q[0], v[1] = q[1], v[2] = q[2], v[3] = q[3];
                    }
                }
    };
    u32x4 xr[C], gr[C];
    float m = 0.f, r = 0.f;
    auto fetch = [&](long row) {
        const bool ok = row < rows;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const Piece<N, WHOLE> piece(c * T + t, cols);
            xr[c] = piece.template load<DT>(x, row * cols, cols, ok);
            gr[c] = piece.template load<DT>(dy, row * cols, cols, ok);
        }
        m = ok ? mean[row] : 0.f;
        r = ok ? rstd[row] : 0.f;
    };
    const long step = (long)gridDim.x * GROUPS;
    long first = (long)blockIdx.x * GROUPS;
    if constexpr (AHEAD) fetch(first + group);
    int turn = 0;
    for (; first < rows; first += step) {
        const long row = first + group;
        if constexpr (!AHEAD) fetch(row);
        u32x4 xv[C], gv[C];
        const float mu = m, rs = r;
#pragma unroll
        for (int c = 0; c < C; ++c) xv[c] = xr[c], gv[c] = gr[c];
        if constexpr (AHEAD) fetch(row + step);            // the next row comes in while this one is added up
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const Piece<N, WHOLE> piece(c * T + t, cols);
            float now[N];
            if constexpr (!AHEAD) load_weight(c, now);
            bring(c, false);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const bool counts = piece.counts(i, cols);
                const float d = counts ? element<DT>(gv[c], i) : 0.f, h = counts ? (element<DT>(xv[c], i) - mu) * rs : 0.f, g = d * (AHEAD ? kept[AHEAD ? c : 0][i] : now[i]);
                s[0] += g;
                s[1] += g * h;
                dw[c][i] += d * h;
                db[c][i] += d;
            }
            bring(c, true);
        }
        group_sums<T>(s, slots[turn] + group * 2 * W);
        turn ^= 1;
        const float a = s[0] / count, b = s[1] / count;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const Piece<N, WHOLE> piece(c * T + t, cols);
            if (row >= rows || !piece.mine()) continue;
            float o[N], now[N];
            if constexpr (!AHEAD) load_weight(c, now);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float g = element<DT>(gv[c], i) * (AHEAD ? kept[AHEAD ? c : 0][i] : now[i]), h = (element<DT>(xv[c], i) - mu) * rs;
                o[i] = rs * (g - a - h * b);
            }
            put16<DT>(stream, dx, row * cols + piece.col, cols - piece.col, o);
        }
    }
    if constexpr (SUMS) {
        // the upper half of the groups hands its sums to the lower half until one is left; dw and db one after the other
        auto join = [&](float(&v)[C][N]) {
#pragma unroll
            for (int half = GROUPS / 2; half >= 1; half /= 2) {
                __syncthreads();
                if (group >= half && group < 2 * half)
#pragma unroll
                    for (int c = 0; c < C; ++c)
#pragma unroll
                        for (int i = 0; i < N; ++i) sums[(c * N + i) * 512 + threadIdx.x - half * T] = v[c][i];
                __syncthreads();
                if (group < half)
#pragma unroll
                    for (int c = 0; c < C; ++c)
#pragma unroll
                        for (int i = 0; i < N; ++i) v[c][i] += sums[(c * N + i) * 512 + threadIdx.x];
            }
        };
        join(dw);
        join(db);
        if (group == 0) {
            float* out = partial + (long)blockIdx.x * 2 * cols;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const Piece<N, WHOLE> piece(c * T + t, cols);
                bring(c, false);
                if ((WHOLE || GROUPS == 1) && piece.skip == 0 && (WHOLE || cols >= N)) {           // (all of them counted: in whole pieces; one by one 5 x 7909 f16, forward and backward, took 18.8 us, 13.1)
#pragma unroll
                    for (int h = 0; h < N; h += 4) {
                        const float w[4] = {dw[c][h], dw[c][h + 1], dw[c][h + 2], dw[c][h + 3]}, b[4] = {db[c][h], db[c][h + 1], db[c][h + 2], db[c][h + 3]};
                        store16<SP_F32>(out, piece.col + h, 4, w);
                        store16<SP_F32>(out, cols + piece.col + h, 4, b);
                    }
                    continue;
                }
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (piece.counts(i, cols)) {
                        out[piece.col + i] = dw[c][i];
                        out[cols + piece.col + i] = db[c][i];
                    }
            }
        }
    }
}

// The sums of `parts` rows of 2 cols columns: dweight, then dbias.  64 columns to a workgroup, its 16 waves take the parts in turn, eight loads of a
// wave under way at a time (one at a time, 256 parts took 10.2 us).
constexpr int SUM_WAVES = 16, SUM_AHEAD = 8;
__global__ __launch_bounds__(SUM_WAVES * 64) void layer_norm_sums_kernel(const float* partial, int parts, int cols, float* dweight, float* dbias) {
    __shared__ float sums[SUM_WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = blockIdx.x * 64 + lane, all = 2 * cols;
    float s = 0.f;
    if (col < all)
        for (int p = wave; p < parts; p += SUM_WAVES * SUM_AHEAD) {
            float v[SUM_AHEAD];
#pragma unroll
            for (int u = 0; u < SUM_AHEAD; ++u) v[u] = p + u * SUM_WAVES < parts ? partial[(long)(p + u * SUM_WAVES) * all + col] : 0.f;
#pragma unroll
            for (int u = 0; u < SUM_AHEAD; ++u) s += v[u];
        }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && col < all) {
#pragma unroll
        for (int w = 1; w < SUM_WAVES; ++w) s += sums[w][lane];
        if (col < cols) dweight[col] = s;
        else dbias[col - cols] = s;
    }
}

// ---- host side -------------------------------------------------------------------------------

struct NormArgs {
    const void *x, *weight, *bias, *dy;
    void *y, *dx;
    float *mean, *rstd;
    const float *mean_in, *rstd_in;
    float *dweight, *dbias, *partial;
    long rows;
    int cols;
    float eps;
    hipStream_t stream;
};

template <int DT>
static bool whole_pieces(const NormArgs& a) { return a.cols % PER16<DT> == 0; }

template <int DT, int WT, int T, int C>
static int launch_forward(const NormArgs& a) {
    constexpr int THREADS = T < 256 ? 256 : T, ROWS = THREADS / T;
    const long blocks = (a.rows + ROWS - 1) / ROWS, most = 1l << 20;       // (a launch counts its work items in 32 bits)
    auto kernel = whole_pieces<DT>(a) ? layer_norm_kernel<DT, WT, T, C, true> : layer_norm_kernel<DT, WT, T, C, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(THREADS), 0, a.stream, a.x,
                       a.weight, a.bias, a.y, a.rows, a.cols, a.eps, a.mean, a.rstd);
    return check_launch("sp_layer_norm");
}

template <int DT, int WT>
static int forward(const NormArgs& a) {
    // few lanes per row as long as a wave can hold it; three pieces per lane where four would leave a quarter of them idle
    const int pieces = (a.cols + PER16<DT> - 1) / PER16<DT>;
    if (pieces <= 8) return launch_forward<DT, WT, 8, 1>(a);
    if (pieces <= 16) return launch_forward<DT, WT, 16, 1>(a);
    if (pieces <= 32) return launch_forward<DT, WT, 32, 1>(a);
    if (pieces <= 64) return launch_forward<DT, WT, 64, 1>(a);
    if (pieces <= 128) return launch_forward<DT, WT, 64, 2>(a);
    if (pieces <= 256) return launch_forward<DT, WT, 64, 4>(a);
    // rows for two workgroups a unit or less: the shortest way through one (us, this / the rules below: 16 x 4096 bf16 3.1 / 3.4, 5 x 7909 f16 4.3 / 6.3,
    // 256 x 8192 bf16 4.5 / 5.1; 16384 x 4096 80 / 68; with two pieces a lane 100 x 12887 6.9 / 7.5, but 512 x 16384 11.1 / 10.4)
    if (a.rows <= 2 * device_cu_count()) {
        if (pieces <= 512) return launch_forward<DT, WT, 512, 1>(a);
        if (pieces <= 1024) return launch_forward<DT, WT, 1024, 1>(a);
    }
    if (pieces <= 512) return launch_forward<DT, WT, 256, 2>(a);
    if (pieces <= 768) return launch_forward<DT, WT, 256, 3>(a);
    if (pieces <= 1024) return launch_forward<DT, WT, 256, 4>(a);
    if (pieces <= 1536) return launch_forward<DT, WT, 512, 3>(a);
    if constexpr (DT == SP_F32)
        if (pieces > 2048) return launch_forward<DT, WT, 1024, 4>(a);
    return launch_forward<DT, WT, 512, 4>(a);
}

static int backward_blocks(int64_t rows) {
    const int cus = device_cu_count();
    return (int)(rows < cus ? rows : cus);
}

template <int DT, int WT, int T, int C, bool SUMS>
static int launch_backward(const NormArgs& a) {
    constexpr int GROUPS = 1024 / T;
    const int blocks = (int)std::min<long>(backward_blocks(a.rows), (a.rows + GROUPS - 1) / GROUPS);
    auto kernel = whole_pieces<DT>(a) ? layer_norm_backward_kernel<DT, WT, T, C, SUMS, true> : layer_norm_backward_kernel<DT, WT, T, C, SUMS, false>;
    constexpr int columns = C * PER16<DT>;               // of a lane
    const int lds_bytes = !SUMS ? 0 : columns > 8 ? 1024 * 2 * columns * 4 : GROUPS > 1 ? 512 * columns * 4 : 0;
    if (const int rc = ensure_dynamic_lds((const void*)kernel, lds_bytes); rc != SP_OK) return rc;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(1024), lds_bytes, a.stream, a.dy, a.x, a.mean_in, a.rstd_in, a.rows, a.cols, a.weight, a.dx, a.partial);
    if (const int rc = check_launch("sp_layer_norm_backward"); rc != SP_OK || !SUMS) return rc;
    hipLaunchKernelGGL(layer_norm_sums_kernel, dim3((2 * a.cols + 63) / 64), dim3(SUM_WAVES * 64), 0, a.stream, a.partial, blocks, a.cols, a.dweight, a.dbias);
    return check_launch("sp_layer_norm_backward");
}

template <int DT, int WT, bool SUMS>
static int backward(const NormArgs& a) {
    constexpr int C = 8 / PER16<DT>;                       // 8 columns per lane
    if (a.cols <= 8 * 8) return launch_backward<DT, WT, 8, C, SUMS>(a);
    if (a.cols <= 16 * 8) return launch_backward<DT, WT, 16, C, SUMS>(a);
    if (a.cols <= 32 * 8) return launch_backward<DT, WT, 32, C, SUMS>(a);
    if (a.cols <= 64 * 8) return launch_backward<DT, WT, 64, C, SUMS>(a);
    if (a.cols <= 128 * 8) return launch_backward<DT, WT, 128, C, SUMS>(a);
    if (a.cols <= 256 * 8) return launch_backward<DT, WT, 256, C, SUMS>(a);
    if (a.cols <= 512 * 8) return launch_backward<DT, WT, 512, C, SUMS>(a);
    if (a.cols <= 1024 * 8) return launch_backward<DT, WT, 1024, C, SUMS>(a);
    return launch_backward<DT, WT, 1024, 2 * C, SUMS>(a);
}

// f<input type, weight type>()
template <typename F>
static int by_types(int dtype, int weight_dtype, F f) {
    typedef std::integral_constant<int, SP_F32> f32;
    typedef std::integral_constant<int, SP_F16> f16;
    typedef std::integral_constant<int, SP_BF16> bf16;
    const bool wide = weight_dtype == SP_F32;
    switch (dtype) {
        case SP_F32: return f(f32{}, f32{});
        case SP_F16: return wide ? f(f16{}, f32{}) : f(f16{}, f16{});
        default: return wide ? f(bf16{}, f32{}) : f(bf16{}, bf16{});
    }
}

static int check_norm(const char* fn, int dtype, int weight_dtype, int64_t rows, int64_t cols) {
    if (dtype != SP_F32 && dtype != SP_F16 && dtype != SP_BF16) return fail(SP_ERR_DTYPE, "%s: dtype must be f32, f16 or bf16, got %d", fn, dtype);
    if (weight_dtype != SP_F32 && weight_dtype != dtype) return fail(SP_ERR_DTYPE, "%s: weights are f32 or of the rows' type, got %d", fn, weight_dtype);
    if (rows <= 0 || cols <= 0) return fail(SP_ERR_SHAPE, "%s: rows and cols must be positive (got %lld, %lld)", fn, (long long)rows, (long long)cols);
    if (cols > NORM_MOST_COLS) return fail(SP_ERR_SHAPE, "%s: cols must be <= %d, got %lld", fn, NORM_MOST_COLS, (long long)cols);
    if (rows > (int64_t)1 << 40) return fail(SP_ERR_SHAPE, "%s: too large", fn);
    return SP_OK;
}

namespace {
struct NormKernelNames {
    NormKernelNames() {
        register_kernel("layer_norm", (const void*)layer_norm_kernel<SP_BF16, SP_F32, 256, 2, true>, 256);
        register_kernel("layer_norm_backward", (const void*)layer_norm_backward_kernel<SP_BF16, SP_F32, 512, 1, true, true>, 1024);
    }
} norm_kernel_names;
}  // namespace

}  // namespace sp

using namespace sp;

extern "C" int sp_layer_norm(int dtype, int weight_dtype, const void* x, const void* weight, const void* bias, void* y, float* mean_out,
                             float* rstd_out, int64_t rows, int64_t cols, float eps, void* stream) {
    SP_REQUIRE_PTR(x);
    SP_REQUIRE_PTR(y);
    SP_OPTIONAL_PTR(weight);
    SP_OPTIONAL_PTR(bias);
    SP_OPTIONAL_PTR(mean_out);
    SP_OPTIONAL_PTR(rstd_out);
    int rc = check_norm(__func__, dtype, weight_dtype, rows, cols);
    if (rc != SP_OK) return rc;
    if (!(eps >= 0.f) || eps > 3.4e38f) return fail(SP_ERR_ARG, "sp_layer_norm: eps must be finite and not negative, got %g", (double)eps);
    rc = require_gfx950(__func__);
    if (rc != SP_OK) return rc;
    NormArgs a{};
    a.x = x; a.weight = weight; a.bias = bias; a.y = y; a.mean = mean_out; a.rstd = rstd_out;
    a.rows = rows; a.cols = (int)cols; a.eps = eps; a.stream = (hipStream_t)stream;
    return by_types(dtype, weight_dtype, [&](auto dt, auto wt) { return forward<decltype(dt)::value, decltype(wt)::value>(a); });
}

extern "C" int64_t sp_layer_norm_backward_workspace_bytes(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0 || cols > NORM_MOST_COLS) return 0;
    return (int64_t)backward_blocks(rows) * 2 * cols * 4;
}

extern "C" int sp_layer_norm_backward(int dtype, int weight_dtype, const void* dy, const void* x, const float* mean, const float* rstd,
                                      const void* weight, void* dx, float* dweight, float* dbias, int64_t rows, int64_t cols,
                                      void* workspace, int64_t workspace_bytes, void* stream) {
    SP_REQUIRE_PTR(dy);
    SP_REQUIRE_PTR(x);
    SP_REQUIRE_PTR(mean);
    SP_REQUIRE_PTR(rstd);
    SP_OPTIONAL_PTR(weight);
    SP_REQUIRE_PTR(dx);
    SP_OPTIONAL_PTR(dweight);
    SP_OPTIONAL_PTR(dbias);
    int rc = check_norm(__func__, dtype, weight_dtype, rows, cols);
    if (rc != SP_OK) return rc;
    if ((dweight == nullptr) != (dbias == nullptr)) return fail(SP_ERR_ARG, "sp_layer_norm_backward: dweight and dbias are both given or both NULL");
    if (dweight != nullptr) {
        SP_REQUIRE_PTR(workspace);
        if (workspace_bytes < sp_layer_norm_backward_workspace_bytes(rows, cols))
            return fail(SP_ERR_ARG, "sp_layer_norm_backward: workspace of %lld bytes, %lld are needed", (long long)workspace_bytes,
                        (long long)sp_layer_norm_backward_workspace_bytes(rows, cols));
    }
    rc = require_gfx950(__func__);
    if (rc != SP_OK) return rc;
    NormArgs a{};
    a.dy = dy; a.x = x; a.mean_in = mean; a.rstd_in = rstd; a.weight = weight; a.dx = dx; a.dweight = dweight; a.dbias = dbias;
    a.partial = (float*)workspace; a.rows = rows; a.cols = (int)cols; a.stream = (hipStream_t)stream;
    return by_types(dtype, weight_dtype, [&](auto dt, auto wt) {
        constexpr int DT = decltype(dt)::value, WT = decltype(wt)::value;
        return dweight != nullptr ? backward<DT, WT, true>(a) : backward<DT, WT, false>(a);
    });
}
