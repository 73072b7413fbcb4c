// Log probabilities of one token per row of logits, the entropy of the row and its most likely tokens; and the gradient of the logits.
//
// With m the largest logit, s = sum exp(x - m) and w = sum exp(x - m) (x - m): lse = m + ln s, log p_t = (x_t - m) - ln s, and the entropy
// -sum p ln p = ln s - w / s, two numbers that are not negative, so nothing cancels.  A row is read once: a lane keeps m, s and w of what it has seen
// and scales s and w where m grows; lanes, waves and chunks of a row then join in an order of the sizes alone.
// Backward: dx_j = d_logp [j = t] - p_j (d_logp + d_entropy (ln p_j + H) - d_lse), one read and one write.  p_j = exp(x_j - lse), of lse rounded to f32: that is a
// relative error of up to |lse| 2^-24 which all p of a row share, no more than half a last place of a f32 logit of that size; m and ln s apart would be two numbers of a row to keep.
//
// What rows may hold: -inf has probability 0 (its terms are left out); a row with nothing above -inf has lse -inf, log probability -inf and entropy 0, and
// gradients of 0; the lowest finite number is a logit like any other (x - m is taken before it is scaled, so that it does not
// overflow to a NaN); +inf or a NaN make the sums NaN.
#include "overlap.h"
#include "vec_io.h"

namespace sp {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr float FAR_BELOW = -1e4f;            // of y = (x - m) log2 e: 2^y is 0 there, and 0 * y stays 0 where y alone would be -inf
constexpr int MOST_TOP = 32;                  // alternatives
constexpr int MOST_CHUNKS = 64;               // of a row: one lane each where they join
constexpr int LIST = 2048;                    // candidates for them that a workgroup can hold

struct TokenArgs {
    const int32_t* tokens;
    float *logp, *entropy, *lse, *top_logp;
    int32_t* top_ids;
    int top;
    float* part;                  // of every (row, chunk): m, s, w, and behind all of them `top` values each, and their columns
    float* part_top;
    int32_t* part_ids;
};

// The sums of some of a row's logits, of e = 2^y with y = (x - m) log2 e.
struct Sums {
    float m, s, w;                // w: of e y
};
__device__ __forceinline__ float finite_reference(float m) { return m == -INFINITY ? 0.f : m; }
// What s and w are from another m, which is no smaller.
__device__ __forceinline__ void move_to(Sums& a, float m) {
    const float y = (a.m - finite_reference(m)) * LOG2E, f = __builtin_amdgcn_exp2f(y);
    a.w = f * __builtin_fmaf(a.s, fmaxf(y, FAR_BELOW), a.w);
    a.s *= f;
    a.m = m;
}
__device__ __forceinline__ float add_f32(float a, float b) { return a + b; }
// most: the largest of a.m and x.
template <int N, bool ENTROPY>
__device__ __forceinline__ void take(Sums& a, const float (&x)[N], float most) {
    move_to(a, most);
    const float from = finite_reference(most);
    float s = 0.f, w = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float y = (x[i] - from) * LOG2E, e = __builtin_amdgcn_exp2f(y);
        s += e;
        if constexpr (ENTROPY) w = __builtin_fmaf(e, fmaxf(y, FAR_BELOW), w);
    }
    a.s += s;
    a.w += w;
}

// A row's results from its sums.
struct RowResult {
    bool none;
    float m, ln_s;
    __device__ __forceinline__ explicit RowResult(const Sums& a) : none(a.m == -INFINITY && a.s == 0.f), m(a.m), ln_s(logf(a.s)) {}
    __device__ __forceinline__ float logp(float x) const { return none ? -INFINITY : (x - m) - ln_s; }
};
template <int DT>
__device__ __forceinline__ float logit_at(const void* logits, long at) {
    if constexpr (DT == SP_F32) return ((const float*)logits)[at];
    else return half_bits_to_f32<DT>(((const unsigned short*)logits)[at]);
}
// x: the token's logit, where it counts.
__device__ __forceinline__ void put_sums(const TokenArgs& a, long row, bool counts, float x, const Sums& sums) {
    const RowResult r(sums);
    a.logp[row] = counts ? r.logp(x) : 0.f;
    if (a.lse != nullptr) a.lse[row] = r.none ? -INFINITY : r.m + r.ln_s;
    if (a.entropy != nullptr) a.entropy[row] = r.none ? 0.f : r.ln_s - LN2 * (sums.w / sums.s);
}
template <int DT>
__device__ __forceinline__ void put_row(const TokenArgs& a, const void* logits, long cols, long row, const Sums& sums) {
    const int token = a.tokens[row];
    const bool counts = (unsigned)token < (unsigned)cols;
    put_sums(a, row, counts, counts ? logit_at<DT>(logits, row * cols + token) : 0.f, sums);
}

// ---- the most likely tokens ----
// A logit and its column as one number: larger for the larger logit, of equal ones for the lower column; 0 for what is never taken, -inf and NaN.
typedef unsigned long long Key;
__device__ __forceinline__ Key key_of(float x, int column) {
    if (!(x > -INFINITY)) return 0;
    const unsigned u = __float_as_uint(x + 0.f);                       // (-0 is +0)
    return (Key)(u ^ ((u >> 31) != 0 ? 0xffffffffu : 0x80000000u)) << 32 | (unsigned)~column;
}
__device__ __forceinline__ float logit_of(Key k) {
    const unsigned u = (unsigned)(k >> 32);
    return __uint_as_float(u ^ ((u >> 31) != 0 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int column_of(Key k) { return (int)~(unsigned)k; }
__device__ __forceinline__ Key larger(Key a, Key b) { return a > b ? a : b; }

template <int T>
struct TopLds {
    Key list[LIST];
    Key lanes[T];
    Key subsets[64];
    Key least;
    int count, found;
    unsigned short who[T];
};

// The `top` largest keys of a workgroup's part of a row, in their order, to put(place, key); places behind the last one get key 0.  mine: at most `slack` below the largest key of this
// lane (0: it has none), pieces: how many pieces a lane has, keys(lane, piece, f): f of every key of that lane's piece.
// The 64 largest of lanes apart by 64 hold `top` keys (or all there are) that are no smaller than the top-th of them, so nothing below that one is taken.  The few lanes that have
// something left are listed, their pieces shared out over all lanes, and what is left of them, some two dozen keys for 20 alternatives, goes to a list, where every key counts the larger
// ones.  Where that list is too short (thousands of the largest logits in a few lanes) the workgroup looks for one key after the other.
template <int T, typename Keys, typename Put>
__device__ __forceinline__ void largest_keys(TopLds<T>& lds, Key mine, Key slack, int top, int pieces, const Keys& keys, const Put& put) {
    const int tid = threadIdx.x;
    lds.lanes[tid] = mine;
    if (tid == 0) {
        lds.count = lds.found = 0;
        lds.least = 1;
    }
    __syncthreads();
    if (tid < 64) {
        Key best = 0;
#pragma unroll
        for (int t = 0; t < T; t += 64) best = larger(best, lds.lanes[t + tid]);
        lds.subsets[tid] = best;                           // (one wave: what it writes it reads in order)
        int above = 0;
#pragma unroll 8
        for (int j = 0; j < 64; ++j) above += lds.subsets[j] > best ? 1 : 0;
        if (best != 0 && above == top - 1) lds.least = best;
    }
    __syncthreads();
    const Key least = lds.least;
    if (mine != 0 && mine + slack >= least) lds.who[atomicAdd(&lds.found, 1)] = (unsigned short)tid;
    __syncthreads();
    const int all = lds.found * pieces;
    for (int i = tid; i < all; i += T)
        keys(lds.who[i / pieces], i % pieces, [&](Key k) {
            if (k < least) return;
            const int at = atomicAdd(&lds.count, 1);
            if (at < LIST) lds.list[at] = k;
        });
    __syncthreads();
    const int n = lds.count;
    if (n <= LIST) {
        for (int i = tid; i < n; i += T) {
            const Key k = lds.list[i];
            int above = 0;
            for (int j = 0; j < n; ++j) above += lds.list[j] > k ? 1 : 0;
            if (above < top) put(above, k);
        }
        for (int i = n + tid; i < top; i += T) put(i, (Key)0);
        return;
    }
    Key last = ~(Key)0;
    for (int place = 0; place < top; ++place) {
        Key best = 0;
        for (int i = 0; i < pieces; ++i)
            keys(tid, i, [&](Key k) {
                if (k < last) best = larger(best, k);
            });
#pragma unroll
        for (int d = 1; d < 64; d *= 2) best = larger(best, __shfl_xor(best, d, WAVE));
        __syncthreads();                                   // (the last round's are read)
        if ((tid & 63) == 0) lds.subsets[tid >> 6] = best;
        __syncthreads();
        best = lds.subsets[0];
#pragma unroll
        for (int w = 1; w < T / 64; ++w) best = larger(best, lds.subsets[w]);
        if (tid == 0) put(place, best);
        last = best;
    }
}

// ---- long rows: a workgroup for a chunk of a row ----
// Bound by HBM with the vector ALU close behind (some 11 instructions and one exponential a logit): 256 x 131072 bf16 with entropy 13.1 us (5.1 TB/s), 4096 x 32003 bf16 50.5 us (5.2 TB/s, the ALU
// 75 % busy).  Five alternatives cost 4.4 us more, a chain of four short steps and a trip to memory that nothing covers with one workgroup a unit; two a unit, of half a row, were slower by the join.
// One row of 32003 f32 logits: 5.8 us in 16 chunks and 4.2 for their join, launch and latency.
constexpr int AT_ONCE = 4;        // 16-byte pieces of a lane between two looks at m

template <int DT, int T, bool ENTROPY, bool TOP>
__global__ __launch_bounds__(T) void token_probs_kernel(const void* logits, long cols, unsigned chunks, long chunk_cols, const TokenArgs a) {
    constexpr int P = PER16<DT>, PIECES = T * P, STEP = AT_ONCE * PIECES, N = AT_ONCE * P;
    const int tid = threadIdx.x;
    const long row = blockIdx.x / chunks;
    const unsigned chunk = blockIdx.x - (unsigned)row * chunks;
    const long c0 = (long)chunk * chunk_cols;
    // pieces are those of memory, 16-byte aligned: the first one may begin up to P - 1 logits in front of the chunk, whose columns count from there
    const int front = (int)((row * cols) & (P - 1)), here = (int)(cols - c0 < chunk_cols ? cols - c0 : chunk_cols) + front;
    const long base = row * cols + c0 - front;
    auto inside = [&](int i) { return i >= front && i < here; };
    // piece u of the step from column i0 on
    auto load = [&](int i0, u32x4 (&raw)[AT_ONCE]) {
        if (i0 + STEP <= here) {                           // (of the whole workgroup)
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) raw[u] = *reinterpret_cast<const u32x4*>((const unsigned char*)logits + (base + i0 + u * PIECES + tid * P) * ELEM_BYTES<DT>);
        } else {
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const int i = i0 + u * PIECES + tid * P;
                raw[u] = load16<DT>(logits, base + i, here - i);
            }
        }
    };
    Sums mine{-INFINITY, 0.f, 0.f};
    int best_piece = 0;                                    // the first piece with this lane's largest logit
    auto consume = [&](int i0, const u32x4 (&raw)[AT_ONCE], auto whole) {
        float x[N];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
            for (int e = 0; e < P; ++e) {
                x[u * P + e] = element<DT>(raw[u], e);
                if (!decltype(whole)::value && !inside(i0 + u * PIECES + tid * P + e)) x[u * P + e] = -INFINITY;
            }
        float most = mine.m;
        if constexpr (TOP) {
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                float of_piece = x[u * P];
#pragma unroll
                for (int e = 1; e < P; ++e) of_piece = fmaxf(of_piece, x[u * P + e]);
                best_piece = of_piece > most ? i0 / PIECES + u : best_piece;
                most = fmaxf(most, of_piece);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) most = fmaxf(most, x[i]);
        }
        take<N, ENTROPY>(mine, x, most);
    };
    u32x4 ahead[AT_ONCE];
    load(0, ahead);
    for (int i0 = 0; i0 < here; i0 += STEP) {
        u32x4 raw[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) raw[u] = ahead[u];
        if (i0 + STEP < here) load(i0 + STEP, ahead);
        if (i0 + STEP <= here && (i0 > 0 || front == 0)) consume(i0, raw, std::true_type{});
        else consume(i0, raw, std::false_type{});
    }
    auto keys_of_piece = [&](int lane, int piece, const auto& f) {
        const int i = piece * PIECES + lane * P;
        const u32x4 raw = load16<DT>(logits, base + i, here - i);
#pragma unroll
        for (int e = 0; e < P; ++e) f(inside(i + e) ? key_of(element<DT>(raw, e), (int)c0 + i + e - front) : (Key)0);
    };
    // the largest logit of this lane, with the last column of its piece: which of the columns it is would be another trip to memory (256 x 131072 bf16, five alternatives: 19.0 us, so 17.8)
    const Key best = TOP && mine.m > -INFINITY ? key_of(mine.m, (int)c0 + best_piece * PIECES + tid * P + P - 1 - front) : (Key)0;
    __shared__ Sums waves[T / 64];
    move_to(mine, group_max<64>(mine.m));
    mine.s = group_reduce<64>(mine.s, add_f32);
    if constexpr (ENTROPY) mine.w = group_reduce<64>(mine.w, add_f32);
    if ((tid & 63) == 0) waves[tid >> 6] = mine;
    __syncthreads();
    if (!TOP && tid != 0) return;
    float most = waves[0].m;
#pragma unroll
    for (int w = 1; w < T / 64; ++w) most = fmaxf(most, waves[w].m);
    Sums sums{most, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < T / 64; ++w) {
        Sums one = waves[w];
        move_to(one, most);
        sums.s += one.s;
        sums.w += one.w;
    }
    if (tid == 0) {
        if (chunks == 1) {
            put_row<DT>(a, logits, cols, row, sums);
        } else {
            a.part[3l * blockIdx.x] = sums.m;
            a.part[3l * blockIdx.x + 1] = sums.s;
            a.part[3l * blockIdx.x + 2] = sums.w;
        }
    }
    if constexpr (TOP) {
        __shared__ TopLds<T> lds;
        const long to = (long)blockIdx.x * a.top;
        const RowResult r(sums);
        largest_keys<T>(lds, best, P - 1, a.top, (here + PIECES - 1) / PIECES, keys_of_piece, [&](int place, Key k) {
            if (chunks == 1) {
                a.top_logp[to + place] = k != 0 ? r.logp(logit_of(k)) : -INFINITY;
                a.top_ids[to + place] = k != 0 ? column_of(k) : -1;
            } else {
                a.part_top[to + place] = k != 0 ? logit_of(k) : -INFINITY;
                a.part_ids[to + place] = k != 0 ? column_of(k) : -1;
            }
        });
    }
}

// A row's chunks, a lane of a wave each.
__device__ __forceinline__ Sums join_chunks(const TokenArgs& a, long row, int chunks, int lane) {
    Sums sums{-INFINITY, 0.f, 0.f};
    if (lane < chunks) {
        const float* at = a.part + 3 * (row * chunks + lane);
        sums = Sums{at[0], at[1], at[2]};
    }
    move_to(sums, group_max<64>(sums.m));
    sums.s = group_reduce<64>(sums.s, add_f32);
    sums.w = group_reduce<64>(sums.w, add_f32);
    return sums;
}
template <int DT>
__global__ __launch_bounds__(256) void token_probs_join_kernel(const void* logits, long cols, long rows, int chunks, const TokenArgs a) {
    const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const Sums sums = join_chunks(a, row, chunks, threadIdx.x & 63);
    if ((threadIdx.x & 63) == 0) put_row<DT>(a, logits, cols, row, sums);
}
// The same with the alternatives, a workgroup for a row: every chunk has left its own, largest first, and the row's are among them.
// With `deep` of them a chunk, the (top / deep)-th largest of the chunks' deep-th ones has `top` above it or equal, so nothing below it is taken; `deep` is such that this is one of the
// larger half (of 34 chunks, for 32 alternatives: the 16th of their second ones, with some 60 keys left; the 32nd of their first has 100).
template <int DT>
__global__ __launch_bounds__(256) void token_probs_join_top_kernel(const void* logits, long cols, int chunks, const TokenArgs a) {
    constexpr int T = 256;
    const int tid = threadIdx.x;
    const long row = blockIdx.x;
    const int n = chunks * a.top;
    __shared__ Key keys[MOST_CHUNKS * MOST_TOP], list[MOST_CHUNKS * MOST_TOP];
    __shared__ Key least;
    __shared__ int count;
    for (int i = tid; i < n; i += T) keys[i] = key_of(a.part_top[row * n + i], a.part_ids[row * n + i]);
    if (tid == 0) {
        least = 1;
        count = 0;
    }
    const Sums sums = join_chunks(a, row, chunks, tid & 63);           // (every wave for itself)
    if (tid == 0) put_row<DT>(a, logits, cols, row, sums);
    const RowResult r(sums);
    __syncthreads();
    if (tid < chunks) {
        int deep = 1;
        while (deep < a.top && 2 * ((a.top + deep - 1) / deep) > chunks) ++deep;
        const int place = (a.top + deep - 1) / deep - 1;
        const Key mine = keys[tid * a.top + deep - 1];
        int above = 0;
        for (int c = 0; c < chunks; ++c) above += keys[c * a.top + deep - 1] > mine ? 1 : 0;
        if (mine != 0 && above == place) least = mine;     // (keys differ, but for 0)
    }
    __syncthreads();
    for (int i = tid; i < n; i += T) {
        const Key k = keys[i];
        if (k >= least) list[atomicAdd(&count, 1)] = k;
    }
    __syncthreads();
    auto put = [&](int place, Key k) {
        a.top_logp[row * a.top + place] = k != 0 ? r.logp(logit_of(k)) : -INFINITY;
        a.top_ids[row * a.top + place] = k != 0 ? column_of(k) : -1;
    };
    for (int i = tid; i < count; i += T) {
        const Key k = list[i];
        int above = 0;
        for (int j = 0; j < count; ++j) above += list[j] > k ? 1 : 0;
        if (above < a.top) put(above, k);
    }
    for (int i = count + tid; i < a.top; i += T) put(i, (Key)0);
}

// ---- short rows: T lanes hold one in C pieces each ----
// Bound by HBM: 65536 x 256 f32 with entropy 11.4 us (5.9 TB/s); 5001 x 1003 f16 5.4 us, launch and latency.
template <int DT, int T, int C, bool ENTROPY>
__global__ __launch_bounds__(256) void token_probs_rows_kernel(const void* logits, long cols, long rows, const TokenArgs a) {
    constexpr int P = PER16<DT>, N = C * P;
    const int lane = threadIdx.x % T;
    const long row = (long)blockIdx.x * (256 / T) + threadIdx.x / T;
    if (row >= rows) return;                               // (all lanes of a row)
    const int token = a.tokens[row];
    u32x4 raw[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = (c * T + lane) * P;
        raw[c] = load16<DT>(logits, row * cols + i, cols - i);
    }
    const bool counts = (unsigned)token < (unsigned)cols;
    const float mine = counts && lane == 0 ? logit_at<DT>(logits, row * cols + token) : 0.f;
    float x[N];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < P; ++e) x[c * P + e] = (c * T + lane) * P + e < cols ? element<DT>(raw[c], e) : -INFINITY;
    float most = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) most = fmaxf(most, x[i]);
    most = group_max<T>(fmaxf(most, -INFINITY));           // (a NaN alone in its lane is not handed on)
    Sums sums{most, 0.f, 0.f};
    take<N, ENTROPY>(sums, x, most);
    sums.s = group_reduce<T>(sums.s, add_f32);
    if constexpr (ENTROPY) sums.w = group_reduce<T>(sums.w, add_f32);
    if (lane == 0) put_sums(a, row, counts, mine, sums);
}

// ---- the gradient ----
struct TokenGradArgs {
    const int32_t* tokens;
    const float *lse, *entropy, *d_logp, *d_entropy, *d_lse;
    void* dx;
};

// Bound by HBM: 4096 x 32003 bf16, 524 MB, 82.5 us (6.4 TB/s); 65536 x 256 f32, 134 MB, 20.4 us (6.6).
// T lanes to a row or a chunk of one, U pieces each.
template <int DT, int T, int U, bool ENTROPY, int POLICY>
__global__ __launch_bounds__(256) void token_grad_kernel(const void* logits, long cols, long rows, unsigned chunks, const TokenGradArgs a) {
    constexpr int P = PER16<DT>;
    const int lane = threadIdx.x % T;
    const long part = (long)blockIdx.x * (256 / T) + threadIdx.x / T;
    const long row = part / chunks;
    if (row >= rows) return;
    const long c0 = (part - row * chunks) * (T * U * P);
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long i = c0 + (u * T + lane) * P;
        raw[u] = load16<DT>(logits, row * cols + i, cols - i);
    }
    const float lse = a.lse[row];
    const int token = a.tokens[row];
    const bool counts = (unsigned)token < (unsigned)cols, none = lse == -INFINITY;
    const float of_token = a.d_logp != nullptr && counts && !none ? a.d_logp[row] : 0.f;
    float slope = 0.f, all = of_token;                     // dx = [j = t] of_token - p (all + slope ln p)
    // (a row of nothing hands an infinity back through an lse of -inf: p is 0 there, and 0 times it must stay 0)
    if (a.d_lse != nullptr && !none) all -= a.d_lse[row];
    if constexpr (ENTROPY) {
        if (!none) {
            slope = a.d_entropy[row];
            all = __builtin_fmaf(slope, a.entropy[row], all);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long i = c0 + (u * T + lane) * P;
        if (i >= cols) break;
        float d[P];
#pragma unroll
        for (int e = 0; e < P; ++e) {
            const float ln_p = element<DT>(raw[u], e) - lse, p = none ? 0.f : __builtin_amdgcn_exp2f(ln_p * LOG2E);
            const float f = ENTROPY ? __builtin_fmaf(slope, fmaxf(ln_p, FAR_BELOW), all) : all;
            d[e] = __builtin_fmaf(-p, f, i + e == token ? of_token : 0.f);
        }
        store16<DT, POLICY>(a.dx, row * cols + i, cols - i, d);
    }
}

// ---- host side -------------------------------------------------------------------------------

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Workgroups of 512 lanes for a row (or chunk) of more than 16384 columns, of 256 for shorter ones (us, 512 / 256: 2048 x 8192 bf16 12.9 / 7.3, 256 x 131072 with five alternatives 18.2 / 22.5);
// rows in chunks where there are fewer of them than compute units, one workgroup a unit (two: 256 x 131072 with alternatives 23.7, one 18.2), of 2048 columns at least.
constexpr int LONG_THREADS = 512, SHORT_THREADS = 256;
constexpr int64_t LONG_COLS = 16384, LEAST_CHUNK = 2048;
constexpr int GRAD_PIECES = 4, FEW_PIECES = 256;    // the gradient: 16-byte pieces of a lane of a long row, of a short row

static int64_t token_chunks(int64_t rows, int64_t cols) {
    const int64_t wanted = ceil_div(device_cu_count(), rows), possible = ceil_div(cols, LEAST_CHUNK);
    const int64_t n = wanted < possible ? wanted : possible;
    return n < MOST_CHUNKS ? n : MOST_CHUNKS;
}
// Columns of a chunk, whole pieces, and lanes of the workgroup that takes one.
static int64_t chunk_columns(int dtype, int64_t cols, int64_t chunks) {
    const int64_t piece = dtype == SP_F32 ? 4 : 8;
    return ceil_div(ceil_div(cols, chunks), piece) * piece;
}
static int chunk_threads(int64_t chunk_cols) { return chunk_cols > LONG_COLS ? LONG_THREADS : SHORT_THREADS; }
// Whether lanes of one wave hold a row: up to 512 of its 16-byte pieces, 1024 where there are waves enough.  (us, so / a workgroup per row: bf16 16384 x 4000 28.6 / 53, 8192 x 8000 33 / 36.8,
// 2048 x 8192 12.5 / 9.1, 16 x 4091 4.2 / 3.5 and 2.5 for the join of two chunks, 256 x 8192 6.2 / 3.5; f32 16384 x 2000 23.6 / 32.9, 8192 x 4000 24.2 / 28.4.)
// With alternatives a workgroup takes a row of any length, whose steps from barrier to barrier then are the time: 16384 x 256 f32 52 us with five of them, 4.9 without.
constexpr int MANY_PIECES = 1024;
static bool short_rows(int dtype, int64_t rows, int64_t cols, int32_t top) {
    const int64_t pieces = ceil_div(cols, dtype == SP_F32 ? 4 : 8);
    return top == 0 && (pieces <= 512 || (pieces <= MANY_PIECES && rows >= 4096));
}

// Lanes to a row of so many 16-byte pieces, and pieces to a lane: few lanes, so that a wave's reductions are of many rows (us, forward and backward of 65536 x 256 f32 on 64 lanes of one
// piece 17.3 + 27.6, on 16 of four 11.6 + 21.2; 65536 x 1024 bf16 on 64 of two 32.8 + 50.4, on 16 of eight 30.1 + 46.4).
template <int MOST, typename F>
static int by_pieces(long pieces, const F& f) {
    typedef std::integral_constant<int, 4> c4;
    typedef std::integral_constant<int, 8> c8;
    typedef std::integral_constant<int, 16> c16;
    typedef std::integral_constant<int, 64> c64;
    if (pieces <= 4) return f(c4{}, std::integral_constant<int, 1>{});
    if (pieces <= 16) return f(c4{}, c4{});
    if (pieces <= 32) return f(c16{}, std::integral_constant<int, 2>{});
    if (pieces <= 64) return f(c16{}, c4{});
    if (pieces <= 128) return f(c16{}, c8{});
    if constexpr (MOST > 256) {
        if (pieces > 512) return f(c64{}, c16{});
        if (pieces > 256) return f(c64{}, c8{});
    }
    return f(c64{}, c4{});
}

template <int DT, bool ENTROPY>
static int launch_rows(const void* logits, long cols, long rows, const TokenArgs& a, hipStream_t stream) {
    return by_pieces<MANY_PIECES>(ceil_div(cols, PER16<DT>), [&](auto t, auto c) {
        constexpr int T = decltype(t)::value, C = decltype(c)::value;
        hipLaunchKernelGGL((token_probs_rows_kernel<DT, T, C, ENTROPY>), dim3((unsigned)ceil_div(rows, 256 / T)), dim3(256), 0, stream, logits, cols, rows, a);
        return check_launch("sp_token_log_probs");
    });
}

template <int DT, bool ENTROPY, bool TOP>
static int launch_long(const void* logits, long cols, long rows, const TokenArgs& a, hipStream_t stream) {
    const long chunks = token_chunks(rows, cols), chunk_cols = chunk_columns(DT, cols, chunks);
    const dim3 blocks((unsigned)(rows * chunks));
    if (chunk_threads(chunk_cols) == LONG_THREADS) hipLaunchKernelGGL((token_probs_kernel<DT, LONG_THREADS, ENTROPY, TOP>), blocks, dim3(LONG_THREADS), 0, stream, logits, cols, (unsigned)chunks, chunk_cols, a);
    else hipLaunchKernelGGL((token_probs_kernel<DT, SHORT_THREADS, ENTROPY, TOP>), blocks, dim3(SHORT_THREADS), 0, stream, logits, cols, (unsigned)chunks, chunk_cols, a);
    if (const int rc = check_launch("sp_token_log_probs"); rc != SP_OK || chunks == 1) return rc;
    if (TOP) hipLaunchKernelGGL(token_probs_join_top_kernel<DT>, dim3((unsigned)rows), dim3(256), 0, stream, logits, cols, (int)chunks, a);
    else hipLaunchKernelGGL(token_probs_join_kernel<DT>, dim3((unsigned)ceil_div(rows, 4)), dim3(256), 0, stream, logits, cols, rows, (int)chunks, a);
    return check_launch("sp_token_log_probs");
}

template <int DT, bool ENTROPY>
static int launch_grad(const void* logits, long cols, long rows, const TokenGradArgs& a, hipStream_t stream) {
    constexpr int P = PER16<DT>;
    auto launch = [&](auto t, auto u) {
        constexpr int T = decltype(t)::value, U = decltype(u)::value;
        const long chunks = ceil_div(cols, T * U * P), blocks = ceil_div(rows * chunks, 256 / T);
        // a gradient that does not stay in the caches (32 MiB of L2) is streamed past them
        if (rows * cols * ELEM_BYTES<DT> > 32l << 20)
            hipLaunchKernelGGL((token_grad_kernel<DT, T, U, ENTROPY, ST_STREAM>), dim3((unsigned)blocks), dim3(256), 0, stream, logits, cols, rows, (unsigned)chunks, a);
        else
            hipLaunchKernelGGL((token_grad_kernel<DT, T, U, ENTROPY, ST_PLAIN>), dim3((unsigned)blocks), dim3(256), 0, stream, logits, cols, rows, (unsigned)chunks, a);
        return check_launch("sp_token_log_probs_backward");
    };
    const long pieces = ceil_div(cols, P);
    if (pieces <= FEW_PIECES) return by_pieces<FEW_PIECES>(pieces, launch);
    return launch(std::integral_constant<int, 256>{}, std::integral_constant<int, GRAD_PIECES>{});
}

namespace {
struct TokenKernelNames {
    TokenKernelNames() {
        register_kernel("token_probs", (const void*)token_probs_kernel<SP_BF16, LONG_THREADS, true, false>, LONG_THREADS);
        register_kernel("token_probs_top", (const void*)token_probs_kernel<SP_BF16, LONG_THREADS, true, true>, LONG_THREADS);
        register_kernel("token_grad", (const void*)token_grad_kernel<SP_BF16, 256, 4, true, ST_STREAM>, 256);
    }
} token_kernel_names;
}  // namespace

}  // namespace sp

using namespace sp;

static int token_sizes(const char* fn, int dtype, int64_t rows, int64_t cols) {
    if (dtype != SP_F32 && dtype != SP_F16 && dtype != SP_BF16) return fail(SP_ERR_DTYPE, "%s: dtype must be f32, f16 or bf16, got %d", fn, dtype);
    if (rows <= 0 || cols <= 0) return fail(SP_ERR_SHAPE, "%s: rows and cols must be positive (got %lld, %lld)", fn, (long long)rows, (long long)cols);
    if (rows > INT32_MAX || cols > (int64_t)1 << 30) return fail(SP_ERR_SHAPE, "%s: too large", fn);     // (columns are counted in 32 bits)
    return SP_OK;
}

// A launch holds fewer than 2^32 work items, whole workgroups of 256.
constexpr int64_t MOST_TOKEN_ITEMS = ((int64_t)1 << 32) - 256;
static int64_t forward_items(int dtype, int64_t rows, int64_t cols, int32_t top) {
    if (short_rows(dtype, rows, cols, top)) return rows * by_pieces<MANY_PIECES>(ceil_div(cols, dtype == SP_F32 ? 4 : 8), [](auto t, auto) { return (int)decltype(t)::value; });
    const int64_t chunks = token_chunks(rows, cols);
    return rows * chunks * chunk_threads(chunk_columns(dtype, cols, chunks));
}
static int64_t backward_items(int dtype, int64_t rows, int64_t cols) {
    const int64_t pieces = ceil_div(cols, dtype == SP_F32 ? 4 : 8);
    return rows * (pieces <= FEW_PIECES ? by_pieces<FEW_PIECES>(pieces, [](auto t, auto) { return (int)decltype(t)::value; }) : 256 * ceil_div(pieces, GRAD_PIECES * 256));
}

extern "C" int64_t sp_token_log_probs_workspace_bytes(int64_t rows, int64_t cols, int32_t top) {
    if (rows <= 0 || cols <= 0 || top < 0 || top > MOST_TOP) return 0;
    const int64_t chunks = token_chunks(rows, cols);
    return chunks > 1 ? rows * chunks * 4 * (3 + 2 * top) : 0;
}

extern "C" int sp_token_log_probs(int dtype, const void* logits, const int32_t* tokens, float* logp, float* entropy, float* lse, int32_t top, float* top_logp, int32_t* top_ids,
                                  int64_t rows, int64_t cols, void* workspace, int64_t workspace_bytes, void* stream) {
    SP_REQUIRE_PTR(logits);
    SP_REQUIRE_PTR(tokens);
    SP_REQUIRE_PTR(logp);
    SP_OPTIONAL_PTR(entropy);
    SP_OPTIONAL_PTR(lse);
    SP_OPTIONAL_PTR(top_logp);
    SP_OPTIONAL_PTR(top_ids);
    if (const int rc = token_sizes(__func__, dtype, rows, cols); rc != SP_OK) return rc;
    if (top < 0 || top > MOST_TOP) return fail(SP_ERR_ARG, "sp_token_log_probs: top must be in [0, 32], got %d", top);
    if (top > 0 && (top_logp == nullptr || top_ids == nullptr)) return fail(SP_ERR_NULL, "sp_token_log_probs: top_logp and top_ids are needed for %d alternatives", top);
    const bool in_registers = short_rows(dtype, rows, cols, top);
    if (forward_items(dtype, rows, cols, top) > MOST_TOKEN_ITEMS) return fail(SP_ERR_SHAPE, "sp_token_log_probs: too large");
    const int64_t need = sp_token_log_probs_workspace_bytes(rows, cols, top);
    if (need > 0) {
        SP_REQUIRE_PTR(workspace);
        if (workspace_bytes < need) return fail(SP_ERR_ARG, "sp_token_log_probs: workspace of %lld bytes, %lld are needed", (long long)workspace_bytes, (long long)need);
    }
    const int64_t es = dtype == SP_F32 ? 4 : 2, of_top = top > 0 ? rows * top * 4 : 0;
    if (const int rc = lie_apart(__func__, {{"logp", logp, rows * 4}, {"entropy", entropy, rows * 4}, {"lse", lse, rows * 4}, {"top_logp", of_top > 0 ? top_logp : nullptr, of_top},
                                            {"top_ids", of_top > 0 ? top_ids : nullptr, of_top}, {"workspace", need > 0 ? workspace : nullptr, need}},
                                 {{"logits", logits, rows * cols * es}, {"tokens", tokens, rows * 4}});
        rc != SP_OK)
        return rc;
    if (const int rc = require_gfx950(__func__); rc != SP_OK) return rc;
    TokenArgs a{};
    a.tokens = tokens; a.logp = logp; a.entropy = entropy; a.lse = lse; a.top = top; a.top_logp = top_logp; a.top_ids = top_ids;
    if (need > 0) {
        const int64_t parts = rows * token_chunks(rows, cols);
        a.part = (float*)workspace; a.part_top = a.part + 3 * parts; a.part_ids = (int32_t*)(a.part_top + parts * top);
    }
    const hipStream_t st = (hipStream_t)stream;
    auto by_entropy = [&](auto dt, auto with) {
        constexpr int DT = decltype(dt)::value;
        constexpr bool ENTROPY = decltype(with)::value;
        if (in_registers) return launch_rows<DT, ENTROPY>(logits, cols, rows, a, st);
        return top > 0 ? launch_long<DT, ENTROPY, true>(logits, cols, rows, a, st) : launch_long<DT, ENTROPY, false>(logits, cols, rows, a, st);
    };
    auto by_type = [&](auto dt) { return entropy != nullptr ? by_entropy(dt, std::true_type{}) : by_entropy(dt, std::false_type{}); };
    if (dtype == SP_F32) return by_type(std::integral_constant<int, SP_F32>{});
    if (dtype == SP_F16) return by_type(std::integral_constant<int, SP_F16>{});
    return by_type(std::integral_constant<int, SP_BF16>{});
}

extern "C" int sp_token_log_probs_backward(int dtype, const void* logits, const int32_t* tokens, const float* lse, const float* entropy, const float* d_logp,
                                           const float* d_entropy, const float* d_lse, void* d_logits, int64_t rows, int64_t cols, void* stream) {
    SP_REQUIRE_PTR(logits);
    SP_REQUIRE_PTR(tokens);
    SP_REQUIRE_PTR(lse);
    SP_REQUIRE_PTR(d_logits);
    SP_OPTIONAL_PTR(entropy);
    SP_OPTIONAL_PTR(d_logp);
    SP_OPTIONAL_PTR(d_entropy);
    SP_OPTIONAL_PTR(d_lse);
    if (const int rc = token_sizes(__func__, dtype, rows, cols); rc != SP_OK) return rc;
    if (d_entropy != nullptr && entropy == nullptr) return fail(SP_ERR_NULL, "sp_token_log_probs_backward: d_entropy needs the entropy");
    if (backward_items(dtype, rows, cols) > MOST_TOKEN_ITEMS) return fail(SP_ERR_SHAPE, "sp_token_log_probs_backward: too large");
    // (every number of the logits is read by the lane that writes its gradient, so they may be the same memory, but not half of it)
    const int64_t all = rows * cols * (dtype == SP_F32 ? 4 : 2);
    if (const int rc = lie_apart(__func__, {{"d_logits", d_logits, all}},
                                 {{"logits", logits == d_logits ? nullptr : logits, all}, {"tokens", tokens, rows * 4}, {"lse", lse, rows * 4},
                                  {"entropy", d_entropy != nullptr ? entropy : nullptr, rows * 4}, {"d_logp", d_logp, rows * 4}, {"d_entropy", d_entropy, rows * 4}, {"d_lse", d_lse, rows * 4}});
        rc != SP_OK)
        return rc;
    if (const int rc = require_gfx950(__func__); rc != SP_OK) return rc;
    TokenGradArgs a{};
    a.tokens = tokens; a.lse = lse; a.entropy = entropy; a.d_logp = d_logp; a.d_entropy = d_entropy; a.d_lse = d_lse; a.dx = d_logits;
    const hipStream_t st = (hipStream_t)stream;
    auto by_type = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        return d_entropy != nullptr ? launch_grad<DT, true>(logits, cols, rows, a, st) : launch_grad<DT, false>(logits, cols, rows, a, st);
    };
    if (dtype == SP_F32) return by_type(std::integral_constant<int, SP_F32>{});
    if (dtype == SP_F16) return by_type(std::integral_constant<int, SP_F16>{});
    return by_type(std::integral_constant<int, SP_BF16>{});
}
