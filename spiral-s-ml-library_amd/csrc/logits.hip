// Logits of a whole vocabulary before a token is chosen: penalties for tokens that stand in the history, biases, temperature and a mask,
// and the largest of what is left.  One pass: every logit is read once and written once, and that bounds it.
//
// A workgroup takes CHUNK columns of one row, and asks for them, and for their mask, before anything else.  What the history and the biases say about
// them is gathered meanwhile in a 32-bit word of LDS per column -- bits 0..19 the count behind the prompt, bit 20 "seen in the prompt", bits 21..31
// the first bias entry that names the column -- with integer atomics, whose order does not matter.  Columns whose word is zero, most of them, then
// cost one LDS read.
// Columns named by several bias entries (rare; a flag says whether there is one at all) have theirs added up in their order, in an LDS sum at the place of the first of them: the
// waves go through the entries once more, each for columns of its own.  1 x 32003, 2047 entries, none twice 11 us, one twice 17, half of them one id (a padded list)
// 51; with every named column going through the entries by itself, once one stood there twice, 10, 1230, 1220.
// The arithmetic is that of the steps written out, each rounded to f32: nothing is contracted.
#include "vec_io.h"

#pragma clang fp contract(off)

namespace sp {

constexpr unsigned COUNT_MASK = (1u << 20) - 1u, SEEN_BIT = 1u << 20;
constexpr int ENTRY_SHIFT = 21, MOST_ENTRIES = 2047;      // entry j is kept as 2047 - j: the first one is the largest, 0 is none
// Columns to a workgroup: enough of them that reading the history again for every chunk of a row does not count; fewer where the large chunks
// would leave most of the chip idle (1 x 32003, a history of 2000, with the token: 4 chunks 13.3 us, 16 chunks 8.5).  (One workgroup for a whole
// row, which needs no second launch to choose the token, is slower than both launches: a compute unit alone brings in 24 bytes a cycle, 16 us for
// 32003 columns.)
constexpr int LARGE_CHUNK = 8192, LARGE_THREADS = 512, SMALL_CHUNK = 2048, SMALL_THREADS = 256;
constexpr int AHEAD = 2;                                  // 16-byte pieces of the history per lane that are asked for at once

struct LogitsArgs {
    float* out;
    int32_t* token;
    const int32_t *tokens, *lengths, *prompt_lengths;
    const float *repetition, *presence, *frequency, *temperature;
    const int32_t* bias_ids;
    const float* bias;
    const unsigned* mask;
    long history, mask_step;      // mask_step: words from a row's mask to the next one's, 0 if all rows have the same
    int n_bias;
    float* best;                  // of every (row, chunk): the largest value, and behind them its column
    int* best_at;
};

struct Best {
    float v;
    int at;
    // the larger value, of equal ones the lower column; a NaN never wins, and -inf never does over "none"
    __device__ __forceinline__ void take(float w, int j) {
        if (w > v || (w == v && (unsigned)j < (unsigned)at)) { v = w; at = j; }
    }
};

__device__ __forceinline__ Best best_of_wave(Best b) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) b.take(__shfl_xor(b.v, d, WAVE), __shfl_xor(b.at, d, WAVE));
    return b;
}

// Four logits: a lane's share of a step, so that the f32 results of a wave are one KiB side by side (eight of 16 bits a lane leave in halves of
// 128-byte lines: 256 x 131072 bf16 and nothing else 44.7 us against 40.6, streamed 70.5 against 33.4).
template <int DT>
using Four = std::conditional_t<DT == SP_F32, u32x4, u32x2>;
template <int DT>
__device__ __forceinline__ Four<DT> load4(const void* p, long at, long left) {
    if constexpr (DT == SP_F32) {
        return load16<DT>(p, at, left);
    } else {
        const unsigned short* q = (const unsigned short*)p + at;
        if (left >= 4) return load_aligned<2, u32x2>(q);
        u32x2 v = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < left) v[i >> 1] |= (unsigned)q[i] << (16 * (i & 1));
        return v;
    }
}
template <int DT>
__device__ __forceinline__ float logit(const Four<DT>& v, int i) {
    if constexpr (DT == SP_F32) return __uint_as_float(v[i]);
    else return half_bits_to_f32<DT>(i & 1 ? v[i >> 1] >> 16 : v[i >> 1] & 0xffffu);
}

// SPARSE: there is a history or there are biases.  POLICY: of the stores.
template <int DT, bool SPARSE, int CHUNK, int THREADS, int POLICY>
__global__ __launch_bounds__(THREADS) void logits_kernel(const void* logits, long cols, unsigned chunks, const LogitsArgs a) {
    constexpr int N = 4, STEP = THREADS * N, PIECES = CHUNK / STEP;
    static_assert(CHUNK % STEP == 0 && CHUNK % 32 == 0, "whole pieces, whole words of the mask");
    extern __shared__ __attribute__((aligned(16))) unsigned words[];       // SPARSE: CHUNK of them, and behind them a sum per bias entry
    __shared__ int again;                                  // a column has more than one bias entry
    __shared__ float wave_v[THREADS / 64];
    __shared__ int wave_at[THREADS / 64];
    const int tid = threadIdx.x;
    const long row = blockIdx.x / chunks;
    const unsigned chunk = blockIdx.x - (unsigned)row * chunks;
    const long c0 = (long)chunk * CHUNK;
    const int here = (int)(cols - c0 < CHUNK ? cols - c0 : CHUNK);     // columns of this workgroup
    Four<DT> raw[PIECES];
    unsigned allowed[PIECES];
    const unsigned* mask = a.mask + row * a.mask_step;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int i = p * STEP + tid * N;
        raw[p] = load4<DT>(logits, row * cols + c0 + i, here - i);
        allowed[p] = a.mask != nullptr && i < here ? mask[(c0 + i) >> 5] : ~0u;
    }
    float rep = 1.f, pres = 0.f, freq = 0.f, temp = 0.f;
    const bool has_rep = a.repetition != nullptr, has_pres = a.presence != nullptr, has_freq = a.frequency != nullptr;
    if (has_rep) rep = a.repetition[row];
    if (has_pres) pres = a.presence[row];
    if (has_freq) freq = a.frequency[row];
    if (a.temperature != nullptr) temp = a.temperature[row];
    const int32_t* ids = a.bias_ids + row * a.n_bias;
    const float* biases = a.bias + row * a.n_bias;
    if constexpr (SPARSE) {
        // the history's first tokens and the first biases' columns are asked for before anything waits
        const int32_t* mine = a.tokens + row * a.history;
        long length = a.tokens != nullptr ? a.history : 0;
        auto tokens_at = [&](int v) { return ((long)v * THREADS + tid) * 4; };
        u32x4 ahead[AHEAD];
#pragma unroll
        for (int v = 0; v < AHEAD; ++v) ahead[v] = load16<SP_F32>(mine, tokens_at(v), length - tokens_at(v));
        const int id = tid < a.n_bias ? ids[tid] : -1;
        if (a.lengths != nullptr) {
            const long given = a.lengths[row];
            length = given < length ? given : length;
        }
        long prompt = a.prompt_lengths != nullptr ? a.prompt_lengths[row] : 0;
        prompt = prompt > 0 ? prompt : 0;
        // (columns are below 2^31: a token in front of the chunk, or below zero, wraps to a column behind it)
        const unsigned first = (unsigned)c0;
        for (int i = tid * 4; i < CHUNK; i += THREADS * 4) *reinterpret_cast<u32x4*>(words + i) = u32x4{0u, 0u, 0u, 0u};
        if (tid == 0) again = 0;
        __syncthreads();
        auto each_bias = [&](auto f) {
            for (int j = tid; j < a.n_bias; j += THREADS) {
                const unsigned at = (unsigned)(j == tid ? id : ids[j]) - first;
                if (at < (unsigned)here) f(at, (unsigned)(MOST_ENTRIES - j));
            }
        };
        if (a.n_bias > 0) {
            each_bias([&](unsigned at, unsigned entry) { atomicMax(&words[at], entry << ENTRY_SHIFT); });
            __syncthreads();
            // (counting goes on meanwhile: it leaves the upper bits alone)
            each_bias([&](unsigned at, unsigned entry) { if (words[at] >> ENTRY_SHIFT != entry) again = 1; });
        }
        auto take = [&](const u32x4& t, long i) {
            const int left = length - i < 4 ? (int)(length - i) : 4, of_prompt = prompt - i < 4 ? (int)(prompt - i) : 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned at = t[e] - first;
                if (at >= (unsigned)here || e >= left) continue;
                if (e < of_prompt) atomicOr(&words[at], SEEN_BIT);
                else atomicAdd(&words[at], 1u);
            }
        };
#pragma unroll
        for (int v = 0; v < AHEAD; ++v)
            if (tokens_at(v) < length) take(ahead[v], tokens_at(v));
        for (long i = tokens_at(AHEAD); i < length; i += THREADS * 4) take(load16<SP_F32>(mine, i, length - i), i);
        __syncthreads();
        if (a.n_bias > 0 && again != 0) {
            float* sums = reinterpret_cast<float*>(words + CHUNK);
            for (int j = tid; j < a.n_bias; j += THREADS) sums[j] = biases[j];
            __syncthreads();
            const int wave = tid >> 6;
            for (int j0 = 0; j0 < a.n_bias; j0 += 64) {
                const int j = j0 + (tid & 63);
                const unsigned at = j < a.n_bias ? (unsigned)ids[j] - first : ~0u;
                const int to = at < (unsigned)here ? MOST_ENTRIES - (int)(words[at] >> ENTRY_SHIFT) : j;      // the column's first entry
                const bool adds = to != j && to % (THREADS / 64) == wave;
                const float b = adds ? biases[j] : 0.f;
                for (unsigned long todo = __ballot(adds); todo != 0;) {
                    const int column = __builtin_amdgcn_readlane(to, __builtin_ctzl(todo));
                    unsigned long same = __ballot(to == column) & todo;
                    todo &= ~same;
                    float s = sums[column];
                    for (; same != 0; same &= same - 1) s = s + __int_as_float(__builtin_amdgcn_readlane(__float_as_int(b), __builtin_ctzl(same)));
                    sums[column] = s;                      // (of all lanes the same)
                }
            }
            __syncthreads();
        }
    }
    Best best{-INFINITY, -1};
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int i = p * STEP + tid * N;
        if (i >= here) break;
        float v[N];
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = logit<DT>(raw[p], e);
        if constexpr (SPARSE) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(words + i);
            if ((w[0] | w[1] | w[2] | w[3]) != 0) {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    if (w[e] == 0) continue;
                    const unsigned count = w[e] & COUNT_MASK;
                    float x = v[e];
                    if (has_rep && (w[e] & (SEEN_BIT | COUNT_MASK)) != 0) x = x > 0.f ? x / rep : x * rep;
                    if (count != 0) {
                        if (has_freq) x = x - freq * (float)count;
                        if (has_pres) x = x - pres;
                    }
                    if (const unsigned entry = w[e] >> ENTRY_SHIFT; entry != 0) {
                        const int first = MOST_ENTRIES - (int)entry;
                        x = x + (again != 0 ? reinterpret_cast<const float*>(words + CHUNK)[first] : biases[first]);
                    }
                    v[e] = x;
                }
            }
        }
        if (temp > 0.f)
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = v[e] / temp;
        if (a.mask != nullptr)
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = (allowed[p] >> ((i & 31) + e)) & 1u ? v[e] : -INFINITY;
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (i + e < here && v[e] > best.v) best = Best{v[e], (int)c0 + i + e};     // (columns go up: the first one stays)
        store16<SP_F32, POLICY>(a.out, row * cols + c0 + i, here - i, v);
    }
    if (a.token == nullptr) return;
    best = best_of_wave(best);
    if ((tid & 63) == 0) {
        wave_v[tid >> 6] = best.v;
        wave_at[tid >> 6] = best.at;
    }
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int w = 1; w < THREADS / 64; ++w) best.take(wave_v[w], wave_at[w]);
        if (chunks == 1) {
            a.token[row] = best.at;
        } else {
            a.best[blockIdx.x] = best.v;
            a.best_at[blockIdx.x] = best.at;
        }
    }
}

// The best of a row's chunks, a wave per row.
__global__ __launch_bounds__(256) void logits_token_kernel(const float* best, const int* best_at, unsigned chunks, long rows, int32_t* token) {
    const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    Best b{-INFINITY, -1};
    for (unsigned c = threadIdx.x & 63; c < chunks; c += 64) b.take(best[row * chunks + c], best_at[row * chunks + c]);
    b = best_of_wave(b);
    if ((threadIdx.x & 63) == 0) token[row] = b.at;
}

// ---- host side -------------------------------------------------------------------------------

static int64_t chunks_of(int64_t cols, int64_t chunk) { return (cols + chunk - 1) / chunk; }
static bool small_chunks(int64_t rows, int64_t cols) { return rows * chunks_of(cols, LARGE_CHUNK) <= device_cu_count() / 2; }
static int64_t logits_chunks(int64_t rows, int64_t cols) { return chunks_of(cols, small_chunks(rows, cols) ? SMALL_CHUNK : LARGE_CHUNK); }

template <int DT, bool SPARSE, int CHUNK, int THREADS, int POLICY>
static int launch_chunks(const void* logits, long rows, long cols, unsigned chunks, const LogitsArgs& a, hipStream_t stream) {
    auto kernel = logits_kernel<DT, SPARSE, CHUNK, THREADS, POLICY>;
    if (const int rc = ensure_dynamic_lds((const void*)kernel, SPARSE ? (CHUNK + MOST_ENTRIES + 1) * 4 : 0); rc != SP_OK) return rc;
    const int lds_bytes = SPARSE ? (CHUNK + (a.n_bias + 3) / 4 * 4) * 4 : 0;
    hipLaunchKernelGGL(kernel, dim3((unsigned)rows * chunks), dim3(THREADS), lds_bytes, stream, logits, cols, chunks, a);
    return check_launch("sp_logits_penalize");
}

// Results that do not stay in the caches (32 MiB of L2) are streamed past them: 256 x 131072 bf16 with a history of 4096 59 -> 53 us, without one and all
// else 41 -> 33.
template <int DT, bool SPARSE>
static int launch_logits(const void* logits, long rows, long cols, unsigned chunks, const LogitsArgs& a, hipStream_t stream) {
    if (small_chunks(rows, cols)) return launch_chunks<DT, SPARSE, SMALL_CHUNK, SMALL_THREADS, ST_PLAIN>(logits, rows, cols, chunks, a, stream);
    if (rows * cols * 4 > 32l << 20) return launch_chunks<DT, SPARSE, LARGE_CHUNK, LARGE_THREADS, ST_STREAM>(logits, rows, cols, chunks, a, stream);
    return launch_chunks<DT, SPARSE, LARGE_CHUNK, LARGE_THREADS, ST_PLAIN>(logits, rows, cols, chunks, a, stream);
}

namespace {
struct LogitsKernelNames {
    LogitsKernelNames() {
        register_kernel("logits", (const void*)logits_kernel<SP_F32, true, LARGE_CHUNK, LARGE_THREADS, ST_STREAM>, LARGE_THREADS);
        register_kernel("logits_bf16", (const void*)logits_kernel<SP_BF16, true, LARGE_CHUNK, LARGE_THREADS, ST_STREAM>, LARGE_THREADS);
    }
} logits_kernel_names;
}  // namespace

}  // namespace sp

using namespace sp;

extern "C" int64_t sp_logits_penalize_workspace_bytes(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0) return 0;
    return rows * logits_chunks(rows, cols) * 8;
}

extern "C" int sp_logits_penalize(int dtype, const void* logits, float* out, int32_t* token, const int32_t* tokens, const int32_t* lengths,
                                  const int32_t* prompt_lengths, int64_t history, const float* repetition, const float* presence,
                                  const float* frequency, const float* temperature, const int32_t* bias_ids, const float* bias, int64_t n_bias,
                                  const int32_t* mask, int64_t mask_rows, int64_t rows, int64_t cols, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
    SP_REQUIRE_PTR(logits);
    SP_REQUIRE_PTR(out);
    SP_OPTIONAL_PTR(token);
    SP_OPTIONAL_PTR(tokens);
    SP_OPTIONAL_PTR(lengths);
    SP_OPTIONAL_PTR(prompt_lengths);
    SP_OPTIONAL_PTR(repetition);
    SP_OPTIONAL_PTR(presence);
    SP_OPTIONAL_PTR(frequency);
    SP_OPTIONAL_PTR(temperature);
    SP_OPTIONAL_PTR(bias_ids);
    SP_OPTIONAL_PTR(bias);
    SP_OPTIONAL_PTR(mask);
    if (dtype != SP_F32 && dtype != SP_F16 && dtype != SP_BF16) return fail(SP_ERR_DTYPE, "sp_logits_penalize: dtype must be f32, f16 or bf16, got %d", dtype);
    if (rows <= 0 || cols <= 0) return fail(SP_ERR_SHAPE, "sp_logits_penalize: rows and cols must be positive (got %lld, %lld)", (long long)rows, (long long)cols);
    if (cols > INT32_MAX || rows > INT32_MAX || rows * chunks_of(cols, LARGE_CHUNK) * LARGE_THREADS >= (int64_t)1 << 32) return fail(SP_ERR_SHAPE, "sp_logits_penalize: too large");
    if (dtype != SP_F32 && (const void*)out == logits) return fail(SP_ERR_ARG, "sp_logits_penalize: only f32 logits can be overwritten");
    if (history < 0 || history > (int64_t)COUNT_MASK) return fail(SP_ERR_SHAPE, "sp_logits_penalize: history must be in [0, 2^20), got %lld", (long long)history);
    if (n_bias < 0 || n_bias > MOST_ENTRIES) return fail(SP_ERR_SHAPE, "sp_logits_penalize: n_bias must be in [0, 2047], got %lld", (long long)n_bias);
    if (history > 0 && tokens == nullptr) return fail(SP_ERR_NULL, "sp_logits_penalize: tokens is NULL");
    if (n_bias > 0 && (bias_ids == nullptr || bias == nullptr)) return fail(SP_ERR_NULL, "sp_logits_penalize: bias_ids and bias go together");
    if (mask != nullptr && mask_rows != 1 && mask_rows != rows) return fail(SP_ERR_SHAPE, "sp_logits_penalize: mask_rows must be 1 or rows, got %lld", (long long)mask_rows);
    if (token != nullptr) {
        SP_REQUIRE_PTR(workspace);
        if (workspace_bytes < sp_logits_penalize_workspace_bytes(rows, cols))
            return fail(SP_ERR_ARG, "sp_logits_penalize: workspace of %lld bytes, %lld are needed", (long long)workspace_bytes,
                        (long long)sp_logits_penalize_workspace_bytes(rows, cols));
    }
    const int rc = require_gfx950(__func__);
    if (rc != SP_OK) return rc;
    LogitsArgs a{};
    a.out = out; a.token = token; a.tokens = history > 0 ? tokens : nullptr; a.lengths = lengths; a.prompt_lengths = prompt_lengths; a.history = history;
    a.repetition = repetition; a.presence = presence; a.frequency = frequency; a.temperature = temperature;
    a.bias_ids = bias_ids; a.bias = bias; a.n_bias = (int)n_bias; a.mask = (const unsigned*)mask;
    a.mask_step = mask_rows == rows ? (cols + 31) / 32 : 0;
    const int64_t chunks = logits_chunks(rows, cols);
    a.best = (float*)workspace; a.best_at = token != nullptr ? (int*)((float*)workspace + rows * chunks) : nullptr;
    auto launch = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        const hipStream_t st = (hipStream_t)stream;
        return a.tokens != nullptr || a.n_bias > 0 ? launch_logits<DT, true>(logits, rows, cols, (unsigned)chunks, a, st) : launch_logits<DT, false>(logits, rows, cols, (unsigned)chunks, a, st);
    };
    const int launched = dtype == SP_F32 ? launch(std::integral_constant<int, SP_F32>{}) : dtype == SP_F16 ? launch(std::integral_constant<int, SP_F16>{})
                                                                                                          : launch(std::integral_constant<int, SP_BF16>{});
    if (launched != SP_OK || token == nullptr || chunks == 1) return launched;
    hipLaunchKernelGGL(logits_token_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, (hipStream_t)stream, a.best, a.best_at, (unsigned)chunks, (long)rows, token);
    return check_launch(__func__);
}
