// Log-probabilities and entropy of actions under a wide categorical head, forward and backward -- gfx950.
//
// The front end that loss.hip's ppo_loss_logits_fwd_bwd has for 2 .. 8 actions (Categorical(logits).log_prob / .entropy,
// reference src/ppo.py:186-189, :212-214), for any number of actions, rows of tokens and 16-bit logits.  With
// z = logits / temperature of one row, top = max z, s = sum e^(z - top), u = sum e^(z - top) (z - top):
//     log p_a = z_a - top - ln s          H = -sum p ln p = ln s - u / s
//     d log p_a / d z_k = [k = a] - p_k   d H / d z_k = -p_k (ln p_k + H)
// One pass over the logits forward (running maximum; s and u are rescaled when it moves), one pass backward that reads
// the logits again and writes their gradient.  Both are bound by HBM: 8192 rows of 131072 f16 logits take 397 us forward (5.4
// TB/s) and 735 us backward (5.8 TB/s); a large copy runs at 4.7 TB/s, a sum over a large array at 4.0.  What is kept per row for the backward pass is the
// PAIR {max logit, ln s}: their sum, the usual log-sum-exp, loses ln s in rows of large magnitude (a row of the type's
// lowest value is a uniform one), and (logit - max) is exact where the two are near.
// All sums are f32 over chunks of at most 32 elements, then over the lanes' chunks, then over lanes: 131072 terms are
// off by a few 1e-7.
#include "token_common.h"

using namespace ppo_token;

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// Stands for -inf, and all that is lower, as the factor of a weight 2^t that is 0 (0 * -inf would be NaN).  2^t is 0 below
// -149 already, and neither a gradient of 1e35 nor a sum of 2^40 weights overflows when it is multiplied by this.
constexpr float LOWEST = -1000.0f;

struct Row {
    float m, s, u;   // max of the raw logits; sum 2^t; sum t 2^t with t = (x - m) * c, c = log2(e) / temperature
};

__device__ __forceinline__ Row row_none() { return Row{-INFINITY, 0.0f, 0.0f}; }

// (m, s, u) seen from the maximum m2 >= m
__device__ __forceinline__ void row_move(Row &r, float m2, float c)
{
    const float base = m2 == -INFINITY ? 0.0f : m2;
    const float t = (r.m - base) * c;                  // -inf for an empty part: s and u are 0 then
    const float f = __builtin_amdgcn_exp2f(t);
    r.u = (r.u + r.s * fmaxf(t, LOWEST)) * f;
    r.s *= f;
    r.m = m2;
}

__device__ __forceinline__ Row row_join(Row a, Row b, float c)
{
    const float m = fmaxf(a.m, b.m);
    row_move(a, m, c);
    row_move(b, m, c);
    return Row{m, a.s + b.s, a.u + b.u};
}

template <int N> __device__ __forceinline__ void row_add(Row &r, const float (&x)[N], float c)
{
    float m = r.m;
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, x[i]);
    if (m > r.m) row_move(r, m, c);
    const float base = r.m == -INFINITY ? 0.0f : r.m;
    float s = 0.0f, u = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float t = (x[i] - base) * c;
        const float e = __builtin_amdgcn_exp2f(t);     // NaN stays in s
        s += e;
        u = __builtin_fmaf(e, fmaxf(t, LOWEST), u);
    }
    r.s += s;
    r.u += u;
}

template <int G> __device__ __forceinline__ Row row_lanes(Row r, float c)
{
#pragma unroll
    for (int off = G / 2; off > 0; off >>= 1) {
        const Row o = {__shfl_xor(r.m, off, 64), __shfl_xor(r.s, off, 64), __shfl_xor(r.u, off, 64)};
        r = row_join(r, o, c);
    }
    return r;
}

struct FwdArgs {
    const void *logits, *actions;
    float *logp, *entropy, *stats;
    long rows, length, A, batch_stride, token_stride, ignore, first;   // first: row of this launch
    float c, inv_t;
    int action_bytes;
};

__device__ __forceinline__ long action_of(const void *actions, int bytes, long row)
{
    return bytes == 8 ? reinterpret_cast<const long *>(actions)[row] : (long)reinterpret_cast<const int *>(actions)[row];
}

__device__ __forceinline__ long row_offset(long row, long rows, long length, long batch_stride, long token_stride)
{
    if (length == rows) return row * token_stride;     // one batch, or evenly spaced ones (even_rows)
    const long b = row / length;
    return b * batch_stride + (row - b * length) * token_stride;
}

__device__ __forceinline__ void write_ignored(const FwdArgs &a, long row)
{
    a.logp[row] = 0.0f;
    if (a.entropy) a.entropy[row] = 0.0f;
    a.stats[2 * row] = 0.0f;
    a.stats[2 * row + 1] = 0.0f;
}

template <class T> __device__ __forceinline__ void write_row(const FwdArgs &a, long row, const typename T::raw *x, long act, Row r)
{
    float logp, H, lns;
    if (act < 0 || act >= a.A) {                       // no such action: the row's outputs and gradients are NaN
        logp = H = lns = __builtin_nanf("");
    } else if (r.m == -INFINITY && r.s == 0.0f) {      // no legal action in the row
        logp = -INFINITY;
        H = lns = 0.0f;
    } else {
        lns = logf(r.s);
        H = lns - LN2 * (r.u / r.s);
        logp = (T::load(x[act]) - r.m) * a.inv_t - lns;
    }
    a.logp[row] = logp;
    if (a.entropy) a.entropy[row] = H;
    a.stats[2 * row] = r.m;
    a.stats[2 * row + 1] = lns;
}

// G lanes a row, at most N elements a lane, all in registers: the lanes find the row's maximum first and then only
// add, where joining running sums would take two exponentials a step
template <class T, int G, int N> __global__ void __launch_bounds__(256) k_logprobs_short(FwdArgs a)
{
    const long row = a.first + (long)blockIdx.x * (256 / G) + threadIdx.x / G;
    const int l = threadIdx.x % G, A = (int)a.A;
    if (row >= a.rows) return;
    const typename T::raw *x = reinterpret_cast<const typename T::raw *>(a.logits) + row_offset(row, a.rows, a.length, a.batch_stride, a.token_stride);
    float v[N];                                        // (on their way while the action, which may be the ignored one, is)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = l + i * G < A ? T::load(x[l + i * G]) : -INFINITY;
    const long act = action_of(a.actions, a.action_bytes, row);
    if (act == a.ignore) {
        if (l == 0) write_ignored(a, row);
        return;
    }
    float m = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);
#pragma unroll
    for (int off = G / 2; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    const float base = m == -INFINITY ? 0.0f : m;
    Row r = {m, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float t = (v[i] - base) * a.c, e = __builtin_amdgcn_exp2f(t);
        r.s += e;
        r.u = __builtin_fmaf(e, fmaxf(t, LOWEST), r.u);
    }
#pragma unroll
    for (int off = G / 2; off > 0; off >>= 1) {
        r.s += __shfl_xor(r.s, off, 64);
        r.u += __shfl_xor(r.u, off, 64);
    }
    if (l == 0) write_row<T>(a, row, x, act, r);
}

// a workgroup of THREADS (a wave, 256 or 1024 threads) a row, 16-byte loads
template <class T, int THREADS> __global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS) k_logprobs_long(FwdArgs a)
{
    constexpr int E = 16 / T::BYTES, CHUNK = 32, U = CHUNK / E;
    const long row = a.first + (THREADS == 64 ? (long)blockIdx.x * 4 + threadIdx.x / 64 : (long)blockIdx.x);
    const int tid = THREADS == 64 ? threadIdx.x % 64 : threadIdx.x;
    if (row >= a.rows) return;
    const long act = action_of(a.actions, a.action_bytes, row);
    if (act == a.ignore) {
        if (tid == 0) write_ignored(a, row);
        return;
    }
    const typename T::raw *x = reinterpret_cast<const typename T::raw *>(a.logits) + row_offset(row, a.rows, a.length, a.batch_stride, a.token_stride);
    Row r = row_none();
    long at = 0;
    for (; at + (long)THREADS * CHUNK <= a.A; at += (long)THREADS * CHUNK) {
        float v[CHUNK];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            float w[E];
            load16<T>(x + at + ((long)i * THREADS + tid) * E, w);
#pragma unroll
            for (int j = 0; j < E; ++j) v[i * E + j] = w[j];
        }
        row_add<CHUNK>(r, v, a.c);
    }
    for (; at + tid * E < a.A; at += (long)THREADS * E) {
        const long k = at + tid * E;
        float w[E];
        if (k + E <= a.A) {
            load16<T>(x + k, w);
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) w[j] = k + j < a.A ? T::load(x[k + j]) : -INFINITY;
        }
        row_add<E>(r, w, a.c);
    }
    r = row_lanes<64>(r, a.c);
    if constexpr (THREADS > 64) {
        __shared__ Row part[THREADS / 64];
        if ((tid & 63) == 0) part[tid >> 6] = r;
        __syncthreads();
        if (tid < 64) {
            r = tid < THREADS / 64 ? part[tid] : row_none();
            r = row_lanes<THREADS / 64>(r, a.c);
        }
    }
    if (tid == 0) write_row<T>(a, row, x, act, r);
}

struct BwdArgs {
    const void *logits, *actions;
    const float *stats, *entropy, *g_logp, *g_entropy;
    void *g;
    long rows, length, A, batch_stride, token_stride, ignore, first;   // first: row of this launch
    float c, inv_t;
    int action_bytes;
};

// d loss / d logit_k = -p_k (ga + gb log2 p_k) + [k = a] gl
struct Grad {
    float base, lns2, ga, gb, gl;
    long act;
    bool live;
};

__device__ __forceinline__ Grad grad_of(const BwdArgs &a, long row)
{
    Grad g;
    g.act = action_of(a.actions, a.action_bytes, row);
    const float m = a.stats[2 * row], lns = a.stats[2 * row + 1];
    const float glp = a.g_logp ? a.g_logp[row] : 0.0f, gh = a.g_entropy ? a.g_entropy[row] : 0.0f;
    const float H = a.g_entropy ? a.entropy[row] : 0.0f;
    // an ignored token and a row without a legal action have no gradient
    g.live = g.act != a.ignore && !(m == -INFINITY && lns == 0.0f);
    g.base = m;
    g.lns2 = lns * LOG2E;
    g.gl = glp * a.inv_t;
    g.ga = g.gl + gh * H * a.inv_t;
    g.gb = gh * LN2 * a.inv_t;
    return g;
}

__device__ __forceinline__ float grad_at(const Grad &g, float x, float c)
{
    const float t = __builtin_fmaf(x - g.base, c, -g.lns2);   // log2 p
    const float p = __builtin_amdgcn_exp2f(t);
    return -p * __builtin_fmaf(g.gb, fmaxf(t, LOWEST), g.ga);
}

template <class T, int G> __global__ void __launch_bounds__(256) k_logprobs_bwd_short(BwdArgs a)
{
    const long row = a.first + (long)blockIdx.x * (256 / G) + threadIdx.x / G;
    const int l = threadIdx.x % G, A = (int)a.A;
    if (row >= a.rows) return;
    const typename T::raw *x = reinterpret_cast<const typename T::raw *>(a.logits) + row_offset(row, a.rows, a.length, a.batch_stride, a.token_stride);
    typename T::raw *o = reinterpret_cast<typename T::raw *>(a.g) + row * a.A;
    const Grad g = grad_of(a, row);
    for (int k = l; k < A; k += 4 * G) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = k + i * G < A ? T::load(x[k + i * G]) : 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = k + i * G;
            if (at < A) o[at] = T::store(g.live ? grad_at(g, v[i], a.c) + (at == g.act ? g.gl : 0.0f) : 0.0f);
        }
    }
}

// (row, chunk of 256 * 32 elements) a workgroup
template <class T> __global__ void __launch_bounds__(256) k_logprobs_bwd_long(BwdArgs a, int chunks)
{
    constexpr int E = 16 / T::BYTES, CHUNK = 32, U = CHUNK / E;
    const long row = a.first + blockIdx.x / chunks;
    const long at = (long)(blockIdx.x % chunks) * (256 * CHUNK);
    const Grad g = grad_of(a, row);
    const typename T::raw *x = reinterpret_cast<const typename T::raw *>(a.logits) + row_offset(row, a.rows, a.length, a.batch_stride, a.token_stride);
    typename T::raw *o = reinterpret_cast<typename T::raw *>(a.g) + row * a.A;
    const bool whole = at + 256 * CHUNK <= a.A;
    float w[U][E];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const long k = at + ((long)i * 256 + threadIdx.x) * E;
        if (g.live && (whole || k + E <= a.A)) {
            load16<T>(x + k, w[i]);
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) w[i][j] = g.live && k + j < a.A ? T::load(x[k + j]) : 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const long k = at + ((long)i * 256 + threadIdx.x) * E;
#pragma unroll
        for (int j = 0; j < E; ++j) w[i][j] = g.live ? grad_at(g, w[i][j], a.c) : 0.0f;
        if (g.live && g.act >= k && g.act < k + E) {
#pragma unroll
            for (int j = 0; j < E; ++j) w[i][j] += k + j == g.act ? g.gl : 0.0f;
        }
        if (whole || k + E <= a.A) {
            store16<T>(o + k, w[i]);
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (k + j < a.A) o[k + j] = T::store(w[i][j]);
        }
    }
}

bool logits_ok(const void *logits, int dtype, long batch, long length, long A, long batch_stride, long token_stride,
               const void *actions, int action_bytes, double temperature)
{
    if (!dtype_known(dtype) || batch < 1 || length < 1 || A < 1 || (action_bytes != 4 && action_bytes != 8)) return false;
    if (!logits || !actions || !ppo_aligned(logits, dtype_bytes(dtype)) || !ppo_aligned(actions, action_bytes)) return false;
    if (!(temperature > 0.0) || !(temperature <= 1e6) || !(temperature >= 1e-6)) return false;
    // the largest index of any element stays far from 2^63, the number of workgroups below 2^31
    const long MOST = 1L << 40;
    if (batch > MOST / length || A > MOST || batch * length > (1L << 31) - 1) return false;
    if (batch_stride < 0 || token_stride < 0) return false;
    return (__int128)(batch - 1) * batch_stride + (__int128)(length - 1) * token_stride + A < ((__int128)1 << 60);
}

// rows whose offsets are row * token_stride throughout need no division by length
template <class Args> void even_rows(Args &a, long batch)
{
    if (batch == 1 || a.batch_stride == a.length * a.token_stride) a.length = a.rows;
}

// A launch has fewer than 2^32 threads: so many rows (of `threads` each, rounded up to whole workgroups) at a time.
template <class Args, class Kernel, class... More>
int launch_rows(Kernel kernel, Args a, long threads, int block, hipStream_t s, More... more)
{
    const long fit = (1L << 31) / threads, most = fit >= 32 ? fit / 32 * 32 : fit;   // (whole workgroups)
    for (a.first = 0; a.first < a.rows; a.first += most) {
        const long rows = a.rows - a.first < most ? a.rows - a.first : most;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((rows * threads + block - 1) / block)), dim3(block), 0, s, a, more...);
        const int rc = ppo_launch_status();
        if (rc) return rc;
    }
    return 0;
}

}  // namespace

extern "C" {

int ppo_token_logprobs_fwd(const void *logits, int dtype, long batch, long length, long num_actions, long batch_stride,
                           long token_stride, const void *actions, int action_bytes, double temperature, long ignore_index,
                           float *logp, float *entropy, float *stats, void *stream)
{
    if (batch == 0 || length == 0) return 0;
    PPO_REQUIRE(logits_ok(logits, dtype, batch, length, num_actions, batch_stride, token_stride, actions, action_bytes, temperature));
    PPO_REQUIRE(logp && stats && ppo_aligned(logp, 4) && ppo_aligned(entropy, 4) && ppo_aligned(stats, 8));
    FwdArgs a;
    a.logits = logits; a.actions = actions; a.logp = logp; a.entropy = entropy; a.stats = stats;
    a.rows = batch * length; a.length = length; a.A = num_actions; a.batch_stride = batch_stride; a.token_stride = token_stride;
    a.ignore = ignore_index; a.action_bytes = action_bytes;
    a.inv_t = (float)(1.0 / temperature);
    a.c = (float)(1.4426950408889634 / temperature);
    even_rows(a, batch);
    hipStream_t s = (hipStream_t)stream;
    return by_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        // the fewest lanes that hold a row in 16 registers each (f32, us, 262144 rows: 64 actions 14 with 8 lanes, 19 with 16; 128
        // actions 22 with 8, 26 with 16; 65536 rows: 256 actions 13 with 16, 16 with 32, 500 actions 22 with 32, 28 with 64, 32
        // with a wave's loop, which is no slower than 32 lanes for 512 in 16 bits); above, a wave a row, above 4096 a workgroup of
        // 256, or of 1024 where rows are few (bf16, a wave / 256 / 1024 threads: 8192 x 4096 15 / 20 / 47, 1024 x 65536 32 / 25 / 27,
        // 64 x 65536 24 / 11 / 11)
        if (a.A <= 32) return launch_rows(k_logprobs_short<T, 8, 4>, a, 8, 256, s);
        if (a.A <= 64) return launch_rows(k_logprobs_short<T, 8, 8>, a, 8, 256, s);
        if (a.A <= 128) return launch_rows(k_logprobs_short<T, 8, 16>, a, 8, 256, s);
        if (a.A <= 256) return launch_rows(k_logprobs_short<T, 16, 16>, a, 16, 256, s);
        if (a.A <= 512) return launch_rows(k_logprobs_short<T, 32, 16>, a, 32, 256, s);
        if (a.A <= 4096) return launch_rows(k_logprobs_long<T, 64>, a, 64, 256, s);
        if (a.rows >= 1024) return launch_rows(k_logprobs_long<T, 256>, a, 256, 256, s);
        return launch_rows(k_logprobs_long<T, 1024>, a, 1024, 1024, s);
    });
}

int ppo_token_logprobs_bwd(const void *logits, int dtype, long batch, long length, long num_actions, long batch_stride,
                           long token_stride, const void *actions, int action_bytes, const float *stats, const float *entropy,
                           const float *g_logp, const float *g_entropy, double temperature, long ignore_index, void *g_logits,
                           void *stream)
{
    if (batch == 0 || length == 0) return 0;
    PPO_REQUIRE(logits_ok(logits, dtype, batch, length, num_actions, batch_stride, token_stride, actions, action_bytes, temperature));
    PPO_REQUIRE(stats && g_logits && (g_logp || g_entropy) && (!g_entropy || entropy));
    PPO_REQUIRE(ppo_aligned(stats, 8) && ppo_aligned(g_logits, dtype_bytes(dtype)) && ppo_aligned(entropy, 4) && ppo_aligned(g_logp, 4) &&
                ppo_aligned(g_entropy, 4));
    BwdArgs a;
    a.logits = logits; a.actions = actions; a.stats = stats; a.entropy = entropy; a.g_logp = g_logp; a.g_entropy = g_entropy;
    a.g = g_logits; a.rows = batch * length; a.length = length; a.A = num_actions; a.batch_stride = batch_stride;
    a.token_stride = token_stride; a.ignore = ignore_index; a.action_bytes = action_bytes;
    a.inv_t = (float)(1.0 / temperature);
    a.c = (float)(1.4426950408889634 / temperature);
    even_rows(a, batch);
    const long chunks = (a.A + 256 * 32 - 1) / (256 * 32);
    const bool chunked = a.A * dtype_bytes(dtype) > 8192;
    PPO_REQUIRE(!chunked || chunks < (1L << 23));      // a row's gradient is one launch at least
    hipStream_t s = (hipStream_t)stream;
    return by_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        // lanes a row, us with 8 / 16 / 64: f32 262144 x 64 23 / 24 / 46, x 128 57 / 51 / 63, 65536 x 300 36 / 29 / 29, x 500 87 / 60 /
        // 45; bf16 262144 x 64 21 / 21 / 45, x 128 35 / 31 / 51.  Rows of 8 KB, a wave against workgroups: f32 16384 x 2048 45 / 63 and
        // 8192 x 4096 52 / 43, bf16 8192 x 4096 27 / 30
        if (a.A <= 64) return launch_rows(k_logprobs_bwd_short<T, 8>, a, 8, 256, s);
        if (a.A <= 320) return launch_rows(k_logprobs_bwd_short<T, 16>, a, 16, 256, s);
        if (!chunked) return launch_rows(k_logprobs_bwd_short<T, 64>, a, 64, 256, s);
        return launch_rows(k_logprobs_bwd_long<T>, a, chunks * 256, 256, s, (int)chunks);
    });
}

}  // extern "C"
