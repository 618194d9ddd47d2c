// Losses over padded token sequences, forward and backward in one call -- gfx950.
//
// ppo_policy_kl_loss: the clipped surrogate of loss.hip (reference src/ppo.py:502-508, :522-525) over [B, L] tokens with a
// mask, asymmetric clip range and a KL term to a reference policy.  Per token, with d = new - old, r = e^d:
//     l = -min(r A, clip(r, 1 - lo, 1 + hi) A) + kl_coef k(e),   e = new - ref
//     k1 = e, k2 = e^2 / 2, k3 = e^-e - 1 + e;   dl/dnew = -(r A unless the clip binds) + kl_coef k'(e)
// and the mean of l over the unmasked tokens, or over the non-empty sequences of their tokens' means.
// ppo_preference_loss: a loss on the paired log ratio of two sequences, D = sum (chosen - ref) - sum (rejected - ref):
// -(1 - e) ln s(bD) - e ln s(-bD), max(0, 1 - bD) or (D - 1 / 2b)^2, the mean over the pairs.
//
// Both stream their inputs once and write one gradient a token: bound by HBM (21 and 13 bytes a token).  4096 x 8192 tokens
// take 167 us (4.2 TB/s, of them 11 for counting the mask), 2048 pairs of 4096 + 4000 tokens 53 us (4.0 TB/s).  Whether the clip
// binds is decided on d in f64 (the difference of two f32 is nearly always exact there) against ln(1 + hi), ln(1 - lo);
// sums are f64 per lane, over the wave, the workgroup and then the workgroups in index order, as in loss.hip: the same
// call gives the same bits.  A masked token is never used in arithmetic: what it holds may be NaN.
#include "token_common.h"

using namespace ppo_token;

namespace {

constexpr int SEQ_BLOCK = 256, SEQ_MAX_BLOCKS = 2048, COUNT_MAX_BLOCKS = 1024;
constexpr int NSUM = 4;                        // policy term, KL, clipped, drift r - 1 - ln r

template <int NV, int THREADS> __device__ __forceinline__ void block_sum(double (&acc)[NV], double (*part)[NV])
{
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
#pragma unroll
    for (int k = 0; k < NV; ++k) acc[k] = wave_sum(acc[k]);
    __syncthreads();                           // the last use of part is over
    if (lane == 0) {
#pragma unroll
        for (int k = 0; k < NV; ++k) part[wid][k] = acc[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        double s = 0.0;
        for (int w = 0; w < THREADS / 64; ++w) s += part[w][k];
        acc[k] = s;
    }
}

struct __attribute__((packed, aligned(1))) Bytes16 { uint32_t w[4]; };
struct __attribute__((packed, aligned(1))) Bytes4 { uint32_t w; };

// e^x - 1 - x for |x| <= 1/2, where it would cancel: the Taylor series (the terms left out are below 2^-27 of it)
__device__ __forceinline__ float expm1mx_near(float x)
{
    float q = 1.0f / 3628800;                  // 1 / 10!
    q = __builtin_fmaf(q, x, 1.0f / 362880);
    q = __builtin_fmaf(q, x, 1.0f / 40320);
    q = __builtin_fmaf(q, x, 1.0f / 5040);
    q = __builtin_fmaf(q, x, 1.0f / 720);
    q = __builtin_fmaf(q, x, 1.0f / 120);
    q = __builtin_fmaf(q, x, 1.0f / 24);
    q = __builtin_fmaf(q, x, 1.0f / 6);
    q = __builtin_fmaf(q, x, 0.5f);
    return q * x * x;
}

struct PolicyArgs {
    const float *lp, *old_lp, *adv, *ref_lp;
    const uint8_t *mask;
    float *g, *out6;
    double *partials;                          // [blocks][NSUM]
    double *counts;                            // [COUNT_MAX_BLOCKS][2]: unmasked tokens, non-empty rows of a counting workgroup
    int *row_counts;                           // [B], sequence means only
    long B, L, lp_stride, old_stride, adv_stride, ref_stride, mask_stride;
    double log_hi, log_lo, kl_coef;
    float hi, lo, kl_coef_f;
    int kl, per_sequence, sequence_mean, count_blocks;
};

// unmasked tokens of the rows that this workgroup visits, LANES lanes a row
template <int LANES> __device__ __forceinline__ void count_rows(const PolicyArgs &a, int *row_counts, long first, long step, double (&tot)[2])
{
    const int lane = threadIdx.x % LANES;
    tot[0] = tot[1] = 0.0;
    for (long b = first + threadIdx.x / LANES; b < a.B; b += step) {
        int n = 0;
        if (a.mask) {
            const uint8_t *m = a.mask + b * a.mask_stride;
            long t = lane * 16L;
#pragma unroll 4
            for (; t + 16 <= a.L; t += LANES * 16) {
                const Bytes16 v = *reinterpret_cast<const Bytes16 *>(m + t);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // one bit a non-zero byte
                    const uint32_t w = v.w[i];
                    n += __popc((((w & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w) & 0x80808080u);
                }
            }
            for (long k = t; k < a.L && k < t + 16; ++k) n += m[k] != 0;
#pragma unroll
            for (int off = LANES / 2; off > 0; off >>= 1) n += __shfl_xor(n, off, 64);
        } else {
            n = (int)a.L;
        }
        if (lane == 0) {
            if (a.sequence_mean) row_counts[b] = n;
            tot[0] += (double)n;
            tot[1] += n > 0 ? 1.0 : 0.0;
        }
    }
}

__global__ void __launch_bounds__(SEQ_BLOCK) k_policy_count(PolicyArgs a)
{
    __shared__ double part[SEQ_BLOCK / 64][2];
    double tot[2];
    // a wave a row, eight rows a wave where they are short (70000 x 128, the whole call: 40 us, 51 with a wave a row; as fast
    // as that for 4096 rows of any length)
    if (a.L > 256)
        count_rows<64>(a, a.row_counts, (long)blockIdx.x * (SEQ_BLOCK / 64), (long)gridDim.x * (SEQ_BLOCK / 64), tot);
    else
        count_rows<8>(a, a.row_counts, (long)blockIdx.x * (SEQ_BLOCK / 8), (long)gridDim.x * (SEQ_BLOCK / 8), tot);
    block_sum<2, SEQ_BLOCK>(tot, part);
    if (threadIdx.x == 0) {
        a.counts[2 * blockIdx.x] = tot[0];
        a.counts[2 * blockIdx.x + 1] = tot[1];
    }
}

template <class V> __device__ __forceinline__ void load4(const float *p, int n, V &v)
{
    if (n == 4) {
        const Vec16<F32> w = *reinterpret_cast<const Vec16<F32> *>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __builtin_bit_cast(float, w.w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = i < n ? p[i] : 0.0f;
    }
}

// groups of four neighbouring tokens of a row
__device__ __forceinline__ void policy_groups(const PolicyArgs &a, const int *row_counts, double tokens, double rows, long first, long step,
                                              double (&acc)[NSUM])
{
    const double whole = a.sequence_mean ? (rows > 0 ? 1.0 / rows : 1.0) : (tokens > 0 ? 1.0 / tokens : 1.0);
    const long per_row = (a.L + 3) / 4, groups = a.B * per_row;
    const bool small = groups < (1L << 31);
    for (long q = first; q < groups; q += step) {
        const long b = small ? (long)((uint32_t)q / (uint32_t)per_row) : q / per_row;
        const long t = (q - b * per_row) * 4;
        const int n = a.L - t < 4 ? (int)(a.L - t) : 4;
        float lp[4], old[4], adv[4], ref[4], g[4];
        uint32_t on = 0x01010101u;
        if (a.mask) {
            const uint8_t *m = a.mask + b * a.mask_stride + t;
            if (n == 4) {
                on = reinterpret_cast<const Bytes4 *>(m)->w;
            } else {
                on = 0;
                for (int i = 0; i < n; ++i) on |= (uint32_t)m[i] << (8 * i);
            }
        }
        load4(a.lp + b * a.lp_stride + t, n, lp);
        load4(a.old_lp + b * a.old_stride + t, n, old);
        if (a.per_sequence) {
            adv[0] = adv[1] = adv[2] = adv[3] = a.adv[b * a.adv_stride];
        } else {
            load4(a.adv + b * a.adv_stride + t, n, adv);
        }
        if (a.ref_lp) load4(a.ref_lp + b * a.ref_stride + t, n, ref);
        double w = 1.0;
        if (a.sequence_mean) {
            const int c = row_counts[b];
            w = 1.0 / (double)(c > 0 ? c : 1);
        }
        const float gw = (float)(w * whole);
        float s_pg = 0.0f, s_kl = 0.0f, s_drift = 0.0f;    // four terms in f32, then f64
        int out = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            g[i] = 0.0f;
            if (i < n && ((on >> (8 * i)) & 0xffu) != 0) {
                const double d = (double)lp[i] - (double)old[i];
                const bool above = d > a.log_hi, below = d < a.log_lo;
                const float df = (float)d, r = expf(df), A = adv[i], rA = r * A;
                const bool cut = A >= 0.0f ? above : below;
                s_pg -= cut ? A * (A >= 0.0f ? a.hi : a.lo) : rA;
                float dl = cut ? 0.0f : -rA;
                out += above || below ? 1 : 0;
                s_drift += fabsf(df) > 0.5f ? r - 1.0f - df : expm1mx_near(df);
                if (a.ref_lp) {
                    const float e = lp[i] - ref[i];
                    float k, dk;
                    if (a.kl == PPO_KL_K1) {
                        k = e; dk = 1.0f;
                    } else if (a.kl == PPO_KL_K2) {
                        k = 0.5f * e * e; dk = e;
                    } else {
                        // 1 - e^-e: as it stands far from 0 (e = inf where the reference's log-prob is -inf: 1), e - k near it
                        const bool far = fabsf(e) > 0.5f;
                        const float x = expf(-e);
                        k = far ? x - 1.0f + e : expm1mx_near(-e);
                        dk = far ? 1.0f - x : e - k;
                    }
                    s_kl += k;
                    if (a.kl_coef_f != 0.0f) dl = __builtin_fmaf(a.kl_coef_f, dk, dl);   // (only reported: an infinite one is no 0 * inf)
                }
                g[i] = gw * dl;
            }
        }
        acc[0] += w * (double)s_pg;
        acc[1] += w * (double)s_kl;
        acc[2] += w * (double)out;
        acc[3] += w * (double)s_drift;
        if (a.g) {
            float *o = a.g + b * a.L + t;
            if (n == 4) {
                store16<F32>(o, g);
            } else {
                for (int i = 0; i < n; ++i) o[i] = g[i];
            }
        }
    }
}

__device__ __forceinline__ void policy_out(const PolicyArgs &a, const double (&s)[NSUM], double tokens, double rows)
{
    const double whole = a.sequence_mean ? (rows > 0 ? 1.0 / rows : 1.0) : (tokens > 0 ? 1.0 / tokens : 1.0);
    const double pg = s[0] * whole, kl = s[1] * whole;
    a.out6[0] = (float)(a.ref_lp && a.kl_coef != 0.0 ? pg + a.kl_coef * kl : pg);
    a.out6[1] = (float)pg;
    a.out6[2] = (float)kl;
    a.out6[3] = (float)(s[2] * whole);
    a.out6[4] = (float)(s[3] * whole);
    a.out6[5] = (float)tokens;
}

template <int THREADS> __device__ __forceinline__ void totals(const PolicyArgs &a, double (*part)[2], double &tokens, double &rows)
{
    double tot[2] = {0.0, 0.0};
#pragma unroll 4
    for (int i = threadIdx.x; i < a.count_blocks; i += THREADS) {
        tot[0] += a.counts[2 * i];
        tot[1] += a.counts[2 * i + 1];
    }
    block_sum<2, THREADS>(tot, part);
    tokens = tot[0];
    rows = tot[1];
}

__global__ void __launch_bounds__(SEQ_BLOCK) k_policy_main(PolicyArgs a)
{
    __shared__ double part2[SEQ_BLOCK / 64][2];
    __shared__ double part[SEQ_BLOCK / 64][NSUM];
    double tokens, rows, acc[NSUM] = {0.0, 0.0, 0.0, 0.0};
    totals<SEQ_BLOCK>(a, part2, tokens, rows);
    policy_groups(a, a.row_counts, tokens, rows, (long)blockIdx.x * SEQ_BLOCK + threadIdx.x, (long)gridDim.x * SEQ_BLOCK, acc);
    block_sum<NSUM, SEQ_BLOCK>(acc, part);
    if (threadIdx.x == 0) {
#pragma unroll
        for (int k = 0; k < NSUM; ++k) a.partials[(long)blockIdx.x * NSUM + k] = acc[k];
    }
}

constexpr int FINAL_BLOCK = 256;
__global__ void __launch_bounds__(FINAL_BLOCK) k_policy_final(PolicyArgs a, int blocks)
{
    __shared__ double part2[FINAL_BLOCK / 64][2];
    __shared__ double part[FINAL_BLOCK / 64][NSUM];
    double tokens, rows, acc[NSUM] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 2
    for (int i = threadIdx.x; i < blocks; i += FINAL_BLOCK) {
#pragma unroll
        for (int k = 0; k < NSUM; ++k) acc[k] += a.partials[(long)i * NSUM + k];
    }
    totals<FINAL_BLOCK>(a, part2, tokens, rows);
    block_sum<NSUM, FINAL_BLOCK>(acc, part);
    if (threadIdx.x == 0) policy_out(a, acc, tokens, rows);
}

// everything in one workgroup: a few thousand tokens, where launches are what costs
constexpr int ONE_BLOCK = 512, ONE_ROWS = 256, ONE_GROUPS = 2048;
__global__ void __launch_bounds__(ONE_BLOCK) k_policy_one(PolicyArgs a)
{
    __shared__ double part2[ONE_BLOCK / 64][2];
    __shared__ double part[ONE_BLOCK / 64][NSUM];
    __shared__ int row_counts[ONE_ROWS];
    double tot[2], acc[NSUM] = {0.0, 0.0, 0.0, 0.0};
    if (a.L > 256)
        count_rows<64>(a, row_counts, 0, ONE_BLOCK / 64, tot);
    else
        count_rows<8>(a, row_counts, 0, ONE_BLOCK / 8, tot);
    block_sum<2, ONE_BLOCK>(tot, part2);           // (its barriers are the row counts' too)
    policy_groups(a, row_counts, tot[0], tot[1], threadIdx.x, ONE_BLOCK, acc);
    block_sum<NSUM, ONE_BLOCK>(acc, part);
    if (threadIdx.x == 0) policy_out(a, acc, tot[0], tot[1]);
}

// ---- preference loss ----------------------------------------------------------------------------------------------
struct PrefSide {
    const float *lp, *ref;
    const uint8_t *mask;
    float *g;
    long L, lp_stride, ref_stride, mask_stride;
};

struct PrefArgs {
    PrefSide side[2];                              // chosen, rejected
    double *partials;                              // [2 B][chunks][2]: sum, tokens of a chunk
    double *pair;                                  // [B][2]: loss, whether z > 0 of a pair (a workgroup a pair)
    float *out2, *rewards;
    long B;
    double beta, smoothing, inv_pairs;             // (1 / B from the host: the division in every wave cost 13 us)
    int kind, average, chunks;
};

// the mask's bytes of tokens t .. t + n - 1
__device__ __forceinline__ uint32_t mask4(const uint8_t *m, long t, int n)
{
    if (!m) return 0x01010101u;
    if (n == 4) return reinterpret_cast<const Bytes4 *>(m + t)->w;
    uint32_t on = 0;
    for (int i = 0; i < n; ++i) on |= (uint32_t)m[t + i] << (8 * i);
    return on;
}

// sum of (lp - ref) and number of tokens over [from, to) of row b, thread tid's share
template <int THREADS> __device__ __forceinline__ void pref_sum(const PrefSide &s, long b, long from, long to, int tid, double (&acc)[2])
{
    const float *lp = s.lp + b * s.lp_stride, *ref = s.ref ? s.ref + b * s.ref_stride : nullptr;
    const uint8_t *m = s.mask ? s.mask + b * s.mask_stride : nullptr;
    acc[0] = 0.0;
    long count = 0;
#pragma unroll 2
    for (long t = from + tid * 4L; t < to; t += THREADS * 4L) {
        const int n = to - t < 4 ? (int)(to - t) : 4;
        float x[4], y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        load4(lp + t, n, x);
        if (ref) load4(ref + t, n, y);
        const uint32_t on = mask4(m, t, n);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i < n && (on >> (8 * i) & 0xffu)) {
                acc[0] += (double)x[i] - (double)y[i];
                ++count;
            }
        }
    }
    acc[1] = (double)count;
}

// z = beta D and D of a pair, and beta times its two sums (means)
struct Margin {
    double z, delta, scale[2], reward[2];
};

__device__ __forceinline__ Margin margin_of(const PrefArgs &a, const double (&sum)[2], const double (&count)[2])
{
    Margin m;
    double mean[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        m.scale[k] = a.average ? 1.0 / (count[k] > 0.0 ? count[k] : 1.0) : 1.0;
        mean[k] = sum[k] * m.scale[k];
        m.reward[k] = a.beta * mean[k];
    }
    m.delta = mean[0] - mean[1];
    m.z = a.beta * m.delta;
    return m;
}

// e^-x for x >= 0 and ln(1 + y) for y in [0, 1]: short chains, since few lanes wait for them.  Taylor's series of e^r,
// |r| <= ln 2 / 2, to r^12 / 12!, where r = -x - k ln 2 in two steps (Cody and Waite's reduction, with fdlibm's ln2HI and ln2LO);
// ln(1 + y) = 2 artanh(y / (2 + y)), whose argument is at most 1/3, to its 19th power: 2e-16 and 1e-11 relative.
__device__ __forceinline__ double exp_minus(double x)
{
    if (x > 700.0) return 0.0;
    const double k = rint(x * -1.4426950408889634), r = __builtin_fma(k, -1.9082149292705877e-10, __builtin_fma(k, -0.6931471803691238, -x));
    double e = 1.0 / 479001600;
    e = __builtin_fma(e, r, 1.0 / 39916800);
    e = __builtin_fma(e, r, 1.0 / 3628800);
    e = __builtin_fma(e, r, 1.0 / 362880);
    e = __builtin_fma(e, r, 1.0 / 40320);
    e = __builtin_fma(e, r, 1.0 / 5040);
    e = __builtin_fma(e, r, 1.0 / 720);
    e = __builtin_fma(e, r, 1.0 / 120);
    e = __builtin_fma(e, r, 1.0 / 24);
    e = __builtin_fma(e, r, 1.0 / 6);
    e = __builtin_fma(e, r, 0.5);
    e = __builtin_fma(e, r, 1.0);
    e = __builtin_fma(e, r, 1.0);
    return ldexp(e, (int)k);
}

__device__ __forceinline__ double log1p_unit(double y)
{
    const double s = y / (2.0 + y), q = s * s;
    double sum = 1.0 / 19;
    sum = __builtin_fma(sum, q, 1.0 / 17);
    sum = __builtin_fma(sum, q, 1.0 / 15);
    sum = __builtin_fma(sum, q, 1.0 / 13);
    sum = __builtin_fma(sum, q, 1.0 / 11);
    sum = __builtin_fma(sum, q, 1.0 / 9);
    sum = __builtin_fma(sum, q, 1.0 / 7);
    sum = __builtin_fma(sum, q, 1.0 / 5);
    sum = __builtin_fma(sum, q, 1.0 / 3);
    sum = __builtin_fma(sum, q, 1.0);
    return 2.0 * s * sum;
}

// d mean loss / d a token's log-prob, chosen (k = 0) or rejected
__device__ __forceinline__ float pair_grad(const PrefArgs &a, const Margin &m, int k)
{
    double g;
    if (a.kind == PPO_PREF_SIGMOID) {
        const double ez = exp_minus(fabs(m.z)), far = 1.0 / (1.0 + ez), near = ez * far;   // s(|z|), s(-|z|)
        const double s_neg = m.z >= 0.0 ? near : far, s_pos = m.z >= 0.0 ? far : near;
        g = -a.beta * ((1.0 - a.smoothing) * s_neg - a.smoothing * s_pos);
        if (m.z != m.z) g = m.z;
    } else if (a.kind == PPO_PREF_HINGE) {
        g = m.z < 1.0 ? -a.beta : (m.z != m.z ? m.z : 0.0);
    } else {
        g = 2.0 * (m.delta - 0.5 / a.beta);
    }
    return (float)((k == 0 ? g * m.scale[0] : -g * m.scale[1]) * a.inv_pairs);
}

__device__ __forceinline__ double pair_loss(const PrefArgs &a, const Margin &m)
{
    if (a.kind == PPO_PREF_SIGMOID) {
        const double sp = log1p_unit(exp_minus(fabs(m.z)));           // softplus(-|z|)
        const double loss_pos = (m.z < 0.0 ? -m.z : 0.0) + sp, loss_neg = (m.z > 0.0 ? m.z : 0.0) + sp;   // -ln s(z), -ln s(-z)
        const double smooth = a.smoothing > 0.0 ? a.smoothing * loss_neg : 0.0;   // (z = inf: 0, not 0 * inf)
        return m.z != m.z ? m.z : (1.0 - a.smoothing) * loss_pos + smooth;
    }
    if (a.kind == PPO_PREF_HINGE) return m.z < 1.0 ? 1.0 - m.z : (m.z != m.z ? m.z : 0.0);
    const double off = m.delta - 0.5 / a.beta;
    return off * off;
}

// the first two groups of four mask bytes that a thread will want in pref_write: asked for before the margin is known
struct Ahead {
    uint32_t on[2];
};

template <int THREADS> __device__ __forceinline__ Ahead pref_ahead(const PrefSide &s, long b, long from, long to, int tid)
{
    Ahead a = {{0x01010101u, 0x01010101u}};
    if (s.mask && s.g) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const long t = from + (tid + i * THREADS) * 4L;
            if (t < to) a.on[i] = mask4(s.mask + b * s.mask_stride, t, to - t < 4 ? (int)(to - t) : 4);
        }
    }
    return a;
}

template <int THREADS> __device__ __forceinline__ void pref_write(const PrefSide &s, long b, long from, long to, int tid, const Ahead &ahead, float g)
{
    if (!s.g) return;
    const uint8_t *m = s.mask ? s.mask + b * s.mask_stride : nullptr;
    float *o = s.g + b * s.L;
    int turn = 0;
    for (long t = from + tid * 4L; t < to; t += THREADS * 4L, ++turn) {
        const int n = to - t < 4 ? (int)(to - t) : 4;
        const uint32_t on = turn == 0 ? ahead.on[0] : turn == 1 ? ahead.on[1] : mask4(m, t, n);
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = on >> (8 * i) & 0xffu ? g : 0.0f;
        if (n == 4) {
            store16<F32>(o + t, v);
        } else {
            for (int i = 0; i < n; ++i) o[t + i] = v[i];
        }
    }
}

__device__ __forceinline__ void pref_rewards(const PrefArgs &a, long b, const Margin &m)
{
    a.rewards[2 * b] = (float)m.reward[0];
    a.rewards[2 * b + 1] = (float)m.reward[1];
}

__device__ __forceinline__ void pref_out(const PrefArgs &a, double loss, double hits)
{
    a.out2[0] = (float)(loss * a.inv_pairs);
    a.out2[1] = (float)(hits * a.inv_pairs);
}

// a workgroup a pair, from pair `first` on
__global__ void __launch_bounds__(SEQ_BLOCK) k_pref_pair(PrefArgs a, long first)
{
    __shared__ double part[SEQ_BLOCK / 64][4];
    const long b = first + blockIdx.x;
    double v[4], acc[2];
    pref_sum<SEQ_BLOCK>(a.side[0], b, 0, a.side[0].L, threadIdx.x, acc);
    v[0] = acc[0]; v[1] = acc[1];
    pref_sum<SEQ_BLOCK>(a.side[1], b, 0, a.side[1].L, threadIdx.x, acc);
    v[2] = acc[0]; v[3] = acc[1];
    const Ahead ahead[2] = {pref_ahead<SEQ_BLOCK>(a.side[0], b, 0, a.side[0].L, threadIdx.x), pref_ahead<SEQ_BLOCK>(a.side[1], b, 0, a.side[1].L, threadIdx.x)};
    block_sum<4, SEQ_BLOCK>(v, part);
    const double sum[2] = {v[0], v[2]}, count[2] = {v[1], v[3]};
    const Margin m = margin_of(a, sum, count);
#pragma unroll
    for (int k = 0; k < 2; ++k) pref_write<SEQ_BLOCK>(a.side[k], b, 0, a.side[k].L, threadIdx.x, ahead[k], pair_grad(a, m, k));
    if (threadIdx.x == 0) {
        pref_rewards(a, b, m);
        a.pair[2 * b] = pair_loss(a, m);
        a.pair[2 * b + 1] = m.z > 0.0 ? 1.0 : 0.0;
    }
}

__global__ void __launch_bounds__(SEQ_BLOCK) k_pref_final(PrefArgs a)
{
    __shared__ double part[SEQ_BLOCK / 64][2];
    double acc[2] = {0.0, 0.0};
#pragma unroll 8
    for (long b = threadIdx.x; b < a.B; b += SEQ_BLOCK) {
        acc[0] += a.pair[2 * b];
        acc[1] += a.pair[2 * b + 1];
    }
    block_sum<2, SEQ_BLOCK>(acc, part);
    if (threadIdx.x == 0) pref_out(a, acc[0], acc[1]);
}

// long rows, few pairs: a workgroup a chunk of one row
__device__ __forceinline__ void chunk_of(const PrefArgs &a, long L, int c, long &from, long &to)
{
    const long size = ((L + a.chunks - 1) / a.chunks + 3) / 4 * 4;
    from = c * size < L ? c * size : L;
    to = from + size < L ? from + size : L;
}

__global__ void __launch_bounds__(SEQ_BLOCK) k_pref_sum(PrefArgs a)
{
    __shared__ double part[SEQ_BLOCK / 64][2];
    const long b = blockIdx.x / (2 * a.chunks);
    const int k = blockIdx.x / a.chunks % 2, c = blockIdx.x % a.chunks;
    long from, to;
    chunk_of(a, a.side[k].L, c, from, to);
    double acc[2];
    pref_sum<SEQ_BLOCK>(a.side[k], b, from, to, threadIdx.x, acc);
    block_sum<2, SEQ_BLOCK>(acc, part);
    if (threadIdx.x == 0) {
        a.partials[2L * blockIdx.x] = acc[0];
        a.partials[2L * blockIdx.x + 1] = acc[1];
    }
}

// the margin of pair b from its chunks' sums: LANES neighbouring lanes together, each gets it
template <int LANES> __device__ __forceinline__ Margin margin_of_chunks(const PrefArgs &a, long b, int lane)
{
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    for (int i = lane; i < a.chunks; i += LANES) {
        const double *p = a.partials + 2 * (b * 2 * a.chunks + i);
        v[0] += p[0];
        v[1] += p[1];
        v[2] += p[2 * a.chunks];
        v[3] += p[2 * a.chunks + 1];
    }
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] += __shfl_xor(v[k], off, 64);
    }
    const double sum[2] = {v[0], v[2]}, count[2] = {v[1], v[3]};
    return margin_of(a, sum, count);
}

// the last workgroup makes the mean over the pairs, the others write the gradients of their chunks
__global__ void __launch_bounds__(SEQ_BLOCK) k_pref_grad(PrefArgs a)
{
    const int lane = threadIdx.x & 63;
    if (blockIdx.x == 2 * a.B * a.chunks) {
        __shared__ double part[SEQ_BLOCK / 64][2];
        double acc[2] = {0.0, 0.0};
        const int lanes = a.chunks <= 8 ? 8 : 64;          // a pair (up to 256 pairs have two chunks: 32 of them at once)
        for (long b = threadIdx.x / lanes; b < a.B; b += SEQ_BLOCK / lanes) {
            const Margin m = lanes == 8 ? margin_of_chunks<8>(a, b, threadIdx.x % 8) : margin_of_chunks<64>(a, b, lane);
            if (threadIdx.x % lanes == 0) {
                acc[0] += pair_loss(a, m);
                acc[1] += m.z > 0.0 ? 1.0 : 0.0;
                pref_rewards(a, b, m);
            }
        }
        block_sum<2, SEQ_BLOCK>(acc, part);
        if (threadIdx.x == 0) pref_out(a, acc[0], acc[1]);
        return;
    }
    const long b = blockIdx.x / (2 * a.chunks);
    const int k = blockIdx.x / a.chunks % 2, c = blockIdx.x % a.chunks;
    long from, to;
    chunk_of(a, a.side[k].L, c, from, to);
    const Ahead ahead = pref_ahead<SEQ_BLOCK>(a.side[k], b, from, to, threadIdx.x);
    const float g = pair_grad(a, margin_of_chunks<64>(a, b, lane), k);   // (every wave for itself)
    pref_write<SEQ_BLOCK>(a.side[k], b, from, to, threadIdx.x, ahead, g);
}

// everything in one workgroup, a wave a pair: a few thousand tokens, where launches are what costs
__global__ void __launch_bounds__(ONE_BLOCK) k_pref_one(PrefArgs a)
{
    __shared__ double part[ONE_BLOCK / 64][2];
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    double tot[2] = {0.0, 0.0};
    for (long b = wid; b < a.B; b += ONE_BLOCK / 64) {
        double sum[2], count[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            double acc[2];
            pref_sum<64>(a.side[k], b, 0, a.side[k].L, lane, acc);
            sum[k] = wave_sum(acc[0]);
            count[k] = wave_sum(acc[1]);
        }
        const Margin m = margin_of(a, sum, count);
#pragma unroll
        for (int k = 0; k < 2; ++k)
            pref_write<64>(a.side[k], b, 0, a.side[k].L, lane, pref_ahead<64>(a.side[k], b, 0, a.side[k].L, lane), pair_grad(a, m, k));
        if (lane == 0) {
            pref_rewards(a, b, m);
            tot[0] += pair_loss(a, m);
            tot[1] += m.z > 0.0 ? 1.0 : 0.0;
        }
    }
    block_sum<2, ONE_BLOCK>(tot, part);
    if (threadIdx.x == 0) pref_out(a, tot[0], tot[1]);
}

// One launch instead of three: 8192 tokens, four turns of a thread.  Measured, us, against three: 8 x 1024 11.9 / 18.8, 128 x 64
// 11.9 / 19.4; 16384 tokens: 16 x 1024 19.5 / 19.5, 64 x 256 18.9 / 18.6, 256 x 64 19.9 / 19.0.
bool one_workgroup(long batch, long length)
{
    return batch <= ONE_ROWS && batch * ((length + 3) / 4) <= ONE_GROUPS;
}

// Workgroups a row is cut into: 0 = one for everything, where that is at most ten turns of a wave (measured, us, against a
// workgroup a pair: 4 pairs of 2 x 1000 15 / 20, 16 of 2 x 512 15 / 19; 16 turns: 32 of 2 x 512 23 / 19, 64 of 2 x 128 31 / 19).
// 1 = one a pair, up to 8192 tokens or where there are 256 pairs (against chunks: 64 of 2 x 8192 20 / 26, 16 of 2 x 8192 20 / 20;
// 1 of 2 x 16384 31 / 19).  Otherwise about 512 in all, of 2048 tokens at least.
int pref_chunks(long B, long Lc, long Lr)
{
    const long L = Lc > Lr ? Lc : Lr, turns = (Lc + 255) / 256 + (Lr + 255) / 256;
    if ((B + ONE_BLOCK / 64 - 1) / (ONE_BLOCK / 64) * (turns > 0 ? turns : 1) <= 10) return 0;   // (a pair without tokens has a loss, too)
    if (B >= 256 || L <= 8192) return 1;
    long c = (512 + 2 * B - 1) / (2 * B);
    const long most = (L + 2047) / 2048;
    if (c > most) c = most;
    return c < 2 ? 2 : (int)c;
}

bool rows_ok(const void *p, long B, long L, long stride)
{
    return p && ppo_aligned(p, 4) && stride >= 0 && (__int128)(B - 1) * stride + L < ((__int128)1 << 60);
}

}  // namespace

extern "C" {

size_t ppo_policy_kl_loss_workspace_bytes(long batch, long length)
{
    return batch < 0 || one_workgroup(batch, length) ? 0 : (size_t)SEQ_MAX_BLOCKS * NSUM * sizeof(double) + (size_t)COUNT_MAX_BLOCKS * 2 * sizeof(double) + (size_t)batch * sizeof(int);
}

int ppo_policy_kl_loss(const float *log_probs, long lp_stride, const float *old_log_probs, long old_stride, const float *advantages,
                       long adv_stride, int per_sequence, const float *ref_log_probs, long ref_stride, const uint8_t *mask,
                       long mask_stride, long batch, long length, double clip_low, double clip_high, double kl_coef, int kl_kind,
                       int sequence_mean, float *out6, float *g_log_probs, void *workspace, size_t workspace_bytes, void *stream)
{
    PPO_REQUIRE(batch >= 1 && length >= 1 && length <= (1L << 31) - 1 && batch <= (1L << 31) - 1 && batch * length < (1L << 40));
    PPO_REQUIRE(rows_ok(log_probs, batch, length, lp_stride) && rows_ok(old_log_probs, batch, length, old_stride));
    PPO_REQUIRE(rows_ok(advantages, batch, per_sequence ? 1 : length, adv_stride));
    PPO_REQUIRE(!ref_log_probs || rows_ok(ref_log_probs, batch, length, ref_stride));
    PPO_REQUIRE(!mask || (mask_stride >= 0 && (__int128)(batch - 1) * mask_stride + length < ((__int128)1 << 60)));
    PPO_REQUIRE(out6 && ppo_aligned(out6, 4) && ppo_aligned(g_log_probs, 4));
    PPO_REQUIRE(clip_low >= 0.0 && clip_low < 1.0 && clip_high >= 0.0 && clip_high <= 1e30 && kl_coef >= -1e30 && kl_coef <= 1e30);
    PPO_REQUIRE(kl_kind == PPO_KL_K1 || kl_kind == PPO_KL_K2 || kl_kind == PPO_KL_K3);
    const bool one = one_workgroup(batch, length);
    PPO_REQUIRE(one || (workspace && ppo_aligned(workspace, 8) && workspace_bytes >= ppo_policy_kl_loss_workspace_bytes(batch, length)));
    PolicyArgs a;
    a.lp = log_probs; a.old_lp = old_log_probs; a.adv = advantages; a.ref_lp = ref_log_probs; a.mask = mask;
    a.g = g_log_probs; a.out6 = out6;
    a.partials = reinterpret_cast<double *>(workspace);
    a.counts = a.partials + (size_t)SEQ_MAX_BLOCKS * NSUM;
    a.row_counts = reinterpret_cast<int *>(a.counts + 2 * COUNT_MAX_BLOCKS);
    a.B = batch; a.L = length; a.lp_stride = lp_stride; a.old_stride = old_stride; a.adv_stride = adv_stride; a.ref_stride = ref_stride;
    a.mask_stride = mask_stride;
    a.log_hi = log1p(clip_high); a.log_lo = log1p(-clip_low); a.kl_coef = kl_coef;
    a.hi = (float)(1.0 + clip_high); a.lo = (float)(1.0 - clip_low); a.kl_coef_f = (float)kl_coef;
    a.kl = kl_kind; a.per_sequence = per_sequence; a.sequence_mean = sequence_mean;
    hipStream_t s = (hipStream_t)stream;
    const long groups = batch * ((length + 3) / 4);
    if (one) {
        a.count_blocks = 0;
        hipLaunchKernelGGL(k_policy_one, dim3(1), dim3(ONE_BLOCK), 0, s, a);
        return ppo_launch_status();
    }
    const long at_once = length > 256 ? SEQ_BLOCK / 64 : SEQ_BLOCK / 8, cb = (batch + at_once - 1) / at_once;
    a.count_blocks = (int)(cb < COUNT_MAX_BLOCKS ? cb : COUNT_MAX_BLOCKS);
    hipLaunchKernelGGL(k_policy_count, dim3(a.count_blocks), dim3(SEQ_BLOCK), 0, s, a);
    int rc = ppo_launch_status();
    if (rc) return rc;
    const long mb = (groups + SEQ_BLOCK - 1) / SEQ_BLOCK;
    const int blocks = (int)(mb < SEQ_MAX_BLOCKS ? mb : SEQ_MAX_BLOCKS);
    hipLaunchKernelGGL(k_policy_main, dim3(blocks), dim3(SEQ_BLOCK), 0, s, a);
    rc = ppo_launch_status();
    if (rc) return rc;
    hipLaunchKernelGGL(k_policy_final, dim3(1), dim3(FINAL_BLOCK), 0, s, a, blocks);
    return ppo_launch_status();
}

size_t ppo_preference_loss_workspace_bytes(long pairs, long chosen_length, long rejected_length)
{
    if (pairs < 0 || chosen_length < 0 || rejected_length < 0) return 0;
    const int chunks = pref_chunks(pairs, chosen_length, rejected_length);
    return chunks == 0 ? 0 : chunks == 1 ? (size_t)pairs * 2 * sizeof(double) : (size_t)pairs * 4 * chunks * sizeof(double);
}

int ppo_preference_loss(const float *chosen, long chosen_stride, const float *ref_chosen, long ref_chosen_stride,
                        const uint8_t *mask_chosen, long mask_chosen_stride, long chosen_length, const float *rejected,
                        long rejected_stride, const float *ref_rejected, long ref_rejected_stride, const uint8_t *mask_rejected,
                        long mask_rejected_stride, long rejected_length, long pairs, int kind, double beta, double label_smoothing,
                        int average, float *out2, float *rewards, float *g_chosen, float *g_rejected, void *workspace,
                        size_t workspace_bytes, void *stream)
{
    PPO_REQUIRE(pairs >= 1 && pairs <= (1L << 28) && chosen_length >= 0 && rejected_length >= 0);
    PPO_REQUIRE(chosen_length <= (1L << 40) && rejected_length <= (1L << 40));
    PPO_REQUIRE(kind == PPO_PREF_SIGMOID || kind == PPO_PREF_HINGE || kind == PPO_PREF_IPO);
    PPO_REQUIRE(beta > 0.0 && beta <= 1e30 && label_smoothing >= 0.0 && label_smoothing < 0.5);
    PPO_REQUIRE(out2 && rewards && ppo_aligned(out2, 4) && ppo_aligned(rewards, 4) && ppo_aligned(g_chosen, 4) && ppo_aligned(g_rejected, 4));
    const int chunks = pref_chunks(pairs, chosen_length, rejected_length);
    PPO_REQUIRE(chunks == 0 || (workspace && ppo_aligned(workspace, 8) &&
                                workspace_bytes >= ppo_preference_loss_workspace_bytes(pairs, chosen_length, rejected_length)));
    PrefArgs a;
    a.side[0] = PrefSide{chosen, ref_chosen, mask_chosen, g_chosen, chosen_length, chosen_stride, ref_chosen_stride, mask_chosen_stride};
    a.side[1] = PrefSide{rejected, ref_rejected, mask_rejected, g_rejected, rejected_length, rejected_stride, ref_rejected_stride, mask_rejected_stride};
    for (const PrefSide &s : a.side) {
        if (s.L == 0) continue;
        PPO_REQUIRE(rows_ok(s.lp, pairs, s.L, s.lp_stride) && (!s.ref || rows_ok(s.ref, pairs, s.L, s.ref_stride)));
        PPO_REQUIRE(!s.mask || (s.mask_stride >= 0 && (__int128)(pairs - 1) * s.mask_stride + s.L < ((__int128)1 << 60)));
    }
    a.pair = a.partials = reinterpret_cast<double *>(workspace);
    a.out2 = out2; a.rewards = rewards; a.B = pairs; a.inv_pairs = 1.0 / (double)pairs; a.beta = beta; a.smoothing = label_smoothing; a.kind = kind; a.average = average;
    a.chunks = chunks;
    hipStream_t s = (hipStream_t)stream;
    if (chunks == 0) {
        hipLaunchKernelGGL(k_pref_one, dim3(1), dim3(ONE_BLOCK), 0, s, a);
        return ppo_launch_status();
    }
    if (chunks == 1) {
        constexpr long MOST = 1L << 20;            // a launch has fewer than 2^32 threads
        for (long first = 0; first < pairs; first += MOST) {
            hipLaunchKernelGGL(k_pref_pair, dim3((unsigned)(pairs - first < MOST ? pairs - first : MOST)), dim3(SEQ_BLOCK), 0, s, a, first);
            const int rc = ppo_launch_status();
            if (rc) return rc;
        }
        hipLaunchKernelGGL(k_pref_final, dim3(1), dim3(SEQ_BLOCK), 0, s, a);
    } else {
        hipLaunchKernelGGL(k_pref_sum, dim3((unsigned)(2 * pairs * chunks)), dim3(SEQ_BLOCK), 0, s, a);
        const int rc = ppo_launch_status();
        if (rc) return rc;
        hipLaunchKernelGGL(k_pref_grad, dim3((unsigned)(2 * pairs * chunks + 1)), dim3(SEQ_BLOCK), 0, s, a);
    }
    return ppo_launch_status();
}

}  // extern "C"
