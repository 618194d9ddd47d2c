// y = act(x W^T + b) + residual, forward and backward, on the matrix cores -- gfx950.
//
// Beside ppo_linear_wgrad (wgrad.hip: layers of at most 64 x 64 over millions of rows) for layers of any size and for
// 16-bit types.  With z = x W^T + b, y = act(z) + r the forward pass also keeps d = act'(z) where a gradient will be
// asked for; then for a gradient g of y
//     u = g d,   g_x = u W,   g_W = u^T x,   g_b = sum over rows of u.
// d is kept rather than z: act'(z) of a z rounded to bf16 is off by 1.5 % for tanh at z = 4.  It is kept in f16 for bf16
// layers (|d| < 1.2; 8 times finer than bf16 for |d| >= 2^-14, steps of 2^-24 below, where g d hardly counts beside others) and in f32
// for the others, so that the one rounding that counts beside the outputs' own is that of u to the inputs' type, which the two
// products need: g_x and g_W are off by sqrt 2 of what the outputs' rounding alone leaves.  g_b sums u unrounded, in f32.
//
// One product, C[m, n] = sum_k A[m, k] B[n, k], serves all three, each operand with its rows along m (n) or along k.
//   * 16-bit inputs: v_mfma_f32_16x16x32_{bf16,f16}, f32 accumulators.
//   * f32 inputs: every operand split in registers into three bf16 pieces that represent it exactly (mfma_split.h), six
//     products of order <= 2 into one f32 accumulator: the three left out are below 2^-23 of the product.  f32 matrix
//     instructions run at 1/16 of the bf16 rate, so six of these are 2.7 times as fast.  Tiles with an infinite operand take those.
// A workgroup of 8 waves computes 256 x 256 of C (4 waves: 128 x 128 where there would be too few of the larger ones, 128 x 64
// or 64 x 128 where C has no more columns or rows), a wave 128 x 64, 64 x 64 or 32 x 64 of it.  Rows of 128 bytes of k (64
// halves, 32 floats; where an operand's rows go along k, as many rows of the tile's width) are brought straight into LDS, the
// next stages on their way while the matrix cores work on this one.  16-byte pieces are swizzled inside their row so that what
// a fragment read touches falls into different banks.  The operands of v_mfma are swapped (B first), so that a lane's
// accumulators run along n.
// Measured: bf16 8192 x 4096 -> 16384 with gelu 875 us forward (1.26 PFLOP/s) and 1715 us backward (1.28, of them 180 for u and
// its column sums); f32 4096 x 4096 -> 4096 608 us forward (226 TFLOP/s, as bf16 products 1.36 PFLOP/s).  Plain library products
// of these sizes reach 1.6 PFLOP/s in bf16 and 0.154 in f32.
#include "token_common.h"
#include "mfma_split.h"

using namespace ppo_token;

namespace {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using h8v = __attribute__((ext_vector_type(8))) _Float16;
using b8v = __attribute__((ext_vector_type(8))) __bf16;

template <class T> __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c)
{
    if constexpr (std::is_same_v<T, F16>)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
}

// ---- activations: value and derivative ------------------------------------------------------------------------------
// No library functions, whose branches cost more than the rest of an epilogue (with them bf16 8192 x 4096 -> 16384 with gelu took
// 1284 us forward, and 970 with no activation at all; f32 191 x 106 -> 607 43 us, 33 with these, and 19 with a piece's values
// worked out together, 15 with no activation).
// FAST, for 16-bit layers: a few 1e-7 of max(1, |value|), far below their half steps.  Otherwise, for f32 ones: the rounding of an
// exponential's argument is put right, a reciprocal gets a Newton step.  Measured on 2^21 arguments up to 12 and up to 100: values
// within 7 half steps of f32, derivatives within 9 of the larger of |d| and 1/4 (gelu's and silu's have a zero, at -0.75 and -1.28).
// The normal distribution's tail is P(> a) = e^(-a^2 / 2) h(t) t, t = 1 / (1 + 0.38 a / sqrt 2), whose exponential is the density that the
// derivative needs as well, h a polynomial fitted by Lawson's iteration for a up to 20: of degree 7, 1.1e-6 of the tail, or 10, 4e-8
// (with the coefficients and t's factor rounded to f32 as they stand here).
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.442695041f); }

// e^x, -208 <= x <= 0
__device__ __forceinline__ float exp_near(float x)
{
    const float t = x * 1.442695041f;
    const float lost = __builtin_fmaf(x, 1.925963e-8f, __builtin_fmaf(x, 1.442695041f, -t));   // of x log2 e
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e, lost * 0.6931471806f, e);
}

// 1 / x, x >= 1
template <bool FAST> __device__ __forceinline__ float inverse(float x)
{
    const float r = __builtin_amdgcn_rcpf(x);
    return FAST ? r : __builtin_fmaf(__builtin_fmaf(-x, r, 1.0f), r, r);
}

template <bool FAST> __device__ __forceinline__ void tanh_of(float z, float &y, float &d)
{
    const float a = fabsf(z);
    const float e = FAST ? exp_fast(-2.0f * a) : exp_near(-2.0f * fminf(a, 52.0f)), r = inverse<FAST>(1.0f + e);
    float t = (1.0f - e) * r;
    if constexpr (FAST) {
        t = a < 0.02f ? a - a * a * a * (1.0f / 3) : t;   // (what is left out: 2 a^5 / 15)
    } else {
        const float q = a * a;                            // the series to a^11: what is left out is below 2^-32
        float p = -1382.0f / 155925;
        p = __builtin_fmaf(p, q, 62.0f / 2835);
        p = __builtin_fmaf(p, q, -17.0f / 315);
        p = __builtin_fmaf(p, q, 2.0f / 15);
        p = __builtin_fmaf(p, q, -1.0f / 3);
        t = a < 0.25f ? __builtin_fmaf(a * q, p, a) : t;
    }
    y = copysignf(t, z);
    d = 4.0f * e * r * r;                               // 1 - tanh^2 without its cancellation
    if constexpr (!FAST) {
        y = z != z ? z : y;
        d = z != z ? z : d;
    }
}

template <bool FAST> __device__ __forceinline__ void gelu_of(float z, float &y, float &d)
{
    float q, g;                                         // P(> |z|) and sqrt(2 pi) times the density
    if constexpr (FAST) {
        const float a = fabsf(z), t = inverse<FAST>(__builtin_fmaf(a, 0.38f * 0.70710678f, 1.0f));
        g = __builtin_amdgcn_exp2f(a * a * -0.7213475204f);
        q = -0.0627071038f;
        q = __builtin_fmaf(q, t, 0.168012768f);
        q = __builtin_fmaf(q, t, -0.0349497572f);
        q = __builtin_fmaf(q, t, 0.123912774f);
        q = __builtin_fmaf(q, t, 0.0902986899f);
        q = __builtin_fmaf(q, t, 0.108288437f);
        q = __builtin_fmaf(q, t, 0.107143678f);
        q = q * t * g;
    } else {
        const float a = fminf(fabsf(z), 20.0f), t = inverse<FAST>(__builtin_fmaf(a, 0.38f * 0.70710678f, 1.0f));
        const float s = a * a, lost = __builtin_fmaf(a, a, -s);
        g = exp_near(-0.5f * s);
        g = __builtin_fmaf(g, -0.5f * lost, g);
        q = -0.015613814815878868f;
        q = __builtin_fmaf(q, t, 0.0887872651219368f);
        q = __builtin_fmaf(q, t, -0.19097009301185608f);
        q = __builtin_fmaf(q, t, 0.18277713656425476f);
        q = __builtin_fmaf(q, t, -0.10117244720458984f);
        q = __builtin_fmaf(q, t, 0.0877317488193512f);
        q = __builtin_fmaf(q, t, 0.04822973534464836f);
        q = __builtin_fmaf(q, t, 0.08668842911720276f);
        q = __builtin_fmaf(q, t, 0.09912792593240738f);
        q = __builtin_fmaf(q, t, 0.10721877962350845f);
        q = __builtin_fmaf(q, t, 0.10719534009695053f);
        q = q * t * g;
    }
    const float phi = z > 0.0f ? 1.0f - q : q;
    const bool far = fabsf(z) > 20.0f;                  // (NaN: near)
    y = far ? fmaxf(z, 0.0f) : z * phi;
    d = far ? (z > 0.0f ? 1.0f : 0.0f) : __builtin_fmaf(z * 0.3989422804f, g, phi);
}

template <bool FAST> __device__ __forceinline__ void silu_of(float z, float &y, float &d)
{
    float s, rest;                                      // s(z), 1 - s(z)
    if constexpr (FAST) {
        s = inverse<FAST>(1.0f + exp_fast(-z));
        rest = 1.0f - s;
    } else {
        const float e = exp_near(-fminf(fabsf(z), 104.0f)), r = inverse<FAST>(1.0f + e), near = e * r;
        s = z >= 0.0f ? r : near;
        rest = z >= 0.0f ? near : r;                    // (a difference would have lost its digits for large z)
    }
    y = z == -INFINITY ? 0.0f : z * s;
    d = fabsf(z) == INFINITY ? s : s * (1.0f + z * rest);
}

// N values at once
template <bool FAST, int N> __device__ __forceinline__ void activate(int act, const float (&z)[N], float (&y)[N], float (&d)[N])
{
    switch (act) {
    case PPO_ACT_TANH:
#pragma unroll
        for (int j = 0; j < N; ++j) tanh_of<FAST>(z[j], y[j], d[j]);
        break;
    case PPO_ACT_RELU:
#pragma unroll
        for (int j = 0; j < N; ++j) {
            y[j] = z[j] > 0.0f ? z[j] : (z[j] != z[j] ? z[j] : 0.0f);
            d[j] = z[j] > 0.0f ? 1.0f : 0.0f;
        }
        break;
    case PPO_ACT_GELU:
#pragma unroll
        for (int j = 0; j < N; ++j) gelu_of<FAST>(z[j], y[j], d[j]);
        break;
    case PPO_ACT_SILU:
#pragma unroll
        for (int j = 0; j < N; ++j) silu_of<FAST>(z[j], y[j], d[j]);
        break;
    default:
#pragma unroll
        for (int j = 0; j < N; ++j) {
            y[j] = z[j];
            d[j] = 1.0f;
        }
    }
}

template <class T> struct DerivOf { using type = F32; };
template <> struct DerivOf<BF16> { using type = F16; };
template <class T> using D = typename DerivOf<T>::type;

// N neighbouring elements of 16 bytes a piece
template <class T, int N> __device__ __forceinline__ void load_n(const typename T::raw *p, float (&v)[N])
{
    constexpr int E = 16 / T::BYTES;
    if constexpr (N <= E) {
        struct __attribute__((packed, aligned(T::BYTES))) Part { typename T::raw r[N]; };
        const Part w = *reinterpret_cast<const Part *>(p);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = T::load(w.r[j]);
    } else {
#pragma unroll
        for (int q = 0; q < N; q += E) {
            float w[E];
            load16<T>(p + q, w);
#pragma unroll
            for (int j = 0; j < E; ++j) v[q + j] = w[j];
        }
    }
}

template <class T, int N> __device__ __forceinline__ void store_n(typename T::raw *p, const float (&v)[N])
{
    constexpr int E = 16 / T::BYTES;
    static_assert(N % E == 0, "whole pieces");
#pragma unroll
    for (int q = 0; q < N; q += E) {
        float w[E];
#pragma unroll
        for (int j = 0; j < E; ++j) w[j] = v[q + j];
        store16<T>(p + q, w);
    }
}

// ---- operand preparation: multiply by d, pad, sum columns ----------------------------------------------------------
// src [R, C] of T with row stride ld (times mul [R, C] of D<T>, contiguous) -> rows [R, Cp] of T, Cp the next multiple of a
// stage's k, zero-filled; sums [tiles of 64 rows][C] f32 = column sums of a tile.
struct PrepArgs {
    const void *src, *mul;
    void *rows;
    float *sums;
    long R, C, ld, Cp;
    int tiles_x;                           // tiles of 64 x 64 a row of tiles
};

// up to three of them in one launch: tiles first[j] .. first[j + 1] - 1 are those of job[j]
struct PrepJobs {
    PrepArgs job[3];
    unsigned first[4];
};

template <class T> __global__ void __launch_bounds__(256) k_prep(PrepJobs jobs)
{
    const int which = blockIdx.x < jobs.first[1] ? 0 : blockIdx.x < jobs.first[2] ? 1 : 2;
    const PrepArgs a = which == 0 ? jobs.job[0] : which == 1 ? jobs.job[1] : jobs.job[2];
    const unsigned id = blockIdx.x - (which == 0 ? 0u : which == 1 ? jobs.first[1] : jobs.first[2]);
    const long tile_y = id / (unsigned)a.tiles_x, tile_x = id % (unsigned)a.tiles_x;
    constexpr int E = 16 / T::BYTES, TPR = 64 / E, RPP = 256 / TPR;   // threads a row of 64, rows a pass
    using raw = typename T::raw;
    __shared__ float colsum[RPP][64];
    const int tc = threadIdx.x % TPR * E, tr = threadIdx.x / TPR;
    const long gc = tile_x * 64 + tc;
    const raw *src = reinterpret_cast<const raw *>(a.src);
    const typename D<T>::raw *mul = reinterpret_cast<const typename D<T>::raw *>(a.mul);
    float sum[E];
#pragma unroll
    for (int j = 0; j < E; ++j) sum[j] = 0.0f;
#pragma unroll
    for (int p = 0; p < 64 / RPP; ++p) {
        const long gr = tile_y * 64 + p * RPP + tr;
        float v[E];
        if (gr < a.R && gc + E <= a.C) {
            load16<T>(src + gr * a.ld + gc, v);
            if (mul) {
                float w[E];
                load_n<D<T>, E>(mul + gr * a.C + gc, w);
#pragma unroll
                for (int j = 0; j < E; ++j) v[j] *= w[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) {
                v[j] = 0.0f;
                if (gr < a.R && gc + j < a.C) {
                    v[j] = T::load(src[gr * a.ld + gc + j]);
                    if (mul) v[j] *= D<T>::load(mul[gr * a.C + gc + j]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < E; ++j) sum[j] += v[j];
        if (a.rows && gr < a.R && gc < a.Cp) store16<T>(reinterpret_cast<raw *>(a.rows) + gr * a.Cp + gc, v);
    }
    if (!a.sums) return;
#pragma unroll
    for (int j = 0; j < E; ++j) colsum[tr][tc + j] = sum[j];
    __syncthreads();
    if (threadIdx.x < 64 && tile_x * 64 + threadIdx.x < a.C) {
        float s = 0.0f;
        for (int k = 0; k < RPP; ++k) s += colsum[k][threadIdx.x];
        a.sums[tile_y * a.C + tile_x * 64 + threadIdx.x] = s;
    }
}

// 64 columns a workgroup, its 16 waves share the tiles of rows
template <class T> __global__ void __launch_bounds__(1024) k_bias_grad(const float *sums, long tiles, long C, typename T::raw *out)
{
    __shared__ float part[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const long c = (long)blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (c < C) {
#pragma unroll 4
        for (long t = w; t < tiles; t += 16) s += sums[t * C + c];
    }
    part[w][lane] = s;
    __syncthreads();
    if (w == 0 && c < C) {
        s = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; ++k) s += part[k][lane];
        out[c] = T::store(s);
    }
}

// ---- the product -----------------------------------------------------------------------------------------------------
constexpr uint32_t KEEP = 0x7fc5a5a5u;        // marks a result that is not written again

struct GemmArgs {
    const void *A, *B;                 // [M, k], [N, k]; rows lda, ldb bytes apart
    long M, N, lda, ldb;
    long K;                            // the last stage's elements from here on count as 0
    int steps, steps_per_split;        // steps of 128 bytes of k
    int tiles_m, tiles_n;
    float *partial;                    // [splits][M][N], or NULL: the epilogue below
    const void *bias, *residual;
    long res_ld;
    void *out, *deriv;                 // [M, N] contiguous
    int act;
};

template <class T> __device__ __forceinline__ void finish(const GemmArgs &g, long m, long n, float z, float &y, float &d)
{
    using raw = typename T::raw;
    if (g.bias) z += T::load(reinterpret_cast<const raw *>(g.bias)[n]);
    const float in[1] = {z};
    float value[1], slope[1];
    activate<T::BYTES == 2, 1>(g.act, in, value, slope);
    y = value[0];
    d = slope[0];
    if (g.residual) y += T::load(reinterpret_cast<const raw *>(g.residual)[m * g.res_ld + n]);
}

// 16 bytes of neighbouring results of row m, or as many as the row still has; `bias` is theirs
template <class T> __device__ __forceinline__ void epilogue(const GemmArgs &g, long m, long n, const float (&z)[16 / T::BYTES], const float (&bias)[16 / T::BYTES])
{
    using raw = typename T::raw;
    constexpr int E = 16 / T::BYTES;
    raw *out = reinterpret_cast<raw *>(g.out) + m * g.N + n;
    typename D<T>::raw *der = g.deriv ? reinterpret_cast<typename D<T>::raw *>(g.deriv) + m * g.N + n : nullptr;
    const bool whole = n + E <= g.N;
    float r[E], v[E], y[E], d[E];
    if (g.residual) {
        const raw *p = reinterpret_cast<const raw *>(g.residual) + m * g.res_ld + n;
        if (whole) {
            load16<T>(p, r);
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) r[j] = n + j < g.N ? T::load(p[j]) : 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = z[j] + bias[j];
    activate<T::BYTES == 2, E>(g.act, v, y, d);             // (together: one after the other they wait for each other)
    if (g.residual) {
#pragma unroll
        for (int j = 0; j < E; ++j) y[j] += r[j];
    }
    if (whole) {
        store16<T>(out, y);
        if (der) store_n<D<T>, E>(der, d);
    } else {
#pragma unroll
        for (int j = 0; j < E; ++j) {
            if (n + j < g.N) {
                out[j] = T::store(y[j]);
                if (der) der[j] = D<T>::store(d[j]);
            }
        }
    }
}

template <class T> __device__ __forceinline__ void load_bias(const GemmArgs &g, long n, float (&bias)[16 / T::BYTES])
{
    constexpr int E = 16 / T::BYTES;
    const typename T::raw *p = reinterpret_cast<const typename T::raw *>(g.bias);
#pragma unroll
    for (int j = 0; j < E; ++j) bias[j] = p && n + j < g.N ? T::load(p[n + j]) : 0.0f;
}

// Swizzles: piece c (16 bytes) of a row of 128 bytes of k lies at c ^ f(row) in LDS.  A ds_read_b128 is served 16 lanes a
// cycle from 64 banks: lanes {0-3, 12-15, 20-23, 24-27}, {4-11, 16-19, 28-31} and these + 32.  In a fragment read lane l wants
// piece l / 16 of the fragment's row l % 16, so with f = a r1 ^ b r2 ^ d r3 (r1 .. r3 the bits 1 .. 3 of the row) the lanes of a
// group fall into different places (row & 1, c ^ f) if 0, b ^ d, 1 ^ b and 1 ^ d differ modulo a: (4, 2, 3).  The f32 fragments'
// pieces are two apart, which makes that 0, b ^ d, 2 ^ b, 2 ^ d: (4, 1, 3).  (f = row & 7 costs twice the cycles a read.)
template <int BYTES> __device__ __forceinline__ int swizzle(int row)
{
    return (row >> 1 & 1) * 4 ^ (row >> 2 & 1) * (BYTES == 2 ? 2 : 1) ^ (row >> 3 & 1) * 3;
}
// Operands whose rows go along k lie in LDS as they come, a row a k.  An f32 fragment is eight reads of a float, one a k, and
// a row's pieces are moved by 4 (k / 8) so that the four k groups of such a read fall into different banks; a 16-bit one is
// two ds_read_b64_tr_b16, which hand lane i of 16 the column i of four rows of 16: 32 bytes of 16 rows a read, moved by 32
// bytes times (k % 4, k / 8 % 2) so that 8 of them fill the banks.
template <int BYTES, int ROW> __device__ __forceinline__ int moved(int k)
{
    if constexpr (BYTES == 4) return (k >> 3) * 4;
    return (ROW == 128 ? (k >> 1 & 1) | (k >> 3 & 1) << 1 : (k & 3) | (k >> 3 & 1) << 2) * 2;   // (rows of 128 bytes: k & 1 moves them already)
}

// 64 lanes bring 16 bytes each from rsrc[voff + soff] to LDS at lds + 16 lane.  In asm because the compiler's own form of
// this load makes every LDS read wait for all of them; it has no destination register, and the loop below waits itself.
__device__ __forceinline__ void load_lds(u32x4 rsrc, uint32_t voff, int soff, uint32_t lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc), "s"(soff) : "memory");
}

__device__ __forceinline__ u32x4 buffer_of(const void *p, long bytes)
{
    const uint64_t at = reinterpret_cast<uint64_t>(p);
    const uint32_t n = bytes > 0xffffffffL ? 0xffffffffu : (uint32_t)bytes;
    return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)at), (uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) & 0xffffu,
                 (uint32_t)__builtin_amdgcn_readfirstlane((int)n), 0x00027000u};
}

// KA, KB: that operand lies [k, M] (or [k, N]), its rows along k
template <class T, int BM, int BN, int WAVES_M, int WAVES_N, bool KA, bool KB>
__global__ void __launch_bounds__(64 * WAVES_M * WAVES_N) k_gemm(GemmArgs g)
{
    constexpr int WAVES = WAVES_M * WAVES_N, WM = BM / WAVES_M, WN = BN / WAVES_N, MI = WM / 16, NI = 4;
    static_assert(WN == 16 * NI && MI * 16 * WAVES_M == BM, "whole 16 x 16 products");
    constexpr int LA = BM / 8 / WAVES, LB = BN / 8 / WAVES;          // loads a wave and stage (8 rows each)
    constexpr int A_STAGE = BM * 128, B_STAGE = BN * 128, B_AT = (T::BYTES == 2 ? 3 : 2) * A_STAGE;
    constexpr int PI = MI < 4 ? MI : 4, ROWS = WAVES_M * 16 * PI, LD = BN * 4 + 16;   // the results' way out, below
    constexpr int STAGES = B_AT + 2 * B_STAGE;
    __shared__ __align__(1024) char lds[STAGES > ROWS * LD ? STAGES : ROWS * LD];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WAVES_N, wn = wave % WAVES_N;

    // tiles: an XCD (workgroups go round them one by one) takes a run of neighbouring ones, in bands of 8 rows of tiles,
    // so that what its L2 holds is used by several of its workgroups
    const int tiles = g.tiles_m * g.tiles_n;
    int id = blockIdx.x;
    {
        const int x = id % 8, q = tiles / 8, rem = tiles % 8;
        id = x * q + (x < rem ? x : rem) + id / 8;
    }
    const int band = 8 * g.tiles_n, first = id / band * 8, high = g.tiles_m - first < 8 ? g.tiles_m - first : 8;
    const long m0 = (long)(first + id % band % high) * BM, n0 = (long)(id % band / high) * BN;
    const int s0 = blockIdx.y * g.steps_per_split, s1 = s0 + g.steps_per_split < g.steps ? s0 + g.steps_per_split : g.steps;

    constexpr int KS = 128 / T::BYTES, ROW_A = BM * T::BYTES, ROW_B = BN * T::BYTES;   // k a stage; bytes of a row along k
    const long kbytes = (g.K * T::BYTES + 3) / 4 * 4;                // (whole dwords: the last may hold an element that is masked)
    const int tail = s1 == g.steps ? (int)(g.K - (g.steps - 1L) * KS) : KS;   // of the last one
    const long rows_a = g.M - m0 < BM ? g.M - m0 : BM, rows_b = g.N - n0 < BN ? g.N - n0 : BN;
    const char *pa0 = reinterpret_cast<const char *>(g.A) + (KA ? m0 * T::BYTES : m0 * g.lda);
    const char *pb0 = reinterpret_cast<const char *>(g.B) + (KB ? n0 * T::BYTES : n0 * g.ldb);
    const u32x4 ra = buffer_of(pa0, KA ? 0 : (rows_a - 1) * g.lda + kbytes), rb = buffer_of(pb0, KB ? 0 : (rows_b - 1) * g.ldb + kbytes);
    // where in the operand what this lane brings in load i lies (256 rows of less than 2^24 bytes: below 2^32)
    auto offset = [&](auto along_k, auto row_bytes, int i, long rows, long ld) {
        if constexpr (along_k()) {
            constexpr int pieces = row_bytes() / 16;
            const int k = (i * WAVES + wave) * (64 / pieces) + lane / pieces;
            return (uint32_t)k * (uint32_t)ld + ((lane % pieces) ^ moved<T::BYTES, row_bytes()>(k)) * 16;
        } else {
            const int row = (i * WAVES + wave) * 8 + lane / 8, have = row < rows ? row : (int)rows - 1;   // rows past the end repeat the last
            return (uint32_t)have * (uint32_t)ld + ((lane % 8) ^ swizzle<T::BYTES>(row)) * 16;
        }
    };
    uint32_t va[LA], vb[LB];
#pragma unroll
    for (int i = 0; i < LA; ++i) va[i] = offset(std::bool_constant<KA>{}, std::integral_constant<int, ROW_A>{}, i, rows_a, g.lda);
#pragma unroll
    for (int i = 0; i < LB; ++i) vb[i] = offset(std::bool_constant<KB>{}, std::integral_constant<int, ROW_B>{}, i, rows_b, g.ldb);
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    // load i of a stage's A or B to the place that begins at `to`.  What is read past a row's end is the next row's beginning,
    // or nothing behind the last row: past K it is masked out of the last stage's fragments, and where the operand's rows go
    // along k it belongs to columns whose results are not kept.
    // Along k the descriptor begins at the stage's first row and goes on to the operand's end; stages are loaded one after the
    // other.  (Worked out anew for each it takes 40 scalar instructions a stage, as long as a tile of 128 x 128's products.)
    struct Along {
        const char *p;
        long left, step;
        __device__ u32x4 take(bool last)
        {
            const u32x4 d = buffer_of(p, left);
            if (last) {
                p += step;
                left -= step;
            }
            return d;
        }
    };
    auto along_a = [&] { return Along{pa0 + (long)s0 * KS * g.lda, (g.K - (long)s0 * KS - 1) * g.lda + ((g.M - m0) * T::BYTES + 3) / 4 * 4, KS * g.lda}; };
    auto along_b = [&] { return Along{pb0 + (long)s0 * KS * g.ldb, (g.K - (long)s0 * KS - 1) * g.ldb + ((g.N - n0) * T::BYTES + 3) / 4 * 4, KS * g.ldb}; };
    Along al = along_a(), bl = along_b();
    auto load_a = [&](int s, int to, int i) {
        const uint32_t at = base + wave * 1024 + to + i * WAVES * 1024;
        if constexpr (KA)
            load_lds(al.take(i == LA - 1), va[i], 0, at);
        else
            load_lds(ra, va[i], s * 128, at);
    };
    auto load_b = [&](int s, int to, int i) {
        const uint32_t at = base + wave * 1024 + B_AT + to + i * WAVES * 1024;
        if constexpr (KB)
            load_lds(bl.take(i == LB - 1), vb[i], 0, at);
        else
            load_lds(rb, vb[i], s * 128, at);
    };
    auto stage_a = [&](int s, int to) {
#pragma unroll
        for (int i = 0; i < LA; ++i) load_a(s, to, i);
    };
    auto stage_b = [&](int s, int to) {
#pragma unroll
        for (int i = 0; i < LB; ++i) load_b(s, to, i);
    };

    // fragment reads: lane q = lane % 16 reads k piece kg = lane / 16 of row q (+ 16 i or 16 j) of a wave's rows
    const int q = lane & 15, kg = lane >> 4;
    const int row_a = wm * WM + q, row_b = wn * WN + q;
    const int pa = row_a * 128, pb = B_AT + row_b * 128, xa = swizzle<T::BYTES>(row_a), xb = swizzle<T::BYTES>(row_b);
    // along k, 16 bits: the lane's four columns of row k of its group; column block i lies at ^ 32 i
    const int tk = kg * 8 + (q >> 2);
    const int ta = tk * ROW_A + ((wm * WM * 2 + (q & 3) * 8) ^ moved<2, ROW_A>(tk) * 16);
    const int tb = B_AT + tk * ROW_B + ((wn * WN * 2 + (q & 3) * 8) ^ moved<2, ROW_B>(tk) * 16);

    f32x4 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    ppo_net::Bf16Select sel;
    if constexpr (T::BYTES == 4) sel.init();

    // acc[i][j][e] is C[m0 + wm WM + 16 i + q][n0 + wn WN + 16 j + 4 kg + e].  The results go through LDS, PI rows of
    // products of every wave at a time, so that a wave finishes and stores whole rows: from the accumulators' layout a
    // store touched 32 cache lines, and each residual and derivative as many again.  (A pad of 16 bytes a row puts the 16
    // rows of a write into different banks.)
    constexpr int E = 16 / T::BYTES, LANES = BN / E, STEP = 64 * WAVES / LANES;
    static_assert(MI % PI == 0, "whole passes");
    const int col = threadIdx.x % LANES * E, row0 = threadIdx.x / LANES;
    const long nn = n0 + col;
    auto leave = [&](auto second, auto value) {             // second: only what is not KEEP
        float bias[E];
        load_bias<T>(g, nn, bias);
#pragma unroll
        for (int pass = 0; pass < MI / PI; ++pass) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < PI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j)
                    *reinterpret_cast<f32x4 *>(lds + ((wm * PI + i) * 16 + q) * LD + (wn * WN + j * 16 + kg * 4) * 4) = value(pass * PI + i, j);
            __syncthreads();
#pragma clang loop unroll(disable)
            for (int r = row0; r < ROWS; r += STEP) {
                const long m = m0 + r / (16 * PI) * WM + pass * 16 * PI + r % (16 * PI);
                if (m >= g.M || nn >= g.N) continue;
                float z[E];
#pragma unroll
                for (int j = 0; j < E; j += 4) {
                    const f32x4 v = *reinterpret_cast<const f32x4 *>(lds + r * LD + (col + j) * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[j + e] = v[e];
                }
                if constexpr (second()) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        if (nn + e >= g.N || __builtin_bit_cast(uint32_t, z[e]) == KEEP) continue;
                        if (g.partial) {
                            g.partial[((long)blockIdx.y * g.M + m) * g.N + nn + e] = z[e];
                        } else {
                            float y, d;
                            finish<T>(g, m, nn + e, z[e], y, d);
                            reinterpret_cast<typename T::raw *>(g.out)[m * g.N + nn + e] = T::store(y);
                            if (g.deriv) reinterpret_cast<typename D<T>::raw *>(g.deriv)[m * g.N + nn + e] = D<T>::store(d);
                        }
                    }
                } else if (g.partial) {
                    float *p = g.partial + ((long)blockIdx.y * g.M + m) * g.N + nn;
                    if (nn + E <= g.N) {
                        store_n<F32, E>(p, z);
                    } else {
#pragma unroll
                        for (int e = 0; e < E; ++e)
                            if (nn + e < g.N) p[e] = z[e];
                    }
                } else {
                    epilogue<T>(g, m, nn, z, bias);
                }
            }
        }
    };

    if constexpr (T::BYTES == 2) {
        // A stage is two halves of 32 k.  While the matrix cores work on one half's fragments the next half's are read, so
        // no product waits for LDS, and the barrier between two stages lies between two runs of products whose operands
        // are in registers already: behind it this stage's places are free (its second half has been read by all) and the
        // next stage has landed.  160 KB hold three stages of A and two of B: B's loads have one stage's time to arrive,
        // A's, which go out behind them, two.  (What bounds this loop is the way from L2 and the last-level cache: without
        // the products it takes 605 of its 790 us for 8192 x 4096 x 16384; with two places for both, sent out together, a
        // load had to arrive within 1.5 us and the loop waited for it.  Rows of 64 bytes in a ring of five stages double
        // the requests and are slower still.)
        struct Half { u32x4 a[MI], b[NI]; };
        Half h0, h1;
        // one read of a half's fragments, in the order in which its products want them
        auto turned = [&](int at, int row_bytes) {
            using s4 = __attribute__((ext_vector_type(4))) short;
            using u2 = __attribute__((ext_vector_type(2))) uint32_t;
            typedef __attribute__((address_space(3))) s4 *ptr;
            const u2 lo = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(lds + at)));
            const u2 hi = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(lds + at + 4 * row_bytes)));
            return u32x4{lo[0], lo[1], hi[0], hi[1]};
        };
        auto fetch = [&](int at_a, int at_b, int half, Half &h, int r) {
            const int c = half * 4 + kg;
            if (r < NI) {
                if constexpr (KB)
                    h.b[r] = turned(((at_b + tb) ^ r * 32) + half * 32 * ROW_B, ROW_B);
                else
                    h.b[r] = *reinterpret_cast<const u32x4 *>(lds + at_b + pb + r * 2048 + (c ^ xb) * 16);
            } else {
                if constexpr (KA)
                    h.a[r - NI] = turned(((at_a + ta) ^ (r - NI) * 32) + half * 32 * ROW_A, ROW_A);
                else
                    h.a[r - NI] = *reinterpret_cast<const u32x4 *>(lds + at_a + pa + (r - NI) * 2048 + (c ^ xa) * 16);
            }
        };
        // a half's products one by one, and between them, in this order, the reads of the next half and the loads: left to
        // itself the compiler sends all loads first, which blocks the wave, and with it its products, until the address
        // unit has taken them
        auto work = [&](const Half &now, auto &&between) {
            constexpr int P = MI * NI;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const int i = p / NI, j = p % NI;
                acc[i][j] = mfma<T>(now.b[j], now.a[i], acc[i][j]);
                __builtin_amdgcn_sched_barrier(0);
                between(p, P);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        constexpr int R = MI + NI, GAP = 2 * R <= MI * NI ? 2 : 1;   // a read to every other product where there are enough
        static_assert(GAP * R <= MI * NI && LA + LB <= MI * NI, "room for the reads and loads");
        const int n = s1 - s0;
        int a_now = 0, a_next = A_STAGE, b_now = 0, b_next = B_STAGE;
        // what lies past K in the last stage is not of this row: 0
        auto cut = [&](Half &h, int half) {
            if (tail < KS) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int in = tail - (half * 32 + kg * 8 + 2 * e);
                    const uint32_t keep = in >= 2 ? 0xffffffffu : in == 1 ? 0xffffu : 0u;
#pragma unroll
                    for (int j = 0; j < NI; ++j) h.b[j][e] &= keep;
#pragma unroll
                    for (int i = 0; i < MI; ++i) h.a[i][e] &= keep;
                }
            }
        };
        auto turn = [&](int s, auto left) {                 // left: stages behind this one, 3 for three or more
            if constexpr (left() == 0) cut(h0, 0);
            work(h0, [&](int p, int) {
                if (p % GAP == 0 && p / GAP < R) fetch(a_now, b_now, 1, h1, p / GAP);
            });
            if constexpr (left() >= 2)
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LA) : "memory");   // A of stage s + 2 may be on its way
            else
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if constexpr (left() == 0) cut(h1, 1);
            __builtin_amdgcn_sched_barrier(0);
            work(h1, [&](int p, int P) {
                constexpr int NL = LB + LA;
                const int l = p * NL / P;
                if (l != (p + 1) * NL / P) {
                    if constexpr (left() >= 2) {
                        if (l < LB) load_b(s0 + s + 2, b_now, l);
                    }
                    if constexpr (left() >= 3) {
                        if (l >= LB) load_a(s0 + s + 3, a_now, l - LB);
                    }
                }
                if constexpr (left() >= 1) {
                    if (p % GAP == 0 && p / GAP < R) fetch(a_next, b_next, 0, h0, p / GAP);
                }
            });
            const int was = b_now;
            b_now = b_next;
            b_next = was;
            a_now = a_next;
            a_next = a_next == 2 * A_STAGE ? 0 : a_next + A_STAGE;
        };
        stage_a(s0, 0);
        stage_b(s0, 0);
        if (n > 1) {
            stage_a(s0 + 1, A_STAGE);
            stage_b(s0 + 1, B_STAGE);
        }
        if (n > 2) {
            stage_a(s0 + 2, 2 * A_STAGE);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * LA + LB) : "memory");
        } else if (n > 1) {
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LA + LB) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int r = 0; r < R; ++r) fetch(0, 0, 0, h0, r);
        int s = 0;
        for (; s + 3 < n; ++s) turn(s, std::integral_constant<int, 3>{});
        if (n > 2) turn(s++, std::integral_constant<int, 2>{});
        if (n > 1) turn(s++, std::integral_constant<int, 1>{});
        turn(s, std::integral_constant<int, 0>{});
        leave(std::false_type{}, [&](int i, int j) { return acc[i][j]; });
    } else {
        // plain: by the f32 matrix instructions, for the few tiles that need it (below)
        auto step = [&](int s, auto last, auto plain) {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();                   // stage s has landed for every wave, and nobody reads the other one
            asm volatile("" ::: "memory");
            const int now = (s - s0) & 1;
            if constexpr (!last()) {
                stage_a(s + 1, (now ^ 1) * A_STAGE);
                stage_b(s + 1, (now ^ 1) * B_STAGE);
            }
            const char *at_a = lds + now * A_STAGE, *at_b = lds + now * B_STAGE;
            auto split = [&](f32x4 lo, f32x4 hi, u32x4(&f)[3]) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t w0, w1, w2;
                    ppo_net::split3_bf16(e < 2 ? lo[2 * e] : hi[2 * e - 4], e < 2 ? lo[2 * e + 1] : hi[2 * e - 3], sel, w0, w1, w2);
                    f[0][e] = w0;
                    f[1][e] = w1;
                    f[2][e] = w2;
                }
            };
            const int c = 2 * kg, ca0 = (c ^ xa) * 16, ca1 = ((c + 1) ^ xa) * 16, cb0 = (c ^ xb) * 16, cb1 = ((c + 1) ^ xb) * 16;
            // eight k of one row: two pieces of it, or a float of each of eight rows of k
            auto read_a = [&](int i, f32x4 &lo, f32x4 &hi) {
                if constexpr (KA) {
                    const char *p = at_a + kg * 8 * ROW_A + ((row_a + i * 16) ^ kg * 16) * 4;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        lo[e] = *reinterpret_cast<const float *>(p + e * ROW_A);
                        hi[e] = *reinterpret_cast<const float *>(p + (e + 4) * ROW_A);
                    }
                } else {
                    lo = *reinterpret_cast<const f32x4 *>(at_a + pa + i * 2048 + ca0);
                    hi = *reinterpret_cast<const f32x4 *>(at_a + pa + i * 2048 + ca1);
                }
            };
            auto read_b = [&](int j, f32x4 &lo, f32x4 &hi) {
                if constexpr (KB) {
                    const char *p = at_b + B_AT + kg * 8 * ROW_B + ((row_b + j * 16) ^ kg * 16) * 4;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        lo[e] = *reinterpret_cast<const float *>(p + e * ROW_B);
                        hi[e] = *reinterpret_cast<const float *>(p + (e + 4) * ROW_B);
                    }
                } else {
                    lo = *reinterpret_cast<const f32x4 *>(at_b + pb + j * 2048 + cb0);
                    hi = *reinterpret_cast<const f32x4 *>(at_b + pb + j * 2048 + cb1);
                }
            };
            auto cut = [&](f32x4 &lo, f32x4 &hi) {          // k past K are not of this row
                if constexpr (last()) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        lo[e] = kg * 8 + e < tail ? lo[e] : 0.0f;
                        hi[e] = kg * 8 + e + 4 < tail ? hi[e] : 0.0f;
                    }
                }
            };
            if constexpr (plain()) {
                // lane q, kg has k = 8 kg + e of row q for e = 0 .. 7: four k of a product of 16 x 16 x 4 for each e
                f32x4 fb[NI][2];
#pragma unroll
                for (int j = 0; j < NI; ++j) {
                    read_b(j, fb[j][0], fb[j][1]);
                    cut(fb[j][0], fb[j][1]);
                }
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    f32x4 fa[2];
                    read_a(i, fa[0], fa[1]);
                    cut(fa[0], fa[1]);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
#pragma unroll
                        for (int j = 0; j < NI; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[j][e / 4][e % 4], fa[e / 4][e % 4], acc[i][j], 0, 0, 0);
                }
            } else {
                u32x4 fb[NI][3];
#pragma unroll
                for (int j = 0; j < NI; ++j) {
                    f32x4 lo, hi;
                    read_b(j, lo, hi);
                    cut(lo, hi);
                    split(lo, hi, fb[j]);
                }
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    f32x4 lo, hi;
                    u32x4 fa[3];
                    read_a(i, lo, hi);
                    cut(lo, hi);
                    split(lo, hi, fa);
#pragma unroll
                    for (int t = 0; t < 6; ++t) {
                        constexpr int PA[6] = {0, 2, 1, 0, 1, 0}, PB[6] = {2, 0, 1, 1, 0, 0};   // small terms first
#pragma unroll
                        for (int j = 0; j < NI; ++j) acc[i][j] = mfma<BF16>(fb[j][PB[t]], fa[PA[t]], acc[i][j]);
                    }
                }
            }
        };
        auto run = [&](auto plain) {
            stage_a(s0, 0);
            stage_b(s0, 0);
            for (int s = s0; s + 1 < s1; ++s) step(s, std::false_type{}, plain);
            step(s1 - 1, std::true_type{}, plain);
        };
        run(std::false_type{});
        // An operand that is infinite, or above 3.38e38, where its first piece is, leaves NaN in every product that it is in, and the first
        // pieces of two large ones may have an infinite product where theirs is finite.  Where a tile holds a result that is not finite
        // it is worked out again by the f32 matrix instructions (4096^3 with a NaN in every tile: 2.1 times as long), and what was not
        // finite is replaced: such operands give what f32 arithmetic gives, as on the vector units, and the other results keep their
        // bits.  (KEEP is a NaN itself, which no product makes and an operand can only pass on: then the result was NaN and stays.)
        uint32_t wild[MI] = {}, found = 0;                  // bit 4 j + e of word i: acc[i][j][e] is not finite
        float sum = 0.0f;                                   // NaN where one is not
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum = __builtin_fmaf(acc[i][j][e], 0.0f, sum);
        if (__any(sum != sum)) {
#pragma unroll
            for (int i = 0; i < MI; ++i) {
#pragma unroll
                for (int j = 0; j < NI; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) wild[i] |= (fabsf(acc[i][j][e]) < INFINITY ? 0u : 1u) << (4 * j + e);
                found |= wild[i];
            }
        }
        leave(std::false_type{}, [&](int i, int j) { return acc[i][j]; });
        __syncthreads();                                    // (the results have left LDS)
        const bool mine = __any(found != 0);
        if (lane == 0) reinterpret_cast<int *>(lds)[wave] = mine;
        __syncthreads();
        int again = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) again |= reinterpret_cast<const int *>(lds)[w];
        if (__builtin_amdgcn_readfirstlane(again) != 0) {
            __syncthreads();                                // (the flags have been read)
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            al = along_a();
            bl = along_b();
            run(std::true_type{});
            leave(std::true_type{}, [&](int i, int j) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = wild[i] >> (4 * j + e) & 1 ? acc[i][j][e] : __builtin_bit_cast(float, KEEP);
                return v;
            });
        }
    }
}

// sums the splits of a row's 16 / BYTES neighbouring results and finishes them.  PARTS threads share the splits, each adds
// its run of them in order, and the first the runs: where there are many splits of few results one thread's loads take long.
template <class T, int PARTS> __global__ void __launch_bounds__(256) k_join(GemmArgs g, int splits)
{
    constexpr int E = 16 / T::BYTES, THREADS = 256 / PARTS;
    const int part = threadIdx.x / THREADS, at = threadIdx.x % THREADS;
    const long per_row = (g.N + E - 1) / E, id = (long)blockIdx.x * THREADS + at;
    const long m = id / per_row, n = (id - m * per_row) * E;
    const bool in = m < g.M;
    float z[E];
#pragma unroll
    for (int j = 0; j < E; ++j) z[j] = 0.0f;
    if (in) {
        const int have = g.N - n < E ? (int)(g.N - n) : E;
        const int s1 = (int)((long)splits * (part + 1) / PARTS);
#pragma unroll 4
        for (int s = (int)((long)splits * part / PARTS); s < s1; ++s) {
            const float *p = g.partial + ((long)s * g.M + m) * g.N + n;
            if (have == E) {
#pragma unroll
                for (int j = 0; j < E; j += 4) {
                    float w[4];
                    load16<F32>(p + j, w);
#pragma unroll
                    for (int k = 0; k < 4; ++k) z[j + k] += w[k];
                }
            } else {
#pragma unroll
                for (int j = 0; j < E; ++j)
                    if (j < have) z[j] += p[j];
            }
        }
    }
    if constexpr (PARTS > 1) {
        __shared__ float runs[PARTS - 1][THREADS][E + 1];
        if (part > 0) {
#pragma unroll
            for (int j = 0; j < E; ++j) runs[part - 1][at][j] = z[j];
        }
        __syncthreads();
        if (part > 0) return;
        for (int k = 0; k < PARTS - 1; ++k) {
#pragma unroll
            for (int j = 0; j < E; ++j) z[j] += runs[k][at][j];
        }
    }
    if (!in) return;
    float bias[E];
    load_bias<T>(g, n, bias);
    epilogue<T>(g, m, n, z, bias);
}

// ---- few rows: the weights are read once, by the vector units --------------------------------------------------------
// a wave COLS rows of W, lanes along k; ROWS rows of x
template <class T, int ROWS, int COLS> __global__ void __launch_bounds__(256) k_few_rows(GemmArgs g, long K)
{
    constexpr int E = 16 / T::BYTES;
    using raw = typename T::raw;
    const int lane = threadIdx.x & 63;
    const long n0 = ((long)blockIdx.x * 4 + (threadIdx.x >> 6)) * COLS, m0 = (long)blockIdx.y * ROWS;
    if (n0 >= g.N) return;
    const raw *x[ROWS], *w[COLS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) x[r] = reinterpret_cast<const raw *>(reinterpret_cast<const char *>(g.A) + (m0 + r < g.M ? m0 + r : g.M - 1) * g.lda);
#pragma unroll
    for (int c = 0; c < COLS; ++c) w[c] = reinterpret_cast<const raw *>(reinterpret_cast<const char *>(g.B) + (n0 + c < g.N ? n0 + c : g.N - 1) * g.ldb);
    float acc[ROWS][COLS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int c = 0; c < COLS; ++c) acc[r][c] = 0.0f;
    long k = (long)lane * E;
    for (; k + E <= K; k += 64 * E) {
        float wv[COLS][E];
#pragma unroll
        for (int c = 0; c < COLS; ++c) load16<T>(w[c] + k, wv[c]);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            float xv[E];
            load16<T>(x[r] + k, xv);
#pragma unroll
            for (int c = 0; c < COLS; ++c)
#pragma unroll
                for (int j = 0; j < E; ++j) acc[r][c] = __builtin_fmaf(xv[j], wv[c][j], acc[r][c]);
        }
    }
    for (; k < K; ++k) {                                    // (at most one lane has a part of 16 bytes left)
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int c = 0; c < COLS; ++c) acc[r][c] = __builtin_fmaf(T::load(x[r][k]), T::load(w[c][k]), acc[r][c]);
        if (k % E == E - 1) break;
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) acc[r][c] += __shfl_xor(acc[r][c], off, 64);
        }
    if (lane < ROWS && m0 + lane < g.M) {
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
            float z = 0.0f;
#pragma unroll
            for (int r = 0; r < ROWS; ++r) z = lane == r ? acc[r][c] : z;
            const float one[1] = {z};
            if (n0 + c < g.N) {
                float y, d;
                finish<T>(g, m0 + lane, n0 + c, one[0], y, d);
                reinterpret_cast<raw *>(g.out)[(m0 + lane) * g.N + n0 + c] = T::store(y);
                if (g.deriv) reinterpret_cast<typename D<T>::raw *>(g.deriv)[(m0 + lane) * g.N + n0 + c] = D<T>::store(d);
            }
        }
    }
}

// ---- host: how a product is cut -------------------------------------------------------------------------------------
// Which calls go to k_few_rows.  Measured, that against the matrix cores, us: weights of a few MB, which stay in L2 when
// they are read once for every 8 rows, 1000 x 1024 and 32 rows 10 / 15 in bf16, 12 / 15 in f32 (40 rows 12 / 14, 14 / 14); bf16
// 4000 x 4096 and 4 rows 12 / 15 (6 rows 27 / 14), 16384 x 4096 25 / 26 (6 rows 37 / 27), the same not in place, where the matrix
// cores need a padded copy of the weights first, 8 rows 44 / 83 (10 rows 87 / 83); f32 4000 x 4096 and 4 rows 20 / 24 (6 rows
// 33 / 24), 268 MB and 8 rows 65 / 72 (10 rows 105 / 73).
bool few_rows(long rows, long N, long K, long e, bool in_place)
{
    if (N * K * e <= 4L << 20) return rows <= 32;
    return rows <= (e == 2 ? (in_place ? 4 : 8) : (N * K * e > 128L << 20 ? 8 : 4));
}
constexpr long MOST_K = (1L << 22) - 128;   // 256 padded rows of so many floats still have 32-bit offsets

long k_padded(long k, long e) { return (k * e + 127) / 128 * 128 / e; }

enum Shape { SMALL, LARGE, NARROW_N, NARROW_M };   // of a tile: 128 x 128, 256 x 256, 128 x 64, 64 x 128

struct Plan {
    Shape shape;
    int tiles_m, tiles_n, steps, per_split, splits;
};

// The tile, and how many workgroups share a tile's k: the cheapest by a model of the 256 CUs fitted to measurements (us; 16-bit /
// f32).  A round of 256 x 256 tiles, one a CU: 19 + 1.4 / 4.6 a stage.  Of 128 x 128: 10 + 0.5 / 1.43 a stage alone on a CU, 0.9 / 2.6
// for two together; of the narrow ones 0.4 / 0.88 and 0.6 / 1.25.  Joining splits: 3 + 8 bytes a partial result at 4.5 TB/s.
// (Constants closer to single runs chose small tiles for bf16 3000 x 3000 x 3000, 85 us against 67.)
// Measured, large against small tiles, best splits of each: bf16 4096 x 4096 x 4096 99 against 115 us, 4096 x 4096 x 1024 35 / 39,
// 6000 x 3000 x 512 41 / 32, 2048 x 2048 x 2048 44 / 24, 1024 x 1024 x 8192 45 (8 splits) / 34 (4; unsplit 57), 300 x 1000 x 1024 22 (4) / 13;
// f32 16384 x 512 x 3136 286 (2) / 259, 512 x 3136 x 16384 314 (8) / 287 (5; unsplit 727).  Small against narrow tiles, at most 64 rows or
// columns: f32 4020 x 33 x 6985 51 (16) / 36 (16), 16384 x 64 x 2048 54 (4) / 37 (4), 65536 x 64 x 64 16 / 12, 64 x 512 x 16384 26 (64) / 20
// (64), 64 x 64 x 65536 33 (256; unsplit 2875) / 28 (256); bf16 4020 x 33 x 6985 47 (16) / 46 (16), 16384 x 64 x 2048 21 (2) / 18, 64 x 64 x
// 65536 17 (64) / 14 (64), 64 x 16384 x 4096 29 (2) / 29 (2).
Plan plan_of(long M, long N, long K, long e)
{
    Plan p{};
    p.steps = (int)(k_padded(K, e) * e / 128);
    double best = 0.0;
    for (Shape shape : {SMALL, LARGE, NARROW_N, NARROW_M}) {
        if ((shape == NARROW_N && N > 64) || (shape == NARROW_M && M > 64)) continue;
        const long bm = shape == LARGE ? 256 : shape == NARROW_M ? 64 : 128, bn = shape == LARGE ? 256 : shape == NARROW_N ? 64 : 128;
        const long tm = (M + bm - 1) / bm, tn = (N + bn - 1) / bn;
        const double fixed = shape == LARGE ? 19.0 : 10.0;
        const double one = shape == LARGE ? (e == 2 ? 1.4 : 4.6) : shape == SMALL ? (e == 2 ? 0.5 : 1.43) : (e == 2 ? 0.4 : 0.88);
        const double two = shape == SMALL ? (e == 2 ? 0.9 : 2.6) : (e == 2 ? 0.6 : 1.25);
        for (int splits : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 24, 32, 48, 64, 96, 128, 192, 256}) {
            if (splits > 1 && (p.steps < 4 * splits || (double)splits * M * N > 2.5e8)) break;
            const int per = (p.steps + splits - 1) / splits;
            const long rounds = (tm * tn * splits + 255) / 256;
            double us = shape == LARGE ? rounds * (fixed + one * per) : rounds / 2 * (fixed + two * per) + rounds % 2 * (fixed + one * per);
            if (splits > 1) us += 3.0 + (double)splits * M * N * 8.0 / 4.5e6;
            if (best != 0.0 && us >= best) continue;
            best = us;
            p.shape = shape;
            p.tiles_m = (int)tm;
            p.tiles_n = (int)tn;
            p.per_split = per;
            p.splits = (p.steps + per - 1) / per;
        }
    }
    return p;
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }
size_t partial_bytes(const Plan &p, long M, long N) { return p.splits > 1 ? round256((size_t)p.splits * M * N * 4) : 0; }

// The loads take 16 bytes from any multiple of 4, so f32 operands are read as they lie, and 16-bit ones whose rows are an
// even number of elements apart (and, along a row, hold an even number of k); the others are copied to padded rows first.
bool in_place_along_k(const void *p, long ld, long e) { return ppo_aligned(p, 4) && (e == 4 || ld % 2 == 0); }
bool in_place(const void *p, long ld, long K, long e) { return in_place_along_k(p, ld, e) && (e == 4 || K % 2 == 0); }

// collects what a call has to prepare, for one launch
template <class T> struct Prep {
    PrepJobs jobs{};
    int count = 0;
    long tiles = 0;

    void add(const void *src, long ld, const void *mul, long R, long C, void *rows, float *sums)
    {
        PrepArgs a{src, mul, rows, sums, R, C, ld, k_padded(C, T::BYTES), 0};
        const long gr = (R + 63) / 64, gc = ((rows ? a.Cp : C) + 63) / 64;   // what lies past a row's end becomes zero
        a.tiles_x = (int)gc;
        jobs.job[count] = a;
        tiles += gr * gc;
        jobs.first[++count] = (unsigned)tiles;
    }

    int launch(hipStream_t s)
    {
        if (count == 0) return 0;
        PPO_REQUIRE(tiles < (1L << 24));     // fewer than 2^32 threads a launch
        for (int j = count; j < 3; ++j) jobs.first[j + 1] = (unsigned)tiles;
        hipLaunchKernelGGL(k_prep<T>, dim3((unsigned)tiles), dim3(256), 0, s, jobs);
        return ppo_launch_status();
    }
};

template <class T, bool KA, bool KB> int gemm(GemmArgs g, long K, const Plan &p, hipStream_t s)
{
    g.K = K;
    g.steps = p.steps;
    g.steps_per_split = p.per_split;
    g.tiles_m = p.tiles_m;
    g.tiles_n = p.tiles_n;
    if (p.splits == 1) g.partial = nullptr;
    const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), (unsigned)p.splits);
    switch (p.shape) {
    case LARGE: hipLaunchKernelGGL((k_gemm<T, 256, 256, 2, 4, KA, KB>), grid, dim3(512), 0, s, g); break;
    case SMALL: hipLaunchKernelGGL((k_gemm<T, 128, 128, 2, 2, KA, KB>), grid, dim3(256), 0, s, g); break;
    case NARROW_N: hipLaunchKernelGGL((k_gemm<T, 128, 64, 4, 1, KA, KB>), grid, dim3(256), 0, s, g); break;
    case NARROW_M: hipLaunchKernelGGL((k_gemm<T, 64, 128, 2, 2, KA, KB>), grid, dim3(256), 0, s, g); break;
    }
    int rc = ppo_launch_status();
    if (rc || p.splits == 1) return rc;
    constexpr long E = 16 / T::BYTES;
    const long threads = g.M * ((g.N + E - 1) / E);
    if (p.splits >= 16)
        hipLaunchKernelGGL((k_join<T, 8>), dim3((unsigned)((threads + 31) / 32)), dim3(256), 0, s, g, p.splits);
    else
        hipLaunchKernelGGL((k_join<T, 1>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, g, p.splits);
    return ppo_launch_status();
}

bool sizes_ok(long rows, long inputs, long outputs, int dtype)
{
    // 32-bit workgroup counts and offsets inside a tile; rows are also the k of the weight gradient
    return dtype_known(dtype) && rows >= 1 && inputs >= 1 && outputs >= 1 && rows <= MOST_K && inputs <= MOST_K && outputs <= MOST_K &&
           (__int128)rows * outputs < ((__int128)1 << 38) && (__int128)rows * inputs < ((__int128)1 << 38) &&
           (__int128)inputs * outputs < ((__int128)1 << 38);
}

bool matrix_ok(const void *p, long ld, long cols, long e) { return p && ppo_aligned(p, e) && ld >= cols && ld <= MOST_K; }

}  // namespace

extern "C" {

size_t ppo_linear_act_fwd_workspace_bytes(long rows, long inputs, long outputs, int dtype)
{
    const long e = dtype_bytes(dtype), Kp = k_padded(inputs, e);
    if (!sizes_ok(rows, inputs, outputs, dtype) || few_rows(rows, outputs, inputs, e, true)) return 0;
    const size_t copies = e == 2 ? round256((size_t)rows * Kp * e) + round256((size_t)outputs * Kp * e) : 0;   // f32 is read as it lies
    return copies + partial_bytes(plan_of(rows, outputs, inputs, e), rows, outputs);
}

int ppo_linear_act_fwd(const void *x, long x_stride, const void *weight, long weight_stride, const void *bias, const void *residual,
                       long residual_stride, int dtype, long rows, long inputs, long outputs, int activation, void *y, void *deriv,
                       void *workspace, size_t workspace_bytes, void *stream)
{
    if (rows == 0) return 0;
    PPO_REQUIRE(sizes_ok(rows, inputs, outputs, dtype));
    const long e = dtype_bytes(dtype);
    PPO_REQUIRE(matrix_ok(x, x_stride, inputs, e) && matrix_ok(weight, weight_stride, inputs, e));
    PPO_REQUIRE(!residual || matrix_ok(residual, residual_stride, outputs, e));
    PPO_REQUIRE(y && ppo_aligned(y, e) && ppo_aligned(deriv, dtype == PPO_DTYPE_BF16 ? 2 : 4) && ppo_aligned(bias, e) && activation >= PPO_ACT_NONE && activation <= PPO_ACT_SILU);
    const bool w_in_place = in_place(weight, weight_stride, inputs, e), few = few_rows(rows, outputs, inputs, e, w_in_place);
    const size_t need = ppo_linear_act_fwd_workspace_bytes(rows, inputs, outputs, dtype);
    PPO_REQUIRE(need == 0 || (workspace && ppo_aligned(workspace, 16) && workspace_bytes >= need));
    hipStream_t s = (hipStream_t)stream;
    return by_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        GemmArgs g{};
        g.A = x; g.B = weight; g.M = rows; g.N = outputs; g.lda = x_stride * e; g.ldb = weight_stride * e;
        g.bias = bias; g.residual = residual; g.res_ld = residual_stride; g.out = y; g.deriv = deriv; g.act = activation;
        if (few) {
            constexpr int COLS = 4;
            const dim3 grid((unsigned)((outputs + 4 * COLS - 1) / (4 * COLS)), (unsigned)((rows + 7) / 8));
            if (rows == 1)
                hipLaunchKernelGGL((k_few_rows<T, 1, COLS>), grid, dim3(256), 0, s, g, inputs);
            else if (rows <= 4)
                hipLaunchKernelGGL((k_few_rows<T, 4, COLS>), grid, dim3(256), 0, s, g, inputs);
            else
                hipLaunchKernelGGL((k_few_rows<T, 8, COLS>), grid, dim3(256), 0, s, g, inputs);
            return ppo_launch_status();
        }
        char *ws = reinterpret_cast<char *>(workspace);
        const long Kp = k_padded(inputs, e);
        Prep<T> prep;
        if (!in_place(x, x_stride, inputs, e)) {
            prep.add(x, x_stride, nullptr, rows, inputs, ws, nullptr);
            g.A = ws;
            g.lda = Kp * e;
        }
        if (e == 2) ws += round256((size_t)rows * Kp * e);
        if (!w_in_place) {
            prep.add(weight, weight_stride, nullptr, outputs, inputs, ws, nullptr);
            g.B = ws;
            g.ldb = Kp * e;
        }
        if (e == 2) ws += round256((size_t)outputs * Kp * e);
        const int rc = prep.launch(s);
        if (rc) return rc;
        g.partial = reinterpret_cast<float *>(ws);
        return gemm<T, false, false>(g, inputs, plan_of(rows, outputs, inputs, e), s);
    });
}

size_t ppo_linear_act_bwd_workspace_bytes(long rows, long inputs, long outputs, int dtype)
{
    if (!sizes_ok(rows, inputs, outputs, dtype)) return 0;
    const long e = dtype_bytes(dtype), Np = k_padded(outputs, e), Kp = k_padded(inputs, e);
    const size_t px = partial_bytes(plan_of(rows, inputs, outputs, e), rows, inputs), pw = partial_bytes(plan_of(outputs, inputs, rows, e), outputs, inputs);
    const size_t copies = e == 2 ? round256((size_t)outputs * Kp * e) + round256((size_t)rows * Kp * e) : 0;   // f32 is read as it lies
    return round256((size_t)rows * Np * e) + copies + round256((size_t)((rows + 63) / 64) * outputs * 4) + (px > pw ? px : pw);
}

int ppo_linear_act_bwd(const void *g_y, long g_stride, const void *x, long x_stride, const void *weight, long weight_stride,
                       const void *deriv, int dtype, long rows, long inputs, long outputs, void *g_x, void *g_weight, void *g_bias,
                       void *workspace, size_t workspace_bytes, void *stream)
{
    PPO_REQUIRE(sizes_ok(rows, inputs, outputs, dtype));
    const long e = dtype_bytes(dtype);
    PPO_REQUIRE(matrix_ok(g_y, g_stride, outputs, e) && matrix_ok(x, x_stride, inputs, e) && matrix_ok(weight, weight_stride, inputs, e));
    PPO_REQUIRE(ppo_aligned(deriv, dtype == PPO_DTYPE_BF16 ? 2 : 4) && ppo_aligned(g_x, e) && ppo_aligned(g_weight, e) && ppo_aligned(g_bias, e));
    PPO_REQUIRE(workspace && ppo_aligned(workspace, 16) && workspace_bytes >= ppo_linear_act_bwd_workspace_bytes(rows, inputs, outputs, dtype));
    if (!g_x && !g_weight && !g_bias) return 0;
    hipStream_t s = (hipStream_t)stream;
    return by_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const long Np = k_padded(outputs, e), Kp = k_padded(inputs, e);
        char *ws = reinterpret_cast<char *>(workspace);
        auto take = [&](size_t n) { char *p = ws; ws += round256(n); return p; };
        char *u = take((size_t)rows * Np * e), *wc = e == 2 ? take((size_t)outputs * Kp * e) : nullptr, *xc = e == 2 ? take((size_t)rows * Kp * e) : nullptr;
        float *sums = reinterpret_cast<float *>(take((size_t)((rows + 63) / 64) * outputs * 4));
        float *partial = reinterpret_cast<float *>(ws);
        GemmArgs gx{}, gw{};               // u W over the outputs, and u^T x over the rows: W, u and x are read along k as they lie
        gx.M = rows; gx.N = inputs; gx.out = g_x; gx.act = PPO_ACT_NONE; gx.partial = partial;
        gw.M = outputs; gw.N = inputs; gw.out = g_weight; gw.act = PPO_ACT_NONE; gw.partial = partial;
        const bool u_in_place = !deriv && in_place(g_y, g_stride, outputs, e), write_u = (g_x || g_weight) && !u_in_place;
        Prep<T> prep;
        if (write_u || g_bias) prep.add(g_y, g_stride, deriv, rows, outputs, write_u ? u : nullptr, g_bias ? sums : nullptr);
        gx.A = gw.A = u_in_place ? g_y : u;
        gx.lda = gw.lda = (u_in_place ? g_stride : Np) * e;
        gx.B = weight; gx.ldb = weight_stride * e;
        if (g_x && !in_place_along_k(weight, weight_stride, e)) {
            prep.add(weight, weight_stride, nullptr, outputs, inputs, wc, nullptr);
            gx.B = wc; gx.ldb = Kp * e;
        }
        gw.B = x; gw.ldb = x_stride * e;
        if (g_weight && !in_place_along_k(x, x_stride, e)) {
            prep.add(x, x_stride, nullptr, rows, inputs, xc, nullptr);
            gw.B = xc; gw.ldb = Kp * e;
        }
        int rc = prep.launch(s);
        if (!rc && g_bias) {
            hipLaunchKernelGGL(k_bias_grad<T>, dim3((unsigned)((outputs + 63) / 64)), dim3(1024), 0, s, sums, (rows + 63) / 64, outputs,
                               reinterpret_cast<typename T::raw *>(g_bias));
            rc = ppo_launch_status();
        }
        if (!rc && g_x) rc = gemm<T, false, true>(gx, outputs, plan_of(rows, inputs, outputs, e), s);
        if (!rc && g_weight) rc = gemm<T, true, true>(gw, rows, plan_of(outputs, inputs, rows, e), s);
        return rc;
    });
}

}  // extern "C"
