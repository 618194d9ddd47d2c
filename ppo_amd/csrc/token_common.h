// Element types, vector access and reductions shared by the token-policy kernels (logprob.hip, seqloss.hip, linear.hip).
#pragma once
#include "common.h"

namespace ppo_token {

struct F32 {
    using raw = float;
    static constexpr int BYTES = 4;
    static __device__ __forceinline__ float load(raw v) { return v; }
    static __device__ __forceinline__ raw store(float v) { return v; }
};
struct BF16 {
    using raw = uint16_t;
    static constexpr int BYTES = 2;
    static __device__ __forceinline__ float load(raw v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }
    static __device__ __forceinline__ raw store(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }   // to nearest even
};
struct F16 {
    using raw = uint16_t;
    static constexpr int BYTES = 2;
    static __device__ __forceinline__ float load(raw v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ __forceinline__ raw store(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};

// 16 bytes at any address that suits the element: global_load / store_dwordx4 need no more than that (a wave's 1 KB
// then touches one more cache line)
template <class T> struct __attribute__((packed, aligned(T::BYTES))) Vec16 {
    uint32_t w[4];
};

// the N = 16 / BYTES elements behind p as floats
template <class T> __device__ __forceinline__ void load16(const typename T::raw *p, float (&out)[16 / T::BYTES])
{
    const Vec16<T> v = *reinterpret_cast<const Vec16<T> *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (T::BYTES == 4) {
            out[i] = __builtin_bit_cast(float, v.w[i]);
        } else {
            out[2 * i] = T::load((uint16_t)v.w[i]);
            out[2 * i + 1] = T::load((uint16_t)(v.w[i] >> 16));
        }
    }
}

template <class T> __device__ __forceinline__ void store16(typename T::raw *p, const float (&in)[16 / T::BYTES])
{
    Vec16<T> v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (T::BYTES == 4)
            v.w[i] = __builtin_bit_cast(uint32_t, in[i]);
        else
            v.w[i] = (uint32_t)T::store(in[2 * i]) | ((uint32_t)T::store(in[2 * i + 1]) << 16);
    }
    *reinterpret_cast<Vec16<T> *>(p) = v;
}

template <class F> static inline int by_dtype(int dtype, F f)
{
    switch (dtype) {
    case PPO_DTYPE_F32: return f(F32{});
    case PPO_DTYPE_BF16: return f(BF16{});
    case PPO_DTYPE_F16: return f(F16{});
    }
    return (int)hipErrorInvalidValue;
}

static inline long dtype_bytes(int dtype) { return dtype == PPO_DTYPE_F32 ? 4 : 2; }
static inline bool dtype_known(int dtype) { return dtype == PPO_DTYPE_F32 || dtype == PPO_DTYPE_BF16 || dtype == PPO_DTYPE_F16; }

}  // namespace ppo_token
