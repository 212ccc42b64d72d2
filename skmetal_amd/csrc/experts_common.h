// experts_common.h -- device helpers shared by the kernels of skmetal_amd.experts.
#pragma once

#include <tuple>
#include <type_traits>
#include <utility>

#include "experts.h"

namespace skm {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }
// Rounded to nearest, ties to even: the one rounding of a result to its type.
template <typename T> __device__ __forceinline__ T from_f(float v) { return (T)v; }

// exp(x) for x <= 0 by the hardware's base-2 exponential.  The product's rounding becomes a relative
// error of up to 2^-24 |x| in the result: 1e-6 at x = -17, where the result is 4e-8 of the row's
// largest and the error 4e-14 of it.  A product in two parts would cost further instructions a
// score, which is what bounds k_route.
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f); }

// ---- loads of 16 bytes of a row, the elements past `left` as 0 ----

template <typename T> constexpr int kVec = 16 / sizeof(T);
template <typename T> using Vec = T __attribute__((ext_vector_type(16 / sizeof(T))));

template <typename T>
__device__ __forceinline__ Vec<T> load16(const T* p)
{
    Vec<T> v;
    __builtin_memcpy(&v, p, 16);  // rows may start at any element
    return v;
}

// 16 bytes that the kernel's caller reads next, from memory: past the caches (a plain store
// would push rows that are still to be read out of them; expanding 8,192 x 4,096 takes 28 us so,
// 36 with plain stores).
template <typename T>
__device__ __forceinline__ void stream16(T* p, Vec<T> v)
{
    typedef unsigned Words __attribute__((ext_vector_type(4), aligned(2)));  // rows may start at any element
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), reinterpret_cast<Words*>(p));
}

template <typename T>
__device__ __forceinline__ Vec<T> load_part(const T* p, int left)
{
    if (left >= kVec<T>) return load16(p);
    Vec<T> v;
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j) v[j] = j < left ? p[j] : (T)0.f;
    return v;
}

// acc += a b^T over the 4 x kVec elements of k that the four lane groups hold (which k a
// lane's elements are makes no difference as long as a and b hold the same).
__device__ __forceinline__ f32x4 mfma16(Vec<bf16> a, Vec<bf16> b, f32x4 acc) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma16(Vec<f16> a, Vec<f16> b, f32x4 acc) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma16(Vec<float> a, Vec<float> b, f32x4 acc)
{
#pragma unroll
    for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], acc, 0, 0, 0);
    return acc;
}

// threadIdx.x / 64, which the compiler then knows to be the same on all lanes.
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// Launches `kernel` and returns that launch's own status (an error that other code left
// on the thread is not taken for it).
template <typename... P, typename... A>
inline hipError_t launch(void (*kernel)(P...), dim3 grid, unsigned block, size_t lds, hipStream_t s, A&&... args)
{
    std::tuple<P...> v{static_cast<P>(std::forward<A>(args))...};
    return std::apply(
        [&](auto&... p) {
            void* ptr[] = {const_cast<void*>(static_cast<const void*>(&p))...};
            return hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(block), ptr, lds, s);
        },
        v);
}
#define SKM_TRY_LAUNCH(...)                                 \
    do {                                                    \
        const hipError_t e_ = skm::launch(__VA_ARGS__);     \
        if (e_ != hipSuccess) return e_;                    \
    } while (0)

// The launcher's choice of element type: f(T{}) for the type of code `type`.
template <typename F>
inline hipError_t with_type(int type, F&& f)
{
    if (type == kBF16) return f(bf16{});
    if (type == kF16) return f(f16{});
    return f(0.f);
}

}  // namespace skm
