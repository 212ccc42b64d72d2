// experts_common.h -- device helpers shared by route_kernels.hip and adapt_kernels.hip.
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
