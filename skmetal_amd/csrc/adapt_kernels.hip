// adapt_kernels.hip -- low-rank adapters of many requests beside a shared projection.
//
// Row i has the adapter q = ids[i], or none when that lies outside [0, a).  With down
// D_q [r x d], up U_q [r x o] (both by rank, so that every product below reads them along
// their rows), gate g_i and scale s_q:
//   t_i = D_q x_i                     f_i = g_i s_q
//   out_i = base_i + f_i U_q^T t_i
// and, from dy_i = the gradient of out_i,
//   u_i = U_q dy_i                    dg_i = s_q <u_i, t_i>
//   dx_i = base_i + f_i D_q^T u_i
//   dD_q = sum_i f_i u_i x_i^T        dU_q = sum_i f_i t_i dy_i^T
#include "experts_common.h"

namespace skm {
namespace {

__device__ __forceinline__ int adapter_of(const int* ids, long stride, long i, int a)
{
    const int q = ids[i * stride];
    return q >= 0 && q < a ? q : -1;
}

// low[i] = M_q v_i; a block per row, a wave per rank.
template <typename T>
__global__ __launch_bounds__(256) void k_low(const T* v, long ld_v, const T* M, long sa, long ld, const int* ids, long ids_stride, int a, int w, int r, float* low)
{
    const long i = blockIdx.x;
    const int q = adapter_of(ids, ids_stride, i, a);
    for (int t = threadIdx.x >> 6; t < r; t += 4) {
        float s = 0.f;
        if (q >= 0)
            for (int j = threadIdx.x & 63; j < w; j += 64) s += to_f(v[i * ld_v + j]) * to_f(M[q * sa + t * ld + j]);
        for (int off = 1; off < 64; off <<= 1) s += __shfl_xor(s, off, 64);
        if ((threadIdx.x & 63) == 0) low[i * r + t] = s;
    }
}

// out[i] = base[i] + f_i M_q^T low[i]; a block per row.
template <typename T>
__global__ __launch_bounds__(256) void k_high(const float* low, const T* M, long sa, long ld, const int* ids, long ids_stride, const float* gates,
                                              long gates_stride, const float* scales, const T* base, long ld_base, T* out, long ld_out, int a, int w, int r)
{
    const long i = blockIdx.x;
    const int q = adapter_of(ids, ids_stride, i, a);
    const float f = q < 0 ? 0.f : (gates ? gates[i * gates_stride] : 1.f) * (scales ? scales[q] : 1.f);
    for (int j = threadIdx.x; j < w; j += 256) {
        float s = 0.f;
        if (q >= 0)
            for (int t = 0; t < r; ++t) s += low[i * r + t] * to_f(M[q * sa + t * ld + j]);
        out[i * ld_out + j] = from_f<T>((base ? to_f(base[i * ld_base + j]) : 0.f) + f * s);
    }
}

// dM_q[t][j] = sum over q's rows of f_i low[i][t] v_i[j]; a block per 256 columns of one (q, t).
template <typename T>
__global__ __launch_bounds__(256) void k_outer(const float* low, const T* v, long ld_v, const int* ids, long ids_stride, const float* gates, long gates_stride,
                                               const float* scales, T* dM, long n, int a, int w, int r)
{
    const int q = blockIdx.z, t = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
    const float sc = scales ? scales[q] : 1.f;
    float s = 0.f;
    for (long i = 0; i < n; ++i)
        if (ids[i * ids_stride] == q && j < w) s += (gates ? gates[i * gates_stride] : 1.f) * sc * low[i * r + t] * to_f(v[i * ld_v + j]);
    if (j < w) dM[((long)q * r + t) * w + j] = from_f<T>(s);
}

// dg_i = s_q <u_i, t_i>
__global__ __launch_bounds__(256) void k_gate(const float* u, const float* t, const int* ids, long ids_stride, const float* scales, float* dg, long n, int a, int r)
{
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int q = adapter_of(ids, ids_stride, i, a);
    float s = 0.f;
    for (int k = 0; k < r; ++k) s += u[i * r + k] * t[i * r + k];
    dg[i] = q < 0 ? 0.f : s * (scales ? scales[q] : 1.f);
}

}  // namespace

// Forward: the low-rank rows where the caller does not want them; backward: u.
size_t adapt_workspace(int, long n, int, int, int r, int, int) { return (size_t)n * r * 4; }

hipError_t launch_adapt(const AdaptArgs& a, hipStream_t s)
{
    if (a.n == 0) return hipSuccess;
    float* low = a.low != nullptr ? a.low : reinterpret_cast<float*>(a.ws);
    return with_type(a.type, [&](auto tag) {
        using T = decltype(tag);
        SKM_TRY_LAUNCH(k_low<T>, dim3((unsigned)a.n), 256, 0, s, (const T*)a.x, a.ld_x, (const T*)a.down, a.down_sa, a.down_ld, a.ids, a.ids_stride, a.a, a.d, a.r, low);
        SKM_TRY_LAUNCH(k_high<T>, dim3((unsigned)a.n), 256, 0, s, low, (const T*)a.up, a.up_sa, a.up_ld, a.ids, a.ids_stride, a.gates, a.gates_stride, a.scales,
                                                (const T*)a.base, a.ld_base, (T*)a.out, a.ld_out, a.a, a.o, a.r);
        return hipSuccess;
    });
}

hipError_t launch_adapt_back(const AdaptBackArgs& a, hipStream_t s)
{
    float* u = reinterpret_cast<float*>(a.ws);
    return with_type(a.type, [&](auto tag) {
        using T = decltype(tag);
        if (a.n > 0) {
            SKM_TRY_LAUNCH(k_low<T>, dim3((unsigned)a.n), 256, 0, s, (const T*)a.dy, a.ld_dy, (const T*)a.up, a.up_sa, a.up_ld, a.ids, a.ids_stride, a.a, a.o, a.r, u);
            SKM_TRY_LAUNCH(k_high<T>, dim3((unsigned)a.n), 256, 0, s, u, (const T*)a.down, a.down_sa, a.down_ld, a.ids, a.ids_stride, a.gates, a.gates_stride, a.scales,
                                                    (const T*)a.base, a.ld_base, (T*)a.dx, a.ld_dx, a.a, a.d, a.r);
            if (a.dgates != nullptr)
                SKM_TRY_LAUNCH(k_gate, (unsigned)((a.n + 255) / 256), 256, 0, s, u, a.low, a.ids, a.ids_stride, a.scales, a.dgates, a.n, a.a, a.r);
        }
        if (a.a > 0) {
            SKM_TRY_LAUNCH(k_outer<T>, dim3((a.d + 255) / 256, a.r, a.a), 256, 0, s, u, (const T*)a.x, a.ld_x, a.ids, a.ids_stride, a.gates, a.gates_stride, a.scales,
                                                                         (T*)a.ddown, a.n, a.a, a.d, a.r);
            SKM_TRY_LAUNCH(k_outer<T>, dim3((a.o + 255) / 256, a.r, a.a), 256, 0, s, a.low, (const T*)a.dy, a.ld_dy, a.ids, a.ids_stride, a.gates, a.gates_stride, a.scales,
                                                                         (T*)a.dup, a.n, a.a, a.o, a.r);
        }
        return hipSuccess;
    });
}

}  // namespace skm
