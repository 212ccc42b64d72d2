// route_kernels.hip -- the router: every row's k largest scores, their softmax weights,
// the experts' counts and the balance loss, and the gradient of the scores.
//
//   p_ij = exp(z_ij - max_j z_ij) / sum_j exp(...)           over the row's scores
//   e_i1 .. e_ik = the k largest scores, equal ones by the lowest index
//   w_it = p_i,e_it, or that divided by its sum over t       (normalize)
//   c_j = rows that take j,  S_j = sum_i p_ij,  N = rows that count
//   loss = E / (k N^2) sum_j c_j S_j
// A score of -inf or NaN is excluded: probability 0, never taken.  A row that is masked
// or has no score left takes no expert (-1, weight 0) and counts nowhere.
#include "experts_common.h"

namespace skm {
namespace {

// One wave per row, each lane the columns lane, lane + 64, ...; k passes over the row for
// the next largest (value, lowest index).
template <typename T>
__global__ __launch_bounds__(256) void k_route(RouteArgs a, int nb, float* psum, int* pcnt, int* prow)
{
    extern __shared__ char lds[];
    float* bs = reinterpret_cast<float*>(lds);       // [E] sums of this block's rows, wave by wave
    int* bc = reinterpret_cast<int*>(bs + a.E);      // [E]
    __shared__ int brow;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int j = threadIdx.x; j < a.E; j += 256) { bs[j] = 0.f; bc[j] = 0; }
    if (threadIdx.x == 0) brow = 0;
    __syncthreads();
    constexpr int V = kRouteMaxE / 64;
    float acc[V];
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = 0.f;
    int mine = 0;
    for (long i = (long)blockIdx.x * 4 + wave; i < a.n; i += (long)nb * 4) {
        const T* z = static_cast<const T*>(a.z) + i * a.ld;
        const bool on = a.mask == nullptr || a.mask[i * a.mask_stride] != 0;
        float x[V];
        float m = -INFINITY;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int j = v * 64 + lane;
            x[v] = on && j < a.E ? to_f(z[j]) : -INFINITY;
            if (x[v] != x[v]) x[v] = -INFINITY;
            m = fmaxf(m, x[v]);
        }
        for (int off = 1; off < 64; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
        const bool live = m > -INFINITY;
        float s = 0.f;
        float p[V];
#pragma unroll
        for (int v = 0; v < V; ++v) { p[v] = live && x[v] > -INFINITY ? __expf(x[v] - m) : 0.f; s += p[v]; }
        for (int off = 1; off < 64; off <<= 1) s += __shfl_xor(s, off, 64);
        const float inv = live ? 1.f / s : 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) { p[v] *= inv; acc[v] += p[v]; }
        mine += live;
        float total = 0.f, wt = 0.f;
        int et = -1;
        for (int t = 0; t < a.k; ++t) {
            float best = -INFINITY, pb = 0.f;
            int at = 0x7fffffff;
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (x[v] > best) { best = x[v]; at = v * 64 + lane; pb = p[v]; }
            for (int off = 1; off < 64; off <<= 1) {
                const float ob = __shfl_xor(best, off, 64), op = __shfl_xor(pb, off, 64);
                const int oa = __shfl_xor(at, off, 64);
                if (ob > best || (ob == best && oa < at)) { best = ob; at = oa; pb = op; }
            }
            if (!(best > -INFINITY)) break;
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v * 64 + lane == at) x[v] = -INFINITY;
            total += pb;
            if (lane == t) { wt = pb; et = at; }
        }
        if (lane < a.k) {
            a.w[i * a.k + lane] = a.normalize && et >= 0 ? wt / total : wt;
            a.ex[i * a.k + lane] = et;
            if (et >= 0) atomicAdd(&bc[et], 1);
        }
    }
    for (int w = 0; w < 4; ++w) {
        if (wave == w) {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v * 64 + lane < a.E) bs[v * 64 + lane] += acc[v];
            if (lane == 0) brow += mine;
        }
        __syncthreads();
    }
    for (int j = threadIdx.x; j < a.E; j += 256) {
        psum[(long)blockIdx.x * a.E + j] = bs[j];
        pcnt[(long)blockIdx.x * a.E + j] = bc[j];
    }
    if (threadIdx.x == 0) prow[blockIdx.x] = brow;
}

// The blocks' sums and counts added in block order, and the loss.
__global__ __launch_bounds__(256) void k_route_total(RouteArgs a, int nb, const float* psum, const int* pcnt, const int* prow)
{
    __shared__ double part[256];
    double dot = 0.0;
    for (int j = threadIdx.x; j < a.E; j += 256) {
        double s = 0.0;
        int c = 0;
        for (int b = 0; b < nb; ++b) { s += psum[(long)b * a.E + j]; c += pcnt[(long)b * a.E + j]; }
        a.sums[j] = (float)s;
        a.counts[j] = c;
        dot += s * c;
    }
    part[threadIdx.x] = dot;
    __syncthreads();
    if (threadIdx.x == 0) {
        int rows = 0;
        for (int b = 0; b < nb; ++b) rows += prow[b];
        double t = 0.0;
        for (int i = 0; i < 256; ++i) t += part[i];
        a.rows[0] = rows;
        a.loss[0] = rows > 0 ? (float)(t * a.E / ((double)a.k * rows * rows)) : 0.f;
    }
}

// dz_ij = p_ij (G_j - sum_j p_ij G_j) + the chosen ones' gate part.
template <typename T>
__global__ __launch_bounds__(256) void k_route_back(RouteBackArgs a, int nb)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    constexpr int V = kRouteMaxE / 64;
    const int N = a.rows[0];
    const float each = a.dloss != nullptr && N > 0 ? (float)((double)a.dloss[0] * a.E / ((double)a.k * N * N)) : 0.f;
    for (long i = (long)blockIdx.x * 4 + wave; i < a.n; i += (long)nb * 4) {
        const T* z = static_cast<const T*>(a.z) + i * a.ld;
        T* dz = static_cast<T*>(a.dz) + i * a.ld_dz;
        const bool on = a.mask == nullptr || a.mask[i * a.mask_stride] != 0;
        float x[V], m = -INFINITY;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int j = v * 64 + lane;
            x[v] = on && j < a.E ? to_f(z[j]) : -INFINITY;
            if (x[v] != x[v]) x[v] = -INFINITY;
            m = fmaxf(m, x[v]);
        }
        for (int off = 1; off < 64; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
        const bool live = m > -INFINITY;
        float s = 0.f, g = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int j = v * 64 + lane;
            x[v] = live && x[v] > -INFINITY ? __expf(x[v] - m) : 0.f;
            s += x[v];
            g += x[v] * (j < a.E ? each * a.counts[j] : 0.f);
        }
        for (int off = 1; off < 64; off <<= 1) { s += __shfl_xor(s, off, 64); g += __shfl_xor(g, off, 64); }
        const float inv = live ? 1.f / s : 0.f;
        g *= inv;
        float wd = 0.f;
        if (a.dw != nullptr)
            for (int t = 0; t < a.k; ++t)
                if (a.ex[i * a.k + t] >= 0) wd += a.w[i * a.k + t] * a.dw[i * a.k + t];
        if (!a.normalize) g += wd;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int j = v * 64 + lane;
            if (j >= a.E) continue;
            float r = x[v] * inv * (each * a.counts[j] - g);
            if (a.dw != nullptr)
                for (int t = 0; t < a.k; ++t)
                    if (a.ex[i * a.k + t] == j) r += a.w[i * a.k + t] * (a.dw[i * a.k + t] - (a.normalize ? wd : 0.f));
            dz[j] = from_f<T>(r);
        }
    }
}

int route_blocks(long n) { return (int)(n < 4 * 512 ? (n + 3) / 4 > 0 ? (n + 3) / 4 : 1 : 512); }

}  // namespace

size_t route_workspace(long n, int E) { return (size_t)route_blocks(n) * (8 * (size_t)E + 4); }

hipError_t launch_route(const RouteArgs& a, hipStream_t s)
{
    const int nb = route_blocks(a.n);
    float* psum = reinterpret_cast<float*>(a.ws);
    int* pcnt = reinterpret_cast<int*>(psum + (size_t)nb * a.E);
    int* prow = pcnt + (size_t)nb * a.E;
    return with_type(a.type, [&](auto t) {
        SKM_TRY_LAUNCH(k_route<decltype(t)>, nb, 256, 8 * (size_t)a.E, s, a, nb, psum, pcnt, prow);
        return launch(k_route_total, 1, 256, 0, s, a, nb, psum, pcnt, prow);
    });
}

hipError_t launch_route_back(const RouteBackArgs& a, hipStream_t s)
{
    if (a.n == 0) return hipSuccess;
    const int nb = (int)((a.n + 3) / 4 < 4096 ? (a.n + 3) / 4 : 4096);
    return with_type(a.type, [&](auto t) {
        return launch(k_route_back<decltype(t)>, nb, 256, 0, s, a, nb);
    });
}

}  // namespace skm
