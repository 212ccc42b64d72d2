// route_kernels.hip -- the router: every row's k largest scores, their softmax weights,
// the experts' counts and the balance loss, and the gradient of the scores.
//
//   p_ij = exp(z_ij - max_j z_ij) / sum_j exp(...)           over the row's scores
//   e_i1 .. e_ik = the k largest scores, equal ones by the lowest index
//   w_it = p_i,e_it, or that divided by its sum over t       (normalize)
//   c_j = rows that take j,  S_j = sum_i p_ij,  N = rows that count
//   loss = E / (k N^2) sum_j c_j S_j
// A score of -inf or NaN is excluded: probability 0, never taken.  A row that is masked
// or has no score left takes no expert (-1, weight 0) and counts nowhere.  +inf is a score:
// the largest, and its row's probabilities are NaN, as inf - inf is.
//
// One pass over the scores each way.  A row lies on L lanes (1, 8, 16 or 64), NC times eight columns a
// lane (column = (c L + lane) 8 + e), so a wave takes 64 / L rows at once and a row's sums
// and its choice need log2(L) exchanges.
#include "experts_common.h"

namespace skm {
namespace {

constexpr int kThreads = 256;
constexpr int kOneThreads = 1024;
constexpr int kMaxBlocks = 768;  // three a CU at once: what the registers of the widest rows allow
constexpr int kOneBlock = kOneThreads / 64;  // groups of 64 / L rows that one block takes at once: no second launch then

// A score as a whole number whose order is that of (score, lowest index first).  The value is
// ordered as its fp32 bits; those of a 16-bit type leave the low 16 (bf16) or 13 bits (fp16) to
// the index, and fp32 scores take 64.  -0 counts as 0; -inf and NaN, the excluded ones, lie
// under every other score's key.
template <typename T>
struct Order {
    using Key = unsigned;
    static constexpr unsigned kIndex = sizeof(T) == 2 && std::is_same_v<T, f16> ? 0x1fff : 0xffff;
    static __device__ __forceinline__ Key of(unsigned ordered, int j) { return (ordered & ~kIndex) | (kIndex - j); }
    static __device__ __forceinline__ unsigned ordered(Key k) { return k & ~kIndex; }
    static __device__ __forceinline__ int index(Key k) { return kIndex - (k & kIndex); }
};
template <>
struct Order<float> {
    using Key = unsigned long long;
    static __device__ __forceinline__ Key of(unsigned ordered, int j) { return (Key)ordered << 32 | (0xffffffffu - (unsigned)j); }
    static __device__ __forceinline__ unsigned ordered(Key k) { return (unsigned)(k >> 32); }
    static __device__ __forceinline__ int index(Key k) { return (int)(0xffffffffu - (unsigned)k); }
};
static_assert(kRouteMaxE <= 0x2000, "the index of an fp16 score has 13 bits");

template <typename T>
__device__ __forceinline__ bool takable(typename Order<T>::Key k) { return Order<T>::ordered(k) >= 0x00800000u; }

template <typename T>
__device__ __forceinline__ float value_of(typename Order<T>::Key k)
{
    const unsigned o = Order<T>::ordered(k), mask = std::is_same_v<T, float> ? 0xffffffffu : ~(std::is_same_v<T, f16> ? 0x1fffu : 0xffffu);
    return __uint_as_float((o & 0x80000000u ? o ^ 0x80000000u : ~o) & mask);
}

// Eight scores of a row: their values (-inf where excluded) and keys from column j on.
template <typename T>
__device__ __forceinline__ void decode8(const T* raw, int j, float* x, typename Order<T>::Key* key)
{
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = fmaxf(to_f(raw[e]) + 0.f, -INFINITY);  // -0 becomes 0, NaN -inf
        const int u = __float_as_int(x[e]);
        key[e] = Order<T>::of((unsigned)(u ^ ((u >> 31) | (int)0x80000000)), j + e);
    }
}

template <typename K>
__device__ __forceinline__ void order(K& hi, K& lo)  // the larger to hi
{
    const K a = hi > lo ? hi : lo, b = hi > lo ? lo : hi;
    hi = a;
    lo = b;
}

// a[0 .. N) falls and then rises (or the other way round): in falling order.
template <int N, typename K>
__device__ __forceinline__ void merge_bitonic(K* a)
{
#pragma unroll
    for (int half = N / 2; half >= 1; half /= 2)
#pragma unroll
        for (int i = 0; i < N; ++i)
            if ((i & half) == 0) order(a[i], a[i + half]);
}

// a[0 .. N) in falling order.
template <int N, typename K>
__device__ __forceinline__ void sort_falling(K* a)
{
#pragma unroll
    for (int size = 2; size <= N; size *= 2)
#pragma unroll
        for (int half = size / 2; half >= 1; half /= 2)
#pragma unroll
            for (int i = 0; i < N; ++i)
                if ((i & half) == 0) {
                    if ((i & size) == 0) order(a[i], a[i + half]); else order(a[i + half], a[i]);
                }
}

// top, in falling order, takes in b, in falling order: of the two lists' N largest, one is
// in each pair of top's i-th and b's i-th from the end.
template <int N, typename K>
__device__ __forceinline__ void merge_top(K* top, const K* b)
{
#pragma unroll
    for (int i = 0; i < N; ++i) top[i] = top[i] > b[N - 1 - i] ? top[i] : b[N - 1 - i];
    merge_bitonic<N>(top);
}

// The value of the lane `off` away (xor), within a butterfly that takes off = 1, 2, 4, ... or starts
// at 8: at 4 the four lanes of a quad hold one value, so the lane opposite within eight
// (7 - lane) serves as well.
__device__ __forceinline__ unsigned across_bits(unsigned v, int off)
{
    switch (off) {
    case 1: return __builtin_amdgcn_update_dpp(0, v, 0xb1, 0xf, 0xf, true);    // quad_perm [1, 0, 3, 2]
    case 2: return __builtin_amdgcn_update_dpp(0, v, 0x4e, 0xf, 0xf, true);    // quad_perm [2, 3, 0, 1]
    case 4: return __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true);   // row_half_mirror
    case 8: return __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, true);   // row_ror:8
    case 16: return __builtin_amdgcn_ds_swizzle(v, 0x401f);                    // xor 16
    default: return __shfl_xor(v, off, 64);
    }
}
__device__ __forceinline__ unsigned across(unsigned v, int off) { return across_bits(v, off); }
__device__ __forceinline__ int across(int v, int off) { return (int)across_bits((unsigned)v, off); }
__device__ __forceinline__ float across(float v, int off) { return __uint_as_float(across_bits(__float_as_uint(v), off)); }
__device__ __forceinline__ unsigned long long across(unsigned long long v, int off)
{
    return (unsigned long long)across_bits((unsigned)(v >> 32), off) << 32 | across_bits((unsigned)v, off);
}

// Sum over a row's lanes, on all of them.
template <int L>
__device__ __forceinline__ float row_sum(float v)
{
#pragma unroll
    for (int off = 1; off < L; off <<= 1) v += across(v, off);
    return v;
}

template <typename T, int L, int NC>
__device__ __forceinline__ void load_row(const void* z, long ld, const uint8_t* mask, long mask_stride, long n, int E, long row, T (*raw)[8], bool& on)
{
    const int j = (threadIdx.x & (L - 1)) * 8;
    on = row < n;
    const long r = on ? row : n - 1;
    const T* p = static_cast<const T*>(z) + r * ld + j;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int col = c * L * 8;
        if (col + L * 8 <= E) {
            __builtin_memcpy(raw[c], p + col, 8 * sizeof(T));
        } else if (col + j + 8 <= E) {
            __builtin_memcpy(raw[c], p + col, 8 * sizeof(T));
        } else if (col < E) {  // the columns past the row as NaN (excluded)
#pragma unroll
            for (int e = 0; e < 8; ++e) raw[c][e] = col + j + e < E ? p[col + e] : (T)__builtin_nanf("");
        }
    }
    if (mask != nullptr) on = on && mask[r * mask_stride] != 0;
}

// The blocks' sums and counts (or the only block's) become the results.
__device__ __forceinline__ float balance_loss(double dot, int E, int k, int rows) { return rows > 0 ? (float)(dot * E / ((double)k * rows * rows)) : 0.f; }

// The choice: every lane sorts its scores eight (or k) at a time by a bitonic network and merges
// the lists, keeping the k largest; the row's lanes then merge theirs log2(L) times.  The
// largest is the softmax's maximum, so the scores are decoded once, and their values stay in
// registers for the exponentials and the column sums, which a wave keeps over all its rows.
// At 131,072 x 256 bf16, k = 8, 40 us (67 MB: 13 us to read): some 900 vector instructions for
// a wave's 8 rows bound it, about 400 of them the choice's.  ONE: a single block, a wave a
// group of rows; 96 x 256, k = 8 takes 12 us on one CU, of which its 12 waves' instructions
// are some 4.5 by their count; the launch and each instruction's first fetch are among the rest.
template <typename T, int L, int NC, int KP, bool ONE>
__global__ __launch_bounds__(ONE ? kOneThreads : kThreads) void k_route(RouteArgs a, int nb, float* psum, int* pcnt, int* prow, unsigned* ticket)
{
    using O = Order<T>;
    using Key = typename O::Key;
    constexpr int NT = ONE ? kOneThreads : kThreads, RW = 64 / L, W = NT / 64, SPAN = L * 8 * NC;
    __shared__ float sums[W][SPAN];
    __shared__ int counts[SPAN];
    __shared__ int rows[W];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & (L - 1);
    for (int i = threadIdx.x; i < SPAN; i += NT) counts[i] = 0;
    if (!ONE && blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
    __syncthreads();
    float acc[NC][8];  // a wave without rows adds zeros
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[c][e] = 0.f;
    int mine = 0;
    const long groups = (a.n + RW - 1) / RW;
    T next[NC][8];
    bool next_on = false;
    long grp = (long)blockIdx.x * W + wave;
    if (grp < groups) load_row<T, L, NC>(a.z, a.ld, a.mask, a.mask_stride, a.n, a.E, grp * RW + lane / L, next, next_on);
    for (; grp < groups; grp += ONE ? groups : (long)nb * W) {
        const long row = grp * RW + lane / L;
        T raw[NC][8];
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) raw[c][e] = next[c][e];
        const bool on = next_on;
        const long after = grp + (long)nb * W;
        if (!ONE && after < groups) load_row<T, L, NC>(a.z, a.ld, a.mask, a.mask_stride, a.n, a.E, after * RW + lane / L, next, next_on);

        float x[NC][8];
        Key top[KP];
#pragma unroll
        for (int t = 0; t < KP; ++t) top[t] = 0;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (c * L * 8 >= a.E) break;
            Key key[8];
            decode8<T>(raw[c], (c * L + j) * 8, x[c], key);
            if constexpr (KP >= 8) {
                // the eight in falling order, and as many zeros
                Key some[KP];
#pragma unroll
                for (int t = 0; t < KP; ++t) some[t] = t < 8 ? key[t] : 0;
                sort_falling<8>(some);
                if (c == 0)
#pragma unroll
                    for (int t = 0; t < KP; ++t) top[t] = some[t];
                else
                    merge_top<KP>(top, some);
            } else {
                // KP at a time; for one or two this is a plain insertion
#pragma unroll
                for (int b = 0; b < 8; b += KP) {
                    sort_falling<KP>(key + b);
                    if (c == 0 && b == 0)
#pragma unroll
                        for (int t = 0; t < KP; ++t) top[t] = key[t];
                    else
                        merge_top<KP>(top, key + b);
                }
            }
        }
#pragma unroll
        for (int off = 1; off < L; off <<= 1) {
            Key other[KP];
#pragma unroll
            for (int t = 0; t < KP; ++t) other[t] = across(top[t], off);
            merge_top<KP>(top, other);
        }
        const bool live = on && takable<T>(top[0]);
        const float m = value_of<T>(top[0]);
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (c * L * 8 >= a.E) break;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[c][e] = live ? exp_of(x[c][e] - m) : 0.f;
                s += x[c][e];
            }
        }
        s = row_sum<L>(s);
        const float inv = live ? 1.f / s : 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (c * L * 8 >= a.E) break;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[c][e] += x[c][e] * inv;
        }
        mine += live && j == 0;

        // slots j, j + L, ... of the row on this lane
        constexpr int SL = (KP + L - 1) / L;
        float w[SL];
        int ex[SL];
        float total = 0.f;
#pragma unroll
        for (int i = 0; i < SL; ++i) {
            Key key = 0;
#pragma unroll
            for (int t = 0; t < KP; ++t)
                if (t % L == j && t / L == i) key = top[t];
            const bool taken = live && takable<T>(key) && i * L + j < a.k;
            w[i] = taken ? exp_of(value_of<T>(key) - m) : 0.f;
            ex[i] = taken ? O::index(key) : -1;
            total += w[i];
        }
        const float scale = a.normalize ? (live ? 1.f / row_sum<L>(total) : 0.f) : inv;
        if (row < a.n)
#pragma unroll
            for (int i = 0; i < SL; ++i) {
                const int t = i * L + j;
                if (t >= a.k) continue;
                a.w[row * a.k + t] = ex[i] >= 0 ? w[i] * scale : 0.f;  // 0 beside a score of +inf too, whose row's scale is NaN
                a.ex[row * a.k + t] = ex[i];
                if (ex[i] >= 0) atomicAdd(&counts[ex[i]], 1);
            }
    }
    // the wave's rows' sums, then the waves', in order
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        if (c * L * 8 >= a.E) break;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
#pragma unroll
            for (int off = L; off < 64; off <<= 1) acc[c][e] += across(acc[c][e], off);
            if (lane < L) sums[wave][(c * L + j) * 8 + e] = acc[c][e];
        }
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) mine += across(mine, off);
    if (lane == 0) rows[wave] = mine;
    __syncthreads();
    if (!ONE) {
        for (int i = threadIdx.x; i < a.E; i += NT) {
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) s += sums[w][i];
            psum[(long)blockIdx.x * a.E + i] = s;
            pcnt[(long)blockIdx.x * a.E + i] = counts[i];
        }
        if (threadIdx.x == 0) prow[blockIdx.x] = rows[0] + rows[1] + rows[2] + rows[3];  // W = 4
        return;
    }
    double dot = 0.0;
    for (int i = threadIdx.x; i < a.E; i += NT) {
        double s = 0.0;
        for (int w = 0; w < W && w < groups; ++w) s += sums[w][i];
        a.sums[i] = (float)s;
        a.counts[i] = counts[i];
        dot += s * counts[i];
    }
    __shared__ double dots[W];
    for (int off = 1; off < 64; off <<= 1) dot += __shfl_xor(dot, off, 64);
    if (lane == 0) dots[wave] = dot;
    __syncthreads();
    if (threadIdx.x == 0) {
        int all = 0;
        double d = 0.0;
        for (int w = 0; w < W; ++w) {
            all += rows[w];
            d += dots[w];
        }
        a.rows[0] = all;
        a.loss[0] = balance_loss(d, a.E, a.k, all);
    }
}

// The blocks' sums and counts added, 16 columns a block, always in the same order; the last
// block to finish adds up the loss.  10 us for 768 blocks' 256 columns, 6 for 64: the chain of
// loads, tree and counter.
constexpr int kTotalThreads = 1024;
__global__ __launch_bounds__(kTotalThreads) void k_route_total(RouteArgs a, int nb, const float* psum, const int* pcnt, const int* prow, double* dots,
                                                               unsigned* ticket)
{
    __shared__ double s16[64][17];
    __shared__ int c16[64][17];
    __shared__ double dot16[16];
    __shared__ bool last;
    const int col = threadIdx.x & 15, part = threadIdx.x >> 4, j = blockIdx.x * 16 + col;
    double s = 0.0;
    int c = 0;
    if (j < a.E) {
#pragma unroll 12
        for (int b = part; b < nb; b += 64) {
            s += psum[(long)b * a.E + j];
            c += pcnt[(long)b * a.E + j];
        }
    }
    s16[part][col] = s;
    c16[part][col] = c;
    __syncthreads();
    for (int half = 32; half >= 1; half /= 2) {
        if (part < half) {
            s16[part][col] += s16[part + half][col];
            c16[part][col] += c16[part + half][col];
        }
        __syncthreads();
    }
    if (threadIdx.x < 16) {
        dot16[col] = 0.0;
        if (j < a.E) {
            a.sums[j] = (float)s16[0][col];
            a.counts[j] = c16[0][col];
            dot16[col] = s16[0][col] * c16[0][col];
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double d = 0.0;
        for (int i = 0; i < 16; ++i) d += dot16[i];
        __hip_atomic_store(dots + blockIdx.x, d, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __threadfence();
        last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    int rows = 0;
    for (int b = threadIdx.x; b < nb; b += kTotalThreads) rows += prow[b];
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) rows += across(rows, off);
    if ((threadIdx.x & 63) == 0) c16[threadIdx.x >> 6][0] = rows;
    __syncthreads();
    if (threadIdx.x == 0) {
        int all = 0;
        for (int w = 0; w < kTotalThreads / 64; ++w) all += c16[w][0];
        double d = 0.0;
        for (unsigned b = 0; b < gridDim.x; ++b) d += __hip_atomic_load(dots + b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        a.rows[0] = all;
        a.loss[0] = balance_loss(d, a.E, a.k, all);
    }
}

// dz_ij = p_ij (G_j - sum_j p_ij G_j) + the chosen ones' gate part, with G_j = dloss E c_j / (k N^2).
// The gate part of a chosen score is w (dw - sum w dw) for normalized weights; otherwise w dw,
// and sum w dw joins the sum over the row.  It reaches its column through LDS.  Probabilities are
// computed anew from the scores, which costs less than keeping them would.  At 131,072 x 256
// bf16 37 us (134 MB, 3.7 TB/s).
template <typename T, int L, int NC>
__global__ __launch_bounds__(kThreads) void k_route_back(RouteBackArgs a, int nb)
{
    constexpr int RW = 64 / L, W = kThreads / 64, SPAN = L * 8 * NC;
    constexpr int kSlots = (kRouteMaxK + L - 1) / L;
    __shared__ __align__(16) float gate[W][RW][SPAN + 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & (L - 1);
    float* mine = &gate[wave][lane / L][0];
    for (int i = lane; i < RW * (SPAN + 4); i += 64) (&gate[wave][0][0])[i] = 0.f;
    const int N = a.rows[0];
    const float each = a.dloss != nullptr && N > 0 ? (float)((double)a.dloss[0] * a.E / ((double)a.k * N * N)) : 0.f;
    float G[NC][8];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int col = (c * L + j) * 8 + e;
            G[c][e] = a.dloss != nullptr && col < a.E ? each * a.counts[col] : 0.f;
        }
    const long groups = (a.n + RW - 1) / RW;
    T next[NC][8];
    bool next_on = false;
    long grp = (long)blockIdx.x * W + wave;
    if (grp < groups) load_row<T, L, NC>(a.z, a.ld, a.mask, a.mask_stride, a.n, a.E, grp * RW + lane / L, next, next_on);
    for (; grp < groups; grp += (long)nb * W) {
        const long row = grp * RW + lane / L;
        // the row's slots
        float w[kSlots], dw[kSlots];
        int ex[kSlots];
        if (a.dw != nullptr)
#pragma unroll
            for (int i = 0; i < kSlots; ++i) {
                const int t = i * L + j;
                const bool there = row < a.n && t < a.k;
                ex[i] = there ? a.ex[row * a.k + t] : -1;
                w[i] = there ? a.w[row * a.k + t] : 0.f;
                dw[i] = there ? a.dw[row * a.k + t] : 0.f;
            }
        float x[NC][8];
        float m = -INFINITY;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (c * L * 8 >= a.E) break;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[c][e] = fmaxf(to_f(next[c][e]), -INFINITY);  // NaN too
                m = fmaxf(m, x[c][e]);
            }
        }
        const bool on = next_on;
        const long after = grp + (long)nb * W;
        if (after < groups) load_row<T, L, NC>(a.z, a.ld, a.mask, a.mask_stride, a.n, a.E, after * RW + lane / L, next, next_on);
#pragma unroll
        for (int off = 1; off < L; off <<= 1) m = fmaxf(m, across(m, off));
        const bool live = on && m > -INFINITY;
        float s = 0.f, g = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (c * L * 8 >= a.E) break;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[c][e] = live ? exp_of(x[c][e] - m) : 0.f;
                s += x[c][e];
                g += x[c][e] * G[c][e];
            }
        }
        s = row_sum<L>(s);
        const float inv = live ? 1.f / s : 0.f;
        g = row_sum<L>(g) * inv;
        if (a.dw != nullptr) {
            float wd = 0.f;
#pragma unroll
            for (int i = 0; i < kSlots; ++i) wd += live && ex[i] >= 0 ? w[i] * dw[i] : 0.f;
            wd = row_sum<L>(wd);
            if (!a.normalize) g += wd;
#pragma unroll
            for (int i = 0; i < kSlots; ++i)
                if (live && ex[i] >= 0 && ex[i] < a.E) mine[ex[i]] = w[i] * (a.normalize ? dw[i] - wd : dw[i]);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        T* dz = static_cast<T*>(a.dz) + row * a.ld_dz;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (c * L * 8 >= a.E) break;
            const int col = (c * L + j) * 8;
            float gt[8] = {};
            if (a.dw != nullptr) __builtin_memcpy(gt, __builtin_assume_aligned(mine + col, 16), 32);
            T out[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) out[e] = from_f<T>(x[c][e] * inv * (G[c][e] - g) + gt[e]);
            if (row < a.n) {
                if ((c + 1) * L * 8 <= a.E || col + 8 <= a.E)
                    __builtin_memcpy(dz + col, out, 8 * sizeof(T));
                else
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (col + e < a.E) dz[col + e] = out[e];
            }
        }
        if (a.dw != nullptr) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < kSlots; ++i)
                if (live && ex[i] >= 0 && ex[i] < a.E) mine[ex[i]] = 0.f;
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// Lanes a row takes: as few as hold it in 32 scores each (one: no exchanges at all), for every
// doubling costs an exchange of the k chosen.  65,536 x 500 fp32, k = 5 take 76 us on sixteen
// lanes, 133 on a wave.
int row_lanes(int E) { return E <= 32 ? 1 : E <= 256 ? 8 : E <= 512 ? 16 : 64; }

int route_blocks(long n, int E)
{
    const long rw = 64 / row_lanes(E), groups = (n + rw - 1) / rw;
    if (groups <= kOneBlock) return 1;
    const long b = (groups + kThreads / 64 - 1) / (kThreads / 64);
    return (int)(b < kMaxBlocks ? b : kMaxBlocks);
}

struct RouteSpace {
    size_t dots, ticket, sum, cnt, row, bytes;
};
RouteSpace route_space(long n, int E)
{
    const size_t nb = (size_t)route_blocks(n, E);
    RouteSpace s{};
    s.dots = 0;
    s.ticket = s.dots + 8 * (size_t)(kRouteMaxE / 16);
    s.sum = s.ticket + 16;
    s.cnt = s.sum + nb * E * 4;
    s.row = s.cnt + nb * E * 4;
    s.bytes = s.row + nb * 4;
    return s;
}

// f(lanes a row, times eight columns a lane)
template <typename F>
hipError_t with_shape(int E, F&& f)
{
    using std::integral_constant;
    switch (row_lanes(E)) {
    case 1: return f(integral_constant<int, 1>{}, integral_constant<int, 4>{});
    case 8:
        if (E <= 64) return f(integral_constant<int, 8>{}, integral_constant<int, 1>{});
        return f(integral_constant<int, 8>{}, integral_constant<int, 4>{});
    case 16: return f(integral_constant<int, 16>{}, integral_constant<int, 4>{});
    default: return f(integral_constant<int, 64>{}, integral_constant<int, 4>{});
    }
}

template <typename F>
hipError_t with_slots(int k, F&& f)
{
    using std::integral_constant;
    if (k <= 1) return f(integral_constant<int, 1>{});
    if (k <= 2) return f(integral_constant<int, 2>{});
    if (k <= 4) return f(integral_constant<int, 4>{});
    if (k <= 8) return f(integral_constant<int, 8>{});
    return f(integral_constant<int, 16>{});
}

}  // namespace

size_t route_workspace(long n, int E) { return route_blocks(n, E) == 1 ? 0 : route_space(n, E).bytes; }

hipError_t launch_route(const RouteArgs& a, hipStream_t s)
{
    const int nb = route_blocks(a.n, a.E);
    const RouteSpace at = route_space(a.n, a.E);
    double* dots = reinterpret_cast<double*>(a.ws + at.dots);
    unsigned* ticket = reinterpret_cast<unsigned*>(a.ws + at.ticket);
    float* psum = reinterpret_cast<float*>(a.ws + at.sum);
    int* pcnt = reinterpret_cast<int*>(a.ws + at.cnt);
    int* prow = reinterpret_cast<int*>(a.ws + at.row);
    const hipError_t e = with_type(a.type, [&](auto t) {
        return with_shape(a.E, [&](auto lanes, auto times) {
            return with_slots(a.k, [&](auto slots) {
                if (nb == 1)
                    return launch(k_route<decltype(t), lanes.value, times.value, slots.value, true>, 1, kOneThreads, 0, s, a, nb, psum, pcnt, prow, ticket);
                return launch(k_route<decltype(t), lanes.value, times.value, slots.value, false>, nb, kThreads, 0, s, a, nb, psum, pcnt, prow, ticket);
            });
        });
    });
    if (e != hipSuccess || nb == 1) return e;
    return launch(k_route_total, (a.E + 15) / 16, kTotalThreads, 0, s, a, nb, psum, pcnt, prow, dots, ticket);
}

hipError_t launch_route_back(const RouteBackArgs& a, hipStream_t s)
{
    if (a.n == 0) return hipSuccess;
    const long rw = 64 / row_lanes(a.E), b = ((a.n + rw - 1) / rw + kThreads / 64 - 1) / (kThreads / 64);
    // A row of one step of columns a lane leaves registers for six blocks a CU.  us with three and with
    // six: bf16, 131,072 x 37 12.8, 11.7; x 64 13.5, 12.7; 50,003 x 37 7.5, 7.2; x 64 7.4, 8.2 (27 blocks
    // past the six); fp32, 131,072 x 37 16.2, 14.7.  Four steps: 131,072 x 256 34.0, 42.7.
    const long most = a.E <= 64 && a.E > 32 ? 2 * kMaxBlocks : kMaxBlocks;
    const int nb = (int)(b < most ? b : most);
    return with_type(a.type, [&](auto t) {
        return with_shape(a.E, [&](auto lanes, auto times) { return launch(k_route_back<decltype(t), lanes.value, times.value>, nb, kThreads, 0, s, a, nb); });
    });
}

}  // namespace skm
