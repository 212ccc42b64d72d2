// drop_kernels.hip -- dropout whose mask is a function of place and key, never stored.
//
//   out_ij = base_ij + (word(i d + j) >= t ? x_ij s : 0),   t = p 2^32,   s = 1 / (1 - p)
//
// word(e) is number e mod 4 of the four 32-bit words that Philox4x32-10 (Salmon, Moraes, Dror,
// Shaw: Parallel random numbers: as easy as 1, 2, 3, 2011) makes of the counter (e / 4: 64 bits, site,
// step) under a 64-bit seed.  The gradient of x is the same call on out's gradient, with the same key:
// the mask is made anew, which costs less than the n d bits it would take to keep.
//
// Bound by memory: Philox is 20 products of 32 x 32 bits and about 60 simple instructions for four
// elements.
#include "experts_common.h"

namespace skm {
namespace {

constexpr int kDropThreads = 256;
constexpr int kChunk = 8;  // elements a lane takes at once: two counters

struct Words {
    unsigned w[4];
};

__device__ __forceinline__ Words philox(unsigned long long block, unsigned site, unsigned step, unsigned k0, unsigned k1)
{
    unsigned c0 = (unsigned)block, c1 = (unsigned)(block >> 32), c2 = site, c3 = step;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long long a = 0xD2511F53ull * c0, b = 0xCD9E8D57ull * c2;
        c0 = (unsigned)(b >> 32) ^ c1 ^ k0;
        c1 = (unsigned)b;
        c2 = (unsigned)(a >> 32) ^ c3 ^ k1;
        c3 = (unsigned)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return Words{{c0, c1, c2, c3}};
}

struct Key {
    unsigned k0, k1, step;
    __device__ explicit Key(const long long* key) : k0((unsigned)key[0]), k1((unsigned)((unsigned long long)key[0] >> 32)), step((unsigned)key[1]) {}
};

template <typename T>
struct DropArgs {
    const T* x; long ld_x;
    const T* base; long ld_base;  // nullable
    T* out; long ld_out;
    long n, d;                    // rows whose elements lie side by side; one row where nothing lies between them
    const long long* key; unsigned site, limit; float scale;
    long chunks;                  // a row
};

template <typename T>
__device__ __forceinline__ T dropped(T x, T base, bool has, unsigned word, unsigned limit, float scale)
{
    const float v = word >= limit ? to_f(x) * scale : 0.f;
    return from_f<T>(has ? to_f(base) + v : v);
}

// Eight elements of a row from an element on whose number is a multiple of four.
template <typename T>
__device__ __forceinline__ void drop8(const DropArgs<T>& p, long row, long col, const Key& key)
{
    constexpr int V = kVec<T>;
    const T* x = p.x + row * p.ld_x + col;
    const T* base = p.base + row * p.ld_base + col;
    T* out = p.out + row * p.ld_out + col;
    const bool has = p.base != nullptr;
    const unsigned long long block = (unsigned long long)(row * p.d + col) >> 2;
    if (col + kChunk <= p.d) {
        Vec<T> xv[kChunk / V], bv[kChunk / V];
#pragma unroll
        for (int u = 0; u < kChunk / V; ++u) xv[u] = load16(x + u * V);
        if (has)
#pragma unroll
            for (int u = 0; u < kChunk / V; ++u) bv[u] = load16(base + u * V);
        else
#pragma unroll
            for (int u = 0; u < kChunk / V; ++u) bv[u] = Vec<T>{};
        const Words w[2] = {philox(block, p.site, key.step, key.k0, key.k1), philox(block + 1, p.site, key.step, key.k0, key.k1)};
#pragma unroll
        for (int u = 0; u < kChunk / V; ++u) {
            Vec<T> v;
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = dropped<T>(xv[u][j], bv[u][j], has, w[(u * V + j) / 4].w[j % 4], p.limit, p.scale);
            stream16(out + u * V, v);
        }
        return;
    }
    const Words w[2] = {philox(block, p.site, key.step, key.k0, key.k1), philox(block + 1, p.site, key.step, key.k0, key.k1)};
#pragma unroll
    for (int j = 0; j < kChunk; ++j)
        if (col + j < p.d) out[j] = dropped<T>(x[j], has ? base[j] : (T)0.f, has, w[j / 4].w[j % 4], p.limit, p.scale);
}

// Rows in chunks of eight elements.  16,384 x 4,096 bf16, one call with a base and one without in turn: 125 us, 5.4 TB/s (over and over
// the same: 66 with, 56 without).
template <typename T>
__global__ __launch_bounds__(kDropThreads) void k_drop(DropArgs<T> p)
{
    const Key key(p.key);
    const long all = p.n * p.chunks, step = (long)gridDim.x * kDropThreads;
    for (long c = (long)blockIdx.x * kDropThreads + threadIdx.x; c < all; c += step) {
        const long row = p.n == 1 ? 0 : all >> 32 ? c / p.chunks : (unsigned)c / (unsigned)p.chunks;
        drop8(p, row, (c - row * p.chunks) * kChunk, key);
    }
}

// Rows apart whose width is not a multiple of four: a lane takes the four elements of a counter one by one, of one row or
// the end of one and the beginning of the next.  16,384 x 777 bf16, rows 780 apart: 24 us, with an element a lane 44 (rows without gaps: 13).
template <typename T>
__global__ __launch_bounds__(kDropThreads) void k_drop_apart(DropArgs<T> p)
{
    const Key key(p.key);
    const long all = p.n * p.d, step = (long)gridDim.x * kDropThreads * 4;
    for (long e = ((long)blockIdx.x * kDropThreads + threadIdx.x) * 4; e < all; e += step) {
        long row = all >> 32 ? e / p.d : (unsigned)e / (unsigned)p.d, col = e - row * p.d;
        const Words w = philox((unsigned long long)e >> 2, p.site, key.step, key.k0, key.k1);
        const bool has = p.base != nullptr;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (e + j < all) p.out[row * p.ld_out + col] = dropped<T>(p.x[row * p.ld_x + col], has ? p.base[row * p.ld_base + col] : (T)0.f, has, w.w[j], p.limit, p.scale);
            if (++col == p.d) {
                col = 0;
                ++row;
            }
        }
    }
}

}  // namespace

hipError_t launch_drop(const DropCall& a, hipStream_t s)
{
    if (a.n == 0 || a.d == 0) return hipSuccess;
    return with_type(a.type, [&](auto tag) {
        using T = decltype(tag);
        DropArgs<T> p{(const T*)a.x, a.ld_x, (const T*)a.base, a.ld_base, (T*)a.out, a.ld_out, a.n, a.d, a.key, a.site, a.limit, a.scale, 0};
        if (a.n == 1 || (a.ld_x == a.d && a.ld_out == a.d && (a.base == nullptr || a.ld_base == a.d))) {
            p.d = a.n * a.d;
            p.n = 1;
        }
        p.chunks = (p.d + kChunk - 1) / kChunk;
        const bool apart = p.n > 1 && p.d % 4 != 0;
        const long blocks = ((apart ? (p.n * p.d + 3) / 4 : p.n * p.chunks) + kDropThreads - 1) / kDropThreads;
        const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536));
        return apart ? launch(k_drop_apart<T>, grid, kDropThreads, 0, s, p) : launch(k_drop<T>, grid, kDropThreads, 0, s, p);
    });
}

}  // namespace skm
