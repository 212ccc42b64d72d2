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
//
// Three products in all: rows to ranks (k_shrink: t, u), ranks to rows (k_expand: out, dx)
// and rows by rows (k_outer: dD, dU).  k_plan_place first puts the rows of each adapter side by
// side (a stable counting sort) and cuts them into tiles of one adapter; with few rows
// every row is its own tile and there is no sort.
#include "experts_common.h"

namespace skm {
namespace {

constexpr int kTile = 64;        // rows of a k_shrink / k_expand tile
constexpr int kPlanRows = 4096;  // rows of a k_plan block, 1024 a wave

struct Tile {
    int q;      // adapter; a: rows without one; -1: an unused entry
    int start;  // first place in perm
    int cnt;
    int slot;   // chunks only: where its partial sums go, -1: they are the whole sum
};

struct PlanArgs {
    const int* ids; long ids_stride; int n, a;
    int* hist;           // [chunks x (a + 1)], more than one chunk only
    int* perm;           // [n] rows in the order of their adapters
    Tile* tiles; int ntiles;    // kTile rows each
    Tile* chunks; int nchunks;  // nullable; `chunk` rows each, one at least per adapter
    int2* merge;         // [a] first slot and number of an adapter's chunks where there are several
    int chunk;
};

__device__ __forceinline__ int adapter_of(const int* ids, long stride, long i, int a)
{
    const int q = ids[i * stride];
    return q >= 0 && q < a ? q : a;
}

// Lanes that hold the same key (of `bits` bits) as this one, among those with `on`.
__device__ __forceinline__ unsigned long long same_key(int key, bool on, int bits)
{
    unsigned long long m = __ballot(on);
    for (int b = 0; b < bits; ++b) {
        const bool one = (key >> b) & 1;
        const unsigned long long v = __ballot(one);
        m &= one ? v : ~v;
    }
    return m;
}

// Exclusive sum of v[0 .. count) in place (256 threads), v[count] = the total.
__device__ void block_scan(int* v, int count, int* tmp)
{
    const int per = (count + 255) / 256, lo = min(count, (int)threadIdx.x * per), hi = min(count, lo + per);
    int s = 0;
    for (int i = lo; i < hi; ++i) s += v[i];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int inc = s;
    for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(inc, off, 64);
        if (lane >= off) inc += o;
    }
    if (lane == 63) tmp[wave] = inc;
    __syncthreads();
    int base = inc - s;
    for (int w = 0; w < wave; ++w) base += tmp[w];
    for (int i = lo; i < hi; ++i) {
        const int x = v[i];
        v[i] = base;
        base += x;
    }
    if (threadIdx.x == 255) v[count] = base;
    __syncthreads();
}

// Per wave of this block's rows, how many have each key (the leaders of equal keys add
// them up, so no two lanes write one place).
__device__ void count_keys(const PlanArgs& p, unsigned short* wh, int K, int bits)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int j = threadIdx.x; j < 4 * K; j += 256) wh[j] = 0;
    __syncthreads();
    for (int it = 0; it < kPlanRows / 256; ++it) {
        const long i = (long)blockIdx.x * kPlanRows + wave * (kPlanRows / 4) + it * 64 + lane;
        const bool on = i < p.n;
        const int key = on ? adapter_of(p.ids, p.ids_stride, i, p.a) : 0;
        const unsigned long long m = same_key(key, on, bits);
        if (on && (m & ((1ull << lane) - 1)) == 0) wh[wave * K + key] += (unsigned short)__popcll(m);
    }
    __syncthreads();
}

__global__ __launch_bounds__(256) void k_plan_count(PlanArgs p, int bits)
{
    extern __shared__ char lds[];
    unsigned short* wh = reinterpret_cast<unsigned short*>(lds);
    const int K = p.a + 1;
    count_keys(p, wh, K, bits);
    for (int k = threadIdx.x; k < K; k += 256)
        p.hist[(long)blockIdx.x * K + k] = wh[k] + wh[K + k] + wh[2 * K + k] + wh[3 * K + k];
}

// `size` = rows per key, consumed: the tiles of `len` rows of every key.
__device__ void write_tiles(const int* off, int* first, int K, int a, int len, bool whole, Tile* out, int bound, int* tmp, int2* merge)
{
    // whole: one tile at least per adapter and none for the rows without one
    for (int k = threadIdx.x; k < K; k += 256) {
        const int c = off[k + 1] - off[k], t = (c + len - 1) / len;
        first[k] = !whole ? t : k == a ? 0 : max(1, t);
    }
    __syncthreads();
    block_scan(first, K, tmp);
    const int total = first[K];
    for (int t = threadIdx.x; t < bound; t += 256) {
        Tile e{-1, 0, 0, -1};
        if (t < total) {
            int lo = 0, hi = K;  // the last key whose tiles start at t or before
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (first[mid] <= t) lo = mid; else hi = mid;
            }
            const int c = off[lo + 1] - off[lo], at = (t - first[lo]) * len;
            e.q = lo;
            e.start = off[lo] + at;
            e.cnt = min(len, c - at);
            if (whole && c > len) e.slot = t;
        }
        out[t] = e;
    }
    __syncthreads();
    if (merge != nullptr)
        for (int k = threadIdx.x; k < a; k += 256) {
            const int t = first[k + 1] - first[k];
            merge[k] = make_int2(first[k], t > 1 ? t : 0);
        }
    __syncthreads();
}

// Places of the rows, and (block 0) the tiles.  Without a histogram this block holds all
// the rows.
__global__ __launch_bounds__(256) void k_plan_place(PlanArgs p, int bits)
{
    extern __shared__ char lds[];
    const int K = p.a + 1;
    int* off = reinterpret_cast<int*>(lds);        // [K + 1] first place of each key, over all rows
    int* at = off + K + 1;                         // [K + 1] first place of this block's
    int* tmp = at + K + 1;                         // [4]
    unsigned short* wh = reinterpret_cast<unsigned short*>(tmp + 4);  // [4 x K]
    count_keys(p, wh, K, bits);
    for (int k = threadIdx.x; k < K; k += 256) {
        int c = 0;
        for (int w = 0; w < 4; ++w) {
            const int x = wh[w * K + k];
            wh[w * K + k] = (unsigned short)c;
            c += x;
        }
        int before = 0;
        if (p.hist != nullptr) {
            c = 0;
            for (int b = 0; b < (int)gridDim.x; ++b) {
                const int x = p.hist[(long)b * K + k];
                if (b < (int)blockIdx.x) before += x;
                c += x;
            }
        }
        off[k] = c;
        at[k] = before;
    }
    __syncthreads();
    block_scan(off, K, tmp);
    for (int k = threadIdx.x; k < K; k += 256) at[k] += off[k];
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    volatile unsigned short* mine = wh + wave * K;
    for (int it = 0; it < kPlanRows / 256; ++it) {
        const long i = (long)blockIdx.x * kPlanRows + wave * (kPlanRows / 4) + it * 64 + lane;
        const bool on = i < p.n;
        const int key = on ? adapter_of(p.ids, p.ids_stride, i, p.a) : 0;
        const unsigned long long m = same_key(key, on, bits), lower = m & ((1ull << lane) - 1);
        if (on) {
            const int seen = mine[key];
            p.perm[at[key] + seen + __popcll(lower)] = (int)i;
            if (lower == 0) mine[key] = (unsigned short)(seen + __popcll(m));
        }
    }
    if (blockIdx.x != 0) return;
    __syncthreads();
    write_tiles(off, at, K, p.a, kTile, false, p.tiles, p.ntiles, tmp, nullptr);
    if (p.chunks != nullptr) write_tiles(off, at, K, p.a, p.chunk, true, p.chunks, p.nchunks, tmp, p.merge);
}

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

struct Rows {  // where the rows of a tile come from
    const Tile* tiles;   // nullable: tile i is row i
    const int* perm;
    const int* ids; long ids_stride; int a;
};

__device__ __forceinline__ Tile tile_at(const Rows& w, int t)
{
    if (w.tiles != nullptr) return w.tiles[t];
    return Tile{adapter_of(w.ids, w.ids_stride, t, w.a), t, 1, -1};
}

__device__ __forceinline__ int row_at(const Rows& w, int place) { return w.tiles != nullptr ? w.perm[place] : place; }

// ---- rows to ranks ----

template <typename T>
struct ShrinkArgs {
    Rows rows;
    const T* v; long ld_v;       // [n x w]
    const T* M; long sa, ld;     // [a][r][w]
    int w, r; long n;
    int splits;                  // of w, one a blockIdx.y
    float* part;                 // [splits][n][r]
};

// part[s][row][t] = sum over the s-th part of the columns of M_q[t] v_row.  A block takes
// RT * 16 rows of one adapter and NB * 16 ranks; its four waves take the columns in turn,
// 128 bytes of each row at a time, and add up their sums at the end, so that rows and
// adapter are read once and go to the matrix cores straight from memory.
template <typename T, int RT, int NB>
__global__ __launch_bounds__(256) void k_shrink(ShrinkArgs<T> p)
{
    constexpr int KS = 128 / sizeof(T);
    __shared__ float sum[2][RT * 16][NB * 16 + 1];
    const Tile t = tile_at(p.rows, blockIdx.x);
    if (t.q < 0 || t.q >= p.rows.a) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
    const int rank0 = blockIdx.z * (NB * 16);
    const T* v[RT];
    const T* m[NB];
#pragma unroll
    for (int i = 0; i < RT; ++i) v[i] = p.v + (long)row_at(p.rows, t.start + min(i * 16 + l16, t.cnt - 1)) * p.ld_v + g * (KS / 4);
#pragma unroll
    for (int b = 0; b < NB; ++b) m[b] = p.M + t.q * p.sa + (long)min(rank0 + b * 16 + l16, p.r - 1) * p.ld + g * (KS / 4);
    f32x4 acc[RT][NB];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[i][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int steps = (p.w + KS - 1) / KS;
    const int s0 = (int)((long)steps * blockIdx.y / p.splits), s1 = (int)((long)steps * (blockIdx.y + 1) / p.splits);
    const int full = p.w / KS;
    for (int s = s0 + wave; s < s1; s += 4) {
        Vec<T> x[RT][2], y[NB][2];
        if (s < full) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < RT; ++i) x[i][h] = load16(v[i] + (long)s * KS + h * kVec<T>);
#pragma unroll
                for (int b = 0; b < NB; ++b) y[b][h] = load16(m[b] + (long)s * KS + h * kVec<T>);
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int left = p.w - (s * KS + g * (KS / 4) + h * kVec<T>);
#pragma unroll
                for (int i = 0; i < RT; ++i) x[i][h] = load_part(v[i] + (long)s * KS + h * kVec<T>, left);
#pragma unroll
                for (int b = 0; b < NB; ++b) y[b][h] = load_part(m[b] + (long)s * KS + h * kVec<T>, left);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int b = 0; b < NB; ++b) acc[i][b] = mfma16(x[i][h], y[b][h], acc[i][b]);
    }
    // waves 2 and 3 hand their sums to 0 and 1, then 1 to 0
    for (int from = 2; from >= 1; --from) {
        if (wave >= from && wave < 2 * from)
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[wave - from][i * 16 + g * 4 + e][b * 16 + l16] = acc[i][b][e];
        __syncthreads();
        if (wave < from)
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][b][e] += sum[wave][i * 16 + g * 4 + e][b * 16 + l16];
        __syncthreads();
    }
    if (wave != 0) return;
    float* out = p.part + (long)blockIdx.y * p.n * p.r;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int at = i * 16 + g * 4 + e;
            if (at >= t.cnt) continue;
            const long row = row_at(p.rows, t.start + at);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int rank = rank0 + b * 16 + l16;
                if (rank < p.r) out[row * p.r + rank] = acc[i][b][e];
            }
        }
}

// ---- ranks to rows ----

template <typename T>
struct ExpandArgs {
    Rows rows;
    const float* part; int splits; long n;   // k_shrink's
    const T* M; long sa, ld;                 // [a][r][w]
    const float* gates; long gates_stride; const float* scales;
    const T* base; long ld_base;             // nullable
    T* out; long ld_out;
    int w, r;
    float* low;                              // nullable: [n x r], the splits' sum (0 for a row without an adapter)
    const float* dot; float* dgates;         // nullable: dgates[i] = s_q <low_i, dot_i>
};

// out_row = base_row + f_row low_row M_q.  A block takes RT * 16 rows of one adapter and
// four waves' columns, 16 * kVec each, of which a wave keeps M_q in registers.  The product is taken
// as (M_q^T)(low^T) on the fp32 matrix cores, four ranks at a time: M_q then needs no
// transposition, low no rounding, and a lane ends up with 16 bytes of a row, four times.
template <typename T, int RT, int NB>
__global__ __launch_bounds__(256) void k_expand(ExpandArgs<T> p)
{
    constexpr int V = kVec<T>;
    const Tile t = tile_at(p.rows, blockIdx.x);
    if (t.q < 0) return;
    const bool has = t.q < p.rows.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
    if (blockIdx.y == 0 && (p.low != nullptr || p.dgates != nullptr)) {
        for (int at = wave; at < t.cnt; at += 4) {
            const long row = row_at(p.rows, t.start + at);
            float d = 0.f;
            for (int k = lane; k < p.r; k += 64) {
                float s = 0.f;
                if (has)
                    for (int c = 0; c < p.splits; ++c) s += p.part[(c * p.n + row) * p.r + k];
                if (p.low != nullptr) p.low[row * p.r + k] = s;
                if (p.dgates != nullptr && has) d += s * p.dot[row * p.r + k];
            }
            if (p.dgates != nullptr) {
                for (int off = 1; off < 64; off <<= 1) d += __shfl_xor(d, off, 64);
                if (lane == 0) p.dgates[row] = has ? d * (p.scales ? p.scales[t.q] : 1.f) : 0.f;
            }
        }
    }
    const int c0 = (blockIdx.y * 4 + wave) * 16 * V;
    if (c0 >= p.w) return;
    Vec<T> m[NB][4];
    const int cm = c0 + ((l16 & 3) * 4 + (l16 >> 2)) * V;  // the columns of M this lane brings
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int rank = b * 16 + g * 4 + s;
            m[b][s] = load_part(p.M + (has ? t.q * p.sa + (long)rank * p.ld + cm : 0), has && rank < p.r ? p.w - cm : 0);
        }
    const float sc = has && p.scales ? p.scales[t.q] : 1.f;
#pragma unroll 1
    for (int i = 0; i < RT; ++i) {
        if (i * 16 >= t.cnt) break;
        const bool on = i * 16 + l16 < t.cnt;
        const long row = row_at(p.rows, t.start + min(i * 16 + l16, t.cnt - 1));
        Vec<T> y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c = c0 + (e * 4 + g) * V;
            y[e] = load_part(p.base + (p.base ? row * p.ld_base + c : 0), p.base && on ? p.w - c : 0);
        }
        f32x4 acc[V];
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        float f = 0.f;
        if (has) {
            f = (p.gates ? p.gates[row * p.gates_stride] : 1.f) * sc;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float lo[4] = {0.f, 0.f, 0.f, 0.f};
                for (int c = 0; c < p.splits; ++c)
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        const int rank = b * 16 + g * 4 + s;
                        if (rank < p.r) lo[s] += p.part[(c * p.n + row) * p.r + rank];
                    }
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int j = 0; j < V; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(to_f(m[b][s][j]), lo[s], acc[j], 0, 0, 0);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c = c0 + (e * 4 + g) * V, left = on ? p.w - c : 0;
            Vec<T> z;
#pragma unroll
            for (int j = 0; j < V; ++j) z[j] = from_f<T>(has ? to_f(y[e][j]) + f * acc[j][e] : to_f(y[e][j]));
            T* o = p.out + row * p.ld_out + c;
            if (left >= V)
                __builtin_memcpy(o, &z, 16);
            else
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (j < left) o[j] = z[j];
        }
    }
}

// ---- rows by rows ----

template <typename T>
struct OuterSide {
    const float* low;                        // [n x r]
    const T* v; long ld_v; int w;            // [n x w]
    T* dM;                                   // [a][r][w]
    float* part;                             // [slots][r][w]
};
template <typename T>
struct OuterArgs {
    const Tile* chunks; const int2* merge; const int* perm; int a, r;
    const float* gates; long gates_stride; const float* scales;
    OuterSide<T> side[2];                    // blockIdx.y < split: side 0
    int split;                               // blocks of side 0's columns
};

constexpr int kMaxChunk = 512;

// dM_q[t] += sum over a chunk's rows of f_row low_row[t] v_row.  A block takes the chunk
// and 16 * kVec columns, its four waves every fourth quad of rows; both operands go to the
// fp32 matrix cores as they lie in memory.
template <typename T, int NB>
__global__ __launch_bounds__(256) void k_outer(OuterArgs<T> p)
{
    constexpr int V = kVec<T>, W = 16 * V;
    __shared__ int rows[kMaxChunk];
    __shared__ float fac[kMaxChunk];
    extern __shared__ char lds[];
    float* sum = reinterpret_cast<float*>(lds);  // [2][NB * 16][W]
    const Tile t = p.chunks[blockIdx.x];
    if (t.q < 0) return;
    const bool second = (int)blockIdx.y >= p.split;
    const OuterSide<T>& s = p.side[second];
    const int c0 = ((int)blockIdx.y - (second ? p.split : 0)) * W, rank0 = blockIdx.z * (NB * 16);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
    const float sc = p.scales ? p.scales[t.q] : 1.f;
    for (int i = threadIdx.x; i < t.cnt; i += 256) {
        const int row = p.perm[t.start + i];
        rows[i] = row;
        fac[i] = (p.gates ? p.gates[row * p.gates_stride] : 1.f) * sc;
    }
    __syncthreads();
    f32x4 acc[NB][V];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < V; ++j) acc[b][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int c = c0 + l16 * V, left = s.w - c;
    const int quads = (t.cnt + 3) / 4;
    for (int k = wave; k < quads; k += 4) {
        const int i = k * 4 + g;
        const bool on = i < t.cnt;
        const long row = rows[on ? i : 0];
        const float f = on ? fac[i] : 0.f;
        const Vec<T> v = load_part(s.v + row * s.ld_v + c, on ? left : 0);
        float lo[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int rank = rank0 + b * 16 + l16;
            lo[b] = on && rank < p.r ? f * s.low[row * p.r + rank] : 0.f;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < V; ++j) acc[b][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(lo[b], to_f(v[j]), acc[b][j], 0, 0, 0);
    }
    for (int from = 2; from >= 1; --from) {
        if (wave >= from && wave < 2 * from)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int j = 0; j < V; ++j) sum[((wave - from) * NB * 16 + b * 16 + g * 4 + e) * W + l16 * V + j] = acc[b][j][e];
        __syncthreads();
        if (wave < from)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int j = 0; j < V; ++j) acc[b][j][e] += sum[(wave * NB * 16 + b * 16 + g * 4 + e) * W + l16 * V + j];
        __syncthreads();
    }
    if (wave != 0) return;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int rank = rank0 + b * 16 + g * 4 + e;
            if (rank >= p.r) continue;
            if (t.slot >= 0) {
                float* o = s.part + ((long)t.slot * p.r + rank) * s.w + c;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (j < left) o[j] = acc[b][j][e];
            } else {
                T* o = s.dM + ((long)t.q * p.r + rank) * s.w + c;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (j < left) o[j] = from_f<T>(acc[b][j][e]);
            }
        }
}

// The chunks' sums of the adapters that have several, added in chunk order.
template <typename T>
__global__ __launch_bounds__(256) void k_outer_merge(OuterArgs<T> p)
{
    const int2 m = p.merge[blockIdx.y];
    if (m.y == 0) return;
    const OuterSide<T>& s = p.side[blockIdx.z];
    const long size = (long)p.r * s.w;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < size; i += (long)gridDim.x * 256) {
        float v = 0.f;
        for (int k = 0; k < m.y; ++k) v += s.part[(m.x + k) * size + i];
        s.dM[blockIdx.y * size + i] = from_f<T>(v);
    }
}

// ---- host ----

// Rows up to which every row is its own tile (no sort): its adapter is then read once a
// row instead of once a tile.
constexpr long kDirectRows = 128;

size_t up16(size_t b) { return (b + 15) & ~size_t(15); }

struct Layout {
    long n; int a, r;
    bool direct;
    int blocks, ntiles, nchunks, chunk;
    int down_splits, up_splits;           // of d (t = D x) and of o (u = U dy)
    size_t hist, perm, tiles, chunks, merge, part, low, dpart, upart, bytes;
};

// Parts of the columns, so that enough blocks read at once; each wave still has a step.
int split_count(long tiles, int w, int type, int zs)
{
    if (tiles < 1) tiles = 1;
    const long steps = (w + 128 / (int)elem_size(type) - 1) / (128 / (int)elem_size(type));
    long s = (1024 + tiles * zs - 1) / (tiles * zs);
    const long most = (steps + 3) / 4;
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s > 16 ? 16 : s);
}

Layout layout(int type, long n, int d, int o, int r, int a, bool backward)
{
    Layout L{};
    L.n = n; L.a = a; L.r = r;
    L.direct = n <= kDirectRows && !backward;
    L.blocks = (int)((n + kPlanRows - 1) / kPlanRows);
    if (L.blocks < 1) L.blocks = 1;
    L.ntiles = L.direct ? (int)n : (int)((n + kTile - 1) / kTile) + a + 1;
    L.chunk = kMaxChunk / 2;
    L.nchunks = (int)(n / L.chunk) + a;
    const int zs = (r + 63) / 64;
    L.down_splits = split_count(L.direct ? n : (n + kTile - 1) / kTile, d, type, zs);
    L.up_splits = split_count(L.direct ? n : (n + kTile - 1) / kTile, o, type, zs);
    size_t at = 0;
    auto take = [&](size_t& where, size_t bytes) { where = at; at += up16(bytes); };
    if (!L.direct) {
        take(L.hist, L.blocks > 1 ? (size_t)L.blocks * (a + 1) * 4 : 0);
        take(L.perm, (size_t)n * 4);
        take(L.tiles, (size_t)L.ntiles * sizeof(Tile));
    }
    take(L.part, (size_t)(backward ? L.up_splits : L.down_splits) * n * r * 4);
    if (backward) {
        take(L.chunks, (size_t)L.nchunks * sizeof(Tile));
        take(L.merge, (size_t)a * sizeof(int2));
        take(L.low, (size_t)n * r * 4);
        take(L.dpart, (size_t)L.nchunks * r * d * 4);
        take(L.upart, (size_t)L.nchunks * r * o * 4);
    }
    L.bytes = at;
    return L;
}

hipError_t launch_plan(const Layout& L, const int* ids, long ids_stride, char* ws, bool backward, hipStream_t s)
{
    PlanArgs p{ids, ids_stride, (int)L.n, L.a, L.blocks > 1 ? reinterpret_cast<int*>(ws + L.hist) : nullptr,
               reinterpret_cast<int*>(ws + L.perm), reinterpret_cast<Tile*>(ws + L.tiles), L.ntiles,
               backward ? reinterpret_cast<Tile*>(ws + L.chunks) : nullptr, L.nchunks,
               backward ? reinterpret_cast<int2*>(ws + L.merge) : nullptr, L.chunk};
    const int K = L.a + 1;
    int bits = 0;
    while ((1 << bits) < K) ++bits;
    if (L.blocks > 1) SKM_TRY_LAUNCH(k_plan_count, L.blocks, 256, 8 * (size_t)K, s, p, bits);
    return launch(k_plan_place, L.blocks, 256, 8 * (size_t)(K + 1) + 16 + 8 * (size_t)K, s, p, bits);
}

template <typename T, int RT>
hipError_t launch_shrink(const ShrinkArgs<T>& p, int ntiles, hipStream_t s)
{
    const dim3 grid(ntiles, p.splits, (p.r + 63) / 64);
    if (p.r <= 16) return launch(k_shrink<T, RT, 1>, grid, 256, 0, s, p);
    if (p.r <= 32) return launch(k_shrink<T, RT, 2>, grid, 256, 0, s, p);
    return launch(k_shrink<T, RT, 4>, grid, 256, 0, s, p);
}

template <typename T, int RT>
hipError_t launch_expand(const ExpandArgs<T>& p, int ntiles, hipStream_t s)
{
    const dim3 grid(ntiles, (p.w + 64 * kVec<T> - 1) / (64 * kVec<T>));
    if (p.r <= 16) return launch(k_expand<T, RT, 1>, grid, 256, 0, s, p);
    if (p.r <= 32) return launch(k_expand<T, RT, 2>, grid, 256, 0, s, p);
    if (p.r <= 64) return launch(k_expand<T, RT, 4>, grid, 256, 0, s, p);
    return launch(k_expand<T, RT, 8>, grid, 256, 0, s, p);
}

template <typename T>
hipError_t shrink_expand(const Layout& L, const Rows& rows, const ShrinkArgs<T>& sh, const ExpandArgs<T>& ex, hipStream_t s)
{
    if (L.direct) {
        const hipError_t e = L.a > 0 ? launch_shrink<T, 1>(sh, L.ntiles, s) : hipSuccess;
        return e != hipSuccess ? e : launch_expand<T, 1>(ex, L.ntiles, s);
    }
    const hipError_t e = L.a > 0 ? launch_shrink<T, kTile / 16>(sh, L.ntiles, s) : hipSuccess;
    return e != hipSuccess ? e : launch_expand<T, kTile / 16>(ex, L.ntiles, s);
}

}  // namespace

size_t adapt_workspace(int type, long n, int d, int o, int r, int a, int backward) { return layout(type, n, d, o, r, a, backward != 0).bytes; }

hipError_t launch_adapt(const AdaptArgs& a, hipStream_t s)
{
    if (a.n == 0) return hipSuccess;
    const Layout L = layout(a.type, a.n, a.d, a.o, a.r, a.a, false);
    if (!L.direct) {
        const hipError_t e = launch_plan(L, a.ids, a.ids_stride, a.ws, false, s);
        if (e != hipSuccess) return e;
    }
    const Rows rows{L.direct ? nullptr : reinterpret_cast<const Tile*>(a.ws + L.tiles), reinterpret_cast<const int*>(a.ws + L.perm), a.ids, a.ids_stride, a.a};
    float* part = reinterpret_cast<float*>(a.ws + L.part);
    return with_type(a.type, [&](auto tag) {
        using T = decltype(tag);
        const ShrinkArgs<T> sh{rows, (const T*)a.x, a.ld_x, (const T*)a.down, a.down_sa, a.down_ld, a.d, a.r, a.n, L.down_splits, part};
        const ExpandArgs<T> ex{rows, part, L.down_splits, a.n, (const T*)a.up, a.up_sa, a.up_ld, a.gates, a.gates_stride, a.scales,
                               (const T*)a.base, a.ld_base, (T*)a.out, a.ld_out, a.o, a.r, a.low, nullptr, nullptr};
        return shrink_expand<T>(L, rows, sh, ex, s);
    });
}

hipError_t launch_adapt_back(const AdaptBackArgs& a, hipStream_t s)
{
    const Layout L = layout(a.type, a.n, a.d, a.o, a.r, a.a, true);
    if (a.n == 0 && a.a == 0) return hipSuccess;
    const hipError_t planned = launch_plan(L, a.ids, a.ids_stride, a.ws, true, s);
    if (planned != hipSuccess) return planned;
    const Rows rows{reinterpret_cast<const Tile*>(a.ws + L.tiles), reinterpret_cast<const int*>(a.ws + L.perm), a.ids, a.ids_stride, a.a};
    float* part = reinterpret_cast<float*>(a.ws + L.part);
    float* u = reinterpret_cast<float*>(a.ws + L.low);
    return with_type(a.type, [&](auto tag) {
        using T = decltype(tag);
        if (a.n > 0) {
            const ShrinkArgs<T> sh{rows, (const T*)a.dy, a.ld_dy, (const T*)a.up, a.up_sa, a.up_ld, a.o, a.r, a.n, L.up_splits, part};
            const ExpandArgs<T> ex{rows, part, L.up_splits, a.n, (const T*)a.down, a.down_sa, a.down_ld, a.gates, a.gates_stride, a.scales,
                                   (const T*)a.base, a.ld_base, (T*)a.dx, a.ld_dx, a.d, a.r, u, a.low, a.dgates};
            const hipError_t e = shrink_expand<T>(L, rows, sh, ex, s);
            if (e != hipSuccess) return e;
        }
        if (a.a == 0) return hipSuccess;
        constexpr int W = 16 * kVec<T>;
        const OuterArgs<T> ou{reinterpret_cast<const Tile*>(a.ws + L.chunks), reinterpret_cast<const int2*>(a.ws + L.merge), rows.perm, a.a, a.r,
                              a.gates, a.gates_stride, a.scales,
                              {{u, (const T*)a.x, a.ld_x, a.d, (T*)a.ddown, reinterpret_cast<float*>(a.ws + L.dpart)},
                               {a.low, (const T*)a.dy, a.ld_dy, a.o, (T*)a.dup, reinterpret_cast<float*>(a.ws + L.upart)}},
                              (a.d + W - 1) / W};
        const int cols = ou.split + (a.o + W - 1) / W;
        if (a.r <= 16)
            SKM_TRY_LAUNCH(k_outer<T, 1>, dim3(L.nchunks, cols, 1), 256, 2 * 16 * W * 4, s, ou);
        else
            SKM_TRY_LAUNCH(k_outer<T, 2>, dim3(L.nchunks, cols, (a.r + 31) / 32), 256, 2 * 32 * W * 4, s, ou);
        const long most = (long)a.r * (a.d > a.o ? a.d : a.o);
        return launch(k_outer_merge<T>, dim3((unsigned)((most + 1023) / 1024), a.a, 2), 256, 0, s, ou);
    });
}

}  // namespace skm
