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
// and rows by rows (k_outer: dD, dU).  k_plan first puts the rows of each adapter side by
// side (a stable counting sort) and cuts them into tiles of one adapter; with few rows
// every row is its own tile and there is no sort; where they are small besides, the first two
// products are one launch (k_direct).
#include "experts_common.h"

namespace skm {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanLoads = 16;     // ids a k_plan lane holds
constexpr int kPlanRows = kPlanThreads * kPlanLoads;

struct Tile {
    int q;      // adapter; a: rows without one; -1: an unused entry
    int start;  // first place in perm
    int cnt;
    int slot;   // chunks only: where its partial sums go, -1: they are the whole sum
};

struct PlanArgs {
    const int* ids; long ids_stride; int n, a;
    int2* seen;          // [a + 1][segments] rows below and of each adapter, more than one segment only
    int* perm;           // [n] rows in the order of their adapters
    Tile* tiles; int ntiles, tile;    // `tile` rows each
    Tile* chunks; int nchunks;  // nullable; `chunk` rows each, one at least per adapter
    int2* merge;         // [a] first slot and number of an adapter's chunks where there are several
    int chunk; bool slot_by_entry;
};

__device__ __forceinline__ int adapter_of(const int* ids, long stride, long i, int a)
{
    const int q = ids[i * stride];
    return q >= 0 && q < a ? q : a;
}

// The tiles of adapter q, of `len` rows each (`whole`: one at least, and none for the rows
// without an adapter).  Tile j of q has the entry start_q / len + q + j: start_(q+1) / len + q + 1
// is at least that many entries on, so q's block needs no other's count; the entries
// between stay unused.  `slot` is the first of the slots that the tiles take where they are several.
__device__ void write_tiles(int q, int a, int start, int cnt, int len, bool whole, Tile* out, int bound, int slot, int2* merge)
{
    const int first = start / len + q;
    const int tiles = !whole ? (cnt + len - 1) / len : q == a ? 0 : max(1, (cnt + len - 1) / len);
    const int next = q == a ? bound : (start + cnt) / len + q + 1;
    for (int j = threadIdx.x; first + j < next; j += kPlanThreads)
        out[first + j] = j < tiles ? Tile{q, start + j * len, min(len, cnt - j * len), whole && tiles > 1 ? slot + j : -1} : Tile{-1, 0, 0, -1};
    if (merge != nullptr && q < a && threadIdx.x == 0) merge[q] = make_int2(slot, tiles > 1 ? tiles : 0);
}

// The keys of a segment of kPlanRows rows, a wave's side by side (a + 1: no row).
__device__ __forceinline__ void plan_keys(const PlanArgs& p, int* key)
{
    const long first = (long)blockIdx.y * kPlanRows + (threadIdx.x >> 6) * (64 * kPlanLoads) + (threadIdx.x & 63);
#pragma unroll
    for (int it = 0; it < kPlanLoads; ++it) key[it] = p.a + 1;
    if (p.n == 0) return;
#pragma unroll
    for (int it = 0; it < kPlanLoads; ++it) key[it] = p.ids[min(first + it * 64, (long)p.n - 1) * p.ids_stride];  // all in flight
#pragma unroll
    for (int it = 0; it < kPlanLoads; ++it) {
        const int k = key[it] >= 0 && key[it] < p.a ? key[it] : p.a;
        key[it] = first + it * 64 < p.n ? k : p.a + 1;
    }
}

// Rows of the segment with keys below q, and with q, per wave.
__device__ __forceinline__ void plan_count(const int* key, int q, int* below, int* equal)
{
    int lo = 0, eq = 0;
#pragma unroll
    for (int it = 0; it < kPlanLoads; ++it) {
        lo += __popcll(__ballot(key[it] < q));
        eq += __popcll(__ballot(key[it] == q));
    }
    if ((threadIdx.x & 63) == 0) {
        below[threadIdx.x >> 6] = lo;
        equal[threadIdx.x >> 6] = eq;
    }
    __syncthreads();
}

__global__ __launch_bounds__(kPlanThreads) void k_plan_count(PlanArgs p)
{
    __shared__ int below[kPlanThreads / 64], equal[kPlanThreads / 64];
    int key[kPlanLoads];
    plan_keys(p, key);
    plan_count(key, blockIdx.x, below, equal);
    if (threadIdx.x != 0) return;
    int2 s = make_int2(0, 0);
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        s.x += below[w];
        s.y += equal[w];
    }
    p.seen[(long)blockIdx.x * gridDim.y + blockIdx.y] = s;
}

// The places of adapter blockIdx.x's rows (a: of the rows without one) among the rows of
// segment blockIdx.y, in their order, and its tiles.  Every block reads the ids anew and counts
// those below its own adapter: 16,384 rows and 64 adapters take 6.5 us, the launch and three
// dependent trips to memory (11 with a wait after each of a lane's ids; one block that sorts all
// the rows took 18).  The work is rows times adapters: with k_plan_count 131,072 rows take 24 us
// for 64 adapters and 403 for 2,048, 1,048,576 rows 5.4 ms for 2,048.
__global__ __launch_bounds__(kPlanThreads) void k_plan(PlanArgs p)
{
    __shared__ int below[kPlanThreads / 64], equal[kPlanThreads / 64], all[3];
    const int q = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, segments = gridDim.y;
    int key[kPlanLoads];
    plan_keys(p, key);
    if (threadIdx.x < 3) all[threadIdx.x] = 0;
    plan_count(key, q, below, equal);
    int start = 0, cnt = 0, place = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        start += below[w];
        if (w < wave) place += equal[w];
        cnt += equal[w];
    }
    if (segments > 1) {  // k_plan_count's numbers of the other segments
        for (int s = threadIdx.x; s < segments; s += kPlanThreads) {
            const int2 v = p.seen[(long)q * segments + s];
            atomicAdd(&all[0], v.x);
            atomicAdd(&all[1], v.y);
            if (s < (int)blockIdx.y) atomicAdd(&all[2], v.y);
        }
        __syncthreads();
        start = all[0];
        cnt = all[1];
        place += all[2];
    }
    place += start;
    const long first = (long)blockIdx.y * kPlanRows + wave * (64 * kPlanLoads) + lane;
#pragma unroll
    for (int it = 0; it < kPlanLoads; ++it) {
        const unsigned long long m = __ballot(key[it] == q);
        if (key[it] == q) p.perm[place + __popcll(m & ((1ull << lane) - 1))] = (int)(first + it * 64);
        place += __popcll(m);
    }
    if (blockIdx.y != 0) return;
    write_tiles(q, p.a, start, cnt, p.tile, false, p.tiles, p.ntiles, 0, nullptr);
    // Slots by the chunks' entries, or, where that takes fewer, from 2 start / chunk on: an adapter of several
    // chunks has more than `chunk` rows, of which floor(2 cnt / chunk) is no less than ceil(cnt / chunk).
    if (p.chunks != nullptr) write_tiles(q, p.a, start, cnt, p.chunk, true, p.chunks, p.nchunks, p.slot_by_entry ? start / p.chunk + q : 2 * start / p.chunk, p.merge);
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

// 16 bytes that this kernel's caller reads next, from memory: past the caches (a plain store
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

struct Rows {  // where the rows of a tile come from
    const Tile* tiles;   // nullable: tile i is row i
    const int* perm;
    const int* ids; long ids_stride; int a;
};

__device__ __forceinline__ Tile tile_at(const Rows& w, int i)
{
    if (w.tiles != nullptr) return w.tiles[i];
    return Tile{adapter_of(w.ids, w.ids_stride, i, w.a), i, 1, -1};
}

// Which of `count` tiles (or chunks) and of `parts` parts of its work block x takes.  Blocks go to the
// 8 XCDs in turn, so an XCD gets an eighth of the tiles side by side, each with all its
// parts one after the other.  Neighbouring tiles share adapters, which that XCD's L2
// then holds.  And the parts are stretches of the rows' columns: were the blocks that run
// together all at one stretch, rows a multiple of 4 KB apart would put them on a quarter of
// the memory channels (k_outer_split at 16,384 x 4,096, rank 64: 298 us that way).
// The grid has ceil(count / 8) * 8 * parts blocks.
struct Place { int tile, part; };
__device__ __forceinline__ Place place_of(unsigned x, int count, int parts)
{
    const int per = (count + 7) / 8, i = x >> 3;
    return Place{(int)(x & 7) * per + i / parts, i % parts};
}
// For k_outer, whose chunks share nothing and differ in length: a chunk's parts on all XCDs.
__device__ __forceinline__ Place place_spread(unsigned x, int parts)
{
    const int chunk = x / parts;
    return Place{chunk, (int)(x + chunk) % parts};
}
inline unsigned place_grid(int count, int parts) { return (unsigned)((count + 7) / 8) * 8u * (unsigned)parts; }

__device__ __forceinline__ int row_at(const Rows& w, int place) { return w.tiles != nullptr ? w.perm[place] : place; }

// ---- rows to ranks ----

template <typename T>
struct ShrinkArgs {
    Rows rows;
    const T* v; long ld_v;       // [n x w]
    const T* M; long sa, ld;     // [a][r][w]
    int w, r; long n;
    int ntiles, splits;          // splits of w
    float* part; int rp;         // [splits][n places][rp], rp = the ranks in whole 16s
};

// part[s][place][t] = sum over the s-th part of the columns of M_q[t] v_row, 0 from r on.  A
// block takes RT * 16 rows of one adapter and NB * 16 ranks; its four waves take the columns
// in turn, 128 bytes of each row at a time, and add up their sums at the end, so that rows
// and adapter are read once and go to the matrix cores straight from memory.  The columns
// are split over blocks where there are too few tiles to keep the memory busy.
//
// Bound by the reading: 8,192 bf16 rows of 4,096, rank 16, take 18 us (3.6 TB/s).  At rank 64
// (16,384 rows, 64 adapters: 58 us) an adapter is as long as its tile's rows, first read
// from memory, and the waves' sums take 7 us to meet.
template <typename T, int RT, int NB>
__global__ __launch_bounds__(256) void k_shrink(ShrinkArgs<T> p)
{
    constexpr int KS = 128 / sizeof(T);
    __shared__ float sum[2][RT * 16][NB * 16 + 1];
    const Place at = place_of(blockIdx.x, p.ntiles, p.splits);
    if (at.tile >= p.ntiles) return;
    const Tile t = tile_at(p.rows, at.tile);
    if (t.q < 0 || t.q >= p.rows.a) return;
    const int lane = threadIdx.x & 63, wave = wave_index(), l16 = lane & 15, g = lane >> 4;
    const int rank0 = blockIdx.z * (NB * 16);
    const T* v[RT];
    const T* m[NB];
#pragma unroll
    for (int i = 0; i < RT; ++i) v[i] = p.v + (long)row_at(p.rows, t.start + min(i * 16 + l16, t.cnt - 1)) * p.ld_v + g * kVec<T>;
#pragma unroll
    for (int b = 0; b < NB; ++b) m[b] = p.M + t.q * p.sa + (long)min(rank0 + b * 16 + l16, p.r - 1) * p.ld + g * kVec<T>;
    f32x4 acc[RT][NB];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[i][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int steps = (p.w + KS - 1) / KS;
    const int s0 = (int)((long)steps * at.part / p.splits), count = (int)((long)steps * (at.part + 1) / p.splits) - s0;
    const int full = p.w / KS;
    for (int k = wave; k < count; k += 4) {
        const int s = s0 + k;
        Vec<T> x[RT][2], y[NB][2];
        if (s < full) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < RT; ++i) x[i][h] = load16(v[i] + (long)s * KS + h * (KS / 2));
#pragma unroll
                for (int b = 0; b < NB; ++b) y[b][h] = load16(m[b] + (long)s * KS + h * (KS / 2));
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int left = p.w - (s * KS + h * (KS / 2) + g * kVec<T>);
#pragma unroll
                for (int i = 0; i < RT; ++i) x[i][h] = load_part(v[i] + (long)s * KS + h * (KS / 2), left);
#pragma unroll
                for (int b = 0; b < NB; ++b) y[b][h] = load_part(m[b] + (long)s * KS + h * (KS / 2), left);
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
    float* out = p.part + ((long)at.part * p.n + t.start) * p.rp;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = i * 16 + g * 4 + e;
            if (row >= t.cnt) continue;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int rank = rank0 + b * 16 + l16;
                if (rank < p.rp) out[row * p.rp + rank] = rank < p.r ? acc[i][b][e] : 0.f;
            }
        }
}

// ---- ranks to rows ----

// v = hi + mid + lo, exactly down to bf16's smallest steps: 8 bits each of the 24 of an fp32.  A
// low-rank value enters products of bf16 matrix cores as three bf16, so that these are
// fp32's; with two, which leave out up to 2^-17 |v|, one bf16 result in 700 came out a step
// off its nearest.
__device__ __forceinline__ void split3(float v, bf16& hi, bf16& mid, bf16& lo)
{
    hi = (bf16)v;
    const float rest = __builtin_isfinite((float)hi) ? v - (float)hi : 0.f;  // an infinity stays one
    mid = (bf16)rest;
    lo = (bf16)(rest - (float)mid);
}

// b[j] = element j of the eight vectors a[0 .. 7]: an 8 x 8 transposition in registers.
__device__ __forceinline__ void transpose8(const Vec<bf16>* a, Vec<bf16>* b)
{
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned x = __builtin_bit_cast(u32x4, a[2 * e])[j / 2], y = __builtin_bit_cast(u32x4, a[2 * e + 1])[j / 2];
            w[e] = __builtin_amdgcn_perm(y, x, j % 2 ? 0x07060302u : 0x05040100u);
        }
        b[j] = __builtin_bit_cast(Vec<bf16>, w);
    }
}

template <typename T>
struct ExpandArgs {
    Rows rows; int ntiles, parts;            // parts: blocks a tile
    const float* part; int splits, rp; long n;   // k_shrink's
    const T* M; long sa, ld;                 // [a][r][w]
    const float* gates; long gates_stride; const float* scales;
    const T* base; long ld_base;             // nullable
    T* out; long ld_out;
    int w, r;
    float* low;                              // nullable: [n x r], the splits' sum (0 for a row without an adapter)
    // backward (else null): the forward call's low, and its products with the splits' sum
    const float* dot; float* dgates;         // dgates[i] = s_q <low_i, dot_i>, nullable
    bf16* low_t; bf16* dot_t; long ld_t;     // f low and f dot for k_outer_split, nullable: [3][r][ld_t], by place
};

// What k_expand keeps of a tile's low-rank rows: f low as three bf16 (bf16 rows) or as it is.
template <typename T, int RT, int KP>
struct LowTile {
    static constexpr bool kSplit = false;
    float v[RT * 16][KP + 4];
    __device__ void set(int i, int k, f32x4 x) { *reinterpret_cast<f32x4*>(&v[i][k]) = x; }
};
template <int RT, int KP>
struct LowTile<bf16, RT, KP> {
    static constexpr bool kSplit = true;
    bf16 v[RT * 16][3 * KP + 8];
    __device__ void set(int i, int k, f32x4 x)
    {
        bf16 __attribute__((ext_vector_type(4))) hi, mid, lo;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            bf16 a, b, c;
            split3(x[u], a, b, c);
            hi[u] = a;
            mid[u] = b;
            lo[u] = c;
        }
        __builtin_memcpy(&v[i][k], &hi, 8);
        __builtin_memcpy(&v[i][KP + k], &mid, 8);
        __builtin_memcpy(&v[i][2 * KP + k], &lo, 8);
    }
};

// A row's own numbers in a tile, which its first threads look up.
template <int RT>
struct __align__(16) TileRows {
    int row[RT * 16];
    float f[RT * 16];
};

template <typename T, int RT>
__device__ __forceinline__ void stage_rows(const ExpandArgs<T>& p, const Tile& t, bool has, float sc, TileRows<RT>& R)
{
    if (threadIdx.x < RT * 16) {
        const int row = row_at(p.rows, t.start + min((int)threadIdx.x, t.cnt - 1));
        R.row[threadIdx.x] = row;
        R.f[threadIdx.x] = has ? (p.gates ? p.gates[(long)row * p.gates_stride] : 1.f) * sc : 0.f;
    }
}

// The splits' sums of a tile's low-rank rows, four ranks a thread at a time, times f into L.
// store: the sums themselves, by row; dgates: s_q times their products with dot.
// Barriers: one before this writes L and reads R, the caller's one after it.
template <typename T, int RT, int KP>
__device__ __forceinline__ void stage_low(const ExpandArgs<T>& p, const Tile& t, bool has, float sc, LowTile<T, RT, KP>& L, const TileRows<RT>& R,
                                          float* store, float* dgates)
{
    constexpr int Q = KP / 4, ALL = RT * 16 * Q, PER = (ALL + 255) / 256;
    f32x4 s[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (has)
        for (int c = 0; c < p.splits; ++c) {
            const float* part = p.part + ((long)c * p.n + t.start) * p.rp;
#pragma unroll
            for (int u = 0; u < PER; ++u) {
                const int idx = threadIdx.x + u * 256, i = idx / Q, k = idx % Q * 4;
                if (idx < ALL && i < t.cnt && k < p.rp) s[u] += *reinterpret_cast<const f32x4*>(part + i * p.rp + k);
            }
        }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const int idx = threadIdx.x + u * 256, i = idx / Q, k = idx % Q * 4;
        if (idx >= ALL) break;
        L.set(i, k, s[u] * R.f[i]);
        if (store == nullptr && dgates == nullptr) continue;
        const long row = R.row[i];
        float d = 0.f;
#pragma unroll
        for (int v = 0; v < 4; ++v)
            if (i < t.cnt && k + v < p.r) {
                if (store != nullptr) store[row * p.r + k + v] = s[u][v];
                if (dgates != nullptr && has) d += s[u][v] * p.dot[row * p.r + k + v];
            }
        if (dgates != nullptr) {
#pragma unroll
            for (int off = 1; off < Q; off <<= 1) d += __shfl_xor(d, off, 64);
            if (k == 0 && i < t.cnt) dgates[row] = has ? d * sc : 0.f;
        }
    }
}

// f dot into L, dot [n x r] by row (R is there).
template <typename T, int RT, int KP>
__device__ __forceinline__ void stage_dot(const ExpandArgs<T>& p, const Tile& t, LowTile<T, RT, KP>& L, const TileRows<RT>& R)
{
    constexpr int Q = KP / 4, ALL = RT * 16 * Q;
#pragma unroll 4
    for (int idx = threadIdx.x; idx < ALL; idx += 256) {
        const int i = idx / Q, k = idx % Q * 4;
        const float* at = p.dot + (long)R.row[i] * p.r + k;
        f32x4 s;
#pragma unroll
        for (int v = 0; v < 4; ++v) s[v] = i < t.cnt && k + v < p.r ? at[v] : 0.f;
        L.set(i, k, s * R.f[i]);
    }
}

// A tile's rows of L by rank, for k_outer_split.
template <typename T, int RT, int KP>
__device__ __forceinline__ void store_by_rank(const ExpandArgs<T>& p, const Tile& t, const LowTile<T, RT, KP>& L, bf16* out)
{
    if constexpr (LowTile<T, RT, KP>::kSplit)
        for (int idx = threadIdx.x; idx < 3 * p.r * RT * 16; idx += 256) {
            const int i = idx % (RT * 16), k = idx / (RT * 16), part = k / p.r;  // k: the ranks' hi, then their mid, then lo
            if (i < t.cnt) out[k * p.ld_t + t.start + i] = L.v[i][part * KP + k - part * p.r];
        }
}

// The rows of a 16-row tile that a lane brings and takes: g * 4 .. + 3 of it.
struct Quad { int row[4]; };

// Their base: 16 bytes of each row a lane, 256 bytes of a row side by side.
template <typename T, bool FULL>
__device__ __forceinline__ void fetch_base(const ExpandArgs<T>& p, const Quad& q, int c, Vec<T>* y)
{
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const T* from = p.base + q.row[e] * p.ld_base + c;
        y[e] = p.base == nullptr ? Vec<T>{} : FULL ? load16(from) : load_part(from, p.w - c);
    }
}

// A wave's M_q and first 16 rows' base of the 16 * kVec columns from c0 on.  A lane brings kVec
// columns of eight ranks at a time: for bf16 g * 8 .. + 7 of every 32 (of the 16, where there
// are no more), else g * 4 .. + 3 of every 16, two such.
template <typename T, int KP>
__device__ __forceinline__ void fetch_stretch(const ExpandArgs<T>& p, int q, bool has, const Quad& rows, int c0, Vec<T> (*m)[8], Vec<T>* y)
{
    constexpr int V = kVec<T>;
    if (c0 >= p.w) return;
    const int lane = threadIdx.x & 63, g = lane >> 4, c = c0 + (lane & 15) * V;
    const bool full = c0 + 16 * V <= p.w;
    if (has) {
#pragma unroll
        for (int b = 0; b < (KP + 31) / 32; ++b) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int rank = std::is_same_v<T, bf16> ? (KP == 16 ? (g & 1) * 8 + e : b * 32 + g * 8 + e) : b * 32 + e / 4 * 16 + g * 4 + e % 4;
                const T* from = p.M + q * p.sa + (long)min(rank, p.r - 1) * p.ld + c;
                m[b][e] = full ? load16(from) : load_part(from, p.w - c);
                if (rank >= p.r) m[b][e] = Vec<T>{};
            }
        }
    }
    if (full)
        fetch_base<T, true>(p, rows, c, y);
    else
        fetch_base<T, false>(p, rows, c, y);
}

// M_q's ranks as the matrix cores want them.
template <typename T, int KP>
__device__ __forceinline__ void turn_ranks(Vec<T> (*m)[8])
{
    if constexpr (std::is_same_v<T, bf16>) {
#pragma unroll
        for (int b = 0; b < (KP + 31) / 32; ++b) {
            Vec<T> x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = m[b][e];
            transpose8(x, m[b]);
        }
    }
}

// The wave's rows and columns of a tile: out = base + L M, with the first 16 rows' base in
// y[0].  A lane ends up with kVec columns (from c on) of four rows.
//
// bf16: lanes hold eight ranks of eight columns each, transposed in registers, so M goes
// to the matrix cores without a detour; L enters as three bf16 (where the ranks fill half of
// a product of 32: hi and mid side by side, M twice, then lo beside zeros).  Other types: fp32 matrix
// cores, four ranks at a time, which need M by columns as it lies and L unrounded.
// FULL: all the columns exist.
//
// The sums start from the base where its type rounds at 2^-8 or 2^-11 anyway; in fp32 they
// would then round at the base's size once for every four ranks, so it is added last.
template <typename T, int RT, int KP, bool FULL>
__device__ __forceinline__ void expand_columns(const ExpandArgs<T>& p, const Tile& t, const Vec<T> (*m)[8], const LowTile<T, RT, KP>& L, const TileRows<RT>& R,
                                               Vec<T> (*y)[4], int c, bool has)
{
    constexpr int V = kVec<T>;
    constexpr bool kBaseFirst = sizeof(T) == 2;
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4, left = p.w - c;
    auto quad = [&](int i) { return *reinterpret_cast<const Quad*>(&R.row[i * 16 + g * 4]); };
    Quad now = quad(0);
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        if (i * 16 >= t.cnt) break;
        Quad next = now;
        if (i + 1 < RT) {
            next = quad(i + 1);
            fetch_base<T, FULL>(p, next, c, y[(i + 1) & 1]);
        }
        f32x4 acc[V];
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][e] = kBaseFirst ? to_f(y[i & 1][e][j]) : 0.f;
        if (has) {
            if constexpr (LowTile<T, RT, KP>::kSplit) {
                auto part = [&](int k) { return *reinterpret_cast<const Vec<T>*>(&L.v[i * 16 + l16][k]); };
                if constexpr (KP == 16) {
                    const Vec<T> hi_mid = part(g * 8), lo = g < 2 ? part(32 + g * 8) : Vec<T>{};
#pragma unroll
                    for (int j = 0; j < V; ++j) acc[j] = mfma16(hi_mid, m[0][j], acc[j]);
#pragma unroll
                    for (int j = 0; j < V; ++j) acc[j] = mfma16(lo, m[0][j], acc[j]);
                } else {
#pragma unroll
                    for (int b = 0; b < KP / 32; ++b)
#pragma unroll
                        for (int of = 0; of < 3; ++of) {
                            const Vec<T> some = part(of * KP + b * 32 + g * 8);
#pragma unroll
                            for (int j = 0; j < V; ++j) acc[j] = mfma16(some, m[b][j], acc[j]);
                        }
                }
            } else {
#pragma unroll
                for (int b = 0; b < KP / 16; ++b) {
                    const f32x4 lo = *reinterpret_cast<const f32x4*>(&L.v[i * 16 + l16][b * 16 + g * 4]);
#pragma unroll
                    for (int s = 0; s < 4; ++s)
#pragma unroll
                        for (int j = 0; j < V; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(lo[s], to_f(m[b / 2][b % 2 * 4 + s][j]), acc[j], 0, 0, 0);
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (i * 16 + g * 4 + e >= t.cnt) continue;
            Vec<T> z;
#pragma unroll
            for (int j = 0; j < V; ++j) z[j] = from_f<T>(kBaseFirst ? acc[j][e] : to_f(y[i & 1][e][j]) + acc[j][e]);
            T* o = p.out + now.row[e] * p.ld_out + c;
            if (FULL || left >= V)
                stream16(o, z);
            else
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (j < left) o[j] = z[j];
        }
        now = next;
    }
}

// out_row = base_row + f_row low_row M_q.  A block takes RT * 16 rows of one adapter and
// every parts-th stretch of 64 * kVec columns, 16 * kVec a wave, which keeps M_q for them in
// registers.  KP: the ranks, rounded up.
//
// Bound by the base read and the result written: 8,192 bf16 rows of 4,096, rank 16, take 27 us
// (5.0 TB/s), 16,384 at rank 64 82 us (3.3 TB/s: the adapters' reads and the low-rank rows
// staged in every block come on top), 105 backward with those written by rank.
template <typename T, int RT, int KP, bool BACK>
__global__ __launch_bounds__(256, KP <= 32 ? 3 : KP <= 64 ? 2 : 1) void k_expand(ExpandArgs<T> p)
{
    constexpr int V = kVec<T>;
    using Low = LowTile<T, RT, KP>;
    __shared__ __align__(16) Low L;
    __shared__ TileRows<RT> R;
    const Place at = place_of(blockIdx.x, p.ntiles, p.parts);
    if (at.tile >= p.ntiles) return;
    const Tile t = tile_at(p.rows, at.tile);
    if (t.q < 0) return;
    const bool has = t.q < p.rows.a;
    const int lane = threadIdx.x & 63, wave = wave_index(), l16 = lane & 15, g = lane >> 4;
    const float sc = has && p.scales ? p.scales[t.q] : 1.f;
    Quad row0;
#pragma unroll
    for (int e = 0; e < 4; ++e) row0.row[e] = row_at(p.rows, t.start + min(g * 4 + e, t.cnt - 1));
    constexpr int NM = (KP + 31) / 32;
    Vec<T> m[NM][8], y[2][4];
    int c0 = (at.part * 4 + wave) * 16 * V;
    fetch_stretch<T, KP>(p, t.q, has, row0, c0, m, y[0]);
    const bool first = at.part == 0;
    stage_rows<T, RT>(p, t, has, sc, R);
    stage_low<T, RT, KP>(p, t, has, sc, L, R, first ? p.low : nullptr, BACK && first ? p.dgates : nullptr);
    __syncthreads();
    if (BACK && Low::kSplit && first && has && p.low_t != nullptr) store_by_rank<T, RT, KP>(p, t, L, p.low_t);
    while (c0 < p.w) {
        if (has) turn_ranks<T, KP>(m);
        if (c0 + 16 * V <= p.w)
            expand_columns<T, RT, KP, true>(p, t, m, L, R, y, c0 + l16 * V, has);
        else
            expand_columns<T, RT, KP, false>(p, t, m, L, R, y, c0 + l16 * V, has);
        c0 += p.parts * 64 * V;
        fetch_stretch<T, KP>(p, t.q, has, row0, c0, m, y[0]);
    }
    if (BACK && Low::kSplit && has && p.dot_t != nullptr && at.part == p.parts - 1) {
        __syncthreads();
        stage_dot<T, RT, KP>(p, t, L, R);
        __syncthreads();
        store_by_rank<T, RT, KP>(p, t, L, p.dot_t);
    }
}

// One row a block (and 128 * kVec of its columns): both products at once, low_row computed
// anew by every block of the row.  Eight waves share its columns, several steps in flight.
// One bf16 row of 1,024, rank 8, takes 6.4 us launch after launch (two kernels: 6.8), 64 of them
// 6.8 (7.6): the launch and the three trips to memory, one after another, bound it.
constexpr int kDirectThreads = 512;
template <typename T, int KP, bool BACK>
__global__ __launch_bounds__(kDirectThreads) void k_direct(ExpandArgs<T> p, const T* v, long ld_v, const T* D, long sa, long ld, int w)
{
    constexpr int V = kVec<T>, NB = KP / 16, KS = 128 / sizeof(T), W = kDirectThreads / 64, U = NB == 1 ? 4 : NB == 2 ? 2 : 1;
    __shared__ __align__(16) LowTile<T, 1, KP> L;
    __shared__ TileRows<1> R;
    __shared__ __align__(16) float sum[W][KP];
    const int i = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
    const Tile t{adapter_of(p.rows.ids, p.rows.ids_stride, i, p.rows.a), i, 1, -1};
    const bool has = t.q < p.rows.a;
    const int lane = threadIdx.x & 63, wave = wave_index(), l16 = lane & 15, g = lane >> 4;
    const float sc = has && p.scales ? p.scales[t.q] : 1.f;
    if (threadIdx.x < 16) {
        R.row[threadIdx.x] = i;
        R.f[threadIdx.x] = has ? (p.gates ? p.gates[i * p.gates_stride] : 1.f) * sc : 0.f;
    }
    Vec<T> m[(KP + 31) / 32][8], y[2][4];
    const int c0 = (part * W + wave) * 16 * V;
    fetch_stretch<T, KP>(p, t.q, has, Quad{{i, i, i, i}}, c0, m, y[0]);
    if (has) {
        const T* x = v + i * ld_v + g * V;
        const T* d[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) d[b] = D + t.q * sa + (long)min(b * 16 + l16, p.r - 1) * ld + g * V;
        f32x4 acc[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int steps = (w + KS - 1) / KS, full = w / KS;
        for (int k = wave; k < steps; k += W * U) {
            Vec<T> a[U][2], b[U][NB][2];
            if (k + (U - 1) * W < full) {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int at = (k + u * W) * KS + h * (KS / 2);
                        a[u][h] = load16(x + at);
#pragma unroll
                        for (int n = 0; n < NB; ++n) b[u][n][h] = load16(d[n] + at);
                    }
            } else {  // the steps past the row, and the last one's columns past it, as 0
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int at = (k + u * W) * KS + h * (KS / 2), left = w - at - g * V;
                        a[u][h] = load_part(x + at, left);
#pragma unroll
                        for (int n = 0; n < NB; ++n) b[u][n][h] = load_part(d[n] + at, left);
                    }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int n = 0; n < NB; ++n) acc[n] = mfma16(a[u][h], b[u][n][h], acc[n]);
        }
        if (g == 0)  // all sixteen rows of the product are this row
#pragma unroll
            for (int b = 0; b < NB; ++b) sum[wave][b * 16 + l16] = acc[b][0];
    }
    __syncthreads();
    if (threadIdx.x < KP / 4) {
        const int k = threadIdx.x * 4;
        f32x4 s{0.f, 0.f, 0.f, 0.f};
        if (has)
#pragma unroll
            for (int u = 0; u < W; ++u) s += *reinterpret_cast<const f32x4*>(&sum[u][k]);
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (k + e >= p.r) s[e] = 0.f;
            if (part == 0 && k + e < p.r) {
                if (p.low != nullptr) p.low[(long)i * p.r + k + e] = s[e];
                if (BACK && p.dgates != nullptr && has) dot += s[e] * p.dot[(long)i * p.r + k + e];
            }
        }
        L.set(0, k, s * R.f[0]);
        if (BACK && part == 0 && p.dgates != nullptr) {
#pragma unroll
            for (int off = 1; off < KP / 4; off <<= 1) dot += __shfl_xor(dot, off, 64);
            if (threadIdx.x == 0) p.dgates[i] = has ? dot * sc : 0.f;
        }
    }
    __syncthreads();
    if (c0 >= p.w) return;
    if (has) turn_ranks<T, KP>(m);
    if (c0 + 16 * V <= p.w)
        expand_columns<T, 1, KP, true>(p, t, m, L, R, y, c0 + l16 * V, has);
    else
        expand_columns<T, 1, KP, false>(p, t, m, L, R, y, c0 + l16 * V, has);
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
    const Tile* chunks;                      // nullable: chunk q is all of adapter q's rows, at most kMaxChunk, found here
    const int2* merge; const int* perm; int a, r;
    const int* ids; long ids_stride; int n;  // for finding them
    const float* gates; long gates_stride; const float* scales;
    OuterSide<T> side[2];                    // parts below `split`: side 0
    int split, parts;                        // parts: of both sides' columns
};

constexpr int kMaxChunk = 512;

// dM_q[t] += sum over a chunk's rows of f_row low_row[t] v_row.  A block takes the chunk
// and 16 * kVec columns, its four waves every fourth quad of rows; both operands go to the
// fp32 matrix cores as they lie in memory.  For fp32 and fp16 rows, and for calls of few
// rows; 4,099 fp16 rows of 777 and 1,001, rank 5, take 14 us, most of it latency (16 MB).
template <typename T, int NB>
__global__ __launch_bounds__(256) void k_outer(OuterArgs<T> p)
{
    constexpr int V = kVec<T>, W = 16 * V;
    __shared__ int rows[kMaxChunk];
    __shared__ float fac[kMaxChunk];
    extern __shared__ char lds[];
    float* sum = reinterpret_cast<float*>(lds);  // [2][NB * 16][W]
    const Place at = place_spread(blockIdx.x, p.parts);
    Tile t{at.tile, 0, 0, -1};
    if (p.chunks != nullptr) t = p.chunks[at.tile];
    if (t.q < 0) return;
    const bool second = at.part >= p.split;
    const OuterSide<T>& s = p.side[second];
    const int c0 = (at.part - (second ? p.split : 0)) * W, rank0 = blockIdx.z * (NB * 16);
    const int lane = threadIdx.x & 63, wave = wave_index(), l16 = lane & 15, g = lane >> 4;
    const float sc = p.scales ? p.scales[t.q] : 1.f;
    if (p.chunks != nullptr) {
        for (int i = threadIdx.x; i < t.cnt; i += 256) rows[i] = p.perm[t.start + i];
    } else {
        __shared__ int found[kMaxChunk / 64];
        unsigned long long m[kMaxChunk / 256];
#pragma unroll
        for (int u = 0; u < kMaxChunk / 256; ++u) {
            const int i = u * 256 + threadIdx.x;
            m[u] = __ballot(i < p.n && p.ids[(long)min(i, p.n - 1) * p.ids_stride] == t.q);
            if (lane == 0) found[u * 4 + wave] = __popcll(m[u]);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kMaxChunk / 256; ++u) {
            int place = __popcll(m[u] & ((1ull << lane) - 1));
            for (int w = 0; w < u * 4 + wave; ++w) place += found[w];
            if (m[u] >> lane & 1) rows[place] = u * 256 + threadIdx.x;
        }
        for (int w = 0; w < kMaxChunk / 64; ++w) t.cnt += found[w];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < t.cnt; i += 256) fac[i] = (p.gates ? p.gates[(long)rows[i] * p.gates_stride] : 1.f) * sc;
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

// The same for bf16 rows on the bf16 matrix cores, 32 rows at a time: a lane's eight rows of
// eight columns are transposed in registers, and f low comes by rank as three bf16 (k_expand's
// low_t, dot_t) through LDS, 64 rows at a time, for the block's four waves.  A block takes a
// chunk and 512 columns, a wave 128 of them.  16,384 rows x 4,096 twice, rank 64: 104 us, of
// which the third part takes 11; with each wave's own loads of f low, 16 lines of 64 bytes
// apiece, it took half as long again.
struct SplitSide {
    const bf16* low;                         // [3][r][ld_t]: hi, mid, lo
    const bf16* v; long ld_v; int w;
    bf16* dM; float* part;
};
struct OuterSplitArgs {
    const Tile* chunks; const int* perm; int r; long ld_t;
    SplitSide side[2]; int split, parts;
};

template <int NB>
__global__ __launch_bounds__(256, 2) void k_outer_split(OuterSplitArgs p)
{
    constexpr int R = NB * 16;
    constexpr int S = 8 * 256 / R;  // rows staged at once: 16 bytes of each part a thread
    __shared__ __align__(16) int rows[kMaxChunk + 32];
    __shared__ __align__(16) bf16 low[2][3][R][S + 8];  // twice: hi, mid and lo of S rows by rank
    const Place at = place_spread(blockIdx.x, p.parts);
    const Tile t = p.chunks[at.tile];
    if (t.q < 0) return;
    const bool second = at.part >= p.split;
    const SplitSide s = second ? p.side[1] : p.side[0];
    const int lane = threadIdx.x & 63, wave = wave_index(), l16 = lane & 15, g = lane >> 4;
    const int c0 = ((at.part - (second ? p.split : 0)) * 4 + wave) * 128, rank0 = blockIdx.z * R;
    const bool active = c0 < s.w, full = c0 + 128 <= s.w;
    const int c = c0 + l16 * 8, left = s.w - c;
    const int seg = threadIdx.x % (S / 8), line = threadIdx.x / (S / 8);
    const bf16* from = s.low + min(rank0 + line, p.r - 1) * p.ld_t + t.start + seg * 8;
    Vec<bf16> mine[3];
    auto fetch_low = [&](int i) {
#pragma unroll
        for (int of = 0; of < 3; ++of) {
            mine[of] = load16(from + of * p.r * p.ld_t + i);
            if (i + S > t.cnt)  // the places past the chunk belong to other adapters
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (i + seg * 8 + e >= t.cnt) mine[of][e] = (bf16)0.f;
        }
    };
    auto stage_low = [&](int turn) {
#pragma unroll
        for (int of = 0; of < 3; ++of) *reinterpret_cast<Vec<bf16>*>(&low[turn][of][line][seg * 8]) = mine[of];
    };
    Vec<bf16> v[8];
    auto fetch_rows = [&](int i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bf16* from = s.v + (long)rows[i + g * 8 + e] * s.ld_v + c;
            v[e] = full ? load16(from) : load_part(from, left);
        }
    };
    if (t.cnt > 0) fetch_low(0);
    for (int i = threadIdx.x; i < ((t.cnt + 31) & ~31); i += 256) rows[i] = p.perm[t.start + min(i, t.cnt - 1)];
    __syncthreads();
    if (active && t.cnt > 0) fetch_rows(0);
    f32x4 acc[NB][8];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[b][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < t.cnt; i += S) {
        const int turn = i / S & 1;
        stage_low(turn);
        __syncthreads();  // one is enough: the other half is written again only after the next
        if (i + S < t.cnt) fetch_low(i + S);
        if (!active) continue;
#pragma unroll
        for (int h = 0; h < S / 32; ++h) {
            const int k = i + h * 32;
            if (k >= t.cnt) break;
            if (k + 32 > t.cnt)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (k + g * 8 + e >= t.cnt) v[e] = Vec<bf16>{};
            Vec<bf16> x[8];
            transpose8(v, x);
            if (k + 32 < t.cnt) fetch_rows(k + 32);  // on their way while these are multiplied
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int of = 0; of < 3; ++of) {
                    const Vec<bf16> f = *reinterpret_cast<const Vec<bf16>*>(&low[turn][of][b * 16 + l16][h * 32 + g * 8]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) acc[b][j] = mfma16(f, x[j], acc[b][j]);
                }
        }
    }
    if (!active) return;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int rank = rank0 + b * 16 + g * 4 + e;
            if (rank >= p.r) continue;
            if (t.slot >= 0) {
                float* o = s.part + ((long)t.slot * p.r + rank) * s.w + c;
                float z[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) z[j] = acc[b][j][e];
                if (full)
                    __builtin_memcpy(o, z, 32);
                else
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j < left) o[j] = z[j];
            } else {
                bf16* o = s.dM + ((long)t.q * p.r + rank) * s.w + c;
                Vec<bf16> z;
#pragma unroll
                for (int j = 0; j < 8; ++j) z[j] = (bf16)acc[b][j][e];
                if (full)
                    stream16(o, z);
                else
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j < left) o[j] = z[j];
            }
        }
}

// The chunks' sums of the adapters that have several, added in chunk order: blockIdx.z and
// every gridDim.z-th such adapter.  Four values a thread (VEC), eight chunks in flight.
// Bound by the partial sums' reading: 14 us at 16,384 rows of 4,096 twice, rank 64.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void k_outer_merge(OuterArgs<T> p)
{
    constexpr int N = VEC ? 4 : 1;
    __shared__ int4 some[256];  // adapter, first slot, chunks
    __shared__ int found[4];
    const OuterSide<T>& s = p.side[blockIdx.y];
    const long size = (long)p.r * s.w;
    const int lane = threadIdx.x & 63, wave = wave_index();
    for (int q0 = 0; q0 < p.a; q0 += 256) {
        const int q = q0 + threadIdx.x;
        const int2 m = q < p.a ? p.merge[q] : make_int2(0, 0);
        const unsigned long long several = __ballot(m.y != 0);
        if (lane == 0) found[wave] = __popcll(several);
        __syncthreads();
        int at = __popcll(several & ((1ull << lane) - 1)), count = 0;
        for (int w = 0; w < 4; ++w) {
            if (w < wave) at += found[w];
            count += found[w];
        }
        if (m.y != 0) some[at] = make_int4(q, m.x, m.y, 0);
        __syncthreads();
        for (int j = blockIdx.z; j < count; j += gridDim.z) {
            const int4 m = some[j];
            const float* part = s.part + m.y * size;
            T* out = s.dM + m.x * size;
            for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * N; i < size; i += (long)gridDim.x * 256 * N) {
                float v[N] = {};
                for (int k = 0; k < m.z; k += 8) {
                    float x[8][N];
#pragma unroll
                    for (int u = 0; u < 8; ++u) __builtin_memcpy(x[u], part + min(k + u, m.z - 1) * size + i, 4 * N);
#pragma unroll
                    for (int u = 0; u < 8; ++u)
#pragma unroll
                        for (int e = 0; e < N; ++e) v[e] += k + u < m.z ? x[u][e] : 0.f;
                }
#pragma unroll
                for (int e = 0; e < N; ++e) out[i + e] = from_f<T>(v[e]);
            }
        }
        __syncthreads();
    }
}

// ---- host ----

// Whether every row is its own tile, without a sort: the call then has a launch less and reads
// an adapter once a row instead of once a tile.  us without and with the sort, bf16, d = o:
//   d = 1,024, rank 16:  256 rows 7, 15;  512 rows 12, 14
//   d = 4,096, rank 16:   64 rows 9, 15;  128 rows 14, 16;  256 rows 17, 16
//   d = 4,096, rank 64:   64 rows 15, 19;  128 rows 24, 20
bool is_direct(long n, int d, int o, int rp)
{
    return n <= kMaxChunk && (size_t)n * rp * ((size_t)d + o) <= (n <= 64 ? size_t(1) << 25 : size_t(1) << 24);
}

// Whether such a call's two products are one launch, every block of a row computing its
// low-rank vector anew: where that reads little, 32 MiB of M in all and 128 KiB a block (64 KiB
// in fp32, whose matrix instructions take four times as long for it).  A second launch and its
// workspace also cost the caller 4 us on the host (300 fp32 rows of 768, rank 16, forward and
// backward from Python: 31.6 us with one, 36.2 with two).  Launch after launch, d = o, two kernels
// and one:
//   bf16:  1 row of 256, rank 64: 8.7, 4.9;   64 of 1,024, rank 8: 7.6, 6.8;   256 of 1,024, rank 8: 8.7, 6.7
//         64 of 1,024, rank 64: 10.9, 9.4;    64 of 4,096, rank 8: 9.5, 7.5;   512 of 512, rank 32: 10.2, 6.9
//         96 of 2,048, rank 32: 10.5, 9.0;   128 of 2,048, rank 32: 11.0, 10.0
//   fp16: 512 of 1,024, rank 8: 11.2, 9.1;   256 of 2,048, rank 8: 11.3, 8.4
//   fp32: 256 of 1,024, rank 8: 10.1, 9.1;   512 of 512, rank 32: 15.8, 12.2
// Within the limits and slower on the device, for the host's sake, where more than 256 blocks
// (one a CU) take a second turn:
//   bf16: 288 of 1,024, rank 8: 9.7, 11.7;   320 of 1,536, rank 8: 10.7, 15.4; 160 of 1,536, rank 32: 11.0, 12.8
//   fp32: 288 of 768, rank 8: 10.4, 11.9
// Beyond the limits:
//   bf16:  72 of 4,096, rank 8: 11.1, 13.3;   96: 10.6, 13.5;   1 of 4,096, rank 64: 10.9, 20.3;   64 of 2,048, rank 64: 11.7, 14.5
//   fp16:  96 of 4,096, rank 8: 11.0, 11.5
//   fp32:   1 of 1,024, rank 32: 8.1, 8.9;    48 of 4,096, rank 8: 10.3, 22.4
bool is_fused(long n, int d, int o, int rp, int type)
{
    const size_t wide = d > o ? d : o, es = elem_size(type), cols = kDirectThreads / 4 * (16 / es);  // columns a block
    const size_t row = rp * wide * es;
    return rp <= 64 && row <= (size_t(type == kF32 ? 64 : 128) << 10) && n * ((wide + cols - 1) / cols) * row <= size_t(32) << 20;
}

size_t up16(size_t b) { return (b + 15) & ~size_t(15); }

struct Layout {
    long n; int a, r;
    bool direct, fused, split;            // fused: k_direct; split: k_outer_split
    int tile, ntiles, nchunks, chunk, segments;
    int slots; bool slot_by_entry;        // partial sums of chunks
    long full_tiles;                      // of n rows, were they all of one adapter
    int rp;
    int down_splits, up_splits;           // of d (t = D x) and of o (u = U dy)
    long ld_t;
    size_t seen, perm, tiles, chunks, merge, part, low, low_t, dot_t, dpart, upart, bytes;
};

// Parts of the columns, so that enough blocks read at once while a wave still has two
// steps of its own.
int split_count(long tiles, int w, int type, int zs)
{
    if (tiles < 1) tiles = 1;
    const long steps = (w + 128 / (int)elem_size(type) - 1) / (128 / (int)elem_size(type));
    long s = (512 + tiles * zs - 1) / (tiles * zs);
    const long most = steps / 8;
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s > 8 ? 8 : s);
}

// Columns in k_expand's stretches.
int stretches(int w, int type)
{
    const int columns = 64 * (16 / (int)elem_size(type));
    return (w + columns - 1) / columns;
}

// Rows a tile: as many as leave about three blocks a CU on the average of both widths, for each
// tile reads its adapter anew.
int tile_rows(long n, int d, int o, int type)
{
    int t = 64;
    while (t > 16 && (n + t - 1) / t * (stretches(d, type) + stretches(o, type)) < 2 * 768) t /= 2;
    return t;
}

// Blocks a k_expand tile: each stages the tile's low-rank rows again, so no more than
// about 1,024 blocks in all.
int part_count(long tiles, int w, int type)
{
    const long most = stretches(w, type), want = tiles > 0 ? (1024 + tiles - 1) / tiles : most;
    return (int)(want < 1 ? 1 : want > most ? most : want);
}

// Rows a k_outer block sums up: as many as leave a block a CU (k_outer_split) or two (k_outer,
// whose waves share a chunk), for every cut costs a partial matrix written and read.
int chunk_rows(long n, int d, int o, int a, int type)
{
    const int cols = type == kBF16 ? 512 : 16 * (16 / (int)elem_size(type)), blocks = type == kBF16 ? 256 : 512;
    const long parts = (d + cols - 1) / cols + (o + cols - 1) / cols;
    int c = kMaxChunk;
    while (c > 64 && (n / c + (a < n / c ? a : n / c)) * parts < blocks) c /= 2;
    return c;
}

Layout layout(int type, long n, int d, int o, int r, int a, AdaptCall call)
{
    const bool backward = call == kAdaptBackward;
    Layout L{};
    L.n = n; L.a = a; L.r = r;
    L.rp = (r + 15) & ~15;
    L.direct = is_direct(n, d, o, L.rp);
    // k_direct's blocks of a row each read all of x while others write out already
    L.fused = L.direct && call != kAdaptInX && is_fused(n, d, o, L.rp, type);
    L.split = type == kBF16 && !L.direct;
    L.tile = L.direct ? 1 : tile_rows(n, d, o, type);
    L.full_tiles = (n + L.tile - 1) / L.tile;
    L.ntiles = L.direct ? (int)n : (int)(n / L.tile + a + 1);
    L.segments = (int)((n + kPlanRows - 1) / kPlanRows);
    if (L.segments < 1) L.segments = 1;
    L.chunk = chunk_rows(n, d, o, a, type);
    L.nchunks = (int)(n / L.chunk) + a;
    L.slot_by_entry = L.nchunks <= 2 * n / L.chunk;
    L.slots = n <= L.chunk ? 0 : L.slot_by_entry ? L.nchunks : (int)(2 * n / L.chunk);
    L.ld_t = ((n + 63) & ~63l) + 160;  // 128 rows past the last (k_outer_split's most at once); not a power of two apart
    const int zs = (r + 63) / 64;
    L.down_splits = split_count(L.full_tiles, d, type, zs);
    L.up_splits = split_count(L.full_tiles, o, type, zs);
    size_t at = 0;
    auto take = [&](size_t& where, size_t bytes) { where = at; at += up16(bytes); };
    if (!L.direct) {
        take(L.seen, L.segments > 1 ? (size_t)L.segments * (a + 1) * sizeof(int2) : 0);
        take(L.perm, (size_t)n * 4);
        take(L.tiles, (size_t)L.ntiles * sizeof(Tile));
    }
    if (!L.fused) take(L.part, (size_t)(backward ? L.up_splits : L.down_splits) * n * L.rp * 4);
    if (backward && L.direct) take(L.low, (size_t)n * r * 4);
    if (backward && !L.direct) {
        take(L.chunks, (size_t)L.nchunks * sizeof(Tile));
        take(L.merge, (size_t)a * sizeof(int2));
        take(L.low, L.split ? 0 : (size_t)n * r * 4);
        take(L.low_t, L.split ? (size_t)3 * r * L.ld_t * 2 : 0);
        take(L.dot_t, L.split ? (size_t)3 * r * L.ld_t * 2 : 0);
        take(L.dpart, (size_t)L.slots * r * d * 4);
        take(L.upart, (size_t)L.slots * r * o * 4);
    }
    L.bytes = at;
    return L;
}

hipError_t launch_plan(const Layout& L, const int* ids, long ids_stride, char* ws, bool backward, hipStream_t s)
{
    const PlanArgs p{ids, ids_stride, (int)L.n, L.a, reinterpret_cast<int2*>(ws + L.seen), reinterpret_cast<int*>(ws + L.perm),
                     reinterpret_cast<Tile*>(ws + L.tiles), L.ntiles, L.tile,
                     backward ? reinterpret_cast<Tile*>(ws + L.chunks) : nullptr, L.nchunks,
                     backward ? reinterpret_cast<int2*>(ws + L.merge) : nullptr, L.chunk, L.slot_by_entry};
    const dim3 grid(L.a + 1, L.segments);
    if (L.segments > 1) SKM_TRY_LAUNCH(k_plan_count, grid, kPlanThreads, 0, s, p);
    return launch(k_plan, grid, kPlanThreads, 0, s, p);
}

template <typename T, int RT>
hipError_t launch_shrink(const ShrinkArgs<T>& p, hipStream_t s)
{
    const dim3 grid(place_grid(p.ntiles, p.splits), 1, (p.r + 63) / 64);
    if (p.r <= 16) return launch(k_shrink<T, RT, 1>, grid, 256, 0, s, p);
    if (p.r <= 32) return launch(k_shrink<T, RT, 2>, grid, 256, 0, s, p);
    return launch(k_shrink<T, RT, 4>, grid, 256, 0, s, p);
}

template <typename T, int RT, bool BACK>
hipError_t launch_expand(const ExpandArgs<T>& p, hipStream_t s)
{
    const dim3 grid(place_grid(p.ntiles, p.parts));
    if (p.r <= 16) return launch(k_expand<T, RT, 16, BACK>, grid, 256, 0, s, p);
    if (p.r <= 32) return launch(k_expand<T, RT, 32, BACK>, grid, 256, 0, s, p);
    if (p.r <= 64) return launch(k_expand<T, RT, 64, BACK>, grid, 256, 0, s, p);
    return launch(k_expand<T, RT, 128, BACK>, grid, 256, 0, s, p);
}

// The row's own kernel, or both of a tile's.
template <typename T, bool BACK>
hipError_t launch_direct(const ShrinkArgs<T>& sh, ExpandArgs<T> ex, hipStream_t s)
{
    ex.parts = (ex.w + kDirectThreads / 4 * kVec<T> - 1) / (kDirectThreads / 4 * kVec<T>);
    const dim3 grid((unsigned)(ex.n * ex.parts));
    if (ex.r <= 16) return launch(k_direct<T, 16, BACK>, grid, kDirectThreads, 0, s, ex, sh.v, sh.ld_v, sh.M, sh.sa, sh.ld, sh.w);
    if (ex.r <= 32) return launch(k_direct<T, 32, BACK>, grid, kDirectThreads, 0, s, ex, sh.v, sh.ld_v, sh.M, sh.sa, sh.ld, sh.w);
    return launch(k_direct<T, 64, BACK>, grid, kDirectThreads, 0, s, ex, sh.v, sh.ld_v, sh.M, sh.sa, sh.ld, sh.w);
}

// f(row tiles of 16 a tile)
template <typename F>
hipError_t with_tile(int tile, F&& f)
{
    if (tile == 64) return f(std::integral_constant<int, 4>{});
    if (tile == 32) return f(std::integral_constant<int, 2>{});
    return f(std::integral_constant<int, 1>{});
}

}  // namespace

bool adapt_fits(int type, long n, int d, int o, int r, int a)
{
    const Layout L = layout(type, n, d, o, r, a, kAdaptBackward);
    const size_t tiles = ((size_t)L.full_tiles + a + 8) * (size_t)(L.down_splits > L.up_splits ? L.down_splits : L.up_splits);
    const size_t wide = ((size_t)L.full_tiles + a + 8) * (size_t)(part_count(L.full_tiles, d, type) > part_count(L.full_tiles, o, type) ? part_count(L.full_tiles, d, type) : part_count(L.full_tiles, o, type));
    const size_t cols = 16 * (16 / elem_size(type)), chunks = (L.direct ? (size_t)a : (size_t)n / L.chunk + a) * ((d + cols - 1) / cols + (o + cols - 1) / cols);
    const size_t most = size_t(1) << 24;  // blocks of 256 threads in a grid that has less than 2^32 threads
    return tiles < most && wide < most && chunks < most && L.segments < 65536;
}

size_t adapt_workspace(int type, long n, int d, int o, int r, int a, AdaptCall call) { return layout(type, n, d, o, r, a, call).bytes; }

hipError_t launch_adapt(const AdaptArgs& a, hipStream_t s)
{
    if (a.n == 0) return hipSuccess;
    const Layout L = layout(a.type, a.n, a.d, a.o, a.r, a.a, a.in_x ? kAdaptInX : kAdapt);
    if (!L.direct) {
        const hipError_t e = launch_plan(L, a.ids, a.ids_stride, a.ws, false, s);
        if (e != hipSuccess) return e;
    }
    const Rows rows{L.direct ? nullptr : reinterpret_cast<const Tile*>(a.ws + L.tiles), reinterpret_cast<const int*>(a.ws + L.perm), a.ids, a.ids_stride, a.a};
    float* part = reinterpret_cast<float*>(a.ws + L.part);
    return with_type(a.type, [&](auto tag) {
        using T = decltype(tag);
        const ShrinkArgs<T> sh{rows, (const T*)a.x, a.ld_x, (const T*)a.down, a.down_sa, a.down_ld, a.d, a.r, a.n, L.ntiles, L.down_splits, part, L.rp};
        const ExpandArgs<T> ex{rows, L.ntiles, part_count(L.full_tiles, a.o, a.type), part, L.down_splits, L.rp, a.n, (const T*)a.up, a.up_sa, a.up_ld, a.gates, a.gates_stride, a.scales,
                               (const T*)a.base, a.ld_base, (T*)a.out, a.ld_out, a.o, a.r, a.low, nullptr, nullptr, nullptr, nullptr, 0};
        if (L.fused) return launch_direct<T, false>(sh, ex, s);
        return with_tile(L.tile, [&](auto rt) {
            const hipError_t e = a.a > 0 ? launch_shrink<T, rt.value>(sh, s) : hipSuccess;
            return e != hipSuccess ? e : launch_expand<T, rt.value, false>(ex, s);
        });
    });
}

hipError_t launch_adapt_back(const AdaptBackArgs& a, hipStream_t s)
{
    const Layout L = layout(a.type, a.n, a.d, a.o, a.r, a.a, kAdaptBackward);
    if (a.n == 0 && a.a == 0) return hipSuccess;
    if (!L.direct) {
        const hipError_t e = launch_plan(L, a.ids, a.ids_stride, a.ws, true, s);
        if (e != hipSuccess) return e;
    }
    const Rows rows{L.direct ? nullptr : reinterpret_cast<const Tile*>(a.ws + L.tiles), reinterpret_cast<const int*>(a.ws + L.perm), a.ids, a.ids_stride, a.a};
    const Tile* chunks = L.direct ? nullptr : reinterpret_cast<const Tile*>(a.ws + L.chunks);
    float* part = reinterpret_cast<float*>(a.ws + L.part);
    float* u = L.split ? nullptr : reinterpret_cast<float*>(a.ws + L.low);
    bf16* u_t = L.split ? reinterpret_cast<bf16*>(a.ws + L.low_t) : nullptr;
    bf16* t_t = L.split ? reinterpret_cast<bf16*>(a.ws + L.dot_t) : nullptr;
    float* dpart = reinterpret_cast<float*>(a.ws + L.dpart);
    float* upart = reinterpret_cast<float*>(a.ws + L.upart);
    return with_type(a.type, [&](auto tag) {
        using T = decltype(tag);
        if (a.n > 0) {
            const ShrinkArgs<T> sh{rows, (const T*)a.dy, a.ld_dy, (const T*)a.up, a.up_sa, a.up_ld, a.o, a.r, a.n, L.ntiles, L.up_splits, part, L.rp};
            const ExpandArgs<T> ex{rows, L.ntiles, part_count(L.full_tiles, a.d, a.type), part, L.up_splits, L.rp, a.n, (const T*)a.down, a.down_sa, a.down_ld,
                                   a.gates, a.gates_stride, a.scales, (const T*)a.base, a.ld_base, (T*)a.dx, a.ld_dx, a.d, a.r, u, a.low, a.dgates, u_t, t_t,
                                   L.ld_t};
            const hipError_t e = L.fused ? launch_direct<T, true>(sh, ex, s) : with_tile(L.tile, [&](auto rt) {
                const hipError_t e = a.a > 0 ? launch_shrink<T, rt.value>(sh, s) : hipSuccess;
                return e != hipSuccess ? e : launch_expand<T, rt.value, true>(ex, s);
            });
            if (e != hipSuccess) return e;
        }
        if (a.a == 0) return hipSuccess;
        constexpr int W = 16 * kVec<T>;
        const OuterArgs<T> ou{chunks, reinterpret_cast<const int2*>(a.ws + L.merge), rows.perm, a.a, a.r, a.ids, a.ids_stride, (int)a.n,
                              a.gates, a.gates_stride, a.scales,
                              {{u, (const T*)a.x, a.ld_x, a.d, (T*)a.ddown, dpart}, {a.low, (const T*)a.dy, a.ld_dy, a.o, (T*)a.dup, upart}},
                              (a.d + W - 1) / W, (a.d + W - 1) / W + (a.o + W - 1) / W};
        if (L.split) {
            if constexpr (std::is_same_v<T, bf16>) {
                const OuterSplitArgs os{chunks, rows.perm, a.r, L.ld_t,
                                        {{u_t, (const T*)a.x, a.ld_x, a.d, (T*)a.ddown, dpart}, {t_t, (const T*)a.dy, a.ld_dy, a.o, (T*)a.dup, upart}},
                                        (a.d + 511) / 512, (a.d + 511) / 512 + (a.o + 511) / 512};
                const unsigned grid = (unsigned)(L.nchunks * os.parts);
                if (a.r <= 16)
                    SKM_TRY_LAUNCH(k_outer_split<1>, dim3(grid), 256, 0, s, os);
                else if (a.r <= 32)
                    SKM_TRY_LAUNCH(k_outer_split<2>, dim3(grid), 256, 0, s, os);
                else
                    SKM_TRY_LAUNCH(k_outer_split<4>, dim3(grid, 1, (a.r + 63) / 64), 256, 0, s, os);
            }
        } else {
            const unsigned grid = (unsigned)((L.direct ? a.a : L.nchunks) * ou.parts);
            if (a.r <= 16)
                SKM_TRY_LAUNCH((k_outer<T, 1>), dim3(grid), 256, 2 * 16 * W * 4, s, ou);
            else
                SKM_TRY_LAUNCH((k_outer<T, 2>), dim3(grid, 1, (a.r + 31) / 32), 256, 2 * 32 * W * 4, s, ou);
        }
        if (L.direct || L.n <= L.chunk) return hipSuccess;  // one chunk an adapter
        const long most = (long)a.r * (a.d > a.o ? a.d : a.o);
        const bool vec = ((long)a.r * a.d % 4 == 0) && ((long)a.r * a.o % 4 == 0);
        const long blocks = (most / (vec ? 4 : 1) + 255) / 256;
        const dim3 grid((unsigned)(blocks < 256 ? blocks : 256), 2, a.a < 8 ? a.a : 8);
        return vec ? launch(k_outer_merge<T, true>, grid, 256, 0, s, ou) : launch(k_outer_merge<T, false>, grid, 256, 0, s, ou);
    });
}

}  // namespace skm
