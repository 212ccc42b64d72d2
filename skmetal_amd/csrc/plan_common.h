// plan_common.h -- rows in the order of their adapters (or experts): the sort in front of
// the products of adapt_kernels.hip and feed_kernels.hip.  Each of the two has its own copy.
#pragma once

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

}  // namespace
}  // namespace skm
