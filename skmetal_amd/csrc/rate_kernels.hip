// rate_kernels.hip -- log probabilities of given targets under rows of scores, with the rows'
// entropy and their largest scores, and the gradient of the scores.
//
//   m = max_j z_j,  S = sum_j exp(z_j - m),  T = sum_j exp(z_j - m) (z_j - m)
//   lse = m + ln S        log p_j = z_j - lse        H = -sum_j p_j log p_j = ln S - T / S
//   dz_j = p_j (g_lse - g_t - g_H (log p_j + H)) + [j = t] g_t
// with g_t the gradient of the target's log p.  A score of -inf or NaN is excluded (p = 0); +inf makes its
// row's results NaN, as inf - inf is.
//
// One pass over the scores each way.  A row's scores are split over blocks where there are few
// rows; a part leaves (m, S, T) and its k largest scores, which a second launch joins.
#include "experts_common.h"

namespace skm {
namespace {

constexpr int kMaxTop = kRateMaxK;
constexpr float kLowest = -3.402823466e38f;
// exp(-200) is 0 in fp32: as a lower bound it also turns the differences of excluded scores (-inf, and NaN, which
// fmaxf leaves for the other operand) into probability 0 without a comparison.
constexpr float kZero = -200.f;

// A score and its place as a whole number, ordered by (score, lowest place first); -0 as 0, 0 for an excluded one.
__device__ __forceinline__ unsigned long long key_of(float z, unsigned j)
{
    if (!(z > -__builtin_inff())) return 0;
    const unsigned u = __float_as_uint(z + 0.f);
    return (unsigned long long)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (0xffffffffu - j);
}
__device__ __forceinline__ float score_of(unsigned long long key)
{
    const unsigned o = (unsigned)(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ int place_of(unsigned long long key) { return (int)(0xffffffffu - (unsigned)key); }

// The softmax's sums relative to a maximum.
struct Sums {
    float m, s, t;  // the largest score (kLowest: none yet), sum e, sum e (z - m), e = exp(z - m)
    __device__ __forceinline__ void raise(float to)
    {
        const float by = fminf(to - m, -kZero), c = exp_of(-by);
        t = c * (t - by * s);
        s *= c;
        m = to;
    }
    __device__ __forceinline__ void add(float z)
    {
        const float d = fmaxf(z - m, kZero), e = exp_of(d);
        s += e;
        t = fmaf(e, d, t);
    }
    __device__ __forceinline__ void join(const Sums& o)
    {
        const float to = fmaxf(m, o.m), a = fminf(to - m, -kZero), b = fminf(to - o.m, -kZero), ca = exp_of(-a), cb = exp_of(-b);
        t = ca * (t - a * s) + cb * (o.t - b * o.s);
        s = ca * s + cb * o.s;
        m = to;
    }
};

// The wave's sums joined, on every lane: relative to its maximum at once, so that a lane takes one exponential.
__device__ __forceinline__ Sums joined(Sums v)
{
    float m = v.m;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
    v.raise(m);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        v.s += __shfl_xor(v.s, x);
        v.t += __shfl_xor(v.t, x);
    }
    return v;
}

// The wave's k-th largest key (1: fewer lanes hold one), on every lane; equal keys are 0.  Bit by bit: a bit belongs to it
// if k lanes reach the number with that bit set, a comparison and a ballot each.  A score of 16 bits shows in the upper 16
// (bf16) or 19 (fp16) alone; the places are asked only where more than k lanes reach the score.  Where just
// k do, the score without its spare bits is returned: no lane's key lies between it and the k-th largest.
// (Every key against every other: 131,072 x 256 bf16 with the 4 largest 139 us, so 99.)
template <typename T>
__device__ __forceinline__ unsigned long long kth_largest(unsigned long long key, int k)
{
    constexpr int SPARE = std::is_same<T, float>::value ? 0 : std::is_same<T, _Float16>::value ? 13 : 16;
    const unsigned o = (unsigned)(key >> 32);
    unsigned t = 0;
#pragma unroll
    for (int b = 31; b >= SPARE; --b) {
        const unsigned with = t | 1u << b;
        t = __popcll(__ballot(o >= with)) >= k ? with : t;
    }
    if (t == 0) return 1;
    if (__popcll(__ballot(o >= t)) == k) return (unsigned long long)t << 32;
    static_assert(kRateMaxV <= 1 << 22, "places in 22 bits");
    const unsigned places = (1u << 22) - 1, place = o >= t ? (o - t) >> SPARE ? places : (unsigned)key & places : 0;
    unsigned at = 0;
#pragma unroll
    for (int b = 21; b >= 0; --b) {
        const unsigned with = at | 1u << b;
        at = __popcll(__ballot(place >= with)) >= k ? with : at;
    }
    if (!(t >> 31)) t |= (1u << SPARE) - 1;  // a negative score's bits are inverted
    return (unsigned long long)t << 32 | ~places | at;
}

// How many of the list's `found` keys are larger.
__device__ __forceinline__ int rank_of(const unsigned long long* list, int found, unsigned long long key)
{
    int place = 0;
#pragma unroll 8
    for (int j = 0; j < found; ++j) place += list[j] > key;
    return place;
}

struct RateOut {
    const int* targets; long target_stride; int v;
    float* log_probs; float* entropy; float* lse; float* rest;  // [n]
    int k; int* top; float* top_log_probs;                      // [n x k]
};

// A row's results from its sums, by one lane.
template <typename T>
__device__ __forceinline__ void finish(const RateOut& o, long row, const Sums& v, const T* z)
{
    const float log_s = logf(v.s);
    const int t = o.targets[row * o.target_stride];
    const bool inf = v.m == __builtin_inff(), none = v.s == 0.f;
    const float lse = none && !inf ? -__builtin_inff() : v.m + log_s;
    // lse to twice fp32's bits, for the gradient: what the sum's rounding left out
    const float part = lse - v.m, rest = (v.m - (lse - part)) + (log_s - part);
    o.lse[row] = inf ? v.m : lse;
    o.rest[row] = none || inf ? 0.f : rest;
    o.entropy[row] = inf ? __builtin_nanf("") : none ? 0.f : fmaxf(log_s - v.t / v.s, 0.f);
    float lp = 0.f;
    if (t >= 0 && t < o.v) {
        const float zt = to_f(z[t]);
        lp = inf ? __builtin_nanf("") : zt > -__builtin_inff() ? (zt - v.m) - log_s : -__builtin_inff();
    }
    o.log_probs[row] = lp;
}

// Place `at` of a row's largest scores.
__device__ __forceinline__ void put_top(const RateOut& o, long row, int at, unsigned long long key, const Sums& v)
{
    o.top[row * o.k + at] = key ? place_of(key) : -1;
    o.top_log_probs[row * o.k + at] = v.m == __builtin_inff() ? __builtin_nanf("") : key ? (score_of(key) - v.m) - logf(v.s) : -__builtin_inff();
}

template <typename T>
struct RateArgs {
    const T* z; long ld;
    long n; int splits;         // parts of a row
    int part;                   // scores a part, a multiple of a block's step
    RateOut out;
    Sums* sums;                 // [n][splits], several parts only
    unsigned long long* keys;   // [n][splits][k]
};

// One part of a row on NT lanes: 16 bytes a lane, UN at once.
//
// The k largest: every lane knows the first place of its own largest score, at no cost but a comparison every 16 bytes.
// The k-th largest of a wave's lanes is a lower bound for the k-th largest of all.  Of the wave that has the
// largest of these bounds k lanes hold scores that reach it, of the others fewer, so a second look at the part
// (from the caches) finds at most k of a lane's share in each wave, and hardly more than k in all as a rule; these
// are ranked by counting.  (With a bound over all lanes through LDS a part of 4,096 scores took 11 us, not 7.)
// The second look reads several vectors at once and passes over those whose largest score is below: 2,000 x 128,256 bf16
// with the 4 largest 145 us (without them 96, a vector at a time and key by key 213).
template <typename T, int NT, bool TOP>
__global__ __launch_bounds__(NT) void k_rate(RateArgs<T> p)
{
    constexpr int V = kVec<T>, UN = 4, STEP = NT * V;
    const long row = blockIdx.x / p.splits;
    const int split = (int)(blockIdx.x % p.splits);
    const T* z = p.z + row * p.ld;
    const int lo = split * p.part, hi = min(p.out.v, lo + p.part), tid = threadIdx.x;
    Sums s{kLowest, 0.f, 0.f};
    int first = -1;  // where a vector held the lane's largest score first
    auto take = [&](const float* x, int at) {
        float top = x[0];
#pragma unroll
        for (int j = 1; j < V; ++j) top = fmaxf(top, x[j]);
        if (top > s.m || (first < 0 && top == kLowest)) {
            s.raise(top);
            first = at;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) s.add(x[j]);
    };
    auto scores = [&](int at, float* x) {  // -inf past the part's end
        if (at + V <= hi) {
            const Vec<T> raw = load16(z + at);
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = to_f(raw[j]);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = at + j < hi ? to_f(z[at + j]) : -__builtin_inff();
        }
    };
    int at = lo + tid * V;
    for (; at + (UN - 1) * STEP + V <= hi; at += UN * STEP) {
        Vec<T> raw[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) raw[u] = load16(z + at + u * STEP);
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            float x[V];
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = to_f(raw[u][j]);
            take(x, at + u * STEP);
        }
    }
    for (; at < hi; at += STEP) {
        float x[V];
        scores(at, x);
        take(x, at);
    }

    __shared__ Sums wave_sums[NT / 64];
    extern __shared__ unsigned long long list[];  // TOP: list_of() keys
    __shared__ unsigned long long bounds[NT / 64];
    __shared__ int count;
    Sums all = joined(s);
    if (NT > 64 && (tid & 63) == 0) wave_sums[tid >> 6] = all;
    if constexpr (TOP) {
        unsigned long long mine = 0;
        if (first >= 0) {
            float x[V];
            scores(first, x);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const unsigned long long key = key_of(x[j], first + j);
                mine = key > mine ? key : mine;
            }
        }
        unsigned long long least = kth_largest<T>(mine, p.out.k);
        if (NT > 64 && (tid & 63) == 0) bounds[tid >> 6] = least;
        if (tid == 0) count = 0;
        __syncthreads();
        if (NT > 64)
#pragma unroll
            for (int w = 0; w < NT / 64; ++w) least = bounds[w] > least ? bounds[w] : least;
        if (mine >= least) {
            const float bound = score_of(least);  // NaN for 1: every key counts
            auto collect = [&](const float* x, int from) {
                float top = x[0];
#pragma unroll
                for (int j = 1; j < V; ++j) top = fmaxf(top, x[j]);
                if (top < bound) return;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const unsigned long long key = key_of(x[j], from + j);
                    if (key >= least) list[atomicAdd(&count, 1)] = key;
                }
            };
            at = lo + tid * V;
            for (; at + (UN - 1) * STEP + V <= hi; at += UN * STEP) {
                Vec<T> raw[UN];
#pragma unroll
                for (int u = 0; u < UN; ++u) raw[u] = load16(z + at + u * STEP);
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    float x[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) x[j] = to_f(raw[u][j]);
                    collect(x, at + u * STEP);
                }
            }
            for (; at < hi; at += STEP) {
                float x[V];
                scores(at, x);
                collect(x, at);
            }
        }
    }
    if (NT > 64 || TOP) __syncthreads();
    if (NT > 64) {
        all = wave_sums[0];
#pragma unroll
        for (int w = 1; w < NT / 64; ++w) all.join(wave_sums[w]);
    }
    const bool whole = p.splits == 1;
    if (tid == 0) {
        if (whole)
            finish(p.out, row, all, z);
        else
            p.sums[row * p.splits + split] = all;
    }
    if constexpr (TOP) {
        const int k = p.out.k, found = count;
        unsigned long long* keys = p.keys + (row * p.splits + split) * k;
        for (int i = tid; i < max(found, k); i += NT) {  // places that no score takes: 0, behind the others
            const unsigned long long key = i < found ? list[i] : 0;
            const int place = i < found ? rank_of(list, found, key) : i;
            if (place >= k) continue;
            if (whole)
                put_top(p.out, row, place, key, all);
            else
                keys[place] = key;
        }
    }
}

// The parts of a row joined, by a wave.  Of the parts' keys, each part's largest first, those count that reach the
// largest of the parts' last ones: a lower bound for the k-th largest of all, which at most k - 1 keys of
// every other part exceed.
template <typename T>
__global__ __launch_bounds__(64) void k_rate_join(RateArgs<T> p)
{
    __shared__ unsigned long long list[kRateSplits * kMaxTop];
    const long row = blockIdx.x;
    const int lane = threadIdx.x, k = p.out.k;
    Sums all{kLowest, 0.f, 0.f};
    unsigned long long least = 1;
    for (int i = lane; i < p.splits; i += 64) {
        all.join(p.sums[row * p.splits + i]);
        if (k > 0) {
            const unsigned long long last = p.keys[(row * p.splits + i) * k + k - 1];
            least = last > least ? last : least;
        }
    }
    all = joined(all);
    if (lane == 0) finish(p.out, row, all, p.z + row * p.ld);
    if (k == 0) return;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        const unsigned long long other = __shfl_xor(least, x);
        least = other > least ? other : least;
    }
    int found = 0;
    for (int i0 = 0; i0 < p.splits * k; i0 += 64) {
        const unsigned long long key = i0 + lane < p.splits * k ? p.keys[row * p.splits * k + i0 + lane] : 0;
        const unsigned long long who = __ballot(key >= least);
        if (key >= least) list[found + __popcll(who & ((1ull << lane) - 1))] = key;
        found += __popcll(who);
    }
    __syncthreads();
    for (int i = lane; i < max(found, k); i += 64) {
        const unsigned long long key = i < found ? list[i] : 0;
        const int place = i < found ? rank_of(list, found, key) : i;
        if (place < k) put_top(p.out, row, place, key, all);
    }
}

template <typename T>
struct RateBackArgs {
    const T* z; long ld;
    const int* targets; long target_stride;
    const float* lse; const float* rest; const float* entropy;
    const float* dlog; const float* dent; const float* dlse;  // nullable
    T* dz; long ld_dz;
    int v, splits, part;
};

template <typename T, int NT>
__global__ __launch_bounds__(NT) void k_rate_back(RateBackArgs<T> p)
{
    constexpr int V = kVec<T>, UN = 4, STEP = NT * V;
    const long row = blockIdx.x / p.splits;
    const int lo = (int)(blockIdx.x % p.splits) * p.part, hi = min(p.v, lo + p.part);
    const T* z = p.z + row * p.ld;
    T* dz = p.dz + row * p.ld_dz;
    int t = p.targets[row * p.target_stride];
    if (t < 0 || t >= p.v) t = -1;
    const float lse = p.lse[row], rest = p.rest[row], ent = p.entropy[row];
    const float gt = p.dlog != nullptr && t >= 0 ? p.dlog[row] : 0.f;
    const float gh = p.dent != nullptr ? p.dent[row] : 0.f, gl = (p.dlse != nullptr ? p.dlse[row] : 0.f) - gt;
    const bool inf = lse == __builtin_inff();
    const float a = gl - gh * ent;  // dz = p (a - gh log p)
    auto one = [&](float x, int j) {
        const float lp = fmaxf((x - lse) - rest, kZero), e = exp_of(lp);
        float g = e > 0.f ? e * fmaf(-gh, lp, a) : 0.f;
        if (j == t && x > -__builtin_inff()) g += gt;
        return inf && x > -__builtin_inff() ? __builtin_nanf("") : g;
    };
    // Stores of whole lines: the lanes' 16 bytes begin where a line of dz does, and what a row has before its first
    // whole 16 bytes is taken one by one.  1,999 x 50,257 fp32: 158 us (from the row's start: 177).
    constexpr int LINE = 128 / (int)sizeof(T);
    int at = lo - (int)((size_t)(dz + lo) / sizeof(T) % LINE) + (int)threadIdx.x * V;
    if (at < lo) {
        for (int j = max(0, lo - at); j < V && at + j < hi; ++j) dz[at + j] = from_f<T>(one(to_f(z[at + j]), at + j));
        at += STEP;
    }
    for (; at + (UN - 1) * STEP + V <= hi; at += UN * STEP) {
        Vec<T> raw[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) raw[u] = load16(z + at + u * STEP);
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            Vec<T> g;
#pragma unroll
            for (int j = 0; j < V; ++j) g[j] = from_f<T>(one(to_f(raw[u][j]), at + u * STEP + j));
            stream16(dz + at + u * STEP, g);
        }
    }
    for (; at < hi; at += STEP) {
        if (at + V <= hi) {
            const Vec<T> raw = load16(z + at);
            Vec<T> g;
#pragma unroll
            for (int j = 0; j < V; ++j) g[j] = from_f<T>(one(to_f(raw[j]), at + j));
            stream16(dz + at, g);
        } else {
            for (int j = 0; at + j < hi; ++j) dz[at + j] = from_f<T>(one(to_f(z[at + j]), at + j));
        }
    }
}

// Rows of at most this many scores take one wave each.
constexpr int kShort = 2048;

struct Parts {
    int threads, splits, part;
};

// Keys that a part's second look collects at most: k lanes' shares in each wave.  Its LDS follows the shape, so that many
// short rows run at once: 131,072 x 256 bf16 with the 4 largest 139 us, with room for kRateList keys in every block 533.
int list_of(const Parts& c, int type, int k)
{
    const int vec = 16 / (int)elem_size(type), step = c.threads * vec;
    return c.threads / 64 * k * ((c.part + step - 1) / step) * vec;
}

// How a row is cut: parts of at least 4,096 scores, as many as leave about four blocks a CU, at most
// kRateSplits; with the k largest none of more scores than a lane's share of the list allows.
Parts parts_of(long n, int v, int type, int k)
{
    const int vec = 16 / (int)elem_size(type);
    if (v <= kShort) return {64, 1, v};
    long splits = n > 0 ? (1024 + n - 1) / n : 1;
    const long most = (v + 4095) / 4096;
    if (splits > most) splits = most;
    if (splits > kRateSplits) splits = kRateSplits;
    const int longest = k > 0 ? kRateList / (4 * k) / vec * vec * 256 : v;  // k lanes of each of four waves
    const long least = ((long)v + longest - 1) / longest;
    if (splits < least) splits = least;
    const int step = 256 * vec;
    const int part = (int)((((v + splits - 1) / splits + step - 1) / step) * step);
    return {256, (v + part - 1) / part, part};
}

size_t up16(size_t b) { return (b + 15) & ~size_t(15); }

}  // namespace

bool rate_fits(long n, int v, int type, int k)
{
    const Parts c = parts_of(n, v, type, k);
    return c.splits <= kRateSplits && (unsigned long long)n * c.splits * c.threads < 1ull << 32;
}

size_t rate_workspace(long n, int v, int type, int k)
{
    const Parts c = parts_of(n, v, type, k);
    return c.splits == 1 ? 0 : up16((size_t)n * c.splits * sizeof(Sums)) + (size_t)n * c.splits * k * 8;
}

hipError_t launch_rate(const RateCall& a, hipStream_t s)
{
    if (a.n == 0) return hipSuccess;
    const Parts c = parts_of(a.n, a.v, a.type, a.k);
    return with_type(a.type, [&](auto tag) {
        using T = decltype(tag);
        RateArgs<T> p{(const T*)a.z, a.ld, a.n, c.splits, c.part,
                      {a.targets, a.target_stride, a.v, a.log_probs, a.entropy, a.lse, a.rest, a.k, a.top, a.top_log_probs},
                      reinterpret_cast<Sums*>(a.ws), reinterpret_cast<unsigned long long*>(a.ws + up16((size_t)a.n * c.splits * sizeof(Sums)))};
        const dim3 grid((unsigned)(a.n * c.splits));
        const size_t lds = (size_t)list_of(c, a.type, a.k) * 8;  // at most kRateList keys
        const hipError_t e = c.threads == 64 ? (a.k > 0 ? launch(k_rate<T, 64, true>, grid, 64, lds, s, p) : launch(k_rate<T, 64, false>, grid, 64, 0, s, p))
                                             : (a.k > 0 ? launch(k_rate<T, 256, true>, grid, 256, lds, s, p) : launch(k_rate<T, 256, false>, grid, 256, 0, s, p));
        if (e != hipSuccess || c.splits == 1) return e;
        return launch(k_rate_join<T>, dim3((unsigned)a.n), 64, 0, s, p);
    });
}

hipError_t launch_rate_back(const RateBackCall& a, hipStream_t s)
{
    if (a.n == 0) return hipSuccess;
    const Parts c = parts_of(a.n, a.v, a.type, 0);
    return with_type(a.type, [&](auto tag) {
        using T = decltype(tag);
        const RateBackArgs<T> p{(const T*)a.z, a.ld, a.targets, a.target_stride, a.lse, a.rest, a.entropy, a.dlog, a.dent, a.dlse, (T*)a.dz, a.ld_dz, a.v, c.splits, c.part};
        const dim3 grid((unsigned)(a.n * c.splits));
        return c.threads == 64 ? launch(k_rate_back<T, 64>, grid, 64, 0, s, p) : launch(k_rate_back<T, 256>, grid, 256, 0, s, p);
    });
}

}  // namespace skm
