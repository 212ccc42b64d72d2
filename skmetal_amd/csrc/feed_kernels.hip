// feed_kernels.hip -- the gated feed-forward block of every row's experts.
//
// Row i goes to the experts q_ij = chosen[i][j], j < k (none outside [0, a)), with the
// weights w_ij; a slot is one such pair.  With expert q's matrices P, Q [f x d] and R [o x f]:
//   g = P x_i, u = Q x_i, h = w act(g) u        out_i = base_i + sum_j R h
// and from dy_i, the gradient of out_i:
//   e = R^T dy_i       dw_ij = <e, act(g) u>     dg = w e u act'(g), du = w e act(g)
//   dx_i = base_i + sum_j P^T dg + Q^T du
//   dP = sum dg x_i^T, dQ = sum du x_i^T, dR = sum dy_i h^T        over the slots of q
//
// k_plan first puts the slots of each expert side by side, cut into tiles of one expert.  Six
// matrix products follow, all by one kernel, k_product: tiles of C = A B^T whose operands are rows in
// memory, either along the sum (a row holds successive terms: "along") or across it (a row holds one term of
// successive results: "across"), gathered through the sort where they are the caller's rows.  Each
// differs in its operands and in what it does with a finished tile.
//
// Between the products h, dg and du are in the rows' type, each rounded once: the matrix cores
// take 16-bit operands, and every result then has one rounding of its terms and one of its own, half
// of what its variance would be with a second rounding.  What enters no product stays fp32: g and u
// (kept from the forward pass for the backward one), e, dw, and the k parts of a row's sum.
#include "plan_common.h"

#include <algorithm>

namespace skm {
namespace {

enum Kind : int { kGated, kDown, kHidden, kRows, kGates, kOuts, kKinds };

// 16 bytes of zeros for loads of what does not exist.
__device__ __attribute__((aligned(16))) unsigned g_zeros[4];

// slot / k for slots below 2^30 and k <= 16.
struct ByK {
    unsigned k, mul, shift;
    __device__ __forceinline__ unsigned row(unsigned slot) const { return (unsigned)(((unsigned long long)slot * mul) >> shift); }
};
ByK by_k(int k)
{
    unsigned l = 0;
    while ((1 << l) < k) ++l;
    return ByK{(unsigned)k, (unsigned)(((1ull << (30 + l)) + k - 1) / k), 30 + l};
}

template <typename T>
struct FeedArgs {
    // tiles of slots (row products) or the slots of each expert (gradients of matrices)
    const Tile* tiles; int ntiles, cut; const int* perm; int slots, a;  // each of the tiles cut in `cut`; tiles null: one expert has all slots in their order
    ByK byk;
    // operands
    const T *A, *A2; long lda;
    const T *B, *B2; long sb, ldb, sb2, ldb2;  // expert and row strides
    int M, N, K;                               // of the result and the sum; what the tiles give is 0
    int nm, nn;                                // tiles of M (kGates, kOuts) and N
    // results
    T *h, *dg, *du; long ldh;                  // [slots][ldh], by place
    float* pre;                                // [slots][2][f], by slot; nullable in kGated
    const float* weights; int act;             // weights nullable
    float* dots; int ndots;                    // [slots][ndots] parts of <e, act(g) u>, nullable
    const T* base; long ld_base; T* out; long ld_out;  // k = 1
    float* sums;                               // [splits][slots][N] by slot: k > 1 or several splits
    T *dm, *dm2; float* part;                  // [a][M][N]; partial sums [splits][a][2 where dm2][M][N] where splits > 1
    int splits;                                // of the sum, over blocks
};

// exp(x) for |x| <= 88: the product with log2 e in two parts, so that its rounding does not grow with x.
__device__ __forceinline__ float exp_near(float x)
{
    const float hi = x * 1.44269502162933349609f, lo = fmaf(x, 1.92596299112661746887e-8f, fmaf(x, 1.44269502162933349609f, -hi));
    const float e = __builtin_amdgcn_exp2f(hi);
    return fmaf(e * 0.69314718055994530942f, lo, e);
}

// act(g) and its derivative.  Both products' tiles end in 64 of these a lane: silu takes 13 instructions so, gelu 32 (with the
// library's expf, division and erfcf, which branch, the gated product of 4,096 x 2,048 by 8,192 took 341 us, not 319).
__device__ __forceinline__ float2 activate(float g, int act)
{
    if (act == kSilu) {
        const float t = g < -88.f ? 0.f : __builtin_amdgcn_rcpf(1.f + exp_near(fminf(fmaxf(-g, -88.f), 88.f)));  // 88 e^-88: 5e-37
        return make_float2(g * t, t * fmaf(g, 1.f - t, 1.f));
    }
    if (act == kGelu) {
        // The normal distribution function of -|g| is 0.5 erfc(x), x = |g| / sqrt(2); erfc(x) = t P(t) exp(-x^2) with t = 1 / (1 + x / 2) and P
        // a polynomial fitted at Chebyshev points of t, relative error 1.5e-7, so that the lower tail keeps its bits.
        const float x = fabsf(g) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(fmaf(0.5f, x, 1.f));
        // g^2 in two parts: what its rounding leaves out is up to 2^-25 g^2 of the exponential (65 2^-24 of the result near -13, 7 so)
        const float sq = g * g, near = exp_near(-0.5f * fminf(sq, 175.f));
        const float e = sq > 175.f ? 0.f : fmaf(near * -0.5f, fmaf(g, g, -sq), near);  // 13.2 times the tail there is 7e-39
        constexpr float P[9] = {0.282087684f, 0.282353491f, 0.24326095f, 0.202070117f, -0.0251784418f, 0.2759794f, -0.485384911f, 0.283702582f, -0.0588909127f};
        float q = P[8];
#pragma unroll
        for (int i = 7; i >= 0; --i) q = fmaf(q, t, P[i]);
        const float tail = 0.5f * t * q * e, c = g > 0.f ? 1.f - tail : tail;
        return make_float2(g * c, fmaf(g * 0.39894228040143268f, e, c));
    }
    return g > 0.f ? make_float2(g, 1.f) : make_float2(g != g ? g : 0.f, 0.f);
}

template <typename T> using Quad = T __attribute__((ext_vector_type(4)));

// Four neighbouring elements of a row, of which `left` exist.
template <typename T>
__device__ __forceinline__ void put4(T* p, f32x4 v, int left)
{
    Quad<T> r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = from_f<T>(v[e]);
    if (left >= 4)
        __builtin_memcpy(p, &r, sizeof r);
    else
        for (int e = 0; e < left; ++e) p[e] = r[e];
}
// The same past the caches, for what only a later launch or the backward pass reads: the gated and down products with their sums at
// 8,192 x 2,048, 8 experts, k = 2, take 580 us so, 626 with plain stores (and h, which the next launch reads, past the caches: 592).
__device__ __forceinline__ void stream4(float* p, f32x4 v, int left)
{
    typedef f32x4 Loose __attribute__((aligned(4)));
    if (left >= 4)
        __builtin_nontemporal_store(v, reinterpret_cast<Loose*>(p));
    else
        for (int e = 0; e < left; ++e) p[e] = v[e];
}
template <typename T>
__device__ __forceinline__ f32x4 get4(const T* p, int left)
{
    Quad<T> r{};
    if (left >= 4)
        __builtin_memcpy(&r, p, sizeof r);
    else
        for (int e = 0; e < left; ++e) r[e] = p[e];
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = to_f(r[e]);
    return v;
}

// Read once and never again: past the caches, which leaves them to h, dg and du (kHidden 337 us with plain loads, 320 so).
__device__ __forceinline__ f32x4 once4(const float* p, int left)
{
    typedef f32x4 Loose __attribute__((aligned(4)));
    return left >= 4 ? __builtin_nontemporal_load(reinterpret_cast<const Loose*>(p)) : get4(p, left);
}

// ---- staging ----

// 16 bytes a lane from memory to LDS, a wave's side by side from byte `to` on.  As assembly, for the compiler waits for
// a load of its own builtin before every transposing read of LDS, and so leaves none in flight
// under a step's products.  m0 is as before after it (a reserved register, which no clobber list covers); landed() waits for the load.
__device__ __forceinline__ void to_lds(const void* from, unsigned to)
{
    unsigned kept;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\ts_mov_b32 m0, %0" : "=&s"(kept) : "s"(to), "v"(from) : "memory");
}
__device__ __forceinline__ unsigned lds_offset(char* p) { return (unsigned)(size_t)(__attribute__((address_space(3))) char*)p; }

constexpr int kStepBytes = 64;  // of a row along the sum: terms a step
template <typename T> constexpr int kStep = kStepBytes / (int)sizeof(T);

// How far the 16-byte chunks of term k's row are displaced in an operand across the sum, so that the lanes of a
// read, which take 16 terms at once, find them in different banks.
template <typename T, int CHUNKS>
__device__ __forceinline__ int displaced(int k)
{
    if constexpr (sizeof(T) == 2) return (((k & 3) | ((k >> 3) & 1) << 2) << 1) & (CHUNKS - 1);
    return (((k >> 2) & 3) << 2) & (CHUNKS - 1);
}

// A block's way to an operand's R rows (or columns) of a tile, a step of terms after another: from memory to
// LDS, 16 bytes a lane.  Along the sum a row takes 64 bytes a step, its chunks exchanged by the row's number, so that
// 16 rows' chunks of the same terms lie in different banks; across it a term's row takes
// R elements.  FAST: every chunk is 16 bytes that exist or not, at addresses of 16 bytes; they go to LDS without
// registers between, and those that do not exist come from g_zeros.
template <typename T, bool ALONG, int R, int NT, bool FAST>
struct Stager {
    static constexpr int V = kVec<T>, C = R * 4 / NT, CHUNKS = ALONG ? 4 : R / V;
    static_assert(C * NT == R * 4, "whole chunks a lane");
    const T* p[C];  // the chunks of the next step
    Vec<T> held[FAST ? 1 : C];

    static __device__ __forceinline__ int index(int c) { return c * NT + (int)threadIdx.x; }
    static __device__ __forceinline__ int line(int c) { return index(c) / CHUNKS; }  // row, or term of the step
    static __device__ __forceinline__ int chunk(int c)
    {
        const int l = line(c), s = index(c) % CHUNKS;
        return ALONG ? s ^ ((l >> 1) & 3) : s ^ displaced<T, CHUNKS>(l);
    }
    // across: where a chunk lies in its row, of which `left` elements are the tile's; FAST reads what exists instead of
    // columns that do not, whose results nothing takes
    static __device__ __forceinline__ int column(int c, int left) { return FAST ? min(chunk(c) * V, left - V) : chunk(c) * V; }

    // along: row(i) is the address of row i of the tile (one that exists, also where the tile has no such row)
    template <typename F>
    __device__ __forceinline__ void rows(F&& row)
    {
#pragma unroll
        for (int c = 0; c < C; ++c) p[c] = row(line(c)) + chunk(c) * V;
    }
    // across: `first` is the address of the first term's row, at column 0 of the tile
    __device__ __forceinline__ void terms(const T* first, long ld, int left)
    {
#pragma unroll
        for (int c = 0; c < C; ++c) p[c] = first + line(c) * ld + column(c, left);
    }

    // Chunk c of a step, from `from` where it is there; `to` is the byte of LDS where the wave's chunks of the step go.
    __device__ __forceinline__ void fetch(int c, const T* from, bool there, int left, unsigned to)
    {
        if constexpr (FAST)
            to_lds(there ? (const void*)from : (const void*)g_zeros, to + c * NT * 16);
        else
            held[c] = there && left > 0 ? load_part(from, left) : Vec<T>{};
    }
    __device__ __forceinline__ void settle(char* to)
    {
        if constexpr (!FAST)
#pragma unroll
            for (int c = 0; c < C; ++c) *reinterpret_cast<Vec<T>*>(to + index(c) * 16) = held[c];
    }

    // Chunk c of the step that begins at term k0 of `count`, the first that was not taken yet.
    __device__ __forceinline__ void along(int c, int k0, int count, unsigned to)
    {
        fetch(c, p[c], chunk(c) * V < count - k0, count - k0 - chunk(c) * V, to);
        p[c] += kStep<T>;
    }
    __device__ __forceinline__ void across(int c, int k0, int count, long ld, int left, unsigned to)
    {
        fetch(c, p[c], line(c) < count - k0, left - chunk(c) * V, to);
        p[c] += kStep<T> * ld;
    }
    // The same for gathered rows; `slots`: those of the step's terms, in LDS, or null where they are the places from `place` on.
    __device__ __forceinline__ void gathered(int c, int k0, int count, const int* slots, int place, const ByK& byk, const T* first, long ld, int left, unsigned to)
    {
        const bool there = line(c) < count - k0;
        const int slot = slots != nullptr ? slots[line(c)] : place + line(c);
        fetch(c, first + (long)byk.row((unsigned)slot) * ld + column(c, left), there, left - chunk(c) * V, to);
    }
};

// All but the last LEFT of this wave's loads to LDS have landed (they do in their order): to be followed by a barrier.
template <int LEFT>
__device__ __forceinline__ void landed()
{
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LEFT) : "memory");
}

// ---- fragments: a lane's terms of one row (or column) for a 16 x 16 product ----

template <typename T, bool ALONG, int R>
struct Reader {
    int at, displacement, first;  // `first`: the wave's first of R rows
    __device__ __forceinline__ explicit Reader(int first_row) : first(first_row)
    {
        const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
        if constexpr (ALONG) {
            at = (first + l16) * kStepBytes + ((g ^ ((l16 >> 1) & 3)) * 16);
            displacement = 0;
        } else if constexpr (sizeof(T) == 2) {  // a lane's terms are 8 g + 0 .. 7; it reads for others 8 bytes of term 8 g + l16 / 4 (+ 4)
            at = (g * 8 + (l16 >> 2)) * R * 2 + ((l16 & 3) >> 1) * 16 + (l16 & 1) * 8;
            displacement = displaced<T, R / 8>(g * 8 + (l16 >> 2));
        } else {
            at = g * 4 * R * 4 + (l16 >> 2) * 16 + (l16 & 3) * 4;
            displacement = displaced<T, R / 4>(g * 4);
        }
    }
    __device__ __forceinline__ Vec<T> read(const char* lds, int tile) const
    {
        if constexpr (ALONG) {
            return *reinterpret_cast<const Vec<T>*>(lds + at + tile * 16 * kStepBytes);
        } else if constexpr (sizeof(T) == 2) {
            // a transposing read: lane i of 16 gets column i of the four rows that each four lanes point at
            typedef short s4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s4* Lds4;
            const char* p = lds + at + ((((first >> 3) + tile * 2) ^ displacement) * 16);
            union { s4 q[2]; Vec<T> v; } r;
            r.q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)p);
            r.q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)(p + 4 * R * 2));
            return r.v;
        } else {
            const char* p = lds + at + ((((first >> 2) + tile * 4) ^ displacement) * 16);
            Vec<T> v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const float*>(p + j * R * 4);
            return v;
        }
    }
};

// The tile that a block takes, of `layers` times nm x nn.  Units of 4 x 4 tiles share operands in an XCD's L2 (blocks go to the
// 8 XCDs in turn) and go to the XCDs in turn themselves, so that tiles which turn out to be empty are missing on all of
// them alike: with an eighth of all tiles side by side on each XCD, the last of them had nothing to do at
// 4,096 rows of one expert (an eighth more tiles than rows for, and 28 % of the time idle).
constexpr int kUnit = 4;
struct Place { int layer, m, n; };
__device__ __forceinline__ Place place_of(unsigned block, int nm, int nn)
{
    const int i = block >> 3, unit = i / (kUnit * kUnit) * 8 + (int)(block & 7), in = i % (kUnit * kUnit);
    const int across = (nn + kUnit - 1) / kUnit, per = (nm + kUnit - 1) / kUnit * across, u = unit % per;
    return Place{unit / per, u / across * kUnit + in % kUnit, u % across * kUnit + in / kUnit};
}
long blocks_of(long layers, int nm, int nn)
{
    const long units = layers * ((nm + kUnit - 1) / kUnit) * ((nn + kUnit - 1) / kUnit);
    return (units + 7) / 8 * 8 * kUnit * kUnit;
}

// ---- the product ----

// A block's tile of WM TM 16 x WN TN 16 results; a wave's is TM 16 x TN 16.
//
// Four stages of LDS: while a step's products run from one, the operands of the three next steps come into the others.  A
// step is TM groups of TN products.  Fragments are read three groups ahead, across the steps too: the barrier stands
// before the last three groups, when every wave has read what it needs of the stage, so that the products of these
// hide it and the first reads of the next stage.
//
// Bound by the way from L2 to LDS and by what nothing hides: at 8,192 x 2,048, 8 experts, k = 2, bf16, both forward products and
// their sums took 617 us (580 since stream4); without the fetches in the loop 457, without the reads of fragments 625, without either 435, of which
// 250 are the products (with 4.25 and 2.1 tiles a CU that take 5 and 3 turns) and 140 the tiles' ends: all CUs write then,
// 8 bytes a result beside h in the gated product, which is the rate of the memory (kHidden reads and writes 22).  One expert, 8,192 x
// 2,048 by 4,096, runs at 930 to 1,080 TFLOP/s where a large library product reaches 1,410; rows a multiple of 4 KB apart, as all
// there are, cost a tenth, for their chunks of the same terms lie in few channels.
// Steps on the way, us (gated, gates, outs):
//   fragments read as they are used, results stored from the registers, one step ahead:  390, 745, 347
//   fragments three groups ahead, results by rows through LDS:                            377, 364, 199
//   three steps ahead:                                                                    372, 268, 159
// 4 waves of 128 x 128 were slower (450 to 460 for the gated one), tiles of 256 x 128, two blocks a CU, too (400): they read
// more from L2.
template <typename T, int KIND, int WM, int WN, int TM, int TN, bool FAST>
__global__ __launch_bounds__(WM* WN * 64, 2) void k_product(FeedArgs<T> p)
{
    constexpr int NT = WM * WN * 64, RA = WM * TM * 16, RB = WN * TN * 16, STAGE = (RA + RB) * kStepBytes;
    constexpr bool MATRIX = KIND == kGates || KIND == kOuts;  // the sum runs over slots
    constexpr bool A_ALONG = !MATRIX, B_ALONG = KIND == kGated || KIND == kDown;
    constexpr bool GATHERED = MATRIX;
    constexpr int STAGES = 4, ASLOTS = 8;  // ASLOTS: the slots of gathered rows, of 8 steps, a copy a wave
    __shared__ __attribute__((aligned(1024))) char lds[STAGES * STAGE + (GATHERED ? NT / 64 * ASLOTS * 256 : 0)];

    const int lane = threadIdx.x & 63, wave = wave_index(), l16 = lane & 15, g = lane >> 4;
    const int wm = wave / WN, wn = wave % WN;
    Tile t;
    int n0, m0 = 0, split = 0;
    const T *A = p.A, *B = p.B, *B2 = p.B2;
    T* dm = p.dm;
    int terms = p.K, from = 0, matrix = 0;
    if constexpr (MATRIX) {
        const int both = KIND == kGates ? 2 : 1;
        const Place at = place_of(blockIdx.x, p.nm, p.nn);
        if (at.layer >= p.a * p.splits * both || at.m >= p.nm || at.n >= p.nn) return;
        m0 = at.m * RA;
        n0 = at.n * RB;
        split = at.layer % p.splits;
        matrix = at.layer / p.splits % both;
        const int q = at.layer / p.splits / both;
        t = p.tiles != nullptr ? p.tiles[q] : Tile{0, 0, p.slots, -1};
        t.q = q;
        if (matrix) {
            A = p.A2;
            dm = p.dm2;
        }
        // this part's slots, whole steps
        const int steps = (t.cnt + kStep<T> - 1) / kStep<T>;
        from = (int)((long)steps * split / p.splits) * kStep<T>;
        terms = max(0, min(t.cnt, (int)((long)steps * (split + 1) / p.splits) * kStep<T>) - from);
    } else {
        const Place at = place_of(blockIdx.x, p.ntiles, p.nn);
        if (at.layer >= p.splits || at.m >= p.ntiles || at.n >= p.nn) return;
        split = at.layer;
        n0 = at.n * (KIND == kGated ? RB / 2 : RB);
        if (p.tiles != nullptr) {
            t = p.tiles[at.m / p.cut];
            const int skip = at.m % p.cut * RA;
            t.start += skip;
            t.cnt = min(RA, t.cnt - skip);
            if (t.cnt <= 0) return;
        } else {
            t = Tile{0, at.m * RA, min(RA, p.slots - at.m * RA), -1};
        }
        if (t.q < 0) return;
        if (t.q >= p.a) {  // slots without an expert
            if constexpr (KIND == kGated) {
                if (p.pre == nullptr) return;
                for (int i = threadIdx.x; i < t.cnt * (RB / 2); i += NT) {
                    const int f = n0 + i % (RB / 2);
                    float* to = p.pre + (long)p.perm[t.start + i / (RB / 2)] * 2 * p.N;
                    if (f < p.N) to[f] = to[p.N + f] = 0.f;
                }
            }
            if constexpr (KIND == kDown || KIND == kRows) {
                if (p.out == nullptr) return;
                for (int i = threadIdx.x; i < t.cnt * RB; i += NT) {
                    const int n = n0 + i % RB;
                    const long row = p.perm[t.start + i / RB];
                    if (n < p.N) p.out[row * p.ld_out + n] = p.base != nullptr ? p.base[row * p.ld_base + n] : (T)0.f;
                }
            }
            return;
        }
        B += t.q * p.sb;
        if constexpr (KIND == kGated || KIND == kRows) B2 += t.q * p.sb2;
        if constexpr (KIND == kDown) {
            const int steps = (p.K + kStep<T> - 1) / kStep<T>;
            from = (int)((long)steps * split / p.splits) * kStep<T>;
            terms = min(p.K, (int)((long)steps * (split + 1) / p.splits) * kStep<T>) - from;
            A += from;
            B += from;
        }
    }
    // P^T dg + Q^T du: one sum after the other, or a block each
    const bool both_sums = KIND == kRows && p.splits == 1;
    long ldb = p.ldb;
    if constexpr (KIND == kRows)
        if (split > 0) {
            A = p.A2;
            B = B2;
            ldb = p.ldb2;
        }
    auto slot_of = [&](int place) -> int { return p.perm != nullptr ? p.perm[place] : place; };

    Stager<T, A_ALONG, RA, NT, FAST> sa;
    Stager<T, B_ALONG, RB, NT, FAST> sb;
    const int steps1 = (terms + kStep<T> - 1) / kStep<T>, steps = both_sums ? 2 * steps1 : steps1;
    const int left_a = p.M - m0, left_b = p.N - n0, start = t.start + (MATRIX ? from : 0);
    auto begin_a = [&](const T* a) {
        if constexpr (KIND == kGated || KIND == kHidden)
            sa.rows([&](int r) { return a + (long)p.byk.row((unsigned)slot_of(t.start + min(r, t.cnt - 1))) * p.lda; });
        if constexpr (KIND == kDown || KIND == kRows) sa.rows([&](int r) { return a + (long)(t.start + min(r, t.cnt - 1)) * p.lda; });
    };
    begin_a(A);
    if constexpr (KIND == kGates) sa.terms(A + m0 + start * p.lda, p.lda, left_a);
    if constexpr (KIND == kGated)  // 16 rows of one matrix beside 16 of the other
        sb.rows([&](int r) {
            const int f = min(n0 + (r >> 5) * 16 + (r & 15), p.N - 1);
            return r & 16 ? B2 + f * p.ldb2 : B + f * p.ldb;
        });
    if constexpr (KIND == kDown) sb.rows([&](int r) { return B + (long)min(n0 + r, p.N - 1) * p.ldb; });
    if constexpr (KIND == kHidden || KIND == kRows) sb.terms(B + n0, ldb, left_b);
    if constexpr (KIND == kOuts) sb.terms(B + n0 + start * p.ldb, p.ldb, left_b);

    // The slots of step `step`'s gathered rows, which are fetched from step - ASLOTS / 2 on.
    const unsigned lds_slots = lds_offset(lds) + STAGES * STAGE + wave * (ASLOTS * 256);
    auto look = [&](int step) {
        if constexpr (GATHERED) {
            const int* from_perm = p.perm + start + min(step * kStep<T> + (lane & (kStep<T> - 1)), max(terms - 1, 0));
            const void* src = p.perm != nullptr ? (const void*)from_perm : (const void*)g_zeros;
            unsigned kept;
            asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %2, off\n\ts_mov_b32 m0, %0"
                         : "=&s"(kept) : "s"(lds_slots + (step & (ASLOTS - 1)) * 256), "v"(src) : "memory");
        }
    };
    // Part c of a step's operands, one chunk a lane: those of A, then those of B.  A step's are taken in their order; steps
    // past the last are zeros.
    constexpr int CHUNKS_A = decltype(sa)::C, CHUNKS = CHUNKS_A + decltype(sb)::C, LOADS = CHUNKS + (GATHERED ? 1 : 0);
    const unsigned lds_wave = lds_offset(lds) + wave * 1024;
    auto fetch = [&](int step, int stage, int c) {
        unsigned to = lds_wave + stage;
        int k0 = step * kStep<T>;
        bool second = false;
        if constexpr (KIND == kRows)
            if (both_sums && step >= steps1) {
                second = true;
                k0 -= steps1 * kStep<T>;
                if (c == 0 && step == steps1) {
                    begin_a(p.A2);
                    sb.terms(B2 + n0, p.ldb2, left_b);
                }
            }
        const int* slots = nullptr;
        if constexpr (GATHERED) {
            if (c == 0) look(step + ASLOTS / 2);  // landed three steps later at the latest, with that step's operands
            if (p.perm != nullptr) slots = reinterpret_cast<const int*>(lds + STAGES * STAGE + wave * (ASLOTS * 256) + (step & (ASLOTS - 1)) * 256);
        }
        if (c < CHUNKS_A) {
            if constexpr (A_ALONG) sa.along(c, k0, terms, to);
            if constexpr (KIND == kGates) sa.across(c, k0, terms, p.lda, left_a, to);
            if constexpr (KIND == kOuts) sa.gathered(c, k0, terms, slots, start + k0, p.byk, A + m0, p.lda, left_a, to);
        } else {
            c -= CHUNKS_A;
            to += RA * kStepBytes;
            if constexpr (B_ALONG) sb.along(c, k0, terms, to);
            if constexpr (KIND == kHidden || KIND == kRows || KIND == kOuts) sb.across(c, k0, terms, second ? p.ldb2 : ldb, left_b, to);
            if constexpr (KIND == kGates) sb.gathered(c, k0, terms, slots, start + k0, p.byk, B + n0, p.ldb, left_b, to);
        }
    };
    auto settle = [&](int stage) {
        sa.settle(lds + stage);
        sb.settle(lds + stage + RA * kStepBytes);
    };

    const Reader<T, A_ALONG, RA> ra(wm * TM * 16);
    const Reader<T, B_ALONG, RB> rb(wn * TN * 16);
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    if (steps > 0) {
        constexpr int AHEAD = TM < 4 ? TM - 1 : 3, RING = AHEAD + 1, EACH = (CHUNKS + TM - 1) / TM;
        static_assert(TM % RING == 0, "a fragment's registers are free when the next step reads into them");
        Vec<T> x[RING], y[2][TN];
        if constexpr (GATHERED) {
#pragma unroll
            for (int i = 0; i < ASLOTS / 2; ++i) look(i);
            landed<0>();
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) {
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) fetch(i, i * STAGE, c);
            settle(i * STAGE);
        }
        landed<FAST ? (STAGES - 2) * LOADS : 0>();
        __syncthreads();
        auto take_y = [&](int stage, Vec<T>* to) {
#pragma unroll
            for (int j = 0; j < TN; ++j) to[j] = rb.read(lds + stage + RA * kStepBytes, j);
        };
        int before = (STAGES - 1) * STAGE, now = 0, next = STAGE;  // bytes: the stages of the last step, this one and the next
        take_y(now, y[0]);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            x[i] = ra.read(lds, i);
#pragma unroll
            for (int e = 0; e < EACH; ++e)
                if (i * EACH + e < CHUNKS) fetch(STAGES - 1, before, i * EACH + e);
        }
        for (int s0 = 0; s0 < steps; s0 += 2) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int s = s0 + h;
#pragma unroll
                for (int u = 0; u < TM; ++u) {
                    const int v = u + AHEAD, v1 = v < TM ? v : v - TM;
                    if (u == TM - AHEAD) {
                        settle(before);
                        landed<FAST ? (STAGES - 2) * LOADS : 0>();
                        __syncthreads();
                        take_y(next, y[h ^ 1]);
                    }
                    x[v % RING] = ra.read(lds + (v < TM ? now : next), v1);
                    // a step's parts are fetched one by one, into the stage that the last barrier freed: all at once they
                    // would fill the queue to memory, and the products behind them would wait
#pragma unroll
                    for (int e = 0; e < EACH; ++e)
                        if (v1 * EACH + e < CHUNKS) fetch((v < TM ? s : s + 1) + STAGES - 1, v < TM ? before : now, v1 * EACH + e);
#pragma unroll
                    for (int j = 0; j < TN; ++j) acc[u][j] = mfma16(y[h][j], x[u % RING], acc[u][j]);
                }
                before = now;
                now = next;
                next = next == (STAGES - 1) * STAGE ? 0 : next + STAGE;
            }
        }
        landed<0>();
        __syncthreads();
    }

    // Results go through LDS, up to 64 rows of a wave at once in its own part of it, so that neighbouring lanes take neighbouring
    // columns: lane (l16, g) holds m = i 16 + l16 and n = j 16 + 4 g + 0 .. 3.  Chunks of 16 bytes are exchanged by the row's number.
    constexpr int WIDE = TN * 16, QUADS = TN * 4, EX = QUADS < 16 ? QUADS - 1 : 15;  // a row of the wave's results: columns, chunks
    constexpr int PART = TM < 4 ? TM : 4;                                          // tiles of 16 rows at once
    static_assert(STAGES * STAGE >= WM * WN * PART * 16 * WIDE * 4 && TM % PART == 0, "the rows of all waves");
    char* mine = lds + wave * (PART * 16 * WIDE * 4);
    auto result = [&](int r, int c) { return *reinterpret_cast<const f32x4*>(mine + r * (WIDE * 4) + ((c ^ (r & EX)) * 16)); };
    for (int part = 0; part < TM / PART; ++part) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
            if (i / PART == part)
#pragma unroll
                for (int j = 0; j < TN; ++j) *reinterpret_cast<f32x4*>(mine + (i % PART * 16 + l16) * (WIDE * 4) + (((j * 4 + g) ^ (l16 & EX)) * 16)) = acc[i][j];
        __builtin_amdgcn_wave_barrier();
        const int first = (wm * TM + part * PART) * 16;  // of the tile's rows
        if constexpr (KIND == kGated) {
#pragma unroll 2
            for (int it = 0; it < PART * QUADS / 8; ++it) {
                const int r = it * (128 / QUADS) + lane / (QUADS / 2), c = lane % (QUADS / 2), m = first + r;  // the c-th four columns of f
                const f32x4 gate = result(r, (c >> 2) * 8 + (c & 3)), up = result(r, (c >> 2) * 8 + 4 + (c & 3));
                const int f = n0 + wn * (TN * 8) + c * 4;
                if (m >= t.cnt || f >= p.ldh) continue;
                const int place = t.start + m, slot = slot_of(place);
                const float w = p.weights != nullptr ? p.weights[slot] : 1.f;
                if (p.pre != nullptr) {
                    float* to = p.pre + (long)slot * 2 * p.N + f;
                    stream4(to, gate, p.N - f);
                    stream4(to + p.N, up, p.N - f);
                }
                f32x4 h;
#pragma unroll
                for (int e = 0; e < 4; ++e) h[e] = f + e < p.N ? w * (activate(gate[e], p.act).x * up[e]) : 0.f;
                put4(p.h + place * p.ldh + f, h, 4);
            }
        } else {
#pragma unroll 2
            for (int it = 0; it < PART * QUADS / 4; ++it) {
                const int r = it * (64 / QUADS) + lane / QUADS, c = lane % QUADS, m = first + r, n = n0 + wn * WIDE + c * 4;
                f32x4 v = result(r, c);
                if constexpr (MATRIX) {
                    if (m0 + m >= p.M || n >= p.N) continue;
                    const long each = (long)p.M * p.N, at = (long)(m0 + m) * p.N + n;
                    if (p.splits == 1)
                        put4(dm + t.q * each + at, v, p.N - n);
                    else
                        stream4(p.part + (((long)split * p.a + t.q) * (KIND == kGates ? 2 : 1) + matrix) * each + at, v, p.N - n);
                } else if constexpr (KIND == kHidden) {
                    const bool there = m < t.cnt && n < p.ldh;
                    const int place = t.start + min(m, t.cnt - 1), slot = slot_of(place);
                    float dot = 0.f;
                    if (there) {
                        const float w = p.weights != nullptr ? p.weights[slot] : 1.f;
                        const float* pre = p.pre + (long)slot * 2 * p.N + n;
                        const f32x4 gate = once4(pre, p.N - n), up = once4(pre + p.N, p.N - n);
                        f32x4 h, dg, du;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 act = activate(gate[e], p.act);
                            const bool in = n + e < p.N;
                            const float hidden = act.x * up[e], err = v[e];
                            dot += in ? err * hidden : 0.f;
                            h[e] = in ? w * hidden : 0.f;
                            dg[e] = in ? w * err * up[e] * act.y : 0.f;
                            du[e] = in ? w * err * act.x : 0.f;
                        }
                        if (p.h != nullptr) put4(p.h + place * p.ldh + n, h, 4);
                        put4(p.dg + place * p.ldh + n, dg, 4);
                        put4(p.du + place * p.ldh + n, du, 4);
                    }
                    if (p.dots != nullptr) {
#pragma unroll
                        for (int x = 1; x < QUADS; x <<= 1) dot += __shfl_xor(dot, x);
                        if (m < t.cnt && c == 0) p.dots[(long)slot * p.ndots + n0 / WIDE + wn] = dot;
                    }
                } else {
                    if (m >= t.cnt || n >= p.N) continue;
                    const long slot = slot_of(t.start + m);
                    if (p.out != nullptr) {
                        if (p.base != nullptr) v += get4(p.base + slot * p.ld_base + n, p.N - n);
                        put4(p.out + slot * p.ld_out + n, v, p.N - n);
                    } else {
                        stream4(p.sums + ((long)split * p.slots + slot) * p.N + n, v, p.N - n);
                    }
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- few slots: each with its expert's matrices as they come from memory ----

constexpr int kFewThreads = 256, kFewRows = 2;  // rows of a matrix that a wave takes

template <typename T>
struct FewArgs {
    const T* x; long ld_x;
    const T* gate; long gate_sa, gate_ld;
    const T* up; long up_sa, up_ld;
    const T* down; long down_sa, down_ld;
    const int* chosen; const float* weights; int act;
    const T* base; long ld_base; T* out; long ld_out;
    T* h; long ldh; float* pre;
    int n, d, f, o, k, a;
};

// acc[i] += this lane's part of <m_i, v>, `terms` long.
template <typename T, int ROWS>
__device__ __forceinline__ void dots_with(const T* v, const T* const (&m)[ROWS], int terms, float (&acc)[ROWS])
{
    constexpr int V = kVec<T>, STEP = 64 * V;
    int at = (int)(threadIdx.x & 63) * V;
    auto add = [&](const Vec<T>& a, const Vec<T> (&b)[ROWS]) {
#pragma unroll
        for (int e = 0; e < V; ++e)
#pragma unroll
            for (int i = 0; i < ROWS; ++i) acc[i] = fmaf(to_f(a[e]), to_f(b[i][e]), acc[i]);
    };
#pragma unroll 4
    for (; at + V <= terms; at += STEP) {
        const Vec<T> a = load16(v + at);
        Vec<T> b[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) b[i] = load16(m[i] + at);
        add(a, b);
    }
    if (at < terms) {
        const Vec<T> a = load_part(v + at, terms - at);
        Vec<T> b[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) b[i] = load_part(m[i] + at, terms - at);
        add(a, b);
    }
}
template <int ROWS>
__device__ __forceinline__ void sum_lanes(float (&acc)[ROWS])
{
#pragma unroll
    for (int x = 1; x < 64; x <<= 1)
#pragma unroll
        for (int i = 0; i < ROWS; ++i) acc[i] += __shfl_xor(acc[i], x);
}

// g, u and the weighted h of kFewRows hidden places of a slot, a wave each.
template <typename T>
__global__ __launch_bounds__(kFewThreads) void k_few_gated(FewArgs<T> p)
{
    const int per = (p.f + kFewRows - 1) / kFewRows, w = (int)blockIdx.x * (kFewThreads / 64) + wave_index();
    const int slot = w / per, f0 = w % per * kFewRows, lane = threadIdx.x & 63;
    if (slot >= p.n * p.k) return;
    const int q = p.chosen != nullptr ? p.chosen[slot] : 0;
    if (q < 0 || q >= p.a) {
        if (p.pre != nullptr && lane < kFewRows && f0 + lane < p.f) {
            float* to = p.pre + (long)slot * 2 * p.f + f0 + lane;
            to[0] = to[p.f] = 0.f;
        }
        return;
    }
    const T* m[2 * kFewRows];
#pragma unroll
    for (int i = 0; i < kFewRows; ++i) {
        const long f = min(f0 + i, p.f - 1);
        m[i] = p.gate + q * p.gate_sa + f * p.gate_ld;
        m[kFewRows + i] = p.up + q * p.up_sa + f * p.up_ld;
    }
    float acc[2 * kFewRows] = {};
    dots_with<T, 2 * kFewRows>(p.x + slot / p.k * p.ld_x, m, p.d, acc);
    sum_lanes(acc);
#pragma unroll
    for (int i = 0; i < kFewRows; ++i) {
        if (lane != i || f0 + i >= p.f) continue;
        const float g = acc[i], u = acc[kFewRows + i], wt = p.weights != nullptr ? p.weights[slot] : 1.f;
        if (p.pre != nullptr) {
            float* to = p.pre + (long)slot * 2 * p.f + f0 + i;
            to[0] = g;
            to[p.f] = u;
        }
        p.h[slot * p.ldh + f0 + i] = from_f<T>(wt * (activate(g, p.act).x * u));
    }
}

// kFewRows results of a row, over all its slots.
template <typename T>
__global__ __launch_bounds__(kFewThreads) void k_few_down(FewArgs<T> p)
{
    const int per = (p.o + kFewRows - 1) / kFewRows, w = (int)blockIdx.x * (kFewThreads / 64) + wave_index();
    const int row = w / per, o0 = w % per * kFewRows, lane = threadIdx.x & 63;
    if (row >= p.n) return;
    float acc[kFewRows] = {};
    for (int j = 0; j < p.k; ++j) {
        const int slot = row * p.k + j, q = p.chosen != nullptr ? p.chosen[slot] : 0;
        if (q < 0 || q >= p.a) continue;
        const T* m[kFewRows];
#pragma unroll
        for (int i = 0; i < kFewRows; ++i) m[i] = p.down + q * p.down_sa + (long)min(o0 + i, p.o - 1) * p.down_ld;
        dots_with<T, kFewRows>(p.h + slot * p.ldh, m, p.f, acc);
    }
    sum_lanes(acc);
#pragma unroll
    for (int i = 0; i < kFewRows; ++i)
        if (lane == i && o0 + i < p.o)
            p.out[row * p.ld_out + o0 + i] = from_f<T>(p.base != nullptr ? to_f(p.base[row * p.ld_base + o0 + i]) + acc[i] : acc[i]);
}

// ---- what joins parts ----

template <typename T>
struct JoinArgs {
    const float* sums; const int* chosen; int n, k, a, w, splits;  // [splits][n k][w]
    const T* base; long ld_base; T* out; long ld_out;
};

// out_i = base_i + the sum of row i's slots, in their order; a block a stretch of 1,024 columns of a row.
template <typename T>
__global__ __launch_bounds__(256) void k_feed_join(JoinArgs<T> p)
{
    const long row = blockIdx.x;
    const int n = ((int)blockIdx.y * 256 + (int)threadIdx.x) * 4;
    if (n >= p.w) return;
    const int left = p.w - n;
    f32x4 v{0.f, 0.f, 0.f, 0.f};
    if (p.base != nullptr) v = get4(p.base + row * p.ld_base + n, left);
    for (int j = 0; j < p.k; ++j) {
        const int q = p.chosen != nullptr ? p.chosen[row * p.k + j] : 0;
        if (q >= 0 && q < p.a)
            for (int s = 0; s < p.splits; ++s) v += get4(p.sums + (((long)s * p.n + row) * p.k + j) * p.w + n, left);
    }
    put4(p.out + row * p.ld_out + n, v, left);
}

// dw of every slot: the sum of its parts in their order, 0 for one without an expert.
__global__ __launch_bounds__(256) void k_feed_dots(const float* dots, int ndots, const int* chosen, int slots, int a, float* dw)
{
    const int i = (int)(blockIdx.x * 256 + threadIdx.x);
    if (i >= slots) return;
    const int q = chosen != nullptr ? chosen[i] : 0;
    float v = 0.f;
    if (q >= 0 && q < a)
        for (int j = 0; j < ndots; ++j) v += dots[(long)i * ndots + j];
    dw[i] = v;
}

// The matrices' gradients from their parts, in their order.
template <typename T>
__global__ __launch_bounds__(256) void k_feed_merge(const float* part, int splits, long each, int both, int a, T* dm, T* dm2)
{
    const long all = each * both * a;
    for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4; i < all; i += (long)gridDim.x * 1024) {
        f32x4 v{0.f, 0.f, 0.f, 0.f};
        const int left = (int)(all - i < 4 ? all - i : 4);
        for (int s = 0; s < splits; ++s) v += get4(part + s * all + i, left);
        for (int e = 0; e < left; ++e) {
            const long at = i + e, q = at / (each * both), in = at - q * each * both;
            (in >= each ? dm2 : dm)[q * each + (in >= each ? in - each : in)] = from_f<T>(v[e]);
        }
    }
}

// ---- launches ----

size_t up16(size_t b) { return (b + 15) & ~size_t(15); }

// Forward calls of few slots may take two launches that read a slot's matrices as they come from memory, an expert's anew for each of
// its slots (from the caches where they hold it), instead of tiles of one expert, which read them once, but by few blocks in
// long chains of steps, behind a sort.  The rule compares estimates of both, us: the slots' reads at 16 TB/s where all matrices
// fit the L2s, down to 7.6 where they do not (16-bit rows off 16 bytes: 9 to 6); the steps' chains, one expert's matrices by the blocks that
// it has, all matrices, the sort.  us, few and tiles, with the matrices from memory at every call, and the slots from which on the rule takes tiles:
//   bf16, d = o = 4,096, f = 11,008,  1 expert:         4 slots 147, 178;  8:  274, 182;  16:   554, 191;  64: 2,279, 257  (from 5 on)
//                       f = 2,048,    1:                8 slots  36,  44; 12:   46,  45;  16:    58,  45;  64:   221,  51  (11)
//                                     4, k = 2:         8 slots  53,  58; 12:   80,  61;  16:   108,  62;  64:   391,  63  (12)
//                                    16, k = 2:         2 slots  24,  43; 16:  125, 133;  24:   175, 142;  64:   448, 173  (20)
//         d = o = 2,048, f = 1,024,   1:                8 slots  15,  26; 16:   21,  26;  24:    26,  27;  64:    53,  30  (20)
//                                     8, k = 2:         2 slots  14,  35; 16:   30,  39;  24:    39,  40;  64:    74,  40  (30)
//         d = o = 512, f = 512,      64, k = 4:         4 slots  10,  22; 16:   13,  30;  64:    23,  33
//         d = o = 4,095, f = 2,047,   1:                8 slots  67, 136; 16:  106, 136;  24:   150, 137;  64:   366, 137  (21)
//   fp32, d = o = 4,096, f = 11,008,  1:                4 slots 312, 619;  8:  611, 624;  16: 1,220, 622;  48: 3,598, 622  (7)
//                       f = 2,048,    1:                8 slots  68, 130; 16:  132, 131;  24:   198, 132;  48:   397, 132  (17)
//                                     8, k = 2:         8 slots 125, 240; 16:  229, 235;  24:   319, 245;  48:   641, 251  (20)
//         d = o = 1,024, f = 1,024,   1:                8 slots  14,  48; 48:   35,  50;  64:    43,  50  (54)
//         d = o = 4,095, f = 2,047,   1:                8 slots  72, 346; 24:  214, 351;  48:   441, 352  (39)
bool is_few(const FeedSizes& z)
{
    const double slots = (double)z.n * z.k;
    if (slots > 64) return false;
    const bool wide = z.type == kF32;
    const double matrix = (double)z.f * (2.0 * z.d + z.o) * elem_size(z.type), all = std::min((double)z.a, slots) * matrix;
    const double few = slots * matrix * (wide || z.aligned ? (1 + 1.1 * std::min(1.0, all / 2e8)) / 16e6 : (1 + 0.5 * std::min(1.0, all / 2e8)) / 9e6);
    const double tiles = (z.sorted ? 10 : 0) + ((double)z.d + z.f) * (wide ? (z.aligned ? 0.02 : 0.056) : z.aligned ? 0.004 : 0.018) + matrix / 4e6 + all / 1e7;
    return few <= tiles;
}

struct Layout {
    int slots, ntiles, segments;
    int tile, r[kKinds];                  // rows of the sort's tiles, and of each product's
    bool few, fast, sorted, joined;       // joined: a launch adds up a row's parts
    int ldh, ndots, rsplits, gsplits, osplits;
    size_t seen, perm, tiles, groups, merge, h, dg, du, dots, sums, part, bytes;
};

int tiles_of(long m, int r) { return (int)((m + r - 1) / r); }

// Rows (and columns) of a block's tile: 256 (one block a CU, FAST only), 128 (two) or 64 (four).  What a tile costs is its
// products over how well they keep the matrix cores busy, which the CU's other blocks help with; what a launch
// costs is that of the CU with most tiles.  us, forward and gradients of rows and of matrices, all products with tiles of 64 / 128 / 256, and
// by the rule:
//   bf16   64 x 4,096 by 2,048, 16 experts, k = 2: 179 193 494 / 193 178 427 / 228 236 375, 181 194 379
//         300 x 1,024 by 1,024,  4, 1:              25  43  50 /  39  69  65 /  72 118  97,  26  44  48
//         512 x 2,048 by 2,048,  8, 2:             101 119 207 /  89 109 184 / 124 198 207,  88 109 167
//       2,048 x 2,048 by 2,048,  8, 2:             268 350 383 / 211 281 331 / 204 256 299, 204 281 294
//       4,096 x 2,048 by 8,192,  1, 1:             813 955 1,263 / 509 603 785 / 453 604 673, 461 577 674
//       8,192 x 1,024 by 1,024,  8, 1:             140 157 199 / 117 153 170 / 130 150 256, 117 151 170
//       1,024 x 1,001 by 777,    4, 2:              69  95 117 /  85 153 141 / -,             69  95 115
//   fp32  256 x 512 by 1,024,    4, 1:              47  79  57 / 120 215 100 / 375 651 235,  47  78  58
//       2,048 x 2,048 by 2,048,  4, 1:             538 572 714 / 655 834 779 / 980 1,538 1,068, 513 567 706
int choose_tile(const FeedSizes& z, long rows, long columns, long layers, int parts, double tail = 1.0)
{
    int best = 0;
    double least = 0;
    for (const int r : {256, 128, 64}) {
        if (r == 256 && !z.aligned) continue;
        const long tiles = layers * tiles_of(rows, r) + (parts > 1 ? std::min<long>(parts, rows) / 2 : 0), busy = (tiles * tiles_of(columns, r) + 255) / 256;
        const double waste = z.type == kF32 ? (r == 256 ? 1.0 : r == 128 ? (busy > 1 ? 1.0 : 1.1) : busy > 1 ? 1.15 : 1.3)
                           : r == 256       ? (busy == 1 && layers > 1 ? 1.4 : 1.0)  // matrices of unlike experts: a second turn evens them out
                           : r == 128       ? (busy > 1 ? 1.35 : z.aligned ? 1.8 : 2.2)
                                            : (busy > 3 ? 2.0 : busy > 1 ? 2.6 : 4.0);
        const double cost = (double)busy * r * r * waste * (r == 256 ? tail : 1.0);
        if (best == 0 || cost < least) {
            best = r;
            least = cost;
        }
    }
    return best;
}

// Parts of the slots for the matrices' gradients: enough for two blocks a CU, each with 8 steps at least.
int matrix_splits(long slots, int a, int m, int n, int both, int r, int step)
{
    const long blocks = (long)a * both * tiles_of(m, r) * tiles_of(n, r);
    long s = 512 / (blocks > 0 ? blocks : 1);
    const long most = slots / a / (8 * step);
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s > 8 ? 8 : s);
}

// Parts of the sum of a product that goes back to the rows, where tiles of 256 leave half of the CUs without work: each part's results cost a
// write and a read in fp32.  4,096 x 2,048 from 8,192 hidden: 197 us in one, 143 in two (tiles of 256 in one: 206).
int row_splits(const FeedSizes& z, int r, long columns, long terms, int most)
{
    const long blocks = ((z.n * z.k + r - 1) / r + z.a / 2) * tiles_of(columns, r);
    if (r != 256 || terms < 4096 || blocks > 128 || blocks == 0) return 1;  // 0: no rows
    const int parts = std::min(most, (int)(256 / blocks));
    return blocks * parts < 192 ? 1 : parts;  // fewer are left to smaller tiles
}

Layout layout(const FeedSizes& z, bool backward)
{
    Layout L{};
    const int vec = 16 / (int)elem_size(z.type), step = 128 / (int)elem_size(z.type);
    L.slots = (int)(z.n * z.k);
    L.few = !backward && is_few(z);
    L.sorted = z.sorted && !L.few;
    L.fast = z.aligned;
    L.ldh = (z.f + vec - 1) / vec * vec;
    if (backward) {
        L.r[kHidden] = choose_tile(z, L.slots, z.f, 1, z.a, 1.15);  // 22 bytes a result at its end, which nothing else hides there: 356 us with 256 rows, 333 with 128
        L.r[kRows] = choose_tile(z, L.slots, z.d, 1, z.a);
        L.r[kGates] = choose_tile(z, z.f, z.d, 2 * z.a, 1);
        L.r[kOuts] = choose_tile(z, z.o, z.f, z.a, 1);
        if (z.type != kF32 && z.aligned && row_splits(z, 256, z.d, 2l * z.f, 2) == 2) L.r[kRows] = 256;
        L.rsplits = row_splits(z, L.r[kRows], z.d, 2l * z.f, 2);
        L.tile = std::max(L.r[kHidden], L.r[kRows]);
    } else {
        L.r[kGated] = choose_tile(z, L.slots, 2l * z.f, 1, z.a);
        L.r[kDown] = choose_tile(z, L.slots, z.o, 1, z.a);
        if (z.type != kF32 && z.aligned && row_splits(z, 256, z.o, z.f, 4) > 1) L.r[kDown] = 256;
        L.rsplits = row_splits(z, L.r[kDown], z.o, z.f, 4);
        L.tile = std::max(L.r[kGated], L.r[kDown]);
    }
    L.ntiles = L.slots / L.tile + z.a + 1;
    L.segments = (L.slots + kPlanRows - 1) / kPlanRows;
    if (L.segments < 1) L.segments = 1;
    if (backward) {
        L.ndots = tiles_of(z.f, L.r[kHidden]) * (L.r[kHidden] == 256 ? 4 : 2);  // one for each wave's columns
        L.gsplits = matrix_splits(L.slots, z.a, z.f, z.d, 2, L.r[kGates], step);
        L.osplits = matrix_splits(L.slots, z.a, z.o, z.f, 1, L.r[kOuts], step);
    }
    size_t at = 0;
    auto take = [&](size_t& where, size_t bytes) { where = at; at += up16(bytes); };
    if (L.sorted) {
        take(L.seen, L.segments > 1 ? (size_t)L.segments * (z.a + 1) * sizeof(int2) : 0);
        take(L.perm, (size_t)L.slots * 4);
        take(L.tiles, (size_t)L.ntiles * sizeof(Tile));
        if (backward) {
            take(L.groups, (size_t)z.a * sizeof(Tile));
            take(L.merge, (size_t)z.a * sizeof(int2));
        }
    }
    const size_t es = elem_size(z.type), hidden = (size_t)L.slots * L.ldh * es;
    take(L.h, hidden);
    const int w = backward ? z.d : z.o;
    L.joined = !L.few && (z.k > 1 || L.rsplits > 1);
    if (L.joined) take(L.sums, (size_t)L.rsplits * L.slots * w * 4);
    if (backward) {
        take(L.dg, hidden);
        take(L.du, hidden);
        take(L.dots, (size_t)L.slots * L.ndots * 4);
        const size_t g = L.gsplits > 1 ? (size_t)L.gsplits * z.a * 2 * z.f * z.d * 4 : 0, o = L.osplits > 1 ? (size_t)L.osplits * z.a * z.o * z.f * 4 : 0;
        take(L.part, g > o ? g : o);
    }
    L.bytes = at;
    return L;
}

hipError_t launch_plan(const Layout& L, const int* chosen, int a, char* ws, bool backward, hipStream_t s)
{
    // "chunks" of the plan: all slots of an expert
    const PlanArgs p{chosen, 1, L.slots, a, reinterpret_cast<int2*>(ws + L.seen), reinterpret_cast<int*>(ws + L.perm),
                     reinterpret_cast<Tile*>(ws + L.tiles), L.ntiles, L.tile,
                     backward ? reinterpret_cast<Tile*>(ws + L.groups) : nullptr, a,
                     backward ? reinterpret_cast<int2*>(ws + L.merge) : nullptr, 1 << 30, true};
    const dim3 grid(a + 1, L.segments);
    if (L.segments > 1) SKM_TRY_LAUNCH(k_plan_count, grid, kPlanThreads, 0, s, p);
    return launch(k_plan, grid, kPlanThreads, 0, s, p);
}

template <typename T, int KIND>
hipError_t launch_product(const Layout& L, FeedArgs<T> p, hipStream_t s)
{
    constexpr bool MATRIX = KIND == kGates || KIND == kOuts;
    const int r = L.r[KIND];
    p.nn = tiles_of(KIND == kGated ? 2l * p.N : p.N, r);
    p.nm = MATRIX ? tiles_of(p.M, r) : 0;
    if (!MATRIX) {
        p.cut = L.tile / r;
        p.ntiles = p.tiles != nullptr ? L.ntiles * p.cut : tiles_of(L.slots, r);
    }
    const dim3 grid((unsigned)(MATRIX ? blocks_of((long)p.a * p.splits * (KIND == kGates ? 2 : 1), p.nm, p.nn) : blocks_of(p.splits, p.ntiles, p.nn)));
    if (r == 256) return launch(k_product<T, KIND, 2, 4, 8, 4, true>, grid, 512, 0, s, p);
    if (r == 128) return L.fast ? launch(k_product<T, KIND, 2, 2, 4, 4, true>, grid, 256, 0, s, p) : launch(k_product<T, KIND, 2, 2, 4, 4, false>, grid, 256, 0, s, p);
    return L.fast ? launch(k_product<T, KIND, 2, 2, 2, 2, true>, grid, 256, 0, s, p) : launch(k_product<T, KIND, 2, 2, 2, 2, false>, grid, 256, 0, s, p);
}

template <typename T>
hipError_t launch_join(const float* sums, const int* chosen, const FeedSizes& z, int splits, int w, const T* base, long ld_base, T* out, long ld_out, hipStream_t s)
{
    const JoinArgs<T> p{sums, chosen, (int)z.n, z.k, z.a, w, splits, base, ld_base, out, ld_out};
    return launch(k_feed_join<T>, dim3((unsigned)z.n, (unsigned)((w + 1023) / 1024)), 256, 0, s, p);
}

}  // namespace

// Whether the rows and matrices of a call lie in whole 16 bytes is not known here: both ways have to fit.
bool feed_fits(FeedSizes z)
{
    if (z.n * z.k >= 1l << 30) return false;
    const long most = 1l << 32, wide = z.d > z.o ? z.d : z.o;  // threads a launch has fewer than
    if (z.n * 256 >= most || (wide + 1023) / 1024 >= 65536 || (z.n * z.k + kPlanRows - 1) / kPlanRows >= 65536) return false;
    const int outer = tiles_of(wide, 64);  // small calls at once: tiles of 64, the most parts
    if (blocks_of(4, (int)(z.n * z.k / 64) + 4 * (z.a + 1), std::max(tiles_of(2l * z.f, 64), outer)) * 512 < most && blocks_of(16l * z.a, tiles_of(z.f, 64), outer) * 512 < most) return true;
    for (int way = 0; way < 4; ++way) {
        z.aligned = (way & 1) != 0;
        const Layout L = layout(z, (way & 2) != 0);
        if (L.few) continue;
        auto fits = [&](int kind, long layers, long m, long n) {
            const long threads = L.r[kind] == 256 ? 512 : 256;
            return blocks_of(layers, (int)m, tiles_of(n, L.r[kind])) * threads < most;
        };
        auto rows = [&](int kind) { return (long)L.ntiles * (L.tile / L.r[kind]); };
        const bool fine = way & 2 ? fits(kHidden, 1, rows(kHidden), z.f) && fits(kRows, L.rsplits, rows(kRows), z.d) &&
                                        fits(kGates, 2l * z.a * L.gsplits, tiles_of(z.f, L.r[kGates]), z.d) &&
                                        fits(kOuts, (long)z.a * L.osplits, tiles_of(z.o, L.r[kOuts]), z.f)
                                  : fits(kGated, 1, rows(kGated), 2l * z.f) && fits(kDown, L.rsplits, rows(kDown), z.o);
        if (!fine) return false;
    }
    return true;
}

size_t feed_workspace(const FeedSizes& z, bool backward) { return layout(z, backward).bytes; }

hipError_t launch_feed(const FeedCall& a, hipStream_t s)
{
    const FeedSizes& z = a.z;
    if (z.n == 0) return hipSuccess;
    const Layout L = layout(z, false);
    if (L.sorted) {
        const hipError_t e = launch_plan(L, a.chosen, z.a, a.ws, false, s);
        if (e != hipSuccess) return e;
    }
    return with_type(z.type, [&](auto tag) {
        using T = decltype(tag);
        if (L.few) {
            const FewArgs<T> p{(const T*)a.x, a.ld_x, (const T*)a.gate, a.gate_sa, a.gate_ld, (const T*)a.up, a.up_sa, a.up_ld, (const T*)a.down, a.down_sa, a.down_ld,
                               a.chosen, a.weights, a.act, (const T*)a.base, a.ld_base, (T*)a.out, a.ld_out, (T*)(a.ws + L.h), L.ldh, a.pre,
                               (int)z.n, z.d, z.f, z.o, z.k, z.a};
            constexpr int EACH = kFewRows * (kFewThreads / 64);
            auto blocks = [&](long vectors, int rows) { return dim3((unsigned)((vectors * ((rows + kFewRows - 1) / kFewRows) * kFewRows + EACH - 1) / EACH)); };
            SKM_TRY_LAUNCH(k_few_gated<T>, blocks(L.slots, z.f), kFewThreads, 0, s, p);
            return launch(k_few_down<T>, blocks(z.n, z.o), kFewThreads, 0, s, p);
        }
        FeedArgs<T> p{};
        p.tiles = L.sorted ? reinterpret_cast<const Tile*>(a.ws + L.tiles) : nullptr;
        p.perm = L.sorted ? reinterpret_cast<const int*>(a.ws + L.perm) : nullptr;
        p.slots = L.slots;
        p.a = z.a;
        p.byk = by_k(z.k);
        p.splits = 1;
        p.h = (T*)(a.ws + L.h);
        p.ldh = L.ldh;
        p.weights = a.weights;
        p.act = a.act;
        FeedArgs<T> q = p;
        p.A = (const T*)a.x; p.lda = a.ld_x;
        p.B = (const T*)a.gate; p.sb = a.gate_sa; p.ldb = a.gate_ld;
        p.B2 = (const T*)a.up; p.sb2 = a.up_sa; p.ldb2 = a.up_ld;
        p.N = z.f; p.K = z.d;
        p.pre = a.pre;
        hipError_t e = launch_product<T, kGated>(L, p, s);
        if (e != hipSuccess) return e;
        q.A = q.h; q.lda = L.ldh;
        q.B = (const T*)a.down; q.sb = a.down_sa; q.ldb = a.down_ld;
        q.N = z.o; q.K = z.f;
        float* sums = reinterpret_cast<float*>(a.ws + L.sums);
        q.splits = L.rsplits;
        if (!L.joined) {
            q.base = (const T*)a.base; q.ld_base = a.ld_base;
            q.out = (T*)a.out; q.ld_out = a.ld_out;
        } else {
            q.sums = sums;
        }
        e = launch_product<T, kDown>(L, q, s);
        if (e != hipSuccess || !L.joined) return e;
        return launch_join<T>(sums, a.chosen, z, L.rsplits, z.o, (const T*)a.base, a.ld_base, (T*)a.out, a.ld_out, s);
    });
}

hipError_t launch_feed_back(const FeedBackCall& a, hipStream_t s)
{
    const FeedSizes& z = a.z;
    const Layout L = layout(z, true);
    const bool matrices = a.dgate != nullptr;
    if (z.n == 0 && !matrices) return hipSuccess;
    if (L.sorted) {
        const hipError_t e = launch_plan(L, a.chosen, z.a, a.ws, true, s);
        if (e != hipSuccess) return e;
    }
    return with_type(z.type, [&](auto tag) {
        using T = decltype(tag);
        FeedArgs<T> p{};
        p.tiles = L.sorted ? reinterpret_cast<const Tile*>(a.ws + L.tiles) : nullptr;
        p.perm = L.sorted ? reinterpret_cast<const int*>(a.ws + L.perm) : nullptr;
        p.slots = L.slots;
        p.a = z.a;
        p.byk = by_k(z.k);
        p.ldh = L.ldh;
        p.splits = 1;
        T *h = (T*)(a.ws + L.h), *dg = (T*)(a.ws + L.dg), *du = (T*)(a.ws + L.du);
        float* part = reinterpret_cast<float*>(a.ws + L.part);
        hipError_t e = hipSuccess;
        if (z.n > 0) {
            FeedArgs<T> q = p;
            q.A = (const T*)a.dy; q.lda = a.ld_dy;
            q.B = (const T*)a.down; q.sb = a.down_sa; q.ldb = a.down_ld;
            q.N = z.f; q.K = z.o;
            q.h = matrices ? h : nullptr;
            q.dg = dg; q.du = du;
            q.pre = const_cast<float*>(a.pre);
            q.weights = a.weights;
            q.act = a.act;
            float* dots = reinterpret_cast<float*>(a.ws + L.dots);
            q.dots = a.dweights != nullptr ? dots : nullptr;
            q.ndots = L.ndots;
            e = launch_product<T, kHidden>(L, q, s);
            if (e != hipSuccess) return e;
            if (a.dweights != nullptr) SKM_TRY_LAUNCH(k_feed_dots, dim3((L.slots + 255) / 256), 256, 0, s, dots, L.ndots, a.chosen, L.slots, z.a, a.dweights);
            if (a.dx != nullptr) {
                FeedArgs<T> r = p;
                r.A = dg; r.A2 = du; r.lda = L.ldh;
                r.B = (const T*)a.gate; r.sb = a.gate_sa; r.ldb = a.gate_ld;
                r.B2 = (const T*)a.up; r.sb2 = a.up_sa; r.ldb2 = a.up_ld;
                r.N = z.d; r.K = z.f;
                float* sums = reinterpret_cast<float*>(a.ws + L.sums);
                r.splits = L.rsplits;
                if (!L.joined) {
                    r.base = (const T*)a.base; r.ld_base = a.ld_base;
                    r.out = (T*)a.dx; r.ld_out = a.ld_dx;
                } else {
                    r.sums = sums;
                }
                e = launch_product<T, kRows>(L, r, s);
                if (e == hipSuccess && L.joined) e = launch_join<T>(sums, a.chosen, z, L.rsplits, z.d, (const T*)a.base, a.ld_base, (T*)a.dx, a.ld_dx, s);
                if (e != hipSuccess) return e;
            }
        }
        if (!matrices) return e;
        auto merge = [&](int splits, long each, int both, T* dm, T* dm2) {
            const long blocks = (each * both * z.a + 1023) / 1024;
            return launch(k_feed_merge<T>, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), 256, 0, s, part, splits, each, both, z.a, dm, dm2);
        };
        FeedArgs<T> u = p;
        u.tiles = L.sorted ? reinterpret_cast<const Tile*>(a.ws + L.groups) : nullptr;
        u.part = part;
        FeedArgs<T> v = u;
        u.A = dg; u.A2 = du; u.lda = L.ldh;
        u.B = (const T*)a.x; u.ldb = a.ld_x;
        u.M = z.f; u.N = z.d;
        u.dm = (T*)a.dgate; u.dm2 = (T*)a.dup;
        u.splits = L.gsplits;
        e = launch_product<T, kGates>(L, u, s);
        if (e == hipSuccess && L.gsplits > 1) e = merge(L.gsplits, (long)z.f * z.d, 2, u.dm, u.dm2);
        if (e != hipSuccess) return e;
        v.A = (const T*)a.dy; v.lda = a.ld_dy;
        v.B = h; v.ldb = L.ldh;
        v.M = z.o; v.N = z.f;
        v.dm = (T*)a.ddown;
        v.splits = L.osplits;
        e = launch_product<T, kOuts>(L, v, s);
        if (e == hipSuccess && L.osplits > 1) e = merge(L.osplits, (long)z.o * z.f, 1, v.dm, nullptr);
        return e;
    });
}

}  // namespace skm
