// experts.h -- the operators of skmetal_amd.experts: argument blocks and launchers
// (route_kernels.hip, adapt_kernels.hip, feed_kernels.hip, drop_kernels.hip, rate_kernels.hip).  Everything is in device memory and every
// launch goes to the caller's stream; nothing here allocates or waits.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace skm {

// Element types of scores, rows and adapters (SKMETAL_F32 ...).
enum ElemType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };
inline size_t elem_size(int t) { return t == kF32 ? 4 : 2; }

// ---- route_kernels.hip ----

constexpr int kRouteMaxE = 2048;  // experts
constexpr int kRouteMaxK = 16;    // experts a row takes

struct RouteArgs {
    const void* z; int type; long n; int E; long ld;   // scores [n x E], rows ld elements apart
    const uint8_t* mask; long mask_stride;             // nullable: rows that count
    int k; int normalize;
    float* w; int* ex;                                 // [n x k]
    int* counts; float* sums;                          // [E]
    int* rows; float* loss;                            // [1]
    char* ws;                                          // route_workspace(n, E) bytes
};
size_t route_workspace(long n, int E);
hipError_t launch_route(const RouteArgs& a, hipStream_t s);

struct RouteBackArgs {
    const void* z; int type; long n; int E; long ld;
    const uint8_t* mask; long mask_stride;
    int k; int normalize;
    const float* w; const int* ex; const int* counts; const int* rows;  // launch_route's
    const float* dw;                                   // nullable, [n x k]
    const float* dloss;                                // nullable, [1]
    void* dz; long ld_dz;                              // [n x E]
};
hipError_t launch_route_back(const RouteBackArgs& a, hipStream_t s);

// ---- adapt_kernels.hip ----

constexpr int kAdaptMaxR = 128;   // rank
constexpr int kAdaptMaxA = 2048;  // adapters

struct AdaptArgs {
    int type; long n; int d, o, r, a;
    const void* x; long ld_x;                          // [n x d]
    const void* down; long down_sa, down_ld;           // [a][r][d]
    const void* up; long up_sa, up_ld;                 // [a][r][o]
    const int* ids; long ids_stride;                   // [n]; outside [0, a): none
    const float* gates; long gates_stride;             // nullable, [n]
    const float* scales;                               // nullable, [a]
    const void* base; long ld_base;                    // nullable, [n x o]
    void* out; long ld_out;                            // [n x o]
    float* low;                                        // nullable, [n x r]
    bool in_x;                                         // out shares memory with x
    char* ws;
};
hipError_t launch_adapt(const AdaptArgs& a, hipStream_t s);

struct AdaptBackArgs {
    int type; long n; int d, o, r, a;
    const void* dy; long ld_dy;                        // [n x o]
    const void* x; long ld_x;
    const void* down; long down_sa, down_ld;
    const void* up; long up_sa, up_ld;
    const int* ids; long ids_stride;
    const float* gates; long gates_stride;
    const float* scales;
    const float* low;                                  // launch_adapt's
    const void* base; long ld_base;                    // nullable, [n x d]: added to dx
    void* dx; long ld_dx;                              // [n x d]
    void* ddown; void* dup;                            // [a][r][d], [a][r][o], dense
    float* dgates;                                     // nullable, [n]
    char* ws;
};
hipError_t launch_adapt_back(const AdaptBackArgs& a, hipStream_t s);
enum AdaptCall : int { kAdapt = 0, kAdaptBackward = 1, kAdaptInX = 2 };
size_t adapt_workspace(int type, long n, int d, int o, int r, int a, AdaptCall call);
// Whether every launch of both directions has a grid that the device takes.
bool adapt_fits(int type, long n, int d, int o, int r, int a);

// ---- feed_kernels.hip ----

constexpr int kFeedMaxK = 16;    // experts of a row
constexpr int kFeedMaxA = 2048;  // experts
enum Activation : int { kSilu = 0, kGelu = 1, kRelu = 2 };

struct FeedSizes {
    int type; long n; int d, f, o, k, a;
    bool sorted;                                       // false: one expert takes every row
    bool aligned;                                      // rows and matrices in whole 16 bytes
};
struct FeedCall {
    FeedSizes z;
    const void* x; long ld_x;                          // [n x d]
    const void* gate; long gate_sa, gate_ld;           // [a][f][d]
    const void* up; long up_sa, up_ld;                 // [a][f][d]
    const void* down; long down_sa, down_ld;           // [a][o][f]
    const int* chosen;                                 // [n x k]; outside [0, a): none; null where not sorted
    const float* weights;                              // nullable, [n x k]
    int act;
    const void* base; long ld_base;                    // nullable, [n x o]
    void* out; long ld_out;                            // [n x o]
    float* pre;                                        // nullable, [n x k][2][f]
    char* ws;
};
hipError_t launch_feed(const FeedCall& a, hipStream_t s);

struct FeedBackCall {
    FeedSizes z;
    const void* dy; long ld_dy;                        // [n x o]
    const void* x; long ld_x;
    const void* gate; long gate_sa, gate_ld;
    const void* up; long up_sa, up_ld;
    const void* down; long down_sa, down_ld;
    const int* chosen; const float* weights; int act;
    const float* pre;                                  // launch_feed's
    const void* base; long ld_base;                    // nullable, [n x d]: added to dx
    void* dx; long ld_dx;                              // nullable, [n x d]
    void *dgate, *dup, *ddown;                         // nullable together; dense
    float* dweights;                                   // nullable, [n x k]
    char* ws;
};
hipError_t launch_feed_back(const FeedBackCall& a, hipStream_t s);
size_t feed_workspace(const FeedSizes& z, bool backward);
// Whether every launch of both directions has a grid that the device takes.
bool feed_fits(FeedSizes z);

// ---- drop_kernels.hip ----

struct DropCall {
    int type; long n, d;
    const void* x; long ld_x;                          // [n x d]
    const void* base; long ld_base;                    // nullable, [n x d]
    void* out; long ld_out;                            // [n x d]; may be x or base
    const long long* key; unsigned site;               // key: seed, step
    unsigned limit; float scale;                       // p 2^32, 1 / (1 - p)
};
hipError_t launch_drop(const DropCall& a, hipStream_t s);

// ---- rate_kernels.hip ----

constexpr int kRateMaxK = 16;       // largest scores a row names
constexpr int kRateMaxV = 1 << 22;  // scores a row
constexpr int kRateSplits = 256;    // parts a row
constexpr int kRateList = 4096;     // scores that a part's choice looks at twice, at most

struct RateCall {
    const void* z; int type; long n; int v; long ld;   // scores [n x v]
    const int* targets; long target_stride;            // [n]; outside [0, v): none
    int k;
    float* log_probs; float* entropy; float* lse; float* rest;  // [n]
    int* top; float* top_log_probs;                    // [n x k]
    char* ws;                                          // rate_workspace() bytes
};
hipError_t launch_rate(const RateCall& a, hipStream_t s);
size_t rate_workspace(long n, int v, int type, int k);
// Whether every launch of both directions has a grid that the device takes.
bool rate_fits(long n, int v, int type, int k);

struct RateBackCall {
    const void* z; int type; long n; int v; long ld;
    const int* targets; long target_stride;
    const float* lse; const float* rest; const float* entropy;   // launch_rate's
    const float* dlog; const float* dent; const float* dlse;     // nullable, [n]
    void* dz; long ld_dz;                              // [n x v]; may be z
};
hipError_t launch_rate_back(const RateBackCall& a, hipStream_t s);

}  // namespace skm
