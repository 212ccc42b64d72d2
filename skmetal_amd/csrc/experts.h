// experts.h -- the operators of skmetal_amd.experts: argument blocks and launchers
// (route_kernels.hip, adapt_kernels.hip).  Everything is in device memory and every
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

}  // namespace skm
