// Stand-in for <hip/hip_runtime.h> for the kernels of hccl_amd/csrc/model_ops in the CPU emulation: test infrastructure
// only.  The runtime API is that of ../../hip/hip_runtime.h; the execution engine is another one (lanes.cc), because these
// kernels exchange values between the lanes of a wavefront all the time.  Here every lane of a workgroup is a fiber of one
// thread, which stops at cross-lane operations until its wavefront has arrived, and at barriers until all have.
#pragma once

#include <math.h>

#include "../../hip/hip_runtime.h"

#undef threadIdx
#undef blockIdx
#undef gridDim
#undef blockDim
#undef __syncthreads
#undef hipLaunchKernelGGL

namespace lanes {
struct Idx {
    unsigned x, y, z;
};
extern Idx g_thread, g_block;      // of the lane in progress

// Runs body() for every lane of every workgroup.  The wavefronts take turns between barriers in an order that changes with
// every turn.
void Launch(dim3 grid, dim3 block, size_t ldsBytes, const std::function<void()>& body);
void SyncThreads();
void* DynamicLds();
// Hands `value` to the wavefront; returns the values of all its lanes, and in `active` which of them take part.
const uint32_t* Exchange(uint32_t value, int site, uint64_t* active, unsigned* lane);

uint32_t UpdateDpp(uint32_t old, uint32_t src, int control, int rowMask, int bankMask, bool boundControl,
                   int site = __builtin_LINE());
uint64_t Ballot(bool value, int site = __builtin_LINE());
uint32_t ReadLane(uint32_t v, uint32_t from, int site = __builtin_LINE());
uint32_t ReadFirstLane(uint32_t v, int site = __builtin_LINE());
uint32_t ShuffleXor(uint32_t v, unsigned distance, int site = __builtin_LINE());
struct Pair {
    uint32_t x, y;
};
Pair SwapRows(uint32_t a, uint32_t b, unsigned distance, int site);
inline Pair Permlane16Swap(uint32_t a, uint32_t b, bool, bool, int site = __builtin_LINE()) { return SwapRows(a, b, 16, site); }
inline Pair Permlane32Swap(uint32_t a, uint32_t b, bool, bool, int site = __builtin_LINE()) { return SwapRows(a, b, 32, site); }
float WidenFp8(int word, int byte);                            // e4m3 with NaN and without infinities
int NarrowFp8Pair(float a, float b, int old, bool upper);      // to nearest even, of what rounds to at most 448
inline float Reciprocal(float x) { return 1.0f / x; }
}  // namespace lanes

#define threadIdx (lanes::g_thread)
#define blockIdx (lanes::g_block)
#define __syncthreads() lanes::SyncThreads()
#define __ballot(x) lanes::Ballot((x) != 0)
#define __shfl_xor(v, distance) lanes::ShuffleXor(v, distance)
#define __ffsll(x) __builtin_ffsll(static_cast<long long>(x))
#define __popc(x) __builtin_popcount(x)
#define hipLaunchKernelGGL(kernel, grid, block, ldsBytes, stream, ...) \
    lanes::Launch((grid), (block), (ldsBytes), [&] { kernel(__VA_ARGS__); })

// On LDS: one lane runs at a time.
template <typename T>
inline T atomicAdd(T* p, T v)
{
    const T old = *p;
    *p = old + v;
    return old;
}
