// Device helpers of the model operators: 16-byte vectors of any element type that may start on any element, conversions,
// and reductions over a wavefront.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace hccl_amd {
namespace model_ops {

#define HCCL_AMD_GLOBAL __attribute__((address_space(1)))
typedef uint32_t U32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t U32x4 __attribute__((ext_vector_type(4)));
typedef U32x2 U32x2Any __attribute__((aligned(1)));
typedef U32x4 U32x4Any __attribute__((aligned(1)));

constexpr uint32_t kWave = 64;

struct F32 {
    typedef uint32_t Raw;
    static constexpr bool kHalf = false;
};
struct B16 {
    typedef uint16_t Raw;
    static constexpr bool kHalf = false;
};
struct F16 {
    typedef uint16_t Raw;
    static constexpr bool kHalf = true;
};

template <typename T>
__device__ __forceinline__ float Widen(typename T::Raw r);
template <>
__device__ __forceinline__ float Widen<F32>(uint32_t r)
{
    return __builtin_bit_cast(float, r);
}
template <>
__device__ __forceinline__ float Widen<B16>(uint16_t r)
{
    return __builtin_bit_cast(float, static_cast<uint32_t>(r) << 16);
}
template <>
__device__ __forceinline__ float Widen<F16>(uint16_t r)
{
    return static_cast<float>(__builtin_bit_cast(_Float16, r));
}

// Rounds once to the element type, to nearest even; a value beyond the type's range becomes an infinity.
template <typename T>
__device__ __forceinline__ typename T::Raw Narrow(float f);
template <>
__device__ __forceinline__ uint32_t Narrow<F32>(float f)
{
    return __builtin_bit_cast(uint32_t, f);
}
template <>
__device__ __forceinline__ uint16_t Narrow<B16>(float f)
{
    return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f));
}
template <>
__device__ __forceinline__ uint16_t Narrow<F16>(float f)
{
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
}

// Elements of a 16-byte vector.
template <typename T>
constexpr uint32_t kPer16 = 16 / sizeof(typename T::Raw);

template <typename T>
__device__ __forceinline__ void Unpack16(U32x4 raw, float* x)
{
    if constexpr (sizeof(typename T::Raw) == 4) {
        for (int i = 0; i < 4; ++i) {
            const uint32_t word = raw[i];     // (a bit cast of the vector's element itself reads element 0)
            x[i] = __builtin_bit_cast(float, word);
        }
    } else {
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = Widen<T>(static_cast<uint16_t>(raw[i] & 0xFFFFu));
            x[2 * i + 1] = Widen<T>(static_cast<uint16_t>(raw[i] >> 16));
        }
    }
}

template <typename T>
__device__ __forceinline__ U32x4 Pack16(const float* x)
{
    U32x4 raw;
    if constexpr (sizeof(typename T::Raw) == 4) {
        for (int i = 0; i < 4; ++i) {
            raw[i] = __builtin_bit_cast(uint32_t, x[i]);
        }
    } else {
        for (int i = 0; i < 4; ++i) {
            raw[i] = static_cast<uint32_t>(Narrow<T>(x[2 * i])) | (static_cast<uint32_t>(Narrow<T>(x[2 * i + 1])) << 16);
        }
    }
    return raw;
}

// Accesses that leave the caches to others: everything here is touched once.  Any address is allowed.
__device__ __forceinline__ U32x4 LoadOnce16(const void* p)
{
    return __builtin_nontemporal_load((const HCCL_AMD_GLOBAL U32x4Any*)p);
}
__device__ __forceinline__ U32x4 Load16(const void* p) { return *((const HCCL_AMD_GLOBAL U32x4Any*)p); }
__device__ __forceinline__ void StoreOnce16(void* p, U32x4 v)
{
    __builtin_nontemporal_store(v, (HCCL_AMD_GLOBAL U32x4Any*)p);
}
__device__ __forceinline__ U32x2 LoadOnce8(const void* p)
{
    return __builtin_nontemporal_load((const HCCL_AMD_GLOBAL U32x2Any*)p);
}
__device__ __forceinline__ void StoreOnce8(void* p, U32x2 v)
{
    __builtin_nontemporal_store(v, (HCCL_AMD_GLOBAL U32x2Any*)p);
}
template <typename V>
__device__ __forceinline__ V LoadOne(const V* p)
{
    return *((const HCCL_AMD_GLOBAL V*)p);
}
template <typename V>
__device__ __forceinline__ void StoreOne(V* p, V v)
{
    *((HCCL_AMD_GLOBAL V*)p) = v;
}

// The value of lane (lane ^ D), for D a power of two, without LDS: permutations within four and sixteen lanes that the
// vector ALU applies to an operand, and the exchanges of 16- and 32-lane rows.
template <int kControl>
__device__ __forceinline__ uint32_t Dpp(uint32_t v)
{
    return __builtin_amdgcn_update_dpp(0, v, kControl, 0xF, 0xF, true);
}
constexpr int kQuadXor1 = 0xB1, kQuadXor2 = 0x4E, kQuadXor3 = 0x1B, kHalfMirror = 0x141, kMirror = 0x140, kRotate8 = 0x128;

// Both values of a pair of lanes 16 or 32 apart: x is the lower lane's, y the upper lane's, on both.
template <uint32_t D>
__device__ __forceinline__ U32x2 RowPair(uint32_t v)
{
    if constexpr (D == 16) {
        return __builtin_bit_cast(U32x2, __builtin_amdgcn_permlane16_swap(v, v, false, false));
    } else {
        return __builtin_bit_cast(U32x2, __builtin_amdgcn_permlane32_swap(v, v, false, false));
    }
}

template <uint32_t D>
__device__ __forceinline__ uint32_t XorLane(uint32_t v)
{
    if constexpr (D == 1) {
        return Dpp<kQuadXor1>(v);
    } else if constexpr (D == 2) {
        return Dpp<kQuadXor2>(v);
    } else if constexpr (D == 4) {
        return Dpp<kQuadXor3>(Dpp<kHalfMirror>(v));     // 7 ^ 3
    } else if constexpr (D == 8) {
        return Dpp<kRotate8>(v);
    } else {
        const U32x2 pair = RowPair<D>(v);
        return (threadIdx.x & D) == 0 ? pair.y : pair.x;
    }
}
template <uint32_t D>
__device__ __forceinline__ float XorLane(float v)
{
    return __builtin_bit_cast(float, XorLane<D>(__builtin_bit_cast(uint32_t, v)));
}
template <uint32_t D>
__device__ __forceinline__ double XorLane(double v)
{
    const U32x2 w = __builtin_bit_cast(U32x2, v);
    return __builtin_bit_cast(double, U32x2{XorLane<D>(w.x), XorLane<D>(w.y)});
}

// Reductions over a wavefront; every lane gets the result, and all the same bits (the operands of a pair only change places).
__device__ __forceinline__ float Larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ uint32_t Larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <typename V>
__device__ __forceinline__ V LaneMax(V v)
{
    v = Larger(v, XorLane<1>(v));
    v = Larger(v, XorLane<2>(v));
    v = Larger(v, XorLane<4>(v));
    v = Larger(v, XorLane<8>(v));
    v = Larger(v, XorLane<16>(v));
    return Larger(v, XorLane<32>(v));
}
template <typename V>
__device__ __forceinline__ V WaveSum(V v)
{
    v += XorLane<1>(v);
    v += XorLane<2>(v);
    v += XorLane<4>(v);
    v += XorLane<8>(v);
    v += XorLane<16>(v);
    v += XorLane<32>(v);
    return v;
}

// Sum over the lanes up to and including the own one.
template <int kControl, int kRows>
__device__ __forceinline__ uint32_t FromLower(uint32_t v)
{
    return __builtin_amdgcn_update_dpp(0, v, kControl, kRows, 0xF, false);      // 0 where there is no such lane
}
__device__ __forceinline__ uint32_t WaveScan(uint32_t v)
{
    v += FromLower<0x111, 0xF>(v);      // shifts by 1, 2, 4, 8 within sixteen lanes
    v += FromLower<0x112, 0xF>(v);
    v += FromLower<0x114, 0xF>(v);
    v += FromLower<0x118, 0xF>(v);
    v += FromLower<0x142, 0xA>(v);      // the last lane of rows 0 and 2 to rows 1 and 3
    v += FromLower<0x143, 0xC>(v);      // lane 31 to the upper half
    return v;
}

// 2^x, one instruction (results below 2^-126 become 0).
__device__ __forceinline__ float Exp2(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace model_ops
}  // namespace hccl_amd
