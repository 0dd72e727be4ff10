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
};
struct B16 {
    typedef uint16_t Raw;
};
struct F16 {
    typedef uint16_t Raw;
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

__device__ __forceinline__ float WaveMax(float v)
{
    for (int d = 32; d > 0; d >>= 1) {
        v = fmaxf(v, __shfl_xor(v, d));
    }
    return v;
}
__device__ __forceinline__ float WaveSum(float v)
{
    for (int d = 32; d > 0; d >>= 1) {
        v += __shfl_xor(v, d);
    }
    return v;
}
__device__ __forceinline__ double WaveSum(double v)
{
    for (int d = 32; d > 0; d >>= 1) {
        v += __shfl_xor(v, d);
    }
    return v;
}

// 2^x, one instruction (results below 2^-126 become 0).
__device__ __forceinline__ float Exp2(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace model_ops
}  // namespace hccl_amd
