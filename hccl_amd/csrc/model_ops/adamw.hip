// One AdamW step over a batch of tensors, states in 32 bits or as e4m3 codes with a scale per 256 elements.
//
// Purely elementwise but for the scales.  A lane owns four neighbouring elements, 16 bytes of a 32-bit tensor, so that every
// access of a wavefront is one run of memory, and a wavefront owns a state block of 256: its largest magnitude takes six
// exchanges between lanes and no memory.  m and v are updated in 32 bits and rounded once on the way out; the weights take
// the unrounded ones.  Of v the root is stored: that halves the exponents it needs, and it is what the step divides by.  A
// root above zero is stored as at least the smallest code: rounded to zero it would leave m / eps as a step.
// The states' products and sums are rounded one by one, and on the way to codes the root and the quotients too: the states
// are then the bits that elementwise 32-bit operations give.  One bit more or less can decide between two codes, 6 %
// apart, and one step later between two scales.  (With fused operations and the one-instruction root, four steps on 2^27
// weights left 1371 codes and two scales that were not the same; 1 % faster with FP8 states, equally fast with 32-bit
// ones.)  In the weights' step the reciprocal, and with 32-bit states the root, are the one-instruction forms (1 ulp): it
// is 1e-7 of itself off, the weight far less.  A v below 2^-126 is scaled for that root, which would be 0 and leave m / eps
// as a step.  (With the correctly rounded root a call for 300 000 weights in 24 tensors
// takes 6.5 us instead of 5.6, the 2^27 weights below as long.)
//
// Bound: every tensor read once and the updated ones written once.  2^27 bf16 weights in 300 tensors with 32-bit master
// weights, four launches: 632 us, 5.9 TB/s of the 6.0 - 6.7 that a copy reaches; with FP8 states 378 us, 5.7 TB/s.  (A lane
// with eight neighbours, two 16-byte accesses 32 bytes apart: 790 and 486.  Chunks of 1024 elements 631 and 393, of 4096
// 676 and 396; stores written through 651 and 391, plain ones 701 and 414.)
#include "model_ops.h"
#include "vec.h"

namespace hccl_amd {
namespace model_ops {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kPer = 4;                                   // elements of a lane
constexpr uint32_t kSteps = kAdamWChunk / (kThreads * kPer);   // per workgroup
constexpr uint32_t kBlock = HCCL_AMD_STATE_BLOCK;
constexpr float kCodeMax = 448.0f;           // largest e4m3 value
constexpr float kCodeMin = 0.001953125f;     // smallest above 0
constexpr float kNoUnit = 1e-35f;            // below it 448 / x is beyond a float: such a block counts as zero
static_assert(kBlock == kWave * kPer && kAdamWChunk % kBlock == 0, "a block is a wavefront and never leaves its chunk");

// Four elements from element `at`, of which `n` (0 .. 4, or more) are in the tensor; the others are 0.
template <typename T>
__device__ __forceinline__ void Load4(uint64_t base, uint64_t at, uint32_t n, float* x)
{
    typedef typename T::Raw Raw;
    const Raw* p = reinterpret_cast<const Raw*>(base) + at;
    if (n >= kPer) {
        if constexpr (sizeof(Raw) == 4) {
            Unpack16<T>(LoadOnce16(p), x);
        } else {
            const U32x2 raw = LoadOnce8(p);
            for (uint32_t i = 0; i < 2; ++i) {
                const uint32_t word = raw[i];
                x[2 * i] = Widen<T>(static_cast<uint16_t>(word & 0xFFFFu));
                x[2 * i + 1] = Widen<T>(static_cast<uint16_t>(word >> 16));
            }
        }
    } else {
        for (uint32_t i = 0; i < kPer; ++i) {
            x[i] = i < n ? Widen<T>(LoadOne(p + i)) : 0.0f;
        }
    }
}

template <typename T>
__device__ __forceinline__ void Store4(uint64_t base, uint64_t at, uint32_t n, const float* x)
{
    typedef typename T::Raw Raw;
    Raw* p = reinterpret_cast<Raw*>(base) + at;
    if (n >= kPer) {
        if constexpr (sizeof(Raw) == 4) {
            StoreOnce16(p, Pack16<T>(x));
        } else {
            U32x2 raw;
            for (uint32_t i = 0; i < 2; ++i) {
                raw[i] = static_cast<uint32_t>(Narrow<T>(x[2 * i])) | (static_cast<uint32_t>(Narrow<T>(x[2 * i + 1])) << 16);
            }
            StoreOnce8(p, raw);
        }
    } else {
        for (uint32_t i = 0; i < kPer; ++i) {
            if (i < n) {
                StoreOne(p + i, Narrow<T>(x[i]));
            }
        }
    }
}

typedef uint32_t CodesAny __attribute__((aligned(1)));
__device__ __forceinline__ uint32_t LoadCodes(uint64_t base, uint64_t at, uint32_t n)
{
    const uint8_t* p = reinterpret_cast<const uint8_t*>(base) + at;
    if (n >= kPer) {
        return __builtin_nontemporal_load((const HCCL_AMD_GLOBAL CodesAny*)p);
    }
    uint32_t codes = 0;
    for (uint32_t i = 0; i < kPer; ++i) {
        codes |= i < n ? static_cast<uint32_t>(LoadOne(p + i)) << (8 * i) : 0u;
    }
    return codes;
}

__device__ __forceinline__ void Decode(uint32_t codes, float scale, float* x)
{
    x[0] = scale * __builtin_amdgcn_cvt_f32_fp8(codes, 0);
    x[1] = scale * __builtin_amdgcn_cvt_f32_fp8(codes, 1);
    x[2] = scale * __builtin_amdgcn_cvt_f32_fp8(codes, 2);
    x[3] = scale * __builtin_amdgcn_cvt_f32_fp8(codes, 3);
}

__device__ __forceinline__ void StoreCodes(uint64_t base, uint64_t at, uint32_t n, const float* x)
{
    uint8_t* p = reinterpret_cast<uint8_t*>(base) + at;
    int packed = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    packed = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], packed, true);
    const uint32_t codes = static_cast<uint32_t>(packed);
    if (n >= kPer) {
        __builtin_nontemporal_store(codes, (HCCL_AMD_GLOBAL CodesAny*)p);
    } else {
        for (uint32_t i = 0; i < kPer; ++i) {
            if (i < n) {
                StoreOne(p + i, static_cast<uint8_t>(codes >> (8 * i)));
            }
        }
    }
}

// The root in one instruction (1 ulp), which takes what is below the smallest normal number as 0: that is scaled for it.
__device__ __forceinline__ float Root(float v)
{
    const bool small = v < 0x1p-126f;
    return __builtin_amdgcn_sqrtf(small ? v * 0x1p64f : v) * (small ? 0x1p-32f : 1.0f);
}

// Largest magnitude of a block.
__device__ __forceinline__ float BlockMax(const float* x)
{
    return LaneMax(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
}

template <typename P, typename G, bool kMaster, bool kFp8>
__global__ __launch_bounds__(kThreads) void AdamWKernel(const AdamWArgs a)
{
    constexpr uint32_t kStride = AdamWTensorWords(kMaster, kFp8);
    uint32_t lo = 0, hi = a.nTensors - 1;      // the first tensor that ends behind this chunk
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (static_cast<uint32_t>(a.table[mid * kStride]) > blockIdx.x) {
            hi = mid;
        } else {
            lo = mid + 1;
        }
    }
    const uint64_t* t = a.table + lo * kStride;
    const uint32_t chunk = blockIdx.x - (lo == 0 ? 0u : static_cast<uint32_t>(a.table[(lo - 1) * kStride]));
    const uint64_t begin = static_cast<uint64_t>(chunk) * kAdamWChunk;
    const uint32_t inChunk = blockIdx.x + 1 == static_cast<uint32_t>(t[0]) ? static_cast<uint32_t>(t[0] >> 32) : kAdamWChunk;
    const uint64_t param = t[1], grad = t[2], expAvg = t[3], expAvgSq = t[4];
    const uint64_t weights = kMaster ? t[5] : param;
    float* const mScales = kFp8 ? reinterpret_cast<float*>(t[kStride - 2]) : nullptr;
    float* const vScales = kFp8 ? reinterpret_cast<float*>(t[kStride - 1]) : nullptr;

    // everything is on its way before the step's numbers are
    float w[kSteps][kPer], g[kSteps][kPer], m[kSteps][kPer], v[kSteps][kPer], mScale[kSteps], vScale[kSteps];
    uint32_t mCodes[kSteps], vCodes[kSteps];
    for (uint32_t s = 0; s < kSteps; ++s) {
        const uint32_t off = (s * kThreads + threadIdx.x) * kPer;
        const uint64_t at = begin + off;
        const uint32_t n = off < inChunk ? inChunk - off : 0;
        if constexpr (kMaster) {
            Load4<F32>(weights, at, n, w[s]);
        } else {
            Load4<P>(weights, at, n, w[s]);
        }
        Load4<G>(grad, at, n, g[s]);
        if constexpr (kFp8) {
            mCodes[s] = LoadCodes(expAvg, at, n);
            vCodes[s] = LoadCodes(expAvgSq, at, n);
            mScale[s] = n != 0 ? LoadOne(mScales + at / kBlock) : 0.0f;
            vScale[s] = n != 0 ? LoadOne(vScales + at / kBlock) : 0.0f;
        } else {
            Load4<F32>(expAvg, at, n, m[s]);
            Load4<F32>(expAvgSq, at, n, v[s]);
        }
    }

    float clip = 1.0f;
    if (a.clip != nullptr) {
        if (a.skipNonFinite && !(fabsf(LoadOne(a.clip)) < __builtin_inff())) {
            return;
        }
        clip = LoadOne(a.clip + 1);
    }
    const float lr = a.lr != nullptr ? LoadOne(a.lr) : a.hostLr;
    float correction1 = a.correction1, rootCorrection2 = a.rootCorrection2;
    if (a.step != nullptr) {
        const float step = static_cast<float>(LoadOne(a.step));
        correction1 = -1.0f / expm1f(step * a.logBeta1);
        rootCorrection2 = 1.0f / sqrtf(-expm1f(step * a.logBeta2));
    }
    const float rate = lr * correction1, keep = 1.0f - lr * a.weightDecay;

    for (uint32_t s = 0; s < kSteps; ++s) {
        const uint32_t off = (s * kThreads + threadIdx.x) * kPer;
        const uint64_t at = begin + off;
        const uint32_t n = off < inChunk ? inChunk - off : 0;
        if constexpr (kFp8) {
            Decode(mCodes[s], mScale[s], m[s]);
            Decode(vCodes[s], vScale[s], v[s]);
        }
        float root[kPer];
        for (uint32_t i = 0; i < kPer; ++i) {
            if constexpr (kFp8) {
                v[s][i] *= v[s][i];
            }
            const float gi = g[s][i] * clip;
            m[s][i] = m[s][i] * a.beta1 + gi * a.oneMinusBeta1;
            v[s][i] = v[s][i] * a.beta2 + gi * gi * a.oneMinusBeta2;
            root[i] = kFp8 ? sqrtf(v[s][i]) : Root(v[s][i]);
            const float step = m[s][i] * __builtin_amdgcn_rcpf(__builtin_fmaf(root[i], rootCorrection2, a.eps));
            w[s][i] = __builtin_fmaf(-rate, step, w[s][i] * keep);
            if constexpr (kMaster) {
                // The 16-bit weights are the rounded master weights: without this the compiler rounds the fused
                // multiply-add to 16 bits in one instruction, past the 32-bit value.
                asm("" : "+v"(w[s][i]));
            }
        }
        if constexpr (kFp8) {
            // (places behind the tensor's end have zeros)
            for (uint32_t i = 0; i < kPer; ++i) {
                m[s][i] = i < n ? m[s][i] : 0.0f;
                root[i] = i < n ? root[i] : 0.0f;
            }
            const float mMost = BlockMax(m[s]), vMost = BlockMax(root);
            const float mUnit = mMost > kNoUnit ? 1.0f / mMost * kCodeMax : 0.0f;
            const float vUnit = vMost > kNoUnit ? 1.0f / vMost * kCodeMax : 0.0f;
            for (uint32_t i = 0; i < kPer; ++i) {
                m[s][i] *= mUnit;
                root[i] = root[i] > 0.0f ? fmaxf(root[i] * vUnit, kCodeMin) : root[i];
            }
            if (n != 0 && threadIdx.x % kWave == 0) {
                StoreOne(mScales + at / kBlock, mMost * (1.0f / kCodeMax));
                StoreOne(vScales + at / kBlock, vMost * (1.0f / kCodeMax));
            }
        }
        if (n != 0) {
            Store4<P>(param, at, n, w[s]);
            if constexpr (kMaster) {
                Store4<F32>(weights, at, n, w[s]);
            }
            if constexpr (kFp8) {
                StoreCodes(expAvg, at, n, m[s]);
                StoreCodes(expAvgSq, at, n, root);
            } else {
                Store4<F32>(expAvg, at, n, m[s]);
                Store4<F32>(expAvgSq, at, n, v[s]);
            }
        }
    }
}

template <typename P, typename G, bool kMaster>
void LaunchState(const AdamWArgs& a, bool fp8State, uint32_t chunks, hipStream_t stream)
{
    if (fp8State) {
        hipLaunchKernelGGL((AdamWKernel<P, G, kMaster, true>), dim3(chunks), dim3(kThreads), 0, stream, a);
    } else {
        hipLaunchKernelGGL((AdamWKernel<P, G, kMaster, false>), dim3(chunks), dim3(kThreads), 0, stream, a);
    }
}

}  // namespace

hipError_t LaunchAdamW(const AdamWArgs& a, HcclDataType paramType, HcclDataType gradType, bool master, bool fp8State,
                       uint32_t chunks, hipStream_t stream)
{
    if (paramType == HCCL_DATA_TYPE_FP32) {
        switch (gradType) {
            case HCCL_DATA_TYPE_FP32: LaunchState<F32, F32, false>(a, fp8State, chunks, stream); break;
            case HCCL_DATA_TYPE_BFP16: LaunchState<F32, B16, false>(a, fp8State, chunks, stream); break;
            default: LaunchState<F32, F16, false>(a, fp8State, chunks, stream); break;
        }
    } else if (paramType == HCCL_DATA_TYPE_BFP16) {
        if (gradType == HCCL_DATA_TYPE_FP32) {
            master ? LaunchState<B16, F32, true>(a, fp8State, chunks, stream)
                   : LaunchState<B16, F32, false>(a, fp8State, chunks, stream);
        } else {
            master ? LaunchState<B16, B16, true>(a, fp8State, chunks, stream)
                   : LaunchState<B16, B16, false>(a, fp8State, chunks, stream);
        }
    } else {
        if (gradType == HCCL_DATA_TYPE_FP32) {
            master ? LaunchState<F16, F32, true>(a, fp8State, chunks, stream)
                   : LaunchState<F16, F32, false>(a, fp8State, chunks, stream);
        } else {
            master ? LaunchState<F16, F16, true>(a, fp8State, chunks, stream)
                   : LaunchState<F16, F16, false>(a, fp8State, chunks, stream);
        }
    }
    return hipGetLastError();
}

}  // namespace model_ops
}  // namespace hccl_amd
