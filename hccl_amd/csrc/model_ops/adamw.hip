// One AdamW step over a batch of tensors, states in 32 bits or as e4m3 codes with a scale per 256 elements.
//
// Purely elementwise but for the scales.  A lane owns eight neighbouring elements, a wavefront 512, so that a block of 256
// is half a wavefront: its largest magnitude takes five exchanges between lanes and no memory.  m and v are updated in
// 32 bits and rounded once on the way out; the weights take the unrounded ones.  Of v the root is stored: that halves the
// exponents it needs, and it is what the step divides by.  A root above zero is stored as at least the smallest code:
// rounded to zero it would leave m / eps as a step.
// Square root and reciprocal are the one-instruction forms (1 ulp): the step is 1e-7 of itself off, the weight far less.
// Bound: every tensor read once and the updated ones written once.
#include "model_ops.h"
#include "vec.h"

namespace hccl_amd {
namespace model_ops {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kPer = 8;                                   // elements of a lane
constexpr uint32_t kSteps = kAdamWChunk / (kThreads * kPer);   // per workgroup
constexpr uint32_t kBlock = HCCL_AMD_STATE_BLOCK;
constexpr uint32_t kBlockLanes = kBlock / kPer;
constexpr float kCodeMax = 448.0f;           // largest e4m3 value
constexpr float kCodeMin = 0.001953125f;     // smallest above 0
constexpr float kNoUnit = 1e-35f;            // below it 448 / x is beyond a float: such a block counts as zero
static_assert(kBlockLanes == 32 && kAdamWChunk % kBlock == 0, "a block is half a wavefront and never leaves its chunk");

// Eight elements from element `at`, which has `n` (1 .. 8) left in the tensor.
template <typename T>
__device__ __forceinline__ void Load8(const void* base, uint64_t at, uint32_t n, float* x)
{
    typedef typename T::Raw Raw;
    const Raw* p = static_cast<const Raw*>(base) + at;
    if (n >= kPer) {
        Unpack16<T>(LoadOnce16(p), x);
        if constexpr (sizeof(Raw) == 4) {
            Unpack16<T>(LoadOnce16(p + 4), x + 4);
        }
    } else {
        for (uint32_t i = 0; i < kPer; ++i) {
            x[i] = i < n ? Widen<T>(LoadOne(p + i)) : 0.0f;
        }
    }
}

template <typename T>
__device__ __forceinline__ void Store8(void* base, uint64_t at, uint32_t n, const float* x)
{
    typedef typename T::Raw Raw;
    Raw* p = static_cast<Raw*>(base) + at;
    if (n >= kPer) {
        StoreOnce16(p, Pack16<T>(x));
        if constexpr (sizeof(Raw) == 4) {
            StoreOnce16(p + 4, Pack16<T>(x + 4));
        }
    } else {
        for (uint32_t i = 0; i < kPer; ++i) {
            if (i < n) {
                StoreOne(p + i, Narrow<T>(x[i]));
            }
        }
    }
}

__device__ __forceinline__ void LoadCodes(const void* base, uint64_t at, uint32_t n, float* x)
{
    const uint8_t* p = static_cast<const uint8_t*>(base) + at;
    U32x2 raw = {0, 0};
    if (n >= kPer) {
        raw = LoadOnce8(p);
    } else {
        for (uint32_t i = 0; i < kPer; ++i) {
            const uint32_t code = i < n ? LoadOne(p + i) : 0;
            raw[i / 4] |= code << (8 * (i % 4));
        }
    }
    for (uint32_t w = 0; w < 2; ++w) {
        x[4 * w] = __builtin_amdgcn_cvt_f32_fp8(raw[w], 0);
        x[4 * w + 1] = __builtin_amdgcn_cvt_f32_fp8(raw[w], 1);
        x[4 * w + 2] = __builtin_amdgcn_cvt_f32_fp8(raw[w], 2);
        x[4 * w + 3] = __builtin_amdgcn_cvt_f32_fp8(raw[w], 3);
    }
}

__device__ __forceinline__ void StoreCodes(void* base, uint64_t at, uint32_t n, const float* x)
{
    uint8_t* p = static_cast<uint8_t*>(base) + at;
    U32x2 raw;
    for (uint32_t w = 0; w < 2; ++w) {
        int packed = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * w], x[4 * w + 1], 0, false);
        packed = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * w + 2], x[4 * w + 3], packed, true);
        raw[w] = static_cast<uint32_t>(packed);
    }
    if (n >= kPer) {
        StoreOnce8(p, raw);
    } else {
        for (uint32_t i = 0; i < kPer; ++i) {
            if (i < n) {
                StoreOne(p + i, static_cast<uint8_t>(raw[i / 4] >> (8 * (i % 4))));
            }
        }
    }
}

// Largest of the eight magnitudes over the 32 lanes of a block.
__device__ __forceinline__ float BlockMax(const float* x)
{
    float most = fabsf(x[0]);
    for (uint32_t i = 1; i < kPer; ++i) {
        most = fmaxf(most, fabsf(x[i]));
    }
    for (uint32_t d = kBlockLanes / 2; d > 0; d >>= 1) {
        most = fmaxf(most, __shfl_xor(most, d));
    }
    return most;
}

template <typename P, typename G, bool kMaster, bool kFp8>
__global__ __launch_bounds__(kThreads) void AdamWKernel(const AdamWArgs a)
{
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

    uint32_t lo = 0, hi = a.nTensors - 1;      // the first tensor that ends behind this chunk
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (a.chunkEnd[mid] > blockIdx.x) {
            hi = mid;
        } else {
            lo = mid + 1;
        }
    }
    const AdamWArgs::Tensor& t = a.t[lo];
    const uint64_t begin = static_cast<uint64_t>(blockIdx.x - (lo == 0 ? 0 : a.chunkEnd[lo - 1])) * kAdamWChunk;
    const uint64_t left = t.count - begin;
    const uint32_t inChunk = left < kAdamWChunk ? static_cast<uint32_t>(left) : kAdamWChunk;

    for (uint32_t s = 0; s < kSteps; ++s) {
        const uint32_t off = (s * kThreads + threadIdx.x) * kPer;
        const uint64_t at = begin + off;
        const uint32_t n = off < inChunk ? inChunk - off : 0;
        float w[kPer], g[kPer], m[kPer], v[kPer];
        float mScale = 0.0f, vScale = 0.0f;
        if (n != 0) {
            if constexpr (kMaster) {
                Load8<F32>(t.master, at, n, w);
            } else {
                Load8<P>(t.param, at, n, w);
            }
            Load8<G>(t.grad, at, n, g);
            if constexpr (kFp8) {
                LoadCodes(t.m, at, n, m);
                LoadCodes(t.v, at, n, v);
                mScale = LoadOne(t.mScale + at / kBlock);
                vScale = LoadOne(t.vScale + at / kBlock);
            } else {
                Load8<F32>(t.m, at, n, m);
                Load8<F32>(t.v, at, n, v);
            }
        } else {
            for (uint32_t i = 0; i < kPer; ++i) {
                w[i] = g[i] = m[i] = v[i] = 0.0f;
            }
        }
        float root[kPer];
        for (uint32_t i = 0; i < kPer; ++i) {
            if constexpr (kFp8) {
                m[i] *= mScale;
                v[i] *= vScale;
                v[i] *= v[i];
            }
            const float gi = g[i] * clip;
            m[i] = __builtin_fmaf(m[i], a.beta1, gi * a.oneMinusBeta1);
            v[i] = __builtin_fmaf(v[i], a.beta2, gi * gi * a.oneMinusBeta2);
            root[i] = __builtin_amdgcn_sqrtf(v[i]);
            const float step = m[i] * __builtin_amdgcn_rcpf(__builtin_fmaf(root[i], rootCorrection2, a.eps));
            w[i] = __builtin_fmaf(-rate, step, w[i] * keep);
            if constexpr (kMaster) {
                // The 16-bit weights are the rounded master weights: without this the compiler rounds the fused
                // multiply-add to 16 bits in one instruction, past the 32-bit value.
                asm("" : "+v"(w[i]));
            }
        }
        if constexpr (kFp8) {
            const float mMost = BlockMax(m), vMost = BlockMax(root);
            const float mUnit = mMost > kNoUnit ? kCodeMax / mMost : 0.0f, vUnit = vMost > kNoUnit ? kCodeMax / vMost : 0.0f;
            for (uint32_t i = 0; i < kPer; ++i) {
                m[i] *= mUnit;
                root[i] = root[i] > 0.0f ? fmaxf(root[i] * vUnit, kCodeMin) : root[i];
            }
            if (n != 0 && threadIdx.x % kBlockLanes == 0) {
                StoreOne(t.mScale + at / kBlock, mMost / kCodeMax);
                StoreOne(t.vScale + at / kBlock, vMost / kCodeMax);
            }
        }
        if (n != 0) {
            Store8<P>(t.param, at, n, w);
            if constexpr (kMaster) {
                Store8<F32>(t.master, at, n, w);
            }
            if constexpr (kFp8) {
                StoreCodes(t.m, at, n, m);
                StoreCodes(t.v, at, n, root);
            } else {
                Store8<F32>(t.m, at, n, m);
                Store8<F32>(t.v, at, n, v);
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
