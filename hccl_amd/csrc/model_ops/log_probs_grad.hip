// Gradient of log probabilities, entropy and alternatives with respect to one rank's part of the logits:
//   d_v = scale ( one-hot terms - p_v (a + e (log p_v + H)) ),  log p_v = scale x_v - lse,  a = g + sum_j h_j.
//
// log p_v takes one rounding from the given lse, and has what that lacks: the 32-bit lse is |lse| 2^-24 off, and every p_v by
// that share.  Beside a p near 1 it is all that 1 - p is right to (1 - p = 1e-5 at lse 40: 20 % off; 1e-2: 2e-4).
//
// Every element needs its logit and half a dozen numbers of its row, so the part is cut into chunks that know nothing of
// each other.  The one-hot terms are added in 32 bits before the only rounding: lane j of every wavefront fetches the j-th
// term of the row, and those that fall into the chunk (rarely any) are walked one by one.
//
// Bound: one read and one write per element; a copy of 1 GiB runs at 6.5 TB/s here with one vector per lane and stores past
// the caches, at 6.0 with four.  A chunk is two vectors per lane, which measured best for 4096 x 131072 bf16 in eight parts
// and for 1001 x 50001 in three, rows on any element, with eight alternatives: 349 us (6.2 TB/s) and 48 us; one vector 357
// and 49, four 353 and 52, stores written through 351 and 52, vectors cut on the gradient's 16-byte lines 351 and 49.
#include "model_ops.h"
#include "vec.h"

namespace hccl_amd {
namespace model_ops {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kUnroll = 2;          // vectors of a lane, see above
constexpr float kLog2E = 1.44269504088896341f;
constexpr float kMaskedRow = -1e30f;      // logSumExp of a row in which no entry can occur
constexpr float kNoProb = -1000.0f;      // log p below this has p = 0 in 32 bits; keeps -inf out of products with p

__device__ __forceinline__ int64_t IdAt(const void* ids, uint32_t wide, uint64_t at)
{
    return wide ? LoadOne(static_cast<const int64_t*>(ids) + at) : LoadOne(static_cast<const int32_t*>(ids) + at);
}

template <typename T, bool kTop>
__global__ __launch_bounds__(kThreads) void LogProbsGradKernel(const LogProbsGradArgs a, uint32_t chunks)
{
    constexpr uint32_t P = kPer16<T>;
    typedef typename T::Raw Raw;
    const uint32_t row32 = blockIdx.x / chunks;
    const uint64_t row = row32;
    const uint32_t begin = (blockIdx.x - row32 * chunks) * (kThreads * kUnroll * P);
    const Raw* x = static_cast<const Raw*>(a.logits) + row * a.rowStride;
    Raw* d = static_cast<Raw*>(a.grad) + row * a.gradRowStride;

    // the logits are on their way before the row's numbers are
    U32x4 raw[kUnroll];
    for (uint32_t u = 0; u < kUnroll; ++u) {
        const uint32_t at = begin + (u * kThreads + threadIdx.x) * P;
        if (at + P <= a.count) {
            raw[u] = LoadOnce16(x + at);
        } else {
            float f[P];
            for (uint32_t i = 0; i < P; ++i) {
                f[i] = at + i < a.count ? Widen<T>(LoadOne(x + at + i)) : 0.0f;
            }
            raw[u] = Pack16<T>(f);
        }
    }
    const float lse = LoadOne(a.logSumExp + row);
    const float e = a.gradEntropy != nullptr ? LoadOne(a.gradEntropy + row) : 0.0f;
    const float h = a.gradEntropy != nullptr ? LoadOne(a.entropy + row) : 0.0f;
    // Lane j has the j-th one-hot term: entry `id` (negative: none) and its gradient t; the given token comes behind the
    // alternatives.  Every wavefront fetches them for itself.
    const uint32_t lane = threadIdx.x & (kWave - 1);
    const uint32_t nTop = kTop ? a.topCount : 0;
    int64_t id = -1;
    float t = 0.0f;
    if (kTop && lane < nTop) {
        id = IdAt(a.topIds, a.wideTokens, row * nTop + lane);
        t = LoadOne(a.gradTop + row * nTop + lane);
    } else if (lane == nTop && a.gradLogProbs != nullptr) {
        id = IdAt(a.tokens, a.wideTokens, row);
        t = LoadOne(a.gradLogProbs + row);
    }
    t = id >= 0 ? t : 0.0f;
    const float sum = kTop ? WaveSum(t) : __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(uint32_t, t)));
    bool zero = __ballot(t != 0.0f) == 0 && e == 0.0f;
    zero = zero || lse < kMaskedRow;
    const float es = e * a.scale, as = sum * a.scale;

    float y[kUnroll][P];
    for (uint32_t u = 0; u < kUnroll; ++u) {
        Unpack16<T>(raw[u], y[u]);
        for (uint32_t i = 0; i < P; ++i) {
            const float logP = __builtin_fmaf(y[u][i], a.scale, -lse);
            const float p = Exp2(logP * kLog2E);
            y[u][i] = zero ? 0.0f : -p * __builtin_fmaf(es, fmaxf(logP, kNoProb) + h, as);
        }
    }
    // Terms that fall into this chunk, one after the other.
    const int64_t local = id - a.vocabStart - begin;      // place in the chunk
    uint64_t hits = __ballot(id >= 0 && local >= 0 && local < static_cast<int64_t>(kThreads * kUnroll * P) && !zero);
    while (hits != 0) {
        const uint32_t j = __ffsll(static_cast<unsigned long long>(hits)) - 1;
        hits &= hits - 1;
        const uint32_t place = __builtin_amdgcn_readlane(static_cast<uint32_t>(local), j);
        const float term = a.scale * __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(uint32_t, t), j));
        const uint32_t vec = place / P;
        if (vec % kThreads == threadIdx.x) {
            const uint32_t element = vec / kThreads * P + place % P;
            for (uint32_t u = 0; u < kUnroll; ++u) {
                for (uint32_t i = 0; i < P; ++i) {
                    y[u][i] += u * P + i == element ? term : 0.0f;
                }
            }
        }
    }
    for (uint32_t u = 0; u < kUnroll; ++u) {
        const uint32_t at = begin + (u * kThreads + threadIdx.x) * P;
        if (at + P <= a.count) {
            StoreOnce16(d + at, Pack16<T>(y[u]));
        } else {
            for (uint32_t i = 0; i < P; ++i) {
                if (at + i < a.count) {
                    StoreOne(d + at + i, Narrow<T>(y[u][i]));
                }
            }
        }
    }
}

template <typename T>
hipError_t Launch(const LogProbsGradArgs& a, uint32_t rows, hipStream_t stream)
{
    constexpr uint32_t chunk = kThreads * kUnroll * kPer16<T>;
    const uint32_t chunks = static_cast<uint32_t>((static_cast<uint64_t>(a.count) + chunk - 1) / chunk);
    // A launch has fewer than 2^32 work items: very many rows take several.
    const uint32_t perLaunch = (1u << 23) / chunks == 0 ? 1 : (1u << 23) / chunks;
    for (uint32_t first = 0; first < rows; first += perLaunch) {
        const uint32_t n = rows - first < perLaunch ? rows - first : perLaunch;
        LogProbsGradArgs b = a;
        const uint64_t at = first;
        b.logits = static_cast<const typename T::Raw*>(a.logits) + at * a.rowStride;
        b.grad = static_cast<typename T::Raw*>(a.grad) + at * a.gradRowStride;
        const uint64_t idBytes = a.wideTokens ? 8 : 4;
        const auto skip = [at](const float* p, uint64_t per) { return p != nullptr ? p + at * per : nullptr; };
        const auto skipIds = [at, idBytes](const void* p, uint64_t per) {
            return p != nullptr ? static_cast<const uint8_t*>(p) + at * per * idBytes : nullptr;
        };
        b.tokens = skipIds(a.tokens, 1);
        b.topIds = skipIds(a.topIds, a.topCount);
        b.logSumExp = skip(a.logSumExp, 1);
        b.entropy = skip(a.entropy, 1);
        b.gradLogProbs = skip(a.gradLogProbs, 1);
        b.gradEntropy = skip(a.gradEntropy, 1);
        b.gradTop = skip(a.gradTop, a.topCount);
        if (b.gradTop != nullptr) {
            hipLaunchKernelGGL((LogProbsGradKernel<T, true>), dim3(n * chunks), dim3(kThreads), 0, stream, b, chunks);
        } else {
            hipLaunchKernelGGL((LogProbsGradKernel<T, false>), dim3(n * chunks), dim3(kThreads), 0, stream, b, chunks);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) {
            return e;
        }
    }
    return hipSuccess;
}

}  // namespace

hipError_t LaunchLogProbsGrad(const LogProbsGradArgs& a, HcclDataType dtype, uint32_t rows, hipStream_t stream)
{
    switch (dtype) {
        case HCCL_DATA_TYPE_FP32: return Launch<F32>(a, rows, stream);
        case HCCL_DATA_TYPE_BFP16: return Launch<B16>(a, rows, stream);
        default: return Launch<F16>(a, rows, stream);
    }
}

}  // namespace model_ops
}  // namespace hccl_amd
