// Gradient of log probabilities, entropy and alternatives with respect to one rank's part of the logits:
//   d_v = scale ( one-hot terms - p_v (a + e (log p_v + H)) ),  log p_v = scale x_v - lse,  a = g + sum_j h_j.
//
// Every element needs its logit and half a dozen numbers of its row, so the part is cut into chunks that know nothing of
// each other.  Bound: one read and one write per element.  The one-hot terms are added in 32 bits before the only rounding:
// a workgroup walks the row's few ids with uniform control flow and skips those outside its chunk.
#include "model_ops.h"
#include "vec.h"

namespace hccl_amd {
namespace model_ops {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kUnroll = 4;
constexpr float kLog2E = 1.44269504088896341f;
constexpr float kMaskedRow = -1e30f;      // logSumExp of a row in which no entry can occur
constexpr float kNoProb = -1000.0f;      // log p below this has p = 0 in 32 bits; keeps -inf out of products with p

__device__ __forceinline__ int64_t IdAt(const void* ids, uint32_t wide, uint64_t at)
{
    return wide ? LoadOne(static_cast<const int64_t*>(ids) + at) : LoadOne(static_cast<const int32_t*>(ids) + at);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void LogProbsGradKernel(const LogProbsGradArgs a, uint32_t chunks)
{
    constexpr uint32_t P = kPer16<T>;
    constexpr uint32_t N = kUnroll * P;
    typedef typename T::Raw Raw;
    const uint32_t block = blockIdx.x;
    const uint64_t row = block / chunks;
    const uint32_t begin = (block - static_cast<uint32_t>(row) * chunks) * (kThreads * N);
    const Raw* x = static_cast<const Raw*>(a.logits) + row * a.rowStride;
    Raw* d = static_cast<Raw*>(a.grad) + row * a.gradRowStride;

    const float lse = LoadOne(a.logSumExp + row);
    const float e = a.gradEntropy != nullptr ? LoadOne(a.gradEntropy + row) : 0.0f;
    const float h = e != 0.0f ? LoadOne(a.entropy + row) : 0.0f;
    float g = 0.0f;
    int64_t token = -1;
    if (a.gradLogProbs != nullptr) {
        token = IdAt(a.tokens, a.wideTokens, row);
        g = token >= 0 ? LoadOne(a.gradLogProbs + row) : 0.0f;
    }
    float sum = g;
    bool zero = g == 0.0f && e == 0.0f;
    if (a.gradTop != nullptr) {
        for (uint32_t j = 0; j < a.topCount; ++j) {
            if (IdAt(a.topIds, a.wideTokens, row * a.topCount + j) >= 0) {
                const float t = LoadOne(a.gradTop + row * a.topCount + j);
                sum += t;
                zero = zero && t == 0.0f;
            }
        }
    }
    zero = zero || lse < kMaskedRow;
    const float es = e * a.scale, as = sum * a.scale;

    float y[kUnroll][P];
    for (uint32_t u = 0; u < kUnroll; ++u) {
        const uint32_t at = begin + (u * kThreads + threadIdx.x) * P;
        if (zero) {
            for (uint32_t i = 0; i < P; ++i) {
                y[u][i] = 0.0f;
            }
        } else if (at + P <= a.count) {
            Unpack16<T>(LoadOnce16(x + at), y[u]);
        } else {
            for (uint32_t i = 0; i < P; ++i) {
                y[u][i] = at + i < a.count ? Widen<T>(LoadOne(x + at + i)) : 0.0f;
            }
        }
    }
    if (!zero) {
        for (uint32_t u = 0; u < kUnroll; ++u) {
            for (uint32_t i = 0; i < P; ++i) {
                const float logP = __builtin_fmaf(y[u][i], a.scale, -lse);
                const float p = Exp2(logP * kLog2E);
                y[u][i] = -p * __builtin_fmaf(es, fmaxf(logP, kNoProb) + h, as);
            }
        }
        const uint32_t nTop = a.gradTop != nullptr ? a.topCount : 0;
        for (uint32_t j = 0; j <= nTop; ++j) {
            // j == nTop: the given token
            const int64_t id = (j < nTop ? IdAt(a.topIds, a.wideTokens, row * a.topCount + j) : token);
            const int64_t local = id - a.vocabStart - begin;
            if (id < 0 || local < 0 || local >= static_cast<int64_t>(kThreads * N)) {
                continue;
            }
            const float t = (j < nTop ? LoadOne(a.gradTop + row * a.topCount + j) : g) * a.scale;
            const uint32_t vec = static_cast<uint32_t>(local) / P, lane = vec % kThreads;
            if (lane == threadIdx.x) {
                const uint32_t element = vec / kThreads * P + static_cast<uint32_t>(local) % P;
                for (uint32_t u = 0; u < kUnroll; ++u) {
                    for (uint32_t i = 0; i < P; ++i) {
                        y[u][i] += u * P + i == element ? t : 0.0f;
                    }
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
        hipLaunchKernelGGL((LogProbsGradKernel<T>), dim3(n * chunks), dim3(kThreads), 0, stream, b, chunks);
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
