// Sum of squares over many tensors, its root and the clip factor.
//
// The tensors of a batch are cut into chunks of 16 KiB and every workgroup sums a run of neighbouring chunks: one 64-bit
// multiply-add per element, which runs at the rate of a 32-bit one here, so that neither the range of the element type nor
// the number of elements costs accuracy.  A workgroup leaves one partial sum and a last workgroup adds them: which elements
// meet in which order depends on the sizes alone.  Bound: one read of the gradients.
#include "model_ops.h"
#include "vec.h"

namespace hccl_amd {
namespace model_ops {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kJoinThreads = 1024;

template <typename T>
__device__ __forceinline__ double ChunkSquares(const void* data, uint32_t elements)
{
    constexpr uint32_t P = kPer16<T>;
    constexpr uint32_t kVecs = kNormChunkBytes / 16 / kThreads;
    typedef typename T::Raw Raw;
    const Raw* x = static_cast<const Raw*>(data);
    double sum = 0.0;
    if (elements == kVecs * kThreads * P) {
        U32x4 raw[kVecs];
        for (uint32_t u = 0; u < kVecs; ++u) {
            raw[u] = LoadOnce16(x + (u * kThreads + threadIdx.x) * P);
        }
        for (uint32_t u = 0; u < kVecs; ++u) {
            float f[P];
            Unpack16<T>(raw[u], f);
            for (uint32_t i = 0; i < P; ++i) {
                const double v = f[i];
                sum = __builtin_fma(v, v, sum);
            }
        }
    } else {
        for (uint32_t at = threadIdx.x * P; at < elements; at += kThreads * P) {
            float f[P];
            if (at + P <= elements) {
                Unpack16<T>(LoadOnce16(x + at), f);
            } else {
                for (uint32_t i = 0; i < P; ++i) {
                    f[i] = at + i < elements ? Widen<T>(LoadOne(x + at + i)) : 0.0f;
                }
            }
            for (uint32_t i = 0; i < P; ++i) {
                const double v = f[i];
                sum = __builtin_fma(v, v, sum);
            }
        }
    }
    return sum;
}

// Sum over a workgroup, valid in thread 0.
template <uint32_t kWavesInGroup>
__device__ __forceinline__ double GroupSum(double v)
{
    __shared__ double wave[kWavesInGroup];
    v = WaveSum(v);
    if ((threadIdx.x & (kWave - 1)) == 0) {
        wave[threadIdx.x / kWave] = v;
    }
    __syncthreads();
    double sum = wave[0];
    for (uint32_t w = 1; w < kWavesInGroup; ++w) {
        sum += wave[w];
    }
    return sum;
}

__global__ __launch_bounds__(kThreads) void NormBatchKernel(const NormArgs a)
{
    const uint32_t first = blockIdx.x * a.perGroup;
    const uint32_t last = first + a.perGroup < a.nChunks ? first + a.perGroup : a.nChunks;
    uint32_t lo = 0, hi = a.nTensors - 1;      // the tensor of the first chunk: the first one that ends behind it
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (a.chunkEnd[mid] > first) {
            hi = mid;
        } else {
            lo = mid + 1;
        }
    }
    uint32_t tensor = lo;
    double sum = 0.0;
    for (uint32_t chunk = first; chunk < last; ++chunk) {
        while (a.chunkEnd[tensor] <= chunk) {
            ++tensor;
        }
        const uint32_t start = tensor == 0 ? 0 : a.chunkEnd[tensor - 1];
        const uint32_t type = a.lastChunk[tensor] & 3u;
        const uint32_t whole = kNormChunkBytes / (type == 0 ? 4 : 2);
        const uint32_t elements = chunk + 1 == a.chunkEnd[tensor] ? a.lastChunk[tensor] >> 2 : whole;
        const void* data = static_cast<const uint8_t*>(a.data[tensor]) + static_cast<uint64_t>(chunk - start) * kNormChunkBytes;
        if (type == 0) {
            sum += ChunkSquares<F32>(data, elements);
        } else if (type == 1) {
            sum += ChunkSquares<B16>(data, elements);
        } else {
            sum += ChunkSquares<F16>(data, elements);
        }
    }
    sum = GroupSum<kThreads / kWave>(sum);
    if (threadIdx.x == 0) {
        StoreOne(a.partial + blockIdx.x, sum);
    }
}

__global__ __launch_bounds__(kJoinThreads) void NormJoinKernel(const NormJoinArgs a)
{
    double sum = 0.0;
    for (uint32_t i = threadIdx.x; i < a.nPartial; i += kJoinThreads) {
        sum += LoadOne(a.partial + i);
    }
    sum = GroupSum<kJoinThreads / kWave>(sum);
    if (threadIdx.x < a.nOut) {
        const double norm = sqrt(sum) * fabs(static_cast<double>(a.scale));
        double factor = a.scale;
        if (a.maxNorm > 0.0f) {
            const double clip = a.maxNorm / (norm + 1e-6);
            factor = clip < 1.0 || clip != clip ? factor * clip : factor;
        }
        StoreOne(a.out[threadIdx.x], static_cast<float>(norm));
        StoreOne(a.out[threadIdx.x] + 1, static_cast<float>(factor));
    }
}

}  // namespace

hipError_t LaunchNormBatch(const NormArgs& a, uint32_t groups, hipStream_t stream)
{
    hipLaunchKernelGGL(NormBatchKernel, dim3(groups), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

hipError_t LaunchNormJoin(const NormJoinArgs& a, hipStream_t stream)
{
    hipLaunchKernelGGL(NormJoinKernel, dim3(1), dim3(kJoinThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace model_ops
}  // namespace hccl_amd
