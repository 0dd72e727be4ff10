// Sum of squares over many tensors, its root and the clip factor.
//
// The tensors of a batch are cut into chunks of 16 KiB and every workgroup sums a run of neighbouring chunks: one 64-bit
// multiply-add per element, which runs at the rate of a 32-bit one here, so that neither the range of the element type nor
// the number of elements costs accuracy.  A workgroup leaves one partial sum and a last workgroup adds them: which elements
// meet in which order depends on the sizes alone.
//
// Bound: one read of the gradients.  1 GiB of bf16 in 960 tensors of eight ranks, three launches and the last one: 173 us, 6.2
// TB/s of the 7.0 that a plain read reaches; about 4 us of each launch is its start and end.  For that reason a tensor's
// address and size share a word: 320 fit the arguments of a launch.  (240 with words of their own: 176 us, and 21 instead of
// 18 for 856 tensors of 40 elements.  Chunks dealt round the workgroups instead of in runs: 182 at best with four launches,
// since every step then passes a dozen tensors.)
#include "model_ops.h"
#include "vec.h"

namespace hccl_amd {
namespace model_ops {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kJoinThreads = 1024;

constexpr uint32_t kVecs = kNormChunkBytes / 16 / kThreads;

// A lane's vectors of a chunk of `bytes` bytes; what lies behind its end is 0.
__device__ __forceinline__ void LoadChunk(const uint8_t* data, uint32_t bytes, uint32_t elementSize, U32x4* raw)
{
    if (bytes == kNormChunkBytes) {
        for (uint32_t u = 0; u < kVecs; ++u) {
            raw[u] = LoadOnce16(data + (u * kThreads + threadIdx.x) * 16);
        }
        return;
    }
    for (uint32_t u = 0; u < kVecs; ++u) {
        const uint32_t at = (u * kThreads + threadIdx.x) * 16;
        raw[u] = U32x4{0, 0, 0, 0};
        if (at + 16 <= bytes) {
            raw[u] = LoadOnce16(data + at);
        } else if (elementSize == 4) {
            for (uint32_t i = 0; i < 4; ++i) {
                raw[u][i] = at + 4 * i < bytes ? LoadOne(reinterpret_cast<const uint32_t*>(data + at + 4 * i)) : 0u;
            }
        } else {
            for (uint32_t i = 0; i < 8; ++i) {
                const uint32_t e = at + 2 * i < bytes ? LoadOne(reinterpret_cast<const uint16_t*>(data + at + 2 * i)) : 0u;
                raw[u][i / 2] |= e << (16 * (i % 2));
            }
        }
    }
}

template <typename T>
__device__ __forceinline__ double Squares(const U32x4* raw, double sum)
{
    for (uint32_t u = 0; u < kVecs; ++u) {
        float f[kPer16<T>];
        Unpack16<T>(raw[u], f);
        for (uint32_t i = 0; i < kPer16<T>; ++i) {
            const double v = f[i];
            sum = __builtin_fma(v, v, sum);
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

// Entries of a sixteen that are at most `chunk`, counted in scalar arithmetic; the sixteen come with one load.
__device__ __forceinline__ uint32_t EndedOf16(const uint32_t* end, uint32_t chunk)
{
    uint32_t n = 0;
    for (uint32_t i = 0; i < 16; ++i) {
        n += end[i] <= chunk ? 1u : 0u;
    }
    return n;
}

__device__ __forceinline__ const uint8_t* Address(uint64_t tensor)
{
    return reinterpret_cast<const uint8_t*>(tensor & ((1ull << kNormAddressBits) - 1));
}

__global__ __launch_bounds__(kThreads) void NormBatchKernel(const NormArgs a)
{
    const uint32_t first = blockIdx.x * a.perGroup;
    const uint32_t last = first + a.perGroup < a.nChunks ? first + a.perGroup : a.nChunks;
    // The tensor of the first chunk, the first one that ends behind it: sixteen by sixteen, not one by one.
    const uint32_t group = EndedOf16(a.groupEnd, first) + EndedOf16(a.groupEnd + 16, first);
    uint32_t tensor = 16 * group + EndedOf16(a.chunkEnd + 16 * group, first);
    uint32_t end = a.chunkEnd[tensor], start = tensor == 0 ? 0u : a.chunkEnd[tensor - 1];
    const uint8_t* data = Address(a.tensor[tensor]);
    uint32_t code = static_cast<uint32_t>(a.tensor[tensor] >> kNormAddressBits);
    double sum = 0.0;
    U32x4 raw[kVecs];
    for (uint32_t chunk = first; chunk < last; ++chunk) {
        if (chunk == end) {
            ++tensor;
            start = end;
            end = a.chunkEnd[tensor];
            data = Address(a.tensor[tensor]);
            code = static_cast<uint32_t>(a.tensor[tensor] >> kNormAddressBits);
        }
        const uint32_t type = code & 3u;
        LoadChunk(data + static_cast<uint64_t>(chunk - start) * kNormChunkBytes, chunk + 1 == end ? (code >> 2) + 1 : kNormChunkBytes,
                  type == 0 ? 4 : 2, raw);
        sum = type == 0 ? Squares<F32>(raw, sum) : type == 1 ? Squares<B16>(raw, sum) : Squares<F16>(raw, sum);
    }
    sum = GroupSum<kThreads / kWave>(sum);
    if (threadIdx.x == 0) {
        StoreOne(a.partial + blockIdx.x, sum);
    }
}

__global__ __launch_bounds__(kJoinThreads) void NormJoinKernel(const NormJoinArgs a)
{
    double sum = 0.0;
    for (uint32_t i = threadIdx.x; i < a.nPartial; i += 4 * kJoinThreads) {
        double part[4];      // loaded together
        for (uint32_t u = 0; u < 4; ++u) {
            part[u] = i + u * kJoinThreads < a.nPartial ? LoadOne(a.partial + i + u * kJoinThreads) : 0.0;
        }
        sum += (part[0] + part[1]) + (part[2] + part[3]);
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
