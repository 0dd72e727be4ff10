// Launch descriptors of the model operators (include/hccl_model_ops.h), shared by their host layer and their kernels.
// Plain data that travels in the kernel-argument segment, below 4 KiB each.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hccl_model_ops.h"

namespace hccl_amd {
namespace model_ops {

constexpr uint32_t kMaxShards = HCCL_AMD_MAX_RANKS;
constexpr uint32_t kMaxTop = HCCL_AMD_MAX_TOP;

// ---- log probabilities ----------------------------------------------------------------------------------------
// Of a set of elements x: the largest, and with y = c (x - m), c = scale * log2(e), the sums of y 2^y and of 2^y.
struct alignas(16) LogProbsStats {
    float m, t;
    double s;
};

// One row of logits is the concatenation of nShards parts.
struct LogProbsArgs {
    const void* logits[kMaxShards];
    uint64_t rowStride[kMaxShards];     // elements
    uint32_t count[kMaxShards];         // elements of the part
    const void* tokens;
    LogProbsStats* stats;   // nSplit > 1: [row][split]
    uint64_t* keys;         //             [row][split][topCount], descending, 0 where there is none
    uint32_t nShards;
    uint32_t nSplit;        // workgroups per row
    uint32_t vocab;
    uint32_t vectors;       // 16-byte vectors of the row, a short one at the end of a part counted
    uint32_t topCount;
    uint32_t slotShift;     // filled by the launcher, see there
    uint32_t wideTokens;    // tokens and topIds are 64-bit
    float scale;
    float exp2Scale;        // scale * log2(e)
    uint32_t nOut;
    struct Out {
        float* logProbs;
        float* logSumExp;
        float* entropy;
        float* topValues;
        void* topIds;
    } out[kMaxShards];
};
static_assert(sizeof(LogProbsArgs) <= 4096, "kernel arguments");

// 16-byte vectors of a part's row.
inline uint64_t LogProbsVectors(uint64_t count, uint32_t elementSize) { return (count * elementSize + 15) / 16; }
// How a call is launched, from its rows and the vectors of a row alone: threads per workgroup and workgroups per row.  More
// vectors never mean fewer workgroups per row (LogProbsWorkspace relies on it).
struct LogProbsForm {
    uint32_t threads;
    uint32_t split;
};
LogProbsForm LogProbsFormOf(uint64_t rows, uint64_t vectors);
// Enough for every type and any parts: 32-bit elements, and a short vector at the end of each part.
inline uint64_t LogProbsWorkspace(uint64_t rows, uint64_t vocab, uint32_t top)
{
    const uint64_t split = rows == 0 ? 1 : LogProbsFormOf(rows, LogProbsVectors(vocab, 4) + kMaxShards).split;
    return split <= 1 ? 0 : rows * split * (4 * sizeof(float) + top * sizeof(uint64_t));
}
// args.vectors and args.nSplit are the form's.
hipError_t LaunchLogProbs(LogProbsArgs& args, HcclDataType dtype, uint32_t rows, hipStream_t stream);

// ---- their gradient ---------------------------------------------------------------------------------------------
struct LogProbsGradArgs {
    const void* logits;
    void* grad;
    uint64_t rowStride;      // elements
    uint64_t gradRowStride;
    uint32_t vocabStart;
    uint32_t count;
    uint32_t topCount;
    uint32_t wideTokens;
    float scale;
    const void* tokens;
    const float* logSumExp;
    const float* entropy;
    const float* gradLogProbs;
    const float* gradEntropy;
    const void* topIds;
    const float* gradTop;
};
hipError_t LaunchLogProbsGrad(const LogProbsGradArgs& args, HcclDataType dtype, uint32_t rows, hipStream_t stream);

// ---- gradient norm ------------------------------------------------------------------------------------------------
// A batch of tensors cut into chunks of kNormChunkBytes; workgroup b sums the chunks [b * perGroup, (b + 1) * perGroup).
constexpr uint32_t kNormBatch = 320;            // tensors per launch, a multiple of 16
constexpr uint32_t kNormAddressBits = 48;       // of a device address
constexpr uint32_t kNormGroups = 4096;          // partial sums per launch, at most
constexpr uint32_t kNormChunkBytes = 16384;
struct NormArgs {
    uint64_t tensor[kNormBatch];        // address, with (bytes of the last chunk - 1) << 2 | type (0 fp32, 1 bf16, 2 fp16) above
    uint32_t chunkEnd[kNormBatch];      // inclusive prefix of the chunk counts, the rest 0xFFFFFFFF
    uint32_t groupEnd[32];              // chunkEnd of every sixteenth tensor, the rest 0xFFFFFFFF
    double* partial;                    // one per workgroup
    uint32_t nChunks;
    uint32_t perGroup;
};
static_assert(sizeof(NormArgs) <= 4096 && kNormBatch % 16 == 0 && kNormBatch / 16 < 32, "kernel arguments");
static_assert(kNormChunkBytes <= 1u << 14, "a last chunk's bytes and type are 16 bits");
struct NormJoinArgs {
    const double* partial;
    uint32_t nPartial;
    float maxNorm;
    float scale;
    uint32_t nOut;
    float* out[kMaxShards];
};
hipError_t LaunchNormBatch(const NormArgs& args, uint32_t groups, hipStream_t stream);
hipError_t LaunchNormJoin(const NormJoinArgs& args, hipStream_t stream);

// ---- AdamW ----------------------------------------------------------------------------------------------------------
constexpr uint32_t kAdamWChunk = 2048;          // elements per workgroup, a multiple of the state block
constexpr uint32_t kAdamWWords = 496;           // words of a launch's table
// Words of one tensor: its last chunk's inclusive prefix with that chunk's elements in the upper half, param, grad, m, v, then
// master and the two scales where there are any.
constexpr uint32_t AdamWTensorWords(bool master, bool fp8State) { return 5u + (master ? 1u : 0u) + (fp8State ? 2u : 0u); }
struct AdamWArgs {
    uint64_t table[kAdamWWords];
    uint32_t nTensors;
    uint32_t skipNonFinite;
    const float* clip;
    const int64_t* step;                // null: the host's factors below
    const float* lr;
    float beta1, oneMinusBeta1, beta2, oneMinusBeta2;
    float eps;
    float weightDecay;
    float hostLr;
    float logBeta1, logBeta2;           // natural logarithms, for a step read on the device
    float correction1, rootCorrection2; // 1 / (1 - beta1^step), 1 / sqrt(1 - beta2^step)
};
static_assert(sizeof(AdamWArgs) <= 4096, "kernel arguments");
hipError_t LaunchAdamW(const AdamWArgs& args, HcclDataType paramType, HcclDataType gradType, bool master, bool fp8State,
                       uint32_t chunks, hipStream_t stream);

}  // namespace model_ops
}  // namespace hccl_amd
