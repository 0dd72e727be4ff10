/*
 * Model operators over loopback worlds: what a training or serving step runs right next to its collectives.
 *
 *   HcclAmdTokenLogProbs      log probabilities of given tokens, entropy and top alternatives of every row of logits
 *                             whose vocabulary is split across the ranks (a collective: every rank calls, every rank
 *                             receives the results)
 *   HcclAmdTokenLogProbsGrad  its gradient with respect to the calling rank's part of the logits (local to the rank)
 *   HcclAmdGradNorm           2-norm over all gradient tensors of all ranks and the factor that clips it (a collective)
 *   HcclAmdAdamW              one AdamW step over many tensors, states in 32 bits or in FP8 blocks (local to the rank)
 *
 * Implemented by libhccl_amd_model_ops.so, which works on the communicators of libhccl_amd.so (hccl.h).  Conventions
 * are those of hccl.h: buffers are device pointers on the world's GPU, work is asynchronous on `stream`, a null stream
 * is refused, results are HcclResult codes, a collective takes one call per rank (HcclGroupStart / HcclGroupEnd for a
 * thread that drives several), and a call that fails its argument checks still takes its place in the sequence of
 * collectives.  The local operators launch at once, also between HcclGroupStart and HcclGroupEnd: a collective of the
 * same group has not been launched then, so what depends on it is called after HcclGroupEnd.  Argument structures and
 * arrays of descriptors are read during the call only.  Nothing here allocates device memory or copies from the host;
 * every call can be captured into a graph (ranks on one stream) and replayed.
 */
#ifndef HCCL_AMD_HCCL_MODEL_OPS_H_
#define HCCL_AMD_HCCL_MODEL_OPS_H_

#include "hccl.h"

#ifdef __cplusplus
extern "C" {
#endif

#define HCCL_AMD_MAX_TOP 32              /* alternatives per row */
#define HCCL_AMD_STATE_BLOCK 256         /* elements that share the scale of an FP8 state */

/*
 * Row i of the logits has V = sum over the ranks of vocabCount entries, rank 0's first.  With x = scale * logits[i],
 * lse = log(sum(exp(x))):
 *   logProbs[i]      x[tokens[i]] - lse; 0 for a negative token (ignored); NaN for a token >= V
 *   logSumExp[i]     lse
 *   entropy[i]       -sum(p log p), p = exp(x - lse)
 *   topIds[i][j]     the j-th most likely entry, the lower index of equal ones; topValues[i][j] = x[topIds[i][j]] - lse
 * Sums are kept in 32 bits or more, relative to the row's maximum: a log p near 0 is right to 3 * 2^-24, not to 24 bits of
 * its own.  -inf logits are entries that cannot occur.  A row of -inf alone has logSumExp -inf, logProbs -inf (0 if
 * ignored), entropy 0, topIds 0, 1, ... and topValues -inf.  A row with a NaN or +inf has NaN in every output but topIds,
 * which are -1, and the 0 of an ignored token.
 * No output, and no workspace, may overlap anything else that the call reads or writes.
 */
typedef struct {
    const void* logits;       /* tokenCount rows of vocabCount elements, rowStride elements apart, element-aligned */
    uint64_t rowStride;       /* >= vocabCount, at most 2^36 */
    uint64_t vocabStart;      /* index of this rank's first entry: the sum of vocabCount over the lower ranks */
    uint64_t vocabCount;      /* may differ between ranks, may be 0; V is 1 .. 2^31 - 1 */
    uint64_t tokenCount;      /* rows, the same on every rank, below 2^24; 0: nothing to do on any rank */
    const void* tokens;       /* tokenCount ids of tokenType, the same on every rank (the lowest rank's are read) */
    HcclDataType dataType;    /* of the logits: FP16, BFP16 or FP32 */
    HcclDataType tokenType;   /* of tokens and topIds: INT32 or INT64 */
    float scale;              /* 1 / temperature, 1e-6 .. 1e6 */
    uint32_t topCount;        /* 0 .. HCCL_AMD_MAX_TOP, at most V */
    float* logProbs;          /* [tokenCount], or null: every output is optional on every rank */
    float* logSumExp;         /* [tokenCount] */
    float* entropy;           /* [tokenCount] */
    float* topValues;         /* [tokenCount][topCount] */
    void* topIds;             /* [tokenCount][topCount] of tokenType */
    void* workspace;          /* 16-byte aligned device memory for calls with few rows, see below */
    uint64_t workspaceBytes;
} HcclAmdTokenLogProbsArgs;

HcclResult HcclAmdTokenLogProbs(const HcclAmdTokenLogProbsArgs* args, HcclComm comm, aclrtStream stream);

/* Bytes of workspace that a call needs on at least one rank (0 where the rows alone fill the GPU); less of it on every
 * rank: HCCL_E_MEMORY.  Its contents need no initialisation and mean nothing afterwards.  Calls that may run at the same
 * time, replays of captured ones included, need different workspaces. */
HcclResult HcclAmdTokenLogProbsWorkspace(uint64_t tokenCount, uint64_t vocabSize, uint32_t topCount, uint64_t* bytes);

/*
 * Gradient of  sum_i gradLogProbs[i] logProbs[i] + gradEntropy[i] entropy[i] + sum_j gradTopValues[i][j] topValues[i][j]
 * with respect to this rank's part of the logits, given the forward pass's logSumExp, entropy and topIds:
 *   gradLogits[i][v] = scale * ([v = tokens[i]] g_i + sum_j [v = topIds[i][j]] h_ij - p_v (a_i + e_i (log p_v + entropy_i)))
 *   a_i = g_i + sum_j h_ij, g_i = 0 for a negative token; a token or topId >= V is not checked for and counts in a_i only
 * rounded once to dataType.  gradLogits may be the logits themselves (same address and stride); other overlaps, with the
 * logits or with an array that is read for the rows, are refused.  A row whose incoming gradients are all 0 gets zeros
 * whatever its logits are; so does a row with logSumExp < -1e30, which -inf or the lowest finite value fills.  A negative
 * topId is skipped with its gradient.
 * log p is formed from the 32-bit logSumExp: it is up to |logSumExp| * 2^-24 off, and p by that share of itself, which next
 * to a p near 1 is also what 1 - p is off by.
 */
typedef struct {
    const void* logits;
    uint64_t rowStride;
    uint64_t vocabStart;
    uint64_t vocabCount;              /* 0: nothing to do */
    uint64_t tokenCount;              /* below 2^24; 0: nothing to do */
    const void* tokens;               /* needed with gradLogProbs */
    HcclDataType dataType;
    HcclDataType tokenType;
    float scale;
    uint32_t topCount;
    const float* logSumExp;
    const float* entropy;             /* needed with gradEntropy */
    const float* gradLogProbs;        /* [tokenCount]; each of the three gradients may be null, not all */
    const float* gradEntropy;         /* [tokenCount] */
    const void* topIds;               /* needed with gradTopValues */
    const float* gradTopValues;       /* [tokenCount][topCount] */
    void* gradLogits;
    uint64_t gradRowStride;
} HcclAmdTokenLogProbsGradArgs;

HcclResult HcclAmdTokenLogProbsGrad(const HcclAmdTokenLogProbsGradArgs* args, HcclComm comm, aclrtStream stream);

/*
 * result[0] = |scale| * sqrt(sum of squares over all tensors of all ranks), result[1] = scale * min(1, maxNorm /
 * (result[0] + 1e-6)), or scale if maxNorm <= 0: what HcclAmdAdamW multiplies the gradients by.  `scale` undoes a loss
 * scale or averages over replicas.  Squares are summed in 64 bits in an order that depends on the sizes only.  A NaN or
 * an infinity in a gradient shows in result[0].  Ranks may pass different tensors, and none; maxNorm and scale are the
 * same on every rank.
 */
typedef struct {
    const void* data;         /* element-aligned */
    uint64_t count;           /* elements, may be 0, below 2^40 */
    HcclDataType dataType;    /* FP16, BFP16 or FP32 */
} HcclAmdNormTensor;

HcclResult HcclAmdGradNorm(const HcclAmdNormTensor* tensors, uint32_t tensorCount, float maxNorm, float scale,
                           float* result /* [2], 4-byte aligned device memory */, void* workspace, uint64_t workspaceBytes,
                           HcclComm comm, aclrtStream stream);

/* Bytes of workspace (16-byte aligned) that a call over `tensorCount` tensors, all ranks' together, needs on at least one
 * rank; the same rules as above. */
HcclResult HcclAmdGradNormWorkspace(uint64_t tensorCount, uint64_t* bytes);

/*
 * One step of Adam with decoupled weight decay, for every element of every tensor:
 *   g = clip * grad;  m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
 *   w = w (1 - lr weightDecay) - lr / (1 - beta1^step) * m / (sqrt(v) / sqrt(1 - beta2^step) + eps)
 * in 32 bits.  w is `master` if given, else `param`; `param` receives w rounded to its type.
 * stateType FP32: expAvg = m and expAvgSq = v are floats.  stateType FP8E4M3: both are e4m3 codes in blocks of
 * HCCL_AMD_STATE_BLOCK elements (the last one short), each with a float scale = largest magnitude * (1 / 448): m = code * scale,
 * and expAvgSq holds the root of v, v = (code * scale)^2, of which a value above 0 is never rounded to 0.  The step uses m
 * and v before they are rounded.
 * The tensors of one call must not overlap.  Zero-filled states and scales are the start.
 */
typedef struct {
    void* param;              /* element-aligned, like every pointer here */
    const void* grad;
    void* expAvg;
    void* expAvgSq;
    float* master;            /* null, or 32-bit weights beside a 16-bit param */
    float* expAvgScale;       /* stateType FP8E4M3 only: [ceil(count / HCCL_AMD_STATE_BLOCK)] */
    float* expAvgSqScale;
    uint64_t count;           /* may be 0, below 2^40 */
    HcclDataType paramType;   /* FP16, BFP16 or FP32 */
    HcclDataType gradType;    /* paramType or FP32; with an FP32 param any of the three */
} HcclAmdAdamWTensor;

typedef struct {
    double lr;
    double beta1, beta2;      /* [0, 1) */
    double eps;               /* >= 2^-126, or 0: elements whose v is 0 then have no defined step */
    double weightDecay;
    uint64_t step;            /* 1 for the first step */
    const int64_t* stepOnDevice;   /* null, or read instead of step when the kernels run (captured steps) */
    const float* lrOnDevice;       /* null, or read instead of lr */
    const float* clip;        /* null, or HcclAmdGradNorm's result: the gradients are multiplied by clip[1] */
    HcclDataType stateType;   /* FP32 or FP8E4M3 */
    int32_t skipNonFinite;    /* with clip: a step whose clip[0] is not finite leaves every tensor as it was */
} HcclAmdAdamWConfig;

HcclResult HcclAmdAdamW(const HcclAmdAdamWTensor* tensors, uint32_t tensorCount, const HcclAmdAdamWConfig* config,
                        HcclComm comm, aclrtStream stream);

#ifdef __cplusplus
}
#endif
#endif /* HCCL_AMD_HCCL_MODEL_OPS_H_ */
