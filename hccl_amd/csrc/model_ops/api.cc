// Entry points of include/hccl_model_ops.h: argument checks, the marshalling of the collective ones through the rendezvous
// of libhccl_amd.so, and what the last arrival launches.
#include <cmath>
#include <cstring>
#include <new>
#include <vector>

#include "../host.h"
#include "hccl_model_ops.h"
#include "model_ops.h"

using namespace hccl_amd;
using namespace hccl_amd::model_ops;

namespace {

bool IsLogitsType(HcclDataType t)
{
    return t == HCCL_DATA_TYPE_FP16 || t == HCCL_DATA_TYPE_BFP16 || t == HCCL_DATA_TYPE_FP32;
}

bool IsTokenType(HcclDataType t) { return t == HCCL_DATA_TYPE_INT32 || t == HCCL_DATA_TYPE_INT64; }

bool Aligned(const void* p, uint64_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

constexpr uint64_t kMaxVocab = 0x7FFFFFFFull;
constexpr uint64_t kMaxRows = (1ull << 24) - 1;
constexpr uint64_t kMaxRowStride = 1ull << 36;      // rows x stride x 4 bytes stays below 2^62

// A structure of a rank's call as the words RankArgs::var carries, and back.
template <typename S>
std::vector<uint64_t> Words(const S& s, size_t more = 0)
{
    std::vector<uint64_t> w((sizeof(S) + 7) / 8 + more);
    memcpy(w.data(), &s, sizeof(S));
    return w;
}
template <typename S>
S FromWords(const std::vector<uint64_t>& w)
{
    S s;
    memcpy(&s, w.data(), sizeof(S));
    return s;
}

// The checks shared by the log probabilities and their gradient.
HcclResult CheckLogits(const char* name, const void* logits, uint64_t rowStride, uint64_t vocabStart, uint64_t vocabCount,
                       uint64_t tokenCount, HcclDataType dataType, HcclDataType tokenType, float scale, uint32_t topCount)
{
    if (!IsLogitsType(dataType) || !IsTokenType(tokenType)) {
        Log(1, "%s: logits of type %d with tokens of type %d are not supported", name, static_cast<int>(dataType),
            static_cast<int>(tokenType));
        return HCCL_E_NOT_SUPPORT;
    }
    if (vocabCount != 0 && logits == nullptr) {
        Log(1, "%s: logits is nullptr", name);
        return HCCL_E_PTR;
    }
    if (tokenCount > kMaxRows || vocabStart > kMaxVocab || vocabCount > kMaxVocab - vocabStart) {
        Log(1, "%s: %llu rows of entries %llu + %llu are out of range", name, (unsigned long long)tokenCount,
            (unsigned long long)vocabStart, (unsigned long long)vocabCount);
        return HCCL_E_PARA;
    }
    if (rowStride < vocabCount || rowStride > kMaxRowStride) {
        Log(1, "%s: a row stride of %llu does not fit %llu entries", name, (unsigned long long)rowStride,
            (unsigned long long)vocabCount);
        return HCCL_E_PARA;
    }
    if (!(scale >= 1e-6f && scale <= 1e6f)) {
        Log(1, "%s: scale %g is not within 1e-6 .. 1e6", name, static_cast<double>(scale));
        return HCCL_E_PARA;
    }
    if (topCount > kMaxTop) {
        Log(1, "%s: %u alternatives, %u at most", name, topCount, kMaxTop);
        return HCCL_E_PARA;
    }
    if (!Aligned(logits, DataTypeSize(dataType))) {
        Log(1, "%s: logits is not element-aligned", name);
        return HCCL_E_PARA;
    }
    return HCCL_SUCCESS;
}

HcclResult CheckAligned(const char* name, const void* p, uint64_t to, const char* what)
{
    if (!Aligned(p, to)) {
        Log(1, "%s: %s is not aligned to %llu bytes", name, what, (unsigned long long)to);
        return HCCL_E_PARA;
    }
    return HCCL_SUCCESS;
}

// Runs the body of an entry point, or of a launch in the rendezvous: no exception leaves through the C boundary, nor past
// the state of a launch in progress.
template <class F>
HcclResult Guarded(const char* name, F body)
{
    try {
        return body();
    } catch (const std::bad_alloc&) {
        Log(1, "%s: out of host memory", name);
        return HCCL_E_MEMORY;
    } catch (...) {
        Log(1, "%s: internal error", name);
        return HCCL_E_INTERNAL;
    }
}

// ---- what the last arrival launches -----------------------------------------------------------------------------
HcclResult LaunchTokenLogProbs(World* w, PendingOp& p, hipStream_t s)
{
    LogProbsArgs a = {};
    const uint64_t rows = p.count;
    uint64_t vocab = 0, vectors = 0;
    std::vector<HcclAmdTokenLogProbsArgs> ranks(w->n);
    for (uint32_t r = 0; r < w->n; ++r) {
        ranks[r] = FromWords<HcclAmdTokenLogProbsArgs>(p.ranks[r].var);
        const HcclAmdTokenLogProbsArgs& x = ranks[r];
        if (x.scale != ranks[0].scale || x.tokenType != ranks[0].tokenType || x.vocabStart != vocab) {
            Log(1, "TokenLogProbs on rank %u: scale %g, token type %d, first entry %llu do not follow the lower ranks' %g, %d, %llu",
                r, static_cast<double>(x.scale), static_cast<int>(x.tokenType), (unsigned long long)x.vocabStart,
                static_cast<double>(ranks[0].scale), static_cast<int>(ranks[0].tokenType), (unsigned long long)vocab);
            return HCCL_E_PARA;
        }
        vocab += x.vocabCount;
        if (x.vocabCount != 0) {
            a.logits[a.nShards] = x.logits;
            a.rowStride[a.nShards] = x.rowStride;
            a.count[a.nShards] = static_cast<uint32_t>(x.vocabCount);
            vectors += LogProbsVectors(x.vocabCount, DataTypeSize(p.dtype));
            a.nShards++;
        }
        if (a.tokens == nullptr) {
            a.tokens = x.tokens;
        }
        if (x.logProbs != nullptr || x.logSumExp != nullptr || x.entropy != nullptr || x.topValues != nullptr ||
            x.topIds != nullptr) {
            a.out[a.nOut++] = {x.logProbs, x.logSumExp, x.entropy, x.topValues, x.topIds};
        }
    }
    const uint32_t top = p.root;
    if (vocab == 0 || vocab > kMaxVocab || top > vocab) {
        Log(1, "TokenLogProbs: %u alternatives of a vocabulary of %llu", top, (unsigned long long)vocab);
        return HCCL_E_PARA;
    }
    if (a.nOut == 0) {
        return HCCL_SUCCESS;
    }
    a.vocab = static_cast<uint32_t>(vocab);
    a.topCount = top;
    a.wideTokens = ranks[0].tokenType == HCCL_DATA_TYPE_INT64 ? 1 : 0;
    a.scale = ranks[0].scale;
    a.exp2Scale = static_cast<float>(static_cast<double>(a.scale) * 1.4426950408889634);
    a.vectors = static_cast<uint32_t>(vectors);
    a.nSplit = LogProbsFormOf(rows, vectors).split;
    if (a.nSplit > 1) {
        const uint64_t need = LogProbsWorkspace(rows, vocab, top);
        void* space = nullptr;
        for (uint32_t r = 0; r < w->n && space == nullptr; ++r) {
            space = ranks[r].workspaceBytes >= need ? ranks[r].workspace : nullptr;
        }
        if (space == nullptr) {
            Log(1, "TokenLogProbs: %llu rows of %llu entries need a workspace of %llu bytes", (unsigned long long)rows,
                (unsigned long long)vocab, (unsigned long long)need);
            return HCCL_E_MEMORY;
        }
        a.stats = static_cast<LogProbsStats*>(space);
        a.keys = reinterpret_cast<uint64_t*>(a.stats + rows * a.nSplit);
    }
    HIP_OK(LaunchLogProbs(a, p.dtype, static_cast<uint32_t>(rows), s));
    return HCCL_SUCCESS;
}

// A rank's call of the norm: these words, then data, count and type of every tensor.
struct NormCall {
    float maxNorm;
    float scale;
    float* result;
    void* workspace;
    uint64_t workspaceBytes;
    uint64_t tensorCount;
};
constexpr size_t kNormCallWords = sizeof(NormCall) / 8;
constexpr uint32_t kMaxChunks = 1u << 30;      // chunks of one launch

uint64_t NormWorkspace(uint64_t tensors)
{
    // Every launch but the last takes kNormBatch tensors, or fewer where they are beyond kMaxChunks chunks together: two
    // launches more than the tensor count asks for, per 2^44 bytes, which the GPU's memory does not hold twice.
    const uint64_t launches = tensors / kNormBatch + 2;
    return launches * kNormGroups * sizeof(double);
}

HcclResult LaunchGradNorm(World* w, PendingOp& p, hipStream_t s)
{
    NormJoinArgs join = {};
    uint64_t tensors = 0;
    std::vector<NormCall> calls(w->n);
    for (uint32_t r = 0; r < w->n; ++r) {
        calls[r] = FromWords<NormCall>(p.ranks[r].var);
        if (memcmp(&calls[r].maxNorm, &calls[0].maxNorm, 2 * sizeof(float)) != 0) {
            Log(1, "GradNorm on rank %u: maxNorm %g and scale %g are not rank 0's", r, static_cast<double>(calls[r].maxNorm),
                static_cast<double>(calls[r].scale));
            return HCCL_E_PARA;
        }
        tensors += calls[r].tensorCount;
        join.out[r] = calls[r].result;
    }
    const uint64_t need = NormWorkspace(tensors);
    double* partial = nullptr;
    for (uint32_t r = 0; r < w->n && partial == nullptr; ++r) {
        partial = calls[r].workspaceBytes >= need ? static_cast<double*>(calls[r].workspace) : nullptr;
    }
    if (partial == nullptr) {
        Log(1, "GradNorm: %llu tensors need a workspace of %llu bytes", (unsigned long long)tensors, (unsigned long long)need);
        return HCCL_E_MEMORY;
    }
    join.partial = partial;
    join.maxNorm = calls[0].maxNorm;
    join.scale = calls[0].scale;
    join.nOut = w->n;
    NormArgs a = {};
    uint32_t nTensors = 0;
    const auto flush = [&]() -> HcclResult {
        if (a.nChunks != 0) {
            if ((join.nPartial + kNormGroups) * sizeof(double) > need) {
                return HCCL_E_INTERNAL;
            }
            a.partial = partial + join.nPartial;
            a.perGroup = (a.nChunks + kNormGroups - 1) / kNormGroups;
            const uint32_t groups = (a.nChunks + a.perGroup - 1) / a.perGroup;
            for (uint32_t i = nTensors; i < kNormBatch; ++i) {
                a.chunkEnd[i] = 0xFFFFFFFFu;
            }
            for (uint32_t i = 0; i < 32; ++i) {
                a.groupEnd[i] = i < kNormBatch / 16 ? a.chunkEnd[16 * i + 15] : 0xFFFFFFFFu;
            }
            HIP_OK(LaunchNormBatch(a, groups, s));
            join.nPartial += groups;
        }
        nTensors = a.nChunks = 0;
        return HCCL_SUCCESS;
    };
    for (uint32_t r = 0; r < w->n; ++r) {
        const uint64_t* d = p.ranks[r].var.data() + kNormCallWords;
        for (uint64_t i = 0; i < calls[r].tensorCount; ++i, d += 3) {
            const HcclDataType type = static_cast<HcclDataType>(d[2]);
            const uint64_t perChunk = kNormChunkBytes / DataTypeSize(type);
            const uint64_t chunks = (d[1] + perChunk - 1) / perChunk;
            if (chunks == 0) {
                continue;
            }
            if (nTensors == kNormBatch || a.nChunks + chunks > kMaxChunks) {
                HcclResult rc = flush();
                if (rc != HCCL_SUCCESS) {
                    return rc;
                }
            }
            a.nChunks += static_cast<uint32_t>(chunks);
            const uint64_t lastChunk = (d[1] - (chunks - 1) * perChunk) * DataTypeSize(type) - 1;
            const uint64_t code = type == HCCL_DATA_TYPE_FP32 ? 0u : type == HCCL_DATA_TYPE_BFP16 ? 1u : 2u;
            a.tensor[nTensors] = d[0] | (lastChunk << 2 | code) << kNormAddressBits;
            a.chunkEnd[nTensors] = a.nChunks;
            nTensors++;
        }
    }
    HcclResult rc = flush();
    if (rc != HCCL_SUCCESS) {
        return rc;
    }
    HIP_OK(LaunchNormJoin(join, s));
    return HCCL_SUCCESS;
}

HcclResult RunTokenLogProbs(World* w, PendingOp& p, hipStream_t s)
{
    return Guarded("HcclAmdTokenLogProbs", [&] { return LaunchTokenLogProbs(w, p, s); });
}

HcclResult RunGradNorm(World* w, PendingOp& p, hipStream_t s)
{
    return Guarded("HcclAmdGradNorm", [&] { return LaunchGradNorm(w, p, s); });
}

// The first checks of every entry point; `ref` is looked up before, so that a collective's call that fails a check keeps
// its place in the sequence.
HcclResult CheckHandles(const char* name, HcclComm comm, const CommRef& ref, aclrtStream stream)
{
    if (stream == nullptr || comm == nullptr) {
        Log(1, "%s: %s is nullptr", name, stream == nullptr ? "stream" : "comm");
        return HCCL_E_PTR;
    }
    if (ref.c == nullptr) {
        Log(1, "%s: comm is not a live communicator", name);
        return HCCL_E_PARA;
    }
    return CheckUserRank(ref.c);
}

// A rank-local operator's last checks: what a collective learns from the rendezvous.
HcclResult CheckLocal(const char* name, const CommRef& ref)
{
    World* w = ref.c->world;
    std::lock_guard<std::mutex> lock(w->mu);
    if (w->envInvalid) {
        return HCCL_E_PARA;
    }
    if (w->destroyed != 0) {
        Log(1, "%s on rank %u: a communicator of this world has been destroyed", name, ref.c->rank);
        return HCCL_E_UNAVAIL;
    }
    return HCCL_SUCCESS;
}

HcclResult CheckTokenLogProbs(const char* name, const HcclAmdTokenLogProbsArgs& a)
{
    HcclResult rc = CheckLogits(name, a.logits, a.rowStride, a.vocabStart, a.vocabCount, a.tokenCount, a.dataType,
                                a.tokenType, a.scale, a.topCount);
    if (rc != HCCL_SUCCESS) {
        return rc;
    }
    if (a.logProbs != nullptr && a.tokens == nullptr) {
        Log(1, "%s: tokens is nullptr", name);
        return HCCL_E_PTR;
    }
    const uint32_t tokenSize = DataTypeSize(a.tokenType);
    if (!Aligned(a.tokens, tokenSize) || !Aligned(a.topIds, tokenSize)) {
        Log(1, "%s: tokens or topIds is not element-aligned", name);
        return HCCL_E_PARA;
    }
    for (const void* p : {a.logProbs, a.logSumExp, a.entropy, a.topValues}) {
        if ((rc = CheckAligned(name, p, 4, "an output")) != HCCL_SUCCESS) {
            return rc;
        }
    }
    return CheckAligned(name, a.workspace, 16, "the workspace");
}

HcclResult CheckNormTensors(const char* name, const HcclAmdNormTensor* tensors, uint32_t tensorCount)
{
    if (tensorCount != 0 && tensors == nullptr) {
        Log(1, "%s: tensors is nullptr", name);
        return HCCL_E_PTR;
    }
    for (uint32_t i = 0; i < tensorCount; ++i) {
        const HcclAmdNormTensor& t = tensors[i];
        if (!IsLogitsType(t.dataType)) {
            Log(1, "%s: tensor %u has type %d", name, i, static_cast<int>(t.dataType));
            return HCCL_E_NOT_SUPPORT;
        }
        if (t.count != 0 && t.data == nullptr) {
            Log(1, "%s: data of tensor %u is nullptr", name, i);
            return HCCL_E_PTR;
        }
        if (t.count >= 1ull << 40 || !Aligned(t.data, DataTypeSize(t.dataType)) ||
            reinterpret_cast<uint64_t>(t.data) >> kNormAddressBits != 0) {
            Log(1, "%s: tensor %u has %llu elements, is not element-aligned or at no device address", name, i, (unsigned long long)t.count);
            return HCCL_E_PARA;
        }
    }
    return HCCL_SUCCESS;
}

HcclResult CheckAdamWTensor(const char* name, uint32_t i, const HcclAmdAdamWTensor& t, bool fp8)
{
    const bool types = IsLogitsType(t.paramType) && IsLogitsType(t.gradType) &&
                       (t.gradType == t.paramType || t.gradType == HCCL_DATA_TYPE_FP32 || t.paramType == HCCL_DATA_TYPE_FP32);
    if (!types || (t.master != nullptr && t.paramType == HCCL_DATA_TYPE_FP32)) {
        Log(1, "%s: tensor %u has weights of type %d%s and gradients of type %d", name, i, static_cast<int>(t.paramType),
            t.master != nullptr ? " with 32-bit master weights" : "", static_cast<int>(t.gradType));
        return HCCL_E_NOT_SUPPORT;
    }
    if (t.count != 0 && (t.param == nullptr || t.grad == nullptr || t.expAvg == nullptr || t.expAvgSq == nullptr ||
                         (fp8 && (t.expAvgScale == nullptr || t.expAvgSqScale == nullptr)))) {
        Log(1, "%s: a buffer of tensor %u is nullptr", name, i);
        return HCCL_E_PTR;
    }
    const uint64_t state = fp8 ? 1 : 4;
    if (t.count >= 1ull << 40 || !Aligned(t.param, DataTypeSize(t.paramType)) || !Aligned(t.grad, DataTypeSize(t.gradType)) ||
        !Aligned(t.expAvg, state) || !Aligned(t.expAvgSq, state) || !Aligned(t.master, 4) || !Aligned(t.expAvgScale, 4) ||
        !Aligned(t.expAvgSqScale, 4)) {
        Log(1, "%s: tensor %u has %llu elements or a buffer that is not element-aligned", name, i, (unsigned long long)t.count);
        return HCCL_E_PARA;
    }
    return HCCL_SUCCESS;
}

HcclResult CheckAdamWConfig(const char* name, const HcclAmdAdamWConfig& c)
{
    if (c.stateType != HCCL_DATA_TYPE_FP32 && c.stateType != HCCL_DATA_TYPE_FP8E4M3) {
        Log(1, "%s: states of type %d are not supported", name, static_cast<int>(c.stateType));
        return HCCL_E_NOT_SUPPORT;
    }
    const bool betas = c.beta1 >= 0 && c.beta1 < 1 && c.beta2 >= 0 && c.beta2 < 1;
    const bool eps = c.eps == 0 || (c.eps >= 0x1p-126 && std::isfinite(c.eps));      // (reciprocals of less are infinite)
    if (!betas || !eps || !std::isfinite(c.weightDecay) ||
        (c.lrOnDevice == nullptr && !std::isfinite(c.lr)) || (c.stepOnDevice == nullptr && c.step == 0)) {
        Log(1, "%s: lr %g, betas %g %g, eps %g, weight decay %g, step %llu are out of range", name, c.lr, c.beta1, c.beta2,
            c.eps, c.weightDecay, (unsigned long long)c.step);
        return HCCL_E_PARA;
    }
    if (!Aligned(c.stepOnDevice, 8) || !Aligned(c.lrOnDevice, 4) || !Aligned(c.clip, 4)) {
        Log(1, "%s: a device scalar is not aligned", name);
        return HCCL_E_PARA;
    }
    return HCCL_SUCCESS;
}

constexpr uint32_t kMaxAdamWChunks = 1u << 23;

// Tensors of one combination of types, in batches.
HcclResult RunAdamW(const HcclAmdAdamWTensor* tensors, uint32_t tensorCount, AdamWArgs& a, bool fp8, hipStream_t s)
{
    std::vector<uint8_t> done(tensorCount, 0);
    for (uint32_t i = 0; i < tensorCount; ++i) {
        if (done[i] || tensors[i].count == 0) {
            continue;
        }
        const HcclAmdAdamWTensor& like = tensors[i];
        const bool master = like.master != nullptr;
        const uint32_t stride = AdamWTensorWords(master, fp8);
        uint32_t chunks = 0;
        a.nTensors = 0;
        const auto flush = [&]() -> HcclResult {
            if (chunks != 0) {
                HIP_OK(LaunchAdamW(a, like.paramType, like.gradType, master, fp8, chunks, s));
            }
            chunks = a.nTensors = 0;
            return HCCL_SUCCESS;
        };
        for (uint32_t j = i; j < tensorCount; ++j) {
            const HcclAmdAdamWTensor& t = tensors[j];
            if (done[j] || t.count == 0 || t.paramType != like.paramType || t.gradType != like.gradType ||
                (t.master != nullptr) != master) {
                continue;
            }
            done[j] = 1;
            const uint64_t ps = DataTypeSize(t.paramType), gs = DataTypeSize(t.gradType), ss = fp8 ? 1 : 4;
            // A launch has fewer than 2^32 work items: a tensor of more than 2^23 chunks takes several pieces.
            for (uint64_t at = 0; at < t.count;) {
                if ((a.nTensors + 1) * stride > kAdamWWords || chunks == kMaxAdamWChunks) {
                    HcclResult rc = flush();
                    if (rc != HCCL_SUCCESS) {
                        return rc;
                    }
                }
                const uint64_t room = static_cast<uint64_t>(kMaxAdamWChunks - chunks) * kAdamWChunk;
                const uint64_t n = t.count - at < room ? t.count - at : room;
                const uint64_t mine = (n + kAdamWChunk - 1) / kAdamWChunk;
                chunks += static_cast<uint32_t>(mine);
                uint64_t* d = a.table + static_cast<size_t>(a.nTensors++) * stride;
                *d++ = chunks | (n - (mine - 1) * kAdamWChunk) << 32;
                *d++ = reinterpret_cast<uint64_t>(t.param) + at * ps;
                *d++ = reinterpret_cast<uint64_t>(t.grad) + at * gs;
                *d++ = reinterpret_cast<uint64_t>(t.expAvg) + at * ss;
                *d++ = reinterpret_cast<uint64_t>(t.expAvgSq) + at * ss;
                if (master) {
                    *d++ = reinterpret_cast<uint64_t>(t.master + at);
                }
                if (fp8) {
                    *d++ = reinterpret_cast<uint64_t>(t.expAvgScale + at / HCCL_AMD_STATE_BLOCK);
                    *d++ = reinterpret_cast<uint64_t>(t.expAvgSqScale + at / HCCL_AMD_STATE_BLOCK);
                }
                at += n;
            }
        }
        HcclResult rc = flush();
        if (rc != HCCL_SUCCESS) {
            return rc;
        }
    }
    return HCCL_SUCCESS;
}

}  // namespace

extern "C" {

HcclResult HcclAmdTokenLogProbs(const HcclAmdTokenLogProbsArgs* args, HcclComm comm, aclrtStream stream)
{
    return Guarded(__func__, [&]() -> HcclResult {
        const char* name = "HcclAmdTokenLogProbs";
        CommRef ref = AsComm(comm);   // looked up first, so that a call that fails any check below keeps its place
        if (args != nullptr && args->tokenCount == 0) {
            return HCCL_SUCCESS;
        }
        HcclResult rc = CheckHandles(name, comm, ref, stream);
        if (rc == HCCL_SUCCESS && args == nullptr) {
            Log(1, "%s: args is nullptr", name);
            rc = HCCL_E_PTR;
        }
        if (rc == HCCL_SUCCESS) {
            rc = CheckTokenLogProbs(name, *args);
        }
        if (rc != HCCL_SUCCESS) {
            return Reject(ref, OpType::TOKEN_LOG_PROBS, rc);
        }
        if (ref.c->world->envInvalid) {
            return HCCL_E_PARA;
        }
        return Submit(ref, OpType::TOKEN_LOG_PROBS, args->dataType, HCCL_REDUCE_RESERVED, args->tokenCount, args->logits,
                      nullptr, static_cast<hipStream_t>(stream), Words(*args), args->topCount, false, RunTokenLogProbs);
    });
}

HcclResult HcclAmdTokenLogProbsWorkspace(uint64_t tokenCount, uint64_t vocabSize, uint32_t topCount, uint64_t* bytes)
{
    if (bytes == nullptr) {
        Log(1, "%s: bytes is nullptr", __func__);
        return HCCL_E_PTR;
    }
    if (tokenCount > kMaxRows || vocabSize > kMaxVocab || topCount > kMaxTop) {
        Log(1, "%s: %llu rows of %llu entries with %u alternatives are out of range", __func__, (unsigned long long)tokenCount,
            (unsigned long long)vocabSize, topCount);
        return HCCL_E_PARA;
    }
    *bytes = LogProbsWorkspace(tokenCount, vocabSize, topCount);
    return HCCL_SUCCESS;
}

HcclResult HcclAmdTokenLogProbsGrad(const HcclAmdTokenLogProbsGradArgs* args, HcclComm comm, aclrtStream stream)
{
    return Guarded(__func__, [&]() -> HcclResult {
        const char* name = "HcclAmdTokenLogProbsGrad";
        CommRef ref = AsComm(comm);
        if (args != nullptr && (args->tokenCount == 0 || args->vocabCount == 0)) {
            return HCCL_SUCCESS;
        }
        HcclResult rc = CheckHandles(name, comm, ref, stream);
        if (rc != HCCL_SUCCESS) {
            return rc;
        }
        if (args == nullptr) {
            Log(1, "%s: args is nullptr", name);
            return HCCL_E_PTR;
        }
        const HcclAmdTokenLogProbsGradArgs& a = *args;
        rc = CheckLogits(name, a.logits, a.rowStride, a.vocabStart, a.vocabCount, a.tokenCount, a.dataType, a.tokenType,
                         a.scale, a.topCount);
        if (rc != HCCL_SUCCESS) {
            return rc;
        }
        const bool top = a.gradTopValues != nullptr && a.topCount != 0;
        if (a.gradLogits == nullptr || a.logSumExp == nullptr || (a.gradLogProbs != nullptr && a.tokens == nullptr) ||
            (a.gradEntropy != nullptr && a.entropy == nullptr) || (top && a.topIds == nullptr) ||
            (a.gradLogProbs == nullptr && a.gradEntropy == nullptr && !top)) {
            Log(1, "%s: a buffer that the gradients need, or every gradient, is nullptr", name);
            return HCCL_E_PTR;
        }
        const uint64_t size = DataTypeSize(a.dataType), idSize = DataTypeSize(a.tokenType);
        if (a.gradRowStride < a.vocabCount || a.gradRowStride > kMaxRowStride) {
            Log(1, "%s: a row stride of %llu does not fit %llu entries", name, (unsigned long long)a.gradRowStride,
                (unsigned long long)a.vocabCount);
            return HCCL_E_PARA;
        }
        if (!Aligned(a.gradLogits, size) || !Aligned(a.tokens, idSize) || !Aligned(a.topIds, idSize) ||
            !Aligned(a.logSumExp, 4) || !Aligned(a.entropy, 4) || !Aligned(a.gradLogProbs, 4) || !Aligned(a.gradEntropy, 4) ||
            !Aligned(a.gradTopValues, 4)) {
            Log(1, "%s: a buffer is not element-aligned", name);
            return HCCL_E_PARA;
        }
        // In place or apart.  (Two parts of one matrix, rows interleaved, are apart: same stride, less than a row away.)
        const uint64_t x = reinterpret_cast<uint64_t>(a.logits), d = reinterpret_cast<uint64_t>(a.gradLogits);
        const uint64_t xEnd = x + ((a.tokenCount - 1) * a.rowStride + a.vocabCount) * size;
        const uint64_t dEnd = d + ((a.tokenCount - 1) * a.gradRowStride + a.vocabCount) * size;
        const uint64_t off = x > d ? x - d : d - x, stride = a.rowStride * size, row = a.vocabCount * size;
        const bool same = x == d && (a.rowStride == a.gradRowStride || a.tokenCount == 1);
        const bool woven = a.rowStride == a.gradRowStride && off % stride >= row && off % stride + row <= stride;
        if (x < dEnd && d < xEnd && !same && !woven) {
            Log(1, "%s: gradLogits overlaps the logits without being them", name);
            return HCCL_E_PARA;
        }
        // What a workgroup reads of its row, others may still need when it writes.
        const uint64_t ids = a.tokenCount * a.topCount, pitch = a.gradRowStride * size;
        const struct {
            const void* data;
            uint64_t bytes;
        } read[] = {{a.logSumExp, 4 * a.tokenCount},
                    {a.gradLogProbs != nullptr ? a.tokens : nullptr, idSize * a.tokenCount},
                    {a.gradLogProbs, 4 * a.tokenCount},
                    {a.gradEntropy != nullptr ? a.entropy : nullptr, 4 * a.tokenCount},
                    {a.gradEntropy, 4 * a.tokenCount},
                    {top ? a.topIds : nullptr, idSize * ids},
                    {top ? a.gradTopValues : nullptr, 4 * ids}};
        for (const auto& r : read) {
            const uint64_t at = reinterpret_cast<uint64_t>(r.data);
            if (r.data == nullptr || at >= dEnd || at + r.bytes <= d) {
                continue;
            }
            const bool between = at >= d && (at - d) % pitch >= row && (at - d) % pitch + r.bytes <= pitch;
            if (!between) {
                Log(1, "%s: gradLogits overlaps an array that the rows' numbers are read from", name);
                return HCCL_E_PARA;
            }
        }
        rc = CheckLocal(name, ref);
        if (rc != HCCL_SUCCESS) {
            return rc;
        }
        LogProbsGradArgs k = {};
        k.logits = a.logits;
        k.grad = a.gradLogits;
        k.rowStride = a.rowStride;
        k.gradRowStride = a.gradRowStride;
        k.vocabStart = static_cast<uint32_t>(a.vocabStart);
        k.count = static_cast<uint32_t>(a.vocabCount);
        k.topCount = top ? a.topCount : 0;
        k.wideTokens = a.tokenType == HCCL_DATA_TYPE_INT64 ? 1 : 0;
        k.scale = a.scale;
        k.tokens = a.tokens;
        k.logSumExp = a.logSumExp;
        k.entropy = a.entropy;
        k.gradLogProbs = a.gradLogProbs;
        k.gradEntropy = a.gradEntropy;
        k.topIds = top ? a.topIds : nullptr;
        k.gradTop = top ? a.gradTopValues : nullptr;
        DeviceScope onWorldDevice(ref.c->world->device);
        HIP_OK(LaunchLogProbsGrad(k, a.dataType, static_cast<uint32_t>(a.tokenCount), static_cast<hipStream_t>(stream)));
        return HCCL_SUCCESS;
    });
}

HcclResult HcclAmdGradNorm(const HcclAmdNormTensor* tensors, uint32_t tensorCount, float maxNorm, float scale, float* result,
                           void* workspace, uint64_t workspaceBytes, HcclComm comm, aclrtStream stream)
{
    return Guarded(__func__, [&]() -> HcclResult {
        const char* name = "HcclAmdGradNorm";
        CommRef ref = AsComm(comm);   // looked up first, so that a call that fails any check below keeps its place
        HcclResult rc = CheckHandles(name, comm, ref, stream);
        if (rc == HCCL_SUCCESS && result == nullptr) {
            Log(1, "%s: result is nullptr", name);
            rc = HCCL_E_PTR;
        }
        if (rc == HCCL_SUCCESS && (!std::isfinite(maxNorm) || !std::isfinite(scale) || !Aligned(result, 4))) {
            Log(1, "%s: maxNorm %g or scale %g is not finite, or result is not aligned", name, static_cast<double>(maxNorm),
                static_cast<double>(scale));
            rc = HCCL_E_PARA;
        }
        if (rc == HCCL_SUCCESS) {
            rc = CheckAligned(name, workspace, 16, "the workspace");
        }
        if (rc == HCCL_SUCCESS) {
            rc = CheckNormTensors(name, tensors, tensorCount);
        }
        if (rc != HCCL_SUCCESS) {
            return Reject(ref, OpType::GRAD_NORM, rc);
        }
        if (ref.c->world->envInvalid) {
            return HCCL_E_PARA;
        }
        const NormCall call = {maxNorm, scale, result, workspace, workspaceBytes, tensorCount};
        std::vector<uint64_t> words = Words(call, 3 * static_cast<size_t>(tensorCount));
        for (uint32_t i = 0; i < tensorCount; ++i) {
            uint64_t* d = words.data() + kNormCallWords + 3 * static_cast<size_t>(i);
            d[0] = reinterpret_cast<uint64_t>(tensors[i].data);
            d[1] = tensors[i].count;
            d[2] = static_cast<uint64_t>(tensors[i].dataType);
        }
        return Submit(ref, OpType::GRAD_NORM, HCCL_DATA_TYPE_FP32, HCCL_REDUCE_RESERVED, 1, result, result,
                      static_cast<hipStream_t>(stream), std::move(words), 0, false, RunGradNorm);
    });
}

HcclResult HcclAmdGradNormWorkspace(uint64_t tensorCount, uint64_t* bytes)
{
    if (bytes == nullptr) {
        Log(1, "%s: bytes is nullptr", __func__);
        return HCCL_E_PTR;
    }
    if (tensorCount > 1ull << 40) {
        Log(1, "%s: %llu tensors are out of range", __func__, (unsigned long long)tensorCount);
        return HCCL_E_PARA;
    }
    *bytes = NormWorkspace(tensorCount);
    return HCCL_SUCCESS;
}

HcclResult HcclAmdAdamW(const HcclAmdAdamWTensor* tensors, uint32_t tensorCount, const HcclAmdAdamWConfig* config,
                        HcclComm comm, aclrtStream stream)
{
    return Guarded(__func__, [&]() -> HcclResult {
        const char* name = "HcclAmdAdamW";
        CommRef ref = AsComm(comm);
        HcclResult rc = CheckHandles(name, comm, ref, stream);
        if (rc != HCCL_SUCCESS) {
            return rc;
        }
        if (config == nullptr || (tensorCount != 0 && tensors == nullptr)) {
            Log(1, "%s: %s is nullptr", name, config == nullptr ? "config" : "tensors");
            return HCCL_E_PTR;
        }
        const HcclAmdAdamWConfig& c = *config;
        rc = CheckAdamWConfig(name, c);
        const bool fp8 = c.stateType == HCCL_DATA_TYPE_FP8E4M3;
        for (uint32_t i = 0; rc == HCCL_SUCCESS && i < tensorCount; ++i) {
            rc = CheckAdamWTensor(name, i, tensors[i], fp8);
        }
        if (rc == HCCL_SUCCESS) {
            rc = CheckLocal(name, ref);
        }
        if (rc != HCCL_SUCCESS) {
            return rc;
        }
        AdamWArgs a = {};
        a.clip = c.clip;
        a.skipNonFinite = c.skipNonFinite != 0 ? 1 : 0;
        a.step = c.stepOnDevice;
        a.lr = c.lrOnDevice;
        a.beta1 = static_cast<float>(c.beta1);
        a.beta2 = static_cast<float>(c.beta2);
        a.oneMinusBeta1 = static_cast<float>(1.0 - c.beta1);
        a.oneMinusBeta2 = static_cast<float>(1.0 - c.beta2);
        a.eps = static_cast<float>(c.eps);
        a.weightDecay = static_cast<float>(c.weightDecay);
        a.hostLr = static_cast<float>(c.lr);
        a.logBeta1 = static_cast<float>(std::log(c.beta1));      // -inf for 0: the correction is then 1
        a.logBeta2 = static_cast<float>(std::log(c.beta2));
        a.correction1 = static_cast<float>(1.0 / (1.0 - std::pow(c.beta1, static_cast<double>(c.step))));
        a.rootCorrection2 = static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(c.beta2, static_cast<double>(c.step))));
        DeviceScope onWorldDevice(ref.c->world->device);
        return RunAdamW(tensors, tensorCount, a, fp8, static_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
