// Log probabilities of given tokens, entropy and top alternatives of rows of logits whose vocabulary lies in up to 64
// parts (one per rank).
//
// With x = scale * logit, one pass over a row keeps, per lane, the largest logit m, s = sum exp(x - scale m) and
// t = sum y exp2(y), y = log2(e) (x - scale m): whenever m grows, s and t are carried over to the new reference,
// s' = s c, t' = c (t + s d), c = exp2(d), d = log2(e) scale (m - m').  Differences to the maximum are formed before they
// are scaled, so that rows of the type's lowest value (a mask) come out like any other row of equal logits.
//   lse = scale m + ln s, entropy = ln s - ln 2 t / s.
//
// Alternatives without a second pass: the k-th largest of the 256 lane maxima bounds the k-th largest element of the row
// from below, since k lanes hold an element at least as large.  Only lanes whose maximum reaches the bound can hold one of
// the k, so their elements alone (k / 256 of the row, still in the cache) are looked at again; what reaches the bound is
// ranked by (logit, lower index).  Rows with so many equal logits that the list overflows are searched exactly instead.
//
// Bound: one read of the logits from HBM.  Every workgroup owns one row; where there are few rows, nSplit workgroups share
// each and a second kernel joins their partial results.
#include "model_ops.h"
#include "vec.h"

namespace hccl_amd {
namespace model_ops {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWaves = kThreads / kWave;
constexpr uint32_t kUnroll = 4;            // vectors a lane loads together
constexpr uint32_t kCandidates = 1024;     // elements of a row that may reach the bound before the exact search takes over
constexpr float kLowest = -3.402823466e38f;
constexpr float kFarBelow = -1e30f;        // stands for -inf where it is multiplied by a zero probability
constexpr float kLn2 = 0.69314718055994531f;

// Order of floats as unsigned integers; both zeros are one value.
__device__ __forceinline__ uint32_t Ordered(float x)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float FromOrdered(uint32_t o)
{
    return __builtin_bit_cast(float, o ^ (static_cast<uint32_t>(static_cast<int32_t>(~o) >> 31) | 0x80000000u));
}
// Larger logit first, then the lower index.  0 is below every element's key.
__device__ __forceinline__ uint64_t Key(uint32_t ordered, uint32_t index)
{
    return (static_cast<uint64_t>(ordered) << 32) | (0xFFFFFFFFu - index);
}

struct Stats {
    float m, s, t;
};

__device__ __forceinline__ void Rescale(Stats& a, float m, float exp2Scale)
{
    const float d = fmaxf((a.m - m) * exp2Scale, kFarBelow);
    const float c = Exp2(d);
    a.t = c * (a.t + a.s * d);
    a.s = a.s * c;
    a.m = m;
}

// The same numbers for the union; both sides end up on the larger maximum.
__device__ __forceinline__ Stats Join(Stats a, Stats b, float exp2Scale)
{
    const float m = fmaxf(a.m, b.m);
    Rescale(a, m, exp2Scale);
    Rescale(b, m, exp2Scale);
    return Stats{m, a.s + b.s, a.t + b.t};
}

__device__ __forceinline__ Stats WaveJoin(Stats a, float exp2Scale)
{
    Stats r;
    r.m = WaveMax(a.m);
    Rescale(a, r.m, exp2Scale);
    r.s = WaveSum(a.s);
    r.t = WaveSum(a.t);
    return r;
}

template <uint32_t N>
__device__ __forceinline__ void Accumulate(Stats& a, const float* x, float exp2Scale)
{
    float most = x[0];
    for (uint32_t i = 1; i < N; ++i) {
        most = fmaxf(most, x[i]);
    }
    if (most > a.m) {
        Rescale(a, most, exp2Scale);
    }
    for (uint32_t i = 0; i < N; ++i) {
        const float y = (x[i] - a.m) * exp2Scale;
        const float e = Exp2(y);
        a.s += e;
        a.t = __builtin_fmaf(fmaxf(y, kFarBelow), e, a.t);
    }
}

// The part of one shard's row that this workgroup reads: vectors [first, last) of which those below `full` are whole.
template <typename T>
struct Range {
    const typename T::Raw* row;
    uint32_t count;
    uint32_t full;
    uint32_t first;
    uint32_t last;

    __device__ __forceinline__ Range(const LogProbsArgs& a, uint32_t shard, uint64_t r, uint32_t split)
    {
        row = static_cast<const typename T::Raw*>(a.logits[shard]) + r * a.rowStride[shard];
        count = a.count[shard];
        full = count / kPer16<T>;
        const uint32_t vectors = (count + kPer16<T> - 1) / kPer16<T>;
        first = static_cast<uint32_t>(static_cast<uint64_t>(vectors) * split / a.nSplit);
        last = static_cast<uint32_t>(static_cast<uint64_t>(vectors) * (split + 1) / a.nSplit);
    }
    // Elements of vector v; the places behind the end of the row get -inf.
    __device__ __forceinline__ void Get(uint32_t v, float* x) const
    {
        if (v < full) {
            Unpack16<T>(Load16(row + static_cast<uint64_t>(v) * kPer16<T>), x);
        } else {
            for (uint32_t i = 0; i < kPer16<T>; ++i) {
                const uint32_t at = v * kPer16<T> + i;
                x[i] = at < count ? Widen<T>(LoadOne(row + at)) : -__builtin_inff();
            }
        }
    }
    __device__ __forceinline__ uint32_t Valid(uint32_t v) const
    {
        return v < full ? kPer16<T> : count - v * kPer16<T>;
    }
};

// Descending bitonic sort of one value per lane.
__device__ __forceinline__ uint32_t WaveSort(uint32_t v, uint32_t lane)
{
    for (uint32_t size = 2; size <= kWave; size <<= 1) {
        for (uint32_t d = size >> 1; d > 0; d >>= 1) {
            const uint32_t o = __shfl_xor(v, d);
            const bool keepMax = ((lane & d) == 0) == ((lane & size) == 0);
            v = keepMax ? (v > o ? v : o) : (v < o ? v : o);
        }
    }
    return v;
}

// Sorts a bitonic sequence of 32 in each half of the wavefront, descending.
__device__ __forceinline__ uint32_t HalfMerge(uint32_t v, uint32_t lane)
{
    for (uint32_t d = 16; d > 0; d >>= 1) {
        const uint32_t o = __shfl_xor(v, d);
        v = (lane & d) == 0 ? (v > o ? v : o) : (v < o ? v : o);
    }
    return v;
}

struct TopSpace {
    uint32_t sorted[kWaves][32];
    uint32_t lanes[kThreads];
    uint64_t candidate[kCandidates];
    uint32_t nLanes;
    uint32_t nCandidates;
    uint32_t bound;
    uint32_t total;
    uint32_t waveCount[kWaves];
};

// Sum over the workgroup; every thread gets it.
__device__ __forceinline__ uint32_t BlockCount(uint32_t v, TopSpace& sh, uint32_t tid)
{
    for (int d = 32; d > 0; d >>= 1) {
        v += __shfl_xor(v, d);
    }
    __syncthreads();
    if ((tid & (kWave - 1)) == 0) {
        sh.waveCount[tid / kWave] = v;
    }
    __syncthreads();
    uint32_t sum = 0;
    for (uint32_t w = 0; w < kWaves; ++w) {
        sum += sh.waveCount[w];
    }
    return sum;
}

// Elements of the workgroup's part of the row whose order is at least (or, above = true, above) `bound`.
template <typename T>
__device__ __forceinline__ uint32_t CountFrom(const LogProbsArgs& a, uint64_t row, uint32_t split, uint32_t bound, bool above, TopSpace& sh,
                              uint32_t tid)
{
    uint32_t n = 0;
    for (uint32_t shard = 0; shard < a.nShards; ++shard) {
        const Range<T> r(a, shard, row, split);
        for (uint32_t v = r.first + tid; v < r.last; v += kThreads) {
            float x[kPer16<T>];
            r.Get(v, x);
            const uint32_t valid = r.Valid(v);
            for (uint32_t i = 0; i < kPer16<T>; ++i) {
                const uint32_t o = Ordered(x[i]);
                n += (i < valid && (above ? o > bound : o >= bound)) ? 1 : 0;
            }
        }
    }
    return BlockCount(n, sh, tid);
}

// The exact search, for rows with more elements at the bound than the list holds: the topCount-th largest logit by
// bisection, then everything above it and, in ascending order, as many equal to it as are still wanted.  A dozen or more
// passes over the (cached) row in general, two where the bound itself is the largest logit, as in a row of equal ones.
template <typename T>
__device__ __forceinline__ void SearchTop(const LogProbsArgs& a, uint64_t row, uint32_t split, uint32_t most, TopSpace& sh,
                                       uint32_t tid)
{
    uint32_t low = sh.bound;       // at least topCount elements reach it
    uint32_t high = most;          // nothing lies above it
    uint32_t above = CountFrom<T>(a, row, split, low, true, sh, tid);
    if (above >= a.topCount) {
        while (low < high) {       // the largest value that topCount elements reach
            const uint32_t mid = low + (high - low + 1) / 2;
            if (CountFrom<T>(a, row, split, mid, false, sh, tid) >= a.topCount) {
                low = mid;
            } else {
                high = mid - 1;
            }
        }
        above = CountFrom<T>(a, row, split, low, true, sh, tid);
    }
    uint32_t want = a.topCount - above;    // of those equal to `low`
    __syncthreads();
    if (tid == 0) {
        sh.nCandidates = 0;
    }
    __syncthreads();
    uint32_t start = 0;
    for (uint32_t shard = 0; shard < a.nShards; ++shard) {
        const Range<T> r(a, shard, row, split);
        for (uint32_t v0 = r.first; v0 < r.last; v0 += kThreads) {
            const uint32_t v = v0 + tid;
            uint32_t equal = 0;     // bit i: element i equals `low`
            if (v < r.last) {
                float x[kPer16<T>];
                r.Get(v, x);
                const uint32_t valid = r.Valid(v);
                for (uint32_t i = 0; i < kPer16<T>; ++i) {
                    const uint32_t o = Ordered(x[i]);
                    if (i < valid && o > low) {
                        sh.candidate[atomicAdd(&sh.nCandidates, 1u)] = Key(o, start + v * kPer16<T> + i);
                    }
                    equal |= (i < valid && o == low) ? 1u << i : 0u;
                }
            }
            if (want != 0) {
                // position of the lane's first equal element among those of all lanes
                const uint32_t mine = __popc(equal);
                uint32_t before = mine;
                for (uint32_t d = 1; d < kWave; d <<= 1) {
                    const uint32_t o = __shfl_up(before, d);
                    before += (tid & (kWave - 1)) >= d ? o : 0;
                }
                __syncthreads();
                if ((tid & (kWave - 1)) == kWave - 1) {
                    sh.waveCount[tid / kWave] = before;
                }
                __syncthreads();
                uint32_t total = 0;
                before -= mine;
                for (uint32_t w = 0; w < kWaves; ++w) {
                    before += w < tid / kWave ? sh.waveCount[w] : 0;
                    total += sh.waveCount[w];
                }
                for (uint32_t i = 0; i < kPer16<T>; ++i) {
                    if ((equal >> i) & 1u) {
                        if (before < want) {
                            sh.candidate[atomicAdd(&sh.nCandidates, 1u)] = Key(low, start + v * kPer16<T> + i);
                        }
                        ++before;
                    }
                }
                want -= total < want ? total : want;
            }
        }
        start += r.count;
    }
    __syncthreads();
}

// Leaves at least the topCount largest keys of the workgroup's part of the row (all keys if it is shorter) in
// sh.candidate, at most kCandidates.  laneMost: order of the lane's largest logit, 0 if it had no element.
template <typename T>
__device__ __forceinline__ void GatherTop(const LogProbsArgs& a, uint64_t row, uint32_t split, uint32_t laneMost, TopSpace& sh, uint32_t tid)
{
    const uint32_t lane = tid & (kWave - 1);
    const uint32_t sorted = WaveSort(laneMost, lane);
    if (lane < 32) {
        sh.sorted[tid / kWave][lane] = sorted;
    }
    if (tid == 0) {
        sh.nLanes = 0;
        sh.nCandidates = 0;
    }
    __syncthreads();
    if (tid < kWave) {
        // lanes 0..31: the 32 largest of wavefronts 0 and 1, lanes 32..63: of 2 and 3; then of both
        const uint32_t i = lane & 31u, pair = (lane >> 5) * 2;
        const uint32_t x = sh.sorted[pair][i], y = sh.sorted[pair + 1][31 - i];
        uint32_t v = HalfMerge(x > y ? x : y, lane);
        const uint32_t o = __shfl(v, 63 - lane);
        v = HalfMerge(v > o ? v : o, lane);
        if (lane == 0) {
            sh.total = v;          // the largest
        }
        if (lane == a.topCount - 1) {
            sh.bound = v;
        }
    }
    __syncthreads();
    const uint32_t bound = sh.bound;
    if (laneMost != 0 && laneMost >= bound) {
        sh.lanes[atomicAdd(&sh.nLanes, 1u)] = tid;
    }
    __syncthreads();
    const uint32_t nLanes = sh.nLanes;
    uint32_t start = 0;
    for (uint32_t shard = 0; shard < a.nShards; ++shard) {
        const Range<T> r(a, shard, row, split);
        const uint32_t perLane = (r.last - r.first + kThreads - 1) / kThreads;
        for (uint32_t item = tid; item < nLanes * perLane; item += kThreads) {
            const uint32_t j = item / nLanes;
            const uint32_t v = r.first + j * kThreads + sh.lanes[item - j * nLanes];
            if (v < r.last) {
                float x[kPer16<T>];
                r.Get(v, x);
                const uint32_t valid = r.Valid(v);
                for (uint32_t i = 0; i < kPer16<T>; ++i) {
                    const uint32_t o = Ordered(x[i]);
                    if (i < valid && o >= bound) {
                        const uint32_t at = atomicAdd(&sh.nCandidates, 1u);
                        if (at < kCandidates) {
                            sh.candidate[at] = Key(o, start + v * kPer16<T> + i);
                        }
                    }
                }
            }
        }
        start += r.count;
    }
    __syncthreads();
    if (sh.nCandidates > kCandidates) {
        SearchTop<T>(a, row, split, sh.total, sh, tid);
    }
}

// What is written for a row once its numbers are known.
struct RowResult {
    float m, logSum, lse, entropy;
    bool none;      // -inf alone
    bool bad;       // a NaN or +inf
};

__device__ __forceinline__ RowResult Finish(Stats a, float scale)
{
    RowResult r;
    r.m = a.m;
    r.none = a.s == 0.0f;
    r.bad = a.s != a.s;
    r.logSum = logf(a.s);
    r.lse = r.none ? -__builtin_inff() : a.m * scale + r.logSum;
    r.entropy = r.none ? 0.0f : r.logSum - kLn2 * (a.t / a.s);
    return r;
}

__device__ __forceinline__ float LogProbOf(const RowResult& r, float x, float scale)
{
    return r.none ? -__builtin_inff() : (x - r.m) * scale - r.logSum;
}

template <typename T>
__device__ __forceinline__ void WriteRow(const LogProbsArgs& a, uint64_t row, const RowResult& r)
{
    float logProb = 0.0f;
    if (a.tokens != nullptr) {
        const int64_t token = a.wideTokens ? LoadOne(static_cast<const int64_t*>(a.tokens) + row)
                                           : LoadOne(static_cast<const int32_t*>(a.tokens) + row);
        if (token >= a.vocab) {
            logProb = __builtin_nanf("");
        } else if (token >= 0) {
            uint32_t at = static_cast<uint32_t>(token);
            uint32_t shard = 0;
            while (at >= a.count[shard]) {
                at -= a.count[shard];
                ++shard;
            }
            const typename T::Raw* p = static_cast<const typename T::Raw*>(a.logits[shard]) + row * a.rowStride[shard] + at;
            logProb = LogProbOf(r, Widen<T>(LoadOne(p)), a.scale);
        }
    }
    for (uint32_t o = 0; o < a.nOut; ++o) {
        if (a.out[o].logProbs != nullptr) {
            StoreOne(a.out[o].logProbs + row, logProb);
        }
        if (a.out[o].logSumExp != nullptr) {
            StoreOne(a.out[o].logSumExp + row, r.lse);
        }
        if (a.out[o].entropy != nullptr) {
            StoreOne(a.out[o].entropy + row, r.entropy);
        }
    }
}

__device__ __forceinline__ void WriteTop(const LogProbsArgs& a, uint64_t row, const RowResult& r, uint32_t rank, uint64_t key)
{
    const float value = r.bad ? __builtin_nanf("") : LogProbOf(r, FromOrdered(static_cast<uint32_t>(key >> 32)), a.scale);
    const int64_t id = r.bad ? -1 : static_cast<int64_t>(0xFFFFFFFFu - static_cast<uint32_t>(key));
    const uint64_t at = row * a.topCount + rank;
    for (uint32_t o = 0; o < a.nOut; ++o) {
        if (a.out[o].topValues != nullptr) {
            StoreOne(a.out[o].topValues + at, value);
        }
        if (a.out[o].topIds != nullptr) {
            if (a.wideTokens) {
                StoreOne(static_cast<int64_t*>(a.out[o].topIds) + at, id);
            } else {
                StoreOne(static_cast<int32_t*>(a.out[o].topIds) + at, static_cast<int32_t>(id));
            }
        }
    }
}

template <typename T, bool kTop>
__global__ __launch_bounds__(kThreads) void LogProbsKernel(const LogProbsArgs a)
{
    constexpr uint32_t P = kPer16<T>;
    __shared__ Stats waveStats[kWaves];
    const uint32_t tid = threadIdx.x;
    const uint32_t split = blockIdx.x % a.nSplit;
    const uint64_t row = blockIdx.x / a.nSplit;
    Stats acc = {kLowest, 0.0f, 0.0f};
    bool any = false;
    for (uint32_t shard = 0; shard < a.nShards; ++shard) {
        const Range<T> r(a, shard, row, split);
        const uint32_t whole = r.last < r.full ? r.last : r.full;
        uint32_t v = r.first;
        for (; v + kThreads * kUnroll <= whole; v += kThreads * kUnroll) {
            U32x4 raw[kUnroll];
            for (uint32_t u = 0; u < kUnroll; ++u) {
                raw[u] = LoadOnce16(r.row + static_cast<uint64_t>(v + u * kThreads + tid) * P);
            }
            float x[kUnroll * P];
            for (uint32_t u = 0; u < kUnroll; ++u) {
                Unpack16<T>(raw[u], x + u * P);
            }
            Accumulate<kUnroll * P>(acc, x, a.exp2Scale);
            any = true;
        }
        for (v += tid; v < r.last; v += kThreads) {
            float x[P];
            r.Get(v, x);
            Accumulate<P>(acc, x, a.exp2Scale);
            any = true;
        }
    }
    const Stats wave = WaveJoin(acc, a.exp2Scale);
    if ((tid & (kWave - 1)) == 0) {
        waveStats[tid / kWave] = wave;
    }
    __syncthreads();
    Stats all = waveStats[0];
    for (uint32_t w = 1; w < kWaves; ++w) {
        all = Join(all, waveStats[w], a.exp2Scale);
    }
    const RowResult result = Finish(all, a.scale);
    if (tid == 0) {
        if (a.nSplit == 1) {
            WriteRow<T>(a, row, result);
        } else {
            float* p = a.stats + (row * a.nSplit + split) * 4;
            StoreOne(p, all.m);
            StoreOne(p + 1, all.s);
            StoreOne(p + 2, all.t);
        }
    }
    if constexpr (kTop) {
        if (result.bad) {     // a NaN has no place in an order: no alternatives
            if (tid < a.topCount) {
                if (a.nSplit == 1) {
                    WriteTop(a, row, result, tid, 0);
                } else {
                    StoreOne(a.keys + (row * a.nSplit + split) * a.topCount + tid, static_cast<uint64_t>(0));
                }
            }
            return;
        }
        __shared__ TopSpace sh;
        const float most = acc.s == 0.0f ? -__builtin_inff() : acc.m;
        GatherTop<T>(a, row, split, any ? Ordered(most) : 0u, sh, tid);
        const uint32_t n = sh.nCandidates;
        uint64_t* keys = a.keys + (row * a.nSplit + split) * a.topCount;
        for (uint32_t c = tid; c < n; c += kThreads) {
            const uint64_t key = sh.candidate[c];
            uint32_t rank = 0;
            for (uint32_t o = 0; o < n; ++o) {
                rank += sh.candidate[o] > key ? 1 : 0;
            }
            if (rank < a.topCount) {
                if (a.nSplit == 1) {
                    WriteTop(a, row, result, rank, key);
                } else {
                    StoreOne(keys + rank, key);
                }
            }
        }
        if (a.nSplit > 1) {
            for (uint32_t c = n + tid; c < a.topCount; c += kThreads) {
                StoreOne(keys + c, static_cast<uint64_t>(0));
            }
        }
    }
}

// Joins the nSplit partial results of a row.
constexpr uint32_t kMaxSplit = 64;
template <typename T>
__global__ __launch_bounds__(kThreads) void LogProbsJoinKernel(const LogProbsArgs a)
{
    const uint32_t tid = threadIdx.x;
    const uint64_t row = blockIdx.x;
    // every wavefront joins the numbers for itself, a lane per split
    Stats mine = {kLowest, 0.0f, 0.0f};
    const uint32_t lane = tid & (kWave - 1);
    if (lane < a.nSplit) {
        const float* p = a.stats + (row * a.nSplit + lane) * 4;
        mine = Stats{LoadOne(p), LoadOne(p + 1), LoadOne(p + 2)};
    }
    const RowResult result = Finish(WaveJoin(mine, a.exp2Scale), a.scale);
    if (tid == 0) {
        WriteRow<T>(a, row, result);
    }
    if (a.topCount == 0) {
        return;
    }
    if (result.bad) {
        if (tid < a.topCount) {
            WriteTop(a, row, result, tid, 0);
        }
        return;
    }
    // The largest topCount-th key of any list bounds the result from below: what is less drops out.
    __shared__ uint64_t kept[kMaxSplit * kMaxTop];
    __shared__ uint32_t nKept;
    const uint64_t* keys = a.keys + row * a.nSplit * a.topCount;
    uint64_t bound = lane < a.nSplit ? LoadOne(keys + static_cast<uint64_t>(lane) * a.topCount + a.topCount - 1) : 0;
    for (int d = 32; d > 0; d >>= 1) {
        const uint64_t o = (static_cast<uint64_t>(__shfl_xor(static_cast<uint32_t>(bound >> 32), d)) << 32) |
                           __shfl_xor(static_cast<uint32_t>(bound), d);
        bound = o > bound ? o : bound;
    }
    if (tid == 0) {
        nKept = 0;
    }
    __syncthreads();
    for (uint32_t c = tid; c < a.nSplit * a.topCount; c += kThreads) {
        const uint64_t key = LoadOne(keys + c);
        if (key != 0 && key >= bound) {
            kept[atomicAdd(&nKept, 1u)] = key;
        }
    }
    __syncthreads();
    const uint32_t n = nKept;
    for (uint32_t c = tid; c < n; c += kThreads) {
        const uint64_t key = kept[c];
        uint32_t rank = 0;
        for (uint32_t o = 0; o < n; ++o) {
            rank += kept[o] > key ? 1 : 0;
        }
        if (rank < a.topCount) {
            WriteTop(a, row, result, rank, key);
        }
    }
}

template <typename T>
hipError_t Launch(const LogProbsArgs& a, uint32_t rows, hipStream_t stream)
{
    const dim3 grid(rows * a.nSplit);
    if (a.topCount != 0) {
        hipLaunchKernelGGL((LogProbsKernel<T, true>), grid, dim3(kThreads), 0, stream, a);
    } else {
        hipLaunchKernelGGL((LogProbsKernel<T, false>), grid, dim3(kThreads), 0, stream, a);
    }
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.nSplit > 1) {
        hipLaunchKernelGGL((LogProbsJoinKernel<T>), dim3(rows), dim3(kThreads), 0, stream, a);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace

// Few rows: as many workgroups per row as bring 1024 in all, each with at least 4096 elements.
uint32_t LogProbsSplit(uint64_t rows, uint64_t vocab)
{
    const uint64_t wanted = rows == 0 ? 1 : (1024 + rows - 1) / rows;
    uint64_t split = vocab / 4096;
    split = split < wanted ? split : wanted;
    split = split < kMaxSplit ? split : kMaxSplit;
    return split < 1 ? 1 : static_cast<uint32_t>(split);
}

hipError_t LaunchLogProbs(const LogProbsArgs& a, HcclDataType dtype, uint32_t rows, hipStream_t stream)
{
    switch (dtype) {
        case HCCL_DATA_TYPE_FP32: return Launch<F32>(a, rows, stream);
        case HCCL_DATA_TYPE_BFP16: return Launch<B16>(a, rows, stream);
        default: return Launch<F16>(a, rows, stream);
    }
}

}  // namespace model_ops
}  // namespace hccl_amd
