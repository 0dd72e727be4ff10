// Log probabilities of given tokens, entropy and top alternatives of rows of logits whose vocabulary lies in up to 64
// parts (one per rank).
//
// One pass over a row keeps, per lane, the largest logit m, s = sum exp2(y) and t = sum y exp2(y) with y = c (x - m),
// c = scale * log2 e.  Whenever m grows, both are carried over: d = c (m - m'), s' = s 2^d, t' = 2^d (t + s d).  Then
//   lse = scale m + ln s, log p = scale (x - m) - ln s, entropy = ln s - ln 2 t / s.
// The difference is formed before it is scaled: the largest logit's y is exactly 0, so that s near 1 does not feel the size of
// the logits, and rows of the type's lowest value (a mask) come out like any other row of equal logits.  (c x - m' in one
// multiply-add saves an instruction per element, not measurably any time, and loses both.)  s is 64 bits wide: eight terms
// are added in 32 bits in three roundings, everything else in 64, and ln s takes the digits that 32 bits lack.  What ln s
// near 0 can be off by are thus the three roundings next to the 1, 3 x 2^-24, at any row length: of a likely token's log p at
// most 2 x 2^-24 was seen, 2.7e-6 of it at -0.05, 1e-4 at -0.001, 1e-3 at -0.0001, for rows of 1000 to 131072 entries
// (torch's 32-bit sums: 3 to 120 x 2^-24).  With s in 32 bits throughout it was seven times as much at 32768 entries
// and a log p of -0.05 to -0.02, and 0.5 % less time.
//
// Alternatives without a second pass over the row: a histogram of the lane maxima, by their distance from the largest,
// yields a bound that topCount lanes reach, and so topCount elements.  Every lane also leaves the largest of each group of
// vectors it loads together in LDS (16 bits of its order), and only groups that reach the bound are read again: four
// vectors for each of the topCount and a few more, instead of the row, which no cache holds any longer.  What reaches the
// bound is ranked by (logit, lower index).  Where too many reach it (equal logits, as in a row that a mask leaves few entries
// of), the exact topCount-th lane maximum takes its place: what lies above is in fewer than topCount lanes, and the rest are
// the first entries equal to it.
//
// Bound: one read of the logits from HBM, closely followed by the vector ALU (about eight instructions and an exponential,
// which takes two slots, per element).  A workgroup owns one row; where there are few rows, nSplit workgroups share each and
// a second kernel joins their partial results.
#include "model_ops.h"
#include "vec.h"

namespace hccl_amd {
namespace model_ops {
namespace {

constexpr uint32_t kUnroll = 4;            // vectors a lane loads together
// Elements, and groups, that may reach the bound before the exact search takes over.
template <uint32_t kThreads>
constexpr uint32_t kCandidates = kThreads == kWave ? 256 : 512;
constexpr uint32_t kGroupBytes = 16384;    // LDS for the groups' maxima, at most
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

typedef LogProbsStats Stats;
constexpr Stats kNoElements = {kLowest, 0.0f, 0.0};      // (or -inf alone)

__device__ __forceinline__ void Rescale(Stats& a, float m, float c)
{
    const float d = fmaxf((a.m - m) * c, kFarBelow);
    const float f = Exp2(d);
    a.t = f * __builtin_fmaf(static_cast<float>(a.s), d, a.t);
    a.s = a.s * static_cast<double>(f);
    a.m = m;
}

// The same for a wavefront's sets together.
__device__ __forceinline__ Stats WaveJoin(Stats a, float c)
{
    Stats r;
    r.m = LaneMax(a.m);
    Rescale(a, r.m, c);
    r.s = WaveSum(a.s);
    r.t = WaveSum(a.t);
    return r;
}

// N more elements, of which the largest is returned.
template <uint32_t N>
__device__ __forceinline__ float Accumulate(Stats& a, const float* x, float c)
{
    float most = x[0];
    for (uint32_t i = 1; i < N; ++i) {
        most = fmaxf(most, x[i]);
    }
    if (most > a.m) {
        Rescale(a, most, c);
    }
    float e[N];
    for (uint32_t i = 0; i < N; ++i) {
        const float y = (x[i] - a.m) * c;
        e[i] = Exp2(y);
        a.t = __builtin_fmaf(fmaxf(y, kFarBelow), e[i], a.t);
    }
    for (uint32_t i = 0; i < N; i += 8) {
        a.s += static_cast<double>(((e[i] + e[i + 1]) + (e[i + 2] + e[i + 3])) + ((e[i + 4] + e[i + 5]) + (e[i + 6] + e[i + 7])));
    }
    return most;
}

// The vectors [first, last) of one part's row that this workgroup reads.  Those below `full` are whole; a shorter end of the
// row is vector `full`, read as the last whole vector's worth of the row with the places before its elements masked.
template <typename T>
struct Part {
    typedef typename T::Raw Raw;
    static constexpr uint32_t P = kPer16<T>;
    static constexpr uint32_t kNone = sizeof(Raw) == 4 ? 0xFF800000u : T::kHalf ? 0xFC00FC00u : 0xFF80FF80u;   // -inf
    const Raw* row;
    uint32_t count;
    uint32_t full;
    uint32_t first;
    uint32_t last;

    // `begin` is the number of vectors of the parts before it; the workgroup has the vectors [from, to) of them all.
    __device__ __forceinline__ Part(const LogProbsArgs& a, uint32_t shard, uint64_t r, uint32_t begin, uint32_t from, uint32_t to)
    {
        row = static_cast<const Raw*>(a.logits[shard]) + r * a.rowStride[shard];
        count = a.count[shard];
        full = count / P;
        const uint32_t end = begin + Vectors();
        first = (from > begin ? from : begin) - begin;
        last = (to < end ? to : end) - begin;
        if (to <= begin || from >= end) {
            first = last = 0;
        }
    }
    __device__ __forceinline__ Part(const Raw* data, uint32_t n, uint32_t f, uint32_t l)
        : row(data), count(n), full(n / P), first(f), last(l)
    {
    }
    __device__ __forceinline__ uint32_t Vectors() const { return (count + P - 1) / P; }
    // Places of vector v that hold an element of it, as bits.
    __device__ __forceinline__ uint32_t Valid(uint32_t v) const
    {
        const uint32_t all = (1u << P) - 1u, rest = count % P;
        return v < full ? all : count >= P ? all & ~(all >> rest) : (1u << rest) - 1u;
    }
    // Index in the part's row of the first place of vector v.
    __device__ __forceinline__ uint32_t Base(uint32_t v) const { return v < full ? v * P : count >= P ? count - P : 0u; }
    __device__ __forceinline__ U32x4 Load(uint32_t v) const
    {
        if (__builtin_expect(v < full, 1)) {
            return LoadOnce16(row + static_cast<uint64_t>(v) * P);
        }
        U32x4 raw = {kNone, kNone, kNone, kNone};
        const uint32_t valid = Valid(v);
        if (count >= P) {
            raw = LoadOnce16(row + (count - P));
        } else {
            for (uint32_t i = 0; i < P; ++i) {
                if (i < count) {
                    Put(raw, i, LoadOne(row + i));
                }
            }
        }
        for (uint32_t i = 0; i < P; ++i) {
            if (!((valid >> i) & 1u)) {
                Put(raw, i, static_cast<Raw>(kNone));
            }
        }
        return raw;
    }
    static __device__ __forceinline__ void Put(U32x4& raw, uint32_t i, Raw e)
    {
        if constexpr (sizeof(Raw) == 4) {
            raw[i] = e;
        } else {
            const uint32_t keep = raw[i / 2] & (0xFFFFu << (16 * ((i + 1) % 2)));
            raw[i / 2] = keep | (static_cast<uint32_t>(e) << (16 * (i % 2)));
        }
    }
};

// Hands out the workgroup's vectors, kUnroll per lane at a time.
template <typename T, uint32_t kThreads>
struct Reader {
    const LogProbsArgs& a;
    uint64_t row;
    uint32_t from, to;       // flat vectors of this workgroup
    uint32_t shard = 0;
    uint32_t begin = 0;      // vectors of the parts before `shard`
    uint32_t next = 0;       // next vector of the current part
    Part<T> part;
    bool any = false;        // the lane has had an element

    __device__ __forceinline__ Reader(const LogProbsArgs& args, uint64_t r, uint32_t f, uint32_t t)
        : a(args), row(r), from(f), to(t), part(args, 0, r, 0, f, t)
    {
        next = part.first;
    }
    __device__ __forceinline__ bool Fetch(U32x4* raw)
    {
        while (next >= part.last) {
            begin += part.Vectors();
            if (++shard >= a.nShards || begin >= to) {
                return false;
            }
            part = Part<T>(a, shard, row, begin, from, to);
            next = part.first;
        }
        const uint32_t v = next + threadIdx.x;
        if (next + kThreads * kUnroll <= (part.last < part.full ? part.last : part.full)) {
            for (uint32_t u = 0; u < kUnroll; ++u) {
                raw[u] = LoadOnce16(part.row + static_cast<uint64_t>(v + u * kThreads) * Part<T>::P);
            }
            any = true;
        } else {
            for (uint32_t u = 0; u < kUnroll; ++u) {
                raw[u] = U32x4{Part<T>::kNone, Part<T>::kNone, Part<T>::kNone, Part<T>::kNone};
                if (v + u * kThreads < part.last) {
                    raw[u] = part.Load(v + u * kThreads);
                    any = true;
                }
            }
        }
        next += kThreads * kUnroll;
        return true;
    }
};

// How many of the n keys are larger; eight at a time, so that their reads do not wait for each other.
__device__ __forceinline__ uint32_t RankOf(uint64_t key, const uint64_t* keys, uint32_t n)
{
    uint32_t rank = 0, o = 0;
    for (; o + 8 <= n; o += 8) {
        uint64_t k[8];
        for (uint32_t i = 0; i < 8; ++i) {
            k[i] = keys[o + i];
        }
        for (uint32_t i = 0; i < 8; ++i) {
            rank += k[i] > key ? 1 : 0;
        }
    }
    for (; o < n; ++o) {
        rank += keys[o] > key ? 1 : 0;
    }
    return rank;
}

constexpr uint32_t kBins = 256;
template <uint32_t kThreads>
struct TopSpace {
    uint32_t bin[kBins];
    uint32_t group[kCandidates<kThreads>];       // groups that reach the bound: slot << 16 | lane
    uint64_t candidate[kCandidates<kThreads>];
    uint64_t top[kMaxTop];
    uint32_t waveCount[kThreads / kWave];
    uint32_t nGroups;
    uint32_t nCandidates;
};

// Sum over the workgroup; every thread gets it.
template <uint32_t kThreads>
__device__ __forceinline__ uint32_t BlockCount(uint32_t v, TopSpace<kThreads>& sh, uint32_t tid)
{
    v = WaveSum(v);
    __syncthreads();
    if ((tid & (kWave - 1)) == 0) {
        sh.waveCount[tid / kWave] = v;
    }
    __syncthreads();
    uint32_t sum = 0;
    for (uint32_t w = 0; w < kThreads / kWave; ++w) {
        sum += sh.waveCount[w];
    }
    return sum;
}

template <uint32_t kThreads>
__device__ __forceinline__ uint32_t BlockMax(uint32_t v, TopSpace<kThreads>& sh, uint32_t tid)
{
    v = LaneMax(v);
    __syncthreads();
    if ((tid & (kWave - 1)) == 0) {
        sh.waveCount[tid / kWave] = v;
    }
    __syncthreads();
    uint32_t most = 0;
    for (uint32_t w = 0; w < kThreads / kWave; ++w) {
        most = sh.waveCount[w] > most ? sh.waveCount[w] : most;
    }
    return most;
}

// Elements of the workgroup's part of the row whose order is at least `bound`.
template <typename T, uint32_t kThreads>
__device__ __forceinline__ uint32_t CountFrom(const LogProbsArgs& a, uint64_t row, uint32_t from, uint32_t to, uint32_t bound,
                                              TopSpace<kThreads>& sh, uint32_t tid)
{
    uint32_t n = 0, begin = 0;
    for (uint32_t shard = 0; shard < a.nShards; ++shard) {
        const Part<T> part(a, shard, row, begin, from, to);
        for (uint32_t v = part.first + tid; v < part.last; v += kThreads) {
            float x[kPer16<T>];
            Unpack16<T>(part.Load(v), x);
            const uint32_t valid = part.Valid(v);
            for (uint32_t i = 0; i < kPer16<T>; ++i) {
                n += ((valid >> i) & 1u) != 0 && Ordered(x[i]) >= bound ? 1 : 0;
            }
        }
        begin += part.Vectors();
    }
    return BlockCount(n, sh, tid);
}

// Appends the first `want` elements of the workgroup's part of the row whose order is `value`, in ascending order.
template <typename T, uint32_t kThreads>
__device__ __forceinline__ void FirstEqual(const LogProbsArgs& a, uint64_t row, uint32_t from, uint32_t to, uint32_t value,
                                           uint32_t want, TopSpace<kThreads>& sh, uint32_t tid)
{
    uint32_t start = 0, begin = 0;
    for (uint32_t shard = 0; shard < a.nShards && want != 0; ++shard) {
        const Part<T> part(a, shard, row, begin, from, to);
        for (uint32_t v0 = part.first; v0 < part.last && want != 0; v0 += kThreads) {
            const uint32_t v = v0 + tid;
            uint32_t equal = 0;     // bit i: place i equals `value`
            if (v < part.last) {
                float x[kPer16<T>];
                Unpack16<T>(part.Load(v), x);
                for (uint32_t i = 0; i < kPer16<T>; ++i) {
                    equal |= Ordered(x[i]) == value ? 1u << i : 0u;
                }
                equal &= part.Valid(v);
            }
            // position of the lane's first one among those of all lanes
            const uint32_t mine = __popc(equal), upTo = WaveScan(mine);
            __syncthreads();
            if ((tid & (kWave - 1)) == kWave - 1) {
                sh.waveCount[tid / kWave] = upTo;
            }
            __syncthreads();
            uint32_t before = upTo - mine, total = 0;
            for (uint32_t w = 0; w < kThreads / kWave; ++w) {
                before += w < tid / kWave ? sh.waveCount[w] : 0;
                total += sh.waveCount[w];
            }
            for (uint32_t i = 0; i < kPer16<T>; ++i) {
                if ((equal >> i) & 1u) {
                    if (before < want) {
                        sh.candidate[atomicAdd(&sh.nCandidates, 1u)] = Key(value, start + part.Base(v) + i);
                    }
                    ++before;
                }
            }
            want -= total < want ? total : want;
        }
        start += part.count;
        begin += part.Vectors();
    }
    __syncthreads();
}

// The search that needs no list, for rows in which a few lanes hold more large elements than the list takes: the
// topCount-th largest logit by bisection, then everything above it.  Returns it; some thirty passes over the row.
template <typename T, uint32_t kThreads>
__device__ __forceinline__ uint32_t SearchTop(const LogProbsArgs& a, uint64_t row, uint32_t from, uint32_t to, uint32_t low,
                                              uint32_t high, TopSpace<kThreads>& sh, uint32_t tid)
{
    // at least topCount elements reach `low`, none lies above `high`
    while (low < high) {       // the largest value that topCount elements reach
        const uint32_t mid = low + (high - low + 1) / 2;
        if (CountFrom<T>(a, row, from, to, mid, sh, tid) >= a.topCount) {
            low = mid;
        } else {
            high = mid - 1;
        }
    }
    __syncthreads();
    if (tid == 0) {
        sh.nCandidates = 0;
    }
    __syncthreads();
    uint32_t start = 0, begin = 0;
    for (uint32_t shard = 0; shard < a.nShards; ++shard) {
        const Part<T> part(a, shard, row, begin, from, to);
        for (uint32_t v = part.first + tid; v < part.last; v += kThreads) {
            float x[kPer16<T>];
            Unpack16<T>(part.Load(v), x);
            const uint32_t valid = part.Valid(v);
            for (uint32_t i = 0; i < kPer16<T>; ++i) {
                const uint32_t o = Ordered(x[i]);
                if (((valid >> i) & 1u) != 0 && o > low) {
                    sh.candidate[atomicAdd(&sh.nCandidates, 1u)] = Key(o, start + part.Base(v) + i);
                }
            }
        }
        start += part.count;
        begin += part.Vectors();
    }
    __syncthreads();
    return low;
}

// A value that `want` lanes reach, or 0 if there are fewer lanes with an element: the lower edge of the first bin of the
// histogram, counted from the largest value on, up to which `want` lane maxima fall; `reaching` counts them and `upper` is
// the bin's upper edge, where the want-th of them lies at most.  Bins are
// 2^shift orders wide, first as fine as bfloat16, and wider where the first 255 do not reach far enough.  Every wavefront
// reads the histogram for itself.
template <uint32_t kThreads>
__device__ __forceinline__ uint32_t TopBound(uint32_t laneMost, uint32_t largest, uint32_t want, uint32_t& reaching,
                                             uint32_t& upper, TopSpace<kThreads>& sh, uint32_t tid)
{
    const uint32_t lane = tid & (kWave - 1);
    for (uint32_t shift = 16;; shift += 4) {
        const uint32_t far = (largest - laneMost) >> shift;
        if (laneMost != 0) {
            atomicAdd(&sh.bin[far < kBins - 1 ? far : kBins - 1], 1u);
        }
        __syncthreads();
        uint32_t n[4], sum = 0;
        for (uint32_t i = 0; i < 4; ++i) {
            n[i] = sh.bin[4 * lane + i];
            sum += n[i];
        }
        const uint32_t upTo = WaveScan(sum);
        const uint64_t reached = __ballot(upTo >= want);
        if (reached == 0) {
            reaching = __builtin_amdgcn_readlane(upTo, kWave - 1);
            upper = largest;
            return 0;
        }
        const uint32_t at = __ffsll(static_cast<unsigned long long>(reached)) - 1;
        uint32_t bin = 4 * at;
        reaching = __builtin_amdgcn_readlane(upTo - sum, at);
        for (uint32_t i = 0; i < 4 && reaching < want; ++i) {
            reaching += __builtin_amdgcn_readlane(n[i], at);
            bin += reaching < want ? 1 : 0;
        }
        if (__builtin_expect(bin < kBins - 1 || shift >= 24, 1)) {
            // the bin holds orders in (largest - ((bin + 1) << shift), largest - (bin << shift)]
            const uint64_t depth = ((static_cast<uint64_t>(bin) + 1) << shift) - 1;
            upper = largest - (bin << shift);
            return depth < largest ? largest - static_cast<uint32_t>(depth) : 1u;
        }
        __syncthreads();
        for (uint32_t i = tid; i < kBins; i += kThreads) {
            sh.bin[i] = 0;
        }
        __syncthreads();
    }
}

// Lists the groups of this lane that reach `bound`, reads them again and lists their elements that do.  False if there are
// more of either than a list takes.
template <typename T, uint32_t kThreads>
__device__ __forceinline__ bool ListElements(const LogProbsArgs& a, uint64_t row, uint32_t from, uint32_t to, uint32_t laneMost,
                                             uint32_t bound, uint32_t nSlots, const uint16_t* groupMost, TopSpace<kThreads>& sh,
                                             uint32_t tid)
{
    constexpr uint32_t P = kPer16<T>;
    if (laneMost != 0 && laneMost >= bound) {
        for (uint32_t slot = 0; slot < nSlots; ++slot) {
            if (groupMost[slot * kThreads + tid] >= bound >> 16) {
                const uint32_t at = atomicAdd(&sh.nGroups, 1u);
                if (at < kCandidates<kThreads>) {
                    sh.group[at] = slot << 16 | tid;
                }
            }
        }
    }
    __syncthreads();
    // A slot is 2^slotShift fetches of kUnroll vectors of the lane; one thread per vector.
    const uint32_t nGroups = sh.nGroups;
    if (nGroups > kCandidates<kThreads>) {
        return false;
    }
    const float least = bound <= Ordered(-__builtin_inff()) ? -__builtin_inff() : FromOrdered(bound);
    const uint32_t shift = a.slotShift;
    for (uint32_t item = tid; item < (nGroups * kUnroll) << shift; item += kThreads) {
        const uint32_t group = sh.group[(item / kUnroll) >> shift];
        const uint32_t fetch = ((group >> 16) << shift) + (item / kUnroll & ((1u << shift) - 1u));
        uint32_t begin = 0, start = 0, before = 0;
        uint32_t v = 0, last = 0, count = 0, index = 0;
        const typename T::Raw* data = nullptr;
        for (uint32_t shard = 0; shard < a.nShards && begin < to; ++shard) {
            const Part<T> part(a, shard, row, begin, from, to);
            const uint32_t per = (part.last - part.first + kThreads * kUnroll - 1) / (kThreads * kUnroll);
            if (fetch - before < per) {       // (below `before` the difference wraps and is not)
                data = part.row;
                v = part.first + ((fetch - before) * kUnroll + item % kUnroll) * kThreads + (group & 0xFFFFu);
                last = part.last;
                count = part.count;
                index = start;
            }
            before += per;
            start += part.count;
            begin += part.Vectors();
        }
        if (v < last) {
            const Part<T> part(data, count, 0, last);
            float x[P];
            Unpack16<T>(part.Load(v), x);
            const uint32_t valid = part.Valid(v);
            index += part.Base(v);
            for (uint32_t e = 0; e < P; ++e) {
                if (x[e] >= least && ((valid >> e) & 1u) != 0) {
                    const uint32_t c = atomicAdd(&sh.nCandidates, 1u);
                    if (c < kCandidates<kThreads>) {
                        sh.candidate[c] = Key(Ordered(x[e]), index + e);
                    }
                }
            }
        }
    }
    __syncthreads();
    return sh.nCandidates <= kCandidates<kThreads>;
}

// Leaves the topCount largest keys of the workgroup's part of the row in sh.top, descending, 0 where there is none.
// laneMost: order of the lane's largest logit, 0 if it had no element; largest: of the workgroup's.  sh.bin, sh.top and the
// counters are zero.
template <typename T, uint32_t kThreads>
__device__ __forceinline__ void GatherTop(const LogProbsArgs& a, uint64_t row, uint32_t from, uint32_t to, uint32_t laneMost,
                                          uint32_t largest, uint32_t nSlots, const uint16_t* groupMost, TopSpace<kThreads>& sh,
                                          uint32_t tid)
{
    uint32_t reaching, upper;
    const uint32_t bound = TopBound<kThreads>(laneMost, largest, a.topCount, reaching, upper, sh, tid);
    // (with fewer lanes than topCount, or a list that a few lanes more than fill, there is nothing to be gained from trying)
    const bool few = reaching <= kCandidates<kThreads> / 4 &&
                     ListElements<T, kThreads>(a, row, from, to, laneMost, bound, nSlots, groupMost, sh, tid);
    if (__builtin_expect(!few, 0)) {
        // The exact topCount-th lane maximum: mostly the largest of its bin, else by bisection.
        uint32_t low = bound;
        if (reaching >= a.topCount) {
            uint32_t high = BlockMax<kThreads>(laneMost <= upper ? laneMost : 0u, sh, tid);
            bool first = true;
            while (low < high) {
                const uint32_t mid = first ? high : low + (high - low + 1) / 2;
                first = false;
                if (BlockCount<kThreads>(laneMost >= mid ? 1 : 0, sh, tid) >= a.topCount) {
                    low = mid;
                } else {
                    high = mid - 1;
                }
            }
        }
        __syncthreads();
        if (tid == 0) {
            sh.nGroups = 0;
            sh.nCandidates = 0;
        }
        __syncthreads();
        if (!ListElements<T, kThreads>(a, row, from, to, laneMost, low + 1, nSlots, groupMost, sh, tid)) {
            low = SearchTop<T, kThreads>(a, row, from, to, low, largest, sh, tid);
        }
        const uint32_t n = sh.nCandidates;
        if (n < a.topCount) {
            FirstEqual<T, kThreads>(a, row, from, to, low, a.topCount - n, sh, tid);
        }
    }
    const uint32_t n = sh.nCandidates;
    for (uint32_t c = tid; c < n; c += kThreads) {
        const uint64_t key = sh.candidate[c];
        const uint32_t rank = RankOf(key, sh.candidate, n);
        if (rank < a.topCount) {
            sh.top[rank] = key;
        }
    }
    __syncthreads();
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
    const float s = static_cast<float>(a.s);
    r.none = s == 0.0f;
    r.bad = s != s;
    r.logSum = logf(s) + static_cast<float>(a.s - static_cast<double>(s)) / s;      // ln s to all 32 bits also next to s = 1
    r.lse = r.none ? -__builtin_inff() : __builtin_fmaf(a.m, scale, r.logSum);
    r.entropy = r.none ? 0.0f : r.logSum - kLn2 * (a.t / s);
    return r;
}

__device__ __forceinline__ float LogProbOf(const RowResult& r, float x, float scale)
{
    return r.none ? -__builtin_inff() : __builtin_fmaf(x - r.m, scale, -r.logSum);
}

// The given token of a row and its logit, fetched before the reductions that the result waits for.
struct Token {
    int64_t id;
    float logit;
};
template <typename T>
__device__ __forceinline__ float TokenLogit(const LogProbsArgs& a, uint64_t row, int64_t token)
{
    if (token < 0 || token >= a.vocab) {
        return 0.0f;
    }
    uint32_t at = static_cast<uint32_t>(token);
    uint32_t shard = 0;
    while (at >= a.count[shard]) {
        at -= a.count[shard];
        ++shard;
    }
    return Widen<T>(LoadOne(static_cast<const typename T::Raw*>(a.logits[shard]) + row * a.rowStride[shard] + at));
}
__device__ __forceinline__ int64_t TokenId(const LogProbsArgs& a, uint64_t row)
{
    return a.tokens == nullptr ? -1
           : a.wideTokens      ? LoadOne(static_cast<const int64_t*>(a.tokens) + row)
                               : LoadOne(static_cast<const int32_t*>(a.tokens) + row);
}

// Every rank's outputs, a wavefront per rank.
template <uint32_t kThreads>
__device__ __forceinline__ void WriteRow(const LogProbsArgs& a, uint64_t row, const RowResult& r, Token token, const uint64_t* top)
{
    const uint32_t lane = threadIdx.x & (kWave - 1);
    float value = 0.0f;
    int64_t id = -1;
    if (lane < a.topCount) {
        value = __builtin_nanf("");
        if (!r.bad) {
            const uint64_t key = top[lane];
            value = LogProbOf(r, FromOrdered(static_cast<uint32_t>(key >> 32)), a.scale);
            id = static_cast<int64_t>(0xFFFFFFFFu - static_cast<uint32_t>(key));
        }
    }
    const float logProb = token.id >= a.vocab ? __builtin_nanf("") : token.id >= 0 ? LogProbOf(r, token.logit, a.scale) : 0.0f;
    for (uint32_t o = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave); o < a.nOut; o += kThreads / kWave) {
        const LogProbsArgs::Out& out = a.out[o];
        if (lane == 0) {
            if (out.logProbs != nullptr) {
                StoreOne(out.logProbs + row, logProb);
            }
            if (out.logSumExp != nullptr) {
                StoreOne(out.logSumExp + row, r.lse);
            }
            if (out.entropy != nullptr) {
                StoreOne(out.entropy + row, r.entropy);
            }
        }
        if (lane < a.topCount) {
            const uint64_t at = row * a.topCount + lane;
            if (out.topValues != nullptr) {
                StoreOne(out.topValues + at, value);
            }
            if (out.topIds != nullptr) {
                if (a.wideTokens) {
                    StoreOne(static_cast<int64_t*>(out.topIds) + at, id);
                } else {
                    StoreOne(static_cast<int32_t*>(out.topIds) + at, static_cast<int32_t>(id));
                }
            }
        }
    }
}

template <typename T, uint32_t kThreads, bool kTop>
__global__ __launch_bounds__(kThreads, kThreads > 256 ? 4 : kTop ? 7 : 8) void LogProbsKernel(const LogProbsArgs a)
{
    constexpr uint32_t P = kPer16<T>, kWaves = kThreads / kWave;
    __shared__ Stats waveStats[kWaves];
    __shared__ TopSpace<kTop ? kThreads : kWave> sh;
    extern __shared__ uint16_t groupMost[];      // [slot][lane]: order, cut to 16 bits, of the largest of 2^slotShift fetches
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1);
    const uint32_t split = blockIdx.x % a.nSplit;
    const uint64_t row = blockIdx.x / a.nSplit;
    const uint32_t from = static_cast<uint32_t>(static_cast<uint64_t>(a.vectors) * split / a.nSplit);
    const uint32_t to = static_cast<uint32_t>(static_cast<uint64_t>(a.vectors) * (split + 1) / a.nSplit);
    Token token = {a.nSplit == 1 ? TokenId(a, row) : -1, 0.0f};
    if constexpr (kTop) {
        for (uint32_t i = tid; i < kBins; i += kThreads) {
            sh.bin[i] = 0;
        }
        if (tid < kMaxTop) {
            sh.top[tid] = 0;
        }
        if (tid == 0) {
            sh.nGroups = 0;
            sh.nCandidates = 0;
        }
    }
    Stats acc = kNoElements;
    Reader<T, kThreads> reader(a, row, from, to);
    U32x4 raw[kUnroll];
    uint32_t fetch = 0, slotMost = 0;
    while (reader.Fetch(raw)) {
        float x[kUnroll * P];
        for (uint32_t u = 0; u < kUnroll; ++u) {
            Unpack16<T>(raw[u], x + u * P);
        }
        if (fetch == 0) {
            token.logit = TokenLogit<T>(a, row, token.id);      // on its way while the row is read
        }
        const float most = Accumulate<kUnroll * P>(acc, x, a.exp2Scale);
        if constexpr (kTop) {
            const uint32_t order = Ordered(most) >> 16;
            slotMost = (fetch & ((1u << a.slotShift) - 1u)) != 0 && slotMost > order ? slotMost : order;
            groupMost[(fetch >> a.slotShift) * kThreads + tid] = static_cast<uint16_t>(slotMost);
        }
        ++fetch;
    }
    const Stats wave = WaveJoin(acc, a.exp2Scale);
    if (lane == 0) {
        waveStats[tid / kWave] = wave;
    }
    __syncthreads();
    const Stats all = WaveJoin(lane < kWaves ? waveStats[lane] : kNoElements, a.exp2Scale);
    const RowResult result = Finish(all, a.scale);
    if constexpr (kTop) {
        if (!result.bad) {     // a NaN has no place in an order: no alternatives
            // (a lane, or a workgroup, that has met nothing but -inf still has the lowest finite value as its largest)
            const float laneMost = acc.s == 0.0 ? -__builtin_inff() : acc.m, most = result.none ? -__builtin_inff() : all.m;
            const uint32_t nSlots = (fetch + (1u << a.slotShift) - 1) >> a.slotShift;
            GatherTop<T>(a, row, from, to, reader.any ? Ordered(laneMost) : 0u, Ordered(most), nSlots, groupMost, sh, tid);
        }
    }
    if (a.nSplit == 1) {
        WriteRow<kThreads>(a, row, result, token, sh.top);
        return;
    }
    const uint64_t at = row * a.nSplit + split;
    if (tid == 0) {
        StoreOne(reinterpret_cast<U32x4*>(a.stats + at), __builtin_bit_cast(U32x4, all));
    }
    if constexpr (kTop) {
        if (tid < a.topCount) {
            StoreOne(a.keys + at * a.topCount + tid, result.bad ? 0 : sh.top[tid]);
        }
    }
}

// Joins the nSplit partial results of a row.
constexpr uint32_t kJoinThreads = 256;
constexpr uint32_t kMaxSplit = 32;
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void LogProbsJoinKernel(const LogProbsArgs a)
{
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1);
    const uint64_t row = blockIdx.x;
    Token token = {TokenId(a, row), 0.0f};
    // every wavefront joins the numbers for itself, a lane per split
    Stats mine = kNoElements;
    const uint64_t* keys = a.keys + row * a.nSplit * a.topCount;
    uint64_t last = 0;      // the lowest key of the lane's list
    if (lane < a.nSplit) {
        mine = __builtin_bit_cast(Stats, LoadOne(reinterpret_cast<const U32x4*>(a.stats + row * a.nSplit + lane)));
        last = a.topCount != 0 ? LoadOne(keys + static_cast<uint64_t>(lane) * a.topCount + a.topCount - 1) : 0;
    }
    token.logit = TokenLogit<T>(a, row, token.id);
    const RowResult result = Finish(WaveJoin(mine, a.exp2Scale), a.scale);
    __shared__ uint64_t top[kMaxTop];
    if (a.topCount != 0 && !result.bad) {
        // The largest topCount-th key of any list bounds the result from below: what is less drops out.
        __shared__ uint64_t kept[kMaxSplit * kMaxTop];
        __shared__ uint32_t nKept;
        for (int d = 32; d > 0; d >>= 1) {
            const uint64_t o = (static_cast<uint64_t>(__shfl_xor(static_cast<uint32_t>(last >> 32), d)) << 32) |
                               __shfl_xor(static_cast<uint32_t>(last), d);
            last = o > last ? o : last;
        }
        if (tid == 0) {
            nKept = 0;
        }
        __syncthreads();
        for (uint32_t c = tid; c < a.nSplit * a.topCount; c += kJoinThreads) {
            const uint64_t key = LoadOne(keys + c);
            if (key != 0 && key >= last) {
                kept[atomicAdd(&nKept, 1u)] = key;
            }
        }
        __syncthreads();
        const uint32_t n = nKept;
        for (uint32_t c = tid; c < n; c += kJoinThreads) {
            const uint64_t key = kept[c];
            const uint32_t rank = RankOf(key, kept, n);
            if (rank < a.topCount) {
                top[rank] = key;
            }
        }
        __syncthreads();
    }
    WriteRow<kJoinThreads>(a, row, result, token, top);
}

template <typename T, uint32_t kThreads>
void LaunchRows(LogProbsArgs& a, uint32_t rows, hipStream_t stream)
{
    const dim3 grid(rows * a.nSplit);
    if (a.topCount == 0) {
        hipLaunchKernelGGL((LogProbsKernel<T, kThreads, false>), grid, dim3(kThreads), 0, stream, a);
        return;
    }
    // Fetches of a workgroup: a short one at the end of every part, and no more than all parts' whole rows take.
    constexpr uint32_t kFetch = kThreads * kUnroll;
    uint32_t fetches = 0;
    for (uint32_t s = 0; s < a.nShards; ++s) {
        fetches += ((a.count[s] + kPer16<T> - 1) / kPer16<T> + kFetch - 1) / kFetch;
    }
    const uint32_t share = (a.vectors / a.nSplit + 1 + kFetch - 1) / kFetch + a.nShards;
    fetches = fetches < share ? fetches : share;
    a.slotShift = 0;
    while (((fetches - 1) >> a.slotShift) + 1 > kGroupBytes / (kThreads * sizeof(uint16_t))) {
        ++a.slotShift;
    }
    const uint32_t lds = (((fetches - 1) >> a.slotShift) + 1) * kThreads * sizeof(uint16_t);
    hipLaunchKernelGGL((LogProbsKernel<T, kThreads, true>), grid, dim3(kThreads), lds, stream, a);
}

template <typename T>
hipError_t Launch(LogProbsArgs& a, uint32_t rows, hipStream_t stream)
{
    switch (LogProbsFormOf(rows, a.vectors).threads) {
        case 64: LaunchRows<T, 64>(a, rows, stream); break;
        case 256: LaunchRows<T, 256>(a, rows, stream); break;
        default: LaunchRows<T, 1024>(a, rows, stream); break;
    }
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.nSplit > 1) {
        hipLaunchKernelGGL((LogProbsJoinKernel<T>), dim3(rows), dim3(kJoinThreads), 0, stream, a);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace

// Measured on MI355X with bf16 rows, no alternatives / eight alternatives, in us (V = 8 vectors):
//   rows x V        wave / row      256 / row       1024 / row      256, row split in
//   4096 x 1000      7.5 / 11.7     18.6 / 25.8     62.9 / 124
//   4096 x 16000    29.4 / 34.3     33.6 / 38.5     64.9 / 144
//   4096 x 65536    92.4 / 99.5     90.5 / 97.8      106 / 180
//   1024 x 4000      7.0 / 10.1      7.6 / 11.2     18.5 / 34.0
//   1024 x 8000      9.5 / 12.9      8.6 / 12.1     18.9 / 36.7
//    512 x 131072   71.8 / 82.7     27.2 / 31.9     29.3 / 38.2     29.7 / 34.9 (2)
//    256 x 32768    19.8 / 25.4      8.8 / 12.2      8.2 / 11.9      9.7 / 14.3 (2)
//    256 x 131072   69.7 / 80.7     23.0 / 27.5     16.6 / 20.4     18.5 / 23.4 (4)
//    255 x 131072                   22.7 / 27.4     16.6 / 20.4     18.1 / 23.5 (4)
//    192 x 131072                   22.4 / 27.1     15.3 / 19.4     15.3 / 20.6 (4)
//    129 x 131072                   21.7 / 26.4     14.5 / 18.7     14.2 / 19.5 (4)
//    129 x 32768                     8.2 / 11.7      7.1 / 10.8      8.4 / 13.2 (4)
//    192 x 16000                     6.9 / 9.8       7.5 / 11.2      8.6 / 12.7 (2)
//    128 x 131072   68.4 / 80.0     21.8 / 26.6     14.5 / 18.6     12.6 / 17.7 (4)
//     64 x 16000    10.4 / 14.1      6.2 / 8.9       7.0 / 10.3      7.1 / 11.5 (4)
//     64 x 65536    35.4 / 42.5     12.4 / 16.4      9.0 / 13.0      8.2 / 12.7 (8)
//     64 x 131072   67.6 / 78.7     21.4 / 25.9     14.0 / 18.3      9.7 / 14.6 (8)
//     16 x 65536    29.2 / 34.2     11.2 / 14.1      8.7 / 12.2      6.7 / 11.0 (8)
//      1 x 131072   46.0 / 55.6     14.3 / 18.4     12.0 / 15.7      6.1 / 10.6 (16)
// With fp32 rows, whose vectors hold half as many:
//   4096 x 16000    45.6 / 51.2     44.8 / 50.2     58.9 / 127      56.6 / 66.4 (2)
//   1024 x 8000     11.9 / 15.5     10.4 / 13.6     16.2 / 32.3     14.5 / 20.6 (2)
//    512 x 50001    46.1 / 53.7     19.8 / 23.8     21.8 / 31.1     23.9 / 28.6 (2)
//    256 x 50001    44.4 / 51.6     16.6 / 20.8     13.6 / 17.1     15.6 / 20.4 (4)
//    160 x 50001    43.8 / 51.3     15.9 / 19.9     10.8 / 14.2     12.5 / 17.3 (4)
//     64 x 65536    52.7 / 61.8     17.4 / 21.9      9.9 / 13.4      8.9 / 13.4 (8)
//     16 x 65536    43.8 / 51.0     15.3 / 19.3      9.3 / 12.7      7.4 / 11.5 (8)
//      1 x 131072   77.6 / 85.4     25.2 / 29.1     13.6 / 17.0      6.1 / 10.4 (16)
// fp16 rows take as long as bf16 in every form, or up to 7 % longer.
// (Loading the next vectors before the present ones are summed: 4096 x 131072 175 against 174, 4096 x 16000 39 against 34,
// 512 x 131072 25 against 27, with alternatives slower everywhere.  128 threads a row: 3 to 10 % faster than
// the form taken for 2048 x 32000 and 16384 x 32000, up to 10 % slower for 4096 x 65536.)
// A split row costs a second kernel of about 3 us, a workgroup of 1024 threads has a CU to itself.
LogProbsForm LogProbsFormOf(uint64_t rows, uint64_t vectors)
{
    if (2 * vectors <= rows) {
        return {64, 1};
    }
    if (rows > 256 || vectors <= 2048) {
        return {256, 1};
    }
    if (rows <= 128 && vectors > (rows <= 32 ? 4096 : 8192)) {
        const uint64_t most = vectors < 65536 ? 16 : 32, wanted = 512 / rows;
        return {256, static_cast<uint32_t>(wanted < most ? wanted : most)};
    }
    return {1024, 1};
}

hipError_t LaunchLogProbs(LogProbsArgs& a, HcclDataType dtype, uint32_t rows, hipStream_t stream)
{
    switch (dtype) {
        case HCCL_DATA_TYPE_FP32: return Launch<F32>(a, rows, stream);
        case HCCL_DATA_TYPE_BFP16: return Launch<B16>(a, rows, stream);
        default: return Launch<F16>(a, rows, stream);
    }
}

}  // namespace model_ops
}  // namespace hccl_amd
