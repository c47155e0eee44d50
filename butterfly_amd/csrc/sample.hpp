// A token for each row of logits, from one random number in [0, 1): with w_i = exp((z_i - max z) / temperature), of the top_k
// largest logits (ties: the lowest indexes) the likeliest ones until their sum reaches top_p of it, of those the ones with
// w_i >= min_p; the token is the first index whose cumulated w, in the order of indexes, exceeds uniform * total.
//
// A workgroup takes a row and keeps it in registers (up to 256 KiB, of the largest 56 to 128 bytes a lane in scratch memory; longer
// rows are read again, out of the caches).  There is no
// sort: what is kept is "logit above t, and the first m of those equal to t", and t is found by histograms of 2048 bins, first
// over the values from the maximum down, then, within the bin where the sum crosses its goal: float by comparing its few entries with
// each other (some 64 of 2^17: one pass less), bfloat16, or many, over the logits' bits.
//
// Weights are whole numbers, w in units of 2^-44: sums do not depend on their order (so the histograms may be filled by
// atomics, and every call gives the same token).  They are off by 2^-37 of themselves: a float exponential would move each border
// between two tokens by some 1e-8 of the total, which with 50000 entries of similar weight is 1e-3 of the distance between two
// borders; these move it by 1e-7 of that.
//
// Measured: 256 rows of 2^17 bfloat16 with top_p 102 us (67 MB: 14 us at a copy's rate), 64 rows of 30001 floats with top_p 34,
// one row of 32768 floats with top_k, top_p and min_p 30.  The large one is bound by the vector unit, busy for 87% of the cycles:
// some 30 operations for each weight, formed for each entry and twice (histogram, sum); the small ones by the chain of
// passes, barriers and scans within a workgroup.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "vec8.hpp"

namespace bf {

struct SampleArgs {
    const void *logits;
    const float *uniform, *temperature, *top_p, *min_p;   // one a row; settings NULL: the ones below for all rows
    const int64_t *top_k;
    double temperature_all, top_p_all, min_p_all;
    int64_t top_k_all;
    int64_t *token;
    int64_t stride;
    int vocab;
};

constexpr int kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64, kSampleBins = 2 * kSampleThreads;
constexpr int kSampleBits = 44, kSampleFine = 4096;
constexpr int kSampleFew = 512;   // entries of a bin that are compared with each other

struct SampleLds {
    unsigned long long powers[kSampleFine];   // 2^(k / 4096), in units of 2^-44
    unsigned long long bins[kSampleBins];
    unsigned long long sums[kSampleWaves];
    float low[kSampleWaves], high[kSampleWaves];
    unsigned long long counts[kSampleWaves];
    unsigned long long above;
    float few[kSampleFew], threshold;
    float lowest;   // no entry below it has a weight
    int at, number;
};

// Order of floats as an order of whole numbers (of bfloat16: 16 bits).
template <typename T>
__device__ __forceinline__ uint32_t sample_key(float v)
{
    const uint32_t bits = __builtin_bit_cast(uint32_t, v);
    const uint32_t key = bits ^ (bits >> 31 ? 0xffffffffu : 0x80000000u);
    return sizeof(T) == 2 ? key >> 16 : key;
}
template <typename T>
__device__ __forceinline__ float sample_value(uint32_t key)
{
    if (sizeof(T) == 2) key = key << 16 | (key >> 15 ? 0u : 0xffffu);
    return __builtin_bit_cast(float, key >> 31 ? key ^ 0x80000000u : ~key);
}

// 16 bytes of a row, NaN and what lies behind its end as -inf, -0 as 0.
template <typename T>
__device__ __forceinline__ uint4 sample_load(const T *row, int64_t col, int vocab)
{
    constexpr int E = 16 / sizeof(T);
    using Quad = std::conditional_t<sizeof(T) == 4, quad_at_4, quad_at_2>;
    uint32_t out[4];
    T part[E];
    if (col + E <= vocab) {
        const Quad v = *reinterpret_cast<const Quad *>(row + col);
        __builtin_memcpy(part, &v, 16);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) part[i] = col + i < vocab ? row[col + i] : (T)-INFINITY;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float f = to_float(part[i]);
        const uint32_t bits = __builtin_bit_cast(uint32_t, f == f ? f + 0.0f : -INFINITY);
        if constexpr (sizeof(T) == 4) out[i] = bits;
        else if (i % 2 == 0) out[i / 2] = bits >> 16;
        else out[i / 2] |= bits & 0xffff0000u;
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}
template <typename T>
__device__ __forceinline__ float sample_element(const uint4 &v, int i)
{
    const uint32_t words[4] = {v.x, v.y, v.z, v.w};
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, words[i]);
    else return __builtin_bit_cast(float, i % 2 ? words[i / 2] & 0xffff0000u : words[i / 2] << 16);
}

template <typename T>
struct SampleWeight {
    const unsigned long long *powers = nullptr;
    float top = 0.0f;
    float high = 0.0f, low = 0.0f;     // 4096 log2 e / temperature as two floats
    float range = 0.0f;                // farther below the maximum a weight is zero

    __device__ __forceinline__ bool reaches(float v) const { return top - v <= range; }

    // 2^44 exp((v - top) / temperature), rounded, of a v that it reaches: off by some 2^-37 of itself.  The exponent, of 2^(1 / 4096),
    // as two floats: a whole number of steps goes through the table, the rest, |x| <= 1/2, through 1 + s = 1 + x l + (x l)^2 / 2 with
    // l = log 2 / 4096 (e is 4096 s).  30 operations; a polynomial in 64-bit numbers took 50, many of them twice as long.
    __device__ __forceinline__ unsigned long long operator()(float v) const
    {
        const float d = top - v, z = d * high;
        float rest = fmaf(d, low, fmaf(d, high, -z));
        if constexpr (sizeof(T) == 4) {
            // (bfloat16: the difference is exact, or that of a number so small that it is exact enough)
            const float back = d - top;
            rest = fmaf((top - (d - back)) - (v + back), high, rest);
        }
        const float steps = rintf(z), s = ((z - steps) + rest) * -0.6931472f, e = fmaf(s * s, 0.5f / kSampleFine, s);
        const int m = -(int)steps;
        const uint64_t power = powers[m & (kSampleFine - 1)];
        // (a step's power times 4096 s: less than 2^32 in units of 2^-43)
        const uint64_t w = power + 2 * (int64_t)(int)((float)(uint32_t)(power >> 13) * e);
        const int down = -(m >> 12);
        return ((w << 1 >> down) + 1) >> 1;
    }
};

__device__ __forceinline__ unsigned long long sample_wave_sum(unsigned long long v)
{
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d, 64);
    return v;
}
__device__ __forceinline__ unsigned long long sample_wave_scan(unsigned long long v)
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const unsigned long long before = __shfl_up(v, d, 64);
        if (lane >= d) v += before;
    }
    return v;
}

// Sum over the threads in front of this one; total: over all.  (Ends behind a barrier of its own.)
__device__ __forceinline__ unsigned long long sample_before(SampleLds &lds, unsigned long long v, unsigned long long &total)
{
    const int wave = threadIdx.x >> 6;
    const unsigned long long inside = sample_wave_scan(v);
    if ((threadIdx.x & 63) == 63) lds.sums[wave] = inside;
    __syncthreads();
    unsigned long long before = 0;
    total = 0;
    for (int w = 0; w < kSampleWaves; ++w) {
        if (w == wave) before = total;
        total += lds.sums[w];
    }
    __syncthreads();
    return before + inside - v;
}

// The bin in which the sum from the first bin on reaches goal(sum of all bins); lds.above: the sum in front of it.  -1: it is never
// reached.
template <typename G>
__device__ __forceinline__ int sample_crossing(SampleLds &lds, G &&goal_of, unsigned long long &goal)
{
    if (threadIdx.x == 0) lds.at = -1;
    const unsigned long long one = lds.bins[2 * threadIdx.x], two = lds.bins[2 * threadIdx.x + 1];
    unsigned long long total;
    const unsigned long long before = sample_before(lds, one + two, total);
    goal = goal_of(total);
    if (before < goal && goal <= before + one + two) {
        const bool second = goal > before + one;
        lds.at = 2 * threadIdx.x + second;
        lds.above = second ? before + one : before;
    }
    __syncthreads();
    return lds.at;
}

// VECTORS: 16-byte pieces of the row that a thread holds; 0: the row is read again in each pass.
template <typename T, int VECTORS>
struct SampleRow {
    static constexpr int E = 16 / sizeof(T);
    const T *row;
    int vocab, span;             // span: pieces of a wavefront, side by side
    uint4 held[VECTORS > 0 ? VECTORS : 1];

    __device__ __forceinline__ int64_t piece(int n) const { return (int64_t)(threadIdx.x >> 6) * span + n * 64 + (threadIdx.x & 63); }

    __device__ __forceinline__ void init(const T *r, int v)
    {
        row = r;
        vocab = v;
        const int pieces = (vocab + E - 1) / E;
        span = VECTORS > 0 ? VECTORS * 64 : (pieces + 64 * kSampleWaves - 1) / (64 * kSampleWaves) * 64;
        if constexpr (VECTORS > 0) {
#pragma unroll
            for (int n = 0; n < VECTORS; ++n) held[n] = sample_load(row, piece(n) * E, vocab);
        }
    }
    // f(value, index) of every entry
    template <typename Fn>
    __device__ __forceinline__ void each(Fn &&f) const
    {
        if constexpr (VECTORS > 0) {
#pragma unroll
            for (int n = 0; n < VECTORS; ++n) {
                // (as something new to the compiler, which would otherwise keep what one pass has formed of every entry for the next)
                uint4 v = held[n];
                asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w));
                piece_of(v, (int)piece(n) * E, f);
            }
        } else {
            for (int n = 0; n < span / 64; ++n) {
                const int64_t at = piece(n);
                if (at * E >= vocab) break;
                piece_of(sample_load(row, at * E, vocab), (int)at * E, f);
            }
        }
    }
    template <typename Fn>
    __device__ __forceinline__ void piece_of(uint4 v, int at, Fn &&f) const
    {
#pragma unroll
        for (int i = 0; i < E; ++i) f(sample_element<T>(v, i), at + i);
    }
};

// The largest value t such that the weights of the logits from t up sum to goal(sum of all) at least; lds.above: the sum of those
// above t.  False: all of them do not.  Weights are those of logits above `floor`, and `ties` for all that are equal to it.
template <typename T, typename Row, typename G, typename W>
__device__ __forceinline__ bool sample_threshold(SampleLds &lds, const Row &row, const SampleWeight<T> &weight, float floor,
                                                 unsigned long long ties, G &&goal_of, W &&of, float &t)
{
    auto clear = [&] {
        lds.bins[2 * threadIdx.x] = lds.bins[2 * threadIdx.x + 1] = 0;
        __syncthreads();
    };
    const float per = weight.range > 0.0f ? kSampleBins / weight.range : 0.0f;
    auto bin_of = [&](float v) { return min((int)((weight.top - v) * per), kSampleBins - 1); };
    clear();
    row.each([&](float v, int) {
        if (weight.reaches(v) & (v > floor)) atomicAdd(&lds.bins[bin_of(v)], of(v));
    });
    if (threadIdx.x == 0 && ties) atomicAdd(&lds.bins[bin_of(floor)], ties);
    __syncthreads();
    unsigned long long goal;
    const int bin = sample_crossing(lds, goal_of, goal);
    if (bin < 0) return false;
    unsigned long long above = lds.above;
    // Few entries in the bin (a vocabulary of 2^17 makes some 64): each sums up those above it.  (The order in which they come
    // does not show in sums of whole numbers.)  bfloat16: a bin holds few distinct values, which the next round tells apart.
    if constexpr (sizeof(T) == 4) {
        if (threadIdx.x == 0) lds.number = 0;
        __syncthreads();
        row.each([&](float v, int) {
            if (weight.reaches(v) & (v > floor))
                if (bin_of(v) == bin) {
                    const int at = atomicAdd(&lds.number, 1);
                    if (at < kSampleFew) lds.few[at] = v;
                }
        });
        __syncthreads();
        const int number = lds.number;
        if (number <= kSampleFew) {
            if (threadIdx.x < number) lds.bins[threadIdx.x] = of(lds.few[threadIdx.x]);
            __syncthreads();
            const bool tied = ties && bin_of(floor) == bin;
            if (threadIdx.x < number + tied) {
                const float v = threadIdx.x < number ? lds.few[threadIdx.x] : floor;
                unsigned long long greater = above, equal = threadIdx.x < number ? 0 : ties;
                for (int j = 0; j < number; ++j) {
                    const float x = lds.few[j];
                    const unsigned long long w = lds.bins[j];
                    greater += x > v ? w : 0;
                    equal += x == v ? w : 0;
                }
                if (greater < goal && goal <= greater + equal) {
                    lds.threshold = v;
                    lds.above = greater;
                }
            }
            __syncthreads();
            t = lds.threshold;
            return true;
        }
    }
    // (bins are off by rounding: a hundredth more on both sides)
    const float width = per > 0.0f ? 1.0f / per : 0.0f;
    uint32_t high = sample_key<T>(fminf(weight.top, weight.top - (bin - 0.01f) * width));
    uint32_t low = bin == kSampleBins - 1 ? sample_key<T>(weight.top - weight.range * 1.001f) : sample_key<T>(weight.top - (bin + 1.01f) * width);
    for (;;) {
        const uint32_t length = high - low;
        const int shift = length < (uint32_t)kSampleBins ? 0 : 32 - __clz((int)length) - 11;
        const float least = sample_value<T>(low), most = sample_value<T>(high);
        __syncthreads();
        clear();
        row.each([&](float v, int) {
            if ((v >= least) & (v <= most) & (v > floor))
                if (weight.reaches(v) && bin_of(v) == bin) atomicAdd(&lds.bins[(high - sample_key<T>(v)) >> shift], of(v));
        });
        if (threadIdx.x == 0 && ties && floor >= least && floor <= most && bin_of(floor) == bin)
            atomicAdd(&lds.bins[(high - sample_key<T>(floor)) >> shift], ties);
        __syncthreads();
        unsigned long long rest;
        const int at = sample_crossing(lds, [&](unsigned long long) { return goal - above; }, rest);
        if (at < 0) return false;   // (cannot be: the bin held it)
        above += lds.above;
        high -= (uint32_t)at << shift;
        if (shift == 0) break;
        const uint32_t lowest = high - ((1u << shift) - 1);
        low = max(low, lowest > high ? 0u : lowest);
    }
    t = sample_value<T>(high);
    __syncthreads();
    if (threadIdx.x == 0) lds.above = above;
    __syncthreads();
    return true;
}

// The largest value whose weight is below `least`, of those from lds.lowest on; the value in front of that one where none is.
template <typename T>
__device__ __forceinline__ float sample_below(const SampleLds &lds, const SampleWeight<T> &weight, unsigned long long least)
{
    // keys low .. high - 1 are unknown, those from high on are not below; 1024 of them at a time
    uint32_t low = sample_key<T>(lds.lowest), high = sample_key<T>(weight.top);
    while (low < high) {
        const uint32_t step = (high - low) / kSampleThreads + 1, key = low + threadIdx.x * step;
        const bool below = key < high && key >= low && weight(sample_value<T>(key)) < least;
        const uint32_t count = (uint32_t)__syncthreads_count(below);
        high = min(high, low + count * step);
        low = count == 0 ? high : min(high, low + (count - 1) * step + 1);
    }
    // (there is no -0 among the entries, and it equals 0)
    const uint32_t key = high - 1, zero = sample_key<T>(0.0f);
    return sample_value<T>(key == zero - 1 ? key - 1 : key);
}

template <typename T, int VECTORS>
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(const SampleArgs a)
{
    __shared__ SampleLds lds;
    constexpr int E = 16 / sizeof(T);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t r = blockIdx.x;
    SampleRow<T, VECTORS> row;
    row.init(static_cast<const T *>(a.logits) + r * a.stride, a.vocab);

    float high = -INFINITY, low = INFINITY;
    row.each([&](float v, int) {
        high = fmaxf(high, v);
        low = fminf(low, v == -INFINITY ? INFINITY : v);
    });
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        high = fmaxf(high, __shfl_xor(high, d, 64));
        low = fminf(low, __shfl_xor(low, d, 64));
    }
    if (lane == 0) {
        lds.high[wave] = high;
        lds.low[wave] = low;
    }
    __syncthreads();
    for (int w = 0; w < kSampleWaves; ++w) {
        high = fmaxf(high, lds.high[w]);
        low = fminf(low, lds.low[w]);
    }
    if (high == -INFINITY) {
        // nothing is possible
        if (threadIdx.x == 0) a.token[r] = -1;
        return;
    }
    const double asked = a.temperature ? (double)a.temperature[r] : a.temperature_all;
    if (!(asked > 0.0)) {
        // the first of the largest
        int first = a.vocab;
        row.each([&](float v, int at) { if (v == high) first = min(first, at); });
#pragma unroll
        for (int d = 1; d < 64; d *= 2) first = min(first, __shfl_xor(first, d, 64));
        if (lane == 0) lds.counts[wave] = (unsigned long long)first;
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned long long least = lds.counts[0];
            for (int w = 1; w < kSampleWaves; ++w) least = min(least, lds.counts[w]);
            a.token[r] = (int64_t)least;
        }
        return;
    }
    // (between 2^-100 and 2^100: what is formed of it stays within the range of floats)
    const double temperature = fmin(fmax(asked, 0x1p-100), 0x1p100);
    const float far = (float)(temperature * ((kSampleBits + 2) * 0.6931471805599453));
    // (the lowest entry itself, where it is not too far: high - low is rounded, and high less that may lie above it)
    if (threadIdx.x == 0) lds.lowest = high - low <= far ? low : high - far;
    // the table: 2^(i / 64) 2^(j / 4096)
    if (threadIdx.x < 128) {
        const int i = threadIdx.x & 63;
        lds.bins[threadIdx.x] = __builtin_bit_cast(unsigned long long, exp2(threadIdx.x < 64 ? i / 64.0 : i / 4096.0));
    }
    __syncthreads();
    for (int k = threadIdx.x; k < kSampleFine; k += kSampleThreads) {
        const double coarse = __builtin_bit_cast(double, lds.bins[k >> 6]), fine = __builtin_bit_cast(double, lds.bins[64 + (k & 63)]);
        lds.powers[k] = (unsigned long long)(coarse * fine * (double)(1ull << kSampleBits) + 0.5);
    }
    __syncthreads();
    const bool infinite = high == INFINITY;
    SampleWeight<T> weight;
    weight.powers = lds.powers;
    weight.top = infinite ? 0.0f : high;
    const double per_nat = kSampleFine * 1.4426950408889634 / temperature;
    weight.high = (float)per_nat;
    weight.low = (float)(per_nat - (double)weight.high);
    weight.range = infinite ? -1.0f : fminf(high - low, far);
    const double min_p = a.min_p ? (double)a.min_p[r] : a.min_p_all;
    const double top_p = a.top_p ? (double)a.top_p[r] : a.top_p_all;
    const int64_t top_k = a.top_k ? a.top_k[r] : a.top_k_all;

    // kept: values above t, and the first m of those equal to it
    float t = -INFINITY;
    unsigned long long m = 0;
    if (infinite) {
        // those alone, all equally likely: the first ones
        unsigned long long mine = 0, all;
        row.each([&](float v, int) { mine += v == INFINITY; });
        sample_before(lds, mine, all);
        t = INFINITY;
        m = top_k > 0 ? min((unsigned long long)top_k, all) : all;
        if (top_p < 1.0) m = max(1ull, min(m, (unsigned long long)ceil(fmax(top_p, 0.0) * (double)m)));
    } else if (top_k > 0 && top_k < a.vocab &&
        sample_threshold<T>(lds, row, weight, t, 0, [&](unsigned long long) { return (unsigned long long)top_k; }, [](float) { return 1ull; }, t))
        m = (unsigned long long)top_k - lds.above;
    if (!infinite && top_p < 1.0) {
        unsigned long long goal = 0;
        auto goal_of = [&](unsigned long long total) {
            goal = max(1ull, min(total, (unsigned long long)ceil(fmax(top_p, 0.0) * (double)total)));
            return goal;
        };
        float tp;
        if (sample_threshold<T>(lds, row, weight, t, m > 0 ? m * weight(t) : 0, goal_of, [&](float v) { return weight(v); }, tp)) {
            const unsigned long long w = weight(tp);
            t = tp;
            m = (goal - lds.above + w - 1) / w;
        }
    }
    if (!infinite && min_p > 0.0) {
        const float unlikely = sample_below<T>(lds, weight, max(1ull, (unsigned long long)ceil(fmin(min_p, 1.0) * (double)(1ull << kSampleBits))));
        if (unlikely >= t) {
            t = unlikely;
            m = 0;
        }
    }
    const unsigned long long tie = infinite ? 1 : m > 0 ? weight(t) : 0;
    unsigned long long sum = 0, ties = 0;
    row.each([&](float v, int) {
        if (weight.reaches(v) & (v > t)) sum += weight(v);
        ties += v == t;
    });
    sum = sample_wave_sum(sum);
    ties = sample_wave_sum(ties);
    __syncthreads();
    if (lane == 0) {
        lds.sums[wave] = sum;
        lds.counts[wave] = ties;
    }
    __syncthreads();
    unsigned long long total = 0, ties_before = 0;
    for (int w = 0; w < kSampleWaves; ++w) {
        const unsigned long long left = m > ties_before ? m - ties_before : 0;
        total += lds.sums[w] + min(left, lds.counts[w]) * tie;
        ties_before += lds.counts[w];
    }
    const double u = fmin(fmax((double)a.uniform[r], 0.0), 1.0);
    unsigned long long target = min((unsigned long long)(u * (double)total), total - 1);
    // the wavefront's part of the row that holds it, read again by all threads in the order of indexes
    int where = 0;
    unsigned long long left = m;
    for (; where < kSampleWaves - 1; ++where) {
        const unsigned long long here = lds.sums[where] + min(left, lds.counts[where]) * tie;
        if (target < here) break;
        target -= here;
        left -= min(left, lds.counts[where]);
    }
    __syncthreads();
    for (int start = 0; start < row.span; start += kSampleThreads) {
        const int64_t piece = (int64_t)where * row.span + start + threadIdx.x;
        const bool mine = start + (int)threadIdx.x < row.span && piece * E < a.vocab;
        const uint4 v = mine ? sample_load(row.row, piece * E, a.vocab) : make_uint4(0, 0, 0, 0);
        unsigned long long mass = 0, equal = 0;
        if (mine) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float x = sample_element<T>(v, i);
                if (weight.reaches(x) & (x > t)) mass += weight(x);
                equal += x == t;
            }
        }
        unsigned long long all_equal, all;
        const unsigned long long equal_before = sample_before(lds, equal, all_equal);
        const unsigned long long allowed = left > equal_before ? min(left - equal_before, equal) : 0;
        const unsigned long long before = sample_before(lds, mass + allowed * tie, all);
        if (target < all) {
            if (before <= target && target < before + mass + allowed * tie) {
                unsigned long long rest = target - before, used = 0;
                for (int i = 0; i < E; ++i) {
                    const float x = sample_element<T>(v, i);
                    unsigned long long w = 0;
                    if (x > t) {
                        if (weight.reaches(x)) w = weight(x);
                    } else if (x == t && used < allowed) {
                        w = tie;
                        ++used;
                    }
                    if (rest < w) {
                        a.token[r] = piece * E + i;
                        break;
                    }
                    rest -= w;
                }
            }
            return;
        }
        target -= all;
        left -= min(left, all_equal);
    }
}

}  // namespace bf
