// sample_kernels.hip -- the next token of each row of fp32 logits from a given
// random number: temperature, top-k, top-p and min-p.
//
// With m the highest logit, token v weighs w(v) = e^((x(v) - m) / T).  Weights
// are whole numbers, w 2^S rounded to nearest, formed in 64-bit floating point,
// so that every sum of them is exact and the same in any order: the token that
// a row draws follows from the row alone.  S = 46, or as much less as keeps the
// sum of a larger vocabulary within 64 bits.
//
// The kept tokens are a run of the order "falling logit, lower token first
// among equals": all up to a last one, whose key (the logit's bits as an
// ordered whole number) and token bound the set.  Block = row, which passes
// over the row's logits, from the caches after the first time:
//   1. the highest logit (and the lowest, which sets the bins);
//   2. where top-k or top-p cut: counts and weights of 1024 bins of the logits,
//      the bin that the cut falls into, its tokens sorted in LDS (bins of more
//      tokens than LDS takes are cut into 1024 again, by their keys);
//   3. the kept tokens' weights, summed by ranges of the vocabulary, the range
//      that the random number falls into, and the token in it.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "attention_common.h"
#include "device_common.h"
#include "runtime_internal.h"

namespace kimkv {
namespace {

constexpr unsigned kBlock = 1024;
constexpr uint32_t kWaves = kBlock / kWave;
constexpr uint32_t kRow = 4 * kBlock;        // tokens of one vector of each thread
constexpr uint32_t kBins = 1024;
constexpr uint32_t kSorted = 2048;           // tokens that are sorted in LDS
constexpr uint32_t kRanges = 32;
constexpr uint32_t kMostTokens = 1u << 20;
constexpr uint32_t kMostRows = kMostTokens / kRow + 1;   // vectors of a thread
constexpr uint32_t kPerRange = (kMostRows + kRanges - 1) / kRanges;

typedef float f32x4_t __attribute__((ext_vector_type(4)));

// ---- whole-number sums over a wave -------------------------------------------

template <int kControl, int kRows>
__device__ inline uint64_t dpp_u64(uint64_t v)
{
    auto const lo = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(static_cast<uint32_t>(v)), kControl, kRows, 0xF, false));
    auto const hi = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(static_cast<uint32_t>(v >> 32)), kControl, kRows, 0xF, false));
    return static_cast<uint64_t>(hi) << 32 | lo;
}

// Each lane's sum of its own and all lower lanes' values.
__device__ inline uint64_t wave_scan(uint64_t v)
{
    v += dpp_u64<0x111, 0xF>(v);   // rows of 16 shifted by 1, 2, 4, 8
    v += dpp_u64<0x112, 0xF>(v);
    v += dpp_u64<0x114, 0xF>(v);
    v += dpp_u64<0x118, 0xF>(v);
    v += dpp_u64<0x142, 0xA>(v);   // the last lane of rows 0 and 2 to rows 1 and 3
    v += dpp_u64<0x143, 0xC>(v);   // lane 31 to rows 2 and 3
    return v;
}

__device__ inline uint64_t lane_u64(uint64_t v, int lane)
{
    auto const lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(v)), lane));
    auto const hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(v >> 32)), lane));
    return static_cast<uint64_t>(hi) << 32 | lo;
}

__device__ inline uint64_t wave_total(uint64_t v) { return lane_u64(wave_scan(v), 63); }

// floor(a b) of a float a in [0, 1] and a whole number, exactly; with `up` the
// least whole number that is not below a b.
__device__ inline uint64_t part_of(float a, uint64_t b, bool up)
{
    uint32_t const bits = __float_as_uint(a);
    uint32_t const e = bits >> 23;
    uint64_t const mantissa = (bits & 0x7FFFFFu) | (e != 0 ? 0x800000u : 0u);
    uint32_t const shift = 150 - (e != 0 ? e : 1);   // a = mantissa 2^-shift, shift 23 .. 149
    uint64_t const high = __umul64hi(mantissa, b);
    uint64_t const low = mantissa * b;
    uint64_t whole;
    bool rest;
    if (shift >= 128) {
        whole = 0;
        rest = (high | low) != 0;
    } else if (shift >= 64) {
        uint32_t const s = shift - 64;
        whole = high >> s;
        rest = low != 0 || (s != 0 && (high << (64 - s)) != 0);
    } else {
        whole = high << (64 - shift) | low >> shift;
        rest = (low << (64 - shift)) != 0;
    }
    return whole + (up && rest ? 1 : 0);
}

// ---- keys and weights --------------------------------------------------------

// An ordered whole number of a logit that is not NaN; 0 is below all of them.
__device__ inline uint32_t key_of(float x)
{
    uint32_t const b = __float_as_uint(x);
    return (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
}
__device__ inline float logit_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) != 0 ? key & 0x7FFFFFFFu : ~key); }

struct Weights {
    double highest;
    double rate;       // log2(e) / T
    uint32_t scale;    // S

    // 2^t of t = (x - m) rate by the exponential's series on [-1/2, 1/2] ln 2: 13
    // terms leave 2^-52 of it.
    __device__ uint64_t of(float x) const
    {
        double const t = (static_cast<double>(x) - highest) * rate;
        if (!(t > -64.0)) return 0;
        double const n = rint(t);
        double const y = (t - n) * 0.6931471805599453;
        double s = 1.0 / 479001600.0;
        s = fma(s, y, 1.0 / 39916800.0);
        s = fma(s, y, 1.0 / 3628800.0);
        s = fma(s, y, 1.0 / 362880.0);
        s = fma(s, y, 1.0 / 40320.0);
        s = fma(s, y, 1.0 / 5040.0);
        s = fma(s, y, 1.0 / 720.0);
        s = fma(s, y, 1.0 / 120.0);
        s = fma(s, y, 1.0 / 24.0);
        s = fma(s, y, 1.0 / 6.0);
        s = fma(s, y, 0.5);
        s = fma(s, y, 1.0);
        s = fma(s, y, 1.0);
        // The sum with 2^52 rounds to whole numbers, which are its low bits.
        double const w = ldexp(s, static_cast<int>(n) + static_cast<int>(scale)) + 4503599627370496.0;
        return static_cast<uint64_t>(__double_as_longlong(w)) & 0xFFFFFFFFFFFFFull;
    }
};

struct SampleLds {
    uint32_t count[kBins];
    uint64_t mass[kBins];
    uint64_t sorted[kSorted];        // key, then ~token, so that falling numbers are the order
    uint64_t range[kRanges * kWaves];
    uint64_t row[kPerRange * kWaves];
    uint64_t wave[kWaves];
    uint64_t found;
    float wave_f[2][kWaves];
    uint32_t word[4];
};

// The row as the block reads it: vector j of thread t is tokens
// 4 (j kBlock + t) - shift + 0 .. 3, at a 16-byte address.
struct Row {
    const float* from;
    uint32_t V;
    uint32_t shift;
    uint32_t vectors;
    bool infinite;       // the highest logit is +inf

    __device__ uint32_t token(uint32_t j) const { return 4 * (j * kBlock + threadIdx.x) - shift; }

    // Tokens past the row, and NaN, are -inf.
    __device__ f32x4_t load(uint32_t j) const
    {
        uint32_t const v = token(j);
        f32x4_t x;
        if (v < V && V - v > 3) {
            x = *reinterpret_cast<const f32x4_t*>(from + v);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) x[i] = v + i < V ? from[v + i] : -INFINITY;
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) x[i] = x[i] != x[i] ? -INFINITY : x[i] + 0.0f;   // no -0
        return x;
    }

    // With logits of +inf, these alone are there, all alike.
    __device__ float value(float x) const { return infinite ? (x == INFINITY ? 0.0f : -INFINITY) : x; }

    // f(token, logit) for every token of this thread that can be drawn.
    template <typename F>
    __device__ void each(F f) const
    {
        for (uint32_t j = 0; j < vectors; ++j) {
            f32x4_t const y = load(j);
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                float const x = value(y[i]);
                if (x != -INFINITY) f(token(j) + i, x);
            }
        }
    }
};

// Sum over the block, in every thread.
__device__ inline uint64_t block_total(uint64_t v, SampleLds& lds)
{
    uint64_t const total = wave_total(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) lds.wave[threadIdx.x / kWave] = total;
    __syncthreads();
    uint64_t sum = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) sum += lds.wave[w];
    return sum;
}

// Sum of the lower threads' values, and of all in *total.
__device__ inline uint64_t block_scan(uint64_t v, SampleLds& lds, uint64_t* total)
{
    uint64_t const upto = wave_scan(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == kWave - 1) lds.wave[threadIdx.x / kWave] = upto;
    __syncthreads();
    uint64_t before = 0, sum = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
        if (w < threadIdx.x / kWave) before += lds.wave[w];
        sum += lds.wave[w];
    }
    *total = sum;
    return before + upto - v;
}

// The ranges' sums of weight(token, logit), and all of them.
template <typename F>
__device__ uint64_t sum_ranges(const Row& row, SampleLds& lds, uint32_t per, F weight)
{
    uint32_t const wave = threadIdx.x / kWave;
    uint32_t const lane = threadIdx.x & (kWave - 1);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kRanges * kWaves; i += kBlock) lds.range[i] = 0;
    __syncthreads();
    uint64_t all = 0, sum = 0;
    uint32_t at = 0;
    auto const flush = [&] {
        if (__ballot(sum != 0) != 0) {
            uint64_t const total = wave_total(sum);
            if (lane == 0) lds.range[at * kWaves + wave] = total;
            all += total;
        }
        sum = 0;
        ++at;
    };
    for (uint32_t j = 0; j < row.vectors; ++j) {
        f32x4_t const y = row.load(j);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            float const x = row.value(y[i]);
            if (x != -INFINITY) sum += weight(row.token(j) + i, x);
        }
        if ((j + 1) % per == 0 || j + 1 == row.vectors) flush();
    }
    if (lane == 0) lds.wave[wave] = all;
    __syncthreads();
    uint64_t total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) total += lds.wave[w];
    return total;
}

// Of sums by (part, wave), in order: the part that the target falls into, and
// what lies before it.  Every thread reads them.
__device__ inline uint32_t part_at(const uint64_t* sums, uint32_t parts, uint64_t target, uint64_t* before)
{
    uint64_t sum = 0;
    for (uint32_t p = 0; p < parts; ++p) {
        uint64_t part = 0;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) part += sums[p * kWaves + w];
        if (target < sum + part) {
            *before = sum;
            return p;
        }
        sum += part;
    }
    *before = sum;
    return parts;   // only for a target that is no part of the sum
}

// The first token at which the running sum exceeds `target`, less than all of
// it; the ranges' sums are in place.  Its weight in *its.
template <typename F>
__device__ uint32_t token_at(const Row& row, SampleLds& lds, uint32_t per, uint64_t target, F weight, uint64_t* its)
{
    uint32_t const wave = threadIdx.x / kWave;
    uint32_t const lane = threadIdx.x & (kWave - 1);
    uint64_t before;
    uint32_t const range = part_at(lds.range, kRanges, target, &before);
    uint32_t const j0 = range * per;
    uint32_t const j1 = min(j0 + per, row.vectors);
    for (uint32_t j = j0; j < j1; ++j) {
        f32x4_t const y = row.load(j);
        uint64_t sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            float const x = row.value(y[i]);
            if (x != -INFINITY) sum += weight(row.token(j) + i, x);
        }
        uint64_t const total = __ballot(sum != 0) != 0 ? wave_total(sum) : 0;
        if (lane == 0) lds.row[(j - j0) * kWaves + wave] = total;
    }
    __syncthreads();
    uint64_t rows_before;
    uint32_t const j = j0 + part_at(lds.row, j1 > j0 ? j1 - j0 : 0, target - before, &rows_before);
    if (j < j1) {
        uint64_t at = before + rows_before;
        for (uint32_t w = 0; w < wave; ++w) at += lds.row[(j - j0) * kWaves + w];
        uint64_t const mine = lds.row[(j - j0) * kWaves + wave];
        if (target >= at && target - at < mine) {   // this wave's
            f32x4_t const y = row.load(j);
            uint64_t w4[4];
            uint64_t sum = 0;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                float const x = row.value(y[i]);
                w4[i] = x != -INFINITY ? weight(row.token(j) + i, x) : 0;
                sum += w4[i];
            }
            at += wave_scan(sum) - sum;
            if (target >= at && target - at < sum) {   // this thread's
                bool found = false;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    if (!found && target - at < w4[i]) {
                        found = true;
                        lds.word[0] = row.token(j) + i;
                        lds.found = w4[i];
                    }
                    if (!found) at += w4[i];
                }
            }
        }
    }
    __syncthreads();
    *its = lds.found;
    return lds.word[0];
}

// The last kept token: its key and its number.  Kept are the higher keys, and
// of its own the tokens up to it.
struct Last {
    uint32_t key;
    uint32_t token;
    __device__ bool keeps(uint32_t k, uint32_t t) const { return k > key || (k == key && t <= token); }
};

// What a cut looks for: the `amount`-th token (from 1) of the order, or the
// first at which the weight reaches `amount`.
struct Cut {
    bool by_mass;
    uint64_t amount;
};

struct Bins {
    float highest;
    float rate;      // bins for a unit of the logit
    bool bounded;    // the last bin holds tokens of weight 0 and of any logit
    __device__ uint32_t of(float x) const { return static_cast<uint32_t>(fminf((highest - x) * rate, static_cast<float>(kBins - 1))); }
};

// The bin of the counted ones that the cut falls into, what lies in the bins
// before it, and how many tokens it holds.
struct Place {
    uint32_t bin;
    uint32_t count;
    uint64_t before_count;
    uint64_t before_mass;
};

__device__ inline Place place_of(SampleLds& lds, const Cut& cut, uint64_t before_count, uint64_t before_mass)
{
    static_assert(kBins == kBlock, "a thread a bin");
    uint32_t const tid = threadIdx.x;
    uint64_t all_count, all_mass;
    uint64_t const count = lds.count[tid];
    uint64_t const mass = lds.mass[tid];
    uint64_t const counts = before_count + block_scan(count, lds, &all_count);
    uint64_t const masses = before_mass + block_scan(mass, lds, &all_mass);
    uint64_t const at = cut.by_mass ? masses : counts;
    uint64_t const mine = cut.by_mass ? mass : count;
    __syncthreads();
    if (tid == 0) lds.word[0] = kBins;
    __syncthreads();
    if (at < cut.amount && cut.amount - at <= mine) {   // one thread at most
        lds.word[0] = tid;
        lds.word[1] = static_cast<uint32_t>(count);
        lds.range[0] = counts;
        lds.range[1] = masses;
    }
    __syncthreads();
    Place const p{lds.word[0], lds.word[1], lds.range[0], lds.range[1]};
    __syncthreads();
    return p;
}

// Sorts lds.sorted[0, n) into falling order; n at most kSorted.
__device__ inline void sort_falling(SampleLds& lds, uint32_t n)
{
    uint32_t size = 2;
    while (size < n) size *= 2;
    for (uint32_t i = n + threadIdx.x; i < size; i += kBlock) lds.sorted[i] = 0;
    for (uint32_t k = 2; k <= size; k *= 2) {
        for (uint32_t j = k / 2; j > 0; j /= 2) {
            __syncthreads();
            for (uint32_t p = threadIdx.x; p < size / 2; p += kBlock) {
                uint32_t const i = 2 * p - (p & (j - 1));
                uint64_t const a = lds.sorted[i];
                uint64_t const b = lds.sorted[i + j];
                if ((a < b) == ((i & k) == 0)) {
                    lds.sorted[i] = b;
                    lds.sorted[i + j] = a;
                }
            }
        }
    }
    __syncthreads();
}

// Where the cut falls, and the weight up to and with its token in *upto.  Bins'
// counts (and weights, where `weigh`) are in lds.
__device__ Last find_cut(const Row& row, SampleLds& lds, const Weights& weights, const Bins& bins, const Cut& cut, bool weigh,
                         uint32_t per, uint64_t* upto)
{
    uint32_t const tid = threadIdx.x;
    Last const everything{0, 0xFFFFFFFFu};
    Place place = place_of(lds, cut, 0, 0);
    *upto = 0;
    // Past the last token, or among tokens that weigh nothing.
    if (place.bin == kBins || (bins.bounded && place.bin == kBins - 1)) return everything;
    // The bin's tokens, and their highest and lowest keys.
    uint32_t const bin = place.bin;
    if (tid < 3) lds.word[tid] = tid == 2 ? 0xFFFFFFFFu : 0;
    __syncthreads();
    row.each([&](uint32_t token, float x) {
        if (bins.of(x) != bin) return;
        uint32_t const key = key_of(x);
        if (place.count <= kSorted) {
            lds.sorted[atomicAdd(&lds.word[0], 1u)] = static_cast<uint64_t>(key) << 32 | (0xFFFFFFFFu - token);
        } else {
            atomicMax(&lds.word[1], key);
            atomicMin(&lds.word[2], key);
        }
    });
    __syncthreads();
    uint32_t high = lds.word[1];
    uint32_t low = lds.word[2];
    while (place.count > kSorted && high != low) {
        // The keys low .. high, cut into bins of 2^shift keys.
        uint32_t shift = 0;
        while (((high - low) >> shift) >= kBins) ++shift;
        __syncthreads();
        lds.count[tid] = 0;
        lds.mass[tid] = 0;
        __syncthreads();
        row.each([&](uint32_t, float x) {
            uint32_t const key = key_of(x);
            if (key < low || key > high) return;
            uint32_t const b = (high - key) >> shift;
            atomicAdd(&lds.count[b], 1u);
            if (weigh) atomicAdd(reinterpret_cast<unsigned long long*>(&lds.mass[b]), static_cast<unsigned long long>(weights.of(x)));
        });
        __syncthreads();
        place = place_of(lds, cut, place.before_count, place.before_mass);
        high -= place.bin << shift;
        uint32_t const keys = 1u << shift;
        low = high - low >= keys ? high - keys + 1 : low;
        if (place.count > kSorted) continue;
        if (tid == 0) lds.word[0] = 0;
        __syncthreads();
        row.each([&](uint32_t token, float x) {
            uint32_t const key = key_of(x);
            if (key >= low && key <= high) lds.sorted[atomicAdd(&lds.word[0], 1u)] = static_cast<uint64_t>(key) << 32 | (0xFFFFFFFFu - token);
        });
        __syncthreads();
    }
    uint64_t const left = cut.amount - (cut.by_mass ? place.before_mass : place.before_count);   // at least 1
    if (place.count > kSorted) {
        // One key: so many of its tokens, the lowest first.
        uint64_t const weight = weights.of(logit_of(high));
        uint64_t const tokens = cut.by_mass ? (left + weight - 1) / weight : left;
        auto const same = [&](uint32_t, float x) { return key_of(x) == high ? uint64_t{1} : uint64_t{0}; };
        static_cast<void>(sum_ranges(row, lds, per, same));
        uint64_t one;
        uint32_t const token = token_at(row, lds, per, tokens - 1, same, &one);
        *upto = place.before_mass + tokens * weight;
        return Last{high, token};
    }
    sort_falling(lds, place.count);
    // Two neighbours of the order a thread.
    uint64_t w[2];
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        uint32_t const n = 2 * tid + i;
        w[i] = n < place.count && weigh ? weights.of(logit_of(static_cast<uint32_t>(lds.sorted[n] >> 32))) : 0;
    }
    uint64_t total = 0;
    uint64_t at = weigh ? block_scan(w[0] + w[1], lds, &total) : 0;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        uint32_t const n = 2 * tid + i;
        bool const here = n < place.count && (cut.by_mass ? at < left && left - at <= w[i] : n + 1 == left);
        at += w[i];
        if (here) {
            lds.word[0] = static_cast<uint32_t>(lds.sorted[n] >> 32);
            lds.word[1] = 0xFFFFFFFFu - static_cast<uint32_t>(lds.sorted[n]);
            lds.found = at;
        }
    }
    __syncthreads();
    *upto = place.before_mass + lds.found;
    Last const last{lds.word[0], lds.word[1]};
    __syncthreads();
    return last;
}

struct SampleArgs {
    const float* logits;
    const kimkv_sample_rule* rules;
    const float* uniforms;
    uint32_t* tokens;
    float* probabilities;
    uint32_t V;
    uint32_t scale;    // S
};

__global__ __launch_bounds__(kBlock) void sample_kernel(SampleArgs a)
{
    __shared__ SampleLds lds;
    uint32_t const tid = threadIdx.x;
    uint32_t const lane = tid & (kWave - 1);
    Row row;
    row.from = a.logits + static_cast<uint64_t>(blockIdx.x) * a.V;
    row.V = a.V;
    row.shift = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row.from) >> 2) & 3u;
    row.vectors = (a.V + row.shift + kRow - 1) / kRow;
    row.infinite = false;
    kimkv_sample_rule const rule = a.rules[blockIdx.x];
    float const uniform = a.uniforms[blockIdx.x];
    auto const answer = [&](uint32_t token, float probability) {
        if (tid != 0) return;
        a.tokens[blockIdx.x] = token;
        if (a.probabilities != nullptr) a.probabilities[blockIdx.x] = probability;
    };
    if (!(rule.temperature >= 0.0f && rule.temperature < INFINITY) || !(rule.top_p > 0.0f && rule.top_p <= 1.0f)
        || !(rule.min_p >= 0.0f && rule.min_p <= 1.0f) || !(uniform >= 0.0f && uniform < 1.0f)) {
        answer(KIMKV_NO_TOKEN, 0.0f);
        return;
    }

    // ---- the highest logit, and the lowest that is not -inf ----
    float high = -INFINITY;
    float low = INFINITY;
    for (uint32_t j = 0; j < row.vectors; ++j) {
        f32x4_t const y = row.load(j);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            high = fmaxf(high, y[i]);
            low = fminf(low, y[i] == -INFINITY ? INFINITY : y[i]);
        }
    }
    high = wave_max(high);
    low = -wave_max(-low);
    if (lane == 0) {
        lds.wave_f[0][tid / kWave] = high;
        lds.wave_f[1][tid / kWave] = low;
    }
    lds.count[tid] = 0;
    lds.mass[tid] = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
        high = fmaxf(high, lds.wave_f[0][w]);
        low = fminf(low, lds.wave_f[1][w]);
    }
    if (high == -INFINITY) {
        answer(KIMKV_NO_TOKEN, 0.0f);
        return;
    }
    row.infinite = high == INFINITY;
    if (row.infinite) high = low = 0.0f;

    bool const greedy = rule.temperature == 0.0f;
    uint32_t const top_k = greedy ? 1 : rule.top_k == 0 || rule.top_k >= a.V ? a.V : rule.top_k;
    bool const cut_k = top_k < a.V;
    bool const cut_p = !greedy && rule.top_p < 1.0f;
    Weights const weights{high, greedy ? 1.0 : 1.4426950408889634 / static_cast<double>(rule.temperature), a.scale};
    // Ranges of `per` vectors.
    uint32_t const per = (row.vectors + kRanges - 1) / kRanges;
    Last last{0, 0xFFFFFFFFu};
    if (cut_k || cut_p) {
        // Tokens 64 T or more below the highest weigh nothing, whatever their order.
        float const span = high - low;
        float const most = greedy ? INFINITY : 64.0f * rule.temperature;
        bool const bounded = span > most;
        Bins const bins{high, span == 0.0f || most == 0.0f ? 0.0f : static_cast<float>(kBins - 1) / fminf(span, most), bounded};
        row.each([&](uint32_t, float x) {
            uint32_t const b = bins.of(x);
            atomicAdd(&lds.count[b], 1u);
            if (cut_p) {
                uint64_t const w = weights.of(x);
                if (w != 0) atomicAdd(reinterpret_cast<unsigned long long*>(&lds.mass[b]), static_cast<unsigned long long>(w));
            }
        });
        __syncthreads();
        uint32_t const count = lds.count[tid];
        uint64_t const mass = lds.mass[tid];
        uint64_t total = 0;
        if (cut_p) total = block_total(mass, lds);
        if (cut_k) {
            uint64_t upto;
            last = find_cut(row, lds, weights, bins, Cut{false, top_k}, cut_p, per, &upto);
            if (last.key != 0) total = upto;
        }
        if (cut_p) {
            __syncthreads();
            lds.count[tid] = count;
            lds.mass[tid] = mass;
            __syncthreads();
            uint64_t upto;
            Last const mine = find_cut(row, lds, weights, bins, Cut{true, part_of(rule.top_p, total, true)}, true, per, &upto);
            if (mine.key > last.key || (mine.key == last.key && mine.token < last.token)) last = mine;
        }
    }

    // ---- the draw ----
    uint64_t const least = part_of(rule.min_p, uint64_t{1} << a.scale, true);
    auto const kept = [&](uint32_t token, float x) -> uint64_t {
        if (!last.keeps(key_of(x), token)) return 0;
        uint64_t const w = weights.of(x);
        return w >= least ? w : 0;
    };
    uint64_t const total = sum_ranges(row, lds, per, kept);
    uint64_t its;
    uint32_t const token = token_at(row, lds, per, part_of(uniform, total, false), kept, &its);
    answer(token, static_cast<float>(static_cast<double>(its) / static_cast<double>(total)));
}

}  // namespace
}  // namespace kimkv

using namespace kimkv;

extern "C" {

size_t kimkv_sample_workspace_bytes(uint32_t, uint32_t) { return 0; }

kimkv_status kimkv_model_sample(const float* logits, uint32_t rows, uint32_t vocabulary, const kimkv_sample_rule* device_rules,
                                const float* device_uniforms, uint32_t* device_tokens, float* probabilities, void*,
                                kimkv_stream_t stream)
{
    if (logits == nullptr || vocabulary == 0 || vocabulary > kMostTokens || device_rules == nullptr || device_uniforms == nullptr
        || device_tokens == nullptr) {
        return KIMKV_INVALID_ARGUMENT;
    }
    uint32_t scale = 63;   // sums of 2^scale for each token stay within 2^63
    while (scale > 0 && (uint64_t{1} << (63 - scale)) < vocabulary) --scale;
    scale = scale > 46 ? 46 : scale;
    SampleArgs a{logits, device_rules, device_uniforms, device_tokens, probabilities, vocabulary, scale};
    constexpr uint32_t kMost = 0x3FFFFFu;   // rows of a launch: fewer than 2^32 threads
    for (uint32_t first = 0; first < rows;) {
        uint32_t const n = rows - first < kMost ? rows - first : kMost;
        sample_kernel<<<n, kBlock, 0, native(stream)>>>(a);
        kimkv_status const status = launch_status();
        if (status != KIMKV_OK) return status;
        first += n;
        a.logits += static_cast<uint64_t>(n) * vocabulary;
        a.rules += n;
        a.uniforms += n;
        a.tokens += n;
        a.probabilities += a.probabilities != nullptr ? n : 0;
    }
    return KIMKV_OK;
}

}  // extern "C"
