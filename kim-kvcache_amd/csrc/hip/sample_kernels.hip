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
// among equals".  Block = row, which passes over the row's logits, from the
// caches after the first time:
//   - The highest logit, and the maxima of 4096 parts of the row.
//   - Short list (top_k of at most 1024): the top_k-th highest of the maxima is
//     reached by at least top_k tokens, and by not many more: those are collected
//     in LDS and sorted, and the cuts and the draw go on there.
//   - Else, where top-k or top-p cut: counts and weights of 1024 bins of the
//     logits, the bin that the cut falls into, its tokens sorted in LDS (bins of
//     more tokens than LDS takes are cut into 1024 again, by their keys), which
//     gives the last kept token.
//   - The draw from a row: the kept tokens' weights summed by ranges of the
//     vocabulary, the range that the random number falls into, the token in it.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "attention_common.h"
#include "device_common.h"
#include "runtime_internal.h"

namespace kimkv {
namespace {

constexpr unsigned kBlock = 1024;
constexpr uint32_t kWaves = kBlock / kWave;
constexpr uint32_t kRow = 4 * kBlock;        // tokens of one vector of each thread
constexpr uint32_t kAhead = 4;               // vectors of a thread in flight
constexpr uint32_t kBins = 1024;
constexpr uint32_t kListed = 2048;           // tokens that are sorted in LDS
constexpr uint32_t kShortList = 1024;        // the largest top_k whose tokens are listed at once
constexpr uint32_t kSmall = 128;             // tokens that are ranked by counting
constexpr uint32_t kBucket = 32;             // tokens of a bucket that are ranked by counting
constexpr uint32_t kRanges = 8;
constexpr uint32_t kMostTokens = 1u << 20;
constexpr uint32_t kMostRows = kMostTokens / kRow + 1;   // vectors of a thread
constexpr uint32_t kPerRange = (kMostRows + kRanges - 1) / kRanges;

typedef float f32x4_t __attribute__((ext_vector_type(4)));

// ---- sums and maxima over a wave and the block ---------------------------------

// A lower lane's value, 0 where there is none.
template <int kControl, int kRows>
__device__ inline uint64_t dpp_u64(uint64_t v)
{
    auto const lo = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(static_cast<uint32_t>(v)), kControl, kRows, 0xF, false));
    auto const hi = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(static_cast<uint32_t>(v >> 32)), kControl, kRows, 0xF, false));
    return static_cast<uint64_t>(hi) << 32 | lo;
}

// Each lane's sum of its own and the lower lanes' values of its row of 16.
__device__ inline uint64_t row_scan(uint64_t v)
{
    v += dpp_u64<0x111, 0xF>(v);   // shifted by 1, 2, 4, 8
    v += dpp_u64<0x112, 0xF>(v);
    v += dpp_u64<0x114, 0xF>(v);
    v += dpp_u64<0x118, 0xF>(v);
    return v;
}

// The same over the wave.
__device__ inline uint64_t wave_scan(uint64_t v)
{
    v = row_scan(v);
    v += dpp_u64<0x142, 0xA>(v);   // the last lane of rows 0 and 2 to rows 1 and 3
    v += dpp_u64<0x143, 0xC>(v);   // lane 31 to rows 2 and 3
    return v;
}

__device__ inline uint64_t lane_u64(uint64_t v, uint32_t lane)
{
    auto const lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(v)), static_cast<int>(lane)));
    auto const hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(v >> 32)), static_cast<int>(lane)));
    return static_cast<uint64_t>(hi) << 32 | lo;
}

__device__ inline uint64_t wave_total(uint64_t v) { return lane_u64(wave_scan(v), kWave - 1); }

// The highest of a row of 16, in each of its lanes.
__device__ inline float row_max(float v)
{
    auto const turned = [&](auto control) {
        return __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(__float_as_uint(v)), decltype(control)::value, 0xF, 0xF, true)));
    };
    v = fmaxf(v, turned(std::integral_constant<int, 0x128>{}));   // rotated by 8, 4, 2, 1
    v = fmaxf(v, turned(std::integral_constant<int, 0x124>{}));
    v = fmaxf(v, turned(std::integral_constant<int, 0x122>{}));
    v = fmaxf(v, turned(std::integral_constant<int, 0x121>{}));
    return v;
}

struct SampleLds {
    uint32_t count[4 * kBlock];      // of 4096 bins of keys, or of kBins
    uint64_t mass[kBins];
    uint64_t listed[kListed];        // key, then ~token, so that falling numbers are the order
    uint64_t other[kListed];         // of a sort, and the listed tokens' weights
    uint64_t range[kRanges * kWaves];
    uint64_t row[kPerRange * kWaves];
    uint64_t wave[kWaves];
    uint64_t found;
    uint64_t before;
    float wave_f[kWaves];
    uint32_t word[4];
};

// Sum of the lower threads' values, and of all in *total.
__device__ inline uint64_t block_scan(uint64_t v, SampleLds& lds, uint64_t* total)
{
    uint32_t const wave = threadIdx.x / kWave;
    uint64_t const upto = wave_scan(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == kWave - 1) lds.wave[wave] = upto;
    __syncthreads();
    static_assert(kWaves == 16, "a row of lanes holds the waves' sums");
    uint64_t const waves = row_scan(lds.wave[threadIdx.x & (kWaves - 1)]);
    *total = lane_u64(waves, kWaves - 1);
    uint64_t const before = wave == 0 ? 0 : lane_u64(waves, __builtin_amdgcn_readfirstlane(static_cast<int>(wave)) - 1u);
    return before + upto - v;
}

__device__ inline uint64_t block_total(uint64_t v, SampleLds& lds)
{
    uint64_t total;
    static_cast<void>(block_scan(v, lds, &total));
    return total;
}

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

// An ordered whole number of a logit that is not NaN (-0 as 0); 0 is below all of them.
__device__ inline uint32_t key_of(float x)
{
    uint32_t const b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
}
__device__ inline float logit_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) != 0 ? key & 0x7FFFFFFFu : ~key); }

// Weights below 2^-48, of tokens this many T under the highest, are 0.
constexpr float kWeightless = 33.5f;

struct Weights {
    double highest;
    double rate;       // log2(e) / T
    uint32_t scale;    // S

    // 2^t of t = (x - m) rate = n + f, n whole: 1 + f q(f) on [-1/2, 1/2], q the
    // polynomial of degree 9 through (2^f - 1) / f at the Chebyshev nodes, off by
    // 2^-50.  Sums with 1.5 2^52 and 2^52 round to whole numbers, in their low
    // bits.  0 for -inf and NaN.
    __device__ uint64_t of(float x) const
    {
        double const t = (static_cast<double>(x) - highest) * rate;
        double const z = t + 6755399441055744.0;
        double const f = t - (z - 6755399441055744.0);
        double s = 7.070968007227213e-09;
        s = fma(s, f, 1.0205905282567993e-07);
        s = fma(s, f, 1.3215451685760035e-06);
        s = fma(s, f, 1.5252672925515726e-05);
        s = fma(s, f, 0.0001540353042468356);
        s = fma(s, f, 0.001333355820079351);
        s = fma(s, f, 0.009618129107618728);
        s = fma(s, f, 0.05550410866465168);
        s = fma(s, f, 0.24022650695910075);
        s = fma(s, f, 0.6931471805599462);
        s = fma(s, f, 1.0);
        int64_t const n = static_cast<int32_t>(__double_as_longlong(z)) + static_cast<int32_t>(scale);
        double const w = __longlong_as_double(__double_as_longlong(s) + (n << 52)) + 4503599627370496.0;
        return t > -64.0 ? static_cast<uint64_t>(__double_as_longlong(w)) & 0xFFFFFFFFFFFFFull : 0;
    }
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

    // -inf past the row.  With logits of +inf, these alone are there, all alike.
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
        return x;
    }
    __device__ f32x4_t as_counted(f32x4_t x) const
    {
        if (infinite) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) x[i] = x[i] == INFINITY ? 0.0f : -INFINITY;
        }
        return x;
    }

    // f(j, vector) for every vector, in order, the next ones on their way.  One
    // vector an iteration: code that a row's block runs through once comes from
    // memory at its own pace, and eight vectors held in registers and passed over
    // in unrolled code took 43 us for 4 rows of 32000 drawn whole, a loop 26.
    template <typename F>
    __device__ __attribute__((always_inline)) void vectors_do(F f) const
    {
        f32x4_t ahead[kAhead];
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) ahead[k] = load(k);
#pragma nounroll
        for (uint32_t j = 0; j < vectors; ++j) {
            f32x4_t const now = as_counted(ahead[0]);
#pragma unroll
            for (uint32_t k = 1; k < kAhead; ++k) ahead[k - 1] = ahead[k];
            ahead[kAhead - 1] = load(j + kAhead);
            f(j, now);
        }
    }

    // f(token, logit) for every token of this thread with a logit in [low, high];
    // vectors without one in any lane cost four comparisons.
    template <typename F>
    __device__ __attribute__((always_inline)) void each_within(float low, float high, F f) const
    {
        vectors_do([&](uint32_t j, f32x4_t const& y) __attribute__((always_inline)) {
            bool in[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) in[i] = y[i] >= low && y[i] <= high;
            if (!(in[0] || in[1] || in[2] || in[3])) return;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                if (in[i]) f(token(j) + i, y[i]);
            }
        });
    }
};

__device__ inline float highest_of(f32x4_t const& y) { return fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])); }

// The last kept token: its logit and its number.  Kept are the higher logits,
// and of its own the tokens up to it.
struct Last {
    float logit;
    uint32_t token;
    __device__ bool keeps(float x, uint32_t t) const { return x > logit || (x == logit && t <= token); }
};

// ---- the draw from a row -------------------------------------------------------

// What a token weighs in a draw.
struct Kept {
    Weights weights;
    Last last;
    uint64_t least;   // weights below it are not kept
    float floor;      // no logit below it is kept or weighs anything

    __device__ __attribute__((always_inline)) uint64_t of(float x, uint32_t token) const
    {
        uint64_t const w = weights.of(x);
        return last.keeps(x, token) && w >= least ? w : 0;
    }
};

// One for each token of a logit.
struct Same {
    float floor;
    __device__ uint64_t of(float x, uint32_t) const { return x == floor ? 1 : 0; }
};

// The sums of the tokens' weights by ranges of `per` vectors, and all of them.
template <typename W>
__device__ __attribute__((always_inline)) inline uint64_t sum_ranges(const Row& row, SampleLds& lds, uint32_t per, const W& weight)
{
    uint32_t const wave = threadIdx.x / kWave;
    uint32_t const lane = threadIdx.x & (kWave - 1);
    __syncthreads();
    if (threadIdx.x < kRanges * kWaves) lds.range[threadIdx.x] = 0;
    __syncthreads();
    uint64_t all = 0, sum = 0;
    uint32_t at = 0, left = per;
    row.vectors_do([&](uint32_t j, f32x4_t const& y) __attribute__((always_inline)) {
        if (highest_of(y) >= weight.floor) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) sum += weight.of(y[i], row.token(j) + i);
        }
        if (--left == 0 || j + 1 == row.vectors) {
            if (__ballot(sum != 0) != 0) {
                uint64_t const total = wave_total(sum);
                if (lane == 0) lds.range[at * kWaves + wave] = total;
                all += total;
            }
            sum = 0;
            ++at;
            left = per;
        }
    });
    return block_total(lane == 0 ? all : 0, lds);
}

// The first token at which the running sum exceeds `target`, less than all of
// it; the ranges' sums are in place.  Its weight in *its.
template <typename W>
__device__ uint32_t token_at(const Row& row, SampleLds& lds, uint32_t per, uint64_t target, const W& weight, uint64_t* its)
{
    uint32_t const wave = threadIdx.x / kWave;
    uint32_t const lane = threadIdx.x & (kWave - 1);
    static_assert(kRanges * kWaves == 2 * kWave, "two a lane, eight lanes a range");
    if (wave == 0) {
        uint64_t const sum = lds.range[2 * lane] + lds.range[2 * lane + 1];
        uint64_t const upto = wave_scan(sum);
        // The lane in which the target lies; its range's first lane knows what lies before.
        uint64_t const hit = __ballot(target >= upto - sum && target - (upto - sum) < sum);
        uint32_t const at = static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(hit)) - 1) & ~7u;
        if (lane == at) {
            lds.word[0] = at / 8;
            lds.before = upto - sum;
        }
    }
    __syncthreads();
    uint32_t const j0 = lds.word[0] * per;
    uint32_t const j1 = min(j0 + per, row.vectors);
    uint64_t at = lds.before;
    uint64_t w4[4] = {};
#pragma nounroll
    for (uint32_t j = j0; j < j1; ++j) {
        f32x4_t const y = row.as_counted(row.load(j));
        uint64_t sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            w4[i] = weight.of(y[i], row.token(j) + i);
            sum += w4[i];
        }
        uint64_t const total = wave_total(sum);
        if (lane == 0) lds.row[(j - j0) * kWaves + wave] = total;
    }
    __syncthreads();
#pragma nounroll
    for (uint32_t j = j0; j < j1; ++j) {
        uint64_t const part = lds.row[(j - j0) * kWaves + (lane & (kWaves - 1))];
        uint64_t const upto = row_scan(part);
        uint64_t const mine = lane_u64(part, __builtin_amdgcn_readfirstlane(static_cast<int>(wave)));
        uint64_t before = at + lane_u64(upto, __builtin_amdgcn_readfirstlane(static_cast<int>(wave))) - mine;
        at += lane_u64(upto, kWaves - 1);
        if (target < before || target - before >= mine) continue;
        // In this vector of this wave.
        if (j + 1 != j1) {
            f32x4_t const y = row.as_counted(row.load(j));
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) w4[i] = weight.of(y[i], row.token(j) + i);
        }
        uint64_t const sum = w4[0] + w4[1] + w4[2] + w4[3];
        before += wave_scan(sum) - sum;
        if (target < before || target - before >= sum) continue;
        bool found = false;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            if (!found && target - before < w4[i]) {
                found = true;
                lds.word[1] = row.token(j) + i;
                lds.found = w4[i];
            }
            if (!found) before += w4[i];
        }
    }
    __syncthreads();
    *its = lds.found;
    return lds.word[1];
}

// ---- sorting ---------------------------------------------------------------------

// Sorts numbers[0, n), all different, into falling order; n at most kListed,
// their upper words within low .. high.
__device__ __attribute__((noinline)) void sort_falling(uint64_t* numbers, SampleLds& lds, uint32_t n, uint32_t low, uint32_t high)
{
    uint32_t const tid = threadIdx.x;
    __syncthreads();
    if (n <= kSmall) {
        // Each goes to the place that the higher ones leave it: eight threads a number.
        uint32_t const mine = tid / (kBlock / kSmall);
        uint32_t const part = tid % (kBlock / kSmall);
        uint64_t const x = mine < n ? numbers[mine] : 0;
        uint32_t higher = 0;
        for (uint32_t i = part; i < n; i += kBlock / kSmall) higher += numbers[i] > x ? 1u : 0u;
#pragma unroll
        for (uint32_t k = 1; k < kBlock / kSmall; k *= 2) higher += static_cast<uint32_t>(__shfl_xor(static_cast<int>(higher), static_cast<int>(k)));
        __syncthreads();
        if (mine < n && part == 0) numbers[higher] = x;
        __syncthreads();
        return;
    }
    // Buckets of the upper words, a thread each; then each number to its place in its bucket.
    static_assert(kBins == kBlock && kListed == 2 * kBlock, "a bucket and two numbers a thread");
    uint32_t shift = 0;
    while (((high - low) >> shift) >= kBins) ++shift;
    lds.count[tid] = 0;
    __syncthreads();
    uint64_t x[2];
    uint32_t bucket[2], place[2];
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        uint32_t const at = tid + i * kBlock;
        if (at >= n) continue;
        x[i] = numbers[at];
        bucket[i] = (high - static_cast<uint32_t>(x[i] >> 32)) >> shift;
        place[i] = atomicAdd(&lds.count[bucket[i]], 1u);
    }
    __syncthreads();
    uint32_t const size = lds.count[tid];
    uint64_t all;
    uint64_t const start = block_scan(size, lds, &all);
    lds.count[kBins + tid] = static_cast<uint32_t>(start);
    if (__syncthreads_or(size > kBucket) == 0) {
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            if (tid + i * kBlock < n) lds.other[lds.count[kBins + bucket[i]] + place[i]] = x[i];
        }
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            if (tid + i * kBlock >= n) continue;
            uint32_t const first = lds.count[kBins + bucket[i]];
            uint32_t const last = first + lds.count[bucket[i]];
            uint32_t higher = 0;
            for (uint32_t k = first; k < last; ++k) higher += lds.other[k] > x[i] ? 1u : 0u;
            numbers[first + higher] = x[i];
        }
        __syncthreads();
        return;
    }
    // Crowded buckets: pairs compared and exchanged.
    uint32_t padded = 2 * kSmall;
    while (padded < n) padded *= 2;
    for (uint32_t i = n + tid; i < padded; i += kBlock) numbers[i] = 0;
    for (uint32_t k = 2; k <= padded; k *= 2) {
        for (uint32_t j = k / 2; j > 0; j /= 2) {
            __syncthreads();
            for (uint32_t p = tid; p < padded / 2; p += kBlock) {
                uint32_t const i = 2 * p - (p & (j - 1));
                uint64_t const a = numbers[i];
                uint64_t const b = numbers[i + j];
                if ((a < b) == ((i & k) == 0)) {
                    numbers[i] = b;
                    numbers[i + j] = a;
                }
            }
        }
    }
    __syncthreads();
}

// ---- the cuts of a row -------------------------------------------------------------

// What a cut looks for: the `amount`-th token (from 1) of the order, or the
// first at which the weight reaches `amount`.
struct Cut {
    bool by_mass;
    uint64_t amount;
};

// Bins of the logits from the highest down to where weights are 0; the last
// one's tokens are not counted.  Half a logit, as the difference of two may be
// past the largest number.
struct Bins {
    float half;      // of the highest logit
    float rate;      // bins for a unit of half a logit, finite
    __device__ uint32_t of(float x) const { return static_cast<uint32_t>(fminf((half - 0.5f * x) * rate, static_cast<float>(kBins - 1))); }
};

// The bin of the counted ones that the cut falls into, how many tokens it
// holds, and what lies before it of what the cut counts.
struct Place {
    uint32_t bin;     // kBins: the cut lies past all that is counted
    uint32_t count;
    uint64_t before;
};

__device__ inline Place place_of(SampleLds& lds, const Cut& cut, uint64_t before)
{
    static_assert(kBins == kBlock, "a thread a bin");
    uint32_t const tid = threadIdx.x;
    uint64_t all;
    uint64_t const mine = cut.by_mass ? lds.mass[tid] : lds.count[tid];
    uint64_t const at = before + block_scan(mine, lds, &all);
    if (tid == 0) lds.word[0] = kBins;
    __syncthreads();
    if (at < cut.amount && cut.amount - at <= mine) {   // one thread at most
        lds.word[0] = tid;
        lds.word[1] = lds.count[tid];
        lds.before = at;
    }
    __syncthreads();
    Place const p{lds.word[0], lds.word[1], lds.before};
    __syncthreads();
    return p;
}

// Where the cut falls; everything is kept where it lies past what is counted.
// The bins' counts and weights are in lds.
__device__ __attribute__((noinline)) Last find_cut(const Row& row, SampleLds& lds, const Weights& weights, const Bins& bins, const Cut& cut,
                                                   uint32_t per)
{
    uint32_t const tid = threadIdx.x;
    Place place = place_of(lds, cut, 0);
    if (place.bin == kBins) return Last{-INFINITY, 0xFFFFFFFFu};
    uint32_t const bin = place.bin;
    // The bin's tokens, and their highest and lowest keys, of the logits that
    // may be in it: its bounds with a part in 2^18 of the largest on the way.
    auto const border = [&](uint32_t b) { return 2.0f * (bins.half - static_cast<float>(b) / bins.rate); };
    float const slack = (fabsf(bins.half) + static_cast<float>(bin + 1) / bins.rate) * 0x1p-17f;
    float const low_x = border(bin + 1) - slack;
    float const high_x = border(bin) + slack;
    if (tid < 3) lds.word[tid] = tid == 2 ? 0xFFFFFFFFu : 0;
    __syncthreads();
    row.each_within(low_x == low_x ? low_x : -INFINITY, high_x == high_x ? high_x : INFINITY, [&](uint32_t token, float x) __attribute__((always_inline)) {
        if (bins.of(x) != bin) return;
        uint32_t const key = key_of(x);
        if (place.count <= kListed) lds.listed[atomicAdd(&lds.word[0], 1u)] = static_cast<uint64_t>(key) << 32 | (0xFFFFFFFFu - token);
        atomicMax(&lds.word[1], key);
        atomicMin(&lds.word[2], key);
    });
    __syncthreads();
    uint32_t high = lds.word[1];
    uint32_t low = lds.word[2];
    while (place.count > kListed && high != low) {
        // The keys low .. high, cut into bins of 2^shift keys.
        uint32_t shift = 0;
        while (((high - low) >> shift) >= kBins) ++shift;
        __syncthreads();
        lds.count[tid] = 0;
        lds.mass[tid] = 0;
        __syncthreads();
        // The keys' own bounds count: that of -0 is no logit's, but compares as 0.
        row.each_within(logit_of(low), logit_of(high), [&](uint32_t, float x) __attribute__((always_inline)) {
            uint32_t const key = key_of(x);
            if (key < low || key > high) return;
            uint32_t const b = (high - key) >> shift;
            atomicAdd(&lds.count[b], 1u);
            if (cut.by_mass) atomicAdd(reinterpret_cast<unsigned long long*>(&lds.mass[b]), static_cast<unsigned long long>(weights.of(x)));
        });
        __syncthreads();
        place = place_of(lds, cut, place.before);
        high -= place.bin << shift;
        uint32_t const keys = 1u << shift;
        low = high - low >= keys ? high - keys + 1 : low;
        if (place.count > kListed) continue;
        if (tid == 0) lds.word[0] = 0;
        __syncthreads();
        row.each_within(logit_of(low), logit_of(high), [&](uint32_t token, float x) __attribute__((always_inline)) {
            uint32_t const key = key_of(x);
            if (key >= low && key <= high) lds.listed[atomicAdd(&lds.word[0], 1u)] = static_cast<uint64_t>(key) << 32 | (0xFFFFFFFFu - token);
        });
        __syncthreads();
    }
    uint64_t const left = cut.amount - place.before;   // at least 1
    if (place.count > kListed) {
        // One key: so many of its tokens, the lowest first.
        uint64_t const weight = cut.by_mass ? weights.of(logit_of(high)) : 1;
        Same const same{logit_of(high)};
        static_cast<void>(sum_ranges(row, lds, per, same));
        uint64_t one;
        uint32_t const token = token_at(row, lds, per, (left - 1) / weight, same, &one);
        return Last{logit_of(high), token};
    }
    sort_falling(lds.listed, lds, place.count, low, high);
    // Two neighbours of the order a thread.
    uint64_t w[2] = {};
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        uint32_t const n = 2 * tid + i;
        if (n < place.count) w[i] = cut.by_mass ? weights.of(logit_of(static_cast<uint32_t>(lds.listed[n] >> 32))) : 1;
    }
    uint64_t total;
    uint64_t at = block_scan(w[0] + w[1], lds, &total);
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        if (at < left && left - at <= w[i]) {
            lds.word[0] = static_cast<uint32_t>(lds.listed[2 * tid + i] >> 32);
            lds.word[1] = 0xFFFFFFFFu - static_cast<uint32_t>(lds.listed[2 * tid + i]);
        }
        at += w[i];
    }
    __syncthreads();
    Last const last{logit_of(lds.word[0]), lds.word[1]};
    __syncthreads();
    return last;
}

// ---- the draw from a short list -----------------------------------------------------

struct Drawn {
    uint32_t token;
    uint64_t weight;
    uint64_t total;
};

// From the list of the highest tokens, keys within low .. high, the first top_k
// of which count.  Each thread has up to two neighbours of the list.
__device__ inline Drawn draw_listed(SampleLds& lds, const Weights& weights, const kimkv_sample_rule& rule, uint32_t listed, uint32_t top_k,
                                    uint32_t low, uint32_t high, float uniform, uint32_t V)
{
    uint32_t const tid = threadIdx.x;
    sort_falling(lds.listed, lds, listed, low, high);
    uint32_t const n = min(listed, top_k);
    uint64_t const least = part_of(rule.min_p, uint64_t{1} << weights.scale, true);
    uint64_t w[2];
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) w[i] = 2 * tid + i < n ? weights.of(logit_of(static_cast<uint32_t>(lds.listed[2 * tid + i] >> 32))) : 0;
    uint64_t total;
    uint64_t at = block_scan(w[0] + w[1], lds, &total);
    // What top-p keeps begins before its part of the weight is reached.
    uint64_t const need = rule.top_p < 1.0f ? part_of(rule.top_p, total, true) : ~uint64_t{0};
    uint32_t kept = 0;
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        if (2 * tid + i < n && at < need && w[i] >= least) {
            kept += 1;
            at += w[i];
        } else {
            at = ~uint64_t{0};   // nor what comes behind
            w[i] = 0;
        }
    }
    uint32_t const m = static_cast<uint32_t>(block_total(kept, lds));
    // The kept ones in the vocabulary's order: ~token, then the place in the list.
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        uint32_t const p = 2 * tid + i;
        if (p < m) lds.listed[p] = lds.listed[p] << 32 | p;
    }
    sort_falling(lds.listed, lds, m, 0xFFFFFFFFu - (V - 1), 0xFFFFFFFFu);
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        if (2 * tid + i < m) lds.other[2 * tid + i] = w[i];
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) w[i] = 2 * tid + i < m ? lds.other[static_cast<uint32_t>(lds.listed[2 * tid + i])] : 0;
    at = block_scan(w[0] + w[1], lds, &total);
    uint64_t const target = part_of(uniform, total, false);
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        if (target >= at && target - at < w[i]) {
            lds.word[0] = 0xFFFFFFFFu - static_cast<uint32_t>(lds.listed[2 * tid + i] >> 32);
            lds.found = w[i];
        }
        at += w[i];
    }
    __syncthreads();
    return Drawn{lds.word[0], lds.found, total};
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
    auto const clear = [&] {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) lds.count[i * kBlock + tid] = 0;
        lds.mass[tid] = 0;
    };
    clear();

    // ---- the highest logit, by place in a vector (NaN is left out) ----
    f32x4_t high4 = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    row.vectors_do([&](uint32_t, f32x4_t const& y) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) high4[i] = fmaxf(high4[i], y[i]);
    });
    float high = row_max(highest_of(high4));
    high = fmaxf(high, xor16(high));
    high = fmaxf(high, xor32(high));
    if (lane == 0) lds.wave_f[tid / kWave] = high;
    __syncthreads();
    high = row_max(lds.wave_f[lane & (kWaves - 1)]);
    if (high == -INFINITY) {
        answer(KIMKV_NO_TOKEN, 0.0f);
        return;
    }
    row.infinite = high == INFINITY;
    high4 = row.as_counted(high4);
    if (row.infinite) high = 0.0f;

    bool const greedy = rule.temperature == 0.0f;
    float const temperature = greedy ? 1.0f : rule.temperature;
    uint32_t const top_k = greedy ? 1 : rule.top_k == 0 || rule.top_k >= a.V ? a.V : rule.top_k;
    bool const cut_k = top_k < a.V || greedy;
    bool const cut_p = !greedy && rule.top_p < 1.0f;
    Weights const weights{high, 1.4426950408889634 / static_cast<double>(temperature), a.scale};

    if (cut_k && top_k <= kShortList) {
        // Bins of the maxima's keys, from the highest down; four of them a thread.
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            if (high4[i] != -INFINITY) atomicAdd(&lds.count[4095u - (key_of(high4[i]) >> 20)], 1u);
        }
        if (tid == 0) {
            lds.word[0] = 0;       // listed tokens
            lds.word[1] = 4095;    // the bound's bin: all, where there are fewer maxima
        }
        __syncthreads();
        uint32_t of[4];
        uint64_t sum = 0, all;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            of[i] = lds.count[4 * tid + i];
            sum += of[i];
        }
        uint64_t at = block_scan(sum, lds, &all);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            if (at < top_k && at + of[i] >= top_k) lds.word[1] = 4 * tid + i;   // one thread at most
            at += of[i];
        }
        __syncthreads();
        uint32_t const bound = max((4095u - lds.word[1]) << 20, 0x00800000u);   // at least the lowest number's key
        row.each_within(logit_of(bound), INFINITY, [&](uint32_t token, float x) __attribute__((always_inline)) {
            uint32_t const at_list = atomicAdd(&lds.word[0], 1u);
            if (at_list < kListed) lds.listed[at_list] = static_cast<uint64_t>(key_of(x)) << 32 | (0xFFFFFFFFu - token);
        });
        __syncthreads();
        uint32_t const listed = lds.word[0];
        if (listed <= kListed) {
            Drawn const d = draw_listed(lds, weights, rule, listed, top_k, bound, key_of(high), uniform, a.V);
            answer(d.token, static_cast<float>(static_cast<double>(d.weight) / static_cast<double>(d.total)));
            return;
        }
        __syncthreads();
        clear();
        __syncthreads();
    }

    // Ranges of `per` vectors.
    uint32_t const per = (row.vectors + kRanges - 1) / kRanges;
    float const weightless = high - kWeightless * temperature;   // no logit below weighs anything; -inf past the largest number
    Last last{-INFINITY, 0xFFFFFFFFu};
    if (cut_k || cut_p) {
        Bins const bins{0.5f * high, fminf(2 * (kBins - 1) / (kWeightless * temperature), 3e38f)};
        row.vectors_do([&](uint32_t, f32x4_t const& y) __attribute__((always_inline)) {
            if (bins.of(highest_of(y)) >= kBins - 1) return;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                uint32_t const b = bins.of(y[i]);
                if (b >= kBins - 1) continue;
                atomicAdd(&lds.count[b], 1u);
                if (cut_p) atomicAdd(reinterpret_cast<unsigned long long*>(&lds.mass[b]), static_cast<unsigned long long>(weights.of(y[i])));
            }
        });
        __syncthreads();
        uint32_t const count = lds.count[tid];
        uint64_t const mass = lds.mass[tid];
        uint64_t total = 0;
        if (cut_p) total = block_total(mass, lds);
        if (cut_k) {
            last = find_cut(row, lds, weights, bins, Cut{false, top_k}, per);
            if (cut_p && last.logit != -INFINITY) total = sum_ranges(row, lds, per, Kept{weights, last, 0, fmaxf(last.logit, weightless)});
        }
        if (cut_p) {
            __syncthreads();
            lds.count[tid] = count;
            lds.mass[tid] = mass;
            __syncthreads();
            Last const mine = find_cut(row, lds, weights, bins, Cut{true, part_of(rule.top_p, total, true)}, per);
            if (mine.logit > last.logit || (mine.logit == last.logit && mine.token < last.token)) last = mine;
        }
    }

    // ---- the draw ----
    float floor = fmaxf(last.logit, weightless);
    if (rule.min_p > 0.0f) {
        // Below min-p's logit by more than what 32 bits lose on the way to it.
        float const under = temperature * logf(rule.min_p);
        floor = fmaxf(floor, high + under - (fabsf(high) - under) * 0x1p-18f);
    }
    Kept const kept{weights, last, part_of(rule.min_p, uint64_t{1} << a.scale, true), floor};
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
