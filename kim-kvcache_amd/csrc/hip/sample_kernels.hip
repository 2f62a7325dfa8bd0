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
//   - The highest logit.  Where a list may do, for each of 4096 parts of the row
//     (columns) the highest, its place and the second.
//   - List (top_k of at most 1024; few tokens that min-p keeps): a bound that
//     top_k columns reach, or min-p's logit.  The tokens from it up are known from
//     the columns, but for those in which two reach it, so the row is not read
//     again.  They are sorted in LDS, and the cuts and the draw go on there.
//   - Else, for top-p: weights of 2048 bins of the logits for each wave's run of
//     the row, with a longer top_k their counts; the bins that the cuts and min-p's
//     border fall into, their tokens sorted in LDS, which gives the last kept token
//     and what is kept of each run.
//   - With a longer top_k alone, or where the bins hold more tokens than LDS takes:
//     counts (and weights) of 4096 bins, the bin of the cut, its tokens sorted, or
//     cut into 4096 again by their keys.
//   - The draw from a row or a run: the kept tokens' weights summed by ranges of
//     the vocabulary, the range that the random number falls into, the token in it.
//
// Bound by the one block of a row, 8 waves, two a SIMD: there is no room for more,
// as the bins take 128 KB of LDS and a thread 185 registers, in rows too that end in
// a list and need neither.  While the block runs, its SIMDs' vector units issue for
// 0.47 of the time in rows from a list, for 0.51 to 0.57 in rows by weights; for the
// rest both waves wait, for loads and for their own chains (256 rows of 128000: 15
// vector instructions for 64 tokens with T = 0, 43 drawn from the row, a weight 26 of
// them, 60 with top-p).  A pass of weights over 32000 tokens takes 11 us, where
// reading the row takes 2.  So a list saves passes: 72 rows of 50255 with top_k 50
// take 16 us (20 us where the list came from a second pass over the row), 256 rows of
// 128000 34 us (58), which is 3.9 TB/s.  16 waves a block left 128 registers a thread,
// which spilled, and these took 17 and 42 us.  Drawn from all the row 28 and 75 us;
// top-p of 0.9 46 and 103, of which one pass of weights (without the runs' own bins a
// second one for the draw: 58 and 140), with min-p 45 and 100, with top_k 3000 56 and
// 125.  Tried and slower for top-p: a list from the highest columns up (256 flat rows
// of 128000 184 us, as it falls back there); counts and mean places of the bins first,
// then one pass of weights that sums by ranges and lists the tokens of the bins in
// question (215 us: a pass of 64-bit additions to LDS takes as long as one with the
// weights).
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "attention_common.h"
#include "device_common.h"
#include "runtime_internal.h"

namespace kimkv {
namespace {

constexpr unsigned kBlock = 512;
constexpr uint32_t kWaves = kBlock / kWave;
constexpr uint32_t kVector = 4 * kWave;      // tokens of one load of a wave
constexpr uint32_t kAhead = 4;               // vectors of a thread in flight
constexpr uint32_t kBins = 4096;
constexpr uint32_t kBinsEach = kBins / kBlock;
constexpr uint32_t kWaveBins = 2048;         // of a wave's own
constexpr uint32_t kWaveBinsEach = kWaveBins / kBlock;
constexpr uint32_t kListed = 2048;           // tokens that are sorted in LDS
constexpr uint32_t kListedEach = kListed / kBlock;
constexpr uint32_t kListedOfWave = kListed / kWaves;
constexpr uint32_t kShortList = 1024;        // the largest top_k whose tokens are listed at once
constexpr uint32_t kCrowded = 96;            // columns that a wave reads again (8, one by one: 72 rows of 50255, top_k 700, 31 us, not 22; no other shape measured)
constexpr uint32_t kAgain = 4;               // of these at once
constexpr uint32_t kSets = 2;                // of a thread's columns
constexpr uint32_t kSmall = 128;             // tokens that are ranked by counting
static_assert(2 * kListed <= kBins, "a sort's counts and starts");
constexpr uint32_t kBucket = 32;             // tokens of a bucket that are ranked by counting
constexpr uint32_t kMostTokens = 1u << 20;
constexpr uint32_t kRange = 4096;            // tokens of a range of a draw
constexpr uint32_t kRangeEach = kRange / kBlock;
constexpr uint32_t kRanges = kMostTokens / kRange + kWaves;   // of all waves, the last of each wave's a part

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
    union {
        uint64_t of_wave[kWaves][kWaveBins];   // weights
        struct {
            uint32_t count[kBins];
            union {
                uint64_t mass[kBins];
                uint64_t other[kListed];       // of a sort, and the listed tokens' weights
            };
        };
    };
    uint64_t listed[kListed];        // key, then ~token, so that falling numbers are the order
    uint64_t range[kRanges];
    uint64_t wave[kWaves];
    uint64_t run[kWaves];            // what is kept of a wave's run
    uint32_t count_of[kWaves];       // what a wave has listed
    uint32_t again[kWaves][kCrowded];   // columns that a wave reads again
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
    static_assert(kWaves <= 16, "a row of lanes holds the waves' sums");
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
        double const t = fmax((static_cast<double>(x) - highest) * rate, -64.0);   // of NaN too
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
        return static_cast<uint64_t>(__double_as_longlong(w)) & 0xFFFFFFFFFFFFFull;
    }
};

// The row as the block reads it: each wave a run of whole vectors, of which
// vector j of lane l is tokens first + kVector j + 4 l + 0 .. 3, at any address of
// 4 bytes.  So the vocabulary's order is the waves', the vectors' and the lanes'.
struct Row {
    const float* from;
    uint32_t V;
    uint32_t run;        // vectors of a wave
    bool infinite;       // the highest logit is +inf
    uint32_t base;       // number of its first token

    __device__ uint32_t first() const { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / kWave))) * run * kVector; }
    __device__ uint32_t place(uint32_t j) const { return first() + j * kVector + 4 * (threadIdx.x & (kWave - 1)); }
    __device__ uint32_t token(uint32_t j) const { return base + place(j); }
    __device__ uint32_t vectors() const
    {
        uint32_t const at = first();
        return at < V ? min(run, (V - at + kVector - 1) / kVector) : 0;
    }

    // Four tokens, -inf past the row.
    __device__ f32x4_t load(uint32_t v) const
    {
        f32x4_t x;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) x[i] = v + i < V ? from[v + i] : -INFINITY;
        return x;
    }
    // With logits of +inf, these alone are there, all alike.
    __device__ f32x4_t as_counted(f32x4_t x) const
    {
        if (infinite) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) x[i] = x[i] == INFINITY ? 0.0f : -INFINITY;
        }
        return x;
    }

    // f(j, vector) for every vector of the wave, in order, the next ones on their
    // way: loads that the hardware bounds to the row, without a branch, behind
    // which the compiler would wait for all of them, each to its own registers,
    // as a copy would wait too; the last vector comes from a load of its own.  A
    // loop of kAhead vectors: code that a row's block runs through once comes from
    // memory at its own pace, and eight vectors held in registers and passed over
    // in unrolled code took 43 us for 4 rows of 32000 drawn whole.
    template <typename F>
    __device__ __attribute__((always_inline)) void vectors_do(F f) const
    {
        uint32_t const n = vectors();
        if (n == 0) return;
        auto const bounded = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(from), 0, static_cast<int>(4 * V), 0x00027000);
        uint32_t const at = 4 * place(0);
        auto const ahead_of = [&](uint32_t j) {
            return __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(bounded, static_cast<int>(at + j * kVector * 4), 0, 0));
        };
        f32x4_t const last = load(place(n - 1));
        f32x4_t ahead[kAhead];
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) ahead[k] = ahead_of(k);
#pragma nounroll
        for (uint32_t j = 0; j < n; j += kAhead) {
#pragma unroll
            for (uint32_t k = 0; k < kAhead; ++k) {
                f32x4_t now = ahead[k];
                if (j + k + 1 >= n) now = last;
                now = as_counted(now);
                ahead[k] = ahead_of(j + k + kAhead);
                if (j + k < n) f(j + k, now);
            }
        }
    }
};

__device__ inline float highest_of(f32x4_t const& y) { return fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])); }

// A token's number of the list: falling numbers are the order.
__device__ inline uint64_t listing(float x, uint32_t token) { return static_cast<uint64_t>(key_of(x)) << 32 | (0xFFFFFFFFu - token); }

__device__ inline uint32_t lanes_below(uint64_t in) { return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(in >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(in), 0)); }

// Places of the list for a wave's tokens, the first of them: one atomic operation
// for all, as the wave waits for it.
__device__ inline uint32_t list_places(SampleLds& lds, uint32_t count)
{
    uint32_t at = 0;
    if (count != 0 && (threadIdx.x & (kWave - 1)) == 0) at = atomicAdd(&lds.word[0], count);
    return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(at)));
}

// Lists the lanes' tokens that are in from place *at on, as far as the list goes.
__device__ inline void list_lanes(SampleLds& lds, uint64_t in, float x, uint32_t token, uint32_t* at)
{
    uint32_t const place = *at + lanes_below(in);
    if ((in >> (threadIdx.x & (kWave - 1)) & 1u) != 0 && place < kListed) lds.listed[place] = listing(x, token);
    *at += static_cast<uint32_t>(__popcll(in));
}

// Lists the tokens of a vector that pass, a lane's bit in[i] for its i-th.
__device__ inline void list_vector(SampleLds& lds, const uint64_t (&in)[4], f32x4_t const& y, uint32_t token)
{
    uint32_t at = list_places(lds, static_cast<uint32_t>(__popcll(in[0]) + __popcll(in[1]) + __popcll(in[2]) + __popcll(in[3])));
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) list_lanes(lds, in[i], y[i], token + i, &at);
}

__device__ inline void start_list(SampleLds& lds)
{
    __syncthreads();
    if (threadIdx.x == 0) lds.word[0] = 0;
    __syncthreads();
}

// Lists the tokens whose logits are in [low, high] and pass; returns how many
// there are.  A wave keeps its own in a part of the list, without waiting for
// places (with that, top-p of 0.9 took 49 and 112 us at the shapes above); where one
// has more, they go into the whole list.
template <typename F>
__device__ __attribute__((always_inline)) inline uint32_t list_tokens(const Row& row, SampleLds& lds, float low, float high, F passes)
{
    uint32_t const lane = threadIdx.x & (kWave - 1);
    uint32_t const wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / kWave)));
    uint64_t* const mine = lds.listed + wave * kListedOfWave;
    auto const each = [&](auto list) __attribute__((always_inline)) {
        row.vectors_do([&](uint32_t j, f32x4_t const& y) __attribute__((always_inline)) {
            bool any = false;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) any = any || (y[i] >= low && y[i] <= high);
            if (__ballot(any) == 0) return;
            uint64_t in[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) in[i] = __ballot(y[i] >= low && y[i] <= high && passes(y[i]));
            list(in, y, row.token(j));
        });
    };
    start_list(lds);
    uint32_t count = 0;
    each([&](const uint64_t (&in)[4], f32x4_t const& y, uint32_t token) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            if (in[i] == 0) continue;
            uint32_t const place = count + lanes_below(in[i]);
            if ((in[i] >> lane & 1u) != 0 && place < kListedOfWave) mine[place] = listing(y[i], token + i);
            count += static_cast<uint32_t>(__popcll(in[i]));
        }
    });
    if (lane == 0) lds.count_of[wave] = count;
    __syncthreads();
    uint32_t before = 0, all = 0, most = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
        uint32_t const n = lds.count_of[w];
        before += w < wave ? n : 0;
        all += n;
        most = max(most, n);
    }
    if (most > kListedOfWave) {
        each([&](const uint64_t (&in)[4], f32x4_t const& y, uint32_t token) __attribute__((always_inline)) { list_vector(lds, in, y, token); });
        __syncthreads();
        return all;
    }
    uint64_t x[kListedOfWave / kWave];
#pragma unroll
    for (uint32_t i = 0; i < kListedOfWave / kWave; ++i) x[i] = mine[i * kWave + lane];
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kListedOfWave / kWave; ++i) {
        if (i * kWave + lane < count) lds.listed[before + i * kWave + lane] = x[i];
    }
    __syncthreads();
    return all;
}

// What a lane's i-th tokens of every kSets-th vector (a column) come to: the
// highest, in which vector it is, and the second.
struct Columns {
    f32x4_t first;
    f32x4_t second;
    uint32_t vector[4];
};

// Lists the tokens from a bound up, and returns how many there are, or more than
// the list takes where they are more than `most`.  Each is in a column whose highest has reached the bound: it is
// that one where the second has not, else the column is read again, its tokens
// side by side in the wave, or the row where a wave has many such columns.
__device__ inline uint32_t list_columns(const Row& row, SampleLds& lds, const Columns (&columns)[kSets], float bound, uint32_t most)
{
    uint32_t const lane = threadIdx.x & (kWave - 1);
    uint32_t least = 0, crowded = 0;
#pragma unroll
    for (uint32_t set = 0; set < kSets; ++set) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            least += static_cast<uint32_t>(__popcll(__ballot(columns[set].first[i] >= bound)));
            crowded += static_cast<uint32_t>(__popcll(__ballot(columns[set].second[i] >= bound)));
        }
    }
    if (block_total(lane == 0 ? least + crowded : 0, lds) > most) return kListed + 1;
    if (__syncthreads_or(crowded > kCrowded) != 0) return list_tokens(row, lds, bound, INFINITY, [](float) { return true; });
    start_list(lds);
    uint32_t const wave = threadIdx.x / kWave;
    uint64_t one[4 * kSets];
    uint32_t alone = 0, again = 0;
#pragma unroll
    for (uint32_t k = 0; k < 4 * kSets; ++k) {
        Columns const& c = columns[k / 4];
        one[k] = __ballot(c.first[k % 4] >= bound && !(c.second[k % 4] >= bound));
        alone += static_cast<uint32_t>(__popcll(one[k]));
        // The numbers of the columns to be read again.
        uint64_t const more = __ballot(c.second[k % 4] >= bound);
        if ((more >> lane & 1u) != 0) lds.again[wave][again + lanes_below(more)] = k / 4 * kVector + 4 * lane + k % 4;
        again += static_cast<uint32_t>(__popcll(more));
    }
    uint32_t at = list_places(lds, alone);
#pragma unroll
    for (uint32_t k = 0; k < 4 * kSets; ++k) {
        Columns const& c = columns[k / 4];
        list_lanes(lds, one[k], c.first[k % 4], row.token(c.vector[k % 4]) + k % 4, &at);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    uint32_t const n = row.vectors();
#pragma nounroll
    for (uint32_t k = 0; k < again; k += kAgain) {
        for (uint32_t first = 0; first < n; first += kSets * kWave) {
            uint32_t token[kAgain];
            float x[kAgain];
            uint64_t in[kAgain];
            uint32_t count = 0;
#pragma unroll
            for (uint32_t e = 0; e < kAgain; ++e) {
                uint32_t const number = lds.again[wave][min(k + e, again - 1)];
                uint32_t const j = first + number / kVector + kSets * lane;
                uint32_t const v = row.first() + j * kVector + number % kVector;
                token[e] = row.base + v;
                x[e] = k + e < again && j < n && v < row.V ? row.from[v] : -INFINITY;
            }
#pragma unroll
            for (uint32_t e = 0; e < kAgain; ++e) {
                if (row.infinite) x[e] = x[e] == INFINITY ? 0.0f : -INFINITY;
                in[e] = __ballot(x[e] >= bound);
                count += static_cast<uint32_t>(__popcll(in[e]));
            }
            at = list_places(lds, count);
#pragma unroll
            for (uint32_t e = 0; e < kAgain; ++e) list_lanes(lds, in[e], x[e], token[e], &at);
        }
    }
    __syncthreads();
    return lds.word[0];
}

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
    float border;     // min-p keeps the logits from it up
    float floor;      // no logit below it is kept or weighs anything
    float sure;       // every logit above it is kept

    __device__ __attribute__((always_inline)) uint64_t of(float x, uint32_t token) const
    {
        uint64_t const w = weights.of(x);
        return last.keeps(x, token) && x >= border ? w : 0;
    }
    __device__ __attribute__((always_inline)) uint64_t of(f32x4_t const& y, uint32_t token) const
    {
        uint64_t sum = 0;
        bool border = false;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) border = border || (y[i] >= floor && y[i] <= sure);
        if (__ballot(border) != 0) {
#pragma nounroll
            for (uint32_t i = 0; i < 4; ++i) sum += of(i < 2 ? (i == 0 ? y[0] : y[1]) : (i == 2 ? y[2] : y[3]), token + i);
        } else {
            // All four at once: a weight is a chain of dependent operations.
            uint64_t w[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) w[i] = weights.of(y[i]);
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) sum += y[i] > sure ? w[i] : 0;
        }
        return sum;
    }
};

// One for each token of a logit.
struct Same {
    float floor;
    __device__ uint64_t of(float x, uint32_t) const { return x == floor ? 1 : 0; }
    __device__ uint64_t of(f32x4_t const& y, uint32_t) const { return of(y[0], 0) + of(y[1], 0) + of(y[2], 0) + of(y[3], 0); }
};

// The lowest logit that min-p keeps: the least number of 32 bits at or above
// m + T log min_p, in 64 bits, as that may lie past the largest of 32.
__device__ inline float min_p_border(double highest, float temperature, float min_p)
{
    if (min_p == 0.0f) return -INFINITY;
    double const at = highest + static_cast<double>(temperature) * log(static_cast<double>(min_p));
    float const near = static_cast<float>(at);
    return static_cast<double>(near) < at ? nextafterf(near, INFINITY) : near;
}

// The kept tokens down to the last one of a cut, of those that min-p keeps.
__device__ inline Kept kept_tokens(const Weights& weights, const Last& last, float temperature, float border)
{
    float const high = static_cast<float>(weights.highest);
    return Kept{weights, last, border, fmaxf(fmaxf(last.logit, high - kWeightless * temperature), border), fmaxf(last.logit, nextafterf(border, -INFINITY))};
}

// Ranges of a wave's run.
__device__ inline uint32_t ranges_of(const Row& row) { return (row.run * kVector + kRange - 1) / kRange; }

// The sums of the tokens' weights by ranges, and all of them.
template <typename W>
__device__ __attribute__((always_inline)) inline uint64_t sum_ranges(const Row& row, SampleLds& lds, const W& weight)
{
    uint32_t const lane = threadIdx.x & (kWave - 1);
    uint32_t const ranges = ranges_of(row);
    uint32_t const mine = threadIdx.x / kWave * ranges;
    __syncthreads();
    // Runs that end before the row's last range leave some of theirs empty.
    for (uint32_t i = threadIdx.x; i < kRanges; i += kBlock) lds.range[i] = 0;
    __syncthreads();
    uint64_t all = 0, sum = 0;
    uint32_t const n = row.vectors();
    row.vectors_do([&](uint32_t j, f32x4_t const& y) __attribute__((always_inline)) {
        if (highest_of(y) >= weight.floor) sum += weight.of(y, row.token(j));
        if (j % (kRange / kVector) == kRange / kVector - 1 || j + 1 == n) {
            uint64_t const total = wave_total(sum);
            if (lane == 0) lds.range[mine + j / (kRange / kVector)] = total;
            all += total;
            sum = 0;
        }
    });
    return block_total(lane == 0 ? all : 0, lds);
}

// The first token at which the running sum exceeds `target`, less than all of
// it; the ranges' sums are in place.  Its weight in *its.
template <typename W>
__device__ __attribute__((always_inline)) inline uint32_t token_at(const Row& row, SampleLds& lds, uint64_t target, const W& weight, uint64_t* its)
{
    static_assert(kRanges <= kBlock, "a thread a range");
    uint32_t const tid = threadIdx.x;
    uint32_t const ranges = ranges_of(row);
    uint64_t all;
    uint64_t sum = tid < ranges * kWaves ? lds.range[tid] : 0;
    uint64_t before = block_scan(sum, lds, &all);
    if (target >= before && target - before < sum) {   // one thread
        lds.word[0] = tid / ranges * row.run * kVector + tid % ranges * kRange;
        lds.word[1] = min((tid / ranges + 1) * row.run * kVector, lds.word[0] + kRange);
        lds.before = before;
    }
    __syncthreads();
    // The range's tokens, neighbours each thread.
    uint32_t const v = lds.word[0] + kRangeEach * tid;
    uint32_t const end = lds.word[1];
    uint64_t w[kRangeEach];
    sum = 0;
#pragma unroll
    for (uint32_t k = 0; k < kRangeEach; k += 4) {
        f32x4_t const y = row.as_counted(row.load(v + k));
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            uint64_t const x = weight.of(y[i], row.base + v + k + i);
            w[k + i] = v + k + i < end ? x : 0;
            sum += w[k + i];
        }
    }
    before = lds.before + block_scan(sum, lds, &all);
    if (target >= before && target - before < sum) {   // one thread
        bool found = false;
#pragma unroll
        for (uint32_t k = 0; k < kRangeEach; ++k) {
            if (!found && target - before < w[k]) {
                found = true;
                lds.word[2] = v + k;
                lds.found = w[k];
            }
            if (!found) before += w[k];
        }
    }
    __syncthreads();
    *its = lds.found;
    return row.base + lds.word[2];
}

// ---- sorting ---------------------------------------------------------------------

// Sorts numbers[0, n), all different, into falling order; n at most kListed.
// Their upper words are keys of logits, or ~tokens, which count as -token;
// these are at most `highest`, and lie within about `width`.
__device__ __attribute__((always_inline)) inline void sort_falling(uint64_t* numbers, SampleLds& lds, uint32_t n, bool logits, float highest, float width)
{
    uint32_t const tid = threadIdx.x;
    __syncthreads();
    if (n <= kSmall) {
        // Each goes to the place that the higher ones leave it: four threads a number.
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
    // Buckets, as many as the list has places; then each number to its place in its bucket.
    float const rate = static_cast<float>(kListed) / width;
    uint32_t* const starts = lds.count + kListed;
#pragma unroll
    for (uint32_t i = 0; i < kListedEach; ++i) lds.count[i * kBlock + tid] = 0;
    __syncthreads();
    uint64_t x[kListedEach];
    uint32_t bucket[kListedEach], place[kListedEach];
#pragma unroll
    for (uint32_t i = 0; i < kListedEach; ++i) {
        uint32_t const at = tid + i * kBlock;
        if (at >= n) continue;
        x[i] = numbers[at];
        uint32_t const word = static_cast<uint32_t>(x[i] >> 32);
        float const value = logits ? logit_of(word) : -static_cast<float>(0xFFFFFFFFu - word);
        bucket[i] = static_cast<uint32_t>(fminf((highest - value) * rate, static_cast<float>(kListed - 1)));   // of NaN the last
        place[i] = atomicAdd(&lds.count[bucket[i]], 1u);
    }
    __syncthreads();
    uint32_t size[kListedEach], sum = 0, most = 0;
#pragma unroll
    for (uint32_t i = 0; i < kListedEach; ++i) {
        size[i] = lds.count[kListedEach * tid + i];
        sum += size[i];
        most = max(most, size[i]);
    }
    uint64_t all;
    uint32_t start = static_cast<uint32_t>(block_scan(sum, lds, &all));
#pragma unroll
    for (uint32_t i = 0; i < kListedEach; ++i) {
        starts[kListedEach * tid + i] = start;
        start += size[i];
    }
    if (__syncthreads_or(most > kBucket) == 0) {
#pragma unroll
        for (uint32_t i = 0; i < kListedEach; ++i) {
            if (tid + i * kBlock < n) lds.other[starts[bucket[i]] + place[i]] = x[i];
        }
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kListedEach; ++i) {
            if (tid + i * kBlock >= n) continue;
            uint32_t const first = starts[bucket[i]];
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

// Bins of the logits from the highest down over `width`; the last one's tokens
// are not counted.  Half a logit, as the difference of two may be
// past the largest number.
struct Bins {
    float high;      // the highest logit
    float half;      // of it: rounded, where it is below the normal numbers
    float rate;      // bins for a unit of half a logit, finite
    float last;      // bin
    __device__ uint32_t of(float x) const { return static_cast<uint32_t>(fminf((half - 0.5f * x) * rate, last)); }
    __device__ Bins(float high, float width, uint32_t n)
        : high(high), half(0.5f * high), rate(fminf(2.0f * static_cast<float>(n - 1) / width, 3e38f)), last(static_cast<float>(n - 1))
    {
    }
    // No logit of the bin is below under(b), and none above over(b): the borders,
    // and what a part in 2^17 of the largest number on the way may take from them.
    __device__ float slack(uint32_t b) const { return (fabsf(half) + static_cast<float>(b + 1) / rate) * 0x1p-17f; }
    __device__ float under(uint32_t b) const
    {
        float const x = 2.0f * (half - static_cast<float>(b + 1) / rate) - slack(b);
        return x == x ? x : -INFINITY;
    }
    __device__ float over(uint32_t b) const
    {
        float const x = 2.0f * (half - static_cast<float>(b) / rate) + slack(b);
        return x == x ? x : INFINITY;
    }
};

// The bin that the cut falls into, and what lies before it of what the cut counts.
struct Place {
    uint32_t bin;     // kBins: the cut lies past all that is counted
    uint64_t before;
};

__device__ inline Place place_of(SampleLds& lds, const Cut& cut, uint64_t before)
{
    uint32_t const tid = threadIdx.x;
    uint64_t of[kBinsEach];
    uint64_t sum = 0, all;
#pragma unroll
    for (uint32_t i = 0; i < kBinsEach; ++i) {
        of[i] = cut.by_mass ? lds.mass[kBinsEach * tid + i] : lds.count[kBinsEach * tid + i];
        sum += of[i];
    }
    uint64_t at = before + block_scan(sum, lds, &all);
    if (tid == 0) lds.word[0] = kBins;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kBinsEach; ++i) {
        if (at < cut.amount && cut.amount - at <= of[i]) {   // one bin at most
            lds.word[0] = kBinsEach * tid + i;
            lds.before = at;
        }
        at += of[i];
    }
    __syncthreads();
    Place const p{lds.word[0], lds.before};
    __syncthreads();
    return p;
}

__device__ inline void clear_bins(SampleLds& lds)
{
#pragma unroll
    for (uint32_t i = 0; i < kBinsEach; ++i) {
        lds.count[i * kBlock + threadIdx.x] = 0;
        lds.mass[i * kBlock + threadIdx.x] = 0;
    }
}

// Where the cut falls; everything is kept where it lies past what is counted.
// The bins' counts (or weights, for a cut by them) are in lds.
__device__ __attribute__((always_inline)) inline Last find_cut(const Row& row, SampleLds& lds, const Weights& weights, const Bins& bins, const Cut& cut)
{
    uint32_t const tid = threadIdx.x;
    Place place = place_of(lds, cut, 0);
    if (place.bin == kBins) return Last{-INFINITY, 0xFFFFFFFFu};
    uint32_t const bin = place.bin;
    // The bin's tokens, and the keys that they can have.
    float const low_x = bins.under(bin);
    float const high_x = bins.over(bin);
    uint32_t low = key_of(fmaxf(low_x, -3.4028234664e38f));
    uint32_t high = key_of(fminf(high_x, bins.high));
    uint32_t listed = list_tokens(row, lds, low_x, high_x, [&](float x) { return bins.of(x) == bin; });
    if (listed > kListed) {
        // Too many: their highest and lowest keys, and bins of these.
        if (tid == 0) {
            lds.word[1] = 0;
            lds.word[2] = 0xFFFFFFFFu;
        }
        __syncthreads();
        uint32_t most = 0, fewest = 0xFFFFFFFFu;
        row.vectors_do([&](uint32_t, f32x4_t const& y) __attribute__((always_inline)) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                if (bins.of(y[i]) != bin) continue;
                most = max(most, key_of(y[i]));
                fewest = min(fewest, key_of(y[i]));
            }
        });
        atomicMax(&lds.word[1], most);
        atomicMin(&lds.word[2], fewest);
        __syncthreads();
        high = lds.word[1];
        low = lds.word[2];
    }
    // A token of the keys low .. high: that of -0 is no logit's, but compares as 0.
    auto const within = [&](float x) {
        uint32_t const key = key_of(x);
        return key >= low && key <= high;
    };
    while (listed > kListed && high != low) {
        // The keys, cut into bins of 2^shift of them.
        uint32_t shift = 0;
        while (((high - low) >> shift) >= kBins) ++shift;
        __syncthreads();
        clear_bins(lds);
        __syncthreads();
        row.vectors_do([&](uint32_t, f32x4_t const& y) __attribute__((always_inline)) {
#pragma nounroll
            for (uint32_t i = 0; i < 4; ++i) {
                float const x = i < 2 ? (i == 0 ? y[0] : y[1]) : (i == 2 ? y[2] : y[3]);
                if (x != x || !within(x)) continue;
                uint32_t const b = (high - key_of(x)) >> shift;
                if (cut.by_mass) {
                    atomicAdd(reinterpret_cast<unsigned long long*>(&lds.mass[b]), static_cast<unsigned long long>(weights.of(x)));
                } else {
                    atomicAdd(&lds.count[b], 1u);
                }
            }
        });
        __syncthreads();
        place = place_of(lds, cut, place.before);
        high -= place.bin << shift;
        uint32_t const keys = 1u << shift;
        low = high - low >= keys ? high - keys + 1 : low;
        listed = list_tokens(row, lds, logit_of(low), logit_of(high), within);
    }
    uint64_t const left = cut.amount - place.before;   // at least 1
    if (listed > kListed) {
        // One key: so many of its tokens, the lowest first.
        uint64_t const weight = cut.by_mass ? weights.of(logit_of(high)) : 1;
        Same const same{logit_of(high)};
        static_cast<void>(sum_ranges(row, lds, same));
        uint64_t one;
        uint32_t const token = token_at(row, lds, (left - 1) / weight, same, &one);
        return Last{logit_of(high), token};
    }
    sort_falling(lds.listed, lds, listed, true, logit_of(high), logit_of(high) - logit_of(low));
    // Neighbours of the order each thread.
    uint64_t w[kListedEach] = {};
#pragma unroll
    for (uint32_t i = 0; i < kListedEach; ++i) {
        uint32_t const n = kListedEach * tid + i;
        if (n < listed) w[i] = cut.by_mass ? weights.of(logit_of(static_cast<uint32_t>(lds.listed[n] >> 32))) : 1;
    }
    uint64_t total, sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < kListedEach; ++i) sum += w[i];
    uint64_t at = block_scan(sum, lds, &total);
#pragma unroll
    for (uint32_t i = 0; i < kListedEach; ++i) {
        if (at < left && left - at <= w[i]) {
            lds.word[0] = static_cast<uint32_t>(lds.listed[kListedEach * tid + i] >> 32);
            lds.word[1] = 0xFFFFFFFFu - static_cast<uint32_t>(lds.listed[kListedEach * tid + i]);
        }
        at += w[i];
    }
    __syncthreads();
    Last const last{logit_of(lds.word[0]), lds.word[1]};
    __syncthreads();
    return last;
}

// ---- top-p's cut, and what it keeps of each wave's run -------------------------------

// The weights in bins of each wave's own give the bin that the cut falls into; the
// tokens of that or of min-p's border's, whichever is first, listed and sorted,
// give the last kept one, and with the bins before it what is kept of every run:
// lds.run.  Top-p's part is of the first top_k tokens' weight (V: of
// all): counts of the bins give the one of the last of them, whose tokens are
// listed and sorted for their weight.  False where a list is too long.
__device__ __attribute__((always_inline)) inline bool cut_of_runs(const Row& row, SampleLds& lds, const Weights& weights, const Bins& bins, float top_p,
                                                                  uint32_t top_k, const Kept& kept, Last* last)
{
    uint32_t const tid = threadIdx.x;
    uint32_t const lane = tid & (kWave - 1);
    uint32_t const wave = tid / kWave;
    auto* const counts = reinterpret_cast<uint32_t*>(lds.listed);   // until there is a list
    static_assert(kWaveBins * sizeof(uint32_t) <= sizeof(lds.listed), "the bins' counts");
    bool const cut_k = top_k < row.V;
    if (cut_k) {
#pragma unroll
        for (uint32_t i = 0; i < kWaveBinsEach; ++i) counts[i * kBlock + tid] = 0;
        __syncthreads();
    }
    row.vectors_do([&](uint32_t, f32x4_t const& y) __attribute__((always_inline)) {
        if (bins.of(highest_of(y)) >= kWaveBins - 1) return;
        uint32_t b[4];
        uint64_t w[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            b[i] = bins.of(y[i]);
            w[i] = weights.of(y[i]);
        }
        // Here, and not each behind its condition.
        asm volatile("" : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3]));
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            if (b[i] < kWaveBins - 1) atomicAdd(reinterpret_cast<unsigned long long*>(&lds.of_wave[wave][b[i]]), static_cast<unsigned long long>(w[i]));
        }
        if (cut_k) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                if (b[i] < kWaveBins - 1) atomicAdd(&counts[b[i]], 1u);
            }
        }
    });
    __syncthreads();
    uint64_t of[kWaveBinsEach];
    uint64_t sum = 0, total;
#pragma unroll
    for (uint32_t i = 0; i < kWaveBinsEach; ++i) {
        of[i] = 0;
#pragma unroll
        for (uint32_t v = 0; v < kWaves; ++v) of[i] += lds.of_wave[v][kWaveBinsEach * tid + i];
        sum += of[i];
    }
    uint64_t const first = block_scan(sum, lds, &total);
    uint64_t at = first;
    if (cut_k) {
        uint32_t n[kWaveBinsEach];
        sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < kWaveBinsEach; ++i) {
            n[i] = counts[kWaveBinsEach * tid + i];
            sum += n[i];
        }
        uint64_t all;
        uint64_t tokens = block_scan(sum, lds, &all);
        if (tid == 0) lds.word[3] = kWaveBins;
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kWaveBinsEach; ++i) {
            if (tokens < top_k && top_k - tokens <= n[i]) {   // one bin, or none where fewer weigh anything
                lds.word[3] = kWaveBinsEach * tid + i;
                lds.word[2] = top_k - static_cast<uint32_t>(tokens);
                lds.before = at;
            }
            tokens += n[i];
            at += of[i];
        }
        __syncthreads();
        uint32_t const bin = lds.word[3];
        uint32_t const its = lds.word[2];
        uint64_t const before = lds.before;
        __syncthreads();
        if (bin < kWaveBins) {
            float const low = fmaxf(bins.under(bin), -3.4028234664e38f);
            float const high = fminf(bins.over(bin), bins.high);
            uint32_t const listed = list_tokens(row, lds, low, high, [&](float x) { return bins.of(x) == bin; });
            if (listed > kListed) return false;
            // What lies where the sort works.
            constexpr uint32_t kSaved = (sizeof(lds.count) + sizeof(lds.other)) / sizeof(uint64_t) / kBlock;
            uint64_t* const there = lds.of_wave[0];
            uint64_t saved[kSaved];
#pragma unroll
            for (uint32_t i = 0; i < kSaved; ++i) saved[i] = there[i * kBlock + tid];
            sort_falling(lds.listed, lds, listed, true, high, high - low);
            sum = 0;
#pragma unroll
            for (uint32_t i = 0; i < kListedEach; ++i) {
                uint32_t const p = i * kBlock + tid;
                if (p < min(its, listed)) sum += weights.of(logit_of(static_cast<uint32_t>(lds.listed[p] >> 32)));
            }
            total = before + block_total(sum, lds);
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < kSaved; ++i) there[i * kBlock + tid] = saved[i];
            __syncthreads();
        }
        at = first;
    }
    uint64_t const amount = part_of(top_p, total, true);   // at least 1, at most the total
#pragma unroll
    for (uint32_t i = 0; i < kWaveBinsEach; ++i) {
        if (at < amount && amount - at <= of[i]) lds.word[3] = kWaveBinsEach * tid + i;   // one bin
        at += of[i];
    }
    __syncthreads();
    uint32_t const bin = lds.word[3];
    uint32_t const end = min(bins.of(kept.floor), bin);
    at = first;
#pragma unroll
    for (uint32_t i = 0; i < kWaveBinsEach; ++i) {
        if (kWaveBinsEach * tid + i == end) lds.before = at;
        at += of[i];
    }
    sum = 0;
    for (uint32_t b = lane; b < end; b += kWave) sum += lds.of_wave[wave][b];
    sum = wave_total(sum);
    if (lane == 0) lds.run[wave] = sum;
    if (tid == 0) {
        lds.word[1] = 0xFFFFFFFFu;   // the last token, where the list holds it
        lds.word[2] = key_of(-INFINITY);
    }
    __syncthreads();
    uint64_t const left = amount - lds.before;   // at least 1
    float const low = fmaxf(bins.under(end), -3.4028234664e38f);
    float const high = fminf(bins.over(end), bins.high);
    uint32_t const listed = list_tokens(row, lds, low, high, [&](float x) { return bins.of(x) == end; });
    if (listed > kListed) return false;
    sort_falling(lds.listed, lds, listed, true, high, high - low);
    // Neighbours of the order each thread.
    uint64_t w[kListedEach];
    sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < kListedEach; ++i) {
        uint32_t const n = kListedEach * tid + i;
        w[i] = n < listed ? weights.of(logit_of(static_cast<uint32_t>(lds.listed[n] >> 32))) : 0;
        sum += w[i];
    }
    at = block_scan(sum, lds, &total);
#pragma unroll
    for (uint32_t i = 0; i < kListedEach; ++i) {
        uint32_t const n = kListedEach * tid + i;
        if (n < listed && at < left) {
            uint32_t const key = static_cast<uint32_t>(lds.listed[n] >> 32);
            uint32_t const token = 0xFFFFFFFFu - static_cast<uint32_t>(lds.listed[n]);
            if (left - at <= w[i]) {
                lds.word[2] = key;
                lds.word[1] = token;
            }
            if (logit_of(key) >= kept.border) atomicAdd(reinterpret_cast<unsigned long long*>(&lds.run[token / (row.run * kVector)]), static_cast<unsigned long long>(w[i]));
        }
        at += w[i];
    }
    __syncthreads();
    *last = Last{logit_of(lds.word[2]), lds.word[1]};
    return true;
}

// ---- the draw from a short list -----------------------------------------------------

struct Drawn {
    uint32_t token;
    uint64_t weight;
    uint64_t total;
};

// From a list of the first top_k tokens and more, or of all that min-p keeps,
// logits within low .. high; top-p's part is of `total`, or where that is 0 of the
// first top_k's weight.  Each thread has neighbours of the list.
__device__ inline Drawn draw_listed(SampleLds& lds, const Kept& of, float top_p, uint32_t listed, uint32_t top_k, uint64_t total, float low,
                                    float high, float uniform, uint32_t V)
{
    uint32_t const tid = threadIdx.x;
    sort_falling(lds.listed, lds, listed, true, high, high - low);
    uint32_t const n = min(listed, top_k);
    uint64_t w[kListedEach];
    bool good[kListedEach];   // as far as min-p goes
    uint64_t sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < kListedEach; ++i) {
        uint32_t const p = kListedEach * tid + i;
        float const x = p < n ? logit_of(static_cast<uint32_t>(lds.listed[p] >> 32)) : -INFINITY;
        w[i] = of.weights.of(x);
        good[i] = p < n && x >= of.border;
        sum += w[i];
    }
    uint64_t all;
    uint64_t at = block_scan(sum, lds, &all);
    // What top-p keeps begins before its part of the weight is reached.
    uint64_t const need = top_p < 1.0f ? part_of(top_p, total != 0 ? total : all, true) : ~uint64_t{0};
    uint32_t kept = 0;
#pragma unroll
    for (uint32_t i = 0; i < kListedEach; ++i) {
        if (good[i] && at < need) {
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
    for (uint32_t i = 0; i < kListedEach; ++i) {
        uint32_t const p = kListedEach * tid + i;
        if (p < m) lds.listed[p] = lds.listed[p] << 32 | p;
    }
    sort_falling(lds.listed, lds, m, false, 0.0f, static_cast<float>(V));
#pragma unroll
    for (uint32_t i = 0; i < kListedEach; ++i) {
        if (kListedEach * tid + i < m) lds.other[kListedEach * tid + i] = w[i];
    }
    __syncthreads();
    sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < kListedEach; ++i) {
        w[i] = kListedEach * tid + i < m ? lds.other[static_cast<uint32_t>(lds.listed[kListedEach * tid + i])] : 0;
        sum += w[i];
    }
    at = block_scan(sum, lds, &all);
    uint64_t const target = part_of(uniform, all, false);
#pragma unroll
    for (uint32_t i = 0; i < kListedEach; ++i) {
        if (target >= at && target - at < w[i]) {
            lds.word[0] = 0xFFFFFFFFu - static_cast<uint32_t>(lds.listed[kListedEach * tid + i] >> 32);
            lds.found = w[i];
        }
        at += w[i];
    }
    __syncthreads();
    return Drawn{lds.word[0], lds.found, all};
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
    row.run = (a.V + kWaves * kVector - 1) / (kWaves * kVector);
    row.infinite = false;
    row.base = 0;
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

    bool const greedy = rule.temperature == 0.0f;
    float const temperature = greedy ? 1.0f : rule.temperature;
    uint32_t const top_k = greedy ? 1 : rule.top_k == 0 || rule.top_k >= a.V ? a.V : rule.top_k;
    bool const cut_k = top_k < a.V || greedy;
    bool const short_k = cut_k && top_k <= kShortList;
    bool const cut_p = !greedy && rule.top_p < 1.0f;
    bool const list = short_k || (!cut_k && rule.min_p > 0.0f);

    bool const runs = cut_p && !short_k;
    if (runs) {
        for (uint32_t b = lane; b < kWaveBins; b += kWave) lds.of_wave[tid / kWave][b] = 0;
    } else {
        clear_bins(lds);
    }

    // ---- the columns' highest logits (NaN is left out) ----
    constexpr f32x4_t kNone{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    static_assert(kAhead % kSets == 0, "a vector's set is known where the code is built");
    Columns columns[kSets];
#pragma unroll
    for (uint32_t set = 0; set < kSets; ++set) columns[set] = Columns{kNone, kNone, {0, 0, 0, 0}};
    if (list) {
        row.vectors_do([&](uint32_t j, f32x4_t const& y) __attribute__((always_inline)) {
            Columns& c = columns[j % kSets];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                c.second[i] = fmaxf(c.second[i], fminf(c.first[i], y[i]));
                c.vector[i] = y[i] > c.first[i] ? j : c.vector[i];
                c.first[i] = fmaxf(c.first[i], y[i]);
            }
        });
    } else {
        row.vectors_do([&](uint32_t j, f32x4_t const& y) __attribute__((always_inline)) {
            Columns& c = columns[j % kSets];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) c.first[i] = fmaxf(c.first[i], y[i]);
        });
    }
    float high = -INFINITY;
#pragma unroll
    for (uint32_t set = 0; set < kSets; ++set) high = fmaxf(high, highest_of(columns[set].first));
    high = row_max(high);
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
    if (row.infinite) high = 0.0f;
    Weights const weights{high, 1.4426950408889634 / static_cast<double>(temperature), a.scale};
    float const border = min_p_border(high, temperature, rule.min_p);
    Kept kept = kept_tokens(weights, Last{-INFINITY, 0xFFFFFFFFu}, temperature, border);

    // ---- from a list ----
    if (list) {
#pragma unroll
        for (uint32_t set = 0; set < kSets; ++set) {
            columns[set].first = row.as_counted(columns[set].first);
            columns[set].second = row.as_counted(columns[set].second);
        }
        // A bound that so many columns reach, to a part in 4096 of what is looked at;
        // what lies below `none` weighs nothing.
        float const none = fmaxf(high - kWeightless * temperature, -3.4028234664e38f);
        float bound = none;
        if (short_k) {
            Bins const near(high, fminf(kWeightless * temperature, 64.0f), kBins);
#pragma unroll
            for (uint32_t set = 0; set < kSets; ++set) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    uint32_t const b = near.of(columns[set].first[i]);
                    if (b < kBins - 1) atomicAdd(&lds.count[b], 1u);
                }
            }
            __syncthreads();
            uint32_t const bin = place_of(lds, Cut{false, top_k}, 0).bin;
            if (bin < kBins) bound = fmaxf(near.under(bin), none);
        }
        // One that min-p leaves out counts where top-p takes its part of the list.
        if (!short_k || !cut_p) bound = fmaxf(bound, kept.floor);
        // A list of min-p's pays while it is a small part of the row: 256 rows of 128000,
        // some 1300 tokens, 42 us, drawn from the row 74; 72 rows of 50255, some 1500
        // tokens, 38, from the row 28; beside top-p, whose pass of weights comes on top,
        // 256 rows of 128000, up to 2000 tokens, 114, without the list 103.  The 48th part
        // lies between these; no other shape was measured.
        uint32_t const listed = list_columns(row, lds, columns, bound, short_k ? kListed : min(cut_p ? kShortList : kListed, a.V / 48));
        if (listed <= kListed) {
            // Min-p leaves the list, and top-p keeps a part of the row.
            uint64_t total = 0;
            if (!short_k && cut_p) {
                row.vectors_do([&](uint32_t, f32x4_t const& y) __attribute__((always_inline)) {
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) total += weights.of(y[i]);
                });
                total = block_total(total, lds);
            }
            Drawn const d = draw_listed(lds, kept, rule.top_p, listed, top_k, total, bound, high, uniform, a.V);
            answer(d.token, static_cast<float>(static_cast<double>(d.weight) / static_cast<double>(d.total)));
            return;
        }
        if (short_k) {
#pragma unroll
            for (uint32_t i = 0; i < kBinsEach; ++i) lds.count[i * kBlock + tid] = 0;
            __syncthreads();
        }
    }

    // ---- the cuts of the row ----
    Last last{-INFINITY, 0xFFFFFFFFu};
    Row drawn = row;           // the part of the row that the draw falls into
    uint64_t sums = 0;         // of all that is kept, where known
    uint64_t before = 0;       // of it before that part
    bool cut = !cut_k && !cut_p;
    if (runs) {
        Bins const bins(high, kWeightless * temperature, kWaveBins);
        cut = cut_of_runs(row, lds, weights, bins, rule.top_p, top_k, kept, &last);
        if (cut) {
            uint64_t const upto = row_scan(lds.run[lane & (kWaves - 1)]);
            sums = lane_u64(upto, kWaves - 1);
            uint64_t const target = part_of(uniform, sums, false);
            uint32_t const wave = static_cast<uint32_t>(__popcll(__ballot(lane < kWaves && upto <= target)));
            before = wave == 0 ? 0 : lane_u64(upto, wave - 1);
            drawn.base = wave * row.run * kVector;
            drawn.from = row.from + drawn.base;
            drawn.V = min(row.V - drawn.base, row.run * kVector);
            drawn.run = (drawn.V + kWaves * kVector - 1) / (kWaves * kVector);
        } else {
            __syncthreads();
            clear_bins(lds);
            __syncthreads();
        }
    }
    if (!cut) {
        Bins const bins(high, kWeightless * temperature, kBins);
        row.vectors_do([&](uint32_t, f32x4_t const& y) __attribute__((always_inline)) {
            if (bins.of(highest_of(y)) >= kBins - 1) return;
            uint32_t b[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) b[i] = bins.of(y[i]);
            if (cut_k) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    if (b[i] < kBins - 1) atomicAdd(&lds.count[b[i]], 1u);
                }
            }
            if (cut_p) {
                uint64_t w[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) w[i] = weights.of(y[i]);
                // Here, and not each behind its condition.
                asm volatile("" : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3]));
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    if (b[i] < kBins - 1) atomicAdd(reinterpret_cast<unsigned long long*>(&lds.mass[b[i]]), static_cast<unsigned long long>(w[i]));
                }
            }
        });
        __syncthreads();
        uint64_t mass[kBinsEach];
        uint64_t total = 0;
        if (cut_p) {
#pragma unroll
            for (uint32_t i = 0; i < kBinsEach; ++i) {
                mass[i] = lds.mass[i * kBlock + tid];
                total += mass[i];
            }
            total = block_total(total, lds);
        }
        // The top_k tokens' cut, then that of top-p's part of their weight.
#pragma nounroll
        for (uint32_t by_mass = cut_k ? 0 : 1; by_mass <= (cut_p ? 1 : 0); ++by_mass) {
            if (by_mass != 0 && cut_k) {
                if (last.logit != -INFINITY) total = sum_ranges(row, lds, kept_tokens(weights, last, temperature, -INFINITY));
                __syncthreads();
#pragma unroll
                for (uint32_t i = 0; i < kBinsEach; ++i) lds.mass[i * kBlock + tid] = mass[i];
                __syncthreads();
            }
            Last const its = find_cut(row, lds, weights, bins, Cut{by_mass != 0, by_mass != 0 ? part_of(rule.top_p, total, true) : top_k});
            if (its.logit > last.logit || (its.logit == last.logit && its.token < last.token)) last = its;
        }
    }

    // ---- the draw ----
    kept = kept_tokens(weights, last, temperature, border);
    uint64_t const found = sum_ranges(drawn, lds, kept);
    if (sums == 0) sums = found;
    uint64_t its;
    uint32_t const token = token_at(drawn, lds, part_of(uniform, sums, false) - before, kept, &its);
    answer(token, static_cast<float>(static_cast<double>(its) / static_cast<double>(sums)));
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
