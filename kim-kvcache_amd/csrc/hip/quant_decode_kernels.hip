// quant_decode_kernels.hip -- GQA paged decode attention over a cache in 8
// bits: one new token a lane, split over the lane's length and joined.
//
// With k_j, v_j the codes of token j and a_j, b_j their scales,
//   s_j = (q . k_j) a_j scale,   o = sum_j e^(s_j - m) b_j v_j / sum_j e^(s_j - m).
// A code is an fp16 number as it stands, so the products run on the fp16
// matrix cores and the scales stay outside of them, in 32 bits: a_j at the
// score, b_j at the weight.
//
// Work: block = unit (a lane, a KV head, a range of its tokens), its waves, four
// or for few units eight, a part of it each, joined in LDS; a lane of one unit a
// head is written at once, the others' parts are merged by a second launch.  A wave
// takes the table entries that begin in its range, so no page is cut; it reads
// 64 of them at a time.  An entry that is a whole page of 64 tokens is a tile;
// the groups of 8 of all others are collected eight to a tile: the order of the
// tokens does not matter to the sums.  Per tile
//   S^T[token][q] = K[token][:] . Q[q][:]           D / 2 / 4 MFMA 16x16x32
//   online softmax (base 2) on the 16 scores of a lane
//   O^T[d][q]    += V^T[d][token] . (b P)[q][token]  D / 4 MFMA, weights in two fp16 parts
// K rows and V^T rows go from memory to the operand registers in 16-byte loads
// (8 for small pages); tokens are numbered so that the scores a lane holds are
// the weights it needs.
//
// Bound by HBM where batches are large: 128 lanes of 32768 tokens, 4 heads of 64
// (2.2 GB) take 350 us, 6.3 TB/s.  A tile's K registers take the next tile's K as
// soon as the scores stand, and V's the next V behind the sums: two sets of
// registers for a tile (128 dims: 108 of them spilled) made 64 ragged lanes of up
// to 6000 tokens, 8 heads of 128, 55 us instead of 27.  Beside the 17 us that
// their 103 MB take from HBM there are the chain of loads to a unit's first page
// and the merge's launch (4.5 us).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "attention_common.h"
#include "quant_common.h"
#include "runtime_internal.h"

namespace kimkv {
namespace {

constexpr unsigned kBlock = 256;
constexpr uint32_t kWaves = kBlock / kWave;
constexpr uint32_t kTile = 64;           // tokens
constexpr uint32_t kColumns = 16;        // query heads of an operand
constexpr uint32_t kDirect = 0xFFFFFFFFu;

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

// Tokens [first, first + count) of a lane of `tokens`, for a KV head; its part
// goes to `slot`, or to the output.
struct QuantUnit {
    uint32_t lane;
    uint32_t head;
    uint32_t first;
    uint32_t count;
    uint32_t tokens;
    uint32_t slot;
    uint32_t reserved[2];
};

// A lane of several parts a head: slots first_slot + head * parts + part.
struct QuantMerge {
    uint32_t lane;
    uint32_t tokens;
    uint32_t first_slot;
    uint32_t parts;
};

struct DecodeArgs {
    const kimkv_decode_item* items;
    const QuantUnit* units;
    float* work;
    uint32_t G;   // query heads of a KV head
};

// A part: [G][D] sums, then [G] of (m, l).
__host__ __device__ inline uint64_t slot_floats(uint32_t G, uint32_t D) { return static_cast<uint64_t>(G) * (D + 2); }

__device__ inline bool item_good(const QuantView& P, const kimkv_decode_item& item, uint32_t tokens)
{
    return item.token_count == tokens && item.descriptors != nullptr && item.descriptor_count != 0 && item.layer < P.layers
        && item.query != nullptr && item.output != nullptr;
}

// Codes are read once a launch: streamed past the caches.
typedef const __attribute__((address_space(1))) u32x4_t global_u32x4_t;
typedef const __attribute__((address_space(1))) u32x2_t global_u32x2_t;
__device__ inline u32x4_t stream16(const uint8_t* p) { return __builtin_nontemporal_load((global_u32x4_t*)(p)); }
__device__ inline u32x2_t stream8(const uint8_t* p) { return __builtin_nontemporal_load((global_u32x2_t*)(p)); }
__device__ inline u32x4_t load16(const uint8_t* p) { return *(global_u32x4_t*)(p); }
constexpr int kStreamed = 2;

// A page's bytes behind a pointer that is the same in all lanes, or none of
// them: loads of it then read nothing and wait for nothing.
struct PageBytes {
    __amdgpu_buffer_rsrc_t bounded;
    __device__ PageBytes(const uint8_t* p, uint32_t bytes)
        : bounded(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, static_cast<int>(p != nullptr ? bytes : 0), 0x00027000))
    {
    }
    __device__ u32x4_t stream16(uint32_t at) const { return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(bounded, static_cast<int>(at), 0, kStreamed)); }
    __device__ u32x2_t stream8(uint32_t at) const { return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(bounded, static_cast<int>(at), 0, kStreamed)); }
    __device__ u32x4_t load16(uint32_t at) const { return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(bounded, static_cast<int>(at), 0, 0)); }
};

__device__ inline uint64_t lane_value(uint64_t v, int lane)
{
    auto const lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(v)), lane));
    auto const hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(v >> 32)), lane));
    return static_cast<uint64_t>(hi) << 32 | lo;
}

// The highest of the four lanes of a query column: a swap with itself leaves a
// lane its own value and its partner's.
__device__ inline float column_max(float v)
{
    auto const rows = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(rows[0]), __uint_as_float(rows[1]));
    auto const halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
}

// ---------------------------------------------------------------------------
// Matrix-core path of one wave.
// ---------------------------------------------------------------------------
// Lane (g, r) holds O^T[d][r], d = 16 db + 4 g + i, in acc[db][i]; the running
// max m and the sum l of query column r.
template <uint32_t kDim>
struct WavePart {
    float4_t acc[kDim / 16];
    float m;
    float l;
};

// A group of 8 tokens of a page that is not read whole.
struct Group {
    const uint8_t* block;
    uint16_t first;    // page token
    uint16_t cap;
    uint32_t valid;    // tokens of it
};
constexpr uint32_t kGroupsOfEntry = kQuantMaxPage / 8;
constexpr uint32_t kMaxGroups = kWave * kGroupsOfEntry;

constexpr bool fast_dim(uint32_t dim) { return dim == 64 || dim == 96 || dim == 128; }

// A query column's weights enter the product as p b 2^15 / c, with c a power of
// two above 2^3 times every p b of the column so far, all to its running max, and
// above the tile's: they stay below 2^15, and two fp16 parts are off by 2^-22 of a
// weight or by 2^-36 of the column's largest (a step of the lower part is 2^-24, and
// c at most 2^4 times that), whichever is more.  So a row of V costs the others bits
// only as far as it is attended to: with c above the scales b, whatever their p, one
// row of 65504 that weighed nothing left rows of 2^-12 off by 2^-7 of themselves.  The
// 2^3 are room for the scales of later tiles, so that c need not follow each: 128
// lanes of 32768 tokens, 4 heads of 64, take 356.6 us (353.1 with c above the scales);
// without the room 357.4.
constexpr uint32_t kWeightRoom = 3;
constexpr uint32_t kWeightLow = 64;     // exponent bits of c's least, 2^-62
__device__ inline float weight_factor(uint32_t e) { return __uint_as_float((127u + 15u + 126u - e) << 23); }    // 2^15 / c, c = 2^(e - 126)
__device__ inline float weight_unit(uint32_t e) { return __uint_as_float((e - 126u + 127u - 15u) << 23); }      // c / 2^15

template <uint32_t kFormat, uint32_t kDim>
struct Decoder {
    static constexpr uint32_t kSteps = kDim / 32;     // of the score product
    static constexpr uint32_t kDb = kDim / 16;
    static constexpr bool kWide = kDim % 64 == 0;     // K in column blocks of 64
    static constexpr uint32_t kKw = kWide ? 64 : kDim;

    struct Ops {
        u32x2_t k[4][kSteps];    // tokens 16 (r / 4) + 4 tau + r % 4
        u32x4_t v[kDb];          // row 16 db + r, tokens 16 g ..
        u32x4_t ks[2];           // scales of tokens 16 g ..
        u32x4_t vs[2];
    };

    half8_t q[kSteps];
    float4_t acc[kDb] = {};
    float m = -INFINITY;
    float l = 0.0f;              // of this lane's tokens
    float scale2;
    float most = 0.0f;           // of the column's p b
    uint32_t e = kWeightLow;     // c = 2^(e - 126)
    uint32_t g;
    uint32_t r;

    __device__ Decoder(const kimkv_decode_item& item, uint32_t h, uint32_t G)
    {
        uint32_t const lane = threadIdx.x & (kWave - 1);
        g = lane >> 4;
        r = lane & 15u;
        scale2 = item.attention_scale * kLog2e;
        const uint16_t* const row = item.query + (static_cast<uint64_t>(h) * G + min(r, G - 1)) * kDim;
        bool const aligned = (reinterpret_cast<uintptr_t>(item.query) & 15u) == 0;
#pragma unroll
        for (uint32_t j = 0; j < kSteps; ++j) {
            // Dims of this lane in step j, as K's loads have them.
            uint32_t const d = kWide ? 64 * (j / 2) + 16 * g + 8 * (j & 1) : 32 * j + 8 * g;
            half8_t v = {};
            if (r < G) {
                if (aligned) {
                    v = load_half8(row + d);
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i) v[i] = __builtin_bit_cast(_Float16, row[d + i]);
                }
            }
            q[j] = v;
        }
    }

    // The tile of a whole page of 64 tokens, its K and its V.
    __device__ void load_page_k(Ops& o, const PageBytes& page, uint32_t codes_at, uint32_t scales_at) const
    {
        uint32_t const row = codes_at + (16 * (r >> 2) + (r & 3u)) * kKw + g * (kWide ? 16 : 8);
#pragma unroll
        for (uint32_t tau = 0; tau < 4; ++tau) {
            if (kWide) {
#pragma unroll
                for (uint32_t b = 0; b < kSteps / 2; ++b) {
                    u32x4_t const w = page.stream16(row + 4 * tau * kKw + b * kTile * 64);
                    o.k[tau][2 * b] = u32x2_t{w[0], w[1]};
                    o.k[tau][2 * b + 1] = u32x2_t{w[2], w[3]};
                }
            } else {
#pragma unroll
                for (uint32_t j = 0; j < kSteps; ++j) o.k[tau][j] = page.stream8(row + 4 * tau * kKw + 32 * j);
            }
        }
#pragma unroll
        for (uint32_t s = 0; s < 2; ++s) o.ks[s] = page.load16(scales_at + 32 * g + 16 * s);
    }
    __device__ void load_page_v(Ops& o, const PageBytes& page, uint32_t codes_at, uint32_t scales_at) const
    {
#pragma unroll
        for (uint32_t s = 0; s < 2; ++s) o.vs[s] = page.load16(scales_at + 2 * kTile + 32 * g + 16 * s);
        uint32_t const column = codes_at + kTile * kDim + r * kTile + 16 * g;
#pragma unroll
        for (uint32_t db = 0; db < kDb; ++db) o.v[db] = page.stream16(column + db * 16 * kTile);
    }

    // A tile of 8 groups of pages of any kind; `count` (1 .. 8) are there.
    static __device__ const uint8_t* codes_of(const Group& x, uint32_t h) { return x.block + static_cast<uint64_t>(h) * 2 * x.cap * kDim; }
    __device__ void load_groups_k(Ops& o, const Group* groups, uint32_t count, uint32_t heads, uint32_t h) const
    {
#pragma unroll
        for (uint32_t s = 0; s < 2; ++s) {
            uint32_t const n = 2 * (r >> 2) + s;
            Group const x = groups[min(n, count - 1)];
            const uint8_t* const codes = codes_of(x, h);
#pragma unroll
            for (uint32_t u = 0; u < 2; ++u) {
                const uint8_t* const row = codes + (x.first + 4 * u + (r & 3u)) * kKw + g * (kWide ? 16 : 8);
                if (kWide) {
#pragma unroll
                    for (uint32_t b = 0; b < kSteps / 2; ++b) {
                        u32x4_t const w = stream16(row + b * x.cap * 64u);
                        o.k[2 * s + u][2 * b] = u32x2_t{w[0], w[1]};
                        o.k[2 * s + u][2 * b + 1] = u32x2_t{w[2], w[3]};
                    }
                } else {
#pragma unroll
                    for (uint32_t j = 0; j < kSteps; ++j) o.k[2 * s + u][j] = stream8(row + 32 * j);
                }
            }
        }
#pragma unroll
        for (uint32_t s = 0; s < 2; ++s) {
            Group const x = groups[min(2 * g + s, count - 1)];
            o.ks[s] = load16(x.block + static_cast<uint64_t>(heads) * 2 * x.cap * kDim + h * 4u * x.cap + 2 * x.first);
        }
    }
    __device__ void load_groups_v(Ops& o, const Group* groups, uint32_t count, uint32_t heads, uint32_t h, uint32_t (&valid)[2]) const
    {
#pragma unroll
        for (uint32_t s = 0; s < 2; ++s) {
            uint32_t const n = 2 * g + s;
            Group const x = groups[min(n, count - 1)];
            valid[s] = n < count ? x.valid : 0;
            const uint8_t* const column = codes_of(x, h) + x.cap * kDim + r * x.cap + x.first;
#pragma unroll
            for (uint32_t db = 0; db < kDb; ++db) {
                u32x2_t const w = stream8(column + db * 16 * x.cap);
                o.v[db][2 * s] = w[0];
                o.v[db][2 * s + 1] = w[1];
            }
            o.vs[s] = load16(x.block + static_cast<uint64_t>(heads) * 2 * x.cap * kDim + h * 4u * x.cap + 2 * x.first + 2 * x.cap);
        }
    }

    // kMasked: only the first valid[s] tokens of a lane's groups s are there.
    // next_k, next_v: the next tile's loads, into the registers that are done with.
    template <bool kMasked, typename K, typename V>
    __device__ __attribute__((always_inline)) void add(Ops& o, uint32_t (&valid)[2], K next_k, V next_v)
    {
        auto const scale_of = [](const u32x4_t& w, uint32_t t) {
            return __uint_as_float((t & 1u) != 0 ? w[t >> 1] & 0xFFFF0000u : w[t >> 1] << 16);
        };
        // ---- scores: token 8 s + 4 u + i of the lane's 16 ----
        float4_t score[4];
        float mx = -INFINITY;
#pragma unroll
        for (uint32_t tau = 0; tau < 4; ++tau) {
            float4_t z = {};
#pragma unroll
            for (uint32_t j = 0; j < kSteps; ++j) z = __builtin_amdgcn_mfma_f32_16x16x32_f16(code_halves<kFormat>(o.k[tau][j]), q[j], z, 0, 0, 0);
            score[tau] = z;
        }
#pragma unroll
        for (uint32_t tau = 0; tau < 4; ++tau) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                uint32_t const t = 4 * (tau & 1) + i;
                float x = score[tau][i] * (scale_of(o.ks[tau >> 1], t) * scale2);
                if (kMasked && t >= valid[tau >> 1]) x = -INFINITY;
                score[tau][i] = x;
                mx = fmaxf(mx, x);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        next_k();
        __builtin_amdgcn_sched_barrier(0);
        float const m_new = fmaxf(m, column_max(mx));
        // While every score is -inf the reference is 0, so the weights are zeros and not NaN.
        float const m_top = m_new == -INFINITY ? 0.0f : m_new;
        float alpha = __builtin_amdgcn_exp2f(m - m_top);
        m = m_new;

        // ---- V's scales: whether one is NaN ----
        if (kMasked) {
#pragma unroll
            for (uint32_t s = 0; s < 2; ++s) {
#pragma unroll
                for (uint32_t t = 0; t < 8; ++t) {
                    if (t >= valid[s]) o.vs[s][t >> 1] &= (t & 1u) != 0 ? 0x0000FFFFu : 0xFFFF0000u;
                }
            }
        }
        u16x2_t top = {0, 0};
#pragma unroll
        for (uint32_t s = 0; s < 2; ++s) {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                uint32_t const pair = o.vs[s][j];   // a bit cast of a vector's element itself takes the first one's bits
                top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, pair));
            }
        }
        uint32_t const lane_top = top[0] > top[1] ? top[0] : top[1];   // of the lane's tokens
        bool const has_nan = __ballot(lane_top >= 0x7F80u) != 0;

        // ---- weights ----
        float sum = 0.0f;
#pragma unroll
        for (uint32_t tau = 0; tau < 4; ++tau) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                uint32_t const t = 4 * (tau & 1) + i;
                float const p = __builtin_amdgcn_exp2f(score[tau][i] - m_top);
                sum += p;
                float w = p * scale_of(o.vs[tau >> 1], t);
                if (has_nan && p == 0.0f) w = 0.0f;   // a value that weighs nothing is left out, whatever it is
                score[tau][i] = w;
            }
        }
        l = l * alpha + sum;
        // c stays while no running max rises and no scale passes it.
        if (__ballot(alpha != 1.0f || lane_top >> 7 > e) != 0) {
            float tile_most = 0.0f;   // NaN is left out
#pragma unroll
            for (uint32_t tau = 0; tau < 4; ++tau) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) tile_most = fmaxf(tile_most, score[tau][i]);
            }
            most = fmaxf(most * alpha, column_max(tile_most));
            uint32_t const e_new = max((__float_as_uint(most) >> 23) + kWeightRoom, kWeightLow);
            alpha *= __uint_as_float((127u + e - e_new) << 23);
            e = e_new;
#pragma unroll
            for (uint32_t db = 0; db < kDb; ++db) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) acc[db][i] = alpha == 0.0f ? 0.0f : acc[db][i] * alpha;
            }
        }
        float const factor = weight_factor(e);
        half8_t hi[2], lo[2];
#pragma unroll
        for (uint32_t tau = 0; tau < 4; ++tau) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                uint32_t const t = 4 * (tau & 1) + i;
                float const w = score[tau][i] * factor;
                _Float16 const part = static_cast<_Float16>(w);
                hi[tau >> 1][t] = part;
                lo[tau >> 1][t] = static_cast<_Float16>(w - static_cast<float>(part));
            }
        }
#pragma unroll
        for (uint32_t s = 0; s < 2; ++s) {
#pragma unroll
            for (uint32_t db = 0; db < kDb; ++db) {
                half8_t const v = code_halves<kFormat>(u32x2_t{o.v[db][2 * s], o.v[db][2 * s + 1]});
                acc[db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, hi[s], acc[db], 0, 0, 0);
                acc[db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, lo[s], acc[db], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        next_v();
        __builtin_amdgcn_sched_barrier(0);
    }

    __device__ WavePart<kDim> part() const
    {
        WavePart<kDim> out;
        float const unit = weight_unit(e);
#pragma unroll
        for (uint32_t db = 0; db < kDb; ++db) out.acc[db] = acc[db] * unit;
        float sum = l + xor16(l);
        sum += xor32(sum);
        out.m = m;
        out.l = sum;
        return out;
    }
};

// The entries that begin within [t0, t1), as far as the lane's tokens go; *bad
// where one names no page of the storage.
template <uint32_t kFormat, uint32_t kDim>
__device__ WavePart<kDim> decode_wave(const QuantView& P, const kimkv_decode_item& item, uint32_t h, uint32_t G, uint32_t t0,
                                      uint32_t t1, uint32_t tokens, Group* groups, bool* bad)
{
    uint32_t const lane = threadIdx.x & (kWave - 1);
    Decoder<kFormat, kDim> d(item, h, G);
    // A short table is read whole, without the search's own read of it.
    uint32_t const count = item.descriptor_count;
    uint32_t idx = t0 >= t1 ? count : count <= kWave ? 0 : find_descriptor_wave(item.descriptors, count, t0);
    uint32_t const codes_at = h * 2 * kTile * kDim;
    uint32_t const scales_at = P.heads * 2 * kTile * kDim + h * 4 * kTile;
    uint32_t const page_bytes = P.heads * kTile * (2 * kDim + 4);
    while (idx < count) {
        // This lane's entry.
        bool const there = count - idx > lane;
        kimkv_block_desc entry{};
        if (there) entry = item.descriptors[idx + lane];
        uint32_t const begin = entry.logical_token_begin;
        uint32_t const cap = entry.page_token_capacity;
        bool const mine = there && begin >= t0 && begin < t1 && entry.valid_tokens != 0;
        uint32_t const valid = mine ? min(static_cast<uint32_t>(entry.valid_tokens), tokens - begin) : 0;
        const uint8_t* block = nullptr;
        if (mine && entry.valid_tokens <= cap) block = quant_block(P, item.layer, entry.kind, entry.slot, cap);
        *bad = *bad || __ballot(mine && block == nullptr) != 0;
        bool const page = block != nullptr && cap == kTile && valid == kTile;
        uint32_t const parts = block != nullptr && !page ? (valid + 7) / 8 : 0;
        uint32_t before = parts;   // groups of the lanes up to this one
#pragma unroll
        for (uint32_t k = 1; k < kWave; k *= 2) {
            uint32_t const v = static_cast<uint32_t>(__shfl_up(static_cast<int>(before), k));
            if (lane >= k) before += v;
        }
        uint32_t const total = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(before), 63));
        for (uint32_t k = 0; k < parts; ++k) {
            groups[before - parts + k] = Group{block, static_cast<uint16_t>(8 * k), static_cast<uint16_t>(cap), min(8u, valid - 8 * k)};
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();

        // Whole pages.
        uint64_t left = __ballot(page);
        if (left != 0) {
            typename Decoder<kFormat, kDim>::Ops o;
            uint32_t whole[2] = {8, 8};
            auto const next = [&] {
                if (left == 0) return PageBytes(nullptr, 0);
                int const j = __ffsll(static_cast<unsigned long long>(left)) - 1;
                return PageBytes(reinterpret_cast<const uint8_t*>(lane_value(reinterpret_cast<uint64_t>(block), j)), page_bytes);
            };
            PageBytes p = next();
            d.load_page_k(o, p, codes_at, scales_at);
            d.load_page_v(o, p, codes_at, scales_at);
            do {
                left &= left - 1;
                p = next();
                d.template add<false>(o, whole, [&] { d.load_page_k(o, p, codes_at, scales_at); }, [&] { d.load_page_v(o, p, codes_at, scales_at); });
            } while (left != 0);
        }
        if (total != 0) {
            typename Decoder<kFormat, kDim>::Ops o;
            uint32_t there_of[2];
            d.load_groups_k(o, groups, min(8u, total), P.heads, h);
            d.load_groups_v(o, groups, min(8u, total), P.heads, h, there_of);
            for (uint32_t k = 0; k < total; k += 8) {
                uint32_t const n = k + 8;
                d.template add<true>(o, there_of,
                    [&] { if (n < total) d.load_groups_k(o, groups + n, min(8u, total - n), P.heads, h); },
                    [&] { if (n < total) d.load_groups_v(o, groups + n, min(8u, total - n), P.heads, h, there_of); });
            }
        }
        // The last entry read decides whether there are more.
        uint32_t const last = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(there ? begin : 0xFFFFFFFFu), 63));
        if (last >= t1) break;
        idx += kWave;
        __builtin_amdgcn_wave_barrier();
    }
    return d.part();
}

// ---- joining parts -------------------------------------------------------------

// What part (m, l) weighs beside the highest reference.
__device__ inline float part_weight(float m, float top) { return __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.0f : top)); }

// sum / l as fp16; 0 where no token had a weight.  A row's largest code times its
// scale can be past fp16's largest number (read_back), and so can this: it stays
// there, and NaN stays NaN.
__device__ inline uint16_t quotient_half(float sum, float l)
{
    float v = l == 0.0f ? 0.0f : sum / l;
    v = v > 65504.0f ? 65504.0f : v;
    v = v < -65504.0f ? -65504.0f : v;
    return __half_as_ushort(__float2half_rn(v));
}

// ---------------------------------------------------------------------------
// General path: any head dim, any group, any table.  One query head at a time;
// lanes own tokens for scores and dims for sums.  Bound by its loads of a byte,
// of the whole cache for each query head: 64 lanes of 2000 tokens, 4 heads of 256
// with 8 query heads each, take 5.2 ms, of 64 with 32 4.4 ms.
// ---------------------------------------------------------------------------
struct WaveTokens {
    float p[kWave];
    float scale[kWave];
    const uint8_t* v[kWave];   // V codes of dim 0
    uint32_t cap[kWave];
};

struct GeneralLds {
    WaveTokens tokens[kWaves];
    float sum[kWaves][kQuantMaxDim];
    float m[kWaves];
    float l[kWaves];
};

template <uint32_t kFormat>
__device__ void decode_general(const QuantView& P, const kimkv_decode_item& item, const QuantUnit& unit, uint32_t G, float* slot,
                               GeneralLds& lds)
{
    uint32_t const tid = threadIdx.x;
    uint32_t const lane = tid & (kWave - 1);
    uint32_t const wave = tid / kWave;
    uint32_t const D = P.dim;
    uint32_t const h = unit.head;
    uint32_t const end = unit.first + unit.count;
    float const scale2 = item.attention_scale * kLog2e;
    WaveTokens& tokens = lds.tokens[wave];
    for (uint32_t j = 0; j < G; ++j) {
        const uint16_t* const query = item.query + (static_cast<uint64_t>(h) * G + j) * D;
        float m = -INFINITY;
        float l = 0.0f;
        float acc[kQuantMaxDim / kWave] = {};
        for (uint32_t t0 = unit.first + wave * kWave; t0 < end; t0 += kBlock) {
            uint32_t const t = t0 + lane;
            // The last entry that begins at or before the token.
            uint32_t lo = 0, hi = item.descriptor_count;
            while (hi - lo > 1) {
                uint32_t const mid = lo + (hi - lo) / 2;
                if (item.descriptors[mid].logical_token_begin <= t) lo = mid; else hi = mid;
            }
            kimkv_block_desc const entry = item.descriptors[lo];
            uint32_t const cap = entry.page_token_capacity;
            bool const covered = t < end && entry.logical_token_begin <= t && t - entry.logical_token_begin < entry.valid_tokens;
            uint8_t* block = nullptr;
            if (covered && entry.valid_tokens <= cap) block = quant_block(P, item.layer, entry.kind, entry.slot, cap);
            if (covered && block == nullptr && P.faults != nullptr) atomicOr(P.faults, KIMKV_FAULT_DECODE_ITEM);
            float s = -INFINITY;
            tokens.scale[lane] = 0.0f;
            if (block != nullptr) {
                uint32_t const pt = t - entry.logical_token_begin;
                const uint8_t* const codes = quant_codes(block, P, cap, h);
                const uint16_t* const scales = quant_scales(block, P, cap, h);
                float dot = 0.0f;
                for (uint32_t d = 0; d < D; ++d) {
                    dot += __half2float(__ushort_as_half(query[d])) * code_value<kFormat>(codes[quant_k_at(cap, D, pt, d)]);
                }
                s = dot * (scale_value(scales[pt]) * scale2);
                tokens.scale[lane] = scale_value(scales[cap + pt]);
                tokens.v[lane] = codes + quant_v_at(cap, D, pt, 0);
                tokens.cap[lane] = cap;
            }
            float const m_new = fmaxf(m, wave_max(s));
            float const m_top = m_new == -INFINITY ? 0.0f : m_new;
            float const alpha = __builtin_amdgcn_exp2f(m - m_top);
            float const p = block != nullptr ? __builtin_amdgcn_exp2f(s - m_top) : 0.0f;
            m = m_new;
            l = l * alpha + wave_sum(p);
            tokens.p[lane] = p;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (uint32_t k = 0; k < kQuantMaxDim / kWave; ++k) acc[k] = alpha == 0.0f ? 0.0f : acc[k] * alpha;
            for (uint32_t i = 0; i < kWave; ++i) {
                float const w = tokens.p[i];
                if (w == 0.0f) continue;
                float const b = w * tokens.scale[i];
#pragma unroll
                for (uint32_t k = 0; k < kQuantMaxDim / kWave; ++k) {
                    uint32_t const d = lane + k * kWave;
                    if (d < D) acc[k] += b * code_value<kFormat>(tokens.v[i][d * tokens.cap[i]]);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
#pragma unroll
        for (uint32_t k = 0; k < kQuantMaxDim / kWave; ++k) lds.sum[wave][lane + k * kWave] = acc[k];
        if (lane == 0) {
            lds.m[wave] = m;
            lds.l[wave] = l;
        }
        __syncthreads();
        float top = -INFINITY;
        for (uint32_t w = 0; w < kWaves; ++w) top = fmaxf(top, lds.m[w]);
        float sum = 0.0f, total = 0.0f;
        for (uint32_t w = 0; w < kWaves; ++w) {
            float const f = part_weight(lds.m[w], top);
            total += lds.l[w] * f;
            if (f != 0.0f) sum += lds.sum[w][tid] * f;
        }
        if (tid < D) {
            if (slot == nullptr) {
                item.output[(static_cast<uint64_t>(h) * G + j) * D + tid] = quotient_half(sum, total);
            } else {
                slot[static_cast<uint64_t>(j) * D + tid] = sum;
                if (tid == 0) {
                    slot[static_cast<uint64_t>(G) * D + 2 * j] = top;
                    slot[static_cast<uint64_t>(G) * D + 2 * j + 1] = total;
                }
            }
        }
        __syncthreads();
    }
}

template <uint32_t kDim, uint32_t kOf>
struct FastLds {
    union {
        Group groups[kOf][kMaxGroups];
        float sum[kOf][kColumns][kDim + 4];
    };
    float m[kOf][kColumns];
    float l[kOf][kColumns];
};

// kDim 0: the general path alone.  kOf: waves of a block.
template <uint32_t kFormat, uint32_t kDim, uint32_t kOf>
__global__ __launch_bounds__(kOf * kWave, 2 * kWaves / kOf) void quant_decode_kernel(QuantView P, DecodeArgs a)
{
    static_assert(kDim != 0 || kOf == kWaves, "the general path's LDS is for kWaves");
    constexpr size_t kFast = kDim != 0 ? sizeof(FastLds<kDim == 0 ? 64 : kDim, kOf>) : 0;
    __shared__ alignas(16) unsigned char lds[kFast > sizeof(GeneralLds) ? kFast : sizeof(GeneralLds)];
    QuantUnit const unit = a.units[blockIdx.x];
    kimkv_decode_item const item = a.items[unit.lane];
    if (!item_good(P, item, unit.tokens)) {
        report_fault(P, KIMKV_FAULT_DECODE_ITEM);
        return;
    }
    uint32_t const G = a.G;
    float* const slot = unit.slot == kDirect ? nullptr : a.work + unit.slot * slot_floats(G, P.dim);
    if constexpr (kDim != 0) {
        auto& f = *reinterpret_cast<FastLds<kDim, kOf>*>(lds);
        uint32_t const tid = threadIdx.x;
        uint32_t const lane = tid & (kWave - 1);
        uint32_t const wave = tid / kWave;
        uint32_t const end = unit.first + unit.count;
        uint32_t const per = ((unit.count + kTile - 1) / kTile + kOf - 1) / kOf * kTile;
        uint32_t const t0 = min(unit.first + wave * per, end);
        bool bad = false;
        WavePart<kDim> const part = decode_wave<kFormat, kDim>(P, item, unit.head, G, t0, min(t0 + per, end), unit.tokens, f.groups[wave], &bad);
        if (bad && lane == 0 && P.faults != nullptr) atomicOr(P.faults, KIMKV_FAULT_DECODE_ITEM);
        __syncthreads();   // every wave is done with its groups
        {
            uint32_t const g = lane >> 4;
            uint32_t const r = lane & 15u;
#pragma unroll
            for (uint32_t db = 0; db < kDim / 16; ++db) *reinterpret_cast<float4_t*>(&f.sum[wave][r][16 * db + 4 * g]) = part.acc[db];
            if (g == 0) {
                f.m[wave][r] = part.m;
                f.l[wave][r] = part.l;
            }
            __syncthreads();
            for (uint32_t i = tid; i < G * (kDim / 4); i += kOf * kWave) {
                uint32_t const j = i / (kDim / 4);
                uint32_t const d = (i - j * (kDim / 4)) * 4;
                float top = -INFINITY;
#pragma unroll
                for (uint32_t w = 0; w < kOf; ++w) top = fmaxf(top, f.m[w][j]);
                float4_t sum = {};
                float total = 0.0f;
#pragma unroll
                for (uint32_t w = 0; w < kOf; ++w) {
                    float const x = part_weight(f.m[w][j], top);
                    total += f.l[w][j] * x;
                    if (x != 0.0f) sum += *reinterpret_cast<const float4_t*>(&f.sum[w][j][d]) * x;
                }
                if (slot == nullptr) {
                    uint16_t* const out = item.output + (static_cast<uint64_t>(unit.head) * G + j) * kDim + d;
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) out[k] = quotient_half(sum[k], total);
                } else {
                    // A slot of an odd number of floats, so no vector store.
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) slot[j * kDim + d + k] = sum[k];
                    if (d == 0) {
                        slot[G * kDim + 2 * j] = top;
                        slot[G * kDim + 2 * j + 1] = total;
                    }
                }
            }
        }
    } else {
        decode_general<kFormat>(P, item, unit, G, slot, *reinterpret_cast<GeneralLds*>(lds));
    }
}

// Block = (merged lane, KV head, kBlock of its values): a thread a value, the
// parts eight at a time in flight.
__global__ __launch_bounds__(kBlock) void quant_merge_kernel(QuantView P, const kimkv_decode_item* items, const QuantMerge* merges,
                                                             const float* work, uint32_t G)
{
    constexpr uint32_t kAtOnce = 8;
    QuantMerge const x = merges[blockIdx.x];
    kimkv_decode_item const item = items[x.lane];
    uint32_t const D = P.dim;
    uint32_t const h = blockIdx.y;
    uint64_t const size = slot_floats(G, D);
    for (uint32_t i = blockIdx.z * kBlock + threadIdx.x; i < G * D; i += gridDim.z * kBlock) {
        const float* const values = work + (x.first_slot + static_cast<uint64_t>(h) * x.parts) * size + i;
        const float* const ml = values - i + static_cast<uint64_t>(G) * D + 2 * (i / D);
        float m = -INFINITY, total = 0.0f, sum = 0.0f;
        for (uint32_t p = 0; p < x.parts; p += kAtOnce) {
            float top[kAtOnce], l[kAtOnce], v[kAtOnce];
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce; ++k) {
                uint64_t const at = min(p + k, x.parts - 1) * size;
                top[k] = ml[at];
                l[k] = ml[at + 1];
                v[k] = values[at];
            }
            float most = m;
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce; ++k) most = fmaxf(most, top[k]);
            float const f = part_weight(m, most);
            sum = f != 0.0f ? sum * f : 0.0f;
            total *= f;
            m = most;
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce; ++k) {
                float const w = p + k < x.parts ? part_weight(top[k], most) : 0.0f;
                total += l[k] * w;
                if (w != 0.0f) sum += v[k] * w;
            }
        }
        // An item that is not as planned is reported by its units, which wrote no parts.
        if (item_good(P, item, x.tokens)) item.output[static_cast<uint64_t>(h) * G * D + i] = quotient_half(sum, total);
    }
}

// ---- plan ------------------------------------------------------------------------

// Parts of a lane of `tiles` tiles when a unit takes at most `most` of them.
inline uint32_t lane_parts(uint32_t tiles, uint32_t most) { return (tiles + most - 1) / most; }

constexpr uint32_t kGridRows = 65535;       // of a launch's third dimension
constexpr uint32_t kMostUnits = 0xFFFFFF;   // times kBlock threads: fewer than 2^32

}  // namespace
}  // namespace kimkv

using namespace kimkv;

extern "C" {

kimkv_status kimkv_quant_decode_plan(uint32_t kv_heads, uint32_t head_dim, uint32_t query_heads, uint32_t compute_units,
                                     const uint32_t* token_counts, uint32_t lane_count, void* entries, uint64_t capacity,
                                     kimkv_quant_plan* plan)
{
    if (plan == nullptr) return KIMKV_INVALID_ARGUMENT;
    *plan = kimkv_quant_plan{};
    if (kv_heads == 0 || kv_heads > 65535 || lane_count > kMostUnits || head_dim == 0 || head_dim > kQuantMaxDim || query_heads == 0 || query_heads % kv_heads != 0
        || static_cast<uint64_t>(query_heads) * head_dim > 0x7FFFFFFFull || (lane_count != 0 && token_counts == nullptr)
        || (capacity != 0 && entries == nullptr)) {
        return KIMKV_INVALID_ARGUMENT;
    }
    uint32_t const G = query_heads / kv_heads;
    uint64_t const slots = 2ull * (compute_units == 0 ? 256 : compute_units);   // units that run at once
    uint64_t tiles = 0;
    uint32_t longest = 0;
    for (uint32_t i = 0; i < lane_count; ++i) {
        if (token_counts[i] >= 0x80000000u) return KIMKV_INVALID_ARGUMENT;
        uint32_t const n = (token_counts[i] + kTile - 1) / kTile;
        tiles += n;
        longest = n > longest ? n : longest;
    }
    // The tiles of a unit: as many as make two units for each place, which evens
    // out lanes that do not divide (one a place, 128 equal lanes of 32768 tokens:
    // 345 us, not 353), 16 at least (8, 64 lanes of up to 6000: 31 us, not 29).
    uint64_t most = tiles / (2 * slots) * kv_heads + tiles % (2 * slots) * kv_heads / (2 * slots);
    most = most < 16 ? 16 : most;
    most = most > longest && longest != 0 ? longest : most;
    auto const counted = [&](uint64_t* units, uint64_t* parts, uint64_t* merges) {
        *units = *parts = *merges = 0;
        for (uint32_t i = 0; i < lane_count; ++i) {
            if (token_counts[i] == 0) continue;
            uint64_t const n = lane_parts((token_counts[i] + kTile - 1) / kTile, static_cast<uint32_t>(most));
            *units += n * kv_heads;
            if (n > 1) {
                *parts += n * kv_heads;
                *merges += 1;
            }
        }
    };
    uint64_t units, parts, merges;
    counted(&units, &parts, &merges);
    while (units > kMostUnits && most < longest) {
        most = most * 2 < longest ? most * 2 : longest;
        counted(&units, &parts, &merges);
    }
    if (units > kMostUnits) return KIMKV_INVALID_ARGUMENT;
    plan->entry_bytes = units * sizeof(QuantUnit) + merges * sizeof(QuantMerge);
    plan->workspace_bytes = parts * slot_floats(G, head_dim) * sizeof(float);
    plan->kv_heads = kv_heads;
    plan->head_dim = head_dim;
    plan->query_heads = query_heads;
    plan->lane_count = lane_count;
    plan->unit_count = static_cast<uint32_t>(units);
    plan->slot_count = static_cast<uint32_t>(parts);
    plan->merge_lanes = static_cast<uint32_t>(merges);
    if (plan->entry_bytes > capacity) return KIMKV_INVALID_ARGUMENT;
    auto* const unit = static_cast<QuantUnit*>(entries);
    auto* const merge = reinterpret_cast<QuantMerge*>(unit + units);
    uint64_t u = 0, m = 0;
    uint32_t slot = 0;
    for (uint32_t i = 0; i < lane_count; ++i) {
        uint32_t const tokens = token_counts[i];
        if (tokens == 0) continue;
        uint32_t const n = (tokens + kTile - 1) / kTile;
        uint32_t const count = lane_parts(n, static_cast<uint32_t>(most));
        if (count > 1) merge[m++] = QuantMerge{i, tokens, slot, count};
        for (uint32_t h = 0; h < kv_heads; ++h) {
            for (uint32_t p = 0; p < count; ++p) {
                auto const tile = [&](uint32_t k) { return static_cast<uint32_t>(static_cast<uint64_t>(n) * k / count); };
                uint32_t const first = tile(p) * kTile;
                uint32_t const end = p + 1 == count ? tokens : tile(p + 1) * kTile;
                unit[u++] = QuantUnit{i, h, first, end - first, tokens, count > 1 ? slot++ : kDirect, {0, 0}};
            }
        }
    }
    std::sort(unit, unit + units, [](const QuantUnit& a, const QuantUnit& b) {
        return a.count != b.count ? a.count > b.count : a.lane != b.lane ? a.lane < b.lane : a.head != b.head ? a.head < b.head : a.first < b.first;
    });
    return KIMKV_OK;
}

kimkv_status kimkv_quant_decode_batch(const kimkv_quant_storage* storage, const kimkv_decode_item* device_items,
                                      const void* device_entries, const kimkv_quant_plan* plan, void* workspace,
                                      kimkv_stream_t stream)
{
    int device = -1;
    if (storage == nullptr || plan == nullptr || plan->kv_heads != storage->layout.kv_heads || plan->head_dim != storage->layout.head_dim
        || plan->query_heads == 0 || plan->query_heads % plan->kv_heads != 0 || plan->unit_count > kMostUnits
        || plan->entry_bytes != plan->unit_count * sizeof(QuantUnit) + plan->merge_lanes * sizeof(QuantMerge)
        || hipGetDevice(&device) != hipSuccess || device != storage->device) {
        return KIMKV_INVALID_ARGUMENT;
    }
    uint32_t const G = plan->query_heads / plan->kv_heads;
    if (plan->workspace_bytes != plan->slot_count * slot_floats(G, plan->head_dim) * sizeof(float)) return KIMKV_INVALID_ARGUMENT;
    if (plan->unit_count == 0) return KIMKV_OK;
    auto const aligned = [](const void* p) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    if (device_items == nullptr || !aligned(device_entries) || (plan->workspace_bytes != 0 && !aligned(workspace))) return KIMKV_INVALID_ARGUMENT;
    QuantView const view = quant_view(*storage);
    auto const* const units = static_cast<const QuantUnit*>(device_entries);
    DecodeArgs const args{device_items, units, static_cast<float*>(workspace), G};
    // A unit for a compute unit or less: twice the waves, as there is room for them
    // (16 lanes of 1000 tokens, 4 heads of 64: 10.7 us, not 12.1).
    bool const few = plan->unit_count <= static_cast<uint32_t>(storage->compute_units);
    auto const launch = [&](auto kernel, uint32_t waves) { kernel<<<plan->unit_count, waves * kWave, 0, native(stream)>>>(view, args); };
    auto const launch_dim = [&](auto format, auto dim) {
        if (few) {
            launch(quant_decode_kernel<format.value, dim.value, 2 * kWaves>, 2 * kWaves);
        } else {
            launch(quant_decode_kernel<format.value, dim.value, kWaves>, kWaves);
        }
    };
    auto const launch_format = [&](auto format) {
        switch (fast_dim(view.dim) && G <= kColumns ? view.dim : 0) {
        case 64: launch_dim(format, std::integral_constant<uint32_t, 64>{}); break;
        case 96: launch_dim(format, std::integral_constant<uint32_t, 96>{}); break;
        case 128: launch_dim(format, std::integral_constant<uint32_t, 128>{}); break;
        default: launch(quant_decode_kernel<format.value, 0, kWaves>, kWaves); break;
        }
    };
    void* start = nullptr;
    kernel_timing_begin(TimedKernel::Decode, native(stream), &start);
    if (storage->format == KIMKV_QUANT_INT8) {
        launch_format(std::integral_constant<uint32_t, KIMKV_QUANT_INT8>{});
    } else {
        launch_format(std::integral_constant<uint32_t, KIMKV_QUANT_E4M3>{});
    }
    kimkv_status const status = launch_status();
    kernel_timing_end(TimedKernel::Decode, native(stream), start);
    if (status != KIMKV_OK || plan->merge_lanes == 0) return status;
    quant_merge_kernel<<<dim3(plan->merge_lanes, plan->kv_heads, std::min((G * view.dim + kBlock - 1) / kBlock, kGridRows)), kBlock, 0, native(stream)>>>(
        view, device_items, reinterpret_cast<const QuantMerge*>(units + plan->unit_count), args.work, G);
    return launch_status();
}

}  // extern "C"
