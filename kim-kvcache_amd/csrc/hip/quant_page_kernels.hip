// quant_page_kernels.hip -- a cache in 8 bits: its storage, append (with fused
// partial-tail copy-on-write), read-back and promotion.  Formats and layout:
// quant_common.h.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <limits>
#include <mutex>
#include <new>
#include <type_traits>

#include "quant_common.h"
#include "runtime_internal.h"

namespace kimkv {
namespace {

constexpr unsigned kBlock = 256;
constexpr uint32_t kTileTokens = kQuantMaxPage;
constexpr uint32_t kGatherAtOnce = 2;
constexpr uint32_t kAtOnce = 4;   // loads of a thread in flight

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

// Bytes (r, c) of four words, byte c of word r, as four words, byte r of word c.
__device__ inline void transpose_bytes(uint32_t (&w)[4])
{
    uint32_t const t0 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u);
    uint32_t const t1 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
    uint32_t const u0 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
    uint32_t const u1 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    w[0] = __builtin_amdgcn_perm(u0, t0, 0x05040100u);
    w[1] = __builtin_amdgcn_perm(u0, t0, 0x07060302u);
    w[2] = __builtin_amdgcn_perm(u1, t1, 0x05040100u);
    w[3] = __builtin_amdgcn_perm(u1, t1, 0x07060302u);
}

__device__ inline float half_value(uint16_t bits) { return __half2float(__ushort_as_half(bits)); }

// Of the power of two that covers n: threads of a row of n pieces, for one.
inline uint32_t log2_of(uint32_t n)
{
    uint32_t log2 = 0;
    while ((1u << log2) < n) ++log2;
    return log2;
}

struct AppendGrid {
    uint32_t heads_log2;   // of a block
    uint32_t lanes_log2;   // of a row
};

// ---------------------------------------------------------------------------
// Append: block = (job, layer, some heads).  A job of fewer than 8 tokens, or
// of rows off 16 bytes, writes V byte by byte; others turn V's codes in LDS.
// Bound by HBM where jobs are many, with operations close behind (113 a piece of
// 8 values kept the units busy for 0.56 of 130 us), so divisions, fallbacks and
// index arithmetic are kept out of the way; a step of 128 lanes is its launch.
// ---------------------------------------------------------------------------
// Tokens [0, n) of one head of a page's block copied to another page, byte for
// byte: the codes and the scales of each.  Only those tokens' bytes are stored:
// others may be writing behind them.
__device__ inline void copy_head(const uint8_t* src, const uint16_t* src_scales, uint32_t scap, uint8_t* dst, uint16_t* dst_scales,
                                 uint32_t dcap, uint32_t D, uint32_t n)
{
    uint32_t const tid = threadIdx.x;
    uint32_t const kw = quant_k_width(D);
    uint32_t const run = n * kw;   // contiguous in both, for each column block
    if (D % 8u == 0) {
        for (uint32_t i = tid * 8; i < n * D; i += kBlock * 8) {
            uint32_t const b = i / run;
            uint32_t const o = i - b * run;
            *reinterpret_cast<u32x2_t*>(dst + b * dcap * kw + o) = *reinterpret_cast<const u32x2_t*>(src + b * scap * kw + o);
        }
    } else {
        for (uint32_t i = tid; i < run; i += kBlock) dst[i] = src[i];
    }
    uint32_t const groups = (n + 7) / 8;
    for (uint32_t i = tid; i < groups * D; i += kBlock) {
        uint32_t const d = i / groups;
        uint32_t const t = (i - d * groups) * 8;
        const uint8_t* from = src + quant_v_at(scap, D, t, d);
        uint8_t* to = dst + quant_v_at(dcap, D, t, d);
        u32x2_t const v = *reinterpret_cast<const u32x2_t*>(from);
        if (n - t >= 8) {
            *reinterpret_cast<u32x2_t*>(to) = v;
        } else {
            for (uint32_t j = 0; j < n - t; ++j) to[j] = static_cast<uint8_t>(v[j >> 2] >> (8 * (j & 3)));
        }
    }
    for (uint32_t i = tid; i < n; i += kBlock) {
        dst_scales[i] = src_scales[i];
        dst_scales[dcap + i] = src_scales[scap + i];
    }
}

// Dims [8 p, 8 p + 8) of a row of D, zeros past its end.
__device__ inline u32x4_t load_piece(const uint16_t* row, uint32_t p, uint32_t D, bool aligned)
{
    u32x4_t w = {};
    if (aligned && 8 * p + 8 <= D) {
        w = *reinterpret_cast<const u32x4_t*>(row + 8 * p);
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            if (8 * p + j < D) w[j >> 1] |= static_cast<uint32_t>(row[8 * p + j]) << (16 * (j & 1));
        }
    }
    return w;
}

// Of what is read once, lines at a time: past the caches.  Appended rows and V's
// codes so, and read-back rows written so: 6 layers of 4 x 4096 tokens, 8 heads of
// 128, appended and read back in 186 us, not 246, the same tensors every time (212
// with others each time, 5.3 TB/s).  With K's codes so too, 199: a wave reads them
// in pieces of 64 bytes.
__device__ inline u32x4_t load_once(const void* p) { return __builtin_nontemporal_load(static_cast<const u32x4_t*>(p)); }

// The largest of the lanes of a row, 2^log2 neighbours.
__device__ inline uint32_t row_largest(uint32_t v, uint32_t lanes)
{
    auto const turned = [&](auto control) {
        return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), decltype(control)::value, 0xF, 0xF, false));
    };
    if (lanes > 1) v = max(v, turned(std::integral_constant<int, 0xB1>{}));    // the neighbour
    if (lanes > 2) v = max(v, turned(std::integral_constant<int, 0x4E>{}));    // the pair beside
    if (lanes > 4) v = max(v, turned(std::integral_constant<int, 0x141>{}));   // eight, turned round
    if (lanes > 8) v = max(v, turned(std::integral_constant<int, 0x140>{}));   // sixteen
    if (lanes > 16) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 16)));
    return v;
}

// Codes of a piece, and the row's scale; the row's other pieces are in the
// other threads of its group.
template <uint32_t kFormat>
__device__ inline u32x2_t quantise_piece(u32x4_t w, uint32_t lanes, uint16_t* scale)
{
    u16x2_t top = {0, 0};   // two fp16 numbers without sign, ordered as whole numbers
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        uint32_t const pair = w[j] & 0x7FFF7FFFu;
        top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, pair));
    }
    *scale = row_scale<kFormat>(row_largest(top[0] > top[1] ? top[0] : top[1], lanes));
    RowQuant const r = row_quant(*scale);
    u32x2_t codes;
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
        float const x[4] = {half_value(static_cast<uint16_t>(w[2 * j])), half_value(static_cast<uint16_t>(w[2 * j] >> 16)),
                            half_value(static_cast<uint16_t>(w[2 * j + 1])), half_value(static_cast<uint16_t>(w[2 * j + 1] >> 16))};
        codes[j] = row_codes<kFormat>(x, r);
    }
    if (__ballot(*scale == kScaleNan) != 0 && *scale == kScaleNan) codes = u32x2_t{no_codes<kFormat>(), no_codes<kFormat>()};
    return codes;
}

__device__ inline void store_key_piece(uint8_t* at, u32x2_t codes, uint32_t p, uint32_t D)
{
    if (D % 8u == 0) {
        *reinterpret_cast<u32x2_t*>(at) = codes;
    } else {
        for (uint32_t j = 0; j < 8 && 8 * p + j < D; ++j) at[j] = static_cast<uint8_t>(codes[j >> 2] >> (8 * (j & 3)));
    }
}

// kDim 0: any head dim.
template <uint32_t kFormat, uint32_t kDim>
__global__ __launch_bounds__(kBlock) void quant_append_kernel(QuantView P, const kimkv_append_job* jobs, AppendGrid g)
{
    __shared__ alignas(16) uint8_t tile[kTileTokens * (kQuantMaxDim + 4)];   // V codes of the heads' tokens
    kimkv_append_job const job = jobs[blockIdx.x];
    if (blockIdx.y >= job.layer_count) return;   // a shorter job of a launch sized for the longest
    uint32_t const layer = job.layer_begin + blockIdx.y;
    uint32_t const D = kDim != 0 ? kDim : P.dim;
    uint32_t const n = job.token_count;
    uint32_t const dcap = quant_page_tokens(P, job.dst_kind);
    uint32_t const scap = quant_page_tokens(P, job.cow_kind);
    uint8_t* const dst = quant_block(P, layer, job.dst_kind, job.dst_slot, dcap);
    uint8_t* const src = job.cow_tokens != 0 ? quant_block(P, layer, job.cow_kind, job.cow_slot, scap) : nullptr;
    // Each block judges the job's whole range of layers, so that a bad one is skipped in all of them.
    if (job.layer_begin >= P.layers || job.layer_count > P.layers - job.layer_begin || job.layer_count > gridDim.y || dst == nullptr
        || n > dcap || job.dst_token > dcap - n
        || (n != 0 && (job.src_key == nullptr || job.src_value == nullptr))
        || (job.cow_tokens != 0 && (src == nullptr || job.cow_tokens > scap || job.cow_tokens > job.dst_token))) {
        report_fault(P, KIMKV_FAULT_APPEND_JOB);
        return;
    }
    uint32_t const tid = threadIdx.x;
    uint32_t const h0 = blockIdx.z << g.heads_log2;
    uint32_t const h1 = min(h0 + (1u << g.heads_log2), P.heads);

    // The copied positions lie below the written ones: neither waits for the other.
    for (uint32_t h = h0; job.cow_tokens != 0 && h < h1; ++h) {
        copy_head(quant_codes(src, P, scap, h), quant_scales(src, P, scap, h), scap, quant_codes(dst, P, dcap, h),
                  quant_scales(dst, P, dcap, h), dcap, D, job.cow_tokens);
    }
    if (n == 0) return;

    uint64_t const layer_off = static_cast<uint64_t>(blockIdx.y) * job.src_layer_stride;
    const uint16_t* const sk = job.src_key + layer_off;
    const uint16_t* const sv = job.src_value + layer_off;
    uint64_t const stride = job.src_token_stride;
    bool const aligned = ((D | stride) & 7u) == 0 && ((reinterpret_cast<uintptr_t>(sk) | reinterpret_cast<uintptr_t>(sv)) & 15u) == 0;
    uint32_t const lanes_log2 = kDim == 64 ? 3 : kDim == 128 ? 4 : g.lanes_log2;
    uint32_t const lanes = 1u << lanes_log2;
    uint32_t const p = tid & (lanes - 1);          // piece of the row
    uint32_t const first = tid >> lanes_log2;
    uint32_t const step = kBlock >> lanes_log2;
    bool const mine = 8 * p < D;
    uint32_t const t0 = job.dst_token;

    if (n < 8 || (kDim != 0 && !aligned)) {
        // A token step: K and V rows of all heads at once, V byte by byte.
        uint32_t const rows = 2 * n * (h1 - h0);
        for (uint32_t base = 0; base < rows; base += step) {
            uint32_t const i = base + first;
            bool const there = i < rows && mine;
            uint32_t const row = min(i, rows - 1);
            uint32_t const h = h0 + row / (2 * n);
            uint32_t const rem = row % (2 * n);
            bool const value = rem >= n;
            uint32_t const t = value ? rem - n : rem;
            u32x4_t w = {};
            if (there) w = load_piece((value ? sv : sk) + t * stride + static_cast<uint64_t>(h) * D, p, D, aligned);
            uint16_t scale;
            u32x2_t const codes = quantise_piece<kFormat>(w, lanes, &scale);
            if (!there) continue;
            uint8_t* const at = quant_codes(dst, P, dcap, h);
            if (p == 0) quant_scales(dst, P, dcap, h)[(value ? dcap : 0) + t0 + t] = scale;
            if (!value) {
                store_key_piece(at + quant_k_at(dcap, D, t0 + t, 8 * p), codes, p, D);
            } else {
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) {
                    if (8 * p + j < D) at[quant_v_at(dcap, D, t0 + t, 8 * p + j)] = static_cast<uint8_t>(codes[j >> 2] >> (8 * (j & 3)));
                }
            }
        }
        return;
    }

    // Rows of all the block's heads, a token's side by side as they are in the source.
    uint32_t const heads = h1 - h0;
    uint32_t const pitch = (D << g.heads_log2) + 4;   // heads of a block: at most kQuantMaxDim dims
    uint32_t const g0 = t0 / 8;                       // groups of 8 page tokens that the job touches
    uint32_t const groups = (t0 + n + 7) / 8 - g0;
    uint32_t const rows = (2 * n) << g.heads_log2;
    for (uint32_t base = 0; base < rows; base += kAtOnce * step) {
        u32x4_t w[kAtOnce];
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k) {
            uint32_t const i = base + first + k * step;
            uint32_t const h = i & ((1u << g.heads_log2) - 1);
            uint32_t const t = i >> g.heads_log2;
            w[k] = u32x4_t{};
            if (t >= 2 * n || h >= heads || !mine) continue;
            const uint16_t* const row = (t >= n ? sv + (t - n) * stride : sk + t * stride) + (h0 + h) * D;
            w[k] = kDim != 0 ? load_once(row + 8 * p) : load_piece(row, p, D, aligned);
        }
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k) {
            if (base + k * step >= rows) break;
            uint32_t const i = base + first + k * step;
            uint32_t const h = i & ((1u << g.heads_log2) - 1);
            bool const value = i >> g.heads_log2 >= n;
            uint32_t const t = (i >> g.heads_log2) - (value ? n : 0);
            uint16_t scale;
            u32x2_t const codes = quantise_piece<kFormat>(w[k], lanes, &scale);
            if (t >= n || h >= heads || !mine) continue;
            if (p == 0) quant_scales(dst, P, dcap, h0 + h)[(value ? dcap : 0) + t0 + t] = scale;
            if (!value) {
                store_key_piece(quant_codes(dst, P, dcap, h0 + h) + quant_k_at(dcap, D, t0 + t, 8 * p), codes, p, D);
            } else {
                // Row t0 % 8 + t of the tile, so that its groups of 8 are the page's.
                uint8_t* const row = tile + ((t0 & 7u) + t) * pitch + h * D + 8 * p;
                if (D % 8u == 0) {
                    reinterpret_cast<uint32_t*>(row)[0] = codes[0];
                    reinterpret_cast<uint32_t*>(row)[1] = codes[1];
                } else {
                    store_key_piece(row, codes, p, D);
                }
            }
        }
    }
    __syncthreads();
    auto const row_of = [&](uint32_t gi, uint32_t j) { return tile + (8 * gi + j) * pitch; };
    if (D % 8u == 0) {
        for (uint32_t i = tid; i < groups * heads * (D / 4); i += kBlock) {
            uint32_t const q = i / groups;
            uint32_t const gi = i - q * groups;
            uint32_t const h = 4 * q / D;
            uint32_t const t = 8 * (g0 + gi);
            uint32_t lo[4], hi[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                lo[j] = *reinterpret_cast<const uint32_t*>(row_of(gi, j) + 4 * q);
                hi[j] = *reinterpret_cast<const uint32_t*>(row_of(gi, j + 4) + 4 * q);
            }
            transpose_bytes(lo);
            transpose_bytes(hi);
            bool const whole = t >= t0 && t + 8 <= t0 + n;
            uint8_t* const codes_at = quant_codes(dst, P, dcap, h0 + h) + quant_v_at(dcap, D, t, 4 * q - h * D);
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                uint8_t* const at = codes_at + k * dcap;
                if (whole) {
                    *reinterpret_cast<u32x2_t*>(at) = u32x2_t{lo[k], hi[k]};
                } else {
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j) {
                        uint32_t const word = j < 4 ? lo[k] : hi[k];
                        if (t + j >= t0 && t + j < t0 + n) at[j] = static_cast<uint8_t>(word >> (8 * (j & 3)));
                    }
                }
            }
        }
    } else {
        for (uint32_t i = tid; i < n * heads * D; i += kBlock) {
            uint32_t const d = i / n;
            uint32_t const t = i - d * n;
            uint32_t const h = d / D;
            quant_codes(dst, P, dcap, h0 + h)[quant_v_at(dcap, D, t0 + t, d - h * D)] = tile[((t0 & 7u) + t) * pitch + d];
        }
    }
}

// ---------------------------------------------------------------------------
// Read-back: block = (table entry, layer, some heads).  V's codes are turned in
// LDS, and rows of up to 256 dims written whole: head after head, 22 layers of
// 16384 tokens of 4 heads of 64 took 123 us with rows through the caches and 137
// a head at a time; 100 us now, all of the same pages every time, and 107 of
// others each time, 5.2 TB/s.
// ---------------------------------------------------------------------------
struct GatherArgs {
    const kimkv_block_desc* descriptors;
    uint16_t* out;
    uint32_t first;        // token
    uint32_t count;
    uint32_t layer_begin;
    uint32_t heads;        // of a block: at most kQuantMaxDim dims
    bool wide;             // rows of 16-byte pieces
};

// Rows that are written once and whole, past the caches.
__device__ inline void store_row(uint16_t* at, code_halves_t v) { __builtin_nontemporal_store(v, reinterpret_cast<code_halves_t*>(at)); }

// kDim 0: any head dim.
template <uint32_t kFormat, uint32_t kDim>
__global__ __launch_bounds__(kBlock) void quant_gather_kernel(QuantView P, GatherArgs a)
{
    __shared__ uint32_t tile[kQuantMaxDim * (kTileTokens / 4 + 1)];   // V codes of the heads' dims, rows of 17 words
    kimkv_block_desc const e = a.descriptors[blockIdx.x];
    uint64_t const begin = e.logical_token_begin;
    uint64_t const last = static_cast<uint64_t>(a.first) + a.count;
    if (begin >= last || begin + e.valid_tokens <= a.first) return;
    uint32_t const cap = e.page_token_capacity;
    uint32_t const layer = a.layer_begin + blockIdx.y;
    uint8_t* const block = e.valid_tokens <= cap ? quant_block(P, layer, e.kind, e.slot, cap) : nullptr;
    if (block == nullptr) {
        report_fault(P, KIMKV_FAULT_GATHER_ENTRY);
        return;
    }
    uint32_t const tid = threadIdx.x;
    uint32_t const D = kDim != 0 ? kDim : P.dim;
    uint32_t const HD = P.heads * D;
    // Page tokens [p0, p1), token p0 of which is row `to` of the output.
    uint32_t const p0 = begin < a.first ? static_cast<uint32_t>(a.first - begin) : 0;
    uint32_t const p1 = static_cast<uint32_t>(min<uint64_t>(e.valid_tokens, last - begin));
    uint32_t const n = p1 - p0;
    uint64_t const to = begin + p0 - a.first;
    uint16_t* const key_out = a.out + (static_cast<uint64_t>(blockIdx.y) * 2 * a.count + to) * HD;
    uint16_t* const value_out = key_out + static_cast<uint64_t>(a.count) * HD;
    uint32_t const h0 = blockIdx.z * a.heads;
    uint32_t const h1 = min(h0 + a.heads, P.heads);
    if (!a.wide) {
        for (uint32_t h = h0; h < h1; ++h) {
            const uint8_t* const codes = quant_codes(block, P, cap, h);
            const uint16_t* const scales = quant_scales(block, P, cap, h);
            for (uint32_t i = tid; i < n * D; i += kBlock) {
                uint32_t const t = i / D;
                uint32_t const d = i - t * D;
                uint64_t const o = static_cast<uint64_t>(t) * HD + h * D + d;
                key_out[o] = read_back(code_value<kFormat>(codes[quant_k_at(cap, D, p0 + t, d)]), scale_value(scales[p0 + t]));
                value_out[o] = read_back(code_value<kFormat>(codes[quant_v_at(cap, D, p0 + t, d)]), scale_value(scales[cap + p0 + t]));
            }
        }
        return;
    }
    // Tokens' rows of all the block's heads, side by side.  V codes into LDS, K in the meantime.
    uint32_t const pieces = D / 8;
    uint32_t const row = (h1 - h0) * pieces;
    uint32_t const eights = D * cap / 8;   // 8 codes each, of a head's V
    uint32_t const words = cap / 4;        // of a dim
    for (uint32_t base = tid; base < (h1 - h0) * eights || base < n * row; base += kGatherAtOnce * kBlock) {
        u32x2_t v[kGatherAtOnce], k[kGatherAtOnce];
        uint16_t s[kGatherAtOnce];
#pragma unroll
        for (uint32_t j = 0; j < kGatherAtOnce; ++j) {
            uint32_t const i = base + j * kBlock;
            if (i >= (h1 - h0) * eights) continue;
            uint32_t const h = i / eights;
            v[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x2_t*>(quant_codes(block, P, cap, h0 + h) + cap * D + 8 * (i - h * eights)));
        }
#pragma unroll
        for (uint32_t j = 0; j < kGatherAtOnce; ++j) {
            uint32_t const i = base + j * kBlock;
            if (i >= n * row) continue;
            uint32_t const t = i / row;
            uint32_t const h = (i - t * row) / pieces;
            uint32_t const piece = i - t * row - h * pieces;
            k[j] = *reinterpret_cast<const u32x2_t*>(quant_codes(block, P, cap, h0 + h) + quant_k_at(cap, D, p0 + t, 8 * piece));
            s[j] = quant_scales(block, P, cap, h0 + h)[p0 + t];
        }
#pragma unroll
        for (uint32_t j = 0; j < kGatherAtOnce; ++j) {
            uint32_t const i = base + j * kBlock;
            if (i >= (h1 - h0) * eights) continue;
            uint32_t const d = 2 * i / words;   // of all heads
            uint32_t* const to_row = tile + d * (kTileTokens / 4 + 1) + (2 * i - d * words);
            to_row[0] = v[j][0];
            to_row[1] = v[j][1];
        }
#pragma unroll
        for (uint32_t j = 0; j < kGatherAtOnce; ++j) {
            uint32_t const i = base + j * kBlock;
            if (i >= n * row) continue;
            uint32_t const t = i / row;
            store_row(key_out + static_cast<uint64_t>(t) * HD + h0 * D + 8 * (i - t * row), read_back<kFormat>(k[j], scale_value(s[j])));
        }
    }
    __syncthreads();
    // Four tokens by 8 dims a thread.
    uint32_t const q0 = p0 / 4;
    uint32_t const quads = (p1 + 3) / 4 - q0;
    for (uint32_t i = tid; i < quads * row; i += kBlock) {
        uint32_t const q = i / row;
        uint32_t const d = (i - q * row) * 8;   // of all heads
        const uint16_t* const scales = quant_scales(block, P, cap, h0 + d / D) + cap;
        uint32_t lo[4], hi[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            lo[j] = tile[(d + j) * (kTileTokens / 4 + 1) + q0 + q];
            hi[j] = tile[(d + 4 + j) * (kTileTokens / 4 + 1) + q0 + q];
        }
        transpose_bytes(lo);
        transpose_bytes(hi);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            uint32_t const t = 4 * (q0 + q) + k;
            if (t < p0 || t >= p1) continue;
            store_row(value_out + static_cast<uint64_t>(t - p0) * HD + h0 * D + d, read_back<kFormat>(u32x2_t{lo[k], hi[k]}, scale_value(scales[t])));
        }
    }
}

// ---------------------------------------------------------------------------
// Promotion: block = (job, layer, some heads).  Eight pages of 8 tokens into
// one of 64: K in runs of 8 tokens of a column block, V and the scales in
// pieces of 8 tokens.  512 jobs in 22 layers (0.8 GB moved) and their read-back
// (1.1 GB) take 331 us, the same pages every time, and 349 other ones; in pieces of
// 8 bytes 391 with the read-back of then.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(kBlock) void quant_promote_kernel(QuantView P, const kimkv_promotion_job* jobs, uint32_t heads)
{
    __shared__ const uint8_t* source[8];
    kimkv_promotion_job const& job = jobs[blockIdx.x];
    uint32_t const layer = blockIdx.y;
    uint32_t const tid = threadIdx.x;
    uint8_t* const dst = quant_block(P, layer, KIMKV_PAGE_EXTENT, job.extent_slot, 64);
    if (tid < 8) source[tid] = quant_block(P, layer, KIMKV_PAGE_MICRO, job.micro_slots[tid], 8);
    __syncthreads();
    bool good = dst != nullptr;
    for (uint32_t m = 0; m < 8; ++m) good = good && source[m] != nullptr;
    if (!good) {
        report_fault(P, KIMKV_FAULT_PROMOTION_JOB);
        return;
    }
    uint32_t const D = P.dim;
    uint32_t const kw = quant_k_width(D);
    uint32_t const run = 8 * kw;   // a micro page's column block
    uint32_t const h0 = blockIdx.z * heads;
    uint32_t const h1 = min(h0 + heads, P.heads);
    if (D % 2u == 0) {
        // 16 bytes at a time: of K a run's; of V two dims of two pages, which are two dims' of the page.
        uint32_t const pieces = D * 4;   // of a head's K; half as many of its V
        for (uint32_t base = tid; base < (h1 - h0) * pieces; base += kAtOnce * kBlock) {
            u32x4_t w[kAtOnce];
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce; ++k) {
                uint32_t const i = base + k * kBlock;
                if (i >= (h1 - h0) * pieces) continue;
                uint32_t const h = i / pieces;
                uint32_t const at = (i - h * pieces) * 16;
                uint32_t const b = at / (8 * run);
                uint32_t const m = at / run & 7u;
                w[k] = load_once(source[m] + static_cast<uint64_t>(h0 + h) * 16 * D + b * run + (at - (8 * b + m) * run));
            }
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce; ++k) {
                uint32_t const i = base + k * kBlock;
                if (i >= (h1 - h0) * pieces) continue;
                uint32_t const h = i / pieces;
                *reinterpret_cast<u32x4_t*>(quant_codes(dst, P, 64, h0 + h) + (i - h * pieces) * 16) = w[k];
            }
        }
        for (uint32_t base = tid; base < (h1 - h0) * pieces / 2; base += kAtOnce / 2 * kBlock) {
            u32x4_t w[kAtOnce / 2][2];
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce / 2; ++k) {
                uint32_t const i = base + k * kBlock;
                if (i >= (h1 - h0) * pieces / 2) continue;
                uint32_t const h = i / (pieces / 2);
                uint32_t const m = 2 * (i & 3u);
                uint32_t const d = (i - h * (pieces / 2)) / 4 * 2;
                uint64_t const at = static_cast<uint64_t>(h0 + h) * 16 * D + 8 * D + d * 8;
                w[k][0] = load_once(source[m] + at);
                w[k][1] = load_once(source[m + 1] + at);
            }
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce / 2; ++k) {
                uint32_t const i = base + k * kBlock;
                if (i >= (h1 - h0) * pieces / 2) continue;
                uint32_t const h = i / (pieces / 2);
                uint32_t const d = (i - h * (pieces / 2)) / 4 * 2;
                uint8_t* const to = quant_codes(dst, P, 64, h0 + h) + 64 * D + d * 64 + 16 * (i & 3u);
                *reinterpret_cast<u32x4_t*>(to) = u32x4_t{w[k][0][0], w[k][0][1], w[k][1][0], w[k][1][1]};
                *reinterpret_cast<u32x4_t*>(to + 64) = u32x4_t{w[k][0][2], w[k][0][3], w[k][1][2], w[k][1][3]};
            }
        }
    } else {
        for (uint32_t h = h0; h < h1; ++h) {
            uint8_t* const to = quant_codes(dst, P, 64, h);
            uint64_t const from = static_cast<uint64_t>(h) * 16 * D;
            for (uint32_t i = tid; i < 8 * D; i += kBlock) {   // of 8 bytes
                uint32_t const m = i / D;
                uint32_t const o = (i - m * D) * 8;
                *reinterpret_cast<u32x2_t*>(to + m * run + o) = *reinterpret_cast<const u32x2_t*>(source[m] + from + o);
                uint32_t const vm = i & 7u;
                uint32_t const d = i >> 3;
                *reinterpret_cast<u32x2_t*>(to + 64 * D + d * 64 + vm * 8) = *reinterpret_cast<const u32x2_t*>(source[vm] + from + 8 * D + d * 8);
            }
        }
    }
    // The scales: of a head, 8 of K and 8 of V a page.
    for (uint32_t i = tid; i < (h1 - h0) * 128; i += kBlock) {
        uint32_t const h = h0 + i / 128;
        uint32_t const m = (i >> 3) & 7u;
        uint32_t const value = (i >> 6) & 1u;
        const uint16_t* const s = reinterpret_cast<const uint16_t*>(source[m] + static_cast<uint64_t>(P.heads) * 16 * D) + h * 16;
        quant_scales(dst, P, 64, h)[i & 127u] = s[value * 8 + (i & 7u)];
    }
}

// Moves the fault word to the mapped host word and clears it in one exchange.
__global__ __launch_bounds__(64) void quant_take_faults_kernel(uint32_t* faults, uint32_t* host_word)
{
    if (threadIdx.x == 0) *host_word = atomicExch(faults, 0u);
}

// Heads a block takes, a power of two: about kQuantMaxDim dims (6 layers of 4 x
// 4096 tokens, 8 heads of 128, all in turn in a block: 265 us, two of them 244),
// fewer where the rest of the grid does not fill the chip.
uint32_t heads_of_block(uint32_t heads, uint32_t dim, uint64_t blocks)
{
    uint32_t per = 1;
    while (per < heads && 2 * per * dim <= kQuantMaxDim) per *= 2;
    while (per > 1 && blocks * ceil_div(heads, per) < 1024) per /= 2;
    return per;
}

// f(format, head dim) of a storage; the dims whose index arithmetic is fixed
// where the code is built, 0 for all others.
template <typename F>
auto with_format(const kimkv_quant_storage& s, F f)
{
    auto const with_dim = [&](auto format) {
        switch (s.layout.head_dim) {
        case 64: return f(format, std::integral_constant<uint32_t, 64>{});
        case 128: return f(format, std::integral_constant<uint32_t, 128>{});
        default: return f(format, std::integral_constant<uint32_t, 0>{});
        }
    };
    return s.format == KIMKV_QUANT_INT8 ? with_dim(std::integral_constant<uint32_t, KIMKV_QUANT_INT8>{})
                                        : with_dim(std::integral_constant<uint32_t, KIMKV_QUANT_E4M3>{});
}

bool on_device(const kimkv_quant_storage* s)
{
    int device = -1;
    return hipGetDevice(&device) == hipSuccess && device == s->device;
}

constexpr uint32_t kGridRows = 65535;   // of a launch's second and third dimension
constexpr uint32_t kGridBlocks = 0xFFFFFFu;   // times kBlock threads: fewer than 2^32

}  // namespace
}  // namespace kimkv

using namespace kimkv;

extern "C" {

kimkv_status kimkv_quant_storage_create(kimkv_quant_storage** out, kimkv_layout layout, uint32_t format, uint32_t micro_capacity,
                                        uint32_t extent_capacity, uint16_t micro_page_tokens, uint16_t extent_page_tokens)
{
    if (out == nullptr) return KIMKV_INVALID_ARGUMENT;
    *out = nullptr;
    auto const page = [](uint32_t tokens) { return tokens != 0 && tokens % 8 == 0 && tokens <= kQuantMaxPage; };
    if (layout.layers == 0 || layout.layers > 0x7FFFu || layout.kv_heads == 0 || layout.kv_heads > kGridRows || layout.head_dim == 0
        || layout.head_dim > kQuantMaxDim || (format != KIMKV_QUANT_INT8 && format != KIMKV_QUANT_E4M3) || !page(micro_page_tokens)
        || !page(extent_page_tokens)) {
        return KIMKV_INVALID_ARGUMENT;
    }
    // At most 2^15 layers x 2^32 pages x 2^16 heads x 2^15 bytes: 2^78.
    uint64_t const layer_bytes_limit = std::numeric_limits<int64_t>::max() / layout.layers / 2;
    uint64_t const micro_slot = quant_slot_bytes(layout, micro_page_tokens);
    uint64_t const extent_slot = quant_slot_bytes(layout, extent_page_tokens);
    if ((micro_capacity != 0 && micro_slot > layer_bytes_limit / micro_capacity)
        || (extent_capacity != 0 && extent_slot > layer_bytes_limit / extent_capacity)) {
        return KIMKV_INVALID_ARGUMENT;
    }
    int count = 0;
    if (hipGetDeviceCount(&count) != hipSuccess || count == 0) return KIMKV_RUNTIME_UNAVAILABLE;
    auto* s = new (std::nothrow) kimkv_quant_storage{};
    if (s == nullptr) return KIMKV_ALLOCATION_FAILED;
    s->layout = layout;
    s->format = format;
    s->micro_capacity = micro_capacity;
    s->extent_capacity = extent_capacity;
    s->micro_tokens = micro_page_tokens;
    s->extent_tokens = extent_page_tokens;
    uint64_t const bytes = (micro_slot * micro_capacity + extent_slot * extent_capacity) * layout.layers;
    hipError_t e = hipGetDevice(&s->device);
    if (e == hipSuccess) e = hipDeviceGetAttribute(&s->compute_units, hipDeviceAttributeMultiprocessorCount, s->device);
    if (e == hipSuccess && bytes != 0) {
        e = hipMalloc(reinterpret_cast<void**>(&s->pool), bytes);
        if (e == hipSuccess) e = hipMemset(s->pool, 0, bytes);
    }
    if (e == hipSuccess) {
        e = hipMalloc(reinterpret_cast<void**>(&s->faults), 256);
        if (e == hipSuccess) e = hipMemset(s->faults, 0, 256);
    }
    if (e == hipSuccess) {
        e = hipHostMalloc(reinterpret_cast<void**>(&s->fault_host), 256, hipHostMallocMapped | hipHostMallocCoherent);
        if (e == hipSuccess) e = hipHostGetDevicePointer(reinterpret_cast<void**>(&s->fault_view), s->fault_host, 0);
    }
    if (e == hipSuccess) e = hipDeviceSynchronize();
    if (e != hipSuccess) {
        record_error(e, KIMKV_ALLOCATION_FAILED);
        if (s->pool) static_cast<void>(hipFree(s->pool));
        if (s->faults) static_cast<void>(hipFree(s->faults));
        if (s->fault_host) static_cast<void>(hipHostFree(s->fault_host));
        delete s;
        return KIMKV_ALLOCATION_FAILED;
    }
    *out = s;
    return KIMKV_OK;
}

kimkv_status kimkv_quant_storage_destroy(kimkv_quant_storage* storage)
{
    if (storage == nullptr) return KIMKV_OK;
    // In-flight work may still read the pools.
    static_cast<void>(hipDeviceSynchronize());
    if (storage->pool) static_cast<void>(hipFree(storage->pool));
    if (storage->faults) static_cast<void>(hipFree(storage->faults));
    if (storage->fault_host) static_cast<void>(hipHostFree(storage->fault_host));
    delete storage;
    return KIMKV_OK;
}

kimkv_status kimkv_quant_storage_query(const kimkv_quant_storage* s, kimkv_quant_storage_info* info)
{
    if (s == nullptr || info == nullptr) return KIMKV_INVALID_ARGUMENT;
    *info = kimkv_quant_storage_info{};
    info->layout = s->layout;
    info->format = s->format;
    info->micro_capacity = s->micro_capacity;
    info->extent_capacity = s->extent_capacity;
    info->micro_page_tokens = s->micro_tokens;
    info->extent_page_tokens = s->extent_tokens;
    info->micro_page_bytes = quant_slot_bytes(s->layout, s->micro_tokens) * s->layout.layers;
    info->extent_page_bytes = quant_slot_bytes(s->layout, s->extent_tokens) * s->layout.layers;
    info->reserved_bytes = info->micro_page_bytes * s->micro_capacity + info->extent_page_bytes * s->extent_capacity;
    info->device = s->device;
    info->compute_units = s->compute_units;
    return KIMKV_OK;
}

kimkv_status kimkv_quant_storage_faults(kimkv_quant_storage* storage, kimkv_stream_t stream, uint32_t* faults)
{
    if (faults != nullptr) *faults = 0;
    if (storage == nullptr || !on_device(storage)) return KIMKV_INVALID_ARGUMENT;
    // One reader of the mapped word at a time.
    static std::mutex mutex;
    std::lock_guard<std::mutex> lock(mutex);
    *reinterpret_cast<volatile uint32_t*>(storage->fault_host) = 0;
    quant_take_faults_kernel<<<1, 64, 0, native(stream)>>>(storage->faults, storage->fault_view);
    kimkv_status const launched = launch_status();
    if (launched != KIMKV_OK) return launched;
    kimkv_status const done = record_error(hipStreamSynchronize(native(stream)), KIMKV_EXECUTION_FAILED);
    if (done != KIMKV_OK) return done;
    uint32_t const bits = *reinterpret_cast<volatile uint32_t*>(storage->fault_host);
    if (faults != nullptr) *faults = bits;
    return bits != 0 ? KIMKV_INVALID_ARGUMENT : KIMKV_OK;
}

kimkv_status kimkv_quant_append_batch(const kimkv_quant_storage* storage, const kimkv_append_job* device_jobs, uint32_t job_count,
                                      uint32_t max_layer_count, kimkv_stream_t stream)
{
    if (storage == nullptr || (job_count != 0 && device_jobs == nullptr) || max_layer_count > storage->layout.layers || !on_device(storage)) {
        return KIMKV_INVALID_ARGUMENT;
    }
    if (job_count == 0 || max_layer_count == 0) return KIMKV_OK;
    QuantView const view = quant_view(*storage);
    uint32_t const heads = heads_of_block(view.heads, view.dim, static_cast<uint64_t>(job_count) * max_layer_count);
    uint32_t const z = ceil_div(view.heads, heads);
    uint32_t const most = kGridBlocks / (max_layer_count * z) == 0 ? 1 : kGridBlocks / (max_layer_count * z);
    auto const kernel = with_format(*storage, [](auto format, auto dim) { return quant_append_kernel<format.value, dim.value>; });
    for (uint32_t first = 0; first < job_count;) {
        uint32_t const jobs = job_count - first < most ? job_count - first : most;
        kernel<<<dim3(jobs, max_layer_count, z), kBlock, 0, native(stream)>>>(view, device_jobs + first, AppendGrid{log2_of(heads), log2_of(ceil_div(view.dim, 8))});
        kimkv_status const status = launch_status();
        if (status != KIMKV_OK) return status;
        first += jobs;
    }
    return KIMKV_OK;
}

kimkv_status kimkv_quant_gather(const kimkv_quant_storage* storage, const kimkv_block_desc* device_descriptors, uint32_t descriptor_count,
                                uint32_t first_token, uint32_t token_count, uint32_t layer_begin, uint32_t layer_count,
                                uint16_t* device_output, kimkv_stream_t stream)
{
    if (storage == nullptr || layer_begin > storage->layout.layers || layer_count > storage->layout.layers - layer_begin
        || token_count > 0xFFFFFFFFu - first_token || !on_device(storage)) {
        return KIMKV_INVALID_ARGUMENT;
    }
    if (token_count == 0 || layer_count == 0) return KIMKV_OK;
    if (device_descriptors == nullptr || descriptor_count == 0 || device_output == nullptr) return KIMKV_INVALID_ARGUMENT;
    QuantView const view = quant_view(*storage);
    uint32_t const heads = heads_of_block(view.heads, view.dim, static_cast<uint64_t>(descriptor_count) * layer_count);
    uint32_t const z = ceil_div(view.heads, heads);
    uint32_t const most = kGridBlocks / (layer_count * z) == 0 ? 1 : kGridBlocks / (layer_count * z);
    bool const wide = view.dim % 8 == 0 && (reinterpret_cast<uintptr_t>(device_output) & 15u) == 0;
    auto const kernel = with_format(*storage, [](auto format, auto dim) { return quant_gather_kernel<format.value, dim.value>; });
    for (uint32_t first = 0; first < descriptor_count;) {
        uint32_t const entries = descriptor_count - first < most ? descriptor_count - first : most;
        GatherArgs const args{device_descriptors + first, device_output, first_token, token_count, layer_begin, heads, wide};
        kernel<<<dim3(entries, layer_count, z), kBlock, 0, native(stream)>>>(view, args);
        kimkv_status const status = launch_status();
        if (status != KIMKV_OK) return status;
        first += entries;
    }
    return KIMKV_OK;
}

kimkv_status kimkv_quant_promote_batch(const kimkv_quant_storage* storage, const kimkv_promotion_job* device_jobs, uint32_t job_count,
                                       kimkv_stream_t stream)
{
    if (storage == nullptr || (job_count != 0 && device_jobs == nullptr) || storage->micro_tokens != 8 || storage->extent_tokens != 64
        || !on_device(storage)) {
        return KIMKV_INVALID_ARGUMENT;
    }
    if (job_count == 0) return KIMKV_OK;
    QuantView const view = quant_view(*storage);
    uint32_t const heads = heads_of_block(view.heads, view.dim, static_cast<uint64_t>(job_count) * view.layers);
    uint32_t const z = ceil_div(view.heads, heads);
    uint32_t const most = kGridBlocks / (view.layers * z) == 0 ? 1 : kGridBlocks / (view.layers * z);
    for (uint32_t first = 0; first < job_count;) {
        uint32_t const jobs = job_count - first < most ? job_count - first : most;
        quant_promote_kernel<<<dim3(jobs, view.layers, z), kBlock, 0, native(stream)>>>(view, device_jobs + first, heads);
        kimkv_status const status = launch_status();
        if (status != KIMKV_OK) return status;
        first += jobs;
    }
    return KIMKV_OK;
}

}  // extern "C"
