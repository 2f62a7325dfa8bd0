// quant_common.h -- pages of a cache in 8 bits: storage, layout, and the two
// number formats of their codes.
//
// A row is the D values of one token's K or V of one head.  With a = max |x|
// of the row and Q = 127 (whole numbers) or 448 (e4m3), its scale s is the
// smallest number of 8 significant bits (a bf16) with Q s >= a, and its codes
// are x / s rounded to nearest, ties to even.  x has 11 significant bits and a
// tie times s at most 13 to 16, so x / s either is a tie or is 2^-19 of itself
// away from one: a quotient that is rounded to 32 bits first rounds to the
// same code.  Likewise a / Q in 32 bits is a bf16 exactly where a is Q times
// one, and else at least 2^-15 away, so rounding it up gives s.  A row of zeros
// has s = 0; one that holds an infinity or a NaN has s = NaN and codes of 0.
//
// Page layout: one layer's block of a page holds, per head, 2 cap D code bytes,
// K first, then V transposed, and behind all heads their scales, per head cap
// of K and cap of V:
//   K(t, d) = (d / kw) cap kw + t kw + d % kw,   kw = 64 where D is a multiple of 64, else D
//   V(d, t) = cap D + d cap + t                  (cap <= 64)
// A matrix-core operand load of 16 tokens x 16 bytes of K, or 16 dims x 16 tokens
// of V, is then 1 KB without gaps.  Scales of a page lie beside its codes rather
// than in a pool of their own: they are 2 / D of a row, and share its
// address translation.
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>

#include <cstdint>

#include "device_common.h"
#include "kimkv_hip.h"

struct kimkv_quant_storage {
    kimkv_layout layout{};
    uint32_t format{0};
    uint32_t micro_capacity{0};
    uint32_t extent_capacity{0};
    uint16_t micro_tokens{0};
    uint16_t extent_tokens{0};
    uint8_t* pool{nullptr};
    uint32_t* faults{nullptr};       // device word, KIMKV_FAULT_* bits
    uint32_t* fault_host{nullptr};   // mapped pinned word kimkv_quant_storage_faults reads
    uint32_t* fault_view{nullptr};   // its device address
    int device{0};
    int compute_units{0};
};

namespace kimkv {

constexpr uint32_t kQuantMaxDim = 256;
constexpr uint32_t kQuantMaxPage = 64;

// Pool view passed to kernels by value.
struct QuantView {
    uint8_t* micro;                // layer 0's micro blocks
    uint8_t* extent;
    uint64_t micro_slot_bytes;     // one micro page's block of one layer
    uint64_t extent_slot_bytes;
    uint64_t layer_bytes;          // one layer's region: every micro, then every extent page
    uint32_t micro_capacity;
    uint32_t extent_capacity;
    uint32_t micro_tokens;
    uint32_t extent_tokens;
    uint32_t layers;
    uint32_t heads;
    uint32_t dim;
    uint32_t* faults;
};

// Bytes of one page's block of one layer; whole 128-byte lines.
inline uint64_t quant_slot_bytes(const kimkv_layout& l, uint32_t cap)
{
    uint64_t const bytes = static_cast<uint64_t>(l.kv_heads) * cap * (2ull * l.head_dim + 4);
    return (bytes + 127) / 128 * 128;
}

inline QuantView quant_view(const kimkv_quant_storage& s)
{
    uint64_t const micro_slot = quant_slot_bytes(s.layout, s.micro_tokens);
    uint64_t const extent_slot = quant_slot_bytes(s.layout, s.extent_tokens);
    return QuantView{s.pool, s.pool + micro_slot * s.micro_capacity, micro_slot, extent_slot,
                     micro_slot * s.micro_capacity + extent_slot * s.extent_capacity,
                     s.micro_capacity, s.extent_capacity, s.micro_tokens, s.extent_tokens,
                     s.layout.layers, s.layout.kv_heads, s.layout.head_dim, s.faults};
}

__device__ inline void report_fault(const QuantView& p, uint32_t bit)
{
    if (threadIdx.x == 0 && p.faults != nullptr) atomicOr(p.faults, bit);
}

__device__ inline uint32_t quant_page_tokens(const QuantView& p, uint32_t kind)
{
    return kind == KIMKV_PAGE_MICRO ? p.micro_tokens : p.extent_tokens;
}

// Block of a (kind, slot) in a layer, or nullptr when the handle does not name
// a page of this storage or its capacity is not the pool's.
__device__ inline uint8_t* quant_block(const QuantView& p, uint32_t layer, uint32_t kind, uint32_t slot, uint32_t capacity)
{
    uint64_t const region = layer * p.layer_bytes;
    if (kind == KIMKV_PAGE_MICRO && slot < p.micro_capacity && capacity == p.micro_tokens) {
        return p.micro + region + slot * p.micro_slot_bytes;
    }
    if (kind == KIMKV_PAGE_EXTENT && slot < p.extent_capacity && capacity == p.extent_tokens) {
        return p.extent + region + slot * p.extent_slot_bytes;
    }
    return nullptr;
}

__host__ __device__ inline uint32_t quant_k_width(uint32_t D) { return D % 64u == 0u ? 64u : D; }

// Byte offsets inside a head's codes.
__device__ inline uint32_t quant_k_at(uint32_t cap, uint32_t D, uint32_t t, uint32_t d)
{
    return D % 64u == 0u ? (d >> 6) * cap * 64u + t * 64u + (d & 63u) : t * D + d;
}
__device__ inline uint32_t quant_v_at(uint32_t cap, uint32_t D, uint32_t t, uint32_t d) { return cap * D + d * cap + t; }

// A head's codes and scales in a page's block.
__device__ inline uint8_t* quant_codes(uint8_t* block, const QuantView& p, uint32_t cap, uint32_t head)
{
    return block + static_cast<uint64_t>(head) * 2u * cap * p.dim;
}
__device__ inline uint16_t* quant_scales(uint8_t* block, const QuantView& p, uint32_t cap, uint32_t head)
{
    return reinterpret_cast<uint16_t*>(block + static_cast<uint64_t>(p.heads) * 2u * cap * p.dim) + static_cast<uint64_t>(head) * 2u * cap;
}

// ---- the two formats ---------------------------------------------------------

template <uint32_t kFormat>
__device__ inline float quant_largest()
{
    return kFormat == KIMKV_QUANT_INT8 ? 127.0f : 448.0f;
}

__device__ inline float scale_value(uint16_t bits) { return __uint_as_float(static_cast<uint32_t>(bits) << 16); }

constexpr uint16_t kScaleNan = 0x7FC0;

// The scale of a row whose |x| are at most the fp16 of these bits: a / Q, by a
// product that is off by 3 steps of 32 bits at most, rounded up.  a / Q is a bf16
// or 256 of these steps away from one, so 64 of them are no part of a larger one.
template <uint32_t kFormat>
__device__ inline uint16_t row_scale(uint32_t largest_bits)
{
    if (largest_bits >= 0x7C00u) return kScaleNan;
    float const q = __half2float(__ushort_as_half(static_cast<uint16_t>(largest_bits))) * (1.0f / quant_largest<kFormat>());
    return static_cast<uint16_t>((__float_as_uint(q) + (0xFFFFu - 64u)) >> 16);
}

// What codes of a row are made with: 1 / s, and s; 0 where every code is 0.
struct RowQuant {
    float scale;
    float inverse;
};

__device__ inline RowQuant row_quant(uint16_t scale_bits)
{
    bool const none = scale_bits == 0 || scale_bits == kScaleNan;
    float const s = none ? 1.0f : scale_value(scale_bits);
    return RowQuant{s, none ? 0.0f : __builtin_amdgcn_rcpf(s)};
}

// x / s rounded to 32 bits: the product with the reciprocal, corrected once by
// its remainder (exact in one fused operation), so that a quotient that 32 bits
// hold, a tie among them, is exact.
__device__ inline float row_quotient(float x, RowQuant r)
{
    float const y = x * r.inverse;
    return __builtin_fmaf(__builtin_fmaf(-y, r.scale, x), r.inverse, y);
}

// Four codes of a row, one a byte.  A whole number is held with 128 added, so
// that the byte under the bits of 1024 is an fp16 number, and read by one
// subtraction.
template <uint32_t kFormat>
__device__ inline uint32_t row_codes(const float (&x)[4], RowQuant r)
{
    float y[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) y[i] = row_quotient(x[i], r);
    if (kFormat == KIMKV_QUANT_INT8) {
        // The sum's last bit is 1: it rounds to the whole number, ties to even.
        uint32_t u[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) u[i] = __float_as_uint(y[i] + 8388736.0f);
        uint32_t const lo = __builtin_amdgcn_perm(u[1], u[0], 0x0C0C0400u);
        uint32_t const hi = __builtin_amdgcn_perm(u[3], u[2], 0x04000C0Cu);
        return lo | hi;
    }
    uint32_t const lo = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false));
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], static_cast<int>(lo), true));
}

// Four codes of 0.
template <uint32_t kFormat>
__device__ inline uint32_t no_codes()
{
    return kFormat == KIMKV_QUANT_INT8 ? 0x80808080u : 0u;
}

// Eight codes as fp16.  A whole number's byte u under the bits of 1024 is
// 1024 + u, and 1152 less is the number, exactly.
typedef uint32_t code_words_t __attribute__((ext_vector_type(2)));
typedef _Float16 code_halves_t __attribute__((ext_vector_type(8)));
template <uint32_t kFormat>
__device__ inline code_halves_t code_halves(code_words_t w)
{
    typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
    code_halves_t out;
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
        half2_t a, b;
        if (kFormat == KIMKV_QUANT_INT8) {
            half2_t const shift = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
            a = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, w[j], 0x04010400u)) + shift;
            b = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, w[j], 0x04030402u)) + shift;
        } else {
            a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w[j]), 1.0f, false);
            b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w[j]), 1.0f, true);
        }
        out[4 * j] = a[0];
        out[4 * j + 1] = a[1];
        out[4 * j + 2] = b[0];
        out[4 * j + 3] = b[1];
    }
    return out;
}

template <uint32_t kFormat>
__device__ inline float code_value(uint8_t code)
{
    return static_cast<float>(code_halves<kFormat>(code_words_t{code, 0})[0]);
}

// A code times its scale as fp16.  The product is exact in 32 bits; the
// largest, 516 * 127 and 147 * 448, are past fp16's and stay at 65504.
__device__ inline uint16_t read_back(float code, float scale)
{
    float v = code * scale;
    v = v > 65504.0f ? 65504.0f : v;
    v = v < -65504.0f ? -65504.0f : v;
    return __half_as_ushort(__float2half_rn(v));
}
// Eight codes of a row; a product past 65504 only with a scale whose largest one is.
template <uint32_t kFormat>
__device__ inline code_halves_t read_back(code_words_t w, float scale)
{
    code_halves_t const code = code_halves<kFormat>(w);
    code_halves_t out;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) out[j] = static_cast<_Float16>(static_cast<float>(code[j]) * scale);
    if (__ballot(scale * quant_largest<kFormat>() > 65504.0f) != 0) {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) out[j] = __builtin_bit_cast(_Float16, read_back(static_cast<float>(code[j]), scale));
    }
    return out;
}

}  // namespace kimkv
