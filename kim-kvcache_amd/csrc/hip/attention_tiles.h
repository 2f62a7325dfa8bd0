// attention_tiles.h -- tiles of one KV head's keys and values in LDS, shared by
// the paged prefill and the shared-prefix decode kernels: the 8-key groups of
// a key range resolved to page addresses, and 256 threads that fetch a tile
// (16-byte loads, one in registers while another is computed from) and store it
// bank-swizzled.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "attention_common.h"
#include "device_common.h"

namespace kimkv {

constexpr unsigned kTileThreads = 256;   // threads that fetch and store a tile

// What depends on the head dim of the tiles (64 or 128).
template <uint32_t kDim>
struct TileDims {
    static_assert(kDim == 64 || kDim == 128, "MFMA path head dims");
    static constexpr uint32_t kTileKeys = 4096 / kDim;   // keys per staged tile: 16 KiB of K and V^T
    static constexpr uint32_t kKB = kTileKeys / 32;      // 32-key halves of a tile
    static constexpr uint32_t kPanels = kDim / 32;       // 32-dim column blocks of K
    static constexpr uint32_t kDb = kDim / 16;           // 16-dim blocks of O
};

// One tile of one KV head staged in LDS, in 16-byte units:
//   K   unit (key t, dim octet o) at t * (D / 8) + (o ^ k_swizzle(t))
//   V^T unit (dim d, key octet c), D = 64 (8 octets):  d * 8 + (c ^ (d & 7))
//                                  D = 128 (4 octets): d * 4 + (c ^ ((d >> 1) & 3))
// The swizzles put the eight 16-byte reads that one LDS cycle serves (lanes
// 8j .. 8j + 7 of an MFMA operand read) on eight different bank groups.
template <uint32_t kDim>
struct KvTile {
    half8_t k[TileDims<kDim>::kTileKeys * (kDim / 8)];
    half8_t v[kDim * (TileDims<kDim>::kTileKeys / 8)];
};

__device__ inline uint32_t k_swizzle(uint32_t t) { return (t & 3u) | (((t >> 3) & 1u) << 2); }
template <uint32_t kDim>
__device__ inline uint32_t k_unit(uint32_t t, uint32_t o)
{
    return t * (kDim / 8) + (o ^ k_swizzle(t));
}
template <uint32_t kDim>
__device__ inline uint32_t v_unit(uint32_t d, uint32_t c)
{
    return kDim == 64 ? d * 8u + (c ^ (d & 7u)) : d * 4u + (c ^ ((d >> 1) & 3u));
}

// One 8-key group of a key range resolved for a layer and KV head:
// k points at the group's first key in K panel 0 (panel p, dims 32 p ..
// 32 p + 31, is p * kpanel elements further), v at the group's first key in
// V^T row 0 (dim d is d * vw elements further).
struct HeadGroup {
    const uint16_t* k;
    const uint16_t* v;
    uint32_t kpanel;
    uint32_t vw;
    uint64_t pad;
};

// Records the 8-key groups of [c0, c1) that entry `e` covers, for layer /
// head.  An entry whose pages do not keep 8-token groups aligned (or that
// names no page of the storage) switches the block to the generic path.
template <uint32_t kDim>
__device__ inline void add_head_groups(const PoolView& P, kimkv_block_desc const& e, uint32_t layer, uint32_t h,
                                       uint32_t c0, uint32_t c1, uint32_t T, HeadGroup* groups, uint32_t* s_generic)
{
    uint32_t const b = e.logical_token_begin;
    uint32_t const end = b + e.valid_tokens;
    uint32_t const lo = max(b, c0);
    uint32_t const hi = min(end, c1);
    if (lo >= hi) return;
    uint32_t const cap = e.page_token_capacity;
    const uint16_t* page = page_base(P, e.kind, e.slot, cap);
    bool const aligned = (b & 7u) == 0 && (cap & 7u) == 0 && e.valid_tokens <= cap
        && ((end & 7u) == 0 || end >= T) && page != nullptr;
    if (!aligned) {
        *s_generic = 1;
        return;
    }
    const uint16_t* hb = page + head_block(P, cap, layer, h);
    uint32_t const vw = v_width(cap);
    for (uint32_t g = (lo - c0) >> 3; g < (hi - c0 + 7) >> 3; ++g) {
        uint32_t const pt0 = c0 + 8 * g - b;
        groups[g] = HeadGroup{hb + k_offset(cap, kDim, pt0, 0), hb + v_offset(cap, kDim, pt0, 0), cap * 32u, vw, 0};
    }
}

// A thread's share of one tile in flight: two K units and two V^T units.
//   K unit j:   chunk c = tid + 256 j -> group c / (D), panel (c / 32) % (D / 32), key (c / 4) % 8, octet c % 4
//               (a wave reads half or all of one 8-key group: contiguous 512-byte runs of the page)
//   V^T unit j: D = 64:  key octet 4 j + tid % 4, dim tid / 4
//               D = 128: key octet tid % 4, dim tid / 4 + 64 j
//               (four consecutive lanes read one dim row of a 32-key V^T panel: 64 contiguous bytes)
struct TileLoad {
    half8_t k[2];
    half8_t v[2];
};

// A wave-uniform 64-bit value in SGPRs.  readfirstlane returns int: each
// half goes through uint32_t so that the low half is not sign-extended.
__device__ __attribute__((always_inline)) inline uint64_t uniform_u64(uint64_t x)
{
    uint32_t const lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x)));
    uint32_t const hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x >> 32)));
    return (static_cast<uint64_t>(hi) << 32) | lo;
}

// kFull: all keys of the tile are below nvalid and every group of the segment
// names a page, so no lane needs a check.  A K unit's group (c / D) is the
// same for the whole wave: its base goes to SGPRs and each lane adds a 32-bit
// offset (panel (tid / 32) % (D / 32), key (tid / 4) % 8, octet tid % 4, the
// same for both units).
template <uint32_t kDim, bool kFull>
__device__ inline void tile_fetch(TileLoad& r, const HeadGroup* groups, uint32_t tg, uint32_t nvalid, uint32_t tid)
{
    using Dims = TileDims<kDim>;
    half8_t const zero8 = {};
    uint32_t const tk = (tid >> 2) & 7u;
    uint32_t const k_off = tk * 64u + (tid & 3u) * 16u;
    uint32_t const k_panel = (tid >> 5) & (Dims::kPanels - 1);
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
        uint32_t const g = (tid + kTileThreads * j) / kDim;
        if (kFull || 8 * g + tk < nvalid) {
            HeadGroup const e = groups[tg + g];
            uint64_t const kb = uniform_u64(reinterpret_cast<uintptr_t>(e.k));
            uint32_t const off = k_off + k_panel * static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(e.kpanel)) * 2u;
            r.k[j] = zero8;
            if (kFull || kb != 0) {
                r.k[j] = __builtin_nontemporal_load(reinterpret_cast<const global_half8_t*>(kb + off));
            }
        } else {
            r.k[j] = zero8;
        }
        uint32_t const ko = kDim == 64 ? 4 * j + (tid & 3u) : tid & 3u;
        uint32_t const d = kDim == 64 ? tid >> 2 : (tid >> 2) + 64 * j;
        if (kFull) {
            HeadGroup const e = groups[tg + ko];
            r.v[j] = load_half8_stream(e.v + d * e.vw);
        } else {
            r.v[j] = zero8;
            if (8 * ko < nvalid) {
                HeadGroup const e = groups[tg + ko];
                if (e.v != nullptr) {
                    r.v[j] = load_half8_stream(e.v + d * e.vw);
                    if (8 * ko + 8 > nvalid) {
                        uint32_t const keep = nvalid - 8 * ko;
#pragma unroll
                        for (uint32_t q = 0; q < 8; ++q) {
                            if (q >= keep) r.v[j][q] = static_cast<_Float16>(0.0f);
                        }
                    }
                }
            }
        }
    }
}

template <uint32_t kDim>
__device__ inline void tile_store(KvTile<kDim>& t, const TileLoad& r, uint32_t tid)
{
    using Dims = TileDims<kDim>;
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
        uint32_t const c = tid + kTileThreads * j;
        uint32_t const key = 8 * (c / kDim) + ((c >> 2) & 7u);
        t.k[k_unit<kDim>(key, 4 * ((c >> 5) & (Dims::kPanels - 1)) + (c & 3u))] = r.k[j];
        if (kDim == 64) {
            t.v[v_unit<kDim>(tid >> 2, 4 * j + (tid & 3u))] = r.v[j];
        } else {
            t.v[v_unit<kDim>((tid >> 2) + 64 * j, tid & 3u)] = r.v[j];
        }
    }
}

}  // namespace kimkv
