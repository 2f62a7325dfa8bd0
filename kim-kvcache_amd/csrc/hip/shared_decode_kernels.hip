// shared_decode_kernels.hip -- paged decode attention of lanes that share
// prefixes, for gfx950.
//
// A group of n lanes forked from one prompt attends to the prompt's pages with
// n * G query rows for each KV head: one matrix product instead of n reads.
// Softmax over a split set of keys is the merge of the parts' (o, m, l):
//   m = max s_t,  l = sum 2^(s_t - m),  o = sum 2^(s_t - m) v_t
//   out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i,  M = max m_i
// so the plan cuts the batch into units, each a run of tokens of one table and
// the lanes that attend to them through it: pieces of the groups' prefixes,
// and of every lane's own tokens.  A unit's workgroup leaves its lanes' parts
// in the launch's workspace (the output itself where a lane has one part), and
// a second launch merges them.
//
// No counterpart in the reference, whose batch kernel reads every lane's whole
// table (src/cuda/attention/paged_decode_kernels.cu:299-474).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <type_traits>
#include <utility>
#include <vector>

#include "attention_common.h"
#include "attention_tiles.h"
#include "device_common.h"
#include "runtime_internal.h"

namespace kimkv {
namespace {

constexpr unsigned kBlock = 512;   // 8 waves
constexpr unsigned kWaves = kBlock / kWave;
constexpr uint32_t kMaxDim = 256;

// How a unit is computed.
constexpr uint8_t kDirect = 0;      // few columns: the waves split heads and tokens; 1, 2, 4: staged tiles, that many
constexpr uint8_t kSingle = 0x80;   // 16-column blocks a wave.  kSingle: the lane has no other part.

// Tokens [begin, end) of table_lane's table for KV heads [head, head + heads).
// Of the score matrix of lanes lane, lane + 1, ... (G query heads of a KV head
// each) it takes columns [col0, col0 + cols): column c is query head c % G of
// the KV head's group, lane lane + c / G, whose part goes to slot + c / G.
// cols = 0: nothing to do.
struct SharedUnit {
    uint32_t table_lane;
    uint32_t lane;
    uint32_t col0;
    uint32_t cols;
    uint32_t begin;
    uint32_t end;
    uint32_t slot;
    uint16_t head;
    uint8_t heads;
    uint8_t kind;
};
static_assert(sizeof(SharedUnit) == 32, "entries are read as 16-byte vectors");

// A lane's parts: prefix_count ones prefix_stride slots apart from
// prefix_slot on, tail_count consecutive ones from tail_slot on.
struct SharedLane {
    uint32_t table_lane;     // whose table holds its prefix
    uint32_t tokens;         // as planned
    uint32_t prefix_slot;
    uint32_t prefix_stride;
    uint32_t prefix_count;
    uint32_t tail_slot;
    uint32_t tail_count;
    uint32_t merged;         // its output comes from the merge
};
static_assert(sizeof(SharedLane) == 32, "entries are read as 16-byte vectors");

// The launch's scratch: each slot's o ([QH][D] floats), then each slot's
// (m, l) ([QH] pairs).
struct Parts {
    float* o;
    float2* ml;
};

__host__ __device__ inline uint64_t parts_o_floats(uint64_t slots, uint32_t QH, uint32_t D) { return slots * QH * D; }

struct SharedArgs {
    const kimkv_decode_item* items;
    const SharedUnit* units;
    const SharedLane* lanes;
    Parts parts;
    uint32_t lane_count;
    uint32_t slot_count;
    uint32_t QH;
};

// Whether a lane can be computed: an item as planned.
__device__ inline bool lane_valid(const PoolView& P, const kimkv_decode_item& item, uint32_t planned_tokens)
{
    return planned_tokens != 0 && item.token_count == planned_tokens && item.descriptors != nullptr
        && item.descriptor_count != 0 && item.query != nullptr && item.output != nullptr && item.layer < P.layers;
}

// Whether a lane's output is made: with its own item also its group's first,
// through whose table its prefix is read, and both of one layer.
__device__ inline bool lane_ok(const PoolView& P, const SharedArgs& a, uint32_t lane)
{
    SharedLane const rec = a.lanes[lane];
    if (rec.table_lane >= a.lane_count) return false;
    kimkv_decode_item const item = a.items[lane];
    if (!lane_valid(P, item, rec.tokens)) return false;
    if (rec.table_lane == lane) return true;
    kimkv_decode_item const first = a.items[rec.table_lane];
    return lane_valid(P, first, a.lanes[rec.table_lane].tokens) && first.layer == item.layer;
}

// One column of a unit: query row, scale, and whether there is one (a lane
// whose item is not as planned, or is of another layer than the table's, has
// none).
struct Column {
    const uint16_t* query;
    float scale2;            // attention scale * log2 e
    bool ok;
};

__device__ inline Column unit_column(const PoolView& P, const SharedArgs& a, const SharedUnit& u, uint32_t layer, uint32_t G,
                                     uint32_t h, uint32_t c)
{
    if (c >= u.cols) return Column{nullptr, 0.0f, false};
    uint32_t const lane = u.lane + (u.col0 + c) / G;
    kimkv_decode_item const item = a.items[lane];
    bool const ok = lane_valid(P, item, a.lanes[lane].tokens) && item.layer == layer;
    return Column{item.query + (static_cast<uint64_t>(h) * G + (u.col0 + c) % G) * P.dim, item.attention_scale * kLog2e, ok};
}

// Where column c's part of KV head h goes.
struct PartOut {
    float* o;
    float2* ml;
    uint16_t* output;   // instead, for a lane of one part
};

__device__ inline PartOut part_out(const SharedArgs& a, const SharedUnit& u, uint32_t D, uint32_t G, uint32_t h, uint32_t c)
{
    uint32_t const i = (u.col0 + c) / G;
    uint32_t const q = h * G + (u.col0 + c) % G;
    if ((u.kind & kSingle) != 0) return PartOut{nullptr, nullptr, a.items[u.lane + i].output + static_cast<uint64_t>(q) * D};
    uint64_t const row = static_cast<uint64_t>(u.slot + i) * a.QH + q;
    return PartOut{a.parts.o + row * D, a.parts.ml + row, nullptr};
}

// o / l as an output: 0 for a row without any weight, l itself where it is not finite or NaN.
__device__ inline uint16_t output_half(float o, float l)
{
    return __half_as_ushort(__float2half_rn(l > 0.0f ? o / l : l == 0.0f ? 0.0f : l));
}

// ---------------------------------------------------------------------------
// Generic path: any table, head dim up to 256, scale, address.  A wave takes
// kRows query rows (columns of the unit's score matrix) at a time; lanes own
// keys for the scores and dims for the output.
// ---------------------------------------------------------------------------
constexpr uint32_t kRows = 8;

__device__ inline float read_lane(float v, uint32_t lane)
{
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), static_cast<int>(lane)));
}

// Parts of kRows rows: lane i holds o[r][k] of dim i + 64 k, every lane m and l.
struct RowParts {
    float o[kRows][4];
    float m[kRows];
    float l[kRows];
};

__device__ void attend_rows_generic(const PoolView& P, const kimkv_decode_item& table, uint32_t h, uint32_t c0,
                                    uint32_t c1, Column const (&rows)[kRows], RowParts& out)
{
    uint32_t const lane = threadIdx.x & (kWave - 1);
    uint32_t const D = P.dim;
    float q[kRows][4];
#pragma unroll
    for (uint32_t r = 0; r < kRows; ++r) {
        out.m[r] = -INFINITY;
        out.l[r] = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            uint32_t const d = lane + 64 * k;
            q[r][k] = rows[r].ok && d < D ? __half2float(__ushort_as_half(rows[r].query[d])) : 0.0f;
            out.o[r][k] = 0.0f;
        }
    }
    for (uint32_t t0 = c0; t0 < c1; t0 += 64) {
        uint32_t const t = t0 + lane;
        uint32_t idx = find_descriptor_wave(table.descriptors, table.descriptor_count, t0);
        const uint16_t* hb = nullptr;
        uint32_t cap = 0;
        uint32_t pt = 0;
        if (t < c1) {
            while (idx + 1 < table.descriptor_count && table.descriptors[idx + 1].logical_token_begin <= t) ++idx;
            kimkv_block_desc const e = table.descriptors[idx];
            if (t >= e.logical_token_begin && t - e.logical_token_begin < e.valid_tokens
                && e.valid_tokens <= e.page_token_capacity) {
                const uint16_t* page = page_base(P, e.kind, e.slot, e.page_token_capacity);
                if (page != nullptr) {
                    cap = e.page_token_capacity;
                    pt = t - e.logical_token_begin;
                    hb = page + head_block(P, cap, table.layer, h);
                }
            }
        }
        float s[kRows] = {};
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            for (uint32_t j = 0; j < 64 && 64 * k + j < D; ++j) {
                float const key = hb != nullptr ? __half2float(__ushort_as_half(hb[k_offset(cap, D, pt, 64 * k + j)])) : 0.0f;
#pragma unroll
                for (uint32_t r = 0; r < kRows; ++r) s[r] += read_lane(q[r][k], j) * key;
            }
        }
        float p[kRows];
#pragma unroll
        for (uint32_t r = 0; r < kRows; ++r) {
            s[r] = hb != nullptr ? s[r] * rows[r].scale2 : -INFINITY;
            float const m_new = fmaxf(out.m[r], wave_max(s[r]));
            float const alpha = m_new == -INFINITY ? 1.0f : exp2f(out.m[r] - m_new);
            p[r] = hb != nullptr && m_new != -INFINITY ? exp2f(s[r] - m_new) : 0.0f;
            out.l[r] = out.l[r] * alpha + wave_sum(p[r]);
            out.m[r] = m_new;
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) out.o[r][k] *= alpha;
        }
        const uint16_t* const vb = hb != nullptr ? hb + v_offset(cap, D, pt, 0) : nullptr;
        auto const vb_lo = static_cast<int>(reinterpret_cast<uintptr_t>(vb));
        auto const vb_hi = static_cast<int>(reinterpret_cast<uintptr_t>(vb) >> 32);
        auto const vb_width = static_cast<int>(v_width(cap));
        uint32_t const nt = min(64u, c1 - t0);
        for (uint32_t tt = 0; tt < nt; ++tt) {
            auto const key = static_cast<int>(tt);
            uint64_t const from = static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(vb_hi, key))) << 32
                | static_cast<uint32_t>(__builtin_amdgcn_readlane(vb_lo, key));
            auto const vw = static_cast<uint32_t>(__builtin_amdgcn_readlane(vb_width, key));
            if (from == 0) continue;
            float v[4];
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                uint32_t const d = lane + 64 * k;
                v[k] = d < D ? __half2float(__ushort_as_half(reinterpret_cast<const uint16_t*>(from)[static_cast<uint64_t>(d) * vw]))
                             : 0.0f;
            }
#pragma unroll
            for (uint32_t r = 0; r < kRows; ++r) {
                float const pp = read_lane(p[r], tt);
                if (pp == 0.0f) continue;   // whatever V holds there
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) out.o[r][k] += pp * v[k];
            }
        }
    }
}

// Rows as the waves leave them in LDS for the workgroup's own merge.
struct GenericLds {
    float o[kWaves][kRows][kMaxDim];
    float m[kWaves][kRows];
    float l[kWaves][kRows];
};

// The whole unit by the generic path.  A task is kRows columns of one KV head;
// where there are fewer tasks than waves, the waves of a task take a part of
// the tokens each.
__device__ void unit_generic(const PoolView& P, const SharedArgs& a, const SharedUnit& u, GenericLds& lds)
{
    uint32_t const tid = threadIdx.x;
    uint32_t const wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint32_t const D = P.dim;
    uint32_t const G = a.QH / P.heads;
    uint32_t const columns = u.cols;
    uint32_t const batches = (columns + kRows - 1) / kRows;
    uint32_t const tasks = u.heads * batches;
    uint32_t const split = tasks >= kWaves ? 1 : kWaves / tasks;
    uint32_t const at_once = kWaves / split;
    uint32_t const piece = ((u.end - u.begin + split - 1) / split + 63) / 64 * 64;
    kimkv_decode_item const table = a.items[u.table_lane];
    for (uint32_t t0 = 0; t0 < tasks; t0 += at_once) {
        uint32_t const task = t0 + wave / split;
        if (wave / split < at_once && task < tasks) {
            uint32_t const h = u.head + task / batches;
            uint32_t const col0 = task % batches * kRows;
            uint32_t const c0 = min(u.begin + wave % split * piece, u.end);
            uint32_t const c1 = min(c0 + piece, u.end);
            Column rows[kRows];
#pragma unroll
            for (uint32_t r = 0; r < kRows; ++r) rows[r] = unit_column(P, a, u, table.layer, G, h, col0 + r);
            RowParts part;
            attend_rows_generic(P, table, h, c0, c1, rows, part);
#pragma unroll
            for (uint32_t r = 0; r < kRows; ++r) {
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) lds.o[wave][r][(tid & 63u) + 64 * k] = part.o[r][k];
                if ((tid & 63u) == 0) {
                    lds.m[wave][r] = part.m[r];
                    lds.l[wave][r] = part.l[r];
                }
            }
        }
        __syncthreads();
        for (uint32_t i = tid; i < at_once * kRows * D; i += kBlock) {
            uint32_t const d = i % D;
            uint32_t const r = i / D % kRows;
            uint32_t const w = i / D / kRows * split;
            uint32_t const mine = t0 + w / split;
            uint32_t const c = mine % batches * kRows + r;
            if (mine >= tasks || !unit_column(P, a, u, table.layer, G, u.head + mine / batches, c).ok) continue;
            float M = -INFINITY;
            for (uint32_t s = 0; s < split; ++s) M = fmaxf(M, lds.m[w + s][r]);
            float o = 0.0f;
            float l = 0.0f;
            for (uint32_t s = 0; s < split; ++s) {
                float const f = lds.m[w + s][r] == -INFINITY ? 0.0f : exp2f(lds.m[w + s][r] - M);
                if (f == 0.0f) continue;   // whatever V made of it, as for a key of weight 0
                o += f * lds.o[w + s][r][d];
                l += f * lds.l[w + s][r];
            }
            PartOut const to = part_out(a, u, D, G, u.head + mine / batches, c);
            if (to.output != nullptr) {
                to.output[d] = output_half(o, l);
            } else {
                to.o[d] = o;
                if (d == 0) *to.ml = make_float2(M, l);
            }
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// Matrix-core path.  A wave holds kCB blocks of 16 columns and takes 32 kKB
// keys a step: S^T = K . Q^T, softmax with a reference point that moves
// lazily, O^T += V^T . P^T, all on v_mfma_f32_16x16x32_f16.  The keys of a
// 32-key block are permuted (HeadGroup readers below) so that the layout S^T
// leaves is the operand layout of P^T: lane l holds keys 8 (l / 16) .. + 7 of
// column l % 16.  Weights go to the matrix cores in two fp16 parts, p = hi +
// lo, which keep what 32-bit weights do to 2^-22.
// ---------------------------------------------------------------------------
constexpr float kLazyRescaleLog2 = 8.0f;
// Weights are 2^(s - m + kWeightShift), at most 2^15, so that lo stays a
// normal fp16 number down to 2^-9 of the largest weight.
constexpr float kWeightShift = 7.0f;

template <uint32_t kDim, uint32_t kCB>
struct Columns {
    static constexpr uint32_t kPanels = kDim / 32;
    static constexpr uint32_t kDb = kDim / 16;
    half8_t q[kCB][kPanels];
    float scale2[kCB];
    float m[kCB];   // reference point, -inf before the first finite score
    float l[kCB];   // of this lane's keys
    float4_t acc[kDb][kCB];   // O^T dims 16 db + 4 (l / 16) + i of column l % 16
    bool ok[kCB];
};

// Eight halves of a caller's row, whose address carries no alignment promise.
__device__ inline half8_t load_row8(const uint16_t* p)
{
    if ((reinterpret_cast<uintptr_t>(p) & 15u) == 0) return load_half8(p);
    half8_t v;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) v[i] = __builtin_bit_cast(_Float16, p[i]);
    return v;
}

// Column blocks from column c0 of the unit on.  Returns false when some
// column's scale does not keep the order of the scores.
template <uint32_t kDim, uint32_t kCB>
__device__ inline bool columns_init(Columns<kDim, kCB>& w, const PoolView& P, const SharedArgs& a, const SharedUnit& u,
                                    uint32_t layer, uint32_t G, uint32_t h, uint32_t c0)
{
    uint32_t const l = threadIdx.x & 63u;
    bool ordered = true;
#pragma unroll
    for (uint32_t cb = 0; cb < kCB; ++cb) {
        Column const c = unit_column(P, a, u, layer, G, h, c0 + 16 * cb + (l & 15u));
        w.ok[cb] = c.ok;
        w.scale2[cb] = c.ok ? c.scale2 : 1.0f;
        ordered = ordered && w.scale2[cb] > 0.0f && w.scale2[cb] < INFINITY;
        w.m[cb] = -INFINITY;
        w.l[cb] = 0.0f;
#pragma unroll
        for (uint32_t p = 0; p < kDim / 32; ++p) {
            w.q[cb][p] = half8_t{};
            if (c.ok) w.q[cb][p] = load_row8(c.query + 32 * p + 8 * (l >> 4));
        }
#pragma unroll
        for (uint32_t db = 0; db < kDim / 16; ++db) w.acc[db][cb] = float4_t{};
    }
    return ordered;
}

// kMasked: only the first nvalid of the step's keys count (their V is finite).
template <uint32_t kDim, uint32_t kCB, uint32_t kKB, bool kMasked>
__device__ __attribute__((always_inline)) inline void attend_step(Columns<kDim, kCB>& w, half8_t const (&k)[kKB][2][kDim / 32],
                                                                  half8_t const (&v)[kKB][kDim / 16], uint32_t nvalid)
{
    uint32_t const a8 = (threadIdx.x & 48u) >> 1;   // 8 (l / 16)
    float4_t s[kCB][kKB][2];
    float mx[kCB];
    bool over = false;
#pragma unroll
    for (uint32_t cb = 0; cb < kCB; ++cb) {
        mx[cb] = -INFINITY;
#pragma unroll
        for (uint32_t kb = 0; kb < kKB; ++kb) {
#pragma unroll
            for (uint32_t e = 0; e < 2; ++e) {
                float4_t z = {};
#pragma unroll
                for (uint32_t p = 0; p < kDim / 32; ++p) {
                    z = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[kb][e][p], w.q[cb][p], z, 0, 0, 0);
                }
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    if (kMasked && 32 * kb + a8 + 4 * e + i >= nvalid) z[i] = -INFINITY;
                    mx[cb] = fmaxf(mx[cb], z[i]);
                }
                s[cb][kb][e] = z;
            }
        }
        over = over || mx[cb] * w.scale2[cb] > w.m[cb] + kLazyRescaleLog2;
    }
    // The reference point moves, and what was summed is rescaled, only when a
    // score passes it by more than 2^8: a column's four lanes then agree on
    // the maximum.
    if (__builtin_expect(__any(over), 0)) {
        __asm__ volatile("" ::: "memory");   // not speculated
#pragma unroll
        for (uint32_t cb = 0; cb < kCB; ++cb) {
            float x = fmaxf(mx[cb], xor16(mx[cb]));
            x = fmaxf(x, xor32(x)) * w.scale2[cb];
            bool const grow = x > w.m[cb] + kLazyRescaleLog2;
            float const alpha = grow ? __builtin_amdgcn_exp2f(w.m[cb] - x) : 1.0f;
            if (grow) w.m[cb] = x;
            w.l[cb] *= alpha;
#pragma unroll
            for (uint32_t db = 0; db < kDim / 16; ++db) w.acc[db][cb] *= alpha;
        }
    }
#pragma unroll
    for (uint32_t cb = 0; cb < kCB; ++cb) {
        // Without a finite score yet the reference is 0: the weights are 2^-inf.
        float const mref = w.m[cb] == -INFINITY ? 0.0f : w.m[cb] - kWeightShift;
#pragma unroll
        for (uint32_t kb = 0; kb < kKB; ++kb) {
            half8_t hi, lo;
#pragma unroll
            for (uint32_t e = 0; e < 2; ++e) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    float const p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[cb][kb][e][i], w.scale2[cb], -mref));
                    _Float16 const h = static_cast<_Float16>(p);
                    w.l[cb] += p;
                    hi[4 * e + i] = h;
                    lo[4 * e + i] = static_cast<_Float16>(p - static_cast<float>(h));
                }
            }
#pragma unroll
            for (uint32_t db = 0; db < kDim / 16; ++db) {
                w.acc[db][cb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[kb][db], hi, w.acc[db][cb], 0, 0, 0);
                w.acc[db][cb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[kb][db], lo, w.acc[db][cb], 0, 0, 0);
            }
        }
    }
}

// The state as a part: denominators summed over the column's lanes, m the
// exponent's whole reference (-inf where there was no weight).  Returns
// whether some value of a column that counts is not finite.
template <uint32_t kDim, uint32_t kCB>
__device__ inline bool columns_finish(Columns<kDim, kCB>& w)
{
    float z = 0.0f;   // stays 0 unless a term is infinite or NaN
#pragma unroll
    for (uint32_t cb = 0; cb < kCB; ++cb) {
        w.l[cb] += xor16(w.l[cb]);
        w.l[cb] += xor32(w.l[cb]);
        w.m[cb] -= kWeightShift;   // -inf stays
        float4_t f = {w.l[cb] * 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t db = 0; db < kDim / 16; ++db) f += w.acc[db][cb] * 0.0f;
        z += w.ok[cb] ? (f[0] + f[1]) + (f[2] + f[3]) : 0.0f;
    }
    return z != 0.0f;
}

// ---- the unit's group table ---------------------------------------------------

constexpr uint32_t kTableGroups = 512;   // 4096 keys: no longer units on the matrix cores

struct TableFlags {
    uint32_t found;
    uint32_t generic;
    uint32_t first;
};

// Resolves the 8-key groups of [u.begin, u.end) for KV head u.head.  False
// where the table does not keep them aligned and whole: the unit then goes the
// generic path.  Called by every thread.
template <uint32_t kDim>
__device__ bool build_groups(const PoolView& P, const kimkv_decode_item& table, const SharedUnit& u, HeadGroup* groups,
                             TableFlags& flags)
{
    uint32_t const tid = threadIdx.x;
    uint32_t const ngroups = (u.end - u.begin + 7) / 8;
    if (ngroups > kTableGroups || (u.begin & 7u) != 0) return false;
    for (uint32_t g = tid; g < ngroups; g += kBlock) groups[g].k = nullptr;
    if (tid == 0) flags = TableFlags{0, 0, 0};
    __syncthreads();
    // The first entry is guessed before it is searched for: when every entry
    // before it is a full extent page of 64 tokens it is entry begin / 64.
    auto add = [&](uint32_t first) {
        for (uint32_t j = tid; j <= ngroups && first + j < table.descriptor_count; j += kBlock) {
            kimkv_block_desc const e = table.descriptors[first + j];
            if (j == 0 && e.logical_token_begin <= u.begin && u.begin - e.logical_token_begin < e.valid_tokens) flags.found = 1;
            add_head_groups<kDim>(P, e, table.layer, u.head, u.begin, u.end, table.token_count, groups, &flags.generic);
        }
        __syncthreads();
    };
    add(min(u.begin / 64u, table.descriptor_count - 1));
    if (flags.found == 0) {
        for (uint32_t g = tid; g < ngroups; g += kBlock) groups[g].k = nullptr;
        if (tid < kWave) {
            uint32_t const first = find_descriptor_wave(table.descriptors, table.descriptor_count, u.begin);
            if (tid == 0) flags.first = first;
        }
        __syncthreads();
        add(flags.first);
    }
    for (uint32_t g = tid; g < ngroups; g += kBlock) {
        if (groups[g].k == nullptr) flags.generic = 1;
    }
    __syncthreads();
    return flags.generic == 0;
}

// ---- direct units ---------------------------------------------------------------
// At most 16 columns.  The waves split the unit's heads, then its tokens, and
// read K and V^T straight into operand registers, two steps in flight: the
// work of lanes' own tokens and of groups too small to share a tile.  Bound by
// the bytes and, for short units, by the chain of reads in front of them.

template <uint32_t kDim>
struct DirectRows {
    static constexpr uint32_t kRow = kDim + 4;   // o, m, l, pad
    float row[kWaves][16][kRow];
    uint32_t ok[16];
};

template <uint32_t kDim>
__device__ bool unit_direct(const PoolView& P, const SharedArgs& a, const SharedUnit& u, const kimkv_decode_item& table,
                            const HeadGroup* groups, DirectRows<kDim>& rows)
{
    constexpr uint32_t kKB = kDim <= 64 ? 2 : 1;   // 32-key blocks a step
    constexpr uint32_t kStep = 32 * kKB;
    constexpr uint32_t kPanels = kDim / 32;
    constexpr uint32_t kDb = kDim / 16;
    uint32_t const tid = threadIdx.x;
    uint32_t const wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint32_t const l = tid & 63u;
    uint32_t const a4 = l >> 4;
    uint32_t const r = l & 15u;
    uint32_t const x = (l >> 2) & 3u;
    uint32_t const G = a.QH / P.heads;
    uint32_t const hs = u.heads <= 1 ? 1 : u.heads <= 2 ? 2 : u.heads <= 4 ? 4 : 8;   // heads' share of the waves
    uint32_t const split = kWaves / hs;
    uint32_t const head = wave % hs;
    uint32_t const piece = ((u.end - u.begin + split - 1) / split + 31) / 32 * 32;
    uint32_t const c0 = min(wave / hs * piece, u.end - u.begin);   // relative to begin
    uint32_t const c1 = min(c0 + piece, u.end - u.begin);
    bool const works = head < u.heads;
    Columns<kDim, 1> w;
    bool ordered = columns_init(w, P, a, u, table.layer, G, works ? u.head + head : u.head, 0);
    if (wave == 0 && l < 16) rows.ok[l] = w.ok[0] ? 1 : 0;
    struct Ops {
        half8_t k[kKB][2][kPanels];
        half8_t v[kKB][kDb];
    };
    auto load = [&](Ops& o, uint32_t t0, auto tail) {
        constexpr bool kTail = decltype(tail)::value;
#pragma unroll
        for (uint32_t kb = 0; kb < kKB; ++kb) {
            uint32_t const tk = t0 + 32 * kb + 8 * x;
            HeadGroup const gk = groups[(kTail ? min(tk, c1 - 1) : tk) / 8];
            const uint16_t* const k0 = gk.k + head * (2u * kDim / 32u) * gk.kpanel;   // 2 cap D a head
#pragma unroll
            for (uint32_t e = 0; e < 2; ++e) {
                const uint16_t* const row = k0 + (4 * e + (l & 3u)) * 32 + a4 * 8;
#pragma unroll
                for (uint32_t p = 0; p < kPanels; ++p) {
                    o.k[kb][e][p] = half8_t{};
                    if (!kTail || tk + 4 * e + (l & 3u) < c1) o.k[kb][e][p] = load_half8_stream(row + p * gk.kpanel);
                }
            }
            uint32_t const tv = t0 + 32 * kb + 8 * a4;
            HeadGroup const gv = groups[(kTail ? min(tv, c1 - 1) : tv) / 8];
            const uint16_t* const v0 = gv.v + head * (2u * kDim / 32u) * gv.kpanel + r * gv.vw;
#pragma unroll
            for (uint32_t db = 0; db < kDb; ++db) {
                o.v[kb][db] = half8_t{};
                if (!kTail || tv < c1) o.v[kb][db] = load_half8_stream(v0 + 16 * db * gv.vw);
            }
            if (kTail && tv < c1 && tv + 8 > c1) {   // keys past the end may hold anything
#pragma unroll
                for (uint32_t db = 0; db < kDb; ++db) {
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j) {
                        if (tv + j >= c1) o.v[kb][db][j] = static_cast<_Float16>(0.0f);
                    }
                }
            }
        }
    };
    auto full = [&](Ops const& o) { attend_step<kDim, 1, kKB, false>(w, o.k, o.v, kStep); };
    std::false_type const whole{};
    if (works && c0 < c1) {
        Ops buf_a, buf_b;
        uint32_t const steps = (c1 - c0) / kStep;
        uint32_t t = c0;
        if (steps > 0) {
            load(buf_a, t, whole);
            uint32_t i = 1;
            for (; i + 1 < steps; i += 2) {
                load(buf_b, t + kStep, whole);
                full(buf_a);
                load(buf_a, t + 2 * kStep, whole);
                full(buf_b);
                t += 2 * kStep;
            }
            if (i < steps) {
                load(buf_b, t + kStep, whole);
                full(buf_a);
                full(buf_b);
                t += 2 * kStep;
            } else {
                full(buf_a);
                t += kStep;
            }
        }
        if (t < c1) {
            load(buf_a, t, std::true_type{});
            attend_step<kDim, 1, kKB, true>(w, buf_a.k, buf_a.v, c1 - t);
        }
    }
    bool const again = columns_finish(w) || !ordered;
    float* const mine = rows.row[wave][r];
#pragma unroll
    for (uint32_t db = 0; db < kDb; ++db) *reinterpret_cast<float4_t*>(mine + 16 * db + 4 * a4) = w.acc[db][0];
    if (l < 16) {
        mine[kDim] = w.m[0];
        mine[kDim + 1] = w.l[0];
    }
    if (__syncthreads_or(again) != 0) return false;
    for (uint32_t i = tid; i < u.heads * 16 * (kDim / 4); i += kBlock) {
        uint32_t const d = i % (kDim / 4) * 4;
        uint32_t const c = i / (kDim / 4) % 16;
        uint32_t const hd = i / (kDim / 4) / 16;
        if (c >= u.cols || rows.ok[c] == 0) continue;
        float M = -INFINITY;
        for (uint32_t s = 0; s < split; ++s) M = fmaxf(M, rows.row[s * hs + hd][c][kDim]);
        float4_t o = {};
        float den = 0.0f;
        for (uint32_t s = 0; s < split; ++s) {
            const float* const part = rows.row[s * hs + hd][c];
            float const f = part[kDim] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(part[kDim] - M);
            o += f * *reinterpret_cast<const float4_t*>(part + d);
            den += f * part[kDim + 1];
        }
        PartOut const to = part_out(a, u, kDim, G, u.head + hd, c);
        if (to.output != nullptr) {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) to.output[d + j] = output_half(o[j], den);
        } else {
            *reinterpret_cast<float4_t*>(to.o + d) = o;
            if (d == 0) *to.ml = make_float2(M, den);
        }
    }
    return true;
}

// ---- staged units ---------------------------------------------------------------
// Whole 64-key blocks of one KV head and up to 64 kCB columns.  Each half of
// the workgroup takes every other tile: its 256 threads stage it in LDS, and
// its four waves compute kCB blocks of 16 columns each from it.  The halves'
// states are merged in LDS, so that a unit leaves one part.

template <uint32_t kDim>
struct StagedLds {
    union {
        KvTile<kDim> tile[2][2];                // [half][buffer]
        struct {
            float4_t acc[4][16][64];            // [column wave][register][lane]
            float2 ml[4][4][64];
        } part;
    };
};

template <uint32_t kDim, uint32_t kCB>
__device__ bool unit_staged(const PoolView& P, const SharedArgs& a, const SharedUnit& u, const kimkv_decode_item& table,
                            const HeadGroup* groups, StagedLds<kDim>& lds)
{
    using Dims = TileDims<kDim>;
    constexpr uint32_t kPanels = kDim / 32;
    constexpr uint32_t kDb = kDim / 16;
    constexpr uint32_t kGroups = Dims::kTileKeys / 8;
    static_assert(kDb * kCB <= 16 && kCB <= 4, "a wave's state fits its part");
    uint32_t const wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t const half = wave >> 2;
    uint32_t const cw = wave & 3u;
    uint32_t const tid = threadIdx.x & (kTileThreads - 1);
    uint32_t const l = tid & 63u;
    uint32_t const a4 = l >> 4;
    uint32_t const r = l & 15u;
    uint32_t const x = (l >> 2) & 3u;
    uint32_t const G = a.QH / P.heads;
    uint32_t const tiles = (u.end - u.begin) / Dims::kTileKeys;
    uint32_t const rounds = (tiles + 1) / 2;
    TileLoad ld;
    if (half < tiles) {
        tile_fetch<kDim, true>(ld, groups, half * kGroups, Dims::kTileKeys, tid);
        tile_store(lds.tile[half][0], ld, tid);
    }
    if (half + 2 < tiles) tile_fetch<kDim, true>(ld, groups, (half + 2) * kGroups, Dims::kTileKeys, tid);
    Columns<kDim, kCB> w;
    bool const ordered = columns_init(w, P, a, u, table.layer, G, u.head, cw * 16 * kCB);
    bool const works = cw * 16 * kCB < u.cols;
    __syncthreads();
    for (uint32_t i = 0; i < rounds; ++i) {
        uint32_t const j = 2 * i + half;
        KvTile<kDim> const& tile = lds.tile[half][i & 1u];
        if (works && j < tiles) {
#pragma unroll
            for (uint32_t kb = 0; kb < Dims::kKB; ++kb) {
                half8_t k[1][2][kPanels];
                half8_t v[1][kDb];
#pragma unroll
                for (uint32_t e = 0; e < 2; ++e) {
#pragma unroll
                    for (uint32_t p = 0; p < kPanels; ++p) {
                        k[0][e][p] = tile.k[k_unit<kDim>(32 * kb + 8 * x + 4 * e + (l & 3u), 4 * p + a4)];
                    }
                }
#pragma unroll
                for (uint32_t db = 0; db < kDb; ++db) v[0][db] = tile.v[v_unit<kDim>(16 * db + r, 4 * kb + a4)];
                attend_step<kDim, kCB, 1, false>(w, k, v, 32);
            }
        }
        if (j + 2 < tiles) tile_store(lds.tile[half][(i + 1) & 1u], ld, tid);
        if (j + 4 < tiles) tile_fetch<kDim, true>(ld, groups, (j + 4) * kGroups, Dims::kTileKeys, tid);
        __syncthreads();
    }
    bool const again = columns_finish(w) || !ordered;
    if (half == 1) {
#pragma unroll
        for (uint32_t cb = 0; cb < kCB; ++cb) {
#pragma unroll
            for (uint32_t db = 0; db < kDb; ++db) lds.part.acc[cw][db * kCB + cb][l] = w.acc[db][cb];
            lds.part.ml[cw][cb][l] = make_float2(w.m[cb], w.l[cb]);
        }
    }
    if (__syncthreads_or(again) != 0) return false;
    if (half == 1 || !works) return true;
#pragma unroll
    for (uint32_t cb = 0; cb < kCB; ++cb) {
        uint32_t const c = (cw * kCB + cb) * 16 + r;
        if (!w.ok[cb]) continue;
        float2 const other = lds.part.ml[cw][cb][l];
        float const M = fmaxf(w.m[cb], other.x);
        float const f0 = w.m[cb] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(w.m[cb] - M);
        float const f1 = other.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(other.x - M);
        float const den = f0 * w.l[cb] + f1 * other.y;
        PartOut const to = part_out(a, u, kDim, G, u.head, c);
#pragma unroll
        for (uint32_t db = 0; db < kDb; ++db) {
            float4_t const o = f0 * w.acc[db][cb] + f1 * lds.part.acc[cw][db * kCB + cb][l];
            uint32_t const d = 16 * db + 4 * a4;
            if (to.output != nullptr) {
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) to.output[d + j] = output_half(o[j], den);
            } else {
                *reinterpret_cast<float4_t*>(to.o + d) = o;
            }
        }
        if (to.output == nullptr && a4 == 0) *to.ml = make_float2(M, den);
    }
    return true;
}

// Dims with a matrix-core path, and with tiles.
constexpr bool direct_dim(uint32_t D) { return D == 64 || D == 96 || D == 128; }
constexpr bool staged_dim(uint32_t D) { return D == 64 || D == 128; }

struct NoLds {};

// kDim: the head dim, or 0 for one that has only the generic path.
template <uint32_t kDim>
__global__ __launch_bounds__(kBlock) __attribute__((amdgpu_waves_per_eu(2, 2))) void shared_decode_kernel(PoolView P,
                                                                                                         SharedArgs a)
{
    // One workgroup a compute unit (its registers see to that), so the paths' memory may be large.
    union Paths {
        GenericLds generic;
        std::conditional_t<direct_dim(kDim), DirectRows<kDim == 0 ? 64 : kDim>, NoLds> direct;
        std::conditional_t<staged_dim(kDim), StagedLds<staged_dim(kDim) ? kDim : 64>, NoLds> staged;
    };
    __shared__ __attribute__((aligned(16))) unsigned char path_lds[sizeof(Paths)];
    __shared__ HeadGroup groups[kDim != 0 ? kTableGroups : 1];
    __shared__ TableFlags flags;
    Paths& lds = *reinterpret_cast<Paths*>(path_lds);
    SharedUnit const u = a.units[xcd_logical_index(blockIdx.x, gridDim.x)];
    if (u.cols == 0) return;
    uint32_t const G = a.QH / P.heads;
    // The entries lie in the caller's memory: nothing outside the launch's buffers is touched, whatever they hold.
    uint64_t const last = (static_cast<uint64_t>(u.col0) + u.cols - 1) / G;   // lane of the last column, from u.lane
    if (u.table_lane >= a.lane_count || u.lane + last >= a.lane_count || u.heads == 0 || u.head + u.heads > P.heads
        || u.begin >= u.end || ((u.kind & kSingle) == 0 && u.slot + last >= a.slot_count)) {
        report_fault(P, KIMKV_FAULT_DECODE_ITEM);
        return;
    }
    kimkv_decode_item const table = a.items[u.table_lane];
    uint32_t const planned = a.lanes[u.table_lane].tokens;
    if (!lane_valid(P, table, planned) || u.end > planned) {
        report_fault(P, KIMKV_FAULT_DECODE_ITEM);
        return;
    }
    bool bad = false;
    for (uint32_t c = threadIdx.x; c < u.cols; c += kBlock) bad |= !unit_column(P, a, u, table.layer, G, u.head, c).ok;
    if (bad && P.faults != nullptr) atomicOr(P.faults, KIMKV_FAULT_DECODE_ITEM);
    if constexpr (kDim != 0) {
        bool done = false;
        uint32_t const kind = u.kind & ~kSingle;
        if (build_groups<kDim>(P, table, u, groups, flags)) {
            if (kind == kDirect) {
                if (u.cols <= 16 && u.heads <= kWaves) done = unit_direct<kDim>(P, a, u, table, groups, lds.direct);
            } else if constexpr (staged_dim(kDim)) {
                bool const whole = u.heads == 1 && (u.begin & 63u) == 0 && (u.end & 63u) == 0 && u.cols <= 64 * kind;
                if (whole && kind == 1) done = unit_staged<kDim, 1>(P, a, u, table, groups, lds.staged);
                if (whole && kind == 2) done = unit_staged<kDim, 2>(P, a, u, table, groups, lds.staged);
                if constexpr (kDim == 64) {
                    if (whole && kind == 4) done = unit_staged<kDim, 4>(P, a, u, table, groups, lds.staged);
                }
            }
        }
        if (done) return;
        __syncthreads();   // the generic path's rows take the same memory
    }
    unit_generic(P, a, u, lds.generic);
}

// Merges the lanes' parts, four dims a thread (one where the head dim is no
// multiple of 4).  Bound by the parts' bytes, which the launch before has just
// written; kBatch parts are in flight together.
constexpr unsigned kMergeBlock = 256;

template <uint32_t kWidth>
__global__ __launch_bounds__(kMergeBlock) void shared_merge_kernel(PoolView P, SharedArgs a)
{
    constexpr uint32_t kBatch = 8;
    typedef float vec_t __attribute__((ext_vector_type(kWidth)));
    uint32_t const lane = blockIdx.x;
    SharedLane const rec = a.lanes[lane];
    if (rec.merged == 0 || !lane_ok(P, a, lane)) return;   // a unit reported it
    uint64_t const last_prefix = rec.prefix_slot + static_cast<uint64_t>(rec.prefix_stride) * (rec.prefix_count - 1ull);
    if (rec.prefix_count > a.slot_count || rec.tail_count > a.slot_count
        || (rec.prefix_count != 0 && last_prefix >= a.slot_count)
        || static_cast<uint64_t>(rec.tail_slot) + rec.tail_count > a.slot_count) {
        return;
    }
    uint32_t const D = P.dim;
    uint32_t const parts = rec.prefix_count + rec.tail_count;
    uint16_t* const output = a.items[lane].output;
    uint32_t const per_row = D / kWidth;
    for (uint32_t x = blockIdx.y * kMergeBlock + threadIdx.x; x < a.QH * per_row; x += gridDim.y * kMergeBlock) {
        uint32_t const q = x / per_row;
        uint32_t const d = (x - q * per_row) * kWidth;
        float M = -INFINITY;
        float l = 0.0f;
        vec_t o = {};
        for (uint32_t i0 = 0; i0 < parts; i0 += kBatch) {
            float2 ml[kBatch];
            vec_t row[kBatch];
#pragma unroll
            for (uint32_t j = 0; j < kBatch; ++j) {
                uint32_t const i = min(i0 + j, parts - 1);
                uint32_t const slot = i < rec.prefix_count ? rec.prefix_slot + i * rec.prefix_stride
                                                           : rec.tail_slot + (i - rec.prefix_count);
                uint64_t const at = static_cast<uint64_t>(slot) * a.QH + q;
                ml[j] = a.parts.ml[at];
                row[j] = *reinterpret_cast<const vec_t*>(a.parts.o + at * D + d);
                if (i0 + j >= parts) ml[j].x = -INFINITY;
            }
            float m_new = M;
#pragma unroll
            for (uint32_t j = 0; j < kBatch; ++j) m_new = fmaxf(m_new, ml[j].x);
            float const c = M == -INFINITY ? 0.0f : exp2f(M - m_new);
            M = m_new;
            o *= c;
            l *= c;
#pragma unroll
            for (uint32_t j = 0; j < kBatch; ++j) {
                float const f = ml[j].x == -INFINITY ? 0.0f : exp2f(ml[j].x - M);
                if (f == 0.0f) continue;   // whatever V made of it, as for a key of weight 0
                o += f * row[j];
                l += f * ml[j].y;
            }
        }
        uint16_t* const to = output + static_cast<uint64_t>(q) * D + d;
#pragma unroll
        for (uint32_t j = 0; j < kWidth; ++j) to[j] = output_half(o[j], l);
    }
}

// ---- planning -----------------------------------------------------------------

constexpr uint32_t kShareBlock = 64;     // tokens: a shared prefix is cut to whole blocks
constexpr uint32_t kMaxUnit = kTableGroups * 8;

// What a unit costs its compute unit, in nanoseconds.
struct UnitCost {
    uint32_t D;
    static constexpr double kStart = 3000;   // the chain of reads in front, the merge and the stores behind
    double direct(uint32_t heads, uint32_t tokens) const { return kStart + 10.0 * D / 64 * heads * tokens; }
    double staged(uint32_t blocks, uint32_t tokens) const { return kStart + 700.0 * blocks + 4.5 * D / 64 * blocks * tokens; }
};

struct Planned {
    std::vector<SharedUnit> units;
    std::vector<double> cost;
    std::vector<SharedLane> lanes;
    uint64_t slots{0};
    uint32_t merge_lanes{0};
};

uint64_t align16(uint64_t n) { return (n + 15) / 16 * 16; }

// Spreads the units over the XCDs (workgroup w runs on XCD w % 8): units of
// one range of keys and head together, whose K and V then stay in one L2, the
// costliest first onto the XCD with least to do, and each XCD's costliest
// first.  Short lists end in idle entries.
void place_units(Planned& p)
{
    size_t const n = p.units.size();
    struct Bundle {
        size_t first, count;
        double cost;
    };
    std::vector<Bundle> bundles;
    for (size_t i = 0; i < n; ++i) {
        SharedUnit const& u = p.units[i];
        if (!bundles.empty()) {
            SharedUnit const& b = p.units[bundles.back().first];
            if (b.table_lane == u.table_lane && b.begin == u.begin && b.end == u.end && b.head == u.head) {
                bundles.back().count += 1;
                bundles.back().cost += p.cost[i];
                continue;
            }
        }
        bundles.push_back(Bundle{i, 1, p.cost[i]});
    }
    std::stable_sort(bundles.begin(), bundles.end(), [](Bundle const& x, Bundle const& y) { return x.cost > y.cost; });
    std::vector<size_t> xcd[kXcds];
    double load[kXcds] = {};
    for (Bundle const& b : bundles) {
        uint32_t best = 0;
        for (uint32_t x = 1; x < kXcds; ++x) {
            if (load[x] < load[best] || (load[x] == load[best] && xcd[x].size() < xcd[best].size())) best = x;
        }
        load[best] += b.cost;
        for (size_t i = 0; i < b.count; ++i) xcd[best].push_back(b.first + i);
    }
    size_t length = 0;
    for (auto& list : xcd) {
        std::stable_sort(list.begin(), list.end(), [&](size_t x, size_t y) { return p.cost[x] > p.cost[y]; });
        length = std::max(length, list.size());
    }
    std::vector<SharedUnit> placed(length * kXcds, SharedUnit{});
    for (uint32_t x = 0; x < kXcds; ++x) {
        for (size_t i = 0; i < xcd[x].size(); ++i) placed[x * length + i] = p.units[xcd[x][i]];
    }
    p.units = std::move(placed);
}

// Tokens of each of the pieces of [0, tokens), in blocks of 64.
uint32_t piece_tokens(uint64_t tokens, double pieces)
{
    uint64_t const n = std::max<uint64_t>(1, std::max<uint64_t>(static_cast<uint64_t>(pieces + 0.5), (tokens + kMaxUnit - 1) / kMaxUnit));
    return static_cast<uint32_t>(std::max<uint64_t>(64, ((tokens + n - 1) / n + 63) / 64 * 64));
}

bool plan_batch(uint32_t H, uint32_t D, uint32_t QH, uint32_t compute_units, const uint32_t* tokens, uint32_t lane_count,
                const kimkv_shared_group* groups, uint32_t group_count, Planned& out)
{
    uint32_t const G = QH / H;
    UnitCost const unit_cost{D};
    uint32_t const max_blocks = D == 64 ? 4 : staged_dim(D) ? 2 : 0;
    out.lanes.resize(lane_count);
    for (uint32_t i = 0; i < lane_count; ++i) out.lanes[i] = SharedLane{i, tokens[i], 0, 0, 0, 0, 0, 0};
    std::vector<uint8_t> grouped(lane_count, 0);
    std::vector<uint32_t> shared(lane_count, 0);   // tokens of the lane that a group's units take
    struct Shared {
        uint32_t lane, lanes, prefix, blocks;   // blocks: of 16 columns a wave, 0 for direct units
        uint64_t tiles;                         // column tiles
    };
    std::vector<Shared> prefixes;
    double total = 0;
    for (uint32_t g = 0; g < group_count; ++g) {
        kimkv_shared_group const& group = groups[g];
        if (group.first_lane > lane_count || group.lane_count > lane_count - group.first_lane) return false;
        uint32_t prefix = group.prefix_tokens;
        for (uint32_t i = group.first_lane; i < group.first_lane + group.lane_count; ++i) {
            if (grouped[i] != 0) return false;
            grouped[i] = 1;
            prefix = std::min(prefix, tokens[i]);
        }
        prefix = prefix / kShareBlock * kShareBlock;
        if (group.lane_count < 2 || prefix == 0) continue;
        uint64_t const columns = static_cast<uint64_t>(group.lane_count) * G;
        if (columns > 0x7FFFFFFFu) return false;
        Shared s{group.first_lane, group.lane_count, prefix, 0, (columns + 15) / 16};
        if (columns > 32 && max_blocks != 0) {
            s.blocks = columns <= 64 ? 1 : columns <= 128 || max_blocks == 2 ? 2 : 4;
            s.tiles = (columns + 64 * s.blocks - 1) / (64 * s.blocks);
        }
        prefixes.push_back(s);
        for (uint32_t i = 0; i < group.lane_count; ++i) shared[group.first_lane + i] = prefix;
        double const whole = s.blocks != 0 ? unit_cost.staged(s.blocks, prefix) : unit_cost.direct(1, prefix);
        total += whole * static_cast<double>(s.tiles) * H;
    }
    uint32_t heads = 1;   // KV heads of a unit of a lane's own tokens
    while (heads < 8 && heads < H) heads *= 2;
    uint64_t own_units = 0;
    for (uint32_t i = 0; i < lane_count; ++i) {
        if (tokens[i] == shared[i]) continue;
        own_units += static_cast<uint64_t>((H + heads - 1) / heads) * ((G + 15) / 16);
        total += unit_cost.direct(H, tokens[i] - shared[i]) * ((G + 15) / 16);
    }
    // Fewer heads a unit, and more waves for each, while the units are few.
    while (heads > 1 && own_units * 4 <= compute_units) {
        heads /= 2;
        own_units *= 2;
    }
    // Each compute unit is to take about the same: pieces of that cost, but
    // none so short that starting it costs more than its work.
    double const share = std::max(total / compute_units, 3 * UnitCost::kStart);
    auto push = [&](SharedUnit u, double cost) {
        out.units.push_back(u);
        out.cost.push_back(cost);
    };
    for (Shared const& s : prefixes) {
        double const whole = s.blocks != 0 ? unit_cost.staged(s.blocks, s.prefix) : unit_cost.direct(1, s.prefix);
        uint32_t const piece = piece_tokens(s.prefix, whole / share);
        uint32_t const pieces = (s.prefix + piece - 1) / piece;
        uint32_t const width = s.blocks != 0 ? 64 * s.blocks : 16;
        uint32_t const columns = s.lanes * G;
        if (out.slots + static_cast<uint64_t>(s.lanes) * pieces > 0x7FFFFFFFu) return false;
        for (uint32_t i = 0; i < s.lanes; ++i) {
            SharedLane& lane = out.lanes[s.lane + i];
            lane.table_lane = s.lane;
            lane.prefix_slot = static_cast<uint32_t>(out.slots + i);
            lane.prefix_stride = s.lanes;
            lane.prefix_count = pieces;
        }
        for (uint64_t at = 0; at < s.prefix; at += piece) {
            auto const b = static_cast<uint32_t>(at);
            auto const end = static_cast<uint32_t>(std::min<uint64_t>(s.prefix, at + piece));
            for (uint32_t h = 0; h < H; ++h) {
                for (uint32_t c = 0; c < columns; c += width) {
                    push(SharedUnit{s.lane, s.lane, c, std::min(width, columns - c), b, end, static_cast<uint32_t>(out.slots),
                                    static_cast<uint16_t>(h), 1, static_cast<uint8_t>(s.blocks)},
                         s.blocks != 0 ? unit_cost.staged(s.blocks, end - b) : unit_cost.direct(1, end - b));
                }
            }
            out.slots += s.lanes;
        }
    }
    for (uint32_t i = 0; i < lane_count; ++i) {
        SharedLane& lane = out.lanes[i];
        uint32_t const own = tokens[i] - shared[i];
        if (own == 0) {
            lane.merged = lane.prefix_count != 0 ? 1 : 0;
            out.merge_lanes += lane.merged;
            continue;
        }
        uint32_t const piece = piece_tokens(own, unit_cost.direct(heads, own) / share);
        uint32_t const pieces = (own + piece - 1) / piece;
        bool const single = pieces == 1 && lane.prefix_count == 0;
        if (out.slots + pieces > 0x7FFFFFFFu) return false;
        lane.tail_slot = static_cast<uint32_t>(out.slots);
        lane.tail_count = single ? 0 : pieces;
        lane.merged = single ? 0 : 1;
        out.merge_lanes += lane.merged;
        for (uint64_t b = shared[i]; b < tokens[i]; b += piece) {
            auto const end = static_cast<uint32_t>(std::min<uint64_t>(tokens[i], b + piece));
            for (uint32_t h = 0; h < H; h += heads) {
                uint32_t const n = std::min(heads, H - h);
                for (uint32_t c = 0; c < G; c += 16) {
                    push(SharedUnit{i, i, c, std::min(16u, G - c), static_cast<uint32_t>(b), end, static_cast<uint32_t>(out.slots),
                                    static_cast<uint16_t>(h), static_cast<uint8_t>(n),
                                    static_cast<uint8_t>(kDirect | (single ? kSingle : 0))},
                         unit_cost.direct(n, end - static_cast<uint32_t>(b)));
                }
            }
            if (!single) out.slots += 1;
        }
    }
    place_units(out);
    return out.slots <= 0x7FFFFFFFu && out.units.size() <= 0x7FFFFFFFu;
}

}  // namespace
}  // namespace kimkv

using namespace kimkv;

extern "C" {

kimkv_status kimkv_shared_decode_plan(uint32_t kv_heads, uint32_t head_dim, uint32_t query_heads,
                                      uint32_t compute_units, const uint32_t* token_counts, uint32_t lane_count,
                                      const kimkv_shared_group* groups, uint32_t group_count, void* entries,
                                      uint64_t capacity, kimkv_shared_plan* plan)
{
    if (plan == nullptr) return KIMKV_INVALID_ARGUMENT;
    *plan = kimkv_shared_plan{};
    if ((lane_count != 0 && token_counts == nullptr) || (group_count != 0 && groups == nullptr) || query_heads == 0
        || kv_heads == 0 || query_heads % kv_heads != 0 || kv_heads > 0xFFFFu || head_dim == 0 || head_dim > kMaxDim
        || lane_count > 0x7FFFFFFFu) {
        return KIMKV_INVALID_ARGUMENT;
    }
    try {
        Planned p;
        if (!plan_batch(kv_heads, head_dim, query_heads, compute_units == 0 ? 256 : compute_units, token_counts, lane_count,
                        groups, group_count, p)) {
            return KIMKV_INVALID_ARGUMENT;
        }
        uint64_t const unit_bytes = p.units.size() * sizeof(SharedUnit);
        uint64_t const lane_bytes = p.lanes.size() * sizeof(SharedLane);
        plan->entry_bytes = unit_bytes + lane_bytes;
        plan->workspace_bytes = align16(parts_o_floats(p.slots, query_heads, head_dim) * sizeof(float))
            + p.slots * query_heads * sizeof(float2);
        plan->kv_heads = kv_heads;
        plan->head_dim = head_dim;
        plan->query_heads = query_heads;
        plan->lane_count = lane_count;
        plan->unit_count = static_cast<uint32_t>(p.units.size());
        plan->slot_count = static_cast<uint32_t>(p.slots);
        plan->merge_lanes = p.merge_lanes;
        if (capacity < plan->entry_bytes || (plan->entry_bytes != 0 && entries == nullptr)) return KIMKV_INVALID_ARGUMENT;
        if (unit_bytes != 0) std::memcpy(entries, p.units.data(), unit_bytes);
        if (lane_bytes != 0) std::memcpy(static_cast<unsigned char*>(entries) + unit_bytes, p.lanes.data(), lane_bytes);
    } catch (std::exception const&) {
        *plan = kimkv_shared_plan{};
        return KIMKV_ALLOCATION_FAILED;
    }
    return KIMKV_OK;
}

kimkv_status kimkv_shared_decode_batch(const kimkv_storage* storage, const kimkv_decode_item* device_items,
                                       const void* device_entries, const kimkv_shared_plan* plan, void* workspace,
                                       kimkv_stream_t stream)
{
    if (storage == nullptr || plan == nullptr) return KIMKV_INVALID_ARGUMENT;
    if (plan->unit_count == 0 && plan->lane_count == 0) return KIMKV_OK;
    uint32_t const H = storage->layout.kv_heads;
    uint32_t const D = storage->layout.head_dim;
    if (plan->kv_heads != H || plan->head_dim != D || !on_current_device(storage)) return KIMKV_INVALID_ARGUMENT;
    if (plan->unit_count == 0) return KIMKV_OK;
    uint64_t const o_bytes = align16(parts_o_floats(plan->slot_count, plan->query_heads, D) * sizeof(float));
    if (device_items == nullptr || device_entries == nullptr || plan->lane_count == 0 || plan->query_heads == 0 || H == 0
        || plan->query_heads % H != 0 || D > kMaxDim || plan->unit_count > 0x7FFFFFFFu
        || (reinterpret_cast<uintptr_t>(device_entries) & 15u) != 0
        || plan->entry_bytes != plan->unit_count * sizeof(SharedUnit) + plan->lane_count * sizeof(SharedLane)
        || plan->workspace_bytes != o_bytes + static_cast<uint64_t>(plan->slot_count) * plan->query_heads * sizeof(float2)
        || (plan->slot_count != 0 && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0))) {
        return KIMKV_INVALID_ARGUMENT;
    }
    hipStream_t const s = native(stream);
    SharedArgs a{};
    a.items = device_items;
    a.units = static_cast<const SharedUnit*>(device_entries);
    a.lanes = reinterpret_cast<const SharedLane*>(a.units + plan->unit_count);
    a.parts.o = static_cast<float*>(workspace);
    a.parts.ml = reinterpret_cast<float2*>(static_cast<unsigned char*>(workspace) + o_bytes);
    a.lane_count = plan->lane_count;
    a.slot_count = plan->slot_count;
    a.QH = plan->query_heads;
    PoolView const pv = pool_view(*storage);
    void* start = nullptr;
    kernel_timing_begin(TimedKernel::Decode, s, &start);
    auto attend = [&](auto dim) { shared_decode_kernel<decltype(dim)::value><<<plan->unit_count, kBlock, 0, s>>>(pv, a); };
    if (D == 64) attend(std::integral_constant<uint32_t, 64>{});
    else if (D == 96) attend(std::integral_constant<uint32_t, 96>{});
    else if (D == 128) attend(std::integral_constant<uint32_t, 128>{});
    else attend(std::integral_constant<uint32_t, 0>{});
    kernel_timing_end(TimedKernel::Decode, s, start);
    kimkv_status const status = launch_status();
    if (status != KIMKV_OK || plan->merge_lanes == 0) return status;
    uint32_t const width = D % 4 == 0 ? 4 : 1;
    uint32_t const blocks = ceil_div(static_cast<uint64_t>(plan->query_heads) * D / width, kMergeBlock);
    dim3 const grid(plan->lane_count, blocks < 65535u ? blocks : 65535u);
    if (width == 4) shared_merge_kernel<4><<<grid, kMergeBlock, 0, s>>>(pv, a);
    else shared_merge_kernel<1><<<grid, kMergeBlock, 0, s>>>(pv, a);
    return launch_status();
}

}  // extern "C"
