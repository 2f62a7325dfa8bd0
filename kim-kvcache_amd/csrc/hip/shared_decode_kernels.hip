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
#include "device_common.h"
#include "runtime_internal.h"

namespace kimkv {
namespace {

// Workgroups of 8 waves, one a compute unit, or of 4, two a compute unit (256
// registers a lane either way): the plan says which.  Two hide one's start and
// end behind the other's keys, which short units gain by (lanes' own tokens;
// 4 lanes of 500 tokens 10.4 and 9.2 us, eight groups of four 21.8 and 20.1);
// one starts half as many units for the same keys, which long ones on many
// columns gain by (64 lanes of 128 dims on 4100 tokens 35.2 and 38.9 us, 128
// lanes on 16384 54.7 and 58.5).  (Passes over one set of inputs, which the
// caches hold in part; the first two take 9.0 and 22.0, the third 36.1 with
// inputs from memory.)
constexpr uint32_t kManyWaves = 8;
constexpr uint32_t kFewWaves = 4;
constexpr uint32_t kMaxDim = 256;

// How a unit is computed.
constexpr uint8_t kSingle = 0x80;   // the lane has no other part; the rest: 1, 2 or 4 blocks of 16 columns a wave

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
    Divisor group;   // query heads a KV head
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

// Reports a column whose lane cannot be computed.
__device__ inline void report_column(const PoolView& P, bool missing)
{
    if (missing && P.faults != nullptr) atomicOr(P.faults, KIMKV_FAULT_DECODE_ITEM);
}

// One column of a unit: its lane's item and query head in the group; !ok
// where the lane is planned with no tokens, or `missing`: its item is not as
// planned, or of another layer than the table's.
struct Column {
    const uint16_t* query;   // row of KV head 0
    uint16_t* output;
    float scale2;            // attention scale * log2 e
    uint32_t lane;           // from u.lane on
    uint32_t q;
    bool ok;
    bool missing;
};

__device__ inline Column unit_column(const PoolView& P, const SharedArgs& a, const SharedUnit& u, uint32_t layer, uint32_t c)
{
    Column out{};
    out.lane = div_mod(u.col0 + min(c, u.cols - 1), a.group, &out.q);
    kimkv_decode_item const item = a.items[u.lane + out.lane];
    uint32_t const planned = a.lanes[u.lane + out.lane].tokens;
    out.ok = c < u.cols && lane_valid(P, item, planned) && item.layer == layer;
    out.missing = c < u.cols && planned != 0 && !out.ok;
    out.query = item.query + out.q * P.dim;
    out.output = item.output + out.q * P.dim;
    out.scale2 = item.attention_scale * kLog2e;
    return out;
}

// Where a column's parts go (KV head h: G h rows further), or its output
// where the lane has one part.
struct ColumnOut {
    uint64_t row;
    uint16_t* output;
    uint32_t ok;
};

__device__ inline ColumnOut column_out(const SharedArgs& a, const SharedUnit& u, const Column& c)
{
    return ColumnOut{static_cast<uint64_t>(u.slot + c.lane) * a.QH + c.q, (u.kind & kSingle) != 0 ? c.output : nullptr,
                     c.ok ? 1u : 0u};
}

// o / l as an output: 0 for a row without any weight, l itself where it is not finite or NaN.
__device__ inline uint16_t output_half(float o, float l)
{
    return __half_as_ushort(__float2half_rn(l > 0.0f ? o / l : l == 0.0f ? 0.0f : l));
}

// kWidth outputs o / l, in one store where the address allows it.
template <uint32_t kWidth, typename Vec>
__device__ inline void store_outputs(uint16_t* to, const Vec& o, float l)
{
    float const inv = l > 0.0f ? 1.0f / l : 0.0f;
    uint16_t v[kWidth];
#pragma unroll
    for (uint32_t j = 0; j < kWidth; ++j) v[j] = l >= 0.0f ? __half_as_ushort(__float2half_rn(o[j] * inv)) : output_half(o[j], l);
    if (kWidth == 4 && (reinterpret_cast<uintptr_t>(to) & 7u) == 0) {
        *reinterpret_cast<uint2*>(to) = make_uint2(v[0] | static_cast<uint32_t>(v[1 % kWidth]) << 16,
                                                   v[2 % kWidth] | static_cast<uint32_t>(v[3 % kWidth]) << 16);
        return;
    }
#pragma unroll
    for (uint32_t j = 0; j < kWidth; ++j) to[j] = v[j];
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

// A sum of weighted values under a new reference: 0 where it weighs nothing, whatever V made of it.
__device__ inline float carried(float o, float factor) { return factor == 0.0f ? 0.0f : o * factor; }

// Whether a part of denominator l that weighs `factor` is left out: where it weighs nothing, unless a score was NaN.
__device__ inline bool left_out(float factor, float l) { return factor == 0.0f && l == l; }

// Parts of kRows rows: lane i holds o[r][k] of dim i + 64 k, every lane m and l.
struct RowParts {
    float o[kRows][4];
    float m[kRows];
    float l[kRows];
};

__device__ void attend_rows_generic(const PoolView& P, const kimkv_decode_item& table, uint32_t G, uint32_t h, uint32_t c0,
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
            q[r][k] = rows[r].ok && d < D ? __half2float(__ushort_as_half(rows[r].query[h * G * D + d])) : 0.0f;
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
            // The maximum passes over NaN scores; their weights carry them into the sum.
            float const m_new = fmaxf(out.m[r], wave_max(s[r]));
            float const m_top = m_new == -INFINITY ? 0.0f : m_new;
            float const alpha = m_new == -INFINITY ? 1.0f : exp2f(out.m[r] - m_new);
            p[r] = hb != nullptr ? exp2f(s[r] - m_top) : 0.0f;
            out.l[r] = out.l[r] * alpha + wave_sum(p[r]);
            out.m[r] = m_new;
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) out.o[r][k] = carried(out.o[r][k], alpha);
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
template <uint32_t kWaves>
struct GenericLds {
    float o[kWaves][kRows][kMaxDim];
    float m[kWaves][kRows];
    float l[kWaves][kRows];
};

// The whole unit by the generic path.  A task is kRows columns of one KV head;
// where there are fewer tasks than waves, the waves of a task take a part of
// the tokens each.
template <uint32_t kWaves>
__device__ void unit_generic(const PoolView& P, const SharedArgs& a, const SharedUnit& u, GenericLds<kWaves>& lds)
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
            for (uint32_t r = 0; r < kRows; ++r) {
                rows[r] = unit_column(P, a, u, table.layer, col0 + r);
                report_column(P, rows[r].missing);
            }
            RowParts part;
            attend_rows_generic(P, table, G, h, c0, c1, rows, part);
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
        for (uint32_t i = tid; i < at_once * kRows * D; i += kWaves * kWave) {
            uint32_t const d = i % D;
            uint32_t const r = i / D % kRows;
            uint32_t const w = i / D / kRows * split;
            uint32_t const mine = t0 + w / split;
            uint32_t const c = mine % batches * kRows + r;
            if (mine >= tasks || c >= columns) continue;
            Column const column = unit_column(P, a, u, table.layer, c);
            if (!column.ok) continue;
            float M = -INFINITY;
            for (uint32_t s = 0; s < split; ++s) M = fmaxf(M, lds.m[w + s][r]);
            float o = 0.0f;
            float l = 0.0f;
            for (uint32_t s = 0; s < split; ++s) {
                float const f = lds.m[w + s][r] == -INFINITY ? 0.0f : exp2f(lds.m[w + s][r] - M);
                if (left_out(f, lds.l[w + s][r])) continue;
                o += f * lds.o[w + s][r][d];
                l += f * lds.l[w + s][r];
            }
            ColumnOut const to = column_out(a, u, column);
            uint32_t const q = (u.head + mine / batches) * G;
            if (to.output != nullptr) {
                to.output[q * D + d] = output_half(o, l);
            } else {
                a.parts.o[(to.row + q) * D + d] = o;
                if (d == 0) a.parts.ml[to.row + q] = make_float2(M, l);
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
// lo, each cut off behind its bits, so a weight is kept to 2^-20 of itself.
// ---------------------------------------------------------------------------
// Weights are 2^(s - m + kWeightShift), at most 2^15, so that lo stays a
// normal fp16 number down to 2^-9 of the largest weight.
constexpr float kWeightShift = 7.0f;

template <uint32_t kDim, uint32_t kCB>
struct Columns {
    static constexpr uint32_t kPanels = kDim / 32;
    static constexpr uint32_t kDb = kDim / 16;
    half8_t q[kCB][kPanels];
    float scale2[kCB];
    float mref[kCB];   // weights are 2^(s - mref); inf (so 0) before the first finite score
    float l[kCB];   // of this lane's keys
    float4_t acc[kDb][kCB];   // O^T dims 16 db + 4 (l / 16) + i of column l % 16
    bool ok[kCB];
};

template <bool kStream>
__device__ __attribute__((always_inline)) inline half8_t load_keys(const uint16_t* p)
{
    return kStream ? load_half8_stream(p) : *reinterpret_cast<const global_half8_t*>(reinterpret_cast<uintptr_t>(p));
}

// Eight halves of a caller's row, whose address carries no alignment promise.
__device__ inline half8_t load_row8(const uint16_t* p)
{
    if ((reinterpret_cast<uintptr_t>(p) & 15u) == 0) return load_half8(p);
    half8_t v;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) v[i] = __builtin_bit_cast(_Float16, p[i]);
    return v;
}

// The unit's column blocks for KV head h, and where their parts go (outs, by
// the first wave).  Returns false when some column's scale does not keep the
// order of the scores.
template <uint32_t kDim, uint32_t kCB>
__device__ inline bool columns_init(Columns<kDim, kCB>& w, const PoolView& P, const SharedArgs& a, const SharedUnit& u,
                                    uint32_t layer, uint32_t h, ColumnOut* outs)
{
    // Lane i looks up column i of the wave's 16 kCB (a lane past them, one again) and hands it to the lanes that hold it.
    uint32_t const l = threadIdx.x & 63u;
    uint32_t const mine = l % (16 * kCB);
    Column const c = unit_column(P, a, u, layer, mine);
    auto const at = reinterpret_cast<uintptr_t>(c.query + h * a.group.d * kDim);
    auto const at_lo = static_cast<int>(at);
    auto const at_hi = static_cast<int>(at >> 32);
    if (threadIdx.x < 16 * kCB) outs[mine] = column_out(a, u, c);
    bool ordered = true;
#pragma unroll
    for (uint32_t cb = 0; cb < kCB; ++cb) {
        auto const from = static_cast<int>(16 * cb + (l & 15u));
        w.ok[cb] = __shfl(static_cast<int>(c.ok), from) != 0;
        auto const lo = static_cast<uint32_t>(__shfl(at_lo, from));
        auto const hi = static_cast<uint32_t>(__shfl(at_hi, from));
        float const scale2 = __shfl(c.scale2, from);
        const uint16_t* const row = reinterpret_cast<const uint16_t*>(static_cast<uint64_t>(hi) << 32 | lo);
#pragma unroll
        for (uint32_t p = 0; p < kDim / 32; ++p) {
            w.q[cb][p] = half8_t{};
            if (w.ok[cb]) w.q[cb][p] = load_row8(row + 32 * p + 8 * (l >> 4));
        }
        w.scale2[cb] = w.ok[cb] ? scale2 : 1.0f;
        ordered = ordered && w.scale2[cb] > 0.0f && w.scale2[cb] < INFINITY;
        w.mref[cb] = INFINITY;
        w.l[cb] = 0.0f;
#pragma unroll
        for (uint32_t db = 0; db < kDim / 16; ++db) w.acc[db][cb] = float4_t{};
    }
    report_column(P, c.missing);
    return ordered;
}

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

// Both rounded toward zero: one instruction for two, and what it leaves of a
// weight is taken up by the weight's second part.
__device__ inline half2_t two_halves(float a, float b)
{
    return __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(a, b));
}

// Only the first nvalid of the step's keys count (the others' V is finite).
// Written so that there is one copy of it in a loop, whatever the step: its
// instructions come from memory the first time, and a short unit runs them
// once or twice.
//
// The weights are made against the reference point as it stands, and their
// sum tells whether one of them passed 2^15: only then, and before the first
// finite score, is the maximum taken, the reference moved and the step's
// weights made anew.  (A maximum of every step's scores first costs half an
// instruction a score and puts it in front of the exponentials.)
template <uint32_t kDim, uint32_t kCB, uint32_t kKB>
__device__ __attribute__((always_inline)) inline void attend_step(Columns<kDim, kCB>& w, half8_t const (&k)[kKB][2][kDim / 32],
                                                                  half8_t const (&v)[kKB][kDim / 16], uint32_t nvalid)
{
    constexpr float kMostWeight = 32768.0f;
    // Not known to be -1, so that p - hi is one mixed-precision multiply-add.
    float minus_one = -1.0f;
    __asm__("" : "+s"(minus_one));
    float4_t s[kCB][kKB][2];
#pragma unroll
    for (uint32_t cb = 0; cb < kCB; ++cb) {
#pragma unroll
        for (uint32_t kb = 0; kb < kKB; ++kb) {
#pragma unroll
            for (uint32_t e = 0; e < 2; ++e) {
                float4_t z = {};
#pragma unroll
                for (uint32_t p = 0; p < kDim / 32; ++p) {
                    z = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[kb][e][p], w.q[cb][p], z, 0, 0, 0);
                }
                s[cb][kb][e] = z;
            }
        }
    }
    if (__builtin_expect(nvalid < 32 * kKB, 0)) {
        uint32_t a8 = (threadIdx.x & 48u) >> 1;   // 8 (l / 16)
        __asm__ volatile("" : "+v"(a8));          // a branch, not a selection of every score
#pragma unroll
        for (uint32_t kb = 0; kb < kKB; ++kb) {
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
                bool const gone = 32 * kb + a8 + j >= nvalid;
#pragma unroll
                for (uint32_t cb = 0; cb < kCB; ++cb) {
                    if (gone) s[cb][kb][j / 4][j % 4] = -INFINITY;
                }
            }
        }
    }
    half8_t hi[kCB][kKB], lo[kCB][kKB];
    float sum[kCB];
    bool over;
    float alpha[kCB];
#pragma unroll
    for (uint32_t cb = 0; cb < kCB; ++cb) alpha[cb] = 1.0f;
    uint32_t pass = 0;
#pragma unroll 1
    for (;;) {
        over = false;
#pragma unroll
        for (uint32_t cb = 0; cb < kCB; ++cb) {
            sum[cb] = 0.0f;
#pragma unroll
            for (uint32_t kb = 0; kb < kKB; ++kb) {
#pragma unroll
                for (uint32_t j = 0; j < 8; j += 2) {
                    float p[2];
#pragma unroll
                    for (uint32_t i = 0; i < 2; ++i) {
                        p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[cb][kb][j / 4][j % 4 + i], w.scale2[cb], -w.mref[cb]));
                    }
                    sum[cb] += p[0] + p[1];
                    half2_t const h = two_halves(p[0], p[1]);
                    half2_t const rest = two_halves(__builtin_fmaf(static_cast<float>(h[0]), minus_one, p[0]),
                                                    __builtin_fmaf(static_cast<float>(h[1]), minus_one, p[1]));
                    hi[cb][kb][j] = h[0];
                    hi[cb][kb][j + 1] = h[1];
                    lo[cb][kb][j] = rest[0];
                    lo[cb][kb][j + 1] = rest[1];
                }
            }
            over = over || !(sum[cb] <= kMostWeight) || w.mref[cb] == INFINITY;
        }
        if (__builtin_expect(!__any(over), 1)) break;
        // A column's four lanes agree on the maximum.  Once the reference
        // stands there the sums are small, unless a score is infinite or NaN,
        // which nothing helps.
        if (pass != 0) break;
        pass = 1;
        __asm__ volatile("" : "+s"(pass));   // a loop of two passes would be made into two copies
#pragma unroll
        for (uint32_t cb = 0; cb < kCB; ++cb) {
            float x = -INFINITY;
#pragma unroll
            for (uint32_t kb = 0; kb < kKB; ++kb) {
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) {
                    float score = s[cb][kb][j / 4][j % 4];
                    __asm__ volatile("" : "+v"(score));   // taken here, not in front of the loop
                    x = fmaxf(x, score);
                }
            }
            x = fmaxf(x, xor16(x));
            x = fmaxf(x, xor32(x)) * w.scale2[cb] - kWeightShift;
            bool const first = w.mref[cb] == INFINITY && x > -INFINITY;
            bool const grow = (first || x > w.mref[cb]) && x < INFINITY;
            if (grow && !first) alpha[cb] = __builtin_amdgcn_exp2f(w.mref[cb] - x);
            if (grow) w.mref[cb] = x;
        }
    }
    if (__builtin_expect(pass != 0, 0)) {
#pragma unroll
        for (uint32_t cb = 0; cb < kCB; ++cb) {
            w.l[cb] *= alpha[cb];
#pragma unroll
            for (uint32_t db = 0; db < kDim / 16; ++db) w.acc[db][cb] *= alpha[cb];
        }
    }
#pragma unroll
    for (uint32_t cb = 0; cb < kCB; ++cb) {
        w.l[cb] += sum[cb];
#pragma unroll
        for (uint32_t kb = 0; kb < kKB; ++kb) {
#pragma unroll
            for (uint32_t db = 0; db < kDim / 16; ++db) {
                w.acc[db][cb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[kb][db], hi[cb][kb], w.acc[db][cb], 0, 0, 0);
            }
#pragma unroll
            for (uint32_t db = 0; db < kDim / 16; ++db) {
                w.acc[db][cb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[kb][db], lo[cb][kb], w.acc[db][cb], 0, 0, 0);
            }
        }
    }
}

// The state as a part: denominators summed over the column's lanes, mref -inf
// where there was no finite score.  Returns whether some value of a column
// that counts is not finite.
template <uint32_t kDim, uint32_t kCB>
__device__ inline bool columns_finish(Columns<kDim, kCB>& w)
{
    float z = 0.0f;   // stays 0 unless a term is infinite or NaN
#pragma unroll
    for (uint32_t cb = 0; cb < kCB; ++cb) {
        w.l[cb] += xor16(w.l[cb]);
        w.l[cb] += xor32(w.l[cb]);
        if (w.mref[cb] == INFINITY) w.mref[cb] = -INFINITY;
        float4_t f = {w.l[cb] * 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t db = 0; db < kDim / 16; ++db) f += w.acc[db][cb] * 0.0f;
        z += w.ok[cb] ? (f[0] + f[1]) + (f[2] + f[3]) : 0.0f;
    }
    return z != 0.0f;
}

// ---- the unit's group table ---------------------------------------------------

// Groups of 8 keys that a workgroup resolves at once, one a thread: a longer
// unit is taken in segments of that.
template <uint32_t kWaves>
constexpr uint32_t kTableGroups = kWaves * kWave;

struct TableFlags {
    uint32_t generic;
    uint32_t first;
};

// The entry that holds group threadIdx.x of keys begin.. in a table of full
// extent pages of 64 tokens, then micro pages of 8; its length tells how many
// there are of each.
__device__ inline kimkv_block_desc guessed_entry(const kimkv_decode_item& table, uint32_t begin)
{
    uint32_t const t = begin + 8 * threadIdx.x;
    uint32_t const micro = (table.token_count + 7) / 8;   // entries without an extent page, which saves seven
    uint32_t const extents = micro > table.descriptor_count ? (micro - table.descriptor_count) / 7 : 0;
    uint32_t const i = t / 64 < extents ? t / 64 : extents + (t - 64 * extents) / 8;
    return table.descriptors[min(i, table.descriptor_count - 1)];
}

// Resolves the 8-key groups of [begin, end) for KV head `head`, group
// threadIdx.x from `guess` (guessed_entry's) where every thread's is right,
// else by searching.  False where the table does not keep the groups aligned
// and whole: the unit then goes the generic path.  Called by every thread.
template <uint32_t kDim, uint32_t kWaves>
__device__ bool build_groups(const PoolView& P, const kimkv_decode_item& table, uint32_t head, uint32_t begin,
                             uint32_t end, kimkv_block_desc const& guess, HeadGroup* groups, TableFlags& flags)
{
    uint32_t const tid = threadIdx.x;
    uint32_t const ngroups = (end - begin + 7) / 8;
    bool right = true;
    if (tid < ngroups) {
        uint32_t const t = begin + 8 * tid;
        uint32_t const cap = guess.page_token_capacity;
        uint32_t const at = t - guess.logical_token_begin;
        const uint16_t* const page = page_base(P, guess.kind, guess.slot, cap);
        right = t >= guess.logical_token_begin && at < guess.valid_tokens && ((guess.logical_token_begin | cap) & 7u) == 0
            && guess.valid_tokens <= cap && page != nullptr
            && (guess.valid_tokens - at >= 8 || guess.logical_token_begin + guess.valid_tokens >= table.token_count);
        if (right) {
            const uint16_t* const block = page + head_block(P, cap, table.layer, head);
            groups[tid] = HeadGroup{block + k_offset(cap, kDim, at, 0), block + v_offset(cap, kDim, at, 0), cap * 32u, v_width(cap), 0};
        }
    }
    if (__syncthreads_and(right) != 0) return true;
    if (tid < ngroups) groups[tid].k = nullptr;
    if (tid == 0) flags.generic = 0;
    if (tid < kWave) {
        uint32_t const first = find_descriptor_wave(table.descriptors, table.descriptor_count, begin);
        if (tid == 0) flags.first = first;
    }
    __syncthreads();
    // At most ngroups + 1 entries reach into the unit.
    uint32_t const first = flags.first;
    for (uint32_t j = tid; j <= ngroups && j < table.descriptor_count - first; j += kWaves * kWave) {
        add_head_groups<kDim>(P, table.descriptors[first + j], table.layer, head, begin, end, table.token_count, groups,
                              &flags.generic);
    }
    __syncthreads();
    bool const hole = tid < ngroups && groups[tid].k == nullptr;
    return __syncthreads_or(hole || flags.generic != 0) == 0;
}

// ---- direct units ---------------------------------------------------------------
// The waves split the unit's heads, then its tokens, and read K and V^T
// straight into operand registers, two steps in flight; at the end they merge
// their parts through LDS.  Each wave holds all of the unit's columns (up to
// 64 of 64 dims, 32 of 128), so every byte enters the compute unit once and
// nothing is staged.
//
// Times of a unit, alone on its compute unit: about 1.1 us until its table is
// known, 1.2 for queries, 0.7 for the pages, 2.4 for the merge and its stores
// (instructions that come from memory once a launch).  Between them 1 us a
// 64-token step of one block of columns is the loads' latency; many columns
// are bound by the weights: 57 cycles for 64 scores a SIMD, of which 44 remain
// without loads (8192 tokens x 64 columns x 64 dims in 71 us, 0.48 PFLOP/s over
// 256 units).  Tiles of 64 keys staged in LDS for 256 columns of 8 waves
// measured 153 us where this took 173 (128 lanes x 65536 tokens), and 62 where
// this took 53 (16384): the barriers cost what the fewer loads save.
template <uint32_t kDim, uint32_t kCB, uint32_t kWaves>
struct DirectRows {
    static constexpr uint32_t kRow = kDim + 4;   // o, m, l, pad
    float row[kWaves][16 * kCB][kRow];
};

// Dims [d, d + 4) of the part o, m, l of query head out's + q.
template <uint32_t kDim>
__device__ inline void store_part(const SharedArgs& a, const ColumnOut& out, uint32_t q, uint32_t d, float4_t o, float m, float l)
{
    if (out.output == nullptr) {
        *reinterpret_cast<float4_t*>(a.parts.o + (out.row + q) * kDim + d) = o;
        if (d == 0) a.parts.ml[out.row + q] = make_float2(m, l);
        return;
    }
    uint16_t* const to = out.output + q * kDim + d;
    store_outputs<4>(to, o, l);
}

template <uint32_t kDim, uint32_t kCB, uint32_t kWaves>
__device__ bool unit_direct(const PoolView& P, const SharedArgs& a, const SharedUnit& u, const kimkv_decode_item& table,
                            HeadGroup* groups, TableFlags& flags, ColumnOut* outs, DirectRows<kDim, kCB, kWaves>& rows)
{
    constexpr uint32_t kSegment = 8 * kTableGroups<kWaves>;
    constexpr uint32_t kKB = kDim <= 64 && kCB == 1 ? 2 : 1;   // 32-key blocks a step
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
    uint32_t const hs = kCB > 1 || u.heads <= 1 ? 1 : u.heads <= 2 ? 2 : u.heads <= 4 ? 4 : kWaves;   // heads' share of the waves
    uint32_t const split = kWaves / hs;
    uint32_t const head = wave % hs;
    bool const works = head < u.heads;
    // The table's entries and the queries are on their way together.
    kimkv_block_desc guess = guessed_entry(table, u.begin);
    Columns<kDim, kCB> w;
    bool const ordered = columns_init(w, P, a, u, table.layer, works ? u.head + head : u.head, outs);
    // Two steps' keys in registers, and values of one where two do not fit.
    constexpr uint32_t kValueSteps = kDim == 128 && kCB > 1 ? 1 : 2;
    struct Keys {
        half8_t k[kKB][2][kPanels];
    };
    struct Values {
        half8_t v[kKB][kDb];
    };
    // Keys past the end are read at the last group's place.
    uint32_t c0 = 0, c1 = 0;   // the wave's keys of the segment
    auto load_k = [&](Keys& o, uint32_t t0) {
#pragma unroll
        for (uint32_t kb = 0; kb < kKB; ++kb) {
            HeadGroup const g = groups[min(t0 / 8 + 4 * kb + x, (c1 - 1) / 8)];
            const uint16_t* const k0 = g.k + head * (2u * kDim / 32u) * g.kpanel + (l & 3u) * 32 + a4 * 8;   // 2 cap D a head
#pragma unroll
            for (uint32_t e = 0; e < 2; ++e) {
#pragma unroll
                for (uint32_t p = 0; p < kPanels; ++p) o.k[kb][e][p] = load_keys<kCB == 1>(k0 + 128 * e + p * g.kpanel);
            }
        }
    };
    auto load_v = [&](Values& o, uint32_t t0) {
#pragma unroll
        for (uint32_t kb = 0; kb < kKB; ++kb) {
            HeadGroup const g = groups[min(t0 / 8 + 4 * kb + a4, (c1 - 1) / 8)];
            const uint16_t* const v0 = g.v + head * (2u * kDim / 32u) * g.kpanel + r * g.vw;
#pragma unroll
            for (uint32_t db = 0; db < kDb; ++db) o.v[kb][db] = load_keys<kCB == 1>(v0 + 16 * db * g.vw);
        }
    };
    auto step = [&](Keys const& k, Values& v, uint32_t t) {
        uint32_t const nvalid = c1 - t;
        if (__builtin_expect(nvalid < kStep, 0)) {   // V of keys past the end may hold anything
            uint32_t first = 8 * a4;
            __asm__ volatile("" : "+v"(first));      // a branch
#pragma unroll
            for (uint32_t kb = 0; kb < kKB; ++kb) {
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) {
                    if (32 * kb + first + j < nvalid) continue;
#pragma unroll
                    for (uint32_t db = 0; db < kDb; ++db) v.v[kb][db][j] = static_cast<_Float16>(0.0f);
                }
            }
        }
        attend_step(w, k.k, v.v, nvalid);
    };
    for (uint32_t s0 = u.begin; s0 < u.end; s0 += kSegment) {
        uint32_t const s1 = min(u.end - s0, kSegment) + s0;
        if (s0 != u.begin) {
            guess = guessed_entry(table, s0);
            __syncthreads();   // the last segment's groups have been read
        }
        if (!build_groups<kDim, kWaves>(P, table, u.head, s0, s1, guess, groups, flags)) return false;
        uint32_t const piece = ((s1 - s0 + split - 1) / split + 31) / 32 * 32;
        c0 = min(wave / hs * piece, s1 - s0);
        c1 = min(c0 + piece, s1 - s0);
        if (works && c0 < c1) {
            Keys k0, k1;
            Values v0, v1;
            load_k(k0, c0);
            if (kValueSteps == 2) load_v(v0, c0);
#pragma unroll 1
            for (uint32_t t = c0;; t += 2 * kStep) {
                bool const second = t + kStep < c1;
                if (kValueSteps == 1) load_v(v0, t);
                if (second) load_k(k1, t + kStep);
                if (kValueSteps == 2 && second) load_v(v1, t + kStep);
                step(k0, v0, t);
                if (!second) break;
                bool const third = t + 2 * kStep < c1;
                if (kValueSteps == 1) load_v(v0, t + kStep);
                if (third) load_k(k0, t + 2 * kStep);
                if (kValueSteps == 2 && third) load_v(v0, t + 2 * kStep);
                if (kValueSteps == 1) {
                    step(k1, v0, t + kStep);
                } else {
                    step(k1, v1, t + kStep);
                }
                if (!third) break;
            }
        }
    }
    bool const again = columns_finish(w) || !ordered;
    if (kCB == 1 && split == 1) {   // a wave's head is its own
        if (__syncthreads_or(again) != 0) return false;
        if (works && w.ok[0]) {
            ColumnOut const out = outs[r];
#pragma unroll
            for (uint32_t db = 0; db < kDb; ++db) {
                store_part<kDim>(a, out, (u.head + head) * G, 16 * db + 4 * a4, w.acc[db][0], w.mref[0], w.l[0]);
            }
        }
        return true;
    }
#pragma unroll
    for (uint32_t cb = 0; cb < kCB; ++cb) {
        float* const mine = rows.row[wave][16 * cb + r];
#pragma unroll
        for (uint32_t db = 0; db < kDb; ++db) *reinterpret_cast<float4_t*>(mine + 16 * db + 4 * a4) = w.acc[db][cb];
        if (l < 16) {
            mine[kDim] = w.mref[cb];
            mine[kDim + 1] = w.l[cb];
        }
    }
    if (__syncthreads_or(again) != 0) return false;
    // Four dims of a column of a head at a time.
    constexpr uint32_t kQuads = kDim / 4;
    for (uint32_t i = tid; i < u.heads * u.cols * kQuads; i += kWaves * kWave) {
        uint32_t const d = i % kQuads * 4;
        uint32_t const c = i / kQuads % u.cols;
        uint32_t const hd = i / kQuads / u.cols;
        ColumnOut const out = outs[c];
        if (out.ok == 0) continue;
        // All the waves' rows are read at once; those of another head count for nothing.
        float m[kWaves];
        float M = -INFINITY;
#pragma unroll
        for (uint32_t v = 0; v < kWaves; ++v) {
            m[v] = v % hs == hd ? rows.row[v][c][kDim] : -INFINITY;
            M = fmaxf(M, m[v]);
        }
        float4_t o = {};
        float den = 0.0f;
#pragma unroll
        for (uint32_t v = 0; v < kWaves; ++v) {
            const float* const part = rows.row[v][c];
            float const f = m[v] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[v] - M);
            if (f != 0.0f) {
                o += f * *reinterpret_cast<const float4_t*>(part + d);
                den += f * part[kDim + 1];
            }
        }
        uint32_t const q = (u.head + hd) * G;   // past the column's query head of KV head 0
        store_part<kDim>(a, out, q, d, o, M, den);
    }
    return true;
}

// Head dims with a matrix-core path, and the most 16-column blocks a wave's
// registers hold at one.
constexpr bool direct_dim(uint32_t D) { return D == 64 || D == 96 || D == 128; }
constexpr uint32_t most_blocks(uint32_t D) { return D == 64 ? 4 : direct_dim(D) ? 2 : 1; }

struct NoLds {};

constexpr size_t kMostLds = 160 * 1024;   // of a compute unit

// kDim: the head dim, or 0 for one that has only the generic path.
template <uint32_t kDim, uint32_t kWaves>
__global__ __launch_bounds__(kWaves * kWave) __attribute__((amdgpu_waves_per_eu(2, 2))) void shared_decode_kernel(PoolView P,
                                                                                                                 SharedArgs a)
{
    // Registers allow 8 waves a compute unit, so a workgroup's memory may take its share of the unit's: all or nearly half.
    union Paths {
        GenericLds<kWaves> generic;
        std::conditional_t<kDim != 0, DirectRows<kDim == 0 ? 64 : kDim, most_blocks(kDim), kWaves>, NoLds> direct;
    };
    __shared__ __attribute__((aligned(16))) unsigned char path_lds[sizeof(Paths)];
    __shared__ ColumnOut outs[64];
    __shared__ HeadGroup groups[kDim != 0 ? kTableGroups<kWaves> : 1];
    __shared__ TableFlags flags;
    static_assert(kMostLds / (kManyWaves / kWaves) >= sizeof path_lds + sizeof outs + sizeof groups + sizeof flags + 64);
    Paths& lds = *reinterpret_cast<Paths*>(path_lds);
    SharedUnit const u = a.units[xcd_logical_index(blockIdx.x, gridDim.x)];
    if (u.cols == 0) return;
    // The entries lie in the caller's memory: nothing outside the launch's buffers is touched, whatever they hold.
    uint32_t rest;
    uint64_t const last = div_mod(u.col0 + (u.cols - 1), a.group, &rest);   // lane of the last column, from u.lane
    if (((u.col0 | (u.cols - 1)) >> 30) != 0 || u.table_lane >= a.lane_count || u.lane + last >= a.lane_count || u.heads == 0
        || u.head + u.heads > P.heads || u.begin >= u.end || ((u.kind & kSingle) == 0 && u.slot + last >= a.slot_count)) {
        report_fault(P, KIMKV_FAULT_DECODE_ITEM);
        return;
    }
    kimkv_decode_item const table = a.items[u.table_lane];
    uint32_t const planned = a.lanes[u.table_lane].tokens;
    if (!lane_valid(P, table, planned) || u.end > planned) {
        report_fault(P, KIMKV_FAULT_DECODE_ITEM);
        return;
    }
    if constexpr (kDim != 0) {
        bool done = false;
        uint32_t const kind = u.kind & ~kSingle;
        auto direct = [&](auto blocks) {
            constexpr uint32_t kCB = decltype(blocks)::value;
            if (u.cols > 16 * kCB || (u.begin & 7u) != 0 || (kCB == 1 ? u.heads > kWaves : u.heads != 1)) return;
            done = unit_direct<kDim, kCB, kWaves>(P, a, u, table, groups, flags, outs,
                                                  *reinterpret_cast<DirectRows<kDim, kCB, kWaves>*>(path_lds));
        };
        if (kind == 1) direct(std::integral_constant<uint32_t, 1>{});
        else if (kind == 2) direct(std::integral_constant<uint32_t, 2>{});
        if constexpr (most_blocks(kDim) == 4) {
            if (kind == 4) direct(std::integral_constant<uint32_t, 4>{});
        }
        if (done) return;
        __syncthreads();   // the generic path's rows take the same memory
    }
    unit_generic<kWaves>(P, a, u, lds.generic);
}

// Merges the lanes' parts, four dims a thread (one where the head dim is no
// multiple of 4), the parts of a row over `split` neighbouring threads where
// they are many.  Bound by the parts' bytes, which the launch before has just
// written, and for many by the rounds of reads (8 lanes of 8192 tokens in 32
// pieces: 23.4 us a pass with a thread a row, 19.5 so); kMergeBatch parts of a
// thread are in flight together.
constexpr unsigned kMergeBlock = 256;
constexpr uint32_t kMergeBatch = 8;

template <uint32_t kWidth>
__global__ __launch_bounds__(kMergeBlock) void shared_merge_kernel(PoolView P, SharedArgs a, uint32_t split)
{
    typedef float vec_t __attribute__((ext_vector_type(kWidth)));
    uint32_t const lane = blockIdx.x;
    SharedLane const rec = a.lanes[lane];
    if (rec.merged == 0) return;
    uint64_t const last_prefix = rec.prefix_slot + static_cast<uint64_t>(rec.prefix_stride) * (rec.prefix_count - 1ull);
    if (rec.prefix_count > a.slot_count || rec.tail_count > a.slot_count
        || (rec.prefix_count != 0 && last_prefix >= a.slot_count)
        || static_cast<uint64_t>(rec.tail_slot) + rec.tail_count > a.slot_count) {
        return;
    }
    uint32_t const D = P.dim;
    uint32_t const parts = rec.prefix_count + rec.tail_count;
    bool const ok = lane_ok(P, a, lane);   // a unit reported it; not waited for before the parts are read
    uint16_t* const output = a.items[lane].output;
    uint32_t const per_row = D / kWidth;
    uint32_t const mine = threadIdx.x & (split - 1);
    uint32_t const at_once = kMergeBlock / split;
    for (uint32_t x0 = blockIdx.y * at_once; x0 < a.QH * per_row; x0 += gridDim.y * at_once) {
        uint32_t const x = min(x0 + threadIdx.x / split, a.QH * per_row - 1);   // past the end: once again
        uint32_t const q = x / per_row;
        uint32_t const d = (x - q * per_row) * kWidth;
        float M = -INFINITY;
        float l = 0.0f;
        vec_t o = {};
        for (uint32_t i0 = 0; i0 < parts; i0 += kMergeBatch * split) {
            float2 ml[kMergeBatch];
            vec_t row[kMergeBatch];
#pragma unroll
            for (uint32_t j = 0; j < kMergeBatch; ++j) {
                uint32_t const n = i0 + j * split + mine;
                uint32_t const i = min(n, parts - 1);
                uint32_t const slot = i < rec.prefix_count ? rec.prefix_slot + i * rec.prefix_stride
                                                           : rec.tail_slot + (i - rec.prefix_count);
                uint64_t const at = static_cast<uint64_t>(slot) * a.QH + q;
                ml[j] = a.parts.ml[at];
                row[j] = *reinterpret_cast<const vec_t*>(a.parts.o + at * D + d);
                if (n >= parts) ml[j].x = -INFINITY;
            }
            float m_new = M;
#pragma unroll
            for (uint32_t j = 0; j < kMergeBatch; ++j) m_new = fmaxf(m_new, ml[j].x);
            float const c = M == -INFINITY ? 0.0f : exp2f(M - m_new);
            M = m_new;
#pragma unroll
            for (uint32_t k = 0; k < kWidth; ++k) o[k] = carried(o[k], c);
            l *= c;
#pragma unroll
            for (uint32_t j = 0; j < kMergeBatch; ++j) {
                float const f = ml[j].x == -INFINITY ? 0.0f : exp2f(ml[j].x - M);
                if (left_out(f, ml[j].y)) continue;
                o += f * row[j];
                l += f * ml[j].y;
            }
        }
        for (uint32_t step = 1; step < split; step *= 2) {
            float const other = __shfl_xor(M, static_cast<int>(step));
            float const m_new = fmaxf(M, other);
            float const f = M == -INFINITY ? 0.0f : exp2f(M - m_new);
            M = m_new;
            l = left_out(f, l) ? 0.0f : f * l;
            l += __shfl_xor(l, static_cast<int>(step));
#pragma unroll
            for (uint32_t k = 0; k < kWidth; ++k) {
                float const v = carried(o[k], f);
                o[k] = v + __shfl_xor(v, static_cast<int>(step));
            }
        }
        if (ok && mine == 0 && x0 + threadIdx.x / split < a.QH * per_row) {
            store_outputs<kWidth>(output + static_cast<uint64_t>(q) * D + d, o, l);
        }
    }
}

// ---- planning -----------------------------------------------------------------

constexpr uint32_t kShareBlock = 64;     // tokens: a shared prefix is cut to whole blocks

// What a unit costs, in nanoseconds, as measured on a full device: the chain of
// reads in front of it and the merge and stores behind it (6.2 to 7.0 us for a
// few tokens, 6.7 to 8.5 with another beside it); the bytes that a workgroup
// streams; the steps of a wave when the loads' latency is all there is; the
// arithmetic of many columns (at D = 64, 64 columns: 25.7 and 71.7 us for 2048
// and 8192 tokens by 8 waves, 28.4 and 77 for 1024 and 4096 by 4).  What the
// bytes of all units take, whoever reads them; and the merge: its launch, a
// round of reads, and what the parts take to write and read.
struct UnitCost {
    uint32_t D;
    uint32_t waves;
    static constexpr double kBytes = 5500;        // HBM's, a nanosecond
    static constexpr double kMergeLaunch = 4000;
    static constexpr double kMergeRound = 1000;
    static constexpr double kPartBytes = 4000;    // a nanosecond
    static constexpr double kLeast = 6500;        // of any unit
    double own_start() const { return waves == kManyWaves ? 6500 : 8000; }
    double prefix_start(uint32_t blocks) const { return 6500.0 + (waves == kManyWaves ? 600 : 800) * blocks; }
    // `split` waves share a head's tokens.
    double own(uint32_t heads, uint32_t split, uint32_t tokens) const
    {
        double const steps = std::ceil(std::ceil(tokens / static_cast<double>(split)) * D / 64 / 64);
        return own_start() + std::max((waves == kManyWaves ? 6.0 : 11.5) * D / 64 * heads * tokens, 700.0 * steps);
    }
    double prefix(uint32_t blocks, uint32_t tokens) const
    {
        double const token = waves == kManyWaves ? std::max(4.9, 1.87 * blocks) : std::max(10.9, 3.9 * blocks);
        return prefix_start(blocks) + token * D / 64 * tokens;
    }
    double bytes(uint32_t heads, uint32_t tokens) const { return 4.0 * D * heads * tokens; }
};

// Threads that share the merge of a row of so many parts.
uint32_t merge_split(uint64_t parts)
{
    uint32_t split = 1;
    while (split < 8 && parts > kMergeBatch * split) split *= 2;
    return split;
}

struct Planned {
    std::vector<SharedUnit> units;
    std::vector<double> cost;
    std::vector<SharedLane> lanes;
    uint64_t slots{0};
    uint32_t merge_lanes{0};
    uint32_t merge_parts{0};   // of the lane that has most
    uint32_t waves{0};         // of a workgroup
};

// A launch takes fewer than 2^32 threads.
constexpr uint32_t most_units(uint32_t waves) { return 0xFFFFFFFFu / (waves * kWave); }
constexpr uint32_t kMostLanes = 0xFFFFFFFFu / kMergeBlock;
constexpr uint32_t kMostRow = 0x7FFFFFFFu;   // elements of a lane's query, indexed in 32 bits

uint64_t align16(uint64_t n) { return (n + 15) / 16 * 16; }

// Spreads the units over the XCDs (workgroup w runs on XCD w % 8): units of
// one range of keys and head together, whose K and V then stay in one L2, the
// costliest first onto the XCD with least to do that still has a compute unit
// for each, and each XCD's costliest first.  Where these are more than an XCD
// runs at once (many lanes' columns on few heads), they are cut every so many
// units, or every eighth of all such units where that is more (256 lanes of 16
// query heads on 8192 tokens, 2 KV heads: 128 units on each of two XCDs and
// none on the others, so 32 on each).  Short lists end in idle entries.
void place_units(Planned& p, uint32_t at_once)
{
    size_t const per_xcd = std::max(1u, at_once / kXcds);
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
    size_t wide = 0;
    for (Bundle const& b : bundles) wide += b.count > per_xcd ? b.count : 0;
    if (wide != 0) {
        size_t const most = std::max<size_t>(per_xcd, (wide + kXcds - 1) / kXcds);
        std::vector<Bundle> cut;
        bool open = false;   // the last one takes more units
        for (Bundle b : bundles) {
            if (b.count <= per_xcd) {
                cut.push_back(b);
                open = false;
                continue;
            }
            double const each = b.cost / static_cast<double>(b.count);
            while (b.count != 0) {
                if (!open) cut.push_back(Bundle{b.first, 0, 0.0});
                Bundle& last = cut.back();
                size_t const n = std::min(b.count, most - last.count);
                last.count += n;
                last.cost += each * static_cast<double>(n);
                b.first += n;
                b.count -= n;
                open = last.count < most;
            }
        }
        bundles = std::move(cut);
    }
    std::stable_sort(bundles.begin(), bundles.end(), [](Bundle const& x, Bundle const& y) { return x.cost > y.cost; });
    std::vector<size_t> xcd[kXcds];
    double load[kXcds] = {};
    for (Bundle const& b : bundles) {
        auto const key = [&](uint32_t x) { return std::make_pair(xcd[x].size() + b.count > per_xcd, load[x]); };
        uint32_t best = 0;
        for (uint32_t x = 1; x < kXcds; ++x) {
            if (key(x) < key(best)) best = x;
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

// Tokens of each of the pieces of [0, tokens), in blocks of 64, when they are
// to be about n.
uint32_t piece_tokens(uint64_t tokens, double n)
{
    auto const each = static_cast<uint64_t>(std::ceil(static_cast<double>(tokens) / std::max(1.0, std::ceil(n - 0.25))));
    return static_cast<uint32_t>(std::max<uint64_t>(64, (each + 63) / 64 * 64));
}

// The lanes' work before it is cut into pieces.
struct Work {
    struct Prefix {
        uint32_t lane, lanes, tokens, blocks;   // blocks: of 16 columns a wave
        uint64_t tiles;                         // units that take all its columns, but those of empty lanes alone
    };
    std::vector<Prefix> prefixes;
    std::vector<uint32_t> shared;   // tokens of each lane that a prefix takes
};

struct Shape {
    uint32_t H, G, D;
    uint32_t waves;     // of a workgroup
    uint32_t at_once;   // workgroups that run at the same time
    const uint32_t* tokens;
    uint32_t lane_count;
};

// How a batch is cut: KV heads of a unit of a lane's own tokens, the costs
// that pieces of prefixes and of lanes' own tokens do not go far past, and what
// that comes to.
struct Cut {
    uint32_t heads{1};
    double share{0};
    double own_share{0};
    double time{0};
};

template <typename PrefixFn, typename OwnFn>
void each_piece(Shape const& s, Work const& work, Cut const& cut, PrefixFn&& prefix_piece, OwnFn&& own_piece)
{
    UnitCost const cost{s.D, s.waves};
    for (Work::Prefix const& p : work.prefixes) {
        double const start = cost.prefix_start(p.blocks);
        double const whole = cost.prefix(p.blocks, p.tokens) - start;
        prefix_piece(p, piece_tokens(p.tokens, whole / std::max(1.0, cut.share - start)));
    }
    uint32_t const split = s.waves / cut.heads;
    for (uint32_t i = 0; i < s.lane_count; ++i) {
        uint32_t const own = s.tokens[i] - work.shared[i];
        if (own == 0) continue;
        double const whole = cost.own(std::min(cut.heads, s.H), split, own) - cost.own_start();
        own_piece(i, own, piece_tokens(own, whole / std::max(1.0, cut.own_share - cost.own_start())));
    }
}

// The time of a cut: units go to compute units as these come free, the costliest
// first, so one starts no later than when the costlier ones' work, spread
// evenly, is done, and the whole takes no longer than rounds of one unit on each
// compute unit (costs within an eighth of each other count as equal); no less
// than what their bytes take; and the merge where a lane has several parts.
double cut_time(Shape const& s, Work const& work, Cut const& cut)
{
    UnitCost const cost{s.D, s.waves};
    constexpr int kLevels = 64;   // 8 an octave from the least cost on
    struct Level {
        double total{0};
        double longest{0};
        uint64_t units{0};
    };
    Level levels[kLevels];
    double bytes = 0;
    uint64_t parts = 0;        // of all lanes
    uint64_t prefix_most = 0;  // of a lane
    uint64_t own_most = 0;
    auto add = [&](double each, uint64_t n) {
        // The exponent and the first three bits behind the leading one.
        auto const ratio = static_cast<float>(each / UnitCost::kLeast);
        uint32_t bits;
        std::memcpy(&bits, &ratio, sizeof bits);
        Level& level = levels[std::min(kLevels - 1, std::max(0, static_cast<int>(bits >> 20) - (127 << 3)))];
        level.total += each * static_cast<double>(n);
        level.longest = std::max(level.longest, each);
        level.units += n;
    };
    each_piece(
        s, work, cut,
        [&](Work::Prefix const& p, uint32_t piece) {
            add(cost.prefix(p.blocks, std::min(piece, p.tokens)), (p.tokens + piece - 1ull) / piece * s.H * p.tiles);
            bytes += cost.bytes(s.H, p.tokens);
            uint64_t const pieces = (p.tokens + piece - 1ull) / piece;
            parts += pieces * p.lanes;
            prefix_most = std::max(prefix_most, pieces);
        },
        [&](uint32_t, uint32_t own, uint32_t piece) {
            uint64_t const pieces = (own + piece - 1ull) / piece;
            add(cost.own(std::min(cut.heads, s.H), s.waves / cut.heads, std::min(piece, own)),
                pieces * ((s.H + cut.heads - 1) / cut.heads) * ((s.G + 15) / 16));
            parts += pieces;
            own_most = std::max(own_most, pieces);
            bytes += cost.bytes(s.H, own);
        });
    double spread = 0;
    double rounds = 0;
    double before = 0;
    uint64_t units = 0;
    auto const rounds_of = [&](uint64_t n) { return (n + s.at_once - 1) / s.at_once; };
    for (int i = kLevels - 1; i >= 0; --i) {
        Level const& level = levels[i];
        if (level.units == 0) continue;
        rounds += static_cast<double>(rounds_of(units + level.units) - rounds_of(units)) * level.longest;
        units += level.units;
        before += level.total;
        double const start = units <= s.at_once ? 0.0 : (before - level.longest) / s.at_once;
        spread = std::max(spread, start + level.longest);
    }
    double const time = std::max(std::min(spread, rounds), UnitCost::kLeast + bytes / UnitCost::kBytes);
    if (prefix_most == 0 && own_most <= 1) return time;
    uint64_t const most = prefix_most + own_most;
    double const merge_rounds = std::ceil(static_cast<double>(most) / (kMergeBatch * merge_split(most)));
    return time + UnitCost::kMergeLaunch + UnitCost::kMergeRound * merge_rounds
        + 4.0 * static_cast<double>(parts) * s.H * s.G * s.D / UnitCost::kPartBytes;
}

// The best of a few cuts: pieces of a few sizes around an equal share for each
// compute unit, and whole ones; lanes' own tokens in pieces alike, or smaller
// ones, which fill the end behind long pieces of prefixes.
Cut best_cut(Shape const& s, Work const& work)
{
    UnitCost const cost{s.D, s.waves};
    // KV heads of a unit of a lane's own tokens: one for each wave, fewer, with
    // more waves for each, while the units are few.
    uint32_t heads = 1;
    while (heads < s.waves && heads < s.H) heads *= 2;
    uint64_t own_units = 0;
    double total = 0;
    uint32_t longest_own = 0;
    for (uint32_t i = 0; i < s.lane_count; ++i) {
        uint32_t const own = s.tokens[i] - work.shared[i];
        if (own == 0) continue;
        longest_own = std::max(longest_own, own);
        own_units += static_cast<uint64_t>((s.H + heads - 1) / heads) * ((s.G + 15) / 16);
        total += cost.own(s.H, s.waves, own) * ((s.G + 15) / 16);
    }
    while (heads > 1 && own_units * 4 <= s.at_once) {
        heads /= 2;
        own_units *= 2;
    }
    for (Work::Prefix const& p : work.prefixes) {
        total += cost.prefix(p.blocks, p.tokens) * static_cast<double>(p.tiles) * s.H;
    }
    double const even = total / s.at_once + UnitCost::kLeast;
    Cut best;
    double const longest = cost.own(std::min(heads, s.H), s.waves / heads, longest_own);
    for (double const part : {1.0, 0.35, 0.15}) {
        for (double const share : {1e12, 0.7 * even, 0.8 * even, 0.9 * even, even, 1.1 * even, 1.25 * even, 1.45 * even, 1.8 * even}) {
            double const own_share = share < 1e12 ? part * share : part < 1.0 ? part * even : share;
            if (part < 1.0 && longest <= own_share) continue;   // cuts nothing more
            Cut c{heads, std::max(share, UnitCost::kLeast + 4000), std::max(own_share, cost.own_start() + 1500), 0};
            c.time = cut_time(s, work, c);
            if (best.share == 0 || c.time < best.time) best = c;
        }
        if (work.prefixes.empty()) break;   // own tokens alone: the shares say it all
    }
    return best;
}

// Whether columns [col, col + 16 p.blocks) of a prefix belong to lanes with tokens, some of them.
bool any_tokens(const uint32_t* tokens, Work::Prefix const& p, uint32_t G, uint32_t col)
{
    uint32_t const end = std::min(p.lanes, (col + 16 * p.blocks - 1) / G + 1);
    for (uint32_t i = col / G; i < end; ++i) {
        if (tokens[p.lane + i] != 0) return true;
    }
    return false;
}

bool plan_batch(uint32_t H, uint32_t D, uint32_t QH, uint32_t compute_units, const uint32_t* tokens, uint32_t lane_count,
                const kimkv_shared_group* groups, uint32_t group_count, Planned& out)
{
    uint32_t const G = QH / H;
    for (uint32_t i = 0; i < lane_count; ++i) {
        if (tokens[i] >> 31 != 0) return false;
    }
    std::vector<uint8_t> grouped(lane_count, 0);
    Work apart;
    apart.shared.assign(lane_count, 0);
    Work work = apart;
    for (uint32_t g = 0; g < group_count; ++g) {
        kimkv_shared_group const& group = groups[g];
        if (group.first_lane > lane_count || group.lane_count > lane_count - group.first_lane) return false;
        uint32_t prefix = group.prefix_tokens;
        // Lanes of no tokens (requests that ended, padding) share nothing and hold nobody up: the prefix is the
        // others', read through the first of them.
        uint32_t live = 0, first = 0, last = 0;
        for (uint32_t i = group.first_lane; i < group.first_lane + group.lane_count; ++i) {
            if (grouped[i] != 0) return false;
            grouped[i] = 1;
            if (tokens[i] == 0) continue;
            if (live == 0) first = i;
            last = i;
            ++live;
            prefix = std::min(prefix, tokens[i]);
        }
        prefix = prefix / kShareBlock * kShareBlock;
        if (live < 2 || prefix == 0) continue;
        uint32_t const run = last - first + 1;
        uint64_t const columns = static_cast<uint64_t>(run) * G;
        if (columns >> 30 != 0) return false;
        Work::Prefix p{first, run, prefix, 1, 0};
        while (p.blocks < most_blocks(D) && 16 * p.blocks < columns) p.blocks *= 2;
        for (uint32_t col = 0; col < columns; col += 16 * p.blocks) p.tiles += any_tokens(tokens, p, G, col) ? 1 : 0;
        work.prefixes.push_back(p);
        for (uint32_t i = first; i <= last; ++i) work.shared[i] = std::min(prefix, tokens[i]);
    }
    // Many waves a workgroup where the prefixes are most of the work.
    auto const shape_of = [&](uint32_t waves) {
        return Shape{H, G, D, waves, std::min(compute_units, 1u << 20) * (kManyWaves / waves), tokens, lane_count};
    };
    UnitCost const rough{D, kManyWaves};
    double prefix_work = 0;
    double own_work = 0;
    for (Work::Prefix const& p : work.prefixes) {
        prefix_work += (rough.prefix(p.blocks, p.tokens) - rough.prefix_start(p.blocks)) * static_cast<double>(p.tiles) * H;
    }
    for (uint32_t i = 0; i < lane_count; ++i) {
        if (tokens[i] != work.shared[i]) own_work += rough.own(H, kManyWaves, tokens[i] - work.shared[i]);
    }
    Shape shape = shape_of(prefix_work > own_work ? kManyWaves : kFewWaves);
    Cut cut = best_cut(shape, work);
    // Short prefixes of few lanes are read faster lane by lane, without a merge.
    if (!work.prefixes.empty()) {
        Shape const other_shape = shape_of(kFewWaves);
        Cut const other = best_cut(other_shape, apart);
        if (other.time <= cut.time) {
            shape = other_shape;
            cut = other;
            work = apart;
        }
    }
    UnitCost const cost{D, shape.waves};
    uint64_t units = 0;
    each_piece(
        shape, work, cut,
        [&](Work::Prefix const& p, uint32_t piece) { units += (p.tokens + piece - 1ull) / piece * H * p.tiles; },
        [&](uint32_t, uint32_t own, uint32_t piece) {
            units += (own + piece - 1ull) / piece * ((H + cut.heads - 1) / cut.heads) * ((G + 15ull) / 16);
        });
    if (units > most_units(shape.waves)) return false;
    out.waves = shape.waves;
    out.lanes.resize(lane_count);
    for (uint32_t i = 0; i < lane_count; ++i) out.lanes[i] = SharedLane{i, tokens[i], 0, 0, 0, 0, 0, 0};
    bool fits = true;
    auto push = [&](SharedUnit const& u, double c) {
        out.units.push_back(u);
        out.cost.push_back(c);
    };
    auto take_slots = [&](uint64_t n) {
        fits = fits && out.slots + n <= 0x7FFFFFFFu;
        return fits;
    };
    each_piece(
        shape, work, cut,
        [&](Work::Prefix const& p, uint32_t piece) {
            uint32_t const pieces = (p.tokens + piece - 1) / piece;
            if (!take_slots(static_cast<uint64_t>(p.lanes) * pieces)) return;
            for (uint32_t i = 0; i < p.lanes; ++i) {
                SharedLane& lane = out.lanes[p.lane + i];
                if (lane.tokens == 0) continue;   // its columns' parts are nobody's
                lane.table_lane = p.lane;
                lane.prefix_slot = static_cast<uint32_t>(out.slots + i);
                lane.prefix_stride = p.lanes;
                lane.prefix_count = pieces;
            }
            uint32_t const columns = p.lanes * shape.G;
            for (uint64_t at = 0; at < p.tokens; at += piece) {
                auto const end = static_cast<uint32_t>(std::min<uint64_t>(p.tokens, at + piece));
                double const c = cost.prefix(p.blocks, end - static_cast<uint32_t>(at));
                for (uint32_t h = 0; h < H; ++h) {
                    for (uint32_t col = 0; col < columns; col += 16 * p.blocks) {
                        if (!any_tokens(tokens, p, shape.G, col)) continue;
                        push(SharedUnit{p.lane, p.lane, col, std::min(16 * p.blocks, columns - col), static_cast<uint32_t>(at), end,
                                        static_cast<uint32_t>(out.slots), static_cast<uint16_t>(h), 1, static_cast<uint8_t>(p.blocks)},
                             c);
                    }
                }
                out.slots += p.lanes;
            }
        },
        [&](uint32_t i, uint32_t own, uint32_t piece) {
            SharedLane& lane = out.lanes[i];
            uint32_t const pieces = static_cast<uint32_t>((own + piece - 1ull) / piece);
            bool const single = pieces == 1 && lane.prefix_count == 0;
            if (!take_slots(single ? 0 : pieces)) return;
            lane.tail_slot = static_cast<uint32_t>(out.slots);
            lane.tail_count = single ? 0 : pieces;
            for (uint64_t at = work.shared[i]; at < tokens[i]; at += piece) {
                auto const end = static_cast<uint32_t>(std::min<uint64_t>(tokens[i], at + piece));
                for (uint32_t h = 0; h < H; h += cut.heads) {
                    uint32_t const n = std::min(cut.heads, H - h);
                    double const c = cost.own(n, shape.waves / cut.heads, end - static_cast<uint32_t>(at));
                    for (uint32_t col = 0; col < shape.G; col += 16) {
                        push(SharedUnit{i, i, col, std::min(16u, shape.G - col), static_cast<uint32_t>(at), end,
                                        static_cast<uint32_t>(out.slots), static_cast<uint16_t>(h), static_cast<uint8_t>(n),
                                        static_cast<uint8_t>(1 | (single ? kSingle : 0))},
                             c);
                    }
                }
                if (!single) out.slots += 1;
            }
        });
    if (!fits) return false;
    for (SharedLane& lane : out.lanes) {
        lane.merged = lane.prefix_count + lane.tail_count != 0 ? 1 : 0;
        out.merge_lanes += lane.merged;
        out.merge_parts = std::max(out.merge_parts, lane.prefix_count + lane.tail_count);
    }
    place_units(out, shape.at_once);
    return out.units.size() <= most_units(shape.waves);
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
        || static_cast<uint64_t>(query_heads) * head_dim > kMostRow || lane_count > kMostLanes) {
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
        plan->merge_split = merge_split(p.merge_parts);
        plan->waves = p.waves;
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
        || plan->query_heads % H != 0 || static_cast<uint64_t>(plan->query_heads) * D > kMostRow || D > kMaxDim
        || (plan->waves != kManyWaves && plan->waves != kFewWaves)
        || plan->merge_split == 0 || plan->merge_split > 8 || (plan->merge_split & (plan->merge_split - 1)) != 0
        || plan->unit_count > most_units(plan->waves) || plan->lane_count > kMostLanes
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
    a.group = divisor(plan->query_heads / H);
    PoolView const pv = pool_view(*storage);
    void* start = nullptr;
    kernel_timing_begin(TimedKernel::Decode, s, &start);
    auto launch = [&](auto dim, auto waves) {
        shared_decode_kernel<decltype(dim)::value, decltype(waves)::value><<<plan->unit_count, plan->waves * kWave, 0, s>>>(pv, a);
    };
    auto attend = [&](auto dim) {
        if (plan->waves == kManyWaves) launch(dim, std::integral_constant<uint32_t, kManyWaves>{});
        else launch(dim, std::integral_constant<uint32_t, kFewWaves>{});
    };
    if (D == 64) attend(std::integral_constant<uint32_t, 64>{});
    else if (D == 96) attend(std::integral_constant<uint32_t, 96>{});
    else if (D == 128) attend(std::integral_constant<uint32_t, 128>{});
    else attend(std::integral_constant<uint32_t, 0>{});
    kernel_timing_end(TimedKernel::Decode, s, start);
    kimkv_status const status = launch_status();
    if (status != KIMKV_OK || plan->merge_lanes == 0) return status;
    uint32_t const width = D % 4 == 0 ? 4 : 1;
    uint32_t const blocks = ceil_div(static_cast<uint64_t>(plan->query_heads) * D / width * plan->merge_split, kMergeBlock);
    dim3 const grid(plan->lane_count, blocks < 65535u ? blocks : 65535u);
    if (width == 4) shared_merge_kernel<4><<<grid, kMergeBlock, 0, s>>>(pv, a, plan->merge_split);
    else shared_merge_kernel<1><<<grid, kMergeBlock, 0, s>>>(pv, a, plan->merge_split);
    return launch_status();
}

}  // extern "C"
