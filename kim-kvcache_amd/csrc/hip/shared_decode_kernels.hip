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
#include <vector>

#include "attention_common.h"
#include "device_common.h"
#include "runtime_internal.h"

namespace kimkv {
namespace {

constexpr unsigned kBlock = 512;   // 8 waves
constexpr unsigned kWaves = kBlock / kWave;
constexpr uint32_t kMaxDim = 256;

// Tokens [begin, end) of table_lane's table for KV heads [head, head + heads),
// attended to by lanes [lane, lane + lanes).  Lane lane + i's part goes to
// slot + i; single: the lane has no other part.  lanes = 0: nothing to do.
struct SharedUnit {
    uint32_t table_lane;
    uint32_t lane;
    uint32_t lanes;
    uint32_t begin;
    uint32_t end;
    uint32_t slot;
    uint16_t head;
    uint16_t heads;
    uint32_t single;
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

// Whether a lane can be computed: an item as planned, on the layer that its
// group's table is read for.
__device__ inline bool lane_valid(const PoolView& P, const kimkv_decode_item& item, uint32_t planned_tokens)
{
    return item.token_count == planned_tokens && item.descriptors != nullptr && item.descriptor_count != 0
        && item.query != nullptr && item.output != nullptr && item.layer < P.layers;
}

__device__ inline bool lane_ok(const PoolView& P, const SharedArgs& a, uint32_t lane)
{
    SharedLane const rec = a.lanes[lane];
    if (rec.table_lane >= a.lane_count || rec.tokens == 0) return false;
    kimkv_decode_item const item = a.items[lane];
    if (!lane_valid(P, item, rec.tokens)) return false;
    if (rec.table_lane == lane) return true;
    kimkv_decode_item const first = a.items[rec.table_lane];
    return lane_valid(P, first, a.lanes[rec.table_lane].tokens) && first.layer == item.layer;
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

// One query row of the unit.
struct QueryRow {
    const uint16_t* query;   // nullptr: no row
    float scale2;            // attention scale * log2 e
};

// Parts of kRows rows: lane i holds o[r][k] of dim i + 64 k, every lane m and l.
struct RowParts {
    float o[kRows][4];
    float m[kRows];
    float l[kRows];
};

__device__ void attend_rows_generic(const PoolView& P, const kimkv_decode_item& table, uint32_t h, uint32_t c0,
                                    uint32_t c1, QueryRow const (&rows)[kRows], RowParts& out)
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
            q[r][k] = rows[r].query != nullptr && d < D ? __half2float(__ushort_as_half(rows[r].query[d])) : 0.0f;
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

// Where the part of (lane index i of the unit, query head q) goes.
struct PartOut {
    float* o;
    float2* ml;
    uint16_t* output;   // instead, for a lane of one part
};

__device__ inline PartOut part_out(const SharedArgs& a, const SharedUnit& u, uint32_t D, uint32_t i, uint32_t q)
{
    uint64_t const row = static_cast<uint64_t>(u.slot + i) * a.QH + q;
    PartOut to{a.parts.o + row * D, a.parts.ml + row, nullptr};
    if (u.single != 0) to.output = a.items[u.lane + i].output + static_cast<uint64_t>(q) * D;
    return to;
}

// The whole unit by the generic path.  A task is kRows columns of one KV head;
// where there are fewer tasks than waves, the waves of a task take a part of
// the tokens each.
__device__ void unit_generic(const PoolView& P, const SharedArgs& a, const SharedUnit& u, GenericLds& lds)
{
    uint32_t const tid = threadIdx.x;
    uint32_t const wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint32_t const D = P.dim;
    uint32_t const G = a.QH / P.heads;
    uint32_t const columns = u.lanes * G;
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
            QueryRow rows[kRows];
#pragma unroll
            for (uint32_t r = 0; r < kRows; ++r) {
                rows[r] = QueryRow{nullptr, 0.0f};
                uint32_t const c = col0 + r;
                if (c < columns && lane_ok(P, a, u.lane + c / G)) {
                    kimkv_decode_item const& item = a.items[u.lane + c / G];
                    rows[r] = QueryRow{item.query + (static_cast<uint64_t>(h) * G + c % G) * D, item.attention_scale * kLog2e};
                }
            }
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
            if (mine >= tasks || c >= columns || !lane_ok(P, a, u.lane + c / G)) continue;
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
            PartOut const to = part_out(a, u, D, c / G, (u.head + mine / batches) * G + c % G);
            if (to.output != nullptr) {
                to.output[d] = __half_as_ushort(__float2half_rn(l > 0.0f ? o / l : l == 0.0f ? 0.0f : l));
            } else {
                to.o[d] = o;
                if (d == 0) *to.ml = make_float2(M, l);
            }
        }
        __syncthreads();
    }
}

__global__ __launch_bounds__(kBlock) void shared_decode_kernel(PoolView P, SharedArgs a)
{
    __shared__ GenericLds lds;
    SharedUnit const u = a.units[xcd_logical_index(blockIdx.x, gridDim.x)];
    if (u.lanes == 0) return;
    // The entries lie in the caller's memory: nothing outside the launch's buffers is touched, whatever they hold.
    if (u.table_lane >= a.lane_count || u.lanes > a.lane_count || u.lane > a.lane_count - u.lanes || u.heads == 0
        || u.head + u.heads > P.heads || u.begin >= u.end
        || (u.single == 0 && (u.lanes > a.slot_count || u.slot > a.slot_count - u.lanes))) {
        report_fault(P, KIMKV_FAULT_DECODE_ITEM);
        return;
    }
    bool bad = false;
    for (uint32_t i = threadIdx.x; i < u.lanes; i += kBlock) bad |= !lane_ok(P, a, u.lane + i);
    if (__syncthreads_or(bad)) report_fault(P, KIMKV_FAULT_DECODE_ITEM);
    if (!lane_valid(P, a.items[u.table_lane], a.lanes[u.table_lane].tokens) || u.end > a.lanes[u.table_lane].tokens) {
        report_fault(P, KIMKV_FAULT_DECODE_ITEM);
        return;
    }
    unit_generic(P, a, u, lds);
}

// Merges the lanes' parts: block = (lane, kMergeRows query heads), kMergeThreads
// threads a head.
constexpr unsigned kMergeBlock = 256;

__global__ __launch_bounds__(kMergeBlock) void shared_merge_kernel(PoolView P, SharedArgs a)
{
    uint32_t const lane = blockIdx.x;
    SharedLane const rec = a.lanes[lane];
    if (rec.merged == 0 || !lane_ok(P, a, lane)) return;   // a unit reported it
    uint64_t const last_prefix = static_cast<uint64_t>(rec.prefix_slot) + static_cast<uint64_t>(rec.prefix_stride) * rec.prefix_count;
    uint64_t const last_tail = static_cast<uint64_t>(rec.tail_slot) + rec.tail_count;
    if (rec.prefix_count > a.slot_count || rec.tail_count > a.slot_count) return;
    if ((rec.prefix_count != 0 && last_prefix - rec.prefix_stride >= a.slot_count) || (rec.tail_count != 0 && last_tail > a.slot_count)) return;
    uint32_t const D = P.dim;
    uint32_t const parts = rec.prefix_count + rec.tail_count;
    auto row = [&](uint32_t i, uint32_t q) {
        uint32_t const slot = i < rec.prefix_count ? rec.prefix_slot + i * rec.prefix_stride : rec.tail_slot + i - rec.prefix_count;
        return static_cast<uint64_t>(slot) * a.QH + q;
    };
    uint16_t* const output = a.items[lane].output;
    for (uint32_t x = blockIdx.y * kMergeBlock + threadIdx.x; x < a.QH * D; x += gridDim.y * kMergeBlock) {
        uint32_t const q = x / D;
        uint32_t const d = x - q * D;
        float M = -INFINITY;
        for (uint32_t i = 0; i < parts; ++i) M = fmaxf(M, a.parts.ml[row(i, q)].x);
        float o = 0.0f;
        float l = 0.0f;
        for (uint32_t i = 0; i < parts; ++i) {
            float2 const ml = a.parts.ml[row(i, q)];
            float const f = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - M);
            if (f == 0.0f) continue;   // whatever V made of it, as for a key of weight 0
            o += f * a.parts.o[row(i, q) * D + d];
            l += f * ml.y;
        }
        output[x] = __half_as_ushort(__float2half_rn(l > 0.0f ? o / l : l == 0.0f ? 0.0f : l));
    }
}

// ---- planning -----------------------------------------------------------------

constexpr uint32_t kShareBlock = 64;     // tokens: a shared prefix is cut to whole blocks
constexpr uint32_t kMinShared = 64;

struct Planned {
    std::vector<SharedUnit> units;
    std::vector<SharedLane> lanes;
    uint64_t slots{0};
    uint32_t merge_lanes{0};
    uint32_t column_blocks{0};
};

uint64_t align16(uint64_t n) { return (n + 15) / 16 * 16; }

bool plan_batch(uint32_t H, uint32_t D, uint32_t QH, uint32_t compute_units, const uint32_t* tokens, uint32_t lane_count,
                const kimkv_shared_group* groups, uint32_t group_count, Planned& out)
{
    out.lanes.resize(lane_count);
    for (uint32_t i = 0; i < lane_count; ++i) out.lanes[i] = SharedLane{i, tokens[i], 0, 0, 0, 0, 0, 0};
    std::vector<uint8_t> grouped(lane_count, 0);
    std::vector<uint32_t> shared(lane_count, 0);   // tokens of the lane that a group's units take
    constexpr uint32_t kPiece = 1024;
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
        if (group.lane_count < 2 || prefix < kMinShared) continue;
        uint32_t const pieces = (prefix + kPiece - 1) / kPiece;
        for (uint32_t i = 0; i < group.lane_count; ++i) {
            SharedLane& lane = out.lanes[group.first_lane + i];
            lane.table_lane = group.first_lane;
            lane.prefix_slot = static_cast<uint32_t>(out.slots + i);
            lane.prefix_stride = group.lane_count;
            lane.prefix_count = pieces;
            shared[group.first_lane + i] = prefix;
        }
        for (uint32_t p = 0; p < pieces; ++p) {
            for (uint32_t h = 0; h < H; ++h) {
                out.units.push_back(SharedUnit{group.first_lane, group.first_lane, group.lane_count, p * kPiece,
                                               std::min(prefix, (p + 1) * kPiece), static_cast<uint32_t>(out.slots),
                                               static_cast<uint16_t>(h), 1, 0});
            }
            out.slots += group.lane_count;
        }
    }
    for (uint32_t i = 0; i < lane_count; ++i) {
        SharedLane& lane = out.lanes[i];
        uint32_t const own = tokens[i] - shared[i];
        uint32_t const pieces = (own + kPiece - 1) / kPiece;
        lane.tail_slot = static_cast<uint32_t>(out.slots);
        lane.tail_count = pieces;
        bool const single = pieces == 1 && lane.prefix_count == 0;
        lane.merged = !single && pieces + lane.prefix_count != 0 ? 1 : 0;
        out.merge_lanes += lane.merged;
        for (uint32_t p = 0; p < pieces; ++p) {
            out.units.push_back(SharedUnit{i, i, 1, shared[i] + p * kPiece, std::min(tokens[i], shared[i] + (p + 1) * kPiece),
                                           static_cast<uint32_t>(out.slots), 0, static_cast<uint16_t>(H), single ? 1u : 0u});
            if (!single) out.slots += 1;
        }
    }
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
        plan->column_blocks = p.column_blocks;
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
    shared_decode_kernel<<<plan->unit_count, kBlock, 0, s>>>(pv, a);
    kernel_timing_end(TimedKernel::Decode, s, start);
    kimkv_status const status = launch_status();
    if (status != KIMKV_OK || plan->merge_lanes == 0) return status;
    uint32_t const blocks = ceil_div(static_cast<uint64_t>(plan->query_heads) * D, kMergeBlock);
    shared_merge_kernel<<<dim3(plan->lane_count, blocks < 65535u ? blocks : 65535u), kMergeBlock, 0, s>>>(pv, a);
    return launch_status();
}

}  // extern "C"
