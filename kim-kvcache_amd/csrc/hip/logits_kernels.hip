// logits_kernels.hip -- penalties, biases and allowed-token masks on rows of
// fp32 logits, and the greedy token of each adjusted row, in one read.
//
// The work follows the vocabulary: block = (slice of kSlice tokens, row).  A
// block counts the history's tokens of its slice and adds up its biases in
// LDS, then takes the slice's logits once: adjusted, stored if wanted, and
// folded into the slice's maximum.  A second, small launch picks the first of
// the slices' maxima.  The reference picks the plain argmax
// (src/cuda/model/kernels.cuh:111-117).
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "device_common.h"
#include "runtime_internal.h"

namespace kimkv {
namespace {

constexpr unsigned kBlock = 256;
constexpr unsigned kWaves = kBlock / kWave;
constexpr uint32_t kSlice = 8192;      // tokens of the vocabulary a block takes
constexpr uint32_t kOwners = 1024;

typedef float f32x4_t __attribute__((ext_vector_type(4)));

// A candidate for a row's token; token KIMKV_NO_TOKEN: none.
struct Best {
    float value;
    uint32_t token;
};

// The first index of the highest value, whatever the order of the calls.
__device__ inline void take_best(Best& best, float value, uint32_t token)
{
    if (token != KIMKV_NO_TOKEN
        && (best.token == KIMKV_NO_TOKEN || value > best.value || (value == best.value && token < best.token))) {
        best = Best{value, token};
    }
}

__device__ inline Best wave_best(Best best)
{
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        float const v = __shfl_xor(best.value, m);
        uint32_t const t = __shfl_xor(best.token, m);
        take_best(best, v, t);
    }
    return best;
}

struct RowRule {
    kimkv_logits_rule r;
    bool valid;
};

__device__ inline RowRule load_rule(const kimkv_logits_rule* rules, uint32_t row)
{
    RowRule rule{};
    rule.r.repetition_penalty = 1.0f;
    rule.valid = true;
    if (rules != nullptr) {
        rule.r = rules[row];
        float const p = rule.r.repetition_penalty;
        rule.valid = p > 0.0f && p < INFINITY && ((rule.r.history_count | rule.r.bias_count) >> 31) == 0
            && (rule.r.history_count == 0 || rule.r.history != nullptr)
            && (rule.r.bias_count == 0 || (rule.r.bias_tokens != nullptr && rule.r.bias_values != nullptr));
    }
    return rule;
}

// The tokens [s0, s1) of a row as the rule changes them.
struct SliceLds {
    uint32_t seen[kSlice];    // times a token occurs in the history
    float bias[kSlice];
    uint32_t owner[kOwners];
    Best best[kWaves];
};

// Adds the biases of the slice's tokens, those of one token in the list's
// order: of the 256 entries a round looks at, each thread holds one, and of
// the entries of one token (of one owner word: tokens that share it wait for
// each other) the first left goes.
__device__ void add_biases(SliceLds& lds, const kimkv_logits_rule& r, uint32_t s0, uint32_t s1)
{
    uint32_t const tid = threadIdx.x;
    for (uint32_t at = 0; at < r.bias_count; at += kBlock) {
        uint32_t token = KIMKV_NO_TOKEN;
        float value = 0.0f;
        if (r.bias_count - at > tid) {
            token = r.bias_tokens[at + tid];
            value = r.bias_values[at + tid];
        }
        bool waits = token >= s0 && token < s1;
        while (__syncthreads_or(waits) != 0) {
            uint32_t* const owner = lds.owner + (token & (kOwners - 1));
            if (waits) atomicMin(owner, tid);
            __syncthreads();
            if (waits && *owner == tid) {
                lds.bias[token - s0] += value;
                *owner = 0xFFFFFFFFu;
                waits = false;
            }
        }
    }
}

// One logit as the rule leaves it.  Each operation rounds by itself.
__device__ inline float adjusted(float x, uint32_t seen, float bias, const kimkv_logits_rule& r)
{
#pragma clang fp contract(off)
    if (seen != 0) {
        x = x > 0.0f ? x / r.repetition_penalty : x * r.repetition_penalty;
        x -= r.frequency_penalty * static_cast<float>(seen) + r.presence_penalty;
    }
    return x + bias;
}

__global__ __launch_bounds__(kBlock) void logits_kernel(const float* logits, uint32_t V, uint32_t per,
                                                        const kimkv_logits_rule* rules, float* out, uint32_t* tokens,
                                                        Best* partial)
{
    __shared__ SliceLds lds;
    uint32_t const tid = threadIdx.x;
    uint32_t const row = blockIdx.y;
    uint32_t const s0 = blockIdx.x * per;
    uint32_t const s1 = min(s0 + per, V);
    RowRule const rule = load_rule(rules, row);
    kimkv_logits_rule const& r = rule.r;
    Best best{-INFINITY, KIMKV_NO_TOKEN};
    if (rule.valid) {
        for (uint32_t i = tid; i < s1 - s0; i += kBlock) {
            lds.seen[i] = 0;
            lds.bias[i] = -0.0f;   // the sum of no biases: x + -0 is x
        }
        for (uint32_t i = tid; i < kOwners; i += kBlock) lds.owner[i] = 0xFFFFFFFFu;
        __syncthreads();
        for (uint32_t i = tid; i < r.history_count; i += kBlock) {
            uint32_t const token = r.history[i];
            if (token >= s0 && token < s1) atomicAdd(&lds.seen[token - s0], 1u);
        }
        add_biases(lds, r, s0, s1);
        __syncthreads();
        uint64_t const at = static_cast<uint64_t>(row) * V;
        for (uint32_t v = s0 + tid; v < s1; v += kBlock) {
            float x = adjusted(logits[at + v], lds.seen[v - s0], lds.bias[v - s0], r);
            bool const allowed = r.allowed == nullptr || ((r.allowed[v >> 5] >> (v & 31u)) & 1u) != 0;
            if (!allowed) x = -INFINITY;
            if (out != nullptr) out[at + v] = x;
            if (allowed && x == x) take_best(best, x, v);
        }
    }
    if (tokens == nullptr) return;
    best = wave_best(best);
    if ((tid & (kWave - 1)) == 0) lds.best[tid / kWave] = best;
    __syncthreads();
    if (tid != 0) return;
    for (uint32_t w = 1; w < kWaves; ++w) take_best(best, lds.best[w].value, lds.best[w].token);
    if (gridDim.x == 1) {
        tokens[row] = best.token;
    } else {
        partial[static_cast<uint64_t>(row) * gridDim.x + blockIdx.x] = best;
    }
}

// One wave a row: the first of the slices' maxima.
__global__ __launch_bounds__(kBlock) void logits_pick_kernel(const Best* partial, uint32_t rows, uint32_t slices,
                                                             uint32_t* tokens)
{
    uint32_t const row = blockIdx.x * kWaves + threadIdx.x / kWave;
    if (row >= rows) return;
    Best best{-INFINITY, KIMKV_NO_TOKEN};
    for (uint32_t i = threadIdx.x & (kWave - 1); i < slices; i += kWave) {
        Best const b = partial[static_cast<uint64_t>(row) * slices + i];
        take_best(best, b.value, b.token);
    }
    best = wave_best(best);
    if ((threadIdx.x & (kWave - 1)) == 0) tokens[row] = best.token;
}

uint32_t logits_slices(uint32_t vocabulary) { return ceil_div(vocabulary, kSlice); }

}  // namespace
}  // namespace kimkv

using namespace kimkv;

extern "C" {

size_t kimkv_logits_workspace_bytes(uint32_t rows, uint32_t vocabulary)
{
    uint32_t const slices = logits_slices(vocabulary);
    return slices <= 1 ? 0 : static_cast<size_t>(rows) * slices * sizeof(Best);
}

kimkv_status kimkv_model_logits_adjust(const float* logits, uint32_t rows, uint32_t vocabulary,
                                       const kimkv_logits_rule* device_rules, float* out, uint32_t* device_tokens,
                                       void* workspace, kimkv_stream_t stream)
{
    if (logits == nullptr || vocabulary == 0 || vocabulary > 0x7FFFFFFFu || (out == nullptr && device_tokens == nullptr)) {
        return KIMKV_INVALID_ARGUMENT;
    }
    uint32_t const slices = logits_slices(vocabulary);
    bool const split = slices > 1 && device_tokens != nullptr;
    if (split && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 7u) != 0) && rows != 0) {
        return KIMKV_INVALID_ARGUMENT;
    }
    uint32_t const per = ceil_div(vocabulary, slices);
    auto* const partial = static_cast<Best*>(workspace);
    // A launch takes 65535 rows of a grid.
    for (uint32_t first = 0; first < rows;) {
        uint32_t const n = rows - first < 65535u ? rows - first : 65535u;
        uint64_t const at = static_cast<uint64_t>(first) * vocabulary;
        Best* const part = split ? partial + static_cast<uint64_t>(first) * slices : nullptr;
        logits_kernel<<<dim3(slices, n), kBlock, 0, native(stream)>>>(
            logits + at, vocabulary, per, device_rules != nullptr ? device_rules + first : nullptr,
            out != nullptr ? out + at : nullptr, device_tokens != nullptr ? device_tokens + first : nullptr, part);
        kimkv_status const status = launch_status();
        if (status != KIMKV_OK) return status;
        first += n;
    }
    if (!split || rows == 0) return KIMKV_OK;
    logits_pick_kernel<<<ceil_div(rows, kWaves), kBlock, 0, native(stream)>>>(partial, rows, slices, device_tokens);
    return launch_status();
}

}  // extern "C"
