// logits_kernels.hip -- penalties, biases and allowed-token masks on rows of
// fp32 logits, and the greedy token of each adjusted row, in one read.
//
// The work follows the vocabulary: block = (slice of the vocabulary, row).  A
// slice's logits are on their way to registers, 16 bytes a lane, while the
// block counts the history's tokens of its slice in LDS, a word a token.  Then
// one thread for each token that occurs, and one for each bias, replaces the
// word by the changed logit: a few hundred of a slice's thousands.  So each
// logit is read once: exchanged where its word says so, stored if wanted (past
// the caches: 67 for 71 us) and folded into the slice's maximum.  A second,
// small launch picks the first of the blocks' maxima where a row takes several.
//
// Bound by HBM where rows are many and wide: 256 rows of 128000, stored, with
// 4000 history tokens, 100 biases and masks take 70 us (265 MB, 3.8 TB/s), the
// rows alone 53.  The lists' share is their chain (entries, counts, logits,
// four barriers) and that every slice looks at the whole history, so slices are
// large: 1024 threads and 16384 tokens, two blocks a compute unit; halves of
// that took 80 for 71.  By the two launches where they are few: 8.2 us for 4
// rows of 32000, 11.5 for 72.  The reference picks the plain argmax
// (src/cuda/model/kernels.cuh:111-117).
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "attention_common.h"
#include "device_common.h"
#include "runtime_internal.h"

namespace kimkv {
namespace {

constexpr unsigned kBlock = 1024;
constexpr uint32_t kVecs = 4;          // 16-byte vectors of a row's logits a thread holds
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

// The wave's: the first token of the highest value.  (No token, the highest number, has the lowest value.)
__device__ inline Best wave_best(Best best)
{
    float const value = wave_max(best.value);
    uint32_t token = best.value == value ? best.token : KIMKV_NO_TOKEN;
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) token = min(token, static_cast<uint32_t>(__shfl_xor(static_cast<int>(token), m)));
    return Best{value, token};
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

// A slice of a row: positions [first, first + count) of its tokens, which
// stand `shift` positions further so that every fourth position is a 16-byte
// address of the row's logits.
struct Slice {
    uint32_t first;
    uint32_t count;
    uint32_t shift;
    uint32_t V;
    // The token's place in the slice; count or more: it is not in it.
    __device__ uint32_t place(uint32_t token) const { return token < V ? token + shift - first : 0xFFFFFFFFu; }
    __device__ float logit(const float* row, uint32_t place) const { return place < count ? row[first + place - shift] : 0.0f; }
};

// A changed logit as its token's word: never 0, which stands for one that is as it was.
__device__ inline uint32_t word_of(float x) { return x == x ? ~__float_as_uint(x) : ~0x7FC00000u; }
__device__ inline float value_of(uint32_t word, float unchanged) { return word != 0 ? __uint_as_float(~word) : unchanged; }

// A logit whose token occurs `seen` times, as the penalties leave it.  Each operation rounds by itself.
__device__ inline float penalized(float x, uint32_t seen, const kimkv_logits_rule& r)
{
#pragma clang fp contract(off)
    x = x > 0.0f ? x / r.repetition_penalty : x * r.repetition_penalty;
    return x - (r.frequency_penalty * static_cast<float>(seen) + r.presence_penalty);
}

// Slices are `per` positions, a multiple of 4 kBlock up to 4 kBlock kVecs.
struct SliceLds {
    uint4 words[kBlock * kVecs];
    uint32_t taken[kBlock * kVecs / 8];   // a bit a token: some thread has it in hand
    uint32_t owners[kOwners];
    Best best[kBlock / kWave];
};

constexpr uint32_t kAhead = 4;   // history entries of a thread in flight
constexpr uint32_t kHistoryStep = kAhead * kBlock;

// kAhead entries from entry `at` on: their places and logits.
struct Entries {
    uint32_t place[kAhead];
    float logit[kAhead];
    __device__ void find(const kimkv_logits_rule& r, const Slice& slice, uint32_t at)
    {
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) {
            uint32_t const n = at + i * kBlock + threadIdx.x;
            place[i] = n < r.history_count ? slice.place(r.history[n]) : 0xFFFFFFFFu;
        }
    }
    __device__ void read(const float* from, const Slice& slice)
    {
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) logit[i] = slice.logit(from, place[i]);
    }
};

// The words of the tokens in the history: how often each occurs, then the
// penalized logit.  The words are 0 before, `e` those of entry 0 on.
__device__ void apply_history(SliceLds& lds, Entries& e, const float* from, const kimkv_logits_rule& r,
                              const Slice& slice)
{
    uint32_t* const words = reinterpret_cast<uint32_t*>(lds.words);
    uint32_t at = 0;
    for (;;) {
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) {
            if (e.place[i] < slice.count) atomicAdd(words + e.place[i], 1u);
        }
        if (r.history_count - at <= kHistoryStep) break;
        at += kHistoryStep;
        e.find(r, slice, at);
        e.read(from, slice);
    }
    __syncthreads();
    // The last entries are still at hand; the others are read again.
    for (;;) {
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) {
            if (e.place[i] >= slice.count) continue;
            uint32_t const bit = 1u << (e.place[i] & 31u);
            if ((atomicOr(lds.taken + (e.place[i] >> 5), bit) & bit) != 0) continue;
            words[e.place[i]] = word_of(penalized(e.logit[i], words[e.place[i]], r));
        }
        if (at == 0) break;
        at -= kHistoryStep;
        e.find(r, slice, at);
        e.read(from, slice);
    }
}

// A bias of the list.
struct Bias {
    uint32_t place;
    float value;
    float logit;   // its token's, unchanged
};

__device__ inline Bias bias_at(const kimkv_logits_rule& r, const Slice& slice, uint32_t i)
{
    if (i >= r.bias_count) return Bias{0xFFFFFFFFu, 0.0f, 0.0f};
    return Bias{slice.place(r.bias_tokens[i]), r.bias_values[i], 0.0f};
}

// Adds the biases of the slice's tokens to their logits, those of one token in
// the list's order: of the entries a round looks at, each thread holds one, and
// of the entries of one token (of one owner word: tokens that share it wait for
// each other) the first left goes.  `bias` is the first round's.
__device__ void apply_biases(SliceLds& lds, Bias bias, const float* from, const kimkv_logits_rule& r, const Slice& slice)
{
    uint32_t const tid = threadIdx.x;
    uint32_t* const words = reinterpret_cast<uint32_t*>(lds.words);
    for (uint32_t at = 0; at < r.bias_count; at += kBlock) {
        if (at != 0) {
            bias = bias_at(r, slice, at + tid);
            bias.logit = slice.logit(from, bias.place);
        }
        bool waits = bias.place < slice.count;
        do {
            uint32_t* const owner = lds.owners + (bias.place & (kOwners - 1));
            if (waits) atomicMin(owner, tid);
            __syncthreads();
            if (waits && *owner == tid) {
                words[bias.place] = word_of(value_of(words[bias.place], bias.logit) + bias.value);
                *owner = 0xFFFFFFFFu;
                waits = false;
            }
        } while (__syncthreads_or(waits) != 0);
    }
}

__global__ __launch_bounds__(kBlock) void logits_kernel(const float* logits, uint32_t V, uint32_t per,
                                                        const kimkv_logits_rule* rules, float* out, uint32_t* tokens,
                                                        Best* partial)
{
    __shared__ SliceLds lds;
    uint32_t const tid = threadIdx.x;
    uint32_t const row = blockIdx.y;
    const float* const from = logits + static_cast<uint64_t>(row) * V;
    Slice const slice{blockIdx.x * per, per, static_cast<uint32_t>(reinterpret_cast<uintptr_t>(from) >> 2) & 3u, V};
    uint32_t const vecs = per / (4 * kBlock);
    // Vector j of this thread holds tokens token(j) + 0 .. 3, those below V (a token in front of the row is a huge one).
    auto const token = [&](uint32_t j) { return slice.first + 4 * (j * kBlock + tid) - slice.shift; };
    auto const whole = [&](uint32_t v) { return v < V && V - v > 3; };
    // The lists are asked for first: loads come back in order.
    RowRule const rule = load_rule(rules, row);
    kimkv_logits_rule const& r = rule.r;
    Entries entries{};
    Bias bias{};
    if (rule.valid) {
        entries.find(r, slice, 0);
        bias = bias_at(r, slice, tid);
    }
    f32x4_t x[kVecs];
#pragma unroll
    for (uint32_t j = 0; j < kVecs; ++j) {
        x[j] = f32x4_t{};
        uint32_t const v = token(j);
        if (j < vecs && whole(v)) {
            x[j] = *reinterpret_cast<const f32x4_t*>(from + v);
        } else if (j < vecs) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                if (v + i < V) x[j][i] = from[v + i];
            }
        }
    }
    if (rule.valid) {
        entries.read(from, slice);
        bias.logit = slice.logit(from, bias.place);
    }
    Best best{-INFINITY, KIMKV_NO_TOKEN};
    if (rule.valid) {
        bool const changes = (r.history_count | r.bias_count) != 0;
        if (changes) {
            for (uint32_t i = tid; i < vecs * kBlock; i += kBlock) lds.words[i] = uint4{0, 0, 0, 0};
            for (uint32_t i = tid; i < vecs * kBlock / 8; i += kBlock) lds.taken[i] = 0;
            for (uint32_t i = tid; i < kOwners; i += kBlock) lds.owners[i] = 0xFFFFFFFFu;
            __syncthreads();
            if (r.history_count != 0) {
                apply_history(lds, entries, from, r, slice);
                __syncthreads();
            }
            apply_biases(lds, bias, from, r, slice);
            __syncthreads();
        }
        float* const to = out + static_cast<uint64_t>(row) * V;
        bool const aligned = ((reinterpret_cast<uintptr_t>(to) >> 2) & 3u) == slice.shift;
#pragma unroll
        for (uint32_t j = 0; j < kVecs; ++j) {
            if (j >= vecs) break;
            uint32_t const v = token(j);
            bool const all = whole(v);
            uint32_t allowed = 15;
            if (r.allowed != nullptr && all) {
                uint64_t const two = r.allowed[v >> 5] | static_cast<uint64_t>(r.allowed[(v + 3) >> 5]) << 32;
                allowed = static_cast<uint32_t>(two >> (v & 31u));
            }
            if (!all) {
                uint32_t there = 0;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    if (v + i >= V) continue;
                    there |= (r.allowed == nullptr ? 1u : r.allowed[(v + i) >> 5] >> ((v + i) & 31u) & 1u) << i;
                }
                allowed = there;
            }
            uint4 word{0, 0, 0, 0};
            if (changes) word = lds.words[j * kBlock + tid];
            uint32_t const w[4] = {word.x, word.y, word.z, word.w};
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                float const value = value_of(w[i], x[j][i]);
                bool const may = (allowed >> i & 1u) != 0;
                x[j][i] = may ? value : -INFINITY;
                // A thread's tokens ascend, so an equal value is no better.
                if (may && (value > best.value || (best.token == KIMKV_NO_TOKEN && value == value))) best = Best{value, v + i};
            }
            if (out == nullptr) continue;
            if (all && aligned) {
                __builtin_nontemporal_store(x[j], reinterpret_cast<f32x4_t*>(to + v));
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    if (v + i < V) to[v + i] = x[j][i];
                }
            }
        }
    }
    if (tokens == nullptr) return;
    best = wave_best(best);
    if ((tid & (kWave - 1)) == 0) lds.best[tid / kWave] = best;
    __syncthreads();
    if (tid >= kWave) return;
    best = wave_best(lds.best[tid < kBlock / kWave ? tid : 0]);
    if (tid != 0) return;
    if (gridDim.x == 1) {
        tokens[row] = best.token;
    } else {
        partial[static_cast<uint64_t>(row) * gridDim.x + blockIdx.x] = best;
    }
}

constexpr unsigned kPickBlock = 256;

// One wave a row: the first of the slices' maxima.
__global__ __launch_bounds__(kPickBlock) void logits_pick_kernel(const Best* partial, uint32_t rows, uint32_t slices,
                                                             uint32_t* tokens)
{
    uint32_t const row = blockIdx.x * (kPickBlock / kWave) + threadIdx.x / kWave;
    if (row >= rows) return;
    Best best{-INFINITY, KIMKV_NO_TOKEN};
    for (uint32_t i = threadIdx.x & (kWave - 1); i < slices; i += kWave) {
        Best const b = partial[static_cast<uint64_t>(row) * slices + i];
        take_best(best, b.value, b.token);
    }
    best = wave_best(best);
    if ((threadIdx.x & (kWave - 1)) == 0) tokens[row] = best.token;
}

// How rows are cut: slices of 4096 positions up to 16384, those whose rounds
// of the blocks that run at once, and the second launch where a row takes
// several, come to least.  A round takes about 3.5 us and 1.2 for each 4096
// positions, the second launch 2.5.  (Slices as large as leave 512 blocks took
// 11.2 us for 101 rows of 20562, 10.7 for 242 of 6793, 11.1 for 153 of 10726
// and 19.0 for 85 of 99226, these 9.9, 7.7, 9.2 and 17.4.  A block of 1024
// threads for a row of 32000 saves the second launch too and loses more: 12.6
// us for 4 rows and 16.2 for 72, where slices took 9.2 and 13.4.)
constexpr uint32_t kBlocksAtOnce = 512;

struct RowCut {
    uint32_t per;
    uint32_t slices;
};

RowCut row_cut(uint32_t rows, uint32_t vocabulary)
{
    RowCut cut{};
    double best = 0.0;
    for (uint32_t vecs = 1; vecs <= kVecs; ++vecs) {
        uint32_t const per = 4 * kBlock * vecs;
        uint32_t const slices = ceil_div(vocabulary + 3ull, per);   // 3: a row's shift
        uint32_t const rounds = ceil_div(static_cast<uint64_t>(rows) * slices, kBlocksAtOnce);
        double const cost = rounds * (3.5 + 1.2 * vecs) + (slices > 1 ? 2.5 : 0.0);
        if (cut.per == 0 || cost < best) {
            best = cost;
            cut = RowCut{per, slices};
        }
    }
    return cut;
}

}  // namespace
}  // namespace kimkv

using namespace kimkv;

extern "C" {

// A row is cut into more slices in a small batch than in a large one, so the
// size is that of the smallest slices, whatever the batch: enough for fewer rows too.
size_t kimkv_logits_workspace_bytes(uint32_t rows, uint32_t vocabulary)
{
    uint32_t const slices = ceil_div(vocabulary + 3ull, 4 * kBlock);
    return slices <= 1 ? 0 : static_cast<size_t>(rows) * slices * sizeof(Best);
}

kimkv_status kimkv_model_logits_adjust(const float* logits, uint32_t rows, uint32_t vocabulary,
                                       const kimkv_logits_rule* device_rules, float* out, uint32_t* device_tokens,
                                       void* workspace, kimkv_stream_t stream)
{
    if (logits == nullptr || vocabulary == 0 || vocabulary > 0x7FFFFFFFu || (out == nullptr && device_tokens == nullptr)) {
        return KIMKV_INVALID_ARGUMENT;
    }
    RowCut const cut = row_cut(rows, vocabulary);
    bool const split = cut.slices > 1 && device_tokens != nullptr;
    if (split && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 7u) != 0) && rows != 0) {
        return KIMKV_INVALID_ARGUMENT;
    }
    auto* const partial = static_cast<Best*>(workspace);
    // A launch takes 65535 rows of a grid.
    for (uint32_t first = 0; first < rows;) {
        uint32_t const n = rows - first < 65535u ? rows - first : 65535u;
        uint64_t const at = static_cast<uint64_t>(first) * vocabulary;
        Best* const part = split ? partial + static_cast<uint64_t>(first) * cut.slices : nullptr;
        logits_kernel<<<dim3(cut.slices, n), kBlock, 0, native(stream)>>>(
            logits + at, vocabulary, cut.per, device_rules != nullptr ? device_rules + first : nullptr,
            out != nullptr ? out + at : nullptr, device_tokens != nullptr ? device_tokens + first : nullptr, part);
        kimkv_status const status = launch_status();
        if (status != KIMKV_OK) return status;
        first += n;
    }
    if (!split || rows == 0) return KIMKV_OK;
    logits_pick_kernel<<<ceil_div(rows, kPickBlock / kWave), kPickBlock, 0, native(stream)>>>(partial, rows, cut.slices,
                                                                                             device_tokens);
    return launch_status();
}

}  // extern "C"
