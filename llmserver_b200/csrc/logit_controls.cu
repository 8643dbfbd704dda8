// A step's logits under its requests' controls, and the token drawn from them.
//
// For token v of row r with logit l, in this order, each step rounded to 32 bits:
//
//   v stands in the request (prompt or answer):    l <- l > 0 ? l / repetition : l * repetition
//   v stands c > 0 times in the answer:            l <- (l - c * frequency) - presence
//   the row's list has a bias for v:               l <- l + bias
//   the row's mask has no bit for v:               l <- -inf
//
// What a request holds is read from its history, a row of token ids of which the first `prompt` are the prompt: nothing is counted
// from call to call, so a call that is repeated gives the same, and a request that was put out and comes back has nothing to rebuild.
// A block takes a slice of the vocabulary of one row and keeps one word per token of the slice in shared memory: the times it stands
// in the answer (30 bits), whether a bias is listed, whether it stands in the prompt.  It walks the row's whole history and marks the
// tokens of its slice (integer atomics: their order does not matter), then walks the slice's logits once.  The logits of its first
// turn are asked for before the history, so that the two reads overlap.
//
// Sampling (sampling.cu's rule) takes the controlled logits as they are made, without writing them.  A second kernel picks the best
// slice of a row, gives -1 where nothing is left to draw from, and writes the token behind the request's history: all histories have
// been read by then, whatever rows share one.
//
// What bounds it: the logits, read once (and written once by the form that returns them).
#include "sampling.cuh"

// (the caller fills this in field by field)
struct LlmControls {
    const float* penalties;             // [rows][3]: repetition, presence, frequency; null: none
    const int* history;                 // [histories][capacity]
    const int* history_rows;            // [rows]; -1: none
    const int* lengths;                 // [rows]
    const int* prompt_lengths;          // [rows]
    int histories, capacity;
    const int* bias_starts;             // [lists + 1]
    const int* bias_ids;                // ascending within a list
    const float* bias_values;
    const int* bias_rows;               // [rows]; -1: none
    int bias_lists, bias_entries;
    const int* masks;                   // [masks][words], bit v % 32 of word v / 32
    const int* mask_rows;               // [rows]; -1: none
    int mask_count, mask_words;
    int* error_flag;
};

namespace {

using Controls = LlmControls;

constexpr uint32_t kPrompt = 0x80000000u, kBias = 0x40000000u, kTimes = 0x3fffffffu;
constexpr int kThreads = 512;
constexpr int kAhead = 8;               // logits a thread asks for at a time
constexpr int kMostSlice = 13824;       // tokens per slice: 54 KiB of words, four blocks of which fit an SM
constexpr int kBadRow = 8;              // error code: a row names a history, list or mask that does not exist

// What a block needs of its row.
struct RowControls {
    float repetition, presence, frequency;
    const int* history;
    int length, prompt;
    const int* bias_ids;
    const float* bias_values;
    int biases;
    const int* mask;
    bool marks;                         // words are kept for the slice
};

__device__ __forceinline__ RowControls controls_of(const Controls& c, int row) {
    RowControls r = {};
    bool bad = false;
    r.repetition = 1.0f;
    if (c.penalties != nullptr && c.history_rows != nullptr) {
        r.repetition = c.penalties[3 * (size_t)row];
        r.presence = c.penalties[3 * (size_t)row + 1];
        r.frequency = c.penalties[3 * (size_t)row + 2];
        const int at = c.history_rows[row];
        bad |= at >= c.histories;
        // penalties that change nothing need no history
        if (at >= 0 && at < c.histories && (r.repetition != 1.0f || r.presence != 0.0f || r.frequency != 0.0f)) {
            r.history = c.history + (size_t)at * c.capacity;
            r.length = min(max(c.lengths[row], 0), c.capacity);
            r.prompt = min(max(c.prompt_lengths[row], 0), r.length);
        }
    }
    if (c.bias_rows != nullptr) {
        const int list = c.bias_rows[row];
        bad |= list >= c.bias_lists;
        if (list >= 0 && list < c.bias_lists) {
            const int first = min(max(c.bias_starts[list], 0), c.bias_entries);
            const int last = min(max(c.bias_starts[list + 1], first), c.bias_entries);
            r.bias_ids = c.bias_ids + first;
            r.bias_values = c.bias_values + first;
            r.biases = last - first;
        }
    }
    if (c.mask_rows != nullptr) {
        const int mask = c.mask_rows[row];
        bad |= mask >= c.mask_count;
        if (mask >= 0 && mask < c.mask_count) r.mask = c.masks + (size_t)mask * c.mask_words;
    }
    if (bad && threadIdx.x == 0 && c.error_flag != nullptr) atomicExch(c.error_flag, kBadRow);
    r.marks = r.length > 0 || r.biases > 0;
    return r;
}

// Marks the tokens begin .. begin + count - 1 of the row's history and bias list.
__device__ __forceinline__ void mark_slice(const RowControls& r, uint32_t* marks, int begin, int count) {
    for (int i = threadIdx.x; i < count; i += blockDim.x) marks[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < r.length; i += blockDim.x) {
        const uint32_t place = (uint32_t)r.history[i] - (uint32_t)begin;
        if (place < (uint32_t)count) {
            if (i < r.prompt) atomicOr(&marks[place], kPrompt);
            else atomicAdd(&marks[place], 1u);
        }
    }
    for (int i = threadIdx.x; i < r.biases; i += blockDim.x) {
        const uint32_t place = (uint32_t)r.bias_ids[i] - (uint32_t)begin;
        if (place < (uint32_t)count) atomicOr(&marks[place], kBias);
    }
    __syncthreads();
}

__device__ float bias_of(const RowControls& r, int token) {
    int low = 0, high = r.biases - 1;
    while (low < high) {
        const int middle = (low + high) >> 1;
        if (r.bias_ids[middle] < token) low = middle + 1;
        else high = middle;
    }
    return r.bias_ids[low] == token ? r.bias_values[low] : 0.0f;
}

// The steps are rounded one by one (no fused multiply-add), as the formula above says.
__device__ __forceinline__ float controlled(const RowControls& r, float logit, uint32_t mark, int token) {
    if (mark != 0) {
        const uint32_t times = mark & kTimes;
        if (times != 0 || (mark & kPrompt)) logit = logit > 0.0f ? __fdiv_rn(logit, r.repetition) : __fmul_rn(logit, r.repetition);
        if (times != 0) logit = __fsub_rn(__fsub_rn(logit, __fmul_rn((float)times, r.frequency)), r.presence);
        if (mark & kBias) logit = __fadd_rn(logit, bias_of(r, token));
    }
    return logit;
}

// SAMPLE: each block leaves its slice's best score and token in `partial`; else the controlled logits go to `out` (which may be
// `logits`).  Slices begin at multiples of 32 tokens, so that a warp's 32 tokens share a word of the mask.
template <bool SAMPLE>
__global__ void __launch_bounds__(kThreads) control_kernel(const float* logits, float* out, const Controls c, int vocab, int per_slice,
                                                           const float* __restrict__ temperatures, const uint64_t* __restrict__ seeds,
                                                           const int* __restrict__ steps, float* __restrict__ partial_scores,
                                                           int* __restrict__ partial_indices) {
    pdl_trigger();
    pdl_wait();
    extern __shared__ uint32_t marks[];
    __shared__ float best_values[kThreads / 32];
    __shared__ int best_indices[kThreads / 32];
    const int row = blockIdx.y;
    const int begin = blockIdx.x * per_slice, end = min(vocab, begin + per_slice);
    const float* src = logits + (size_t)row * vocab;
    float values[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
        const int i = begin + (int)threadIdx.x + a * kThreads;
        values[a] = i < end ? src[i] : 0.0f;
    }
    const RowControls r = controls_of(c, row);
    if (r.marks) mark_slice(r, marks, begin, end - begin);
    float temperature = 0.0f;
    uint64_t seed = 0;
    uint32_t step = 0;
    if (SAMPLE && temperatures != nullptr) {
        temperature = temperatures[row];
        seed = seeds[row];
        step = (uint32_t)steps[row];
    }
    float best = -INFINITY;
    int best_index = 0x7fffffff;
    for (int first = begin + (int)threadIdx.x; first < end; first += kAhead * kThreads) {
        if (first >= begin + kAhead * kThreads) {
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                const int i = first + a * kThreads;
                values[a] = i < end ? src[i] : 0.0f;
            }
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int i = first + a * kThreads;
            if (i >= end) break;
            float logit = values[a];
            if (r.marks) logit = controlled(r, logit, marks[i - begin], i);
            if (r.mask != nullptr && ((uint32_t)__ldg(r.mask + (i >> 5)) >> (i & 31) & 1u) == 0) logit = -INFINITY;
            if (SAMPLE) {
                if (temperature > 0.0f) logit = logit / temperature - logf(-logf(uniform_for(seed, step, (uint32_t)i)));
                if (logit != logit) logit = -INFINITY;      // a NaN never wins
                take_better(best, best_index, logit, i);
            } else {
                out[(size_t)row * vocab + i] = logit;
            }
        }
    }
    if (!SAMPLE) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, best, offset);
        const int other_index = __shfl_xor_sync(0xffffffffu, best_index, offset);
        take_better(best, best_index, other, other_index);
    }
    if (lane == 0) {
        best_values[warp] = best;
        best_indices[warp] = best_index;
    }
    __syncthreads();
    if (warp != 0) return;
    best = lane < kThreads / 32 ? best_values[lane] : -INFINITY;
    best_index = lane < kThreads / 32 ? best_indices[lane] : 0x7fffffff;
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, best, offset);
        const int other_index = __shfl_xor_sync(0xffffffffu, best_index, offset);
        take_better(best, best_index, other, other_index);
    }
    if (lane == 0) {
        partial_scores[(size_t)row * gridDim.x + blockIdx.x] = best;
        partial_indices[(size_t)row * gridDim.x + blockIdx.x] = best_index;
    }
}

// One warp per row.
__global__ void control_pick_kernel(const float* __restrict__ partial_scores, const int* __restrict__ partial_indices, int slices,
                                    int* __restrict__ out, int* history, const Controls c, int note, const int* __restrict__ flag_a,
                                    const int* __restrict__ flag_b) {
    pdl_trigger();
    pdl_wait();
    const int row = blockIdx.x, lane = threadIdx.x;
    float best = -INFINITY;
    int best_index = 0x7fffffff;
    for (int s = lane; s < slices; s += 32)
        take_better(best, best_index, partial_scores[(size_t)row * slices + s], partial_indices[(size_t)row * slices + s]);
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, best, offset);
        const int other_index = __shfl_xor_sync(0xffffffffu, best_index, offset);
        take_better(best, best_index, other, other_index);
    }
    if (lane != 0) return;
    const int token = best == -INFINITY ? -1 : best_index;
    out[row] = token;
    if (note && token >= 0) {
        const int at = c.history_rows[row], place = c.lengths[row];
        if (at >= 0 && at < c.histories && place >= 0 && place < c.capacity) history[(size_t)at * c.capacity + place] = token;
    }
    if (row == 0) leave_flags(out + gridDim.x, flag_a, flag_b);
}

// Tokens per slice: whole waves of blocks (four share an SM), slices of at most kMostSlice and, where rows are few, of no fewer than
// 2048 tokens.
int slice_of(int rows, int vocab) {
    const long long wave = 4LL * llm_sm_count();
    int per_slice = kMostSlice;
    for (int waves = 1; waves <= 64; ++waves) {
        const long long slices = wave * waves / rows;
        if (slices < 1) continue;
        const long long size = (vocab + slices - 1) / slices;
        if (size <= kMostSlice) {
            per_slice = size < 2048 ? 2048 : (int)size;
            break;
        }
    }
    return (per_slice + 31) / 32 * 32;
}

int refuse_controls(const char* what, const Controls& c, int rows, int vocab) {
    if (rows < 0 || rows > 65535 || vocab < 1) {
        llm_set_error("%s: %d rows of %d logits (1 to 65535 rows per launch)", what, rows, vocab);
        return LLM_REFUSED;
    }
    if (c.masks != nullptr && c.mask_words < (vocab + 31) / 32) {
        llm_set_error("%s: masks of %d words do not cover %d tokens", what, c.mask_words, vocab);
        return LLM_REFUSED;
    }
    return LLM_OK;
}

template <bool SAMPLE>
int launch_control(const float* logits, float* out, const Controls& c, int rows, int vocab, int per_slice, const float* temperatures,
                   const uint64_t* seeds, const int* steps, float* scores, int* indices, cudaStream_t stream) {
    const int slices = (vocab + per_slice - 1) / per_slice;
    const size_t shared = (size_t)(per_slice < vocab ? per_slice : vocab) * sizeof(uint32_t);
    if (int status = llm_raise_shared_limit((const void*)control_kernel<SAMPLE>, shared, "control_logits", true)) return status;
    llm_launch(control_kernel<SAMPLE>, dim3(slices, rows), kThreads, shared, stream, logits, out, c, vocab, per_slice, temperatures, seeds,
               steps, scores, indices);
    return llm_check_launch("control_logits");
}

}  // namespace

// How many slices a row is scanned in: the scratch of llm_control_sample holds that many scores and tokens per row.
LLM_EXPORT int llm_control_slices(int rows, int vocab) {
    if (rows < 1 || vocab < 1) return 1;
    const int per_slice = slice_of(rows, vocab);
    return (vocab + per_slice - 1) / per_slice;
}

LLM_EXPORT int llm_control_logits(const float* logits, float* out, int rows, int vocab, const LlmControls* controls, cudaStream_t stream) {
    if (int status = refuse_controls("control_logits", *controls, rows, vocab)) return status;
    if (rows == 0) return LLM_OK;
    return launch_control<false>(logits, out, *controls, rows, vocab, slice_of(rows, vocab), nullptr, nullptr, nullptr, nullptr, nullptr, stream);
}

// `history`: where tokens are noted, or null.  `scores` / `indices`: [rows][llm_control_slices].
LLM_EXPORT int llm_control_sample(const float* logits, const float* temperatures, const uint64_t* seeds, const int* steps, int* out, int rows,
                                  int vocab, const LlmControls* controls, int* history, float* scores, int* indices, const int* flag_a,
                                  const int* flag_b, cudaStream_t stream) {
    if (int status = refuse_controls("sample", *controls, rows, vocab)) return status;
    if (rows == 0) return LLM_OK;
    const int per_slice = slice_of(rows, vocab);
    if (int status = launch_control<true>(logits, nullptr, *controls, rows, vocab, per_slice, temperatures, seeds, steps, scores, indices, stream))
        return status;
    llm_launch(control_pick_kernel, rows, 32, 0, stream, scores, indices, (vocab + per_slice - 1) / per_slice, out, history, *controls,
               (int)(history != nullptr), flag_a, flag_b);
    return llm_check_launch("control_pick");
}
