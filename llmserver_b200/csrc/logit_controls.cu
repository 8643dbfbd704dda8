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
// A block takes a slice of the vocabulary of one row and keeps a mark per token of the slice in shared memory: the times it stands in the
// answer, whether a bias is listed, whether it stands in the prompt; 16 bits where histories have room for fewer than 16384 tokens, so that
// one round of blocks holds large steps, else 32.  It walks the row's whole history and marks the tokens of its slice (integer atomics: their
// order does not matter); whoever marks a token first puts it on a list.  The tokens of the list, a few hundred of many thousand, are worked
// out by themselves, a token per thread.  The walk over the slice's logits then knows nothing of them: the form that returns logits
// writes theirs over what the walk wrote, and the one that samples looks at a mark only where a logit would win.  (With the marks looked up
// for every token the walk took twice as long, and worked out where it met them half as long again: it is bound by instructions.)  A list
// that overflows is not used: marks are then worked out in the walk.
//
// Sampling (sampling.cu's rule) takes the controlled logits as they are made, without writing them.  A second kernel picks the best
// slice of a row, gives -1 where a row's controls leave nothing to draw from, and writes the token behind the request's history: all histories have
// been read by then, whatever rows share one.
//
// What bounds it: the logits, read once (and written once by the form that returns them), and behind that the block's phases, which all blocks go
// through at the same time.  In a graph of such steps over logits from memory, 64 rows of 151936: returned 15.6 us without controls (5 TB/s) and 24.7 with
// histories of 4096 tokens, 50 biases and masks (29.4 call after call); drawn greedily 15.7 and 23.0, at temperatures 24.4 and 30.4 (31.1 call after call; 20
// instructions a token for its random word and the bound).  1 row and a short history: returned 3.7, drawn 7.7.
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

constexpr int kThreads = 512;
constexpr int kPerSm = 3;               // blocks that share an SM
constexpr int kAhead = 8;               // logits a thread asks for at a time
constexpr int kIdsAhead = 8;            // ids of the history
constexpr int kListed = 2048;           // marked tokens of a slice that are worked out by themselves
constexpr int kMostShared = 68 << 10;   // of a block
constexpr int kLeastSlice = 2048;       // tokens
constexpr int kListByScan = 8 * kThreads;      // slices of so many tokens and fewer are marked first and looked through for marks afterwards
constexpr int kMostVocab = 0x7ffe0000;  // places are counted in 32 bits, up to a slice and a lap behind the last
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
    // asked for together, looked at afterwards
    int at = -1, list = -1, mask = -1, length = 0, prompt = 0;
    RowControls r = {};
    r.repetition = 1.0f;
    if (c.history_rows != nullptr) at = c.history_rows[row];      // also where tokens are only noted there: a bad one is reported here, so that
                                                                   // the flag is settled when control_pick_kernel hands it on
    if (c.penalties != nullptr) {
        length = c.lengths[row];
        prompt = c.prompt_lengths[row];
        r.repetition = c.penalties[3 * (size_t)row];
        r.presence = c.penalties[3 * (size_t)row + 1];
        r.frequency = c.penalties[3 * (size_t)row + 2];
    }
    if (c.bias_rows != nullptr) list = c.bias_rows[row];
    if (c.mask_rows != nullptr) mask = c.mask_rows[row];
    if (list >= 0 && list < c.bias_lists) {
        const int first = min(max(c.bias_starts[list], 0), c.bias_entries);
        const int last = min(max(c.bias_starts[list + 1], first), c.bias_entries);
        r.bias_ids = c.bias_ids + first;
        r.bias_values = c.bias_values + first;
        r.biases = last - first;
    }
    // penalties that change nothing need no history
    if (at >= 0 && at < c.histories && (r.repetition != 1.0f || r.presence != 0.0f || r.frequency != 0.0f)) {
        r.history = c.history + (size_t)at * c.capacity;
        r.length = min(max(length, 0), c.capacity);
        r.prompt = min(max(prompt, 0), r.length);
    }
    if (mask >= 0 && mask < c.mask_count) r.mask = c.masks + (size_t)mask * c.mask_words;
    if (threadIdx.x == 0 && (at >= c.histories || list >= c.bias_lists || mask >= c.mask_count) && c.error_flag != nullptr) atomicExch(c.error_flag, kBadRow);
    r.marks = r.length > 0 || r.biases > 0;
    return r;
}

// The marks of a slice: SMALL of them share a word two by two.
template <bool SMALL>
struct Marks {
    static constexpr uint32_t kPrompt = SMALL ? 0x8000u : 0x80000000u, kBias = SMALL ? 0x4000u : 0x40000000u, kTimes = kBias - 1;
    uint32_t* words;
    static constexpr int kPerVector = SMALL ? 8 : 4;      // marks in 16 bytes
    static __host__ __device__ int vectors_of(int count) { return (count + kPerVector - 1) / kPerVector; }
    // Adds a flag or one more time; gives what the mark was.
    __device__ __forceinline__ uint32_t touch(uint32_t place, uint32_t flag) const {
        uint32_t* word = &words[SMALL ? place >> 1 : place];
        const int shift = SMALL ? 16 * (place & 1) : 0;
        return cut(flag ? atomicOr(word, flag << shift) : atomicAdd(word, 1u << shift), place);
    }
    static __device__ __forceinline__ uint32_t cut(uint32_t word, uint32_t place) { return SMALL ? word >> (16 * (place & 1)) & 0xffffu : word; }
    __device__ __forceinline__ uint32_t of(uint32_t place) const { return cut(words[SMALL ? place >> 1 : place], place); }
};

// Marks the tokens begin .. begin + count - 1 of the row's history and bias list and lists them, each once; more than kListed are counted, and
// only the first of them listed.  The words are zero.  Large slices list a token when it is marked first, small ones look through the
// marks at the end: an atomic that has to answer costs more than one that has not, and a small slice belongs to a step of few rows whose
// histories may be long.
template <bool SMALL>
__device__ __forceinline__ void mark_slice(const RowControls& r, Marks<SMALL> marks, uint16_t* listed, int* n_listed, int begin, int count) {
    const bool scan = count <= kListByScan;
    auto put = [&](int place) {
        const int at = atomicAdd(n_listed, 1);
        if (at < kListed) listed[at] = (uint16_t)place;
    };
    auto batch = [&](const int (&ids)[kIdsAhead], const uint32_t (&flags)[kIdsAhead]) {
        if (scan) {
#pragma unroll
            for (int a = 0; a < kIdsAhead; ++a)
                if ((uint32_t)ids[a] - (uint32_t)begin < (uint32_t)count) marks.touch((uint32_t)ids[a] - (uint32_t)begin, flags[a]);
            return;
        }
        uint32_t before[kIdsAhead];
#pragma unroll
        for (int a = 0; a < kIdsAhead; ++a)
            before[a] = (uint32_t)ids[a] - (uint32_t)begin < (uint32_t)count ? marks.touch((uint32_t)ids[a] - (uint32_t)begin, flags[a]) : 1;
#pragma unroll
        for (int a = 0; a < kIdsAhead; ++a)
            if (before[a] == 0) put(ids[a] - begin);
    };
    // (asked for one after the other, 24 thousand ids of a row took 26 us: every turn waits for memory)
    int next[kIdsAhead];
    auto ask = [&](const int* from, int first, int most) {
#pragma unroll
        for (int a = 0; a < kIdsAhead; ++a) next[a] = first + a * kThreads < most ? from[first + a * kThreads] : -1;      // (no token: begin is not negative)
    };
    ask(r.history, threadIdx.x, r.length);
    for (int first = threadIdx.x; first < r.length; first += kIdsAhead * kThreads) {
        int ids[kIdsAhead];
        uint32_t flags[kIdsAhead];
#pragma unroll
        for (int a = 0; a < kIdsAhead; ++a) {
            ids[a] = next[a];
            flags[a] = first + a * kThreads < r.prompt ? Marks<SMALL>::kPrompt : 0;
        }
        ask(r.history, first + kIdsAhead * kThreads, r.length);
        batch(ids, flags);
    }
    for (int first = threadIdx.x; first < r.biases; first += kIdsAhead * kThreads) {
        uint32_t flags[kIdsAhead];
        ask(r.bias_ids, first, r.biases);
#pragma unroll
        for (int a = 0; a < kIdsAhead; ++a) flags[a] = Marks<SMALL>::kBias;
        batch(next, flags);
    }
    if (scan) {
        __syncthreads();
        constexpr int kEach = Marks<SMALL>::kPerVector;
        for (int v = threadIdx.x; v < Marks<SMALL>::vectors_of(count); v += kThreads) {
            const uint4 words = reinterpret_cast<const uint4*>(marks.words)[v];
            if ((words.x | words.y | words.z | words.w) == 0) continue;
            const uint32_t word[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
            for (int e = 0; e < kEach; ++e)
                if (Marks<SMALL>::cut(word[SMALL ? e / 2 : e], e) != 0) put(v * kEach + e);
        }
    }
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
template <bool SMALL>
__device__ __forceinline__ float controlled(const RowControls& r, float logit, uint32_t mark, int token) {
    const uint32_t times = mark & Marks<SMALL>::kTimes;
    if (times != 0 || (mark & Marks<SMALL>::kPrompt)) logit = logit > 0.0f ? __fdiv_rn(logit, r.repetition) : __fmul_rn(logit, r.repetition);
    if (times != 0) logit = __fsub_rn(__fsub_rn(logit, __fmul_rn((float)times, r.frequency)), r.presence);
    if (mark & Marks<SMALL>::kBias) logit = __fadd_rn(logit, bias_of(r, token));
    return logit;
}

// A score in the order of whole numbers.
__device__ __forceinline__ int ordered(float v) {
    const int bits = __float_as_int(v);
    return bits >= 0 ? bits : bits ^ 0x7fffffff;
}
__device__ __forceinline__ float unordered(int v) { return __int_as_float(v >= 0 ? v : v ^ 0x7fffffff); }

// The draw of a row at a temperature.  Most tokens cannot win, and an upper bound of their score says so for a fifth of its price: with
// -log u >= 1 - u > v, the noise -log(-log u) is below -log v (v is 0 for the last of the words, and the bound infinite); the noise itself, with
// u at most 1 - 2^-24, is below 17.  The bound's own errors (the approximate logarithm's,
// the product's for the quotient) are below a thousandth and a millionth of the quotient, and a quotient that needs noise to reach a score is within 17 of
// it: the score is lowered by as much, once for many tokens.
struct Draw {
    float temperature, inverse;
    uint32_t word;      // of seed and step
    __device__ __forceinline__ void begin(float t, uint64_t seed, uint32_t step) {
        temperature = t;
        inverse = 1.0f / t;
        if (inverse > 3.4028234e38f) inverse = NAN;      // a temperature below the normal numbers: no bound
        word = mix32(mix32(mix32((uint32_t)seed ^ 0x9E3779B9u) ^ (uint32_t)(seed >> 32)) ^ step);
    }
    // What the bound of a token that may reach `best` is not below.
    static __device__ __forceinline__ float floor_of(float best) { return best - fmaf(fabsf(best) + 17.0f, 1e-6f, 1e-3f); }
    __device__ __forceinline__ bool may_reach(float logit, int token, float floor) const {
        const uint32_t k = mix32(word ^ (uint32_t)token) >> 9;
        const float v = 1.99999988f - __uint_as_float(0x3f800000u | k);      // exact: 1 - (k + 1) / 2^23, a little below 1 - u
        float log2_v;
        asm("lg2.approx.f32 %0, %1;" : "=f"(log2_v) : "f"(v));
        return !(fmaf(-0.69314718f, log2_v, logit * inverse) < floor);      // true where anything is a NaN
    }
    __device__ __forceinline__ float score(float logit, int token) const {
        const uint32_t k = mix32(word ^ (uint32_t)token) >> 9;
        const float u = ((float)k + 0.5f) * (1.0f / 8388608.0f);
        const float score = logit / temperature - logf(-logf(u));
        return score != score ? -INFINITY : score;      // a NaN never wins
    }
};

// SAMPLE: each block leaves its slice's best score and token in `partial`; else the controlled logits go to `out` (which may be
// `logits`).  FOUR: rows begin at multiples of 16 bytes, and a thread takes four tokens side by side.
template <bool SAMPLE, bool SMALL, bool FOUR>
__global__ void __launch_bounds__(kThreads, kPerSm) control_kernel(const float* logits, float* out, const Controls c, int vocab, int per_slice,
                                                                   const float* __restrict__ temperatures, const uint64_t* __restrict__ seeds,
                                                                   const int* __restrict__ steps, float* __restrict__ partial_scores,
                                                                   int* __restrict__ partial_indices) {
    pdl_trigger();
    pdl_wait();
    extern __shared__ uint4 slice_vectors[];      // the marks, then the slice of the mask
    __shared__ float best_values[kThreads / 32];
    __shared__ int best_indices[kThreads / 32];
    __shared__ uint16_t listed[kListed];
    __shared__ int n_listed;
    __shared__ int bar;      // SAMPLE: a score that some token of the slice reaches; raised as the walk goes on (left at the first lap's, 64 rows took 32 us and not 30)
    const int row = blockIdx.y;
    const int begin = blockIdx.x * per_slice, end = min(vocab, begin + per_slice), count = end - begin;
    const float* src = logits + (size_t)row * vocab;
    float* dst = out + (size_t)row * vocab;
    const RowControls r = controls_of(c, row);
    const Marks<SMALL> marks{reinterpret_cast<uint32_t*>(slice_vectors)};
    uint32_t* allowed = reinterpret_cast<uint32_t*>(slice_vectors + Marks<SMALL>::vectors_of(per_slice));
    if (r.mask != nullptr)
        for (int i = threadIdx.x; i < (count + 31) / 32; i += kThreads) allowed[i] = (uint32_t)r.mask[begin / 32 + i];      // (slices begin at multiples of 32)
    if (threadIdx.x == 0) {
        n_listed = 0;
        bar = ordered(-INFINITY);
    }
    if (r.marks) {
        for (int i = threadIdx.x; i < Marks<SMALL>::vectors_of(count); i += kThreads) slice_vectors[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        mark_slice<SMALL>(r, marks, listed, &n_listed, begin, count);
    }
    Draw draw = {};
    if (SAMPLE && temperatures != nullptr && temperatures[row] > 0.0f) draw.begin(temperatures[row], seeds[row], (uint32_t)steps[row]);
    const bool warm = draw.temperature > 0.0f;
    __syncthreads();

    const bool apart = r.marks && n_listed <= kListed, inside = r.marks && !apart;      // where what is marked is worked out
    float best = -INFINITY;
    int best_index = 0x7fffffff;
    constexpr int kEach = FOUR ? 4 : 1, kGroups = kAhead / kEach;      // tokens that lie side by side, groups of them
    for (int lap = 0; lap < count; lap += kAhead * kThreads) {
        auto place = [&](int a) { return lap + (a / kEach * kThreads + (int)threadIdx.x) * kEach + a % kEach; };
        auto token = [&](int a) { return begin + place(a); };
        float now[kAhead];
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int i = token(g * kEach);
            if constexpr (FOUR) {
                const float4 v = i < end ? *reinterpret_cast<const float4*>(src + i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                now[4 * g] = v.x, now[4 * g + 1] = v.y, now[4 * g + 2] = v.z, now[4 * g + 3] = v.w;
            } else {
                now[g] = i < end ? src[i] : -INFINITY;
            }
        }
        if (inside) {
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                const uint32_t mark = token(a) < end ? marks.of(place(a)) : 0;
                if (mark != 0) now[a] = controlled<SMALL>(r, now[a], mark, token(a));
            }
        }
        if (r.mask != nullptr) {
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const uint32_t bits = token(g * kEach) < end ? allowed[place(g * kEach) >> 5] >> (place(g * kEach) & 31) : 0;
#pragma unroll
                for (int e = 0; e < kEach; ++e) now[g * kEach + e] = bits >> e & 1u ? now[g * kEach + e] : -INFINITY;
            }
        }
        if (!SAMPLE) {
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const int i = token(g * kEach);
                if (i >= end) break;
                if constexpr (FOUR) *reinterpret_cast<float4*>(dst + i) = make_float4(now[4 * g], now[4 * g + 1], now[4 * g + 2], now[4 * g + 3]);
                else dst[i] = now[g];
            }
            continue;
        }
        const float least = unordered(bar);      // (the first lap's is below everything)
        auto take = [&](int a) {
            if (apart && marks.of(place(a)) != 0) return;      // has been dealt with
            take_better(best, best_index, warm ? draw.score(now[a], token(a)) : now[a], token(a));
        };
        if (warm) {
            int from = 0;
            if (lap == 0) {
                // the first of each thread's logits set the bar for the others
                if (now[0] > -INFINITY) take(0);
                const int high = __reduce_max_sync(0xffffffffu, ordered(best));
                if ((threadIdx.x & 31) == 0) atomicMax(&bar, high);
                __syncthreads();
                from = 1;
            }
            const float set = unordered(bar), floor = Draw::floor_of(fmaxf(best, set));
#pragma unroll
            for (int a = 0; a < kAhead; ++a)
                if (a >= from && now[a] > -INFINITY && draw.may_reach(now[a], token(a), floor)) take(a);
            if (best > set) atomicMax(&bar, ordered(best));      // for everybody's next laps
        } else {
            float high = now[0];
#pragma unroll
            for (int a = 1; a < kAhead; ++a) high = fmaxf(high, now[a]);      // (a NaN is not)
            // equal scores go to the lower token, whoever holds it
            if (high >= fmaxf(best, least) && high > -INFINITY) {
#pragma unroll
                for (int a = 0; a < kAhead; ++a)
                    if (now[a] >= best && now[a] > -INFINITY) take(a);
            }
            if (lap == 0) {
                const int highest = __reduce_max_sync(0xffffffffu, ordered(best));
                if ((threadIdx.x & 31) == 0) atomicMax(&bar, highest);
                __syncthreads();
            }
        }
    }
    if (apart) {
        // Behind the walk these logits come from L2 (in front of it they waited for memory behind the walks of other blocks).  Where the result goes
        // to the logits' own place the walk has written each back as it was, or -inf where the mask bans it, which it then stays.
        if (!SAMPLE) __syncthreads();
#pragma unroll
        for (int k = 0; k < kListed / kThreads; ++k) {
            const int e = threadIdx.x + k * kThreads;
            if (e >= n_listed) break;
            const int place = listed[e], i = begin + place;
            float logit = controlled<SMALL>(r, src[i], marks.of(place), i);
            if (r.mask != nullptr && (allowed[place >> 5] >> (i & 31) & 1u) == 0) logit = -INFINITY;
            if (!SAMPLE) dst[i] = logit;
            else if (logit > -INFINITY) take_better(best, best_index, warm ? draw.score(logit, i) : logit, i);
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

// Whether anything is said about a row (an index that names nothing says nothing).
__device__ __forceinline__ bool any_controls(const Controls& c, int row) {
    auto names = [&](const int* rows, int count) { return rows != nullptr && rows[row] >= 0 && rows[row] < count; };
    return (c.penalties != nullptr && names(c.history_rows, c.histories)) || names(c.bias_rows, c.bias_lists) || names(c.mask_rows, c.mask_count);
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
    int token = best_index;
    if (best == -INFINITY) {      // a quotient may be too large for 32 bits: the token is then still one that is left
        if (!any_controls(c, row)) token = 0;      // as sampling.cu has it, whoever shares the step
        else if (best_index == 0x7fffffff) token = -1;
    }
    if (note) {
        const int at = c.history_rows[row], place = c.lengths[row];
        // of rows with one place the last has it
        bool last = true;
        for (int other = row + 1 + lane; other < (int)gridDim.x; other += 32)
            if (c.history_rows[other] == at && c.lengths[other] == place) last = false;
        last = __all_sync(0xffffffffu, last);
        if (lane == 0 && last && token >= 0 && at >= 0 && at < c.histories && place >= 0 && place < c.capacity)
            history[(size_t)at * c.capacity + place] = token;
    }
    if (lane != 0) return;
    out[row] = token;
    if (row == 0) leave_flags(out + gridDim.x, flag_a, flag_b);
}

// Whether 16 bits hold every count, and the bytes of shared memory that a slice needs.
bool small_marks(const Controls& c) { return c.capacity <= (int)Marks<true>::kTimes; }
size_t shared_of(int places, bool small) {
    return (size_t)(small ? Marks<true>::vectors_of(places) : Marks<false>::vectors_of(places)) * sizeof(uint4) + places / 32 * sizeof(uint32_t);
}

// Tokens per slice, a multiple of 32: whole rounds of blocks, as few as the shared memory lets, and no fewer than kLeastSlice tokens.
int slice_of(int rows, int vocab, bool small) {
    const long long round = (long long)kPerSm * llm_sm_count();
    for (long long rounds = 1;; ++rounds) {
        const long long slices = round * rounds / rows;
        if (slices < 1) continue;
        const long long each = (vocab + slices - 1) / slices;
        if (each <= kLeastSlice) return kLeastSlice;
        const long long size = (each + 31) / 32 * 32;
        if (size <= 1 << 16 && shared_of((int)size, small) <= (size_t)kMostShared) return (int)size;
    }
}
int refuse_controls(const char* what, const Controls& c, int rows, int vocab) {
    if (rows < 0 || rows > 65535 || vocab < 1 || vocab > kMostVocab) {
        llm_set_error("%s: %d rows of %d logits (1 to 65535 rows per launch, of 1 to %d)", what, rows, vocab, kMostVocab);
        return LLM_REFUSED;
    }
    if (c.masks != nullptr && c.mask_words < (vocab + 31) / 32) {
        llm_set_error("%s: masks of %d words do not cover %d tokens", what, c.mask_words, vocab);
        return LLM_REFUSED;
    }
    return LLM_OK;
}

template <bool SAMPLE, bool SMALL, bool FOUR>
int launch_form(const float* logits, float* out, const Controls& c, int rows, int vocab, int per_slice, const float* temperatures,
                const uint64_t* seeds, const int* steps, float* scores, int* indices, cudaStream_t stream) {
    if (int status = llm_raise_shared_limit((const void*)control_kernel<SAMPLE, SMALL, FOUR>, kMostShared, "control_logits", true)) return status;
    llm_launch(control_kernel<SAMPLE, SMALL, FOUR>, dim3((unsigned)(((long long)vocab + per_slice - 1) / per_slice), rows), kThreads,
               shared_of(per_slice, SMALL), stream, logits, out, c, vocab, per_slice, temperatures, seeds, steps, scores, indices);
    return llm_check_launch("control_logits");
}

template <bool SAMPLE>
int launch_control(const float* logits, float* out, const Controls& c, int rows, int vocab, const float* temperatures,
                   const uint64_t* seeds, const int* steps, float* scores, int* indices, cudaStream_t stream) {
    const bool small = small_marks(c), four = vocab % 4 == 0 && aligned16(logits) && (SAMPLE || aligned16(out));
    const auto form = small ? (four ? launch_form<SAMPLE, true, true> : launch_form<SAMPLE, true, false>)
                            : (four ? launch_form<SAMPLE, false, true> : launch_form<SAMPLE, false, false>);
    return form(logits, out, c, rows, vocab, slice_of(rows, vocab, small), temperatures, seeds, steps, scores, indices, stream);
}

}  // namespace

LLM_EXPORT int llm_control_logits(const float* logits, float* out, int rows, int vocab, const LlmControls* controls, cudaStream_t stream) {
    if (int status = refuse_controls("control_logits", *controls, rows, vocab)) return status;
    if (rows == 0) return LLM_OK;
    return launch_control<false>(logits, out, *controls, rows, vocab, nullptr, nullptr, nullptr, nullptr, nullptr, stream);
}

// `history`: where tokens are noted, or null.  `scores` / `indices`: a number each for every slice of every row, of which there are at most
// ceil(vocab / 2048).
LLM_EXPORT int llm_control_sample(const float* logits, const float* temperatures, const uint64_t* seeds, const int* steps, int* out, int rows,
                                  int vocab, const LlmControls* controls, int* history, float* scores, int* indices, const int* flag_a,
                                  const int* flag_b, cudaStream_t stream) {
    if (int status = refuse_controls("sample", *controls, rows, vocab)) return status;
    if (rows == 0) return LLM_OK;
    const int per_slice = slice_of(rows, vocab, small_marks(*controls));
    if (int status = launch_control<true>(logits, nullptr, *controls, rows, vocab, temperatures, seeds, steps, scores, indices, stream)) return status;
    llm_launch(control_pick_kernel, rows, 32, 0, stream, scores, indices, (int)(((long long)vocab + per_slice - 1) / per_slice), out, history, *controls, (int)(history != nullptr), flag_a, flag_b);
    return llm_check_launch("control_pick");
}
