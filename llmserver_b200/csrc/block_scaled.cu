// Rows and matrices in 8 bits (e4m3) with a 32-bit scale for each block: 1 x 128 for a row's groups, 128 x 128 for a matrix.
//
//   scale = 2^e, e the least (not below -126) for which max |x| of the block <= 448 * 2^e;   value = e4m3(x / scale)
//
// A power of two as scale makes the quotient exact, so every number is rounded once, to the nearest of e4m3's (ties to even), and
// since e4m3 is itself a floating format nothing is lost against a scale of max / 448 but half a binade or so below its normal range.  A block
// that holds an infinity or a NaN (e4m3 has no infinity) becomes NaN whole, values and scale.
//
// What bounds it: reading x and writing a byte for each number.  Half a warp takes 128 numbers of a row, eight a lane, as they lie in
// memory; what a thread needs of x is asked for all at once, before anything is looked at (a branch around each load, for rows that begin
// anywhere, made the loads wait for one another: 24576 x 4096 bfloat16 in blocks of 128 x 128 took 218 us and not 45, 6.7 TB/s).  Rows that do not begin at
// multiples of 16 bytes are read number by number, by kernels of their own.
#include "block_scaled.cuh"

#include <string.h>

namespace {

using namespace block_scaled;

constexpr int kThreads = 256;

// Eight numbers of a row as they lie in memory.
template <typename T>
struct Eight {
    uint4 words[sizeof(T) / 2];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i) words[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void ask(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i) words[i] = *(reinterpret_cast<const uint4*>(p) + i);
    }
    __device__ __forceinline__ void ask_singly(const T* row, int first, int inner) {      // those that exist, from wherever the row begins
        T each[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) Num<T>::store(&each[c], first + c < inner ? Num<T>::load(row + first + c) : 0.0f);
        memcpy(words, each, sizeof(each));
    }
    // The bits of the largest magnitude: as whole numbers magnitudes are ordered, NaN above infinity above all others.
    __device__ __forceinline__ uint32_t largest() const {
        if constexpr (sizeof(T) == 2) {
            const uint32_t sign = 0x7fff7fffu;
            const uint32_t both = __vmaxu2(__vmaxu2(words[0].x & sign, words[0].y & sign), __vmaxu2(words[0].z & sign, words[0].w & sign));
            return max(both & 0xffff0000u, both << 16);
        } else {
            uint32_t found = 0;
#pragma unroll
            for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
                found = max(max(found, max(words[i].x & 0x7fffffffu, words[i].y & 0x7fffffffu)), max(words[i].z & 0x7fffffffu, words[i].w & 0x7fffffffu));
            return found;
        }
    }
    __device__ __forceinline__ uint2 rounded(float inverse) const {
        float v[8];
        load8<T>(reinterpret_cast<const T*>(words), v);
        return make_uint2(four_of(v[0], v[1], v[2], v[3], inverse), four_of(v[4], v[5], v[6], v[7], inverse));
    }
};

__device__ __forceinline__ uint32_t half_warp_max(uint32_t v) {
#pragma unroll
    for (int offset = 8; offset > 0; offset >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, offset));
    return v;
}

// The successor may read what does not depend on these kernels as soon as it runs, so it is let in only when everything in front of them is
// complete.  The rows of `out` begin at multiples of 16 bytes; bytes behind a row's end, up to there, may be written.
//
// Rows that are whole groups long: the groups lie one after the other, and half a warp takes AT_ONCE of them at a time.
template <typename T, int AT_ONCE>
__global__ void __launch_bounds__(kThreads) quantize_groups_kernel(const T* __restrict__ x, unsigned char* __restrict__ out, float* __restrict__ scales,
                                                                   long long total) {
    pdl_wait();
    pdl_trigger();
    const int place = threadIdx.x & 15;
    const long long halves = (long long)gridDim.x * (kThreads / 16);
    // (a warp's two halves run side by side to the end: the groups that one of them lacks are left out)
    for (long long g0 = ((long long)blockIdx.x * kThreads + (threadIdx.x & ~31)) >> 4; g0 < total; g0 += halves * AT_ONCE) {
        const long long first = g0 + ((threadIdx.x >> 4) & 1);
        Eight<T> numbers[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const long long g = first + i * halves;
            if (g < total) numbers[i].ask(x + g * kBlock + 8 * place);
            else numbers[i].clear();
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const long long g = first + i * halves;
            const Rounding r = rounding_of(half_warp_max(numbers[i].largest()));
            if (g < total) {
                *reinterpret_cast<uint2*>(out + g * kBlock + 8 * place) = numbers[i].rounded(r.inverse);
                if (place == 0) scales[g] = r.scale;
            }
        }
    }
}

// Any other rows, AT_ONCE groups at a time (WHOLE: they begin at multiples of 16 bytes).  A half warp's next group is step_rows and step_groups further on:
// found by divisions of 64 bits and one at a time, 16384 rows of 6000 bfloat16 took 68 us and not 61.
template <typename T, bool WHOLE, int AT_ONCE>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const T* __restrict__ x, unsigned char* __restrict__ out, float* __restrict__ scales,
                                                                 int rows, int inner, int groups, long long pitch, int step_rows, int step_groups) {
    pdl_wait();
    pdl_trigger();
    const int place = threadIdx.x & 15;
    const long long half = ((long long)blockIdx.x * kThreads + threadIdx.x) >> 4;
    long long row = half / groups;
    int group = (int)(half - row * groups);
    // (a warp's halves go on together: as long as one of them has a group left)
    while (__any_sync(0xffffffffu, row < rows)) {
        Eight<T> numbers[AT_ONCE];
        long long rows_of[AT_ONCE];
        int groups_of[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            rows_of[i] = row, groups_of[i] = group;
            const int first = group * kBlock + 8 * place;
            if (WHOLE && row < rows && first + 8 <= inner) numbers[i].ask(x + (size_t)row * inner + first);
            else numbers[i].clear();
            if (!WHOLE || first + 8 > inner)
                if (row < rows) numbers[i].ask_singly(x + (size_t)row * inner, first, inner);
            row += step_rows, group += step_groups;
            if (group >= groups) group -= groups, ++row;
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const Rounding r = rounding_of(half_warp_max(numbers[i].largest()));
            if (rows_of[i] >= rows) continue;
            const int first = groups_of[i] * kBlock + 8 * place;
            if (first < inner) *reinterpret_cast<uint2*>(out + (size_t)rows_of[i] * pitch + first) = numbers[i].rounded(r.inverse);
            if (place == 0) scales[(size_t)rows_of[i] * groups + groups_of[i]] = r.scale;
        }
    }
}

// Block (column of blocks, row of blocks); a warp takes 16 of its 128 rows, two at a time.  WHOLE: rows begin at multiples of 16 bytes.
template <typename T, bool WHOLE>
__global__ void __launch_bounds__(kThreads) quantize_matrix_kernel(const T* __restrict__ x, unsigned char* __restrict__ out, float* __restrict__ scales,
                                                                   int rows, int inner, int groups, long long pitch) {
    pdl_wait();
    pdl_trigger();
    constexpr int kTurns = kBlock / (kThreads / 16);
    __shared__ uint32_t parts[kThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int first = blockIdx.x * kBlock + 8 * (lane & 15);
    const long long row0 = (long long)blockIdx.y * kBlock + warp * 2 * kTurns + (lane >> 4);
    Eight<T> numbers[kTurns];
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
        const long long row = row0 + 2 * i;
        if (WHOLE && row < rows && first + 8 <= inner) numbers[i].ask(x + (size_t)row * inner + first);
        else numbers[i].clear();
        if (!WHOLE || first + 8 > inner)
            if (row < rows) numbers[i].ask_singly(x + (size_t)row * inner, first, inner);
    }
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < kTurns; ++i) largest = max(largest, numbers[i].largest());
    largest = __reduce_max_sync(0xffffffffu, largest);
    if (lane == 0) parts[warp] = largest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) largest = max(largest, parts[w]);
    const Rounding r = rounding_of(largest);
    if (first < inner)
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            const long long row = row0 + 2 * i;
            if (row < rows) *reinterpret_cast<uint2*>(out + (size_t)row * pitch + first) = numbers[i].rounded(r.inverse);
        }
    if (threadIdx.x == 0) scales[(size_t)blockIdx.y * groups + blockIdx.x] = r.scale;
}

}  // namespace

// x [rows, inner] (float or bfloat16, contiguous) -> out [rows, pitch] bytes and scales [ceil(rows / block_rows), ceil(inner / 128)];
// pitch a multiple of 16 and at least inner, out 16-byte aligned.
LLM_EXPORT int llm_quantize_blocks(const void* x, int dtype, void* out, float* scales, int rows, int inner, long long pitch, int block_rows,
                                   cudaStream_t stream) {
    if (rows < 0 || rows > kMostAlong || inner < 1 || inner > kMostAlong || pitch < inner || pitch % 16 != 0 || !aligned16(out) || (block_rows != 1 && block_rows != kBlock)) {
        llm_set_error("quantize_blocks: %d rows of %d (pitch %lld) in blocks of %d rows", rows, inner, pitch, block_rows);
        return LLM_REFUSED;
    }
    if (rows == 0) return LLM_OK;
    const int groups = (inner + kBlock - 1) / kBlock, row_blocks = (rows + kBlock - 1) / kBlock;
    if (block_rows != 1 && row_blocks > 65535) {
        llm_set_error("quantize_blocks: at most %d rows, got %d", 65535 * kBlock, rows);
        return LLM_REFUSED;
    }
    LLM_DISPATCH_DTYPE(dtype, {
        const T* from = reinterpret_cast<const T*>(x);
        unsigned char* to = reinterpret_cast<unsigned char*>(out);
        // rows that begin at multiples of 16 bytes are read 16 bytes at a time
        const bool whole = inner % (16 / (int)sizeof(T)) == 0 && aligned16(x);
        if (block_rows == 1) {
            const long long total = (long long)rows * groups, blocks = (total + kThreads / 16 - 1) / (kThreads / 16);
            const long long room = 8LL * llm_sm_count();      // blocks that run at a time
            const dim3 grid((unsigned)(blocks < room ? blocks : room));
            const long long halves = (long long)grid.x * (kThreads / 16);
            if (whole && inner % kBlock == 0 && pitch == inner) {
                // several at once where there are as many for each half warp (500 rows of 4096 bfloat16: one 2.8 us, four 4.0; 4096 rows level)
                constexpr int kMost = sizeof(T) == 2 ? 4 : 2;
                llm_launch(total >= kMost * halves ? quantize_groups_kernel<T, kMost> : quantize_groups_kernel<T, 1>, grid, kThreads, 0, stream, from, to, scales, total);
            } else {
                const int step_rows = (int)(halves / groups), step_groups = (int)(halves % groups);
                // four at once where there are as many for each half warp (4096 rows of 1000: one 4.7 us, four 6.2); of 32-bit numbers one (8192 rows of 4100: one
                // 27.5 us, two 31.5), and of rows that are read number by number
                constexpr int kMost = sizeof(T) == 2 ? 4 : 1;
                const auto kernel = !whole ? quantize_rows_kernel<T, false, 1> : total >= kMost * halves ? quantize_rows_kernel<T, true, kMost> : quantize_rows_kernel<T, true, 1>;
                llm_launch(kernel, grid, kThreads, 0, stream, from, to, scales, rows, inner, groups, pitch, step_rows, step_groups);
            }
        } else {
            const dim3 grid(groups, row_blocks);
            if (whole) llm_launch(quantize_matrix_kernel<T, true>, grid, kThreads, 0, stream, from, to, scales, rows, inner, groups, pitch);
            else llm_launch(quantize_matrix_kernel<T, false>, grid, kThreads, 0, stream, from, to, scales, rows, inner, groups, pitch);
        }
    });
    return llm_check_launch("quantize_blocks");
}
