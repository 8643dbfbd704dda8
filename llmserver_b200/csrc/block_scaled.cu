// Rows and matrices in 8 bits (e4m3) with a 32-bit scale for each block: 1 x 128 for a row's groups, 128 x 128 for a matrix.
//
//   scale = 2^e, e the least (not below -126) for which max |x| of the block <= 448 * 2^e;   value = e4m3(x / scale)
//
// A power of two as scale makes the quotient exact, so every number is rounded once, to the nearest of e4m3's (ties to even), and
// since e4m3 is itself a floating format nothing is lost against a scale of max / 448 but half a binade or so below its normal range.  A block
// that holds an infinity or a NaN (e4m3 has no infinity) becomes NaN whole, values and scale.
//
// What bounds it: reading x and writing a byte for each number.  Rows: a warp takes groups of 128 one after the other, four numbers a
// lane.  Matrices: a block of threads keeps the 128 x 128 numbers in registers between the maximum and the rounding.
#include "block_scaled.cuh"

namespace {

using namespace block_scaled;

constexpr int kGroup = kBlock;
constexpr int kThreads = 256;

__device__ __forceinline__ uint32_t warp_max_bits(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

// Numbers 4 i .. 4 i + 3 of a row (those that exist; zeros behind them).  `whole`: the row begins where 4 numbers can be read at once.
template <typename T>
__device__ __forceinline__ void load4(const T* row, int first, int inner, bool whole, float (&v)[4]) {
    if (whole && first + 4 <= inner) {
        if constexpr (sizeof(T) == 4) {
            const float4 raw = *reinterpret_cast<const float4*>(row + first);
            v[0] = raw.x, v[1] = raw.y, v[2] = raw.z, v[3] = raw.w;
        } else {
            const uint2 raw = *reinterpret_cast<const uint2*>(row + first);
            const float2 low = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.x));
            const float2 high = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.y));
            v[0] = low.x, v[1] = low.y, v[2] = high.x, v[3] = high.y;
        }
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = first + c < inner ? Num<T>::load(row + first + c) : 0.0f;
    }
}

// The rows of `out` begin at multiples of 16 bytes; bytes behind a row's end (up to there) may be written.
template <typename T>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const T* __restrict__ x, unsigned char* __restrict__ out, float* __restrict__ scales,
                                                                 int rows, int inner, int groups, long long pitch, int whole) {
    // The successor may read what does not depend on this kernel as soon as it runs, so it is let in only when everything in front of
    // this kernel is complete.
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const long long warp = ((long long)blockIdx.x * kThreads + threadIdx.x) >> 5, warps = (long long)gridDim.x * (kThreads / 32);
    const long long total = (long long)rows * groups;
    for (long long g = warp; g < total; g += warps) {
        const int row = (int)(g / groups), group = (int)(g - (long long)row * groups);
        const int first = group * kGroup + 4 * lane;
        float v[4];
        load4(x + (size_t)row * inner, first, inner, whole != 0, v);
        const uint32_t largest = warp_max_bits(max(max(magnitude(v[0]), magnitude(v[1])), max(magnitude(v[2]), magnitude(v[3]))));
        const Rounding r = rounding_of(largest);
        if (first < inner) *reinterpret_cast<uint32_t*>(out + (size_t)row * pitch + first) = four_of(v[0], v[1], v[2], v[3], r.inverse);
        if (lane == 0) scales[g] = r.scale;
    }
}

// Block (column of blocks, row of blocks); a warp takes 16 of its 128 rows.
template <typename T>
__global__ void __launch_bounds__(kThreads) quantize_matrix_kernel(const T* __restrict__ x, unsigned char* __restrict__ out, float* __restrict__ scales,
                                                                   int rows, int inner, int groups, long long pitch, int whole) {
    pdl_wait();
    pdl_trigger();
    constexpr int kRows = kGroup / (kThreads / 32);
    __shared__ uint32_t parts[kThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int first = blockIdx.x * kGroup + 4 * lane;
    const long long row0 = (long long)blockIdx.y * kGroup + warp * kRows;
    float v[kRows][4];
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
#pragma unroll
        for (int c = 0; c < 4; ++c) v[i][c] = 0.0f;
        if (row0 + i < rows) load4(x + (size_t)(row0 + i) * inner, first, inner, whole != 0, v[i]);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) largest = max(largest, magnitude(v[i][c]));
    largest = warp_max_bits(largest);
    if (lane == 0) parts[warp] = largest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) largest = max(largest, parts[w]);
    const Rounding r = rounding_of(largest);
    if (first < inner)
#pragma unroll
        for (int i = 0; i < kRows; ++i)
            if (row0 + i < rows) *reinterpret_cast<uint32_t*>(out + (size_t)(row0 + i) * pitch + first) = four_of(v[i][0], v[i][1], v[i][2], v[i][3], r.inverse);
    if (threadIdx.x == 0) scales[(size_t)blockIdx.y * groups + blockIdx.x] = r.scale;
}

}  // namespace

// x [rows, inner] (float or bfloat16, contiguous) -> out [rows, pitch] bytes and scales [ceil(rows / block_rows), ceil(inner / 128)];
// pitch a multiple of 16 and at least inner, out 16-byte aligned.
LLM_EXPORT int llm_quantize_blocks(const void* x, int dtype, void* out, float* scales, int rows, int inner, long long pitch, int block_rows,
                                   cudaStream_t stream) {
    if (rows < 0 || inner < 1 || pitch < inner || pitch % 16 != 0 || !aligned16(out) || (block_rows != 1 && block_rows != kGroup)) {
        llm_set_error("quantize_blocks: %d rows of %d (pitch %lld) in blocks of %d rows", rows, inner, pitch, block_rows);
        return LLM_REFUSED;
    }
    if (rows == 0) return LLM_OK;
    const int groups = (inner + kGroup - 1) / kGroup, row_blocks = (rows + kGroup - 1) / kGroup;
    if (block_rows != 1 && row_blocks > 65535) {
        llm_set_error("quantize_blocks: at most %d rows, got %d", 65535 * kGroup, rows);
        return LLM_REFUSED;
    }
    LLM_DISPATCH_DTYPE(dtype, {
        // four numbers of every row can be read at once: the rows begin at multiples of four numbers
        const int whole = inner % 4 == 0 && reinterpret_cast<uintptr_t>(x) % (4 * sizeof(T)) == 0;
        if (block_rows == 1) {
            const long long warps = (long long)rows * groups, blocks = (warps + kThreads / 32 - 1) / (kThreads / 32);
            const long long room = 8LL * llm_sm_count();      // blocks that run at a time
            llm_launch(quantize_rows_kernel<T>, dim3((unsigned)(blocks < room ? blocks : room)), kThreads, 0, stream,
                       reinterpret_cast<const T*>(x), reinterpret_cast<unsigned char*>(out), scales, rows, inner, groups, pitch, whole);
        } else {
            llm_launch(quantize_matrix_kernel<T>, dim3(groups, row_blocks), kThreads, 0, stream, reinterpret_cast<const T*>(x),
                       reinterpret_cast<unsigned char*>(out), scales, rows, inner, groups, pitch, whole);
        }
    });
    return llm_check_launch("quantize_blocks");
}
