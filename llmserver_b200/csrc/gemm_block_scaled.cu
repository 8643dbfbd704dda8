// y[m, n] = sum over blocks b of 128 along k:  xs[m, b] * ws[n / 128, b] * sum_{k in b} xq[m, k] wq[n, k]
//
// Both operands are e4m3 with 32-bit scales, one for each row and 128 columns of x, one for each 128 x 128 of W.  The products of a
// block are summed by tcgen05.mma (kind::f8f6f4: exact products, 32-bit sums) into tensor memory; from there they are read back,
// multiplied with the block's two scales and added up in registers, 32-bit as well: the scales are any 32-bit numbers, so blocks
// cannot be added before they are scaled.
//
// For up to 64 tokens (more, and from 33 on large matrices: gemm_block_scaled_many.cu).  The roles of the operands are swapped for the hardware, as in gemm_tcgen05.cu:
// 128 rows of W are the MMA's M, the tokens (16, 32 or 64) its N, so that a product of few tokens streams W and wastes nothing on rows
// that do not exist.  A stage of the ring is one block of 128 along k: 16 KiB of W and 2 to 8 KiB of x, which are one swizzle atom wide.  The MMAs of a block go to one of several
// buffers of tensor memory, so that they run ahead of the warps that scale and add.
//
// What bounds it: W's bytes.  8 rows by 151936 x 4096 98 us, 6.4 TB/s, 0.97 of a copy; 1 row by 24576 x 4096 20.3 us with the kernel that
// brings the row to 8 bits, 5.0 TB/s in all, 6.1 once the rings are full.
//
// Where tiles do not come out even on the SMs, k is split over a cluster and the parts are added through distributed shared memory in
// the order of k (see split_of).
//
// Roles: warp 0 copies (TMA), warp 1 issues the MMAs, warp 2 leaves each unit's scales (a token's times W's) in shared
// memory, warp 3 holds the tensor memory, and the other four scale and add, a row of W per thread.  All waits are
// bounded: one that runs out sets error code 2, every role leaves its loop, and the block still frees its tensor memory and meets its
// cluster.
//
// k need not be a multiple of 128 nor n of 128 nor m of anything: what lies outside is read as zeros (TMA) and not written.
#include "block_scaled_mma.cuh"

namespace {

using namespace block_scaled;

constexpr int kRows = 128;            // rows of W per tile (UMMA M)
constexpr int kAdders = 4;            // warps that scale and add
constexpr int kThreads = 128 + 32 * kAdders;
constexpr int kPerSm = 2;             // blocks that share an SM: one streams while the other begins or ends
constexpr uint32_t kRingBytes = 96 << 10;
constexpr int kMaxStages = 6;
constexpr int kMaxSplit = 8;
constexpr int kScaleSlots = 8;        // units whose scales wait to be used
constexpr int kScalesAhead = 4;       // and those on their way from memory
constexpr int kMaxBuffers = 8;
constexpr uint32_t kWBytes = kRows * kBlock;

struct BlockParams {
    const float* x_scales;            // [m][groups]
    const float* w_scales;            // [ceil(n / 128)][groups]
    void* out;
    int out_is_f32;
    int m, n, groups;
    int stages, split;
    int early;                        // W may be asked for before the kernel in front is complete
    int* error_flag;
};

__device__ __forceinline__ void store_result(const BlockParams& p, int token, int row, float v) {
    const size_t at = (size_t)token * p.n + row;
    if (p.out_is_f32) reinterpret_cast<float*>(p.out)[at] = v;
    else reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
}

constexpr uint32_t stage_bytes(int tokens) { return kWBytes + (uint32_t)tokens * kBlock; }
constexpr int buffers_of(int tokens) { return 256 / tokens < kMaxBuffers ? 256 / tokens : kMaxBuffers; }

template <int TOKENS>
__global__ void __launch_bounds__(kThreads, kPerSm)
    gemm_block_scaled_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const BlockParams p) {
    constexpr int kBuffers = buffers_of(TOKENS);
    constexpr uint32_t kColumns = kBuffers * TOKENS;
    constexpr uint32_t kStageBytes = stage_bytes(TOKENS);
    constexpr int kPart = TOKENS < 32 ? TOKENS : 32;      // tokens read from tensor memory at a time
    extern __shared__ unsigned char block_shared[];
    __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], sums_full[kMaxBuffers], sums_empty[kMaxBuffers],
        scale_full[kScaleSlots], scale_empty[kScaleSlots];
    __shared__ __align__(16) float scales[kScaleSlots][TOKENS];      // of a unit: each token's times W's
    __shared__ uint32_t tmem_slot;
    __shared__ int failed;
    const uint32_t ring = (tma::smem_u32(block_shared) + 1023u) & ~1023u;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = p.split > 1 ? (int)cluster_rank() : 0;
    const int tile = blockIdx.x / p.split;
    const int first = p.groups * rank / p.split, count = p.groups * (rank + 1) / p.split - first;      // this block's units

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            tma::mbar_init(tma::smem_u32(&full[s]), 1);
            tma::mbar_init(tma::smem_u32(&empty[s]), 1);
        }
        for (int b = 0; b < kBuffers; ++b) {
            tma::mbar_init(tma::smem_u32(&sums_full[b]), 1);
            tma::mbar_init(tma::smem_u32(&sums_empty[b]), kAdders);
        }
        for (int s = 0; s < kScaleSlots; ++s) {
            tma::mbar_init(tma::smem_u32(&scale_full[s]), 1);
            tma::mbar_init(tma::smem_u32(&scale_empty[s]), kAdders);
        }
        tma::mbar_fence_init();
        failed = 0;
        if (p.early)
            for (int s = 0; s < p.stages && s < count; ++s) {
                tma::mbar_expect_tx(tma::smem_u32(&full[s]), kStageBytes);
                tma::load_2d(ring + s * kStageBytes, &map_w, tma::smem_u32(&full[s]), (first + s) * kBlock, tile * kRows);
            }
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
    }
    pdl_wait();
    // Tensor memory is taken when the kernel in front has given its own back, and the successor is let in when this block has its share:
    // two kernels never wait for each other's.
    if (warp == 3) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tma::smem_u32(&tmem_slot)), "r"(kColumns));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc5::fence_before();
    __syncthreads();
    tc5::fence_after();
    pdl_trigger();
    const uint32_t tmem = tmem_slot;

    if (warp == 0) {
        bool ok = true;
        Turn turn;
        for (int i = 0; i < count && ok; ++i) {
            const uint32_t stage = ring + turn.at * kStageBytes, bar = tma::smem_u32(&full[turn.at]);
            if (i >= p.stages) ok = __all_sync(0xffffffffu, tma::mbar_wait(tma::smem_u32(&empty[turn.at]), turn.parity ^ 1));
            if (!ok) break;
            if (elect_one()) {
                if (!p.early || i >= p.stages) {
                    tma::mbar_expect_tx(bar, kStageBytes);
                    tma::load_2d(stage, &map_w, bar, (first + i) * kBlock, tile * kRows);
                }
                tma::load_2d(stage + kWBytes, &map_x, bar, (first + i) * kBlock, 0);
            }
            turn.step(p.stages);
        }
        // the last MMAs signal this block's barriers: it may not leave before they have
        for (int back = count < p.stages ? count : p.stages; back > 0 && ok; --back)
            ok = tma::mbar_wait(tma::smem_u32(&empty[(count - back) % p.stages]), ((count - back) / p.stages) & 1);
        if (!ok) failed = 1;
    } else if (warp == 1) {
        const uint32_t idesc = instruction_f8(kRows, TOKENS);
        const uint64_t desc_w = tc5::desc_k_major(ring, 1024u), desc_x = tc5::desc_k_major(ring + kWBytes, 1024u);
        bool ok = true;
        Turn turn, buffer;
        for (int i = 0; i < count && ok; ++i) {
            if (i >= kBuffers) ok = tma::mbar_wait(tma::smem_u32(&sums_empty[buffer.at]), buffer.parity ^ 1);
            ok = __all_sync(0xffffffffu, ok && tma::mbar_wait(tma::smem_u32(&full[turn.at]), turn.parity));
            if (!ok) break;
            tc5::fence_after();
            const uint64_t stage = turn.at * (kStageBytes >> 4);      // descriptors hold addresses in units of 16 bytes
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < kBlock / 32; ++k) mma_f8(tmem + buffer.at * TOKENS, desc_w + stage + k * 2, desc_x + stage + k * 2, idesc, k > 0);
                tc5::mma_commit(tma::smem_u32(&empty[turn.at]));
                tc5::mma_commit(tma::smem_u32(&sums_full[buffer.at]));
            }
            turn.step(p.stages);
            buffer.step(kBuffers);
        }
        if (!ok) failed = 1;
    } else if (warp == 2) {
        // A lane's tokens' scales times W's, asked for kScalesAhead units before.
        constexpr int kMine = TOKENS < 32 ? 1 : TOKENS / 32;
        const float* w_scales = p.w_scales + (size_t)tile * p.groups + first;
        float x_scale[kScalesAhead][kMine], w_scale[kScalesAhead];
        auto ask = [&](int i, float (&x)[kMine], float& w) {
            w = w_scales[i];
#pragma unroll
            for (int t = 0; t < kMine; ++t) {
                const int token = t * 32 + lane;
                x[t] = token < p.m && t * 32 + lane < TOKENS ? p.x_scales[(size_t)token * p.groups + first + i] : 0.0f;
            }
        };
#pragma unroll
        for (int d = 0; d < kScalesAhead; ++d)
            if (d < count) ask(d, x_scale[d], w_scale[d]);
        bool ok = true;
        Turn slot;
        for (int i = 0; i < count && ok; i += kScalesAhead) {
#pragma unroll
            for (int d = 0; d < kScalesAhead; ++d) {
                if (i + d >= count || !ok) break;
                if (i + d >= kScaleSlots) ok = __all_sync(0xffffffffu, tma::mbar_wait(tma::smem_u32(&scale_empty[slot.at]), slot.parity ^ 1));
                if (!ok) break;
#pragma unroll
                for (int t = 0; t < kMine; ++t)
                    if (t * 32 + lane < TOKENS) scales[slot.at][t * 32 + lane] = x_scale[d][t] * w_scale[d];
                __syncwarp();
                if (lane == 0) tma::mbar_arrive(tma::smem_u32(&scale_full[slot.at]));
                slot.step(kScaleSlots);
                if (i + d + kScalesAhead < count) ask(i + d + kScalesAhead, x_scale[d], w_scale[d]);
            }
        }
        if (!ok) failed = 1;
    } else if (warp >= 4) {
        const int row = (warp & 3) * 32 + lane;      // its row of W in the tile
        const uint32_t address = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        uint64_t sums[TOKENS / 2];      // of two tokens each
#pragma unroll
        for (int c = 0; c < TOKENS / 2; ++c) sums[c] = 0;
        bool ok = true;
        Turn slot, buffer;
        for (int i = 0; i < count && ok; ++i) {
            ok = __all_sync(0xffffffffu, tma::mbar_wait(tma::smem_u32(&scale_full[slot.at]), slot.parity) &&
                                             tma::mbar_wait(tma::smem_u32(&sums_full[buffer.at]), buffer.parity));
            if (!ok) break;
            tc5::fence_after();
#pragma unroll
            for (int part = 0; part < TOKENS; part += kPart) {
                uint32_t r[kPart];
                tmem_ask<kPart>(address + buffer.at * TOKENS + part, r);
                tmem_wait<kPart>(r);
                if (part + kPart == TOKENS) {      // all of the buffer is in registers
                    tc5::fence_before();
                    __syncwarp();
                    if (lane == 0) tma::mbar_arrive(tma::smem_u32(&sums_empty[buffer.at]));
                }
#pragma unroll
                for (int c = 0; c < kPart; c += 4) {
                    const ulonglong2 scale = *reinterpret_cast<const ulonglong2*>(&scales[slot.at][part + c]);
                    uint64_t& low = sums[(part + c) / 2];
                    uint64_t& high = sums[(part + c) / 2 + 1];
                    low = tc5::fma_pair(tc5::pair_of(__uint_as_float(r[c]), __uint_as_float(r[c + 1])), scale.x, low);
                    high = tc5::fma_pair(tc5::pair_of(__uint_as_float(r[c + 2]), __uint_as_float(r[c + 3])), scale.y, high);
                }
            }
            __syncwarp();
            if (lane == 0) tma::mbar_arrive(tma::smem_u32(&scale_empty[slot.at]));
            slot.step(kScaleSlots);
            buffer.step(kBuffers);
        }
        if (!ok) failed = 1;
        const int w_row = tile * kRows + row;
#pragma unroll
        for (int c = 0; c < TOKENS; c += 2) {
            float low, high;
            tc5::halves_of(sums[c / 2], low, high);
            if (p.split > 1) {
                // all copies into the ring and all MMAs that read it are complete: [token][row of W]
                if (ok) {
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(ring + (c * kRows + row) * 4), "f"(low) : "memory");
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(ring + ((c + 1) * kRows + row) * 4), "f"(high) : "memory");
                }
            } else if (w_row < p.n) {
                if (c < p.m) store_result(p, c, w_row, low);
                if (c + 1 < p.m) store_result(p, c + 1, w_row, high);
            }
        }
    }
    __syncwarp();
    tc5::fence_before();
    __syncthreads();
    tc5::fence_after();
    if (failed)      // a wait ran out: copies that may still be in flight get time to land
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    // given back in front of the cluster's barriers: a block that holds tensor memory waits for nobody who may be waiting for some
    if (warp == 3) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns));
    if (p.split > 1) {
        cluster_sync();
        // the tokens of a tile are dealt to the blocks of the cluster, a warp each
        for (int t = rank + warp * p.split; t < TOKENS && t < p.m; t += kThreads / 32 * p.split) {
            float4 sum = load_peer4(ring + (t * kRows + lane * 4) * 4, 0);
            for (int peer = 1; peer < p.split; ++peer) {
                const float4 part = load_peer4(ring + (t * kRows + lane * 4) * 4, peer);
                sum.x += part.x, sum.y += part.y, sum.z += part.z, sum.w += part.w;
            }
            const float values[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (tile * kRows + lane * 4 + c < p.n) store_result(p, t, tile * kRows + lane * 4 + c, values[c]);
        }
        cluster_sync();      // nobody leaves while others read its shared memory
    }
    if (failed && threadIdx.x == 0 && p.error_flag) atomicExch(p.error_flag, 2);
}

// Whether the tokens are the MMA's M (gemm_block_scaled_many.cu): beyond 64 of them, and beyond 32 where W's tiles are enough for every other SM, so that
// that kernel need not split k (40 rows by 8192 x 2048 11.4 us here and 12.6 there, by 10240 x 4096 15.8 and 15.0, by 24576 x 4096 25.3 and 23.4; 64 rows
// by 4096 x 4096 13.4 and 13.7, by 24576 x 4096 26.9 and 23.7; 32 rows by 24576 x 4096, in tiles of 32, 22.4 here).
bool many_rows(int m, int n) { return m > 64 || (m > 32 && 2 * ((n + kRows - 1LL) / kRows) > llm_sm_count()); }

int tokens_per_tile(int m) { return m <= 16 ? 16 : m <= 32 ? 32 : 64; }

// Into how many parts k is split: as many as one round of blocks holds (a second round waits for the first to give up its share of an SM:
// 1 row by 24576 x 4096, 192 tiles on 296 places, 19.1 us whole, 23.4 in two parts, 26.6 in three), a power of two (clusters of 3, 5, 6 and 7 leave
// places empty: 1 row by 6144 x 4096 in four parts 8.3 us, in six 12.5), each of two units at least.
int split_of(long long tiles, int groups) {
    const long long room = (long long)kPerSm * llm_sm_count();
    int split = 1;
    while (2 * split <= kMaxSplit && tiles * 2 * split <= room && groups / (2 * split) >= 2) split *= 2;
    return split;
}

template <int TOKENS>
int launch_block_scaled(const void* x, long long x_pitch, const void* w, long long w_pitch, BlockParams p, int inner, cudaStream_t stream) {
    CUtensorMap map_w, map_x;
    if (!make_map_f8(&map_w, w, (uint64_t)p.n, (uint64_t)inner, (uint64_t)w_pitch, kRows) ||
        !make_map_f8(&map_x, x, (uint64_t)p.m, (uint64_t)inner, (uint64_t)x_pitch, TOKENS)) {
        llm_set_error("block_linear: the tensor maps could not be made");
        return LLM_REFUSED;
    }
    const int tiles = (p.n + kRows - 1) / kRows;
    p.split = split_of(tiles, p.groups);
    p.stages = (int)(kRingBytes / stage_bytes(TOKENS));
    const size_t shared = (size_t)p.stages * stage_bytes(TOKENS) + 1024;
    if (int status = llm_raise_shared_limit((const void*)gemm_block_scaled_kernel<TOKENS>, shared, "block_linear", true)) return status;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(tiles * p.split), 1, 1);
    config.blockDim = dim3(kThreads, 1, 1);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    cudaLaunchAttribute attribute[2];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim.x = (unsigned)p.split;
    attribute[0].val.clusterDim.y = 1;
    attribute[0].val.clusterDim.z = 1;
    attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attribute;
    config.numAttrs = llm_pdl_enabled() ? 2 : 1;
    const cudaError_t status = cudaLaunchKernelEx(&config, gemm_block_scaled_kernel<TOKENS>, map_w, map_x, p);
    if (status != cudaSuccess) {
        llm_set_error("block_linear launch: %s", cudaGetErrorString(status));
        return (int)status;
    }
    return llm_check_launch("block_linear");
}

int refuse_product(long long m, int n, int inner, long long x_pitch, long long w_pitch) {
    if (m < 0 || n < 1 || n > kMostAlong || inner < 1 || inner > kMostAlong || x_pitch < inner || x_pitch % 16 != 0 || w_pitch < inner || w_pitch % 16 != 0 || m > 65535 * 128LL ||
        (m + 127) / 128 * ((n + 127LL) / 128) * ((inner + 127LL) / 128) > 0x7fffffffLL / kMaxSplit) {
        llm_set_error("block_linear: [%lld, %d] x [%d, %d]^T with rows %lld and %lld bytes apart is not supported", m, inner, n, inner, x_pitch, w_pitch);
        return LLM_REFUSED;
    }
    return LLM_OK;
}

}  // namespace

int llm_block_linear_many(const void* x, long long x_pitch, const float* x_scales, const void* w, long long w_pitch, const float* w_scales, void* out,
                          int out_is_f32, int m, int n, int inner, int early, int* error_flag, cudaStream_t stream);
extern "C" int llm_quantize_blocks(const void* x, int dtype, void* out, float* scales, int rows, int inner, long long pitch, int block_rows,
                                   cudaStream_t stream);

// out[m, n] (float or bfloat16) = x W^T.  `x` [m, inner]: float or bfloat16 (x_dtype 0 or 1, contiguous), or (x_dtype -1) 8 bits with rows
// x_pitch bytes apart and x_scales [m, ceil(inner / 128)].  The former are brought to 8 bits in `scratch`: m rows of x_pitch bytes, then
// m * ceil(inner / 128) scales.
LLM_EXPORT int llm_block_linear(const void* x, int x_dtype, long long x_pitch, const float* x_scales, const void* w, long long w_pitch,
                                const float* w_scales, void* out, int out_is_f32, int m, int n, int inner, void* scratch, int* error_flag,
                                cudaStream_t stream) {
    if (int status = refuse_product(m, n, inner, x_pitch, w_pitch)) return status;
    if (!aligned16(w) || (x_dtype < 0 && !aligned16(x)) || !aligned16(scratch)) {
        llm_set_error("block_linear: operands in 8 bits begin at multiples of 16 bytes");
        return LLM_REFUSED;
    }
    if (x_dtype >= 0 && m > 0 && scratch == nullptr) {
        llm_set_error("block_linear: %d rows are brought to 8 bits in scratch, and there is none", m);
        return LLM_REFUSED;
    }
    if (x_dtype > LLM_BF16) {
        llm_set_error("unknown dtype code %d", x_dtype);
        return LLM_REFUSED;
    }
    if (m == 0) return LLM_OK;
    BlockParams p = {};
    p.groups = (inner + kBlock - 1) / kBlock;
    p.x_scales = x_scales;
    p.w_scales = w_scales;
    p.out = out;
    p.out_is_f32 = out_is_f32;
    p.m = m;
    p.n = n;
    p.error_flag = error_flag;
    const void* rows = x;
    if (x_dtype >= 0) {
        float* made = reinterpret_cast<float*>(static_cast<unsigned char*>(scratch) + (size_t)m * x_pitch);
        if (int status = llm_quantize_blocks(x, x_dtype, scratch, made, m, inner, x_pitch, 1, stream)) return status;
        rows = scratch;
        p.x_scales = made;
        p.early = 1;      // that kernel lets this one in only when all in front of it is complete
    }
    if (many_rows(m, n))
        return llm_block_linear_many(rows, x_pitch, p.x_scales, w, w_pitch, w_scales, out, out_is_f32, m, n, inner, p.early, error_flag, stream);
    switch (tokens_per_tile(m)) {
        case 16: return launch_block_scaled<16>(rows, x_pitch, w, w_pitch, p, inner, stream);
        case 32: return launch_block_scaled<32>(rows, x_pitch, w, w_pitch, p, inner, stream);
        default: return launch_block_scaled<64>(rows, x_pitch, w, w_pitch, p, inner, stream);
    }
}
