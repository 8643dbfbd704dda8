// y[m, n] = sum over blocks b of 128 along k:  xs[m, b] * ws[n / 128, b] * sum_{k in b} xq[m, k] wq[n, k]
//
// Both operands are e4m3 with 32-bit scales, one for each row and 128 columns of x, one for each 128 x 128 of W.  The products of a
// block are summed by tcgen05.mma (kind::f8f6f4: exact products, 32-bit sums) into tensor memory; from there they are read back,
// multiplied with the block's two scales and added up in registers, 32-bit as well: the scales are any 32-bit numbers, so blocks
// cannot be added before they are scaled.
//
// The roles of the operands are swapped for the hardware, as in gemm_tcgen05.cu: 128 rows of W are the MMA's M, the tokens (16 to
// 128) its N, so that a product of few tokens streams W and wastes nothing on rows that do not exist.  A stage of the ring is one
// block of 128 along k: 16 KiB of W and up to 16 KiB of x, which are one swizzle atom wide.  The MMAs of a block go to one of several
// buffers of tensor memory, so that they run ahead of the four warps that scale and add.  Where tiles are too few for the SMs, k is
// split over a cluster and the parts are added through distributed shared memory in the order of k.
//
// Roles: warp 0 copies (TMA), warp 1 issues the MMAs, warp 2 brings the tokens' scales (asynchronous copies of 4 bytes, several
// blocks ahead), warp 3 holds the tensor memory, warps 4 to 7 scale and add, a row of W per thread.  All waits are bounded: one that runs out
// sets error code 2, every role leaves its loop, and the block still frees its tensor memory and meets its cluster.
//
// k need not be a multiple of 128 nor n of 128 nor m of anything: what lies outside is read as zeros (TMA) and not written.
#include "common.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace {

constexpr int kRows = 128;            // rows of W per tile (UMMA M)
constexpr int kBlock = 128;           // of k: one stage, one pair of scales
constexpr int kThreads = 256;
constexpr int kMaxStages = 12;
constexpr int kScaleSlots = 8;        // blocks whose token scales are on their way or waiting
constexpr int kMaxBuffers = 8;
constexpr int kMaxSplit = 8;
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

__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// e4m3 x e4m3 -> float32, both operands K-major.
__device__ __forceinline__ uint32_t instruction_f8(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

__device__ __forceinline__ void tmem_load_16(uint32_t address, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(address)
        : "memory");
}

// 4 bytes from global to shared memory (zeros where `present` is false), and this thread's arrival on a barrier once all its copies
// so far have landed.
__device__ __forceinline__ void copy_4(uint32_t dst, const float* src, bool present) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(present ? 4u : 0u) : "memory");
}
__device__ __forceinline__ void arrive_when_copied(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    return rank;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 load_peer4(uint32_t local_address, uint32_t rank) {
    uint32_t remote;
    float4 value;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_address), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(value.x), "=f"(value.y), "=f"(value.z), "=f"(value.w) : "r"(remote) : "memory");
    return value;
}

__device__ __forceinline__ void store_result(const BlockParams& p, int token, int row, float v) {
    const size_t at = (size_t)token * p.n + row;
    if (p.out_is_f32) reinterpret_cast<float*>(p.out)[at] = v;
    else reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
}

constexpr int buffers_of(int tokens) { return 256 / tokens < kMaxBuffers ? 256 / tokens : kMaxBuffers; }
constexpr uint32_t stage_bytes(int tokens) { return kWBytes + (uint32_t)tokens * kBlock; }

// Up to 64 tokens two blocks share an SM; with 128 a thread's sums alone are 128 registers, and a block has the SM to itself.
template <int TOKENS>
__global__ void __launch_bounds__(kThreads, TOKENS <= 64 ? 2 : 1)
    gemm_block_scaled_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const BlockParams p) {
    constexpr int kBuffers = buffers_of(TOKENS);
    constexpr uint32_t kColumns = kBuffers * TOKENS;
    constexpr uint32_t kStageBytes = stage_bytes(TOKENS);
    extern __shared__ unsigned char block_shared[];
    __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], sums_full[kMaxBuffers], sums_empty[kMaxBuffers],
        scale_full[kScaleSlots], scale_empty[kScaleSlots];
    __shared__ __align__(16) float token_scales[kScaleSlots][TOKENS];
    __shared__ uint32_t tmem_slot;
    __shared__ int failed;
    const uint32_t ring = (tma::smem_u32(block_shared) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = p.split > 1 ? (int)cluster_rank() : 0;
    const int tile = blockIdx.x / p.split, token0 = blockIdx.y * TOKENS;
    const int first = (int)((long long)p.groups * rank / p.split), count = (int)((long long)p.groups * (rank + 1) / p.split) - first;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            tma::mbar_init(tma::smem_u32(&full[s]), 1);
            tma::mbar_init(tma::smem_u32(&empty[s]), 1);
        }
        for (int b = 0; b < kBuffers; ++b) {
            tma::mbar_init(tma::smem_u32(&sums_full[b]), 1);
            tma::mbar_init(tma::smem_u32(&sums_empty[b]), 4);
        }
        for (int s = 0; s < kScaleSlots; ++s) {
            tma::mbar_init(tma::smem_u32(&scale_full[s]), 32);
            tma::mbar_init(tma::smem_u32(&scale_empty[s]), 4);
        }
        tma::mbar_fence_init();
        failed = 0;
        if (p.early)
            for (int s = 0; s < p.stages && s < count; ++s) {
                tma::mbar_expect_tx(tma::smem_u32(&full[s]), kStageBytes);
                tma::load_2d(ring + s * kStageBytes, &map_w, tma::smem_u32(&full[s]), (first + s) * kBlock, tile * kRows);
            }
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
    float sums[TOKENS];
#pragma unroll
    for (int c = 0; c < TOKENS; ++c) sums[c] = 0.0f;

    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            for (int i = 0; i < count && ok; ++i) {
                const int s = i % p.stages;
                const uint32_t stage = ring + s * kStageBytes, bar = tma::smem_u32(&full[s]);
                if (i >= p.stages) ok = tma::mbar_wait(tma::smem_u32(&empty[s]), ((i / p.stages) - 1) & 1);
                if (!ok) break;
                if (!p.early || i >= p.stages) {
                    tma::mbar_expect_tx(bar, kStageBytes);
                    tma::load_2d(stage, &map_w, bar, (first + i) * kBlock, tile * kRows);
                }
                tma::load_2d(stage + kWBytes, &map_x, bar, (first + i) * kBlock, token0);
            }
            // the last MMAs signal this block's barriers: it may not leave before they have
            for (int back = count < p.stages ? count : p.stages; back > 0 && ok; --back)
                ok = tma::mbar_wait(tma::smem_u32(&empty[(count - back) % p.stages]), ((count - back) / p.stages) & 1);
            if (!ok) failed = 1;
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = instruction_f8(kRows, TOKENS);
            bool ok = true;
            for (int i = 0; i < count && ok; ++i) {
                const int s = i % p.stages, b = i % kBuffers;
                if (i >= kBuffers) ok = tma::mbar_wait(tma::smem_u32(&sums_empty[b]), ((i / kBuffers) - 1) & 1);
                if (ok) ok = tma::mbar_wait(tma::smem_u32(&full[s]), (i / p.stages) & 1);
                if (!ok) break;
                tc5::fence_after();
                const uint32_t stage = ring + s * kStageBytes;
#pragma unroll
                for (int k = 0; k < kBlock / 32; ++k)
                    mma_f8(tmem + b * TOKENS, tc5::desc_k_major(stage + k * 32, 1024u), tc5::desc_k_major(stage + kWBytes + k * 32, 1024u), idesc, k > 0);
                tc5::mma_commit(tma::smem_u32(&empty[s]));
                tc5::mma_commit(tma::smem_u32(&sums_full[b]));
            }
            if (!ok) failed = 1;
        }
    } else if (warp == 2) {
        bool ok = true;
        for (int i = 0; i < count && ok; ++i) {
            const int s = i % kScaleSlots;
            if (i >= kScaleSlots) ok = tma::mbar_wait(tma::smem_u32(&scale_empty[s]), ((i / kScaleSlots) - 1) & 1);
            if (!ok) break;
            for (int t = lane; t < TOKENS; t += 32) {
                const bool present = token0 + t < p.m;
                copy_4(tma::smem_u32(&token_scales[s][t]), p.x_scales + (present ? (size_t)(token0 + t) * p.groups + first + i : 0), present);
            }
            arrive_when_copied(tma::smem_u32(&scale_full[s]));
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (!ok) failed = 1;
    } else if (warp >= 4) {
        const uint32_t address = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const float* w_scales = p.w_scales + (size_t)tile * p.groups + first;
        bool ok = true;
        float w_scale = count > 0 ? w_scales[0] : 0.0f;
        for (int i = 0; i < count && ok; ++i) {
            const int s = i % kScaleSlots, b = i % kBuffers;
            const float scale = w_scale;
            if (i + 1 < count) w_scale = w_scales[i + 1];
            ok = __all_sync(0xffffffffu, tma::mbar_wait(tma::smem_u32(&scale_full[s]), (i / kScaleSlots) & 1) &&
                                             tma::mbar_wait(tma::smem_u32(&sums_full[b]), (i / kBuffers) & 1));
            if (!ok) break;
            tc5::fence_after();
#pragma unroll
            for (int part = 0; part < TOKENS / 16; ++part) {
                uint32_t r[16];
                tmem_load_16(address + b * TOKENS + part * 16, r);
#pragma unroll
                for (int c = 0; c < 16; ++c)
                    sums[part * 16 + c] = fmaf(__uint_as_float(r[c]), token_scales[s][part * 16 + c] * scale, sums[part * 16 + c]);
            }
            tc5::fence_before();
            __syncwarp();
            if (lane == 0) {
                tma::mbar_arrive(tma::smem_u32(&sums_empty[b]));
                tma::mbar_arrive(tma::smem_u32(&scale_empty[s]));
            }
        }
        if (!ok) failed = 1;
        const int row = (warp & 3) * 32 + lane;
        if (p.split == 1) {
            if (tile * kRows + row < p.n)
#pragma unroll
                for (int c = 0; c < TOKENS; ++c)
                    if (token0 + c < p.m) store_result(p, token0 + c, tile * kRows + row, sums[c]);
        } else if (ok) {
            // all copies into the ring and all MMAs that read it are complete: [token][row of W]
#pragma unroll
            for (int c = 0; c < TOKENS; ++c)
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(ring + (c * kRows + row) * 4), "f"(sums[c]) : "memory");
        }
    }
    __syncwarp();
    tc5::fence_before();
    __syncthreads();
    tc5::fence_after();
    if (failed)      // a wait ran out: copies that may still be in flight get time to land
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    if (p.split > 1) {
        cluster_sync();
        // the tokens of a tile are dealt to the blocks of the cluster, a warp each
        for (int t = rank + warp * p.split; t < TOKENS && token0 + t < p.m; t += kThreads / 32 * p.split) {
            float4 sum = load_peer4(ring + (t * kRows + lane * 4) * 4, 0);
            for (int peer = 1; peer < p.split; ++peer) {
                const float4 part = load_peer4(ring + (t * kRows + lane * 4) * 4, peer);
                sum.x += part.x, sum.y += part.y, sum.z += part.z, sum.w += part.w;
            }
            const float values[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (tile * kRows + lane * 4 + c < p.n) store_result(p, token0 + t, tile * kRows + lane * 4 + c, values[c]);
        }
        cluster_sync();      // nobody leaves while others read its shared memory
    }
    if (failed && threadIdx.x == 0 && p.error_flag) atomicExch(p.error_flag, 2);
    if (warp == 3) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns));
}

// Tensor map of bytes [rows, columns] with `pitch` bytes between rows, box = [box_rows, 128 columns], 128-byte swizzle, zeros outside.
bool make_map_f8(CUtensorMap* map, const void* pointer, uint64_t rows, uint64_t columns, uint64_t pitch, uint32_t box_rows) {
    tma::EncodeTiled encode = tma::encode_tiled();
    if (encode == nullptr) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)columns, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)pitch};
    const cuuint32_t box[2] = {(cuuint32_t)kBlock, box_rows};
    const cuuint32_t ones[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(pointer), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int TOKENS>
int launch_block_scaled(const void* x, long long x_pitch, const void* w, long long w_pitch, BlockParams p, int inner, cudaStream_t stream) {
    CUtensorMap map_w, map_x;
    if (!make_map_f8(&map_w, w, (uint64_t)p.n, (uint64_t)inner, (uint64_t)w_pitch, kRows) ||
        !make_map_f8(&map_x, x, (uint64_t)p.m, (uint64_t)inner, (uint64_t)x_pitch, TOKENS)) {
        llm_set_error("block_linear: the tensor maps could not be made");
        return LLM_REFUSED;
    }
    const int tiles = (p.n + kRows - 1) / kRows, token_tiles = (p.m + TOKENS - 1) / TOKENS;
    const int per_sm = TOKENS <= 64 ? 2 : 1;
    const long long room = (long long)per_sm * llm_sm_count();
    p.split = 1;
    while (2 * p.split <= kMaxSplit && (long long)tiles * token_tiles * 2 * p.split <= room && p.groups / (2 * p.split) >= 2) p.split *= 2;
    const uint32_t ring_bytes = per_sm == 2 ? 96u << 10 : 200u << 10;
    p.stages = (int)(ring_bytes / stage_bytes(TOKENS));
    if (p.stages > kMaxStages) p.stages = kMaxStages;
    size_t shared = (size_t)p.stages * stage_bytes(TOKENS) + 1024;
    if (int status = llm_raise_shared_limit((const void*)gemm_block_scaled_kernel<TOKENS>, shared, "block_linear", true)) return status;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(tiles * p.split), (unsigned)token_tiles, 1);
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

}  // namespace

extern "C" int llm_quantize_blocks(const void* x, int dtype, void* out, float* scales, int rows, int inner, long long pitch, int block_rows,
                                   cudaStream_t stream);

// out[m, n] (float or bfloat16) = x W^T.  `x` [m, inner] float or bfloat16 (x_dtype), brought to 8 bits in xq [m, x_pitch] and
// x_scales [m, ceil(inner / 128)] first; null: xq and x_scales hold it already.
LLM_EXPORT int llm_block_linear(const void* x, int x_dtype, void* xq, long long x_pitch, float* x_scales, const void* w, long long w_pitch,
                                const float* w_scales, void* out, int out_is_f32, int m, int n, int inner, int* error_flag, cudaStream_t stream) {
    if (m < 0 || n < 1 || inner < 1 || x_pitch < inner || x_pitch % 16 != 0 || w_pitch < inner || w_pitch % 16 != 0 || !aligned16(xq) || !aligned16(w)) {
        llm_set_error("block_linear: [%d, %d] x [%d, %d]^T with rows %lld and %lld bytes apart is not supported", m, inner, n, inner, x_pitch, w_pitch);
        return LLM_REFUSED;
    }
    if (m == 0) return LLM_OK;
    if (m > 65535 * 128) {
        llm_set_error("block_linear: at most %d rows, got %d", 65535 * 128, m);
        return LLM_REFUSED;
    }
    if (x != nullptr)
        if (int status = llm_quantize_blocks(x, x_dtype, xq, x_scales, m, inner, x_pitch, 1, stream)) return status;
    BlockParams p = {};
    p.x_scales = x_scales;
    p.w_scales = w_scales;
    p.out = out;
    p.out_is_f32 = out_is_f32;
    p.m = m;
    p.n = n;
    p.groups = (inner + kBlock - 1) / kBlock;
    p.early = x != nullptr;
    p.error_flag = error_flag;
    if (m <= 16) return launch_block_scaled<16>(xq, x_pitch, w, w_pitch, p, inner, stream);
    if (m <= 32) return launch_block_scaled<32>(xq, x_pitch, w, w_pitch, p, inner, stream);
    if (m <= 64) return launch_block_scaled<64>(xq, x_pitch, w, w_pitch, p, inner, stream);
    return launch_block_scaled<128>(xq, x_pitch, w, w_pitch, p, inner, stream);
}
