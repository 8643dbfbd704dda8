// The product of gemm_block_scaled.cu for many tokens: y[m, n] = sum_b xs[m, b] ws[n / 128, b] (xq wq^T over block b of k), operands e4m3.
//
// Here the tokens are the MMA's M = 128 and 128 or 256 rows of W its N.  A lane of tensor memory is then a token, and what a block's sums
// are multiplied with is one number per thread and 128 rows of W, which the adders read from shared memory as one word a unit.  (With a
// token per column every thread has to read the numbers of all its columns: 64 KiB of registers filled from shared memory per unit of
// 128 x 128 x 128, 512 cycles beside the MMA's 256.)
//
// A block has its SM to itself and walks tiles c, c + blocks, ...; the ring of stages (128 of k each: 16 KiB of x, 16 or 32 KiB of W) and the
// buffers of tensor memory run on across tiles.  Eight warps scale and add: two share the lanes of a quarter, each half of the columns, 64 or
// 128 sums a thread.  A finished tile goes from registers through 2 KiB of shared memory per warp, so that it leaves in pieces of 64 bytes a row.
// Where there are few tiles of 128 columns, k is split over a cluster and the parts are added through distributed shared memory in the
// order of k.
//
// Roles, bounded waits and the treatment of ragged sizes are those of gemm_block_scaled.cu.
#include "block_scaled_mma.cuh"

namespace {

using namespace block_scaled;

constexpr int kTokens = 128;          // per tile (UMMA M)
constexpr int kAdders = 8;
constexpr int kThreads = 128 + 32 * kAdders;
constexpr int kMaxStages = 6;
constexpr int kMaxBuffers = 4;
constexpr int kMaxSplit = 4;
constexpr int kRun = 4;               // units whose scales are handed over together: a wait costs 100 cycles even where it need not wait
constexpr int kScaleSlots = 2;        // runs of units whose scales wait to be used; another is on its way from memory
constexpr uint32_t kXBytes = kTokens * kBlock;
constexpr uint32_t kPieceBytes = 32 * 64;

struct ManyParams {
    const float* x_scales;            // [m][groups]
    const float* w_scales;            // [ceil(n / 128)][groups]
    void* out;
    int out_is_f32;
    int m, n, groups;
    int row_tiles, col_tiles, row_group;      // row tiles that are walked together for each column tile
    int split;
    int bulk_out;                     // rows of the output begin at multiples of 16 bytes: pieces leave as bulk stores
    int early;                        // W may be asked for before the kernel in front is complete
    int* error_flag;
};

constexpr uint32_t stage_bytes(int cols) { return kXBytes + (uint32_t)cols * kBlock; }
constexpr int stages_of(int cols) { return cols == 128 ? 6 : 4; }
constexpr uint32_t shared_bytes(int cols) { return stages_of(cols) * stage_bytes(cols) + kAdders * kPieceBytes + 1024; }

// Tile t of the walk: row_group row tiles through all column tiles before the next ones, so that these rows of x stay in L2 while W passes.
struct Tile {
    int token0, col0;
};
template <int COLS>
__device__ __forceinline__ Tile tile_of(const ManyParams& p, int t) {
    const int per_group = p.row_group * p.col_tiles, group = t / per_group, rest = t - group * per_group;
    const int in_group = min(p.row_group, p.row_tiles - group * p.row_group);
    return Tile{(group * p.row_group + rest % in_group) * kTokens, rest / in_group * COLS};
}

// The units of this block, one after the other.
template <int COLS>
struct Walk {
    int t, group, first, last;
    Tile tile;
    __device__ __forceinline__ void begin(const ManyParams& p, int t0, int from, int to) {
        t = t0, group = first = from, last = to;
        tile = tile_of<COLS>(p, t);
    }
    __device__ __forceinline__ bool ends() const { return group + 1 == last; }
    __device__ __forceinline__ void step(const ManyParams& p, int stride, int total) {
        if (++group < last) return;
        group = first;
        t += stride;
        if (t < total) tile = tile_of<COLS>(p, t);
    }
};

// 64 bytes of each of a warp's 32 rows, through its 2 KiB of shared memory: a lane hands in its row's; where the rows of the output begin at
// multiples of 16 bytes the piece leaves as one bulk store, which leaves out what does not exist, else four lanes store a row's four 16-byte words
// number by number.  The words of a row are swapped by the row's number (the 64-byte swizzle), free of bank conflicts both ways.
template <int ELEMENT>
__device__ __forceinline__ void put_piece(const ManyParams& p, const CUtensorMap* map_out, uint32_t buffer, int lane, int row0, int column,
                                          const uint32_t (&words)[16]) {
    if (p.bulk_out) {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // the piece before has been read
        __syncwarp();
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(buffer + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)), "r"(words[4 * c]),
                     "r"(words[4 * c + 1]), "r"(words[4 * c + 2]), "r"(words[4 * c + 3]) : "memory");
    if (p.bulk_out) {
        tma::fence_proxy_async();
        __syncwarp();
        if (lane == 0 && row0 < p.m && column < p.n) {
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
                         ::"l"(map_out), "r"(buffer), "r"(column), "r"(row0) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        return;
    }
    __syncwarp();
    constexpr int kEach = 16 / ELEMENT;
    const int c = lane & 3, at = column + c * kEach;
#pragma unroll
    for (int it = 0; it < 4; ++it) {
        const int row = it * 8 + (lane >> 2);
        uint32_t w[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(buffer + row * 64 + ((c ^ ((row >> 1) & 3)) << 4)) : "memory");
        if (row0 + row >= p.m || at >= p.n) continue;
        unsigned char* to = reinterpret_cast<unsigned char*>(p.out) + ((size_t)(row0 + row) * p.n + at) * ELEMENT;
#pragma unroll
        for (int e = 0; e < kEach; ++e)
            if (at + e < p.n) {
                if (ELEMENT == 4) reinterpret_cast<uint32_t*>(to)[e] = w[e];
                else reinterpret_cast<uint16_t*>(to)[e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
            }
    }
    __syncwarp();
}

template <int COLS>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_block_scaled_many_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                                  const __grid_constant__ CUtensorMap map_out, const ManyParams p) {
    constexpr int kBuffers = 512 / COLS, kStages = stages_of(COLS), kHalves = COLS / 128;
    constexpr uint32_t kStageBytes = stage_bytes(COLS);
    constexpr int kWidth = COLS / 2;      // columns of an adder
    constexpr bool kSplits = COLS == 128;      // the narrow tiles alone
    static_assert(kBuffers <= kMaxBuffers && kStages <= kMaxStages, "the barriers are enough");
    extern __shared__ unsigned char many_shared[];
    __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], sums_full[kMaxBuffers], sums_empty[kMaxBuffers],
        scale_full[kScaleSlots], scale_empty[kScaleSlots];
    __shared__ float scales[kScaleSlots][kRun][kHalves][kTokens];      // of a unit: each token's times W's
    __shared__ uint32_t tmem_slot;
    __shared__ int failed;
    const uint32_t ring = (tma::smem_u32(many_shared) + 1023u) & ~1023u;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = kSplits && p.split > 1 ? (int)cluster_rank() : 0;
    const int total = p.row_tiles * p.col_tiles, stride = (int)gridDim.x / p.split, t0 = (int)blockIdx.x / p.split;
    const int first = (int)((long long)p.groups * rank / p.split), last = (int)((long long)p.groups * (rank + 1) / p.split);
    const int tiles = (total - t0 + stride - 1) / stride, count = tiles * (last - first);      // this block's units
    Walk<COLS> walk;
    walk.begin(p, t0, first, last);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
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
        if (p.early) {
            Walk<COLS> ahead = walk;
            for (int s = 0; s < kStages && s < count; ++s) {
                tma::mbar_expect_tx(tma::smem_u32(&full[s]), kStageBytes);
                tma::load_2d(ring + s * kStageBytes + kXBytes, &map_w, tma::smem_u32(&full[s]), ahead.group * kBlock, ahead.tile.col0);
                ahead.step(p, stride, total);
            }
        }
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
    }
    pdl_wait();
    // tensor memory: taken behind the wait, and the successor let in behind that, as in gemm_block_scaled.cu
    if (warp == 3) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tma::smem_u32(&tmem_slot)), "r"(512));
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
            if (i >= kStages) ok = __all_sync(0xffffffffu, tma::mbar_wait(tma::smem_u32(&empty[turn.at]), turn.parity ^ 1));
            if (!ok) break;
            if (elect_one()) {
                if (!p.early || i >= kStages) {
                    tma::mbar_expect_tx(bar, kStageBytes);
                    tma::load_2d(stage + kXBytes, &map_w, bar, walk.group * kBlock, walk.tile.col0);
                }
                tma::load_2d(stage, &map_x, bar, walk.group * kBlock, walk.tile.token0);
            }
            walk.step(p, stride, total);
            turn.step(kStages);
        }
        // the last MMAs signal this block's barriers: it may not leave before they have
        for (int back = count < kStages ? count : kStages; back > 0 && ok; --back)
            ok = tma::mbar_wait(tma::smem_u32(&empty[(count - back) % kStages]), ((count - back) / kStages) & 1);
        if (!ok) failed = 1;
    } else if (warp == 1) {
        const uint32_t idesc = instruction_f8(kTokens, COLS);
        const uint64_t desc_x = tc5::desc_k_major(ring, 1024u), desc_w = tc5::desc_k_major(ring + kXBytes, 1024u);
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
                for (int k = 0; k < kBlock / 32; ++k) mma_f8(tmem + buffer.at * COLS, desc_x + stage + k * 2, desc_w + stage + k * 2, idesc, k > 0);
                tc5::mma_commit(tma::smem_u32(&empty[turn.at]));
                tc5::mma_commit(tma::smem_u32(&sums_full[buffer.at]));
            }
            turn.step(kStages);
            buffer.step(kBuffers);
        }
        if (!ok) failed = 1;
    } else if (warp == 2) {
        // A lane's four tokens' scales times W's, asked for a run of units before.
        const int col_blocks = (p.n + 127) / 128;
        float x_scale[kRun][4], w_scale[kRun][kHalves];
        auto ask = [&](float (&x)[4], float (&w)[kHalves]) {
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                const int block = walk.tile.col0 / 128 + h;
                w[h] = block < col_blocks ? p.w_scales[(size_t)block * p.groups + walk.group] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int token = walk.tile.token0 + j * 32 + lane;
                x[j] = token < p.m ? p.x_scales[(size_t)token * p.groups + walk.group] : 0.0f;
            }
            walk.step(p, stride, total);
        };
#pragma unroll
        for (int d = 0; d < kRun; ++d)
            if (d < count) ask(x_scale[d], w_scale[d]);
        bool ok = true;
        Turn slot;
        for (int i = 0; i < count && ok; i += kRun) {
            if (i >= kScaleSlots * kRun) ok = __all_sync(0xffffffffu, tma::mbar_wait(tma::smem_u32(&scale_empty[slot.at]), slot.parity ^ 1));
            if (!ok) break;
#pragma unroll
            for (int d = 0; d < kRun; ++d) {
                if (i + d >= count) break;
#pragma unroll
                for (int h = 0; h < kHalves; ++h)
#pragma unroll
                    for (int j = 0; j < 4; ++j) scales[slot.at][d][h][j * 32 + lane] = x_scale[d][j] * w_scale[d][h];
                if (i + d + kRun < count) ask(x_scale[d], w_scale[d]);
            }
            __syncwarp();
            if (lane == 0) tma::mbar_arrive(tma::smem_u32(&scale_full[slot.at]));
            slot.step(kScaleSlots);
        }
        if (!ok) failed = 1;
    } else if (warp >= 4) {
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        const int row = quarter * 32 + lane;      // its token in the tile
        const uint32_t address = tmem + ((uint32_t)(quarter * 32) << 16) + half * kWidth;
        const uint32_t buffer_of_warp = ring + kStages * kStageBytes + (warp - 4) * kPieceBytes;
        float sums[kWidth];
#pragma unroll
        for (int c = 0; c < kWidth; ++c) sums[c] = 0.0f;
        bool ok = true;
        Turn slot, buffer;
        for (int i = 0; i < count && ok; ++i) {
            const int in_run = i % kRun;
            if (in_run == 0) ok = tma::mbar_wait(tma::smem_u32(&scale_full[slot.at]), slot.parity);
            const float scale = scales[slot.at][in_run][kHalves > 1 ? half : 0][row];
            ok = __all_sync(0xffffffffu, ok && tma::mbar_wait(tma::smem_u32(&sums_full[buffer.at]), buffer.parity));
            if (!ok) break;
            tc5::fence_after();
#pragma unroll
            for (int part = 0; part < kWidth; part += 32) {
                uint32_t r[32];
                tmem_ask<32>(address + buffer.at * COLS + part, r);
                tmem_wait<32>(r);
                if (part + 32 == kWidth) {      // all of the buffer is in registers
                    tc5::fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        tma::mbar_arrive(tma::smem_u32(&sums_empty[buffer.at]));
                        if (in_run == kRun - 1) tma::mbar_arrive(tma::smem_u32(&scale_empty[slot.at]));
                    }
                }
#pragma unroll
                for (int c = 0; c < 32; ++c) sums[part + c] = fmaf(__uint_as_float(r[c]), scale, sums[part + c]);
            }
            if (in_run == kRun - 1) slot.step(kScaleSlots);
            buffer.step(kBuffers);
            if (walk.ends() && !(kSplits && p.split > 1)) {
                const int row0 = walk.tile.token0 + quarter * 32, column0 = walk.tile.col0 + half * kWidth;
                if (p.out_is_f32) {
#pragma unroll
                    for (int c0 = 0; c0 < kWidth; c0 += 16) {
                        uint32_t words[16];
#pragma unroll
                        for (int c = 0; c < 16; ++c) words[c] = __float_as_uint(sums[c0 + c]);
                        put_piece<4>(p, &map_out, buffer_of_warp, lane, row0, column0 + c0, words);
                    }
                } else {
#pragma unroll
                    for (int c0 = 0; c0 < kWidth; c0 += 32) {
                        uint32_t words[16];
#pragma unroll
                        for (int c = 0; c < 16; ++c) words[c] = tc5::pack2(sums[c0 + 2 * c], sums[c0 + 2 * c + 1]);
                        put_piece<2>(p, &map_out, buffer_of_warp, lane, row0, column0 + c0, words);
                    }
                }
#pragma unroll
                for (int c = 0; c < kWidth; ++c) sums[c] = 0.0f;
            }
            walk.step(p, stride, total);
        }
        if (!ok) failed = 1;
        if (kSplits && p.split > 1 && ok) {
            // all copies into the ring and all MMAs that read it are complete: [column][token]
#pragma unroll
            for (int c = 0; c < kWidth; ++c)
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(ring + ((half * kWidth + c) * kTokens + row) * 4), "f"(sums[c]) : "memory");
        }
    }
    __syncwarp();
    tc5::fence_before();
    __syncthreads();
    tc5::fence_after();
    if (failed)      // a wait ran out: copies that may still be in flight get time to land
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    if (kSplits && p.split > 1) {
        cluster_sync();
        const Tile tile = tile_of<COLS>(p, t0);
        // pieces of 32 tokens by 64 bytes of columns, dealt to the cluster's adders
        const int each = p.out_is_f32 ? 16 : 32, pieces = 4 * (COLS / each);
        if (warp >= 4 && !failed)
            for (int piece = rank + (warp - 4) * p.split; piece < pieces; piece += kAdders * p.split) {
                const int quarter = piece & 3, c0 = (piece >> 2) * each;
                uint32_t words[16];
                float sums[32];
                const uint32_t place = ring + (c0 * kTokens + quarter * 32 + lane) * 4;
#pragma unroll
                for (int c = 0; c < 32; ++c) sums[c] = c < each ? load_peer(place + c * kTokens * 4, 0) : 0.0f;
                for (int peer = 1; peer < p.split; ++peer) {
                    float more[32];      // asked for together
#pragma unroll
                    for (int c = 0; c < 32; ++c) more[c] = c < each ? load_peer(place + c * kTokens * 4, peer) : 0.0f;
#pragma unroll
                    for (int c = 0; c < 32; ++c) sums[c] += more[c];
                }
                const uint32_t buffer_of_warp = ring + kStages * kStageBytes + (warp - 4) * kPieceBytes;
                if (p.out_is_f32) {
#pragma unroll
                    for (int c = 0; c < 16; ++c) words[c] = __float_as_uint(sums[c]);
                    put_piece<4>(p, &map_out, buffer_of_warp, lane, tile.token0 + quarter * 32, tile.col0 + c0, words);
                } else {
#pragma unroll
                    for (int c = 0; c < 16; ++c) words[c] = tc5::pack2(sums[2 * c], sums[2 * c + 1]);
                    put_piece<2>(p, &map_out, buffer_of_warp, lane, tile.token0 + quarter * 32, tile.col0 + c0, words);
                }
            }
        cluster_sync();      // nobody leaves while others read its shared memory
    }
    // nothing may be left in shared memory, or on its way out of it, when the block leaves
    if (warp >= 4 && lane == 0 && p.bulk_out) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    if (failed && threadIdx.x == 0 && p.error_flag) atomicExch(p.error_flag, 2);
    if (warp == 3) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// Tensor map of the output [rows, columns] (float or bfloat16) for pieces of 32 rows x 64 bytes; what lies outside is not written.
bool make_piece_map(CUtensorMap* map, void* pointer, uint64_t rows, uint64_t columns, bool wide) {
    tma::EncodeTiled encode = tma::encode_tiled();
    if (encode == nullptr) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)columns, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)columns * (wide ? 4 : 2)};
    const cuuint32_t box[2] = {wide ? 16u : 32u, 32u};
    const cuuint32_t ones[2] = {1, 1};
    return encode(map, wide ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, pointer, dims, strides, box, ones,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int COLS>
int launch_many(const CUtensorMap& map_x, const CUtensorMap& map_out, const void* w, long long w_pitch, ManyParams p, int inner, cudaStream_t stream) {
    CUtensorMap map_w;
    if (!make_map_f8(&map_w, w, (uint64_t)p.n, (uint64_t)inner, (uint64_t)w_pitch, COLS)) {
        llm_set_error("block_linear: the tensor maps could not be made");
        return LLM_REFUSED;
    }
    const int sms = llm_sm_count();
    p.row_tiles = (p.m + kTokens - 1) / kTokens;
    p.col_tiles = (p.n + COLS - 1) / COLS;
    const long long total = (long long)p.row_tiles * p.col_tiles;
    // row tiles whose rows of x stay in L2 together while W passes: at most 32 MiB of them
    const long long fit = (32LL << 20) / ((long long)kTokens * inner);
    p.row_group = (int)(fit < 1 ? 1 : fit < p.row_tiles ? fit : p.row_tiles);
    p.split = 1;
    if (COLS == 128)
        while (2 * p.split <= kMaxSplit && total * 2 * p.split <= sms && p.groups / (2 * p.split) >= 4) p.split *= 2;
    const size_t shared = shared_bytes(COLS);
    if (int status = llm_raise_shared_limit((const void*)gemm_block_scaled_many_kernel<COLS>, shared, "block_linear", true)) return status;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)((total < sms ? total : sms) * p.split), 1, 1);
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
    const cudaError_t status = cudaLaunchKernelEx(&config, gemm_block_scaled_many_kernel<COLS>, map_w, map_x, map_out, p);
    if (status != cudaSuccess) {
        llm_set_error("block_linear launch: %s", cudaGetErrorString(status));
        return (int)status;
    }
    return llm_check_launch("block_linear");
}

}  // namespace

// The product for rows in 8 bits (called by llm_block_linear, which has checked its arguments).
int llm_block_linear_many(const void* x, long long x_pitch, const float* x_scales, const void* w, long long w_pitch, const float* w_scales, void* out,
                          int out_is_f32, int m, int n, int inner, int early, int* error_flag, cudaStream_t stream) {
    ManyParams p = {};
    p.x_scales = x_scales;
    p.w_scales = w_scales;
    p.out = out;
    p.out_is_f32 = out_is_f32;
    p.m = m;
    p.n = n;
    p.groups = (inner + kBlock - 1) / kBlock;
    p.bulk_out = n % (out_is_f32 ? 4 : 8) == 0 && aligned16(out);
    p.early = early;
    p.error_flag = error_flag;
    CUtensorMap map_x, map_out;
    if (!make_map_f8(&map_x, x, (uint64_t)m, (uint64_t)inner, (uint64_t)x_pitch, kTokens) ||
        (p.bulk_out && !make_piece_map(&map_out, out, (uint64_t)m, (uint64_t)n, out_is_f32 != 0))) {
        llm_set_error("block_linear: the tensor maps could not be made");
        return LLM_REFUSED;
    }
    if (!p.bulk_out) map_out = map_x;      // not used
    // Tiles of 256 columns need 48 KiB a unit and 740 cycles for them, tiles of 128 need 32 KiB and 500: the wider ones unless the
    // narrower ones fill the SMs better by more than that.
    const long long sms = llm_sm_count(), rows = (m + kTokens - 1) / kTokens;
    const long long wide = (rows * ((n + 255) / 256) + sms - 1) / sms, narrow = (rows * ((n + 127) / 128) + sms - 1) / sms;
    if (2 * narrow < 3 * wide) return launch_many<128>(map_x, map_out, w, w_pitch, p, inner, stream);
    return launch_many<256>(map_x, map_out, w, w_pitch, p, inner, stream);
}
