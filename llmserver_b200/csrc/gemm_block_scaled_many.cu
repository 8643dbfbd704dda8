// The product of gemm_block_scaled.cu for many tokens: y[m, n] = sum_b xs[m, b] ws[n / 128, b] (xq wq^T over block b of k), operands e4m3.
//
// Here the tokens are the MMA's M = 128 and 128 or 256 rows of W its N.  A lane of tensor memory is then a token, and what a block's sums
// are multiplied with is one number per thread and 128 rows of W, which the adders read from shared memory as one word a unit.  (With a
// token per column every thread has to read the numbers of all its columns: 64 KiB of registers filled from shared memory per unit of
// 128 x 128 x 128, 512 cycles beside the MMA's 256.)
//
// A block has its SM to itself and walks tiles c, c + blocks, ...; the ring of stages and the buffers of tensor memory run on across tiles.  Eight
// warps scale and add, 32 tokens by half the columns each.  A finished tile goes from registers through two KiB of shared memory per warp, so that
// it leaves in pieces of 32 bytes a row while the next piece is written.  Tiles of 128 columns, where they are few, split k over a cluster; the
// parts are added through distributed shared memory in the order of k.
//
// A unit of the ring is a block of 128 along k for tiles of 256 columns and two blocks for tiles of 128, 48 and 64 KiB: every unit costs each role its
// waits and signals, some 300 cycles, and both fill 256 columns of tensor memory.  (With units of a single block tiles of 128 columns took 620 cycles a
// block, 500 x 4096 -> 4096 14.2 us behind 8-bit rows and not 13.1.)
//
// What bounds it, in SM cycles for a unit of 128 x 256: the MMAs alone 513, with copies, waits and signals 540, with the adders' reads and 32768
// products and sums 670 in a loop of nothing else; this kernel 800.  Counted in time the power limit comes first: with random operands the SMs run
// at 1.3 to 1.4 GHz, and even the MMAs with their copies alone take 422 ns of the 580 of a unit.
// Behind 8-bit rows, over fresh operands for two seconds on end (and in a burst of a few milliseconds, before the power limit holds the clock down):
// 8192 x 4096 -> 24576 856 us, 1926 TFLOP/s (756); 500 x 4096 -> 4096 14.0 us (12.8); 100 x 4096 -> 24576 24.3 us, W at 4.1 TB/s (22.3).
// Sixteen adders of half the columns take 830 to 1050 cycles, reads of 16 columns at a time 980, and sums kept as single numbers 1440 (they spill).
//
// Roles, bounded waits and the treatment of ragged sizes are those of gemm_block_scaled.cu.
#include "block_scaled_mma.cuh"

namespace {

using namespace block_scaled;

constexpr int kTokens = 128;          // per tile (UMMA M)
constexpr int kAdders = 8;            // warps; an adder has 32 tokens and half the columns
constexpr int kThreads = 128 + 32 * kAdders;
constexpr int kBuffers = 2;           // of 256 columns of tensor memory, a unit's sums
constexpr int kRun = 4;               // most units whose scales are handed over together: a wait costs 100 cycles
constexpr int kMaxStages = 4;
constexpr int kMaxSplit = 4;
constexpr int kScaleSlots = 2;        // runs of units whose scales wait to be used; another is on its way from memory
constexpr uint32_t kXBytes = kTokens * kBlock;
constexpr int kPieceRow = 32;         // bytes of a row that leave together
constexpr uint32_t kPieceBytes = 32 * kPieceRow;

struct ManyParams {
    const float* x_scales;            // [m][groups]
    const float* w_scales;            // [ceil(n / 128)][groups]
    void* out;
    int m, n, groups, units;          // blocks of 128 along k, and units of them
    int row_tiles, col_tiles, row_group;      // row tiles that are walked together for each column tile
    int split;
    int early;                        // W may be asked for before the kernel in front is complete
    int* error_flag;
};

// A unit is 128 of k for tiles of 256 columns and 256 of k, two blocks, for tiles of 128.
constexpr int blocks_of(int cols) { return 256 / cols; }
constexpr uint32_t stage_bytes(int cols) { return (uint32_t)blocks_of(cols) * (kXBytes + (uint32_t)cols * kBlock); }
constexpr int stages_of(int cols) { return cols == 128 ? 3 : 4; }
constexpr int lap_of(int cols) { return cols == 128 ? 6 : 4; }      // units after which stages and buffers are where they were
constexpr uint32_t shared_bytes(int cols) { return stages_of(cols) * stage_bytes(cols) + kAdders * 2 * kPieceBytes + 1024; }

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
    int t, unit, first, last;
    Tile tile;
    __device__ __forceinline__ void begin(const ManyParams& p, int t0, int from, int to) {
        t = t0, unit = first = from, last = to;
        tile = tile_of<COLS>(p, t);
    }
    __device__ __forceinline__ void step(const ManyParams& p, int stride, int total) {
        if (++unit < last) return;
        unit = first;
        t += stride;
        if (t < total) tile = tile_of<COLS>(p, t);
    }
};

// 32 bytes of each of a warp's 32 rows, through a KiB of shared memory, of which a warp has two: a lane hands in its row's; where the rows of the output begin at
// multiples of 16 bytes the piece leaves as one bulk store, which leaves out what does not exist, else two lanes store a row's two 16-byte words
// number by number.
template <int ELEMENT, bool BULK>
__device__ __forceinline__ void put_piece(const ManyParams& p, const CUtensorMap* map_out, uint32_t buffer, int lane, int row0, int column,
                                          const uint32_t (&words)[8]) {
    if (BULK) {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");      // the piece that lay here has been read
        __syncwarp();
    }
#pragma unroll
    for (int c = 0; c < 2; ++c)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(buffer + lane * kPieceRow + c * 16), "r"(words[4 * c]), "r"(words[4 * c + 1]),
                     "r"(words[4 * c + 2]), "r"(words[4 * c + 3]) : "memory");
    if (BULK) {
        tma::fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
            if (row0 < p.m && column < p.n)
                asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
                             ::"l"(map_out), "r"(buffer), "r"(column), "r"(row0) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");      // an empty one too: the groups are counted
        }
        return;
    }
    __syncwarp();
    constexpr int kEach = 16 / ELEMENT;
    const int c = lane & 1, at = column + c * kEach;
#pragma unroll
    for (int it = 0; it < 2; ++it) {
        const int row = it * 16 + (lane >> 1);
        uint32_t w[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(buffer + row * kPieceRow + c * 16) : "memory");
        if (row0 + row >= p.m) continue;
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

// Columns FIRST to FIRST + COUNT of this lane's row, held as pairs, piece by piece.
template <int COUNT, int ELEMENT, bool BULK>
__device__ __forceinline__ void put_row(const ManyParams& p, const CUtensorMap* map_out, uint32_t buffer, int lane, int row0, int column,
                                        const uint64_t (&v)[COUNT / 2]) {
    constexpr int kEach = kPieceRow / ELEMENT;
#pragma unroll
    for (int c0 = 0; c0 < COUNT; c0 += kEach) {
        uint32_t words[8];
#pragma unroll
        for (int c = 0; c < kEach; c += 2) {
            float lo, hi;
            tc5::halves_of(v[(c0 + c) / 2], lo, hi);
            if (ELEMENT == 4) words[c] = __float_as_uint(lo), words[c + 1] = __float_as_uint(hi);
            else words[c / 2] = tc5::pack2(lo, hi);
        }
        put_piece<ELEMENT, BULK>(p, map_out, buffer + c0 / kEach % 2 * kPieceBytes, lane, row0, column + c0, words);
    }
}

// COLS: columns of a tile; ELEMENT: bytes of a number of the output; BULK: its rows begin at multiples of 16 bytes.
template <int COLS, int ELEMENT, bool BULK>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_block_scaled_many_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                                  const __grid_constant__ CUtensorMap map_out, const ManyParams p) {
    constexpr int kStages = stages_of(COLS), kLap = lap_of(COLS), kBlocks = blocks_of(COLS), kWidth = COLS / 2;
    constexpr uint32_t kStageBytes = stage_bytes(COLS), kWBytes = COLS * kBlock, kUnitW = kBlocks * kXBytes;      // the last: where a stage's W begins
    constexpr bool kSplits = COLS == 128;      // the narrow tiles alone
    static_assert(kStages <= kMaxStages && kLap % kStages == 0 && kLap % kBuffers == 0, "the barriers are enough, and a lap is whole");
    extern __shared__ unsigned char many_shared[];
    __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], sums_bars[2][kBuffers],
        scale_full[kScaleSlots], scale_empty[kScaleSlots];
    __shared__ float scales[kScaleSlots][kRun][2][kTokens];      // of a unit's two blocks of W: each token's times W's
    __shared__ uint32_t tmem_slot;
    __shared__ int failed;
    const uint32_t ring = (tma::smem_u32(many_shared) + 1023u) & ~1023u;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = kSplits && p.split > 1 ? (int)cluster_rank() : 0, in_cluster = kSplits ? p.split : 1;
    const int total = p.row_tiles * p.col_tiles, stride = (int)gridDim.x / in_cluster, t0 = (int)blockIdx.x / in_cluster;
    const int first = (int)((long long)p.units * rank / in_cluster), last = (int)((long long)p.units * (rank + 1) / in_cluster);
    const int tiles = (total - t0 + stride - 1) / stride, count = tiles * (last - first);      // this block's units
    Walk<COLS> walk;
    walk.begin(p, t0, first, last);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            tma::mbar_init(tma::smem_u32(&full[s]), 1);
            tma::mbar_init(tma::smem_u32(&empty[s]), 1);
        }
        for (int b = 0; b < kBuffers; ++b) {
            tma::mbar_init(tma::smem_u32(&sums_bars[0][b]), 1);
            tma::mbar_init(tma::smem_u32(&sums_bars[1][b]), kAdders);
        }
        for (int s = 0; s < kScaleSlots; ++s) {
            tma::mbar_init(tma::smem_u32(&scale_full[s]), 1);
            tma::mbar_init(tma::smem_u32(&scale_empty[s]), kAdders);
        }
        tma::mbar_fence_init();
        failed = 0;
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
    }
    if (threadIdx.x == 0 && p.early) {
        Walk<COLS> ahead = walk;
        for (int s = 0; s < kStages && s < count; ++s) {
            tma::mbar_expect_tx(tma::smem_u32(&full[s]), kStageBytes);
#pragma unroll
            for (int k = 0; k < kBlocks; ++k)
                tma::load_2d(ring + s * kStageBytes + kUnitW + k * kWBytes, &map_w, tma::smem_u32(&full[s]), (ahead.unit * kBlocks + k) * kBlock, ahead.tile.col0);
            ahead.step(p, stride, total);
        }
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
        if (elect_one()) {
            bool ok = true;
            uint32_t lap = 0;      // of stages and buffers; a stage's barriers complete kLap / kStages times in it
            for (int i0 = 0; i0 < count && ok; i0 += kLap, ++lap) {
#pragma unroll
                for (int s = 0; s < kLap; ++s) {
                    const int at = s % kStages;
                    const uint32_t stage = ring + at * kStageBytes, bar = tma::smem_u32(&full[at]), turn = lap * (kLap / kStages) + s / kStages;
                    if (i0 + s >= count) break;
                    if (turn > 0 && !(ok = tma::mbar_wait(tma::smem_u32(&empty[at]), (turn & 1) ^ 1))) break;
                    if (!p.early || turn > 0) tma::mbar_expect_tx(bar, kStageBytes);
#pragma unroll
                    for (int k = 0; k < kBlocks; ++k) {      // what lies beyond the last of k is zeros
                        const int x = (walk.unit * kBlocks + k) * kBlock;
                        if (!p.early || turn > 0) tma::load_2d(stage + kUnitW + k * kWBytes, &map_w, bar, x, walk.tile.col0);
                        tma::load_2d(stage + k * kXBytes, &map_x, bar, x, walk.tile.token0);
                    }
                    walk.step(p, stride, total);
                }
            }
            // the last MMAs signal this block's barriers: it may not leave before they have
            for (int back = count < kStages ? count : kStages; back > 0 && ok; --back)
                ok = tma::mbar_wait(tma::smem_u32(&empty[(count - back) % kStages]), ((count - back) / kStages) & 1);
            if (!ok) failed = 1;
        }
    } else if (warp == 1) {
        // A lap is written out, so that every place and buffer is a constant, and one lane walks it: with places counted up beside the warp's vote a
        // unit took this warp 390 cycles with one wait and no work for anybody else, like this 297.
        if (elect_one()) {
            const uint32_t idesc = instruction_f8(kTokens, COLS);
            const uint64_t desc_x = tc5::desc_k_major(ring, 1024u), desc_w = tc5::desc_k_major(ring + kUnitW, 1024u);
            bool ok = true;
            uint32_t lap = 0;
            for (int i0 = 0; i0 < count && ok; i0 += kLap, ++lap) {
#pragma unroll
                for (int s = 0; s < kLap; ++s) {
                    const int at = s % kStages, b = s % kBuffers;
                    const uint32_t turn = lap * (kLap / kBuffers) + s / kBuffers;      // of the buffer
                    if (i0 + s >= count) break;
                    ok = tma::mbar_wait(tma::smem_u32(&full[at]), (lap * (kLap / kStages) + s / kStages) & 1);
                    if (ok && (s >= kBuffers || lap > 0)) ok = tma::mbar_wait(tma::smem_u32(&sums_bars[1][b]), (turn & 1) ^ 1);
                    if (!ok) break;
                    tc5::fence_after();
#pragma unroll
                    for (int k = 0; k < kBlocks * (kBlock / 32); ++k) {
                        const int block = k / (kBlock / 32), in_block = k % (kBlock / 32);
                        // descriptors hold addresses in units of 16 bytes
                        const uint64_t x_at = (at * kStageBytes + block * kXBytes) >> 4, w_at = (at * kStageBytes + block * kWBytes) >> 4;
                        mma_f8(tmem + b * 256 + block * COLS, desc_x + x_at + in_block * 2, desc_w + w_at + in_block * 2, idesc, in_block > 0);
                    }
                    tc5::mma_commit(tma::smem_u32(&sums_bars[0][b]));
                    tc5::mma_commit(tma::smem_u32(&empty[at]));
                }
            }
            if (!ok) failed = 1;
        }
    } else if (warp == 2) {
        // A lane's four tokens' scales times W's, asked for a run of units before: up to kRun units of one tile.  (Addresses are made once a tile: with
        // them and their bounds made for each unit a unit took 20 cycles more.)
        const int col_blocks = (p.n + 127) / 128;
        const float *x_from[4], *w_from[2 / kBlocks];
        float x_scale[kRun][kBlocks][4], w_scale[kRun][2];
        int t = t0, next = last;      // the tile and the unit to ask for next
        auto ask = [&](int units) {
            if (next == last) {      // a new tile; what lies outside the matrices reads something that does not
                const Tile tile = tile_of<COLS>(p, t);
#pragma unroll
                for (int j = 0; j < 4; ++j) x_from[j] = p.x_scales + (size_t)min(tile.token0 + j * 32 + lane, p.m - 1) * p.groups;
#pragma unroll
                for (int h = 0; h < 2 / kBlocks; ++h) w_from[h] = p.w_scales + (size_t)min(tile.col0 / 128 + h, col_blocks - 1) * p.groups;
                t += stride;
                next = first;
            }
#pragma unroll
            for (int d = 0; d < kRun; ++d)
                if (d < units) {
#pragma unroll
                    for (int k = 0; k < kBlocks; ++k) {      // beyond the last block of k there are zeros to be multiplied
                        const int group = (next + d) * kBlocks + k;
                        const bool there = kBlocks == 1 || group < p.groups;
#pragma unroll
                        for (int h = 0; h < 2 / kBlocks; ++h) w_scale[d][kBlocks == 1 ? h : k] = there ? w_from[h][group] : 0.0f;
#pragma unroll
                        for (int j = 0; j < 4; ++j) x_scale[d][k][j] = there ? x_from[j][group] : 0.0f;
                    }
                }
            next += units;
        };
        int units = min(kRun, last - first);      // of the run that was asked for
        if (count > 0) ask(units);
        bool ok = true;
        Turn slot;
        for (int i = 0, run = 0; i < count && ok; ++run) {
            if (run >= kScaleSlots) ok = __all_sync(0xffffffffu, tma::mbar_wait(tma::smem_u32(&scale_empty[slot.at]), slot.parity ^ 1));
            if (!ok) break;
#pragma unroll
            for (int d = 0; d < kRun; ++d)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < 4; ++j) scales[slot.at][d][h][j * 32 + lane] = x_scale[d][kBlocks == 1 ? 0 : h][j] * w_scale[d][h];
            i += units;
            units = next == last ? min(kRun, last - first) : min(kRun, last - next);
            if (i < count) ask(units);
            __syncwarp();
            if (lane == 0) tma::mbar_arrive(tma::smem_u32(&scale_full[slot.at]));
            slot.step(kScaleSlots);
        }
        if (!ok) failed = 1;
    } else if (warp >= 4) {
        const int quarter = warp & 3, share = (warp - 4) >> 2;      // its lanes of tensor memory, its columns
        const uint32_t address = tmem + ((uint32_t)(quarter * 32) << 16) + share * kWidth;
        uint64_t sums[kWidth / 2];      // pairs of numbers, which one instruction adds to
#pragma unroll
        for (int c = 0; c < kWidth / 2; ++c) sums[c] = 0;
        // Addresses and parities go on by additions, in registers of the lanes, which the shuffle keeps them in: with places counted up and multiplied
        // with sizes, in the warp's uniform registers, a unit of 256 columns took 885 cycles and not 825.
        const uint32_t vary = (uint32_t)__shfl_sync(0xffffffffu, 0, lane);      // 0
        const uint32_t bars = tma::smem_u32(&sums_bars[0][0]) + vary, my_scales = tma::smem_u32(&scales[0][0][kBlocks == 1 ? share : 0][quarter * 32 + lane]);
        uint32_t bar = bars, parity = vary, from = address;      // of the buffer: sums_full's address
        bool ok = true;
        Turn slot;
        for (int t = t0; t < total && ok; t += stride) {
            for (int unit = first; unit < last && ok; unit += kRun) {
                uint32_t scale_at = my_scales + slot.at * (uint32_t)sizeof(scales[0]);
                ok = tma::mbar_wait(tma::smem_u32(&scale_full[slot.at]), slot.parity);
#pragma unroll 1
                for (int units = min(kRun, last - unit); units > 0; --units) {
                    float scale[kBlocks];
#pragma unroll
                    for (int k = 0; k < kBlocks; ++k) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(scale[k]) : "r"(scale_at + k * kTokens * 4) : "memory");
                    scale_at += (uint32_t)sizeof(scales[0][0]);
                    ok = __all_sync(0xffffffffu, ok && tma::mbar_wait(bar, parity));
                    if (!ok) break;
                    tc5::fence_after();
                    // read from tensor memory at a time: 32 columns, or with half the sums to hold a block's 64
                    constexpr int kPart = kBlocks == 1 ? 32 : 64;
#pragma unroll
                    for (int part = 0; part < 128; part += kPart) {
                        const int k = kBlocks == 1 ? 0 : part / kWidth, first_column = kBlocks == 1 ? part : 0;
                        uint32_t r[kPart / 32][32];
#pragma unroll
                        for (int c = 0; c < kPart; c += 32) tmem_ask<32>(from + k * COLS + first_column + c, r[c / 32]);
#pragma unroll
                        for (int c = 0; c < kPart; c += 32) tmem_wait<32>(r[c / 32]);
                        if (part + kPart == 128) {      // all of the buffer is in registers
                            tc5::fence_before();
                            __syncwarp();
                            if (lane == 0) tma::mbar_arrive(bar + kBuffers * 8);
                        }
                        const uint64_t both = tc5::pair_of(scale[k], scale[k]);
#pragma unroll
                        for (int c = 0; c < kPart; c += 2) {
                            uint64_t& sum = sums[(first_column + c) / 2];
                            sum = tc5::fma_pair(tc5::pair_of(__uint_as_float(r[c / 32][c % 32]), __uint_as_float(r[c / 32][c % 32 + 1])), both, sum);
                        }
                    }
                    bar += 8, from += 256;
                    if (bar == bars + kBuffers * 8) bar = bars, from = address, parity ^= 1;
                }
                __syncwarp();
                if (lane == 0) tma::mbar_arrive(tma::smem_u32(&scale_empty[slot.at]));
                slot.step(kScaleSlots);
            }
            if (kSplits && p.split > 1) break;      // one tile, whose parts are added below
            if (!ok) break;
            const Tile tile = tile_of<COLS>(p, t);
            put_row<kWidth, ELEMENT, BULK>(p, &map_out, ring + kStages * kStageBytes + (warp - 4) * 2 * kPieceBytes, lane, tile.token0 + quarter * 32,
                                           tile.col0 + share * kWidth, sums);
#pragma unroll
            for (int c = 0; c < kWidth / 2; ++c) sums[c] = 0;
        }
        if (!ok) failed = 1;
        if (kSplits && p.split > 1 && ok) {
            // all copies into the ring and all MMAs that read it are complete: [column][token]
#pragma unroll
            for (int c = 0; c < kWidth; c += 2) {
                float lo, hi;
                tc5::halves_of(sums[c / 2], lo, hi);
                const uint32_t place = ring + ((share * kWidth + c) * kTokens + quarter * 32 + lane) * 4;
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(place), "f"(lo) : "memory");
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(place + kTokens * 4), "f"(hi) : "memory");
            }
        }
    }
    __syncwarp();
    tc5::fence_before();
    __syncthreads();
    tc5::fence_after();
    if (failed)      // a wait ran out: copies that may still be in flight get time to land
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    if (warp == 3) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    if (kSplits && p.split > 1) {
        cluster_sync();
        const Tile tile = tile_of<COLS>(p, t0);
        // pieces of 32 tokens by 32 columns, dealt to the cluster's adders
        constexpr int kEach = 32;
        if (warp >= 4 && !failed)
            for (int piece = rank + (warp - 4) * p.split; piece < 4 * (COLS / kEach); piece += kAdders * p.split) {
                const int quarter = piece & 3, c0 = (piece >> 2) * kEach;
                float sums[kEach];
                uint64_t pairs[kEach / 2];
                const uint32_t place = ring + (c0 * kTokens + quarter * 32 + lane) * 4;
#pragma unroll
                for (int c = 0; c < kEach; ++c) sums[c] = load_peer(place + c * kTokens * 4, 0);
                for (int peer = 1; peer < p.split; ++peer) {
                    float more[kEach];      // asked for together
#pragma unroll
                    for (int c = 0; c < kEach; ++c) more[c] = load_peer(place + c * kTokens * 4, peer);
#pragma unroll
                    for (int c = 0; c < kEach; ++c) sums[c] += more[c];
                }
#pragma unroll
                for (int c = 0; c < kEach; c += 2) pairs[c / 2] = tc5::pair_of(sums[c], sums[c + 1]);
                put_row<kEach, ELEMENT, BULK>(p, &map_out, ring + kStages * kStageBytes + (warp - 4) * 2 * kPieceBytes, lane, tile.token0 + quarter * 32,
                                              tile.col0 + c0, pairs);
            }
        cluster_sync();      // nobody leaves while others read its shared memory
    }
    // nothing may be left in shared memory, or on its way out of it, when the block leaves
    if (BULK && warp >= 4 && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    if (failed && threadIdx.x == 0 && p.error_flag) atomicExch(p.error_flag, 2);
}

// Tensor map of the output [rows, columns] (float or bfloat16) for pieces of 32 rows x 32 bytes; what lies outside is not written.
bool make_piece_map(CUtensorMap* map, void* pointer, uint64_t rows, uint64_t columns, bool wide) {
    tma::EncodeTiled encode = tma::encode_tiled();
    if (encode == nullptr) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)columns, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)columns * (wide ? 4 : 2)};
    const cuuint32_t box[2] = {(cuuint32_t)kPieceRow / (wide ? 4 : 2), 32u};
    const cuuint32_t ones[2] = {1, 1};
    return encode(map, wide ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, pointer, dims, strides, box, ones,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int COLS, int ELEMENT, bool BULK>
int launch_many(const CUtensorMap& map_x, const CUtensorMap& map_out, const void* w, long long w_pitch, ManyParams p, int inner, cudaStream_t stream) {
    CUtensorMap map_w;
    if (!make_map_f8(&map_w, w, (uint64_t)p.n, (uint64_t)inner, (uint64_t)w_pitch, COLS)) {
        llm_set_error("block_linear: the tensor maps could not be made");
        return LLM_REFUSED;
    }
    const int places = llm_sm_count();
    p.row_tiles = (p.m + kTokens - 1) / kTokens;
    p.col_tiles = (p.n + COLS - 1) / COLS;
    p.units = (p.groups + blocks_of(COLS) - 1) / blocks_of(COLS);
    const long long total = (long long)p.row_tiles * p.col_tiles;
    // row tiles whose rows of x stay in L2 together while W passes: at most 32 MiB of them
    const long long fit = (32LL << 20) / ((long long)kTokens * inner);
    p.row_group = (int)(fit < 1 ? 1 : fit < p.row_tiles ? fit : p.row_tiles);
    p.split = 1;
    if (COLS == 128)
        while (2 * p.split <= kMaxSplit && total * 2 * p.split <= places && p.units / (2 * p.split) >= 2) p.split *= 2;
    const size_t shared = shared_bytes(COLS);
    if (int status = llm_raise_shared_limit((const void*)gemm_block_scaled_many_kernel<COLS, ELEMENT, BULK>, shared, "block_linear", true)) return status;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)((total < places ? total : places) * p.split), 1, 1);
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
    const cudaError_t status = cudaLaunchKernelEx(&config, gemm_block_scaled_many_kernel<COLS, ELEMENT, BULK>, map_w, map_x, map_out, p);
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
    p.m = m;
    p.n = n;
    p.groups = (inner + kBlock - 1) / kBlock;
    const bool bulk = n % (out_is_f32 ? 4 : 8) == 0 && aligned16(out);
    p.early = early;
    p.error_flag = error_flag;
    CUtensorMap map_x, map_out;
    if (!make_map_f8(&map_x, x, (uint64_t)m, (uint64_t)inner, (uint64_t)x_pitch, kTokens) ||
        (bulk && !make_piece_map(&map_out, out, (uint64_t)m, (uint64_t)n, out_is_f32 != 0))) {
        llm_set_error("block_linear: the tensor maps could not be made");
        return LLM_REFUSED;
    }
    if (!bulk) map_out = map_x;      // not used
    // A block of k of a tile of 256 columns takes 800 cycles, of 128 columns 530: the wider ones unless the narrower ones fill the SMs better by that
    // (384 x 4096 -> 6144, one tile an SM either way: 17.1 us narrow, 22.3 wide; 900 rows, 3 and 2: 35.8 and 37.9; 700 rows, 2 and 1: 28.9 and 23.5).
    const long long sms = llm_sm_count(), rows = (m + kTokens - 1) / kTokens;
    const long long wide = (rows * ((n + 255) / 256) + sms - 1) / sms, narrow = (rows * ((n + 127) / 128) + sms - 1) / sms;
    const int form = 2 * narrow <= 3 * wide ? 0 : 1;
    using Launch = int (*)(const CUtensorMap&, const CUtensorMap&, const void*, long long, ManyParams, int, cudaStream_t);
    static const Launch launches[2][2][2] = {
        {{launch_many<128, 2, false>, launch_many<128, 2, true>}, {launch_many<128, 4, false>, launch_many<128, 4, true>}},
        {{launch_many<256, 2, false>, launch_many<256, 2, true>}, {launch_many<256, 4, false>, launch_many<256, 4, true>}}};
    return launches[form][out_is_f32 != 0][bulk](map_x, map_out, w, w_pitch, p, inner, stream);
}
