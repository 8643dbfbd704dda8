// What the products of e4m3 operands with a scale per block share: places in rings, the MMA and its descriptor, tensor-memory loads that are waited
// for together, cluster helpers and tensor maps of bytes.
#pragma once

#include "block_scaled.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace block_scaled {

// A place in a ring and the parity of its turn.  It moves by additions: a division of integers is a hundred cycles for a role that one warp
// plays, and with five of them per unit a unit took 1150 cycles, whatever its size.
struct Turn {
    int at = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void step(int size) {
        if (++at == size) at = 0, parity ^= 1;
    }
};

__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// e4m3 x e4m3 -> float32, both operands K-major.
__device__ __forceinline__ uint32_t instruction_f8(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

// One lane of the warp, chosen by the hardware.  What it issues is then known to come from one thread, with operands that the whole
// warp shares: under `lane == 0` each MMA and copy cost 70 to 200 cycles more, and a unit 880 however small.
__device__ __forceinline__ bool elect_one() {
    uint32_t elected;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
    return elected != 0;
}

// COUNT columns of this warp's rows; the caller waits once for all loads that it has issued.
template <int COUNT>
__device__ __forceinline__ void tmem_ask(uint32_t address, uint32_t (&r)[COUNT]);
template <>
__device__ __forceinline__ void tmem_ask<16>(uint32_t address, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(address) : "memory");
}
template <>
__device__ __forceinline__ void tmem_ask<32>(uint32_t address, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
                   "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
                   "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(address) : "memory");
}
// The array is an operand, so that nothing reads it before the wait.
template <int COUNT>
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[COUNT]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < COUNT; ++i) asm volatile("" : "+r"(r[i]));
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

__device__ __forceinline__ float load_peer(uint32_t local_address, uint32_t rank) {
    uint32_t remote;
    float value;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_address), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(value) : "r"(remote) : "memory");
    return value;
}

// Tensor map of bytes [rows, columns] with `pitch` bytes between rows, box = [box_rows, 128 columns], 128-byte swizzle, zeros outside.
inline bool make_map_f8(CUtensorMap* map, const void* pointer, uint64_t rows, uint64_t columns, uint64_t pitch, uint32_t box_rows) {
    tma::EncodeTiled encode = tma::encode_tiled();
    if (encode == nullptr) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)columns, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)pitch};
    const cuuint32_t box[2] = {(cuuint32_t)kBlock, box_rows};
    const cuuint32_t ones[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(pointer), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace block_scaled
