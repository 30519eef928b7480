// row_tiles.cuh — rows brought to shared memory by cp.async and read back as operands of mma.sync.
#pragma once

#include <stdint.h>

namespace drkv {

// A tile is rows of ROWB bytes in shared memory; chunks of 16 bytes are permuted so that both access patterns are free
// of bank conflicts: rows (g) x chunks (t) for K, rows (2t) x chunks (g) for V, g = lane / 4, t = lane % 4.
template <int ROWB>
__device__ __forceinline__ uint32_t tile_off(int row, int chunk) {
    if (ROWB == 64)                    // two rows share a 128-byte line
        return (row >> 1) * 128 + (((((row & 1) << 2) | chunk) ^ (((row >> 1) & 3) << 1)) << 4);
    return row * ROWB + ((chunk ^ ((((row >> 1) & 3) << 1) ^ ((row & 1) << 2))) << 4);
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
// 16 bytes from global to shared memory; the second form writes zeros where !live
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16_or_zero(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

}  // namespace drkv
