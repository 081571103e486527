// How tiles of fp16 key and value rows lie in LDS and are read as matrix operands (sq_attn.hip, sq_prefix_attn.hip,
// sq_evict.hip).
#pragma once
#include "sq_common.h"

namespace sq {

// Chunk permutations inside a tile row of D halves (D / 8 chunks of 16 bytes).
// K is read 128 bits wide by 32 lanes = rows at one chunk: 16 consecutive rows (256 bytes of LDS banks) must differ.
template <int D>
__device__ __forceinline__ int k_swz(int row) {
    return D == 128 ? (row & 15) : ((row & 7) ^ ((row >> 3) & 1));
}
// V is read 64 bytes of a row by 8 lanes, four consecutive rows by a transposing read: the rows' 64-byte pieces must differ.
template <int D>
__device__ __forceinline__ int v_swz(int row) {
    return D == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1);
}

typedef short short4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ short4_t lds_read_tr(const uint8_t* p) {
    typedef __attribute__((address_space(3))) short4_t* lp;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p));
}

// A pointer that is the same in all lanes, in scalar registers, for the direct loads.  A memory instruction may read a scalar
// register five wait states after a vector instruction has written it (v_readfirstlane is one), and the compiler does not
// count them in front of inline assembly: they are here.
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
    const uint64_t u = (uint64_t)(uintptr_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)u), hi = __builtin_amdgcn_readfirstlane((int)(u >> 32));
    uint64_t both = ((uint64_t)hi << 32) | lo;
    asm volatile("s_nop 4" : "+s"(both));
    return (const uint8_t*)(uintptr_t)both;
}

}  // namespace sq
