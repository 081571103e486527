// A key/value cache held in 4 bits: what its kernels share.
//
// The cache is a pool of pages of 64 rows; pool [pages][H][record] bytes, one record per page and key/value head:
//   offset        what
//   0             keys, uint32 [64][4][D/32]: nibble n of word w of chunk c = element
//                 64 (w/2) + 32 (n%2) + 8 c + 4 (n/2%2) + 2 (w%2) + n/4
//   32 D          values, uint32 [16][D/8][4]: row 4 a + t, word w; nibble n = element 16 n + w (D = 128) or
//                 16 (n%4) + 8 (n/4) + w (D = 64)
//   64 D          fp16 [D/g][16][2][4] of the keys: scales and minima of rows 4 a .. 4 a + 3 by group
//   + 256 D/g     the same of the values
//   + 256 D/g     fp16 [2][D]: largest and smallest key of the page, by element, as the rows were given
// The orders are those in which the attention's matrix operands lie in registers: a 16-byte load of the keys is a
// lane's share of a row for two or four products, a 16-byte load of the values is four rows of the same eight columns.
#pragma once
#include "sq_common.h"

namespace sq {

constexpr int KV4_PAGE = 64;

__host__ __device__ constexpr int kv4_record_bytes(int D, int g) { return 68 * D + 512 * (D / g); }

// The cache as a kernel sees it.  Whatever the tables and lengths on the device say, nothing outside the pool is
// read or written: a page outside [0, num_pages) does not exist, and neither do rows that the table has no place for.
struct Kv4Cache {
    uint8_t* pool;
    const int* table;    // [B][table_stride], `width` entries used
    const int* lengths;  // [B], rows of a sequence with those of this call
    const int* starts;   // [B + 1] or null: `each` tokens per sequence
    int B, T, H, num_pages, width, table_stride, each;
};

// Of a sequence's rows, those that its table has places for.
__device__ __forceinline__ int kv4_inside(const Kv4Cache& c, int rows) {
    const int most = c.width * KV4_PAGE;
    return rows < 0 ? 0 : (rows > most ? most : rows);
}
__device__ __forceinline__ int kv4_length(const Kv4Cache& c, int b) { return kv4_inside(c, c.lengths[b]); }

// First token of sequence b and behind its last, inside [0, T].
__device__ __forceinline__ void kv4_tokens(const Kv4Cache& c, int b, int& first, int& count) {
    if (c.starts) {
        const int s0 = c.starts[b], s1 = c.starts[b + 1];
        first = s0 < 0 ? 0 : (s0 > c.T ? c.T : s0);
        const int end = s1 > c.T ? c.T : s1;
        count = end > first ? end - first : 0;
    } else {
        first = b * c.each;
        count = c.each;
    }
}

__device__ __forceinline__ int imax(int a, int b) { return a > b ? a : b; }

// Inclusive sum over the lanes of a wave, by data-parallel moves (a shuffle through LDS costs 60 cycles a step).
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);   // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);   // row_shr:2
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);   // row_shr:4
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);   // row_shr:8
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
    return v;
}
__device__ __forceinline__ int wave_sum(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }

// A value and that of the lane 16 (32) away, on every lane.
__device__ __forceinline__ void pair16(float v, float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(bit_cast<uint32_t>(v), bit_cast<uint32_t>(v), false, false);
    a = bit_cast<float>((uint32_t)r[0]);
    b = bit_cast<float>((uint32_t)r[1]);
}
__device__ __forceinline__ void pair32(float v, float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(bit_cast<uint32_t>(v), bit_cast<uint32_t>(v), false, false);
    a = bit_cast<float>((uint32_t)r[0]);
    b = bit_cast<float>((uint32_t)r[1]);
}
__device__ __forceinline__ float rows_sum(float v) {  // over the four lanes of a column
    float a, b;
    pair16(v, a, b);
    pair32(a + b, a, b);
    return a + b;
}
__device__ __forceinline__ float rows_max(float v) {
    float a, b;
    pair16(v, a, b);
    pair32(fmaxf(a, b), a, b);
    return fmaxf(a, b);
}
}  // namespace sq
