// One row of keys and values into a page of a 4-bit cache (layout: sq_kv4.h), by the lanes of a wave.
//
// Per group of g elements: m = min x, s = fp16((max x - m) / 15), code = round((x - m) / s) in 0..15, the element then
// reads as s * code + m.  All steps in fp32 with one rounding each (the division included), so that the codes are those of
// any IEEE implementation.  An infinity or a NaN in a group makes its scale a NaN: the group reads as NaN.
//
// Division.  A group divides all its elements by one scale, so its reciprocal is worked out once (a Newton step on the
// hardware's, within one ulp: correctly rounded for every significand of fp16, checked one by one) and an element takes three
// operations instead of ten: q = d r, then q + (d - q s) r, which Markstein's theorem makes the correctly rounded quotient.
// All exchanges between lanes are data-parallel moves: a row's group lies in 4, 8 or 16 lanes, a word's codes in eight.
#pragma once
#include "sq_kv4.h"

#include <type_traits>

namespace sq {

template <int CTRL>
__device__ __forceinline__ uint32_t lane_move(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
}
template <int CTRL>
__device__ __forceinline__ float lane_move(float v) {
    return bit_cast<float>(lane_move<CTRL>(bit_cast<uint32_t>(v)));
}
// The value of the lane whose number differs by X (1, 2, 4 or 8).
template <int X>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
    if constexpr (X == 1) return lane_move<0xB1>(v);   // quad_perm 1,0,3,2
    if constexpr (X == 2) return lane_move<0x4E>(v);   // quad_perm 2,3,0,1
    if constexpr (X == 4) return lane_move<0x141>(lane_move<0x1B>(v));  // 3 apart, then 7 apart (row_half_mirror)
    return lane_move<0x128>(v);                        // row_ror:8
}

// What a row's group became: lanes that hold eight of its elements each agree on it.
struct Group {
    float s, m, r;  // scale, minimum, 1 / scale
    half_t sh, mh;
};

// The lowest and highest of pairs, a NaN left aside.
__device__ __forceinline__ half2_t pair_min(half2_t a, half2_t b) { return __builtin_elementwise_min(a, b); }
__device__ __forceinline__ half2_t pair_max(half2_t a, half2_t b) { return __builtin_elementwise_max(a, b); }

// Eight elements (of the lane's part of a group of g) -> the group and the eight codes, whole numbers.
template <int g>
__device__ __forceinline__ Group kv4_quantise8(half8_t x8, float (&code)[8]) {
    half2_t lo2 = {x8[0], x8[1]}, hi2 = lo2;
    float bad = 0.f;  // 0, or NaN where an element is no finite number
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const half2_t x = {x8[e], x8[e + 1]};
        lo2 = pair_min(lo2, x);
        hi2 = pair_max(hi2, x);
        bad = __builtin_amdgcn_fdot2(x, (half2_t){(half_t)0.f, (half_t)0.f}, bad, false);
    }
    float lo = fminf((float)lo2[0], (float)lo2[1]), hi = fmaxf((float)hi2[0], (float)hi2[1]);
    auto step = [&](auto ctrl) {
        constexpr int C = decltype(ctrl)::value;
        lo = fminf(lo, lane_move<C>(lo));
        hi = fmaxf(hi, lane_move<C>(hi));
        bad += lane_move<C>(bad);
    };
    step(std::integral_constant<int, 0xB1>{});
    step(std::integral_constant<int, 0x4E>{});
    if constexpr (g >= 64) step(std::integral_constant<int, 0x141>{});   // row_half_mirror: the other quad of eight lanes
    if constexpr (g >= 128) step(std::integral_constant<int, 0x140>{});  // row_mirror: the other eight
    Group q;
    q.sh = (half_t)((hi - lo) / 15.f + bad);
    q.mh = (half_t)lo;
    q.s = (float)q.sh;
    q.m = lo;
    const float r0 = __builtin_amdgcn_rcpf(q.s);
    q.r = q.s > 0.f ? __builtin_fmaf(__builtin_fmaf(-q.s, r0, 1.f), r0, r0) : 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float d = (float)x8[e] - q.m, c = d * q.r;
        const float quotient = __builtin_fmaf(__builtin_fmaf(-c, q.s, d), q.r, c);
        code[e] = __builtin_amdgcn_fmed3f(__builtin_rintf(quotient), 0.f, 15.f);
    }
    return q;
}
// Four codes as the bytes of a word.
__device__ __forceinline__ uint32_t four_bytes(float a, float b, float c, float d) {
    uint32_t w = __builtin_amdgcn_cvt_pk_u8_f32(a, 0, 0);
    w = __builtin_amdgcn_cvt_pk_u8_f32(b, 1, w);
    w = __builtin_amdgcn_cvt_pk_u8_f32(c, 2, w);
    return __builtin_amdgcn_cvt_pk_u8_f32(d, 3, w);
}

struct RowOut {  // where what the row reads as goes to, or null
    half_t *k, *v;
};

// D / 8 lanes have a row, eight elements k8 and v8 each from 8 (lane % (D / 8)) on; `live`: whether this lane's row is
// stored.
template <int D, int G>
__device__ __forceinline__ void kv4_store_row(uint8_t* rec, int row, half8_t k8, half8_t v8, bool live, const RowOut& hat) {
    constexpr int g = D / G, LPR = D / 8;
    const int sub = (threadIdx.x & 63) % LPR;
    const int quad = row >> 2, in_quad = row & 3;
    auto finish = [&](const Group& q, const float (&code)[8], half_t* to, int what) {
        if (!live) return;
        if (to) {
            half8_t y;
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = (half_t)(q.s * code[e] + q.m);
            *(half8_t*)(to + 8 * sub) = y;
        }
        if (sub % (g / 8) == 0) {
            half_t* const sm = (half_t*)(rec + 64 * D + 256 * G * what) + ((sub / (g / 8)) * 16 + quad) * 8 + in_quad;
            sm[0] = q.sh;
            sm[4] = q.mh;
        }
    };
    float code[8];
    // Keys: the lane's eight elements share words 2 p and 2 p + 1 of chunk sub % 4 with those of the lane four away.
    {
        const Group q = kv4_quantise8<g>(k8, code);
        const int h = (sub >> 2) & 1;
        const uint32_t w0 = four_bytes(code[0], code[4], code[1], code[5]) << (4 * h);
        const uint32_t w1 = four_bytes(code[2], code[6], code[3], code[7]) << (4 * h);
        const uint32_t o0 = lane_xor<4>(w0), o1 = lane_xor<4>(w1);
        if (live) *(uint32_t*)(rec + row * (D / 2) + ((sub & 3) * (D / 32) + 2 * (sub >> 3) + h) * 4) = h ? (w1 | o1) : (w0 | o0);
        finish(q, code, hat.k, 0);
    }
    // Values: a word has one element of each of eight lanes.  The lanes' words of eight codes are transposed in three
    // exchanges of halves, quarters and eighths.
    {
        const Group q = kv4_quantise8<g>(v8, code);
        uint32_t w = four_bytes(code[0], code[2], code[4], code[6]) | four_bytes(code[1], code[3], code[5], code[7]) << 4;
        // n, the lane's nibble in the words: elements 16 n + w (D = 128) or 16 (n % 4) + 8 (n / 4) + w
        const int n = D == 128 ? sub >> 1 : (sub >> 1 | (sub & 1) << 2);
        auto swap = [&](uint32_t other, uint32_t low, int shift, int bit) {
            w = bit ? (w & ~low) | ((other >> shift) & low) : (w & low) | ((other & low) << shift);
        };
        swap(lane_xor<2>(w), 0x0F0F0F0Fu, 4, n & 1);
        swap(lane_xor<4>(w), 0x00FF00FFu, 8, n & 2);
        swap(lane_xor<D == 128 ? 8 : 1>(w), 0x0000FFFFu, 16, n & 4);
        const int word = D == 128 ? n + 8 * (sub & 1) : n;
        if (live) *(uint32_t*)(rec + 32 * D + (quad * (D / 8) + word) * 16 + in_quad * 4) = w;
        finish(q, code, hat.v, 1);
    }
}

}  // namespace sq
