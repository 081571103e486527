// What the kernels of attention over a 4-bit cache share (sq_kv4_attn.hip: few rows; sq_kv4_chunk.hip: many).
#pragma once
#include "sq_kv4.h"

#include <type_traits>

namespace sq {

template <int N>
using Int = std::integral_constant<int, N>;

struct Kv4AttnArgs {
    Kv4Cache c;
    const half_t* q;
    half_t* out;          // [T][share * H][D]
    const int* selected;  // [B][H][count] or null
    float* ws;            // partial states, or null: no sequence is split
    long q_ts, q_hs;      // element strides of q over token and head
    int share;            // query heads of a key/value head
    int count;
    float scale;          // sm_scale * log2(e)
    const half_t* k_new;  // the row of every sequence's one token, stored by the kernel first, or null
    const half_t* v_new;
    long k_ts, k_hs, v_ts, v_hs;
    int rows_min, rows_max;  // sequences with fewer or more rows (token, query head) per head are another launch's (with starts)
};

// How a launch's work is dealt.  A tile is R of the rows (token, query head) of a sequence and key/value head; a
// workgroup takes one tile over a share of its pages.  The share's length follows from the lengths on the device: the pages
// of all tiles over 256 per_cu workgroups, `least` at the fewest.
struct Deal {
    int per_cu, least;
    __host__ __device__ int wgs() const { return 256 * per_cu; }
};
constexpr long KA_MOST_PAGES = 1l << 38;  // of all tiles, that `deal` can count: beyond it nothing is shared
struct Piece {
    int b, tile, head, share, shares;  // share of how many
    int slot;                          // where its partial state goes (shares > 1)
    int first, count, len;             // tokens of the sequence, and its rows inside the table
    int end;                           // behind the row of its last token (which the table may have no place for)
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// A sequence's tokens, rows (see Piece), pages and tiles.
struct Sizes {
    int first, count, len, end, pages, tiles;
};
template <int R>
__device__ __forceinline__ Sizes sizes_of(const Kv4AttnArgs& a, int b) {
    Sizes s = {0, 0, 0, 0, 0, 0};
    if (b < a.c.B) {
        kv4_tokens(a.c, b, s.first, s.count);
        s.end = imax(a.c.lengths[b], 0);
        s.len = kv4_inside(a.c, s.end);
        s.pages = ceil_div(s.len, KV4_PAGE);
        if (a.selected) s.pages = imin(s.pages, a.count);
        const int rows = s.count * a.share;
        s.tiles = rows >= a.rows_min && rows <= a.rows_max ? ceil_div(rows, R) * a.c.H : 0;
    }
    return s;
}

// The piece of workgroup `index` (SPLIT: of the index-th tile among those that are shared), by every wave alone: lane i
// looks at sequence 64 k + i.
template <int R, bool SPLIT>
__device__ __forceinline__ bool deal(const Kv4AttnArgs& a, const Deal& d, int index, Piece& out) {
    const int lane = threadIdx.x & 63;
    const int B = a.c.B;
    if (!SPLIT && !a.ws && !a.c.starts) {  // nothing is shared, every sequence has as many tiles: no length is waited for here
        const int tiles = ceil_div(a.c.each * a.share, R) * a.c.H;
        out.b = index / tiles;
        const int tile = index - out.b * tiles;
        out.tile = tile / a.c.H;
        out.head = tile - out.tile * a.c.H;
        out.share = out.slot = 0;
        out.shares = 1;
        out.first = out.b * a.c.each;
        out.count = a.c.each;
        if (out.b >= B) return false;
        out.end = imax(a.c.lengths[out.b], 0);
        out.len = kv4_inside(a.c, out.end);
        return true;
    }
    Sizes s = sizes_of<R>(a, lane);
    int least = 1 << 30;
    if (a.ws) {
        unsigned long long units = 0;
        for (int b0 = 0; b0 < B; b0 += 64) {
            const Sizes t = b0 ? sizes_of<R>(a, b0 + lane) : s;
            const unsigned long long mine = (unsigned long long)t.tiles * t.pages;
            units += (unsigned)wave_sum((int)(mine & 0xffff)) + ((unsigned long long)(unsigned)wave_sum((int)(mine >> 16)) << 16);
        }
        // (tokens counted once: below KA_MOST_PAGES; starts that let sequences overlap may pass it, and then nothing is shared)
        const unsigned long long per = (units + 255) >> 8;
        const int even = ceil_div((int)(per < (1u << 30) ? per : 1u << 30), d.per_cu);
        least = imax(even, d.least);
    }
    int slots = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        if (b0) s = sizes_of<R>(a, b0 + lane);
        const int shares = s.pages > least ? ceil_div(s.pages, least) : 1;
        const int mine = SPLIT ? (shares > 1 ? s.tiles : 0) : s.tiles * shares;
        const int upto = wave_scan(mine);
        const int taken = shares > 1 ? s.tiles * shares : 0;
        const int slots_upto = wave_scan(taken);
        const unsigned long long past = __ballot(upto > index);
        if (past) {
            const int at = __ffsll(past) - 1;
            const int rest = index - __builtin_amdgcn_readlane(upto - mine, at);
            out.shares = __builtin_amdgcn_readlane(shares, at);
            const int tile = SPLIT || out.shares == 1 ? rest : rest / out.shares;
            out.b = b0 + at;
            out.share = SPLIT ? 0 : rest - tile * out.shares;
            out.head = tile % a.c.H;
            out.tile = tile / a.c.H;
            out.slot = slots + __builtin_amdgcn_readlane(slots_upto - taken, at) + tile * out.shares + out.share;
            out.first = __builtin_amdgcn_readlane(s.first, at);
            out.count = __builtin_amdgcn_readlane(s.count, at);
            out.len = __builtin_amdgcn_readlane(s.len, at);
            out.end = __builtin_amdgcn_readlane(s.end, at);
            return true;
        }
        index -= __builtin_amdgcn_readlane(upto, 63);
        slots += __builtin_amdgcn_readlane(slots_upto, 63);
    }
    return false;
}

template <int CTRL>
__device__ __forceinline__ float row_move(float v) {
    return bit_cast<float>(__builtin_amdgcn_mov_dpp(bit_cast<int>(v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, row_move<0x121>(v));  // row_ror:1
    v = fmaxf(v, row_move<0x122>(v));
    v = fmaxf(v, row_move<0x124>(v));
    v = fmaxf(v, row_move<0x128>(v));
    return rows_max(v);
}

// The softmax's reference moves when a score is more than KA_LAZY beyond it (in powers of two): P is at most 2^KA_LAZY, and
// P' = fp16(P s KA_TOP / sref), with sref a power of two above the scales so far, at most 2^15.  The factor is as large as that
// allows because sref follows the largest scale whatever its row counts for: below 2^-14, where fp16 numbers become denormal,
// P' is held to 2^-25 only, so that terms P s below 2^(KA_LAZY - 29) sref are held to 2^(KA_LAZY - 40) sref each instead of to
// 2^-11 of themselves.  2 / 3 / 4 / 8: 1024 tokens over 16384 rows 454 / 451 / 448 / 447 us, with scores three times as wide
// 460 / 457 / 453 / 448; single tokens and drafts alike within 1 %.
constexpr int KA_LAZY = 4;
constexpr float KA_TOP = 1 << (15 - KA_LAZY);

// Shares of a tile's pages, joined: a workgroup has ROWS rows of a shared tile, 256 / ROWS threads each, of which D / 4 hold
// four columns each of every so many-th share.  (LAST: tiles are worked on from the last to the first.)  3.8 to 4.7 us where
// a tile has up to a few dozen shares, nearly all of it the launch and two rounds of loads; 18 us for the 35 MB of 1024 tokens.
template <int D, int R, int ROWS, bool LAST>
__global__ __launch_bounds__(256) void kv4_join_kernel(Kv4AttnArgs a, Deal d) {
    constexpr int C4 = D / 4, LANES = 256 / C4 / ROWS;
    static_assert(LANES >= 1 && R % ROWS == 0);
    __shared__ __attribute__((aligned(16))) float part[ROWS][LANES][D];
    __shared__ float state[ROWS][LANES][2];
    Piece pc;
    if (!deal<R, true>(a, d, blockIdx.x, pc)) return;
    if (pc.slot + pc.shares > 2 * d.wgs()) return;  // (only where lengths change under the launch)
    const int c4 = threadIdx.x % C4, lane = threadIdx.x / C4 % LANES, sub = threadIdx.x / (C4 * LANES);
    const int r = blockIdx.y * ROWS + sub;
    const int rr = (LAST ? ceil_div(pc.count * a.share, R) - 1 - pc.tile : pc.tile) * R + r;
    const bool live = rr < pc.count * a.share;
    const float* const base = a.ws + (long)pc.slot * R * (D + 2);
    float m = -INFINITY, sum = 0.f;
    float4_t o = {0.f, 0.f, 0.f, 0.f};
    constexpr int AHEAD = 4;  // shares whose states are asked for at once
    if (live)
        for (int s0 = lane; s0 < pc.shares; s0 += LANES * AHEAD) {
            float ms[AHEAD], ls[AHEAD];
            float4_t v[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const float* const src = base + (long)imin(s0 + LANES * i, pc.shares - 1) * R * (D + 2);
                ms[i] = src[R * D + 2 * r];
                ls[i] = src[R * D + 2 * r + 1];
                v[i] = *(const float4_t*)(src + r * D + 4 * c4);
            }
#pragma unroll
            for (int i = 0; i < AHEAD; i++)
                if (s0 + LANES * i < pc.shares) {
                    const float to = fmaxf(m, ms[i]);
                    const float f0 = m == to ? 1.f : __builtin_amdgcn_exp2f(m - to);
                    const float f1 = ms[i] == to ? 1.f : __builtin_amdgcn_exp2f(ms[i] - to);
                    sum = sum * f0 + ls[i] * f1;
                    o = o * f0 + v[i] * f1;
                    m = to;
                }
        }
    *(float4_t*)&part[sub][lane][4 * c4] = o;
    if (c4 == 0) {
        state[sub][lane][0] = m;
        state[sub][lane][1] = sum;
    }
    __syncthreads();
    if (lane != 0 || !live) return;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < LANES; w++) mx = fmaxf(mx, state[sub][w][0]);
    sum = 0.f;
    o = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < LANES; w++) {
        const float mw = state[sub][w][0];
        const float f = mw == mx ? 1.f : __builtin_amdgcn_exp2f(mw - mx);
        sum += state[sub][w][1] * f;
        o += *(const float4_t*)&part[sub][w][4 * c4] * f;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    half4_t h;
#pragma unroll
    for (int e = 0; e < 4; e++) h[e] = (half_t)(o[e] * inv);
    *(half4_t*)(a.out + ((long)(pc.first + rr / a.share) * a.c.H * a.share + pc.head * a.share + rr % a.share) * D + 4 * c4) = h;
}

// Many rows per sequence and key/value head (no selected pages): sq_kv4_chunk.hip.
size_t kv4_chunk_workspace_bytes(int D, int pages);
hipError_t launch_kv4_chunk(Kv4AttnArgs a, int D, int g, hipStream_t st);

}  // namespace sq
