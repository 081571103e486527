// Causal attention of a batch of sequences that share a long prefix (fp16 in and out, fp32 softmax and sums).
//
//   out[t, h, :] = sum_j P[j] v_j,  P = softmax_j(sm_scale q[t, h, :] . k_j)  over the P rows of the prefix, which all
//   sequences see whole, and the rows of t's own sequence up to t's.
//
// The softmax splits: with (m, l, o) = (max s, sum exp(s - m), sum exp(s - m) v) over a part of the rows, parts join as
//   m = max m_i, l = sum l_i exp(m_i - m), o = sum o_i exp(m_i - m), out = o / l.
// So the prefix can be read once for all sequences: the rows (token, query head) of a key/value head, whatever sequence they
// belong to, are packed into tiles and meet the prefix as one dense product without masks; each sequence's rows meet its own
// cache apart; a second launch joins the parts.  Where a sequence has many rows itself (a prompt) nothing is gained by packing:
// its tiles go through the prefix and on through their own rows, and write the result.
//
// What bounds it: one token of each sequence the bytes, long ones at 3.1 TB/s with the second launch (64 ragged sequences of up to
// 1000 rows behind 8192, 32 heads over 8 of 128: 131 MB in 42 us, 31 of the first launch and 5.6 of the second), short ones
// the chain of launch, first rows, softmax, join (8 sequences behind 512 rows 12.3 us, the host's two launches 9 of them);
// prompts the vector instructions of the softmax beside the products, which overlap in part (16 ragged ones of up to 512 tokens
// behind 4096 rows: 141 GFLOP in 176 us, 0.8 PFLOP/s; per 32 x 32 scores 16 products of 32 cycles, and 16 exponentials of 8
// with about five other instructions of 4 each).  Four waves of 32 rows on two workgroups a CU: products and exponentials of
// different waves fill each other's gaps better than one wave's own interleaved (202 us as it was then, 226 to 243 interleaved).
#include "sq_attn_rows.h"
#include "sq_kernels.h"

#include <algorithm>
#include <type_traits>

namespace sq {

namespace {

constexpr int PA_STEP = 64;  // keys of a step

// How a call is cut.  Packed: rows of all sequences against pieces of the prefix (a), a sequence's against pieces of its own rows
// (b).  Otherwise tiles of a sequence's rows against the prefix and its own rows, as `Deal` has it.
struct PrefixPlan {
    float* po;  // partial outputs, then (reference, sum) of each
    float2* pml;
    int packed, qa, qb, rows_b;                                // tiles of 32 qa and 32 qb rows
    int tiles_a, parts_a, steps_a, tiles_b, parts_b, steps_b;  // steps of 64 keys of a part
    int units_a, units_b, grid_a, grid_b, most;                // most: parts that a tile may be cut into
    Divisor by_share, by_tiles_a, by_parts_a, by_tiles_b, by_parts_b;
};

struct PrefixArgs {
    PrefixAttn t;
    PrefixPlan p;
    float qk_scale;  // sm_scale * log2(e)
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }
__device__ __forceinline__ int imax(int a, int b) { return a > b ? a : b; }

// Tokens of sequence b of the call: [first, first + count), whatever `starts` holds inside [0, T].
__device__ __forceinline__ void tokens_of(const PrefixAttn& t, int b, int& first, int& count) {
    if (t.starts) {
        first = imin(imax(t.starts[b], 0), t.T);
        count = imax(imin(imax(t.starts[b + 1], 0), t.T) - first, 0);
    } else {
        first = b * t.each;
        count = t.each;
    }
}

// The sequence of a token (-1: behind the last), by a wave together.
__device__ __forceinline__ int sequence_of(const PrefixAttn& t, int token) {
    if (!t.starts) return token / t.each;
    const int lane = threadIdx.x & 63;
    int upto = 0;
    for (int b0 = 0; b0 <= t.B; b0 += 64) {
        const int b = b0 + lane;
        upto += __popcll(__ballot(b <= t.B && t.starts[imin(b, t.B)] <= token));
    }
    return upto > t.B ? -1 : upto - 1;
}

struct Tile {
    int b, tile, first, count;
};
// The index-th tile of ROWS rows among those of all sequences, by a wave together.
__device__ __forceinline__ bool tile_of(const PrefixAttn& t, int rows_of_tile, int index, Tile& out) {
    if (!t.starts) {
        const int tiles = ceil_div(t.each * t.share, rows_of_tile);
        out.b = index / tiles;
        out.tile = index - out.b * tiles;
        out.first = out.b * t.each;
        out.count = t.each;
        return out.b < t.B;
    }
    const int lane = threadIdx.x & 63;
    for (int b0 = 0; b0 < t.B; b0 += 64) {
        int first = 0, count = 0;
        if (b0 + lane < t.B) tokens_of(t, b0 + lane, first, count);
        const int mine = ceil_div(count * t.share, rows_of_tile);
        int upto = mine;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) {
            const int v = __shfl_up(upto, x);
            if (lane >= x) upto += v;
        }
        const unsigned long long past = __ballot(upto > index);
        if (past) {
            const int at = __ffsll(past) - 1;
            out.b = b0 + at;
            out.tile = index - __builtin_amdgcn_readlane(upto - mine, at);
            out.first = __builtin_amdgcn_readlane(first, at);
            out.count = __builtin_amdgcn_readlane(count, at);
            return true;
        }
        index -= __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// What the rows of a tile of a sequence see: own rows [0, own) of the cache, and in steps.
struct Reach {
    int before;    // own rows that were there before the call's
    int own;       // rows that the tile's last row sees
    int own_first; // rows that the tile's first row sees
    int pre_steps, steps;
};
__device__ __forceinline__ Reach reach_of(const PrefixAttn& t, const PrefixPlan& p, const Tile& tl) {
    Reach r;
    r.before = imax(t.lengths[tl.b], 0) - tl.count;
    const int row0 = tl.tile * p.rows_b;
    const int row1 = imin(row0 + p.rows_b, tl.count * t.share) - 1;
    r.own = imin(imax(r.before + p.by_share(row1) + 1, 0), t.Lmax);
    r.own_first = imin(imax(r.before + p.by_share(row0) + 1, 0), t.Lmax);
    r.pre_steps = p.packed ? 0 : ceil_div(t.P, PA_STEP);
    r.steps = r.pre_steps + ceil_div(r.own, PA_STEP);
    return r;
}

// Tiles that go through the prefix and on through their own rows.  A launch has room for PA_SLOTS workgroups at a time and the
// tiles take about as long as each other: those of the full rounds are a workgroup's each, the rest, which would leave most of
// the last round empty, is cut into as many parts as fill it (616 tiles: 2 rounds, now 1 and a fifth).
constexpr int PA_SLOTS = 512;
struct Deal {
    int tiles;              // of a head
    int full, rest, parts;  // tiles of full rounds, the others, and the parts of each of those
};
__host__ __device__ __forceinline__ Deal deal_of(int tiles, int heads, int most) {
    Deal d;
    const int all = tiles * heads;
    d.tiles = tiles;
    d.full = all / PA_SLOTS * PA_SLOTS;
    d.rest = all - d.full;
    d.parts = d.rest ? PA_SLOTS / d.rest : 1;
    d.parts = d.parts < 1 ? 1 : d.parts > most ? most : d.parts;
    return d;
}
__device__ __forceinline__ Deal deal_of(const PrefixAttn& t, const PrefixPlan& p) {
    int tiles = p.tiles_b;
    if (t.starts) {
        const int lane = threadIdx.x & 63;
        tiles = 0;
        for (int b0 = 0; b0 < t.B; b0 += 64) {
            int first = 0, count = 0;
            if (b0 + lane < t.B) tokens_of(t, b0 + lane, first, count);
            int sum = ceil_div(count * t.share, p.rows_b);
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
            // (starts of any content may let sequences overlap: what the launch has no workgroups for is left out)
            tiles = imin(tiles + sum, p.tiles_b);
        }
        tiles = __builtin_amdgcn_readfirstlane(tiles);
    }
    return deal_of(tiles, t.H, p.most);
}

// A piece of work: rows of a key/value head against a range of steps.
struct Work {
    int head, row0, rows;  // rows row0 .. row0 + rows - 1 of the head's T * share
    int s0, s1;            // steps
    bool shared;           // against the prefix alone
    bool direct;           // all that the rows see: the result; otherwise a part of it, row r at place + r of the parts
    long place;
    Tile tl;
    Reach rc;
};

__device__ __forceinline__ const half_t* prefix_row(const PrefixAttn& t, const Work& w, bool value, int key) {
    return (value ? t.vp : t.kp) + (long)w.head * t.p_hs + (long)key * t.p_rs;
}
__device__ __forceinline__ const half_t* cache_row(const PrefixAttn& t, const Work& w, bool value, int key) {
    return (value ? t.vc : t.kc) + (long)w.tl.b * t.c_bs + (long)w.head * t.c_hs + (long)key * t.c_rs;
}
// Own rows from here on are the call's: they are taken from there, other workgroups are storing them to the cache.
__device__ __forceinline__ int fresh_from(const PrefixAttn& t, const Work& w) { return t.kn ? w.rc.before : t.Lmax; }
__device__ __forceinline__ const half_t* own_row(const PrefixAttn& t, const Work& w, bool value, int key) {
    const int fresh = fresh_from(t, w);
    if (key >= fresh) return (value ? t.vn : t.kn) + (long)(w.tl.first + key - fresh) * t.n_ts + (long)w.head * t.n_hs;
    return cache_row(t, w, value, key);
}

// Infinities and NaN among the values must reach the rows that see them and no others, and 0 times them is no 0: in steps
// with a causal mask they count as 0 in the product, and are added behind the last step to the rows that see them.
template <int D>
__device__ __forceinline__ bool clear_odd(uint8_t* tile, int rows, int first, int stride) {
    bool odd = false;
#pragma unroll 1
    for (int i = first; i < rows * (D / 8); i += stride) {
        half8_t x = *(half8_t*)(tile + i * 16);
        bool any = false;
#pragma unroll
        for (int v = 0; v < 8; v++) {
            const bool finite = __builtin_fabsf((float)x[v]) <= 65504.f;
            any |= !finite;
            x[v] = finite ? x[v] : (half_t)0.f;
        }
        if (any) *(half8_t*)(tile + i * 16) = x;
        odd |= any;
    }
    return odd;
}
template <int D>
__device__ __forceinline__ void add_odd(const PrefixAttn& t, const Work& w, int last, float16_t (&acc)[D / 32]) {
    const int lc = (threadIdx.x & 63) >> 5;
    const int k0 = imax(imax(w.s0 - w.rc.pre_steps, 0) * PA_STEP, w.rc.own_first / PA_STEP * PA_STEP);
    const int k1 = imin((w.s1 - w.rc.pre_steps) * PA_STEP, w.rc.own);
#pragma unroll 1
    for (int key = k0; key < k1; key++) {
        const half_t* const v = own_row(t, w, true, key) + 4 * lc;
#pragma unroll
        for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const half4_t h = *(const half4_t*)(v + 32 * dt + 8 * i);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    acc[dt][4 * i + j] += key <= last && !(__builtin_fabsf((float)h[j]) <= 65504.f) ? (float)h[j] : 0.f;
            }
    }
}

// Four columns of a row's sums: the result, or a part of it.
template <int D>
__device__ __forceinline__ void store_row(const PrefixArgs& a, const Work& w, int row, int col, float4_t o, float m, float l) {
    const PrefixAttn& t = a.t;
    if (w.direct) {
        const int token = a.p.by_share(row);
        const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing: 0
        half4_t h;
#pragma unroll
        for (int j = 0; j < 4; j++) h[j] = (half_t)(o[j] * inv);
        *(half4_t*)(t.o + ((long)token * (t.H * t.share) + w.head * t.share + row - token * t.share) * D + col) = h;
    } else {
        *(float4_t*)(a.p.po + (w.place + row) * D + col) = o;
        if (col == 0) a.p.pml[w.place + row] = make_float2(m, l);
    }
}

// Up to 32 rows: the waves go round the keys.
template <int D>
__device__ __forceinline__ void few_rows(const PrefixArgs& a, const Work& w, uint8_t* lds, float2* stat) {
    typedef RowsAttn<D> R;
    const PrefixAttn& t = a.t;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = w.row0 + imin(lane & 31, w.rows - 1);
    const int token = a.p.by_share(row);
    R r;
    r.load_query(t.q + (long)token * t.q_ts + (long)(w.head * t.share + row - token * t.share) * t.q_hs + 8 * (lane >> 5));
    const int limit = imin(w.rc.before + token - w.tl.first, t.Lmax - 1);  // the last own row that it sees
    const int pre = w.shared ? 2 * w.s1 : 2 * w.rc.pre_steps;              // blocks of the prefix
    const int plain_own = imin(w.rc.own, fresh_from(t, w));
    const int end = imin(2 * w.s1, w.shared ? ceil_div(t.P, RA_BLOCK) : pre + ceil_div(w.rc.own, RA_BLOCK));
    bool odd = false;
    r.template run<false>(
        lds, 2 * w.s0 + wave, end, a.qk_scale, []() {},
        [&](int blk, bool value, uint32_t at) {
            const bool is_pre = blk < pre;
            const int n = (is_pre ? blk : blk - pre) * RA_BLOCK;
            if (n + RA_BLOCK <= (is_pre ? t.P : plain_own))
                R::request((const uint8_t*)(is_pre ? prefix_row(t, w, value, n) : cache_row(t, w, value, n)),
                           (uint32_t)(is_pre ? t.p_rs : t.c_rs) * 2, value, at);
            else
                R::request_each(value, at, [&](int i) {  // rows past the end re-read the last one
                    return is_pre ? prefix_row(t, w, value, imin(n + i, t.P - 1)) : own_row(t, w, value, imin(n + i, w.rc.own - 1));
                });
        },
        [&](int blk, int& n, int& full, int& last) {
            const bool is_pre = blk < pre;
            n = (is_pre ? blk : blk - pre) * RA_BLOCK;
            full = is_pre ? t.P : w.rc.own_first;
            last = is_pre ? t.P - 1 : limit;
        },
        [](int, uint8_t*) {},
        [&](int blk, uint8_t* tile) {
            const bool is_pre = blk < pre;
            const int n = (is_pre ? blk : blk - pre) * RA_BLOCK;
            const int past = (is_pre ? t.P : w.rc.own) - n;
            if (past < RA_BLOCK) R::clear_from(tile, imax(past, 0));
            if (!is_pre && n + RA_BLOCK > w.rc.own_first && w.rc.own_first < w.rc.own) odd |= clear_odd<D>(tile, RA_BLOCK, lane, 64);
        },
        [](int, const float16_t&) {});
    if (!w.shared && w.rc.own_first < w.rc.own && __syncthreads_or(odd) && wave == 0) add_odd<D>(t, w, limit, r.acc);
    r.join(lds, stat, w.rows, [&](int i, int col, float4_t o, float m, float l) { store_row<D>(a, w, w.row0 + i, col, o, m, l); });
}

// 32 QG rows: wave (qg, kg) has rows 32 qg .. + 31 and a KG-th of the keys of a step; the steps' tiles are shared, in two stages.
template <int D, int QG>
__device__ __forceinline__ void many_rows(const PrefixArgs& a, const Work& w, uint8_t* lds) {
    constexpr int KG = 4 / QG;
    constexpr int KS = PA_STEP / (32 * KG);  // 32-key blocks of a wave and step
    constexpr int ROW = D * 2;               // bytes of a tile row
    constexpr int TILE = PA_STEP * ROW;
    constexpr int SB = 2 * TILE;             // a stage: K tile, V tile
    constexpr int NK = D / 16;
    constexpr int DT = D / 32;
    constexpr int NL = TILE / 1024 / 4;      // direct loads per wave, operand and stage
    constexpr int RPL = 1024 / ROW;          // tile rows per load
    constexpr int CPR = D / 8;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    const PrefixAttn& t = a.t;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ln = lane & 31, lc = lane >> 5;
    const int qg = wave / KG, kg = wave % KG;
    const bool idle = 32 * qg >= w.rows;
    const int row = w.row0 + imin(32 * qg + ln, w.rows - 1);
    const int token = a.p.by_share(row);
    const int limit = imin(w.rc.before + token - w.tl.first, t.Lmax - 1);
    half8_t qf[NK];
    {
        const half_t* qp = t.q + (long)token * t.q_ts + (long)(w.head * t.share + row - token * t.share) * t.q_hs + 8 * lc;
#pragma unroll
        for (int s = 0; s < NK; s++) qf[s] = *(const half8_t*)(qp + 16 * s);
    }
    const int pre_steps = w.shared ? w.s1 : w.rc.pre_steps;
    const int plain_own = imin(w.rc.own, fresh_from(t, w));
    const int lrow = lane / CPR, lchunk = lane % CPR;
    const int row_w = RPL * NL * wave + lrow;  // of this lane's first load in the tile
    auto issue = [&](int s, uint32_t stage) {
        const bool pre = s < pre_steps;
        const int n = (pre ? s : s - pre_steps) * PA_STEP;
        const uint32_t l0 = lds0 + stage + wave * (NL * 1024);
        if (n + PA_STEP <= (pre ? t.P : plain_own)) {
            const uint32_t rs = (uint32_t)(pre ? t.p_rs : t.c_rs) * 2;
            const uint8_t* const kb = uniform((const uint8_t*)(pre ? prefix_row(t, w, false, n) : cache_row(t, w, false, n)));
            const uint8_t* const vb = uniform((const uint8_t*)(pre ? prefix_row(t, w, true, n) : cache_row(t, w, true, n)));
            uint32_t off = row_w * rs;
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const int r = row_w + RPL * j;
                load_to_lds_x4(kb, off + ((lchunk ^ k_swz<D>(r)) * 16), l0 + j * 1024);
                load_to_lds_x4(vb, off + ((lchunk ^ v_swz<D>(r)) * 16), l0 + TILE + j * 1024);
                off += RPL * rs;
            }
        } else {  // rows past the end re-read the last one
#pragma unroll 1
            for (int j = 0; j < NL; j++) {
                const int r = row_w + RPL * j;
                const int key = imin(n + r, (pre ? t.P : w.rc.own) - 1);
                const half_t* const k = pre ? prefix_row(t, w, false, key) : own_row(t, w, false, key);
                const half_t* const v = pre ? prefix_row(t, w, true, key) : own_row(t, w, true, key);
                load_to_lds_x4((const uint8_t*)k + ((lchunk ^ k_swz<D>(r)) * 16), l0 + j * 1024);
                load_to_lds_x4((const uint8_t*)v + ((lchunk ^ v_swz<D>(r)) * 16), l0 + TILE + j * 1024);
            }
        }
    };
    if (w.s0 < w.s1) issue(w.s0, 0);

    // LDS byte offsets of the operand reads (of the other stage: with SB flipped).
    int kread[NK], vread[DT];
#pragma unroll
    for (int s = 0; s < NK; s++) kread[s] = (32 * KS * kg + ln) * ROW + (((2 * s + lc) ^ k_swz<D>(ln)) * 16);
    {
        const int key = 4 * lc + ((lane & 15) >> 2);  // + 32 b + 16 s + 8 i, which leave v_swz unchanged
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
            vread[dt] = TILE + (32 * KS * kg + key) * ROW +
                        (((4 * dt + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ v_swz<D>(key)) * 16) + 8 * (lane & 1);
    }

    // Reference of the row (0 while unset), the score above it at which it moves (any score while unset), and this lane's share
    // of the row sum.
    float ref = 0.f, top = -INFINITY, l_i = 0.f;
    float16_t acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int v = 0; v < 16; v++) acc[dt][v] = 0.f;
#pragma unroll
    for (int s = 0; s < NK; s++) {
        u32x4_t x = bit_cast<u32x4_t>(qf[s]);
        asm volatile("" : "+v"(x));
        qf[s] = bit_cast<half8_t>(x);
    }
    const bool causal = !w.shared && w.rc.own_first < w.rc.own;  // (or all rows of the tile see all own rows up to the last)
    bool odd = false;
    uint32_t stage = 0;
#pragma unroll 1
    for (int s = w.s0; s < w.s1; s++, stage ^= SB) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (s + 1 < w.s1) issue(s + 1, stage ^ SB);
        const bool pre = s < pre_steps;
        const int n = (pre ? s : s - pre_steps) * PA_STEP;
        // Masks (only where the step touches the end of the rows or the causal diagonal; the test is uniform).
        const bool masked = n + PA_STEP > (pre ? t.P : w.rc.own_first);
        if (masked) {
            uint8_t* const vt = lds + stage + TILE;
            for (int i = imax((pre ? t.P : w.rc.own) - n, 0) * CPR + tid; i < PA_STEP * CPR; i += 256)
                *(u32x4_t*)(vt + i * 16) = (u32x4_t){0u, 0u, 0u, 0u};
            if (!pre && causal) odd |= clear_odd<D>(vt, imin(w.rc.own - n, PA_STEP), tid, 256);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
        if (idle) continue;
        const uint8_t* const l = lds + stage;
        float16_t st[KS];
#pragma unroll
        for (int b = 0; b < KS; b++) {
            half8_t kf[NK];
#pragma unroll
            for (int i = 0; i < NK; i++) kf[i] = *(const half8_t*)(l + kread[i] + b * (32 * ROW));
#pragma unroll
            for (int v = 0; v < 16; v++) st[b][v] = 0.f;
#pragma unroll
            for (int i = 0; i < NK; i++) st[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i], qf[i], st[b], 0, 0, 0);
        }
#pragma unroll
        for (int b = 0; b < KS; b++)
#pragma unroll
            for (int v = 0; v < 16; v++) st[b][v] = __builtin_fmaf(st[b][v], a.qk_scale, -ref);
        if (masked) {
            const int last = pre ? t.P - 1 : limit;
#pragma unroll
            for (int b = 0; b < KS; b++)
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const int key = n + 32 * (KS * kg + b) + 8 * (v >> 2) + 4 * lc + (v & 3);
                    st[b][v] = key <= last ? st[b][v] : -INFINITY;
                }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < KS; b++)
#pragma unroll
            for (int v = 0; v < 16; v++) mx = fmaxf(mx, st[b][v]);
        if (__builtin_amdgcn_ballot_w64(mx > top) != 0) {
            const float mq = fmaxf(mx, __shfl_xor(mx, 32));
            const bool upd = mq > top;
            const float delta = upd ? mq - REF_BELOW : 0.f;
            const float alpha = (upd && top != -INFINITY) ? __builtin_amdgcn_exp2f(-delta) : 1.f;
            ref += delta;
            top = upd ? REF_MOVES : top;
            l_i *= alpha;
#pragma unroll
            for (int b = 0; b < KS; b++)
#pragma unroll
                for (int v = 0; v < 16; v++) st[b][v] -= delta;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int v = 0; v < 16; v++) acc[dt][v] *= alpha;
        }
        // p is rounded to fp16 for the second product (its operands are), and the row sum is that of the rounded ones.
        half8_t pk[2 * KS];
        float rs = 0.f;
#pragma unroll
        for (int b = 0; b < KS; b++)
#pragma unroll
            for (int v = 0; v < 16; v += 2) {
                const half2_t pp = {(half_t)__builtin_amdgcn_exp2f(st[b][v]), (half_t)__builtin_amdgcn_exp2f(st[b][v + 1])};
                rs = __builtin_amdgcn_fdot2(pp, (half2_t){(half_t)1.f, (half_t)1.f}, rs, false);
                pk[2 * b + (v >> 3)][v & 7] = pp.x;
                pk[2 * b + (v >> 3)][(v & 7) + 1] = pp.y;
            }
        l_i += rs;
#pragma unroll
        for (int i = 0; i < 2 * KS; i++)
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                const u32x2_t lo = bit_cast<u32x2_t>(lds_read_tr(l + vread[dt] + 16 * i * ROW));
                const u32x2_t hi = bit_cast<u32x2_t>(lds_read_tr(l + vread[dt] + (16 * i + 8) * ROW));
                const u32x4_t x = {lo.x, lo.y, hi.x, hi.y};
                acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bit_cast<half8_t>(x), pk[i], acc[dt], 0, 0, 0);
            }
    }
    if (causal && __syncthreads_or(odd) && kg == 0) add_odd<D>(t, w, limit, acc);

    // ---- the row's state: over its two lanes, then over the key groups
    l_i += __shfl_xor(l_i, 32);
    float m_i = top == -INFINITY ? -INFINITY : ref;
    const bool valid = 32 * qg + ln < w.rows;
    __syncthreads();
    if constexpr (KG == 1) {
        if (valid) {
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    store_row<D>(a, w, row, 32 * dt + 8 * i + 4 * lc,
                                 (float4_t){acc[dt][4 * i], acc[dt][4 * i + 1], acc[dt][4 * i + 2], acc[dt][4 * i + 3]}, m_i, l_i);
        }
    } else {
        // each wave hands half of its columns to the other key group's wave and finishes the others
        constexpr int OWN = DT / 2;
        float4_t* red = reinterpret_cast<float4_t*>(lds);                 // [wave][OWN][4][64]
        float2* state = reinterpret_cast<float2*>(lds + 4 * OWN * 4096);  // [wave][64]
        static_assert(4 * OWN * 4096 + 4 * 512 <= 2 * SB, "fits");
#pragma unroll
        for (int d = 0; d < OWN; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float4_t x;
#pragma unroll
                for (int j = 0; j < 4; j++) x[j] = kg == 0 ? acc[OWN + d][4 * i + j] : acc[d][4 * i + j];
                red[((wave * OWN + d) * 4 + i) * 64 + lane] = x;
            }
        state[wave * 64 + lane] = make_float2(m_i, l_i);
        __syncthreads();
        const int peer = wave ^ 1;
        const float2 mine = make_float2(m_i, l_i), theirs = state[peer * 64 + lane];
        const float m = fmaxf(mine.x, theirs.x);
        const float f = share_of(mine, m), g = share_of(theirs, m);
        const float l = mine.y * f + theirs.y * g;
        if (valid) {
#pragma unroll
            for (int d = 0; d < OWN; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float4_t o = red[((peer * OWN + d) * 4 + i) * 64 + lane];
                    float4_t x;
#pragma unroll
                    for (int j = 0; j < 4; j++) x[j] = (kg == 0 ? acc[d][4 * i + j] : acc[OWN + d][4 * i + j]) * f + o[j] * g;
                    store_row<D>(a, w, row, 32 * (d + kg * OWN) + 8 * i + 4 * lc, x, m, l);
                }
        }
    }
}

template <int D, int QG>
__device__ __forceinline__ void attend(const PrefixArgs& a, const Work& w, uint8_t* lds, float2* stat) {
    if constexpr (QG == 1) few_rows<D>(a, w, lds, stat);
    else many_rows<D, QG>(a, w, lds);
}

// QA, QB: groups of 32 rows of the tiles against the prefix (0: none) and of a sequence's.
template <int D, int QA, int QB>
__global__ __launch_bounds__(256, 2) void prefix_attn_kernel(PrefixArgs a) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[RowsAttn<D>::LDS];
    __shared__ float2 stat[4 * 32];
    static_assert(RowsAttn<D>::LDS == 4 * PA_STEP * D * 2);
    const PrefixAttn& t = a.t;
    const PrefixPlan& p = a.p;
    int index = blockIdx.x;
    Work w = {};
    if constexpr (QA > 0) {
        // (a part's place: [head][parts_a, then parts_b][T * share])
        const int parts = p.parts_a + p.parts_b, all = t.T * t.share;
        if (index < p.grid_a) {
            const int work = (index & 7) * (p.grid_a >> 3) + (index >> 3);  // an eighth of the list per XCD: a piece's tiles share an L2
            if (work >= p.units_a) return;
            const int rest = p.by_tiles_a(work);
            w.row0 = (work - rest * p.tiles_a) * (32 * QA);
            w.head = p.by_parts_a(rest);
            const int part = rest - w.head * p.parts_a;
            w.rows = imin(32 * QA, all - w.row0);
            w.s0 = part * p.steps_a;
            w.s1 = imin(w.s0 + p.steps_a, ceil_div(t.P, PA_STEP));
            w.shared = true;
            w.place = ((long)w.head * parts + part) * all;
            if constexpr (QA != QB) {
                attend<D, QA>(a, w, lds, stat);
                return;
            }
        }
        index -= p.grid_a;
        if (index < p.grid_b) {
            if (!w.shared) {
                const int work = (index & 7) * (p.grid_b >> 3) + (index >> 3);
                if (work >= p.units_b) return;
                const int rest = p.by_tiles_b(work);
                w.head = p.by_parts_b(rest);
                const int part = rest - w.head * p.parts_b;
                if (!tile_of(t, 32 * QB, p.tiles_b - 1 - (work - rest * p.tiles_b), w.tl)) return;
                w.rc = reach_of(t, p, w.tl);
                w.row0 = w.tl.first * t.share + w.tl.tile * (32 * QB);
                w.rows = imin(32 * QB, w.tl.count * t.share - w.tl.tile * (32 * QB));
                w.s0 = part * p.steps_b;
                w.s1 = imin(w.s0 + p.steps_b, w.rc.steps);
                if (w.s0 >= w.s1 && part > 0) return;  // (the first part also stands for rows that see nothing)
                w.place = ((long)w.head * parts + p.parts_a + part) * all;
            }
            attend<D, QB>(a, w, lds, stat);
            return;
        }
    } else if (index < p.grid_b) {
        const Deal d = deal_of(t, p);
        int at = index, part = 0;
        if (index < d.full) {
            at = (index & 7) * (d.full >> 3) + (index >> 3);  // an eighth of the list per XCD: a head's tiles share an L2
        } else {
            at = index - d.full;
            if (at >= d.rest * d.parts) return;
            part = at / d.rest;
            at += d.full - part * d.rest;
        }
        w.head = at / d.tiles;
        if (!tile_of(t, 32 * QB, at - w.head * d.tiles, w.tl)) return;
        w.rc = reach_of(t, p, w.tl);
        w.row0 = w.tl.first * t.share + w.tl.tile * (32 * QB);
        w.rows = imin(32 * QB, w.tl.count * t.share - w.tl.tile * (32 * QB));
        w.s1 = w.rc.steps;
        w.direct = index < d.full || d.parts == 1;
        if (!w.direct) {
            const int each = ceil_div(w.rc.steps, d.parts);
            w.s0 = imin(part * each, w.rc.steps);
            w.s1 = imin(w.s0 + each, w.rc.steps);
            w.place = (long)((at - d.full) * d.parts + part) * (32 * QB) - w.row0;
        }
        attend<D, QB>(a, w, lds, stat);
        return;
    }
    // the call's own rows into the cache, a token per wave
    const int lane = threadIdx.x & 63;
    const int token = (index - p.grid_b) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (token >= t.T) return;
    const int b = sequence_of(t, token);
    if (b < 0) return;
    int first, count;
    tokens_of(t, b, first, count);
    const int at = t.lengths[b] - count + token - first;
    if (at < 0 || at >= t.Lmax) return;
    constexpr int CPR = D / 8;
    for (int i = lane; i < t.H * CPR; i += 64) {
        const int h = i / CPR, c = 8 * (i % CPR);
        const long from = (long)token * t.n_ts + (long)h * t.n_hs + c;
        const long to = (long)b * t.c_bs + (long)h * t.c_hs + (long)at * t.c_rs + c;
        *(u32x4_t*)(t.kc + to) = *(const u32x4_t*)(t.kn + from);
        *(u32x4_t*)(t.vc + to) = *(const u32x4_t*)(t.vn + from);
    }
}

// The parts of a row, `apart` places from each other, by a wave: its output.
template <int D>
__device__ __forceinline__ void join_row(const PrefixPlan& p, long place, long apart, int parts, half_t* out) {
    constexpr int EPL = D / 64;
    typedef float vec_t __attribute__((ext_vector_type(EPL)));
    typedef half_t hvec_t __attribute__((ext_vector_type(EPL)));
    const int lane = threadIdx.x & 63;
    float m = -INFINITY, l = 0.f;
    vec_t o = {};
    for (int s0 = 0; s0 < parts; s0 += 64) {
        float2 ml = make_float2(-INFINITY, 0.f);
        if (s0 + lane < parts) ml = p.pml[place + (s0 + lane) * apart];
        const int n = imin(parts - s0, 64);
        vec_t x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = *(const vec_t*)(p.po + (place + (s0 + imin(j, n - 1)) * apart) * D + EPL * lane);
        float mx = ml.x;
#pragma unroll
        for (int y = 1; y < 64; y <<= 1) mx = fmaxf(mx, __shfl_xor(mx, y));
        mx = fmaxf(mx, m);
        const float w = share_of(ml, mx);
        float ls = ml.y * w;
#pragma unroll
        for (int y = 1; y < 64; y <<= 1) ls += __shfl_xor(ls, y);
        const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mx);
        l = l * f + ls;
        o *= f;
        m = mx;
#pragma unroll 1
        for (int s = 0; s < n; s += 8) {
            if (s > 0) {
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = *(const vec_t*)(p.po + (place + (s0 + imin(s + j, n - 1)) * apart) * D + EPL * lane);
            }
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (s + j < n) o += x[j] * bit_cast<float>(__builtin_amdgcn_readlane(bit_cast<int>(w), s + j));
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    hvec_t h;
#pragma unroll
    for (int i = 0; i < EPL; i++) h[i] = (half_t)(o[i] * inv);
    *(hvec_t*)(out + EPL * lane) = h;
}

// Packed: a row (token, query head) per wave.
template <int D>
__global__ __launch_bounds__(256) void prefix_join_kernel(PrefixArgs a) {
    const PrefixAttn& t = a.t;
    const PrefixPlan& p = a.p;
    const int index = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int heads = t.H * t.share;
    const int token = index / heads;
    if (token >= t.T) return;
    const int qhead = index - token * heads, head = p.by_share(qhead);
    Tile tl;
    tl.b = sequence_of(t, token);
    if (tl.b < 0) return;
    tokens_of(t, tl.b, tl.first, tl.count);
    const int row = token * t.share + qhead - head * t.share;
    tl.tile = (row - tl.first * t.share) / p.rows_b;
    const Reach rc = reach_of(t, p, tl);
    const int total = p.parts_a + p.parts_b;
    const long rows = (long)t.T * t.share;
    join_row<D>(p, (long)head * total * rows + row, rows, p.parts_a + imin(imax(ceil_div(rc.steps, p.steps_b), 1), p.parts_b),
                t.o + (long)index * D);
}

// Otherwise: 16 rows of a tile that was cut, four per wave.
template <int D>
__global__ __launch_bounds__(256) void prefix_join_tiles_kernel(PrefixArgs a) {
    const PrefixAttn& t = a.t;
    const PrefixPlan& p = a.p;
    const Deal d = deal_of(t, p);
    const int at = blockIdx.y;
    if (d.parts == 1 || at >= d.rest) return;
    const int head = (d.full + at) / d.tiles;
    Tile tl;
    if (!tile_of(t, p.rows_b, d.full + at - head * d.tiles, tl)) return;
    const int row0 = tl.first * t.share + tl.tile * p.rows_b;
    const int rows = imin(p.rows_b, tl.count * t.share - tl.tile * p.rows_b);
    for (int i = 0; i < 4; i++) {
        const int r = blockIdx.x * 16 + 4 * i + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        if (r >= rows) return;
        const int token = p.by_share(row0 + r);
        join_row<D>(p, (long)at * d.parts * p.rows_b + r, p.rows_b, d.parts,
                    t.o + ((long)token * (t.H * t.share) + head * t.share + row0 + r - token * t.share) * D);
    }
}

int div_up(long a, long b) { return (int)((a + b - 1) / b); }
// Steps of a piece where `steps` in all are cut for so many workgroups.
int cut(long steps, int wgs, int most) { return (int)std::max<long>(std::min<long>((steps + wgs - 1) / wgs, most), 1); }
int pad8(long n) { return (int)((n + 7) / 8 * 8); }

// Workgroups that packed rows' pieces are cut for (us).  Against the prefix a piece writes its rows' sums, and up to 256 rows the
// prefix's bytes bound it: two pieces per three CUs (64 sequences of 32 heads behind 8192 rows, 8 key/value heads: 42.0 with 160,
// 44.8 with 256, 56 with 512).  Beyond, behind a long prefix, the products do: one per CU (64 x 4 tokens behind 4096 rows
// 50.5 with 160, 47.5 with 256, 57 with 512; 64 x 8 88, 70 and 76; behind 1024 32.6 and 37.6).
constexpr int PA_WGS_MANY = 160, PA_WGS_FULL = 256, PA_WGS_FEW = 256;
// Against their own rows, of different numbers and up to the caches' room: four per CU (ragged up to 1000 rows 46.1 us with 512,
// 42.8 with 1024, 48 with 4096).
constexpr int PA_WGS_OWN = 1024;
// Packing pays where the prefix is long: it costs a second launch and the rows' sums, and saves each sequence's tile the way through
// the prefix (from L2).  Packed / not, us, 32 heads over 8: 64 x 1 token behind 512 rows 23.5 / 20.3, 1024 23.5 / 26.6, 8192
// 44 / 125; 64 x 8 behind 1024 45 / 32, 2048 52 / 45, 4096 70 / 74; where the tiles do not fill the chip 16 x 1 behind 64 12.2 / 9.0,
// 256 12.7 / 12.3, 1024 13.8 / 16.2; 16 x 8 16.9 / 11.8, 17.9 / 19.3, 19.2 / 23.6.  More than 32 rows of a sequence (64 x 16 tokens
// behind 4096) 107 / 102.  The average number of rows decides, since only the device knows each sequence's: one prompt of 1024
// tokens beside 63 single ones behind 4096 rows takes 231, the two apart 116 and 32.
bool pack(int P, int B, long each, long tiles) {
    return B > 1 && each <= 32 && P > (tiles >= PA_SLOTS ? 512 + 64 * each : PA_STEP);
}

}  // namespace

PrefixPlan prefix_plan(int T, int B, int H, int share, int P, int Lmax, bool ragged) {
    PrefixPlan p = {};
    const long rows = (long)T * share;     // of a key/value head
    const long each = (rows + B - 1) / B;  // of a sequence, on average
    const bool packed = pack(P, B, each, (long)B * H);
    p.packed = packed;
    p.qa = !packed ? 0 : rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
    // (tiles of 128 rows where that makes more than 64 of them: 1 x 32 tokens behind 4096 rows 27.1 us instead of 22.3 with 64,
    // 8 x 32 44.5 and 42.0, 8 x 64 58 and 62.5, 16 x 128 159 and 190)
    p.qb = each <= 32 ? 1 : each <= 64 || (rows + 127) / 128 * H <= 64 ? 2 : 4;
    p.rows_b = 32 * p.qb;
    const int pre = div_up(P, PA_STEP), own = div_up(Lmax, PA_STEP);
    if (packed) {
        p.tiles_a = div_up(rows, 32 * p.qa);
        const long steps = (long)H * p.tiles_a * pre;
        p.steps_a = cut(steps, p.qa == 1 ? PA_WGS_FEW : p.tiles_a > 2 && P >= 2048 ? PA_WGS_FULL : PA_WGS_MANY, pre);
        if (p.qa == 1) p.steps_a = (p.steps_a + 1) / 2 * 2;
        p.parts_a = div_up(pre, p.steps_a);
        p.units_a = H * p.parts_a * p.tiles_a;
    }
    p.tiles_b = ragged ? (int)(rows / p.rows_b + B) : B * div_up((long)(T / B) * share, p.rows_b);
    if (packed) {
        p.steps_b = cut((long)p.tiles_b * H * own, PA_WGS_OWN, own);
        p.steps_b = (p.steps_b + 1) / 2 * 2;  // (four waves' blocks of 32)
        p.parts_b = std::max(div_up(own, p.steps_b), 1);
        p.units_b = H * p.parts_b * p.tiles_b;
        p.grid_b = pad8(p.units_b);
    } else {
        p.steps_b = p.parts_b = 1;
        // Parts of four steps or more; many of them take longer to join than to go through (us, 8 heads x 4: 1 token behind 8192 rows
        // 18.4 with up to 8 parts, 13.6 with 24, 17.4 with 64, behind 16384 34.4, 21.8 and 24.4; 64 tokens 37.7 with 8, 31.2 with 16;
        // 2 x 64 behind 4096, of four steps each, 29.8 and 33.3).
        const int steps = own + pre;
        p.most = std::max(p.qb == 1 ? std::min(steps / 4, 24) : std::max(std::min(steps / 4, 8), std::min(steps / 8, 16)), 1);
        const int all = p.tiles_b * H;
        p.grid_b = all / PA_SLOTS * PA_SLOTS + (ragged ? PA_SLOTS : all % PA_SLOTS * deal_of(p.tiles_b, H, p.most).parts);
    }
    p.grid_a = pad8(p.units_a);
    p.by_share = Divisor::of(share);
    p.by_tiles_a = Divisor::of(std::max(p.tiles_a, 1));
    p.by_parts_a = Divisor::of(std::max(p.parts_a, 1));
    p.by_tiles_b = Divisor::of(std::max(p.tiles_b, 1));
    p.by_parts_b = Divisor::of(p.parts_b);
    return p;
}

namespace {
// Rows that parts have room for.
size_t part_rows(const PrefixPlan& p, int T, int H, int share, bool ragged) {
    if (p.packed) return (size_t)(p.parts_a + p.parts_b) * H * T * share;
    const Deal d = deal_of(p.tiles_b, H, p.most);
    if (!ragged) return d.parts == 1 ? 0 : (size_t)d.rest * d.parts * p.rows_b;
    // (fewer tiles than the launch has room for may be cut into more parts, of up to PA_SLOTS in all)
    return p.most == 1 ? 0 : (size_t)std::min<long>(PA_SLOTS, (long)p.tiles_b * H * p.most) * p.rows_b;
}
}  // namespace

size_t prefix_attention_workspace_bytes(int T, int B, int H, int share, int D, int P, int Lmax, bool ragged) {
    return part_rows(prefix_plan(T, B, H, share, P, Lmax, ragged), T, H, share, ragged) * (D + 2) * sizeof(float);
}

hipError_t launch_prefix_attention(const PrefixAttn& t, int D, float sm_scale, void* workspace, hipStream_t st) {
    PrefixArgs a;
    a.t = t;
    a.p = prefix_plan(t.T, t.B, t.H, t.share, t.P, t.Lmax, t.starts != nullptr);
    a.qk_scale = sm_scale * 1.44269504f;
    const size_t rows = part_rows(a.p, t.T, t.H, t.share, t.starts != nullptr);
    a.p.po = (float*)workspace;
    a.p.pml = (float2*)(a.p.po + rows * D);
    const dim3 pieces(a.p.grid_a + a.p.grid_b + (t.kn ? (t.T + 3) / 4 : 0));
#define SQ_PREFIX_LAUNCH(QA_, QB_)                                                                  \
    if (D == 64) hipLaunchKernelGGL((prefix_attn_kernel<64, QA_, QB_>), pieces, dim3(256), 0, st, a); \
    else hipLaunchKernelGGL((prefix_attn_kernel<128, QA_, QB_>), pieces, dim3(256), 0, st, a)
    if (a.p.qa == 1) {
        SQ_PREFIX_LAUNCH(1, 1);
    } else if (a.p.qa == 2) {
        SQ_PREFIX_LAUNCH(2, 1);
    } else if (a.p.qa == 4) {
        SQ_PREFIX_LAUNCH(4, 1);
    } else if (a.p.qb == 1) {
        SQ_PREFIX_LAUNCH(0, 1);
    } else if (a.p.qb == 2) {
        SQ_PREFIX_LAUNCH(0, 2);
    } else {
        SQ_PREFIX_LAUNCH(0, 4);
    }
#undef SQ_PREFIX_LAUNCH
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || rows == 0) return e;
    if (a.p.packed) {
        const dim3 grid(div_up((long)t.T * t.H * t.share, 4));
        if (D == 64) hipLaunchKernelGGL((prefix_join_kernel<64>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((prefix_join_kernel<128>), grid, dim3(256), 0, st, a);
    } else {
        const dim3 grid(a.p.rows_b / 16, std::min(PA_SLOTS - 1, a.p.tiles_b * t.H));
        if (D == 64) hipLaunchKernelGGL((prefix_join_tiles_kernel<64>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((prefix_join_tiles_kernel<128>), grid, dim3(256), 0, st, a);
    }
    return hipGetLastError();
}

}  // namespace sq
