// A key/value cache of a fixed number of rows that evicts by accumulated attention weight (fp16, one token per sequence).
//
// A step: where the cache is not full the token's row goes behind the others; where it is, the row of the lowest weight among
// those that are neither of the first `first` nor of the last `last` tokens makes way for it.  The token attends over the rows,
// its own among them, and every row's weight grows by what the token's heads give it:
//   P = softmax_j(scale q . k_j),  out = sum_j P_j v_j,  weight_j += sum over the query heads of the key/value head of P_j
// The probabilities are known only behind the last row, so the scores wait in the workspace (4 bytes of a row's 512 at D = 128).
//
// What bounds it: the bytes, 4.6 TB/s of them (32 sequences x 8 heads x 4000 rows of 128, four query heads each: 487 MB in 106 us);
// where there are few the chain of launch, first rows, the lowest weight, softmax, join and weights (8 sequences of 32 heads x 512
// rows, 57 MB in 13.0 us, one launch).  The weights are looked through behind the first requests, by every workgroup of a head, which
// costs 8 bytes a row from L2 and saves a launch in front.
#include "sq_attn_rows.h"
#include "sq_kernels.h"

#include <algorithm>
#include <type_traits>

namespace sq {

namespace {

constexpr int EV_TILE = 32;  // query heads of a workgroup

struct EvictArgs {
    EvictStep t;
    float* scores;  // [B][H][share][pitch], in units of log2
    float* po;      // [B][H][parts][share][D]
    float2* pml;    // [B][H][parts][share]
    int pitch, parts, blocks, tiles;
    Divisor by_parts, by_tiles, by_heads;
    float qk_scale;
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }
__device__ __forceinline__ int imax(int a, int b) { return a > b ? a : b; }

// Order of weights as unsigned numbers; a NaN is the lowest, and both zeros are the same (-0 + 0 is 0).
__device__ __forceinline__ uint32_t order_of(float w) {
    const uint32_t u = bit_cast<uint32_t>(w + 0.f);
    return w != w ? 0u : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ uint64_t wave_min64(uint64_t v) {
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        const uint64_t o = ((uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), x) << 32) | (uint32_t)__shfl_xor((int)v, x);
        v = o < v ? o : v;
    }
    return v;
}

// A sequence that has seen nothing.
template <int D>
__device__ __forceinline__ void nothing_seen(const EvictStep& t, int bh) {
    half_t* const out = t.o + (long)bh * t.share * D;
    for (int i = threadIdx.x; i < t.share * D; i += 256) out[i] = (half_t)0.f;
    if (threadIdx.x == 0) t.slot[bh] = -1;
}

// What the query heads g0 .. g0 + heads - 1 give to the rows r0 .. r0 + EJ_ROWS - 1 is added to their weights; state holds the
// heads' reference (in units of log2) and the reciprocal of their sum.  The row of the slot begins anew, with the first heads.
constexpr int EJ_ROWS = 1024;
__device__ __forceinline__ void add_weights(const EvictArgs& a, int bh, int r0, int n, int seen, int slot, const float2* state, int g0,
                                            int heads) {
    const EvictStep& t = a.t;
    const int r = r0 + 4 * threadIdx.x;
    if (r >= n) return;
    float* const w = t.weight + (long)bh * t.R + r;
    float4_t sum;
#pragma unroll
    for (int j = 0; j < 4; j++) sum[j] = r + j < n && !(r + j == slot && g0 == 0) ? w[j] : 0.f;
    const float* const from = a.scores + ((long)bh * t.share + g0) * a.pitch + r;
#pragma unroll 4
    for (int g = 0; g < heads; g++) {
        const float4_t s = *(const float4_t*)(from + (long)g * a.pitch);
        const float2 st = state[g];
#pragma unroll
        for (int j = 0; j < 4; j++) sum[j] += __builtin_amdgcn_exp2f(s[j] - st.x) * st.y;
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (r + j < n) w[j] = sum[j];
    if (slot >= r && slot < r + 4) t.position[(long)bh * t.R + slot] = seen - 1;
}

template <int D>
__global__ __launch_bounds__(256, 2) void evict_attn_kernel(EvictArgs a) {
    typedef RowsAttn<D> R;
    constexpr int CPR = R::CPR;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[R::LDS];
    __shared__ float2 stat[RA_WAVES * RA_BLOCK];
    __shared__ uint64_t least[RA_WAVES];
    __shared__ float2 state[EV_TILE];
    const EvictStep& t = a.t;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ln = lane & 31, lc = lane >> 5;
    const int rest = a.by_parts(blockIdx.x);
    const int part = blockIdx.x - rest * a.parts;
    const int bh = a.by_tiles(rest);
    const int tile = rest - bh * a.tiles;
    const int b = a.by_heads(bh), h = bh - b * t.H;
    const int seen = t.seen[b];
    const int n = imin(seen, t.R);  // rows attended
    const int blk0 = part * a.blocks, blk1 = imin(blk0 + a.blocks, ceil_div(n, RA_BLOCK));
    if (blk0 >= blk1) {  // (where there is a second launch it writes the zeros of a sequence that has seen nothing)
        if (a.parts == 1 && a.tiles == 1) nothing_seen<D>(t, bh);
        return;
    }

    const int rows = imin(EV_TILE, t.share - tile * EV_TILE);
    const int g = tile * EV_TILE + imin(ln, rows - 1);
    R r;
    r.load_query(t.q + (long)b * t.q_bs + (long)(h * t.share + g) * t.q_hs + 8 * lc);
    // The new row, a chunk of it per lane.
    const int chunk = lane % CPR;
    const long n_at = (long)b * t.n_bs + (long)h * t.n_hs + 8 * chunk;
    const u32x4_t fresh_k = *(const u32x4_t*)(t.kn + n_at);
    const u32x4_t fresh_v = *(const u32x4_t*)(t.vn + n_at);
    int slot = seen - 1;  // where it goes
    const long c_at = (long)b * t.c_bs + (long)h * t.c_hs;
    float* const scores = a.scores + ((long)bh * t.share + g) * a.pitch + 4 * lc;
    const bool valid = ln < rows;
    r.template run<true>(
        lds, blk0 + wave, blk1, a.qk_scale,
        [&]() {
            if (seen <= t.R) return;
            const float* const w = t.weight + (long)bh * t.R;
            const int* const pos = t.position + (long)bh * t.R;
            uint64_t best = ~0ull;
#pragma unroll 1
            for (int i0 = tid; i0 < t.R; i0 += 8 * 256) {
                int p[8];
                float v[8];
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    const int i = imin(i0 + u * 256, t.R - 1);  // (the last one again behind the last)
                    p[u] = pos[i];
                    v[u] = w[i];
                }
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    const uint32_t o = p[u] >= t.first && p[u] < seen - t.last ? order_of(v[u]) : ~0u;
                    const uint64_t key = ((uint64_t)o << 32) | (uint32_t)imin(i0 + u * 256, t.R - 1);
                    best = key < best ? key : best;
                }
            }
            best = wave_min64(best);
            if (lane == 0) least[wave] = best;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < RA_WAVES; i++) best = least[i] < best ? least[i] : best;
            slot = __builtin_amdgcn_readfirstlane((int)(uint32_t)best);
        },
        [&](int blk, bool value, uint32_t at) {
            const half_t* const base = (value ? t.vc : t.kc) + c_at;
            const int first = blk * RA_BLOCK;
            if (first + RA_BLOCK <= n)
                R::request((const uint8_t*)(base + (long)first * t.c_rs), (uint32_t)t.c_rs * 2, value, at);
            else  // rows past the end re-read the last one
                R::request_each(value, at, [&](int i) { return base + (long)imin(first + i, n - 1) * t.c_rs; });
        },
        [&](int blk, int& first, int& full, int& last) {
            first = blk * RA_BLOCK;
            full = n;
            last = n - 1;
        },
        [&](int blk, uint8_t* tile_at) {
            const int i = slot - blk * RA_BLOCK;
            if (i >= 0 && i < RA_BLOCK && lane < CPR) {  // the new row takes its place
                R::put(tile_at, false, i, chunk, fresh_k);
                if (tile == 0) *(u32x4_t*)(t.kc + c_at + (long)slot * t.c_rs + 8 * chunk) = fresh_k;
                if (tile == 0 && lane == 0) t.slot[bh] = slot;
            }
        },
        [&](int blk, uint8_t* tile_at) {
            const int i = slot - blk * RA_BLOCK;
            if (i >= 0 && i < RA_BLOCK && lane < CPR) {
                R::put(tile_at, true, i, chunk, fresh_v);
                if (tile == 0) *(u32x4_t*)(t.vc + c_at + (long)slot * t.c_rs + 8 * chunk) = fresh_v;
            }
            const int past = n - blk * RA_BLOCK;
            if (past < RA_BLOCK) R::clear_from(tile_at, past);
        },
        [&](int blk, const float16_t& st) {
            if (valid) {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    *(float4_t*)(scores + blk * RA_BLOCK + 8 * i) = (float4_t){st[4 * i], st[4 * i + 1], st[4 * i + 2], st[4 * i + 3]};
            }
        });
    const bool whole = a.parts == 1 && a.tiles == 1;  // nothing is left for a second launch
    half_t* const out = t.o + (long)bh * t.share * D;
    r.join(lds, stat, rows, [&](int i, int col, float4_t o, float m, float l) {
        if (whole) {
            half4_t x;
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = (half_t)(o[j] / l);
            *(half4_t*)(out + i * D + col) = x;
            if (col == 0) state[i] = make_float2(m, 1.f / l);
            return;
        }
        const long at = ((long)bh * a.parts + part) * t.share + tile * EV_TILE + i;
        *(float4_t*)(a.po + at * D + col) = o;
        if (col == 0) a.pml[at] = make_float2(m, l);
    });
    if (whole) {
        __syncthreads();  // (the scores are in L2, and so is what the waves wrote)
        for (int r0 = 0; r0 < n; r0 += EJ_ROWS) add_weights(a, bh, r0, n, seen, slot, state, 0, rows);
    }
}

// The parts of a (sequence, key/value head): its outputs (first chunk of rows), and the weights of a chunk of rows.
constexpr int EJ_HEADS = 64;  // whose maxima and sums are held at once

template <int D>
__global__ __launch_bounds__(256) void evict_join_kernel(EvictArgs a) {
    __shared__ float2 state[EJ_HEADS];
    const EvictStep& t = a.t;
    const int tid = threadIdx.x;
    const int bh = blockIdx.x, b = a.by_heads(bh);
    const int r0 = blockIdx.y * EJ_ROWS;
    const int seen = t.seen[b];
    const int n = imin(seen, t.R);
    if (r0 >= n && r0 > 0) return;
    if (seen <= 0) {
        nothing_seen<D>(t, bh);
        return;
    }
    half_t* const out = t.o + (long)bh * t.share * D;
    const int slot = t.slot[bh];
    const int parts = ceil_div(ceil_div(n, RA_BLOCK), a.blocks);
    for (int g0 = 0; g0 < t.share; g0 += EJ_HEADS) {
        const int heads = imin(EJ_HEADS, t.share - g0);
        const long first = (long)bh * a.parts * t.share + g0;
        __syncthreads();
        // a wave per head, lane s looks at part s
        for (int g = tid >> 6; g < heads; g += 4) {
            float2 all = make_float2(-INFINITY, 0.f);
            for (int s0 = 0; s0 < parts; s0 += 64) {
                const int s = s0 + (tid & 63);
                const float2 x = s < parts ? a.pml[first + (long)s * t.share + g] : make_float2(-INFINITY, 0.f);
                float m = fmaxf(x.x, all.x);
#pragma unroll
                for (int y = 1; y < 64; y <<= 1) m = fmaxf(m, __shfl_xor(m, y));
                float l = x.y * share_of(x, m);
#pragma unroll
                for (int y = 1; y < 64; y <<= 1) l += __shfl_xor(l, y);
                all = make_float2(m, all.y * share_of(all, m) + l);
            }
            if ((tid & 63) == 0) state[g] = make_float2(all.x, 1.f / all.y);
        }
        __syncthreads();
        add_weights(a, bh, r0, n, seen, slot, state, g0, heads);
        if (blockIdx.y == 0) {
            for (int i = tid; i < heads * (D / 4); i += 256) {
                const int g = i / (D / 4), c = 4 * (i % (D / 4));
                const float2 st = state[g];
                float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
                for (int s = 0; s < parts; s++) {
                    const long at = first + (long)s * t.share + g;
                    o += *(const float4_t*)(a.po + at * D + c) * share_of(a.pml[at], st.x);
                }
                half4_t x;
#pragma unroll
                for (int j = 0; j < 4; j++) x[j] = (half_t)(o[j] * st.y);
                *(half4_t*)(out + (g0 + g) * D + c) = x;
            }
        }
    }
}

// Workgroups that the caches' rows are cut for: one per CU, so that a chip full of heads needs no second launch (us, with 256 / 512 /
// 1024: 8 x 32 heads x 512 rows 16.6 / 19.6 / 24.1; 32 x 8 x 4000 107.5 / 109.4 / 109.0; 2 x 32 x 2000 22.4 / 22.3 / 27.9; 4 x 8 x 4000
// 24.7 / 24.6 / 31.5).
constexpr int EV_WGS = 256;

EvictArgs plan(int B, int H, int share, int R) {
    EvictArgs a = {};
    a.pitch = (R + 31) / 32 * 32;
    a.tiles = (share + EV_TILE - 1) / EV_TILE;
    const long units = (long)B * H * a.tiles;
    const int rounds = (a.pitch / RA_BLOCK + RA_WAVES - 1) / RA_WAVES;  // of the waves over the rows
    const int each = (int)std::max<long>((units * rounds + EV_WGS - 1) / EV_WGS, 1);
    a.blocks = each * RA_WAVES;
    a.parts = (rounds + each - 1) / each;
    a.by_parts = Divisor::of(a.parts);
    a.by_tiles = Divisor::of(a.tiles);
    a.by_heads = Divisor::of(H);
    return a;
}

// ------------------------------------------------------------------------------------------------ a prompt's rows

constexpr int KEEP_THREADS = 1024;
constexpr int KEEP_BINS = 2048;

// Of prompts of any length.  Which rows stay: the R of the highest weight, the first and last ones above all, the lower row among equals.  A search for
// the R-th highest weight by its digits from the top (11, 11 and 10 bits, counted in LDS), then one pass that writes the rows
// in their order.  One workgroup reads a head's weights four times, which bounds it (8 heads: 4 prompts of 40000 rows into 2000 89 us,
// of 131072 into 4000 279, one of a million 1670).
__global__ __launch_bounds__(KEEP_THREADS) void keep_select_kernel(EvictKeep t) {
    __shared__ int bins[KEEP_BINS];
    __shared__ int sums[KEEP_THREADS / 64][2];
    __shared__ int found[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int bh = blockIdx.x, b = bh / t.H, h = bh - b * t.H;
    int n = t.lengths ? t.lengths[b] : t.S;
    n = n < 0 ? 0 : imin(n, t.S);
    int* const rows = t.rows + (long)bh * t.R;
    if (n <= t.R) {
        for (int i = tid; i < t.R; i += KEEP_THREADS) rows[i] = i < n ? i : -1;
        return;
    }
    const float* const w = t.weight + (long)b * t.w_bs + (long)h * t.w_hs;
    auto key_of = [&](int r) { return r < t.first || r >= n - t.last ? ~0u : order_of(w[r]); };
    uint32_t prefix = 0;
    int need = t.R, shift = 32;  // of the keys that begin with `prefix`, so many
    for (int pass = 0; pass < 3; pass++) {
        const int bits = pass < 2 ? 11 : 10;
        const int low = shift - bits;
        for (int i = tid; i < KEEP_BINS; i += KEEP_THREADS) bins[i] = 0;
        __syncthreads();
        for (int r = tid; r < n; r += KEEP_THREADS) {
            const uint32_t key = key_of(r);
            if (pass == 0 || (key >> shift) == prefix) atomicAdd(&bins[(key >> low) & ((1u << bits) - 1)], 1);
        }
        __syncthreads();
        // counts from the highest bin down: thread i has bins 2047 - 2 i and 2046 - 2 i
        const int hi = bins[KEEP_BINS - 1 - 2 * tid], lo = bins[KEEP_BINS - 2 - 2 * tid];
        int upto = hi + lo;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) {
            const int v = __shfl_up(upto, x);
            if (lane >= x) upto += v;
        }
        if (lane == 63) sums[wave][0] = upto;
        __syncthreads();
        for (int i = 0; i < wave; i++) upto += sums[i][0];
        const int before = upto - hi - lo;
        if (before < need && before + hi >= need) {
            found[0] = KEEP_BINS - 1 - 2 * tid;
            found[1] = need - before;
        } else if (before + hi < need && upto >= need) {
            found[0] = KEEP_BINS - 2 - 2 * tid;
            found[1] = need - before - hi;
        }
        __syncthreads();
        prefix = (prefix << bits) | (uint32_t)found[0];
        need = found[1];
        shift = low;
        __syncthreads();
    }
    // keys above `prefix`, and of those equal to it the first `need`
    int taken = 0, equal = 0;
    for (int r0 = 0; r0 < n; r0 += KEEP_THREADS) {
        const int r = r0 + tid;
        const uint32_t key = r < n ? key_of(r) : 0u;
        const bool eq = r < n && key == prefix;
        const uint64_t below = (1ull << lane) - 1;
        const uint64_t eqs = __ballot(eq);
        const uint64_t above = __ballot(r < n && key > prefix);
        if (lane == 0) {
            sums[wave][0] = __popcll(eqs);
            sums[wave][1] = __popcll(above);
        }
        __syncthreads();
        int e = equal, k = taken;
        for (int i = 0; i < KEEP_THREADS / 64; i++) {
            if (i < wave) {
                e += sums[i][0];
                k += sums[i][1];
            }
            equal += sums[i][0];
            taken += sums[i][1];
        }
        // rows taken so far: those above, and of the equal ones at most `need`
        const int e_mine = e + __popcll(eqs & below);
        const int place = k + __popcll(above & below) + imin(e_mine, need);
        if (r < n && (key > prefix || (eq && e_mine < need))) rows[place] = r;
        __syncthreads();
    }
}

template <int D>
__global__ __launch_bounds__(256) void keep_gather_kernel(EvictKeep t) {
    constexpr int CPR = D / 8;
    constexpr int RPW = 256 / CPR;  // rows of a workgroup and pass
    const int bh = blockIdx.y, b = bh / t.H, h = bh - b * t.H;
    const int c = threadIdx.x % CPR;
    const int j = blockIdx.x * RPW + threadIdx.x / CPR;
    if (j >= t.R) return;
    const int r = t.rows[(long)bh * t.R + j];
    if (r < 0) return;
    const long from = (long)b * t.k_bs + (long)h * t.k_hs + (long)r * t.k_rs + 8 * c;
    const long to = (long)b * t.c_bs + (long)h * t.c_hs + (long)j * t.c_rs + 8 * c;
    *(u32x4_t*)(t.kc + to) = *(const u32x4_t*)(t.k + from);
    *(u32x4_t*)(t.vc + to) = *(const u32x4_t*)(t.v + from);
    if (c == 0) {
        t.cweight[(long)bh * t.R + j] = t.weight[(long)b * t.w_bs + (long)h * t.w_hs + r];
        t.cposition[(long)bh * t.R + j] = r;
    }
}

// The same for prompts whose weights fit LDS, and the rows copied by the same workgroup (in two launches 16 x 8 heads of 20000 rows
// take 95 us instead of 69, 8 x 32 of 512 rows 24.5 instead of 17.4): several share a head where there are few, and each of
// them makes the choice.  (With the weights in registers the code is a copy of each loop for every one of them,
// and fetching it takes longer than the loops.)  The threshold is found between the
// lowest and the highest weight, of whose distance every pass looks at 11 bits: counted by the weights' own digits, most of
// them fall on a few counters (the numbers of one power of two have one), and LDS takes them one at a time.
constexpr int KEEP_LIST = 4096;  // places of a workgroup
// Workgroups that the places are cut for, of 256 places or more each (us, with 128 / 256 / 512 / 1024: 16 x 8 heads, 20000 rows into 2000
// 94 / 68.7 / 69.7 / 81; 32 x 8, 2000 into 500 28.3 / 28.3 / 31.9 / 31.7; 8 x 32, 512 into 256, two workgroups of 128
// places a head instead of one 23.6 / 17.4).
constexpr int KEEP_WGS = 256;

constexpr int KEEP_MOST = 32 * KEEP_THREADS;  // rows of a prompt

template <int D>
__global__ __launch_bounds__(KEEP_THREADS) void keep_kernel(EvictKeep t, int each) {
    constexpr int WAVES = KEEP_THREADS / 64;
    __shared__ int bins[KEEP_BINS];
    extern __shared__ uint32_t keys[];  // a thread reads its own
    __shared__ uint32_t counts[KEEP_MOST / 64];  // of a wave's 64 rows: above the threshold (from bit 16 on), equal to it
    __shared__ uint32_t sums[WAVES];
    __shared__ uint32_t found[4];
    __shared__ uint64_t left[64];
    __shared__ int list[KEEP_LIST];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int bh = blockIdx.y, b = bh / t.H, h = bh - b * t.H;
    const int j0 = blockIdx.x * each, j1 = imin(j0 + each, t.R);  // the places that are this workgroup's
    int n = t.lengths ? t.lengths[b] : t.S;
    n = n < 0 ? 0 : imin(n, t.S);
    int* const rows = t.rows + (long)bh * t.R;
    const float* const w = t.weight + (long)b * t.w_bs + (long)h * t.w_hs;
    if (n <= t.R) {
        for (int j = j0 + tid; j < j1; j += KEEP_THREADS) {
            rows[j] = j < n ? j : -1;
            list[j - j0] = j < n ? j : -1;
        }
    } else {
        uint32_t low = ~0u, high = 0u;
        const int last = n - t.last, groups = ceil_div(n, KEEP_THREADS);
#pragma unroll 4
        for (int r = tid; r < n; r += KEEP_THREADS) {
            const bool forced = r < t.first || r >= last;
            const uint32_t key = forced ? ~0u : order_of(w[r]);
            keys[r] = key;
            low = !forced && key < low ? key : low;
            high = !forced && key > high ? key : high;
        }
        if (tid == 0) found[0] = ~0u, found[1] = 0u;
        __syncthreads();
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) {
            const uint32_t l = __shfl_xor((int)low, x), g = __shfl_xor((int)high, x);
            low = l < low ? l : low;
            high = g > high ? g : high;
        }
        if (lane == 0) {
            atomicMin(&found[0], low);
            atomicMax(&found[1], high);
        }
        __syncthreads();
        low = found[0], high = found[1];
        int need = t.R - imin(t.first, n) - t.last;  // of the keys in [low, high] the highest
        if (need <= 0) low = high = ~0u;             // (only the forced ones)
        while (low < high) {
            const int shift = imax(32 - __builtin_clz(high - low) - 11, 0);
            for (int i = tid; i < KEEP_BINS; i += KEEP_THREADS) bins[i] = 0;
            __syncthreads();
#pragma unroll 4
            for (int r = tid; r < n; r += KEEP_THREADS) {
                const uint32_t key = keys[r];
                if (key >= low && key <= high) atomicAdd(&bins[(key - low) >> shift], 1);
            }
            __syncthreads();
            // counts from the highest bin down: thread i has bins 2047 - 2 i and 2046 - 2 i
            const int hi = bins[KEEP_BINS - 1 - 2 * tid], lo = bins[KEEP_BINS - 2 - 2 * tid];
            int upto = hi + lo;
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) {
                const int v = __shfl_up(upto, x);
                if (lane >= x) upto += v;
            }
            if (lane == 63) sums[wave] = upto;
            __syncthreads();
            for (int i = 0; i < wave; i++) upto += sums[i];
            const int before = upto - hi - lo;
            if (before < need && upto >= need) {
                const bool first = before + hi >= need;
                found[2] = KEEP_BINS - (first ? 1 : 2) - 2 * tid;
                found[3] = need - before - (first ? 0 : hi);
                found[1] = first ? hi : lo;
                found[0] = 0;
            }
            __syncthreads();
            const uint32_t from = low + (found[2] << shift);
            need = (int)found[3];
            const uint32_t to = from + ((1u << shift) - 1);
            high = to < high ? to : high;
            low = from;
            const int count = (int)found[1];
            if (shift == 0 || count > 64) continue;
            // few are left: each is compared with all of them
            for (int r = tid; r < n; r += KEEP_THREADS) {
                const uint32_t key = keys[r];
                if (key >= low && key <= high) left[atomicAdd(&found[0], 1u)] = ((uint64_t)key << 32) | (uint32_t)~r;
            }
            __syncthreads();
            if (tid < count) {
                const uint64_t mine = left[tid];
                int better = 0, higher = 0;
                for (int i = 0; i < count; i++) {
                    better += left[i] > mine;
                    higher += (left[i] >> 32) > (mine >> 32);
                }
                if (better == need - 1) {  // the last that stays
                    found[2] = (uint32_t)(mine >> 32);
                    found[3] = need - higher;
                }
            }
            __syncthreads();
            low = high = found[2];
            need = (int)found[3];
        }
        // rows above the threshold (the forced ones are), of those equal to it the first `need`: how many each wave's 64 have
        if (low == ~0u) low = ~0u - 1, need = 0;
        const uint64_t below = (1ull << lane) - 1;
        for (int i = 0; i < groups; i++) {
            const int r = i * KEEP_THREADS + tid;
            const uint32_t key = r < n ? keys[r] : 0u;
            const uint64_t above = __ballot(r < n && key > low), equal = __ballot(r < n && key == low);
            if (lane == 0) counts[i * WAVES + wave] = ((uint32_t)__popcll(above) << 16) | (uint32_t)__popcll(equal);
        }
        __syncthreads();
        uint32_t upto = tid < groups * WAVES ? counts[tid] : 0u;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) {
            const uint32_t v = __shfl_up((int)upto, x);
            if (lane >= x) upto += v;
        }
        if (lane == 63) sums[wave] = upto;
        __syncthreads();
        if (tid < groups * WAVES) {
            for (int i = 0; i < wave; i++) upto += sums[i];
            counts[tid] = upto - counts[tid];
        }
        __syncthreads();
        for (int i = 0; i < groups; i++) {
            const int r = i * KEEP_THREADS + tid;
            const uint32_t key = r < n ? keys[r] : 0u;
            const bool is_above = r < n && key > low, is_equal = r < n && key == low;
            const uint64_t above = __ballot(is_above), equal = __ballot(is_equal);
            const uint32_t front = counts[i * WAVES + wave];
            const int e = (int)(front & 0xffffu) + __popcll(equal & below);
            const int place = (int)(front >> 16) + __popcll(above & below) + imin(e, need);
            if (is_above || (is_equal && e < need)) {
                if (blockIdx.x == 0) rows[place] = r;
                if (place >= j0 && place < j1) list[place - j0] = r;
            }
        }
    }
    __syncthreads();
    constexpr int CPR = D / 8, RPP = KEEP_THREADS / CPR, AHEAD = 4;  // rows of a pass, passes under way
    const int c = tid % CPR;
    for (int i0 = tid / CPR; i0 < j1 - j0; i0 += AHEAD * RPP) {
        u32x4_t k[AHEAD], v[AHEAD];
        int r[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            r[u] = i0 + u * RPP < j1 - j0 ? list[i0 + u * RPP] : -1;
            const long from = (long)b * t.k_bs + (long)h * t.k_hs + (long)imax(r[u], 0) * t.k_rs + 8 * c;
            if (r[u] >= 0) {
                k[u] = __builtin_nontemporal_load((const u32x4_t*)(t.k + from));
                v[u] = __builtin_nontemporal_load((const u32x4_t*)(t.v + from));
            }
        }
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            if (r[u] < 0) continue;
            const int j = j0 + i0 + u * RPP;
            const long to = (long)b * t.c_bs + (long)h * t.c_hs + (long)j * t.c_rs + 8 * c;
            *(u32x4_t*)(t.kc + to) = k[u];
            *(u32x4_t*)(t.vc + to) = v[u];
            if (c == 0) {
                t.cweight[(long)bh * t.R + j] = w[r[u]];
                t.cposition[(long)bh * t.R + j] = r[u];
            }
        }
    }
}

}  // namespace

size_t evict_attention_workspace_bytes(int B, int H, int share, int D, int R) {
    const EvictArgs a = plan(B, H, share, R);
    return ((size_t)B * H * share * a.pitch + (size_t)B * H * share * a.parts * (D + 2)) * sizeof(float);
}

hipError_t launch_evict_attention(const EvictStep& t, int D, float sm_scale, void* workspace, hipStream_t st) {
    EvictArgs a = plan(t.B, t.H, t.share, t.R);
    a.t = t;
    a.qk_scale = sm_scale * 1.44269504f;
    a.scores = (float*)workspace;
    a.po = a.scores + (size_t)t.B * t.H * t.share * a.pitch;
    a.pml = (float2*)(a.po + (size_t)t.B * t.H * t.share * a.parts * D);
    const dim3 grid(t.B * t.H * a.tiles * a.parts), join(t.B * t.H, (t.R + EJ_ROWS - 1) / EJ_ROWS);
    if (D == 64) hipLaunchKernelGGL((evict_attn_kernel<64>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((evict_attn_kernel<128>), grid, dim3(256), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || (a.parts == 1 && a.tiles == 1)) return e;
    if (D == 64) hipLaunchKernelGGL((evict_join_kernel<64>), join, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((evict_join_kernel<128>), join, dim3(256), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_evict_keep(const EvictKeep& t, int D, hipStream_t st) {
    const int heads = t.B * t.H;
    if (t.S <= KEEP_MOST) {
        // (every workgroup of a head makes the whole choice)
        const int share = std::max((t.R + KEEP_LIST - 1) / KEEP_LIST, std::min((KEEP_WGS + heads - 1) / heads, (t.R + 255) / 256));
        const int each = (t.R + share - 1) / share;
        const dim3 grid((t.R + each - 1) / each, heads);
        const int lds = t.S * 4;
        if (lds > 32 * 1024) {
            const hipError_t e = hipFuncSetAttribute(D == 64 ? (const void*)keep_kernel<64> : (const void*)keep_kernel<128>,
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, KEEP_MOST * 4);
            if (e != hipSuccess) return e;
        }
        if (D == 64) hipLaunchKernelGGL((keep_kernel<64>), grid, dim3(KEEP_THREADS), lds, st, t, each);
        else hipLaunchKernelGGL((keep_kernel<128>), grid, dim3(KEEP_THREADS), lds, st, t, each);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(keep_select_kernel, dim3(heads), dim3(KEEP_THREADS), 0, st, t);
    const int per = 256 / (D / 8);
    const dim3 grid((t.R + per - 1) / per, heads);
    if (D == 64)
        hipLaunchKernelGGL((keep_gather_kernel<64>), grid, dim3(256), 0, st, t);
    else
        hipLaunchKernelGGL((keep_gather_kernel<128>), grid, dim3(256), 0, st, t);
    return hipGetLastError();
}

}  // namespace sq
