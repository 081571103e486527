// Attention over a key/value cache held in 4 bits (layout: sq_kv4.h).
//
//   out[t, h, :] = sum_j P[j] v_hat[j, :],  P = softmax_j(sm_scale * q[t, h, :] . k_hat[j, :])
//
// over the rows j of token t's sequence up to its own (its last `count` rows are those of this call), or over the rows
// of selected pages only; x_hat = s code + m per row and group of g elements.
//
// Neither operand is ever dequantised.  Per row j and group: q . k_hat = s (q . code) + m sum(q), and with P' = P s:
// sum_j P k_hat = sum_j P' code + sum_j P m.  Codes enter the matrix instruction as they are: a nibble masked in
// place is the denormal fp16 number code * 2^-24 (bits 0..3) or code * 2^-20 (bits 4..7), exact, so eight codes cost a
// shift and four masks, nothing is subtracted, and the powers of two leave with the fp32 result.
//   S   = K Q^T  v_mfma_f32_16x16x32_f16, A = codes (row = key), B = q: a lane has one query and four keys of 16
//   O^T = V^T P' A = codes (row = column of V), B = P': the keys that the lane already has, in that order; the two rows
//                whose codes share a register come together by one byte permutation of two words
// The sum is one of P' (code - 8) and of P (m + 8 s): a second product of P' with the constant -8 follows the codes' own,
// within every 32 rows.  The rounding of P' to fp16 then acts on s (code - 8), about the size of v, and not on s code, which
// is twice that; and the fp32 sums stay as small as the result, where those of positive codes alone, which the matrix
// instruction rounds towards zero, lose the more of it the longer the cache is (131072 rows: error 5.4e-4 of the result
// instead of 2.8e-4, the rounding of P' and of the output).  P' is kept inside fp16's range by a power of two per group that
// follows the scales.
#include "sq_kernels.h"
#include "sq_kv4.h"

#include <type_traits>

namespace sq {

namespace {

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
};

// How a launch's work is dealt.  A tile is R of the rows (token, query head) of a sequence and key/value head; a
// workgroup takes one tile over a share of its pages.  The share's length follows from the lengths on the device: the pages
// of all tiles over 2^log_wgs workgroups, `least` at the fewest.
struct Deal {
    int log_wgs, least;
};
struct Piece {
    int b, tile, head, share, shares;  // share of how many
    int slot;                          // where its partial state goes (shares > 1)
    int first, count, len;             // tokens and rows of the sequence
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <int R>
__device__ __forceinline__ int deal_sizes(const Kv4AttnArgs& a, int b, int& first, int& count, int& len, int& pages) {
    kv4_tokens(a.c, b, first, count);
    len = kv4_length(a.c, b);
    pages = ceil_div(len, KV4_PAGE);
    if (a.selected && pages > a.count) pages = a.count;
    return ceil_div(count * a.share, R) * a.c.H;  // tiles
}

// The piece of workgroup `index` (SPLIT: of the index-th tile among those that are shared), by every wave alone.
template <int R, bool SPLIT>
__device__ __forceinline__ bool deal(const Kv4AttnArgs& a, const Deal& d, int index, Piece& out) {
    const int lane = threadIdx.x & 63;
    const int B = a.c.B;
    int least = d.least;
    if (a.ws) {
        unsigned long long units = 0;
        for (int b = lane; b < B; b += 64) {
            int f, n, l, p;
            const int tiles = deal_sizes<R>(a, b, f, n, l, p);
            units += (unsigned long long)tiles * p;
        }
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) units += __shfl_xor(units, x, 64);
        const int even = (int)((units + (1ull << d.log_wgs) - 1) >> d.log_wgs);
        least = even > least ? even : least;
    } else {
        least = 1 << 30;
    }
    int slots = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        const int b = b0 + lane;
        int f = 0, n = 0, l = 0, p = 0, tiles = 0;
        if (b < B) tiles = deal_sizes<R>(a, b, f, n, l, p);
        const int shares = p > least ? ceil_div(p, least) : 1;
        const int mine = SPLIT ? (shares > 1 ? tiles : 0) : tiles * shares;
        const int upto = wave_scan(mine);
        const int taken = shares > 1 ? tiles * shares : 0;
        const int slots_upto = wave_scan(taken);
        const unsigned long long past = __ballot(upto > index);
        if (past) {
            const int at = __ffsll(past) - 1;
            const int rest = index - __shfl(upto - mine, at, 64);
            out.shares = __shfl(shares, at, 64);
            const int tile = SPLIT ? rest : rest / out.shares;
            out.b = b0 + at;
            out.share = SPLIT ? 0 : rest - tile * out.shares;
            out.head = tile % a.c.H;
            out.tile = tile / a.c.H;
            out.slot = slots + __shfl(slots_upto - taken, at, 64) + tile * out.shares + out.share;
            out.first = __shfl(f, at, 64);
            out.count = __shfl(n, at, 64);
            out.len = __shfl(l, at, 64);
            return true;
        }
        index -= __shfl(upto, 63, 64);
        slots += __shfl(slots_upto, 63, 64);
    }
    return false;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) v = fmaxf(v, __shfl_xor(v, x, 64));
    return v;
}
__device__ __forceinline__ float rows_sum(float v) {  // over the four lanes of a query
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}
__device__ __forceinline__ float rows_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}

constexpr int KA_WAVES = 4;
constexpr int KA_ROWS = 16;
constexpr float KA_LAZY = 8.f;  // the softmax's reference moves when a score is 2^8 beyond it

// Half a page (32 rows) as a lane holds it.
template <int D, int G>
struct Half {
    uint32_t k[2][D / 32];  // [16 rows][words of the lane's row and chunk]
    u32x4_t v[2];
    half8_t ksm[2][G], vsm[2][G];  // scales and minima of four rows
};

template <int D, int G>
__global__ __launch_bounds__(64 * KA_WAVES) void kv4_attn_kernel(Kv4AttnArgs a, Deal d) {
    constexpr int g = D / G;
    constexpr int REC = kv4_record_bytes(D, g);
    constexpr int NT = D / 16;    // tiles of 16 columns
    constexpr int PITCH = D + 4;  // of a row of partial outputs: the 16 queries of a store fall on different banks
    __shared__ __attribute__((aligned(16))) float part[KA_WAVES][KA_ROWS][PITCH];
    __shared__ float state[KA_WAVES][KA_ROWS][2];

    const Kv4Cache& c = a.c;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Piece pc;
    if (!deal<KA_ROWS, false>(a, d, blockIdx.x, pc)) return;
    if (pc.shares > 1 && pc.slot >= 2 << d.log_wgs) return;  // (only where lengths change under the launch)
    const int b = __builtin_amdgcn_readfirstlane(pc.b), head = __builtin_amdgcn_readfirstlane(pc.head);
    const int tile = __builtin_amdgcn_readfirstlane(pc.tile), shares = __builtin_amdgcn_readfirstlane(pc.shares);
    const int share = __builtin_amdgcn_readfirstlane(pc.share), slot = __builtin_amdgcn_readfirstlane(pc.slot);
    const int first = __builtin_amdgcn_readfirstlane(pc.first), count = __builtin_amdgcn_readfirstlane(pc.count);
    const int len = __builtin_amdgcn_readfirstlane(pc.len);

    // This lane's query: row n of the tile.
    const int n = lane & 15, l4 = lane >> 4;
    const int rows = imin(count * a.share - tile * KA_ROWS, KA_ROWS);
    const int row = tile * KA_ROWS + imin(n, rows - 1);
    const int token = row / a.share, qhead = head * a.share + row % a.share;
    const int limit = len - count + token;  // the last row it sees
    const int limit_lo = len - count + tile * KA_ROWS / a.share;
    const int limit_hi = len - count + (tile * KA_ROWS + rows - 1) / a.share;
    const int all_pages = ceil_div(imin(limit_hi + 1, len) > 0 ? imin(limit_hi + 1, len) : 0, KV4_PAGE);
    // (selected pages are for single tokens: limit_hi + 1 = len)
    const int pages = a.selected ? imin(all_pages, a.count) : all_pages;
    const int p0 = (int)((long)pages * share / shares), p1 = (int)((long)pages * (share + 1) / shares);

    half8_t qf[D / 32];
    float qsum[G];
    {
        const half_t* src = a.q + (long)(first + token) * a.q_ts + (long)qhead * a.q_hs + 8 * l4;
#pragma unroll
        for (int i = 0; i < G; i++) qsum[i] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
            qf[i] = *(const half8_t*)(src + 32 * i);
#pragma unroll
            for (int e = 0; e < 8; e++) qsum[32 * i / g] += (float)qf[i][e];
        }
#pragma unroll
        for (int i = 0; i < G; i++) qsum[i] = rows_sum(qsum[i]) * a.scale;
    }

    float4_t acc[NT];
#pragma unroll
    for (int i = 0; i < NT; i++) acc[i] = (float4_t){0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;     // the reference of the softmax (of this query), the lane's share of the sum
    float mins[G], sref[G];           // sum P (m + 8 s) (the lane's share), power of two in P'
#pragma unroll
    for (int i = 0; i < G; i++) mins[i] = 0.f, sref[i] = 0x1p-30f;
    const half8_t eight[2] = {bit_cast<half8_t>((u32x4_t){0x80088008u, 0x80088008u, 0x80088008u, 0x80088008u}),   // -8 * 2^-24
                              bit_cast<half8_t>((u32x4_t){0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u})};  // -8 * 2^-20
    const float scale24 = a.scale * 0x1p24f;
    const NibbleMasks nm = nibble_masks();
    const uint32_t voff = (D == 128 ? n : (n & 7)) * 16;
    const uint32_t vsel = D == 64 && n >= 8 ? 0x07060302u : 0x05040100u;

    const int* const table = c.table + (long)b * c.table_stride;
    const int* const chosen = a.selected ? a.selected + ((long)b * c.H + head) * a.count : nullptr;
    // Pages are looked up 64 at a time: lane i has the i-th one's place in the sequence and in the pool.
    for (int pb = p0; pb < p1; pb += 64) {
        int place = pb + lane, id = -1;
        if (place < p1) {
            if (chosen) place = chosen[place];
            if ((unsigned)place < (unsigned)all_pages) id = table[place];
            if ((unsigned)id >= (unsigned)c.num_pages) id = -1;
        }
        if (id < 0) place = 0;  // a page that does not exist: its rows lie behind every query's last
        const int units = 2 * imin(64, p1 - pb);
        auto load = [&](int u, Half<D, G>& x) {
            const int pid = __builtin_amdgcn_readlane(id, u >> 1);
            const uint8_t* const rec = c.pool + ((long)(pid < 0 ? 0 : pid) * c.H + head) * REC;
            const int r0 = 32 * (u & 1);
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const uint8_t* ks = rec + (r0 + 16 * t + n) * (D / 2) + l4 * (D / 8);
                if constexpr (D == 128) {
                    const u32x4_t w = *(const u32x4_t*)ks;
#pragma unroll
                    for (int i = 0; i < 4; i++) x.k[t][i] = w[i];
                } else {
                    const u32x2_t w = *(const u32x2_t*)ks;
                    x.k[t][0] = w[0];
                    x.k[t][1] = w[1];
                }
                const int quad = (r0 + 16 * t) / 4 + l4;
                x.v[t] = *(const u32x4_t*)(rec + 32 * D + quad * (2 * D) + voff);
#pragma unroll
                for (int i = 0; i < G; i++) {
                    x.ksm[t][i] = *(const half8_t*)(rec + 64 * D + (i * 16 + quad) * 16);
                    x.vsm[t][i] = *(const half8_t*)(rec + 64 * D + 256 * G + (i * 16 + quad) * 16);
                }
            }
        };
        auto consume = [&](int u, const Half<D, G>& x) {
            const int pid = __builtin_amdgcn_readlane(id, u >> 1);
            const int pos0 = __builtin_amdgcn_readlane(place, u >> 1) * KV4_PAGE + 32 * (u & 1);
            float s[8];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                float4_t even[G], odd[G];
#pragma unroll
                for (int i = 0; i < G; i++) even[i] = odd[i] = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int p = 0; p < D / 64; p++) {
                    const uint32_t w0 = x.k[t][2 * p], w1 = x.k[t][2 * p + 1], h0 = w0 >> 8, h1 = w1 >> 8;
                    const u32x4_t lo = {w0 & nm.lo, w1 & nm.lo, h0 & nm.lo, h1 & nm.lo};
                    const u32x4_t hi = {w0 & nm.hi, w1 & nm.hi, h0 & nm.hi, h1 & nm.hi};
                    const int ie = 64 * p / g, io = (64 * p + 32) / g;
                    even[ie] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bit_cast<half8_t>(lo), qf[2 * p], even[ie], 0, 0, 0);
                    odd[io] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bit_cast<half8_t>(hi), qf[2 * p + 1], odd[io], 0, 0, 0);
                }
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float codes = 0.f, shift = 0.f;
#pragma unroll
                    for (int i = 0; i < G; i++) {
                        const float sum = odd[i][r] * 0.0625f + even[i][r];
                        codes += (float)x.ksm[t][i][r] * sum;
                        shift += (float)x.ksm[t][i][4 + r] * qsum[i];
                    }
                    s[4 * t + r] = codes * scale24 + shift;
                }
            }
            bool vis[8];
#pragma unroll
            for (int j = 0; j < 8; j++) vis[j] = true;
            if (pid < 0 || pos0 + 31 > limit_lo) {  // some row is not there, or not for every query
                const int last = pid < 0 ? -1 : limit;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    vis[j] = pos0 + 16 * (j >> 2) + 4 * l4 + (j & 3) <= last;
                    if (!vis[j]) s[j] = -INFINITY;
                }
            }
            float top = s[0];
#pragma unroll
            for (int j = 1; j < 8; j++) top = fmaxf(top, s[j]);
            if (__ballot(top > m + KA_LAZY)) {
                const float to = fmaxf(rows_max(top), m);
                const float f = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - to);
                m = to;
                l *= f;
#pragma unroll
                for (int i = 0; i < NT; i++) acc[i] *= f;
#pragma unroll
                for (int i = 0; i < G; i++) mins[i] *= f;
            }
            const float ref = m == -INFINITY ? 0.f : m;
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                p[j] = __builtin_amdgcn_exp2f(s[j] - ref);
                l += p[j];
            }
            half8_t pf[G];
#pragma unroll
            for (int i = 0; i < G; i++) {
                float sv[8], mv[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    sv[j] = (float)x.vsm[j >> 2][i][j & 3];
                    mv[j] = (float)x.vsm[j >> 2][i][4 + (j & 3)];
                    if (!vis[j]) sv[j] = mv[j] = 0.f;  // whatever lies there
                }
                float big = sv[0];
#pragma unroll
                for (int j = 1; j < 8; j++) big = fmaxf(big, sv[j]);
                if (__ballot(big > 8.f * sref[i])) {
                    const float to = bit_cast<float>(bit_cast<uint32_t>(wave_max(big)) & 0x7f800000u) * 2.f;
                    const float f = sref[i] / to;
                    sref[i] = to;
#pragma unroll
                    for (int k = i * g / 16; k < (i + 1) * g / 16; k++) acc[k] *= f;
                }
                const float inv = 16.f / sref[i];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    pf[i][j] = (half_t)(p[j] * (sv[j] * inv));
                    mins[i] += p[j] * (8.f * sv[j] + mv[j]);
                }
            }
            uint32_t lo[4];
            auto products = [&](int tile0) {
                uint32_t up[4];
#pragma unroll
                for (int j = 0; j < 4; j++) up[j] = lo[j] >> 8;
                const u32x4_t a0 = {lo[0] & nm.lo, lo[1] & nm.lo, lo[2] & nm.lo, lo[3] & nm.lo};
                const u32x4_t a1 = {lo[0] & nm.hi, lo[1] & nm.hi, lo[2] & nm.hi, lo[3] & nm.hi};
                const u32x4_t a2 = {up[0] & nm.lo, up[1] & nm.lo, up[2] & nm.lo, up[3] & nm.lo};
                const u32x4_t a3 = {up[0] & nm.hi, up[1] & nm.hi, up[2] & nm.hi, up[3] & nm.hi};
                const u32x4_t op[4] = {a0, a1, a2, a3};
#pragma unroll
                for (int k = 0; k < 4; k++)
                    acc[tile0 + k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bit_cast<half8_t>(op[k]), pf[16 * (tile0 + k) / g],
                                                                            acc[tile0 + k], 0, 0, 0);
#pragma unroll
                for (int k = 0; k < 4; k++)
                    acc[tile0 + k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight[k & 1], pf[16 * (tile0 + k) / g], acc[tile0 + k],
                                                                            0, 0, 0);
            };
#pragma unroll
            for (int j = 0; j < 4; j++)
                lo[j] = __builtin_amdgcn_perm(x.v[j >> 1][2 * (j & 1) + 1], x.v[j >> 1][2 * (j & 1)], vsel);
            products(0);
            if constexpr (D == 128) {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    lo[j] = __builtin_amdgcn_perm(x.v[j >> 1][2 * (j & 1) + 1], x.v[j >> 1][2 * (j & 1)], 0x07060302u);
                products(4);
            }
        };
        Half<D, G> x0, x1;
        int u = wave;
        if (u < units) {
            load(u, x0);
            while (u < units) {
                if (u + KA_WAVES < units) load(u + KA_WAVES, x1);
                consume(u, x0);
                u += KA_WAVES;
                if (u >= units) break;
                if (u + KA_WAVES < units) load(u + KA_WAVES, x0);
                consume(u, x1);
                u += KA_WAVES;
            }
        }
    }

    // The wave's output over its rows, then the workgroup's.
    l = rows_sum(l);
#pragma unroll
    for (int i = 0; i < G; i++) mins[i] = rows_sum(mins[i]);
    if (n < rows) {
#pragma unroll
        for (int i = 0; i < NT; i++) {
            const int gi = 16 * i / g;
            const float f = sref[gi] * 0.0625f, fc = f * (i & 1 ? 0x1p20f : 0x1p24f), base = mins[gi];
            *(float4_t*)&part[wave][n][16 * i + 4 * l4] = (float4_t){acc[i][0] * fc + base, acc[i][1] * fc + base,
                                                                     acc[i][2] * fc + base, acc[i][3] * fc + base};
        }
        if (l4 == 0) {
            state[wave][n][0] = m;
            state[wave][n][1] = l;
        }
    }
    __syncthreads();
    constexpr int C4 = D / 4;
    for (int i = threadIdx.x; i < rows * C4; i += 64 * KA_WAVES) {
        const int r = i / C4, c4 = i % C4;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < KA_WAVES; w++) mx = fmaxf(mx, state[w][r][0]);
        float sum = 0.f;
        float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < KA_WAVES; w++) {
            const float mw = state[w][r][0];
            const float f = mw == -INFINITY ? (mx == -INFINITY ? 1.f : 0.f) : __builtin_amdgcn_exp2f(mw - mx);
            sum += state[w][r][1] * f;
            o += *(const float4_t*)&part[w][r][4 * c4] * f;
        }
        if (shares == 1) {
            const int rr = tile * KA_ROWS + r;
            const float inv = sum == 0.f ? 0.f : 1.f / sum;  // nothing visible: 0
            half4_t h;
#pragma unroll
            for (int e = 0; e < 4; e++) h[e] = (half_t)(o[e] * inv);
            *(half4_t*)(a.out + ((long)(first + rr / a.share) * c.H * a.share + head * a.share + rr % a.share) * D + 4 * c4) = h;
        } else {
            float* const dst = a.ws + (long)slot * KA_ROWS * (D + 2);
            *(float4_t*)(dst + r * D + 4 * c4) = o;
            if (c4 == 0) {
                dst[KA_ROWS * D + 2 * r] = mx;
                dst[KA_ROWS * D + 2 * r + 1] = sum;
            }
        }
    }
}

// Shares of a tile's pages, joined: a workgroup per row of a shared tile.
template <int D, int R>
__global__ __launch_bounds__(256) void kv4_join_kernel(Kv4AttnArgs a, Deal d) {
    constexpr int C4 = D / 4, LANES = 256 / C4;
    __shared__ __attribute__((aligned(16))) float part[LANES][D];
    __shared__ float state[LANES][2];
    Piece pc;
    if (!deal<R, true>(a, d, blockIdx.x, pc)) return;
    if (pc.slot + pc.shares > 2 << d.log_wgs) return;  // (only where lengths change under the launch)
    const int r = blockIdx.y;
    const int rr = pc.tile * R + r;
    if (rr >= pc.count * a.share) return;
    const float* const base = a.ws + (long)pc.slot * R * (D + 2);
    const int c4 = threadIdx.x % C4, part0 = threadIdx.x / C4;
    float m = -INFINITY, sum = 0.f;
    float4_t o = {0.f, 0.f, 0.f, 0.f};
    for (int s = part0; s < pc.shares; s += LANES) {
        const float* const src = base + (long)s * R * (D + 2);
        const float ms = src[R * D + 2 * r], ls = src[R * D + 2 * r + 1];
        const float4_t v = *(const float4_t*)(src + r * D + 4 * c4);
        const float to = fmaxf(m, ms);
        const float f0 = m == to ? 1.f : __builtin_amdgcn_exp2f(m - to), f1 = ms == to ? 1.f : __builtin_amdgcn_exp2f(ms - to);
        sum = sum * f0 + ls * f1;
        o = o * f0 + v * f1;
        m = to;
    }
    *(float4_t*)&part[part0][4 * c4] = o;
    if (c4 == 0) {
        state[part0][0] = m;
        state[part0][1] = sum;
    }
    __syncthreads();
    if (threadIdx.x >= C4) return;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < LANES; w++) mx = fmaxf(mx, state[w][0]);
    sum = 0.f;
    o = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < LANES; w++) {
        const float mw = state[w][0];
        const float f = mw == mx ? 1.f : __builtin_amdgcn_exp2f(mw - mx);
        sum += state[w][1] * f;
        o += *(const float4_t*)&part[w][4 * c4] * f;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    half4_t h;
#pragma unroll
    for (int e = 0; e < 4; e++) h[e] = (half_t)(o[e] * inv);
    *(half4_t*)(a.out + ((long)(pc.first + rr / a.share) * a.c.H * a.share + pc.head * a.share + rr % a.share) * D + 4 * c4) = h;
}

constexpr Deal KA_DEAL = {10, 4};

}  // namespace

// At most 2^(log_wgs + 1) shares of shared tiles: every one but a tile's last holds `least` pages or more, of which
// there are 2^log_wgs times as many as in all, and there are fewer shared tiles than that.
size_t kv4_attention_workspace_bytes(int D) { return (size_t)(2 << KA_DEAL.log_wgs) * KA_ROWS * (D + 2) * sizeof(float); }

hipError_t launch_kv4_attention(const Kv4Cache& c, const void* q, void* out, const int* selected, void* workspace, int D, int g,
                                int share, int count, long q_ts, long q_hs, float sm_scale, hipStream_t st) {
    Kv4AttnArgs a;
    a.c = c;
    a.q = (const half_t*)q;
    a.out = (half_t*)out;
    a.selected = selected;
    a.q_ts = q_ts;
    a.q_hs = q_hs;
    a.share = share;
    a.count = count;
    a.scale = sm_scale * 1.44269504088896340736f;
    const int most = selected && count < c.width ? count : c.width;
    const bool split = workspace != nullptr && most > KA_DEAL.least;
    a.ws = split ? (float*)workspace : nullptr;
    const long tiles = (c.starts ? (long)c.T * share / KA_ROWS + c.B : (long)c.B * (((long)c.each * share + KA_ROWS - 1) / KA_ROWS)) *
                       c.H;
    const long wgs = split ? tiles + (1l << KA_DEAL.log_wgs) : tiles;
    auto go = [&](auto d, auto groups) {
        hipLaunchKernelGGL((kv4_attn_kernel<d.value, groups.value>), dim3((unsigned)wgs), dim3(64 * KA_WAVES), 0, st, a, KA_DEAL);
        if (!split) return;
        const long tokens = c.starts ? KA_ROWS : c.each;
        const unsigned rows = (unsigned)(tokens * share < KA_ROWS ? tokens * share : KA_ROWS);
        const long shared = tiles < (1l << KA_DEAL.log_wgs) ? tiles : (1l << KA_DEAL.log_wgs);
        hipLaunchKernelGGL((kv4_join_kernel<d.value, KA_ROWS>), dim3((unsigned)shared, rows), dim3(256), 0, st, a, KA_DEAL);
    };
    if (D == 128 && g == 128) go(std::integral_constant<int, 128>{}, std::integral_constant<int, 1>{});
    if (D == 128 && g == 64) go(std::integral_constant<int, 128>{}, std::integral_constant<int, 2>{});
    if (D == 128 && g == 32) go(std::integral_constant<int, 128>{}, std::integral_constant<int, 4>{});
    if (D == 64 && g == 64) go(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    if (D == 64 && g == 32) go(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    return hipGetLastError();
}

}  // namespace sq
