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
// shift and four masks, and the powers of two leave with the fp32 result.
//   S   = K Q^T  v_mfma_f32_16x16x32_f16, A = codes (row = key), B = q: a lane has one query and four keys of 16
//   O^T = V^T P' A = codes (row = column of V), B = P': the keys that the lane already has, in that order; the two rows
//                whose codes share a register come together by one byte permutation of two words
// The sum is one of P' (code - 8) and of P (m + 8 s): 8 is taken off the values' codes, which is exact among denormals too.
// The rounding of P' to fp16 then acts on s (code - 8), about the size of v, and not on s code, which is twice that; and the
// fp32 sums stay as small as the result, where those of positive codes, which the matrix instruction rounds towards zero, lose
// the more of it the longer the cache is (131072 rows: error 5.4e-4 of the result; 3.7e-4 with the constant -8 as a product of
// its own after every 32 rows' codes, 2 % faster; 2.9e-4 so, nearly all of it the rounding of P' and of the output).  P' is kept
// inside fp16's range by a power of two per group that follows the scales.
#include "sq_kernels.h"
#include "sq_kv4_attn.h"
#include "sq_kv4_row.h"

namespace sq {

namespace {

// The kernel for few rows.  A workgroup's waves take units of a page (PACK = 1: half of one) in turn, each with a softmax
// of its own, and join them in LDS.
//
// What bounds it: over long caches the stream of records (64 ragged sequences, 221 MB, 49 us = 4.5 TB/s; 131072 rows of one,
// 151 MB, 37.5 us = 4.0 TB/s), with which the work on the codes just keeps up; over short ones latency, one after the other:
// launch, lengths and table, records, join (640 rows of one sequence 8.1 us, of eight 9.9 us = 2.4 TB/s); with 20 queries
// to a key the work per row (5 tokens of 16 sequences 22.5 us).
//
// PACK.  The matrix instruction has 16 columns for the tile's rows; with 4 rows, 12 of them would be empty, and so would
// be three quarters of all that follows per score.  So 4 (2) tiles of 16 cache rows share one result: the tile's queries stand
// in columns 4 j .. 4 j + 3 of the operand that meets the j-th of them and the other columns are 0, so that the four products
// add up to four tiles side by side.  Each column is then a softmax over its own cache rows, and P' meets the values the same
// way round: of its operand, the columns of other tiles are masked off.
template <int D, int G, int PACK>
struct Unit {
    static constexpr int TILES = PACK > 1 ? 4 : 2, SETS = TILES / PACK, ROWS = 16 * TILES;
    uint32_t k[TILES][D / 32];  // [words of the lane's row and chunk]
    u32x4_t v[TILES];
    half8_t ksm[SETS][G], vsm[SETS][G];  // scales and minima of four rows
};

template <int D, int G, int PACK, int RT, int WAVES, bool NEW>
__global__ __launch_bounds__(64 * WAVES) void kv4_attn_kernel(Kv4AttnArgs a, Deal d) {
    constexpr int g = D / G;
    constexpr int REC = kv4_record_bytes(D, g);
    constexpr int NT = D / 16;        // tiles of 16 columns of the values
    constexpr int COLS = 16 / PACK;   // of a tile of cache rows
    constexpr int R = COLS * RT;      // rows of the tile
    constexpr int PITCH = D + 4;      // of a row of partial outputs: the queries of a store fall on different banks
    typedef Unit<D, G, PACK> U;
    static_assert(RT == 1 || PACK == 1);
    // The queries as the products take them, lane by lane, and as many zeros for the columns that a product leaves out: one
    // copy for all waves, read where it is used (kept in registers, 64 of them with PACK = 4, other things would be spilled).
    constexpr int QBYTES = RT * (D / 32) * 1024;
    __shared__ __attribute__((aligned(16))) uint8_t queries[PACK > 1 ? 2 : 1][QBYTES];
    __shared__ __attribute__((aligned(16))) float part[WAVES][R][PITCH];
    __shared__ float state[WAVES][R][2];

    const Kv4Cache& c = a.c;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Piece pc;
    if (!deal<R, false>(a, d, blockIdx.x, pc)) return;
    if (pc.shares > 1 && pc.slot >= 2 * d.wgs()) return;  // (only where lengths change under the launch)
    const int head = pc.head, tile = pc.tile, len = pc.len, before = pc.end - pc.count;  // (rows before the call's)
    const int* const table = c.table + (long)pc.b * c.table_stride;
    const int* const chosen = a.selected ? a.selected + ((long)pc.b * c.H + head) * a.count : nullptr;
    // The first 64 pages, or the places of the selected ones, without waiting for the length.
    int ahead = -1;
    if (lane < (chosen ? a.count : c.width)) ahead = chosen ? chosen[lane] : table[lane];

    const int n = lane & 15, l4 = lane >> 4;
    const int col = n & (COLS - 1), part_of = n / COLS;  // the lane's query, and which of PACK tiles of cache rows
    const int rows = imin(pc.count * a.share - tile * R, R);
    // Queries of this lane: rows col + 16 rt of the tile; the last cache row that each sees.
    int limit[RT], token[RT], qhead[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const int row = tile * R + imin(col + 16 * rt, rows - 1);
        token[rt] = pc.count == 1 ? 0 : row / a.share;
        qhead[rt] = head * a.share + row - token[rt] * a.share;
        limit[rt] = before + token[rt];
    }
    const int limit_hi = before + (pc.count == 1 ? 0 : (tile * R + rows - 1) / a.share);
    const int all_pages = limit_hi < 0 ? 0 : imin(limit_hi / KV4_PAGE + 1, ceil_div(len, KV4_PAGE));
    // (selected pages are for single tokens: limit_hi is the sequence's last row)
    const int pages = a.selected ? imin(all_pages, a.count) : all_pages;
    int p0 = 0, p1 = pages;
    if (pc.shares > 1) {
        const int each = pages / pc.shares, more = pages - each * pc.shares;
        p0 = pc.share * each + imin(pc.share, more);
        p1 = p0 + each + (pc.share < more ? 1 : 0);
    }

    float qsum[RT][G];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const half_t* src = a.q + (long)(pc.first + token[rt]) * a.q_ts + (long)qhead[rt] * a.q_hs + 8 * l4;
#pragma unroll
        for (int i = 0; i < G; i++) qsum[rt][i] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
            const half8_t x = *(const half8_t*)(src + 32 * i);
            if (wave == 0) {
                *(half8_t*)(queries[0] + (rt * (D / 32) + i) * 1024 + lane * 16) = x;
                if (PACK > 1) *(half8_t*)(queries[PACK > 1] + i * 1024 + lane * 16) = (half8_t){};
            }
#pragma unroll
            for (int e = 0; e < 8; e += 2)
                qsum[rt][32 * i / g] = __builtin_amdgcn_fdot2((half2_t){x[e], x[e + 1]}, (half2_t){(half_t)1.f, (half_t)1.f},
                                                              qsum[rt][32 * i / g], false);
        }
#pragma unroll
        for (int i = 0; i < G; i++) qsum[rt][i] = rows_sum(qsum[rt][i]) * a.scale;
    }
    const uint8_t* qat[PACK];  // the lane's place in the queries, or in the zeros for a product that leaves its column out
#pragma unroll
    for (int j = 0; j < PACK; j++) qat[j] = queries[PACK > 1 && part_of != j ? 1 : 0] + lane * 16;
    __syncthreads();

    float4_t acc[RT][NT];
    float m[RT], l[RT];            // the reference of the softmax (of this column), the lane's share of the sum
    float mins[RT][G];             // sum P (m + 8 s) (the lane's share)
    float sref[G], sinv[G];        // power of two in P', and KA_TOP over it
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        m[rt] = -INFINITY, l[rt] = 0.f;
#pragma unroll
        for (int i = 0; i < NT; i++) acc[rt][i] = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < G; i++) mins[rt][i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < G; i++) sref[i] = 0x1p-30f, sinv[i] = KA_TOP * 0x1p30f;
    const half8_t eight[2] = {bit_cast<half8_t>((u32x4_t){0x80088008u, 0x80088008u, 0x80088008u, 0x80088008u}),   // -8 * 2^-24
                              bit_cast<half8_t>((u32x4_t){0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u})};  // -8 * 2^-20
    const float scale24 = a.scale * 0x1p24f;
    const NibbleMasks nm = nibble_masks();
    uint32_t own[PACK];  // all ones where the column is of the j-th tile
#pragma unroll
    for (int j = 0; j < PACK; j++) own[j] = part_of == j ? ~0u : 0u;
    const uint32_t koff = n * (D / 2) + l4 * (D / 8);
    const uint32_t voff = 32 * D + l4 * (2 * D) + (D == 128 ? n : (n & 7)) * 16;
    const uint32_t smoff = 64 * D + (4 * part_of + l4) * 16;
    const uint32_t vsel = D == 64 && n >= 8 ? 0x07060302u : 0x05040100u;
    constexpr int PER = KV4_PAGE / U::ROWS;  // units of a page

    // Pages are looked up 64 at a time: lane i has the i-th one's place in the sequence and in the pool.
    for (int pb = p0; pb < p1; pb += 64) {
        int place = pb + lane, id = -1;
        if (place < p1) {
            if (chosen) place = pb == 0 ? ahead : chosen[place];
            if ((unsigned)place < (unsigned)all_pages) id = pb == 0 && !chosen ? ahead : table[place];
            if ((unsigned)id >= (unsigned)c.num_pages) id = -1;
        }
        if (id < 0) place = 0;  // a page that does not exist: its rows lie behind every query's last
        const int units = PER * imin(64, p1 - pb);
        U x;
        // (uniform base, 32-bit offset of the lane, the rest an immediate)
        auto record = [&](int u) {
            const int pid = __builtin_amdgcn_readlane(id, u / PER);
            return c.pool + ((long)(pid < 0 ? 0 : pid) * c.H + head) * REC;
        };
        auto load_keys = [&](int u) {
            const uint8_t* const rec = record(u);
            const int t0 = PER == 1 ? 0 : u % PER * U::TILES;
            const uint8_t* const ks = rec + t0 * (8 * D);
            const uint8_t* const sm = rec + t0 * 64;
#pragma unroll
            for (int t = 0; t < U::TILES; t++) {
                if constexpr (D == 128) {
                    const u32x4_t w = __builtin_nontemporal_load((const u32x4_t*)(ks + (koff + t * (8 * D))));
#pragma unroll
                    for (int i = 0; i < 4; i++) x.k[t][i] = w[i];
                } else {
                    const u32x2_t w = __builtin_nontemporal_load((const u32x2_t*)(ks + (koff + t * (8 * D))));
                    x.k[t][0] = w[0];
                    x.k[t][1] = w[1];
                }
            }
#pragma unroll
            for (int i = 0; i < U::SETS; i++)
#pragma unroll
                for (int j = 0; j < G; j++) x.ksm[i][j] = *(const half8_t*)(sm + (smoff + PACK * i * 64 + j * 256));
        };
        auto load_values = [&](int u) {
            const uint8_t* const rec = record(u);
            const int t0 = PER == 1 ? 0 : u % PER * U::TILES;
            const uint8_t* const vs = rec + t0 * (8 * D);
            const uint8_t* const sm = rec + t0 * 64;
#pragma unroll
            for (int i = 0; i < U::SETS; i++)
#pragma unroll
                for (int j = 0; j < G; j++) x.vsm[i][j] = *(const half8_t*)(sm + (smoff + 256 * G + PACK * i * 64 + j * 256));
#pragma unroll
            for (int t = 0; t < U::TILES; t++)
                x.v[t] = __builtin_nontemporal_load((const u32x4_t*)(vs + (voff + t * (8 * D))));
        };
        // One unit.  The next one's keys are asked for where this one's have met the queries, its values where these have met P.
        auto consume = [&](int u) {
            constexpr int NS = 4 * U::SETS;  // scores of a lane and query
            float s[RT][NS];
            float4_t even[U::SETS][RT][G], odd[U::SETS][RT][G];
#pragma unroll
            for (int i = 0; i < U::SETS; i++)
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
#pragma unroll
                    for (int j = 0; j < G; j++) even[i][rt][j] = odd[i][rt][j] = (float4_t){0.f, 0.f, 0.f, 0.f};
            asm volatile("" ::: "memory");  // the queries are read anew
#pragma unroll
            for (int t = 0; t < U::TILES; t++) {
                const int set = t / PACK, j = t % PACK;
#pragma unroll
                for (int p = 0; p < D / 64; p++) {
                    const uint32_t w0 = x.k[t][2 * p], w1 = x.k[t][2 * p + 1], h0 = w0 >> 8, h1 = w1 >> 8;
                    const half8_t lo = bit_cast<half8_t>((u32x4_t){w0 & nm.lo, w1 & nm.lo, h0 & nm.lo, h1 & nm.lo});
                    const half8_t hi = bit_cast<half8_t>((u32x4_t){w0 & nm.hi, w1 & nm.hi, h0 & nm.hi, h1 & nm.hi});
                    const int ie = 64 * p / g, io = (64 * p + 32) / g;
#pragma unroll
                    for (int rt = 0; rt < RT; rt++) {
                        const half8_t* const q = (const half8_t*)(qat[j] + (rt * (D / 32) + 2 * p) * 1024);
                        even[set][rt][ie] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, q[0], even[set][rt][ie], 0, 0, 0);
                        odd[set][rt][io] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, q[64], odd[set][rt][io], 0, 0, 0);
                    }
                }
            }
            // Where the lane's scores stand: rows pos + 16 PACK set + r.
            const int pid = __builtin_amdgcn_readlane(id, u / PER);
            const int pos = __builtin_amdgcn_readlane(place, u / PER) * KV4_PAGE + u % PER * U::ROWS + 16 * part_of + 4 * l4;
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                const int last = pid < 0 ? -1 : limit[rt];
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < NS; i++) {
                    const int set = i / 4, r = i % 4;
                    float codes = 0.f, shift = 0.f;
#pragma unroll
                    for (int j = 0; j < G; j++) {
                        const float sum = odd[set][rt][j][r] * 0.0625f + even[set][rt][j][r];
                        codes += (float)x.ksm[set][j][r] * sum;
                        shift += (float)x.ksm[set][j][4 + r] * qsum[rt][j];
                    }
                    s[rt][i] = codes * scale24 + shift;
                    if (pos + 16 * PACK * set + r > last) s[rt][i] = -INFINITY;
                    top = fmaxf(top, s[rt][i]);
                }
                if (rt == RT - 1) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (u + WAVES < units) load_keys(u + WAVES);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (__ballot(top > m[rt] + (float)KA_LAZY)) {
                    const float to = fmaxf(rows_max(top), m[rt]);
                    const float f = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[rt] - to);
                    m[rt] = to;
                    l[rt] *= f;
#pragma unroll
                    for (int i = 0; i < NT; i++) acc[rt][i] *= f;
#pragma unroll
                    for (int i = 0; i < G; i++) mins[rt][i] *= f;
                }
                const float ref = m[rt] == -INFINITY ? 0.f : m[rt];
#pragma unroll
                for (int i = 0; i < NS; i++) {
                    s[rt][i] = __builtin_amdgcn_exp2f(s[rt][i] - ref);
                    l[rt] += s[rt][i];
                }
            }
            // P' of every group, as the operand's halves.
            const int seen_to = RT == 1 ? limit[0] : limit_hi;
            uint32_t pf[RT][U::SETS][G][2];
#pragma unroll
            for (int j = 0; j < G; j++) {
                float sv[NS], mid[NS], big = 0.f;
#pragma unroll
                for (int i = 0; i < NS; i++) {
                    const int set = i / 4, r = i % 4;
                    sv[i] = (float)x.vsm[set][j][r];
                    mid[i] = 8.f * sv[i] + (float)x.vsm[set][j][4 + r];
                    if (pid < 0 || pos + 16 * PACK * set + r > seen_to) sv[i] = mid[i] = 0.f;  // whatever lies where nobody looks
                    big = fmaxf(big, sv[i]);
                }
                if (__ballot(big >= sref[j])) {
                    const float to = bit_cast<float>(bit_cast<uint32_t>(wave_max(big)) & 0x7f800000u) * 2.f;
                    const float f = sref[j] / to;
                    sref[j] = to;
                    sinv[j] = KA_TOP / to;
#pragma unroll
                    for (int rt = 0; rt < RT; rt++)
#pragma unroll
                        for (int k = j * g / 16; k < (j + 1) * g / 16; k++) acc[rt][k] *= f;
                }
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
#pragma unroll
                    for (int i = 0; i < NS; i += 2) {
                        float x0 = s[rt][i] * (sv[i] * sinv[j]), x1 = s[rt][i + 1] * (sv[i + 1] * sinv[j]);
                        float y0 = s[rt][i] * mid[i], y1 = s[rt][i + 1] * mid[i + 1];
                        if (RT > 1) {  // a row that another query sees
                            const int set = i / 4, r = i % 4;
                            if (pos + 16 * PACK * set + r > limit[rt]) x0 = y0 = 0.f;
                            if (pos + 16 * PACK * set + r + 1 > limit[rt]) x1 = y1 = 0.f;
                        }
                        mins[rt][j] += y0;
                        mins[rt][j] += y1;
                        pf[rt][i / 4][j][i % 4 / 2] = bit_cast<uint32_t>((half2_t){(half_t)x0, (half_t)x1});
                    }
            }
#pragma unroll
            for (int t = 0; t < U::TILES; t += 2) {
                const int s0 = t / PACK, s1 = (t + 1) / PACK, j0 = t % PACK, j1 = (t + 1) % PACK;
                half8_t b[RT][G];
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
#pragma unroll
                    for (int j = 0; j < G; j++) {
                        u32x4_t w = {pf[rt][s0][j][0], pf[rt][s0][j][1], pf[rt][s1][j][0], pf[rt][s1][j][1]};
                        if (PACK > 1) w = (u32x4_t){w[0] & own[j0], w[1] & own[j0], w[2] & own[j1], w[3] & own[j1]};
                        b[rt][j] = bit_cast<half8_t>(w);
                    }
#pragma unroll
                for (int hf = 0; hf < D / 64; hf++) {  // low halves of the words (D = 64: the lane's half), high halves
                    const uint32_t sel = hf ? 0x07060302u : vsel;
                    uint32_t lo[4], up[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        lo[j] = __builtin_amdgcn_perm(x.v[t + (j >> 1)][2 * (j & 1) + 1], x.v[t + (j >> 1)][2 * (j & 1)], sel);
                        up[j] = lo[j] >> 8;
                    }
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t mask = k & 1 ? nm.hi : nm.lo;
                        const half8_t op = (k < 2 ? bit_cast<half8_t>((u32x4_t){lo[0] & mask, lo[1] & mask, lo[2] & mask, lo[3] & mask})
                                                  : bit_cast<half8_t>((u32x4_t){up[0] & mask, up[1] & mask, up[2] & mask, up[3] & mask})) +
                                           eight[k & 1];
                        const int i = 4 * hf + k;
#pragma unroll
                        for (int rt = 0; rt < RT; rt++)
                            acc[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(op, b[rt][16 * i / g], acc[rt][i], 0, 0, 0);
                    }
                }
            }
        };
        // The new row, if this is the share that sees it: stored by the wave whose unit it is in, before it asks for that
        // unit; the others do not wait.  (All queries of a head stand in one tile here.)
        const int fresh = NEW && pb + 64 >= p1 && p1 == all_pages && len > 0 && pc.end == len  // (inside the table)
                              ? PER * (p1 - pb - 1) + (len - 1) % KV4_PAGE / U::ROWS : -1;
        const bool mine = fresh >= 0 && fresh % WAVES == wave;
        if (wave < units && !(mine && fresh == wave)) {
            load_keys(wave);
            load_values(wave);
        }
        if (NEW && mine) {
            const int pid = __builtin_amdgcn_readlane(id, fresh / PER);
            if (pid >= 0) {
                uint8_t* const rec = c.pool + ((long)pid * c.H + head) * REC;
                const int row = (len - 1) % KV4_PAGE, sub = lane % (D / 8);
                const half8_t k8 = *(const half8_t*)(a.k_new + (long)pc.first * a.k_ts + (long)head * a.k_hs + 8 * sub);
                const half8_t v8 = *(const half8_t*)(a.v_new + (long)pc.first * a.v_ts + (long)head * a.v_hs + 8 * sub);
                half8_t* const bounds = (half8_t*)(rec + 64 * D + 512 * G) + sub;
                half8_t hi, lo;
#pragma unroll
                for (int e = 0; e < 8; e++) hi[e] = (half_t)-INFINITY, lo[e] = (half_t)INFINITY;
                if (row > 0) hi = bounds[0], lo = bounds[D / 8];
                hi = __builtin_elementwise_max(hi, k8);
                lo = __builtin_elementwise_min(lo, k8);
                kv4_store_row<D, G>(rec, row, k8, v8, lane < D / 8, RowOut{nullptr, nullptr});
                if (lane < D / 8) {
                    bounds[0] = hi;
                    bounds[D / 8] = lo;
                }
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            if (fresh == wave) {
                load_keys(wave);
                load_values(wave);
            }
        }
        for (int u = wave; u < units; u += WAVES) {
            consume(u);
            __builtin_amdgcn_sched_barrier(0);
            if (u + WAVES < units) load_values(u + WAVES);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // Of the wave: sums over the lanes of a column, then the columns of one query, which have seen different rows.
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        l[rt] = rows_sum(l[rt]);
#pragma unroll
        for (int i = 0; i < G; i++) mins[rt][i] = rows_sum(mins[rt][i]);
#pragma unroll
        for (int i = 0; i < NT; i++) {
            const int gi = 16 * i / g;
            const float f = sref[gi] * ((i & 1 ? 0x1p20f : 0x1p24f) / KA_TOP);
#pragma unroll
            for (int e = 0; e < 4; e++) acc[rt][i][e] = acc[rt][i][e] * f + mins[rt][gi];
        }
        if constexpr (PACK > 1) {
            float to = fmaxf(m[rt], row_move<0x128>(m[rt]));          // row_ror:8
            if (PACK == 4) to = fmaxf(to, row_move<0x124>(to));        // row_ror:4
            const float f = m[rt] == to ? 1.f : __builtin_amdgcn_exp2f(m[rt] - to);
            m[rt] = to;
            l[rt] *= f;
            l[rt] += row_move<0x128>(l[rt]);
            if (PACK == 4) l[rt] += row_move<0x124>(l[rt]);
#pragma unroll
            for (int i = 0; i < NT; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float v = acc[rt][i][e] * f;
                    v += row_move<0x128>(v);
                    if (PACK == 4) v += row_move<0x124>(v);
                    acc[rt][i][e] = v;
                }
        }
        const int row = n + 16 * rt;
        if (n < COLS && row < rows) {
#pragma unroll
            for (int i = 0; i < NT; i++) *(float4_t*)&part[wave][row][16 * i + 4 * l4] = acc[rt][i];
            if (l4 == 0) {
                state[wave][row][0] = m[rt];
                state[wave][row][1] = l[rt];
            }
        }
    }
    __syncthreads();
    constexpr int C4 = D / 4;
    for (int i = threadIdx.x; i < rows * C4; i += 64 * WAVES) {
        const int r = i / C4, c4 = i % C4;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < WAVES; w++) mx = fmaxf(mx, state[w][r][0]);
        float sum = 0.f;
        float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const float mw = state[w][r][0];
            const float f = mw == mx ? 1.f : __builtin_amdgcn_exp2f(mw - mx);
            sum += state[w][r][1] * f;
            o += *(const float4_t*)&part[w][r][4 * c4] * f;
        }
        if (pc.shares == 1) {
            const int rr = tile * R + r, t = pc.count == 1 ? 0 : rr / a.share;
            const float inv = sum == 0.f ? 0.f : 1.f / sum;  // nothing visible: 0
            half4_t h;
#pragma unroll
            for (int e = 0; e < 4; e++) h[e] = (half_t)(o[e] * inv);
            *(half4_t*)(a.out + ((long)(pc.first + t) * c.H * a.share + head * a.share + rr - t * a.share) * D + 4 * c4) = h;
        } else {
            float* const dst = a.ws + (long)pc.slot * R * (D + 2);
            *(float4_t*)(dst + r * D + 4 * c4) = o;
            if (c4 == 0) {
                dst[R * D + 2 * r] = mx;
                dst[R * D + 2 * r + 1] = sum;
            }
        }
    }
}

// Workgroups per CU that a launch's pages are dealt to, and a share's fewest pages.  Two (64 ragged sequences / one of
// 131072 rows: 48.9 / 38.0 us; 59 / 45 with three, 54 / 46 with four: more partial states and no more loads under way than
// the registers allow).  Sixteen pages, so that up to 1024 rows nothing is shared: with eight, 640 rows of one sequence
// take 10.5 instead of 8.1 us, of eight 14 instead of 9.9 (the second launch is dearer than what it saves), 5 tokens of
// 16 sequences 28.7 instead of 22.5.
// Two things hang on these sixteen pages, and neither fits every call.  Whether a launch shares at all goes by the table's width,
// which is what the host knows: through a table of more than 16 pages 640 rows of one sequence take 11.0 instead of 8.6 us, of
// eight 13.3 instead of 10.6 (four waves, a look at all lengths, a second launch that finds nothing).  And once it does, a share
// has sixteen pages at the fewest: one sequence of 8 heads goes to 8 workgroups at 1024 rows (10.6 us), to 64 at 8000 (16.3).
constexpr Deal KA_DEAL = {2, 16};
constexpr int KA_ROWS = 32;  // of a tile at the most

}  // namespace

// At most 2 wgs() shares of shared tiles: a tile of p pages has fewer than p / least + 1, there are at most wgs() * least
// pages in all, and every shared tile has more than `least` of them.
size_t kv4_attention_workspace_bytes(int T, int B, int share, int D, int pages) {
    const long mean = ((long)T * share + B - 1) / B;
    if (mean > KA_ROWS) return kv4_chunk_workspace_bytes(D, pages);
    if (pages <= KA_DEAL.least) return 0;
    const int rows = mean <= 4 ? 4 : mean <= 8 ? 8 : mean <= 16 ? 16 : KA_ROWS;
    return (size_t)(2 * KA_DEAL.wgs()) * rows * (D + 2) * sizeof(float);
}

hipError_t launch_kv4_attention(const Kv4Cache& c, const void* q, void* out, const int* selected, void* workspace, int D, int g,
                                int share, int count, long q_ts, long q_hs, float sm_scale, const void* k_new, const void* v_new,
                                const long* new_strides, hipStream_t st) {
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
    a.k_new = a.v_new = nullptr;
    a.k_ts = a.k_hs = a.v_ts = a.v_hs = 0;
    // Rows of a sequence and key/value head (of the average one where they differ).
    long mean = ((long)c.T * share + c.B - 1) / c.B;
    a.rows_min = 0, a.rows_max = 1 << 30;
    if (k_new && !c.starts && c.each == 1 && mean <= KA_ROWS) {
        a.k_new = (const half_t*)k_new;
        a.v_new = (const half_t*)v_new;
        a.k_ts = new_strides[0];
        a.k_hs = new_strides[1];
        a.v_ts = new_strides[2];
        a.v_hs = new_strides[3];
    } else if (k_new) {
        const hipError_t e = launch_kv4_append(c, k_new, v_new, nullptr, nullptr, D, g, new_strides, st);
        if (e != hipSuccess) return e;
    }
    // Prompts beside single tokens: where sequences differ and the average is above KA_ROWS and up to 1024 rows, the kernel for many
    // rows takes those with more than KA_ROWS and this one the others, which there would fill a thirtieth of a tile (4 query
    // heads; 1024 tokens over 4096 rows beside 63 sequences of one token: 589 us without, 213 so).  Where nothing is left for
    // this kernel its launches are lost: 8 prompts of 30 to 58 tokens 9.4 and 11.2, of 100 to 300 18.9 and 20.8.
    // Neither bound tells all calls apart, for the host knows the average alone.  Up to KA_ROWS this kernel takes all: by both, 64
    // sequences of 1 to 5 tokens over 2000 rows would take 82 us instead of 69, but 256 tokens over 4096 rows beside 63 single
    // ones 123 instead of 268.  Above 1024 the other takes all: by both, 1024 tokens over 16384 rows beside 5 over 1300 would take
    // 471 instead of 454 and 8 prompts of 512 66 instead of 64, but 4096 beside 7 single ones 278 instead of 425.
    const bool both = c.starts && !selected && mean > KA_ROWS && mean <= 1024 && share <= KA_ROWS && c.B > 1;
    if (mean > KA_ROWS && !selected) {
        a.ws = (float*)workspace;
        if (both) a.rows_min = KA_ROWS + 1;
        const hipError_t e = launch_kv4_chunk(a, D, g, st);
        if (e != hipSuccess || !both) return e;
        a.rows_min = 0, a.rows_max = KA_ROWS;
        mean = share;  // (those with few rows mostly have one token)
    }
    const int most = selected && count < c.width ? count : c.width;
    auto tiles_of = [&](int R) {
        if (both && (long)c.T * share > (long)c.B * KA_ROWS) return (long)c.B * (KA_ROWS / R) * c.H;
        return (c.starts ? (long)c.T * share / R + c.B : (long)c.B * (((long)c.each * share + R - 1) / R)) * c.H;
    };
    const bool split = workspace != nullptr && most > KA_DEAL.least && tiles_of(4) < KA_MOST_PAGES / most;
    a.ws = split ? (float*)workspace : nullptr;
    auto go = [&](auto d, auto groups, auto pack, auto rt, auto waves) {
        constexpr int R = 16 / pack.value * rt.value;
        const long tiles = tiles_of(R);
        const long wgs = split ? tiles + KA_DEAL.wgs() : tiles;
        if (a.k_new)
            hipLaunchKernelGGL((kv4_attn_kernel<d.value, groups.value, pack.value, rt.value, waves.value, true>),
                               dim3((unsigned)wgs), dim3(64 * waves.value), 0, st, a, KA_DEAL);
        else
            hipLaunchKernelGGL((kv4_attn_kernel<d.value, groups.value, pack.value, rt.value, waves.value, false>),
                               dim3((unsigned)wgs), dim3(64 * waves.value), 0, st, a, KA_DEAL);
        if (!split) return;
        const long tokens = c.starts ? R : c.each;
        const unsigned rows = (unsigned)(tokens * share < R ? tokens * share : R);
        const long shared = tiles < KA_DEAL.wgs() ? tiles : KA_DEAL.wgs();
        hipLaunchKernelGGL((kv4_join_kernel<d.value, R, 1, false>), dim3((unsigned)shared, rows), dim3(256), 0, st, a, KA_DEAL);
    };
    // Where nothing is shared and there are no more workgroups than CUs, eight waves take the pages of one (8 x 640 rows of 32
    // heads 11.2 -> 10.1 us); otherwise four, of which two or three workgroups fit on a CU (64 ragged sequences 65 -> 49).
    auto waves_for = [&](auto d, auto groups, auto pack, auto rt) {
        if (!split && tiles_of(16 / pack.value * rt.value) <= 256)
            go(d, groups, pack, rt, Int<8>{});
        else
            go(d, groups, pack, rt, Int<4>{});
    };
    // Rows of a tile: the fewest that hold the average sequence's, so that few columns of the products are empty.  17 to 32
    // rows: two operands of queries per unpacked code by 8 waves (5 tokens of 4 query heads 22.5 us, by 4 waves 25.9; two
    // tiles of 16 rows instead 26.9 and, by 4 waves, 24.3).
    auto by_rows = [&](auto d, auto groups) {
        if (mean <= 4)
            waves_for(d, groups, Int<4>{}, Int<1>{});
        else if (mean <= 8)
            waves_for(d, groups, Int<2>{}, Int<1>{});
        else if (mean <= 16)
            waves_for(d, groups, Int<1>{}, Int<1>{});
        else
            go(d, groups, Int<1>{}, Int<2>{}, Int<8>{});
    };
    if (D == 128 && g == 128) by_rows(Int<128>{}, Int<1>{});
    if (D == 128 && g == 64) by_rows(Int<128>{}, Int<2>{});
    if (D == 128 && g == 32) by_rows(Int<128>{}, Int<4>{});
    if (D == 64 && g == 64) by_rows(Int<64>{}, Int<1>{});
    if (D == 64 && g == 32) by_rows(Int<64>{}, Int<2>{});
    return hipGetLastError();
}

}  // namespace sq
