// Attention over a 4-bit cache for many rows (prompts, chunks of them; the mathematics: sq_kv4_attn.hip, the layout: sq_kv4.h).
//
// A workgroup of four waves owns 128 rows (token, query head) of a sequence and key/value head, 32 per wave, and goes through
// their pages.  Each page's codes are unpacked once for all of them, into LDS, as the whole numbers they are (exact in fp16),
// in the order of the matrix operands; scales and minima stay apart and meet the fp32 results:
//   S^T = s (K Q^T) + m sum(q)   v_mfma_f32_32x32x16_f16, A = key codes, B = q: a lane has one query and 16 keys of 32
//   O^T = (V - 8)^T P'           A = value codes less 8, B = P' = fp16(P s'): what the lane has, in that order
//   and sum P (m + 8 s) per query and group by vector instructions.  m + 8 s, about the middle of a group, is rounded to fp16,
//   as the values themselves were that the group was made of: up to 2^-11 of the result where values lie far from zero beside
//   their spread (in fp32: 454 instead of 442 us at 2 x 1024 new tokens of 8192 rows, 53 instead of 47 at 8 prompts of 512
//   tokens with heads of 64).
// s' = KA_TOP s over a power of two that follows the scales (of the largest so far), so that P' stays inside fp16's range.
// While a page is worked on, the next one's codes are unpacked into the other half of LDS and the one behind it is on its way to
// registers; one barrier a page, which does not wait for those.
//
// What bounds it: vector instructions, by the counters 533 of them beside 32 matrix instructions per wave and page (16.7 for each
// of a lane's 32 scores), which the two waves of a SIMD hardly overlap (heads of 128 in groups of 64, 1024 tokens of 32 heads over
// 16384 rows: 440 us = 604 TFLOP/s with the join; vector units busy 0.63, matrix units 0.26, LDS 0.34 of 976 thousand cycles, no
// bank conflicts).  Groups of 128 take 0.84 of the time of groups of 64, of 32 1.5 times.
#include "sq_kernels.h"
#include "sq_kv4_attn.h"

namespace sq {

namespace {

constexpr int KC_WAVES = 4;
constexpr int KC_ROWS = 32 * KC_WAVES;

template <int D, int G>
__global__ __launch_bounds__(64 * KC_WAVES, 2) void kv4_chunk_kernel(Kv4AttnArgs a, Deal d) {
    constexpr int g = D / G;
    constexpr int REC = kv4_record_bytes(D, g);
    constexpr int DT = D / 32;  // tiles of 32 columns of the values
    constexpr int ST = D / 16;  // steps of 16 elements of a key
    struct Stage {
        u32x4_t k[D / 8][64];         // [8 elements][key]
        u32x4_t v[8][D];              // [16-key step, half][column]: eight keys
        u32x4_t ksm[G][16], vsm[G][16];  // of four keys: scales, minima; s', m + 8 s
        float sref[G];
    };
    __shared__ __attribute__((aligned(16))) Stage stages[2];

    const Kv4Cache& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Piece pc;
    if (!deal<KC_ROWS, false>(a, d, blockIdx.x, pc)) return;
    if (pc.shares > 1 && pc.slot >= 2 * d.wgs()) return;  // (only where lengths change under the launch)
    const int head = pc.head, len = pc.len;
    const int tile = ceil_div(pc.count * a.share, KC_ROWS) - 1 - pc.tile;  // those that see most come first

    const int n = lane & 31, hl = lane >> 5;
    const int rows = imin(pc.count * a.share - tile * KC_ROWS, KC_ROWS);
    const int row = tile * KC_ROWS + imin(32 * wave + n, rows - 1);
    const int token = row / a.share, qhead = head * a.share + row - token * a.share;
    const int before = pc.end - pc.count;  // rows before the call's
    const int limit = before + token;      // the last row it sees
    const int limit_lo = before + tile * KC_ROWS / a.share;
    const int limit_hi = before + (tile * KC_ROWS + rows - 1) / a.share;
    const int pages = limit_hi < 0 ? 0 : imin(limit_hi / KV4_PAGE + 1, ceil_div(len, KV4_PAGE));
    int p0 = 0, p1 = pages;
    if (pc.shares > 1) {
        const int each = pages / pc.shares, more = pages - each * pc.shares;
        p0 = pc.share * each + imin(pc.share, more);
        p1 = p0 + each + (pc.share < more ? 1 : 0);
    }

    const int* const table = c.table + (long)pc.b * c.table_stride;
    auto page_at = [&](int p) {  // of the pool, -1: none
        const int id = p < p1 ? table[p] : -1;
        return (unsigned)id < (unsigned)c.num_pages ? id : -1;
    };

    // ---- a page on its way: registers, then LDS
    u32x4_t rk, rv[2], rsm;
    const int kkey = lane, kchunk = wave;                                            // keys: 16 (8) bytes of a row
    const int vw = tid % (D / 8), vhf = tid / (D / 8) % 2, vqp = tid / (D / 4);      // values: word, half of it, eight keys
    const bool vtask = vqp < 8;                                                      // (D = 64: half of the threads)
    const int vquad = 4 * (vqp >> 1) + (vqp & 1);
    auto request = [&](int id) __attribute__((always_inline)) {
        const uint8_t* const rec = c.pool + ((long)(id < 0 ? 0 : id) * c.H + head) * REC;
        if constexpr (D == 128)
            rk = *(const u32x4_t*)(rec + kkey * 64 + kchunk * 16);
        else {
            const u32x2_t w = *(const u32x2_t*)(rec + kkey * 32 + kchunk * 8);
            rk[0] = w[0];
            rk[1] = w[1];
        }
        if (vtask) {
            rv[0] = *(const u32x4_t*)(rec + 32 * D + (vquad * (D / 8) + vw) * 16);
            rv[1] = *(const u32x4_t*)(rec + 32 * D + ((vquad + 2) * (D / 8) + vw) * 16);
        }
        if (wave < 2 && lane < 16 * G) rsm = *(const u32x4_t*)(rec + 64 * D + wave * 256 * G + lane * 16);
    };
    float run = 0x1p-24f;  // (second wave, lane i: of group i / 16) the largest scale so far, as a power of two above it
    const NibbleMasks nm = nibble_masks();
    auto unpack = [&](int p, int id, Stage& st) __attribute__((always_inline)) {
        const half2_t k1024 = {(half_t)1024.f, (half_t)1024.f}, k64 = {(half_t)64.f, (half_t)64.f};
#pragma unroll
        for (int q = 0; q < D / 64; q++) {
            const uint32_t w0 = rk[2 * q], w1 = rk[2 * q + 1], h0 = w0 >> 8, h1 = w1 >> 8;
            auto low = [&](uint32_t w) { return bit_cast<uint32_t>(bit_cast<half2_t>((w & nm.lo) | 0x64006400u) - k1024); };
            auto high = [&](uint32_t w) { return bit_cast<uint32_t>(bit_cast<half2_t>((w & nm.hi) | 0x54005400u) - k64); };
            st.k[8 * q + kchunk][kkey] = (u32x4_t){low(w0), low(w1), low(h0), low(h1)};
            st.k[8 * q + 4 + kchunk][kkey] = (u32x4_t){high(w0), high(w1), high(h0), high(h1)};
        }
        if (vtask) {
            const half2_t k1032 = {(half_t)1032.f, (half_t)1032.f}, k72 = {(half_t)72.f, (half_t)72.f};
            const uint32_t sel = vhf ? 0x07060302u : 0x05040100u;
            uint32_t x[4];
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = __builtin_amdgcn_perm(rv[j >> 1][2 * (j & 1) + 1], rv[j >> 1][2 * (j & 1)], sel);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                u32x4_t o;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t w = k >= 2 ? x[j] >> 8 : x[j];
                    o[j] = k & 1 ? bit_cast<uint32_t>(bit_cast<half2_t>((w & nm.hi) | 0x54005400u) - k72)
                                 : bit_cast<uint32_t>(bit_cast<half2_t>((w & nm.lo) | 0x64006400u) - k1032);
                }
                st.v[vqp][(D == 128 ? 16 * (4 * vhf + k) : 16 * k + 8 * vhf) + vw] = o;
            }
        }
        if (wave < 2 && lane < 16 * G) {
            const int key = p * KV4_PAGE + 4 * (lane & 15);
            half8_t sm = bit_cast<half8_t>(rsm);
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (id < 0 || key + r > limit_hi) sm[r] = sm[4 + r] = (half_t)0.f;  // whatever lies where nobody looks
            if (wave == 1) {
                float big = 0.f;
#pragma unroll
                for (int r = 0; r < 4; r++) big = fmaxf(big, (float)sm[r]);
                big = fmaxf(big, row_move<0x121>(big));
                big = fmaxf(big, row_move<0x122>(big));
                big = fmaxf(big, row_move<0x124>(big));
                big = fmaxf(big, row_move<0x128>(big));
                if (big > run) run = bit_cast<float>(bit_cast<uint32_t>(big) & 0x7f800000u) * 2.f;
                const float inv = KA_TOP / run;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float s = (float)sm[r];
                    sm[4 + r] = (half_t)(8.f * s + (float)sm[4 + r]);
                    sm[r] = (half_t)(s * inv);
                }
                st.vsm[lane >> 4][lane & 15] = bit_cast<u32x4_t>(sm);
                if ((lane & 15) == 0) st.sref[lane >> 4] = run;
            } else {
                st.ksm[lane >> 4][lane & 15] = bit_cast<u32x4_t>(sm);
            }
        }
    };
    auto barrier = [&]() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

    int id0 = page_at(p0), id1 = page_at(p0 + 1), id2 = page_at(p0 + 2);
    if (p0 < p1) request(id0);

    half8_t qf[ST];
    float qsum[G];
    {
        const half_t* src = a.q + (long)(pc.first + token) * a.q_ts + (long)qhead * a.q_hs + 8 * hl;
#pragma unroll
        for (int i = 0; i < G; i++) qsum[i] = 0.f;
#pragma unroll
        for (int i = 0; i < ST; i++) {
            const u32x4_t bits = *(const u32x4_t*)(src + 16 * i);
            const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
            qf[i] = bit_cast<half8_t>((u32x4_t){bits[0] ^ flip, bits[1] ^ flip, bits[2] ^ flip, bits[3] ^ flip});
#pragma unroll
            for (int e = 0; e < 8; e += 2)
                qsum[16 * i / g] = __builtin_amdgcn_fdot2((half2_t){qf[i][e], qf[i][e + 1]}, (half2_t){(half_t)1.f, (half_t)1.f},
                                                          qsum[16 * i / g], false);
        }
#pragma unroll
        for (int i = 0; i < G; i++) {
            float x, y;
            pair32(qsum[i], x, y);
            qsum[i] = x + y;
        }
    }

    float16_t acc[DT];
    // Scores stay in units of 1 / scale (its sign went into the queries); 0 is as good as 1e-30.
    const float scale = fmaxf(fabsf(a.scale), 1e-30f), lazy = (float)KA_LAZY / scale;
    float m = -INFINITY, l = 0.f;  // the reference of the softmax, the lane's share of the sum
    float mins[G], sref[G];
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
        for (int v = 0; v < 16; v++) acc[i][v] = 0.f;
#pragma unroll
    for (int i = 0; i < G; i++) mins[i] = 0.f, sref[i] = 0x1p-24f;

    auto dots = [&](const Stage& st, int kb, float16_t (&dot)[G]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < G; i++)
#pragma unroll
            for (int v = 0; v < 16; v++) dot[i][v] = 0.f;
        u32x4_t kf[ST];  // all asked for before the first product
#pragma unroll
        for (int i = 0; i < ST; i++) kf[i] = st.k[2 * i + hl][32 * kb + n];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < ST; i++)
            dot[16 * i / g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bit_cast<half8_t>(kf[i]), qf[i], dot[16 * i / g], 0, 0, 0);
    };
    auto block = [&](auto masked, int pos, const Stage& st, int kb, const float16_t (&dot)[G]) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(masked)::value;
        u32x4_t vf[2][DT];  // and these before the softmax
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int t = 0; t < DT; t++) vf[u][t] = st.v[2 * (2 * kb + u) + hl][32 * t + n];
        __builtin_amdgcn_sched_barrier(0);
        float s[16], top = -INFINITY;
#pragma unroll
        for (int qd = 0; qd < 4; qd++) {
            half8_t sm[G];
#pragma unroll
            for (int i = 0; i < G; i++) sm[i] = bit_cast<half8_t>(st.ksm[i][8 * kb + 2 * qd + hl]);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float x = 0.f;
#pragma unroll
                for (int i = 0; i < G; i++) {
                    x += (float)sm[i][r] * dot[i][4 * qd + r];
                    x += (float)sm[i][4 + r] * qsum[i];
                }
                if (MASKED && pos + 8 * qd + 4 * hl + r > limit) x = -INFINITY;
                s[4 * qd + r] = x;
                top = fmaxf(top, x);
            }
        }
        if (__ballot(top > m + lazy)) {
            float x, y;
            pair32(top, x, y);
            const float to = fmaxf(fmaxf(x, y), m);
            const float f = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - to) * scale);
            m = to;
            l *= f;
#pragma unroll
            for (int i = 0; i < DT; i++) acc[i] *= f;
#pragma unroll
            for (int i = 0; i < G; i++) mins[i] *= f;
        }
        const float ref = m == -INFINITY ? 0.f : -m * scale;
#pragma unroll
        for (int v = 0; v < 16; v++) {
            s[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], scale, ref));
            l += s[v];
        }
        half8_t pf[2][G];
#pragma unroll
        for (int qd = 0; qd < 4; qd++)
#pragma unroll
            for (int i = 0; i < G; i++) {
                const half8_t sm = bit_cast<half8_t>(st.vsm[i][8 * kb + 2 * qd + hl]);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float x = __builtin_fmaf(s[4 * qd + r], (float)sm[r], 0.f);  // (with the rounding below one instruction)
                    float y = s[4 * qd + r] * (float)sm[4 + r];
                    if (MASKED && pos + 8 * qd + 4 * hl + r > limit) x = y = 0.f;  // a row that another query sees
                    pf[qd >> 1][i][4 * (qd & 1) + r] = (half_t)x;
                    mins[i] += y;
                }
            }
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int t = 0; t < DT; t++)
                acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bit_cast<half8_t>(vf[u][t]), pf[u][32 * t / g], acc[t], 0, 0, 0);
    };

    if (p0 < p1) {
        unpack(p0, id0, stages[0]);
        if (p0 + 1 < p1) request(id1);
    }
    barrier();
    // Pages that every query sees whole, then those that end or begin to be hidden in one.
    const int whole = imin(imax((limit_lo + 1) / KV4_PAGE, p0), p1);
    auto step = [&](auto masked, int p) __attribute__((always_inline)) {
        const Stage& st = stages[(p - p0) & 1];
        if (p + 1 < p1) {
            unpack(p + 1, id1, stages[(p - p0 + 1) & 1]);
            if (p + 2 < p1) request(id2);
        }
        const int id = id0;
        id0 = id1, id1 = id2, id2 = page_at(p + 3);
#pragma unroll
        for (int i = 0; i < G; i++) {
            const float to = bit_cast<float>(__builtin_amdgcn_readfirstlane(bit_cast<int>(st.sref[i])));
            if (to != sref[i]) {
                const float f = sref[i] / to;
                sref[i] = to;
#pragma unroll
                for (int t = i * g / 32; t < (i + 1) * g / 32; t++) acc[t] *= f;
            }
        }
        if (id >= 0) {  // a page that does not exist is seen by nobody
            float16_t dot[G];
            dots(st, 0, dot);
            block(masked, p * KV4_PAGE, st, 0, dot);
            dots(st, 1, dot);
            block(masked, p * KV4_PAGE + 32, st, 1, dot);
        }
        barrier();
    };
    int p = p0;
    for (; p < whole; p++) step(std::false_type{}, p);
    for (; p < p1; p++) step(std::true_type{}, p);

    {
        float x, y;
        pair32(l, x, y);
        l = x + y;
#pragma unroll
        for (int i = 0; i < G; i++) {
            pair32(mins[i], x, y);
            mins[i] = x + y;
        }
    }
    if (32 * wave + n >= rows) return;
    if (pc.shares == 1) {
        const float inv = l == 0.f ? 0.f : 1.f / l;  // nothing visible: 0
        half_t* const dst = a.out + ((long)(pc.first + token) * c.H * a.share + qhead) * D + 4 * hl;
#pragma unroll
        for (int t = 0; t < DT; t++) {
            const int gi = 32 * t / g;
            const float f = sref[gi] * (1.f / KA_TOP);
#pragma unroll
            for (int qd = 0; qd < 4; qd++) {
                half4_t h;
#pragma unroll
                for (int r = 0; r < 4; r++) h[r] = (half_t)((acc[t][4 * qd + r] * f + mins[gi]) * inv);
                *(half4_t*)(dst + 32 * t + 8 * qd) = h;
            }
        }
    } else {
        float* const dst = a.ws + (long)pc.slot * KC_ROWS * (D + 2);
        const int r = 32 * wave + n;
#pragma unroll
        for (int t = 0; t < DT; t++) {
            const int gi = 32 * t / g;
            const float f = sref[gi] * (1.f / KA_TOP);
#pragma unroll
            for (int qd = 0; qd < 4; qd++) {
                float4_t o;
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] = acc[t][4 * qd + e] * f + mins[gi];
                *(float4_t*)(dst + r * D + 32 * t + 8 * qd + 4 * hl) = o;
            }
        }
        if (hl == 0) {
            dst[KC_ROWS * D + 2 * r] = m * scale;
            dst[KC_ROWS * D + 2 * r + 1] = l;
        }
    }
}

// Workgroups per CU that the pages are dealt to (1 / 2 / 3 / 4 / 6 / 8: 645 / 449 / 478 / 466 / 473 / 493 us at 1024 tokens
// over 16384 rows: two fit on a CU, and a share's partial state is 66 KB to write and read), and a share's fewest pages.
constexpr Deal KC_DEAL = {2, 8};

}  // namespace

size_t kv4_chunk_workspace_bytes(int D, int pages) {
    return pages > KC_DEAL.least ? (size_t)(2 * KC_DEAL.wgs()) * KC_ROWS * (D + 2) * sizeof(float) : 0;
}

hipError_t launch_kv4_chunk(Kv4AttnArgs a, int D, int g, hipStream_t st) {
    const Kv4Cache& c = a.c;
    const long tiles =
        (c.starts ? (long)c.T * a.share / KC_ROWS + c.B : (long)c.B * (((long)c.each * a.share + KC_ROWS - 1) / KC_ROWS)) * c.H;
    const bool split = a.ws != nullptr && c.width > KC_DEAL.least && tiles < KA_MOST_PAGES / c.width;
    if (!split) a.ws = nullptr;
    const long wgs = split ? tiles + KC_DEAL.wgs() : tiles;
    auto go = [&](auto d, auto groups) {
        hipLaunchKernelGGL((kv4_chunk_kernel<d.value, groups.value>), dim3((unsigned)wgs), dim3(64 * KC_WAVES), 0, st, a, KC_DEAL);
        if (!split) return;
        const long shared = tiles < KC_DEAL.wgs() ? tiles : KC_DEAL.wgs();
        hipLaunchKernelGGL((kv4_join_kernel<d.value, KC_ROWS, 4, true>), dim3((unsigned)shared, KC_ROWS / 4), dim3(256), 0, st, a,
                           KC_DEAL);
    };
    if (D == 128 && g == 128) go(Int<128>{}, Int<1>{});
    if (D == 128 && g == 64) go(Int<128>{}, Int<2>{});
    if (D == 128 && g == 32) go(Int<128>{}, Int<4>{});
    if (D == 64 && g == 64) go(Int<64>{}, Int<1>{});
    if (D == 64 && g == 32) go(Int<64>{}, Int<2>{});
    return hipGetLastError();
}

}  // namespace sq
