// The attention weight that a prompt's queries give to each of its keys, summed over the queries (all, or the last so many)
// and over the query heads of a key/value head:
//   w[j] = sum_{g, i >= j} exp(scale q_{g,i} . k_j - lse_{g,i}),  lse_{g,i} = log sum_{j <= i} exp(scale q_{g,i} . k_j)
// Two passes over the same products: the sums of the rows first, then the sums of the columns.  The rows (query, head) of a
// key/value head are packed, so that its keys are read once for all of its heads.
//
// What bounds it: vector instructions beside the products; an exponential of 8 cycles and two to three others of 4 per score and pass,
// and a score's share of the products is 4 (D = 128).  8 prompts of 2048, 32 heads: 275 GFLOP in both passes, 350 us, 0.78 PFLOP/s
// (vector issue 0.81 of the time in both, matrix pipes 0.56 and 0.44); the two products alone would take 236 at a large product's
// rate.  Where queries and keys are all that is given the second product cannot be avoided: the sums are known only behind a
// row's last key, and the scores in memory would be 1 GB.  (A prompt's attention forms the same sums; it does not hand them on, so
// that a cache that evicts pays for the first pass again.)  A window of 64 queries over 4 x 8191 rows takes 43 us for 26 MB:
// two launches, of which the first goes through all keys with one tile of queries a workgroup.
#include "sq_attn_rows.h"
#include "sq_kernels.h"

#include <algorithm>
#include <type_traits>

namespace sq {

namespace {

constexpr int WG_STEP = 64;   // keys of a step of the first pass
constexpr int WG_ROWS = 128;  // rows of its workgroups

struct WeighPlan {
    WeighArgs t;
    float2* ml;  // [B][H][parts][pitch]: reference (in units of log2) and sum of a row over a part of the keys
    long pitch;
    int tiles, parts, steps, queries;
    int even;  // a step of the second pass holds whole queries, within 32 bits of bytes
    float qk_scale;
    // by_pairs: (sequence, head) pairs that are worked on at a time, a multiple of 8 where there are more: workgroups go round
    // the eight XCDs, so that all tiles of a pair, which read the same rows, share an L2, and 8 pairs' keys fit one.
    Divisor by_share, by_heads, by_parts, by_steps, by_pairs, by_tiles, by_key_tiles;
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Rows of sequence b, and how many of them are its queries.
__device__ __forceinline__ void sizes_of(const WeighPlan& a, int b, int& n, int& queries) {
    n = a.t.lengths ? a.t.lengths[b] : a.t.S;
    n = n < 0 ? 0 : imin(n, a.t.S);
    queries = imin(n, a.queries);
}

template <int D>
__global__ __launch_bounds__(256, 4) void weigh_rows_kernel(WeighPlan a) {
    constexpr int ROW = D * 2;
    constexpr int TILE = WG_STEP * ROW;
    constexpr int NK = D / 16;
    constexpr int NL = TILE / 1024 / 4;
    constexpr int RPL = 1024 / ROW;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * TILE];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    const WeighArgs& t = a.t;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ln = lane & 31, lc = lane >> 5;
    const int rest = a.by_pairs(blockIdx.x), per = a.by_tiles(rest), in = rest - per * (int)a.by_tiles.value;
    const int bh = per * (int)a.by_pairs.value + blockIdx.x - rest * (int)a.by_pairs.value;
    const int back = a.by_parts(in), part = in - back * a.parts;
    const int tile = a.tiles - 1 - back;  // those that see most come first
    if (bh >= t.B * t.H) return;
    const int b = a.by_heads(bh), h = bh - b * t.H;
    int n, queries;
    sizes_of(a, b, n, queries);
    const int rows = queries * t.share;
    const int row0 = tile * WG_ROWS;
    if (row0 >= rows) return;
    const int first = n - queries;  // the first of its queries
    const int row = imin(row0 + 32 * wave + ln, rows - 1);
    const int place = a.by_share(row);
    const int query = first + place;
    const int seen_lo = first + a.by_share(row0) + 1;                              // keys of the tile's first row
    const int seen = first + a.by_share(imin(row0 + WG_ROWS, rows) - 1) + 1;       // ... and of its last
    const int s0 = part * a.steps;
    const int s1 = imin(s0 + a.steps, ceil_div(seen, WG_STEP));

    half8_t qf[NK];
    {
        const half_t* qp = t.q + (long)b * t.q_bs + (long)(h * t.share + row - place * t.share) * t.q_hs + (long)query * t.q_rs + 8 * lc;
#pragma unroll
        for (int s = 0; s < NK; s++) qf[s] = *(const half8_t*)(qp + 16 * s);
    }
    const half_t* const kb = t.k + (long)b * t.k_bs + (long)h * t.k_hs;
    const int rs = (int)t.k_rs * 2;
    const int lrow = lane / (D / 8), lchunk = lane % (D / 8);
    const int row_w = RPL * NL * wave + lrow;
    uint32_t off[NL];
#pragma unroll
    for (int j = 0; j < NL; j++) off[j] = (row_w + RPL * j) * rs + ((lchunk ^ k_swz<D>(row_w + RPL * j)) * 16);
    auto issue = [&](int s, uint32_t stage) {
        const int at = s * WG_STEP;
        const uint8_t* const base = uniform((const uint8_t*)kb + (long)at * rs);
        const uint32_t l0 = lds0 + stage + wave * (NL * 1024);
        if (at + WG_STEP <= seen) {
#pragma unroll
            for (int j = 0; j < NL; j++) load_to_lds_x4(base, off[j], l0 + j * 1024);
        } else {  // rows past the end re-read the last one
#pragma unroll 1
            for (int j = 0; j < NL; j++) {
                const int r = row_w + RPL * j;
                load_to_lds_x4(base, (uint32_t)(imin(r, seen - 1 - at) * rs + ((lchunk ^ k_swz<D>(r)) * 16)), l0 + j * 1024);
            }
        }
    };
    if (s0 < s1) issue(s0, 0);
    int kread[NK];
#pragma unroll
    for (int s = 0; s < NK; s++) kread[s] = ln * ROW + (((2 * s + lc) ^ k_swz<D>(ln)) * 16);
    // A lane's reference: the largest of the first scores that it sees.  The sums are fp32 and unrounded, so that later scores may
    // exceed it by 2^100 before it has to move: no maximum is formed in the loop.
    constexpr float MOST = 0x1p100f;
    float ref = 0.f, sum = 0.f;
    bool unset = true;
#pragma unroll
    for (int s = 0; s < NK; s++) {
        u32x4_t x = bit_cast<u32x4_t>(qf[s]);
        asm volatile("" : "+v"(x));
        qf[s] = bit_cast<half8_t>(x);
    }
    uint32_t stage = 0;
    const int plain = imin(s1, seen_lo / WG_STEP);  // steps in which every row sees every key
    for (int s = s0; s < s1; s++, stage ^= TILE) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (s + 1 < s1) issue(s + 1, stage ^ TILE);
        const uint8_t* const l = lds + stage;
        float16_t st[2];
#pragma unroll
        for (int v = 0; v < 16; v++) st[0][v] = st[1][v] = 0.f;
#pragma unroll
        for (int k = 0; k < NK; k++)
#pragma unroll
            for (int i = 0; i < 2; i++)
                st[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const half8_t*)(l + kread[k] + i * (32 * ROW)), qf[k], st[i], 0, 0, 0);
        // Score e is at place_of(e) + 4 lc of the step's keys, of which places up to `visible` are seen.
        auto place_of = [](int e) { return 32 * (e >> 4) + 8 * ((e & 15) >> 2) + (e & 3); };
        int visible = query - s * WG_STEP - 4 * lc;
        asm volatile("" : "+v"(visible));  // (or 32 differences to it would be kept over the loop)
        float four[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 32; e++) st[e >> 4][e & 15] = __builtin_fmaf(st[e >> 4][e & 15], a.qk_scale, -ref);
        if (s >= plain) {
#pragma unroll
            for (int e = 0; e < 32; e++) st[e >> 4][e & 15] = place_of(e) <= visible ? st[e >> 4][e & 15] : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 32; e++) four[e & 3] += __builtin_amdgcn_exp2f(st[e >> 4][e & 15]);
        float more = (four[0] + four[1]) + (four[2] + four[3]);
        if (__builtin_amdgcn_ballot_w64(unset || !(more < MOST)) != 0) {
            float mx = -INFINITY;
#pragma unroll
            for (int e = 0; e < 32; e++) mx = fmaxf(mx, st[e >> 4][e & 15]);
            const float delta = mx == -INFINITY ? 0.f : unset ? mx : fmaxf(mx, 0.f);
            // (while it is unset the sum is 0, or NaN where a score was, and 2^-delta of a first score below -128 is infinite)
            sum = unset ? sum : sum * __builtin_amdgcn_exp2f(-delta);
            unset = unset && mx == -INFINITY;
            ref += delta;
            more = 0.f;
#pragma unroll
            for (int e = 0; e < 32; e++) more += __builtin_amdgcn_exp2f(st[e >> 4][e & 15] - delta);
        }
        sum += more;
    }
    const float m = unset ? -INFINITY : ref;
    const float2 mine = make_float2(m, sum), other = make_float2(__shfl_xor(m, 32), __shfl_xor(sum, 32));
    const float top = fmaxf(mine.x, other.x);
    const float l = mine.y * share_of(mine, top) + other.y * share_of(other, top);
    if (lc == 0 && row0 + 32 * wave + ln < rows) a.ml[((long)bh * a.parts + part) * a.pitch + row] = make_float2(top, l);
}

// KG groups of 32 keys, RG groups of rows: wave (kg, rg) sums the weights of 32 keys over an RG-th of the rows of a step.
template <int D, int KG, int RG>
__global__ __launch_bounds__(256, RG == 1 ? 4 : 2) void weigh_keys_kernel(WeighPlan a) {
    constexpr int BLK = RG == 1 ? 2 : 1;    // 32-row blocks of a wave and step
    constexpr int STEP = 32 * BLK * RG;     // rows of a step
    constexpr int CHUNK = 512;              // rows whose sums are fetched at once
    constexpr int ROW = D * 2;
    constexpr int TILE = STEP * ROW;
    constexpr int NK = D / 16;
    constexpr int NL = TILE / 1024 / 4;
    constexpr int RPL = 1024 / ROW;
    static_assert(KG * RG == 4);
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * TILE];
    __shared__ __attribute__((aligned(16))) float lse[2][CHUNK];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    const WeighArgs& t = a.t;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ln = lane & 31, lc = lane >> 5;
    const int kg = wave % KG, rg = wave / KG;
    const int rest = a.by_pairs(blockIdx.x), per = a.by_key_tiles(rest);
    const int bh = per * (int)a.by_pairs.value + blockIdx.x - rest * (int)a.by_pairs.value;
    const int tile = rest - per * (int)a.by_key_tiles.value;  // those that are seen most come first
    if (bh >= t.B * t.H) return;
    const int b = a.by_heads(bh), h = bh - b * t.H;
    int n, queries;
    sizes_of(a, b, n, queries);
    const int key0 = tile * 32 * KG;
    const int key = key0 + 32 * kg + ln;
    float* const out = t.w + (long)bh * t.S;
    if (key0 >= n) {
        if (rg == 0 && lc == 0 && key < t.S) out[key] = 0.f;
        return;
    }
    const int first = n - queries;
    const int rows = queries * t.share;
    const int end = ceil_div(rows, STEP);
    const int begin = imin((key0 > first ? key0 - first : 0) * t.share / STEP, end);

    half8_t kf[NK];
    {
        const half_t* p = t.k + (long)b * t.k_bs + (long)h * t.k_hs + (long)imin(key, n - 1) * t.k_rs + 8 * lc;
#pragma unroll
        for (int s = 0; s < NK; s++) kf[s] = *(const half8_t*)(p + 16 * s);
    }
    const half_t* const qb = t.q + (long)b * t.q_bs + (long)h * t.share * t.q_hs;
    const int lrow = lane / (D / 8), lchunk = lane % (D / 8);
    const int row_w = RPL * NL * wave + lrow;
    // Where a step holds whole queries a lane's places in it are the same in every step.
    uint32_t off[NL];
#pragma unroll
    for (int j = 0; j < NL; j++) {
        const int i = row_w + RPL * j, q = a.by_share(i);
        off[j] = (uint32_t)((i - q * t.share) * t.q_hs + q * t.q_rs + 8 * (lchunk ^ k_swz<D>(i))) * 2;
    }
    auto issue = [&](int s, int slot) {
        if (a.even && (s + 1) * STEP <= rows) {
            const uint8_t* const base = uniform((const uint8_t*)(qb + (long)(first + a.by_share(s * STEP)) * t.q_rs));
#pragma unroll
            for (int j = 0; j < NL; j++) load_to_lds_x4(base, off[j], lds0 + slot * TILE + wave * (NL * 1024) + j * 1024);
            return;
        }
#pragma unroll 1
        for (int j = 0; j < NL; j++) {
            const int i = row_w + RPL * j;
            const int r = imin(s * STEP + i, rows - 1);
            const int q = a.by_share(r);
            load_to_lds_x4(qb + (long)(r - q * t.share) * t.q_hs + (long)(first + q) * t.q_rs + 8 * (lchunk ^ k_swz<D>(i)),
                           lds0 + slot * TILE + wave * (NL * 1024) + j * 1024);
        }
    };
    // The logarithms of the sums of a chunk's rows, infinite for rows that are none: they give nothing.
    const float2* const ml = a.ml + (long)bh * a.parts * a.pitch;
    auto fetch = [&](int chunk) {
#pragma unroll
        for (int i = 0; i < CHUNK / 256; i++) {
            const int r = chunk * CHUNK + i * 256 + tid;
            float x = INFINITY;
            if (r < rows) {
                // (the parts that hold keys of the row: others were not written, or hold nothing of it)
                const int parts = a.by_steps((first + a.by_share(r)) / WG_STEP) + 1;
                float2 v = make_float2(-INFINITY, 0.f);
                for (int p0 = 0; p0 < parts; p0 += 8) {
                    float2 u[8];
                    float m = v.x;
#pragma unroll
                    for (int p = 0; p < 8; p++) {  // (the last one again behind the last)
                        u[p] = ml[imin(p0 + p, parts - 1) * a.pitch + r];
                        m = fmaxf(m, u[p].x);
                    }
                    v.y *= share_of(v, m);
#pragma unroll
                    for (int p = 0; p < 8; p++) v.y += p0 + p < parts ? u[p].y * share_of(u[p], m) : 0.f;
                    v.x = m;
                }
                x = v.x + __builtin_amdgcn_logf(v.y);
            }
            lse[chunk & 1][i * 256 + tid] = x;
        }
    };
    constexpr int PER = CHUNK / STEP;
    if (begin < end) {
        issue(begin, 0);
        fetch(begin / PER);
    }
    int qread[NK];
#pragma unroll
    for (int s = 0; s < NK; s++) qread[s] = (32 * BLK * rg + ln) * ROW + (((2 * s + lc) ^ k_swz<D>(ln)) * 16);
#pragma unroll
    for (int s = 0; s < NK; s++) {
        u32x4_t x = bit_cast<u32x4_t>(kf[s]);
        asm volatile("" : "+v"(x));
        kf[s] = bit_cast<half8_t>(x);
    }
    float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int s = begin; s < end; s++) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int slot = (s - begin) & 1;
        const uint8_t* l = lds + slot * TILE;
        if ((s == begin || s % PER == 0) && (s / PER + 1) * PER < end) fetch(s / PER + 1);
        if (s + 1 < end) issue(s + 1, 1 - slot);
        const float* const from = &lse[(s / PER) & 1][s % PER * STEP];
        const bool masked = first + a.by_share(s * STEP) < key0 + 32 * KG - 1;
#pragma unroll
        for (int i = 0; i < BLK; i++) {
            float16_t st;
#pragma unroll
            for (int v = 0; v < 16; v++) st[v] = 0.f;
#pragma unroll
            for (int k = 0; k < NK; k++) {
                const half8_t qf = *(const half8_t*)(l + qread[k] + i * (32 * ROW));
                st = __builtin_amdgcn_mfma_f32_32x32x16_f16(qf, kf[k], st, 0, 0, 0);
            }
            const int r0 = 32 * (BLK * rg + i) + 4 * lc;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float4_t x = *(const float4_t*)(from + r0 + 8 * j);
#pragma unroll
                for (int v = 0; v < 4; v++) st[4 * j + v] = __builtin_fmaf(st[4 * j + v], a.qk_scale, -x[v]);
            }
            if (masked) {
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const int r = s * STEP + r0 + 8 * (v >> 2) + (v & 3);
                    st[v] = key <= first + a.by_share(r) ? st[v] : -INFINITY;
                }
            }
#pragma unroll
            for (int v = 0; v < 16; v++) sums[v & 3] += __builtin_amdgcn_exp2f(st[v]);
        }
    }
    float sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    sum += __shfl_xor(sum, 32);
    if constexpr (RG > 1) {
        __syncthreads();
        float* red = reinterpret_cast<float*>(lds);
        if (lc == 0) red[wave * 32 + ln] = sum;
        __syncthreads();
        if (rg != 0) return;
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < RG; i++) sum += red[(i * KG + kg) * 32 + ln];
    }
    if (lc == 0 && key < t.S) out[key] = key < n ? sum : 0.f;
}

// Workgroups that the keys are cut for in the first pass where there are few rows.  The second pass joins the parts, each time it
// needs a row: the last 64 queries of ragged prompts of up to 8191 rows, 4 x 8 heads (us): 45.7 with 512, 46.5 with 1024, 53.1
// with 2048, 67.3 with 4096; one such prompt 25.2, 29.5, 39.6, 39.6.
constexpr int WG_WGS = 512;
constexpr int WG_PAIRS = 128;  // (8 x 32 heads x 2048: 425 us with 64, 413 with 128)
// Workgroups below which a tile of the second pass is 32 keys wide instead of 128 (8 heads x 4096 keys, 4 query heads each: 263 us
// instead of 346; 8191 keys and 64 queries of one prompt 57 instead of 30: its tiles are shorter than their beginning).
constexpr int WG_NARROW = 512;

WeighPlan plan(int B, int H, int share, int S, int window) {
    WeighPlan a = {};
    a.queries = window > 0 ? std::min(window, S) : S;
    a.pitch = (long)a.queries * share;
    a.tiles = (int)((a.pitch + WG_ROWS - 1) / WG_ROWS);
    const int steps = (S + WG_STEP - 1) / WG_STEP;
    a.steps = (int)std::max<long>(((long)B * H * a.tiles * steps + WG_WGS - 1) / WG_WGS, 1);
    if ((long)B * H * a.tiles >= WG_NARROW) a.steps = steps;
    a.parts = (steps + a.steps - 1) / a.steps;
    a.by_share = Divisor::of(share);
    a.by_heads = Divisor::of(H);
    a.by_parts = Divisor::of(a.parts);
    a.by_pairs = Divisor::of(B * H > 8 ? std::min((B * H + 7) / 8 * 8, WG_PAIRS) : B * H);
    a.by_tiles = Divisor::of(std::max(a.tiles * a.parts, 1));
    a.by_steps = Divisor::of(a.steps);
    return a;
}

}  // namespace

size_t attention_weights_workspace_bytes(int B, int H, int share, int S, int window) {
    const WeighPlan a = plan(B, H, share, S, window);
    return (size_t)B * H * a.parts * a.pitch * sizeof(float2);
}

hipError_t launch_attention_weights(const WeighArgs& t, int D, float sm_scale, void* workspace, hipStream_t st) {
    WeighPlan a = plan(t.B, t.H, t.share, t.S, t.window);
    a.t = t;
    a.ml = (float2*)workspace;
    a.qk_scale = sm_scale * 1.44269504f;
    const int pairs = (int)a.by_pairs.value, groups = (t.B * t.H + pairs - 1) / pairs;
    const dim3 rows((unsigned)groups * pairs * a.tiles * a.parts);
    const long wide = (long)t.B * t.H * ((t.S + 127) / 128);
    const bool narrow = wide < WG_NARROW;
    a.by_key_tiles = Divisor::of(narrow ? (t.S + 31) / 32 : (t.S + 127) / 128);
    const dim3 keys((unsigned)groups * pairs * a.by_key_tiles.value);
    const int step = narrow ? 128 : 64;
    a.even = step % t.share == 0 && (t.share * t.q_hs + step / t.share * t.q_rs) * 2 < (1L << 31);
    if (D == 64) {
        hipLaunchKernelGGL((weigh_rows_kernel<64>), rows, dim3(256), 0, st, a);
        if (narrow) hipLaunchKernelGGL((weigh_keys_kernel<64, 1, 4>), keys, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((weigh_keys_kernel<64, 4, 1>), keys, dim3(256), 0, st, a);
    } else {
        hipLaunchKernelGGL((weigh_rows_kernel<128>), rows, dim3(256), 0, st, a);
        if (narrow) hipLaunchKernelGGL((weigh_keys_kernel<128, 1, 4>), keys, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((weigh_keys_kernel<128, 4, 1>), keys, dim3(256), 0, st, a);
    }
    return hipGetLastError();
}

}  // namespace sq
