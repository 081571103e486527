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
#include "sq_attn_tile.h"
#include "sq_kernels.h"

#include <algorithm>
#include <type_traits>

namespace sq {

namespace {

constexpr int PA_STEP = 64;  // keys of a step

struct PrefixArgs {
    PrefixAttn t;
    PrefixPlan p;
    float qk_scale;  // sm_scale * log2(e)
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }
__device__ __forceinline__ int imax(int a, int b) { return a > b ? a : b; }

// All bits of the halves of a word that are infinities or NaN.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    return ((w & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((w & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
}

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
    const int row0 = tl.tile * p.rows;
    const int row1 = imin(row0 + p.rows, tl.count * t.share) - 1;
    r.own = imin(imax(r.before + row1 / t.share + 1, 0), t.Lmax);
    r.own_first = imin(imax(r.before + row0 / t.share + 1, 0), t.Lmax);
    r.pre_steps = p.packed ? 0 : ceil_div(t.P, PA_STEP);
    r.steps = r.pre_steps + ceil_div(r.own, PA_STEP);
    return r;
}

// QG groups of 32 rows, KG groups of keys: wave (qg, kg) has rows 32 qg .. + 31 and a KG-th of the keys of a step.
template <int D, int QG, int KG>
__global__ __launch_bounds__(64 * QG * KG, QG == 1 ? 1 : 2) void prefix_attn_kernel(PrefixArgs a) {
    constexpr int NW = QG * KG;
    constexpr int KS = PA_STEP / (32 * KG);  // 32-key blocks of a wave and step
    constexpr int ROW = D * 2;               // bytes of a tile row
    constexpr int TILE = PA_STEP * ROW;
    constexpr int SB = 2 * TILE;             // a stage: K tile, V tile
    constexpr int NK = D / 16;
    constexpr int DT = D / 32;
    constexpr int NL = TILE / 1024 / NW;     // direct loads per wave, operand and stage
    constexpr int RPL = 1024 / ROW;          // tile rows per load
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * SB];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;

    const PrefixAttn& t = a.t;
    const PrefixPlan& p = a.p;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ln = lane & 31, lc = lane >> 5;
    const int qg = wave / KG, kg = wave % KG;

    // ---- which piece of work this is
    int index = blockIdx.x;
    int head, part, row0, rows, s0, s1;  // rows row0 .. row0 + rows - 1 of the head's T * share; steps s0 .. s1 - 1
    Tile tl = {0, 0, 0, 0};
    Reach rc = {0, 0, 0, 0, 0};
    const bool shared = index < p.grid_a;
    if (shared) {
        const int per = p.grid_a >> 3;
        const int work = (index & 7) * per + (index >> 3);  // an eighth of the list per XCD: a prefix piece's tiles share an L2
        if (work >= p.units_a) return;
        const int tile = work % p.tiles_a;
        part = work / p.tiles_a % p.parts_a;
        head = work / p.tiles_a / p.parts_a;
        row0 = tile * p.rows;
        rows = imin(p.rows, t.T * t.share - row0);
        s0 = part * p.steps_a;
        s1 = imin(s0 + p.steps_a, ceil_div(t.P, PA_STEP));
    } else if ((index -= p.grid_a) < p.grid_b) {
        const int per = p.grid_b >> 3;
        const int work = (index & 7) * per + (index >> 3);
        if (work >= p.units_b) return;
        const int b_part = work / p.tiles_b % p.parts_b;
        head = work / p.tiles_b / p.parts_b;
        if (!tile_of(t, p.rows, p.tiles_b - 1 - work % p.tiles_b, tl)) return;
        rc = reach_of(t, p, tl);
        row0 = tl.first * t.share + tl.tile * p.rows;
        rows = imin(p.rows, tl.count * t.share - tl.tile * p.rows);
        s0 = b_part * p.steps_b;
        s1 = imin(s0 + p.steps_b, rc.steps);
        if (s0 >= s1 && b_part > 0) return;  // (the first part also stands for rows that see nothing)
        part = p.parts_a + b_part;
    } else {
        // the call's own rows into the cache, a token per wave
        index -= p.grid_b;
        const int token = index * NW + wave;
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
        return;
    }

    const bool idle = 32 * qg >= rows;  // (a sequence's tile may be shorter than the workgroup's)
    const int row = row0 + imin(32 * qg + ln, rows - 1);
    const int token = row / t.share;
    const int qhead = head * t.share + row - token * t.share;
    const int limit = imin(rc.before + token - tl.first, t.Lmax - 1);  // the last own row that it sees
    // own rows from here on come from the call's rows, not from the cache, which other workgroups are storing them to
    const int fresh = t.kn ? rc.before : t.Lmax;

    half8_t qf[NK];
    {
        const half_t* qp = t.q + (long)token * t.q_ts + (long)qhead * t.q_hs + 8 * lc;
#pragma unroll
        for (int s = 0; s < NK; s++) qf[s] = *(const half8_t*)(qp + 16 * s);
    }

    const half_t* const kp = t.kp + (long)head * t.p_hs;
    const half_t* const vp = t.vp + (long)head * t.p_hs;
    const long own_at = (long)tl.b * t.c_bs + (long)head * t.c_hs;
    const half_t* const ko = t.kc + own_at;
    const half_t* const vo = t.vc + own_at;
    const long new_at = (long)tl.first * t.n_ts + (long)head * t.n_hs;

    const int pre_steps = shared ? s1 : rc.pre_steps;
    const int lrow = lane / (D / 8), lchunk = lane % (D / 8);
    const int row_w = RPL * NL * wave + lrow;  // of this lane's first load in the tile
    auto issue = [&](int s, int slot) {
        const bool pre = s < pre_steps;
        const int n = (pre ? s : s - pre_steps) * PA_STEP;
        const int end = pre ? t.P : rc.own;
        const int rs = (int)(pre ? t.p_rs : t.c_rs) * 2;
        const half_t* const kb = pre ? kp : ko;
        const half_t* const vb = pre ? vp : vo;
        const uint32_t l0 = lds0 + slot * SB + wave * (NL * 1024);
        if (n + PA_STEP <= (pre ? end : imin(end, fresh))) {
            const uint8_t* const kbase = uniform((const uint8_t*)kb + (long)n * rs);
            const uint8_t* const vbase = uniform((const uint8_t*)vb + (long)n * rs);
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const int r = row_w + RPL * j;
                load_to_lds_x4(kbase, (uint32_t)(r * rs + ((lchunk ^ k_swz<D>(r)) * 16)), l0 + j * 1024);
            }
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const int r = row_w + RPL * j;
                load_to_lds_x4(vbase, (uint32_t)(r * rs + ((lchunk ^ v_swz<D>(r)) * 16)), l0 + TILE + j * 1024);
            }
        } else {  // rows past the end re-read the last one (their scores are masked)
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const int r = row_w + RPL * j;
                const int key = imin(n + r, end - 1);
                const bool is_new = !pre && key >= fresh;
                const uint8_t* const kr = is_new ? (const uint8_t*)(t.kn + new_at + (long)(key - fresh) * t.n_ts)
                                                 : (const uint8_t*)kb + (long)key * rs;
                const uint8_t* const vr = is_new ? (const uint8_t*)(t.vn + new_at + (long)(key - fresh) * t.n_ts)
                                                 : (const uint8_t*)vb + (long)key * rs;
                load_to_lds_x4(kr + (lchunk ^ k_swz<D>(r)) * 16, l0 + j * 1024);
                load_to_lds_x4(vr + (lchunk ^ v_swz<D>(r)) * 16, l0 + TILE + j * 1024);
            }
        }
    };
    if (s0 < s1) issue(s0, 0);

    // LDS byte offsets of the operand reads.
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

    // Reference maximum of the row (0 while unset), the score above it at which it moves (any score while unset), and
    // this lane's share of the row sum.
    constexpr float LAZY = 8.f;
    float ref = 0.f, top = -INFINITY, l_i = 0.f;
    float16_t acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int v = 0; v < 16; v++) acc[dt][v] = 0.f;

    // Keys 16 i .. + 15 of this wave's, columns 32 dt .. + 31.
    auto values = [&](const uint8_t* l, int i, int dt) {
        const u32x2_t lo = bit_cast<u32x2_t>(lds_read_tr(l + vread[dt] + 16 * i * ROW));
        const u32x2_t hi = bit_cast<u32x2_t>(lds_read_tr(l + vread[dt] + (16 * i + 8) * ROW));
        return (u32x4_t){lo.x, lo.y, hi.x, hi.y};
    };
    auto visit = [&](int s, auto slot_, bool more) {
        constexpr int SLOT = decltype(slot_)::value;
        const uint8_t* l = lds + SLOT * SB;
        if (more) issue(s + 1, 1 - SLOT);
        if (idle) return;
        __builtin_amdgcn_sched_barrier(0);
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
        const bool pre = s < pre_steps;
        const int n = (pre ? s : s - pre_steps) * PA_STEP;
        // Masks (only where the step touches the end of the rows or the causal diagonal; the test is uniform).
        const bool masked = n + PA_STEP > (pre ? t.P : rc.own_first);
        const int last = pre ? t.P - 1 : limit;
        if (masked) {
#pragma unroll
            for (int b = 0; b < KS; b++)
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const int key = n + 32 * (KS * kg + b) + 8 * (v >> 2) + 4 * lc + (v & 3);
                    st[b][v] = key <= last ? st[b][v] : -INFINITY;
                }
        }
        // The reference maximum moves only when a score exceeds it by more than 2^LAZY (or when it is still unset): until
        // then p = exp2(score) stays inside fp16 and nothing needs rescaling.
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < KS; b++)
#pragma unroll
            for (int v = 0; v < 16; v++) mx = fmaxf(mx, st[b][v]);
        if (__builtin_amdgcn_ballot_w64(mx > top) != 0) {
            const float mq = fmaxf(mx, __shfl_xor(mx, 32));
            const bool upd = mq > top;
            const float delta = upd ? mq : 0.f;
            const float alpha = (upd && top != -INFINITY) ? __builtin_amdgcn_exp2f(-delta) : 1.f;
            ref += delta;
            top = upd ? LAZY : top;
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
        uint32_t odd = 0;  // whether a value that some row must not see is no finite number
#pragma unroll
        for (int i = 0; i < 2 * KS; i++)
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                u32x4_t vt = values(l, i, dt);
                if (masked) {
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        const uint32_t m = not_finite(vt[w]);
                        odd |= m;
                        vt[w] &= ~m;
                    }
                }
                acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bit_cast<half8_t>(vt), pk[i], acc[dt], 0, 0, 0);
            }
        // Infinities and NaN reach the rows that see them and no others: a product of its own for each of the keys, of which
        // these rows take their part (0 times them is no 0).
        if (masked && __builtin_amdgcn_ballot_w64(odd != 0) != 0) {
#pragma unroll
            for (int i = 0; i < 2 * KS; i++)
#pragma unroll 1
                for (int e = 0; e < 16; e++) {
                    const bool mine = ((e >> 2) & 1) == lc;
                    const int el = (e & 3) + 4 * (e >> 3);
                    const bool visible = n + 32 * KS * kg + 16 * i + e <= last;
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) {
                        u32x4_t vt = values(l, i, dt);
#pragma unroll
                        for (int w = 0; w < 4; w++)
                            vt[w] = mine && (el >> 1) == w ? vt[w] & not_finite(vt[w]) & (el & 1 ? 0xffff0000u : 0xffffu) : 0u;
                        float16_t x;
#pragma unroll
                        for (int v = 0; v < 16; v++) x[v] = 0.f;
                        x = __builtin_amdgcn_mfma_f32_32x32x16_f16(bit_cast<half8_t>(vt), pk[i], x, 0, 0, 0);
#pragma unroll
                        for (int v = 0; v < 16; v++) acc[dt][v] += visible ? x[v] : 0.f;
                    }
                }
        }
    };

    auto landed = []() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
#pragma unroll
    for (int s = 0; s < NK; s++) {
        u32x4_t x = bit_cast<u32x4_t>(qf[s]);
        asm volatile("" : "+v"(x));
        qf[s] = bit_cast<half8_t>(x);
    }
    for (int s = s0; s < s1; s += 2) {
        landed();
        visit(s, std::integral_constant<int, 0>{}, s + 1 < s1);
        if (s + 1 >= s1) break;
        landed();
        visit(s + 1, std::integral_constant<int, 1>{}, s + 2 < s1);
    }

    // ---- the row's state: over its two lanes, then over the key groups
    l_i += __shfl_xor(l_i, 32);
    float m_i = top == -INFINITY ? -INFINITY : ref;
    float w_own = 1.f;
    constexpr int OWN = KG == 2 ? DT / 2 : DT;  // column tiles that a wave finishes
    __syncthreads();
    float4_t other[OWN][4];
    float w_peer = 0.f;
    if constexpr (KG == 2) {
        // each wave hands half of its columns to the other key group's wave and finishes the others
        float4_t* red = reinterpret_cast<float4_t*>(lds);                        // [wave][OWN][4][64]
        float2* stat = reinterpret_cast<float2*>(lds + NW * OWN * 4096);         // [wave][64]
        static_assert(NW * OWN * 4096 + NW * 512 <= 2 * SB, "fits");
#pragma unroll
        for (int d = 0; d < OWN; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float4_t x;
#pragma unroll
                for (int j = 0; j < 4; j++) x[j] = kg == 0 ? acc[OWN + d][4 * i + j] : acc[d][4 * i + j];
                red[((wave * OWN + d) * 4 + i) * 64 + lane] = x;
            }
        stat[wave * 64 + lane] = make_float2(m_i, l_i);
        __syncthreads();
        const int peer = wave ^ 1;
        const float2 ps = stat[peer * 64 + lane];
        const float mm = fmaxf(m_i, ps.x);
        w_own = m_i == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_i - mm);
        w_peer = ps.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ps.x - mm);
        l_i = l_i * w_own + ps.y * w_peer;
        m_i = mm;
#pragma unroll
        for (int d = 0; d < OWN; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) other[d][i] = red[((peer * OWN + d) * 4 + i) * 64 + lane];
    }
    const bool valid = 32 * qg + ln < rows;
    const bool direct = p.parts_a + p.parts_b == 1;
    const float inv = direct ? (l_i == 0.f ? 0.f : 1.f / l_i) : 1.f;  // a row that sees nothing: 0
    const long slot = ((long)head * (p.parts_a + p.parts_b) + part) * ((long)t.T * t.share) + row;
    const long o_at = ((long)token * (t.H * t.share) + qhead) * D;
    if (!valid) return;
#pragma unroll
    for (int d = 0; d < OWN; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float4_t x;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (KG == 2)
                    x[j] = ((kg == 0 ? acc[d][4 * i + j] : acc[OWN + d][4 * i + j]) * w_own + other[d][i][j] * w_peer) * inv;
                else
                    x[j] = acc[d][4 * i + j] * inv;
            }
            const int col = 32 * (d + (KG == 2 && kg ? OWN : 0)) + 8 * i + 4 * lc;
            if (direct) {
                half4_t h;
#pragma unroll
                for (int j = 0; j < 4; j++) h[j] = (half_t)x[j];
                *(half4_t*)(t.o + o_at + col) = h;
            } else {
                *(float4_t*)(p.po + slot * D + col) = x;
            }
        }
    if (!direct && lc == 0 && kg == 0) p.pml[slot] = make_float2(m_i, l_i);
}

// The parts of a row (token, query head), a row per wave.
template <int D>
__global__ __launch_bounds__(256) void prefix_join_kernel(PrefixArgs a) {
    const PrefixAttn& t = a.t;
    const PrefixPlan& p = a.p;
    constexpr int EPL = D / 64;
    typedef float vec_t __attribute__((ext_vector_type(EPL)));
    typedef half_t hvec_t __attribute__((ext_vector_type(EPL)));
    const int lane = threadIdx.x & 63;
    const int index = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int heads = t.H * t.share;
    const int token = index / heads;
    if (token >= t.T) return;
    const int qhead = index - token * heads;
    const int head = qhead / t.share;
    Tile tl;
    tl.b = sequence_of(t, token);
    if (tl.b < 0) return;
    tokens_of(t, tl.b, tl.first, tl.count);
    const int row = token * t.share + qhead - head * t.share;
    tl.tile = (row - tl.first * t.share) / p.rows;
    const Reach rc = reach_of(t, p, tl);
    const int total = p.parts_a + p.parts_b;
    const int parts = p.parts_a + imin(imax(ceil_div(rc.steps, p.steps_b), 1), p.parts_b);
    const long rows = (long)t.T * t.share;
    const long slot = (long)head * total * rows + row;
    float m = -INFINITY, l = 0.f;
    vec_t o = {};
    for (int s0 = 0; s0 < parts; s0 += 64) {
        float2 ml = make_float2(-INFINITY, 0.f);
        if (s0 + lane < parts) ml = p.pml[slot + (s0 + lane) * rows];
        float mx = ml.x;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) mx = fmaxf(mx, __shfl_xor(mx, x));
        mx = fmaxf(mx, m);
        const float w = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - mx);
        float ls = ml.y * w;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) ls += __shfl_xor(ls, x);
        const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mx);
        l = l * f + ls;
        o *= f;
        m = mx;
        const int n = imin(parts - s0, 64);
        for (int s = 0; s < n; s += 8) {
            vec_t x[8];
#pragma unroll
            for (int j = 0; j < 8; j++)
                x[j] = *(const vec_t*)(p.po + (slot + (s0 + imin(s + j, n - 1)) * rows) * D + EPL * lane);
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (s + j < n) o += x[j] * bit_cast<float>(__builtin_amdgcn_readlane(bit_cast<int>(w), s + j));
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    hvec_t h;
#pragma unroll
    for (int i = 0; i < EPL; i++) h[i] = (half_t)(o[i] * inv);
    *(hvec_t*)(t.o + ((long)token * heads + qhead) * D + EPL * lane) = h;
}

int div_up(long a, long b) { return (int)((a + b - 1) / b); }
int pad8(long n) { return (int)((n + 7) / 8 * 8); }

// Workgroups that the pieces of a launch are cut for: two per CU.
constexpr int PA_WGS = 512;

}  // namespace

PrefixPlan prefix_plan(int T, int B, int H, int share, int P, int Lmax, bool ragged) {
    PrefixPlan p = {};
    const long rows = (long)T * share;          // of a key/value head
    const long each = (rows + B - 1) / B;       // of a sequence, on average
    p.packed = P > 0 && B > 1 && each < 64;
    const long most = p.packed ? rows : each;
    p.qg = most <= 32 ? 1 : most <= 64 ? 2 : 4;
    p.rows = 32 * p.qg;
    const int pre = div_up(P, PA_STEP), own = div_up(Lmax, PA_STEP);
    if (p.packed) {
        p.tiles_a = div_up(rows, p.rows);
        const long steps = (long)H * p.tiles_a * pre;
        p.steps_a = std::max(div_up(steps, PA_WGS), 1);
        p.parts_a = div_up(pre, p.steps_a);
        p.units_a = (long)H * p.parts_a * p.tiles_a;
    }
    p.tiles_b = ragged ? (int)(rows / p.rows + B) : B * div_up((long)(T / B) * share, p.rows);
    const int steps_b = own + (p.packed ? 0 : pre);
    p.steps_b = std::max(div_up((long)p.tiles_b * H * steps_b, PA_WGS), 1);
    p.parts_b = std::max(div_up(steps_b, p.steps_b), 1);
    p.units_b = (long)H * p.parts_b * p.tiles_b;
    p.grid_a = pad8(p.units_a);
    p.grid_b = pad8(p.units_b);
    return p;
}

size_t prefix_attention_workspace_bytes(int T, int B, int H, int share, int D, int P, int Lmax, bool ragged) {
    const PrefixPlan p = prefix_plan(T, B, H, share, P, Lmax, ragged);
    const size_t parts = p.parts_a + p.parts_b;
    return parts == 1 ? 0 : parts * H * T * share * (D + 2) * sizeof(float);
}

hipError_t launch_prefix_attention(const PrefixAttn& t, int D, float sm_scale, void* workspace, hipStream_t st) {
    PrefixArgs a;
    a.t = t;
    a.p = prefix_plan(t.T, t.B, t.H, t.share, t.P, t.Lmax, t.starts != nullptr);
    a.qk_scale = sm_scale * 1.44269504f;
    const int parts = a.p.parts_a + a.p.parts_b;
    a.p.po = (float*)workspace;
    a.p.pml = (float2*)(a.p.po + (size_t)parts * t.H * t.T * t.share * D);
#define SQ_PREFIX_LAUNCH(D_, QG_, KG_)                                                                                     \
    hipLaunchKernelGGL((prefix_attn_kernel<D_, QG_, KG_>),                                                                 \
                       dim3(a.p.grid_a + a.p.grid_b + (t.kn ? (t.T + QG_ * KG_ - 1) / (QG_ * KG_) : 0)), dim3(64 * QG_ * KG_), 0, \
                       st, a)
    if (D == 64) {
        if (a.p.qg == 1) SQ_PREFIX_LAUNCH(64, 1, 2);
        else if (a.p.qg == 2) SQ_PREFIX_LAUNCH(64, 2, 2);
        else SQ_PREFIX_LAUNCH(64, 4, 1);
    } else {
        if (a.p.qg == 1) SQ_PREFIX_LAUNCH(128, 1, 2);
        else if (a.p.qg == 2) SQ_PREFIX_LAUNCH(128, 2, 2);
        else SQ_PREFIX_LAUNCH(128, 4, 1);
    }
#undef SQ_PREFIX_LAUNCH
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || parts == 1) return e;
    const dim3 grid(div_up((long)t.T * t.H * t.share, 4));
    if (D == 64)
        hipLaunchKernelGGL((prefix_join_kernel<64>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((prefix_join_kernel<128>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace sq
