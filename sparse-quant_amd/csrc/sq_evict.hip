// A key/value cache of a fixed number of rows that evicts by accumulated attention weight (fp16, one token per sequence).
//
// A step: where the cache is not full the token's row goes behind the others; where it is, the row of the lowest weight among
// those that are neither of the first `first` nor of the last `last` tokens makes way for it.  The token attends over the rows,
// its own among them, and every row's weight grows by what the token's heads give it:
//   P = softmax_j(scale q . k_j),  out = sum_j P_j v_j,  weight_j += sum over the query heads of the key/value head of P_j
// The probabilities are known only behind the last row, so the scores wait in the workspace (4 bytes of a row's 512 at D = 128).
#include "sq_attn_tile.h"
#include "sq_kernels.h"

#include <algorithm>
#include <type_traits>

namespace sq {

namespace {

constexpr int EV_STEP = 64;   // rows of a step
constexpr int EV_TILE = 32;   // query heads of a workgroup
constexpr int EV_WAVES = 2;

struct EvictArgs {
    EvictStep t;
    float* scores;  // [B][H][share][pitch], in units of log2
    float* po;      // [B][H][parts][share][D]
    float2* pml;    // [B][H][parts][share]
    int pitch, parts, steps, tiles;
    float qk_scale;
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }
__device__ __forceinline__ int imax(int a, int b) { return a > b ? a : b; }

// Order of weights as unsigned numbers; a NaN is the lowest.
__device__ __forceinline__ uint32_t order_of(float w) {
    const uint32_t u = bit_cast<uint32_t>(w);
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

template <int D>
__global__ __launch_bounds__(64 * EV_WAVES, 1) void evict_attn_kernel(EvictArgs a) {
    constexpr int ROW = D * 2;
    constexpr int TILE = EV_STEP * ROW;
    constexpr int SB = 2 * TILE;
    constexpr int NK = D / 16;
    constexpr int DT = D / 32;
    constexpr int NL = TILE / 1024 / EV_WAVES;
    constexpr int RPL = 1024 / ROW;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * SB];
    __shared__ uint64_t least[EV_WAVES];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;

    const EvictStep& t = a.t;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ln = lane & 31, lc = lane >> 5;
    const int part = blockIdx.x % a.parts;
    const int tile = blockIdx.x / a.parts % a.tiles;
    const int bh = blockIdx.x / a.parts / a.tiles;
    const int b = bh / t.H, h = bh - b * t.H;
    const int seen = t.seen[b];
    const int n = imin(seen, t.R);  // rows attended
    const int s0 = part * a.steps;
    const int s1 = imin(s0 + a.steps, ceil_div(n, EV_STEP));
    if (s0 >= s1) return;  // (also where nothing was seen: the second launch writes zeros)

    const int rows = imin(EV_TILE, t.share - tile * EV_TILE);
    const int g = tile * EV_TILE + imin(ln, rows - 1);
    half8_t qf[NK];
    {
        const half_t* qp = t.q + (long)b * t.q_bs + (long)(h * t.share + g) * t.q_hs + 8 * lc;
#pragma unroll
        for (int s = 0; s < NK; s++) qf[s] = *(const half8_t*)(qp + 16 * s);
    }
    const long c_at = (long)b * t.c_bs + (long)h * t.c_hs;
    const half_t* const kb = t.kc + c_at;
    const half_t* const vb = t.vc + c_at;
    const int rs = (int)t.c_rs * 2;
    const int lrow = lane / (D / 8), lchunk = lane % (D / 8);
    const int row_w = RPL * NL * wave + lrow;
    auto issue = [&](int s, int slot) {
        const int at = s * EV_STEP;
        const uint8_t* const kbase = uniform((const uint8_t*)kb + (long)at * rs);
        const uint8_t* const vbase = uniform((const uint8_t*)vb + (long)at * rs);
        const uint32_t l0 = lds0 + slot * SB + wave * (NL * 1024);
#pragma unroll
        for (int j = 0; j < NL; j++) {  // rows past the end re-read the last one (their scores are masked)
            const int r = row_w + RPL * j;
            load_to_lds_x4(kbase, (uint32_t)(imin(r, n - 1 - at) * rs + ((lchunk ^ k_swz<D>(r)) * 16)), l0 + j * 1024);
        }
#pragma unroll
        for (int j = 0; j < NL; j++) {
            const int r = row_w + RPL * j;
            load_to_lds_x4(vbase, (uint32_t)(imin(r, n - 1 - at) * rs + ((lchunk ^ v_swz<D>(r)) * 16)), l0 + TILE + j * 1024);
        }
    };
    issue(s0, 0);

    // The new row, a chunk of it per thread.
    constexpr int CPR = D / 8;
    const int chunk = tid % CPR;
    const long n_at = (long)b * t.n_bs + (long)h * t.n_hs + 8 * chunk;
    u32x4_t fresh_k = *(const u32x4_t*)(t.kn + n_at);
    u32x4_t fresh_v = *(const u32x4_t*)(t.vn + n_at);
    // Where it goes.
    int slot = seen - 1;
    if (seen > t.R) {
        const float* const w = t.weight + (long)bh * t.R;
        const int* const pos = t.position + (long)bh * t.R;
        uint64_t best = ~0ull;
        for (int r = tid; r < t.R; r += 64 * EV_WAVES) {
            const int p = pos[r];
            const uint32_t o = p >= t.first && p < seen - t.last ? order_of(w[r]) : ~0u;
            const uint64_t key = ((uint64_t)o << 32) | (uint32_t)r;
            best = key < best ? key : best;
        }
        best = wave_min64(best);
        if (lane == 0) least[wave] = best;
        __syncthreads();
        uint64_t v = least[0];
#pragma unroll
        for (int i = 1; i < EV_WAVES; i++) v = least[i] < v ? least[i] : v;
        slot = __builtin_amdgcn_readfirstlane((int)(uint32_t)v);
    }

    int kread[NK], vread[DT];
#pragma unroll
    for (int s = 0; s < NK; s++) kread[s] = (32 * wave + ln) * ROW + (((2 * s + lc) ^ k_swz<D>(ln)) * 16);
    {
        const int key = 4 * lc + ((lane & 15) >> 2);
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
            vread[dt] = TILE + (32 * wave + key) * ROW + (((4 * dt + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ v_swz<D>(key)) * 16) +
                        8 * (lane & 1);
    }

    float ref = 0.f, top = -INFINITY, l_i = 0.f;
    constexpr float LAZY = 8.f;
    float16_t acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int v = 0; v < 16; v++) acc[dt][v] = 0.f;
    float* const scores = a.scores + ((long)bh * t.share + g) * a.pitch;
    const bool valid = ln < rows;

    auto visit = [&](int s, auto slot_, bool more) {
        constexpr int SLOT = decltype(slot_)::value;
        uint8_t* l = lds + SLOT * SB;
        const int at = s * EV_STEP;
        const bool here = slot >= at && slot < at + EV_STEP;
        if (here || at + EV_STEP > n) {
            if (here) {  // the new row takes its place
                const int r = slot - at;
                if (tid < CPR) {
                    *(u32x4_t*)(l + r * ROW + ((chunk ^ k_swz<D>(r)) * 16)) = fresh_k;
                    *(u32x4_t*)(l + TILE + r * ROW + ((chunk ^ v_swz<D>(r)) * 16)) = fresh_v;
                    if (tile == 0) {
                        *(u32x4_t*)(t.kc + c_at + (long)slot * t.c_rs + 8 * chunk) = fresh_k;
                        *(u32x4_t*)(t.vc + c_at + (long)slot * t.c_rs + 8 * chunk) = fresh_v;
                    }
                }
                if (tid == 0 && tile == 0) t.slot[bh] = slot;
            }
            // values behind the last row meet probabilities of 0: they must be numbers
            for (int i = imax(n - at, 0) + tid / CPR; i < EV_STEP; i += 64 * EV_WAVES / CPR)
                *(u32x4_t*)(l + TILE + i * ROW + ((chunk ^ v_swz<D>(i)) * 16)) = (u32x4_t){0u, 0u, 0u, 0u};
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
        if (more) issue(s + 1, 1 - SLOT);
        __builtin_amdgcn_sched_barrier(0);
        float16_t st;
#pragma unroll
        for (int v = 0; v < 16; v++) st[v] = 0.f;
        half8_t kf[NK];
#pragma unroll
        for (int i = 0; i < NK; i++) kf[i] = *(const half8_t*)(l + kread[i]);
#pragma unroll
        for (int i = 0; i < NK; i++) st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i], qf[i], st, 0, 0, 0);
        const int k0 = at + 32 * wave + 4 * lc;
#pragma unroll
        for (int v = 0; v < 16; v++) {
            const int key = k0 + 8 * (v >> 2) + (v & 3);
            st[v] = key < n ? st[v] * a.qk_scale : -INFINITY;
        }
        if (valid) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                *(float4_t*)(scores + k0 + 8 * i) = (float4_t){st[4 * i], st[4 * i + 1], st[4 * i + 2], st[4 * i + 3]};
        }
        float mx = -INFINITY;
#pragma unroll
        for (int v = 0; v < 16; v++) {
            st[v] -= ref;
            mx = fmaxf(mx, st[v]);
        }
        if (__builtin_amdgcn_ballot_w64(mx > top) != 0) {
            const float mq = fmaxf(mx, __shfl_xor(mx, 32));
            const bool upd = mq > top;
            const float delta = upd ? mq : 0.f;
            const float alpha = (upd && top != -INFINITY) ? __builtin_amdgcn_exp2f(-delta) : 1.f;
            ref += delta;
            top = upd ? LAZY : top;
            l_i *= alpha;
#pragma unroll
            for (int v = 0; v < 16; v++) st[v] -= delta;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int v = 0; v < 16; v++) acc[dt][v] *= alpha;
        }
        // The sum is that of the unrounded exponentials: the weights are divided by it and keep 32 bits.
        half8_t pk[2];
#pragma unroll
        for (int v = 0; v < 16; v++) {
            const float p = __builtin_amdgcn_exp2f(st[v]);
            l_i += p;
            pk[v >> 3][v & 7] = (half_t)p;
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                const u32x2_t lo = bit_cast<u32x2_t>(lds_read_tr(l + vread[dt] + 16 * i * ROW));
                const u32x2_t hi = bit_cast<u32x2_t>(lds_read_tr(l + vread[dt] + (16 * i + 8) * ROW));
                u32x4_t vt = {lo.x, lo.y, hi.x, hi.y};
                acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bit_cast<half8_t>(vt), pk[i], acc[dt], 0, 0, 0);
            }
    };
    auto landed = []() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
#pragma unroll
    for (int s = 0; s < NK; s++) {
        u32x4_t x = bit_cast<u32x4_t>(qf[s]);
        asm volatile("" : "+v"(x));
        qf[s] = bit_cast<half8_t>(x);
    }
    asm volatile("" : "+v"(fresh_k), "+v"(fresh_v));
    for (int s = s0; s < s1; s += 2) {
        landed();
        visit(s, std::integral_constant<int, 0>{}, s + 1 < s1);
        if (s + 1 >= s1) break;
        landed();
        visit(s + 1, std::integral_constant<int, 1>{}, s + 2 < s1);
    }

    l_i += __shfl_xor(l_i, 32);
    float m_i = top == -INFINITY ? -INFINITY : ref;
    __syncthreads();
    constexpr int OWN = DT / 2;
    float4_t* red = reinterpret_cast<float4_t*>(lds);                       // [wave][OWN][4][64]
    float2* stat = reinterpret_cast<float2*>(lds + EV_WAVES * OWN * 4096);  // [wave][64]
#pragma unroll
    for (int d = 0; d < OWN; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float4_t x;
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = wave == 0 ? acc[OWN + d][4 * i + j] : acc[d][4 * i + j];
            red[((wave * OWN + d) * 4 + i) * 64 + lane] = x;
        }
    stat[wave * 64 + lane] = make_float2(m_i, l_i);
    __syncthreads();
    const float2 ps = stat[(wave ^ 1) * 64 + lane];
    const float mm = fmaxf(m_i, ps.x);
    const float w_own = m_i == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_i - mm);
    const float w_peer = ps.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ps.x - mm);
    if (!valid) return;
    const long slot_at = ((long)bh * a.parts + part) * t.share + g;
#pragma unroll
    for (int d = 0; d < OWN; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4_t o = red[(((wave ^ 1) * OWN + d) * 4 + i) * 64 + lane];
            float4_t x;
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = (wave == 0 ? acc[d][4 * i + j] : acc[OWN + d][4 * i + j]) * w_own + o[j] * w_peer;
            *(float4_t*)(a.po + slot_at * D + 32 * (d + wave * OWN) + 8 * i + 4 * lc) = x;
        }
    if (lc == 0 && wave == 0) a.pml[slot_at] = make_float2(mm, l_i * w_own + ps.y * w_peer);
}

// The parts of a (sequence, key/value head): its outputs (first chunk of rows), and the weights of a chunk of rows.
constexpr int EJ_ROWS = 1024;
constexpr int EJ_HEADS = 64;  // whose maxima and sums are held at once

template <int D>
__global__ __launch_bounds__(256) void evict_join_kernel(EvictArgs a) {
    __shared__ float2 state[EJ_HEADS];
    const EvictStep& t = a.t;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int bh = blockIdx.x, b = bh / t.H;
    const int r0 = blockIdx.y * EJ_ROWS;
    const int seen = t.seen[b];
    const int n = imin(seen, t.R);
    if (r0 >= n && r0 > 0) return;
    half_t* const out = t.o + (long)bh * t.share * D;
    if (seen <= 0) {
        for (int i = tid; i < t.share * D; i += 256) out[i] = (half_t)0.f;
        if (tid == 0) t.slot[bh] = -1;
        return;
    }
    const int parts = ceil_div(ceil_div(n, EV_STEP), a.steps);
    float acc[EJ_ROWS / 256];
#pragma unroll
    for (int i = 0; i < EJ_ROWS / 256; i++) acc[i] = 0.f;
    for (int g0 = 0; g0 < t.share; g0 += EJ_HEADS) {
        const int heads = imin(EJ_HEADS, t.share - g0);
        __syncthreads();
        for (int g = tid; g < heads; g += 256) {
            const float2* ml = a.pml + (long)bh * a.parts * t.share + g0 + g;
            float m = -INFINITY, l = 0.f;
            for (int s = 0; s < parts; s++) m = fmaxf(m, ml[(long)s * t.share].x);
            for (int s = 0; s < parts; s++) {
                const float2 x = ml[(long)s * t.share];
                l += x.x == -INFINITY ? 0.f : x.y * __builtin_amdgcn_exp2f(x.x - m);
            }
            state[g] = make_float2(m, 1.f / l);
        }
        __syncthreads();
        for (int g = 0; g < heads; g++) {
            const float2 st = state[g];
            const float* s = a.scores + ((long)bh * t.share + g0 + g) * a.pitch;
#pragma unroll
            for (int i = 0; i < EJ_ROWS / 256; i++) {
                const int r = r0 + 256 * i + tid;
                if (r < n) acc[i] += __builtin_amdgcn_exp2f(s[r] - st.x) * st.y;
            }
        }
        if (blockIdx.y == 0) {
            for (int g = wave; g < heads; g += 4) {
                const float2 st = state[g];
                const long at = (long)bh * a.parts * t.share + g0 + g;
                for (int c = lane; c < D; c += 64) {
                    float o = 0.f;
                    for (int s = 0; s < parts; s++) {
                        const float m = a.pml[at + (long)s * t.share].x;
                        const float w = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - st.x);
                        o += a.po[(at + (long)s * t.share) * D + c] * w;
                    }
                    out[(g0 + g) * D + c] = (half_t)(o * st.y);
                }
            }
        }
    }
    const int slot = t.slot[bh];
#pragma unroll
    for (int i = 0; i < EJ_ROWS / 256; i++) {
        const int r = r0 + 256 * i + tid;
        if (r < n) {
            float* w = t.weight + (long)bh * t.R + r;
            *w = r == slot ? acc[i] : *w + acc[i];
            if (r == slot) t.position[(long)bh * t.R + r] = seen - 1;
        }
    }
}

// Workgroups that the caches' rows are cut for: two per CU.
constexpr int EV_WGS = 512;

EvictArgs plan(int B, int H, int share, int R) {
    EvictArgs a = {};
    a.pitch = (R + 63) / 64 * 64;
    a.tiles = (share + EV_TILE - 1) / EV_TILE;
    const long units = (long)B * H * a.tiles;
    const int steps = a.pitch / 64;
    a.steps = (int)std::max<long>((units * steps + EV_WGS - 1) / EV_WGS, 1);
    a.parts = (steps + a.steps - 1) / a.steps;
    return a;
}

// ------------------------------------------------------------------------------------------------ a prompt's rows

constexpr int KEEP_THREADS = 1024;
constexpr int KEEP_BINS = 2048;

// Which rows stay: the R of the highest weight, the first and last ones above all, the lower row among equals.  A search for
// the R-th highest weight by its digits from the top (11, 11 and 10 bits, counted in LDS), then one pass that writes the rows
// in their order.
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
    if (D == 64) {
        hipLaunchKernelGGL((evict_attn_kernel<64>), grid, dim3(64 * EV_WAVES), 0, st, a);
        hipLaunchKernelGGL((evict_join_kernel<64>), join, dim3(256), 0, st, a);
    } else {
        hipLaunchKernelGGL((evict_attn_kernel<128>), grid, dim3(64 * EV_WAVES), 0, st, a);
        hipLaunchKernelGGL((evict_join_kernel<128>), join, dim3(256), 0, st, a);
    }
    return hipGetLastError();
}

hipError_t launch_evict_keep(const EvictKeep& t, int D, hipStream_t st) {
    hipLaunchKernelGGL(keep_select_kernel, dim3(t.B * t.H), dim3(KEEP_THREADS), 0, st, t);
    const int per = 256 / (D / 8);
    const dim3 grid((t.R + per - 1) / per, t.B * t.H);
    if (D == 64)
        hipLaunchKernelGGL((keep_gather_kernel<64>), grid, dim3(256), 0, st, t);
    else
        hipLaunchKernelGGL((keep_gather_kernel<128>), grid, dim3(256), 0, st, t);
    return hipGetLastError();
}

}  // namespace sq
