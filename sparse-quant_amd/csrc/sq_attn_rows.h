// Attention of up to 32 rows (token, query head) of one key/value head over fp16 keys and values, by a workgroup of four waves:
// what single tokens and short tails are served with (sq_prefix_attn.hip, sq_evict.hip).
//
// The keys go round the waves in blocks of 32.  A wave works by itself: it requests its block's keys and values straight into
// its own part of LDS, and the next block's keys as soon as the scores are formed, its values behind the second product, so that
// no barrier stands in the stream and a wave always has 8 KB or more on the way (D = 128; eight waves on a CU).  Products as in
// sq_attn.hip: S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_32x32x16_f16, a lane has one row, P^T is where it is needed.  With few
// rows most of a product is unused, and it does not matter: at the memory's rate a wave has 7 us for a block's 16 KB, and
// takes 0.5.  What does matter for a short call is the length of the code, which comes from memory on every launch:
// blocks that are not plain take the rolled form of the requests.
#pragma once
#include "sq_attn_tile.h"

namespace sq {

constexpr int RA_WAVES = 4;
constexpr int RA_BLOCK = 32;  // keys

// Division of 32-bit numbers by one that the host knows: a multiplication instead of twenty instructions (Granlund and Montgomery,
// Division by invariant integers using multiplication, 1994: the multiplier rounded up).
struct Divisor {
    uint32_t mul, shift, value;
    __host__ static Divisor of(uint32_t d) {
        Divisor r;
        uint32_t l = 0;
        while (l < 32 && (1ull << l) < d) l++;
        r.mul = (uint32_t)(((((1ull << l) - d) << 32) / d) + 1);
        r.shift = l;
        r.value = d;
        return r;
    }
    __device__ __forceinline__ int operator()(int n) const {
        const uint32_t h = __umulhi((uint32_t)n, mul);
        const uint32_t q = (uint32_t)(((uint64_t)h + (uint32_t)n) >> shift);
        return (int)q;
    }
};

// How much of a state (reference, sum) counts beside the highest reference m.  One without a reference has seen nothing, sum 0, or
// scores that are no numbers, sum NaN: it counts as its sum.
__device__ __forceinline__ float share_of(float2 s, float m) {
    return s.x == -INFINITY ? s.y : __builtin_amdgcn_exp2f(s.x - m);
}

// Probabilities meet the values in fp16, as 2^(score - reference): the reference lies 2^7 below the largest score when it is set and
// moves when one exceeds it by more than 2^15, so that p stays inside fp16 and nothing needs rescaling until then, and what is
// 2^-32 of the largest or more is not 0.  (With the largest at 1, a million rows of 2^-26 beside it, 1.5 % of the sum, were lost.)
constexpr float REF_BELOW = 7.f, REF_MOVES = 15.f;

template <int D>
struct RowsAttn {
    static constexpr int ROW = D * 2;
    static constexpr int TILE = RA_BLOCK * ROW;      // a block's keys, or its values
    static constexpr int LDS = RA_WAVES * 2 * TILE;  // of the workgroup
    static constexpr int NK = D / 16;
    static constexpr int DT = D / 32;
    static constexpr int NL = TILE / 1024;           // direct loads of a tile
    static constexpr int RPL = 1024 / ROW;           // rows of a load
    static constexpr int CPR = D / 8;                // chunks of a row

    half8_t qf[NK];
    float16_t acc[DT];
    float ref, top, sum;  // reference (0 while unset), the score above it at which it moves, this lane's share of the sum

    static __device__ __forceinline__ int swz(bool value, int row) { return value ? v_swz<D>(row) : k_swz<D>(row); }

    __device__ __forceinline__ void load_query(const half_t* row) {  // + 8 * (lane / 32)
#pragma unroll
        for (int s = 0; s < NK; s++) qf[s] = *(const half8_t*)(row + 16 * s);
    }

    // A block whose rows lie rs bytes apart from `base` on.
    static __device__ __forceinline__ void request(const uint8_t* base, uint32_t rs, bool value, uint32_t at) {
        const int lane = threadIdx.x & 63;
        const uint32_t lrow = lane / CPR, lchunk = lane % CPR;
        uint32_t off = lrow * rs;
        base = uniform(base);
#pragma unroll
        for (int j = 0; j < NL; j++) {
            load_to_lds_x4(base, off + (lchunk ^ swz(value, RPL * j + lrow)) * 16, at + j * 1024);
            off += RPL * rs;
        }
    }
    // Any rows: row_of(i) is where row i of the block lies.
    template <class F>
    static __device__ __forceinline__ void request_each(bool value, uint32_t at, F row_of) {
        const int lane = threadIdx.x & 63;
        const int lrow = lane / CPR, lchunk = lane % CPR;
#pragma unroll 1
        for (int j = 0; j < NL; j++) {
            const int r = RPL * j + lrow;
            load_to_lds_x4((const uint8_t*)row_of(r) + (lchunk ^ swz(value, r)) * 16, at + j * 1024);
        }
    }
    // Row r of a tile <- a chunk per lane.
    static __device__ __forceinline__ void put(uint8_t* tile, bool value, int r, int chunk, u32x4_t x) {
        *(u32x4_t*)(tile + r * ROW + ((chunk ^ swz(value, r)) * 16)) = x;
    }
    static __device__ __forceinline__ void clear_from(uint8_t* tile, int r0) {  // of a tile of values
        const int lane = threadIdx.x & 63;
        for (int r = r0 + lane / CPR; r < RA_BLOCK; r += 64 / CPR) put(tile, true, r, lane % CPR, (u32x4_t){0u, 0u, 0u, 0u});
    }

    // Blocks blk, blk + RA_WAVES, .. below blk1 of this wave.  issue(block, value, at) requests a tile; keys(block, tile) and
    // values(block, tile) may change what has landed; seen(block, first, full, last): the block's first key, the keys below which
    // all rows see, and the last that this lane's row sees; scored(block, st) is given the scores in units of log2 (this lane's
    // row, keys 8 i + 4 (lane / 32) + 0..3).  EXACT: the sum is that of the unrounded exponentials, otherwise of those that meet
    // the values.
    // prepare() is called by all waves, behind the first requests.
    template <bool EXACT, class Prepare, class Issue, class Seen, class Keys, class Values, class Scored>
    __device__ __forceinline__ void run(uint8_t* lds, int blk, int blk1, float qk_scale, Prepare prepare, Issue issue, Seen seen,
                                        Keys keys, Values values, Scored scored) {
        const int lane = threadIdx.x & 63, ln = lane & 31, lc = lane >> 5;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        uint8_t* const kt = lds + wave * 2 * TILE;
        uint8_t* const vt = kt + TILE;
        const uint32_t kt0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)kt;
        ref = 0.f, top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int v = 0; v < 16; v++) acc[dt][v] = 0.f;
        if (blk < blk1) {
            issue(blk, false, kt0);
            issue(blk, true, kt0 + TILE);
        }
        prepare();
        if (blk >= blk1) return;
        const int vkey = 4 * lc + ((lane & 15) >> 2);  // + 16 s + 8 i, which leave v_swz unchanged
        const int vchunk = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
        const uint8_t* const vread = vt + vkey * ROW + 8 * (lane & 1);
        for (;;) {
            const int next = blk + RA_WAVES;
            int n, full, last;
            seen(blk, n, full, last);
            wait_landed();
            keys(blk, kt);
            float16_t st;
#pragma unroll
            for (int v = 0; v < 16; v++) st[v] = 0.f;
            {
                half8_t kf[NK];
#pragma unroll
                for (int s = 0; s < NK; s++) kf[s] = *(const half8_t*)(kt + ln * ROW + (((2 * s + lc) ^ k_swz<D>(ln)) * 16));
#pragma unroll
                for (int s = 0; s < NK; s++) st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[s], qf[s], st, 0, 0, 0);
            }
            if (n + RA_BLOCK > full) {
#pragma unroll
                for (int v = 0; v < 16; v++) st[v] = n + 8 * (v >> 2) + 4 * lc + (v & 3) <= last ? st[v] * qk_scale : -INFINITY;
            } else {
#pragma unroll
                for (int v = 0; v < 16; v++) st[v] *= qk_scale;
            }
            scored(blk, st);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (next < blk1) issue(next, false, kt0);  // (the keys are in registers)
            float mx = -INFINITY;
#pragma unroll
            for (int v = 0; v < 16; v++) {
                st[v] -= ref;
                mx = fmaxf(mx, st[v]);
            }
            if (__builtin_amdgcn_ballot_w64(mx > top) != 0) {
                const float mq = fmaxf(mx, __shfl_xor(mx, 32));
                const bool upd = mq > top;
                const float delta = upd ? mq - REF_BELOW : 0.f;
                const float alpha = (upd && top != -INFINITY) ? __builtin_amdgcn_exp2f(-delta) : 1.f;
                ref += delta;
                top = upd ? REF_MOVES : top;
                sum *= alpha;
#pragma unroll
                for (int v = 0; v < 16; v++) st[v] -= delta;
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int v = 0; v < 16; v++) acc[dt][v] *= alpha;
            }
            half8_t pk[2];  // rounded to fp16 as the second product's operands are
#pragma unroll
            for (int v = 0; v < 16; v++) {
                const float p = __builtin_amdgcn_exp2f(st[v]);
                const half_t h = (half_t)p;
                sum += EXACT ? p : (float)h;
                pk[v >> 3][v & 7] = h;
            }
            if (next < blk1) wait_landed();
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            values(blk, vt);
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int dt = 0; dt < DT; dt++) {
                    const uint8_t* const p = vread + (((4 * dt + vchunk) ^ v_swz<D>(vkey)) * 16) + 16 * i * ROW;
                    const u32x2_t lo = bit_cast<u32x2_t>(lds_read_tr(p)), hi = bit_cast<u32x2_t>(lds_read_tr(p + 8 * ROW));
                    const u32x4_t x = {lo.x, lo.y, hi.x, hi.y};
                    acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bit_cast<half8_t>(x), pk[i], acc[dt], 0, 0, 0);
                }
            blk = next;
            if (blk >= blk1) break;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            issue(blk, true, kt0 + TILE);
        }
        sum += __shfl_xor(sum, 32);
    }
    // All requests but the last tile's have landed.
    static __device__ __forceinline__ void wait_landed() {
        if constexpr (NL == 8) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
        static_assert(NL == 8 || NL == 4);
    }

    // The waves' states of a row joined: emit(row, column, four sums, reference, sum) for the first `rows` rows.  stat: [4][32].
    template <class Emit>
    __device__ __forceinline__ void join(uint8_t* lds, float2* stat, int rows, Emit emit) {
        const int tid = threadIdx.x, lane = tid & 63, ln = lane & 31, lc = lane >> 5;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        __syncthreads();  // (the tiles are the waves' own, but a wave's sums cover others' tiles)
        if (ln < rows) {
            float4_t* const mine = (float4_t*)lds + (wave * RA_BLOCK + ln) * (D / 4);
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    mine[(8 * dt + 2 * i + lc) ^ (ln & 7)] =
                        (float4_t){acc[dt][4 * i], acc[dt][4 * i + 1], acc[dt][4 * i + 2], acc[dt][4 * i + 3]};
        }
        if (lc == 0) stat[wave * RA_BLOCK + ln] = make_float2(top == -INFINITY ? -INFINITY : ref, sum);
        __syncthreads();
        for (int i = tid; i < rows * (D / 4); i += 64 * RA_WAVES) {
            const int row = i / (D / 4), c = i % (D / 4);
            float2 s[RA_WAVES];
            float m = -INFINITY;
#pragma unroll
            for (int w = 0; w < RA_WAVES; w++) {
                s[w] = stat[w * RA_BLOCK + row];
                m = fmaxf(m, s[w].x);
            }
            float l = 0.f;
            float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < RA_WAVES; w++) {
                const float f = share_of(s[w], m);
                l += s[w].y * f;
                const float4_t x = ((const float4_t*)lds)[(w * RA_BLOCK + row) * (D / 4) + (c ^ (row & 7))];
                o += x * f;
            }
            emit(row, 4 * c, o, m, l);
        }
    }
};

}  // namespace sq
