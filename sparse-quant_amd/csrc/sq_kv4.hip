// A key/value cache held in 4 bits: quantising new rows into it, choosing pages by a bound of their scores, copying
// pages (layout: sq_kv4.h; attention: sq_kv4_attn.hip).
#include "sq_kernels.h"
#include "sq_kv4_row.h"

#include <type_traits>

namespace sq {

namespace {

// ------------------------------------------------------------------------------------------------------- append
//
// A workgroup owns one page of one head and with it the page's bounds, so nothing is shared between workgroups and nothing is
// atomic (the row itself: sq_kv4_row.h).  One wave where a sequence gets one row; four otherwise, each with every fourth
// pass of rows (6421 tokens of 12 prompts, 8 heads in groups of 32: 22.1 / 20.0 / 22.2 / 30.8 us with 2 / 4 / 8 / 16 waves).
// Bounds: a step of 8 sequences 3.65 us, of which a launch that does nothing is 1.7; the prompts move 61 MB in 18 to 20 us
// (3.1 to 3.4 TB/s; a copy of as many bytes 12.3) and spend as long on the codes as on the loads.
struct Kv4AppendArgs {
    Kv4Cache c;
    const half_t* k;
    const half_t* v;
    half_t* k_hat;  // what the rows read as, contiguous [T][H][D], or null
    half_t* v_hat;
    long k_ts, k_hs, v_ts, v_hs;  // element strides over token and head
};

template <int D, int G, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void kv4_append_kernel(Kv4AppendArgs a) {
    constexpr int g = D / G;
    constexpr int LPR = D / 8;     // lanes of a row
    constexpr int RPW = 64 / LPR;  // rows of a wave
    constexpr int REC = kv4_record_bytes(D, g);
    __shared__ __attribute__((aligned(16))) half2_t ext[WAVES][2][D / 2];
    const Kv4Cache& c = a.c;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int head = blockIdx.x % c.H;
    int unit = blockIdx.x / c.H;

    // The sequence and its unit-th page that gets rows.
    int b = 0, first = 0, count = 0, len = 0;
    if (!c.starts) {
        const int per = (c.each + KV4_PAGE - 2) / KV4_PAGE + 1;
        b = unit / per;
        unit -= b * per;
        if (b >= c.B) return;
        kv4_tokens(c, b, first, count);
        len = c.lengths[b];
    } else {
        bool found = false;
        for (int b0 = 0; b0 < c.B && !found; b0 += 64) {
            int f = 0, n = 0, l = 0, touched = 0;
            if (b0 + lane < c.B) {
                kv4_tokens(c, b0 + lane, f, n);
                l = c.lengths[b0 + lane];
                touched = n > 0 ? (n + KV4_PAGE - 2) / KV4_PAGE + 1 : 0;
            }
            const int upto = wave_scan(touched);
            const unsigned long long past = __ballot(upto > unit);
            if (past) {
                const int at = __ffsll(past) - 1;
                b = b0 + at;
                unit -= __shfl(upto - touched, at, 64);
                first = __shfl(f, at, 64);
                count = __shfl(n, at, 64);
                len = __shfl(l, at, 64);
                found = true;
            } else {
                unit -= __shfl(upto, 63, 64);
            }
        }
        if (!found) return;
    }
    if (len <= 0 || count <= 0) return;
    // Rows [len - count, len), those inside the table; rows of this page [r0, r1).
    const long begin = (long)len - count;
    const long row_lo = begin < 0 ? 0 : begin;
    const long row_hi = len < (long)c.width * KV4_PAGE ? len : (long)c.width * KV4_PAGE;
    const long page = row_lo / KV4_PAGE + unit;
    const long pr = page * KV4_PAGE;
    const int r0 = (int)((row_lo > pr ? row_lo : pr) - pr);
    const int r1 = (int)((row_hi < pr + KV4_PAGE ? row_hi : pr + KV4_PAGE) - pr);
    if (r0 >= r1) return;
    const int id = c.table[(long)b * c.table_stride + page];
    if ((unsigned)id >= (unsigned)c.num_pages) return;
    uint8_t* const rec = c.pool + ((long)id * c.H + head) * REC;
    const long token0 = first + (pr - begin);  // token of row 0 of the page (it may lie before the first)

    const int sub = lane % LPR, slot = lane / LPR;
    half_t* const bounds = (half_t*)(rec + 64 * D + 512 * G);
    half8_t old_hi, old_lo;  // what the page had, unless its row 0 is among the rows of this call
#pragma unroll
    for (int e = 0; e < 8; e++) old_hi[e] = (half_t)-INFINITY, old_lo[e] = (half_t)INFINITY;
    if (r0 > 0 && threadIdx.x < LPR) {
        old_hi = *(const half8_t*)(bounds + 8 * sub);
        old_lo = *(const half8_t*)(bounds + D + 8 * sub);
    }
    half2_t top[4], bottom[4];  // of the lane's elements over its rows
#pragma unroll
    for (int j = 0; j < 4; j++)
        top[j] = (half2_t){(half_t)-INFINITY, (half_t)-INFINITY}, bottom[j] = (half2_t){(half_t)INFINITY, (half_t)INFINITY};

    // A pass of the workgroup is WAVES * RPW rows; the next one's are asked for ahead.
    const half_t* const kp = a.k + head * a.k_hs + 8 * sub;
    const half_t* const vp = a.v + head * a.v_hs + 8 * sub;
    int row = r0 + wave * RPW + slot;
    long t = token0 + imin(row, r1 - 1);
    half8_t k8 = *(const half8_t*)(kp + t * a.k_ts), v8 = *(const half8_t*)(vp + t * a.v_ts);
#pragma unroll 1
    while (true) {
        const int next = row + WAVES * RPW;
        const long tn = token0 + imin(next, r1 - 1);
        const half8_t kn = *(const half8_t*)(kp + tn * a.k_ts), vn = *(const half8_t*)(vp + tn * a.v_ts);
        const RowOut hat = {a.k_hat ? a.k_hat + (t * c.H + head) * D : nullptr, a.v_hat ? a.v_hat + (t * c.H + head) * D : nullptr};
        kv4_store_row<D, G>(rec, row, k8, v8, row < r1, hat);
        // (a row behind the last is the last once more)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const half2_t x = {k8[2 * j], k8[2 * j + 1]};
            top[j] = pair_max(top[j], x);
            bottom[j] = pair_min(bottom[j], x);
        }
        if (__ballot(next < r1) == 0) break;
        row = next, t = tn, k8 = kn, v8 = vn;
    }
    // Bounds: over the wave's rows, the waves', and the page's before.
#pragma unroll
    for (int j = 0; j < 4; j++) {
        auto fold = [&](half2_t v, auto join) {
            if constexpr (LPR == 8) v = join(v, bit_cast<half2_t>(lane_move<0x128>(bit_cast<uint32_t>(v))));  // row_ror:8
            float x, y;
            pair16(bit_cast<float>(v), x, y);
            v = join(bit_cast<half2_t>(x), bit_cast<half2_t>(y));
            pair32(bit_cast<float>(v), x, y);
            return join(bit_cast<half2_t>(x), bit_cast<half2_t>(y));
        };
        top[j] = fold(top[j], pair_max);
        bottom[j] = fold(bottom[j], pair_min);
    }
    if constexpr (WAVES > 1) {
        if (slot == 0) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                ext[wave][0][4 * sub + j] = top[j];
                ext[wave][1][4 * sub + j] = bottom[j];
            }
        }
        __syncthreads();
    }
    if (threadIdx.x < LPR) {
        half8_t hi8, lo8;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            half2_t hi = top[j], lo = bottom[j];
#pragma unroll
            for (int w = 1; w < WAVES; w++) {
                hi = pair_max(hi, ext[w][0][4 * sub + j]);
                lo = pair_min(lo, ext[w][1][4 * sub + j]);
            }
            hi = pair_max(hi, (half2_t){old_hi[2 * j], old_hi[2 * j + 1]});
            lo = pair_min(lo, (half2_t){old_lo[2 * j], old_lo[2 * j + 1]});
            hi8[2 * j] = hi[0], hi8[2 * j + 1] = hi[1];
            lo8[2 * j] = lo[0], lo8[2 * j + 1] = lo[1];
        }
        *(half8_t*)(bounds + 8 * sub) = hi8;
        *(half8_t*)(bounds + D + 8 * sub) = lo8;
    }
}

// --------------------------------------------------------------------------------------------------------- copy

// Pages of all layers, src[i] to dst[i]; a pair with an index outside the pool is left out.  16 KB of a page per workgroup,
// four 16-byte loads of a thread under way at once: 195 MB of 8 layers in 39 to 42 us, what a large copy reaches (5 TB/s);
// one page of 32 layers 3.15 us.
__global__ __launch_bounds__(256) void kv4_copy_kernel(uint8_t* pool, const int* src, const int* dst, int num_pages,
                                                       int parts, long page_bytes, long layer_bytes) {
    const int pair = blockIdx.x / parts, part = blockIdx.x % parts;
    const int from = src[pair], to = dst[pair];
    if ((unsigned)from >= (unsigned)num_pages || (unsigned)to >= (unsigned)num_pages || from == to) return;
    uint8_t* const base = pool + (long)blockIdx.y * layer_bytes;
    const u32x4_t* s = (const u32x4_t*)(base + from * page_bytes);
    u32x4_t* d = (u32x4_t*)(base + to * page_bytes);
    const int n = (int)(page_bytes / 16);
    const int i0 = part * 1024 + threadIdx.x;
    u32x4_t t[4];
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (i0 + 256 * j < n) t[j] = s[i0 + 256 * j];
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (i0 + 256 * j < n) d[i0 + 256 * j] = t[j];
}

// ------------------------------------------------------------------------------------------------------- select
//
// score(page) = max over the head's queries of sum_d max(q_d hi_d, q_d lo_d), hi and lo the page's largest and
// smallest keys: no key of the page can score higher.  Which of two pages is the better one must not hang on the order
// of a sum: products of fp16 numbers are exact in fp32, their sums are taken in 64 bits.
// 16 (D = 64: 8) lanes share a page, 8 elements each; the choice between hi and lo goes by the signs of the queries, which
// a lane keeps as masks of pairs.  A wave takes SELECT_PAGES pages, all their bounds asked for at once (8 sequences of up
// to 32768 rows and 8 heads: 7.1 us, up to 17 MB of bounds in pieces of 512 bytes; 125 pages of 8 heads 16.9 us for all three
// launches with 8 pages a wave, 17.3 with 16).  A launch of its own: with the choice in the same one, by the workgroup that
// ends last, the two took 8.5 instead of 8.4 and 20 instead of 11 us.
constexpr int SELECT_QUERIES = 4;  // of a round
constexpr int SELECT_PAGES = 8;    // of a wave

struct Kv4SelectArgs {
    Kv4Cache c;
    const half_t* q;
    int* selected;   // [B][H][count]
    double* scores;  // [B][H][width]
    long q_ts, q_hs;
    int share, count, keep_first, keep_last;
};

typedef short short2_t __attribute__((ext_vector_type(2)));

template <int CTRL>
__device__ __forceinline__ double row_move(double v) {
    const u32x2_t u = bit_cast<u32x2_t>(v);
    return bit_cast<double>((u32x2_t){lane_move<CTRL>(u.x), lane_move<CTRL>(u.y)});
}

template <int D>
__global__ __launch_bounds__(64) void kv4_score_kernel(Kv4SelectArgs a, int rec_bytes) {
    constexpr int LPP = D / 8, PPI = 64 / LPP, N = SELECT_PAGES / PPI;
    const Kv4Cache& c = a.c;
    const int lane = threadIdx.x;
    const int head = blockIdx.y % c.H, b = blockIdx.y / c.H;
    const int pages = (kv4_length(c, b) + KV4_PAGE - 1) / KV4_PAGE;
    const int first = blockIdx.x * SELECT_PAGES;
    if (pages <= a.count || first >= pages) return;
    const int sub = lane % LPP, slot = lane / LPP;
    int id = first + lane < pages && lane < SELECT_PAGES ? c.table[(long)b * c.table_stride + first + lane] : -1;
    u32x4_t hi[N], lo[N];
    bool real[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        int p = __shfl(id, PPI * i + slot, 64);
        real[i] = (unsigned)p < (unsigned)c.num_pages;
        if (!real[i]) p = 0;
        const uint8_t* const bounds = c.pool + ((long)p * c.H + head) * rec_bytes + rec_bytes - 4 * D + 16 * sub;
        hi[i] = *(const u32x4_t*)bounds;
        lo[i] = *(const u32x4_t*)(bounds + 2 * D);
    }
    double best[N];
#pragma unroll
    for (int i = 0; i < N; i++) best[i] = -INFINITY;
    for (int g0 = 0; g0 < a.share; g0 += SELECT_QUERIES) {
        half8_t q[SELECT_QUERIES];
#pragma unroll
        for (int g = 0; g < SELECT_QUERIES; g++)  // (a round's queries beyond the last are the last again)
            q[g] = *(const half8_t*)(a.q + (long)b * a.q_ts + (long)(head * a.share + imin(g0 + g, a.share - 1)) * a.q_hs + 8 * sub);
#pragma unroll
        for (int g = 0; g < SELECT_QUERIES; g++) {
            const u32x4_t qb = bit_cast<u32x4_t>(q[g]);
            uint32_t minus[4];
#pragma unroll
            for (int j = 0; j < 4; j++) minus[j] = bit_cast<uint32_t>(bit_cast<short2_t>(qb[j]) >> (short)15);
#pragma unroll
            for (int i = 0; i < N; i++) {
                double s = 0.0;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const half2_t x = bit_cast<half2_t>((lo[i][j] & minus[j]) | (hi[i][j] & ~minus[j]));
                    s += (double)((float)x[0] * (float)q[g][2 * j]);
                    s += (double)((float)x[1] * (float)q[g][2 * j + 1]);
                }
                s += row_move<0xB1>(s);                // quad_perm 1,0,3,2
                s += row_move<0x4E>(s);                // quad_perm 2,3,0,1
                s += row_move<0x141>(s);               // row_half_mirror: the other quad of eight
                if (D == 128) s += row_move<0x140>(s);  // row_mirror: the other eight
                if (s > best[i]) best[i] = s;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int page = first + PPI * i + slot;
        if (sub == 0 && page < pages) a.scores[((long)b * c.H + head) * c.width + page] = real[i] ? best[i] : -INFINITY;
    }
}

// A double as an unsigned number of the same order; one that is no number is the lowest.
__device__ __forceinline__ unsigned long long ordered(double x) {
    if (!(x == x)) return 0;
    const unsigned long long u = bit_cast<unsigned long long>(x + 0.0);
    return u & 0x8000000000000000ull ? ~u : u | 0x8000000000000000ull;
}

// (1024 / 512 / 256: 17.7 / 17.3 / 17.2 us for all three launches at 125 pages, 30.0 / 29.6 / 30.2 at 512)
constexpr int SELECT_THREADS = 512;

// The `count` best pages of a head in ascending order, ties to the lowest; -1 behind the last where there are fewer.
// The count-th largest key is found digit by digit, from the top, until no other key shares its digits.  4 to 5 us, most of it
// the barriers of two or three digits.
__global__ __launch_bounds__(SELECT_THREADS) void kv4_select_kernel(Kv4SelectArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned long long keys[];
    __shared__ unsigned hist[256];
    __shared__ unsigned waves[SELECT_THREADS / 64][2];
    __shared__ unsigned digit_at, left_at, shared_by;
    const Kv4Cache& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int b = blockIdx.x / c.H;
    const int pages = (kv4_length(c, b) + KV4_PAGE - 1) / KV4_PAGE;
    int* const out = a.selected + (long)blockIdx.x * a.count;
    if (pages <= a.count) {
        for (int i = tid; i < a.count; i += SELECT_THREADS) out[i] = i < pages ? i : -1;
        return;
    }
    const double* const scores = a.scores + (long)blockIdx.x * c.width;
    for (int i = tid; i < pages; i += SELECT_THREADS)
        keys[i] = i < a.keep_first || i >= pages - a.keep_last ? ~0ull : ordered(scores[i]);
    unsigned long long prefix = 0, mask = 0;
    unsigned left = a.count;  // of the keys that share the prefix, how many are taken
    for (int shift = 56; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < pages; i += SELECT_THREADS)
            if ((keys[i] & mask) == prefix) atomicAdd(&hist[(keys[i] >> shift) & 255], 1u);
        __syncthreads();
        if (tid < 64) {
            // keys of digits above: lane l has digits 255 - 4 l downwards
            unsigned n[4], sum = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) sum += n[j] = hist[255 - 4 * lane - j];
            unsigned before = (unsigned)wave_scan((int)sum) - sum;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (before < left && before + n[j] >= left) {
                    digit_at = 255 - 4 * lane - j;
                    left_at = left - before;
                    shared_by = n[j];
                }
                before += n[j];
            }
        }
        __syncthreads();
        prefix |= (unsigned long long)digit_at << shift;
        mask |= 255ull << shift;
        left = left_at;
        if (shared_by == left) break;  // every key that shares the prefix is taken
        // (the next pass writes these three behind its second barrier)
    }
    // Keys above the prefix are taken, of those that share it the first `left`.
    unsigned taken = 0, ties = 0;
    for (int i0 = 0; i0 < pages; i0 += SELECT_THREADS) {
        const int i = i0 + tid;
        const unsigned long long key = i < pages ? keys[i] & mask : 0;
        const bool above = i < pages && key > prefix, tie = i < pages && key == prefix;
        const unsigned long long am = __ballot(above), tm = __ballot(tie);
        __syncthreads();
        if (lane == 0) {
            waves[wave][0] = __popcll(am);
            waves[wave][1] = __popcll(tm);
        }
        __syncthreads();
        unsigned a_before = 0, t_before = 0, a_all = 0, t_all = 0;
#pragma unroll
        for (int w = 0; w < SELECT_THREADS / 64; w++) {
            if (w == wave) a_before = a_all, t_before = t_all;
            a_all += waves[w][0];
            t_all += waves[w][1];
        }
        const unsigned long long below = (1ull << lane) - 1;
        a_before += __popcll(am & below);
        t_before += __popcll(tm & below) + ties;
        const unsigned at = taken + a_before + (t_before < left ? t_before : left) - (ties < left ? ties : left);
        if (above || (tie && t_before < left)) out[at] = i;
        const unsigned t_new = ties + t_all;
        taken += a_all + (t_new < left ? t_new : left) - (ties < left ? ties : left);
        ties = t_new;
    }
}

}  // namespace

hipError_t launch_kv4_append(const Kv4Cache& c, const void* k, const void* v, void* k_hat, void* v_hat, int D, int g,
                             const long* strides, hipStream_t st) {
    Kv4AppendArgs a;
    a.c = c;
    a.k = (const half_t*)k;
    a.v = (const half_t*)v;
    a.k_hat = (half_t*)k_hat;
    a.v_hat = (half_t*)v_hat;
    a.k_ts = strides[0];
    a.k_hs = strides[1];
    a.v_ts = strides[2];
    a.v_hs = strides[3];
    // Pages that get rows: n tokens touch at most (n + 62) / 64 + 1 of them.
    const long units = c.starts ? c.T / KV4_PAGE + 2l * (c.B < c.T ? c.B : c.T)
                                : (long)c.B * ((c.each + KV4_PAGE - 2) / KV4_PAGE + 1);
    const dim3 grid((unsigned)(units * c.H));
    auto go = [&](auto d, auto groups) {
        // one row per sequence: one wave; otherwise four share a page
        if (!c.starts && c.each == 1)
            hipLaunchKernelGGL((kv4_append_kernel<d.value, groups.value, 1>), grid, dim3(64), 0, st, a);
        else
            hipLaunchKernelGGL((kv4_append_kernel<d.value, groups.value, 4>), grid, dim3(256), 0, st, a);
    };
    if (D == 128 && g == 128) go(std::integral_constant<int, 128>{}, std::integral_constant<int, 1>{});
    if (D == 128 && g == 64) go(std::integral_constant<int, 128>{}, std::integral_constant<int, 2>{});
    if (D == 128 && g == 32) go(std::integral_constant<int, 128>{}, std::integral_constant<int, 4>{});
    if (D == 64 && g == 64) go(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    if (D == 64 && g == 32) go(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    return hipGetLastError();
}

hipError_t launch_kv4_copy_pages(void* pool, const int* src, const int* dst, int n, int num_pages, int layers,
                                 long page_bytes, long layer_bytes, hipStream_t st) {
    const int parts = (int)((page_bytes / 16 + 1023) / 1024);
    hipLaunchKernelGGL(kv4_copy_kernel, dim3((unsigned)n * parts, layers), dim3(256), 0, st, (uint8_t*)pool, src, dst, num_pages,
                       parts, page_bytes, layer_bytes);
    return hipGetLastError();
}

hipError_t launch_kv4_select(const Kv4Cache& c, const void* q, void* selected, void* workspace, int D, int g, int share,
                             long q_ts, long q_hs, int count, int keep_first, int keep_last, hipStream_t st) {
    Kv4SelectArgs a;
    a.c = c;
    a.q = (const half_t*)q;
    a.selected = (int*)selected;
    a.scores = (double*)workspace;
    a.q_ts = q_ts;
    a.q_hs = q_hs;
    a.share = share;
    a.count = count;
    a.keep_first = keep_first;
    a.keep_last = keep_last;
    const int heads = c.B * c.H;
    if (c.width > count) {
        const dim3 grid((c.width + SELECT_PAGES - 1) / SELECT_PAGES, heads);
        if (D == 128)
            hipLaunchKernelGGL(kv4_score_kernel<128>, grid, dim3(64), 0, st, a, kv4_record_bytes(D, g));
        else
            hipLaunchKernelGGL(kv4_score_kernel<64>, grid, dim3(64), 0, st, a, kv4_record_bytes(D, g));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(kv4_select_kernel, dim3(heads), dim3(SELECT_THREADS), (size_t)c.width * 8, st, a);
    return hipGetLastError();
}

}  // namespace sq
