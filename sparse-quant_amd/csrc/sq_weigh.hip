// The attention weight that a prompt's queries give to each of its keys, summed over the queries (all, or the last so many)
// and over the query heads of a key/value head:
//   w[j] = sum_{g, i >= j} exp(scale q_{g,i} . k_j - lse_{g,i}),  lse_{g,i} = log sum_{j <= i} exp(scale q_{g,i} . k_j)
// Two passes over the same products: the sums of the rows first, then the sums of the columns.  The rows (query, head) of a
// key/value head are packed, so that its keys are read once for all of its heads.
#include "sq_attn_tile.h"
#include "sq_kernels.h"

#include <algorithm>
#include <type_traits>

namespace sq {

namespace {

constexpr int WG_STEP = 64;   // keys of a step of the first pass
constexpr int WG_ROWS = 128;  // rows of its workgroups

struct WeighPlan {
    WeighArgs t;
    float2* ml;  // [B][H][parts][pitch]: maximum (in units of log2) and sum of a row over a part of the keys
    long pitch;
    int tiles, parts, steps, queries;
    float qk_scale;
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Rows of sequence b, and how many of them are its queries.
__device__ __forceinline__ void sizes_of(const WeighPlan& a, int b, int& n, int& queries) {
    n = a.t.lengths ? a.t.lengths[b] : a.t.S;
    n = n < 0 ? 0 : imin(n, a.t.S);
    queries = imin(n, a.queries);
}

template <int D>
__global__ __launch_bounds__(256, 2) void weigh_rows_kernel(WeighPlan a) {
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
    const int per = gridDim.x >> 3;
    const int work = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    const int part = work % a.parts;
    const int tile = a.tiles - 1 - work / a.parts % a.tiles;  // those that see most come first
    const int bh = work / a.parts / a.tiles;
    if (bh >= t.B * t.H) return;
    const int b = bh / t.H, h = bh - b * t.H;
    int n, queries;
    sizes_of(a, b, n, queries);
    const int rows = queries * t.share;
    const int row0 = tile * WG_ROWS;
    if (row0 >= rows) return;
    const int first = n - queries;  // the first of its queries
    const int row = imin(row0 + 32 * wave + ln, rows - 1);
    const int query = first + row / t.share;
    const int seen_lo = first + row0 / t.share + 1;                               // keys of the tile's first row
    const int seen = first + (imin(row0 + WG_ROWS, rows) - 1) / t.share + 1;      // ... and of its last
    const int s0 = part * a.steps;
    const int s1 = imin(s0 + a.steps, ceil_div(seen, WG_STEP));

    half8_t qf[NK];
    {
        const half_t* qp = t.q + (long)b * t.q_bs + (long)(h * t.share + row % t.share) * t.q_hs + (long)query * t.q_rs + 8 * lc;
#pragma unroll
        for (int s = 0; s < NK; s++) qf[s] = *(const half8_t*)(qp + 16 * s);
    }
    const half_t* const kb = t.k + (long)b * t.k_bs + (long)h * t.k_hs;
    const int rs = (int)t.k_rs * 2;
    const int lrow = lane / (D / 8), lchunk = lane % (D / 8);
    const int row_w = RPL * NL * wave + lrow;
    auto issue = [&](int s, int slot) {
        const int at = s * WG_STEP;
        const uint8_t* const base = uniform((const uint8_t*)kb + (long)at * rs);
#pragma unroll
        for (int j = 0; j < NL; j++) {
            const int r = row_w + RPL * j;
            load_to_lds_x4(base, (uint32_t)(imin(r, seen - 1 - at) * rs + ((lchunk ^ k_swz<D>(r)) * 16)),
                           lds0 + slot * TILE + wave * (NL * 1024) + j * 1024);
        }
    };
    if (s0 < s1) issue(s0, 0);
    int kread[NK];
#pragma unroll
    for (int s = 0; s < NK; s++) kread[s] = ln * ROW + (((2 * s + lc) ^ k_swz<D>(ln)) * 16);
    float m = -INFINITY, l_i = 0.f;
#pragma unroll
    for (int s = 0; s < NK; s++) {
        u32x4_t x = bit_cast<u32x4_t>(qf[s]);
        asm volatile("" : "+v"(x));
        qf[s] = bit_cast<half8_t>(x);
    }
    for (int s = s0; s < s1; s++) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const uint8_t* l = lds + ((s - s0) & 1) * TILE;
        if (s + 1 < s1) issue(s + 1, 1 - ((s - s0) & 1));
        float16_t st[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
#pragma unroll
            for (int v = 0; v < 16; v++) st[i][v] = 0.f;
#pragma unroll
            for (int k = 0; k < NK; k++) {
                const half8_t kf = *(const half8_t*)(l + kread[k] + i * (32 * ROW));
                st[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[k], st[i], 0, 0, 0);
            }
        }
        if (s * WG_STEP + WG_STEP > seen_lo) {
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const int key = s * WG_STEP + 32 * i + 8 * (v >> 2) + 4 * lc + (v & 3);
                    st[i][v] = key <= query ? st[i][v] * a.qk_scale : -INFINITY;
                }
        } else {
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int v = 0; v < 16; v++) st[i][v] *= a.qk_scale;
        }
        float mx = m;
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int v = 0; v < 16; v++) mx = fmaxf(mx, st[i][v]);
        const float base = mx == -INFINITY ? 0.f : mx;
        l_i *= __builtin_amdgcn_exp2f(m - base);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int v = 0; v < 16; v++) sum += __builtin_amdgcn_exp2f(st[i][v] - base);
        l_i += sum;
        m = mx;
    }
    const float mo = __shfl_xor(m, 32), lo = __shfl_xor(l_i, 32);
    const float mm = fmaxf(m, mo);
    const float l = (m == -INFINITY ? 0.f : l_i * __builtin_amdgcn_exp2f(m - mm)) + (mo == -INFINITY ? 0.f : lo * __builtin_amdgcn_exp2f(mo - mm));
    if (lc == 0 && row0 + 32 * wave + ln < rows) a.ml[((long)bh * a.parts + part) * a.pitch + row] = make_float2(mm, l);
}

// KG groups of 32 keys, RG groups of rows: wave (kg, rg) sums the weights of 32 keys over an RG-th of the rows of a step.
template <int D, int KG, int RG>
__global__ __launch_bounds__(256, 2) void weigh_keys_kernel(WeighPlan a) {
    constexpr int BLK = RG == 1 ? 2 : 1;    // 32-row blocks of a wave and step
    constexpr int STEP = 32 * BLK * RG;     // rows of a step
    constexpr int ROW = D * 2;
    constexpr int TILE = STEP * ROW;
    constexpr int NK = D / 16;
    constexpr int NL = TILE / 1024 / 4;
    constexpr int RPL = 1024 / ROW;
    static_assert(KG * RG == 4);
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * TILE];
    __shared__ __attribute__((aligned(16))) float lse[2][STEP];
    __shared__ __attribute__((aligned(16))) int last[2][STEP];  // the last key that a row sees
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    const WeighArgs& t = a.t;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ln = lane & 31, lc = lane >> 5;
    const int kg = wave % KG, rg = wave / KG;
    const int tiles = ceil_div(t.S, 32 * KG);
    const int per = gridDim.x >> 3;
    const int work = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    const int tile = work % tiles;  // (those that are seen most come first)
    const int bh = work / tiles;
    if (bh >= t.B * t.H) return;
    const int b = bh / t.H, h = bh - b * t.H;
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
    const int begin = imin((key0 > first ? key0 - first : 0) * t.share / STEP, ceil_div(rows, STEP));
    const int end = ceil_div(rows, STEP);

    half8_t kf[NK];
    {
        const half_t* p = t.k + (long)b * t.k_bs + (long)h * t.k_hs + (long)imin(key, n - 1) * t.k_rs + 8 * lc;
#pragma unroll
        for (int s = 0; s < NK; s++) kf[s] = *(const half8_t*)(p + 16 * s);
    }
    const half_t* const qb = t.q + (long)b * t.q_bs + (long)h * t.share * t.q_hs;
    const int lrow = lane / (D / 8), lchunk = lane % (D / 8);
    const int row_w = RPL * NL * wave + lrow;
    const float2* const ml = a.ml + (long)bh * a.parts * a.pitch;
    auto issue = [&](int s, int slot) {
        if (tid < STEP) {
            const int r = s * STEP + tid;
            float x = INFINITY;  // a row that is none gives nothing
            int q = -1;
            if (r < rows) {
                q = first + r / t.share;
                const int parts = ceil_div(q / WG_STEP + 1, a.steps);  // (those of the row alone: others hold nothing of it)
                float m = -INFINITY, l = 0.f;
                for (int i = 0; i < parts; i++) m = fmaxf(m, ml[i * a.pitch + r].x);
                for (int i = 0; i < parts; i++) {
                    const float2 v = ml[i * a.pitch + r];
                    l += v.x == -INFINITY ? 0.f : v.y * __builtin_amdgcn_exp2f(v.x - m);
                }
                x = m + __builtin_amdgcn_logf(l);
            }
            lse[slot][tid] = x;
            last[slot][tid] = q;
        }
#pragma unroll
        for (int j = 0; j < NL; j++) {
            const int i = row_w + RPL * j;
            const int r = imin(s * STEP + i, rows - 1);
            const int q = r / t.share;
            load_to_lds_x4(qb + (long)(r - q * t.share) * t.q_hs + (long)(first + q) * t.q_rs + 8 * (lchunk ^ k_swz<D>(i)),
                           lds0 + slot * TILE + wave * (NL * 1024) + j * 1024);
        }
    };
    if (begin < end) issue(begin, 0);
    int qread[NK];
#pragma unroll
    for (int s = 0; s < NK; s++) qread[s] = (32 * BLK * rg + ln) * ROW + (((2 * s + lc) ^ k_swz<D>(ln)) * 16);
#pragma unroll
    for (int s = 0; s < NK; s++) {
        u32x4_t x = bit_cast<u32x4_t>(kf[s]);
        asm volatile("" : "+v"(x));
        kf[s] = bit_cast<half8_t>(x);
    }
    float sum = 0.f;
    for (int s = begin; s < end; s++) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int slot = (s - begin) & 1;
        const uint8_t* l = lds + slot * TILE;
        if (s + 1 < end) issue(s + 1, 1 - slot);
        const bool masked = first + s * STEP / t.share < key0 + 32 * KG - 1;
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
            float part = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int r = 32 * (BLK * rg + i) + 8 * j + 4 * lc;
                const float4_t x = *(const float4_t*)&lse[slot][r];
                float p[4];
#pragma unroll
                for (int v = 0; v < 4; v++) p[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[4 * j + v], a.qk_scale, -x[v]));
                if (masked) {
#pragma unroll
                    for (int v = 0; v < 4; v++) p[v] = key <= last[slot][r + v] ? p[v] : 0.f;
                }
                part += (p[0] + p[1]) + (p[2] + p[3]);
            }
            sum += part;
        }
    }
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

constexpr int WG_WGS = 512;

WeighPlan plan(int B, int H, int share, int S, int window) {
    WeighPlan a = {};
    a.queries = window > 0 ? std::min(window, S) : S;
    a.pitch = (long)a.queries * share;
    a.tiles = (int)((a.pitch + WG_ROWS - 1) / WG_ROWS);
    const int steps = (S + WG_STEP - 1) / WG_STEP;
    a.steps = (int)std::max<long>(((long)B * H * a.tiles * steps + WG_WGS - 1) / WG_WGS, 1);
    if ((long)B * H * a.tiles >= WG_WGS) a.steps = steps;
    a.parts = (steps + a.steps - 1) / a.steps;
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
    auto pad8 = [](long n) { return dim3((unsigned)((n + 7) / 8 * 8)); };
    const dim3 rows = pad8((long)t.B * t.H * a.tiles * a.parts);
    const long wide = (long)t.B * t.H * ((t.S + 127) / 128);
    const bool narrow = wide < WG_WGS;
    const dim3 keys = pad8(narrow ? (long)t.B * t.H * ((t.S + 31) / 32) : wide);
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
