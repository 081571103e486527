// Rules on a row of logits, and its best token:
//   x > 0 ? x / r : x r     where the token stands in the row's text (r: repetition)
//   x - f c - p             where it stands c > 0 times in the generated part of it (f: frequency, p: presence)
//   x + b                   where it has a bias (the last entry of those that name it)
//   -inf                    where its bit in the mask is 0
// each step rounded once in fp32, the result once more to the logits' type.
#include "sq_common.h"
#include "sq_kernels.h"

#include <algorithm>

namespace sq {

namespace {

struct LogitArgs {
    LogitRules t;
    float* best;  // [M][slices]
    int* arg;
    int slices;
};

__device__ __forceinline__ void wave_best(float& best, int& arg) {
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        const float ob = __shfl_xor(best, x);
        const int oa = __shfl_xor(arg, x);
        if (ob > best || (ob == best && oa < arg)) best = ob, arg = oa;
    }
}

// A workgroup has W tokens of a row: it counts those of the text that fall on them in LDS, and goes through their logits.
template <typename T, int W, int THREADS>
__global__ __launch_bounds__(THREADS) void logit_rules_kernel(LogitArgs a) {
    constexpr int VEC = 16 / sizeof(T);
    typedef T vec_t __attribute__((ext_vector_type(VEC)));
    __shared__ unsigned count[W];          // of the generated part; the top bit: stands in the text before it
    __shared__ unsigned short entry[W];    // 1 + the last of the row's biases that names the token
    __shared__ float wbest[THREADS / 64];
    __shared__ int warg[THREADS / 64];
    const LogitRules& t = a.t;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int m = blockIdx.y;
    const T* const x = (const T*)t.x + (long)m * t.x_rs;
    T* const y = (T*)t.y + (long)m * t.y_rs;
    // slices begin where the row's memory is aligned to 16 bytes
    const int shift = (int)(((uintptr_t)x / sizeof(T)) % VEC);
    const bool aligned = ((uintptr_t)y / sizeof(T)) % VEC == shift;
    const int base = blockIdx.x * W - shift;
    const bool penalties = t.repetition || t.presence || t.frequency;

    if (penalties)
        for (int i = tid; i < W; i += THREADS) count[i] = 0u;
    if (t.nb)
        for (int i = tid; i < W; i += THREADS) entry[i] = 0;
    __syncthreads();
    float r = 1.f, f = 0.f, p = 0.f;
    if (penalties) {
        if (t.repetition) r = t.repetition[m];
        if (t.frequency) f = t.frequency[m];
        if (t.presence) p = t.presence[m];
        const long long len = t.lengths ? t.lengths[m * t.len_s] : t.L;
        const long long from = t.generated ? t.generated[m * t.gen_s] : 0;
        const int n = len < 0 ? 0 : len > t.L ? t.L : (int)len;
        const long long* ids = t.ids + (long)m * t.id_rs;
        for (int i = tid; i < n; i += THREADS) {
            const long long id = ids[(long)i * t.id_ps];
            const long long at = id - base;
            if (id >= 0 && id < t.V && at >= 0 && at < W) {
                if (i >= from) atomicAdd(&count[at], 1u);
                else atomicOr(&count[at], 0x80000000u);
            }
        }
    }
    if (t.nb) {
        const int* ids = t.bias_ids + (long)m * t.bid_rs;
        // (the entries are set in their order: a later one that names the same token waits for the pass it is in)
        for (int i0 = 0; i0 < t.nb; i0 += THREADS) {
            const int i = i0 + tid;
            int at = -1;
            if (i < t.nb) {
                const int id = ids[i];
                if (id >= 0 && id < t.V && id - base >= 0 && id - base < W) at = id - base;
            }
            bool todo = at >= 0;
            while (__syncthreads_or(todo)) {
                if (todo) entry[at] = (unsigned short)(i + 1);
                __syncthreads();
                todo = todo && entry[at] < i + 1;
                __syncthreads();
            }
        }
    }
    __syncthreads();

    const unsigned* const mask = t.mask ? t.mask + (long)m * t.mask_rs : nullptr;
    const int words = (t.V + 31) >> 5;
    float best = -INFINITY;
    int arg = 0x7fffffff;
    for (int i = tid * VEC; i < W; i += THREADS * VEC) {
        const int e = base + i;
        if (e >= t.V) break;
        const bool whole = e >= 0 && e + VEC <= t.V;
        vec_t v;
        if (whole) v = *(const vec_t*)(x + e);
        else
#pragma unroll
            for (int k = 0; k < VEC; k++) v[k] = e + k >= 0 && e + k < t.V ? x[e + k] : (T)0.f;
        unsigned allowed = ~0u;
        if (mask) {
            const int e0 = e < 0 ? 0 : e;
            const unsigned lo = mask[e0 >> 5], hi = mask[imin((e0 >> 5) + 1, words - 1)];
            allowed = (unsigned)((((unsigned long long)hi << 32) | lo) >> (e0 & 31)) << (e0 - e);
        }
        vec_t o;
#pragma unroll
        for (int k = 0; k < VEC; k++) {
#pragma clang fp contract(off)
            float s = (float)v[k];
            if (penalties) {
                const unsigned c = count[i + k];
                if (c) {
                    if (t.repetition) s = s > 0.f ? s / r : s * r;
                    const unsigned g = c & 0x7fffffffu;
                    if (g) {
                        if (t.frequency) s = s - f * (float)g;
                        if (t.presence) s = s - p;
                    }
                }
            }
            if (t.nb) {
                const int j = entry[i + k];
                if (j) s = s + t.bias[(long)m * t.b_rs + j - 1];
            }
            if (!((allowed >> k) & 1u)) s = -INFINITY;
            o[k] = (T)s;
            if (e + k >= 0 && e + k < t.V) {
                const float w = (float)o[k];
                if (w > best || (w == best && e + k < arg)) best = w, arg = e + k;
            }
        }
        if (whole && aligned) *(vec_t*)(y + e) = o;
        else
#pragma unroll
            for (int k = 0; k < VEC; k++)
                if (e + k >= 0 && e + k < t.V) y[e + k] = o[k];
    }
    wave_best(best, arg);
    if (lane == 0) {
        wbest[wave] = best;
        warg[wave] = arg;
    }
    __syncthreads();
    if (wave == 0) {
        best = lane < THREADS / 64 ? wbest[lane] : -INFINITY;
        arg = lane < THREADS / 64 ? warg[lane] : 0x7fffffff;
        wave_best(best, arg);
        if (lane == 0) {
            a.best[(long)m * a.slices + blockIdx.x] = best;
            a.arg[(long)m * a.slices + blockIdx.x] = arg;
        }
    }
}

__global__ __launch_bounds__(64) void logit_token_kernel(LogitArgs a) {
    const int lane = threadIdx.x;
    const int m = blockIdx.x;
    float best = -INFINITY;
    int arg = 0x7fffffff;
    for (int i = lane; i < a.slices; i += 64) {
        const float v = a.best[(long)m * a.slices + i];
        const int k = a.arg[(long)m * a.slices + i];
        if (v > best || (v == best && k < arg)) best = v, arg = k;
    }
    wave_best(best, arg);
    if (lane == 0) a.t.token[m] = arg == 0x7fffffff ? 0 : arg;
}

constexpr int NARROW = 2048, WIDE = 8192;
bool narrow(int M, int V) { return (long)M * ((V + NARROW - 1) / NARROW) <= 1024; }
int slices_of(int M, int V) {  // (one more than the tokens need: a row may begin inside 16 bytes)
    const int w = narrow(M, V) ? NARROW : WIDE;
    return (V + 7 + w - 1) / w;
}

}  // namespace

size_t logit_rules_workspace_bytes(int M, int V) { return (size_t)M * slices_of(M, V) * 8; }

hipError_t launch_logit_rules(const LogitRules& t, int elem_bytes, void* workspace, hipStream_t st) {
    LogitArgs a;
    a.t = t;
    a.slices = slices_of(t.M, t.V);
    a.best = (float*)workspace;
    a.arg = (int*)(a.best + (size_t)t.M * a.slices);
    const dim3 grid(a.slices, t.M);
    if (narrow(t.M, t.V)) {
        if (elem_bytes == 2) hipLaunchKernelGGL((logit_rules_kernel<half_t, NARROW, 256>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((logit_rules_kernel<float, NARROW, 256>), grid, dim3(256), 0, st, a);
    } else {
        if (elem_bytes == 2) hipLaunchKernelGGL((logit_rules_kernel<half_t, WIDE, 512>), grid, dim3(512), 0, st, a);
        else hipLaunchKernelGGL((logit_rules_kernel<float, WIDE, 512>), grid, dim3(512), 0, st, a);
    }
    hipLaunchKernelGGL(logit_token_kernel, dim3(t.M), dim3(64), 0, st, a);
    return hipGetLastError();
}

}  // namespace sq
