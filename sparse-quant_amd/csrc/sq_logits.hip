// Rules on a row of logits, and its best token:
//   x > 0 ? x / r : x r     where the token stands in the row's text (r: repetition)
//   x - f c, then x - p     where it stands c > 0 times in the generated part of it (f: frequency, p: presence)
//   x + b                   where it has a bias (the last entry of those that name it)
//   -inf                    where its bit in the mask is 0
// each step rounded once in fp32, the result once more to the logits' type; the best token is that of the results.
//
// A row is cut into slices, a workgroup each.  What the rules ask of a slice's tokens is counted in LDS, in whole numbers, so that
// the order of the atomics does not matter; whoever touches a token first puts it on a list.  Then the logits, which were
// requested in front of all that, go through registers once, masked, with the listed tokens as they are, and behind that the
// list is worked off, one token a lane.  Every slice looks through the row's whole text for its tokens (from L2), so that with
// many rows the slices are wide.  A second launch joins the slices' best tokens.
//
// What bounds it: few rows the host (a call of two launches from Python takes 9 us; they take 5); many rows, the text and what hangs on
// it: 200 rows of 131077 fp32 logits, 210 MB, take 41 us where nothing is asked (the copy's rate), 11 more with a mask, 17 more
// with a text of 5000 tokens, which each of 17 slices looks through, 5 to 9 with biases, 77 with all.
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

// (From -inf and no token on: -inf is better than none, a NaN never is.)
__device__ __forceinline__ void better(float v, int i, float& best, int& arg) {
    if (v > best || (v == best && i < arg)) best = v, arg = i;
}
__device__ __forceinline__ void wave_best(float& best, int& arg) {
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        const float ob = __shfl_xor(best, x);
        const int oa = __shfl_xor(arg, x);
        better(ob, oa, best, arg);
    }
}
// ... of a workgroup, in its first lane.
template <int THREADS>
__device__ __forceinline__ void group_best(float& best, int& arg) {
    __shared__ float wbest[THREADS / 64];
    __shared__ int warg[THREADS / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
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
    }
}

// A row: its memory, what it is penalised with, and the part of its text that counts.
template <typename T>
struct Row {
    static constexpr int VEC = 16 / sizeof(T);
    typedef T vec_t __attribute__((ext_vector_type(VEC)));
    const T* x;
    T* y;
    int shift;  // elements of the row's first 16 bytes that lie in front of it: pieces begin where memory is aligned
    bool aligned, penalties;
    float r, f, p;
    const long long* ids;
    int n;
    long long from;
    const unsigned* mask;
    const float* bias;

    __device__ __forceinline__ Row(const LogitRules& t, int m) {
        x = (const T*)t.x + (long)m * t.x_rs;
        y = (T*)t.y + (long)m * t.y_rs;
        shift = (int)(((uintptr_t)x / sizeof(T)) % VEC);
        aligned = ((uintptr_t)y / sizeof(T)) % VEC == shift;
        penalties = t.repetition || t.presence || t.frequency;
        r = t.repetition ? t.repetition[m] : 1.f;
        f = t.frequency ? t.frequency[m] : 0.f;
        p = t.presence ? t.presence[m] : 0.f;
        const long long len = t.lengths ? t.lengths[m * t.len_s] : t.L;
        n = !penalties || len < 0 ? 0 : len > t.L ? t.L : (int)len;
        from = t.generated ? t.generated[m * t.gen_s] : 0;
        ids = t.ids + (long)m * t.id_rs;
        mask = t.mask ? t.mask + (long)m * t.mask_rs : nullptr;
        bias = t.bias + (long)m * t.b_rs;
    }
    __device__ __forceinline__ vec_t load(int e, int V) const {
        vec_t v;
        if (e >= 0 && e + VEC <= V) v = *(const vec_t*)(x + e);
        else
#pragma unroll
            for (int k = 0; k < VEC; k++) v[k] = e + k >= 0 && e + k < V ? x[e + k] : (T)0.f;
        return v;
    }
    __device__ __forceinline__ void store(int e, int V, vec_t o) const {
        if (aligned && e >= 0 && e + VEC <= V) *(vec_t*)(y + e) = o;
        else
#pragma unroll
            for (int k = 0; k < VEC; k++)
                if (e + k >= 0 && e + k < V) y[e + k] = o[k];
    }
    // Bit k: whether token e + k may be chosen.
    __device__ __forceinline__ unsigned allowed(int e, int V) const {
        if (!mask || e >= V) return ~0u;
        const int e0 = e < 0 ? 0 : e, last = (V - 1) >> 5;
        const unsigned lo = mask[e0 >> 5], hi = mask[imin((e0 >> 5) + 1, last)];
        return (unsigned)((((unsigned long long)hi << 32) | lo) >> (e0 & 31)) << (e0 - e);
    }
    // A vector of logits under the mask, those that are marked as they are.
    template <class Marked>
    __device__ __forceinline__ void pass(int e, int V, vec_t v, unsigned bits, Marked marked, float& best, int& arg) const {
        vec_t o;
#pragma unroll
        for (int k = 0; k < VEC; k++) {
            const bool listed = marked(k);
            o[k] = ((bits >> k) & 1u) || listed ? v[k] : (T)-INFINITY;
            if (!listed && e + k >= 0 && e + k < V) better((float)o[k], e + k, best, arg);
        }
        store(e, V, o);
    }
    // A listed token: in the text or not, `made` times in its generated part, with entry j of the biases (from 1; 0: none).
    __device__ __forceinline__ void finish(const LogitRules& t, int e, bool text, unsigned made, unsigned j, float& best, int& arg) const {
#pragma clang fp contract(off)
        float s = (float)x[e];
        if (text || made) {
            if (t.repetition) s = s > 0.f ? s / r : s * r;
            if (made) {
                if (t.frequency) s = s - f * (float)made;
                if (t.presence) s = s - p;
            }
        }
        if (j) s = s + bias[j - 1];
        if (mask && !((mask[e >> 5] >> (e & 31)) & 1u)) s = -INFINITY;
        const T o = (T)s;
        y[e] = o;
        better((float)o, e, best, arg);
    }
};

// ---- a slice of W tokens by one workgroup

// A token's word: from the top one bit, it stands in the text in front of the generated part; the last of the row's biases that
// names it, counted from 1; in the lower half, how often it stands in the generated part.
template <typename T, typename Word, int W, int THREADS>
__global__ __launch_bounds__(THREADS) void logit_slice_kernel(LogitArgs a) {
    constexpr int VEC = Row<T>::VEC, VECS = W / (THREADS * VEC), HALF = 4 * sizeof(Word);
    constexpr Word TEXT = (Word)1 << (2 * HALF - 1);
    __shared__ __attribute__((aligned(16))) Word words[W];
    __shared__ unsigned short list[W];
    __shared__ unsigned listed;
    const LogitRules& t = a.t;
    const int tid = threadIdx.x, m = blockIdx.y;
    const Row<T> row(t, m);
    const int base = blockIdx.x * W - row.shift;
    typename Row<T>::vec_t v[VECS];
    unsigned allowed[VECS];
#pragma unroll
    for (int u = 0; u < VECS; u++) {  // on their way while the text is looked through
        const int e = base + (u * THREADS + tid) * VEC;
        v[u] = row.load(e, t.V);
        allowed[u] = row.allowed(e, t.V);
    }
    // The first tokens of the text as well (a lane's eight), and its first bias.
    constexpr int AHEAD = 8;
    const int* const bias_ids = t.bias_ids + (long)m * t.bid_rs;
    long long id[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; u++) id[u] = tid + u * THREADS < row.n ? row.ids[(long)(tid + u * THREADS) * t.id_ps] : -1;
    int named = tid < t.nb ? bias_ids[tid] : -1;
    const bool marks = row.n > 0 || t.nb > 0;
    auto enlist = [&](int at, Word was) {
        if (was == 0) list[atomicAdd(&listed, 1u)] = (unsigned short)at;
    };
    if (marks) {
        if (tid == 0) listed = 0;
        for (int i = tid * (int)(16 / sizeof(Word)); i < W; i += THREADS * (int)(16 / sizeof(Word)))
            *(u32x4_t*)&words[i] = (u32x4_t){0u, 0u, 0u, 0u};
        __syncthreads();
    }
    auto place = [&](long long id) { return id >= 0 && id < t.V && id >= base && id < base + W ? (int)(id - base) : -1; };
    if (t.nb > 0) {
        for (int i = tid; i < t.nb; i += THREADS) {
            const int at = place(named);
            if (at >= 0) enlist(at, atomicMax(&words[at], (Word)(i + 1) << HALF));
            named = i + THREADS < t.nb ? bias_ids[i + THREADS] : -1;
        }
        __syncthreads();
    }
    if (row.n > 0) {
        for (int i0 = tid; i0 < row.n; i0 += AHEAD * THREADS) {
            if (i0 != tid) {
#pragma unroll
                for (int u = 0; u < AHEAD; u++) id[u] = i0 + u * THREADS < row.n ? row.ids[(long)(i0 + u * THREADS) * t.id_ps] : -1;
            }
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                const int at = place(id[u]);
                if (at < 0) continue;
                enlist(at, i0 + u * THREADS >= row.from ? atomicAdd(&words[at], (Word)1) : atomicOr(&words[at], TEXT));
            }
        }
        __syncthreads();
    }
    float best = -INFINITY;
    int arg = 0x7fffffff;
#pragma unroll
    for (int u = 0; u < VECS; u++) {
        const int i = (u * THREADS + tid) * VEC, e = base + i;
        if (e >= t.V) break;
        row.pass(e, t.V, v[u], allowed[u], [&](int k) { return marks && words[i + k] != 0; }, best, arg);
    }
    if (marks) {
        __syncthreads();  // (a vector's store lies in front of its listed tokens' own)
        for (unsigned i = tid; i < listed; i += THREADS) {
            const Word w = words[list[i]];
            const unsigned made = (unsigned)(w & (((Word)1 << HALF) - 1)), j = (unsigned)((w & ~TEXT) >> HALF);
            row.finish(t, base + list[i], (w & TEXT) != 0, made, j, best, arg);
        }
    }
    group_best<THREADS>(best, arg);
    if (tid == 0) {
        a.best[(long)m * a.slices + blockIdx.x] = best;
        a.arg[(long)m * a.slices + blockIdx.x] = arg;
    }
}

__global__ __launch_bounds__(64) void logit_token_kernel(LogitArgs a) {
    const int lane = threadIdx.x, m = blockIdx.x;
    float best = -INFINITY;
    int arg = 0x7fffffff;
    for (int i = lane; i < a.slices; i += 64) better(a.best[(long)m * a.slices + i], a.arg[(long)m * a.slices + i], best, arg);
    wave_best(best, arg);
    if (lane == 0) a.t.token[m] = arg == 0x7fffffff ? 0 : arg;
}

// Slices: wide ones look through the text less often, narrow ones fill the chip (200 rows of 131072 fp32 logits with all rules, us: 76
// with 8192 tokens by 512 threads, 78 with 4096 by 256, 91 with 4096 by 512 and with 2048 by 256; 4 rows 13.6 with the widest
// and 13.1 with the narrowest, 16 rows 16.1 and 16.9, 32 rows 19.5 and 23.1).
constexpr int NARROW = 2048, WIDE = 8192, LONG = 4096;
// Words of 32 bits count 65535 of a token; longer texts take 64 and half the width.
bool long_text(int L, int nb) { return L > 0xffff || nb > 0x7ffe; }
bool narrow(int M, int V) { return (long)M * ((V + NARROW - 1) / NARROW) <= 1024; }
int slices_of(int M, int V, int L, int nb) {  // (7 more than the tokens: a row may begin inside 16 bytes)
    const int w = long_text(L, nb) ? LONG : narrow(M, V) ? NARROW : WIDE;
    return (V + 7 + w - 1) / w;
}

}  // namespace

size_t logit_rules_workspace_bytes(int M, int V, int L, int nb) {
    return (size_t)M * slices_of(M, V, L, nb) * 8;
}

hipError_t launch_logit_rules(const LogitRules& t, int elem_bytes, void* workspace, hipStream_t st) {
    LogitArgs a;
    a.t = t;
    a.slices = slices_of(t.M, t.V, t.L, t.nb);
    a.best = (float*)workspace;
    a.arg = (int*)(a.best + (size_t)t.M * a.slices);
    const dim3 grid(a.slices, t.M);
#define SQ_LOGITS(WORD_, W_, THREADS_)                                                                                        \
    if (elem_bytes == 2) hipLaunchKernelGGL((logit_slice_kernel<half_t, WORD_, W_, THREADS_>), grid, dim3(THREADS_), 0, st, a); \
    else hipLaunchKernelGGL((logit_slice_kernel<float, WORD_, W_, THREADS_>), grid, dim3(THREADS_), 0, st, a)
    if (long_text(t.L, t.nb)) {
        SQ_LOGITS(unsigned long long, LONG, 512);
    } else if (narrow(t.M, t.V)) {
        SQ_LOGITS(unsigned, NARROW, 256);
    } else {
        SQ_LOGITS(unsigned, WIDE, 512);
    }
#undef SQ_LOGITS
    hipLaunchKernelGGL(logit_token_kernel, dim3(t.M), dim3(64), 0, st, a);
    return hipGetLastError();
}

}  // namespace sq
