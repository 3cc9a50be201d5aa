// Sampling over rows of the vocabulary for gfx950 (CDNA4): the code object
// cima_sample.hsaco.  Softmax of rows of logits at a temperature, log probabilities
// of given tokens with the rows' entropy and likeliest alternatives, and the
// verification of drafted tokens.
#include "gguf_formats.h"

// ------------------------------------------------------------------ softmax
//
// A row's logits are read into registers: the maximum first, then the sum of
// e^((f(x) - m) / T) = 2^((f(x) - m) log2(e) / T), then the same again times 1 /
// sum.  Rows up to 65536 logits go to a workgroup each, in one launch.  Longer
// ones, and few long ones, are split over `parts` workgroups of 8192 logits, or
// of 2048 where those are at most four to a CU: the first launch leaves each
// part's maximum, its place and its sum, the second joins a row's parts, reads
// its own logits once more and writes the probabilities.
// Bound by memory: the probabilities go past the caches, which keep the logits
// for the second reading.  Measured on MI355X, us: 384 rows of 128256 f16 61
// (393 MB moved, 6.5 TB/s; through the caches 83, a row per workgroup in 32
// words a thread 73); 256 rows of 60000 in one launch 20.6, in two 22.5; 64 of
// 30000 6.9 and 8.6.  Parts of 2048 / 8192: one row of 151936 6.2 / 7.5, capped 3
// of 40000 8.0 / 14.8, eight of 151936 7.7 / 8.2; 384 of 128256 72 / 62.

struct SmPart {
    float m, l;
    int at, pad;
};

// V logits from element i on, those behind n as -inf: a lane's word.  Four, so
// that the probabilities of a wave are written contiguously; eight of f16 where
// nothing is written.
template <bool F32, int V>
DEV void sm_load(const void* __restrict__ x, size_t row, int i, int n, uint32_t (&v)[F32 ? V : V / 2]) {
    if (i + V <= n) {
        if constexpr (F32) __builtin_memcpy(v, __builtin_assume_aligned((const float*)x + row + i, 4), 4 * V);
        else __builtin_memcpy(v, __builtin_assume_aligned((const uint16_t*)x + row + i, 2), 2 * V);
    } else if constexpr (F32) {
#pragma unroll
        for (int j = 0; j < V; j++) v[j] = i + j < n ? ((const uint32_t*)x)[row + i + j] : 0xff800000u;
    } else {
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            const uint32_t a = i + j < n ? ((const uint16_t*)x)[row + i + j] : 0xfc00u;
            const uint32_t b = i + j + 1 < n ? ((const uint16_t*)x)[row + i + j + 1] : 0xfc00u;
            v[j / 2] = a | b << 16;
        }
    }
}
template <bool F32, int V>
DEV float sm_get(const uint32_t (&v)[F32 ? V : V / 2], int j) {
    if constexpr (F32) {
        const uint32_t a = v[j];
        return __builtin_bit_cast(float, a);
    } else {
        return h2f(j & 1 ? v[j / 2] >> 16 : v[j / 2] & 0xffffu);
    }
}
DEV float uniform(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}
// c / T within fp32's range, so that no difference of logits becomes 0 * inf at a
// temperature that is infinite or next to nothing
DEV float sm_scale(float c, float T) { return fminf(fmaxf(c / T, 1e-37f), 1e38f); }
// f of a logit, cap * tanh(x / cap).  Infinite ones stay as they are: -inf is a
// token that may not be taken (or no logit, behind n), and -cap would give it a
// share.
DEV float sm_f(float x, float cap) { return __builtin_isinf(x) ? x : cap * tanhf(x / cap); }

// a logit of a pair less c: of f16 logits as x * 1 - c, one instruction with the
// conversion, the same number
DEV float mix_less(uint32_t pair, bool high, float c) {
    float d;
    if (high)
        __asm__("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(pair), "v"(c));
    else
        __asm__("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel_hi:[1,0,0]" : "=v"(d) : "v"(pair), "v"(c));
    return d;
}

// R words of V logits a thread of a row by NT threads: the maximum, the first place of it
// (T <= 0) or the sum (T > 0).  CAP: f is applied when the logits are loaded,
// which are fp32 from there on.
template <bool F32, bool CAP, int NT, int R, int V = 4>
struct SmRow {
    static constexpr bool W32 = F32 || CAP;
    uint32_t v[R][W32 ? V : V / 2];
    int base;
    float m, l;
    int at;

    DEV float get(int r, int j) const { return sm_get<W32, V>(v[r], j); }
    DEV float less(int r, int j, float c) const {
        if constexpr (W32) return get(r, j) - c;
        else return mix_less(v[r][j / 2], j & 1, c);
    }
    // keeps the compiler from holding all logits as fp32 from one pass to the next
    DEV void fresh() {
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int k = 0; k < (W32 ? V : V / 2); k++) __asm__ volatile("" : "+v"(v[r][k]));
    }
    DEV void load(const void* __restrict__ x, size_t row, int first, int n, float cap) {
        base = first + threadIdx.x * V;
#pragma unroll
        for (int r = 0; r < R; r++) {
            if constexpr (CAP) {
                uint32_t w[F32 ? V : V / 2];
                sm_load<F32, V>(x, row, base + r * NT * V, n, w);
#pragma unroll
                for (int j = 0; j < V; j++) v[r][j] = __builtin_bit_cast(uint32_t, sm_f(sm_get<F32, V>(w, j), cap));
            } else {
                sm_load<F32, V>(x, row, base + r * NT * V, n, v[r]);
            }
        }
    }
    DEV void stats(float T) {
        __shared__ float red[2][NT / 64];
        __shared__ int place[NT / 64];
        const int w = threadIdx.x >> 6;
        m = -INFINITY;
        if constexpr (W32) {
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int j = 0; j < V; j++) m = fmaxf(m, get(r, j));
        } else {  // two f16 at a time, exact
            typedef _Float16 hp __attribute__((ext_vector_type(2)));
            hp h = {(_Float16)-INFINITY, (_Float16)-INFINITY};
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int k = 0; k < V / 2; k++) h = __builtin_elementwise_max(h, __builtin_bit_cast(hp, v[r][k]));
            m = fmaxf((float)h[0], (float)h[1]);
        }
        m = wave_max_u(m);
        if ((threadIdx.x & 63) == 0) red[0][w] = m;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NT / 64; k++) m = fmaxf(m, red[0][k]);
        fresh();
        l = 0.f;
        at = 0x7fffffff;
        if (T > 0.f) {
            const float c = m == -INFINITY ? 0.f : m, s = sm_scale(1.44269504088896340736f, T);
#pragma unroll
            for (int r = 0; r < R; r++) {
                float p = 0.f;
#pragma unroll
                for (int j = 0; j < V; j++) p += __builtin_amdgcn_exp2f(less(r, j, c) * s);
                l += p;
            }
            l = wave_sum_u(l);
            if ((threadIdx.x & 63) == 0) red[1][w] = l;
        } else {
            // behind a row or part of -inf alone there is no place to find
#pragma unroll
            for (int r = R - 1; r >= 0; r--)
#pragma unroll
                for (int j = V - 1; j >= 0; j--)
                    if (get(r, j) == m && m != -INFINITY) at = base + r * NT * V + j;
#pragma unroll
            for (int o = 32; o; o >>= 1) at = min(at, __shfl_xor(at, o));
            if ((threadIdx.x & 63) == 0) place[w] = at;
        }
        __syncthreads();
        if (T > 0.f) {
            l = 0.f;
#pragma unroll
            for (int k = 0; k < NT / 64; k++) l += red[1][k];
        } else {
#pragma unroll
            for (int k = 0; k < NT / 64; k++) at = min(at, place[k]);
        }
        // the same in every lane: out of the vector registers, which the row fills
        m = uniform(m), l = uniform(l);
        at = __builtin_amdgcn_readfirstlane(at);
        fresh();
    }
    // the probabilities of a row of maximum M at place A and sum L, by the square
    // of the half exponent's power: the exponential itself would flush results
    // below 2^-126
    DEV void write(float* __restrict__ y, size_t row, int n, float T, float M, int A, float L) const {
        static_assert(V == 4, "a 16-byte store a word");
        const bool none = M == -INFINITY && L == 0.f;  // -inf alone
        const float c = M == -INFINITY ? 0.f : M, inv = none ? 0.f : 1.f / L;
        const float s = sm_scale(0.72134752044448170368f, T);
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int i = base + r * NT * V;
            float p[4];
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float h = __builtin_amdgcn_exp2f(less(r, j, c) * s);
                p[j] = T > 0.f ? h * (h * inv) : (i + j == A ? 1.f : 0.f);
            }
            float* o = y + row + i;
            if (i + 4 <= n) {
                typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
                __builtin_nontemporal_store((f4u){p[0], p[1], p[2], p[3]}, (f4u*)o);
            } else {
#pragma unroll
                for (int j = 0; j < V; j++)
                    if (i + j < n) o[j] = p[j];
            }
            __builtin_amdgcn_sched_barrier(0);  // a word at a time: the row fills the registers
        }
    }
};

constexpr int SM_T = 256;  // threads of a part, of R words a thread

// a row's parts joined by every wave: lane i takes parts i, i + 64, ...
DEV float sm_join(const SmPart* __restrict__ p, int parts, float T, int* at, float* L) {
    const int lane = threadIdx.x & 63;
    float m = -INFINITY, l = 0.f;
    for (int i = lane; i < parts; i += 64) m = fmaxf(m, p[i].m);
    m = wave_max_u(m);
    int a = 0x7fffffff;
    if (T > 0.f) {
        const float c = m == -INFINITY ? 0.f : m, s = sm_scale(1.44269504088896340736f, T);
        for (int i = lane; i < parts; i += 64)
            l += p[i].l * (p[i].m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((p[i].m - c) * s));
    } else {
        // the first of the parts that have the maximum has its first place
        for (int i = lane; i < parts; i += 64)
            if (p[i].m == m) a = min(a, p[i].at);
#pragma unroll
        for (int o = 32; o; o >>= 1) a = min(a, __shfl_xor(a, o));
    }
    *L = wave_sum_u(l);
    *at = a;
    return m;
}
#define SOFTMAX_PARTS(NAME, F32, CAP, R)                                                                               \
    extern "C" __global__ __launch_bounds__(SM_T) void cima_softmax_stats_w##R##_##NAME(                               \
        const void* __restrict__ x, SmPart* __restrict__ part, int n, const float* __restrict__ temp,                  \
        int rows_per_temp, float cap, int parts) {                                                                     \
        const int row = blockIdx.x / parts, pt = blockIdx.x % parts;                                                   \
        SmRow<F32, CAP, SM_T, F32 ? R : R / 2, F32 ? 4 : 8> S;                                                         \
        S.load(x, (size_t)row * n, pt * SM_T * R * 4, n, cap);                                                         \
        S.stats(temp ? temp[row / rows_per_temp] : 1.f);                                                               \
        if (threadIdx.x == 0) part[blockIdx.x] = SmPart{S.m, S.l, S.at, 0};                                            \
    }                                                                                                                  \
    extern "C" __global__ __launch_bounds__(SM_T) void cima_softmax_probs_w##R##_##NAME(                               \
        const void* __restrict__ x, float* __restrict__ y, const SmPart* __restrict__ part, int n,                     \
        const float* __restrict__ temp, int rows_per_temp, float cap, int parts) {                                     \
        const int row = blockIdx.x / parts, pt = blockIdx.x % parts;                                                   \
        const float T = temp ? temp[row / rows_per_temp] : 1.f;                                                        \
        SmRow<F32, CAP, SM_T, R> S;                                                                                    \
        S.load(x, (size_t)row * n, pt * SM_T * R * 4, n, cap);                                                         \
        float L;                                                                                                       \
        int at;                                                                                                        \
        const float m = sm_join(part + (size_t)row * parts, parts, T, &at, &L);                                        \
        S.write(y, (size_t)row * n, n, T, m, at, L);                                                                   \
    }
#define SOFTMAX_WHOLE(NAME, F32, CAP, NT, WORDS)                                                                       \
    extern "C" __global__ __launch_bounds__(NT) void cima_softmax_t##NT##_w##WORDS##_##NAME(                           \
        const void* __restrict__ x, float* __restrict__ y, int n, const float* __restrict__ temp, int rows_per_temp,   \
        float cap) {                                                                                                   \
        const int row = blockIdx.x;                                                                                    \
        const float T = temp ? temp[row / rows_per_temp] : 1.f;                                                        \
        SmRow<F32, CAP, NT, WORDS> R;                                                                                  \
        R.load(x, (size_t)row * n, 0, n, cap);                                                                         \
        R.stats(T);                                                                                                    \
        R.write(y, (size_t)row * n, n, T, R.m, R.at, R.l);                                                             \
    }
#define SOFTMAX(NAME, F32, CAP)            \
    SOFTMAX_PARTS(NAME, F32, CAP, 2)       \
    SOFTMAX_PARTS(NAME, F32, CAP, 8)       \
    SOFTMAX_WHOLE(NAME, F32, CAP, 256, 2)  \
    SOFTMAX_WHOLE(NAME, F32, CAP, 256, 8)  \
    SOFTMAX_WHOLE(NAME, F32, CAP, 1024, 8)
SOFTMAX(f16, false, false)
SOFTMAX(f32, true, false)
SOFTMAX(cap_f16, false, true)
SOFTMAX(cap_f32, true, true)
SOFTMAX_WHOLE(f16, false, false, 1024, 16)
SOFTMAX_WHOLE(f32, true, false, 1024, 16)

// v of the lane that a DPP pattern names, 0 where there is none
template <int CTRL, int ROWS>
DEV double dpp_d(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)u, CTRL, ROWS, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// inclusive running sum over the wave: within rows of 16, then from row to row
DEV double wave_scan_d(double v) {
    v += dpp_d<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
    v += dpp_d<0x112, 0xf>(v);
    v += dpp_d<0x114, 0xf>(v);
    v += dpp_d<0x118, 0xf>(v);
    v += dpp_d<0x142, 0xa>(v);  // row_bcast:15 into rows 1, 3
    v += dpp_d<0x143, 0xc>(v);  // row_bcast:31 into rows 2, 3
    return v;
}
DEV double lane_d(double v, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)u, lane), hi = __builtin_amdgcn_readlane((uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// ------------------------------------------------------- log probabilities
//
// With z = (f(x) - m) / T and L = sum e^z over a row: a token's log probability is z -
// ln L, the row's entropy ln L - sum e^z z / L.  One reading: a part's logits stay in
// registers, first their largest, then the two sums.  The likeliest n_top of a part
// are found from the threads' largest: each wave takes the n_top-th largest of its
// lanes', which bounds the row's n_top-th from below, and the highest of these bounds
// leaves the few logits that are looked at one by one, ranked by counting (value
// first, then the lower id).  A second launch joins rows of several parts.  Parts
// as in the softmax above; sums of parts are joined in fp64.
constexpr int LP_TOP = 32;    // most alternatives
constexpr int LP_LIST = 1024;  // logits looked at one by one

struct LpArgs {
    const void* x;
    const int* tokens;
    float* logprob;
    float* entropy;
    int* top_ids;
    float* top_logprobs;
    const float* temp;
    float4* stats;                // [rows][parts]: m, l, sum of e^z z in log2's unit
    unsigned long long* keys;     // [rows][parts][kept]
    int n, n_top, kept, rows_per_temp, parts;  // kept: keys of a part, n_top or 1
    float cap;
};

// logits in order as whole numbers; -0 as 0
DEV uint32_t lp_order(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.f);
    return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
DEV float lp_value(unsigned long long key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __builtin_bit_cast(float, u ^ (u >> 31 ? 0x80000000u : 0xffffffffu));
}
constexpr uint32_t LP_NONE = 0x007fffffu;  // of -inf: a token that may not be taken
DEV unsigned long long lp_key(uint32_t order, int at) { return (unsigned long long)order << 32 | (uint32_t)~at; }
DEV int lp_id(unsigned long long key) { return (int)~(uint32_t)key; }

DEV unsigned long long wave_max_key(unsigned long long v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        const unsigned long long w = __shfl_xor(v, o);
        v = w > v ? w : v;
    }
    return v;
}
template <int NT>
struct LpTop {  // shared between the threads of a workgroup
    unsigned long long list[LP_LIST], top[LP_TOP], best[NT / 64];
    int count;
};
// the `kept` largest of the listed keys to S.top in order, zeros behind them;
// each(f) calls f with every key of this thread, for lists that are too short
template <int NT, typename E>
DEV void lp_rank(LpTop<NT>& S, int kept, E each) {
    __syncthreads();
    const int count = S.count;
    if (count <= 64) {  // a lane each: no loads from list to list
        if (threadIdx.x < 64) {
            const unsigned long long k = (int)threadIdx.x < count ? S.list[threadIdx.x] : 0;
            const uint32_t lo = (uint32_t)k, hi = (uint32_t)(k >> 32);
            int rank = 0;
            for (int j = 0; j < count; j++) {
                const uint32_t a = __builtin_amdgcn_readlane(lo, j), b = __builtin_amdgcn_readlane(hi, j);
                rank += ((unsigned long long)b << 32 | a) > k;
            }
            if ((int)threadIdx.x < count) {
                if (rank < kept) S.top[rank] = k;
            } else if ((int)threadIdx.x < kept) {
                S.top[threadIdx.x] = 0;
            }
        }
    } else if (count <= LP_LIST) {
        for (int i = threadIdx.x; i < count; i += NT) {
            const unsigned long long k = S.list[i];
            int rank = 0;
            for (int j = 0; j < count; j++) rank += S.list[j] > k;
            if (rank < kept) S.top[rank] = k;
        }
    } else {  // more equal logits than the list holds: one after the other
        unsigned long long last = ~0ull;
        for (int i = 0; i < kept; i++) {
            unsigned long long b = 0;
            each([&](unsigned long long k) { b = k < last && k > b ? k : b; });
            b = wave_max_key(b);
            __syncthreads();
            if ((threadIdx.x & 63) == 0) S.best[threadIdx.x >> 6] = b;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NT / 64; w++) b = S.best[w] > b ? S.best[w] : b;
            if (threadIdx.x == 0) S.top[i] = b;
            last = b;
            if (!b) last = 0;
        }
    }
    __syncthreads();
}
// a row's results: largest f(x) m, sums L and H as in LpArgs, the best keys in top
DEV void lp_finish(const LpArgs& A, int row, float T, float m, double L, double H, const unsigned long long* top, float xt,
                   bool cap) {
    const double ln = log(L);
    auto logprob = [&](float x) -> float {
        if (x == -INFINITY) return -INFINITY;
        const float f = cap ? sm_f(x, A.cap) : x;
        return (float)((double)(f - m) / (double)T - ln);
    };
    const bool one = !(T > 0.f);  // the largest logit alone
    const int first = one && top[0] ? lp_id(top[0]) : -1;
    const int t = threadIdx.x;
    if (t == 0) {
        const int id = A.tokens ? A.tokens[row] : -1;
        const bool known = (unsigned)id < (unsigned)A.n;
        if (A.logprob) A.logprob[row] = !known ? -INFINITY : one ? (id == first ? 0.f : -INFINITY) : logprob(xt);
        if (A.entropy) A.entropy[row] = one || L == 0. ? 0.f : (float)(ln - 0.69314718055994530942 * H / L);
    }
    if (t < A.n_top) {
        const unsigned long long k = top[t];
        A.top_ids[(size_t)row * A.n_top + t] = k ? lp_id(k) : -1;
        A.top_logprobs[(size_t)row * A.n_top + t] = !k ? -INFINITY : one ? (t ? -INFINITY : 0.f) : logprob(lp_value(k));
    }
}
template <bool F32>
DEV float lp_token_logit(const LpArgs& A, int row) {
    const int id = A.tokens ? A.tokens[row] : -1;
    if ((unsigned)id >= (unsigned)A.n) return -INFINITY;
    const size_t at = (size_t)row * A.n + id;
    if constexpr (F32) return ((const float*)A.x)[at];
    else return h2f(((const uint16_t*)A.x)[at]);
}

// R words of V logits a thread
template <bool F32, bool CAP, int NT, int R, int V>
DEV void lp_part(const LpArgs& A) {
    __shared__ LpTop<NT> S;
    __shared__ float red[3][NT / 64];
    __shared__ uint32_t bound[2][NT / 64];
    constexpr int W = F32 ? V : V / 2;
    static_assert(R * V == 32 || R * V == 8, "a bit for each logit of a thread");
    const int row = blockIdx.x / A.parts, part = blockIdx.x % A.parts, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int base = part * NT * R * V + threadIdx.x * V;
    uint32_t v[R][W];
#pragma unroll
    for (int r = 0; r < R; r++) sm_load<F32, V>(A.x, (size_t)row * A.n, base + r * NT * V, A.n, v[r]);
    const float T = A.temp ? A.temp[row / A.rows_per_temp] : 1.f;
    const float xt = lp_token_logit<F32>(A, row);
    auto get = [&](int r, int j) { return sm_get<F32, V>(v[r], j); };
    // f of a logit less c (SmRow::less)
    auto less = [&](int r, int j, float c) {
        if constexpr (CAP) return sm_f(get(r, j), A.cap) - c;
        else if constexpr (F32) return get(r, j) - c;
        else return mix_less(v[r][j / 2], j & 1, c);
    };
    // ---- the thread's and the part's largest
    float mine = -INFINITY;
    if constexpr (F32) {
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int j = 0; j < V; j++) mine = fmaxf(mine, get(r, j));
    } else {
        typedef _Float16 hp __attribute__((ext_vector_type(2)));
        hp h = {(_Float16)-INFINITY, (_Float16)-INFINITY};
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int k = 0; k < W; k++) h = __builtin_elementwise_max(h, __builtin_bit_cast(hp, v[r][k]));
        mine = fmaxf((float)h[0], (float)h[1]);
    }
    float m = wave_max_u(mine);
    if (lane == 0) red[0][w] = m;
    const int kept = A.n_top ? A.n_top : T > 0.f ? 0 : 1;
    const uint32_t order = lp_order(mine);
    if (kept) {
        // the need-th largest of the lanes' or less, by its bits from the highest on
        // (f16 logits have no more than 19)
        auto nth = [&](int need) {
            uint32_t t = 0;
            for (int b = 31; b >= (F32 ? 0 : 13); b--) {
                const int c = __popcll(__ballot(order >= (t | 1u << b)));
                if (c >= need) t |= 1u << b;
                if (c == need) break;
            }
            return t;
        };
        // `kept` logits are not below any wave's kept-th, nor below the least of the
        // waves' (kept / waves)-th, which is the higher where the waves are alike
        const uint32_t a = nth(kept), b = nth((kept + NT / 64 - 1) / (NT / 64));
        if (lane == 0) bound[0][w] = a, bound[1][w] = b;
    }
    if (threadIdx.x == 0) S.count = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NT / 64; k++) m = fmaxf(m, red[0][k]);
    // ---- the sums
    m = uniform(CAP ? sm_f(m, A.cap) : m);
    const float c = m == -INFINITY ? 0.f : m, s = sm_scale(1.44269504088896340736f, T > 0.f ? T : 1.f);
    float l = 0.f, h = 0.f;
#pragma unroll
    for (int r = 0; r < R; r++) {
        float pl = 0.f, ph = 0.f;
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float z = less(r, j, c) * s, e = __builtin_amdgcn_exp2f(z);
            pl += e;
            ph = fmaf(e, fmaxf(z, -1e30f), ph);
        }
        l += pl, h += ph;
    }
    l = wave_sum_u(l), h = wave_sum_u(h);
    if (lane == 0) red[1][w] = l, red[2][w] = h;
    // ---- the part's likeliest
    if (kept) {
        uint32_t t = LP_NONE + 1, all = 0xffffffffu;
#pragma unroll
        for (int k = 0; k < NT / 64; k++) t = max(t, bound[0][k]), all = min(all, bound[1][k]);
        t = max(t, all);
        const float least = lp_value((unsigned long long)t << 32);  // or NaN: more than any logit
        // which of the thread's logits are not below the bound, then those few from
        // memory once more
        uint32_t some = 0;
        if (order >= t) {
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int j = 0; j < V; j++) some |= get(r, j) >= least ? 1u << (r * V + j) : 0u;
        }
        auto each = [&](auto f) {
            for (uint32_t left = some; left; left &= left - 1) {
                const int i = __ffs(left) - 1, at = base + i / V * NT * V + i % V;
                const size_t e = (size_t)row * A.n + at;
                float x;
                if constexpr (F32) x = ((const float*)A.x)[e];
                else x = h2f(((const uint16_t*)A.x)[e]);
                f(lp_key(lp_order(x), at));
            }
        };
        each([&](unsigned long long k) {
            const int at = atomicAdd(&S.count, 1);
            if (at < LP_LIST) S.list[at] = k;
        });
        lp_rank<NT>(S, kept, each);
    } else {
        __syncthreads();
    }
    l = red[1][0], h = red[2][0];
#pragma unroll
    for (int k = 1; k < NT / 64; k++) l += red[1][k], h += red[2][k];
    if (A.parts == 1) {
        lp_finish(A, row, T, m, l, h, S.top, xt, CAP);
    } else {
        if (threadIdx.x == 0) A.stats[blockIdx.x] = make_float4(m, l, h, 0.f);
        if ((int)threadIdx.x < kept) A.keys[(size_t)blockIdx.x * kept + threadIdx.x] = S.top[threadIdx.x];
    }
}

// A row's parts joined: their sums brought to the largest m, and of their keys those
// that are not below the largest of the parts' last ones, which bounds the row's
// last one.
template <bool F32, bool CAP>
DEV void lp_join(const LpArgs& A) {
    constexpr int NT = 256;
    __shared__ LpTop<NT> S;
    __shared__ float red[4];
    __shared__ double sums[2][4];
    __shared__ unsigned long long bound[4];
    const int row = blockIdx.x, t = threadIdx.x, w = t >> 6, lane = t & 63;
    const float4* st = A.stats + (size_t)row * A.parts;
    const float T = A.temp ? A.temp[row / A.rows_per_temp] : 1.f;
    const float xt = lp_token_logit<F32>(A, row);
    const int kept = A.n_top ? A.n_top : T > 0.f ? 0 : 1;
    const unsigned long long* keys = A.keys + (size_t)row * A.parts * kept;
    // the first of a thread's stats and keys are fetched together
    constexpr int U = 4;
    const long long many = (long long)A.parts * kept;
    const float4 mine = st[min(t, A.parts - 1)];
    unsigned long long key[U];
#pragma unroll
    for (int u = 0; u < U; u++) key[u] = t + u * NT < many ? keys[t + u * NT] : 0;
    float m = -INFINITY;
    unsigned long long last = 1;
    for (int p = t; p < A.parts; p += NT) m = fmaxf(m, p == t ? mine.x : st[p].x);
    // a key at a part's end
#pragma unroll
    for (int u = 0; u < U; u++)
        if (t + u * NT < many && (t + u * NT) % kept == kept - 1) last = max(last, key[u]);
    for (long long i = t + U * NT; i < many; i += NT)
        if (i % kept == kept - 1) last = max(last, keys[i]);
    m = wave_max_u(m);
    last = wave_max_key(last);
    if (lane == 0) red[w] = m, bound[w] = last;
    if (t == 0) S.count = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; k++) m = fmaxf(m, red[k]), last = max(last, bound[k]);
    const float c = m == -INFINITY ? 0.f : m, s = sm_scale(1.44269504088896340736f, T > 0.f ? T : 1.f);
    double L = 0, H = 0;
    for (int p = t; p < A.parts; p += NT) {
        const float4 q = p == t ? mine : st[p];
        const float z = (q.x - c) * s, a = q.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(z);
        L += (double)q.y * a;
        H += a != 0.f ? a * ((double)q.z + (double)q.y * (q.x == -INFINITY ? 0.f : z)) : 0.;
    }
    L = lane_d(wave_scan_d(L), 63), H = lane_d(wave_scan_d(H), 63);
    if (lane == 0) sums[0][w] = L, sums[1][w] = H;
    if (kept) {
        auto each = [&](auto f) {
#pragma unroll
            for (int u = 0; u < U; u++)
                if (key[u] >= last) f(key[u]);
            for (long long i = t + U * NT; i < many; i += NT) {
                const unsigned long long k = keys[i];
                if (k >= last) f(k);
            }
        };
        each([&](unsigned long long k) {
            const int at = atomicAdd(&S.count, 1);
            if (at < LP_LIST) S.list[at] = k;
        });
        lp_rank<NT>(S, kept, each);
    } else {
        __syncthreads();
    }
    L = (sums[0][0] + sums[0][1]) + (sums[0][2] + sums[0][3]);
    H = (sums[1][0] + sums[1][1]) + (sums[1][2] + sums[1][3]);
    lp_finish(A, row, T, m, L, H, S.top, xt, CAP);
}
#define LOGPROBS_PART(NAME, F32, CAP, NT, R)                                                              \
    extern "C" __global__ __launch_bounds__(NT) void cima_logprobs_t##NT##_w##R##_##NAME(const LpArgs A) { \
        lp_part<F32, CAP, NT, F32 ? R : R / 2, F32 ? 4 : 8>(A);                                            \
    }
#define LOGPROBS(NAME, F32, CAP)                                                                          \
    LOGPROBS_PART(NAME, F32, CAP, 256, 2)                                                                 \
    LOGPROBS_PART(NAME, F32, CAP, 256, 8)                                                                 \
    LOGPROBS_PART(NAME, F32, CAP, 1024, 8)                                                                \
    extern "C" __global__ __launch_bounds__(256) void cima_logprobs_join_##NAME(const LpArgs A) {         \
        lp_join<F32, CAP>(A);                                                                              \
    }
LOGPROBS(f16, false, false)
LOGPROBS(f32, true, false)
LOGPROBS(cap_f16, false, true)
LOGPROBS(cap_f32, true, true)

// ------------------------------------------------------------- verification
//
// Which drafts are kept needs one probability of p and q a draft; the token
// that follows needs one row of each.  The first launch sums that row's
// max(p - q, 0) in at most 64 parts (fp64), the second finds the part that holds
// u times the whole, a wave's running sum, and looks through it.  Every
// workgroup of the first works out the kept drafts itself, one round of loads.
// Bound by reading the two rows, short batches by the chain of loads.  Measured
// on MI355X: 192 slots of 128256 (197 MB) 28.2 us, 7.0 TB/s, and 4.7 for the second
// launch; two of 151936 3.7 + 4.1.

constexpr int VF_T = 256, VF_V = 8, VF_STEP = VF_T * VF_V;

struct VfArgs {
    const float* p;
    const float* q;
    const int* drafts;
    const int* counts;
    const float* u;
    int* accepted;
    int* tokens;
    int* lens;
    double* sums;  // [seqs][parts]
    int* state;    // [seqs]: kept drafts, + KEPT_REFUSED where the next was refused; -1: not in use
    int n_draft, vocab, parts, part_len;  // at most 64 parts, part_len a multiple of VF_STEP
};
constexpr int KEPT_REFUSED = 1 << 30;

// Drafts kept of slot s (-1: the slot is not in use), by the whole wave; the
// row whose residual is drawn from is p[kept] less q[kept] where `*refused`.
DEV int vf_kept(const VfArgs& A, int s, bool* refused) {
    const int lane = threadIdx.x & 63;
    // what the answer needs is fetched together, whether it is used or not
    const int len = A.lens ? A.lens[s] : 0;
    int count = A.counts ? A.counts[s] : A.n_draft;
    int d = -1;
    float u = 0.f;
    auto fetch = [&](int i) {
        d = i < A.n_draft ? A.drafts[(size_t)s * A.n_draft + i] : -1;
        u = i < A.n_draft ? A.u[(size_t)s * (A.n_draft + 1) + i] : 0.f;
    };
    fetch(lane);
    count = max(0, min(count, A.n_draft));
    *refused = false;
    if (len < 0) return -1;
    for (int i0 = 0; i0 < count; i0 += 64) {
        const int i = i0 + lane;
        if (i0) fetch(i);
        bool no = false;
        if (i < count) {
            no = true;
            if ((unsigned)d < (unsigned)A.vocab) {
                const double pd = A.p[((size_t)s * (A.n_draft + 1) + i) * A.vocab + d];
                const double qd = A.q ? A.q[((size_t)s * A.n_draft + i) * A.vocab + d] : 1.f;
                no = !((double)u * qd < pd);
            }
        }
        const unsigned long long b = __ballot(no);
        if (b) {
            *refused = true;
            return i0 + __ffsll(b) - 1;
        }
    }
    return count;
}
// eight entries of the residual from i on, those behind the vocabulary 0
struct VfRow {
    const float* p;
    const float* q;  // null: nothing is taken off but at `one`
    int one;         // the draft that was certain (-1: none)
};
DEV VfRow vf_row(const VfArgs& A, int s, int kept, bool refused) {
    VfRow r{A.p + ((size_t)s * (A.n_draft + 1) + kept) * A.vocab, nullptr, -1};
    if (refused) {
        if (A.q) r.q = A.q + ((size_t)s * A.n_draft + kept) * A.vocab;
        else r.one = A.drafts[(size_t)s * A.n_draft + kept];
    }
    return r;
}
DEV void ld8f(const float* p, float (&v)[8]) {
    __builtin_memcpy(v, __builtin_assume_aligned(p, 4), 32);
}
DEV void vf_load(const VfRow& r, int i, int n, float (&v)[8]) {
    float w[8];
    if (i + 8 <= n) {
        ld8f(r.p + i, v);
        if (r.q) ld8f(r.q + i, w);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            v[j] = i + j < n ? r.p[i + j] : 0.f;
            w[j] = r.q && i + j < n ? r.q[i + j] : 0.f;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if (r.q) v[j] -= w[j];
        v[j] = v[j] > 0.f && i + j != r.one ? v[j] : 0.f;
    }
}
// sum of one part by the workgroup
DEV double vf_part(const VfArgs& A, const VfRow& r, int part) {
    __shared__ double red[4];
    double s = 0;
    for (int i = part * A.part_len; i < min((part + 1) * A.part_len, A.vocab); i += VF_STEP) {
        float v[8];
        vf_load(r, i + threadIdx.x * VF_V, A.vocab, v);
#pragma unroll
        for (int j = 0; j < 8; j++) s += v[j];
    }
    s = wave_scan_d(s);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = s;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

extern "C" __global__ __launch_bounds__(VF_T) void cima_verify_sums(const VfArgs A) {
    const int s = blockIdx.x / A.parts, part = blockIdx.x % A.parts;
    bool refused = false;
    const int kept = vf_kept(A, s, &refused);
    if (part == 0 && threadIdx.x == 0) A.state[s] = kept < 0 ? -1 : kept + (refused ? KEPT_REFUSED : 0);
    if (kept < 0) return;
    const double v = vf_part(A, vf_row(A, s, kept, refused), part);
    if (threadIdx.x == 0) A.sums[blockIdx.x] = v;
}

extern "C" __global__ __launch_bounds__(VF_T) void cima_verify_draw(const VfArgs A) {
    const int s = blockIdx.x, t = threadIdx.x, lane = t & 63, w = t >> 6;
    double* sums = A.sums + (size_t)s * A.parts;
    const int state = A.state[s];
    double v = lane < A.parts ? sums[lane] : 0.0;  // a slot not in use has none: not used below
    const float u = A.u[(size_t)s * (A.n_draft + 1) + A.n_draft];
    const bool refused = state >= 0 && state & KEPT_REFUSED;
    const int kept = state < 0 ? -1 : state & (KEPT_REFUSED - 1);
    int* out = A.tokens + (size_t)s * (A.n_draft + 1);
    for (int i = t; i <= A.n_draft; i += VF_T)
        if (i != kept) out[i] = i < kept ? A.drafts[(size_t)s * A.n_draft + i] : -1;
    if (t == 0) A.accepted[s] = max(kept, 0);
    if (kept < 0) return;
    VfRow r = vf_row(A, s, kept, refused);
    double x = wave_scan_d(v), whole = lane_d(x, 63);
    if (!(whole > 0) && refused) {  // nothing left of p: from p itself
        r.q = nullptr;
        r.one = -1;
        for (int i = 0; i < A.parts; i++) {
            const double z = vf_part(A, r, i);
            if (lane == i) v = z;
        }
        x = wave_scan_d(v), whole = lane_d(x, 63);
    }
    __shared__ double wsum[4];
    __shared__ int found, last;
    int token = -1;
    if (whole > 0) {
        const double goal = (double)u * whole;
        // the part that passes the goal, else the last that holds anything
        const unsigned long long some = __ballot(v > 0), past = __ballot(v > 0 && x > goal);
        const int part = past ? __ffsll(past) - 1 : 63 - __clzll(some);
        double before = lane_d(x, part) - lane_d(v, part);
        if (t == 0) found = 0x7fffffff, last = -1;
        for (int i0 = part * A.part_len; i0 < min((part + 1) * A.part_len, A.vocab); i0 += VF_STEP) {
            float p[8];
            vf_load(r, i0 + t * VF_V, A.vocab, p);
            double mine = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) mine += p[j];
            const double y = wave_scan_d(mine);
            __syncthreads();
            if (lane == 63) wsum[w] = y;
            __syncthreads();
            double run = before;
            for (int i = 0; i < w; i++) run += wsum[i];
            run += y - mine;
            int hit = 0x7fffffff, end = -1;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                run += p[j];
                if (p[j] > 0.f) {
                    end = i0 + t * VF_V + j;
                    if (run > goal && hit == 0x7fffffff) hit = end;
                }
            }
            // a wave's entries follow its lanes
            const unsigned long long hits = __ballot(hit != 0x7fffffff), ends = __ballot(end >= 0);
            if (hits && lane == __ffsll(hits) - 1) atomicMin(&found, hit);
            if (ends && lane == 63 - __clzll(ends)) atomicMax(&last, end);
            __syncthreads();
            if (found != 0x7fffffff) break;
            before += (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]);
        }
        token = found != 0x7fffffff ? found : last;
    }
    if (t == 0) {
        out[kept] = token;
        if (A.lens) A.lens[s] += kept + 1;
    }
}
