// Sampling over rows of the vocabulary for gfx950 (CDNA4): the code object
// cima_sample.hsaco.  Softmax of rows of logits at a temperature, log probabilities
// of given tokens with the rows' entropy and likeliest alternatives, and the
// verification of drafted tokens.
#include "gguf_formats.h"

#include <type_traits>

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

// a logit of a pair times s less c
DEV float mix_fma(uint32_t pair, bool high, float s, float c) {
    float d;
    if (high)
        __asm__("v_fma_mix_f32 %0, %1, %2, -%3 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(pair), "v"(s), "v"(c));
    else
        __asm__("v_fma_mix_f32 %0, %1, %2, -%3 op_sel_hi:[1,0,0]" : "=v"(d) : "v"(pair), "v"(s), "v"(c));
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
            if (!(T > 0.f)) {  // by comparisons: a maximum loses what it had at a signalling NaN
                m = -INFINITY;
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int j = 0; j < V; j++) m = get(r, j) > m ? get(r, j) : m;
            }
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
// ln L, the row's entropy ln L - sum e^z z / L.  One reading of the logits, each thread
// to its own running maximum and sums.  The likeliest n_top are found from the
// largest logits of groups of 32 (neighbours, or a thread's in a row of one workgroup):
// the n_top-th of 64 samples, each the largest of a 64th of the threads' groups, bounds
// the row's n_top-th from below, and what the few groups that reach it hold is
// looked at one by one and ranked by counting (value first, then the lower id).
// Rows up to 32768 logits go to a workgroup each, in one launch; of longer ones the
// parts leave their sums and groups' largest, and a second launch joins them (in
// fp64) and finds the likeliest: looked for in each part they took as long as the
// sums did.  Measured on MI355X: 384 rows of 128256 f16 with 20 alternatives 21.5 us (4.6
// TB/s) and 8.4 for the join, capped 37.4 and 8.6, f32 35.9 and 8.1, both 43.6 and 8.2;
// 777 rows of 151936 without 41.5 (5.7 TB/s) and 4.6; one of them with 5 3.3 and 6.8, a
// chain of three loads, a search by bits and a ranking; 384 rows of 2000 in one launch
// 6.8.  Bound by vector instructions: a logit is a fused
// multiply-add, an exponential at half rate, a maximum, an addition and another
// multiply-add, and a share of finding its group's largest.

constexpr int LP_TOP = 32;     // most alternatives
constexpr int LP_LIST = 1024;  // logits looked at one by one
constexpr int LP_GROUPS = 256;

struct LpArgs {
    const void* x;
    const int* tokens;
    float* logprob;
    float* entropy;
    int* top_ids;
    float* top_logprobs;
    const float* temp;
    float4* stats;  // [rows][parts]: m, l, sum of e^z z in log2's unit
    void* largest;  // [rows][parts][groups of a part], f32 or f16 as the logits
    int n, n_top, rows_per_temp, parts, chunk_shift;  // 2^chunk_shift chunks a part
    float cap;
};

// logits in order as whole numbers; -0 as 0
DEV uint32_t lp_order(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.f);
    return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
DEV float lp_value(uint32_t order) {
    return __builtin_bit_cast(float, order ^ (order >> 31 ? 0x80000000u : 0xffffffffu));
}
constexpr uint32_t LP_NONE = 0x007fffffu;  // of -inf: a token that may not be taken
DEV unsigned long long lp_key(uint32_t order, int at) { return (unsigned long long)order << 32 | (uint32_t)~at; }
DEV int lp_id(unsigned long long key) { return (int)~(uint32_t)key; }
template <bool F32>
DEV float lp_load(const void* x, size_t row0, int i, int n) {
    if ((unsigned)i >= (unsigned)n) return -INFINITY;
    if constexpr (F32) return ((const float*)x)[row0 + i];
    else return h2f(((const uint16_t*)x)[row0 + i]);
}
DEV int lanes_below(unsigned long long m) { return __popcll(m & ((1ull << (threadIdx.x & 63)) - 1)); }

template <int NT>
struct LpTop {  // shared between the threads of a workgroup
    unsigned long long list[LP_LIST + 8], top[LP_TOP];
    int group[LP_GROUPS];
    int count, groups, found[2][NT / 64], bits[32];
    uint32_t sample[64], bound[NT / 64];
};
// the `kept` largest of the listed keys to S.top in order, zeros behind them, while
// the second wave does something else
template <int NT, typename B>
DEV void lp_rank(LpTop<NT>& S, int kept, B beside) {
    const int count = S.count;
    if (count <= 64) {  // a lane each: no loads from list to list
        if (threadIdx.x < 64) {
            const unsigned long long k = (int)threadIdx.x < count ? S.list[threadIdx.x] : 0;
            const uint32_t lo = (uint32_t)k, hi = (uint32_t)(k >> 32);
            int rank = 0;
            for (int j0 = 0; j0 < count; j0 += 4)
#pragma unroll
                for (int j = j0; j < j0 + 4; j++) {
                    const uint32_t a = __builtin_amdgcn_readlane(lo, j), b = __builtin_amdgcn_readlane(hi, j);
                    rank += ((unsigned long long)b << 32 | a) > k;
                }
            if ((int)threadIdx.x < count) {
                if (rank < kept) S.top[rank] = k;
            } else if ((int)threadIdx.x < kept) {
                S.top[threadIdx.x] = 0;
            }
        } else if (threadIdx.x < 128) {
            beside();
        }
    } else {
        if (threadIdx.x >= 64 && threadIdx.x < 128) beside();
        if (threadIdx.x < 7) S.list[count + threadIdx.x] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < count; i += NT) {
            const unsigned long long k = S.list[i];
            int rank = 0;
            for (int j = 0; j < count; j += 8)
#pragma unroll
                for (int u = 0; u < 8; u++) rank += S.list[j + u] > k;
            if (rank < kept) S.top[rank] = k;
        }
    }
    __syncthreads();
}
// those of R words of V logits, `step` apart from `at` of the row on, that are not below
// `least` to S.list, as far as there is room
template <int NT, bool F32, int V, int R>
DEV void lp_list(LpTop<NT>& S, const uint32_t (&v)[R][F32 ? V : V / 2], int at, int step, float least) {
    int mine = 0;
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int j = 0; j < V; j++) mine += sm_get<F32, V>(v[r], j) >= least;
    if (!mine) return;
    int to = atomicAdd(&S.count, mine);
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float y = sm_get<F32, V>(v[r], j);
            if (y >= least && to < LP_LIST) S.list[to++] = lp_key(lp_order(y), at + r * step + j);
        }
}
// The same of every group whose largest is not below `least`: each_group(f): f(largest,
// group) for every group of this thread, `most` the largest of them; place(g, p): where
// in the row piece p of PIECES of V logits of group g begins.  A barrier is behind it.
template <int NT, bool F32, int V, int PIECES, typename G, typename P>
DEV void lp_gather(LpTop<NT>& S, const void* x, size_t row0, int n, float least, G each_group, float most, P place) {
    if (most >= least)
        each_group([&](float y, int g) {
            if (y >= least) {
                const int to = atomicAdd(&S.groups, 1);
                if (to < LP_GROUPS) S.group[to] = g;
            }
        });
    __syncthreads();
    const int many = min(S.groups, LP_GROUPS) * PIECES;
    for (int i = threadIdx.x; i < many; i += NT) {
        const int at = place(S.group[i / PIECES], i % PIECES);
        uint32_t v[1][F32 ? V : V / 2];
        sm_load<F32, V>(x, row0, at, n, v[0]);
        lp_list<NT, F32, V>(S, v, at, 0, least);
    }
    __syncthreads();
}
// The row's `kept` likeliest to S.top.  `most`: the largest of this thread's groups;
// gather(least): logits of the groups whose largest is not below `least` that are not
// below it themselves to S.list, with a barrier behind; each_group(f): f(largest) for
// every group of this thread; beside(): something that the second wave has to do once.
template <int NT, bool F32, typename L, typename G, typename B>
DEV void lp_select(LpTop<NT>& S, int kept, const void* x, size_t row0, int n, float most, L gather, G each_group, B beside) {
    const int t = threadIdx.x, w = t >> 6, lane = t & 63;
    const uint32_t best = lp_order(most);
    // the kept-th largest of the lanes' or less, by its bits from the highest on (f16
    // logits have no more than 19) until as many are left and an eighth of it is known
    auto nth = [&](uint32_t of) {
        uint32_t v = 0;
        for (int b = 31; b >= (F32 ? 0 : 13); b--) {
            const int c = __popcll(__ballot(of >= (v | 1u << b)));
            if (c >= kept) v |= 1u << b;
            if (c == kept && b <= 20) break;
        }
        return v;
    };
    constexpr int LANES = NT / 64;  // that are one of 64 samples
    static_assert(LANES == 4 || LANES == 16, "a quad or a row of lanes");
    uint32_t many = best;
    many = max(many, (uint32_t)__builtin_amdgcn_mov_dpp((int)many, 0xB1, 0xf, 0xf, false));
    many = max(many, (uint32_t)__builtin_amdgcn_mov_dpp((int)many, 0x4E, 0xf, 0xf, false));
    if constexpr (LANES == 16) {
        many = max(many, (uint32_t)__builtin_amdgcn_mov_dpp((int)many, 0x141, 0xf, 0xf, false));
        many = max(many, (uint32_t)__builtin_amdgcn_mov_dpp((int)many, 0x140, 0xf, 0xf, false));
    }
    if (t % LANES == 0) S.sample[t / LANES] = many;
    if (t == 0) S.count = S.groups = 0;
    if (t < 32) S.bits[t] = 0;
    __syncthreads();
    uint32_t v = nth(S.sample[lane]);
    if (v <= LP_NONE) {  // few logits, or of tokens that may not be taken: any wave's kept-th
        const uint32_t b = nth(best);
        if (lane == 0) S.bound[w] = b;
        __syncthreads();
        v = LP_NONE + 1;
#pragma unroll
        for (int k = 0; k < NT / 64; k++) v = max(v, S.bound[k]);
    }
    // Logits that are not below v, from the groups whose largest is not, to S.list.  Where
    // there are too many, such as equal ones, once more from v + 1 on, v then the kept-th
    // largest of the groups' exactly: what is above it lies in less than `kept` groups.
    bool exact = false;
    while (true) {
        gather(lp_value(exact ? v + 1 : v));
        if (exact || (S.groups <= LP_GROUPS && S.count <= LP_LIST)) break;
        v = 0;
        for (int b = 31; b >= 0; b--) {
            int c = 0;
            each_group([&](float x) { c += lp_order(x) >= (v | 1u << b); });
            if (c) atomicAdd(&S.bits[b], c);
            __syncthreads();
            if (S.bits[b] >= kept) v |= 1u << b;
        }
        v = max(v, LP_NONE);
        if (t == 0) S.count = S.groups = 0;
        __syncthreads();
        exact = true;
    }
    lp_rank<NT>(S, kept, beside);
    if (!exact) return;
    // of v's equals the first follow
    int have = min(S.count, kept);
    for (int i0 = 0, k = 0; i0 < n && have < kept && v > LP_NONE; i0 += NT, k ^= 1) {
        const float y = lp_load<F32>(x, row0, i0 + t, n);
        const unsigned long long hit = __ballot(lp_order(y) == v);
        if (lane == 0) S.found[k][w] = __popcll(hit);
        __syncthreads();
        int to = have + lanes_below(hit), all = 0;
#pragma unroll
        for (int u = 0; u < NT / 64; u++) {
            if (u < w) to += S.found[k][u];
            all += S.found[k][u];
        }
        if (lp_order(y) == v && to < kept) S.top[to] = lp_key(v, i0 + t);
        have += all;
    }
    __syncthreads();
}
// f of a logit, cap tanh(x / cap), by two forms that are off by 2^-22 of it at most (as tanhf
// is), whatever the cap.  Up to the cap, u = x / cap: x (1 + t P(t)), t = u^2, P fitted to
// (tanh(u) / u - 1) / t for the least relative error, 5.5e-8; its highest coefficient is positive,
// so that infinities stay.  Above it cap - 2 cap / (1 + e^(2 |u|)), which cancels no
// more there: the quotient is 0.24 or less.  A wave takes the first for words of which no
// logit is above the cap, ten instructions at the full rate a logit.
struct LpCap {
    float cap, inv, s;  // 1 / cap; 2 log2(e) / cap
    uint32_t least, span;  // as bits, of f16 logits twice: above these finite logits may be above the cap; how far
};
template <bool F32>
DEV LpCap lp_cap(float cap) {
    LpCap C;
    C.cap = cap;
    C.inv = fminf(1.f / cap, 1e38f);
    C.s = 2.88539008177792681472f * C.inv;
    const float least = cap * 0.999999f;  // the rounding of u
    if constexpr (F32) {
        C.least = __builtin_bit_cast(uint32_t, least) + 1;
        C.span = 0x7f800000u - C.least;
    } else {
        uint32_t h = least < 65504.f ? f2h(least) : 0x7bffu;
        if (h2f(h) > least) h--;
        C.least = (h + 1) * 0x10001u, C.span = 0x7c00u - (h + 1);
    }
    return C;
}
DEV float lp_low(float x, const LpCap& C) {
    const float u = x * C.inv, t = u * u;
    float p = fmaf(t, 0.0010582645928059005f, -0.006259339200112074f);
    p = fmaf(t, p, 0.020359759264195577f);
    p = fmaf(t, p, -0.053498707589033995f);
    p = fmaf(t, p, 0.13326408874426884f);
    p = fmaf(t, p, -0.3333298677943413f);
    return fmaf(x * t, p, x);
}
DEV float lp_f(float x, const LpCap& C) {
    const float e = __builtin_amdgcn_exp2f(fabsf(x) * C.s);
    const float high = copysignf(fmaf(-2.f * __builtin_amdgcn_rcpf(1.f + e), C.cap, C.cap), x);
    return __builtin_isinf(x) ? x : fabsf(x * C.inv) <= 1.f ? lp_low(x, C) : high;
}
// whether any finite logit of a wave's words may be above the cap
template <bool F32, int W>
DEV bool lp_any_high(const uint32_t (&v)[W], const LpCap& C) {
    if constexpr (F32) {
        uint32_t m = 0xffffffffu;
#pragma unroll
        for (int i = 0; i < W; i++) m = min(m, (v[i] & 0x7fffffffu) - C.least);
        return __any(m < C.span);
    } else {
        typedef unsigned short us2 __attribute__((ext_vector_type(2)));
        us2 m = {0xffff, 0xffff};
#pragma unroll
        for (int i = 0; i < W; i++)
            m = __builtin_elementwise_min(m, __builtin_bit_cast(us2, v[i] & 0x7fff7fffu) - __builtin_bit_cast(us2, C.least));
        return __any(m[0] < C.span || m[1] < C.span);
    }
}
// The token that is left at T <= 0 under a cap: of the largest f(x) the first, as softmax_rows
// finds it, by its sm_f.  Several logits may have that f, the largest logit not the first
// of them.
struct LpBest {
    float f = -INFINITY;
    int at = 0x7fffffff;
    DEV void take(float y, int i) {
        if (y > f || (y == f && i < at)) f = y, at = i;
    }
    DEV void wave() {
#pragma unroll
        for (int o = 32; o; o >>= 1) take(__shfl_xor(f, o), __shfl_xor(at, o));
    }
    DEV int id() const { return f == -INFINITY ? -1 : at; }
};
// Below this no logit's sm_f is as large as that of `most`.  sm_f is off by 2^-21 of itself at
// most (the quotient, tanhf, the product), and by cap 2^-149 where the quotient is next to
// nothing; from 0 on tanh rises by its slope at the end of a stretch or more, 1 - tanh^2,
// and from 6.5 to 8 by 4.3e-6.
DEV float lp_as_large(float most, float cap) {
    if (!(most > 0.f)) return -INFINITY;
    if (__builtin_isinf(most)) return most;
    const float u = most / cap;
    if (u >= 8.f) return 6.5f * cap;
    const float th = tanhf(u);
    return most - cap * (th * 0x1p-19f / ((1.f - th) * (1.f + th)) + 0x1p-147f);
}
// of logits [lo, hi) of a row of n, by the workgroup (one call in a kernel), the largest of
// which that a thread looked at is `most`; the result in every thread
template <int NT, bool F32, int V>
DEV LpBest lp_best(const void* x, size_t row0, int lo, int hi, int n, float cap, float most) {
    __shared__ float best[NT / 64];
    __shared__ int place[NT / 64];
    LpBest b;
    const float least = lp_as_large(wave_max_u(most), cap);
#pragma unroll 4
    for (int i = lo + threadIdx.x * V; i < hi; i += NT * V) {
        uint32_t v[F32 ? V : V / 2];
        sm_load<F32, V>(x, row0, i, n, v);
        uint32_t near = 0;  // bit j: logit j may be it
#pragma unroll
        for (int j = 0; j < V; j++) near |= sm_get<F32, V>(v, j) >= least ? 1u << j : 0;
        for (; near; near &= near - 1) {
            const int j = __builtin_ctz(near);
            b.take(sm_f(lp_load<F32>(x, row0, i + j, n), cap), i + j);
        }
    }
    b.wave();
    if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = b.f, place[threadIdx.x >> 6] = b.at;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NT / 64; k++) b.take(best[k], place[k]);
    return b;
}
// alternatives that are looked for: where T <= 0 and there is no cap, the one token
DEV int lp_kept(const LpArgs& A, float T, bool cap) { return A.n_top ? A.n_top : T > 0.f || cap ? 0 : 1; }
// a row's results: largest f(x) m, sums L (and its logarithm) and H as in LpArgs, the
// best keys in top; under a cap at T <= 0 the token that is left (LpBest::id), without one
// the first of top
DEV void lp_finish(const LpArgs& A, int row, float T, float m, double ln, double L, double H,
                   const unsigned long long* top, float xt, bool cap, int left) {
    const LpCap C = lp_cap<true>(A.cap);
    auto logprob = [&](float x) -> float {
        if (x == -INFINITY) return -INFINITY;
        const float f = cap ? lp_f(x, C) : x;
        return (float)(((double)f - m) / T - ln);
    };
    const bool one = !(T > 0.f);  // the largest logit alone
    const int first = !one ? -1 : cap ? left : top[0] ? lp_id(top[0]) : -1;
    const int t = threadIdx.x;
    if (t == 0) {
        const int id = A.tokens ? A.tokens[row] : -1;
        const bool known = (unsigned)id < (unsigned)A.n;
        if (A.logprob) A.logprob[row] = !known ? -INFINITY : one ? (id == first ? 0.f : -INFINITY) : logprob(xt);
        if (A.entropy) A.entropy[row] = one || L == 0. ? 0.f : (float)(ln - 0.69314718055994530942 * H / L);
    }
    if (t < A.n_top) {
        unsigned long long k = top[t];
        if (one && cap && first >= 0) {  // it comes before those with larger logits
            bool behind = false;
            for (int i = 0; i < t; i++) behind |= lp_id(top[i]) == first;
            if (!behind) k = t ? top[t - 1] : lp_key(0, first);
        }
        A.top_ids[(size_t)row * A.n_top + t] = k ? lp_id(k) : -1;
        A.top_logprobs[(size_t)row * A.n_top + t] =
            !k ? -INFINITY : one ? (t ? -INFINITY : 0.f) : logprob(lp_value((uint32_t)(k >> 32)));
    }
}

// The largest number of W words, of f16 that of their lower halves beside that of
// their upper ones
template <bool F32, int W>
DEV uint32_t lp_largest(const uint32_t* v) {
    uint32_t p = v[0];
#pragma unroll
    for (int i = 1; i < W; i++) {
        if constexpr (F32) p = __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, p), __builtin_bit_cast(float, v[i])));
        else {
            uint32_t q;  // a register of its own: no copy of v[0] before it
            __asm__("v_pk_max_f16 %0, %1, %2" : "=v"(q) : "v"(p), "v"(v[i]));
            p = q;
        }
    }
    return p;
}
// Signalling NaN hides what a maximum had before it.  Where a thread's sum says that one of
// its logits is NaN, the largest of V from element i on is found anew, NaN as -inf; from
// memory, so that no register is held for it.
template <bool F32>
DEV uint32_t lp_number(uint32_t v) {
    if constexpr (F32) return (v & 0x7fffffffu) > 0x7f800000u ? 0xff800000u : v;
    const uint32_t lo = v & 0xffffu, hi = v >> 16;
    return ((lo & 0x7fffu) > 0x7c00u ? 0xfc00u : lo) | ((hi & 0x7fffu) > 0x7c00u ? 0xfc00u : hi) << 16;
}
template <bool F32, int V>
DEV uint32_t lp_largest_number(const void* x, size_t row0, int i, int n) {
    constexpr int W = F32 ? V : V / 2;
    uint32_t v[W];
    sm_load<F32, V>(x, row0, i, n, v);
#pragma unroll
    for (int k = 0; k < W; k++) v[k] = lp_number<F32>(v[k]);
    return lp_largest<F32, W>(v);
}
// (NaN alone: -inf)
template <bool F32>
DEV float lp_of(uint32_t p) {
    if constexpr (F32) return fmaxf(__builtin_bit_cast(float, p), -INFINITY);
    else return fmaxf(fmaxf(h2f(p & 0xffffu), h2f(p >> 16)), -INFINITY);
}
// the largest of aligned groups of 4 or 8 lanes
template <bool F32, int LANES>
DEV uint32_t lp_lanes(uint32_t p) {
    auto other = [&](uint32_t q) {
        const uint32_t both[2] = {p, q};
        p = lp_largest<F32, 2>(both);
    };
    other(__builtin_amdgcn_mov_dpp(p, 0xB1, 0xf, 0xf, false));
    other(__builtin_amdgcn_mov_dpp(p, 0x4E, 0xf, 0xf, false));
    if constexpr (LANES == 8) other(__builtin_amdgcn_mov_dpp(p, 0x141, 0xf, 0xf, false));
    return p;
}
// a row's temperature: 2^-127 where it is positive and less, whose reciprocal is none
DEV float lp_temp(const LpArgs& A, int row) {
    const float T = A.temp ? A.temp[row / A.rows_per_temp] : 1.f;
    return T > 0.f ? fmaxf(T, 0x1p-127f) : T;
}
// z = (half y - half c) s, s = log2(e) / (half T): the halves of two fp32 logits differ by a
// number, they themselves may not; at low temperatures, where halving could round, they
// are near each other or z is far below 0.  At an infinite one s is the least number, so that
// -inf stays what it is.
struct LpScale {
    float s, half;
};
template <bool F32>
DEV LpScale lp_scale(float T) {
    const float half = F32 && T >= 1.f ? 0.5f : 1.f;
    return {T > 0.f ? fmaxf(1.44269504088896340736f / T, 0x1p-149f) / half : 1.f, half};
}
// A thread's running sums of 2^z and 2^z z, R words of V logits at a time: z = (f(x) -
// c) s, c f of the largest so far (0: none), half of it as LpScale says; FAST, of f16
// logits, z = x s - b in one instruction, b = c s as fp32 holds it, which the end puts
// right.  It takes |c s| up to 2^20, so that b is near enough: s up to LP_FAST.
constexpr float LP_FAST = 16.f;
template <bool F32, bool CAP, int R, int V>
struct LpSums {
    static constexpr int W = F32 ? V : V / 2;
    using Words = uint32_t[R][W];
    float mine = -INFINITY, c = 0.f, b = 0.f, l = 0.f, h = 0.f;

    // to another largest
    template <bool FAST>
    DEV void bring(float to, const LpScale& Z) {
        const float nc = F32 ? to * Z.half : to, nb = to * Z.s, z = mine == -INFINITY ? 0.f : FAST ? b - nb : (c - nc) * Z.s;
        const float a = __builtin_amdgcn_exp2f(z);
        h = a * fmaf(fmaxf(z, -1e30f), l, h), l *= a;
        c = nc, b = nb;
    }
    // words whose largest is m
    template <bool FAST>
    DEV void add(const Words& v, float m, const LpCap& C, const LpScale& Z) {
        if (m > mine) {
            bring<FAST>(CAP ? lp_f(m, C) : m, Z);
            mine = m;
        }
        const float least = -1e30f;  // for a product with 0
        const float s = Z.s;
        auto less = [&](float y) { return F32 ? fmaf(y, Z.half, -c) : y - c; };
        // z of logit j of word r: of(r, j)
        auto word = [&](int r, auto of) {
            float pl, ph;
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float z = of(r, j);
                float y;
                const float e = __builtin_amdgcn_exp2f(z);
                // (fmaxf of what an asm returns is two instructions, the first for NaN, which e has)
                __asm__("v_max_f32 %0, %1, %2" : "=v"(y) : "s"(least), "v"(z));
                pl = j ? pl + e : e;
                ph = j ? fmaf(e, y, ph) : e * y;
            }
            l += pl, h += ph;
        };
#pragma unroll
        for (int r = 0; r < R; r++) {
            if constexpr (CAP) {
                if (lp_any_high<F32>(v[r], C)) word(r, [&](int r, int j) { return less(lp_f(sm_get<F32, V>(v[r], j), C)) * s; });
                else word(r, [&](int r, int j) { return less(lp_low(sm_get<F32, V>(v[r], j), C)) * s; });
            } else {
                word(r, [&](int r, int j) {
                    if constexpr (FAST) return mix_fma(v[r][j / 2], j & 1, s, b);
                    else if constexpr (F32) return less(sm_get<F32, V>(v[r], j)) * s;
                    else return mix_less(v[r][j / 2], j & 1, c) * s;
                });
            }
        }
    }
    // the workgroup's: *m is f of its largest
    template <int NT, bool FAST>
    DEV void join(float* m, const LpCap& C, const LpScale& Z) {
        __shared__ float red[3][NT / 64];
        const int w = threadIdx.x >> 6;
        const float a = wave_max_u(mine);
        if ((threadIdx.x & 63) == 0) red[0][w] = a;
        __syncthreads();
        float g = red[0][0];
#pragma unroll
        for (int k = 1; k < NT / 64; k++) g = fmaxf(g, red[0][k]);
        *m = uniform(CAP ? lp_f(g, C) : g);
        bring<FAST>(*m, Z);
        l = wave_sum_u(l), h = wave_sum_u(h);
        if ((threadIdx.x & 63) == 0) red[1][w] = l, red[2][w] = h;
        __syncthreads();
        l = red[1][0], h = red[2][0];
#pragma unroll
        for (int k = 1; k < NT / 64; k++) l += red[1][k], h += red[2][k];
        if (FAST && *m != -INFINITY) {  // z less what b was rounded by
            const float off = -fmaf(*m, Z.s, -b), e = __builtin_amdgcn_exp2f(off);
            h = e * fmaf(off, l, h), l *= e;
        }
    }
};

// a row in R words of V logits a thread
template <bool F32, bool CAP, int NT, int R, int V>
DEV void lp_whole(const LpArgs& A) {
    __shared__ LpTop<NT> S;
    const int row = blockIdx.x, t = threadIdx.x;
    const size_t row0 = (size_t)row * A.n;
    const LpCap C = lp_cap<F32>(A.cap);
    LpSums<F32, CAP, R, V> P;
    typename decltype(P)::Words v;
#pragma unroll
    for (int r = 0; r < R; r++) sm_load<F32, V>(A.x, row0, t * V + r * NT * V, A.n, v[r]);
    const float T = lp_temp(A, row);
    const LpScale Z = lp_scale<F32>(T);
    const float xt = lp_load<F32>(A.x, row0, A.tokens ? A.tokens[row] : -1, A.n);
    const bool one = CAP && !(T > 0.f);  // no sums are asked for, but the token that is left
    float mine = -INFINITY, m = 0.f;
    if (!one) {
        mine = lp_of<F32>(lp_largest<F32, R * P.W>(&v[0][0]));
        P.template add<false>(v, mine, C, Z);
    }
    if (one || __any(P.l != P.l)) {
        mine = -INFINITY;
#pragma unroll 1
        for (int r = 0; r < R; r++)
            mine = fmaxf(mine, lp_of<F32>(lp_largest_number<F32, V>(A.x, row0, t * V + r * NT * V, A.n)));
    }
    if (!one) P.template join<NT, false>(&m, C, Z);
    const int kept = lp_kept(A, T, CAP);
    if (kept)
        lp_select<NT, F32>(
            S, kept, A.x, row0, A.n, mine,
            [&](float least) {  // a thread's logits are its group
                // few are listed from the registers (2000 logits, 20 alternatives 7.1 -> 6.2
                // us), more read again by many threads (8000 7.6, from the registers 8.4)
                if constexpr (R * V <= 8) {
                    if (mine >= least) lp_list<NT, F32, V>(S, v, t * V, NT * V, least);
                    __syncthreads();
                } else {
                    lp_gather<NT, F32, V, R>(
                        S, A.x, row0, A.n, least, [&](auto f) { f(mine, t); }, mine,
                        [&](int g, int p) { return p * NT * V + g * V; });
                }
            },
            [&](auto f) { f(mine); }, [] {});
    int left = -1;
    if constexpr (CAP)
        if (one) left = lp_best<NT, F32, V>(A.x, row0, 0, A.n, A.n, A.cap, mine).id();
    lp_finish(A, row, T, m, log((double)P.l), P.l, P.h, S.top, xt, CAP, left);
}

// Parts of rows: 256 threads, 2^chunk_shift chunks of 32 logits a thread (SMALL: one
// of 8).  A group is 32 logits that lie together, a word of LANES threads: what is
// looked at again is a line of memory, not four.
template <bool F32, bool SMALL>
struct LpShape {
    static constexpr int V = F32 ? 4 : 8, R = (SMALL ? 8 : 32) / V, CHUNK = 256 * R * V, LANES = 32 / V;
    static constexpr int GROUPS = CHUNK / 32;  // of a chunk; that of word r of threads LANES i, ... is R i + r
    static_assert(R <= LANES, "a thread for each word");
    using Largest = std::conditional_t<F32, float, uint16_t>;
    DEV static int place(int g, int piece) {
        const int chunk = g / GROUPS, i = g % GROUPS;
        return chunk * CHUNK + i % R * (256 * V) + i / R * 32 + piece * V;
    }
};
template <bool F32, bool CAP, bool SMALL>
DEV void lp_part(const LpArgs& A) {
    using P = LpShape<F32, SMALL>;
    const int row = blockIdx.x / A.parts, part = blockIdx.x % A.parts, t = threadIdx.x;
    const int first = part << A.chunk_shift, all = (A.n - 1) / P::CHUNK + 1, last = min(first + (1 << A.chunk_shift), all);
    const size_t row0 = (size_t)row * A.n;
    const float T = lp_temp(A, row);
    const LpScale Z = lp_scale<F32>(T);
    const bool kept = lp_kept(A, T, CAP);
    typename P::Largest* to = (typename P::Largest*)A.largest + (size_t)row * all * P::GROUPS;
    const LpCap C = lp_cap<F32>(A.cap);
    LpSums<F32, CAP, P::R, P::V> S;
    using Words = typename decltype(S)::Words;
    auto load = [&](int k, Words& v) {
        if ((k + 1) * P::CHUNK <= A.n) {
            const size_t at = row0 + (size_t)k * P::CHUNK + t * P::V;
            // past the caches: read once (777 rows of 151936 46.6 -> 42.0 us)
            typedef uint32_t word4 __attribute__((ext_vector_type(4), aligned(2)));
#pragma unroll
            for (int r = 0; r < P::R; r++) {
                word4 q;
                if constexpr (F32) q = __builtin_nontemporal_load((const word4*)((const float*)A.x + at + r * 256 * P::V));
                else q = __builtin_nontemporal_load((const word4*)((const uint16_t*)A.x + at + r * 256 * P::V));
#pragma unroll
                for (int i = 0; i < 4; i++) v[r][i] = q[i];
            }
        } else {
#pragma unroll
            for (int r = 0; r < P::R; r++) sm_load<F32, P::V>(A.x, row0, k * P::CHUNK + t * P::V + r * 256 * P::V, A.n, v[r]);
        }
    };
    // the largest of the group that word r of this thread is in
    auto put = [&](int k, int r, uint32_t g) {
        typename P::Largest* o = to + k * P::GROUPS + t / P::LANES * P::R + r;
        if constexpr (F32) *o = lp_of<F32>(g);
        else *o = (uint16_t)f2h(lp_of<F32>(g));
    };
    // the groups alone, NaN as -inf; the largest of this thread's logits
    auto find_groups = [&] {
        float most = -INFINITY;
#pragma unroll P::R
        for (int i = first * P::R; i < last * P::R; i++) {
            const int k = i / P::R, r = i % P::R, at = k * P::CHUNK + t * P::V + r * 256 * P::V;
            uint32_t p = lp_largest_number<F32, P::V>(A.x, row0, at, A.n);
            most = fmaxf(most, lp_of<F32>(p));
            p = lp_lanes<F32, P::LANES>(p);
            if (kept && t % P::LANES == r) put(k, r, p);  // by the same lane as add's
        }
        return most;
    };
    auto all_chunks = [&](auto fast) {
        auto add = [&](int k, const Words& v) {
            uint32_t word[P::R];
#pragma unroll
            for (int r = 0; r < P::R; r++) word[r] = lp_largest<F32, S.W>(v[r]);
            const float m = lp_of<F32>(lp_largest<F32, P::R>(word));
            if (kept) {
                const int i = t % P::LANES;
                uint32_t g = 0;
#pragma unroll
                for (int r = 0; r < P::R; r++) {
                    const uint32_t p = lp_lanes<F32, P::LANES>(word[r]);
                    g = i == r ? p : g;
                }
                if (i < P::R) put(k, i, g);
            }
            S.template add<fast>(v, m, C, Z);
        };
        Words v, next;
        load(first, v);
        for (int k = first; k < last; k += 2) {
            if (k + 1 < last) load(k + 1, next);
            add(k, v);
            if (k + 1 == last) break;
            if (k + 2 < last) load(k + 2, v);
            add(k + 1, next);
        }
        if (kept && __any(S.l != S.l)) find_groups();
        float m;
        S.template join<256, fast>(&m, C, Z);
        if (t == 0) A.stats[blockIdx.x] = make_float4(m, S.l, S.h, 0.f);
    };
    if constexpr (CAP)
        if (!(T > 0.f)) {  // no sums are asked for, but the token that is left: {f, id, 0, 0}
            const float most = find_groups();
            const LpBest b = lp_best<256, F32, P::V>(A.x, row0, first * P::CHUNK, min(last * P::CHUNK, A.n), A.n, A.cap, most);
            if (t == 0) A.stats[blockIdx.x] = make_float4(b.f, __builtin_bit_cast(float, b.at), 0.f, 0.f);
            return;
        }
    if constexpr (F32 || CAP) all_chunks(std::false_type{});
    else if (Z.s <= LP_FAST && Z.s >= 1e-30f) all_chunks(std::true_type{});
    else all_chunks(std::false_type{});
}

// A row's parts joined: their sums brought to the largest m, its likeliest looked for.
template <bool F32, bool CAP, bool SMALL>
DEV void lp_join(const LpArgs& A) {
    using P = LpShape<F32, SMALL>;
    constexpr int NT = 256, VG = F32 ? 4 : 8;  // groups of a load
    __shared__ LpTop<NT> S;
    const int row = blockIdx.x, t = threadIdx.x, lane = t & 63;
    const size_t row0 = (size_t)row * A.n;
    const float T = lp_temp(A, row);
    const double s = 1.44269504088896340736 / T;
    const float xt = lp_load<F32>(A.x, row0, A.tokens ? A.tokens[row] : -1, A.n);
    const int kept = lp_kept(A, T, CAP);
    __shared__ double sums[3];
    __shared__ float largest;
    __shared__ int left;
    // the sums, by one wave
    const float4* st = A.stats + (size_t)row * A.parts;
    const float4 first = st[min(lane, A.parts - 1)];
    auto join = [&] {
        if constexpr (CAP)
            if (!(T > 0.f)) {
                LpBest b;
                for (int p = lane; p < A.parts; p += 64) {
                    const float4 q = p < 64 ? first : st[p];
                    b.take(q.x, __builtin_bit_cast(int, q.y));
                }
                b.wave();
                left = b.id();
                return;
            }
        float m = -INFINITY;
        for (int p = lane; p < A.parts; p += 64) m = fmaxf(m, p < 64 ? first.x : st[p].x);
        m = wave_max_u(m);
        const float c = m == -INFINITY ? 0.f : m;
        double L = 0, H = 0;
        for (int p = lane; p < A.parts; p += 64) {
            const float4 q = p < 64 ? first : st[p];
            const float z = (float)(((double)q.x - c) * s), a = q.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(z);
            L += (double)q.y * a;
            H += a != 0.f ? a * ((double)q.z + (double)q.y * (q.x == -INFINITY ? 0.f : z)) : 0.;
        }
        L = lane_d(wave_scan_d(L), 63), H = lane_d(wave_scan_d(H), 63);
        sums[0] = log(L), sums[1] = L, sums[2] = H;
        largest = m;
    };
    if (!kept) {
        if (t >= 64) return;
        join();
    } else {
        // loads that a thread keeps, of rows up to 32768 VG logits (f16 262144, f32 131072);
        // those behind are read again
        constexpr int K = 4;
        const int loads = ((A.n - 1) / P::CHUNK + 1) * P::GROUPS / VG;
        const uint4* from = (const uint4*)((const typename P::Largest*)A.largest + (size_t)row * loads * VG);
        uint4 q[K];
#pragma unroll
        for (int u = 0; u < K; u++) {
            constexpr uint32_t NONE = F32 ? 0xff800000u : 0xfc00fc00u;
            q[u] = u * NT + t < loads ? from[u * NT + t] : make_uint4(NONE, NONE, NONE, NONE);
        }
        uint32_t a[K * 4];
#pragma unroll
        for (int u = 0; u < K; u++) a[4 * u] = q[u].x, a[4 * u + 1] = q[u].y, a[4 * u + 2] = q[u].z, a[4 * u + 3] = q[u].w;
        float most = lp_of<F32>(lp_largest<F32, K * 4>(a));
        for (int i = K * NT + t; i < loads; i += NT) {
            const uint4 z = from[i];
            const uint32_t b[4] = {z.x, z.y, z.z, z.w};
            most = fmaxf(most, lp_of<F32>(lp_largest<F32, 4>(b)));
        }
        auto each_group = [&](auto f) {
            auto eight = [&](const uint4& v, int i) {
                const uint32_t a[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int k = 0; k < VG; k++) {
                    const float x = F32 ? __builtin_bit_cast(float, a[k]) : h2f(k & 1 ? a[k / 2] >> 16 : a[k / 2] & 0xffffu);
                    f(x, i * VG + k);
                }
            };
#pragma unroll
            for (int u = 0; u < K; u++)
                if (u * NT + t < loads) eight(q[u], u * NT + t);
            for (int i = K * NT + t; i < loads; i += NT) eight(from[i], i);
        };
        lp_select<NT, F32>(
            S, kept, A.x, row0, A.n, most,
            [&](float least) {
                lp_gather<NT, F32, P::V, P::LANES>(S, A.x, row0, A.n, least, each_group, most, P::place);
            },
            [&](auto f) { each_group([&](float x, int) { f(x); }); }, join);
        if (t >= 64) return;
    }
    lp_finish(A, row, T, largest, sums[0], sums[1], sums[2], S.top, xt, CAP, left);
}
#define LOGPROBS_WHOLE(NAME, F32, CAP, NT, R)                                                             \
    extern "C" __global__ __launch_bounds__(NT) void cima_logprobs_t##NT##_w##R##_##NAME(const LpArgs A) { \
        lp_whole<F32, CAP, NT, F32 ? R : R / 2, F32 ? 4 : 8>(A);                                           \
    }
#define LOGPROBS_PARTS(NAME, F32, CAP, R, SMALL)                                                           \
    extern "C" __global__ __launch_bounds__(256) void cima_logprobs_part_w##R##_##NAME(const LpArgs A) {  \
        lp_part<F32, CAP, SMALL>(A);                                                                        \
    }                                                                                                      \
    extern "C" __global__ __launch_bounds__(256) void cima_logprobs_join_w##R##_##NAME(const LpArgs A) {  \
        lp_join<F32, CAP, SMALL>(A);                                                                        \
    }
#define LOGPROBS(NAME, F32, CAP)            \
    LOGPROBS_WHOLE(NAME, F32, CAP, 256, 2)  \
    LOGPROBS_WHOLE(NAME, F32, CAP, 256, 8)  \
    LOGPROBS_WHOLE(NAME, F32, CAP, 1024, 8) \
    LOGPROBS_PARTS(NAME, F32, CAP, 2, true) \
    LOGPROBS_PARTS(NAME, F32, CAP, 8, false)
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
