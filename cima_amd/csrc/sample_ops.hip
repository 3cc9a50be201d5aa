// Sampling over rows of the vocabulary for gfx950 (CDNA4): the code object
// cima_sample.hsaco.  Softmax of rows of logits at a temperature, and the
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
    // a logit less c: of f16 logits as x * 1 - c, one instruction with the
    // conversion, the same number
    DEV float less(int r, int j, float c) const {
        if constexpr (W32) return get(r, j) - c;
        float d;
        if (j & 1)
            __asm__("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(v[r][j / 2]), "v"(c));
        else
            __asm__("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel_hi:[1,0,0]" : "=v"(d) : "v"(v[r][j / 2]), "v"(c));
        return d;
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
