// Sampling over rows of the vocabulary for gfx950 (CDNA4): the code object
// cima_sample.hsaco.  Softmax of rows of logits at a temperature, and the
// verification of drafted tokens.
#include "gguf_formats.h"

// ------------------------------------------------------------------ softmax
//
// A row is taken by `parts` workgroups, PART logits each.  The first launch
// leaves each part's maximum, its place and the sum of e^((f(x) - m) / T); the
// second joins a row's parts, reads its own logits once more (from the caches)
// and writes the probabilities.

constexpr int SM_T = 256, SM_V = 8, SM_R = 4;     // threads, logits a word, words a thread
constexpr int SM_PART = SM_T * SM_V * SM_R;       // logits of a part
struct SmPart {
    float m, l;
    int at, pad;
};

// eight logits from element i on (i < n), those behind n as -inf
template <bool F32>
DEV void sm_load(const void* __restrict__ x, size_t row, int i, int n, float (&v)[8]) {
    if (i + 8 <= n) {
        if (F32) {
            const float* p = (const float*)x + row + i;
            uint4 a, b;
            __builtin_memcpy(&a, __builtin_assume_aligned(p, 4), 16);
            __builtin_memcpy(&b, __builtin_assume_aligned(p + 4, 4), 16);
            const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = __builtin_bit_cast(float, u[j]);
        } else {
            const uint4 a = ld16u((const uint8_t*)((const uint16_t*)x + row + i));
            const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int j = 0; j < 4; j++) v[2 * j] = h2f(u[j] & 0xffffu), v[2 * j + 1] = h2f(u[j] >> 16);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++)
        v[j] = i + j >= n ? -INFINITY : F32 ? ((const float*)x)[row + i + j] : h2f(((const uint16_t*)x)[row + i + j]);
}
// f(x) of the same eight; those behind n stay -inf
DEV void sm_cap(float (&v)[8], int i, int n, float cap) {
    if (cap > 0.f) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = i + j < n ? cap * tanhf(v[j] / cap) : v[j];
    }
}
// whether (a, i) ranks before (b, j): larger, or equal and at a lower place
DEV bool sm_before(float a, int i, float b, int j) { return a > b || (a == b && i < j); }

template <bool F32>
DEV void sm_stats(const void* __restrict__ x, SmPart* __restrict__ part, int n, const float* __restrict__ temp,
                  int rows_per_temp, float cap, int parts) {
    __shared__ float rm[4], rl[4];
    __shared__ int ra[4];
    const int row = blockIdx.x / parts, pt = blockIdx.x % parts, t = threadIdx.x;
    const float T = temp ? temp[row / rows_per_temp] : 1.f;
    float v[SM_R][8];
#pragma unroll
    for (int r = 0; r < SM_R; r++) sm_load<F32>(x, (size_t)row * n, pt * SM_PART + (r * SM_T + t) * SM_V, n, v[r]);
    float m = -INFINITY;
    int at = 0x7fffffff;
#pragma unroll
    for (int r = 0; r < SM_R; r++) {
        sm_cap(v[r], pt * SM_PART + (r * SM_T + t) * SM_V, n, cap);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int i = pt * SM_PART + (r * SM_T + t) * SM_V + j;
            if (v[r][j] > m) m = v[r][j], at = i;
        }
    }
    // a thread's first largest is its lowest place; across threads the place decides
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        const float om = __shfl_xor(m, o);
        const int oa = __shfl_xor(at, o);
        if (sm_before(om, oa, m, at)) m = om, at = oa;
    }
    if ((t & 63) == 0) rm[t >> 6] = m, ra[t >> 6] = at;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; w++)
        if (sm_before(rm[w], ra[w], m, at)) m = rm[w], at = ra[w];
    float l = 0.f;
    if (T > 0.f) {
        // a part of -inf alone adds nothing
        const float c = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int r = 0; r < SM_R; r++)
#pragma unroll
            for (int j = 0; j < 8; j++) l += expf((v[r][j] - c) / T);
    }
    l = wave_sum_u(l);
    if ((t & 63) == 0) rl[t >> 6] = l;
    __syncthreads();
    if (t == 0) part[blockIdx.x] = SmPart{m, (rl[0] + rl[1]) + (rl[2] + rl[3]), at, 0};
}

template <bool F32>
DEV void sm_probs(const void* __restrict__ x, float* __restrict__ y, const SmPart* __restrict__ part, int n,
                  const float* __restrict__ temp, int rows_per_temp, float cap, int parts) {
    const int row = blockIdx.x / parts, pt = blockIdx.x % parts, t = threadIdx.x;
    const float T = temp ? temp[row / rows_per_temp] : 1.f;
    float m = -INFINITY;
    int at = 0x7fffffff;
    const SmPart* p = part + (size_t)row * parts;
    for (int i = 0; i < parts; i++)
        if (sm_before(p[i].m, p[i].at, m, at)) m = p[i].m, at = p[i].at;
    const float c = m == -INFINITY ? 0.f : m;
    float L = 0.f;
    if (T > 0.f)
        for (int i = 0; i < parts; i++) L += p[i].l * (p[i].m == -INFINITY ? 1.f : expf((p[i].m - c) / T));
    const bool none = m == -INFINITY && L == 0.f;
    const float inv = none ? 0.f : 1.f / L;
#pragma unroll
    for (int r = 0; r < SM_R; r++) {
        const int i = pt * SM_PART + (r * SM_T + t) * SM_V;
        if (i >= n) break;
        float v[8];
        sm_load<F32>(x, (size_t)row * n, i, n, v);
        sm_cap(v, i, n, cap);
        float* o = y + (size_t)row * n + i;
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = T > 0.f ? expf((v[j] - c) / T) * inv : (i + j == at ? 1.f : 0.f);
        if (i + 8 <= n) {
            __builtin_memcpy(__builtin_assume_aligned(o, 4), v, 32);
        } else {
            for (int j = 0; j < 8 && i + j < n; j++) o[j] = v[j];
        }
    }
}
#define SOFTMAX(NAME, F32)                                                                                             \
    extern "C" __global__ __launch_bounds__(SM_T) void cima_softmax_stats_##NAME(                                      \
        const void* __restrict__ x, SmPart* __restrict__ part, int n, const float* __restrict__ temp,                  \
        int rows_per_temp, float cap, int parts) {                                                                     \
        sm_stats<F32>(x, part, n, temp, rows_per_temp, cap, parts);                                                    \
    }                                                                                                                  \
    extern "C" __global__ __launch_bounds__(SM_T) void cima_softmax_probs_##NAME(                                      \
        const void* __restrict__ x, float* __restrict__ y, const SmPart* __restrict__ part, int n,                     \
        const float* __restrict__ temp, int rows_per_temp, float cap, int parts) {                                     \
        sm_probs<F32>(x, y, part, n, temp, rows_per_temp, cap, parts);                                                 \
    }
SOFTMAX(f16, false)
SOFTMAX(f32, true)

// ------------------------------------------------------------- verification
//
// Which drafts are kept needs one probability of p and q a draft; the token
// that follows needs one row of each.  The first launch sums that row's
// max(p - q, 0) in parts of VF_PART entries (fp64), the second finds the part
// that holds u times the whole and looks through it.  Every workgroup works
// out the kept drafts itself: one round of loads.

constexpr int VF_T = 256, VF_V = 8, VF_PART = VF_T * VF_V;

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
    int n_draft, vocab, parts;
};

// Drafts kept of slot s (-1: the slot is not in use), by the whole wave; the
// row whose residual is drawn from is p[kept] less q[kept] where `*refused`.
DEV int vf_kept(const VfArgs& A, int s, bool* refused) {
    if (A.lens && A.lens[s] < 0) return -1;
    int count = A.counts ? A.counts[s] : A.n_draft;
    count = max(0, min(count, A.n_draft));
    const int lane = threadIdx.x & 63;
    for (int i0 = 0; i0 < count; i0 += 64) {
        const int i = i0 + lane;
        bool no = false;
        if (i < count) {
            const int d = A.drafts[(size_t)s * A.n_draft + i];
            no = true;
            if ((unsigned)d < (unsigned)A.vocab) {
                const double pd = A.p[((size_t)s * (A.n_draft + 1) + i) * A.vocab + d];
                const double qd = A.q ? A.q[((size_t)s * A.n_draft + i) * A.vocab + d] : 1.f;
                no = !((double)A.u[(size_t)s * (A.n_draft + 1) + i] * qd < pd);
            }
        }
        const unsigned long long b = __ballot(no);
        if (b) {
            *refused = true;
            return i0 + __ffsll((unsigned long long)b) - 1;
        }
    }
    *refused = false;
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
DEV double wave_sum_d(double v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// sum of one part by the workgroup
DEV double vf_part(const VfRow& r, int part, int n) {
    __shared__ double red[4];
    float v[8];
    vf_load(r, part * VF_PART + threadIdx.x * VF_V, n, v);
    double s = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) s += v[j];
    s = wave_sum_d(s);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

extern "C" __global__ __launch_bounds__(VF_T) void cima_verify_sums(const VfArgs A) {
    const int s = blockIdx.x / A.parts, part = blockIdx.x % A.parts;
    bool refused;
    const int kept = vf_kept(A, s, &refused);
    if (kept < 0) return;
    const double v = vf_part(vf_row(A, s, kept, refused), part, A.vocab);
    if (threadIdx.x == 0) A.sums[blockIdx.x] = v;
}

extern "C" __global__ __launch_bounds__(VF_T) void cima_verify_draw(const VfArgs A) {
    const int s = blockIdx.x, t = threadIdx.x, n = A.vocab;
    bool refused = false;
    const int kept = vf_kept(A, s, &refused);
    int* out = A.tokens + (size_t)s * (A.n_draft + 1);
    for (int i = t; i <= A.n_draft; i += VF_T)
        if (i != kept) out[i] = i < kept ? A.drafts[(size_t)s * A.n_draft + i] : -1;
    if (t == 0) A.accepted[s] = max(kept, 0);
    if (kept < 0) return;
    VfRow r = vf_row(A, s, kept, refused);
    double* sums = A.sums + (size_t)s * A.parts;
    double whole = 0;
    for (int i = 0; i < A.parts; i++) whole += sums[i];
    if (!(whole > 0) && refused) {  // nothing left of p: from p itself
        r.q = nullptr;
        r.one = -1;
        whole = 0;
        for (int i = 0; i < A.parts; i++) {
            const double v = vf_part(r, i, n);
            if (t == 0) sums[i] = v;
            whole += v;
        }
        __syncthreads();
    }
    __shared__ double wsum[4];
    __shared__ int found, last;
    int token = -1;
    if (whole > 0) {
        const double goal = (double)A.u[(size_t)s * (A.n_draft + 1) + A.n_draft] * whole;
        // the part that passes the goal, else the last that holds anything
        double before = 0, run = 0;
        int part = 0;
        for (int i = 0; i < A.parts; i++) {
            const double v = sums[i];
            if (v > 0) {
                part = i;
                before = run;
            }
            run += v;
            if (run > goal) break;
        }
        float v[8];
        vf_load(r, part * VF_PART + t * VF_V, n, v);
        double mine = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) mine += v[j];
        double x = mine;
        const int lane = t & 63, w = t >> 6;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double y = __shfl_up(x, o);
            if (lane >= o) x += y;
        }
        if (t == 0) found = 0x7fffffff, last = -1;
        if (lane == 63) wsum[w] = x;
        __syncthreads();
        double run2 = before;
        for (int i = 0; i < w; i++) run2 += wsum[i];
        run2 += x - mine;
        int hit = 0x7fffffff, end = -1;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            run2 += v[j];
            const int i = part * VF_PART + t * VF_V + j;
            if (v[j] > 0.f) {
                end = i;
                if (run2 > goal && hit == 0x7fffffff) hit = i;
            }
        }
        if (hit != 0x7fffffff) atomicMin(&found, hit);
        if (end >= 0) atomicMax(&last, end);
        __syncthreads();
        token = found != 0x7fffffff ? found : last;
    }
    if (t == 0) {
        out[kept] = token;
        if (A.lens) A.lens[s] += kept + 1;
    }
}
