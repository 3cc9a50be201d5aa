// Attention of a batch over a paged KV cache for gfx950 (CDNA4): the code
// object cima_paged_attn.hsaco.
//
// out = sum_t w_t v_t / sum_t w_t, w_t = e^(scale q.k_t - m), over the positions
// t that a row sees.  The rows of a kv head are its query heads times the
// step's tokens; those of all slots share the prefix's pages, so one workgroup
// takes up to 256 of them through a range of the prefix and its keys and values
// are read once for all (prefix tasks).  A slot's own pages are seen by its own
// rows alone (own tasks).  Both kinds run the same code on a tile of rows and a
// range of positions and leave {m, l, sum} per row; a second launch joins them.
//
// Both products run on the matrix cores with 32 x 32 x 16 f16 MFMA.  S^T = K
// Q^T: a lane then holds the scores of ONE row (column lane % 32) for half of
// the 32 keys, so that the row maximum and sum are per-lane operations and one
// exchange between the halves of the wave, and the probabilities are in the
// lane that multiplies them: as the B operand of O^T = V^T P^T, whose order of
// keys is chosen to be that of S^T's registers.  V^T's fragments come from
// row-major LDS through transposing reads (ds_read_b64_tr_b16).  Keys and
// values reach LDS by direct copies (global_load_lds_dwordx4) a ring of tiles
// ahead; the 16-byte words of a row are stored permuted so that neither kind
// of read meets bank conflicts.
#include "gguf_formats.h"

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef float f2 __attribute__((ext_vector_type(2)));

// every lane copies the 16 bytes at g to LDS byte lds + 16 * lane; written in
// asm so that the compiler's wait counting leaves the copies alone (their
// waits are explicit)
DEV void dma16(const void* g, uint32_t lds) {
    asm volatile("global_load_lds_dwordx4 %0, off" ::"v"(g), "{m0}"(__builtin_amdgcn_readfirstlane(lds)) : "memory");
}
template <int N>
DEV void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// workgroup barrier that does not wait for copies in flight
DEV void barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// v of this lane and of the lane in the other half of the wave
DEV f2 halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v),
                                                    false, false);
    const uint32_t a = r[0], b = r[1];  // a bit cast of r[1] itself would take r[0]
    return f2{__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}

struct AttnArgs {
    const uint16_t* q;
    const uint16_t* kp;  // planes of the layer
    const uint16_t* vp;
    const int* table;
    const int* lens;
    uint16_t* out;
    float* acc;  // [rows * q_heads][parts][D]
    f2* ml;      // [rows * q_heads][parts]
    int seqs, n_new, q_heads, kv_heads, page_shift, n_pages, table_stride;
    int prefix_pages, prefix_slot, window;
    int prefix_parts, own_parts, row_tiles;  // row tiles of the prefix tasks
    float scale2;                            // scale * log2(e)
};

constexpr int IDS = 1024;         // page ids of a task kept in LDS at a time
constexpr float LOWEST = -1e30f;  // below any score: the running maximum's start
// The running maximum is raised only where a score passes it by 2^14, and then
// to 2^6 above the score's: probabilities stay between 2^-14 * 2^6 and 2^14 of
// the largest, clear of f16's subnormals, and most tiles skip the rescaling.
constexpr float RAISE = 14.f, ABOVE = 6.f;

template <int D, int WR, int WK>
struct Tile {
    static constexpr int NW = WR * WK;
    static constexpr int KB = WK == 1 ? 2 : 1;      // 32-key blocks of a wave
    static constexpr int KT = 32 * KB * WK;         // keys of a tile
    static constexpr int BYTES = KT * D * 2;        // of its keys (or values)
    static constexpr int ST = 2 * BYTES * 3 <= 98304 ? 3 : 2;  // ring of tiles
    static constexpr int UNITS = 2 * (KT / 16) / NW;  // 16-row copies of a wave
    static constexpr int DPW = UNITS * (D / 32);      // copy instructions of a wave and tile
    static constexpr int RING = ST * 2 * BYTES;
    // the merge of WK waves' sums reuses the ring
    static_assert((WK - 1) * WR * 64 * (D / 32) * 16 * 4 <= RING, "merge space");
    static constexpr int LDS = RING + IDS * 4 + NW * 32;
};

// Rows [r0, r0 + 32 WR) of [ra, rb) (row r of a kv head: head r % g, token r /
// g), positions [plo, phi), part `part` of `parts`, results to column `col`.
template <int D, int WR, int WK>
DEV void attn_task(const AttnArgs& A, uint8_t* lds, int kvh, int r0, int rb, int plo, int phi, const int* trow,
                   int part, int parts, int col) {
    using T = Tile<D, WR, WK>;
    constexpr int ROWB = D * 2, STEPS = D / 16, MT = D / 32, CH = D / 8;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave % WR, wk = wave / WR;
    const int half = lane >> 5;
    int* ids = reinterpret_cast<int*>(lds + T::RING);
    int* red = ids + IDS;  // per wave 8 ints

    // ---- this lane's row
    const int g = A.q_heads / A.kv_heads;
    const int r = r0 + 32 * wr + (lane & 31);
    const bool valid = r < rb;
    const int sj = (valid ? r : r0) / g, s = sj / A.n_new;
    const int len = A.lens[s], pos = len + (sj - s * A.n_new);
    int hi = min(min(pos + 1, phi), A.table_stride << A.page_shift);
    int lo = max(plo, A.window ? pos + 1 - A.window : 0);
    const bool live = valid && len >= 0 && lo < hi;
    const size_t qrow = (size_t)sj * A.q_heads + kvh * g + ((valid ? r : r0) - sj * g);
    h8 qf[STEPS];
    {
        const uint16_t* qp = A.q + qrow * D + 8 * half;
#pragma unroll
        for (int i = 0; i < STEPS; i++) {
            uint4 v = *reinterpret_cast<const uint4*>(qp + 16 * i);
            if (!live) v = make_uint4(0, 0, 0, 0);
            qf[i] = __builtin_bit_cast(h8, v);
        }
    }
    // ---- the positions that rows of the workgroup see: any of [lo, hi), all of
    // [lo_all, hi_all)
    int lo_any = live ? lo : 0x7fffffff, hi_any = live ? hi : 0, lo_all = live ? lo : 0, hi_all = live ? hi : 0x7fffffff;
    if (!live) lo = 0, hi = 0x7fffffff;  // masked by its l at the end
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        lo_any = min(lo_any, __shfl_xor(lo_any, o));
        hi_any = max(hi_any, __shfl_xor(hi_any, o));
        lo_all = max(lo_all, __shfl_xor(lo_all, o));
        hi_all = min(hi_all, __shfl_xor(hi_all, o));
    }
    if (WR > 1) {
        if (lane == 0) red[8 * wave] = lo_any, red[8 * wave + 1] = hi_any, red[8 * wave + 2] = lo_all, red[8 * wave + 3] = hi_all;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WR; w++) {
            lo_any = min(lo_any, red[8 * w]);
            hi_any = max(hi_any, red[8 * w + 1]);
            lo_all = max(lo_all, red[8 * w + 2]);
            hi_all = min(hi_all, red[8 * w + 3]);
        }
    }
    lo_any = __builtin_amdgcn_readfirstlane(lo_any);
    hi_any = __builtin_amdgcn_readfirstlane(hi_any);
    lo_all = __builtin_amdgcn_readfirstlane(lo_all);
    hi_all = __builtin_amdgcn_readfirstlane(hi_all);
    const int base = lo_any & ~15;
    const int tiles = hi_any > lo_any ? (hi_any - base + T::KT - 1) / T::KT : 0;
    const int each = (tiles + parts - 1) / parts;
    const int t0 = min(part * each, tiles), t1 = min(t0 + each, tiles);

    f16v o[MT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[m][i] = 0.f;
    float m = LOWEST, l = 0.f;

    // ---- copies: unit u of this wave is 16 rows of keys or values, a page
    // holds them all; rows that no one sees are replaced by the nearest that
    // someone does, so that what they hold is never multiplied
    const int page = 1 << A.page_shift;
    int ids_from = -IDS;  // first page of the ids in LDS
    auto fill_ids = [&](int first) {
        // all waves are past their last use of the ids (barrier before)
        for (int i = threadIdx.x; i < IDS; i += 64 * T::NW) {
            const int e = min(first + i, A.table_stride - 1);
            ids[i] = (int)min((unsigned)max(trow[e], 0), (unsigned)A.n_pages - 1u);
        }
        ids_from = first;
    };
    auto page_of = [&](int p) { return min(max(p, lo_any), hi_any - 1) >> A.page_shift; };
    auto issue = [&](int t) {
        const uint32_t dst = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + (uint32_t)(t % T::ST) * (2 * T::BYTES);
#pragma unroll
        for (int u = 0; u < T::UNITS; u++) {
            const int unit = wave * T::UNITS + u;
            const bool isv = unit >= T::KT / 16;
            const int grp = isv ? unit - T::KT / 16 : unit;
            const int p0 = base + t * T::KT + 16 * grp;
            const int id = __builtin_amdgcn_readfirstlane(ids[page_of(p0) - ids_from]);
            const uint16_t* src = (isv ? A.vp : A.kp) + ((size_t)id * A.kv_heads + kvh) * page * D;
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
                const int row = c * (64 / CH) + lane / CH, w = lane % CH;  // row of 16, stored word
                const int p = min(max(p0 + row, lo_any), hi_any - 1) & (page - 1);
                int f;
                if (D == 128) f = isv ? ((row & 3) << 2 | row >> 2) : row;
                else f = isv ? ((row >> 1 & 1) << 2 | row >> 2) : row >> 1;
                dma16(src + (size_t)p * D + 8 * (w ^ f), dst + (isv ? T::BYTES : 0) + (uint32_t)(grp * 16 * ROWB + c * 1024));
            }
        }
    };

    if (t0 < t1) {
        __syncthreads();
        fill_ids(page_of(base + t0 * T::KT));
        __syncthreads();
        // first tile whose pages are not in LDS
        auto beyond = [&](int t) { return page_of(base + (t + 1) * T::KT - 1) - ids_from >= IDS; };
#pragma unroll
        for (int i = 0; i < T::ST - 1; i++)
            if (t0 + i < t1) issue(t0 + i);
        for (int t = t0; t < t1; t++) {
            if (t + T::ST - 2 < t1) wait_vm<(T::ST - 2) * T::DPW>();
            else wait_vm<0>();
            barrier();
            if (t + T::ST - 1 < t1) {
                if (beyond(t + T::ST - 1)) {
                    fill_ids(page_of(base + (t + T::ST - 1) * T::KT));
                    __syncthreads();
                }
                issue(t + T::ST - 1);
            }
            const uint8_t* K = lds + (t % T::ST) * (2 * T::BYTES);
            const uint8_t* V = K + T::BYTES;
            const int kw = wk * 32 * T::KB;  // this wave's keys of the tile
            f16v sc[T::KB];
#pragma unroll
            for (int b = 0; b < T::KB; b++) {
#pragma unroll
                for (int i = 0; i < 16; i++) sc[b][i] = 0.f;
                const int row = lane & 31, fk = D == 128 ? row & 15 : row >> 1 & 7;
                const uint8_t* kr = K + (kw + 32 * b + row) * ROWB;
#pragma unroll
                for (int i = 0; i < STEPS; i++) {
                    const h8 kf = *reinterpret_cast<const h8*>(kr + ((2 * i + half) ^ fk) * 16);
                    sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[i], sc[b], 0, 0, 0);
                }
            }
            const int p0 = base + t * T::KT;
            if (p0 < lo_all || p0 + T::KT > hi_all) {
#pragma unroll
                for (int b = 0; b < T::KB; b++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int p = p0 + kw + 32 * b + (i & 3) + 8 * (i >> 2) + 4 * half;
                        sc[b][i] = p >= lo && p < hi ? sc[b][i] : -INFINITY;
                    }
            }
            // ---- running maximum and sum
            float mx = sc[0][0];
#pragma unroll
            for (int b = 0; b < T::KB; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) mx = fmaxf(mx, sc[b][i]);
            const f2 hm = halves(mx);
            mx = fmaxf(hm[0], hm[1]) * A.scale2;
            if (__any(mx > m + RAISE)) {
                const float mn = mx > m + RAISE ? mx - ABOVE : m;
                const float a = __builtin_amdgcn_exp2f(m - mn);
                l *= a;
#pragma unroll
                for (int x = 0; x < MT; x++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[x][i] *= a;
                m = mn;
            }
            h8 pf[T::KB * 2];
#pragma unroll
            for (int b = 0; b < T::KB; b++)
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const float e0 = __builtin_amdgcn_exp2f(fmaf(sc[b][i], A.scale2, -m));
                    const float e1 = __builtin_amdgcn_exp2f(fmaf(sc[b][i + 1], A.scale2, -m));
                    l += e0 + e1;
                    const h2 v = __builtin_convertvector((f2{e0, e1}), h2);
                    pf[2 * b + (i >> 3)][i & 7] = v[0];
                    pf[2 * b + (i >> 3)][(i & 7) + 1] = v[1];
                }
            // ---- O^T += V^T P^T
            const int gi = lane >> 4, li = lane & 15;
            typedef __attribute__((address_space(3))) s4* lp;
            __attribute__((address_space(3))) uint8_t* V3 = (__attribute__((address_space(3))) uint8_t*)V;
#pragma unroll
            for (int b = 0; b < 2 * T::KB; b++)
#pragma unroll
                for (int x = 0; x < MT; x++) {
                    s4 vv[2];
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const int row = 16 * b + 8 * u + 4 * half + (li >> 2);  // key of the wave's
                        const int word = 4 * x + 2 * (gi & 1) + ((li & 3) >> 1);
                        const int f = D == 128 ? ((li >> 2) << 2 | 2 * u + half) : ((li >> 3) << 2 | 2 * u + half);
                        vv[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (lp)(V3 + (kw + row) * ROWB + ((word ^ f) * 16 + (li & 1) * 8)));
                    }
                    typedef short s8 __attribute__((ext_vector_type(8)));
                    const s8 vf = __builtin_shufflevector(vv[0], vv[1], 0, 1, 2, 3, 4, 5, 6, 7);
                    o[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, vf), pf[b], o[x], 0, 0, 0);
                }
        }
    }
    const f2 hl = halves(l);
    l = hl[0] + hl[1];

    // ---- waves that shared rows: sums brought to the largest maximum and
    // added in wave order
    if (WK > 1) {
        float* mm = reinterpret_cast<float*>(red);  // [NW][8]: not enough for 32 rows, so in the ring
        (void)mm;
        __syncthreads();
        float* ro = reinterpret_cast<float*>(lds);
        constexpr int N = MT * 16;
        // {m, l} of a wave's rows through the ids' space
        f2* rm = reinterpret_cast<f2*>(ids);
        if (half == 0) rm[(wk * WR + wr) * 32 + (lane & 31)] = f2{m, l};
        __syncthreads();
        float M = LOWEST;
#pragma unroll
        for (int w = 0; w < WK; w++) M = fmaxf(M, rm[(w * WR + wr) * 32 + (lane & 31)][0]);
        const float a = __builtin_amdgcn_exp2f(m - M);
        float L = 0.f;
#pragma unroll
        for (int w = 0; w < WK; w++) {
            const f2 v = rm[(w * WR + wr) * 32 + (lane & 31)];
            L += v[1] * __builtin_amdgcn_exp2f(v[0] - M);
        }
        if (wk > 0) {
            float* to = ro + (size_t)((wk - 1) * WR + wr) * N * 64 + lane;
#pragma unroll
            for (int x = 0; x < MT; x++)
#pragma unroll
                for (int i = 0; i < 16; i++) to[(x * 16 + i) * 64] = o[x][i] * a;
        }
        __syncthreads();
        if (wk > 0) return;
#pragma unroll
        for (int x = 0; x < MT; x++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[x][i] *= a;
#pragma unroll
        for (int w = 1; w < WK; w++) {
            const float* from = ro + (size_t)((w - 1) * WR + wr) * N * 64 + lane;
#pragma unroll
            for (int x = 0; x < MT; x++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[x][i] += from[(x * 16 + i) * 64];
        }
        m = M;
        l = L;
    }
    if (!valid) return;
    const bool some = live && t0 < t1;
    const int all = A.prefix_parts + A.own_parts;
    if (all == 1) {
        // nothing to join: the result, rounded once
        const float inv = some && l != 0.f ? 1.f / l : 0.f;
        uint16_t* to = A.out + qrow * D + 4 * half;
#pragma unroll
        for (int x = 0; x < MT; x++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                uint2 w = make_uint2(0, 0);
                if (some) w = make_uint2(f2h2(o[x][i] * inv, o[x][i + 1] * inv), f2h2(o[x][i + 2] * inv, o[x][i + 3] * inv));
                *reinterpret_cast<uint2*>(to + 32 * x + 2 * i) = w;
            }
        return;
    }
    if (half == 0) A.ml[qrow * all + col] = f2{some ? m : LOWEST, some ? l : 0.f};
    if (!some) return;
    float* to = A.acc + (qrow * all + col) * D + 4 * half;
#pragma unroll
    for (int x = 0; x < MT; x++)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<float4*>(to + 32 * x + 2 * i) = make_float4(o[x][i], o[x][i + 1], o[x][i + 2], o[x][i + 3]);
}

// Prefix tasks.  Workgroups go to the XCDs in turn; the row tiles of one range
// of one kv head follow each other on the same XCD, so that all but the first
// find its pages in that XCD's L2.
template <int D, int WR, int WK>
DEV void attn_prefix_body(const AttnArgs& A, uint8_t* lds) {
    const int slot = blockIdx.x >> 3, xcd = blockIdx.x & 7;
    const int grp = slot / A.row_tiles * 8 + xcd, tile = slot % A.row_tiles;
    if (grp >= A.kv_heads * A.prefix_parts) return;
    const int kvh = grp / A.prefix_parts, part = grp % A.prefix_parts;
    const int rows = A.seqs * A.n_new * (A.q_heads / A.kv_heads);
    attn_task<D, WR, WK>(A, lds, kvh, tile * 32 * WR, rows, 0, A.prefix_pages << A.page_shift,
                         A.table + (size_t)A.prefix_slot * A.table_stride, part, A.prefix_parts, part);
}
// Own tasks: one slot's rows, 32 at a time.
template <int D, int WK>
DEV void attn_own_body(const AttnArgs& A, uint8_t* lds) {
    const int rows = A.n_new * (A.q_heads / A.kv_heads), tiles = (rows + 31) / 32;
    int b = blockIdx.x;
    const int part = b % A.own_parts;
    b /= A.own_parts;
    const int tile = b % tiles;
    b /= tiles;
    const int kvh = b % A.kv_heads, s = b / A.kv_heads;
    attn_task<D, 1, WK>(A, lds, kvh, s * rows + tile * 32, (s + 1) * rows, A.prefix_pages << A.page_shift, 0x7fffffff,
                        A.table + (size_t)s * A.table_stride, part, A.own_parts, A.prefix_parts + part);
}
#define ATTN_PREFIX(D, WR, WK)                                                                                       \
    extern "C" __global__ __launch_bounds__(64 * WR * WK) void cima_attn_paged_prefix_d##D##_r##WR##k##WK(           \
        const AttnArgs A) {                                                                                          \
        extern __shared__ __align__(1024) uint8_t lds[];                                                             \
        attn_prefix_body<D, WR, WK>(A, lds);                                                                         \
    }
#define ATTN_OWN(D, WK)                                                                                              \
    extern "C" __global__ __launch_bounds__(64 * WK) void cima_attn_paged_own_d##D##_k##WK(const AttnArgs A) {       \
        extern __shared__ __align__(1024) uint8_t lds[];                                                             \
        attn_own_body<D, WK>(A, lds);                                                                                \
    }
#define ATTN_ALL(D)         \
    ATTN_PREFIX(D, 1, 4)    \
    ATTN_PREFIX(D, 2, 2)    \
    ATTN_PREFIX(D, 4, 1)    \
    ATTN_PREFIX(D, 8, 1)    \
    ATTN_OWN(D, 4)
ATTN_ALL(64)
ATTN_ALL(128)

// The parts of a row joined: out = sum_c 2^(m_c - M) acc_c / sum_c 2^(m_c - M)
// l_c.  D / 4 threads a row, four elements each.  A row without any part (a
// slot not in use) becomes zeros.
template <int D>
DEV void attn_join_body(const float* __restrict__ acc, const f2* __restrict__ ml, uint16_t* __restrict__ out, int rows,
                        int parts) {
    constexpr int TR = D / 4;
    const int r = blockIdx.x * (256 / TR) + threadIdx.x / TR, e = threadIdx.x % TR * 4;
    if (r >= rows) return;
    const f2* p = ml + (size_t)r * parts;
    const float* a = acc + (size_t)r * parts * D + e;
    float M = LOWEST;
    for (int c = 0; c < parts; c++) M = fmaxf(M, p[c][0]);
    float L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = 0; c < parts; c++) {
        const f2 v = p[c];
        if (v[1] == 0.f) continue;  // nothing seen there, acc is not written
        const float w = __builtin_amdgcn_exp2f(v[0] - M);
        const float4 x = *reinterpret_cast<const float4*>(a + (size_t)c * D);
        L += v[1] * w;
        o.x += x.x * w;
        o.y += x.y * w;
        o.z += x.z * w;
        o.w += x.w * w;
    }
    const float inv = L != 0.f ? 1.f / L : 0.f;
    *reinterpret_cast<uint2*>(out + (size_t)r * D + e) = make_uint2(f2h2(o.x * inv, o.y * inv), f2h2(o.z * inv, o.w * inv));
}
extern "C" __global__ __launch_bounds__(256) void cima_attn_paged_join_d64(const float* __restrict__ acc,
                                                                           const f2* __restrict__ ml,
                                                                           uint16_t* __restrict__ out, int rows,
                                                                           int parts) {
    attn_join_body<64>(acc, ml, out, rows, parts);
}
extern "C" __global__ __launch_bounds__(256) void cima_attn_paged_join_d128(const float* __restrict__ acc,
                                                                            const f2* __restrict__ ml,
                                                                            uint16_t* __restrict__ out, int rows,
                                                                            int parts) {
    attn_join_body<128>(acc, ml, out, rows, parts);
}
