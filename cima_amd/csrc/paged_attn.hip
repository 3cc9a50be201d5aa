// Attention of a batch over a paged KV cache for gfx950 (CDNA4): the code
// object cima_paged_attn.hsaco.
//
// out = sum_t w_t v_t / sum_t w_t, w_t = e^(scale q.k_t - m), over the positions
// t that a row sees.  The rows of a kv head are its query heads times the
// step's tokens; those of all slots share the prefix's pages, so one workgroup
// takes up to 128 of them through a range of the prefix and its keys and values
// are read once for all (prefix tasks).  A slot's own pages are seen by its own
// rows alone (own tasks).  Both take a tile of rows through a range of positions
// and leave {m, l, sum} per row, which a second launch joins; a row's only part
// is its result.
//
// Rounding: q, keys and values are f16 as given; scores, maxima, sums of weights
// and of values are fp32.  The weights are rounded to f16 for the second product,
// by at most 2^-11 of each, their sum l is not: an error of at most 2^-11 of sum
// w |v| / sum w, as the result's own rounding.  Partial sums stay fp32.
//
// Both products of a row tile run on the matrix cores with 32 x 32 x 16 f16 MFMA.  S^T = K
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

#include <type_traits>

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef float f2 __attribute__((ext_vector_type(2)));

// every lane copies the 16 bytes at g to LDS byte lds + 16 * lane; written in
// asm so that the compiler's wait counting leaves the copies alone (their
// waits are explicit)
DEV void dma16(const void* g, uint32_t lds) {
    asm volatile("global_load_lds_dwordx4 %0, off" ::"v"(g), "{m0}"(__builtin_amdgcn_readfirstlane(lds)) : "memory");
}
// the same with a wave-uniform address and a byte offset per lane
DEV void dma16(const void* base, uint32_t off, uint32_t lds) {
    asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(__builtin_amdgcn_readfirstlane(lds))
                 : "memory");
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

// maximum over the four lanes that hold a row of a 16-row block (lanes 16 apart)
DEV float quarters_max(float v) {
    const f2 h = halves(v);
    const uint32_t x = __builtin_bit_cast(uint32_t, fmaxf(h[0], h[1]));
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    const uint32_t a = r[0], b = r[1];
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
DEV float quarters_sum(float v) {
    const f2 h = halves(v);
    const uint32_t x = __builtin_bit_cast(uint32_t, h[0] + h[1]);
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    const uint32_t a = r[0], b = r[1];
    return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}

// this lane, anew: where it is needed rarely, nothing made of it is kept in a
// register until then
DEV int lane_now() {
    int lane = __builtin_amdgcn_mbcnt_hi(-1, __builtin_amdgcn_mbcnt_lo(-1, 0));
    __asm__ volatile("" : "+v"(lane));
    return lane;
}

// minimum over aligned groups of 16 lanes
template <int CTRL>
DEV int dpp_min(int v) {
    return min(v, __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, false));
}
DEV int min16(int v) {
    v = dpp_min<0xB1>(v);      // quad_perm [1,0,3,2]
    v = dpp_min<0x4E>(v);      // quad_perm [2,3,0,1]
    v = dpp_min<0x141>(v);     // row_half_mirror
    return dpp_min<0x140>(v);  // row_mirror
}
DEV int max16(int v) { return -min16(-v); }

// Values of positions that have no page (a table entry that is no page's id) or
// lie between the windows of a task's rows: their scores are masked, and a weight
// of 0 multiplies what is read for them.
__device__ const uint4 no_page[256 * 128 * 2 / 16] = {};

struct AttnArgs {
    const uint16_t* q;
    const uint16_t* kp;  // planes of the layer
    const uint16_t* vp;
    const int* table;
    const int* lens;
    uint16_t* out;
    // partial sums, R = seqs * n_new * q_heads / kv_heads rows of a kv head: {m,
    // l} of (part, kv head, row) at ml[(part * kv_heads + head) * R + row]; the
    // sums of a tile of rows [r0, r0 + cols) from acc + ((part * kv_heads + head)
    // * R + r0) * D on, four elements d of all its rows after the other ([D /
    // 4][cols][4]), which is how the matrix cores leave them
    float* acc;
    f2* ml;
    int seqs, n_new, q_heads, kv_heads, page_shift, n_pages, table_stride;
    int prefix_pages, prefix_slot, window;
    int prefix_parts, own_parts, row_tiles;  // row tiles of the prefix tasks
    int prefix_tile, own_tile;               // their rows, and those of the own tasks
    int prefix_wgs;                          // workgroups of prefix tasks
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
    static constexpr int KB = WK == 1 && WR > 1 ? 2 : 1;  // 32-key blocks of a wave
    static constexpr int KT = 32 * KB * WK;         // keys of a tile
    static constexpr int BYTES = KT * D * 2;        // of its keys (or values)
    static_assert(KT == 16 * NW, "a wave copies 16 rows of keys and of values");
    static constexpr int RING = 2 * 2 * BYTES;        // two tiles: one being read, one on its way
    // the merge of WK waves' sums reuses the ring
    static_assert(WK == 1 || (WK - 1) * WR * 64 * (D / 32) * 16 * 4 <= RING, "merge space");
    static constexpr int LDS = RING + IDS * 4 + NW * 32 + WR * 32 * 8;
    static_assert(LDS <= 80 * 1024, "two workgroups to a CU");
};

// Rows [r0, r0 + 32 WR) of [0, rb) (row r of a kv head: head r % g, token r /
// g), positions [plo, phi), part `part` of `parts`, results to column `col`.
//
// 64 positions a tile, two tiles in LDS (64 KB), two workgroups of four waves to
// a CU: 250 registers hold 32 rows' sums, two tiles' scores and q, and the two
// workgroups cover each other's barriers.  Measured on MI355X, 128 slots of 4 x 8
// heads of 128 over 65536 positions (137 GFLOP): 153 us, 899 TFLOP/s, the matrix
// cores 0.47 busy at the 1.9 GHz that the card holds under this load.  No one part
// bounds it: of 155 us, without the copies 133, without reads from LDS 123, without
// the weights 138, with the products alone 85; reading fragments 2 to 8 products
// ahead changes nothing.  One workgroup of eight waves and 256 rows, which copies half
// as much: 176; 64 rows a wave: 572, its registers spill.
template <int D, int WR, int WK>
DEV void attn_task(const AttnArgs& A, uint8_t* lds, int kvh, int r0, int rb, int plo, int phi, const int* trow,
                   int part, int parts, int col) {
    using T = Tile<D, WR, WK>;
    constexpr int ROWB = D * 2, STEPS = D / 16, MT = D / 32, CH = D / 8;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave % WR, wk = wave / WR;
    const int half = lane >> 5;
    int* ids = reinterpret_cast<int*>(lds + T::RING);
    int* red = ids + IDS;  // per wave 8 ints; [4]: an id of the task names no page
    int2* span = reinterpret_cast<int2*>(red + 8 * T::NW);  // the positions that each row sees
    if (threadIdx.x == 0) red[4] = 0;

    // the ids of pages about where the part begins if all of [plo, phi) is seen, a
    // page a thread, fetched before the lengths are known
    const int guess =
        max(0, (plo + ((phi - plo + T::KT - 1) / T::KT + parts - 1) / parts * part * T::KT >> A.page_shift) - 64);
    const int guess_id = trow[min(guess + (int)threadIdx.x, A.table_stride - 1)];
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
    if (wk == 0 && half == 0) span[32 * wr + lane] = live ? make_int2(lo, hi) : make_int2(0, 0);
    if (!live) lo = 0, hi = 0x7fffffff;  // masked by its l at the end
    lo_any = min16(lo_any), hi_any = max16(hi_any), lo_all = max16(lo_all), hi_all = min16(hi_all);
    lo_any = min(lo_any, __builtin_amdgcn_readlane(lo_any, 16));
    hi_any = max(hi_any, __builtin_amdgcn_readlane(hi_any, 16));
    lo_all = max(lo_all, __builtin_amdgcn_readlane(lo_all, 16));
    hi_all = min(hi_all, __builtin_amdgcn_readlane(hi_all, 16));
    lo_any = __builtin_amdgcn_readfirstlane(lo_any);
    hi_any = __builtin_amdgcn_readfirstlane(hi_any);
    lo_all = __builtin_amdgcn_readfirstlane(lo_all);
    hi_all = __builtin_amdgcn_readfirstlane(hi_all);
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

    // ---- copies: a wave brings 16 rows of a tile's keys and of its values, which
    // a page holds all; rows that no one sees are replaced by the nearest that
    // someone does, so that what they hold is never multiplied, and values without
    // a page by zeros.  Where the rows have no position in common their windows may
    // lie apart (slots that end within the prefix): values that none sees are zeros
    const int page = 1 << A.page_shift;
    auto page_of = [&](int p) { return min(max(p, lo_any), hi_any - 1) >> A.page_shift; };
    int ids_from = -IDS;  // first page of the ids in LDS
    auto fill_ids = [&](int first, auto begin) {
        // all waves are past their last use of the ids (barrier before)
        const int n = min(IDS, page_of(base + t1 * T::KT - 1) - first + 1);
        auto put = [&](int i, int id) {
            const bool none = (unsigned)id >= (unsigned)A.n_pages;
            ids[i] = none ? -1 : id;
            if (none) red[4] = 1;
        };
        if (begin && first >= guess && first + n <= guess + 64 * T::NW) {
            const int i = guess + (int)threadIdx.x - first;
            if (i >= 0 && i < n) put(i, guess_id);
        } else {
            for (int i = 64 * wave + lane_now(); i < n; i += 64 * T::NW) put(i, trow[first + i]);
        }
        ids_from = first;
    };
    // A copy instruction c takes 1024 bytes of the 16 rows: this lane's row and
    // 16-byte word of the stored order.  Word w of row r holds the row's word w ^
    // f(r) -- keys: f = r (D = 64: r / 2), so that 16 rows' reads of one word
    // spread over the banks; values: f = r % 4 * 4 + r / 4 (D = 64: r / 2 % 2 * 4 +
    // r / 4), so that four rows' transposing reads of four words do.  c enters by
    // an exclusive or of constants.
    const int lrow = lane / CH, lword = lane % CH;
    const uint32_t kword = (uint32_t)(lword ^ (D == 128 ? lrow : lrow >> 1)) * 16;
    const uint32_t vword = (uint32_t)(lword ^ (D == 128 ? lrow << 2 : ((lrow >> 1 & 1) << 2 | lrow >> 2))) * 16;
    constexpr uint32_t KX = 64, VX = D == 128 ? 16 : 32;
    const size_t page_elems = (size_t)A.kv_heads * page * D;
    const uint16_t* kplane = A.kp + (size_t)kvh * page * D;
    const uint16_t* vplane = A.vp + (size_t)kvh * page * D;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + wave * 16 * ROWB;
    auto id_at = [&](int t) { return ids[page_of(base + t * T::KT + 16 * wave) - ids_from]; };
    auto issue = [&](int t, int id, const uint16_t* plane, uint32_t word, uint32_t flip, uint32_t ring) {
        const int p0 = base + t * T::KT + 16 * wave;
        id = __builtin_amdgcn_readfirstlane(id);
        const uint16_t* src = plane + (size_t)max(id, 0) * page_elems;
        if (ring && id < 0) src = reinterpret_cast<const uint16_t*>(no_page);
        const uint32_t dst = lds0 + ring + (uint32_t)(t & 1) * T::BYTES;
        if (p0 >= lo_any && p0 + 16 <= hi_any) {
            src += (size_t)(p0 & (page - 1)) * D;
#pragma unroll
            for (int c = 0; c < D / 32; c++)
                dma16(src, (((uint32_t)lrow * ROWB + word) ^ c * flip) + c * 1024, dst + c * 1024);
        } else {
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
                const int p = min(max(p0 + c * (64 / CH) + lrow, lo_any), hi_any - 1) & (page - 1);
                dma16(src, (uint32_t)p * ROWB + (word ^ c * flip), dst + c * 1024);
            }
        }
    };
    // the wave's 16 rows of tile t's values, which have arrived: zeros where none of
    // the workgroup's rows sees the position
    auto clear = [&](int t) {
        const int ln = lane_now();
        const int2 a = span[ln & (32 * WR - 1)], b = span[(64 + ln) & (32 * WR - 1)];
        uint32_t seen = 0;  // bit i: position p0 + i
        for (int i = 0, p = base + t * T::KT + 16 * wave; i < 16; i++, p++)
            if (__ballot((a.x <= p && p < a.y) || (b.x <= p && p < b.y))) seen |= 1u << i;
        uint4* v = reinterpret_cast<uint4*>(lds + 2 * T::BYTES + (t & 1) * T::BYTES + wave * 16 * ROWB) + ln;
#pragma unroll
        for (int c = 0; c < D / 32; c++)
            if (!(seen >> (c * (64 / CH) + ln / CH) & 1)) v[64 * c] = make_uint4(0, 0, 0, 0);
    };
    const int kw = wk * 32 * T::KB;  // this wave's keys of a tile
    f16v zero16;
#pragma unroll
    for (int i = 0; i < 16; i++) zero16[i] = 0.f;
    // fragments of keys and of transposed values: one address a lane each, the
    // rest enters by an exclusive or and an offset
    const int gi = lane >> 4, li = lane & 15, krow = lane & 31;
    const uint32_t lbase = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    const uint32_t kread = lbase + (kw + krow) * ROWB + (half ^ (D == 128 ? krow & 15 : krow >> 1 & 7)) * 16;
    const uint32_t vread = lbase + 2 * T::BYTES + (kw + 4 * half + (li >> 2)) * ROWB + (li & 1) * 8 +
                           ((2 * (gi & 1) + ((li & 3) >> 1)) ^ ((D == 128 ? li >> 2 : li >> 3) << 2 | half)) * 16;
    typedef short s8 __attribute__((ext_vector_type(8)));
    typedef __attribute__((address_space(3))) s4* s4p;
    typedef const __attribute__((address_space(3))) h8* h8p;
    auto kfrag = [&](uint32_t at, int i) {
        return *(h8p)(uintptr_t)((at ^ i / T::KB * 32) + (i % T::KB) * 32 * ROWB);
    };
    auto vfrag = [&](uint32_t at, int n) {
        const int b = n / MT, x = n % MT;
        const s4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s4p)(uintptr_t)((at ^ x * 64) + 16 * b * ROWB));
        const s4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s4p)(uintptr_t)((at ^ x * 64 ^ 32) + (16 * b + 8) * ROWB));
        const s8 v = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(h8, v);
    };
    // the scores of tile t that a row does not see, or that have no page, become
    // -inf; the largest left
    bool holes = false;  // an id among those that were in LDS names no page
    auto mask = [&](int t, f16v (&sc)[T::KB]) {
        const int p0 = base + t * T::KT;
        int end[2 * T::KB];  // of the wave's 16 keys from 16 j on
#pragma unroll
        for (int j = 0; j < 2 * T::KB; j++) end[j] = hi;
        if (holes) {
#pragma unroll
            for (int j = 0; j < 2 * T::KB; j++)
                if (ids[page_of(p0 + kw + 16 * j) - ids_from] < 0) end[j] = 0;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < T::KB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int p = p0 + kw + 32 * b + (i & 3) + 8 * (i >> 2) + 4 * half;
                sc[b][i] = p >= lo && p < end[2 * b + (i >> 3)] ? sc[b][i] : -INFINITY;
                mx = fmaxf(mx, sc[b][i]);
            }
        return mx;
    };
    auto raise = [&](float mx) {
        const f2 h = halves(mx);
        mx = fmaxf(h[0], h[1]) * A.scale2;
        if (!__any(mx > m + RAISE)) return;
        const float mn = mx > m + RAISE ? mx - ABOVE : m;
        const float a = __builtin_amdgcn_exp2f(m - mn);
        l *= a;
#pragma unroll
        for (int x = 0; x < MT; x++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[x][i] *= a;
        m = mn;
    };

    // The loop is two tiles deep, so that the exponentials of one tile run beside
    // the next one's products: the scores of tile t are there when its turn
    // begins, its values and the keys of tile t + 1 have arrived.  A short task (7
    // tiles of 64) spends 0.7 us on the lengths, 0.2 on the ids, 0.4 to 0.8 on the
    // first keys and 1 us a tile; around them stand the launch and, at its end, the
    // write-back of the partial sums (2.7 us for 6 MB).
    if (t0 < t1) {
        __syncthreads();
        fill_ids(page_of(base + t0 * T::KT), std::true_type{});
        __syncthreads();
        holes = __builtin_amdgcn_readfirstlane(red[4]);
        f16v sa[T::KB], sb[T::KB];  // scores of even and of odd tiles from t0 on
        int id = id_at(t0);
        // the first keys, waited for alone, the first values and the second keys
        issue(t0, id, kplane, kword, KX, 0);
        issue(t0, id, vplane, vword, VX, 2 * T::BYTES);
        if (t0 + 1 < t1) {
            id = id_at(t0 + 1);
            issue(t0 + 1, id, kplane, kword, KX, 0);
            wait_vm<2 * (D / 32)>();
        } else {
            wait_vm<D / 32>();
        }
        barrier();
        {
            const uint32_t kr = kread + (uint32_t)(t0 & 1) * T::BYTES;
#pragma unroll
            for (int b = 0; b < T::KB; b++) sa[b] = zero16;
#pragma unroll
            for (int i = 0; i < T::KB * STEPS; i++) {
                const int b = i % T::KB;
                sa[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kfrag(kr, i), qf[i / T::KB], sa[b], 0, 0, 0);
            }
        }
        raise(mask(t0, sa));
        // tile t, whose scores are in sc; those of the next go to sn
        auto turn = [&](int t, f16v (&sc)[T::KB], f16v (&sn)[T::KB]) {
            const bool more = t + 1 < t1;
            wait_vm<0>();
            if (lo_all > hi_all) clear(t);
            barrier();
            if (more) {
                issue(t + 1, id, vplane, vword, VX, 2 * T::BYTES);
                if (t + 2 < t1) {
                    if (page_of(base + (t + 3) * T::KT - 1) - ids_from >= IDS) {
                        fill_ids(page_of(base + (t + 1) * T::KT), std::false_type{});  // its mask looks them up
                        __syncthreads();
                        holes = __builtin_amdgcn_readfirstlane(red[4]);
                    }
                    id = id_at(t + 2);
                    issue(t + 2, id, kplane, kword, KX, 0);
                }
            }
            h8 pf[T::KB * 2];
            // two weights: elements i, i + 1 of block j / 8
            auto pair = [&](int j) {
                const int b = j / 8, i = j % 8 * 2;
                const float e0 = __builtin_amdgcn_exp2f(fmaf(sc[b][i], A.scale2, -m));
                const float e1 = __builtin_amdgcn_exp2f(fmaf(sc[b][i + 1], A.scale2, -m));
                l += e0 + e1;
                const h2 v = __builtin_convertvector((f2{e0, e1}), h2);
                pf[2 * b + (i >> 3)][i & 7] = v[0];
                pf[2 * b + (i >> 3)][(i & 7) + 1] = v[1];
            };
            // ---- the next tile's scores beside the first half of the weights
            // (behind the last tile LDS holds older keys: not used)
            {
                constexpr int N = T::KB * STEPS, AHEAD = 4, PAIRS = 4 * T::KB;
                const uint32_t kr = kread + (uint32_t)((t + 1) & 1) * T::BYTES;
                h8 kf[AHEAD];
                auto frag = [&](int i) { return kfrag(kr, i); };
#pragma unroll
                for (int i = 0; i < AHEAD; i++) kf[i] = frag(i);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const int b = i % T::KB;
                    if (i < T::KB)
                        sn[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i % AHEAD], qf[i / T::KB], zero16, 0, 0, 0);
                    else
                        sn[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i % AHEAD], qf[i / T::KB], sn[b], 0, 0, 0);
                    if (i + AHEAD < N) kf[i % AHEAD] = frag(i + AHEAD);
#pragma unroll
                    for (int j = i * PAIRS / N; j < (i + 1) * PAIRS / N; j++) pair(j);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            // ---- O^T += V^T P^T, beside the other weights and the next tile's
            // largest score
            const uint32_t vr = vread + (uint32_t)(t & 1) * T::BYTES;
            float mx = -INFINITY;
            {
                constexpr int N = 2 * T::KB * MT, AHEAD = 2;
                h8 vf[AHEAD];
#pragma unroll
                for (int i = 0; i < AHEAD; i++) vf[i] = vfrag(vr, i);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < N; i++) {
                    o[i % MT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[i % AHEAD], pf[i / MT], o[i % MT], 0, 0, 0);
                    if (i + AHEAD < N) vf[i % AHEAD] = vfrag(vr, i + AHEAD);
                    if (i < N / 2) {
#pragma unroll
                        for (int j = 0; j < 4 / MT + (4 % MT != 0); j++) pair(4 * T::KB + i * 4 / MT + j);
                    } else {
                        constexpr int E = 16 / MT;  // scores looked at beside a product
#pragma unroll
                        for (int j = (i - N / 2) * E; j < (i - N / 2 + 1) * E; j++) mx = fmaxf(mx, sn[j / 16][j % 16]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            __asm__ volatile("" : "+v"(mx));  // found beside the products, not behind them
            if (more) {
                const int p0 = base + (t + 1) * T::KT;
                if (p0 < lo_all || p0 + T::KT > hi_all || holes) mx = mask(t + 1, sn);
                raise(mx);
            }
        };
        for (int t = t0; t < t1; t += 2) {
            turn(t, sa, sb);
            if (t + 1 < t1) turn(t + 1, sb, sa);
        }
    }
    const f2 hl = halves(l);
    l = hl[0] + hl[1];

    // ---- waves that shared rows: sums brought to the largest maximum and
    // added in wave order
    if (WK > 1) {
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
    const int R = A.seqs * A.n_new * g;
    const size_t at = (size_t)(col * A.kv_heads + kvh) * R;
    const int c0 = r0 + 32 * wr, cols = min(32, rb - c0), ln = lane_now();
    if (ln < 32) A.ml[at + c0 + ln] = f2{some ? m : LOWEST, some ? l : 0.f};
    if (!some) return;
    float4* to = reinterpret_cast<float4*>(A.acc + (at + c0) * D) + (ln >> 5) * cols + (ln & 31);
#pragma unroll
    for (int x = 0; x < MT; x++)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            to[(8 * x + i / 2) * cols] = make_float4(o[x][i], o[x][i + 1], o[x][i + 2], o[x][i + 3]);
}

// ------------------------------------------------------------- few rows
//
// Tasks of up to 16 NB rows (own tasks; prefix tasks of up to 16 rows): bound by
// reading the keys and values, and short ones by the latency of their chain of
// loads (lengths, ids, pages).  The four waves of a workgroup take 32-position
// tiles in turn and do not wait for each other: keys go straight from memory
// to the registers of the A operand (16 x 16 x 32 MFMA: a lane holds 16 bytes
// of a key), values by direct copies to the wave's own LDS.  The waves' sums are
// added at the end, in wave order.  Rounding: the weights to f16, as in the row
// tiles; sums, maxima and the waves' joining are fp32.
//
// BUFS 2: a tile is on its way while the one before it is computed, 64 KB of LDS
// a workgroup, two of them to a CU.  BUFS 1: the loads of a tile are waited for,
// but the registers and LDS suffice for four workgroups to a CU, whose waves
// cover each other; it is taken where the launch holds nothing larger and more
// than two workgroups to a CU.
// Measured on MI355X, 8 kv heads of 128, one / two in flight: 64 slots of up
// to 4000 positions (524 MB) 107 / 146 us (4.9 TB/s), 128 of up to 500 27 / 33;
// 128 full slots of 8192 (4.3 GB) 765 us with the join, 5.6 TB/s.  Values by
// loads to registers and LDS writes: 127 and 36 us.
constexpr int few_bufs(int D, int mode, int nb) { return mode == 0 && !(D == 128 && nb == 2) ? 1 : 2; }
constexpr int few_wgs(int D, int mode, int nb) { return few_bufs(D, mode, nb) == 1 ? 4 : 2; }
constexpr int OWN_LEAST = 4;  // tiles that a part of an own task has at least, where there are
template <int D, int NB, int BUFS>
struct Few {
    static constexpr int VT = 32 * D * 2;                  // bytes of a tile's values
    static constexpr int OB = NB * (D / 16) * 64 * 16;     // of a wave's sums
    static constexpr int WAVE = BUFS * VT > OB ? BUFS * VT : OB;  // LDS of a wave
    static constexpr int LDS = 4 * WAVE + 4 * NB * 16 * 8;
    static_assert(LDS <= (BUFS == 1 ? 40 : 80) * 1024, "workgroups to a CU");
};
template <int D, int NB, int BUFS>
DEV void few_task(const AttnArgs& A, uint8_t* lds, int kvh, int r0, int rb, int plo, int phi, const int* trow, int part,
                  int parts, int col, int guess, int least, bool slots) {
    using F = Few<D, NB, BUFS>;
    constexpr int STEPS = D / 32, XT = D / 16, CH = D / 8;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, q4 = lane >> 4;
    const int g = A.q_heads / A.kv_heads;
    // the ids of the 64 pages that the part most likely begins with, fetched
    // before the lengths are known; lane i: id of page ids_from + i, -1: none
    auto fetch_ids = [&](int first) {
        const int id = trow[min(first + lane, A.table_stride - 1)];
        return (unsigned)id < (unsigned)A.n_pages ? id : -1;
    };
    int ids_from = guess, ids = fetch_ids(guess);
    // ---- this lane's rows
    bool valid[NB], live[NB];
    int lo[NB], hi[NB], len[NB], tok[NB];
    size_t qrow[NB];
    h8 qf[NB][STEPS];
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const int r = r0 + 16 * b + li;
        valid[b] = r < rb;
        const int rr = valid[b] ? r : r0, sj = rr / g, s = sj / A.n_new;
        len[b] = A.lens[s];
        tok[b] = sj - s * A.n_new;
        qrow[b] = (size_t)sj * A.q_heads + kvh * g + (rr - sj * g);
#pragma unroll
        for (int i = 0; i < STEPS; i++)
            qf[b][i] = *reinterpret_cast<const h8*>(A.q + qrow[b] * D + 32 * i + 8 * q4);
    }
    int lo_any = 0x7fffffff, hi_any = 0, lo_all = 0, hi_all = 0x7fffffff;
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const int pos = len[b] + tok[b];
        hi[b] = min(min(pos + 1, phi), A.table_stride << A.page_shift);
        lo[b] = max(plo, A.window ? pos + 1 - A.window : 0);
        live[b] = valid[b] && len[b] >= 0 && lo[b] < hi[b];
        if (live[b]) {
            lo_any = min(lo_any, lo[b]);
            hi_any = max(hi_any, hi[b]);
            lo_all = max(lo_all, lo[b]);
            hi_all = min(hi_all, hi[b]);
        } else {
            lo[b] = 0, hi[b] = 0x7fffffff;  // masked by its l at the end
        }
    }
    lo_any = __builtin_amdgcn_readfirstlane(min16(lo_any));
    hi_any = __builtin_amdgcn_readfirstlane(max16(hi_any));
    lo_all = __builtin_amdgcn_readfirstlane(max16(lo_all));
    hi_all = __builtin_amdgcn_readfirstlane(min16(hi_all));
    const int base = lo_any & ~15;
    const int tiles = hi_any > lo_any ? (hi_any - base + 31) / 32 : 0;
    const int each = max((tiles + parts - 1) / parts, least);
    const int t0 = min(part * each, tiles), t1 = min(t0 + each, tiles);

    f4 o[NB][XT];
    float m[NB], l[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) {
        m[b] = LOWEST, l[b] = 0.f;
#pragma unroll
        for (int x = 0; x < XT; x++) o[b][x] = f4{0.f, 0.f, 0.f, 0.f};
    }
    // ---- loads of a tile: two groups of 16 positions, each within a page; rows
    // that no one sees are replaced by the nearest that someone does, values
    // without a page by zeros, and where the windows of several slots' rows lie
    // apart what is between them too
    const int page = 1 << A.page_shift;
    const uint32_t vbase = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + wave * F::WAVE;
    h8 kf[BUFS][2][STEPS];
    uint32_t gone[BUFS];  // bit u: group u of the tile has no page
    auto issue = [&](int t, auto buf) {
        gone[buf] = 0;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int p0 = base + 32 * t + 16 * u;
            const int pg = min(max(p0, lo_any), hi_any - 1) >> A.page_shift;
            if ((unsigned)(pg - ids_from) >= 64u) {
                ids = fetch_ids(pg);
                ids_from = pg;
            }
            const int id = __builtin_amdgcn_readlane(ids, pg - ids_from);
            gone[buf] |= (uint32_t)id >> 31 << u;
            const size_t off = ((size_t)max(id, 0) * A.kv_heads + kvh) * page * D;
            uint32_t seen = 0xffff;  // bit i: position p0 + i
            if (slots && lo_all > hi_all) {
                seen = 0;
                for (int i = 0, p = p0; i < 16; i++, p++)
                    if (__ballot(live[0] && lo[0] <= p && p < hi[0])) seen |= 1u << i;
            }
            const uint16_t* vsrc = id < 0 ? reinterpret_cast<const uint16_t*>(no_page) : A.vp + off;
            const int pk = min(max(p0 + li, lo_any), hi_any - 1) & (page - 1);
#pragma unroll
            for (int i = 0; i < STEPS; i++)
                kf[buf][u][i] = *reinterpret_cast<const h8*>(A.kp + off + (size_t)pk * D + 32 * i + 8 * q4);
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
                const int row = c * (64 / CH) + lane / CH, w = lane % CH;
                const int p = min(max(p0 + row, lo_any), hi_any - 1) & (page - 1);
                const int f = D == 128 ? (row & 7) << 1 : (row >> 1 & 3) << 1;
                const uint16_t* at = vsrc + (size_t)p * D;
                if (slots && !(seen >> row & 1)) at = reinterpret_cast<const uint16_t*>(no_page);
                dma16(at + 8 * (w ^ f), vbase + buf * F::VT + u * 16 * D * 2 + c * 1024);
            }
        }
    };
    auto step = [&](int t, auto buf) {
        if constexpr (BUFS == 1) issue(t, buf);
        wait_vm<0>();
        if constexpr (BUFS == 2)
            if (t + 4 < t1) issue(t + 4, std::integral_constant<int, 1 - buf>{});
        const int p0 = base + 32 * t;
        __asm__ volatile("" : "+s"(gone[buf]));  // one path for the tile, by one test
        h8 pf[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            f4 sc[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                sc[u] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < STEPS; i++)
                    sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[buf][u][i], qf[b][i], sc[u], 0, 0, 0);
            }
            if (p0 < lo_all || p0 + 32 > hi_all || gone[buf]) {
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int end = gone[buf] >> u & 1 ? 0 : hi[b];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int p = p0 + 16 * u + 4 * q4 + i;
                        sc[u][i] = p >= lo[b] && p < end ? sc[u][i] : -INFINITY;
                    }
                }
            }
            float mx = sc[0][0];
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) mx = fmaxf(mx, sc[u][i]);
            mx = quarters_max(mx) * A.scale2;
            if (__any(mx > m[b] + RAISE)) {
                const float mn = mx > m[b] + RAISE ? mx - ABOVE : m[b];
                const float a = __builtin_amdgcn_exp2f(m[b] - mn);
                l[b] *= a;
#pragma unroll
                for (int x = 0; x < XT; x++) o[b][x] *= a;
                m[b] = mn;
            }
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float e0 = __builtin_amdgcn_exp2f(fmaf(sc[u][i], A.scale2, -m[b]));
                    const float e1 = __builtin_amdgcn_exp2f(fmaf(sc[u][i + 1], A.scale2, -m[b]));
                    l[b] += e0 + e1;
                    const h2 v = __builtin_convertvector((f2{e0, e1}), h2);
                    pf[b][4 * u + i] = v[0];
                    pf[b][4 * u + i + 1] = v[1];
                }
        }
        typedef __attribute__((address_space(3))) s4* lp;
        typedef short s8 __attribute__((ext_vector_type(8)));
#pragma unroll
        for (int x = 0; x < XT; x++) {
            s4 vv[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int row = 16 * u + 4 * q4 + (li >> 2), w = 2 * x + ((li & 3) >> 1);
                const int f = D == 128 ? (row & 7) << 1 : (row >> 1 & 3) << 1;
                vv[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lp)(uintptr_t)(vbase + buf * F::VT + row * D * 2 + (w ^ f) * 16 + (li & 1) * 8));
            }
            const s8 vf = __builtin_shufflevector(vv[0], vv[1], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
            for (int b = 0; b < NB; b++)
                o[b][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, vf), pf[b], o[b][x], 0, 0, 0);
        }
        // the next copies into this buffer follow the reads
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };
    using B0 = std::integral_constant<int, 0>;
    using B1 = std::integral_constant<int, 1>;
    int t = t0 + wave;
    if constexpr (BUFS == 1) {
        for (; t < t1; t += 4) step(t, B0{});
    } else if (t < t1) {
        issue(t, B0{});
        while (true) {
            step(t, B0{});
            if ((t += 4) >= t1) break;
            step(t, B1{});
            if ((t += 4) >= t1) break;
        }
    }
    // ---- the waves' sums, brought to the largest maximum
    f2* rm = reinterpret_cast<f2*>(lds + 4 * F::WAVE);
#pragma unroll
    for (int b = 0; b < NB; b++) {
        l[b] = quarters_sum(l[b]);
        if (q4 == 0) rm[(wave * NB + b) * 16 + li] = f2{m[b], l[b]};
    }
    __syncthreads();
    float M[NB], L[NB];
    float4* mine = reinterpret_cast<float4*>(lds + wave * F::WAVE);
#pragma unroll
    for (int b = 0; b < NB; b++) {
        M[b] = LOWEST, L[b] = 0.f;
#pragma unroll
        for (int w = 0; w < 4; w++) M[b] = fmaxf(M[b], rm[(w * NB + b) * 16 + li][0]);
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const f2 v = rm[(w * NB + b) * 16 + li];
            L[b] += v[1] * __builtin_amdgcn_exp2f(v[0] - M[b]);
        }
        const float a = __builtin_amdgcn_exp2f(m[b] - M[b]);
#pragma unroll
        for (int x = 0; x < XT; x++) {
            const f4 v = o[b][x] * a;
            mine[(b * XT + x) * 64 + lane] = make_float4(v[0], v[1], v[2], v[3]);
        }
    }
    __syncthreads();
    const int R = A.seqs * A.n_new * g, all = A.prefix_parts + A.own_parts, cols = min(16 * NB, rb - r0);
    const size_t at = (size_t)(col * A.kv_heads + kvh) * R;
#pragma unroll
    for (int b = 0; b < NB; b++) {
        if (!valid[b]) continue;
        const bool some = live[b] && t0 < t1;
        if (all > 1 && wave == 0 && q4 == 0) A.ml[at + r0 + 16 * b + li] = f2{some ? M[b] : LOWEST, some ? L[b] : 0.f};
        if (all > 1 && !some) continue;
        const float inv = some && L[b] != 0.f ? 1.f / L[b] : 0.f;
#pragma unroll
        for (int y = 0; y < XT / 4; y++) {
            const int x = wave * (XT / 4) + y;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float4 z = reinterpret_cast<const float4*>(lds + w * F::WAVE)[(b * XT + x) * 64 + lane];
                v.x += z.x, v.y += z.y, v.z += z.z, v.w += z.w;
            }
            if (all > 1) {
                reinterpret_cast<float4*>(A.acc + (at + r0) * D)[(4 * x + q4) * cols + 16 * b + li] = v;
            } else {  // nothing to join: the result, rounded once
                uint2 z = make_uint2(0, 0);
                if (some) z = make_uint2(f2h2(v.x * inv, v.y * inv), f2h2(v.z * inv, v.w * inv));
                *reinterpret_cast<uint2*>(A.out + qrow[b] * D + 16 * x + 4 * q4) = z;
            }
        }
    }
}
// One launch: first the prefix tasks (MODE 0: as few-row tasks, up to 16 rows; 1
// and 2: tiles of 64 and 128 rows), then the own tasks, one slot's rows 16 NB at
// a time, so that they fill what the prefix tasks leave.  Workgroups go to the XCDs in turn; the row tiles
// of one range of one kv head follow each other on the same XCD, so that all but
// the first find its pages in that XCD's L2.
template <int D, int MODE, int NB>
DEV void attn_body(const AttnArgs& A, uint8_t* lds) {
    constexpr int BUFS = few_bufs(D, MODE, NB);
    const int rows = A.n_new * (A.q_heads / A.kv_heads);
    int b = blockIdx.x;
    if (b < A.prefix_wgs) {
        const int slot = b >> 3, grp = slot / A.row_tiles * 8 + (b & 7), tile = slot % A.row_tiles;
        if (grp >= A.kv_heads * A.prefix_parts) return;
        const int kvh = grp / A.prefix_parts, part = grp % A.prefix_parts, phi = A.prefix_pages << A.page_shift;
        const int* trow = A.table + (size_t)A.prefix_slot * A.table_stride;
        if constexpr (MODE == 0 && NB == 1)
            few_task<D, NB, BUFS>(A, lds, kvh, 0, A.seqs * rows, 0, phi, trow, part, A.prefix_parts, part,
                            ((phi + 31) / 32 + A.prefix_parts - 1) / A.prefix_parts * part * 32 >> A.page_shift, 1, true);
        else if constexpr (MODE == 1)
            attn_task<D, 2, 2>(A, lds, kvh, tile * 64, A.seqs * rows, 0, phi, trow, part, A.prefix_parts, part);
        else if constexpr (MODE == 2)
            attn_task<D, 4, 1>(A, lds, kvh, tile * 128, A.seqs * rows, 0, phi, trow, part, A.prefix_parts, part);
        return;
    }
    b -= A.prefix_wgs;
    const int tiles = (rows + 16 * NB - 1) / (16 * NB);
    const int part = b % A.own_parts;
    b /= A.own_parts;
    const int tile = b % tiles;
    b /= tiles;
    const int kvh = b % A.kv_heads, s = b / A.kv_heads;
    few_task<D, NB, BUFS>(A, lds, kvh, s * rows + tile * 16 * NB, (s + 1) * rows, A.prefix_pages << A.page_shift, 0x7fffffff,
                    A.table + (size_t)s * A.table_stride, part, A.own_parts, A.prefix_parts + part, A.prefix_pages, OWN_LEAST, false);
}
#define ATTN(D, MODE, NB)                                                                                            \
    extern "C" __global__ __launch_bounds__(256, few_wgs(D, MODE, NB)) void cima_attn_paged_d##D##_m##MODE##_n##NB(const AttnArgs A) {  \
        extern __shared__ __align__(1024) uint8_t lds[];                                                             \
        attn_body<D, MODE, NB>(A, lds);                                                                              \
    }
#define ATTN_ALL(D) \
    ATTN(D, 0, 1)   \
    ATTN(D, 1, 1)   \
    ATTN(D, 2, 1)   \
    ATTN(D, 0, 2)   \
    ATTN(D, 1, 2)   \
    ATTN(D, 2, 2)
ATTN_ALL(64)
ATTN_ALL(128)

// The parts of a row joined: out = sum_c 2^(m_c - M) acc_c / sum_c 2^(m_c - M)
// l_c.  A workgroup takes 16 rows and 16 elements.  First all parts' {m, l} of
// the rows are read together and become weights in LDS, and the parts that any
// of the rows has are listed; then each wave sums every fourth of them, a lane
// four elements of a row, and the waves' sums are added in wave order.  A row
// without any part (a slot not in use) becomes zeros.
constexpr int MAX_PARTS = 192;
template <int D>
DEV void attn_join_body(const AttnArgs& A) {
    __shared__ float wt[MAX_PARTS][16], red[16][16];
    __shared__ int list[MAX_PARTS], count;
    __shared__ float4 ro[4][64];
    const int g = A.q_heads / A.kv_heads, rows = A.n_new * g, R = A.seqs * rows, all = A.prefix_parts + A.own_parts;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, li = lane & 15, q4 = lane >> 4;
    int b = blockIdx.x;
    const int x = b % (D / 16);
    b /= D / 16;
    const int rts = (R + 15) / 16, r = min(b % rts * 16 + li, R - 1), kvh = b / rts;
    const bool valid = b % rts * 16 + li < R;
    const size_t step = (size_t)A.kv_heads * R, head = (size_t)kvh * R;
    // where the row's elements 16 x + 4 q4 are in a prefix part and in an own part
    const int pr0 = r / A.prefix_tile * A.prefix_tile, pc = min(A.prefix_tile, R - pr0);
    const int s0 = r / rows * rows, or0 = s0 + (r - s0) / A.own_tile * A.own_tile, oc = min(A.own_tile, s0 + rows - or0);
    const float4* ap = reinterpret_cast<const float4*>(A.acc + (head + pr0) * D) + (4 * x + q4) * pc + (r - pr0);
    const float4* ao = reinterpret_cast<const float4*>(A.acc + (head + or0) * D) + (4 * x + q4) * oc + (r - or0);
    auto part = [&](int c) { return (c < A.prefix_parts ? ap : ao)[c * step * (D / 4)]; };
    // few parts: their sums are fetched beside the weights, needed or not
    const bool few = all <= 8;
    float4 e0 = make_float4(0.f, 0.f, 0.f, 0.f), e1 = e0;
    if (few) {
        e0 = part(min(wave, all - 1));
        e1 = part(min(wave + 4, all - 1));
    }
    // ---- weights: thread (t / 16, row t % 16) takes parts t / 16 + 16 k
    const f2* ml = A.ml + head + r;
    f2 v[MAX_PARTS / 16];
    float M = LOWEST;
#pragma unroll
    for (int k = 0; k < MAX_PARTS / 16; k++) {
        v[k] = f2{LOWEST, 0.f};
        if (t / 16 + 16 * k < all) v[k] = ml[(t / 16 + 16 * k) * step];
    }
#pragma unroll
    for (int k = 0; k < MAX_PARTS / 16; k++) M = fmaxf(M, v[k][0]);
    red[t / 16][li] = M;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; i++) M = fmaxf(M, red[i][li]);
    __syncthreads();
    float L = 0.f;
#pragma unroll
    for (int k = 0; k < MAX_PARTS / 16; k++) {
        const int c = t / 16 + 16 * k;
        if (c >= all) break;
        // a part that saw nothing has not written its sums
        const float w = v[k][1] == 0.f ? 0.f : __builtin_amdgcn_exp2f(v[k][0] - M);
        L += v[k][1] * w;
        wt[c][li] = w;
    }
    red[t / 16][li] = L;
    __syncthreads();
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    // what a weight of 0 stands for may hold anything
    auto add = [&](const float4& z, float w) {
        o.x += w != 0.f ? z.x * w : 0.f;
        o.y += w != 0.f ? z.y * w : 0.f;
        o.z += w != 0.f ? z.z * w : 0.f;
        o.w += w != 0.f ? z.w * w : 0.f;
    };
    if (few) {
        add(e0, wave < all ? wt[wave][li] : 0.f);
        add(e1, wave + 4 < all ? wt[wave + 4][li] : 0.f);
    } else {
        if (wave == 0) {
            int n = 0;
            for (int c0 = 0; c0 < all; c0 += 64) {
                bool any = false;
                if (c0 + lane < all)
#pragma unroll
                    for (int i = 0; i < 16; i++) any |= wt[c0 + lane][i] != 0.f;
                const unsigned long long m = __ballot(any);
                if (any) list[n + __popcll(m & ((1ull << lane) - 1))] = c0 + lane;
                n += __popcll(m);
            }
            if (lane == 0) count = n;
        }
        __syncthreads();
        const int n = count;
        constexpr int U = 8;
        for (int k0 = wave; k0 < n; k0 += 4 * U) {
            float4 z[U];
            float w[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int k = k0 + 4 * u, c = list[min(k, n - 1)];
                w[u] = k < n ? wt[c][li] : 0.f;
                z[u] = part(c);
            }
#pragma unroll
            for (int u = 0; u < U; u++) add(z[u], w[u]);
        }
    }
    ro[wave][lane] = o;
    __syncthreads();
    if (wave || !valid) return;
    L = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) L += red[i][li];
#pragma unroll
    for (int w = 1; w < 4; w++) {
        const float4 z = ro[w][lane];
        o.x += z.x, o.y += z.y, o.z += z.z, o.w += z.w;
    }
    const float inv = L != 0.f ? 1.f / L : 0.f;
    const int sj = r / g;
    const size_t qrow = (size_t)sj * A.q_heads + kvh * g + (r - sj * g);
    *reinterpret_cast<uint2*>(A.out + qrow * D + 16 * x + 4 * q4) = make_uint2(f2h2(o.x * inv, o.y * inv), f2h2(o.z * inv, o.w * inv));
}
extern "C" __global__ __launch_bounds__(256) void cima_attn_paged_join_d64(const AttnArgs A) { attn_join_body<64>(A); }
extern "C" __global__ __launch_bounds__(256) void cima_attn_paged_join_d128(const AttnArgs A) { attn_join_body<128>(A); }
