// Paged KV cache for gfx950 (CDNA4): the code object cima_paged.hsaco.  RoPE
// with the append of a step's keys and values, the read back, and the operations
// on pages: copy, reserve, fork, free, compact.  The cache's layout is
// cima_kv_pages in include/cima_hip.h.
#include "gguf_formats.h"
#include "kv_quant.h"

// ---------------------------------------------------------- RoPE and append

// One row of qkv per workgroup: the D/2 angles of the row's position go to LDS
// once (pos * theta^(-2i/D) in fp64, reduced to a fraction of a turn there, so
// that far positions keep their angle), then every thread rotates eight pairs
// of a head, two 16-byte words.  Keys and values go to the row's place in its
// page.  Rotated in fp32 (the angle's sine and cosine are rounded to it) and
// rounded to f16 once.  Bound by memory: 2048 rows of 48 heads of 128 (50 MB read
// and written) 9.8 us on MI355X, 5.1 TB/s; four rows 3 us, the chain lens, table,
// sine.
template <int D>
DEV void rope_append_body(const uint16_t* __restrict__ qkv, uint16_t* __restrict__ q, uint16_t* __restrict__ kp,
                          uint16_t* __restrict__ vp, const int* __restrict__ table, const int* __restrict__ lens,
                          int n_new, int q_heads, int kv_heads, int page_shift, int n_pages, int table_stride,
                          int rotate, double log2_theta) {
    constexpr int H8 = D / 16;  // 8-pair words of a head
    __shared__ float cs[D / 2], sn[D / 2];
    const int row = blockIdx.x, s = row / n_new, t = threadIdx.x;
    const int len = lens[s];
    if (len < 0) return;
    const int pos = len + (row - s * n_new);
    const int at = pos >> page_shift;
    int id = -1;
    if ((unsigned)at < (unsigned)table_stride) id = table[(size_t)s * table_stride + at];
    if (t < D / 2) {
        float sv = 0.f, cv = 1.f;
        if (rotate) {
            const double turns = (double)pos * (exp2(log2_theta * (-2.0 * t / D)) * 0.15915494309189533577);
            sincospif((float)(2.0 * (turns - rint(turns))), &sv, &cv);
        }
        cs[t] = cv;
        sn[t] = sv;
    }
    __syncthreads();
    const uint16_t* x = qkv + (size_t)row * (q_heads + 2 * kv_heads) * D;
    const bool keep = (unsigned)id < (unsigned)n_pages;
    const int page = 1 << page_shift;
    // head h of the cached row: offset of its first element
    auto place = [&](int h) { return (((size_t)id * kv_heads + h) * page + (pos & (page - 1))) * D; };
    for (int e = t; e < (q_heads + kv_heads) * H8; e += 256) {
        const int h = e / H8, i = e % H8 * 8;
        const uint4 a = *reinterpret_cast<const uint4*>(x + (size_t)h * D + i);
        const uint4 b = *reinterpret_cast<const uint4*>(x + (size_t)h * D + D / 2 + i);
        const uint32_t au[4] = {a.x, a.y, a.z, a.w}, bu[4] = {b.x, b.y, b.z, b.w};
        uint32_t oa[4], ob[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float a0 = h2f(au[j] & 0xffffu), a1 = h2f(au[j] >> 16);
            const float b0 = h2f(bu[j] & 0xffffu), b1 = h2f(bu[j] >> 16);
            const float c0 = cs[i + 2 * j], c1 = cs[i + 2 * j + 1], s0 = sn[i + 2 * j], s1 = sn[i + 2 * j + 1];
            oa[j] = f2h2(a0 * c0 - b0 * s0, a1 * c1 - b1 * s1);
            ob[j] = f2h2(a0 * s0 + b0 * c0, a1 * s1 + b1 * c1);
        }
        uint16_t* y;
        if (h < q_heads) y = q + ((size_t)row * q_heads + h) * D;
        else if (keep) y = kp + place(h - q_heads);
        else continue;
        *reinterpret_cast<uint4*>(y + i) = make_uint4(oa[0], oa[1], oa[2], oa[3]);
        *reinterpret_cast<uint4*>(y + D / 2 + i) = make_uint4(ob[0], ob[1], ob[2], ob[3]);
    }
    if (!keep) return;
    for (int e = t; e < kv_heads * (D / 8); e += 256) {
        const int h = e / (D / 8), i = e % (D / 8) * 8;
        *reinterpret_cast<uint4*>(vp + place(h) + i) =
            *reinterpret_cast<const uint4*>(x + (size_t)(q_heads + kv_heads + h) * D + i);
    }
}
#define ROPE_APPEND(D)                                                                                               \
    extern "C" __global__ __launch_bounds__(256) void cima_rope_append_paged_d##D(                                   \
        const uint16_t* __restrict__ qkv, uint16_t* __restrict__ q, uint16_t* __restrict__ kp,                       \
        uint16_t* __restrict__ vp, const int* __restrict__ table, const int* __restrict__ lens, int n_new,           \
        int q_heads, int kv_heads, int page_shift, int n_pages, int table_stride, int rotate,                          \
        double log2_theta) {                                                                                         \
        rope_append_body<D>(qkv, q, kp, vp, table, lens, n_new, q_heads, kv_heads, page_shift, n_pages,              \
                            table_stride, rotate, log2_theta);                                                       \
    }
ROPE_APPEND(64)
ROPE_APPEND(128)

// The same into a quantised cache.  A row's keys are rotated in fp64 and rounded to
// f16, what an f16 cache would hold, so that the codes do not hang on fp32's last
// bits (with an fp32 rotation one key in 10^4 is off by an f16 step, and now and
// then a code or its group's scale with it); queries as above.  A thread has eight
// elements of a group, a quad the group: its extremes are two exchanges in the quad.
// Bound by memory: 2048 rows of 32/8 heads of 128 as Q4_1 (45 MB read and written) 11 us
// on MI355X, 4.1 TB/s; four rows 4 us, the chain above and the extremes.
template <int D, int BITS>
DEV void rope_append_quant_body(const uint16_t* __restrict__ qkv, uint16_t* __restrict__ q, uint8_t* __restrict__ kp,
                                uint8_t* __restrict__ vp, const int* __restrict__ table, const int* __restrict__ lens,
                                int n_new, int q_heads, int kv_heads, int page_shift, int n_pages, int table_stride,
                                int rotate, double log2_theta) {
    using Q = KvQ<BITS>;
    constexpr int H8 = D / 16;  // 8-pair words of a head
    __shared__ float cs[D / 2], sn[D / 2];
    __shared__ double cd[D / 2], sd[D / 2];
    const int row = blockIdx.x, s = row / n_new, t = threadIdx.x;
    const int len = lens[s];
    if (len < 0) return;
    const int pos = len + (row - s * n_new);
    const int at = pos >> page_shift;
    int id = -1;
    if ((unsigned)at < (unsigned)table_stride) id = table[(size_t)s * table_stride + at];
    if (t < D / 2) {
        double sv = 0., cv = 1.;
        if (rotate) {
            const double turns = (double)pos * (exp2(log2_theta * (-2.0 * t / D)) * 0.15915494309189533577);
            sincospi(2.0 * (turns - rint(turns)), &sv, &cv);
        }
        cs[t] = (float)cv, sn[t] = (float)sv;
        cd[t] = cv, sd[t] = sv;
    }
    __syncthreads();
    const uint16_t* x = qkv + (size_t)row * (q_heads + 2 * kv_heads) * D;
    const bool keep = (unsigned)id < (unsigned)n_pages;
    const int page = 1 << page_shift, r = pos & (page - 1);
    for (int e = t; e < q_heads * H8; e += 256) {
        const int h = e / H8, i = e % H8 * 8;
        const uint4 a = *reinterpret_cast<const uint4*>(x + (size_t)h * D + i);
        const uint4 b = *reinterpret_cast<const uint4*>(x + (size_t)h * D + D / 2 + i);
        const uint32_t au[4] = {a.x, a.y, a.z, a.w}, bu[4] = {b.x, b.y, b.z, b.w};
        uint32_t oa[4], ob[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float a0 = h2f(au[j] & 0xffffu), a1 = h2f(au[j] >> 16);
            const float b0 = h2f(bu[j] & 0xffffu), b1 = h2f(bu[j] >> 16);
            const float c0 = cs[i + 2 * j], c1 = cs[i + 2 * j + 1], s0 = sn[i + 2 * j], s1 = sn[i + 2 * j + 1];
            oa[j] = f2h2(a0 * c0 - b0 * s0, a1 * c1 - b1 * s1);
            ob[j] = f2h2(a0 * s0 + b0 * c0, a1 * s1 + b1 * c1);
        }
        uint16_t* y = q + ((size_t)row * q_heads + h) * D;
        *reinterpret_cast<uint4*>(y + i) = make_uint4(oa[0], oa[1], oa[2], oa[3]);
        *reinterpret_cast<uint4*>(y + D / 2 + i) = make_uint4(ob[0], ob[1], ob[2], ob[3]);
    }
    if (!keep) return;
    // keys, then values, eight elements a thread: 8 heads of 128 are one pass
    for (int e = t; e < 2 * kv_heads * (D / 8); e += 256) {
        const int h = e / (D / 8), i = e % (D / 8) * 8;
        const uint16_t* from = x + (size_t)(q_heads + h) * D;
        const uint4 own = *reinterpret_cast<const uint4*>(from + i);
        uint32_t v[4] = {own.x, own.y, own.z, own.w};
        if (h < kv_heads) {
            const uint4 other = *reinterpret_cast<const uint4*>(from + (i ^ (D / 2)));
            const uint32_t o[4] = {other.x, other.y, other.z, other.w};
            const int at = i & (D / 2 - 1);
            const double sign = i < D / 2 ? -1. : 1.;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const double a0 = h2f(v[j] & 0xffffu), a1 = h2f(v[j] >> 16);
                const double b0 = h2f(o[j] & 0xffffu), b1 = h2f(o[j] >> 16);
                v[j] = d2h(fma(a0, cd[at + 2 * j], sign * b0 * sd[at + 2 * j])) |
                       d2h(fma(a1, cd[at + 2 * j + 1], sign * b1 * sd[at + 2 * j + 1])) << 16;
            }
        }
        uint32_t w[Q::WORDS];
        const uint32_t sc = kv_encode<BITS>(v, w);
        uint8_t* head = (h < kv_heads ? kp : vp) + ((size_t)id * kv_heads + (h < kv_heads ? h : h - kv_heads)) * page * Q::row(D);
        uint32_t* c = reinterpret_cast<uint32_t*>(head + r * Q::codes(D) + i * BITS / 8);
#pragma unroll
        for (int k = 0; k < Q::WORDS; k++) c[k] = w[k];
        if ((i & 31) == 0) {
            uint8_t* z = head + page * Q::codes(D) + r * Q::scales(D) + i / 32 * Q::SCALE;
            if constexpr (BITS == 4) *reinterpret_cast<uint32_t*>(z) = sc;
            else *reinterpret_cast<uint16_t*>(z) = (uint16_t)sc;
        }
    }
}
#define ROPE_APPEND_QUANT(D, BITS)                                                                                   \
    extern "C" __global__ __launch_bounds__(256) void cima_rope_append_paged_q##BITS##_d##D(                         \
        const uint16_t* __restrict__ qkv, uint16_t* __restrict__ q, uint8_t* __restrict__ kp,                        \
        uint8_t* __restrict__ vp, const int* __restrict__ table, const int* __restrict__ lens, int n_new,            \
        int q_heads, int kv_heads, int page_shift, int n_pages, int table_stride, int rotate,                        \
        double log2_theta) {                                                                                         \
        rope_append_quant_body<D, BITS>(qkv, q, kp, vp, table, lens, n_new, q_heads, kv_heads, page_shift, n_pages,  \
                                        table_stride, rotate, log2_theta);                                           \
    }
ROPE_APPEND_QUANT(64, 4)
ROPE_APPEND_QUANT(128, 4)
ROPE_APPEND_QUANT(64, 8)
ROPE_APPEND_QUANT(128, 8)

// ---------------------------------------------------------------- read back

// Positions first + j of slots as f16 rows [slot][head][max_seq][D]: a thread has
// eight elements of ROWS rows of the keys and of the values, whose loads go out
// together.  Positions without a page are zeros.  Bound by memory, past the caches
// both ways: 24 slots of 5000 positions, 8 heads of 128, Q4_1 (154 MB read, 491
// written) 115 us on MI355X, 5.6 TB/s, Q8_0 133; through the caches 127 and 145.
// Where there are few rows (`all`, of all heads one after the other) a
// thread has one: one slot of 4003, 2 heads of 64, Q8_0 4.1 -> 3.3 us, 8 rows of 256 slots
// 5.9 -> 5.0; but the 24 slots 133.
constexpr int READ_ROWS = 4;
typedef uint32_t word4 __attribute__((ext_vector_type(4)));
template <int D, int BITS, int ROWS>
DEV void kv_read_body(const uint8_t* __restrict__ kp, const uint8_t* __restrict__ vp, const int* __restrict__ table,
                      const int* __restrict__ slots, const int* __restrict__ first, uint16_t* __restrict__ k,
                      uint16_t* __restrict__ v, int kv_heads, int page_shift, int n_pages, int table_stride,
                      int max_seqs, int n, int blocks, int all, long long max_seq) {
    using Q = KvQ<BITS>;
    constexpr int W8 = D / 8, PASS = 256 / W8;  // threads of a row, rows of a pass
    const int row = threadIdx.x / W8, w8 = threadIdx.x % W8, page = 1 << page_shift;
    // the head, and the first row's position less the slot's first
    int sh, j0;
    if constexpr (ROWS == 1) {
        const int at = blockIdx.x * PASS + row;
        if (at >= all) return;
        sh = (int)((uint32_t)at / (uint32_t)n), j0 = at - sh * n;
    } else {
        sh = blockIdx.x / blocks, j0 = blockIdx.x % blocks * ROWS * PASS + row;
    }
    const int i = sh / kv_heads, h = sh % kv_heads;
    const int slot = slots ? slots[i] : i;
    const long long from = first ? first[i] : 0;
    const size_t out = (size_t)sh * max_seq * D + w8 * 8;
    uint32_t w[2][ROWS][Q::WORDS], sc[2][ROWS];
    bool has[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; u++) {
        const int j = j0 + u * PASS;
        const long long pos = from + j, e = pos >> page_shift;
        int id = -1;
        if (j < n && pos >= 0 && e < table_stride && (unsigned)slot < (unsigned)max_seqs)
            id = table[(size_t)slot * table_stride + e];
        has[u] = (unsigned)id < (unsigned)n_pages;
        const int r = (int)(pos & (page - 1));
        const size_t head = ((size_t)(has[u] ? id : 0) * kv_heads + h) * page * Q::row(D);
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const uint8_t* p = (c ? vp : kp) + head;
            const uint32_t* at = reinterpret_cast<const uint32_t*>(p + (size_t)r * Q::codes(D)) + w8 * Q::WORDS;
#pragma unroll
            for (int x = 0; x < Q::WORDS; x++) w[c][u][x] = __builtin_nontemporal_load(at + x);
            sc[c][u] = Q::load_scale(p, page, D, r, w8 / 4);
        }
    }
#pragma unroll
    for (int u = 0; u < ROWS; u++) {
        const int j = j0 + u * PASS;
        if (j >= n) break;
#pragma unroll
        for (int c = 0; c < 2; c++) {
            uint32_t o[4];
            Q::decode(w[c][u], sc[c][u], o);
            const uint4 z = has[u] ? make_uint4(o[0], o[1], o[2], o[3]) : make_uint4(0, 0, 0, 0);
            __builtin_nontemporal_store((word4){z.x, z.y, z.z, z.w}, (word4*)((c ? v : k) + out + (size_t)j * D));
        }
    }
}
#define KV_READ_AS(NAME, D, BITS, ROWS)                                                                              \
    extern "C" __global__ __launch_bounds__(256) void cima_kv_pages_##NAME##_b##BITS##_d##D(                         \
        const uint8_t* __restrict__ kp, const uint8_t* __restrict__ vp, const int* __restrict__ table,               \
        const int* __restrict__ slots, const int* __restrict__ first, uint16_t* __restrict__ k,                      \
        uint16_t* __restrict__ v, int kv_heads, int page_shift, int n_pages, int table_stride, int max_seqs, int n,  \
        int blocks, int all, long long max_seq) {                                                                    \
        kv_read_body<D, BITS, ROWS>(kp, vp, table, slots, first, k, v, kv_heads, page_shift, n_pages, table_stride,  \
                                    max_seqs, n, blocks, all, max_seq);                                              \
    }
#define KV_READ(D, BITS)                  \
    KV_READ_AS(read, D, BITS, READ_ROWS)  \
    KV_READ_AS(read_few, D, BITS, 1)
KV_READ(64, 4)
KV_READ(128, 4)
KV_READ(64, 8)
KV_READ(128, 8)
KV_READ(64, 16)
KV_READ(128, 16)

// -------------------------------------------------------------- page copies

// The copies go in pieces of 16 KB (256 threads, four 16-byte words each), a
// workgroup a piece as far as the grid goes, past the caches both ways: what is
// moved once is not read soon.  Measured on MI355X, 52 pages in 32 planes (220
// MB): 92 us, 4.8 TB/s read and written, as fast as a large copy; through the
// caches 107, eight words a thread 93, eight workgroups to a CU 99.
constexpr int PIECE = 1024;  // 16-byte words of a piece

DEV void copy_piece(const word4* __restrict__ src, word4* __restrict__ dst, long long words, long long first) {
    word4 v[4];
    const long long i = first + threadIdx.x;
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = __builtin_nontemporal_load(&src[min(i + 256 * j, words - 1)]);
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (i + 256 * j < words) __builtin_nontemporal_store(v[j], &dst[i + 256 * j]);
}

// Unit u of `pages` pages in n_planes planes: (plane, page pair, piece).
DEV void copy_unit(word4* pool, long long plane_words, long long page_words, int pieces, int pages, long long u,
                   const int* __restrict__ src, const int* __restrict__ dst, int n_pages) {
    const int piece = (int)(u % pieces);
    const long long v = u / pieces;
    const int k = (int)(v % pages);
    const int a = src[k], b = dst[k];
    if ((unsigned)a >= (unsigned)n_pages || (unsigned)b >= (unsigned)n_pages || a == b) return;
    word4* plane = pool + (v / pages) * plane_words;
    copy_piece(plane + a * page_words, plane + b * page_words, page_words, (long long)piece * PIECE);
}

extern "C" __global__ __launch_bounds__(256) void cima_kv_pages_copy(word4* pool, long long plane_words,
                                                                     long long page_words, int pieces, int n,
                                                                     long long units, const int* __restrict__ src,
                                                                     const int* __restrict__ dst, int n_pages) {
    for (long long u = blockIdx.x; u < units; u += gridDim.x)
        copy_unit(pool, plane_words, page_words, pieces, n, u, src, dst, n_pages);
}

// ------------------------------------------------------- the lowest free pages
//
// One workgroup of 1024 threads (16 waves) looks at every count: pages in
// chunks of 1024, a wave a chunk, 16 counts a lane.  `sum` is the exclusive
// running sum of the chunks' counts, so any rank's chunk is known.

constexpr int CH = 1024;         // pages of a chunk
constexpr int MAX_CHUNKS = 1024;  // n_pages <= 1048576
constexpr int MAX_SLOTS = 4096;

template <int CTRL, int ROWS>
DEV int dpp_i(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
// inclusive running sum within rows of 16 lanes, and over the wave
DEV int row_scan(int v) {
    v += dpp_i<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
    v += dpp_i<0x112, 0xf>(v);
    v += dpp_i<0x114, 0xf>(v);
    return v + dpp_i<0x118, 0xf>(v);
}
DEV int wave_scan(int v) {
    v = row_scan(v);
    v += dpp_i<0x142, 0xa>(v);         // row_bcast:15 into rows 1, 3
    return v + dpp_i<0x143, 0xc>(v);   // row_bcast:31 into rows 2, 3
}
// Exclusive prefix sum of v over the 1024 threads of the workgroup, the whole
// in *total.
DEV int block_scan(int v, int* total) {
    __shared__ int part[16];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int x = wave_scan(v);
    __syncthreads();
    if (lane == 63) part[w] = x;
    __syncthreads();
    const int p = row_scan(part[lane & 15]);
    *total = __builtin_amdgcn_readlane(p, 15);
    return (w ? __builtin_amdgcn_readlane(p, w - 1) : 0) + x - v;
}

// bit i of the result: page first + 64 i + lane of a chunk exists and is free
// (FREE) or held
template <bool FREE>
DEV uint32_t chunk_bits(const int* refs, int n_pages, int first) {
    const int lane = threadIdx.x & 63;
    int r[16];
#pragma unroll
    for (int i = 0; i < 16; i++) r[i] = refs[min(first + 64 * i + lane, n_pages - 1)];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; i++)
        if (first + 64 * i + lane < n_pages && (r[i] == 0) == FREE) m |= 1u << i;
    return m;
}
DEV int below_lane(unsigned long long m) { return __popcll(m & ((1ull << (threadIdx.x & 63)) - 1)); }
// sum[c] = pages of the kind in chunks before c; returns how many there are.
// *bits: those of this wave's first chunk, for each_lowest
template <bool FREE>
DEV int count_chunks(const int* refs, int n_pages, int* sum, uint32_t* bits) {
    const int chunks = (n_pages + CH - 1) / CH, w = threadIdx.x >> 6;
    *bits = 0;
    for (int c = w; c < chunks; c += 16) {
        const uint32_t b = chunk_bits<FREE>(refs, n_pages, c * CH);
        if (c == w) *bits = b;
        int n = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) n += __popcll(__ballot(b >> i & 1));
        if ((threadIdx.x & 63) == 0) sum[c] = n;
    }
    __syncthreads();
    const int mine = (int)threadIdx.x < chunks ? sum[threadIdx.x] : 0;
    int total;
    const int before = block_scan(mine, &total);
    if ((int)threadIdx.x < chunks) sum[threadIdx.x] = before;
    __syncthreads();
    return total;
}
// emit(rank, page) for the `need` lowest pages of the kind
template <bool FREE, typename F>
DEV void each_lowest(const int* refs, int n_pages, const int* sum, uint32_t bits, int need, F emit) {
    const int chunks = (n_pages + CH - 1) / CH, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (int c = w; c < chunks && sum[c] < need; c += 16) {
        const uint32_t m = c == w ? bits : chunk_bits<FREE>(refs, n_pages, c * CH);
        int rank = sum[c];
        for (int i = 0; i < 16 && rank < need; i++) {
            const unsigned long long b = __ballot(m >> i & 1);
            const int mine = rank + below_lane(b);
            if ((m >> i & 1) && mine < need) emit(mine, c * CH + 64 * i + lane);
            rank += __popcll(b);
        }
    }
}

// Room for n_new tokens in slots [0, seqs): slot s lacks the entries from its
// first -1 in [lens / page, end) on (entries are filled from the left).  The
// page of rank r goes to the slot whose running sum holds r.  Bound by the
// latency of its loads: the counts are read beside the lengths.  9 slots in 1024
// pages 4.6 us on MI355X.
extern "C" __global__ __launch_bounds__(1024) void cima_kv_pages_reserve(int* refs, int n_pages, int* table,
                                                                         const int* lens, int seqs, int table_stride,
                                                                         int page_shift, int n_new, int* status) {
    __shared__ int sum[MAX_CHUNKS], base[MAX_SLOTS + 1], from[MAX_SLOTS], behind;
    const int t = threadIdx.x, page = 1 << page_shift;
    if (t == 0) behind = 0;
    int len = t < seqs ? lens[t] : -1;
    uint32_t bits;
    const int have = count_chunks<true>(refs, n_pages, sum, &bits);
    int need = 0;  // pages wanted by the slots so far
    for (int s0 = 0; s0 < seqs; s0 += 1024) {
        const int s = s0 + t;
        if (s0) len = s < seqs ? lens[s] : -1;
        int lack = 0, lo = 0;
        if (len >= 0) {
            const int* row = table + (size_t)s * table_stride;
            lo = len >> page_shift;
            int end = (int)(((long long)len + n_new + page - 1) >> page_shift);
            const int off = end - max(lo, table_stride);  // entries behind the row
            if (off > 0) atomicAdd(&behind, min(off, 1 << 18));
            end = min(end, table_stride);
            int hi = max(end, lo);
            if (hi - lo <= 4) {  // a few entries: looked at together
                int e[4];
#pragma unroll
                for (int i = 0; i < 4; i++) e[i] = lo + i < hi ? row[lo + i] : -1;
#pragma unroll
                for (int i = 3; i >= 0; i--)
                    if (e[i] < 0) hi = min(hi, lo + i);
                lo = hi;
            } else {
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (row[mid] < 0) hi = mid;
                    else lo = mid + 1;
                }
            }
            lack = max(0, end - lo);
        }
        int n;
        const int before = block_scan(lack, &n);
        if (s < seqs) {
            base[s] = need + before;
            from[s] = lo;
        }
        need += n;
    }
    __syncthreads();
    const int missing = (int)min((long long)max(0, need - have) + behind, 0x7fffffffLL);
    if (t == 0) *status = missing;
    if (missing || need == 0) return;
    each_lowest<true>(refs, n_pages, sum, bits, need, [&](int rank, int id) {
        int lo = 0, hi = seqs - 1;  // the last slot whose base is at most rank
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (base[mid] <= rank) lo = mid;
            else hi = mid - 1;
        }
        table[(size_t)lo * table_stride + from[lo] + (rank - base[lo])] = id;
        refs[id] = 1;
    });
}

// Fork, first launch: the slots are looked over and claimed (a child's lens
// goes from -1 to -2 - i, so that one named twice shows), pages are found for
// the children whose parent has begun a page, and entered.  8 children in 1024
// pages 4.5 us on MI355X, the second launch 3.5.
extern "C" __global__ __launch_bounds__(1024) void cima_kv_pages_fork(int* refs, int n_pages, int* table, int* lens,
                                                                      int max_seqs, int table_stride, int page_shift,
                                                                      const int* __restrict__ parents,
                                                                      const int* __restrict__ children, int n,
                                                                      int* status) {
    __shared__ int sum[MAX_CHUNKS], entry[MAX_SLOTS], wrong;
    constexpr int K = MAX_SLOTS / 1024;
    const int t = threadIdx.x, page = 1 << page_shift;
    int p[K], c[K], len[K];
    bool mine[K];
    if (t == 0) wrong = 0;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int i = t + 1024 * k;
        p[k] = i < n ? parents[i] : 0;
        c[k] = i < n ? children[i] : -1;
    }
    uint32_t bits;
    const int have = count_chunks<true>(refs, n_pages, sum, &bits);
    int need = 0;
#pragma unroll
    for (int k = 0; k < K; k++) {
        mine[k] = false;
        if (1024 * k >= n) continue;
        const int i = t + 1024 * k;
        if (i < n) {
            bool ok = (unsigned)p[k] < (unsigned)max_seqs && (unsigned)c[k] < (unsigned)max_seqs;
            if (ok) {
                len[k] = lens[p[k]];
                ok = len[k] >= 0 && len[k] <= table_stride << page_shift;
                if (ok) {
                    // the page that the parent has begun is copied: it has to be one
                    const bool begun = len[k] & (page - 1);
                    const int id = begun ? table[(size_t)p[k] * table_stride + (len[k] >> page_shift)] : 0;
                    mine[k] = atomicCAS(&lens[c[k]], -1, -2 - i) == -1;
                    ok = mine[k] && (unsigned)id < (unsigned)n_pages;
                }
            }
            if (!ok) wrong = 1;
        }
        int m;
        const int part = mine[k] && len[k] & (page - 1);
        const int before = block_scan(part, &m);
        if (part) entry[need + before] = c[k] * table_stride + (len[k] >> page_shift);
        need += m;
    }
    __syncthreads();
    const int missing = max(0, need - have);
    const bool fine = !wrong && !missing;
    if (t == 0) *status = wrong ? -1 : missing;
#pragma unroll
    for (int k = 0; k < K; k++)
        if (mine[k]) lens[c[k]] = fine ? len[k] : -1;
    if (!fine || need == 0) return;
    each_lowest<true>(refs, n_pages, sum, bits, need, [&](int rank, int id) {
        table[entry[rank]] = id;
        refs[id] = 1;
    });
}

// Fork, second launch: workgroups [0, n) write the children's rows and count
// the shared pages, the others copy the rows of the pages begun (and a quantised
// cache's scales of them), one child and plane each.
extern "C" __global__ __launch_bounds__(256) void cima_kv_pages_fork_copy(
    uint4* pool, long long plane_words, int* refs, int n_pages, int* table, const int* __restrict__ lens,
    int table_stride, int page_shift, int kv_heads, int row_words, int scale_words, const int* __restrict__ parents,
    const int* __restrict__ children, int n, const int* __restrict__ status) {
    if (*status != 0) return;
    const int b = blockIdx.x, i = b % n;
    const int p = parents[i], c = children[i], len = lens[p];
    const int full = len >> page_shift, rest = len & ((1 << page_shift) - 1);
    const int* from = table + (size_t)p * table_stride;
    int* to = table + (size_t)c * table_stride;
    if (b < n) {
        for (int e = threadIdx.x; e < table_stride; e += 256) {
            if (e < full) {
                const int id = from[e];
                to[e] = id;
                if ((unsigned)id < (unsigned)n_pages) atomicAdd(&refs[id], 1);
            } else if (e > full || rest == 0) {
                to[e] = -1;
            }
        }
        return;
    }
    if (rest == 0) return;
    const int src = from[full], dst = to[full];
    if ((unsigned)src >= (unsigned)n_pages || (unsigned)dst >= (unsigned)n_pages) return;
    uint4* plane = pool + (long long)(b / n - 1) * plane_words;
    // 16-byte words of rows copied and held per head, behind them 4-byte words of
    // rows' scales
    const int live = rest * row_words, rows = row_words << page_shift, live4 = rest * scale_words;
    const int head = rows + ((scale_words << page_shift) >> 2);
    const uint4* s = plane + (long long)src * kv_heads * head;
    uint4* d = plane + (long long)dst * kv_heads * head;
    for (int e = threadIdx.x; e < kv_heads * live; e += 256) {
        const int w = e / live * head + e % live;
        d[w] = s[w];
    }
    for (int e = threadIdx.x; e < kv_heads * live4; e += 256) {
        const int w = (e / live4 * head + rows) * 4 + e % live4;
        reinterpret_cast<uint32_t*>(d)[w] = reinterpret_cast<const uint32_t*>(s)[w];
    }
}

// Every entry is taken out once (an exchange), so that a slot named twice
// gives its pages back once.
extern "C" __global__ __launch_bounds__(256) void cima_kv_pages_free(int* refs, int n_pages, int* table, int* lens,
                                                                     int max_seqs, int table_stride,
                                                                     const int* __restrict__ slots, int parts) {
    const int s = slots[blockIdx.x / parts];
    if ((unsigned)s >= (unsigned)max_seqs) return;
    const int first = blockIdx.x % parts * 1024;
    if (first == 0 && threadIdx.x == 0) lens[s] = -1;
    int* row = table + (size_t)s * table_stride;
    for (int e = first + threadIdx.x; e < min(first + 1024, table_stride); e += 256) {
        if (row[e] == -1) continue;
        const int id = atomicExch(&row[e], -1);
        if ((unsigned)id < (unsigned)n_pages) atomicSub(&refs[id], 1);
    }
}

// Compaction, first launch: the moves (work = {count, -, src[n_pages],
// dst[n_pages], remap[n_pages]}) and the new counts.
extern "C" __global__ __launch_bounds__(1024) void cima_kv_pages_compact(const int* refs, int n_pages, int* refs_out,
                                                                         int* n_live, int* work) {
    __shared__ int held[MAX_CHUNKS];
    int* src = work + 16;
    int* dst = src + n_pages;
    int* remap = dst + n_pages;
    uint32_t bits;
    const int live = count_chunks<false>(refs, n_pages, held, &bits), lane = threadIdx.x & 63;
    const int chunks = (n_pages + CH - 1) / CH;
    // ranks: of a held page among the held, of a free one among the free
    auto each = [&](auto f) {
        for (int c = threadIdx.x >> 6; c < chunks; c += 16) {
            const uint32_t m = chunk_bits<false>(refs, n_pages, c * CH);
            int rank = held[c];
            for (int i = 0; i < 16; i++) {
                const unsigned long long b = __ballot(m >> i & 1);
                const int p = c * CH + 64 * i + lane, r = rank + below_lane(b);
                const bool h = m >> i & 1;
                if (p < n_pages) f(p, h, h ? r : p - r);
                rank += __popcll(b);
            }
        }
    };
    // holes below `live`: as many as there are held pages from `live` on, so
    // the last of these have the ranks [live - holes, live)
    __shared__ int holes;
    if (threadIdx.x == 0) holes = 0;
    __syncthreads();
    int mine = 0;
    each([&](int p, bool h, int) { mine += !h && p < live; });
    if (mine) atomicAdd(&holes, mine);
    __syncthreads();
    const int moves = holes;
    each([&](int p, bool h, int rank) {
        if (h && p >= live) src[rank - (live - moves)] = p;
        if (!h && p < live) dst[rank] = p;
        if (p < live || !h) remap[p] = p;
    });
    __threadfence_block();
    __syncthreads();
    for (int k = threadIdx.x; k < moves; k += 1024) remap[src[k]] = dst[k];
    for (int p = threadIdx.x; p < live; p += 1024)
        if (refs_out != refs) refs_out[p] = refs[p];
    __threadfence_block();
    __syncthreads();
    for (int k = threadIdx.x; k < moves; k += 1024) refs_out[dst[k]] = refs[src[k]];
    __syncthreads();
    for (int p = live + threadIdx.x; p < n_pages; p += 1024) refs_out[p] = 0;
    if (threadIdx.x == 0) {
        work[0] = moves;
        *n_live = live;
    }
}

// Compaction, second launch: the pages are moved and the table's entries
// renamed; entries of pages that are not held stay.
extern "C" __global__ __launch_bounds__(256) void cima_kv_pages_compact_move(
    word4* pool, long long plane_words, long long page_words, int pieces, int n_planes, int n_pages,
    const int* table, int* table_out, long long entries, const int* __restrict__ work) {
    const int moves = work[0];
    const int* src = work + 16;
    const int* dst = src + n_pages;
    const int* remap = dst + n_pages;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < entries; e += (long long)gridDim.x * 256) {
        const int id = table[e];
        table_out[e] = (unsigned)id < (unsigned)n_pages ? remap[id] : id;
    }
    if (moves == 0) return;
    const long long units = (long long)n_planes * moves * pieces;
    for (long long u = blockIdx.x; u < units; u += gridDim.x)
        copy_unit(pool, plane_words, page_words, pieces, moves, u, src, dst, n_pages);
}
