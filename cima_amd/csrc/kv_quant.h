// Elements of a quantised paged cache for gfx950 (CDNA4), cima_kv_pages with a
// ggml_type: how a group of 32 is stored and what it stands for.  Included by
// paged_ops.hip and paged_attn.hip.
//
// Q4_1: codes 0 to 15, f16 scale d and least value m; value f16(c d + m).  d is the
// least f16 that is not below (max - m) / 15, so that no code is cut off and a value
// is off by at most d / 2 (and its rounding to f16).  Q8_0: codes -127 to 127, kept
// with 128 added, f16 scale d, the least not below max|x| / 127 but at most 515.5, above
// which 127 d would pass f16; value f16(c d).  A code is the nearest to the quotient, half
// to even.
//
// A head's page is its rows' codes, then its rows' scales ({d, m} or d, in the
// groups' order).  Eight elements of Q4_1 are a 32-bit word: element 2 k in nibble
// k, element 2 k + 1 in nibble k + 4, so that a shift and a mask leave a pair of
// neighbours in the halves of the word, as the f16 instructions take it.
#pragma once
#include "gguf_formats.h"

typedef _Float16 kvh2 __attribute__((ext_vector_type(2)));

// BITS 4: Q4_1, 8: Q8_0, 16: f16 as it is
template <int BITS>
struct KvQ {
    static constexpr int WORDS = BITS / 4;                             // 32-bit words of eight elements
    static constexpr int SCALE = BITS == 4 ? 4 : BITS == 8 ? 2 : 0;    // bytes of a group's scales
    // bytes of a row's codes and scales, and of a head's page
    static constexpr int codes(int dim) { return dim * BITS / 8; }
    static constexpr int scales(int dim) { return dim / 32 * SCALE; }
    static constexpr int row(int dim) { return codes(dim) + scales(dim); }

    // eight elements from their words, s as load_scale gives it
    DEV static void decode(const uint32_t (&w)[WORDS], uint32_t s, uint32_t (&o)[4]) {
        if constexpr (BITS == 16) {
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = w[i];
        } else {
            const kvh2 sc = __builtin_bit_cast(kvh2, s);
            const kvh2 d = {sc[0], sc[0]};
            if constexpr (BITS == 4) {
                const kvh2 m = {sc[1], sc[1]};
                // 1024 + c by the exponent's bits; of the pair in bits 4 to 7 1024 + 16 c,
                // whose 16th less 64 is c, exactly
                const kvh2 off = {(_Float16)-1024.f, (_Float16)-1024.f}, off4 = {(_Float16)-64.f, (_Float16)-64.f};
                const kvh2 down4 = {(_Float16)0.0625f, (_Float16)0.0625f};
                const uint32_t v = w[0] >> 8;
                // in a vector register: and, or in one instruction, which takes one scalar
                uint32_t one = 0x64006400u;
                __asm__("" : "+v"(one));
                kvh2 c[4];
                c[0] = __builtin_bit_cast(kvh2, (w[0] & 0x000f000fu) | one) + off;
                c[1] = __builtin_elementwise_fma(__builtin_bit_cast(kvh2, (w[0] & 0x00f000f0u) | one), down4, off4);
                c[2] = __builtin_bit_cast(kvh2, (v & 0x000f000fu) | one) + off;
                c[3] = __builtin_elementwise_fma(__builtin_bit_cast(kvh2, (v & 0x00f000f0u) | one), down4, off4);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    o[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(c[i], d, m));
            } else {
                const kvh2 off = {(_Float16)-1152.f, (_Float16)-1152.f};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    // bytes 2 i, 2 i + 1 under the exponent of 1024
                    const uint32_t u = __builtin_amdgcn_perm(0x64646464u, w[i / 2], i & 1 ? 0x07030602u : 0x05010400u);
                    // the bias in a value of its own: as part of the product it would be rounded
                    const kvh2 c = __builtin_bit_cast(kvh2, u) + off;
                    o[i] = __builtin_bit_cast(uint32_t, c * d);
                }
            }
        }
    }
    // scales of group g of row r in a head's page: {d, m} or d
    DEV static uint32_t load_scale(const uint8_t* head, int page, int dim, int r, int g) {
        const uint8_t* p = head + (uint32_t)(page * codes(dim) + r * scales(dim) + g * SCALE);
        if constexpr (BITS == 4) return *reinterpret_cast<const uint32_t*>(p);
        else if constexpr (BITS == 8) return *reinterpret_cast<const uint16_t*>(p);
        else return 0;
    }
};

// ---------------------------------------------------------------- storing

// fp64 -> f16 bits, rounded once: an fp32 that is not exact is made odd on the way,
// and no odd one lies half way between two f16
DEV uint32_t d2h(double v) {
    const float f = (float)v;
    uint32_t u = __builtin_bit_cast(uint32_t, f);
    if ((double)f != v) u = (u - (fabs((double)f) > fabs(v) ? 1u : 0u)) | 1u;
    return f2h(__builtin_bit_cast(float, u));
}
// max over the four lanes of a quad
DEV float quad_max(float v) {
    v = fmaxf(v, dpp_xor1(v));
    return fmaxf(v, dpp_xor2(v));
}
// f16 bits of the least f16 that is not below w / steps, w >= 0 and finite
DEV uint32_t scale_up(double w, float steps) {
    uint32_t c = f2h((float)w / steps);
    if (c) c--;  // the quotient's rounding is off by one at most
#pragma unroll
    for (int i = 0; i < 2; i++)
        if ((double)(h2f(c) * steps) < w) c++;
    return c;
}
// the code nearest to (x - m) / d, by exact products in fp64 where the fp32 quotient
// (off by less than `near`) lies that close to half way
DEV float code_of(float x, float m, float d, float inv, float near) {
    const float z = (x - m) * inv;
    float r = rintf(z);
    if (fabsf(z - r) > 0.5f - near) {
        const float k = floorf(z);
        const double two = 2. * ((double)x - (double)m), half = (2. * k + 1.) * (double)d;
        r = two > half || (two == half && ((int)k & 1)) ? k + 1.f : k;
    }
    return r;
}
// Eight f16 elements of a group that a quad's lanes hold in order: their words, and
// the group's scales (the same in all four lanes).  A group that is not finite
// gets NaN as its scale.
template <int BITS>
DEV uint32_t kv_encode(const uint32_t (&x)[4], uint32_t (&w)[KvQ<BITS>::WORDS]) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = h2f(i & 1 ? x[i / 2] >> 16 : x[i / 2] & 0xffffu);
    float hi = v[0], lo = v[0];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        hi = fmaxf(hi, v[i]), lo = fminf(lo, v[i]);
        bad |= !__builtin_isfinite(v[i]);
    }
    hi = quad_max(hi), lo = -quad_max(-lo);
    bad = quad_max(bad ? 1.f : 0.f) > 0.f;
    constexpr float STEPS = BITS == 4 ? 15.f : 127.f;
    const float m = BITS == 4 ? lo + 0.f : 0.f;  // a least value of -0 as 0, whichever came first
    const double width = BITS == 4 ? (double)hi - (double)lo : (double)fmaxf(hi, -lo);
    uint32_t db = bad ? 0x7e00u : scale_up(width, STEPS);
    // of 65472 and 65504 516, whose 127th multiple is no f16: 515.5, the nearest code still 127
    if (BITS == 8 && db == 0x6008u) db = 0x6007u;
    const float d = h2f(db), inv = d > 0.f ? __builtin_amdgcn_rcpf(d) : 0.f;
    // the quotient's fp32 roundings (the reciprocal's 2^-23) at its largest, 15 or 127
    constexpr float NEAR = BITS == 4 ? 1e-5f : 1e-4f;
    int c[8];
#pragma unroll
    for (int i = 0; i < 8; i++) c[i] = d > 0.f ? (int)code_of(v[i], m, d, inv, NEAR) : 0;
    if constexpr (BITS == 4) {
        w[0] = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) w[0] |= (uint32_t)(c[i] & 15) << (i / 2 * 4 + (i & 1) * 16);
        return db | f2h(m) << 16;
    } else {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            w[k] = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) w[k] |= (uint32_t)((c[4 * k + i] + 128) & 255) << 8 * i;
        }
        return db;
    }
}
