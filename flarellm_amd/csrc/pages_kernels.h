// Kernels of the paged KV cache: attention of a batch of queries over the pages of
// their sequences, and the stores, reads and copies of pages.
#pragma once

#include <type_traits>

#include "bgemm_pack.h"
#include "pages_args.h"

namespace fl {

typedef _Float16 ph8_t __attribute__((ext_vector_type(8)));
typedef float pf4_t __attribute__((ext_vector_type(4)));
typedef float pf16_t __attribute__((ext_vector_type(16)));
typedef uint32_t pu4_t __attribute__((ext_vector_type(4)));
typedef uint32_t pu2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ pf4_t pg_mfma_h(pu4_t a, pu4_t b, pf4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ph8_t, a), __builtin_bit_cast(ph8_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ pf16_t pg_mfma_w(pu4_t a, pu4_t b, pf16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(ph8_t, a), __builtin_bit_cast(ph8_t, b), c, 0, 0, 0);
}

// Mixed multiply-adds of f32 and binary16 (v_fma_mix*: exact products, one rounding), as
// expressions that the compiler selects them from: written as assembly, nothing would keep
// them the distance from matrix products, exponentials and half-register writes that
// these need.  The multiplier of -1 is opaque, or the compiler makes two instructions of it.
typedef _Float16 ph2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float pg_minus_one() {
    float m = -1.0f;
    asm("" : "+v"(m));
    return m;
}
__device__ __forceinline__ float pg_fma_mix(float a, uint32_t b, int half, float c) {
    return __builtin_fmaf(a, (float)__builtin_bit_cast(ph2_t, b)[half], c);
}
// 2 floats as two binary16 parts: round toward zero, then the rest.  (The first part is
// rounded by an instruction of its own: of (_Float16)(x * y) the compiler makes v_fma_mixlo's
// one rounding in one place and two in another, and the parts no longer fit together.)
__device__ __forceinline__ void pg_split2(float x0, float x1, float minus, uint32_t &hi, uint32_t &lo) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(x0, x1);
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, ph2_t{(_Float16)__builtin_fmaf((float)h[0], minus, x0),
                                            (_Float16)__builtin_fmaf((float)h[1], minus, x1)});
}
// 8 floats
__device__ __forceinline__ void pg_split(const float *x, pu4_t &hi, pu4_t &lo) {
    const float minus = pg_minus_one();
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t h, l;
        pg_split2(x[2 * i], x[2 * i + 1], minus, h, l);
        hi[i] = h;
        lo[i] = l;
    }
}

// A power of two that brings a query's largest value x to 2^13, so that the low parts
// of the others stay normal (zero, denormal and non-finite rows stay), and the score
// scale c for it.
__device__ __forceinline__ void pg_q_scale(float x, float &mul, float &c) {
    const int e = (int)((__float_as_uint(x) >> 23) & 0xFF);
    if (e <= 13 || e == 255) return;
    const int s = min(max(140 - e, -100), 100);
    mul = __uint_as_float((uint32_t)(127 + s) << 23);
    c *= __uint_as_float((uint32_t)(127 - s) << 23);
}

// 8 signed bytes as 8 binary16 values, exactly: byte b ^ 0x80 under the exponent of
// 1024 is 1024 + 128 + b
__device__ __forceinline__ pu4_t pg_bytes(pu2_t x) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    pu4_t r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = x[i >> 1] ^ 0x80808080u;
        const uint32_t u = __builtin_amdgcn_perm(0x64646464u, w, (i & 1) ? 0x04030402u : 0x04010400u);
        r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, u) - off);
    }
    return r;
}

__device__ __forceinline__ float pg_max16(float v) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float pg_sum16(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// A value of the cache, one by one (KV: element of K, or of V in its blocks)
template <int FMT, int D>
__device__ __forceinline__ float pg_k(const PagePool &p, size_t head, int slot, int d) {
    const size_t e = (head * p.P + slot) * D + d;
    if constexpr (FMT == FL_KV_F32) return ((const float *)p.k)[e];
    if constexpr (FMT == FL_KV_F16) return h2f(((const uint16_t *)p.k)[e]);
    return (float)((const int8_t *)p.k)[e] * h2f(p.ks[(head * p.P + slot) * (D / 32) + (d >> 5)]);
}
template <int FMT, int D>
__device__ __forceinline__ float pg_v(const PagePool &p, size_t head, int slot, int d) {
    const size_t e = head * p.P * D + ((size_t)(slot >> 5) * D + d) * 32 + (slot & 31);
    if constexpr (FMT == FL_KV_F32) return ((const float *)p.v)[e];
    if constexpr (FMT == FL_KV_F16) return h2f(((const uint16_t *)p.v)[e]);
    return (float)((const int8_t *)p.v)[e] * h2f(p.vs[(head * p.P + slot) * (D / 32) + (d >> 5)]);
}

// Scale of a block of 32 channels, and the factor that its codes are rounded from:
// amax / 127 and 127 / amax from one division (quantize_input_q8_0_into, model.rs:
// 5557-5570, has two: a scale may differ from its in the last place, a code by one
// where the value is next to a half).
__device__ __forceinline__ void pg_q8_scale(float amax, float &scale, float &factor) {
    scale = amax * (1.0f / 127.0f);
    asm("" : "+v"(scale));  // rounded to f32 before binary16 (not v_fma_mixlo_f16's one rounding)
    factor = amax > 0.0f ? 1.0f / amax * 127.0f : 0.0f;
}

// A row's O and sum are kept relative to a maximum that follows its scores only when one
// is over it by 2^kPageLag (nearly every block has a new maximum of some row, and
// bringing O to it is a third of a block's vector work).  p is kept times 2^kPageShift
// where its parts are binary16: at most 2^15, and what its low part loses below 2^-14, if
// products take smaller numbers for 0, is 2^-23 of the largest p.  In 8 bits the parts are
// those of p times V's scale, so the maximum is over the scores with the scale's exponent.
constexpr float kPageLag = 6.0f;
template <int FMT>
constexpr float kPageShift = FMT == FL_KV_F32 ? 0.0f : 9.0f;

// The operands of a 32-slot block of one (page, kv head), in registers.  Scores are
// formed transposed, S^T = K Q^T, with 16 x 16 products: a query row is a lane (mod
// 16), and the K rows of the two tiles t enter so that lane group g = lane / 16 gets
// the scores of slots 8 g + 4 t + 0..3: its probabilities are already the operand of
// O^T = V^T P^T, whose V operand is 8 consecutive slots of a channel, one piece of a
// V block.
//
// K and V in binary16 (or int8, exact in binary16) against q and p in two binary16
// parts: 22 bits of each, so the products lose nothing that f32 would keep.  f32
// caches take the f32 matrix product, K = 4.
template <int FMT, int D>
struct PgBlock;

template <int D>
struct PgBlock<FL_KV_F16, D> {
    static constexpr int QP = D / 32 * 2;  // q operands (pu4_t) of a 16-row tile
    pu4_t k[2][D / 32], v[D / 16];

    __device__ __forceinline__ void load_k(const PagePool &p, size_t head, int slot, int m, int g) {
        const uint16_t *b = (const uint16_t *)p.k + (head * p.P + slot) * D;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int c = 0; c < D / 32; c++)
                k[t][c] = *(const pu4_t *)(b + (8 * (m >> 2) + 4 * t + (m & 3)) * D + 32 * c + 8 * g);
    }
    __device__ __forceinline__ void load_v(const PagePool &p, size_t head, int slot, int m, int g) {
        const uint16_t *b = (const uint16_t *)p.v + (head * p.P + slot) * D;
#pragma unroll
        for (int c = 0; c < D / 16; c++) v[c] = *(const pu4_t *)(b + (16 * c + m) * 32 + 8 * g);
    }
    // slots from `n` on hold no token: whatever is there must not meet a zero
    __device__ __forceinline__ void clip_v(int n, int g) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int s = 8 * g + 2 * i;
            const uint32_t keep = (s < n ? 0xFFFFu : 0u) | (s + 1 < n ? 0xFFFF0000u : 0u);
#pragma unroll
            for (int c = 0; c < D / 16; c++) v[c][i] &= keep;
        }
    }
    static __device__ __forceinline__ void make_q(const float *q, float mul, int g, pu4_t *o) {
#pragma unroll
        for (int c = 0; c < D / 32; c++) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = q[32 * c + 8 * g + j] * mul;
            pg_split(x, o[2 * c], o[2 * c + 1]);
        }
    }
    __device__ __forceinline__ float v_exponent() const { return 0.0f; }
    // of NT tiles of 16 rows: what is made of k and v is made once
    template <int NT, typename Q>
    __device__ __forceinline__ void scores(const Q &q, pf4_t (*s)[2]) const {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                pf4_t lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < D / 32; c++) {
                    lo = pg_mfma_h(k[t][c], q(n, 2 * c + 1), lo);
                    hi = pg_mfma_h(k[t][c], q(n, 2 * c), hi);
                }
                s[n][t] = hi + lo;
            }
    }
    template <int NT>
    __device__ __forceinline__ void add_pv(const float (*p)[8], pf4_t (*o)[D / 16]) const {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            pu4_t hi, lo;
            pg_split(p[n], hi, lo);
#pragma unroll
            for (int c = 0; c < D / 16; c++) {
                o[n][c] = pg_mfma_h(v[c], lo, o[n][c]);
                o[n][c] = pg_mfma_h(v[c], hi, o[n][c]);
            }
        }
    }
};

template <int D>
struct PgBlock<FL_KV_Q8, D> {
    static constexpr int QP = D / 32 * 2;
    pu2_t k[2][D / 32], v[D / 16];
    pu4_t ks[D / 32], vs[D / 32];  // scales of slots 8 g + 0..7: value i of [slot][D / 32]

    __device__ __forceinline__ void load_k(const PagePool &p, size_t head, int slot, int m, int g) {
        const int8_t *b = (const int8_t *)p.k + (head * p.P + slot) * D;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int c = 0; c < D / 32; c++)
                k[t][c] = *(const pu2_t *)(b + (8 * (m >> 2) + 4 * t + (m & 3)) * D + 32 * c + 8 * g);
        const pu4_t *s = (const pu4_t *)(p.ks + (head * p.P + slot + 8 * g) * (D / 32));
#pragma unroll
        for (int i = 0; i < D / 32; i++) ks[i] = s[i];
    }
    __device__ __forceinline__ void load_v(const PagePool &p, size_t head, int slot, int m, int g) {
        const int8_t *b = (const int8_t *)p.v + (head * p.P + slot) * D;
#pragma unroll
        for (int c = 0; c < D / 16; c++) v[c] = *(const pu2_t *)(b + (16 * c + m) * 32 + 8 * g);
        const pu4_t *s = (const pu4_t *)(p.vs + (head * p.P + slot + 8 * g) * (D / 32));
#pragma unroll
        for (int i = 0; i < D / 32; i++) vs[i] = s[i];
    }
    // (codes are finite: only the scales of slots without a token must not meet a zero)
    __device__ __forceinline__ void clip_v(int n, int g) {
#pragma unroll
        for (int i = 0; i < D / 32; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int s0 = 8 * g + (8 * i + 2 * j) / (D / 32), s1 = 8 * g + (8 * i + 2 * j + 1) / (D / 32);
                vs[i][j] &= (s0 < n ? 0xFFFFu : 0u) | (s1 < n ? 0xFFFF0000u : 0u);
            }
    }
    // a power of two over the scales of the lane's slots
    __device__ __forceinline__ float v_exponent() const {
        typedef uint16_t u2 __attribute__((ext_vector_type(2)));
        u2 m = {0, 0};
#pragma unroll
        for (int i = 0; i < D / 32; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) m = __builtin_elementwise_max(m, __builtin_bit_cast(u2, vs[i][j]));
        return (float)(max((int)m[0], (int)m[1]) >> 10) - 14.0f;
    }
    static __device__ __forceinline__ void make_q(const float *q, float mul, int g, pu4_t *o) {
        PgBlock<FL_KV_F16, D>::make_q(q, mul, g, o);
    }
    template <int NT, typename Q>
    __device__ __forceinline__ void scores(const Q &q, pf4_t (*s)[2]) const {
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int n = 0; n < NT; n++) s[n][t] = pf4_t{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
                const pu4_t a = pg_bytes(k[t][c]);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    pf4_t d = pg_mfma_h(a, q(n, 2 * c + 1), pf4_t{0, 0, 0, 0});
                    d = pg_mfma_h(a, q(n, 2 * c), d);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int at = (4 * t + i) * (D / 32) + c;  // (even D / 32: its parity is c's)
                        s[n][t][i] = pg_fma_mix(d[i], ks[at >> 3][(at & 7) >> 1], c & 1, s[n][t][i]);
                    }
                }
            }
        }
    }
    template <int NT>
    __device__ __forceinline__ void add_pv(const float (*p)[8], pf4_t (*o)[D / 16]) const {
        const float minus = pg_minus_one();
#pragma unroll
        for (int c = 0; c < D / 32; c++) {
            pu4_t hi[NT], lo[NT];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                // the scales of two neighbouring slots, side by side
                const int a0 = 2 * j * (D / 32) + c, a1 = a0 + D / 32;
                const uint32_t w0 = vs[a0 >> 3][(a0 & 7) >> 1], w1 = vs[a1 >> 3][(a1 & 7) >> 1];
                const uint32_t s = __builtin_amdgcn_perm(w1, w0, (c & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    uint32_t h, l;
                    pg_split2(pg_fma_mix(p[n][2 * j], s, 0, 0.0f), pg_fma_mix(p[n][2 * j + 1], s, 1, 0.0f), minus, h, l);
                    hi[n][j] = h;
                    lo[n][j] = l;
                }
            }
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const pu4_t a = pg_bytes(v[2 * c + u]);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    o[n][2 * c + u] = pg_mfma_h(a, lo[n], o[n][2 * c + u]);
                    o[n][2 * c + u] = pg_mfma_h(a, hi[n], o[n][2 * c + u]);
                }
            }
        }
    }
};

template <int D>
struct PgBlock<FL_KV_F32, D> {
    static constexpr int QP = D / 16;
    pf4_t k[2][D / 16], v[D / 16][2];

    __device__ __forceinline__ void load_k(const PagePool &p, size_t head, int slot, int m, int g) {
        const float *b = (const float *)p.k + (head * p.P + slot) * D;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int c = 0; c < D / 16; c++)
                k[t][c] = *(const pf4_t *)(b + (8 * (m >> 2) + 4 * t + (m & 3)) * D + 16 * c + 4 * g);
    }
    __device__ __forceinline__ void load_v(const PagePool &p, size_t head, int slot, int m, int g) {
        const float *b = (const float *)p.v + (head * p.P + slot) * D;
#pragma unroll
        for (int c = 0; c < D / 16; c++)
#pragma unroll
            for (int t = 0; t < 2; t++) v[c][t] = *(const pf4_t *)(b + (16 * c + m) * 32 + 8 * g + 4 * t);
    }
    __device__ __forceinline__ void clip_v(int n, int g) {
#pragma unroll
        for (int c = 0; c < D / 16; c++)
#pragma unroll
            for (int j = 0; j < 8; j++) v[c][j >> 2][j & 3] = 8 * g + j < n ? v[c][j >> 2][j & 3] : 0.0f;
    }
    __device__ __forceinline__ float v_exponent() const { return 0.0f; }
    static __device__ __forceinline__ void make_q(const float *q, float mul, int g, pu4_t *o) {
#pragma unroll
        for (int c = 0; c < D / 16; c++)
#pragma unroll
            for (int j = 0; j < 4; j++) o[c][j] = __float_as_uint(q[16 * c + 4 * g + j] * mul);
    }
    template <int NT, typename Q>
    __device__ __forceinline__ void scores(const Q &q, pf4_t (*s)[2]) const {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                s[n][t] = pf4_t{0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < D / 16; c++) {
                    const pu4_t w = q(n, c);
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        s[n][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][c][j], __uint_as_float(w[j]), s[n][t], 0, 0, 0);
                }
            }
    }
    template <int NT>
    __device__ __forceinline__ void add_pv(const float (*p)[8], pf4_t (*o)[D / 16]) const {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int c = 0; c < D / 16; c++)
#pragma unroll
                for (int j = 0; j < 8; j++)
                    o[n][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[c][j >> 2][j & 3], p[n][j], o[n][c], 0, 0, 0);
    }
};

constexpr bool pg_q_in_lds(int fmt, int D, int nt) { return fmt == FL_KV_Q8 && nt == 2 && D == 128; }
// The query operands of NT tiles: registers, or (LDS) the same of all waves in LDS, for the
// forms whose registers would not do for two waves a SIMD.
template <int NT, int QP, bool LDS>
struct PgQ {
    pu4_t r[NT][QP];
    __device__ __forceinline__ const pu4_t &operator()(int n, int i) const { return r[n][i]; }
};
template <int NT, int QP>
struct PgQ<NT, QP, true> {
    const pu4_t *base;
    int at;  // the lane's
    __device__ __forceinline__ pu4_t operator()(int n, int i) const { return base[at + (n * QP + i) * 64]; }
};

// Where an item's blocks are.  Its page numbers go through the scalar cache, asked for a
// block (or step) ahead: as vector loads they would wait behind the keys' and values'.
struct PgWalk {
    const __attribute__((address_space(4))) int *ids;
    int blk0, first, per;
    uint32_t inv;
    __device__ __forceinline__ int page_of(int blk) const { return inv ? (int)(((uint64_t)(uint32_t)blk * inv) >> 32) : blk; }
    __device__ __forceinline__ PgWalk(const PageAttnArgs &a, const PageItem &it)
        : ids((const __attribute__((address_space(4))) int *)(a.page_ids + it.page0)), blk0(it.slot0 >> 5), per(a.pool.per),
          inv(a.pool.per_inv) {
        first = page_of(blk0);
    }
    __device__ __forceinline__ int page(int b) const { return ids[page_of(blk0 + b) - first]; }
    // first slot of block b in its page
    __device__ __forceinline__ int slot(int b) const { return 32 * (blk0 + b - page_of(blk0 + b) * per); }
};
// An item, through the scalar cache
__device__ __forceinline__ PageItem pg_item(const PageAttnArgs &a, int i) {
    typedef int i8_t __attribute__((ext_vector_type(8)));
    const i8_t w = ((const __attribute__((address_space(4))) i8_t *)a.items)[i];
    return PageItem{w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]};
}

// A value of a partial result.  HERE: another workgroup of the launch reads it.
template <bool HERE>
__device__ __forceinline__ void pg_put(float *p, float v) {
    if constexpr (HERE) st_agent(p, v);
    else *p = v;
}

// An item's rows key by key, where some value was not finite: 2^kShift times the
// sum and O, in base 2 relative to the largest score, as the tiles have them (all rows
// of the item; this is rare).  lds: 260 floats.
template <int FMT, int D, bool HERE>
__device__ __forceinline__ void pg_rows_again(const PageAttnArgs &a, const PageItem &it, int kvh, float *lds) {
    const int nkv = a.pool.nkv, G = a.group, nh = nkv * G, P = a.pool.P, rows = it.nq * G;
    const size_t layer_pages = (size_t)a.layer * a.pool.pages;
    const int tid = threadIdx.x;
    float *sc = lds, *red = lds + 256;
    auto head_of = [&](int t) { return (layer_pages + a.page_ids[it.page0 + t / P - it.slot0 / P]) * nkv + kvh; };
    for (int row = 0; row < rows; row++) {
        const int qi = row / G, hd = kvh * G + row % G;
        const PageQuery pq = a.order[it.q0 + qi];
        const float *qp = a.q + pq.query * a.q_stride + (size_t)hd * D;
        const int end = min(pq.seen, it.slot1);
        float mx = -INFINITY, sum = 0.0f, acc = 0.0f;
        for (int t0 = it.slot0; t0 < end; t0 += 256) {
            const int t = t0 + tid;
            float x = -INFINITY;
            if (tid < 256 && t < end) {
                x = 0.0f;
                for (int d = 0; d < D; d++) x = __builtin_fmaf(qp[d], pg_k<FMT, D>(a.pool, head_of(t), t % P, d), x);
                x *= a.scale;
            }
            __syncthreads();
            if (tid < 256) sc[tid] = x;
            for (int i = 1; i < 64; i <<= 1) x = fmaxf(x, __shfl_xor(x, i, 64));
            if (tid < 256 && (tid & 63) == 0) red[tid >> 6] = x;
            __syncthreads();
            const float mn = fmaxf(mx, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
            const float al = mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mx - mn);
            sum *= al;
            acc *= al;
            mx = mn;
            for (int i = 0; i < 256 && t0 + i < end; i++) {
                const float y = sc[i], p = y == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(y - mx + kPageShift<FMT>);
                sum += p;
                if (tid < D) acc = __builtin_fmaf(p, pg_v<FMT, D>(a.pool, head_of(t0 + i), (t0 + i) % P, tid), acc);
            }
        }
        __syncthreads();
        if (tid >= D) continue;
        if (it.unit < 0) {
            a.out[((size_t)pq.query * nh + hd) * D + tid] = acc / sum;
        } else {
            const size_t u = (size_t)(it.unit + qi) * nh + hd;
            pg_put<HERE>(a.part + u * D + tid, acc);
            if (tid == 0) {
                pg_put<HERE>(a.ml + u * 2, mx);
                pg_put<HERE>(a.ml + u * 2 + 1, sum);
            }
        }
    }
}

// An item's query rows into LDS, LROW floats apart (read from memory by the lanes that
// need them, a load is 32 or 64 lines: 10 us of a 128-row item's prologue).
template <int D, int LROW, int NTHR>
__device__ __forceinline__ void pg_stage_q(const PageAttnArgs &a, const PageItem &it, int kvh, float *lds) {
    constexpr int TR = D / 4;
    const int G = a.group, rows = it.nq * G, c = threadIdx.x % TR * 4;
#pragma unroll 4
    for (int r = threadIdx.x / TR; r < rows; r += NTHR / TR) {
        const int qi = r / G;
        const float *src = a.q + a.order[it.q0 + qi].query * a.q_stride + (size_t)(kvh * G + r - qi * G) * D + c;
        *(pf4_t *)(lds + r * LROW + c) = pf4_t{src[0], src[1], src[2], src[3]};
    }
}

// A row of an item's result: channels ch .. ch + 3 from the KL partial results at
// lds[i * step], each [D] O, max, sum.  Sets *bad where a value is not finite.
template <int D, int KL, bool HERE>
__device__ __forceinline__ void pg_join_row(const PageAttnArgs &a, const PageItem &it, int kvh, int row, int ch,
                                            const float *lds, int step, int *bad) {
    float mx = -INFINITY, sum = 0.0f, wt[KL];
#pragma unroll
    for (int i = 0; i < KL; i++) mx = fmaxf(mx, lds[i * step + D]);
#pragma unroll
    for (int i = 0; i < KL; i++) {
        const float mi = lds[i * step + D];
        wt[i] = mi == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mi - mx);
        sum = __builtin_fmaf(lds[i * step + D + 1], wt[i], sum);
    }
    float odd = sum * 0.0f;
    const int G = a.group, nh = a.pool.nkv * G, qi = row / G, hd = kvh * G + row % G;
    const size_t u = (size_t)(it.unit < 0 ? a.order[it.q0 + qi].query : it.unit + qi) * nh + hd;
    float *op = (it.unit < 0 ? a.out : a.part) + u * D + ch;
    const float il = it.unit < 0 ? 1.0f / sum : 1.0f;
    pf4_t y = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < KL; i++) {
        const pf4_t x = *(const pf4_t *)(lds + i * step + ch);
#pragma unroll
        for (int k = 0; k < 4; k++) y[k] = __builtin_fmaf(x[k], wt[i], y[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
        y[k] *= il;
        odd = __builtin_fmaf(y[k], 0.0f, odd);
    }
    if (!HERE || it.unit < 0) {
        *(pf4_t *)op = y;
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) st_agent(op + k, y[k]);
    }
    if (it.unit >= 0 && ch == 0) {
        pg_put<HERE>(a.ml + u * 2, mx);
        pg_put<HERE>(a.ml + u * 2 + 1, sum);
    }
    if (odd != 0.0f) *bad = 1;  // 0 * Inf and 0 * NaN are NaN
}

// Items of up to 16 NT rows (query x head): NW waves, wave w takes the item's 32-slot
// blocks w, w + NW, ..  Each keeps (max, sum, O) of its blocks for NT x 16 rows, joined
// through LDS at the end ([NW][16][D + 4] floats: O, max, sum of one tile).  K of a wave's
// next block is loaded when the scores have been formed, V when O has been: half a
// block ahead.  Bound by the memory: a block is 16 NT products for 16 KB (D = 128, binary16).
//
// Values that are not finite: slots behind the item's last token are taken out of V;
// a token that some of the item's queries see and others do not has p = 0 for the
// latter, and 0 * Inf is NaN, as is an Inf against a zero low part.  Every such case
// leaves a NaN or Inf in O: such a row is then formed again, key by key.
template <int FMT, int D, int NT, int NW, bool HERE>
__device__ __forceinline__ void pg_narrow(const PageAttnArgs &a, const PageItem &it, int kvh, float *lds, int *bad) {
    using Block = PgBlock<FMT, D>;
    constexpr bool QL = pg_q_in_lds(FMT, D, NT);
    constexpr int QP = Block::QP, DT = D / 16, LROW = D + 4;
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nkv = a.pool.nkv, G = a.group;
    const int rows = it.nq * G, P = a.pool.P;
    const int nb = (it.slot1 - it.slot0 + 31) >> 5;
    const size_t layer_pages = (size_t)a.layer * a.pool.pages;

    const PgWalk walk(a, it);
    const int last = nb - 1;
    Block blk;
    int b0 = min(wave, last), b1 = min(wave + NW, last);  // this block and the next: past the end, the last one
    int page = walk.page(b1);
    {
        const size_t head = (layer_pages + walk.page(b0)) * nkv + kvh;
        blk.load_k(a.pool, head, walk.slot(b0), m, g);
        blk.load_v(a.pool, head, walk.slot(b0), m, g);
    }

    pg_stage_q<D, LROW, 64 * NW>(a, it, kvh, lds);
    __syncthreads();
    PgQ<NT, QP, QL> q;
    pu4_t *ql = (pu4_t *)(lds + NW * 16 * LROW);  // behind the join's
    float c[NT];
    int seen[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int r = min(16 * n + m, rows - 1);
        seen[n] = a.order[it.q0 + r / G].seen;
        const float *qp = lds + r * LROW;
        c[n] = a.scale;
        float mul = 1.0f;
        if constexpr (FMT != FL_KV_F32) {
            float x = 0.0f;
#pragma unroll
            for (int k = 0; k < D / 32; k++)
#pragma unroll
                for (int j = 0; j < 8; j++) x = fmaxf(x, fabsf(qp[32 * k + 8 * g + j]));
            pg_q_scale(pg_max16(x), mul, c[n]);
        }
        if constexpr (QL) {
            if (wave != n) continue;
            pu4_t w[QP];
            Block::make_q(qp, mul, g, w);
#pragma unroll
            for (int i = 0; i < QP; i++) ql[(n * QP + i) * 64 + lane] = w[i];
        } else {
            Block::make_q(qp, mul, g, q.r[n]);
        }
    }
    if constexpr (QL) {
        q.base = ql;
        q.at = lane;
        __syncthreads();
    }
    pf4_t o[NT][DT];
    float m_run[NT], l_run[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        m_run[n] = -INFINITY;
        l_run[n] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++) o[n][d] = pf4_t{0, 0, 0, 0};
    }

    for (int b = wave; b < nb; b += NW) {
        const int tok = it.slot0 + 32 * b;  // first token of the block
        pf4_t s[NT][2];
        if constexpr (QL) asm volatile("" : "+v"(q.at));  // read again, not kept in registers
        blk.template scores<NT>(q, s);
        const size_t head = (layer_pages + page) * nkv + kvh;
        const int slot = walk.slot(b1);
        blk.load_k(a.pool, head, slot, m, g);
        b1 = min(b1 + NW, last);
        page = walk.page(b1);
        if (tok + 32 > it.smin) {  // some query does not see every token
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (tok + 8 * g + j >= min(seen[n], it.slot1)) s[n][j >> 2][j & 3] = -INFINITY;
            if (tok + 32 > it.slot1) blk.clip_v(it.slot1 - tok, g);
        }
        float p[NT][8];
        const float ve = blk.v_exponent();
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float x = s[n][0][0];
#pragma unroll
            for (int j = 1; j < 8; j++) x = fmaxf(x, s[n][j >> 2][j & 3]);
            x = pg_max16(__builtin_fmaf(x, c[n], ve));
            if (__any(x > m_run[n] + kPageLag)) {
                const float mn = fmaxf(m_run[n], x);
                const float al = m_run[n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run[n] - mn);
                m_run[n] = mn;
                l_run[n] *= al;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[n][d][i] *= al;
            }
            // (a row that has seen no token yet has scores of -Inf alone, and p = 0)
            const float off = m_run[n] == -INFINITY ? -INFINITY : kPageShift<FMT> - m_run[n];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                p[n][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][j >> 2][j & 3], c[n], off));
                l_run[n] += p[n][j];
            }
        }
        blk.template add_pv<NT>(p, o);
        blk.load_v(a.pool, head, slot, m, g);
    }

    // join the waves, one 16-row tile at a time
#pragma unroll
    for (int n = 0; n < NT; n++) {
        if (16 * n >= rows) break;
        __syncthreads();
        float *w = lds + (16 * wave + m) * LROW;
#pragma unroll
        for (int d = 0; d < DT; d++) *(pf4_t *)(w + 16 * d + 4 * g) = o[n][d];
        const float l = pg_sum16(l_run[n]);
        if (g == 0) {
            w[D] = m_run[n];
            w[D + 1] = l;
        }
        __syncthreads();
        for (int r = threadIdx.x / (D / 4); r < min(16, rows - 16 * n); r += 64 * NW / (D / 4))
            pg_join_row<D, NW, HERE>(a, it, kvh, 16 * n + r, threadIdx.x % (D / 4) * 4, lds + r * LROW, 16 * LROW, bad);
    }
}

// Items of up to 32 R rows, binary16: 8 waves, R row groups of 32 x 8 / R key lanes.  A step
// is 128 tokens, K and V of its four 32-slot blocks copied memory -> LDS one step ahead
// (wave w copies K or V of one block); a key lane takes R / 2 of them.  Products are
// 32 x 32 x 16: a query row is a lane (mod 32), the K rows enter with index bits 2 and 3
// swapped so that scores i = 8 mm + j of a lane are slots 16 mm + 8 (lane / 32) + j, the
// operand of O^T = V^T P^T.  smem: two steps of K and V; at the end [8][32][D + 4] floats.
template <int D, int R, bool HERE>
__device__ __forceinline__ void pg_wide(const PageAttnArgs &a, const PageItem &it, int kvh, char *smem, int *bad) {
    constexpr int FMT = FL_KV_F16, KL = 8 / R, NB = 4 / KL;
    constexpr int KS = D / 16, DT = D / 32, CH = D / 8, BLK = 32 * D * 2;  // BLK: bytes of a block's K (or V)
    constexpr int LROW = D + 4;
    const int lane = threadIdx.x & 63, l31 = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rg = wave % R, kl = wave / R;
    const int nkv = a.pool.nkv, G = a.group;
    const int rows = it.nq * G, P = a.pool.P;
    const int nb = (it.slot1 - it.slot0 + 31) >> 5, nit = (nb + 3) >> 2;
    const size_t layer_pages = (size_t)a.layer * a.pool.pages;
    const bool live = 32 * rg < rows;  // wave-uniform

    // chunk p (16 B) of a K block in LDS holds chunk c ^ g(row) of its row, g from row bits
    // 0, 1, 3 (the rows that 8 lanes read together differ in those); of a V block, chunk
    // c ^ (channel >> 1 & 3) of its channel.  A copy of 64 chunks: the lane's place among
    // them, but for row bit 3, which is a bit of the copy's number.
    const int r8 = lane / CH;
    const int kplace = 16 * (r8 * CH + ((lane % CH) ^ (r8 & 3))), vplace = 16 * ((lane & ~3) | ((lane & 3) ^ ((lane >> 3) & 3)));
    const PgWalk walk(a, it);
    int page = walk.page(min(wave & 3, nb - 1));
    auto copy = [&](int step, int buf) {
        const int b = min(4 * step + (wave & 3), nb - 1);
        const size_t at = (((layer_pages + page) * nkv + kvh) * P + walk.slot(b)) * D * 2;
        page = walk.page(min(b + 4, nb - 1));  // the next step's
        char *dst = smem + (size_t)(8 * buf + wave) * BLK;
        if (wave < 4) {
#pragma unroll
            for (int u = 0; u < BLK / 1024; u++)
                copy_to_lds((const char *)a.pool.k + at + u * 1024 + (((u * 64 / CH) & 8) ? kplace ^ 64 : kplace), dst + u * 1024);
        } else {
#pragma unroll
            for (int u = 0; u < BLK / 1024; u++)
                copy_to_lds((const char *)a.pool.v + at + u * 1024 + vplace, dst + u * 1024);
        }
    };
    copy(0, 0);

    // the queries, in the second buffer until its first copy
    float *lds = (float *)smem, *ql = (float *)(smem + 8 * BLK);
    pg_stage_q<D, LROW, 512>(a, it, kvh, ql);
    __syncthreads();
    const int r0 = min(32 * rg + l31, rows - 1);
    const int seen = a.order[it.q0 + r0 / G].seen;
    const float *qp = ql + r0 * LROW + 8 * h;
    float c = a.scale, mul = 1.0f, x0 = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
        for (int j = 0; j < 8; j++) x0 = fmaxf(x0, fabsf(qp[16 * k + j]));
    pg_q_scale(fmaxf(x0, __shfl_xor(x0, 32, 64)), mul, c);
    pu4_t q[KS][2];
#pragma unroll
    for (int k = 0; k < KS; k++) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = qp[16 * k + j] * mul;
        pg_split(x, q[k][0], q[k][1]);
    }
    const pf16_t zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    pf16_t o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = zero;
    float m_run = -INFINITY, l_run = 0.0f;
    const int krow = (l31 & 0x13) | ((l31 & 4) << 1) | ((l31 & 8) >> 1);
    const int kg = (krow & 3) | ((krow >> 1) & 4);
    // of its K row, chunk 2 k + h: 4 places, and those 128 B behind; of a V block, chunk 2 mm + h of channel l31
    int kat[4], vat[2];
#pragma unroll
    for (int k = 0; k < 4; k++) kat[k] = krow * D * 2 + (((2 * k + h) ^ kg) * 16);
#pragma unroll
    for (int mm = 0; mm < 2; mm++) vat[mm] = l31 * 64 + (((2 * mm + h) ^ ((l31 >> 1) & 3)) * 16);

    for (int step = 0; step < nit; step++) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();  // this step has landed, and nobody reads the other buffer
        asm volatile("" ::: "memory");
        const int buf = step & 1;
        if (step + 1 < nit) {
            copy(step + 1, buf ^ 1);
        } else if (const int over = (it.slot1 - it.slot0) & 31; over) {
            // slots behind the item's last token: whatever is there must not meet a zero
            char *vb = smem + (size_t)(8 * buf + 4 + ((nb - 1) & 3)) * BLK;
            for (int i = threadIdx.x; i < 32 * D; i += 512) {
                const int d = i >> 5, s = i & 31;
                if (s >= over) *(uint16_t *)(vb + d * 64 + (((s >> 3) ^ ((d >> 1) & 3)) * 16) + (s & 7) * 2) = 0;
            }
            __syncthreads();
        }
        if (!live) continue;
        // Operands are read from LDS a phase ahead: V before the softmax, the next
        // block's K between the products with V.
        pu4_t kf[KS], vf[DT][2];
        auto load_k = [&](int bi) {
            const char *kt = smem + (size_t)(8 * buf + bi) * BLK;
#pragma unroll
            for (int k = 0; k < KS; k++) kf[k] = *(const pu4_t *)(kt + kat[k & 3] + (k >> 2) * 128);
        };
        load_k(NB * kl);
#pragma unroll
        for (int i = 0; i < NB; i++) {
            const int bi = NB * kl + i, tok = it.slot0 + 32 * (4 * step + bi);
            if (tok >= it.slot1) break;
            pf16_t s = zero;
#pragma unroll
            for (int k = 0; k < KS; k++) s = pg_mfma_w(kf[k], q[k][1], s);
#pragma unroll
            for (int k = 0; k < KS; k++) s = pg_mfma_w(kf[k], q[k][0], s);
            const char *vt = smem + (size_t)(8 * buf + 4 + bi) * BLK;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int mm = 0; mm < 2; mm++) vf[d][mm] = *(const pu4_t *)(vt + vat[mm] + d * 2048);
            __builtin_amdgcn_sched_barrier(0);
            if (tok + 32 > it.smin) {  // some query does not see every token
                const int end = min(seen, it.slot1) - tok;
#pragma unroll
                for (int j = 0; j < 16; j++)
                    if (16 * (j >> 3) + 8 * h + (j & 7) >= end) s[j] = -INFINITY;
            }
            float m = s[0];
#pragma unroll
            for (int j = 1; j < 16; j++) m = fmaxf(m, s[j]);
            m = fmaxf(m, __shfl_xor(m, 32, 64)) * c;
            if (__any(m > m_run + kPageLag)) {
                const float mn = fmaxf(m_run, m);
                const float al = m_run == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - mn);
                m_run = mn;
                l_run *= al;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int j = 0; j < 16; j++) o[d][j] *= al;
            }
            // (a row that has seen no token yet has scores of -Inf alone, and p = 0)
            const float off = m_run == -INFINITY ? -INFINITY : kPageShift<FMT> - m_run;
            float p[16];
#pragma unroll
            for (int j = 0; j < 16; j++) {
                p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j], c, off));
                l_run += p[j];
            }
            pu4_t pf[2][2];
            pg_split(p, pf[0][0], pf[0][1]);
            pg_split(p + 8, pf[1][0], pf[1][1]);
#pragma unroll
            for (int mm = 0; mm < 2; mm++) {
#pragma unroll
                for (int u = 1; u >= 0; u--)
#pragma unroll
                    for (int d = 0; d < DT; d++) o[d] = pg_mfma_w(vf[d][mm], pf[mm][u], o[d]);
                if (mm == 0) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (i + 1 < NB) load_k(bi + 1);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    }
    __syncthreads();
    if (live) {
        float *w = lds + (size_t)(32 * wave + l31) * LROW;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                *(pf4_t *)(w + 32 * d + 8 * i + 4 * h) = pf4_t{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
        const float l = l_run + __shfl_xor(l_run, 32, 64);
        if (h == 0) {
            w[D] = m_run;
            w[D + 1] = l;
        }
    }
    __syncthreads();
    for (int r = threadIdx.x / (D / 4); r < rows; r += 512 / (D / 4))
        pg_join_row<D, KL, HERE>(a, it, kvh, r, threadIdx.x % (D / 4) * 4, lds + (size_t)r * LROW, 32 * R * LROW, bad);
}

// Partial results of a query and head, N of them in flight, into o, l relative to mx
struct PgSum {
    float mx = -INFINITY, l = 0.0f;
    pf4_t o = {0, 0, 0, 0};
    // parts first, first + step, ..; value(unit index, ml, o)
    template <int N, typename F>
    __device__ __forceinline__ void add(int first, int end, int step, F value) {
        for (int i = first; i < end; i += step * N) {
            float2 ml[N];
            pf4_t p[N];
#pragma unroll
            for (int k = 0; k < N; k++) value(min(i + step * k, end - 1), ml[k], p[k]);
            float mn = mx;
#pragma unroll
            for (int k = 0; k < N; k++) mn = fmaxf(mn, ml[k].x);
            const float al = mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mx - mn);
            mx = mn;
            l *= al;
#pragma unroll
            for (int x = 0; x < 4; x++) o[x] *= al;
#pragma unroll
            for (int k = 0; k < N; k++) {
                if (i + step * k >= end) break;
                const float w = ml[k].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml[k].x - mx);
                l = __builtin_fmaf(ml[k].y, w, l);
#pragma unroll
                for (int x = 0; x < 4; x++) o[x] = __builtin_fmaf(p[k][x], w, o[x]);
            }
        }
    }
};

// At the end of an item: joins the queries of which this workgroup has the last part for
// its kv head to arrive, in the order of the plan whichever that is.  Parts are stored and
// read past the XCDs' caches (st_agent, ld_agent), a wave's before its workgroup counts.
// last: NTHR / 4 ints of LDS (an item has as many queries at most).
template <int D, int NTHR>
__device__ __forceinline__ void pg_join_here(const PageAttnArgs &a, const PageItem &it, int kvh, int *last) {
    const int nkv = a.pool.nkv, G = a.group, nh = nkv * G, tid = threadIdx.x;
    if (blockIdx.x < (unsigned)nkv)
        for (int i = tid; i < a.nempty * G * D; i += NTHR)
            a.out[((size_t)a.joins[a.njoins - 1 - i / (G * D)].query * nh + kvh * G) * D + i % (G * D)] = 0.0f;
    if (it.unit < 0) return;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid < it.nq) {
        const int j = a.join_of[a.order[it.q0 + tid].query];
        int *c = a.arrived + (size_t)j * nkv + kvh;
        const bool mine = __hip_atomic_fetch_add(c, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.joins[j].count - 1;
        if (mine) __hip_atomic_store(c, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last[tid] = mine ? j : -1;
    }
    __syncthreads();
    const int per = G * (D / 4);  // threads of a query
    for (int i = tid; i < it.nq * per; i += NTHR) {
        const int qi = i / per, e = i - qi * per, hd = kvh * G + e / (D / 4), ch = e % (D / 4) * 4;
        if (last[qi] < 0) continue;
        const PageJoin j = a.joins[last[qi]];
        PgSum s;
        s.add<8>(0, j.count, 1, [&](int k, float2 &ml, pf4_t &p) {
            const size_t u = (size_t)a.units[j.first + k] * nh + hd;
            ml = ld_agent2(a.ml + u * 2);
            const float2 x = ld_agent2(a.part + u * D + ch), y = ld_agent2(a.part + u * D + ch + 2);
            p = pf4_t{x.x, x.y, y.x, y.y};
        });
        const float il = 1.0f / s.l;
        *(pf4_t *)(a.out + ((size_t)j.query * nh + hd) * D + ch) = pf4_t{s.o[0] * il, s.o[1] * il, s.o[2] * il, s.o[3] * il};
    }
}

// One item (PageItem) and kv head per workgroup; the kv head is the faster index, so that
// with 8 of them the items of a head share an XCD's L2.

// Items of up to 16 rows (FORMS = 1), or up to 32: 4 waves.  HERE: partial results are joined in
// the launch (a kernel of its own: with the code of it, but not taken, 32 sequences over 8 bits
// 25.2 us against 24.4).
template <int FMT, int D, int FORMS, bool HERE>
__global__ __launch_bounds__(256, page_waves(FMT, D, FORMS)) void k_pages_attn(PageAttnArgs a) {
    __shared__ __align__(16) float lds[4 * 16 * (D + 4) + (pg_q_in_lds(FMT, D, FORMS) ? FORMS * PgBlock<FMT, D>::QP * 256 : 0)];
    __shared__ int bad;
    const int kvh = blockIdx.x % a.pool.nkv;
    const PageItem it = pg_item(a, blockIdx.x / a.pool.nkv);
    if (threadIdx.x == 0) bad = 0;
    if (FORMS == 1 || it.form == 0) pg_narrow<FMT, D, 1, 4, HERE>(a, it, kvh, lds, &bad);
    else pg_narrow<FMT, D, FORMS, 4, HERE>(a, it, kvh, lds, &bad);
    __syncthreads();
    if (bad) pg_rows_again<FMT, D, HERE>(a, it, kvh, lds);
    if constexpr (HERE) pg_join_here<D, 256>(a, it, kvh, (int *)lds);
}

// binary16, items of up to 128 rows: 8 waves, one workgroup a CU.  (In one launch, so that
// items of many rows, which the matrix cores bound, run beside those of few, which the
// memory does.)
template <int D, bool HERE>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_pages_attn_wide(PageAttnArgs a) {
    extern __shared__ __align__(16) char smem[];
    __shared__ int bad;
    const int kvh = blockIdx.x % a.pool.nkv;
    const PageItem it = pg_item(a, blockIdx.x / a.pool.nkv);
    if (threadIdx.x == 0) bad = 0;
    if (it.form == 0) pg_narrow<FL_KV_F16, D, 1, 8, HERE>(a, it, kvh, (float *)smem, &bad);
    else if (it.form == 1) pg_wide<D, 2, HERE>(a, it, kvh, smem, &bad);
    else pg_wide<D, 4, HERE>(a, it, kvh, smem, &bad);
    __syncthreads();
    if (bad) pg_rows_again<FL_KV_F16, D, HERE>(a, it, kvh, (float *)smem);
    if constexpr (HERE) pg_join_here<D, 512>(a, it, kvh, (int *)smem);
}

// Partial results of a query joined: a workgroup takes 128 channels, 4 a thread, and
// 8 of its threads share each channel's parts (one thread for all of them took 25 us for
// the 64 parts of a single query of 16384 tokens, so 4).  grid (queries, heads * D / 128)
template <int D>
__global__ __launch_bounds__(256) void k_pages_join(PageJoinArgs a) {
    constexpr int U = 4;
    __shared__ __align__(16) float lds[8][32][4];
    __shared__ float lml[8][32][2];
    const PageJoin j = a.joins[blockIdx.x];
    const int c = threadIdx.x & 31, s = threadIdx.x >> 5;
    const int e = blockIdx.y * 128 + 4 * c, ec = min(e, a.heads * D - 4), hd = ec / D, n = j.count;
    PgSum part;
    part.add<U>(s, n, 8, [&](int i, float2 &ml, pf4_t &p) {
        const size_t u = (size_t)a.units[j.first + i] * a.heads + hd;
        ml = *(const float2 *)(a.ml + u * 2);
        p = *(const pf4_t *)(a.part + u * D + ec % D);
    });
    *(pf4_t *)lds[s][c] = part.o;
    lml[s][c][0] = part.mx;
    lml[s][c][1] = part.l;
    __syncthreads();
    if (s) return;
    float mx = part.mx, l;
    for (int i = 1; i < 8; i++) mx = fmaxf(mx, lml[i][c][0]);
    float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float mi = lml[i][c][0], w = mi == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mi - mx);
        l = __builtin_fmaf(lml[i][c][1], w, l);
#pragma unroll
        for (int x = 0; x < 4; x++) y[x] = __builtin_fmaf(lds[i][c][x], w, y[x]);
    }
    const float il = n ? 1.0f / l : 0.0f;
    if (e < a.heads * D) *(pf4_t *)(a.out + (size_t)j.query * a.heads * D + e) = pf4_t{y[0] * il, y[1] * il, y[2] * il, y[3] * il};
}

__device__ __forceinline__ PageRun pg_run(const PageRuns &r, int i) { return r.list ? r.list[i] : r.some[i]; }
// A value as the cache holds it
template <int FMT>
using PgElem = std::conditional_t<FMT == FL_KV_F32, float, std::conditional_t<FMT == FL_KV_F16, uint16_t, int8_t>>;

// f32 rows into the slots of a block: a workgroup takes the tokens of one run, one kv head
// and layer.  A thread has 4 channels of a token; V is turned in LDS, so that a full block
// leaves in pieces of 16 bytes and a part of one in consecutive slots.  Bound by the memory
// (a thread for 32 channels with 32 scattered stores took 39 us for 2209 tokens of 8 x 128 in
// 8 bits, this 9.2).  grid (runs, kv heads, layers)
template <int FMT, int D>
__global__ __launch_bounds__(256) void k_pages_write(PageWriteArgs a, PageRuns runs) {
    using E = PgElem<FMT>;
    constexpr int TR = D / 4, PAD = 36;  // threads of a row; elements between V's channels in LDS
    __shared__ __align__(16) E vt[D * PAD];
    const PageRun run = pg_run(runs, blockIdx.x);
    const int kvh = blockIdx.y, layer = blockIdx.z;
    const int page = run.block / a.pool.per, slot0 = 32 * (run.block - page * a.pool.per);
    const size_t head = ((size_t)(a.layer0 + layer) * a.pool.pages + page) * a.pool.nkv + kvh;
    E *kb = (E *)a.pool.k + (head * a.pool.P + slot0) * D, *vb = (E *)a.pool.v + (head * a.pool.P + slot0) * D;
    uint16_t *ks = a.pool.ks + (head * a.pool.P + slot0) * (D / 32), *vs = a.pool.vs + (head * a.pool.P + slot0) * (D / 32);
    const int c = threadIdx.x % TR * 4;
    for (int i = threadIdx.x / TR; i < 2 * run.count; i += 256 / TR) {
        const int r = i >> 1, isv = i & 1, slot = run.slot + r;
        const float *x = (isv ? a.v : a.k) + ((long long)layer * a.n + run.token + r) * a.stride + kvh * D + c;
        float y[4] = {x[0], x[1], x[2], x[3]};
        E e[4];
        if constexpr (FMT == FL_KV_Q8) {
            float amax = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
#pragma unroll
            for (int m = 1; m < 8; m <<= 1) amax = fmaxf(amax, __shfl_xor(amax, m, 64));  // 8 threads: 32 channels
            float d, id;
            pg_q8_scale(amax, d, id);
#pragma unroll
            for (int k = 0; k < 4; k++) e[k] = q8_code(y[k] * id);
            if (c % 32 == 0) (isv ? vs : ks)[slot * (D / 32) + c / 32] = f2h(d);
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if constexpr (FMT == FL_KV_F32) e[k] = y[k];
                else e[k] = f2h(y[k]);
            }
        }
        if (isv) {
#pragma unroll
            for (int k = 0; k < 4; k++) vt[(c + k) * PAD + r] = e[k];
        } else {
            struct alignas(4 * sizeof(E)) E4 {
                E x[4];
            };
            *(E4 *)(kb + slot * D + c) = E4{{e[0], e[1], e[2], e[3]}};
        }
    }
    __syncthreads();
    if (run.count == 32) {
        constexpr int N = 4;  // elements of a piece
        struct alignas(N * sizeof(E)) EN {
            E x[N];
        };
        for (int i = threadIdx.x; i < D * 32 / N; i += 256)
            ((EN *)vb)[i] = *(const EN *)(vt + (i / (32 / N)) * PAD + i % (32 / N) * N);
    } else {
        for (int i = threadIdx.x; i < D * run.count; i += 256) {
            const int d = i / run.count, r = i - d * run.count;
            vb[d * 32 + run.slot + r] = vt[d * PAD + r];
        }
    }
}

// The values of runs of slots, as f32 rows: a workgroup takes one run and kv head; a thread
// has 4 channels of a token's K, then 4 slots of a channel's V, turned in LDS.  grid (runs,
// kv heads)
template <int FMT, int D>
__global__ __launch_bounds__(256) void k_pages_read(PageReadArgs a, PageRuns runs) {
    using E = PgElem<FMT>;
    constexpr int TR = D / 4, PAD = D + 1;
    struct alignas(4 * sizeof(E)) E4 {
        E x[4];
    };
    __shared__ float vt[32 * PAD];
    const PageRun run = pg_run(runs, blockIdx.x);
    const int kvh = blockIdx.y;
    const int page = run.block / a.pool.per, slot0 = 32 * (run.block - page * a.pool.per);
    const size_t head = ((size_t)a.layer * a.pool.pages + page) * a.pool.nkv + kvh;
    const E *kb = (const E *)a.pool.k + (head * a.pool.P + slot0) * D, *vb = (const E *)a.pool.v + (head * a.pool.P + slot0) * D;
    const uint16_t *ks = a.pool.ks + (head * a.pool.P + slot0) * (D / 32), *vs = a.pool.vs + (head * a.pool.P + slot0) * (D / 32);
    const size_t row = (size_t)a.pool.nkv * D;
    auto value = [&](E x, const uint16_t *s, int slot, int d) -> float {
        if constexpr (FMT == FL_KV_F32) return x;
        else if constexpr (FMT == FL_KV_F16) return h2f(x);
        else return (float)x * h2f(s[slot * (D / 32) + (d >> 5)]);
    };
    const int c = threadIdx.x % TR * 4;
    if (a.k)
        for (int r = threadIdx.x / TR; r < run.count; r += 256 / TR) {
            const int slot = run.slot + r;
            const E4 x = *(const E4 *)(kb + slot * D + c);
            float *o = a.k + (size_t)(run.token + r) * row + kvh * D + c;
#pragma unroll
            for (int k = 0; k < 4; k++) o[k] = value(x.x[k], ks, slot, c + k);
        }
    if (!a.v) return;
    for (int i = threadIdx.x; i < D * 8; i += 256) {
        const int d = i >> 3, s = (i & 7) * 4;
        const E4 x = *(const E4 *)(vb + d * 32 + s);
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (s + k >= run.slot && s + k < run.slot + run.count) vt[(s + k - run.slot) * PAD + d] = value(x.x[k], vs, s + k, d);
    }
    __syncthreads();
    for (int r = threadIdx.x / TR; r < run.count; r += 256 / TR) {
        float *o = a.v + (size_t)(run.token + r) * row + kvh * D + c;
#pragma unroll
        for (int k = 0; k < 4; k++) o[k] = vt[r * PAD + c + k];
    }
}

// Blocks of pages to other pages: grid (copies, layers * kv heads); `unit` bytes of
// a 32-slot block of K (and of V), `sunit` of its scales
static __global__ __launch_bounds__(256) void k_pages_copy(PagePool p, PageCopies c, int unit, int sunit) {
    const PageCopy x = c.list ? c.list[blockIdx.x] : c.some[blockIdx.x];
    const int layer = blockIdx.y / p.nkv, kvh = blockIdx.y % p.nkv;
    const size_t per = p.P / kPageBlock;
    const size_t from = (((size_t)layer * p.pages + x.src) * p.nkv + kvh) * per;
    const size_t to = (((size_t)layer * p.pages + x.dst) * p.nkv + kvh) * per;
    const int n = x.blocks * unit / 16, ns = x.blocks * sunit / 16;
    // U pieces of K and of V of a thread in flight together: 63 copies of 96 tokens of 32 layers
    // x 8 x 128, binary16, 186 us one by one, 150 by two, 141 so
    constexpr int U = 8;
    for (int i = threadIdx.x; i < n; i += 256 * U) {
        pu4_t x[2 * U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = min(i + 256 * u, n - 1);
            x[u] = ((const pu4_t *)((const char *)p.k + from * unit))[j];
            x[U + u] = ((const pu4_t *)((const char *)p.v + from * unit))[j];
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (i + 256 * u >= n) break;
            ((pu4_t *)((char *)p.k + to * unit))[i + 256 * u] = x[u];
            ((pu4_t *)((char *)p.v + to * unit))[i + 256 * u] = x[U + u];
        }
    }
    for (int i = threadIdx.x; i < ns; i += 256) {
        ((pu4_t *)((char *)p.ks + to * sunit))[i] = ((const pu4_t *)((const char *)p.ks + from * sunit))[i];
        ((pu4_t *)((char *)p.vs + to * sunit))[i] = ((const pu4_t *)((const char *)p.vs + from * sunit))[i];
    }
}

}  // namespace fl
