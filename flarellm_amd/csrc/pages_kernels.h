// Kernels of the paged KV cache: attention of a batch of queries over the pages of
// their sequences, and the stores, reads and copies of pages.
#pragma once

#include "pages_args.h"

namespace fl {

typedef _Float16 ph8_t __attribute__((ext_vector_type(8)));
typedef float pf4_t __attribute__((ext_vector_type(4)));
typedef uint32_t pu4_t __attribute__((ext_vector_type(4)));
typedef uint32_t pu2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ pf4_t pg_mfma_h(pu4_t a, pu4_t b, pf4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ph8_t, a), __builtin_bit_cast(ph8_t, b), c, 0, 0, 0);
}

// 8 floats as two binary16 parts (round toward zero, then the rest)
__device__ __forceinline__ void pg_split(const float *x, pu4_t &hi, pu4_t &lo) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const auto h = __builtin_amdgcn_cvt_pkrtz(x[2 * i], x[2 * i + 1]);
        const auto l = __builtin_amdgcn_cvt_pkrtz(x[2 * i] - (float)h[0], x[2 * i + 1] - (float)h[1]);
        hi[i] = __builtin_bit_cast(uint32_t, h);
        lo[i] = __builtin_bit_cast(uint32_t, l);
    }
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
    __device__ __forceinline__ void scores(const pu4_t *q, int, pf4_t *s) const {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            pf4_t lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
                lo = pg_mfma_h(k[t][c], q[2 * c + 1], lo);
                hi = pg_mfma_h(k[t][c], q[2 * c], hi);
            }
            s[t] = hi + lo;
        }
    }
    __device__ __forceinline__ void add_pv(const float *p, int, pf4_t *o) const {
        pu4_t hi, lo;
        pg_split(p, hi, lo);
#pragma unroll
        for (int c = 0; c < D / 16; c++) {
            o[c] = pg_mfma_h(v[c], lo, o[c]);
            o[c] = pg_mfma_h(v[c], hi, o[c]);
        }
    }
};

template <int D>
struct PgBlock<FL_KV_Q8, D> {
    static constexpr int QP = D / 32 * 2;
    pu2_t k[2][D / 32], v[D / 16];
    uint16_t ks[8][D / 32], vs[8][D / 32];  // scales of slots 8 g + 0..7

    __device__ __forceinline__ void load_s(const uint16_t *b, uint16_t (*s)[D / 32]) {
        // 8 slots' scales are contiguous
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
            const pu4_t w = ((const pu4_t *)b)[i];
#pragma unroll
            for (int j = 0; j < 8; j++) s[(8 * i + j) / (D / 32)][(8 * i + j) % (D / 32)] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
        }
    }
    __device__ __forceinline__ void load_k(const PagePool &p, size_t head, int slot, int m, int g) {
        const int8_t *b = (const int8_t *)p.k + (head * p.P + slot) * D;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int c = 0; c < D / 32; c++)
                k[t][c] = *(const pu2_t *)(b + (8 * (m >> 2) + 4 * t + (m & 3)) * D + 32 * c + 8 * g);
        load_s(p.ks + (head * p.P + slot + 8 * g) * (D / 32), ks);
    }
    __device__ __forceinline__ void load_v(const PagePool &p, size_t head, int slot, int m, int g) {
        const int8_t *b = (const int8_t *)p.v + (head * p.P + slot) * D;
#pragma unroll
        for (int c = 0; c < D / 16; c++) v[c] = *(const pu2_t *)(b + (16 * c + m) * 32 + 8 * g);
        load_s(p.vs + (head * p.P + slot + 8 * g) * (D / 32), vs);
    }
    // (codes are finite: only the scales of slots without a token must not meet a zero)
    __device__ __forceinline__ void clip_v(int n, int g) {
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int c = 0; c < D / 32; c++) vs[i][c] = 8 * g + i < n ? vs[i][c] : (uint16_t)0;
    }
    static __device__ __forceinline__ void make_q(const float *q, float mul, int g, pu4_t *o) {
        PgBlock<FL_KV_F16, D>::make_q(q, mul, g, o);
    }
    __device__ __forceinline__ void scores(const pu4_t *q, int, pf4_t *s) const {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            s[t] = pf4_t{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
                const pu4_t a = pg_bytes(k[t][c]);
                pf4_t d = pg_mfma_h(a, q[2 * c + 1], pf4_t{0, 0, 0, 0});
                d = pg_mfma_h(a, q[2 * c], d);
#pragma unroll
                for (int i = 0; i < 4; i++) s[t][i] = __builtin_fmaf(d[i], h2f(ks[4 * t + i][c]), s[t][i]);
            }
        }
    }
    __device__ __forceinline__ void add_pv(const float *p, int, pf4_t *o) const {
#pragma unroll
        for (int c = 0; c < D / 32; c++) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = p[j] * h2f(vs[j][c]);
            pu4_t hi, lo;
            pg_split(x, hi, lo);
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const pu4_t a = pg_bytes(v[2 * c + u]);
                o[2 * c + u] = pg_mfma_h(a, lo, o[2 * c + u]);
                o[2 * c + u] = pg_mfma_h(a, hi, o[2 * c + u]);
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
    static __device__ __forceinline__ void make_q(const float *q, float mul, int g, pu4_t *o) {
#pragma unroll
        for (int c = 0; c < D / 16; c++)
#pragma unroll
            for (int j = 0; j < 4; j++) o[c][j] = __float_as_uint(q[16 * c + 4 * g + j] * mul);
    }
    __device__ __forceinline__ void scores(const pu4_t *q, int, pf4_t *s) const {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            s[t] = pf4_t{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < D / 16; c++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][c][j], __uint_as_float(q[c][j]), s[t], 0, 0, 0);
        }
    }
    __device__ __forceinline__ void add_pv(const float *p, int, pf4_t *o) const {
#pragma unroll
        for (int c = 0; c < D / 16; c++)
#pragma unroll
            for (int j = 0; j < 8; j++)
                o[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[c][j >> 2][j & 3], p[j], o[c], 0, 0, 0);
    }
};

// One item (PageItem) and kv head per workgroup of 4 waves; wave w takes the item's
// 32-slot blocks w, w + 4, ..  Each keeps (max, sum, O) of its blocks for NT x 16
// rows (query x head), joined through LDS at the end.  K of a wave's next block is
// loaded when the scores have been formed, V when O has been: half a block ahead.
//
// Values that are not finite: slots behind the item's last token are taken out of V;
// a token that some of the item's queries see and others do not has p = 0 for the
// latter, and 0 * Inf is NaN, as is an Inf against a zero low part.  Every such case
// leaves a NaN or Inf in O: such a row is then formed again, key by key.
template <int FMT, int D, int NT>
__global__ __launch_bounds__(256) void k_pages_attn(PageAttnArgs a) {
    using Block = PgBlock<FMT, D>;
    constexpr int QP = Block::QP, DT = D / 16;
    constexpr float kShift = FMT == FL_KV_F32 ? 0.0f : 15.0f;  // p is kept times 2^15: its parts hold 22 bits
    // [4 waves][16 rows][D + 4]: O, max, sum (of one 16-row tile at a time)
    constexpr int LROW = D + 4;
    __shared__ __align__(16) float lds[4 * 16 * LROW];
    __shared__ int bad_rows;
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nkv = a.pool.nkv, kvh = blockIdx.x % nkv, G = a.group, nh = nkv * G;
    const PageItem it = a.items[blockIdx.x / nkv];
    const int rows = it.nq * G, P = a.pool.P;
    const int nb = (it.slot1 - it.slot0 + 31) >> 5;
    const size_t layer_pages = (size_t)a.layer * a.pool.pages;
    if (threadIdx.x == 0) bad_rows = 0;

    // block b: its (page, kv head), and its first slot in the page
    auto locate = [&](int b, size_t &head, int &slot) {
        const int tok = it.slot0 + 32 * b, first = it.slot0 / P;
        const int page = __builtin_amdgcn_readfirstlane(a.page_ids[it.page0 + tok / P - first]);
        slot = tok % P;
        head = (layer_pages + page) * nkv + kvh;
    };

    Block blk;
    size_t head;
    int slot;
    const int last = max(0, nb - 1);
    locate(min(wave, last), head, slot);
    blk.load_k(a.pool, head, slot, m, g);
    blk.load_v(a.pool, head, slot, m, g);

    pu4_t q[NT][QP];
    float c[NT];
    int seen[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int r = min(16 * n + m, rows - 1), qi = r / G;
        const PageQuery pq = a.order[it.q0 + qi];
        seen[n] = pq.seen;
        const float *qp = a.q + pq.query * a.q_stride + (size_t)(kvh * G + r % G) * D;
        c[n] = a.scale;
        float mul = 1.0f;
        if constexpr (FMT != FL_KV_F32) {
            // the row's largest value is brought to 2^13, so that the low parts stay normal
            float x = 0.0f;
#pragma unroll
            for (int k = 0; k < D / 32; k++)
#pragma unroll
                for (int j = 0; j < 8; j++) x = fmaxf(x, fabsf(qp[32 * k + 8 * g + j]));
            x = pg_max16(x);
            const int e = (int)((__float_as_uint(x) >> 23) & 0xFF);
            if (e > 13 && e < 255) {
                const int s = min(max(140 - e, -100), 100);
                mul = __uint_as_float((uint32_t)(127 + s) << 23);
                c[n] *= __uint_as_float((uint32_t)(127 - s) << 23);
            }
        }
        Block::make_q(qp, mul, g, q[n]);
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

    for (int b = wave; b < nb; b += 4) {
        const int tok = it.slot0 + 32 * b;  // first token of the block
        pf4_t s[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) blk.scores(q[n], g, s[n]);
        size_t head2;
        int slot2;
        locate(min(b + 4, last), head2, slot2);  // past the end: loaded, not used
        blk.load_k(a.pool, head2, slot2, m, g);
        if (tok + 32 > it.smin) {  // some query does not see every token
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (tok + 8 * g + j >= min(seen[n], it.slot1)) s[n][j >> 2][j & 3] = -INFINITY;
            if (tok + 32 > it.slot1) blk.clip_v(it.slot1 - tok, g);
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float x = s[n][0][0];
#pragma unroll
            for (int j = 1; j < 8; j++) x = fmaxf(x, s[n][j >> 2][j & 3]);
            x = pg_max16(x) * c[n];
            if (__any(x > m_run[n])) {
                const float mn = fmaxf(m_run[n], x);
                const float al = m_run[n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run[n] - mn);
                m_run[n] = mn;
                l_run[n] *= al;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[n][d][i] *= al;
            }
            // a row that has seen no token yet keeps p = 0
            const float off = m_run[n] == -INFINITY ? -INFINITY : kShift - m_run[n];
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float y = s[n][j >> 2][j & 3];
                p[j] = y == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(__builtin_fmaf(y, c[n], off));
                l_run[n] += p[j];
            }
            blk.add_pv(p, g, o[n]);
        }
        blk.load_v(a.pool, head2, slot2, m, g);
    }

    // join the waves, one 16-row tile at a time: thread t has row t / 16 and the
    // channels of t % 16
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
        const int r = threadIdx.x >> 4, ch = (threadIdx.x & 15) * (D / 16), row = 16 * n + r;
        float mx = -INFINITY, sum = 0.0f, wt[4];
#pragma unroll
        for (int i = 0; i < 4; i++) mx = fmaxf(mx, lds[(16 * i + r) * LROW + D]);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float mi = lds[(16 * i + r) * LROW + D];
            wt[i] = mi == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mi - mx);
            sum = __builtin_fmaf(lds[(16 * i + r) * LROW + D + 1], wt[i], sum);
        }
        float y[D / 16], odd = sum * 0.0f;
#pragma unroll
        for (int j = 0; j < D / 16; j++) y[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < D / 16; j++) y[j] = __builtin_fmaf(lds[(16 * i + r) * LROW + ch + j], wt[i], y[j]);
        const float il = it.unit < 0 ? 1.0f / sum : 1.0f;
#pragma unroll
        for (int j = 0; j < D / 16; j++) {
            y[j] *= il;
            odd = __builtin_fmaf(y[j], 0.0f, odd);
        }
        if (row < rows) {
            const int qi = row / G, hd = kvh * G + row % G;
            float *op;
            if (it.unit < 0) {
                op = a.out + ((size_t)a.order[it.q0 + qi].query * nh + hd) * D;
            } else {
                op = a.part + ((size_t)(it.unit + qi) * nh + hd) * D;
                if (ch == 0) {
                    float *ml = a.ml + ((size_t)(it.unit + qi) * nh + hd) * 2;
                    ml[0] = mx;
                    ml[1] = sum;
                }
            }
#pragma unroll
            for (int j = 0; j < D / 16; j += 4) *(pf4_t *)(op + ch + j) = pf4_t{y[j], y[j + 1], y[j + 2], y[j + 3]};
            if (odd != 0.0f) bad_rows = 1;  // 0 * Inf and 0 * NaN are NaN
        }
    }
    __syncthreads();
    if (!bad_rows) return;

    // Rows key by key, in the same terms: max of scores in base 2, sum and O times
    // 2^kShift (all rows of the item; this is rare).
    float *sc = lds, *red = lds + 256;
    for (int row = 0; row < rows; row++) {
        const int qi = row / G, hd = kvh * G + row % G;
        const PageQuery pq = a.order[it.q0 + qi];
        const float *qp = a.q + pq.query * a.q_stride + (size_t)hd * D;
        const int end = min(pq.seen, it.slot1);
        float mx = -INFINITY, sum = 0.0f, acc = 0.0f;
        for (int t0 = it.slot0; t0 < end; t0 += 256) {
            const int t = t0 + threadIdx.x;
            float x = -INFINITY;
            if (t < end) {
                const size_t h = (layer_pages + a.page_ids[it.page0 + t / P - it.slot0 / P]) * nkv + kvh;
                x = 0.0f;
                for (int d = 0; d < D; d++) x = __builtin_fmaf(qp[d], pg_k<FMT, D>(a.pool, h, t % P, d), x);
                x *= a.scale;
            }
            __syncthreads();
            sc[threadIdx.x] = x;
            for (int i = 1; i < 64; i <<= 1) x = fmaxf(x, __shfl_xor(x, i, 64));
            if (lane == 0) red[wave] = x;
            __syncthreads();
            const float mn = fmaxf(mx, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
            const float al = mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mx - mn);
            sum *= al;
            acc *= al;
            mx = mn;
            for (int i = 0; i < 256 && t0 + i < end; i++) {
                const float y = sc[i], p = y == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(y - mx + kShift);
                sum += p;
                if (threadIdx.x < D) {
                    const int t2 = t0 + i;
                    const size_t h = (layer_pages + a.page_ids[it.page0 + t2 / P - it.slot0 / P]) * nkv + kvh;
                    acc = __builtin_fmaf(p, pg_v<FMT, D>(a.pool, h, t2 % P, threadIdx.x), acc);
                }
            }
        }
        __syncthreads();
        if (threadIdx.x < D) {
            if (it.unit < 0) {
                a.out[((size_t)pq.query * nh + hd) * D + threadIdx.x] = acc / sum;
            } else {
                const size_t u = (size_t)(it.unit + qi) * nh + hd;
                a.part[u * D + threadIdx.x] = acc;
                if (threadIdx.x == 0) {
                    a.ml[u * 2] = mx;
                    a.ml[u * 2 + 1] = sum;
                }
            }
        }
    }
}

// Partial results of a query joined; 4 channels a thread.  grid (queries, heads * D / 1024 rounded up)
template <int D>
__global__ __launch_bounds__(256) void k_pages_join(PageJoinArgs a) {
    const PageJoin j = a.joins[blockIdx.x];
    const int e = blockIdx.y * 1024 + 4 * threadIdx.x;
    if (e >= a.heads * D) return;
    const int hd = e / D;
    float mx = -INFINITY, l = 0.0f;
    for (int i = 0; i < j.count; i++) mx = fmaxf(mx, a.ml[((size_t)a.units[j.first + i] * a.heads + hd) * 2]);
    pf4_t o = {0, 0, 0, 0};
    for (int i = 0; i < j.count; i++) {
        const size_t u = (size_t)a.units[j.first + i] * a.heads + hd;
        const float mi = a.ml[u * 2], w = mi == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mi - mx);
        l = __builtin_fmaf(a.ml[u * 2 + 1], w, l);
        const pf4_t p = *(const pf4_t *)(a.part + u * D + e % D);
#pragma unroll
        for (int k = 0; k < 4; k++) o[k] = __builtin_fmaf(p[k], w, o[k]);
    }
    const float il = j.count ? 1.0f / l : 0.0f;
#pragma unroll
    for (int k = 0; k < 4; k++) o[k] *= il;
    *(pf4_t *)(a.out + (size_t)j.query * a.heads * D + e) = o;
}

// f32 rows into their slots: a thread takes 32 channels of K or V of one token,
// layer and kv head (as fl_kv_write's Q8 writer, its arithmetic)
template <int FMT, int D>
__global__ __launch_bounds__(256) void k_pages_write(PageWriteArgs a) {
    constexpr int NB = D / 32;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long total = (long long)a.layers * a.n * a.pool.nkv * NB * 2;
    if (i >= total) return;
    const int isv = (int)(i & 1), b = (int)(i >> 1) % NB;
    long long j = (i >> 1) / NB;
    const int kvh = (int)(j % a.pool.nkv);
    j /= a.pool.nkv;
    const int t = (int)(j % a.n), l = (int)(j / a.n);
    const int at = a.slots[t], page = at / a.pool.P, slot = at % a.pool.P;
    const float *x = (isv ? a.v : a.k) + ((long long)l * a.n + t) * a.stride + kvh * D + 32 * b;
    const size_t head = ((size_t)(a.layer0 + l) * a.pool.pages + page) * a.pool.nkv + kvh;
    const size_t base = isv ? head * a.pool.P * D + ((size_t)(slot >> 5) * D + 32 * b) * 32 + (slot & 31)
                            : (head * a.pool.P + slot) * D + 32 * b;
    const int step = isv ? 32 : 1;
    void *o = isv ? a.pool.v : a.pool.k;
    if constexpr (FMT == FL_KV_Q8) {
        float amax = 0.0f;
        for (int e = 0; e < 32; e++) amax = fmaxf(amax, fabsf(x[e]));
        const float d = amax / 127.0f;
        const float id = (d != 0.0f) ? 127.0f / amax : 0.0f;
        for (int e = 0; e < 32; e++) ((int8_t *)o)[base + (size_t)e * step] = q8_code(x[e] * id);
        (isv ? a.pool.vs : a.pool.ks)[(head * a.pool.P + slot) * NB + b] = f2h(d);
    } else {
        for (int e = 0; e < 32; e++) {
            if constexpr (FMT == FL_KV_F32) ((float *)o)[base + (size_t)e * step] = x[e];
            else ((uint16_t *)o)[base + (size_t)e * step] = f2h(x[e]);
        }
    }
}

// The values of slots, as f32 rows: a thread per (token, kv head, channel)
template <int FMT, int D>
__global__ __launch_bounds__(256) void k_pages_read(PageReadArgs a) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)a.n * a.pool.nkv * D) return;
    const int d = (int)(i % D), kvh = (int)(i / D % a.pool.nkv), t = (int)(i / D / a.pool.nkv);
    const int at = a.slots[t], page = at / a.pool.P, slot = at % a.pool.P;
    const size_t head = ((size_t)a.layer * a.pool.pages + page) * a.pool.nkv + kvh;
    if (a.k) a.k[i] = pg_k<FMT, D>(a.pool, head, slot, d);
    if (a.v) a.v[i] = pg_v<FMT, D>(a.pool, head, slot, d);
}

// Blocks of pages to other pages: grid (copies, layers * kv heads); `unit` bytes of
// a 32-slot block of K (and of V), `sunit` of its scales
static __global__ __launch_bounds__(256) void k_pages_copy(PagePool p, const PageCopy *c, int unit, int sunit) {
    const PageCopy x = c[blockIdx.x];
    const int layer = blockIdx.y / p.nkv, kvh = blockIdx.y % p.nkv;
    const size_t per = p.P / kPageBlock;
    const size_t from = (((size_t)layer * p.pages + x.src) * p.nkv + kvh) * per;
    const size_t to = (((size_t)layer * p.pages + x.dst) * p.nkv + kvh) * per;
    const int n = x.blocks * unit / 16, ns = x.blocks * sunit / 16;
    for (int i = threadIdx.x; i < n; i += 256) {
        const pu4_t k = ((const pu4_t *)((const char *)p.k + from * unit))[i];
        const pu4_t v = ((const pu4_t *)((const char *)p.v + from * unit))[i];
        ((pu4_t *)((char *)p.k + to * unit))[i] = k;
        ((pu4_t *)((char *)p.v + to * unit))[i] = v;
    }
    for (int i = threadIdx.x; i < ns; i += 256) {
        ((pu4_t *)((char *)p.ks + to * sunit))[i] = ((const pu4_t *)((const char *)p.ks + from * sunit))[i];
        ((pu4_t *)((char *)p.vs + to * sunit))[i] = ((const pu4_t *)((const char *)p.vs + from * sunit))[i];
    }
}

}  // namespace fl
