// Attention over the paged KV cache: amv_paged_attn (a ragged batch over its pages), amv_paged_attn_shared (sequences behind one
// prefix) and amv_paged_attn_sparse (selected pages).
//
//   out[t][h] = sum_j w_j v_j / sum_j w_j,  w_j = 2^(s_j - m),  s_j = scale log2(e) q[t][h] . k_j,  m a running reference
//
// The query rows of a sequence and a KV head, its tokens times the group's heads, are tiles of 16 rows; a wave takes RT tiles over
// 32 keys at a time, straight from memory to registers, no LDS and no barrier on the way:
//   S^T (keys x rows) = K Q^T with v_mfma_f32_16x16x32_f16, two products of 16 keys: lane (c = l % 16, g = l / 16) reads elements
//     32 s + 8 g .. + 7 of key 8 (c / 4) + 4 u + c % 4 for product u. In the results the lane then holds keys 8 g .. 8 g + 7 of row c,
//     which is just what the second product wants of it:
//   O^T (elements x rows) += V^T P^T: the lane's k slots are its own keys 8 g + 0 .. 7. It reads the elements (D / 16) c + t, one for
//     each of the D / 16 products t, of those 8 keys (16 lanes a whole row), and v_perm_b32 pairs the keys: one instruction for two
//     operand elements is all the transposing there is.
// q and the weights are f32; f16 alone would cost them 2^-11. Each enters its product as two f16, the value rounded and the rest
// (22 bits together): twice the matrix work, at less than a fifth of their rate where keys come from memory. q is scaled by a power
// of two to below 2 first (from 2^103 on by 2^-102, so that q times scale log2(e) leaves f16's range at 2^118); the weights' reference is
// kept 12 to 15 below the running maximum, so that the rest keeps its bits beside a dominating key.
// Quantized caches: the integers are exact in f16. Block b of a key is one product of K's (its own accumulator, then times the
// block's scale in f32), and two of V's products, whose weights are multiplied by the value's scale before they are split. The
// scales are brought to at most 1 by a power of two that follows the largest met (as the maximum does), which keeps weight times
// scale in f16's range whatever the values' size.
//
// Four waves of a workgroup take the 32-key tiles of a range in turn and join in LDS; ranges of a long sequence go to several
// workgroups, joined by k_paged_merge from (m, l, O) in the workspace. Tiles of many rows share K and V through LDS (pg_many).
//
// Measured (32 query and 8 KV heads of 128), and what bounds it:
//   64 sequences of up to 4096 f16 keys, 684 MB: 123 us, 5.5 TB/s (equally long ones 6.6, where a copy of 4 GiB reaches 5.0): memory
//   3 of up to 65536 Q8_0 keys, 331 MB: 66 us and 5 the merge, 4.7 TB/s (96 equal ones 6.0): memory, VALU a third of the SIMD cycles
//   96 of 4096 Q4_0 keys: 104 us, 4.4 TB/s: VALU, as much work a key as Q8_0's for half the bytes
//   one of 777 f16 keys: 7.7 us and 2.4 the merge: two launches, a tile's latency and the join
//   2 x 1024 tokens, up to 3000 f16 keys: 138 us, 0.76 PFLOP/s of products, which are twice the formula's (8192 tokens 1.1, a library's
//     product 1.17): matrix cores 30 %, VALU 35 % of the SIMD cycles at two waves a SIMD; over Q8_0 keys 232 us, Q4_0 231: half as many
//     products again and the bringing of integers to LDS
//   128 tokens behind 16384 shared f16 keys: 107 us and 7 the merge: the same, and the first steps of 384 workgroups
//   32 sequences of up to 8 tokens after up to 4096 keys (17 to 32 rows a KV head): f16 84 us, 70 of them the bytes; Q8_0 142, half of the
//     waves of tiles of 64 rows having no rows; Q4_0 121, VALU (29 %) and the way of 64 spilled registers
#include "amv_paged.h"

#include <algorithm>
#include <type_traits>

typedef _Float16 pg_h8 __attribute__((ext_vector_type(8)));
typedef float pg_f4 __attribute__((ext_vector_type(4)));

struct PgAttn {
    PgBatch b;
    const uint8_t *k, *v;
    const float* q;
    float* out;
    float2* ml;        // (reference, sum) of each part of a row's keys, [row][n_split]; NULL: the output is written instead
    float* acc;        // its weighted values [row][n_split][D]
    const int32_t* list;  // selected pages [n_tok][n_head_kv][n_list], or the prefix's pages
    int64_t q_stride, page_stride;
    float scale2;      // scale * log2(e)
    int n_pages, n_head, n_head_kv, G;
    int kind;          // PG_ONE, PG_FIND, PG_PREFIX, PG_LIST
    int ta;            // row tiles of a sequence (PG_ONE) or a token (PG_LIST)
    int rows_most;     // PG_ONE: sequences of at most, PG_FIND: of more than so many rows
    int n_list;        // selected pages, or the prefix's keys
    int tiles, n_split, split_len;  // row tiles (of one KV head), parts of their keys and the parts' length
};
enum { PG_ONE, PG_FIND, PG_PREFIX, PG_LIST };

__device__ __forceinline__ uint32_t pg_bits(amv_h2 x) { return __builtin_bit_cast(uint32_t, x); }

template <int N>
__device__ __forceinline__ void pg_load(uint32_t* to, const uint8_t* from) {  // N bytes, aligned to min(N, 16)
    if constexpr (N >= 16) {
#pragma unroll
        for (int i = 0; i < N / 16; ++i) {
            const amv_v4u x = *reinterpret_cast<const amv_v4u*>(from + 16 * i);
            to[4 * i] = x.x;
            to[4 * i + 1] = x.y;
            to[4 * i + 2] = x.z;
            to[4 * i + 3] = x.w;
        }
    } else if constexpr (N == 8) {
        const uint2 x = *reinterpret_cast<const uint2*>(from);
        to[0] = x.x;
        to[1] = x.y;
    } else if constexpr (N == 4) {
        to[0] = *reinterpret_cast<const uint32_t*>(from);
    } else {
        to[0] = *reinterpret_cast<const uint16_t*>(from);
    }
}

// N bytes that no other instruction reads a part of the lines of: past the caches (64 sequences of 4096 f16 keys: 180 us, with the
// values read so 162)
template <int N>
__device__ __forceinline__ void pg_load_once(uint32_t* to, const uint8_t* from) {
    if constexpr (N == 16) {
        const amv_v4u x = __builtin_nontemporal_load(reinterpret_cast<const amv_v4u*>(from));
        to[0] = x.x;
        to[1] = x.y;
        to[2] = x.z;
        to[3] = x.w;
    } else {
        typedef uint32_t v2u __attribute__((ext_vector_type(2)));
        const v2u x = __builtin_nontemporal_load(reinterpret_cast<const v2u*>(from));
        to[0] = x.x;
        to[1] = x.y;
    }
}

// 32 keys of a wave, as they come from memory. KPL: scores a lane holds, of its keys 8 g + 4 u .. (u 0 where KPL is 8)
template <int TYPE, int D, int KPL>
struct PgK {
    static constexpr int NB = D / 32, W = TYPE == AMV_T_F16 ? 4 * NB : TYPE == AMV_T_Q8_0 ? 2 * NB : NB;
    uint32_t k[2][W];                                  // product u's key, the lane's elements
    uint32_t s[TYPE == AMV_T_F16 ? 1 : KPL * NB / 2];  // scales f16 [key][NB] of the lane's scores
};
template <int TYPE, int D, int KPL>
struct PgV {
    static constexpr int NB = D / 32, BYTES = TYPE == AMV_T_F16 ? D / 8 : TYPE == AMV_T_Q8_0 ? D / 16 : D / 32;
    static constexpr int W = BYTES < 4 ? 1 : BYTES / 4;
    uint32_t v[8][W];                                  // key 8 g + j, the lane's D / 16 elements
    uint32_t s[TYPE == AMV_T_F16 ? 1 : KPL * NB / 2];
};
// where a wave's 32 keys are, the same in every lane: their halves' places, bytes of their rows in the pool; e: the physical pages, -1
// for no keys
struct PgAt {
    int e0, e1, p0, p1;
};
// a lane's parts of the addresses
struct PgLane {
    int k, v, s;   // of its K row and elements, its first V row and elements, its first scales
    bool k1, v1;   // whether they are in the second half
};

template <int TYPE, int D>
__device__ __forceinline__ int64_t pg_off(const PgAttn& a, int e, int p, bool scales) {  // uniform
    using R = PgRow<TYPE, D>;
    const int row = p & ((1 << a.b.pshift) - 1);
    return (int64_t)max(e, 0) * a.page_stride + (scales ? (int64_t)(R::ROW << a.b.pshift) + row * R::SC : (int64_t)row * R::ROW);
}
template <int TYPE, int D, int KPL>
__device__ __forceinline__ void pg_load_k(PgK<TYPE, D, KPL>& t, const PgAttn& a, const uint8_t* kc, const PgAt& at, const PgLane& ln) {
    using R = PgRow<TYPE, D>;
    const int64_t o0 = pg_off<TYPE, D>(a, at.e0, at.p0, false), o1 = pg_off<TYPE, D>(a, at.e1, at.p1, false);
    const uint8_t* p = kc + (ln.k1 ? o1 : o0) + ln.k;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        if constexpr (TYPE == AMV_T_F16) {
#pragma unroll
            for (int s = 0; s < R::NB; ++s) pg_load<16>(&t.k[u][4 * s], p + 4 * u * R::ROW + 64 * s);
        } else {
            pg_load<R::ROW / 4>(t.k[u], p + 4 * u * R::ROW);
        }
    }
    if constexpr (TYPE != AMV_T_F16) {
        const int64_t s0 = pg_off<TYPE, D>(a, at.e0, at.p0, true), s1 = pg_off<TYPE, D>(a, at.e1, at.p1, true);
        pg_load<KPL * R::SC>(t.s, kc + (ln.v1 ? s1 : s0) + ln.s);
    }
}
template <int TYPE, int D, int KPL>
__device__ __forceinline__ void pg_load_v(PgV<TYPE, D, KPL>& t, const PgAttn& a, const uint8_t* vc, const PgAt& at, const PgLane& ln) {
    using R = PgRow<TYPE, D>;
    const int64_t o0 = pg_off<TYPE, D>(a, at.e0, at.p0, false), o1 = pg_off<TYPE, D>(a, at.e1, at.p1, false);
    const uint8_t* p = vc + (ln.v1 ? o1 : o0) + ln.v;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if constexpr (R::ROW >= 128) pg_load_once<PgV<TYPE, D, KPL>::BYTES>(t.v[j], p + j * R::ROW);
        else pg_load<PgV<TYPE, D, KPL>::BYTES>(t.v[j], p + j * R::ROW);
    }
    if constexpr (TYPE != AMV_T_F16) {
        const int64_t s0 = pg_off<TYPE, D>(a, at.e0, at.p0, true), s1 = pg_off<TYPE, D>(a, at.e1, at.p1, true);
        pg_load<KPL * R::SC>(t.s, vc + (ln.v1 ? s1 : s0) + ln.s);
    }
}

// Integers u = value + bias in the low bits of a word's two halves are, as they stand, the f16 u 2^-24. Values become operands times
// 2^-10: u 2^-24 2^14 - bias 2^-10 is exact.
template <int TYPE>
__device__ __forceinline__ uint32_t pg_f16_of(uint32_t u) {
    constexpr float bias = (TYPE == AMV_T_Q8_0 ? 128.0f : 8.0f) / 1024.0f;
    const amv_h2 m = {(_Float16)16384.0f, (_Float16)16384.0f}, b = {(_Float16)-bias, (_Float16)-bias};
    return pg_bits(__builtin_elementwise_fma(__builtin_bit_cast(amv_h2, u), m, b));
}
// The operand of product s of K: 8 f16; of quantized keys (value + bias) 2^-24 (Q4_0: times 16), whose product begins at -128 2^-24
// times the sum of q's elements, so that no instruction is spent on the bias (96 sequences of 4096 Q4_0 keys 105 us, so 100). The matrix
// cores align such f16 by their exponent, which is the least for all of them: with Q4_0's integers in the lowest 4 of the 10 bits the
// sums lost 6 bits (an error of 4.6e-6 for 24 selected pages), in bits 4 to 7, as with Q8_0's 8 bits, they lose 2.
template <int TYPE, int D>
__device__ __forceinline__ pg_h8 pg_k_operand(const uint32_t* k, int s) {
    amv_v4u x;
    if constexpr (TYPE == AMV_T_F16) {
        x = amv_v4u{k[4 * s], k[4 * s + 1], k[4 * s + 2], k[4 * s + 3]};
    } else if constexpr (TYPE == AMV_T_Q8_0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t w = k[2 * s + h] ^ 0x80808080u;
            x[2 * h] = __builtin_amdgcn_perm(0u, w, 0x0C010C00u);
            x[2 * h + 1] = __builtin_amdgcn_perm(0u, w, 0x0C030C02u);
        }
    } else {
        const uint32_t even = (k[s] << 4) & 0xF0F0F0F0u, odd = k[s] & 0xF0F0F0F0u;
        x[0] = __builtin_amdgcn_perm(odd, even, 0x0C040C00u);
        x[1] = __builtin_amdgcn_perm(odd, even, 0x0C050C01u);
        x[2] = __builtin_amdgcn_perm(odd, even, 0x0C060C02u);
        x[3] = __builtin_amdgcn_perm(odd, even, 0x0C070C03u);
    }
    return __builtin_bit_cast(pg_h8, x);
}
// the operand of product t of V: element t of keys 0 .. 7
template <int TYPE, int D, int KPL>
__device__ __forceinline__ pg_h8 pg_v_operand(const PgV<TYPE, D, KPL>& v, int t) {
    amv_v4u x;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        if constexpr (TYPE == AMV_T_F16) {
            x[p] = __builtin_amdgcn_perm(v.v[2 * p + 1][t >> 1], v.v[2 * p][t >> 1], (t & 1) ? 0x07060302u : 0x05040100u);
        } else {
            uint32_t lo, hi;
            int b;
            if constexpr (TYPE == AMV_T_Q8_0) {
                lo = v.v[2 * p][t >> 2] ^ 0x80808080u;
                hi = v.v[2 * p + 1][t >> 2] ^ 0x80808080u;
                b = t & 3;
            } else {
                lo = (v.v[2 * p][t >> 3] >> ((t & 1) * 4)) & 0x0F0F0F0Fu;
                hi = (v.v[2 * p + 1][t >> 3] >> ((t & 1) * 4)) & 0x0F0F0F0Fu;
                b = (t >> 1) & 3;
            }
            x[p] = pg_f16_of<TYPE>(__builtin_amdgcn_perm(hi, lo, 0x0C040C00u + 0x00010001u * b));
        }
    }
    return __builtin_bit_cast(pg_h8, x);
}
// 1 in the halves of a word that are infinite or no number
__device__ __forceinline__ uint32_t pg_strange(uint32_t w) { return (((w & 0x7C007C00u) + 0x04000400u) >> 15) & 0x00010001u; }
// Values that are infinite or no number, where a tile's rows see different keys: a row that does not see such a value has the weight 0
// for it, and the product would make no number of it. Such keys (bits j: the lane's keys 8 g + j) leave the products, and a row that sees
// one gets a sum that is no number.
__device__ __forceinline__ uint32_t pg_row16_or(uint32_t x) {
    x |= (uint32_t)amv_dpp_i<0xB1>((int)x);
    x |= (uint32_t)amv_dpp_i<0x4E>((int)x);
    x |= (uint32_t)amv_dpp_i<0x141>((int)x);
    return x | (uint32_t)amv_dpp_i<0x140>((int)x);
}
// 8 values as f16 and the rest as f16
__device__ __forceinline__ void pg_split(const float (&x)[8], pg_h8& hi, pg_h8& lo) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        hi[j] = (_Float16)x[j];
        lo[j] = (_Float16)fmaf((float)hi[j], -1.0f, x[j]);
    }
}
// the f16 of a value (part 0) or the rest (part 1)
__device__ __forceinline__ _Float16 pg_part(float x, float part) { return (_Float16)fmaf((float)(_Float16)x, -part, x); }
template <int C>
__device__ __forceinline__ float pg_dpp(float x) { return __int_as_float(amv_dpp_i<C>(__float_as_int(x))); }
#define PG_ROR8 0x128        // lane c of a row of 16 and c ^ 8
#define PG_HALF_MIRROR 0x141 // c and 7 - c (of its 8)
#define PG_MIRROR 0x140      // c and 15 - c
__device__ __forceinline__ pg_f4 pg_mfma(pg_h8 a, pg_h8 b, pg_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float pg_half(const uint32_t* s, int i) { return amv_h2f(s[i >> 1] >> (16 * (i & 1))); }

// A tile's rows: rows r0 .. r_last of the n_rows of tokens tok0 .., row r is head r % G of token tok0 + r / G, whose place is place0 +
// r / G; keys: how many there are to see, see_all: that each of the rows sees, see_any: that any does
struct PgRows {
    int tok0, r0, r_last, n_rows, place0, keys, see_all, see_any;
    const int32_t* pages;  // the physical pages, or the sequence's table where `list` says which
    const int32_t* list;
    int64_t part0;         // PG_ONE: where the rows of the sequence are in ml; else -1
    __device__ void see(const PgAttn& a, int from, int to) {
        r0 = from;
        r_last = to;
        see_all = see_any = keys;
        if (a.kind != PG_PREFIX) {
            see_all = min(keys, place0 + r0 / a.G + 1);
            see_any = min(keys, place0 + r_last / a.G + 1);
        }
    }
};
// the rows of tile `tile` of `rows` rows; false where there are none (the same for the whole workgroup)
__device__ __forceinline__ bool pg_rows(const PgAttn& a, int hk, int tile, int rows, PgRows& t) {
    t.list = nullptr;
    t.part0 = -1;
    int in = tile;
    if (a.kind == PG_PREFIX) {
        t.tok0 = 0;
        t.n_rows = a.b.last(a.b.n_seq - 1) * a.G;  // (not the rows behind the last sequence, whatever is in them)
        t.keys = t.place0 = a.n_list;
        t.pages = a.list;
    } else {
        int s;
        if (a.kind == PG_LIST) {
            t.tok0 = tile / a.ta;
            in = tile % a.ta;
            s = pg_seq_of(a.b, t.tok0);
        } else if (a.kind == PG_ONE) {
            s = tile / a.ta;
            in = tile % a.ta;
        } else {
            pg_find(a.b.n_seq, tile, [&](int q) {
                const int r = (a.b.last(q) - a.b.first(q)) * a.G;
                return r > a.rows_most ? (r + rows - 1) / rows : 0;
            }, s, in);
        }
        if (s >= a.b.n_seq) return false;
        const int first = a.b.first(s), n_q = a.b.last(s) - first;
        t.place0 = a.b.end(s) - n_q;
        t.keys = a.b.keys(s);
        t.pages = a.b.table + s * a.b.table_stride;
        if (a.kind == PG_LIST) {
            t.place0 += t.tok0 - first;
            t.n_rows = a.G;
            t.list = a.list + ((int64_t)t.tok0 * a.n_head_kv + hk) * a.n_list;
        } else {
            t.tok0 = first;
            t.n_rows = n_q * a.G;
            if (a.kind == PG_ONE && t.n_rows > a.rows_most) return false;
            if (a.kind == PG_ONE) t.part0 = ((int64_t)s * a.n_head_kv + hk) * a.rows_most;
            if (a.kind == PG_FIND) in = (t.n_rows + rows - 1) / rows - 1 - in;  // the rows with the most keys first
        }
    }
    if (in * rows >= t.n_rows) return false;
    t.see(a, in * rows, min(in * rows + rows, t.n_rows) - 1);
    return true;
}
// where keys 32 i .. 32 i + 31 are (i: uniform over the wave)
__device__ __forceinline__ PgAt pg_where(const PgAttn& a, const int32_t* pages, int keys, int i) {
    PgAt at;
    at.p0 = i * 32;
    at.p1 = at.p0 + 16;
    at.e0 = pages[at.p0 >> a.b.pshift];
    at.e1 = at.p1 < keys ? pages[at.p1 >> a.b.pshift] : -1;
    if ((uint32_t)at.e0 >= (uint32_t)a.n_pages) at.e0 = -1;
    if ((uint32_t)at.e1 >= (uint32_t)a.n_pages) at.e1 = -1;
    return at;
}
// elements 32 s + 8 g .. of row r of a tile, times scale log2(e) 2^-e below 2; returns 2^e
template <int D>
__device__ __forceinline__ float pg_query(const PgAttn& a, const PgRows& t, int hk, int r, int g, float (&x)[D / 32][8]) {
    const int tr = r / a.G;
    const float* src = a.q + (t.tok0 + tr) * a.q_stride + (int64_t)(hk * a.G + r - tr * a.G) * D + 8 * g;
    float am = 0.0f;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
        const float4 y = *reinterpret_cast<const float4*>(src + 32 * s), z = *reinterpret_cast<const float4*>(src + 32 * s + 4);
        const float yz[8] = {y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[s][j] = yz[j] * a.scale2;
            am = fmaxf(am, fabsf(x[s][j]));
        }
    }
    am = amv_max_x32(amv_max_x16(am));
    const uint32_t e = max(1u, min(229u, __float_as_uint(am) >> 23));  // (2^e 2^24 is a number)
    const float down = __uint_as_float((254u - e) << 23);
#pragma unroll
    for (int s = 0; s < D / 32; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[s][j] *= down;
    return __uint_as_float(e << 23);
}
// the weights w of a row's scores s, whose units are f; m the running reference, l and o the sums so far
template <int P, int N, int T>
__device__ __forceinline__ void pg_soften(const float (&s)[N], float f, float& m, float& l, pg_f4 (&o)[T], float (&w)[N]) {
    float mx = s[0];
#pragma unroll
    for (int j = 1; j < N; ++j) mx = fmaxf(mx, s[j]);
    if constexpr (P == 4) mx = fmaxf(mx, pg_dpp<PG_ROR8>(mx));
    mx = amv_max_x32(amv_max_x16(mx)) * f;  // (f a power of two: exact)
    // the reference moves when a weight would pass 2^15 (or there is none yet), to 2^-12 of the maximum; where no difference of 12 is
    // exact, to the maximum
    const bool grow = mx > m + 15.0f;
    if (__builtin_amdgcn_ballot_w64(grow)) {
        const float to = fabsf(mx) > 0x1p20f ? mx : mx - 12.0f;
        const float alpha = grow ? __builtin_amdgcn_exp2f(m - to) : 1.0f;
        if (grow) m = to;
        l *= alpha;
#pragma unroll
        for (int t = 0; t < T; ++t) o[t] *= alpha;
    }
    const float ref = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        w[j] = __builtin_amdgcn_exp2f(fmaf(s[j], f, -ref));
        sum += w[j];
    }
    l += sum;
}
// where a row's result goes: the output, or (*ml not NULL) its part z
template <int D>
__device__ __forceinline__ float* pg_to(const PgAttn& a, const PgRows& t, int hk, int r, int z, float2** ml) {
    const int tr = r / a.G;
    const int64_t row = (int64_t)(t.tok0 + tr) * a.n_head + hk * a.G + (r - tr * a.G);
    const int64_t part = (t.part0 >= 0 ? t.part0 + r : row) * a.n_split + z;
    *ml = a.ml ? a.ml + part : nullptr;
    return a.ml ? a.acc + part * D : a.out + row * D;
}

// The waves of the workgroup take the tile's keys in turn, each for all its rows: rows 16 RT / P sub .. of tile `tile` of `rows`
template <int TYPE, int D, int RT, int P>
__device__ __forceinline__ void pg_few(const PgAttn& a, int hk, int tile, int rows, int sub, int z, float* so0, float* so1) {
    using R = PgRow<TYPE, D>;
    constexpr int NB = D / 32, T = D / 16, ROWS = 16 / P, KPL = P == 4 ? 4 : 8;
    constexpr bool QUANT = TYPE != AMV_T_F16;
    static_assert(P == 1 || RT == 1, "rows that share a product's columns are one tile");
    // a row tile's O^T of waves 0 and 1, 2 and 3: [wave][register][product][lane]
    const auto so = [&](int w, int r, int v) -> float& { return (w < 2 ? so0 : so1)[(((w & 1) * 4 + r) * T + v) * 64 + (threadIdx.x & 63)]; };
    __shared__ float sm[4][16 * RT], sl[4][16 * RT];
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    // what column c of the products is: row `col` of its tile, rounded (part 0) or the rest (part 1); u: whose keys it keeps
    const int u = P == 4 ? c >> 3 : 0;
    const bool rest = P == 4 ? (c & 4) != 0 : P == 2 && c >= 8;
    const int col = P == 4 ? (rest ? 3 - (c & 3) : c & 3) : P == 2 ? (rest ? 15 - c : c) : c;
    const float part = rest ? 1.0f : 0.0f;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int psh = a.b.pshift, ps = 1 << psh;
    PgRows t;
    if (!pg_rows(a, hk, tile, rows, t)) return;
    if (rows > ROWS * RT) {
        const int r0 = t.r0 + ROWS * RT * sub;
        if (r0 > t.r_last) return;
        t.see(a, r0, min(r0 + ROWS * RT - 1, t.r_last));
    }

    // the walk: 32-key tiles i = begin + w, begin + w + 4, ... of the keys (of the listed pages' keys)
    int walk = t.see_any;
    if (t.list) {
        walk = 0;
        for (int i = lane; i < (a.n_list + 63) / 64 * 64; i += 64) {
            const uint64_t m = __builtin_amdgcn_ballot_w64(i < a.n_list && t.list[min(i, a.n_list - 1)] >= 0);
            if (m) walk = ((i - lane) + 64 - __builtin_clzll(m)) << psh;
        }
        walk = __builtin_amdgcn_readfirstlane(walk);
    }
    const int end = (min(walk, (z + 1) * a.split_len) + 31) >> 5;
    int i = (z * a.split_len >> 5) + w;

    const auto where = [&](int i) {
        if (!t.list) return pg_where(a, t.pages, t.keys, i);
        PgAt at;
        const int j0 = i * 32 >> psh, j1 = min(i * 32 + 16, walk - 1) >> psh, off = (i * 32) & (ps - 1);
        const int l0 = t.list[j0], l1 = t.list[j1], most = (a.b.max_kv - 1) >> psh;
        at.e0 = l0 >= 0 && l0 <= most ? t.pages[l0] : -1;
        at.e1 = i * 32 + 16 < walk && l1 >= 0 && l1 <= most ? t.pages[l1] : -1;
        at.p0 = (l0 << psh) + off;
        at.p1 = psh == 4 ? l1 << psh : at.p0 + 16;
        if ((uint32_t)at.e0 >= (uint32_t)a.n_pages) at.e0 = -1;
        if ((uint32_t)at.e1 >= (uint32_t)a.n_pages) at.e1 = -1;
        return at;
    };

    const size_t chunk = (size_t)ps * (R::ROW + R::SC);
    const uint8_t *kc = a.k + hk * chunk, *vc = a.v + hk * chunk;
    PgK<TYPE, D, KPL> tk;
    PgV<TYPE, D, KPL> tv;
    const PgLane ln = {(8 * ((c >> 2) & 1) + (c & 3)) * R::ROW + (QUANT ? g * (R::ROW / 4) : 16 * g),
                       8 * (g & 1) * R::ROW + PgV<TYPE, D, KPL>::BYTES * c, (8 * (g & 1) + 4 * u) * R::SC, c >= 8, g >= 2};
    PgAt at = {-1, -1, 0, 0};
    if (i < end) {
        at = where(i);
        pg_load_k(tk, a, kc, at, ln);
        pg_load_v(tv, a, vc, at, ln);
    }

    // Q^T operands: values times scale log2(e) 2^-e below 2, P = 1: as f16 and the rest in two operands, P = 2: in the two halves of
    // the columns of one, P = 4 and quantized keys: of two, one for each product u, that is 0 where the columns keep the other's keys,
    // so that the products add up to what each column keeps (f16 keys may be infinite or no number where nobody sees them: 0 times
    // them would not be 0, so there each column picks its product). f: 2^e (for quantized keys times what their operands
    // lack); lim: keys the row sees; q0: where the products of quantized keys begin
    pg_h8 qa[RT][P == 2 || (P == 4 && !QUANT) ? 1 : 2][NB];
    float f[RT], q0[RT][QUANT ? NB : 1];
    int lim[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = min(t.r0 + 16 * rt + col, t.r_last);
        lim[rt] = a.kind == PG_PREFIX ? t.keys : min(t.keys, t.place0 + r / a.G + 1);
        float x[NB][8];
        f[rt] = pg_query<D>(a, t, hk, r, g, x);
#pragma unroll
        for (int s = 0; s < NB; ++s) {
            if constexpr (P == 1) {
                pg_split(x[s], qa[rt][0][s], qa[rt][1][s]);
            } else {
                pg_h8 h;
#pragma unroll
                for (int j = 0; j < 8; ++j) h[j] = pg_part(x[s][j], part);
                if constexpr (P == 2 || !QUANT) {
                    qa[rt][0][s] = h;
                } else {
                    const amv_v4u hw = __builtin_bit_cast(amv_v4u, h);
                    const uint32_t k0 = u ? 0u : 0xFFFFFFFFu;
                    qa[rt][0][s] = __builtin_bit_cast(pg_h8, hw & k0);
                    qa[rt][1][s] = __builtin_bit_cast(pg_h8, hw & ~k0);
                }
            }
            if constexpr (QUANT) {
                float sum = 0.0f;  // of what the products multiply: the two parts, or the column's
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    sum += P == 2 ? (float)qa[rt][0][s][j] : (float)qa[rt][0][s][j] + (float)qa[rt][1][s][j];
                q0[rt][s] = amv_sum_x32(amv_sum_x16(sum)) * (-128.0f * 0x1p-24f);
            }
        }
        if constexpr (QUANT) f[rt] *= TYPE == AMV_T_Q8_0 ? 0x1p24f : 0x1p20f;
    }

    float m[RT], l[RT];
    pg_f4 o[RT][T];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY;
        l[rt] = 0.0f;
#pragma unroll
        for (int v = 0; v < T; ++v) o[rt][v] = pg_f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    float vref = 0.0f, vdown = 0.0f;  // the power of two that values' scales are held below, its inverse

    // one tile, with the wave's next one on its way into the registers as they fall free (`more`: there is one. The last tile has
    // its own copy of this code: to load it again instead cost a tenth of the time of a wave of 8 tiles)
    const auto step = [&](auto more) {
        const PgAt now = at;
        if constexpr (more()) at = where(i + 4);
        // scores of the lane's keys 8 g + 4 u + j
        float s[RT][KPL];
        if constexpr (QUANT) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int j = 0; j < KPL; ++j) s[rt][j] = 0.0f;
        }
        constexpr int X = P == 4 && QUANT ? 1 : 2;
        pg_f4 x[RT][X];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (QUANT || b == 0) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int h = 0; h < X; ++h) {
                        const float y = QUANT ? q0[rt][QUANT ? b : 0] : 0.0f;
                        x[rt][h] = pg_f4{y, y, y, y};
                    }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const pg_h8 kf = pg_k_operand<TYPE, D>(tk.k[h], b);
                if constexpr (P == 4 && QUANT) {
                    x[0][0] = pg_mfma(kf, qa[0][h][b], x[0][0]);
                } else {
#pragma unroll
                    for (int k = P == 1 ? 1 : 0; k >= 0; --k)
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) x[rt][h] = pg_mfma(kf, qa[rt][k][b], x[rt][h]);
                }
            }
            if constexpr (QUANT) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int j = 0; j < KPL; ++j) s[rt][j] = fmaf(x[rt][j >> 2][j & 3], pg_half(tk.s, j * NB + b), s[rt][j]);
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int j = 0; j < KPL; ++j) {
                if constexpr (!QUANT) s[rt][j] = P == 4 ? (u ? x[rt][1][j & 3] : x[rt][0][j & 3]) : x[rt][j >> 2][j & 3];
                if constexpr (P == 2) s[rt][j] += pg_dpp<PG_MIRROR>(s[rt][j]);  // the rounded q's and the rest's
                if constexpr (P == 4) s[rt][j] += pg_dpp<PG_HALF_MIRROR>(s[rt][j]);
            }
        if constexpr (more()) pg_load_k(tk, a, kc, at, ln);
        // keys that are not there, or not seen by every row
        const int p = (g >= 2 ? now.p1 : now.p0) + 8 * (g & 1);
        const bool there = (g >= 2 ? now.e1 : now.e0) >= 0;
        const bool some = now.e0 < 0 || now.e1 < 0 || max(now.p0, now.p1) + 16 > t.see_all;
        if (some) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int j = 0; j < KPL; ++j) s[rt][j] = there && p + 4 * u + j < lim[rt] ? s[rt][j] : -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) {  // what lies there must not matter, 0 times infinity is no number
                const uint32_t keep = there && p + j < t.see_any ? 0xFFFFFFFFu : 0u;
#pragma unroll
                for (int x = 0; x < PgV<TYPE, D, KPL>::W; ++x) tv.v[j][x] &= keep;
            }
            if constexpr (QUANT) {
#pragma unroll
                for (int j = 0; j < KPL; ++j) {
                    const uint32_t keep = there && p + 4 * u + j < t.see_any ? 0xFFFFFFFFu : 0u;
#pragma unroll
                    for (int b = 0; b < NB; b += 2) tv.s[(j * NB + b) >> 1] &= keep;
                }
            }
        }
        pg_h8 ph[RT], pl[RT];  // P^T operands: the weights and their rest, or (P > 1) both in one
        float pw[RT][KPL];
        const auto operand = [&](int rt, const float (&y)[KPL]) {
            if constexpr (P == 1) {
                pg_split(y, ph[rt], pl[rt]);
            } else if constexpr (P == 2) {
#pragma unroll
                for (int j = 0; j < 8; ++j) ph[rt][j] = pg_part(y[j], part);
            } else {  // columns c and c ^ 8 have the same row's keys of product 0 and of 1: each takes the other's
                amv_v4u o4;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int mine = (int)pg_bits(amv_h2{pg_part(y[2 * h], part), pg_part(y[2 * h + 1], part)});
                    o4[h] = (uint32_t)__builtin_amdgcn_update_dpp(mine, mine, PG_ROR8, 0xF, 0xC, false);
                    o4[2 + h] = (uint32_t)__builtin_amdgcn_update_dpp(mine, mine, PG_ROR8, 0xF, 0x3, false);
                }
                ph[rt] = __builtin_bit_cast(pg_h8, o4);
            }
        };
        if (some && t.see_all < t.see_any) {
            uint32_t strange = 0;  // bits of the lane's keys
            if constexpr (QUANT) {  // (a scale is a whole block's)
#pragma unroll
                for (int x = 0; x < KPL * NB / 2; ++x) {
                    const uint32_t b = pg_strange(tv.s[x]);
                    strange |= b ? 1u << (4 * u + 2 * x / NB) : 0u;
                    tv.s[x] &= ~(b * 0xFFFFu);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int x = 0; x < PgV<TYPE, D, KPL>::W; ++x) {
                        const uint32_t b = pg_strange(tv.v[j][x]);
                        strange |= b ? 1u << j : 0u;
                        tv.v[j][x] &= ~(b * 0xFFFFu);
                    }
                strange = pg_row16_or(strange);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
                if (strange & ((1u << max(0, min(8, lim[rt] - p))) - 1)) l[rt] = __uint_as_float(0x7FC00000u);
        }
        if constexpr (QUANT) {  // the values' largest scale
            amv_h2 big = {(_Float16)0.0f, (_Float16)0.0f};
#pragma unroll
            for (int x = 0; x < KPL * NB / 2; ++x)
                big = __builtin_elementwise_max(big, __builtin_bit_cast(amv_h2, tv.s[x] & 0x7FFF7FFFu));
            float top = amv_max_x32(amv_max_x16(fmaxf((float)big.x, (float)big.y)));
            if constexpr (P == 4) top = fmaxf(top, pg_dpp<PG_ROR8>(top));
            if (__builtin_amdgcn_readfirstlane(top == INFINITY)) {  // (it is its own rows' matter: the largest of the others)
                float y = 0.0f;
#pragma unroll
                for (int x = 0; x < KPL * NB; ++x) {
                    const float z = fabsf(pg_half(tv.s, x));
                    y = z < INFINITY ? fmaxf(y, z) : y;
                }
                top = amv_max_x32(amv_max_x16(y));
                if constexpr (P == 4) top = fmaxf(top, pg_dpp<PG_ROR8>(top));
            }
            if (__builtin_amdgcn_readfirstlane(top > vref)) {
                const uint32_t e = min(253u, (__float_as_uint(top) >> 23) + 1u);
                const float up = __uint_as_float(e << 23), by = vref * __uint_as_float((254u - e) << 23);
                vref = up;
                vdown = __uint_as_float((254u - e) << 23);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int v = 0; v < T; ++v) o[rt][v] *= by;
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            pg_soften<P>(s[rt], f[rt], m[rt], l[rt], o[rt], pw[rt]);
            if constexpr (QUANT) {
#pragma unroll
                for (int j = 0; j < KPL; ++j) pw[rt][j] *= vdown;
            } else {
                operand(rt, pw[rt]);
            }
        }
#pragma unroll
        for (int v = 0; v < T; ++v) {
            const pg_h8 vf = pg_v_operand<TYPE, D>(tv, v);
            if constexpr (QUANT) {
                if ((v & 1) == 0) {  // products 2 b and 2 b + 1 are block b
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        float y[KPL];
#pragma unroll
                        for (int j = 0; j < KPL; ++j) {
                            y[j] = pw[rt][j] * pg_half(tv.s, j * NB + (v >> 1));
                            // The compiler would round the unrounded product to f16 (v_fma_mixlo_f16) but take the rest from the
                            // f16 of the rounded one; where the two differ, next to a tie, the parts do not sum to y.
                            asm("" : "+v"(y[j]));
                        }
                        operand(rt, y);
                    }
                }
            }
            if constexpr (P == 1) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) o[rt][v] = pg_mfma(vf, pl[rt], o[rt][v]);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) o[rt][v] = pg_mfma(vf, ph[rt], o[rt][v]);
        }
        if constexpr (more()) pg_load_v(tv, a, vc, at, ln);
    };
    for (; i + 4 < end; i += 4) step(std::true_type{});
    if (i < end) step(std::false_type{});

    // the waves' parts together. Lane (c, g) of wave w takes register w of every product: elements of row c that lie side by side
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float lt = amv_sum_x32(amv_sum_x16(l[rt]));
        if constexpr (P == 4) lt += pg_dpp<PG_ROR8>(lt);
        if (g == 0) {
            sm[w][16 * rt + c] = m[rt];
            sl[w][16 * rt + c] = lt;
        }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        if (rt) __syncthreads();
        const float back = QUANT ? vref * 1024.0f : 1.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int v = 0; v < T; ++v) {
                float y = o[rt][v][r];
                if constexpr (P == 2) y += pg_dpp<PG_MIRROR>(y);  // (lanes of part 0 end with their row's)
                if constexpr (P == 4) y += pg_dpp<PG_HALF_MIRROR>(y);
                so(w, r, v) = y * back;
            }
        __syncthreads();
        const int r = t.r0 + 16 * rt + c;
        float M = -INFINITY, L = 0.0f, x[T];
#pragma unroll
        for (int j = 0; j < 4; ++j) M = fmaxf(M, sm[j][16 * rt + c]);
#pragma unroll
        for (int v = 0; v < T; ++v) x[v] = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float mj = sm[j][16 * rt + c], by = mj == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mj - M);
            L = fmaf(sl[j][16 * rt + c], by, L);
#pragma unroll
            for (int v = 0; v < T; ++v) x[v] = fmaf(so(j, w, v), by, x[v]);
        }
        if (r < t.n_rows && c < ROWS) {
            float2* ml;
            float* to = pg_to<D>(a, t, hk, r, z, &ml);
            if (!ml) {
                const float inv = L > 0.0f ? 1.0f / L : L;  // (no keys: 0; a weight that is no number stays one)
#pragma unroll
                for (int v = 0; v < T; ++v) x[v] *= inv;
            } else if (w == 0 && g == 0) {
                *ml = make_float2(M, L);
            }
            const int d = 4 * g + w;  // the operand row
            if constexpr (QUANT) {
#pragma unroll
                for (int v = 0; v < T; v += 2)
                    *reinterpret_cast<float2*>(to + 16 * v + 2 * d) = make_float2(x[v], x[v + 1]);
            } else {
#pragma unroll
                for (int v = 0; v < T; v += 4)
                    *reinterpret_cast<float4*>(to + T * d + v) = make_float4(x[v], x[v + 1], x[v + 2], x[v + 3]);
            }
        }
    }
}

// Many rows (prompts, a prefix): tiles of 32 RW rows, 32 of each wave, whose keys come from memory once for the workgroup: read by each
// wave for itself (pg_few), K's pieces of 16 bytes from 16 rows an instruction keep the loads' address unit busy for all of the time.
// RW = 4: every wave goes over all keys; RW = 2: two waves a row range, each with one half of every step's keys, joined at the end. f16
// K and V rows of 64 keys, a step, go to LDS without registers (global_load_lds), one step ahead in two buffers; the products are those
// of pg_few with RT = 2. The loads write LDS in lane order, so a row's pieces are exchanged on the memory side: K's 16-byte pieces by a
// number of the key that differs among the 16 keys of an operand read, V's 32-byte units by one that takes each value twice among the
// 16 keys of a transposing read (ds_read_b64_tr_b16: 16 lanes pointing at 4 keys' 8-byte quarters of a unit get an element of the 4
// keys each), so both reads meet all banks.
typedef __attribute__((address_space(3))) void pg_lds;
typedef __attribute__((address_space(1))) const void pg_glb;
typedef short pg_s4 __attribute__((ext_vector_type(4)));
typedef short pg_s8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) pg_s4 pg_lds_s4;
// every wave's LDS accesses and vector memory loads (those into LDS too) done, then the workgroup's barrier
#define PG_BARRIER()                        \
    do {                                    \
        asm volatile("" ::: "memory");      \
        __builtin_amdgcn_s_waitcnt(0x0070); \
        __builtin_amdgcn_s_barrier();       \
        asm volatile("" ::: "memory");      \
    } while (0)
// the same without the loads into registers, which may still be on their way
#define PG_BARRIER_LDS()                    \
    do {                                    \
        asm volatile("" ::: "memory");      \
        __builtin_amdgcn_s_waitcnt(0xC07F); \
        __builtin_amdgcn_s_barrier();       \
        asm volatile("" ::: "memory");      \
    } while (0)
__device__ __align__(16) const uint8_t pg_zeros[16] = {};

// Quantized keys and values come through registers, a quarter of a key's row a lane: the integers become f16 (the low bits of 1024 plus
// the value), times the scales in packed f16, the product rounded and the rest (exact, by an fma), each a buffer of its own in LDS, one
// step at a time; the next step's bytes are on their way while this one is worked on. A power of two per key brings its largest scale to
// 2^7 .. 2^8, so that blocks down to 2^-20 of it keep 20 bits; it meets the scores and the weights in f32. Three products of the parts in
// place of two (the rests' own is below 2^-22), but the scales no longer cost an instruction for each row and block: the 2 x 1024 tokens
// over Q8_0 keys took 418 us with every wave working from its own registers (pg_few of 32 rows).
// (true: nothing is written, as a sum is no number and a value that not all rows see may be the reason, which pg_few leaves out)
template <int TYPE, int D, int RW>
__device__ __forceinline__ bool pg_many(const PgAttn& a, int hk, int tile, int z, uint16_t* sKa, uint16_t* sKb, uint16_t* sVa,
                                        uint16_t* sVb) {
    using R = PgRow<TYPE, D>;
    constexpr bool QUANT = TYPE != AMV_T_F16;
    constexpr int NB = D / 32, T = D / 16, PIECES = D / 8;  // (of 16 bytes a row)
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ps = 1 << a.b.pshift;
    PgRows t;
    if (!pg_rows(a, hk, tile, 32 * RW, t)) return false;
    // steps of 64 keys
    const int begin = z * a.split_len >> 6, end = (min(t.see_any, (z + 1) * a.split_len) + 63) >> 6;
    const int seen = t.see_all;  // (by all rows of the tile)
    // the wave's own rows, and which half of a step's keys it takes
    const int rw = w & (RW - 1), kw = w / RW, wr0 = t.r0 + 32 * rw, wr1 = min(wr0 + 31, t.r_last);
    const bool idle = wr0 > t.r_last;
    t.see(a, idle ? t.r_last : wr0, idle ? t.r_last : wr1);
    const int mine = idle ? 0 : min(end, (t.see_any + 63) >> 6);  // steps that its rows see a part of

    // staging: the wave's 16 rows of a step; lane: row `row` of an instruction's, place x of its pieces
    constexpr int RPI = 64 / PIECES, LOADS = 16 / RPI;  // rows of an instruction
    const int row = lane / PIECES, x = lane % PIECES;
    const auto hash_k = [](int key) { return D == 128 ? ((key >> 3 & 3) << 2 | (key & 3)) : ((key >> 3 & 3) << 1 | (key >> 1 & 1)); };
    const auto hash_v = [](int key) { return D == 128 ? ((key & 3) | (key >> 3 & 1) << 2) : ((key >> 1 & 1) | (key >> 3 & 1) << 1); };
    uint32_t ko[LOADS], vo[LOADS];  // bytes from the wave's first row
#pragma unroll
    for (int y = 0; y < LOADS; ++y) {
        const int key = 16 * w + RPI * y + row;
        ko[y] = (RPI * y + row) * 2 * D + 16 * (x ^ hash_k(key));
        vo[y] = (RPI * y + row) * 2 * D + 16 * ((((x >> 1) ^ hash_v(key)) << 1) | (x & 1));
    }
    const size_t chunk = (size_t)ps * (R::ROW + R::SC);
    const uint8_t *kc = a.k + hk * chunk, *vc = a.v + hk * chunk;
    struct Step {
        PgAt a, b;  // its 32-key halves
    };
    const auto where = [&](int i) {
        Step s;
        s.a = pg_where(a, t.pages, t.keys, 2 * i);
        if (64 * i + 32 < t.keys) s.b = pg_where(a, t.pages, t.keys, 2 * i + 1);
        else s.b = {-1, -1, 64 * i + 32, 64 * i + 48};
        return s;
    };
    const auto stage = [&](const Step& s, uint16_t* sK, uint16_t* sV) {
        const int e = w == 0 ? s.a.e0 : w == 1 ? s.a.e1 : w == 2 ? s.b.e0 : s.b.e1;
        const int64_t off = pg_off<AMV_T_F16, D>(a, e, s.a.p0 + 16 * w, false);
        const bool whole = e >= 0 && s.a.p0 + 16 * w + 16 <= t.keys;
        // (scalar: a base in scalar registers and the lane's bytes, not a sum for each load that is kept over the steps)
        const int64_t so = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(off >> 32)) << 32 |
                                     (uint32_t)__builtin_amdgcn_readfirstlane((int)off));
        const uint8_t *ks = kc + so, *vs = vc + so;
#pragma unroll
        for (int y = 0; y < LOADS; ++y) {
            asm volatile("" : "+v"(ko[y]), "+v"(vo[y]));
            __builtin_amdgcn_global_load_lds((pg_glb*)(ks + (size_t)ko[y]), (pg_lds*)(sK + (16 * w + RPI * y) * D), 16, 0, 0);
            if (whole) {
                __builtin_amdgcn_global_load_lds((pg_glb*)(vs + (size_t)vo[y]), (pg_lds*)(sV + (16 * w + RPI * y) * D), 16, 0, 0);
            } else {  // zeros where there is no key: what lies there must not matter, and 0 times infinity is no number
                const uint8_t* from = e >= 0 && s.a.p0 + 16 * w + RPI * y + row < t.keys ? vs + vo[y] : pg_zeros;
                __builtin_amdgcn_global_load_lds((pg_glb*)from, (pg_lds*)(sV + (16 * w + RPI * y) * D), 16, 0, 0);
            }
        }
    };
    // quantized: a lane has a quarter of a key's row (8 elements of each block) in registers, from where put() brings it to LDS
    __shared__ float sF[QUANT ? 2 : 1][QUANT ? 64 : 1];
    constexpr int RAW = QUANT ? R::ROW / 16 : 1, RSC = QUANT ? NB / 2 : 1;
    uint32_t rk[RAW], rv[RAW], sk[RSC], sv[RSC];
    const int key = 16 * w + (lane >> 2), j4 = lane & 3;
    const auto fetch = [&](const Step& s) {
        if constexpr (QUANT) {
            const int e = w == 0 ? s.a.e0 : w == 1 ? s.a.e1 : w == 2 ? s.b.e0 : s.b.e1, p = s.a.p0 + 16 * w;
            const int64_t off = pg_off<TYPE, D>(a, e, p, false) + (lane >> 2) * R::ROW + j4 * (R::ROW / 4);
            const int64_t sof = pg_off<TYPE, D>(a, e, p, true) + (lane >> 2) * R::SC;
            pg_load<R::ROW / 4>(rk, kc + off);
            pg_load<R::SC>(sk, kc + sof);
            pg_load<R::ROW / 4>(rv, vc + off);
            pg_load<R::SC>(sv, vc + sof);
            const uint32_t keep = e >= 0 && p + (lane >> 2) < t.keys ? 0xFFFFFFFFu : 0u;  // values of no key: 0
#pragma unroll
            for (int i = 0; i < RSC; ++i) sv[i] &= keep;
        }
    };
    const auto put = [&]() {
        if constexpr (QUANT) {
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const uint32_t(&x)[RAW] = v ? rv : rk;
                const uint32_t(&sc)[RSC] = v ? sv : sk;
                // the key's scales times the power of two that brings the largest to 2^7 .. 2^8
                amv_h2 big = __builtin_bit_cast(amv_h2, sc[0] & 0x7FFF7FFFu);
                if constexpr (RSC > 1) big = __builtin_elementwise_max(big, __builtin_bit_cast(amv_h2, sc[RSC - 1] & 0x7FFF7FFFu));
                const uint32_t e = max(103u, min(142u, __float_as_uint(fmaxf((float)big.x, (float)big.y)) >> 23));
                const float norm = __uint_as_float((261u - e) << 23);
                if (j4 == 0) sF[v][key] = __uint_as_float((e - 7u) << 23);
                constexpr float zero = TYPE == AMV_T_Q8_0 ? -1152.0f : -1032.0f;  // integers in the low bits of 1024 are 1024 more
                const amv_h2 bias = {(_Float16)zero, (_Float16)zero};
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    uint32_t n[4];
                    if constexpr (TYPE == AMV_T_Q8_0) {
#pragma unroll
                        for (int m = 0; m < 4; ++m) {
                            const uint32_t word = (v ? x[m * (D / 64) + (b >> 1)] : x[2 * b + (m >> 1)]) ^ 0x80808080u;
                            n[m] = __builtin_amdgcn_perm(0x64646464u, word, ((v ? b : m) & 1) ? 0x04030402u : 0x04010400u);
                        }
                    } else if (v) {  // elements 0, 2, 1, 3 and 4, 6, 5, 7
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            uint32_t z;
                            if constexpr (D == 128) {  // byte b of words 2 m and 2 m + 1
                                z = __builtin_amdgcn_perm(x[(2 * m + 1) % RAW], x[2 * m % RAW], 0x0C040C00u + 0x00010001u * b);
                            } else {                   // bytes b and 2 + b of word m
                                z = (x[m] >> (8 * b)) & 0x00FF00FFu;
                            }
                            n[2 * m] = (z & 0x000F000Fu) | 0x64006400u;
                            n[2 * m + 1] = ((z >> 4) & 0x000F000Fu) | 0x64006400u;
                        }
                    } else {  // elements 0, 4, 1, 5, 2, 6, 3, 7
#pragma unroll
                        for (int m = 0; m < 4; ++m) n[m] = ((x[b] >> (4 * m)) & 0x000F000Fu) | 0x64006400u;
                    }
                    const _Float16 s1 = (_Float16)(pg_half(sc, b) * norm);
                    const amv_h2 s2 = {s1, s1};
                    amv_v4u hi, lo;
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        const amv_h2 y = __builtin_bit_cast(amv_h2, n[m]) + bias, h = y * s2;
                        hi[m] = pg_bits(h);
                        lo[m] = pg_bits(__builtin_elementwise_fma(y, s2, -h));
                    }
                    const int piece = 4 * b + j4;
                    const int to = key * D + 8 * (v ? (((piece >> 1) ^ hash_v(key)) << 1) | (piece & 1) : piece ^ hash_k(key));
                    *reinterpret_cast<amv_v4u*>((v ? sVa : sKa) + to) = hi;
                    *reinterpret_cast<amv_v4u*>((v ? sVb : sKb) + to) = lo;
                }
            }
        }
    };
    Step at = {};
    if (begin < end) {
        at = where(begin);
        if constexpr (QUANT) fetch(at);
        else stage(at, sKa, sVa);
    }
    pg_h8 qh[2][NB], ql[2][NB];
    float f[2], m[2], l[2];
    int lim[2];
    pg_f4 o[2][T];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
        const int r = min(t.r0 + 16 * rt + c, t.r_last);
        lim[rt] = a.kind == PG_PREFIX ? t.keys : min(t.keys, t.place0 + r / a.G + 1);
        float y[NB][8];
        f[rt] = pg_query<D>(a, t, hk, r, g, y);
#pragma unroll
        for (int s = 0; s < NB; ++s) {
            if constexpr (TYPE == AMV_T_Q4_0) {  // in put()'s order
                const float z[8] = {y[s][0], y[s][4], y[s][1], y[s][5], y[s][2], y[s][6], y[s][3], y[s][7]};
                pg_split(z, qh[rt][s], ql[rt][s]);
            } else {
                pg_split(y[s], qh[rt][s], ql[rt][s]);
            }
        }
        m[rt] = -INFINITY;
        l[rt] = 0.0f;
#pragma unroll
        for (int v = 0; v < T; ++v) o[rt][v] = pg_f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // the lane's places in the rows of 32 keys: K's key of product 0 and its piece g (+ 4 b: by XOR), V's key and unit 0 (v: by XOR)
    const int kx = (8 * (c >> 2) + (c & 3)) * D + 8 * (g ^ (D == 128 ? c : c >> 1));  // (hash_k of both products' key)
    const int vx = (8 * g + (c >> 2)) * D + 16 * hash_v(8 * g + (c >> 2)) + 4 * (c & 3);  // (and hash_v of key + 4)
    float vref = 0.0f;  // quantized: the largest power of two of a key's values met
    const auto half = [&](const PgAt& now, const uint16_t* sK, const uint16_t* sV, int h32) {  // 32 keys
        int kx0 = kx, vx0 = vx;  // (not known to be the same each time: their sums would be kept, in registers that are not there)
        asm volatile("" : "+v"(kx0), "+v"(vx0));
        pg_f4 y[2][2];
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) y[rt][0] = y[rt][1] = pg_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const pg_h8 kf = *reinterpret_cast<const pg_h8*>(&sK[(kx0 ^ (32 * b)) + 4 * h * D]);
                if constexpr (QUANT) {
                    const pg_h8 kr = *reinterpret_cast<const pg_h8*>(&sKb[32 * D * h32 + (kx0 ^ (32 * b)) + 4 * h * D]);
#pragma unroll
                    for (int rt = 0; rt < 2; ++rt) y[rt][h] = pg_mfma(kr, qh[rt][b], y[rt][h]);
                }
#pragma unroll
                for (int rt = 0; rt < 2; ++rt) y[rt][h] = pg_mfma(kf, ql[rt][b], y[rt][h]);
#pragma unroll
                for (int rt = 0; rt < 2; ++rt) y[rt][h] = pg_mfma(kf, qh[rt][b], y[rt][h]);
            }
        float s[2][8], pw[8];
#pragma unroll
        for (int rt = 0; rt < 2; ++rt)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                s[rt][j] = y[rt][j >> 2][j & 3];
                if constexpr (QUANT) s[rt][j] *= sF[0][32 * h32 + 8 * g + j];
            }
        if (now.e0 < 0 || now.e1 < 0 || now.p1 + 16 > t.see_all) {
            const int p = now.p0 + 8 * g;
            const bool there = (g >= 2 ? now.e1 : now.e0) >= 0;
#pragma unroll
            for (int rt = 0; rt < 2; ++rt)
#pragma unroll
                for (int j = 0; j < 8; ++j) s[rt][j] = there && p + j < lim[rt] ? s[rt][j] : -INFINITY;
        }
        pg_h8 ph[2], pl[2];
        float fv[QUANT ? 8 : 1];
        if constexpr (QUANT) {
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                fv[j] = sF[1][32 * h32 + 8 * g + j];
                top = fmaxf(top, fv[j]);
            }
            top = amv_max_x32(amv_max_x16(top));
            if (__builtin_amdgcn_readfirstlane(top > vref)) {
                const float by = vref * __uint_as_float((254u << 23) - __float_as_uint(top));
                vref = top;
#pragma unroll
                for (int rt = 0; rt < 2; ++rt)
#pragma unroll
                    for (int v = 0; v < T; ++v) o[rt][v] *= by;
            }
            const float down = __uint_as_float((254u << 23) - __float_as_uint(vref));  // (1 / vref: powers of two)
#pragma unroll
            for (int j = 0; j < 8; ++j) fv[j] *= down;
        }
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
            pg_soften<1>(s[rt], f[rt], m[rt], l[rt], o[rt], pw);
            if constexpr (QUANT) {
#pragma unroll
                for (int j = 0; j < 8; ++j) pw[j] *= fv[j];
            }
            pg_split(pw, ph[rt], pl[rt]);
        }
#pragma unroll
        for (int v = 0; v < T; ++v) {
            const auto value = [&](const uint16_t* at0) {
                const pg_s4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pg_lds_s4*)(__attribute__((address_space(3))) uint16_t*)at0);
                const pg_s4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pg_lds_s4*)(__attribute__((address_space(3))) uint16_t*)(at0 + 4 * D));
                const pg_s8 ab = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
                return __builtin_bit_cast(pg_h8, ab);
            };
            const pg_h8 vf = value(&sV[vx0 ^ (16 * v)]);
            if constexpr (QUANT) {
                const pg_h8 vr = value(&sVb[32 * D * h32 + (vx0 ^ (16 * v))]);
#pragma unroll
                for (int rt = 0; rt < 2; ++rt) o[rt][v] = pg_mfma(vr, ph[rt], o[rt][v]);
            }
#pragma unroll
            for (int rt = 0; rt < 2; ++rt) o[rt][v] = pg_mfma(vf, pl[rt], o[rt][v]);
#pragma unroll
            for (int rt = 0; rt < 2; ++rt) o[rt][v] = pg_mfma(vf, ph[rt], o[rt][v]);
        }
    };
    const auto step = [&](const Step& now, const uint16_t* sK, const uint16_t* sV) {
        if constexpr (RW == 4) {
            half(now.a, sK, sV, 0);
            half(now.b, sK + 32 * D, sV + 32 * D, 1);
        } else {
            half(kw ? now.b : now.a, sK + 32 * D * kw, sV + 32 * D * kw, kw);
        }
    };
    if constexpr (QUANT) {
        for (int i = begin; i < end; ++i) {
            put();
            PG_BARRIER();
            Step next = at;
            if (i + 1 < end) {
                next = where(i + 1);
                fetch(next);
            }
            if (i < mine) step(at, sKa, sVa);
            at = next;
            PG_BARRIER_LDS();
        }
#pragma unroll
        for (int rt = 0; rt < 2; ++rt)
#pragma unroll
            for (int v = 0; v < T; ++v) o[rt][v] *= vref;
    }
    if constexpr (!QUANT) PG_BARRIER();
    for (int i = QUANT ? end : begin; i < end; i += 2) {
        Step next = at;
        if (i + 1 < end) {
            next = where(i + 1);
            stage(next, sKb, sVb);
        }
        if (i < mine) step(at, sKa, sVa);
        PG_BARRIER();
        if (i + 1 >= end) break;
        if (i + 2 < end) {
            at = where(i + 2);
            stage(at, sKa, sVa);
        }
        if (i + 1 < mine) step(next, sKb, sVb);
        PG_BARRIER();
    }
    float* const ex = reinterpret_cast<float*>(rw ? sKb : sKa) + lane;  // [row tile][product][register][lane]
    float* const ml = reinterpret_cast<float*>(sVa) + 256 * rw + lane;  // [row tile][m, l][lane]
    float sum = 0.0f;  // no number: one of the sums is none, or infinite
    if (!idle)
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
            sum = fmaf(l[rt], 0.0f, sum);
#pragma unroll
            for (int v = 0; v < T; ++v)
#pragma unroll
                for (int r = 0; r < 4; ++r) sum = fmaf(o[rt][v][r], 0.0f, sum);
        }
    if constexpr (RW == 2) {  // the second half's sums go to the first's, through the buffers
        if (kw) {
#pragma unroll
            for (int rt = 0; rt < 2; ++rt) {
                ml[128 * rt] = m[rt];
                ml[128 * rt + 64] = l[rt];
#pragma unroll
                for (int v = 0; v < T; ++v)
#pragma unroll
                    for (int r = 0; r < 4; ++r) ex[64 * ((rt * T + v) * 4 + r)] = o[rt][v][r];
            }
        }
    }
    bool again = __builtin_amdgcn_readfirstlane(__syncthreads_or(sum != sum));
    if (again) {
        // A sum that is no number is its own rows' matter (a query, a key, a value that they see), unless a value that not all rows see
        // is infinite or no number. Only those keys' values are looked at, a row tile's tokens and a step of them at most: 2 x 1024
        // tokens, those of one sequence no number, take 143 us in place of 139; all of pg_few again would be 956.
        bool strange = false;
        constexpr int UNITS = QUANT ? 1 : PIECES;  // of a value: its scales, or 16 bytes each
        for (int i = (int)threadIdx.x; i < (min(64 * end, t.keys) - max(64 * begin, seen)) * UNITS; i += 256) {
            const int key = max(64 * begin, seen) + i / UNITS, e = t.pages[key >> a.b.pshift];
            if ((uint32_t)e >= (uint32_t)a.n_pages) continue;
            uint32_t v[QUANT ? RSC : 4];
            pg_load<QUANT ? R::SC : 16>(v, vc + pg_off<TYPE, D>(a, e, key, QUANT) + 16 * (i % UNITS));
#pragma unroll
            for (int x = 0; x < (QUANT ? RSC : 4); ++x) strange |= pg_strange(v[x]) != 0;
        }
        again = __builtin_amdgcn_readfirstlane(__syncthreads_or(strange));
    }
    if (again) return true;
    if (idle || (RW == 2 && kw)) return false;
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
        float L = l[rt];
        if constexpr (RW == 2) {
            const float m1 = ml[128 * rt], M = fmaxf(m[rt], m1);
            const float f0 = m[rt] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[rt] - M);
            const float f1 = m1 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m1 - M);
            L = fmaf(L, f0, ml[128 * rt + 64] * f1);
            m[rt] = M;
#pragma unroll
            for (int v = 0; v < T; ++v)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[rt][v][r] = fmaf(o[rt][v][r], f0, ex[64 * ((rt * T + v) * 4 + r)] * f1);
        }
        L = amv_sum_x32(amv_sum_x16(L));
        const int r = t.r0 + 16 * rt + c;
        if (r > t.r_last) continue;
        float2* part;
        float* to = pg_to<D>(a, t, hk, r, z, &part);
        float inv = 1.0f;
        if (!part) inv = L > 0.0f ? 1.0f / L : L;
        else if (g == 0) *part = make_float2(m[rt], L);
#pragma unroll
        for (int v = 0; v < T; ++v) {
            pg_f4 y = o[rt][v] * inv;
            if constexpr (TYPE == AMV_T_Q4_0) y = pg_f4{y.x, y.z, y.y, y.w};  // (put()'s order)
            *reinterpret_cast<pg_f4*>(to + 16 * v + 4 * g) = y;
        }
    }
    return false;
}

// A launch has up to three jobs, one after the other over the workgroups, so that one's reading fills the other's computing: tiles of
// many rows (of the prefix, of sequences with many tokens), then those of few.
struct PgJobs {
    PgAttn a[3];
    int n[3];  // workgroups
};
__device__ __forceinline__ void pg_place_of(const PgAttn& a, int b, int& hk, int& tile, int& z) {
    hk = b % a.n_head_kv;
    b /= a.n_head_kv;
    tile = b % a.tiles;
    z = b / a.tiles;
}
template <int TYPE, int D, int RT, int P>
__global__ __launch_bounds__(256, 2) void k_paged_few(PgJobs jobs) {  // jobs 1 and 2
    __shared__ float so[2][32 * D];
    const int b = (int)blockIdx.x, k = b < jobs.n[1] ? 1 : 2;
    int hk, tile, z;
    pg_place_of(jobs.a[k], k == 1 ? b : b - jobs.n[1], hk, tile, z);
    pg_few<TYPE, D, RT, P>(jobs.a[k], hk, tile, 16 * RT / P, 0, z, so[0], so[1]);
}
template <int TYPE, int D, int RT, int P, int RW>
__global__ __launch_bounds__(256, 2) void k_paged_many_few(PgJobs jobs) {  // jobs 0 and 1 of many rows, 2 of few
    // buffers as variables of their own: reads of one do not wait for the loads into another
    __shared__ __align__(16) uint16_t sKa[64 * D], sKb[64 * D], sVa[64 * D], sVb[64 * D];
    float *so0 = reinterpret_cast<float*>(sKa), *so1 = reinterpret_cast<float*>(sKb);
    int b = (int)blockIdx.x, hk, tile, z;
    const int k = b < jobs.n[0] ? 0 : b < jobs.n[0] + jobs.n[1] ? 1 : 2;
    if (k > 0) b -= jobs.n[0];
    if (k > 1) b -= jobs.n[1];
    pg_place_of(jobs.a[k], b, hk, tile, z);
    constexpr int ROWS = 16 * RT / P;
    if (k < 2 && !pg_many<TYPE, D, RW>(jobs.a[k], hk, tile, z, sKa, sKb, sVa, sVb)) return;
    const int rows = k < 2 ? 32 * RW : ROWS;
    for (int sub = 0; sub < rows / ROWS; ++sub) {
        if (sub) __syncthreads();
        pg_few<TYPE, D, RT, P>(jobs.a[k], hk, tile, rows, sub, z, so0, so1);
    }
}

// out = sum_z w_z O_z / sum_z w_z l_z over the parts z of a row's keys, w_z = 2^(m_z - max m): one wave per row. A row has parts of
// its own keys, laid out by sequence where that has at most rows_most rows and else by row, and of the prefix. Bound: the launch and
// two dependent reads (2.4 us for 32 rows of 7 parts, 4.5 for 96 of 21; reads of 8 parts at once, and 4 or 2 where no more are left,
// are a microsecond less than always 8 for 32 rows of 6 parts).
struct PgParts {
    const float2* ml;
    const float* acc;
    int n;
};
struct PgMerge {
    PgBatch b;
    PgParts one, many, pre;
    float* out;
    int n_head, n_head_kv, G, rows_most;
    int by_seq;  // only sequences of few rows have parts: the waves go over their rows, not over all tokens'
};
template <int D>
__global__ __launch_bounds__(256) void k_paged_merge(PgMerge a) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63;
    const int64_t at = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int64_t row = at, own_row;
    PgParts own = a.one;
    if (a.by_seq) {
        if (at >= (int64_t)a.b.n_seq * a.n_head_kv * a.rows_most) return;
        const int hs = (int)(at / a.rows_most), r = (int)(at - (int64_t)hs * a.rows_most), s = hs / a.n_head_kv;
        const int first = a.b.first(s), n_rows = (a.b.last(s) - first) * a.G;
        if (n_rows > a.rows_most || r >= n_rows) return;
        own_row = at;
        row = (int64_t)(first + r / a.G) * a.n_head + (hs - s * a.n_head_kv) * a.G + r % a.G;
    } else {
        const int tok = (int)(row / a.n_head), h = (int)(row - (int64_t)tok * a.n_head);
        if (tok >= a.b.n_tok) return;
        const int s = pg_seq_of(a.b, tok);
        if (s >= a.b.n_seq) return;
        const int first = a.b.first(s);
        const bool few = (a.b.last(s) - first) * a.G <= a.rows_most;
        if (!few) own = a.many;
        if (!own.n) return;  // its workgroup wrote the row
        own_row = few ? ((int64_t)s * a.n_head_kv + h / a.G) * a.rows_most + (tok - first) * a.G + h % a.G : row;
    }
    const float2 *ml0 = own.ml + own_row * own.n, *ml1 = a.pre.ml + row * a.pre.n;
    const float *acc0 = own.acc + own_row * own.n * D, *acc1 = a.pre.acc + row * a.pre.n * D;
    float M = -INFINITY;
    for (int z = lane; z < own.n; z += 64) M = fmaxf(M, ml0[z].x);
    for (int z = lane; z < a.pre.n; z += 64) M = fmaxf(M, ml1[z].x);
    M = amv_wave_max_u(M);
    float x[E] = {}, L = 0.0f;
    const auto join = [&](const float2* ml, const float* acc, int n) {
        for (int z0 = 0; z0 < n; z0 += 64) {
            const float2 p = z0 + lane < n ? ml[z0 + lane] : make_float2(-INFINITY, 0.0f);
            const float wz = p.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(p.x - M);
            L = fmaf(wz, p.y, L);
            const uint64_t has = __builtin_amdgcn_ballot_w64(p.x != -INFINITY);
            const int n_here = has ? 64 - __builtin_clzll(has) : 0;  // up to the last part that has keys
            const auto some = [&](auto width, int j0) {  // parts j0 .. j0 + width - 1, their reads on the way together
                constexpr int W = width();
                float y[W][E];
#pragma unroll
                for (int j = 0; j < W; ++j)
#pragma unroll
                    for (int e = 0; e < E; ++e) y[j][e] = acc[(int64_t)(z0 + min(j0 + j, n_here - 1)) * D + E * lane + e];
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    const float by = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wz), min(j0 + j, 63)));
#pragma unroll
                    for (int e = 0; e < E; ++e) x[e] = j0 + j < n_here ? fmaf(by, y[j][e], x[e]) : x[e];
                }
            };
            int j0 = 0;
            for (; j0 + 4 < n_here; j0 += 8) some(std::integral_constant<int, 8>{}, j0);
            if (j0 + 2 < n_here) some(std::integral_constant<int, 4>{}, j0);
            else if (j0 < n_here) some(std::integral_constant<int, 2>{}, j0);
        }
    };
    join(ml1, acc1, a.pre.n);
    join(ml0, acc0, own.n);
    L = amv_wave_sum(L);
    const float inv = L > 0.0f ? 1.0f / L : L;
#pragma unroll
    for (int e = 0; e < E; ++e) a.out[row * D + E * lane + e] = x[e] * inv;
}

// ---------------------------------------------------------------------------------------------------------------- host
// Row tiles: rt times 16 rows, or 16 / pack of them where rows are few: the products' 16 columns then hold the two f16 of every row side
// by side, and with pack 4 the two products' keys too, so that each lane's scores are of use to half the lanes rather than an eighth.
struct PgTiles {
    int rt, pack;
    int rows() const { return 16 * rt / pack; }
    int of(int64_t n) const { return (int)((n + rows() - 1) / rows()); }
};
// Two row tiles (17 to 32 rows) of heads of 128 need more than the 256 registers of two waves a SIMD: 3 are spilled over f16 keys, 64
// over Q4_0, 86 over Q8_0, and 41, 103 and 119 in the kernels that have tiles of many rows too. 32 sequences of up to 4096 keys in
// groups of 32 heads take 30, 42 and 54 us, their bytes 18, 5 and 10; 64 of up to 5 tokens in groups of 4 behind 8192 keys (their own up
// to 512 in such tiles) 88 over f16 and 130 over Q4_0.
static PgTiles pg_tiles(int64_t rows) { return {rows > 16 ? 2 : 1, rows <= 4 ? 4 : rows <= 8 ? 2 : 1}; }
// How a call is launched, and the workspace of the parts
struct PgPlan {
    PgTiles few;                            // tiles of few rows: sequences (or listed tokens), ta tiles each, and a small batch's prefix
    int ta, n_one, len_one;                 // their parts
    int many_rows;                          // rows of the other tiles: 64 or 128
    int find, rows_most, n_find, len_find;  // sequences of more rows than rows_most
    int64_t find_tiles;
    bool pre_many;                          // the prefix in tiles of many rows
    int pre_tiles, n_pre, len_pre;
    int64_t w_one, w_many, w_pre;           // parts in the workspace
    int64_t bytes(int64_t D) const { return (w_one + w_many + w_pre) * (8 + 4 * D); }
};
// parts of `keys` keys for `units` workgroups' worth of rows: two workgroups a CU, none of less than 128 keys (a tile for each of its
// waves), and up to 256 keys no parts, as their merge is a launch of its own. More and shorter parts cost their prologues and the merge
// (us at 512 / 1024 / 2048 workgroups: 64 sequences of up to 4096 f16 keys 136 / 147 / 144, 3 of 65536 Q8_0 keys 78 / 78 / 82; one of 777
// with parts of 256 keys 9.6, of 128 9.3)
static int pg_parts(int64_t units, int64_t keys, int* len, int target = 512) {
    units = std::max<int64_t>(1, units);
    const int64_t n = keys <= 256 ? 1 : std::max<int64_t>(1, std::min<int64_t>(target / units, (keys + 127) / 128));
    int64_t l = ((keys + n - 1) / n + 127) / 128 * 128;
    l = std::max<int64_t>(128, l);
    *len = (int)l;
    return (int)std::max<int64_t>(1, (keys + l - 1) / l);
}
static PgPlan pg_plan(const amv_paged_kv* kv, const amv_paged_batch* b, int64_t n_head, int64_t n_prefix, int64_t n_sel) {
    PgPlan p = {};
    const int64_t G = n_head / kv->n_head_kv, all = b->n_tok * G;
    if (n_sel > 0) {
        p.few = pg_tiles(G);
        p.ta = p.few.of(G);
        p.n_one = pg_parts(b->n_tok * kv->n_head_kv * p.ta, n_sel * kv->page_size, &p.len_one);
        if (p.n_one > 1) p.w_many = b->n_tok * n_head * p.n_one;
        return p;
    }
    const int64_t rows = std::min(b->max_q, b->n_tok) * G;
    // 17 to 32 rows are one tile of few rows, but not of Q8_0 keys, whose registers for it suffice least (32 sequences of up to 8 tokens
    // after up to 4096 keys 147 us, in half a tile of 64 rows 141; Q4_0 122 and 140)
    const int64_t most = kv->type == AMV_T_Q8_0 ? 16 : 32;
    p.pre_many = all > most;
    p.few = pg_tiles(n_prefix > 0 && !p.pre_many ? all : rows <= most ? rows : G);
    p.rows_most = (int)std::max<int64_t>(p.few.rows(), G);
    p.ta = p.few.of(p.rows_most);
    p.n_one = pg_parts(b->n_seq * kv->n_head_kv * p.ta, b->max_kv, &p.len_one);
    p.find = rows > p.rows_most;
    // Tiles of 128 rows do more with a step (8192 tokens 996 us, with 64 rows 1150; 512 after 7488 others 174 and 219; 128 sequences
    // behind 16384 keys 107 and 119), those of 64 rows share the GPU more evenly where the larger are no more than a few for each CU and
    // not cut into parts (2048 tokens 104 and 113, 512 28 and 35), and read a prefix for up to 64 rows as soon.
    const int64_t large = all / 128 * kv->n_head_kv;
    const bool even = (!p.find || rows <= 64 || b->max_kv <= 1024 || (large >= 256 && large < 1024)) && (n_prefix == 0 || all <= 64);
    p.many_rows = even ? 64 : 128;
    if (p.find) {
        p.find_tiles = all / p.many_rows + b->n_seq;
        p.n_find = pg_parts(all / p.many_rows * kv->n_head_kv + 1, b->max_kv, &p.len_find);
    }
    if (n_prefix > 0) {
        p.pre_tiles = p.pre_many ? (int)((all + p.many_rows - 1) / p.many_rows) : p.few.of(all);
        // (fewer parts: each is all rows' sums again. 32 sequences behind 8192 keys 39 us with 512, 31 with 384)
        p.n_pre = pg_parts(p.pre_tiles * kv->n_head_kv, n_prefix, &p.len_pre, p.pre_many ? 384 : 512);
    }
    if (p.n_one > 1 || p.n_pre) p.w_one = b->n_seq * kv->n_head_kv * p.rows_most * p.n_one;
    if (p.find && (p.n_find > 1 || p.n_pre)) p.w_many = b->n_tok * n_head * p.n_find;
    p.w_pre = b->n_tok * n_head * p.n_pre;
    return p;
}

extern "C" int64_t amv_paged_attn_workspace_bytes(const amv_paged_kv* kv, const amv_paged_batch* batch, int64_t n_head,
                                                  int64_t n_prefix, int64_t n_sel) {
    if (pg_check("amv_paged_attn_workspace_bytes", kv, batch, n_head) || n_prefix < 0 || n_sel < 0) return -1;
    return pg_plan(kv, batch, n_head, n_prefix, n_sel).bytes(kv->D);
}

template <int TYPE, int D, int RT, int P>
static void pg_launch(const PgJobs& j, int many, hipStream_t st) {
    const dim3 grid((unsigned)(j.n[0] + j.n[1] + j.n[2]));
    if (many == 64) hipLaunchKernelGGL((k_paged_many_few<TYPE, D, RT, P, 2>), grid, dim3(256), 0, st, j);
    else if (many) hipLaunchKernelGGL((k_paged_many_few<TYPE, D, RT, P, 4>), grid, dim3(256), 0, st, j);
    else hipLaunchKernelGGL((k_paged_few<TYPE, D, RT, P>), grid, dim3(256), 0, st, j);
}
template <int TYPE, int D>
static void pg_launch(const PgJobs& j, PgTiles t, int many, hipStream_t st) {
    if (t.pack == 4) pg_launch<TYPE, D, 1, 4>(j, many, st);
    else if (t.pack == 2) pg_launch<TYPE, D, 1, 2>(j, many, st);
    else if (t.rt == 1) pg_launch<TYPE, D, 1, 1>(j, many, st);
    else pg_launch<TYPE, D, 2, 1>(j, many, st);
}
static void pg_launch(int type, int D, const PgJobs& j, PgTiles t, int many, hipStream_t st) {
    if (D == 128) {
        if (type == AMV_T_F16) pg_launch<AMV_T_F16, 128>(j, t, many, st);
        else if (type == AMV_T_Q8_0) pg_launch<AMV_T_Q8_0, 128>(j, t, many, st);
        else pg_launch<AMV_T_Q4_0, 128>(j, t, many, st);
    } else {
        if (type == AMV_T_F16) pg_launch<AMV_T_F16, 64>(j, t, many, st);
        else if (type == AMV_T_Q8_0) pg_launch<AMV_T_Q8_0, 64>(j, t, many, st);
        else pg_launch<AMV_T_Q4_0, 64>(j, t, many, st);
    }
}

static int pg_attn(const char* what, const amv_paged_kv* kv, const amv_paged_batch* b, const int32_t* list, int64_t n_prefix,
                   int64_t n_sel, const float* q, int64_t q_stride, float* out, int64_t n_head, float scale, void* workspace,
                   int64_t workspace_bytes, void* stream) {
    if (const int rc = pg_check(what, kv, b, n_head)) return rc;
    if (b->n_tok == 0) return AMV_OK;
    AMV_REQUIRE(q && out, "%s: null pointer", what);
    AMV_REQUIRE(q_stride >= n_head * kv->D && q_stride % 4 == 0 && ((uintptr_t)q & 15) == 0 && ((uintptr_t)out & 15) == 0,
                "%s: q rows too short, or q or out not 16-byte aligned", what);
    const PgPlan p = pg_plan(kv, b, n_head, n_prefix, n_sel);
    const int64_t rows = b->n_tok * n_head, need = p.bytes(kv->D);
    AMV_REQUIRE(need == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need),
                "%s: workspace of %lld bytes, %lld needed (16-byte aligned)", what, (long long)workspace_bytes, (long long)need);
    PgAttn a = {};
    a.b = pg_batch(kv, b);
    a.k = (const uint8_t*)kv->k;
    a.v = (const uint8_t*)kv->v;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.page_stride = kv->page_stride;
    a.scale2 = scale * AMV_LOG2E;
    a.n_pages = (int)kv->n_pages;
    a.n_head = (int)n_head;
    a.n_head_kv = kv->n_head_kv;
    a.G = (int)(n_head / kv->n_head_kv);
    a.list = list;
    // workspace: the weighted values of the parts of own keys (by sequence, by row) and of the prefix, then their (m, l)
    float* const acc = (float*)workspace;
    float2* const ml = (float2*)(acc + (p.w_one + p.w_many + p.w_pre) * kv->D);
    PgMerge m = {a.b, {ml, acc, p.w_one ? p.n_one : 0},
                 {ml + p.w_one, acc + p.w_one * kv->D, p.w_many ? (n_sel > 0 ? p.n_one : p.n_find) : 0},
                 {ml + p.w_one + p.w_many, acc + (p.w_one + p.w_many) * kv->D, p.n_pre},
                 out, (int)n_head, kv->n_head_kv, a.G, n_sel > 0 ? -1 : p.rows_most, n_sel == 0 && !p.w_many && !p.w_pre};
    PgJobs jobs = {};
    int64_t groups = 0;
    const auto job = [&](int k, int kind, int64_t tiles, int parts, int len, const PgParts& into) {
        PgAttn& x = jobs.a[k] = a;
        x.kind = kind;
        x.n_list = (int)(kind == PG_PREFIX ? n_prefix : n_sel);
        x.ta = p.ta;
        x.rows_most = p.rows_most;
        x.tiles = (int)tiles;
        x.n_split = parts;
        x.split_len = len;
        x.ml = into.n ? const_cast<float2*>(into.ml) : nullptr;
        x.acc = const_cast<float*>(into.acc);
        jobs.n[k] = (int)(tiles * parts * kv->n_head_kv);
        groups += tiles * parts * kv->n_head_kv;
    };
    if (p.find) job(0, PG_FIND, p.find_tiles, p.n_find, p.len_find, m.many);
    if (p.n_pre) job(1, PG_PREFIX, p.pre_tiles, p.n_pre, p.len_pre, m.pre);
    if (n_sel > 0) job(2, PG_LIST, b->n_tok * p.ta, p.n_one, p.len_one, m.many);
    else job(2, PG_ONE, b->n_seq * p.ta, p.n_one, p.len_one, m.one);
    AMV_REQUIRE(groups <= PG_MAX_GROUPS, "%s: batch too large", what);
    hipStream_t st = amv_stream(stream);
    pg_launch(kv->type, kv->D, jobs, p.few, p.find || (p.n_pre && p.pre_many) ? p.many_rows : 0, st);
    if (p.w_one + p.w_many + p.w_pre) {
        const dim3 grid((unsigned)(((m.by_seq ? b->n_seq * kv->n_head_kv * p.rows_most : rows) + 3) / 4));
        if (kv->D == 128) hipLaunchKernelGGL(k_paged_merge<128>, grid, dim3(256), 0, st, m);
        else hipLaunchKernelGGL(k_paged_merge<64>, grid, dim3(256), 0, st, m);
    }
    return amv_check_launch(what);
}

extern "C" int amv_paged_attn(const amv_paged_kv* kv, const amv_paged_batch* batch, const float* q, int64_t q_stride, float* out,
                              int64_t n_head, float scale, void* workspace, int64_t workspace_bytes, void* stream) {
    return pg_attn("amv_paged_attn", kv, batch, nullptr, 0, 0, q, q_stride, out, n_head, scale, workspace, workspace_bytes, stream);
}

extern "C" int amv_paged_attn_shared(const amv_paged_kv* kv, const amv_paged_batch* batch, const int32_t* prefix_table,
                                     int64_t n_prefix, const float* q, int64_t q_stride, float* out, int64_t n_head, float scale,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
    AMV_REQUIRE(n_prefix >= 0 && n_prefix <= (int64_t)1 << 30 && (n_prefix == 0 || prefix_table),
                "amv_paged_attn_shared: a prefix of %lld keys without pages", (long long)n_prefix);
    return pg_attn("amv_paged_attn_shared", kv, batch, prefix_table, n_prefix, 0, q, q_stride, out, n_head, scale, workspace,
                   workspace_bytes, stream);
}

extern "C" int amv_paged_attn_sparse(const amv_paged_kv* kv, const amv_paged_batch* batch, const int32_t* sel, int64_t n_sel,
                                     const float* q, int64_t q_stride, float* out, int64_t n_head, float scale, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
    AMV_REQUIRE((sel || (batch && batch->n_tok == 0)) && n_sel > 0 && n_sel <= PG_MAX_PAGES, "amv_paged_attn_sparse: %lld selected pages", (long long)n_sel);
    return pg_attn("amv_paged_attn_sparse", kv, batch, sel, 0, n_sel, q, q_stride, out, n_head, scale, workspace, workspace_bytes,
                   stream);
}
