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
// of two to below 2 first, so that no f32 is out of f16's range; the weights' reference is kept 12 to 15 below the running maximum, so
// that the rest keeps its bits beside a dominating key.
// Quantized caches: the integers are exact in f16. Block b of a key is one product of K's (its own accumulator, then times the
// block's scale in f32), and two of V's products, whose weights are multiplied by the value's scale before they are split. The
// scales are brought to at most 1 by a power of two that follows the largest met (as the maximum does), which keeps weight times
// scale in f16's range whatever the values' size.
//
// Four waves of a workgroup take the 32-key tiles of a range in turn and join in LDS; ranges of a long sequence go to several
// workgroups (blockIdx.y), joined by k_paged_merge from
// (m, l, O) in the workspace.
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
    int n_split, split_len;  // parts (blockIdx.y) of the keys and their length
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

// integers u (value + 8 or + 128) in the low bits of a word's two halves, as f16 values times 2^-10: such a half is the f16 u 2^-24,
// and u 2^-24 2^14 - bias 2^-10 is exact
template <int TYPE>
__device__ __forceinline__ uint32_t pg_f16_of(uint32_t u) {
    constexpr float bias = (TYPE == AMV_T_Q8_0 ? 128.0f : 8.0f) / 1024.0f;
    const amv_h2 m = {(_Float16)16384.0f, (_Float16)16384.0f}, b = {(_Float16)-bias, (_Float16)-bias};
    return pg_bits(__builtin_elementwise_fma(__builtin_bit_cast(amv_h2, u), m, b));
}
// the operand of product s of K: 8 f16
template <int TYPE, int D>
__device__ __forceinline__ pg_h8 pg_k_operand(const uint32_t* k, int s) {
    amv_v4u x;
    if constexpr (TYPE == AMV_T_F16) {
        x = amv_v4u{k[4 * s], k[4 * s + 1], k[4 * s + 2], k[4 * s + 3]};
    } else if constexpr (TYPE == AMV_T_Q8_0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t w = k[2 * s + h] ^ 0x80808080u;
            x[2 * h] = pg_f16_of<TYPE>(__builtin_amdgcn_perm(0u, w, 0x0C010C00u));
            x[2 * h + 1] = pg_f16_of<TYPE>(__builtin_amdgcn_perm(0u, w, 0x0C030C02u));
        }
    } else {
        const uint32_t even = k[s] & 0x0F0F0F0Fu, odd = (k[s] >> 4) & 0x0F0F0F0Fu;
        x[0] = pg_f16_of<TYPE>(__builtin_amdgcn_perm(odd, even, 0x0C040C00u));
        x[1] = pg_f16_of<TYPE>(__builtin_amdgcn_perm(odd, even, 0x0C050C01u));
        x[2] = pg_f16_of<TYPE>(__builtin_amdgcn_perm(odd, even, 0x0C060C02u));
        x[3] = pg_f16_of<TYPE>(__builtin_amdgcn_perm(odd, even, 0x0C070C03u));
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

template <int TYPE, int D, int RT, int P>
__global__ __launch_bounds__(256, 2) void k_paged_attn(PgAttn a) {
    using R = PgRow<TYPE, D>;
    constexpr int NB = D / 32, T = D / 16, ROWS = 16 / P, KPL = P == 4 ? 4 : 8;
    constexpr bool QUANT = TYPE != AMV_T_F16;
    static_assert(P == 1 || RT == 1, "rows that share a product's columns are one tile");
    __shared__ float so[4][4][T][64];  // a row tile's O^T of the four waves, [wave][register][product][lane]
    __shared__ float sm[4][16 * RT], sl[4][16 * RT];
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    // what column c of the products is: row `col` of its tile, rounded (part 0) or the rest (part 1); u: whose keys it keeps
    const int u = P == 4 ? c >> 3 : 0;
    const bool rest = P == 4 ? (c & 4) != 0 : P == 2 && c >= 8;
    const int col = P == 4 ? (rest ? 3 - (c & 3) : c & 3) : P == 2 ? (rest ? 15 - c : c) : c;
    const float part = rest ? 1.0f : 0.0f;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hk = (int)blockIdx.x % a.n_head_kv, tile = (int)blockIdx.x / a.n_head_kv, z = blockIdx.y;
    const int psh = a.b.pshift, ps = 1 << psh;

    // the tile's rows: rows r0 .. of the n_rows of tokens tok0 .., row r is head r % G of token tok0 + r / G, whose place is
    // place0 + r / G; keys: how many there are to see
    int tok0, r0, n_rows, place0, keys;
    const int32_t* pages;  // the physical pages, or the sequence's table where `list` says which
    const int32_t* list = nullptr;
    int64_t part0 = -1;  // PG_ONE: where the rows of the sequence are in ml
    if (a.kind == PG_PREFIX) {
        tok0 = 0;
        r0 = tile * ROWS * RT;
        n_rows = a.b.n_tok * a.G;
        keys = a.n_list;
        place0 = keys;  // (every row sees them all)
        pages = a.list;
    } else {
        int s, in;
        if (a.kind == PG_LIST) {
            tok0 = tile / a.ta;
            in = tile % a.ta;
            s = pg_seq_of(a.b, tok0);
        } else if (a.kind == PG_ONE) {
            s = tile / a.ta;
            in = tile % a.ta;
        } else {
            pg_find(a.b.n_seq, tile, [&](int q) {
                const int r = (a.b.last(q) - a.b.first(q)) * a.G;
                return r > a.rows_most ? (r + ROWS * RT - 1) / (ROWS * RT) : 0;
            }, s, in);
        }
        if (s >= a.b.n_seq) return;
        const int first = a.b.first(s), n_q = a.b.last(s) - first;
        place0 = a.b.end(s) - n_q;
        keys = a.b.keys(s);
        pages = a.b.table + s * a.b.table_stride;
        if (a.kind == PG_LIST) {
            place0 += tok0 - first;
            n_rows = a.G;
            list = a.list + ((int64_t)tok0 * a.n_head_kv + hk) * a.n_list;
        } else {
            tok0 = first;
            n_rows = n_q * a.G;
            if (a.kind == PG_ONE && n_rows > a.rows_most) return;
            if (a.kind == PG_ONE) part0 = ((int64_t)s * a.n_head_kv + hk) * a.rows_most;
            if (a.kind == PG_FIND) in = (n_rows + ROWS * RT - 1) / (ROWS * RT) - 1 - in;  // the rows with the most keys first
        }
        r0 = in * ROWS * RT;
        if (r0 >= n_rows) return;
    }
    const int r_last = min(r0 + ROWS * RT, n_rows) - 1;
    // keys that every row of the tile sees, and the last that any does
    int see_all = keys, see_any = keys;
    if (a.kind != PG_PREFIX) {
        see_all = min(keys, place0 + r0 / a.G + 1);
        see_any = min(keys, place0 + r_last / a.G + 1);
    }
    // the walk: 32-key tiles i = begin + w, begin + w + 4, ... of the keys (of the listed pages' keys)
    int walk = see_any;
    if (list) {
        walk = 0;
        for (int i = lane; i < (a.n_list + 63) / 64 * 64; i += 64) {
            const uint64_t m = __builtin_amdgcn_ballot_w64(i < a.n_list && list[min(i, a.n_list - 1)] >= 0);
            if (m) walk = ((i - lane) + 64 - __builtin_clzll(m)) << psh;
        }
        walk = __builtin_amdgcn_readfirstlane(walk);
    }
    const int end = (min(walk, (z + 1) * a.split_len) + 31) >> 5;
    int i = (z * a.split_len >> 5) + w;

    const auto where = [&](int i) {  // i: uniform over the wave
        PgAt at;
        if (list) {
            const int j0 = i * 32 >> psh, j1 = min(i * 32 + 16, walk - 1) >> psh, off = (i * 32) & (ps - 1);
            const int l0 = list[j0], l1 = list[j1], most = (a.b.max_kv - 1) >> psh;
            at.e0 = l0 >= 0 && l0 <= most ? pages[l0] : -1;
            at.e1 = i * 32 + 16 < walk && l1 >= 0 && l1 <= most ? pages[l1] : -1;
            at.p0 = (l0 << psh) + off;
            at.p1 = psh == 4 ? l1 << psh : at.p0 + 16;
        } else {
            at.p0 = i * 32;
            at.p1 = at.p0 + 16;
            at.e0 = pages[at.p0 >> psh];
            at.e1 = at.p1 < keys ? pages[at.p1 >> psh] : -1;
        }
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
    // them would not be 0, so there each column picks its product). f: 2^e (for quantized keys times the 2^10 that their operands
    // lack); lim: keys the row sees
    pg_h8 qa[RT][P == 2 || (P == 4 && !QUANT) ? 1 : 2][NB];
    float f[RT];
    int lim[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = min(r0 + 16 * rt + col, r_last), t = r / a.G;
        lim[rt] = a.kind == PG_PREFIX ? keys : min(keys, place0 + t + 1);
        const float* src = a.q + (tok0 + t) * a.q_stride + (int64_t)(hk * a.G + r - t * a.G) * D + 8 * g;
        float x[NB][8], am = 0.0f;
#pragma unroll
        for (int s = 0; s < NB; ++s) {
            const float4 y = *reinterpret_cast<const float4*>(src + 32 * s), z = *reinterpret_cast<const float4*>(src + 32 * s + 4);
            const float yz[8] = {y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[s][j] = yz[j] * a.scale2;
                am = fmaxf(am, fabsf(x[s][j]));
            }
        }
        am = amv_max_x32(amv_max_x16(am));
        const uint32_t e = max(1u, min(253u, __float_as_uint(am) >> 23));
        const float down = __uint_as_float((254u - e) << 23);
        f[rt] = __uint_as_float(e << 23);
#pragma unroll
        for (int s = 0; s < NB; ++s) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[s][j] *= down;
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
        }
        if constexpr (QUANT) f[rt] *= 1024.0f;
    }

    float m[RT], l[RT];
    pg_f4 o[RT][T];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY;
        l[rt] = 0.0f;
#pragma unroll
        for (int t = 0; t < T; ++t) o[rt][t] = pg_f4{0.0f, 0.0f, 0.0f, 0.0f};
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
                    for (int h = 0; h < X; ++h) x[rt][h] = pg_f4{0.0f, 0.0f, 0.0f, 0.0f};
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const pg_h8 kf = pg_k_operand<TYPE, D>(tk.k[h], b);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    if constexpr (P == 4 && QUANT) {
                        x[rt][0] = pg_mfma(kf, qa[rt][h][b], x[rt][0]);
                    } else {
                        if constexpr (P == 1) x[rt][h] = pg_mfma(kf, qa[rt][1][b], x[rt][h]);
                        x[rt][h] = pg_mfma(kf, qa[rt][0][b], x[rt][h]);
                    }
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
        const bool some = now.e0 < 0 || now.e1 < 0 || max(now.p0, now.p1) + 16 > see_all;
        if (some) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int j = 0; j < KPL; ++j) s[rt][j] = there && p + 4 * u + j < lim[rt] ? s[rt][j] : -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) {  // what lies there must not matter, 0 times infinity is no number
                const uint32_t keep = there && p + j < keys ? 0xFFFFFFFFu : 0u;
#pragma unroll
                for (int x = 0; x < PgV<TYPE, D, KPL>::W; ++x) tv.v[j][x] &= keep;
            }
            if constexpr (QUANT) {
#pragma unroll
                for (int j = 0; j < KPL; ++j) {
                    const uint32_t keep = there && p + 4 * u + j < keys ? 0xFFFFFFFFu : 0u;
#pragma unroll
                    for (int b = 0; b < NB; b += 2) tv.s[(j * NB + b) >> 1] &= keep;
                }
            }
        }
        if constexpr (QUANT) {  // the values' largest scale
            amv_h2 big = {(_Float16)0.0f, (_Float16)0.0f};
#pragma unroll
            for (int x = 0; x < KPL * NB / 2; ++x)
                big = __builtin_elementwise_max(big, __builtin_bit_cast(amv_h2, tv.s[x] & 0x7FFF7FFFu));
            float top = amv_max_x32(amv_max_x16(fmaxf((float)big.x, (float)big.y)));
            if constexpr (P == 4) top = fmaxf(top, pg_dpp<PG_ROR8>(top));
            if (__builtin_amdgcn_readfirstlane(top > vref)) {
                const uint32_t e = min(253u, (__float_as_uint(top) >> 23) + 1u);
                const float up = __uint_as_float(e << 23), by = vref * __uint_as_float((254u - e) << 23);
                vref = up;
                vdown = __uint_as_float((254u - e) << 23);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int t = 0; t < T; ++t) o[rt][t] *= by;
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
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float mx = s[rt][0];
#pragma unroll
            for (int j = 1; j < KPL; ++j) mx = fmaxf(mx, s[rt][j]);
            if constexpr (P == 4) mx = fmaxf(mx, pg_dpp<PG_ROR8>(mx));
            mx = amv_max_x32(amv_max_x16(mx)) * f[rt];  // (f a power of two: exact)
            // the reference moves when a weight would pass 2^15 (or there is none yet), to 2^-12 of the maximum; where no difference
            // of 12 is exact, to the maximum
            const bool grow = mx > m[rt] + 15.0f;
            if (__builtin_amdgcn_ballot_w64(grow)) {
                const float to = fabsf(mx) > 0x1p20f ? mx : mx - 12.0f;
                const float alpha = grow ? __builtin_amdgcn_exp2f(m[rt] - to) : 1.0f;
                if (grow) m[rt] = to;
                l[rt] *= alpha;
#pragma unroll
                for (int t = 0; t < T; ++t) o[rt][t] *= alpha;
            }
            const float ref = m[rt] == -INFINITY ? 0.0f : m[rt];
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < KPL; ++j) {
                pw[rt][j] = __builtin_amdgcn_exp2f(fmaf(s[rt][j], f[rt], -ref));
                sum += pw[rt][j];
            }
            l[rt] += sum;
            if constexpr (QUANT) {
#pragma unroll
                for (int j = 0; j < KPL; ++j) pw[rt][j] *= vdown;
            } else {
                operand(rt, pw[rt]);
            }
        }
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const pg_h8 vf = pg_v_operand<TYPE, D>(tv, t);
            if constexpr (QUANT) {
                if ((t & 1) == 0) {  // products 2 b and 2 b + 1 are block b
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        float y[KPL];
#pragma unroll
                        for (int j = 0; j < KPL; ++j) {
                            y[j] = pw[rt][j] * pg_half(tv.s, j * NB + (t >> 1));
                            // The compiler would round the unrounded product to f16 (v_fma_mixlo_f16) but take the rest from the
                            // f16 of the rounded one; where the two differ, next to a tie, the parts do not sum to y.
                            asm("" : "+v"(y[j]));
                        }
                        operand(rt, y);
                    }
                }
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                if constexpr (P == 1) o[rt][t] = pg_mfma(vf, pl[rt], o[rt][t]);
                o[rt][t] = pg_mfma(vf, ph[rt], o[rt][t]);
            }
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
            for (int t = 0; t < T; ++t) {
                float y = o[rt][t][r];
                if constexpr (P == 2) y += pg_dpp<PG_MIRROR>(y);  // (lanes of part 0 end with their row's)
                if constexpr (P == 4) y += pg_dpp<PG_HALF_MIRROR>(y);
                so[w][r][t][lane] = y * back;
            }
        __syncthreads();
        const int r = r0 + 16 * rt + c;
        float M = -INFINITY, L = 0.0f, x[T];
#pragma unroll
        for (int j = 0; j < 4; ++j) M = fmaxf(M, sm[j][16 * rt + c]);
#pragma unroll
        for (int t = 0; t < T; ++t) x[t] = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float mj = sm[j][16 * rt + c], by = mj == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mj - M);
            L = fmaf(sl[j][16 * rt + c], by, L);
#pragma unroll
            for (int t = 0; t < T; ++t) x[t] = fmaf(so[j][w][t][lane], by, x[t]);
        }
        if (r < n_rows && c < ROWS) {
            const int tr = r / a.G;
            const int64_t row = (int64_t)(tok0 + tr) * a.n_head + hk * a.G + (r - tr * a.G);
            float* to = a.out + row * D;
            if (!a.ml) {
                const float inv = L > 0.0f ? 1.0f / L : L;  // (no keys: 0; a weight that is no number stays one)
#pragma unroll
                for (int t = 0; t < T; ++t) x[t] *= inv;
            } else {
                const int64_t part = (part0 >= 0 ? part0 + r : row) * a.n_split + z;
                to = a.acc + part * D;
                if (w == 0 && g == 0) a.ml[part] = make_float2(M, L);
            }
            const int d = 4 * g + w;  // the operand row
            if constexpr (QUANT) {
#pragma unroll
                for (int t = 0; t < T; t += 2)
                    *reinterpret_cast<float2*>(to + 16 * t + 2 * d) = make_float2(x[t], x[t + 1]);
            } else {
#pragma unroll
                for (int t = 0; t < T; t += 4)
                    *reinterpret_cast<float4*>(to + T * d + t) = make_float4(x[t], x[t + 1], x[t + 2], x[t + 3]);
            }
        }
    }
}

// out = sum_z w_z O_z / sum_z w_z l_z over the parts z of a row's keys, w_z = 2^(m_z - max m): one wave per row. A row has parts of
// its own keys, laid out by sequence where that has at most rows_most rows and else by row, and of the prefix.
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
};
template <int D>
__global__ __launch_bounds__(256) void k_paged_merge(PgMerge a) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tok = (int)(row / a.n_head), h = (int)(row - (int64_t)tok * a.n_head);
    if (tok >= a.b.n_tok) return;
    const int s = pg_seq_of(a.b, tok);
    if (s >= a.b.n_seq) return;
    const int first = a.b.first(s);
    const bool few = (a.b.last(s) - first) * a.G <= a.rows_most;
    const PgParts own = few ? a.one : a.many;
    if (!own.n) return;  // its workgroup wrote the row
    const int64_t own_row = few ? ((int64_t)s * a.n_head_kv + h / a.G) * a.rows_most + (tok - first) * a.G + h % a.G : row;
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
            for (int j0 = 0; j0 < n_here; j0 += 8) {
                float y[8][E];
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int e = 0; e < E; ++e) y[j][e] = acc[(int64_t)(z0 + min(j0 + j, n_here - 1)) * D + E * lane + e];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float by = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wz), min(j0 + j, 63)));
#pragma unroll
                    for (int e = 0; e < E; ++e) x[e] = j0 + j < n_here ? fmaf(by, y[j][e], x[e]) : x[e];
                }
            }
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
// Row tiles of a launch: rt times 16 rows, or 16 / pack of them where rows are few: the products' 16 columns then hold the two f16 of
// every row side by side, and with pack 4 the two products' keys too, so that each lane's scores are of use to half the lanes
// rather than an eighth.
struct PgTiles {
    int rt, pack;
    int rows() const { return 16 * rt / pack; }
    int of(int64_t n) const { return (int)((n + rows() - 1) / rows()); }
};
static PgTiles pg_tiles(int64_t rows) { return {rows > 16 ? 2 : 1, rows <= 4 ? 4 : rows <= 8 ? 2 : 1}; }
// How a call is launched: up to two launches over the sequences' own keys and one over the prefix, and the workspace of the parts.
struct PgPlan {
    PgTiles one, pre;                       // sequences (or listed tokens) of few rows, ta tiles each; the prefix's
    int ta, n_one, len_one;                 // their parts
    int find, rows_most, n_find, len_find;  // sequences of more rows than rows_most, tiles of 32
    int64_t find_tiles;
    int n_pre, len_pre;                     // parts of the prefix
    int64_t w_one, w_many, w_pre;           // parts in the workspace
    int64_t bytes(int64_t D) const { return (w_one + w_many + w_pre) * (8 + 4 * D); }
};
// parts of `keys` keys for `units` workgroups' worth of rows: two workgroups a CU, none of less than 128 keys (a tile for each of its
// waves). More and shorter parts cost their prologues and the merge (us at 512 / 1024 / 2048 workgroups: 64 sequences of up to 4096
// f16 keys 136 / 147 / 144, 3 of 65536 Q8_0 keys 78 / 78 / 82, one of 777 with parts of 256 keys 9.6, of 128 9.3)
static int pg_parts(int64_t units, int64_t keys, int* len) {
    units = std::max<int64_t>(1, units);
    const int64_t n = std::max<int64_t>(1, std::min<int64_t>(512 / units, (keys + 127) / 128));
    int64_t l = ((keys + n - 1) / n + 127) / 128 * 128;
    l = std::max<int64_t>(128, l);
    *len = (int)l;
    return (int)std::max<int64_t>(1, (keys + l - 1) / l);
}
static PgPlan pg_plan(const amv_paged_kv* kv, const amv_paged_batch* b, int64_t n_head, int64_t n_prefix, int64_t n_sel) {
    PgPlan p = {};
    const int64_t G = n_head / kv->n_head_kv;
    if (n_sel > 0) {
        p.one = pg_tiles(G);
        p.ta = p.one.of(G);
        p.n_one = pg_parts(b->n_tok * kv->n_head_kv * p.ta, n_sel * kv->page_size, &p.len_one);
        if (p.n_one > 1) p.w_many = b->n_tok * n_head * p.n_one;
        return p;
    }
    const int64_t rows = std::min(b->max_q, b->n_tok) * G;
    p.one = pg_tiles(rows <= 32 ? rows : G);
    p.rows_most = (int)std::max<int64_t>(p.one.rows(), G);
    p.ta = p.one.of(p.rows_most);
    p.n_one = pg_parts(b->n_seq * kv->n_head_kv * p.ta, b->max_kv, &p.len_one);
    p.find = rows > p.rows_most;
    if (p.find) {
        p.find_tiles = b->n_tok * G / 32 + b->n_seq;
        p.n_find = pg_parts(b->n_tok * G / 32 * kv->n_head_kv + 1, b->max_kv, &p.len_find);
    }
    p.pre = pg_tiles(b->n_tok * G);
    if (n_prefix > 0) p.n_pre = pg_parts(p.pre.of(b->n_tok * G) * kv->n_head_kv, n_prefix, &p.len_pre);
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

template <int TYPE, int D>
static void pg_launch(const PgAttn& a, PgTiles t, int64_t tiles, int parts, hipStream_t st) {
    const dim3 grid((unsigned)(tiles * a.n_head_kv), (unsigned)parts);
    if (t.pack == 4) hipLaunchKernelGGL((k_paged_attn<TYPE, D, 1, 4>), grid, dim3(256), 0, st, a);
    else if (t.pack == 2) hipLaunchKernelGGL((k_paged_attn<TYPE, D, 1, 2>), grid, dim3(256), 0, st, a);
    else if (t.rt == 1) hipLaunchKernelGGL((k_paged_attn<TYPE, D, 1, 1>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_paged_attn<TYPE, D, 2, 1>), grid, dim3(256), 0, st, a);
}
static void pg_launch(int type, int D, const PgAttn& a, PgTiles t, int64_t tiles, int parts, hipStream_t st) {
    if (D == 128) {
        if (type == AMV_T_F16) pg_launch<AMV_T_F16, 128>(a, t, tiles, parts, st);
        else if (type == AMV_T_Q8_0) pg_launch<AMV_T_Q8_0, 128>(a, t, tiles, parts, st);
        else pg_launch<AMV_T_Q4_0, 128>(a, t, tiles, parts, st);
    } else {
        if (type == AMV_T_F16) pg_launch<AMV_T_F16, 64>(a, t, tiles, parts, st);
        else if (type == AMV_T_Q8_0) pg_launch<AMV_T_Q8_0, 64>(a, t, tiles, parts, st);
        else pg_launch<AMV_T_Q4_0, 64>(a, t, tiles, parts, st);
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
                 out, (int)n_head, kv->n_head_kv, a.G, n_sel > 0 ? -1 : p.rows_most};
    const auto into = [&](const PgParts& parts) {
        a.ml = parts.n ? const_cast<float2*>(parts.ml) : nullptr;
        a.acc = const_cast<float*>(parts.acc);
    };
    hipStream_t st = amv_stream(stream);
    if (p.n_pre) {
        a.kind = PG_PREFIX;
        a.n_list = (int)n_prefix;
        a.n_split = p.n_pre;
        a.split_len = p.len_pre;
        into(m.pre);
        pg_launch(kv->type, kv->D, a, p.pre, p.pre.of(b->n_tok * a.G), p.n_pre, st);
    }
    if (p.find) {
        a.kind = PG_FIND;
        a.rows_most = p.rows_most;
        a.n_split = p.n_find;
        a.split_len = p.len_find;
        into(m.many);
        pg_launch(kv->type, kv->D, a, PgTiles{2, 1}, p.find_tiles, p.n_find, st);
    }
    a.kind = n_sel > 0 ? PG_LIST : PG_ONE;
    a.n_list = (int)n_sel;
    a.ta = p.ta;
    a.rows_most = p.rows_most;
    a.n_split = p.n_one;
    a.split_len = p.len_one;
    into(n_sel > 0 ? m.many : m.one);
    pg_launch(kv->type, kv->D, a, p.one, (n_sel > 0 ? b->n_tok : b->n_seq) * p.ta, p.n_one, st);
    if (p.w_one + p.w_many + p.w_pre) {
        const dim3 grid((unsigned)((rows + 3) / 4));
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
