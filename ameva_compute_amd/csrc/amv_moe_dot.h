// Dot products of weight rows with activation rows, lanes along k: a lane has a 32-element block, or a super-block's 16-byte slice, of two
// neighbouring weight rows, so that a load of a wave is one run of memory; 4 x 8-bit dot products, a block's or slice's integer exact.
#pragma once
#include "amv_moe.h"

struct MoAct {  // the activation rows of a call: integers; Q8_0: {d, sum} per block; Q8_K: d per super-block, sums per 16
    const int8_t* q;
    const int2* ds;
    const float* d;
    const int32_t* s16;
};

__device__ __forceinline__ int mo_dot16(const uint4& w, const int4& a, int s) {
    return amv_dot4((int)w.w, a.w, amv_dot4((int)w.z, a.z, amv_dot4((int)w.y, a.y, amv_dot4((int)w.x, a.x, s))));
}

// Per weight type: W, unit j (a block, or a slice of 32 elements) of rows n and n + 1 of the matrix at m; A, the same unit of the activation
// row; add: acc[r][i0 + i] += the product of rows n + i and a[r]. units: of a row.
template <int WT>
struct Mo;

template <>
struct Mo<AMV_T_Q4_0> {
    struct W {
        uint4 q[2];
        uint32_t d;  // both rows' scales
    };
    struct A {
        int4 lo, hi;
        int2 ds;
    };
    static __device__ __forceinline__ void load(W& w, const uint8_t* m, int rows, int units, int n, int j) {
        w.q[0] = amv_ld_stream(reinterpret_cast<const uint4*>(m + (uint32_t)(n * units + j) * 16u));
        w.q[1] = amv_ld_stream(reinterpret_cast<const uint4*>(m + (uint32_t)((n + 1) * units + j) * 16u));
        w.d = amv_ld_stream(reinterpret_cast<const uint32_t*>(m + (uint32_t)(rows * units) * 16u + (uint32_t)((n >> 1) * units + j) * 4u));
    }
    static __device__ __forceinline__ void load(A& a, const MoAct& act, int64_t row, int units, int j) {
        const int4* q = reinterpret_cast<const int4*>(act.q + row * units * 32);
        a.lo = q[2 * j];
        a.hi = q[2 * j + 1];
        a.ds = act.ds[row * units + j];
    }
    template <int C, int S>
    static __device__ __forceinline__ void add(const W& w, const A (&a)[C], int, float (&acc)[C][S], int i0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 q = w.q[i];
            const uint4 lo = make_uint4(q.x & 0x0F0F0F0Fu, q.y & 0x0F0F0F0Fu, q.z & 0x0F0F0F0Fu, q.w & 0x0F0F0F0Fu);
            const uint4 hi = make_uint4((q.x >> 4) & 0x0F0F0F0Fu, (q.y >> 4) & 0x0F0F0F0Fu, (q.z >> 4) & 0x0F0F0F0Fu, (q.w >> 4) & 0x0F0F0F0Fu);
            const float d = amv_h2f(i ? w.d >> 16 : w.d & 0xFFFFu);
#pragma unroll
            for (int r = 0; r < C; ++r) {
                const int s = mo_dot16(hi, a[r].hi, mo_dot16(lo, a[r].lo, -8 * a[r].ds.y));
                acc[r][i0 + i] = fmaf((float)s, d * __int_as_float(a[r].ds.x), acc[r][i0 + i]);
            }
        }
    }
};

template <>
struct Mo<AMV_T_Q8_0> {
    struct W {
        uint4 q[2][2];
        uint16_t d[2];
    };
    using A = Mo<AMV_T_Q4_0>::A;
    static __device__ __forceinline__ void load(W& w, const uint8_t* m, int rows, int units, int n, int j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            // (a block's two halves: lines that the wave touches twice, so not streamed)
            const uint4* q = reinterpret_cast<const uint4*>(m + (uint32_t)((n + i) * units + j) * 32u);
            w.q[i][0] = q[0];
            w.q[i][1] = q[1];
            w.d[i] = amv_ld_stream(reinterpret_cast<const uint16_t*>(m + (uint32_t)(rows * units) * 32u + (uint32_t)((n + i) * units + j) * 2u));
        }
    }
    static __device__ __forceinline__ void load(A& a, const MoAct& act, int64_t row, int units, int j) {
        Mo<AMV_T_Q4_0>::load(a, act, row, units, j);
    }
    template <int C, int S>
    static __device__ __forceinline__ void add(const W& w, const A (&a)[C], int, float (&acc)[C][S], int i0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float d = amv_h2f(w.d[i]);
#pragma unroll
            for (int r = 0; r < C; ++r) {
                const int s = mo_dot16(w.q[i][1], a[r].hi, mo_dot16(w.q[i][0], a[r].lo, 0));
                acc[r][i0 + i] = fmaf((float)s, d * __int_as_float(a[r].ds.x), acc[r][i0 + i]);
            }
        }
    }
};

struct MoAK {  // 16 + 16 activations of a slice, their sums, the super-block's scale
    int4 lo, hi;
    int slo, shi;
    float d;
};

// Q4_K: slice t of a super-block has the low nibbles of elements 64 (t / 2) + 16 (t % 2) .. and the high ones of those 32 further on: halves
// of units 2 (t / 2) and 2 (t / 2) + 1
template <>
struct Mo<AMV_T_Q4_K> {
    struct W {
        uint4 q[2];
        uint32_t h[2];  // a word of the super-block's head, lane % 4: the lanes of four have one super-block
    };
    using A = MoAK;
    static __device__ __forceinline__ void load(W& w, const uint8_t* m, int rows, int units, int n, int j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            w.q[i] = amv_ld_stream(reinterpret_cast<const uint4*>(m + (uint32_t)((n + i) * units + j) * 16u));
            w.h[i] = amv_ld_stream(reinterpret_cast<const uint32_t*>(m + (uint32_t)(rows * units) * 16u + (uint32_t)((n + i) * (units >> 3) + (j >> 3)) * 16u +
                                                                     4u * (threadIdx.x & 3)));
        }
    }
    static __device__ __forceinline__ void load(A& a, const MoAct& act, int64_t row, int units, int j) {
        const int64_t sb = row * (units >> 3) + (j >> 3);
        const int at = 4 * ((j & 7) >> 1) + (j & 1);
        a.lo = reinterpret_cast<const int4*>(act.q)[sb * 16 + at];
        a.hi = reinterpret_cast<const int4*>(act.q)[sb * 16 + at + 2];
        a.d = act.d[sb];
        a.slo = act.s16[sb * 16 + at];
        a.shi = act.s16[sb * 16 + at + 2];
    }
    template <int C, int S>
    static __device__ __forceinline__ void add(const W& w, const A (&a)[C], int j, float (&acc)[C][S], int i0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t h = w.h[i];
            const uint32_t x = amv_dpp_i<0x00>((int)h), y = amv_dpp_i<0x55>((int)h), z = amv_dpp_i<0xAA>((int)h), v = amv_dpp_i<0xFF>((int)h);
            int sl, ml, sh, mh;
            k4_scale_min_pair((j & 7) >> 1, y, z, v, sl, ml, sh, mh);
            const uint4 q = w.q[i];
            const uint4 lo = make_uint4(q.x & 0x0F0F0F0Fu, q.y & 0x0F0F0F0Fu, q.z & 0x0F0F0F0Fu, q.w & 0x0F0F0F0Fu);
            const uint4 hi = make_uint4((q.x >> 4) & 0x0F0F0F0Fu, (q.y >> 4) & 0x0F0F0F0Fu, (q.z >> 4) & 0x0F0F0F0Fu, (q.w >> 4) & 0x0F0F0F0Fu);
            const float d = amv_h2f(x & 0xFFFFu), dmin = amv_h2f(x >> 16);
#pragma unroll
            for (int r = 0; r < C; ++r) {
                const int s = sl * mo_dot16(lo, a[r].lo, 0) + sh * mo_dot16(hi, a[r].hi, 0), mins = ml * a[r].slo + mh * a[r].shi;
                acc[r][i0 + i] = fmaf(d * a[r].d, (float)s, acc[r][i0 + i]);
                acc[r][i0 + i] = fmaf(-(dmin * a[r].d), (float)mins, acc[r][i0 + i]);
            }
        }
    }
};

// Q6_K: slice t = 4 hh + r has the low nibbles of elements 128 hh + 16 r .. and the high ones of those 64 further on; their upper two bits are
// in 16 bytes of qh
template <>
struct Mo<AMV_T_Q6_K> {
    struct W {
        uint4 l[2], h[2];
        uint2 sc[2];  // the half's eight scales
        uint16_t d[2];
    };
    using A = MoAK;
    static __device__ __forceinline__ void load(W& w, const uint8_t* m, int rows, int units, int n, int j) {
        const uint32_t all = (uint32_t)rows * (units >> 3);  // super-blocks
        const int hh = (j & 7) >> 2, r = j & 3;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t sb = (uint32_t)(n + i) * (units >> 3) + (j >> 3);
            w.l[i] = amv_ld_stream(reinterpret_cast<const uint4*>(m + (uint32_t)((n + i) * units + j) * 16u));
            w.h[i] = *reinterpret_cast<const uint4*>(m + (all * 128u + sb * 64u + 32u * hh + 16u * (r & 1)));
            w.sc[i] = *reinterpret_cast<const uint2*>(m + (all * 192u + sb * 16u + 8u * hh));
            w.d[i] = *reinterpret_cast<const uint16_t*>(m + (all * 208u + sb * 2u));
        }
    }
    static __device__ __forceinline__ void load(A& a, const MoAct& act, int64_t row, int units, int j) {
        const int64_t sb = row * (units >> 3) + (j >> 3);
        const int at = 8 * ((j & 7) >> 2) + (j & 3);
        a.lo = reinterpret_cast<const int4*>(act.q)[sb * 16 + at];
        a.hi = reinterpret_cast<const int4*>(act.q)[sb * 16 + at + 4];
        a.d = act.d[sb];
        a.slo = act.s16[sb * 16 + at];
        a.shi = act.s16[sb * 16 + at + 4];
    }
    template <int C, int S>
    static __device__ __forceinline__ void add(const W& w, const A (&a)[C], int j, float (&acc)[C][S], int i0) {
        const int q = j & 3, lo = 2 * (q >> 1), hi = lo + 4;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 L = w.l[i], H = w.h[i];
            const auto q6 = [](uint32_t l, uint32_t h) { return (l & 0x0F0F0F0Fu) | ((h & 0x03030303u) << 4); };
            const uint4 vl = make_uint4(q6(L.x, H.x >> lo), q6(L.y, H.y >> lo), q6(L.z, H.z >> lo), q6(L.w, H.w >> lo));
            const uint4 vh = make_uint4(q6(L.x >> 4, H.x >> hi), q6(L.y >> 4, H.y >> hi), q6(L.z >> 4, H.z >> hi), q6(L.w >> 4, H.w >> hi));
            const int sl = (int)(int8_t)(w.sc[i].x >> (8 * q)), sh = (int)(int8_t)(w.sc[i].y >> (8 * q));
            const float d = amv_h2f(w.d[i]);
#pragma unroll
            for (int r = 0; r < C; ++r) {
                const int s = sl * (mo_dot16(vl, a[r].lo, -32 * a[r].slo)) + sh * (mo_dot16(vh, a[r].hi, -32 * a[r].shi));
                acc[r][i0 + i] = fmaf(d * a[r].d, (float)s, acc[r][i0 + i]);
            }
        }
    }
};
