// The experts' products of a token by itself (no plan): each pair is a product of one row. A wave has two neighbouring weight rows, its
// lanes the 32-element blocks (or a super-block's 16-byte slices) along them, so that a load of the wave is one run of memory;
// all loads of a step of 64 lanes, four weight rows, are on their way before the first product. (On the matrix core, with 16 weight rows a wave
// and 64 bytes of each a load, the same bytes take a third longer.)
// Gate and up: a workgroup has 32 columns of a pair, a wave two of them in both matrices. Down: a workgroup has a few columns of
// a token, its waves the token's experts, parts of a long k and columns, and adds the weighted products up: no second launch.
// Measured, with cold weights: two experts of 4096 x 14336 with their sum, Q6_K 18 us, 5.3 TB/s, Q8_0 28, Q4_0 13; gate and up of eight
// experts of 2048 x 4096 Q4_K 16 us, of 1024 x 2048 5.6, of which the bytes are 4.
#include "amv_moe.h"

#include <algorithm>

struct MoAct {  // the activation rows of a call: integers; Q8_0: {d, sum} per block; Q8_K: d per super-block, sums per 16
    const int8_t* q;
    const int2* ds;
    const float* d;
    const int32_t* s16;
};

// Per weight type: W, unit j (a block, or a slice of 32 elements) of rows n and n + 1 of the matrix at m; A, the same unit of the activation
// row; add: acc[i] += their product for row n + i. units: of a row.
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
    static __device__ __forceinline__ void add(const W& w, const A& a, int, float (&acc)[2]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 q = w.q[i];
            int s = -8 * a.ds.y;
            s = amv_dot4((int)(q.x & 0x0F0F0F0Fu), a.lo.x, s);
            s = amv_dot4((int)(q.y & 0x0F0F0F0Fu), a.lo.y, s);
            s = amv_dot4((int)(q.z & 0x0F0F0F0Fu), a.lo.z, s);
            s = amv_dot4((int)(q.w & 0x0F0F0F0Fu), a.lo.w, s);
            s = amv_dot4((int)((q.x >> 4) & 0x0F0F0F0Fu), a.hi.x, s);
            s = amv_dot4((int)((q.y >> 4) & 0x0F0F0F0Fu), a.hi.y, s);
            s = amv_dot4((int)((q.z >> 4) & 0x0F0F0F0Fu), a.hi.z, s);
            s = amv_dot4((int)((q.w >> 4) & 0x0F0F0F0Fu), a.hi.w, s);
            acc[i] = fmaf((float)s, amv_h2f(i ? w.d >> 16 : w.d & 0xFFFFu) * __int_as_float(a.ds.x), acc[i]);
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
    static __device__ __forceinline__ void add(const W& w, const A& a, int, float (&acc)[2]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 p = w.q[i][0], q = w.q[i][1];
            int s = amv_dot4((int)p.x, a.lo.x, 0);
            s = amv_dot4((int)p.y, a.lo.y, s);
            s = amv_dot4((int)p.z, a.lo.z, s);
            s = amv_dot4((int)p.w, a.lo.w, s);
            s = amv_dot4((int)q.x, a.hi.x, s);
            s = amv_dot4((int)q.y, a.hi.y, s);
            s = amv_dot4((int)q.z, a.hi.z, s);
            s = amv_dot4((int)q.w, a.hi.w, s);
            acc[i] = fmaf((float)s, amv_h2f(w.d[i]) * __int_as_float(a.ds.x), acc[i]);
        }
    }
};

__device__ __forceinline__ int mo_dot16(const uint4& w, const int4& a) {
    return amv_dot4((int)w.w, a.w, amv_dot4((int)w.z, a.z, amv_dot4((int)w.y, a.y, amv_dot4((int)w.x, a.x, 0))));
}
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
    static __device__ __forceinline__ void add(const W& w, const A& a, int j, float (&acc)[2]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t h = w.h[i];
            const uint32_t x = amv_dpp_i<0x00>((int)h), y = amv_dpp_i<0x55>((int)h), z = amv_dpp_i<0xAA>((int)h), v = amv_dpp_i<0xFF>((int)h);
            int sl, ml, sh, mh;
            k4_scale_min_pair((j & 7) >> 1, y, z, v, sl, ml, sh, mh);
            const uint4 q = w.q[i];
            const uint4 lo = make_uint4(q.x & 0x0F0F0F0Fu, q.y & 0x0F0F0F0Fu, q.z & 0x0F0F0F0Fu, q.w & 0x0F0F0F0Fu);
            const uint4 hi = make_uint4((q.x >> 4) & 0x0F0F0F0Fu, (q.y >> 4) & 0x0F0F0F0Fu, (q.z >> 4) & 0x0F0F0F0Fu, (q.w >> 4) & 0x0F0F0F0Fu);
            const int s = sl * mo_dot16(lo, a.lo) + sh * mo_dot16(hi, a.hi), mins = ml * a.slo + mh * a.shi;
            acc[i] = fmaf(amv_h2f(x & 0xFFFFu) * a.d, (float)s, acc[i]);
            acc[i] = fmaf(-(amv_h2f(x >> 16) * a.d), (float)mins, acc[i]);
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
    static __device__ __forceinline__ void add(const W& w, const A& a, int j, float (&acc)[2]) {
        const int r = j & 3, lo = 2 * (r >> 1), hi = lo + 4;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 L = w.l[i], H = w.h[i];
            const auto q6 = [](uint32_t l, uint32_t h) { return (l & 0x0F0F0F0Fu) | ((h & 0x03030303u) << 4); };
            const uint4 vl = make_uint4(q6(L.x, H.x >> lo), q6(L.y, H.y >> lo), q6(L.z, H.z >> lo), q6(L.w, H.w >> lo));
            const uint4 vh = make_uint4(q6(L.x >> 4, H.x >> hi), q6(L.y >> 4, H.y >> hi), q6(L.z >> 4, H.z >> hi), q6(L.w >> 4, H.w >> hi));
            const int sl = (int)(int8_t)(w.sc[i].x >> (8 * r)), sh = (int)(int8_t)(w.sc[i].y >> (8 * r));
            const int s = sl * (mo_dot16(vl, a.lo) - 32 * a.slo) + sh * (mo_dot16(vh, a.hi) - 32 * a.shi);
            acc[i] = fmaf(amv_h2f(w.d[i]) * a.d, (float)s, acc[i]);
        }
    }
};

// rows n[i] and n[i] + 1 of matrix m[i], M times, times activation row `row`, part of parts of k. All loads of a step before its products;
// the loads of a second step beside them were slower (two experts of 4096 x 14336 Q4_0 14 us, so 13; 32 rows of 2048 x 4096 Q6_K 24, so 22).
template <int WT, int M>
__device__ __forceinline__ void mo_rows(const uint8_t* const (&m)[M], int rows, int units, const int (&n)[M], const MoAct& act, int64_t row, int part,
                                        int parts, float (&acc)[M][2]) {
    using T = Mo<WT>;
    const int lane = threadIdx.x & 63;
    for (int s = 64 * part; s < units; s += 64 * parts) {
        typename T::W w[M];
        typename T::A a;
        const int j = min(s + lane, units - 1);
#pragma unroll
        for (int i = 0; i < M; ++i) T::load(w[i], m[i], rows, units, n[i], j);
        T::load(a, act, row, units, j);
        __builtin_amdgcn_sched_barrier(0);
        if (s + lane < units)
#pragma unroll
            for (int i = 0; i < M; ++i) T::add(w[i], a, j, acc[i]);
    }
#pragma unroll
    for (int i = 0; i < M; ++i) {
        acc[i][0] = amv_wave_sum(acc[i][0]);
        acc[i][1] = amv_wave_sum(acc[i][1]);
    }
}

#define MO_PAIRS 2  // pairs of columns of a wave of the down product

struct MoArgs {
    const uint8_t *w0, *w1;
    int64_t stride;
    int rows, units, n_expert, n_used, n_cols, groups, parts;
    MoAct act;
    const int32_t* ids;
    const float *weights, *add;
    float* out;
    AmvActOut q;
};

template <int WT>
__global__ __launch_bounds__(1024) void k_moe_one_gate_up(const MoArgs p) {
    __shared__ __align__(16) float s_red[16][4];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int pair = blockIdx.x / p.n_cols, n0 = 32 * (blockIdx.x % p.n_cols), e = p.ids[pair];
    float acc[2][2] = {};
    if (e >= 0 && e < p.n_expert) {
        const uint8_t* const m[2] = {p.w0 + e * p.stride, p.w1 + e * p.stride};
        const int n[2] = {n0 + 2 * wv, n0 + 2 * wv};
        mo_rows<WT, 2>(m, p.rows, p.units, n, p.act, pair / p.n_used, 0, 1, acc);
    }
    if (lane == 0) *reinterpret_cast<float4*>(s_red[wv]) = make_float4(acc[0][0], acc[0][1], acc[1][0], acc[1][1]);
    __syncthreads();
    if (tid >= 32) return;
    const float g = s_red[tid >> 1][tid & 1], u = s_red[tid >> 1][2 + (tid & 1)];
    const float h = g / (1.0f + expf(-g)) * u;
    if (p.out) p.out[(int64_t)pair * p.rows + n0 + tid] = h;
    if (p.q.type) {
        const AmvActOut o = amv_act_row(p.q, pair, p.rows);
        moe_q8_0(h, o.rule, tid, o.qs + n0, reinterpret_cast<int2*>(o.meta) + n0 / 32);
    }
}

template <int WT>
__global__ __launch_bounds__(1024) void k_moe_one_down(const MoArgs p) {
    constexpr int G = MO_PAIRS;
    __shared__ __align__(16) float s_red[MOE_MAX_USED][2 * G];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int t = blockIdx.x / p.n_cols, n0 = 2 * G * p.groups * (blockIdx.x % p.n_cols);
    // job: 2 G columns, expert, part (in turns where there are more than waves)
    for (int job = wv; job < p.groups * p.n_used * p.parts; job += blockDim.x >> 6) {
        const int part = job % p.parts, j = job / p.parts % p.n_used, c = n0 + 2 * G * (job / (p.parts * p.n_used));
        const int e = p.ids[t * p.n_used + j];
        float acc[G][2] = {};
        if (e >= 0 && e < p.n_expert) {
            const uint8_t* m[G];
            int n[G];
#pragma unroll
            for (int i = 0; i < G; ++i) {
                m[i] = p.w0 + e * p.stride;
                n[i] = min(c + 2 * i, p.rows - 2);
            }
            mo_rows<WT, G>(m, p.rows, p.units, n, p.act, (int64_t)t * p.n_used + j, part, p.parts, acc);
        }
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < G; ++i) *reinterpret_cast<float2*>(s_red[job] + 2 * i) = make_float2(acc[i][0], acc[i][1]);
    }
    __syncthreads();
    if (tid >= 2 * G * p.groups || n0 + tid >= p.rows) return;
    const int64_t at = (int64_t)t * p.rows + n0 + tid;
    float v = p.add ? p.add[at] : 0.0f;
    for (int j = 0; j < p.n_used; ++j) {
        const int e = p.ids[t * p.n_used + j];
        if (e < 0 || e >= p.n_expert) continue;
        float y = 0.0f;
        for (int z = 0; z < p.parts; ++z) y += s_red[(tid / (2 * G) * p.n_used + j) * p.parts + z][tid % (2 * G)];
        v = fmaf(p.weights[t * p.n_used + j], y, v);
    }
    p.out[at] = v;
}

template <int WT>
static void mo_go(MoArgs a, int64_t n, bool gu, hipStream_t st) {
    if (gu) {
        a.n_cols = a.rows / 32;
        k_moe_one_gate_up<WT><<<(unsigned)(n * a.n_cols), 1024, 0, st>>>(a);
        return;
    }
    // eight waves (a wave an expert where there are more): parts of k, as many as bring eight waves a CU, then columns. Sixteen were slower or equal
    // (two experts of 4096 x 14336 Q4_0 20 us, so 13), two columns a wave too (eight of 4096 x 2048 Q4_0 15, so 12); of one expert of 2048 x 8192
    // Q8_0 one part takes 9, two 7, four 6.
    const int room = std::max(1, 8 / a.n_used), steps = (a.units + 63) / 64;
    const int64_t waves = n * (a.rows / (2 * MO_PAIRS)) * a.n_used;
    a.parts = (int)std::min<int64_t>(std::min(room, steps), std::max<int64_t>(1, 2048 / waves));
    a.groups = std::max(1, room / a.parts);
    a.n_cols = (a.rows + 2 * MO_PAIRS * a.groups - 1) / (2 * MO_PAIRS * a.groups);
    k_moe_one_down<WT><<<(unsigned)(n * a.n_cols), 64 * std::min(16, a.n_used * a.parts * a.groups), 0, st>>>(a);
}

int moe_one(const MoeProduct& p) {
    const bool kq = p.type == AMV_T_Q4_K || p.type == AMV_T_Q6_K, gu = p.w1 != nullptr;
    const int8_t* aq = (const int8_t*)p.act;
    const int8_t* meta = aq + p.act_rows * p.k;
    const int64_t n = gu ? p.n_tok * p.n_used : p.n_tok;
    AMV_REQUIRE(p.n_tok * p.n_used * p.rows < 1 << 26, "moe: %lld pairs of %lld without a plan are too many", (long long)(p.n_tok * p.n_used),
                (long long)p.rows);
    const MoArgs a{(const uint8_t*)p.w0, (const uint8_t*)p.w1, p.stride, (int)p.rows, (int)(p.k / 32), p.n_expert, p.n_used, 0, 0, 0,
                   {aq, (const int2*)meta, (const float*)meta, kq ? (const int32_t*)(meta + p.act_rows * (p.k / 64)) : nullptr}, p.ids, p.weights,
                   p.add, p.out, p.q};
    if (p.type == AMV_T_Q4_0) mo_go<AMV_T_Q4_0>(a, n, gu, p.st);
    else if (p.type == AMV_T_Q8_0) mo_go<AMV_T_Q8_0>(a, n, gu, p.st);
    else if (p.type == AMV_T_Q4_K) mo_go<AMV_T_Q4_K>(a, n, gu, p.st);
    else mo_go<AMV_T_Q6_K>(a, n, gu, p.st);
    return amv_check_launch("amv_moe products");
}
