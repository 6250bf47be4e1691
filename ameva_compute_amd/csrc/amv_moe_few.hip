// The experts' products with few rows each (decode steps, small batches): a tile is up to 16 rows (pairs) of one expert.
//
// One v_mfma_i32_16x16x64_i8 multiplies 16 A rows of 64 bytes with 16 weight rows. A lane of the weights holds 16 bytes of weight
// row l % 16, and quarter q = l / 16 of the wave holds block q of four: the 64-long contraction would add four blocks up, each of
// which has a scale of its own. So A row 4 t + b has token t's integers in the bytes of quarter b and zeros in the others: of four
// tokens and four blocks, each comes out as an integer of its own, exact. Weights go from memory to the lanes as they lie (16 bytes a lane),
// and one instruction in four would do for the arithmetic, but these products are bound by the weights' bytes.
// Result D of lane l: weight row l % 16, token l / 16, blocks 0..3 in its four registers: the block epilogue is a sum within the lane.
#include "amv_moe.h"

#include <algorithm>

typedef int mf_v4i __attribute__((ext_vector_type(4)));

__device__ __forceinline__ mf_v4i mf_mma(const uint4& a, const uint4& b, const mf_v4i& c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(mf_v4i{(int)a.x, (int)a.y, (int)a.z, (int)a.w},
                                                 mf_v4i{(int)b.x, (int)b.y, (int)b.z, (int)b.w}, c, 0, 0, 0);
}
__device__ __forceinline__ uint4 mf_each(const uint4& v, uint32_t (*f)(uint32_t)) { return make_uint4(f(v.x), f(v.y), f(v.z), f(v.w)); }
__device__ __forceinline__ uint32_t mf_m8(uint32_t v) { return (v + 0x78787878u) ^ 0x80808080u; }  // nibble - 8 per byte

// A wave's operands of one matrix and one step (four blocks of 32, or a super-block), and what one step adds to a row's sum.
// act row r: q + r * k integers, then the type's scales and sums.
struct MfAct {
    const int8_t* q;
    const float2* d0;     // Q8_0: {d, sum} per block
    const float* dk;      // Q8_K: d per super-block
    const int32_t* s16;   // Q8_K: sums per 16
};

template <int WT>
struct Mf;

template <int WT>
struct Mf32 {  // Q4_0, Q8_0
    static constexpr bool Q4 = WT == AMV_T_Q4_0;
    static constexpr int STEP = 4;  // blocks of 32
    struct W {
        uint4 q[Q4 ? 1 : 2];
        float d[4];
    };
    struct A {
        uint4 q[2];
        float d[4];
    };
    static __host__ __device__ int steps(int64_t k) { return (int)((k / 32 + 3) / 4); }
    // rows n of a matrix of `rows`; blocks past the end count nothing: their scales are 0, their integers another block's
    static __device__ __forceinline__ void load_w(W& w, const uint8_t* m, int rows, int nb, int n, int q, int s) {
        const int b = min(4 * s + q, nb - 1);
        const uint4* p = reinterpret_cast<const uint4*>(m + ((size_t)n * nb + b) * (Q4 ? 16 : 32));
        w.q[0] = p[0];
        if constexpr (!Q4) w.q[1] = p[1];
        const uint16_t* d = reinterpret_cast<const uint16_t*>(m + (size_t)rows * nb * (Q4 ? 16 : 32));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int bb = min(4 * s + i, nb - 1);
            const uint16_t h = Q4 ? d[((size_t)(n >> 1) * nb + bb) * 2 + (n & 1)] : d[(size_t)n * nb + bb];
            w.d[i] = 4 * s + i < nb ? amv_h2f(h) : 0.0f;
        }
    }
    static __device__ __forceinline__ void load_a(A& a, const MfAct& act, int64_t mine, int64_t row, int nb, bool diag, int q, int s) {
        const int b = min(4 * s + q, nb - 1);
        const uint4* p = reinterpret_cast<const uint4*>(act.q + (mine * nb + b) * 32);
        const uint4 z = make_uint4(0, 0, 0, 0);
        a.q[0] = diag ? p[0] : z;
        a.q[1] = diag ? p[1] : z;
#pragma unroll
        for (int i = 0; i < 4; ++i) a.d[i] = act.d0[row * nb + min(4 * s + i, nb - 1)].x;
    }
    static __device__ __forceinline__ float add(const W& w, const A& a, float acc) {
        mf_v4i c = {0, 0, 0, 0};
        if constexpr (Q4) {
            const uint4 x = w.q[0];
            c = mf_mma(a.q[0], mf_each(x, [](uint32_t v) { return mf_m8(v & 0x0F0F0F0Fu); }), c);
            c = mf_mma(a.q[1], mf_each(x, [](uint32_t v) { return mf_m8((v >> 4) & 0x0F0F0F0Fu); }), c);
        } else {
            c = mf_mma(a.q[0], w.q[0], c);
            c = mf_mma(a.q[1], w.q[1], c);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) acc = fmaf((float)c[i], w.d[i] * a.d[i], acc);
        return acc;
    }
};
template <>
struct Mf<AMV_T_Q4_0> : Mf32<AMV_T_Q4_0> {};
template <>
struct Mf<AMV_T_Q8_0> : Mf32<AMV_T_Q8_0> {};

// Q4_K: quarter q has the 32 bytes of units 2 q (low nibbles) and 2 q + 1 (high) of a super-block
template <>
struct Mf<AMV_T_Q4_K> {
    struct W {
        uint4 q[2];
        uint4 head;
    };
    struct A {
        uint4 q[4];
        int u[8];  // sums of the units
        float d;
    };
    static __host__ __device__ int steps(int64_t k) { return (int)(k / 256); }
    static __device__ __forceinline__ void load_w(W& w, const uint8_t* m, int rows, int nsb, int n, int q, int s) {
        const size_t sb = (size_t)n * nsb + s;
        const uint4* p = reinterpret_cast<const uint4*>(m) + sb * 8 + 2 * q;
        w.q[0] = p[0];
        w.q[1] = p[1];
        w.head = reinterpret_cast<const uint4*>(m)[(size_t)rows * nsb * 8 + sb];
    }
    static __device__ __forceinline__ void load_a(A& a, const MfAct& act, int64_t mine, int64_t row, int nsb, bool diag, int q, int s) {
        const uint4* p = reinterpret_cast<const uint4*>(act.q + (mine * nsb + s) * 256 + 64 * q);
        const uint4 z = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) a.q[i] = diag ? p[i] : z;
        const moe_i4* u = reinterpret_cast<const moe_i4*>(act.s16 + (row * nsb + s) * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const moe_i4 v = u[i];
            a.u[2 * i] = v.x + v.y;
            a.u[2 * i + 1] = v.z + v.w;
        }
        a.d = act.dk[row * nsb + s];
    }
    static __device__ __forceinline__ float add(const W& w, const A& a, float acc) {
        const mf_v4i z = {0, 0, 0, 0};
        mf_v4i lo = z, hi = z;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            lo = mf_mma(a.q[i], mf_each(w.q[i], [](uint32_t v) { return v & 0x0F0F0F0Fu; }), lo);
            hi = mf_mma(a.q[2 + i], mf_each(w.q[i], [](uint32_t v) { return (v >> 4) & 0x0F0F0F0Fu; }), hi);
        }
        // scales and mins of units 0-3 and 4-7, one per byte
        const uint32_t sc[2] = {w.head.y & 0x3F3F3F3Fu, (w.head.w & 0x0F0F0F0Fu) | ((w.head.y >> 2) & 0x30303030u)};
        const uint32_t mn[2] = {w.head.z & 0x3F3F3F3Fu, ((w.head.w >> 4) & 0x0F0F0F0Fu) | ((w.head.z >> 2) & 0x30303030u)};
        int I1 = 0, I2 = 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            I1 += __mul24(u & 1 ? hi[u >> 1] : lo[u >> 1], (int)((sc[u >> 2] >> (8 * (u & 3))) & 0xFF));
            I2 += __mul24(a.u[u], (int)((mn[u >> 2] >> (8 * (u & 3))) & 0xFF));
        }
        return fmaf(fmaf(amv_h2f(w.head.x), (float)I1, -(amv_h2f(w.head.x >> 16) * (float)I2)), a.d, acc);
    }
};

// Q6_K: quarter q = 2 h + p has elements 128 h + 16 p + {0, 32, 64, 96} .. + 15, four sub-blocks of 16
template <>
struct Mf<AMV_T_Q6_K> {
    struct W {
        uint4 l0, l1, h, sc;
        uint32_t d;
    };
    struct A {
        uint4 q[4];
        float d;
    };
    static __host__ __device__ int steps(int64_t k) { return (int)(k / 256); }
    static __device__ __forceinline__ void load_w(W& w, const uint8_t* m, int rows, int nsb, int n, int q, int s) {
        const size_t sb = (size_t)n * nsb + s, all = (size_t)rows * nsb;
        const uint4* l = reinterpret_cast<const uint4*>(m) + sb * 8 + 4 * (q >> 1) + (q & 1);
        w.l0 = l[0];
        w.l1 = l[2];
        w.h = reinterpret_cast<const uint4*>(m)[all * 8 + sb * 4 + q];
        w.sc = reinterpret_cast<const uint4*>(m)[all * 12 + sb];
        w.d = reinterpret_cast<const uint16_t*>(m + all * 208)[sb];
    }
    static __device__ __forceinline__ void load_a(A& a, const MfAct& act, int64_t mine, int64_t row, int nsb, bool diag, int q, int s) {
        const uint4* p = reinterpret_cast<const uint4*>(act.q + (mine * nsb + s) * 256 + 128 * (q >> 1) + 16 * (q & 1));
        const uint4 z = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) a.q[i] = diag ? p[2 * i] : z;
        a.d = act.dk[row * nsb + s];
    }
    static __device__ __forceinline__ float add(const W& w, const A& a, float acc) {
        const uint32_t L[2][4] = {{w.l0.x, w.l0.y, w.l0.z, w.l0.w}, {w.l1.x, w.l1.y, w.l1.z, w.l1.w}};
        const uint32_t H[4] = {w.h.x, w.h.y, w.h.z, w.h.w}, S[4] = {w.sc.x, w.sc.y, w.sc.z, w.sc.w};
        const mf_v4i z = {0, 0, 0, 0};
        int I = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // elements 32 e: low (e < 2) or high nibbles of l0 or l1, bits 2 e of h; minus 32
            uint32_t b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                b[i] = ((((L[e & 1][i] >> (e < 2 ? 0 : 4)) & 0x0F0F0F0Fu) | (((H[i] >> (2 * e)) & 0x03030303u) << 4)) + 0x60606060u) ^ 0x80808080u;
            const mf_v4i c = mf_mma(a.q[e], make_uint4(b[0], b[1], b[2], b[3]), z);
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // sub-block 8 (i / 2) + 2 e + i % 2
                const int sub = 8 * (i >> 1) + 2 * e + (i & 1);
                I += __mul24(c[i], (int)(int8_t)(S[sub >> 2] >> (8 * (sub & 3))));
            }
        }
        return fmaf(a.d * amv_h2f(w.d), (float)I, acc);
    }
};

// Workgroup: one tile of rows and, of each of its two matrices, 32 weight rows (gate and up; the down product's second matrix
// is the 32 rows after the first's), two waves of 16 weight rows on each quarter of k. The quarters' sums meet in LDS.
#define MF_KG 4
struct MfArgs {
    const uint8_t *w0, *w1;
    int64_t stride;
    int rows, n_k, n_expert, n_used, steps, n_tiles, act_div;
    MfAct act;
    const int32_t* ids;
    const int2* tiles;
    const int32_t* order;
    float* out;
    AmvActOut q;
};

template <int WT, bool GU, int G>
__global__ __launch_bounds__(128 * MF_KG) void k_moe_few(const MfArgs p) {
    __shared__ float s_red[MF_KG][2][4 * G][33];
    __shared__ int s_pair[4 * G];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nw = wv & 1, kw = wv >> 1, c16 = lane & 15, q = lane >> 4;
    int e, first, count;
    if (p.tiles) {
        const int2 tile = p.tiles[blockIdx.y];
        e = tile.x & 0xFFFF;
        count = tile.x >> 16;
        first = tile.y;
        if (!count) return;
    } else {
        e = p.ids[blockIdx.y];
        e = e >= 0 && e < p.n_expert ? e : p.n_expert;
        first = blockIdx.y;
        count = 1;
    }
    const int n0 = blockIdx.x * (GU ? 32 : 64);
    const auto pair = [&](int i) { return p.tiles ? p.order[first + min(i, count - 1)] : first; };
    float acc[2][G];
#pragma unroll
    for (int g = 0; g < G; ++g) acc[0][g] = acc[1][g] = 0.0f;
    if (tid < 4 * G) s_pair[tid] = pair(tid);
    if (e < p.n_expert) {
        const uint8_t* m0 = p.w0 + e * p.stride;
        const uint8_t* m1 = GU ? p.w1 + e * p.stride : m0;
        const int r0 = n0 + 16 * nw + c16, r1 = GU ? r0 : min(r0 + 32, p.rows - 1);
        const int n_g = (count + 3) >> 2;
        // the lane's tokens: of the integers (A row c16: token c16 / 4, block c16 % 4) and of the scales (token q)
        int64_t mine[G], row[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            mine[g] = pair(4 * g + (c16 >> 2)) / p.act_div;
            row[g] = pair(4 * g + q) / p.act_div;
        }
        const bool diag = (c16 & 3) == q;
        const int per = (p.steps + MF_KG - 1) / MF_KG, s_end = min(p.steps, (kw + 1) * per);
        for (int s = kw * per; s < s_end; ++s) {
            typename Mf<WT>::W w0, w1;
            Mf<WT>::load_w(w0, m0, p.rows, p.n_k, r0, q, s);
            Mf<WT>::load_w(w1, m1, p.rows, p.n_k, r1, q, s);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                if (g >= n_g) break;
                typename Mf<WT>::A a;
                Mf<WT>::load_a(a, p.act, mine[g], row[g], p.n_k, diag, q, s);
                acc[0][g] = Mf<WT>::add(w0, a, acc[0][g]);
                acc[1][g] = Mf<WT>::add(w1, a, acc[1][g]);
            }
        }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
        s_red[kw][0][4 * g + q][16 * nw + c16] = acc[0][g];
        s_red[kw][1][4 * g + q][16 * nw + c16] = acc[1][g];
    }
    __syncthreads();
    // thread: token i and column f of the 32 (a block of the 8-bit output is 32 lanes)
    for (int i = tid >> 5; i < count; i += 4 * MF_KG) {
        const int f = tid & 31;
        float v[2] = {0.0f, 0.0f};
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int z = 0; z < MF_KG; ++z) v[m] += s_red[z][m][i][f];
        const int64_t pr = s_pair[i];
        if constexpr (GU) {
            const float h = v[0] / (1.0f + expf(-v[0])) * v[1];
            if (p.out) p.out[pr * p.rows + n0 + f] = h;
            if (p.q.type) {
                const AmvActOut o = amv_act_row(p.q, pr, p.rows);
                int2* const meta = reinterpret_cast<int2*>(o.meta) + n0 / 32;
                amv_q8_0_lanes32(h, o.rule, f, o.qs + n0, meta);
                // (a scale that is none where an element is: moe_act_store4)
                const uint64_t bad = __ballot(!(fabsf(h) < INFINITY));
                if (f == 0 && (uint32_t)(bad >> (lane & 32))) meta->x = 0x7FC00000;
            }
        } else if (e < p.n_expert) {
            p.out[pr * p.rows + n0 + f] = v[0];
            if (n0 + 32 + f < p.rows) p.out[pr * p.rows + n0 + 32 + f] = v[1];
        }
    }
}

template <int WT, bool GU>
static void mf_go(const MfArgs& a, bool one, hipStream_t st) {
    const dim3 grid((unsigned)((a.rows + (GU ? 31 : 63)) / (GU ? 32 : 64)), (unsigned)a.n_tiles);
    if (one) k_moe_few<WT, GU, 1><<<grid, 128 * MF_KG, 0, st>>>(a);
    else k_moe_few<WT, GU, 4><<<grid, 128 * MF_KG, 0, st>>>(a);
}

int moe_few(const MoeProduct& p) {
    const int64_t pairs = p.n_tok * p.n_used;
    const MoePlanView v = moe_plan_view(p.plan, pairs, p.n_expert);
    const bool kq = p.type == AMV_T_Q4_K || p.type == AMV_T_Q6_K, gu = p.w1 != nullptr;
    const int8_t* aq = (const int8_t*)p.act;
    const int8_t* meta = aq + p.act_rows * p.k;
    MfArgs a{(const uint8_t*)p.w0, (const uint8_t*)p.w1, p.stride, (int)p.rows, (int)(p.k / (kq ? 256 : 32)), p.n_expert, p.n_used, 0,
             v.n_few, gu ? p.n_used : 1, {aq, (const float2*)meta, (const float*)meta, (const int32_t*)(meta + p.act_rows * (p.k / 64))},
             p.ids, v.few, v.order, p.out, p.q};
    a.steps = kq ? a.n_k : (a.n_k + 3) / 4;
    const int64_t all = a.n_tiles;
    for (int64_t t0 = 0; t0 < all; t0 += 65535) {
        a.n_tiles = (int)std::min<int64_t>(65535, all - t0);
        if (p.plan) a.tiles = v.few + t0;
        else AMV_REQUIRE(all <= 65535, "moe: %lld pairs without a plan", (long long)all);
        const bool one = !p.plan;
#define GO(T) (gu ? mf_go<T, true>(a, one, p.st) : mf_go<T, false>(a, one, p.st))
        if (p.type == AMV_T_Q4_0) GO(AMV_T_Q4_0);
        else if (p.type == AMV_T_Q8_0) GO(AMV_T_Q8_0);
        else if (p.type == AMV_T_Q4_K) GO(AMV_T_Q4_K);
        else GO(AMV_T_Q6_K);
#undef GO
    }
    return amv_check_launch("amv_moe products");
}
