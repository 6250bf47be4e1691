// The experts' products with few rows each (decode steps, small batches): a tile is up to 16 rows (pairs) of one expert.
//
// One v_mfma_i32_16x16x64_i8 multiplies 16 A rows of 64 bytes with 16 weight rows. A lane of the weights holds 16 bytes of weight
// row l % 16, and quarter q = l / 16 of the wave holds block q of four: the 64-long contraction would add four blocks up, each of
// which has a scale of its own. So A row 4 t + b has token t's integers in the bytes of quarter b and zeros in the others: of four
// tokens and four blocks, each comes out as an integer of its own, exact. Weights go from memory to the lanes as they lie (16 bytes a
// lane), and one instruction in four would do for the arithmetic, but these products are bound by the weights' bytes.
// Result D of lane l: weight row l % 16, token l / 16, blocks 0..3 in its four registers: the block epilogue is a sum within the lane.
#include "amv_moe.h"

#include <algorithm>

typedef int mf_v4i __attribute__((ext_vector_type(4)));
typedef short mf_s2 __attribute__((ext_vector_type(2)));
// two or four 32-bit words at an address of any 16 or 32 bits
typedef uint32_t mf_u2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t mf_u4 __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ mf_v4i mf_mma(const uint4& a, const uint4& b, const mf_v4i& c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(mf_v4i{(int)a.x, (int)a.y, (int)a.z, (int)a.w},
                                                 mf_v4i{(int)b.x, (int)b.y, (int)b.z, (int)b.w}, c, 0, 0, 0);
}
template <typename F>
__device__ __forceinline__ uint4 mf_each(const uint4& v, F f) { return make_uint4(f(v.x), f(v.y), f(v.z), f(v.w)); }
__device__ __forceinline__ uint32_t mf_m8(uint32_t v) { return (v + 0x78787878u) ^ 0x80808080u; }  // nibble - 8 per byte
// register x of quarter j (lanes 16 j .. 16 j + 15) in every quarter, for the four j
__device__ __forceinline__ void mf_quarters(uint32_t x, uint32_t (&o)[4]) {
    const auto h = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    const auto a = __builtin_amdgcn_permlane16_swap(h[0], h[0], false, false), b = __builtin_amdgcn_permlane16_swap(h[1], h[1], false, false);
    o[0] = a[0];
    o[1] = a[1];
    o[2] = b[0];
    o[3] = b[1];
}

// the activation rows of a call: integers, and scales (Q8_0: {d, sum} per block; Q8_K: d per super-block) and sums per 16 (Q8_K)
struct MfAct {
    const int8_t* q;
    const float2* d0;
    const float* dk;
    const int32_t* s16;
};

// Per weight type: a step (STEP k) is four blocks of 32 or a super-block; U steps are loaded at once (struct W, one matrix). The
// activations come from LDS: rows of integers LD bytes apart, their scales at s (float [row][STEPS * 4 or 1]), unit sums at u.
template <int WT>
struct Mf32 {  // Q4_0, Q8_0
    static constexpr bool Q4 = WT == AMV_T_Q4_0;
    static constexpr int STEP = 128, U = Q4 ? 4 : 2, PER = 4;  // PER: scales of a row and step
    struct W {
        uint4 q[U][Q4 ? 1 : 2];
        uint2 d[Q4 ? 1 : U];  // four f16; Q4_0: quarter j of the wave holds step j's
    };
    // steps s .. of weight row n of a matrix of `rows`; blocks past the end: another block's integers, scales 0
    static __device__ __forceinline__ void load(W& w, const uint8_t* m, int rows, int nb, int n, int q, int s) {
        const uint8_t* const d = m + (size_t)rows * nb * (Q4 ? 16 : 32);
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const uint4* p = reinterpret_cast<const uint4*>(m + ((size_t)n * nb + min(4 * (s + j) + q, nb - 1)) * (Q4 ? 16 : 32));
            w.q[j][0] = p[0];
            if constexpr (!Q4) w.q[j][1] = p[1];
        }
        if constexpr (Q4) {
            // the scales of rows 2 p and 2 p + 1 side by side: lane quarter q takes blocks 4 (s + q) .. + 3, its own row's halves
            const uint32_t* p = reinterpret_cast<const uint32_t*>(d) + (size_t)(n >> 1) * nb;
            uint32_t x[4];
            if (4 * (s + 4) <= nb) {
                const mf_u4 v = *reinterpret_cast<const mf_u4*>(p + 4 * (s + q));
                x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = 4 * (s + q) + i < nb ? p[min(4 * (s + q) + i, nb - 1)] : 0u;
            }
            const uint32_t sel = n & 1 ? 0x07060302u : 0x05040100u;  // the upper or the lower halves of two words
            w.d[0] = make_uint2(__builtin_amdgcn_perm(x[1], x[0], sel), __builtin_amdgcn_perm(x[3], x[2], sel));
        } else {
            const uint16_t* p = reinterpret_cast<const uint16_t*>(d) + (size_t)n * nb;
#pragma unroll
            for (int j = 0; j < U; ++j) {
                if (4 * (s + j + 1) <= nb) {
                    const mf_u2 v = *reinterpret_cast<const mf_u2*>(p + 4 * (s + j));
                    w.d[j] = make_uint2(v.x, v.y);
                } else {
                    uint32_t x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = 4 * (s + j) + i < nb ? p[min(4 * (s + j) + i, nb - 1)] : 0u;
                    w.d[j] = make_uint2(x[0] | x[1] << 16, x[2] | x[3] << 16);
                }
            }
        }
    }
    // what the steps need of the weights alone, once for all tokens: operands and scales of step j
    struct B {
        uint4 q[2];
        float d[4];
    };
    struct Scales {
        uint32_t lo[4], hi[4];
    };
    static __device__ __forceinline__ void scales(const W& w, Scales& c) {
        if constexpr (Q4) {
            mf_quarters(w.d[0].x, c.lo);
            mf_quarters(w.d[0].y, c.hi);
        } else {
#pragma unroll
            for (int j = 0; j < U; ++j) {
                c.lo[j] = w.d[j].x;
                c.hi[j] = w.d[j].y;
            }
        }
    }
    static __device__ __forceinline__ void operands(const W& w, const Scales& c, int j, B& o) {
        if constexpr (Q4) {
            o.q[0] = mf_each(w.q[j][0], [](uint32_t v) { return mf_m8(v & 0x0F0F0F0Fu); });
            o.q[1] = mf_each(w.q[j][0], [](uint32_t v) { return mf_m8((v >> 4) & 0x0F0F0F0Fu); });
        } else {
            o.q[0] = w.q[j][0];
            o.q[1] = w.q[j][1];
        }
        o.d[0] = amv_h2f(c.lo[j]);
        o.d[1] = amv_h2f(c.lo[j] >> 16);
        o.d[2] = amv_h2f(c.hi[j]);
        o.d[3] = amv_h2f(c.hi[j] >> 16);
    }
    struct A {
        uint4 q[2];
        float4 d;
    };
    // a: the lane's integers of the step (or zeros, `on` 0), s: its token's scales of the step
    static __device__ __forceinline__ void read(A& a, const uint8_t* p, int on, int q, const float* s, const int16_t*) {
        const uint4* v = reinterpret_cast<const uint4*>(p + on * 32 * q);
        a.q[0] = v[0];
        a.q[1] = v[1];
        a.d = *reinterpret_cast<const float4*>(s);
    }
    static __device__ __forceinline__ float add(const B& w, const A& a, float acc) {
        mf_v4i c = {0, 0, 0, 0};
        c = mf_mma(a.q[0], w.q[0], c);
        c = mf_mma(a.q[1], w.q[1], c);
        acc = fmaf((float)c[0], w.d[0] * a.d.x, acc);
        acc = fmaf((float)c[1], w.d[1] * a.d.y, acc);
        acc = fmaf((float)c[2], w.d[2] * a.d.z, acc);
        return fmaf((float)c[3], w.d[3] * a.d.w, acc);
    }
};
template <int WT>
struct Mf : Mf32<WT> {};

// Q4_K: quarter q has the 32 bytes of units 2 q (low nibbles) and 2 q + 1 (high) of a super-block
template <>
struct Mf<AMV_T_Q4_K> {
    static constexpr int STEP = 256, U = 2, PER = 1;
    struct W {
        uint4 q[U][2], head[U];
    };
    static __device__ __forceinline__ void load(W& w, const uint8_t* m, int rows, int nsb, int n, int q, int s) {
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const size_t sb = (size_t)n * nsb + min(s + j, nsb - 1);
            const uint4* p = reinterpret_cast<const uint4*>(m) + sb * 8 + 2 * q;
            w.q[j][0] = p[0];
            w.q[j][1] = p[1];
            w.head[j] = reinterpret_cast<const uint4*>(m)[(size_t)rows * nsb * 8 + sb];
        }
    }
    struct B {
        uint4 lo[2], hi[2];
        int sc[8];
        mf_s2 mn[4];
        float d, dm;
    };
    struct Scales {};
    static __device__ __forceinline__ void scales(const W&, Scales&) {}
    static __device__ __forceinline__ void operands(const W& w, const Scales&, int j, B& o) {
        const uint4 h = w.head[j];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            o.lo[i] = mf_each(w.q[j][i], [](uint32_t v) { return v & 0x0F0F0F0Fu; });
            o.hi[i] = mf_each(w.q[j][i], [](uint32_t v) { return (v >> 4) & 0x0F0F0F0Fu; });
        }
        // scales and mins of units 0-3 and 4-7, one per byte
        const uint32_t sc[2] = {h.y & 0x3F3F3F3Fu, (h.w & 0x0F0F0F0Fu) | ((h.y >> 2) & 0x30303030u)};
        const uint32_t mn[2] = {h.z & 0x3F3F3F3Fu, ((h.w >> 4) & 0x0F0F0F0Fu) | ((h.z >> 2) & 0x30303030u)};
#pragma unroll
        for (int u = 0; u < 8; ++u) o.sc[u] = (int)((sc[u >> 2] >> (8 * (u & 3))) & 0xFF);
#pragma unroll
        for (int u = 0; u < 4; ++u)  // bytes 2 u, 2 u + 1 as two 16-bit numbers
            o.mn[u] = __builtin_bit_cast(mf_s2, __builtin_amdgcn_perm(0u, mn[u >> 1], u & 1 ? 0x0C030C02u : 0x0C010C00u));
        o.d = amv_h2f(h.x);
        o.dm = amv_h2f(h.x >> 16);
    }
    struct A {
        uint4 q[4], u;
        float d;
    };
    static __device__ __forceinline__ void read(A& a, const uint8_t* p, int on, int q, const float* s, const int16_t* u) {
        const uint4* v = reinterpret_cast<const uint4*>(p + on * 64 * q);
#pragma unroll
        for (int i = 0; i < 4; ++i) a.q[i] = v[on * i];
        a.u = *reinterpret_cast<const uint4*>(u);
        a.d = *s;
    }
    static __device__ __forceinline__ float add(const B& w, const A& a, float acc) {
        mf_v4i lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            lo = mf_mma(a.q[i], w.lo[i], lo);
            hi = mf_mma(a.q[2 + i], w.hi[i], hi);
        }
        const uint32_t us[4] = {a.u.x, a.u.y, a.u.z, a.u.w};
        int I1 = 0, I2 = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            I1 += __mul24(lo[u], w.sc[2 * u]);
            I1 += __mul24(hi[u], w.sc[2 * u + 1]);
            I2 = __builtin_amdgcn_sdot2(__builtin_bit_cast(mf_s2, us[u]), w.mn[u], I2, false);
        }
        return fmaf(fmaf(w.d, (float)I1, -(w.dm * (float)I2)), a.d, acc);
    }
};

// Q6_K: quarter q = 2 h + p has elements 128 h + 16 p + {0, 32, 64, 96} .. + 15, four sub-blocks of 16
template <>
struct Mf<AMV_T_Q6_K> {
    static constexpr int STEP = 256, U = 1, PER = 1;
    struct W {
        uint4 l0[U], l1[U], h[U], sc[U];
        uint32_t d[U];
    };
    static __device__ __forceinline__ void load(W& w, const uint8_t* m, int rows, int nsb, int n, int q, int s) {
        const size_t all = (size_t)rows * nsb;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const size_t sb = (size_t)n * nsb + min(s + j, nsb - 1);
            const uint4* l = reinterpret_cast<const uint4*>(m) + sb * 8 + 4 * (q >> 1) + (q & 1);
            w.l0[j] = l[0];
            w.l1[j] = l[2];
            w.h[j] = reinterpret_cast<const uint4*>(m)[all * 8 + sb * 4 + q];
            w.sc[j] = reinterpret_cast<const uint4*>(m)[all * 12 + sb];
            w.d[j] = reinterpret_cast<const uint16_t*>(m + all * 208)[sb];
        }
    }
    struct B {
        uint4 q[4], sc;
        float d;
    };
    struct Scales {};
    static __device__ __forceinline__ void scales(const W&, Scales&) {}
    static __device__ __forceinline__ void operands(const W& w, const Scales&, int j, B& o) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // elements 32 e: low (e < 2) or high nibbles of l0 or l1, bits 2 e of h; minus 32
            const uint4 l = e & 1 ? w.l1[j] : w.l0[j];
            const auto one = [&](uint32_t x, uint32_t y) {
                return ((((x >> (e < 2 ? 0 : 4)) & 0x0F0F0F0Fu) | (((y >> (2 * e)) & 0x03030303u) << 4)) + 0x60606060u) ^ 0x80808080u;
            };
            o.q[e] = make_uint4(one(l.x, w.h[j].x), one(l.y, w.h[j].y), one(l.z, w.h[j].z), one(l.w, w.h[j].w));
        }
        o.sc = w.sc[j];
        o.d = amv_h2f(w.d[j]);
    }
    struct A {
        uint4 q[4];
        float d;
    };
    static __device__ __forceinline__ void read(A& a, const uint8_t* p, int on, int q, const float* s, const int16_t*) {
        const uint4* v = reinterpret_cast<const uint4*>(p + on * (128 * (q >> 1) + 16 * (q & 1)));
#pragma unroll
        for (int i = 0; i < 4; ++i) a.q[i] = v[on * 2 * i];
        a.d = *s;
    }
    static __device__ __forceinline__ float add(const B& w, const A& a, float acc) {
        const uint32_t S[4] = {w.sc.x, w.sc.y, w.sc.z, w.sc.w};
        const mf_v4i z = {0, 0, 0, 0};
        int I = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const mf_v4i c = mf_mma(a.q[e], w.q[e], z);
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // sub-block 8 (i / 2) + 2 e + i % 2
                const int sub = 8 * (i >> 1) + 2 * e + (i & 1);
                I += __mul24(c[i], (int)(int8_t)(S[sub >> 2] >> (8 * (sub & 3))));
            }
        }
        return fmaf(a.d * w.d, (float)I, acc);
    }
};

// Workgroup: eight waves, NW = 8 / KG of them side by side (16 weight rows each, of NM matrices: gate and up, or one), KG on parts of k.
// The tile's activation rows go to LDS, MF_KC k at a time (all of k in most models), where every wave takes a part of it; the waves'
// weights are loaded U steps ahead of their use, the first of them before the rows. The parts' sums meet in LDS.
struct MfArgs {
    const uint8_t *w0, *w1;
    int64_t stride;
    int rows, n_k, n_expert, act_div;
    MfAct act;
    const int32_t* ids;
    const int2* tiles;
    const int32_t* order;
    float* out;
    AmvActOut q;
};

template <int WT, int NM, int KG, int G>
__global__ __launch_bounds__(512) void k_moe_few(const MfArgs p) {
    using T = Mf<WT>;
    constexpr int NW = 8 / KG, KC = G == 1 ? 8192 : 4096, CS = KC / T::STEP, LD = KC + 32, LS = CS * T::PER + 4;
    constexpr int R = 4 * G, COLS = 16 * NW;
    constexpr bool SUMS = WT == AMV_T_Q4_K, KQ = T::STEP == 256;
    __shared__ __align__(16) uint8_t s_q[32 + R * LD];  // 32 zeros, then the rows
    __shared__ __align__(16) float s_d[R * LS];
    __shared__ __align__(16) int16_t s_u[SUMS ? R * CS * 8 : 8];
    float(*const s_red)[NM][R][COLS + 1] = reinterpret_cast<float(*)[NM][R][COLS + 1]>(s_q);  // when the rows are done with
    static_assert(sizeof(float[KG][NM][R][COLS + 1]) <= 32 + R * LD, "the parts' sums take the rows' place");
    __shared__ int s_pair[R];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nw = wv % NW, kw = wv / NW, c16 = lane & 15, q = lane >> 4;
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
    const int n0 = blockIdx.x * COLS, n_g = (count + 3) >> 2;
    float acc[NM][G];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int m = 0; m < NM; ++m) acc[m][g] = 0.0f;
    if (tid < R) s_pair[tid] = p.tiles ? p.order[first + min(tid, count - 1)] : first;
    if (e < p.n_expert) {
        const uint8_t* const m[2] = {p.w0 + e * p.stride, NM == 2 ? p.w1 + e * p.stride : nullptr};
        const int n = n0 + 16 * nw + c16, nc = min(n, p.rows - 1);
        const int steps = KQ ? p.n_k : (p.n_k + 3) / 4;
        const int64_t k = (int64_t)p.n_k * (KQ ? 256 : 32);
        const int t4 = c16 >> 2, on = (c16 & 3) == q;
        if (tid < 2) reinterpret_cast<uint4*>(s_q)[tid] = make_uint4(0, 0, 0, 0);
        for (int c0 = 0; c0 < steps; c0 += CS) {
            const int ns = min(CS, steps - c0), per = (ns + KG - 1) / KG, s0 = kw * per, s1 = min(ns, s0 + per);
            typename T::W wa[NM], wb[NM];
            const auto load = [&](typename T::W (&w)[NM], int s) {
#pragma unroll
                for (int i = 0; i < NM; ++i) T::load(w[i], m[i], p.rows, p.n_k, nc, q, c0 + s);
            };
            if (s0 < s1) load(wa, s0);
            __syncthreads();  // (the first time: the pairs; then the rows before these are read)
            // rows c0 .. c0 + ns of the tile: integers in pieces of 16, zeros past k
            const int pieces = ns * (T::STEP / 16), k_left = (int)min((int64_t)KC, k - (int64_t)c0 * T::STEP) / 16;
            for (int r = wv; r < count; r += 8) {
                const int64_t row = s_pair[r] / p.act_div;
                const uint4* src = reinterpret_cast<const uint4*>(p.act.q + row * k + (int64_t)c0 * T::STEP);
                for (int i = lane; i < pieces; i += 64)
                    *reinterpret_cast<uint4*>(s_q + 32 + r * LD + 16 * i) = i < k_left ? src[i] : make_uint4(0, 0, 0, 0);
            }
            for (int x = tid; x < 4 * n_g * ns * T::PER; x += 512) {
                const int r = x / (ns * T::PER), b = x % (ns * T::PER), at = c0 * T::PER + b;
                const int64_t i = (int64_t)(s_pair[r] / p.act_div) * p.n_k + min(at, p.n_k - 1);
                const bool in = r < count && at < p.n_k;
                s_d[r * LS + b] = in ? (KQ ? p.act.dk[i] : p.act.d0[i].x) : 0.0f;
                if constexpr (SUMS) {
                    const moe_i4* u = reinterpret_cast<const moe_i4*>(p.act.s16 + i * 16);
                    uint32_t o[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const moe_i4 v = u[j];
                        o[j] = (uint32_t)((v.x + v.y) & 0xFFFF) | (uint32_t)(v.z + v.w) << 16;
                    }
                    reinterpret_cast<uint4*>(s_u)[r * CS + b] = make_uint4(o[0], o[1], o[2], o[3]);
                }
            }
            __syncthreads();
            const auto compute = [&](const typename T::W (&w)[NM], int s) {
                typename T::Scales c[NM];
#pragma unroll
                for (int i = 0; i < NM; ++i) T::scales(w[i], c[i]);
#pragma unroll
                for (int j = 0; j < T::U; ++j) {
                    if (s + j >= s1) break;
                    typename T::B b[NM];
#pragma unroll
                    for (int i = 0; i < NM; ++i) T::operands(w[i], c[i], j, b[i]);
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        if (g >= n_g) break;
                        typename T::A a;
                        const int live = on & (4 * g + t4 < count);
                        T::read(a, live ? s_q + 32 + (4 * g + t4) * LD + (s + j) * T::STEP : s_q, live, q,
                                s_d + (4 * g + q) * LS + (s + j) * T::PER, SUMS ? s_u + ((4 * g + q) * CS + s + j) * 8 : nullptr);
#pragma unroll
                        for (int i = 0; i < NM; ++i) acc[i][g] = T::add(b[i], a, acc[i][g]);
                    }
                }
            };
            for (int s = s0; s < s1; s += 2 * T::U) {
                if (s + T::U < s1) load(wb, s + T::U);
                compute(wa, s);
                if (s + T::U >= s1) break;
                if (s + 2 * T::U < s1) load(wa, s + 2 * T::U);
                compute(wb, s + T::U);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < NM; ++i) s_red[kw][i][4 * g + q][16 * nw + c16] = acc[i][g];
    __syncthreads();
    // thread: token i and column f (a block of the 8-bit output is 32 lanes)
    constexpr int PW = 512 / COLS;
    for (int i = tid / COLS; i < count; i += PW) {
        const int f = tid % COLS;
        float v[NM];
#pragma unroll
        for (int j = 0; j < NM; ++j) {
            v[j] = 0.0f;
#pragma unroll
            for (int z = 0; z < KG; ++z) v[j] += s_red[z][j][i][f];
        }
        const int64_t pr = s_pair[i];
        if constexpr (NM == 2) {
            if (n0 + f >= p.rows) continue;  // (whole blocks of 32)
            const float h = v[0] / (1.0f + expf(-v[0])) * v[NM - 1];
            if (p.out) p.out[pr * p.rows + n0 + f] = h;
            if (p.q.type) {
                const AmvActOut o = amv_act_row(p.q, pr, p.rows);
                int2* const meta = reinterpret_cast<int2*>(o.meta) + (n0 + f) / 32;
                amv_q8_0_lanes32(h, o.rule, f & 31, o.qs + n0 + (f & ~31), meta);
                // (a scale that is none where an element is: moe_act_store4)
                const uint64_t bad = __ballot(!(fabsf(h) < INFINITY));
                if ((f & 31) == 0 && (uint32_t)(bad >> (lane & 32))) meta->x = 0x7FC00000;
            }
        } else if (e < p.n_expert && n0 + f < p.rows) {
            p.out[pr * p.rows + n0 + f] = v[0];
        }
    }
}

template <int WT, int NM, int KG>
static void mf_go(const MfArgs& a, int n_tiles, hipStream_t st) {
    constexpr int COLS = 16 * (8 / KG);
    const dim3 grid((unsigned)((a.rows + COLS - 1) / COLS), (unsigned)n_tiles);
    if (!a.tiles) k_moe_few<WT, NM, KG, 1><<<grid, 512, 0, st>>>(a);
    else k_moe_few<WT, NM, KG, 4><<<grid, 512, 0, st>>>(a);
}

int moe_few(const MoeProduct& p) {
    const int64_t pairs = p.n_tok * p.n_used;
    const MoePlanView v = moe_plan_view(p.plan, pairs, p.n_expert);
    const bool kq = p.type == AMV_T_Q4_K || p.type == AMV_T_Q6_K, gu = p.w1 != nullptr;
    const int8_t* aq = (const int8_t*)p.act;
    const int8_t* meta = aq + p.act_rows * p.k;
    MfArgs a{(const uint8_t*)p.w0, (const uint8_t*)p.w1, p.stride, (int)p.rows, (int)(p.k / (kq ? 256 : 32)), p.n_expert, gu ? p.n_used : 1,
             {aq, (const float2*)meta, (const float*)meta, (const int32_t*)(meta + p.act_rows * (p.k / 64))}, p.ids, v.few, v.order, p.out, p.q};
    AMV_REQUIRE(p.plan || v.n_few <= 65535, "moe: %d pairs without a plan", v.n_few);
    for (int64_t t0 = 0; t0 < v.n_few; t0 += 65535) {
        const int n = (int)std::min<int64_t>(65535, v.n_few - t0);
        if (p.plan) a.tiles = v.few + t0;
#define GO(T) (gu ? mf_go<T, 2, 4>(a, n, p.st) : mf_go<T, 1, 4>(a, n, p.st))
        if (p.type == AMV_T_Q4_0) GO(AMV_T_Q4_0);
        else if (p.type == AMV_T_Q8_0) GO(AMV_T_Q8_0);
        else if (p.type == AMV_T_Q4_K) GO(AMV_T_Q4_K);
        else GO(AMV_T_Q6_K);
#undef GO
    }
    return amv_check_launch("amv_moe products");
}
