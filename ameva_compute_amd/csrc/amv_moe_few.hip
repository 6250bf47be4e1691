// The experts' products with few rows each (decode steps, small batches): a tile is up to 16 rows (pairs) of one expert.
//
// One v_mfma_i32_16x16x64_i8 multiplies 16 A rows of 64 bytes with 16 weight rows. A lane of the weights holds 16 bytes of weight
// row l % 16, and quarter q = l / 16 of the wave holds block q of four: the 64-long contraction would add four blocks up, each of
// which has a scale of its own. So A row 4 t + b has token t's integers in the bytes of quarter b and zeros in the others: of four
// tokens and four blocks, each comes out as an integer of its own, exact. Weights go from memory to the lanes as they lie (16 bytes a
// lane), and one instruction in four would do for the arithmetic, but these products are bound by the weights' bytes.
// Result D of lane l: weight row l % 16, token l / 16, blocks 0..3 in its four registers: the block epilogue is a sum within the lane.
// Measured, with cold weights: gate and up of 48 tokens with 8 of 64 experts of 1024 x 2048 Q4_0 40 us, 3.8 TB/s; down of 40 tokens,
// 2048 x 1408 Q8_0, 44 us, 4.4 TB/s.
#include "amv_moe_dot.h"

#include <type_traits>

typedef int mf_v4i __attribute__((ext_vector_type(4)));
typedef short mf_s2 __attribute__((ext_vector_type(2)));
// two 32-bit words at an address of any 16 bits
typedef uint32_t mf_u2 __attribute__((ext_vector_type(2), aligned(2)));

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

#define MF_RSRC(p, bytes) __builtin_amdgcn_make_buffer_rsrc((void*)(p), 0, (uint32_t)(bytes), 0x00027000)
__device__ __forceinline__ uint4 mf_load(__amdgpu_buffer_rsrc_t r, uint32_t off) {  // 0 past the buffer's end
    const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// the activation rows of a call: integers, and scales (Q8_0: {d, sum} per block; Q8_K: d per super-block) and sums per 16 (Q8_K)
struct MfAct {
    const int8_t* q;
    const float2* d0;
    const float* dk;
    const int32_t* s16;
};

// Per weight type: a step (STEP k) is four blocks of 32 or a super-block, U steps are loaded at once (struct W) of row n of the matrix at
// m (buffer r). The activations come from LDS: a row's integers of the step, the lane's own quarter of them, at p, its scales at s, its
// sums at u.
template <int WT, int U>
struct Mf32 {  // Q4_0, Q8_0
    static constexpr bool Q4 = WT == AMV_T_Q4_0;
    static constexpr int STEP = 128, PER = 4;      // PER: scales of a row and step
    static constexpr int SUMS = 0, AT = 32;  // SUMS: words of sums of a row and step; AT: bytes between the quarters' integers
    static_assert(!Q4 || U == 4, "a quarter of the wave holds a step's scales");
    struct W {
        uint4 q[U][Q4 ? 1 : 2];
        std::conditional_t<Q4, uint4, uint2> d[Q4 ? 1 : U];  // four f16; Q4_0: four pairs, quarter j of the wave holds step j's
    };
    // blocks past the end: other integers (their activations are zeros) and scales 0
    static __device__ __forceinline__ void load(W& w, __amdgpu_buffer_rsrc_t r, const uint8_t* m, int rows, int nb, int n, int q, int s) {
        const uint32_t at = ((uint32_t)n * nb + 4 * s + q) * (Q4 ? 16 : 32);
#pragma unroll
        for (int j = 0; j < U; ++j) {
            w.q[j][0] = mf_load(r, at + j * (Q4 ? 64 : 128));
            if constexpr (!Q4) w.q[j][1] = mf_load(r, at + j * 128 + 16);
        }
        if constexpr (Q4) {
            // the scales of rows 2 p and 2 p + 1 side by side: lane quarter q takes blocks 4 (s + q) .. + 3 (of both rows: what is done
            // to them here would wait for them)
            w.d[0] = mf_load(r, (uint32_t)rows * nb * 16 + ((uint32_t)(n >> 1) * nb + 4 * (s + q)) * 4);
        } else {
            const uint16_t* p = reinterpret_cast<const uint16_t*>(m + (size_t)rows * nb * 32) + (size_t)n * nb;
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
    // what a step needs of the weights alone, once for all tokens
    struct B {
        uint4 q[2];
        float d[4];
    };
    struct Scales {
        uint32_t lo[4], hi[4];
    };
    static __device__ __forceinline__ void scales(const W& w, Scales& c, int nb, int n, int q, int s) {
        if constexpr (Q4) {
            uint32_t x[4] = {w.d[0].x, w.d[0].y, w.d[0].z, w.d[0].w};
            if (4 * (s + 4) > nb)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = 4 * (s + q) + i < nb ? x[i] : 0u;
            const uint32_t sel = n & 1 ? 0x07060302u : 0x05040100u;  // the upper or the lower halves of two words
            mf_quarters(__builtin_amdgcn_perm(x[1], x[0], sel), c.lo);
            mf_quarters(__builtin_amdgcn_perm(x[3], x[2], sel), c.hi);
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
    static __device__ __forceinline__ float add(const B& w, const uint8_t* p, const float* s, const int*, float acc) {
        const uint4* v = reinterpret_cast<const uint4*>(p);
        const float4 d = *reinterpret_cast<const float4*>(s);
        mf_v4i c = {0, 0, 0, 0};
        c = mf_mma(v[0], w.q[0], c);
        c = mf_mma(v[1], w.q[1], c);
        acc = fmaf((float)c[0], w.d[0] * d.x, acc);
        acc = fmaf((float)c[1], w.d[1] * d.y, acc);
        acc = fmaf((float)c[2], w.d[2] * d.z, acc);
        return fmaf((float)c[3], w.d[3] * d.w, acc);
    }
};
template <int WT, int U>
struct Mf : Mf32<WT, U> {};

// Q4_K: quarter q has the 32 bytes of units 2 q (low nibbles) and 2 q + 1 (high) of a super-block
template <int U>
struct Mf<AMV_T_Q4_K, U> {
    static constexpr int STEP = 256, PER = 1, SUMS = 4, AT = 64;
    struct W {
        uint4 q[U][2], head[U];
    };
    static __device__ __forceinline__ void load(W& w, __amdgpu_buffer_rsrc_t r, const uint8_t*, int rows, int nsb, int n, int q, int s) {
        const uint32_t sb = (uint32_t)n * nsb + s, h = (uint32_t)rows * nsb * 128;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            w.q[j][0] = mf_load(r, (sb + j) * 128 + 32 * q);
            w.q[j][1] = mf_load(r, (sb + j) * 128 + 32 * q + 16);
            w.head[j] = mf_load(r, h + (sb + j) * 16);
        }
    }
    struct B {
        uint4 q[2];
        uint32_t sc[2];
        mf_s2 mn[4];
        float d, dm;
    };
    struct Scales {};
    static __device__ __forceinline__ void scales(const W&, Scales&, int, int, int, int) {}
    static __device__ __forceinline__ void operands(const W& w, const Scales&, int j, B& o) {
        const uint4 h = w.head[j];
        o.q[0] = w.q[j][0];
        o.q[1] = w.q[j][1];
        // scales and mins of units 0-3 and 4-7, one per byte
        o.sc[0] = h.y & 0x3F3F3F3Fu;
        o.sc[1] = (h.w & 0x0F0F0F0Fu) | ((h.y >> 2) & 0x30303030u);
        const uint32_t mn[2] = {h.z & 0x3F3F3F3Fu, ((h.w >> 4) & 0x0F0F0F0Fu) | ((h.z >> 2) & 0x30303030u)};
#pragma unroll
        for (int u = 0; u < 4; ++u)  // bytes 2 u, 2 u + 1 as two 16-bit numbers
            o.mn[u] = __builtin_bit_cast(mf_s2, __builtin_amdgcn_perm(0u, mn[u >> 1], u & 1 ? 0x0C030C02u : 0x0C010C00u));
        o.d = amv_h2f(h.x);
        o.dm = amv_h2f(h.x >> 16);
    }
    static __device__ __forceinline__ float add(const B& w, const uint8_t* p, const float* s, const int* u, float acc) {
        const uint4* v = reinterpret_cast<const uint4*>(p);
        mf_v4i lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            lo = mf_mma(v[i], mf_each(w.q[i], [](uint32_t x) { return x & 0x0F0F0F0Fu; }), lo);
            hi = mf_mma(v[2 + i], mf_each(w.q[i], [](uint32_t x) { return (x >> 4) & 0x0F0F0F0Fu; }), hi);
        }
        const uint4 us = *reinterpret_cast<const uint4*>(u);
        const uint32_t uw[4] = {us.x, us.y, us.z, us.w};
        int I1 = 0, I2 = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t c = w.sc[i >> 1] >> (16 * (i & 1));
            I1 += __mul24(lo[i], (int)(c & 0xFF));
            I1 += __mul24(hi[i], (int)((c >> 8) & 0xFF));
            I2 = __builtin_amdgcn_sdot2(__builtin_bit_cast(mf_s2, uw[i]), w.mn[i], I2, false);
        }
        return fmaf(fmaf(w.d, (float)I1, -(w.dm * (float)I2)), *s, acc);
    }
};

// Q6_K: quarter q = 2 h + p has elements 128 h + 16 p + {0, 32, 64, 96} .. + 15, four sub-blocks of 16
template <int U>
struct Mf<AMV_T_Q6_K, U> {
    static constexpr int STEP = 256, PER = 1, SUMS = 0, AT = 0;
    struct W {
        uint4 l0[U], l1[U], h[U], sc[U];
        uint32_t d[U];
    };
    static __device__ __forceinline__ void load(W& w, __amdgpu_buffer_rsrc_t r, const uint8_t* m, int rows, int nsb, int n, int q, int s) {
        const uint32_t all = (uint32_t)rows * nsb, sb = (uint32_t)n * nsb + s;
        const uint16_t* d = reinterpret_cast<const uint16_t*>(m + (size_t)all * 208);
#pragma unroll
        for (int j = 0; j < U; ++j) {
            w.l0[j] = mf_load(r, (sb + j) * 128 + 64 * (q >> 1) + 16 * (q & 1));
            w.l1[j] = mf_load(r, (sb + j) * 128 + 64 * (q >> 1) + 16 * (q & 1) + 32);
            w.h[j] = mf_load(r, all * 128 + (sb + j) * 64 + 16 * q);
            w.sc[j] = mf_load(r, all * 192 + (sb + j) * 16);
            w.d[j] = d[min(sb + j, all - 1)];
        }
    }
    struct B {
        uint4 l0, l1, h, sc;
        float d;
    };
    struct Scales {};
    static __device__ __forceinline__ void scales(const W&, Scales&, int, int, int, int) {}
    static __device__ __forceinline__ void operands(const W& w, const Scales&, int j, B& o) {
        o.l0 = w.l0[j];
        o.l1 = w.l1[j];
        o.h = w.h[j];
        o.sc = w.sc[j];
        o.d = amv_h2f(w.d[j]);
    }
    static __device__ __forceinline__ float add(const B& w, const uint8_t* p, const float* s, const int*, float acc) {
        const uint4* v = reinterpret_cast<const uint4*>(p);
        const uint32_t S[4] = {w.sc.x, w.sc.y, w.sc.z, w.sc.w};
        const mf_v4i z = {0, 0, 0, 0};
        int I = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // elements 32 e: low (e < 2) or high nibbles of l0 or l1, bits 2 e of h; minus 32
            const uint4 l = e & 1 ? w.l1 : w.l0;
            const auto one = [&](uint32_t x, uint32_t y) {
                return ((((x >> (e < 2 ? 0 : 4)) & 0x0F0F0F0Fu) | (((y >> (2 * e)) & 0x03030303u) << 4)) + 0x60606060u) ^ 0x80808080u;
            };
            const mf_v4i c = mf_mma(v[2 * e], make_uint4(one(l.x, w.h.x), one(l.y, w.h.y), one(l.z, w.h.z), one(l.w, w.h.w)), z);
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // sub-block 8 (i / 2) + 2 e + i % 2
                const int sub = 8 * (i >> 1) + 2 * e + (i & 1);
                I += __mul24(c[i], (int)(int8_t)(S[sub >> 2] >> (8 * (sub & 3))));
            }
        }
        return fmaf(*s * w.d, (float)I, acc);
    }
};

// Workgroup: one tile and NW groups of 16 weight rows (gate and up: half of them each), a wave a
// group on one of KG parts of k. The rows go to LDS, KC k at a time (all of k but where that is very long), a wave's first weights
// are on their way meanwhile; then a wave goes through its weights by itself, and the parts' sums meet in LDS. What carries it is
// several workgroups on a CU, whose chains (tile, order, rows; weights; sums) overlap: so few registers, one buffer of weights a wave.
struct MfArgs {
    const uint8_t *w0, *w1;
    int64_t stride, bytes;
    int rows, n_k, n_expert, act_div, n_cols, kc, dot;  // dot: tiles of up to so many rows by dot products
    MfAct act;
    const int2* tiles;
    const int32_t* order;
    float* out;
    AmvActOut q;
};
// LDS, in bytes: a row of zeros and the rows' integers, their scales, their sums, the parts' sums
struct MfLds {
    int ld, ls, d, u, red, total;
};
template <int STEP, int PER, int SUMS>
__host__ __device__ inline MfLds mf_lds(int kc, int r, int kg, int nw) {
    MfLds l;
    const int cs = kc / STEP;
    l.ld = kc + 32;
    l.ls = cs * PER + 4;
    l.d = (r + 1) * l.ld;
    l.u = l.d + 4 * r * l.ls;
    l.red = l.u + 4 * SUMS * r * (cs + 1);
    l.total = l.red + 4 * kg * r * nw * 17;
    return l;
}

// sums over each half of the wave, for the 16 lanes of a row: x's in rows 0 and 2, y's in rows 1 and 3
__device__ __forceinline__ float mf_sum2(float x, float y) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return amv_row16_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}
// sums over the wave: v[0], v[2], v[1], v[3] in its four rows
__device__ __forceinline__ float mf_sum4(const float (&v)[4]) {
    const auto half = [](float x, float y) {  // x in the lower half, y in the upper one
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
        return __uint_as_float(r[0]) + __uint_as_float(r[1]);
    };
    return mf_sum2(half(v[0], v[1]), half(v[2], v[3]));
}

// A tile of up to NR rows by dot products, lanes along the weight rows: its loads are runs of 1 KB where the matrix core's operand wants 64 bytes of
// 16 rows, but each row costs vector work, so it is for one or two rows (Q8_0, without nibbles to take apart: four), and for a k that fills the
// lanes. us, matrix core / dot products: 64 experts of gate and up 1024 x 2048, 16 tokens x 8, Q4_0 34 / 28, Q4_K 36 / 30, Q6_K 48 / 44, Q8_0 54 /
// 51; 8 experts of 6144 x 4096, 6 x 2, Q4_0 45 / 35, Q6_K 67 / 55; with tiles of up to four rows Q4_0 32, Q4_K 36; with half of
// the lanes idle, 8 tokens' down Q4_K 18 / 24. A wave has WR weight rows, four at a time (gate and up: two columns of both), over all of k;
// sums to red[group of 16 weight rows][row][weight row % 16]. H: the wave's parts of 64 / H lanes have four weight rows each (a short k).
template <int WT, int NR, bool GU, int NW, int WR, int H>
__device__ __forceinline__ void mf_dot(const uint8_t* m0, const uint8_t* m1, int rows, int units, int n0, int wave, const MoAct& act, const int32_t* order,
                                       int count, int act_div, float (*red)[MOE_FEW][17]) {
    using T = Mo<WT>;
    static_assert(!GU || H == 1, "");
    constexpr int L = 64 / H;
    const int lane = threadIdx.x & 63, at_k = lane % L;
    int row[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) row[r] = order[min(r, count - 1)] / act_div;
    for (int g0 = wave * (WR / 4); g0 < (wave + 1) * (WR / 4); g0 += H) {
        const int g = g0 + lane / L;
        const uint8_t* const m[2] = {m0, GU ? m1 : m0};
        const int n[2] = {min(GU ? n0 + 2 * g : n0 + 4 * g, rows - 2), min(GU ? n0 + 2 * g : n0 + 4 * g + 2, rows - 2)};
        float acc[NR][4];
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[r][i] = 0.0f;
        for (int s = 0; s < units; s += L) {
            const int j = min(s + at_k, units - 1);
            typename T::W w[2];
            typename T::A a[NR];
            T::load(w[0], m[0], rows, units, n[0], j);
            T::load(w[1], m[1], rows, units, n[1], j);
#pragma unroll
            for (int r = 0; r < NR; ++r) T::load(a[r], act, row[r], units, j);
            __builtin_amdgcn_sched_barrier(0);  // (all loads before the first product)
            if (s + at_k < units)
#pragma unroll
                for (int i = 0; i < 2; ++i) T::add(w[i], a, j, acc, 2 * i);
        }
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            if constexpr (H == 2) {
                const float v = mf_sum2(acc[r][0], acc[r][1]), u = mf_sum2(acc[r][2], acc[r][3]);
                const int c = 4 * g + ((lane >> 4) & 1);
                if ((lane & 15) == 0) {
                    red[c >> 4][r][c & 15] = v;
                    red[c >> 4][r][(c & 15) + 2] = u;
                }
                continue;
            }
            const float v = mf_sum4(acc[r]);
            const int at = ((lane >> 4) & 1) * 2 + (lane >> 5);  // which of the four
            const int c = GU ? (at >> 1) * (8 * NW) + 2 * g + (at & 1) : 4 * g + at;
            if ((lane & 15) == 0) red[c >> 4][r][c & 15] = v;
        }
    }
}

template <int WT, int U, bool GU, int NW, int KG>
__global__ __launch_bounds__(64 * NW * KG) __attribute__((amdgpu_waves_per_eu(4))) void k_moe_few(const MfArgs p) {
    using T = Mf<WT, U>;
    constexpr int G = MOE_FEW / 4, R = MOE_FEW, NT = 64 * NW * KG, COLS = 16 * (GU ? NW / 2 : NW);
    constexpr bool KQ = T::STEP == 256;
    constexpr int SUMS = T::SUMS;
    extern __shared__ __align__(16) uint8_t s_mem[];
    const MfLds L = mf_lds<T::STEP, T::PER, SUMS>(p.kc, R, KG, NW);
    float* const s_d = reinterpret_cast<float*>(s_mem + L.d);
    int* const s_u = reinterpret_cast<int*>(s_mem + L.u);
    float(*const s_red)[NW][R][17] = reinterpret_cast<float(*)[NW][R][17]>(s_mem + L.red);
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nw = wv % NW, kw = wv / NW, c16 = lane & 15, q = lane >> 4;
    // the workgroups of a tile's columns one after another over the XCDs (a run of tiles for each XCD leaves the last ones idle, where a
    // plan's last tiles are not taken: 48 tokens x 8 of 64 experts of 1024 x 2048 Q4_0 63 us, so 50)
    const int col = blockIdx.x % p.n_cols, tile = blockIdx.x / p.n_cols, n0 = col * COLS;
    const int2 t = p.tiles[tile];
    const int e = t.x & 0xFFFF, count = t.x >> 16;
    if (!count) return;
    const int n_g = (count + 3) >> 2;
    const auto pair = [&](int i) { return p.order[t.y + i]; };
    float acc[G];
#pragma unroll
    for (int g = 0; g < G; ++g) acc[g] = 0.0f;
    constexpr int WR = 16 * NW / (NW * KG);  // weight rows of a wave
    // (an expert's only tile: which of its rows are in a last small tile is chance, and the two ways round differently)
    const int2 prev = p.tiles[max(tile - 1, 0)];
    const bool dot = count <= p.dot && e < p.n_expert && !(tile && prev.x >> 16 && (prev.x & 0xFFFF) == e);
    if (dot) {
        const MoAct act{p.act.q, reinterpret_cast<const int2*>(p.act.d0), p.act.dk, p.act.s16};
        const uint8_t *const m0 = p.w0 + e * p.stride, *const m1 = GU ? p.w1 + e * p.stride : m0;
        const int units = KQ ? 8 * p.n_k : p.n_k;
        const auto go = [&](auto nr) __attribute__((always_inline)) {
            constexpr int N = decltype(nr)::value;
            if (!GU && units <= 32) mf_dot<WT, N, GU, NW, WR, GU ? 1 : 2>(m0, m1, p.rows, units, n0, wv, act, p.order + t.y, count, p.act_div, s_red[0]);
            else mf_dot<WT, N, GU, NW, WR, 1>(m0, m1, p.rows, units, n0, wv, act, p.order + t.y, count, p.act_div, s_red[0]);
        };
        if (count == 1) go(std::integral_constant<int, 1>());
        else if (count == 2) go(std::integral_constant<int, 2>());
        else if constexpr (WT == AMV_T_Q8_0) go(std::integral_constant<int, 4>());
        if constexpr (KG > 1)
            for (int i = tid; i < (KG - 1) * NW * R * 17; i += NT) (&s_red[1][0][0][0])[i] = 0.0f;
    } else if (e < p.n_expert) {
        const uint8_t* const m = (GU && nw >= NW / 2 ? p.w1 : p.w0) + e * p.stride;
        const __amdgpu_buffer_rsrc_t buf = MF_RSRC(m, p.bytes);
        const int n = min(n0 + 16 * (GU ? nw % (NW / 2) : nw) + c16, p.rows - 1);
        const int steps = KQ ? p.n_k : (p.n_k + 3) / 4, cs = p.kc / T::STEP;
        const int64_t k = (int64_t)p.n_k * (KQ ? 256 : 32);
        const int t4 = c16 >> 2, on = (c16 & 3) == q;
        for (int i = tid; i < L.ld / 16; i += NT) reinterpret_cast<uint4*>(s_mem)[i] = make_uint4(0, 0, 0, 0);
        for (int c0 = 0; c0 < steps; c0 += cs) {
            const int ns = min(cs, steps - c0), per = (ns + KG - 1) / KG, s0 = kw * per, s1 = min(ns, s0 + per);
            typename T::W w;
            if (s0 < s1) T::load(w, buf, m, p.rows, p.n_k, n, q, c0 + s0);
            if (c0) __syncthreads();  // (the rows before these are read)
            // steps c0 .. c0 + ns of the rows, a wave a row: integers in pieces of 16 (zeros past k), scales, sums of the units
            const int pieces = ns * (T::STEP / 16), k_left = (int)min((int64_t)p.kc, k - (int64_t)c0 * T::STEP) / 16;
            for (int r = wv; r < 4 * n_g && r < R; r += NT / 64) {
                const bool in = r < count;
                const int64_t row = pair(in ? r : 0) / p.act_div;
                if (in) {
                    const uint4* src = reinterpret_cast<const uint4*>(p.act.q + row * k + (int64_t)c0 * T::STEP);
                    for (int i = lane; i < pieces; i += 64)
                        *reinterpret_cast<uint4*>(s_mem + (r + 1) * L.ld + 16 * i) = i < k_left ? src[i] : make_uint4(0, 0, 0, 0);
                }
                for (int b = lane; b < ns * T::PER; b += 64) {
                    const int blk = c0 * T::PER + b;
                    const int64_t i = row * p.n_k + min(blk, p.n_k - 1);
                    const bool has = in && blk < p.n_k;
                    if constexpr (KQ) {
                        s_d[r * L.ls + b] = has ? p.act.dk[i] : 0.0f;
                    } else {
                        s_d[r * L.ls + b] = has ? p.act.d0[i].x : 0.0f;
                    }
                    if constexpr (KQ && SUMS) {  // the units' sums, two in a word
                        const moe_i4* u = reinterpret_cast<const moe_i4*>(p.act.s16 + i * 16);
                        uint32_t o[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const moe_i4 v = u[j];
                            o[j] = (uint32_t)((v.x + v.y) & 0xFFFF) | (uint32_t)(v.z + v.w) << 16;
                        }
                        reinterpret_cast<uint4*>(s_u)[r * (cs + 1) + b] = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                }
            }
            __syncthreads();
            // all steps for n groups of four rows, two groups at a time side by side (one after the other, a chain of a row's read, its
            // products and its sums would be waited for at every turn; more than two take too many registers)
            const auto go = [&](auto n_groups) {
                constexpr int NG = decltype(n_groups)::value;
                // where the lane's integers are (in the row of zeros, for the quarters that are not its block's), its row's scales and sums
                const uint8_t* a[NG];
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const int at = T::AT ? T::AT * q : 128 * (q >> 1) + 16 * (q & 1);
                    a[g] = s_mem + (on && 4 * g + t4 < count ? (4 * g + t4 + 1) * L.ld + at : 0) + s0 * T::STEP;
                }
                const float* d = s_d + q * L.ls + s0 * T::PER;
                const int* u = s_u + (q * (cs + 1) + s0) * SUMS;
                for (int s = s0; s < s1; s += U) {
                    if (s > s0) T::load(w, buf, m, p.rows, p.n_k, n, q, c0 + s);
                    typename T::Scales c;
                    T::scales(w, c, p.n_k, n, q, c0 + s);
#pragma unroll
                    for (int j = 0; j < U; ++j) {
                        if (s + j >= s1) break;
                        typename T::B b;
                        T::operands(w, c, j, b);
#pragma unroll
                        for (int g = 0; g < NG; ++g) {
                            acc[g] = T::add(b, a[g] + j * T::STEP, d + 4 * g * L.ls + j * T::PER, u + (4 * g * (cs + 1) + j) * SUMS, acc[g]);
                            if (NG > 2 && (g & 1)) __builtin_amdgcn_sched_barrier(0);
                        }
                    }
#pragma unroll
                    for (int g = 0; g < NG; ++g) a[g] += U * T::STEP;
                    d += U * T::PER;
                    u += U * SUMS;
                }
            };
            if (n_g == 1) go(std::integral_constant<int, 1>());
            else if (n_g == 2) go(std::integral_constant<int, 2>());
            else if (n_g == 3) go(std::integral_constant<int, 3>());
            else go(std::integral_constant<int, G>());
        }
    }
    if (!dot)
#pragma unroll
        for (int g = 0; g < G; ++g) s_red[kw][nw][4 * g + q][c16] = acc[g];
    __syncthreads();
    // thread: row i and column f (a block of the 8-bit output is 32 lanes)
    for (int i = tid / COLS; i < count; i += NT / COLS) {
        const int f = tid % COLS;
        if (n0 + f >= p.rows) continue;  // (columns come in blocks of 32)
        float v[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < (GU ? 2 : 1); ++j)
#pragma unroll
            for (int z = 0; z < KG; ++z) v[j] += s_red[z][j * (NW / 2) + (f >> 4)][i][f & 15];
        const int64_t pr = pair(i);
        if constexpr (GU) {
            const float h = v[0] / (1.0f + expf(-v[0])) * v[1];
            if (p.out) p.out[pr * p.rows + n0 + f] = h;
            if (p.q.type) {
                const AmvActOut o = amv_act_row(p.q, pr, p.rows);
                moe_q8_0(h, o.rule, f & 31, o.qs + n0 + (f & ~31), reinterpret_cast<int2*>(o.meta) + (n0 + f) / 32);
            }
        } else if (e < p.n_expert) {
            p.out[pr * p.rows + n0 + f] = v[0];
        }
    }
}

// k that a workgroup's LDS holds of a tile's rows
#define MF_KC 3584

template <int WT, int U, bool GU, int NW, int KG>
static void mf_go(MfArgs a, int64_t tiles, int64_t k, hipStream_t st) {
    using T = Mf<WT, U>;
    constexpr int COLS = 16 * (GU ? NW / 2 : NW);
    a.n_cols = (a.rows + COLS - 1) / COLS;
    // all of k, or even parts of it, in whole steps
    const int64_t steps = (k + T::STEP - 1) / T::STEP, most = MF_KC / T::STEP, parts = (steps + most - 1) / most;
    a.kc = (int)((steps + parts - 1) / parts * T::STEP);
    const MfLds l = mf_lds<T::STEP, T::PER, T::SUMS>(a.kc, MOE_FEW, KG, NW);
    k_moe_few<WT, U, GU, NW, KG><<<(unsigned)(tiles * a.n_cols), 64 * NW * KG, l.total, st>>>(a);
}
template <int WT>
static void mf_type(const MfArgs& a, int64_t tiles, int64_t k, bool gu, hipStream_t st) {
    constexpr int U = WT == AMV_T_Q4_0 ? 4 : WT == AMV_T_Q8_0 ? 2 : 1;
    if (k <= 2560) {
        if (gu) mf_go<WT, U, true, 8, 1>(a, tiles, k, st);
        else mf_go<WT, U, false, 8, 1>(a, tiles, k, st);
    } else {
        if (gu) mf_go<WT, U, true, 4, 2>(a, tiles, k, st);
        else mf_go<WT, U, false, 4, 2>(a, tiles, k, st);
    }
}

int moe_few(const MoeProduct& p) {
    const int64_t pairs = p.n_tok * p.n_used;
    const MoePlanView v = moe_plan_view(p.plan, pairs, p.n_expert);
    const bool kq = p.type == AMV_T_Q4_K || p.type == AMV_T_Q6_K, gu = p.w1 != nullptr;
    const int8_t* aq = (const int8_t*)p.act;
    const int8_t* meta = aq + p.act_rows * p.k;
    const int units = (int)(p.k / 32), lanes = !gu && units <= 32 ? 32 : (units + 63) / 64 * 64;
    const int dot = 4 * units < 3 * lanes ? 0 : p.type == AMV_T_Q8_0 ? 4 : 2;
    const MfArgs a{(const uint8_t*)p.w0, (const uint8_t*)p.w1, p.stride, amv_weight_bytes(p.type, p.rows, p.k), (int)p.rows,
                   (int)(p.k / (kq ? 256 : 32)), p.n_expert, gu ? p.n_used : 1, 0, 0, dot,
                   {aq, (const float2*)meta, (const float*)meta, (const int32_t*)(meta + p.act_rows * (p.k / 64))}, v.few, v.order,
                   p.out, p.q};
    AMV_REQUIRE((int64_t)v.n_few * ((p.rows + 31) / 32) < 1 << 23, "moe: %d tiles of %lld columns are too many", v.n_few, (long long)p.rows);
    if (p.type == AMV_T_Q4_0) mf_type<AMV_T_Q4_0>(a, v.n_few, p.k, gu, p.st);
    else if (p.type == AMV_T_Q8_0) mf_type<AMV_T_Q8_0>(a, v.n_few, p.k, gu, p.st);
    else if (p.type == AMV_T_Q4_K) mf_type<AMV_T_Q4_K>(a, v.n_few, p.k, gu, p.st);
    else mf_type<AMV_T_Q6_K>(a, v.n_few, p.k, gu, p.st);
    return amv_check_launch("amv_moe products");
}
