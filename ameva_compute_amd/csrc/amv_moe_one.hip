// The experts' products of a token by itself (no plan): each pair is a product of one row, by dot products with the lanes along the weight
// rows; all loads of a step of 64 lanes, four weight rows, are on their way before the first product. (On the matrix core, with 16 weight rows a wave
// and 64 bytes of each a load, the same bytes take a third longer.)
// Gate and up: a workgroup has 32 columns of a pair, a wave two of them in both matrices. Down: a workgroup has a few columns of
// a token, its waves the token's experts, parts of a long k and columns, and adds the weighted products up: no second launch.
// Measured, with cold weights: two experts of 4096 x 14336 with their sum, Q6_K 18 us, 5.3 TB/s, Q8_0 28, Q4_0 13; gate and up of eight
// experts of 2048 x 4096 Q4_K 16 us, of 1024 x 2048 6, of which the bytes are 4.
#include "amv_moe_dot.h"

#include <algorithm>

// rows n[i] and n[i] + 1 of matrix m[i], M times, times activation row `row`, part of parts of k; H: the wave's parts of 64 / H lanes have rows
// of their own (n then differs between them). All loads of a step before its products;
// the loads of a second step beside them were slower (two experts of 4096 x 14336 Q4_0 14 us, so 13; 32 rows of 2048 x 4096 Q6_K 24, so 22).
template <int WT, int M, int H>
__device__ __forceinline__ void mo_rows(const uint8_t* const (&m)[M], int rows, int units, const int (&n)[M], const MoAct& act, int64_t row, int part,
                                        int parts, float (&acc)[1][2 * M]) {
    using T = Mo<WT>;
    constexpr int L = 64 / H;
    const int lane = threadIdx.x % L;
    for (int s = L * part; s < units; s += L * parts) {
        typename T::W w[M];
        typename T::A a[1];
        const int j = min(s + lane, units - 1);
#pragma unroll
        for (int i = 0; i < M; ++i) T::load(w[i], m[i], rows, units, n[i], j);
        T::load(a[0], act, row, units, j);
        __builtin_amdgcn_sched_barrier(0);
        if (s + lane < units)
#pragma unroll
            for (int i = 0; i < M; ++i) T::add(w[i], a, j, acc, 2 * i);
    }
#pragma unroll
    for (int i = 0; i < 2 * M; ++i) acc[0][i] = H == 1 ? amv_wave_sum(acc[0][i]) : amv_sum_x16(amv_row16_sum(acc[0][i]));
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
    float acc[1][4] = {};
    if (e >= 0 && e < p.n_expert) {
        const uint8_t* const m[2] = {p.w0 + e * p.stride, p.w1 + e * p.stride};
        const int n[2] = {n0 + 2 * wv, n0 + 2 * wv};
        mo_rows<WT, 2, 1>(m, p.rows, p.units, n, p.act, pair / p.n_used, 0, 1, acc);
    }
    if (lane == 0) *reinterpret_cast<float4*>(s_red[wv]) = make_float4(acc[0][0], acc[0][1], acc[0][2], acc[0][3]);
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

template <int WT, int H>
__global__ __launch_bounds__(1024) void k_moe_one_down(const MoArgs p) {
    constexpr int G = MO_PAIRS, C = 2 * G * H;  // columns of a wave
    __shared__ __align__(16) float s_red[MOE_MAX_USED][C];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int t = blockIdx.x / p.n_cols, n0 = C * p.groups * (blockIdx.x % p.n_cols);
    // job: C columns, expert, part (in turns where there are more than waves)
    for (int job = wv; job < p.groups * p.n_used * p.parts; job += blockDim.x >> 6) {
        const int part = job % p.parts, j = job / p.parts % p.n_used, c = n0 + C * (job / (p.parts * p.n_used)) + 2 * G * (lane / (64 / H));
        const int e = p.ids[t * p.n_used + j];
        float acc[1][2 * G] = {};
        if (e >= 0 && e < p.n_expert) {
            const uint8_t* m[G];
            int n[G];
#pragma unroll
            for (int i = 0; i < G; ++i) {
                m[i] = p.w0 + e * p.stride;
                n[i] = min(c + 2 * i, p.rows - 2);
            }
            mo_rows<WT, G, H>(m, p.rows, p.units, n, p.act, (int64_t)t * p.n_used + j, part, p.parts, acc);
        }
        if (lane % (64 / H) == 0)
#pragma unroll
            for (int i = 0; i < G; ++i) *reinterpret_cast<float2*>(s_red[job] + 2 * G * (lane / (64 / H)) + 2 * i) = make_float2(acc[0][2 * i], acc[0][2 * i + 1]);
    }
    __syncthreads();
    if (tid >= C * p.groups || n0 + tid >= p.rows) return;
    const int64_t at = (int64_t)t * p.rows + n0 + tid;
    float v = p.add ? p.add[at] : 0.0f;
    for (int j = 0; j < p.n_used; ++j) {
        const int e = p.ids[t * p.n_used + j];
        if (e < 0 || e >= p.n_expert) continue;
        float y = 0.0f;
        for (int z = 0; z < p.parts; ++z) y += s_red[(tid / C * p.n_used + j) * p.parts + z][tid % C];
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
    // H: a k of up to 32 units leaves room for the rows of two waves in one
    const int H = a.units <= 32 ? 2 : 1, C = 2 * MO_PAIRS * H;
    const int room = std::max(1, 8 / a.n_used), steps = (a.units + 63) / 64;
    const int64_t waves = n * (a.rows / C) * a.n_used;
    a.parts = (int)std::min<int64_t>(std::min(room, steps), std::max<int64_t>(1, 2048 / waves));
    a.groups = std::max(1, room / a.parts);
    a.n_cols = (a.rows + C * a.groups - 1) / (C * a.groups);
    const dim3 grid((unsigned)(n * a.n_cols)), block(64 * std::min(16, a.n_used * a.parts * a.groups));
    if (H == 2) k_moe_one_down<WT, 2><<<grid, block, 0, st>>>(a);
    else k_moe_one_down<WT, 1><<<grid, block, 0, st>>>(a);
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
