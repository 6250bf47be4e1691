// What the kernels of a mixture of experts share: the plan of a call's (token, slot) pairs, and checks of their arguments.
#pragma once
#include "amv_common.h"

// A plan, int32 words: tiles of up to MOE_FEW rows, tiles of up to MOE_MANY rows, then the pairs in the order of their experts
// (those of one in any order: a tile's rows are computed alike, each by itself). A tile is two words: expert | rows << 16, place of its first pair in the order;
// rows 0: no tile. Pairs without an expert stand last, in tiles of the expert n_expert. n_used >= 1, n_expert <= MOE_MAX_EXPERTS.
#define MOE_MAX_EXPERTS 1024
#define MOE_MAX_USED 64
#define MOE_MAX_PAIRS (1 << 22)
#define MOE_FEW 16
#define MOE_MANY 64
// up to this many pairs one workgroup makes the plan, its tiles side by side; above it each expert has places of its own for
// them, the unused ones among them
#define MOE_PLAN_ONE 4096

static inline int64_t moe_tiles(int64_t pairs, int64_t n_expert, int64_t rows) {
    const int64_t e = n_expert + 1;
    if (pairs > MOE_PLAN_ONE) return pairs / rows + e;
    const int64_t most = pairs < e ? pairs : e;  // experts that have a pair
    const int64_t n = (pairs + (rows - 1) * most) / rows;
    return n < pairs ? n : pairs;
}
struct MoePlanView {
    const int2* few;
    const int2* many;
    const int32_t* order;
    int n_few, n_many;
};
static inline MoePlanView moe_plan_view(const void* plan, int64_t pairs, int64_t n_expert) {
    MoePlanView v;
    v.n_few = (int)moe_tiles(pairs, n_expert, MOE_FEW);
    v.n_many = (int)moe_tiles(pairs, n_expert, MOE_MANY);
    v.few = (const int2*)plan;
    v.many = v.few + v.n_few;
    v.order = (const int32_t*)(v.many + v.n_many);
    return v;
}

// the experts' matrices of a product: rows x k of `type` each, `stride` bytes apart; a gate has its up beside it
struct MoeProduct {
    int type, n_expert, n_used;
    int64_t rows, k, stride, n_tok;
    const void *w0, *w1;
    const void* act;
    int64_t act_rows;
    const int32_t* ids;
    const void* plan;
    // gate and up: f32 [pairs][rows] and / or the 8-bit output; down: f32 [pairs][rows], but moe_one's f32 [n_tok][rows], the sum
    float* out;
    AmvActOut q;
    const float *weights, *add;  // of moe_one's sum
    hipStream_t st;
};
int moe_one(const MoeProduct& p);   // amv_moe_one.hip: without a plan
int moe_few(const MoeProduct& p);   // amv_moe_few.hip
int moe_many(const MoeProduct& p);  // amv_moe_many.hip

// amv_ld_stream of four floats
__device__ __forceinline__ float4 moe_ld_stream(const float4* p) {
    const uint4 v = amv_ld_stream(reinterpret_cast<const uint4*>(p));
    return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
}

// four int32 at an address of any whole int32 (a Q8_K buffer's sums begin where its scales end)
typedef int moe_i4 __attribute__((ext_vector_type(4), aligned(4)));

// amv_act_store4 for a block with an element that is infinite or no number: integers cannot say so and the largest value passes over
// it, so the block's scale is made none, and whatever reads it learns of it. Called as amv_act_store4.
__device__ __forceinline__ void moe_act_store4(const AmvActOut& o, int c, const float (&v)[4]) {
    amv_act_store4(o, c, v);
    const bool bad = !(fabsf(v[0]) < INFINITY && fabsf(v[1]) < INFINITY && fabsf(v[2]) < INFINITY && fabsf(v[3]) < INFINITY);
    const uint64_t any = __ballot(bad);
    if (!any) return;
    const int lane = threadIdx.x & 63;
    if (o.type == AMV_T_Q8_0) {
        if ((c & 7) == 0 && ((any >> (lane & 56)) & 0xFF)) reinterpret_cast<int2*>(o.meta)[c >> 3].x = 0x7FC00000;
    } else if ((c & 63) == 0) {
        reinterpret_cast<int*>(o.meta)[c >> 6] = 0x7FC00000;
    }
}

// Q8_0 of a block of 32 that 32 lanes hold, an element each: amv_q8_0_lanes32's rules and bytes, the largest and the sum by DPP; a block
// with an element that is infinite or no number gets a scale that is none (moe_act_store4)
__device__ __forceinline__ void moe_q8_0(float v, int rule, int j, int8_t* qs, int2* meta) {
    float a = fabsf(v);
    a = fmaxf(a, __int_as_float(amv_dpp_i<0xB1>(__float_as_int(a))));
    a = fmaxf(a, __int_as_float(amv_dpp_i<0x4E>(__float_as_int(a))));
    a = fmaxf(a, __int_as_float(amv_dpp_i<0x141>(__float_as_int(a))));
    a = fmaxf(a, __int_as_float(amv_dpp_i<0x140>(__float_as_int(a))));
    a = amv_max_x16(a);
    const float d = a / 127.0f;
    const float id = rule == AMV_Q8_X86 ? (a != 0.0f ? 127.0f / a : 0.0f) : (d != 0.0f ? 1.0f / d : 0.0f);
    const float t = v * id;
    const int q = (int)fminf(127.0f, fmaxf(-127.0f, rule == AMV_Q8_REF ? roundf(t) : rintf(t)));
    int s = q;
    s += amv_dpp_i<0xB1>(s);
    s += amv_dpp_i<0x4E>(s);
    s += amv_dpp_i<0x141>(s);
    s += amv_dpp_i<0x140>(s);
    const auto o = __builtin_amdgcn_permlane16_swap((uint32_t)s, (uint32_t)s, false, false);
    const uint64_t bad = __ballot(!(fabsf(v) < INFINITY));
    qs[j] = (int8_t)q;
    if (j == 0)
        *meta = make_int2((uint32_t)(bad >> (threadIdx.x & 32)) ? 0x7FC00000 : __float_as_int(amv_h2f(amv_f2h(d))), (int)(o[0] + o[1]));
}
