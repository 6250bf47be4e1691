// A mixture of experts' feed-forward part: the residual's addition with the norm and its 8-bit output, the routing, the plan of the
// pairs that the products go by, and the entry points of the products (their kernels are in amv_moe_one.hip, amv_moe_few.hip and
// amv_moe_many.hip).
#include "amv_moe.h"

#include <algorithm>

// ---------------------------------------------------------------------------------------------------------------- norm
// sum = x + add; o = sum / sqrt(mean(sum^2) + eps) * w, act = o in 8 bits, one workgroup per row, the row in registers in
// between. The squares are f32 products summed in 64 bits and mean, root and quotient are rounded as amv_rms_norm's. Bound by memory: 4096
// rows of 4096 with a Q8_K output are 0.29 GB in 54 us, 5.4 TB/s; one row takes 4 to 6, a launch and two dependent passes. Loads past the caches
// against loads through them, by events around the launch: x and add last written some passes before 55 / 71 us; add by the launch before,
// as an attention's output is, 61 / 63 to 64; both by the two launches before 52 / 62. The choice between w4[c]
// and z is one between places, so the forms of R > 1 keep z in scratch (32 bytes a lane; 182 MB written where the outputs are 155).
template <int NT, int R>
__global__ __launch_bounds__(NT) void k_add_rms_norm(const float* x, const float* add, int n4, float eps,
                                                     const float* __restrict__ w, float* sum, float* __restrict__ o,
                                                     const AmvActOut act) {
    __shared__ double s_part[NT / 64];
    const size_t row = blockIdx.x;
    const float4* x4 = reinterpret_cast<const float4*>(x) + row * n4;
    const float4* a4 = reinterpret_cast<const float4*>(add) + row * n4;
    float4* s4 = reinterpret_cast<float4*>(sum) + row * n4;
    const float4* w4 = reinterpret_cast<const float4*>(w);
    const int tid = threadIdx.x;
    float4 v[R], ww[R];
    double t = 0.0;
    for (int c0 = 0; c0 < n4; c0 += NT * R) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = c0 + tid + NT * r;
            const float4 z = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const float4 a = c < n4 ? moe_ld_stream(x4 + c) : z, b = c < n4 ? moe_ld_stream(a4 + c) : z;
            if (n4 <= NT * R) ww[r] = c < n4 && w ? w4[c] : z;
            v[r] = make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = c0 + tid + NT * r;
            if (c < n4) s4[c] = v[r];
            t += (double)(v[r].x * v[r].x);
            t += (double)(v[r].y * v[r].y);
            t += (double)(v[r].z * v[r].z);
            t += (double)(v[r].w * v[r].w);
        }
    }
    t = amv_wave_sum_d_u(t);
    if ((tid & 63) == 0) s_part[tid >> 6] = t;
    __syncthreads();
    double tot = 0.0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) tot += s_part[i];
    const float scale = amv_rms_scale(tot, 4 * n4, eps);
    const AmvActOut q = amv_act_row(act, row, 4 * (int64_t)n4);
    const auto finish = [&](int c, const float4& s, const float4& g) __attribute__((always_inline)) {
        float y[4] = {s.x * scale, s.y * scale, s.z * scale, s.w * scale};
        if (w) {
            y[0] *= g.x;
            y[1] *= g.y;
            y[2] *= g.z;
            y[3] *= g.w;
        }
        if (o) reinterpret_cast<float4*>(o)[row * n4 + c] = make_float4(y[0], y[1], y[2], y[3]);
        if (q.type) moe_act_store4(q, c, y);
    };
    if (n4 <= NT * R) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = tid + NT * r;
            if (c < n4) finish(c, v[r], ww[r]);
        }
    } else {  // a thread reads back the sums that it stored itself
        for (int c = tid; c < n4; c += NT) finish(c, s4[c], w ? w4[c] : make_float4(0.0f, 0.0f, 0.0f, 0.0f));
    }
}

extern "C" int amv_add_rms_norm_act(const float* x, const float* add, int64_t n_rows, int64_t n, float eps, const float* w,
                                    float* sum, float* o, void* act, int act_type, int rule, void* stream) {
    AMV_REQUIRE(x && add && sum, "amv_add_rms_norm: null input or sum");
    AMV_REQUIRE(n_rows >= 0 && n > 0 && n_rows < 1 << 22 && n <= 1 << 24, "amv_add_rms_norm: bad shape");
    AMV_REQUIRE(n % 4 == 0, "amv_add_rms_norm: n %% 4 != 0");
    AMV_REQUIRE((((uintptr_t)x | (uintptr_t)add | (uintptr_t)w | (uintptr_t)sum | (uintptr_t)o | (uintptr_t)act) & 15) == 0,
                "amv_add_rms_norm: buffers must be 16-byte aligned");
    AMV_REQUIRE(!act || act_type == AMV_T_Q8_0 || act_type == AMV_T_Q8_K, "amv_add_rms_norm: act_type %d (Q8_0 or Q8_K)", act_type);
    AMV_REQUIRE(!act || n % (act_type == AMV_T_Q8_K ? 256 : 32) == 0,
                "amv_add_rms_norm: the fused quantization needs n %% block size == 0");
    AMV_REQUIRE(rule >= AMV_Q8_X86 && rule <= AMV_Q8_REF, "amv_add_rms_norm: bad rule");
    if (!n_rows) return AMV_OK;
    const AmvActOut q = amv_act_out(act, n, act ? act_type : 0, rule, n_rows);
    const int n4 = (int)(n / 4);
    const dim3 grid((unsigned)n_rows);
    // few rows: as many threads a row as load it at once; many: the waves of several rows on a CU hide one another's latencies, so fewer
    // (4096 rows of 4096, us: 1024 threads 71, 256 threads of 4 chunks 68, both with loads through the caches)
    if (n4 <= 256) k_add_rms_norm<256, 1><<<grid, 256, 0, amv_stream(stream)>>>(x, add, n4, eps, w, sum, o, q);
    else if (n_rows >= 1024 && n4 <= 512) k_add_rms_norm<256, 2><<<grid, 256, 0, amv_stream(stream)>>>(x, add, n4, eps, w, sum, o, q);
    else if (n_rows >= 1024 && n4 <= 1024) k_add_rms_norm<256, 4><<<grid, 256, 0, amv_stream(stream)>>>(x, add, n4, eps, w, sum, o, q);
    else if (n4 > 1024 && n4 <= 4096) k_add_rms_norm<1024, 4><<<grid, 1024, 0, amv_stream(stream)>>>(x, add, n4, eps, w, sum, o, q);
    else k_add_rms_norm<1024, 1><<<grid, 1024, 0, amv_stream(stream)>>>(x, add, n4, eps, w, sum, o, q);
    return amv_check_launch("amv_add_rms_norm");
}

// the values an activation buffer stands for (its integers times their block's scale), as f32 or f16
template <typename T>
__global__ __launch_bounds__(256) void k_act_values(const int8_t* __restrict__ q, const float* __restrict__ d, int shift, int step,
                                                    int64_t n4, T* __restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n4) return;
    const float s = d[((4 * i) >> shift) * step];
    const char4 v = reinterpret_cast<const char4*>(q)[i];
    out[4 * i] = (T)((float)v.x * s);
    out[4 * i + 1] = (T)((float)v.y * s);
    out[4 * i + 2] = (T)((float)v.z * s);
    out[4 * i + 3] = (T)((float)v.w * s);
}

extern "C" int amv_act_values(int act_type, const void* act, int64_t m, int64_t k, int out_type, void* out, void* stream) {
    AMV_REQUIRE(act && out, "amv_act_values: null pointer");
    AMV_REQUIRE(act_type == AMV_T_Q8_0 || act_type == AMV_T_Q8_K, "amv_act_values: type %d (Q8_0 or Q8_K)", act_type);
    const bool kq = act_type == AMV_T_Q8_K;
    AMV_REQUIRE(m >= 0 && k > 0 && k % (kq ? 256 : 32) == 0 && k <= INT32_MAX && m <= INT32_MAX, "amv_act_values: bad shape");
    // (four values a thread, 256 threads a workgroup, less than 2^32 threads a launch)
    AMV_REQUIRE(m * k <= ((int64_t)1 << 34) - 1024, "amv_act_values: too many values");
    AMV_REQUIRE(out_type == AMV_T_F32 || out_type == AMV_T_F16, "amv_act_values: output type %d (F32 or F16)", out_type);
    AMV_REQUIRE((((uintptr_t)act | (uintptr_t)out) & 7) == 0, "amv_act_values: buffers must be 8-byte aligned");
    if (!m) return AMV_OK;
    const int8_t* q = (const int8_t*)act;
    const float* d = (const float*)(q + m * k);
    const int64_t n4 = m * k / 4;
    const dim3 grid((unsigned)((n4 + 255) / 256));
    if (out_type == AMV_T_F32)
        k_act_values<float><<<grid, 256, 0, amv_stream(stream)>>>(q, d, kq ? 8 : 5, kq ? 1 : 2, n4, (float*)out);
    else
        k_act_values<_Float16><<<grid, 256, 0, amv_stream(stream)>>>(q, d, kq ? 8 : 5, kq ? 1 : 2, n4, (_Float16*)out);
    return amv_check_launch("amv_act_values");
}

// ---------------------------------------------------------------------------------------------------------------- routing
// One wave per token; lane l holds experts l, l + 64, ... Scores, their sums and the choices are in 64 bits: which of two close
// experts is the larger must not hang on a rounding. A choice becomes a whole number of the same order (0: not to be chosen), and
// n_used times the largest one is taken, the lower index first where they are equal. 4096 tokens of 256 experts in 8 groups take 11.9 us
// (vector work: 930 instructions a wave, a third of them the 64-bit exponentials and quotients), one token of 128 experts 3.4.
__device__ __forceinline__ uint64_t moe_key(double v) {  // NaN and minus infinity: 0
    const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);  // (-0 and 0 are one)
    return v > -INFINITY ? ((b >> 63) ? ~b : b | ((uint64_t)1 << 63)) : 0;
}
__device__ __forceinline__ uint64_t moe_lane(uint64_t v, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane) |
           (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32;
}
__device__ __forceinline__ uint32_t moe_wave_max(uint32_t v) {
    v = max(v, (uint32_t)amv_dpp_i<0xB1>((int)v));
    v = max(v, (uint32_t)amv_dpp_i<0x4E>((int)v));
    v = max(v, (uint32_t)amv_dpp_i<0x141>((int)v));
    v = max(v, (uint32_t)amv_dpp_i<0x140>((int)v));
    const auto lane = [&](int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
    return max(max(lane(0), lane(16)), max(lane(32), lane(48)));
}
// the lanes with the largest key, none where all are 0 (a key that is not 0 has an upper half that is not 0: others are no number)
__device__ __forceinline__ uint64_t moe_largest(uint64_t key) {
    const uint32_t hi = (uint32_t)(key >> 32), m = moe_wave_max(hi);
    if (!m) return 0;
    const uint64_t who = __ballot(hi == m);
    if (!(who & (who - 1))) return who;
    const uint32_t lo = hi == m ? (uint32_t)key : 0u, l = moe_wave_max(lo);
    return __ballot(hi == m && lo == l);
}
// b0, b1: the two largest so far (a c that is no number is in no comparison the larger)
__device__ __forceinline__ void moe_take(double& b0, double& b1, double c) {
    const bool up = c > b0;
    const double low = up ? b0 : c;
    b0 = up ? c : b0;
    b1 = low > b1 ? low : b1;
}
__device__ __forceinline__ double moe_lane_d(double v, int lane) {
    return __longlong_as_double((long long)moe_lane((uint64_t)__double_as_longlong(v), lane));
}

struct MoeRoute {
    const float* logits;
    const float* bias;
    int32_t* ids;
    float* weights;
    int64_t stride;
    double scale;
    int n_tok, n_expert, n_used, n_group, top_group, group_best, sigmoid, renorm;
};

template <int PER, bool GROUPS>
__global__ __launch_bounds__(64) void k_moe_route(const MoeRoute a) {
    __shared__ double s_choice[GROUPS ? 64 * PER : 1];
    const int lane = threadIdx.x, t = blockIdx.x;
    const float* lg = a.logits + t * a.stride;
    float l[PER];
    double p[PER], choice[PER];
    float top = -INFINITY;
#pragma unroll
    for (int v = 0; v < PER; ++v) {
        const int e = 64 * v + lane;
        l[v] = e < a.n_expert ? lg[e] : -INFINITY;
        top = fmaxf(top, l[v]);
    }
    double sum = 0.0;
    if (a.sigmoid) {
#pragma unroll
        for (int v = 0; v < PER; ++v) p[v] = 1.0 / (1.0 + exp(-(double)l[v]));
    } else {
        top = amv_wave_max_u(top);
#pragma unroll
        for (int v = 0; v < PER; ++v) {
            p[v] = exp((double)l[v] - (double)top);
            sum += p[v];
        }
        sum = amv_wave_sum_d_u(sum);
#pragma unroll
        for (int v = 0; v < PER; ++v) p[v] = p[v] / sum;
    }
    // softmax without a bias keeps the order of the logits
    const bool by_logit = !a.sigmoid && !a.bias && (!GROUPS || a.group_best == 1);
    uint64_t key[PER];
#pragma unroll
    for (int v = 0; v < PER; ++v) {
        const int e = 64 * v + lane;
        choice[v] = by_logit ? (double)l[v] : a.bias && e < a.n_expert ? p[v] + (double)a.bias[e] : p[v];
        key[v] = l[v] > -INFINITY ? moe_key(choice[v]) : 0;
    }
    if constexpr (GROUPS) {
        const int size = a.n_expert / a.n_group;
        const float inv = 1.0f / (float)size;
#pragma unroll
        for (int v = 0; v < PER; ++v) s_choice[64 * v + lane] = key[v] ? choice[v] : __longlong_as_double(0x7FF8000000000000ll);
        __syncthreads();
        // 2^sh lanes for a group, then its first one: the sum of the group's best choices
        const int sh = __builtin_clz(a.n_group - 1) - 26, per = 1 << sh, group = lane >> sh;
        double b0 = -INFINITY, b1 = -INFINITY;
        if (group < a.n_group)
            for (int i = lane & (per - 1); i < size; i += per) moe_take(b0, b1, s_choice[group * size + i]);
        for (int o = 1; o < per; o <<= 1) {
            const double c0 = __shfl_xor(b0, o, 64), c1 = __shfl_xor(b1, o, 64);
            moe_take(b0, b1, c0);
            moe_take(b0, b1, c1);
        }
        uint64_t g = lane & (per - 1) ? 0 : moe_key(a.group_best == 2 && b1 > -INFINITY ? b0 + b1 : b0), kept = 0;
        for (int i = 0; i < a.top_group; ++i) {
            const uint64_t who = moe_largest(g);
            if (!who) break;
            const int first = __builtin_ctzll(who);
            kept |= (uint64_t)1 << (first >> sh);
            if (lane == first) g = 0;
        }
#pragma unroll
        for (int v = 0; v < PER; ++v) {
            const int e = 64 * v + lane;
            const int of = (int)(((float)e + 0.5f) * inv);  // e / size: at least 1 / (2 size) from a whole number, off by 2^-22 of itself
            if (!((kept >> (of & 63)) & 1)) key[v] = 0;
        }
    }
    // lane i keeps the i-th choice
    int my_id = -1;
    double my_p = 0.0, total = 0.0;
    for (int i = 0; i < a.n_used; ++i) {
        uint64_t best = key[0];
        int at = 0;
#pragma unroll
        for (int v = 1; v < PER; ++v)
            if (key[v] > best) {
                best = key[v];
                at = v;
            }
        const uint64_t who = moe_largest(best);
        if (!who) break;
        int first = __builtin_ctzll(who), v_at = __builtin_amdgcn_readlane(at, first);
        if (who & (who - 1)) {  // equal ones: the lowest index, so the lowest v first
            for (uint64_t rest = who & (who - 1); rest; rest &= rest - 1) {
                const int o = __builtin_ctzll(rest), vo = __builtin_amdgcn_readlane(at, o);
                if (vo < v_at) {
                    v_at = vo;
                    first = o;
                }
            }
        }
        double pv = p[0];
#pragma unroll
        for (int v = 1; v < PER; ++v) pv = v == v_at ? p[v] : pv;
        pv = moe_lane_d(pv, first);
#pragma unroll
        for (int v = 0; v < PER; ++v)
            if (v == v_at && lane == first) key[v] = 0;
        total += pv;
        if (lane == i) {
            my_id = 64 * v_at + first;
            my_p = pv;
        }
    }
    if (lane < a.n_used) {
        const double w = a.renorm ? (total == 0.0 ? 0.0 : my_p / total) : my_p;
        a.ids[(int64_t)t * a.n_used + lane] = my_id;
        a.weights[(int64_t)t * a.n_used + lane] = my_id < 0 ? 0.0f : (float)(w * a.scale);
    }
}

extern "C" int amv_moe_route(const float* logits, int64_t logits_stride, int64_t n_tok, int64_t n_expert, int64_t n_used, int score,
                             const float* bias, int64_t n_group, int64_t top_group, int group_best, int renorm, float scale,
                             int32_t* ids, float* weights, void* stream) {
    AMV_REQUIRE(logits && ids && weights, "amv_moe_route: null pointer");
    AMV_REQUIRE(n_tok >= 0 && n_expert > 0 && n_expert <= MOE_MAX_EXPERTS, "amv_moe_route: %lld tokens, %lld experts (1 to %d are supported)",
                (long long)n_tok, (long long)n_expert, MOE_MAX_EXPERTS);
    AMV_REQUIRE(n_used > 0 && n_used <= MOE_MAX_USED && n_used <= n_expert, "amv_moe_route: %lld of %lld experts a token (up to %d)",
                (long long)n_used, (long long)n_expert, MOE_MAX_USED);
    AMV_REQUIRE(n_tok <= MOE_MAX_PAIRS / n_used, "amv_moe_route: more than %d pairs", MOE_MAX_PAIRS);
    AMV_REQUIRE(logits_stride >= n_expert || n_tok <= 1, "amv_moe_route: row stride < n_expert");
    AMV_REQUIRE(score == AMV_MOE_SOFTMAX || score == AMV_MOE_SIGMOID, "amv_moe_route: score %d", score);
    AMV_REQUIRE(n_group > 0 && n_group <= 64 && n_expert % n_group == 0 && top_group > 0 && top_group <= n_group,
                "amv_moe_route: %lld of %lld groups of %lld experts", (long long)top_group, (long long)n_group, (long long)n_expert);
    AMV_REQUIRE(group_best == 1 || group_best == 2, "amv_moe_route: group_best %d (1 or 2)", group_best);
    if (!n_tok) return AMV_OK;
    const MoeRoute a{logits, bias, ids, weights, logits_stride, (double)scale, (int)n_tok, (int)n_expert, (int)n_used,
                     (int)n_group, (int)top_group, group_best, score == AMV_MOE_SIGMOID, renorm != 0};
    const bool g = top_group < n_group;
    hipStream_t st = amv_stream(stream);
    const dim3 grid((unsigned)n_tok);
#define ROUTE(PER) (g ? k_moe_route<PER, true><<<grid, 64, 0, st>>>(a) : k_moe_route<PER, false><<<grid, 64, 0, st>>>(a))
    if (n_expert <= 64) ROUTE(1);
    else if (n_expert <= 128) ROUTE(2);
    else if (n_expert <= 256) ROUTE(4);
    else if (n_expert <= 512) ROUTE(8);
    else ROUTE(16);
#undef ROUTE
    return amv_check_launch("amv_moe_route");
}

// ---------------------------------------------------------------------------------------------------------------- plan
__device__ __forceinline__ void moe_put_tiles(int2* tiles, int at, int e, int first, int count, int rows) {
    for (int i = 0; i * rows < count; ++i) tiles[at + i] = make_int2(e | min(rows, count - i * rows) << 16, first + i * rows);
}

// Few pairs: one workgroup counts the experts' pairs in LDS, adds the counts up and puts each pair at its place.
__global__ __launch_bounds__(1024) void k_moe_plan_one(const int32_t* __restrict__ ids, int pairs, int n_expert, int2* few, int n_few,
                                                       int2* many, int n_many, int32_t* __restrict__ order) {
    __shared__ int s_count[MOE_MAX_EXPERTS + 1], s_first[MOE_MAX_EXPERTS + 1], s_sum[3][16];
    __shared__ int16_t s_id[MOE_PLAN_ONE];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    for (int e = tid; e <= n_expert; e += 1024) s_count[e] = 0;
    __syncthreads();
    for (int p = tid; p < pairs; p += 1024) {
        int e = ids[p];
        e = e >= 0 && e < n_expert ? e : n_expert;
        s_id[p] = (int16_t)e;
        atomicAdd(&s_count[e], 1);
    }
    __syncthreads();
    // sums over the experts before one: of pairs, of tiles of both sizes (thread e for expert e, and one for what is left)
    int base[3] = {0, 0, 0};
    for (int e0 = 0; e0 <= n_expert; e0 += 1024) {
        const int e = e0 + tid, c = e <= n_expert ? s_count[e] : 0;
        const int own[3] = {c, (c + MOE_FEW - 1) / MOE_FEW, (c + MOE_MANY - 1) / MOE_MANY};
        int before[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            int s = own[i];
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int u = __shfl_up(s, o, 64);
                s += lane >= o ? u : 0;
            }
            before[i] = s - own[i];
            if (lane == 63) s_sum[i][wv] = s;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            int all = 0;
            for (int j = 0; j < 16; ++j) {
                if (j == wv) before[i] += base[i] + all;
                all += s_sum[i][j];
            }
            base[i] += all;
        }
        if (e <= n_expert) {
            s_first[e] = before[0];
            moe_put_tiles(few, before[1], e, before[0], c, MOE_FEW);
            moe_put_tiles(many, before[2], e, before[0], c, MOE_MANY);
        }
        __syncthreads();
    }
    for (int i = base[1] + tid; i < n_few; i += 1024) few[i] = make_int2(0, 0);
    for (int i = base[2] + tid; i < n_many; i += 1024) many[i] = make_int2(0, 0);
    // the order of an expert's pairs does not enter into any result: the rows of a tile are computed alike, each by itself
    for (int p = tid; p < pairs; p += 1024) order[atomicAdd(&s_first[s_id[p]], 1)] = p;
}

// Many pairs: workgroup e reads all of them, counts those of lower experts and its own, and puts its own at their places. A lane has
// 4 consecutive pairs of each of B runs of 256, all loaded at once: 32768 pairs of 128 experts are one round trip (11 us; 23 with 64
// pairs a load and a ballot for each). The work is pairs times experts: 2^18 pairs of 128 take 50 us, 2^20 204 (of 1024 experts 883), 2^22 of
// 1024 4066.
__global__ __launch_bounds__(1024) void k_moe_plan(const int32_t* __restrict__ ids, int pairs, int n_expert, int2* few, int2* many,
                                                   int32_t* __restrict__ order) {
    constexpr int B = 8;
    __shared__ int s_low[16], s_own[16];
    const int e = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    // wave w: pairs from w * per on, per a multiple of 256
    const int per = ((pairs + 15) / 16 + 255) / 256 * 256, p0 = wv * per, p1 = min(pairs, p0 + per);
    int id[B][4];
    const auto load = [&](int p) {  // the experts of 256 B pairs from p on, -1 past p1
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int at = p + 256 * b + 4 * lane;
            moe_i4 v = {0, 0, 0, 0};
            if (at + 3 < p1) v = *reinterpret_cast<const moe_i4*>(ids + at);
            else
#pragma unroll
                for (int c = 0; c < 4; ++c) v[c] = at + c < p1 ? ids[at + c] : 0;
#pragma unroll
            for (int c = 0; c < 4; ++c) id[b][c] = at + c >= p1 ? -1 : v[c] >= 0 && v[c] < n_expert ? v[c] : n_expert;
        }
    };
    int low = 0, own = 0;
    for (int p = p0; p < p1; p += 256 * B) {
        load(p);
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                low += id[b][c] >= 0 && id[b][c] < e;
                own += id[b][c] == e;
            }
    }
    int before = own;  // the own pairs of the lanes up to this one
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(before, o, 64);
        before += lane >= o ? u : 0;
    }
    const int wave_low = amv_wave_sum_i_u(low);
    if (lane == 63) {
        s_low[wv] = wave_low;
        s_own[wv] = before;
    }
    before -= own;
    __syncthreads();
    int first = 0, count = 0;
    for (int j = 0; j < 16; ++j) {
        first += s_low[j];
        before += j < wv ? s_own[j] : 0;
        count += s_own[j];
    }
    int at = first + before;
    for (int p = p0; p < p1; p += 256 * B) {
        if (p1 - p0 > 256 * B) load(p);  // (else they are still here)
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (id[b][c] == e) order[at++] = p + 256 * b + 4 * lane + c;
    }
    // places for tiles: enough of them for any counts, the same ones by every workgroup's reckoning
    const auto places = [&](int2* tiles, int rows) {
        const int t0 = first / rows + e, t1 = (first + count) / rows + e + 1, n = (count + rows - 1) / rows;
        const int last = e == n_expert ? pairs / rows + n_expert + 1 : t1;
        for (int i = tid; t0 + i < last; i += 1024)
            tiles[t0 + i] = i < n ? make_int2(e | min(rows, count - i * rows) << 16, first + i * rows) : make_int2(0, 0);
    };
    places(few, MOE_FEW);
    places(many, MOE_MANY);
}

static int moe_check_pairs(const char* what, int64_t n_tok, int64_t n_used, int64_t n_expert) {
    AMV_REQUIRE(n_tok >= 0 && n_used > 0 && n_used <= MOE_MAX_USED && n_expert > 0 && n_expert <= MOE_MAX_EXPERTS,
                "%s: %lld tokens with %lld of %lld experts (up to %d of %d)", what, (long long)n_tok, (long long)n_used,
                (long long)n_expert, MOE_MAX_USED, MOE_MAX_EXPERTS);
    AMV_REQUIRE(n_tok <= MOE_MAX_PAIRS / n_used, "%s: more than %d pairs", what, MOE_MAX_PAIRS);
    return AMV_OK;
}

extern "C" int64_t amv_moe_plan_bytes(int64_t n_tok, int64_t n_used, int64_t n_expert) {
    if (moe_check_pairs("amv_moe_plan_bytes", n_tok, n_used, n_expert)) return -1;
    const int64_t pairs = n_tok * n_used;
    return 8 * (moe_tiles(pairs, n_expert, MOE_FEW) + moe_tiles(pairs, n_expert, MOE_MANY)) + 4 * pairs;
}

extern "C" int amv_moe_plan(const int32_t* ids, int64_t n_tok, int64_t n_used, int64_t n_expert, void* plan, void* stream) {
    const int rc = moe_check_pairs("amv_moe_plan", n_tok, n_used, n_expert);
    if (rc) return rc;
    AMV_REQUIRE(ids && plan && ((uintptr_t)plan & 7) == 0, "amv_moe_plan: null pointer or a plan that is not 8-byte aligned");
    const int64_t pairs = n_tok * n_used;
    if (!pairs) return AMV_OK;
    const MoePlanView v = moe_plan_view(plan, pairs, n_expert);
    hipStream_t st = amv_stream(stream);
    if (pairs <= MOE_PLAN_ONE)
        k_moe_plan_one<<<1, 1024, 0, st>>>(ids, (int)pairs, (int)n_expert, (int2*)v.few, v.n_few, (int2*)v.many, v.n_many, (int32_t*)v.order);
    else
        k_moe_plan<<<(unsigned)n_expert + 1, 1024, 0, st>>>(ids, (int)pairs, (int)n_expert, (int2*)v.few, (int2*)v.many, (int32_t*)v.order);
    return amv_check_launch("amv_moe_plan");
}

// ---------------------------------------------------------------------------------------------------------------- products
// rows of f32 to the 8-bit output, a float4 a thread (a row holds whole blocks, so that a block's threads leave together)
__global__ __launch_bounds__(256) void k_moe_quantize(const float4* __restrict__ x, int64_t total4, int n4, const AmvActOut act) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total4) return;
    const int64_t r = i / n4;
    const float4 v = x[i];
    const float h[4] = {v.x, v.y, v.z, v.w};
    moe_act_store4(amv_act_row(act, r, 4 * (int64_t)n4), (int)(i - r * n4), h);
}

// Tiles of many rows from so many rows an expert on that their products beside the weights' bytes cost less than the few rows' kernel,
// which does four times the matrix work; later where the tiles are too few to fill the GPU (us, few / many, at the rows an expert below
// and above the choice): 64 experts of gate and up 1024 x 2048 Q4_0 8: 50 / 51, 16: 65 / 60; Q8_0 4: 61 / 66, 8: 75 / 71; Q4_K 4: 44 / 46,
// 8: 54 / 50; Q6_K 8: 67 / 74, 16: 83 / 82; down 2048 x 1024 Q4_0 6: 28 / 30, 12: 36 / 33; Q8_0 4: 38 / 38, 8: 45 / 40; Q4_K 4: 25 / 26,
// 6: 28 / 25; Q6_K 8: 40 / 42, 12: 44 / 43; 8 experts of 4096 x 6144 Q4_0 24: 68 / 75, 32: 87 / 78; Q8_0 8: 65 / 64, 16: 85 / 79; Q4_K 8:
// 43 / 45, 24: 67 / 60; Q6_K 8: 57 / 62, 16: 78 / 74; of gate and up 2048 x 4096 Q4_K 16: 38 / 43, 32: 59 / 51; of 4096 x 14336 Q6_K 8:
// 126 / 136, 16: 168 / 160
static int moe_product(const MoeProduct& p) {
    if (!p.plan) return moe_one(p);
    const int64_t wgs = p.n_expert * ((p.rows + (p.w1 ? 63 : 127)) / (p.w1 ? 64 : 128));
    const int rows = p.type == AMV_T_Q4_0 ? (wgs >= 512 ? 10 : 28) : p.type == AMV_T_Q8_0 ? (wgs >= 512 ? 6 : 8)
                     : p.type == AMV_T_Q4_K ? (wgs >= 512 ? 5 : 20) : (wgs >= 512 ? 12 : 16);
    const bool many = p.n_tok * p.n_used >= (int64_t)rows * p.n_expert;
    return many ? moe_many(p) : moe_few(p);
}

// (p's counts are checked before, in the 64 bits they come in: moe_check_pairs)
static int moe_check_product(const char* what, const MoeProduct& p) {
    AMV_REQUIRE(p.type == AMV_T_Q4_0 || p.type == AMV_T_Q8_0 || p.type == AMV_T_Q4_K || p.type == AMV_T_Q6_K,
                "%s: weight type %d is not supported (Q4_0, Q8_0, Q4_K, Q6_K are)", what, p.type);
    const bool kq = p.type == AMV_T_Q4_K || p.type == AMV_T_Q6_K;
    AMV_REQUIRE(p.rows > 0 && p.k > 0 && p.k % (kq ? 256 : 32) == 0 && p.rows % 32 == 0, "%s: experts of %lld x %lld (rows a multiple of 32, k of %d)",
                what, (long long)p.rows, (long long)p.k, kq ? 256 : 32);
    AMV_REQUIRE(p.rows <= 1 << 20 && p.k <= 1 << 20 && p.rows * p.k < (int64_t)1 << 31, "%s: experts of %lld x %lld are too large", what,
                (long long)p.rows, (long long)p.k);
    AMV_REQUIRE(p.w0 && p.w1 && p.ids && (((uintptr_t)p.w0 | (uintptr_t)p.w1) & 15) == 0, "%s: null or unaligned weights, or no ids", what);
    AMV_REQUIRE(p.stride % 16 == 0 && p.stride >= amv_weight_bytes(p.type, p.rows, p.k), "%s: experts %lld bytes apart", what,
                (long long)p.stride);
    AMV_REQUIRE(p.act && ((uintptr_t)p.act & 15) == 0 && ((uintptr_t)p.plan & 7) == 0, "%s: null or unaligned activations or plan", what);
    AMV_REQUIRE(p.n_tok * p.n_used * std::max(p.rows, p.k) < (int64_t)1 << 32, "%s: %lld pairs of %lld are too many", what,
                (long long)(p.n_tok * p.n_used), (long long)std::max(p.rows, p.k));
    return AMV_OK;
}

// bytes of the pairs' rows in f32; -1 for counts that the products refuse
static int64_t moe_rows_bytes(const char* what, int64_t n_tok, int64_t n_used, int64_t rows) {
    if (moe_check_pairs(what, n_tok, n_used, 1)) return -1;
    AMV_REQUIRE(rows > 0 && rows <= 1 << 20 && n_tok * n_used * rows < (int64_t)1 << 32, "%s: %lld pairs of %lld", what,
                (long long)(n_tok * n_used), (long long)rows);
    return 4 * n_tok * n_used * rows;
}

extern "C" int64_t amv_moe_gate_up_workspace_bytes(int64_t n_tok, int64_t n_used, int64_t rows, int act_type) {
    const int64_t n = moe_rows_bytes("amv_moe_gate_up_workspace_bytes", n_tok, n_used, rows);
    return n < 0 || act_type == AMV_T_Q8_K ? n : 0;
}

extern "C" int amv_moe_gate_up(int wtype, const void* w_gate, const void* w_up, int64_t expert_stride, int64_t n_expert, int64_t rows,
                               int64_t k, const void* act, int64_t n_tok, int64_t n_used, const int32_t* ids, const void* plan,
                               float* eout, void* act_out, int act_type, int rule, void* workspace, int64_t workspace_bytes,
                               void* stream) {
    const char* what = "amv_moe_gate_up";
    int rc = moe_check_pairs(what, n_tok, n_used, n_expert);
    if (rc) return rc;
    MoeProduct p{wtype, (int)n_expert, (int)n_used, rows, k, expert_stride, n_tok, w_gate, w_up, act, n_tok, ids, plan, eout, {}, nullptr,
                 nullptr, amv_stream(stream)};
    rc = moe_check_product(what, p);
    if (rc) return rc;
    AMV_REQUIRE(eout || act_out, "%s: no output requested", what);
    AMV_REQUIRE((((uintptr_t)eout | (uintptr_t)act_out | (uintptr_t)workspace) & 15) == 0, "%s: buffers must be 16-byte aligned", what);
    AMV_REQUIRE(!act_out || act_type == AMV_T_Q8_0 || act_type == AMV_T_Q8_K, "%s: act_type %d (Q8_0 or Q8_K)", what, act_type);
    AMV_REQUIRE(!act_out || act_type != AMV_T_Q8_K || rows % 256 == 0, "%s: a Q8_K output of rows of %lld", what, (long long)rows);
    AMV_REQUIRE(rule >= AMV_Q8_X86 && rule <= AMV_Q8_REF, "%s: bad rule", what);
    const int64_t pairs = n_tok * n_used;
    if (!pairs) return AMV_OK;
    // blocks of 256 columns lie across the products' workgroups (32 or 64 columns of a row) and are quantized in a second launch, from f32
    // rows: of 4096 tokens with 8 experts of 1024 columns, all types, 9 to 15 us more than a Q8_0 output
    const bool late = act_out && act_type == AMV_T_Q8_K;
    if (late && !eout) {
        AMV_REQUIRE(workspace && workspace_bytes >= amv_moe_gate_up_workspace_bytes(n_tok, n_used, rows, act_type),
                    "%s: a workspace of %lld bytes, %lld needed", what, (long long)workspace_bytes,
                    (long long)amv_moe_gate_up_workspace_bytes(n_tok, n_used, rows, act_type));
        p.out = (float*)workspace;
    }
    if (act_out && !late) p.q = amv_act_out(act_out, rows, act_type, rule, pairs);
    const int r = moe_product(p);
    if (r || !late) return r;
    const int64_t total4 = pairs * rows / 4;
    k_moe_quantize<<<(unsigned)((total4 + 255) / 256), 256, 0, p.st>>>((const float4*)p.out, total4, (int)(rows / 4),
                                                                        amv_act_out(act_out, rows, act_type, rule, pairs));
    return amv_check_launch(what);
}

// out[t][n] = add[t][n] + sum_j weights[t][j] y[t n_used + j][n] over the pairs with an expert, in the order of j: 32768 pairs of 2048 are
// 0.34 GB in 48 us. (The products cannot add to out themselves: the sums' order would not be one.)
__global__ __launch_bounds__(256) void k_moe_combine(const float* __restrict__ y, const int32_t* __restrict__ ids,
                                                     const float* __restrict__ weights, int n_used, int n_expert, int n4,
                                                     const float* add, float* out) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    const int64_t t = blockIdx.y;
    if (c >= n4) return;
    float4 s = add ? moe_ld_stream(reinterpret_cast<const float4*>(add) + t * n4 + c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int j = 0; j < n_used; ++j) {
        const int e = ids[t * n_used + j];
        if (e < 0 || e >= n_expert) continue;
        const float w = weights[t * n_used + j];
        const float4 v = moe_ld_stream(reinterpret_cast<const float4*>(y) + (t * n_used + j) * n4 + c);
        s = make_float4(fmaf(w, v.x, s.x), fmaf(w, v.y, s.y), fmaf(w, v.z, s.z), fmaf(w, v.w, s.w));
    }
    reinterpret_cast<float4*>(out)[t * n4 + c] = s;
}

extern "C" int64_t amv_moe_down_workspace_bytes(int64_t n_tok, int64_t n_used, int64_t rows) {
    return moe_rows_bytes("amv_moe_down_workspace_bytes", n_tok, n_used, rows);
}

extern "C" int amv_moe_down(int wtype, const void* w, int64_t expert_stride, int64_t n_expert, int64_t rows, int64_t k, const void* act,
                            int64_t n_tok, int64_t n_used, const int32_t* ids, const void* plan, const float* weights,
                            const float* add, float* dst, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "amv_moe_down";
    int rc = moe_check_pairs(what, n_tok, n_used, n_expert);
    if (rc) return rc;
    MoeProduct p{wtype, (int)n_expert, (int)n_used, rows, k, expert_stride, n_tok, w, w, act, n_tok * n_used, ids, plan,
                 plan ? (float*)workspace : dst, {}, weights, add, amv_stream(stream)};
    rc = moe_check_product(what, p);
    if (rc) return rc;
    AMV_REQUIRE(weights && dst && (((uintptr_t)dst | (uintptr_t)add | (uintptr_t)workspace) & 15) == 0,
                "%s: null weights or dst, or a buffer that is not 16-byte aligned", what);
    const int64_t need = amv_moe_down_workspace_bytes(n_tok, n_used, rows);
    if (!n_tok) return AMV_OK;
    AMV_REQUIRE(!plan || (workspace && workspace_bytes >= need), "%s: a workspace of %lld bytes, %lld needed", what,
                (long long)workspace_bytes, (long long)need);
    p.w1 = nullptr;
    const int r = moe_product(p);
    if (r || !plan) return r;
    const int n4 = (int)(rows / 4);
    for (int64_t t0 = 0; t0 < n_tok; t0 += 65535) {
        const int64_t n = std::min<int64_t>(65535, n_tok - t0);
        k_moe_combine<<<dim3((unsigned)((n4 + 255) / 256), (unsigned)n), 256, 0, p.st>>>(
            p.out + t0 * n_used * rows, ids + t0 * n_used, weights + t0 * n_used, (int)n_used, (int)n_expert, n4,
            add ? add + t0 * rows : nullptr, dst + t0 * rows);
    }
    return amv_check_launch("amv_moe_down");
}
