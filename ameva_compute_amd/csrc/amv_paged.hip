// The paged KV cache: keys and values appended with the position rotation on the way, and the choice of the pages that a
// token's attention reads (amv_paged_rope_append, amv_paged_select; the attention is in amv_paged_attn.hip).
#include "amv_paged.h"

// ---------------------------------------------------------------------------------------------------------------- checks
extern "C" int64_t amv_paged_chunk_bytes(int type, int64_t D, int64_t page_size) {
    if ((D != 64 && D != 128) || page_size < 16 || page_size > 1024 || (page_size & (page_size - 1))) return -1;
    if (type == AMV_T_F16) return page_size * 2 * D;
    if (type == AMV_T_Q8_0) return page_size * (D + D / 16);
    if (type == AMV_T_Q4_0) return page_size * (D / 2 + D / 16);
    return -1;
}

PgBatch pg_batch(const amv_paged_kv* kv, const amv_paged_batch* b) {
    return {b->cu_q, b->n_kv, b->table, b->table_stride, (int)b->n_seq, (int)b->n_tok, (int)b->max_kv,
            __builtin_ctz((unsigned)kv->page_size)};
}

int pg_check(const char* what, const amv_paged_kv* kv, const amv_paged_batch* b, int64_t n_head) {
    AMV_REQUIRE(kv && b, "%s: null pool or batch", what);
    const int64_t chunk = amv_paged_chunk_bytes(kv->type, kv->D, kv->page_size);
    AMV_REQUIRE(chunk > 0, "%s: type %d with heads of %d and pages of %d is not supported (F16, Q8_0, Q4_0; 64, 128; powers of two "
                "from 16 to 1024 are)", what, kv->type, kv->D, kv->page_size);
    AMV_REQUIRE(kv->k && kv->v && kv->n_pages > 0 && kv->n_pages < (int64_t)1 << 31, "%s: pool without pages", what);
    AMV_REQUIRE(kv->n_head_kv > 0 && kv->n_head_kv <= 1024 && kv->page_stride >= kv->n_head_kv * chunk &&
                    kv->page_stride % 16 == 0 && ((uintptr_t)kv->k & 15) == 0 && ((uintptr_t)kv->v & 15) == 0 &&
                    ((uintptr_t)kv->bounds & 15) == 0,
                "%s: pages of %lld bytes for %d KV heads of %lld each, or a pool that is not 16-byte aligned", what,
                (long long)kv->page_stride, kv->n_head_kv, (long long)chunk);
    AMV_REQUIRE(n_head > 0 && n_head % kv->n_head_kv == 0 && n_head / kv->n_head_kv <= 1024, "%s: %lld heads over %d KV heads",
                what, (long long)n_head, kv->n_head_kv);
    AMV_REQUIRE(b->n_kv && b->table && b->n_seq > 0 && b->n_tok >= 0 && b->max_q > 0 && b->max_kv >= 0,
                "%s: null lengths or table, or a bad size", what);
    AMV_REQUIRE(b->n_seq <= 65535 && b->n_tok <= (int64_t)1 << 24 && b->max_kv <= (int64_t)1 << 30 &&
                    b->n_tok * n_head <= 4 * (int64_t)PG_MAX_GROUPS,
                "%s: batch too large", what);
    AMV_REQUIRE(b->cu_q || (b->n_tok == b->n_seq && b->max_q == 1), "%s: without cu_q there is one token a sequence", what);
    AMV_REQUIRE(b->table_stride >= (b->max_kv + kv->page_size - 1) / kv->page_size,
                "%s: %lld columns of the table for %lld keys", what, (long long)b->table_stride, (long long)b->max_kv);
    return AMV_OK;
}

// ---------------------------------------------------------------------------------------------------------------- append
// One workgroup per KV head and per run of a sequence's tokens that share a page, so that the page's bounds have one writer. Four
// waves (one where every sequence has one token), D / 2 lanes per token, two elements a lane: the lanes' angle, sine and cosine
// are computed once per token in f64 and used by the G query heads and the key head. Elements are rotated in f64 and rounded to
// f32, which fixes the f32 value, and so the stored f16 or integer, up to one in 2^29 borderline cases, however a machine orders
// the sum. What bounds it: memory (4226 tokens of 32 and 8 heads of 128 into f16 pages of 16, 193 MB: 40 us, 4.8 TB/s, where a copy
// of 4 GiB reaches 5.0; into pages of 64, a quarter of the workgroups, 60 the call), at one token a sequence the launch (48 tokens: 4.5 us).
struct PgAppend {
    PgBatch b;
    const float* qkv;
    float* q_out;
    const int32_t* pos;
    uint8_t *k, *v;
    uint16_t* bounds;
    unsigned int* bad;
    int64_t qkv_stride, out_stride, page_stride;
    double lf, freq_scale, attn;  // a pair's turns per position: freq_scale * 2^(lf * pair)
    int n_pages, n_head, n_head_kv, G, n_dims, neox, rule, one;
};

__device__ __forceinline__ int pg_place_k(int d, int D) { return ((d >> 3) & 3) * (D / 4) + (d >> 5) * 8 + (d & 7); }
__device__ __forceinline__ int pg_place_v(int d, int D) { return ((d & 31) >> 1) * (D / 16) + (d >> 5) * 2 + (d & 1); }

__device__ __forceinline__ float pg_row16_max(float v) {
    v = fmaxf(v, __int_as_float(amv_dpp_i<0xB1>(__float_as_int(v))));
    v = fmaxf(v, __int_as_float(amv_dpp_i<0x4E>(__float_as_int(v))));
    v = fmaxf(v, __int_as_float(amv_dpp_i<0x141>(__float_as_int(v))));
    return fmaxf(v, __int_as_float(amv_dpp_i<0x140>(__float_as_int(v))));
}
// elements 2 i, 2 i + 1 of a row (lane i of its D / 2; a block of 32 is a DPP row of 16 lanes) into row `slot` of a chunk; every lane
// of the wave calls it, `live` ones store. Integers cannot say that an element is no number, and the maxima pass over it: the scale of
// its block is none instead, so that whoever reads the key or the value learns of it
template <int TYPE, int D, bool V>
__device__ __forceinline__ void pg_store_pair(uint8_t* chunk, int ps, int slot, int i, float x0, float x1, int rule, bool live) {
    using R = PgRow<TYPE, D>;
    const int at = V ? pg_place_v(2 * i, D) : pg_place_k(2 * i, D);
    if constexpr (TYPE == AMV_T_F16) {
        const amv_h2 h = {(_Float16)x0, (_Float16)x1};
        if (live) *reinterpret_cast<amv_h2*>(chunk + (size_t)slot * R::ROW + 4 * i) = h;
    } else {
        uint16_t* scale = reinterpret_cast<uint16_t*>(chunk + (size_t)ps * R::ROW + (size_t)slot * R::SC) + (i >> 4);
        const uint64_t none = __builtin_amdgcn_ballot_w64(x0 != x0 || x1 != x1);
        const bool no_number = (none >> (threadIdx.x & 48) & 0xFFFF) != 0;  // in the lane's block
        if constexpr (TYPE == AMV_T_Q8_0) {
            const float amax = pg_row16_max(fmaxf(fabsf(x0), fabsf(x1)));
            const float d = amax / 127.0f;
            float id;
            if (rule == AMV_Q8_X86) id = amax != 0.0f ? 127.0f / amax : 0.0f;
            else id = d != 0.0f ? 1.0f / d : 0.0f;
            const float t0 = x0 * id, t1 = x1 * id;
            const int q0 = (int)fminf(127.0f, fmaxf(-127.0f, rule == AMV_Q8_REF ? roundf(t0) : rintf(t0)));
            const int q1 = (int)fminf(127.0f, fmaxf(-127.0f, rule == AMV_Q8_REF ? roundf(t1) : rintf(t1)));
            if (live) {
                *reinterpret_cast<uint16_t*>(chunk + (size_t)slot * R::ROW + at) = (uint16_t)((q0 & 0xFF) | (q1 & 0xFF) << 8);
                if ((i & 15) == 0) *scale = no_number ? 0x7E00 : amv_f2h(d);
            }
        } else {
            // the element of largest magnitude, the first on ties
            const bool second = fabsf(x1) > fabsf(x0);
            float am = second ? fabsf(x1) : fabsf(x0), mx = second ? x1 : x0;
            int ai = 2 * i + second;
            const auto pick = [&](float om, float ox, int oi) {
                if (om > am || (om == am && oi < ai)) { am = om; mx = ox; ai = oi; }
            };
#define PG_PICK(C) pick(__int_as_float(amv_dpp_i<C>(__float_as_int(am))), __int_as_float(amv_dpp_i<C>(__float_as_int(mx))), amv_dpp_i<C>(ai))
            PG_PICK(0xB1);
            PG_PICK(0x4E);
            PG_PICK(0x141);
            PG_PICK(0x140);
#undef PG_PICK
            const float d = mx / -8.0f, id = d != 0.0f ? 1.0f / d : 0.0f;
            const int q0 = min(15, max(0, (int)(x0 * id + 8.5f))), q1 = min(15, max(0, (int)(x1 * id + 8.5f)));
            if (live) {
                chunk[(size_t)slot * R::ROW + (at >> 1)] = (uint8_t)(q0 | q1 << 4);
                if ((i & 15) == 0) *scale = no_number ? 0x7E00 : amv_f2h(d);
            }
        }
    }
}

template <int TYPE, int D>
__global__ __launch_bounds__(256) void k_paged_append(PgAppend a) {
    using R = PgRow<TYPE, D>;
    constexpr int LPR = D / 2, TPW = 64 / LPR;  // lanes per token, tokens per wave
    __shared__ float red[4 * TPW][4][LPR];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
    const int i = lane % LPR, sub = lane / LPR;
    const int hk = (int)blockIdx.x % a.n_head_kv, item = (int)blockIdx.x / a.n_head_kv;
    const int psh = a.b.pshift, ps = 1 << psh;
    int s, run = 0;
    if (a.one) s = item;  // one token a sequence, one run each
    else
        pg_find(a.b.n_seq, item, [&](int q) {
            const int n = a.b.last(q) - a.b.first(q), p1 = a.b.end(q);
            return n ? ((p1 - 1) >> psh) - ((p1 - n) >> psh) + 1 : 0;
        }, s, run);
    if (s >= a.b.n_seq) return;
    const int t_first = a.b.first(s), n_q = a.b.last(s) - t_first;
    if (n_q == 0) return;
    const int p_first = a.b.end(s) - n_q;                    // place of the sequence's first token of this call
    const int page = (p_first >> psh) + run;                  // the run's page in the sequence
    const int p0 = max(p_first, page << psh), p1 = min(p_first + n_q, (page + 1) << psh);
    const int n = p1 - p0, tok0 = t_first + p0 - p_first;
    const int phys = page >= 0 && page < a.b.table_stride ? a.b.table[s * a.b.table_stride + page] : -1;
    const bool stored = phys >= 0 && phys < a.n_pages;
    const int lost = stored ? max(0, p1 - max(p0, a.b.max_kv)) : n;
    if (lost && a.bad && threadIdx.x == 0) atomicAdd(a.bad, (unsigned)lost);
    const size_t chunk = (size_t)ps * (R::ROW + R::SC);
    const size_t off = (size_t)(stored ? phys : 0) * a.page_stride + hk * chunk;

    const int nd2 = a.n_dims / 2;
    const bool turns = i < nd2;
    const int e0 = !a.neox ? 2 * i : turns ? i : a.n_dims + 2 * (i - nd2), e1 = !a.neox ? e0 + 1 : turns ? i + nd2 : e0 + 1;
    const double freq = a.freq_scale * exp2(a.lf * i);
    // NEOX: where elements 2 i and 2 i + 1 of a row are after the rotation (lane, first or second)
    const auto owner = [&](int d, int& l, bool& sec) {
        if (d < nd2) { l = d; sec = false; }
        else if (d < a.n_dims) { l = d - nd2; sec = true; }
        else { l = nd2 + (d - a.n_dims) / 2; sec = (d - a.n_dims) & 1; }
        l += sub * LPR;
    };
    int l0, l1;
    bool s0, s1;
    owner(2 * i, l0, s0);
    owner(2 * i + 1, l1, s1);

    float lo0 = INFINITY, lo1 = INFINITY, hi0 = -INFINITY, hi1 = -INFINITY;
    for (int t = wave * TPW; t < n; t += nw * TPW) {
        const bool live = t + sub < n;
        const int tok = tok0 + min(t + sub, n - 1), place = p0 + min(t + sub, n - 1), slot = place & (ps - 1);
        const bool store = live && stored && place < a.b.max_kv;
        const float* row = a.qkv + tok * a.qkv_stride;
        float* orow = a.q_out + tok * a.out_stride + (int64_t)hk * a.G * D;
        const float* qr = row + (int64_t)hk * a.G * D;
        const float* kr = row + (int64_t)(a.n_head + hk) * D;
        const float k0 = kr[e0], k1 = kr[e1];
        const float2 vv = *reinterpret_cast<const float2*>(row + (int64_t)(a.n_head + a.n_head_kv + hk) * D + 2 * i);
        const double p = a.pos ? a.pos[tok] : place;
        const double turn = p * freq;  // in full turns: the whole ones go, exactly
        double sn, cs;
        sincospi(2.0 * (turn - rint(turn)), &sn, &cs);
        sn *= a.attn;
        cs *= a.attn;
        const auto rotate = [&](float x0, float x1, float& y0, float& y1) {
            if (turns) {
                y0 = (float)fma((double)x0, cs, -((double)x1 * sn));
                y1 = (float)fma((double)x0, sn, (double)x1 * cs);
            } else {
                y0 = x0;
                y1 = x1;
            }
        };
        for (int g = 0; g < a.G; g += 4) {
            float x0[4], x1[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float* src = qr + (int64_t)min(g + j, a.G - 1) * D;
                x0[j] = src[e0];
                x1[j] = src[e1];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float y0, y1;
                rotate(x0[j], x1[j], y0, y1);
                if (g + j < a.G && live) {
                    orow[(g + j) * D + e0] = y0;
                    orow[(g + j) * D + e1] = y1;
                }
            }
        }
        float y0, y1;
        rotate(k0, k1, y0, y1);
        if (a.neox) {
            const float a0 = __shfl(y0, l0, AMV_WAVE), b0 = __shfl(y1, l0, AMV_WAVE);
            const float a1 = __shfl(y0, l1, AMV_WAVE), b1 = __shfl(y1, l1, AMV_WAVE);
            y0 = s0 ? b0 : a0;
            y1 = s1 ? b1 : a1;
        }
        pg_store_pair<TYPE, D, false>(a.k + off, ps, slot, i, y0, y1, a.rule, store);
        pg_store_pair<TYPE, D, true>(a.v + off, ps, slot, i, vv.x, vv.y, a.rule, store);
        if (!store) continue;
        const float r0 = amv_round_f16(y0), r1 = amv_round_f16(y1);
        lo0 = fminf(lo0, r0);
        lo1 = fminf(lo1, r1);
        hi0 = fmaxf(hi0, r0);
        hi1 = fmaxf(hi1, r1);
    }
    if (!a.bounds || !stored || p0 >= a.b.max_kv) return;
    float* mine = &red[wave * TPW + sub][0][0];
    mine[i] = lo0;
    mine[LPR + i] = lo1;
    mine[2 * LPR + i] = hi0;
    mine[3 * LPR + i] = hi1;
    __syncthreads();
    if (threadIdx.x >= LPR) return;
    for (int w = 0; w < nw * TPW; ++w) {
        lo0 = fminf(lo0, red[w][0][i]);
        lo1 = fminf(lo1, red[w][1][i]);
        hi0 = fmaxf(hi0, red[w][2][i]);
        hi1 = fmaxf(hi1, red[w][3][i]);
    }
    amv_h2* low = reinterpret_cast<amv_h2*>(a.bounds + ((size_t)phys * a.n_head_kv + hk) * 2 * D) + i;
    amv_h2* high = low + D / 2;
    if ((p0 & (ps - 1)) != 0) {  // the page had keys before (and perhaps some at these places: their bounds stay, wider than need be)
        const amv_h2 l = *low, h = *high;
        lo0 = fminf(lo0, (float)l.x);
        lo1 = fminf(lo1, (float)l.y);
        hi0 = fmaxf(hi0, (float)h.x);
        hi1 = fmaxf(hi1, (float)h.y);
    }
    *low = amv_h2{(_Float16)lo0, (_Float16)lo1};
    *high = amv_h2{(_Float16)hi0, (_Float16)hi1};
}

extern "C" int amv_paged_rope_append(const amv_paged_kv* kv, const amv_paged_batch* batch, const float* qkv,
                                     int64_t qkv_stride, int64_t n_head, const int32_t* pos, int n_dims, int mode,
                                     float freq_base, float freq_scale, float attn_factor, int rule, float* q_out,
                                     int64_t out_stride, unsigned int* bad, void* stream) {
    const char* what = "amv_paged_rope_append";
    if (const int rc = pg_check(what, kv, batch, n_head)) return rc;
    if (batch->n_tok == 0) return AMV_OK;
    AMV_REQUIRE(qkv && q_out, "%s: null pointer", what);
    AMV_REQUIRE(qkv_stride >= (n_head + 2 * kv->n_head_kv) * kv->D && out_stride >= n_head * kv->D && qkv_stride % 4 == 0 &&
                    out_stride % 4 == 0 && ((uintptr_t)qkv & 15) == 0 && ((uintptr_t)q_out & 15) == 0,
                "%s: rows too short or not 16-byte aligned", what);
    AMV_REQUIRE(mode == 0 || mode == 2, "%s: rope mode %d (0 NORMAL, 2 NEOX)", what, mode);
    AMV_REQUIRE(n_dims >= 0 && n_dims <= kv->D && n_dims % 2 == 0, "%s: %d of %d elements rotated", what, n_dims, kv->D);
    AMV_REQUIRE(freq_base > 0.0f, "%s: frequency base %g", what, freq_base);
    AMV_REQUIRE(rule >= AMV_Q8_X86 && rule <= AMV_Q8_REF, "%s: Q8_0 rule %d", what, rule);
    const bool one = batch->max_q == 1;
    PgAppend a = {pg_batch(kv, batch), qkv, q_out, pos, (uint8_t*)kv->k, (uint8_t*)kv->v, (uint16_t*)kv->bounds, bad, qkv_stride,
                  out_stride, kv->page_stride, n_dims ? -2.0 * log2((double)freq_base) / n_dims : 0.0,
                  (double)freq_scale / 6.283185307179586476925, (double)attn_factor, (int)kv->n_pages, (int)n_head, kv->n_head_kv,
                  (int)(n_head / kv->n_head_kv), n_dims, mode == 2, rule, one};
    // n tokens touch at most (n - 1) / page_size + 2 pages
    const int64_t items = one ? batch->n_seq : batch->n_tok / kv->page_size + 2 * batch->n_seq;
    AMV_REQUIRE(items * kv->n_head_kv <= PG_MAX_GROUPS, "%s: batch too large", what);
    const dim3 grid((unsigned)(items * kv->n_head_kv)), block(one ? 64 : 256);
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, amv_stream(stream), a); };
    if (kv->D == 128) {
        if (kv->type == AMV_T_F16) go(k_paged_append<AMV_T_F16, 128>);
        else if (kv->type == AMV_T_Q8_0) go(k_paged_append<AMV_T_Q8_0, 128>);
        else go(k_paged_append<AMV_T_Q4_0, 128>);
    } else {
        if (kv->type == AMV_T_F16) go(k_paged_append<AMV_T_F16, 64>);
        else if (kv->type == AMV_T_Q8_0) go(k_paged_append<AMV_T_Q8_0, 64>);
        else go(k_paged_append<AMV_T_Q4_0, 64>);
    }
    return amv_check_launch(what);
}

// ---------------------------------------------------------------------------------------------------------------- select
// A page's score for a token and a KV head: sum over the group's heads h and the elements d of max(q_hd low_d, q_hd high_d). As
// max(q low, q high) = max(q, 0) high + min(q, 0) low, the heads join before the pages are met: score = up . high + down . low with
// up = sum_h max(q_h, 0), down = sum_h min(q_h, 0), one product of 2 D elements a page whatever the group. In f64 (a product of f32
// and f16 is exact there), so that which page comes first does not hang on the order of a sum. 16 lanes a page, each D / 16
// elements of both bounds. Bound: reading the bounds, 4 D bytes a page, and the launch (16 tokens over up to 512 pages of 8 KV heads:
// 10.3 us; one over 250: 4.6).
struct PgSelect {
    PgBatch b;
    const float* q;
    const uint16_t* bounds;
    double* score;  // [n_tok][n_head_kv][most]
    int32_t* sel;
    int64_t q_stride;
    int n_pages, n_head_kv, G, most, n_sel, n_first, n_last;
};
#define PG_SCORE_PAGES 64  // pages of a workgroup

// pages that token t of sequence s sees (those of its keys up to its own), at most `most`
__device__ __forceinline__ int pg_pages_seen(const PgBatch& b, int s, int t, int most) {
    const int seen = min(b.keys(s), b.end(s) - b.last(s) + t + 1);
    return seen <= 0 ? 0 : min(most, ((seen - 1) >> b.pshift) + 1);
}

template <int D>
__global__ __launch_bounds__(256) void k_paged_score(PgSelect a) {
    constexpr int E = D / 16;
    const int lane = threadIdx.x & 63, i = lane & 15;
    const int hk = (int)blockIdx.x % a.n_head_kv, tok = (int)blockIdx.x / a.n_head_kv;
    const int s = pg_seq_of(a.b, tok);
    if (s >= a.b.n_seq) return;
    const int n = pg_pages_seen(a.b, s, tok, a.most), p0 = (int)blockIdx.y * PG_SCORE_PAGES;
    if (p0 >= n || n <= a.n_sel) return;  // (all of them are selected)
    const int32_t* table = a.b.table + s * a.b.table_stride;
    double up[E] = {}, down[E] = {};
    for (int g = 0; g < a.G; ++g) {
        const float* q = a.q + tok * a.q_stride + (int64_t)(hk * a.G + g) * D + E * i;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float x = q[e];
            up[e] += x > 0.0f ? (double)x : 0.0;
            down[e] += x > 0.0f ? 0.0 : (double)x;  // (what is no number goes here)
        }
    }
    typedef _Float16 hv __attribute__((ext_vector_type(E)));
    hv low[4], high[4];
    int phys[4];
    const int first = p0 + (int)(threadIdx.x >> 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) phys[j] = table[min(first + 16 * j, n - 1)];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool in = (uint32_t)phys[j] < (uint32_t)a.n_pages;
        const uint16_t* b = a.bounds + ((int64_t)(in ? phys[j] : 0) * a.n_head_kv + hk) * 2 * D + E * i;
        low[j] = *reinterpret_cast<const hv*>(b);
        high[j] = *reinterpret_cast<const hv*>(b + D);
        if (!in) phys[j] = -1;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        double x = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) x = fma(up[e], (double)(float)high[j][e], fma(down[e], (double)(float)low[j][e], x));
        if (x != x) {  // 0 times infinity: a side without a bound, where no q asks for it, does not enter
            const auto add = [&](double q, double b, double none) { x = q == 0.0 && b == none ? x : fma(q, b, x); };
            x = 0.0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                add(down[e], (double)(float)low[j][e], -INFINITY);
                add(up[e], (double)(float)high[j][e], INFINITY);
            }
        }
        x += amv_dpp_d<0xB1>(x);
        x += amv_dpp_d<0x4E>(x);
        x += amv_dpp_d<0x141>(x);
        x += amv_dpp_d<0x140>(x);
        const int p = first + 16 * j;
        if (i == 0 && p < n) a.score[((int64_t)tok * a.n_head_kv + hk) * a.most + p] = phys[j] >= 0 ? x : __longlong_as_double(0x7FF8000000000000ll);
    }
}

// The n_sel pages of a token and a KV head: one workgroup, the candidates' scores in LDS as integers of the same order (0 for what is
// no number). The least selected score is found by digits of 8 bits: the candidates between lo and hi are counted in 256 equal
// ranges, and the range in which the count from above passes what is wanted becomes the next lo .. hi; starting at the scores'
// own least and largest, a few hundred pages are told apart after two counts. Bound: its chain of barriers, 5.1 us at 250 pages, 7.1 at
// 512 (scores and choice in one launch, a workgroup reading all bounds of its token: 10.4 and 14.5 us in place of 9.3 and 9.6).
__global__ __launch_bounds__(256) void k_paged_top(PgSelect a) {
    extern __shared__ uint64_t key[];  // [most]
    __shared__ uint64_t s_lo[4], s_hi[4];
    __shared__ unsigned hist[256];
    __shared__ int s_n[4][2];
    __shared__ int s_bin, s_need, s_in;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hk = (int)blockIdx.x % a.n_head_kv, tok = (int)blockIdx.x / a.n_head_kv;
    const int s = pg_seq_of(a.b, tok);
    if (s >= a.b.n_seq) return;
    const int n = pg_pages_seen(a.b, s, tok, a.most);
    int32_t* out = a.sel + ((int64_t)tok * a.n_head_kv + hk) * a.n_sel;
    if (n <= a.n_sel) {
        for (int i = tid; i < a.n_sel; i += 256) out[i] = i < n ? i : -1;
        return;
    }
    // candidates c0 .. c1 - 1; the pages before and behind them are selected
    const int c0 = a.n_first, c1 = n - a.n_last, want = a.n_sel - a.n_first - a.n_last;
    const double* score = a.score + ((int64_t)tok * a.n_head_kv + hk) * a.most;
    uint64_t lo = ~0ull, hi = 0;
    for (int i = c0 + tid; i < c1; i += 256) {
        const double x = score[i];
        const uint64_t u = (uint64_t)__double_as_longlong(x);
        const uint64_t k = x != x ? 0 : (u >> 63) ? ~u : u | 1ull << 63;  // (-0 comes before +0: a score of 0 is +0 here)
        key[i] = k;
        lo = k < lo ? k : lo;
        hi = k > hi ? k : hi;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t l = __shfl_xor(lo, o, AMV_WAVE), h = __shfl_xor(hi, o, AMV_WAVE);
        lo = l < lo ? l : lo;
        hi = h > hi ? h : hi;
    }
    if (lane == 0) {
        s_lo[w] = lo;
        s_hi[w] = hi;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        lo = s_lo[j] < lo ? s_lo[j] : lo;
        hi = s_hi[j] > hi ? s_hi[j] : hi;
    }
    // need of the candidates in lo .. hi are selected, and all above
    int need = want;
    uint64_t above = hi;  // keys larger than this are selected; of those from lo to it, `need` are
    while (need > 0 && lo < above) {
        const uint64_t range = above - lo;
        const int bits = 64 - __builtin_clzll(range), shift = bits > 8 ? bits - 8 : 0;
        hist[tid] = 0;
        __syncthreads();
        for (int i = c0 + tid; i < c1; i += 256) {
            const uint64_t k = key[i];
            if (k >= lo && k <= above) atomicAdd(&hist[(k - lo) >> shift], 1u);
        }
        __syncthreads();
        if (w == 0) {  // lane l: bins 255 - 4 l .. 252 - 4 l, the largest first
            int c[4], sum = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                c[j] = (int)hist[255 - 4 * lane - j];
                sum += c[j];
            }
            int upto = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int v = __shfl_up(upto, o, AMV_WAVE);
                if (lane >= o) upto += v;
            }
            int past = upto - sum;
            if (past < need && upto >= need) {  // one lane
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (past < need && past + c[j] >= need) {
                        s_bin = 255 - 4 * lane - j;
                        s_need = need - past;
                        s_in = c[j];
                    }
                    past += c[j];
                }
            }
        }
        __syncthreads();
        const uint64_t from = lo + ((uint64_t)s_bin << shift);
        need = s_need;
        lo = from;
        if ((above - from) >> shift) above = from + ((1ull << shift) - 1);  // (where it is not past `above`: +infinity's key is near 2^64)
        const bool all = s_in == need;
        __syncthreads();
        if (all) {  // the whole range: nothing is left to be told apart
            above = lo - 1;  // (lo > 0: the range above the least score)
            if (lo == 0) above = 0, need = s_in;
            else need = 0;
            break;
        }
    }
    // selected: keys above `above`, and the first `need` of those from lo to it (equal ones). Wave w writes its quarter in order
    const int per = ((n + 255) >> 8) << 6, i0 = w * per, i1 = min(n, i0 + per);
    const bool none = need == 0;
    const auto kind = [&](int i) {  // 2 selected, 1 equal to the least, 0 not
        if (i >= i1) return 0;
        if (i < c0 || i >= c1) return 2;
        const uint64_t k = key[i];
        return k > above ? 2 : !none && k >= lo ? 1 : 0;
    };
    int sure = 0, even = 0;
    for (int i = i0; i < i1; i += 64) {
        const int k = kind(i + lane);
        sure += __popcll(__builtin_amdgcn_ballot_w64(k == 2));
        even += __popcll(__builtin_amdgcn_ballot_w64(k == 1));
    }
    if (lane == 0) {
        s_n[w][0] = sure;
        s_n[w][1] = even;
    }
    __syncthreads();
    int at = 0, ties = 0;  // selected and equal ones before the wave's
    for (int j = 0; j < w; ++j) {
        at += s_n[j][0] + max(0, min(s_n[j][1], need - ties));
        ties += s_n[j][1];
    }
    for (int i = i0; i < i1; i += 64) {
        const int k = kind(i + lane);
        const uint64_t before = (1ull << lane) - 1, eq = __builtin_amdgcn_ballot_w64(k == 1);
        const bool take = k == 2 || (k == 1 && ties + __popcll(eq & before) < need);
        const uint64_t all = __builtin_amdgcn_ballot_w64(take);
        const int to = at + __popcll(all & before);
        if (take && to < a.n_sel) out[to] = i + lane;
        at += __popcll(all);
        ties += __popcll(eq);
    }
}

extern "C" int64_t amv_paged_select_workspace_bytes(const amv_paged_kv* kv, const amv_paged_batch* batch) {
    if (pg_check("amv_paged_select_workspace_bytes", kv, batch, kv ? kv->n_head_kv : 0)) return -1;
    return batch->n_tok * kv->n_head_kv * ((batch->max_kv + kv->page_size - 1) / kv->page_size) * 8;
}

extern "C" int amv_paged_select(const amv_paged_kv* kv, const amv_paged_batch* batch, const float* q, int64_t q_stride,
                                int64_t n_head, int64_t n_sel, int64_t n_first, int64_t n_last, int32_t* sel, void* workspace,
                                int64_t workspace_bytes, void* stream) {
    const char* what = "amv_paged_select";
    if (const int rc = pg_check(what, kv, batch, n_head)) return rc;
    if (batch->n_tok == 0) return AMV_OK;
    AMV_REQUIRE(q && sel, "%s: null pointer", what);
    AMV_REQUIRE(kv->bounds, "%s: the pool has no bounds", what);
    AMV_REQUIRE(q_stride >= n_head * kv->D, "%s: q rows too short", what);
    AMV_REQUIRE(n_first >= 0 && n_last >= 0 && n_sel > 0 && n_first + n_last <= n_sel && n_sel <= PG_MAX_PAGES,
                "%s: %lld pages with the first %lld and the last %lld", what, (long long)n_sel, (long long)n_first, (long long)n_last);
    const int64_t most = (batch->max_kv + kv->page_size - 1) / kv->page_size;
    AMV_REQUIRE(most <= PG_MAX_PAGES, "%s: %lld pages a sequence, more than %d", what, (long long)most, PG_MAX_PAGES);
    const int64_t need = batch->n_tok * kv->n_head_kv * most * 8;
    AMV_REQUIRE(need == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need),
                "%s: workspace of %lld bytes, %lld needed (16-byte aligned)", what, (long long)workspace_bytes, (long long)need);
    AMV_REQUIRE(batch->n_tok * kv->n_head_kv <= PG_MAX_GROUPS, "%s: batch too large", what);
    PgSelect a = {pg_batch(kv, batch), q, (const uint16_t*)kv->bounds, (double*)workspace, sel, q_stride, (int)kv->n_pages,
                  kv->n_head_kv, (int)(n_head / kv->n_head_kv), (int)most, (int)n_sel, (int)n_first, (int)n_last};
    hipStream_t st = amv_stream(stream);
    const unsigned units = (unsigned)(batch->n_tok * kv->n_head_kv);
    if (most > n_sel) {
        const dim3 grid(units, (unsigned)((most + PG_SCORE_PAGES - 1) / PG_SCORE_PAGES));
        if (kv->D == 128) hipLaunchKernelGGL(k_paged_score<128>, grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL(k_paged_score<64>, grid, dim3(256), 0, st, a);
    }
    const size_t lds = (size_t)most * 8;
    if (lds > 60 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k_paged_top), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        AMV_REQUIRE(e == hipSuccess, "%s: %zu bytes of LDS: %s", what, lds, hipGetErrorString(e));
    }
    hipLaunchKernelGGL(k_paged_top, dim3(units), dim3(256), lds, st, a);
    return amv_check_launch(what);
}
