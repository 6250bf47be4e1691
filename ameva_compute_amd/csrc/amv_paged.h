// What the kernels over the paged KV cache share: the layout of a page, the checks of a pool and a batch, and how a workgroup
// finds its part of a ragged batch whose lengths are in device memory.
#pragma once
#include "amv_common.h"

#define PG_MAX_GROUPS (1 << 23)  // workgroups of a launch (of up to 256 threads: a grid has less than 2^32)
#define PG_MAX_PAGES 16384  // pages of one sequence that amv_paged_select ranks (their scores are in LDS, 8 bytes each)

// one key's (or value's) integers and scales in a chunk
template <int TYPE, int D>
struct PgRow {
    static constexpr int NB = D / 32;                                                            // blocks of 32 elements
    static constexpr int ROW = TYPE == AMV_T_F16 ? 2 * D : TYPE == AMV_T_Q8_0 ? D : D / 2;       // bytes of integers (f16)
    static constexpr int SC = TYPE == AMV_T_F16 ? 0 : 2 * NB;                                    // bytes of scales
};

// device view of amv_paged_batch with the lengths made safe: whatever is in device memory, tokens stay inside the n_tok rows and
// keys inside the table's columns
struct PgBatch {
    const int32_t *cu_q, *n_kv, *table;
    int64_t table_stride;
    int n_seq, n_tok, max_kv, pshift;
    __device__ int first(int s) const { return cu_q ? max(0, min(cu_q[s], n_tok)) : s; }
    __device__ int last(int s) const { return cu_q ? max(first(s), min(cu_q[s + 1], n_tok)) : s + 1; }  // one past
    __device__ int end(int s) const { return max(-(1 << 30), min(n_kv[s], 1 << 30)); }  // place behind the last key
    __device__ int keys(int s) const { return max(0, min(n_kv[s], max_kv)); }           // keys there are to see
};

// For work that sequences have count(s) items of: the sequence of item i and the item's index in it, or s = n_seq where there are
// fewer items. Every lane of the wave calls it with the same i; 64 sequences a step.
template <class F>
__device__ __forceinline__ void pg_find(int n_seq, int i, F count, int& s, int& in) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int s0 = 0; s0 < n_seq; s0 += 64) {
        const int mine = s0 + lane < n_seq ? count(s0 + lane) : 0;
        int sum = mine;  // inclusive sums over the lanes
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int up = __shfl_up(sum, o, AMV_WAVE);
            if (lane >= o) sum += up;
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(before + sum > i);
        if (past) {
            const int l = __builtin_ctzll(past);
            s = s0 + l;
            in = i - before - __shfl(sum - mine, l, AMV_WAVE);
            s = __builtin_amdgcn_readfirstlane(s);
            in = __builtin_amdgcn_readfirstlane(in);
            return;
        }
        before += __shfl(sum, 63, AMV_WAVE);
    }
    s = n_seq;
    in = 0;
}

// the sequence that owns token t, or n_seq (rows before the first or behind the last)
__device__ __forceinline__ int pg_seq_of(const PgBatch& b, int t) {
    if (!b.cu_q) return t < b.n_seq ? t : b.n_seq;
    const int lane = threadIdx.x & 63;
    for (int s0 = 0; s0 < b.n_seq; s0 += 64) {
        const int s = min(s0 + lane, b.n_seq - 1);
        const uint64_t in = __builtin_amdgcn_ballot_w64(s0 + lane < b.n_seq && b.first(s) <= t && t < b.last(s));
        if (in) return __builtin_amdgcn_readfirstlane(s0 + __builtin_ctzll(in));
    }
    return b.n_seq;
}

// host
PgBatch pg_batch(const amv_paged_kv* kv, const amv_paged_batch* b);
int pg_check(const char* what, const amv_paged_kv* kv, const amv_paged_batch* b, int64_t n_head);
