// The experts' products with many rows each (prompts): tiles of 64 rows (pairs) of one expert on v_mfma_i32_32x32x32_i8, as
// the dense products of amv_qgemm.hip, with the rows gathered through the plan's order and gate and up side by side.
//
// Operands: A = rows, B = weight rows; lane l has row l % 32 and 16 bytes l / 32 of a 32-block; result D of lane l: weight row
// l % 32, rows 8 (r / 4) + 4 (l / 32) + r % 4. A workgroup's tile is 64 rows x 128 weight rows, a wave's 64 x 32; for gate and up, the
// waves of weight rows take them in turn, so that 64 columns of both meet in the workgroup. Steps of 128 k go from memory to LDS without
// registers, one step ahead; the 16-byte pieces of an LDS row are exchanged by an XOR with the row index on the memory side, so that
// the fragments' reads hit all banks. Rows past the end of a buffer read as zero (the buffers' own range check).
// The work beside the matrix core bounds these kernels where an expert's rows are many: of a 32-block's 32 x 32 integers, each is converted
// and added with its scale (Q4_0, Q8_0; the scale products are one outer product on the matrix core), or multiplied by its unit's scale
// and added up for the super-block (K-quants: a multiplication and an addition per output and unit, of which Q4_K has 8 and Q6_K 16).
// Measured: gate and up of 4096 tokens with 8 of 128 experts of 1024 x 2048 Q4_0 460 us, 600 TFLOP/s (vector instructions 89 % of the
// cycles, the matrix core 29 %, 0.9 GB read), Q4_K 420, Q6_K 570, Q8_0 500; down of the same pairs, 2048 x 1024 Q4_K, 206 us (76 %; 0.5 GB of
// weights read and 0.27 of sums written for the next launch); 1200 pairs of 8 experts of 4096 x 6144 Q4_0 117 us (58 %; 770 workgroups, three a CU,
// so that little follows where one ends). With some 22 rows an expert memory bounds them: 331 tokens with 4 of 60 experts of 1408 x 2048 Q8_0 96 us, 0.42
// GB read for 0.37 of weights; a k of 2080, whose rows begin anywhere in a 128-byte line, so that a step's 128 bytes are parts of two, 0.58 GB, 116 us.
// Not faster: tiles of 128 rows, workgroups that go on to further tiles, a start of k that turns with the workgroup, two sets of waves on halves of
// k (but for a dozen rows an expert). Not tried for Q4_K: unit scales times nibbles as f16 operands (exact, sums of 128 products below 2^24), without
// the multiplication per unit; Q6_K's need more than f16's 11 bits.
#include "amv_moe.h"

#include <type_traits>

typedef int mm_v4i __attribute__((ext_vector_type(4)));
typedef int mm_v16i __attribute__((ext_vector_type(16)));
typedef _Float16 mm_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 mm_h2 __attribute__((ext_vector_type(2)));
typedef float mm_f16v __attribute__((ext_vector_type(16)));
typedef float mm_f32v __attribute__((ext_vector_type(32)));
typedef __attribute__((address_space(3))) void mm_lds;
#define MM_RSRC(p, bytes) __builtin_amdgcn_make_buffer_rsrc((void*)(p), 0, (uint32_t)(bytes), 0x00027000)
// wait for every vector memory load (the other counters are left alone)
#define MM_WAIT_LOADS() __builtin_amdgcn_s_waitcnt(0x0f70)

// 16 bytes a lane from byte `off` of a buffer to LDS, the wave's 64 side by side from `to` on
__device__ __forceinline__ void mm_to_lds(__amdgpu_buffer_rsrc_t from, uint4* to, uint32_t off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (mm_lds*)to, 16, off, 0, 0, 0);
}

#define MM_BM MOE_MANY
#define MM_BN 128  // weight rows of a workgroup (gate and up: 64 of each)

struct MmArgs {
    const uint8_t *w0, *w1;
    int64_t stride;
    int rows, n_k, n_expert, act_div, n_tw;
    const int8_t* aq;       // integers [act_rows][k]
    const uint8_t* meta;    // Q8_0: {d, sum} [act_rows][k / 32]; Q8_K: d [act_rows][k / 256], sums [act_rows][k / 16]
    int64_t act_rows;
    const int2* tiles;
    const int32_t* order;
    float* out;
    AmvActOut q;
};

// what a workgroup works on: its tile of rows and its weight rows; LDS: the rows' pairs
struct MmTile {
    int e, count, n0;  // n0: first weight row (gate and up: of each)
};
template <bool GU>
__device__ __forceinline__ MmTile mm_tile(const MmArgs& p, int* s_pair) {
    // An XCD (workgroup i runs on XCD i % 8) takes every eighth column tile of all row tiles, so the row tiles of an expert read a column
    // tile's weights from one L2; which column tiles these are turns with the expert, as their number need not be a multiple of eight.
    // (A run of tiles for each XCD leaves the last ones idle, where a plan's last tiles are not taken.)
    const int x = blockIdx.x & 7, j = blockIdx.x >> 3, per = (p.n_tw + 7) >> 3;
    MmTile m;
    const int2 t = p.tiles[j / per];
    m.e = t.x & 0xFFFF;
    const int col = 8 * (j % per) + ((x + m.e) & 7);
    m.count = col < p.n_tw ? t.x >> 16 : 0;
    m.n0 = col * (GU ? MM_BN / 2 : MM_BN);
    if (m.count && (int)threadIdx.x < MM_BM) s_pair[threadIdx.x] = p.order[t.y + min((int)threadIdx.x, m.count - 1)];
    return m;
}

// The end of a tile. acc[i][r] of wave wn: row 32 i + 8 (r / 4) + 4 h + r % 4, weight row 32 wn + l % 32.
// Down: stored as they lie, 32 lanes a row's 32 floats. Gate and up: 16 rows at a time through LDS (the first A buffer, free by then),
// where four columns of a row come to a thread: h = silu(g) u, its store and its block's quantization (8 lanes).
template <bool GU>
__device__ __forceinline__ void mm_finish(const MmArgs& p, const MmTile& tile, const int* s_pair, uint4* sA, mm_f16v (&acc)[2], int wn) {
    const int t = threadIdx.x, lane = t & 63, c32 = lane & 31, h = lane >> 5;
    if constexpr (!GU) {
        const int n = tile.n0 + 32 * wn + c32;
        if (n >= p.rows) return;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int m = 32 * i + 8 * (r >> 2) + 4 * h + (r & 3);
                if (m < tile.count) p.out[(int64_t)s_pair[m] * p.rows + n] = acc[i][r];
            }
    } else {
        float* const s = reinterpret_cast<float*>(sA);  // gate [16][64], up [16][64]
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            __syncthreads();
#pragma unroll
            for (int r = 0; r < 8; ++r)
                s[(wn & 1) * 1024 + (8 * (r >> 2) + 4 * h + (r & 3)) * 64 + 32 * (wn >> 1) + c32] = acc[q >> 1][8 * (q & 1) + r];
            __syncthreads();
            const int lr = t >> 4, c = t & 15, m = 16 * q + lr, col = tile.n0 + 4 * c;
            if (m < tile.count && col < p.rows) {  // (eight lanes at a time: columns come in blocks of 32)
                const float4 g = reinterpret_cast<const float4*>(s)[lr * 16 + c], u = reinterpret_cast<const float4*>(s)[256 + lr * 16 + c];
                const float v[4] = {g.x / (1.0f + expf(-g.x)) * u.x, g.y / (1.0f + expf(-g.y)) * u.y, g.z / (1.0f + expf(-g.z)) * u.z,
                                    g.w / (1.0f + expf(-g.w)) * u.w};
                const int64_t pr = s_pair[m];
                if (p.out) *reinterpret_cast<float4*>(p.out + pr * p.rows + col) = make_float4(v[0], v[1], v[2], v[3]);
                if (p.q.type) moe_act_store4(amv_act_row(p.q, pr, p.rows), col / 4, v);
            }
        }
    }
}

// f with the number of 32-row halves of the tile that hold rows: the second half's products are half the work
template <typename F>
__device__ __forceinline__ void mm_halves(const MmTile& tile, F f) {
    if (tile.count > 32) f(std::integral_constant<int, 2>());
    else f(std::integral_constant<int, 1>());
}

// pairs without an expert: zeros from gate and up, nothing from down (their rows are left out of the sum)
template <bool GU>
__device__ __forceinline__ void mm_none(const MmArgs& p, const MmTile& tile, const int* s_pair) {
    if constexpr (GU) {
        const int lane = threadIdx.x & 63;
        for (int m = threadIdx.x >> 6; m < tile.count; m += blockDim.x >> 6)
            if (lane < 16 && tile.n0 + 4 * lane < p.rows) {
                const int64_t pr = s_pair[m];
                const float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (p.out) *reinterpret_cast<float4*>(p.out + pr * p.rows + tile.n0 + 4 * lane) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (p.q.type) moe_act_store4(amv_act_row(p.q, pr, p.rows), tile.n0 / 4 + lane, v);
            }
    }
}

// byte-wise 16 (n - 8) of the nibbles n that are the bytes' high halves (one v_bitop3; n - 8 itself takes two operations more)
__device__ __forceinline__ int mm_m8(uint32_t v) { return (int)((v & 0xF0F0F0F0u) ^ 0x80808080u); }

// Q8_0's integers as floats: the product's C operand is the word of 1 / (2 pi), whose mantissa leaves room for sums of 520192 on both
// sides, so its bits plus the sum are a float of the same binade, and the float less 1 / (2 pi) is 2^-26 times the sum, exactly. A
// subtraction is half of a conversion's time (8 experts of 4096 x 6144, 256 rows each, us: 655 with conversions, 635 so). As it is written here, an
// operand that several products use, the compiler builds it in 16 registers, which Q4_0's kernel does not have at four waves a SIMD
// (it spills; at three waves it loses more than it gains), so Q4_0 converts. The instruction could take 1 / (2 pi) as an inline constant,
// without registers; that is not tried.
#define MM_ORIGIN 0x3E22F983

// ---------------------------------------------------------------------------------------------------------------- Q4_0, Q8_0
template <int WT, bool GU>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4))) void k_moe_many(const MmArgs p) {
    constexpr bool Q4 = WT == AMV_T_Q4_0;
    constexpr int BM = MM_BM, BN = MM_BN, NT = 256;
    constexpr int WB = Q4 ? 16 : 32, WP = 4 * WB / 16;          // bytes of a weight block, 16-byte pieces of a step's row
    constexpr int RA = BM * 8 / NT, RW = BN * WP / NT;          // rounds of the threads over a step's pieces
    constexpr int RDW = BN * 4 / NT;                            // and over its weight scales (its rows': one)
    constexpr int LA = BM * 8, LW = BN * WP;
    // the buffers of even and odd steps are variables of their own: reads of one do not wait for the loads into the other
    __shared__ __align__(16) uint4 sAa[LA], sAb[LA], sWa[LW], sWb[LW];
    __shared__ __align__(16) float sDa[2][4 * BM];
    __shared__ __align__(16) uint16_t sDw[2][4 * BN];  // (f16: three workgroups of Q8_0 on a CU)
    __shared__ int s_pair[BM];
    const MmTile tile = mm_tile<GU>(p, s_pair);
    if (!tile.count) return;
    __syncthreads();
    if (tile.e >= p.n_expert) return mm_none<GU>(p, tile, s_pair);
    const int t = threadIdx.x, lane = t & 63, c32 = lane & 31, h = lane >> 5;
    const int wv = __builtin_amdgcn_readfirstlane(t >> 6), wn = wv;
    const int nb = p.n_k, N = p.rows, nsteps = (nb + 3) / 4;
    const uint32_t K = 32u * nb;

    const uint8_t* const m0 = p.w0 + tile.e * p.stride;
    const uint8_t* const m1 = GU ? p.w1 + tile.e * p.stride : m0;
    const uint32_t wbytes = (uint32_t)N * nb * WB;
    const __amdgpu_buffer_rsrc_t ra = MM_RSRC(p.aq, p.act_rows * K), rw0 = MM_RSRC(m0, wbytes), rw1 = MM_RSRC(m1, wbytes);
    // weight row of a tile's row r (past the last one: none, which reads as zero)
    const auto wrow = [&](int r) { return GU ? tile.n0 + 32 * (r >> 6) + (r & 31) : tile.n0 + r; };
    const bool half_only = tile.count <= 32;  // (the second round loads the second half's rows)
    static_assert(RA == 2, "a round loads half of the rows");
    uint32_t oa[RA], ow[RW];
#pragma unroll
    for (int i = 0; i < RA; ++i)
        oa[i] = (uint32_t)(s_pair[(t >> 3) + NT / 8 * i] / p.act_div) * K + 16 * ((t & 7) ^ ((t >> 4) & 7));
#pragma unroll
    for (int i = 0; i < RW; ++i) {
        const int r = t / WP + NT / WP * i, n = wrow(r);
        ow[i] = n < N ? (uint32_t)n * (nb * WB) + 16 * (Q4 ? (t & 3) ^ ((t >> 4) & 3) : (t & 7) ^ ((t >> 4) & 7)) : 0x80000000u;
    }
    const auto load = [&](uint4* sA, uint4* sW, int b) {
#pragma unroll
        for (int i = 0; i < RA; ++i)
            if (!i || !half_only) mm_to_lds(ra, sA + NT * i + 64 * wv, oa[i] + 32u * b);
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            const bool up = GU && (((NT * i + 64 * wv) / WP) & 32);
            if (up) mm_to_lds(rw1, sW + NT * i + 64 * wv, ow[i] + (uint32_t)WB * b);
            else mm_to_lds(rw0, sW + NT * i + 64 * wv, ow[i] + (uint32_t)WB * b);
        }
    };
    // scales, through registers: row x / 4 of the block x % 4 of the step; 0 past the last block
    const float2* const pda = reinterpret_cast<const float2*>(p.meta) + (int64_t)(s_pair[t >> 2] / p.act_div) * nb;
    float da;
    uint32_t dw[RDW];
    const uint16_t* pdw[RDW];
#pragma unroll
    for (int i = 0; i < RDW; ++i) {
        const int r = (t + NT * i) >> 2, n = min(wrow(r), N - 1);
        const uint16_t* d = reinterpret_cast<const uint16_t*>((GU && (r & 32) ? m1 : m0) + wbytes);
        pdw[i] = Q4 ? d + (size_t)(n >> 1) * nb * 2 + (n & 1) : d + (size_t)n * nb;
    }
    const auto load_s = [&](int b) {
        const int bb = min(b + (t & 3), nb - 1);
        da = pda[bb].x;
#pragma unroll
        for (int i = 0; i < RDW; ++i) dw[i] = pdw[i][Q4 ? 2 * bb : bb];
    };
    const auto store_s = [&](int b, int buf) {
        const bool in = b + (t & 3) < nb;
        sDa[buf][(t & 3) * BM + (t >> 2)] = in ? da : 0.0f;
#pragma unroll
        for (int i = 0; i < RDW; ++i) {
            const int x = t + NT * i;
            sDw[buf][(x & 3) * BN + (x >> 2)] = in ? (uint16_t)dw[i] : (uint16_t)0;
        }
    };

    mm_f16v acc[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = 0.0f;
    const int ar = c32, wr = 32 * wn + c32;
    const int ax = (c32 >> 1) & 7, wx = Q4 ? (c32 >> 2) & 3 : ax;  // the rows' XOR (32 i, 32 wn do not change them)
    const auto compute = [&](auto ni, const uint4* sA, const uint4* sW, int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int bl = 0; bl < 4; ++bl) {
            const mm_f32v zero = {};
            const mm_f32v o = __builtin_amdgcn_mfma_f32_32x32x1f32(sDa[buf][bl * BM + lane], amv_h2f(sDw[buf][bl * BN + wr]), zero, 0, 0, 0);
            mm_v4i B;
            if constexpr (Q4) {  // element e < 16: low nibble of byte e (lane half 0); 16 + e: its high nibble (half 1)
                const uint4 x = sW[wr * 4 + (bl ^ wx)];
                const int s = 4 - 4 * h;
                B = mm_v4i{mm_m8(x.x << s), mm_m8(x.y << s), mm_m8(x.z << s), mm_m8(x.w << s)};
            } else {
                const uint4 x = sW[wr * 8 + ((2 * bl + h) ^ wx)];
                B = mm_v4i{(int)x.x, (int)x.y, (int)x.z, (int)x.w};
            }
#pragma unroll
            for (int i = 0; i < decltype(ni)::value; ++i) {
                const uint4 a = sA[(ar + 32 * i) * 8 + ((2 * bl + h) ^ ax)];
                mm_v16i z;
#pragma unroll
                for (int r = 0; r < 16; ++r) z[r] = Q4 ? 0 : MM_ORIGIN;
                const mm_v16i C = __builtin_amdgcn_mfma_i32_32x32x32_i8(mm_v4i{(int)a.x, (int)a.y, (int)a.z, (int)a.w}, B, z, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    acc[i][r] = fmaf(Q4 ? (float)C[r] : __int_as_float(C[r]) - __int_as_float(MM_ORIGIN), o[16 * i + r], acc[i][r]);
            }
            // one block's results at a time (more do not fit the registers), added up here (the compiler would move the
            // additions behind the next barrier and keep the results until then)
            asm volatile("" : "+v"(acc[0]), "+v"(acc[1]));
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    load(sAa, sWa, 0);
    load_s(0);
    store_s(0, 0);
    MM_WAIT_LOADS();
    __syncthreads();
    const auto steps = [&](auto ni) __attribute__((always_inline)) {
        for (int s = 0;; s += 2) {
            const bool more = s + 1 < nsteps, again = s + 2 < nsteps;
            if (more) {
                load(sAb, sWb, 4 * (s + 1));
                load_s(4 * (s + 1));
            }
            compute(ni, sAa, sWa, 0);
            if (!more) break;
            store_s(4 * (s + 1), 1);
            MM_WAIT_LOADS();
            __syncthreads();
            if (again) {
                load(sAa, sWa, 4 * (s + 2));
                load_s(4 * (s + 2));
            }
            compute(ni, sAb, sWb, 1);
            if (!again) break;
            store_s(4 * (s + 2), 0);
            MM_WAIT_LOADS();
            __syncthreads();
        }
    };
    mm_halves(tile, steps);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] *= Q4 ? 0x1p-4f : 0x1p26f;
    mm_finish<GU>(p, tile, s_pair, sAa, acc, wn);
}

// ---------------------------------------------------------------------------------------------------------------- Q4_K
// Steps of half a super-block. Heads go to LDS with the first half, the activation sums per 16 (as f16, exact) and scales through
// registers; the mins' sum is one f16 matrix product of the units' mins against the sums, exact in f32.
__device__ __forceinline__ uint32_t mm_h2bits(int a, int b) {
    return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)(float)a) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)(float)b) << 16);
}

// (gate and up's form has two registers too few at four waves a SIMD: 12 bytes of scratch a lane)
template <bool GU>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4))) void k_moe_many_q4k(const MmArgs p) {
    constexpr int BM = MM_BM, BN = MM_BN, NT = 256;
    constexpr int RA = BM * 8 / NT, RW = BN * 4 / NT;
    constexpr int LA = BM * 8, LW = BN * 4;
    // the buffers of even and odd steps are variables of their own: reads of one do not wait for the loads into the other
    __shared__ __align__(16) uint4 sAa[LA], sAb[LA], sWa[LW], sWb[LW];
    __shared__ __align__(16) uint4 sHd[BN];
    __shared__ __align__(16) uint2 sBs[BM * 4];
    __shared__ __align__(16) float sDa[BM];
    __shared__ int s_pair[BM];
    const MmTile tile = mm_tile<GU>(p, s_pair);
    if (!tile.count) return;
    __syncthreads();
    if (tile.e >= p.n_expert) return mm_none<GU>(p, tile, s_pair);
    const int t = threadIdx.x, lane = t & 63, c32 = lane & 31, h = lane >> 5;
    const int wv = __builtin_amdgcn_readfirstlane(t >> 6), wn = wv;
    const int nsb = p.n_k, N = p.rows, j_last = nsb - 1;
    const uint32_t K = 256u * nsb;

    const uint8_t* const m0 = p.w0 + tile.e * p.stride;
    const uint8_t* const m1 = GU ? p.w1 + tile.e * p.stride : m0;
    const uint32_t wbytes = (uint32_t)N * nsb * 128;
    const __amdgpu_buffer_rsrc_t ra = MM_RSRC(p.aq, p.act_rows * K);
    const __amdgpu_buffer_rsrc_t rw0 = MM_RSRC(m0, wbytes), rw1 = MM_RSRC(m1, wbytes);
    const __amdgpu_buffer_rsrc_t rh0 = MM_RSRC(m0 + wbytes, N * nsb * 16);
    const auto wrow = [&](int r) { return GU ? tile.n0 + 32 * (r >> 6) + (r & 31) : tile.n0 + r; };
    const bool half_only = tile.count <= 32;  // (the second round loads the second half's rows)
    static_assert(RA == 2, "a round loads half of the rows");
    uint32_t oa[RA], ow[RW];
#pragma unroll
    for (int i = 0; i < RA; ++i)
        oa[i] = (uint32_t)(s_pair[(t >> 3) + NT / 8 * i] / p.act_div) * K + 16 * ((t & 7) ^ ((t >> 4) & 7));
#pragma unroll
    for (int i = 0; i < RW; ++i) {
        const int n = wrow((t >> 2) + NT / 4 * i);
        ow[i] = n < N ? (uint32_t)n * (nsb * 128) + 16 * ((t & 3) ^ ((t >> 4) & 3)) : 0x80000000u;
    }
    const auto load = [&](uint4* sA, uint4* sW, int j, int half) {
#pragma unroll
        for (int i = 0; i < RA; ++i)
            if (!i || !half_only) mm_to_lds(ra, sA + NT * i + 64 * wv, oa[i] + 256u * j + 128 * half);
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            if (GU && (((NT * i + 64 * wv) / 4) & 32))
                mm_to_lds(rw1, sW + NT * i + 64 * wv, ow[i] + 128u * j + 64 * half);
            else
                mm_to_lds(rw0, sW + NT * i + 64 * wv, ow[i] + 128u * j + 64 * half);
        }
    };
    // a row's head is loaded by lane r % 64 of wave r / 64: of gate and up, 32 lanes each
    const int hn = wrow(min(t, BN - 1));
    const uint32_t oh = hn < N ? (uint32_t)hn * (nsb * 16) : 0x80000000u;
    const uint8_t* const ph = (GU && (t & 32) ? m1 : m0) + wbytes;
    const auto load_head = [&](int j) {
        if (wv < BN / 64) {
            if constexpr (GU) sHd[t] = hn < N ? *reinterpret_cast<const uint4*>(ph + oh + 16 * j) : make_uint4(0, 0, 0, 0);
            else mm_to_lds(rh0, sHd + 64 * wv, oh + 16u * j);
        }
    };
    // activation sums (thread: row t / 4, 4 of the 16) and scale of super-block j, through registers
    const uint8_t* const sums = p.meta + p.act_rows * nsb * 4;
    const uint32_t os = (uint32_t)(s_pair[t >> 2] / p.act_div) * (nsb * 64) + 16 * (t & 3), od = (uint32_t)(s_pair[min(t, BM - 1)] / p.act_div) * (nsb * 4);
    moe_i4 bs;
    float da0;
    const auto load_sb = [&](int j) {
        bs = *reinterpret_cast<const moe_i4*>(sums + (os + 64u * j));
        da0 = *reinterpret_cast<const float*>(p.meta + (od + 4u * j));
    };
    const auto store_sb = [&]() {
        sBs[t] = make_uint2(mm_h2bits(bs.x, bs.y), mm_h2bits(bs.z, bs.w));
        if (t < BM) sDa[t] = da0;
    };

    mm_f16v acc[2];
    mm_v16i I1[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = 0.0f;
    const int ar = c32, wr = 32 * wn + c32;
    const int ax = (c32 >> 1) & 7, wx = (c32 >> 2) & 3;
    const auto half_step = [&](auto ni, const uint4* sA, const uint4* sW, uint32_t scw, bool first) __attribute__((always_inline)) {
#pragma unroll
        for (int cp = 0; cp < 2; ++cp) {
            const uint4 x = sW[wr * 4 + ((2 * cp + h) ^ wx)];
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const int u = 2 * cp + v, s = 4 * v;
                const mm_v4i B = mm_v4i{(int)((x.x >> s) & 0x0F0F0F0Fu), (int)((x.y >> s) & 0x0F0F0F0Fu), (int)((x.z >> s) & 0x0F0F0F0Fu),
                                        (int)((x.w >> s) & 0x0F0F0F0Fu)};
                const int sc = (int)((scw >> (8 * u)) & 0xFFu);
#pragma unroll
                for (int i = 0; i < decltype(ni)::value; ++i) {
                    const uint4 a = sA[(ar + 32 * i) * 8 + ((2 * u + h) ^ ax)];
                    const mm_v16i z = {};
                    const mm_v16i C = __builtin_amdgcn_mfma_i32_32x32x32_i8(mm_v4i{(int)a.x, (int)a.y, (int)a.z, (int)a.w}, B, z, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 16; ++r) I1[i][r] = first && u == 0 ? __mul24(C[r], sc) : I1[i][r] + __mul24(C[r], sc);
                }
                asm volatile("" : "+v"(I1[0]), "+v"(I1[1]));  // (as in k_moe_many)
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };

    load_head(0);
    load(sAa, sWa, 0, 0);
    MM_WAIT_LOADS();
    __syncthreads();
    const auto steps = [&](auto ni) __attribute__((always_inline)) {
        for (int j = 0; j < nsb; ++j) {
            const int jn = min(j + 1, j_last);
            load(sAb, sWb, j, 1);
            load_sb(j);
            const uint4 hd = sHd[wr];
            // scales and mins of units 0-3 and 4-7, one per byte
            const uint32_t sc0 = hd.y & 0x3F3F3F3Fu, sc1 = (hd.w & 0x0F0F0F0Fu) | ((hd.y >> 2) & 0x30303030u);
            const uint32_t mw = h ? ((hd.w >> 4) & 0x0F0F0F0Fu) | ((hd.z >> 2) & 0x30303030u) : hd.z & 0x3F3F3F3Fu;
            half_step(ni, sAa, sWa, sc0, true);
            store_sb();
            MM_WAIT_LOADS();
            __syncthreads();
            load(sAa, sWa, jn, 0);
            load_head(jn);
            half_step(ni, sAb, sWb, sc1, false);
            // the mins, each on its unit's two 16-sum slots, against the sums
            mm_h8 Bmn;
            {
                const uint32_t off = 0xE400E400u;  // -1024, -1024: 0x6400 | m is the f16 1024 + m
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t q = __builtin_amdgcn_perm(0x64646464u, mw, 0x04000400u + 0x00010001u * e);
                    const mm_h2 v = __builtin_bit_cast(mm_h2, q) + __builtin_bit_cast(mm_h2, off);
                    Bmn[2 * e] = v.x;
                    Bmn[2 * e + 1] = v.y;
                }
            }
            const float d = amv_h2f(hd.x), dm = amv_h2f(hd.x >> 16);
#pragma unroll
            for (int i = 0; i < decltype(ni)::value; ++i) {
                const int tl = 32 * i;
                const mm_h8 Abs = *reinterpret_cast<const mm_h8*>(&sBs[(tl + c32) * 4 + 2 * h]);
                const mm_f16v zf = {};
                const mm_f16v I2 = __builtin_amdgcn_mfma_f32_32x32x16_f16(Abs, Bmn, zf, 0, 0, 0);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float4 v = *reinterpret_cast<const float4*>(&sDa[tl + 4 * h + 8 * q]);
                    const float da[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        acc[i][4 * q + r] = fmaf(fmaf(d, (float)I1[i][4 * q + r], -(dm * I2[4 * q + r])), da[r], acc[i][4 * q + r]);
                }
            }
            MM_WAIT_LOADS();
            __syncthreads();
        }
    };
    mm_halves(tile, steps);
    mm_finish<GU>(p, tile, s_pair, sAa, acc, wn);
}

// ---------------------------------------------------------------------------------------------------------------- Q6_K
// Steps of half a super-block: elements 128 n + {l, 32 + l, 64 + l, 96 + l} (l < 32) from the low nibbles of ql[l], ql[32 + l], then the
// high ones, with bits 0-1, 2-3, 4-5, 6-7 of qh[l]; sub-blocks of 16 have scales of their own, so the matrix core takes 16 k at a time
// (v_mfma_i32_32x32x16_i8, lane half h the bytes 8 h .. 8 h + 7 of a sub-block).
template <bool GU>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3))) void k_moe_many_q6k(const MmArgs p) {
    constexpr int BM = MM_BM, BN = MM_BN, NT = 256;
    constexpr int RA = BM * 8 / NT, RW = BN * 4 / NT;
    constexpr int LA = BM * 8, LW = BN * 4, LH = BN * 2;
    // the buffers of even and odd steps are variables of their own: reads of one do not wait for the loads into the other
    __shared__ __align__(16) uint4 sAa[LA], sAb[LA], sWa[LW], sWb[LW], sHa[LH], sHb[LH];
    __shared__ __align__(16) uint4 sSc[2][BN];
    __shared__ __align__(16) float sD[2][BN], sDa[2][BM];
    __shared__ int s_pair[BM];
    const MmTile tile = mm_tile<GU>(p, s_pair);
    if (!tile.count) return;
    __syncthreads();
    if (tile.e >= p.n_expert) return mm_none<GU>(p, tile, s_pair);
    const int t = threadIdx.x, lane = t & 63, c32 = lane & 31, h = lane >> 5;
    const int wv = __builtin_amdgcn_readfirstlane(t >> 6), wn = wv;
    const int nsb = p.n_k, N = p.rows, j_last = nsb - 1;
    const uint32_t K = 256u * nsb;

    const uint8_t* const m0 = p.w0 + tile.e * p.stride;
    const uint8_t* const m1 = GU ? p.w1 + tile.e * p.stride : m0;
    const uint32_t nblk = (uint32_t)N * nsb;
    const __amdgpu_buffer_rsrc_t ra = MM_RSRC(p.aq, p.act_rows * K);
    const __amdgpu_buffer_rsrc_t rw0 = MM_RSRC(m0, nblk * 128), rw1 = MM_RSRC(m1, nblk * 128);
    const __amdgpu_buffer_rsrc_t rq0 = MM_RSRC(m0 + nblk * 128, nblk * 64), rq1 = MM_RSRC(m1 + nblk * 128, nblk * 64);
    const auto wrow = [&](int r) { return GU ? tile.n0 + 32 * (r >> 6) + (r & 31) : tile.n0 + r; };
    const bool half_only = tile.count <= 32;  // (the second round loads the second half's rows)
    static_assert(RA == 2, "a round loads half of the rows");
    uint32_t oa[RA], ow[RW];
#pragma unroll
    for (int i = 0; i < RA; ++i)
        oa[i] = (uint32_t)(s_pair[(t >> 3) + NT / 8 * i] / p.act_div) * K + 16 * ((t & 7) ^ ((t >> 4) & 7));
#pragma unroll
    for (int i = 0; i < RW; ++i) {
        const int n = wrow((t >> 2) + NT / 4 * i);
        ow[i] = n < N ? (uint32_t)n * (nsb * 128) + 16 * ((t & 3) ^ ((t >> 4) & 3)) : 0x80000000u;
    }
    // qh: two pieces a row, the first 2 BN threads
    const int qn = wrow(min(t >> 1, BN - 1));
    const uint32_t oq = qn < N ? (uint32_t)qn * (nsb * 64) + 16 * ((t & 1) ^ ((t >> 3) & 1)) : 0x80000000u;
    const auto load = [&](uint4* sA, uint4* sW, uint4* sH, int j, int half) {
#pragma unroll
        for (int i = 0; i < RA; ++i)
            if (!i || !half_only) mm_to_lds(ra, sA + NT * i + 64 * wv, oa[i] + 256u * j + 128 * half);
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            if (GU && (((NT * i + 64 * wv) / 4) & 32))
                mm_to_lds(rw1, sW + NT * i + 64 * wv, ow[i] + 128u * j + 64 * half);
            else
                mm_to_lds(rw0, sW + NT * i + 64 * wv, ow[i] + 128u * j + 64 * half);
        }
        if (wv < BN * 2 / 64) {
            if (GU && (wv & 1)) mm_to_lds(rq1, sH + 64 * wv, oq + 64u * j + 32 * half);
            else mm_to_lds(rq0, sH + 64 * wv, oq + 64u * j + 32 * half);
        }
    };
    // scales of super-block j: 16 bytes and d of the first BN threads' weight rows, d of the first BM threads' rows, through registers
    const int sr = min(t, BN - 1), sn = min(wrow(sr), N - 1);
    const uint8_t* const ms = GU && (sr & 32) ? m1 : m0;
    const uint4* const psc = reinterpret_cast<const uint4*>(ms + (size_t)nblk * 192) + (size_t)sn * nsb;
    const uint16_t* const pd = reinterpret_cast<const uint16_t*>(ms + (size_t)nblk * 208) + (size_t)sn * nsb;
    const float* const pda = reinterpret_cast<const float*>(p.meta) + (int64_t)(s_pair[min(t, BM - 1)] / p.act_div) * nsb;
    uint4 scr;
    uint32_t dr;
    float dar;
    const auto load_sb = [&](int j) {
        scr = psc[j];
        dr = pd[j];
        dar = pda[j];
    };
    const auto store_sb = [&](int buf) {
        if (t < BN) {
            sSc[buf][t] = scr;
            sD[buf][t] = 0.25f * amv_h2f(dr);  // (the integers are four times q - 32)
        }
        if (t < BM) sDa[buf][t] = dar;
    };

    mm_f16v acc[2];
    mm_v16i I[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            acc[i][r] = 0.0f;
            I[i][r] = 0;
        }
    const int ar = c32, wr = 32 * wn + c32;
    const int ax = (c32 >> 1) & 7, wx = (c32 >> 2) & 3, hx = (c32 >> 2) & 1;
    // sw: the half's eight scales (bytes 2 e + pp: sub-block of elements 32 e + 16 pp ..)
    const auto half_step = [&](auto ni, const uint4* sA, const uint4* sW, const uint4* sH, uint32_t s0, uint32_t s1) __attribute__((always_inline)) {
#pragma unroll
        for (int pp = 0; pp < 2; ++pp) {
            const uint2 l0 = reinterpret_cast<const uint2*>(sW + wr * 4 + (pp ^ wx))[h];
            const uint2 l1 = reinterpret_cast<const uint2*>(sW + wr * 4 + ((2 + pp) ^ wx))[h];
            uint2 qh = reinterpret_cast<const uint2*>(sH + wr * 2 + (pp ^ hx))[h];
            qh = make_uint2(qh.x ^ 0xAAAAAAAAu, qh.y ^ 0xAAAAAAAAu);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint2 l = e & 1 ? l1 : l0;
                // 4 (q - 32): the six bits at the byte's top, the highest one turned over (above, for all e)
                const auto q6 = [&](uint32_t lo, uint32_t hi) {
                    return ((e < 2 ? lo << 2 : lo >> 2) & 0x3C3C3C3Cu) | ((hi << (6 - 2 * e)) & 0xC0C0C0C0u);
                };
                const uint2 b = make_uint2(q6(l.x, qh.x), q6(l.y, qh.y));
                const int sub = 2 * e + pp, sc = (int)(int8_t)((sub < 4 ? s0 : s1) >> (8 * (sub & 3)));
#pragma unroll
                for (int i = 0; i < decltype(ni)::value; ++i) {
                    const uint2 a = reinterpret_cast<const uint2*>(sA + (ar + 32 * i) * 8 + ((2 * e + pp) ^ ax))[h];
                    const mm_v16i z = {};
                    const mm_v16i C = __builtin_amdgcn_mfma_i32_32x32x16_i8(__builtin_bit_cast(long, a), __builtin_bit_cast(long, b), z, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 16; ++r) I[i][r] += __mul24(C[r], sc);
                }
                asm volatile("" : "+v"(I[0]), "+v"(I[1]));  // (as in k_moe_many)
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };

    load(sAa, sWa, sHa, 0, 0);
    load_sb(0);
    store_sb(0);
    MM_WAIT_LOADS();
    __syncthreads();
    const auto steps = [&](auto ni) __attribute__((always_inline)) {
        for (int j = 0; j < nsb; ++j) {
            const int jn = min(j + 1, j_last), buf = j & 1;
            load(sAb, sWb, sHb, j, 1);
            load_sb(jn);
            const uint4 sc = sSc[buf][wr];
            half_step(ni, sAa, sWa, sHa, sc.x, sc.y);
            store_sb(buf ^ 1);
            MM_WAIT_LOADS();
            __syncthreads();
            load(sAa, sWa, sHa, jn, 0);
            half_step(ni, sAb, sWb, sHb, sc.z, sc.w);
            const float d = sD[buf][wr];
#pragma unroll
            for (int i = 0; i < decltype(ni)::value; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float4 v = *reinterpret_cast<const float4*>(&sDa[buf][32 * i + 4 * h + 8 * q]);
                    const float da[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        acc[i][4 * q + r] = fmaf(d * da[r], (float)I[i][4 * q + r], acc[i][4 * q + r]);
                        I[i][4 * q + r] = 0;
                    }
                }
            MM_WAIT_LOADS();
            __syncthreads();
        }
    };
    mm_halves(tile, steps);
    mm_finish<GU>(p, tile, s_pair, sAa, acc, wn);
}

// ---------------------------------------------------------------------------------------------------------------- host
int moe_many(const MoeProduct& p) {
    const int64_t pairs = p.n_tok * p.n_used;
    const MoePlanView v = moe_plan_view(p.plan, pairs, p.n_expert);
    const bool kq = p.type == AMV_T_Q4_K || p.type == AMV_T_Q6_K, gu = p.w1 != nullptr;
    const int8_t* aq = (const int8_t*)p.act;
    MmArgs a{(const uint8_t*)p.w0, (const uint8_t*)p.w1, p.stride, (int)p.rows, (int)(p.k / (kq ? 256 : 32)), p.n_expert, gu ? p.n_used : 1,
             0, aq, (const uint8_t*)aq + p.act_rows * p.k, p.act_rows, v.many, v.order, p.out, p.q};
    a.n_tw = (int)((p.rows + (gu ? MM_BN / 2 : MM_BN) - 1) / (gu ? MM_BN / 2 : MM_BN));
    const int64_t wgs = (int64_t)((a.n_tw + 7) / 8 * 8) * v.n_many;
    AMV_REQUIRE(wgs < 1 << 24, "moe: %d tiles of %lld columns are too many", v.n_many, (long long)p.rows);
    const unsigned grid = (unsigned)wgs;
#define GO(GATE_UP, DOWN) hipLaunchKernelGGL((gu ? GATE_UP : DOWN), dim3(grid), dim3(256), 0, p.st, a)
    if (p.type == AMV_T_Q4_0) GO((k_moe_many<AMV_T_Q4_0, true>), (k_moe_many<AMV_T_Q4_0, false>));
    else if (p.type == AMV_T_Q8_0) GO((k_moe_many<AMV_T_Q8_0, true>), (k_moe_many<AMV_T_Q8_0, false>));
    else if (p.type == AMV_T_Q4_K) GO(k_moe_many_q4k<true>, k_moe_many_q4k<false>);
    else GO(k_moe_many_q6k<true>, k_moe_many_q6k<false>);
#undef GO
    return amv_check_launch("amv_moe products");
}
