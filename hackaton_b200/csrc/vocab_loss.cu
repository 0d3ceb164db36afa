// Softmax cross-entropy over the vocabulary straight from the hidden states, in pieces of the vocabulary: the logits
// l = h . w_v exist only in tensor memory, a tile at a time, and of the softmax there is one piece at a time.
//   forward    lse = log sum_v exp(l_v),  loss = lse - l_t = log(1 + sum_{v != t} exp(l_v - l_t))
//   backward   with b = d loss, c = d lse:  dl_v = (b + c) p_v - b [v = t];  dH = dl . W,  dW = dl^T . H
// Rows whose target is negative take no part: the others are gathered first, everything behind that works on as many
// rows as there are (the count stays on the device), and what an ignored row holds is never read.
//
// dH is linear in two things that the forward knows up to a row's factors:
//   dH = (b + c) U + (c p_t - b (1 - p_t)) w_t,   U = sum_{v != t} p_v w_v
// so the forward forms U in the same sweep over the vocabulary as the statistics, two matrix products of 2 R V K
// operations (R rows, V words, K features) instead of three: a piece's exponentials are taken relative to a reference
// per row that is fixed before the sweep (from the first words and the target's own logit), and the sum's 1 / s comes
// at the end. The target is left out of U and of the sums, so that 1 - p_t and a loss near zero keep their digits, and its
// share is added in fp32. A row that meets a logit too far above its reference for the 16-bit type has its piece done
// again with a new one (its sums so far scaled by a power of two); launches for that look at a flag and leave. dW needs
// the final lse: the logits once more, in 16-bit dl this time, and one product.
//
// All products run in one kernel, vl_gemm_kernel, in modes that differ in the operands' layouts and the epilogue; it
// is bound by the tensor cores. CTA pairs (tcgen05.mma.cta_group::2) own a 256 x 256 tile, 128 rows by 256 columns of
// fp32 in each CTA's tensor memory, twice: while eight warps work on one tile's values the next one is being
// multiplied. Operands come by TMA in 64-deep steps through a ring of six. The 16-bit piece is laid out in blocks of
// [rows][64 words], which is how TMA reads it along either side, and its size is chosen on the device: whole waves of
// tiles for the rows there are, within a buffer that stays in L2.
// Nothing is added atomically: results do not depend on timing.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "kernels.h"
#include "ptx.cuh"

namespace nf4 {

constexpr float VL_LOG2E = 1.4426950408889634f;
constexpr float VL_LN2 = 0.6931471805599453f;
constexpr float VL_NEG = -1.0e30f;         // a finite "minus infinity"
constexpr float VL_P_SCALE = 8192.f;       // of the 16-bit gradient: below 4 * 2^13, down to 2^-24 / 2^13
// A row's reference for its exponentials (base 2): the larger of the first words' maximum less VL_BELOW and the
// target's logit less VL_BELOW_TARGET; fp16 takes what lies up to 2^15 above it, bf16 2^100.
constexpr float VL_BELOW = 3.f, VL_BELOW_TARGET = 10.f;
constexpr float VL_ROOM_F16 = 15.f, VL_ROOM_BF16 = 100.f;
constexpr int VL_PROBE_TILES = 8;          // tiles of words that the reference is taken from
constexpr int VL_PIECE_UNITS = 512;        // tiles of 256 x 256 that a piece may have: 64 MiB

constexpr int VL_TILE = 256;               // rows and columns of a pair's tile
constexpr int VL_BK = 64;
constexpr int VL_EPI_WARPS = 8;
constexpr int VL_SMEM_MAX = 232448;
// Shared memory of a CTA: the ring (128 rows of A and ROWS of B per step), a box of 32 rows x 128 bytes per epilogue warp
// on its way out (OUT), barriers.
template <int ROWS, int STAGES_, bool OUT>
struct VlSmem {
    static constexpr int STAGES = STAGES_;
    static constexpr int A_BYTES = 128 * VL_BK * 2, B_BYTES = ROWS * VL_BK * 2;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int STAGING_OFF = STAGES * STAGE_BYTES;
    static constexpr int BAR_OFF = STAGING_OFF + (OUT ? VL_EPI_WARPS * 4096 : 0);
    static constexpr int TOTAL = BAR_OFF + 8 * (3 * STAGES + 4) + 8 + 1024;    // + slack for 1024-byte alignment
    static_assert(TOTAL <= VL_SMEM_MAX && BAR_OFF % 8 == 0, "exceeds the 227 KB of shared memory per CTA");
};
constexpr int VL_THREADS = 64 + VL_EPI_WARPS * 32;

enum VlMode {
    VL_STATS = 0,    // A = gathered rows [R, K], B = W [V, K]                -> maximum and sum per row and half tile
    VL_SOFT = 1,     // the same operands, one piece                          -> exponentials in 16 bits, the same statistics
    VL_GRAD = 2,     // the same                                              -> dl in 16 bits
    VL_HIDDEN = 3,   // A = the piece [R, words], B = its rows of W, N along K   -> fp32 planes [slices][R, K]
    VL_WEIGHT = 4,   // A = the piece transposed, B = gathered rows, N along K   -> 16-bit dW rows of the piece
    VL_FEW = 5       // A = W, B = at most 64 gathered rows, words as M                 -> maximum and sum per row and warp
};

struct VlMaps {
    CUtensorMap a, b, c;     // c: where the epilogue's boxes go (not VL_STATS)
};

struct VlParams {
    const int* count;        // rows that take part
    int* status;
    int bf16;
    int vocab, hidden;
    int word_tiles;          // of the whole vocabulary (VL_STATS: of what is to be looked at)
    int index;               // of the piece
    int capacity;            // tiles that a piece may have
    int slots;               // pairs that pieces and slices are planned for
    int n_rows;              // VL_FEW: columns of the accumulator, 32 or 64
    const int* target;       // per gathered row
    // VL_STATS, VL_SOFT
    float2* parts;           // [2 * word tiles][rows_pad]: maximum (base 2), sum (relative to it; VL_SOFT: to the reference)
    long long rows_pad;
    // VL_SOFT, VL_HIDDEN
    float* refs;             // [pieces + 1][rows_pad]: a row's reference before each piece and after the last
    int* flags;              // [pieces][1 + row tiles]: whether any row, and which tiles' rows, need the piece again
    int flags_pitch;
    int again;               // VL_SOFT: this launch does flagged pieces again
    // VL_GRAD
    const float* lse2;
    const float* rest;       // 1 - p of the target
    const float4* coef;      // ((b + c), b, c) over the common power of two, times VL_P_SCALE
    // VL_SOFT, VL_GRAD: the 16-bit piece, [block of 64 words][rows of the tiles][64]
    void* piece;
    // VL_HIDDEN
    float* planes;           // [slices][rows of the tiles][hidden]
    // VL_WEIGHT
    void* d_weight;          // [vocab, hidden]
    const float* weight_scale;
};

__host__ __device__ inline int vl_div_up(int a, int b) { return (a + b - 1) / b; }

// Tiles of words in a piece: what the buffer holds for so many row tiles, cut to whole waves of the pairs.
__host__ __device__ inline int vl_piece_tiles(int row_tiles, int word_tiles, int capacity, int slots) {
    int t = capacity / row_tiles;
    if (t >= word_tiles) return word_tiles;
    const int waves = row_tiles * t / slots;
    if (waves > 0) t = waves * slots / row_tiles;
    return t > 0 ? t : 1;
}

// Slices of a piece's words for U: as many as keep the pairs busiest, with at least eight steps each; none is empty.
constexpr int VL_MAX_SLICES = 16;
__host__ __device__ inline int vl_slices(int tiles, int steps, int slots) {
    int best = 1, best_cost = 0x7FFFFFFF;
    for (int s = 1; s <= VL_MAX_SLICES && (s == 1 || steps / s >= 8); ++s) {
        const int per = vl_div_up(steps, s);
        const int cost = vl_div_up(tiles * vl_div_up(steps, per), slots) * (per + 6);
        if (cost < best_cost) { best_cost = cost; best = s; }
    }
    return vl_div_up(steps, vl_div_up(steps, best));
}

__device__ __forceinline__ float vl_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t vl_pack(float a, float b, int bf16) {
    if (bf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void vl_sts128(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

struct VlPlan {      // what a launch's units are, from the device's row count
    int rows, row_tiles, v0, tiles;            // first word and tiles of the piece
    int m_tiles, units, steps, slices, per_slice;
};

template <int MODE>
__device__ __forceinline__ VlPlan vl_plan(const VlParams& p, int rows) {
    VlPlan w;
    w.rows = rows;
    w.row_tiles = vl_div_up(rows, VL_TILE);
    w.slices = 1;
    const int feature_tiles = vl_div_up(p.hidden, VL_TILE);
    w.v0 = 0;
    w.tiles = p.word_tiles;
    int first_tiles = p.word_tiles;
    if (MODE != VL_STATS && MODE != VL_FEW) {
        first_tiles = vl_piece_tiles(max(w.row_tiles, 1), p.word_tiles, p.capacity, p.slots);
        const int before = min((long long)first_tiles * p.index, (long long)p.word_tiles);
        w.v0 = before * VL_TILE;
        w.tiles = min(first_tiles, p.word_tiles - before);
    }
    if (MODE == VL_WEIGHT) {
        w.m_tiles = w.tiles;
        w.steps = vl_div_up(rows, VL_BK);
        w.units = w.tiles * feature_tiles;
    } else if (MODE == VL_HIDDEN) {
        w.m_tiles = w.row_tiles;
        w.steps = w.tiles * (VL_TILE / VL_BK);
        const int tiles = w.row_tiles * feature_tiles;
        if (rows > 0) w.slices = vl_slices(tiles, first_tiles * (VL_TILE / VL_BK), p.slots);
        w.units = w.tiles > 0 ? tiles * w.slices : 0;
    } else if (MODE == VL_FEW) {
        w.m_tiles = w.tiles;
        w.steps = vl_div_up(p.hidden, VL_BK);
        w.units = rows > 0 ? w.tiles : 0;
    } else {
        w.m_tiles = w.row_tiles;
        w.steps = vl_div_up(p.hidden, VL_BK);
        w.units = w.row_tiles * w.tiles;
    }
    w.per_slice = vl_div_up(w.steps, w.slices);
    return w;
}

template <int MODE>
using VlSmemOf = VlSmem<MODE == VL_FEW ? 32 : 128, MODE == VL_FEW ? 11 : MODE == VL_STATS ? 7 : 6, MODE != VL_STATS && MODE != VL_FEW>;

struct VlUnit {
    int mt, nt, slice, begin, steps;
};

template <int MODE>
__device__ __forceinline__ VlUnit vl_unit(int u, const VlPlan& w) {
    VlUnit r;
    r.slice = 0;
    if (MODE == VL_HIDDEN) {       // slices outermost: the units of a wave read the same words
        const int tiles = w.units / w.slices;
        r.slice = u / tiles;
        u -= r.slice * tiles;
    }
    r.mt = u % w.m_tiles;
    r.nt = u / w.m_tiles;
    r.begin = r.slice * w.per_slice;
    r.steps = min(w.per_slice, w.steps - r.begin);
    return r;
}

template <int MODE>
__global__ void __launch_bounds__(VL_THREADS, 1)
vl_gemm_kernel(const __grid_constant__ VlMaps maps, const __grid_constant__ VlParams p) {
    constexpr bool A_MN = MODE == VL_WEIGHT, B_MN = MODE == VL_HIDDEN || MODE == VL_WEIGHT;
    constexpr bool A_PIECE = MODE == VL_HIDDEN || MODE == VL_WEIGHT;      // A comes from the 16-bit piece
    using L = VlSmemOf<MODE>;
    constexpr int STAGES = L::STAGES;
    extern __shared__ uint8_t vl_smem[];
    const uint32_t base = (smem_u32(vl_smem) + 1023u) & ~1023u;
    uint8_t* gen = vl_smem + (base - smem_u32(vl_smem));
    const uint32_t bar = base + L::BAR_OFF;
    auto bar_full = [&](int s) { return bar + 8u * s; };                        // leader: both CTAs' operands
    auto bar_landed = [&](int s) { return bar + 8u * (STAGES + s); };        // peer: its own
    auto bar_empty = [&](int s) { return bar + 8u * (2 * STAGES + s); };
    auto bar_done = [&](int b) { return bar + 8u * (3 * STAGES + b); };      // accumulator complete
    auto bar_drained = [&](int b) { return bar + 8u * (3 * STAGES + 2 + b); };
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + L::BAR_OFF + 8 * (3 * STAGES + 4));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + L::BAR_OFF + 8 * (3 * STAGES + 4) + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int pair = (int)(blockIdx.x >> 1), pairs = (int)(gridDim.x >> 1);
    const int* flags = p.flags + (long long)p.index * p.flags_pitch;
    if (MODE == VL_SOFT && p.again) {     // nearly always there is nothing to do again
        grid_dep_wait();
        if (flags[0] == 0) return;
    }

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(bar_full(s), 2);       // the leader's expect_tx and the peer's word that its share is there
            mbar_init(bar_landed(s), 1);
            mbar_init(bar_empty(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(bar_done(b), 1);
            mbar_init(bar_drained(b), 2 * VL_EPI_WARPS);
        }
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&maps.a);
        tma_prefetch_desc(&maps.b);
        if (MODE != VL_STATS) tma_prefetch_desc(&maps.c);
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
        tmem_relinquish_pair();
    }
    grid_dep_wait();
    grid_dep_launch();
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    const int rows = *p.count;
    const VlPlan plan = vl_plan<MODE>(p, rows);
    const int rows_dev = plan.row_tiles * VL_TILE;
    // (what all roles leave out: slices that the last piece has no steps for, row tiles that need not be done again)
    const auto skip = [&](const VlUnit& w) {
        return w.steps <= 0 || (MODE == VL_SOFT && p.again && flags[1 + w.mt] == 0);
    };
    int fail = 0;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t g = 0;
            for (int u = pair; u < plan.units && !fail; u += pairs) {
                const VlUnit w = vl_unit<MODE>(u, plan);
                if (skip(w)) continue;
                for (int it = 0; it < w.steps; ++it, ++g) {
                    const int s = (int)(g % STAGES);
                    const uint32_t ph = (g / STAGES) & 1u;
                    if (!mbar_wait_cluster(bar_empty(s), ph ^ 1u, abort_flag)) { fail = 1; break; }
                    const uint32_t landed = rank == 0 ? bar_full(s) : bar_landed(s);
                    const uint32_t sa = base + (uint32_t)s * L::STAGE_BYTES, sb = sa + L::A_BYTES;
                    const int k = (w.begin + it) * VL_BK;
                    const int am = w.mt * VL_TILE + (int)rank * 128;
                    const int bn = MODE == VL_FEW ? (int)rank * (p.n_rows / 2) : w.nt * VL_TILE + (int)rank * 128;
                    mbar_arrive_expect_tx(landed, L::A_BYTES + (MODE == VL_FEW ? p.n_rows * 64 : L::B_BYTES));
                    if (A_MN) {             // words as M, rows as steps
                        tma_load_2d(sa, &maps.a, 0, (am >> 6) * rows_dev + k, landed);
                        tma_load_2d(sa + 8192, &maps.a, 0, ((am >> 6) + 1) * rows_dev + k, landed);
                    } else if (A_PIECE) {   // rows as M, words as steps
                        tma_load_2d(sa, &maps.a, 0, (k >> 6) * rows_dev + am, landed);
                    } else {
                        tma_load_2d(sa, &maps.a, k, am, landed);
                    }
                    if (B_MN) {     // VL_HIDDEN: rows of W from the piece's first word on; VL_WEIGHT: gathered rows
                        const int y = MODE == VL_HIDDEN ? plan.v0 + k : k;
                        tma_load_2d(sb, &maps.b, bn, y, landed);
                        tma_load_2d(sb + 8192, &maps.b, bn + 64, y, landed);
                    } else {
                        tma_load_2d(sb, &maps.b, k, plan.v0 + bn, landed);
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            // tcgen05 descriptors: K-major tiles are rows of 128 bytes, eight rows 1024 bytes apart; MN-major ones 64 steps
            // of 128 bytes (64 values along M or N), the next 64 values 8192 bytes on
            constexpr uint64_t K_MAJOR = make_smem_desc(0, 16, 1024, LAYOUT_SW128);
            constexpr uint64_t MN_MAJOR = make_smem_desc(0, 8192, 1024, LAYOUT_SW128);
            constexpr uint64_t A_DESC = A_MN ? MN_MAJOR : K_MAJOR, B_DESC = B_MN ? MN_MAJOR : K_MAJOR;
            constexpr uint32_t A_STEP = (A_MN ? 16 * 128 : 32) >> 4, B_STEP = (B_MN ? 16 * 128 : 32) >> 4;
            const uint32_t idesc = make_idesc_f16(MODE == VL_FEW ? (uint32_t)p.n_rows : VL_TILE, A_MN ? 1u : 0u, B_MN ? 1u : 0u, VL_TILE) |
                                   (p.bf16 ? (1u << 7) | (1u << 10) : 0u);
            const uint32_t base4 = (base & 0x3FFFFu) >> 4;
            uint32_t g = 0, n = 0;
            for (int u = pair; u < plan.units && !fail; u += pairs) {
                const VlUnit w = vl_unit<MODE>(u, plan);
                if (skip(w)) continue;
                const int b = (int)(n & 1u);
                if (!mbar_wait_cluster(bar_drained(b), ((n >> 1) & 1u) ^ 1u, abort_flag)) { fail = 6; break; }
                tc_fence_after_sync();
                for (int it = 0; it < w.steps; ++it, ++g) {
                    const int s = (int)(g % STAGES);
                    if (!mbar_wait_cluster(bar_full(s), (g / STAGES) & 1u, abort_flag)) { fail = 3; break; }
                    tc_fence_after_sync();
                    const uint32_t a4 = base4 + (uint32_t)s * (L::STAGE_BYTES >> 4), b4 = a4 + (L::A_BYTES >> 4);
#pragma unroll
                    for (int k = 0; k < VL_BK / 16; ++k)
                        umma_f16_words<2>(tmem + b * VL_TILE, a4 + (uint32_t)(A_DESC & 0xFFFFFFFFu) + A_STEP * k,
                                          (uint32_t)(A_DESC >> 32), b4 + (uint32_t)(B_DESC & 0xFFFFFFFFu) + B_STEP * k,
                                          (uint32_t)(B_DESC >> 32), idesc, it > 0 || k > 0 ? 1u : 0u);
                    umma_commit_pair(bar_empty(s), (uint16_t)3);
                }
                if (fail) break;
                umma_commit_pair(bar_done(b), (uint16_t)3);
                ++n;
            }
        } else if (lane == 0) {
            const uint32_t lead_full0 = mapa_shared(bar_full(0), 0u);
            uint32_t g = 0;
            for (int u = pair; u < plan.units && !fail; u += pairs) {
                const VlUnit w = vl_unit<MODE>(u, plan);
                if (skip(w)) continue;
                for (int it = 0; it < w.steps; ++it, ++g) {
                    const int s = (int)(g % STAGES);
                    if (!mbar_wait(bar_landed(s), (g / STAGES) & 1u, abort_flag)) { fail = 8; break; }
                    mbar_arrive_cluster(lead_full0 + 8u * s);
                }
            }
        }
    } else if constexpr (MODE == VL_FEW) {
        // ------------------------------------------------------------------ epilogue: a word's values of half the rows
        // A thread keeps maximum and sum of the words that come by its lane, for each of its 16 or 32 rows, over all tiles;
        // the lanes of a warp meet at the end.
        const int q = warp & 3, half = (warp - 2) >> 2, n = p.n_rows / 2, row0 = half * n;
        const uint32_t lead_drained = mapa_shared(bar_drained(0), 0u);
        const int target = lane < n && row0 + lane < rows ? p.target[row0 + lane] : -1;
        float m[32], s[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) { m[j] = VL_NEG; s[j] = 0.f; }
        uint32_t it = 0;
        for (int u = pair; u < plan.units && !fail; u += pairs, ++it) {
            const int b = (int)(it & 1u);
            if (!mbar_wait(bar_done(b), (it >> 1) & 1u, abort_flag)) { fail = 5; break; }
            tc_fence_after_sync();
            const int word0 = u * VL_TILE + (int)rank * 128 + q * 32;
            uint32_t r[32];
            const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + b * VL_TILE + row0;
            if (n == 32) {
                tmem_ld_32x32(at, r);
            } else {
                uint32_t h[16];
                tmem_ld_32x16(at, h);
#pragma unroll
                for (int j = 0; j < 32; ++j) r[j] = j < 16 ? h[j] : 0u;
            }
            tmem_ld_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(lead_drained + 8u * b);
            const bool there = word0 + lane < p.vocab;
            const unsigned hits = __ballot_sync(0xffffffffu, (unsigned)(target - word0) < 32u);    // rows whose target is here
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                if (j >= n) break;
                float x2 = there ? __uint_as_float(r[j]) * VL_LOG2E : VL_NEG;
                if (hits >> j & 1u) x2 = __shfl_sync(0xffffffffu, target, j) == word0 + lane ? VL_NEG : x2;
                const float top = fmaxf(m[j], x2);
                s[j] = fmaf(s[j], vl_ex2(m[j] - top), there && x2 != VL_NEG ? vl_ex2(x2 - top) : 0.f);
                m[j] = top;
            }
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            if (j >= n) break;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float om = __shfl_xor_sync(0xffffffffu, m[j], o), os = __shfl_xor_sync(0xffffffffu, s[j], o);
                const float top = fmaxf(m[j], om);
                s[j] = s[j] * vl_ex2(m[j] - top) + os * vl_ex2(om - top);
                m[j] = top;
            }
            if (lane == 0) p.parts[(long long)(blockIdx.x * 4 + q) * p.rows_pad + row0 + j] = make_float2(m[j], s[j]);
        }
    } else {
        // ------------------------------------------------------------------ epilogue: a row's half tile per thread
        const int q = warp & 3, half = (warp - 2) >> 2;
        const uint32_t lead_drained = mapa_shared(bar_drained(0), 0u);
        const uint32_t staging = base + L::STAGING_OFF + (uint32_t)(warp - 2) * 4096u;
        uint32_t n = 0;
        for (int u = pair; u < plan.units && !fail; u += pairs) {
            const VlUnit w = vl_unit<MODE>(u, plan);
            const int row = w.mt * VL_TILE + (int)rank * 128 + q * 32 + lane;     // VL_WEIGHT: word of the piece
            const int col0 = w.nt * VL_TILE + half * 128;
            if (MODE == VL_WEIGHT && plan.steps <= 0) {
                // no row takes part: the gradient of the head is zero
                if (plan.v0 + row < p.vocab)
                    for (int c = col0; c < col0 + 128 && c < p.hidden; ++c)
                        static_cast<unsigned short*>(p.d_weight)[(long long)(plan.v0 + row) * p.hidden + c] = 0;
                continue;
            }
            const bool live = row < rows;
            float scale = 1.f;
            if (MODE == VL_HIDDEN && live && p.index > 0)
                scale = exp2f(p.refs[p.index * p.rows_pad + row] - p.refs[(p.index + 1) * p.rows_pad + row]);
            if (skip(w)) {
                if (MODE == VL_HIDDEN && live && scale != 1.f) {     // nothing to add, but the reference has moved
                    float* plane = p.planes + ((long long)w.slice * rows_dev + row) * p.hidden;
                    for (int c = col0; c < col0 + 128 && c < p.hidden; ++c) plane[c] *= scale;
                }
                continue;
            }
            const int b = (int)(n & 1u);
            // what the values meet, asked for before the tile is complete
            int target = -1;
            float lse2 = 0.f, rest = 0.f, ref = 0.f;
            float4 coef = make_float4(0.f, 0.f, 0.f, 0.f);
            if (MODE <= VL_GRAD && live) target = p.target[row] - plan.v0 - col0;   // column of this thread's share
            if (MODE == VL_GRAD && live) {
                lse2 = p.lse2[row];
                rest = p.rest[row];
                coef = p.coef[row];
            }
            if (MODE == VL_SOFT && live) {
                ref = p.refs[p.index * p.rows_pad + row];
                if (p.again) {
                    // the piece's largest decides whether this row changes its reference (the sums are not read:
                    // they may have overflowed, and other units replace them)
                    float top = VL_NEG;
                    for (int i = 0; i < 2 * plan.tiles; ++i)
                        top = fmaxf(top, p.parts[(plan.v0 / VL_TILE * 2 + i) * p.rows_pad + row].x);
                    if (top > ref + (p.bf16 ? VL_ROOM_BF16 : VL_ROOM_F16)) ref = ceilf(top) - 6.f;
                }
                if (w.nt == 0 && half == 0) p.refs[(p.index + 1) * p.rows_pad + row] = ref;
            }
            if (MODE == VL_WEIGHT) scale = *p.weight_scale;
            if (!mbar_wait(bar_done(b), (n >> 1) & 1u, abort_flag)) { fail = 5; break; }
            tc_fence_after_sync();
            const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + b * VL_TILE + half * 128;
            auto release = [&]() {
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(lead_drained + 8u * b);
            };
            // The box's memory is free again once the store before has read it; what is in it goes out as 32 whole lines.
            auto box_begin = [&]() {
                if (lane == 0) bulk_wait_read();
                __syncwarp();
            };
            auto box_put = [&](int chunk, uint32_t x, uint32_t y, uint32_t z, uint32_t t) {    // 16 bytes of this lane's row
                vl_sts128(staging + lane * 128 + ((chunk ^ (lane & 7)) << 4), x, y, z, t);
            };
            auto box_end = [&](int x, int y, bool add) {
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    if (add) tma_reduce_add_2d(&maps.c, staging, x, y);
                    else     tma_store_2d(&maps.c, staging, x, y);
                    bulk_commit();
                }
            };
            const int row0 = row - lane;
            // 32 values in 16 bits: half a box
            auto put16 = [&](const float (&v)[32], int c) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    box_put((c & 32) / 8 + i, vl_pack(v[8 * i], v[8 * i + 1], p.bf16), vl_pack(v[8 * i + 2], v[8 * i + 3], p.bf16),
                            vl_pack(v[8 * i + 4], v[8 * i + 5], p.bf16), vl_pack(v[8 * i + 6], v[8 * i + 7], p.bf16));
            };
            // values of the 16-bit piece (columns col0 + c ..)
            auto store_piece = [&](const float (&v)[32], int c) {
                if ((c & 32) == 0) box_begin();
                put16(v, c);
                if ((c & 32) != 0) box_end(0, ((col0 + c) >> 6) * rows_dev + row0, false);
            };
            float m2 = VL_NEG, sum = 0.f;
#pragma unroll 1
            for (int c = 0; c < 128; c += 32) {
                uint32_t r[32];
                tmem_ld_32x32(at + c, r);
                tmem_ld_wait();
                if (c == 96) release();
                if (MODE <= VL_SOFT) {
                    const int words = p.vocab - plan.v0 - col0 - c;       // words there are in this chunk
                    const bool cut = words < 32 || (unsigned)(target - c) < 32u;
                    if (__any_sync(0xffffffffu, cut)) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (e >= words || e == target - c) r[e] = __float_as_uint(VL_NEG);
                    }
                    float top = __uint_as_float(r[0]);
#pragma unroll
                    for (int e = 1; e < 32; ++e) top = fmaxf(top, __uint_as_float(r[e]));
                    const float top2 = top * VL_LOG2E;
                    float part[4] = {0.f, 0.f, 0.f, 0.f};
                    if (MODE == VL_STATS) {
                        if (top2 > m2) {
                            sum *= vl_ex2(m2 - top2);
                            m2 = top2;
                        }
#pragma unroll
                        for (int e = 0; e < 32; ++e) part[e & 3] += vl_ex2(fmaf(__uint_as_float(r[e]), VL_LOG2E, -m2));
                    } else {
                        m2 = fmaxf(m2, top2);
                        float v[32];
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            v[e] = live ? vl_ex2(fmaf(__uint_as_float(r[e]), VL_LOG2E, -ref)) : 0.f;
                            part[e & 3] += v[e];
                        }
                        store_piece(v, c);
                    }
                    sum += (part[0] + part[1]) + (part[2] + part[3]);
                } else if (MODE == VL_GRAD) {
                    const int words = p.vocab - plan.v0 - col0 - c;
                    float v[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[e] = vl_ex2(fmaf(__uint_as_float(r[e]), VL_LOG2E, -lse2)) * coef.x;
                    const bool cut = words < 32 || (unsigned)(target - c) < 32u || !live;
                    if (__any_sync(0xffffffffu, cut)) {
                        const float hit = coef.z * (1.f - rest) - coef.y * rest;    // c p_t - b (1 - p_t)
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            if (e == target - c) v[e] = hit;
                            if (e >= words || !live) v[e] = 0.f;
                        }
                    }
                    store_piece(v, c);
                } else if (MODE == VL_HIDDEN) {
                    if (col0 + c >= p.hidden) continue;
                    if (__any_sync(0xffffffffu, scale != 1.f)) {       // a reference has moved: sums so far go along
                        float* out = p.planes + ((long long)w.slice * rows_dev + row) * p.hidden + col0 + c;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (col0 + c + e < p.hidden) out[e] = fmaf(out[e], scale, __uint_as_float(r[e]));
                        continue;
                    }
                    box_begin();
#pragma unroll
                    for (int i = 0; i < 8; ++i) box_put(i, r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
                    box_end(col0 + c, w.slice * rows_dev + row0, p.index > 0);
                } else {
                    if (col0 + (c & 64) >= p.hidden) continue;
                    if ((c & 32) == 0) box_begin();
                    float v[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(r[e]) * scale;
                    put16(v, c);
                    if ((c & 32) != 0) box_end(col0 + (c & 64), plan.v0 + row0, false);
                }
            }
            if (MODE <= VL_SOFT) {
                p.parts[(long long)(plan.v0 / VL_TILE * 2 + 2 * w.nt + half) * p.rows_pad + row] = make_float2(m2, sum);
                if (MODE == VL_SOFT && live && !p.again && m2 > ref + (p.bf16 ? VL_ROOM_BF16 : VL_ROOM_F16)) {
                    int* f = p.flags + (long long)p.index * p.flags_pitch;      // (several threads write the same)
                    f[0] = 1;
                    f[1 + w.mt] = 1;
                }
            }
            ++n;
        }
        if (MODE != VL_STATS && lane == 0) bulk_wait();
    }

    if (fail) {
        atomicCAS(p.status, 0, 100 + fail);
        // copies and MMAs in flight get time to land before shared memory and TMEM go away
        const unsigned long long t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem, 512);
    }
}

// ------------------------------------------------------------------------------------- rows that take part
__device__ __forceinline__ float vl_float(unsigned short x, int bf16) {
    return bf16 ? __uint_as_float((uint32_t)x << 16) : __half2float(__ushort_as_half(x));
}
__device__ __forceinline__ float2 vl_two(uint32_t w, int bf16) {
    if (bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

constexpr int VL_GATHER_WARPS = 8;

// A CTA takes `per` rows of the caller's. Where they go follows from the targets before them, which it counts itself.
__global__ void __launch_bounds__(VL_GATHER_WARPS * 32)
vl_gather_kernel(const VocabLossArgs a, int per) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ int before[VL_GATHER_WARPS];
    __shared__ int place[32], total;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long row0 = (long long)blockIdx.x * per;
    const auto takes_part = [&](long long t) { return t >= 0 && t < a.vocab; };
    int n = 0;
    for (long long i = threadIdx.x; i < row0; i += VL_GATHER_WARPS * 32) n += takes_part(a.targets[i]) ? 1 : 0;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) before[warp] = n;
    if (a.flags != nullptr)
        for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < a.n_flags; i += (long long)gridDim.x * blockDim.x)
            a.flags[i] = 0;
    __syncthreads();
    if (warp == 0) {
        int start = 0;
        for (int i = 0; i < VL_GATHER_WARPS; ++i) start += before[i];
        const long long row = row0 + lane;
        const bool in = lane < per && row < a.rows;
        const long long t = in ? a.targets[row] : -1;
        const bool part = in && takes_part(t);
        if (in && t >= a.vocab) atomicCAS(a.status, 0, STATUS_CE_TARGET_RANGE);   // treated as ignored, and recorded
        const unsigned mask = __ballot_sync(0xffffffffu, part);
        const int at = start + __popc(mask & ((1u << lane) - 1u));
        place[lane] = part ? at : -1;
        if (in) {
            a.place[row] = part ? at : -1;
            if (part) {
                a.target[at] = (int)t;
                a.source[at] = (int)row;
            } else {
                a.losses[row] = 0.f;
                a.lse[row] = 0.f;
            }
        }
        if (lane == 0) {
            total = start + __popc(mask);
            if (row0 + per >= a.rows) *a.count = total;      // (the last CTA)
        }
    }
    __syncthreads();
    const int vecs = (int)(a.hidden / 8);
    for (int i = warp; i < per; i += VL_GATHER_WARPS) {
        const int at = place[i];
        if (at < 0) continue;
        const long long row = row0 + i;
        const uint4* h = reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(a.x) + row * a.ld_x);
        const uint4* w = reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(a.weight) + (long long)a.targets[row] * a.ld_w);
        uint4* out = reinterpret_cast<uint4*>(static_cast<unsigned short*>(a.gathered) + (long long)at * a.hidden);
        float dot = 0.f;
#pragma unroll 4
        for (int c = lane; c < vecs; c += 32) {
            const uint4 x = __ldg(h + c), y = __ldg(w + c);
            out[c] = x;
            const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
            float d = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = vl_two(xs[e], a.bf16), g = vl_two(ys[e], a.bf16);
                d = fmaf(f.x, g.x, d);
                d = fmaf(f.y, g.y, d);
            }
            dot += d;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (lane == 0) a.target_logit[at] = dot;
    }
    // the last CTA fills the last tile's empty rows with zeros: they meet the others' in sums over rows
    if (row0 + per >= a.rows) {
        const int end = vl_div_up(total, VL_TILE) * VL_TILE;
        uint4* out = reinterpret_cast<uint4*>(a.gathered);
        for (long long i = (long long)total * vecs + threadIdx.x; i < (long long)end * vecs; i += VL_GATHER_WARPS * 32)
            out[i] = make_uint4(0u, 0u, 0u, 0u);
    }
}

// Joins a row's statistics, 32 rows by 32 shares of the parts per CTA. PROBE: the first words' maxima give the row's
// reference. Otherwise the whole vocabulary's give loss and lse; `soft`: the sums are relative to the row's references,
// of which the parts of `piece` word tiles each had one.
template <bool PROBE>
__global__ void __launch_bounds__(1024)
vl_merge_kernel(const VocabLossArgs a, int n_parts, int word_tiles, int soft) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ float2 join[32][33];
    const int rows = *a.count, row = blockIdx.x * 32 + threadIdx.x;
    if (blockIdx.x * 32 >= rows) return;
    const int piece = soft ? vl_piece_tiles(vl_div_up(rows, VL_TILE), word_tiles, a.capacity, a.slots) : 1;
    float m = VL_NEG, s = 0.f;
    if (row < rows) {
#pragma unroll 4
        for (int i = threadIdx.y; i < n_parts; i += 32) {
            float2 x = a.parts[(long long)i * a.rows_pad + row];
            if (soft) x.x = a.refs[(long long)(i / 2 / piece + 1) * a.rows_pad + row];
            const float top = fmaxf(m, x.x);
            s = s * vl_ex2(m - top) + x.y * vl_ex2(x.x - top);
            m = top;
        }
    }
    join[threadIdx.x][threadIdx.y] = make_float2(m, s);
    __syncthreads();
    // a warp joins one row's shares
    float2 x = join[threadIdx.y][threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, x.x, o), os = __shfl_xor_sync(0xffffffffu, x.y, o);
        const float top = fmaxf(x.x, om);
        x.y = x.y * vl_ex2(x.x - top) + os * vl_ex2(om - top);
        x.x = top;
    }
    const int at = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x != 0 || at >= rows) return;
    const float logit = a.target_logit[at], logit2 = logit * VL_LOG2E;
    if (PROBE) {
        // (fmaxf leaves out a NaN; within what a float keeps whole numbers of)
        const float ref = fmaxf(fmaxf(x.x - VL_BELOW, logit2 - VL_BELOW_TARGET), -1.0e6f);
        a.refs[at] = floorf(fminf(ref, 1.0e6f));
        return;
    }
    const float d = x.x - logit2;      // log2 of what the others' sum is relative to, over the target's
    float loss, rest, norm;
    if (d <= 0.f) {
        const float f = exp2f(d), r = x.y * f;
        loss = log1pf(r);
        rest = r / (1.f + r);
        norm = f / (1.f + r);
    } else {
        const float t = x.y + exp2f(-d);
        loss = d * VL_LN2 + logf(t);
        rest = x.y / t;
        norm = 1.f / t;
    }
    a.lse_rows[at] = logit2 + loss * VL_LOG2E;
    a.rest[at] = rest;
    if (soft) a.norm[at] = norm;
    a.losses[a.source[at]] = loss;
    a.lse[a.source[at]] = logit + loss;
}

// U: the planes' sum over the row's sum of exponentials.
__global__ void __launch_bounds__(256)
vl_mean_kernel(const VocabLossArgs a, int word_tiles) {
    grid_dep_wait();
    grid_dep_launch();
    const int rows = *a.count, quads = (int)(a.hidden / 4);
    if (rows == 0) return;
    const int row_tiles = vl_div_up(rows, VL_TILE);
    const int steps = vl_piece_tiles(row_tiles, word_tiles, a.capacity, a.slots) * (VL_TILE / VL_BK);
    const int slices = vl_slices(row_tiles * vl_div_up((int)a.hidden, VL_TILE), steps, a.slots);
    const long long plane = (long long)row_tiles * VL_TILE * a.hidden;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)rows * quads; i += (long long)gridDim.x * 256) {
        const float norm = a.norm[i / quads];
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int z = 0; z < slices; ++z) {
            const float4 x = *reinterpret_cast<const float4*>(a.planes + z * plane + i * 4);
            v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
        }
        reinterpret_cast<float4*>(a.mean)[i] = make_float4(v.x * norm, v.y * norm, v.z * norm, v.w * norm);
    }
}

// ------------------------------------------------------------------------------------- backward
// Power of two at or above x >= 0, from 2^-95 to 2^126: 0 for zero, 1 for what is not finite.
__device__ __forceinline__ float vl_power(float x) {
    const uint32_t bits = __float_as_uint(x);
    if (bits == 0u || bits >= 0x7F800000u) return bits == 0u ? 0.f : 1.f;
    return __uint_as_float(min(max((bits + 0x007FFFFFu) >> 23, 32u), 253u) << 23);
}

__device__ __forceinline__ float vl_upstream(const float* g, long long stride, long long row) {
    return g == nullptr ? 0.f : g[row * stride];
}

// One CTA: per row that takes part (b + c, b, c) over the power of two above the largest |b|, |c|, times VL_P_SCALE. (A
// row far below the largest keeps its digits down to 2^-27 of it, and adds nothing that the others' rounding would not
// cover below.)
__global__ void __launch_bounds__(1024)
vl_coef_kernel(const VocabLossArgs a) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ float part[32];
    float top = 0.f;
    const int rows = *a.count;
    for (int at = threadIdx.x; at < rows; at += 1024) {
        const long long row = a.source[at];
        top = fmaxf(top, fmaxf(fabsf(vl_upstream(a.d_losses, a.d_losses_stride, row)), fabsf(vl_upstream(a.d_lse, a.d_lse_stride, row))));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
    __syncthreads();
    top = part[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float power = vl_power(top), inv = power > 0.f ? VL_P_SCALE / power : 0.f;
    for (int at = threadIdx.x; at < rows; at += 1024) {
        const long long row = a.source[at];
        const float b = vl_upstream(a.d_losses, a.d_losses_stride, row), c = vl_upstream(a.d_lse, a.d_lse_stride, row);
        a.coef[at] = make_float4((b + c) * inv, b * inv, c * inv, 0.f);
    }
    if (threadIdx.x == 0) *a.weight_scale = power / VL_P_SCALE;
}

// dH of the caller's rows; zeros where the row took no part.
__global__ void __launch_bounds__(256)
vl_hidden_kernel(const VocabLossArgs a) {
    grid_dep_wait();
    grid_dep_launch();
    const int vecs = (int)(a.hidden / 8);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < a.rows * vecs; i += (long long)gridDim.x * 256) {
        const long long row = i / vecs;
        const int c = (int)(i - row * vecs), at = a.place[row];
        uint4 out = make_uint4(0u, 0u, 0u, 0u);
        if (at >= 0) {
            const float b = vl_upstream(a.d_losses, a.d_losses_stride, row), z = vl_upstream(a.d_lse, a.d_lse_stride, row);
            const float rest = a.rest[at], mean = b + z, hit = z * (1.f - rest) - b * rest;
            const float4* u = reinterpret_cast<const float4*>(a.mean + (long long)at * a.hidden) + 2 * c;
            const float4 x = u[0], y = u[1];
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(a.weight) + (long long)a.target[at] * a.ld_w) + c);
            const float2 w0 = vl_two(w.x, a.bf16), w1 = vl_two(w.y, a.bf16), w2 = vl_two(w.z, a.bf16), w3 = vl_two(w.w, a.bf16);
            out = make_uint4(vl_pack(fmaf(mean, x.x, hit * w0.x), fmaf(mean, x.y, hit * w0.y), a.bf16),
                             vl_pack(fmaf(mean, x.z, hit * w1.x), fmaf(mean, x.w, hit * w1.y), a.bf16),
                             vl_pack(fmaf(mean, y.x, hit * w2.x), fmaf(mean, y.y, hit * w2.y), a.bf16),
                             vl_pack(fmaf(mean, y.z, hit * w3.x), fmaf(mean, y.w, hit * w3.y), a.bf16));
        }
        reinterpret_cast<uint4*>(a.d_x)[i] = out;
    }
}

// ------------------------------------------------------------------------------------------- host side
static size_t vl_align(size_t n) { return (n + 255) / 256 * 256; }

static long long vl_rows_pad(long long rows) { return (rows + VL_TILE - 1) / VL_TILE * VL_TILE; }

static int vl_word_tiles(long long vocab) { return (int)((vocab + VL_TILE - 1) / VL_TILE); }

// Tiles that the 16-bit piece has room for, the most pieces that any number of rows up to `rows` makes of the
// vocabulary, and the planes of U they need, in units of rows_pad rows.
struct VlRoom {
    int capacity, pieces, planes;
};
static VlRoom vl_room(long long rows, long long vocab, long long hidden, int slots) {
    VlRoom r = {VL_PIECE_UNITS, 1, 1};
    const long long row_tiles = vl_rows_pad(rows) / VL_TILE;
    const int word_tiles = vl_word_tiles(vocab), feature_tiles = vl_div_up((int)hidden, VL_TILE);
    if (r.capacity < 4 * row_tiles) r.capacity = (int)(4 * row_tiles);
    if (r.capacity > row_tiles * word_tiles) r.capacity = (int)(row_tiles * word_tiles);
    long long most = row_tiles;
    for (long long t = 1; t <= row_tiles; ++t) {
        const int tiles = vl_piece_tiles((int)t, word_tiles, r.capacity, slots), pieces = vl_div_up(word_tiles, tiles);
        if (pieces > r.pieces) r.pieces = pieces;
        const long long planes = t * vl_slices((int)t * feature_tiles, tiles * (VL_TILE / VL_BK), slots);
        if (planes > most) most = planes;
    }
    r.planes = (int)((most + row_tiles - 1) / row_tiles);
    return r;
}

// What the forward keeps for the backward.
struct VlKept {
    size_t count, place, source, target, lse, rest, gathered, mean, bytes;
};
static VlKept vl_kept(long long rows, long long hidden, int grads) {
    VlKept k = {};
    const size_t pad = (size_t)vl_rows_pad(rows);
    size_t at = 0;
    const auto take = [&](size_t n) { const size_t r = at; at += vl_align(n); return r; };
    k.count = take(4);
    k.place = take((size_t)rows * 4);
    k.source = take(pad * 4);
    k.target = take(pad * 4);
    k.lse = take(pad * 4);
    k.rest = take(pad * 4);
    if (grads & 1) k.mean = take((size_t)rows * (size_t)hidden * 4);
    k.gathered = at;                       // last: without a gradient of the weight it is scratch of the forward
    if (grads & 2) take(pad * (size_t)hidden * 2);
    k.bytes = at;
    return k;
}

struct VlScratch {
    size_t parts, target_logit, norm, refs, flags, gathered, coef, weight_scale, piece, planes, bytes;
    VlRoom room;
};

static VlScratch vl_scratch(const VocabLossArgs& a, bool backward) {
    VlScratch s = {};
    const size_t pad = (size_t)vl_rows_pad(a.rows);
    size_t at = 0;
    const auto take = [&](size_t n) { const size_t r = at; at += vl_align(n); return r; };
    if ((backward && a.d_weight != nullptr) || (!backward && (a.grads & 1)))
        s.room = vl_room(a.rows, a.vocab, a.hidden, a.sm_count / 2);
    if (!backward) {
        const size_t n_parts = (size_t)vl_word_tiles(a.vocab) * 2, few_parts = (size_t)a.sm_count * 4;
        s.parts = take((n_parts > few_parts ? n_parts : few_parts) * 8 * pad);
        s.target_logit = take(pad * 4);
        if (!(a.grads & 2)) s.gathered = take(pad * (size_t)a.hidden * 2);
        if (a.grads & 1) {
            s.norm = take(pad * 4);
            s.refs = take((size_t)(s.room.pieces + 1) * pad * 4);
            s.flags = take((size_t)s.room.pieces * (1 + pad / VL_TILE) * 4);
            s.piece = take((size_t)s.room.capacity * VL_TILE * VL_TILE * 2);
            s.planes = take((size_t)s.room.planes * pad * (size_t)a.hidden * 4);
        }
    } else if (a.d_weight != nullptr) {
        s.coef = take(pad * 16);
        s.weight_scale = take(4);
        s.piece = take((size_t)s.room.capacity * VL_TILE * VL_TILE * 2);
    }
    s.bytes = at;
    return s;
}

size_t vocab_loss_kept_bytes(long long rows, long long hidden, int grads) { return vl_kept(rows, hidden, grads).bytes; }

size_t vocab_loss_workspace_bytes(const VocabLossArgs& a, bool backward) { return vl_scratch(a, backward).bytes; }

template <int MODE>
static cudaError_t vl_launch(const VlMaps& maps, const VlParams& p, long long units, int sm_count, cudaStream_t stream,
                             int* ctas = nullptr) {
    auto kernel = vl_gemm_kernel<MODE>;
    constexpr int VL_SMEM = VlSmemOf<MODE>::TOTAL;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, VL_SMEM);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(VL_THREADS);
    cfg.dynamicSmemBytes = VL_SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    // pairs that can be resident at once: a pair sits in one GPC, so the runtime knows (asked once)
    static const int most = [&] {
        cfg.gridDim = dim3((unsigned)(sm_count / 2 * 2));
        int n = 0;
        return cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess && n > 0 ? n : 0x7FFFFFFF;
    }();
    long long pairs = sm_count / 2 < most ? sm_count / 2 : most;
    if (units < pairs) pairs = units;
    if (pairs < 1) pairs = 1;
    cfg.gridDim = dim3((unsigned)(2 * pairs));
    if (ctas != nullptr) *ctas = (int)(2 * pairs);
    return cudaLaunchKernelEx(&cfg, kernel, maps, p);
}

static bool vl_map(CUtensorMap* map, int bf16, const void* base, long long inner, long long outer, long long pitch, int box_outer) {
    return make_map_2d(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, base, (uint64_t)inner,
                       (uint64_t)outer, (uint64_t)pitch * 2, VL_BK, (uint32_t)box_outer, CU_TENSOR_MAP_SWIZZLE_128B);
}

// The 16-bit piece: blocks of [rows][64 words], read in boxes of 128 rows (rows as M) or 64 (as steps), written in 32.
static bool vl_piece_map(CUtensorMap* map, const VocabLossArgs& a, int box_outer) {
    return vl_map(map, a.bf16, a.piece, VL_BK, (long long)a.capacity * VL_TILE * (VL_TILE / VL_BK), VL_BK, box_outer);
}

static void vl_use_kept(VocabLossArgs& a) {
    const VlKept k = vl_kept(a.rows, a.hidden, a.grads);
    char* base = static_cast<char*>(a.kept);
    a.count = reinterpret_cast<int*>(base + k.count);
    a.place = reinterpret_cast<int*>(base + k.place);
    a.source = reinterpret_cast<int*>(base + k.source);
    a.target = reinterpret_cast<int*>(base + k.target);
    a.lse_rows = reinterpret_cast<float*>(base + k.lse);
    a.rest = reinterpret_cast<float*>(base + k.rest);
    a.mean = reinterpret_cast<float*>(base + k.mean);
    a.gathered = base + k.gathered;
    a.rows_pad = vl_rows_pad(a.rows);
    a.slots = a.sm_count / 2;
}

static VlParams vl_params(const VocabLossArgs& a) {
    VlParams p = {};
    p.count = a.count; p.status = a.status; p.bf16 = a.bf16;
    p.vocab = (int)a.vocab; p.hidden = (int)a.hidden; p.word_tiles = vl_word_tiles(a.vocab);
    p.capacity = a.capacity; p.slots = a.slots;
    p.target = a.target; p.parts = a.parts; p.rows_pad = a.rows_pad;
    p.refs = a.refs; p.flags = a.flags; p.flags_pitch = 1 + (int)(a.rows_pad / VL_TILE);
    p.lse2 = a.lse_rows; p.rest = a.rest; p.coef = a.coef;
    p.piece = a.piece; p.planes = a.planes; p.d_weight = a.d_weight; p.weight_scale = a.weight_scale;
    return p;
}

cudaError_t launch_vocab_loss_fwd(const VocabLossArgs& a_in, cudaStream_t stream, const char** why) {
    *why = "";
    VocabLossArgs a = a_in;
    if (a.rows <= 0) return cudaSuccess;
    vl_use_kept(a);
    const VlScratch s = vl_scratch(a, false);
    char* ws = static_cast<char*>(a.workspace);
    a.parts = reinterpret_cast<float2*>(ws + s.parts);
    a.target_logit = reinterpret_cast<float*>(ws + s.target_logit);
    if (!(a.grads & 2)) a.gathered = ws + s.gathered;
    const bool soft = (a.grads & 1) != 0;
    if (soft) {
        a.norm = reinterpret_cast<float*>(ws + s.norm);
        a.refs = reinterpret_cast<float*>(ws + s.refs);
        a.flags = reinterpret_cast<int*>(ws + s.flags);
        a.n_flags = s.room.pieces * (1 + a.rows_pad / VL_TILE);
        a.piece = ws + s.piece;
        a.planes = reinterpret_cast<float*>(ws + s.planes);
        a.capacity = s.room.capacity;
    }
    const int per = a.rows <= 4096 ? 8 : 32;
    cudaError_t e = launch_pdl(vl_gather_kernel, dim3((unsigned)((a.rows + per - 1) / per)), dim3(VL_GATHER_WARPS * 32), 0, stream, a, per);
    if (e != cudaSuccess) { *why = "gather"; return e; }
    VlMaps logits = {}, hidden = {};
    // Up to 64 rows without a gradient of x: the words take the tensor cores' long side. (64 rows of 3584 features against
    // 151,936 words: 216 us with the rows there, which costs four times the products; the weight alone takes 168.)
    const bool few = !soft && a.rows <= 64;
    const int few_rows = a.rows <= 32 ? 32 : 64;
    bool ok = few ? vl_map(&logits.a, a.bf16, a.weight, a.hidden, a.vocab, a.ld_w, 128) &&
                        vl_map(&logits.b, a.bf16, a.gathered, a.hidden, a.rows_pad, a.hidden, few_rows / 2)
                  : vl_map(&logits.a, a.bf16, a.gathered, a.hidden, a.rows_pad, a.hidden, 128) &&
                        vl_map(&logits.b, a.bf16, a.weight, a.hidden, a.vocab, a.ld_w, 128);
    if (ok && soft)
        ok = vl_piece_map(&logits.c, a, 32) && vl_piece_map(&hidden.a, a, 128) &&
             vl_map(&hidden.b, a.bf16, a.weight, a.hidden, a.vocab, a.ld_w, 64) &&
             make_map_2d(&hidden.c, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, a.planes, (uint64_t)a.hidden,
                         (uint64_t)s.room.planes * (uint64_t)a.rows_pad, (uint64_t)a.hidden * 4, 32, 32, CU_TENSOR_MAP_SWIZZLE_128B);
    if (!ok) { *why = "cuTensorMapEncodeTiled"; return cudaErrorInvalidValue; }
    VlParams base = vl_params(a);
    base.n_rows = few_rows;
    int n_parts = 2 * base.word_tiles;
    const long long row_tiles = a.rows_pad / VL_TILE;
    const dim3 merge_grid((unsigned)((a.rows + 31) / 32)), merge_block(32, 32);
    if (!soft) {
        int ctas = 0;
        e = few ? vl_launch<VL_FEW>(logits, base, base.word_tiles, a.sm_count, stream, &ctas)
                : vl_launch<VL_STATS>(logits, base, row_tiles * base.word_tiles, a.sm_count, stream);
        if (few) n_parts = 4 * ctas;
        if (e != cudaSuccess) { *why = "statistics"; return e; }
    } else {
        VlParams probe = base;
        if (probe.word_tiles > VL_PROBE_TILES) probe.word_tiles = VL_PROBE_TILES;
        e = vl_launch<VL_STATS>(logits, probe, row_tiles * probe.word_tiles, a.sm_count, stream);
        if (e == cudaSuccess) e = launch_pdl(vl_merge_kernel<true>, merge_grid, merge_block, 0, stream, a, 2 * probe.word_tiles, probe.word_tiles, 0);
        if (e != cudaSuccess) { *why = "references"; return e; }
        const long long units = row_tiles * base.word_tiles < a.capacity ? row_tiles * base.word_tiles : a.capacity;
        for (int i = 0; i < s.room.pieces; ++i) {
            VlParams p = base;
            p.index = i;
            e = vl_launch<VL_SOFT>(logits, p, units, a.sm_count, stream);
            p.again = 1;
            if (e == cudaSuccess) e = vl_launch<VL_SOFT>(logits, p, units, a.sm_count, stream);
            if (e != cudaSuccess) { *why = "softmax"; return e; }
            e = vl_launch<VL_HIDDEN>(hidden, p, row_tiles * vl_div_up(p.hidden, VL_TILE) * VL_MAX_SLICES, a.sm_count, stream);
            if (e != cudaSuccess) { *why = "gradient of the hidden states"; return e; }
        }
    }
    e = launch_pdl(vl_merge_kernel<false>, merge_grid, merge_block, 0, stream, a, n_parts, base.word_tiles, soft ? 1 : 0);
    if (e == cudaSuccess && soft)
        e = launch_pdl(vl_mean_kernel, dim3((unsigned)(a.sm_count * 8)), dim3(256), 0, stream, a, base.word_tiles);
    if (e != cudaSuccess) *why = "merge";
    return e;
}

cudaError_t launch_vocab_loss_bwd(const VocabLossArgs& a_in, cudaStream_t stream, const char** why) {
    *why = "";
    VocabLossArgs a = a_in;
    if (a.rows <= 0) return cudaSuccess;
    vl_use_kept(a);
    const VlScratch s = vl_scratch(a, true);
    char* ws = static_cast<char*>(a.workspace);
    cudaError_t e = cudaSuccess;
    if (a.d_x != nullptr) {
        e = launch_pdl(vl_hidden_kernel, dim3((unsigned)(a.sm_count * 8)), dim3(256), 0, stream, a);
        if (e != cudaSuccess) { *why = "gradient of the hidden states"; return e; }
    }
    if (a.d_weight == nullptr) return e;
    a.coef = reinterpret_cast<float4*>(ws + s.coef);
    a.weight_scale = reinterpret_cast<float*>(ws + s.weight_scale);
    a.piece = ws + s.piece;
    a.capacity = s.room.capacity;
    e = launch_pdl(vl_coef_kernel, dim3(1), dim3(1024), 0, stream, a);
    if (e != cudaSuccess) { *why = "row factors"; return e; }
    VlMaps logits = {}, weight = {};
    if (!vl_map(&logits.a, a.bf16, a.gathered, a.hidden, a.rows_pad, a.hidden, 128) ||
        !vl_map(&logits.b, a.bf16, a.weight, a.hidden, a.vocab, a.ld_w, 128) ||
        !vl_piece_map(&logits.c, a, 32) || !vl_piece_map(&weight.a, a, 64) ||
        !vl_map(&weight.b, a.bf16, a.gathered, a.hidden, a.rows_pad, a.hidden, 64) ||
        !vl_map(&weight.c, a.bf16, a.d_weight, a.hidden, a.vocab, a.hidden, 32)) {
        *why = "cuTensorMapEncodeTiled";
        return cudaErrorInvalidValue;
    }
    VlParams p = vl_params(a);
    const long long units = a.rows_pad / VL_TILE * p.word_tiles < a.capacity ? a.rows_pad / VL_TILE * p.word_tiles : a.capacity;
    for (p.index = 0; p.index < s.room.pieces; ++p.index) {
        e = vl_launch<VL_GRAD>(logits, p, units, a.sm_count, stream);
        if (e != cudaSuccess) { *why = "gradient of the logits"; return e; }
        e = vl_launch<VL_WEIGHT>(weight, p, (long long)p.word_tiles * vl_div_up(p.hidden, VL_TILE), a.sm_count, stream);
        if (e != cudaSuccess) { *why = "gradient of the head"; return e; }
    }
    return e;
}

}  // namespace nf4
