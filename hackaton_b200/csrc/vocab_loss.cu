// Softmax cross-entropy over the vocabulary straight from the hidden states, in pieces of the vocabulary: the logits
// l = h . w_v exist only in tensor memory, a tile at a time, and of their gradient there is one piece at a time.
//   forward    lse = log sum_v exp(l_v),  loss = lse - l_t = log(1 + sum_{v != t} exp(l_v - l_t))
//   backward   with b = d loss, c = d lse:  dl_v = (b + c) p_v - b [v = t];  dH = dl . W,  dW = dl^T . H
// Rows whose target is negative take no part: the others are gathered first, everything behind that works on as many
// rows as there are (the count stays on the device), and what an ignored row holds is never read.
//
// Four matrix products of 2 R V K operations each (R rows, V words, K features): the logits for the statistics,
// once more for the gradient, then dH and dW. All run in one kernel, vl_gemm_kernel, in four modes that differ in
// the operands' layouts and the epilogue; it is bound by the tensor cores. CTA pairs (tcgen05.mma.cta_group::2) own a
// 256 x 256 tile, 128 rows by 256 columns of fp32 in each CTA's tensor memory, twice: while eight warps work on one
// tile's values the next one is being multiplied. Operands come by TMA in 64-deep steps through a ring of six.
//   statistics: a thread has a row's 128 columns; running maximum and sum of exponentials in the base-2 domain, the
//     target left out, so that 1 - p_t and a loss near zero keep their digits; one pair of numbers per row and half
//     tile goes out, which vl_merge_kernel joins in order. The target's own logit is a dot product in fp32 (vl_gather).
//   gradient: dl in 16 bits, each row scaled by a power of two (exact) so that fp16 keeps small probabilities
//   dH: fp32 planes, one per slice of the piece, added to from piece to piece; vl_hidden_kernel joins them in order
//   dW: the rows of the piece, in 16 bits
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

constexpr int VL_TILE = 256;               // rows and columns of a pair's tile
constexpr int VL_BK = 64;
constexpr int VL_STAGES = 6;
constexpr int VL_HALF_BYTES = 128 * VL_BK * 2;      // one CTA's share of either operand
constexpr int VL_STAGE_BYTES = 2 * VL_HALF_BYTES;
constexpr int VL_BAR_OFF = VL_STAGES * VL_STAGE_BYTES;
constexpr int VL_SMEM = VL_BAR_OFF + 256 + 1024;    // + slack for 1024-byte alignment
constexpr int VL_EPI_WARPS = 8;
constexpr int VL_THREADS = 64 + VL_EPI_WARPS * 32;

enum VlMode {
    VL_STATS = 0,    // A = gathered rows [R, K], B = W [V, K]                  -> maximum and sum per row and half tile
    VL_GRAD = 1,     // the same operands, one piece                            -> dl in 16 bits [R, piece]
    VL_HIDDEN = 2,   // A = dl [R, piece], B = W rows of the piece, N along K   -> fp32 planes [slices][R, K]
    VL_WEIGHT = 3    // A = dl^T, B = scaled rows [R, K], N along K             -> 16-bit rows of the piece [piece, K]
};

struct VlMaps {
    CUtensorMap a, b;
};

struct VlParams {
    const int* count;        // rows that take part
    int* status;
    int mode_bf16;
    int vocab, hidden;
    int v0, piece;           // first word of the piece, its words (a multiple of 256 unless it is the last)
    int n_tiles;             // tiles along the words (VL_STATS, VL_GRAD, VL_WEIGHT: as M) or features
    int slots;               // pairs that the slices are planned for
    // VL_STATS
    float2* parts;           // [2 * n_tiles][rows_pad]
    long long rows_pad;
    const int* target;       // per gathered row
    // VL_GRAD
    const float* lse2;
    const float* rest;       // 1 - p of the target
    const float4* coef;      // (b + c, b, c, -) over the row's scale, times VL_P_SCALE
    void* dl;
    long long ld_dl;
    // VL_HIDDEN
    float* planes;           // [slices][row tiles * 256][hidden]
    int first;               // the piece that fills the planes
    int first_steps;         // its steps, which decide on the slices
    // VL_WEIGHT
    void* d_weight;
    long long ld_dw;
    const float* weight_scale;
};

__host__ __device__ inline int vl_div_up(int a, int b) { return (a + b - 1) / b; }

// Slices of a piece's words for dH: as many as keep the pairs busiest, with at least eight steps each; none is empty.
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

struct VlPlan {      // what a mode's units are, from the device's row count
    int m_tiles, units, steps, slices, per_slice;
};

template <int MODE>
__device__ __forceinline__ VlPlan vl_plan(const VlParams& p, int rows) {
    VlPlan w;
    const int row_tiles = vl_div_up(rows, VL_TILE);
    w.slices = 1;
    if (MODE == VL_WEIGHT) {
        w.m_tiles = p.n_tiles;                                  // words of the piece
        w.steps = vl_div_up(rows, VL_BK);
        w.units = w.m_tiles * vl_div_up(p.hidden, VL_TILE);
    } else if (MODE == VL_HIDDEN) {
        w.m_tiles = row_tiles;
        w.steps = vl_div_up(p.piece, VL_BK);
        const int tiles = row_tiles * vl_div_up(p.hidden, VL_TILE);
        w.slices = rows > 0 ? vl_slices(tiles, p.first_steps, p.slots) : 1;
        w.units = tiles * w.slices;
    } else {
        w.m_tiles = row_tiles;
        w.steps = vl_div_up(p.hidden, VL_BK);
        w.units = row_tiles * p.n_tiles;
    }
    w.per_slice = vl_div_up(w.steps, w.slices);
    return w;
}

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
    constexpr bool A_MN = MODE == VL_WEIGHT, B_MN = MODE >= VL_HIDDEN;
    extern __shared__ uint8_t vl_smem[];
    const uint32_t base = (smem_u32(vl_smem) + 1023u) & ~1023u;
    uint8_t* gen = vl_smem + (base - smem_u32(vl_smem));
    const uint32_t bar = base + VL_BAR_OFF;
    auto bar_full = [&](int s) { return bar + 8u * s; };                        // leader: both CTAs' operands
    auto bar_landed = [&](int s) { return bar + 8u * (VL_STAGES + s); };        // peer: its own
    auto bar_empty = [&](int s) { return bar + 8u * (2 * VL_STAGES + s); };
    auto bar_done = [&](int b) { return bar + 8u * (3 * VL_STAGES + b); };      // accumulator complete
    auto bar_drained = [&](int b) { return bar + 8u * (3 * VL_STAGES + 2 + b); };
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + VL_BAR_OFF + 8 * (3 * VL_STAGES + 4));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + VL_BAR_OFF + 8 * (3 * VL_STAGES + 4) + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int pair = (int)(blockIdx.x >> 1), pairs = (int)(gridDim.x >> 1);

    if (threadIdx.x == 0) {
        for (int s = 0; s < VL_STAGES; ++s) {
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
    int fail = 0;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t g = 0;
            for (int u = pair; u < plan.units && !fail; u += pairs) {
                const VlUnit w = vl_unit<MODE>(u, plan);
                for (int it = 0; it < w.steps; ++it, ++g) {
                    const int s = (int)(g % VL_STAGES);
                    const uint32_t ph = (g / VL_STAGES) & 1u;
                    if (!mbar_wait_cluster(bar_empty(s), ph ^ 1u, abort_flag)) { fail = 1; break; }
                    const uint32_t landed = rank == 0 ? bar_full(s) : bar_landed(s);
                    const uint32_t sa = base + (uint32_t)s * VL_STAGE_BYTES, sb = sa + VL_HALF_BYTES;
                    const int k = (w.begin + it) * VL_BK;
                    const int am = w.mt * VL_TILE + (int)rank * 128, bn = w.nt * VL_TILE + (int)rank * 128;
                    mbar_arrive_expect_tx(landed, VL_STAGE_BYTES);
                    if (A_MN) {     // (the piece's words as M: columns of dl)
                        tma_load_2d(sa, &maps.a, am, k, landed);
                        tma_load_2d(sa + 8192, &maps.a, am + 64, k, landed);
                    } else {
                        tma_load_2d(sa, &maps.a, k, am, landed);
                    }
                    if (B_MN) {     // VL_HIDDEN: rows of W from the piece's first word on; VL_WEIGHT: gathered rows
                        const int y = MODE == VL_HIDDEN ? p.v0 + k : k;
                        tma_load_2d(sb, &maps.b, bn, y, landed);
                        tma_load_2d(sb + 8192, &maps.b, bn + 64, y, landed);
                    } else {
                        tma_load_2d(sb, &maps.b, k, p.v0 + bn, landed);
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
            const uint32_t idesc = make_idesc_f16(VL_TILE, A_MN ? 1u : 0u, B_MN ? 1u : 0u, VL_TILE) |
                                   (p.mode_bf16 ? (1u << 7) | (1u << 10) : 0u);
            const uint32_t base4 = (base & 0x3FFFFu) >> 4;
            uint32_t g = 0, n = 0;
            for (int u = pair; u < plan.units && !fail; u += pairs) {
                const VlUnit w = vl_unit<MODE>(u, plan);
                if (w.steps <= 0) continue;
                const int b = (int)(n & 1u);
                if (!mbar_wait_cluster(bar_drained(b), ((n >> 1) & 1u) ^ 1u, abort_flag)) { fail = 6; break; }
                tc_fence_after_sync();
                for (int it = 0; it < w.steps; ++it, ++g) {
                    const int s = (int)(g % VL_STAGES);
                    if (!mbar_wait_cluster(bar_full(s), (g / VL_STAGES) & 1u, abort_flag)) { fail = 3; break; }
                    tc_fence_after_sync();
                    const uint32_t a4 = base4 + (uint32_t)s * (VL_STAGE_BYTES >> 4), b4 = a4 + (VL_HALF_BYTES >> 4);
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
                for (int it = 0; it < w.steps; ++it, ++g) {
                    const int s = (int)(g % VL_STAGES);
                    if (!mbar_wait(bar_landed(s), (g / VL_STAGES) & 1u, abort_flag)) { fail = 8; break; }
                    mbar_arrive_cluster(lead_full0 + 8u * s);
                }
            }
        }
    } else {
        // ------------------------------------------------------------------ epilogue: a row's half tile per thread
        const int q = warp & 3, half = (warp - 2) >> 2;
        const uint32_t lead_drained = mapa_shared(bar_drained(0), 0u);
        uint32_t n = 0;
        for (int u = pair; u < plan.units && !fail; u += pairs) {
            const VlUnit w = vl_unit<MODE>(u, plan);
            const int row = w.mt * VL_TILE + (int)rank * 128 + q * 32 + lane;     // VL_WEIGHT: word of the piece
            const int col0 = w.nt * VL_TILE + half * 128;
            if (w.steps <= 0) {
                // no rows take part: the gradient of the head is zero (other modes have no units then)
                if (MODE == VL_WEIGHT && p.v0 + row < p.vocab && row < p.piece)
                    for (int c = col0; c < col0 + 128 && c < p.hidden; ++c)
                        static_cast<unsigned short*>(p.d_weight)[(long long)(p.v0 + row) * p.ld_dw + c] = 0;
                continue;
            }
            const int b = (int)(n & 1u);
            // what the values meet, asked for before the tile is complete
            int target = -1;
            float lse2 = 0.f, rest = 0.f, scale = 1.f;
            float4 coef = make_float4(0.f, 0.f, 0.f, 0.f);
            const bool live = row < rows;
            if (MODE <= VL_GRAD && live) target = p.target[row] - p.v0 - col0;   // column of this thread's share
            if (MODE == VL_GRAD && live) {
                lse2 = p.lse2[row];
                rest = p.rest[row];
                coef = p.coef[row];
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
            float m2 = VL_NEG, sum = 0.f;
#pragma unroll 1
            for (int c = 0; c < 128; c += 32) {
                uint32_t r[32];
                tmem_ld_32x32(at + c, r);
                tmem_ld_wait();
                if (c == 96) release();
                if (MODE == VL_STATS) {
                    const int words = p.vocab - p.v0 - col0 - c;       // words there are in this chunk
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
                    if (top2 > m2) {
                        sum *= vl_ex2(m2 - top2);
                        m2 = top2;
                    }
                    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int e = 0; e < 32; ++e) part[e & 3] += vl_ex2(fmaf(__uint_as_float(r[e]), VL_LOG2E, -m2));
                    sum += (part[0] + part[1]) + (part[2] + part[3]);
                } else if (MODE == VL_GRAD) {
                    const int words = p.vocab - p.v0 - col0 - c;
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
                    uint4* out = reinterpret_cast<uint4*>(static_cast<unsigned short*>(p.dl) + (long long)row * p.ld_dl + col0 + c);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        out[i] = make_uint4(vl_pack(v[8 * i], v[8 * i + 1], p.mode_bf16), vl_pack(v[8 * i + 2], v[8 * i + 3], p.mode_bf16),
                                            vl_pack(v[8 * i + 4], v[8 * i + 5], p.mode_bf16), vl_pack(v[8 * i + 6], v[8 * i + 7], p.mode_bf16));
                } else if (MODE == VL_HIDDEN) {
                    if (live && col0 + c < p.hidden) {
                        float4* out = reinterpret_cast<float4*>(p.planes + ((long long)w.slice * plan.m_tiles * VL_TILE + row) * p.hidden + col0 + c);
                        const int n4 = min(8, (p.hidden - col0 - c) >> 2);       // (hidden is a multiple of 8)
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            if (i >= n4) break;
                            float4 v = make_float4(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]),
                                                   __uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3]));
                            if (!p.first) {
                                const float4 o = out[i];
                                v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
                            }
                            out[i] = v;
                        }
                    }
                } else {
                    if (p.v0 + row < p.vocab && row < p.piece && col0 + c < p.hidden) {
                        unsigned short* out = static_cast<unsigned short*>(p.d_weight) + (long long)(p.v0 + row) * p.ld_dw + col0 + c;
                        const int n8 = min(4, (p.hidden - col0 - c) >> 3);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (i >= n8) break;
                            uint32_t o[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                o[j] = vl_pack(__uint_as_float(r[8 * i + 2 * j]) * scale, __uint_as_float(r[8 * i + 2 * j + 1]) * scale, p.mode_bf16);
                            reinterpret_cast<uint4*>(out)[i] = make_uint4(o[0], o[1], o[2], o[3]);
                        }
                    }
                }
            }
            if (MODE == VL_STATS) p.parts[(long long)(2 * w.nt + half) * p.rows_pad + row] = make_float2(m2, sum);
            ++n;
        }
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
    __syncthreads();
    if (warp == 0) {
        int start = 0;
        for (int i = 0; i < VL_GATHER_WARPS; ++i) start += before[i];
        for (int c = 0; c < per; c += 32) {
            const long long row = row0 + c + lane;
            const bool in = c + lane < per && row < a.rows;
            const long long t = in ? a.targets[row] : -1;
            const bool part = in && takes_part(t);
            if (in && t >= a.vocab) atomicCAS(a.status, 0, STATUS_CE_TARGET_RANGE);   // treated as ignored, and recorded
            const unsigned mask = __ballot_sync(0xffffffffu, part);
            const int at = start + __popc(mask & ((1u << lane) - 1u));
            if (c + lane < per) place[c + lane] = part ? at : -1;
            if (in) {
                a.place[row] = part ? at : -1;
                if (part) a.target[at] = (int)t;
                else { a.losses[row] = 0.f; a.lse[row] = 0.f; }
            }
            start += __popc(mask);
        }
        if (lane == 0 && row0 + per >= a.rows) *a.count = start;      // (the last CTA)
        if (lane == 0) total = start;
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
        const int count = total, end = vl_div_up(count, VL_TILE) * VL_TILE;
        uint4* out = reinterpret_cast<uint4*>(a.gathered);
        for (long long i = (long long)count * vecs + threadIdx.x; i < (long long)end * vecs; i += VL_GATHER_WARPS * 32)
            out[i] = make_uint4(0u, 0u, 0u, 0u);
    }
}

// Joins a row's maxima and sums: 32 rows by 32 shares of the parts per CTA.
__global__ void __launch_bounds__(1024)
vl_merge_kernel(const VocabLossArgs a, int n_parts) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ float2 join[32][33];
    const int rows = *a.count, row = blockIdx.x * 32 + threadIdx.x;
    if (blockIdx.x * 32 >= rows) return;
    float m = VL_NEG, s = 0.f;
    if (row < rows) {
#pragma unroll 4
        for (int i = threadIdx.y; i < n_parts; i += 32) {
            const float2 x = a.parts[(long long)i * a.rows_pad + row];
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
    const float logit = a.target_logit[at], d = x.x - logit * VL_LOG2E;    // log2 of the others' largest over the target's
    float loss, rest;
    if (d <= 0.f) {
        const float r = x.y * exp2f(d);
        loss = log1pf(r);
        rest = r / (1.f + r);
    } else {
        const float t = x.y + exp2f(-d);
        loss = d * VL_LN2 + logf(t);
        rest = x.y / t;
    }
    a.lse_rows[at] = logit * VL_LOG2E + loss * VL_LOG2E;
    a.rest[at] = rest;
    a.loss_rows[at] = make_float2(loss, logit + loss);
}

// To where the caller's rows are.
__global__ void __launch_bounds__(256)
vl_scatter_kernel(const VocabLossArgs a) {
    grid_dep_wait();
    grid_dep_launch();
    const long long row = (long long)blockIdx.x * 256 + threadIdx.x;
    if (row >= a.rows) return;
    const int at = a.place[row];
    if (at < 0) return;
    const float2 x = a.loss_rows[at];
    a.losses[row] = x.x;
    a.lse[row] = x.y;
}

// ------------------------------------------------------------------------------------- backward's row factors
// Power of two at or above x >= 0, from 2^-95 to 2^126: 0 for zero, 1 for what is not finite.
__device__ __forceinline__ float vl_power(float x) {
    const uint32_t bits = __float_as_uint(x);
    if (bits == 0u || bits >= 0x7F800000u) return bits == 0u ? 0.f : 1.f;
    return __uint_as_float(min(max((bits + 0x007FFFFFu) >> 23, 32u), 253u) << 23);
}

// One CTA: per row that takes part (b + c, b, c) over the row's power of two, times VL_P_SCALE; the largest power.
__global__ void __launch_bounds__(1024)
vl_coef_kernel(const VocabLossArgs a) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ float part[32];
    float top = 0.f;
    for (long long row = threadIdx.x; row < a.rows; row += 1024) {
        const int at = a.place[row];
        if (at < 0) continue;
        const float b = a.d_losses == nullptr ? 0.f : a.d_losses[row * a.d_losses_stride];
        const float c = a.d_lse == nullptr ? 0.f : a.d_lse[row * a.d_lse_stride];
        const float power = vl_power(fmaxf(fabsf(b), fabsf(c)));
        const float inv = power > 0.f ? VL_P_SCALE / power : 0.f;
        a.coef[at] = make_float4((b + c) * inv, b * inv, c * inv, power);
        top = fmaxf(top, power);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x < 32) {
        top = part[threadIdx.x];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (threadIdx.x == 0) {
            a.scales[0] = top;
            a.scales[1] = top / VL_P_SCALE;
        }
    }
}

// The rows times their power over the largest one, exact but for what falls out of the type's range below.
__global__ void __launch_bounds__(256)
vl_scale_rows_kernel(const VocabLossArgs a) {
    grid_dep_wait();
    grid_dep_launch();
    const int rows = *a.count, vecs = (int)(a.hidden / 8), end = vl_div_up(rows, VL_TILE) * VL_TILE;
    const float top = a.scales[0];
    const uint4* in = reinterpret_cast<const uint4*>(a.gathered);
    uint4* out = reinterpret_cast<uint4*>(a.scaled);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)end * vecs; i += (long long)gridDim.x * 256) {
        const int row = (int)(i / vecs);
        const float power = row < rows ? a.coef[row].w : 0.f;
        uint4 v = in[i];
        if (power != top) {
            const float f = power > 0.f ? power / top : 0.f;
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 x = vl_two(w[e], a.bf16);
                w[e] = f > 0.f ? vl_pack(x.x * f, x.y * f, a.bf16) : 0u;
            }
            v = make_uint4(w[0], w[1], w[2], w[3]);
        }
        out[i] = v;
    }
}

// dH of the caller's rows: the planes' sum times the row's power; zeros where the row took no part.
__global__ void __launch_bounds__(256)
vl_hidden_kernel(const VocabLossArgs a, int steps, int slots) {
    grid_dep_wait();
    grid_dep_launch();
    const int rows = *a.count, vecs = (int)(a.hidden / 8);
    const int row_tiles = vl_div_up(rows, VL_TILE);
    const int slices = rows > 0 ? vl_slices(row_tiles * vl_div_up((int)a.hidden, VL_TILE), steps, slots) : 1;
    const long long plane = (long long)row_tiles * VL_TILE * a.hidden;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < a.rows * vecs; i += (long long)gridDim.x * 256) {
        const long long row = i / vecs;
        const int c = (int)(i - row * vecs) * 8, at = a.place[row];
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (at >= 0) {
            const float power = a.coef[at].w * (1.f / VL_P_SCALE);
            const float* src = a.planes + (long long)at * a.hidden + c;
#pragma unroll 4
            for (int z = 0; z < slices; ++z) {
                const float4 x = *reinterpret_cast<const float4*>(src + z * plane), y = *reinterpret_cast<const float4*>(src + z * plane + 4);
                v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
                v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= power;
        }
        reinterpret_cast<uint4*>(static_cast<unsigned short*>(a.d_x) + row * a.hidden)[c / 8] =
            make_uint4(vl_pack(v[0], v[1], a.bf16), vl_pack(v[2], v[3], a.bf16), vl_pack(v[4], v[5], a.bf16), vl_pack(v[6], v[7], a.bf16));
    }
}

// ------------------------------------------------------------------------------------------- host side
static size_t vl_align(size_t n) { return (n + 255) / 256 * 256; }

static long long vl_rows_pad(long long rows) { return (rows + VL_TILE - 1) / VL_TILE * VL_TILE; }

// What the forward keeps for the backward.
struct VlKept {
    size_t count, place, target, lse, rest, gathered, bytes;
};
static VlKept vl_kept(long long rows, long long hidden) {
    VlKept k;
    const size_t pad = (size_t)vl_rows_pad(rows);
    size_t at = 0;
    const auto take = [&](size_t n) { const size_t r = at; at += vl_align(n); return r; };
    k.count = take(4);
    k.place = take((size_t)rows * 4);
    k.target = take(pad * 4);
    k.lse = take(pad * 4);
    k.rest = take(pad * 4);
    k.gathered = take(pad * (size_t)hidden * 2);
    k.bytes = at;
    return k;
}

// Words of a piece: its 16-bit gradient takes at most 64 MiB (it is read back from L2), in whole tiles.
static int vl_piece(long long rows, long long vocab) {
    const long long pad = vl_rows_pad(rows), all = (vocab + VL_TILE - 1) / VL_TILE * VL_TILE;
    long long piece = (64ll << 20) / 2 / pad / VL_TILE * VL_TILE;
    if (piece < 1024) piece = 1024;
    return (int)(piece < all ? piece : all);
}

// Planes of dH in units of rows_pad rows: what any count of rows up to `rows` asks for.
static int vl_planes(long long rows, long long hidden, int piece, int slots) {
    const long long tiles = vl_rows_pad(rows) / VL_TILE;
    long long most = tiles;
    for (long long t = 1; t <= tiles && t <= 4096; ++t) {     // (more tiles than that are one slice)
        const long long n = t * vl_slices((int)t * vl_div_up((int)hidden, VL_TILE), vl_div_up(piece, VL_BK), slots);
        if (n > most) most = n;
    }
    return (int)((most + tiles - 1) / tiles);
}

struct VlScratch {
    size_t parts, loss_rows, target_logit, coef, scales, scaled, dl, planes, bytes;
    int piece;
};

static VlScratch vl_scratch(const VocabLossArgs& a, bool backward) {
    VlScratch s = {};
    const size_t pad = (size_t)vl_rows_pad(a.rows);
    size_t at = 0;
    const auto take = [&](size_t n) { const size_t r = at; at += vl_align(n); return r; };
    if (!backward) {
        s.parts = take((size_t)((a.vocab + VL_TILE - 1) / VL_TILE) * 2 * 8 * pad);
        s.loss_rows = take(pad * 8);
        s.target_logit = take(pad * 4);
    } else {
        s.piece = vl_piece(a.rows, a.vocab);
        s.coef = take(pad * 16);
        s.scales = take(16);
        s.dl = take(pad * (size_t)s.piece * 2);
        if (a.d_x != nullptr)
            s.planes = take((size_t)vl_planes(a.rows, a.hidden, s.piece, a.sm_count / 2) * pad * (size_t)a.hidden * 4);
        if (a.d_weight != nullptr) s.scaled = take(pad * (size_t)a.hidden * 2);
    }
    s.bytes = at;
    return s;
}

size_t vocab_loss_kept_bytes(long long rows, long long hidden) { return vl_kept(rows, hidden).bytes; }

size_t vocab_loss_workspace_bytes(const VocabLossArgs& a, bool backward) { return vl_scratch(a, backward).bytes; }

template <int MODE>
static cudaError_t vl_launch(const VlMaps& maps, const VlParams& p, long long units, int sm_count, cudaStream_t stream) {
    auto kernel = vl_gemm_kernel<MODE>;
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
    cfg.gridDim = dim3((unsigned)(2 * pairs));
    return cudaLaunchKernelEx(&cfg, kernel, maps, p);
}

static bool vl_map(CUtensorMap* map, int bf16, const void* base, long long inner, long long outer, long long pitch, int box_outer) {
    return make_map_2d(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, base, (uint64_t)inner,
                       (uint64_t)outer, (uint64_t)pitch * 2, VL_BK, (uint32_t)box_outer, CU_TENSOR_MAP_SWIZZLE_128B);
}

static void vl_use_kept(VocabLossArgs& a) {
    const VlKept k = vl_kept(a.rows, a.hidden);
    char* base = static_cast<char*>(a.kept);
    a.count = reinterpret_cast<int*>(base + k.count);
    a.place = reinterpret_cast<int*>(base + k.place);
    a.target = reinterpret_cast<int*>(base + k.target);
    a.lse_rows = reinterpret_cast<float*>(base + k.lse);
    a.rest = reinterpret_cast<float*>(base + k.rest);
    a.gathered = base + k.gathered;
    a.rows_pad = vl_rows_pad(a.rows);
}

cudaError_t launch_vocab_loss_fwd(const VocabLossArgs& a_in, cudaStream_t stream, const char** why) {
    *why = "";
    VocabLossArgs a = a_in;
    if (a.rows <= 0) return cudaSuccess;
    vl_use_kept(a);
    const VlScratch s = vl_scratch(a, false);
    char* ws = static_cast<char*>(a.workspace);
    a.parts = reinterpret_cast<float2*>(ws + s.parts);
    a.loss_rows = reinterpret_cast<float2*>(ws + s.loss_rows);
    a.target_logit = reinterpret_cast<float*>(ws + s.target_logit);
    const int per = a.rows <= 4096 ? 8 : 32;
    cudaError_t e = launch_pdl(vl_gather_kernel, dim3((unsigned)((a.rows + per - 1) / per)), dim3(VL_GATHER_WARPS * 32), 0, stream, a, per);
    if (e != cudaSuccess) { *why = "gather"; return e; }
    VlMaps maps;
    if (!vl_map(&maps.a, a.bf16, a.gathered, a.hidden, a.rows_pad, a.hidden, 128) ||
        !vl_map(&maps.b, a.bf16, a.weight, a.hidden, a.vocab, a.ld_w, 128)) {
        *why = "cuTensorMapEncodeTiled";
        return cudaErrorInvalidValue;
    }
    VlParams p = {};
    p.count = a.count; p.status = a.status; p.mode_bf16 = a.bf16;
    p.vocab = (int)a.vocab; p.hidden = (int)a.hidden;
    p.v0 = 0; p.piece = (int)a.vocab;
    p.n_tiles = (int)((a.vocab + VL_TILE - 1) / VL_TILE);
    p.parts = a.parts; p.rows_pad = a.rows_pad; p.target = a.target;
    e = vl_launch<VL_STATS>(maps, p, a.rows_pad / VL_TILE * p.n_tiles, a.sm_count, stream);
    if (e != cudaSuccess) { *why = "statistics"; return e; }
    e = launch_pdl(vl_merge_kernel, dim3((unsigned)((a.rows + 31) / 32)), dim3(32, 32), 0, stream, a, 2 * p.n_tiles);
    if (e != cudaSuccess) { *why = "merge"; return e; }
    e = launch_pdl(vl_scatter_kernel, dim3((unsigned)((a.rows + 255) / 256)), dim3(256), 0, stream, a);
    if (e != cudaSuccess) *why = "scatter";
    return e;
}

cudaError_t launch_vocab_loss_bwd(const VocabLossArgs& a_in, cudaStream_t stream, const char** why) {
    *why = "";
    VocabLossArgs a = a_in;
    if (a.rows <= 0) return cudaSuccess;
    vl_use_kept(a);
    const VlScratch s = vl_scratch(a, true);
    char* ws = static_cast<char*>(a.workspace);
    a.coef = reinterpret_cast<float4*>(ws + s.coef);
    a.scales = reinterpret_cast<float*>(ws + s.scales);
    a.scaled = ws + s.scaled;
    a.planes = reinterpret_cast<float*>(ws + s.planes);
    void* dl = ws + s.dl;
    cudaError_t e = launch_pdl(vl_coef_kernel, dim3(1), dim3(1024), 0, stream, a);
    if (e != cudaSuccess) { *why = "row factors"; return e; }
    if (a.d_weight != nullptr) {
        e = launch_pdl(vl_scale_rows_kernel, dim3((unsigned)(a.sm_count * 8)), dim3(256), 0, stream, a);
        if (e != cudaSuccess) { *why = "row scales"; return e; }
    }
    const int feature_tiles = (int)((a.hidden + VL_TILE - 1) / VL_TILE);
    VlMaps logits, hidden, weight;
    if (!vl_map(&logits.a, a.bf16, a.gathered, a.hidden, a.rows_pad, a.hidden, 128) ||
        !vl_map(&logits.b, a.bf16, a.weight, a.hidden, a.vocab, a.ld_w, 128) ||
        !vl_map(&hidden.a, a.bf16, dl, s.piece, a.rows_pad, s.piece, 128) ||
        !vl_map(&hidden.b, a.bf16, a.weight, a.hidden, a.vocab, a.ld_w, 64) ||
        !vl_map(&weight.a, a.bf16, dl, s.piece, a.rows_pad, s.piece, 64) ||
        !vl_map(&weight.b, a.bf16, a.d_weight != nullptr ? a.scaled : a.gathered, a.hidden, a.rows_pad, a.hidden, 64)) {
        *why = "cuTensorMapEncodeTiled";
        return cudaErrorInvalidValue;
    }
    VlParams p = {};
    p.count = a.count; p.status = a.status; p.mode_bf16 = a.bf16;
    p.vocab = (int)a.vocab; p.hidden = (int)a.hidden;
    p.rows_pad = a.rows_pad; p.target = a.target;
    p.lse2 = a.lse_rows; p.rest = a.rest; p.coef = a.coef; p.dl = dl; p.ld_dl = s.piece;
    p.planes = a.planes; p.slots = a.sm_count / 2; p.first_steps = vl_div_up((int)(a.vocab < s.piece ? a.vocab : s.piece), VL_BK);
    p.d_weight = a.d_weight; p.ld_dw = a.hidden; p.weight_scale = a.scales + 1;
    for (long long v0 = 0; v0 < a.vocab; v0 += s.piece) {
        p.v0 = (int)v0;
        p.piece = (int)(a.vocab - v0 < s.piece ? a.vocab - v0 : s.piece);
        p.n_tiles = vl_div_up(p.piece, VL_TILE);
        const long long row_tiles = a.rows_pad / VL_TILE;
        e = vl_launch<VL_GRAD>(logits, p, row_tiles * p.n_tiles, a.sm_count, stream);
        if (e != cudaSuccess) { *why = "gradient of the logits"; return e; }
        if (a.d_x != nullptr) {
            p.first = v0 == 0 ? 1 : 0;
            e = vl_launch<VL_HIDDEN>(hidden, p, row_tiles * feature_tiles * VL_MAX_SLICES, a.sm_count, stream);
            if (e != cudaSuccess) { *why = "gradient of the hidden states"; return e; }
        }
        if (a.d_weight != nullptr) {
            e = vl_launch<VL_WEIGHT>(weight, p, (long long)p.n_tiles * feature_tiles, a.sm_count, stream);
            if (e != cudaSuccess) { *why = "gradient of the head"; return e; }
        }
    }
    if (a.d_x != nullptr) {
        e = launch_pdl(vl_hidden_kernel, dim3((unsigned)(a.sm_count * 8)), dim3(256), 0, stream, a,
                       p.first_steps, p.slots);
        if (e != cudaSuccess) *why = "sum of the planes";
    }
    return e;
}

}  // namespace nf4
