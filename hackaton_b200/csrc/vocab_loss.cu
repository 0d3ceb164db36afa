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
// per row that is fixed before the sweep (from the first words, in bf16 also the target's own logit), and the sum's 1 / s
// comes at the end. The target is left out of U and of the sums, so that 1 - p_t and a loss near zero keep their digits, and its
// share is added in fp32. Where a row meets a logit too far above its reference for the 16-bit type, its row tile's sweep
// is done again with references from the maxima; the launch for that looks at a flag and leaves. dW needs the final
// lse: the logits once more, in 16-bit dl this time, and one product. A word's row of dW is mostly what its own
// rows' targets add, so that what those dl lose in 16 bits shows: it is kept and added in fp32, for four rows of a word.
// (1229 rows, 5000 words: dW is 2.1e-4 of itself off in fp16, as much as its own rounding alone; without this 3.0e-4.) What the
// probabilities of other words lose is not given back: where one of those holds most of its rows, dH and dW are 1.08 to 1.19 times as far
// off as products and sums in fp32 with the same rounding at the end (at most 1.5 times over 40,000 small random cases).
//
// The tensor cores bound it, and their clock the power that the chip may take, so what counts is that they never pause
// and that little moves. CTA pairs (tcgen05.mma.cta_group::2) own a 256 x 256 tile, 128 rows by 256 columns of fp32 in
// each CTA's tensor memory, twice: while eight warps work on one tile's values the next one is being multiplied.
// Operands come by TMA in 64-deep steps through a ring of six. A sweep is one kernel (vl_sweep_kernel): first logits, then
// the product with the 16-bit piece, as units of one list that the pairs draw tickets from,
//     P(0) P(1)  P(2) Q(0)  P(3) Q(1)  ...  Q(last)     P(i): logits tiles of piece i, Q(i): tiles of the product with it
// (here two pieces behind), each unit waiting, with counters in memory, for what it reads or overwrites; all of that has
// smaller tickets, which running CTAs have drawn, so that nothing depends on how many CTAs are resident. (As a launch per
// piece and product, a pair idled 11 of 66 us per launch. Tickets handed on with fences of cluster scope cost the thread
// that issues the products 2300 of 21,400 cycles a unit; as asynchronous stores that a barrier counts, 200.) The 16-bit
// piece is laid out in blocks of [rows][64 words], which is how TMA reads it along either side. Measured, 151,936 words x
// 1536, mean of 500 in a row (the chip at its power limit, 1.1 to 1.2 GHz): U and the sums for 2048 rows 1651 us
// (1158 TFLOP/s), for 1229 rows 1088 us (1054), dW of 1229 rows 1038 us (1105); a library's product of 8192^3 then 1340.
// Nothing is added in an order that depends on timing: U's tiles take the pieces' products one after the other.
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
constexpr float VL_P_SCALE = 8192.f;       // of the 16-bit gradient: at most 2 * 2^13, down to 2^-24 / 2^13
// A row's reference for its exponentials (base 2): the first words' maximum less VL_BELOW; fp16 takes what lies up to 2^15 above it,
// bf16 2^100. The target has no part in it, as it has none in the sums: fp16 then holds each word to 2^-28 of the largest or better,
// however certain the row is. (With 2^10 below the target as the least, a target 19 nats above the next word left dH 1.8e-3 of itself off,
// one 23 above 7e-2. 151,936 words, one of them 4 to 20 nats above all others, those spread by 1 to 3: the largest at 2^3 costs dH 4e-5 at
// most, at 1 4e-4, at 2^-3 2e-3.) bf16's range has room for 2^10 below the target too, which spares second sweeps.
constexpr float VL_BELOW = 3.f, VL_BELOW_TARGET_BF16 = 10.f;
constexpr float VL_ROOM_F16 = 15.f, VL_ROOM_BF16 = 100.f;
constexpr int VL_TILE = 256;               // rows and columns of a pair's tile
constexpr int VL_PROBE_TILES = 8;          // tiles of words that the reference is taken from
// Pieces (vl_shape). Forward as large as VL_PIECE_UNITS tiles of 256 x 256 allow (67 MB): each adds to all of U, which costs
// more than a piece that leaves L2. (U of 2048 rows, 151,936 words x 1536, the mean of 500 in a row: 75 pieces 1674 us, 38
// pieces, three of which fill L2, 1745, 10 pieces 1651, 5 of twice the size 1627.) Few row tiles: pieces so small that
// there are VL_PRODUCTS units of the product, two for each of 74 pairs (256 rows in one plane: 24 tiles of words 320 us, 8
// 671, 64 366). The backward's product is written, not added: small pieces that stay in L2 (1229 rows: 8 tiles of words 1030 us, 16
// 1053, 64 1069). With many rows at least VL_PIECE_LEAST tiles of words up to VL_PIECE_MOST tiles (a gigabyte of scratch),
// one behind that.
// A piece's product comes `lag` pieces behind its logits in the list, so many that VL_AHEAD_ units of logits (and as much work
// on products) lie between: what a unit waits for was drawn well before it, not a moment ago by a pair that is still at it.
// (U of 1229 rows, 80 units to a piece: one piece behind 1201 us, two 1107; of 256 rows, 24 units: six 304, eight 287,
// twelve 276. dW of 16 rows x 3584, 8 units: two 880, four 717, eight 692; of 1229 rows, 40 units: two 1030, three 1038.)
constexpr int VL_PIECE_UNITS = 512, VL_PIECE_TILES = 64, VL_BWD_TILES = 8, VL_PIECE_LEAST = 8, VL_PIECE_MOST = 2048;
constexpr int VL_AHEAD_FWD = 278, VL_AHEAD_BWD = 111, VL_MOST_LAG = 24;
constexpr int VL_PRODUCTS = 148;
constexpr int VL_PLANE_ROWS = 1024;

constexpr int VL_BK = 64;
// The tensor cores cut off what an addition to an accumulator leaves behind its 24 bits, always in one direction, so
// that a logit's error grows with the length of its chain of additions. A chain of logits is at most VL_CHAIN steps of 64;
// longer ones are cut, and the parts added in the epilogue's registers with rounding. (3584 features, losses against 64 bits: one
// chain 1.2e-6 in norm, chains of 32 steps 4e-7, of 8 1.2e-7; fp32 products and sums 1.5e-7.) Up to VL_CHAIN_ROWS row tiles,
// among few rows, a single confident one's small loss shows (2 rows of 2920 features, chains of 32 3.0e-6, of 8 below 1e-6), and the
// cuts cost nothing: at most VL_CHAIN_FEW steps, and so where the words take the long side (64 x 3584 against 151,936 words 180.0 us
// in four chains of 14 steps, 180.5 in seven of 8). (2048 rows x 1536, U: 1725 us in one chain, 1760 in two, 1797 in three.)
constexpr int VL_CHAIN = 32, VL_CHAIN_FEW = 8, VL_CHAIN_ROWS = 2;
constexpr int VL_LINKS = 16;               // rows of a word (or that share its place in the table) up to which they are looked up
constexpr int VL_FEW_CHAINS = 4;           // that share a buffer, 64 columns each
constexpr int VL_EPI_WARPS = 8;
constexpr int VL_SMEM_MAX = 232448, VL_BAR_ROOM = 512;
// Shared memory of a CTA: the ring (128 rows of A and ROWS of B per step), a box of 32 rows x 128 bytes per epilogue warp
// on its way out (OUT), barriers.
template <int ROWS, int STAGES_, bool OUT>
struct VlSmem {
    static constexpr int STAGES = STAGES_;
    static constexpr int A_BYTES = 128 * VL_BK * 2, B_BYTES = ROWS * VL_BK * 2;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int STAGING_OFF = STAGES * STAGE_BYTES;
    static constexpr int BAR_OFF = STAGING_OFF + (OUT ? VL_EPI_WARPS * 4096 : 0);
    static constexpr int TOTAL = BAR_OFF + VL_BAR_ROOM + 1024;    // + slack for 1024-byte alignment
    static_assert(TOTAL <= VL_SMEM_MAX && BAR_OFF % 8 == 0, "exceeds the 227 KB of shared memory per CTA");
};
constexpr int VL_THREADS = 64 + VL_EPI_WARPS * 32;

// Statistics alone (no gradient of the hidden states): one product, nothing to write but a maximum and a sum.
enum VlMode {
    VL_STATS = 0,    // A = gathered rows [R, K], B = W [V, K]         -> maximum and sum per row and half tile
    VL_FEW = 1       // A = W, B = at most 64 gathered rows, words as M -> per row and warp
};

struct VlMaps {
    CUtensorMap a, b;
};

struct VlParams {
    const int* count;        // rows that take part
    int* status;
    int bf16;
    int vocab, hidden;
    int word_tiles;          // to be looked at
    int n_rows;              // VL_FEW: columns of the accumulator, 32 or 64
    int cta_tiles;           // VL_FEW: tiles of a CTA, one behind the other,
    int tile_words;          // and the words of each, at most 128
    const int* target;       // per gathered row
    float2* parts;           // [parts][rows_pad]: maximum (base 2), sum relative to it
    long long rows_pad;
};

struct VlSweepMaps {
    CUtensorMap rows, words;      // P: gathered rows, W
    CUtensorMap piece_in;         // Q: the piece, as rows (forward) or as words (backward) of the product
    CUtensorMap other;            // Q: W with features along N (forward), gathered rows with features along N (backward)
    CUtensorMap piece_out;        // P writes the piece
    CUtensorMap out;              // Q adds to U (forward, fp32), writes dW (backward)
};

struct VlSweepParams {
    const int* count;
    int* status;
    int bf16;
    int vocab, hidden;
    int word_tiles;
    long long rows_pad;
    const int* target;
    void* piece;             // [buffer][block of 64 words][rows of the tiles][64]
    // counters, zero before: units drawn; per piece and row tile (backward: word tile) warps that have written their
    // part of the piece, units that have read it; per tile of U warps that have added theirs
    int* ticket;
    int* written;
    int* read;
    int* added;
    int pitch;               // counters per piece
    // forward
    float2* parts;           // [2 * word tiles][rows_pad]: maximum (base 2), sum relative to the reference
    const float* refs;       // [rows_pad]
    int* flags;              // [row tiles]: whether a row outgrew its reference
    const int* list;         // a sweep done again: number of row tiles, their indexes
    int again;
    // backward
    const float* lse2;
    const float* rest;       // 1 - p of the target
    const float4* coef;      // ((b + c), b, c) over the common power of two, times VL_P_SCALE, and what the target's dl loses
    const int* links;
    const int* first;
    const int* next;
    const void* gathered;
    void* d_weight;          // [vocab, hidden]
    const float* weight_scale;
};

__host__ __device__ inline int vl_div_up(int a, int b) { return (a + b - 1) / b; }

// Rows that U's planes have together. Pieces add to the planes in turn, as many as there is room for: where there are few
// row tiles, one addition behind the other, 8 us each, would be most of the time (256 rows: 341 us, with four planes 287).
__host__ __device__ inline long long vl_plane_rows(long long rows_pad) { return rows_pad > VL_PLANE_ROWS ? rows_pad : VL_PLANE_ROWS; }
__host__ __device__ inline int vl_planes(long long rows_pad, int row_tiles) {
    return row_tiles > 0 ? (int)(vl_plane_rows(rows_pad) / VL_TILE / row_tiles) : 1;
}

struct VlShape {
    int tiles, pieces, lag, buffers;      // tiles of words in a piece; pieces that have a buffer at a time
};
__host__ __device__ inline VlShape vl_shape(int row_tiles, int word_tiles, int feature_tiles, bool backward) {
    VlShape s;
    const int a = row_tiles > 0 ? row_tiles : 1;
    int least = VL_PIECE_MOST / a;
    if (least > VL_PIECE_LEAST) least = VL_PIECE_LEAST;
    if (least < 1) least = 1;
    long long t = VL_BWD_TILES;
    if (!backward) {
        t = (long long)word_tiles * a * feature_tiles / VL_PRODUCTS;
        if (t > VL_PIECE_TILES) t = VL_PIECE_TILES;
    }
    if (t > VL_PIECE_UNITS / a) t = VL_PIECE_UNITS / a;
    if (t < least) t = least;
    if (t > word_tiles) t = word_tiles;
    s.tiles = (int)t;
    s.pieces = vl_div_up(word_tiles, s.tiles);
    const long long units = (long long)a * s.tiles;
    const int ahead = backward ? VL_AHEAD_BWD : VL_AHEAD_FWD;
    s.lag = units >= ahead ? 1 : vl_div_up(ahead, (int)units);
    if (s.lag > VL_MOST_LAG) s.lag = VL_MOST_LAG;
    if (s.lag > s.pieces) s.lag = s.pieces;
    s.buffers = s.lag + 2 < s.pieces ? s.lag + 2 : s.pieces;
    return s;
}

__device__ __forceinline__ float vl_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void vl_sts128(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// dl of the target: c p_t - b (1 - p_t).
__device__ __forceinline__ float vl_hit(float b, float c, float rest) { return c * (1.f - rest) - b * rest; }

// Steps of a chain where there are so many.
__device__ __forceinline__ int vl_chain(int steps, int row_tiles) {
    return vl_div_up(steps, vl_div_up(steps, row_tiles <= VL_CHAIN_ROWS ? VL_CHAIN_FEW : VL_CHAIN));
}

// acc += a thread's 128 columns of a chain that is not the last.
__device__ __forceinline__ void vl_add_chain(float (&acc)[128], uint32_t at) {
#pragma unroll
    for (int c = 0; c < 128; c += 16) {
        uint32_t r[16];
        tmem_ld_32x16(at + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[c + e] += __uint_as_float(r[e]);
    }
}

// The largest of 32 accumulator values (a NaN left out).
__device__ __forceinline__ float vl_top(const uint32_t (&r)[32]) {
    float top = __uint_as_float(r[0]);
#pragma unroll
    for (int e = 1; e < 32; ++e) top = fmaxf(top, __uint_as_float(r[e]));
    return top;
}

// Of 32 words' logits, what lies behind the vocabulary and the target's own count as nothing.
__device__ __forceinline__ void vl_leave_out(uint32_t (&r)[32], int words, int target) {
    if (!__any_sync(0xffffffffu, words < 32 || (unsigned)target < 32u)) return;
#pragma unroll
    for (int e = 0; e < 32; ++e)
        if (e >= words || e == target) r[e] = __float_as_uint(VL_NEG);
}

// A word to a CTA of the cluster, its arrival and its bytes counted by a barrier there.
__device__ __forceinline__ void vl_send(uint32_t cluster_addr, int value, uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], 4;" ::"r"(cluster_bar) : "memory");
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];"
                 ::"r"(cluster_addr), "r"(value), "r"(cluster_bar) : "memory");
}

__device__ __forceinline__ float2 vl_two(uint32_t w, int bf16) {
    if (bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

__device__ __forceinline__ uint32_t vl_pack(float a, float b, int bf16) {
    if (bf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <int MODE>
using VlSmemOf = VlSmem<MODE == VL_FEW ? 32 : 128, MODE == VL_FEW ? 10 : 7, false>;
constexpr int VL_FEW_DEEP = 2;             // steps of the ring that come and go together

__device__ __forceinline__ float2 vl_join(float2 x, float2 y) {
    const float top = fmaxf(x.x, y.x);
    return make_float2(top, x.y * vl_ex2(x.x - top) + y.y * vl_ex2(y.x - top));
}

// tcgen05 descriptors: K-major tiles are rows of 128 bytes, eight rows 1024 bytes apart; MN-major ones 64 steps of 128
// bytes (64 values along M or N), the next 64 values 8192 bytes on.
constexpr uint64_t VL_K_MAJOR = make_smem_desc(0, 16, 1024, LAYOUT_SW128);
constexpr uint64_t VL_MN_MAJOR = make_smem_desc(0, 8192, 1024, LAYOUT_SW128);

// One 64-deep step of a pair's tile.
__device__ __forceinline__ void vl_mma_step(uint32_t d_tmem, uint32_t a4, uint32_t b4, bool a_mn, bool b_mn, uint32_t idesc, bool first) {
    const uint32_t a_lo = a4 + (uint32_t)((a_mn ? VL_MN_MAJOR : VL_K_MAJOR) & 0xFFFFFFFFu), a_hi = (uint32_t)((a_mn ? VL_MN_MAJOR : VL_K_MAJOR) >> 32);
    const uint32_t b_lo = b4 + (uint32_t)((b_mn ? VL_MN_MAJOR : VL_K_MAJOR) & 0xFFFFFFFFu), b_hi = (uint32_t)((b_mn ? VL_MN_MAJOR : VL_K_MAJOR) >> 32);
    const uint32_t a_step = (a_mn ? 16 * 128 : 32) >> 4, b_step = (b_mn ? 16 * 128 : 32) >> 4;
#pragma unroll
    for (int k = 0; k < VL_BK / 16; ++k)
        umma_f16_words<2>(d_tmem, a_lo + a_step * k, a_hi, b_lo + b_step * k, b_hi, idesc, first && k == 0 ? 0u : 1u);
}

__device__ __forceinline__ uint32_t vl_idesc(int n, bool a_mn, bool b_mn, int bf16) {
    return make_idesc_f16((uint32_t)n, a_mn ? 1u : 0u, b_mn ? 1u : 0u, VL_TILE) | (bf16 ? (1u << 7) | (1u << 10) : 0u);
}

template <int MODE>
__global__ void __launch_bounds__(VL_THREADS, 1)
vl_stats_kernel(const __grid_constant__ VlMaps maps, const __grid_constant__ VlParams p) {
    using L = VlSmemOf<MODE>;
    constexpr int DEEP = MODE == VL_FEW ? VL_FEW_DEEP : 1, STAGES = L::STAGES / DEEP, STAGE_BYTES = DEEP * L::STAGE_BYTES;
    extern __shared__ uint8_t vl_smem[];
    const uint32_t base = (smem_u32(vl_smem) + 1023u) & ~1023u;
    uint8_t* gen = vl_smem + (base - smem_u32(vl_smem));
    const uint32_t bar = base + L::BAR_OFF;
    auto bar_full = [&](int s) { return bar + 8u * s; };                        // leader: both CTAs' operands
    auto bar_landed = [&](int s) { return bar + 8u * (STAGES + s); };           // peer: its own
    auto bar_empty = [&](int s) { return bar + 8u * (2 * STAGES + s); };
    auto bar_done = [&](int b) { return bar + 8u * (3 * STAGES + b); };         // accumulator complete
    auto bar_drained = [&](int b) { return bar + 8u * (3 * STAGES + 2 + b); };
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + L::BAR_OFF + 8 * (3 * STAGES + 4));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + L::BAR_OFF + 8 * (3 * STAGES + 4) + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int pair = (int)(blockIdx.x >> 1), pairs = (int)(gridDim.x >> 1);

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
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
        tmem_relinquish_pair();
    }
    // The first words come to L2 while the kernel before gathers the rows.
    const int word_begin = MODE == VL_FEW ? (int)blockIdx.x * p.cta_tiles * p.tile_words : 0;
    if (MODE == VL_FEW && warp == 0 && lane == 0 && word_begin < p.vocab)
        for (int k = 0; k < L::STAGES && k * VL_BK < p.hidden; ++k) tma_prefetch_2d(&maps.a, k * VL_BK, word_begin);
    grid_dep_wait();
    grid_dep_launch();
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    const int rows = *p.count, row_tiles = vl_div_up(rows, VL_TILE), steps = vl_div_up(p.hidden, VL_BK * DEEP);
    const int chain = MODE == VL_FEW ? vl_div_up(steps, vl_div_up(steps, VL_CHAIN_FEW / DEEP)) : vl_chain(steps, row_tiles);
    // Few rows: a pair's units are its tiles.
    const int units = rows == 0 ? 0 : MODE == VL_FEW ? (pair + 1) * p.cta_tiles : row_tiles * p.word_tiles;
    const int unit0 = MODE == VL_FEW ? pair * p.cta_tiles : pair, stride = MODE == VL_FEW ? 1 : pairs;
    int fail = 0;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t g = 0;
            for (int u = unit0; u < units && !fail; u += stride) {
                const int am = MODE == VL_FEW ? word_begin + (u - unit0) * p.tile_words : u % row_tiles * VL_TILE + (int)rank * 128;
                const int bn = MODE == VL_FEW ? (int)rank * (p.n_rows / 2) : u / row_tiles * VL_TILE + (int)rank * 128;
                const int bytes = DEEP * (MODE == VL_FEW ? p.tile_words * 128 + p.n_rows * 64 : L::A_BYTES + L::B_BYTES);
                for (int it = 0; it < steps; ++it, ++g) {
                    const int s = (int)(g % STAGES);
                    if (!mbar_wait_cluster(bar_empty(s), ((g / STAGES) & 1u) ^ 1u, abort_flag)) { fail = 1; break; }
                    const uint32_t landed = rank == 0 ? bar_full(s) : bar_landed(s);
                    const uint32_t sa = base + (uint32_t)s * STAGE_BYTES, sb = sa + DEEP * L::A_BYTES;
                    mbar_arrive_expect_tx(landed, bytes);
#pragma unroll
                    for (int k = 0; k < DEEP; ++k) {       // (behind the features: zeros)
                        const int x = (it * DEEP + k) * VL_BK;
                        tma_load_2d(sa + k * L::A_BYTES, &maps.a, x, am, landed);
                        tma_load_2d(sb + k * L::B_BYTES, &maps.b, x, bn, landed);
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            const uint32_t idesc = vl_idesc(MODE == VL_FEW ? p.n_rows : VL_TILE, false, false, p.bf16);
            const uint32_t base4 = (base & 0x3FFFFu) >> 4;
            uint32_t g = 0, n = 0;
            for (int u = unit0; u < units && !fail; u += stride) {
                uint32_t d = 0;
                for (int at = 0, k = 0; at < steps && !fail; at += chain, ++k) {
                    if (MODE != VL_FEW || k % VL_FEW_CHAINS == 0) {      // a buffer to a chain, or (few rows) to some of a tile's
                        if (!mbar_wait_cluster(bar_drained(n & 1u), ((n >> 1) & 1u) ^ 1u, abort_flag)) { fail = 6; break; }
                        tc_fence_after_sync();
                        d = tmem + (n & 1u) * VL_TILE;
                    }
                    const int end = min(at + chain, steps);
                    for (int it = at; it < end; ++it, ++g) {
                        const int s = (int)(g % STAGES);
                        if (!mbar_wait_cluster(bar_full(s), (g / STAGES) & 1u, abort_flag)) { fail = 3; break; }
                        tc_fence_after_sync();
                        const uint32_t a4 = base4 + (uint32_t)s * (STAGE_BYTES >> 4), b4 = a4 + DEEP * (L::A_BYTES >> 4);
#pragma unroll
                        for (int k = 0; k < DEEP; ++k)
                            vl_mma_step(d, a4 + k * (L::A_BYTES >> 4), b4 + k * (L::B_BYTES >> 4), false, false, idesc, it == at && k == 0);
                        umma_commit_pair(bar_empty(s), (uint16_t)3);
                    }
                    d += 64;
                    if (!fail && (MODE != VL_FEW || end == steps || k % VL_FEW_CHAINS == VL_FEW_CHAINS - 1))
                        umma_commit_pair(bar_done(n++ & 1u), (uint16_t)3);
                }
            }
        } else if (lane == 0) {
            const uint32_t lead_full0 = mapa_shared(bar_full(0), 0u);
            uint32_t g = 0;
            for (int u = unit0; u < units && !fail; u += stride) {
                for (int it = 0; it < steps; ++it, ++g) {
                    const int s = (int)(g % STAGES);
                    if (!mbar_wait(bar_landed(s), (g / STAGES) & 1u, abort_flag)) { fail = 8; break; }
                    mbar_arrive_cluster(lead_full0 + 8u * s);
                }
            }
        }
    } else if constexpr (MODE == VL_FEW) {
        // ------------------------------------------------------------------ epilogue: a word's values of half the rows
        // (Lanes behind a tile's words hold what the ring held before.) A thread keeps maximum and sum of the words that come by its lane, for each of its 16 or 32 rows, over all tiles;
        // the lanes of a warp meet at the end.
        const int q = warp & 3, half = (warp - 2) >> 2, n = p.n_rows / 2, row0 = half * n;
        const uint32_t lead_drained = mapa_shared(bar_drained(0), 0u);
        const int target = lane < n && row0 + lane < rows ? p.target[row0 + lane] : -1;
        float m[32], s[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) { m[j] = VL_NEG; s[j] = 0.f; }
        uint32_t buffer = 0;
        for (int u = unit0; u < units && !fail; u += stride) {
            const int word0 = word_begin + (u - unit0) * p.tile_words + q * 32;
            float r[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = 0.f;
            for (int it = 0; it < steps; it += VL_FEW_CHAINS * chain, ++buffer) {
                const int b = (int)(buffer & 1u);
                if (!mbar_wait(bar_done(b), (buffer >> 1) & 1u, abort_flag)) { fail = 5; break; }
                tc_fence_after_sync();
                for (int c = 0; c < VL_FEW_CHAINS && it + c * chain < steps; ++c) {
                    const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + b * VL_TILE + c * 64 + row0;
#pragma unroll
                    for (int j = 0; j < 32; j += 16) {
                        if (j >= n) break;
                        uint32_t h[16];
                        tmem_ld_32x16(at + j, h);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; ++e) r[j + e] += __uint_as_float(h[e]);
                    }
                }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(lead_drained + 8u * b);
            }
            if (fail) break;
            const bool there = word0 + lane < p.vocab && q * 32 + lane < p.tile_words;
            const unsigned hits = __ballot_sync(0xffffffffu, (unsigned)(target - word0) < 32u);    // rows whose target is here
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                if (j >= n) break;
                float x2 = there ? r[j] * VL_LOG2E : VL_NEG;
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
                const float2 x = vl_join(make_float2(m[j], s[j]), make_float2(__shfl_xor_sync(0xffffffffu, m[j], o),
                                                                              __shfl_xor_sync(0xffffffffu, s[j], o)));
                m[j] = x.x;
                s[j] = x.y;
            }
            if (lane == 0) p.parts[(long long)(blockIdx.x * 4 + q) * p.rows_pad + row0 + j] = make_float2(m[j], s[j]);
        }
    } else {
        // ------------------------------------------------------------------ epilogue: a row's half tile per thread
        const int q = warp & 3, half = (warp - 2) >> 2;
        const uint32_t lead_drained = mapa_shared(bar_drained(0), 0u);
        uint32_t n = 0;
        for (int u = pair; u < units && !fail; u += pairs, ++n) {
            float acc[128];
#pragma unroll
            for (int e = 0; e < 128; ++e) acc[e] = 0.f;
            for (int it = chain; it < steps; it += chain, ++n) {
                if (!mbar_wait(bar_done(n & 1u), (n >> 1) & 1u, abort_flag)) { fail = 5; break; }
                tc_fence_after_sync();
                vl_add_chain(acc, tmem + ((uint32_t)(q * 32) << 16) + (n & 1u) * VL_TILE + half * 128);
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(lead_drained + 8u * (n & 1u));
            }
            if (fail) break;
            const int row = u % row_tiles * VL_TILE + (int)rank * 128 + q * 32 + lane, nt = u / row_tiles;
            const int col0 = nt * VL_TILE + half * 128, b = (int)(n & 1u);
            const int target = row < rows ? p.target[row] - col0 : -1;      // column of this thread's share
            if (!mbar_wait(bar_done(b), (n >> 1) & 1u, abort_flag)) { fail = 5; break; }
            tc_fence_after_sync();
            const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + b * VL_TILE + half * 128;
            float m2 = VL_NEG, sum = 0.f;
#pragma unroll
            for (int c = 0; c < 128; c += 32) {
                uint32_t r[32];
                tmem_ld_32x32(at + c, r);
                tmem_ld_wait();
                if (c == 96) {
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(lead_drained + 8u * b);
                }
#pragma unroll
                for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) + acc[c + e]);
                vl_leave_out(r, p.vocab - col0 - c, target - c);
                const float top2 = vl_top(r) * VL_LOG2E;
                if (top2 > m2) {
                    sum *= vl_ex2(m2 - top2);
                    m2 = top2;
                }
                float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 32; ++e) part[e & 3] += vl_ex2(fmaf(__uint_as_float(r[e]), VL_LOG2E, -m2));
                sum += (part[0] + part[1]) + (part[2] + part[3]);
            }
            p.parts[(long long)(2 * nt + half) * p.rows_pad + row] = make_float2(m2, sum);
        }
    }

    if (fail) give_up(p.status, 100 + fail);
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem, 512);
    }
}

// ------------------------------------------------------------------------------------- the sweep
struct VlUnit {
    bool q;              // a tile of the product with the piece, not of the logits
    int piece, tiles;    // the piece, its tiles of words
    int mt;              // row tile (P, forward's Q)
    int slot;            // where its counters are: row tile among those of the sweep (forward), word tile of the piece
    int nt;              // P: word tile of the piece; Q: feature tile
    int steps, chain;    // of 64; accumulated in one go
};

struct VlList {          // the list of units
    int rows, row_tiles, active, feature_tiles, tiles, pieces, lag, buffers, planes, last_tiles, p, q, p_last, q_last, total;
};

template <bool BWD>
__device__ __forceinline__ VlList vl_list(const VlSweepParams& p) {
    VlList w;
    w.rows = *p.count;
    w.row_tiles = vl_div_up(w.rows, VL_TILE);
    w.active = p.again ? p.list[0] : w.row_tiles;
    w.feature_tiles = vl_div_up(p.hidden, VL_TILE);
    const VlShape s = vl_shape(w.row_tiles, p.word_tiles, w.feature_tiles, BWD);
    w.tiles = s.tiles;
    w.pieces = s.pieces;
    w.lag = s.lag;
    w.buffers = s.buffers;
    w.planes = vl_planes(p.rows_pad, w.row_tiles);
    w.last_tiles = p.word_tiles - (w.pieces - 1) * w.tiles;
    w.p = w.active * w.tiles;
    w.p_last = w.active * w.last_tiles;
    w.q = (BWD ? w.tiles : w.active) * w.feature_tiles;
    w.q_last = (BWD ? w.last_tiles : w.active) * w.feature_tiles;
    w.total = (w.pieces - 1) * (w.p + w.q) + w.p_last + w.q_last;
    return w;
}

template <bool BWD>
__device__ __forceinline__ VlUnit vl_unit(int k, const VlSweepParams& p, const VlList& w) {
    VlUnit r;
    const int p_units = max(w.p, 1), lead = w.lag;           // pieces of which only the logits come first
    const int head = w.pieces > w.lag ? w.lag * w.p : (w.pieces - 1) * w.p + w.p_last;
    r.q = k >= head;
    if (!r.q) {
        r.piece = min(k / p_units, lead - 1);
        k -= r.piece * w.p;
    } else {
        k -= head;
        const int blocks = w.pieces - lead;      // each P(block + lag), Q(block); behind the last the Q that are left
        int first = 0;
        if (blocks > 0) {
            first = min(k / (w.p + w.q), blocks - 1);
            k -= first * (w.p + w.q);
            const int ps = first == blocks - 1 ? w.p_last : w.p;
            r.q = k >= ps;
            r.piece = first + w.lag;
            if (r.q) k -= ps;
        }
        if (r.q) {
            const int more = first >= blocks - 1 ? min(k / w.q, w.pieces - 1 - first) : 0;
            r.piece = first + more;
            k -= more * w.q;
        }
    }
    r.tiles = r.piece == w.pieces - 1 ? w.last_tiles : w.tiles;
    const int width = r.q && BWD ? r.tiles : w.active, first = k % width;
    r.nt = k / width;
    r.mt = r.q && BWD ? 0 : p.again ? p.list[1 + first] : first;
    r.slot = BWD ? (r.q ? first : r.nt) : first;
    r.steps = !r.q ? vl_div_up(p.hidden, VL_BK) : BWD ? vl_div_up(w.rows, VL_BK) : r.tiles * (VL_TILE / VL_BK);
    r.chain = r.q ? r.steps : vl_chain(r.steps, w.row_tiles);
    return r;
}

__device__ __forceinline__ int vl_counted(const int* counter) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(counter) : "memory");
    return v;
}

// Bounded wait for a counter in memory. What its writers wrote before is visible behind it, to TMA too. `before`: done
// once, before there is anything to wait for.
template <typename F>
__device__ __forceinline__ bool vl_wait_count(const int* counter, int least, volatile int* abort_flag, F before) {
    if (least <= 0) return true;
    unsigned long long t0 = 0;
    for (;;) {
        if (vl_counted(counter) >= least) break;
        if (t0 == 0) before();
        const unsigned long long now = globaltimer_ns();
        if (t0 == 0) t0 = now;
        if (*abort_flag) return false;
        if (now - t0 > WAIT_TIMEOUT_NS) {
            *abort_flag = 1;
            return false;
        }
        __nanosleep(100);
    }
    asm volatile("fence.proxy.async;" ::: "memory");
    return true;
}

// Counts one more, behind everything this thread wrote or waited for, its TMA stores included.
__device__ __forceinline__ void vl_count(int* counter) {
    asm volatile("fence.proxy.async;" ::: "memory");
    asm volatile("red.release.gpu.global.add.s32 [%0], 1;" ::"l"(counter) : "memory");
}

constexpr int VL_TICKETS = 2;        // units that a pair has drawn and its epilogue not begun, at most
constexpr int VL_SWEEP_THREADS = VL_THREADS + 32;

template <bool BWD>
__global__ void __launch_bounds__(VL_SWEEP_THREADS, 1)
vl_sweep_kernel(const __grid_constant__ VlSweepMaps maps, const __grid_constant__ VlSweepParams p) {
    using L = VlSmem<128, 6, true>;
    constexpr int STAGES = L::STAGES;
    constexpr int BARS = 3 * STAGES + 4 + 2 * VL_TICKETS;
    constexpr uint32_t ALL = 2 * (VL_EPI_WARPS + 2) + 1;  // who reads a ticket: both CTAs' TMA, MMA (peer: its word) and epilogue, the counter
    extern __shared__ uint8_t vl_smem[];
    const uint32_t base = (smem_u32(vl_smem) + 1023u) & ~1023u;
    uint8_t* gen = vl_smem + (base - smem_u32(vl_smem));
    const uint32_t bar = base + L::BAR_OFF;
    auto bar_full = [&](int s) { return bar + 8u * s; };
    auto bar_landed = [&](int s) { return bar + 8u * (STAGES + s); };
    auto bar_empty = [&](int s) { return bar + 8u * (2 * STAGES + s); };
    auto bar_done = [&](int b) { return bar + 8u * (3 * STAGES + b); };
    auto bar_drained = [&](int b) { return bar + 8u * (3 * STAGES + 2 + b); };
    auto bar_drawn = [&](int k) { return bar + 8u * (3 * STAGES + 4 + k); };                    // a ticket is there
    auto bar_taken = [&](int k) { return bar + 8u * (3 * STAGES + 4 + VL_TICKETS + k); };       // leader: all have read it
    static_assert(8 * BARS + 8 + 4 * VL_TICKETS <= VL_BAR_ROOM, "barrier area");
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + L::BAR_OFF + 8 * BARS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + L::BAR_OFF + 8 * BARS + 4);
    const uint32_t tickets = base + L::BAR_OFF + 8 * BARS + 8;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    if (!BWD && p.again) {     // nearly always there is nothing to do again
        grid_dep_wait();
        if (p.list[0] == 0) return;
    }

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(bar_full(s), 2);
            mbar_init(bar_landed(s), 1);
            mbar_init(bar_empty(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(bar_done(b), 1);
            mbar_init(bar_drained(b), 2 * VL_EPI_WARPS + 1);
        }
        for (int k = 0; k < VL_TICKETS; ++k) {
            mbar_init(bar_drawn(k), 1);
            mbar_init(bar_taken(k), ALL);
        }
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&maps.rows);
        tma_prefetch_desc(&maps.words);
        tma_prefetch_desc(&maps.piece_in);
        tma_prefetch_desc(&maps.other);
        tma_prefetch_desc(&maps.piece_out);
        tma_prefetch_desc(&maps.out);
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
    const VlList list = vl_list<BWD>(p);
    const int rows = list.rows, rows_dev = list.row_tiles * VL_TILE;
    const int buffer_rows = list.tiles * (VL_TILE / 64) * rows_dev;     // of 64 words, in one buffer
    int fail = 0;

    // The next unit's ticket, or -1 behind the last; every reader takes them in turn: one lane for itself, or a warp, of
    // which all lanes have read before one says so.
    const uint32_t lead_taken0 = mapa_shared(bar_taken(0), 0u);
    uint32_t drawn = 0;
    auto next_ticket = [&](bool whole_warp) -> int {
        const int k = (int)(drawn % VL_TICKETS);
        if (!mbar_wait(bar_drawn(k), (drawn / VL_TICKETS) & 1u, abort_flag)) { fail = 9; return -1; }
        int t;
        asm volatile("ld.shared.s32 %0, [%1];" : "=r"(t) : "r"(tickets + 4u * k) : "memory");
        if (whole_warp) t = __shfl_sync(0xffffffffu, t, 0);       // (all have read it)
        if (!whole_warp || lane == 0) mbar_arrive_cluster(lead_taken0 + 8u * k);
        ++drawn;
        return t;
    };

    if (warp == 0) {
        if (lane == 0) {
            uint32_t g = 0;
            for (int t; !fail && (t = next_ticket(false)) >= 0;) {
                const VlUnit w = vl_unit<BWD>(t, p, list);
                const int in_buffer = w.piece % list.buffers * buffer_rows, v0 = w.piece * list.tiles * VL_TILE;
                if (w.q) {     // the piece has to be there
                    const int least = 2 * VL_EPI_WARPS * (BWD ? list.active : w.tiles);
                    if (!vl_wait_count(p.written + w.piece * p.pitch + w.slot, least, abort_flag, [] {})) { fail = 10; break; }
                }
                const int am = (w.q && BWD ? w.slot : w.mt) * VL_TILE + (int)rank * 128, bn = w.nt * VL_TILE + (int)rank * 128;
                for (int it = 0; it < w.steps; ++it, ++g) {
                    const int s = (int)(g % STAGES);
                    if (!mbar_wait_cluster(bar_empty(s), ((g / STAGES) & 1u) ^ 1u, abort_flag)) { fail = 1; break; }
                    const uint32_t landed = rank == 0 ? bar_full(s) : bar_landed(s);
                    const uint32_t sa = base + (uint32_t)s * L::STAGE_BYTES, sb = sa + L::A_BYTES;
                    mbar_arrive_expect_tx(landed, L::STAGE_BYTES);
                    if (!w.q) {
                        tma_load_2d(sa, &maps.rows, it * VL_BK, am, landed);
                        tma_load_2d(sb, &maps.words, it * VL_BK, v0 + bn, landed);
                    } else if (!BWD) {       // rows as M, words as steps; features as N
                        tma_load_2d(sa, &maps.piece_in, 0, in_buffer + it * rows_dev + am, landed);
                        tma_load_2d(sb, &maps.other, bn, v0 + it * VL_BK, landed);
                        tma_load_2d(sb + 8192, &maps.other, bn + 64, v0 + it * VL_BK, landed);
                    } else {                 // words as M, rows as steps; features as N
                        tma_load_2d(sa, &maps.piece_in, 0, in_buffer + (am >> 6) * rows_dev + it * VL_BK, landed);
                        tma_load_2d(sa + 8192, &maps.piece_in, 0, in_buffer + ((am >> 6) + 1) * rows_dev + it * VL_BK, landed);
                        tma_load_2d(sb, &maps.other, bn, it * VL_BK, landed);
                        tma_load_2d(sb + 8192, &maps.other, bn + 64, it * VL_BK, landed);
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            const uint32_t idesc_p = vl_idesc(VL_TILE, false, false, p.bf16), idesc_q = vl_idesc(VL_TILE, BWD, true, p.bf16);
            const uint32_t base4 = (base & 0x3FFFFu) >> 4;
            uint32_t g = 0, n = 0;
            for (int t; !fail && (t = next_ticket(false)) >= 0;) {
                const VlUnit w = vl_unit<BWD>(t, p, list);
                for (int at = 0; at < w.steps && !fail; at += w.chain, ++n) {
                    const int b = (int)(n & 1u), end = min(at + w.chain, w.steps);
                    if (!mbar_wait_cluster(bar_drained(b), ((n >> 1) & 1u) ^ 1u, abort_flag)) { fail = 6; break; }
                    tc_fence_after_sync();
                    for (int it = at; it < end; ++it, ++g) {
                        const int s = (int)(g % STAGES);
                        if (!mbar_wait_cluster(bar_full(s), (g / STAGES) & 1u, abort_flag)) { fail = 3; break; }
                        tc_fence_after_sync();
                        const uint32_t a4 = base4 + (uint32_t)s * (L::STAGE_BYTES >> 4), b4 = a4 + (L::A_BYTES >> 4);
                        if (w.q) vl_mma_step(tmem + b * VL_TILE, a4, b4, BWD, true, idesc_q, it == at);
                        else     vl_mma_step(tmem + b * VL_TILE, a4, b4, false, false, idesc_p, it == at);
                        umma_commit_pair(bar_empty(s), (uint16_t)3);
                    }
                    if (!fail) umma_commit_pair(bar_done(b), (uint16_t)3);
                }
            }
        } else if (lane == 0) {
            const uint32_t lead_full0 = mapa_shared(bar_full(0), 0u);
            uint32_t g = 0;
            for (int t; !fail && (t = next_ticket(false)) >= 0;) {
                const VlUnit w = vl_unit<BWD>(t, p, list);
                for (int it = 0; it < w.steps; ++it, ++g) {
                    const int s = (int)(g % STAGES);
                    if (!mbar_wait(bar_landed(s), (g / STAGES) & 1u, abort_flag)) { fail = 8; break; }
                    mbar_arrive_cluster(lead_full0 + 8u * s);
                }
            }
        }
    } else if (warp == VL_EPI_WARPS + 2) {
        // ------------------------------------------------------------------ draws the pair's tickets
        if (lane == 0 && rank == 0) {
            const uint32_t tickets0[2] = {mapa_shared(tickets, 0u), mapa_shared(tickets, 1u)};
            const uint32_t drawn0[2] = {mapa_shared(bar_drawn(0), 0u), mapa_shared(bar_drawn(0), 1u)};
            for (uint32_t n = 0;; ++n) {
                const int k = (int)(n % VL_TICKETS);
                if (!mbar_wait_cluster(bar_taken(k), ((n / VL_TICKETS) & 1u) ^ 1u, abort_flag)) { fail = 11; break; }
                int t = atomicAdd(p.ticket, 1);
                if (t >= list.total) t = -1;
                for (int c = 0; c < 2; ++c) vl_send(tickets0[c] + 4u * k, t, drawn0[c] + 8u * k);
                if (t < 0) break;
            }
        } else if (lane == 0) {
            // ---------------------------------------------------------- the peer: counts the units that have read a piece
            // (A fence and a count take 2700 cycles: in an epilogue warp a third of its time for a tile of few rows' dW.)
            const uint32_t lead_drained = mapa_shared(bar_drained(0), 0u);
            uint32_t n = 0;
            for (int t; !fail && (t = next_ticket(false)) >= 0;) {
                const VlUnit w = vl_unit<BWD>(t, p, list);
                for (int it = 0; it < w.steps; it += w.chain, ++n) {
                    if (!mbar_wait(bar_done(n & 1u), (n >> 1) & 1u, abort_flag)) { fail = 5; break; }
                    mbar_arrive_cluster(lead_drained + 8u * (n & 1u));
                }
                if (!fail && w.q && w.steps > 0) vl_count(p.read + w.piece * p.pitch + w.slot);
            }
        }
    } else {
        // ------------------------------------------------------------------ epilogue: a row's half tile per thread
        const int q = warp & 3, half = (warp - 2) >> 2;
        const uint32_t lead_drained = mapa_shared(bar_drained(0), 0u);
        const uint32_t staging = base + L::STAGING_OFF + (uint32_t)(warp - 2) * 4096u;
        // The box's memory is free again once the store before has read it; what is in it goes out as 32 whole lines.
        auto box_begin = [&]() {
            if (lane == 0) bulk_wait_read();
            __syncwarp();
        };
        auto box_put = [&](int chunk, uint32_t x, uint32_t y, uint32_t z, uint32_t t) {    // 16 bytes of this lane's row
            vl_sts128(staging + lane * 128 + ((chunk ^ (lane & 7)) << 4), x, y, z, t);
        };
        auto box_end = [&](const CUtensorMap* map, int x, int y, bool add) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (add) tma_reduce_add_2d(map, staging, x, y);
                else     tma_store_2d(map, staging, x, y);
                bulk_commit();
            }
        };
        // 32 values in 16 bits: half a box
        auto put16 = [&](const float (&v)[32], int c) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                box_put((c & 32) / 8 + i, vl_pack(v[8 * i], v[8 * i + 1], p.bf16), vl_pack(v[8 * i + 2], v[8 * i + 3], p.bf16),
                        vl_pack(v[8 * i + 4], v[8 * i + 5], p.bf16), vl_pack(v[8 * i + 6], v[8 * i + 7], p.bf16));
        };
        // A unit's stores are counted once they are done, which takes a microsecond: not waited for where the next
        // tile is there already, but before anything that could have to wait for what they lead to.
        int* owed = nullptr;       // the counter
        auto settle = [&]() {
            if (lane == 0 && owed != nullptr) {
                bulk_wait();
                vl_count(owed);
            }
            owed = nullptr;
        };
        // Lane 0 waits for a counter, everybody for lane 0.
        auto wait_count = [&](const int* counter, int least) -> bool {
            int ok = 1;
            if (lane == 0) ok = vl_wait_count(counter, least, abort_flag, settle) ? (owed == nullptr ? 3 : 1) : 0;
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (ok & 2) owed = nullptr;
            return ok != 0;
        };
        uint32_t n = 0;
        for (int t; !fail && (t = next_ticket(true)) >= 0;) {
            const VlUnit w = vl_unit<BWD>(t, p, list);
            const int v0 = w.piece * list.tiles * VL_TILE;
            const int row0 = (w.q && BWD ? w.slot : w.mt) * VL_TILE + (int)rank * 128 + q * 32, row = row0 + lane;   // backward's Q: word of the piece
            const int col0 = w.nt * VL_TILE + half * 128;      // word of the piece, feature
            if (BWD && w.q && w.steps <= 0) {
                // no row takes part: the gradient of the head is zero
                if (v0 + row < p.vocab)
                    for (int c = col0; c < col0 + 128 && c < p.hidden; ++c)
                        static_cast<unsigned short*>(p.d_weight)[(long long)(v0 + row) * p.hidden + c] = 0;
                continue;
            }
            if (owed != nullptr && (w.q || !__all_sync(0xffffffffu, mbar_test(bar_done(n & 1u), (n >> 1) & 1u)))) settle();
            float acc[128];
#pragma unroll
            for (int e = 0; e < 128; ++e) acc[e] = 0.f;
            for (int it = w.chain; it < w.steps; it += w.chain, ++n) {       // (logits alone)
                if (!mbar_wait(bar_done(n & 1u), (n >> 1) & 1u, abort_flag)) { fail = 5; break; }
                tc_fence_after_sync();
                vl_add_chain(acc, tmem + ((uint32_t)(q * 32) << 16) + (n & 1u) * VL_TILE + half * 128);
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(lead_drained + 8u * (n & 1u));
            }
            if (fail) break;
            const int b = (int)(n & 1u);
            // what the values meet, asked for before the tile is complete
            int target = -1;
            float lse2 = 0.f, rest = 0.f, ref = 0.f, scale = 1.f;
            float4 coef = make_float4(0.f, 0.f, 0.f, 0.f);
            const bool live = row < rows;
            if (!w.q && live) {
                target = p.target[row] - v0 - col0;     // column of this thread's share
                if (BWD) {
                    lse2 = p.lse2[row];
                    rest = p.rest[row];
                    coef = p.coef[row];
                } else {
                    ref = p.refs[row];
                }
            }
            // backward's Q: the last four rows whose target is this thread's word. (Where there are many, what they lose
            // averages out.)
            int hits[4] = {-1, -1, -1, -1};
            if (BWD && w.q) {
                scale = *p.weight_scale;
                const int key = (v0 + row) % (int)p.rows_pad, links = p.links[key], first = p.first[key];
                if (v0 + row < p.vocab && links <= VL_LINKS)
                    for (int r = first; r >= 0; r = p.next[r]) {
                        if (p.target[r] != v0 + row) continue;
                        int x = r;
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (x > hits[k]) {
                                const int y = hits[k];
                                hits[k] = x;
                                x = y;
                            }
                    }
                __syncwarp();
            }
            const bool any_hit = BWD && w.q && __any_sync(0xffffffffu, hits[0] >= 0);
            // what is about to be overwritten has been read; what is about to be added to has the pieces before
            if (!w.q && w.piece >= list.buffers &&
                !wait_count(p.read + (w.piece - list.buffers) * p.pitch + w.slot, list.feature_tiles)) { fail = 12; break; }
            const int plane = w.piece % list.planes;
            int* const added = p.added + (plane * list.row_tiles + w.mt) * list.feature_tiles + w.nt;
            if (!BWD && w.q && !wait_count(added, 2 * VL_EPI_WARPS * (w.piece / list.planes))) { fail = 13; break; }
            if (!mbar_wait(bar_done(b), (n >> 1) & 1u, abort_flag)) { fail = 5; break; }
            tc_fence_after_sync();
            const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + b * VL_TILE + half * 128;
            float m2 = VL_NEG, sum = 0.f;
            const int piece_row = w.piece % list.buffers * buffer_rows + row0;
            auto load = [&](int c, uint32_t (&r)[32]) {        // the last chunk's makes room for the unit after the next
                tmem_ld_32x32(at + c, r);
                tmem_ld_wait();
                if (c == 96) {
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(lead_drained + 8u * b);
                }
            };
            if (!w.q) {
#pragma unroll
                for (int c = 0; c < 128; c += 32) {
                    uint32_t r[32];
                    load(c, r);
#pragma unroll
                    for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) + acc[c + e]);
                    const int words = p.vocab - v0 - col0 - c;       // words there are in this chunk
                    float v[32];
                    if (!BWD) {
                        vl_leave_out(r, words, target - c);
                        m2 = fmaxf(m2, vl_top(r) * VL_LOG2E);
                        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            v[e] = live ? vl_ex2(fmaf(__uint_as_float(r[e]), VL_LOG2E, -ref)) : 0.f;
                            part[e & 3] += v[e];
                        }
                        sum += (part[0] + part[1]) + (part[2] + part[3]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = vl_ex2(fmaf(__uint_as_float(r[e]), VL_LOG2E, -lse2)) * coef.x;
                        if (__any_sync(0xffffffffu, words < 32 || (unsigned)(target - c) < 32u || !live)) {
                            const float hit = vl_hit(coef.y, coef.z, rest);
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                if (e == target - c) v[e] = hit;
                                if (e >= words || !live) v[e] = 0.f;
                            }
                        }
                    }
                    if ((c & 32) == 0) box_begin();
                    put16(v, c);
                    if ((c & 32) != 0) box_end(&maps.piece_out, 0, piece_row + ((col0 + c) >> 6) * rows_dev, false);
                    if (c == 32 && owed != nullptr) {
                        if (lane == 0) {
                            bulk_wait_but<1>();
                            vl_count(owed);
                        }
                        owed = nullptr;
                    }
                }
            } else {
#pragma unroll 1
                for (int c = 0; c < 128; c += 32) {
                    uint32_t r[32];
                    load(c, r);
                    if (!BWD) {
                        if (col0 + c >= p.hidden) continue;
                        box_begin();
#pragma unroll
                        for (int i = 0; i < 8; ++i) box_put(i, r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
                        box_end(&maps.out, col0 + c, plane * rows_dev + row0, w.piece >= list.planes);
                    } else {
                        if (col0 + (c & 64) >= p.hidden) continue;
                        if ((c & 32) == 0) box_begin();
                        float v[32];
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(r[e]);
                        if (any_hit) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                if (hits[k] < 0) continue;
                                const float lost = p.coef[hits[k]].w;
                                const uint4* h = reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(p.gathered) +
                                                                               (long long)hits[k] * p.hidden + col0 + c);
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    if (col0 + c + 8 * i >= p.hidden) break;
                                    const uint4 x = h[i];
                                    const uint32_t two[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                                    for (int e = 0; e < 4; ++e) {
                                        const float2 y = vl_two(two[e], p.bf16);
                                        v[8 * i + 2 * e] = fmaf(lost, y.x, v[8 * i + 2 * e]);
                                        v[8 * i + 2 * e + 1] = fmaf(lost, y.y, v[8 * i + 2 * e + 1]);
                                    }
                                }
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] *= scale;
                        put16(v, c);
                        if ((c & 32) != 0) box_end(&maps.out, col0 + (c & 64), v0 + row0, false);
                    }
                }
            }
            ++n;
            if (!w.q && !BWD) {
                p.parts[(long long)(v0 / VL_TILE * 2 + 2 * w.nt + half) * p.rows_pad + row] = make_float2(m2, sum);
                // (several threads write the same)
                if (live && m2 > ref + (p.bf16 ? VL_ROOM_BF16 : VL_ROOM_F16)) p.flags[w.mt] = 1;
            }
            if (!w.q || !BWD)       // (backward's Q writes what nobody waits for)
                owed = w.q ? added : p.written + w.piece * p.pitch + w.slot;
        }
        settle();
        if (lane == 0) bulk_wait();
    }

    if (fail) give_up(p.status, 100 + fail);
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem, 512);
    }
}

// ------------------------------------------------------------------------------------- rows that take part
constexpr int VL_GATHER_WARPS = 8;

// Rows that take part among VL_COUNT_ROWS each, and how many come before each such block: where there are so many rows that a
// CTA of the gather would count too long. (8 words x 8 features, every CTA counting all targets before its own, and this way: 16,384 rows
// 41 and 44 us, 32,768 65 and 66, 131,072 254 and 183, 2,097,152 25.0 and 2.8 ms.)
constexpr int VL_COUNT_ROWS = 1024, VL_COUNT_FROM = 32768;

__device__ __forceinline__ bool vl_takes_part(const VocabLossArgs& a, long long t) { return t >= 0 && t < a.vocab; }

__global__ void __launch_bounds__(256)
vl_count_kernel(const VocabLossArgs a) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ int part[8];
    const long long row0 = (long long)blockIdx.x * VL_COUNT_ROWS;
    int n = 0;
#pragma unroll
    for (int k = 0; k < VL_COUNT_ROWS; k += 256) {
        const long long row = row0 + k + threadIdx.x;
        n += row < a.rows && vl_takes_part(a, a.targets[row]) ? 1 : 0;
    }
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = n;
    __syncthreads();
    if (threadIdx.x != 0) return;
    n = 0;
    for (int i = 0; i < 8; ++i) n += part[i];
    a.before[blockIdx.x] = n;
}

// Counts to sums of those before, by one CTA.
__global__ void __launch_bounds__(1024)
vl_before_kernel(const VocabLossArgs a, int blocks) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ int part[32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int start = 0;
    for (int i0 = 0; i0 < blocks; i0 += 1024) {
        const int i = i0 + threadIdx.x, n = i < blocks ? a.before[i] : 0;
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        if (lane == 31) part[warp] = sum;
        __syncthreads();
        int all = part[lane];        // every warp adds up the warps
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, all, o);
            if (lane >= o) all += x;
        }
        const int warps_before = __shfl_sync(0xffffffffu, all, (warp + 31) & 31);
        if (i < blocks) a.before[i] = start + (warp > 0 ? warps_before : 0) + sum - n;
        start += __shfl_sync(0xffffffffu, all, 31);
        __syncthreads();
    }
}

// A CTA takes `per` rows of the caller's. Where they go follows from the targets before them, which it counts itself, from the
// beginning of its block where there are sums for blocks.
__global__ void __launch_bounds__(VL_GATHER_WARPS * 32)
vl_gather_kernel(const VocabLossArgs a, int per) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ int before[VL_GATHER_WARPS];
    __shared__ int place[32];
    __shared__ float dots[VL_GATHER_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long row0 = (long long)blockIdx.x * per;
    const long long block = a.before != nullptr ? row0 / VL_COUNT_ROWS : 0;
    int n = 0;
    for (long long i = block * VL_COUNT_ROWS + threadIdx.x; i < row0; i += VL_GATHER_WARPS * 32) n += vl_takes_part(a, a.targets[i]) ? 1 : 0;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) before[warp] = n;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < a.n_counters; i += (long long)gridDim.x * blockDim.x)
        a.counters[i] = 0;
    if (a.grads & 2)
        for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < a.rows_pad; i += (long long)gridDim.x * blockDim.x) {
            a.links[i] = 0;
            a.first[i] = -1;
        }
    __syncthreads();
    if (warp == 0) {
        int start = a.before != nullptr ? a.before[block] : 0;
        for (int i = 0; i < VL_GATHER_WARPS; ++i) start += before[i];
        const long long row = row0 + lane;
        const bool in = lane < per && row < a.rows;
        const long long t = in ? a.targets[row] : -1;
        const bool part = in && vl_takes_part(a, t);
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
        if (lane == 0 && row0 + per >= a.rows) *a.count = start + __popc(mask);      // (the last CTA)
    }
    __syncthreads();
    const int vecs = (int)(a.hidden / 8);
    // a row to a warp, or to several where there are few rows
    const int shares = per < VL_GATHER_WARPS ? VL_GATHER_WARPS / per : 1, share = warp % shares;
    for (int i = warp / shares; i < per; i += VL_GATHER_WARPS / shares) {
        const int at = place[i];
        if (at < 0) continue;
        const long long row = row0 + i;
        const uint4* h = reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(a.x) + row * a.ld_x);
        const uint4* w = reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(a.weight) + (long long)a.targets[row] * a.ld_w);
        uint4* out = reinterpret_cast<uint4*>(static_cast<unsigned short*>(a.gathered) + (long long)at * a.hidden);
        float dot = 0.f;
#pragma unroll 4
        for (int c = share * 32 + lane; c < vecs; c += shares * 32) {
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
        if (lane == 0) {
            if (shares > 1) dots[warp] = dot;
            else            a.target_logit[at] = dot;
        }
    }
    if (shares == 1) return;
    __syncthreads();
    if (threadIdx.x < per && place[threadIdx.x] >= 0) {
        float dot = 0.f;
        for (int k = 0; k < shares; ++k) dot += dots[threadIdx.x * shares + k];
        a.target_logit[place[threadIdx.x]] = dot;
    }
}

// Joins a row's statistics, 8 rows by 128 shares of the parts per CTA. (32 by 32: 8.5 us for 64 rows of 151,936 words, so 5.0.)
// Where the head's gradient is to come, the last tile's empty rows become zeros: they meet the others' in sums over rows,
// and nowhere else does what lies there reach a result. PROBE: the first words' maxima give the row's
// reference. Otherwise the whole vocabulary's give loss and lse; `soft`: the sums are relative to the row's reference.
constexpr int VL_MERGE_ROWS = 8, VL_MERGE_SHARES = 1024 / VL_MERGE_ROWS;

template <bool PROBE>
__global__ void __launch_bounds__(1024)
vl_merge_kernel(const VocabLossArgs a, int n_parts, int soft) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ float2 join[VL_MERGE_ROWS][VL_MERGE_SHARES + 1];
    const int rows = *a.count, row = blockIdx.x * VL_MERGE_ROWS + threadIdx.x;
    if (!PROBE && (a.grads & 2)) {
        const long long vecs = a.hidden / 8, end = (long long)vl_div_up(rows, VL_TILE) * VL_TILE * vecs;
        uint4* out = reinterpret_cast<uint4*>(a.gathered);
        for (long long i = rows * vecs + blockIdx.x * 1024 + threadIdx.y * VL_MERGE_ROWS + threadIdx.x; i < end; i += gridDim.x * 1024)
            out[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    const int thread = threadIdx.y * VL_MERGE_ROWS + threadIdx.x, warp = thread >> 5, lane = thread & 31;
    if (blockIdx.x * VL_MERGE_ROWS >= rows) return;
    float m = VL_NEG, s = 0.f;
    if (row < rows) {
        const float ref = soft ? a.refs[row] : 0.f;
#pragma unroll 4
        for (int i = threadIdx.y; i < n_parts; i += VL_MERGE_SHARES) {
            float2 x = a.parts[(long long)i * a.rows_pad + row];
            if (soft) x.x = ref;
            x = vl_join(make_float2(m, s), x);
            m = x.x;
            s = x.y;
        }
    }
    join[threadIdx.x][threadIdx.y] = make_float2(m, s);
    __syncthreads();
    // a warp joins one row's shares
    if (warp >= VL_MERGE_ROWS) return;
    float2 x = join[warp][lane];
#pragma unroll
    for (int i = 32; i < VL_MERGE_SHARES; i += 32) x = vl_join(x, join[warp][lane + i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        x = vl_join(x, make_float2(__shfl_xor_sync(0xffffffffu, x.x, o), __shfl_xor_sync(0xffffffffu, x.y, o)));
    }
    const int at = blockIdx.x * VL_MERGE_ROWS + warp;
    if (lane != 0 || at >= rows) return;
    const float logit = a.target_logit[at], logit2 = logit * VL_LOG2E;
    if (PROBE) {
        // (fmaxf leaves out a NaN; where there is nothing finite to go by, any number will do)
        float ref = x.x - VL_BELOW;
        if (a.bf16 || x.x <= 0.5f * VL_NEG) ref = fmaxf(ref, logit2 - VL_BELOW_TARGET_BF16);
        a.refs[at] = fabsf(ref) < 1.0e29f ? floorf(ref) : 0.f;
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
    if (a.grads & 2) {        // (their order is of no account: who reads them sorts)
        const int key = a.target[at] % (int)a.rows_pad;
        a.next[at] = atomicExch(a.first + key, at);
        atomicAdd(a.links + key, 1);
    }
    a.losses[a.source[at]] = loss;
    a.lse[a.source[at]] = logit + loss;
}

// A CTA per row tile: where a row outgrew its reference, the tile goes onto the list (in any order), with new references from
// the maxima.
__global__ void __launch_bounds__(VL_TILE)
vl_again_kernel(const VocabLossArgs a, int word_tiles) {
    grid_dep_wait();
    grid_dep_launch();
    if (a.flags[blockIdx.x] == 0) return;
    if (threadIdx.x == 0) a.list[1 + atomicAdd(a.list, 1)] = blockIdx.x;
    const int rows = *a.count, row = blockIdx.x * VL_TILE + threadIdx.x;
    if (row >= rows) return;
    float top = VL_NEG;
#pragma unroll 8
    for (int i = 0; i < 2 * word_tiles; ++i) top = fmaxf(top, a.parts[(long long)i * a.rows_pad + row].x);
    if (top > a.refs[row] + (a.bf16 ? VL_ROOM_BF16 : VL_ROOM_F16)) a.refs[row] = ceilf(top) - 6.f;
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

// One CTA: per row that takes part (b + c, b, c) over a common power of two, times VL_P_SCALE, and what the target's dl of that
// size loses in 16 bits. The power is the one above the largest |b| (1 - p_t) and |c|: no dl is more than twice that, and the
// largest are near it however certain the rows are. (Above the largest |b|, rows 22 nats above their other words alone left dW's rows
// of those a percent off in fp16.) A row far below the largest keeps its digits down to 2^-27 of it, and adds nothing that the others'
// rounding would not cover below. VL_B_MOST keeps b over the power finite.
constexpr float VL_B_MOST = 5.421010862427522e-20f;      // 2^-64
__global__ void __launch_bounds__(1024)
vl_coef_kernel(const VocabLossArgs a) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ float part[32];
    float top = 0.f;
    const int rows = *a.count;
    for (long long i = threadIdx.x; i < a.n_counters; i += 1024) a.counters[i] = 0;
    for (int at = threadIdx.x; at < rows; at += 1024) {
        const long long row = a.source[at];
        const float b = fabsf(vl_upstream(a.d_losses, a.d_losses_stride, row)), c = fabsf(vl_upstream(a.d_lse, a.d_lse_stride, row));
        top = fmaxf(top, fmaxf(b * fmaxf(a.rest[at], VL_B_MOST), c));
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
        const float rest = a.rest[at], hit = vl_hit(b * inv, c * inv, rest);
        const float there = a.bf16 ? __bfloat162float(__float2bfloat16_rn(hit)) : __half2float(__float2half_rn(hit));
        a.coef[at] = make_float4((b + c) * inv, b * inv, c * inv, hit - there);
    }
    if (threadIdx.x == 0) *a.weight_scale = power / VL_P_SCALE;
}

// dH of the caller's rows; zeros where the row took no part.
__global__ void __launch_bounds__(256)
vl_hidden_kernel(const VocabLossArgs a) {
    grid_dep_wait();
    grid_dep_launch();
    const int vecs = (int)(a.hidden / 8), row_tiles = vl_div_up(*a.count, VL_TILE);
    const int planes = min(vl_planes(a.rows_pad, row_tiles),
                           vl_shape(row_tiles, vl_div_up((int)a.vocab, VL_TILE), vl_div_up((int)a.hidden, VL_TILE), false).pieces);
    const long long plane = (long long)row_tiles * VL_TILE * a.hidden / 4;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < a.rows * vecs; i += (long long)gridDim.x * 256) {
        const long long row = i / vecs;
        const int c = (int)(i - row * vecs), at = a.place[row];
        uint4 out = make_uint4(0u, 0u, 0u, 0u);
        if (at >= 0) {
            const float b = vl_upstream(a.d_losses, a.d_losses_stride, row), z = vl_upstream(a.d_lse, a.d_lse_stride, row);
            const float rest = a.rest[at], mean = (b + z) * a.norm[at], hit = vl_hit(b, z, rest);
            const float4* u = reinterpret_cast<const float4*>(a.sums + (long long)at * a.hidden) + 2 * c;
            float4 x = u[0], y = u[1];
            for (int k = 1; k < planes; ++k) {
                const float4 v = u[k * plane], w = u[k * plane + 1];
                x = make_float4(x.x + v.x, x.y + v.y, x.z + v.z, x.w + v.w);
                y = make_float4(y.x + w.x, y.y + w.y, y.z + w.z, y.w + w.w);
            }
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

// Tiles of 256 x 256 that the pieces' buffers need, and the most pieces, for any number of rows up to `rows`.
struct VlRoom {
    long long units;
    int pieces;
};
static VlRoom vl_room(long long rows, long long vocab, long long hidden, bool backward) {
    const int row_tiles = (int)(vl_rows_pad(rows) / VL_TILE), word_tiles = vl_word_tiles(vocab);
    VlRoom r = {0, 1};
    for (int a = 1; a <= row_tiles; ++a) {
        const VlShape s = vl_shape(a, word_tiles, vl_div_up((int)hidden, VL_TILE), backward);
        const long long units = (long long)s.buffers * s.tiles * a;
        if (units > r.units) r.units = units;
        if (s.pieces > r.pieces) r.pieces = s.pieces;
    }
    return r;
}

// What the forward keeps for the backward.
struct VlKept {
    size_t count, place, source, target, lse, rest, norm, links, first, next, sums, gathered, bytes;
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
    k.norm = take(pad * 4);
    if (grads & 2) {
        k.links = take(pad * 4);
        k.first = take(pad * 4);
        k.next = take(pad * 4);
    }
    if (grads & 1) k.sums = take((size_t)vl_plane_rows((long long)pad) * (size_t)hidden * 4);
    k.gathered = at;                       // last: without a gradient of the weight it is scratch of the forward
    if (grads & 2) take(pad * (size_t)hidden * 2);
    k.bytes = at;
    return k;
}

// Counters of a sweep, and of the forward's two.
struct VlCounters {
    long long ticket, written, read, added, each, flags, list, total;
    int pitch;
};
static VlCounters vl_counters(const VocabLossArgs& a, const VlRoom& room, bool backward) {
    VlCounters c = {};
    const long long row_tiles = vl_rows_pad(a.rows) / VL_TILE, feature_tiles = vl_div_up((int)a.hidden, VL_TILE);
    c.pitch = backward ? VL_BWD_TILES : (int)row_tiles;
    c.ticket = 0;
    c.written = 32;
    c.read = c.written + (long long)room.pieces * c.pitch;
    c.added = c.read + (long long)room.pieces * c.pitch;
    c.each = c.added + (backward ? 0 : vl_plane_rows(vl_rows_pad(a.rows)) / VL_TILE * feature_tiles);
    c.flags = (backward ? 1 : 2) * c.each;
    c.list = c.flags + (backward ? 0 : row_tiles);
    c.total = c.list + (backward ? 0 : 1 + row_tiles);
    return c;
}

struct VlScratch {
    size_t parts, target_logit, before, refs, counters, gathered, coef, weight_scale, piece, bytes;
    VlRoom room;
};

static VlScratch vl_scratch(const VocabLossArgs& a, bool backward) {
    VlScratch s = {};
    const size_t pad = (size_t)vl_rows_pad(a.rows);
    size_t at = 0;
    const auto take = [&](size_t n) { const size_t r = at; at += vl_align(n); return r; };
    s.room = vl_room(a.rows, a.vocab, a.hidden, backward);
    const size_t piece = (size_t)s.room.units * VL_TILE * VL_TILE * 2;
    const size_t counters = (size_t)vl_counters(a, s.room, backward).total * 4;
    if (!backward) {
        const size_t n_parts = (size_t)vl_word_tiles(a.vocab) * 2, few_parts = (size_t)a.sm_count * 4;
        s.parts = take((n_parts > few_parts ? n_parts : few_parts) * 8 * pad);
        s.target_logit = take(pad * 4);
        s.before = take(a.rows > VL_COUNT_FROM ? pad / VL_COUNT_ROWS * 4 + 4 : 0);
        if (!(a.grads & 2)) s.gathered = take(pad * (size_t)a.hidden * 2);
        if (a.grads & 1) {
            s.refs = take(pad * 4);
            s.counters = take(counters);
            s.piece = take(piece);
        }
    } else if (a.d_weight != nullptr) {
        s.coef = take(pad * 16);
        s.weight_scale = take(4);
        s.counters = take(counters);
        s.piece = take(piece);
    }
    s.bytes = at;
    return s;
}

size_t vocab_loss_kept_bytes(long long rows, long long hidden, int grads) { return vl_kept(rows, hidden, grads).bytes; }

size_t vocab_loss_workspace_bytes(const VocabLossArgs& a, bool backward) { return vl_scratch(a, backward).bytes; }

// CTA pairs: one per pair of SMs as far as there are units.
static long long vl_pairs(long long units, int sm_count) {
    const long long pairs = units < sm_count / 2 ? units : sm_count / 2;
    return pairs < 1 ? 1 : pairs;
}

// A kernel of CTA pairs that takes tensor maps and parameters.
template <typename Maps, typename Params>
static cudaError_t vl_launch(void (*kernel)(Maps, Params), int threads, int smem, const Maps& maps, const Params& p, long long units,
                             int sm_count, cudaStream_t stream) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
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
    cfg.gridDim = dim3((unsigned)(2 * vl_pairs(units, sm_count)));
    return cudaLaunchKernelEx(&cfg, kernel, maps, p);
}

static bool vl_map(CUtensorMap* map, int bf16, const void* base, long long inner, long long outer, long long pitch, int box_outer) {
    return make_map_2d(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, base, (uint64_t)inner,
                       (uint64_t)outer, (uint64_t)pitch * 2, VL_BK, (uint32_t)box_outer, CU_TENSOR_MAP_SWIZZLE_128B);
}

// The 16-bit pieces: blocks of [rows][64 words], read in boxes of 128 rows (rows as M) or 64 (as steps), written in 32.
static bool vl_piece_map(CUtensorMap* map, const VocabLossArgs& a, int box_outer) {
    return vl_map(map, a.bf16, a.piece, VL_BK, a.piece_units * VL_TILE * (VL_TILE / VL_BK), VL_BK, box_outer);
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
    a.norm = reinterpret_cast<float*>(base + k.norm);
    a.links = reinterpret_cast<int*>(base + k.links);
    a.first = reinterpret_cast<int*>(base + k.first);
    a.next = reinterpret_cast<int*>(base + k.next);
    a.sums = reinterpret_cast<float*>(base + k.sums);
    a.gathered = base + k.gathered;
    a.rows_pad = vl_rows_pad(a.rows);
}

static VlSweepParams vl_sweep_params(const VocabLossArgs& a, const VlCounters& c, int sweep) {
    VlSweepParams p = {};
    p.count = a.count; p.status = a.status; p.bf16 = a.bf16;
    p.vocab = (int)a.vocab; p.hidden = (int)a.hidden; p.word_tiles = vl_word_tiles(a.vocab);
    p.rows_pad = a.rows_pad; p.target = a.target; p.piece = a.piece;
    int* counters = a.counters + sweep * c.each;
    p.ticket = counters + c.ticket; p.written = counters + c.written; p.read = counters + c.read; p.added = counters + c.added;
    p.pitch = c.pitch;
    p.parts = a.parts; p.refs = a.refs; p.flags = a.flags; p.list = a.list; p.again = sweep;
    p.lse2 = a.lse_rows; p.rest = a.rest; p.coef = a.coef; p.links = a.links; p.first = a.first; p.next = a.next; p.gathered = a.gathered; p.d_weight = a.d_weight; p.weight_scale = a.weight_scale;
    return p;
}

constexpr int VL_SWEEP_SMEM = VlSmem<128, 6, true>::TOTAL;

cudaError_t launch_vocab_loss_fwd(const VocabLossArgs& a_in, cudaStream_t stream, const char** why) {
    *why = "";
    VocabLossArgs a = a_in;
    if (a.rows <= 0) return cudaSuccess;
    vl_use_kept(a);
    const VlScratch s = vl_scratch(a, false);
    const VlCounters counters = vl_counters(a, s.room, false);
    char* ws = static_cast<char*>(a.workspace);
    a.parts = reinterpret_cast<float2*>(ws + s.parts);
    a.target_logit = reinterpret_cast<float*>(ws + s.target_logit);
    if (!(a.grads & 2)) a.gathered = ws + s.gathered;
    const bool soft = (a.grads & 1) != 0;
    if (soft) {
        a.refs = reinterpret_cast<float*>(ws + s.refs);
        a.counters = reinterpret_cast<int*>(ws + s.counters);
        a.n_counters = counters.total;
        a.flags = a.counters + counters.flags;
        a.list = a.counters + counters.list;
        a.piece = ws + s.piece;
        a.piece_units = s.room.units;
    }
    cudaError_t e = cudaSuccess;
    if (a.rows > VL_COUNT_FROM) {
        a.before = reinterpret_cast<int*>(ws + s.before);
        const int blocks = (int)((a.rows + VL_COUNT_ROWS - 1) / VL_COUNT_ROWS);
        e = launch_pdl(vl_count_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a);
        if (e == cudaSuccess) e = launch_pdl(vl_before_kernel, dim3(1), dim3(1024), 0, stream, a, blocks);
        if (e != cudaSuccess) { *why = "counts"; return e; }
    }
    const int per = a.rows <= 512 ? 2 : a.rows <= 4096 ? 8 : 32;     // rows of a CTA (64 x 3584: a row to a warp 11.5 us, to four 5.7)
    e = launch_pdl(vl_gather_kernel, dim3((unsigned)((a.rows + per - 1) / per)), dim3(VL_GATHER_WARPS * 32), 0, stream, a, per);
    if (e != cudaSuccess) { *why = "gather"; return e; }
    // Up to 64 rows without a gradient of x: the words take the tensor cores' long side. (64 rows of 3584 features against
    // 151,936 words: with the rows there, which costs four times the products, 216 us; this way all three kernels take 176, the
    // weight's 1.09 GB alone 168.) Every CTA has as many words, in tiles of one size (9 of 115 here): as shares of tiles of
    // 128, of which there are 8.03 to a CTA, 197 us, as eight of them and a rest in boxes of 16 words 187.
    const bool few = !soft && a.rows <= 64;
    const int few_rows = a.rows <= 32 ? 32 : 64;
    VlMaps logits = {};
    VlSweepMaps maps = {};
    const long long few_ctas = 2 * vl_pairs(vl_word_tiles(a.vocab), a.sm_count);
    const int cta_tiles = vl_div_up((int)a.vocab, (int)few_ctas * 128), tile_words = vl_div_up((int)a.vocab, (int)few_ctas * cta_tiles);
    bool ok = few ? vl_map(&logits.a, a.bf16, a.weight, a.hidden, a.vocab, a.ld_w, tile_words) &&
                        vl_map(&logits.b, a.bf16, a.gathered, a.hidden, a.rows_pad, a.hidden, few_rows / 2)
                  : vl_map(&logits.a, a.bf16, a.gathered, a.hidden, a.rows_pad, a.hidden, 128) &&
                        vl_map(&logits.b, a.bf16, a.weight, a.hidden, a.vocab, a.ld_w, 128);
    if (ok && soft) {
        maps.rows = logits.a;
        maps.words = logits.b;
        ok = vl_piece_map(&maps.piece_in, a, 128) && vl_map(&maps.other, a.bf16, a.weight, a.hidden, a.vocab, a.ld_w, 64) &&
             vl_piece_map(&maps.piece_out, a, 32) &&
             make_map_2d(&maps.out, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, a.sums, (uint64_t)a.hidden, (uint64_t)vl_plane_rows(a.rows_pad),
                         (uint64_t)a.hidden * 4, 32, 32, CU_TENSOR_MAP_SWIZZLE_128B);
    }
    if (!ok) { *why = "cuTensorMapEncodeTiled"; return cudaErrorInvalidValue; }
    VlParams p = {};
    p.count = a.count; p.status = a.status; p.bf16 = a.bf16;
    p.vocab = (int)a.vocab; p.hidden = (int)a.hidden; p.word_tiles = vl_word_tiles(a.vocab); p.n_rows = few_rows;
    p.target = a.target; p.parts = a.parts; p.rows_pad = a.rows_pad;
    const long long row_tiles = a.rows_pad / VL_TILE;
    const dim3 merge_grid((unsigned)((a.rows + VL_MERGE_ROWS - 1) / VL_MERGE_ROWS)), merge_block(VL_MERGE_ROWS, VL_MERGE_SHARES);
    int n_parts = 2 * p.word_tiles;
    if (few) {
        p.cta_tiles = cta_tiles;
        p.tile_words = tile_words;
        e = vl_launch(vl_stats_kernel<VL_FEW>, VL_THREADS, VlSmemOf<VL_FEW>::TOTAL, logits, p, p.word_tiles, a.sm_count, stream);
        n_parts = (int)(4 * few_ctas);
    } else if (!soft) {
        e = vl_launch(vl_stats_kernel<VL_STATS>, VL_THREADS, VlSmemOf<VL_STATS>::TOTAL, logits, p, row_tiles * p.word_tiles, a.sm_count, stream);
    } else {
        VlParams probe = p;
        if (probe.word_tiles > VL_PROBE_TILES) probe.word_tiles = VL_PROBE_TILES;
        e = vl_launch(vl_stats_kernel<VL_STATS>, VL_THREADS, VlSmemOf<VL_STATS>::TOTAL, logits, probe, row_tiles * probe.word_tiles, a.sm_count, stream);
        if (e == cudaSuccess) e = launch_pdl(vl_merge_kernel<true>, merge_grid, merge_block, 0, stream, a, 2 * probe.word_tiles, 0);
        if (e != cudaSuccess) { *why = "references"; return e; }
        const long long units = row_tiles * (p.word_tiles + vl_div_up(p.hidden, VL_TILE));
        // (no row outgrows a reference that all words were asked for)
        const bool sure = p.word_tiles <= VL_PROBE_TILES;
        for (int sweep = 0; sweep < (sure ? 1 : 2) && e == cudaSuccess; ++sweep) {
            e = vl_launch(vl_sweep_kernel<false>, VL_SWEEP_THREADS, VL_SWEEP_SMEM, maps, vl_sweep_params(a, counters, sweep), units, a.sm_count, stream);
            if (!sure && sweep == 0 && e == cudaSuccess)
                e = launch_pdl(vl_again_kernel, dim3((unsigned)row_tiles), dim3(VL_TILE), 0, stream, a, p.word_tiles);
        }
    }
    if (e != cudaSuccess) { *why = "statistics"; return e; }
    e = launch_pdl(vl_merge_kernel<false>, merge_grid, merge_block, 0, stream, a, n_parts, soft ? 1 : 0);
    if (e != cudaSuccess) *why = "merge";
    return e;
}

cudaError_t launch_vocab_loss_bwd(const VocabLossArgs& a_in, cudaStream_t stream, const char** why) {
    *why = "";
    VocabLossArgs a = a_in;
    if (a.rows <= 0) return cudaSuccess;
    vl_use_kept(a);
    const VlScratch s = vl_scratch(a, true);
    const VlCounters counters = vl_counters(a, s.room, true);
    char* ws = static_cast<char*>(a.workspace);
    cudaError_t e = cudaSuccess;
    if (a.d_x != nullptr) {
        e = launch_pdl(vl_hidden_kernel, dim3((unsigned)(a.sm_count * 8)), dim3(256), 0, stream, a);
        if (e != cudaSuccess) { *why = "gradient of the hidden states"; return e; }
    }
    if (a.d_weight == nullptr) return e;
    a.coef = reinterpret_cast<float4*>(ws + s.coef);
    a.weight_scale = reinterpret_cast<float*>(ws + s.weight_scale);
    a.counters = reinterpret_cast<int*>(ws + s.counters);
    a.n_counters = counters.total;
    a.piece = ws + s.piece;
    a.piece_units = s.room.units;
    e = launch_pdl(vl_coef_kernel, dim3(1), dim3(1024), 0, stream, a);
    if (e != cudaSuccess) { *why = "row factors"; return e; }
    VlSweepMaps maps = {};
    if (!vl_map(&maps.rows, a.bf16, a.gathered, a.hidden, a.rows_pad, a.hidden, 128) ||
        !vl_map(&maps.words, a.bf16, a.weight, a.hidden, a.vocab, a.ld_w, 128) ||
        !vl_piece_map(&maps.piece_in, a, 64) || !vl_map(&maps.other, a.bf16, a.gathered, a.hidden, a.rows_pad, a.hidden, 64) ||
        !vl_piece_map(&maps.piece_out, a, 32) || !vl_map(&maps.out, a.bf16, a.d_weight, a.hidden, a.vocab, a.hidden, 32)) {
        *why = "cuTensorMapEncodeTiled";
        return cudaErrorInvalidValue;
    }
    const long long units = (long long)vl_word_tiles(a.vocab) * (a.rows_pad / VL_TILE + vl_div_up((int)a.hidden, VL_TILE));
    e = vl_launch(vl_sweep_kernel<true>, VL_SWEEP_THREADS, VL_SWEEP_SMEM, maps, vl_sweep_params(a, counters, 0), units, a.sm_count, stream);
    if (e != cudaSuccess) *why = "gradient of the head";
    return e;
}

}  // namespace nf4
