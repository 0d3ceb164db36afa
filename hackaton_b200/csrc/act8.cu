// Activations kept in 8 bits for the backward pass (the form: act8.cuh), and what reads them there:
//   quantize / dequantize   the values of a tensor to codes and steps, and back
//   SwiGLU                  hidden = gate * sigmoid(gate) * up with gate and up kept in the same pass; the
//                           backward from the codes (the arithmetic of swiglu.cuh)
//   LoRA gradient           dA[r, k] = sum_m s[m, r] * x[m, k] from the codes of x
// All are bound by memory: per value quantize 3.03 bytes, dequantize 3.03, SwiGLU forward 8.06, backward 8.06,
// the gradient 1.03 and a share of s.
// A thread takes 16 values (32 bytes of fp16 in two 16-byte accesses, one 16-byte access of codes), two
// threads a block of 32, whose largest magnitude is one shuffle away. Rows that are not whole blocks or not 16-byte
// aligned go a warp per block, a lane per value, several times as long: 16,384 x 3592 quantise 161 us, read back 149 (3584: 28 and 30);
// SwiGLU both ways 4096 x 8968 300 us (8960: 101). The gradient takes 29 us at 3592 or 3616 (22 at 3584), where a row's step bytes are
// no whole words.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "act8.cuh"
#include "kernels.h"
#include "ptx.cuh"
#include "swiglu.cuh"

namespace nf4 {

constexpr int A8_THREADS = 256;

// 16 values as they lie in memory.
template <typename T>
struct A8Raw {
    uint4 q[sizeof(T)];   // 2 or 4 pieces of 16 bytes
    static constexpr int N = (int)sizeof(T);
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < N; ++i) q[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ void load(const void* p, long long i) {
        const uint4* s = static_cast<const uint4*>(p) + i * N;
#pragma unroll
        for (int j = 0; j < N; ++j) q[j] = __ldcs(s + j);
    }
    __device__ __forceinline__ void values(float (&v)[16]) const {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t w[4] = {q[j].x, q[j].y, q[j].z, q[j].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (sizeof(T) == 4) {
                    v[4 * j + e] = __uint_as_float(w[e]);
                } else {
                    const float2 f = A8Source<T>::two(w[e]);
                    v[8 * j + 2 * e] = f.x;
                    v[8 * j + 2 * e + 1] = f.y;
                }
            }
        }
    }
};

template <typename T>
__device__ __forceinline__ void a8_store16(void* p, long long i, const float (&v)[16]) {
    uint4* d = static_cast<uint4*>(p) + i * (int)sizeof(T);
#pragma unroll
    for (int j = 0; j < (int)sizeof(T); ++j) {
        if constexpr (sizeof(T) == 4)
            d[j] = make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]),
                              __float_as_uint(v[4 * j + 3]));
        else
            d[j] = make_uint4(A8Source<T>::pack(v[8 * j], v[8 * j + 1]), A8Source<T>::pack(v[8 * j + 2], v[8 * j + 3]),
                              A8Source<T>::pack(v[8 * j + 4], v[8 * j + 5]), A8Source<T>::pack(v[8 * j + 6], v[8 * j + 7]));
    }
}

// Codes of this thread's half block; both halves' threads take part.
__device__ __forceinline__ uint4 a8_encode16(const float (&v)[16], uint32_t& step) {
    uint32_t top = 0u;
#pragma unroll
    for (int e = 0; e < 16; ++e) top = max(top, a8_bits(v[e]));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    step = a8_step(top);
    const float inv = a8_inverse(step);
    return make_uint4(a8_code4(v[0], v[1], v[2], v[3], inv), a8_code4(v[4], v[5], v[6], v[7], inv),
                      a8_code4(v[8], v[9], v[10], v[11], inv), a8_code4(v[12], v[13], v[14], v[15], inv));
}

__device__ __forceinline__ void a8_decode16(const uint4& q, uint32_t step, float (&v)[16]) {
    const float s = a8_value_of_step(step);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float f[4];
        a8_values4(w[j], s, f);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * j + e] = f[e];
    }
}

// The largest of a warp's magnitudes, in every lane.
__device__ __forceinline__ uint32_t a8_warp_top(float x) { return __reduce_max_sync(0xffffffffu, a8_bits(x)); }

__device__ __forceinline__ float a8_decode1(const int8_t* codes, const uint8_t* steps, long long block, int lane) {
    return (float)codes[block * A8_BLOCK + lane] * a8_value_of_step(steps[block]);
}

// `n16`: half blocks of a flat array of whole blocks.
template <typename T>
__global__ void __launch_bounds__(A8_THREADS)
act8_quantize_kernel(const void* __restrict__ x, uint4* __restrict__ codes, uint8_t* __restrict__ steps, long long n16) {
    grid_dep_wait();
    grid_dep_launch();
    const long long i = (long long)blockIdx.x * A8_THREADS + threadIdx.x;
    const bool here = i < n16;
    A8Raw<T> raw;
    raw.zero();
    if (here) raw.load(x, i);
    float v[16];
    raw.values(v);
    uint32_t step;
    const uint4 q = a8_encode16(v, step);
    if (!here) return;
    codes[i] = q;
    if ((i & 1) == 0) steps[i >> 1] = (uint8_t)step;
}

template <typename T>
__global__ void __launch_bounds__(A8_THREADS)
act8_dequantize_kernel(const uint4* __restrict__ codes, const uint8_t* __restrict__ steps, void* __restrict__ x,
                       long long n16) {
    grid_dep_wait();
    grid_dep_launch();
    const long long i = (long long)blockIdx.x * A8_THREADS + threadIdx.x;
    if (i >= n16) return;
    float v[16];
    a8_decode16(__ldcs(codes + i), steps[i >> 1], v);
    a8_store16<T>(x, i, v);
}

// Any width: a warp per block, a lane per value.
struct A8Rows {
    long long rows, blocks;   // blocks of a row
    int cols;
};

template <typename T>
__global__ void __launch_bounds__(A8_THREADS)
act8_quantize_any_kernel(const void* __restrict__ x, int8_t* __restrict__ codes, uint8_t* __restrict__ steps, const A8Rows g) {
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31;
    const long long total = g.rows * g.blocks, stride = (long long)gridDim.x * (A8_THREADS / 32);
    for (long long b = (long long)blockIdx.x * (A8_THREADS / 32) + (threadIdx.x >> 5); b < total; b += stride) {
        const long long row = b / g.blocks;
        const int col = (int)(b - row * g.blocks) * A8_BLOCK + lane;
        const float v = col < g.cols ? A8Source<T>::load(x, row * g.cols + col) : 0.f;
        const uint32_t step = a8_step(a8_warp_top(v));
        codes[b * A8_BLOCK + lane] = (int8_t)(a8_code(v, a8_inverse(step)) & 255u);
        if (lane == 0) steps[b] = (uint8_t)step;
    }
}

template <typename T>
__global__ void __launch_bounds__(A8_THREADS)
act8_dequantize_any_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ steps, void* __restrict__ x,
                           const A8Rows g) {
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31;
    const long long total = g.rows * g.blocks, stride = (long long)gridDim.x * (A8_THREADS / 32);
    for (long long b = (long long)blockIdx.x * (A8_THREADS / 32) + (threadIdx.x >> 5); b < total; b += stride) {
        const long long row = b / g.blocks;
        const int col = (int)(b - row * g.blocks) * A8_BLOCK + lane;
        if (col < g.cols) A8Source<T>::store(x, row * g.cols + col, a8_decode1(codes, steps, b, lane));
    }
}

// ---------------------------------------------------------------------------------------------- SwiGLU
__global__ void __launch_bounds__(A8_THREADS)
act8_swiglu_fwd_kernel(const Act8Swiglu a, long long n16) {
    grid_dep_wait();
    grid_dep_launch();
    const long long i = (long long)blockIdx.x * A8_THREADS + threadIdx.x;
    const bool here = i < n16;
    A8Raw<__half> rg, ru;
    rg.zero();
    ru.zero();
    if (here) {
        rg.load(a.gate, i);
        ru.load(a.up, i);
    }
    float g[16], u[16];
    rg.values(g);
    ru.values(u);
    uint32_t sg, su;
    const uint4 qg = a8_encode16(g, sg), qu = a8_encode16(u, su);
    if (!here) return;
    reinterpret_cast<uint4*>(a.gate_codes)[i] = qg;
    reinterpret_cast<uint4*>(a.up_codes)[i] = qu;
    if ((i & 1) == 0) {
        a.gate_steps[i >> 1] = (uint8_t)sg;
        a.up_steps[i >> 1] = (uint8_t)su;
    }
    uint4* h = reinterpret_cast<uint4*>(a.hidden) + 2 * i;
#pragma unroll
    for (int j = 0; j < 2; ++j)
        h[j] = make_uint4(swiglu2(rg.q[j].x, ru.q[j].x), swiglu2(rg.q[j].y, ru.q[j].y), swiglu2(rg.q[j].z, ru.q[j].z),
                          swiglu2(rg.q[j].w, ru.q[j].w));
}

__global__ void __launch_bounds__(A8_THREADS)
act8_swiglu_bwd_kernel(const Act8Swiglu a, long long n16) {
    grid_dep_wait();
    grid_dep_launch();
    const long long i = (long long)blockIdx.x * A8_THREADS + threadIdx.x;
    if (i >= n16) return;
    A8Raw<__half> rd;
    rd.load(a.d_hidden, i);
    const uint4 qg = __ldcs(reinterpret_cast<const uint4*>(a.gate_codes) + i);
    const uint4 qu = __ldcs(reinterpret_cast<const uint4*>(a.up_codes) + i);
    float d[16], g[16], u[16];
    a8_decode16(qg, a.gate_steps[i >> 1], g);
    a8_decode16(qu, a.up_steps[i >> 1], u);
    rd.values(d);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        float dg, du;
        swiglu_bwd1(d[e], g[e], u[e], dg, du);
        g[e] = dg;
        u[e] = du;
    }
    a8_store16<__half>(a.d_gate, i, g);
    a8_store16<__half>(a.d_up, i, u);
}

__global__ void __launch_bounds__(A8_THREADS)
act8_swiglu_any_kernel(const Act8Swiglu a, const A8Rows g, int backward) {
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31;
    const long long total = g.rows * g.blocks, stride = (long long)gridDim.x * (A8_THREADS / 32);
    for (long long b = (long long)blockIdx.x * (A8_THREADS / 32) + (threadIdx.x >> 5); b < total; b += stride) {
        const long long row = b / g.blocks;
        const int col = (int)(b - row * g.blocks) * A8_BLOCK + lane;
        const long long at = row * g.cols + col;
        const bool in = col < g.cols;
        if (!backward) {
            const float x = in ? __half2float(a.gate[at]) : 0.f, u = in ? __half2float(a.up[at]) : 0.f;
            const uint32_t sg = a8_step(a8_warp_top(x)), su = a8_step(a8_warp_top(u));
            a.gate_codes[b * A8_BLOCK + lane] = (int8_t)(a8_code(x, a8_inverse(sg)) & 255u);
            a.up_codes[b * A8_BLOCK + lane] = (int8_t)(a8_code(u, a8_inverse(su)) & 255u);
            if (lane == 0) {
                a.gate_steps[b] = (uint8_t)sg;
                a.up_steps[b] = (uint8_t)su;
            }
            if (in) a.hidden[at] = __float2half_rn(x * sigmoid_fast(x) * u);
        } else if (in) {
            float dg, du;
            swiglu_bwd1(__half2float(a.d_hidden[at]), a8_decode1(a.gate_codes, a.gate_steps, b, lane),
                        a8_decode1(a.up_codes, a.up_steps, b, lane), dg, du);
            a.d_gate[at] = __float2half_rn(dg);
            a.d_up[at] = __float2half_rn(du);
        }
    }
}

// ---------------------------------------------------------------------------------------- LoRA gradient
// out[r, k] = sum_m s[m, r] * x[m, k] as mma.sync m16n8k16 with the 16 ranks as M, 8 columns as N and 16 rows
// as the contraction: reading the codes once bounds it, so the warp-level instruction is ample (without it 1.5 us
// less, when the kernel took 25). A warp walks 16 rows x 128 columns per step; its steps' codes, rows of s and step bytes are on their way to
// shared memory, four steps ahead and nobody else's (one step ahead in registers, 64 columns: 16,384 x 3584 40 us). Lane
// (g = lane / 4, t = lane % 4) takes 16 codes, columns 16g .. 16g + 15, of rows
// t, t + 4, t + 8 and t + 12, and column 16g + j of them is its part of the j-th of 16 products. (The contraction may
// visit the rows in any order that both operands share.) The values are fp16 numbers: a code on top of 1536, times the
// step, less 1536 steps, in one fma that is exact. (Steps outside 2^-24 .. 2^5 take another branch: below, of blocks below 2^-18,
// they go in as two factors; what they hold are multiples of 2^-24 like their source. s and
// x as bf16 need no such care but two products for the 11 bits of s: 32 us. A block of zeros has step byte 1 and takes that branch too: half of
// the rows zero, 23.2 us.) Sums are fp32 throughout: a warp's in its
// accumulators, the CTA's warps' in shared memory, row shares' in planes that a second kernel adds in order, so that
// results do not depend on timing. 16,384 x 3584 takes 22 us behind a kernel that wrote 117 MB, of which as much as is
// read here has to leave L2 meanwhile: 122 MB, 5.5 TB/s; copies by TMA in place of cp.async change nothing.
constexpr int A8G_WARPS = 8;
constexpr int A8G_COLS = 128;
constexpr int A8G_DEPTH = 4;
constexpr int A8G_PITCH = A8G_COLS + 32;      // of a row of codes: the four rows and two columns of eight lanes lie in as many banks
constexpr int A8G_CODES = 16 * A8G_PITCH, A8G_STEP_BYTES = A8G_CODES + 16 * 32 + 64;      // codes, s, step bytes
constexpr int A8G_SMEM = A8G_WARPS * A8G_DEPTH * A8G_STEP_BYTES;
constexpr int A8G_SUM_PITCH = A8G_COLS / 32 * 36;
static_assert(A8G_SMEM >= A8G_WARPS * 16 * A8G_SUM_PITCH * 4, "the warps' sums meet in the same memory");

__device__ __forceinline__ void a8_mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__global__ void __launch_bounds__(A8G_WARPS * 32, 2)
act8_lora_grad_kernel(const Act8LoraGrad a) {
    grid_dep_wait();
    grid_dep_launch();
    extern __shared__ uint4 a8_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int col0 = blockIdx.x * A8G_COLS;
    const long long row_begin = (long long)blockIdx.y * a.rows_per_split;
    const long long row_end = min(row_begin + a.rows_per_split, a.rows);
    const long long blocks = a.pitch / A8_BLOCK;
    const bool step_words = blocks % 4 == 0 && (reinterpret_cast<uintptr_t>(a.steps) & 3) == 0;
    const uint32_t ring = smem_u32(a8_smem) + (uint32_t)warp * (A8G_DEPTH * A8G_STEP_BYTES);
    float acc[16][4];
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;

    // where this lane's copies come from in the step at row 0, and go to
    const int piece = lane & 7, prow = lane >> 3;
    const bool piece_ok = col0 + piece * 16 < a.pitch;
    const long long first = row_begin + warp * 16;
    int todo = (int)(row_end - first);         // rows from the step to fetch to the end
    const int8_t* from_codes = a.codes + (first + prow) * a.pitch + (piece_ok ? col0 + piece * 16 : 0);
    const char* from_s = reinterpret_cast<const char*>(a.s) + first * 32 + lane * 16;
    const uint8_t* from_steps = a.steps + (first + (lane & 15)) * blocks + col0 / A8_BLOCK;    // (a tile begins at a multiple of four blocks)
    const long long row4 = 4 * a.pitch, ahead_codes = A8G_WARPS * 16 * a.pitch, ahead_steps = A8G_WARPS * 16 * blocks;
    const uint32_t to_codes = prow * A8G_PITCH + piece * 16;
    const auto fetch = [&](uint32_t at) {
        if (todo >= 16 && piece_ok) {
            const int8_t* p = from_codes;
#pragma unroll
            for (int i = 0; i < 4; ++i, p += row4) cp_async16(at + to_codes + i * 4 * A8G_PITCH, p);      // 8 pieces of 16 bytes a row
        } else if (todo > 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool there = piece_ok && i * 4 + prow < todo;
                cp_async16_or_zero(at + to_codes + i * 4 * A8G_PITCH, there ? from_codes + i * row4 : a.codes, there);
            }
        }
        if (todo > 0) {
            const bool there = (lane >> 1) < todo;
            cp_async16_or_zero(at + A8G_CODES + lane * 16, there ? from_s : reinterpret_cast<const char*>(a.s), there);
            if (lane < 16 && step_words) {
                const bool in = lane < todo;
                cp_async4_or_zero(at + A8G_CODES + 512 + lane * 4, in ? from_steps : a.steps, in);
            }
        }
        cp_async_commit();
        from_codes += ahead_codes;
        from_s += A8G_WARPS * 16 * 32;
        from_steps += ahead_steps;
        todo -= A8G_WARPS * 16;
    };
    for (int k = 0; k < A8G_DEPTH; ++k) fetch(ring + k * A8G_STEP_BYTES);
    // the fragment of s, rank-major: contraction index 2t is row t, 2t + 1 row t + 4, 2t + 8 and 2t + 9 rows t + 8, t + 12
    const int k8 = (lane & 7) + (lane >= 16 ? 8 : 0);      // (matrices 0, 1: indices 0 .. 7; 2, 3: 8 .. 15)
    const uint32_t at_s = A8G_CODES + (((k8 & 7) >> 1) + (k8 & 1) * 4 + (k8 & 8)) * 32 + ((lane >> 3) & 1) * 16;
    const uint32_t at_codes = t * A8G_PITCH + g * 16, at_steps = A8G_CODES + 512 + t * 4 + (g >> 1);
    const __half2 bias = __float2half2_rn(1536.f);
    uint32_t at = ring;
    for (int left = (int)(row_end - first); left > 0; left -= A8G_WARPS * 16) {
        cp_async_wait<A8G_DEPTH - 1>();
        __syncwarp();
        uint32_t q[4][4], st[4];
        bool plain = true;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(q[i][0]), "=r"(q[i][1]), "=r"(q[i][2]), "=r"(q[i][3])
                         : "r"(at + at_codes + i * 4 * A8G_PITCH));
            if (step_words) {
                asm volatile("ld.shared.u8 %0, [%1];" : "=r"(st[i]) : "r"(at + at_steps + i * 16));
            } else {
                const long long b = col0 / A8_BLOCK + (g >> 1), row = row_end - left + t + 4 * i;
                st[i] = t + 4 * i < left && b < blocks ? a.steps[row * blocks + b] : 0u;
            }
            plain = plain && (st[i] == 0u || st[i] - 103u <= 132u - 103u);
        }
        uint32_t f[4];
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(f[0]), "=r"(f[1]), "=r"(f[2]), "=r"(f[3]) : "r"(at + at_s));
        // A code of each of two rows, sign-extended; 0x6600 plus a number from -128 to 127 is 1536 plus it in fp16, and the
        // sum's upper byte is 0x66, or 0x65 where the number is negative.
        const auto two = [&](int w, int e, int p) {
            uint32_t x;
            asm("prmt.b32 %0, %1, %2, %3;" : "=r"(x) : "r"(q[2 * p][w]), "r"(q[2 * p + 1][w]), "r"(0xC480 + 0x1111 * e));
            x = (x & 0x03FF03FFu) ^ 0x66006600u;
            return *reinterpret_cast<const __half2*>(&x);
        };
        __half2 large[2];
        if (__all_sync(0xffffffffu, plain)) {      // steps of 2^-24 to 2^5 (or of nothing): 1536 steps are a number too
            __half2 off[2];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                large[p] = __floats2half2_rn(__uint_as_float(st[2 * p] << 23), __uint_as_float(st[2 * p + 1] << 23));
                off[p] = __hneg2(__hmul2(bias, large[p]));
            }
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t b[2];
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        const __half2 v = __hfma2(two(w, e, p), large[p], off[p]);
                        b[p] = *reinterpret_cast<const uint32_t*>(&v);
                    }
                    a8_mma16816(acc[4 * w + e], f, b[0], b[1]);
                }
        } else {                                   // a step below 2^-24: that, and a second factor. (NaN stays)
            __half2 small[2];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                float s1[2], s2[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    s1[i] = a8_value_of_step(st[2 * p + i]);
                    const bool below = s1[i] < 5.9604644775390625e-8f;
                    s2[i] = below ? s1[i] * 16777216.f : 1.f;
                    s1[i] = below ? 5.9604644775390625e-8f : s1[i];
                }
                large[p] = __floats2half2_rn(s1[0], s1[1]);
                small[p] = __floats2half2_rn(s2[0], s2[1]);
            }
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t b[2];
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        const __half2 v = __hmul2(__hmul2(__hsub2(two(w, e, p), bias), small[p]), large[p]);
                        b[p] = *reinterpret_cast<const uint32_t*>(&v);
                    }
                    a8_mma16816(acc[4 * w + e], f, b[0], b[1]);
                }
        }
        __syncwarp();      // (every lane has read the slot)
        fetch(at);
        at = at == ring + (A8G_DEPTH - 1) * A8G_STEP_BYTES ? ring : at + A8G_STEP_BYTES;
    }
    cp_async_wait<0>();
    __syncthreads();
    // acc[j]: ranks g, g, g + 8, g + 8 of columns 16 * (2t) + j and 16 * (2t + 1) + j (N index n stands for the column
    // group of the lanes with g = n). Every warp lays its sums down, every thread adds the warps' for some outputs. A rank's
    // 32-column quarters are 36 values apart: the banks of eight lanes with two ranks and four t differ.
    const uint32_t sums = smem_u32(a8_smem);
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int j = 0; j < 16; j += 4)
            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};"
                         ::"r"(sums + 4 * ((warp * 16 + g + (h >> 1) * 8) * A8G_SUM_PITCH + t * 36 + (h & 1) * 16 + j)),
                           "f"(acc[j][h]), "f"(acc[j + 1][h]), "f"(acc[j + 2][h]), "f"(acc[j + 3][h]) : "memory");
    __syncthreads();
    float* out = a.splits > 1 ? a.planes + (long long)blockIdx.y * 16 * a.cols : a.out;
    for (int i = threadIdx.x; i < 16 * A8G_COLS / 4; i += A8G_WARPS * 32) {
        const int r = i / (A8G_COLS / 4), c = i % (A8G_COLS / 4) * 4;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < A8G_WARPS; ++w) {
            float x[4];
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3])
                         : "r"(sums + 4 * ((w * 16 + r) * A8G_SUM_PITCH + c / 32 * 36 + c % 32)));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += x[e];
        }
        float* to = out + (long long)r * a.cols + col0 + c;
        if (a.cols % 4 == 0 && col0 + c < a.cols && (reinterpret_cast<uintptr_t>(out) & 15) == 0) {
            *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (col0 + c + e < a.cols) to[e] = v[e];
        }
    }
}

__global__ void __launch_bounds__(256)
act8_lora_sum_kernel(const float* __restrict__ planes, float* __restrict__ out, long long n, int splits) {
    grid_dep_wait();
    grid_dep_launch();
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float v = 0.f;
#pragma unroll 8
    for (int z = 0; z < splits; ++z) v += planes[z * n + i];
    out[i] = v;
}

// ------------------------------------------------------------------------------------------- host side
static bool a8_whole(const void* a, const void* b, long long cols) {
    return cols % A8_BLOCK == 0 && ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0;
}

static A8Rows a8_rows(long long rows, long long cols) {
    return A8Rows{rows, (cols + A8_BLOCK - 1) / A8_BLOCK, (int)cols};
}

static dim3 a8_grid(const A8Rows& g, int sm_count) {
    const long long ctas = (g.rows * g.blocks + A8_THREADS / 32 - 1) / (A8_THREADS / 32), cap = (long long)sm_count * 32;
    return dim3((unsigned)(ctas < cap ? ctas : cap));
}

static dim3 a8_flat_grid(long long n16) { return dim3((unsigned)((n16 + A8_THREADS - 1) / A8_THREADS)); }

template <typename T>
static cudaError_t quantize_as(const Act8Convert& a, cudaStream_t stream) {
    if (a8_whole(a.x, a.codes, a.cols)) {
        const long long n16 = a.rows * a.cols / 16;
        return launch_pdl(act8_quantize_kernel<T>, a8_flat_grid(n16), dim3(A8_THREADS), 0, stream, (const void*)a.x,
                          reinterpret_cast<uint4*>(a.codes), a.steps, n16);
    }
    const A8Rows g = a8_rows(a.rows, a.cols);
    return launch_pdl(act8_quantize_any_kernel<T>, a8_grid(g, a.sm_count), dim3(A8_THREADS), 0, stream,
                      (const void*)a.x, a.codes, a.steps, g);
}

template <typename T>
static cudaError_t dequantize_as(const Act8Convert& a, cudaStream_t stream) {
    if (a8_whole(a.x, a.codes, a.cols)) {
        const long long n16 = a.rows * a.cols / 16;
        return launch_pdl(act8_dequantize_kernel<T>, a8_flat_grid(n16), dim3(A8_THREADS), 0, stream,
                          reinterpret_cast<const uint4*>(a.codes), (const uint8_t*)a.steps, a.x, n16);
    }
    const A8Rows g = a8_rows(a.rows, a.cols);
    return launch_pdl(act8_dequantize_any_kernel<T>, a8_grid(g, a.sm_count), dim3(A8_THREADS), 0, stream,
                      (const int8_t*)a.codes, (const uint8_t*)a.steps, a.x, g);
}

cudaError_t launch_act8_quantize(const Act8Convert& a, cudaStream_t stream) {
    if (a.rows <= 0 || a.cols <= 0) return cudaSuccess;
    return a.dtype == 0 ? quantize_as<__half>(a, stream) : a.dtype == 1 ? quantize_as<__nv_bfloat16>(a, stream)
                                                                        : quantize_as<float>(a, stream);
}

cudaError_t launch_act8_dequantize(const Act8Convert& a, cudaStream_t stream) {
    if (a.rows <= 0 || a.cols <= 0) return cudaSuccess;
    return a.dtype == 0 ? dequantize_as<__half>(a, stream) : a.dtype == 1 ? dequantize_as<__nv_bfloat16>(a, stream)
                                                                          : dequantize_as<float>(a, stream);
}

cudaError_t launch_act8_swiglu(const Act8Swiglu& a, bool backward, cudaStream_t stream) {
    if (a.rows <= 0 || a.cols <= 0) return cudaSuccess;
    const bool whole = a8_whole(a.gate_codes, a.up_codes, a.cols) &&
                       (backward ? a8_whole(a.d_hidden, a.d_gate, a.cols) && a8_whole(a.d_up, a.d_up, a.cols)
                                 : a8_whole(a.gate, a.up, a.cols) && a8_whole(a.hidden, a.hidden, a.cols));
    if (whole) {
        const long long n16 = a.rows * a.cols / 16;
        return launch_pdl(backward ? act8_swiglu_bwd_kernel : act8_swiglu_fwd_kernel, a8_flat_grid(n16), dim3(A8_THREADS),
                          0, stream, a, n16);
    }
    const A8Rows g = a8_rows(a.rows, a.cols);
    return launch_pdl(act8_swiglu_any_kernel, a8_grid(g, a.sm_count), dim3(A8_THREADS), 0, stream, a, g, backward ? 1 : 0);
}

// Row shares: two CTAs per SM as far as that goes without a third wave, each of at least a step of every warp.
int act8_lora_grad_splits(long long rows, long long cols, int sm_count) {
    const long long tiles = (cols + A8G_COLS - 1) / A8G_COLS, step = A8G_WARPS * 16;
    long long splits = 2ll * sm_count / tiles;
    const long long most = (rows + step - 1) / step;
    if (splits > most) splits = most;
    return splits < 1 ? 1 : (int)splits;
}

cudaError_t launch_act8_lora_grad(const Act8LoraGrad& a_in, cudaStream_t stream) {
    Act8LoraGrad a = a_in;
    const long long step = A8G_WARPS * 16;
    a.pitch = (a.cols + A8_BLOCK - 1) / A8_BLOCK * A8_BLOCK;
    a.splits = act8_lora_grad_splits(a.rows, a.cols, a.sm_count);
    a.rows_per_split = (a.rows + a.splits - 1) / a.splits;
    a.rows_per_split = (a.rows_per_split + step - 1) / step * step;
    a.splits = (int)((a.rows + a.rows_per_split - 1) / a.rows_per_split);   // no empty share
    const dim3 grid((unsigned)((a.cols + A8G_COLS - 1) / A8G_COLS), (unsigned)a.splits);
    cudaError_t e = cudaFuncSetAttribute(act8_lora_grad_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, A8G_SMEM);
    if (e != cudaSuccess) return e;
    e = launch_pdl(act8_lora_grad_kernel, grid, dim3(A8G_WARPS * 32), A8G_SMEM, stream, a);
    if (e != cudaSuccess || a.splits == 1) return e;
    const long long n = 16 * a.cols;
    return launch_pdl(act8_lora_sum_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream,
                      (const float*)a.planes, a.out, n, a.splits);
}

}  // namespace nf4
