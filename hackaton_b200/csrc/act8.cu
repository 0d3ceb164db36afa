// Activations kept in 8 bits for the backward pass (the form: act8.cuh), and what reads them there:
//   quantize / dequantize   the values of a tensor to codes and steps, and back
//   SwiGLU                  hidden = gate * sigmoid(gate) * up with gate and up kept in the same pass; the
//                           backward from the codes (the arithmetic of swiglu.cuh)
//   LoRA gradient           dA[r, k] = sum_m s[m, r] * x[m, k] from the codes of x
// All are bound by memory: per value quantize 3.03 bytes, dequantize 3.03, SwiGLU forward 8.06, backward 8.06,
// the gradient 1.03 and a share of s.
// A thread takes 16 values (32 bytes of fp16 in two 16-byte accesses, one 16-byte access of codes), two
// threads a block of 32, whose largest magnitude is one shuffle away. Rows that are not whole blocks or not 16-byte
// aligned go a warp per block, a lane per value.
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
// as the contraction: bound by reading the codes once, so the warp-level instruction is ample. A warp walks
// 16 rows x 64 columns per step: lane (g = lane / 4, t = lane % 4) reads 8 codes, columns 8g .. 8g + 7, of rows
// 2t, 2t + 1, 2t + 8 and 2t + 9, and column 8g + j of them is its part of the j-th of 8 products. The values go in as bf16, which holds a code times a power of two exactly, over
// fp32's range (fp16 would lose blocks below 2^-18); s, fp16 with 11 significant bits, as the sum of two bf16 numbers,
// also exact. Sums are fp32 throughout: a warp's in its accumulators, the CTA's warps' in shared memory, row
// shares' in planes that a second kernel adds in order, so that results do not depend on timing.
constexpr int A8G_WARPS = 8;
constexpr int A8G_COLS = 64;

__device__ __forceinline__ void a8_mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two fp16 numbers as the sum of two pairs of bf16 numbers.
__device__ __forceinline__ void a8_split(uint32_t x0, uint32_t x1, uint32_t& hi, uint32_t& lo) {
    const float2 f = A8Source<__half>::two(x0 | x1 << 16);
    hi = A8Source<__nv_bfloat16>::pack(f.x, f.y);
    const float2 h = A8Source<__nv_bfloat16>::two(hi);
    lo = A8Source<__nv_bfloat16>::pack(f.x - h.x, f.y - h.y);
}

__global__ void __launch_bounds__(A8G_WARPS * 32, 2)
act8_lora_grad_kernel(const Act8LoraGrad a) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ float sums[A8G_WARPS / 2][16][A8G_COLS + 4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int col0 = blockIdx.x * A8G_COLS, col = col0 + 8 * g;
    const bool col_ok = col < a.pitch;
    const long long row_begin = (long long)blockIdx.y * a.rows_per_split;
    const long long row_end = min(row_begin + a.rows_per_split, a.rows);
    const uint2* codes = reinterpret_cast<const uint2*>(a.codes + col);
    const long long pitch8 = a.pitch / 8, steps_pitch = a.pitch / A8_BLOCK;
    const uint8_t* steps = a.steps + col / A8_BLOCK;
    const unsigned short* s = reinterpret_cast<const unsigned short*>(a.s) + g;
    const int at[4] = {2 * t, 2 * t + 1, 2 * t + 8, 2 * t + 9};
    float acc[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;

    struct Step {
        uint2 q[4];
        uint32_t st[4], lo[4], hi[4];
    } next;
    const auto fetch = [&](long long r0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long long r = r0 + at[i];
            const bool ok = r < row_end;
            next.q[i] = make_uint2(0u, 0u);
            next.st[i] = 0u;
            next.lo[i] = next.hi[i] = 0u;
            if (ok && col_ok) {
                next.q[i] = __ldcs(codes + r * pitch8);
                next.st[i] = __ldg(steps + r * steps_pitch);
            }
            if (ok) {
                next.lo[i] = __ldg(s + r * 16);
                next.hi[i] = __ldg(s + r * 16 + 8);
            }
        }
    };
    long long r0 = row_begin + warp * 16;
    fetch(r0);
    for (; r0 < row_end; r0 += A8G_WARPS * 16) {
        const Step now = next;
        fetch(r0 + A8G_WARPS * 16);
        uint32_t hi[4], lo[4];
        a8_split(now.lo[0], now.lo[1], hi[0], lo[0]);
        a8_split(now.hi[0], now.hi[1], hi[1], lo[1]);
        a8_split(now.lo[2], now.lo[3], hi[2], lo[2]);
        a8_split(now.hi[2], now.hi[3], hi[3], lo[3]);
        float scale[4], shift[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            scale[i] = a8_value_of_step(now.st[i]);
            shift[i] = -8388736.f * scale[i];
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            uint32_t word[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                word[i] = (w == 0 ? now.q[i].x : now.q[i].y) ^ 0x80808080u;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t v[4], b[2];
#pragma unroll
                for (int i = 0; i < 4; ++i)   // (2^23 + 128 + q) * step - (2^23 + 128) * step: exact, seven bits
                    v[i] = __float_as_uint(fmaf(__uint_as_float(__byte_perm(word[i], 0x4B000000u, 0x7440 + e)),
                                                scale[i], shift[i]));
                b[0] = __byte_perm(v[0], v[1], 0x7632);   // their upper halves are the bf16 numbers
                b[1] = __byte_perm(v[2], v[3], 0x7632);
                a8_mma16816(acc[4 * w + e], hi, b[0], b[1]);
                a8_mma16816(acc[4 * w + e], lo, b[0], b[1]);
            }
        }
    }
    // acc[j]: ranks g, g, g + 8, g + 8 of columns 8 * (2t) + j and 8 * (2t + 1) + j (N index n stands for the column
    // group of the lanes with g = n)
    for (int half = A8G_WARPS / 2; half >= 1; half >>= 1) {
        if (warp >= half && warp < 2 * half) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                sums[warp - half][g][16 * t + j] = acc[j][0];
                sums[warp - half][g][16 * t + 8 + j] = acc[j][1];
                sums[warp - half][g + 8][16 * t + j] = acc[j][2];
                sums[warp - half][g + 8][16 * t + 8 + j] = acc[j][3];
            }
        }
        __syncthreads();
        if (warp < half) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                acc[j][0] += sums[warp][g][16 * t + j];
                acc[j][1] += sums[warp][g][16 * t + 8 + j];
                acc[j][2] += sums[warp][g + 8][16 * t + j];
                acc[j][3] += sums[warp][g + 8][16 * t + 8 + j];
            }
        }
        __syncthreads();
    }
    if (warp == 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            sums[0][g][16 * t + j] = acc[j][0];
            sums[0][g][16 * t + 8 + j] = acc[j][1];
            sums[0][g + 8][16 * t + j] = acc[j][2];
            sums[0][g + 8][16 * t + 8 + j] = acc[j][3];
        }
    }
    __syncthreads();
    float* out = a.splits > 1 ? a.planes + (long long)blockIdx.y * 16 * a.cols : a.out;
    for (int i = threadIdx.x; i < 16 * A8G_COLS; i += A8G_WARPS * 32) {
        const int r = i / A8G_COLS, c = i % A8G_COLS;
        if (col0 + c < a.cols) out[(long long)r * a.cols + col0 + c] = sums[0][r][c];
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

// Row shares: about two CTAs per SM, each of at least a step of every warp.
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
    cudaError_t e = launch_pdl(act8_lora_grad_kernel, grid, dim3(A8G_WARPS * 32), 0, stream, a);
    if (e != cudaSuccess || a.splits == 1) return e;
    const long long n = 16 * a.cols;
    return launch_pdl(act8_lora_sum_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream,
                      (const float*)a.planes, a.out, n, a.splits);
}

}  // namespace nf4
