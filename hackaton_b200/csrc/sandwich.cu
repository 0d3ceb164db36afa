// The norm behind a block, its gate, the scaled residual and the norm before the next block in one pass each
// way, on the fp32 stream:
//   n = delta * rd * post              rd = 1 / sqrt(mean(delta^2) + eps)
//   s = scale * residual + gate * n    gate: none, or [gates, hidden], a row for rows / gates rows in a row
//   y = s * rs * pre                   rs = 1 / sqrt(mean(s^2) + eps)
// and, from d_stream (what reaches s directly) and dy, with dh = delta * rd, sh = s * rs, w = dy * pre, g = gate * post:
//   ds = d_stream + rs * (w - sh * mean(w * sh))
//   d_residual = scale * ds            d_delta = rd * (g ds - dh * mean(g ds * dh))
//   d_gate = post * sum ds dh          d_post = sum gate * ds dh        d_pre = sum dy * sh      (over rows)
// The backward's second mean is linear in ds, so that both means come out of one reduction of three sums:
//   mean(g ds dh) = mean(g dh (d_stream + rs w)) - rs mean(w sh) mean(g dh sh)
// Memory bound: 4 + 4 bytes per value of the stream and 2 + 2 of 16-bit delta and y forward (12), 18 backward. A CTA
// keeps a thread's columns of the weights in registers over all its rows; rows to come are on their way to shared
// memory, each thread's own columns into slots that nobody else reads (cp.async, no barrier), four rows ahead forward and
// three backward, since two or three CTAs of an SM with one row each in flight leave most of the bandwidth idle (one row
// ahead in registers: 16,384 x 1536 82 and 129 us). Column sums of the weights' gradients stay in registers; a second
// kernel adds the CTAs' sums in order, so that results do not depend on timing. All sums are fp32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.h"
#include "ptx.cuh"

namespace nf4 {

// VEC values of a type as they lie in memory.
template <typename T, int VEC> struct SwRaw;

template <> struct SwRaw<float, 4> {
    static __device__ __forceinline__ void copy(uint32_t dst, const void* p, long long i) { cp_async16(dst, static_cast<const float*>(p) + i); }
    float4 v;
    __device__ __forceinline__ void load(const void* p, long long i) { v = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i)); }
    __device__ __forceinline__ void get(float (&f)[4]) const { f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
    static __device__ __forceinline__ void store(void* p, long long i, const float (&f)[4]) {
        *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(f[0], f[1], f[2], f[3]);
    }
};
template <> struct SwRaw<__half, 4> {
    static __device__ __forceinline__ void copy(uint32_t dst, const void* p, long long i) { cp_async8(dst, static_cast<const __half*>(p) + i); }
    uint2 v;
    __device__ __forceinline__ void load(const void* p, long long i) { v = __ldg(reinterpret_cast<const uint2*>(static_cast<const __half*>(p) + i)); }
    __device__ __forceinline__ void get(float (&f)[4]) const {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
        f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
    }
    static __device__ __forceinline__ void store(void* p, long long i, const float (&f)[4]) {
        const __half2 a = __floats2half2_rn(f[0], f[1]), b = __floats2half2_rn(f[2], f[3]);
        *reinterpret_cast<uint2*>(static_cast<__half*>(p) + i) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
};
template <> struct SwRaw<__nv_bfloat16, 4> {
    static __device__ __forceinline__ void copy(uint32_t dst, const void* p, long long i) { cp_async8(dst, static_cast<const __nv_bfloat16*>(p) + i); }
    uint2 v;
    __device__ __forceinline__ void load(const void* p, long long i) { v = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p) + i)); }
    __device__ __forceinline__ void get(float (&f)[4]) const {
        f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xFFFF0000u);
        f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xFFFF0000u);
    }
    static __device__ __forceinline__ void store(void* p, long long i, const float (&f)[4]) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p) + i) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
};
__device__ __forceinline__ float sw_float(float x) { return x; }
__device__ __forceinline__ float sw_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float sw_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void sw_round(float x, float& y) { y = x; }
__device__ __forceinline__ void sw_round(float x, __half& y) { y = __float2half_rn(x); }
__device__ __forceinline__ void sw_round(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }
template <typename T> struct SwRaw<T, 1> {
    T v;
    __device__ __forceinline__ void load(const void* p, long long i) { v = static_cast<const T*>(p)[i]; }
    __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = sw_float(v); }
    static __device__ __forceinline__ void store(void* p, long long i, const float (&f)[1]) { sw_round(f[0], static_cast<T*>(p)[i]); }
};

// Rows on their way: `depth` slots of what a thread's columns take of one array, [slot][i][thread]. Rows of single
// values (VEC = 1) go through registers, one row ahead.
template <typename T, int NV, int VEC>
struct SwRing {
    SwRaw<T, VEC> next[VEC == 4 ? 1 : NV];
    uint32_t base;     // this thread's place in slot 0
    // Bytes of the ring; `at` moves behind it.
    __device__ __forceinline__ void place(uint32_t& at, int depth) {
        if (VEC != 4) return;
        base = at + threadIdx.x * (4 * sizeof(T));
        at += depth * NV * blockDim.x * (4 * sizeof(T));
    }
    __device__ __forceinline__ void ask(int slot, int i, const void* p, long long index) {
        if constexpr (VEC == 4) SwRaw<T, 4>::copy(base + (slot * NV + i) * blockDim.x * (4 * sizeof(T)), p, index);
        else                    next[i].load(p, index);
    }
    __device__ __forceinline__ void get(int slot, int i, float (&f)[VEC]) const {
        if constexpr (VEC == 4) {
            const uint32_t a = base + (slot * NV + i) * blockDim.x * (4 * sizeof(T));
            SwRaw<T, 4> raw;
            if constexpr (sizeof(T) == 4)
                asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(raw.v.x), "=f"(raw.v.y), "=f"(raw.v.z), "=f"(raw.v.w) : "r"(a));
            else
                asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(raw.v.x), "=r"(raw.v.y) : "r"(a));
            raw.get(f);
        } else {
            next[i].get(f);
        }
    }
};

// Threads up to which a kernel may take 80 registers each forward and 128 backward.
constexpr int SW_FEW_FWD = 256, SW_FEW_BWD = 512;
constexpr int SW_FWD_DEPTH = 4, SW_BWD_DEPTH = 3;      // where shared memory allows

// Waits for this thread's copies of the oldest of `depth` rows.
__device__ __forceinline__ void sw_oldest(int depth) {
    if (depth >= 4)      cp_async_wait<3>();
    else if (depth == 3) cp_async_wait<2>();
    else if (depth == 2) cp_async_wait<1>();
    else                 cp_async_wait<0>();
}

// Sums of N values over the CTA, the same in every thread: a warp's by shuffles, the warps' by every thread for itself
// (a broadcast load per four warps; shuffles are what a row of few columns per thread spends its time on). `part` has two
// halves that successive calls take in turn: who writes a half again has passed the barrier behind which everybody
// had read it. What belongs to warps that are not there is zero from the start.
template <int N>
__device__ __forceinline__ void sw_block_sum(float (&v)[N], float (*part)[N][32], int& turn) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (warps > 1) {
        if (lane == 0)
#pragma unroll
            for (int n = 0; n < N; ++n) part[turn][n][threadIdx.x >> 5] = v[n];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = 0.f;
        for (int w = 0; w < warps; w += 4)
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const float4 x = *reinterpret_cast<const float4*>(&part[turn][n][w]);
                v[n] += (x.x + x.y) + (x.z + x.w);
            }
        turn ^= 1;
    }
}

// (the barrier in the first sum comes behind this for every half that is read)
template <int N>
__device__ __forceinline__ void sw_clear(float (*part)[N][32]) {
    for (int i = threadIdx.x; i < 2 * N * 32; i += blockDim.x)
        if ((i & 31) >= (int)(blockDim.x >> 5)) (&part[0][0][0])[i] = 0.f;
}

template <int NV, int VEC>
__device__ __forceinline__ void sw_weights(const float* p, int hidden, float fill, float (&w)[NV][VEC]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (threadIdx.x + i * blockDim.x) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[i][e] = fill;
        if (p != nullptr && c < hidden) {
            SwRaw<float, VEC> raw;
            raw.load(p, c);
            raw.get(w[i]);
        }
    }
}

template <int NV, int VEC, typename TD, typename TY, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT <= SW_FEW_FWD ? 3 : 1)
sandwich_fwd_kernel(const SandwichArgs a) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ __align__(16) float part[2][1][32];
    int turn = 0;
    sw_clear<1>(part);
    const int hidden = a.hidden;
    const float inv_h = 1.f / (float)hidden;
    float post[NV][VEC], pre[NV][VEC];
    sw_weights<NV, VEC>(a.post, hidden, 0.f, post);
    sw_weights<NV, VEC>(a.pre, hidden, 0.f, pre);
    if (a.gates == 1) {
        float gate[NV][VEC];
        sw_weights<NV, VEC>(a.gate, hidden, 0.f, gate);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) post[i][e] *= gate[i][e];
    }
    const int depth = VEC == 4 ? a.depth : 1;
    extern __shared__ uint4 sw_smem[];
    uint32_t room = smem_u32(sw_smem);
    SwRing<float, NV, VEC> ring_r;
    SwRing<TD, NV, VEC> ring_d;
    ring_r.place(room, depth);
    ring_d.place(room, depth);
    const auto fetch = [&](long long row, int slot) {
        if (row < a.rows) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (threadIdx.x + i * blockDim.x) * VEC;
                if (c < hidden) {
                    ring_d.ask(slot, i, a.delta, row * hidden + c);
                    ring_r.ask(slot, i, a.residual, row * hidden + c);
                }
            }
        }
        if (VEC == 4) cp_async_commit();
    };
    long long row = blockIdx.x;
    for (int k = 0; k < depth; ++k) fetch(row + (long long)k * gridDim.x, k);
    for (int slot = 0; row < a.rows; row += gridDim.x, slot = slot + 1 == depth ? 0 : slot + 1) {
        if (VEC == 4) sw_oldest(depth);
        float d[NV][VEC], s[NV][VEC], sum[1] = {0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (threadIdx.x + i * blockDim.x) * VEC;
#pragma unroll
            for (int e = 0; e < VEC; ++e) d[i][e] = s[i][e] = 0.f;
            if (c < hidden) {
                ring_d.get(slot, i, d[i]);
                ring_r.get(slot, i, s[i]);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum[0] += d[i][e] * d[i][e];
        }
        if (VEC != 4) fetch(row + gridDim.x, 0);
        sw_block_sum<1>(sum, part, turn);
        const float rd = 1.f / sqrtf(sum[0] * inv_h + a.eps);
        if (VEC == 4) fetch(row + (long long)depth * gridDim.x, slot);    // (behind the barrier: the slot has been read)
        sum[0] = 0.f;
        const float* gate_row = a.gates > 1 ? a.gate + row / a.group_rows * hidden : nullptr;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (threadIdx.x + i * blockDim.x) * VEC;
            float n[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) n[e] = d[i][e] * rd * post[i][e];
            if (gate_row != nullptr && c < hidden) {
                SwRaw<float, VEC> raw;
                float gate[VEC];
                raw.load(gate_row, c);
                raw.get(gate);
#pragma unroll
                for (int e = 0; e < VEC; ++e) n[e] *= gate[e];
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                s[i][e] = fmaf(a.scale, s[i][e], n[e]);
                sum[0] += s[i][e] * s[i][e];
            }
            if (c < hidden) SwRaw<float, VEC>::store(a.stream, row * hidden + c, s[i]);
        }
        sw_block_sum<1>(sum, part, turn);
        const float rs = 1.f / sqrtf(sum[0] * inv_h + a.eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (threadIdx.x + i * blockDim.x) * VEC;
            float y[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) y[e] = pre[i][e] * (s[i][e] * rs);
            if (c < hidden) SwRaw<TY, VEC>::store(a.normed, row * hidden + c, y);
        }
        if (threadIdx.x == 0 && a.rstd != nullptr) {
            a.rstd[2 * row] = rd;
            a.rstd[2 * row + 1] = rs;
        }
    }
}

// A unit is a share of the rows that one gate row serves; a CTA takes units blockIdx.x, + gridDim.x, ...
template <int NV, int VEC, typename TD, typename TY, int MAXT>
__global__ void __launch_bounds__(MAXT, 1)
sandwich_bwd_kernel(const SandwichArgs a) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ __align__(16) float part[2][3][32];
    int turn = 0;
    sw_clear<3>(part);
    const int hidden = a.hidden;
    const float inv_h = 1.f / (float)hidden;
    float post[NV][VEC], pre[NV][VEC], gate[NV][VEC], sum_post[NV][VEC], sum_pre[NV][VEC], sum_unit[NV][VEC];
    sw_weights<NV, VEC>(a.post, hidden, 0.f, post);
    sw_weights<NV, VEC>(a.pre, hidden, 0.f, pre);
    sw_weights<NV, VEC>(a.gates == 1 ? a.gate : nullptr, hidden, 1.f, gate);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum_post[i][e] = sum_pre[i][e] = sum_unit[i][e] = 0.f;

    const int depth = VEC == 4 ? a.depth : 1;
    extern __shared__ uint4 sw_smem[];
    uint32_t room = smem_u32(sw_smem);
    SwRing<float, NV, VEC> ring_s, ring_t;
    SwRing<TD, NV, VEC> ring_d;
    SwRing<TY, NV, VEC> ring_y;
    ring_s.place(room, depth);
    ring_t.place(room, depth);
    ring_d.place(room, depth);
    ring_y.place(room, depth);
    const uint32_t ring_rstd = room + threadIdx.x * 8;      // (a copy for every thread)
    float2 next_rstd = make_float2(0.f, 0.f);
    const auto fetch = [&](int row, int slot) {      // (a negative row: nothing)
        if (row >= 0) {
            const long long at = (long long)row * hidden;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (threadIdx.x + i * blockDim.x) * VEC;
                if (c < hidden) {
                    ring_s.ask(slot, i, a.stream, at + c);
                    ring_d.ask(slot, i, a.delta, at + c);
                    ring_y.ask(slot, i, a.d_normed, at + c);
                    if (a.d_stream != nullptr) ring_t.ask(slot, i, a.d_stream, at + c);
                }
            }
            if (VEC == 4) cp_async8(ring_rstd + slot * blockDim.x * 8, a.rstd + 2ll * row);
            else          next_rstd = *reinterpret_cast<const float2*>(a.rstd + 2ll * row);
        }
        if (VEC == 4) cp_async_commit();
    };
    // two walks over this CTA's rows: the one that asks for them is depth rows ahead of the one that works on them
    const int shares = (int)a.shares, share_rows = (int)a.share_rows, group_rows = (int)a.group_rows, units = (int)a.units;
    struct Walk {
        int unit, row, end;
    };
    const auto enter = [&](Walk& w) {
        const int group = w.unit / shares, share = w.unit - group * shares;
        w.row = group * group_rows + share * share_rows;
        w.end = min(w.row + share_rows, (group + 1) * group_rows);
    };
    const auto step = [&](Walk& w) {     // row -1 behind the last one
        if (w.row < 0 || ++w.row < w.end) return;
        w.unit += gridDim.x;
        if (w.unit < units) enter(w);
        else                w.row = -1;
    };
    Walk ahead;
    ahead.unit = blockIdx.x;   // (gridDim.x <= units)
    enter(ahead);
    Walk now = ahead;
    for (int k = 0; k < depth; ++k) {
        fetch(ahead.row, k);
        step(ahead);
    }
    bool new_unit = true;
    for (int slot = 0; now.row >= 0; slot = slot + 1 == depth ? 0 : slot + 1) {
        if (VEC == 4) sw_oldest(depth);
        if (a.gates > 1 && new_unit) sw_weights<NV, VEC>(a.gate + (long long)(now.unit / shares) * hidden, hidden, 0.f, gate);
        float2 rstd = next_rstd;
        if (VEC == 4) asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(rstd.x), "=f"(rstd.y) : "r"(ring_rstd + slot * blockDim.x * 8));
        const float rd = rstd.x, rs = rstd.y;
        float s[NV][VEC], t[NV][VEC], d[NV][VEC], y[NV][VEC], sum[3] = {0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (threadIdx.x + i * blockDim.x) * VEC;
#pragma unroll
            for (int e = 0; e < VEC; ++e) s[i][e] = t[i][e] = d[i][e] = y[i][e] = 0.f;
            if (c < hidden) {
                ring_s.get(slot, i, s[i]);
                ring_d.get(slot, i, d[i]);
                ring_y.get(slot, i, y[i]);
                if (a.d_stream != nullptr) ring_t.get(slot, i, t[i]);
            }
        }
        const long long at = (long long)now.row * hidden;
        const int this_unit = now.unit;
        step(now);
        const bool unit_done = now.row < 0 || now.unit != this_unit;
        new_unit = unit_done;
        if (VEC != 4) {
            fetch(ahead.row, 0);
            step(ahead);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                s[i][e] *= rs;                                      // sh
                d[i][e] *= rd;                                      // dh
                const float w = y[i][e] * pre[i][e], gd = gate[i][e] * post[i][e] * d[i][e];
                t[i][e] = fmaf(rs, w, t[i][e]);                     // ds but for the mean
                sum[0] += w * s[i][e];
                sum[1] += gd * t[i][e];
                sum[2] += gd * s[i][e];
                sum_pre[i][e] += y[i][e] * s[i][e];
            }
        sw_block_sum<3>(sum, part, turn);
        if (VEC == 4) {       // (behind the barrier: the slot has been read)
            fetch(ahead.row, slot);
            step(ahead);
        }
        const float m1 = rs * (sum[0] * inv_h);
        const float m2 = (sum[1] - m1 * sum[2]) * inv_h;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (threadIdx.x + i * blockDim.x) * VEC;
            float dr[VEC], dd[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float ds = fmaf(-m1, s[i][e], t[i][e]);
                dr[e] = a.scale * ds;
                dd[e] = rd * (ds * (gate[i][e] * post[i][e]) - d[i][e] * m2);
                sum_unit[i][e] = fmaf(ds, d[i][e], sum_unit[i][e]);
            }
            if (c < hidden) {
                if (a.d_residual != nullptr) SwRaw<float, VEC>::store(a.d_residual, at + c, dr);
                if (a.d_delta != nullptr) SwRaw<TD, VEC>::store(a.d_delta, at + c, dd);
            }
        }
        if (unit_done) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (threadIdx.x + i * blockDim.x) * VEC;
                float dg[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    dg[e] = post[i][e] * sum_unit[i][e];
                    sum_post[i][e] = fmaf(gate[i][e], sum_unit[i][e], sum_post[i][e]);
                    sum_unit[i][e] = 0.f;
                }
                // (one share per gate row: the row itself; otherwise the shares' plane)
                if (a.d_gate != nullptr && c < hidden)
                    SwRaw<float, VEC>::store(shares == 1 ? a.d_gate : a.planes_gate, (long long)this_unit * hidden + c, dg);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (threadIdx.x + i * blockDim.x) * VEC;
        if (c >= hidden) continue;
        if (a.d_post != nullptr) SwRaw<float, VEC>::store(a.planes_post, (long long)blockIdx.x * hidden + c, sum_post[i]);
        if (a.d_pre != nullptr) SwRaw<float, VEC>::store(a.planes_pre, (long long)blockIdx.x * hidden + c, sum_pre[i]);
    }
}

// Adds the planes in order: blockIdx.y 0 d_post, 1 d_pre, then a gate row each. 32 columns by 32 shares of the planes.
__global__ void __launch_bounds__(1024)
sandwich_sum_kernel(const SandwichArgs a) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ float part[32][33];
    const int col = blockIdx.x * 32 + threadIdx.x;
    for (long long job = blockIdx.y; job < 2 + (a.shares > 1 ? a.groups : 0); job += gridDim.y) {
        const float* planes = job == 0 ? a.planes_post : job == 1 ? a.planes_pre : a.planes_gate + (job - 2) * a.shares * a.hidden;
        float* out = job == 0 ? a.d_post : job == 1 ? a.d_pre : a.d_gate == nullptr ? nullptr : a.d_gate + (job - 2) * a.hidden;
        const long long count = job < 2 ? a.grid : a.shares;
        float v = 0.f;
        if (out != nullptr && col < a.hidden) {
#pragma unroll 4
            for (long long p = threadIdx.y; p < count; p += 32) v += planes[p * a.hidden + col];
        }
        part[threadIdx.y][threadIdx.x] = v;
        __syncthreads();
        float t = part[threadIdx.x][threadIdx.y];   // transposed: a warp holds one column's shares
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        const int c = blockIdx.x * 32 + threadIdx.y;
        if (out != nullptr && threadIdx.x == 0 && c < a.hidden) out[c] = t;
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------- host side
struct SandwichShape {
    int vec, nv, threads, depth;
    size_t smem;      // of the rings
};

// Columns per thread: two or four float4 where a row is then left to eight warps or fewer (its sums cost every warp ten
// shuffles and more: 16,384 x 1536 with one float4 74 and 97 us, PLACEHOLDER), as many as registers hold backward; one where there
// are few rows and latency counts; single values for rows that are no whole float4, not aligned, or too long for one of
// them in shared memory.
static SandwichShape sandwich_shape(int hidden, bool vec, bool few, bool backward, int delta_type, int normed_type) {
    const size_t room = (227 << 10) - 2048;
    SandwichShape s = {};
    s.vec = vec && hidden % 4 == 0 ? 4 : 1;
    for (;;) {
        const int items = (hidden + s.vec - 1) / s.vec;
        if (s.vec == 4) s.nv = items <= (few ? 1024 : backward ? 192 : 256) ? 1 : items <= (few ? 2048 : backward ? 1024 : 512) ? 2 : 4;
        else            s.nv = items <= 4096 ? 4 : 16;
        s.threads = ((items + s.nv - 1) / s.nv + 31) / 32 * 32;
        if (s.vec != 4) return s;
        const size_t d = delta_type == 2 ? 16 : 8, y = normed_type == 2 ? 16 : 8;
        const size_t row = (size_t)s.nv * s.threads * (backward ? 32 + d + y : 16 + d) + (backward ? (size_t)s.threads * 8 : 0);
        s.depth = backward ? SW_BWD_DEPTH : SW_FWD_DEPTH;
        while (s.depth > 0 && s.depth * row > room) --s.depth;
        s.smem = s.depth * row;
        if (s.depth > 0) return s;
        s.vec = 1;
        s.smem = 0;
    }
}

// CTAs that an SM holds, by registers and the rings.
static long long sandwich_resident(const SandwichShape& s, bool backward) {
    long long n = backward ? (s.threads <= SW_FEW_BWD ? SW_FEW_BWD / s.threads : 1) : (s.threads <= SW_FEW_FWD ? 768 : 1024) / s.threads;
    if (s.smem > 0 && (long long)((227 << 10) / (s.smem + 2048)) < n) n = (long long)((227 << 10) / (s.smem + 2048));
    return n < 1 ? 1 : n > 16 ? 16 : n;
}

// Backward: CTAs, and how the rows of a gate row are shared among them.
static void sandwich_plan(SandwichArgs& a, const SandwichShape& s) {
    a.groups = a.gates > 0 ? a.gates : 1;
    a.group_rows = a.rows / a.groups;
    const long long target = a.sm_count * sandwich_resident(s, true);
    long long shares = target / a.groups;
    if (shares > a.group_rows) shares = a.group_rows;
    if (shares < 1) shares = 1;
    a.share_rows = (a.group_rows + shares - 1) / shares;
    a.shares = (a.group_rows + a.share_rows - 1) / a.share_rows;
    a.units = a.groups * a.shares;
    a.grid = a.units < target ? a.units : target;
}

long long sandwich_workspace_floats(long long rows, int hidden, long long gates, int sm_count) {
    long long most = 0;
    const bool few = rows <= 2 * sm_count;
    for (int k = 0; k < 8; ++k) {   // (alignment and types are not known yet)
        SandwichArgs a = {};
        a.rows = rows; a.hidden = hidden; a.gates = gates; a.sm_count = sm_count;
        a.delta_type = k & 2; a.normed_type = k & 4 ? 2 : 0;
        sandwich_plan(a, sandwich_shape(hidden, (k & 1) != 0, few, true, a.delta_type, a.normed_type));
        const long long planes = 2 * a.grid + (a.gates > 0 && a.shares > 1 ? a.units : 0);
        if (planes > most) most = planes;
    }
    return most * hidden;
}

template <int NV, int VEC, typename TD, typename TY>
static cudaError_t sandwich_with(const SandwichArgs& a, const SandwichShape& s, bool backward, unsigned grid, cudaStream_t stream) {
    auto kernel = backward ? (s.threads > SW_FEW_BWD ? sandwich_bwd_kernel<NV, VEC, TD, TY, 1024> : sandwich_bwd_kernel<NV, VEC, TD, TY, SW_FEW_BWD>)
                           : (s.threads > SW_FEW_FWD ? sandwich_fwd_kernel<NV, VEC, TD, TY, 1024> : sandwich_fwd_kernel<NV, VEC, TD, TY, SW_FEW_FWD>);
    if (s.smem > (40 << 10)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)s.smem);
        if (e != cudaSuccess) return e;
    }
    return launch_pdl(kernel, dim3(grid), dim3((unsigned)s.threads), s.smem, stream, a);
}

template <typename TD, typename TY>
static cudaError_t sandwich_as(const SandwichArgs& a, const SandwichShape& s, bool backward, unsigned grid, cudaStream_t stream) {
    if (s.vec == 4) {
        if (s.nv == 1) return sandwich_with<1, 4, TD, TY>(a, s, backward, grid, stream);
        if (s.nv == 2) return sandwich_with<2, 4, TD, TY>(a, s, backward, grid, stream);
        return sandwich_with<4, 4, TD, TY>(a, s, backward, grid, stream);
    }
    if (s.nv == 4) return sandwich_with<4, 1, TD, TY>(a, s, backward, grid, stream);
    return sandwich_with<16, 1, TD, TY>(a, s, backward, grid, stream);
}

cudaError_t launch_sandwich(const SandwichArgs& a_in, bool backward, cudaStream_t stream) {
    SandwichArgs a = a_in;
    if (a.rows <= 0) return cudaSuccess;
    uintptr_t bits = 0;
    for (const void* p : {(const void*)a.residual, a.delta, (const void*)a.post, (const void*)a.pre, (const void*)a.gate,
                          (const void*)a.stream, (const void*)a.normed, (const void*)a.d_stream, a.d_normed,
                          (const void*)a.d_residual, (const void*)a.d_delta, (const void*)a.d_post, (const void*)a.d_pre,
                          (const void*)a.d_gate, (const void*)a.planes_post})
        bits |= reinterpret_cast<uintptr_t>(p);
    const SandwichShape s = sandwich_shape(a.hidden, (bits & 15) == 0, a.rows <= 2 * a.sm_count, backward, a.delta_type, a.normed_type);
    a.depth = s.depth;
    sandwich_plan(a, s);
    unsigned grid;
    if (backward) {
        a.planes_pre = a.planes_post + a.grid * a.hidden;
        a.planes_gate = a.planes_pre + a.grid * a.hidden;
        grid = (unsigned)a.grid;
    } else {
        const long long target = a.sm_count * sandwich_resident(s, false);
        grid = (unsigned)(a.rows < target ? a.rows : target);
    }
    cudaError_t e;
    if (a.delta_type == 0)
        e = a.normed_type == 2 ? sandwich_as<__half, float>(a, s, backward, grid, stream)
                               : sandwich_as<__half, __half>(a, s, backward, grid, stream);
    else if (a.delta_type == 1)
        e = a.normed_type == 2 ? sandwich_as<__nv_bfloat16, float>(a, s, backward, grid, stream)
                               : sandwich_as<__nv_bfloat16, __nv_bfloat16>(a, s, backward, grid, stream);
    else
        e = sandwich_as<float, float>(a, s, backward, grid, stream);
    if (e != cudaSuccess || !backward) return e;
    const bool gate_planes = a.d_gate != nullptr && a.shares > 1;
    if (a.d_post == nullptr && a.d_pre == nullptr && !gate_planes) return e;
    long long jobs = 2 + (a.shares > 1 ? a.groups : 0);
    if (jobs > 4096) jobs = 4096;
    return launch_pdl(sandwich_sum_kernel, dim3((unsigned)((a.hidden + 31) / 32), (unsigned)jobs), dim3(32, 32), 0, stream, a);
}

}  // namespace nf4
