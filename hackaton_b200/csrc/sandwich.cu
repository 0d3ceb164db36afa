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
// keeps a thread's columns of the weights in registers over all its rows. Rows to come are on their way to shared
// memory, four ahead forward and three backward, a bulk copy per array and row that one thread asks for: two or three CTAs
// of an SM with one row each in flight leave most of the bandwidth idle, and every instruction that a thread spends
// on addresses counts where it has eight values of a row. 16,384 x 1536 (302 and 453 MB): forward 51 us (6.0 TB/s),
// backward 76 (6.0 TB/s) and 4 for its sums; a row ahead in registers 82 and 129. Column sums of the weights'
// gradients stay in registers; a second kernel adds the CTAs' sums in order, so that results do not depend on timing.
// All sums are fp32.
// Beside that (16-bit delta, both ways, in brackets what the bytes alone take): 8192 x 4096 173 us (156); wider rows, whose values do not fit the
// registers backward (stack of 0.3 to 0.5 KB a thread), 8192 x 5000 467 (190), 8192 x 8192 553 (311), 4096 x 16,384 820 (311), the last
// by single values, since no row fits shared memory; widths that are no multiple of 8, by single values a row ahead in registers, 16,384 x 1537
// 242 (117). fp32 delta 16,384 x 1536 179 (156).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.h"
#include "ptx.cuh"

namespace nf4 {

// VEC values of a type as they lie in memory.
template <typename T, int VEC> struct SwRaw;

template <> struct SwRaw<float, 4> {
    float4 v;
    __device__ __forceinline__ void load(const void* p, long long i) { v = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i)); }
    __device__ __forceinline__ void get(float (&f)[4]) const { f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
    static __device__ __forceinline__ void store(void* p, long long i, const float (&f)[4]) {
        *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(f[0], f[1], f[2], f[3]);
    }
};
template <> struct SwRaw<__half, 4> {
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

// What a thread's columns take of one array's rows. VEC = 4: from a slot in shared memory, where the row lies as in memory;
// VEC = 1: through registers, one row ahead.
template <typename T, int NV, int VEC>
struct SwRow {
    SwRaw<T, VEC> next[VEC == 4 ? 1 : NV];
    __device__ __forceinline__ void ask(const T* row, const int (&cols)[NV]) {      // (VEC = 1)
        if constexpr (VEC == 1)
#pragma unroll
            for (int i = 0; i < NV; ++i) next[i].load(row, cols[i]);
    }
    __device__ __forceinline__ void get(uint32_t slot, const int (&cols)[NV], float (&f)[NV][VEC]) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (VEC == 4) {
                const uint32_t x = slot + cols[i] * (int)sizeof(T);
                SwRaw<T, 4> raw;
                if constexpr (sizeof(T) == 4)
                    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(raw.v.x), "=f"(raw.v.y), "=f"(raw.v.z), "=f"(raw.v.w) : "r"(x));
                else
                    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(raw.v.x), "=r"(raw.v.y) : "r"(x));
                raw.get(f[i]);
            } else {
                next[i].get(f[i]);
            }
        }
    }
};

// Threads up to which a kernel may take 80 registers each forward and 128 backward.
constexpr int SW_FEW_FWD = 256, SW_FEW_BWD = 512;
constexpr int SW_FWD_DEPTH = 4, SW_BWD_DEPTH = 3;      // where shared memory allows

// The slots' barriers: a slot's copies count towards its own.
struct SwBars {
    uint32_t first;
    volatile int* abort_flag;
    __device__ __forceinline__ void init(unsigned long long* room, int* flag, int depth) {
        first = smem_u32(room);
        abort_flag = flag;
        if (threadIdx.x == 0) {
            for (int k = 0; k < depth; ++k) mbar_init(first + 8 * k, 1);
            *flag = 0;
            fence_barrier_init();
        }
        __syncthreads();
    }
    __device__ __forceinline__ uint32_t operator[](int slot) const { return first + 8 * slot; }
};

// Sums of N values over the CTA, the same in every thread: a warp's by shuffles; of the warps' every fourth by each
// lane (a load that is mostly a broadcast), the four shares by shuffles again. `part` has two halves that successive calls
// take in turn: who writes a half again has passed the barrier behind which everybody had read it.
template <int N>
__device__ __forceinline__ void sw_block_sum(float (&v)[N], float4 (*part)[32], int& turn) {
    static_assert(N <= 4, "one float4 per warp");
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (warps > 1) {
        if (lane == 0) part[turn][threadIdx.x >> 5] = make_float4(v[0], N > 1 ? v[N > 1 ? 1 : 0] : 0.f, N > 2 ? v[N > 2 ? 2 : 0] : 0.f, 0.f);
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = 0.f;
        for (int w = lane & 3; w < warps; w += 4) {
            const float4 x = part[turn][w];
            v[0] += x.x;
            if (N > 1) v[N > 1 ? 1 : 0] += x.y;
            if (N > 2) v[N > 2 ? 2 : 0] += x.z;
        }
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int o = 2; o > 0; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
        turn ^= 1;
    } else {
        __syncwarp();      // (what the lanes read may be written again)
    }
}

// A thread's columns. Where a row ends before them they stand for its last ones, with weights of zero: nothing needs
// a guard but what is added up or written.
template <int NV, int VEC>
__device__ __forceinline__ void sw_columns(int hidden, int (&cols)[NV], bool (&in)[NV]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (threadIdx.x + i * blockDim.x) * VEC;
        in[i] = c < hidden;
        cols[i] = in[i] ? c : hidden - VEC;
    }
}

template <int NV, int VEC>
__device__ __forceinline__ void sw_weights(const float* p, const int (&cols)[NV], const bool (&in)[NV], float (&w)[NV][VEC]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        SwRaw<float, VEC> raw;
        raw.load(p, cols[i]);
        raw.get(w[i]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[i][e] = in[i] ? w[i][e] : 0.f;
    }
}

// Weights behind the block with their gate row.
template <int NV, int VEC>
__device__ __forceinline__ void sw_gated(const SandwichArgs& a, long long gate_row, const int (&cols)[NV], const bool (&in)[NV],
                                         float (&w)[NV][VEC]) {
    sw_weights<NV, VEC>(a.post, cols, in, w);
    if (a.gates == 0) return;
    float gate[NV][VEC];
    sw_weights<NV, VEC>(a.gate + gate_row * a.hidden, cols, in, gate);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[i][e] *= gate[i][e];
}

// A CTA's rows: units (gate row, share) blockIdx.x, + gridDim.x, ...; of a gate row's rows a share is every shares-th, so
// that what the CTAs read at a time lies together (shares of consecutive rows: 16,384 x 1536 forward 55 us, so 51).
struct SwWalk {
    int unit, row, end;      // row -1 behind the last one
    __device__ __forceinline__ void enter(const SandwichArgs& a) {
        if (unit >= (int)a.units) {
            row = -1;
            return;
        }
        const int group = unit / (int)a.shares;
        row = group * (int)a.group_rows + unit - group * (int)a.shares;
        end = (group + 1) * (int)a.group_rows;
    }
    __device__ __forceinline__ void step(const SandwichArgs& a) {
        if (row < 0) return;
        row += (int)a.shares;
        if (row < end) return;
        unit += gridDim.x;
        enter(a);
    }
};

template <int NV, int VEC, typename TD, typename TY, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT <= SW_FEW_FWD ? 3 : 1)
sandwich_fwd_kernel(const SandwichArgs a) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ float4 part[2][32];
    __shared__ unsigned long long bar_room[4];
    __shared__ int abort_room;
    int turn = 0;
    const int hidden = a.hidden;
    const float inv_h = 1.f / (float)hidden;
    int cols[NV];
    bool in[NV];
    sw_columns<NV, VEC>(hidden, cols, in);
    float post[NV][VEC], pre[NV][VEC];      // post: times the gate
    sw_weights<NV, VEC>(a.pre, cols, in, pre);
    const int depth = VEC == 4 ? a.depth : 1;
    extern __shared__ uint4 sw_smem[];
    const uint32_t room = smem_u32(sw_smem), bytes_r = hidden * 4, bytes_d = hidden * (int)sizeof(TD), slot_bytes = bytes_r + bytes_d;
    SwBars bars;
    SwRow<float, NV, VEC> in_r;
    SwRow<TD, NV, VEC> in_d;
    if (VEC == 4) bars.init(bar_room, &abort_room, depth);
    const auto fetch = [&](int r, int slot) {      // (a negative row: nothing)
        if (r < 0) return;
        const long long at = (long long)r * hidden;
        const TD* const d_row = static_cast<const TD*>(a.delta) + at;
        if (VEC == 1) {
            in_d.ask(d_row, cols);
            in_r.ask(a.residual + at, cols);
        } else if (threadIdx.x == 0) {
            const uint32_t to = room + slot * slot_bytes;
            mbar_arrive_expect_tx(bars[slot], slot_bytes);
            bulk_load(to, a.residual + at, bytes_r, bars[slot]);
            bulk_load(to + bytes_r, d_row, bytes_d, bars[slot]);
        }
    };
    SwWalk ahead = {(int)blockIdx.x, 0, 0};      // asks for rows, `depth` of them before the one that works on them
    ahead.enter(a);
    SwWalk now = ahead;
    for (int k = 0; k < depth; ++k) {
        fetch(ahead.row, k);
        ahead.step(a);
    }
    uint32_t phase = 0;
    int unit = -1;
    for (int slot = 0; now.row >= 0; now.step(a)) {
        const uint32_t from = room + slot * slot_bytes;
        const int row = now.row;
        if (VEC == 4 && !mbar_wait(bars[slot], phase, bars.abort_flag)) {
            if (threadIdx.x == 0) give_up(a.status, STATUS_ROW_WAIT);
            return;
        }
        if (now.unit != unit) {
            unit = now.unit;
            sw_gated<NV, VEC>(a, unit / (int)a.shares, cols, in, post);
        }
        float d[NV][VEC], s[NV][VEC], sum[1] = {0.f};
        in_d.get(from + bytes_r, cols, d);
        in_r.get(from, cols, s);
        if (VEC != 4) {
            fetch(ahead.row, 0);
            ahead.step(a);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (in[i])
#pragma unroll
                for (int e = 0; e < VEC; ++e) sum[0] = fmaf(d[i][e], d[i][e], sum[0]);
        sw_block_sum<1>(sum, part, turn);
        const float rd = 1.f / sqrtf(sum[0] * inv_h + a.eps);
        if (VEC == 4) {       // (behind the barrier: the slot has been read)
            fetch(ahead.row, slot);
            ahead.step(a);
            if (++slot == depth) {
                slot = 0;
                phase ^= 1u;
            }
        }
        sum[0] = 0.f;
        const long long at = (long long)row * hidden;
        float* const out = a.stream + at;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) s[i][e] = fmaf(d[i][e] * rd, post[i][e], a.scale * s[i][e]);
            if (in[i]) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) sum[0] = fmaf(s[i][e], s[i][e], sum[0]);
                SwRaw<float, VEC>::store(out, cols[i], s[i]);
            }
        }
        sw_block_sum<1>(sum, part, turn);
        const float rs = 1.f / sqrtf(sum[0] * inv_h + a.eps);
        TY* const normed = static_cast<TY*>(a.normed) + at;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float y[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) y[e] = pre[i][e] * (s[i][e] * rs);
            if (in[i]) SwRaw<TY, VEC>::store(normed, cols[i], y);
        }
        if (threadIdx.x == 0 && a.rstd != nullptr) *reinterpret_cast<float4*>(a.rstd + 4ll * row) = make_float4(rd, rs, 0.f, 0.f);
    }
}

template <int NV, int VEC, typename TD, typename TY, int MAXT>
__global__ void __launch_bounds__(MAXT, 1)
sandwich_bwd_kernel(const SandwichArgs a) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ float4 part[2][32];
    __shared__ unsigned long long bar_room[4];
    __shared__ int abort_room;
    int turn = 0;
    const int hidden = a.hidden;
    const float inv_h = 1.f / (float)hidden;
    int cols[NV];
    bool in[NV];
    sw_columns<NV, VEC>(hidden, cols, in);
    float post[NV][VEC], pre[NV][VEC], sum_post[NV][VEC], sum_pre[NV][VEC], sum_unit[NV][VEC];   // post: times the gate
    sw_weights<NV, VEC>(a.pre, cols, in, pre);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum_post[i][e] = sum_pre[i][e] = sum_unit[i][e] = 0.f;

    const int depth = VEC == 4 ? a.depth : 1;
    const bool direct = a.d_stream != nullptr;
    extern __shared__ uint4 sw_smem[];
    const uint32_t room = smem_u32(sw_smem), bytes_s = hidden * 4, bytes_t = direct ? bytes_s : 0, bytes_d = hidden * (int)sizeof(TD),
                   bytes_y = hidden * (int)sizeof(TY), at_t = bytes_s, at_d = at_t + bytes_t, at_y = at_d + bytes_d,
                   at_rstd = at_y + bytes_y, slot_bytes = at_rstd + 16;
    SwBars bars;
    SwRow<float, NV, VEC> in_s, in_t;
    SwRow<TD, NV, VEC> in_d;
    SwRow<TY, NV, VEC> in_y;
    if (VEC == 4) bars.init(bar_room, &abort_room, depth);
    float2 next_rstd = make_float2(0.f, 0.f);
    const auto fetch = [&](int row, int slot) {      // (a negative row: nothing)
        if (row < 0) return;
        const long long at = (long long)row * hidden;
        const TD* const d_row = static_cast<const TD*>(a.delta) + at;
        const TY* const y_row = static_cast<const TY*>(a.d_normed) + at;
        if (VEC == 1) {
            in_s.ask(a.stream + at, cols);
            in_d.ask(d_row, cols);
            in_y.ask(y_row, cols);
            if (direct) in_t.ask(a.d_stream + at, cols);
            next_rstd = *reinterpret_cast<const float2*>(a.rstd + 4ll * row);
        } else if (threadIdx.x == 0) {
            const uint32_t to = room + slot * slot_bytes, bar = bars[slot];
            mbar_arrive_expect_tx(bar, slot_bytes);
            bulk_load(to, a.stream + at, bytes_s, bar);
            if (direct) bulk_load(to + at_t, a.d_stream + at, bytes_t, bar);
            bulk_load(to + at_d, d_row, bytes_d, bar);
            bulk_load(to + at_y, y_row, bytes_y, bar);
            bulk_load(to + at_rstd, a.rstd + 4ll * row, 16, bar);
        }
    };
    const int shares = (int)a.shares;
    SwWalk ahead = {(int)blockIdx.x, 0, 0};      // as in the forward   (gridDim.x <= units)
    ahead.enter(a);
    SwWalk now = ahead;
    for (int k = 0; k < depth; ++k) {
        fetch(ahead.row, k);
        ahead.step(a);
    }
    bool new_unit = true;
    uint32_t phase = 0;
    for (int slot = 0; now.row >= 0;) {
        const uint32_t from = room + slot * slot_bytes;
        if (VEC == 4 && !mbar_wait(bars[slot], phase, bars.abort_flag)) {
            if (threadIdx.x == 0) give_up(a.status, STATUS_ROW_WAIT);
            return;
        }
        if (new_unit) sw_gated<NV, VEC>(a, now.unit / shares, cols, in, post);
        float2 rstd = next_rstd;
        if (VEC == 4) asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(rstd.x), "=f"(rstd.y) : "r"(from + at_rstd));
        const float rd = rstd.x, rs = rstd.y;
        float s[NV][VEC], t[NV][VEC], d[NV][VEC], y[NV][VEC], sum[3] = {0.f, 0.f, 0.f};
        in_s.get(from, cols, s);
        in_d.get(from + at_d, cols, d);
        in_y.get(from + at_y, cols, y);
        if (direct) {
            in_t.get(from + at_t, cols, t);
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) t[i][e] = 0.f;
        }
        const long long at = (long long)now.row * hidden;
        const int this_unit = now.unit;
        now.step(a);
        const bool unit_done = now.row < 0 || now.unit != this_unit;
        new_unit = unit_done;
        if (VEC != 4) {
            fetch(ahead.row, 0);
            ahead.step(a);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                s[i][e] *= rs;                                      // sh
                d[i][e] *= rd;                                      // dh
                const float w = y[i][e] * pre[i][e], gd = post[i][e] * d[i][e];      // (both zero behind the row)
                t[i][e] = fmaf(rs, w, t[i][e]);                     // ds but for the mean
                sum[0] = fmaf(w, s[i][e], sum[0]);
                sum[1] = fmaf(gd, t[i][e], sum[1]);
                sum[2] = fmaf(gd, s[i][e], sum[2]);
                sum_pre[i][e] = fmaf(y[i][e], s[i][e], sum_pre[i][e]);
            }
        sw_block_sum<3>(sum, part, turn);
        if (VEC == 4) {       // (behind the barrier: the slot has been read)
            fetch(ahead.row, slot);
            ahead.step(a);
            if (++slot == depth) {
                slot = 0;
                phase ^= 1u;
            }
        }
        const float m1 = rs * (sum[0] * inv_h);
        const float m2 = (sum[1] - m1 * sum[2]) * inv_h, rd_m2 = rd * m2;
        float* const d_residual = a.d_residual + at;
        TD* const d_delta = static_cast<TD*>(a.d_delta) + at;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float dr[VEC], dd[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float ds = fmaf(-m1, s[i][e], t[i][e]);
                dr[e] = a.scale * ds;
                dd[e] = rd * (ds * post[i][e]) - d[i][e] * rd_m2;
                sum_unit[i][e] = fmaf(ds, d[i][e], sum_unit[i][e]);
            }
            if (in[i]) {
                if (a.d_residual != nullptr) SwRaw<float, VEC>::store(d_residual, cols[i], dr);
                if (a.d_delta != nullptr) SwRaw<TD, VEC>::store(d_delta, cols[i], dd);
            }
        }
        if (unit_done) {
            float own[NV][VEC], gate[NV][VEC];
            sw_weights<NV, VEC>(a.post, cols, in, own);
            if (a.gates > 0) sw_weights<NV, VEC>(a.gate + (long long)(this_unit / shares) * hidden, cols, in, gate);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float dg[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    dg[e] = own[i][e] * sum_unit[i][e];
                    sum_post[i][e] = fmaf(a.gates > 0 ? gate[i][e] : 1.f, sum_unit[i][e], sum_post[i][e]);
                    sum_unit[i][e] = 0.f;
                }
                // (one share per gate row: the row itself; otherwise the shares' plane)
                if (a.d_gate != nullptr && in[i])
                    SwRaw<float, VEC>::store(shares == 1 ? a.d_gate : a.planes_gate, (long long)this_unit * hidden + cols[i], dg);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (!in[i]) continue;
        const long long at = (long long)blockIdx.x * hidden + cols[i];
        if (a.d_post != nullptr) SwRaw<float, VEC>::store(a.planes_post, at, sum_post[i]);
        if (a.d_pre != nullptr) SwRaw<float, VEC>::store(a.planes_pre, at, sum_pre[i]);
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
// shuffles and more: 16,384 x 1536 with one float4 74 and 97 us, so 51 and 76), as many as registers hold backward; one where there
// are few rows and latency counts; single values for rows that are no whole float4, not aligned, or too long for one of
// them in shared memory.
static SandwichShape sandwich_shape(int hidden, bool vec, bool few, bool backward, int delta_type, int normed_type) {
    const size_t room = (227 << 10) - 2048;
    SandwichShape s = {};
    s.vec = vec && hidden % (delta_type == 2 && normed_type == 2 ? 4 : 8) == 0 ? 4 : 1;     // (rows of whole 16 bytes)
    for (;;) {
        const int items = (hidden + s.vec - 1) / s.vec;
        if (s.vec == 4) s.nv = items <= (few ? 1024 : backward ? 192 : 256) ? 1 : items <= (few ? 2048 : backward ? 1024 : 512) ? 2 : 4;
        else            s.nv = items <= 4096 ? 4 : 16;
        s.threads = ((items + s.nv - 1) / s.nv + 31) / 32 * 32;
        if (s.vec != 4) return s;
        const size_t d = delta_type == 2 ? 4 : 2, y = normed_type == 2 ? 4 : 2;
        const size_t row = backward ? (size_t)hidden * (8 + d + y) + 16 : (size_t)hidden * (4 + d);
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

// CTAs, and how the rows of a gate row are shared among them.
static void sandwich_plan(SandwichArgs& a, const SandwichShape& s, bool backward) {
    a.groups = a.gates > 0 ? a.gates : 1;
    a.group_rows = a.rows / a.groups;
    const long long target = a.sm_count * sandwich_resident(s, backward);
    long long shares = target / a.groups;
    if (shares > a.group_rows) shares = a.group_rows;
    a.shares = shares < 1 ? 1 : shares;
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
        sandwich_plan(a, sandwich_shape(hidden, (k & 1) != 0, few, true, a.delta_type, a.normed_type), true);
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
                          (const void*)a.d_gate, (const void*)a.planes_post, (const void*)a.rstd})
        bits |= reinterpret_cast<uintptr_t>(p);
    const SandwichShape s = sandwich_shape(a.hidden, (bits & 15) == 0, a.rows <= 2 * a.sm_count, backward, a.delta_type, a.normed_type);
    a.depth = s.depth;
    sandwich_plan(a, s, backward);
    const unsigned grid = (unsigned)a.grid;
    if (backward) {
        a.planes_pre = a.planes_post + a.grid * a.hidden;
        a.planes_gate = a.planes_pre + a.grid * a.hidden;
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
