// Activations in 8 bits: 32 consecutive values of a row share one power of two as their step.
//   step 2^e with e = floor(log2 max|x|) - 6, at least -126 (a normal fp32 number)
//   code q = rint(x / 2^e) held within -127 .. 127, value q * 2^e
// (the MXINT8 form of the OCP microscaling formats, with the step's exponent moved by the elements' six
// fraction bits). Every operation but the rounding to a whole number is exact, so that the values are the
// same whichever precision they are computed in, and q * 2^e is exact in the source's type. The largest value of
// a block lies between 64 and 128 steps: the error of a value is at most half a step (a whole one above
// 127.5 steps), 2^-7 of the block's largest. A block with an infinity or a NaN is held as NaN as a whole.
// Layout: codes int8 [rows, blocks * 32] (the last block of a row filled up with zeros), steps uint8
// [rows, blocks] = e + 127, 255 for a block of NaN.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace nf4 {

constexpr int A8_BLOCK = 32;

// Magnitudes are compared as their bits: a NaN is then larger than an infinity, and neither gets lost.
template <typename T> struct A8Source;

template <> struct A8Source<float> {
    static constexpr uint32_t INF_BITS = 0x7F800000u;
    static __device__ __forceinline__ float load(const void* p, long long i) { return static_cast<const float*>(p)[i]; }
    static __device__ __forceinline__ void store(void* p, long long i, float v) { static_cast<float*>(p)[i] = v; }
};
template <> struct A8Source<__half> {
    static __device__ __forceinline__ float load(const void* p, long long i) {
        return __half2float(static_cast<const __half*>(p)[i]);
    }
    static __device__ __forceinline__ void store(void* p, long long i, float v) {
        static_cast<__half*>(p)[i] = __float2half_rn(v);
    }
    static __device__ __forceinline__ float2 two(uint32_t w) {
        return __half22float2(*reinterpret_cast<const __half2*>(&w));
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <> struct A8Source<__nv_bfloat16> {
    static __device__ __forceinline__ float load(const void* p, long long i) {
        return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    }
    static __device__ __forceinline__ void store(void* p, long long i, float v) {
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    }
    static __device__ __forceinline__ float2 two(uint32_t w) {
        return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};

__device__ __forceinline__ uint32_t a8_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// Step byte of a block whose largest magnitude has these fp32 bits, and 1 / step.
__device__ __forceinline__ uint32_t a8_step(uint32_t top_bits) {
    const int field = (int)(top_bits >> 23);                    // exponent + 127
    return field == 255 ? 255u : (uint32_t)max(field - 6, 1);
}
__device__ __forceinline__ float a8_inverse(uint32_t step) {    // (255: any finite number)
    return __uint_as_float((254u - min(step, 253u)) << 23);
}
__device__ __forceinline__ float a8_value_of_step(uint32_t step) {
    return __uint_as_float(step == 255u ? 0x7FFFFFFFu : step << 23);
}

// The code of x, in the low byte. x / step is exact and below 128 in magnitude; adding 1.5 * 2^23 rounds it to
// a whole number, ties to even, whose low byte stands in the low byte of the sum. (fminf and fmaxf drop a NaN; its
// block is marked in the step.)
__device__ __forceinline__ uint32_t a8_code(float x, float inverse) {
    const float magic = 12582912.f;
    const float r = fmaf(x, inverse, magic);
    return __float_as_uint(fmaxf(fminf(r, magic + 127.f), magic - 127.f));
}

__device__ __forceinline__ uint32_t a8_code4(float a, float b, float c, float d, float inverse) {
    const uint32_t lo = __byte_perm(a8_code(a, inverse), a8_code(b, inverse), 0x0040);
    const uint32_t hi = __byte_perm(a8_code(c, inverse), a8_code(d, inverse), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
}

// Four values from four codes: a byte with its sign bit flipped, put under the exponent of 2^23, is 2^23 + 128 + q.
__device__ __forceinline__ void a8_values4(uint32_t codes, float step, float (&v)[4]) {
    const uint32_t u = codes ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = (__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 + i)) - 8388736.f) * step;
}

}  // namespace nf4
