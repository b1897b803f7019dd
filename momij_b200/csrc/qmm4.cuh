// qmm4.cuh -- what the two kernels of the 4-bit product share: its arguments, and
// x as both see it.
#pragma once

#include "host.cuh"
#include "pack.cuh"

namespace momij {

struct Qmm4Call {
    const uint16_t* x;
    const uint32_t* w;
    const uint16_t* s;
    const uint16_t* b;
    uint16_t* y;
    long long ldx, ldy;
    int M, N, K, gs, dtype;
};

// Two results rounded to the activations' type, in one word.
template <int DT>
__device__ __forceinline__ uint32_t rounded2(float lo, float hi) {
    if (DT == MOMIJ_DTYPE_F16) return f16x2(lo, hi);
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// The two 16-bit values of a word as floats.
template <int DT>
__device__ __forceinline__ float half_of(uint32_t w, int hi) {
    if (DT == MOMIJ_DTYPE_BF16) return __uint_as_float(hi ? w & 0xffff0000u : w << 16);
    return Half<DT>::to_f((uint16_t)(hi ? w >> 16 : w & 0xffffu));
}
// Eight elements of x from device memory, aligned to 16 bytes (vec) or not.
__device__ __forceinline__ uint4 qmm4_piece(const uint16_t* src, bool vec) {
    if (vec) return __ldg(reinterpret_cast<const uint4*>(src));
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __ldg(src + 2 * i) | ((uint32_t)__ldg(src + 2 * i + 1) << 16);
    return make_uint4(v[0], v[1], v[2], v[3]);
}
// The largest magnitude's bits among eight elements (so that NaN counts as the largest).
__device__ __forceinline__ uint32_t qmm4_top(const uint4& v) {
    const uint32_t t[4] = {v.x, v.y, v.z, v.w};
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, max(t[i] & 0x7fffu, (t[i] >> 16) & 0x7fffu));
    return top;
}
// A token's biased exponent, from which x is scaled so that its largest magnitude
// becomes 2^14 .. 2^15; 141 (a factor of one) for zeros, infinities and NaN.
// Tokens below 2^-112 stay smaller.
template <int DT>
__device__ __forceinline__ int qmm4_exponent(uint32_t top) {
    const uint32_t u = __float_as_uint(Half<DT>::to_f((uint16_t)top));
    return u == 0 || u >= 0x7f800000u ? 141 : max((int)(u >> 23), 15);
}
// Eight elements as the operand's 16 bytes: scaled by f, in the order in which a
// word's codes come apart (elements 0 and 4; 1 and 5 sixteen times smaller; 2 and 6;
// 3 and 7 likewise); and their sum.
template <int DT>
__device__ __forceinline__ uint4 qmm4_operand(const uint4& v, float f, float& sum) {
    const uint32_t t[4] = {v.x, v.y, v.z, v.w};
    float e[8];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        e[2 * q] = half_of<DT>(t[q], 0) * f;
        e[2 * q + 1] = half_of<DT>(t[q], 1) * f;
    }
    sum = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) sum += e[q];
    return make_uint4(f16x2(e[0], e[4]), f16x2(e[1] * 0.0625f, e[5] * 0.0625f), f16x2(e[2], e[6]), f16x2(e[3] * 0.0625f, e[7] * 0.0625f));
}
constexpr float kQmm4Unit = 5.9604644775390625e-08f;  // 2^-24, the unit of the codes' products

// qmm4_tc.cu: whether it takes these arguments, and the call itself.
bool qmm4_tc_takes(const Qmm4Call& c);
int qmm4_tc_launch(const Qmm4Call& c, momij_stream_t st);

}  // namespace momij
