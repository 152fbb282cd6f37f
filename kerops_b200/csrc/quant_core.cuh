// Rows of 16-bit values as 8-bit integers and a scale per row:  s = max|x| / 127,  q = round-half-even(x * 127 / max|x|).
//
// q is the exactly rounded quotient.  With m = max|x|, x' = 127 x (at most 18 significant bits, exact in fp32) and m (11
// bits), a quotient in [2^k, 2^(k+1)) that is no half differs from every half by at least 2^(k-19): in units of the last
// bit of x' it is |2 x' - (2n+1) m| / 2m >= 1 / 2m, and m < 2^(18-k) such units.  The quotient is computed as
//     h = x' r,   v = h + (x' - h m) r        with r = fl(1 / m), two fused multiply-adds,
// whose error is far below that, and a quotient that IS a half comes out exactly (the remainder x' - h m is exact, its
// product with r is off by less than half a unit of the result's last bit).  Adding 1.5 * 2^23 then rounds to the nearest
// integer, halves to even, and leaves it in the low byte: five operations on the fp32 pipes and none on the slower
// conversion unit.
#pragma once

#include "kdw_common.cuh"

namespace kdw {

#ifdef __CUDACC__

__device__ __forceinline__ float half_bits_to_float(uint32_t b, bool bf16) {
    return bf16 ? __uint_as_float(b << 16) : __half2float(__ushort_as_half((unsigned short)b));
}

// The row's maximum as bits: magnitudes of 16-bit floats order like integers, infinities above all numbers, NaN above.
__device__ __forceinline__ uint32_t max_bits(uint4 v, uint32_t m) {
    uint32_t a = __vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu);
    const uint32_t b = __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu);
    a = __vmaxu2(a, b);
    const uint32_t lo = a & 0xffff, hi = a >> 16;
    m = lo > m ? lo : m;
    return hi > m ? hi : m;
}

// How a row is quantised, from the bits of its maximum.
struct QuantRow {
    float scale;   // max / 127; NaN where the row holds a NaN or an infinity
    float pre;     // 127 times a power of two that keeps the products inside the range of fp32
    float m, r;    // the maximum after that power of two, and its reciprocal
    bool fine;     // false: a row of zeros, or with a NaN or an infinity; its q are 0
};
__device__ __forceinline__ QuantRow quant_row(uint32_t bits, bool bf16) {
    QuantRow q;
    const uint32_t inf = bf16 ? 0x7f80u : 0x7c00u;
    const float m = half_bits_to_float(bits, bf16);
    const float p = m > 1.8446744073709552e19f ? 5.4210108624275222e-20f : m < 5.4210108624275222e-20f ? 1.8446744073709552e19f : 1.f;
    q.fine = bits > 0 && bits < inf;
    q.scale = bits >= inf ? __uint_as_float(0x7fffffffu) : __fdiv_rn(m, 127.f);
    q.pre = 127.f * p;
    q.m = m * p;
    q.r = q.fine ? __frcp_rn(q.m) : 0.f;
    return q;
}
__device__ __forceinline__ uint32_t quant_one(uint32_t bits, const QuantRow& q, bool bf16) {
    const float x = half_bits_to_float(bits, bf16) * q.pre;
    const float h = x * q.r;
    return __float_as_uint(fmaf(fmaf(-h, q.m, x), q.r, h) + 12582912.f);  // its low byte
}
__device__ __forceinline__ uint2 quant8(uint4 v, const QuantRow& q, bool bf16) {
    if (!q.fine) return make_uint2(0, 0);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t o[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t a = __byte_perm(quant_one(w[2 * j] & 0xffff, q, bf16), quant_one(w[2 * j] >> 16, q, bf16), 0x0040);
        const uint32_t b = __byte_perm(quant_one(w[2 * j + 1] & 0xffff, q, bf16), quant_one(w[2 * j + 1] >> 16, q, bf16), 0x0040);
        o[j] = __byte_perm(a, b, 0x5410);
    }
    return make_uint2(o[0], o[1]);
}

#endif  // __CUDACC__

}  // namespace kdw
