// Rows of 16-bit values as 8-bit integers and a scale per row:  s = max|x| / 127,  q = round-half-even(x * 127 / max|x|).
//
// q is the exactly rounded quotient.  With m = max|x|, x' = 127 x (at most 18 significant bits, exact in fp32) and m (11
// bits), a quotient in [2^k, 2^(k+1)) that is no half differs from every half by at least 2^(k-19): in units of the last
// bit of x' it is |2 x' - (2n+1) m| / 2m >= 1 / 2m, and m < 2^(18-k) such units.  The quotient is computed as
//     h = x' r,   h + (x' - h m) r        with r = fl(1 / m), two fused multiply-adds,
// whose error is far below that, and a quotient that IS a half comes out exactly (the remainder x' - h m is exact, its
// product with r is off by less than half a unit of the result's last bit).  Three operations in place of a division.
//
// Bound by memory: 2 bytes read and 1 written per value.
#include "../../include/kdw.h"
#include "linear_core.cuh"
#include "linear_plan.h"

namespace kdw {

constexpr int kQuantKeep = 4;  // vectors of 8 values that a thread keeps in registers between the two passes

__device__ __forceinline__ float half_bits_to_float(uint32_t b, bool bf16) {
    return bf16 ? __uint_as_float(b << 16) : __half2float(__ushort_as_half((unsigned short)b));
}

template <bool VEC>
__device__ __forceinline__ uint4 load8(const uint16_t* row, int c, int cols) {
    if (VEC) return *reinterpret_cast<const uint4*>(row + c);  // cols is a multiple of 8
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? row[c + j] : 0;
    return make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
}

// The row's maximum as bits: magnitudes of 16-bit floats order like integers, infinities above all numbers, NaN above.
__device__ __forceinline__ uint32_t max_bits(uint4 v, uint32_t m) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t lo = w[j] & 0x7fff, hi = (w[j] >> 16) & 0x7fff;
        m = lo > m ? lo : m;
        m = hi > m ? hi : m;
    }
    return m;
}

// How a row is quantised, from the bits of its maximum.
struct QuantRow {
    float scale;     // max / 127; NaN where the row holds a NaN or an infinity
    float pre;       // a power of two that keeps the products inside the range of fp32
    float m, r;      // maximum and reciprocal after `pre`; 0 and 0 for rows of zeros and rows with a NaN or an infinity
};
__device__ __forceinline__ QuantRow quant_row(uint32_t bits, bool bf16) {
    QuantRow q;
    const uint32_t inf = bf16 ? 0x7f80u : 0x7c00u;
    const float m = half_bits_to_float(bits, bf16);
    q.pre = m > 1.8446744073709552e19f ? 5.4210108624275222e-20f : m < 5.4210108624275222e-20f ? 1.8446744073709552e19f : 1.f;
    const bool fine = bits > 0 && bits < inf;
    q.scale = bits >= inf ? __uint_as_float(0x7fffffffu) : __fdiv_rn(m, 127.f);
    q.m = fine ? m * q.pre : 0.f;
    q.r = fine ? __frcp_rn(q.m) : 0.f;
    return q;
}
__device__ __forceinline__ uint32_t quant_one(uint32_t bits, const QuantRow& q, bool bf16) {
    const float x = half_bits_to_float(bits, bf16) * q.pre * 127.f;
    const float h = x * q.r;
    const float v = fmaf(fmaf(-h, q.m, x), q.r, h);
    return q.r == 0.f ? 0u : (uint32_t)__float2int_rn(v) & 255u;
}
__device__ __forceinline__ uint2 quant8(uint4 v, const QuantRow& q, bool bf16) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t o[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
        o[j] = quant_one(w[2 * j] & 0xffff, q, bf16) | quant_one(w[2 * j] >> 16, q, bf16) << 8 |
               quant_one(w[2 * j + 1] & 0xffff, q, bf16) << 16 | quant_one(w[2 * j + 1] >> 16, q, bf16) << 24;
    return make_uint2(o[0], o[1]);
}

// TPR threads to a row (a warp or the CTA).  VEC: rows of the input are 16-byte aligned, QVEC: rows of the output 8-byte.
template <int TPR, bool VEC, bool QVEC>
__global__ __launch_bounds__(256) void quant_rows_kernel(const uint16_t* __restrict__ x, int8_t* __restrict__ q,
                                                         float* __restrict__ scale, long long rows, int cols,
                                                         long long x_stride, long long q_stride, int bf16) {
    __shared__ uint32_t s_max[8];
    constexpr int RPB = 256 / TPR;
    const int sub = threadIdx.x / TPR, t = threadIdx.x % TPR;
    grid_dependency_wait();
    for (long long r0 = (long long)blockIdx.x * RPB; r0 < rows; r0 += (long long)gridDim.x * RPB) {
        const long long r = r0 + sub;
        const bool live = r < rows;
        const uint16_t* row = x + (live ? r : 0) * x_stride;
        uint4 keep[kQuantKeep];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < kQuantKeep; ++i) {
            const int c = (i * TPR + t) * 8;
            keep[i] = live && c < cols ? load8<VEC>(row, c, cols) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < kQuantKeep; ++i) m = max_bits(keep[i], m);
        for (int c = (kQuantKeep * TPR + t) * 8; live && c < cols; c += TPR * 8) m = max_bits(load8<VEC>(row, c, cols), m);
        m = __reduce_max_sync(0xffffffffu, m);
        if (TPR > 32) {
            __syncthreads();
            if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
            __syncthreads();
            for (int i = 0; i < 8; ++i) m = s_max[i] > m ? s_max[i] : m;
        }
        if (!live) continue;
        const QuantRow qr = quant_row(m, bf16);
        if (t == 0) scale[r] = qr.scale;
        int8_t* out = q + r * q_stride;
        auto put = [&](int c, uint4 v) {
            const uint2 o = quant8(v, qr, bf16);
            if (QVEC) {
                *reinterpret_cast<uint2*>(out + c) = o;
            } else {
                const uint32_t w[2] = {o.x, o.y};
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (c + j < cols) out[c + j] = (int8_t)(w[j >> 2] >> (8 * (j & 3)));
            }
        };
#pragma unroll
        for (int i = 0; i < kQuantKeep; ++i) {
            const int c = (i * TPR + t) * 8;
            if (c < cols) put(c, keep[i]);
        }
        for (int c = (kQuantKeep * TPR + t) * 8; c < cols; c += TPR * 8) put(c, load8<VEC>(row, c, cols));
    }
}

template <int TPR>
static int quant_launch(const void* x, void* q, float* scale, int64_t rows, int64_t cols, int64_t x_stride, int64_t q_stride,
                        int bf16, bool vec, bool qvec, cudaStream_t st) {
    int sms = 0;
    int rc = device_sm_count(&sms);
    if (rc) return rc;
    const int64_t blocks = (rows + 256 / TPR - 1) / (256 / TPR);
    const unsigned grid = (unsigned)(blocks < 8 * sms ? blocks : 8 * sms);
    auto* k = vec ? (qvec ? quant_rows_kernel<TPR, true, true> : quant_rows_kernel<TPR, true, false>)
                  : (qvec ? quant_rows_kernel<TPR, false, true> : quant_rows_kernel<TPR, false, false>);
    KDW_CUDA(launch_overlapping_previous(k, grid, 256u, st, (const uint16_t*)x, (int8_t*)q, scale, (long long)rows, (int)cols,
                                         (long long)x_stride, (long long)q_stride, bf16));
    return 0;
}

int quant_rows(const void* x, void* q, float* scale, int64_t rows, int64_t cols, int64_t x_stride, int64_t q_stride, int bf16,
               bool q_padded, cudaStream_t st) {
    const bool vec = ((uintptr_t)x & 15) == 0 && x_stride % 8 == 0 && cols % 8 == 0;
    // a last piece may run into the padding of its row, but not into the next row
    const bool qvec = ((uintptr_t)q & 7) == 0 && q_stride % 8 == 0 && (cols % 8 == 0 || q_padded);
    // a warp keeps 1024 values in registers, the CTA 8192
    return cols <= 1024 ? quant_launch<32>(x, q, scale, rows, cols, x_stride, q_stride, bf16, vec, qvec, st)
                        : quant_launch<256>(x, q, scale, rows, cols, x_stride, q_stride, bf16, vec, qvec, st);
}

}  // namespace kdw

extern "C" int kdw_quant_rows(const void* x, int8_t* q, float* scale, int64_t rows, int64_t cols, int64_t x_stride, int dtype,
                              void* stream) {
    using namespace kdw;
    if (!x || !q || !scale) {
        set_error("quant_rows: null pointer");
        return KDW_ERR_ARG;
    }
    if (rows < 1 || cols < 1 || cols > INT32_MAX - 65536 || x_stride < cols || (dtype != KDW_F16 && dtype != KDW_BF16)) {
        set_error("quant_rows: rows=%lld cols=%lld x_stride=%lld dtype=%d out of range", (long long)rows, (long long)cols,
                  (long long)x_stride, dtype);
        return KDW_ERR_ARG;
    }
    if (((uintptr_t)x & 1) || ((uintptr_t)scale & 3)) {
        set_error("quant_rows: a pointer is not aligned to its elements");
        return KDW_ERR_ALIGN;
    }
    return quant_rows(x, q, scale, rows, cols, x_stride, cols, dtype == KDW_BF16, false, (cudaStream_t)stream);
}
