// Quantises rows of 16-bit values (the arithmetic: quant_core.cuh).  Bound by memory: 2 bytes read and 1 written per value.
#include <type_traits>

#include "../../include/kdw.h"
#include "linear_core.cuh"
#include "linear_plan.h"
#include "quant_core.cuh"

namespace kdw {

template <bool VEC>
__device__ __forceinline__ uint4 load8(const uint16_t* row, int c, int cols) {
    if (VEC) return __ldg(reinterpret_cast<const uint4*>(row + c));  // cols is a multiple of 8
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? __ldg(row + c + j) : 0;
    return make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
}

// TPR threads to a row (a part of a warp, a warp or the CTA), KEEP vectors of 8 values of a thread stay in registers between
// the two passes over the row; what is longer is read again.  CTAs from `ctas` on copy weights instead.  VEC: rows of the
// input are 16-byte aligned, QVEC: rows of the output 8-byte.
template <int TPR, int KEEP, bool VEC, bool QVEC, int THREADS>
__global__ __launch_bounds__(THREADS) void quant_rows_kernel(const uint16_t* __restrict__ x, int8_t* __restrict__ q,
                                                         float* __restrict__ scale, long long rows, int cols,
                                                         long long x_stride, long long q_stride, int bf16,
                                                         const __grid_constant__ PackRows pack, int ctas) {
    __shared__ uint32_t s_max[8];
    constexpr int RPB = THREADS / TPR;
    const int sub = threadIdx.x / TPR, t = threadIdx.x % TPR;
    grid_dependency_wait();
    grid_launch_dependents();
    if ((int)blockIdx.x >= ctas) {
        pack_rows_part<uint8_t>(pack, blockIdx.x - ctas, gridDim.x - ctas, THREADS);
        return;
    }
    for (long long r0 = (long long)blockIdx.x * RPB; r0 < rows; r0 += (long long)ctas * RPB) {
        const long long r = r0 + sub;
        const bool live = r < rows;
        const uint16_t* row = x + (live ? r : 0) * x_stride;
        uint4 keep[KEEP];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < KEEP; ++i) {
            const int c = (i * TPR + t) * 8;
            keep[i] = live && c < cols ? load8<VEC>(row, c, cols) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < KEEP; ++i) m = max_bits(keep[i], m);
        for (int c = (KEEP * TPR + t) * 8; live && c < cols; c += TPR * 8) m = max_bits(load8<VEC>(row, c, cols), m);
        if constexpr (TPR >= 32) {
            m = __reduce_max_sync(0xffffffffu, m);
        } else {
#pragma unroll
            for (int d = TPR / 2; d; d /= 2) {
                const uint32_t o = __shfl_xor_sync(0xffffffffu, m, d);
                m = o > m ? o : m;
            }
        }
        if (TPR > 32) {
            __syncthreads();
            if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
            __syncthreads();
            for (int i = 0; i < THREADS / 32; ++i) m = s_max[i] > m ? s_max[i] : m;
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
        for (int i = 0; i < KEEP; ++i) {
            const int c = (i * TPR + t) * 8;
            if (c < cols) put(c, keep[i]);
        }
        for (int c = (KEEP * TPR + t) * 8; c < cols; c += TPR * 8) put(c, load8<VEC>(row, c, cols));
    }
}

// IN: 0 rows of any alignment, 1 only aligned ones, 2 only others.
template <int TPR, int KEEP, int THREADS, int IN>
static int quant_launch(const void* x, void* q, float* scale, int64_t rows, int64_t cols, int64_t x_stride, int64_t q_stride,
                        int bf16, bool vec, bool qvec, const PackRows* pack, cudaStream_t st) {
    int sms = 0;
    int rc = device_facts(nullptr, &sms);
    if (rc) return rc;
    const int64_t blocks = (rows + THREADS / TPR - 1) / (THREADS / TPR);
    const int grid = (int)(blocks < 2048 / THREADS * sms ? blocks : 2048 / THREADS * sms);
    const int more = pack ? pack_ctas(*pack, 1, sms) * (256 / THREADS) : 0;
    constexpr bool V = IN != 2, S = IN == 1;  // what the two choices below stand for, where one of them is not made
    auto* k = vec ? (qvec ? quant_rows_kernel<TPR, KEEP, V, true, THREADS> : quant_rows_kernel<TPR, KEEP, V, false, THREADS>)
                  : (qvec ? quant_rows_kernel<TPR, KEEP, S, true, THREADS> : quant_rows_kernel<TPR, KEEP, S, false, THREADS>);
    KDW_CUDA(launch_overlapping_previous(k, (unsigned)(grid + more), (unsigned)THREADS, st, (const uint16_t*)x, (int8_t*)q, scale, (long long)rows, (int)cols,
                                         (long long)x_stride, (long long)q_stride, bf16, pack ? *pack : PackRows{}, grid));
    return 0;
}

int quant_rows(const void* x, void* q, float* scale, int64_t rows, int64_t cols, int64_t x_stride, int64_t q_stride, int bf16,
               bool q_padded, const PackRows* pack, cudaStream_t st) {
    const bool vec = ((uintptr_t)x & 15) == 0 && x_stride % 8 == 0 && cols % 8 == 0;
    // a last piece may run into the padding of its row, but not into the next row
    const bool qvec = ((uintptr_t)q & 7) == 0 && q_stride % 8 == 0 && (cols % 8 == 0 || q_padded);
    int sms = 0;
    int rc = device_facts(nullptr, &sms);
    if (rc) return rc;
    auto go = [&](auto tpr, auto keep, auto threads, auto in) {
        return quant_launch<decltype(tpr)::value, decltype(keep)::value, decltype(threads)::value, decltype(in)::value>(
            x, q, scale, rows, cols, x_stride, q_stride, bf16, vec, qvec, pack, st);
    };
    using std::integral_constant;
    const integral_constant<int, 0> any;
    const integral_constant<int, 1> k1, aligned;
    const integral_constant<int, 2> k2, unaligned;
    const integral_constant<int, 4> k4;
    const integral_constant<int, 8> k8;
    const integral_constant<int, 16> k16;
    const integral_constant<int, 32> warp;
    const integral_constant<int, 128> cta;
    const integral_constant<int, 256> wide;
    // A warp to a row needs no barrier, and no more registers than the row fills; with few rows, or rows that a warp cannot
    // keep, the CTA takes a row together.  bf16, us with a warp and with the CTA: 8192 x 4096 17.8 and 19.6 (0.86 and 0.79
    // of the measured bandwidth), 8192 x 1024 5.2 and 9.9, 500 x 4096 3.0 and 2.5.
    if (cols > 4096) return go(wide, k4, wide, any);
    if (rows < 8 * sms) return cols <= 1024 ? go(cta, k1, cta, any) : go(cta, k4, cta, any);
    // Short rows: several to a warp, few lanes without a piece, and the more pieces a thread has on their way the better, as
    // long as a row is still read in whole lines.  us with a warp to a row, and with the threads below: 15.68 M x 8 3122 and
    // 114, 15.68 M x 32 3099 and 320, 8 M x 64 1621 and 273, 4 M x 128 840 and 283 (0.84 of the measured bandwidth), 2 M x 256
    // 441 and 249, 1 M x 512 306 and 242 (0.97); 8192 x 1024 5.5 and 6.0, so 1024 keep the warp.
    if (vec && cols <= 8) return go(k1, k1, cta, aligned);
    if (vec && cols <= 16) return go(k1, k2, cta, aligned);
    if (vec && cols <= 32) return go(k2, k2, cta, aligned);
    if (vec && cols <= 64) return go(k2, k4, cta, aligned);
    if (vec && cols <= 128) return go(k4, k4, cta, aligned);
    if (vec && cols <= 256) return go(k4, k8, cta, aligned);
    if (vec && cols <= 512) return go(k8, k8, cta, aligned);
    // Unaligned ones are read value by value, where lanes side by side count more: 4 M x 100 1054 and 597 with one piece to a
    // thread, 1241 with four.
    if (cols <= 8) return go(k1, k1, cta, unaligned);
    if (cols <= 16) return go(k2, k1, cta, unaligned);
    if (cols <= 32) return go(k4, k1, cta, unaligned);
    if (cols <= 64) return go(k8, k1, cta, unaligned);
    if (cols <= 128) return go(k16, k1, cta, unaligned);
    if (cols <= 256) return go(warp, k1, cta, unaligned);
    if (cols <= 512) return go(warp, k2, cta, unaligned);
    if (cols <= 1024) return go(warp, k4, cta, any);
    if (cols <= 2048) return go(warp, k8, cta, any);
    return go(warp, k16, cta, any);
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
    return quant_rows(x, q, scale, rows, cols, x_stride, cols, dtype == KDW_BF16, false, nullptr, (cudaStream_t)stream);
}
