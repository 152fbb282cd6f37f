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

// TPR threads to a row (a warp or the CTA), KEEP vectors of 8 values of a thread stay in registers between the two passes
// over the row; what is longer is read again.  CTAs from `ctas` on copy weights instead.  VEC: rows of the input are 16-byte aligned, QVEC: rows of the output 8-byte.
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
        m = __reduce_max_sync(0xffffffffu, m);
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

template <int TPR, int KEEP, int THREADS>
static int quant_launch(const void* x, void* q, float* scale, int64_t rows, int64_t cols, int64_t x_stride, int64_t q_stride,
                        int bf16, bool vec, bool qvec, const PackRows* pack, cudaStream_t st) {
    int sms = 0;
    int rc = device_facts(nullptr, &sms);
    if (rc) return rc;
    const int64_t blocks = (rows + THREADS / TPR - 1) / (THREADS / TPR);
    const int grid = (int)(blocks < 2048 / THREADS * sms ? blocks : 2048 / THREADS * sms);
    const int more = pack ? pack_ctas(*pack, 1, sms) * (256 / THREADS) : 0;
    auto* k = vec ? (qvec ? quant_rows_kernel<TPR, KEEP, true, true, THREADS> : quant_rows_kernel<TPR, KEEP, true, false, THREADS>)
                  : (qvec ? quant_rows_kernel<TPR, KEEP, false, true, THREADS> : quant_rows_kernel<TPR, KEEP, false, false, THREADS>);
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
    auto go = [&](auto tpr, auto keep, auto threads) {
        return quant_launch<decltype(tpr)::value, decltype(keep)::value, decltype(threads)::value>(
            x, q, scale, rows, cols, x_stride, q_stride, bf16, vec, qvec, pack, st);
    };
    using std::integral_constant;
    const integral_constant<int, 1> k1;
    const integral_constant<int, 2> k2;
    const integral_constant<int, 4> k4;
    const integral_constant<int, 8> k8;
    const integral_constant<int, 16> k16;
    const integral_constant<int, 32> warp;
    const integral_constant<int, 128> cta;
    const integral_constant<int, 256> wide;
    // A warp to a row needs no barrier, and no more registers than the row fills; with few rows, or rows that a warp cannot
    // keep, the CTA takes a row together.  bf16, us with a warp and with the CTA: 8192 x 4096 17.8 and 19.6 (0.86 and 0.79
    // of the measured bandwidth), 8192 x 1024 5.2 and 9.9, 500 x 4096 3.0 and 2.5.
    if (cols > 4096) return go(wide, k4, wide);
    if (rows < 8 * sms) return cols <= 1024 ? go(cta, k1, cta) : go(cta, k4, cta);
    if (cols <= 256) return go(warp, k1, cta);
    if (cols <= 512) return go(warp, k2, cta);
    if (cols <= 1024) return go(warp, k4, cta);
    if (cols <= 2048) return go(warp, k8, cta);
    return go(warp, k16, cta);
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
