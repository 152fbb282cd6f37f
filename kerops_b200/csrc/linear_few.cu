// Products of few rows with large weights (single tokens while a model answers): bound by reading the weights once.
//
// The weights take the M side of mma.sync (m16n8k16 for 16-bit, m16n8k32 for 8-bit operands), the rows the N side, eight to
// a tile.  A lane loads 16 contiguous bytes of a weight row and the same 16 bytes of an input row; the order of the
// contraction inside a fragment is free as long as both operands agree, so the four words of such a piece are, as they
// come, the operands of two products.  The weights go from memory to registers to the tensor pipe, without shared memory;
// the tensor pipe is idle almost always.  A CTA takes 16 output channels of one group and splits the contraction over its
// eight warps in pieces of 64 bytes, so that it reads runs of 512 bytes, or 32 channels with four warps to each half and runs
// of 256 bytes; the warps' sums are added in shared memory.
//
// One row of 4096 x 4096 takes 6.7 us in bf16 and 4.2-4.5 us in 8 bits, 5.1 with its quantisation (0.77 and 0.6 of the measured
// bandwidth: some 2 us are the launch, the first load's latency and the last sums), 8192 x 16384 in bf16 48 us (0.86).
//
// 8-bit products of 16-bit rows: with at most eight rows every CTA quantises the rows it needs itself (they come from L2),
// which is cheaper than a kernel in front.
#include "../../include/kdw.h"
#include "linear_core.cuh"
#include "linear_plan.h"
#include "quant_core.cuh"

namespace kdw {

struct FewParams {
    const char *x, *w;        // rows and weights
    long long x_pitch;        // bytes between rows
    int len;                  // bytes of a row of x (QUANT: of its quantised form) and of w
    const float *x_scale, *w_scale;
    void* y;
    const int* ends;
    int T, E, N;
    int x_bf16, y_bf16;
    int q_pitch;              // QUANT: bytes between the quantised rows in shared memory
};

template <bool STREAM>
__device__ __forceinline__ uint4 load_16(const char* p) {
    uint4 v;
    if (STREAM)
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    else
        v = __ldg(reinterpret_cast<const uint4*>(p));
    return v;
}

// Bytes [at, at + 16) of a row of `len` bytes, zeros beyond it: issue() starts the loads, get() waits for them.  VEC: rows
// start on 16-byte boundaries and len is a multiple of 16.  Otherwise the piece is shifted together from the two aligned
// pieces that hold its bytes.  No piece without a byte of the row is read (in its place one that has some), and the loads
// stand outside branches, so that all of a lane's are in flight at once.
template <bool VEC>
struct Piece {
    uint4 v;
    template <bool STREAM>
    __device__ __forceinline__ void issue(const char* row, int at, int len) {
        v = make_uint4(0, 0, 0, 0);
        if (at < len) v = load_16<STREAM>(row + at);
    }
    __device__ __forceinline__ uint4 get() const { return v; }
};
template <>
struct Piece<false> {
    uint4 v0, v1;
    int lead, n;
    template <bool STREAM>
    __device__ __forceinline__ void issue(const char* row, int at, int len) {
        n = len - at < 16 ? len - at : 16;
        const uintptr_t p = (uintptr_t)(row + (n > 0 ? at : 0));
        lead = (int)(p & 15);
        const char* aligned = reinterpret_cast<const char*>(p - lead);
        v0 = load_16<false>(aligned);
        v1 = load_16<false>(lead + n > 16 ? aligned + 16 : aligned);
    }
    __device__ __forceinline__ uint4 get() const {
        uint32_t w[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w}, o[4];
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = lead & 8 ? w[i + 2] : w[i];
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = lead & 4 ? w[i + 1] : w[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int left = n - 4 * i;
            const uint32_t keep = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : 0xffffffffu >> (8 * (4 - left));
            o[i] = __funnelshift_r(w[i], w[i + 1], (lead & 3) * 8) & keep;
        }
        return make_uint4(o[0], o[1], o[2], o[3]);
    }
};
template <bool VEC>
__device__ __forceinline__ uint4 load_piece(const char* row, int at, int len) {
    Piece<VEC> p;
    p.template issue<false>(row, at, len);
    return p.get();
}

template <bool I8, bool BF16>
__device__ __forceinline__ void few_mma(uint32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    if constexpr (I8) {
        asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else {
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(c[i]);
        if constexpr (BF16)
            asm volatile(
                "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                : "+f"(f[0]), "+f"(f[1]), "+f"(f[2]), "+f"(f[3])
                : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
        else
            asm volatile(
                "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                : "+f"(f[0]), "+f"(f[1]), "+f"(f[2]), "+f"(f[3])
                : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = __float_as_uint(f[i]);
    }
}

// Rows [begin, end) of the slot-th group that has rows, or an empty range; also the end of the last group (one warp).
__device__ __forceinline__ void few_group(const FewParams& p, int slot, int lane, int* g, int* begin, int* end, int* last) {
    int before = 0, seen = 0;
    *g = -1;
    *begin = *end = 0;
    int next = lane < p.E ? __ldg(p.ends + lane) : 0;
    for (int base = 0; base < p.E; base += 32) {
        const int e = base + lane;
        int stop = next;
        next = e + 32 < p.E ? __ldg(p.ends + e + 32) : 0;
        stop = stop < 0 ? 0 : (stop > p.T ? p.T : stop);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, stop, d);
            if (lane >= d && o > stop) stop = o;
        }
        if (stop < before) stop = before;
        int start = __shfl_up_sync(0xffffffffu, stop, 1);
        if (lane == 0) start = before;
        const unsigned has = __ballot_sync(0xffffffffu, e < p.E && stop > start);
        const int n = __popc(has);
        if (*g < 0 && slot < seen + n) {
            const int l = __fns(has, 0, slot - seen + 1);
            *g = base + l;
            *begin = __shfl_sync(0xffffffffu, start, l);
            *end = __shfl_sync(0xffffffffu, stop, l);
        }
        seen += n;
        before = __shfl_sync(0xffffffffu, stop, 31);
    }
    *last = before;
}

// NT: tiles of eight rows that share one pass over the weights.  QUANT: x holds 16-bit rows (NT == 1).
template <bool I8, bool BF16, bool QUANT, int NT, bool VEC, int WARPS, int U, int CH>
__global__ __launch_bounds__(32 * WARPS, 2) void linear_few_kernel(const __grid_constant__ FewParams p) {
    extern __shared__ __align__(16) char s_q[];
    constexpr int KW = WARPS * 16 / CH;  // warps along the contraction
    __shared__ uint32_t s_sum[KW][NT * 8][CH + 1];
    __shared__ int s_group[4];
    __shared__ uint32_t s_max[8];
    __shared__ float s_scale[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
    const int n0 = blockIdx.x * CH, kw = warp % KW, ch = warp / KW * 16;
    grid_dependency_wait();
    grid_launch_dependents();
    int g = 0, begin = 0, end = p.T, last = p.T;
    if (p.ends) {
        if (warp == 0) {
            few_group(p, blockIdx.y, lane, &g, &begin, &end, &last);
            if (lane == 0) {
                s_group[0] = g;
                s_group[1] = begin;
                s_group[2] = end;
                s_group[3] = last;
            }
        }
        __syncthreads();
        g = s_group[0];
        begin = s_group[1];
        end = s_group[2];
        last = s_group[3];
    }
    uint16_t* const y = reinterpret_cast<uint16_t*>(p.y);
    if (blockIdx.y == 0)
        for (int i = threadIdx.x; i < (p.T - last) * CH; i += 32 * WARPS)
            if (n0 + i % CH < p.N) y[(long long)(last + i / CH) * p.N + n0 + i % CH] = 0;
    if (end <= begin) return;

    const char* wr[2];
    int wlen[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int n = n0 + ch + gid + 8 * h;
        wlen[h] = n < p.N ? p.len : 0;
        wr[h] = p.w + ((long long)g * p.N + (n < p.N ? n : 0)) * p.len;
    }
    const int pieces = (p.len + 63) >> 6;

    for (int t0 = begin; t0 < end; t0 += NT * 8) {
        Piece<VEC> wp[U][2];
        auto load_weights = [&](int u, int c) {
#pragma unroll
            for (int h = 0; h < 2; ++h) wp[u][h].template issue<true>(wr[h], c * 64 + tig * 16, wlen[h]);
        };
#pragma unroll
        for (int u = 0; u < U; ++u) load_weights(u, kw + u * KW);
        if constexpr (QUANT) {
            // the rows of this tile, quantised into shared memory while the first weights are on their way
            const int rows = end - t0 < 8 ? end - t0 : 8;
            const int vecs = (p.len + 7) >> 3;
            if (threadIdx.x < 8) s_max[threadIdx.x] = 0;
            __syncthreads();
            for (int r = 0; r < rows; ++r) {
                const char* row = p.x + (t0 + r) * p.x_pitch;
                uint32_t m = 0;
                for (int i = threadIdx.x; i < vecs; i += 32 * WARPS)
                    m = max_bits(load_piece<VEC>(row, i * 16, 2 * p.len), m);
                m = __reduce_max_sync(0xffffffffu, m);
                if (lane == 0 && m) atomicMax(&s_max[r], m);
            }
            __syncthreads();
            for (int r = 0; r < rows; ++r) {
                const char* row = p.x + (t0 + r) * p.x_pitch;
                const QuantRow q = quant_row(s_max[r], p.x_bf16);
                if (threadIdx.x == 0) s_scale[r] = q.scale;
                for (int i = threadIdx.x; i < p.q_pitch / 8; i += 32 * WARPS) {
                    uint2 o = make_uint2(0, 0);
                    if (i < vecs) o = quant8(load_piece<VEC>(row, i * 16, 2 * p.len), q, p.x_bf16);
                    *reinterpret_cast<uint2*>(s_q + r * p.q_pitch + i * 8) = o;
                }
            }
            __syncthreads();
        }
        uint32_t acc[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][i] = 0;
        const char* xr[NT];
        int xlen[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int t = t0 + j * 8 + gid;
            xlen[j] = t < end ? p.len : 0;
            xr[j] = QUANT ? s_q + gid * p.q_pitch : p.x + (t < end ? t : t0) * p.x_pitch;
        }
        Piece<VEC || QUANT> xp[U][NT];
        auto load_rows = [&](int u, int c) {
            const int at = c * 64 + tig * 16;
#pragma unroll
            for (int j = 0; j < NT; ++j)
                if constexpr (QUANT)
                    xp[u][j].v = at < xlen[j] ? *reinterpret_cast<const uint4*>(xr[j] + at) : make_uint4(0, 0, 0, 0);
                else
                    xp[u][j].template issue<false>(xr[j], at, xlen[j]);
        };
        if (!QUANT) {  // quantised rows wait in shared memory
#pragma unroll
            for (int u = 0; u < U; ++u) load_rows(u, kw + u * KW);
        }
        for (int c = kw; c < pieces; c += U * KW) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (QUANT) load_rows(u, c + u * KW);
                const uint4 w0 = wp[u][0].get(), w1 = wp[u][1].get();
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const uint4 x = xp[u][j].get();
                    few_mma<I8, BF16>(acc[j], w0.x, w1.x, w0.y, w1.y, x.x, x.y);
                    few_mma<I8, BF16>(acc[j], w0.z, w1.z, w0.w, w1.w, x.z, x.w);
                }
                // the piece that takes this one's place is on its way while the others are used
                if (c + U * KW < pieces) {
                    load_weights(u, c + (u + U) * KW);
                    if (!QUANT) load_rows(u, c + (u + U) * KW);
                }
            }
        }
        if (t0 != begin) __syncthreads();
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) s_sum[kw][j * 8 + tig * 2 + (i & 1)][ch + gid + 8 * (i >> 1)] = acc[j][i];
        __syncthreads();
        for (int i = threadIdx.x; i < NT * 8 * CH; i += 32 * WARPS) {
            const int r = i / CH, c = i % CH, t = t0 + r, n = n0 + c;
            if (t >= end || n >= p.N) continue;
            float v = 0.f;
            if constexpr (I8) {
                int s = 0;
#pragma unroll
                for (int k = 0; k < KW; ++k) s += (int)s_sum[k][r][c];
                v = RowScale(QUANT ? s_scale[r] : __ldg(p.x_scale + t)).of(s, __ldg(p.w_scale + (long long)g * p.N + n));
            } else {
#pragma unroll
                for (int k = 0; k < KW; ++k) v += __uint_as_float(s_sum[k][r][c]);
            }
            y[(long long)t * p.N + n] = (uint16_t)pack2(v, 0.f, p.y_bf16);
        }
        if (QUANT) __syncthreads();
    }
}

template <bool I8, bool BF16, bool QUANT, int NT, bool VEC, int WARPS, int U, int CH>
static int few_warps(const FewParams& p, cudaStream_t st) {
    const dim3 grid((unsigned)((p.N + CH - 1) / CH), (unsigned)(p.ends ? (p.E < p.T ? p.E : p.T) : 1));
    if (QUANT) {
        static KernelSetup setup;
        int sms = 0, occ = 0;
        int rc = setup.get((const void*)linear_few_kernel<I8, BF16, QUANT, NT, VEC, WARPS, U, CH>, 32 * WARPS, 8 * kFewQuantPitch, &sms, &occ);
        if (rc) return rc;
    }
    KDW_CUDA(launch_overlapping_previous_grid(linear_few_kernel<I8, BF16, QUANT, NT, VEC, WARPS, U, CH>, grid, dim3(32 * WARPS),
                                              (size_t)(QUANT ? p.q_pitch * 8 : 0), st, 1, p));
    return 0;
}
template <bool I8, bool BF16, bool QUANT, int NT, bool VEC>
static int few_launch(const FewParams& p, cudaStream_t st) {
    // Pieces in flight per lane and weight row.  One row of 4096 x 4096 in bf16: 8.2 us with eight, 10.5 us with four (6.7 us
    // now that a piece's successor is loaded as soon as it has been used).
    constexpr int U = (NT == 1 ? 8 : 4) / (VEC ? 1 : 4);
    int sms = 0;
    int rc = device_facts(nullptr, &sms);
    if (rc) return rc;
    if (few_channels(p.N, p.ends ? (p.E < p.T ? p.E : p.T) : 1, sms) == 32) return few_warps<I8, BF16, QUANT, NT, VEC, 8, U, 32>(p, st);
    return few_warps<I8, BF16, QUANT, NT, VEC, 8, U, 16>(p, st);
}
template <bool I8, bool BF16, bool VEC>
static int few_rows(const FewParams& p, cudaStream_t st) {
    return p.T <= 8 ? few_launch<I8, BF16, false, 1, VEC>(p, st) : few_launch<I8, BF16, false, 2, VEC>(p, st);
}

int linear_few(const LinArgs& a, int x_type, cudaStream_t st) {
    FewParams p;
    p.x = (const char*)a.a;
    p.w = (const char*)a.b;
    const bool quant = a.esize == 1 && x_type != KDW_I8;
    const int x_size = quant ? 2 : a.esize;
    p.x_pitch = a.a_stride * x_size;
    p.len = (int)(a.K * a.esize);
    p.x_scale = a.row_scale;
    p.w_scale = a.col_scale;
    p.y = a.out;
    p.ends = a.ends;
    p.T = (int)a.T;
    p.E = (int)a.E;
    p.N = (int)a.N;
    p.x_bf16 = x_type == KDW_BF16;
    p.y_bf16 = a.out_bf16;
    p.q_pitch = quant ? (p.len + 127) / 128 * 128 + 64 : 0;  // eight lanes then read all 32 banks
    const bool vec = ((uintptr_t)p.x & 15) == 0 && ((uintptr_t)p.w & 15) == 0 && p.x_pitch % 16 == 0 && p.len % 16 == 0;
    if (quant) return vec ? few_launch<true, false, true, 1, true>(p, st) : few_launch<true, false, true, 1, false>(p, st);
    if (a.esize == 1) return vec ? few_rows<true, false, true>(p, st) : few_rows<true, false, false>(p, st);
    if (a.in_bf16) return vec ? few_rows<false, true, true>(p, st) : few_rows<false, true, false>(p, st);
    return vec ? few_rows<false, false, true>(p, st) : few_rows<false, false, false>(p, st);
}

}  // namespace kdw
