// Products of many rows with one narrow weight matrix (the pointwise product behind a depthwise convolution on a volume:
// 8 to 128 channels, millions of voxels): bound by reading and writing the rows once.
//
// Rows of 16 to 256 bytes are too short for the TMA unit, which moves 40-50 G box rows per second whatever their length;
// here a warp loads them straight into the operand registers of mma.sync, 16 rows to a tile, in runs of contiguous memory.
// The weights stay in registers as the other operand for the whole kernel.  The order of the contraction and of the output
// columns inside a fragment is free: a lane's words of a 16-byte piece of a row are the operands of two products as they
// come, and the columns are dealt to the fragments so that a lane's results are 16 contiguous bytes of an output row.
//
// 4.48 M rows, fp16: 32 -> 32 channels 95 us, 128 -> 8 184 us (0.92 and 1.01 of the measured copy bandwidth), 64 -> 64, whose
// weights fill the registers, 181 us (0.97); the tensor-core kernel of linear_mma.cu took 295 us for 64 -> 32 (now 137 us).
#include "../../include/kdw.h"
#include "linear_core.cuh"
#include "linear_plan.h"

namespace kdw {

struct NarrowParams {
    const char* x;
    const uint16_t* w;
    char* y;
    const int* ends;          // one end, or null
    long long x_pitch;        // bytes
    long long T;
    int K, N;                 // contraction and output columns, multiples of 8
    int across;               // 1: the contraction runs along the rows of the weights
};

template <bool BF16>
__device__ __forceinline__ void narrow_mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
    if constexpr (BF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// WORDS 32-bit words of a lane's piece of a row.
template <int WORDS>
__device__ __forceinline__ void narrow_load(uint32_t (&v)[WORDS], const char* p, bool live) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) v[i] = 0;
    if (!live) return;
    if constexpr (WORDS == 4)
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "l"(p));
    else if constexpr (WORDS == 2)
        asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "l"(p));
    else
        asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(v[0]) : "l"(p));
}

// KP, NP: contraction and columns rounded up to 8, 16, 32, 64 or 128; KP * NP <= 4096, so that the weights fit the registers.
template <bool BF16_, int KP_, int NP_>
struct NCfg {
    static constexpr bool BF16 = BF16_;
    static constexpr int KP = KP_, NP = NP_;
    static constexpr int WORDS = KP >= 32 ? 4 : KP / 8;         // words of a lane's piece: a row is PIECES x 4 lanes x WORDS
    static constexpr int PIECES = KP >= 32 ? KP / 32 : 1;
    static constexpr int STEPS = KP >= 16 ? KP / 16 : 1;        // products of a tile and eight columns
    static constexpr int COLS = NP >= 32 ? 32 : NP;             // columns whose results a lane stores as one piece
    static constexpr int GROUPS = NP / COLS, TILES = COLS / 8;  // of eight columns, per piece
    static constexpr int AHEAD = PIECES >= 4 ? 1 : PIECES == 2 ? 2 : 4;  // row tiles whose loads are in flight
    // The tiles of a warp in flight are neighbours, or spread over the warps' tiles where rows of 256 bytes are written and those
    // read have 32 bytes and more.  4.48 M rows, us, neighbours and spread: 64 -> 64 181 and 187, 32 -> 64 149 and 154, 8 -> 128
    // 212 and 208, 16 -> 128 255 and 231, 32 -> 128 257 and 254.
    static constexpr bool SPREAD = NP == 128 && KP >= 16;
    static constexpr int THREADS = 128;
    static constexpr int CTAS = KP * NP >= 4096 ? 3 : 4;        // to an SM at least: what the registers have to allow
};

template <class C>
__global__ __launch_bounds__(C::THREADS, C::CTAS) void linear_narrow_kernel(const __grid_constant__ NarrowParams p) {
    const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
    const long long warp = ((long long)blockIdx.x * C::THREADS + threadIdx.x) >> 5, warps = (long long)gridDim.x * (C::THREADS / 32);
    grid_dependency_wait();
    grid_launch_dependents();
    // The weights, through shared memory: read in order, then picked by every lane.  [w_rows][w_cols] in memory; 16 bytes
    // between the rows keep the picks out of each other's banks.
    __shared__ __align__(16) uint16_t s_w[C::KP * C::NP + 8 * (C::KP > C::NP ? C::KP : C::NP)];
    const bool across = p.across;
    const int w_rows = across ? p.K : p.N, pieces = (across ? p.N : p.K) >> 3, pitch = pieces * 8 + 8;
    for (int i = threadIdx.x; i < w_rows * pieces; i += C::THREADS) {
        const int r = i / pieces, c = i - r * pieces;
        *reinterpret_cast<uint4*>(s_w + r * pitch + c * 8) = __ldg(reinterpret_cast<const uint4*>(p.w) + i);
    }
    __syncthreads();
    long long rows = p.T;
    if (p.ends) {
        const int e = __ldg(p.ends);
        rows = e < 0 ? 0 : (e < p.T ? e : p.T);
    }
    // Weights.  Step s of piece q covers, for this lane, contraction indexes q * 32 + tig * 8 + (s & 1) * 4 + {0, 1} and
    // + {2, 3} (KP >= 32); the slot `gid` of tile j of a column group is column (gid / 2) * 2 TILES + 2 j + (gid & 1).
    uint32_t b[C::GROUPS][C::TILES][C::STEPS][2];
#pragma unroll
    for (int g = 0; g < C::GROUPS; ++g)
#pragma unroll
        for (int j = 0; j < C::TILES; ++j)
#pragma unroll
            for (int s = 0; s < C::STEPS; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int n = g * C::COLS + (gid >> 1) * 2 * C::TILES + 2 * j + (gid & 1);
                    const int k = C::KP >= 32 ? (s >> 1) * 32 + tig * 8 + (s & 1) * 4 + h * 2 : tig * C::KP / 4 + h * 2;
                    uint32_t v = 0;
                    if (n < p.N && k < p.K && (C::KP > 8 || h == 0)) {
                        if (across)
                            v = s_w[k * pitch + n] | (uint32_t)s_w[(k + 1) * pitch + n] << 16;
                        else
                            v = *reinterpret_cast<const uint32_t*>(s_w + n * pitch + k);
                    }
                    b[g][j][s][h] = v;
                }
    const long long tiles = (p.T + 15) >> 4;
    const int kbytes = p.K * 2;
    auto load = [&](uint32_t (&a)[C::PIECES][2][C::WORDS], long long t) {
#pragma unroll
        for (int q = 0; q < C::PIECES; ++q)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const long long r = t * 16 + gid + 8 * h;
                const int at = q * 64 + tig * C::WORDS * 4;
                narrow_load<C::WORDS>(a[q][h], p.x + r * p.x_pitch + at, r < rows && at < kbytes);
            }
    };
    uint32_t a[C::AHEAD][C::PIECES][2][C::WORDS];
#pragma unroll
    for (int i = 0; i < C::AHEAD; ++i) load(a[i], C::SPREAD ? warp + i * warps : warp * C::AHEAD + i);
    for (long long t0 = C::SPREAD ? warp : warp * C::AHEAD; t0 < tiles; t0 += C::AHEAD * warps) {
#pragma unroll
        for (int i = 0; i < C::AHEAD; ++i) {
            const long long t = t0 + (C::SPREAD ? i * warps : i);
            if (t >= tiles) break;
#pragma unroll
            for (int g = 0; g < C::GROUPS; ++g) {
                float c[C::TILES][4];
#pragma unroll
                for (int j = 0; j < C::TILES; ++j) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[j][e] = 0.f;
#pragma unroll
                    for (int s = 0; s < C::STEPS; ++s) {
                        constexpr int M = C::WORDS - 1;
                        const int q = C::KP >= 32 ? s >> 1 : 0, o = C::KP >= 32 ? (s & 1) * 2 : 0;
                        narrow_mma16<C::BF16>(c[j], a[i][q][0][o], a[i][q][1][o], C::KP > 8 ? a[i][q][0][(o + 1) & M] : 0u,
                                              C::KP > 8 ? a[i][q][1][(o + 1) & M] : 0u, b[g][j][s][0], b[g][j][s][1]);
                    }
                }
                if (g + 1 == C::GROUPS) load(a[i], t + C::AHEAD * warps);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const long long r = t * 16 + gid + 8 * h;
                    const int col = g * C::COLS + tig * 2 * C::TILES;
                    if (r >= p.T || col >= p.N) continue;
                    uint32_t o[C::TILES];
#pragma unroll
                    for (int j = 0; j < C::TILES; ++j) o[j] = r < rows ? pack2(c[j][2 * h], c[j][2 * h + 1], C::BF16) : 0u;
                    char* dst = p.y + (r * p.N + col) * 2;
                    if constexpr (C::TILES == 4)
                        *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
                    else if constexpr (C::TILES == 2)
                        *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
                    else
                        *reinterpret_cast<uint32_t*>(dst) = o[0];
                }
            }
        }
    }
}

template <class C>
static int narrow_launch(const NarrowParams& p, cudaStream_t st) {
    static KernelSetup setup;
    int sms = 0, occ = 0;
    int rc = setup.get((const void*)linear_narrow_kernel<C>, C::THREADS, 0, &sms, &occ);
    if (rc) return rc;
    const long long want = ((p.T + 15) / 16 + C::THREADS / 32 - 1) / (C::THREADS / 32);
    const long long most = (long long)sms * occ;
    KDW_CUDA(launch_overlapping_previous(linear_narrow_kernel<C>, (unsigned)(want < most ? want : most), (unsigned)C::THREADS, st, p));
    return 0;
}
template <bool BF16, int KP>
static int narrow_cols(const NarrowParams& p, cudaStream_t st) {
    if (p.N <= 8) return narrow_launch<NCfg<BF16, KP, 8>>(p, st);
    if (p.N <= 16) return narrow_launch<NCfg<BF16, KP, 16>>(p, st);
    if (p.N <= 32) return narrow_launch<NCfg<BF16, KP, 32>>(p, st);
    if constexpr (KP <= 64) {
        if (p.N <= 64) return narrow_launch<NCfg<BF16, KP, 64>>(p, st);
    }
    if constexpr (KP <= 32) {
        if (p.N <= 128) return narrow_launch<NCfg<BF16, KP, 128>>(p, st);
    }
    set_error("linear: %d x %d weights are not narrow", p.K, p.N);
    return KDW_ERR_ARG;
}
template <bool BF16>
static int narrow_rows(const NarrowParams& p, cudaStream_t st) {
    if (p.K <= 8) return narrow_cols<BF16, 8>(p, st);
    if (p.K <= 16) return narrow_cols<BF16, 16>(p, st);
    if (p.K <= 32) return narrow_cols<BF16, 32>(p, st);
    if (p.K <= 64) return narrow_cols<BF16, 64>(p, st);
    return narrow_cols<BF16, 128>(p, st);
}

// ------------------------------------------------------------------------------------------------------------------
// Both gradients of such a product in one pass over the gradient g and the rows x:  dx = g W,  dw = g^T x.  dx as above.  For
// dw the rows are the contraction: the 8 x 8 blocks (rows x channels) that a warp's words form are transposed in registers
// (movmatrix) and are then, as they come, the fragments of both operands; the sums stay in registers for the whole kernel, so
// K N <= 2048.  A CTA's warps add theirs in shared memory, the CTAs' are added by a second kernel in their order.
// Bytes: g and x read, dx written, once each; two kernels read g twice.  4.48 M rows, 32 and 64 channels: 207 us, 0.84 of the
// measured bandwidth; the two products took 137 and 134 us.
// ------------------------------------------------------------------------------------------------------------------
struct NarrowGradsParams {
    const char *x, *g;
    const uint16_t* w;        // [N][K]
    char* dx;
    float* partial;           // [CTA][NG][KX]
    const int* ends;
    long long x_pitch, g_pitch;  // bytes
    long long T;
    int K, N;
};

template <bool BF16_, int KX_, int NG_>
struct GCfg {
    static constexpr bool BF16 = BF16_;
    static constexpr int KX = KX_, NG = NG_;                    // channels of x and g, rounded up
    static constexpr int XW = KX >= 32 ? 4 : KX / 8, XP = KX >= 32 ? KX / 32 : 1, XM = KX / 8;  // words, pieces, 8-channel blocks
    static constexpr int GW = NG >= 32 ? 4 : NG / 8, GP = NG >= 32 ? NG / 32 : 1, GM = NG / 8;
    static constexpr int GB = (GM + 1) / 2;                     // blocks of 16 output rows of dw
    static constexpr int STEPS = NG >= 16 ? NG / 16 : 1;        // products of dx: contraction over g's channels
    static constexpr int COLS = KX >= 32 ? 32 : KX, GROUPS = KX / COLS, TILES = COLS / 8;
    static constexpr int AHEAD = XP + GP >= 5 ? 1 : 2;
    static constexpr int THREADS = 128;
};

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// Channel of slot `slot` of block m = piece * WORDS + word.
template <int WORDS>
__device__ __forceinline__ int block_channel(int m, int slot) {
    return m / WORDS * 32 + (slot >> 1) * 2 * WORDS + 2 * (m % WORDS) + (slot & 1);
}

template <class C>
__global__ __launch_bounds__(C::THREADS, 2) void linear_narrow_grads_kernel(const __grid_constant__ NarrowGradsParams p) {
    __shared__ __align__(16) uint16_t s_w[C::KX * C::NG + 8 * C::NG];
    __shared__ float s_dw[C::NG * C::KX];
    const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3, warp_in = threadIdx.x >> 5;
    const long long warp = ((long long)blockIdx.x * C::THREADS + threadIdx.x) >> 5, warps = (long long)gridDim.x * (C::THREADS / 32);
    grid_dependency_wait();
    grid_launch_dependents();
    // weights [N][K] in shared memory, then in the registers as the operand of dx: contraction along their rows
    const int pieces = p.K >> 3, pitch = p.K + 8;
    for (int i = threadIdx.x; i < p.N * pieces; i += C::THREADS) {
        const int r = i / pieces, c = i - r * pieces;
        *reinterpret_cast<uint4*>(s_w + r * pitch + c * 8) = __ldg(reinterpret_cast<const uint4*>(p.w) + i);
    }
    __syncthreads();
    long long rows = p.T;
    if (p.ends) {
        const int e = __ldg(p.ends);
        rows = e < 0 ? 0 : (e < p.T ? e : p.T);
    }
    uint32_t b[C::GROUPS][C::TILES][C::STEPS][2];
#pragma unroll
    for (int o = 0; o < C::GROUPS; ++o)
#pragma unroll
        for (int j = 0; j < C::TILES; ++j)
#pragma unroll
            for (int s = 0; s < C::STEPS; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int k = o * C::COLS + (gid >> 1) * 2 * C::TILES + 2 * j + (gid & 1);
                    const int n = C::NG >= 32 ? (s >> 1) * 32 + tig * 8 + (s & 1) * 4 + h * 2 : tig * C::NG / 4 + h * 2;
                    b[o][j][s][h] = k < p.K && n < p.N && (C::NG > 8 || h == 0)
                                        ? s_w[n * pitch + k] | (uint32_t)s_w[(n + 1) * pitch + k] << 16
                                        : 0u;
                }
    float dw[C::GB][C::XM][4];
#pragma unroll
    for (int i = 0; i < C::GB; ++i)
#pragma unroll
        for (int j = 0; j < C::XM; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) dw[i][j][e] = 0.f;

    const long long tiles = (p.T + 15) >> 4;
    uint32_t g[C::AHEAD][C::GP][2][C::GW], x[C::AHEAD][C::XP][2][C::XW];
    auto load = [&](int i, long long t) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const long long r = t * 16 + gid + 8 * h;
#pragma unroll
            for (int q = 0; q < C::GP; ++q) {
                const int at = q * 64 + tig * C::GW * 4;
                narrow_load<C::GW>(g[i][q][h], p.g + r * p.g_pitch + at, r < rows && at < 2 * p.N);
            }
#pragma unroll
            for (int q = 0; q < C::XP; ++q) {
                const int at = q * 64 + tig * C::XW * 4;
                narrow_load<C::XW>(x[i][q][h], p.x + r * p.x_pitch + at, r < rows && at < 2 * p.K);
            }
        }
    };
#pragma unroll
    for (int i = 0; i < C::AHEAD; ++i) load(i, warp * C::AHEAD + i);
    for (long long t0 = warp * C::AHEAD; t0 < tiles; t0 += C::AHEAD * warps) {
#pragma unroll
        for (int i = 0; i < C::AHEAD; ++i) {
            const long long t = t0 + i;
            if (t >= tiles) break;
            // dx of 16 rows
#pragma unroll
            for (int o = 0; o < C::GROUPS; ++o) {
                float c[C::TILES][4];
#pragma unroll
                for (int j = 0; j < C::TILES; ++j) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[j][e] = 0.f;
#pragma unroll
                    for (int s = 0; s < C::STEPS; ++s) {
                        constexpr int M = C::GW - 1;
                        const int q = C::NG >= 32 ? s >> 1 : 0, a = C::NG >= 32 ? (s & 1) * 2 : 0;
                        narrow_mma16<C::BF16>(c[j], g[i][q][0][a], g[i][q][1][a], C::NG > 8 ? g[i][q][0][(a + 1) & M] : 0u,
                                              C::NG > 8 ? g[i][q][1][(a + 1) & M] : 0u, b[o][j][s][0], b[o][j][s][1]);
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const long long r = t * 16 + gid + 8 * h;
                    const int col = o * C::COLS + tig * 2 * C::TILES;
                    if (r >= p.T || col >= p.K) continue;
                    uint32_t v[C::TILES];
#pragma unroll
                    for (int j = 0; j < C::TILES; ++j) v[j] = r < rows ? pack2(c[j][2 * h], c[j][2 * h + 1], C::BF16) : 0u;
                    char* dst = p.dx + (r * p.K + col) * 2;
                    if constexpr (C::TILES == 4)
                        *reinterpret_cast<uint4*>(dst) = make_uint4(v[0], v[1], v[2], v[3]);
                    else if constexpr (C::TILES == 2)
                        *reinterpret_cast<uint2*>(dst) = make_uint2(v[0], v[1]);
                    else
                        *reinterpret_cast<uint32_t*>(dst) = v[0];
                }
            }
            // dw of the same rows
            __syncwarp();
            uint32_t xt[C::XM][2];
#pragma unroll
            for (int m = 0; m < C::XM; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) xt[m][h] = transpose_8x8(x[i][m / C::XW][h][m % C::XW]);
#pragma unroll
            for (int n = 0; n < C::GB; ++n) {
                uint32_t a[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (2 * n + k < C::GM)
#pragma unroll
                        for (int h = 0; h < 2; ++h) a[k + 2 * h] = transpose_8x8(g[i][(2 * n + k) / C::GW][h][(2 * n + k) % C::GW]);
#pragma unroll
                for (int m = 0; m < C::XM; ++m) narrow_mma16<C::BF16>(dw[n][m], a[0], a[1], a[2], a[3], xt[m][0], xt[m][1]);
            }
            load(i, t + C::AHEAD * warps);
        }
    }
    // the warps' sums, one after the other
    for (int k = 0; k < C::THREADS / 32; ++k) {
        if (warp_in == k)
#pragma unroll
            for (int n = 0; n < C::GB; ++n)
#pragma unroll
                for (int m = 0; m < C::XM; ++m)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (2 * n + (e >> 1) >= C::GM) continue;
                        float& s = s_dw[block_channel<C::GW>(2 * n + (e >> 1), gid) * C::KX + block_channel<C::XW>(m, 2 * tig + (e & 1))];
                        s = k == 0 ? dw[n][m][e] : s + dw[n][m][e];
                    }
        __syncthreads();
    }
    float* out = p.partial + (long long)blockIdx.x * C::NG * C::KX;
    for (int i = threadIdx.x; i < C::NG * C::KX; i += C::THREADS) out[i] = s_dw[i];
}

// Adds the CTAs' sums in their order (eight threads to a value, every eighth CTA each) and rounds once.
__global__ __launch_bounds__(256) void linear_narrow_sum_kernel(const float* __restrict__ partial, uint16_t* dw, int ctas, int NG, int KX,
                                                               int N, int K, int bf16) {
    __shared__ float s[8][32];
    grid_dependency_wait();
    grid_launch_dependents();
    const int o = threadIdx.x & 31, l = threadIdx.x >> 5, at = blockIdx.x * 32 + o;  // NG * KX is a multiple of 32
    float sum = 0.f;
#pragma unroll 8
    for (int c = l; c < ctas; c += 8) sum += __ldcg(partial + (long long)c * NG * KX + at);
    s[l][o] = sum;
    __syncthreads();
    if (l != 0) return;
    for (int i = 1; i < 8; ++i) sum += s[i][o];
    const int n = at / KX, k = at - n * KX;
    if (n < N && k < K) dw[(long long)n * K + k] = (uint16_t)pack2(sum, 0.f, bf16);
}

template <class C>
static int grads_launch(NarrowGradsParams p, void* dw, float* ws, int64_t ws_bytes, int64_t* need, cudaStream_t st) {
    static KernelSetup setup;
    int sms = 0, occ = 0;
    int rc = setup.get((const void*)linear_narrow_grads_kernel<C>, C::THREADS, 0, &sms, &occ);
    if (rc) return rc;
    const long long want = ((p.T + 15) / 16 + C::THREADS / 32 - 1) / (C::THREADS / 32), most = (long long)sms * occ;
    const int grid = (int)(want < most ? want : most);
    *need = (int64_t)grid * C::NG * C::KX * 4;
    if (!dw) return 0;
    if (ws_bytes < *need) {
        set_error("linear_grads_f16: workspace of %lld bytes needed, %lld given", (long long)*need, (long long)ws_bytes);
        return KDW_ERR_WORKSPACE;
    }
    p.partial = ws;
    KDW_CUDA(launch_overlapping_previous(linear_narrow_grads_kernel<C>, (unsigned)grid, (unsigned)C::THREADS, st, p));
    KDW_CUDA(launch_overlapping_previous(linear_narrow_sum_kernel, (unsigned)(C::NG * C::KX / 32), 256u, st, (const float*)ws, (uint16_t*)dw,
                                         grid, C::NG, C::KX, p.N, p.K, (int)C::BF16));
    return 0;
}
template <bool BF16, int KX>
static int grads_cols(const NarrowGradsParams& p, void* dw, float* ws, int64_t bytes, int64_t* need, cudaStream_t st) {
    if (p.N <= 8) return grads_launch<GCfg<BF16, KX, 8>>(p, dw, ws, bytes, need, st);
    if (p.N <= 16) return grads_launch<GCfg<BF16, KX, 16>>(p, dw, ws, bytes, need, st);
    if constexpr (KX <= 64) {
        if (p.N <= 32) return grads_launch<GCfg<BF16, KX, 32>>(p, dw, ws, bytes, need, st);
    }
    if constexpr (KX <= 32) {
        if (p.N <= 64) return grads_launch<GCfg<BF16, KX, 64>>(p, dw, ws, bytes, need, st);
    }
    if constexpr (KX <= 16) {
        if (p.N <= 128) return grads_launch<GCfg<BF16, KX, 128>>(p, dw, ws, bytes, need, st);
    }
    set_error("linear: %d x %d weights are not narrow", p.N, p.K);
    return KDW_ERR_ARG;
}
template <bool BF16>
static int grads_rows(const NarrowGradsParams& p, void* dw, float* ws, int64_t bytes, int64_t* need, cudaStream_t st) {
    if (p.K <= 8) return grads_cols<BF16, 8>(p, dw, ws, bytes, need, st);
    if (p.K <= 16) return grads_cols<BF16, 16>(p, dw, ws, bytes, need, st);
    if (p.K <= 32) return grads_cols<BF16, 32>(p, dw, ws, bytes, need, st);
    return grads_cols<BF16, 64>(p, dw, ws, bytes, need, st);
}

static int64_t narrow_pad(int64_t v) { return v <= 8 ? 8 : v <= 16 ? 16 : v <= 32 ? 32 : v <= 64 ? 64 : 128; }

bool is_narrow(const LinArgs& a) {
    if (a.op == LIN_WGRAD || a.esize != 2 || a.E != 1 || a.K > 128 || a.N > 128) return false;
    if (narrow_pad(a.K) * narrow_pad(a.N) > 4096) return false;
    // (the weights are read by elements; a base that TMA cannot address would need a workspace on the other path)
    return a.K % 8 == 0 && a.N % 8 == 0 && ((uintptr_t)a.a & 15) == 0 && ((uintptr_t)a.b & 15) == 0 && a.a_stride % 8 == 0;
}

// One pass pays with rows enough (20000 rows, 32 and 64 channels: 15.9 us, the two products 13.1) and where the sums leave
// registers for the loads (128 and 16 channels: 434 us, the two products 426).
bool is_narrow_grads(const LinArgs& d, const LinArgs& g) {
    return is_narrow(d) && narrow_pad(d.K) * narrow_pad(d.N) <= 2048 && d.K <= 64 && d.T >= 32768 && ((uintptr_t)g.b & 15) == 0 && g.b_stride % 8 == 0;
}

int linear_narrow_grads(const LinArgs& d, const LinArgs& g, void* ws, int64_t ws_bytes, int64_t* need, cudaStream_t st) {
    NarrowGradsParams p;
    p.x = (const char*)g.b;
    p.g = (const char*)d.a;
    p.w = (const uint16_t*)d.b;
    p.dx = (char*)d.out;
    p.partial = nullptr;
    p.ends = d.ends;
    p.x_pitch = g.b_stride * 2;
    p.g_pitch = d.a_stride * 2;
    p.T = d.T;
    p.K = (int)d.K;
    p.N = (int)d.N;
    return d.in_bf16 ? grads_rows<true>(p, g.out, (float*)ws, ws_bytes, need, st)
                     : grads_rows<false>(p, g.out, (float*)ws, ws_bytes, need, st);
}

int linear_narrow(const LinArgs& a, cudaStream_t st) {
    NarrowParams p;
    const bool fwd = a.op == LIN_FWD;
    p.x = (const char*)a.a;
    p.w = (const uint16_t*)a.b;
    p.y = (char*)a.out;
    p.ends = a.ends;
    p.x_pitch = a.a_stride * 2;
    p.T = a.T;
    p.K = (int)(fwd ? a.K : a.N);
    p.N = (int)(fwd ? a.N : a.K);
    p.across = !fwd;
    return a.in_bf16 ? narrow_rows<true>(p, st) : narrow_rows<false>(p, st);
}

}  // namespace kdw
