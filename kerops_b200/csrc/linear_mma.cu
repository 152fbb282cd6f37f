// Channel-mixing products of ragged row groups: forward, input gradient, weight gradient (16-bit operands) and the
// 8-bit integer product with a scale per row and per output channel.
#include <limits.h>
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "../../include/kdw.h"
#include "linear_core.cuh"
#include "linear_plan.h"

namespace kdw {

// ------------------------------------------------------------------------------------------------------------------
// The product kernel.  One persistent CTA per SM:
//   warp 2       finds the CTA's units and hands their descriptions to the others through a ring in shared memory
//   warp 0       loads operand tiles with TMA into a ring of stages
//   warp 1       issues the tensor-core products into accumulators in tensor memory
//   warps 4-11 and 12-19  take finished accumulators in turn and bring them to memory while the next tiles are being
//                multiplied (eight warps to an accumulator: a warp reads 32 of its lanes and every other 32 of its columns)
//   warp 3       clears the output rows behind the last group
//   M side: weights (row products; stored with the contraction contiguous for the forward pass, across it for the input
//           gradient) or the gradient's rows, transposed (weight gradient).  N side: rows, or their transpose.
//   PAIR: two CTAs of a cluster share a 256 x BN tile.  Each loads its 128 of M and half of N; the tensor cores of both
//         read both halves of N, so a byte that enters shared memory is used for twice the products (a 128 x 256 tile of
//         one CTA is bound by shared memory: 768 cycles to a stage where the products take 512).  CTA 0 waits for the
//         loads of both and issues the products.
// Large products are bound by the tensor cores (87 % of their cycles busy on 16384 rows of 8 groups, 2048 -> 4096): 18944 x
// 4096 -> 2048 in bf16 takes 204-212 us on different boards, 1500-1560 TFLOP/s (the library's product beside 209 and 212: 204, 205);
// 8192 x 4096 -> 8192 in 8-bit integers 165-173 us, 3180-3330 TOP/s.
// Many small groups are bound by their weights' bytes (64 groups of about 8 rows, 2048 -> 1024: 46 us,
// 0.90 of the measured bandwidth), short contractions by bringing the results to memory (18944 x 64 -> 2048: 21 us; with
// eight warps instead of sixteen and 16-byte pieces instead of transposing matrix stores 26 us).
// Tried and left: asking L2 for the next unit's boxes ahead of their loads (the TMA unit does twice the work: 430 instead of
// 385 us on 32768 rows of 16 groups, 2048 -> 4096), or for its first blocks alone (no difference).
// ------------------------------------------------------------------------------------------------------------------
template <int OP_, bool I8_, int BN_, bool PAIR_>
struct LCfg {
    static constexpr bool I8 = I8_, WGRAD = OP_ == LIN_WGRAD, PAIR = PAIR_;
    static constexpr bool A_ACROSS = OP_ != LIN_FWD, B_ACROSS = WGRAD;  // memory rows run across the contraction
    static constexpr int BN = BN_;
    static constexpr int LOAD_N = PAIR ? BN / 2 : BN;  // of the N side, what a CTA loads
    static constexpr int THREADS = 640;
    static constexpr int A_BYTES = kLinTileM * kLinSpan;
    static constexpr int B_BYTES = LOAD_N * kLinSpan;
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGING = 16 * (1024 + (I8 ? 128 : 0));  // 16 rows of 64 bytes for each warp, and its rows' scales
    static constexpr int STAGES = (232448 - 1024 - STAGING - (int)sizeof(LinTable) - 768) / STAGE;
    static constexpr int ACCS = BN == 256 ? 2 : 4;
    static constexpr int TMEM_COLS = ACCS * BN;
    static constexpr int UNITS = 4;  // descriptions on their way
    static constexpr int BARS = 3 * STAGES + 2 * ACCS + 1 + 2 * UNITS;
    static constexpr int SMEM = 1024 + STAGES * STAGE + STAGING + UNITS * (int)sizeof(LinUnit) + (int)sizeof(LinTable) + BARS * 8 + 16;
    static constexpr int K_ELEMS = I8 ? 128 : 64;  // contraction steps of a stage
    static_assert(LOAD_N >= 64 && TMEM_COLS >= 32 && TMEM_COLS <= 512, "");
    static_assert(SMEM <= 232448 && BARS * 8 + 16 + UNITS * (int)sizeof(LinUnit) <= 768, "");
};

// 16 staged rows of 64 bytes; the 16-byte pieces of a row change places so that neither columns nor rows of pieces meet in
// a bank.
__device__ __forceinline__ int staged(int row, int piece) { return row * 64 + ((piece ^ (row >> 1)) & 3) * 16; }

// Writes the first `rows` of 16 staged rows of `cols` (<= 32) values of one warp to memory.
__device__ __forceinline__ void store_staged(const char* stage, char* dst, long long dst_pitch, int rows, int cols, bool vec,
                                             int lane) {
    if (vec) {  // 16-byte pieces, four lanes to a row
        const int c = lane & 3, r = lane >> 2;
        const uint4 v0 = *reinterpret_cast<const uint4*>(stage + staged(r, c));
        const uint4 v1 = *reinterpret_cast<const uint4*>(stage + staged(r + 8, c));
        dst += r * dst_pitch + c * 16;
        if (r < rows && c * 8 < cols) *reinterpret_cast<uint4*>(dst) = v0;
        if (r + 8 < rows && c * 8 < cols) *reinterpret_cast<uint4*>(dst + 8 * dst_pitch) = v1;
    } else if (lane < cols) {
        for (int r = 0; r < (rows < 16 ? rows : 16); ++r)
            *reinterpret_cast<uint16_t*>(dst + r * dst_pitch + lane * 2) =
                *reinterpret_cast<const uint16_t*>(stage + staged(r, lane >> 3) + (lane & 7) * 2);
    }
}

// Clears the output rows that belong to no group: every CTA takes its share.
__device__ __forceinline__ void clear_rows(const LinParams& p, int first_row, int tid, int nthreads) {
    const long long begin = (long long)first_row * p.out_cols * 2, end = (long long)p.T * p.out_cols * 2;
    char* out = reinterpret_cast<char*>(p.out);
    const long long head = begin + ((16 - ((uintptr_t)(out + begin) & 15)) & 15);
    const long long id = (long long)blockIdx.x * nthreads + tid, n = (long long)gridDim.x * nthreads;
    if (head >= end) {
        for (long long i = begin + 2 * id; i < end; i += 2 * n) *reinterpret_cast<uint16_t*>(out + i) = 0;
        return;
    }
    const long long tail = head + (end - head) / 16 * 16;
    for (long long i = begin + 2 * id; i < head; i += 2 * n) *reinterpret_cast<uint16_t*>(out + i) = 0;
    for (long long i = head + 16 * id; i < tail; i += 16 * n) *reinterpret_cast<uint4*>(out + i) = make_uint4(0, 0, 0, 0);
    for (long long i = tail + 2 * id; i < end; i += 2 * n) *reinterpret_cast<uint16_t*>(out + i) = 0;
}

// Panels of 64 columns of a tile `width` wide that hold any of the `left` columns from its first on.
__device__ __forceinline__ int boxes_inside(int left, int width) {
    const int n = (left + 63) >> 6;
    return n < 0 ? 0 : n > width / 64 ? width / 64 : n;
}

// What a CTA loads for a unit.  Boxes wholly beyond the output are not loaded: what is left in their place reaches only
// rows and columns of the accumulator that are not stored.
template <class C>
struct LinLoad {
    int g, c0, t0, kb, ke, k_row, k_rows, a_boxes, b_boxes;
    uint32_t bytes;
    __device__ __forceinline__ LinLoad(const LinParams& p, const LinUnit& w, uint32_t rank) {
        g = w.g;
        kb = w.kb;
        ke = w.ke;
        k_row = w.k_row;
        k_rows = w.k_rows;
        c0 = w.c0 + (int)rank * kLinTileM;
        t0 = w.t0 + (int)rank * (C::WGRAD ? C::LOAD_N : w.width >> 1);
        a_boxes = C::A_ACROSS ? boxes_inside((C::WGRAD ? p.out_rows : p.out_cols) - c0, kLinTileM) : 1;
        b_boxes = C::WGRAD ? boxes_inside(p.out_cols - t0, C::LOAD_N) : 1;
        bytes = (C::A_ACROSS ? a_boxes * 8192 : C::A_BYTES) + (C::WGRAD ? b_boxes * 8192 : C::B_BYTES);
    }
    __device__ __forceinline__ void load_a(const CUtensorMap* ma, int k, uint32_t a, uint32_t bar) const {
        if constexpr (C::WGRAD) {
#pragma unroll
            for (int j = 0; j < kLinTileM / 64; ++j)
                if (j < a_boxes) tma_load_2d<C::PAIR>(a + j * 8192, ma, bar, c0 + j * 64, k_row + k * 64);
        } else if constexpr (C::A_ACROSS) {
#pragma unroll
            for (int j = 0; j < kLinTileM / 64; ++j)
                if (j < a_boxes) tma_load_3d<C::PAIR>(a + j * 8192, ma, bar, c0 + j * 64, k * 64, g);
        } else {
            tma_load_3d<C::PAIR>(a, ma, bar, k * C::K_ELEMS, c0, g);
        }
    }
    __device__ __forceinline__ void load_b(const CUtensorMap* mb, int k, uint32_t b, uint32_t bar) const {
        if constexpr (C::WGRAD) {
#pragma unroll
            for (int j = 0; j < C::LOAD_N / 64; ++j)
                if (j < b_boxes) tma_load_2d<C::PAIR>(b + j * 8192, mb, bar, t0 + j * 64, k_row + k * 64);
        } else {
            tma_load_2d<C::PAIR>(b, mb, bar, k * C::K_ELEMS, t0);
        }
    }
};

template <bool I8>
__device__ __forceinline__ void add_share(uint4& sum, const uint4& v) {
    if (I8) {
        sum.x += v.x;
        sum.y += v.y;
        sum.z += v.z;
        sum.w += v.w;
    } else {
        sum.x = __float_as_uint(__uint_as_float(sum.x) + __uint_as_float(v.x));
        sum.y = __float_as_uint(__uint_as_float(sum.y) + __uint_as_float(v.y));
        sum.z = __float_as_uint(__uint_as_float(sum.z) + __uint_as_float(v.z));
        sum.w = __float_as_uint(__uint_as_float(sum.w) + __uint_as_float(v.w));
    }
}

// The CTAs of a cluster add their parts of a tile (of their 128 of its M): CTA `part` takes its share of the column
// quadruples, in the order of the parts.
template <class C, int PARTS>
__device__ __forceinline__ void add_parts(const LinParams& p, const LinUnit& w, int part, uint32_t rank, uint32_t tile) {
    const int m = threadIdx.x & 127, c = w.c0 + (int)rank * kLinTileM + m;
    const int cols = C::WGRAD ? (p.out_cols - w.t0 < C::BN ? p.out_cols - w.t0 : C::BN) : w.rows;
    const bool live = c < (C::WGRAD ? p.out_rows : p.out_cols);
    float cs = 1.f;
    if (C::I8 && live) cs = __ldg(p.col_scale + (long long)w.g * p.out_cols + c);
    uint16_t* out = reinterpret_cast<uint16_t*>(p.out) +
                    (C::WGRAD ? ((long long)w.g * p.out_rows + c) * p.out_cols + w.t0 : (long long)w.t0 * p.out_cols + c);
    const int quads = (cols + 3) >> 2, end = quads * (part + 1) / PARTS;
    uint32_t src[PARTS];
#pragma unroll
    for (int k = 0; k < PARTS; ++k) src[k] = cluster_addr(tile + m * 16, C::PAIR ? 2 * k + rank : k);
    for (int j = quads * part / PARTS + (threadIdx.x >> 7); j < end; j += C::THREADS / 128) {
        uint4 v[PARTS];
#pragma unroll
        for (int k = 0; k < PARTS; ++k) v[k] = cluster_load(src[k] + j * kLinTileM * 16);
#pragma unroll
        for (int k = 1; k < PARTS; ++k) add_share<C::I8>(v[0], v[k]);
        if (!live) continue;
        const uint32_t s[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
        float f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[e] = __uint_as_float(s[e]);
            if (C::I8) f[e] = 4 * j + e < cols ? RowScale(__ldg(p.row_scale + w.t0 + 4 * j + e)).of((int)s[e], cs) : 0.f;
        }
        const uint32_t lo = pack2(f[0], f[1], p.out_bf16), hi = pack2(f[2], f[3], p.out_bf16);
        if (C::WGRAD && p.out_vec) {
            *reinterpret_cast<uint2*>(out + 4 * j) = make_uint2(lo, hi);  // rows are multiples of 8 values
        } else {
            const long long next = C::WGRAD ? 1 : p.out_cols;
            uint16_t* o = out + 4 * j * next;
            if (4 * j < cols) o[0] = (uint16_t)lo;
            if (4 * j + 1 < cols) o[next] = (uint16_t)(lo >> 16);
            if (4 * j + 2 < cols) o[2 * next] = (uint16_t)hi;
            if (4 * j + 3 < cols) o[3 * next] = (uint16_t)(hi >> 16);
        }
    }
}

// The next unit's description; lanes of a warp take it together and give the place back.
__device__ __forceinline__ bool take_unit(LinUnit& w, const LinUnit* ring, uint32_t full, uint32_t empty, int& slot, uint32_t& phase,
                                          int slots, int lane, const LinParams& p) {
    const bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(full + 8 * slot, phase, p.limit_ns));
    if (!ok) {
        if (lane == 0) atomicExch(p.status, (int)KDW_STATUS_TMA_TIMEOUT);
        return false;
    }
    w = ring[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + 8 * slot);
    if (++slot == slots) {
        slot = 0;
        phase ^= 1;
    }
    return w.u >= 0;
}

template <class C>
__global__ __launch_bounds__(C::THREADS, 1) void linear_kernel(const __grid_constant__ CUtensorMap map_a,
                                                               const __grid_constant__ CUtensorMap map_b,
                                                               const __grid_constant__ LinParams p) {
    extern __shared__ char smem_raw[];
    char* const base = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    char* const staging = base + C::STAGES * C::STAGE;
    LinUnit* const ring = reinterpret_cast<LinUnit*>(staging + C::STAGING);
    LinTable* const tab = reinterpret_cast<LinTable*>(ring + C::UNITS);
    uint64_t* const bars = reinterpret_cast<uint64_t*>(tab + 1);
    uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(bars + C::BARS);
    const uint32_t full = smem_u32(bars), empty = full + 8 * C::STAGES, partly = empty + 8 * C::STAGES,
                   acc_full = partly + 8 * C::STAGES, acc_empty = acc_full + 8 * C::ACCS, drain = acc_empty + 8 * C::ACCS,
                   unit_full = drain + 8, unit_empty = unit_full + 8 * C::UNITS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // Few tiles: a cluster takes one tile, its CTAs (pairs) a part of the contraction each, and adds the parts at the end.
    const bool shared_tile = p.splits > 1;
    const uint32_t in_cluster = C::PAIR || shared_tile ? cluster_rank() : 0;
    const uint32_t rank = C::PAIR ? in_cluster & 1 : 0, leader = in_cluster & ~1u, both = 3u << leader;  // of the pair
    const int part = !shared_tile ? 0 : C::PAIR ? (int)(in_cluster >> 1) : (int)in_cluster;
    const int ctas = (C::PAIR ? 2 : 1) * p.splits;  // that share a tile

    if (warp == 0 && lane == 0) {
        prefetch_tmap(&map_a);
        prefetch_tmap(&map_b);
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(full + 8 * i, C::PAIR ? 2 : 1);
            mbar_init(empty + 8 * i, 1);
            mbar_init(partly + 8 * i, 1);
        }
        for (int i = 0; i < C::ACCS; ++i) {
            mbar_init(acc_full + 8 * i, 1);
            mbar_init(acc_empty + 8 * i, C::PAIR ? 16 : 8);
        }
        mbar_init(drain, 1);
        for (int i = 0; i < C::UNITS; ++i) {
            mbar_init(unit_full + 8 * i, 1);
            mbar_init(unit_empty + 8 * i, 18);  // warps 0, 1 and 4-19
        }
        mbar_fence_init();
    } else if (warp == 1) {
        tmem_alloc<C::PAIR>(smem_u32(s_tmem), C::TMEM_COLS);
    }
    // Operands, scales and `ends` may be the work of the kernel before this one.  EARLY: that kernel is this call's own (it
    // quantises the rows), and it let this one start only after its own wait, so whatever came before it has completed: only
    // the rows and their scales have to be waited for, and the first weights are loaded while they are being made (64 rows,
    // 4096 -> 8192: 12.0 us instead of 12.9, 4096 rows of 32 groups, 1024 -> 2048: 24.4 instead of 25.1).
    const bool early = !C::WGRAD && p.early;
    if (!early) {
        grid_dependency_wait();
        grid_launch_dependents();
    }
    if (warp == 2) lin_build_table(p, tab->row, tab->unit, lane);
    tc_fence_before();
    __syncthreads();
    if (C::PAIR) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    int slot = 0;  // of the ring of units
    uint32_t slot_phase = 0;
    LinUnit w;

    if (warp == 0) {
        int loads = 0, stage = 0;
        uint32_t phase = 0, partly_stages = 0, partly_phase = 0;  // stages whose last load reported to `partly`, and its parity
        bool ok = true;
        if (early && p.stop_after >= 0) grid_dependency_wait();
        while (ok && take_unit(w, ring, unit_full, unit_empty, slot, slot_phase, C::UNITS, lane, p)) {
            const LinLoad<C> l(p, w, rank);
            int ahead = 0;
            if (early && loads == 0 && p.stop_after < 0) {
                // the ring is empty: weights for all of it, then the wait, then the rows beside them
                const int n = l.ke - l.kb < C::STAGES ? l.ke - l.kb : C::STAGES;
                for (int h = 0; h < 2; ++h) {
                    if (h == 1) grid_dependency_wait();
                    if (elect_one())
                        for (int i = 0; i < n; ++i) {
                            const uint32_t a = smem_u32(base) + i * C::STAGE;
                            const uint32_t bar = rank == 0 ? full + 8 * i : cluster_addr(full + 8 * i, leader);
                            if (h == 1) {
                                l.load_b(&map_b, l.kb + i, a + C::A_BYTES, bar);
                                continue;
                            }
                            if (rank == 0)
                                mbar_expect_tx(bar, l.bytes);
                            else
                                cluster_expect_tx(bar, l.bytes);
                            l.load_a(&map_a, l.kb + i, a, bar);
                        }
                    __syncwarp();
                }
                loads = ahead = n;
                stage = n == C::STAGES ? 0 : n;
                phase = n == C::STAGES ? 1 : 0;
            }
            for (int k = l.kb + ahead; k < l.ke; ++k) {
                if (p.stop_after >= 0 && loads >= p.stop_after) {
                    ok = false;
                    break;
                }
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(empty + 8 * stage, phase ^ 1, p.limit_ns));
                if (!ok) {
                    if (lane == 0) atomicExch(p.status, (int)KDW_STATUS_TMA_TIMEOUT);
                    break;
                }
                const bool own = C::PAIR && C::WGRAD && rank != 0 && l.k_rows - k * 64 < 64;
                partly_stages = own ? partly_stages | 1u << stage : partly_stages & ~(1u << stage);
                partly_phase ^= (uint32_t)own << stage;
                if (elect_one()) {
                    const uint32_t a = smem_u32(base) + stage * C::STAGE, b = a + C::A_BYTES;
                    uint32_t bar = full + 8 * stage;
                    if (rank == 0) {
                        mbar_expect_tx(bar, l.bytes);
                    } else if (own) {
                        bar = partly + 8 * stage;  // warp 1 clears the rows beyond the share first and then tells CTA 0
                        mbar_expect_tx(bar, l.bytes);
                    } else {
                        bar = cluster_addr(bar, leader);  // CTA 0 waits for the loads of both
                        cluster_expect_tx(bar, l.bytes);
                    }
                    l.load_a(&map_a, k, a, bar);
                    l.load_b(&map_b, k, b, bar);
                }
                __syncwarp();
                ++loads;
                if (++stage == C::STAGES) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
        // A CTA leaves only when its last copies have landed and the products' reports on its stages have arrived.  CTA 0 of a
        // pair sends those to both CTAs and waits for its own last one in warp 1.  CTA 1's copies report to CTA 0, but for
        // blocks that its warp 1 clears in part.
        const int last = loads < C::STAGES ? loads : C::STAGES;
        bool ok_last = true;
        for (int i = 0; i < last; ++i) {
            if (stage == 0) {
                stage = C::STAGES;
                phase ^= 1;
            }
            --stage;
            if (rank == 0) {
                ok_last &= mbar_wait_bounded(full + 8 * stage, phase, p.limit_ns);
            } else {
                if (partly_stages >> stage & 1) ok_last &= mbar_wait_bounded(partly + 8 * stage, partly_phase >> stage & 1 ^ 1, p.limit_ns);
                ok_last = ok_last && mbar_wait_bounded(empty + 8 * stage, phase, p.limit_ns);
            }
        }
        if (!ok_last) atomicExch(p.status, (int)KDW_STATUS_TMA_TIMEOUT);
        __syncwarp();
    } else if (warp == 1) {
        int stage = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0, partly_phase = 0;
        bool ok = true;
        while (ok && take_unit(w, ring, unit_full, unit_empty, slot, slot_phase, C::UNITS, lane, p)) {
            if (w.kb == w.ke) continue;
            if (rank == 0) {
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(acc_empty + 8 * acc, acc_phase ^ 1, p.limit_ns));
                if (!ok) break;
                tc_fence_after();
            }
            const uint32_t d = tmem + acc * C::BN, idesc = p.idesc | (uint32_t)(w.width >> 3) << 17;
            for (int k = w.kb; k < w.ke; ++k) {
                char* const sa = base + stage * C::STAGE;
                // rows beyond the share are another group's (or of no group): their products must vanish even where
                // one of the factors is a NaN or an infinity, so both operands are cleared
                const int valid = C::WGRAD ? w.k_rows - k * 64 : 64;
                if (rank == 0 || valid < 64) {
                    // (CTA 0 also waits for what CTA 1 cleared: ordinary writes that the products are to read)
                    ok = rank != 0 ? mbar_wait_bounded(partly + 8 * stage, partly_phase >> stage & 1, p.limit_ns)
                         : C::PAIR && valid < 64 ? cluster_wait_bounded(full + 8 * stage, phase, p.limit_ns)
                                                 : mbar_wait_bounded(full + 8 * stage, phase, p.limit_ns);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                }
                if (C::WGRAD && valid < 64) {
                    for (int i = valid * 8 + lane; i < 512; i += 32)
#pragma unroll
                        for (int j = 0; j < C::STAGE / 8192; ++j)
                            *reinterpret_cast<uint4*>(sa + j * 8192 + i * 16) = make_uint4(0, 0, 0, 0);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (rank != 0) {
                        partly_phase ^= 1u << stage;  // one parity bit per stage
                        if (lane == 0) cluster_release_arrive(cluster_addr(full + 8 * stage, leader));
                    }
                }
                if (rank == 0) {
                    tc_fence_after();
                    const uint32_t el = elect_one();
                    const uint64_t da = smem_desc(smem_u32(sa), C::A_ACROSS);
                    const uint64_t db = smem_desc(smem_u32(sa) + C::A_BYTES, C::B_ACROSS);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        tc_mma<C::I8, C::PAIR>(el, d, da + i * (C::A_ACROSS ? 2048 >> 4 : 32 >> 4),
                                               db + i * (C::B_ACROSS ? 2048 >> 4 : 32 >> 4), idesc, k > w.kb || i > 0);
                    tc_commit<C::PAIR>(el, empty + 8 * stage, both);
                    if (k + 1 == w.ke) tc_commit<C::PAIR>(el, acc_full + 8 * acc, both);
                }
                if (++stage == C::STAGES) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (++acc == C::ACCS) {
                acc = 0;
                acc_phase ^= 1;
            }
        }
        if (!ok && lane == 0) atomicExch(p.status, (int)KDW_STATUS_TMA_TIMEOUT);
        // products in flight still read shared memory and write tensor memory
        if (rank == 0) {
            tc_commit<C::PAIR>(elect_one(), drain, both);
            if (!mbar_wait_bounded(drain, 0, p.limit_ns)) atomicExch(p.status, (int)KDW_STATUS_TMA_TIMEOUT);
        }
        __syncwarp();
    } else if (warp == 2) {
        const int units = tab->unit[p.E];
        const int first = blockIdx.x / ctas;
        const int step = shared_tile ? units : gridDim.x / ctas;  // a shared tile is the cluster's only one
        for (int u = first;; u += step) {
            const bool more = u < units;
            if (more)
                w = lin_unit(p, tab->row, tab->unit, u, part);
            else
                w.u = -1;
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(unit_empty + 8 * slot, slot_phase ^ 1, p.limit_ns))) {
                if (lane == 0) atomicExch(p.status, (int)KDW_STATUS_TMA_TIMEOUT);
                break;
            }
            if (lane == 0) {
                ring[slot] = w;
                mbar_arrive(unit_full + 8 * slot);
            }
            __syncwarp();
            if (++slot == C::UNITS) {
                slot = 0;
                slot_phase ^= 1;
            }
            if (!more) break;
        }
    } else if (warp == 3) {
        if (early) {
            grid_dependency_wait();
            grid_launch_dependents();
        }
        if (!C::WGRAD) clear_rows(p, tab->row[p.E], lane, 32);
        if (p.table && blockIdx.x == 0)
            for (int i = lane; i <= p.E; i += 32) {
                p.table[i] = tab->row[i];
                p.table[p.E + 1 + i] = tab->unit[i];
            }
    } else {
        const int q = warp & 3, turn = (warp - 4) >> 3, odd = (warp >> 2) & 1 ^ 1;
        char* const stg = staging + (warp - 4) * 1024;
        if (early) grid_dependency_wait();
        int acc = 0, count = 0;  // accumulators used so far: the two groups of warps take them in turn
        uint32_t acc_phase = 0;
        while (take_unit(w, ring, unit_full, unit_empty, slot, slot_phase, C::UNITS, lane, p)) {
            const bool any = w.ke > w.kb;
            const bool mine = (count & 1) == turn;
            if (any) ++count;
            if (!mine) {
                if (any && ++acc == C::ACCS) {
                    acc = 0;
                    acc_phase ^= 1;
                }
                continue;
            }
            if (any) {
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(acc_full + 8 * acc, acc_phase, p.limit_ns))) {
                    if (lane == 0) atomicExch(p.status, (int)KDW_STATUS_TMA_TIMEOUT);
                    break;
                }
                tc_fence_after();
            }
            const uint32_t d = tmem + acc * C::BN + ((uint32_t)(q * 32) << 16);
            const int c0 = w.c0 + (int)rank * kLinTileM + q * 32;  // of this warp's 32 lanes
            const long long pitch = (long long)p.out_cols * 2;
            if ((C::WGRAD && p.partial && !(w.whole && p.fold == 1)) || shared_tile) {
                // a share of a tile: column quadruples of a lane side by side over the lanes, in memory or, where the CTAs
                // of a cluster add them, in the ring of stages (the tile is the CTA's only one: its loads have been used)
                uint4* out = shared_tile ? reinterpret_cast<uint4*>(base)
                                         : reinterpret_cast<uint4*>(p.partial) + ((long long)w.u * (C::PAIR ? 2 : 1) + rank) * (C::BN / 4) * kLinTileM;
                out += q * 32 + lane;
#pragma unroll 1
                for (int n = 32 * odd; n < w.width; n += 64) {
                    uint32_t v[32];
                    if (any) {
                        tmem_load_32(d + n, v);
                        tmem_wait(v);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = 0u;
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        out[(long long)((n + i) / 4) * kLinTileM] = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                }
            } else if constexpr (C::WGRAD) {
                // lanes are output rows, accumulator columns output columns
                char* out = reinterpret_cast<char*>(p.out) + lin_out_offset((long long)w.g * p.out_rows + c0, 0, p.out_cols);
                const int rows = p.out_rows - c0;
#pragma unroll 1
                for (int n = 32 * odd; n < C::BN; n += 64) {
                    int cols = p.out_cols - w.t0 - n;
                    if (cols <= 0 || rows <= 0) break;
                    cols = cols > 32 ? 32 : cols;
                    uint32_t v[32];
                    if (any) {
                        tmem_load_32(d + n, v);
                        tmem_wait(v);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = 0u;
                    }
                    uint4 o[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        o[i].x = pack2(__uint_as_float(v[8 * i]), __uint_as_float(v[8 * i + 1]), p.out_bf16);
                        o[i].y = pack2(__uint_as_float(v[8 * i + 2]), __uint_as_float(v[8 * i + 3]), p.out_bf16);
                        o[i].z = pack2(__uint_as_float(v[8 * i + 4]), __uint_as_float(v[8 * i + 5]), p.out_bf16);
                        o[i].w = pack2(__uint_as_float(v[8 * i + 6]), __uint_as_float(v[8 * i + 7]), p.out_bf16);
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (lane >> 4 == h) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(stg + staged(lane & 15, i)) = o[i];
                        }
                        __syncwarp();
                        store_staged(stg, out + 16 * h * pitch + (long long)(w.t0 + n) * 2, pitch, rows - 16 * h, cols, p.out_vec, lane);
                        __syncwarp();
                    }
                }
            } else {
                // lanes are output channels, accumulator columns rows of the output: blocks are transposed on their way
                // into shared memory
                int cols = p.out_cols - c0;
                cols = cols > 32 ? 32 : cols;
                float cs[4];  // of channels l / 4 + 8 i
                float* const srs = reinterpret_cast<float*>(staging + 16 * 1024) + (warp - 4) * 32;
                if constexpr (C::I8) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int c = (lane >> 2) + 8 * i;
                        cs[i] = c < cols ? __ldg(p.col_scale + (long long)w.g * p.out_cols + c0 + c) : 0.f;
                    }
                }
                char* out = reinterpret_cast<char*>(p.out) + lin_out_offset(w.t0 + 32ll * odd, c0, p.out_cols);
                const uint32_t mat = smem_u32(stg) + staged(lane & 7, lane >> 3);
#pragma unroll 1
                for (int n = 32 * odd; n < w.rows; n += 64) {
                    if (cols <= 0) break;
                    const int rows = w.rows - n;
                    bool large = false;
                    if constexpr (C::I8) {
                        const float s = lane < rows ? __ldg(p.row_scale + w.t0 + n + lane) : 0.f;
                        srs[lane] = s;
                        large = __any_sync(0xffffffffu, RowScale::is_large(s));
                        __syncwarp();
                    }
                    uint32_t v[32];
                    tmem_load_frag(d + n, v);
                    tmem_wait(v);
                    // LARGE: RowScale's third product, which blocks of ordinary rows go without (8 M int8 rows, 64 -> 64: 573 us,
                    // 617 with it everywhere)
                    auto write = [&](auto LARGE) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const int j = 2 * h + k;
                                float2 rs = make_float2(1.f, 1.f);
                                if constexpr (C::I8) rs = *reinterpret_cast<const float2*>(srs + 8 * j + 2 * (lane & 3));
                                uint32_t o[4];
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const uint32_t a = v[16 * (i >> 1) + 4 * j + 2 * (i & 1)], b = v[16 * (i >> 1) + 4 * j + 2 * (i & 1) + 1];
                                    if constexpr (C::I8 && decltype(LARGE)::value)
                                        o[i] = pack2(RowScale(rs.x).of((int)a, cs[i]), RowScale(rs.y).of((int)b, cs[i]), p.out_bf16);
                                    else if constexpr (C::I8)
                                        o[i] = pack2((float)(int)a * rs.x * cs[i], (float)(int)b * rs.y * cs[i], p.out_bf16);
                                    else
                                        o[i] = pack2(__uint_as_float(a), __uint_as_float(b), p.out_bf16);
                                }
                                store_matrix_trans(mat + k * 512, o[0], o[1], o[2], o[3]);
                            }
                            __syncwarp();
                            store_staged(stg, out + 16 * h * pitch, pitch, rows - 16 * h, cols, p.out_vec, lane);
                            __syncwarp();
                        }
                    };
                    if (large)
                        write(std::true_type());
                    else
                        write(std::false_type());
                    out += 64 * pitch;
                }
            }
            if (any) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (C::PAIR)
                        cluster_arrive(cluster_addr(acc_empty + 8 * acc, leader));
                    else
                        mbar_arrive(acc_empty + 8 * acc);
                }
                if (++acc == C::ACCS) {
                    acc = 0;
                    acc_phase ^= 1;
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (C::PAIR || shared_tile) cluster_sync();
    tc_fence_after();
    // CTA 0's last report goes to both CTAs, and it has waited for its own: CTA 1 leaves when the other has arrived too
    if (warp == 1) {
        if (C::PAIR && rank != 0 && !mbar_wait_bounded(drain, 0, p.limit_ns)) atomicExch(p.status, (int)KDW_STATUS_TMA_TIMEOUT);
        __syncwarp();  // (lanes may leave the wait one after the other; what follows is executed by the warp as one)
        tmem_free<C::PAIR>(tmem, C::TMEM_COLS);
    }
    if (shared_tile) {
        if (early) grid_dependency_wait();  // (of the warps that have not waited)
        w = ring[0];
        if (w.u >= 0) {
            if (p.splits == 2)
                add_parts<C, 2>(p, w, part, rank, smem_u32(base));
            else if (p.splits == 4)
                add_parts<C, 4>(p, w, part, rank, smem_u32(base));
            else if constexpr (!C::PAIR)
                add_parts<C, 8>(p, w, part, rank, smem_u32(base));
        }
        cluster_sync();  // the others may still read this CTA's part
    }
}

// Weight gradient: adds the shares of the tiles that have several, and rounds once.  A CTA takes four columns of 256 / L
// rows of a tile; L threads to a row add every L-th share each, and their sums are added in order: the same bits every call.
template <int L>
__global__ __launch_bounds__(256) void linear_sum_kernel(const __grid_constant__ LinParams p) {
    constexpr int R = 256 / L;  // rows at a time
    __shared__ uint4 s[L][R];
    const int r = threadIdx.x % R, l = threadIdx.x / R;
    const int quads = p.bn / 4, blocks = p.tile_m / R * quads;  // of a tile
    const int tiles = p.m_tiles * p.n_tiles;                    // of a group
    const int* row = p.table;
    const int* unit = p.table + p.E + 1;
    grid_dependency_wait();
    grid_launch_dependents();
    for (int i = blockIdx.x; i < p.E * tiles * blocks; i += gridDim.x) {
        const int t = i / blocks, part = i - t * blocks, g = t / tiles;
        const int shares = lin_shares(p, row[g + 1] - row[g]);
        if (shares == 1) continue;
        const int u = unit[g] + t - g * tiles;
        const LinUnit w = lin_unit(p, row, unit, u);
        const int n = part % quads * 4, m = part / quads * R + r;  // of the tile
        if (w.t0 + n >= p.out_cols) continue;
        const long long halves = p.tile_m / kLinTileM, step = tiles * halves * quads * kLinTileM;
        const uint4* src = reinterpret_cast<const uint4*>(p.partial) +
                           ((u * halves + m / kLinTileM) * quads + n / 4) * kLinTileM + m % kLinTileM;
        uint4 sum = make_uint4(0, 0, 0, 0);
#pragma unroll 8
        for (int k = l; k < shares; k += L) add_share<false>(sum, __ldcg(src + k * step));
        __syncthreads();
        s[l][r] = sum;
        __syncthreads();
        if (l != 0 || w.c0 + m >= p.out_rows) continue;
#pragma unroll
        for (int k = 1; k < L; ++k) add_share<false>(sum, s[k][r]);
        const uint32_t v[4] = {sum.x, sum.y, sum.z, sum.w};
        uint16_t* out = reinterpret_cast<uint16_t*>(p.out) + ((long long)g * p.out_rows + w.c0 + m) * p.out_cols + w.t0 + n;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (w.t0 + n + j < p.out_cols) out[j] = (uint16_t)pack2(__uint_as_float(v[j]), 0.f, p.out_bf16);
    }
}

// The weight gradient from a folded product (see linear_plan): the sum over the shares and over the f blocks on the
// diagonal.  A CTA adds four neighbouring values of a row, its threads the (share, block) pairs, in a fixed order.
__global__ __launch_bounds__(256) void linear_fold_kernel(const __grid_constant__ LinParams p, int BN, int N, int K) {
    __shared__ float4 s[8];
    const int lane = threadIdx.x & 31, quads = K / 4, tiles = p.m_tiles * p.n_tiles;
    grid_dependency_wait();
    grid_launch_dependents();
    const int shares = p.table[p.E + 1 + p.E] / tiles;
    for (int i = blockIdx.x; i < N * quads; i += gridDim.x) {
        const int n = i / quads, k = (i - n * quads) * 4;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int j = threadIdx.x; j < shares * p.fold; j += 256) {
            const int share = j / p.fold, block = j - share * p.fold;
            const int m = block * N + n, c = block * K + k;
            const int mt = m / p.tile_m, nt = c / BN, band = nt / kLinBand;
            const int wide = p.n_tiles - band * kLinBand < kLinBand ? p.n_tiles - band * kLinBand : kLinBand;
            const long long u = (long long)share * tiles + (p.m_tiles > 1 ? band * kLinBand * p.m_tiles + mt * wide + nt - band * kLinBand : nt);
            const long long half = u * (p.tile_m / kLinTileM) + (m % p.tile_m) / kLinTileM;
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p.partial) + (half * (BN / 4) + (c % BN) / 4) * kLinTileM + m % kLinTileM);
            sum.x += v.x;
            sum.y += v.y;
            sum.z += v.z;
            sum.w += v.w;
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            sum.x += __shfl_xor_sync(0xffffffffu, sum.x, d);
            sum.y += __shfl_xor_sync(0xffffffffu, sum.y, d);
            sum.z += __shfl_xor_sync(0xffffffffu, sum.z, d);
            sum.w += __shfl_xor_sync(0xffffffffu, sum.w, d);
        }
        __syncthreads();
        if (lane == 0) s[threadIdx.x >> 5] = sum;
        __syncthreads();
        if (threadIdx.x < 4) {
            float v = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) v += reinterpret_cast<const float*>(&s[j])[threadIdx.x];
            reinterpret_cast<uint16_t*>(p.out)[(long long)n * K + k + threadIdx.x] = (uint16_t)pack2(v, 0.f, p.out_bf16);
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void pack_rows_kernel(const __grid_constant__ PackRows a, const __grid_constant__ PackRows b,
                                                        const __grid_constant__ PackRows c, int split_b, int split_c) {
    grid_dependency_wait();
    grid_launch_dependents();
    const int cta = blockIdx.x;
    if (cta < split_b)
        pack_rows_part<T>(a, cta, split_b);
    else if (cta < split_c)
        pack_rows_part<T>(b, cta - split_b, split_c - split_b);
    else
        pack_rows_part<T>(c, cta - split_c, gridDim.x - split_c);
}

// ------------------------------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------------------------------
template <class C>
static int launch_product(const LinPlan& pl, const CUtensorMap& ma, const CUtensorMap& mb, const LinParams& p,
                          cudaStream_t st) {
    static KernelSetup setup;
    int sms = 0, occ = 0;
    int rc = setup.get((const void*)linear_kernel<C>, C::THREADS, C::SMEM, &sms, &occ);
    if (rc) return rc;
    const int cluster = (C::PAIR ? 2 : 1) * p.splits;
    const int64_t slots = p.splits > 1 ? INT_MAX : C::PAIR ? sms / 2 : sms;  // shared tiles: a cluster to each, in waves
    const int64_t grid = std::max<int64_t>(1, std::min(pl.max_units, slots)) * cluster;
    KDW_CUDA(launch_overlapping_previous_grid(linear_kernel<C>, dim3((unsigned)grid), dim3(C::THREADS), (size_t)C::SMEM, st, cluster,
                                              ma, mb, p));
    if (p.fold > 1) {
        const int N = pl.out_rows / p.fold, K = pl.out_cols / p.fold;
        const int quads = N * (K / 4);
        KDW_CUDA(launch_overlapping_previous(linear_fold_kernel, (unsigned)std::min(quads, 8 * sms), 256u, st, p, C::BN, N, K));
    } else if (p.partial) {
        const bool many = pl.max_units >= 8 * pl.max_tiles;
        const int64_t blocks = pl.max_tiles * (C::BN / 4) * (p.tile_m / (many ? 32 : 128));
        KDW_CUDA(launch_overlapping_previous(many ? linear_sum_kernel<8> : linear_sum_kernel<2>,
                                             (unsigned)std::min<int64_t>(blocks, 8 * sms), 256u, st, p));
    }
    return 0;
}

template <int OP, bool I8>
static int launch_width(const LinPlan& pl, const CUtensorMap& ma, const CUtensorMap& mb, const LinParams& p,
                        cudaStream_t st) {
    if (pl.tile_m == 256) return launch_product<LCfg<OP, I8, 256, true>>(pl, ma, mb, p, st);
    switch (pl.bn) {
        case 64: return launch_product<LCfg<OP, I8, 64, false>>(pl, ma, mb, p, st);
        case 128: return launch_product<LCfg<OP, I8, 128, false>>(pl, ma, mb, p, st);
        default: return launch_product<LCfg<OP, I8, 256, false>>(pl, ma, mb, p, st);
    }
}

int pack_ctas(const PackRows& r, int esize, int sms) {
    const int64_t want = (r.rows * ((r.cols * (int64_t)esize + 15) / 16) + 255) / 256;
    return (int)std::min<int64_t>(want, 8 * sms);
}

int pack_rows(const PackRows* r, int count, int esize, cudaStream_t st) {
    int sms = 0, rc = device_facts(nullptr, &sms);
    if (rc) return rc;
    const PackRows none = {};
    const PackRows &a = r[0], &b = count > 1 ? r[1] : none, &c = count > 2 ? r[2] : none;
    const int na = pack_ctas(a, esize, sms), nb = pack_ctas(b, esize, sms), nc = pack_ctas(c, esize, sms);
    if (na + nb + nc == 0) return 0;
    KDW_CUDA(launch_overlapping_previous(esize == 2 ? pack_rows_kernel<uint16_t> : pack_rows_kernel<uint8_t>,
                                         (unsigned)(na + nb + nc), 256u, st, a, b, c, na, na + nb));
    return 0;
}

int linear_run(const LinPlan& pl, const LinArgs& a, void* ws, cudaStream_t st) {
    int* status = nullptr;
    int sms = 0, rc = device_facts(&status, &sms);  // (launch_product asks for the SMs itself)
    if (rc) return rc;
    char* w = (char*)ws;
    const void* pa = a.a;
    const void* pb = a.b;
    int64_t sa = a.a_stride * pl.fold, sb = a.b_stride * pl.fold;
    if (pl.pack_a || pl.pack_b) {
        const PackRows r[2] = {{pa, w + pl.off_a, pl.pack_a ? pl.a_rows : 0, sa, pl.a_pitch, (int)pl.a_cols},
                               {pb, w + pl.off_b, pl.pack_b ? pl.b_rows : 0, sb, pl.b_pitch, (int)pl.b_cols}};
        rc = pack_rows(r, 2, pl.esize, st);
        if (rc) return rc;
        if (pl.pack_a) {
            pa = w + pl.off_a;
            sa = pl.a_pitch;
        }
        if (pl.pack_b) {
            pb = w + pl.off_b;
            sb = pl.b_pitch;
        }
    }
    LinParams p;
    memset(&p, 0, sizeof(p));
    p.ends = a.ends;
    p.T = (int)(a.T / pl.fold);
    p.fold = pl.fold;
    p.E = (int)a.E;
    p.wgrad = a.op == LIN_WGRAD;
    p.tile_m = pl.tile_m;
    p.bn = pl.bn;
    p.bn_log = pl.bn == 256 ? 8 : pl.bn == 128 ? 7 : 6;
    p.m_tiles = pl.m_tiles;
    p.n_tiles = pl.n_tiles;
    p.out_rows = pl.out_rows;
    p.out_cols = pl.out_cols;
    p.k_blocks = pl.k_blocks;
    p.splits = pl.splits;
    p.chunk = pl.chunk;
    p.out = a.out;
    p.partial = pl.off_partial >= 0 ? (float*)(w + pl.off_partial) : nullptr;
    p.table = pl.off_partial >= 0 ? (int*)(w + pl.off_table) : nullptr;
    p.row_scale = a.row_scale;
    p.col_scale = a.col_scale;
    p.out_bf16 = a.out_bf16;
    p.out_vec = (pl.out_cols % 8 == 0) && ((uintptr_t)a.out & 15) == 0;
    p.status = status;
    const WaitTest wt = wait_test();
    p.limit_ns = wt.limit_ns;
    p.stop_after = wt.stop_after;
    p.early = a.rows_fresh;
    // accumulator fp32 (1) or int32 (2); operands fp16 (0) / bf16 (1) / int8 (1); which run across the contraction; M
    const uint32_t fmt = pl.esize == 1 ? 1u : (uint32_t)a.in_bf16;
    p.idesc = (pl.esize == 1 ? 2u : 1u) << 4 | fmt << 7 | fmt << 10 | (uint32_t)(a.op != LIN_FWD) << 15 |
              (uint32_t)p.wgrad << 16 | (uint32_t)(pl.tile_m >> 4) << 24;
    // the M side is the weights (row products) or the gradient, the N side the rows
    CUtensorMap ma, mb;
    const int span = kLinSpan / pl.esize, load_n = pl.tile_m == 256 ? pl.bn / 2 : pl.bn;
    if (p.wgrad) {
        rc = encode_rows_map(&ma, pa, pl.esize, pl.a_cols, pl.a_rows, sa, 0, 0, span, 64);
        if (!rc) rc = encode_rows_map(&mb, pb, pl.esize, pl.b_cols, pl.b_rows, sb, 0, 0, span, 64);
        return rc ? rc : launch_width<LIN_WGRAD, false>(pl, ma, mb, p, st);
    }
    const int64_t wrows = pl.b_rows / a.E;
    rc = encode_rows_map(&ma, pb, pl.esize, pl.b_cols, wrows, sb, a.E, wrows * sb, span, a.op == LIN_FWD ? kLinTileM : 64);
    if (!rc) rc = encode_rows_map(&mb, pa, pl.esize, pl.a_cols, pl.a_rows, sa, 0, 0, span, load_n);
    if (rc) return rc;
    if (pl.esize == 1) return launch_width<LIN_FWD, true>(pl, ma, mb, p, st);
    if (a.op == LIN_DGRAD) return launch_width<LIN_DGRAD, false>(pl, ma, mb, p, st);
    return launch_width<LIN_FWD, false>(pl, ma, mb, p, st);
}

}  // namespace kdw
