// C entry points of the channel-mixing products: argument checks, the plan and the workspace layout.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "../../include/kdw.h"
#include "linear_core.cuh"
#include "linear_plan.h"

namespace kdw {

static inline int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
static inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Rows of few channels are short, and the TMA unit moves rows at a fixed rate.  In the weight gradient of one group of dense
// rows, f neighbouring rows can be read as one of f times the channels: the product of the folded operands holds f x f
// blocks, of which those on the diagonal are summed and the others, which mix rows, are left.  (In a row product the
// others would multiply zeros with other rows' values, which may be infinite.)
static int fold_of(const LinArgs& a) {
    if (a.op != LIN_WGRAD || a.ends || a.E != 1 || a.a_stride != a.N || a.b_stride != a.K || a.K % 8 || a.N % 8) return 1;
    if (((uintptr_t)a.a & 15) || ((uintptr_t)a.b & 15) || a.T < 8192) return 1;
    const int64_t narrow = std::min(a.K, a.N);
    int f = 1;
    while (f < 8 && narrow * f * 2 <= 64 && a.T % (f * 2) == 0) f *= 2;
    return f;
}

int device_facts(int** status, int* sms) {
    struct Facts {
        int* status;
        std::atomic<int> sms;  // set last; a race only repeats the lookup
    };
    static Facts facts[KernelSetup::kMaxDevices];
    int dev = 0;
    KDW_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= KernelSetup::kMaxDevices) {
        set_error("device index %d is outside the supported range 0..%d", dev, KernelSetup::kMaxDevices - 1);
        return KDW_ERR_ARG;
    }
    // A thread that has made no runtime call yet (a worker of an autograd engine) has no current context, which encoding a
    // tensor map needs.
    static thread_local int bound = -1;
    if (bound != dev) {
        KDW_CUDA(cudaSetDevice(dev));  // (allowed while a stream is being captured, unlike an allocation)
        bound = dev;
    }
    Facts& f = facts[dev];
    if (f.sms.load(std::memory_order_acquire) == 0) {
        int* p = nullptr;
        int n = 0, rc = status_ptr(&p);
        if (!rc) rc = device_sm_count(&n);
        if (rc) return rc;
        f.status = p;
        f.sms.store(n, std::memory_order_release);
    }
    if (status) *status = f.status;
    *sms = f.sms.load(std::memory_order_relaxed);
    return 0;
}

int linear_plan(LinPlan* pl, const LinArgs& given, int sms) {
    LinArgs a = given;
    const bool wgrad = a.op == LIN_WGRAD;
    pl->fold = fold_of(a);
    a.T /= pl->fold;
    a.K *= wgrad ? pl->fold : 1;
    a.N *= wgrad ? pl->fold : 1;
    a.a_stride *= pl->fold;
    a.b_stride *= pl->fold;
    pl->esize = a.esize;
    const int64_t con = a.op == LIN_FWD ? a.K : a.op == LIN_DGRAD ? a.N : a.T;  // length of the contraction
    pl->out_cols = (int)(a.op == LIN_FWD ? a.N : a.K);
    pl->out_rows = wgrad ? (int)a.N : 0;
    pl->a_rows = a.T;
    pl->a_cols = a.op == LIN_FWD ? a.K : a.N;
    pl->b_rows = wgrad ? a.T : a.E * a.N;
    pl->b_cols = a.K;
    // TMA wants 16-byte bases and pitches
    const int64_t per16 = 16 / a.esize;
    pl->pack_a = ((uintptr_t)a.a & 15) != 0 || a.a_stride % per16 != 0 || a.a_stride < pl->a_cols;
    pl->pack_b = ((uintptr_t)a.b & 15) != 0 || a.b_stride % per16 != 0 || a.b_stride < pl->b_cols;
    pl->a_pitch = round_up(pl->a_cols, per16);
    pl->b_pitch = round_up(pl->b_cols, per16);

    const int64_t k_elems = 128 / a.esize;
    pl->k_blocks = wgrad ? 0 : (int)ceil_div(con, k_elems);
    // Tile and parts: the smallest estimate of the cycles on the busiest SM.  A stage of 64 (128 bytes of) contraction
    // steps costs a CTA the larger of the products, 2 cycles a column, and shared memory, which writes and reads the stage
    // at 128 bytes a cycle: 256 cycles for the M side and 2 a column of the N side it loads (a pair: half of them).  A
    // tile costs some 1500 cycles more that the next one does not hide, a pair's 1200 on top, and 4000 to 10000 where two
    // to eight parts of a cluster share it (measured at 64 x 4096 -> 4096 on 128 x 64 tiles: 15.8 us for 64 blocks on one
    // CTA, 12.0 on two, 10.8 on four).
    // Shares of the weight gradient that are added in memory cost another kernel and their bytes, written and read.
    const int64_t groups = std::min(a.E, a.T);
    const double rows = (double)a.T / groups;  // of a group, about
    const int cluster_slots[] = {0, sms, sms, 0, 132 * sms / 148, 0, 0, 0, 120 * sms / 148};  // CTAs in clusters that fit at once
    double best = 1e300;  // (a tile of one CTA without parts is always considered, or shares of folded rows)
    auto consider = [&](double cost, int tile_m, int bn, int splits, int64_t chunk) {
        if (cost >= best) return;
        best = cost;
        pl->tile_m = tile_m;
        pl->bn = bn;
        pl->splits = splits;
        pl->chunk = (int)chunk;
    };
    static const struct { int tile_m, bn; } shapes[] = {{256, 256}, {128, 256}, {128, 128}, {128, 64}};
    for (auto& c : shapes) {
        const bool pair = c.tile_m == 256;
        const int slots = pair ? sms / 2 : sms;
        const double m_tiles = (double)ceil_div(wgrad ? a.N : pl->out_cols, c.tile_m);
        // (groups of unlike sizes have half a tile more than their rows fill, one group as many as it needs)
        const double n_tiles = wgrad ? (double)ceil_div(pl->out_cols, c.bn)
                                     : groups == 1 ? std::ceil(rows / c.bn) : std::max(1.0, rows / c.bn + 0.5);
        const double width = wgrad ? c.bn : std::min<double>(c.bn, std::ceil(rows / n_tiles / 32) * 32);
        const double tiles = m_tiles * n_tiles * (wgrad ? a.E : groups);
        const double block = std::max(2 * width, 256 + (pair ? 1 : 2) * (double)c.bn);
        const double blocks = wgrad ? std::ceil(rows / 64) : pl->k_blocks;
        if (pl->fold == 1) {
            const double extra = pair ? 1200 : 0;
            consider(std::ceil(tiles / slots) * (blocks * block + 1500) + extra, c.tile_m, c.bn, 1, INT32_MAX);
            for (int splits = 2; splits <= (pair ? 4 : 8); splits *= 2)
                if (blocks / splits >= 2 && tiles * splits * (pair ? 2 : 1) <= cluster_slots[splits * (pair ? 2 : 1)])
                    consider(std::ceil(blocks / splits) * block + 3500 + 1000 * splits + extra, c.tile_m, c.bn, splits, INT32_MAX);
        }
        if (!wgrad || (pl->fold == 1 && (tiles > slots || rows < 1024))) continue;
        for (int waves = 1; waves <= 2; ++waves) {
            const double shares = std::max(1.0, std::floor(waves * slots / tiles));
            const int64_t chunk = std::max<int64_t>(256, round_up((int64_t)std::ceil(rows / shares), 64));
            const double units = tiles * std::ceil(rows / chunk), bytes = units * c.tile_m * c.bn * 4;
            consider(std::ceil(units / slots) * (chunk / 64 * block + 1500) + 6000 + bytes / (sms * 10.0), c.tile_m, c.bn, 1,
                     std::min<int64_t>(chunk, 1 << 30));
        }
    }
    pl->m_tiles = (int)ceil_div(wgrad ? a.N : pl->out_cols, pl->tile_m);
    pl->n_tiles = wgrad ? (int)ceil_div(pl->out_cols, pl->bn) : 0;
    // the most there can be, however the rows are distributed
    pl->max_tiles = pl->m_tiles * (wgrad ? pl->n_tiles * a.E : ceil_div(a.T, pl->bn) + groups - 1);
    pl->max_units = pl->max_tiles;
    // (the folded product's blocks are summed from the shares, whatever their number)
    const bool split = wgrad && (pl->chunk < a.T || pl->fold > 1);
    if (split) pl->max_units = (int64_t)pl->m_tiles * pl->n_tiles * (a.T / pl->chunk + a.E);
    int64_t off = 0;
    pl->off_a = pl->off_b = pl->off_table = 0;
    pl->off_partial = -1;
    if (pl->pack_a) {
        pl->off_a = off;
        off = round_up(off + pl->a_rows * pl->a_pitch * a.esize, 256);
    }
    if (pl->pack_b) {
        pl->off_b = off;
        off = round_up(off + pl->b_rows * pl->b_pitch * a.esize, 256);
    }
    if (split) {
        pl->off_table = off;
        off = round_up(off + 2 * (a.E + 1) * 4, 256);
        pl->off_partial = off;
        off += pl->max_units * pl->tile_m * pl->bn * 4;
    }
    pl->bytes = off;
    if (pl->max_units > INT32_MAX) {
        set_error("linear: %lld tiles are more than one call takes", (long long)pl->max_units);
        return KDW_ERR_ARG;
    }
    return 0;
}

static int check_sizes(const char* what, int64_t T, int64_t E, int64_t K, int64_t N) {
    const int64_t most = INT32_MAX - 1024;
    if (T < 1 || E < 1 || K < 1 || N < 1 || T > most || K > most || N > most) {
        set_error("%s: T=%lld E=%lld K=%lld N=%lld out of range", what, (long long)T, (long long)E, (long long)K,
                  (long long)N);
        return KDW_ERR_ARG;
    }
    if (E > kLinMaxGroups) {
        set_error("%s: %lld groups, at most %d", what, (long long)E, kLinMaxGroups);
        return KDW_ERR_ARG;
    }
    if (E * N > most) {
        set_error("%s: E*N=%lld out of range", what, (long long)(E * N));
        return KDW_ERR_ARG;
    }
    return 0;
}

static int f16_args(LinArgs* a, int op, const void* pa, const void* pb, int64_t T, int64_t E, int64_t K, int64_t N,
                    int64_t a_stride, int64_t b_stride, int dtype) {
    int rc = check_sizes("linear_f16", T, E, K, N);
    if (rc) return rc;
    if (op < LIN_FWD || op > LIN_WGRAD || (dtype != KDW_F16 && dtype != KDW_BF16)) {
        set_error("linear_f16: op=%d dtype=%d unknown", op, dtype);
        return KDW_ERR_ARG;
    }
    const int64_t a_cols = op == LIN_FWD ? K : N;
    if (a_stride < a_cols || (op == LIN_WGRAD && b_stride < K)) {
        set_error("linear_f16: row strides %lld, %lld are shorter than the rows", (long long)a_stride, (long long)b_stride);
        return KDW_ERR_ARG;
    }
    *a = LinArgs();
    a->op = op;
    a->a = pa;
    a->b = pb;
    a->T = T;
    a->E = E;
    a->K = K;
    a->N = N;
    a->a_stride = a_stride;
    a->b_stride = op == LIN_WGRAD ? b_stride : K;
    a->esize = 2;
    a->in_bf16 = a->out_bf16 = dtype == KDW_BF16;
    return 0;
}

static bool is_few(const LinArgs& a) { return a.op == LIN_FWD && a.T <= kFewRows && a.K <= (1 << 28); }  // byte offsets in 32 bits

// The 8-bit product: the rows are int8 with their scales, or 16-bit rows that are quantised into the workspace first.
struct I8Layout {
    int64_t q_pitch, off_scale, off_w, off_rest;  // bytes; quantised rows at 0
    bool pack_w;                                  // the kernel that quantises copies the weights to a pitch of 16 bytes too
};
static int i8_args(LinArgs* a, I8Layout* l, const void* x, const void* w, int64_t T, int64_t E, int64_t K, int64_t N,
                   int64_t x_stride, int x_type, int dtype) {
    int rc = check_sizes("linear_i8", T, E, K, N);
    if (rc) return rc;
    if ((x_type != KDW_I8 && x_type != KDW_F16 && x_type != KDW_BF16) || (dtype != KDW_F16 && dtype != KDW_BF16)) {
        set_error("linear_i8: x_type=%d dtype=%d unknown", x_type, dtype);
        return KDW_ERR_ARG;
    }
    if (K > 131071) {  // 2^14 (K - 1) < 2^31 - 2^14: no sum leaves 32 bits
        set_error("linear_i8: K=%lld, at most 131071 (32-bit sums)", (long long)K);
        return KDW_ERR_ARG;
    }
    if (x_stride < K) {
        set_error("linear_i8: row stride %lld is shorter than the rows", (long long)x_stride);
        return KDW_ERR_ARG;
    }
    *a = LinArgs();
    l->q_pitch = l->off_scale = l->off_w = l->off_rest = 0;
    l->pack_w = false;
    a->op = LIN_FWD;
    a->a = x;
    a->a_stride = x_stride;
    a->b = w;
    a->b_stride = K;
    if (x_type != KDW_I8) {
        l->q_pitch = round_up(K, 16);
        l->off_scale = round_up(T * l->q_pitch, 256);
        l->off_w = l->off_rest = round_up(l->off_scale + 4 * T, 256);
        a->a = nullptr;  // its copy in the workspace is aligned
        a->a_stride = l->q_pitch;
        l->pack_w = T > kFewRows && (((uintptr_t)w & 15) != 0 || K % 16 != 0);
        if (l->pack_w) {
            l->off_rest = round_up(l->off_w + E * N * l->q_pitch, 256);
            a->b = nullptr;
            a->b_stride = l->q_pitch;
        }
    }
    a->T = T;
    a->E = E;
    a->K = K;
    a->N = N;
    a->esize = 1;
    a->out_bf16 = dtype == KDW_BF16;
    return 0;
}

// Both gradients of one product: operands that TMA cannot address are copied once for the two.
struct GradsLayout {
    bool pack_g, pack_x, pack_w;
    int64_t g_pitch, k_pitch;               // elements
    int64_t off_g, off_x, off_w, off_rest;  // bytes
};
static int grads_args(LinArgs* d, LinArgs* g, GradsLayout* l, const void* x, const void* w, const void* grad, int64_t T, int64_t E,
                      int64_t K, int64_t N, int64_t x_stride, int64_t grad_stride, int dtype) {
    int rc = f16_args(d, LIN_DGRAD, grad, w, T, E, K, N, grad_stride, 0, dtype);
    if (!rc) rc = f16_args(g, LIN_WGRAD, grad, x, T, E, K, N, grad_stride, x_stride, dtype);
    if (rc) return rc;
    auto odd = [](const void* p, int64_t stride) { return ((uintptr_t)p & 15) != 0 || stride % 8 != 0; };
    l->pack_g = odd(grad, grad_stride);
    l->pack_x = odd(x, x_stride);
    l->pack_w = odd(w, K);
    l->g_pitch = round_up(N, 8);
    l->k_pitch = round_up(K, 8);
    l->off_g = 0;
    l->off_x = round_up(l->pack_g ? T * l->g_pitch * 2 : 0, 256);
    l->off_w = round_up(l->off_x + (l->pack_x ? T * l->k_pitch * 2 : 0), 256);
    l->off_rest = round_up(l->off_w + (l->pack_w ? E * N * l->k_pitch * 2 : 0), 256);
    if (l->pack_g) {
        d->a = g->a = nullptr;  // the copies in the workspace are aligned
        d->a_stride = g->a_stride = l->g_pitch;
    }
    if (l->pack_x) {
        g->b = nullptr;
        g->b_stride = l->k_pitch;
    }
    if (l->pack_w) {
        d->b = nullptr;
        d->b_stride = l->k_pitch;
    }
    return 0;
}

// Few 16-bit rows that every CTA of the product quantises itself.
static bool quant_inside(const LinArgs& a, int x_type) {
    return x_type != KDW_I8 && a.T <= kFewQuantRows && (a.K + 127) / 128 * 128 + 64 <= kFewQuantPitch;
}

static int plan_and_run(LinArgs* a, void* workspace, int64_t workspace_bytes, void* stream) {
    LinPlan pl;
    int sms = 0;
    int rc = device_facts(nullptr, &sms);
    if (!rc) rc = linear_plan(&pl, *a, sms);
    if (rc) return rc;
    if (pl.bytes > 0 && (!workspace || workspace_bytes < pl.bytes || ((uintptr_t)workspace & 255) != 0)) {
        set_error("linear: workspace of %lld bytes (256-byte aligned) needed, %lld given", (long long)pl.bytes,
                  (long long)(workspace ? workspace_bytes : 0));
        return KDW_ERR_WORKSPACE;
    }
    return linear_run(pl, *a, workspace, (cudaStream_t)stream);
}

}  // namespace kdw

extern "C" {

int kdw_linear_auto_variant(int op, int type, int64_t T, int64_t E, int64_t K, int64_t N, int sms) {
    using namespace kdw;
    LinArgs args;
    I8Layout l;
    const void* aligned = (const void*)4096;
    int rc = type == KDW_I8 ? i8_args(&args, &l, aligned, aligned, T, E, K, N, K, type, KDW_F16)
                            : f16_args(&args, op, aligned, aligned, T, E, K, N, op == LIN_FWD ? K : N, K, type);
    if (rc) return rc;
    if (sms < 1) {
        set_error("linear_auto_variant: sms=%d", sms);
        return KDW_ERR_ARG;
    }
    if (is_few(args)) return 1;
    if (is_narrow(args)) return 2;
    LinPlan pl;
    rc = linear_plan(&pl, args, sms);
    if (rc) return rc;
    const int parts = pl.fold > 1 ? 32 : pl.off_partial >= 0 ? 16 : pl.splits;
    return parts * 1000000 + pl.tile_m * 1000 + pl.bn;
}

int64_t kdw_linear_f16_workspace_bytes(int op, const void* a, const void* b, int64_t T, int64_t E, int64_t K, int64_t N,
                                       int64_t a_stride, int64_t b_stride, int dtype) {
    using namespace kdw;
    LinArgs args;
    LinPlan pl;
    int sms = 0;
    int rc = f16_args(&args, op, a, b, T, E, K, N, a_stride, b_stride, dtype);
    if (!rc) rc = device_facts(nullptr, &sms);
    if (!rc && (is_few(args) || is_narrow(args))) return 0;
    if (!rc) rc = linear_plan(&pl, args, sms);
    int64_t bytes = rc ? 0 : pl.bytes;
    if (!rc && pl.fold > 1) {  // the call may bring its one group's end, and then folds no rows
        const int32_t any = 0;
        args.ends = &any;
        rc = linear_plan(&pl, args, sms);
        bytes = std::max(bytes, pl.bytes);
    }
    return rc ? (rc < 0 ? rc : -rc) : bytes;
}

int kdw_linear_f16(int op, const void* a, const void* b, void* out, const int32_t* ends, void* workspace,
                   int64_t workspace_bytes, int64_t T, int64_t E, int64_t K, int64_t N, int64_t a_stride,
                   int64_t b_stride, int dtype, void* stream) {
    using namespace kdw;
    if (!a || !b || !out || (!ends && E != 1)) {
        set_error("linear_f16: null pointer (ends may be null only with one group)");
        return KDW_ERR_ARG;
    }
    LinArgs args;
    int rc = f16_args(&args, op, a, b, T, E, K, N, a_stride, b_stride, dtype);
    if (rc) return rc;
    if (((uintptr_t)a & 1) || ((uintptr_t)b & 1) || ((uintptr_t)out & 1) || ((uintptr_t)ends & 3)) {
        set_error("linear_f16: a pointer is not aligned to its elements");
        return KDW_ERR_ALIGN;
    }
    args.out = out;
    args.ends = ends;
    if (is_few(args)) return linear_few(args, dtype, (cudaStream_t)stream);
    // 16-byte stores: an output that does not allow them takes the other path, which copies nothing of operands like these
    if (is_narrow(args) && ((uintptr_t)out & 15) == 0) return linear_narrow(args, (cudaStream_t)stream);
    return plan_and_run(&args, workspace, workspace_bytes, stream);
}

int64_t kdw_linear_grads_f16_workspace_bytes(const void* x, const void* w, const void* grad, int has_ends, int64_t T, int64_t E,
                                             int64_t K, int64_t N, int64_t x_stride, int64_t grad_stride, int dtype) {
    using namespace kdw;
    LinArgs d, g;
    GradsLayout l;
    LinPlan pl;
    int sms = 0;
    int rc = grads_args(&d, &g, &l, x, w, grad, T, E, K, N, x_stride, grad_stride, dtype);
    if (!rc) rc = device_facts(nullptr, &sms);
    const int32_t any = 0;
    d.ends = g.ends = has_ends ? &any : nullptr;
    int64_t bytes = 0;
    if (!rc && is_narrow_grads(d, g)) rc = linear_narrow_grads(d, g, nullptr, 0, &bytes, nullptr);
    for (const LinArgs* a : {&d, &g})  // (also where both gradients go in one pass: an unaligned dx takes two products)
        if (!rc && !is_narrow(*a)) {  // (a narrow product needs none on either path)
            rc = linear_plan(&pl, *a, sms);
            bytes = std::max<int64_t>(bytes, rc ? 0 : pl.bytes);
        }
    return rc ? (rc < 0 ? rc : -rc) : l.off_rest + bytes;
}

int kdw_linear_grads_f16(const void* x, const void* w, const void* grad, void* dx, void* dw, const int32_t* ends, void* workspace,
                         int64_t workspace_bytes, int64_t T, int64_t E, int64_t K, int64_t N, int64_t x_stride,
                         int64_t grad_stride, int dtype, void* stream) {
    using namespace kdw;
    if (!x || !w || !grad || !dx || !dw || (!ends && E != 1)) {
        set_error("linear_grads_f16: null pointer (ends may be null only with one group)");
        return KDW_ERR_ARG;
    }
    LinArgs d, g;
    GradsLayout l;
    int rc = grads_args(&d, &g, &l, x, w, grad, T, E, K, N, x_stride, grad_stride, dtype);
    if (rc) return rc;
    if (((uintptr_t)x & 1) || ((uintptr_t)w & 1) || ((uintptr_t)grad & 1) || ((uintptr_t)dx & 1) || ((uintptr_t)dw & 1) ||
        ((uintptr_t)ends & 3)) {
        set_error("linear_grads_f16: a pointer is not aligned to its elements");
        return KDW_ERR_ALIGN;
    }
    if (l.off_rest > 0 && (!workspace || workspace_bytes < l.off_rest || ((uintptr_t)workspace & 255) != 0)) {
        set_error("linear_grads_f16: workspace of at least %lld bytes (256-byte aligned) needed", (long long)l.off_rest);
        return KDW_ERR_WORKSPACE;
    }
    char* ws = (char*)workspace;
    if (l.off_rest > 0) {
        const PackRows r[3] = {{grad, ws + l.off_g, l.pack_g ? T : 0, grad_stride, l.g_pitch, (int)N},
                               {x, ws + l.off_x, l.pack_x ? T : 0, x_stride, l.k_pitch, (int)K},
                               {w, ws + l.off_w, l.pack_w ? E * N : 0, K, l.k_pitch, (int)K}};
        rc = pack_rows(r, 3, 2, (cudaStream_t)stream);
        if (rc) return rc;
        if (l.pack_g) d.a = g.a = ws + l.off_g;
        if (l.pack_x) g.b = ws + l.off_x;
        if (l.pack_w) d.b = ws + l.off_w;
    }
    d.out = dx;
    g.out = dw;
    d.ends = g.ends = ends;
    // the second product's kernels touch the workspace only when the first one's have completed
    ws = ws ? ws + l.off_rest : ws;
    if (is_narrow_grads(d, g) && ((uintptr_t)dx & 15) == 0) {
        int64_t need = 0;
        return linear_narrow_grads(d, g, ws, ws ? workspace_bytes - l.off_rest : 0, &need, (cudaStream_t)stream);
    }
    rc = is_narrow(d) && ((uintptr_t)dx & 15) == 0 ? linear_narrow(d, (cudaStream_t)stream)
                                                   : plan_and_run(&d, ws, workspace_bytes - l.off_rest, stream);
    return rc ? rc : plan_and_run(&g, ws, workspace_bytes - l.off_rest, stream);
}

int64_t kdw_linear_i8_workspace_bytes(const void* x, const void* w, int64_t T, int64_t E, int64_t K, int64_t N,
                                      int64_t x_stride, int x_type, int dtype) {
    using namespace kdw;
    LinArgs args;
    LinPlan pl;
    I8Layout l;
    int sms = 0;
    int rc = i8_args(&args, &l, x, w, T, E, K, N, x_stride, x_type, dtype);
    if (!rc) rc = device_facts(nullptr, &sms);
    if (!rc && is_few(args)) return quant_inside(args, x_type) ? 0 : l.off_rest;
    if (!rc) rc = linear_plan(&pl, args, sms);
    return rc ? (rc < 0 ? rc : -rc) : l.off_rest + pl.bytes;
}

int kdw_linear_i8(const void* x, const float* x_scale, const int8_t* w, const float* w_scale, void* y, const int32_t* ends,
                  void* workspace, int64_t workspace_bytes, int64_t T, int64_t E, int64_t K, int64_t N, int64_t x_stride,
                  int x_type, int dtype, void* stream) {
    using namespace kdw;
    if (!x || !w || !w_scale || !y || (!ends && E != 1) || (x_type == KDW_I8 && !x_scale)) {
        set_error("linear_i8: null pointer (x_scale may be null only with 16-bit x, ends only with one group)");
        return KDW_ERR_ARG;
    }
    LinArgs args;
    I8Layout l;
    int rc = i8_args(&args, &l, x, w, T, E, K, N, x_stride, x_type, dtype);
    if (rc) return rc;
    if ((x_type != KDW_I8 && ((uintptr_t)x & 1)) || ((uintptr_t)x_scale & 3) || ((uintptr_t)w_scale & 3) || ((uintptr_t)y & 1) ||
        ((uintptr_t)ends & 3)) {
        set_error("linear_i8: a pointer is not aligned to its elements");
        return KDW_ERR_ALIGN;
    }
    args.out = y;
    args.ends = ends;
    args.row_scale = x_scale;
    args.col_scale = w_scale;
    char* ws = (char*)workspace;
    if (is_few(args) && quant_inside(args, x_type)) {
        args.a = x;
        args.a_stride = x_stride;
        return linear_few(args, x_type, (cudaStream_t)stream);
    }
    if (x_type != KDW_I8) {
        if (!workspace || workspace_bytes < l.off_rest || ((uintptr_t)workspace & 255) != 0) {
            set_error("linear_i8: workspace of at least %lld bytes (256-byte aligned) needed", (long long)l.off_rest);
            return KDW_ERR_WORKSPACE;
        }
        args.a = ws;
        args.row_scale = (const float*)(ws + l.off_scale);
        const PackRows pack = {w, ws + l.off_w, E * N, K, l.q_pitch, (int)K};
        rc = quant_rows(x, ws, (float*)(ws + l.off_scale), T, K, x_stride, l.q_pitch, x_type == KDW_BF16, true,
                        l.pack_w ? &pack : nullptr, (cudaStream_t)stream);
        if (rc) return rc;
        if (l.pack_w) args.b = ws + l.off_w;
        args.rows_fresh = !l.pack_w;
        ws += l.off_rest;
    }
    if (is_few(args)) return linear_few(args, KDW_I8, (cudaStream_t)stream);
    return plan_and_run(&args, ws, workspace_bytes - l.off_rest, stream);
}

}  // extern "C"
