// Host-side plan of one channel-mixing product: tile width, shares of the contraction, packed copies and the
// layout of the workspace.  The workspace query and the launch both build it from the same arguments.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace kdw {

struct LinArgs {
    int op;               // LinOp
    const void *a, *b;    // rows [T][.] and: weights [E][N][K] (row products) or rows [T][K] (weight gradient)
    void* out;
    const int* ends;
    int64_t T, E, K, N;
    int64_t a_stride, b_stride;  // elements between rows; of the weights: K
    int esize;            // bytes of an operand element (2 or 1)
    int in_bf16, out_bf16;
    const float *row_scale, *col_scale;
    int rows_fresh;       // 1: the kernel enqueued just before is this call's own and wrote the rows and row_scale only
};

struct LinPlan {
    int esize, bn, tile_m;  // tile_m 256: a pair of CTAs to a tile
    int m_tiles, n_tiles, out_rows, out_cols, k_blocks, splits, chunk;
    int fold;                // weight gradient: rows that are taken as one (see linear_plan)
    bool pack_a, pack_b;
    int64_t a_rows, a_cols, a_pitch, b_rows, b_cols, b_pitch;  // pitches of the packed copies, in elements
    int64_t off_a, off_b, off_table, off_partial;              // off_partial < 0: no tile has several shares
    int64_t bytes;
    int64_t max_tiles, max_units;                              // over all row distributions
};

// The library's status word on the current device and its SMs, looked up once per device.
int device_facts(int** status, int* sms);

int linear_plan(LinPlan* pl, const LinArgs& a, int sms);
int linear_run(const LinPlan& pl, const LinArgs& a, void* ws, cudaStream_t st);

// Products of few rows, without a workspace (linear_few.cu).  x_type: KDW_I8, or 16-bit rows to quantise within the kernel.
constexpr int kFewRows = 16;
constexpr int kFewQuantRows = 8, kFewQuantPitch = 128 * 96 + 64;  // rows and bytes of a row that a CTA quantises itself
int linear_few(const LinArgs& a, int x_type, cudaStream_t st);
// Output channels of a CTA: 32 where CTAs of 16 would not all be resident at once (two to an SM; `groups` at most that have
// rows).  8 rows of 8 groups, 2048 -> 1024, 9.1 us instead of 10.3 (7.0 now that pieces run ahead); with fewer CTAs the
// contraction is better split further (4096 x 4096: 8.5 and 11.2 us, measured before that too).
inline int few_channels(int64_t N, int64_t groups, int sms) { return (N + 15) / 16 * groups > 2 * (int64_t)sms ? 32 : 16; }

// Products of many rows with one narrow weight matrix, without a workspace (linear_narrow.cu).
bool is_narrow(const LinArgs& a);
int linear_narrow(const LinArgs& a, cudaStream_t st);
// Both gradients in one pass; `need`: the workspace.  Without g.out (the weight gradient) it only says what it needs.
bool is_narrow_grads(const LinArgs& d, const LinArgs& g);
int linear_narrow_grads(const LinArgs& d, const LinArgs& g, void* ws, int64_t ws_bytes, int64_t* need, cudaStream_t st);

// Rows to copy to a pitch of 16 bytes, because TMA cannot address them where they are; strides in elements.
struct PackRows {
    const void* src;
    void* dst;
    long long rows, src_stride, dst_stride;
    int cols;
};
// CTAs of 256 threads that copy them; 0: there is nothing to copy.
int pack_ctas(const PackRows& r, int esize, int sms);
// Copies up to three operands with one kernel.
int pack_rows(const PackRows* r, int count, int esize, cudaStream_t st);

// Quantises rows of 16-bit values (see quant_rows.cu); q_padded: what lies between `cols` and q_stride may be written.
// `pack`, if given, are rows of 8-bit weights that the same kernel copies.
int quant_rows(const void* x, void* q, float* scale, int64_t rows, int64_t cols, int64_t x_stride, int64_t q_stride, int bf16,
               bool q_padded, const PackRows* pack, cudaStream_t st);

// Rows of `cols` elements (1 or 2 bytes each) `stride` elements apart, in `groups` matrices `group_stride` elements
// apart (0 groups: one matrix, a 2-D map); a box of `box_cols` x `box_rows`, 128-byte swizzle, zeros outside.
int encode_rows_map(CUtensorMap* map, const void* base, int esize, int64_t cols, int64_t rows, int64_t stride,
                    int64_t groups, int64_t group_stride, int box_cols, int box_rows);

}  // namespace kdw
