// Host-side interface of the token operators (kernels/rotary.hip, kernels/gated_ffn*.hip) to their C entry points (token_ops.cpp).
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/gddim_amd.h"

namespace gd {

constexpr int ROT_MAX_AXES = 4;
constexpr int ROT_MAX_HEAD_DIM = 512;
constexpr int ROT_BWD_BLOCKS = 512;  // partial rows of the weight gradients
constexpr int ROT_BWD_THREADS = 512;

// one (B, N, heads, D) tensor: strides in elements, channels adjacent
struct HeadsView {
    void *p;
    long long sb, sn, sh;
};

// segment 0 = queries, segment 1 = keys (heads[1] = 0: absent)
struct RotaryParams {
    HeadsView x[2];    // inputs
    HeadsView dy[2];   // backward: gradients of the outputs
    HeadsView out[2];  // outputs (backward: gradients of the inputs)
    int heads[2];
    int batch, tokens, D, R;
    const void *pos;
    int pos_type;  // GD_POS_*
    long long pos_sb, pos_sn, pos_sa;
    int n_axes;
    int axis_end[ROT_MAX_AXES];  // pairs [axis_end[a - 1], axis_end[a]) turn with axis a
    const double *freq;          // R / 2 radians per unit of position
    int halves;                  // pairs (i, i + R/2) instead of (2i, 2i + 1)
    float sign;                  // -1: turn back
    const void *w[2];            // norm weights (D) or null
    int w_f32;                   // weights are float32 whatever the tensors' type
    float eps;
    float *dw_part;  // [blocks][2][D]
    // filled in by the launcher
    int rows_per_item, items_per_token;
    int group;  // tokens of an item
    unsigned items;
};

enum RotaryMode { ROT_PLAIN = 0, ROT_NORM = 1, ROT_NORM_BWD = 2 };
int launch_rotary(RotaryParams p, int dtype, RotaryMode mode, void *dw0, void *dw1, hipStream_t s);

// ---- gated feed-forward block (kernels/gated_ffn_gemm.h) ----
enum GemmKind { GEMM_GATE_UP, GEMM_DOWN, GEMM_DHIDDEN, GEMM_DX, GEMM_DW };
enum GemmEpilogue { EPI_STORE, EPI_GATED, EPI_GATED_BWD };
enum GemmTile { TILE_128, TILE_256, TILE_NARROW, TILE_SKINNY };  // NARROW: 128 x 64

// C[m][n] = sum over parts and k of A[m][k] B[n][k]
struct GemmProblem {
    const void *a[2], *b[2];     // two-part sums: a[1], b[1]; GEMM_GATE_UP: b = {Wg, Wu}
    long long lda, ldb;          // bytes from row to row of the matrix as it lies in memory
    long long a_bytes, b_bytes;  // extent of a matrix in memory
    int M, N, K, parts;
    void *out[3];                // rows of N elements, dense; EPI_GATED: h, gate and up (float32 or null); EPI_GATED_BWD: dgate, dup
    const void *in[2];           // EPI_GATED_BWD: gate, up (float32)
    int short_rows;              // N < 2^23: 32 rows of four-byte elements stay under 2^30 bytes
    int splits, stages_per_split;
    float *partial;
    // filled in by the launcher
    int tiles_m, tiles_n, blocks;
    long long join_threads;
};

struct GemmLaunch {
    GemmProblem q[3];
    int problems, act, direct, join_blocks;
    int blocks, grid;            // pieces of work; workgroups
    int skinny_m, skinny_rows;   // TILE_SKINNY: blocks of 16 rows of x and rows of the weights a workgroup takes
    GemmTile tile;
};

int launch_ffn_gemm_bf16(const GemmLaunch &p, GemmKind kind, hipStream_t s);
int launch_ffn_gemm_f16(const GemmLaunch &p, GemmKind kind, hipStream_t s);
int launch_ffn_gemm_f32(const GemmLaunch &p, GemmKind kind, hipStream_t s);

}  // namespace gd
