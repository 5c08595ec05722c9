// Host-side interface of the token operators (kernels/rotary.hip, kernels/gated_ffn*.hip) to their C entry points (token_ops.cpp).
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/gddim_amd.h"

namespace gd {

constexpr int ROT_MAX_AXES = 4;
constexpr int ROT_MAX_HEAD_DIM = 512;
constexpr int ROT_BWD_BLOCKS = 1024;  // partial rows of the weight gradients

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
    unsigned items;
};

enum RotaryMode { ROT_PLAIN = 0, ROT_NORM = 1, ROT_NORM_BWD = 2 };
int launch_rotary(RotaryParams p, int dtype, RotaryMode mode, void *dw0, void *dw1, hipStream_t s);

}  // namespace gd
