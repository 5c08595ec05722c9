// C entry points of the token operators: argument checks, then the launchers of kernels/.
#include <cstdint>

#include "common.h"
#include "token_ops.h"

using namespace gd;

namespace {

int fill_rotary(RotaryParams &p, const gd_rotary_desc *d, const char *who) {
    GD_CHECK(d, "%s: null description", who);
    GD_CHECK(d->dtype == GD_F32 || d->dtype == GD_BF16 || d->dtype == GD_F16, "%s: unknown element type %d", who, d->dtype);
    GD_CHECK(d->pos_type == GD_POS_I32 || d->pos_type == GD_POS_I64 || d->pos_type == GD_POS_F32, "%s: unknown position type %d", who, d->pos_type);
    GD_CHECK(d->batch >= 0 && d->tokens >= 0, "%s: negative batch %d or tokens %d", who, d->batch, d->tokens);
    GD_CHECK((long long)d->batch * d->tokens < (1LL << 31), "%s: %d x %d tokens do not fit 31 bits", who, d->batch, d->tokens);
    GD_CHECK(d->head_dim >= 2 && d->head_dim <= ROT_MAX_HEAD_DIM, "%s: head_dim %d outside [2, %d]", who, d->head_dim, ROT_MAX_HEAD_DIM);
    GD_CHECK(d->n_axes >= 1 && d->n_axes <= ROT_MAX_AXES, "%s: %d axes outside [1, %d]", who, d->n_axes, ROT_MAX_AXES);
    GD_CHECK(d->freq && (d->pos || (long long)d->batch * d->tokens == 0), "%s: null positions or frequencies", who);
    int R = 0;
    for (int a = 0; a < d->n_axes; ++a) {
        GD_CHECK(d->section[a] >= 2 && d->section[a] % 2 == 0 && d->section[a] <= ROT_MAX_HEAD_DIM, "%s: section %d of axis %d is not an even number of channels", who, d->section[a], a);
        R += d->section[a];
        p.axis_end[a] = R / 2;
    }
    GD_CHECK(R <= d->head_dim, "%s: sections of %d channels exceed head_dim %d", who, R, d->head_dim);
    p.batch = d->batch; p.tokens = d->tokens; p.D = d->head_dim; p.R = R; p.n_axes = d->n_axes;
    p.pos = d->pos; p.pos_type = d->pos_type;
    p.pos_sb = d->pos_stride_b; p.pos_sn = d->pos_stride_n; p.pos_sa = d->pos_stride_axis;
    p.freq = d->freq; p.halves = d->paired_halves != 0; p.sign = 1.f;
    return 0;
}

int view(HeadsView &v, const gd_heads *h, bool empty, const char *who, const char *name) {
    GD_CHECK(h && (h->data || empty), "%s: null %s", who, name);
    v.p = h->data; v.sb = h->stride_b; v.sn = h->stride_n; v.sh = h->stride_h;
    return 0;
}

}  // namespace

extern "C" {

int gd_rotary(const gd_rotary_desc *d, const gd_heads *x, const gd_heads *out, int heads, int inverse, void *stream) {
    RotaryParams p{};
    GD_TRY(fill_rotary(p, d, "rotary"));
    GD_CHECK(heads >= 1 && heads <= 65535, "rotary: %d heads outside [1, 65535]", heads);
    const bool empty = (long long)p.batch * p.tokens == 0;
    GD_TRY(view(p.x[0], x, empty, "rotary", "x"));
    GD_TRY(view(p.out[0], out, empty, "rotary", "out"));
    p.heads[0] = heads;
    if (inverse) p.sign = -1.f;
    return launch_rotary(p, d->dtype, ROT_PLAIN, nullptr, nullptr, (hipStream_t)stream);
}

int gd_qk_norm_rotary(const gd_rotary_desc *d, const gd_heads *q, const gd_heads *k, const gd_heads *q_out, const gd_heads *k_out, int heads_q,
                      int heads_k, const void *w_q, const void *w_k, int w_f32, float eps, void *stream) {
    static const char *who = "qk_norm_rotary";
    RotaryParams p{};
    GD_TRY(fill_rotary(p, d, who));
    GD_CHECK(heads_q >= 1 && heads_k >= 1 && heads_q <= 65535 && heads_k <= 65535, "%s: %d / %d heads outside [1, 65535]", who, heads_q, heads_k);
    GD_CHECK(eps >= 0.f, "%s: negative eps", who);
    const bool empty = (long long)p.batch * p.tokens == 0;
    GD_TRY(view(p.x[0], q, empty, who, "q"));
    GD_TRY(view(p.x[1], k, empty, who, "k"));
    GD_TRY(view(p.out[0], q_out, empty, who, "q_out"));
    GD_TRY(view(p.out[1], k_out, empty, who, "k_out"));
    p.heads[0] = heads_q; p.heads[1] = heads_k;
    p.w[0] = w_q; p.w[1] = w_k; p.w_f32 = w_f32; p.eps = eps;
    return launch_rotary(p, d->dtype, ROT_NORM, nullptr, nullptr, (hipStream_t)stream);
}

long long gd_qk_norm_rotary_backward_workspace(int head_dim) {
    return head_dim < 1 ? 0 : (long long)ROT_BWD_BLOCKS * 2 * head_dim * (long long)sizeof(float);
}

int gd_qk_norm_rotary_backward(const gd_rotary_desc *d, const gd_heads *dq_out, const gd_heads *dk_out, const gd_heads *q, const gd_heads *k,
                               const gd_heads *dq, const gd_heads *dk, int heads_q, int heads_k, const void *w_q, const void *w_k, int w_f32,
                               float eps, void *workspace_dev, void *dw_q, void *dw_k, void *stream) {
    static const char *who = "qk_norm_rotary_backward";
    RotaryParams p{};
    GD_TRY(fill_rotary(p, d, who));
    GD_CHECK(heads_q >= 1 && heads_k >= 1 && heads_q <= 65535 && heads_k <= 65535, "%s: %d / %d heads outside [1, 65535]", who, heads_q, heads_k);
    GD_CHECK(eps >= 0.f, "%s: negative eps", who);
    GD_CHECK(workspace_dev, "%s: null workspace", who);
    const bool empty = (long long)p.batch * p.tokens == 0;
    GD_TRY(view(p.dy[0], dq_out, empty, who, "dq_out"));
    GD_TRY(view(p.dy[1], dk_out, empty, who, "dk_out"));
    GD_TRY(view(p.x[0], q, empty, who, "q"));
    GD_TRY(view(p.x[1], k, empty, who, "k"));
    GD_TRY(view(p.out[0], dq, empty, who, "dq"));
    GD_TRY(view(p.out[1], dk, empty, who, "dk"));
    p.heads[0] = heads_q; p.heads[1] = heads_k;
    p.w[0] = w_q; p.w[1] = w_k; p.w_f32 = w_f32; p.eps = eps;
    p.sign = -1.f;
    p.dw_part = static_cast<float *>(workspace_dev);
    return launch_rotary(p, d->dtype, ROT_NORM_BWD, dw_q, dw_k, (hipStream_t)stream);
}

}  // extern "C"
