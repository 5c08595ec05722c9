// C entry points of the token operators: argument checks, then the launchers of kernels/.
#include <cfloat>
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

// ---- gated feed-forward block ----
size_t elem_size(int dtype) { return dtype == GD_F32 ? 4 : 2; }

int check_ffn(const gd_ffn_desc *d, const char *who) {
    GD_CHECK(d, "%s: null description", who);
    GD_CHECK(d->dtype == GD_F32 || d->dtype == GD_BF16 || d->dtype == GD_F16, "%s: unknown element type %d", who, d->dtype);
    GD_CHECK(d->act == GD_ACT_SILU || d->act == GD_ACT_GELU || d->act == GD_ACT_GELU_TANH, "%s: unknown activation %d", who, d->act);
    GD_CHECK(d->rows >= 0 && d->in >= 1 && d->hidden >= 1 && d->out >= 1, "%s: bad sizes rows=%d in=%d hidden=%d out=%d", who, d->rows, d->in, d->hidden, d->out);
    const long long most = 1LL << 30;
    GD_CHECK(d->rows <= most && d->in <= most && d->hidden <= most && d->out <= most, "%s: sizes past 2^30", who);
    GD_CHECK((d->rows <= 1 || d->ld_x >= d->in) && (d->hidden <= 1 || d->ld_w_in >= d->in) && (d->out <= 1 || d->ld_w_down >= d->hidden),
             "%s: a leading dimension is shorter than its row", who);
    return 0;
}

struct Matrix {
    const void *p;
    long long rows, cols, ld;  // elements
};

bool pieces_ok(const Matrix &m, bool k_adjacent, size_t es) {
    const long long ld = m.ld * (long long)es;
    return (uintptr_t)m.p % 16 == 0 && ld % 16 == 0 && ld <= (1LL << 22) && (!k_adjacent || m.cols * (long long)es % 16 == 0);
}

// C (M, N) = sum of parts A B; operands as they lie in memory, k adjacent or not
GemmProblem problem(const Matrix *a, bool akc, const Matrix *b, bool bkc, int parts, bool gated, size_t es, int *direct) {
    GemmProblem q{};
    q.M = (int)(akc ? a[0].rows : a[0].cols);
    q.N = (int)(bkc ? b[0].rows : b[0].cols);
    q.K = (int)(akc ? a[0].cols : a[0].rows);
    q.parts = parts;
    // Whole dwords: a read is held against the end dword by dword, and of a 16-bit matrix with an odd number of columns the last element lies in the first half of
    // one (the other half is padding of the row, or memory of the same aligned dword; it only meets columns that are not stored)
    auto bytes = [&](const Matrix &m) { return m.rows ? (((m.rows - 1) * m.ld + m.cols) * (long long)es + 3) / 4 * 4 : 0; };
    q.lda = a[0].ld * es; q.ldb = b[0].ld * es;
    q.a_bytes = bytes(a[0]); q.b_bytes = bytes(b[0]);
    for (int s = 0; s < 2; ++s) {
        const Matrix &ma = a[parts == 2 ? s : 0], &mb = b[parts == 2 || gated ? s : 0];
        q.a[s] = ma.p; q.b[s] = mb.p;
        if (!pieces_ok(ma, akc, es) || !pieces_ok(mb, bkc, es)) *direct = 0;
    }
    return q;
}

constexpr long long MAX_THREADS = (1LL << 32) - 1;  // of a launch: more are refused

// tile and split of a launch; returns the floats of partial sums it needs, or -1 (more workgroups than a grid holds)
long long plan_gemm(GemmLaunch &l, int dtype, GemmKind kind) {
    const bool gated = kind == GEMM_GATE_UP;
    const long long cus = device_cus();
    // Few rows: the weight-streaming kernel, where it is estimated to be faster than tiles.  Its time is what its workgroups read, mostly from L2: their rows of
    // the weights and their rows of x, once for each workgroup.  us of gate and up, then of y, in this kernel and (in brackets) in the best tiles, joins with them:
    // 64 x 1024 x 4096 in fp16 12.9 (14.1), 9.6 (18.6); 96 rows 16.1 (15.6), 12.9 (19.2); 128 x 256 x 688 bf16 5.0 (7.2), 3.6 (10.8); 1 x 4096 x 14336 70 (79), 32 (63);
    // 64 rows 147 (90), 88 (41); 96 x 2048 x 8192 51 (29), 34 (22); 96 x 1024 x 4096 float32 32 (29), 27 (23).  16 x 4096 x 14336 is where the estimate errs most:
    // 79 here for gate and up, 97 in the tiles it takes.
    double skinny_us = 1e30;
    int skinny_m = 0, skinny_rows = 16, skinny_tiles = 0;
    long long skinny_grid = 0;
    if ((kind == GEMM_GATE_UP || kind == GEMM_DOWN) && l.direct && l.q[0].M >= 1 && l.q[0].M <= 256) {
        const GemmProblem &q = l.q[0];
        const int m_tiles = (q.M + 15) / 16;
        const long long slices = (q.N + 15) / 16;
        int groups = (m_tiles + 2) / 3;
        while (groups < m_tiles && slices * groups < cus) ++groups;
        skinny_m = (m_tiles + groups - 1) / groups;
        skinny_tiles = (m_tiles + skinny_m - 1) / skinny_m;
        while (skinny_m == 1 && skinny_rows > 4 && 2LL * m_tiles * ((q.N + skinny_rows - 1) / skinny_rows) <= cus) skinny_rows /= 2;
        skinny_grid = (q.N + 8LL * skinny_rows - 1) / (8LL * skinny_rows) * 8 * skinny_tiles;
        const int rows_read = skinny_rows * (gated ? 2 : 1) + (16 * skinny_m < q.M ? 16 * skinny_m : q.M);
        if (skinny_grid * 1024 <= MAX_THREADS) skinny_us = 3 + (dtype == GD_F32 ? 0.2e-6 : 0.14e-6) * (double)skinny_grid * q.K * (double)elem_size(dtype) * rows_read;
    }
    const int kstage = 128 / (int)elem_size(dtype);  // gated_ffn_gemm.h: bytes of k a stage
    struct Shape { GemmTile tile; int m, n; };
    const Shape shapes[3] = {{TILE_128, 128, 128}, {TILE_256, 256, 256}, {TILE_NARROW, 128, 64}};
    auto tiles_n = [&](const GemmProblem &q, int bn) { const int n = gated ? bn / 2 : bn; return (q.N + n - 1LL) / n; };
    auto stages_of = [&](const GemmProblem &q) { return q.K ? (long long)q.parts * ((q.K + kstage - 1) / kstage) : 1; };
    // Tile and split of the sums by estimated time, in us.  A 256 x 256 tile holds a CU, smaller ones share it by two or more; a CU with c tiles takes c times a
    // stage's time per stage, and a fixed time for the way in and out.  Split sums are written and read again by the join.  The constants are fits to y
    // = h Wd^T of 16384 x 1024, K = 256, 512, 1024, 4096, in bf16 (256: 16.5, 24.0, 40.3, 139.6 us; 128: 18.3, 26.9, 42.5, 163.2) and to one and two 128 tiles a CU
    // (17, 24 us at K = 1024); operands whose k is not adjacent cost the small tile more (the weights' gradients of 16384 x 1024 x 4096: 392 us with 256,
    // 488 with 128); split four ways over all CUs these gradients' 192 tiles take 369 us and the join 44.
    // Tiles of 128 x 64 cost more per product but fill narrow matrices and the last round of tiles better.  float32, whose matrix core is 16 times slower: 8192
    // x 1024 x 4096 gate and up 1.11 ms (1.03 with 128 x 128), 6080 x 192 x 2464 down 63 us (92), dx 110 (166), the weights' gradients 174 (200); gate and up of
    // 4096 x 256 x 684 34.8 (40.9).  bf16: 2048 x 1024 x 4096 down 44 us (37), 10069 x 344 x 1208 25 (28), dhidden 51 (58; 66 with 256), of 658 x 184 x 2712 12 (17):
    // each tile of dhidden waits for the projections it reads, once for every 32 rows of a wave (one, two or four times in a tile).  Through registers a stage takes two to three times as long
    // (428 x 884 x 2764 in fp16: dhidden 28 us, 45 with 128 x 128; dx 28, 58).
    // Where it errs: gate and up that are kept, with few stages (16384 x 64 x 512: 30 us with 256, 18 with 128); profiles/token_ops_tile_times.csv holds these and more.
    struct Cost { double alone, shared; };  // us a stage and tile
    const bool f32 = dtype == GD_F32, dhidden = kind == GEMM_DHIDDEN;
    const Cost wide = f32 ? Cost{2.45, 2.0} : Cost{1.05, kind == GEMM_DW ? 0.6 : dhidden || kind == GEMM_DX ? 0.65 : 0.57};
    const Cost narrow = f32 ? Cost{1.45, 1.09} : Cost{0.85, kind == GEMM_DW ? 0.5 : dhidden ? 0.53 : 0.43};
    const long long stages = stages_of(l.q[0]);
    double best = 1e30;
    long long best_split = 1;
    Shape chosen = shapes[0];
    for (const Shape &t : shapes) {
        if (t.tile == TILE_256 && (dtype == GD_F32 || !l.direct)) continue;
        long long n = 0, joins = 0;
        double out = 0;
        for (int i = 0; i < l.problems; ++i) {
            joins += (l.q[i].M * ((l.q[i].N + 3LL) / 4) + 255) / 256 * 256;
            n += ((l.q[i].M + t.m - 1LL) / t.m) * tiles_n(l.q[i], t.n);
            out += (double)l.q[i].M * l.q[i].N * (gated ? 2 : 1);
        }
        if (n > (1LL << 30)) {
            if (skinny_us < 1e30) continue;
            return -1;
        }
        for (long long s = 1; s <= 16 && s <= stages && (s == 1 || stages / s >= 4); ++s) {
            if (s > 1 && joins > MAX_THREADS) break;
            const double per = (double)((stages + s - 1) / s), c = (double)((n * s + cus - 1) / cus);
            double us;
            if (t.tile == TILE_256) us = c * ((kind != GEMM_DW ? 1.9 : n * s < cus ? 1.7 : 2.1) * per + 3) + 5;
            else {
                const Cost &k = t.tile == TILE_NARROW ? narrow : wide;
                us = c <= 1 ? k.alone * per + 5 : k.shared * c * per + 8;
                if (!f32 && !l.direct) us += (kind == GEMM_DW ? 1.5 : t.tile == TILE_NARROW ? 0.7 : 1.1) * (c <= 1 ? k.alone : k.shared * c) * per;
            }
            if (dhidden && f32) us += c <= 1 ? out * 16 / 4.5e6 : 0;
            else if (dhidden) us += out * 12 / 7e6 / (t.tile == TILE_256 ? c : c > 2 ? c / 2 : 1) + (t.tile == TILE_256 ? 16 : t.tile == TILE_128 ? 8 : 4);
            if (s > 1) us += 4 + (double)s * out * 8 / 4.5e6;
            if (us < best) {
                best = us;
                best_split = s;
                chosen = t;
            }
        }
    }
    if (skinny_us <= best && skinny_us < 1e30) {
        l.tile = TILE_SKINNY;
        l.skinny_m = skinny_m;
        l.skinny_rows = skinny_rows;
        l.q[0].tiles_m = skinny_tiles;
        l.q[0].splits = 1;
        l.grid = l.blocks = (int)skinny_grid;
        l.join_blocks = 0;
        return 0;
    }
    l.tile = chosen.tile;
    const long long room = l.tile == TILE_256 ? cus : 2 * cus;
    long long floats = 0, join = 0, blocks = 0;
    for (int i = 0; i < l.problems; ++i) {
        GemmProblem &q = l.q[i];
        q.tiles_m = (int)((q.M + chosen.m - 1LL) / chosen.m);
        q.tiles_n = (int)tiles_n(q, chosen.n);
        q.stages_per_split = (int)((stages_of(q) + best_split - 1) / best_split);
        q.splits = (int)((stages_of(q) + q.stages_per_split - 1) / q.stages_per_split);
        q.blocks = q.tiles_m * q.tiles_n * q.splits;
        blocks += q.blocks;
        q.join_threads = 0;
        if (q.splits > 1) {
            const long long n4 = (q.N + 3LL) / 4 * 4;
            q.join_threads = ((long long)q.M * (n4 / 4) + 255) / 256 * 256;
            floats += (long long)q.splits * (gated ? 2 : 1) * q.M * n4;
        }
        join += q.join_threads;
    }
    if (blocks > (1LL << 30)) return -1;
    l.join_blocks = (int)(join / 256);
    l.blocks = (int)blocks;
    l.grid = (int)(blocks < room ? blocks : room / 8 * 8);  // a workgroup's pieces stay on its XCD
    return floats;
}

int run_gemm(GemmLaunch &l, int dtype, GemmKind kind, float *partial, hipStream_t s, const char *who) {
    const bool gated = kind == GEMM_GATE_UP;
    GD_CHECK(plan_gemm(l, dtype, kind) >= 0, "%s: too many tiles for one launch", who);
    for (int i = 0; i < l.problems; ++i) {
        GemmProblem &q = l.q[i];
        q.short_rows = q.N < (1 << 23);
        q.partial = partial;
        if (q.splits > 1) partial += (long long)q.splits * (gated ? 2 : 1) * q.M * ((q.N + 3LL) / 4 * 4);
    }
    switch (dtype) {
        case GD_BF16: return launch_ffn_gemm_bf16(l, kind, s);
        case GD_F16: return launch_ffn_gemm_f16(l, kind, s);
        default: return launch_ffn_gemm_f32(l, kind, s);
    }
}

struct FfnLaunches {
    GemmLaunch l[5];  // by GemmKind
};

// the block's five launches, without what is only known at the call (outputs); null pointers count as aligned
FfnLaunches ffn_launches(const gd_ffn_desc *d, const void *x, const void *wg, const void *wu, const void *wd, const void *hidden, const void *dy,
                         long long ld_dy, const void *dgate, const void *dup) {
    const size_t es = elem_size(d->dtype);
    auto matrix = [](const void *p, long long rows, long long cols, long long ld) { return Matrix{p, rows, cols, rows <= 1 ? cols : ld}; };
    const Matrix X = matrix(x, d->rows, d->in, d->ld_x), Wg = matrix(wg, d->hidden, d->in, d->ld_w_in), Wu = matrix(wu, d->hidden, d->in, d->ld_w_in),
                 Wd = matrix(wd, d->out, d->hidden, d->ld_w_down), H = matrix(hidden, d->rows, d->hidden, d->hidden),
                 DY = matrix(dy, d->rows, d->out, ld_dy), DG = matrix(dgate, d->rows, d->hidden, d->hidden), DU = matrix(dup, d->rows, d->hidden, d->hidden);
    FfnLaunches f{};
    for (auto &l : f.l) { l.problems = 1; l.direct = !d->unaligned; l.act = d->act; }
    const Matrix w_in[2] = {Wg, Wu}, d_in[2] = {DG, DU};
    f.l[GEMM_GATE_UP].q[0] = problem(&X, true, w_in, true, 1, true, es, &f.l[GEMM_GATE_UP].direct);
    f.l[GEMM_DOWN].q[0] = problem(&H, true, &Wd, true, 1, false, es, &f.l[GEMM_DOWN].direct);
    f.l[GEMM_DHIDDEN].q[0] = problem(&DY, true, &Wd, false, 1, false, es, &f.l[GEMM_DHIDDEN].direct);
    f.l[GEMM_DX].q[0] = problem(d_in, true, w_in, false, 2, false, es, &f.l[GEMM_DX].direct);
    GemmLaunch &w = f.l[GEMM_DW];
    w.problems = 3;
    w.q[0] = problem(&DG, false, &X, false, 1, false, es, &w.direct);
    w.q[1] = problem(&DU, false, &X, false, 1, false, es, &w.direct);
    w.q[2] = problem(&DY, false, &H, false, 1, false, es, &w.direct);
    return f;
}

long long align_up(long long n) { return (n + 255) / 256 * 256; }

// the same as the workspace's size is computed from: aligned tensors, dense rows of dy
FfnLaunches ffn_sizing(const gd_ffn_desc *d) {
    return ffn_launches(d, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, d->out, nullptr, nullptr);
}

// floats of partial sums that the given launches need
long long partial_floats(FfnLaunches f, int dtype, int first, int last) {
    long long most = 0;
    for (int k = first; k <= last; ++k) {
        const long long n = plan_gemm(f.l[k], dtype, (GemmKind)k);
        if (n > most) most = n;
    }
    return most;
}

// The launches take the path that the workspace was sized for.  Rows of dy may be aligned where dense ones, which that takes for granted, are not
int as_sized(FfnLaunches &f, const gd_ffn_desc *d, int first, int last, const char *who) {
    const FfnLaunches sized = ffn_sizing(d);
    for (int k = first; k <= last; ++k) {
        GD_CHECK(f.l[k].direct || !sized.l[k].direct, "%s: a tensor does not start (or rows of dy are not apart by) a multiple of 16 bytes: set unaligned", who);
        f.l[k].direct = sized.l[k].direct;
    }
    return 0;
}

}  // namespace

extern "C" {

long long gd_gated_ffn_workspace(const gd_ffn_desc *d, int backward) {
    if (check_ffn(d, "gated_ffn_workspace")) return -1;
    const FfnLaunches f = ffn_sizing(d);
    if (!backward) return partial_floats(f, d->dtype, GEMM_GATE_UP, GEMM_DOWN) * (long long)sizeof(float);
    const long long grad = align_up((long long)d->rows * d->hidden * (long long)elem_size(d->dtype));
    return 2 * grad + partial_floats(f, d->dtype, GEMM_DHIDDEN, GEMM_DW) * (long long)sizeof(float);
}

int gd_gated_ffn(const gd_ffn_desc *d, const void *x, const void *w_gate, const void *w_up, const void *w_down, float *gate_dev, float *up_dev,
                 void *hidden_dev, void *y, void *workspace_dev, void *stream) {
    static const char *who = "gated_ffn";
    GD_TRY(check_ffn(d, who));
    const bool empty = d->rows == 0;
    GD_CHECK(w_gate && w_up && w_down && (empty || (x && hidden_dev && y)), "%s: null pointer", who);
    GD_CHECK(!gate_dev == !up_dev, "%s: gate and up are kept both or neither", who);
    if (empty) return 0;
    GD_CHECK((uintptr_t)workspace_dev % 16 == 0, "%s: workspace not aligned to 16 bytes", who);
    GD_CHECK(workspace_dev || gd_gated_ffn_workspace(d, 0) == 0, "%s: null workspace", who);
    FfnLaunches f = ffn_launches(d, x, w_gate, w_up, w_down, hidden_dev, nullptr, d->out, nullptr, nullptr);
    GD_TRY(as_sized(f, d, GEMM_GATE_UP, GEMM_DOWN, who));
    GemmLaunch &g = f.l[GEMM_GATE_UP], &o = f.l[GEMM_DOWN];
    g.q[0].out[0] = hidden_dev; g.q[0].out[1] = gate_dev; g.q[0].out[2] = up_dev;
    o.q[0].out[0] = y;
    GD_TRY(run_gemm(g, d->dtype, GEMM_GATE_UP, static_cast<float *>(workspace_dev), (hipStream_t)stream, who));
    return run_gemm(o, d->dtype, GEMM_DOWN, static_cast<float *>(workspace_dev), (hipStream_t)stream, who);
}

int gd_gated_ffn_backward(const gd_ffn_desc *d, const void *dy, long long ld_dy, const void *x, const void *w_gate, const void *w_up,
                          const void *w_down, const float *gate, const float *up, const void *hidden, void *dx, void *dw_gate, void *dw_up,
                          void *dw_down, void *workspace_dev, void *stream) {
    static const char *who = "gated_ffn_backward";
    GD_TRY(check_ffn(d, who));
    const bool empty = d->rows == 0;
    GD_CHECK(w_gate && w_up && w_down && dw_gate && dw_up && dw_down && (empty || (dy && x && gate && up && hidden && dx && workspace_dev)), "%s: null pointer", who);
    GD_CHECK(d->rows <= 1 || ld_dy >= d->out, "%s: a leading dimension is shorter than its row", who);
    GD_CHECK((uintptr_t)workspace_dev % 16 == 0, "%s: workspace not aligned to 16 bytes", who);
    const long long grad = align_up((long long)d->rows * d->hidden * (long long)elem_size(d->dtype));
    char *ws = static_cast<char *>(workspace_dev);
    void *dgate = ws, *dup = ws ? ws + grad : nullptr;
    float *partial = reinterpret_cast<float *>(ws ? ws + 2 * grad : nullptr);
    FfnLaunches f = ffn_launches(d, x, w_gate, w_up, w_down, hidden, dy, ld_dy, dgate, dup);
    GD_TRY(as_sized(f, d, empty ? GEMM_DW : GEMM_DHIDDEN, GEMM_DW, who));
    hipStream_t s = (hipStream_t)stream;
    if (!empty) {
        GemmProblem &h = f.l[GEMM_DHIDDEN].q[0];
        h.out[0] = dgate; h.out[1] = dup;
        h.in[0] = gate; h.in[1] = up;
        GD_TRY(run_gemm(f.l[GEMM_DHIDDEN], d->dtype, GEMM_DHIDDEN, partial, s, who));
        f.l[GEMM_DX].q[0].out[0] = dx;
        GD_TRY(run_gemm(f.l[GEMM_DX], d->dtype, GEMM_DX, partial, s, who));
    }
    GemmLaunch &w = f.l[GEMM_DW];
    w.q[0].out[0] = dw_gate; w.q[1].out[0] = dw_up; w.q[2].out[0] = dw_down;
    return run_gemm(w, d->dtype, GEMM_DW, partial, s, who);
}

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
    GD_CHECK(eps >= 0.f && eps <= FLT_MAX, "%s: eps %g is negative or not a finite float32", who, eps);
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
    GD_CHECK(eps >= 0.f && eps <= FLT_MAX, "%s: eps %g is negative or not a finite float32", who, eps);
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
