// Host side of the token operators with launchers that write down what they are asked for: the launches' shapes are checked without a GPU.
#include "../gddim_amd/csrc/token_ops.cpp"

namespace gd {

void set_error(const char *, ...) {}
int device_cus() { return 256; }

static GemmLaunch asked[8];
static int kinds[8], count;

static int write_down(const GemmLaunch &p, GemmKind kind) {
    if (count < 8) {
        asked[count] = p;
        kinds[count++] = kind;
    }
    return 0;
}

int launch_ffn_gemm_bf16(const GemmLaunch &p, GemmKind kind, hipStream_t) { return write_down(p, kind); }
int launch_ffn_gemm_f16(const GemmLaunch &p, GemmKind kind, hipStream_t) { return write_down(p, kind); }
int launch_ffn_gemm_f32(const GemmLaunch &p, GemmKind kind, hipStream_t) { return write_down(p, kind); }
int launch_rotary(RotaryParams, int, RotaryMode, void *, void *, hipStream_t) { return 0; }

}  // namespace gd

extern "C" {

void forget_launches() { gd::count = 0; }
int launches() { return gd::count; }
// kind, tile, workgroups, threads of a workgroup, workgroups of the join, furthest byte of partial sums
void launch(int i, long long *out) {
    const gd::GemmLaunch &l = gd::asked[i];
    out[0] = gd::kinds[i];
    out[1] = l.tile;
    out[2] = l.grid;
    out[3] = l.tile == gd::TILE_SKINNY ? 1024 : l.tile == gd::TILE_256 ? 512 : 256;
    out[4] = l.join_blocks;
    out[5] = 0;
    for (int k = 0; k < l.problems; ++k) {
        const gd::GemmProblem &q = l.q[k];
        if (q.splits > 1)
            out[5] = (long long)(size_t)(q.partial + (long long)q.splits * (gd::kinds[i] == gd::GEMM_GATE_UP ? 2 : 1) * q.M * ((q.N + 3LL) / 4 * 4));
    }
}

}  // extern "C"
