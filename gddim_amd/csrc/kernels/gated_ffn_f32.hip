// Gated feed-forward block, element type float.
#include "gated_ffn_gemm.h"

namespace gd {

int launch_ffn_gemm_f32(const GemmLaunch &p, GemmKind kind, hipStream_t s) { return ffn::launch_type<float>(p, kind, s); }

}  // namespace gd
