// Gated feed-forward block, element type _Float16.
#include "gated_ffn_gemm.h"

namespace gd {

int launch_ffn_gemm_f16(const GemmLaunch &p, GemmKind kind, hipStream_t s) { return ffn::launch_type<_Float16>(p, kind, s); }

}  // namespace gd
