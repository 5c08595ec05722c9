// Gated feed-forward block, element type __bf16.
#include "gated_ffn_gemm.h"

namespace gd {

int launch_ffn_gemm_bf16(const GemmLaunch &p, GemmKind kind, hipStream_t s) { return ffn::launch_type<__bf16>(p, kind, s); }

}  // namespace gd
