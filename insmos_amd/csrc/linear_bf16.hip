// insmos_amd/csrc/linear_bf16.hip -- the matrix product of linear.h for bf16 (one source per type: they compile side by side).
#include "linear.h"

namespace insmos {
namespace lin {
int launch_gemm_bf16(const GemmP& p, int la, int lb, int tile, hipStream_t s) { return launch_gemm<__bf16>(p, la, lb, tile, s); }
}  // namespace lin
}  // namespace insmos
