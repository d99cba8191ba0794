// insmos_amd/csrc/linear_f16.hip -- the matrix product of linear.h for f16 (one source per type: they compile side by side).
#include "linear.h"

namespace insmos {
namespace lin {
int launch_gemm_f16(const GemmP& p, int la, int lb, int tile, hipStream_t s) { return launch_gemm<_Float16>(p, la, lb, tile, s); }
}  // namespace lin
}  // namespace insmos
