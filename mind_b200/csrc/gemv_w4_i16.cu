// The 4-bit matrix-vector kernels for int16 activations (two bytes each).
#include "gemv_w4.cuh"

namespace mb200 {
namespace w4 {

int64_t launch_i16(DeviceCtx* ctx, const CUtensorMap& tm, const Plan& plan, int nt) {
    if (nt == 0) return launch_gb<2, 1, true>(ctx, tm, plan);
    if (nt <= 1) return launch_gb<2, 1, false>(ctx, tm, plan);
    if (nt == 2) return launch_gb<2, 2, false>(ctx, tm, plan);
    return launch_gb<2, 4, false>(ctx, tm, plan);
}

}  // namespace w4
}  // namespace mb200
