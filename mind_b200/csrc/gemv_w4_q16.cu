// The 4-bit matrix-vector kernels for Q16.16 activations (four bytes each).
#include "gemv_w4.cuh"

namespace mb200 {
namespace w4 {

int64_t launch_q16(DeviceCtx* ctx, const CUtensorMap& tm, const Plan& plan, int tc) {
    return launch_tc<4>(ctx, tm, plan, tc);
}

}  // namespace w4
}  // namespace mb200
