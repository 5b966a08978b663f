// The 4-bit matrix-vector kernels for int16 activations (two bytes each).
#include "gemv_w4.cuh"

namespace mb200 {
namespace w4 {

int64_t launch_i16(DeviceCtx* ctx, const CUtensorMap& tm, const Plan& plan, int tc) {
    return launch_tc<2>(ctx, tm, plan, tc);
}

}  // namespace w4
}  // namespace mb200
