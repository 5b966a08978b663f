// The 4-bit matrix-vector kernels for int8 activations (one byte each).
#include "gemv_w4.cuh"

namespace mb200 {
namespace w4 {

int cluster_fit(DeviceCtx* ctx, int cs) {
    if (cs == 1) return ctx->sm_count;
    static thread_local int dev = -1, fit[9];
    if (dev != ctx->device) {
        dev = ctx->device;
        for (int& f : fit) f = -1;
    }
    if (fit[cs] >= 0) return fit[cs];
    auto kern = gemv_w4_mma_kernel<1, 1, 4>;
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX);
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)(ctx->sm_count / cs * cs), 1, 1);
    lc.blockDim = dim3(THREADS, 1, 1);
    lc.dynamicSmemBytes = SMEM_MAX;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cs;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    lc.attrs = at;
    lc.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &lc) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
    }
    return fit[cs] = n;
}

int64_t launch_i8(DeviceCtx* ctx, const CUtensorMap& tm, const Plan& plan, int tc) {
    return launch_tc<1>(ctx, tm, plan, tc);
}

}  // namespace w4
}  // namespace mb200
