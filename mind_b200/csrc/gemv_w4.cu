// Matrix-vector products with 4-bit weights and group scales.
//
//   d[t,r,g] = sum_{k in group g} w[r,k] * x[t,k]            w in [-8, 7], x int8 / int16 / Q16.16
//   y[t,r]   = (i32)( ( sum_g scale[r,g] * d[t,r,g] ) >> shift )
//
// The sum over groups is taken mod 2^64 and is exact for every operand a model holds
// (|sum| < 2^49 * cols for Q16.16, 2^33 * cols for int16, 2^25 * cols for int8); it is shifted
// once and truncated once, so any order of accumulation gives the same bits.
//
// Weights: two a byte, the even column in the low half, rows of ceil(cols / 2) bytes.
#include "common.h"

namespace mb200 {
namespace {

template <int KIND>
__device__ __forceinline__ int32_t load_x(const void* x, int64_t i) {
    if (KIND == 0) return static_cast<const int8_t*>(x)[i];
    if (KIND == 1) return static_cast<const int16_t*>(x)[i];
    return static_cast<const int32_t*>(x)[i];
}

// The expert of output row p, or -1, for a whole warp: bounds run no lower than the one before, so the
// first offset above p ends the rows of the expert before it.
__device__ __forceinline__ int expert_of(const int32_t* offsets, int64_t experts, int64_t p, int lane) {
    if (!offsets) return 0;
    for (int64_t j0 = 0; j0 <= experts; j0 += 32) {
        const unsigned above = __ballot_sync(0xffffffffu, j0 + lane <= experts && offsets[min(j0 + lane, experts)] > p);
        if (above) return (int)j0 + __ffs(above) - 2;
    }
    return -1;
}

// One warp per output: the cross-check kernel, any size and alignment.
template <int KIND>
__global__ void __launch_bounds__(256)
gemv_w4_warp_kernel(const W4Args a) {
    const int lane = threadIdx.x & 31;
    const int64_t warp = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5;
    const int64_t nwarps = ((int64_t)gridDim.x * blockDim.x) >> 5;
    const int64_t pitch = (a.cols + 1) / 2, groups = (a.cols + a.group - 1) / a.group;
    for (int64_t o = warp; o < a.m * a.rows; o += nwarps) {
        const int64_t p = o / a.rows, r = o - p * a.rows;
        const int e = expert_of(a.offsets, a.experts, p, lane);
        if (e < 0) continue;
        const int64_t xr = a.rows_of ? a.rows_of[p] : p;
        const bool has_x = xr >= 0 && xr < a.x_rows;
        const int8_t* w = a.w + ((int64_t)e * a.rows + r) * pitch;
        const int16_t* s = a.scale + ((int64_t)e * a.rows + r) * groups;
        uint64_t acc = 0;
        for (int64_t i = lane; has_x && i < pitch; i += 32) {
            const int32_t b = w[i];
            const int64_t k = 2 * i;
            int64_t d = (int64_t)((int32_t)((uint32_t)b << 28) >> 28) * load_x<KIND>(a.x, xr * a.cols + k);
            if (k + 1 < a.cols) d += (int64_t)(b >> 4) * load_x<KIND>(a.x, xr * a.cols + k + 1);
            acc += (uint64_t)(d * s[k / a.group]);
        }
        for (int q = 16; q > 0; q >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, q);
        if (lane == 0) a.y[o] = (int32_t)((int64_t)acc >> a.shift);
    }
}

}  // namespace

int64_t launch_gemv_w4(DeviceCtx* ctx, const W4Args& a) {
    int64_t blocks = (a.m * a.rows + 7) / 8;
    if (blocks > (int64_t)ctx->sm_count * 64) blocks = (int64_t)ctx->sm_count * 64;
    prof_begin(ctx);
    if (a.kind == 0)
        gemv_w4_warp_kernel<0><<<(unsigned)blocks, 256, 0, ctx->stream>>>(a);
    else if (a.kind == 1)
        gemv_w4_warp_kernel<1><<<(unsigned)blocks, 256, 0, ctx->stream>>>(a);
    else
        gemv_w4_warp_kernel<2><<<(unsigned)blocks, 256, 0, ctx->stream>>>(a);
    prof_end(ctx);
    count_launch();
    return check_launch("gemv_w4_warp_kernel");
}

}  // namespace mb200
