// Grouping of routed tokens by expert: a stable counting sort of small integers.
//
//   offsets[e] = #{ i : 0 <= ids[i] < e }          (e = 0 .. experts)
//   the kept i, in order of (ids[i], i), are p = 0, 1, ...:  rows[p] = i / per,  place[i] = p
//   place[i] = -1 where ids[i] names no expert (padding)
//
// One block.  Every warp owns a contiguous piece of the ids and a histogram of its own in shared
// memory; two passes over the ids (count, then place) with a scan of the histograms between them,
// expert-major and warp-minor, which is what makes the order stable.  Inside 32 ids the rank of a
// lane among the lanes of the same expert is a population count of __match_any_sync's mask, so no
// atomics are used and the result does not depend on timing.
#include "common.h"

namespace mb200 {
namespace {

__global__ void __launch_bounds__(1024)
expert_plan_kernel(const int32_t* __restrict__ ids, int32_t* __restrict__ offsets, int32_t* __restrict__ rows,
                   int32_t* __restrict__ place, int64_t count, int experts, int64_t per) {
    extern __shared__ int32_t hist[];  // [warps][experts]
    __shared__ int32_t warp_sum[32];
    __shared__ int32_t carry;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    for (int i = threadIdx.x; i < warps * experts; i += blockDim.x) hist[i] = 0;
    if (threadIdx.x == 0) carry = 0;
    __syncthreads();
    const int64_t piece = (count + warps - 1) / warps;
    const int64_t first = warp * piece, last = first + piece < count ? first + piece : count;
    int32_t* const mine = hist + warp * experts;

    // pass 1: how many ids of each expert this warp's piece holds
    for (int64_t i0 = first; i0 < last; i0 += 32) {
        const int64_t i = i0 + lane;
        const int32_t id = i < last ? ids[i] : -1;
        const bool ok = id >= 0 && id < experts;
        const unsigned same = __match_any_sync(0xffffffffu, ok ? id : -1);
        if (ok && (same & ((1u << lane) - 1u)) == 0) mine[id] += __popc(same);
        __syncwarp();
    }
    __syncthreads();

    // exclusive scan over (expert, warp), a block of experts at a time; hist becomes first positions
    for (int e0 = 0; e0 < experts; e0 += blockDim.x) {
        const int e = e0 + threadIdx.x;
        int32_t total = 0;
        if (e < experts)
            for (int w = 0; w < warps; ++w) total += hist[w * experts + e];
        int32_t incl = total;
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) warp_sum[warp] = incl;
        __syncthreads();
        int32_t before = carry;
        for (int w = 0; w < warp; ++w) before += warp_sum[w];
        int32_t at = before + incl - total;
        if (e < experts) {
            offsets[e] = at;
            for (int w = 0; w < warps; ++w) {
                const int32_t n = hist[w * experts + e];
                hist[w * experts + e] = at;
                at += n;
            }
        }
        __syncthreads();
        if (threadIdx.x == blockDim.x - 1) carry = before + incl;
        __syncthreads();
    }
    if (threadIdx.x == 0) offsets[experts] = carry;

    // pass 2: every id takes the next position of its expert within its warp's share
    for (int64_t i0 = first; i0 < last; i0 += 32) {
        const int64_t i = i0 + lane;
        const int32_t id = i < last ? ids[i] : -1;
        const bool ok = id >= 0 && id < experts;
        const unsigned same = __match_any_sync(0xffffffffu, ok ? id : -1);
        const int rank = __popc(same & ((1u << lane) - 1u));
        int32_t base = 0;
        if (ok) base = mine[id];
        __syncwarp();
        if (ok && rank == 0) mine[id] = base + __popc(same);
        __syncwarp();
        if (i < last) {
            if (ok) rows[base + rank] = (int32_t)(i / per);
            place[i] = ok ? base + rank : -1;
        }
    }
}

}  // namespace

int64_t launch_expert_plan(DeviceCtx* ctx, const int32_t* ids, int32_t* offsets, int32_t* rows, int32_t* place,
                           int64_t count, int64_t experts, int64_t per) {
    // as many warps as the histograms leave room for (at least four: 4096 experts take 64 KiB)
    int warps = 32;
    while (warps > 4 && (size_t)warps * experts * 4 > (size_t)128 << 10) warps >>= 1;
    const size_t smem = (size_t)warps * experts * 4;
    MB200_CUDA(cudaFuncSetAttribute(expert_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 << 10));
    prof_begin(ctx);
    expert_plan_kernel<<<1, warps * 32, smem, ctx->stream>>>(ids, offsets, rows, place, count, (int)experts, per);
    prof_end(ctx);
    count_launch();
    return check_launch("expert_plan_kernel");
}

}  // namespace mb200
