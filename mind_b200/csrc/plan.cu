// Grouping of routed tokens by expert: a stable counting sort of small integers.
//
//   offsets[e] = #{ i : 0 <= ids[i] < e }          (e = 0 .. experts)
//   the kept i, in order of (ids[i], i), are p = 0, 1, ...:  rows[p] = i / per,  place[i] = p
//   place[i] = -1 where ids[i] names no expert (padding)
//
// Every warp owns a contiguous piece of the ids and a
// histogram of its own in shared memory; two passes over the ids (count, then place) with a scan of the
// histograms between them, expert-major and (block, warp)-minor, which is what makes the order stable.
// Up to 16384 ids take one launch of one cluster of 1, 2, 4 or 8 blocks, which meet in shared memory: each
// publishes its totals per expert and reads the others' remotely.  More ids take two launches of up to one
// block per SM: the first leaves the blocks' totals in scratch, the second counts again, adds them up and
// places (300126 ids over 160 experts: 75 us on a cluster, whose eight SMs are bound by their scattered
// stores).  Either way no block waits for one that may not be running.
//
// Inside 32 ids the rank of a lane among the lanes of the same expert is a population count of
// __match_any_sync's mask, so no atomics are used and the result does not depend on timing.
// Bound by latency: a warp's 32 ids at a time depend on the histogram the 32 before them left, which is
// why many short pieces (up to 8 x 32 warps) and not a few long ones.
#include "common.h"
#include "ptx.cuh"

namespace mb200 {
using namespace ptx;
namespace {

constexpr int MAX_CLUSTER = 8;

// Expert e's count over the warps (a multiple of four), four loads at a time.
__device__ __forceinline__ int32_t column(const int32_t* hist, int warps, int experts, int e) {
    int32_t n[4] = {0, 0, 0, 0};
    for (int w = 0; w < warps; w += 4)
#pragma unroll
        for (int j = 0; j < 4; ++j) n[j] += hist[(w + j) * experts + e];
    return n[0] + n[1] + n[2] + n[3];
}

// Shared memory: hist[warps][experts], then (clusters) total[experts].
__global__ void __launch_bounds__(1024)
expert_plan_kernel(const int32_t* __restrict__ ids, int32_t* __restrict__ offsets, int32_t* __restrict__ rows,
                   int32_t* __restrict__ place, int64_t count, int experts, unsigned per, int blocks, int phase,
                   int32_t* __restrict__ totals) {  // phase 0: a cluster does it all; 1: count; 2: place
    extern __shared__ int32_t hist[];
    __shared__ int32_t warp_sum[32];
    __shared__ int32_t carry;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int block = blockIdx.x;
    const bool cluster = phase == 0 && blocks > 1;  // the grid is one cluster
    int32_t* const total = hist + warps * experts;
    griddep_launch_dependents();
    for (int i = threadIdx.x; i < warps * experts; i += blockDim.x) hist[i] = 0;
    if (threadIdx.x == 0) carry = 0;
    griddep_wait();  // the ids may be the work of the kernel before this one
    __syncthreads();
    // this warp's piece, a multiple of 32 ids
    const int64_t groups = (count + 31) / 32, pieces = (int64_t)warps * blocks;
    const int64_t piece = (groups + pieces - 1) / pieces * 32;
    const int64_t first = min((int64_t)(block * warps + warp) * piece, count), last = min(first + piece, count);
    int32_t* const mine = hist + warp * experts;
    constexpr int U = 4;  // groups of 32 ids fetched at a time

    // pass 1: how many ids of each expert this warp's piece holds
    for (int64_t i0 = first; i0 < last; i0 += 32 * U) {
        int32_t id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = i0 + 32 * u + lane;
            id[u] = i < last ? ids[i] : -1;
            if ((unsigned)id[u] >= (unsigned)experts) id[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const unsigned same = __match_any_sync(0xffffffffu, id[u]);
            if (id[u] >= 0 && (same & ((1u << lane) - 1u)) == 0) mine[id[u]] += __popc(same);
            __syncwarp();
        }
    }
    __syncthreads();
    if (phase == 1) {
        for (int e = threadIdx.x; e < experts; e += blockDim.x) {
            totals[block * experts + e] = column(hist, warps, experts, e);
        }
        return;
    }
    if (cluster) {  // publish this block's totals
        for (int e = threadIdx.x; e < experts; e += blockDim.x) {
            total[e] = column(hist, warps, experts, e);
        }
        cluster_arrive();
        cluster_wait();
    }

    // exclusive scan over (expert, block, warp), a block of experts at a time; hist becomes first positions
    for (int e0 = 0; e0 < experts; e0 += blockDim.x) {
        const int e = e0 + threadIdx.x;
        int32_t all = 0, before_me = 0;  // of this expert: everywhere, and in the blocks before this one
        if (e < experts) {
            if (phase == 2) {
#pragma unroll 8
                for (int b = 0; b < blocks; ++b) {
                    const int32_t n = totals[b * experts + e];
                    all += n;
                    before_me += b < block ? n : 0;
                }
            } else if (cluster) {
                int32_t n[MAX_CLUSTER];
                const uint32_t at = smem_u32(total + e);
#pragma unroll
                for (int b = 0; b < MAX_CLUSTER; ++b) {
                    n[b] = 0;
                    if (b < blocks) asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(n[b]) : "r"(mapa(at, (uint32_t)b)) : "memory");
                }
#pragma unroll
                for (int b = 0; b < MAX_CLUSTER; ++b) {
                    all += n[b];
                    before_me += b < block ? n[b] : 0;
                }
            } else {
                all = column(hist, warps, experts, e);
            }
        }
        int32_t incl = all;
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) warp_sum[warp] = incl;
        __syncthreads();
        int32_t before = carry;
        for (int w = 0; w < warp; ++w) before += warp_sum[w];
        if (e < experts) {
            int32_t at = before + incl - all;
            if (block == 0) offsets[e] = at;
            at += before_me;
            for (int w = 0; w < warps; w += 4) {
                int32_t n[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) n[j] = hist[(w + j) * experts + e];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    hist[(w + j) * experts + e] = at;
                    at += n[j];
                }
            }
        }
        __syncthreads();
        if (threadIdx.x == blockDim.x - 1) carry = before + incl;
        __syncthreads();
    }
    if (block == 0 && threadIdx.x == 0) offsets[experts] = carry;

    // pass 2: every id takes the next position of its expert within its warp's share
    for (int64_t i0 = first; i0 < last; i0 += 32 * U) {
        int32_t id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = i0 + 32 * u + lane;
            id[u] = i < last ? ids[i] : -1;
            if ((unsigned)id[u] >= (unsigned)experts) id[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = i0 + 32 * u + lane;
            const unsigned same = __match_any_sync(0xffffffffu, id[u]);
            const int rank = __popc(same & ((1u << lane) - 1u));
            int32_t base = 0;
            if (id[u] >= 0) base = mine[id[u]];
            __syncwarp();
            if (id[u] >= 0 && rank == 0) mine[id[u]] = base + __popc(same);
            __syncwarp();
            if (i < last) {
                if (id[u] >= 0) rows[base + rank] = (int32_t)((unsigned)i / per);
                place[i] = id[u] >= 0 ? base + rank : -1;
            }
        }
    }
    if (cluster) {  // no block leaves while another may still read its totals
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    }
}

}  // namespace

int64_t launch_expert_plan(DeviceCtx* ctx, const int32_t* ids, int32_t* offsets, int32_t* rows, int32_t* place,
                           int64_t count, int64_t experts, int64_t per) {
    // As many warps as the histograms leave room for (at least four: 4096 experts take 64 KiB), and no more
    // than there are groups of 32 ids; blocks once every warp of one would have more than a few groups.
    int warps = 32;
    while (warps > 4 && (size_t)warps * experts * 4 > (size_t)128 << 10) warps >>= 1;
    const int64_t groups = (count + 31) / 32;
    while (warps > 4 && warps / 2 >= groups) warps >>= 1;
    // blocks of the two-launch form: as many as keep the table of totals, which every block reads, small
    int64_t wide = 80000 / experts;
    if (wide > ctx->sm_count) wide = ctx->sm_count;
    const bool two = count > 16384 && wide > 2 * MAX_CLUSTER;
    int blocks = 1;
    while (!two && blocks < MAX_CLUSTER && groups > (int64_t)4 * warps * blocks) blocks *= 2;
    int32_t* totals = nullptr;
    if (two) {
        warps = warps < 16 ? warps : 16;
        blocks = (int)(wide < groups / warps ? wide : groups / warps);
        MB200_TRY(arena_reserve(ctx, ctx->scratch, (size_t)blocks * experts * 4 + 2048));
        totals = static_cast<int32_t*>(arena_take(ctx->scratch, (size_t)blocks * experts * 4));
    }
    const size_t smem = (size_t)(warps + 1) * experts * 4;
    static thread_local int done_for = -1;
    if (done_for != ctx->device) {
        MB200_CUDA(cudaFuncSetAttribute(expert_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 << 10));
        done_for = ctx->device;
    }
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)blocks, 1, 1);
    lc.blockDim = dim3((unsigned)warps * 32, 1, 1);
    lc.dynamicSmemBytes = smem;
    lc.stream = ctx->stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)blocks;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    lc.attrs = at;
    lc.numAttrs = !two && blocks > 1 ? 2 : 1;
    const unsigned div = (unsigned)(per < 0x7fffffff ? per : 0x7fffffff);
    prof_begin(ctx);
    if (two) {
        MB200_CUDA(cudaLaunchKernelEx(&lc, expert_plan_kernel, ids, offsets, rows, place, count, (int)experts, div, blocks, 1, totals));
        count_launch();
    }
    MB200_CUDA(cudaLaunchKernelEx(&lc, expert_plan_kernel, ids, offsets, rows, place, count, (int)experts, div, blocks, two ? 2 : 0, totals));
    prof_end(ctx);
    count_launch();
    return check_launch("expert_plan_kernel");
}

}  // namespace mb200
