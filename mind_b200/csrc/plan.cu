// Grouping of routed tokens by expert: a stable counting sort of small integers.
//
//   offsets[e] = #{ i : 0 <= ids[i] < e }          (e = 0 .. experts)
//   the kept i, in order of (ids[i], i), are p = 0, 1, ...:  rows[p] = i / per,  place[i] = p
//   place[i] = -1 where ids[i] names no expert (padding)
//
// Every warp owns a contiguous piece of the ids and a histogram of its own in shared memory; two passes
// over the ids (count, then place) with a scan of the histograms between them, expert-major and (block,
// warp)-minor, which is what makes the order stable.
// Up to 16384 ids take one launch of one cluster of 1, 2, 4 or 8 blocks, which meet in shared memory: each
// publishes its totals per expert and reads the others' remotely.  More ids take two launches of up to one
// block per SM: the first leaves the blocks' totals in scratch; the second counts again, beside the first,
// adds the totals up and places (32768 ids over 64 experts: 6.3 us against 9.8 on a cluster, whose eight
// SMs are bound by their scattered stores).  Either way no block waits for one that may not be running.
//
// Inside 32 ids the rank of a lane among the lanes of the same expert is a population count of the lanes
// that agree in every bit of the id, a ballot per bit.  (__match_any_sync finds them one value after the
// other: 300126 ids over 160 experts took 12.2 us, 65536 over 256 11.6, with ballots 9.2 and 7.5.)  The only
// atomics are sums of integers in shared memory, so the result does not depend on timing.
// Bound by latency: launch, load, count, meet, scan, load, place, store are one chain (64 ids: 2.8 us a call
// in a graph, where the host does not count; 8192: 5; 16384 over 256: 6.7), from a million ids on by the
// scattered stores of rows (4194304 over 256: 40 us).
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

// Shared memory: hist[warps][experts], then total[experts] and (two launches) prior[experts].
__global__ void __launch_bounds__(1024)
expert_plan_kernel(const int32_t* ids, int32_t* __restrict__ offsets, int32_t* __restrict__ rows,
                   int32_t* __restrict__ place, int64_t count, int experts, unsigned per, int blocks, int phase,
                   int32_t* totals) {  // phase 0: a cluster does it all; 1: count; 2: place
    extern __shared__ int32_t hist[];
    __shared__ int32_t warp_sum[32];
    __shared__ int32_t carry;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int block = blockIdx.x;
    const bool cluster = phase == 0 && blocks > 1;  // the grid is one cluster
    int32_t* const total = hist + warps * experts;
    int32_t* const prior = total + experts;
    // (The second launch says nothing: blocks of the kernel behind it, waiting beside it, moved its own blocks
    // off their SMs - 300126 ids over 160 experts 11.2 us against 9.1; other sizes differ by 0.4 at most.)
    if (phase == 0) griddep_launch_dependents();
    for (int i = threadIdx.x; i < (warps + 2) * experts; i += blockDim.x) hist[i] = 0;
    if (threadIdx.x == 0) carry = 0;
    // The ids may be the work of the kernel before this one.  The first of two launches lets the second
    // start when that is over, so the second may read the ids (and count) beside it.
    if (phase != 2) griddep_wait();
    if (phase == 1) griddep_launch_dependents();
    __syncthreads();
    // this warp's piece, a multiple of 32 ids
    const int64_t groups = (count + 31) / 32, pieces = (int64_t)warps * blocks;
    const int64_t piece = (groups + pieces - 1) / pieces * 32;
    const int64_t first = min((int64_t)(block * warps + warp) * piece, count), last = min(first + piece, count);
    int32_t* const mine = hist + warp * experts;
    const int pitch = (experts + 3) & ~3;  // of the blocks' totals
    constexpr int U = 4;  // groups of 32 ids fetched at a time

    // pass 1: how many ids of each expert this warp's piece holds
    for (int64_t i0 = first; i0 < last; i0 += 32 * U) {
        int32_t id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = i0 + 32 * u + lane;
            id[u] = i < last ? __ldcg(ids + i) : -1;
            if ((unsigned)id[u] >= (unsigned)experts) id[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (id[u] >= 0) atomicAdd(mine + id[u], 1);
        }
    }
    __syncthreads();
    if (phase == 1) {
        for (int e = threadIdx.x; e < experts; e += blockDim.x) {
            totals[block * pitch + e] = column(hist, warps, experts, e);
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
    if (phase == 2) {  // add up the blocks' totals: a thread four experts, of every parts-th block
        griddep_wait();
        const int quads = pitch / 4, parts = max(1, min((int)blockDim.x / quads, blocks));
        for (int i = threadIdx.x; i < quads * parts; i += blockDim.x) {
            const int part = i / quads, e = 4 * (i - part * quads);
            int32_t all[4] = {0, 0, 0, 0}, before_me[4] = {0, 0, 0, 0};
            constexpr int B = 8;
            for (int b0 = part; b0 < blocks; b0 += B * parts) {
                int4 n[B];
#pragma unroll
                for (int j = 0; j < B; ++j) {
                    const int b = b0 + j * parts;
                    n[j] = b < blocks ? __ldcg(reinterpret_cast<const int4*>(totals + b * pitch + e)) : make_int4(0, 0, 0, 0);
                }
#pragma unroll
                for (int j = 0; j < B; ++j) {
                    const int32_t v[4] = {n[j].x, n[j].y, n[j].z, n[j].w};
                    const bool mine_after = b0 + j * parts < block;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        all[q] += v[q];
                        before_me[q] += mine_after ? v[q] : 0;
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (e + q < experts) {
                    atomicAdd(total + e + q, all[q]);
                    atomicAdd(prior + e + q, before_me[q]);
                }
        }
        __syncthreads();
    }

    // exclusive scan over (expert, block, warp), a block of experts at a time; hist becomes first positions
    for (int e0 = 0; e0 < experts; e0 += blockDim.x) {
        const int e = e0 + threadIdx.x;
        int32_t all = 0, before_me = 0;  // of this expert: everywhere, and in the blocks before this one
        if (e < experts) {
            if (phase == 2) {
                all = total[e];
                before_me = prior[e];
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

    const int bits = 32 - __clz(experts);
    // pass 2: every id takes the next position of its expert within its warp's share
    for (int64_t i0 = first; i0 < last; i0 += 32 * U) {
        int32_t id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = i0 + 32 * u + lane;
            id[u] = i < last ? __ldcg(ids + i) : -1;
            if ((unsigned)id[u] >= (unsigned)experts) id[u] = -1;
        }
        // The lanes of a group with the same id: those that agree in every bit.  Ids that name no expert have
        // the bits of `experts`, which no other has.
        unsigned same[U];
#pragma unroll
        for (int u = 0; u < U; ++u) same[u] = 0xffffffffu;
        for (int b = 0; b < bits; ++b)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool set = (id[u] < 0 ? experts : id[u]) >> b & 1;
                const unsigned with = __ballot_sync(0xffffffffu, set);
                same[u] &= set ? with : ~with;
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = i0 + 32 * u + lane;
            const int rank = __popc(same[u] & ((1u << lane) - 1u));
            int32_t base = 0;
            if (id[u] >= 0) base = mine[id[u]];
            __syncwarp();
            if (id[u] >= 0 && rank == 0) mine[id[u]] = base + __popc(same[u]);
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
    // than there are groups of 32 ids.
    int warps = 32;
    while (warps > 4 && (size_t)warps * experts * 4 > (size_t)128 << 10) warps >>= 1;
    const int64_t groups = (count + 31) / 32;
    while (warps > 4 && warps / 2 >= groups) warps >>= 1;
    // Blocks of the two-launch form: what keeps the table of totals, which every block reads, small.
    int64_t wide = 80000 / experts;
    if (wide > ctx->sm_count) wide = ctx->sm_count;
    const bool two = count > 16384;
    int blocks = 1;
    if (!two) {
        // Blocks of eight warps with one group of 32 each while that lasts (8192 ids over 64 experts: 4.8 us, of
        // 16 warps 5.3, of 32 7.0), of 16 once eight would have more than four (16384 over 256: 6.7 against 7.2).
        const int most = groups > 4 * 8 * MAX_CLUSTER ? 16 : 8;
        if (warps > most) warps = most;
        while (blocks < MAX_CLUSTER && groups > (int64_t)warps * blocks) blocks *= 2;
    }
    int32_t* totals = nullptr;
    if (two) {
        // Blocks of 16 warps with four groups each, which are loaded at once (65536 ids over 256 experts: 7.5 us
        // with 32 blocks, 10.5 with 128), or every SM where that takes most of them; 32 warps once 16 would have
        // more than eight groups (2^20 ids over 64 experts: 15.8 us against 19.5, 300126 over 160: 10.7 against 9.2).
        const int most = groups > 8 * 16 * wide ? 32 : 16;
        if (warps > most) warps = most;
        const int64_t want = (groups + 4 * warps - 1) / (4 * warps);
        blocks = (int)(want > wide || (2 * want > wide && wide == ctx->sm_count) ? wide : want);
        MB200_TRY(arena_reserve(ctx, ctx->scratch, (size_t)blocks * align_up((size_t)experts, 4) * 4 + 2048));
        totals = static_cast<int32_t*>(arena_take(ctx->scratch, (size_t)blocks * align_up((size_t)experts, 4) * 4));
    }
    const size_t smem = (size_t)(warps + 2) * experts * 4;
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
