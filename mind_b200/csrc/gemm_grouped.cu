// int8 products grouped by expert: rows [offsets[e], offsets[e+1]) of C belong to expert e,
//
//   acc    = (i32) sum_k A[row(p), k] * B[e][k, n]          row(p) = rows[p], or p without `rows`
//   C[p,n] = acc,  or  (i32)( (acc * scale[e, n]) >> shift )
//
// B is experts x K x N (N contiguous) or, transposed, experts x N x K.
//
// gemm_grouped_tc_kernel, the default, is a persistent warp-specialised tcgen05 kernel:
//   warp 0     : TMA producer - tiles of A and of the expert's B into a ring of shared-memory stages of
//                128 of K;
//   warp 1     : one thread issues tcgen05.mma kind::i8 into two TMEM accumulators in turn;
//   warps 2..5 : drain an accumulator (each warp 32 rows), scale, store.
// The groups' bounds are read on the device: every CTA turns the offsets into a table of tiles per
// expert, and tile i of that list goes to CTA i mod grid.  A tile never spans two experts, so its
// last rows may belong to the next one: they are multiplied and not stored.
//
// What bounds it.  Few rows an expert: the weights (64 experts, 128 gathered rows, 2048 x 2816: 47 to 53 us a
// call; about 41 experts get a row, whose 241 MB would take 37 us: ncu shows no byte read twice, at 4.3 TB/s in
// the product itself).  Many: the tensor pipe under the power cap (32768 x 4096 x
// 4096 over 16 experts: 390 us = 2.82 POP/s in a burst, the dense kernel's rate at that size; 516 us back to
// back with rows gathered, of which their copy is 45).  Between: whole waves of tiles.
#include "common.h"
#include "ptx.cuh"

namespace mb200 {
using namespace ptx;
namespace {

__device__ __forceinline__ int32_t finish(int32_t acc, const int32_t* scale, int64_t i, int shift) {
    return scale ? (int32_t)(((int64_t)acc * scale[i]) >> shift) : acc;
}

// 32 x 32 outputs per block, one block column per 32 rows of C; the cross-check kernel, any size
// and alignment.  A block's rows may belong to several experts: it takes them one expert at a time.
__global__ void __launch_bounds__(256)
gemm_grouped_simt_kernel(const GroupedArgs g) {
    __shared__ int8_t as[32][33], bs[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;  // column, rows ty, ty + 8, ...
    const int64_t n_tiles = (g.n + 31) / 32, m_tiles = (g.m + 31) / 32;
    for (int64_t tile = blockIdx.x; tile < n_tiles * m_tiles; tile += gridDim.x) {
        const int64_t p0 = tile / n_tiles * 32, n0 = tile % n_tiles * 32;
        int64_t lo = min((int64_t)max(g.offsets[0], 0), g.m);
        for (int64_t e = 0; e < g.experts; ++e) {
            const int64_t hi = min(max((int64_t)g.offsets[e + 1], lo), g.m);
            const int64_t first = max(p0, lo), last = min(p0 + 32, hi);
            lo = hi;
            if (first >= last) continue;
            uint32_t acc[4] = {0, 0, 0, 0};
            const int8_t* b = g.b + e * g.k * g.n;
            for (int64_t k0 = 0; k0 < g.k; k0 += 32) {
                __syncthreads();
                for (int j = ty; j < 32; j += 8) {
                    const int64_t p = p0 + j, k = k0 + tx;
                    int8_t v = 0;
                    if (p >= first && p < last && k < g.k) {
                        const int64_t r = g.rows ? g.rows[p] : p;
                        if (r >= 0 && r < g.a_rows) v = g.a[r * g.k + k];
                    }
                    as[j][tx] = v;
                    if (g.bt) {
                        const int64_t n = n0 + j;
                        bs[tx][j] = (n < g.n && k < g.k) ? b[n * g.k + k] : (int8_t)0;
                    } else {
                        const int64_t kk = k0 + j, n = n0 + tx;
                        bs[j][tx] = (n < g.n && kk < g.k) ? b[kk * g.n + n] : (int8_t)0;
                    }
                }
                __syncthreads();
                for (int k = 0; k < 32; ++k)
                    for (int j = 0; j < 4; ++j) acc[j] += (uint32_t)((int32_t)as[ty + 8 * j][k] * bs[k][tx]);
            }
            for (int j = 0; j < 4; ++j) {
                const int64_t p = p0 + ty + 8 * j, n = n0 + tx;
                if (p >= first && p < last && n < g.n) g.c[p * g.n + n] = finish((int32_t)acc[j], g.scale, e * g.n + n, g.shift);
            }
        }
    }
}

// ------------------------------------------------------------------ rows made ready
// dst[i][0 .. pitch) = src[idx ? idx[i] : i][0 .. cols), zeros behind; a row outside [0, src_rows) is
// zeros.  A warp takes a row, a lane 16 bytes at a time; a source that is not 16-byte aligned is read
// as the aligned words around the bytes (only words that lie wholly inside src) and shifted together.
// Bound by memory: cols read, pitch written.  One launch may copy two matrices: the first `first_blocks`
// blocks one, the others the other.
__global__ void __launch_bounds__(256)
copy_rows_kernel(const CopyJob job0, const CopyJob job1, int first_blocks) {
    // Everything before this kernel is complete here, and the product behind it may start only now:
    // it relies on that for all that this kernel does not write.
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31;
    const bool second = (int)blockIdx.x >= first_blocks;
    const CopyJob job = second ? job1 : job0;
    const int block = (int)blockIdx.x - (second ? first_blocks : 0), blocks = second ? (int)gridDim.x - first_blocks : first_blocks;
    const int64_t warp = (block * (int64_t)blockDim.x + threadIdx.x) >> 5;
    const int64_t nwarps = ((int64_t)blocks * blockDim.x) >> 5;
    const int8_t* const src = job.src;
    const int32_t* const idx = job.idx;
    const int64_t rows = job.rows, cols = job.cols, pitch = job.pitch, src_rows = job.src_rows;
    const int8_t* const end = src + src_rows * cols;
    for (int64_t i = warp; i < rows; i += nwarps) {
        const int64_t r = idx ? idx[i] : i;
        const bool inside = r >= 0 && r < src_rows;
        const int8_t* const row = src + (inside ? r : 0) * cols;
        int8_t* const to = job.dst + i * pitch;
        const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15);
#pragma unroll 4
        for (int64_t c = lane * 16; c < pitch; c += 512) {
            uint4 v = make_uint4(0, 0, 0, 0);
            const int64_t left = cols - c;  // bytes of the row from here on
            if (inside && left >= 16 && off == 0) {
                v = __ldg(reinterpret_cast<const uint4*>(row + c));
            } else if (inside && left > 0) {
                const int by = off & 3;
                const uint32_t* w = reinterpret_cast<const uint32_t*>(row + c - by);  // 4-byte aligned, by bytes early
                uint32_t x[5];
#pragma unroll
                for (int j = 0; j < 5; ++j) {
                    const int8_t* at = reinterpret_cast<const int8_t*>(w + j);
                    const int64_t first = 4 * j - by;  // its first byte, counted from c
                    x[j] = 0;
                    if (first >= left || first >= 16) continue;
                    if (at >= src && at + 4 <= end) {
                        x[j] = __ldg(w + j);
                    } else {
                        for (int b = 0; b < 4; ++b)
                            if (at + b >= src && at + b < end) x[j] |= (uint32_t)(uint8_t)at[b] << (8 * b);
                    }
                }
                uint32_t y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    y[j] = __funnelshift_r(x[j], x[j + 1], 8 * by);
                    const int64_t keep = left - 4 * j;  // bytes of this word that belong to the row
                    if (keep < 4) y[j] = keep <= 0 ? 0u : y[j] & ((1u << (8 * keep)) - 1u);
                }
                v = make_uint4(y[0], y[1], y[2], y[3]);
            }
            *reinterpret_cast<uint4*>(to + c) = v;
        }
    }
}

}  // namespace

int64_t launch_copy_rows(DeviceCtx* ctx, const CopyJob& a, const CopyJob* b) {
    const int64_t most = (int64_t)ctx->sm_count * 8;
    auto blocks_of = [](const CopyJob& j) { return (j.rows + 7) / 8; };
    int64_t na = blocks_of(a), nb = b ? blocks_of(*b) : 0;
    if (na + nb > most) {  // shared out by the bytes
        const double wa = (double)a.rows * a.pitch, wb = b ? (double)b->rows * b->pitch : 0.0;
        if (b) {
            nb = (int64_t)(most * (wb / (wa + wb)));
            nb = nb < 1 ? 1 : (nb > most - 1 ? most - 1 : nb);
        }
        na = most - nb;
    }
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)(na + nb), 1, 1);
    lc.blockDim = dim3(256, 1, 1);
    lc.stream = ctx->stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at;
    lc.numAttrs = 1;
    MB200_CUDA(cudaLaunchKernelEx(&lc, copy_rows_kernel, a, b ? *b : a, (int)na));
    count_launch();
    return check_launch("copy_rows_kernel");
}

namespace {
// ------------------------------------------------------------------ tensor cores
constexpr int BLOCK_K = 128;  // bytes of K per stage
constexpr int UMMA_K = 32;
constexpr int GT_THREADS = 192;
constexpr int PATCH_BYTES = 32 * 32 * 4;  // one 32 x 32 block of outputs
constexpr int SMEM_MAX = 232448;
constexpr int BAR_BYTES = 1024;

struct GtParams {
    const int32_t* offsets;
    const int32_t* scale;
    int32_t* c;
    int m, k, n, experts;
    int early;             // the kernel before this one is a copy_rows_kernel that makes A, and B is the caller's
    int n_tiles, stages, patches;  // ring depth and patches per epilogue warp: what the expert table leaves room for
    int group_m, hint_a, hint_b;
    int shift;
    int tma_store;
    int* err;
};

__device__ __forceinline__ int tiles_of(int rows, int tile) { return rows / tile + (rows % tile != 0); }

// Tile of the list: expert, its tile row and the tile column.  Items of one thread only grow, so
// the expert is found by moving on from the last one.
struct Tile {
    int e = 0, tm = 0, tn = 0;
    __device__ __forceinline__ void locate(int item, const int* cum, int n_tiles, int group_m) {
        while (item >= cum[e + 1] * n_tiles) ++e;
        const int m_tiles = cum[e + 1] - cum[e];
        const int local = item - cum[e] * n_tiles;
        // groups of group_m tile rows walked together, odd groups backwards (the order of the dense kernel)
        const int per_group = group_m * n_tiles, g = local / per_group, r = local - g * per_group;
        const int gm0 = g * group_m, gsize = min(group_m, m_tiles - gm0);
        tm = gm0 + r % gsize;
        tn = r / gsize;
        if (g & 1) tn = n_tiles - 1 - tn;
    }
};

// A_ROWS rows of A per CTA and tile.  The MMA always takes 128: with A_ROWS = 32 it reads on into the
// B tile behind them, and what it makes of that lands in accumulator rows that nobody stores.
template <int A_ROWS, int BLOCK_N, int PAIR, bool BMN>
__global__ void __launch_bounds__(GT_THREADS, 1)
gemm_grouped_tc_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                       const __grid_constant__ CUtensorMap tm_c, const GtParams p) {
    static_assert(PAIR == 1 || A_ROWS == 128, "a pair of CTAs multiplies 2 x 128 rows");
    constexpr int TILE_M = A_ROWS * PAIR;
    constexpr int B_ROWS = BLOCK_N / PAIR;  // columns of C this CTA stages
    constexpr int A_BYTES = A_ROWS * BLOCK_K, B_BYTES = B_ROWS * BLOCK_K, STAGE_BYTES = A_BYTES + B_BYTES;
    static_assert(A_BYTES + B_BYTES >= 128 * BLOCK_K, "the MMA's 128 rows of A stay inside the stage");
    constexpr int ACC_STAGES = 2, TMEM_COLS = ACC_STAGES * BLOCK_N;
    static_assert(TMEM_COLS == 512 || TMEM_COLS == 256, "TMEM is allocated in powers of two");
    constexpr int UMMA_M = 128 * PAIR;
    constexpr int EPI_WARPS = 4;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t tiles0 = (raw + 1023u) & ~1023u;
    const uint32_t patches0 = tiles0 + p.stages * STAGE_BYTES;
    const uint32_t bars = patches0 + EPI_WARPS * p.patches * PATCH_BYTES;
    const uint32_t full0 = bars, empty0 = bars + 128;                 // up to 16 stages
    const uint32_t tfull0 = bars + 256, tempty0 = bars + 288;
    int* const misc = reinterpret_cast<int*>(smem_raw + (bars + 320 - raw));  // TMEM address, abort flag
    int* const warp_max = misc + 4;                                   // scratch of the table's scans
    int* const warp_sum = misc + 16;
    int* const bound = reinterpret_cast<int*>(smem_raw + (bars + BAR_BYTES - raw));  // [experts + 1] first row of each
    int* const cum = bound + p.experts + 1;                                          // [experts + 1] tile rows before each
    volatile int* const abort_s = misc + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t cta = PAIR == 2 ? cluster_ctarank() : 0u;
    const bool leader = cta == 0;

    griddep_launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int s = 0; s < ACC_STAGES; ++s) {
            mbar_init(tfull0 + 8 * s, 1);
            mbar_init(tempty0 + 8 * s, EPI_WARPS * PAIR);
        }
        misc[1] = 0;
        fence_mbar_init();
        prefetch_tensormap(&tm_a);
        prefetch_tensormap(&tm_b);
    }
    if (warp == 1) {
        tmem_alloc<PAIR>(smem_u32(misc), TMEM_COLS);
        tmem_relinquish<PAIR>();
    }
    // From here on global memory is read, so the kernel before this one must be done.  Unless that one
    // is the copy of A's rows (p.early), which lets this one start only when all before it are done:
    // then nothing but A has to be waited for, and the first tiles of B are fetched beside the copy.
    if (!p.early) griddep_wait();
    // ---- the table of tiles: bound = running maximum of the offsets within [0, m], cum = running
    // sum of ceil(rows / TILE_M).  Every thread owns a run of experts.
    {
        const int per = (p.experts + GT_THREADS - 1) / GT_THREADS;
        const int e0 = min((int)threadIdx.x * per, p.experts), e1 = min(e0 + per, p.experts);
        int mx = min(max(__ldcg(p.offsets), 0), p.m);  // (from L2: this kernel may start before the copy's end)
        const int first = mx;
        for (int e = e0; e < e1; ++e) {
            const int at = min(__ldcg(p.offsets + e + 1), p.m);
            bound[e + 1] = at;
            mx = max(mx, at);
        }
        int incl = mx;
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl = max(incl, v);
        }
        if (lane == 31) warp_max[warp] = incl;
        int before = __shfl_up_sync(0xffffffffu, incl, 1);
        if (lane == 0) before = first;
        __syncthreads();
        for (int w = 0; w < warp; ++w) before = max(before, warp_max[w]);
        int tiles = 0, lo = before;
        for (int e = e0; e < e1; ++e) {
            const int hi = max(lo, bound[e + 1]);
            bound[e + 1] = hi;
            tiles += tiles_of(hi - lo, TILE_M);
            lo = hi;
        }
        int sum = tiles;
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        if (lane == 31) warp_sum[warp] = sum;
        __syncthreads();
        int at = sum - tiles;
        for (int w = 0; w < warp; ++w) at += warp_sum[w];
        lo = before;
        for (int e = e0; e < e1; ++e) {
            const int hi = bound[e + 1];
            at += tiles_of(hi - lo, TILE_M);
            cum[e + 1] = at;
            lo = hi;
        }
        if (threadIdx.x == 0) {
            bound[0] = first;
            cum[0] = 0;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR == 2) {
        cluster_arrive();
        cluster_wait();
    }
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(misc);

    const int total = cum[p.experts] * p.n_tiles;
    const int k_blocks = (p.k + BLOCK_K - 1) / BLOCK_K;
    const int step = gridDim.x / PAIR, first_item = blockIdx.x / PAIR;
    const int stages = p.stages;

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer
        if (lane == 0) {
            const uint64_t pol_a = l2_policy(p.hint_a), pol_b = l2_policy(p.hint_b);
            Tile t;
            int row0 = 0, col0 = 0;
            auto start = [&](int item) {
                t.locate(item, cum, p.n_tiles, p.group_m);
                row0 = bound[t.e] + t.tm * TILE_M + (int)cta * A_ROWS;
                col0 = t.tn * BLOCK_N + (int)cta * B_ROWS;
            };
            // with a pair, both CTAs' copies complete on the leader's barrier, which alone expects them
            auto full = [&](uint32_t s) { return PAIR == 2 ? mapa(full0 + 8 * s, 0) : full0 + 8 * s; };
            auto load_b = [&](uint32_t s, int kx) {
                const uint32_t db = tiles0 + s * STAGE_BYTES + A_BYTES, bar = full(s);
                if (leader) mbar_arrive_expect_tx(full0 + 8 * s, PAIR * STAGE_BYTES);
#pragma unroll
                for (int j = 0; j < (BMN ? B_ROWS / 128 : 1); ++j) {
                    const int x = BMN ? col0 + 128 * j : kx, y = BMN ? kx : col0;
                    if (PAIR == 2) tma_load_3d_pair(db + j * 128 * BLOCK_K, &tm_b, bar, x, y, t.e, pol_b);
                    else tma_load_3d(db + j * 128 * BLOCK_K, &tm_b, bar, x, y, t.e, pol_b);
                }
            };
            auto load_a = [&](uint32_t s, int kx) {
                if (PAIR == 2) tma_load_2d_pair(tiles0 + s * STAGE_BYTES, &tm_a, full(s), kx, row0, pol_a);
                else tma_load_2d(tiles0 + s * STAGE_BYTES, &tm_a, full(s), kx, row0, pol_a);
            };
            int early = 0;  // stages whose B was asked for before the rows of A were ready
            if (p.early) {
                if (first_item < total) {
                    start(first_item);
                    for (; early < stages && early < k_blocks; ++early) load_b(early, early * BLOCK_K);
                }
                griddep_wait();
            }
            uint32_t s = 0, ph = 1;
            bool ok = true;
            for (int item = first_item; ok && item < total; item += step) {
                start(item);
                for (int kb = 0; kb < k_blocks; ++kb) {
                    if (!wait_bounded(empty0 + 8 * s, ph, abort_s, p.err, 1)) {
                        ok = false;
                        break;
                    }
                    if (early > 0) --early;
                    else load_b(s, kb * BLOCK_K);
                    load_a(s, kb * BLOCK_K);
                    if (++s == (uint32_t)stages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
        }
    } else if (warp == 1) {
        // -------------------------------------------------------------- MMA issuer
        if (lane == 0 && leader) {
            constexpr uint32_t ID = idesc_i8(UMMA_M, BLOCK_N, true, true, BMN);
            constexpr uint64_t B_KSTEP = BMN ? (UMMA_K * 128) >> 4 : UMMA_K >> 4;
            uint32_t s = 0, ph = 0, tcount = 0;
            bool ok = true;
            for (int item = first_item; ok && item < total; item += step, ++tcount) {
                const uint32_t as = tcount % ACC_STAGES, aph = (tcount / ACC_STAGES) & 1u;
                if (!wait_bounded(tempty0 + 8 * as, aph ^ 1u, abort_s, p.err, 2)) break;
                tc_fence_after();
                const uint32_t d = tmem_base + as * BLOCK_N;
                for (int kb = 0; kb < k_blocks; ++kb) {
                    if (!wait_bounded(full0 + 8 * s, ph, abort_s, p.err, 3)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sa = tiles0 + s * STAGE_BYTES, sb = sa + A_BYTES;
                    const uint64_t da = smem_desc_k_sw128(sa);
                    const uint64_t db = BMN ? smem_desc_mn_sw128(sb, 128 * BLOCK_K) : smem_desc_k_sw128(sb);
#pragma unroll
                    for (int ks = 0; ks < BLOCK_K / UMMA_K; ++ks)
                        mma_i8<PAIR>(d, da + (uint64_t)((ks * UMMA_K) >> 4), db + (uint64_t)ks * B_KSTEP, ID,
                                     (kb | ks) ? 1u : 0u);
                    if (PAIR == 1) mma_commit(empty0 + 8 * s);
                    else mma_commit_pair(empty0 + 8 * s, 3);
                    if (++s == (uint32_t)stages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
                if (!ok) break;
                if (PAIR == 1) mma_commit(tfull0 + 8 * as);
                else mma_commit_pair(tfull0 + 8 * as, 3);
            }
        }
    } else {
        // ---------------------------------------------------------------- epilogue
        const int q = warp & 3;  // TMEM lane quadrant this warp may read
        const uint32_t patch_first = patches0 + (uint32_t)(warp - 2) * p.patches * PATCH_BYTES;
        uint32_t* const patch = reinterpret_cast<uint32_t*>(smem_raw + (patch_first - raw));
        uint32_t stored = 0, tcount = 0;
        Tile t;
        for (int item = first_item; item < total; item += step, ++tcount) {
            t.locate(item, cum, p.n_tiles, p.group_m);
            const uint32_t as = tcount % ACC_STAGES, aph = (tcount / ACC_STAGES) & 1u;
            const int row_first = bound[t.e] + t.tm * TILE_M + (int)cta * A_ROWS + q * 32;
            const int valid = q * 32 < A_ROWS ? bound[t.e + 1] - row_first : 0;  // rows of this expert in the block
            const int col_tile = t.tn * BLOCK_N;
            const uint32_t t0 = tmem_base + ((uint32_t)(q * 32) << 16) + as * BLOCK_N;
            const int32_t* const scale = p.scale ? p.scale + (size_t)t.e * p.n : nullptr;
            int f_next = scale && col_tile + lane < p.n ? __ldg(scale + col_tile + lane) : 0;
            // (all lanes give up together: what follows is done by whole warps)
            if (!__all_sync(0xffffffffu, wait_bounded(tfull0 + 8 * as, aph, abort_s, p.err, 4))) break;
            tc_fence_after();
            for (int c0 = 0; c0 < BLOCK_N && valid > 0; c0 += 32) {
                const int col = col_tile + c0;
                if (col >= p.n) break;
                uint32_t v[32];
                tmem_ld32(t0 + c0, v);
                tmem_ld_wait();
                if (scale) {
                    // lane j holds the scale of column j; the next block's is fetched before it is needed
                    const int f = f_next;
                    f_next = col + 32 + lane < p.n ? __ldg(scale + col + 32 + lane) : 0;
                    if (p.shift < 32) {  // the low 32 bits of the shifted 64-bit product: a funnel shift
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const int64_t prod = (int64_t)(int32_t)v[j] * __shfl_sync(0xffffffffu, f, j);
                            v[j] = __funnelshift_r((uint32_t)prod, (uint32_t)((uint64_t)prod >> 32), p.shift);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            v[j] = (uint32_t)(__mulhi((int32_t)v[j], __shfl_sync(0xffffffffu, f, j)) >> (p.shift - 32));
                    }
                }
                if (valid >= 32 && p.tma_store) {
                    // 32 rows of 128 bytes in the 128-byte swizzle, written out by one tensor store
                    // (columns past the matrix are clipped by the hardware)
                    if (lane == 0) {
                        if (p.patches == 2) bulk_wait_group_read<1>();
                        else bulk_wait_group_read<0>();
                    }
                    __syncwarp();
                    const uint32_t patch_addr = patch_first + (p.patches == 2 ? (stored & 1u) * PATCH_BYTES : 0u);
                    ++stored;
                    const uint32_t prow = patch_addr + (uint32_t)lane * 128u;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        st_shared_v4(prow + (uint32_t)((j ^ (lane & 7)) << 4), v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tm_c, patch_addr, col, row_first);
                        bulk_commit_group();
                    }
                    continue;
                }
                // A block that ends inside (the rows below it are the next expert's), or a C the tensor
                // stores cannot address: transposed through the patch, one 128-byte line per store.
                if (lane == 0) bulk_wait_group_read<0>();
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 32; ++j) patch[lane * 32 + (j ^ lane)] = v[j];
                __syncwarp();
                if (col + lane < p.n) {
                    int32_t* dst = p.c + (size_t)row_first * (size_t)p.n + col + lane;
                    const int rows = min(valid, 32);
#pragma unroll 4
                    for (int r = 0; r < rows; ++r) {
                        *dst = (int32_t)patch[r * 32 + (lane ^ r)];
                        dst += p.n;
                    }
                }
                __syncwarp();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR == 1) mbar_arrive(tempty0 + 8 * as);
                else mbar_arrive_cluster(tempty0 + 8 * as, 0);
            }
        }
        if (lane == 0) bulk_wait_group<0>();
    }

    // ------------------------------------------------------------------ teardown
    __syncwarp();
    if (*abort_s) __nanosleep(200000);  // let copies / MMAs still in flight land before freeing
    tc_fence_before();
    __syncthreads();
    if (PAIR == 2) {
        cluster_arrive();
        cluster_wait();
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<PAIR>(tmem_base, TMEM_COLS);
    }
}

}  // namespace

// Map over a stack of `experts` row-major 8-bit matrices [rows][cols] of row pitch `pitch`: boxes of
// 128 columns by box_rows rows in the 128-byte swizzle.  Reads past cols or rows return zeros.
int64_t make_tmap_stack(CUtensorMap* tm, const void* base, int64_t cols, int64_t rows, int64_t experts, int64_t pitch,
                        int box_rows) {
    struct Key {
        const void* base;
        int64_t cols, rows, experts, pitch;
        int box_rows;
        bool operator==(const Key& o) const {
            return base == o.base && cols == o.cols && rows == o.rows && experts == o.experts && pitch == o.pitch &&
                   box_rows == o.box_rows;
        }
    };
    constexpr int N = 8;  // a map is a pure function of these arguments: the last few are kept per thread
    static thread_local struct {
        Key key[N];
        CUtensorMap map[N];
        int used = 0, next = 0;
    } cache;
    const Key want{base, cols, rows, experts, pitch, box_rows};
    for (int i = 0; i < cache.used; ++i)
        if (cache.key[i] == want) {
            *tm = cache.map[i];
            return 0;
        }
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return fail(MIND_B200_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)experts};
    cuuint64_t strides[2] = {(cuuint64_t)pitch, (cuuint64_t)pitch * (cuuint64_t)rows};
    cuuint32_t box[3] = {BLOCK_K, (cuuint32_t)box_rows, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(MIND_B200_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d (%lld x %lld x %lld, pitch %lld)", (int)r,
                    (long long)experts, (long long)rows, (long long)cols, (long long)pitch);
    cache.key[cache.next] = want;
    cache.map[cache.next] = *tm;
    cache.next = (cache.next + 1) % N;
    if (cache.used < N) ++cache.used;
    return 0;
}

namespace {

// a: pitch pa, b: pitch pb (both 16-byte multiples on 16-byte bases).
template <int A_ROWS, int BLOCK_N, int PAIR, bool BMN>
int64_t launch_grouped_tc(DeviceCtx* ctx, const GroupedArgs& g, const int8_t* a, int64_t pa, const int8_t* b, int64_t pb,
                          bool early) {
    constexpr int B_ROWS = BLOCK_N / PAIR;
    constexpr int STAGE_BYTES = (A_ROWS + B_ROWS) * BLOCK_K;
    CUtensorMap ta, tb, tc;
    MB200_TRY(make_tmap_u8(&ta, a, g.k, g.m, pa, A_ROWS, BLOCK_K));
    if (BMN) MB200_TRY(make_tmap_stack(&tb, b, g.n, g.k, g.experts, pb, BLOCK_K));
    else MB200_TRY(make_tmap_stack(&tb, b, g.k, g.n, g.experts, pb, B_ROWS));
    GtParams p;
    p.tma_store = g.n % 4 == 0 && reinterpret_cast<uintptr_t>(g.c) % 16 == 0 ? 1 : 0;
    tc = ta;
    if (p.tma_store) MB200_TRY(make_tmap_c32(&tc, g.c, g.n, g.m));
    p.offsets = g.offsets;
    p.scale = g.scale;
    p.c = g.c;
    p.m = (int)g.m;
    p.k = (int)g.k;
    p.n = (int)g.n;
    p.experts = (int)g.experts;
    p.early = early ? 1 : 0;
    p.n_tiles = (int)((g.n + BLOCK_N - 1) / BLOCK_N);
    p.group_m = 8;
    p.hint_a = 1;
    p.hint_b = 0;
    p.shift = g.shift;
    p.err = ctx->err_word;
    const int64_t most = (g.m / (A_ROWS * PAIR) + g.experts) * p.n_tiles;  // tiles, however the rows are spread
    if (most > 0x7fffffff - 4096) return fail(MIND_B200_ERR_TOO_LARGE, "too many output tiles");
    // Shared memory: the table of tiles, two patches per epilogue warp if that still leaves four stages, stages
    const int table = (int)align_up((size_t)(g.experts + 1) * 8, 16);
    const int room = SMEM_MAX - 1024 - BAR_BYTES - table;
    p.patches = (room - 8 * PATCH_BYTES) / STAGE_BYTES >= (PAIR == 2 ? 6 : 4) ? 2 : 1;
    p.stages = (room - 4 * p.patches * PATCH_BYTES) / STAGE_BYTES;
    if (p.stages > 16) p.stages = 16;
    const int smem = 1024 + p.stages * STAGE_BYTES + 4 * p.patches * PATCH_BYTES + BAR_BYTES + table;
    auto kern = gemm_grouped_tc_kernel<A_ROWS, BLOCK_N, PAIR, BMN>;
    static thread_local int done_for = -1;
    if (done_for != ctx->device) {
        MB200_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX));
        done_for = ctx->device;
    }
    int64_t units = ctx->sm_count / PAIR;
    if (most < units) units = most;
    cudaLaunchConfig_t lc = {};
    lc.blockDim = dim3(GT_THREADS, 1, 1);
    lc.dynamicSmemBytes = smem;
    lc.stream = ctx->stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    lc.numAttrs = 1;
    if (PAIR == 2) {
        at[1].id = cudaLaunchAttributeClusterDimension;
        at[1].val.clusterDim.x = PAIR;
        at[1].val.clusterDim.y = 1;
        at[1].val.clusterDim.z = 1;
        lc.numAttrs = 2;
    }
    lc.attrs = at;
    if (PAIR == 2) {  // the pairs that are resident at once (not every SM need be pairable)
        static thread_local int fit_dev = -1, fit = 0;
        if (fit_dev != ctx->device) {
            lc.gridDim = dim3((unsigned)(ctx->sm_count / PAIR * PAIR), 1, 1);
            lc.dynamicSmemBytes = SMEM_MAX;
            if (cudaOccupancyMaxActiveClusters(&fit, kern, &lc) != cudaSuccess) {
                cudaGetLastError();
                fit = 0;
            }
            fit_dev = ctx->device;
            lc.dynamicSmemBytes = smem;
        }
        if (fit > 0 && fit < units) units = fit;
    }
    lc.gridDim = dim3((unsigned)(units * PAIR), 1, 1);
    prof_begin(ctx);
    MB200_CUDA(cudaLaunchKernelEx(&lc, kern, ta, tb, tc, p));
    prof_end(ctx);
    count_launch();
    return check_launch("gemm_grouped_tc_kernel");
}

template <bool BMN>
int64_t launch_grouped_any(DeviceCtx* ctx, const GroupedArgs& g, const int8_t* a, int64_t pa, const int8_t* b, int64_t pb,
                           bool early) {
    // (a kernel may be asked for by name: mind_b200_set_gemm_path 10 / 5 / 3 / 2)
    const int pair = tuning().pair_mode.load(), small = tuning().small_tile.load();
    if (small == 1) return launch_grouped_tc<32, 128, 1, BMN>(ctx, g, a, pa, b, pb, early);
    if (pair == 2) return launch_grouped_tc<128, 256, 2, BMN>(ctx, g, a, pa, b, pb, early);
    if (pair == 1 && tuning().force_transpose.load()) return launch_grouped_tc<128, 128, 1, BMN>(ctx, g, a, pa, b, pb, early);
    if (pair == 1) return launch_grouped_tc<128, 256, 1, BMN>(ctx, g, a, pa, b, pb, early);
    // The host knows the rows and the experts, not how the rows are spread: tiles are counted as if every
    // expert had the average, half of its last tile empty.
    const double m = (double)g.m, half = g.experts / 2.0, n256 = (double)((g.n + 255) / 256);
    const double avg = m / g.experts;
    const double single_tiles = (m / 128 + half) * n256, pair_tiles = (m / 256 + half) * n256;
    // 32-row tiles where the weights are most of the traffic (2048 x 2816, 64 experts: 58.5 us against 58.2 of
    // 128-row tiles at 8 rows an expert, 70 against 63 at 16; with fewer rows they are ahead).
    if (avg <= 8) return launch_grouped_tc<32, 128, 1, BMN>(ctx, g, a, pa, b, pb, early);
    // 128 x 128 tiles while they fit one wave: twice the CTAs, half the epilogue (4096 x 1024, 8 experts, 512
    // rows: 16.6 us against 21.0 of 128 x 256; in more than a wave, 4096 x 2048, 1024 rows: 26.6 against 23.7).
    if ((m / 128 + half) * (double)((g.n + 127) / 128) <= ctx->sm_count)
        return launch_grouped_tc<128, 128, 1, BMN>(ctx, g, a, pa, b, pb, early);
    // Pairs of CTAs move a third less per product (32768 x 4096 x 4096: 390 us against 443), unless their
    // coarser tiles cost a wave (4096 x 4096 x 2048, 8 experts: 42 us in three waves against 38 in two).
    const double single_waves = single_tiles / ctx->sm_count, pair_waves = pair_tiles / (ctx->sm_count / 2);
    const auto up = [](double w) { return w < 8 ? (double)(int64_t)(w + 0.999) : w; };
    if (up(pair_waves) <= 1.13 * up(single_waves)) return launch_grouped_tc<128, 256, 2, BMN>(ctx, g, a, pa, b, pb, early);
    return launch_grouped_tc<128, 256, 1, BMN>(ctx, g, a, pa, b, pb, early);
}

}  // namespace

int64_t launch_gemm_grouped_i8(DeviceCtx* ctx, const GroupedArgs& g) {
    if (tuning().gemm_path.load() != 1 && g.k > 0 && g.a_rows > 0) {
        // The rows of A as the tiles take them: one under the other in the order of C, on 16-byte pitches and
        // bases (TMA's rule).  Rows to be gathered, or not aligned, are copied there first; so is an unaligned B.
        const int64_t b_cols = g.bt ? g.k : g.n, b_rows = g.experts * (g.bt ? g.n : g.k);
        const int64_t pa = (int64_t)align_up((size_t)g.k, 16), pb = (int64_t)align_up((size_t)b_cols, 16);
        const bool a_direct = !g.rows && pa == g.k && reinterpret_cast<uintptr_t>(g.a) % 16 == 0;
        const bool b_direct = pb == b_cols && reinterpret_cast<uintptr_t>(g.b) % 16 == 0;
        const int8_t *a = g.a, *b = g.b;
        if (!a_direct || !b_direct) {
            const size_t sa = a_direct ? 0 : (size_t)g.m * pa, sb = b_direct ? 0 : (size_t)b_rows * pb;
            MB200_TRY(arena_reserve(ctx, ctx->scratch, align_up(sa, 1024) + align_up(sb, 1024) + 2048));
            CopyJob ja, jb;
            if (!b_direct) {
                jb = CopyJob{g.b, nullptr, static_cast<int8_t*>(arena_take(ctx->scratch, sb)), b_rows, b_cols, pb, b_rows};
                b = jb.dst;
            }
            if (!a_direct) {
                ja = CopyJob{g.a, g.rows, static_cast<int8_t*>(arena_take(ctx->scratch, sa)), g.m, g.k, pa, g.a_rows};
                a = ja.dst;
            }
            MB200_TRY(launch_copy_rows(ctx, a_direct ? jb : ja, !a_direct && !b_direct ? &jb : nullptr));
        }
        // Where the copy makes A alone, B is complete when it lets the product start.
        const bool early = !a_direct && b_direct;
        return g.bt ? launch_grouped_any<false>(ctx, g, a, pa, b, pb, early)
                    : launch_grouped_any<true>(ctx, g, a, pa, b, pb, early);
    }
    int64_t blocks = ((g.n + 31) / 32) * ((g.m + 31) / 32);
    if (blocks > (int64_t)ctx->sm_count * 32) blocks = (int64_t)ctx->sm_count * 32;
    prof_begin(ctx);
    gemm_grouped_simt_kernel<<<(unsigned)blocks, 256, 0, ctx->stream>>>(g);
    prof_end(ctx);
    count_launch();
    return check_launch("gemm_grouped_simt_kernel");
}

}  // namespace mb200
