// Matrix-vector products with 4-bit weights and group scales.
//
//   d[t,r,g] = sum_{k in group g} w[r,k] * x[t,k]            w in [-8, 7], x int8 / int16 / Q16.16
//   y[t,r]   = (i32)( ( sum_g scale[r,g] * d[t,r,g] ) >> shift )
//
// The sum over groups is taken mod 2^64 (the low 60 bits decide the output; a model's sums are far smaller:
// |sum| < 2^49 * cols for Q16.16, 2^33 * cols for int16, 2^25 * cols for int8); it is shifted
// once and truncated once, so any order of accumulation gives the same bits.
//
// Weights: two a byte, the even column in the low half, rows of ceil(cols / 2) bytes.
//
// gemv_w4.cuh holds the kernel that runs by default; here are the choice of its shape, the operands
// it cannot address, and the cross-check kernel.
#include "gemv_w4.cuh"

#include <cmath>

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

// What mind_b200_set_w4_shape asks for (0: nothing).
struct Asked {
    int cs, rt, tb;
    bool operator==(const Asked& o) const { return cs == o.cs && rt == o.rt && tb == o.tb; }
    bool any() const { return cs || rt || tb; }
};
Asked asked_shape() {
    const Tuning& t = tuning();
    return Asked{t.w4_cluster.load(), t.w4_row_tiles.load(), t.w4_tokens.load()};
}

// How a call runs on the tensor-core kernel: blocks of at most tb tokens, clusters of cs blocks over the
// columns, rt row tiles to a round.  Every choice gives the same bytes; the one with the least estimated
// time is taken.  The estimate is in clocks of the busiest block; its constants were fitted to 33 cases (1 .. 64
// tokens, 1024 .. 32768 rows, one matrix and 8 .. 128 of them) timed in every shape that fits (as
// mind_b200_set_w4_shape asks for them): the shape taken is 1.2 % slower than the fastest on the geometric mean,
// 9 % at worst (int16, 8 tokens through 4 of 32 experts of 2048 x 4096: 31.0 against 28.5 us).
// fits: clusters of 1, 2, 4 and 8 blocks that the device holds at once.
bool make_plan(const int (&fits)[4], const Asked& asked, const W4Args& a, int tb, int tc, w4::Plan* out) {
    const int L = a.kind == 0 ? 1 : (a.kind == 1 ? 2 : 4);
    const int ac = tc <= 8 ? 8 : tc, tok8 = (tb + 7) / 8;
    const bool pack = L > 1 && L * tc <= 8;
    const int kb_total = (int)((a.cols + w4::KB - 1) / w4::KB);
    const int g32 = (int)(a.group / 32 % 4), gb = g32 == 0 ? 4 : (g32 == 2 ? 2 : 1);
    const size_t table = align_up((size_t)(a.experts + 1) * 8, 128);
    const size_t part = align_up((size_t)w4::WARPS * ac * 17 * 8, 1024);
    // Instructions of a warp per unit, and the clocks of a unit that nothing overlaps
    const double mmas = pack ? 2.0 : (double)L * tok8;                                     // per 32 columns
    const double per32 = 8.0 + mmas + (pack ? 1.0 : mmas) * (gb == 1 ? 1.0 : 0.5) + (pack ? 4.0 : 0.0);
    const double scaling = 8.0 + 4.0 * (pack ? 2.0 : (L == 4 ? 6.0 : L == 2 ? 3.0 : 2.0) * tok8);
    const double unit = 110.0 + 16.0 * per32 + 16.0 / gb * scaling;
    const double fill = 30.0 + 30.0 * L;                                                  // per eight activations
    const int64_t tiles = (a.rows + 15) / 16;
    // Blocks of tokens: of grouped rows the host does not know how they are spread.  Counted as if every expert had
    // the average, half of its last block empty, and as no fewer than the experts that rows drawn by chance meet.
    int64_t blocks = (a.m + tb - 1) / tb;
    if (a.offsets) {
        blocks += (a.experts < a.m ? a.experts : a.m) / 2;
        const int64_t met = (int64_t)((double)a.experts * (1.0 - std::pow(1.0 - 1.0 / (double)a.experts, (double)a.m)) + 0.5);
        if (blocks < met) blocks = met;
    }
    double best = 0;
    for (int cs = 1; cs <= 8; cs *= 2) {
        if (cs > kb_total) break;
        const int fit = fits[cs == 8 ? 3 : cs / 2];
        if (fit < 1 || (asked.cs && asked.cs != cs)) continue;
        const int kb_slice = (kb_total + cs - 1) / cs;
        const size_t x_bytes = (size_t)kb_slice * w4::KB * L * tc;
        for (int rt = 1; rt <= w4::WARPS; ++rt) {
            if (asked.rt && asked.rt != rt) continue;
            const int wpr = w4::WARPS / rt, steps = (kb_slice + wpr - 1) / wpr;
            const int64_t row_rounds = (tiles + rt - 1) / rt, rounds = blocks * row_rounds;
            if (rounds > 0x1fffffff) continue;  // (the kernel counts them, at most twice as many, in 32 bits)
            const int64_t clusters = rounds < fit ? rounds : fit;
            const int64_t most = (rounds + clusters - 1) / clusters;  // rounds of the busiest cluster
            const bool once = most == 1 && !a.offsets;
            const size_t fixed = 1024 + w4::HEAD_BYTES + (once ? 0 : part) + x_bytes + table;
            if (fixed + 2 * w4::RING_BYTES > (size_t)w4::SMEM_MAX) continue;
            int slots = (int)((w4::SMEM_MAX - fixed) / w4::RING_BYTES);
            if (slots > w4::MAX_SLOTS) slots = w4::MAX_SLOTS;
            if (once && (size_t)slots * w4::RING_BYTES < part) continue;
            const double active = (double)clusters * cs;
            const int warps = rt * (wpr < kb_slice ? wpr : kb_slice);
            const double issue = unit * ((warps + 3) / 4) / 0.7, alone = 500.0 + unit * 1.5;
            const double step = issue > alone ? issue : alone;
            // the memory's share: all blocks together at 3400 bytes a clock, one at 60 at most
            const double bytes = (double)rt * kb_slice * 4096.0;
            const double mem = bytes * (active / 3400.0 > 1.0 / 60.0 ? active / 3400.0 : 1.0 / 60.0);
            const double work = steps * step;
            const double round = (mem > work ? mem : work) + 0.15 * (mem > work ? work : mem) + (cs > 1 ? 2800.0 : 700.0);
            // (a cluster's rounds wait for one another's remote reads: 4 us each were measured)
            const double cost = most * round + (cs > 1 ? (most - 1) * 7000.0 : 0.0) + (double)kb_slice * w4::KB / 8 * tb / w4::THREADS * fill * 4.5;
            if (best == 0 || cost < best) {
                best = cost;
                w4::Params& p = out->p;
                p.kb_total = kb_total;
                p.cs = cs;
                p.cs_log2 = cs == 8 ? 3 : cs / 2;
                p.rt = rt;
                p.tb = tb;
                p.slots = slots;
                p.row_rounds = (int)row_rounds;
                p.once = once ? 1 : 0;
                const uint32_t ring_end = (uint32_t)(w4::HEAD_BYTES + slots * w4::RING_BYTES);
                p.off_part = once ? (uint32_t)w4::HEAD_BYTES : ring_end;
                p.off_x = ring_end + (once ? 0 : (uint32_t)part);
                p.off_table = p.off_x + (uint32_t)x_bytes;
                out->grid = (int)(clusters * cs);
                out->rounds = rounds;
                out->smem = (int)(1024 + p.off_table + table);
            }
        }
    }
    return best != 0;
}

// Tokens per block: all of them up to 32, in blocks of equal size beyond; of grouped rows the kernel
// learns the groups' sizes itself, and twice the average leaves few experts with a second block.  The
// choice is a pure function of the sizes, so the last few are kept per thread (it costs as much as a launch).
bool plan_search(const int (&fits)[4], const Asked& asked, const W4Args& a, w4::Plan* plan, int* tc, int* tries) {
    int64_t want = a.m;
    if (a.offsets) {
        const int64_t twice = 2 * ((a.m + a.experts - 1) / a.experts) + 2;
        if (want > twice) want = twice;
    }
    if (asked.tb && want > asked.tb) want = asked.tb;
    *tc = *tries = 0;
    // More blocks where the activations of one would not fit.  What fits goes by the power of two above tb, so only
    // those are tried: six at most, whatever the number of tokens.
    for (int64_t most = 32;;) {
        const int64_t passes = (want + most - 1) / most;
        const int tb = (int)((want + passes - 1) / passes);
        int t = 1;
        while (t < tb) t *= 2;
        ++*tries;
        if (make_plan(fits, asked, a, tb, t, plan)) {
            *tc = t;
            return true;
        }
        if (tb == 1 || asked.tb) return false;
        most = t / 2;
    }
}

void fits_of(DeviceCtx* ctx, int (&fits)[4]) {
    for (int i = 0; i < 4; ++i) fits[i] = w4::cluster_fit(ctx, 1 << i);
}

bool plan_for(DeviceCtx* ctx, const W4Args& a, w4::Plan* plan, int* tc) {
    struct Entry {
        int64_t m, rows, cols, group, experts;
        int kind, grouped, device, tc;
        Asked asked;
        w4::Plan plan;
    };
    const Asked asked = asked_shape();
    static thread_local Entry cache[8];
    static thread_local int used = 0, next = 0;
    const int grouped = a.offsets ? 1 : 0;
    for (int i = 0; i < used; ++i) {
        const Entry& e = cache[i];
        if (e.m == a.m && e.rows == a.rows && e.cols == a.cols && e.group == a.group && e.experts == a.experts &&
            e.kind == a.kind && e.grouped == grouped && e.device == ctx->device && e.asked == asked) {
            *plan = e.plan;
            *tc = e.tc;
            return e.tc != 0;
        }
    }
    int fits[4], tries;
    fits_of(ctx, fits);
    plan_search(fits, asked, a, plan, tc, &tries);
    cache[next] = Entry{a.m, a.rows, a.cols, a.group, a.experts, a.kind, grouped, ctx->device, *tc, asked, *plan};
    next = (next + 1) % 8;
    if (used < 8) ++used;
    return *tc != 0;
}

int64_t launch_warp_kernel(DeviceCtx* ctx, const W4Args& a) {
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

}  // namespace

void describe_gemv_w4(DeviceCtx* ctx, const W4Args& a, int64_t* out) {
    int fits[4] = {148, 74, 33, 15}, tc, tries;  // of a whole B200
    if (ctx) fits_of(ctx, fits);
    w4::Plan plan;
    const bool found = plan_search(fits, asked_shape(), a, &plan, &tc, &tries);
    for (int i = 0; i < 6; ++i) out[i] = 0;
    out[6] = tries;
    if (!found) return;
    const w4::Params& p = plan.p;
    const int64_t shape[6] = {p.cs, p.rt, p.tb, p.slots, plan.grid / p.cs, plan.rounds};
    for (int i = 0; i < 6; ++i) out[i] = shape[i];
}

int64_t launch_gemv_w4(DeviceCtx* ctx, const W4Args& a) {
    if (tuning().gemm_path.load() == 1 || a.cols == 0 || a.x_rows == 0) return launch_warp_kernel(ctx, a);
    const int L = a.kind == 0 ? 1 : (a.kind == 1 ? 2 : 4);
    w4::Plan plan;
    int tc = 0;
    if (!plan_for(ctx, a, &plan, &tc)) {
        if (asked_shape().any())
            return fail(MIND_B200_ERR_INVALID, "the shape that mind_b200_set_w4_shape asks for does not fit this call");
        return launch_warp_kernel(ctx, a);  // a row of activations too long for eight blocks
    }
    // TMA reads rows whose pitch and base are multiples of 16 bytes; others are copied to padded rows first
    const int64_t bytes = (a.cols + 1) / 2, pitch = (int64_t)align_up((size_t)bytes, 16);
    const int8_t* w = a.w;
    if (pitch != bytes || reinterpret_cast<uintptr_t>(w) % 16 != 0) {
        const size_t size = (size_t)(a.experts * a.rows) * pitch;
        MB200_TRY(arena_reserve(ctx, ctx->scratch, size + 2048));
        int8_t* to = static_cast<int8_t*>(arena_take(ctx->scratch, size));
        MB200_TRY(launch_copy_rows(ctx, CopyJob{w, nullptr, to, a.experts * a.rows, bytes, pitch, a.experts * a.rows}, nullptr));
        w = to;
    }
    CUtensorMap tm;
    MB200_TRY(make_tmap_stack(&tm, w, bytes, a.rows, a.experts, pitch, 16));
    w4::Params& p = plan.p;
    p.a = a;
    p.groups = (int)((a.cols + a.group - 1) / a.group);
    p.group32 = (int)(a.group / 32);
    const int gb = p.group32 % 4 == 0 ? 4 : (p.group32 % 2 == 0 ? 2 : 1), ns = w4::KB / 128 / gb;
    p.group_shift = -1;
    for (int i = 0; i < 31; ++i)
        if (p.group32 == 1 << i) p.group_shift = i;
    p.scale_vec = p.group32 == gb && p.groups % ns == 0 && reinterpret_cast<uintptr_t>(a.scale) % (2 * ns) == 0 ? 1 : 0;
    p.x_vec = a.cols % 8 == 0 && reinterpret_cast<uintptr_t>(a.x) % (L == 1 ? 8 : 16) == 0 ? 1 : 0;
    p.err = ctx->err_word;
    if (a.kind == 0) return w4::launch_i8(ctx, tm, plan, tc);
    if (a.kind == 1) return w4::launch_i16(ctx, tm, plan, tc);
    return w4::launch_q16(ctx, tm, plan, tc);
}

}  // namespace mb200
