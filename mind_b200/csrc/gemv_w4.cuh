// The tensor-core kernel of the 4-bit matrix-vector products (see gemv_w4.cu for the rule).
//
// Memory-bound: every weight is read once, half a byte each, and meets 1 .. 32 tokens.  The products run
// on mma.sync.m16n8k32 (s8 weights x u8 / s8 activation bytes, exact int32 sums): 16 rows of W meet eight
// columns at once, so a warp spends a handful of instructions per 512 weights whatever the number of
// columns up to eight; one multiply-add instruction per four weights and column (dp4a) would be the bound
// from three columns on.  tcgen05 would want the 4-bit weights unpacked into shared memory first.
//
// * Activations become columns of bytes: x = sum_i limb_i * 256^i, all but the top limb unsigned.  With
//   few tokens one set of accumulators holds all limbs as columns (PACK: two MMAs, unsigned and signed
//   columns, the other ones zero); with more, eight tokens and one limb make an MMA.
// * Weights arrive as they lie, in boxes of 16 rows x 256 columns, by TMA into a ring of 2 KiB slots that
//   each warp keeps for itself: no barrier between warps in the main loop.  A word of eight weights
//   becomes two registers of four by masking, as 16 times the weight: the factor leaves with the final
//   shift.
// * After GB x 32 columns (GB = 4, 2 or 1: a divisor of the group) the int32 sums are multiplied by the
//   group's scale and added up in 64 bits, in registers.  Lane t of a row's four takes GB consecutive
//   words of those columns with one load, and the MMAs take the words in turn: MMA i has the columns
//   8 GB t + 8 i + {0,2,4,6} / {1,3,5,7} at its k = 4 t + {0..3} / 16 + 4 t + {0..3}.  The activations
//   are laid out in shared memory in that order, once per block of tokens.
// * 16 warps share `rt` row tiles, 16 / rt warps to a tile, which take its units of 512 columns in turn; a
//   cluster of up to eight blocks shares the columns where a block's activations would not fit beside
//   the ring, or where there are fewer row tiles than warps.  The partial sums meet in shared memory,
//   across the cluster by remote reads: integer sums, so no order changes a bit, and nothing is kept in
//   global memory.
//
// What bounds it.  One or two tokens: memory behind a set-up of about 5 us (28672 x 8192 int8: 24.9 to 26.0
// us a call, 4.8 TB/s of weights and scales, 0.73 of the copy bandwidth; int16 and Q16.16 31 us; 4096 x 4096
// Q16.16: 6.4 us, of which the host needs about as much to make the call).  More: the latency of the main loop
// on four warps a scheduler (8192 x 8192 Q16.16, eight tokens, groups of 32: 22.4 us against 5.9 us of memory
// time; 0.44 instructions a clock and scheduler, no pipe more than half busy).  MMAs run at 8.2 clocks a
// scheduler whatever their operands.
#pragma once
#include "common.h"
#include "ptx.cuh"

namespace mb200 {
namespace w4 {
using namespace ptx;

constexpr int WARPS = 16, THREADS = 32 * WARPS;
constexpr int BOX_BYTES = 2048;                     // 16 rows x 128 bytes: one TMA box
constexpr int RING_BYTES = WARPS * BOX_BYTES;       // one slot of every warp
constexpr int KB = 512;                             // columns of a unit: two boxes
constexpr int SMEM_MAX = 232448;
constexpr int MAX_SLOTS = 8;
constexpr int HEAD_BYTES = 2048;                    // barriers and scan scratch

struct Params {
    W4Args a;
    int kb_total;         // units of 512 columns
    int cs, cs_log2, rt;  // cluster size; row tiles per round
    int tb;               // tokens per block, at most
    int slots;            // ring depth, in boxes
    int row_rounds;       // rounds of 16 * rt rows per matrix
    int once;             // no cluster has more than one round: the partial sums take the ring's place
    int groups, group32;  // groups per row; 32-column blocks per group
    int group_shift;      // log2 of group32, or -1
    int x_vec;            // x may be read eight elements at a time
    int scale_vec;        // a group is one scaling, and a lane's scales of a unit are one aligned load
    uint32_t off_part, off_x, off_table;  // shared-memory layout, from the aligned base
    int* err;
};

// D (+)= A . B, 16 x 32 weights (s8) by 32 x 8 activation bytes.  FIRST: D = A . B.
template <bool SIGNED, bool FIRST>
__device__ __forceinline__ void mma(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
#define MB200_W4_MMA(T, C, ...)                                                                                          \
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8." T ".s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, " C ";" __VA_ARGS__)
#define MB200_W4_IN "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1)
#define MB200_W4_NEW : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : MB200_W4_IN, "r"(0)
#define MB200_W4_ADD : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : MB200_W4_IN
    if constexpr (SIGNED && FIRST) MB200_W4_MMA("s8", "{%10,%10,%10,%10}", MB200_W4_NEW);
    else if constexpr (SIGNED) MB200_W4_MMA("s8", "{%0,%1,%2,%3}", MB200_W4_ADD);
    else if constexpr (FIRST) MB200_W4_MMA("u8", "{%10,%10,%10,%10}", MB200_W4_NEW);
    else MB200_W4_MMA("u8", "{%0,%1,%2,%3}", MB200_W4_ADD);
#undef MB200_W4_MMA
#undef MB200_W4_IN
#undef MB200_W4_NEW
#undef MB200_W4_ADD
}
template <bool SIGNED>
__device__ __forceinline__ void mma_step(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool first) {
    if (first) mma<SIGNED, true>(d, a, b0, b1);
    else mma<SIGNED, false>(d, a, b0, b1);
}
// 4 * N bytes of shared memory.
template <int N>
__device__ __forceinline__ void lds(uint32_t (&v)[N], uint32_t addr) {
    if constexpr (N == 4)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
    else if constexpr (N == 2)
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(addr) : "memory");
    else
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(addr) : "memory");
}
// Bytes of activations of one column that lane t holds for GB MMAs: in pieces of at most 16, so that
// the lanes of a load lie side by side.
template <int GB>
struct XPiece {
    static constexpr int BYTES = GB == 1 ? 8 : 16, PIECES = 8 * GB / BYTES, MMAS = BYTES / 8;
};

// Eight activations from element `at` on, as they lie in memory: 2 * L words, aligned.
template <int L>
__device__ __forceinline__ void load8_vec(const void* x, int64_t at, uint32_t (&v)[2 * L]) {
    const char* const p = static_cast<const char*>(x) + at * L;
    if constexpr (L == 1) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        v[0] = w.x;
        v[1] = w.y;
    } else {
#pragma unroll
        for (int i = 0; i < L / 2; ++i) {
            const uint4 w = *reinterpret_cast<const uint4*>(p + 16 * i);
            v[4 * i] = w.x;
            v[4 * i + 1] = w.y;
            v[4 * i + 2] = w.z;
            v[4 * i + 3] = w.w;
        }
    }
}
// The same of row xr from column k on, at any alignment, with zeros past the end.
template <int L>
__device__ __forceinline__ void load8(const Params& p, int64_t xr, int64_t k, uint32_t (&v)[2 * L]) {
    const char* const at = static_cast<const char*>(p.a.x) + (xr * p.a.cols + k) * L;
#pragma unroll
    for (int i = 0; i < 2 * L; ++i) v[i] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (k + i < p.a.cols) {
            if constexpr (L == 1) v[i / 4] |= (uint32_t)*reinterpret_cast<const uint8_t*>(at + i) << (8 * (i % 4));
            else if constexpr (L == 2) v[i / 2] |= (uint32_t)*reinterpret_cast<const uint16_t*>(at + 2 * i) << (16 * (i % 2));
            else v[i] = *reinterpret_cast<const uint32_t*>(at + 4 * i);
        }
}
// Limb l of the activations 0, 2, 4, 6 (odd = 0) or 1, 3, 5, 7 (odd = 1) of such words.
template <int L>
__device__ __forceinline__ uint32_t limb4(const uint32_t (&v)[2 * L], int l, int odd) {
    if constexpr (L == 1) return __byte_perm(v[0], v[1], odd ? 0x7531 : 0x6420);
    if constexpr (L == 2) {
        const uint32_t sel = (l + 2 * odd) | ((l + 2 * odd + 4) << 4);
        return __byte_perm(__byte_perm(v[0], v[1], sel), __byte_perm(v[2], v[3], sel), 0x5410);
    } else if constexpr (L == 4) {
        const uint32_t sel = l | ((l + 4) << 4);
        return __byte_perm(__byte_perm(v[odd], v[2 + odd], sel), __byte_perm(v[4 + odd], v[6 + odd], sel), 0x5410);
    }
    return 0;
}
// The rest of a wait that did not end at once.
static __device__ __noinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile int* abort_s, int* err) {
    return wait_bounded(bar, parity, abort_s, err, 5);
}

// L: limbs of an activation (1 = int8, 2 = int16, 4 = Q16.16).  TC: tokens that a block has room for (the
// layout of the activations, and with it every address of the main loop, is fixed by it).  GB: 32-column
// blocks between two scalings.
template <int L, int TC, int GB>
__global__ void __launch_bounds__(THREADS, 1) gemv_w4_mma_kernel(const __grid_constant__ CUtensorMap tm_w, const Params p) {
    constexpr bool PACK = L > 1 && L * TC <= 8;  // all limbs of the tokens in one set of accumulators
    constexpr int NT = (TC + 7) / 8;      // blocks of eight tokens
    constexpr int LT = PACK ? 1 : L;      // accumulator sets between scalings
    constexpr int AC = 8 * NT;            // accumulator columns of a warp
    constexpr int PS = 17;                // partial sums: a column's 16 rows lie side by side, so that remote reads are whole lines
    constexpr int TP = PACK ? 8 / L : 1;  // tokens per limb in a packed set
    constexpr int NF = KB / 32 / GB;      // scalings per unit
    constexpr int FB = NF / 2;            // per box
    constexpr int NS = NF / 4;            // of which every lane of four holds NS consecutive ones
    using XP = XPiece<GB>;
    constexpr int XCOLS = L * TC;              // columns of activation bytes
    constexpr int CSTRIDE = XCOLS * 32 * GB;   // bytes of the activations between two scalings
    constexpr int LIMB_STRIDE = TC * 4 * XP::BYTES, PIECE_STRIDE = XCOLS * 4 * XP::BYTES;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* const gbase = smem_raw + (base - raw);
    const uint32_t ring0 = base + HEAD_BYTES;
    int* const misc = reinterpret_cast<int*>(gbase + WARPS * MAX_SLOTS * 8);
    volatile int* const abort_s = misc;
    uint64_t* const part = reinterpret_cast<uint64_t*>(gbase + p.off_part);  // [warp][AC][PS]
    const uint32_t xs = base + p.off_x;
    int* const bound = reinterpret_cast<int*>(gbase + p.off_table);  // [experts + 1] first row of each
    int* const cumb = bound + p.a.experts + 1;                       // [experts + 1] token blocks before each

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // The row of the tile that MMA row g stands for: with its bits reversed the lanes of one phase of a
    // load fall on different 16-byte columns of the swizzled box, whatever GB.
    const int row = ((g & 1) << 2) | (g & 2) | (g >> 2);
    const int rt = p.rt, wpr = WARPS / rt;       // warps beyond rt * wpr only help with the activations
    const int my_tile = warp % rt, my_part = warp / rt;
    const uint32_t rank = p.cs > 1 ? cluster_ctarank() : 0u;
    const int clusters = gridDim.x / p.cs, cluster = blockIdx.x / p.cs;
    const uint32_t bars = base + warp * MAX_SLOTS * 8, slots0 = ring0 + warp * BOX_BYTES;

    griddep_launch_dependents();
    if (lane == 0)
        for (int s = 0; s < p.slots; ++s) mbar_init(bars + 8 * s, 1);
    if (threadIdx.x == 0) {
        *abort_s = 0;
        prefetch_tensormap(&tm_w);
    }
    if (lane == 0) fence_mbar_init();
    // Before the wait for the kernel in front nothing may be read that it could have written: grouped rows
    // wait here, for their offsets; one matrix waits behind the set-up.
    if (p.a.offsets) griddep_wait();

    // ---- token blocks: bound = running maximum of the offsets within [0, m], cumb = running sum of
    // the blocks of at most tb rows
    if (!p.a.offsets) {
        if (threadIdx.x == 0) {
            bound[0] = cumb[0] = 0;
            bound[1] = (int)p.a.m;
            cumb[1] = ((int)p.a.m + p.tb - 1) / p.tb;
        }
    } else {
        const int experts = (int)p.a.experts, m = (int)p.a.m;
        auto offset = [&](int e) { return min(max(p.a.offsets[e], 0), m); };
        const int per = (experts + THREADS - 1) / THREADS;
        const int e0 = min((int)threadIdx.x * per, experts), e1 = min(e0 + per, experts);
        const int first = offset(0);
        int mx = first;
        for (int e = e0; e < e1; ++e) {
            bound[e + 1] = offset(e + 1);
            mx = max(mx, bound[e + 1]);
        }
        int incl = mx;
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl = max(incl, v);
        }
        if (lane == 31) misc[4 + warp] = incl;
        int before = __shfl_up_sync(0xffffffffu, incl, 1);
        if (lane == 0) before = first;
        __syncthreads();
        for (int w = 0; w < warp; ++w) before = max(before, misc[4 + w]);
        int blocks = 0, lo = before;
        for (int e = e0; e < e1; ++e) {
            const int hi = max(lo, bound[e + 1]);
            bound[e + 1] = hi;
            blocks += (hi - lo + p.tb - 1) / p.tb;
            lo = hi;
        }
        int sum = blocks;
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        if (lane == 31) misc[24 + warp] = sum;
        __syncthreads();
        int at = sum - blocks;
        for (int w = 0; w < warp; ++w) at += misc[24 + w];
        lo = before;
        for (int e = e0; e < e1; ++e) {
            const int hi = bound[e + 1];
            at += (hi - lo + p.tb - 1) / p.tb;
            cumb[e + 1] = at;
            lo = hi;
        }
        if (threadIdx.x == 0) {
            bound[0] = first;
            cumb[0] = 0;
        }
    }
    __syncthreads();
    if (p.cs > 1) {  // every block of the cluster is running before any writes into another
        cluster_arrive();
        cluster_wait();
    }
    // Rounds (token block, 16 * rt rows) are handed out in equal runs, one run to a cluster.
    const unsigned rounds = (unsigned)cumb[p.a.experts] * (unsigned)p.row_rounds;
    const unsigned run = rounds / (unsigned)clusters, more = rounds - run * (unsigned)clusters;
    const int u0 = (int)(run * cluster + min((unsigned)cluster, more)), u1 = u0 + (int)run + ((unsigned)cluster < more ? 1 : 0);
    const int kb_lo = (int)((unsigned)p.kb_total * rank >> p.cs_log2), kb_hi = (int)((unsigned)p.kb_total * (rank + 1) >> p.cs_log2);
    const int kb_first = my_part < wpr ? kb_lo + my_part : kb_hi;
    const uint64_t policy = l2_policy(0);

    // This warp's units of a round: columns kb_first, kb_first + wpr, ...  Its boxes, in order: two a unit, but
    // for a last unit that ends in its first.
    const int steps = kb_first < kb_hi ? (kb_hi - kb_first + wpr - 1) / wpr : 0;
    const int boxes = 2 * steps - (steps && (int64_t)(kb_first + (steps - 1) * wpr) * KB + KB / 2 >= p.a.cols ? 1 : 0);
    auto group_of = [&](int blk) { return p.group_shift >= 0 ? blk >> p.group_shift : blk / p.group32; };
    // the scales of row r of expert e (rows past the end meet zero weights: any scale will do)
    auto scale_row = [&](int e, int r) {
        return p.a.scale + ((int64_t)e * p.a.rows + min((int64_t)r, p.a.rows - 1)) * p.groups;
    };
    bool lead = lane == 0;  // asks for the boxes; nobody does any more once a wait has run out

    int is_u = boxes ? u0 : u1, is_e = 0, is_row0 = 0, is_box = 0, is_x = kb_first * (KB / 2), fill = 0;  // next load
    auto place = [&]() {
        const int q = (int)((unsigned)is_u / (unsigned)p.row_rounds);
        while (q >= cumb[is_e + 1]) ++is_e;
        is_row0 = ((is_u - q * p.row_rounds) * rt + my_tile) * 16;
    };
    auto issue = [&](bool done) {  // done: the slot's last box has been multiplied (or it never held one)
        if (is_u >= u1) return;
        if (lead && done) {
            mbar_arrive_expect_tx(bars + 8 * fill, BOX_BYTES);
            tma_load_3d(slots0 + fill * RING_BYTES, &tm_w, bars + 8 * fill, is_x, is_row0, is_e, policy);
        }
        fill = fill + 1 == p.slots ? 0 : fill + 1;
        if (++is_box == boxes) {
            is_box = 0;
            is_x = kb_first * (KB / 2);
            if (++is_u < u1) place();
        } else {
            is_x += (is_box & 1) ? 128 : wpr * (KB / 2) - 128;
        }
    };
    if (is_u < u1) place();
    // A round's scales, towards L2: the warps of a row tile share the sectors of its rows.
    auto prefetch_scales = [&](int u, int e) {
        const int q = (int)((unsigned)u / (unsigned)p.row_rounds);
        while (q >= cumb[e + 1]) ++e;
        const int r = ((u - q * p.row_rounds) * rt + my_tile) * 16 + row;
        const int g0 = group_of(kb_lo * (KB / 32)), g1 = min(group_of(kb_hi * (KB / 32) - 1), p.groups - 1);
        const int16_t* const a0 = scale_row(e, r);
        const int16_t* const a8 = scale_row(e, r + 8);
        for (int gi = g0 + (my_part * 4 + t) * 16; gi <= g1 + 15 && my_part < wpr; gi += wpr * 64) {
            const int at = min(gi, g1);
            asm volatile("prefetch.global.L2 [%0];" ::"l"(a0 + at));
            asm volatile("prefetch.global.L2 [%0];" ::"l"(a8 + at));
        }
    };

    // Scales of a unit: lane t holds those of scalings t * NS .. t * NS + NS - 1, of two rows.  (Past the last
    // group the weights are zeros, and the last scales are as good as any.)
    int sc0[NS], sc1[NS];
    auto load_scales = [&](const int16_t* s, const int16_t* s8, int kb) {
        if (p.scale_vec) {  // a group is one scaling, and a lane's are one aligned load
            const int gi = min(kb * NF + t * NS, p.groups - NS);
            auto fetch = [&](const int16_t* q, int (&sc)[NS]) {
                if constexpr (NS == 1) {
                    sc[0] = __ldg(q);
                } else if constexpr (NS == 2) {
                    const int v = __ldg(reinterpret_cast<const int*>(q));
                    sc[0] = (int)(int16_t)v;
                    sc[1] = v >> 16;
                } else {
                    const int2 v = __ldg(reinterpret_cast<const int2*>(q));
                    sc[0] = (int)(int16_t)v.x;
                    sc[1] = v.x >> 16;
                    sc[2] = (int)(int16_t)v.y;
                    sc[3] = v.y >> 16;
                }
            };
            fetch(s + gi, sc0);
            fetch(s8 + gi, sc1);
        } else {
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const int gi = min(group_of(kb * (KB / 32) + (t * NS + i) * GB), p.groups - 1);
                sc0[i] = __ldg(s + gi);
                sc1[i] = __ldg(s8 + gi);
            }
        }
    };

    int take = 0;
    uint32_t phase = 0;
    int block = -1, ntok = 0, p0 = 0, e_now = 0;
    const int rows_round = 16 * rt;

    if (!p.a.offsets) griddep_wait();
    bool asked = false;  // the ring's first loads go out behind the first loads of activations
    for (int u = u0; u < u1; ++u) {
        const int q = (int)((unsigned)u / (unsigned)p.row_rounds);
        if (q != block) {
            // ---- a new block of tokens: its activations, as bytes in the order the MMAs take them
            block = q;
            while (q >= cumb[e_now + 1]) ++e_now;
            const unsigned nb = cumb[e_now + 1] - cumb[e_now], i = q - cumb[e_now];
            const unsigned rows_e = bound[e_now + 1] - bound[e_now], per = rows_e / nb, extra = rows_e - per * nb;
            p0 = bound[e_now] + (int)(i * per + min(i, extra));
            ntok = (int)per + (i < extra ? 1 : 0);
            // A thread owns groups of eight columns and takes them token by token (the block several tokens at once
            // where the columns are few): 16 or 32 registers of loads before the first store (more lengthen the
            // code: 4096 x 4096 int8 of eight tokens 8.7 us with 16, 9.6 with 32), and the weights are asked for
            // behind the last of them, not before, where the activations would have to queue.
            const int octs = (kb_hi - kb_lo) * (KB / 8);
            const int width = octs < THREADS ? octs : THREADS, tstep = THREADS / width;
            const int tok0 = (int)threadIdx.x / width, o0 = (int)threadIdx.x - tok0 * width;
            constexpr int BATCH = TC <= 2 ? 2 * TC : (L == 1 ? 8 : 4);
            int lo = o0, lt = tok0, so = o0, st = tok0;  // next to load, next to store: columns, token
            if (tok0 >= tstep || tok0 >= ntok) lo = so = octs;
            while (so < octs) {
                uint32_t v[BATCH][2 * L];
                if (p.x_vec) {
                    // No branch between the loads, which would end one before the next begins: what is not there is
                    // read from the first row and replaced by zeros.
                    int64_t at[BATCH];
                    unsigned there = 0;
#pragma unroll
                    for (int b = 0; b < BATCH; ++b) {
                        const int tok = min(lt, ntok - 1);
                        const int64_t xr = p.a.rows_of ? p.a.rows_of[p0 + tok] : p0 + tok, k = (int64_t)kb_lo * KB + 8 * lo;
                        const bool ok = lo < octs && k < p.a.cols && xr >= 0 && xr < p.a.x_rows;
                        at[b] = ok ? xr * p.a.cols + k : 0;
                        there |= ok ? 1u << b : 0u;
                        lt += tstep;
                        lo += lt >= ntok ? width : 0;
                        lt = lt >= ntok ? tok0 : lt;
                    }
#pragma unroll
                    for (int b = 0; b < BATCH; ++b) load8_vec<L>(p.a.x, at[b], v[b]);
#pragma unroll
                    for (int b = 0; b < BATCH; ++b)
#pragma unroll
                        for (int j = 0; j < 2 * L; ++j) v[b][j] = there >> b & 1u ? v[b][j] : 0u;
                } else {
#pragma unroll
                    for (int b = 0; b < BATCH; ++b) {
#pragma unroll
                        for (int j = 0; j < 2 * L; ++j) v[b][j] = 0;
                        if (lo >= octs) continue;
                        const int64_t xr = p.a.rows_of ? p.a.rows_of[p0 + lt] : p0 + lt;
                        if (xr >= 0 && xr < p.a.x_rows) load8<L>(p, xr, (int64_t)kb_lo * KB + 8 * lo, v[b]);
                        lt += tstep;
                        if (lt >= ntok) {
                            lt = tok0;
                            lo += width;
                        }
                    }
                }
                if (!asked && lo >= octs) {
                    asked = true;
                    for (int s = 0; s < p.slots; ++s) issue(true);
                }
#pragma unroll
                for (int b = 0; b < BATCH; ++b) {
                    if (so >= octs) break;
                    const int m = so % GB;  // MMA that takes these eight columns
                    const uint32_t at = xs + so / (4 * GB) * CSTRIDE + (m / XP::MMAS) * PIECE_STRIDE +
                                        (st * 4 + (so / GB & 3)) * XP::BYTES + (m % XP::MMAS) * 8;
#pragma unroll
                    for (int l = 0; l < L; ++l)
                        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at + l * LIMB_STRIDE),
                                     "r"(limb4<L>(v[b], l, 0)), "r"(limb4<L>(v[b], l, 1))
                                     : "memory");
                    st += tstep;
                    if (st >= ntok) {
                        st = tok0;
                        so += width;
                    }
                }
            }
            if (!asked) {
                asked = true;
                for (int s = 0; s < p.slots; ++s) issue(true);
            }
            if (u == u0) prefetch_scales(u0, e_now);
            __syncthreads();
        }
        // ---- this warp's units of the round
        int64_t acc64[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc64[n][i] = 0;
        // Packed: column g is limb g / TP of token g % TP.  A column without a token takes another's bytes
        // (its sums are never looked at), so that no load is conditional.
        const bool col_top = PACK && g / TP == L - 1;
        int xtok[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) xtok[n] = (PACK ? (g % TP < ntok ? g % TP : 0) : (n * 8 + g < ntok ? n * 8 + g : 0)) * 4 * XP::BYTES;
        const uint32_t xcol = xs + (PACK ? g / TP : 0) * LIMB_STRIDE + t * XP::BYTES;
        const int tile_row0 = ((u - q * p.row_rounds) * rt + my_tile) * 16;
        const int16_t* const srow = scale_row(e_now, tile_row0 + row);
        const int16_t* const srow8 = scale_row(e_now, tile_row0 + row + 8);
        load_scales(srow, srow8, kb_first);
        if (u + 1 < u1) prefetch_scales(u + 1, e_now);
        uint32_t xnext = xcol + (kb_first - kb_lo) * NF * CSTRIDE;  // activations of the next scaling
        for (int j = 0, kb = kb_first; j < steps; ++j, kb += wpr) {
            int sc[2][NS];
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                sc[0][i] = sc0[i];
                sc[1][i] = sc1[i];
            }
            load_scales(srow, srow8, kb + wpr);
            uint32_t xat = xnext;
            xnext += wpr * NF * CSTRIDE;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
            if (h == 1 && 2 * j + 1 == boxes) break;
            if (!mbar_try_wait(bars + 8 * take, phase)) lead = wait_on(bars + 8 * take, phase, abort_s, p.err) && lead;
            // this lane's words of scaling f of the box lie at wbase ^ (f * 16 GB), the box's swizzle included
            const uint32_t wbase = slots0 + take * RING_BYTES + row * 128 +
                                   (((t * GB / 4) ^ row) << 4) + (t * GB % 4) * 4;
            int used = 0;  // depends on every word of the box
#pragma unroll
            for (int f = 0; f < FB; ++f) {
                const int m0 = __shfl_sync(0xffffffffu, sc[0][f % NS], (lane & 28) | (h * (FB / NS) + f / NS));
                const int m1 = __shfl_sync(0xffffffffu, sc[1][f % NS], (lane & 28) | (h * (FB / NS) + f / NS));
                uint32_t w0[GB], w1[GB], a[GB][4];
                const uint32_t at = wbase ^ (f * 16 * GB);
                lds<GB>(w0, at);
                lds<GB>(w1, at + 1024);
#pragma unroll
                for (int b = 0; b < GB; ++b) {
                    a[b][0] = (w0[b] << 4) & 0xf0f0f0f0u;
                    a[b][1] = (w1[b] << 4) & 0xf0f0f0f0u;
                    a[b][2] = w0[b] & 0xf0f0f0f0u;
                    a[b][3] = w1[b] & 0xf0f0f0f0u;
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (NT > 1 && n * 8 >= ntok) break;
                    int acc[LT][4];
                    const uint32_t xb = xat + xtok[n];
                    uint32_t x[LT][XP::PIECES][2 * XP::MMAS];
#pragma unroll
                    for (int l = 0; l < LT; ++l)
#pragma unroll
                        for (int q = 0; q < XP::PIECES; ++q) lds<2 * XP::MMAS>(x[l][q], xb + l * LIMB_STRIDE + q * PIECE_STRIDE);
                    // one word of every limb's chain after the other: LT sums that do not wait for each other
#pragma unroll
                    for (int b = 0; b < GB; ++b)
#pragma unroll
                        for (int l = 0; l < LT; ++l) {
                            const uint32_t x0 = x[l][b / XP::MMAS][2 * (b % XP::MMAS)], x1 = x[l][b / XP::MMAS][2 * (b % XP::MMAS) + 1];
                            if (PACK) {  // the unsigned columns, then the signed ones
                                mma_step<false>(acc[0], a[b], col_top ? 0u : x0, col_top ? 0u : x1, b == 0);
                                mma_step<true>(acc[0], a[b], col_top ? x0 : 0u, col_top ? x1 : 0u, false);
                            } else if (l < L - 1) {
                                mma_step<false>(acc[l], a[b], x0, x1, b == 0);
                            } else {
                                mma_step<true>(acc[l], a[b], x0, x1, b == 0);
                            }
                        }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (n == 0 && i == 0) used ^= acc[LT - 1][0];
                        const int m = i < 2 ? m0 : m1;
                        if (PACK || L == 1) {
                            acc64[n][i] += (int64_t)m * acc[0][i];
                        } else if (L == 2) {
                            acc64[n][i] += (int64_t)m * (acc[0][i] + 256 * acc[LT - 1][i]);
                        } else {
                            acc64[n][i] += (int64_t)m * (acc[0][i] + 256 * acc[LT > 1 ? 1 : 0][i]);
                            acc64[n][i] += (int64_t)(int32_t)((uint32_t)m << 16) * (acc[LT > 2 ? 2 : 0][i] + 256 * acc[LT - 1][i]);
                        }
                    }
                }
                xat += CSTRIDE;
            }
            // The slot may be filled again once every lane's words of the box have been USED: nothing else keeps a
            // load of them from following the refill (the compiler sees no address in common, and an order left to
            // it failed in the fused Q16.16 kernel).  So the refill is predicated on a vote over sums that each
            // scaling's words went through.  They stay below 2^23 in magnitude, so bits 30 and 31 agree in all of
            // them: the vote always succeeds, which the compiler cannot know.
            const bool done = __all_sync(0xffffffffu, used != 0x40000000);
            take = take + 1 == p.slots ? 0 : take + 1;
            phase ^= take == 0 ? 1u : 0u;
            issue(done);
            }
        }
        // ---- the round's partial sums: of wpr warps here, and of the cluster's other columns
        if (p.once) __syncthreads();  // every box has been multiplied: the sums may take the ring's place
        uint64_t* const mine = part + warp * AC * PS;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) mine[(n * 8 + 2 * t + (i & 1)) * PS + row + 8 * (i >> 1)] = (uint64_t)acc64[n][i];
        __syncwarp();
        if (p.cs > 1) {
            cluster_arrive();
            cluster_wait();
        } else {
            __syncthreads();
        }
        const int row_first = (u - q * p.row_rounds) * rows_round;
        const int outs = rows_round * ntok;
        const unsigned by = (unsigned)rows_round;
        const int all = p.cs * wpr;
        // A thread adds up an output: the partial sums of all the cluster's warps as one list, four (remote) loads
        // at a time.  (Eight: 24.4 against 23.0 us for 8192 x 8192 Q16.16 of eight tokens; eight outputs of one
        // warp each 25.9.  Several of these forms, chosen by the sizes, are behind one again: their code is long.)
        constexpr int AT_ONCE = 4, LS = PACK ? L : 1;
        for (int o = (int)rank * THREADS + threadIdx.x; o < outs; o += p.cs * THREADS) {
            const int tok = (int)((unsigned)o / by), rr = o - tok * rows_round, r = row_first + rr;
            const uint32_t from = smem_u32(part + ((rr >> 4) * AC + tok) * PS + (rr & 15));
            uint64_t sum = 0;
            int c = 0, w = 0;
            for (int j0 = 0; j0 < all; j0 += AT_ONCE) {
                uint64_t v[AT_ONCE][LS];
#pragma unroll
                for (int k = 0; k < AT_ONCE; ++k) {
#pragma unroll
                    for (int l = 0; l < LS; ++l)  // (one too many repeats the last; a block's own memory is rank 0 of one)
                        asm volatile("ld.shared::cluster.u64 %0, [%1];"
                                     : "=l"(v[k][l])
                                     : "r"(mapa(from + (uint32_t)((w * rt * AC + l * TP) * PS * 8), (uint32_t)c))
                                     : "memory");
                    if (j0 + k + 1 < all) {
                        c += w + 1 == wpr ? 1 : 0;
                        w = w + 1 == wpr ? 0 : w + 1;
                    }
                }
#pragma unroll
                for (int k = 0; k < AT_ONCE; ++k)
#pragma unroll
                    for (int l = 0; l < LS; ++l) sum += j0 + k < all ? v[k][l] << (PACK ? 8 * l : 0) : 0;
            }
            if (r < p.a.rows) p.a.y[(int64_t)(p0 + tok) * p.a.rows + r] = (int32_t)((int64_t)sum >> (p.a.shift + 4));
        }
        // the sums and the activations may be overwritten (and no block leaves while another reads from it)
        __syncwarp();
        if (p.cs > 1) {
            cluster_arrive();
            cluster_wait();
        } else if (!p.once) {
            __syncthreads();
        }
    }
    if (*abort_s) __nanosleep(200000);  // let copies still in flight land
}

struct Plan {
    Params p;
    int grid, smem;
    int64_t rounds;  // of all clusters together (of grouped rows: as estimated)
};

template <int L, int TC, int GB>
int64_t launch(DeviceCtx* ctx, const CUtensorMap& tm, const Plan& plan) {
    auto kern = gemv_w4_mma_kernel<L, TC, GB>;
    static thread_local int done_for = -1;
    if (done_for != ctx->device) {
        MB200_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX));
        done_for = ctx->device;
    }
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)plan.grid, 1, 1);
    lc.blockDim = dim3(THREADS, 1, 1);
    lc.dynamicSmemBytes = plan.smem;
    lc.stream = ctx->stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = plan.p.cs;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    lc.attrs = at;
    lc.numAttrs = plan.p.cs > 1 ? 2 : 1;
    prof_begin(ctx);
    MB200_CUDA(cudaLaunchKernelEx(&lc, kern, tm, plan.p));
    prof_end(ctx);
    count_launch();
    return check_launch("gemv_w4_mma_kernel");
}

template <int L, int TC>
int64_t launch_gb(DeviceCtx* ctx, const CUtensorMap& tm, const Plan& plan) {
    const int g32 = plan.p.group32;
    if (g32 % 4 == 0) return launch<L, TC, 4>(ctx, tm, plan);
    if (g32 % 2 == 0) return launch<L, TC, 2>(ctx, tm, plan);
    return launch<L, TC, 1>(ctx, tm, plan);
}

// tc: tokens per block of the kernel, a power of two up to 32.
template <int L>
int64_t launch_tc(DeviceCtx* ctx, const CUtensorMap& tm, const Plan& plan, int tc) {
    if (tc == 1) return launch_gb<L, 1>(ctx, tm, plan);
    if (tc == 2) return launch_gb<L, 2>(ctx, tm, plan);
    if (tc == 4) return launch_gb<L, 4>(ctx, tm, plan);
    if (tc == 8) return launch_gb<L, 8>(ctx, tm, plan);
    if (tc == 16) return launch_gb<L, 16>(ctx, tm, plan);
    return launch_gb<L, 32>(ctx, tm, plan);
}

// Clusters of `cs` blocks that the device holds at once (asked once per device).
int cluster_fit(DeviceCtx* ctx, int cs);
int64_t launch_i8(DeviceCtx* ctx, const CUtensorMap& tm, const Plan& plan, int tc);
int64_t launch_i16(DeviceCtx* ctx, const CUtensorMap& tm, const Plan& plan, int tc);
int64_t launch_q16(DeviceCtx* ctx, const CUtensorMap& tm, const Plan& plan, int tc);

}  // namespace w4
}  // namespace mb200
