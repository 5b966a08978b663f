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
// * Weights arrive as they lie, 16 rows x 256 columns at a time, by TMA into a ring of 2 KiB slots that
//   each warp keeps for itself: no barrier between warps in the main loop.  A word of eight weights
//   becomes two registers of four by masking, as 16 times the weight: the factor leaves with the final
//   shift.  The columns 32 j + 8 t + {0,2,4,6} / {1,3,5,7} go where the MMA has k = 4 t + {0..3} /
//   16 + 4 t + {0..3}; the activations are laid out in shared memory in that order once per block.
// * After GB x 32 columns (a divisor of the group, at most 128 columns) the int32 sums are multiplied by
//   the group's scale and added up in 64 bits, in registers.
// * 16 warps share `rt` row tiles, 16 / rt warps to a tile, which take its 256-column blocks in turn; a
//   cluster of up to eight blocks shares the columns where a block's activations would not fit beside
//   the ring.  Partial sums meet in shared memory (across the cluster, too): integer sums, so no order
//   of arrival changes a bit, and nothing is kept in global memory.
#pragma once
#include "common.h"
#include "ptx.cuh"

namespace mb200 {
namespace w4 {
using namespace ptx;

constexpr int WARPS = 16, THREADS = 32 * WARPS;
constexpr int SLOT_BYTES = 2048;                    // 16 rows x 128 bytes
constexpr int RING_BYTES = WARPS * SLOT_BYTES;      // one slot of every warp
constexpr int KB = 256;                             // columns of a slot
constexpr int SMEM_MAX = 232448;
constexpr int MAX_SLOTS = 8;
constexpr int HEAD_BYTES = 2048;                    // barriers and scan scratch

struct Params {
    W4Args a;
    int kb_total;         // 256-column blocks
    int cs, rt_log2;      // cluster size; row tiles per round
    int tb;               // tokens per block, at most
    int slots;            // ring depth
    int row_rounds;       // rounds of 16 * rt rows per matrix
    int groups, group32;  // groups per row; 32-column blocks per group
    int x_vec;            // x may be read eight elements at a time
    uint32_t off_part, off_sums, off_x, off_table;  // shared-memory layout, from the aligned base
    int* err;
};

struct Cursor {  // one unit of a warp: row tile and 256-column block
    int u, kb, e, row0;
};

__device__ __forceinline__ void mma_s8s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool zero) {
    if (zero)
        asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
    else
        asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8u8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool zero) {
    if (zero)
        asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
    else
        asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}

// Eight activations k .. k + 7 of row xr as int32 (zeros past the end).
template <int L>
__device__ __forceinline__ void load8(const Params& p, int64_t xr, int64_t k, int32_t (&v)[8]) {
    const int64_t at = xr * p.a.cols + k;
    if (p.x_vec && k + 8 <= p.a.cols) {
        if (L == 1) {
            const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(p.a.x) + at);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = (int32_t)(w.x << (24 - 8 * i)) >> 24;
                v[i + 4] = (int32_t)(w.y << (24 - 8 * i)) >> 24;
            }
        } else if (L == 2) {
            const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const int16_t*>(p.a.x) + at);
            const uint32_t s[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = (int32_t)(s[i] << 16) >> 16;
                v[2 * i + 1] = (int32_t)s[i] >> 16;
            }
        } else {
            const int4 lo = *reinterpret_cast<const int4*>(static_cast<const int32_t*>(p.a.x) + at);
            const int4 hi = *reinterpret_cast<const int4*>(static_cast<const int32_t*>(p.a.x) + at + 4);
            v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
            v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = 0;
        if (k + i < p.a.cols)
            v[i] = L == 1 ? static_cast<const int8_t*>(p.a.x)[at + i]
                          : L == 2 ? static_cast<const int16_t*>(p.a.x)[at + i] : static_cast<const int32_t*>(p.a.x)[at + i];
    }
}

// L: limbs of an activation (1 = int8, 2 = int16, 4 = Q16.16).  NT: blocks of eight tokens.  PACK: all
// limbs of 8 / L tokens in one set of accumulators.  GB: 32-column blocks between two scalings.
template <int L, int NT, bool PACK, int GB>
__global__ void __launch_bounds__(THREADS, 1) kernel(const __grid_constant__ CUtensorMap tm_w, const Params p) {
    static_assert(!PACK || (NT == 1 && L > 1), "packing is for few tokens of several limbs");
    constexpr int LT = PACK ? 1 : L;      // accumulator sets between scalings
    constexpr int AC = 8 * NT;            // accumulator columns of a warp
    constexpr int TP = PACK ? 8 / L : 1;  // tokens per limb in a packed set
    constexpr int NF = 8 / GB;            // scalings per slot
    constexpr int NS = (NF + 3) / 4;      // scale registers per lane and row

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* const gbase = smem_raw + (base - raw);
    const uint32_t ring0 = base + HEAD_BYTES;
    int* const misc = reinterpret_cast<int*>(gbase + WARPS * MAX_SLOTS * 8);
    volatile int* const abort_s = misc;
    uint64_t* const part = reinterpret_cast<uint64_t*>(gbase + p.off_part);  // [warp][16][AC]
    uint64_t* const sums = reinterpret_cast<uint64_t*>(gbase + p.off_sums);  // [2][cs][outputs / cs]
    const uint32_t xs = base + p.off_x;
    int* const bound = reinterpret_cast<int*>(gbase + p.off_table);  // [experts + 1] first row of each
    int* const cumb = bound + p.a.experts + 1;                       // [experts + 1] token blocks before each

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rt = 1 << p.rt_log2, wpr = WARPS >> p.rt_log2;
    const uint32_t rank = p.cs > 1 ? cluster_ctarank() : 0u;
    const int clusters = gridDim.x / p.cs, cluster = blockIdx.x / p.cs;
    const uint32_t bars = base + warp * MAX_SLOTS * 8, slots0 = ring0 + warp * SLOT_BYTES;

    griddep_launch_dependents();
    if (lane == 0)
        for (int s = 0; s < p.slots; ++s) mbar_init(bars + 8 * s, 1);
    if (threadIdx.x == 0) {
        *abort_s = 0;
        prefetch_tensormap(&tm_w);
    }
    if (lane == 0) fence_mbar_init();
    griddep_wait();  // from here on global memory is read

    // ---- token blocks: bound = running maximum of the offsets within [0, m], cumb = running sum of
    // the blocks of at most tb rows
    {
        const int experts = (int)p.a.experts, m = (int)p.a.m;
        auto offset = [&](int e) { return p.a.offsets ? min(max(p.a.offsets[e], 0), m) : (e ? m : 0); };
        const int per = (experts + THREADS - 1) / THREADS;
        const int e0 = min((int)threadIdx.x * per, experts), e1 = min(e0 + per, experts);
        const int first = offset(0);
        int mx = first;
        for (int e = e0; e < e1; ++e) mx = max(mx, offset(e + 1));
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
            const int hi = max(lo, offset(e + 1));
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
        __syncthreads();
        if (p.cs > 1) {  // every block of the cluster is running before any writes into another
            cluster_arrive();
            cluster_wait();
        }
    }
    // Rounds (token block, 16 * rt rows) are handed out in equal runs, one run to a cluster.
    const int64_t rounds = (int64_t)cumb[p.a.experts] * p.row_rounds;
    const int u0 = (int)(rounds * cluster / clusters), u1 = (int)(rounds * (cluster + 1) / clusters);
    const int kb_lo = (int)((int64_t)p.kb_total * rank / p.cs), kb_hi = (int)((int64_t)p.kb_total * (rank + 1) / p.cs);
    const int kb_first = kb_lo + (warp >> p.rt_log2);
    const uint64_t policy = l2_policy(0);

    auto place = [&](Cursor& c) {  // expert and row tile of round c.u
        const int q = c.u / p.row_rounds;
        while (q >= cumb[c.e + 1]) ++c.e;
        c.row0 = (((c.u - q * p.row_rounds) << p.rt_log2) + (warp & (rt - 1))) * 16;
    };
    auto advance = [&](Cursor& c) {
        c.kb += wpr;
        if (c.kb >= kb_hi) {
            c.kb = kb_first;
            if (++c.u < u1) place(c);
        }
    };
    Cursor is = {kb_first < kb_hi ? u0 : u1, kb_first, 0, 0}, nx = is;
    if (is.u < u1) place(is);
    nx = is;
    int fill = 0;  // slot of the next load
    auto issue = [&]() {
        if (is.u >= u1) return;
        if (lane == 0 && !*abort_s) {
            mbar_arrive_expect_tx(bars + 8 * fill, SLOT_BYTES);
            tma_load_3d(slots0 + fill * RING_BYTES, &tm_w, bars + 8 * fill, is.kb * (KB / 2), is.row0, is.e, policy);
        }
        if (++fill == p.slots) fill = 0;
        advance(is);
    };
    for (int s = 0; s < p.slots; ++s) issue();

    // scales of a unit: lane t holds those of scalings t and t + 4, for rows g and g + 8
    int sc0[NS], sc1[NS];
    auto load_scales = [&](const Cursor& c) {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int f = t + 4 * i, gi = (c.kb * 8 + f * GB) / p.group32, r = c.row0 + g;
            const bool ok = f < NF && gi < p.groups && c.u < u1;
            const int16_t* const s = p.a.scale + ((int64_t)c.e * p.a.rows + r) * p.groups + gi;
            sc0[i] = ok && r < p.a.rows ? __ldg(s) : 0;
            sc1[i] = ok && r + 8 < p.a.rows ? __ldg(s + 8 * (int64_t)p.groups) : 0;
        }
    };
    load_scales(nx);

    const int cstride = L * p.tb * 32;  // bytes of one 32-column block of activations
    const uint32_t g7 = (uint32_t)(g & 7);
    int take = 0;
    uint32_t phase = 0;
    int block = -1, ntok = 0, p0 = 0, e_now = 0;
    bool pending = false;       // a round's sums are on their way through the cluster
    int pend_row0 = 0, pend_ntok = 0, pend_p0 = 0;
    uint32_t pend_buf = 0, buf = 0;
    const int rows_round = 16 * rt;

    auto finish_pending = [&]() {  // this block's share of the last round's outputs: add up the cluster's sums
        cluster_wait();
        const int outs = rows_round * pend_ntok;
        const int per_rank = (rows_round * p.tb + p.cs - 1) / p.cs;
        for (int i = threadIdx.x; i * p.cs + (int)rank < outs; i += THREADS) {
            const int o = i * p.cs + (int)rank, r = pend_row0 + o % rows_round, tok = o / rows_round;
            uint64_t s = 0;
            for (int c = 0; c < p.cs; ++c) s += sums[(pend_buf * p.cs + c) * per_rank + i];
            if (r < p.a.rows) p.a.y[(int64_t)(pend_p0 + tok) * p.a.rows + r] = (int32_t)((int64_t)s >> (p.a.shift + 4));
        }
        pending = false;
    };

    for (int u = u0; u < u1; ++u) {
        const int q = u / p.row_rounds;
        if (q != block) {
            // ---- a new block of tokens: its activations, as bytes in the order the MMAs take them
            block = q;
            while (q >= cumb[e_now + 1]) ++e_now;
            const int nb = cumb[e_now + 1] - cumb[e_now], i = q - cumb[e_now];
            const int64_t rows_e = bound[e_now + 1] - bound[e_now];
            p0 = bound[e_now] + (int)(rows_e * i / nb);
            ntok = bound[e_now] + (int)(rows_e * (i + 1) / nb) - p0;
            const int octs = (kb_hi - kb_lo) * (KB / 8);
            for (int tok = 0; tok < ntok; ++tok) {
                const int64_t xr = p.a.rows_of ? p.a.rows_of[p0 + tok] : p0 + tok;
                const bool inside = xr >= 0 && xr < p.a.x_rows;
                for (int o = threadIdx.x; o < octs; o += THREADS) {
                    int32_t v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                    if (inside) load8<L>(p, xr, (int64_t)kb_lo * KB + 8 * o, v);
                    const uint32_t at = xs + (o >> 2) * cstride + tok * 32 + (o & 3) * 8;
#pragma unroll
                    for (int l = 0; l < L; ++l) {
                        const uint32_t sel = l | ((l + 4) << 4);
                        const uint32_t b0 = __byte_perm(__byte_perm(v[0], v[2], sel), __byte_perm(v[4], v[6], sel), 0x5410);
                        const uint32_t b1 = __byte_perm(__byte_perm(v[1], v[3], sel), __byte_perm(v[5], v[7], sel), 0x5410);
                        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at + l * p.tb * 32), "r"(b0), "r"(b1) : "memory");
                    }
                }
            }
            __syncthreads();
        }
        // ---- this warp's units of the round
        int64_t acc64[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc64[n][i] = 0;
        // packed: column g is limb g / TP of token g % TP
        const bool col_ok = PACK ? g % TP < ntok : true;
        const bool col_top = PACK && g / TP == L - 1;
        const uint32_t xcol = xs + (PACK ? ((g / TP) * p.tb + g % TP) * 32 : g * 32) + t * 8;
        for (int kb = kb_first; kb < kb_hi; kb += wpr) {
            int s0[NS], s1[NS];
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                s0[i] = sc0[i];
                s1[i] = sc1[i];
            }
            advance(nx);
            load_scales(nx);
            if (!*abort_s) wait_bounded(bars + 8 * take, phase, abort_s, p.err, 5);
            __syncwarp();
            const uint32_t wrow = slots0 + take * RING_BYTES + g * 128 + t * 4;
            const uint32_t xblk = xcol + (kb - kb_lo) * 8 * cstride;
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const int m0 = __shfl_sync(0xffffffffu, s0[f >> 2], (lane & 28) | (f & 3));
                const int m1 = __shfl_sync(0xffffffffu, s1[f >> 2], (lane & 28) | (f & 3));
                uint32_t a[GB][4];
#pragma unroll
                for (int b = 0; b < GB; ++b) {
                    const uint32_t at = wrow + (((uint32_t)(f * GB + b) ^ g7) << 4);
                    const uint32_t w0 = lds32(at), w1 = lds32(at + 1024);
                    a[b][0] = (w0 << 4) & 0xf0f0f0f0u;
                    a[b][1] = (w1 << 4) & 0xf0f0f0f0u;
                    a[b][2] = w0 & 0xf0f0f0f0u;
                    a[b][3] = w1 & 0xf0f0f0f0u;
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (NT > 1 && n * 8 >= ntok) break;
                    int acc[LT][4];
#pragma unroll
                    for (int b = 0; b < GB; ++b) {
                        const uint32_t xb = xblk + (f * GB + b) * cstride + n * 256;
                        if (PACK) {
                            uint2 v = make_uint2(0, 0);
                            if (col_ok) v = lds64(xb);
                            mma_s8u8(acc[0], a[b], col_top ? 0u : v.x, col_top ? 0u : v.y, b == 0);
                            mma_s8s8(acc[0], a[b], col_top ? v.x : 0u, col_top ? v.y : 0u, false);
                        } else {
#pragma unroll
                            for (int l = 0; l < L; ++l) {
                                uint2 v = make_uint2(0, 0);
                                if (n * 8 + g < ntok) v = lds64(xb + l * p.tb * 32);
                                if (l < L - 1) mma_s8u8(acc[l < LT ? l : 0], a[b], v.x, v.y, b == 0);
                                else mma_s8s8(acc[l < LT ? l : 0], a[b], v.x, v.y, b == 0);
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
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
            }
            // The slot's words have been multiplied (the MMAs above took them), so it may be filled again.
            if (++take == p.slots) {
                take = 0;
                phase ^= 1u;
            }
            __syncwarp();
            issue();
        }
        // ---- partial sums of the block
        uint64_t* const mine = part + warp * 16 * AC;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                *reinterpret_cast<ulonglong2*>(mine + (g + 8 * h) * AC + n * 8 + 2 * t) =
                    make_ulonglong2((uint64_t)acc64[n][2 * h], (uint64_t)acc64[n][2 * h + 1]);
        if (pending) finish_pending();
        __syncthreads();
        const int row_first = (u - q * p.row_rounds) * rows_round;
        const int outs = rows_round * ntok;
        for (int o = threadIdx.x; o < outs; o += THREADS) {
            const int rr = o % rows_round, tok = o / rows_round;
            uint64_t s = 0;
            const uint64_t* from = part + ((rr >> 4) * 16 + (rr & 15)) * AC;
            for (int w = 0; w < wpr; ++w, from += (size_t)rt * 16 * AC) {
                if (PACK) {
#pragma unroll
                    for (int l = 0; l < L; ++l) s += from[l * TP + tok] << (8 * l);
                } else {
                    s += from[tok];
                }
            }
            if (p.cs == 1) {
                const int r = row_first + rr;
                if (r < p.a.rows) p.a.y[(int64_t)(p0 + tok) * p.a.rows + r] = (int32_t)((int64_t)s >> (p.a.shift + 4));
            } else {
                const int per_rank = (rows_round * p.tb + p.cs - 1) / p.cs;
                const uint32_t local = smem_u32(&sums[(buf * p.cs + rank) * per_rank + o / p.cs]);
                const uint32_t to = mapa(local, (uint32_t)(o % p.cs));
                asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(s) : "memory");
            }
        }
        if (p.cs > 1) {
            cluster_arrive();
            pending = true;
            pend_row0 = row_first;
            pend_ntok = ntok;
            pend_p0 = p0;
            pend_buf = buf;
            buf ^= 1u;
        }
        __syncthreads();  // the partial sums and the activations may be overwritten
    }
    if (p.cs > 1) {
        if (pending) finish_pending();
        // no block leaves while another may still write into it
        cluster_arrive();
        cluster_wait();
    }
    if (*abort_s) __nanosleep(200000);  // let copies still in flight land
}

struct Plan {
    Params p;
    int grid, smem;
};

template <int L, int NT, bool PACK, int GB>
int64_t launch(DeviceCtx* ctx, const CUtensorMap& tm, const Plan& plan) {
    auto kern = kernel<L, NT, PACK, GB>;
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
    return check_launch("gemv_w4 kernel");
}

template <int L, int NT, bool PACK>
int64_t launch_gb(DeviceCtx* ctx, const CUtensorMap& tm, const Plan& plan) {
    const int g32 = plan.p.group32;
    if (g32 % 4 == 0) return launch<L, NT, PACK, 4>(ctx, tm, plan);
    if (g32 % 2 == 0) return launch<L, NT, PACK, 2>(ctx, tm, plan);
    return launch<L, NT, PACK, 1>(ctx, tm, plan);
}

// Clusters of `cs` blocks that the device holds at once (asked once per device).
int cluster_fit(DeviceCtx* ctx, int cs);
// nt: blocks of eight tokens of the kernel; 0 = packed.
int64_t launch_i8(DeviceCtx* ctx, const CUtensorMap& tm, const Plan& plan, int nt);
int64_t launch_i16(DeviceCtx* ctx, const CUtensorMap& tm, const Plan& plan, int nt);
int64_t launch_q16(DeviceCtx* ctx, const CUtensorMap& tm, const Plan& plan, int nt);

}  // namespace w4
}  // namespace mb200
