// int8 products grouped by expert: rows [offsets[e], offsets[e+1]) of C belong to expert e,
//
//   acc    = (i32) sum_k A[row(p), k] * B[e][k, n]          row(p) = rows[p], or p without `rows`
//   C[p,n] = acc,  or  (i32)( (acc * scale[e, n]) >> shift )
//
// B is experts x K x N (N contiguous) or, transposed, experts x N x K.
#include "common.h"

namespace mb200 {
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

}  // namespace

int64_t launch_gemm_grouped_i8(DeviceCtx* ctx, const GroupedArgs& g) {
    int64_t blocks = ((g.n + 31) / 32) * ((g.m + 31) / 32);
    if (blocks > (int64_t)ctx->sm_count * 32) blocks = (int64_t)ctx->sm_count * 32;
    prof_begin(ctx);
    gemm_grouped_simt_kernel<<<(unsigned)blocks, 256, 0, ctx->stream>>>(g);
    prof_end(ctx);
    count_launch();
    return check_launch("gemm_grouped_simt_kernel");
}

}  // namespace mb200
