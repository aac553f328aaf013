// The decode kernel of a paged cache for chains of tokens, and the merge of parts that several kernels leave in the workspace.
#include "varq_paged_attn_decode.cuh"

namespace varq {
namespace {

// W warps per output row (more where there are many splits): the splits' numerators and sums, by the log-sum-exp rule, always in the same order
template <int D, int W>
__global__ void __launch_bounds__(128) paged_attn_merge_kernel(PagedAttnArgs a, int splits, const float* ws_o, const float* ws_ml) {
    constexpr int V = D / 32;
    __shared__ float part[4][D + 1];
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w0 = warp % W;
    const long long n_rows = (long long)a.T * a.Hq, row = (long long)blockIdx.x * (4 / W) + warp / W, token = row / a.Hq;
    const bool mine = row < n_rows && token >= __ldg(a.q_starts) && token < __ldg(a.q_starts + a.B);      // nobody left parts of the others
    float num[V], den = 0.f, M = -FLT_MAX;
#pragma unroll
    for (int i = 0; i < V; ++i) num[i] = 0.f;
    if (mine) {
        for (int s = lane; s < splits; s += 32) M = fmaxf(M, ws_ml[(s * n_rows + row) * 2]);
#pragma unroll
        for (int z = 16; z; z >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, z));
#pragma unroll 8
        for (int s = w0; s < splits; s += W) {
            const float2 ml = *reinterpret_cast<const float2*>(ws_ml + (s * n_rows + row) * 2);
            const float w = pd_ex2(ml.x - M);
            den = fmaf(w, ml.y, den);
            const float* o = ws_o + (s * n_rows + row) * D + lane * V;
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const float2 x = *reinterpret_cast<const float2*>(o + i);
                num[i] = fmaf(w, x.x, num[i]); num[i + 1] = fmaf(w, x.y, num[i + 1]);
            }
        }
    }
    if constexpr (W > 1) {
#pragma unroll
        for (int i = 0; i < V; ++i) part[warp][lane * V + i] = num[i];
        if (lane == 0) part[warp][D] = den;
        __syncthreads();
        if (w0) return;
#pragma unroll
        for (int w = 1; w < W; ++w) {
            den += part[warp + w][D];
#pragma unroll
            for (int i = 0; i < V; ++i) num[i] += part[warp + w][lane * V + i];
        }
    }
    if (!mine) return;
    const int head = (int)(row - token * a.Hq);
    const float inv = den != 0.f ? 1.f / den : 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) store_o_elem(a.out, a.dtype, token * a.os_t + head * a.os_h + lane * V + i, num[i] * inv);
    if (lane == 0 && a.lse) a.lse[row] = den != 0.f ? (M + __log2f(den)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace

int paged_attn_decode_run(const PagedAttnArgs& a, int rows, int splits, bool in_cluster, int tiles_per_split, float* ws_o, float* ws_ml, int* status, cudaStream_t st) {
    return launch_bits<false>(a, rows, splits, in_cluster, tiles_per_split, ws_o, ws_ml, status, st);
}

int paged_attn_merge_run(const PagedAttnArgs& a, int splits, const float* ws_o, const float* ws_ml, cudaStream_t st) {
    const int w = splits > 8 ? 4 : 1;
    const long long blocks = ((long long)a.T * a.Hq * w + 3) / 4;
    if (blocks > 0x7fffffffLL) return fail(VARQ_ERR_UNSUPPORTED, "varq_paged_attn: more than 2^31 thread blocks");
#define GO(D_, W_) if (a.c.D == D_ && w == W_) VARQ_CUDA_TRY(launch_pdl(paged_attn_merge_kernel<D_, W_>, (unsigned)blocks, 128, 0, st, 1, a, splits, ws_o, ws_ml));
    GO(64, 1) GO(64, 4) GO(128, 1) GO(128, 4)
#undef GO
    count_launches(1);
    return VARQ_OK;
}

}  // namespace varq
