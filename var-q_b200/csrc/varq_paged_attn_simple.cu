// Attention over a paged cache, one warp per query row: the plain form of the mathematics.
#include "varq_attn.cuh"
#include "varq_paged.cuh"

namespace varq {
namespace {

template <int D>
__global__ void __launch_bounds__(128) paged_attn_simple_kernel(PagedAttnArgs a, int* status) {
    constexpr int V = D / 32;
    const int b = blockIdx.z, i = blockIdx.x, hq = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const PagedSeq s = paged_seq(a, b, status);
    if (i >= s.nq || hq >= a.Hq) return;
    const int h = hq / a.G, page = 1 << a.c.page_shift;
    const long long qo = (long long)(s.q0 + i) * a.qs_t + hq * a.qs_h;
    float q[V], o[V], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) { q[j] = load_q_elem(a.q, a.dtype, qo + lane * V + j); o[j] = 0.f; }
    const PagedSpan sp = paged_span(a, s.kv - s.nq + i, s.kv);
    const int kw = D * a.c.kb / 32, vw = D * a.c.vb / 32;
    for (int key = 0; key < sp.hi; ++key) {
        if (key < sp.lo && key >= a.sinks) { key = sp.lo - 1; continue; }
        const int p = paged_page(a, __ldg(a.table + b * a.table_stride + (key >> a.c.page_shift)), status);
        const long long row = ((long long)p * a.c.H + h) * page + (key & (page - 1));
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int e = (lane * V + j) * a.c.kb;
            const int w = __ldg(a.c.kc + row * kw + (e >> 5));
            dot += q[j] * (float)((w << (32 - a.c.kb - (e & 31))) >> (32 - a.c.kb));
        }
#pragma unroll
        for (int z = 16; z; z >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, z);
        const float x = dot * __ldg(a.c.ks + row) * a.scale_log2, vs = __ldg(a.c.vs + row);
        const float mn = fmaxf(m, x), alpha = exp2f(m - mn), w = exp2f(x - mn);
        m = mn;
        l = l * alpha + w;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int e = (lane * V + j) * a.c.vb;
            const int c = __ldg(a.c.vc + row * vw + (e >> 5));
            o[j] = o[j] * alpha + w * vs * (float)((c << (32 - a.c.vb - (e & 31))) >> (32 - a.c.vb));
        }
    }
    const long long oo = (long long)(s.q0 + i) * a.os_t + hq * a.os_h;
    const bool any = sp.hi > 0;
#pragma unroll
    for (int j = 0; j < V; ++j) store_o_elem(a.out, a.dtype, oo + lane * V + j, any ? o[j] / l : 0.f);
    if (a.lse && lane == 0) a.lse[(long long)(s.q0 + i) * a.Hq + hq] = any ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace

int paged_attn_simple_run(const PagedAttnArgs& a, cudaStream_t st) {
    int* status = paged_status_word();
    const dim3 grid(a.max_q, (a.Hq + 3) / 4, a.B);
    if (a.c.D == 64) paged_attn_simple_kernel<64><<<grid, 128, 0, st>>>(a, status);
    else paged_attn_simple_kernel<128><<<grid, 128, 0, st>>>(a, status);
    VARQ_CUDA_TRY(cudaGetLastError());
    count_launches(1);
    return VARQ_OK;
}

}  // namespace varq
