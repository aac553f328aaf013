// Pages and tokens of paged caches on the move: copies of whole pages (forked sequences, compacted pools) and tokens that go to other slots (accepted
// drafts, kept tokens), for all layers in one launch: one page table serves them all, and a launch per layer would cost more than the copies.
//
// A page of a cache is four contiguous pieces (codes and scales of K and V, multiples of 64 bytes each); blocks take spans of a page's 16-byte units.
// Tokens: a block takes one group (sequence) of moves of one head of one cache, chunk by chunk: all reads of a chunk, a barrier, all its writes.  What a later chunk reads
// no earlier one writes, because no destination is the source of a later move.
#include "varq_paged.cuh"

namespace varq {
namespace {

struct CopyCache {
    unsigned char *kc, *vc;
    float *ks, *vs;
    int n_pages, H;
    int krow, vrow;                    // bytes of a row of codes
};
constexpr int MOST_CACHES = 64;        // of a launch: their descriptors are its parameters
struct CopyArgs {
    CopyCache c[MOST_CACHES];
    const long long *src, *dst;
    long long n;
    int page_shift;
    const int32_t* starts;
    int n_groups;
};

constexpr int COPY_THREADS = 256, COPY_UNITS = 8;      // 16-byte units of a thread

__global__ void __launch_bounds__(COPY_THREADS) paged_copy_pages_kernel(const __grid_constant__ CopyArgs a) {
    pdl_trigger();
    pdl_wait();
    const CopyCache& c = a.c[blockIdx.z];
    const long long src = __ldg(a.src + blockIdx.x), dst = __ldg(a.dst + blockIdx.x);
    if ((unsigned long long)src >= (unsigned long long)c.n_pages || (unsigned long long)dst >= (unsigned long long)c.n_pages) return;
    const uint32_t tokens = (uint32_t)c.H << a.page_shift, ku = tokens * (c.krow / 16), vu = tokens * (c.vrow / 16), su = tokens / 4, all = ku + vu + 2 * su;
    const uint32_t u0 = blockIdx.y * (COPY_THREADS * COPY_UNITS) + threadIdx.x;
    uint4 x[COPY_UNITS];
    auto at = [&](uint32_t u, long long page) -> uint4* {
        if (u < ku) return reinterpret_cast<uint4*>(c.kc) + (size_t)page * ku + u;
        u -= ku;
        if (u < vu) return reinterpret_cast<uint4*>(c.vc) + (size_t)page * vu + u;
        u -= vu;
        if (u < su) return reinterpret_cast<uint4*>(c.ks) + (size_t)page * su + u;
        return reinterpret_cast<uint4*>(c.vs) + (size_t)page * su + (u - su);
    };
#pragma unroll
    for (int i = 0; i < COPY_UNITS; ++i) {
        const uint32_t u = u0 + i * COPY_THREADS;
        if (u < all) x[i] = *at(u, src);
    }
#pragma unroll
    for (int i = 0; i < COPY_UNITS; ++i) {
        const uint32_t u = u0 + i * COPY_THREADS;
        if (u < all) *at(u, dst) = x[i];
    }
}

constexpr int MOVE_THREADS = 256, MOVE_ROWS = 64;      // moves of a chunk

__global__ void __launch_bounds__(MOVE_THREADS) paged_move_kernel(const __grid_constant__ CopyArgs a, int* status) {
    __shared__ long long s_at[2][MOVE_ROWS];           // rows of the pools, source and destination, -1: nothing moves
    pdl_trigger();
    pdl_wait();
    const CopyCache& c = a.c[blockIdx.z];
    const int g = blockIdx.x, h = blockIdx.y;
    if (h >= c.H) return;
    const int s0 = __ldg(a.starts + g), s1 = __ldg(a.starts + g + 1);
    const int begin = (int)min((long long)max(s0, 0), a.n), end = (int)min((long long)max(s1, begin), a.n);
    if ((s0 != begin || s1 != end) && threadIdx.x == 0) atomicCAS(status, 0, PAGED_BAD_STARTS);
    const long long n_slots = (long long)c.n_pages << a.page_shift;
    const int page_mask = (1 << a.page_shift) - 1;
    const int kp = c.krow / 16, vp = c.vrow / 16, pieces = kp + vp;                  // 16-byte pieces of a token's codes
    constexpr int U = MOVE_ROWS * 16 / MOVE_THREADS;   // of a thread, at most: 8 pieces of K and of V
    for (int m0 = begin; m0 < end; m0 += MOVE_ROWS) {
        const int n = min(MOVE_ROWS, end - m0);
        __syncthreads();
        if (threadIdx.x < MOVE_ROWS) {
            long long r[2] = {-1, -1};
            if (threadIdx.x < n) {
                const long long s = __ldg(a.src + m0 + threadIdx.x), d = __ldg(a.dst + m0 + threadIdx.x);
                if ((unsigned long long)s < (unsigned long long)n_slots && (unsigned long long)d < (unsigned long long)n_slots && s != d) {
                    r[0] = (((s >> a.page_shift) * c.H + h) << a.page_shift) + (s & page_mask);
                    r[1] = (((d >> a.page_shift) * c.H + h) << a.page_shift) + (d & page_mask);
                }
            }
            s_at[0][threadIdx.x] = r[0]; s_at[1][threadIdx.x] = r[1];
        }
        __syncthreads();
        uint4 x[U];
        float sc = 0.f;
        const int srow = threadIdx.x >> 1;             // scale of K (even threads) or V
        auto at = [&](int u, int which) -> uint4* {    // unit u of the chunk, in its source (0) or destination (1)
            const int row = u / pieces, p = u - row * pieces;
            const long long r = s_at[which][row];
            return p < kp ? reinterpret_cast<uint4*>(c.kc + r * c.krow) + p : reinterpret_cast<uint4*>(c.vc + r * c.vrow) + (p - kp);
        };
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = threadIdx.x + i * MOVE_THREADS;
            if (u < n * pieces && s_at[0][u / pieces] >= 0) x[i] = *at(u, 0);
        }
        if (srow < n && s_at[0][srow] >= 0) sc = (threadIdx.x & 1 ? c.vs : c.ks)[s_at[0][srow]];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = threadIdx.x + i * MOVE_THREADS;
            if (u < n * pieces && s_at[0][u / pieces] >= 0) *at(u, 1) = x[i];
        }
        if (srow < n && s_at[0][srow] >= 0) (threadIdx.x & 1 ? c.vs : c.ks)[s_at[1][srow]] = sc;
    }
}

int copy_caches(const char* who, const varq_paged_t* caches, int n_caches, CopyArgs& a, int from) {
    const int n = n_caches - from < MOST_CACHES ? n_caches - from : MOST_CACHES;
    for (int i = 0; i < n; ++i) {
        PagedView v;
        if (int rc = paged_check_cache(who, caches + from + i, v)) return rc;
        if (caches[from + i].page_size != caches[0].page_size) return fail(VARQ_ERR_ARG, "%s: caches with pages of %d and %d tokens", who, caches[0].page_size, caches[from + i].page_size);
        a.page_shift = v.page_shift;
        a.c[i] = {reinterpret_cast<unsigned char*>(v.kc), reinterpret_cast<unsigned char*>(v.vc), v.ks, v.vs, v.n_pages, v.H, v.D * v.kb / 8, v.D * v.vb / 8};
    }
    return VARQ_OK;
}
int check_caches(const char* who, const varq_paged_t* caches, int n_caches, CopyArgs& a) {
    if (n_caches < 0) return fail(VARQ_ERR_ARG, "%s: %d caches", who, n_caches);
    if (n_caches && !caches) return fail(VARQ_ERR_ARG, "%s: null caches", who);
    for (int from = 0; from < n_caches; from += MOST_CACHES)
        if (int rc = copy_caches(who, caches, n_caches, a, from)) return rc;
    return VARQ_OK;
}

struct TreeArgs {
    const int32_t *parents, *kv_lens, *q_starts;
    int32_t *masks, *positions;
    int B, T, max_q, words;
};
constexpr int TREE_THREADS = 128;

// A token's mask: up the tree from it, word by word as the numbers fall (parents have smaller ones).  Block b: sequence b; the last one: rows of no sequence.
__global__ void __launch_bounds__(TREE_THREADS) paged_tree_kernel(TreeArgs a, int* status) {
    pdl_trigger();
    pdl_wait();
    const int b = blockIdx.x;
    if (b == a.B) {
        const int front = min(max(__ldg(a.q_starts), 0), a.T), behind = min(max(__ldg(a.q_starts + a.B), front), a.T);
        for (long long i = threadIdx.x; i < (long long)(front + a.T - behind) * (a.words + 1); i += TREE_THREADS) {
            const long long row = i / (a.words + 1), w = i - row * (a.words + 1), t = row < front ? row : row - front + behind;
            if (w < a.words) a.masks[t * a.words + w] = 0;
            else a.positions[t] = 0;
        }
        return;
    }
    const int s0 = __ldg(a.q_starts + b), s1 = __ldg(a.q_starts + b + 1), kv = __ldg(a.kv_lens + b);
    const int q0 = min(max(s0, 0), a.T), end = min(max(s1, q0), a.T), n = min(end - q0, a.max_q);
    if ((q0 != s0 || n != s1 - s0) && threadIdx.x == 0) atomicCAS(status, 0, PAGED_BAD_STARTS);
    for (int i = threadIdx.x; i < end - q0; i += TREE_THREADS) {
        int32_t* row = a.masks + (long long)(q0 + i) * a.words;
        int at = i < n ? i : -1, depth = -1;
        for (int w = a.words - 1; w >= 0; --w) {
            uint32_t bits = 0;
            while (at >= 32 * w && at >= 0) {
                bits |= 1u << (at & 31);
                ++depth;
                int p = __ldg(a.parents + q0 + at);
                if (p >= at || p < -1) { atomicCAS(status, 0, PAGED_BAD_PARENT); p = -1; }
                at = p;
            }
            row[w] = (int32_t)bits;
        }
        a.positions[q0 + i] = i < n ? kv - n + depth : 0;
    }
}

}  // namespace
}  // namespace varq

using namespace varq;

extern "C" int varq_paged_copy_pages(const varq_paged_t* caches, int32_t n_caches, const int64_t* src_pages, const int64_t* dst_pages, int64_t n_pages, void* stream) {
    CopyArgs a{};
    if (int rc = check_caches("varq_paged_copy_pages", caches, n_caches, a)) return rc;
    if (n_pages < 0 || n_pages > 0x7fffffffLL) return fail(VARQ_ERR_ARG, "varq_paged_copy_pages: %lld pages", (long long)n_pages);
    if (n_pages == 0 || n_caches == 0) return VARQ_OK;
    if (!src_pages || !dst_pages) return fail(VARQ_ERR_ARG, "varq_paged_copy_pages: null pointer");
    if (((uintptr_t)src_pages | (uintptr_t)dst_pages) % 8) return fail(VARQ_ERR_ARG, "varq_paged_copy_pages: misaligned pointer");
    a.src = reinterpret_cast<const long long*>(src_pages); a.dst = reinterpret_cast<const long long*>(dst_pages); a.n = n_pages;
    for (int from = 0; from < n_caches; from += MOST_CACHES) {
        if (int rc = copy_caches("varq_paged_copy_pages", caches, n_caches, a, from)) return rc;
        const int n = n_caches - from < MOST_CACHES ? n_caches - from : MOST_CACHES;
        unsigned long long units = 0;
        for (int i = 0; i < n; ++i) {
            const unsigned long long u = ((unsigned long long)a.c[i].H << a.page_shift) * (a.c[i].krow / 16 + a.c[i].vrow / 16) + 2 * (((unsigned long long)a.c[i].H << a.page_shift) / 4);
            units = u > units ? u : units;
        }
        const unsigned long long blocks = (units + COPY_THREADS * COPY_UNITS - 1) / (COPY_THREADS * COPY_UNITS);
        if (blocks > 65535) return fail(VARQ_ERR_UNSUPPORTED, "varq_paged_copy_pages: pages of 2 GB or more");
        VARQ_CUDA_TRY(launch_pdl(paged_copy_pages_kernel, dim3((unsigned)n_pages, (unsigned)blocks, (unsigned)n), COPY_THREADS, 0, (cudaStream_t)stream, 1, a));
        count_launches(1);
    }
    return VARQ_OK;
}

extern "C" int varq_paged_move_tokens(const varq_paged_t* caches, int32_t n_caches, const int64_t* src, const int64_t* dst, int64_t n_moves, const int32_t* starts,
                                      int32_t n_groups, int32_t max_moves, void* stream) {
    CopyArgs a{};
    if (int rc = check_caches("varq_paged_move_tokens", caches, n_caches, a)) return rc;
    if (n_moves < 0 || n_moves > 0x7fffffffLL || n_groups < 0 || max_moves < 0) return fail(VARQ_ERR_ARG, "varq_paged_move_tokens: %lld moves, %d groups, %d at most", (long long)n_moves, n_groups, max_moves);
    if (n_moves == 0 || n_caches == 0 || n_groups == 0) return VARQ_OK;
    if (!src || !dst || !starts) return fail(VARQ_ERR_ARG, "varq_paged_move_tokens: null pointer");
    if (((uintptr_t)src | (uintptr_t)dst) % 8 || (uintptr_t)starts % 4) return fail(VARQ_ERR_ARG, "varq_paged_move_tokens: misaligned pointer");
    a.src = reinterpret_cast<const long long*>(src); a.dst = reinterpret_cast<const long long*>(dst); a.n = n_moves; a.starts = starts; a.n_groups = n_groups;
    int* status = nullptr;
    if (int rc = paged_status_word(&status)) return rc;
    for (int from = 0; from < n_caches; from += MOST_CACHES) {
        if (int rc = copy_caches("varq_paged_move_tokens", caches, n_caches, a, from)) return rc;
        const int n = n_caches - from < MOST_CACHES ? n_caches - from : MOST_CACHES;
        int heads = 0;
        for (int i = 0; i < n; ++i) heads = a.c[i].H > heads ? a.c[i].H : heads;
        if (heads > 65535) return fail(VARQ_ERR_UNSUPPORTED, "varq_paged_move_tokens: %d heads (65535 at most)", heads);
        VARQ_CUDA_TRY(launch_pdl(paged_move_kernel, dim3((unsigned)n_groups, (unsigned)heads, (unsigned)n), MOVE_THREADS, 0, (cudaStream_t)stream, 1, a, status));
        count_launches(1);
    }
    return VARQ_OK;
}

extern "C" int varq_paged_tree(const int32_t* parents, const int32_t* kv_lens, const int32_t* q_starts, int32_t n_seqs, int64_t n_tokens, int32_t max_q, int32_t words,
                               int32_t* masks, int32_t* positions, void* stream) {
    if (n_seqs < 0 || n_tokens < 0 || max_q < 0 || words < 0) return fail(VARQ_ERR_ARG, "varq_paged_tree: negative size");
    if (n_tokens > 0x7fffffffLL || n_seqs == 0x7fffffff) return fail(VARQ_ERR_UNSUPPORTED, "varq_paged_tree: 2^31 tokens or sequences or more");
    if (words > (1 << 26) || (long long)words * 32 < max_q) return fail(VARQ_ERR_ARG, "varq_paged_tree: %d words for %d tokens of a sequence", words, max_q);
    if (n_tokens == 0) return VARQ_OK;
    if (!parents || !q_starts || !positions || (words && !masks) || (n_seqs && !kv_lens)) return fail(VARQ_ERR_ARG, "varq_paged_tree: null pointer");
    if (((uintptr_t)parents | (uintptr_t)kv_lens | (uintptr_t)q_starts | (uintptr_t)masks | (uintptr_t)positions) % 4) return fail(VARQ_ERR_ARG, "varq_paged_tree: misaligned pointer");
    TreeArgs a{parents, kv_lens, q_starts, masks, positions, n_seqs, (int)n_tokens, max_q, words};
    int* status = nullptr;
    if (int rc = paged_status_word(&status)) return rc;
    VARQ_CUDA_TRY(launch_pdl(paged_tree_kernel, (unsigned)n_seqs + 1u, TREE_THREADS, 0, (cudaStream_t)stream, 1, a, status));
    count_launches(1);
    return VARQ_OK;
}
