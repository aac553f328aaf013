// Pages and tokens of paged caches on the move: copies of whole pages (forked sequences, compacted pools) and tokens that go to other slots (accepted
// drafts, kept tokens), for all layers in one launch: one page table serves them all, and a launch per layer would cost more than the copies.
//
// A page of a cache is four contiguous pieces (codes and scales of K and V, multiples of 64 bytes each); blocks take spans of a page's 16-byte units.
// Tokens: a block takes one group (sequence) of moves of some heads of some caches, chunk by chunk: all reads of a chunk, a barrier, all its writes.  What a later chunk
// reads no earlier one writes, because no destination is the source of a later move.
//
// What bounds them (B200): their bytes, read and written.  301 pages of 64 tokens, 8 heads x 128, 8 and 4 bits, 16 caches: 986 MB in 148 us, 6.7 TB/s, the copy rate.
// 16000 tokens of 8 sequences of 1000 to 3000 to other pages, 8 caches: 551 MB in 107 us, 5.1 TB/s; its blocks are chains of chunks, the longest of which the others wait for
// (8 times 2000 tokens: 98; in registers, one chunk after the other, 216).  Accepted paths of 64 sequences, one to six tokens, 32 caches: 10.6 us for 32 MB, chains of a launch,
// starts, slots, then three caches after one another (a block per head 31 us; per cache, in two and a half waves, 15).  Pages of four sequences, 32 caches: 5.1 us, by
// bytes 5.3 (part of it stays in L2).
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

// Block (x, y, cache): span y of page x, or, where pages are smaller than a block's units (MANY), `each` pages
template <bool MANY>
__global__ void __launch_bounds__(COPY_THREADS) paged_copy_pages_kernel(const __grid_constant__ CopyArgs a, int each) {
    pdl_trigger();
    pdl_wait();
    const CopyCache& c = a.c[blockIdx.z];
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
    auto there = [&](long long src, long long dst) { return (unsigned long long)src < (unsigned long long)c.n_pages && (unsigned long long)dst < (unsigned long long)c.n_pages; };
    if constexpr (MANY) {
        const long long first = (long long)blockIdx.x * each;
        const uint32_t here = (uint32_t)min((long long)each, a.n - first);
        uint4* to[COPY_UNITS];                         // null: nothing to copy
#pragma unroll
        for (int i = 0; i < COPY_UNITS; ++i) {
            const uint32_t v = u0 + i * COPY_THREADS, p = v / all, u = v - p * all;
            to[i] = nullptr;
            if (p < here) {
                const long long src = __ldg(a.src + first + p), dst = __ldg(a.dst + first + p);
                if (there(src, dst)) { x[i] = *at(u, src); to[i] = at(u, dst); }
            }
        }
#pragma unroll
        for (int i = 0; i < COPY_UNITS; ++i)
            if (to[i]) *to[i] = x[i];
    } else {
        const long long src = __ldg(a.src + blockIdx.x), dst = __ldg(a.dst + blockIdx.x);
        if (!there(src, dst)) return;
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
}

constexpr int MOVE_UNITS = 4, MOVE_AHEAD = 3;           // 16-byte units of a thread in a chunk; stages
template <int THREADS> constexpr int MOVE_BLOCKS = THREADS == 128 ? 7 : 3;      // on an SM
template <int THREADS> struct MoveStage {
    uint4 units[MOVE_UNITS * THREADS];
    float scales[THREADS];
    uint2 at[THREADS];                 // rows of the pools at head 0, source and destination; equal: nothing moves
};

// A block: one group, `heads` heads of `each` caches of one shape, K or V of them or both (parts).  A unit is 16 bytes of codes of a (move, head); a chunk is as many moves of a
// cache as fill the threads' units, in shared memory on its way: two chunks are being read while one is written.
template <int THREADS>
__global__ void __launch_bounds__(THREADS, MOVE_BLOCKS<THREADS>) paged_move_kernel(const __grid_constant__ CopyArgs a, int n_caches, int each, int heads, int parts, int* status) {
    extern __shared__ __align__(16) unsigned char move_smem[];
    using Stage = MoveStage<THREADS>;
    Stage* const stages = reinterpret_cast<Stage*>(move_smem);
    pdl_trigger();
    pdl_wait();
    const int first = (int)blockIdx.z * each, behind = min(first + each, n_caches);
    const CopyCache& shape = a.c[first];
    const int tid = threadIdx.x, g = blockIdx.x, h0 = ((int)blockIdx.y / parts) * heads, hn = min(heads, shape.H - h0), part = (int)blockIdx.y % parts;
    if (hn <= 0) return;
    const int s0 = __ldg(a.starts + g), s1 = __ldg(a.starts + g + 1);
    const int begin = (int)min((long long)max(s0, 0), a.n), end = (int)min((long long)max(s1, begin), a.n);
    if ((s0 != begin || s1 != end) && tid == 0) atomicCAS(status, 0, PAGED_BAD_STARTS);
    if (begin == end) return;
    const int page_mask = (1 << a.page_shift) - 1, shift = a.page_shift;
    const int kp = part == 1 ? 0 : shape.krow / 16, vp = parts == 2 && part == 0 ? 0 : shape.vrow / 16;      // units of a row
    const int per = (kp + vp) * hn, kinds = (kp > 0) + (vp > 0), rows = max(min(MOVE_UNITS * THREADS / per, THREADS / (kinds * hn)), 1);
    // this thread's units and its scale: move of the chunk (-1: none), head, piece
    int row[MOVE_UNITS], piece[MOVE_UNITS];
    uint32_t head[MOVE_UNITS];
#pragma unroll
    for (int i = 0; i < MOVE_UNITS; ++i) {
        const int u = tid + i * THREADS, r = u / per, in = u - r * per, h = in / (kp + vp);
        row[i] = r < rows ? r : -1;
        head[i] = (uint32_t)(h0 + h) << shift;
        piece[i] = in - h * (kp + vp);
    }
    const int s_r = tid / (kinds * hn), s_in = tid - s_r * (kinds * hn), s_row = s_r < rows ? s_r : -1;
    const uint32_t s_head = (uint32_t)(h0 + s_in / kinds) << shift;
    const bool s_v = kinds == 2 ? (s_in & 1) != 0 : kp == 0;
    auto unit = [&](const CopyCache& c, int i, uint32_t at) -> uint4* {
        const size_t r = (size_t)(at + head[i]);
        return piece[i] < kp ? reinterpret_cast<uint4*>(c.kc + r * c.krow) + piece[i] : reinterpret_cast<uint4*>(c.vc + r * c.vrow) + (piece[i] - kp);
    };
    auto scale = [&](const CopyCache& c, uint32_t at) -> float* { return (s_v ? c.vs : c.ks) + (at + s_head); };
    // chunks: those of a cache, then those of the next one
    struct Chunk { int cache, m; };
    auto behind_it = [&](Chunk& x) {
        if (x.m < end - rows) x.m += rows;
        else { x.m = begin; ++x.cache; }
    };
    auto slots = [&](const Chunk& x) -> uint2 {        // of move x.m + this thread's number
        if (x.cache < behind && tid < rows && x.m < end - tid) {
            const CopyCache& c = a.c[x.cache];
            const long long s = __ldg(a.src + x.m + tid), d = __ldg(a.dst + x.m + tid), n_slots = (long long)c.n_pages << shift;
            if ((unsigned long long)s < (unsigned long long)n_slots && (unsigned long long)d < (unsigned long long)n_slots)
                return make_uint2(((uint32_t)(s >> shift) * c.H << shift) + ((uint32_t)s & page_mask), ((uint32_t)(d >> shift) * c.H << shift) + ((uint32_t)d & page_mask));
        }
        return make_uint2(0u, 0u);
    };
    Chunk ahead{first, begin};                         // the next one to be read
    uint2 next = slots(ahead);
    auto copy = [&](Stage& t) {
        __syncthreads();                               // (everybody's copies of an earlier chunk are there, and) this place is written out
        if (tid < rows) t.at[tid] = next;
        const CopyCache& c = a.c[min(ahead.cache, behind - 1)];
        behind_it(ahead);
        next = slots(ahead);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MOVE_UNITS; ++i) {
            const uint2 at = row[i] < 0 ? make_uint2(0u, 0u) : t.at[row[i]];
            if (at.x != at.y)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(&t.units[tid + i * THREADS])), "l"(unit(c, i, at.x)) : "memory");
        }
        const uint2 at = s_row < 0 ? make_uint2(0u, 0u) : t.at[s_row];
        if (at.x != at.y) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(&t.scales[tid])), "l"(scale(c, at.x)) : "memory");
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll 1
    for (int i = 0; i < MOVE_AHEAD - 1; ++i) copy(stages[i]);
    int stage = 0;
#pragma unroll 1
    for (Chunk x{first, begin}; x.cache < behind; behind_it(x)) {
        Stage& t = stages[stage];
        asm volatile("cp.async.wait_group %0;" ::"n"(MOVE_AHEAD - 2) : "memory");
        copy(stages[stage == 0 ? MOVE_AHEAD - 1 : stage - 1]);
        const CopyCache& c = a.c[x.cache];
#pragma unroll
        for (int i = 0; i < MOVE_UNITS; ++i) {
            const uint2 at = row[i] < 0 ? make_uint2(0u, 0u) : t.at[row[i]];
            if (at.x != at.y) *unit(c, i, at.y) = t.units[tid + i * THREADS];
        }
        const uint2 at = s_row < 0 ? make_uint2(0u, 0u) : t.at[s_row];
        if (at.x != at.y) *scale(c, at.y) = t.scales[tid];
        stage = stage == MOVE_AHEAD - 1 ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// How moves are shared out: a block per head, K and V apart, as long as all blocks are resident at once; else, and where a group does not fill a block's units, more heads, then more
// caches of one shape.  Blocks of 128 threads, 7 on an SM / of 256, 3 on an SM, us: accepted paths as above 10.6 / 11.8, of 200 sequences, 4 heads x 64, 2 bits, 64 caches
// 18.8 / 36.1; 8 times 2000 tokens, 8 caches 98 / 109; but where few blocks are long chains, 2000 tokens of one sequence, 16 caches 54.7 / 35.7, one cache 38.6 / 22.0.
template <int THREADS>
int launch_move(const CopyArgs& a, int n, int heads, int max_moves, int* status, cudaStream_t st) {
    const long long room = (long long)MOVE_BLOCKS<THREADS> * sm_count();
    bool alike = true;
    for (int i = 1; i < n; ++i) alike = alike && a.c[i].H == a.c[0].H && a.c[i].krow == a.c[0].krow && a.c[i].vrow == a.c[0].vrow;
    int each = 1, parts = 2;
    auto blocks = [&] { return (long long)a.n_groups * ((heads + each - 1) / each) * parts * n; };
    while (each < heads && 32 * each <= MOVE_UNITS * THREADS && (blocks() > room || 32ll * each * max_moves <= MOVE_UNITS * THREADS)) { each *= 2; parts = 1; }
    const int share = !alike || blocks() <= room ? 1 : (int)(blocks() / room < n ? (blocks() + room - 1) / room : n);
    constexpr int SMEM = MOVE_AHEAD * (int)sizeof(MoveStage<THREADS>);
    static bool configured[64] = {false};
    int dev = 0;
    VARQ_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        VARQ_CUDA_TRY(cudaFuncSetAttribute(paged_move_kernel<THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    const dim3 grid((unsigned)a.n_groups, (unsigned)((heads + each - 1) / each * parts), (unsigned)((n + share - 1) / share));
    VARQ_CUDA_TRY(launch_pdl(paged_move_kernel<THREADS>, grid, THREADS, SMEM, st, 1, a, n, share, each, parts, status));
    count_launches(1);
    return VARQ_OK;
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
// all of them checked, and the first ones in `a`
int check_caches(const char* who, const varq_paged_t* caches, int n_caches, CopyArgs& a) {
    if (n_caches < 0) return fail(VARQ_ERR_ARG, "%s: %d caches", who, n_caches);
    if (n_caches && !caches) return fail(VARQ_ERR_ARG, "%s: null caches", who);
    for (int from = n_caches > 0 ? (n_caches - 1) / MOST_CACHES * MOST_CACHES : 0; from >= 0; from -= MOST_CACHES)
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
    CopyArgs a;
    if (int rc = check_caches("varq_paged_copy_pages", caches, n_caches, a)) return rc;
    if (n_pages < 0 || n_pages > 0x7fffffffLL) return fail(VARQ_ERR_ARG, "varq_paged_copy_pages: %lld pages", (long long)n_pages);
    if (n_pages == 0 || n_caches == 0) return VARQ_OK;
    if (!src_pages || !dst_pages) return fail(VARQ_ERR_ARG, "varq_paged_copy_pages: null pointer");
    if (((uintptr_t)src_pages | (uintptr_t)dst_pages) % 8) return fail(VARQ_ERR_ARG, "varq_paged_copy_pages: misaligned pointer");
    a.src = reinterpret_cast<const long long*>(src_pages); a.dst = reinterpret_cast<const long long*>(dst_pages); a.n = n_pages;
    for (int from = 0; from < n_caches; from += MOST_CACHES) {
        if (from)
            if (int rc = copy_caches("varq_paged_copy_pages", caches, n_caches, a, from)) return rc;
        const int n = n_caches - from < MOST_CACHES ? n_caches - from : MOST_CACHES;
        unsigned long long units = 0;
        for (int i = 0; i < n; ++i) {
            const unsigned long long u = ((unsigned long long)a.c[i].H << a.page_shift) * (a.c[i].krow / 16 + a.c[i].vrow / 16) + 2 * (((unsigned long long)a.c[i].H << a.page_shift) / 4);
            units = u > units ? u : units;
        }
        const unsigned long long blocks = (units + COPY_THREADS * COPY_UNITS - 1) / (COPY_THREADS * COPY_UNITS);
        if (blocks > 65535) return fail(VARQ_ERR_UNSUPPORTED, "varq_paged_copy_pages: pages of 2 GB or more");
        const int each = (int)(COPY_THREADS * COPY_UNITS / units > 1 ? COPY_THREADS * COPY_UNITS / units : 1);
        VARQ_CUDA_TRY(launch_pdl(each > 1 ? paged_copy_pages_kernel<true> : paged_copy_pages_kernel<false>, dim3((unsigned)((n_pages + each - 1) / each), (unsigned)blocks, (unsigned)n),
                                 COPY_THREADS, 0, (cudaStream_t)stream, 1, a, each));
        count_launches(1);
    }
    return VARQ_OK;
}

extern "C" int varq_paged_move_tokens(const varq_paged_t* caches, int32_t n_caches, const int64_t* src, const int64_t* dst, int64_t n_moves, const int32_t* starts,
                                      int32_t n_groups, int32_t max_moves, void* stream) {
    CopyArgs a;
    if (int rc = check_caches("varq_paged_move_tokens", caches, n_caches, a)) return rc;
    if (n_moves < 0 || n_moves > 0x7fffffffLL || n_groups < 0 || max_moves < 0) return fail(VARQ_ERR_ARG, "varq_paged_move_tokens: %lld moves, %d groups, %d at most", (long long)n_moves, n_groups, max_moves);
    if (n_moves == 0 || n_caches == 0 || n_groups == 0) return VARQ_OK;
    if (!src || !dst || !starts) return fail(VARQ_ERR_ARG, "varq_paged_move_tokens: null pointer");
    if (((uintptr_t)src | (uintptr_t)dst) % 8 || (uintptr_t)starts % 4) return fail(VARQ_ERR_ARG, "varq_paged_move_tokens: misaligned pointer");
    for (int i = 0; i < n_caches; ++i)
        for (int j = 0; j < i; ++j)
            if (caches[i].k_codes == caches[j].k_codes) return fail(VARQ_ERR_ARG, "varq_paged_move_tokens: caches %d and %d are one", j, i);      // its tokens would move twice
    a.src = reinterpret_cast<const long long*>(src); a.dst = reinterpret_cast<const long long*>(dst); a.n = n_moves; a.starts = starts; a.n_groups = n_groups;
    int* status = nullptr;
    if (int rc = paged_status_word(&status)) return rc;
    for (int from = 0; from < n_caches; from += MOST_CACHES) {
        if (from)
            if (int rc = copy_caches("varq_paged_move_tokens", caches, n_caches, a, from)) return rc;
        const int n = n_caches - from < MOST_CACHES ? n_caches - from : MOST_CACHES;
        int heads = 0;
        for (int i = 0; i < n; ++i) heads = a.c[i].H > heads ? a.c[i].H : heads;
        if (heads > 32767) return fail(VARQ_ERR_UNSUPPORTED, "varq_paged_move_tokens: %d heads (32767 at most)", heads);
        const bool few = 2ll * n_groups * heads * n <= (long long)MOVE_BLOCKS<256> * sm_count() && max_moves > 64;
        if (int rc = (few ? launch_move<256> : launch_move<128>)(a, n, heads, max_moves, status, (cudaStream_t)stream)) return rc;
    }
    return VARQ_OK;
}

extern "C" int varq_paged_tree(const int32_t* parents, const int32_t* kv_lens, const int32_t* q_starts, int32_t n_seqs, int64_t n_tokens, int32_t max_q, int32_t words,
                               int32_t* masks, int32_t* positions, void* stream) {
    if (n_seqs < 0 || n_tokens < 0 || max_q < 0 || words < 0) return fail(VARQ_ERR_ARG, "varq_paged_tree: negative size");
    if (n_tokens >= (1ll << 31) - 512 || n_seqs == 0x7fffffff)          // a block's threads step through a sequence's tokens, and one step behind them, in an int
        return fail(VARQ_ERR_UNSUPPORTED, "varq_paged_tree: 2^31 - 512 tokens or 2^31 sequences or more");
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
