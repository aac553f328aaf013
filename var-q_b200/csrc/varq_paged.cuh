// What the kernels over a paged cache share: where a token's codes lie, what a sequence holds, which keys a query sees.
#pragma once
#include "varq_common.cuh"

namespace varq {

// Division of numbers below 2^31 by one that is fixed for a launch: multiply by ceil(2^(32 + s) / d) - 2^32, add, shift (Granlund and
// Montgomery, "Division by invariant integers using multiplication").
struct FastDiv {
    uint32_t d, m, s;
    explicit FastDiv(uint32_t d_ = 1) : d(d_), s(0) {
        while ((1ull << s) < d) ++s;
        m = (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (uint32_t)(((unsigned long long)__umulhi(n, m) + n) >> s); }
};

// The pools: codes [page][head][offset][words of a row], scales [page][head][offset]
struct PagedView {
    int32_t *kc, *vc;
    float *ks, *vs;
    int n_pages, page_shift, H, D, kb, vb;
};

struct PagedAttnArgs {
    PagedView c;
    const void* q; int dtype; long long qs_t, qs_h;
    void* out; long long os_t, os_h;
    float* lse;                        // [T][Hq] or null
    const int32_t *q_starts, *kv_lens, *table;
    long long table_stride; int table_pages;
    int B, T, Hq, G;                   // sequences, query tokens of all of them, query heads, query heads per head of the cache
    int max_q, max_kv;
    float scale_log2;                  // softmax_scale * log2(e)
    int causal, window, sinks;         // window 0: none
};

constexpr int PAGED_MOST_KEYS = 0x7fffffff - 4095;      // tokens of a sequence: the numbers of the keys that a warp asks for next, 32 x 64 of them, stay below 2^31

// First thing that was wrong with numbers that only the device sees (lengths, starts, page numbers): the access is clamped into the
// tensors' bounds and the code is kept for varq_device_status.
enum PagedStatus : int { PAGED_BAD_STARTS = 64, PAGED_BAD_LENGTH = 65, PAGED_BAD_PAGE = 66 };
int paged_status_word(int** out);      // its device address
int paged_status(int* out);            // its value where *out is 0; clears it

// Sequence b: its first query token, number of queries, tokens in the cache, query token behind its last one
struct PagedSeq { int q0, nq, kv, end; };
__device__ __forceinline__ PagedSeq paged_seq(const PagedAttnArgs& a, int b, int* status) {
    const int s0 = __ldg(a.q_starts + b), s1 = __ldg(a.q_starts + b + 1), kv = __ldg(a.kv_lens + b);
    PagedSeq s;
    s.q0 = min(max(s0, 0), a.T);
    s.end = min(max(s1, s.q0), a.T);
    s.nq = min(s.end - s.q0, a.max_q);
    s.kv = (int)min((long long)min(max(kv, 0), PAGED_MOST_KEYS), (long long)a.table_pages << a.c.page_shift);
    if (s.q0 != s0 || s.nq != s1 - s0) atomicCAS(status, 0, PAGED_BAD_STARTS);
    if (s.kv != kv) atomicCAS(status, 0, PAGED_BAD_LENGTH);
    return s;
}
__device__ __forceinline__ int paged_page(const PagedAttnArgs& a, int p, int* status) {
    if ((unsigned)p < (unsigned)a.c.n_pages) return p;
    atomicCAS(status, 0, PAGED_BAD_PAGE);
    return 0;
}

// First key of the window of a query at position p, max(p - window + 1, 0), with no number outside an int on the way (p may be negative)
__device__ __forceinline__ int paged_window(const PagedAttnArgs& a, int p) { return a.window ? max(p, a.window - 1) - (a.window - 1) : 0; }
// Keys that a query at position p sees: [0, min(sinks, hi)) and [lo, hi); none where hi <= 0
struct PagedSpan { int lo, hi; };
__device__ __forceinline__ PagedSpan paged_span(const PagedAttnArgs& a, int p, int kv) {
    PagedSpan s;
    s.hi = a.causal ? min(p + 1, kv) : kv;
    s.lo = paged_window(a, p);
    return s;
}

// Query rows in front of the first sequence's and behind the last one's belong to no sequence.  They get zeros and -inf, as rows that see nothing: from the CTAs of
// those two sequences, each thread (number `i` of `step`) a share of the rows of its head of the cache.
struct PagedPad { unsigned short* out; long long os_t, os_h; float* lse; int D, G, Hq, h, front, behind, T; };
__device__ __forceinline__ bool paged_pad_any(const PagedAttnArgs& a, const PagedSeq& seq, int b) { return (b == 0 && seq.q0 > 0) || (b == a.B - 1 && seq.end < a.T); }
__device__ __forceinline__ PagedPad paged_pad_rows(const PagedAttnArgs& a, const PagedSeq& seq, int b, int h) {
    return {reinterpret_cast<unsigned short*>(a.out), a.os_t, a.os_h, a.lse, a.c.D, a.G, a.Hq, h, b == 0 ? seq.q0 : 0, b == a.B - 1 ? seq.end : a.T, a.T};
}
__device__ __forceinline__ void paged_pad(const PagedPad p, long long i, long long step) {
    const int chunks = p.D / 8;
    for (const long long n = (long long)(p.front + p.T - p.behind) * p.G * chunks; i < n; i += step) {
        const long long row = i / chunks, at = row / p.G, token = at < p.front ? at : at - p.front + p.behind;
        const int c = (int)(i - row * chunks), head = p.h * p.G + (int)(row % p.G);
        unsigned short* o = p.out + token * p.os_t + head * p.os_h + 8 * c;
        if ((reinterpret_cast<uintptr_t>(o) & 15u) == 0) *reinterpret_cast<uint4*>(o) = make_uint4(0, 0, 0, 0);
        else
            for (int e = 0; e < 8; ++e) o[e] = 0;
        if (c == 0 && p.lse) p.lse[token * p.Hq + head] = -INFINITY;
    }
}

// What the V scale of a key puts into the exponent, and the factor that takes it out of the sum again: log2 of it, 1 / it.  A scale below 2^-100, 0 among them,
// counts as 2^-100: the key keeps its weight, its value is as good as zero.  One that is no size of values (NaN, infinite, negative) spoils the rows that see
// it and no other: the inverse is finite whatever lies there, and a key that is not seen has weight 0, which times its inverse has to be 0.
__device__ __forceinline__ float paged_exponent(float scale) {
    float y;
    asm("{\n\t.reg .f32 t;\n\tlg2.approx.ftz.f32 t, %1;\n\tmax.NaN.f32 %0, t, %2;\n\t}" : "=f"(y) : "f"(scale), "f"(-100.f));
    return y;
}
__device__ __forceinline__ float paged_inverse(float scale) {      // above 2^126 it is subnormal, which the reciprocal alone (and __fdividef) would flush
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaxf(scale, 0x1p-100f) * 0.25f));
    return r * 0.25f;
}

// Where a row's reference lies: its largest weight times V scale is held as 2^PAGED_SET when the reference is set or raised, and the reference is raised when one
// passes 2^PAGED_TOP.  fp16 ends at 2^16, its normal numbers at 2^-14: what is 2^-21 of the largest or more is rounded by itself, what is less by 2^-32 of the largest.
// (With the largest held as 1 to 2^8, one V row 2^13 times the others', at 2^13 times their weight, took the others out of all columns in which its codes are zero.)
// 8 between the two: raising costs the chunk kernel a tile, and with less of it happens more than once or twice in a long row.
constexpr float PAGED_SET = 7.f, PAGED_TOP = 15.f;

constexpr int PAGED_CLUSTER = 8;       // up to so many parts of the decode kernel can meet in a cluster, without a workspace
// Parts of the key range (splits) leave numerators ws_o [split][query row][D] and (reference, sum) ws_ml [split][query row][2]; a second launch merges them
int paged_attn_tc_run(const PagedAttnArgs& a, int splits, float* ws_o, float* ws_ml, int* status, cudaStream_t st);
// rows: query rows of a CTA, 8, 16 or 24
int paged_attn_decode_run(const PagedAttnArgs& a, int rows, int splits, bool in_cluster, int tiles_per_split, float* ws_o, float* ws_ml, int* status, cudaStream_t st);
int paged_attn_merge_run(const PagedAttnArgs& a, int splits, const float* ws_o, const float* ws_ml, cudaStream_t st);
int paged_attn_tc_status(int* out);
int forced_attn_path();                // varq_attn_force_path

}  // namespace varq
