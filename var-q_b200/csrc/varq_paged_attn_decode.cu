// Attention of a few query rows (8, 16 or 24 per CTA) over a paged cache: warp-level tensor-core instructions fed straight from the pages.
//
// The work is to stream the codes once, so the kernel is built around instructions per key and bytes in flight.  A warp takes 16 keys at a time, which lie
// in one page, 16 rows one behind the other: its lanes copy them (cp.async, 16 bytes each) to a ring of its own in shared memory, several tiles ahead.  The
// 16-byte chunks of a row are permuted by the row's number, so that the fragments below come out without bank conflicts.
// mma.sync m16n8k16 takes the codes as its A operand, and every thread unpacks whole words:
//   S^T = K Q^T     thread (g, c) (g = lane / 4, c = lane % 4) holds keys g and g + 8 and a quarter of the head_dim, contiguous in memory (the order
//                   of the contraction index is free as long as Q follows it); the eight columns are query rows (token, head of the group);
//   O^T = V^T P^T   thread (g, c) holds an eighth of the head_dim of keys 2c, 2c + 1, 2c + 8, 2c + 9; pairs of keys are joined by byte
//                   permutes, and P^T is the transpose of S^T's fragment (movmatrix).
// As in the chunk kernel the V scale goes into the exponent: x = S * (K scale * factor of the row) + log2(V scale), P = 2^(x - m) in fp16,
// l += P / V scale in fp32; the reference m is set 7 below the largest x and raised only when an x passes it by more than 15.  What is held in fewer than 32 bits:
// P, the operand of a 16-bit product (weight times V scale of 2^-21 of the row's largest or more is rounded by itself, 2^-12 of it, a smaller one by 2^-32 of the
// largest), and the queries, fp16 times a power of two per row: exact but for elements below 2^-22 of the row's largest, which are off by 2^-33 of it at most.
// Warps and CTAs (key ranges) are merged by the log-sum-exp rule: where all CTAs are resident at once, up to eight of a row tile are a cluster and read one
// another's shared memory; else they leave parts in the workspace for a second launch.
//
// What bounds it (B200): no unit is full.  64 sequences of 2000 to 10520 keys, 16 heads x 128, 4 bits: 239 us, 3.9 TB/s, DRAM 47 % busy (its bytes alone take 142 us).  Its
// instructions, 365 per 16 keys and warp, about half of them the conversion of the codes, would fill a scheduler for some 140 us; it issues in 65 % of the cycles
// in which it has warps: four of them, each a chain of products, exponentials and unpacking.  Lengths that differ and parts cut by the longest leave an SM without warps for
// another 6 % of the time.  One sequence of 1000 keys, 8 heads: 7.4 us, a chain of latencies (launch, lengths, pages, rows, two products, the cluster's merge).  Four tokens
// over a window of 1024 (20 rows of a head) on 24 sequences: 31 us.  With rows straight from the pages into registers, a tile ahead, instead of the ring: 290 us.
#include <cooperative_groups.h>

#include <cfloat>
#include <type_traits>

#include "varq_attn.cuh"
#include "varq_codes.cuh"
#include "varq_paged.cuh"

namespace varq {
namespace {

constexpr int PD_WARPS = 4, PD_KEYS = 16;

__device__ __forceinline__ void pd_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pd_transpose(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float pd_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <int BITS> __host__ __device__ constexpr uint32_t pd_neg_base(int cls) {      // fp16 pairs of -(1024 / 2^p + bias), by class of bit position
    return BITS == 8 ? 0xE480E480u : BITS == 4 ? (cls == 0 ? 0xE408E408u : 0xD480D480u)
                                               : (cls == 0 ? 0xE402E402u : cls == 1 ? 0xDC08DC08u : cls == 2 ? 0xD420D420u : 0xCC80CC80u);
}
template <int BITS> __device__ __forceinline__ void pd_codes(const uint32_t* w, uint32_t (&h)[8], const CodeMagic<BITS>& cm) {
    Item<BITS>::raw(w, h, cm);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = Item<BITS>::minus_zp(h[i], i, pd_neg_base<BITS>(i % Item<BITS>::CLS));
}
template <int BYTES> struct PdRaw {        // `BYTES` of a row in shared memory (two bytes: the low half of one word)
    static constexpr int NW = BYTES < 4 ? 1 : BYTES / 4;
    uint32_t w[NW];
};
// A tile of 16 rows of RB bytes in shared memory: chunk of 16 bytes `ch` of row `r`
template <int RB> __device__ __forceinline__ int pd_chunk(int r, int ch) { return r * RB + ((RB == 128 ? ch ^ (r & 7) : RB == 64 ? ch ^ ((r >> 1) & 3) : ch) << 4); }
template <int RB, int BYTES> __device__ __forceinline__ void pd_read(PdRaw<BYTES>& o, const unsigned char* tile, int r, int part) {      // part: in units of BYTES
    if constexpr (BYTES == 32) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 v = *reinterpret_cast<const uint4*>(tile + pd_chunk<RB>(r, 2 * part + i));
            o.w[4 * i] = v.x; o.w[4 * i + 1] = v.y; o.w[4 * i + 2] = v.z; o.w[4 * i + 3] = v.w;
        }
    } else {
        const unsigned char* p = tile + pd_chunk<RB>(r, part * BYTES / 16) + (part * BYTES & 15);
        if constexpr (BYTES == 16) { const uint4 v = *reinterpret_cast<const uint4*>(p); o.w[0] = v.x; o.w[1] = v.y; o.w[2] = v.z; o.w[3] = v.w; }
        else if constexpr (BYTES == 8) { const uint2 v = *reinterpret_cast<const uint2*>(p); o.w[0] = v.x; o.w[1] = v.y; }
        else if constexpr (BYTES == 4) o.w[0] = *reinterpret_cast<const uint32_t*>(p);
        else o.w[0] = *reinterpret_cast<const unsigned short*>(p);
    }
}
template <int RB> __device__ __forceinline__ void pd_copy(unsigned char* tile, const unsigned char* src, int lane) {      // 16 rows, contiguous in memory
#pragma unroll
    for (int i = 0; i < (RB + 31) / 32; ++i) {
        const int ch = lane + 32 * i;                       // of 16 * RB / 16 = RB
        if (RB >= 32 || ch < RB)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(tile + pd_chunk<RB>(ch / (RB / 16), ch % (RB / 16)))), "l"(src + ch * 16) : "memory");
    }
}
template <int KB, int VB, int D> struct PdPlan {
    static constexpr int KROW = D * KB / 8, VROW = D * VB / 8, TILE = 16 * (KROW + VROW) + 128;      // rows, then 16 scales of K and of V
    // Some ten KB a warp, which leaves room for as many CTAs on an SM as its registers allow
    static constexpr int ST = TILE > 3000 ? 4 : TILE > 1500 ? 5 : 6;                                 // tiles of a warp's ring
    static constexpr int SMEM = PD_WARPS * ST * TILE;
};
// the words of two keys -> words that unpack to pairs (first key, second key) of one head_dim element each, in element order
template <int BITS, int NW> __device__ __forceinline__ void pd_join(const uint32_t (&a)[NW], const uint32_t (&b)[NW], uint32_t (&o)[2 * NW]) {
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        o[2 * i] = __byte_perm(a[i], b[i], BITS == 8 ? 0x5140 : 0x5410);
        o[2 * i + 1] = __byte_perm(a[i], b[i], BITS == 8 ? 0x7362 : 0x7632);
    }
}

// A call, and behind the keys' loop: inlined in front of it, it took 1.3 % of a long call
__device__ __noinline__ void pd_pad(PagedPad p, long long i, long long step) { paged_pad(p, i, step); }

template <int KB, int VB, int D, int NT>
__global__ void __launch_bounds__(PD_WARPS * 32, NT > 2 ? (D == 128 ? 2 : 3) : NT > 1 ? (D == 128 ? 3 : 4) : D == 128 ? (KB == 8 && VB == 8 ? 3 : 4) : 5)
paged_attn_decode_kernel(PagedAttnArgs a, int n_rowtiles, int splits, int in_cluster, int tiles_per_split, float* ws_o, float* ws_ml, int* status) {
    using P = PdPlan<KB, VB, D>;
    constexpr int KBYTES = D / 4 * KB / 8, VBYTES = D / 8 * VB / 8;       // of a row and thread
    constexpr int KROW = P::KROW, VROW = P::VROW, ST = P::ST;
    constexpr int ITEMS = D / 64, KSTEPS = D / 16, MT = D / 16, ROWS = 8 * NT;
    extern __shared__ __align__(128) unsigned char pd_smem[];
    float (*s_part)[ROWS][D + 2] = reinterpret_cast<float (*)[ROWS][D + 2]>(pd_smem);      // behind the last use of the rings

    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    const int split = (int)(blockIdx.x % (unsigned)splits);
    const unsigned item = blockIdx.x / (unsigned)splits;
    const int rt = (int)(item % (unsigned)n_rowtiles), bh = (int)(item / (unsigned)n_rowtiles), b = bh / a.c.H, h = bh - b * a.c.H;
    const PagedSeq seq = paged_seq(a, b, status);
    const int rows = seq.nq * a.G, row0 = rt * ROWS, p_first = seq.kv - seq.nq;
    if (row0 >= rows && !paged_pad_any(a, seq, b)) return;

    // ---- the 16-key tiles: first tokens, then the window (or everything)
    const int t0 = row0 / a.G, t1 = (min(row0 + ROWS, rows) - 1) / a.G;
    const int hi = max(a.causal ? min(seq.kv, p_first + t1 + 1) : seq.kv, 0), lo = paged_window(a, p_first + t0) & ~(PD_KEYS - 1);
    const int ns = min((a.sinks + PD_KEYS - 1) / PD_KEYS, lo / PD_KEYS), n_tiles = hi > 0 && row0 < rows ? ns + (max(hi - lo, 0) + PD_KEYS - 1) / PD_KEYS : 0;
    const int begin = (int)min((long long)split * tiles_per_split, (long long)n_tiles), end = split == splits - 1 ? n_tiles : min(begin + tiles_per_split, n_tiles);
    const int all_hi = a.causal ? min(p_first + t0 + 1, seq.kv) : seq.kv, all_lo = paged_window(a, p_first + t1);      // what every row sees
    auto key_of = [&](int i) { return i < ns ? i * PD_KEYS : lo + (i - ns) * PD_KEYS; };

    // ---- Q fragments: column g is row t * 8 + g, scaled by a power of two to use fp16's range
    uint32_t qf[NT][KSTEPS][2];
    float qfac[NT][2];                 // of this thread's two score columns: softmax scale in the log2 domain / power of two
    int col_hi[NT][2], col_lo[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float v[D / 4], mx = 0.f;
        const int row = row0 + t * 8 + g, token = row / a.G, head = h * a.G + row - token * a.G;
#pragma unroll
        for (int j = 0; j < D / 4; j += 8) {
            float e[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (row < rows) load_q8(a.q, a.dtype, (long long)(seq.q0 + token) * a.qs_t + head * a.qs_h + c * (D / 4) + j, e);
#pragma unroll
            for (int i = 0; i < 8; ++i) { v[j + i] = e[i]; mx = fmaxf(mx, fabsf(e[i])); }
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1)); mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // 2^(8 - exponent of the largest element), inside fp32's range
        const int ex = min(max((int)(__float_as_uint(mx) >> 23), 40), 240);
        const float f = __uint_as_float((uint32_t)(262 - ex) << 23), fi = __uint_as_float((uint32_t)(ex - 8) << 23);
#pragma unroll
        for (int s = 0; s < KSTEPS; ++s)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int p = 2 * s + r, d = (p >> 3) * 16;
                const __half2 hh = __floats2half2_rn(v[d + code_at(KB, 2 * (p & 7))] * f, v[d + code_at(KB, 2 * (p & 7) + 1)] * f);
                qf[t][s][r] = *reinterpret_cast<const uint32_t*>(&hh);
            }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r2 = row0 + t * 8 + 2 * c + e;
            qfac[t][e] = __shfl_sync(0xffffffffu, fi, (2 * c + e) * 4) * a.scale_log2;
            const PagedSpan s = paged_span(a, p_first + r2 / a.G, seq.kv);
            col_hi[t][e] = r2 < rows ? s.hi : 0; col_lo[t][e] = s.lo;      // a column without a row sees nothing: what it saw would move the references
        }
    }

    float o[NT][MT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int i = 0; i < MT; ++i) { o[t][i][0] = 0.f; o[t][i][1] = 0.f; o[t][i][2] = 0.f; o[t][i][3] = 0.f; }
#pragma unroll
        for (int e = 0; e < 2; ++e) { m[t][e] = -1e30f; l[t][e] = 0.f; }
    }
    CodeMagic<KB> kmagic;
    CodeMagic<VB> vmagic;
    kmagic.init();
    vmagic.init();
    const int32_t* table = a.table + b * a.table_stride;
    const int page_mask = (1 << a.c.page_shift) - 1;
    unsigned char* ring = pd_smem + warp * (ST * P::TILE);
    // A warp takes the tiles begin + warp, + PD_WARPS, ...: `n` of them.  Lane x keeps the page of tile (x mod 32) of the next 32.
    const int n = begin + warp < end ? (end - begin - warp + PD_WARPS - 1) / PD_WARPS : 0;
    int pages = 0;
    auto request = [&](int i) {                  // tile i of the warp, into its place in the ring; an empty group behind the last
        if (i < n) {
            const int key = key_of(begin + warp + i * PD_WARPS);
            if ((i & 31) == 0) {
                const int mine = i + lane;
                pages = mine < n ? __ldg(table + (key_of(begin + warp + mine * PD_WARPS) >> a.c.page_shift)) : 0;
            }
            const int page = paged_page(a, __shfl_sync(0xffffffffu, pages, i & 31), status);
            const uint32_t at = (uint32_t)((page * a.c.H + h) << a.c.page_shift) + (key & page_mask);      // whole tiles: a page's rows behind the sequence's end may be
            unsigned char* t = ring + (i % ST) * P::TILE;                                                  // copied, not used
            pd_copy<KROW>(t, reinterpret_cast<const unsigned char*>(a.c.kc) + (size_t)at * KROW, lane);
            pd_copy<VROW>(t + 16 * KROW, reinterpret_cast<const unsigned char*>(a.c.vc) + (size_t)at * VROW, lane);
            if (lane < 8) {
                const float* src = (lane < 4 ? a.c.ks : a.c.vs) + at + (lane & 3) * 4;
                asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(t + 16 * (KROW + VROW) + lane * 16)), "l"(src) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    struct Tile {
        PdRaw<KBYTES> k[2];                // keys g, g + 8
        PdRaw<VBYTES> v[4];                // keys 2c, 2c + 1, 2c + 8, 2c + 9
        float ks[2], vs[2];                // of keys g, g + 8
    };
    auto read = [&](Tile& t, int i) {
        const unsigned char *p = ring + (i % ST) * P::TILE, *pv = p + 16 * KROW;
        const float* ps = reinterpret_cast<const float*>(p + 16 * (KROW + VROW));
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            pd_read<KROW>(t.k[r], p, g + 8 * r, c);
            t.ks[r] = ps[g + 8 * r]; t.vs[r] = ps[16 + g + 8 * r];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) pd_read<VROW>(t.v[r], pv, 2 * c + (r & 1) + 8 * (r >> 1), g);
    };
    auto process = [&](const Tile& cur, int k0, auto masked_) {
        constexpr bool MASKED = decltype(masked_)::value;
        float s[NT][4];
        {
            float s2[NT][2][4];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int z = 0; z < 2; ++z) { s2[t][z][0] = 0.f; s2[t][z][1] = 0.f; s2[t][z][2] = 0.f; s2[t][z][3] = 0.f; }
#pragma unroll
            for (int it = 0; it < ITEMS; ++it) {
                uint32_t ka[8], kb[8];
                pd_codes<KB>(cur.k[0].w + it * Item<KB>::NW, ka, kmagic);
                pd_codes<KB>(cur.k[1].w + it * Item<KB>::NW, kb, kmagic);
#pragma unroll
                for (int s4 = 0; s4 < 4; ++s4) {
                    const uint32_t af[4] = {ka[2 * s4], kb[2 * s4], ka[2 * s4 + 1], kb[2 * s4 + 1]};
#pragma unroll
                    for (int t = 0; t < NT; ++t) pd_mma(s2[t][s4 & 1], af, qf[t][it * 4 + s4][0], qf[t][it * 4 + s4][1]);
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[t][i] = s2[t][0][i] + s2[t][1][i];
        }
        uint32_t pf[NT][2];
        float lv[2], rv[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            lv[r] = paged_exponent(cur.vs[r]);
            rv[r] = paged_inverse(cur.vs[r]);
        }
        bool over = false;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = fmaf(cur.ks[r], s[t][2 * r + e] * qfac[t][e], lv[r]);
                    if (MASKED) {
                        const int key = k0 + g + 8 * r;
                        if (!(key < col_hi[t][e] && (key >= col_lo[t][e] || key < a.sinks))) x = -INFINITY;
                    }
                    s[t][2 * r + e] = x;
                    over = over | (x > m[t][e] + PAGED_TOP);
                }
        if (__any_sync(0xffffffffu, over)) {
            // rare after the first tile: new references, the same in every lane of a row, and everything accumulated is rescaled
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = fmaxf(s[t][e], s[t][2 + e]);
#pragma unroll
                    for (int z = 4; z < 32; z <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, z));
                    const float mn = fmaxf(m[t][e], x - PAGED_SET), alpha = pd_ex2(m[t][e] - mn);
                    m[t][e] = mn;
                    l[t][e] *= alpha;
#pragma unroll
                    for (int i = 0; i < MT; ++i) { o[t][i][e] *= alpha; o[t][i][2 + e] *= alpha; }
                }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float p0 = pd_ex2(s[t][2 * r] - m[t][0]), p1 = pd_ex2(s[t][2 * r + 1] - m[t][1]);
                l[t][0] = fmaf(p0, rv[r], l[t][0]); l[t][1] = fmaf(p1, rv[r], l[t][1]);
                const __half2 hh = __floats2half2_rn(p0, p1);
                pf[t][r] = pd_transpose(*reinterpret_cast<const uint32_t*>(&hh));
            }
        uint32_t ja[2 * PdRaw<VBYTES>::NW], jb[2 * PdRaw<VBYTES>::NW];
        pd_join<VB>(cur.v[0].w, cur.v[1].w, ja);
        pd_join<VB>(cur.v[2].w, cur.v[3].w, jb);
#pragma unroll
        for (int it = 0; it < ITEMS; ++it) {
            uint32_t va[8], vb_[8];
            pd_codes<VB>(ja + it * Item<VB>::NW, va, vmagic);
            pd_codes<VB>(jb + it * Item<VB>::NW, vb_, vmagic);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t af[4] = {va[2 * i], va[2 * i + 1], vb_[2 * i], vb_[2 * i + 1]};
#pragma unroll
                for (int t = 0; t < NT; ++t) pd_mma(o[t][it * 4 + i], af, pf[t][0], pf[t][1]);
            }
        }
    };
#pragma unroll 1
    for (int i = 0; i < ST - 1; ++i) request(i);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
        __syncwarp();                            // all lanes' copies of tile i are there, and all lanes are done with tile i - 1
        Tile t;
        read(t, i);
        request(i + ST - 1);
        const int k0 = key_of(begin + warp + i * PD_WARPS);
        if (k0 + PD_KEYS > all_hi || (k0 < all_lo && k0 + PD_KEYS > a.sinks)) process(t, k0, std::true_type());
        else process(t, k0, std::false_type());
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    // ---- a warp's partial result
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int z = 4; z < 32; z <<= 1) l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], z);
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int z = 0; z < 4; ++z)      // row g (z < 2) or g + 8 of row tile j = elements 2 j, 2 j + 1 of this thread's eighth of the head_dim
                s_part[warp][t * 8 + 2 * c + (z & 1)][g * (D / 8) + 2 * j + (z >> 1)] = o[t][j][z];
        if (g == 0) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                s_part[warp][t * 8 + 2 * c + e][D] = m[t][e];
                s_part[warp][t * 8 + 2 * c + e][D + 1] = l[t][e];
            }
        }
    }
    __syncthreads();
    // ---- merge the warps, then write the output, meet the cluster, or leave this split's part
    const long long n_rows = (long long)a.T * a.Hq;
    auto finish = [&](int row, int d, float num, float den, float M) {
        const int token = row / a.G, head = h * a.G + row - token * a.G;
        store_o_elem(a.out, a.dtype, (long long)(seq.q0 + token) * a.os_t + head * a.os_h + d, den != 0.f ? num / den : 0.f);
        if (d == 0 && a.lse) a.lse[(long long)(seq.q0 + token) * a.Hq + head] = den != 0.f ? (M + __log2f(den)) * 0.6931471805599453f : -INFINITY;
    };
    float (*s_cta)[D + 2] = reinterpret_cast<float (*)[D + 2]>(pd_smem + PD_WARPS * ROWS * (D + 2) * 4);
    for (int j = threadIdx.x; j < ROWS * D; j += PD_WARPS * 32) {
        const int r = j / D, d = j - r * D, row = row0 + r;
        if (row >= rows) break;
        float M = -FLT_MAX;
#pragma unroll
        for (int w = 0; w < PD_WARPS; ++w) M = fmaxf(M, s_part[w][r][D]);
        float num = 0.f, den = 0.f;
#pragma unroll
        for (int w = 0; w < PD_WARPS; ++w) {
            const float wt = pd_ex2(s_part[w][r][D] - M);
            num = fmaf(wt, s_part[w][r][d], num);
            den = fmaf(wt, s_part[w][r][D + 1], den);
        }
        if (splits == 1) finish(row, d, num, den, M);
        else if (in_cluster) {
            s_cta[r][d] = num;
            if (d == 0) { s_cta[r][D] = M; s_cta[r][D + 1] = den; }
        } else {
            const int token = row / a.G, head = h * a.G + row - token * a.G;
            const long long out_row = (long long)(seq.q0 + token) * a.Hq + head;
            ws_o[(split * n_rows + out_row) * D + d] = num;
            if (d == 0) *reinterpret_cast<float2*>(ws_ml + (split * n_rows + out_row) * 2) = make_float2(M, den);
        }
    }
    if (paged_pad_any(a, seq, b)) pd_pad(paged_pad_rows(a, seq, b, h), (long long)(rt * splits + split) * (PD_WARPS * 32) + threadIdx.x, (long long)n_rowtiles * splits * (PD_WARPS * 32));
    if (in_cluster) {
        const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
        cluster.sync();
        for (int j = threadIdx.x + split * (PD_WARPS * 32); j < ROWS * D; j += splits * (PD_WARPS * 32)) {      // the CTAs share out the elements
            const int r = j / D, d = j - r * D;
            if (row0 + r >= rows) break;
            float M = -FLT_MAX, num = 0.f, den = 0.f;
            for (int s = 0; s < splits; ++s) M = fmaxf(M, cluster.map_shared_rank(&s_cta[r][D], s)[0]);
            for (int s = 0; s < splits; ++s) {
                const float* p = cluster.map_shared_rank(&s_cta[r][0], s);
                const float wt = pd_ex2(p[D] - M);
                num = fmaf(wt, p[d], num);
                den = fmaf(wt, p[D + 1], den);
            }
            finish(row0 + r, d, num, den, M);
        }
        cluster.sync();                          // nobody leaves while its shared memory is read
    }
}

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

template <int KB, int VB, int D, int NT>
int launch_nt(const PagedAttnArgs& a, int splits, bool in_cluster, int tiles_per_split, float* ws_o, float* ws_ml, int* status, cudaStream_t st) {
    constexpr int PART = (PD_WARPS + 1) * 8 * NT * (D + 2) * 4, SMEM = PdPlan<KB, VB, D>::SMEM > PART ? PdPlan<KB, VB, D>::SMEM : PART;
    const long long rows = (long long)a.max_q * a.G;
    const int n_rowtiles = (int)((rows + 8 * NT - 1) / (8 * NT));
    const long long blocks = (long long)a.B * a.c.H * n_rowtiles * splits;
    if (blocks > 0x7fffffffLL) return fail(VARQ_ERR_UNSUPPORTED, "varq_paged_attn: more than 2^31 thread blocks");
    static bool configured[64] = {false};
    int dev = 0;
    VARQ_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        VARQ_CUDA_TRY(cudaFuncSetAttribute(paged_attn_decode_kernel<KB, VB, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    VARQ_CUDA_TRY(launch_pdl(paged_attn_decode_kernel<KB, VB, D, NT>, (unsigned)blocks, PD_WARPS * 32, SMEM, st, in_cluster ? splits : 1, a, n_rowtiles, splits, in_cluster, tiles_per_split, ws_o, ws_ml,
                             status));
    count_launches(1);
    return VARQ_OK;
}
template <int KB, int VB, int D>
int launch(const PagedAttnArgs& a, int rows, int splits, bool in_cluster, int tiles_per_split, float* ws_o, float* ws_ml, int* status, cudaStream_t st) {
    switch (rows) {
        case 8: return launch_nt<KB, VB, D, 1>(a, splits, in_cluster, tiles_per_split, ws_o, ws_ml, status, st);
        case 16: return launch_nt<KB, VB, D, 2>(a, splits, in_cluster, tiles_per_split, ws_o, ws_ml, status, st);
        default: return launch_nt<KB, VB, D, 3>(a, splits, in_cluster, tiles_per_split, ws_o, ws_ml, status, st);
    }
}

}  // namespace

int paged_attn_decode_run(const PagedAttnArgs& a, int rows, int splits, bool in_cluster, int tiles_per_split, float* ws_o, float* ws_ml, int* status, cudaStream_t st) {
#define GO(K_, V_) \
    if (a.c.kb == K_ && a.c.vb == V_) return a.c.D == 64 ? launch<K_, V_, 64>(a, rows, splits, in_cluster, tiles_per_split, ws_o, ws_ml, status, st) : launch<K_, V_, 128>(a, rows, splits, in_cluster, tiles_per_split, ws_o, ws_ml, status, st);
    GO(8, 8) GO(8, 4) GO(8, 2) GO(4, 8) GO(4, 4) GO(4, 2) GO(2, 8) GO(2, 4) GO(2, 2)
#undef GO
    return fail(VARQ_ERR_ARG, "varq_paged_attn: bits must be 2, 4 or 8");
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
