// Attention of a chunk over a paged cache on the 5th-generation tensor cores (tcgen05 + TMEM).
//
// One CTA = one (sequence, head of the cache) x 256 query rows, two tiles of 128; a row is a (token, query head of the group) pair, so query
// heads that share a head of the cache share its converted tiles.  It walks over tiles of 64 keys; those of first tokens (sinks) and those of the window
// are lists of tiles one behind the other.  Per key tile and query tile
//   S = Q K^T       Q fp16 in shared memory, K integer codes as exact fp16; S fp32 in tensor memory
//   x = S a_j + b_j with a_j = K scale * softmax_scale * log2 e and b_j = log2 of the V scale
//   P = 2^(x - m)   fp16, written over S in tensor memory, = weight * V scale relative to the row's reference m
//   l += P / V scale in fp32, from the unrounded P;      O += P V, V integer codes as exact fp16, O fp32 in tensor memory
// and at the end out = O / l, log-sum-exp = (m + log2 l) ln 2.  The reference m is that of weight times V scale, which is what bounds O: it is set 7 below a row's first
// largest x, and raised, again to 7 below, only when an x passes it by more than 15 (P then stays below 2^15, fp16 ends at 2^16).  The tile's scores are then taken
// again against the new one, O, l and the weights of the tile's first half rescaled in fp32.
// What is held in fewer than 32 bits: P, because it is the operand of a 16-bit product.  A weight times V scale of 2^-21 of the row's largest or more is rounded by
// itself, 2^-12 of it; a smaller one by 2^-32 of the largest.  (Where one V row is far larger than the others, the others' part in the columns in which its codes are
// zero is off by as much of *its* size.)  Weights of the first half of a tile whose second half raises the
// reference are rounded twice.  Codes are exact in fp16, and so are fp16 queries; bf16 queries
// too, but for elements below 2^-13 of their row's largest, which are off by 2^-21 of it at most: a row whose largest element lies outside [2^-4, 2^15) is scaled by a
// power of two (then S a_j takes a factor).
//
// Warps: 0-3 and 4-7 softmax of the two query tiles; 8-11 and 12-15 convert K and V: packed rows from shared memory to 128B-swizzled fp16 tiles, scales to the
// tables a, b, 1 / V scale; 16 and 17 issue the products of the two query tiles; 18 and 19 fetch packed rows and scales of K and V with a bulk copy for every
// run of keys in one page, RST tiles ahead.  Two or three score tiles per query tile (what tensor memory holds beside O) are in flight, so that a softmax warp
// finds the next scores there while the tensor pipe works on its weights.
// Every wait is bounded: on expiry the kernel records a status code and all roles drain out.
//
// What bounds it (B200, 1965 MHz): the softmax warps.  At 128 columns and 8-bit codes a tile of 64 keys takes ~2470 cycles of a CTA, of which the exponentials
// alone are 1024 (8 cycles a warp instruction on each of the four schedulers); the products by themselves take 440 us of the first case, 240 of the second.  Measured:
//   2048 queries behind 16384 keys, 32 query / 8 cache heads, 128 columns, 8 bits   736 us   794 TFLOP/s (359 us at the dense rate)
//   16 sequences, 1024 queries on 2240 keys each, 30 heads, 64 columns, 4 bits       640 us   440 TFLOP/s (173 us at the dense rate; the exponentials alone would take 245)
//   4096 queries, window 2048, 128 columns                                          121 us   573 TFLOP/s
// No unit is full (first case: issue 49 %, exponentials' unit 42 %, tensor pipe 35 % of 86 that 256 CTAs on 148 SMs can reach): two softmax warps on a scheduler run load,
// maximum, vote, exponentials and store as a chain.
// Measured on the way, one step after another, so that the last figure of a line is that of its day.  Tiles tried: 128 keys with one score tile each 784 / 721 / 137 us (the softmax waits for its scores); 64 keys, packed rows straight from the pages into the
// converters' registers 770 / 680 / 125 us (a converter waits out its loads at the proxy fence, which lets no load pass); bulk copies 740 / 638 / 120 us.
// Turned down: the first scores of the next tile under the last exponentials of this one, 876 / 687 / 137 us (P comes later, and the products with it); weights
// first and one vote on them for the whole tile, 716 / 646 / 119 us, but 1 to 2 us more on a call of 14 to 24 us.
// Register shares 152 / 64 (softmax / converters) 768 / 638, 144 / 72 740 / 638, 160 / 56 756 / 638 us.
#include "varq_paged_attn_tc.cuh"

namespace varq {
namespace {

template <int D> struct PtPlan {
    static constexpr int SB = D == 64 ? 3 : 2;                     // score tiles per query tile
    static constexpr int KST = D == 64 ? 4 : 3, VST = KST;         // stages of K and V as fp16
    static constexpr int RST = D == 64 ? 6 : 3;                    // stages of K and V as they lie in the pages
    static constexpr int TS = KST + SB;                            // tables: a table is read until its P is written, SB tiles behind its K
    static constexpr int Q_BYTES = PT_M * D * 2, T_BYTES = PT_N * D * 2, R_BYTES = PT_N * D, RAW_BYTES = R_BYTES + PT_N * 4;     // packed rows, then scales
    static constexpr int TAB_FLOATS = 3 * PT_N;
    static constexpr int OFF_Q = 0, OFF_K = OFF_Q + 2 * Q_BYTES, OFF_V = OFF_K + KST * T_BYTES, OFF_RK = OFF_V + VST * T_BYTES, OFF_RV = OFF_RK + RST * RAW_BYTES,
                         OFF_TAB = OFF_RV + RST * RAW_BYTES;
    // barriers: K, V written and free; packed K, V there and free; tables written; queries; S, P of every score tile; O (a ring of four tiles); end
    static constexpr int B_K = 0, B_KF = B_K + KST, B_V = B_KF + KST, B_VF = B_V + VST, B_RK = B_VF + VST, B_RKF = B_RK + RST, B_RV = B_RKF + RST, B_RVF = B_RV + RST,
                         B_TAB = B_RVF + RST, B_Q = B_TAB + TS, B_S = B_Q + 2, B_P = B_S + 2 * SB, B_O = B_P + 2 * SB, B_END = B_O + 8, N_BARS = B_END + 2;
    static constexpr int OFF_BAR = OFF_TAB + TS * TAB_FLOATS * 4;
    static constexpr int OFF_QF = (OFF_BAR + N_BARS * 8 + 15) / 16 * 16;              // factors of the queries [2][128]
    static constexpr int OFF_MISC = OFF_QF + 2 * PT_M * 4, SMEM = OFF_MISC + 16 + 1024;
    static constexpr int COL_O = 0, COL_S = 2 * D, TMEM_COLS = 512;
    static_assert(COL_S + 2 * SB * PT_N <= TMEM_COLS && SMEM <= 227 * 1024 && OFF_RK % 128 == 0, "plan");
    static constexpr int SOFT = 8, K_WARP0 = SOFT, V_WARP0 = K_WARP0 + 4, MMA_WARP = V_WARP0 + 4, LOAD_WARP = MMA_WARP + 2, THREADS = (LOAD_WARP + 2) * 32;
    static constexpr int REGS = 96, REGS_SOFT = 144, REGS_CONV = 72, REGS_MISC = 48;
    static_assert(SOFT * 32 * REGS_SOFT + 256 * REGS_CONV + 128 * REGS_MISC <= THREADS * REGS, "register plan");
};

template <int D>
__global__ void __launch_bounds__(PtPlan<D>::THREADS, 1) paged_attn_tc_kernel(PagedAttnArgs a, int n_qblocks, int splits, float* ws_o, float* ws_ml, int* status) {
    using P = PtPlan<D>;
    constexpr int KST = P::KST, VST = P::VST, TS = P::TS, SB = P::SB;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + P::OFF_BAR);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + P::OFF_MISC);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + P::OFF_MISC + 8);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    if (warp == P::LOAD_WARP) {
        for (int i = lane; i < P::N_BARS; i += 32) {        // warps that arrive
            auto in = [&](int lo, int hi) { return i >= lo && i < hi; };
            const bool by_8 = in(P::B_TAB, P::B_Q);
            const bool by_4 = in(P::B_K, P::B_KF) || in(P::B_V, P::B_VF) || in(P::B_RKF, P::B_RV) || in(P::B_RVF, P::B_TAB) || in(P::B_Q, P::B_S) || in(P::B_P, P::B_O);
            const bool by_2 = in(P::B_KF, P::B_V) || in(P::B_VF, P::B_RK);
            mbar_init(&bars[i], by_8 ? 8u : by_4 ? 4u : by_2 ? 2u : 1u);
        }
        if (lane == 0) *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == P::MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)P::TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_wait();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();       // behind the allocation: a CTA of a next launch must not take tensor memory that one of this launch still asks for
    const uint32_t tmem_base = *tmem_slot;

    // ---- what this CTA does: late query blocks, which see the most keys, first
    const int split = (int)(blockIdx.x % (unsigned)splits);
    const unsigned item = blockIdx.x / (unsigned)splits, heads = (unsigned)(a.B * a.c.H);
    const int bh = (int)(item % heads), qb = n_qblocks - 1 - (int)(item / heads), b = bh / a.c.H, h = bh - b * a.c.H;
    const PagedSeq seq = paged_seq(a, b, status);
    const int rows = seq.nq * a.G, row0 = qb * (2 * PT_M);                   // rows of the (sequence, head); first one of this CTA
    const int p_first = seq.kv - seq.nq;                                     // position of the first query
    PtTiles tiles;
    int n_t[2], tile0 = 0;                                                   // key tiles of the two query tiles
    {
        const int t0 = row0 / a.G, t1 = (min(row0 + 2 * PT_M, rows) - 1) / a.G, t_mid = (min(row0 + PT_M, rows) - 1) / a.G;
        const int hi = max(a.causal ? min(seq.kv, p_first + t1 + 1) : seq.kv, 0), hi0 = max(a.causal ? min(seq.kv, p_first + t_mid + 1) : seq.kv, 0);
        tiles.first = paged_window(a, p_first + t0);
        tiles.lo = tiles.first & ~(PT_N - 1);
        tiles.ns = min((a.sinks + PT_N - 1) / PT_N, tiles.lo / PT_N);
        const int n = hi > 0 ? tiles.ns + (max(hi - tiles.lo, 0) + PT_N - 1) / PT_N : 0, n0 = hi0 > 0 ? tiles.ns + (max(hi0 - tiles.lo, 0) + PT_N - 1) / PT_N : 0;
        tile0 = (int)((long long)n * split / splits);
        tiles.n = row0 < rows ? (int)((long long)n * (split + 1) / splits) - tile0 : 0;
        n_t[0] = min(max(n0 - tile0, 0), tiles.n);
        n_t[1] = row0 + PT_M < rows ? tiles.n : 0;
    }
    const int n_all = max(n_t[0], n_t[1]);
    const int page_mask = (1 << a.c.page_shift) - 1;
    const int32_t* table = a.table + b * a.table_stride;

    if (warp < P::SOFT) {
        // =============================================================== softmax, epilogue
        set_registers<P::REGS_SOFT, P::REGS>();
        const int t = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane, row = row0 + t * PT_M + r;
        const bool live = row < rows;
        const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16), col_s0 = lane_base + P::COL_S + t * (SB * PT_N), col_o = lane_base + P::COL_O + t * D;
        if (row0 + t * PT_M < rows) {
            const int token = live ? row / a.G : 0, head = h * a.G + (live ? row - token * a.G : 0);
            // ---- queries -> fp16 in shared memory, in the order in which the codes of K are unpacked
            float q_factor = 1.f;
            {
                uint4 raw[D / 8];
                const long long off = (long long)(seq.q0 + token) * a.qs_t + head * a.qs_h;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) raw[i] = live ? load_q16<2>(a.q, off + 8 * i) : make_uint4(0, 0, 0, 0);
                float f = 1.f;
                if (a.dtype == VARQ_BF16) {
                    uint32_t top = 0;                                        // bits of the largest absolute value
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) top = max(top, max(w[j] & 0x7fffu, (w[j] >> 16) & 0x7fffu));
                    }
                    const int ex = (int)(top >> 7);                          // exponent: 2^(ex - 127)
                    if (top && (ex < 123 || ex > 141)) {                     // -> largest element in [2^8, 2^9); NaN and infinity stay what they are
                        const int e = min(max(ex, 40), 240);
                        f = __uint_as_float((uint32_t)(262 - e) << 23);
                        q_factor = __uint_as_float((uint32_t)(e - 8) << 23);
                    }
                }
                unsigned char* qs = smem + P::OFF_Q + t * P::Q_BYTES;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    uint32_t w[8] = {raw[2 * i].x, raw[2 * i].y, raw[2 * i].z, raw[2 * i].w, raw[2 * i + 1].x, raw[2 * i + 1].y, raw[2 * i + 1].z, raw[2 * i + 1].w};
                    if (a.dtype == VARQ_BF16) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) w[j] = pack_half2(__uint_as_float(w[j] << 16) * f, __uint_as_float(w[j] & 0xffff0000u) * f);
                    }
                    q_operand_order(w, a.c.kb);
                    sts128(qs + pt_chunk<PT_M>(r, 2 * i), w[0], w[1], w[2], w[3]);
                    sts128(qs + pt_chunk<PT_M>(r, 2 * i + 1), w[4], w[5], w[6], w[7]);
                }
            }
            fence_async_smem();
            warp_arrive(&bars[P::B_Q + t], lane);
            const bool scaled = __any_sync(0xffffffffu, q_factor != 1.f);
            if (scaled) reinterpret_cast<float*>(smem + P::OFF_QF)[t * PT_M + r] = q_factor;
            __syncwarp();
            // keys between which every row of the query tile sees everything
            const int tl = min(row0 + t * PT_M + PT_M, rows) - 1, all_hi = a.causal ? p_first + (row0 + t * PT_M) / a.G + 1 : 0x7fffffff,
                      all_lo = paged_window(a, p_first + tl / a.G);
            // A thread holds, of every eight columns of S, two of the rows g, g + 8, g + 16, g + 24 of its warp's 32 (g = lane / 4): it needs a quarter of
            // the keys' tables and uses an entry for four rows
            const int g = lane >> 2, cq = lane & 3;
            int pos[4];                                                     // positions of the four rows' tokens
#pragma unroll
            for (int i = 0; i < 4; ++i) pos[i] = p_first + min(row0 + t * PT_M + quarter * 32 + g + 8 * i, rows - 1) / a.G;
            pair nm[4] = {0ull, 0ull, 0ull, 0ull};                          // minus the reference, twice
            pair l[4] = {0ull, 0ull, 0ull, 0ull};
            unsigned unset = 15u;                                           // rows that have no reference yet: they have seen no key
            bool ok = true;
            const int n = n_t[t];
            auto by_lane = [&](const float (&v)[4]) {                        // rows g + 8 i of a thread -> row `lane`
                float o = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) { const float x = __shfl_sync(0xffffffffu, v[i], (lane & 7) * 4); o = (lane >> 3) == i ? x : o; }
                return o;
            };
#pragma unroll 1
            for (int j = 0; j < n; ++j) {
                const int key0 = tiles.key(tile0 + j);
                {
                    uint64_t *tab_bar = &bars[P::B_TAB + j % TS], *s_bar = &bars[P::B_S + t * SB + j % SB];
                    const bool there = mbar_test(tab_bar, (j / TS) & 1) & mbar_test(s_bar, (j / SB) & 1);        // both at once: that is a round trip less
                    if (!__all_sync(0xffffffffu, there))
                        ok = mbar_wait_warp(tab_bar, (j / TS) & 1, abort_flag, 201) && mbar_wait_warp(s_bar, (j / SB) & 1, abort_flag, 202);
                    if (!ok) break;
                }
                const uint32_t col_s = col_s0 + (j % SB) * PT_N;
                tc_fence_after();
                const float* tab = reinterpret_cast<const float*>(smem + P::OFF_TAB) + (j % TS) * P::TAB_FLOATS;
                // Two forms of a tile, so that the usual one carries neither masks nor factors: as branches inside they cost 10 % of a long call.  The scores of a
                // chunk of 32 keys come with their maximum and the vote on it while the exponentials of the chunk before are at work: alone the chain of load,
                // maximum, vote and branch takes as long as those (613 cycles a chunk one after the other, 341 so; 280 with two warps on a scheduler, 256 the
                // exponentials alone).
                auto tile = [&](auto special_) {
                    constexpr bool SPECIAL = decltype(special_)::value != 0;
                    // x - m of 32 columns: [half of the rows][eight columns][row g, g + 8]; true where a row needs another reference
                    auto scores = [&](pair (&x)[16], int c) -> bool {
                        uint32_t s[32];
                        tmem_ld_16x256(col_s + 32 * c, s);
                        tmem_ld_16x256(col_s + 32 * c + (16u << 16), s + 16);
                        tmem_loaded(s);
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[i] = pair_of_bits(s[2 * i], s[2 * i + 1]);
                        if (SPECIAL && scaled) {
                            const float* qf = reinterpret_cast<const float*>(smem + P::OFF_QF) + t * PT_M + quarter * 32 + g;
#pragma unroll
                            for (int i = 0; i < 16; ++i) { const float f = qf[8 * ((i >> 3) * 2 + (i & 1))]; x[i] = mul2(x[i], pair_of(f, f)); }
                        }
#pragma unroll
                        for (int v = 0; v < 4; ++v) {
                            const ulonglong2 ab = *reinterpret_cast<const ulonglong2*>(tab + (c * 16 + v * 4 + cq) * 4);
#pragma unroll
                            for (int i = 0; i < 4; ++i) { pair& y = x[(i >> 1) * 8 + v * 2 + (i & 1)]; y = add2(fma2(y, ab.x, ab.y), nm[i]); }
                        }
                        if (SPECIAL) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const PagedSpan sp = paged_span(a, pos[i], seq.kv);
                                // bit k: this thread's column 2c + k of the 32 is seen
                                auto below = [](int k) { return k <= 0 ? 0u : k >= 32 ? ~0u : (1u << k) - 1u; };
                                const int c0 = key0 + 32 * c + 2 * cq;
                                const uint32_t sees = below(sp.hi - c0) & (~below(sp.lo - c0) | below(a.sinks - c0));
#pragma unroll
                                for (int v = 0; v < 4; ++v) {
                                    pair& y = x[(i >> 1) * 8 + v * 2 + (i & 1)];
                                    y = pair_of(sees >> (8 * v) & 1u ? pair_x(y) : -INFINITY, sees >> (8 * v + 1) & 1u ? pair_y(y) : -INFINITY);
                                }
                            }
                        }
                        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int i = 0; i < 16; ++i) top[i & 3] = fmaxf(top[i & 3], fmaxf(pair_x(x[i]), pair_y(x[i])));
                        return __any_sync(0xffffffffu, unset != 0u || fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) > PAGED_TOP) != 0;
                    };
                    // new references from the scores of chunk c, whose predecessors are done; the chunk's scores are then computed once more (changed in place they
                    // would be copied on the way that is always taken)
                    auto raise = [&](pair (&x)[16], int c) {
                        float alpha[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float up = -INFINITY;                        // how far the row's largest x is above its reference
#pragma unroll
                            for (int v = 0; v < 4; ++v) { const pair y = x[(i >> 1) * 8 + v * 2 + (i & 1)]; up = fmaxf(up, fmaxf(pair_x(y), pair_y(y))); }
                            up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, 1));
                            up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, 2));
                            const bool first = (unset >> i & 1u) && up > -INFINITY;
                            // to the largest x itself, which is then a power of two in fp16: where it is most of the sum, so is its exactness
                            up = first || (up > PAGED_TOP && !(unset >> i & 1u)) ? up - PAGED_SET : 0.f;
                            alpha[i] = first ? 1.f : ex2(-up);           // (nothing is accumulated where the reference is the first)
                            if (first) unset &= ~(1u << i);
                            nm[i] = add2(nm[i], pair_of(-up, -up));
                            l[i] = mul2(l[i], pair_of(alpha[i], alpha[i]));
                        }
                        const float al = by_lane(alpha);
                        tmem_wait_st();
#pragma unroll 1
                        for (int z = 0; z < c; ++z) {                    // P of the tile's chunks before this one
                            uint32_t o[16];
                            tmem_ld16(col_s + 16 * z, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) {                // (the factor may be too small for fp16)
                                const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&o[i]));
                                o[i] = pack_half2(p.x * al, p.y * al);
                            }
                            tmem_st16(col_s + 16 * z, o);
                        }
                        if (j > 0) {                                     // behind the products of the tile before
                            ok = __all_sync(0xffffffffu, mbar_wait(&bars[P::B_O + 4 * t + ((j - 1) & 3)], ((j - 1) >> 2) & 1, abort_flag, 203));
                            tc_fence_after();
#pragma unroll 1
                            for (int z = 0; z < D && ok; z += 16) {
                                uint32_t o[16];
                                tmem_ld16(col_o + z, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * al);
                                tmem_st16(col_o + z, o);
                            }
                        }
                        scores(x, c);
                    };
                    // P of a chunk: 16 columns over scores that are read already
                    auto weights = [&](const pair (&x)[16], int c) {
                        uint32_t pk[16];
#pragma unroll
                        for (int v = 0; v < 4; ++v) {
                            const pair vc = *reinterpret_cast<const pair*>(tab + 2 * PT_N + c * 32 + v * 8 + 2 * cq);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const pair y = x[(i >> 1) * 8 + v * 2 + (i & 1)];
                                const float p0 = ex2(pair_x(y)), p1 = ex2(pair_y(y));
                                l[i] = fma2(pair_of(p0, p1), vc, l[i]);
                                pk[(i >> 1) * 8 + v * 2 + (i & 1)] = pack_half2(p0, p1);
                            }
                        }
                        tmem_st_16x128(col_s + 16 * c, pk);
                        tmem_st_16x128(col_s + 16 * c + (16u << 16), pk + 8);
                    };
                    pair xa[16], xb[16];
                    if (scores(xa, 0)) raise(xa, 0);
                    const bool other = scores(xb, 1);
                    weights(xa, 0);
                    if (other) raise(xb, 1);
                    weights(xb, 1);
                };
                if (scaled || key0 + PT_N > all_hi || (key0 < all_lo && key0 + PT_N > a.sinks)) tile(IntC<1>()); else tile(IntC<0>());
                if (!ok) break;
                tmem_wait_st();
                tc_fence_before();
                warp_arrive(&bars[P::B_P + t * SB + j % SB], lane);
            }
            float row_l, row_m;
            {
                float v[4], m[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[i] = pair_x(l[i]) + pair_y(l[i]);
                    v[i] += __shfl_xor_sync(0xffffffffu, v[i], 1);
                    v[i] += __shfl_xor_sync(0xffffffffu, v[i], 2);
                    m[i] = unset >> i & 1u ? -1e30f : -pair_x(nm[i]);
                }
                row_l = by_lane(v);
                row_m = by_lane(m);
            }
            // ---- O / l, or this split's part
            if (ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars[P::B_O + 4 * t + ((n - 1) & 3)], ((n - 1) >> 2) & 1, abort_flag, 203));
            tc_fence_after();
            if (ok) {
                const float inv = row_l != 0.f ? 1.f / row_l : 0.f;       // (a NaN stays one)
                const long long out_row = (long long)(seq.q0 + token) * a.Hq + head, n_rows = (long long)a.T * a.Hq;
                const long long oo = (long long)(seq.q0 + token) * a.os_t + head * a.os_h;
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    float v[32];
                    if (n > 0) { tmem_ld32(col_o + c, o); tmem_wait_ld(); }
                    else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = 0u;
                    }
                    if (a.c.vb == 8) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(o[i]);
                    } else if (a.c.vb == 4) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(o[(i & 16) + code_pos(4, i & 15)]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(o[(i & 16) + code_pos(2, i & 15)]);
                    }
                    if (!live) continue;
                    if (splits == 1) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] *= inv;
                        store_o_row32(a.out, a.dtype, oo + c, v);
                    } else {
                        store_o_row32(ws_o, VARQ_F32, (split * n_rows + out_row) * D + c, v);
                    }
                }
                if (live && splits > 1) *reinterpret_cast<float2*>(ws_ml + (split * n_rows + out_row) * 2) = make_float2(row_m, row_l);
                if (live && splits == 1 && a.lse) a.lse[out_row] = row_l != 0.f ? (row_m + __log2f(row_l)) * 0.6931471805599453f : -INFINITY;
            }
        }
    } else if (warp < P::MMA_WARP) {
        // =============================================================== converters
        set_registers<P::REGS_CONV, P::REGS>();
        const bool is_k = warp < P::V_WARP0;
        const int ptid = tid & 127, it = ptid & 3, kq = ptid >> 2;       // 16-code item of a 64-column block; keys kq and kq + 32
        unsigned char* stages = smem + (is_k ? P::OFF_K : P::OFF_V);
        const unsigned char* raw_stages = smem + (is_k ? P::OFF_RK : P::OFF_RV);
        uint64_t *full = bars + (is_k ? P::B_K : P::B_V), *freed = bars + (is_k ? P::B_KF : P::B_VF);
        uint64_t *raw_full = bars + (is_k ? P::B_RK : P::B_RV), *raw_freed = bars + (is_k ? P::B_RKF : P::B_RVF);
        auto loop = [&](auto bits_) {
            constexpr int BITS = decltype(bits_)::value, NW = BITS / 2, ROW = D * BITS / 8, NB = D / 64;
            CodeMagic<BITS> magic;
            magic.init();
            // Rows of two 64-column blocks: every other group of rows begins with the second, so that the rows that are read together lie in all banks
            const int nb0 = NB == 2 ? kq >> (BITS == 8 ? 0 : BITS == 4 ? 1 : 2) & 1 : 0;
            const uint32_t d0 = pt_chunk<PT_N>(kq, 2 * it), d1 = pt_chunk<PT_N>(kq, 2 * it + 1);
            int st = 0, rst = 0, ts = 0;
            uint32_t st_ph = 1, rst_ph = 0;
#pragma unroll 1
            for (int j = 0; j < n_all; ++j) {
                const int k = kq + 32 * it;
                if (!mbar_wait_warp(&raw_full[rst], rst_ph, abort_flag, is_k ? 211 : 212)) break;
                const unsigned char* raw = raw_stages + rst * P::RAW_BYTES;
                uint32_t w[2][NB][NW];                 // rows that were not fetched: whatever lay there (any codes are finite; the tables hide them)
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        const unsigned char* src = raw + (kq + 32 * p) * ROW + (nb ^ nb0) * (8 * BITS) + it * (NW * 4);
                        if constexpr (NW == 4) {
                            const uint4 x = *reinterpret_cast<const uint4*>(src);
                            w[p][nb][0] = x.x; w[p][nb][1] = x.y; w[p][nb][2] = x.z; w[p][nb][3] = x.w;
                        } else if constexpr (NW == 2) {
                            const uint2 x = *reinterpret_cast<const uint2*>(src);
                            w[p][nb][0] = x.x; w[p][nb][1] = x.y;
                        } else w[p][nb][0] = *reinterpret_cast<const uint32_t*>(src);
                    }
                const float sc = reinterpret_cast<const float*>(raw + P::R_BYTES)[k & (PT_N - 1)];
                if (j >= KST && !mbar_wait_warp(&freed[st], st_ph, abort_flag, is_k ? 204 : 205)) break;
                float* tab = reinterpret_cast<float*>(smem + P::OFF_TAB) + ts * P::TAB_FLOATS;
                if (it < 2) {
                    float* tab_a = tab + (k >> 1) * 4 + (k & 1);
                    const int key = tiles.key(tile0 + j) + k;
                    const bool there = key < seq.kv && (key >= tiles.first || key < a.sinks);      // a run that no row sees is not fetched
                    if (is_k) tab_a[0] = there ? sc * a.scale_log2 : 0.f;
                    else {
                        tab_a[2] = there ? paged_exponent(sc) : -INFINITY;
                        tab[2 * PT_N + k] = there ? paged_inverse(sc) : 0.f;
                    }
                }
                unsigned char* tile = stages + st * P::T_BYTES;
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        uint32_t hw[8];
                        Item<BITS>::raw(w[p][nb], hw, magic);
#pragma unroll
                        for (int i = 0; i < 8; ++i) hw[i] = Item<BITS>::minus_zp(hw[i], i, pt_neg_base<BITS>(i % Item<BITS>::CLS));
                        unsigned char* block = tile + (nb ^ nb0) * (PT_N * 128) + p * (32 * 128);
                        sts128(block + d0, hw[0], hw[1], hw[2], hw[3]);
                        sts128(block + d1, hw[4], hw[5], hw[6], hw[7]);
                    }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) { mbar_arrive(&full[st]); mbar_arrive(&bars[P::B_TAB + ts]); mbar_arrive(&raw_freed[rst]); }
                if (++st == KST) { st = 0; st_ph ^= 1u; }
                if (++rst == P::RST) { rst = 0; rst_ph ^= 1u; }
                if (++ts == TS) ts = 0;
            }
        };
        const int bits = is_k ? a.c.kb : a.c.vb;
        if (bits == 8) loop(IntC<8>()); else if (bits == 4) loop(IntC<4>()); else loop(IntC<2>());
    } else {
        set_registers<P::REGS_MISC, P::REGS>();
        if (warp < P::MMA_WARP + 2) {
            // =============================================================== products of query tile t (the whole warp waits; one elected lane issues)
            // S(0) .. S(SB - 1), then for every key tile j: P(j) -> O += P(j) V(j) -> S(j + SB) over the columns of P(j)
            constexpr uint32_t IDESC_S = instr_desc(PT_M, PT_N, 0), IDESC_O = instr_desc(PT_M, D, 1);
            const int t = warp - P::MMA_WARP, n = n_t[t];
            const uint64_t qd = smem_desc(smem_u32(smem + P::OFF_Q + t * P::Q_BYTES), 16, 1024), kd = smem_desc(smem_u32(smem + P::OFF_K), 16, 1024);
            const uint64_t vd = smem_desc(smem_u32(smem + P::OFF_V), PT_N * 128, 1024);
            const uint32_t col_s = tmem_base + P::COL_S + t * (SB * PT_N), col_o = tmem_base + P::COL_O + t * D;
            bool ok = true;
            auto issue_s = [&](int j) {
                if (!(ok = mbar_wait_warp(&bars[P::B_K + j % KST], (j / KST) & 1, abort_flag, 207))) return;
                tc_fence_after();
                if (j < n) {
                    const uint64_t bd = kd + (uint64_t)(((j % KST) * P::T_BYTES) >> 4);
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
                        tc_mma_ss(col_s + (j % SB) * PT_N, qd + (uint64_t)(((kk >> 2) * (PT_M * 128) + (kk & 3) * 32) >> 4),
                                  bd + (uint64_t)(((kk >> 2) * (PT_N * 128) + (kk & 3) * 32) >> 4), IDESC_S, kk ? 1u : 0u);
                    tc_commit(&bars[P::B_S + t * SB + j % SB]);
                }
                tc_commit(&bars[P::B_KF + j % KST]);
            };
            if (n > 0) ok = mbar_wait_warp(&bars[P::B_Q + t], 0, abort_flag, 206);
            for (int j = 0; j < SB && j < n_all && ok; ++j) issue_s(j);
#pragma unroll 1
            for (int j = 0; j < n_all && ok; ++j) {
                if (!(ok = mbar_wait_warp(&bars[P::B_V + j % VST], (j / VST) & 1, abort_flag, 208))) break;
                if (j < n) {
                    if (!(ok = mbar_wait_warp(&bars[P::B_P + t * SB + j % SB], (j / SB) & 1, abort_flag, 210))) break;
                    tc_fence_after();
                    const uint64_t bd = vd + (uint64_t)(((j % VST) * P::T_BYTES) >> 4);
#pragma unroll
                    for (int kk = 0; kk < PT_N / 16; ++kk)
                        tc_mma_ts(col_o, col_s + (j % SB) * PT_N + kk * 8, bd + (uint64_t)((kk * 2048) >> 4), IDESC_O, j || kk ? 1u : 0u);
                    tc_commit(&bars[P::B_O + 4 * t + (j & 3)]);
                }
                tc_commit(&bars[P::B_VF + j % VST]);
                if (j + SB < n_all) issue_s(j + SB);
            }
            // nothing of this CTA may be in flight when its memory goes
            tc_commit(&bars[P::B_END + t]);
            for (uint32_t i = 0; i < TC_SPIN_LIMIT && !__all_sync(0xffffffffu, mbar_try(&bars[P::B_END + t], 0)); ++i) {}
        } else {
            // =============================================================== packed rows and scales of K (V): a bulk copy for every run of keys in one page of which
            // some row of the CTA sees a key (pages in front of the window may be gone)
            const bool is_k = warp == P::LOAD_WARP;
            if (paged_pad_any(a, seq, b)) paged_pad(paged_pad_rows(a, seq, b, h), (long long)(qb * splits + split) * 64 + (tid & 63), (long long)n_qblocks * splits * 64);
            const int bits = is_k ? a.c.kb : a.c.vb, row = D / 8 * bits, run = min(PT_N, page_mask + 1), last_key = max(seq.kv - 1, 0);
            const unsigned char* pool = reinterpret_cast<const unsigned char*>(is_k ? a.c.kc : a.c.vc);
            const float* scales = is_k ? a.c.ks : a.c.vs;
            unsigned char* raw_stages = smem + (is_k ? P::OFF_RK : P::OFF_RV);
            uint64_t *raw_full = bars + (is_k ? P::B_RK : P::B_RV), *raw_freed = bars + (is_k ? P::B_RKF : P::B_RVF);
            auto page_of = [&](int i) { return __ldg(table + (min(tiles.key(tile0 + min(i, n_all - 1)) + lane * run, last_key) >> a.c.page_shift)); };
            int page = n_all > 0 ? page_of(0) : 0, j = 0;
#pragma unroll 1
            for (; j < n_all; ++j) {
                const int st = j % P::RST, key = tiles.key(tile0 + j) + lane * run;
                const int next = page_of(j + 1);
                if (j >= P::RST && !mbar_wait_warp(&raw_freed[st], (j / P::RST - 1) & 1, abort_flag, is_k ? 213 : 214)) break;
                const bool there = lane * run < PT_N && key < seq.kv && (key + run > tiles.first || key < a.sinks);
                const int runs = __popc(__ballot_sync(0xffffffffu, there));
                if (lane == 0) mbar_expect_tx(&raw_full[st], (uint32_t)(runs * run * (row + 4)));
                __syncwarp();
                if (there) {
                    const uint32_t own = (uint32_t)((paged_page(a, page, status) * a.c.H + h) << a.c.page_shift) + (key & page_mask);
                    unsigned char* raw = raw_stages + st * P::RAW_BYTES;
                    bulk_copy_g2s(raw + lane * run * row, pool + (size_t)own * row, (uint32_t)(run * row), &raw_full[st]);
                    bulk_copy_g2s(raw + P::R_BYTES + lane * run * 4, scales + own, (uint32_t)(run * 4), &raw_full[st]);
                }
                page = next;
            }
            // no copy of this CTA may be in flight when its memory goes
            for (int i = max(j - P::RST, 0); i < j; ++i)
                for (uint32_t n = 0; n < TC_SPIN_LIMIT && !__all_sync(0xffffffffu, mbar_try(&raw_full[i % P::RST], (i / P::RST) & 1)); ++n) {}
        }
    }
    __syncthreads();
    if (warp == P::MMA_WARP) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)P::TMEM_COLS) : "memory");
    }
}

template <int D> int launch_tc(const PagedAttnArgs& a, int n_qblocks, int splits, float* ws_o, float* ws_ml, int* status, cudaStream_t st) {
    using P = PtPlan<D>;
    static bool configured[64] = {false};
    int dev = 0;
    VARQ_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        VARQ_CUDA_TRY(cudaFuncSetAttribute(paged_attn_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, P::SMEM));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    const long long blocks = (long long)a.B * a.c.H * n_qblocks * splits;
    if (blocks > 0x7fffffffLL) return fail(VARQ_ERR_UNSUPPORTED, "varq_paged_attn: more than 2^31 thread blocks");
    VARQ_CUDA_TRY(launch_pdl(paged_attn_tc_kernel<D>, (unsigned)blocks, P::THREADS, P::SMEM, st, 1, a, n_qblocks, splits, ws_o, ws_ml, status));
    count_launches(1);
    return VARQ_OK;
}

}  // namespace

int paged_attn_tc_run(const PagedAttnArgs& a, int splits, float* ws_o, float* ws_ml, int* status, cudaStream_t st) {
    const int n_qblocks = (int)(((long long)a.max_q * a.G + 2 * PT_M - 1) / (2 * PT_M));
    return a.c.D == 64 ? launch_tc<64>(a, n_qblocks, splits, ws_o, ws_ml, status, st) : launch_tc<128>(a, n_qblocks, splits, ws_o, ws_ml, status, st);
}
int paged_attn_tc_status(int* out) { return tc_file_status(out); }

}  // namespace varq
