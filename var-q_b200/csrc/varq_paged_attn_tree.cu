// Attention of trees of drafted tokens over a paged cache, on the 5th-generation tensor cores.
//
// The arithmetic of a tile of 64 keys is the chunk kernel's (varq_paged_attn_tc.cu: what P, m, l and O are, what is rounded): conversion to fp16 tiles, products, softmax on
// tensor memory by the same roles.  One CTA = one (sequence, head of the cache) x up to 256 rows x part of the keys.  What differs:
//
// * A draft has few rows to a head of the cache, often no more than one tile of 128.  Then both groups of softmax warps have the same rows and take every other tile of
//   keys, an accumulator each, merged on tensor memory at the end; with more rows each group has a tile of 128 of its own.  Warps without a row skip the exponentials.
// * A query sees the context by its own position (window, first tokens) and of the drafted tokens those of its row of bits.  Tiles with drafted tokens or an end of a
//   window take the form with masks; there a lane makes the bits of one row of its warp, and the threads that hold the row's scores get them by shuffles.
// * Contexts and drafts differ, and the CTAs of the sequences with most work begin first where a call has more CTAs than SMs.
//
// What bounds it (B200): the softmax warps' chain, 2500 cycles for a tile of 64 keys (450 instructions; its 64 exponentials take 512 of them), which two warps on a scheduler
// do not fill, and about 15000 cycles of a CTA around its tiles (lengths, queries, the first tile's copies and conversion, the output).  32 sequences, drafts of 64, 2000 to 8000
// keys, 32 query / 8 cache heads x 128, 8 bits: 223 us, 765 TFLOP/s (102 us at the dense rate, 58 by bytes); the chunk kernel with masks looked up by each thread took 304.
// Drafts of 26 of 16 sequences, window 1024, groups of five heads: 40 us (52); drafts of 32 (one tile of rows), 16 sequences of 1000 to 4000 keys: 63 us (78).  (Times of replayed
// graphs, without the masks' launch.  Called one by one, the masks among them, the first takes 236 to 250 us, 683 TFLOP/s, the second 42.)
// On the way (us for the first and the second): two groups over one tile of rows, bits by lane 256 / 48; the form with masks a loop 233 / 43; queries by a thread per row
// through their own places in shared memory 224 / 40 (by registers and shuffles 11000 cycles of a CTA, so 6000).  Turned down: equal pieces of all sequences' tiles
// for 148 CTAs that stay, whatever the lengths, 283 / 81: the parts' store and merge and the list of a CTA's items cost more than the last wave; both chunks' scores first,
// then both chunks' weights 257 / 46; the output through shared memory, so that a store covers whole rows (64 rows of a head, 32 sequences of up to 3000 keys, 12 heads x 64:
// 80, with it 84: what runs once costs its instructions).
#include "varq_paged_attn_tc.cuh"

#include <climits>

namespace varq {
namespace {

template <int D> struct TrPlan {
    static constexpr int SB = D == 64 ? 3 : 2;                     // score tiles of a group
    static constexpr int KST = D == 64 ? 4 : 3, VST = KST;         // stages of K and V as fp16
    static constexpr int RST = D == 64 ? 6 : 3;                    // stages of K and V as they lie in the pages
    // Tables: tile j's is written once K's stage of tile j - KST is free, so both groups have asked for that tile's scores, each behind the weights of all its tiles up to
    // 2 SB before it: what is 2 SB + KST tiles old is not read any more
    static constexpr int TS = KST + 2 * SB;
    static constexpr int Q_BYTES = PT_M * D * 2, T_BYTES = PT_N * D * 2, R_BYTES = PT_N * D, RAW_BYTES = R_BYTES + PT_N * 4;     // packed rows, then scales
    static constexpr int TAB_FLOATS = 3 * PT_N;
    static constexpr int OFF_Q = 0, OFF_K = OFF_Q + 2 * Q_BYTES, OFF_V = OFF_K + KST * T_BYTES, OFF_RK = OFF_V + VST * T_BYTES, OFF_RV = OFF_RK + RST * RAW_BYTES,
                         OFF_TAB = OFF_RV + RST * RAW_BYTES;
    // barriers: K, V written and free; packed K, V there and free; tables written; queries; S, P of every score tile; O (a ring of four tiles); end
    static constexpr int B_K = 0, B_KF = B_K + KST, B_V = B_KF + KST, B_VF = B_V + VST, B_RK = B_VF + VST, B_RKF = B_RK + RST, B_RV = B_RKF + RST, B_RVF = B_RV + RST,
                         B_TAB = B_RVF + RST, B_Q = B_TAB + TS, B_S = B_Q + 2, B_P = B_S + 2 * SB, B_O = B_P + 2 * SB, B_END = B_O + 8, N_BARS = B_END + 2;
    static constexpr int OFF_BAR = OFF_TAB + TS * TAB_FLOATS * 4;
    static constexpr int OFF_QF = (OFF_BAR + N_BARS * 8 + 15) / 16 * 16;              // factors of the queries [2][128]
    static constexpr int OFF_ML = OFF_QF + 2 * PT_M * 4;                              // reference and sum of the two groups' rows [2][128][2]
    static constexpr int OFF_MISC = OFF_ML + 2 * PT_M * 8, SMEM = OFF_MISC + 32 + 1024;
    static constexpr int COL_O = 0, COL_S = 2 * D, TMEM_COLS = 512;
    static_assert(COL_S + 2 * SB * PT_N <= TMEM_COLS && SMEM <= 227 * 1024 && OFF_RK % 128 == 0, "plan");
    static constexpr int SOFT = 8, K_WARP0 = SOFT, V_WARP0 = K_WARP0 + 4, MMA_WARP = V_WARP0 + 4, LOAD_WARP = MMA_WARP + 2, THREADS = (LOAD_WARP + 2) * 32;
    static constexpr int REGS = 96, REGS_SOFT = 144, REGS_CONV = 72, REGS_MISC = 48;
    static_assert(SOFT * 32 * REGS_SOFT + 256 * REGS_CONV + 128 * REGS_MISC <= THREADS * REGS, "register plan");
};

__device__ __forceinline__ void pair_sync(int quarter) { asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory"); }      // the two warps that share rows

template <int D>
__global__ void __launch_bounds__(TrPlan<D>::THREADS, 1) paged_attn_tree_kernel(PagedAttnArgs a, int n_qblocks, int splits, int ranked, float* ws_o, float* ws_ml, int* status) {
    using P = TrPlan<D>;
    constexpr int KST = P::KST, VST = P::VST, TS = P::TS, SB = P::SB;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + P::OFF_BAR);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + P::OFF_MISC);
    int* my_seq = reinterpret_cast<int*>(smem + P::OFF_MISC + 16);          // its number; starts and length
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
    // ---- what this CTA does: sequences by rank, then heads, row blocks, parts
    const int split = (int)(blockIdx.x % (unsigned)splits);
    const unsigned item = blockIdx.x / (unsigned)splits, per_seq = (unsigned)(a.c.H * n_qblocks);
    const int rank = (int)(item / per_seq), hq = (int)(item - rank * per_seq), h = hq / n_qblocks, row0 = (hq - h * n_qblocks) * (2 * PT_M);
    if (warp == 0 && ranked) {
        PagedGiven given;
        const int b = paged_ranked(a, rank, 2 * PT_M, given);
        if (lane == 0) { my_seq[0] = b; my_seq[1] = given.s0; my_seq[2] = given.s1; my_seq[3] = given.kv; }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();       // behind the allocation: a CTA of a next launch must not take tensor memory that one of this launch still asks for
    const uint32_t tmem_base = *tmem_slot;
    const int b = ranked ? my_seq[0] : rank, page_mask = (1 << a.c.page_shift) - 1;
    const PagedSeq seq = paged_seq(a, ranked ? PagedGiven{my_seq[1], my_seq[2], my_seq[3]} : paged_given(a, b), status);
    const int rows = seq.nq * a.G, p_first = seq.kv - seq.nq;               // rows of the (sequence, head); position of the first drafted token
    const bool both = rows - row0 > PT_M;                                   // each group has rows of its own
    PtTiles tiles;
    int n = 0, tile0 = 0;                                                   // key tiles of this CTA
    {
        tiles.first = paged_window(a, p_first - 1);
        tiles.lo = tiles.first & ~(PT_N - 1);
        tiles.ns = min((a.sinks + PT_N - 1) / PT_N, tiles.lo / PT_N);
        tiles.n = seq.kv > 0 ? tiles.ns + (seq.kv - tiles.lo + PT_N - 1) / PT_N : 0;
        tile0 = (int)((long long)tiles.n * split / splits);
        if (row0 < rows) n = (int)((long long)tiles.n * (split + 1) / splits) - tile0;
    }

    if (warp < P::SOFT) {
        // =============================================================== softmax, epilogue
        set_registers<P::REGS_SOFT, P::REGS>();
        const int t = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane, g = lane >> 2, cq = lane & 3;
        const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16), col_s0 = lane_base + P::COL_S + t * (SB * PT_N), col_o = lane_base + P::COL_O + t * D;
        bool ok = true, scaled = false;
        const int row_t = row0 + (both ? t * PT_M : 0), row_w = row_t + quarter * 32, n_own = both ? n : (n + 1 - t) >> 1;
        const bool busy = row_w < rows;                                     // this warp has rows
        // ---- queries -> fp16 in shared memory, in the order in which the codes of K are unpacked; with 128 rows or less both groups have the same ones.  A thread copies its
        // row to its place and changes it there: this code runs once, where every instruction counts (by registers and shuffles it took 11000 cycles of a CTA)
        if (row0 < rows) {
            if (busy) {
                const bool live = row_t + r < rows, bf16 = a.dtype == VARQ_BF16;
                const int at = min(row_t + r, rows - 1), token = at / a.G, head = h * a.G + at - token * a.G;
                const unsigned short* const src = reinterpret_cast<const unsigned short*>(a.q) + (long long)(seq.q0 + token) * a.qs_t + (long long)head * a.qs_h;
                unsigned char* const qs = smem + P::OFF_Q + t * P::Q_BYTES;
                if (__all_sync(0xffffffffu, (reinterpret_cast<uintptr_t>(src) & 15u) == 0)) {
                    const int size = live ? 16 : 0;
#pragma unroll
                    for (int i = 0; i < D / 8; ++i)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(qs + pt_chunk<PT_M>(r, i))), "l"(src + 8 * i), "r"(size) : "memory");
                    asm volatile("cp.async.wait_all;" ::: "memory");
                } else {
#pragma unroll 1
                    for (int i = 0; i < D; ++i)
                        reinterpret_cast<unsigned short*>(qs + pt_chunk<PT_M>(r, i >> 3))[i & 7] = live ? __ldg(src + i) : (unsigned short)0;
                }
                float f = 1.f, back = 1.f;
                if (bf16) {
                    uint32_t top = 0;                                        // bits of the largest absolute value, of the even and the odd elements
#pragma unroll 4
                    for (int i = 0; i < D / 8; ++i) {
                        const uint4 u = *reinterpret_cast<const uint4*>(qs + pt_chunk<PT_M>(r, i));
                        top = __vmaxu2(top, __vmaxu2(__vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu), __vmaxu2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu)));
                    }
                    const int ex = (int)(max(top & 0xffffu, top >> 16) >> 7);      // exponent: 2^(ex - 127)
                    if (top && (ex < 123 || ex > 141)) {                     // -> largest element in [2^8, 2^9); NaN and infinity stay what they are
                        const int e = min(max(ex, 40), 240);
                        f = __uint_as_float((uint32_t)(262 - e) << 23);
                        back = __uint_as_float((uint32_t)(e - 8) << 23);
                    }
                    scaled = __any_sync(0xffffffffu, f != 1.f);
                    if (scaled) reinterpret_cast<float*>(smem + P::OFF_QF)[t * PT_M + r] = back;
                }
                if (bf16 || a.c.kb != 8) {
#pragma unroll 2
                    for (int i = 0; i < D / 8; i += 2) {
                        uint4 *const p0 = reinterpret_cast<uint4*>(qs + pt_chunk<PT_M>(r, i)), *const p1 = reinterpret_cast<uint4*>(qs + pt_chunk<PT_M>(r, i + 1));
                        const uint4 u0 = *p0, u1 = *p1;
                        uint32_t w[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
                        if (bf16) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) w[j] = pack_half2(__uint_as_float(w[j] << 16) * f, __uint_as_float(w[j] & 0xffff0000u) * f);
                        }
                        q_operand_order(w, a.c.kb);
                        *p0 = make_uint4(w[0], w[1], w[2], w[3]);
                        *p1 = make_uint4(w[4], w[5], w[6], w[7]);
                    }
                }
                __syncwarp();
            }
            fence_async_smem();
            warp_arrive(&bars[P::B_Q + t], lane);
            const int all_hi = p_first, all_lo = paged_window(a, p_first + seq.nq - 1);      // keys between which every row sees everything
            // for tiles with masks: row `lane` of the warp's 32, its token and the first key of its window
            const int m_token = seq.q0 + min(row_t + r, rows - 1) / a.G, m_lo = a.window ? paged_window(a, paged_tree_position(a, m_token, p_first, seq.nq)) : 0;
            // A thread holds, of every eight columns of S, two of the rows g, g + 8, g + 16, g + 24 of its warp's 32
            pair nm[4] = {0ull, 0ull, 0ull, 0ull};                          // minus the reference, twice
            pair l[4] = {0ull, 0ull, 0ull, 0ull};
            unsigned unset = 15u;                                           // rows that have no reference yet: they have seen no key
            auto by_lane = [&](const float (&v)[4]) {                        // rows g + 8 i of a thread -> row `lane`
                float o = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) { const float y = __shfl_sync(0xffffffffu, v[i], (lane & 7) * 4); o = (lane >> 3) == i ? y : o; }
                return o;
            };
#pragma unroll 1
            for (int own = 0; own < n_own; ++own) {
                const int j = both ? own : 2 * own + t, slot = own % SB, key0 = tiles.key(tile0 + j);
                {
                    uint64_t *tab_bar = &bars[P::B_TAB + j % TS], *s_bar = &bars[P::B_S + t * SB + slot];
                    const bool there = mbar_test(tab_bar, (j / TS) & 1) & mbar_test(s_bar, (own / SB) & 1);        // both at once: that is a round trip less
                    if (!__all_sync(0xffffffffu, there))
                        ok = mbar_wait_warp(tab_bar, (j / TS) & 1, abort_flag, 221) && mbar_wait_warp(s_bar, (own / SB) & 1, abort_flag, 222);
                    if (!ok) break;
                }
                if (busy) {
                    const uint32_t col_s = col_s0 + slot * PT_N;
                    tc_fence_after();
                    const float* tab = reinterpret_cast<const float*>(smem + P::OFF_TAB) + (j % TS) * P::TAB_FLOATS;
                    // Two forms of a tile.  The usual one carries neither masks nor factors nor new references, and nothing of them lies between its instructions: a CTA's roles
                    // share the instruction cache, and a warp that is alone on its scheduler waits for every line of it.  The other one is a loop over the two chunks.
                    // x - m of 32 columns: [half of the rows][eight columns][row g, g + 8]; true where a row needs another reference
                    auto scores = [&](auto special_, pair (&x)[16], int c) -> bool {
                        constexpr bool SPECIAL = decltype(special_)::value != 0;
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
                            // bit k: key k of the chunk is seen by row `lane`; then by the thread's rows, from its first column on
                            auto below = [](int k) { return k <= 0 ? 0u : k >= 32 ? ~0u : (1u << k) - 1u; };
                            const int c0 = key0 + 32 * c;
                            const uint32_t sees = below(seq.kv - c0) & (~below(m_lo - c0) | below(a.sinks - c0)) & paged_tree_bits(a, m_token, c0 - p_first);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t m = __shfl_sync(0xffffffffu, sees, g + 8 * i) >> (2 * cq);
#pragma unroll
                                for (int v = 0; v < 4; ++v) {
                                    pair& y = x[(i >> 1) * 8 + v * 2 + (i & 1)];
                                    y = pair_of(m >> (8 * v) & 1u ? pair_x(y) : -INFINITY, m >> (8 * v + 1) & 1u ? pair_y(y) : -INFINITY);
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
                    auto raise = [&](auto sp_, pair (&x)[16], int c) {
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
                        if (own > 0) {                                 // behind the products of the tile before
                            ok = __all_sync(0xffffffffu, mbar_wait(&bars[P::B_O + 4 * t + ((own - 1) & 3)], ((own - 1) >> 2) & 1, abort_flag, 223));
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
                        scores(sp_, x, c);
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
                    auto tile = [&](auto sp) {
                        pair xa[16], xb[16];
                        if (scores(sp, xa, 0)) raise(sp, xa, 0);
                        const bool other = scores(sp, xb, 1);
                        weights(xa, 0);
                        if (other) raise(sp, xb, 1);
                        weights(xb, 1);
                    };
                    if (scaled || key0 + PT_N > all_hi || (key0 < all_lo && key0 + PT_N > a.sinks)) {
#pragma unroll 1
                        for (int c = 0; c < 2; ++c) {
                            pair x[16];
                            if (scores(IntC<1>(), x, c)) raise(IntC<1>(), x, c);
                            weights(x, c);
                        }
                    } else tile(IntC<0>());
                    if (!ok) break;
                    tmem_wait_st();
                    tc_fence_before();
                }
                warp_arrive(&bars[P::B_P + t * SB + slot], lane);
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
            // ---- O / l, or this split's part.  Where the groups share rows each merges both accumulators on half of the columns (the pair meets whatever happened)
            if (ok && n_own > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars[P::B_O + 4 * t + ((n_own - 1) & 3)], ((n_own - 1) >> 2) & 1, abort_flag, 223));
            float w_own = 1.f, w_other = 0.f;
            int c_lo = 0, c_hi = D;
            bool other = false;                                             // the other group has an accumulator of these rows
            if (!both) {
                float2* ml = reinterpret_cast<float2*>(smem + P::OFF_ML);
                ml[t * PT_M + r] = make_float2(row_m, row_l);
                tc_fence_before();
                pair_sync(quarter);
                const float2 o = ml[(1 - t) * PT_M + r];
                other = t ? n > 0 : n > 1;
                if (other) {
                    const float m = fmaxf(row_m, o.x);
                    w_own = ex2(row_m - m); w_other = ex2(o.x - m);
                    row_l = fmaf(w_own, row_l, w_other * o.y);
                    row_m = m;
                }
                c_lo = t * (D / 2); c_hi = c_lo + D / 2;
            }
            tc_fence_after();
            const int row = row_t + r;
            const bool live = row < rows;
            if (ok && busy) {
                const int token = live ? row / a.G : 0, head = h * a.G + (live ? row - token * a.G : 0);
                const float inv = row_l != 0.f ? 1.f / row_l : 0.f;         // (a NaN stays one)
                const long long out_row = (long long)(seq.q0 + token) * a.Hq + head, oo = (long long)(seq.q0 + token) * a.os_t + head * a.os_h;
                const long long part_row = (long long)split * ((long long)a.T * a.Hq) + out_row;
                if (splits == 1) { w_own *= inv; w_other *= inv; }
                const uint32_t col_other = lane_base + P::COL_O + (1 - t) * D;
#pragma unroll 1
                for (int c = c_lo; c < c_hi; c += 16) {
                    uint32_t o[16];
                    float y[16];
                    if (n_own > 0) tmem_ld16(col_o + c, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] = n_own > 0 ? __uint_as_float(o[i]) * w_own : 0.f;
                    if (other) {
                        tmem_ld16(col_other + c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) y[i] = fmaf(__uint_as_float(o[i]), w_other, y[i]);
                    }
                    float v[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = a.c.vb == 8 ? y[i] : a.c.vb == 4 ? y[code_pos(4, i)] : y[code_pos(2, i)];
                    if (!live) continue;
                    if (splits > 1) {
                        float4* to = reinterpret_cast<float4*>(ws_o + part_row * D + c);
#pragma unroll
                        for (int i = 0; i < 4; ++i) to[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                    } else {
                        uint32_t h[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const __nv_bfloat162 b2 = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                            h[i] = a.dtype == VARQ_F16 ? pack_half2(v[2 * i], v[2 * i + 1]) : *reinterpret_cast<const uint32_t*>(&b2);
                        }
                        unsigned short* to = reinterpret_cast<unsigned short*>(a.out) + oo + c;
                        if ((reinterpret_cast<uintptr_t>(to) & 15u) == 0) {
                            reinterpret_cast<uint4*>(to)[0] = make_uint4(h[0], h[1], h[2], h[3]);
                            reinterpret_cast<uint4*>(to)[1] = make_uint4(h[4], h[5], h[6], h[7]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i) to[i] = (unsigned short)(h[i >> 1] >> (16 * (i & 1)));
                        }
                    }
                }
                if (live && c_lo == 0) {
                    if (splits > 1) *reinterpret_cast<float2*>(ws_ml + part_row * 2) = make_float2(row_m, row_l);
                    else if (a.lse) a.lse[out_row] = row_l != 0.f ? (row_m + __log2f(row_l)) * 0.6931471805599453f : -INFINITY;
                }
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
                for (int j = 0; j < n; ++j) {
                    const int k = kq + 32 * it;
                    if (!mbar_wait_warp(&raw_full[rst], rst_ph, abort_flag, is_k ? 231 : 232)) break;
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
                    if (j >= KST && !mbar_wait_warp(&freed[st], st_ph, abort_flag, is_k ? 224 : 225)) break;
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
            // =============================================================== products of group t (the whole warp waits; one elected lane issues)
            // Of the tiles those of the group: S of the first ones, then for every tile j: P(j) -> O += P(j) V(j) -> S of the tile as far ahead as score tiles
            // reach, over the columns of P(j).  The other tiles are let go as soon as they are there.
            constexpr uint32_t IDESC_S = instr_desc(PT_M, PT_N, 0), IDESC_O = instr_desc(PT_M, D, 1);
            const int t = warp - P::MMA_WARP;
            const uint64_t qd = smem_desc(smem_u32(smem + P::OFF_Q + t * P::Q_BYTES), 16, 1024), kd = smem_desc(smem_u32(smem + P::OFF_K), 16, 1024);
            const uint64_t vd = smem_desc(smem_u32(smem + P::OFF_V), PT_N * 128, 1024);
            const uint32_t col_s = tmem_base + P::COL_S + t * (SB * PT_N), col_o = tmem_base + P::COL_O + t * D;
            bool ok = true;
            int s_own = 0, o_own = 0;                                       // tiles of the group whose S, O are issued
            const int ahead = both ? SB : 2 * SB;
            auto issue_s = [&](int j) {
                if (!(ok = mbar_wait_warp(&bars[P::B_K + j % KST], (j / KST) & 1, abort_flag, 227))) return;
                if (!both && (j & 1) != t) {
                    if (lane == 0) mbar_arrive(&bars[P::B_KF + j % KST]);
                    return;
                }
                tc_fence_after();
                const uint64_t bd = kd + (uint64_t)(((j % KST) * P::T_BYTES) >> 4);
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    tc_mma_ss(col_s + (s_own % SB) * PT_N, qd + (uint64_t)(((kk >> 2) * (PT_M * 128) + (kk & 3) * 32) >> 4),
                              bd + (uint64_t)(((kk >> 2) * (PT_N * 128) + (kk & 3) * 32) >> 4), IDESC_S, kk ? 1u : 0u);
                tc_commit(&bars[P::B_S + t * SB + s_own % SB]);
                tc_commit(&bars[P::B_KF + j % KST]);
                ++s_own;
            };
            if (n > 0) ok = mbar_wait_warp(&bars[P::B_Q + t], 0, abort_flag, 226);
            for (int j = 0; j < ahead && j < n && ok; ++j) issue_s(j);
#pragma unroll 1
            for (int j = 0; j < n && ok; ++j) {
                if (!(ok = mbar_wait_warp(&bars[P::B_V + j % VST], (j / VST) & 1, abort_flag, 228))) break;
                if (both || (j & 1) == t) {
                    if (!(ok = mbar_wait_warp(&bars[P::B_P + t * SB + o_own % SB], (o_own / SB) & 1, abort_flag, 230))) break;
                    tc_fence_after();
                    const uint64_t bd = vd + (uint64_t)(((j % VST) * P::T_BYTES) >> 4);
#pragma unroll
                    for (int kk = 0; kk < PT_N / 16; ++kk)
                        tc_mma_ts(col_o, col_s + (o_own % SB) * PT_N + kk * 8, bd + (uint64_t)((kk * 2048) >> 4), IDESC_O, o_own || kk ? 1u : 0u);
                    tc_commit(&bars[P::B_O + 4 * t + (o_own & 3)]);
                    tc_commit(&bars[P::B_VF + j % VST]);
                    ++o_own;
                } else if (lane == 0) mbar_arrive(&bars[P::B_VF + j % VST]);
                if (j + ahead < n) issue_s(j + ahead);
            }
            // nothing of this CTA may be in flight when its memory goes
            tc_commit(&bars[P::B_END + t]);
            for (uint32_t i = 0; i < TC_SPIN_LIMIT && !__all_sync(0xffffffffu, mbar_try(&bars[P::B_END + t], 0)); ++i) {}
        } else {
            // =============================================================== packed rows and scales of K (V): a bulk copy for every run of keys in one page of which
            // some row sees a key (pages in front of the window may be gone)
            const bool is_k = warp == P::LOAD_WARP;
            const int bits = is_k ? a.c.kb : a.c.vb, row = D / 8 * bits, run = min(PT_N, page_mask + 1);
            const unsigned char* pool = reinterpret_cast<const unsigned char*>(is_k ? a.c.kc : a.c.vc);
            const float* scales = is_k ? a.c.ks : a.c.vs;
            unsigned char* raw_stages = smem + (is_k ? P::OFF_RK : P::OFF_RV);
            uint64_t *raw_full = bars + (is_k ? P::B_RK : P::B_RV), *raw_freed = bars + (is_k ? P::B_RKF : P::B_RVF);
            if (paged_pad_any(a, seq, b)) paged_pad(paged_pad_rows(a, seq, b, h), (long long)(row0 / (2 * PT_M) * splits + split) * 64 + (tid & 63), (long long)n_qblocks * splits * 64);
            const int32_t* table = a.table + b * a.table_stride;
            auto page_of = [&](int i) { return __ldg(table + (min(tiles.key(tile0 + min(i, n - 1)) + lane * run, seq.kv - 1) >> a.c.page_shift)); };
            int page = n > 0 ? page_of(0) : 0, j = 0;
#pragma unroll 1
            for (; j < n; ++j) {
                const int st = j % P::RST, key = tiles.key(tile0 + j) + lane * run;
                const int next = page_of(j + 1);
                if (j >= P::RST && !mbar_wait_warp(&raw_freed[st], (j / P::RST - 1) & 1, abort_flag, is_k ? 233 : 234)) break;
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

template <int D> int launch_tree(const PagedAttnArgs& a, int n_qblocks, int splits, float* ws_o, float* ws_ml, int* status, cudaStream_t st) {
    using P = TrPlan<D>;
    static bool configured[64] = {false};
    int dev = 0;
    VARQ_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        VARQ_CUDA_TRY(cudaFuncSetAttribute(paged_attn_tree_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, P::SMEM));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    const long long blocks = (long long)a.B * a.c.H * n_qblocks * splits;
    if (blocks > 0x7fffffffLL) return fail(VARQ_ERR_UNSUPPORTED, "varq_paged_attn: more than 2^31 thread blocks");
    const int ranked = a.B > 1 && a.B <= PAGED_RANKED && blocks > sm_count();
    VARQ_CUDA_TRY(launch_pdl(paged_attn_tree_kernel<D>, (unsigned)blocks, P::THREADS, P::SMEM, st, 1, a, n_qblocks, splits, ranked, ws_o, ws_ml, status));
    count_launches(1);
    return VARQ_OK;
}

}  // namespace

int paged_attn_tree_run(const PagedAttnArgs& a, int splits, float* ws_o, float* ws_ml, int* status, cudaStream_t st) {
    const int n_qblocks = (int)(((long long)a.max_q * a.G + 2 * PT_M - 1) / (2 * PT_M));
    return a.c.D == 64 ? launch_tree<64>(a, n_qblocks, splits, ws_o, ws_ml, status, st) : launch_tree<128>(a, n_qblocks, splits, ws_o, ws_ml, status, st);
}
int paged_attn_tree_status(int* out) { return tc_file_status(out); }

}  // namespace varq
